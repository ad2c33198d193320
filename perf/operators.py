"""Measured cases of three operators of a transformer block over long token sequences:

  attention  softmax attention inside a sliding window, with a few first tokens that stay visible (grouped heads, padded batches), forward, backward
             and for single tokens against a long cache
  rope       rotary positions with several axes (time, height, width) on queries and keys, and the transposed map for their gradients
  norm       the norm behind a block, its gate and the scaled residual sum, and the norm in front of the next block, forward and backward

With ``own`` False a pass computes the plain form (elementary torch operations in 32 bits, rounded once at the end); with ``own`` True it makes the calls that
a user of ``smb_vision_amd.ops`` makes.  ``exact`` restates the definitions in 64 bits, apart from both.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------------------------------------------------------------------------ the cases
def _attn(name, mode, dtype, B, Sq, Sk, H, Hk, D, left, right, sinks, ragged=False):
    return {"name": name, "op": "attention", "mode": mode, "dtype": dtype, "B": B, "Sq": Sq, "Sk": Sk, "H": H, "Hk": Hk, "D": D, "left": left, "right": right,
            "sinks": sinks, "ragged": ragged}


def _rope(name, mode, dtype, B, S, H, Hk, D, pairs, axes, interleaved, far):
    return {"name": name, "op": "rope", "mode": mode, "dtype": dtype, "B": B, "S": S, "H": H, "Hk": Hk, "D": D, "pairs": pairs, "axes": axes,
            "interleaved": interleaved, "far": far}


def _norm(name, mode, dtype, stream, rows, d, gates, post, pre, res_scale):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "stream": stream, "rows": rows, "d": d, "gates": gates, "post": post, "pre": pre,
            "res_scale": res_scale}


def listed():
    return [
        # one token of one short sequence against its cache, ViT-base heads: the smallest call, where latency counts
        _attn("attention_token_short", "infer", "bf16", 1, 1, 577, 12, 12, 64, 255, 0, 4),
        # one token each of 16 sequences against long caches of uneven length, grouped heads: a serving step
        _attn("attention_token_batch", "infer", "bf16", 16, 1, 16384, 32, 8, 128, 8191, 0, 4, True),
        # an odd piece of a prompt appended to an odd cache, fp16
        _attn("attention_append_odd", "infer", "fp16", 2, 333, 4001, 16, 4, 80, 1500, 0, 7, True),
        # embedding export of one 512 x 512 x 320 volume: 20,480 tokens, ViT-base heads, a window to both sides and a few register tokens
        _attn("attention_volume_infer", "infer", "bf16", 1, 20480, 20480, 12, 12, 64, 1024, 1024, 8),
        # the same tokens through a training step of the decoder (6 heads of 64)
        _attn("attention_volume_train", "train", "bf16", 1, 20480, 20480, 6, 6, 64, 2048, 2048, 8),
        # a padded batch of uneven sequences, causal window, grouped heads of 128: a language model's training step
        _attn("attention_ragged_train", "train", "bf16", 4, 4093, 4093, 16, 4, 128, 1023, 0, 4, True),
        # queries and keys of the volume's 20,480 tokens on the (20, 32, 32) grid of bricks, ViT-base heads, on the way to the attention
        _rope("rope_volume", "forward", "bf16", 1, 20480, 12, 12, 64, 32, 3, False, False),
        # their gradients on the way back, grouped heads, interleaved pairs, part of the channels left as they are, odd length, fp32, far positions
        _rope("rope_odd_grad", "transpose", "fp32", 3, 1999, 16, 4, 80, 30, 3, True, True),
        # the new tokens of 16 sequences: latency
        _rope("rope_token_batch", "forward", "bf16", 16, 1, 32, 8, 128, 64, 1, False, True),
        # the volume's tokens of a ViT-base training step: fp32 residual stream, LayerNorms on both sides, one gate
        _norm("norm_volume_train", "train", "bf16", "fp32", 20480, 768, 1, "layer", "layer", 1.0),
        # a language model's rows with RMS norms, a gate for each of 4 sequences, an odd width and a scaled residual
        _norm("norm_odd_train", "train", "bf16", "bf16", 4 * 1777, 1001, 4, "rms", "rms", 0.70710678),
        # the new tokens of 16 sequences: latency
        _norm("norm_token_batch", "infer", "fp16", "fp16", 16, 4096, 1, "rms", "rms", 1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    """One more case of the same ranges; one that would cost more than its operator's largest listed case is made shorter."""
    case = _draw(rng)
    most = [work(c) for c in listed() if c["op"] == case["op"]]
    most = {n: max(w[n] for w in most) for n in ("bytes", "flops")}
    while any(w > most[n] for n, w in work(case).items()):
        if case.get("B", 1) > 1:
            case["B"] = (case["B"] + 1) // 2
        elif case["op"] == "attention":
            case["Sq"], case["Sk"] = (case["Sq"] + 1) // 2, (case["Sk"] + 1) // 2
        elif case["op"] == "rope":
            case["S"] = (case["S"] + 1) // 2
        else:
            groups = max(1, case["gates"])
            case["rows"] = groups * ((case["rows"] // groups + 1) // 2)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(["token", "append", "infer", "train", "rope", "rope", "norm", "norm"])
    if kind in ("token", "append", "infer", "train"):
        D = rng.choice([32, 64, 64, 80, 128, 128, 8 * rng.randint(1, 16)])
        Hk = rng.choice([1, 2, 4, 6, 8])
        H = Hk * rng.choice([1, 1, 2, 3, 4, 8])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        sinks = rng.choice([0, 1, 4, 4, 16, 130])
        left = rng.choice([-1, _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)])
        ragged = rng.random() < 0.5
        if kind == "token":
            return _attn(None, "infer", dtype, _log_int(rng, 1, 32), 1, _log_int(rng, 1, 16384), H, Hk, D, left, 0, sinks, ragged)
        S = _log_int(rng, 1, 20480)
        B = _log_int(rng, 1, max(1, min(8, 20480 // S)))
        right = rng.choice([0, 0, _log_int(rng, 1, 2048), -1])
        if kind == "append":
            return _attn(None, "infer", dtype, B, _log_int(rng, 1, S), S, H, Hk, D, left, 0, sinks, ragged)
        if H * D > 1536:
            H = Hk
        return _attn(None, kind, dtype, B, S, S, H, Hk, D, left, right, sinks, ragged)
    if kind == "rope":
        D = rng.choice([32, 64, 80, 128, 2 * rng.randint(4, 80)])
        pairs = rng.choice([D // 2, D // 2, max(1, D // 3)])
        axes = min(rng.choice([1, 2, 3, 3, 4]), pairs)
        S = _log_int(rng, 1, 20480)
        Hk = rng.choice([1, 2, 4, 8])
        return _rope(None, rng.choice(["forward", "transpose"]), rng.choice(["bf16", "fp16", "fp32"]), _log_int(rng, 1, max(1, min(16, 20480 // S))), S,
                     Hk * rng.choice([1, 2, 3]), Hk, D, pairs, axes, rng.random() < 0.4, rng.random() < 0.5)
    gates = rng.choice([0, 1, 1, 2, 3, 16])
    rows = max(1, gates) * _log_int(rng, 1, 20480 // max(1, gates))
    d = rng.choice([768, 1024, 384, _log_int(rng, 8, 2048), _log_int(rng, 8, 4096)])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    return _norm(None, rng.choice(["infer", "train", "train"]), dtype, rng.choice([dtype, "fp32"]), rows, d, gates, rng.choice(["layer", "rms", "rms", "none"]),
                 rng.choice(["layer", "rms"]), rng.choice([1.0, 0.70710678]))


# -------------------------------------------------------------------------------------------------------------------------------------- inputs
def _lens(case):
    """Lengths of a ragged batch: a rule of the case alone, so that the work of a pass is known (the first sequence is the longest)."""
    B, Sk = case["B"], case["Sk"]
    if not case["ragged"]:
        return [Sk] * B, [case["Sq"]] * B
    k = [max(1, Sk - (b * 5 * Sk) // (8 * B) - (b % 3)) for b in range(B)]
    q = k if case["Sq"] == Sk else [min(case["Sq"], n) for n in k]
    return k, q


def _sections(pairs, axes):
    base = [pairs // axes] * axes
    base[0] += pairs - sum(base)
    return tuple(base)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed) * 2 + 1)
    dt = DTYPES[case["dtype"]]

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    if case["op"] == "attention":
        B, Sq, Sk, H, Hk, D = (case[n] for n in ("B", "Sq", "Sk", "H", "Hk", "D"))
        klen, qlen = _lens(case)
        st = {"case": case, "klen_host": klen, "qlen_host": qlen, "k_lens": None, "q_lens": None}
        if case["ragged"]:
            st["k_lens"] = torch.tensor(klen, dtype=torch.int32, device=dev)
            st["q_lens"] = torch.tensor(qlen, dtype=torch.int32, device=dev)
        if Sq == Sk and Sk > 1:
            # the output of one projection, split into heads without a copy
            packed = rnd(B, Sq, (H + 2 * Hk) * D)
            st["q"] = packed[..., :H * D].unflatten(-1, (H, D))
            st["k"] = packed[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
            st["v"] = packed[..., (H + Hk) * D:].unflatten(-1, (Hk, D))
        else:
            st["q"] = rnd(B, Sq, H, D)
            st["k"] = rnd(B, Sk, Hk, D)
            st["v"] = rnd(B, Sk, Hk, D)
        if case["mode"] == "train":
            st["do"] = rnd(B, Sq, H, D, scale=0.1)
        return st
    if case["op"] == "rope":
        B, S, H, Hk, D, P, A = (case[n] for n in ("B", "S", "H", "Hk", "D", "pairs", "axes"))
        idx = torch.arange(S, device=dev)
        side = 32
        axes = [idx // (side * side), (idx // side) % side, idx % side, idx % 7] if A > 1 else [idx]
        pos = torch.stack(axes[:A]).to(torch.int32)[:, None, :].repeat(1, B, 1)
        start = torch.randint(0, 1000000 if case["far"] else 64, (1, B, 1), generator=g, device=dev, dtype=torch.int32)
        pos[:1] += start
        inv = 10000.0 ** (-torch.arange(P, device=dev, dtype=torch.float64) / P)
        return {"case": case, "q": rnd(B, S, H, D), "k": rnd(B, S, Hk, D), "pos": pos.contiguous(), "inv_freq": inv.float(), "sections": _sections(P, A)}
    rows, d = case["rows"], case["d"]
    sdt = DTYPES[case["stream"]]
    st = {"case": case, "h": rnd(rows, d, scale=2.0), "x": rnd(rows, d, dtype=sdt), "post_w": None, "post_b": None, "pre_b": None, "gate": None,
          "pre_w": 1 + rnd(d, scale=0.1, dtype=torch.float32)}
    if case["post"] != "none":
        st["post_w"] = 1 + rnd(d, scale=0.1, dtype=torch.float32)
    if case["post"] == "layer":
        st["post_b"] = rnd(d, scale=0.1, dtype=torch.float32)
    if case["pre"] == "layer":
        st["pre_b"] = rnd(d, scale=0.1, dtype=torch.float32)
    if case["gates"]:
        st["gate"] = rnd(case["gates"], d, scale=0.5, dtype=torch.float32)
    if case["mode"] == "train":
        st["dx1"] = rnd(rows, d, dtype=sdt)
        st["dy"] = rnd(rows, d)
    return st


# ----------------------------------------------------------------------------------------------------------------------------------- the passes
def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _attention_own(state) if own else _attention_plain(state)
    if op == "rope":
        return _rope_own(state) if own else _rope_plain(state)
    return _norm_own(state) if own else _norm_plain(state)


def _attention_own(st):
    from smb_vision_amd import ops
    c = st["case"]
    kw = dict(left=c["left"], right=c["right"], sinks=c["sinks"], q_lens=st["q_lens"], k_lens=st["k_lens"])
    q, k, v = st["q"], st["k"], st["v"]
    if c["mode"] == "infer":
        return ops.window_attention_fwd(q, k, v, **kw)[0]
    o, lse, o_lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    return (o, *ops.window_attention_bwd(q, k, v, o, st["do"], lse, o_lo=o_lo, **kw))


def _rope_own(st):
    from smb_vision_amd import ops
    c = st["case"]
    return ops.rope_axes(st["q"], st["k"], st["pos"], st["inv_freq"], st["sections"], interleaved=c["interleaved"], transpose=c["mode"] == "transpose")


def _norm_own(st):
    from smb_vision_amd import ops
    c = st["case"]
    kw = dict(post=None if c["post"] == "none" else c["post"], post_w=st["post_w"], post_b=st["post_b"], gate=st["gate"], res_scale=c["res_scale"],
              pre=c["pre"], pre_w=st["pre_w"], pre_b=st["pre_b"])
    x1, y, stats = ops.gated_norm_fwd(st["h"], st["x"], eps=1e-6, **kw)
    if c["mode"] == "infer":
        return x1, y
    gr = ops.gated_norm_bwd(st["dx1"], st["dy"], st["h"], st["x"], stats, **kw)
    return [x1, y] + [gr[n] for n in ("dh", "dx", "gate", "post_w", "post_b", "pre_w", "pre_b") if gr[n] is not None]


def _band(case, i0, i1, klen, qlen):
    """Keys that the queries i0 .. i1 - 1 of one sequence can see: (first keys that stay, start and end of the window)."""
    shift = klen - qlen
    hi = klen if case["right"] < 0 else max(0, min(klen, i1 - 1 + shift + case["right"] + 1))
    lo = 0 if case["left"] < 0 else max(0, min(hi, i0 + shift - case["left"]))
    ns = min(case["sinks"], hi)
    if ns >= lo:
        return 0, 0, hi
    return ns, lo, hi


def _visible(case, qpos, keys):
    d = keys[None, :] - qpos[:, None]
    vis = torch.ones_like(d, dtype=torch.bool)
    if case["right"] >= 0:
        vis &= d <= case["right"]
    if case["left"] >= 0:
        vis &= (d >= -case["left"]) | (keys[None, :] < case["sinks"])
    return vis


def _attention_plain(st):
    c = st["case"]
    q, k, v = st["q"], st["k"], st["v"]
    B, Sq, H, D = q.shape
    Hk, G = k.shape[2], H // k.shape[2]
    scale = D ** -0.5
    train = c["mode"] == "train"
    o = torch.zeros(B, Sq, H, D, dtype=q.dtype, device=q.device)
    if train:
        dq = torch.zeros_like(o)
        dk = torch.zeros(B, k.shape[1], Hk, D, device=q.device)
        dv = torch.zeros_like(dk)
    step = 1024
    for b in range(B):
        klen, qlen = st["klen_host"][b], st["qlen_host"][b]
        for i0 in range(0, qlen, step):
            i1 = min(i0 + step, qlen)
            ns, lo, hi = _band(c, i0, i1, klen, qlen)
            if ns + hi - lo <= 0:
                continue
            n = i1 - i0
            keys = torch.cat([torch.arange(ns, device=q.device), torch.arange(lo, hi, device=q.device)])
            qf = q[b, i0:i1].float().view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
            if ns:
                kf = torch.cat([k[b, :ns], k[b, lo:hi]]).float().transpose(0, 1).contiguous()
                vf = torch.cat([v[b, :ns], v[b, lo:hi]]).float().transpose(0, 1).contiguous()
            else:
                kf, vf = k[b, lo:hi].float().transpose(0, 1).contiguous(), v[b, lo:hi].float().transpose(0, 1).contiguous()
            s = (torch.matmul(qf, kf.transpose(1, 2).contiguous()) * scale).view(Hk, G, n, -1)
            vis = _visible(c, torch.arange(i0, i1, device=q.device) + (klen - qlen), keys)
            s = s.masked_fill(~vis, float("-inf"))
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m.masked_fill(m == float("-inf"), 0.0))
            den = p.sum(-1, keepdim=True)
            p = (p / den.masked_fill(den == 0, 1.0)).view(Hk, G * n, -1)
            of = torch.matmul(p, vf)
            o[b, i0:i1] = of.view(Hk, G, n, D).permute(2, 0, 1, 3).reshape(n, H, D).to(o.dtype)
            if train:
                dof = st["do"][b, i0:i1].float().view(n, Hk, G, D).permute(1, 2, 0, 3).reshape(Hk, G * n, D)
                dp = torch.matmul(dof, vf.transpose(1, 2).contiguous())
                ds = p * (dp - (dof * of).sum(-1, keepdim=True)) * scale
                dq[b, i0:i1] = torch.matmul(ds, kf).view(Hk, G, n, D).permute(2, 0, 1, 3).reshape(n, H, D).to(dq.dtype)
                dkf = torch.matmul(ds.transpose(1, 2).contiguous(), qf).transpose(0, 1)
                dvf = torch.matmul(p.transpose(1, 2).contiguous(), dof).transpose(0, 1)
                if ns:
                    dk[b, :ns] += dkf[:ns]
                    dv[b, :ns] += dvf[:ns]
                dk[b, lo:hi] += dkf[ns:]
                dv[b, lo:hi] += dvf[ns:]
    if train:
        return o, dq, dk.to(q.dtype), dv.to(q.dtype)
    return o


def _rope_plain(st):
    c = st["case"]
    P = c["pairs"]
    axis = torch.cat([torch.full((n,), a, dtype=torch.long, device=st["pos"].device) for a, n in enumerate(st["sections"])])
    ang = st["pos"].double()[axis].permute(1, 2, 0) * st["inv_freq"].double()   # far positions: the angle needs 64 bits
    turn = 2 * math.pi
    ang = ang - torch.floor(ang / turn) * turn
    cos, sin = torch.cos(ang).float()[:, :, None], torch.sin(ang).float()[:, :, None]
    if c["mode"] == "transpose":
        sin = -sin
    out = []
    for t in (st["q"], st["k"]):
        f = t.float()
        if c["interleaved"]:
            a, b = f[..., 0:2 * P:2], f[..., 1:2 * P:2]
            r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = f[..., :P], f[..., P:2 * P]
            r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        out.append(torch.cat([r, f[..., 2 * P:]], -1).to(t.dtype))
    return tuple(out)


def _norm_plain(st):
    c = st["case"]
    rows, d = c["rows"], c["d"]
    h, x = st["h"].float(), st["x"].float()
    eps = 1e-6

    def normed(t, kind):
        mu = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
        rs = torch.rsqrt(((t - mu) ** 2).mean(-1, keepdim=True) + eps)
        return (t - mu) * rs, rs

    def normed_grad(dz, hat, rs, kind):
        r = dz - hat * (dz * hat).mean(-1, keepdim=True)
        if kind == "layer":
            r = r - dz.mean(-1, keepdim=True)
        return r * rs

    if c["post"] == "none":
        n = h
    else:
        hhat, hrs = normed(h, c["post"])
        n = hhat * st["post_w"] + (st["post_b"] if st["post_b"] is not None else 0.0)
    G = max(1, c["gates"])
    gate = st["gate"].repeat_interleave(rows // G, 0) if c["gates"] else torch.ones(1, d, device=h.device)
    x1 = c["res_scale"] * x + gate * n
    xhat, xrs = normed(x1, c["pre"])
    y = xhat * st["pre_w"] + (st["pre_b"] if st["pre_b"] is not None else 0.0)
    outs = [x1.to(st["x"].dtype), y.to(st["h"].dtype)]
    if c["mode"] == "infer":
        return tuple(outs)
    dy, dx1 = st["dy"].float(), st["dx1"].float()
    tot = dx1 + normed_grad(dy * st["pre_w"], xhat, xrs, c["pre"])
    dn = tot * gate
    if c["post"] == "none":
        dh = dn
    else:
        dh = normed_grad(dn * st["post_w"], hhat, hrs, c["post"])
    outs += [dh.to(st["h"].dtype), (c["res_scale"] * tot).to(st["x"].dtype)]
    if c["gates"]:
        outs.append((tot * n).view(G, rows // G, d).sum(1))
    if st["post_w"] is not None:
        outs.append((dn * hhat).sum(0))
    if st["post_b"] is not None:
        outs.append(dn.sum(0))
    outs.append((dy * xhat).sum(0))
    if st["pre_b"] is not None:
        outs.append(dy.sum(0))
    return outs


# ------------------------------------------------------------------------------------------------------------------------------ the definitions
def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _attention_exact, "rope": _rope_exact, "norm": _norm_exact}[case["op"]](case, st)


def _attention_exact(case, st):
    q, k, v = (st[n].double() for n in ("q", "k", "v"))
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    train = case["mode"] == "train"
    o = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    j = torch.arange(Sk, device=q.device)
    for b in range(B):
        nk, nq = st["klen_host"][b], st["qlen_host"][b]
        for h in range(H):
            kh, vh = k[b, :nk, h // (H // Hk)], v[b, :nk, h // (H // Hk)]
            for a in range(0, nq, 4096):
                z = min(a + 4096, nq)
                pos = torch.arange(a, z, device=q.device)[:, None] + nk - nq
                jj = j[None, :nk]
                ok = torch.ones(z - a, nk, dtype=torch.bool, device=q.device)
                if case["right"] >= 0:
                    ok = ok & (jj <= pos + case["right"])
                if case["left"] >= 0:
                    ok = ok & ((jj + case["left"] >= pos) | (jj < case["sinks"]))
                logit = torch.where(ok, (q[b, a:z, h] @ kh.T) / math.sqrt(D), -math.inf)
                lse = torch.logsumexp(logit, -1, keepdim=True)
                w = torch.where(ok, torch.exp(logit - torch.where(torch.isinf(lse), 0.0, lse)), 0.0)
                o[b, a:z, h] = w @ vh
                if train:
                    g = st["do"][b, a:z, h].double()
                    dv[b, :nk, h // (H // Hk)] += w.T @ g
                    dw = g @ vh.T
                    dl = w * (dw - (w * dw).sum(-1, keepdim=True)) / math.sqrt(D)
                    dq[b, a:z, h] = dl @ kh
                    dk[b, :nk, h // (H // Hk)] += dl.T @ q[b, a:z, h]
    return (o, dq, dk, dv) if train else o


def _rope_exact(case, st):
    P = case["pairs"]
    sign = -1.0 if case["mode"] == "transpose" else 1.0
    outs = []
    angle = torch.empty(case["B"], case["S"], P, dtype=torch.float64, device=st["pos"].device)
    p = 0
    for a, n in enumerate(st["sections"]):
        angle[..., p:p + n] = st["pos"][a].double()[..., None] * st["inv_freq"][p:p + n].double()
        p += n
    turn = torch.polar(torch.ones_like(angle), sign * angle)[:, :, None]
    for t in (st["q"], st["k"]):
        r = t.double().clone()
        first, second = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if case["interleaved"] else (slice(0, P), slice(P, 2 * P))
        z = torch.complex(r[..., first].contiguous(), r[..., second].contiguous()) * turn
        r[..., first], r[..., second] = z.real, z.imag
        outs.append(r)
    return tuple(outs)


def _norm_exact(case, st):
    d = case["d"]
    leaves = {n: st[n].double().requires_grad_(True) for n in ("h", "x", "gate", "post_w", "post_b", "pre_w", "pre_b") if st[n] is not None}

    def norm(t, kind, w, b):
        if kind == "none":
            return t
        if kind == "layer":
            t = t - t.sum(-1, keepdim=True) / d
        t = t / torch.sqrt((t * t).sum(-1, keepdim=True) / d + 1e-6)
        t = t * w
        return t if b is None else t + b

    n = norm(leaves["h"], case["post"], leaves.get("post_w"), leaves.get("post_b"))
    if case["gates"]:
        n = (n.view(case["gates"], -1, d) * leaves["gate"][:, None]).view(-1, d)
    x1 = leaves["x"] * case["res_scale"] + n
    y = norm(x1, case["pre"], leaves["pre_w"], leaves.get("pre_b"))
    if case["mode"] == "infer":
        return x1.detach(), y.detach()
    names = [m for m in ("h", "x", "gate", "post_w", "post_b", "pre_w", "pre_b") if m in leaves]
    total = (x1 * st["dx1"].double()).sum() + (y * st["dy"].double()).sum()
    return [x1.detach(), y.detach(), *torch.autograd.grad(total, [leaves[m] for m in names])]


# -------------------------------------------------------------------------------------------------------------------------------------- the work
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "attention":
        klen, qlen = _lens(case)
        B, H, Hk, D = case["B"], case["H"], case["Hk"], case["D"]
        pairs = seen = 0
        for nk, nq in zip(klen, qlen):
            first = nk
            for i in range(nq):
                ns, lo, hi = _band(case, i, i + 1, nk, nq)
                pairs += ns + hi - lo
                first = min(first, lo)
            ns, lo, hi = _band(case, 0, nq, nk, nq)
            seen += ns + hi - lo
        rows, outs = sum(qlen), B * case["Sq"]
        if case["mode"] == "infer":
            return {"bytes": e * D * (rows * H + 2 * seen * Hk + outs * H), "flops": 4 * D * H * pairs}
        # forward: q, k, v read, o written; backward: q, k, v, o, do read, dq, dk, dv written
        return {"bytes": e * D * (H * (4 * rows + 2 * outs) + Hk * (4 * seen + 2 * B * case["Sk"])), "flops": 14 * D * H * pairs}
    if case["op"] == "rope":
        tok = case["B"] * case["S"]
        return {"bytes": 2 * e * tok * (case["H"] + case["Hk"]) * case["D"] + 4 * case["axes"] * tok + 4 * case["pairs"],
                "flops": 6 * tok * (case["H"] + case["Hk"]) * case["pairs"]}
    n, s = case["rows"] * case["d"], BYTES[case["stream"]]
    small = 4 * case["d"] * (case["gates"] + 4)
    if case["mode"] == "infer":
        return {"bytes": n * (2 * e + 2 * s) + small, "flops": 14 * n}
    # forward: h, x read, x1, y written; backward: dx1, dy, h, x read, dh, dx written
    return {"bytes": n * (2 * e + 2 * s) + n * (3 * e + 3 * s) + 2 * small, "flops": 44 * n}
