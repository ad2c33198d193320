"""Windowed attention with sinks (ops.window_attention_fwd / _bwd) against its definition in 64 bits.

Tolerances are worst cases by element, from the definition's own magnitudes.  u is half a step of the type (bf16 2^-8, fp16 2^-11).  The kernels round P (u),
dS (u) and the results (u); what they hold in 32 bits - scores, exponentials, sums over up to a few thousand terms - is within T = 2^-13 relative for the
operands used here (128 * 2^-24 * scale * sum |q||k|, about 7, is 2^-14).  With A = sum_j P |V|:
    |O - o|   <= u A + u |o| + 4 T A                      <= (2 u + 5 T) A
    |delta|   :  O's error from the rounding of P, u A in every channel, and T:  E = sum_d |dO_d| (u + 5 T) A_d   (the residual of O's own rounding is kept)
    |dS|      <= P (E + (u + 4 T) (|dP| + |delta|) + 2 T sum |dO||V|)      (sum |dO||V| bounds what 32-bit accumulation of dP can lose)
    dQ, dK    <= scale * sum of those |K|, |Q|, + u times the result;     dV <= (u + 4 T) sum P |dO| + u |dV|
fp16 has steps of 2^-24 below 2^-14: P and dS (dS in units of the largest |dO|) can be off by 2^-25 more, an output by 2^-25.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

T = 2.0 ** -13
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from smb_vision_amd import ops as o
    return o


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def lens_of(kind, B, n, seed):
    if kind is None:
        return None
    if kind == "ragged":
        g = torch.Generator().manual_seed(seed)
        out = torch.randint(1, n + 1, (B,), generator=g)
        out[0] = n
        return out.int()
    return torch.tensor((list(kind) * B)[:B], dtype=torch.int32)


def definition(q, k, v, do, left, right, sinks, scale, q_lens, k_lens):
    """o, lse, dq, dk, dv and the tolerances' sums, everything in 64 bits; rows and keys past a length do not take part."""
    dtype = q.dtype
    u, sub = half_step(dtype), (2.0 ** -25 if dtype == HF else 0.0)
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    dev = q.device
    out = {n: torch.zeros(s, dtype=torch.float64, device=dev) for n, s in
           (("o", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape), ("to", q.shape), ("tq", q.shape), ("tk", k.shape), ("tv", v.shape))}
    lse = torch.full((B, H, Sq), -float("inf"), dtype=torch.float64, device=dev)
    for b in range(B):
        nk = Sk if k_lens is None else max(0, min(Sk, int(k_lens[b])))
        nq = Sq if q_lens is None else max(0, min(Sq, int(q_lens[b])))
        if nk == 0 or nq == 0:
            continue
        pos = torch.arange(nq, device=dev)[:, None] + (nk - nq)
        key = torch.arange(nk, device=dev)[None]
        vis = torch.ones(nq, nk, dtype=torch.bool, device=dev)
        if right >= 0:
            vis &= key <= pos + right
        if left >= 0:
            vis &= (key >= pos - left) | (key < sinks)
        gmax = do[b, :nq].double().abs().amax() if do is not None else 0.0
        for h in range(H):
            hk = h // G
            qq, kk, vv = q[b, :nq, h].double(), k[b, :nk, hk].double(), v[b, :nk, hk].double()
            s = (qq @ kk.T * scale).masked_fill(~vis, -float("inf"))
            ls = torch.logsumexp(s, 1)
            lse[b, h, :nq] = ls
            p = torch.where(vis, torch.exp(s - torch.where(torch.isinf(ls), 0.0, ls)[:, None]), 0.0)
            some = vis.any(1, keepdim=True).double()
            a = p @ vv.abs()
            o = p @ vv
            out["o"][b, :nq, h] = o
            out["to"][b, :nq, h] = (2 * u + 5 * T) * a + some * sub * (1 + nk * vv.abs().amax())
            if do is None:
                continue
            g = do[b, :nq, h].double()
            dp = g @ vv.T
            delta = (g * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            e_delta = (g.abs() * ((u + 5 * T) * a + sub * nk * vv.abs().amax())).sum(1, keepdim=True)
            e = p * (e_delta + (u + 4 * T) * (dp.abs() + delta.abs()) + 2 * T * (g.abs() @ vv.abs().T))
            eq, ek = e + vis * sub * g.abs().amax(1, keepdim=True), e + vis * sub * gmax
            out["dq"][b, :nq, h] = scale * ds @ kk
            out["tq"][b, :nq, h] = scale * (eq @ kk.abs()) + u * (scale * ds @ kk).abs() + some * sub
            out["dk"][b, :nk, hk] += scale * ds.T @ qq
            out["tk"][b, :nk, hk] += scale * (ek.T @ qq.abs())
            out["dv"][b, :nk, hk] += p.T @ g
            out["tv"][b, :nk, hk] += (u + 4 * T) * (p.T @ g.abs()) + sub * (vis.double().T @ g.abs())
    out["tk"] += u * out["dk"].abs() + (sub if do is not None else 0)
    out["tv"] += u * out["dv"].abs() + (sub if do is not None else 0)
    return out, lse


def close(got, ref, tol, what):
    bad = ~((got.double() - ref).abs() <= tol * (1 + 1e-6))
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                                 f"{got[bad][0].item()} for {ref[bad][0].item()} +- {tol[bad][0].item()}")


def close_lse(got, ref):
    assert torch.equal(torch.isinf(got), torch.isinf(ref)) and bool((got[torch.isinf(got)] < 0).all())
    fin = ~torch.isinf(ref)
    assert bool(((got.double() - ref)[fin].abs() <= 2 * T + T * ref[fin].abs() * 2 ** -6).all())


def operands(dtype, B, Sq, Sk, H, Hk, D, seed=0, packed=False):
    g = torch.Generator().manual_seed(seed)
    if packed:
        p = torch.randn(B, Sq, (H + 2 * Hk) * D, generator=g).to(dtype).cuda()
        return (p[..., :H * D].unflatten(-1, (H, D)), p[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)), p[..., (H + Hk) * D:].unflatten(-1, (Hk, D)))
    return tuple(torch.randn(B, n, h, D, generator=g).to(dtype).cuda() for n, h in ((Sq, H), (Sk, Hk), (Sk, Hk)))


def check(ops, dtype, B, Sq, Sk, H, Hk, D, left, right, sinks, ql=None, kl=None, scale=None, packed=False, backward=True, resid=True, seed=0):
    q, k, v = operands(dtype, B, Sq, Sk, H, Hk, D, seed, packed)
    do = (torch.randn(B, Sq, H, D, generator=torch.Generator().manual_seed(seed + 100)) * 0.1).to(dtype).cuda() if backward else None
    q_lens, k_lens = lens_of("ragged" if ql == "same" else ql, B, Sq, 11), lens_of(kl, B, Sk, 12)
    if ql == "same":
        k_lens = q_lens
    sc = D ** -0.5 if scale is None else scale
    ref, lse_ref = definition(q, k, v, do, left, right, sinks, sc, q_lens, k_lens)
    dev = lambda t: None if t is None else t.cuda()
    kw = dict(left=left, right=right, sinks=sinks, scale=scale, q_lens=dev(q_lens), k_lens=dev(k_lens))
    res = ops.window_attention_fwd(q, k, v, resid=resid, **kw)
    close(res[0], ref["o"], ref["to"], "o")
    close_lse(res[1], lse_ref)
    if backward:
        dq, dk, dv = ops.window_attention_bwd(q, k, v, res[0], do, res[1], o_lo=res[2], **kw)
        for n, t in (("q", dq), ("k", dk), ("v", dv)):
            close(t, ref["d" + n], ref["t" + n], "d" + n)


SELF = [  # dtype, B, S, H, Hk, D, left, right, sinks
    (HF, 1, 1, 1, 1, 8, 0, 0, 0), (BF, 2, 3, 2, 1, 64, 1, 0, 1), (HF, 1, 63, 2, 2, 64, 5, 0, 2), (HF, 1, 64, 3, 1, 32, 7, 9, 3), (HF, 2, 65, 4, 2, 64, 16, 0, 4),
    (BF, 1, 127, 2, 2, 128, 40, 3, 0), (HF, 1, 129, 6, 2, 128, 33, 0, 5), (HF, 1, 200, 5, 1, 80, 20, 0, 70), (BF, 2, 257, 3, 3, 40, 64, 64, 1),
    (HF, 1, 300, 2, 1, 96, -1, 0, 0), (BF, 1, 333, 2, 2, 64, -1, -1, 0), (HF, 1, 511, 4, 4, 24, 100, -1, 3), (HF, 1, 640, 2, 1, 120, 0, 200, 130),
    (BF, 1, 777, 8, 1, 64, 255, 0, 4), (HF, 1, 1000, 7, 1, 48, 129, 0, 4), (HF, 3, 130, 2, 2, 128, 63, 64, 0), (BF, 1, 2049, 1, 1, 128, 511, 511, 16),
]


@pytest.mark.parametrize("dtype,B,S,H,Hk,D,left,right,sinks", SELF)
def test_self_attention(ops, dtype, B, S, H, Hk, D, left, right, sinks):
    check(ops, dtype, B, S, S, H, Hk, D, left, right, sinks, packed=True)


@pytest.mark.parametrize("dtype,B,S,H,Hk,D,left,right,sinks", [(HF, 4, 150, 4, 2, 64, 31, 0, 4), (BF, 5, 97, 2, 2, 128, -1, 0, 0), (HF, 3, 260, 3, 1, 32, 50, 20, 2)])
def test_padded_batch(ops, dtype, B, S, H, Hk, D, left, right, sinks):
    check(ops, dtype, B, S, S, H, Hk, D, left, right, sinks, ql="same", kl=None)
    check(ops, dtype, B, S, S, H, Hk, D, left, right, sinks, ql="ragged", kl="ragged")


QUERIES = [  # dtype, B, Sq, Sk, H, Hk, D, left, right, sinks, q lens, k lens
    (HF, 1, 1, 1, 4, 4, 64, -1, 0, 0, None, None), (HF, 3, 1, 77, 8, 2, 128, 30, 0, 4, None, "ragged"), (BF, 2, 1, 1500, 12, 12, 64, 255, 0, 4, None, None),
    (HF, 16, 1, 2111, 8, 1, 128, 1000, 0, 4, None, "ragged"), (HF, 1, 1, 4097, 32, 4, 64, -1, 0, 0, None, None), (HF, 2, 5, 900, 4, 2, 80, 300, 0, 1, None, "ragged"),
    (HF, 2, 40, 700, 6, 3, 64, 64, 0, 65, None, None), (BF, 1, 333, 1001, 4, 1, 128, 400, 0, 7, None, None), (HF, 2, 33, 20, 2, 2, 64, 4, 0, 2, None, None),
    (HF, 4, 9, 50, 2, 1, 64, 8, 0, 3, (0, 9, 4, 1), (0, 3, 50, 0)), (HF, 2, 17, 64, 2, 2, 32, 3, 0, 0, (17, 40), (1000, -5)), (HF, 1, 200, 3, 2, 1, 64, 1, 1, 0, None, None),
]


@pytest.mark.parametrize("dtype,B,Sq,Sk,H,Hk,D,left,right,sinks,ql,kl", QUERIES)
def test_queries_at_the_end_of_a_cache(ops, dtype, B, Sq, Sk, H, Hk, D, left, right, sinks, ql, kl):
    """Single tokens, appended pieces, more queries than keys (the first rows see nothing), lengths of zero and out of range."""
    check(ops, dtype, B, Sq, Sk, H, Hk, D, left, right, sinks, ql, kl)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_other_scales(ops, dtype, scale):
    # (scale 1 at D 32: scores up to ~30, the softmax is nearly one key; 32 * 2^-24 * sum |q||k| ~ 20 stays within T)
    check(ops, dtype, 1, 190, 190, 2, 1, 32, 60, 0, 2, scale=scale)


@pytest.mark.parametrize("Sq,Sk,H,Hk,left,right,sinks", [(5000, 5000, 1, 1, 1023, 0, 4), (4100, 4100, 2, 1, 700, 900, 70), (1, 20480, 4, 1, 9999, 0, 5), (20, 16000, 4, 2, -1, 0, 0)])
def test_which_keys_are_seen(ops, Sq, Sk, H, Hk, left, right, sinks):
    """q = 0 makes every visible key weigh the same: O is a mean of small integers, rounded once (the sum and the count are exact in 32 bits, the division and
    the scaling are off by 2^-23), so one key too many or too few shows at any length."""
    D = 64
    q = torch.zeros(1, Sq, H, D, dtype=BF, device="cuda")
    k = torch.randn(1, Sk, Hk, D, device="cuda").to(BF)
    v = ((torch.arange(Sk * Hk * D, device="cuda") * 7919) % 31 - 15).to(BF).view(1, Sk, Hk, D)
    o, lse = ops.window_attention_fwd(q, k, v, left=left, right=right, sinks=sinks)
    vs = torch.cat([torch.zeros(1, Hk, D, dtype=torch.float64, device="cuda"), v[0].double().cumsum(0)])
    p = torch.arange(Sq, device="cuda") + Sk - Sq
    hi = (p + right + 1).clamp(0, Sk) if right >= 0 else torch.full_like(p, Sk)
    lo = (p - left).clamp(min=0) if left >= 0 else torch.zeros_like(p)
    lo = torch.minimum(lo, hi)
    ns = torch.minimum(torch.full_like(p, sinks), lo)
    n = ns + hi - lo
    ref = ((vs[hi] - vs[lo] + vs[ns]) / n[:, None, None]).repeat_interleave(H // Hk, 1)[None]
    close(o, ref, ref.abs() * (half_step(BF) + 2.0 ** -21), "o")
    close_lse(lse, n.double().log().expand(1, H, Sq))


def test_strides_and_output_views(ops):
    """Head-major operands, a batch broadcast over the sequences, gradients into column blocks of one packed tensor; what lies beside them stays."""
    B, S, H, Hk, D = 2, 140, 4, 2, 64
    q, k, v = operands(HF, B, S, S, H, Hk, D)
    do = (torch.randn(B, S, H, D, device="cuda") * 0.1).to(HF)
    kw = dict(left=50, right=0, sinks=3)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    g = ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw)
    hm = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    big = torch.full((B, S + 3, H + 1, D), 7.0, dtype=HF, device="cuda")
    o2, lse2, lo2 = ops.window_attention_fwd(hm(q), hm(k), hm(v), resid=True, out=big[:, :S, :H], **kw)
    assert torch.equal(o2, o) and torch.equal(lse2, lse) and torch.equal(lo2, lo)
    assert bool((big[:, S:] == 7).all()) and bool((big[:, :, H] == 7).all())
    pk = torch.full((B, S, (H + 2 * Hk) * D + 8), 7.0, dtype=HF, device="cuda")
    views = (pk[..., :H * D].unflatten(-1, (H, D)), pk[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)), pk[..., (H + Hk) * D:-8].unflatten(-1, (Hk, D)))
    g2 = ops.window_attention_bwd(hm(q), hm(k), hm(v), o2, hm(do), lse2, o_lo=lo2, out=views, **kw)
    assert all(torch.equal(a, b) for a, b in zip(g, g2)) and bool((pk[..., -8:] == 7).all())
    kb, vb = k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1)
    o3, lse3 = ops.window_attention_fwd(q, kb, vb, **kw)
    o4, _ = ops.window_attention_fwd(q, kb.contiguous(), vb.contiguous(), **kw)
    assert torch.equal(o3, o4)
    g3 = ops.window_attention_bwd(q, kb, vb, o3, do, lse3, **kw)   # the gradients of the expanded operands, one for each sequence
    g4 = ops.window_attention_bwd(q, kb.contiguous(), vb.contiguous(), o3, do, lse3, **kw)
    assert all(torch.equal(a, b) for a, b in zip(g3, g4))


@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
@pytest.mark.parametrize("Sq", [1, 70])
def test_what_nobody_sees_does_not_matter(ops, junk, Sq):
    """NaN and infinities in padded rows, in keys past a length and in keys of a cache that lie between the sinks and every row's window."""
    B, Sk, H, Hk, D, left, sinks = 2, 300, 4, 2, 64, 40, 4
    q, k, v = operands(HF, B, Sq, Sk, H, Hk, D)
    do = (torch.randn(B, Sq, H, D, device="cuda") * 0.1).to(HF)
    ql, kl = torch.tensor([Sq, max(1, Sq - 3)], dtype=torch.int32, device="cuda"), torch.tensor([290, 300], dtype=torch.int32, device="cuda")
    kw = dict(left=left, right=0, sinks=sinks, q_lens=ql, k_lens=kl)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    g = ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw)
    q2, k2, v2, do2 = q.clone(), k.clone(), v.clone(), do.clone()
    for t in (k2, v2):
        t[0, 290:] = junk
        t[:, sinks:300 - Sq - left - 20] = junk
    for t in (q2, do2):
        t[1, int(ql[1]):] = junk
    o2, lse2, lo2 = ops.window_attention_fwd(q2, k2, v2, resid=True, **kw)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    o2[1, int(ql[1]):] = junk
    lo2[1, int(ql[1]):] = junk
    g2 = ops.window_attention_bwd(q2, k2, v2, o2, do2, lse2, o_lo=lo2, **kw)
    assert all(torch.equal(a, b) for a, b in zip(g, g2))


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 10])
def test_fp16_gradients_of_any_size(ops, size):
    """dS is formed in units of the largest |dO|: gradients far below (and above) one keep their digits."""
    B, S, H, D = 1, 200, 2, 64
    q, k, v = operands(HF, B, S, S, H, H, D)
    do = (torch.randn(B, S, H, D, generator=torch.Generator().manual_seed(5)) * size).to(HF).cuda()
    do[:, 100:] *= 2.0 ** -3   # (rows of very different size in one call)
    kw = dict(left=60, right=0, sinks=2)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    ref, _ = definition(q, k, v, do, 60, 0, 2, D ** -0.5, None, None)
    for n, t in zip("qkv", ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw)):
        close(t, ref["d" + n], ref["t" + n], "d" + n)


def test_finite_differences(ops):
    """The gradient against differences of the forward: fp16, a step of 2^-4 along a random direction.  The two forwards are each off by at most their
    tolerance (weighted by |dO|), the difference quotient by its third derivative, below 2 % here (|d| ~ 0.1 a score)."""
    B, S, H, D = 1, 96, 2, 32
    q, k, v = operands(HF, B, S, S, H, H, D)
    do = torch.randn(B, S, H, D, device="cuda").to(HF)
    kw = dict(left=20, right=0, sinks=3)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    grads = ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw)
    step = 2.0 ** -4
    for i, name in enumerate("qkv"):
        t = (q, k, v)[i]
        d = grads[i].double() / grads[i].double().abs().amax()   # along the gradient: the largest change
        plus, minus = [(t.double() + s * step * d).to(HF) for s in (1, -1)]
        f = []
        for x in (plus, minus):
            a = [q, k, v]
            a[i] = x
            r, _ = definition(*a, None, 20, 0, 3, D ** -0.5, None, None)
            y = ops.window_attention_fwd(*a, **kw)[0]
            f.append(((y.double() * do.double()).sum(), (r["to"] * do.double().abs()).pow(2).sum().sqrt()))
        got = (f[0][0] - f[1][0]).item()
        want = (grads[i].double() * (plus.double() - minus.double())).sum().item()
        assert abs(got - want) <= 0.02 * abs(want) + 4 * (f[0][1] + f[1][1]).item(), (name, got, want)


def test_a_repeated_call_gives_the_same_bits(ops):
    q, k, v = operands(BF, 2, 700, 700, 4, 1, 128)
    do = torch.randn(2, 700, 4, 128, device="cuda").to(BF)
    kw = dict(left=150, right=0, sinks=5)
    first = None
    for _ in range(3):
        o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
        res = (o, lse, lo, *ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw))
        first = first or res
        assert all(torch.equal(a, b) for a, b in zip(first, res))


@pytest.mark.parametrize("Sq,Sk,H,Hk", [(400, 400, 4, 2), (1, 5000, 8, 1)])
def test_captured_into_graphs_and_on_another_stream(ops, Sq, Sk, H, Hk):
    """Two captured graphs (their workspaces are theirs) replayed in turn with changed operands, eager calls between the replays; an own stream."""
    D = 64
    kw = dict(left=3000 if Sq == 1 else 90, right=0, sinks=4)
    sets = [operands(BF, 1, Sq, Sk, H, Hk, D, seed=s) for s in (1, 2, 3)]
    dos = [torch.randn(1, Sq, H, D, generator=torch.Generator().manual_seed(s)).to(BF).cuda() for s in (1, 2, 3)]

    def call(q, k, v, do):
        o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
        return (o, lse, *ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw))

    want = [[t.clone() for t in call(*s, do)] for s, do in zip(sets, dos)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(*sets[1], dos[1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in (*sets[0], dos[0])]
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            res = call(*static)
        graphs.append((g, static, res))
    for turn in range(4):
        for n, (g, static, res) in enumerate(graphs):
            i = (turn + n) % 3
            for a, b in zip(static, (*sets[i], dos[i])):
                a.copy_(b)
            g.replay()
        eager = call(*sets[turn % 3], dos[turn % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[turn % 3]))
        for n, (_, _, res) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(res, want[(turn + n) % 3])), (turn, n)


def test_empty_calls(ops):
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 5), (2, 3, 0)):
        q, k, v = operands(BF, B, Sq, Sk, 2, 1, 64)
        o, lse = ops.window_attention_fwd(q, k, v, left=3, right=0)
        assert o.shape == q.shape and not bool(o.any()) and bool((lse == -float("inf")).all())
        for t in ops.window_attention_bwd(q, k, v, o, torch.ones_like(q), lse, left=3, right=0):
            assert not bool(t.any())


def test_a_cache_beyond_32_bit_offsets(ops):
    """One sequence whose keys and values span more than 2^32 bytes: a few rows of a wide buffer, the rest never touched."""
    Sk, Hk, D, width = 36000, 1, 64, 64 * 1024   # 128 KiB between the rows: 4.7 GB
    buf = torch.empty(Sk, width, dtype=BF, device="cuda")
    k, v = torch.randn(1, Sk, Hk, D, device="cuda").to(BF), torch.randn(1, Sk, Hk, D, device="cuda").to(BF)
    kb, vb = buf[:, :D].view(1, Sk, Hk, D), buf[:, D:2 * D].view(1, Sk, Hk, D)
    kb.copy_(k)
    vb.copy_(v)
    for Sq, H in ((1, 4), (300, 2)):
        q = torch.randn(1, Sq, H, D, device="cuda").to(BF)
        for left in (500, -1):
            kw = dict(left=left, right=0, sinks=4)
            o, lse = ops.window_attention_fwd(q, k, v, **kw)
            o2, lse2 = ops.window_attention_fwd(q, kb, vb, **kw)
            assert torch.equal(o, o2) and torch.equal(lse, lse2)
            if left > 0:
                do = torch.randn_like(q)
                assert all(torch.equal(a, b) for a, b in zip(ops.window_attention_bwd(q, k, v, o, do, lse, **kw), ops.window_attention_bwd(q, kb, vb, o, do, lse, **kw)))


def apart(t, gap):
    """t [B, S, H, D] as a head-major view whose heads lie `gap` elements apart."""
    B, S, H, D = t.shape
    buf = torch.empty((H - 1) * gap + B * S * D, dtype=t.dtype, device="cuda")
    return buf.as_strided((B, S, H, D), (S * D, D, gap, 1)).copy_(t)


@pytest.mark.parametrize("H,Hk,gap", [(2, 1, 2 ** 31 + 64), (8, 8, 2 ** 24 + 8), (4, 1, 2 ** 28)])
def test_heads_far_apart(ops, H, Hk, gap):
    """Head-major operands with 2^24 elements and more between the heads (caches of 131,072 keys of 128 channels and longer), beyond 32-bit offsets too."""
    B, S, D = 1, 300, 64
    q, k, v = operands(BF, B, S, S, H, Hk, D)
    do = torch.randn(B, S, H, D, generator=torch.Generator().manual_seed(9)).to(BF).cuda()
    kw = dict(left=60, right=0, sinks=3)
    o, lse = ops.window_attention_fwd(q, k, v, **kw)
    want = ops.window_attention_bwd(q, k, v, o, do, lse, **kw)
    fq, fk, fv, fdo = (apart(t, gap) for t in (q, k, v, do))
    o2, lse2 = ops.window_attention_fwd(fq, fk, fv, **kw)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    assert all(torch.equal(a, b) for a, b in zip(want, ops.window_attention_bwd(fq, fk, fv, o2, fdo, lse2, **kw)))
    outs = [apart(torch.zeros_like(t), gap) for t in (q, k, v)]
    fo = apart(torch.zeros_like(o), gap)
    ops.window_attention_fwd(fq, fk, fv, out=fo, **kw)
    ops.window_attention_bwd(fq, fk, fv, fo, fdo, lse, out=outs, **kw)
    assert torch.equal(fo, o) and all(torch.equal(a, b) for a, b in zip(want, outs))
    for t in (1, 7):   # few rows: the other forward kernel
        assert torch.equal(ops.window_attention_fwd(fq[:, :t], fk, fv, **kw)[0], ops.window_attention_fwd(q[:, :t], k, v, **kw)[0])


@pytest.mark.parametrize("S,H,Hk,D,left,right,sinks", [(300, 2, 1, 64, 5, 0, 2), (200, 2, 2, 128, 20, 10, 0), (700, 3, 1, 32, 40, 0, 40), (130, 1, 1, 80, -1, 0, 0)])
def test_fp16_gradients_beside_a_row_that_a_key_does_not_see(ops, S, H, Hk, D, left, right, sinks):
    """One query's gradient is 2^24 times the others'.  The keys that it does not see keep their digits: their gradients are those of the call without it, bit
    for bit, and within the definition's tolerance for that call."""
    q, k, v = operands(HF, 1, S, S, H, Hk, D)
    small = (torch.randn(1, S, H, D, generator=torch.Generator().manual_seed(8)) * 2.0 ** -13).to(HF).cuda()
    kw = dict(left=left, right=right, sinks=sinks)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    for at in (S // 3, S - 1):
        big, none = small.clone(), small.clone()
        big[:, at], none[:, at] = 2.0 ** 12, 0
        seen = (torch.arange(S) <= at + right) if right >= 0 else torch.ones(S, dtype=torch.bool)
        if left >= 0:
            seen &= (torch.arange(S) >= at - left) | (torch.arange(S) < sinks)
        g, g0 = ([t.clone() for t in ops.window_attention_bwd(q, k, v, o, d, lse, o_lo=lo, **kw)] for d in (big, none))
        ref, _ = definition(q, k, v, none, left, right, sinks, D ** -0.5, None, None)
        assert bool((~seen).any()) or at == S - 1
        for n, a, b in zip("qkv", g, g0):
            close(b, ref["d" + n], ref["t" + n], "d" + n)
            if n != "q":
                assert torch.equal(a[:, ~seen.cuda()], b[:, ~seen.cuda()]), (at, n)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("junk", [float("nan"), float("inf")])
def test_rows_that_see_nothing_give_no_gradient(ops, dtype, junk):
    """More queries than keys: the first rows see nothing.  Whatever their query and their gradient hold, their dQ is 0 and no other gradient changes."""
    B, Sq, Sk, H, Hk, D = 2, 90, 50, 4, 2, 64
    q, k, v = operands(dtype, B, Sq, Sk, H, Hk, D)
    do = (torch.randn(B, Sq, H, D, generator=torch.Generator().manual_seed(4)) * 0.1).to(dtype).cuda()
    kl = torch.tensor([50, 31], dtype=torch.int32, device="cuda")
    kw = dict(left=20, right=0, sinks=2, k_lens=kl)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    want = ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw)
    q2, do2 = q.clone(), do.clone()
    for b, n in enumerate((50, 31)):
        assert bool((lse[b, :, :Sq - n] == -float("inf")).all()) and not bool(o[b, :Sq - n].any()) and not bool(want[0][b, :Sq - n].any())
        q2[b, :Sq - n] = junk
        do2[b, :Sq - n] = junk
    o2, lse2, lo2 = ops.window_attention_fwd(q2, k, v, resid=True, **kw)
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and torch.equal(lo, lo2)
    for n, a, b in zip("qkv", want, ops.window_attention_bwd(q2, k, v, o2, do2, lse2, o_lo=lo2, **kw)):
        assert torch.equal(a, b), n


@pytest.mark.parametrize("Sq,Sk,H", [(90, 50, 2), (12, 5, 2), (40, 20, 1)])
def test_rows_that_see_nothing_beside_infinite_values(ops, Sq, Sk, H):
    """An infinity in a value that other rows of the tile see: the rows that see nothing are 0 with lse -inf, their dQ is 0."""
    q, k, v = operands(BF, 1, Sq, Sk, H, 1, 64)
    do = torch.ones_like(q)
    v[:, :3] = float("inf")
    kw = dict(left=20, right=0, sinks=1)
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
    n = Sq - Sk
    assert not bool(o[:, :n].any()) and not bool(lo[:, :n].any()) and bool((lse[:, :, :n] == -float("inf")).all()) and bool((lse[:, :, n:] > -float("inf")).all())
    assert not bool(ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, **kw)[0][:, :n].any())
