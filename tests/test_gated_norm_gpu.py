"""The norm behind a block, its gate, the scaled residual sum and the norm in front of the next block (ops.gated_norm_fwd / _bwd) against the definition in
64 bits (torch's autograd for the gradients).

Tolerances by element.  A sum over a row in 32 bits is a tree of at most 32 + 8 terms deep: 40 * 2^-24 < 2^-18 of the sum of magnitudes.  A normalised value
hat = (t - mean) / dev is then off by E(hat) = 2^-17 (kappa + |hat|), kappa = max(1, mean|t| / dev).  Through the formulas, with margins of 4 for the handful
of further roundings (each 2^-24 of a term):
    x1: T1 = 2^-15 (|s x| + |gate| ((kappa + |hhat|) |w| + |b|))          y: 2^-13 ((kappa' + |xhat|) |w| + |b|) + max over the row of T1 times |w| / dev
    gradients: 2^-12 times the sum of the magnitudes that the formula adds up (every hat as kappa + |hat|), parameters' gradients: their sum over the rows
and half a step of the result's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from smb_vision_amd import ops as o
    return o


def norm(t, kind, eps):
    """hat, 1 / dev, kappa"""
    if kind is None:
        return t, torch.ones_like(t[:, :1]), torch.zeros_like(t[:, :1])
    mu = t.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
    rs = ((t - mu).pow(2).mean(1, keepdim=True) + eps).rsqrt()
    return (t - mu) * rs, rs, (t.abs().mean(1, keepdim=True) * rs).clamp(min=1)


def close(got, ref, tol, what):
    tol = tol + ref.abs() * torch.finfo(got.dtype).eps / 2 + (2.0 ** -25 if got.dtype == HF else 0)
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][0].item(), ref[bad][0].item(), tol[bad][0].item())


def make(rows, d, ht, xt, post, pre, gates, seed=0, mean=0.0, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    t = dict(h=(2 * r(rows, d) + mean).to(ht), x=(r(rows, d) + mean).to(xt), dx1=r(rows, d).to(xt), dy=r(rows, d).to(ht),
             post_w=1 + 0.2 * r(d) if post else None, post_b=0.3 * r(d) if post and bias else None, gate=r(gates, d) if gates else None,
             pre_w=1 + 0.2 * r(d) if pre else None, pre_b=0.3 * r(d) if pre and bias else None)
    return {k: None if v is None else v.cuda() for k, v in t.items()}


def verify(ops, t, post, pre, s, eps=1e-6, use_dx1=True):
    names = ("post_w", "post_b", "gate", "pre_w", "pre_b")
    kw = dict(post=post, pre=pre, res_scale=s, **{n: t[n] for n in names})
    x1, y, stats = ops.gated_norm_fwd(t["h"], t["x"], eps=eps, **kw)
    assert x1.dtype == t["x"].dtype and (y is None) == (pre is None)
    rows, d = t["h"].shape
    leaf = {n: t[n].double().requires_grad_(True) for n in ("h", "x", *names) if t[n] is not None}
    one, zero = torch.ones(d, dtype=torch.float64, device="cuda"), torch.zeros(d, dtype=torch.float64, device="cuda")
    w, b, pw, pb = leaf.get("post_w", one), leaf.get("post_b", zero), leaf.get("pre_w", one), leaf.get("pre_b", zero)
    gate = leaf["gate"].repeat_interleave(rows // t["gate"].shape[0], 0) if t["gate"] is not None else torch.ones(rows, 1, dtype=torch.float64, device="cuda")
    hh, rh, kh = norm(leaf["h"], post, eps)
    n = hh * w + b if post else hh
    rx1 = s * leaf["x"] + gate * n
    xh, rx, kx = norm(rx1, pre, eps)
    ry = xh * pw + pb
    ah = kh + hh.abs()
    an = ah * w.abs() + b.abs()
    t1 = 2.0 ** -15 * ((s * leaf["x"]).abs() + gate.abs() * an)
    close(x1, rx1.detach(), t1.detach(), "x1")
    ax = kx + xh.abs()
    if pre:
        ty = 2.0 ** -13 * (ax * pw.abs() + pb.abs()) + 2 * t1.amax(1, keepdim=True) * rx * ax * pw.abs()
        close(y, ry.detach(), ty.detach(), "y")
    dy, dx1 = t["dy"] if pre else None, t["dx1"] if use_dx1 else None
    gr = ops.gated_norm_bwd(dx1, dy, t["h"], t["x"], stats, **kw)
    total = (rx1 * (dx1.double() if use_dx1 else 0)).sum() + ((ry * dy.double()).sum() if pre else 0)
    ref = dict(zip(leaf, torch.autograd.grad(total, list(leaf.values()))))
    with torch.no_grad():
        m = dx1.double().abs() if use_dx1 else torch.zeros_like(rx1)
        if pre:
            z = dy.double().abs() * pw.abs()
            m = m + rx * (z + z.mean(1, keepdim=True) + ax * (z * ax).mean(1, keepdim=True))
        zh = m * gate.abs() * (w.abs() if post else 1)
        mh = rh * (zh + zh.mean(1, keepdim=True) + ah * (zh * ah).mean(1, keepdim=True)) if post else zh
        c = 2.0 ** -12
        tol = {"h": c * mh, "x": c * abs(s) * m, "post_w": c * (m * gate.abs() * ah).sum(0), "post_b": c * (m * gate.abs()).sum(0)}
        if pre:
            tol["pre_w"], tol["pre_b"] = c * (dy.double().abs() * ax).sum(0), c * dy.double().abs().sum(0)
        if t["gate"] is not None:
            tol["gate"] = c * (m * an).view(t["gate"].shape[0], -1, d).sum(1)
    for name, r in ref.items():
        got = gr[{"h": "dh", "x": "dx"}.get(name, name)]
        assert got.dtype == t[name].dtype and got.shape == t[name].shape
        close(got, r, tol[name], "d " + name)
    assert all(gr[n] is None for n in names if t[n] is None)


WIDTHS = [(1, 1), (5, 3), (33, 8), (130, 64), (7, 100), (257, 384), (66, 768), (40, 1001), (9, 1024), (21, 1536), (6, 2048), (10, 2500), (3, 4096), (2, 5001), (2, 8192)]


@pytest.mark.parametrize("rows,d", WIDTHS)
@pytest.mark.parametrize("ht,xt", [(BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)])
def test_widths_and_types(ops, rows, d, ht, xt):
    i = WIDTHS.index((rows, d))
    post, pre = [("layer", "layer"), ("rms", "rms"), ("rms", "layer"), ("layer", "rms")][i % 4]
    verify(ops, make(rows, d, ht, xt, post, pre, 1, seed=i), post, pre, 0.75)


@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("pre", [None, "rms", "layer"])
@pytest.mark.parametrize("gates", [0, 1, 3, 30, 90])
def test_norms_and_gates(ops, post, pre, gates):
    """One gate for all rows, for runs of rows that one or several workgroups share, for every row, and none."""
    verify(ops, make(90, 200, BF, FP, post, pre, gates, bias=gates != 3), post, pre, 1.0)


@pytest.mark.parametrize("rows,d,gates", [(20000, 64, 7 - 2), (3000, 136, 1000), (3001, 96, 3001), (2600, 520, 2), (1, 72, 1), (70000, 8, 35000)])
def test_many_rows(ops, rows, d, gates):
    verify(ops, make(rows, d, BF, BF, "rms", "layer", gates), "rms", "layer", 0.5)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_without_variance_and_far_from_zero(ops, kind):
    t = make(12, 300, FP, FP, kind, kind, 1)
    t["h"][3] = 0
    t["h"][4] = 2.5
    t["x"][5] = -t["h"][5]
    verify(ops, t, kind, kind, 1.0, eps=1e-5)
    verify(ops, make(12, 300, FP, FP, kind, kind, 1, mean=50.0), kind, kind, 1.0)


def test_missing_gradients_and_parameters(ops):
    t = make(50, 192, BF, FP, "layer", "layer", 0)
    t["post_w"] = t["pre_w"] = t["pre_b"] = None
    verify(ops, t, "layer", "layer", 1.0)
    verify(ops, make(50, 192, BF, FP, "rms", "rms", 2), "rms", "rms", 1.0, use_dx1=False)


def test_leading_dimensions_strides_and_in_place(ops):
    B, S, d = 3, 17, 96
    t = make(B * S, d, BF, FP, "rms", "layer", B)
    kw = dict(post="rms", pre="layer", **{n: t[n] for n in ("post_w", "post_b", "pre_w", "pre_b")})
    x1, y, st = ops.gated_norm_fwd(t["h"], t["x"], gate=t["gate"], **kw)
    g = ops.gated_norm_bwd(t["dx1"], t["dy"], t["h"], t["x"], st, gate=t["gate"], **kw)
    v = {n: t[n].view(B, S, d) for n in ("h", "x", "dx1", "dy")}
    for gate in (t["gate"], t["gate"][:, None]):
        a = ops.gated_norm_fwd(v["h"], v["x"], gate=gate, **kw)
        assert torch.equal(a[0].view(-1, d), x1) and torch.equal(a[1].view(-1, d), y) and torch.equal(a[2], st)
        b = ops.gated_norm_bwd(v["dx1"], v["dy"], v["h"], v["x"], st, gate=gate, **kw)
        assert b["gate"].shape == gate.shape and torch.equal(b["gate"].view(B, d), g["gate"]) and torch.equal(b["dh"].view(-1, d), g["dh"])

    def strided(x, pad):
        return torch.full((B * S, d + pad), 7.0, dtype=x.dtype, device="cuda")[:, pad // 2:pad // 2 + d].copy_(x)

    for pad in (8, 3, 32):   # (row starts off the vector width among them)
        s = {n: strided(t[n], pad) for n in ("h", "x", "dx1", "dy")}
        ox, oy = strided(t["x"], pad), strided(t["h"], pad)
        a = ops.gated_norm_fwd(s["h"], s["x"], gate=t["gate"], out=(ox, oy), **kw)
        close(a[0], x1.double(), x1.double().abs() * 2.0 ** -20 + 2.0 ** -18, "x1")
        assert a[0] is ox and bool((ox._base[:, :pad // 2] == 7).all()) and bool((ox._base[:, pad // 2 + d:] == 7).all())
        b = ops.gated_norm_bwd(s["dx1"], s["dy"], s["h"], s["x"], a[2], gate=t["gate"], out=(oy, ox), **kw)
        close(b["dx"], g["dx"].double(), g["dx"].double().abs() * 2.0 ** -16 + 2.0 ** -14, "dx")
    x = t["x"].clone()
    a = ops.gated_norm_fwd(t["h"], x, gate=t["gate"], out=(x, torch.empty_like(t["h"])), **kw)
    assert torch.equal(x, x1) and torch.equal(a[1], y)


def test_repeats_bit_for_bit_and_in_graphs(ops):
    t = [make(1500, 264, BF, FP, "rms", "rms", 4, seed=s) for s in (1, 2)]
    names = ("post_w", "gate", "pre_w")

    def call(c):
        kw = {n: c[n] for n in names}
        x1, y, st = ops.gated_norm_fwd(c["h"], c["x"], **kw)
        g = ops.gated_norm_bwd(c["dx1"], c["dy"], c["h"], c["x"], st, **kw)
        return [x1, y, g["dh"], g["dx"], *(g[n] for n in names)]

    want = [[r.clone() for r in call(c)] for c in t]
    graphs = []
    for _ in range(2):
        static = {n: None if v is None else v.clone() for n, v in t[0].items()}
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = call(static)
        graphs.append((g, static, res))
    for turn in range(4):
        for n, (g, static, res) in enumerate(graphs):
            for name, v in static.items():
                if v is not None:
                    v.copy_(t[(turn + n) % 2][name])
            g.replay()
        assert all(torch.equal(a, b) for a, b in zip(call(t[turn % 2]), want[turn % 2]))
        torch.cuda.synchronize()
        for n, (_, _, res) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(res, want[(turn + n) % 2]))


def test_no_rows(ops):
    t = make(0, 64, BF, FP, "rms", "rms", 1)
    kw = dict(post_w=t["post_w"], gate=t["gate"], pre_w=t["pre_w"])
    x1, y, st = ops.gated_norm_fwd(t["h"], t["x"], **kw)
    g = ops.gated_norm_bwd(t["dx1"], t["dy"], t["h"], t["x"], st, **kw)
    assert x1.shape == (0, 64) and not any(bool(g[n].any()) for n in ("gate", "post_w", "pre_w"))
