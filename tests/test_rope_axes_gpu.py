"""Rotary positions with several axes (ops.rope_axes) against the definition in 64 bits.

Tolerance by element: the angle, reduced in 64 bits, is rounded to 2^-26 of a turn (2^-23 rad), its cosine and sine are good to 2^-22, the two products and
their sum to 2^-23: (|x0| + |x1|) 2^-20, and half a step of the type for the result.  At positions near 2^31 the 64-bit product itself is off by 2^-24 of a
turn: 2^-19."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    from smb_vision_amd import ops as o
    return o


def definition(t, pos, inv, sections, interleaved, sign, far):
    P = sum(sections)
    ang = torch.empty(t.shape[0], t.shape[1], P, dtype=torch.float64, device=t.device)
    p = 0
    for a, n in enumerate(sections):
        ang[..., p:p + n] = (pos[a] if pos.dim() == 3 else pos[a][None]).double()[..., None] * inv[p:p + n].double()
        p += n
    c, s = torch.cos(ang)[:, :, None], sign * torch.sin(ang)[:, :, None]
    f = t.double()
    i0, i1 = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    x0, x1 = f[..., i0], f[..., i1]
    ref, tol = f.clone(), torch.zeros_like(f)
    ref[..., i0], ref[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    tol[..., i0] = tol[..., i1] = (x0.abs() + x1.abs()) * 2.0 ** (-19 if far else -20)
    tol[..., :2 * P] += ref[..., :2 * P].abs() * torch.finfo(t.dtype).eps / 2 + (2.0 ** -25 if t.dtype == torch.float16 else 0)
    return ref, tol


def close(got, ref, tol):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[0].tolist(), got[bad][0].item(), ref[bad][0].item(), tol[bad][0].item())


CASES = [  # B, S, H, Hk, D, sections, interleaved, int64, shared positions, far
    (1, 1, 1, 1, 2, (1,), False, False, False, False), (2, 5, 3, 1, 64, (12, 10, 10), False, True, False, False), (1, 20, 12, 12, 64, (32,), True, False, True, True),
    (3, 7, 4, 2, 80, (10, 10, 10), True, True, False, True), (2, 33, 2, 2, 34, (5, 0, 3, 4), False, False, False, False), (1, 130, 5, 0, 96, (16, 16, 16), False, False, True, False),
    (2, 9, 2, 1, 128, (16, 24, 24), False, True, False, True), (1, 3, 1, 1, 1024, (300, 100, 112), False, False, False, False), (1, 4000, 2, 1, 32, (4, 4), True, False, False, False),
    (2, 11, 3, 1, 22, (3, 3, 3), True, False, False, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("B,S,H,Hk,D,sections,interleaved,wide,shared,far", CASES)
def test_against_the_definition(ops, dtype, transpose, B, S, H, Hk, D, sections, interleaved, wide, shared, far):
    g = torch.Generator().manual_seed(B * 100 + S)
    q = torch.randn(B, S, H, D, generator=g).to(dtype).cuda()
    k = torch.randn(B, S, Hk, D, generator=g).to(dtype).cuda() if Hk else None
    pos = torch.randint(-50 if not far else 2 ** 31 - 3000, 2 ** 31 - 1 if far else 5000, (len(sections), S) if shared else (len(sections), B, S), generator=g)
    pos = pos.to(torch.int64 if wide else torch.int32).cuda()
    P = sum(sections)
    inv = (10000.0 ** (-torch.arange(P) / P)).float().cuda()
    qo, ko = ops.rope_axes(q, k, pos, inv, sections, interleaved=interleaved, transpose=transpose)
    close(qo, *definition(q, pos, inv, sections, interleaved, -1 if transpose else 1, far))
    assert torch.equal(qo[..., 2 * P:], q[..., 2 * P:])
    if Hk:
        close(ko, *definition(k, pos, inv, sections, interleaved, -1 if transpose else 1, far))
    else:
        assert ko is None


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_views_in_place_and_alignment(ops, dtype, interleaved):
    """Column blocks of one packed projection, turned in place; the same through a buffer that starts one element off; what lies beside stays."""
    B, S, H, Hk, D, sections = 2, 37, 3, 1, 64, (10, 10, 8)
    packed = torch.randn(B, S, (H + 2 * Hk) * D, device="cuda").to(dtype)
    q, k = packed[..., :H * D].unflatten(-1, (H, D)), packed[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
    pos = torch.randint(0, 1000, (3, B, S), dtype=torch.int32, device="cuda")
    inv = torch.rand(28, device="cuda")
    want = ops.rope_axes(q, k, pos, inv, sections, interleaved=interleaved)
    odd = torch.empty(packed.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(packed).copy_(packed)
    oq, ok = odd[..., :H * D].unflatten(-1, (H, D)), odd[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D))
    assert all(torch.equal(a, b) for a, b in zip(want, ops.rope_axes(oq, ok, pos, inv, sections, interleaved=interleaved)))
    v = packed[..., (H + Hk) * D:].clone()
    res = ops.rope_axes(q, k, pos, inv, sections, interleaved=interleaved, out=(q, k))
    assert res[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(packed[..., (H + Hk) * D:], v)
    back = ops.rope_axes(q.double().float(), None, pos, inv, sections, interleaved=interleaved, transpose=True)[0] if dtype == torch.float32 else None
    if back is not None:   # the transposed map is the inverse
        close(back, odd[..., :H * D].unflatten(-1, (H, D)).double(), torch.full_like(back, 1e-5).double())
    out = torch.full((B, S + 2, H + 1, D), 7.0, dtype=dtype, device="cuda")
    ops.rope_axes(oq, None, pos, inv, sections, interleaved=interleaved, out=(out[:, :S, :H], None))
    assert torch.equal(out[:, :S, :H], want[0]) and bool((out[:, S:] == 7).all()) and bool((out[:, :, H] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_every_alignment_rounds_alike(ops, dtype, interleaved):
    """262,144 elements through the vector kernel and, one element further on, through the one for any alignment."""
    g = torch.Generator().manual_seed(7)
    q = torch.randn(4, 512, 2, 64, generator=g).to(dtype).cuda()
    pos, inv = torch.randint(0, 5000, (2, 4, 512), dtype=torch.int32, generator=g).cuda(), torch.rand(32, generator=g).cuda()
    odd = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(q).copy_(q)
    want = ops.rope_axes(q, None, pos, inv, (12, 20), interleaved=interleaved)[0]
    assert torch.equal(want, ops.rope_axes(odd, None, pos, inv, (12, 20), interleaved=interleaved)[0])


def test_captured_and_empty(ops):
    q, k = torch.randn(2, 9, 2, 64, device="cuda"), torch.randn(2, 9, 1, 64, device="cuda")
    pos = torch.arange(9, dtype=torch.int32, device="cuda").repeat(2, 2, 1)
    inv = torch.rand(32, device="cuda")
    want = ops.rope_axes(q, k, pos, inv, (16, 16))
    pos5 = pos + 5
    want5 = ops.rope_axes(q, k, pos5, inv, (16, 16))
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        res = ops.rope_axes(q, k, pos, inv, (16, 16))
    keep = pos.clone()
    for turn in range(4):
        pos.copy_(pos5 if turn % 2 else keep)
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(res, want5 if turn % 2 else want))
    qo, ko = ops.rope_axes(q[:0], k[:0], pos[:, :0], inv, (16, 16))
    assert qo.shape[0] == 0 and ko.shape[0] == 0
