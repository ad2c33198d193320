"""Per-op Python wrappers over the C ABI (torch tensors in, torch tensors out; all work happens in libsmbv.so on the
current HIP stream).  These are what the GPU parity tests call; the model itself drives the fused whole-step entry
points (see modeling_videomae.py).  Nothing here computes with PyTorch — tensors are only device memory."""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import GemmEpi, check


def _need_gpu(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise _lib.SmbvError("smb_vision_amd ops need tensors on a HIP device (no CPU fallback)")


def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ws(nbytes, dev):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=dev)


def gemm_nt(A, B, *, bias=None, rowadd=None, rowidx=None, gelu=False, save_pre=False, dgelu_pre=None, out_bf16=True, out_f32=False,
            alpha=1.0, grp=None, out_rows=None, reuse=None, splitk=False, rope=None):
    """C = epi(A[M,K] @ B[N,K]^T).  Returns dict with 'bf16', 'f32', 'pre' entries as requested.  reuse: a dict returned by an earlier call of the
    same shape - its tensors are written again instead of allocating (and zero-filling) new ones (timing loops).  splitk: smbv_gemm_nt_splitk (two K
    halves per 256 x 128 tile; raises ValueError for a product that form does not take).  rope: dict(table, pos (or None), S, grid, Dh, head_stride, wa) -
    smbv_gemm_nt_rope, the 3-axis rotary embedding of the q | k sections applied in the epilogue."""
    _need_gpu(A, B)
    lib = _lib.load()
    M, K = A.shape
    N = B.shape[0]
    rows = out_rows or M
    res = {}
    e = GemmEpi()
    e.alpha = alpha
    e.bias = _p(bias)
    e.rowadd, e.rowidx, e.ldr = _p(rowadd), _p(rowidx), (rowadd.stride(0) if rowadd is not None else 0)
    e.dgelu_pre, e.ld_pre = _p(dgelu_pre), (dgelu_pre.stride(0) if dgelu_pre is not None else 0)
    e.act_gelu = int(gelu)
    if save_pre:
        res["pre"] = reuse["pre"] if reuse else torch.empty(rows, N, dtype=torch.bfloat16, device=A.device)
        e.aux_pre, e.ld_aux = res["pre"].data_ptr(), N
    if out_bf16:
        res["bf16"] = reuse["bf16"] if reuse else torch.zeros(rows, N, dtype=torch.bfloat16, device=A.device)
        e.out_bf16, e.ld_ob = res["bf16"].data_ptr(), N
    if out_f32:
        res["f32"] = reuse["f32"] if reuse else torch.zeros(rows, N, dtype=torch.float32, device=A.device)
        e.out_f32, e.ld_of = res["f32"].data_ptr(), N
    if grp:
        e.grp_in, e.grp_out = grp
    if splitk:
        ws = (reuse or {}).get("splitk_ws")
        if ws is None:
            ws = _ws(lib.smbv_gemm_nt_splitk_workspace_bytes(M, N), A.device)
        res["splitk_ws"] = ws
        check(lib.smbv_gemm_nt_splitk(_p(A), A.stride(0), _p(B), B.stride(0), M, N, K, C.byref(e), _p(ws), ws.numel(), _stream()), "smbv_gemm_nt_splitk")
        return res
    if rope is not None:
        rc = rope_cfg(**{k: v for k, v in rope.items() if k != "wa"})
        check(lib.smbv_gemm_nt_rope(_p(A), A.stride(0), _p(B), B.stride(0), M, N, K, C.byref(e), C.byref(rc), rope["wa"], _stream()), "smbv_gemm_nt_rope")
        return res
    check(lib.smbv_gemm_nt(_p(A), A.stride(0), _p(B), B.stride(0), M, N, K, C.byref(e), _stream()), "smbv_gemm_nt")
    return res


def rope_cfg(table, pos, S, grid, Dh, head_stride, table_rows=None):
    """smbv_rope3d_cfg over live tensors (the caller keeps them alive for the call).  table_rows: default the table's extent; 0 = "unknown" (the map then
    runs as the stand-alone launch)."""
    rc = _lib.Rope3dCfg()
    rc.table, rc.pos, rc.S, rc.grid, rc.Dh, rc.head_stride = table.data_ptr(), (pos.data_ptr() if pos is not None else None), S, grid, Dh, head_stride
    rc.table_rows = table.shape[0] if table_rows is None else table_rows
    return rc


def rope3d_(qkv, wa, H, rope, transpose=False):
    """smbv_rope3d in place on the q | k sections of qkv [rows, ld] (rope: the dict gemm_nt takes, wa / table_rows ignored)."""
    lib = _lib.load()
    check(lib.smbv_rope3d(_p(qkv), qkv.stride(0), wa, qkv.shape[0], rope["S"], H, rope["head_stride"], rope["Dh"], rope["grid"],
                          (rope["pos"].data_ptr() if rope["pos"] is not None else None), rope["table"].data_ptr(), int(transpose), _stream()), "smbv_rope3d")
    return qkv


def gemm_tn(X, Y):
    """out[N1,N2] fp32 = X[M,N1]^T @ Y[M,N2]."""
    _need_gpu(X, Y)
    lib = _lib.load()
    M, N1 = X.shape
    N2 = Y.shape[1]
    out = torch.empty(N1, N2, dtype=torch.float32, device=X.device)
    ws = _ws(lib.smbv_gemm_tn_workspace_bytes(M, N1, N2), X.device)
    check(lib.smbv_gemm_tn(_p(X), X.stride(0), _p(Y), Y.stride(0), M, N1, N2, _p(out), _p(ws), ws.numel(), _stream()), "smbv_gemm_tn")
    return out


def gemm_tn_bias(X, Y):
    """(X^T @ Y fp32 [N1,N2], column sums of X fp32 [N1]): weight and bias gradient of a linear in one launch."""
    _need_gpu(X, Y)
    lib = _lib.load()
    M, N1 = X.shape
    N2 = Y.shape[1]
    out = torch.empty(N1, N2, dtype=torch.float32, device=X.device)
    xs = torch.empty(N1, dtype=torch.float32, device=X.device)
    ws = _ws(lib.smbv_gemm_tn_workspace_bytes(M, N1, N2), X.device)
    check(lib.smbv_gemm_tn_bias(_p(X), X.stride(0), _p(Y), Y.stride(0), M, N1, N2, _p(out), _p(xs), _p(ws), ws.numel(), _stream()), "smbv_gemm_tn_bias")
    return out, xs


def gemm_tn_grouped(pairs, sums=None, out=None, split=False):
    """pairs: list of (X [M,N1], Y [M,N2]) bf16; returns the list of X^T @ Y (fp32) from ONE launch (smbv_gemm_tn_grouped).  sums: per job None or a
    segment count (1..3): also returns that job's column sums of X as a list of `segments` tensors.  split: every tile's token range as two halves by two
    workgroups (smbv_gemm_tn_grouped_split)."""
    lib = _lib.load()
    n = len(pairs)
    jobs = (_lib.TnJob * n)()
    outs, xs = [], []
    for i, (X, Y) in enumerate(pairs):
        _need_gpu(X, Y)
        M, N1 = X.shape
        N2 = Y.shape[1]
        o = out[i] if out is not None else torch.empty(N1, N2, dtype=torch.float32, device=X.device)
        outs.append(o)
        j = jobs[i]
        j.X, j.Y, j.out, j.ldx, j.ldy, j.M, j.N1, j.N2 = X.data_ptr(), Y.data_ptr(), o.data_ptr(), X.stride(0), Y.stride(0), M, N1, N2
        nseg = sums[i] if sums else None
        if nseg:
            segs = [torch.empty(N1 // nseg, dtype=torch.float32, device=X.device) for _ in range(nseg)]
            j.seg = N1 // nseg
            for k, t in enumerate(segs):
                j.sum_dst[k] = t.data_ptr()
            xs.append(segs)
        else:
            j.seg = 0
            xs.append(None)
    if split:
        ws = _ws(max(256, lib.smbv_gemm_tn_grouped_split_workspace_bytes(jobs, n)), pairs[0][0].device)
        check(lib.smbv_gemm_tn_grouped_split(jobs, n, _p(ws), ws.numel(), _stream()), "smbv_gemm_tn_grouped_split")
    else:
        check(lib.smbv_gemm_tn_grouped(jobs, n, _stream()), "smbv_gemm_tn_grouped")
    return (outs, xs) if sums else outs


def layernorm_fwd(x, gamma, beta, eps, rows=None, grp=(0, 0, 0)):
    _need_gpu(x, gamma, beta)
    lib = _lib.load()
    D = x.shape[-1]
    rows = rows if rows is not None else x.numel() // D
    y = torch.empty(rows, D, dtype=torch.bfloat16, device=x.device)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    check(lib.smbv_layernorm_fwd(_p(x), _p(gamma), _p(beta), _p(y), _p(mean), _p(rstd), rows, D, eps, *grp, _stream()), "smbv_layernorm_fwd")
    return y, mean, rstd


def layernorm_bwd(dy, x, mean, rstd, gamma, dres=None, grp=(0, 0, 0)):
    _need_gpu(dy, x)
    lib = _lib.load()
    rows, D = dy.shape
    dx = torch.zeros_like(x, dtype=torch.float32)
    dxb = torch.zeros_like(x, dtype=torch.bfloat16)
    dg = torch.empty(D, dtype=torch.float32, device=x.device)
    db = torch.empty(D, dtype=torch.float32, device=x.device)
    ws = _ws(lib.smbv_layernorm_bwd_workspace_bytes(rows, D), x.device)
    check(lib.smbv_layernorm_bwd(_p(dy), _p(x), _p(mean), _p(rstd), _p(gamma), _p(dres), _p(dx), _p(dxb), _p(dg), _p(db), rows, D, *grp,
                                 _p(ws), ws.numel(), _stream()), "smbv_layernorm_bwd")
    return dx, dxb, dg, db


def attention_fwd(qkv, B, S, H, scale=None, Sq=0, q_off=0, Dh=64, resid=False):
    """qkv: bf16 [B*S, 3*H*Dh] (q | k | v column blocks), Dh 64 or 32.  Returns (O bf16 [B*S, H*Dh], LSE fp32 [B,H,S]); with ``resid`` also
    O_lo = bf16(O_fp32 - O), which attention_bwd takes to form delta from the output to 16 significant bits."""
    _need_gpu(qkv)
    lib = _lib.load()
    w = H * Dh
    scale = scale if scale is not None else Dh ** -0.5
    O = torch.zeros(B * S, w, dtype=torch.bfloat16, device=qkv.device)
    O_lo = torch.zeros_like(O) if resid else None
    lse = torch.empty(B, H, Sq if Sq > 0 else S, dtype=torch.float32, device=qkv.device)
    base = qkv.data_ptr()
    check(lib.smbv_attention_fwd(base, base + 2 * w, base + 4 * w, qkv.stride(0), _p(O), _p(O_lo), w, _p(lse), B, S, H, Dh, scale, Sq, q_off, _stream()),
          "smbv_attention_fwd")
    return (O, lse, O_lo) if resid else (O, lse)


def attention_fwd_fp8(qkv, B, S, H, scale=None, Sq=0, q_off=0):
    """As attention_fwd, on the block-scaled fp8 (OCP e4m3) MFMA path (smbv_attention_fwd_fp8)."""
    _need_gpu(qkv)
    lib = _lib.load()
    w = H * 64
    scale = scale if scale is not None else 64 ** -0.5
    O = torch.zeros(B * S, w, dtype=torch.bfloat16, device=qkv.device)
    lse = torch.empty(B, H, Sq if Sq > 0 else S, dtype=torch.float32, device=qkv.device)
    ws = _ws(lib.smbv_attention_fp8_workspace_bytes(B, S, H), qkv.device)
    base = qkv.data_ptr()
    check(lib.smbv_attention_fwd_fp8(base, base + 2 * w, base + 4 * w, qkv.stride(0), _p(O), w, _p(lse), B, S, H, 64, scale, Sq, q_off, _p(ws), ws.numel(),
                                     _stream()), "smbv_attention_fwd_fp8")
    return O, lse


def attention_bwd(qkv, O, dO, lse, B, S, H, scale=None, parts=7, out=None, Sq=0, q_off=0, Dh=64, O_lo=None, fp8=False, fp8_ws_short=0, split=None, rope=None):
    """rope: dict(table, pos (or None), S, grid, Dh (the real head_dim), head_stride) - smbv_attention_bwd_rope: dQ / dK leave through the transposed rotary map
    (split: None / False = no half sweeps).  fp8: the query-owner blocks recompute S and dP on the block-scaled fp8 MFMA (smbv_attention_bwd_fp8; head_dim 64).  fp8_ws_short: declare the
    workspace that many bytes smaller than it is (the error-path test).  split: True (a fresh scratch) or a uint8 scratch tensor - smbv_attention_bwd_split, the
    form the steps run (the last tiles of each role as two half sweeps)."""
    _need_gpu(qkv, O, dO, lse)
    lib = _lib.load()
    w = H * Dh
    scale = scale if scale is not None else Dh ** -0.5
    dqkv, delta = out if out is not None else (torch.zeros_like(qkv), torch.empty(B, H, Sq if Sq > 0 else S, dtype=torch.float32, device=qkv.device))
    base, dbase = qkv.data_ptr(), dqkv.data_ptr()
    if rope is not None:
        use_split = split is not None and split is not False
        ws = (split if torch.is_tensor(split) else _ws(max(256, lib.smbv_attention_bwd_split_workspace_bytes(B, S, H, Dh)), qkv.device)) if use_split else None
        f8 = _ws(lib.smbv_attention_bwd_fp8_workspace_bytes(B, S, H), qkv.device) if fp8 else None
        rc = rope_cfg(**{k: v for k, v in rope.items() if k != "wa"})
        check(lib.smbv_attention_bwd_rope(base, base + 2 * w, base + 4 * w, qkv.stride(0), _p(O), _p(O_lo), _p(dO), w, _p(lse), _p(delta), dbase, dbase + 2 * w,
                                          dbase + 4 * w, dqkv.stride(0), B, S, H, Dh, scale, parts, Sq, q_off, _p(ws), ws.numel() if use_split else 0, _p(f8),
                                          f8.numel() if fp8 else 0, C.byref(rc), _stream()), "smbv_attention_bwd_rope")
        return dqkv, delta
    if fp8 and (split is None or split is False):
        ws = _ws(lib.smbv_attention_bwd_fp8_workspace_bytes(B, S, H), qkv.device)
        check(lib.smbv_attention_bwd_fp8(base, base + 2 * w, base + 4 * w, qkv.stride(0), _p(O), _p(O_lo), _p(dO), w, _p(lse), _p(delta), dbase, dbase + 2 * w,
                                         dbase + 4 * w, dqkv.stride(0), B, S, H, Dh, scale, parts, Sq, q_off, _p(ws), ws.numel() - fp8_ws_short, _stream()), "smbv_attention_bwd_fp8")
        return dqkv, delta
    if split is not None and split is not False:
        ws = split if torch.is_tensor(split) else _ws(max(256, lib.smbv_attention_bwd_split_workspace_bytes(B, S, H, Dh)), qkv.device)
        f8 = _ws(lib.smbv_attention_bwd_fp8_workspace_bytes(B, S, H), qkv.device) if fp8 else None
        check(lib.smbv_attention_bwd_split(base, base + 2 * w, base + 4 * w, qkv.stride(0), _p(O), _p(O_lo), _p(dO), w, _p(lse), _p(delta), dbase, dbase + 2 * w,
                                           dbase + 4 * w, dqkv.stride(0), B, S, H, Dh, scale, parts, Sq, q_off, _p(ws), ws.numel(), _p(f8), f8.numel() if fp8 else 0,
                                           _stream()), "smbv_attention_bwd_split")
        return dqkv, delta
    check(lib.smbv_attention_bwd(base, base + 2 * w, base + 4 * w, qkv.stride(0), _p(O), _p(O_lo), _p(dO), w, _p(lse), _p(delta), dbase, dbase + 2 * w,
                                 dbase + 4 * w, dqkv.stride(0), B, S, H, Dh, scale, parts, Sq, q_off, _stream()), "smbv_attention_bwd")
    return dqkv, delta


def gather_bricks(pix, idx, per_batch, ts, ps):
    _need_gpu(pix, idx)
    lib = _lib.load()
    B, T, Cc, H, W = pix.shape
    rows = idx.numel()
    out = torch.empty(rows, ts * ps * ps, dtype=torch.bfloat16, device=pix.device)
    check(lib.smbv_gather_bricks(_p(pix), _p(idx), rows, per_batch, _p(out), T, H, W, ts, ps, _stream()), "smbv_gather_bricks")
    return out


def brick_stats(pix, idx, per_batch, ts, ps):
    _need_gpu(pix, idx)
    lib = _lib.load()
    B, T, Cc, H, W = pix.shape
    rows = idx.numel()
    mean = torch.empty(rows, dtype=torch.float32, device=pix.device)
    rinv = torch.empty(rows, dtype=torch.float32, device=pix.device)
    check(lib.smbv_brick_stats(_p(pix), _p(idx), rows, per_batch, _p(mean), _p(rinv), T, H, W, ts, ps, _stream()), "smbv_brick_stats")
    return mean, rinv


def mse_fwd(pix, idx, per_batch, mean, rinv, logits, ts, ps):
    lib = _lib.load()
    B, T, Cc, H, W = pix.shape
    rows = idx.numel()
    part = torch.empty(rows, dtype=torch.float32, device=pix.device)
    loss = torch.empty(1, dtype=torch.float32, device=pix.device)
    check(lib.smbv_mse_fwd(_p(pix), _p(idx), rows, per_batch, _p(mean), _p(rinv), _p(logits), _p(part), _p(loss), T, H, W, ts, ps, _stream()),
          "smbv_mse_fwd")
    return loss


def mse_bwd(pix, idx, per_batch, mean, rinv, logits, ts, ps, gscale=None):
    lib = _lib.load()
    B, T, Cc, H, W = pix.shape
    rows = idx.numel()
    dl = torch.empty_like(logits)
    check(lib.smbv_mse_bwd(_p(pix), _p(idx), rows, per_batch, _p(mean), _p(rinv), _p(logits), _p(dl), _p(gscale), T, H, W, ts, ps, _stream()),
          "smbv_mse_bwd")
    return dl


def cast_bf16(x):
    lib = _lib.load()
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    check(lib.smbv_cast_f32_bf16(_p(x), _p(out), x.numel(), _stream()), "smbv_cast_f32_bf16")
    return out


def transpose_cast_bf16(x):
    lib = _lib.load()
    R, Cc = x.shape
    out = torch.empty(Cc, R, dtype=torch.bfloat16, device=x.device)
    check(lib.smbv_transpose_cast_f32_bf16(_p(x), _p(out), R, Cc, R, _stream()), "smbv_transpose_cast_f32_bf16")
    return out


def colsum_bf16(X):
    lib = _lib.load()
    M, N = X.shape
    out = torch.empty(N, dtype=torch.float32, device=X.device)
    ws = _ws(lib.smbv_colsum_workspace_bytes(M, N), X.device)
    check(lib.smbv_colsum_bf16(_p(X), X.stride(0), M, N, _p(out), _p(ws), ws.numel(), _stream()), "smbv_colsum_bf16")
    return out


# ---- operators of a transformer block over long token sequences: windowed attention with sinks, rotary positions with several axes, gated norms ------------
# A call's checks and its C arguments but for the addresses follow from shapes, strides, types and numbers alone: they are worked out once for each such
# signature (a call for one token is bound by what the host does for it: 38 us without, 9 with, 3.5 of them the launch).
_NORMS = {None: 0, "rms": 1, "layer": 2}
_EL16 = {torch.bfloat16: 0, torch.float16: 1}
_EL = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_PLANS = {}


def _meta(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _packed(shape):
    """The strides of a contiguous tensor."""
    out, n = [], 1
    for x in reversed(shape):
        out.append(n)
        n *= max(x, 1)
    return tuple(reversed(out))


class _Plan:
    """One signature's C arguments without addresses, and the outputs to allocate; the entry point and its workspace's size once it has been called."""
    __slots__ = ("args", "new", "fn", "ws_bytes")

    def __init__(self, args, device, *new):
        self.args, self.fn, self.ws_bytes = args, None, 0
        # (a stated layout is the quickest way to an empty tensor: 1.3 us; torch.empty 1.8)
        self.new = [(tuple(shape), _packed(shape), dtype, device) for shape, dtype in new]

    def empty(self, i):
        shape, stride, dtype, device = self.new[i]
        return _empty_strided(shape, stride, dtype=dtype, device=device)


_empty_strided = torch.empty_strided


def _keep(key, plan):
    if len(_PLANS) >= 1024:
        _PLANS.clear()
    _PLANS[key] = plan
    return plan


def _call(plan, name, args, device, workspace=True):
    """The entry point on the tensors' device and the current stream."""
    if torch._C._cuda_getDevice() != device.index:
        with torch.cuda.device(device):
            return _call(plan, name, args, device, workspace)
    if plan.fn is None:
        lib = _lib.load()
        size = getattr(lib, name + "_workspace_bytes", None) if workspace else None
        plan.ws_bytes = int(size(C.byref(args))) if size else 0
        plan.fn = getattr(lib, name)
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if not workspace:
        check(plan.fn(C.byref(args), stream), name)
    elif plan.ws_bytes == 0:
        check(plan.fn(C.byref(args), None, 0, stream), name)
    else:
        ws = torch.empty(plan.ws_bytes, dtype=torch.uint8, device=device)
        check(plan.fn(C.byref(args), ws.data_ptr(), plan.ws_bytes, stream), name)


def _same_device(first, *ts):
    for t in ts:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")


def _ll3(t):
    """Strides of the first three dimensions (a dimension of one element has no stride to speak of)."""
    return _lib.c_ll3(*(0 if t.shape[i] <= 1 else t.stride(i) for i in range(3)))


def _ll3_packed(shape):
    _, r, h, c = shape
    return _lib.c_ll3(r * h * c, h * c, c)


def _heads4(t, name, shape, dtype):
    if t.dim() != 4 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name}: the channels must be contiguous")


def _extent(t):
    if t.numel() == 0:
        return 0, 0
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _writable(t, name, inputs=()):
    """A caller's output: its elements lie apart from each other and from every input."""
    span = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if s < span:
            raise ValueError(f"{name}: elements of an output must not share memory")
        span = (n - 1) * s + span
    lo, hi = _extent(t)
    for x in inputs:
        if x is not None:
            a, b = _extent(x)
            if a < hi and lo < b:
                raise ValueError(f"{name}: an output must not overlap an operand")


def _apart(*ts):
    """Tensors [B, S, H, D] of one call, of which at least one of any two is written, lie apart: nowhere near each other, or as columns of one packed tensor (equal
    steps between rows, other places in them)."""
    ts = [t for t in ts if t is not None and t.numel()]
    for n, a in enumerate(ts):
        for b in ts[n + 1:]:
            (lo, hi), (lo2, hi2) = _extent(a), _extent(b)
            if hi <= lo2 or hi2 <= lo:
                continue
            steps = [i for i in (0, 1) if a.shape[i] > 1 or b.shape[i] > 1]
            row = min((a.stride(i) for i in steps), default=0)
            wa, wb = ((t.shape[2] - 1) * t.stride(2) + t.shape[3] for t in (a, b))
            if row > 0 and all(a.stride(i) == b.stride(i) and a.stride(i) % row == 0 for i in steps):
                at = (lo2 - lo) // a.element_size() % row
                if at >= wa and at + wb <= row:
                    continue
            raise ValueError("out: tensors that share no memory")


def _window_args(q, k, v, left, right, sinks, scale, q_lens, k_lens):
    _need_gpu(q, k, v, q_lens, k_lens)
    _same_device(q, k, v, q_lens, k_lens)
    if q.dtype not in _EL16:
        raise ValueError(f"window attention: bf16 or fp16, got {q.dtype}")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"window attention: q [B, Sq, H, D] and k, v [B, Sk, Hk, D], got {tuple(q.shape)}, {tuple(k.shape)}")
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1], k.shape[2]
    _heads4(q, "q", (B, Sq, H, D), q.dtype)
    _heads4(k, "k", (B, Sk, Hk, D), q.dtype)
    _heads4(v, "v", (B, Sk, Hk, D), q.dtype)
    for name, t in (("q_lens", q_lens), ("k_lens", k_lens)):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous()):
            raise ValueError(f"{name}: a contiguous int32 tensor of {B} lengths")
    a = _lib.WindowAttn()
    a.dtype, a.B, a.Sq, a.Sk, a.H, a.Hk, a.Dh = _EL16[q.dtype], B, Sq, Sk, H, Hk, D
    a.left, a.right = (min(max(x, -1), 2 ** 31 - 1) for x in (left, right))
    if not 0 <= sinks < 2 ** 31:
        raise ValueError(f"sinks: {sinks}")
    a.sinks, a.scale = sinks, D ** -0.5 if scale is None else scale
    a.sq, a.sk, a.sv = _ll3(q), _ll3(k), _ll3(v)
    return a


def window_attention_fwd(q, k, v, *, left=-1, right=-1, sinks=0, scale=None, q_lens=None, k_lens=None, resid=False, out=None):
    """Softmax attention inside a sliding window, with a few first tokens that stay visible (smbv_window_attention_fwd).

    q [B, Sq, H, D], k / v [B, Sk, Hk, D] (bf16 or fp16, any batch / row / head strides that are multiples of 8 elements - rows of k and v less than 2^24
    elements apart -, H a multiple of Hk, D a multiple of 8 up to 128).  Query i stands at position p = i + k_len - q_len and sees key j iff j < k_len, j <= p + right (right < 0: no bound; 0: causal) and
    (j >= p - left (left < 0: no bound) or j < sinks).  q_lens / k_lens: int32 [B] on the device (None: Sq / Sk), so the queries are the last rows of their
    sequence: all of them in training, the newest tokens against a cache in serving (Sq = 1; the whole cache with k_lens keeps the call's signature).  A row that sees nothing, padded rows included, is 0 with lse -inf.
    Keys that no row of a call can see do not take part, whatever they hold; a NaN or infinity in a value that SOME rows see can reach other rows near them that
    see something.

    Returns (o [B, Sq, H, D], lse fp32 [B, H, Sq]) and with ``resid`` also the residual of o's rounding, which window_attention_bwd takes as ``o_lo``.
    out: a tensor for o (its strides free; with ``resid`` the residual gets a tensor of the same strides)."""
    left, right, sinks, scale = int(left), int(right), int(sinks), None if scale is None else float(scale)
    device = q.device
    key = ("window_fwd", q.shape, q.stride(), q.dtype, device, k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device,
           left, right, sinks, scale, _meta(q_lens), _meta(k_lens), _meta(out))
    plan = _PLANS.get(key)
    if plan is None:
        a = _window_args(q, k, v, left, right, sinks, scale, q_lens, k_lens)
        if out is not None:
            _need_gpu(out)
            _same_device(q, out)
            _heads4(out, "out", q.shape, q.dtype)
        a.so = _ll3_packed(q.shape) if out is None else _ll3(out)
        plan = _keep(key, _Plan(a, device, (q.shape, q.dtype), ((a.B, a.H, a.Sq), torch.float32)))
    if out is None:
        o = plan.empty(0)
    else:
        _writable(out, "out", (q, k, v, q_lens, k_lens))
        o = out
    o_lo = _empty_strided(o.shape, o.stride(), dtype=o.dtype, device=device) if resid else None
    lse = plan.empty(1)
    a = _lib.WindowAttn.from_buffer_copy(plan.args)
    a.q_lens, a.k_lens, a.q, a.k, a.v, a.o, a.o_lo, a.lse = _p(q_lens), _p(k_lens), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _p(o_lo), lse.data_ptr()
    _call(plan, "smbv_window_attention_fwd", a, device)
    return (o, lse, o_lo) if resid else (o, lse)


def window_attention_bwd(q, k, v, o, do, lse, *, left=-1, right=-1, sinks=0, scale=None, q_lens=None, k_lens=None, o_lo=None, out=None):
    """Gradients (dq, dk, dv) of window_attention_fwd (the same keyword arguments; o, lse and o_lo as it returned them; do: the gradient of o, any strides).
    A key head's gradient is the sum over its query heads.  Every element is written; the same call gives the same bits.  In fp16, |v| above 16000 / D with
    signs that agree can overflow (dS is held in units of the largest |do|).  out: three tensors for the gradients, for instance the column blocks of one
    packed gradient."""
    left, right, sinks, scale = int(left), int(right), int(sinks), None if scale is None else float(scale)
    outs = (None,) * 3 if out is None else tuple(out)
    key = ("window_bwd", _meta(q), _meta(k), _meta(v), _meta(o), _meta(do), _meta(lse), left, right, sinks, scale, _meta(q_lens), _meta(k_lens), _meta(o_lo),
           out is None, *(_meta(t) for t in outs))
    plan = _PLANS.get(key)
    if plan is None:
        a = _window_args(q, k, v, left, right, sinks, scale, q_lens, k_lens)
        _need_gpu(o, do, lse, o_lo)
        _same_device(q, o, do, lse, o_lo)
        for name, t in (("o", o), ("do", do), ("o_lo", o_lo)):
            if t is not None:
                _heads4(t, name, q.shape, q.dtype)
        if o_lo is not None and list(_ll3(o_lo)) != list(_ll3(o)):
            raise ValueError("o_lo: the strides of o")
        if lse.dtype != torch.float32 or tuple(lse.shape) != (a.B, a.H, a.Sq) or not lse.is_contiguous():
            raise ValueError(f"lse: a contiguous fp32 tensor of shape {(a.B, a.H, a.Sq)}")
        for name, t, like in zip(("dq", "dk", "dv"), outs, (q, k, v)):
            if out is not None:
                if t is None:
                    raise ValueError("out: three tensors")
                _need_gpu(t)
                _same_device(q, t)
                _heads4(t, name, like.shape, q.dtype)
        a.so, a.sdo = _ll3(o), _ll3(do)
        a.sdq, a.sdk, a.sdv = (_ll3_packed(like.shape) if t is None else _ll3(t) for t, like in zip(outs, (q, k, v)))
        plan = _keep(key, _Plan(a, q.device, *((t.shape, q.dtype) for t in (q, k, v))))
    if out is None:
        dq, dk, dv = plan.empty(0), plan.empty(1), plan.empty(2)
    else:
        dq, dk, dv = outs
        for name, t in zip(("dq", "dk", "dv"), outs):
            _writable(t, name, (q, k, v, o, do, o_lo, lse, q_lens, k_lens))
        _apart(*outs)
    a = _lib.WindowAttn.from_buffer_copy(plan.args)
    a.q_lens, a.k_lens, a.q, a.k, a.v = _p(q_lens), _p(k_lens), q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.o, a.o_lo, a.lse, a.d_o, a.dq, a.dk, a.dv = o.data_ptr(), _p(o_lo), lse.data_ptr(), do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    _call(plan, "smbv_window_attention_bwd", a, q.device)
    return dq, dk, dv


def rope_axes(q, k, pos, inv_freq, sections, *, interleaved=False, transpose=False, out=None):
    """Rotary positions with several axes on queries and keys (smbv_rope_axes).  q [B, S, H, D], k [B, S, Hk, D] or None (bf16, fp16 or fp32, any strides with
    contiguous channels, D even up to 1024); pos: int32 or int64 positions [axes, B, S] or [axes, S]; sections: how many pairs each of up to four axes owns,
    in order; inv_freq: fp32 [sum(sections)].  Pair p turns by pos[its axis] * inv_freq[p]; the first 2 * sum(sections) channels of a head are the pairs
    (p, p + sum(sections)), or (2p, 2p + 1) with ``interleaved``; the rest stays.  transpose: the inverse turn - what a gradient goes through on the way back.
    Returns (q', k'); out: tensors for them, (q, k) themselves to turn in place."""
    sections = tuple(map(int, sections))
    qo, ko = (None, None) if out is None else out
    device = q.device
    key = ("rope_axes", q.shape, q.stride(), q.dtype, device, _meta(k), pos.shape, pos.stride(), pos.dtype, pos.device, inv_freq.shape, inv_freq.stride(),
           inv_freq.dtype, inv_freq.device, sections, interleaved, transpose, out is None, _meta(qo), _meta(ko))
    plan = _PLANS.get(key)
    if plan is None:
        _need_gpu(q, k, pos, inv_freq)
        _same_device(q, k, pos, inv_freq)
        if q.dtype not in _EL:
            raise ValueError(f"rope_axes: bf16, fp16 or fp32, got {q.dtype}")
        if q.dim() != 4:
            raise ValueError(f"q: expected [B, S, H, D], got {tuple(q.shape)}")
        B, S, H, D = q.shape
        Hk = 0 if k is None else (k.shape[2] if k.dim() == 4 else -1)
        _heads4(q, "q", (B, S, H, D), q.dtype)
        if k is not None:
            _heads4(k, "k", (B, S, Hk, D), q.dtype)
        if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) <= 0 or 2 * sum(sections) > D:
            raise ValueError(f"sections {sections}: one to four axes that own between them 1 .. {D // 2} pairs")
        if pos.dtype not in (torch.int32, torch.int64) or tuple(pos.shape) not in ((len(sections), B, S), (len(sections), S)):
            raise ValueError(f"pos: int32 or int64 of shape {(len(sections), B, S)} or {(len(sections), S)}, got {pos.dtype} {tuple(pos.shape)}")
        if inv_freq.dtype != torch.float32 or tuple(inv_freq.shape) != (sum(sections),) or not inv_freq.is_contiguous():
            raise ValueError(f"inv_freq: a contiguous fp32 tensor of {sum(sections)} frequencies")
        a = _lib.RopeAxesCfg()
        a.dtype, a.B, a.S, a.H, a.Hk, a.Dh, a.axes = _EL[q.dtype], B, S, H, Hk, D, len(sections)
        a.section = (C.c_int * 4)(*sections)
        a.interleaved, a.transpose, a.pos64 = int(interleaved), int(transpose), int(pos.dtype == torch.int64)
        for name, t, like, s_in, s_out in (("q", qo, q, "sq", "sqo"), ("k", ko, k, "sk", "sko")):
            if out is not None and (t is None) != (like is None):
                raise ValueError("out: one tensor for each of q and k")
            if like is None:
                continue
            setattr(a, s_in, _ll3(like))
            setattr(a, s_out, _ll3_packed(like.shape) if t is None else _ll3(t))
            if t is not None:
                _need_gpu(t)
                _same_device(q, t)
                _heads4(t, f"out of {name}", like.shape, q.dtype)
        a.spos = _lib.c_ll3(pos.stride(0), pos.stride(1) if pos.dim() == 3 else 0, pos.stride(-1))
        plan = _keep(key, _Plan(a, device, (q.shape, q.dtype), *(() if k is None else ((k.shape, q.dtype),))))
    if out is None:
        qo = plan.empty(0)
        ko = None if k is None else plan.empty(1)
    else:
        for name, t, like, other in (("q", qo, q, k), ("k", ko, k, q)):
            if t is not None:
                in_place = t.data_ptr() == like.data_ptr() and list(_ll3(t)) == list(_ll3(like))
                _writable(t, f"out of {name}", (pos, inv_freq) if in_place else (q, k, pos, inv_freq))
                if in_place:   # beside the other operand's columns of one packed projection is fine, on elements that are still to be read is not
                    _apart(t, other)
        _apart(qo, ko)
    a = _lib.RopeAxesCfg.from_buffer_copy(plan.args)
    a.q, a.k, a.qo, a.ko, a.pos, a.inv_freq = q.data_ptr(), _p(k), qo.data_ptr(), _p(ko), pos.data_ptr(), inv_freq.data_ptr()
    _call(plan, "smbv_rope_axes", a, device, False)
    return qo, ko


def _rows2(t, name, lead, d, dtype):
    """The stride between the rows of t [*lead, d]."""
    if t.dtype != dtype or tuple(t.shape) != (*lead, d):
        raise ValueError(f"{name}: expected {dtype} {(*lead, d)}, got {t.dtype} {tuple(t.shape)}")
    if d > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: rows must be contiguous")
    try:
        r = t.view(-1, d) if t.numel() else t.reshape(0, d)
    except RuntimeError:
        raise ValueError(f"{name}: the leading dimensions must have one stride between rows") from None
    return r.stride(0) if r.shape[0] > 1 else d


def _gated_norm_args(h, x, post, post_w, post_b, gate, res_scale, pre, pre_w, pre_b, eps):
    _need_gpu(h, x, post_w, post_b, gate, pre_w, pre_b)
    _same_device(h, x, post_w, post_b, gate, pre_w, pre_b)
    if post not in _NORMS or pre not in _NORMS:
        raise ValueError(f"norms: 'rms', 'layer' or None, got {post!r}, {pre!r}")
    if h.dtype not in _EL or x.dtype not in (h.dtype, torch.float32):
        raise ValueError(f"h: bf16, fp16 or fp32; x: the same or fp32; got {h.dtype}, {x.dtype}")
    if h.dim() < 1 or h.shape[-1] == 0:
        raise ValueError(f"h: rows of at least one element, got {tuple(h.shape)}")
    d, lead = h.shape[-1], tuple(h.shape[:-1])
    a = _lib.GatedNorm()
    a.ldh = _rows2(h, "h", lead, d, h.dtype)
    a.ldx = _rows2(x, "x", lead, d, x.dtype)
    rows = h.numel() // d
    for name, t in (("post_w", post_w), ("post_b", post_b), ("pre_w", pre_w), ("pre_b", pre_b)):
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (d,) or not t.is_contiguous()):
            raise ValueError(f"{name}: a contiguous fp32 tensor of {d} elements")
    a.h_type, a.x_type, a.d, a.post, a.pre, a.eps, a.res_scale, a.rows = _EL[h.dtype], _EL[x.dtype], d, _NORMS[post], _NORMS[pre], eps, res_scale, rows
    a.rows_per_gate = max(rows, 1)
    if gate is not None:
        if gate.dtype != torch.float32 or gate.dim() < 1 or gate.shape[-1] != d or not gate.is_contiguous():
            raise ValueError(f"gate: a contiguous fp32 tensor of rows of {d}")
        of = list(gate.shape[:-1])
        while of and of[-1] == 1:
            of.pop()
        groups = gate.numel() // d
        if (len(lead) != 1 and tuple(of) != lead[:len(of)]) or (groups == 0) != (rows == 0 and groups == 0) or (groups and rows % groups):
            raise ValueError(f"gate {tuple(gate.shape)}: one row, or one for each of h's leading dimensions {lead}")
        if groups:
            a.rows_per_gate = max(rows // groups, 1)
    return a, lead, d


def gated_norm_fwd(h, x, *, post="rms", post_w=None, post_b=None, gate=None, res_scale=1.0, pre="rms", pre_w=None, pre_b=None, eps=1e-6, out=None):
    """The norm behind a block, its gate, the scaled residual sum and the norm in front of the next block (smbv_gated_norm_fwd):

        x1 = res_scale * x + gate * post(h),    y = pre(x1)

    h [..., d]: the block's output (bf16, fp16, fp32); x: the residual stream (h's type or fp32); post / pre: "rms", "layer" or None, their weights and biases
    fp32 [d] or None (1 and 0); gate: fp32 [d], or one row for each of h's leading dimensions ([B, d] or [B, 1, d] for h [B, S, d]; for h [rows, d] any
    [n, d] whose n divides the rows: one gate for rows / n consecutive rows).  y is formed from x1 before its rounding.  Rows up to 8192 wide.

    Returns (x1 in x's type, y in h's type or None without ``pre``, stats fp32 [rows, 4] for gated_norm_bwd).  out: (x1, y), x1 may be x itself."""
    eps, res_scale = float(eps), float(res_scale)
    x1, y = (None, None) if out is None else out
    device = h.device
    key = ("gated_norm_fwd", h.shape, h.stride(), h.dtype, device, x.shape, x.stride(), x.dtype, x.device, post, _meta(post_w), _meta(post_b), _meta(gate), res_scale,
           pre, _meta(pre_w), _meta(pre_b), eps, out is None, _meta(x1), _meta(y))
    plan = _PLANS.get(key)
    if plan is None:
        a, lead, d = _gated_norm_args(h, x, post, post_w, post_b, gate, res_scale, pre, pre_w, pre_b, eps)
        if out is not None:
            if x1 is None or (y is None) != (pre is None):
                raise ValueError("out: (x1, y), y None exactly when there is no norm in front of the next block")
            _need_gpu(x1, y)
            _same_device(h, x1, y)
        a.ldx1 = d if x1 is None else _rows2(x1, "x1", lead, d, x.dtype)
        a.ldy = d if y is None else _rows2(y, "y", lead, d, h.dtype)
        plan = _keep(key, _Plan(a, device, (x.shape, x.dtype), (h.shape, h.dtype), ((a.rows, 4), torch.float32)))
    if out is None:
        x1 = plan.empty(0)
        y = plan.empty(1) if pre else None
    else:
        params = (h, post_w, post_b, gate, pre_w, pre_b)
        _writable(x1, "x1", params if x1.data_ptr() == x.data_ptr() and plan.args.ldx1 == plan.args.ldx else (*params, x))
        if y is not None:
            _writable(y, "y", (*params, x, x1))
    stats = plan.empty(2)
    a = _lib.GatedNorm.from_buffer_copy(plan.args)
    a.h, a.x, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b = h.data_ptr(), x.data_ptr(), _p(post_w), _p(post_b), _p(gate), _p(pre_w), _p(pre_b)
    a.x1, a.y, a.stats = x1.data_ptr(), _p(y), stats.data_ptr()
    _call(plan, "smbv_gated_norm_fwd", a, device, False)
    return x1, y, stats


def gated_norm_bwd(dx1, dy, h, x, stats, *, post="rms", post_w=None, post_b=None, gate=None, res_scale=1.0, pre="rms", pre_w=None, pre_b=None, out=None):
    """Gradients of gated_norm_fwd (the same keyword arguments; h, x: its inputs; stats as it returned them).  dx1: the gradient that reaches x1 from elsewhere
    (x's type, or None), dy: that of y (h's type; None without ``pre``).  Returns a dict: "dh", "dx" and, for every parameter that was given, its fp32
    gradient under its name ("gate", "post_w", "post_b", "pre_w", "pre_b"; None for the others).  The same call gives the same bits.  out: (dh, dx)."""
    res_scale = float(res_scale)
    dh, dx = (None, None) if out is None else out
    key = ("gated_norm_bwd", _meta(dx1), _meta(dy), _meta(h), _meta(x), _meta(stats), post, _meta(post_w), _meta(post_b), _meta(gate), res_scale,
           pre, _meta(pre_w), _meta(pre_b), out is None, _meta(dh), _meta(dx))
    plan = _PLANS.get(key)
    if plan is None:
        a, lead, d = _gated_norm_args(h, x, post, post_w, post_b, gate, res_scale, pre, pre_w, pre_b, 0.0)
        _need_gpu(dx1, dy, stats, dh, dx)
        _same_device(h, dx1, dy, stats, dh, dx)
        if (dy is None) != (pre is None) or (dx1 is None and dy is None):
            raise ValueError("dy: given exactly when there is a norm in front of the next block; without it dx1 is needed")
        if out is not None and (dh is None or dx is None):
            raise ValueError("out: (dh, dx)")
        if stats.dtype != torch.float32 or tuple(stats.shape) != (a.rows, 4) or not stats.is_contiguous():
            raise ValueError(f"stats: a contiguous fp32 tensor of shape {(a.rows, 4)}")
        if dx1 is not None:
            a.lddx1 = _rows2(dx1, "dx1", lead, d, x.dtype)
        if dy is not None:
            a.lddy = _rows2(dy, "dy", lead, d, h.dtype)
        a.lddh = d if out is None else _rows2(dh, "dh", lead, d, h.dtype)
        a.lddx = d if out is None else _rows2(dx, "dx", lead, d, x.dtype)
        plan = _keep(key, _Plan(a, h.device, (h.shape, h.dtype), (x.shape, x.dtype)))
    if out is None:
        dh, dx = plan.empty(0), plan.empty(1)
    else:
        ins = (h, x, dx1, dy, stats, post_w, post_b, gate, pre_w, pre_b)
        _writable(dh, "dh", (*ins, dx))
        _writable(dx, "dx", ins)
    new = torch.empty_like if plan.args.rows else torch.zeros_like  # (no rows: nothing is launched, the sums are empty)
    gr = {n: None if t is None else new(t) for n, t in (("gate", gate), ("post_w", post_w), ("post_b", post_b), ("pre_w", pre_w), ("pre_b", pre_b))}
    a = _lib.GatedNorm.from_buffer_copy(plan.args)
    a.h, a.x, a.post_w, a.post_b, a.gate, a.pre_w, a.pre_b = h.data_ptr(), x.data_ptr(), _p(post_w), _p(post_b), _p(gate), _p(pre_w), _p(pre_b)
    a.dx1, a.dy, a.stats, a.dh, a.dx = _p(dx1), _p(dy), stats.data_ptr(), dh.data_ptr(), dx.data_ptr()
    a.dgate, a.dpost_w, a.dpost_b, a.dpre_w, a.dpre_b = (_p(gr[n]) for n in ("gate", "post_w", "post_b", "pre_w", "pre_b"))
    _call(plan, "smbv_gated_norm_bwd", a, h.device)
    return {"dh": dh, "dx": dx, **gr}


def device_status(clear=False) -> int:
    """smbv_device_status: 0, or SMBV_ERR_STATE (-5) once a kernel of an earlier call has recorded a fault on the current device (text: _lib.last_error())."""
    return int(_lib.load().smbv_device_status(1 if clear else 0))


def debug_pair_state(op: int):
    """smbv_debug_pair_state: 0 = restore the library's device-side scheduling state (attention backward tile queues / tickets / split-sweep flags, the split
    weight-gradient launch's tickets / flags) and the host's launch epochs; test hooks: 1 = dirty the slots, 2 + 4 e = raise every hand-off flag as an unfinished
    launch of epoch e would have left it."""
    check(_lib.load().smbv_debug_pair_state(int(op), _stream()), "smbv_debug_pair_state")

