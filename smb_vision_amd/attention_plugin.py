"""The MI355X attention kernels behind the reference's own operator plug-in point.

Both reference models pick their attention implementation from transformers' registry by name:
`ALL_ATTENTION_FUNCTIONS[config._attn_implementation]` (src/models/vjepa/modeling_vjepa.py:345-364, 790-809, 865-884;
src/models/videomae/modeling_videomae.py:270-289), called as

    attention_interface(module, query[B,H,S,Dh], key, value, mask_or_None, is_causal=..., scaling=..., dropout=...)
        -> (context[B,S,H,Dh], attention_probs_or_None)

and the reference's launch scripts select `flash_attention_2` there (src/run_vjepa.py:230-231).  `register()` adds the name "smbv":
a model built from the reference's unmodified classes runs `smbv_attention_fwd` / `smbv_attention_bwd` (include/smbv.h) for its
softmax(QK^T * scaling) V and everything else in PyTorch.  This is the operator-level drop-in; the fused train step
(modeling_videomae.py / modeling_vjepa.py) is the shipped path and avoids the head-major <-> token-major copies this interface forces.

No fallback: anything the kernels do not compute (masks, dropout, causal, head widths other than 64 / 32, no GPU) raises.

`register_window()` adds "smbv_window": smbv_window_attention_fwd / _bwd under the same interface - a sliding window (bound at registration, or the model's own
`sliding_window`), first tokens that stay visible, causal models, grouped key heads, queries at the end of a longer cache, bf16 and fp16, head widths that are
multiples of 8 up to 128 - and without copies, since those kernels take the head-major strides as they are.  With the name goes a mask function: a model that
builds masks has them turned into the window that they say, and one that is no window of full sequences (padding, packed documents, blocks, a cache with empty
slots) raises.
"""
import functools

import torch

from . import ops

NAME = "smbv"
WINDOW_NAME = "smbv_window"


class _SmbvAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, scaling):
        B, H, S, Dh = query.shape
        # the kernels read token-major rows [B*S, q | k | v column blocks of H*Dh]
        qkv = torch.empty(B * S, 3 * H * Dh, dtype=torch.bfloat16, device=query.device)
        packed = qkv.view(B, S, 3, H, Dh)
        packed[:, :, 0].copy_(query.transpose(1, 2))
        packed[:, :, 1].copy_(key.transpose(1, 2))
        packed[:, :, 2].copy_(value.transpose(1, 2))
        out, lse, out_lo = ops.attention_fwd(qkv, B, S, H, scale=scaling, Dh=Dh, resid=True)  # (+ the bf16 residual of the fp32 output, for delta)
        ctx.save_for_backward(qkv, out, lse, out_lo)
        ctx.dims = (B, H, S, Dh, scaling, query.dtype)
        return out.view(B, S, H, Dh).to(query.dtype)

    @staticmethod
    def backward(ctx, d_out):
        qkv, out, lse, out_lo = ctx.saved_tensors
        B, H, S, Dh, scaling, dtype = ctx.dims
        d_rows = d_out.reshape(B * S, H * Dh).to(torch.bfloat16).contiguous()
        d_qkv, _ = ops.attention_bwd(qkv, out, d_rows, lse, B, S, H, scale=scaling, Dh=Dh, O_lo=out_lo)
        d = d_qkv.view(B, S, 3, H, Dh)
        return (d[:, :, 0].transpose(1, 2).to(dtype), d[:, :, 1].transpose(1, 2).to(dtype), d[:, :, 2].transpose(1, 2).to(dtype), None)


def smbv_attention(module, query, key, value, attention_mask=None, *, scaling=None, dropout=0.0, is_causal=False, **kwargs):
    """transformers attention-interface function (same contract as its `eager_attention_forward`): bf16 MFMA arithmetic, fp32 softmax
    statistics; returns (context [B, S, H, Dh] in the dtype of `query`, None)."""
    _refuse(kwargs)
    if attention_mask is not None and not (isinstance(attention_mask, _WindowMask) and (attention_mask.left, attention_mask.right) == (-1, -1)):
        raise ValueError("smbv attention: attention / head masks are not supported (the reference's training path passes None), nor is a model's causal or sliding one")
    if dropout:
        raise ValueError("smbv attention: attention dropout is not supported (the reference trains with attention_probs_dropout_prob = 0)")
    if is_causal:
        raise ValueError("smbv attention: bidirectional attention only")
    if query.dim() != 4 or key.shape != query.shape or value.shape != query.shape:
        raise ValueError(f"smbv attention: expected query / key / value of one shape [B, H, S, Dh], got {tuple(query.shape)}, "
                         f"{tuple(key.shape)}, {tuple(value.shape)}")
    if query.shape[-1] not in (64, 32):
        raise ValueError(f"smbv attention: head width {query.shape[-1]} has no native build (64 and 32 do)")
    if not _on_gpu(query):
        raise RuntimeError("smbv attention needs an MI355X: there is no CPU path")
    if scaling is None:
        scaling = query.shape[-1] ** -0.5
    return _SmbvAttentionFn.apply(query, key, value, float(scaling)), None


def register(name=NAME):
    """Make `config._attn_implementation = name` select the MI355X kernels (transformers.AttentionInterface); a model's own masks raise
    unless they show everything (transformers.AttentionMaskInterface)."""
    from transformers import AttentionInterface, AttentionMaskInterface
    AttentionInterface.register(name, smbv_attention)
    AttentionMaskInterface.register(name, _window_mask)
    return name


def _not_captured():
    # (autograd's own nodes of a leaf stay on the stream that first used them: a backward pass captured while an eager graph of the same leaves lives ends the
    # process.  ops.window_attention_fwd / _bwd are what a captured training step calls.)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("smbv window attention: training through autograd cannot be captured into a graph; capture ops.window_attention_fwd / _bwd instead")


class _SmbvWindowAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kw, train):
        if not train:
            return ops.window_attention_fwd(q, k, v, **kw)[0]
        _not_captured()
        out, lse, out_lo = ops.window_attention_fwd(q, k, v, resid=True, **kw)
        ctx.save_for_backward(q, k, v, out, lse, out_lo)
        ctx.kw = kw
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        _not_captured()
        q, k, v, out, lse, out_lo = ctx.saved_tensors
        return (*ops.window_attention_bwd(q, k, v, out, _rows_of_heads(d_out.to(q.dtype)), lse, o_lo=out_lo, **ctx.kw), None, None)


# Arguments that models hand on and that change nothing here: what positions, masks and outputs they name is settled before the attention or behind it.
_HARMLESS = {"position_ids", "cache_position", "use_cache", "output_attentions", "output_hidden_states", "output_router_logits", "return_dict",
             "encoder_hidden_states", "num_items_in_batch", "deterministic"}   # (the kernels always are)


def _refuse(kwargs):
    for name, x in kwargs.items():
        if x is not None and name not in _HARMLESS:
            raise ValueError(f"smbv attention: the argument {name!r} is not supported (a cap on the scores, learned sinks, a bias: they change the result)")


def _on_gpu(t):
    return t.is_cuda


class _WindowMask:
    """What a model's mask says: query i, at position p = i + keys - queries, sees key j iff p - left <= j <= p + right (-1: no bound); `dropped`
    positions in front of the first key are no longer in the cache."""
    __slots__ = ("queries", "keys", "left", "right", "dropped")

    def __init__(self, queries, keys, left, right, dropped):
        self.queries, self.keys, self.left, self.right, self.dropped = queries, keys, left, right, dropped


_EMPTY_SLOTS = "smbv attention: {} positions hold tokens and there are {} keys: no preallocated cache with empty slots"


def _window_mask(*, batch_size, q_length, kv_length, q_offset=0, kv_offset=0, mask_function, attention_mask=None, device=None, **unused):
    """transformers mask-interface function: the window that `mask_function(batch, head, query, key)` is over these queries and keys, as a _WindowMask.

    The last query's first key and the first query's last key give the two bounds (none where they reach the ends); every query then has to see the first and the
    last key of its window and nothing next to it, which a padded, packed or blocked mask does not pass.  attention_mask: which positions hold tokens - all."""
    n, m, q0, k0 = int(q_length), int(kv_length), int(q_offset), int(kv_offset)
    if attention_mask is not None:
        if attention_mask.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("smbv attention: a padding mask cannot be looked at inside a graph capture; pass none (every position holds a token)")
        if attention_mask.shape[-1] < k0 + m:
            raise ValueError(_EMPTY_SLOTS.format(attention_mask.shape[-1], k0 + m))
        if attention_mask.dim() != 2 or not bool(attention_mask[:, k0:k0 + m].all()):
            raise ValueError("smbv attention: padded batches are not supported (every position of the attention mask has to hold a token); "
                             "ops.window_attention_fwd takes per-sequence lengths")

    def sees(dev, qi, kj):
        b = torch.arange(int(batch_size), device=dev).view(-1, 1, 1)
        qi, kj = qi.to(dev), kj.to(dev)
        r = mask_function(b, torch.zeros((), dtype=torch.long, device=dev), qi + q0, kj + k0)
        return r.broadcast_to(torch.broadcast_shapes(r.shape, b.shape, qi.shape, kj.shape)).cpu()

    def window(dev):
        if n == 0 or m == 0:
            return -1, -1
        i, j = torch.arange(n).view(1, n, 1), torch.arange(m).view(1, 1, m)
        first, last = sees(dev, i[:, :1], j)[0, 0].nonzero(), sees(dev, i[:, -1:], j)[0, 0].nonzero()
        if first.numel() == 0 or last.numel() == 0:
            return None
        lo, hi = int(last[0]), int(first[-1])
        left, right = -1 if lo == 0 else m - 1 - lo, -1 if hi == m - 1 else hi - (m - n)
        if (lo and left < 0) or (hi < m - 1 and right < 0) or last.numel() != int(last[-1]) - lo + 1 or first.numel() != hi - int(first[0]) + 1:
            return None
        p = i + (m - n)
        a = torch.zeros_like(p) if left < 0 else (p - left).clamp(min=0)
        z = torch.full_like(p, m - 1) if right < 0 else (p + right).clamp(max=m - 1)
        inside = sees(dev, i, torch.cat([a, (a + z) // 2, z], 2)).all()
        outside = (sees(dev, i, (a - 1).clamp(min=0)) & (a > 0)).any() | (sees(dev, i, (z + 1).clamp(max=m - 1)) & (z < m - 1)).any()
        return (left, right) if bool(inside) and not bool(outside) else None

    try:   # (in host memory, without waiting for the device - unless the function looks something up there)
        found = window("cpu")
    except RuntimeError:
        if device is None or torch.device(device).type == "cpu":
            raise
        found = window(device)
    if found != (-1, -1) and q0 - k0 != m - n:
        raise ValueError(_EMPTY_SLOTS.format(q0 - k0 + n, m))
    if found is None:
        raise ValueError("smbv attention: the model's mask is no sliding window over full sequences (packed documents, blocks and prefixes are not supported)")
    return _WindowMask(n, m, *found, k0)


def _rows_of_heads(t):
    """t [B, S, H, D] as the kernels can read it: contiguous channels, 16-byte steps."""
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in range(3)):
        return t.contiguous()
    return t


def smbv_window_attention(module, query, key, value, attention_mask=None, *, scaling=None, dropout=0.0, is_causal=None, sliding_window=None, sinks=0, **kwargs):
    """transformers attention-interface function for query [B, H, Sq, D], key / value [B, Hk, Sk, D]; returns (context [B, Sq, H, D] in the dtype of query, None).

    sliding_window: None, or W - keys closer than W positions, in both directions unless the attention is causal -, or (left, right) - as many keys to either
    side, -1 for all.  is_causal: None takes the module's own `is_causal` (False if it has none).  The queries are the last Sq of the Sk positions, all of which
    hold tokens: no preallocated cache with empty slots.  sinks: first keys that stay visible to every later query; the cache has to keep them, so a model's own
    sliding_window, whose cache forgets them, takes sinks only while they are there, and, without a mask to tell, only with as many keys as queries.  fp32
    operands are rounded to bf16.
    attention_mask: None, or what the mask function of register_window() made of the model's mask, which then says what is seen in place of is_causal and of the
    model's own sliding_window.  Other arguments raise, but for None and a few that change nothing."""
    _refuse(kwargs)
    return _window_attention(module, query, key, value, attention_mask, scaling, dropout, is_causal, sliding_window, None, sinks)


def _bounds(window):
    if window is None:
        return -1, -1
    if isinstance(window, int):
        if window < 1:
            raise ValueError(f"smbv window attention: sliding_window {window}")
        return window - 1, window - 1
    left, right = (int(x) for x in window)
    return left, right


def _narrower(a, b):
    return max(a, b) if a < 0 or b < 0 else min(a, b)


def _window_attention(module, query, key, value, mask, scaling, dropout, is_causal, sliding_window, bound, sinks):
    """bound: the window of register_window(), for models that pass no `sliding_window`."""
    if mask is not None and not isinstance(mask, _WindowMask):
        raise ValueError("smbv window attention: masks are not supported (the window, causality and the first tokens are arguments)")
    if dropout:
        raise ValueError("smbv window attention: attention dropout is not supported")
    if query.dim() != 4 or key.dim() != 4 or key.shape != value.shape or key.shape[0] != query.shape[0] or key.shape[3] != query.shape[3] or query.shape[1] % max(key.shape[1], 1):
        raise ValueError(f"smbv window attention: expected query [B, H, Sq, D] and key, value [B, Hk, Sk, D] with H a multiple of Hk, got {tuple(query.shape)}, "
                         f"{tuple(key.shape)}, {tuple(value.shape)}")
    if query.shape[3] % 8 or not 0 < query.shape[3] <= 128:
        raise ValueError(f"smbv window attention: head width {query.shape[3]} (a multiple of 8 up to 128)")
    if not _on_gpu(query):
        raise RuntimeError("smbv window attention needs an MI355X: there is no CPU path")
    left, right = _bounds(bound if sliding_window is None else sliding_window)
    if sinks > 0 and (mask.dropped > 0 if mask is not None else isinstance(sliding_window, int) and key.shape[2] > query.shape[2]):
        raise ValueError("smbv window attention: sinks with a cache that does not keep the first tokens (use a full cache, the window bound by register_window())")
    if mask is None:
        if bool(getattr(module, "is_causal", False) if is_causal is None else is_causal):
            right = 0
    else:
        if (mask.queries, mask.keys) != (query.shape[2], key.shape[2]):
            raise ValueError(f"smbv window attention: a mask for {mask.queries} queries and {mask.keys} keys, got {query.shape[2]} and {key.shape[2]}")
        if sliding_window is not None or bound is None:
            left, right = mask.left, mask.right
        else:
            left, right = _narrower(left, mask.left), _narrower(right, mask.right)
    dtype = query.dtype if query.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
    q, k, v = (_rows_of_heads(t.transpose(1, 2).to(dtype)) for t in (query, key, value))
    kw = dict(left=left, right=right, sinks=int(sinks), scale=None if scaling is None else float(scaling))
    # (through the autograd function also without gradients: forward-mode tangents, which it has no rule for, then raise instead of being dropped)
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _SmbvWindowAttentionFn.apply(q, k, v, kw, train).to(query.dtype), None


def register_window(name=WINDOW_NAME, *, window=None, sinks=0):
    """Make `config._attn_implementation = name` select the windowed kernels.  window: what takes the place of `sliding_window` in models that pass none (the
    reference's encoders among them); sinks: first tokens that stay visible, with a cache that keeps them (the sliding cache of a model with a window of its own
    does not: generation past it raises)."""
    from transformers import AttentionInterface, AttentionMaskInterface

    @functools.wraps(smbv_window_attention)
    def attend(module, query, key, value, attention_mask=None, *, scaling=None, dropout=0.0, is_causal=None, sliding_window=None, **kwargs):
        _refuse(kwargs)
        return _window_attention(module, query, key, value, attention_mask, scaling, dropout, is_causal, sliding_window, window, sinks)

    AttentionInterface.register(name, attend)
    AttentionMaskInterface.register(name, _window_mask)
    return name
