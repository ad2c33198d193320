"""Windowed attention behind transformers' attention registry (smb_vision_amd/attention_plugin.py register_window), and the block operators run together.

The registered function is the operator of tests/test_window_attention_gpu.py under another interface: its outputs and gradients have to be that operator's, bit
for bit.  The unmodified VideoMAE class by name is compared with its eager attention as tests/test_attention_plugin_gpu.py does, with that file's tolerances."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def rms_err(a, b):
    return float((a.detach().double() - b.detach().double()).pow(2).mean().sqrt() / (b.detach().double().pow(2).mean().sqrt() + 1e-30))


@pytest.mark.parametrize("dtype,H,Hk,Sq,Sk,D,causal,window,left,right", [
    (BF, 4, 2, 70, 70, 64, True, 20, 19, 0), (HF, 3, 3, 45, 45, 80, False, 9, 8, 8), (BF, 8, 1, 1, 130, 128, True, None, -1, 0), (torch.float32, 2, 2, 33, 50, 32, True, (7, 3), 7, 0),
    (BF, 2, 2, 40, 40, 64, False, (5, -1), 5, -1)])
def test_registered_function_is_the_operator(dtype, H, Hk, Sq, Sk, D, causal, window, left, right):
    from smb_vision_amd import ops
    from smb_vision_amd.attention_plugin import smbv_window_attention
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, h, s, D, generator=g).cuda().to(dtype).requires_grad_(True) for h, s in ((H, Sq), (Hk, Sk), (Hk, Sk)))
    module = torch.nn.Module()
    module.is_causal = causal
    out, probs = smbv_window_attention(module, q, k, v, None, scaling=0.2, sliding_window=window, sinks=3)
    assert probs is None and out.shape == (2, Sq, H, D) and out.dtype == dtype
    t = BF if dtype == torch.float32 else dtype
    rows = [x.detach().transpose(1, 2).to(t) for x in (q, k, v)]
    kw = dict(left=left, right=right, sinks=3, scale=0.2)
    o, lse, lo = ops.window_attention_fwd(*rows, resid=True, **kw)
    assert torch.equal(out.detach(), o.to(dtype))
    do = torch.randn(2, Sq, H, D, generator=g).cuda().to(dtype)
    out.backward(do)
    for a, b in zip((q, k, v), ops.window_attention_bwd(*rows, o, do.to(t), lse, o_lo=lo, **kw)):
        assert a.grad.dtype == dtype and torch.equal(a.grad, b.transpose(1, 2).to(dtype))
    with torch.no_grad():
        assert torch.equal(smbv_window_attention(module, q, k, v, None, scaling=0.2, sliding_window=window, sinks=3)[0], o.to(dtype))


def test_reference_class_by_name():
    """The unmodified VideoMAE class: without a window it is full attention and has to match eager; with one it has to match eager under the window's mask."""
    from transformers import VideoMAEConfig, VideoMAEForPreTraining
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    from smb_vision_amd import attention_plugin
    kw = dict(image_size=64, patch_size=16, num_channels=1, num_frames=64, tubelet_size=16, hidden_size=192, num_hidden_layers=2, num_attention_heads=3, intermediate_size=384,
              decoder_num_attention_heads=3, decoder_hidden_size=96, decoder_num_hidden_layers=1, decoder_intermediate_size=192, norm_pix_loss=True)

    def masked_eager(module, query, key, value, attention_mask=None, *, scaling=None, **unused):
        n = query.shape[2]
        d = torch.arange(n, device=query.device)[None] - torch.arange(n, device=query.device)[:, None]
        seen = ((d >= -6) | (torch.arange(n, device=query.device)[None] < 2)) & (d <= 6)
        s = (query.float() @ key.float().transpose(2, 3)) * scaling
        return (torch.softmax(s.masked_fill(~seen, -torch.inf), -1) @ value.float()).transpose(1, 2).contiguous().to(query.dtype), None

    ALL_ATTENTION_FUNCTIONS.register("masked_eager_for_test", masked_eager)
    full = attention_plugin.register_window("smbv_window_full")
    windowed = attention_plugin.register_window("smbv_window_6", window=(6, 6), sinks=2)
    g = torch.Generator().manual_seed(1)
    x = torch.rand(2, 64, 1, 64, 64, generator=g).cuda()
    mask = torch.zeros(2, 64, dtype=torch.bool)
    for b in range(2):
        mask[b, torch.randperm(64, generator=g)[:40]] = True
    for ours_name, ref_name in ((full, "eager"), (windowed, "masked_eager_for_test")):
        torch.manual_seed(0)
        ref = VideoMAEForPreTraining(VideoMAEConfig(**kw, attn_implementation=ref_name)).cuda().train()
        ours = VideoMAEForPreTraining(VideoMAEConfig(**kw, attn_implementation=ours_name)).cuda().train()
        ours.load_state_dict(ref.state_dict())
        outs = []
        for m in (ref, ours):
            with torch.autocast("cuda", dtype=BF):
                o = m(pixel_values=x, bool_masked_pos=mask.cuda())
            o.loss.backward()
            outs.append(o)
        assert abs(float(outs[0].loss) - float(outs[1].loss)) < 5e-3 * abs(float(outs[0].loss))
        assert rms_err(outs[1].logits, outs[0].logits) < 2e-2
        pr, po = dict(ref.named_parameters()), dict(ours.named_parameters())
        worst = max((rms_err(po[n].grad, pr[n].grad), n) for n in pr if pr[n].grad is not None and not n.endswith("key.bias"))
        assert worst[0] < 3e-2, (ours_name, worst)


def test_plugin_refusals():
    from smb_vision_amd.attention_plugin import smbv_window_attention
    q = torch.zeros(1, 2, 16, 64, device="cuda", dtype=BF)
    m = torch.nn.Module()
    for args, kw in (((q, q, q, torch.zeros(1, 1, 16, 16, device="cuda")), {}), ((q, q, q), dict(dropout=0.1)), ((q, q[:, :, :8], q), {}), ((q[..., :60], q[..., :60], q[..., :60]), {}),
                     ((q, q, q), dict(sliding_window=0)), ((q[:, :1], q, q), {}), ((q, q, q), dict(scaling=-1.0)), ((q, q, q), dict(sinks=-1))):
        with pytest.raises((ValueError, RuntimeError)):
            smbv_window_attention(m, *args, **kw)


def test_training_is_not_captured():
    from smb_vision_amd.attention_plugin import smbv_window_attention
    q = torch.randn(1, 2, 16, 64, device="cuda").to(BF).requires_grad_(True)
    m = torch.nn.Module()
    smbv_window_attention(m, q, q, q)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        with torch.no_grad():
            out = smbv_window_attention(m, q, q, q)[0]
        with pytest.raises(RuntimeError):
            smbv_window_attention(m, q, q, q)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, smbv_window_attention(m, q, q, q)[0].detach())


def test_a_block_of_them():
    """norm - projection - rotary positions - windowed attention - projection - norm, gate and residual - and back, as one block of a model runs them, with the
    framework's matrix products between them, against the same block in 64 bits.

    Tolerance: every tensor that passes between the operators is rounded to bf16 once (2^-8 at worst, 2^-9 / sqrt(3) = 1.1e-3 rms), about a dozen of them in a row
    forward and as many again backward; independent roundings add up to 1.1e-3 * sqrt(24) = 5.5e-3 rms of a tensor whose parts do not cancel.  Twice that."""
    from smb_vision_amd import ops
    B, S, H, Hk, D, d = 2, 150, 4, 2, 32, 128
    g = torch.Generator().manual_seed(3)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).cuda()
    x, h0 = r(B, S, d), r(B, S, d).to(BF)
    wq, wo = r((H + 2 * Hk) * D, d, scale=d ** -0.5).to(BF), r(d, H * D, scale=(H * D) ** -0.5).to(BF)
    w1, w2, w3, w4 = (1 + r(d, scale=0.1) for _ in range(4))
    g1, g2 = r(B, d, scale=0.5), r(B, d, scale=0.5)
    pos = torch.stack([torch.arange(S) // 25, (torch.arange(S) // 5) % 5, torch.arange(S) % 5])[:, None].repeat(1, B, 1).int().cuda()
    inv, sec = (100.0 ** (-torch.arange(16) / 16)).float().cuda(), (6, 5, 5)
    win = dict(left=40, right=0, sinks=3)
    heads = lambda t: (t[..., :H * D].unflatten(-1, (H, D)), t[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)), t[..., (H + Hk) * D:].unflatten(-1, (Hk, D)))
    dx, dy = r(B, S, d), r(B, S, d).to(BF)

    k1, k2 = dict(post_w=w1, gate=g1, pre_w=w2), dict(post_w=w3, gate=g2, pre_w=w4, res_scale=0.9)
    x1, y1, st1 = ops.gated_norm_fwd(h0, x, **k1)
    qkv = ops.gemm_nt(y1.view(-1, d), wq)["bf16"].view(B, S, -1)
    q, k, v = heads(qkv)
    ops.rope_axes(q, k, pos, inv, sec, out=(q, k))
    o, lse, lo = ops.window_attention_fwd(q, k, v, resid=True, **win)
    h1 = ops.gemm_nt(o.view(-1, H * D), wo)["bf16"].view(B, S, d)
    x2, y2, st2 = ops.gated_norm_fwd(h1, x1, **k2)
    b2 = ops.gated_norm_bwd(dx, dy, h1, x1, st2, **k2)
    do = ops.gemm_nt(b2["dh"].view(-1, d), wo.T.contiguous())["bf16"].view(B, S, H, D)
    dwo = ops.gemm_tn(b2["dh"].view(-1, d), o.view(-1, H * D))
    dqkv = torch.empty_like(qkv)
    dq, dk, dv = ops.window_attention_bwd(q, k, v, o, do, lse, o_lo=lo, out=heads(dqkv), **win)
    ops.rope_axes(dq, dk, pos, inv, sec, transpose=True, out=(dq, dk))
    dy1 = ops.gemm_nt(dqkv.view(B * S, -1), wq.T.contiguous())["bf16"].view(B, S, d)
    dwq = ops.gemm_tn(dqkv.view(B * S, -1), y1.view(-1, d))
    b1 = ops.gated_norm_bwd(b2["dx"], dy1, h0, x, st1, **k1)

    leaf = [t.double().requires_grad_(True) for t in (x, h0, wq, wo, w1, w2, w3, w4, g1, g2)]
    X, H0, WQ, WO, W1, W2, W3, W4, G1, G2 = leaf
    rms = lambda t, w: t * (t.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w
    X1 = X + G1[:, None] * rms(H0, W1)
    Q, K, V = heads(rms(X1, W2) @ WQ.T)
    ang = torch.cat([pos[a].double()[..., None] * inv[s:e].double() for a, (s, e) in enumerate(((0, 6), (6, 11), (11, 16)))], -1)[:, :, None]
    turn = lambda t: torch.cat([t[..., :16] * ang.cos() - t[..., 16:] * ang.sin(), t[..., :16] * ang.sin() + t[..., 16:] * ang.cos()], -1)
    Q, K = turn(Q), turn(K)
    i = torch.arange(S, device="cuda")
    seen = (i[None] <= i[:, None]) & ((i[None] >= i[:, None] - 40) | (i[None] < 3))
    P = torch.softmax((torch.einsum("bihd,bjhd->bhij", Q, K.repeat_interleave(2, 2)) * D ** -0.5).masked_fill(~seen, -torch.inf), -1)
    O = torch.einsum("bhij,bjhd->bihd", P, V.repeat_interleave(2, 2)).flatten(2)
    X2 = 0.9 * X1 + G2[:, None] * rms(O @ WO.T, W3)
    Y2 = rms(X2, W4)
    grads = torch.autograd.grad((X2 * dx.double()).sum() + (Y2 * dy.double()).sum(), leaf)
    got = (x2, y2, b1["dx"], b1["dh"], dwq, dwo, b1["post_w"], b1["pre_w"], b2["post_w"], b2["pre_w"], b1["gate"], b2["gate"])
    for n, a, b in zip(("x2", "y2", "dx", "dh", "dwq", "dwo", "dw1", "dw2", "dw3", "dw4", "dg1", "dg2"), got, (X2, Y2, *grads)):
        assert rms_err(a, b) < 1.1e-2, (n, rms_err(a, b))


@pytest.mark.parametrize("kind", ["mistral", "llama"])
def test_causal_models_by_name(kind):
    """Mistral (a sliding window and a sliding cache) and Llama by name: a prompt, its gradients, and token by token, against their eager attention in fp32.
    Tolerances as above for a whole model under bf16 operands: 2e-2 of the logits, 3e-2 of the gradients (rms)."""
    import transformers as t
    from smb_vision_amd import attention_plugin
    name = attention_plugin.register_window()
    base = dict(vocab_size=64, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2)
    make = {"mistral": lambda a: t.MistralForCausalLM(t.MistralConfig(**base, sliding_window=24, attn_implementation=a)),
            "llama": lambda a: t.LlamaForCausalLM(t.LlamaConfig(**base, attn_implementation=a))}[kind]
    torch.manual_seed(0)
    ref, ours = make("eager").cuda().train(), make(name).cuda().train()
    ours.load_state_dict(ref.state_dict())
    ids = torch.randint(0, 64, (2, 70), generator=torch.Generator().manual_seed(2)).cuda()
    outs = [m(ids, attention_mask=torch.ones_like(ids), labels=ids) for m in (ref, ours)]
    for o in outs:
        o.loss.backward()
    assert rms_err(outs[1].logits, outs[0].logits) < 2e-2
    pr, po = dict(ref.named_parameters()), dict(ours.named_parameters())
    worst = max((rms_err(po[n].grad, pr[n].grad), n) for n in pr)
    assert worst[0] < 3e-2, worst
    ours.eval()
    cache, got = None, []
    with torch.no_grad():
        for n, at in ((40, 0), *((1, i) for i in range(40, 70))):
            o = ours(ids[:, at:at + n], past_key_values=cache, use_cache=True)
            cache = o.past_key_values
            got.append(o.logits)
    assert rms_err(torch.cat(got, 1), outs[0].logits) < 2e-2
    mask = torch.ones_like(ids)
    mask[1, :5] = 0
    with pytest.raises(ValueError):
        ours(ids, attention_mask=mask)


def test_mask_that_looks_something_up_on_the_device():
    """Packed documents are a table on the model's device: looked up there, and refused."""
    from smb_vision_amd import attention_plugin
    doc = torch.tensor([0] * 6 + [1] * 14, device="cuda")
    kw = dict(batch_size=2, q_length=20, kv_length=20, dtype=BF, config=None, device=torch.device("cuda"))
    with pytest.raises(ValueError):
        attention_plugin._window_mask(mask_function=lambda b, h, q, k: (k <= q) & (doc[q] == doc[k]), **kw)
    one = torch.zeros(20, dtype=torch.long, device="cuda")
    m = attention_plugin._window_mask(mask_function=lambda b, h, q, k: (k <= q) & (one[q] == one[k]), **kw)
    assert (m.left, m.right) == (-1, 0)
