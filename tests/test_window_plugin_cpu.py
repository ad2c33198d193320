"""Models by name (smb_vision_amd/attention_plugin.py register_window) without a GPU: the windowed attention is replaced by its definition, so what is tested is
what the registered functions make of a model's masks, arguments and caches - against the same model's eager attention, or its refusal."""
import pytest
import torch

from smb_vision_amd import attention_plugin, ops


def definition(q, k, v, *, left=-1, right=-1, sinks=0, scale=None, resid=False):
    G, n, m = q.shape[2] // k.shape[2], q.shape[1], k.shape[1]
    d = torch.arange(m)[None] - (torch.arange(n)[:, None] + m - n)
    seen = torch.ones(n, m, dtype=torch.bool)
    if right >= 0:
        seen &= d <= right
    if left >= 0:
        seen &= (d >= -left) | (torch.arange(m)[None] < sinks)
    s = torch.einsum("bihd,bjhd->bhij", q.float(), k.float().repeat_interleave(G, 2)) * (q.shape[3] ** -0.5 if scale is None else scale)
    return torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~seen, -torch.inf), -1), v.float().repeat_interleave(G, 2)), None


@pytest.fixture()
def calls(monkeypatch):
    made = []

    def fwd(q, k, v, **kw):
        made.append((q.shape[1], k.shape[1], kw["left"], kw["right"], kw["sinks"]))
        return definition(q, k, v, **kw)

    monkeypatch.setattr(attention_plugin, "_on_gpu", lambda t: True)
    monkeypatch.setattr(ops, "window_attention_fwd", fwd)
    return made


def rms_err(a, b):
    return float((a - b).pow(2).mean().sqrt() / b.pow(2).mean().sqrt())


def lm(kind, name, **kw):
    import transformers as t
    torch.manual_seed(0)
    base = dict(vocab_size=50, hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, attn_implementation=name)
    if kind == "gpt2":
        return t.GPT2LMHeadModel(t.GPT2Config(vocab_size=50, n_embd=64, n_layer=2, n_head=2, attn_implementation=name)).eval()
    if kind == "bert":
        base.pop("num_key_value_heads")
        return t.BertModel(t.BertConfig(**base)).eval()
    config, model = {"mistral": (t.MistralConfig, t.MistralForCausalLM), "llama": (t.LlamaConfig, t.LlamaForCausalLM), "gemma2": (t.Gemma2Config, t.Gemma2ForCausalLM),
                     "gemma3": (t.Gemma3TextConfig, t.Gemma3ForCausalLM), "gpt_oss": (t.GptOssConfig, t.GptOssForCausalLM)}[kind]
    if kind != "llama":
        kw = dict(sliding_window=8, **kw)
    if kind in ("gemma2", "gemma3", "gpt_oss"):
        kw = dict(head_dim=16, **kw)
    if kind == "gpt_oss":
        kw = dict(num_local_experts=2, num_experts_per_tok=1, **kw)
    return model(config(**base, **kw)).eval()


def both(kind, **register):
    name = attention_plugin.register_window("smbv_window_for_test", **register)
    ref, ours = lm(kind, "eager"), lm(kind, name)
    ours.load_state_dict(ref.state_dict())
    return ref, ours


IDS = torch.randint(1, 50, (2, 20), generator=torch.Generator().manual_seed(0))
ONES = torch.ones(2, 20, dtype=torch.long)


def out(m, *a, **kw):
    with torch.no_grad():
        r = m(*a, **kw)
    return r.logits if "logits" in r else r.last_hidden_state


# (operands are rounded to bf16: 2^-9 a value and a layer; a wrong mask is off by tenths)
@pytest.mark.parametrize("kind,bounds", [("mistral", {(7, 0)}), ("llama", {(-1, 0)}), ("gemma3", {(7, 0)}), ("gpt2", {(-1, 0)}), ("bert", {(-1, -1)})])
def test_models_see_what_their_masks_say(calls, kind, bounds):
    ref, ours = both(kind)
    for kw in ({}, dict(attention_mask=ONES)):
        calls.clear()
        assert rms_err(out(ours, IDS, **kw), out(ref, IDS, **kw)) < 2e-2
        assert {c[:4] for c in calls} == {(20, 20, *b) for b in bounds}


@pytest.mark.parametrize("kind", ["mistral", "llama"])
def test_token_by_token_and_in_pieces(calls, kind):
    ref, ours = both(kind)
    want = out(ref, IDS)
    for steps in ((1,) * 20, (12, 1, 1, 1, 1, 1, 3), (3, 9, 8)):
        cache, got, at = None, [], 0
        for n in steps:
            with torch.no_grad():
                o = ours(IDS[:, at:at + n], past_key_values=cache, use_cache=True)
            cache, at = o.past_key_values, at + n
            got.append(o.logits)
        assert rms_err(torch.cat(got, 1), want) < 2e-2


@pytest.mark.parametrize("kind", ["mistral", "llama", "gpt2", "bert"])
@pytest.mark.parametrize("pad", [slice(0, 3), slice(17, 20), slice(8, 9)])
def test_padded_batches_are_refused(calls, kind, pad):
    _, ours = both(kind)
    mask = ONES.clone()
    mask[1, pad] = 0
    with pytest.raises(ValueError, match="padded"):
        out(ours, IDS, attention_mask=mask)
    assert not calls


def test_other_masks_are_refused(calls):
    _, ours = both("llama")
    for mask in (torch.zeros(2, 1, 20, 20), torch.ones(2, 1, 20, 20, dtype=torch.bool)):   # one that the caller made
        with pytest.raises(ValueError, match="masks are not supported"):
            out(ours, IDS, attention_mask=mask)
    with pytest.raises(ValueError, match="empty slots"):
        ours.generate(IDS[:1, :5], max_new_tokens=4, do_sample=False, pad_token_id=0, cache_implementation="static")
    assert not calls


def fn(name, B=1, seed=0):
    doc = torch.tensor([0] * 6 + [1] * 14)
    return {"causal": lambda b, h, q, k: k <= q, "full": lambda b, h, q, k: q >= 0, "sliding": lambda b, h, q, k: (k <= q) & (k > q - 5),
            "both sides": lambda b, h, q, k: (k - q).abs() <= 3, "uneven": lambda b, h, q, k: (k <= q + 2) & (k >= q - 6),
            "packed": lambda b, h, q, k: (k <= q) & (doc[q] == doc[k]), "chunked": lambda b, h, q, k: (k <= q) & (k // 8 == q // 8),
            "prefix": lambda b, h, q, k: (k <= q) | (k < 4), "block": lambda b, h, q, k: (k <= q) | ((q >= 5) & (q < 9) & (k >= 5) & (k < 9)),
            "nothing": lambda b, h, q, k: (k < q) & (q < 0), "hole": lambda b, h, q, k: (k <= q) & (k != 9), "second": lambda b, h, q, k: (k <= q) & ((b == 0) | (k > 2)),
            "ahead only": lambda b, h, q, k: k > q}[name]


@pytest.mark.parametrize("name,want", [("causal", (-1, 0)), ("full", (-1, -1)), ("sliding", (4, 0)), ("both sides", (3, 3)), ("uneven", (6, 2)), ("packed", None), ("chunked", None),
                                       ("prefix", None), ("block", None), ("nothing", None), ("hole", None), ("second", None), ("ahead only", None)])
def test_mask_functions(name, want):
    make = lambda **kw: attention_plugin._window_mask(**{**dict(batch_size=2, q_length=20, kv_length=20, mask_function=fn(name), dtype=torch.float32, config=None), **kw})
    if want is None:
        with pytest.raises(ValueError):
            make()
        return
    m = make()
    assert (m.left, m.right, m.queries, m.keys) == (*want, 20, 20)
    m = make(q_length=1, q_offset=19)   # the newest token against all of them
    assert m.left == (-1 if want[0] < 0 else want[0]) and m.right == -1
    m = make(q_length=4, kv_length=12, q_offset=16, kv_offset=8)   # against a cache that holds the last 12
    assert (m.left, m.right) == (want[0], -1 if want[1] >= 3 else want[1])   # (the first of them, at 8, reaches the last key, 11, with 3)


@pytest.mark.parametrize("bound,want", [(5, (4, 0)), ((30, 30), (30, 0)), ((2, -1), (2, 0)), (None, (-1, 0))])
def test_bound_window_narrows_a_mask(calls, bound, want):
    _, ours = both("llama", window=bound)
    out(ours, IDS)
    assert {c[2:4] for c in calls} == {want}
    _, ours = both("mistral", window=bound)   # (its own window stands)
    calls.clear()
    out(ours, IDS)
    assert {c[2:4] for c in calls} == {(7, 0)}


@pytest.mark.parametrize("kind,argument", [("gemma2", "softcap"), ("gpt_oss", "s_aux")])
def test_models_with_another_softmax_are_refused(calls, kind, argument):
    _, ours = both(kind)
    with pytest.raises(ValueError, match=argument):
        out(ours, IDS)
    assert not calls


@pytest.mark.parametrize("extra", [dict(softcap=50.0), dict(s_aux=torch.zeros(2)), dict(position_bias=torch.zeros(1)), dict(head_mask=torch.ones(2)),
                                   dict(cu_seq_lens_q=torch.tensor([0, 4])), dict(never_heard_of=0)], ids=lambda d: next(iter(d)))
def test_unknown_arguments_are_refused(calls, extra):
    q, m = torch.zeros(1, 2, 8, 64), torch.nn.Module()
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    named = ALL_ATTENTION_FUNCTIONS[attention_plugin.register_window("smbv_window_for_test")]
    for f in (attention_plugin.smbv_window_attention, named):
        with pytest.raises(ValueError, match=next(iter(extra))):
            f(m, q, q, q, **extra)
        f(m, q, q, q, **{n: None for n in extra}, position_ids=torch.arange(8)[None], use_cache=True)


def test_sinks_need_a_cache_that_keeps_them(calls):
    """A full cache with the window bound at registration gives token by token what a prompt gives; a sliding cache, which forgets the first tokens, raises."""
    _, full = both("llama", window=(7, -1), sinks=4)
    want, cache, got = out(full, IDS), None, []
    for n, at in ((12, 0), *((1, i) for i in range(12, 20))):
        with torch.no_grad():
            o = full(IDS[:, at:at + n], past_key_values=cache, use_cache=True)
        cache = o.past_key_values
        got.append(o.logits)
    assert rms_err(torch.cat(got, 1), want) < 2e-2 and {c[4] for c in calls} == {4}
    _, sliding = both("mistral", sinks=4)   # (its window is 8: the cache keeps 7)
    with torch.no_grad():
        short = sliding(IDS[:, :6], use_cache=True).past_key_values
        sliding(IDS[:, 6:7], past_key_values=short, use_cache=True)   # the first tokens are still there
        long = sliding(IDS[:, :12], use_cache=True).past_key_values
        with pytest.raises(ValueError, match="first tokens"):
            sliding(IDS[:, 12:13], past_key_values=long, use_cache=True)
    q, k, m = torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 8, 64), torch.nn.Module()
    with pytest.raises(ValueError, match="first tokens"):
        attention_plugin.smbv_window_attention(m, q, k, k, sliding_window=8, sinks=4)
    attention_plugin.smbv_window_attention(m, q, k, k, sliding_window=(7, 0), sinks=4)
    attention_plugin.smbv_window_attention(m, k, k, k, sliding_window=8, sinks=4)
    attention_plugin.smbv_window_attention(m, q, k, k, sliding_window=8)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_tangents_are_not_dropped(calls, grad):
    import torch.autograd.forward_ad as fwd
    x, m = torch.randn(1, 2, 8, 64), torch.nn.Module()
    for n in range(3):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            t = [x, x, x]
            t[n] = fwd.make_dual(x, torch.randn_like(x))
            with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                attention_plugin.smbv_window_attention(m, *t)
    o = attention_plugin.smbv_window_attention(m, x, x, x)[0]
    assert not o.requires_grad and o.grad_fn is None
    with torch.no_grad():
        assert torch.equal(attention_plugin.smbv_window_attention(m, x.clone().requires_grad_(True), x, x)[0], o)


def test_full_attention_by_name_refuses_other_masks(monkeypatch):
    """The name "smbv" computes attention of everything to everything: a model that asks for less raises, and one that does not gets what eager gives."""
    monkeypatch.setattr(attention_plugin, "_on_gpu", lambda t: True)
    monkeypatch.setattr(attention_plugin._SmbvAttentionFn, "apply", lambda q, k, v, scale: definition(*(t.transpose(1, 2) for t in (q, k, v)), scale=scale)[0])
    name = attention_plugin.register("smbv_for_test")
    import transformers as t
    base = dict(vocab_size=50, hidden_size=128, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, attn_implementation=name)
    bert = t.BertModel(t.BertConfig(**base)).eval()
    ref = t.BertModel(t.BertConfig(**{**base, "attn_implementation": "eager"})).eval()
    ref.load_state_dict(bert.state_dict())
    for mask in (None, ONES):
        assert rms_err(out(bert, IDS, attention_mask=mask), out(ref, IDS, attention_mask=mask)) < 1e-5
    mask = ONES.clone()
    mask[1, :3] = 0
    with pytest.raises(ValueError, match="padded"):
        out(bert, IDS, attention_mask=mask)
    llama = t.LlamaForCausalLM(t.LlamaConfig(**base)).eval()
    with pytest.raises(ValueError, match="causal"):
        out(llama, IDS)
    q = torch.zeros(1, 2, 8, 64)
    with pytest.raises(ValueError, match="softcap"):
        attention_plugin.smbv_attention(torch.nn.Module(), q, q, q, softcap=50.0)
