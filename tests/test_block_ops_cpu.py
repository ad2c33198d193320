"""What the operators of a transformer block refuse - through the C ABI (with made-up addresses: a refused call touches none) and through ops - without a GPU."""
import ctypes as C

import pytest
import torch

from smb_vision_amd import _lib, ops

P = 1 << 20  # a made-up, aligned address
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def attn(**kw):
    a = _lib.WindowAttn()
    a.dtype, a.B, a.Sq, a.Sk, a.H, a.Hk, a.Dh, a.left, a.right, a.sinks, a.scale = 0, 2, 16, 16, 4, 2, 64, 4, 0, 1, 0.125
    for n in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv"):
        setattr(a, n, P)
    for n in ("sq", "so", "sdo", "sdq"):
        setattr(a, n, _lib.c_ll3(16 * 4 * 64, 4 * 64, 64))
    for n in ("sk", "sv", "sdk", "sdv"):
        setattr(a, n, _lib.c_ll3(16 * 2 * 64, 2 * 64, 64))
    for n, v in kw.items():
        setattr(a, n, v)
    return a


ATTN = [dict(struct_bytes=8), dict(dtype=2), dict(dtype=-1), dict(B=-1), dict(Sq=-1), dict(Sk=-2), dict(H=3), dict(Hk=0), dict(H=0), dict(Dh=0), dict(Dh=60), dict(Dh=136),
        dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(sinks=-1), dict(q=0), dict(k=0), dict(v=0), dict(o=0), dict(lse=0),
        dict(q=P + 2), dict(k=P + 8), dict(o=P + 4), dict(o_lo=P + 2), dict(sq=_lib.c_ll3(4100, 260, 65)), dict(sk=_lib.c_ll3(-2048, 128, 64)), dict(Sk=1 << 30),
        dict(Sq=1 << 28, H=64, Hk=1), dict(B=1 << 30)]


@pytest.mark.parametrize("bad", ATTN, ids=str)
def test_window_attention_refusals(bad):
    lib = _lib.load()
    for fn in ("smbv_window_attention_fwd", "smbv_window_attention_bwd"):
        assert getattr(lib, fn)(C.byref(attn(**bad)), P, 1 << 40, None) < 0
        assert fn[5:] in _lib.last_error()


@pytest.mark.parametrize("bad", [dict(d_o=0), dict(dq=0), dict(dk=0), dict(dv=0), dict(dq=P + 2), dict(sdk=_lib.c_ll3(2048, 128, 4))], ids=str)
def test_window_attention_backward_refusals(bad):
    assert _lib.load().smbv_window_attention_bwd(C.byref(attn(**bad)), P, 1 << 40, None) < 0


@pytest.mark.parametrize("many", [dict(B=1 << 23, Hk=2), dict(Sk=1 << 28, B=8), dict(B=1 << 12, H=1024, Hk=1, Sq=64)], ids=str)
def test_window_attention_more_rows_than_a_launch_takes(many):
    lib = _lib.load()
    for fn in ("smbv_window_attention_fwd", "smbv_window_attention_bwd"):
        assert getattr(lib, fn + "_workspace_bytes")(C.byref(attn(**many))) == 0
        assert getattr(lib, fn)(C.byref(attn(**many)), P, 1 << 60, None) < 0 and "many" in _lib.last_error()
    assert lib.smbv_rope_axes(C.byref(rope(B=1 << 10, S=(1 << 21) - 1, Dh=1024, section=sec(512, 0, 0, 0))), None) < 0 and "many" in _lib.last_error()


def test_workspaces():
    lib = _lib.load()
    a = attn()
    need = lib.smbv_window_attention_bwd_workspace_bytes(C.byref(a))
    assert need > 0 and lib.smbv_window_attention_fwd_workspace_bytes(C.byref(a)) >= 0
    for ws, n in ((P, need - 1), (P + 16, need), (0, need)):
        assert lib.smbv_window_attention_bwd(C.byref(a), ws, n, None) == -4
    g = norm()
    need = lib.smbv_gated_norm_bwd_workspace_bytes(C.byref(g))
    assert need > 0
    for ws, n in ((P, need - 1), (P + 16, need), (0, need)):
        assert lib.smbv_gated_norm_bwd(C.byref(g), ws, n, None) == -4
    assert lib.smbv_window_attention_fwd_workspace_bytes(None) == 0 and lib.smbv_window_attention_bwd_workspace_bytes(None) == 0
    assert lib.smbv_gated_norm_bwd_workspace_bytes(None) == 0


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.smbv_window_attention_fwd(C.byref(attn(B=0)), None, 0, None) == 0
    assert lib.smbv_window_attention_bwd(C.byref(attn(B=0)), None, 0, None) == 0
    assert lib.smbv_rope_axes(C.byref(rope(S=0)), None) == 0
    assert lib.smbv_gated_norm_fwd(C.byref(norm(rows=0)), None) == 0 and lib.smbv_gated_norm_bwd(C.byref(norm(rows=0)), None, 0, None) == 0


def rope(**kw):
    a = _lib.RopeAxesCfg()
    a.dtype, a.B, a.S, a.H, a.Hk, a.Dh, a.axes = 0, 2, 8, 4, 2, 64, 3
    a.section = (C.c_int * 4)(12, 10, 10, 0)
    a.q, a.k, a.qo, a.ko, a.pos, a.inv_freq = P, 2 * P, 3 * P, 4 * P, 5 * P, 6 * P
    a.sq = a.sqo = _lib.c_ll3(8 * 256, 256, 64)
    a.sk = a.sko = _lib.c_ll3(8 * 128, 128, 64)
    a.spos = _lib.c_ll3(16, 8, 1)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def sec(*n):
    return (C.c_int * 4)(*n)


@pytest.mark.parametrize("bad", [dict(struct_bytes=0), dict(dtype=3), dict(axes=0), dict(axes=5), dict(section=sec(12, -1, 10, 0)), dict(section=sec(0, 0, 0, 0)),
                                 dict(section=sec(20, 10, 10, 0)), dict(section=sec(2 ** 31 - 1, 2 ** 31 - 1, 5, 0)), dict(Dh=65), dict(Dh=1026), dict(B=-1), dict(S=-1),
                                 dict(H=-1), dict(q=0), dict(ko=0), dict(pos=0), dict(inv_freq=0), dict(q=P + 1), dict(B=1 << 16, S=1 << 16)], ids=str)
def test_rope_axes_refusals(bad):
    assert _lib.load().smbv_rope_axes(C.byref(rope(**bad)), None) < 0
    assert "rope_axes" in _lib.last_error()


def norm(**kw):
    a = _lib.GatedNorm()
    a.h_type, a.x_type, a.d, a.post, a.pre, a.eps, a.res_scale, a.rows, a.rows_per_gate = 0, 2, 64, 1, 2, 1e-6, 1.0, 12, 4
    for i, n in enumerate(("h", "x", "post_w", "post_b", "gate", "pre_w", "pre_b", "x1", "y", "stats", "dx1", "dy", "dh", "dx", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")):
        setattr(a, n, P * (i + 1))
    for n in ("ldh", "ldx", "ldx1", "ldy", "lddx1", "lddy", "lddh", "lddx"):
        setattr(a, n, 64)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


NORM = [dict(struct_bytes=1), dict(h_type=3), dict(x_type=1), dict(h_type=2, x_type=0), dict(d=0), dict(d=8193), dict(rows=-1), dict(rows=1 << 31), dict(post=3), dict(pre=-1),
        dict(post=0), dict(pre=0), dict(rows_per_gate=5), dict(rows_per_gate=0), dict(eps=-1.0), dict(eps=float("nan")), dict(h=0), dict(x=0), dict(stats=0), dict(ldh=63),
        dict(h=P + 1), dict(x=P + 2), dict(gate=P + 2), dict(stats=P + 4)]


@pytest.mark.parametrize("bad", NORM, ids=str)
def test_gated_norm_refusals(bad):
    lib = _lib.load()
    assert lib.smbv_gated_norm_fwd(C.byref(norm(**bad)), None) < 0 and "gated_norm_fwd" in _lib.last_error()
    assert lib.smbv_gated_norm_bwd(C.byref(norm(**bad)), P, 1 << 40, None) < 0 and "gated_norm_bwd" in _lib.last_error()


@pytest.mark.parametrize("bad", [dict(dy=0), dict(dh=0), dict(dx=0), dict(dgate=0), dict(post_w=0), dict(pre_b=0), dict(pre=0, pre_w=0, pre_b=0, dpre_w=0, dpre_b=0, dx1=0)], ids=str)
def test_gated_norm_backward_refusals(bad):
    assert _lib.load().smbv_gated_norm_bwd(C.byref(norm(**bad)), P, 1 << 40, None) < 0


# ---- through ops: the checks come before the library is reached -------------------------------------------------------------------------------------
class Unreachable:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def dry(monkeypatch):
    monkeypatch.setattr(ops, "_need_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "load", lambda: Unreachable())


def test_operators_need_a_gpu():
    q = torch.zeros(1, 4, 2, 64, dtype=BF)
    with pytest.raises(_lib.SmbvError):
        ops.window_attention_fwd(q, q, q)
    with pytest.raises(_lib.SmbvError):
        ops.window_attention_bwd(q, q, q, q, q, torch.zeros(1, 2, 4))
    with pytest.raises(_lib.SmbvError):
        ops.rope_axes(q, q, torch.zeros(1, 4, dtype=torch.int32), torch.ones(32), (32,))
    with pytest.raises(_lib.SmbvError):
        ops.gated_norm_fwd(q, q)
    with pytest.raises(_lib.SmbvError):
        ops.gated_norm_bwd(q, q, q, q, torch.zeros(8, 4))


Z = torch.zeros


@pytest.mark.parametrize("args,kw", [
    ((Z(1, 4, 2, 64), Z(1, 4, 2, 64), Z(1, 4, 2, 64)), {}),                                                           # fp32
    ((Z(1, 4, 2, 64, dtype=BF), Z(1, 4, 2, 64, dtype=HF), Z(1, 4, 2, 64, dtype=BF)), {}),
    ((Z(4, 2, 64, dtype=BF), Z(1, 4, 2, 64, dtype=BF), Z(1, 4, 2, 64, dtype=BF)), {}),
    ((Z(1, 4, 2, 64, dtype=BF), Z(2, 4, 2, 64, dtype=BF), Z(2, 4, 2, 64, dtype=BF)), {}),
    ((Z(1, 4, 2, 64, dtype=BF), Z(1, 4, 2, 64, dtype=BF), Z(1, 5, 2, 64, dtype=BF)), {}),
    ((Z(1, 4, 2, 64, dtype=BF), Z(1, 4, 2, 32, dtype=BF), Z(1, 4, 2, 32, dtype=BF)), {}),
    ((Z(1, 4, 2, 64, dtype=BF), Z(1, 4, 64, 2, dtype=BF).transpose(2, 3), Z(1, 4, 2, 64, dtype=BF)), {}),            # channels not contiguous
    ((Z(1, 4, 2, 64, dtype=BF),) * 3, dict(q_lens=Z(1, dtype=torch.int64))),
    ((Z(1, 4, 2, 64, dtype=BF),) * 3, dict(k_lens=Z(2, dtype=torch.int32))),
    ((Z(1, 4, 2, 64, dtype=BF),) * 3, dict(sinks=-1)),
    ((Z(1, 4, 2, 64, dtype=BF),) * 3, dict(out=Z(1, 4, 2, 64))),
    ((Z(1, 4, 2, 64, dtype=BF),) * 3, dict(out=Z(1, 1, 2, 64, dtype=BF).expand(1, 4, 2, 64))),
], ids=range(12))
def test_window_attention_arguments(dry, args, kw):
    with pytest.raises(ValueError):
        ops.window_attention_fwd(*args, **kw)


def test_window_attention_outputs_apart(dry):
    q, k, v = (Z(1, 4, 2, 64, dtype=BF) for _ in range(3))
    lse, o = Z(1, 2, 4), Z(1, 4, 2, 64, dtype=BF)
    with pytest.raises(ValueError):
        ops.window_attention_fwd(q, k, v, out=q)
    for kw in (dict(out=(q, Z(1, 4, 2, 64, dtype=BF), Z(1, 4, 2, 64, dtype=BF))), dict(out=(o.clone(),) + (k.clone(),) * 1 + (o,)), dict(o_lo=Z(1, 2, 4, 64, dtype=BF).transpose(1, 2))):
        with pytest.raises(ValueError):
            ops.window_attention_bwd(q, k, v, o, o.clone(), lse, **kw)
    same = Z(1, 4, 2, 64, dtype=BF)
    with pytest.raises(ValueError):
        ops.window_attention_bwd(q, k, v, o, o.clone(), lse, out=(same, same, same))
    for bad in (lse.double(), Z(1, 4, 2), Z(1, 4, 2).transpose(1, 2)):
        with pytest.raises(ValueError):
            ops.window_attention_bwd(q, k, v, o, o.clone(), bad)


@pytest.mark.parametrize("change", [dict(q=Z(1, 4, 2, 64, dtype=torch.float64)), dict(q=Z(4, 2, 64)), dict(k=Z(1, 4, 1, 32)), dict(k=Z(1, 4, 1, 64, dtype=BF)), dict(k=Z(1, 5, 1, 64)),
                                    dict(pos=Z(3, 1, 4)), dict(pos=Z(2, 1, 4, dtype=torch.int32)), dict(pos=Z(4, dtype=torch.int32)), dict(inv=Z(31)),
                                    dict(inv=Z(32, dtype=torch.float64)), dict(sections=()), dict(sections=(8,) * 5), dict(sections=(40, -4, -4)), dict(sections=(20, 20, 20)),
                                    dict(out=(None, None)), dict(out=(Z(1, 4, 2, 64), Z(1, 4, 1, 32)))], ids=str)
def test_rope_axes_arguments(dry, change):
    a = dict(q=Z(1, 4, 2, 64), k=Z(1, 4, 1, 64), pos=Z(3, 1, 4, dtype=torch.int32), inv=Z(32), sections=(12, 10, 10), out=None)
    a.update(change)
    with pytest.raises(ValueError):
        ops.rope_axes(a["q"], a["k"], a["pos"], a["inv"], a["sections"], out=a["out"])


def test_rope_axes_partial_overlap(dry):
    buf = Z(1, 5, 2, 64)
    with pytest.raises(ValueError):
        ops.rope_axes(buf[:, :4], None, Z(1, 4, dtype=torch.int32), Z(32), (32,), out=(buf[:, 1:], None))


def test_outputs_are_tensors_of_their_own(dry, monkeypatch):
    made = []
    monkeypatch.setattr(ops, "_call", lambda plan, name, *a, **kw: made.append(name))
    q, k, pos = Z(1, 4, 1, 64), Z(1, 4, 1, 64), Z(1, 4, dtype=torch.int32)
    same = Z(1, 4, 1, 64)
    with pytest.raises(ValueError):
        ops.rope_axes(q, k, pos, Z(32), (32,), out=(same, same))
    packed = Z(2, 4, 6, 64)
    pos = Z(1, 2, 4, dtype=torch.int32)
    for a, b in ((packed[:, :, :4], packed[:, :, 3:5]), (packed[:, :, 2:], packed[:, :, :3]), (packed[:, :3], packed[:, 1:]), (packed, packed)):
        with pytest.raises(ValueError):   # turned in place, some heads twice
            ops.rope_axes(a, b, pos[..., :a.shape[1]], Z(32), (32,), out=(a, b))
    ops.rope_axes(packed[:, :, :4], packed[:, :, 4:], pos, Z(32), (32,), out=(packed[:, :, :4], packed[:, :, 4:]))   # the columns of one packed tensor
    q, k, v = (Z(2, 4, n, 64, dtype=BF) for n in (2, 1, 1))
    o, lse, grad = q.clone(), Z(2, 2, 4), Z(2, 4, 4, 64, dtype=BF)
    ops.window_attention_bwd(q, k, v, o, o.clone(), lse, out=(grad[:, :, :2], grad[:, :, 2:3], grad[:, :, 3:]))
    assert made == ["smbv_rope_axes", "smbv_window_attention_bwd"]
    for a, b, c in ((2, 2, 3), (1, 4, 3)):   # dk inside dq, dk on dv
        with pytest.raises(ValueError):
            ops.window_attention_bwd(q, k, v, o, o.clone(), lse, out=(grad[:, :, a - 1:a + 1], grad[:, :, b - 1:b], grad[:, :, c:]))
    a = dict(GOOD)
    h, x = a.pop("h"), a.pop("x")
    with pytest.raises(ValueError):
        ops.gated_norm_fwd(h, x, out=(None, h.clone()), **a)
    for out in ((None, x.clone()), (h.clone(), None)):
        with pytest.raises(ValueError):
            ops.gated_norm_bwd(x.clone(), h.clone(), h, x, Z(12, 4), out=out, **a)


GOOD = dict(h=Z(2, 6, 64, dtype=BF), x=Z(2, 6, 64), post="rms", pre="layer", post_w=Z(64), post_b=None, gate=Z(2, 64), pre_w=Z(64), pre_b=Z(64))


@pytest.mark.parametrize("change", [dict(post="batch"), dict(pre=True), dict(h=Z(2, 6, 64, dtype=torch.float64)), dict(x=Z(2, 6, 64, dtype=HF)), dict(x=Z(2, 5, 64)), dict(h=Z(2, 6, 0, dtype=BF)),
                                    dict(post_w=Z(63)), dict(post_w=Z(64, dtype=BF)), dict(pre_b=Z(128)[::2]), dict(gate=Z(6, 64)), dict(gate=Z(1, 6, 64)), dict(gate=Z(2, 32)),
                                    dict(gate=Z(2, 64, dtype=BF)), dict(gate=Z(64, 2).T), dict(h=Z(2, 64, 6, dtype=BF).transpose(1, 2)), dict(x=Z(6, 2, 64).transpose(0, 1))], ids=str)
def test_gated_norm_arguments(dry, change):
    a = {**GOOD, **change}
    h, x = a.pop("h"), a.pop("x")
    with pytest.raises(ValueError):
        ops.gated_norm_fwd(h, x, **a)
    with pytest.raises(ValueError):
        ops.gated_norm_bwd(Z(2, 6, 64), Z(2, 6, 64, dtype=BF), h, x, Z(12, 4), **a)


def test_gated_norm_more_arguments(dry):
    a = dict(GOOD)
    h, x = a.pop("h"), a.pop("x")
    for out in ((x.bfloat16(), h.clone()), (x.clone(), h), (x.clone(), None), (x[:, :, :1].expand(2, 6, 64), h.clone()), (x.clone(), x.bfloat16()[:, :5])):
        with pytest.raises(ValueError):
            ops.gated_norm_fwd(h, x, out=out, **a)
    dx1, dy, st = x.clone(), h.clone(), Z(12, 4)
    for args in ((None, None, h, x, st), (dx1, None, h, x, st), (dx1.bfloat16(), dy, h, x, st), (dx1, dy.float(), h, x, st), (dx1, dy, h, x, Z(12, 3)), (dx1, dy, h, x, Z(4, 12).T)):
        with pytest.raises(ValueError):
            ops.gated_norm_bwd(*args, **a)
    with pytest.raises(ValueError):
        ops.gated_norm_bwd(dx1, dy, h, x, st, out=(h, x.clone()), **a)
    with pytest.raises(ValueError):
        ops.gated_norm_bwd(None, dy, h, x, st, **{**a, "pre": None, "pre_w": None, "pre_b": None})


def test_window_plugin_registers_and_refuses_cpu():
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    from smb_vision_amd import attention_plugin
    name = attention_plugin.register_window(window=(8, 8), sinks=2)
    assert name == "smbv_window" and name in ALL_ATTENTION_FUNCTIONS
    q = Z(1, 2, 16, 64)
    with pytest.raises(RuntimeError):
        ALL_ATTENTION_FUNCTIONS[name](torch.nn.Module(), q, q, q, None, scaling=0.125, dropout=0.0)
    with pytest.raises(ValueError):
        ALL_ATTENTION_FUNCTIONS[name](torch.nn.Module(), q, q, q, Z(1, 1, 16, 16))


def test_turned_in_place_beside_an_operand_that_is_still_read(dry, monkeypatch):
    made = []
    monkeypatch.setattr(ops, "_call", lambda plan, name, *a, **kw: made.append(name))
    packed, pos = Z(2, 4, 6, 64), Z(1, 2, 4, dtype=torch.int32)
    q, k, new = packed[:, :, :4], packed[:, :, 4:], lambda n: Z(2, 4, n, 64)
    for a, b, out in ((q, q, (q, new(4))), (q, packed[:, :, 3:5], (q, new(2))), (packed[:, :, 2:4], q, (new(2), q)), (q, packed[:, :, 1:2], (q, new(1)))):
        with pytest.raises(ValueError):
            ops.rope_axes(a, b, pos, Z(32), (32,), out=out)
    assert not made
    ops.rope_axes(q, k, pos, Z(32), (32,), out=(q, new(2)))
    ops.rope_axes(q, k, pos, Z(32), (32,), out=(new(4), k))
    ops.rope_axes(q, k, pos, Z(32), (32,), out=(q, k))
    ops.rope_axes(q, None, pos, Z(32), (32,), out=(q, None))
    assert made == ["smbv_rope_axes"] * 4


def test_heads_may_lie_far_apart():
    """Head-major operands [B, H, S, D] of any length: the call gets as far as its workspace (too small here, so nothing is launched)."""
    lib = _lib.load()
    for S, D in ((1 << 17, 128), (1 << 18, 64), (1 << 22, 128)):
        q, k = _lib.c_ll3(4 * S * D, D, S * D), _lib.c_ll3(2 * S * D, D, S * D)
        a = attn(B=1, Sq=S, Sk=S, Dh=D, sq=q, so=q, sdo=q, sdq=q, sk=k, sv=k, sdk=k, sdv=k)
        assert lib.smbv_window_attention_bwd(C.byref(a), P, 256, None) == -4, _lib.last_error()
        a.Sq, a.H, a.left = 1, 8, -1   # one token: the shares of its keys need a workspace
        assert lib.smbv_window_attention_fwd(C.byref(a), P, 256, None) == -4, _lib.last_error()
    for far in (dict(sk=_lib.c_ll3(0, 1 << 24, 64)), dict(sv=_lib.c_ll3(0, 1 << 24, 64)), dict(sq=_lib.c_ll3(0, 256, 1 << 40)), dict(so=_lib.c_ll3(0, 1 << 40, 64))):
        assert lib.smbv_window_attention_fwd(C.byref(attn(**far)), P, 1 << 40, None) == -1 and "apart" in _lib.last_error()


def test_outputs_lie_apart_from_the_lengths(dry):
    q, k, v = (Z(2, 4, n, 64, dtype=BF) for n in (2, 1, 1))
    o, lse, fresh = q.clone(), Z(2, 2, 4), lambda: [t.clone() for t in (q, k, v)]
    for name in ("q_lens", "k_lens"):
        out = fresh()
        lens = {name: out[0].view(-1)[8:12].view(torch.int32)}
        with pytest.raises(ValueError, match="overlap"):
            ops.window_attention_fwd(q, k, v, out=out[0], **lens)
        for n in range(3):
            out = fresh()
            with pytest.raises(ValueError, match="overlap"):
                ops.window_attention_bwd(q, k, v, o, o.clone(), lse, out=out, **{name: out[n].view(-1)[8:12].view(torch.int32)})
