"""The token operators' refusals and layouts, without a GPU: the C entry points check their arguments before any launch,
the Python ones before they touch a device."""
import ctypes
import math

import pytest
import torch

from vision_assist_amd import _lib
from vision_assist_amd.tokens import (AttnArgs, Linear, LinearArgs, QKArgs, QKNorm, Rotary, TokenCache, _apart, _interleaved,
                                      _own_elements, attend)

ERR = _lib.VA_ERR_ARG
P = 4096  # a pointer that is aligned and never read


def linear(**kw):
    a = dict(x=P, w=P, y=P, ldx=64, ldr=0, ldy=64, M=0, N=64, K=64, Npad=64, Kpad=64, dtype=1, w8=0, act=0, out_f32=0)
    return _lib.load().va_tok_linear(None, ctypes.byref(LinearArgs(**{**a, **kw})))


def qk(**kw):
    a = dict(q=P, k=P, q_out=P, k_out=P, eps=1e-6, B=0, S=1, Hq=1, Hk=1, D=64, dtype=1)
    return _lib.load().va_tok_qk(None, ctypes.byref(QKArgs(**{**a, **kw})))


ATTN = dict(q=P, k=P, v=P, o=P, scale=0.1, B=0, S=1, Hq=2, Hk=1, D=64, Dv=64, slots=8, frame=1, dtype=1)


def attn(**kw):
    a = AttnArgs(**{**ATTN, **kw})
    lib = _lib.load()
    rc = lib.va_tok_attn(None, ctypes.byref(a))
    assert (lib.va_tok_attn_workspace_bytes(ctypes.byref(a)) < 0) == (rc != 0)
    return rc


def test_struct_sizes():
    out = (ctypes.c_int64 * 14)()
    assert _lib.load().va_abi_struct_sizes(out, 14) == 14
    assert list(out)[11:] == [ctypes.sizeof(t) for t in (LinearArgs, QKArgs, AttnArgs)]


def test_nothing_to_do_is_fine():
    assert linear() == qk() == attn() == 0
    assert linear(x=None) == 0 and qk(B=3, S=0) == 0 and qk(B=3, Hq=0, Hk=0) == 0 and attn(B=2, S=0, q=None) == 0


@pytest.mark.parametrize("kw", [dict(M=-1), dict(N=0), dict(K=0), dict(w=None), dict(y=None), dict(M=1, x=None), dict(dtype=0),
                                dict(dtype=3), dict(w8=1), dict(w8=2, wscale=P), dict(wscale=P), dict(w8=1, wscale=P, dtype=2),
                                dict(act=5), dict(act=-1), dict(N=65, ldy=65), dict(Npad=96), dict(K=65, ldx=65), dict(Kpad=96),
                                dict(w=P + 8), dict(ldx=63), dict(ldy=63), dict(res=P, ldr=63), dict(x=P + 1), dict(y=P + 1),
                                dict(y=P + 2, out_f32=1), dict(bias=P + 2), dict(x=P + 2, dtype=2)])
def test_linear_refuses(kw):
    assert linear(**kw) == ERR


@pytest.mark.parametrize("kw", [dict(B=-1), dict(S=-1), dict(Hq=-1), dict(Hk=-1), dict(D=0), dict(D=257), dict(dtype=3), dict(rot=3),
                                dict(rot=66), dict(rot=64), dict(rot=64, turns=P, axis=P), dict(rot=64, turns=P, axis=P, pos=P),
                                dict(rot=64, turns=P + 4, axis=P, pos=P, axes=1), dict(layout=2), dict(eps=-1.0), dict(eps=math.nan),
                                dict(B=1, q=None), dict(B=1, k_out=None), dict(slots=-1), dict(slots=4, sinks=4), dict(sinks=-1),
                                dict(B=1, slots=4), dict(B=1, slots=4, v=P, v_out=P, Dv=0), dict(Hq=1 << 21)])
def test_qk_refuses(kw):
    assert qk(**kw) == ERR


@pytest.mark.parametrize("kw", [dict(B=-1), dict(S=-1), dict(Hk=0), dict(Hq=0), dict(Hq=3, Hk=2), dict(slots=-1), dict(D=60), dict(D=136),
                                dict(D=0), dict(Dv=4), dict(Dv=160), dict(frame=-1), dict(window=-1), dict(sinks=-1), dict(sinks=8),
                                dict(frame=0, window=4), dict(frame=0, sinks=1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf),
                                dict(scale=math.nan), dict(dtype=3), dict(q_ss=4), dict(o_sh=7), dict(k_sb=12), dict(B=1, q=None),
                                dict(B=1, k=None), dict(B=1, o=None), dict(q=P + 8), dict(v=P + 2), dict(S=2 ** 31 - 1)])
def test_attn_refuses(kw):
    assert attn(**kw) == ERR


def test_null_arguments():
    lib = _lib.load()
    assert lib.va_tok_linear(None, None) == lib.va_tok_qk(None, None) == lib.va_tok_attn(None, None) == ERR
    assert lib.va_tok_attn_workspace_bytes(None) == ERR


def test_ops_of_a_list_pass_refusals_on():
    from vision_assist_amd.seg import ConvArgs, SegOp
    a = LinearArgs(M=-1)
    ops = (SegOp * 1)(SegOp(kind=10, a=ConvArgs(x=ctypes.addressof(a))))
    assert _lib.load().va_seg_run(None, ops, 1) == ERR - 1000
    for kind in (10, 11, 12):
        assert _lib.load().va_seg_run(None, (SegOp * 1)(SegOp(kind=kind)), 1) == ERR - 1000


def test_overlaps():
    x = torch.zeros(3, 5, 12, 8)
    q, k, v = x[:, :, :4], x[:, :, 4:8], x[:, :, 8:]
    assert _interleaved(q, k) and _interleaved(k, q) and _interleaved(q, v) and not _interleaved(q, x[:, :, 3:7])
    y = torch.zeros(3, 12, 5, 8).transpose(1, 2)
    assert _interleaved(y[:, :, :4], y[:, :, 4:9]) and not _interleaved(y[:, :, :5], y[:, :, 4:9])
    _apart(q, k, "k")
    _apart(q, q, "q", same_ok=True)
    for bad in (x[:, :, 3:7], x, q[:, :, :2]):
        with pytest.raises(_lib.VaError):
            _apart(q, bad, "x", same_ok=True)
    with pytest.raises(_lib.VaError):
        _apart(q, q, "q")
    _own_elements(q)
    with pytest.raises(_lib.VaError):
        _own_elements(torch.zeros(1, 4).expand(3, 4))


@pytest.mark.parametrize("kw", [dict(frame=-1), dict(window=-2), dict(sinks=-1), dict(sinks=10), dict(frame=0, window=3), dict(scale=0.0),
                                dict(scale=math.inf), dict(scale=-0.5), dict(frame=2 ** 31)])
def test_attend_refuses(kw):
    q, k = torch.zeros(2, 3, 4, 64), torch.zeros(2, 10, 2, 64)
    with pytest.raises(_lib.VaError):
        attend(q, k, k, **kw)


@pytest.mark.parametrize("q,k,v", [((2, 3, 4, 64), (2, 10, 3, 64), (2, 10, 3, 64)), ((2, 3, 4, 64), (1, 10, 2, 64), (1, 10, 2, 64)),
                                   ((2, 3, 4, 60), (2, 10, 2, 60), (2, 10, 2, 64)), ((2, 3, 4, 64), (2, 10, 2, 64), (2, 9, 2, 64)),
                                   ((2, 3, 4, 64), (2, 10, 2, 64), (2, 10, 2, 136)), ((2, 3, 4, 64), (2, 10, 2, 32), (2, 10, 2, 64)),
                                   ((3, 4, 64), (2, 10, 2, 64), (2, 10, 2, 64)), ((2, 3, 4, 256), (2, 10, 2, 256), (2, 10, 2, 256))])
def test_attend_refuses_shapes(q, k, v):
    with pytest.raises(_lib.VaError):
        attend(torch.zeros(q), torch.zeros(k), torch.zeros(v))


def test_attend_refuses_types_and_places():
    q, k = torch.zeros(2, 3, 4, 64), torch.zeros(2, 10, 2, 64)
    for a in ((q.half(), k.half(), k.half()), (q, k.bfloat16(), k), (q, k, k.double())):
        with pytest.raises(_lib.VaError):
            attend(*a)
    with pytest.raises(_lib.VaError):
        attend(q, k, k, q_len=torch.zeros(2))
    with pytest.raises(_lib.VaError):
        attend(q, k, k, kv_len=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(_lib.VaError):  # no GPU tensors: nothing computes on the host
        attend(q, k, k)


BIG = 2 ** 31 - 1


@pytest.mark.parametrize("call,kw", [(linear, dict(M=BIG)), (linear, dict(Npad=BIG - 63, N=BIG - 100, ldy=BIG)),
                                     (linear, dict(Kpad=BIG - 63, K=BIG - 100, ldx=BIG)), (attn, dict(slots=BIG)), (attn, dict(k_ss=-8)),
                                     (attn, dict(v_ss=-64)), (attn, dict(k_ss=1 << 22)), (attn, dict(v_ss=1 << 24)),
                                     (qk, dict(B=1, slots=4, v=P, v_out=P, Hk=1 << 12, Dv=1 << 19))])
def test_sides_and_strides_that_the_kernels_do_not_count(call, kw):
    assert call(**kw) == ERR


@pytest.mark.parametrize("call,kw", [(linear, dict(M=1 << 30, N=1 << 30, Npad=1 << 30, ldy=1 << 30)),
                                     (linear, dict(M=1 << 30, N=1 << 30, Npad=1 << 30, ldy=1 << 30, K=63)),
                                     (qk, dict(B=1 << 20, S=1 << 20)), (qk, dict(B=1 << 20, S=1 << 20, D=33))])
def test_more_workgroups_than_a_launch_has(call, kw):
    rc = call(**{**dict(x=P), **kw} if call is linear else kw)
    assert rc == _lib.VA_ERR_RANGE


def test_more_workgroups_than_a_launch_has_attention():
    lib = _lib.load()
    a = AttnArgs(**{**ATTN, "B": 1 << 20, "S": 1 << 20, "ws": P, "ws_bytes": 1 << 62})
    assert lib.va_tok_attn(None, ctypes.byref(a)) == _lib.VA_ERR_RANGE


def test_tensors_whose_addresses_calls_take_are_not_replaced():
    c = TokenCache.of(torch.zeros(2, 8, 3, 16), torch.zeros(2, 8, 3, 8), sinks=2)
    for n in ("k", "v", "sinks", "len"):
        with pytest.raises(AttributeError):
            setattr(c, n, getattr(c, n))
    before = c.len.data_ptr()
    assert c.advance(3).advance(torch.tensor([1, 2])).len.tolist() == [4, 5] and c.len.data_ptr() == before
    for cls, names in ((Linear, ("w", "wscale", "bias")), (Rotary, ("turns", "axis")), (QKNorm, ("wq", "wk", "rotary"))):
        for n in names:
            with pytest.raises(AttributeError):
                setattr(cls.__new__(cls), n, None)
