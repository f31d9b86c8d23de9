"""Edges of the token operators that need no GPU: the terms of float weights, refusals, the counts of a cache."""
import math

import pytest
import torch

from vision_assist_amd import _lib
from vision_assist_amd.tokens import _terms


def test_terms_of_any_weight():
    big, top = torch.finfo(torch.float32).max, torch.finfo(torch.bfloat16).max
    edge = float.fromhex("0x1.ffp127")  # the first value whose nearest bf16 is an infinity
    under = torch.nextafter(torch.tensor(edge), torch.tensor(0.0)).item()
    w = torch.tensor([[0.0, 1.0, -1.7, 3e-20, big, -big, edge, under, top, -under, 1e38, math.pi, -2.0 ** -100, 7.0, 65535.0, -0.1]])
    t = _terms(w)
    assert t.dtype == torch.bfloat16 and t.isfinite().all()
    assert torch.equal(t.double().sum(0), w.double())
    w[0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    t = _terms(w).float()
    assert t[:, 0, 0].tolist() == [1, 0, math.inf] and t[:, 0, 1].tolist() == [-1, 0, -math.inf] and t[:, 0, 2].isnan().any()
    assert torch.equal(t[:, :, 3:].double().sum(0), w[:, 3:].double())


def test_attend_refuses_to_lose_a_gradient():
    from vision_assist_amd.tokens import attend
    for i in range(3):
        a = [torch.zeros(2, 3, 4, 64), torch.zeros(2, 10, 2, 64), torch.zeros(2, 10, 2, 64)]
        a[i].requires_grad_()
        with pytest.raises(_lib.VaError, match="gradient"):
            attend(*a)
        with torch.no_grad(), pytest.raises(_lib.VaError, match="on the GPU"):
            attend(*a)


@pytest.mark.parametrize("slots,sinks,frame", [(300, 4, 1), (2804, 4, 400), (1000, 0, 0), (77, 76, 25)])
def test_rebase_sets_large_counts_back_by_rings_and_frames(slots, sinks, frame):
    from vision_assist_amd.tokens import TokenCache
    n = [0, 5, slots, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 12345678, 2 ** 31 - 1]
    k = torch.zeros(len(n), slots, 1, 8)
    c = TokenCache.of(k, k.clone(), sinks=sinks, length=torch.tensor(n, dtype=torch.int32))
    at = c.len.data_ptr()
    turn = math.lcm(slots - sinks, frame or 1)
    got = c.rebase(frame).len.tolist()
    assert c.len.data_ptr() == at and got[:5] == n[:5]
    assert all((a - b) % turn == 0 and 2 ** 30 <= a < 2 ** 30 + turn for a, b in zip(got[4:], n[4:]))
    assert c.rebase(frame).len.tolist() == got


def test_rebase_refuses():
    from vision_assist_amd.tokens import TokenCache
    k = torch.zeros(1, 1009, 1, 8)
    c = TokenCache.of(k, k.clone())
    for frame in (-1, 2 ** 20 + 7):
        with pytest.raises(_lib.VaError):
            c.rebase(frame)


def layer(N=6, K=4, dtype=torch.bfloat16):
    """A Linear without weights on the CPU: what its calls check comes before they are read."""
    from vision_assist_amd.tokens import Linear
    lin = Linear.__new__(Linear)
    lin.device, lin.N, lin.K, lin.tdtype = torch.device("cpu"), N, K, dtype
    lin._ptrs, lin._ints = (4096, 0, 0), (N, K, 64, 64, 1, 0, 0)
    return lin


def test_args_of_an_op_list_are_checked():
    lin, z = layer(), lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)
    x, y = z(5, 4), z(5, 6)
    a = lin.args(x, y, residual=y)
    assert (a.M, a.N, a.K, a.ldx, a.ldy, a.ldr, a.x, a.y, a.res) == (5, 6, 4, 4, 6, 6, x.data_ptr(), y.data_ptr(), y.data_ptr())
    wide = z(5, 20)
    assert lin.args(wide[:, 3:7], wide[:, 10:16]).ldx == 20 and lin.args(x, z(5, 6, dtype=torch.float32)).out_f32 == 1
    for bad in ((z(5, 3), y), (z(2, 5, 4), y), (z(4, 5).t(), y), (z(1, 4).expand(5, 4), y), (z(5, 4, dtype=torch.float32), y), (x, z(5, 5)),
                (x, z(4, 6)), (x, z(6, 5).t()), (x, z(5, 6, dtype=torch.float16)), (wide[:, 2:6], wide[:, 4:10]),
                (x, y, z(5, 5)), (x, y, z(5, 6, dtype=torch.float32)), (x, y, z(1, 6).expand(5, 6)), (x, wide[:, :6], wide[:, 1:7]),
                (x, z(1, 6).expand(5, 6))):
        with pytest.raises(_lib.VaError):
            lin.args(*bad)


def test_the_form_of_a_call():
    import ctypes

    from vision_assist_amd.tokens import LinearArgs
    lib, a = _lib.load(), dict(x=4096, w=4096, y=4096, ldx=64, ldy=64, N=64, K=64, Npad=64, Kpad=64, dtype=1)
    form = lambda **kw: lib.va_tok_linear_form(ctypes.byref(LinearArgs(**{**a, **kw})))
    assert lib.va_tok_linear_form(None) == form(M=-1) == form(dtype=3) == _lib.VA_ERR_ARG
    assert form(M=1) == form(M=64) == form(M=1, dtype=2) == 1 and form(M=1, x=4098) == form(M=1, K=63) == 0
    assert form(M=20000) == form(M=1 << 20, dtype=2) == 2 and form(M=20000, dtype=2) == 3
    assert form(M=1 << 20) == form(M=1 << 20, w8=1, wscale=4096) == 4
