"""The token operators (vision_assist_amd.tokens) against plain float64 implementations on the CPU.

Tolerances, per element, from the roundings a result goes through (half a step relative to the value: bf16 2^-8, float
2^-24):

* Linear, float sums of K products: |error| <= (K + 8) 2^-24 sum |x w| in any order of summation; the six-term form of a
  float product adds 2^-25 of it; the activations have a slope of at most 1.13 (SiLU 1.10, GELU 1.13) and a few float
  roundings of their value; then one rounding to the output's type.
* QKNorm: the mean of squares and its root, weight and rotation: about 16 float roundings of values bounded by the pair's
  norm, and the angle's float sine and cosine (2^-22 absolute); then one rounding to the output's type.
* attend: scores err by (D + 4) 2^-24 scale sum |q k| plus 2^-23 of themselves, so a probability errs by that factor
  (e^x - 1, twice: numerator and denominator); bf16 rounds a probability once more (2^-8 of it at most); then the
  output's rounding.  Against sum p |v|.
"""
import math

import pytest
import torch

from vision_assist_amd import _lib

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32, "w8a16": torch.bfloat16}
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rnd(g, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(shape, generator=g) * by).to(dtype)


def act64(y, act):
    F = torch.nn.functional
    return {None: lambda t: t, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh"),
            "relu": F.relu}[act](y)


# ------------------------------------------------------------------ Linear
def linear_ref(x, w, bias, act, res, scale):
    """-> (value, bound of the float sums) in float64; w as the kernel holds it."""
    x, w = x.double(), w.double()
    if scale is not None:
        w = w * scale.double()[:, None]
    y, mag = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    y = act64(y, act)
    return (y if res is None else y + res.double()), (x.shape[1] + 8) * 2.0 ** -24 * mag


def check(got, want, bound, what=""):
    got = got.double().cpu()
    u = U[torch.bfloat16] if bound[1] == "bf16" else U[torch.float32]
    tol = bound[0] + u * (want.abs() + bound[0])
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).max():.3g} x"


def run_linear(dtype, M, K, N, act=None, bias=True, res=False, seed=0, out_f32=False, x=None, out=None, stream=None):
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(seed)
    t = DT[dtype]
    xh = rnd(g, M, K, dtype=t)
    w = rnd(g, N, K, by=K ** -0.5)
    b = rnd(g, N, by=0.3) if bias else None
    r = rnd(g, M, N, dtype=t) if res else None
    scale = None
    if dtype == "w8a16":
        scale = w.abs().amax(1) / 448
        w = (w / scale[:, None]).to(torch.float8_e4m3fn)
    elif dtype == "bf16":
        w = w.to(torch.bfloat16)
    lin = Linear(w, b, act=act, dtype=dtype, scale=scale, device="cuda")
    o = torch.full((M, N), 7.0, dtype=torch.float32, device="cuda") if out_f32 else None
    got = lin(xh.cuda(), residual=None if r is None else r.cuda(), out=o)
    want, sums = linear_ref(xh, w.float(), b, act, r, scale)
    check(got, want, (1.2 * sums + 2.0 ** -21 * want.abs() + 2.0 ** -30, "f32" if out_f32 or dtype == "f32" else "bf16"),
          f"{dtype} {M}x{K}x{N} {act}")
    return lin, xh, got


@pytest.mark.parametrize("dtype", ["bf16", "w8a16", "f32"])
@pytest.mark.parametrize("M,K,N", [(1, 64, 64), (1, 1024, 520), (2, 72, 130), (5, 1, 1), (15, 40, 1001), (16, 512, 256),
                                   (17, 333, 77), (32, 4096, 192), (33, 128, 2048), (64, 64, 64), (100, 520, 1000),
                                   (129, 200, 257), (400, 256, 512), (777, 1000, 65), (2049, 96, 300)])
def test_linear_sizes(dtype, M, K, N):
    run_linear(dtype, M, K, N, act="silu" if M % 2 else None, bias=N % 2 == 0, res=K % 3 == 0, seed=M + K + N)


@pytest.mark.parametrize("dtype", ["bf16", "w8a16", "f32"])
@pytest.mark.parametrize("act", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("M", [3, 300])
def test_linear_epilogue(dtype, act, M):
    for bias, res, f in ((True, True, False), (False, False, dtype != "f32"), (False, True, dtype != "f32")):
        run_linear(dtype, M, 136, 192, act, bias, res, seed=M, out_f32=f)


@pytest.mark.parametrize("dtype", ["bf16", "w8a16", "f32"])
@pytest.mark.parametrize("M,K,N", [(1024, 512, 1024), (1300, 1032, 1536), (4096, 256, 768)])
def test_linear_large(dtype, M, K, N):
    run_linear(dtype, M, K, N, act="gelu", res=True, seed=K)


@pytest.mark.parametrize("dtype", ["bf16", "w8a16", "f32"])
@pytest.mark.parametrize("M", [4, 160, 1100])
def test_linear_strides(dtype, M):
    """Rows inside wider rows, odd strides and offsets, a transposed x, three leading sizes, out = residual.  Rows that
    cannot be read in 16-byte pieces take another kernel, whose float sums run in another order: two such sums differ by
    at most 2 (K + 8) 2^-24 sum |x w| (each is within half of that of the exact one), and their roundings to the type by a
    step more."""
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(3)
    t, K, N = DT[dtype], 128, 320
    w, b = rnd(g, N, K, by=0.1), rnd(g, N)
    lin = Linear(w, b, act="relu", dtype=dtype, device="cuda")
    wide = rnd(g, M, 2 * K + 5, dtype=t).cuda()

    def near(got, want, x):
        mag = (x.double().abs().cpu() @ w.double().abs().t() + b.double().abs()) * (1 + 2.0 ** -4)  # (e4m3: 2^-4 more)
        tol = 2 * (K + 8) * 2.0 ** -24 * mag + 2 * U[t] * want.double().abs().cpu()
        return bool(((got.double() - want.double()).abs().cpu() <= tol).all())

    for x in (wide[:, 5:5 + K], wide[:, 8:8 + K], rnd(g, K, M, dtype=t).cuda().t(), wide[:, :K].reshape(2, M // 2, K)):
        assert near(lin(x), lin(x.contiguous()), x)
    x, res = wide[:, :K], rnd(g, M, N, dtype=t).cuda()
    base = lin(x, residual=res)
    for width, off in ((N + 7, 3), (N + 8, 8)):
        buf = torch.full((M, width), 5.0, dtype=t, device="cuda")
        buf[:, off:off + N] = res
        o = buf[:, off:off + N]
        assert lin(x, residual=o, out=o) is o and torch.equal(o, base)
        assert (buf[:, :off] == 5).all() and (buf[:, off + N:] == 5).all()
    one = wide[:1, :K].contiguous()
    assert torch.equal(lin(one.expand(M, K)), lin(one.expand(M, K).contiguous()))


@pytest.mark.parametrize("dtype", ["bf16", "w8a16", "f32"])
@pytest.mark.parametrize("M", [1, 24, 200, 2048])
def test_linear_nonfinite_stay_in_their_rows(dtype, M):
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(4)
    t, K, N = DT[dtype], 200, 576
    lin = Linear(rnd(g, N, K, by=0.1), None, dtype=dtype, device="cuda")
    x = rnd(g, M, K, dtype=t)
    clean = lin(x.cuda())
    x[M // 2, K - 1] = math.nan
    x[M - 1, 0] = math.inf
    got = lin(x.cuda())
    hit = {M // 2, M - 1}
    rows = torch.tensor([i for i in range(M) if i not in hit], dtype=torch.long)
    assert torch.equal(got[rows.cuda()], clean[rows.cuda()])
    assert got[M // 2].isnan().all() and not got[M - 1].isfinite().any()


def test_linear_empty_and_one():
    from vision_assist_amd.tokens import Linear
    lin = Linear(torch.randn(48, 24), torch.randn(48), device="cuda")
    assert lin(torch.empty(0, 24, dtype=torch.bfloat16, device="cuda")).shape == (0, 48)
    assert lin(torch.empty(2, 0, 24, dtype=torch.bfloat16, device="cuda")).shape == (2, 0, 48)
    x = torch.randn(24, device="cuda").bfloat16()
    assert torch.equal(lin(x), lin(x[None])[0])


@pytest.mark.parametrize("dtype", ["bf16", "w8a16", "f32"])
def test_linear_rows_do_not_depend_on_their_number(dtype):
    """A row of a batch is the row alone to within the order of its sums, and the same call gives the same bits."""
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(5)
    lin = Linear(rnd(g, 700, 1000, by=0.03), rnd(g, 700), act="gelu", dtype=dtype, device="cuda")
    x = rnd(g, 1500, 1000, dtype=DT[dtype]).cuda()
    full = lin(x)
    assert torch.equal(full, lin(x))
    for M in (1, 16, 40, 200, 700):
        part = lin(x[:M])
        tol = 2.0 ** -7 if dtype != "f32" else 2e-5
        assert (part.float() - full[:M].float()).abs().max() <= tol * full.float().abs().max()


# ------------------------------------------------------------------ QKNorm
def qk_ref(x, w, eps, pos, rot):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if rot is None:
        return x
    R, axis = rot["dim"], [a for a, n in enumerate(rot["sections"]) for _ in range(n)]
    if rot.get("freqs", "shared") == "shared":
        f = torch.tensor([rot.get("base", 10000.0) ** (-2 * i / R) for i in range(R // 2)], dtype=torch.float64)
    else:
        f = torch.tensor([rot.get("base", 10000.0) ** (-i / n) for n in rot["sections"] for i in range(n)], dtype=torch.float64)
    th = pos.double()[..., axis] * f
    c, s = torch.cos(th)[:, :, None], torch.sin(th)[:, :, None]
    y = x.clone()
    a, b = (slice(0, R // 2), slice(R // 2, R)) if rot["layout"] == "half" else (slice(0, R, 2), slice(1, R, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def qk_check(got, want, x, w, dtype, what):
    """Bound: 24 float roundings and 2^-21 of angle on the head's largest normed value, then the type's rounding."""
    big = want.abs().amax(-1, keepdim=True) * 1.5
    tol = (24 * 2.0 ** -24 + 2.0 ** -21) * big + U[dtype] * want.abs() + 1e-30
    bad = (got.double().cpu() - want).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {((got.double().cpu() - want).abs() / tol).max():.3g} x"


QK_CASES = [(64, dict(dim=64, sections=[32], layout="half")), (64, dict(dim=64, sections=[11, 11, 10], layout="pairs")),
            (128, dict(dim=128, sections=[16, 24, 24], layout="half")), (80, dict(dim=80, sections=[20, 20], layout="half")),
            (80, dict(dim=64, sections=[32], layout="pairs")), (72, dict(dim=32, sections=[4, 6, 6], layout="half")),
            (96, dict(dim=96, sections=[16, 16, 16], layout="half", freqs="axis")), (32, dict(dim=32, sections=[16], layout="pairs", base=500.0)),
            (8, dict(dim=8, sections=[4], layout="half")), (256, dict(dim=256, sections=[64, 64], layout="half")),
            (256, dict(dim=128, sections=[64], layout="pairs")), (40, dict(dim=20, sections=[10], layout="half")),
            (33, dict(dim=10, sections=[5], layout="pairs")), (1, None), (7, dict(dim=2, sections=[1], layout="half")), (128, None)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,rot", QK_CASES)
@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 1, 1, 1), (2, 37, 6, 2), (3, 5, 16, 16), (1, 700, 3, 1)])
def test_qk(dtype, D, rot, B, S, Hq, Hk):
    from vision_assist_amd.tokens import QKNorm, Rotary
    g = torch.Generator().manual_seed(D + S)
    t = DT[dtype]
    qkv = rnd(g, B, S, Hq + 2 * Hk, D, dtype=t)
    wq, wk = 1 + rnd(g, D, by=0.2), 1 + rnd(g, D, by=0.2)
    axes = len(rot["sections"]) if rot else 0
    pos = torch.randint(0, 5000, (B, S, max(axes, 1)), generator=g, dtype=torch.int32)
    pos[:, S // 2] *= 3000  # far positions
    r = Rotary(rot["dim"], rot["sections"], rot.get("base", 10000.0), rot["layout"], rot.get("freqs", "shared"), device="cuda") if rot else None
    for a, b in ((wq, wk), (wq, None), (None, None)):
        qk = QKNorm(D, r, a, b, eps=1e-5, device="cuda")
        dev = qkv.cuda()
        q, k = dev[:, :, :Hq], dev[:, :, Hq:Hq + Hk]
        p = pos.cuda() if rot else None
        qo, ko = qk(q, k, p)
        qk_check(qo, qk_ref(qkv[:, :, :Hq], a, 1e-5, pos, rot), qkv, a, t, "q")
        qk_check(ko, qk_ref(qkv[:, :, Hq:Hq + Hk], b, 1e-5, pos, rot), qkv, b, t, "k")
        rest = dev[:, :, Hq + Hk:].clone()
        qk(q, k, p, q_out=q, k_out=k)  # in place, inside the product's output
        assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(dev[:, :, Hq + Hk:], rest)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_qk_layouts(dtype):
    """Odd strides and offsets, heads before tokens, expanded positions, a zero vector, tiny and huge values."""
    from vision_assist_amd.tokens import QKNorm, Rotary
    g = torch.Generator().manual_seed(9)
    t, B, S, H, D = DT[dtype], 2, 19, 3, 64
    x = rnd(g, B, S, H, D, dtype=t)
    x[0, 0] = 0
    x[0, 1] *= 1e-18
    x[1, 2] *= 1e15
    w = 1 + rnd(g, D, by=0.1)
    qk = QKNorm(D, Rotary(64, device="cuda"), w, w, device="cuda")
    pos = torch.arange(S, dtype=torch.int32, device="cuda").expand(B, S)
    want_q, want_k = qk(x.cuda(), x.cuda(), pos)
    rot = dict(dim=64, sections=[32], layout="half")
    qk_check(want_q, qk_ref(x, w, 1e-6, pos.cpu()[..., None], rot), x, w, t, "layout")
    assert torch.equal(want_q, want_k) and (want_q[0, 0] == 0).all()
    for view in (x.transpose(1, 2).contiguous().cuda().transpose(1, 2), torch.nn.functional.pad(x, (1, 2)).cuda()[..., 1:1 + D],
                 x.permute(3, 0, 1, 2).contiguous().cuda().permute(1, 2, 3, 0)):
        buf = torch.full((B, S, H, D + 3), 2.0, dtype=t, device="cuda")
        o = buf[..., 3:]
        a, b = qk(view, view, pos[..., None], q_out=o)
        assert a is o and torch.equal(o, want_q) and torch.equal(b, want_k) and (buf[..., :3] == 2).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,S,H,D,slots,sinks", [(1, 1, 1, 64, 8, 2), (3, 1, 4, 128, 40, 4), (2, 30, 2, 80, 17, 3), (4, 9, 2, 33, 9, 0),
                                                 (2, 64, 3, 32, 64, 0), (1, 5, 2, 64, 2, 1)])
def test_qk_store_rings(dtype, B, S, H, D, slots, sinks):
    """Several calls into one cache: the kept tokens are the sinks and the newest ones, rows behind q_len stay."""
    from vision_assist_amd.tokens import QKNorm, Rotary, TokenCache
    g = torch.Generator().manual_seed(slots)
    t = DT[dtype]
    w = 1 + rnd(g, D, by=0.1)
    rd = D // 2 * 2
    qk = QKNorm(D, Rotary(rd, layout="pairs", device="cuda"), w, w, device="cuda")
    cache = TokenCache(B, slots, H, D, sinks=sinks, dtype=dtype, device="cuda")
    want_k, want_v, seen = cache.k.cpu().clone(), cache.v.cpu().clone(), [0] * B
    for step in range(4):
        q, k, v = (rnd(g, B, S, H, D, dtype=t) for _ in range(3))
        ql = [min(S, (b * 2 + step * 3) % (S + 1)) for b in range(B)]
        q_len = torch.tensor(ql, dtype=torch.int32, device="cuda")
        cache.advance(q_len)
        pos = torch.stack([torch.arange(S) + seen[b] for b in range(B)]).to(torch.int32).cuda()
        out = torch.full((B, S, H, D), 9.0, dtype=t, device="cuda")
        qk.store(q.cuda(), k.cuda(), v.cuda(), pos, cache, q_len=q_len, q_out=out)
        full_q, full_k = qk(q.cuda(), k.cuda(), pos)
        full_k = full_k.cpu()
        for b in range(B):
            assert torch.equal(out[b, :ql[b]], full_q[b, :ql[b]]) and (out[b, ql[b]:] == 9).all()
            for s in range(ql[b]):
                p = seen[b] + s
                slot = p if p < sinks else sinks + (p - sinks) % (slots - sinks)
                want_k[b, slot], want_v[b, slot] = full_k[b, s], v[b, s]
            seen[b] += ql[b]
        assert cache.len.tolist() == seen
        assert torch.equal(cache.k.cpu(), want_k) and torch.equal(cache.v.cpu(), want_v), step


# ------------------------------------------------------------------ attend
def visible(S, slots, frame, window, sinks, ql, kv):
    """bool [S, slots]: what each query sees of each slot; and the slots' positions."""
    see, at = torch.zeros(S, slots, dtype=torch.bool), [-1] * slots
    for p in range(max(kv, 0)):
        at[p if p < sinks or p < slots else sinks + (p - sinks) % (slots - sinks)] = p
    at = torch.tensor(at)
    for s in range(ql):
        i = kv - ql + s
        if i < 0:
            continue
        e = (i // frame + 1) * frame if frame else 1 << 40
        see[s] = (at >= 0) & (at < min(e, kv)) & ((at < sinks) | (at >= (e - window if window else 0)))
    return see


def attend_ref(q, k, v, scale, frame, window, sinks, q_len, kv_len):
    """-> (value, bound) in float64, rows behind q_len NaN."""
    B, S, Hq, D = q.shape
    slots, Hk, Dv = k.shape[1], k.shape[2], v.shape[3]
    out = torch.full((B, S, Hq, Dv), math.nan, dtype=torch.float64)
    tol = torch.zeros_like(out)
    up = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -24
    for b in range(B):
        see = visible(S, slots, frame, window, sinks, q_len[b], kv_len[b])[:q_len[b]]
        for h in range(Hq):
            kk, vv = k[b, :, h // (Hq // Hk)].double(), v[b, :, h // (Hq // Hk)].double()
            qq = q[b, :q_len[b], h].double()
            any_seen = see.any(0)
            kk, vv = kk[any_seen], vv[any_seen]
            m = see[:, any_seen]
            a = scale * (qq @ kk.t())
            mag = scale * (qq.abs() @ kk.abs().t())
            a = a.masked_fill(~m, -math.inf)
            top = a.amax(-1, keepdim=True) if a.shape[1] else torch.zeros(a.shape[0], 1, dtype=torch.float64)
            e = torch.exp(a - top.clamp(min=-1e300))
            tot = e.sum(-1, keepdim=True)
            p = torch.where(m, e / torch.where(tot > 0, tot, 1.0), 0.0)
            out[b, :q_len[b], h] = p @ vv
            # a score's error, its maximum's, exp2's argument and result, and the sums over the keys
            ds = ((D + 4) * 2.0 ** -24 * mag + 2.0 ** -22 * a.masked_fill(~m, 0).abs()).masked_fill(~m, 0)
            dm = ds.amax(-1, keepdim=True) if ds.shape[1] else 0
            rel = torch.expm1(2 * (ds + dm)) + 2.0 ** -21 + up
            tol[b, :q_len[b], h] = (p * rel) @ vv.abs() + (see.shape[1] * 2.0 ** -24) * (p @ vv.abs()) + \
                (p * rel).sum(-1, keepdim=True) * (p @ vv.abs())
    return out, tol


def run_attend(dtype, B, S, Hq, Hk, D, Dv, slots, frame=1, window=0, sinks=0, q_len=None, kv_len=None, seed=0, scale=None, spread=1.0):
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(seed)
    t = DT[dtype]
    q, k, v = rnd(g, B, S, Hq, D, dtype=t, by=spread), rnd(g, B, slots, Hk, D, dtype=t), rnd(g, B, slots, Hk, Dv, dtype=t)
    ql, kl = q_len or [S] * B, kv_len or [slots] * B
    dev = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")
    out = torch.full((B, S, Hq, Dv), 3.0, dtype=t, device="cuda")
    got = attend(q.cuda(), k.cuda(), v.cuda(), scale=scale, frame=frame, window=window, sinks=sinks, q_len=dev(q_len),
                 kv_len=dev(kv_len), out=out)
    want, tol = attend_ref(q, k, v, D ** -0.5 if scale is None else scale, frame, window, sinks, ql, kl)
    got = got.double().cpu()
    for b in range(B):
        assert (got[b, ql[b]:] == 3).all(), "rows behind the sequence were written"
    m = ~want.isnan()
    tol = tol + U[t] * want.abs() + 1e-30
    bad = (got[m] - want[m]).abs() > tol[m]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got[m] - want[m]).abs() / tol[m]).max():.3g} x"


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (32, 64), (80, 80), (72, 72), (8, 8), (96, 96), (128, 32), (104, 120)])
@pytest.mark.parametrize("S,slots,frame,window,sinks", [(1, 1, 1, 0, 0), (1, 300, 1, 0, 0), (70, 70, 1, 0, 0), (130, 130, 0, 0, 0),
                                                        (65, 200, 1, 33, 3), (96, 96, 24, 48, 7), (40, 129, 10, 20, 0)])
def test_attend(dtype, D, Dv, S, slots, frame, window, sinks):
    run_attend(dtype, 2, S, 4, 2, D, Dv, slots, frame, window, sinks, seed=D + S)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 1), (6, 2), (12, 12), (40, 8), (33, 1), (64, 2)])
@pytest.mark.parametrize("S", [1, 3, 50])
def test_attend_heads(dtype, Hq, Hk, S):
    run_attend(dtype, 2, S, Hq, Hk, 64, 64, 160, window=100, sinks=5, seed=Hq + S)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_ragged_and_empty_rows(dtype):
    """Lengths of zero and one, more queries than positions, a window of one, kv 0, sinks longer than a sequence."""
    run_attend(dtype, 6, 20, 4, 2, 64, 64, 90, window=16, sinks=4, q_len=[20, 0, 1, 20, 7, 20], kv_len=[90, 50, 1, 6, 64, 0])
    run_attend(dtype, 3, 5, 2, 2, 32, 32, 40, window=1, sinks=0, q_len=[5, 5, 2], kv_len=[40, 5, 2])
    run_attend(dtype, 3, 33, 2, 1, 64, 64, 70, frame=8, window=8, sinks=30, q_len=[33, 33, 10], kv_len=[70, 33, 10])
    run_attend(dtype, 2, 6, 2, 1, 64, 64, 6, frame=0, q_len=[6, 3], kv_len=[6, 4])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S", [1, 4, 50, 160])
@pytest.mark.parametrize("slots,sinks,window,frame", [(300, 4, 130, 1), (260, 0, 100, 1), (333, 50, 100, 25), (211, 1, 50, 7)])
def test_attend_rings(dtype, S, slots, sinks, window, frame):
    run_attend(dtype, 3, S, 4, 2, 64, 64, slots, frame, window, sinks, q_len=[S, S, max(1, S - 3)], kv_len=[slots + 1, 3 * slots + 17, 5000],
               seed=slots)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_small_rings(dtype):
    """Rings shorter than a tile, wrapped many times."""
    for slots, sinks, window in ((3, 2, 1), (9, 1, 4), (20, 0, 20), (40, 8, 30)):
        run_attend(dtype, 2, 1, 4, 1, 64, 64, slots, 1, window, sinks, kv_len=[1000, slots], seed=slots)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,slots", [(1, 5000), (2, 3001), (7, 900)])
def test_attend_long_steps(dtype, B, slots):
    """Single tokens over long caches (the work of a row is split over the keys)."""
    run_attend(dtype, B, 1, 8, 2, 128, 128, slots, kv_len=[slots - 13 * b for b in range(B)], seed=slots)
    run_attend(dtype, B, 2, 8, 2, 64, 64, slots, window=slots // 2, sinks=9, kv_len=[slots + 333 * b for b in range(B)], seed=slots)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_large_scores(dtype):
    """Scores of some hundreds: the running maximum moves by far more than the sums can hold."""
    run_attend(dtype, 1, 90, 2, 2, 64, 64, 400, window=300, sinks=2, spread=30.0, seed=1)
    run_attend(dtype, 2, 1, 4, 1, 64, 64, 3000, spread=30.0, seed=2)
    run_attend(dtype, 1, 40, 1, 1, 64, 64, 40, scale=2.0, seed=3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("S,frame,window,sinks", [(1, 1, 20, 3), (70, 1, 20, 3), (70, 14, 28, 3), (3, 1, 40, 0)])
def test_attend_what_is_not_seen_has_no_part(dtype, bad, S, frame, window, sinks):
    """Non-finite keys and values at positions: behind the sequence, in unused slots, and at places that some rows see."""
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(8)
    t, B, slots, H, D = DT[dtype], 2, 150, 2, 64
    q, k, v = rnd(g, B, S, 2 * H, D, dtype=t), rnd(g, B, slots, H, D, dtype=t), rnd(g, B, slots, H, D, dtype=t)
    kl = [110, 150]
    kv = torch.tensor(kl, dtype=torch.int32, device="cuda")
    call = lambda k, v: attend(q.cuda(), k.cuda(), v.cuda(), frame=frame, window=window, sinks=sinks, kv_len=kv).cpu()
    clean = call(k, v)
    assert clean.isfinite().all()
    k2, v2 = k.clone(), v.clone()
    k2[0, 110:], v2[0, 110:] = bad, bad  # slots that hold nothing
    assert torch.equal(call(k2, v2), clean)
    for place in (2, 60, 95, 109):
        k2, v2 = k.clone(), v.clone()
        v2[0, place, 1, 5] = bad
        k2[1, place, 0, 7] = bad
        got = call(k2, v2)
        for b in range(B):
            see = visible(S, slots, frame, window, sinks, S, kl[b])[:, place]
            assert torch.equal(got[b, ~see], clean[b, ~see])
            if b == 0:  # only column 5 of the heads over key head 1
                rest = [d for d in range(D) if d != 5]
                assert torch.equal(got[b][:, :H], clean[b][:, :H]) and torch.equal(got[b][..., rest], clean[b][..., rest])
                assert not got[b, see][:, H:, 5].isfinite().any()
            else:
                assert torch.equal(got[b][:, H:], clean[b][:, H:])
                if math.isnan(bad):
                    assert got[b, see][:, :H].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_strides(dtype):
    """Views of one product's output, heads before tokens, odd offsets, an out inside a wider buffer."""
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(6)
    t, B, S, H, D = DT[dtype], 2, 50, 3, 64
    qkv = rnd(g, B, S, 3 * H, D, dtype=t).cuda()
    q, k, v = qkv[:, :, :H], qkv[:, :, H:2 * H], qkv[:, :, 2 * H:]
    want = attend(q.contiguous(), k.contiguous(), v.contiguous(), window=20, sinks=1)
    assert torch.equal(attend(q, k, v, window=20, sinks=1), want)
    hs = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(attend(*hs, window=20, sinks=1), want)
    odd = [torch.nn.functional.pad(x, (1, 2))[..., 1:1 + D] for x in (q, k, v)]
    for width, off in ((D + 3, 1), (D + 8, 8)):
        buf = torch.full((B, S, H, width), 4.0, dtype=t, device="cuda")
        o = buf[..., off:off + D]
        assert attend(*odd, window=20, sinks=1, out=o) is o
        assert torch.equal(o, want) and (buf[..., :off] == 4).all() and (buf[..., off + D:] == 4).all()
    one = rnd(g, 1, S, 1, D, dtype=t).cuda()
    ex = one.expand(B, S, H, D)
    assert torch.equal(attend(q, ex, ex), attend(q, ex.contiguous(), ex.contiguous()))


def test_attend_same_bits_every_time():
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(2)
    q, k, v = rnd(g, 3, 1, 8, 128, dtype=torch.bfloat16).cuda(), *(rnd(g, 3, 4000, 2, 128, dtype=torch.bfloat16).cuda() for _ in range(2))
    first = attend(q, k, v)
    for _ in range(5):
        assert torch.equal(attend(q, k, v), first)
    for b in range(3):  # a sequence does not depend on its batch
        assert (attend(q[b:b + 1], k[b:b + 1], v[b:b + 1]).float() - first[b:b + 1].float()).abs().max() <= 2.0 ** -7


# ------------------------------------------------------------------ together, as a stream uses them
class Layer:
    """One attention layer over a stream: product, norms and rotation into the cache, attention, product + residual."""

    def __init__(self, dtype, C=256, Hq=4, Hk=2, D=64, frame=25, window=50, sinks=25, seed=0):
        from vision_assist_amd.tokens import Linear, QKNorm, Rotary
        g = torch.Generator().manual_seed(seed)
        self.t = DT[dtype]
        self.p = dict(C=C, Hq=Hq, Hk=Hk, D=D, frame=frame, window=window, sinks=sinks)
        self.wi, self.bi = rnd(g, (Hq + 2 * Hk) * D, C, by=C ** -0.5), rnd(g, (Hq + 2 * Hk) * D, by=0.1)
        self.wo = rnd(g, C, Hq * D, by=(Hq * D) ** -0.5)
        self.nq, self.nk = 1 + rnd(g, D, by=0.1), 1 + rnd(g, D, by=0.1)
        self.inp = Linear(self.wi, self.bi, dtype=dtype, device="cuda")
        self.outp = Linear(self.wo, dtype=dtype, device="cuda")
        self.norm = QKNorm(D, Rotary(D, [D // 4, D // 8, D // 8], device="cuda"), self.nq, self.nk, device="cuda")

    def pos(self, n, first):
        i = torch.arange(first, first + n)
        f = self.p["frame"]
        return torch.stack([i // f, i % f // 5, i % 5], -1).to(torch.int32)

    def step(self, x, cache, pos, q_len=None):
        B, S, _ = x.shape
        h = self.inp(x).view(B, S, -1, self.p["D"])
        Hq, Hk = self.p["Hq"], self.p["Hk"]
        cache.advance(S if q_len is None else q_len)
        q = self.norm.store(h[:, :, :Hq], h[:, :, Hq:Hq + Hk], h[:, :, Hq + Hk:], pos, cache, q_len=q_len)
        from vision_assist_amd.tokens import attend
        o = attend(q, cache.k, cache.v, frame=self.p["frame"], window=self.p["window"], sinks=self.p["sinks"], q_len=q_len,
                   kv_len=cache.len)
        return self.outp(o.view(B, S, -1), residual=x)

    def ref(self, x):
        """The whole sequence [N, C] at once in float64."""
        p, t = self.p, (lambda y: y.to(self.t).double())
        w = (lambda y: y.to(self.t).double()) if self.t == torch.bfloat16 else (lambda y: y.double())
        h = (x.double() @ w(self.wi).t() + self.bi.double()).view(1, len(x), -1, p["D"])
        rot = dict(dim=p["D"], sections=[p["D"] // 4, p["D"] // 8, p["D"] // 8], layout="half")
        pos = self.pos(len(x), 0)[None]
        q, k = qk_ref(h[:, :, :p["Hq"]], self.nq, 1e-6, pos, rot), qk_ref(h[:, :, p["Hq"]:p["Hq"] + p["Hk"]], self.nk, 1e-6, pos, rot)
        o, _ = attend_ref(q, k, h[:, :, p["Hq"] + p["Hk"]:], p["D"] ** -0.5, p["frame"], p["window"], p["sinks"], [len(x)], [len(x)])
        return x.double() + o.reshape(len(x), -1) @ w(self.wo).t()


@pytest.mark.parametrize("dtype,tol", [("f32", 2e-5), ("bf16", 0.04)])
def test_layer_streams_frame_by_frame(dtype, tol):
    """Twelve frames of 25 tokens, one call a frame over a ring that holds the first frame, the window and the new one,
    equal the whole sequence at once.  bf16: h, q, k, o, y are rounded between the operators (five roundings of 2^-8 of
    values of size 1 to 4, averaged by the sums they enter)."""
    from vision_assist_amd.tokens import TokenCache
    L = Layer(dtype)
    p, n = L.p, 12
    g = torch.Generator().manual_seed(1)
    x = rnd(g, 2, n * 25, p["C"], dtype=L.t)
    cache = TokenCache(2, p["sinks"] + p["window"] + 25, p["Hk"], p["D"], sinks=p["sinks"], dtype=dtype, device="cuda")
    got = torch.cat([L.step(x[:, 25 * f:25 * f + 25].cuda(), cache, L.pos(25, 25 * f).cuda().expand(2, 25, 3)) for f in range(n)], 1)
    assert cache.len.tolist() == [n * 25] * 2
    for b in range(2):
        err = (got[b].double().cpu() - L.ref(x[b])).abs().max()
        assert err <= tol, err


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_captured_and_replayed(dtype):
    """A step captured into a graph: several replays with eager work between them, each against the eager layer."""
    from vision_assist_amd.tokens import TokenCache
    L = Layer(dtype, frame=1, window=60, sinks=4)
    p = L.p
    g = torch.Generator().manual_seed(2)
    xs = rnd(g, 30, 3, 1, p["C"], dtype=L.t).cuda()
    make = lambda: TokenCache(3, 64, p["Hk"], p["D"], sinks=4, dtype=dtype, device="cuda")
    eager, cache = make(), make()
    want = [L.step(xs[i], eager, torch.full((3, 1, 3), i, dtype=torch.int32, device="cuda")) for i in range(30)]
    x, pos = xs[0].clone(), torch.zeros(3, 1, 3, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        L.step(x, make(), pos)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = L.step(x, cache, pos)
    for i in range(30):
        x.copy_(xs[i])
        pos.fill_(i)
        graph.replay()
        assert torch.equal(y, want[i]), i
        if i % 7 == 3:
            L.step(xs[i], make(), pos)
            torch.cuda.synchronize()
    assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)


def test_layer_as_ops_of_a_list():
    """VA_OP_TOK_*: the layer's launches as one op list, on lanes too."""
    import ctypes

    from vision_assist_amd.seg import ConvArgs, SegOp
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(3)
    a, b = (Linear(rnd(g, 96, 96, by=0.1), act="gelu", device="cuda") for _ in range(2))
    x = rnd(g, 40, 96, dtype=torch.bfloat16).cuda()
    y, z = torch.empty_like(x), torch.empty_like(x)
    args = [a.args(x, y), b.args(y, z, residual=x)]
    ops = (SegOp * 3)(SegOp(kind=8, a=ConvArgs(N=1)), *(SegOp(kind=10, lane=1, a=ConvArgs(x=ctypes.addressof(t))) for t in args))
    _lib.check(_lib.load().va_seg_run(_lib.stream_ptr(), ops, 3), "va_seg_run")
    torch.cuda.synchronize()
    assert torch.equal(z, b(a(x), residual=x))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_calls_on_another_stream_and_two_at_once(dtype):
    """Work on a stream of the caller's, beside the same operators on the current one, gives what the current one gives."""
    from vision_assist_amd.tokens import Linear, QKNorm, Rotary, attend
    g = torch.Generator().manual_seed(4)
    t = DT[dtype]
    lin = Linear(rnd(g, 512, 512, by=0.05), act="silu", dtype=dtype, device="cuda")
    norm = QKNorm(64, Rotary(64, device="cuda"), torch.ones(64), torch.ones(64), device="cuda")
    xs = [rnd(g, 4, 200, 512, dtype=t).cuda() for _ in range(2)]
    pos = torch.arange(200, dtype=torch.int32, device="cuda").expand(4, 200)

    def go(x, stream=None):
        h = lin(x, stream=stream).view(4, 200, 8, 64)
        q, k = norm(h[:, :, :4], h[:, :, 4:6], pos, stream=stream)
        return attend(q, k, h[:, :, 6:], window=50, sinks=2, stream=stream), attend(q[:, -1:], k, h[:, :, 6:], stream=stream)

    want = [[y.clone() for y in go(x)] for x in xs]
    side = [torch.cuda.Stream() for _ in range(2)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = [go(x, s) for x, s in zip(xs, side)]
        here = go(xs[0])
        torch.cuda.synchronize()
        for a, b in zip(got + [here], want + [want[0]]):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------ far ends of the counts
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,frame,window", [(1, 1, 0), (1, 1, 90), (3, 1, 90), (160, 1, 90), (160, 32, 64)])
@pytest.mark.parametrize("slots,sinks", [(300, 4), (333, 0), (352, 32)])
def test_attend_positions_up_to_the_last_one(dtype, S, frame, window, slots, sinks):
    """A ring's result depends on positions by their differences: lengths a whole number of rings (and frames) apart agree."""
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(S + slots)
    t = DT[dtype]
    q, k, v = (rnd(g, *s, dtype=t).cuda() for s in ((2, S, 4, 64), (2, slots, 2, 64), (2, slots, 2, 64)))
    turn = math.lcm(slots - sinks, frame)
    far = [2 ** 31 - 1, 2 ** 31 - 60]
    near = [n - (n - 4 * slots) // turn * turn for n in far]
    out = [attend(q, k, v, frame=frame, window=window, sinks=sinks, kv_len=torch.tensor(n, dtype=torch.int32, device="cuda"))
           for n in (far, near)]
    assert torch.equal(*out)


def test_qk_lengths_behind_the_call_are_the_calls():
    """q_len[b] > S counts as S, as it does for attention: the tokens stand at the last S positions."""
    from vision_assist_amd.tokens import QKNorm, TokenCache
    g = torch.Generator().manual_seed(3)
    q, k, v = (rnd(g, 2, 5, 2, 32, dtype=torch.float32).cuda() for _ in range(3))
    caches = []
    for n in ([5, 3], [9, 3]):
        c = TokenCache(2, 16, 2, 32, dtype="f32").advance(5)
        QKNorm(32).store(q, k, v, None, c, q_len=torch.tensor(n, dtype=torch.int32, device="cuda"))
        caches.append(c)
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


@pytest.mark.parametrize("M,K", [(1, 64), (65, 64), (3, 60)])
def test_linear_offsets_behind_31_bits(M, K):
    """Channels from 2^26 on: offsets of their packed rows pass 2^31.  Weights of 1 in one column each: copies of x."""
    from vision_assist_amd.tokens import Linear
    N = (1 << 26) + 32
    lin = Linear.__new__(Linear)
    from vision_assist_amd import _lib
    lin.lib, lin.device, lin.N, lin.K, lin.dtype, lin.tdtype = _lib.load(), torch.device("cuda", 0), N, K, "bf16", torch.bfloat16
    w = torch.zeros(2, (N + 63) // 64 * 2, 32, 32, dtype=torch.bfloat16, device="cuda")
    at = [0, 31, (1 << 25) - 1, 1 << 25, (1 << 25) + 77, (1 << 26) - 1, 1 << 26, N - 1]
    for i, n in enumerate(at):  # w[n][i] = 1: row n % 32's place, its first eight columns' piece
        r = next(r for r in range(32) if 16 * (r // 4 % 2) + 4 * (r // 8) + r % 4 == n % 32)
        w[0, n // 32, r, 8 * (0 ^ (r // 4 % 4)) + i] = 1
    lin._w, lin._wscale, lin._bias = w, None, None
    lin._ptrs, lin._ints = (w.data_ptr(), 0, 0), (N, K, w.shape[1] * 32, 64, 1, 0, 0)
    x = torch.randn(M, K, device="cuda").to(torch.bfloat16)
    y = lin(x)
    for i, n in enumerate(at):
        assert torch.equal(y[:, n], x[:, i]), f"channel {n}"
    y[:, at] = 0
    assert not y.any()


@pytest.mark.parametrize("S", [1, 5, 300])
def test_attend_keys_that_sequences_share(S):
    """Keys and values expanded over the sequences (stride 0) are those of copies."""
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(S)
    q, k, v = (rnd(g, *s, dtype=torch.bfloat16).cuda() for s in ((3, S, 4, 64), (1, 700, 2, 64), (1, 700, 2, 64)))
    shared = attend(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1))
    assert torch.equal(shared, attend(q, k.repeat(3, 1, 1, 1), v.repeat(3, 1, 1, 1)))
