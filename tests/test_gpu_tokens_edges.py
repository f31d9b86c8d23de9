"""Edges of the token operators: what enters a product as it is, values that are not finite, far ends of a stream's
life, and each form that a product's size chooses.  Plain implementations in float64; tolerances as in test_gpu_tokens.py
(half a step of a rounding relative to the value: bf16 2^-8, float 2^-24), with what is added derived beside each test."""
import math

import pytest
import torch

from tests.test_gpu_tokens import DT, U, attend_ref, rnd

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ attend
@pytest.mark.parametrize("B,S,Hq,Hk,D,slots,kv", [(3, 1, 8, 2, 128, 2500, 2500), (2, 2, 4, 4, 64, 700, 1900), (1, 4, 8, 1, 80, 333, 333),
                                                  (5, 1, 32, 1, 32, 60, 60)])
def test_attend_few_rows_round_once(B, S, Hq, Hk, D, slots, kv):
    """bf16, up to 32 rows of a key head: the probabilities enter the second product as two bf16 terms, each within 2^-8 of
    what it stands for, so 2^-16 of a probability is left out; the rest is the float form's bound and the output's rounding."""
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(slots)
    t = torch.bfloat16
    q, k, v = rnd(g, B, S, Hq, D, dtype=t), rnd(g, B, slots, Hk, D, dtype=t), rnd(g, B, slots, Hk, D, dtype=t)
    kl = [kv - 7 * b for b in range(B)]
    got = attend(q.cuda(), k.cuda(), v.cuda(), kv_len=torch.tensor(kl, dtype=torch.int32, device="cuda")).double().cpu()
    args = (D ** -0.5, 1, 0, 0, [S] * B, kl)
    want, tol = attend_ref(q.float(), k, v, *args)
    size, _ = attend_ref(q.float(), k, v.abs(), *args)
    tol = tol + 2.0 ** -16 * size + U[t] * want.abs()
    assert float(((got - want).abs() / tol).max()) <= 1


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,Hk,slots,frame,window,sinks,kv", [(1, 2, 3000, 1, 0, 0, 3000), (1, 1, 500, 1, 200, 5, 1900), (5, 2, 200, 1, 0, 0, 200),
                                                              (200, 2, 200, 1, 0, 0, 200), (260, 1, 260, 20, 80, 9, 260),
                                                              (70, 2, 400, 1, 250, 3, 1111), (150, 1, 150, 0, 0, 0, 150)])
def test_attend_infinite_values_whatever_their_probability(dtype, S, Hk, slots, frame, window, sinks, kv):
    """Scores of some hundreds, so that most probabilities come out 0: a seen infinity is an infinity all the same, NaN and
    both infinities are NaN, wherever tiles begin; other columns and rows are those of the call without them, bit by bit."""
    from tests.test_gpu_tokens import visible
    from vision_assist_amd.tokens import attend
    g = torch.Generator().manual_seed(S)
    t, B, D = DT[dtype], 2, 64
    q, k, v = rnd(g, B, S, 2 * Hk, D, dtype=t, by=60.0), rnd(g, B, slots, Hk, D, dtype=t), rnd(g, B, slots, Hk, D, dtype=t)
    lens = torch.tensor([kv, kv - 9], dtype=torch.int32, device="cuda")
    call = lambda v: attend(q.cuda(), k.cuda(), v.cuda(), frame=frame, window=window, sinks=sinks, kv_len=lens).cpu().double()
    clean = call(v)
    spots = torch.randperm(slots, generator=g)[:8].tolist()
    put = [(3, math.inf, spots[0]), (4, -math.inf, spots[1]), (5, math.inf, spots[2]), (5, -math.inf, spots[3]), (6, math.nan, spots[4]),
           (40, math.inf, spots[5]), (63, -math.inf, spots[6]), (63, -math.inf, spots[7])]
    bad = v.clone()
    for col, x, slot in put:
        bad[:, slot, :, col] = x
    want = clean.clone()
    for b, n in enumerate(lens.tolist()):
        see = visible(S, slots, frame, window, sinks, S, n)
        for col in {c for c, _, _ in put}:
            hit = [torch.zeros(S, dtype=torch.bool) for _ in range(2)]
            for c, x, slot in put:
                if c == col:
                    for i, sign in enumerate((1, -1)):
                        if math.isnan(x) or x * sign > 0:
                            hit[i] |= see[:, slot]
            for rows, x in ((hit[0] & ~hit[1], math.inf), (hit[1] & ~hit[0], -math.inf), (hit[0] & hit[1], math.nan)):
                want[b, rows, :, col] = x
    got = call(bad)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.5, math.inf, -math.inf), want.nan_to_num(0.5, math.inf, -math.inf))
    assert not want.isfinite().all()


# ------------------------------------------------------------------ Linear
# the float forms: rows few enough to split K over waves, unaligned rows, tiles with K halved between two groups, tiles
F32_FORMS = [(1, 200, 96), (40, 264, 160), (70, 131, 130), (1300, 264, 576), (2112, 136, 1024)]


@pytest.mark.parametrize("M,K,N", F32_FORMS)
def test_linear_f32_infinities_and_the_largest_values(M, K, N):
    """What the definition gives: an infinity's row is infinities of the weights' signs (NaN at a weight of 0), and values
    beyond bf16's largest are values like others.  Those rows' bound is that of test_gpu_tokens.py: (K + 8) 2^-24 sum |x w|."""
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(M)
    big = torch.finfo(torch.float32).max
    w = rnd(g, N, K, by=K ** -0.5)
    w[3, K - 1] = 0.0
    lin = Linear(w, dtype="f32", device="cuda")
    x = rnd(g, M, K)
    clean = lin(x.cuda()).cpu()
    plus, minus, both, large, nan = (i * M // 5 for i in range(5)) if M > 4 else (0,) * 5

    def row(at, i, value):
        y = x.clone()
        for j, v in zip(i, value):
            y[at, j] = v
        got = lin(y.cuda()).cpu()
        rest = torch.arange(M) != at
        assert torch.equal(got[rest], clean[rest])
        return got[at].double()

    s = torch.sign(w[:, K - 1].double())
    want = torch.where(s == 0, math.nan, s * math.inf)
    assert torch.equal(row(plus, [K - 1], [math.inf]).nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(row(minus, [K - 1], [-math.inf]).nan_to_num(7.0), (-want).nan_to_num(7.0))
    s0 = torch.sign(w[:, 0].double())
    two = torch.where((s == s0) & (s != 0), s * math.inf, math.nan)
    assert torch.equal(row(both, [0, K - 1], [math.inf, math.inf]).nan_to_num(7.0), two.nan_to_num(7.0))
    assert row(nan, [K // 2], [math.nan]).isnan().all()
    got = row(large, [K - 1], [big])
    y = x.double()[large].clone()
    y[K - 1] = big
    cols = w[:, K - 1].abs() <= 0.2  # (sums that stay within the range)
    mag = y.abs() @ w.double().abs().t()
    ref = y @ w.double().t()
    tol = (K + 8) * 2.0 ** -24 * mag + 2.0 ** -24 * ref.abs()
    assert cols.any() and bool(((got - ref).abs() <= tol)[cols].all())


@pytest.mark.parametrize("M,K,N", F32_FORMS)
def test_linear_f32_infinite_weights(M, K, N):
    from vision_assist_amd.tokens import Linear
    g = torch.Generator().manual_seed(N)
    w = rnd(g, N, K)
    w[5, 2], w[9, K - 1] = math.inf, -math.inf
    x = rnd(g, M, K)
    x[0, 2], x[M // 2, K - 1] = 0.0, math.inf
    got = Linear(w, dtype="f32", device="cuda")(x.cuda()).double().cpu()
    ref = x.double() @ w.double().t()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.isinf(), ref.isinf())
    assert torch.equal(got[got.isinf()], ref[ref.isinf()])


def test_layers_refuse_to_lose_a_gradient():
    from vision_assist_amd import _lib
    from vision_assist_amd.tokens import Linear, QKNorm, TokenCache
    lin, norm = Linear(torch.nn.Parameter(torch.randn(64, 64)), device="cuda"), QKNorm(64, device="cuda")
    t = lambda grad: torch.randn(2, 3, 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=grad)
    cache = TokenCache(2, 8, 4, 64).advance(3)
    x, y = t(True), t(False)
    calls = [lambda: lin(x), lambda: lin(y, residual=x), lambda: norm(x, y), lambda: norm(y, x), lambda: norm.store(x, y, y, None, cache),
             lambda: norm.store(y, x, y, None, cache), lambda: norm.store(y, y, x, None, cache)]
    for call in calls:
        with pytest.raises(_lib.VaError, match="gradient"):
            call()
        with torch.no_grad():
            call()
    assert not lin(y).requires_grad


# ------------------------------------------------------------------ a stream without an end
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,slots,sinks,frame,window", [(1, 90, 4, 1, 80), (20, 120, 20, 20, 60), (3, 64, 0, 1, 0)])
def test_a_stream_goes_on_past_32_bits(dtype, S, slots, sinks, frame, window):
    """Steps across position 2^31 of a stream that is rebased are those of a young one whose count is whole rings and
    frames apart: eager, and by one captured graph."""
    from vision_assist_amd.tokens import QKNorm, Rotary, TokenCache, attend
    g = torch.Generator().manual_seed(S)
    t, B, H, D = DT[dtype], 2, 2, 64
    norm = QKNorm(D, Rotary(D, device="cuda"), torch.ones(D), torch.ones(D), device="cuda")
    turn = math.lcm(slots - sinks, frame)
    near = (4 * slots // frame + 1) * frame
    far = near + (2 ** 31 - 1 - 4 * S - near) // turn * turn
    k0, v0 = (rnd(g, B, slots, H, D, dtype=t).cuda() for _ in range(2))
    steps = max(12, 2 * turn // S + 8) if turn < 400 else 40
    xs = rnd(g, steps, 3, B, S, H, D, dtype=t).cuda()

    def cache(n):
        return TokenCache.of(k0.clone(), v0.clone(), sinks=sinks, length=torch.full((B,), n, dtype=torch.int32, device="cuda"))

    def step(c, x, pos, rebase):
        if rebase:
            c.rebase(frame)
        c.advance(S)
        q = norm.store(x[0], x[1], x[2], pos, c)
        return attend(q, c.k, c.v, frame=frame, window=window, sinks=sinks, kv_len=c.len)

    young, old, replayed = cache(near), cache(far), cache(far)
    pos = torch.zeros(B, S, dtype=torch.int32, device="cuda")
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache(far), x, pos, True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(replayed, x, pos, True)
    for i in range(steps):
        pos.copy_((torch.arange(S) + i * S).expand(B, S))
        x.copy_(xs[i])
        want = step(young, xs[i], pos, False)
        assert torch.equal(step(old, xs[i], pos, True), want), i
        graph.replay()
        assert torch.equal(y, want), i
    assert int(old.len.max()) < 2 ** 31 - 1 and far + steps * S > 2 ** 31
    assert torch.equal(old.k, young.k) and torch.equal(replayed.v, young.v) and torch.equal(old.len, replayed.len)


# ------------------------------------------------------------------ QKNorm
@pytest.mark.parametrize("S,D", [(3000, 64), (1, 64), (500, 66)])
def test_angles_keep_floats_accuracy(S, D):
    """Pairs (1, 0) without a norm: the result is the cosine and the sine.  Half steps relative to them: two for each of
    the sine's or cosine's evaluation (two units in the last place), one of the sum; and the angle's float64 roundings, two
    here (frequency and product) and two in the reference: 4 x 2^-53 of it."""
    from vision_assist_amd.tokens import QKNorm, Rotary
    g = torch.Generator().manual_seed(D)
    n = D // 2
    x = torch.zeros(1, S, 1, D)
    x[..., 0::2] = 1.0
    pos = torch.randint(0, 1 << 20, (1, S), generator=g, dtype=torch.int32)
    q, _ = QKNorm(D, Rotary(D, layout="pairs", device="cuda"), device="cuda")(x.cuda(), x.cuda(), pos.cuda())
    th = pos.double()[0, :, None] * torch.tensor([10000.0 ** (-2 * i / D) for i in range(n)], dtype=torch.float64)
    got = q[0, :, 0].double().cpu()
    for part, want in ((got[:, 0::2], torch.cos(th)), (got[:, 1::2], torch.sin(th))):
        tol = 5 * 2.0 ** -24 * want.abs() + 4 * 2.0 ** -53 * th
        assert float(((part - want).abs() / (tol + 1e-300)).max()) <= 1


@pytest.mark.parametrize("K", [1, 8])
def test_gelu_keeps_its_left_tail(K):
    """bf16: every value from -12 to -2^-7, the activation alone.  The tail's fit is 2.8e-5 of it off, hardware reciprocal,
    exponential and their arguments (x^2 / 2 up to 72) some 2e-5: 2^-14 together, and the result's half step."""
    from vision_assist_amd.tokens import Linear
    bits = torch.arange(0x10000, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    x = x[(x >= -12) & (x <= -2.0 ** -7)]
    w = torch.zeros(1, K)
    w[0, 0] = 1
    rows = torch.zeros(len(x), K, dtype=torch.bfloat16)
    rows[:, 0] = x
    got = Linear(w, act="gelu", device="cuda")(rows.cuda())[:, 0].double().cpu()
    want = 0.5 * x.double() * torch.erfc(x.double() * -(0.5 ** 0.5))
    assert float(((got - want).abs() / ((2.0 ** -8 + 2.0 ** -14) * want.abs())).max()) <= 1


def test_layers_are_made_on_a_gpu():
    from vision_assist_amd import _lib
    from vision_assist_amd.tokens import Linear, QKNorm, Rotary, TokenCache
    for make in (lambda d: Linear(torch.zeros(8, 8), device=d), lambda d: Rotary(8, device=d), lambda d: QKNorm(8, device=d),
                 lambda d: TokenCache(1, 4, 1, 8, device=d)):
        with pytest.raises(_lib.VaError, match="device cpu"):
            make("cpu")
    here = torch.device("cuda", torch.cuda.current_device())
    for d in (None, "cuda", here):
        assert Linear(torch.zeros(8, 8), device=d).device == QKNorm(8, Rotary(8, device=d), device=d).device == here
        assert TokenCache(1, 4, 1, 8, device=d).k.device == here


ANY, FEW, TILE, TILE_2K, LARGE = range(5)  # VA_TOK_LINEAR_*
FORMS = [(ANY, "bf16", 130, 131, 201), (ANY, "w8a16", 130, 131, 201), (ANY, "f32", 130, 131, 201),
         (FEW, "bf16", 9, 1032, 300), (FEW, "bf16", 30, 520, 301), (FEW, "w8a16", 9, 1032, 300), (FEW, "w8a16", 61, 520, 301),
         (FEW, "f32", 29, 516, 300), (FEW, "bf16", 300, 200, 500),
         (TILE, "bf16", 1301, 328, 1001), (TILE, "w8a16", 2115, 328, 1044), (TILE, "f32", 2115, 332, 1044),
         (TILE_2K, "w8a16", 1301, 456, 1001), (TILE_2K, "f32", 1301, 332, 1001), (TILE_2K, "f32", 1301, 64, 580),
         (LARGE, "bf16", 3700, 328, 2101), (LARGE, "w8a16", 4500, 328, 2101)]


@pytest.mark.parametrize("form,dtype,M,K,N", FORMS)
def test_linear_forms(form, dtype, M, K, N):
    """Each kernel form over several turns of its ring, at ragged rows, channels and K: every activation, bias, residual,
    result = residual, float results, and rows of the result that take stores of eight, four and single values.  Bound: float
    sums (K + 8) 2^-24 sum |x w| with the activations' slope, 2^-14 of a bf16 result for its hardware activation (float: 2^-21),
    and the result's half step."""
    import ctypes

    from vision_assist_amd import _lib
    from vision_assist_amd.tokens import Linear
    from tests.test_gpu_tokens import act64
    g = torch.Generator().manual_seed(M + K + N)
    t = DT[dtype]
    x, w, b, r = rnd(g, M, K, dtype=t), rnd(g, N, K, by=K ** -0.5), rnd(g, N, by=0.3), rnd(g, M, N, dtype=t)
    scale = None
    if dtype == "w8a16":
        scale = w.abs().amax(1) / 448
        w = (w / scale[:, None]).to(torch.float8_e4m3fn)
    elif dtype == "bf16":
        w = w.to(t)
    wd = w.double() if scale is None else w.double() * scale.double()[:, None]
    raw, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    sums = 1.2 * (K + 8) * 2.0 ** -24 * (mag + b.double().abs()) + 2.0 ** -30
    x, rd = x.cuda(), r.cuda()
    # (activation, bias, residual, float result, width of the result's rows, first column; None: a tensor of the call's own)
    calls = [(None, False, False, False, None, 0), ("silu", True, True, False, (N + 15) // 8 * 8, 8), ("gelu", True, False, False, None, 0),
             ("gelu_tanh", False, True, False, (N + 7) // 4 * 4 // 8 * 8 + 4, 4), ("relu", True, True, False, N + 4 - N % 2, 1),
             ("gelu", True, True, True, (N + 15) // 8 * 8, 4), ("silu", False, False, True, N | 1, 0), (None, True, True, True, (N + 7) // 4 * 4, 4)]
    for act, bias, res, f32, width, first in calls:
        lin = Linear(w, b if bias else None, act=act, dtype=dtype, scale=scale, device="cuda")
        ot = torch.float32 if f32 else t
        buf = torch.full((M, N if width is None else width + first), 3.0, dtype=ot, device="cuda")
        out = buf[:, first:first + N]
        same = res and ot == t and width is not None  # the result is the residual
        if same:
            out.copy_(rd)
        arg = out if same else rd if res else None
        assert _lib.load().va_tok_linear_form(ctypes.byref(lin.args(x, out, arg))) == form
        assert lin(x, residual=arg, out=out) is out
        y = act64(raw + b.double() if bias else raw, act)
        want = y + r.double() if res else y
        got = out.double().cpu()
        u = U[torch.float32] if f32 or dtype == "f32" else U[torch.bfloat16]
        tol = sums + (2.0 ** -21 if u < 2.0 ** -20 else 2.0 ** -14) * (y.abs() + want.abs()) + u * (want.abs() + sums)
        worst = float(((got - want).abs() / tol).max())
        assert worst <= 1, (act, bias, res, f32, width, first, worst)
        assert (buf[:, :first] == 3).all() and (buf[:, first + N:] == 3).all()


def test_layers_keep_their_own_weights():
    """What a layer was made of may change afterwards, all of it or none: the layer is what it was."""
    from vision_assist_amd.tokens import Linear, QKNorm
    g = torch.Generator().manual_seed(7)
    w, b, n = rnd(g, 96, 64).cuda(), rnd(g, 96).cuda(), 1 + rnd(g, 64).cuda()
    x = rnd(g, 2, 5, 3, 64, dtype=torch.float32).cuda()
    layers = [Linear(w, b, dtype="f32"), Linear(w, b, dtype="w8a16"), QKNorm(64, q_weight=n, k_weight=n)]
    calls = [lambda: layers[0](x), lambda: layers[1](x.bfloat16()), lambda: torch.stack(layers[2](x, x))]
    want = [c() for c in calls]
    for t in (w, b, n):
        t.add_(1)
    assert all(torch.equal(c(), y) for c, y in zip(calls, want))
