"""What the dense operators promise beyond the general tolerances of test_gpu_dense.py, on the GPU: how many bits weights and planes keep, and
what does not change a result at all.  u, e and the counts of roundings are those of that file."""
import math

import numpy as np
import pytest
import torch

from test_gpu_dense import DEV, DT, E, HALF_STEP, TINY, _attention_inputs, _d, _rand, _visible, _within, ctx  # noqa: F401 (ctx: the fixture)

pytestmark = pytest.mark.gpu

# relative error of a softmax weight as it is multiplied: two bf16 (f16) numbers hold it to half a step of half a step
WEIGHT = {"f32": 0.0, "f16": 2.0 ** -22, "bf16": 2.0 ** -16}


def _exact(q, k, v, scale, left, right, sinks, dt):
    """one batch entry in 64 bits -> (o, tolerance); the weights are not rounded to the type of v"""
    ql, Hq, D = q.shape
    kl, Hk = k.shape[0], k.shape[1]
    o, tol = torch.zeros(ql, Hq, D, dtype=torch.float64), torch.zeros(ql, Hq, D, dtype=torch.float64)
    see = _visible(ql, kl, left, right, sinks)
    n = see.sum(1, keepdim=True)
    for h in range(Hq):
        Q, K, V = _d(q[:, h]), _d(k[:, h * Hk // Hq]), _d(v[:, h * Hk // Hq])
        S = torch.where(see, (Q @ K.t()) * scale, -math.inf)
        ds = torch.where(see, 2 * (D + 8) * E * (Q.abs() @ K.abs().t()) * scale + 4 * E * S.abs(), 0.0).amax(1, keepdim=True)
        P = torch.softmax(S, 1)
        o[:, h] = P @ V
        # (f16: the second number ends at 2^-25, and the weights of a row sum up to 2^7 at least)
        low = 2.0 ** -32 * (see.double() @ V.abs()) if dt == "f16" else 0.0
        tol[:, h] = HALF_STEP[dt] * o[:, h].abs() + ((2 * ds + WEIGHT[dt] + 2 * (n + 64) * E) * (P @ V.abs()) + low) * (1 + 2 * HALF_STEP[dt]) + TINY[dt]
    return o, tol


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk,D,window,layout", [
    (130, 130, 4, 2, 32, (24, 24), "packed"), (200, 200, 4, 1, 128, (-1, 0), "packed"), (150, 300, 2, 2, 64, (-1, -1), "plain"),
    (100, 100, 3, 3, 65, (40, 0), "odd"), (1, 300, 8, 2, 64, (-1, 0), "plain"), (3, 5000, 2, 1, 128, (-1, -1), "heads"), (40, 9, 2, 1, 32, (-1, -1), "plain")])
def test_attention_weights_keep_their_bits(ctx, dt, Lq, Lk, Hq, Hk, D, window, layout):
    """f16 and bf16 results are off by their own rounding and little more: in 2-norm a tenth of it, element by element the counted roundings"""
    q, k, v = _attention_inputs(dt, 1, Lq, Lk, Hq, Hk, D, layout)
    got = ctx.attention(q, k, v, window=window)[0]
    want, tol = _exact(q[0], k[0], v[0], D ** -0.5, window[0], window[1], 0, dt)
    _within(got, want, tol, (dt, Lq, Lk, D))
    rounded = (want.to(DT[dt]).double() - want).norm()
    assert float((_d(got) - want).norm()) <= 1.1 * float(rounded)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk,D,at", [(260, 260, 2, 1, 32, 90), (260, 260, 2, 1, 64, 210), (260, 400, 1, 1, 128, 341), (260, 260, 4, 1, 128, 150),
                                              (8, 900, 4, 1, 64, 896), (3, 9000, 2, 2, 128, 8998), (260, 260, 3, 1, 40, 77)])
def test_attention_hidden_keys_change_no_bit(ctx, dt, Lq, Lk, Hq, Hk, D, at):
    """causal rows in front of a key give the same bits whatever finite numbers that key and those behind it hold, also where the rows that
    share a wave with them do see it and find it far above all others"""
    q, k, v = _attention_inputs(dt, 1, Lq, Lk, Hq, Hk, D)
    first = ctx.attention(q, k, v, window=(-1, 0)).clone()
    front = at - (Lk - Lq)                                   # the first row that sees key `at`
    assert 0 < front < Lq
    for scale in (6.0, -40.0):
        k2, v2 = k.clone(), v.clone()
        k2[:, at:] = k2[:, at:] * scale
        v2[:, at:] = 3.0
        got = ctx.attention(q, k2, v2, window=(-1, 0))
        assert torch.equal(got[:, :front], first[:, :front]), (scale, int((got[:, :front] != first[:, :front]).sum()))
        assert not torch.equal(got[:, front:], first[:, front:])


@pytest.mark.parametrize("Lq,Lk", [(1, 256), (1, 9000), (5, 700), (40, 9000), (40, 300), (200, 300)])
@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("at", [3.0, 555.0, -1300.0])
@pytest.mark.parametrize("spoilt", [False, True])
def test_attention_far_scores_keep_their_weights(ctx, Lq, Lk, D, at, spoilt):
    """f32 weights do not suffer where scores lie far from zero: one key of every tile counts, with a score that f32 holds exactly, so that all a
    weight loses is lost in the softmax.  `spoilt`: an infinity has the first tiles summed row by row, beside others that are not.
    Scores are up to 3 apart: 2^-24 of that by scale * log2(e), three roundings of the difference, 2^-23 by each power (the weight's, and twice in
    joining, above and below the line), sums of at most 150 terms in groups of up to 64: 3 e + 3 e + 6 * 2 e + (64 + 4) e, at most 90 e."""
    rng = np.random.default_rng(Lk + D)
    score = np.full(Lk, at - 2000.0, dtype=np.float32)
    some = np.arange(5, Lk, 64)
    score[some] = at + 3.0 * rng.random(len(some))
    k = torch.zeros(1, Lk, 1, D, device=DEV)
    k[0, :, 0, 0] = torch.tensor(score)
    q = torch.zeros(1, Lq, 1, D, device=DEV)
    q[..., 0] = 1.0
    v = _rand(rng, (1, Lk, 1, D), "f32").abs() + 1.0
    if spoilt:
        v[0, some[0], 0, 7] = math.inf
    got = _d(ctx.attention(q, k, v, scale=1.0))[0, :, 0]
    P = torch.softmax(torch.tensor(score[some], dtype=torch.float64), 0)
    want = P @ _d(v)[0, some, 0]
    keep = [d for d in range(D) if d != 7]
    assert float((got[:, keep] / want[keep] - 1).abs().max()) <= 90 * E
    assert not spoilt or bool((got[:, 7] == math.inf).all())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Lq,Lk", [(1, 200), (1, 9000), (40, 200), (130, 500), (40, 9000)])
@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("steps", [1.0, 90.0])
def test_attention_steep_scores(ctx, dt, Lq, Lk, D, sign, steps):
    """scores that f32 holds exactly, 2^30 (f16) or 2^40 away from zero, which times the scale differ by `steps` times a whole number, in
    units of 2^7 (2^17) before it: the weights go by the differences, which are exact.  The same count of roundings as for far scores, and 2^-23 of
    a score difference of up to 255 that a power still sees (those of more than 126 have no weight): 90 e + 2 * 126 e."""
    big, unit = (2.0 ** 15, 2.0 ** 7) if dt == "f16" else (2.0 ** 20, 2.0 ** 17)
    rng = np.random.default_rng(Lq + Lk + D)
    j = rng.integers(0, 256, Lk)
    k = torch.zeros(1, Lk, 1, D, dtype=DT[dt], device=DEV)
    k[..., 0] = sign * big
    k[0, :, 0, 1] = torch.tensor(j, dtype=DT[dt])
    q = torch.zeros(1, Lq, 1, D, dtype=DT[dt], device=DEV)
    q[..., 0], q[..., 1] = big, unit
    v = _rand(rng, (1, Lk, 1, D), dt).abs() + 1.0
    got = _d(ctx.attention(q, k, v, scale=steps / unit))[0, :, 0]
    want = torch.softmax(torch.tensor(j, dtype=torch.float64) * float(np.float32(steps / unit)) * unit, 0) @ _d(v)[0, :, 0]
    n = min(Lk, 9000)
    assert float((got / want - 1).abs().max()) <= HALF_STEP[dt] * (1 + 2 * HALF_STEP[dt]) + WEIGHT[dt] + (90 + 252 + 2 * n / 64) * E


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("Lq,Lk,D", [(1, 200, 64), (32, 256, 64), (64, 256, 128), (256, 192, 32), (64, 192, 65), (64, 9024, 128), (130, 190, 32)])
def test_attention_large_values(ctx, dt, Lq, Lk, D):
    """values of up to 2^127 / Lk and scores that rise by 5 along the keys: sums of weights of at most 1 times values stay in f32's range"""
    rng = np.random.default_rng(D)
    q, k = torch.zeros(1, Lq, 1, D, dtype=DT[dt], device=DEV), torch.zeros(1, Lk, 1, D, dtype=DT[dt], device=DEV)
    q[..., 0] = 1.0
    k[0, :, 0, 0] = torch.arange(Lk, device=DEV) * (5.0 / Lk)
    v = torch.tensor((0.5 + 0.5 * rng.random((1, Lk, 1, D))) * 2.0 ** 127 / Lk, dtype=torch.float32).to(DT[dt]).to(DEV)
    want, tol = _exact(q[0], k[0], v[0], 1.0, -1, -1, 0, dt)
    _within(ctx.attention(q, k, v, scale=1.0)[0], want, tol)


@pytest.mark.parametrize("power", [48, 51, 52, 53, 54, 56, 60, 64, 90, 127, 300, 900, 1023])
@pytest.mark.parametrize("pairs,whole", [("half", False), ("interleaved", True)])
def test_rope_far_angles(ctx, power, pairs, whole):
    """angles of up to 2^1024 rad are turned by, not scaled by: sine and cosine of the binary64 product, each off by half a step of f32 (and 7e-10
    where the product is close to 2^52), three products and a sum: 8 e (|a| + |b|)"""
    T, D = 40, 24
    rng = np.random.default_rng(power)
    x = _rand(rng, (T, 2, D), "f32")
    p = rng.integers(-2 ** 31 + 1, 2 ** 31 - 1, (T, 1)) | 2 ** 30 if whole else (rng.random((T, 1)) + 1) * rng.choice([-1.0, 1.0], (T, 1))
    p = torch.tensor(p, dtype=torch.int32 if whole else torch.float32, device=DEV)
    freqs = torch.tensor((0.5 + 0.5 * rng.random(8)) * 2.0 ** (power - (31 if whole else 1)), dtype=torch.float64, device=DEV)
    y = _d(ctx.qk_norm_rope(x, None, p, freqs, (8,), norm="none", pairs=pairs)[0])
    t = (_d(p) * _d(freqs)).numpy()
    assert np.isfinite(t).all() and np.abs(t).max() >= 2.0 ** (power - 2)
    cos, sin = (torch.tensor(np.vectorize(f)(t))[:, None] for f in (math.cos, math.sin))
    X = _d(x)
    i = torch.arange(8) if pairs == "half" else 2 * torch.arange(8)
    j = i + 8 if pairs == "half" else i + 1
    a, b = X[..., i], X[..., j]
    tol = (8 * E + 1e-9) * (a.abs() + b.abs())
    assert bool(((y[..., i] - (a * cos - b * sin)).abs() <= tol).all()) and bool(((y[..., j] - (b * cos + a * sin)).abs() <= tol).all())
    assert torch.equal(y[..., 16:], X[..., 16:])


def test_rope_angles_that_are_none(ctx):
    """an infinite or undefined angle leaves NaN in its pairs and nothing anywhere else"""
    x = _rand(np.random.default_rng(0), (4, 1, 8), "f32")
    p = torch.tensor([[1.0], [math.inf], [math.nan], [-3e38]], device=DEV)
    freqs = torch.tensor([0.0, 1.0, 1e300], dtype=torch.float64, device=DEV)
    y = ctx.qk_norm_rope(x, None, p, freqs, (3,), norm="none")[0][:, 0]
    nan = torch.zeros(4, 8, dtype=torch.bool)
    nan[1, :6] = nan[2, :6] = True                           # (0 * inf too)
    nan[3, 2] = nan[3, 5] = True                             # 3e38 * 1e300
    assert torch.equal(torch.isnan(y).cpu(), nan) and torch.equal(y[:, 6:], x[:, 0, 6:])


@pytest.mark.parametrize("norm", ["l2", "rms"])
def test_head_norm_divides(ctx, norm):
    """heads (a, 0, b, 0) of whole numbers whose length d is one: the norm is exact and each element is rounded once, as a division does it"""
    m, n = np.meshgrid(np.arange(2, 60), np.arange(1, 59))
    m, n = m[m > n], n[m > n]
    keep = m * m + n * n < 4096                              # (d^2 < 2^24: the sum of squares is exact in f32)
    m, n = m[keep], n[keep]
    x = np.zeros((len(m), 1, 4))
    x[:, 0, 0], x[:, 0, 2] = m * m - n * n, 2 * m * n
    d = (m * m + n * n)[:, None, None] / (2.0 if norm == "rms" else 1.0)
    y = _d(ctx.qk_norm_rope(torch.tensor(x, dtype=torch.float32, device=DEV), None, torch.zeros(len(m), 1, device=DEV),
                            torch.zeros(0, dtype=torch.float64, device=DEV), (0,), norm=norm, eps=0.0)[0])
    want = torch.tensor(x / d)
    assert bool(((y - want).abs() <= HALF_STEP["f32"] * (1 + 2.0 ** -20) * want).all())


@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("scale", [2.0 ** -110, 2.0 ** -60, 2.0 ** -30, 2.0 ** 55, 2.0 ** 63, 2.0 ** 100])
def test_head_norm_far_from_one(ctx, norm, scale):
    """what a head norm gives does not depend on a power of two in front of its elements, also where their squares leave f32's range"""
    x = _rand(np.random.default_rng(1), (50, 3, 16), "f32")
    args = (None, torch.zeros(50, 1, device=DEV), torch.zeros(0, dtype=torch.float64, device=DEV), (0,))
    y = ctx.qk_norm_rope(x, *args, norm=norm, eps=0.0)[0]
    got = ctx.qk_norm_rope(x * scale, *args, norm=norm, eps=0.0)[0]
    assert bool(((got - y).abs() <= 2 * E * y.abs()).all()) and bool(torch.isfinite(got).all())


@pytest.mark.parametrize("norm", ["l2", "rms"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("scale,eps", [(1e30, 1e-6), (1e25, 3e38), (1e-30, 1e-6), (1e-30, 1e-30), (1e-25, 0.0), (1e-38, 1e-37)])
def test_head_norm_of_any_size(ctx, norm, dt, scale, eps):
    """heads between large and small ones, with and without an eps that decides, against 64 bits: (D + 16) e of the factor and a division, the weight's
    product and the result's rounding"""
    D = 48
    x = _rand(np.random.default_rng(2), (30, 2, D), "f32")
    x[::3] *= scale
    x = x.to(DT[dt])
    w = _rand(np.random.default_rng(3), (D,), dt)
    y = ctx.qk_norm_rope(x, None, torch.zeros(30, 1, device=DEV), torch.zeros(0, dtype=torch.float64, device=DEV), (0,), norm=norm, eps=eps, q_weight=w)[0]
    X, e = _d(x), float(np.float32(eps))
    d = torch.sqrt((X * X).mean(-1, keepdim=True) + e) if norm == "rms" else torch.clamp(X.norm(dim=-1, keepdim=True), min=e)
    want = X / d * _d(w)
    _within(y, want, HALF_STEP[dt] * want.abs() + (D + 20) * E * want.abs() * (1 + 2 * HALF_STEP[dt]) + TINY[dt])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(5, 64, 40), (700, 64, 40), (3000, 160, 333)])
def test_linear_beside_its_input(ctx, dt, M, K, N):
    """rows [x | y | residual] of one buffer: the same bits as apart, and nothing else is written"""
    rng = np.random.default_rng(M)
    rows = _rand(rng, (M, K + 2 * N + 3), dt)
    x, y, r, rest = rows[:, :K], rows[:, K:K + N], rows[:, K + N:K + 2 * N], rows[:, K + 2 * N:]
    w = _rand(rng, (N, K), dt, K ** -0.5)
    want = ctx.linear(x, w, act="silu", residual=r)
    before = rows.clone()
    ctx.linear(x, w, act="silu", residual=r, out=y)
    assert torch.equal(y, want) and torch.equal(x, before[:, :K]) and torch.equal(r, before[:, K + N:K + 2 * N]) and torch.equal(rest, before[:, K + 2 * N:])


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("L,D", [(1, 64), (300, 32), (300, 40), (200, 128)])
def test_attention_beside_its_inputs(ctx, dt, L, D):
    """rows [q | k | v | o] of one buffer"""
    rows = _rand(np.random.default_rng(L + D), (2, L, 12, D), dt)
    q, k, v, o = rows[:, :, :4], rows[:, :, 4:6], rows[:, :, 6:8], rows[:, :, 8:]
    want = ctx.attention(q, k, v, window=(30, 0), sinks=2)
    before = rows[:, :, :8].clone()
    ctx.attention(q, k, v, window=(30, 0), sinks=2, out=o)
    assert torch.equal(o, want) and torch.equal(rows[:, :, :8], before)


@pytest.mark.parametrize("M", [1, 70, 3000])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_silu_of_far_negative_numbers(ctx, M, dt):
    """v / (1 + exp(-v)) down to the smallest normal numbers (v about -92), through products with one: the power's argument off by 2 e of itself and the
    power by 4 e, twice, four products: (16 + 4 |v|) e"""
    v = torch.linspace(-91, -60, M).to(DT[dt]).to(DEV)[:, None]
    got = _d(ctx.linear(v, torch.ones((40, 1), dtype=DT[dt], device=DEV), act="silu"))
    want = (_d(v) / (1 + torch.exp(-_d(v)))).expand(M, 40)
    assert bool(((got - want).abs() <= (HALF_STEP[dt] + (16 + 4 * 91) * E) * want.abs() * (1 + HALF_STEP[dt]) + TINY[dt]).all())


def test_attention_workspace_of_no_type(ctx):
    import ctypes as C
    from bufferx_amd import dense
    q, k, v = _attention_inputs("bf16", 1, 1, 9000, 2, 2, 64)
    a, _ = dense.attention_args(torch, torch.device(DEV), q, k, v, None, (-1, -1), 0, None, None, None)
    assert ctx.lib.bx_attention_workspace(ctx.handle, C.byref(a)) > 0
    for a.dtype in (-1, 3):
        assert ctx.lib.bx_attention_workspace(ctx.handle, C.byref(a)) == -1 and b"bad argument" in ctx.lib.bx_last_error()
