"""The dense operators over keypoints on the GPU (lib.Context.linear / qk_norm_rope / attention) against their definitions in 64 bits.

Tolerances count roundings, element by element.  u = half a step of the result's type (2^-24, 2^-11, 2^-8 relative), e = 2^-24:
  * every result is rounded once:                                                                              u |y|
  * a sum of n products in f32, in any order and with either rounding of the adder:                            2 (n + 8) e sum |x w|
  * an activation of v in f32 (slope at most 1.13; erfc and exp at an argument that is off by 2 e of itself):  1.13 dv + (16 + 4 v^2) e |act(v)|
  * a head norm: (D + 16) e on the factor; sin and cos are rounded to f32; three products and a sum:           (D + 32) e (|a| + |b|)
  * a softmax weight whose score (times scale) is off by ds has a relative error of 2 ds (weight and sum); the weights of halves are
    rounded to u of the weight;  the sums over keys as above:                                                  (2 ds + u_w + 2 (n + 64) e) sum p |v|
plus the type's smallest step where results are subnormal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}
E = 2.0 ** -24
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ctx(bx, packed):
    from bufferx_amd import lib
    cfg = bx.make_cfg("3DMatch")
    cfg.patch.num_fps, cfg.patch.num_points_per_patch, cfg.patch.num_scales = 512, 64, 1
    cfg.patch.search_radius_thresholds = [2]
    cfg.patch.num_points_radius_estimate = 64
    c = lib.Context(cfg, max_points=1024, device=0, packed_weights=packed)
    yield c
    c.close()


def _rand(rng, shape, dt, scale=1.0):
    return torch.tensor(rng.standard_normal(shape) * scale, dtype=torch.float32).to(DT[dt]).to(DEV)


def _d(t):
    return t.detach().double().cpu()


def _within(got, want, tol, what=""):
    got = _d(got)
    assert got.shape == want.shape
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)]), what
    off = (got - want).abs()[finite] - tol[finite]
    assert off.numel() == 0 or float(off.max()) <= 0.0, (what, float(off.max()), float((got - want).abs()[finite].max()))


# ------------------------------------------------------------------ linear
ACT = {"none": lambda v: v, "relu": lambda v: torch.clamp(v, min=0.0), "silu": lambda v: v * torch.sigmoid(v),
       "gelu": lambda v: 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))}


def _linear_ref(x, w, bias, act, residual, dt):
    X, W = _d(x), _d(w)
    b = _d(bias) if bias is not None else torch.zeros(W.shape[0], dtype=torch.float64)
    v = X @ W.t() + b
    mag = X.abs() @ W.abs().t() + b.abs()
    a = ACT[act](v)
    y = a + _d(residual) if residual is not None else a
    dv = 2 * (X.shape[1] + 8) * E * mag
    tol = HALF_STEP[dt] * y.abs() + (1.13 * dv + (16 + 4 * v * v) * E * a.abs() + 4 * E * (a.abs() + y.abs())) * (1 + 2 * HALF_STEP[dt]) + TINY[dt]
    return y, tol


def _linear_case(ctx, dt, M, N, K, act="none", bias=True, residual=True, pads=(0, 0, 0, 0), seed=0, offset=0):
    rng = np.random.default_rng(seed + M * 7 + N * 3 + K)
    x = _rand(rng, (M, K + pads[0] + offset), dt)[:, offset:offset + K]
    w = _rand(rng, (N, K + pads[1]), dt, 1 / math.sqrt(max(K, 1)))[:, :K]
    b = _rand(rng, (N,), dt) if bias else None
    r = _rand(rng, (M, N + pads[2]), dt)[:, :N] if residual else None
    out = torch.full((M, N + pads[3]), 7.0, dtype=DT[dt], device=DEV)
    y = ctx.linear(x, w, bias=b, act=act, residual=r, out=out[:, :N])
    assert y.data_ptr() == out.data_ptr() or M * N == 0
    assert bool((out[:, N:] == 7.0).all())
    want, tol = _linear_ref(x, w, b, act, r, dt)
    _within(y, want, tol, (dt, M, N, K, act))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 8), (1, 130, 257), (3, 5, 7), (16, 16, 32), (17, 40, 1030), (33, 64, 64), (40, 72, 300),
                                   (64, 64, 64), (65, 63, 129), (200, 333, 77), (257, 517, 333), (1000, 128, 48), (2049, 260, 96), (3000, 24, 8)])
def test_linear(ctx, dt, M, N, K):
    _linear_case(ctx, dt, M, N, K, act=["none", "relu", "gelu", "silu"][(M + N + K) % 4], bias=(M + K) % 3 != 0, residual=(N + K) % 2 == 0)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_activations(ctx, dt, act):
    _linear_case(ctx, dt, 96, 80, 72, act=act, residual=False)
    # the whole range of arguments through a product with one: far negative values, zero, large ones
    v = torch.cat([torch.linspace(-14, 14, 1021), torch.tensor([0.0, -0.0, 1e4])]).to(DT[dt]).to(DEV)[:, None]
    one = torch.ones((1, 1), dtype=DT[dt], device=DEV)
    want, tol = _linear_ref(v, one, None, act, None, dt)
    _within(ctx.linear(v, one, act=act), want, tol, act)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pads,offset", [((8, 8, 8, 8), 0), ((1, 3, 5, 7), 0), ((0, 1, 0, 0), 0), ((8, 0, 0, 0), 1), ((0, 0, 1, 0), 0), ((0, 0, 0, 1), 0)])
@pytest.mark.parametrize("M,N,K", [(5, 48, 96), (300, 48, 96), (2100, 144, 136)])
def test_linear_strides(ctx, dt, pads, offset, M, N, K):
    _linear_case(ctx, dt, M, N, K, act="relu", pads=pads, offset=offset)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_linear_big_tiles(ctx, dt):
    _linear_case(ctx, dt, 4200, 1100, 200, act="gelu")
    _linear_case(ctx, dt, 4096, 1024, 256, act="none", residual=False)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("M,N,K", [(20, 2100, 300), (31, 1056, 1024), (100, 1100, 520), (129, 640, 136), (300, 2000, 264), (1100, 300, 1031)])
def test_linear_few_tiles(ctx, dt, pad, M, N, K):
    """outputs that do not fill the card: the slices of K are dealt to groups of waves"""
    _linear_case(ctx, dt, M, N, K, act="silu", pads=(pad, pad, 0, 0))


@pytest.mark.parametrize("dt,M,N,K", [("f32", 8200, 1100, 264), ("bf16", 8230, 1030, 256), ("bf16", 33000, 1100, 72), ("f16", 33000, 1027, 100), ("f16", 33000, 1027, 203),
                                       ("bf16", 9000, 700, 203), ("f16", 40000, 30, 200), ("f32", 40000, 17, 9), ("bf16", 140000, 64, 16),
                                       ("f32", 70000, 64, 136)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_many_tiles(ctx, dt, M, N, K, act):
    _linear_case(ctx, dt, M, N, K, act=act, residual=act == "none")


def test_linear_zero_sizes(ctx):
    for M, N, K in ((0, 5, 3), (5, 0, 3), (0, 0, 0)):
        assert ctx.linear(torch.zeros(M, K, device=DEV), torch.zeros(N, K, device=DEV)).shape == (M, N)
    b = torch.tensor([1.0, -2.0], device=DEV)                  # K = 0: the epilogue alone
    y = ctx.linear(torch.zeros(70, 0, device=DEV), torch.zeros(2, 0, device=DEV), bias=b, act="relu", residual=torch.ones(70, 2, device=DEV))
    assert torch.equal(y, torch.tensor([[2.0, 1.0]], device=DEV).expand(70, 2))


@pytest.mark.parametrize("M,N,K", [(24, 40, 64), (700, 96, 64), (5000, 512, 64)])
@pytest.mark.parametrize("share", [-0.1, 0.0, 0.37, 1.0, 2.0])
def test_linear_live_rows(ctx, M, N, K, share):
    rng = np.random.default_rng(M)
    live = int(share * M)
    x, w, r = _rand(rng, (M, K), "bf16"), _rand(rng, (N, K), "bf16", 0.1), _rand(rng, (M, N), "bf16")
    n = max(0, min(M, live))
    x[n:] = float("nan")
    r[n:] = float("nan")
    out = torch.full((M, N), 3.0, dtype=torch.bfloat16, device=DEV)
    ctx.linear(x, w, residual=r, out=out, m_dev=torch.tensor([live], dtype=torch.int32, device=DEV))
    assert bool((out[n:] == 3.0).all())
    want, tol = _linear_ref(x[:n], w, None, "none", r[:n], "bf16")
    _within(out[:n], want, tol)


def test_linear_residual_in_place_and_broadcast_rows(ctx):
    rng = np.random.default_rng(5)
    for M, N, K in ((9, 32, 64), (800, 96, 64)):
        x, w, y = _rand(rng, (1, K), "f32").expand(M, K), _rand(rng, (N, K), "f32"), _rand(rng, (M, N), "f32")
        want, tol = _linear_ref(x, w, None, "silu", y, "f32")
        assert ctx.linear(x, w, act="silu", residual=y, out=y) is y
        _within(y, want, tol)


def test_linear_nonfinite_stays_in_its_row(ctx):
    rng = np.random.default_rng(6)
    for M in (20, 400):
        x, w = _rand(rng, (M, 64), "f32"), _rand(rng, (48, 64), "f32")
        x[3, 5], x[7, 1], x[11] = float("nan"), float("inf"), 0.0
        for act in ("none", "relu"):
            y = ctx.linear(x, w, act=act)
            want = ACT[act](_d(x) @ _d(w).t())
            assert bool(torch.isnan(y[3]).all()) and torch.equal(_d(y[7]), want[7]) and bool((y[11] == 0).all())
            rest = [i for i in range(M) if i not in (3, 7)]
            assert bool(torch.isfinite(y[rest]).all())


@pytest.mark.parametrize("M,N,K", [(3000, 400, 160), (9000, 1024, 256), (25000, 1100, 136)])
def test_linear_f32_long_sums(ctx, M, N, K):
    """f32 outputs large enough to be summed by planes: roundings as f32's, and rows with NaN, infinities or the largest numbers as f32 has them"""
    rng = np.random.default_rng(K)
    x, w = _rand(rng, (M, K), "f32"), _rand(rng, (N, K), "f32", K ** -0.5)
    x[5] *= 1e30
    x[6] *= 1e-30
    x[9, 3], x[17, 1], x[23, 2], x[40] = float("nan"), float("inf"), -float("inf"), 0.0
    x[31, 7] = torch.finfo(torch.float32).max
    w[:, 7] *= 0.25                                          # |w| < 1: the products of the largest number stay finite
    y = ctx.linear(x, w)
    want, tol = _linear_ref(x, w, None, "none", None, "f32")
    _within(y, want, tol, (M, N, K))


def test_linear_far_rows(ctx):
    """row offsets past 2^31 elements"""
    ld = (1 << 30) + 8
    x = torch.empty(3 * ld, dtype=torch.bfloat16, device=DEV).as_strided((3, 64), (ld, 1))
    x.copy_(_rand(np.random.default_rng(1), (3, 64), "bf16"))
    w = _rand(np.random.default_rng(2), (40, 64), "bf16")
    want, tol = _linear_ref(x, w, None, "none", None, "bf16")
    _within(ctx.linear(x, w), want, tol)
    y = torch.empty(3 * ld, dtype=torch.bfloat16, device=DEV).as_strided((3, 40), (ld, 1))
    ctx.linear(x, w, out=y)
    _within(y, want, tol)


# ------------------------------------------------------------------ norm + rotation
def _rope_ref(x, weight, pos, freqs, sections, norm, eps, pairs, dt):
    X = _d(x)
    D = X.shape[-1]
    if norm == "rms":
        f = 1.0 / torch.sqrt((X * X).mean(-1, keepdim=True) + eps)
    elif norm == "l2":
        f = 1.0 / torch.clamp(torch.sqrt((X * X).sum(-1, keepdim=True)), min=eps)
    else:
        f = torch.ones(X.shape[:-1] + (1,), dtype=torch.float64)
    X = X * f * (_d(weight) if weight is not None else 1.0)
    P = sum(sections)
    axis = np.repeat(np.arange(len(sections)), sections)
    t = (_d(pos)[:, axis] * _d(freqs))[:, None]
    i = torch.arange(P) if pairs == "half" else 2 * torch.arange(P)
    j = i + P if pairs == "half" else i + 1
    y, mag = X.clone(), X.abs()
    a, b = X[..., i], X[..., j]
    y[..., i], y[..., j] = a * torch.cos(t) - b * torch.sin(t), b * torch.cos(t) + a * torch.sin(t)
    mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return y, HALF_STEP[dt] * y.abs() + (D + 32) * E * mag * (1 + 2 * HALF_STEP[dt]) + TINY[dt]


def _rope_case(ctx, dt, T, Hq, Hk, D, sections, norm="rms", pairs="half", weight=True, pos="metric", packed=False, inplace=False, seed=0, eps=1e-6, scale=1.0):
    rng = np.random.default_rng(seed + T + D)
    rows = _rand(rng, (T, Hq + 2 * Hk, D), dt, scale)
    q, k = rows[:, :Hq], rows[:, Hq:Hq + Hk]
    if not packed:
        q, k = q.contiguous(), k.contiguous()
    if pos == "metric":
        p = torch.tensor(rng.random((T, len(sections))) * 60 - 20, dtype=torch.float32, device=DEV)
        freqs = torch.tensor(2 * np.pi / (0.05 * 400.0 ** rng.random(sum(sections))), dtype=torch.float64, device=DEV)
    else:
        p = torch.tensor(rng.integers(-5, 2000000, (T, len(sections))), dtype=torch.int32, device=DEV)
        freqs = torch.tensor(10000.0 ** -rng.random(sum(sections)), dtype=torch.float64, device=DEV)
    qw = (1 + 0.3 * _rand(rng, (D,), dt)) if weight else None
    kw = (1 + 0.3 * _rand(rng, (D,), dt)) if weight else None
    wq, tq = _rope_ref(q, qw, p, freqs, sections, norm, eps, pairs, dt)
    wk, tk = _rope_ref(k, kw, p, freqs, sections, norm, eps, pairs, dt)
    rest = rows[:, Hq + Hk:].clone()
    qo, ko = ctx.qk_norm_rope(q, k, p, freqs, sections, norm=norm, eps=eps, q_weight=qw, k_weight=kw, pairs=pairs, q_out=q if inplace else None,
                              k_out=k if inplace else None)
    _within(qo, wq, tq, "q")
    _within(ko, wk, tk, "k")
    assert torch.equal(rest, rows[:, Hq + Hk:])
    return q, k, p, freqs, qw, kw, qo, ko


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,Hq,Hk,D,sections", [(1, 1, 1, 2, (1,)), (1, 32, 8, 128, (64,)), (5, 3, 1, 20, (3, 3, 3)), (33, 8, 8, 32, (6, 5, 5)),
                                                (7, 4, 2, 80, (8, 0, 12)), (130, 2, 2, 256, (32, 32, 32, 32)), (9, 1, 1, 1, (0,)), (64, 5, 3, 33, (4, 7)),
                                                (3, 2, 1, 128, (16, 20, 20)), (19, 6, 2, 64, (32,)), (11, 2, 2, 24, (4, 4, 4)), (4, 3, 3, 100, (7,))])
@pytest.mark.parametrize("norm,pairs,weight,pos", [("rms", "half", True, "whole"), ("l2", "interleaved", False, "metric"), ("none", "half", False, "metric"),
                                                   ("none", "interleaved", True, "whole")])
def test_rope(ctx, dt, T, Hq, Hk, D, sections, norm, pairs, weight, pos):
    _rope_case(ctx, dt, T, Hq, Hk, D, sections, norm, pairs, weight, pos)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("D,sections", [(64, (12, 10, 10)), (72, (36,)), (30, (5, 5))])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
def test_rope_packed_rows(ctx, dt, inplace, D, sections, pairs):
    """q and k side by side in one projection's rows, out of place and in place (the values behind them stay)"""
    _rope_case(ctx, dt, 77, 4, 2, D, sections, pairs=pairs, packed=True, inplace=inplace)


def test_rope_one_side_and_live_tokens(ctx):
    q, k, p, freqs, qw, kw, qo, ko = _rope_case(ctx, "bf16", 50, 4, 2, 64, (12, 10, 10))
    only_q, none = ctx.qk_norm_rope(q, None, p, freqs, (12, 10, 10), q_weight=qw)
    assert none is None and torch.equal(only_q, qo)
    none, only_k = ctx.qk_norm_rope(None, k, p, freqs, (12, 10, 10), k_weight=kw)
    assert none is None and torch.equal(only_k, ko)
    for live in (-3, 0, 17, 50, 99):
        a, b = torch.full_like(qo, 5.0), torch.full_like(ko, 5.0)
        ctx.qk_norm_rope(q, k, p, freqs, (12, 10, 10), q_weight=qw, k_weight=kw, q_out=a, k_out=b, m_dev=torch.tensor([live], dtype=torch.int32, device=DEV))
        n = max(0, min(50, live))
        assert torch.equal(a[:n], qo[:n]) and torch.equal(b[:n], ko[:n]) and bool((a[n:] == 5).all()) and bool((b[n:] == 5).all())


def test_rope_zero_rows_and_degenerate_heads(ctx):
    e = torch.ones(4, dtype=torch.float64, device=DEV)
    qo, ko = ctx.qk_norm_rope(torch.zeros(0, 2, 8, device=DEV), torch.zeros(0, 1, 8, device=DEV), torch.zeros(0, 1, device=DEV), e, (4,))
    assert qo.shape == (0, 2, 8) and ko.shape == (0, 1, 8)
    for norm in ("rms", "l2", "none"):                       # a head of zeros stays zero, a NaN stays in its head
        x = torch.ones(3, 2, 8, device=DEV)
        x[1, 0] = 0.0
        x[2, 1, 6] = float("nan")
        y, _ = ctx.qk_norm_rope(x, None, torch.ones(3, 1, device=DEV), e, (4,), norm=norm)
        assert bool((y[1, 0] == 0).all()) and bool(torch.isfinite(y[:2]).all()) and bool(torch.isfinite(y[2, 0]).all()) and bool(torch.isnan(y[2, 1, 6]))


def test_rope_far_positions(ctx):
    """angles of 1e9 rad and more keep their phase: they are formed and reduced in binary64"""
    T, D = 64, 32
    rng = np.random.default_rng(3)
    x = _rand(rng, (T, 1, D), "f32")
    p = torch.tensor(rng.integers(2**30, 2**31 - 1, (T, 1)), dtype=torch.int32, device=DEV)
    freqs = torch.tensor(1.0 + rng.random(16) * 2.0, dtype=torch.float64, device=DEV)
    y, _ = ctx.qk_norm_rope(x, None, p, freqs, (16,), norm="none")
    want, tol = _rope_ref(x, None, p, freqs, (16,), "none", 0.0, "half", "f32")
    _within(y, want, tol + 2.0 ** -53 * 2.0 ** 33 * 4)       # the product itself is rounded to 53 bits on both sides: 2^33 * 2^-53


# ------------------------------------------------------------------ attention
def _visible(ql, kl, left, right, sinks):
    i, j = torch.arange(ql)[:, None] + (kl - ql), torch.arange(kl)[None]
    see = torch.ones(ql, kl, dtype=torch.bool)
    if right >= 0:
        see &= j <= i + right
    if left >= 0:
        see &= (j >= i - left) | (j < sinks)
    return see


def _attention_ref(q, k, v, scale, left, right, sinks, dt):
    """one batch entry: q [ql, Hq, D], k / v [kl, Hk, D] -> (o, tolerance); keys that a row does not see are left out of its sums"""
    ql, Hq, D = q.shape
    kl, Hk = k.shape[0], k.shape[1]
    o, tol = torch.zeros(ql, Hq, D, dtype=torch.float64), torch.zeros(ql, Hq, D, dtype=torch.float64)
    see = _visible(ql, kl, left, right, sinks)
    for h in range(Hq):
        Q, K, V = _d(q[:, h]), _d(k[:, h * Hk // Hq]), _d(v[:, h * Hk // Hq])
        S = torch.where(see, (Q @ torch.nan_to_num(K, 0, 0, 0).t()) * scale, -math.inf)
        ds = 2 * (D + 8) * E * (Q.abs() @ torch.nan_to_num(K, 0, 0, 0).abs().t()) * scale + 4 * E * torch.where(see, S.abs(), 0.0)
        ds = torch.where(see, ds, 0.0).amax(1, keepdim=True) if kl else torch.zeros(ql, 1, dtype=torch.float64)
        m = S.amax(1, keepdim=True) if kl else torch.zeros(ql, 1, dtype=torch.float64)
        P = torch.where(see, torch.exp(S - torch.where(torch.isfinite(m), m, 0.0)), 0.0)
        L = P.sum(1, keepdim=True)
        P = torch.where(L > 0, P / L, 0.0)
        Vf = torch.nan_to_num(V, 0, 0, 0)
        o[:, h] = P @ Vf
        n = see.sum(1, keepdim=True)
        uw = 0.0 if dt == "f32" else HALF_STEP[dt]
        tol[:, h] = HALF_STEP[dt] * o[:, h].abs() + (2 * ds + uw + 2 * (n + 64) * E) * (P @ Vf.abs()) * (1 + 2 * HALF_STEP[dt]) + TINY[dt]
    return o, tol


def _attention_inputs(dt, B, Lq, Lk, Hq, Hk, D, layout="plain", seed=0):
    rng = np.random.default_rng(seed + 31 * Lq + Lk + D)
    if layout == "packed":
        rows = _rand(rng, (B, Lq, Hq + 2 * Hk, D), dt)
        return rows[:, :, :Hq], rows[:, :, Hq:Hq + Hk], rows[:, :, Hq + Hk:]
    if layout == "heads":                                    # [B, H, L, D] in memory
        return tuple(_rand(rng, (B, H, L, D), dt).transpose(1, 2) for H, L in ((Hq, Lq), (Hk, Lk), (Hk, Lk)))
    if layout == "odd":                                      # rows one element longer than the heads: nothing is aligned
        return tuple(_rand(rng, (B, L, H, D + 1), dt)[..., 1:] for H, L in ((Hq, Lq), (Hk, Lk), (Hk, Lk)))
    return tuple(_rand(rng, (B, L, H, D), dt) for H, L in ((Hq, Lq), (Hk, Lk), (Hk, Lk)))


def _attention_case(ctx, dt, B, Lq, Lk, Hq, Hk, D, window=(-1, -1), sinks=0, layout="plain", lens=None, scale=None, seed=0):
    q, k, v = _attention_inputs(dt, B, Lq, Lk, Hq, Hk, D, layout, seed)
    out = torch.full((B, Lq, Hq, D), 9.0, dtype=DT[dt], device=DEV)
    ql = kl = None
    if lens is not None:
        ql, kl = (torch.tensor([x[i] for x in lens], dtype=torch.int32, device=DEV) for i in (0, 1))
    got = ctx.attention(q, k, v, scale=scale, window=window, sinks=sinks, q_lens=ql, k_lens=kl, out=out)
    assert got is out
    for b in range(B):
        nq, nk = lens[b] if lens is not None else (Lq, Lk)
        nq, nk = max(0, min(Lq, nq)), max(0, min(Lk, nk))
        want, tol = _attention_ref(q[b, :nq], k[b, :nk], v[b, :nk], scale or D ** -0.5, window[0], window[1], sinks, dt)
        _within(out[b, :nq], want, tol, (b, dt, Lq, Lk, Hq, Hk, D, window, sinks, layout))
        assert bool((out[b, nq:] == 9.0).all())


SHAPES = [(1, 1, 1, 1, 1, 8), (1, 1, 700, 4, 1, 64), (2, 3, 65, 6, 2, 40), (1, 64, 64, 2, 2, 32), (2, 130, 130, 3, 1, 128), (1, 257, 190, 4, 4, 20),
          (1, 100, 333, 2, 1, 96), (3, 31, 33, 1, 1, 1), (1, 513, 513, 2, 2, 33), (1, 5, 2, 2, 1, 16)]
MASKS = [((-1, -1), 0), ((-1, 0), 0), ((40, 0), 3), ((17, 9), 1), ((0, 0), 0), ((3, 200), 70)]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("window,sinks", MASKS)
def test_attention(ctx, dt, shape, window, sinks):
    _attention_case(ctx, dt, *shape, window=window, sinks=sinks)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["packed", "heads", "odd"])
@pytest.mark.parametrize("D", [24, 32, 64, 128])
def test_attention_layouts(ctx, dt, layout, D):
    _attention_case(ctx, dt, 2, 150, 150, 4, 2, D, window=(60, 0), sinks=2, layout=layout)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D,layout", [(32, "plain"), (64, "odd"), (128, "heads")])
@pytest.mark.parametrize("sinks", [1, 63, 64, 65, 130])
def test_attention_gap_behind_the_first_keys(ctx, dt, D, layout, sinks):
    """windows that begin one key before, at, one and many keys behind the end of the first keys, for many rows and for one"""
    for gap in (-1, 0, 1, 100):
        _attention_case(ctx, dt, 1, 150, 400, 2, 1, D, window=(250 - sinks - gap, 20), sinks=sinks, layout=layout)
        _attention_case(ctx, dt, 2, 1, 1200, 4, 1, D, window=(1199 - sinks - gap, 0), sinks=sinks, layout=layout, lens=[(1, 1200), (1, 1190)])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("Lk", [63, 64, 65, 1000, 4096, 9001])
@pytest.mark.parametrize("window,sinks", [((-1, 0), 0), ((511, 0), 4), ((100, 0), 150)])
def test_attention_one_query(ctx, dt, Lk, window, sinks):
    """one token against a long store: the keys are split over workgroups and joined"""
    _attention_case(ctx, dt, 2, 1, Lk, 8, 2, 64, window=window, sinks=sinks)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("Lq,Lk,Hq,Hk,D", [(1, 1, 3, 3, 128), (1, 64, 4, 1, 100), (2, 5, 6, 2, 64), (4, 4, 9, 3, 33), (1, 65, 2, 2, 128), (3, 40, 1, 1, 7)])
@pytest.mark.parametrize("window,sinks,layout", [((-1, 0), 0, "plain"), ((2, 0), 1, "odd"), ((-1, -1), 0, "heads")])
def test_attention_few_keys(ctx, dt, Lq, Lk, Hq, Hk, D, window, sinks, layout):
    _attention_case(ctx, dt, 70, Lq, Lk, Hq, Hk, D, window=window, sinks=sinks, layout=layout,
                    lens=[(1 + b % Lq, (7 * b) % (Lk + 1)) for b in range(70)])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((-1, 0), 0), ((30, 5), 2)])
def test_attention_ragged(ctx, dt, window, sinks):
    """lengths on the device: whole, partial, none, one, negative, too large; more queries than keys leaves rows that see nothing"""
    lens = [(90, 200), (90, 77), (0, 50), (1, 1), (60, 0), (50, 20), (-4, 9), (400, 900)]
    _attention_case(ctx, dt, len(lens), 90, 200, 4, 2, 32, window=window, sinks=sinks, lens=lens)
    _attention_case(ctx, dt, 3, 2, 2000, 2, 1, 32, window=window, sinks=sinks, lens=[(2, 2000), (1, 700), (2, 3)])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("Lq,Lk", [(70, 300), (1, 2500)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_attention_hidden_keys_hold_anything(ctx, dt, Lq, Lk, what):
    """keys and values behind the sequence, before the window and between rows' windows may hold anything"""
    what = torch.finfo(DT[dt]).min if what == "lowest" else what
    q, k, v = _attention_inputs(dt, 1, Lq, Lk, 4, 2, 64)
    nk = Lk - 20
    lens = (torch.tensor([Lq], dtype=torch.int32, device=DEV), torch.tensor([nk], dtype=torch.int32, device=DEV))
    k[:, nk:], v[:, nk:] = what, what
    window, sinks = (40, 0), 3
    low = nk - Lq - 40
    k[:, sinks:low], v[:, sinks:low] = what, what            # no row sees these
    got = ctx.attention(q, k, v, window=window, sinks=sinks, q_lens=lens[0], k_lens=lens[1])
    want, tol = _attention_ref(q[0], k[0, :nk], v[0, :nk], 64 ** -0.5, 40, 0, sinks, dt)
    _within(got[0], want, tol)
    if Lq == 1:
        return
    # a value that only some rows see: it reaches those and no others
    at = nk - Lq + 30                                        # rows 30 .. 70 see it (p_i = nk - Lq + i, window 40 back)
    v[0, at, :, 5], v[0, at, :, 60] = what, what
    v[0, at + 1, :, 60] = -what if what == what else what
    got = _d(ctx.attention(q, k, v, window=window, sinks=sinks, q_lens=lens[0], k_lens=lens[1]))[0]
    dims = [d for d in range(64) if d not in (5, 60)]
    _within(got[:, :, dims], want[:, :, dims], tol[:, :, dims])
    _within(got[:30], want[:30], tol[:30])
    if math.isfinite(what):
        return
    reach = got[30:, :, 5]
    assert bool(torch.isnan(reach).all()) if what != what else torch.equal(reach, torch.full_like(reach, what))
    assert bool(torch.isnan(got[31:, :, 60]).all())          # +inf and -inf, or NaN


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_attention_extreme_scores(ctx, dt):
    """scores far apart (one key takes all), rows of equal scores, and a visible row whose scores are all -inf (0 / 0)"""
    q, k, v = _attention_inputs(dt, 1, 40, 200, 2, 2, 32)
    q *= 30
    want, tol = _attention_ref(q[0], k[0], v[0], 1.0, -1, -1, 0, dt)
    _within(ctx.attention(q, k, v, scale=1.0)[0], want, tol)
    q.zero_()
    want, tol = _attention_ref(q[0], k[0], v[0], 1.0, -1, -1, 0, dt)
    _within(ctx.attention(q, k, v, scale=1.0)[0], want, tol)
    q.fill_(1.0)
    k[:, :, 0] = -float("inf")
    got = ctx.attention(q, k, v, scale=1.0)
    assert bool(torch.isnan(got[:, :, 0]).all()) and bool(torch.isfinite(got[:, :, 1]).all())


def test_attention_f32_infinite_and_large(ctx):
    """f32 keys of -inf get no weight, values of +-inf reach the rows that see them, large and small values keep their digits"""
    q, k, v = _attention_inputs("f32", 1, 90, 150, 2, 1, 32)
    q = q.abs()
    k[:, 40] = -float("inf")                                 # scores -inf in every row
    v[:, :, :, 3] *= 1e30
    v[:, :, :, 4] *= 1e-30
    got = ctx.attention(q, k, v)
    keep = [j for j in range(150) if j != 40]
    want, tol = _attention_ref(q[0], k[0, keep], v[0, keep], 32 ** -0.5, -1, -1, 0, "f32")
    _within(got[0], want, tol)
    v[0, 60, 0, 5], v[0, 61, 0, 6], v[0, 62, 0, 6] = float("inf"), float("inf"), -float("inf")
    got = _d(ctx.attention(q, k, v))[0]
    assert bool((got[:, :, 5] == math.inf).all()) and bool(torch.isnan(got[:, :, 6]).all())
    dims = [d for d in range(32) if d not in (5, 6)]
    _within(got[:, :, dims], want[:, :, dims], tol[:, :, dims])


def test_attention_zero_sizes(ctx):
    z = lambda *s: torch.zeros(s, device=DEV)
    assert ctx.attention(z(0, 4, 2, 8), z(0, 4, 2, 8), z(0, 4, 2, 8)).shape == (0, 4, 2, 8)
    assert ctx.attention(z(2, 0, 2, 8), z(2, 4, 2, 8), z(2, 4, 2, 8)).shape == (2, 0, 2, 8)
    got = ctx.attention(z(2, 3, 2, 8) + 1, z(2, 0, 2, 8), z(2, 0, 2, 8), out=z(2, 3, 2, 8) + 4)
    assert bool((got == 0).all())                            # no keys at all: zeros


def test_attention_far_keys(ctx):
    """key offsets past 2^31 elements in a long store"""
    rng = np.random.default_rng(8)
    st = (1 << 30) + 16
    q = _rand(rng, (1, 2, 2, 64), "bf16")
    k = torch.empty(3 * st, dtype=torch.bfloat16, device=DEV).as_strided((1, 3, 2, 64), (0, st, 64, 1))
    v = torch.empty(3 * st, dtype=torch.bfloat16, device=DEV).as_strided((1, 3, 2, 64), (0, st, 64, 1))
    k.copy_(_rand(rng, (1, 3, 2, 64), "bf16"))
    v.copy_(_rand(rng, (1, 3, 2, 64), "bf16"))
    want, tol = _attention_ref(q[0], k[0], v[0], 0.125, -1, -1, 0, "bf16")
    _within(ctx.attention(q, k, v)[0], want, tol)


def test_attention_workspace_too_small(ctx):
    import ctypes as C
    from bufferx_amd import dense, lib
    q, k, v = _attention_inputs("bf16", 1, 1, 9000, 2, 2, 64)
    a, out = dense.attention_args(torch, torch.device(DEV), q, k, v, None, (-1, -1), 0, None, None, None)
    need = ctx.lib.bx_attention_workspace(ctx.handle, C.byref(a))
    assert need > 0
    for ws in (None, torch.empty(need - 4, dtype=torch.uint8, device=DEV)):
        a.workspace, a.workspace_bytes = (ws.data_ptr(), need - 4) if ws is not None else (None, need)
        assert ctx.lib.bx_attention(ctx.handle, None, C.byref(a)) == 3 and b"workspace" in ctx.lib.bx_last_error()


# ------------------------------------------------------------------ streams, graphs, repetition
def _some_calls(ctx, s):
    y = ctx.linear(s["x"], s["w"], bias=s["b"], act="gelu", residual=s["r"])
    small = ctx.linear(s["x"][:3], s["w"])
    qo, ko = ctx.qk_norm_rope(s["q"], s["k"], s["pos"], s["freqs"], (12, 10, 10))
    o = ctx.attention(qo[None], ko[None], s["v"][None], window=(50, 0), sinks=2)
    one = ctx.attention(qo[None, -1:], s["far"][None], s["far"][None])       # split over the keys, joined
    return y, small, qo, ko, o, one


def _some_state(seed):
    rng = np.random.default_rng(seed)
    return {"x": _rand(rng, (500, 96), "bf16"), "w": _rand(rng, (200, 96), "bf16", 0.1), "b": _rand(rng, (200,), "bf16"), "r": _rand(rng, (500, 200), "bf16"),
            "q": _rand(rng, (300, 4, 64), "bf16"), "k": _rand(rng, (300, 2, 64), "bf16"), "v": _rand(rng, (300, 2, 64), "bf16"),
            "pos": torch.tensor(rng.random((300, 3)), dtype=torch.float32, device=DEV), "far": _rand(rng, (5000, 2, 64), "bf16"),
            "freqs": torch.tensor(rng.random(32) * 20, dtype=torch.float64, device=DEV)}


def test_same_bits_on_other_streams_and_again(ctx):
    s = _some_state(1)
    first = [t.clone() for t in _some_calls(ctx, s)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st in streams * 2:                                   # two streams at once, one context
        with torch.cuda.stream(st):
            got.append(_some_calls(ctx, s))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(first, g))


def test_graph_replays(ctx):
    """two graphs of the same calls on their own inputs, replayed in turn between eager work, follow their inputs"""
    states = [_some_state(2), _some_state(3)]
    for s in states:
        _some_calls(ctx, s)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_some_calls(ctx, s))
        graphs.append(g)
    for turn in range(3):
        for i in (0, 1):
            fresh = _some_state(10 * turn + i + 20)
            for name in states[i]:
                states[i][name].copy_(fresh[name])
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            eager = _some_calls(ctx, states[i])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager, outs[i])), (turn, i)


def test_refusals_name_their_fault(ctx):
    from bufferx_amd.lib import BxError
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(BxError, match="overlaps"):
        ctx.linear(x, torch.zeros(8, 8, device=DEV), out=x)
    with pytest.raises(ValueError, match="context is on"):
        ctx.linear(x.cpu(), torch.zeros(8, 8))
    with pytest.raises(BxError, match="D="):
        ctx.attention(torch.zeros(1, 1, 1, 129, device=DEV), torch.zeros(1, 1, 1, 129, device=DEV), torch.zeros(1, 1, 1, 129, device=DEV))
    assert bool((ctx.linear(x + 1, torch.ones(8, 8, device=DEV)) == 8).all())           # the context is as good as before


# ------------------------------------------------------------------ as they are used: between the descriptors and the matching
def test_descriptors_see_the_other_cloud_before_matching(ctx, oracle):
    """One cross-attention layer over the keypoints of two clouds (f32): projections, head norm with the rotation by the keypoints'
    coordinates in place, attention of each cloud over the other with live counts, output projection onto the residual, then bx_mutual."""
    rng = np.random.default_rng(12)
    K, H, D, C = 300, 2, 32, 32
    n = (300, 271)
    desc, kpts = _rand(rng, (2, K, C), "f32"), torch.tensor(rng.random((2, K, 3)) * 4, dtype=torch.float32, device=DEV)
    wqkv, bqkv = _rand(rng, (3 * H * D, C), "f32", C ** -0.5), _rand(rng, (3 * H * D,), "f32", 0.1)
    wo = _rand(rng, (C, H * D), "f32", (H * D) ** -0.5)
    sections, freqs = (6, 5, 5), torch.tensor(2 * np.pi / (0.1 * 40.0 ** rng.random(16)), dtype=torch.float64, device=DEV)
    rows = ctx.linear(desc.view(2 * K, C), wqkv, bias=bqkv).view(2 * K, 3 * H, D)
    q, k = rows[:, :H], rows[:, H:2 * H]
    ctx.qk_norm_rope(q, k, kpts.view(2 * K, 3), freqs, sections, norm="l2", q_out=q, k_out=k)
    rows = rows.view(2, K, 3 * H, D)
    lens = torch.tensor(n, dtype=torch.int32, device=DEV)
    cross = torch.zeros(2, K, H, D, device=DEV)
    for b in (0, 1):
        ctx.attention(rows[b:b + 1, :, :H], rows[1 - b:2 - b, :, H:2 * H], rows[1 - b:2 - b, :, 2 * H:], scale=8.0, q_lens=lens[b:b + 1],
                      k_lens=lens[1 - b:2 - b], out=cross[b:b + 1])
    new = ctx.linear(cross.view(2 * K, H * D), wo, residual=desc.view(2 * K, C)).view(2, K, C)

    X = _d(desc)
    R = (X @ _d(wqkv).t() + _d(bqkv)).view(2, K, 3 * H, D)
    qk = R[:, :, :2 * H]
    qk = qk / qk.norm(dim=-1, keepdim=True).clamp(min=1e-6)
    t = (_d(kpts)[..., np.repeat([0, 1, 2], sections)] * _d(freqs))[:, :, None]
    a, b = qk[..., :16], qk[..., 16:]
    qk = torch.cat([a * torch.cos(t) - b * torch.sin(t), b * torch.cos(t) + a * torch.sin(t)], -1)
    want = X.clone()
    for c in (0, 1):
        S = torch.einsum("ihd,jhd->hij", qk[c, :n[c], :H], qk[1 - c, :n[1 - c], H:]) * 8.0
        O = torch.einsum("hij,jhd->ihd", torch.softmax(S, -1), R[1 - c, :n[1 - c], 2 * H:])
        want[c, :n[c]] += O.reshape(n[c], H * D) @ _d(wo).t()
    # f32 all the way.  An error of a projection (38 terms of size ~1: 2 * 40 e * 6) reaches the scores times 8 * 2 and the weights
    # times 2, then values of size ~4 and 64 products of 1/8: under 3000 * 2 * 16 * e * 4 is 1.2e-2 at the worst; the bound below
    # is the same count with the sums' errors adding as squares (a sum of n roundings ~ sqrt(n) e): sqrt(40) * 6 * 16 * 2 * 4 * e
    assert float((_d(new) - want).abs().max()) < math.sqrt(40) * 6 * 16 * 2 * 4 * E
    s, tt, count = ctx.mutual(new[0, :n[0]].contiguous(), new[1, :n[1]].contiguous())
    m = int(count.cpu())
    rs, rt, _, _ = oracle.mutual(new[0, :n[0]].cpu().numpy(), new[1, :n[1]].cpu().numpy())
    assert m == len(rs) and np.array_equal(s.cpu().numpy()[:m], rs) and np.array_equal(tt.cpu().numpy()[:m], rt)
