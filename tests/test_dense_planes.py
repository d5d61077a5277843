"""f32 on the bf16 matrix units: every operand is three bf16 numbers, a = a0 + a1 + a2, and six of the nine products are multiplied.  Each of the six is
decided by inputs whose larger products cancel, so that a lost plane or a wrong index shows; on the CPU the inputs themselves are tried with each product
left out."""
import math

import numpy as np
import pytest
import torch

from test_gpu_dense import DEV, E, _d, _rand, ctx  # noqa: F401 (ctx: the fixture)

SIX = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]
WHOLE = [1.0, 1.0 + 2.0 ** -9, 1.0 + 2.0 ** -9 + 2.0 ** -18]          # planes (1), (1, 2^-9), (1, 2^-9, 2^-18)
PLANE = [1.0, 2.0 ** -9, 2.0 ** -18]


def _planes(x):
    out = []
    for _ in range(3):
        out.append(x.to(torch.bfloat16).float())
        x = x - out[-1]
    return out


def _sum_of(products, x, w):
    """x w^T from some of the products of planes"""
    px, pw = _planes(x), _planes(w)
    return sum(px[i].double() @ pw[j].double().t() for i, j in products)


def _deciding(i, j, length, rng):
    """(a row of x, a row of w) whose product is a_i b_j alone: all that is larger, and all else, is taken off by terms of single planes"""
    x, w = np.zeros(length), np.zeros(length)
    at = rng.permutation(length)
    x[at[0]], w[at[0]] = WHOLE[i], WHOLE[j]
    k = 1
    for m in range(i + 1):
        for n in range(j + 1):
            if (m, n) != (i, j) and m + n <= 2:
                x[at[k]], w[at[k]] = -PLANE[m], PLANE[n]
                k += 1
    return x, w


def test_the_inputs_decide():
    """without its product each of them is off by the whole result; with all six none is, beyond the 2^-24 that the three left out may reach"""
    rng = np.random.default_rng(0)
    for i, j in SIX:
        x, w = (torch.tensor(r, dtype=torch.float32)[None] for r in _deciding(i, j, 8, rng))
        want = PLANE[i] * PLANE[j]
        assert float((x.double() @ w.double().t())[0, 0]) == pytest.approx(want, abs=2.0 ** -26)
        assert abs(float(_sum_of(SIX, x, w)) - want) <= 2.0 ** -26
        for left_out in SIX:
            off = abs(float(_sum_of([p for p in SIX if p != left_out], x, w)) - want)
            assert left_out != (i, j) or off >= 0.9 * want


def test_what_is_left_out():
    """a1 b2 + a2 b1 + a2 b2 is at most 2^-24 |a b| (|a1| <= 2^-8 |a|, |a2| <= 2^-17 |a|), and comes close to it"""
    x = torch.tensor(1 + 2.0 ** -8 * (1 + np.random.default_rng(1).random(200000)), dtype=torch.float32)
    six = sum(_planes(x)[i].double() * _planes(x)[j].double() for i, j in SIX)
    off = ((six - x.double() ** 2).abs() / x.double() ** 2).max()
    assert 2.0 ** -25 < float(off) <= 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1300, 1300), (4160, 2070), (5000, 5000)])       # the three tile sizes
@pytest.mark.parametrize("K", [128, 259])
def test_linear_multiplies_six_products(ctx, M, N, K):
    """every pair of rows against 64 bits: the sums are exact but for the products left out (2^-27 and less each, up to four terms)"""
    rng = np.random.default_rng(N + K)
    x, w = np.zeros((len(SIX), K)), np.zeros((len(SIX), K))
    for r, (i, j) in enumerate(SIX):
        x[r], w[r] = _deciding(i, j, K, rng)
    x, w = torch.tensor(x, dtype=torch.float32, device=DEV), torch.tensor(w, dtype=torch.float32, device=DEV)
    want = _d(x) @ _d(w).t()
    assert all(float(want[r, r]) == pytest.approx(PLANE[i] * PLANE[j], abs=2.0 ** -26) for r, (i, j) in enumerate(SIX))
    got = _d(ctx.linear(x.repeat(-(-M // 6), 1)[:M], w.repeat(-(-N // 6), 1)[:N]))
    assert float((got - want.repeat(-(-M // 6), -(-N // 6))[:M, :N]).abs().max()) <= 2.0 ** -25


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1300, 1300, 200), (4160, 2070, 128), (5000, 5000, 136), (3000, 700, 1024)])
def test_linear_f32_error(ctx, M, N, K):
    """2-norm against 64 bits.  A result is rounded by every instruction that adds to it, n = 6 K / 16 of them (8 terms more at the ends), each time by
    half a step of the sum so far, e of it at the most; the sum after k of n steps of random terms is sqrt(k / n) of the whole, and roundings of either
    sign add up as squares: sqrt(sum k / n) e = sqrt((n + 1) / 2) e, and two roundings more for the terms within an instruction and the result.  That
    is 3e-7 to 8e-7 here; sums without one of the products are 2.4e-6 off and more."""
    rng = np.random.default_rng(K)
    x, w = _rand(rng, (M, K), "f32"), _rand(rng, (N, K), "f32", K ** -0.5)
    want = _d(x) @ _d(w).t()
    n = 6 * (-(-K // 16) + 8)
    assert float((_d(ctx.linear(x, w)) - want).norm() / want.norm()) <= (math.sqrt((n + 1) / 2) + 2) * E


@pytest.mark.gpu
@pytest.mark.parametrize("D,Lq", [(32, 64), (64, 200), (128, 64), (65, 64)])
@pytest.mark.parametrize("i,j", SIX)
def test_attention_scores_multiply_six_products(ctx, D, Lq, i, j):
    """one key whose score is a_i b_j, scaled to 1, among keys of score 0: its weight is e / (e + n), and would be 1 / (1 + n) without the product.
    The score is exact but for 2^-26 before the scale of up to 2^18: ds = 2^-8."""
    rng = np.random.default_rng(D)
    x, w = _deciding(i, j, D, rng)
    n = 99
    q = torch.tensor(x, dtype=torch.float32, device=DEV).expand(1, Lq, 1, D).contiguous()
    k = torch.zeros(1, n + 1, 1, D, device=DEV)
    k[0, 70, 0] = torch.tensor(w, dtype=torch.float32)
    v = torch.zeros(1, n + 1, 1, D, device=DEV)
    v[0, 70] = 1.0
    got = _d(ctx.attention(q, k, v, scale=1.0 / (PLANE[i] * PLANE[j])))
    assert float((got / (math.e / (math.e + n)) - 1).abs().max()) <= 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("D,Lq", [(32, 64), (64, 200), (128, 64), (65, 64)])
@pytest.mark.parametrize("s", [-0.3, -1.7, -4.1])
def test_attention_weights_multiply_six_products(ctx, D, Lq, s):
    """two keys of weights p and 1 and values v and -f32(p v): what is left is the roundings.  p from the power instruction (an argument off by 2 e |s c|,
    2 e itself), the product 4 e, the second value's rounding e, the sums 4 e: with |s c| < 6 at most 24 e of p v + p v.  A lost product is 2^-18 of it
    for most of the D values v that are tried."""
    rng = np.random.default_rng(int(-10 * s))
    q, k = torch.zeros(1, Lq, 1, D, device=DEV), torch.zeros(1, 2, 1, D, device=DEV)
    q[..., 0] = 1.0
    k[0, 0, 0, 0] = s
    p = math.exp(float(np.float32(s)))
    v = torch.zeros(1, 2, 1, D, dtype=torch.float64)
    v[0, 0, 0] = torch.tensor((1 + rng.random(D)).astype(np.float32)).double()
    v[0, 1, 0] = (-p * v[0, 0, 0]).float().double()
    got = _d(ctx.attention(q, k, v.float().to(DEV), scale=1.0))[0, :, 0] * (1 + p)
    left = p * v[0, 0, 0] + v[0, 1, 0]
    assert float(((got - left).abs() / (p * v[0, 0, 0])).max()) <= 24 * E


@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64, 128, 65])
def test_attention_f32_error(ctx, D):
    """2-norm against 64 bits of random rows: scores of about 1 off by sqrt(D) roundings, weights and sums by a few more: 2^-20 is 16 roundings"""
    rng = np.random.default_rng(D)
    q, k, v = (_rand(rng, (1, 300, 1, D), "f32") for _ in range(3))
    Q, K, V = (_d(t)[0, :, 0] for t in (q, k, v))
    want = torch.softmax(Q @ K.t() * D ** -0.5, -1) @ V
    assert float((_d(ctx.attention(q, k, v))[0, :, 0] - want).norm() / want.norm()) <= 2.0 ** -20
