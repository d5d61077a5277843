"""Tensors that the dense operators over keypoints refuse because their memory is not their value, or because the call around them would be lost
(bufferx_amd.dense), without a GPU."""
import pytest
import torch

CPU = torch.device("cpu")


def _calls():
    """{operator: (its argument check on CPU tensors, its operands)}"""
    from bufferx_amd import dense
    t = lambda *s: torch.randn(s)
    linear = {"x": t(4, 8), "weight": t(6, 8), "bias": t(6), "residual": t(4, 6), "out": t(4, 6), "m_dev": torch.ones(1, dtype=torch.int32)}
    rope = {"q": t(5, 2, 8), "k": t(5, 1, 8), "pos": t(5, 1), "freqs": torch.ones(4, dtype=torch.float64), "q_weight": t(8), "k_weight": t(8),
            "q_out": t(5, 2, 8), "k_out": t(5, 1, 8), "m_dev": torch.ones(1, dtype=torch.int32)}
    attention = {"q": t(2, 3, 4, 8), "k": t(2, 5, 2, 8), "v": t(2, 5, 2, 8), "q_lens": torch.ones(2, dtype=torch.int32),
                 "k_lens": torch.ones(2, dtype=torch.int32), "out": t(2, 3, 4, 8)}
    return {
        "linear": (lambda x, weight, bias, residual, out, m_dev: dense.linear_args(torch, CPU, x, weight, bias, "none", residual, out, m_dev), linear),
        "rope": (lambda q, k, pos, freqs, q_weight, k_weight, q_out, k_out, m_dev: dense.qk_norm_rope_args(
            torch, CPU, q, k, pos, freqs, (4,), "rms", 1e-6, q_weight, k_weight, "half", q_out, k_out, m_dev), rope),
        "attention": (lambda q, k, v, q_lens, k_lens, out: dense.attention_args(torch, CPU, q, k, v, None, (-1, -1), 0, q_lens, k_lens, out), attention)}


OPERANDS = [("linear", n) for n in ("x", "weight", "bias", "residual", "out")] + \
           [("rope", n) for n in ("q", "k", "pos", "freqs", "q_weight", "k_weight", "q_out", "k_out")] + [("attention", n) for n in ("q", "k", "v", "out")]


@pytest.mark.parametrize("op,name", OPERANDS)
def test_values_that_are_not_in_memory(op, name):
    call, operands = _calls()[op]
    call(**operands)                                         # as they are they are taken
    t = operands[name]
    with pytest.raises(ValueError, match="negated"):
        call(**{**operands, name: torch._neg_view(t)})
    call(**{**operands, name: torch._neg_view(torch._neg_view(t))})
    with pytest.raises(ValueError, match="no memory"):
        call(**{**operands, name: torch._efficientzerotensor(t.shape, dtype=t.dtype)})
    freed = t.clone()
    freed.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="no memory"):
        call(**{**operands, name: freed})


def test_lazily_conjugated_parts():
    """the imaginary part of a conjugated tensor has the sign of the one before it in memory"""
    call, operands = _calls()["linear"]
    z = torch.randn(4, 1, dtype=torch.complex64)
    operands.update(x=z.conj().imag, weight=torch.randn(6, 1))
    with pytest.raises(ValueError, match="negated"):
        call(**operands)
    call(**{**operands, "x": z.conj().imag.resolve_neg()})
    call(**{**operands, "x": z.conj().real})


@pytest.mark.parametrize("op,name", [o for o in OPERANDS if o[1] != "freqs"])
def test_tangents(op, name):
    import torch.autograd.forward_ad as fwd
    call, operands = _calls()[op]
    with fwd.dual_level():
        call(**operands)                                     # none of them carries one
        with pytest.raises(ValueError, match="tangent"):
            call(**{**operands, name: fwd.make_dual(operands[name], torch.ones_like(operands[name]))})
    call(**operands)


@pytest.mark.parametrize("op", ["linear", "rope", "attention"])
@pytest.mark.parametrize("given_out", [True, False])
def test_tracers(op, given_out):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, operands = _calls()[op]
    outs = [n for n in operands if n in ("out", "q_out", "k_out")]
    ins = {n: t for n, t in operands.items() if n not in outs}
    rest = {n: operands[n] if given_out else None for n in outs}

    def f(*tensors):
        got = call(**dict(zip(ins, tensors)), **rest)
        return got[-1]
    f(*ins.values())
    with pytest.raises(ValueError, match="traced"):
        torch.jit.trace(f, tuple(ins.values()), check_trace=False)
    for mode in ("real", "fake"):
        with pytest.raises(ValueError, match="traced"):
            make_fx(f, tracing_mode=mode)(*ins.values())
    f(*ins.values())


# ------------------------------------------------------------------ operands that share a buffer (the C entry points' checks; a call that passes
# them ends at the null context)
@pytest.fixture(scope="module")
def lib():
    from bufferx_amd import lib as L
    L.build()
    L.load()
    return L


def _refusal(lib, fn, args):
    import ctypes
    assert getattr(lib.load(), fn)(None, None, ctypes.byref(args)) == 1
    said = lib.load().bx_last_error().decode()
    return None if said == "null context" else said


def _linear(lib, **kw):
    a = lib.BxLinearArgs(dtype=2, act=0, M=4, N=8, K=16, ldx=16, ldw=16, ldr=8, ldy=8, x=0x10000, w=0x20000, y=0x50000)
    for k, v in kw.items():
        setattr(a, k, v)
    return _refusal(lib, "bx_linear", a)


def _attention(lib, **kw):
    a = lib.BxAttentionArgs(dtype=0, B=2, Lq=3, Lk=3, Hq=4, Hk=2, D=8, left=-1, right=-1, sinks=0, scale=0.3,
                            q_stride_b=96, q_stride_t=32, q_stride_h=8, k_stride_b=48, k_stride_t=16, k_stride_h=8, v_stride_b=48, v_stride_t=16,
                            v_stride_h=8, o_stride_b=96, o_stride_t=32, o_stride_h=8, q=0x10000, k=0x20000, v=0x30000, o=0x40000)
    for k, v in kw.items():
        setattr(a, k, v)
    return _refusal(lib, "bx_attention", a)


def _strides(name, b, t, h):
    return {f"{name}_stride_b": b, f"{name}_stride_t": t, f"{name}_stride_h": h}


def test_linear_results_beside_their_input(lib):
    """x and y as columns of one buffer of rows [16 | 8], in both orders; one column more and they share an element"""
    assert _linear(lib, ldx=24, ldy=24, y=0x10000 + 16 * 2) is None
    assert _linear(lib, ldx=24, ldy=24, x=0x10000 + 8 * 2, y=0x10000) is None
    assert "overlaps" in _linear(lib, ldx=24, ldy=24, y=0x10000 + 15 * 2)
    assert "overlaps" in _linear(lib, ldx=24, ldy=24, x=0x10000 + 7 * 2, y=0x10000)
    assert "overlaps" in _linear(lib, ldx=24, ldy=25, y=0x10000 + 16 * 2)
    assert _linear(lib, ldr=24, ldy=24, residual=0x50000 + 8 * 2, ldx=24, x=0x50000 + 16 * 2, K=8, ldw=8) is None           # [y | residual | x]
    assert "without being it" in _linear(lib, ldr=24, ldy=24, residual=0x50000 + 6 * 2)
    assert _linear(lib, ldy=16, bias=0x50000 + 8 * 2) is None                      # the bias in the gap behind y's first row
    assert "overlaps" in _linear(lib, ldy=16, bias=0x50000 + 9 * 2)


def test_attention_results_beside_their_inputs(lib):
    # one buffer of rows [q 4 | k 2 | v 2 | o 4] of heads of 8 floats
    at = lambda heads: 0x10000 + 4 * 8 * heads
    one = {**_strides("q", 3 * 96, 96, 8), **_strides("k", 3 * 96, 96, 8), **_strides("v", 3 * 96, 96, 8), **_strides("o", 3 * 96, 96, 8)}
    assert _attention(lib, **one, q=at(0), k=at(4), v=at(6), o=at(8)) is None
    assert _attention(lib, **one, q=at(4), k=at(8), v=at(10), o=at(0)) is None
    assert "overlaps" in _attention(lib, **one, q=at(0), k=at(4), v=at(6), o=at(7))
    # heads of q and o side by side: [q 8 | o 8] per head
    assert _attention(lib, **_strides("q", 192, 64, 16), **_strides("o", 192, 64, 16), o=0x10000 + 32) is None
    assert "overlaps" in _attention(lib, **_strides("q", 192, 64, 16), **_strides("o", 192, 64, 16), o=0x10000 + 28)
    # heads before tokens in memory, q and o in halves of each head's stretch
    assert _attention(lib, **_strides("q", 192, 8, 48), **_strides("o", 192, 8, 48), o=0x10000 + 4 * 24) is None
    # a workspace behind every batch entry is still one stretch of memory
    assert "workspace" in _attention(lib, **_strides("o", 200, 32, 8), workspace=0x40000, workspace_bytes=64)


def test_refusals_find_every_shared_element(lib):
    """random strided operands: what passes shares no element with the output, and parts of one row pass"""
    import itertools
    import random
    rng = random.Random(5)
    cells = lambda p, e, row, dims: {p + e * (sum(i * s for i, s in zip(at, [s for _, s in dims])) + c) + byte
                                     for at in itertools.product(*(range(n) for n, _ in dims)) for c in range(row) for byte in range(e)}
    passed = refused = 0
    for _ in range(3000):
        M, K, N, e = rng.randint(1, 5), rng.randint(1, 6), rng.randint(1, 6), rng.choice([2, 4])
        ldx, ldy = rng.randint(0, 14), rng.randint(N, 14)
        if rng.random() < 0.5:
            ldx = ldy
        x, y = 0x10000 + e * rng.randint(0, 30), 0x10000 + e * rng.randint(0, 30)
        said = _linear(lib, dtype=0 if e == 4 else 1, M=M, N=N, K=K, ldx=ldx, ldw=K, ldy=ldy, x=x, w=0x90000, y=y)
        shared = bool(cells(x, e, K, [(M, ldx)]) & cells(y, e, N, [(M, ldy)]))
        assert said is None or "overlaps" in said, said
        assert not (shared and said is None), (M, K, N, ldx, ldy, x, y)
        passed, refused = passed + (said is None), refused + (said is not None)
        if ldx == ldy and K + N <= ldx and (y - x) % (e * ldx) >= e * K and (y - x) % (e * ldx) + e * N <= e * ldx:
            assert said is None
    assert passed > 500 and refused > 500
    for _ in range(3000):
        B, L, H, D = (rng.randint(1, 3) for _ in range(4))
        order = rng.sample(range(3), 3)
        strides, step = [0, 0, 0], rng.randint(D, 2 * D + 2)
        for i in order:                                      # nested dimensions in any order, with gaps
            strides[i] = step
            step = step * (B, L, H)[i] + rng.randint(0, 6)
        o_strides = strides if rng.random() < 0.7 else [s + rng.randint(0, 3) for s in strides]
        q, o = 0x10000 + 4 * rng.randint(0, 20), 0x10000 + 4 * rng.randint(0, 20)
        said = _attention(lib, B=B, Lq=L, Lk=L, Hq=H, Hk=1, D=D, **_strides("q", *strides), **_strides("o", *o_strides), **_strides("k", 0, 0, 0),
                          **_strides("v", 0, 0, 0), q=q, o=o)
        dims = lambda s: list(zip((B, L, H), s))
        if said is None:
            assert not cells(q, 4, D, dims(strides)) & cells(o, 4, D, dims(o_strides)), (B, L, H, D, strides, o_strides, q, o)
