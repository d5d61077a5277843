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
