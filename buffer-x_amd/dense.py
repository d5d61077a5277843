"""Arguments of the dense operators over keypoints (include/bufferx.h bx_linear, bx_qk_norm_rope, bx_attention) from torch tensors:
types, shapes, devices and strides are checked here, overlaps and ranges in the library.  lib.Context.linear / qk_norm_rope / attention
are the calls; nothing here touches the GPU.

Unlike the stage entry points these operators neither convert nor copy what they are given: a tensor of another type, on another
device, with a strided innermost dimension or whose memory does not hold its values is refused (ValueError).  They have no derivatives and
refuse tensors that ask for one, and they are nothing that a tracer can record.
"""
import sys

from . import lib

ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
NORMS = {"none": 0, "rms": 1, "l2": 2}
PAIRS = {"half": 0, "interleaved": 1}
_TYPES = {}


def _type(torch, t):
    if not _TYPES:
        _TYPES.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"type {t.dtype} is not float32, float16 or bfloat16")
    return code


def _need(ok, what):
    if not ok:
        raise ValueError(what)


_STATE = []


def _eager(torch):
    """refuses what would see only the tensors around a call and not the call: a tracer would record an output that nothing writes.  Returns the
    check that its operands need."""
    if not _STATE:
        from torch.autograd import forward_ad
        _STATE.extend((torch.jit.is_tracing, forward_ad))
    if _STATE[0]():
        raise ValueError("these operators cannot be traced (torch.jit.trace)")
    proxy = sys.modules.get("torch.fx.experimental.proxy_tensor")             # (not there: nobody traces with it)
    if proxy is not None and proxy.get_proxy_mode() is not None:
        raise ValueError("these operators cannot be traced (make_fx)")
    # (a level of 0 and more: forward-mode derivatives are being taken)
    return _operand if getattr(_STATE[1], "_current_level", 0) < 0 else _checked


def _operand(torch, name, t, device, dtype, shape):
    """the address of `t`, an operand of this type and shape on this device; its innermost dimension has to be contiguous"""
    try:                                                      # the checks below in one go: a call of a few microseconds pays for each
        if (t.dtype is dtype and t.shape == shape and t.device == device and not t.requires_grad and (t.stride(-1) == 1 or shape[-1] <= 1) and
                not t.is_neg()):
            at = t.data_ptr()
            if at:
                return at
    except AttributeError:
        pass
    return _checked(torch, name, t, device, dtype, shape)


def _checked(torch, name, t, device, dtype, shape):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} is not a tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the context is on {device}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} has type {t.dtype}, expected {dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the innermost dimension has to be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: these operators have no backward pass (use torch.no_grad() or detach())")
    if _STATE[1].unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent: these operators have no derivatives")
    if t.is_neg():
        raise ValueError(f"{name} is a negated view, whose memory holds other values (use resolve_neg())")
    at = t.data_ptr()
    if not at and t.numel():
        raise ValueError(f"{name} has no memory")
    return at


def _sized(torch, name, t, dims, what):
    if not (isinstance(t, torch.Tensor) and t.dim() == dims):
        raise ValueError(f"{name} has to be a tensor {what}")
    return t.shape


def linear_args(torch, device, x, weight, bias, act, residual, out, m_dev):
    operand = _eager(torch)
    M, K = _sized(torch, "x", x, 2, "[M, K]")
    N = _sized(torch, "weight", weight, 2, "[N, K]")[0]
    dt, code = x.dtype, _type(torch, x)
    if act not in ACTS:
        raise ValueError(f"unknown activation {act!r} (known: {tuple(ACTS)})")
    px, pw = operand(torch, "x", x, device, dt, (M, K)), operand(torch, "weight", weight, device, dt, (N, K))
    pb = None if bias is None else operand(torch, "bias", bias, device, dt, (N,))
    pr, ldr = (None, 0) if residual is None else (operand(torch, "residual", residual, device, dt, (M, N)), residual.stride(0))
    pm = None if m_dev is None else operand(torch, "m_dev", m_dev, device, torch.int32, (1,))
    if out is None:
        out = torch.empty((M, N), dtype=dt, device=device)
        py, ldy = out.data_ptr(), N
    else:
        py, ldy = operand(torch, "out", out, device, dt, (M, N)), out.stride(0)
    return lib.BxLinearArgs(code, ACTS[act], M, N, K, x.stride(0), weight.stride(0), ldr, ldy, px, pw, pb, pr, py, pm), out


def _heads(operand, torch, name, t, weight, out, device, dt, T, D):
    """(heads, address, token and head stride, weight's address, out, its address and strides) of q or k; absent: all zero"""
    if t is None:
        if out is not None or weight is not None:
            raise ValueError(f"{name}_out and {name}_weight need {name}")
        return 0, None, 0, 0, None, None, None, 0, 0
    H = _sized(torch, name, t, 3, "[T, heads, D]")[1]
    _need(H < 2**31 and D < 2**31, "sizes of 2^31 or more")
    at = operand(torch, name, t, device, dt, (T, H, D))
    w = None if weight is None else operand(torch, name + "_weight", weight, device, dt, (D,))
    st, sh, _ = t.stride()
    if out is None:
        out = torch.empty((T, H, D), dtype=dt, device=device)
        return H, at, st, sh, w, out, out.data_ptr(), H * D, D
    ot, oh, _ = out.stride() if isinstance(out, torch.Tensor) and out.dim() == 3 else (0, 0, 0)
    return H, at, st, sh, w, out, operand(torch, name + "_out", out, device, dt, (T, H, D)), ot, oh


def qk_norm_rope_args(torch, device, q, k, pos, freqs, sections, norm, eps, q_weight, k_weight, pairs, q_out, k_out, m_dev):
    operand = _eager(torch)
    if norm not in NORMS:
        raise ValueError(f"unknown norm {norm!r} (known: {tuple(NORMS)})")
    if pairs not in PAIRS:
        raise ValueError(f"unknown order of pairs {pairs!r} (known: {tuple(PAIRS)})")
    axes = len(sections)
    _need(1 <= axes <= 4 and 0 <= min(sections) and max(sections) < 2**31, "sections: the rotation pairs of 1 to 4 axes")
    first = q if q is not None else k
    T, _, D = _sized(torch, "q (or k, where q is None)", first, 3, "[T, heads, D]")
    dt, code = first.dtype, _type(torch, first)
    is_i32 = isinstance(pos, torch.Tensor) and pos.dtype is torch.int32
    pp = operand(torch, "pos (float32 or int32)", pos, device, torch.int32 if is_i32 else torch.float32, (T, axes))
    pf = operand(torch, "freqs", freqs, device, torch.float64, (sum(sections),))
    pm = None if m_dev is None else operand(torch, "m_dev", m_dev, device, torch.int32, (1,))
    Hq, aq, qt, qh, wq, q_out, oq, oqt, oqh = _heads(operand, torch, "q", q, q_weight, q_out, device, dt, T, D)
    Hk, ak, kt, kh, wk, k_out, ok, okt, okh = _heads(operand, torch, "k", k, k_weight, k_out, device, dt, T, D)
    return lib.BxQkNormRopeArgs(code, NORMS[norm], PAIRS[pairs], int(is_i32), T, Hq, Hk, D, axes, tuple(sections), eps, 0, qt, qh, kt, kh, oqt, oqh, okt,
                                okh, pos.stride(0), aq, ak, wq, wk, pp, pf, oq, ok, pm), q_out, k_out


def attention_args(torch, device, q, k, v, scale, window, sinks, q_lens, k_lens, out):
    operand = _eager(torch)
    B, Lq, Hq, D = _sized(torch, "q", q, 4, "[B, Lq, heads, D]")
    _, Lk, Hk, _ = _sized(torch, "k", k, 4, "[B, Lk, heads, D]")
    dt, code, big = q.dtype, _type(torch, q), 2**31 - 1
    left, right = window
    _need(max(B, Lq, Lk, Hq, Hk, D) <= big, "sizes of 2^31 or more")          # (what the structure's 32 bits would cut off is seen here)
    left, right, sinks = (max(-1, min(int(n), big)) for n in (left, right, sinks))
    scale = float(scale) if scale is not None else D ** -0.5 if D > 0 else 0.0
    pq = operand(torch, "q", q, device, dt, (B, Lq, Hq, D))
    pk, pv = operand(torch, "k", k, device, dt, (B, Lk, Hk, D)), operand(torch, "v", v, device, dt, (B, Lk, Hk, D))
    pql = None if q_lens is None else operand(torch, "q_lens", q_lens, device, torch.int32, (B,))
    pkl = None if k_lens is None else operand(torch, "k_lens", k_lens, device, torch.int32, (B,))
    if out is None:
        out = torch.empty((B, Lq, Hq, D), dtype=dt, device=device)
        po = out.data_ptr()
    else:
        po = operand(torch, "out", out, device, dt, (B, Lq, Hq, D))
    return lib.BxAttentionArgs(code, B, Lq, Lk, Hq, Hk, D, left, right, sinks, scale, 0, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                               *out.stride()[:3], pq, pk, pv, po, pql, pkl, None, 0), out
