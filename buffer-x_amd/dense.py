"""Arguments of the dense operators over keypoints (include/bufferx.h bx_linear, bx_qk_norm_rope, bx_attention) from torch tensors:
types, shapes, devices and strides are checked here, overlaps and ranges in the library.  lib.Context.linear / qk_norm_rope / attention
are the calls; nothing here touches the GPU.

Unlike the stage entry points these operators neither convert nor copy what they are given: a tensor of another type, on another
device or with a strided innermost dimension is refused (ValueError).  They have no backward pass and refuse tensors that ask for one.
"""
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


def _operand(torch, name, t, device, dtype, shape):
    """the address of `t`, an operand of this type and shape on this device; its innermost dimension has to be contiguous"""
    try:                                                      # the checks below in one go: a call of a few microseconds pays for each
        if t.dtype is dtype and t.shape == shape and t.device == device and not t.requires_grad and (t.stride(-1) == 1 or shape[-1] <= 1):
            return t.data_ptr()
    except AttributeError:
        pass
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
    return t.data_ptr()


def linear_args(torch, device, x, weight, bias, act, residual, out, m_dev):
    _need(isinstance(x, torch.Tensor) and x.dim() == 2, "x has to be a tensor [M, K]")
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight has to be a tensor [N, K]")
    _need(act in ACTS, f"unknown activation {act!r} (known: {tuple(ACTS)})")
    (M, K), N, dt = x.shape, weight.shape[0], x.dtype
    a = lib.BxLinearArgs()
    a.dtype, a.act, a.M, a.N, a.K = _type(torch, x), ACTS[act], M, N, K
    a.x, a.ldx = _operand(torch, "x", x, device, dt, (M, K)), x.stride(0)
    a.w, a.ldw = _operand(torch, "weight", weight, device, dt, (N, K)), weight.stride(0)
    if bias is not None:
        a.bias = _operand(torch, "bias", bias, device, dt, (N,))
    if residual is not None:
        a.residual, a.ldr = _operand(torch, "residual", residual, device, dt, (M, N)), residual.stride(0)
    if m_dev is not None:
        a.m_dev = _operand(torch, "m_dev", m_dev, device, torch.int32, (1,))
    if out is None:
        out = torch.empty((M, N), dtype=dt, device=device)
    a.y, a.ldy = _operand(torch, "out", out, device, dt, (M, N)), out.stride(0)
    return a, out


def qk_norm_rope_args(torch, device, q, k, pos, freqs, sections, norm, eps, q_weight, k_weight, pairs, q_out, k_out, m_dev):
    _need(norm in NORMS, f"unknown norm {norm!r} (known: {tuple(NORMS)})")
    _need(pairs in PAIRS, f"unknown order of pairs {pairs!r} (known: {tuple(PAIRS)})")
    sections = tuple(int(s) for s in sections)
    _need(1 <= len(sections) <= 4 and min(sections) >= 0, "sections: the rotation pairs of 1 to 4 axes")
    first = q if q is not None else k
    _need(isinstance(first, torch.Tensor) and first.dim() == 3, "q and / or k have to be tensors [T, heads, D]")
    T, _, D = first.shape
    dt = first.dtype
    a = lib.BxQkNormRopeArgs()
    a.dtype, a.norm, a.pairs, a.T, a.D, a.axes, a.eps = _type(torch, first), NORMS[norm], PAIRS[pairs], T, D, len(sections), eps
    for i, s in enumerate(sections):
        a.sections[i] = s
    _need(isinstance(pos, torch.Tensor) and pos.dtype in (torch.float32, torch.int32), "pos has to be a float32 or int32 tensor [T, axes]")
    a.pos_dtype = 0 if pos.dtype is torch.float32 else 1
    a.pos, a.pos_stride_t = _operand(torch, "pos", pos, device, pos.dtype, (T, len(sections))), pos.stride(0)
    a.freqs = _operand(torch, "freqs", freqs, device, torch.float64, (sum(sections),))
    if q is not None:
        _need(isinstance(q, torch.Tensor) and q.dim() == 3, "q has to be a tensor [T, heads, D]")
        shape = (T, q.shape[1], D)
        a.Hq, a.q, a.q_stride_t, a.q_stride_h = shape[1], _operand(torch, "q", q, device, dt, shape), q.stride(0), q.stride(1)
        if q_out is None:
            q_out = torch.empty(shape, dtype=dt, device=device)
        a.q_out, a.q_out_stride_t, a.q_out_stride_h = _operand(torch, "q_out", q_out, device, dt, shape), q_out.stride(0), q_out.stride(1)
        if q_weight is not None:
            a.q_weight = _operand(torch, "q_weight", q_weight, device, dt, (D,))
    else:
        _need(q_out is None and q_weight is None, "q_out and q_weight need q")
    if k is not None:
        _need(isinstance(k, torch.Tensor) and k.dim() == 3, "k has to be a tensor [T, heads, D]")
        shape = (T, k.shape[1], D)
        a.Hk, a.k, a.k_stride_t, a.k_stride_h = shape[1], _operand(torch, "k", k, device, dt, shape), k.stride(0), k.stride(1)
        if k_out is None:
            k_out = torch.empty(shape, dtype=dt, device=device)
        a.k_out, a.k_out_stride_t, a.k_out_stride_h = _operand(torch, "k_out", k_out, device, dt, shape), k_out.stride(0), k_out.stride(1)
        if k_weight is not None:
            a.k_weight = _operand(torch, "k_weight", k_weight, device, dt, (D,))
    else:
        _need(k_out is None and k_weight is None, "k_out and k_weight need k")
    if m_dev is not None:
        a.m_dev = _operand(torch, "m_dev", m_dev, device, torch.int32, (1,))
    return a, q_out, k_out


def attention_args(torch, device, q, k, v, scale, window, sinks, q_lens, k_lens, out):
    _need(isinstance(q, torch.Tensor) and q.dim() == 4, "q has to be a tensor [B, Lq, heads, D]")
    _need(isinstance(k, torch.Tensor) and k.dim() == 4, "k has to be a tensor [B, Lk, heads, D]")
    B, Lq, Hq, D = q.shape
    Lk, Hk, dt = k.shape[1], k.shape[2], q.dtype
    a = lib.BxAttentionArgs()
    a.dtype, a.B, a.Lq, a.Lk, a.Hq, a.Hk, a.D = _type(torch, q), B, Lq, Lk, Hq, Hk, D
    a.left, a.right = (max(-1, min(int(w), 2**31 - 1)) for w in window)
    a.sinks = min(int(sinks), 2**31 - 1)
    a.scale = D ** -0.5 if scale is None and D > 0 else float(scale or 0.0)
    a.q = _operand(torch, "q", q, device, dt, (B, Lq, Hq, D))
    a.k = _operand(torch, "k", k, device, dt, (B, Lk, Hk, D))
    a.v = _operand(torch, "v", v, device, dt, (B, Lk, Hk, D))
    a.q_stride_b, a.q_stride_t, a.q_stride_h, _ = q.stride()
    a.k_stride_b, a.k_stride_t, a.k_stride_h, _ = k.stride()
    a.v_stride_b, a.v_stride_t, a.v_stride_h, _ = v.stride()
    if q_lens is not None:
        a.q_lens = _operand(torch, "q_lens", q_lens, device, torch.int32, (B,))
    if k_lens is not None:
        a.k_lens = _operand(torch, "k_lens", k_lens, device, torch.int32, (B,))
    if out is None:
        out = torch.empty((B, Lq, Hq, D), dtype=dt, device=device)
    a.o = _operand(torch, "out", out, device, dt, (B, Lq, Hq, D))
    a.o_stride_b, a.o_stride_t, a.o_stride_h, _ = out.stride()
    return a, out
