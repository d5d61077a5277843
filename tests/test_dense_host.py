"""Refusals of the dense operators over keypoints (bx_linear, bx_qk_norm_rope, bx_attention) without a GPU: the tensor checks of
bufferx_amd.dense on CPU tensors, and the argument checks of the C entry points, which come before the context is looked at -- a call
that passes them ends at the null context, one that does not names its fault."""
import ctypes as C

import pytest
import torch

CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def lib():
    from bufferx_amd import lib as L
    L.build()
    L.load()
    return L


def _ends(lib, fn, args):
    rc = getattr(lib.load(), fn)(None, None, C.byref(args))
    return rc, lib.load().bx_last_error().decode()


def _linear(lib, **kw):
    a = lib.BxLinearArgs(dtype=2, act=0, M=4, N=8, K=16, ldx=16, ldw=16, ldr=8, ldy=8, x=0x10000, w=0x20000, bias=0x30000, residual=0x40000,
                         y=0x50000)
    for k, v in kw.items():
        setattr(a, k, v)
    return _ends(lib, "bx_linear", a)


@pytest.mark.parametrize("kw", [{}, dict(ldx=0), dict(ldw=0, ldr=0), dict(residual=0x50000), dict(M=0, x=None, y=None), dict(N=0, y=None),
                                dict(K=0, x=None, w=None), dict(bias=None, residual=None), dict(ldx=20, ldy=9), dict(x=0x10002), dict(M=1, ldy=0),
                                dict(m_dev=0x60000)])
def test_linear_accepts(lib, kw):
    rc, msg = _linear(lib, **kw)
    assert rc == 1 and msg == "null context"


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=3), "type"), (dict(dtype=-1), "type"), (dict(act=4), "activation"), (dict(M=-1), "range"), (dict(K=2**31), "range"), (dict(M=2**30 + 1), "range"), (dict(K=2**30 + 1), "range"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(ldx=-1), "stride"), (dict(ldy=7), "overlap"),
    (dict(ldx=2**50), "stride"), (dict(x=0x10001), "aligned"), (dict(m_dev=0x60002), "aligned"), (dict(y=0x10000), "overlaps"),
    (dict(y=0x20010), "overlaps"), (dict(y=0x30000), "overlaps"), (dict(residual=0x50002), "residual"), (dict(residual=0x50000, ldr=9), "residual"),
    (dict(m_dev=0x50008), "overlaps")])
def test_linear_refuses(lib, kw, says):
    rc, msg = _linear(lib, **kw)
    assert rc == 1 and says in msg, msg


def _rope(lib, sections=(3, 2, 2), **kw):
    a = lib.BxQkNormRopeArgs(dtype=0, norm=1, pairs=0, pos_dtype=0, T=5, Hq=4, Hk=2, D=16, axes=len(sections), eps=1e-6,
                             q_stride_t=64, q_stride_h=16, k_stride_t=32, k_stride_h=16, q_out_stride_t=64, q_out_stride_h=16, k_out_stride_t=32,
                             k_out_stride_h=16, pos_stride_t=3, q=0x10000, k=0x20000, q_weight=0x30000, k_weight=0x31000, pos=0x32000, freqs=0x33000,
                             q_out=0x40000, k_out=0x50000)
    for i, s in enumerate(sections):
        a.sections[i] = s
    for k, v in kw.items():
        setattr(a, k, v)
    return _ends(lib, "bx_qk_norm_rope", a)


# one buffer of rows [q heads 0..3 | k heads 0..1 | v heads 0..1]: 8 heads of 16 floats, rotated in place
PACKED = dict(q_stride_t=128, k_stride_t=128, q_out_stride_t=128, k_out_stride_t=128, k=0x10000 + 4 * 64, q_out=0x10000, k_out=0x10000 + 4 * 64)


@pytest.mark.parametrize("kw", [{}, dict(k=None, k_out=None), dict(q=None, q_out=None), dict(q_out=0x10000), dict(T=0), dict(norm=0, q_weight=None),
                                PACKED, dict(sections=(8,)), dict(sections=(0,), pos=None, freqs=None), dict(sections=(2, 2, 2, 2)), dict(q_stride_t=0),
                                dict(pos_stride_t=0), dict(eps=0.0)])
def test_rope_accepts(lib, kw):
    rc, msg = _rope(lib, **kw)
    assert rc == 1 and msg == "null context"


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=7), "type"), (dict(norm=3), "norm"), (dict(pairs=2), "pairs"), (dict(pos_dtype=2), "positions"), (dict(D=0), "D="),
    (dict(D=257), "D="), (dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(sections=(3, -1)), "negative"), (dict(sections=(5, 4)), "fit"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"), (dict(T=-1), "range"), (dict(q_out=None), "null"),
    (dict(pos=None), "null"), (dict(freqs=None), "null"), (dict(freqs=0x33004), "aligned"), (dict(q=0x10002), "aligned"), (dict(reserved=1), "reserved"),
    (dict(k_stride_t=-4), "stride"), (dict(q_out_stride_h=15), "overlap"), (dict(q_out_stride_t=0), "overlap"), (dict(q_out=0x10040), "without being it"),
    (dict(q_out=0x20000), "without being it"), (dict(q_out=0x10000, q_out_stride_t=65), "without being it"), (dict(k_out=0x40000), "outputs overlap"),
    (dict(q_out=0x32000), "overlaps an input"), (dict(PACKED, k_out=0x10000 + 3 * 64), "overlap")])
def test_rope_refuses(lib, kw, says):
    rc, msg = _rope(lib, **kw)
    assert rc == 1 and says in msg, msg


def _attention(lib, **kw):
    a = lib.BxAttentionArgs(dtype=0, B=2, Lq=3, Lk=5, Hq=4, Hk=2, D=8, left=-1, right=-1, sinks=0, scale=0.3,
                            q_stride_b=96, q_stride_t=32, q_stride_h=8, k_stride_b=80, k_stride_t=16, k_stride_h=8, v_stride_b=80, v_stride_t=16,
                            v_stride_h=8, o_stride_b=96, o_stride_t=32, o_stride_h=8, q=0x10000, k=0x20000, v=0x30000, o=0x40000, q_lens=0x50000,
                            k_lens=0x51000)
    for k, v in kw.items():
        setattr(a, k, v)
    return _ends(lib, "bx_attention", a)


@pytest.mark.parametrize("kw", [{}, dict(q_lens=None, k_lens=None), dict(Lk=0, k=None, v=None), dict(B=0), dict(Lq=0), dict(left=2**31 - 1, right=2**31 - 1),
                                dict(k_stride_b=0, v_stride_b=0), dict(o_stride_h=24, o_stride_t=8), dict(v=0x20000), dict(D=1), dict(D=128, q_stride_h=0,
                                k_stride_h=0, v_stride_h=0, o_stride_h=128, o_stride_t=512, o_stride_b=1536)])
def test_attention_accepts(lib, kw):
    rc, msg = _attention(lib, **kw)
    assert rc == 1 and msg == "null context"


@pytest.mark.parametrize("kw,says", [
    (dict(dtype=3), "type"), (dict(D=0), "D="), (dict(D=129), "D="), (dict(Hq=3), "share"), (dict(Hk=0), "share"), (dict(Lk=-1), "range"),
    (dict(Lk=2**30), "range"), (dict(Lq=2**29, Hq=4), "range"), (dict(sinks=-1), "negative"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=2.0**101), "scale"), (dict(scale=2.0**-101), "scale"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(o=None), "null"),
    (dict(v_stride_t=-1), "stride"), (dict(q=0x10001), "aligned"), (dict(k_lens=0x51002), "aligned"), (dict(workspace=0x60008, workspace_bytes=64), "aligned"),
    (dict(o_stride_h=7), "rows of o"), (dict(o_stride_b=0), "rows of o"), (dict(o=0x10000), "overlaps"), (dict(o=0x30010), "overlaps"),
    (dict(workspace=0x40000, workspace_bytes=64), "workspace"), (dict(workspace=0x20000, workspace_bytes=64), "workspace"), (dict(reserved=1), "reserved")])
def test_attention_refuses(lib, kw, says):
    rc, msg = _attention(lib, **kw)
    assert rc == 1 and says in msg, msg


def test_attention_workspace_refuses(lib):
    so = lib.load()
    assert so.bx_attention_workspace(None, None) == -1


def test_null_arguments(lib):
    for fn in ("bx_linear", "bx_qk_norm_rope", "bx_attention"):
        assert getattr(lib.load(), fn)(None, None, None) == 1 and b"null" in lib.load().bx_last_error()


# ------------------------------------------------------------------ tensor checks
def _t(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype)


def test_linear_tensors():
    from bufferx_amd import dense
    call = lambda x, w, bias=None, act="none", residual=None, out=None, m_dev=None, device=CPU: dense.linear_args(torch, device, x, w, bias, act, residual, out, m_dev)
    a, out = call(_t(4, 6)[:, 1:], _t(8, 5), _t(8), "gelu", _t(4, 8))
    assert (a.M, a.N, a.K, a.ldx, a.ldw, a.ldr, a.ldy, a.dtype, a.act) == (4, 8, 5, 6, 5, 8, 8, 1, 2) and out.shape == (4, 8) and out.dtype == torch.float16
    for bad in (lambda: call(_t(4, 5, 1), _t(8, 5)), lambda: call(_t(4, 5), _t(8, 6)), lambda: call(_t(4, 5), _t(8, 5), act="tanh"),
                lambda: call(_t(4, 5), _t(8, 5, dtype=torch.float32)), lambda: call(_t(4, 5, dtype=torch.float64), _t(8, 5, dtype=torch.float64)),
                lambda: call(_t(4, 5), _t(5, 8).t()), lambda: call(_t(4, 5), _t(8, 5), _t(7)), lambda: call(_t(4, 5), _t(8, 5), residual=_t(8)),
                lambda: call(_t(4, 5), _t(8, 5), m_dev=torch.zeros(1, dtype=torch.int64)), lambda: call(_t(4, 5), _t(8, 5), out=_t(4, 8, dtype=torch.float32)),
                lambda: call(_t(4, 5), _t(8, 5), device=torch.device("cuda", 0)), lambda: call(_t(4, 5), _t(8, 5).requires_grad_()),
                lambda: call([[1.0]], _t(8, 5))):
        with pytest.raises(ValueError):
            bad()
    with torch.no_grad():
        call(_t(4, 5), _t(8, 5).requires_grad_())


def test_rope_tensors():
    from bufferx_amd import dense
    f64 = lambda n: torch.ones(n, dtype=torch.float64)
    call = lambda q, k, pos, freqs, sections, norm="rms", eps=1e-6, qw=None, kw=None, pairs="half", qo=None, ko=None, m=None: dense.qk_norm_rope_args(
        torch, CPU, q, k, pos, freqs, sections, norm, eps, qw, kw, pairs, qo, ko, m)
    pos = torch.zeros(7, 2)
    rows = _t(7, 5, 12)
    a, qo, ko = call(rows[:, :3], rows[:, 3:4], pos, f64(5), (2, 3))
    assert (a.T, a.Hq, a.Hk, a.D, a.axes, a.q_stride_t, a.k_stride_h, a.q_out_stride_t) == (7, 3, 1, 12, 2, 60, 12, 36) and ko.shape == (7, 1, 12)
    a, qo, ko = call(None, rows, pos, f64(5), (2, 3))
    assert qo is None and a.Hq == 0 and a.Hk == 5
    for bad in (lambda: call(None, None, pos, f64(5), (2, 3)), lambda: call(rows, None, pos, f64(4), (2, 3)), lambda: call(rows, None, pos[:, :1], f64(5), (2, 3)),
                lambda: call(rows, None, pos.double(), f64(5), (2, 3)), lambda: call(rows, None, pos, f64(5).float(), (2, 3)),
                lambda: call(rows, None, pos, f64(5), (2, 3), norm="layer"), lambda: call(rows, None, pos, f64(5), (2, 3), pairs="quarter"),
                lambda: call(rows, None, pos, f64(5), (2, 3), kw=_t(12)), lambda: call(rows, None, pos, f64(5), (2, 3), qw=_t(3, 12)),
                lambda: call(rows, _t(6, 5, 12), pos, f64(5), (2, 3)), lambda: call(rows, rows.float(), pos, f64(5), (2, 3)),
                lambda: call(rows, None, pos, f64(5), ()), lambda: call(rows.transpose(1, 2), None, pos, f64(5), (2, 3))):
        with pytest.raises(ValueError):
            bad()


def test_attention_tensors():
    from bufferx_amd import dense
    call = lambda q, k, v, scale=None, window=(-1, -1), sinks=0, ql=None, kl=None, out=None: dense.attention_args(torch, CPU, q, k, v, scale, window, sinks, ql, kl, out)
    rows = _t(2, 9, 8, 16)
    q, k, v = rows[:, :, :4], rows[:, :, 4:6], rows[:, :, 6:]
    a, out = call(q, k, v, window=(5, 0), sinks=2)
    assert (a.B, a.Lq, a.Lk, a.Hq, a.Hk, a.D, a.left, a.right, a.sinks, a.k_stride_t, a.o_stride_t) == (2, 9, 9, 4, 2, 16, 5, 0, 2, 128, 64)
    assert abs(a.scale - 0.25) < 1e-7
    a, _ = call(q, k, v, window=(-7, 2**40))
    assert (a.left, a.right) == (-1, 2**31 - 1)
    for bad in (lambda: call(q[0], k, v), lambda: call(q, k, v[:, :5]), lambda: call(q, k, v.float()), lambda: call(q, k[:1], v[:1]),
                lambda: call(q, k, v, ql=torch.zeros(3, dtype=torch.int32)), lambda: call(q, k, v, kl=torch.zeros(2)), lambda: call(q, k, v, out=_t(2, 9, 4, 15)),
                lambda: call(q.transpose(2, 3), k, v), lambda: call(q.clone().requires_grad_(), k, v)):
        with pytest.raises(ValueError):
            bad()


def test_sizes_beyond_the_structures():
    """what 32 bits of the argument structs would cut off: expanded tensors reach such sizes with one element of memory"""
    from bufferx_amd import dense
    far = 2**32 + 1
    attention = lambda q, k, sinks=0: dense.attention_args(torch, CPU, q, k, k, None, (-1, -1), sinks, None, None, _t(1, 1, 1, 8).expand(q.shape))
    one = _t(1, 1, 1, 8)
    for q, k in ((one, one.expand(1, far, 1, 8)), (one.expand(1, far, 1, 8), one), (one.expand(far, 1, 1, 8), one.expand(far, 1, 1, 8)), (one.expand(1, 1, far, 8), one)):
        with pytest.raises(ValueError):
            attention(q, k)
    assert attention(one, one, sinks=-2**32)[0].sinks == -1            # which the library refuses
    assert attention(one, one, sinks=2**32)[0].sinks == 2**31 - 1
    q = _t(1, 1, 8).expand(1, far, 8)
    with pytest.raises(ValueError):
        dense.qk_norm_rope_args(torch, CPU, q, None, torch.zeros(1, 1), torch.ones(4, dtype=torch.float64), (4,), "rms", 1e-6, None, None, "half", q, None, None)
    with pytest.raises(ValueError):
        dense.qk_norm_rope_args(torch, CPU, q[:, :1], None, torch.zeros(1, 1), torch.ones(4, dtype=torch.float64), (far,), "rms", 1e-6, None, None, "half", None, None, None)


def test_struct_layouts_match_header(lib):
    """ctypes mirrors of the three argument structs: size and the offset of every field, from a C program compiled against the header."""
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    structs = {"bx_linear_args": lib.BxLinearArgs, "bx_qk_norm_rope_args": lib.BxQkNormRopeArgs, "bx_attention_args": lib.BxAttentionArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "bufferx.h"', "int main(void) {"]
    for name, cls in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for f, _ in cls._fields_]
    lines.append("return 0; }")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "o.c"), os.path.join(d, "o")
        open(src, "w").write("\n".join(lines))
        subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(root, "include"), src, "-o", exe])
        got = dict(l.split() for l in subprocess.check_output([exe], text=True).splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (name, f)]) == getattr(cls, f).offset, (name, f)
