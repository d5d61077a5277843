"""Timed cases of the dense operators over keypoints: the linear layer, the norm of queries and keys with a rotation by position, and attention.

They are the parts of a layer that lets the keypoint descriptors of two clouds see each other before they are matched.  `own` selects
the framework's calls (bufferx_amd.lib.Context); without it the same passes run as elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_DEVICE = "cuda:0"
_HELD = {}


def _context():
    """The handle that a program keeps for its device (a small one: these operators need none of the registration workspace)."""
    if "context" not in _HELD:
        import bufferx_amd
        from bufferx_amd import lib
        cfg = bufferx_amd.make_cfg("3DMatch")
        cfg.patch.num_fps, cfg.patch.num_points_per_patch, cfg.patch.num_scales = 64, 64, 1
        cfg.patch.search_radius_thresholds = [2]
        cfg.patch.num_points_radius_estimate = 64
        _HELD["context"] = lib.Context(cfg, max_points=1024, device=0)
    return _HELD["context"]


# ---------------------------------------------------------------------------------------------------------------- the cases
def _linear(name, dtype, m, k, n, act="none", bias=True, residual=False, live=-1, pad=0):
    """x [m, k] times weight [n, k]; `live` rows of the m are filled (-1: all), rows of x lie k + pad elements apart."""
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual,
            "live": live, "pad": pad}


def _rope(name, dtype, tokens, q_heads, k_heads, dim, norm, weight, pairs, pos, sec0, sec1=0, sec2=0, packed=False):
    """Rotation pairs of each axis in sec0..sec2 (0: the axis is absent); `packed`: q and k are parts of one projection's rows."""
    return {"name": name, "op": "rope", "dtype": dtype, "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim, "norm": norm,
            "weight": weight, "pairs": pairs, "pos": pos, "sec0": sec0, "sec1": sec1, "sec2": sec2, "packed": packed}


def _attention(name, dtype, batch, q_len, k_len, q_heads, k_heads, dim, left=-1, right=-1, sinks=0, ragged=False, packed=False):
    """`ragged`: batch entry b has its own, shorter lengths (see _lens); `packed`: q, k and v are parts of one projection's rows."""
    return {"name": name, "op": "attention", "dtype": dtype, "batch": batch, "q_len": q_len, "k_len": k_len, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "left": left, "right": right, "sinks": sinks, "ragged": ragged, "packed": packed}


def listed():
    return [
        # one descriptor through one layer: the latency of a call, and the rate at which the weights are read
        _linear("linear_one_row", "bf16", 1, 1024, 1024),
        # the keypoints of both clouds (5000 each) through a hidden layer with its skip connection
        _linear("linear_keypoints", "f32", 10000, 256, 256, act="relu", residual=True),
        # every position of the equivariant maps (7 x 20 of 5000 patches) through a pointwise layer: bound by memory
        _linear("linear_maps", "f32", 700000, 32, 64, act="relu"),
        # sizes that divide nothing, a count on the device that fills part of the rows, rows that lie apart
        _linear("linear_odd", "f16", 4871, 333, 517, act="silu", residual=True, live=4500, pad=3),
        # a wide hidden layer over a batch of clouds: bound by the matrix units
        _linear("linear_wide", "bf16", 16384, 1024, 4096, act="gelu"),
        # one new token of a sequence far out
        _rope("rope_one_token", "bf16", 1, 32, 8, 128, "rms", True, "half", "sequence", 64),
        # the keypoints of both clouds, rotated by their metric coordinates along three axes
        _rope("rope_keypoints", "f32", 10000, 8, 8, 32, "l2", False, "interleaved", "metric", 6, 5, 5),
        # many frames of a grid (time, height, width), q and k inside one projection's rows, part of each head left unrotated
        _rope("rope_frames", "bf16", 65536, 16, 4, 128, "rms", True, "half", "frames", 16, 20, 20, packed=True),
        # one query against a long store of keys that shares each key head among four query heads
        _attention("attention_one_query", "bf16", 1, 1, 32768, 32, 8, 128, left=8191, right=0, sinks=4),
        # the keypoints of two clouds against each other's, with the counts of each on the device
        _attention("attention_clouds", "f32", 2, 5000, 5000, 8, 8, 32, ragged=True),
        # the 140 positions of each patch among themselves, in a band of neighbours and with the first position always seen
        _attention("attention_patches", "f16", 1500, 140, 140, 2, 1, 32, left=24, right=24, sinks=1, packed=True),
        # a long sequence in a causal window with its first tokens always seen
        _attention("attention_window", "bf16", 1, 32768, 32768, 16, 4, 128, left=1023, right=0, sinks=4, packed=True),
    ]


def _log(rng, low, high):
    """A size whose logarithm is uniform over [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "rope", "attention"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "linear":
        k, n = _log(rng, 8, 2048), _log(rng, 8, 4096)
        m = _log(rng, 1, max(1, min(700000, (1 << 35) // (k * n), (1 << 27) // (k + n))))
        case = _linear("", dtype, m, k, n, act=rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.8,
                       residual=rng.random() < 0.5, live=rng.randint(0, m) if rng.random() < 0.3 else -1, pad=rng.choice([0, 0, 1, 8]))
    elif op == "rope":
        dim = 2 * rng.randint(4, 64)
        k_heads = rng.choice([1, 2, 3, 4, 8])
        q_heads = k_heads * rng.choice([1, 2, 4])
        tokens = _log(rng, 1, min(200000, (1 << 27) // (dim * (q_heads + k_heads))))
        room = dim // 2
        sec0 = rng.randint(1, room)
        sec1 = rng.randint(0, room - sec0)
        sec2 = rng.randint(0, room - sec0 - sec1) if sec1 else 0
        case = _rope("", dtype, tokens, q_heads, k_heads, dim, rng.choice(["none", "rms", "l2"]), rng.random() < 0.5,
                     rng.choice(["half", "interleaved"]), rng.choice(["sequence", "metric", "frames"]), sec0, sec1, sec2,
                     packed=rng.random() < 0.5)
    else:
        dim = rng.choice([20, 32, 40, 64, 80, 96, 128, rng.randint(8, 128)])
        k_heads = rng.choice([1, 2, 3, 4])
        q_heads = k_heads * rng.choice([1, 2, 3, 4])
        if rng.random() < 0.3:
            batch, q_len, k_len = rng.randint(1, 8), rng.randint(1, 3), _log(rng, 1, 32768)
            left, right, sinks = rng.choice([(-1, 0, 0), (_log(rng, 16, 8192) - 1, 0, rng.randint(0, 8))])
        else:
            q_len = _log(rng, 1, 6000)
            left, right, sinks = rng.choice([(-1, -1, 0), (-1, 0, 0), (_log(rng, 8, 2048) - 1, 0, rng.randint(0, 8)),
                                             (_log(rng, 8, 512), _log(rng, 8, 512), rng.randint(0, 8))])
            k_len = q_len if rng.random() < 0.6 else _log(rng, 1, 6000)
            batch = _log(rng, 1, max(1, min(1000, 400000000 // (q_heads * q_len * k_len + 1), (1 << 24) // (q_len * q_heads * dim + 1))))
        packed = q_len == k_len and rng.random() < 0.5
        case = _attention("", dtype, batch, q_len, k_len, q_heads, k_heads, dim, left, right, sinks, ragged=rng.random() < 0.4, packed=packed)
    del case["name"]
    return case


def _sections(case):
    return [s for s in (case["sec0"], case["sec1"], case["sec2"]) if s]


def _lens(case):
    """Query and key lengths of each batch entry, as numpy arrays; they go by the case alone."""
    b = np.arange(case["batch"], dtype=np.int64)
    q, k = np.full(len(b), case["q_len"], np.int64), np.full(len(b), case["k_len"], np.int64)
    if case["ragged"]:
        q = np.maximum(1, q - (q * (5 * b % 17)) // 64)
        k = np.maximum(1, k - (k * (7 * b % 13)) // 64)
    return q, k


def _visible(case):
    """How many (query, key) pairs the mask leaves, and how many keys of each batch entry any query sees."""
    pairs = keys = 0
    q_lens, k_lens = _lens(case)
    for (ql, kl), times in zip(*np.unique(np.stack([q_lens, k_lens], 1), axis=0, return_counts=True)):
        p = np.arange(ql) + (kl - ql)
        high = np.minimum(kl, p + 1 + case["right"]) if case["right"] >= 0 else np.full(ql, kl)
        low = np.maximum(0, p - case["left"]) if case["left"] >= 0 else np.zeros(ql, np.int64)
        first = np.minimum(min(case["sinks"], kl), np.minimum(low, np.maximum(high, 0)))
        band = np.maximum(0, high - low)
        pairs += int(times) * int((band + np.maximum(0, first)).sum())
        seen = np.zeros(kl + 1, np.int64)
        some = band > 0
        np.add.at(seen, low[some], 1)
        np.add.at(seen, high[some], -1)
        covered = np.cumsum(seen)[:kl] > 0
        covered[:max(0, int(first.max()))] = True
        keys += int(times) * int(covered.sum())
    return pairs, keys


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = (case["live"] if case["live"] >= 0 else case["m"]), case["k"], case["n"]
        moved = m * k + k * n + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        return {"bytes": e * moved, "flops": 2 * m * k * n}
    if case["op"] == "rope":
        values = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": 2 * e * values + 4 * case["tokens"] * len(_sections(case)), "flops": 8 * values}
    pairs, keys = _visible(case)
    q_lens, _ = _lens(case)
    moved = 2 * int(q_lens.sum()) * case["q_heads"] + 2 * keys * case["k_heads"]
    return {"bytes": e * moved * case["dim"], "flops": 4 * pairs * case["q_heads"] * case["dim"]}


# ---------------------------------------------------------------------------------------------------------------- the inputs
def _normal(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=_DEVICE, dtype=torch.float32) * scale).to(dtype)


def _positions(case, gen, seed):
    """[tokens, axes]: whole numbers along a sequence or a grid of frames, or metric coordinates in a room."""
    tokens, axes = case["tokens"], len(_sections(case))
    if case["pos"] == "metric":
        return torch.rand((tokens, axes), generator=gen, device=_DEVICE) * 6.0 - 2.0
    at = torch.arange(tokens, device=_DEVICE, dtype=torch.int32)
    if case["pos"] == "sequence":
        return (at[:, None] + (100000 + 13 * (seed % 1000))).repeat(1, axes).contiguous()
    grid = torch.stack([at // 140 + 7 * (seed % 1000), at // 20 % 7, at % 20], 1)
    return grid[:, :axes].contiguous()


def _frequencies(case):
    """Radians per unit of position of every rotation pair, in 64 bits."""
    parts = []
    for s in _sections(case):
        j = torch.arange(s, device=_DEVICE, dtype=torch.float64) / s
        parts.append(2.0 * math.pi / (0.05 * 400.0 ** j) if case["pos"] == "metric" else 10000.0 ** -j)
    return torch.cat(parts)


def prepare(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(1000003 * seed + 17)
    dtype = _TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        state["x"] = _normal((m, k + case["pad"]), gen, dtype)[:, :k]
        state["weight"] = _normal((n, k), gen, dtype, 1.0 / math.sqrt(k))
        state["bias"] = _normal((n,), gen, dtype, 0.5) if case["bias"] else None
        state["residual"] = _normal((m, n), gen, dtype) if case["residual"] else None
        state["count"] = torch.tensor([case["live"]], dtype=torch.int32, device=_DEVICE) if case["live"] >= 0 else None
        state["out"] = torch.zeros((m, n), dtype=dtype, device=_DEVICE) if case["live"] >= 0 else None
    elif case["op"] == "rope":
        tokens, hq, hk, dim = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
        rows = _normal((tokens, hq + (2 if case["packed"] else 1) * hk, dim), gen, dtype)
        state["q"], state["k"] = rows[:, :hq], rows[:, hq:hq + hk]
        if not case["packed"]:
            state["q"], state["k"] = state["q"].contiguous(), state["k"].contiguous()
        state["pos"] = _positions(case, gen, seed)
        state["freqs"] = _frequencies(case)
        weighted = case["weight"] and case["norm"] != "none"
        state["q_weight"] = (1.0 + _normal((dim,), gen, torch.float32, 0.2)).to(dtype) if weighted else None
        state["k_weight"] = (1.0 + _normal((dim,), gen, torch.float32, 0.2)).to(dtype) if weighted else None
    else:
        b, lq, lk, hq, hk, dim = (case[n] for n in ("batch", "q_len", "k_len", "q_heads", "k_heads", "dim"))
        if case["packed"]:
            rows = _normal((b, lq, hq + 2 * hk, dim), gen, dtype)
            state["q"], state["k"], state["v"] = rows[:, :, :hq], rows[:, :, hq:hq + hk], rows[:, :, hq + hk:]
        else:
            state["q"] = _normal((b, lq, hq, dim), gen, dtype)
            state["k"] = _normal((b, lk, hk, dim), gen, dtype)
            state["v"] = _normal((b, lk, hk, dim), gen, dtype)
        q_lens, k_lens = _lens(case)
        state["q_lens"] = torch.tensor(q_lens, dtype=torch.int32, device=_DEVICE) if case["ragged"] else None
        state["k_lens"] = torch.tensor(k_lens, dtype=torch.int32, device=_DEVICE) if case["ragged"] else None
        state["out"] = torch.zeros((b, lq, hq, dim), dtype=dtype, device=_DEVICE) if case["ragged"] else None
    return state


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _plain_linear(s):
    case = s["case"]
    y = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["act"] == "relu":
        y = torch.clamp(y, min=0.0)
    elif case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(s["x"].dtype)
    if s["count"] is None:
        return y
    return torch.where((torch.arange(y.shape[0], device=y.device) < s["count"])[:, None], y, s["out"])


def _plain_rotate(x, weight, cos, sin, case):
    y = x.float()
    if case["norm"] == "rms":
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6)
    elif case["norm"] == "l2":
        y = y / torch.clamp(torch.sqrt((y * y).sum(-1, keepdim=True)), min=1e-6)
    if weight is not None:
        y = y * weight.float()
    pairs = cos.shape[-1]
    turned = y.clone()
    first, second = (slice(0, pairs), slice(pairs, 2 * pairs)) if case["pairs"] == "half" else (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2))
    a, b = y[..., first], y[..., second]
    turned[..., first] = a * cos - b * sin
    turned[..., second] = b * cos + a * sin
    return turned.to(x.dtype)


def _plain_rope(s):
    case = s["case"]
    axis = torch.repeat_interleave(torch.arange(len(_sections(case)), device=s["pos"].device),
                                   torch.tensor(_sections(case), device=s["pos"].device), output_size=s["freqs"].numel())
    angle = s["pos"].double()[:, axis] * s["freqs"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    return _plain_rotate(s["q"], s["q_weight"], cos, sin, case), _plain_rotate(s["k"], s["k_weight"], cos, sin, case)


def _plain_attention(s):
    case = s["case"]
    q, k, v = s["q"], s["k"], s["v"]
    batch, q_len, q_heads, dim = q.shape
    k_len, k_heads = k.shape[1], k.shape[2]
    group = q_heads // k_heads
    left, right, sinks = case["left"], case["right"], case["sinks"]
    ql = s["q_lens"].long() if s["q_lens"] is not None else torch.full((batch,), q_len, device=q.device)
    kl = s["k_lens"].long() if s["k_lens"] is not None else torch.full((batch,), k_len, device=q.device)
    behind = (kl - ql).view(batch, 1, 1)
    # queries in blocks, each against the first tokens and the stretch of keys that its window can reach
    banded = left >= 0 and right >= 0 and left + right + 1 < k_len
    size = min(q_len, max(64, left + right + 1)) if banded else q_len
    blocks = -(-q_len // size)
    if banded:
        start = torch.arange(blocks, device=q.device).view(1, blocks, 1) * size + behind - left
        stretch = start + torch.arange(size + left + right, device=q.device)
        stretch = torch.where(stretch >= sinks, stretch, -1)
        index = torch.cat([torch.arange(sinks, device=q.device).expand(batch, blocks, sinks), stretch], 2)
        entry = torch.arange(batch, device=q.device).view(batch, 1, 1)
        kk, vv = k[entry, index.clamp(0, k_len - 1)].float(), v[entry, index.clamp(0, k_len - 1)].float()
    else:
        index = torch.arange(k_len, device=q.device).expand(batch, 1, k_len)
        kk, vv = k.float()[:, None], v.float()[:, None]
    inside = (index >= 0) & (index < kl.view(batch, 1, 1))
    at = (torch.arange(blocks * size, device=q.device).view(1, blocks, size) + behind)[..., None]
    key = index[:, :, None, :]
    seen = inside[:, :, None, :].expand(batch, blocks, size, index.shape[2])
    if right >= 0:
        seen = seen & (key <= at + right)
    if left >= 0:
        seen = seen & ((key >= at - left) | (key < sinks))
    qq = torch.nn.functional.pad(q.float(), (0, 0, 0, 0, 0, blocks * size - q_len))
    qq = qq.view(batch, blocks, size, k_heads, group, dim).permute(0, 1, 3, 4, 2, 5).reshape(batch, blocks, k_heads, group * size, dim)
    score = torch.matmul(qq, kk.permute(0, 1, 3, 4, 2).contiguous()).view(batch, blocks, k_heads, group, size, -1) / math.sqrt(dim)
    score = score.masked_fill(~seen[:, :, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(most == -math.inf, 0.0, most))
    del score
    total = p.sum(-1, keepdim=True)
    vv = vv.masked_fill(~inside[..., None, None], 0.0).permute(0, 1, 3, 2, 4).contiguous()
    o = torch.matmul(p.view(batch, blocks, k_heads, group * size, -1), vv).view(batch, blocks, k_heads, group, size, dim)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 1, 4, 2, 3, 5).reshape(batch, blocks * size, q_heads, dim)[:, :q_len].to(q.dtype)
    if s["q_lens"] is None:
        return o
    return torch.where((torch.arange(q_len, device=q.device) < ql[:, None])[..., None, None], o, s["out"])


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        ctx = _context()
        if case["op"] == "linear":
            return ctx.linear(state["x"], state["weight"], bias=state["bias"], act=case["act"], residual=state["residual"],
                              out=state["out"], m_dev=state["count"])
        if case["op"] == "rope":
            return ctx.qk_norm_rope(state["q"], state["k"], state["pos"], state["freqs"], _sections(case), norm=case["norm"], eps=1e-6,
                                    q_weight=state["q_weight"], k_weight=state["k_weight"], pairs=case["pairs"])
        return ctx.attention(state["q"], state["k"], state["v"], window=(case["left"], case["right"]), sinks=case["sinks"],
                             q_lens=state["q_lens"], k_lens=state["k_lens"], out=state["out"])
    if case["op"] == "linear":
        return _plain_linear(state)
    if case["op"] == "rope":
        return _plain_rope(state)
    return _plain_attention(state)


# ---------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_linear(s):
    case = s["case"]
    y = torch.mm(s["x"].double(), s["weight"].double().t().contiguous())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "relu":
        y = torch.maximum(y, torch.zeros((), dtype=torch.float64, device=y.device))
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "gelu":
        y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2.0))
    if s["residual"] is not None:
        y += s["residual"].double()
    if case["live"] >= 0:
        y[case["live"]:] = s["out"][case["live"]:].double()
    return y


def _exact_rope(s):
    case, sections = s["case"], _sections(s["case"])
    angles, at = [], 0
    for axis, count in enumerate(sections):
        angles.append(s["pos"][:, axis].double()[:, None] * s["freqs"][None, at:at + count])
        at += count
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=_DEVICE), torch.cat(angles, 1))[:, None]
    found = []
    for x, weight in ((s["q"].double(), s["q_weight"]), (s["k"].double(), s["k_weight"])):
        if case["norm"] == "rms":
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6)
        elif case["norm"] == "l2":
            x = x / torch.linalg.vector_norm(x, dim=-1, keepdim=True).clamp_min(1e-6)
        if weight is not None:
            x = x * weight.double()
        head, rest = x[..., :2 * at], x[..., 2 * at:]
        pairs = head.unflatten(-1, (2, at)).transpose(-1, -2) if case["pairs"] == "half" else head.unflatten(-1, (at, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(-1, -2) if case["pairs"] == "half" else z
        found.append(torch.cat([z.flatten(-2), rest], -1))
    return tuple(found)


def _exact_attention(s):
    case = s["case"]
    q_lens, k_lens = _lens(case)
    batch, q_len, q_heads, dim = s["q"].shape
    group = q_heads // s["k"].shape[2]
    out = s["out"].double().clone() if s["out"] is not None else torch.empty(s["q"].shape, dtype=torch.float64, device=_DEVICE)
    together = max(1, int(5e7 // (case["q_len"] * case["k_len"] * q_heads))) if not case["ragged"] else 1
    for b0 in range(0, batch, together):
        b1, ql, kl = min(batch, b0 + together), int(q_lens[b0]), int(k_lens[b0])
        for i0 in range(0, ql, 512):
            i1 = min(ql, i0 + 512)
            low, high = i0 + kl - ql - case["left"] if case["left"] >= 0 else 0, i1 + kl - ql + case["right"] if case["right"] >= 0 else kl
            j = torch.arange(kl, device=_DEVICE)
            j = j[((j >= low) | (j < case["sinks"])) & (j < high)]
            query = s["q"][b0:b1, i0:i1].double().transpose(1, 2).contiguous()
            key = s["k"][b0:b1, j].double().permute(0, 2, 3, 1).repeat_interleave(group, 1)
            value = s["v"][b0:b1, j].double().transpose(1, 2).repeat_interleave(group, 1)
            far = j[None, :] - (torch.arange(i0, i1, device=_DEVICE) + (kl - ql))[:, None]
            hidden = torch.zeros(far.shape, dtype=torch.bool, device=_DEVICE)
            if case["right"] >= 0:
                hidden |= far > case["right"]
            if case["left"] >= 0:
                hidden |= (far < -case["left"]) & (j[None, :] >= case["sinks"])
            weight = torch.softmax((torch.matmul(query, key) * dim ** -0.5).masked_fill(hidden, -math.inf), -1)
            weight = weight.masked_fill(hidden.all(-1)[:, None], 0.0)
            out[b0:b1, i0:i1] = torch.matmul(weight, value.contiguous()).transpose(1, 2)
    return out


def exact(case, seed):
    if case["op"] == "attention" and 4 * _visible(case)[0] * case["q_heads"] * case["dim"] > 4e12:
        return None
    state = prepare(case, seed)
    return {"linear": _exact_linear, "rope": _exact_rope, "attention": _exact_attention}[case["op"]](state)
