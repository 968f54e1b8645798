"""Performance cases of dropout without a stored mask, of the RMSNorm of a
residual's sum (with an output in 8 bits, or with gradients), and of the rotation
of queries and keys by positions on several axes.

Kinds of call:
  dropout  rows, forward + backward
  norm     h = residual + dropout(x) and its RMSNorm: a serving call whose norm
           leaves in 8 bits, or forward + backward, with or without an 8-bit
           checkpoint of h
  rope     queries and keys turned by positions on 2 to 4 axes, alone or after
           the RMSNorm of every head: a serving step, or forward + backward

Dropout's numbers come from Philox4x32-10: the block of channels 8 j .. 8 j + 7
of row i has the counter (i ceil(C / 8) + j, offset), two 64-bit numbers, and the
seed as key; its four words are eight numbers of 16 bits, the low half first.
With t = round(p 2^16) a value is kept, times 2^16 / (2^16 - t), where its
number is at least t.

8 bits: blocks of 32 consecutive values of a row (the last one may be shorter).
With a = max |x| of a block, M = 127 ("int8") or 448 ("e4m3") and e the least
integer with a <= M 2^e, at least -100, it holds x 2^-e rounded to nearest even
in that format.  A backward pass over a checkpoint is the operator's at those
values.
"""
import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # A branch's rows at the paper sweep's smallest training call.
        _dropout("dropout_small", 320, 1280, "f32", 0.1),
        # The rows of one layer at the benchmark's training size.
        _dropout("dropout_train", 32768, 4096, "bf16", 0.1),
        # A serving step: one new token for each of 16 sequences, an 8-bit product behind it.
        _norm("norm_decode", 16, 4096, "bf16", "bf16", 0.0, False, "e4m3"),
        # A long prompt on the same path.
        _norm("norm_prompt", 16384, 4096, "bf16", "bf16", 0.0, False, "e4m3"),
        # Training at the benchmark's RMSNorm rows, dropout on the branch.
        _norm("norm_train", 16384, 4096, "bf16", "bf16", 0.1, True, ""),
        # A bf16 branch on the fp32 rows that the residual wrapper returns, h kept in 8 bits.
        _norm("norm_mixed", 8192, 4096, "bf16", "f32", 0.0, True, "int8"),
        # A row length and count with no convenient factor.
        _norm("norm_ragged", 2999, 1001, "f32", "f32", 0.25, True, "e4m3"),
        # A serving step of text behind a video: one new token for each of 16 sequences.
        _rope("rope_decode", 16, 32, 8, 128, 128, "bf16", 131072, "24,20,20", True, False, False, False),
        # Training on text and video, heads normed: grouped heads at the benchmark's width.
        _rope("rope_norm_train", 8192, 32, 8, 128, 128, "bf16", 8192, "16,24,24", False, False, True, True),
        # As many key heads as query heads, rotation alone, pairs dealt to the axes in turn.
        _rope("rope_train", 16384, 32, 32, 128, 128, "bf16", 16384, "24,20,20", True, False, False, True),
        # Images: two axes on half of each head of 80, neighbouring pairs, an odd token count.
        _rope("rope_ragged", 2999, 13, 13, 80, 40, "f32", 4096, "10,10", False, True, True, True),
    ]


def _named(c, name):
    if name is not None:
        c["name"] = name
    return c


def _dropout(name, rows, hidden, dtype, p):
    return _named({"kind": "dropout", "rows": rows, "hidden": hidden, "dtype": dtype, "p": p}, name)


def _norm(name, rows, hidden, dtype, residual, p, train, fmt):
    return _named({"kind": "norm", "rows": rows, "hidden": hidden, "dtype": dtype, "residual": residual, "p": p,
                   "train": train, "format": fmt}, name)


def _rope(name, tokens, heads, kv_heads, head_dim, rotary, dtype, context, sections, dealt, interleaved, norm, train):
    return _named({"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                   "rotary": rotary, "dtype": dtype, "context": context, "sections": sections, "dealt": dealt,
                   "interleaved": interleaved, "norm": norm, "train": train}, name)


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("dropout", "norm", "norm", "rope", "rope"))
    dtype = rng.choice(("f32", "bf16"))
    p = rng.choice((0.05, 0.1, 0.2, 0.3, 0.5))
    if kind in ("dropout", "norm"):
        hidden = _log(rng, 64, 7168)
        if rng.random() < 0.7:  # a transformer's width
            hidden = max(8, hidden // 8 * 8)
        if kind == "dropout":
            most = 32768 * 4096 * 2 // (hidden * (4 if dtype == "f32" else 2))
            return _dropout(None, _log(rng, 16, min(most, 65536)), hidden, dtype, p)
        residual = rng.choice((dtype, dtype, "f32"))
        train = rng.random() < 0.6
        most = min(16384 * 4096 * 2 // (hidden * (4 if residual == "f32" else 2)), 65536)
        return _norm(None, _log(rng, 16 if train else 1, most), hidden, dtype, residual,
                     rng.choice((0.0, p)) if train else 0.0, train, rng.choice(("", "int8", "e4m3") if train else ("int8", "e4m3")))
    head_dim = rng.choice((64, 128, 128, 128, 80, 96, 112, 192, 256, 72))
    rotary = rng.choice((head_dim, head_dim, head_dim, head_dim // 2 // 2 * 2))
    axes = rng.choice((2, 3, 3, 3, 4))
    rest = [rng.randint(rotary // 2 // axes // 2, rotary // 2 // axes) for _ in range(axes - 1)]
    sections = ",".join(str(s) for s in [rotary // 2 - sum(rest)] + rest)
    kv = rng.choice((1, 2, 4, 8, 8, 13))
    heads = min(kv * rng.choice((1, 4, 5, 8)), 64)
    train = rng.random() < 0.7
    most = 16384 * 64 * 128 // ((heads + kv) * head_dim * (2 if dtype == "f32" else 1))
    tokens = _log(rng, 16, min(most, 16384)) if train else _log(rng, 1, 1024)
    return _rope(None, tokens, heads, kv, head_dim, rotary, dtype, _log(rng, 4096, 131072), sections,
                 rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.5, train)


# ---------------------------------------------------------------------------
# State: inputs, parameters, cotangents
# ---------------------------------------------------------------------------

def _randn(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    t = torch.randn(*shape, device="cuda", generator=g)
    return t.mul_(std).add_(mean).to(dtype)


def _rows(g, shape, dtype):
    """Activations: a transformer's rows have a few channels that are much
    larger than the others."""
    t = torch.randn(*shape, device="cuda", generator=g)
    big = torch.rand(shape[-1], device="cuda", generator=g) < 0.005
    return t.mul_(torch.where(big, 12.0, 1.0)).to(dtype)


def _positions(case, g):
    """int64 [axes, tokens]: a serving step's positions are far along and equal
    on every axis; a training row holds text, then frames of 24 x 32 patches."""
    T, axes = case["tokens"], len(case["sections"].split(","))
    if not case["train"]:
        return torch.randint(case["context"], (T,), device="cuda", generator=g).expand(axes, T).contiguous()
    text = T // 8
    i = torch.arange(T, device="cuda")
    j = i - text
    grid = torch.stack([j // 768, j // 32 % 24, j % 32, j // 1536][:axes]) + text
    return torch.where(i < text, i.expand(axes, T), grid).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    kind = case["kind"]
    s = {"case": case}
    if kind != "rope":
        # a training program's seed of the step, and the number of the call site
        s["seed"] = torch.randint(2 ** 62, (1,), device="cuda", generator=g)
        s["offset"] = 7
        T, C = case["rows"], case["hidden"]
        s["x"] = _rows(g, (T, C), dt)
        if kind == "dropout":
            s["x"].requires_grad_(True)
            s["cot"] = _randn(g, T, C, dtype=dt)
            return s
        s["residual"] = _rows(g, (T, C), _DTYPES[case["residual"]])
        s["weight"] = _randn(g, C, std=0.1, mean=1.0, dtype=dt)
        if case["train"]:
            for k in ("x", "residual", "weight"):
                s[k].requires_grad_(True)
            s["cot"] = [_randn(g, T, C, dtype=dt), _randn(g, T, C, dtype=_DTYPES[case["residual"]])]
        return s
    T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    # queries, keys and values as one projection leaves them
    qkv = _rows(g, (T, H + 2 * K, D), dt)
    s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + K]
    s["sections"] = [int(n) for n in case["sections"].split(",")]
    s["params"] = [_randn(g, D, std=0.1, mean=1.0, dtype=dt) for _ in range(2)] if case["norm"] else []
    freq = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
    angle = torch.arange(case["context"], device="cuda", dtype=torch.float64).unsqueeze(1) * freq
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["positions"] = _positions(case, g)
    if case["train"]:
        for t in (s["q"], s["k"], *s["params"]):
            t.requires_grad_(True)
        s["cot"] = [_randn(g, T, H, D, dtype=dt), _randn(g, T, K, D, dtype=dt)]
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import mhc_ascend_amd as mhc

    case = s["case"]
    kind = case["kind"]
    if kind == "dropout":
        out = mhc.dropout(s["x"], case["p"], seed=s["seed"], offset=s["offset"])
        return out.detach(), *torch.autograd.grad(out, [s["x"]], [s["cot"]])
    if kind == "norm":
        call = (s["x"], s["residual"], s["weight"], _EPS)
        if not case["train"]:
            packed, h = mhc.rmsnorm_residual(*call, format=case["format"])
            if case["format"] == "int8":  # the values it stands for, exact in bf16
                return mhc.activation_unpack(packed, torch.bfloat16), h
            return (packed.values[:, :case["hidden"]].view(torch.float8_e4m3fn),
                    packed.scales.view(torch.float8_e8m0fnu), h)
        out = mhc.rmsnorm_residual(*call, dropout=case["p"], seed=s["seed"], offset=s["offset"],
                                   checkpoint=case["format"] or None)
        grads = torch.autograd.grad(out, [s["x"], s["residual"], s["weight"]], s["cot"])
        return (*[o.detach() for o in out], *grads)
    how = {"positions": s["positions"], "interleaved": case["interleaved"], "sections": s["sections"],
           "sections_dealt": case["dealt"]}
    if case["norm"]:
        out = mhc.qk_norm_rope(s["q"], s["k"], *s["params"], s["cos"], s["sin"], eps=_EPS, **how)
    else:
        out = mhc.qk_rope(s["q"], s["k"], s["cos"], s["sin"], **how)
    if not case["train"]:
        return out
    grads = torch.autograd.grad(out, [s["q"], s["k"], *s["params"]], s["cot"])
    return (*[o.detach() for o in out], *grads)


# The plain form: 32-bit torch operations, rounded once at the end.

_LOW = 0xFFFFFFFF


def _kept(rows, hidden, p, seed, offset):
    """1 / (1 - p) where a value is kept, 0 where it is not: fp32 [rows, hidden]."""
    t = round(p * 65536)
    per = (hidden + 7) // 8
    block = torch.arange(rows * per, device=seed.device)
    c0, c1 = block & _LOW, block >> 32
    c2, c3 = torch.full_like(block, offset & _LOW), torch.full_like(block, offset >> 32)
    k0, k1 = seed & _LOW, seed >> 32 & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = (b >> 32 & _LOW) ^ c1 ^ k0, b & _LOW, (a >> 32 & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = k0 + 0x9E3779B9 & _LOW, k1 + 0xBB67AE85 & _LOW
    words = torch.stack([c0, c1, c2, c3], -1)
    u = torch.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, per * 8)[:, :hidden]
    return torch.where(u >= t, 65536.0 / (65536 - t), 0.0)


def _blocks(x):
    pad = -x.shape[-1] % 32
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], -1)
    return x.reshape(*x.shape[:-1], -1, 32)


def _packed(x, fmt):
    """(values before the scale, scales) of fp32 x, in bit arithmetic on fp32 numbers."""
    b = _blocks(x)
    a = b.abs().amax(-1, keepdim=True).view(torch.int32)
    # e + 127: the exponent field less that of the format's largest value, one
    # more where the mantissa is past its mantissa (127 = 1.984375 * 2^6, 448 =
    # 1.75 * 2^8)
    past, top = (0x7E0000, 6) if fmt == "int8" else (0x600000, 8)
    e = (((a + (0x7FFFFF - past)) >> 23) - top).clamp_min_(27)
    v = b * ((254 - e) << 23).view(torch.float32)
    if fmt == "int8":
        v = v.round()
    else:
        # three mantissa bits, subnormal steps of 2^-9 below 2^-6
        step = (v.view(torch.int32) >> 23 & 255).clamp_min_(121) - 3
        v = (v * ((254 - step) << 23).view(torch.float32)).round() * (step << 23).view(torch.float32)
    return v, (e << 23).view(torch.float32)


def _held(x, fmt):
    if not fmt:
        return x
    v, scale = _packed(x, fmt)
    return (v * scale).reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def _normed(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w


def _columns(s):
    """cos and sin [tokens, 1, rotary / 2] of every pair's axis."""
    pairs = torch.arange(s["cos"].shape[1], device="cuda")
    sizes = torch.tensor(s["sections"], device="cuda")
    if s["case"]["dealt"]:
        a = pairs % len(s["sections"])
        axis = torch.where(pairs // len(s["sections"]) < sizes[a], a, 0)
    else:
        axis = torch.searchsorted(sizes.cumsum(0), pairs, right=True)
    row = s["positions"][axis].t()
    return s["cos"][row, pairs].unsqueeze(1), s["sin"][row, pairs].unsqueeze(1)


def _turned(y, c, s, interleaved):
    R = 2 * c.shape[-1]
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    pair = (a * c - b * s, b * c + a * s)
    rot = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([rot, y[..., R:]], -1)


def _run_plain(s):
    case = s["case"]
    dt = _DTYPES[case["dtype"]]
    if case["kind"] == "dropout":
        with torch.no_grad():
            kept = _kept(case["rows"], case["hidden"], case["p"], s["seed"], s["offset"])
            return (s["x"].float() * kept).to(dt), (s["cot"].float() * kept).to(dt)
    if case["kind"] == "norm":
        return _plain_norm(s, case, dt)
    with torch.no_grad():
        c, sn = _columns(s)
    turn = lambda x, w: _turned(_normed(x, w) if case["norm"] else x, c, sn, case["interleaved"])  # noqa: E731
    ins = [s["q"].detach().float(), s["k"].detach().float()]
    ps = [t.detach().float() for t in s["params"]]
    if case["train"]:
        ins = [t.requires_grad_(True) for t in ins]
        ps = [t.requires_grad_(True) for t in ps]
    outs = [turn(x, w) for x, w in zip(ins, ps or (None, None))]
    if not case["train"]:
        return tuple(o.to(dt) for o in outs)
    grads = torch.autograd.grad(outs, ins + ps, [t.float() for t in s["cot"]])
    return (*[o.detach().to(dt) for o in outs], *[g.to(dt) for g in grads])


def _plain_norm(s, case, dt):
    rt, fmt = _DTYPES[case["residual"]], case["format"]
    with torch.no_grad():
        x, w = s["x"].float(), s["weight"].float()
        kept = _kept(case["rows"], case["hidden"], case["p"], s["seed"], s["offset"]) if case["p"] else 1.0
        h = (s["residual"].float() + x * kept).to(rt)
        y = _normed(h.float(), w)
        if not case["train"]:
            v, scale = _packed(y, fmt)
            if fmt == "int8":
                return (v * scale).reshape(case["rows"], -1)[:, :case["hidden"]].to(torch.bfloat16), h
            return (v.reshape(case["rows"], -1)[:, :case["hidden"]].to(torch.float8_e4m3fn),
                    scale.squeeze(-1).to(torch.float8_e8m0fnu), h)
    hat, w = _held(h.float(), fmt).requires_grad_(True), w.requires_grad_(True)
    dt_h, dw = torch.autograd.grad(_normed(hat, w), [hat, w], s["cot"][0].float())
    dh = dt_h + s["cot"][1].float()
    return y.to(dt), h, (dh * kept).to(dt), dh.to(rt), dw.to(dt)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    """Rows or a checkpoint that the forward leaves for the backward count where
    they are written and where they are read: the rest of the step runs between
    the two.  Dropout's integer work is ten rounds of two products and about
    eight other operations for eight values."""
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "dropout":
        E = case["rows"] * case["hidden"]
        return {"bytes": 4 * E * size, "flops": 2 * E * 14}
    if case["kind"] == "norm":
        rows, C = case["rows"], case["hidden"]
        E, rsize = rows * C, 2 if case["residual"] == "bf16" else 4
        held = rows * (C + (C + 31) // 32)
        if not case["train"]:  # x, residual in; h, 8 bits out
            return {"bytes": E * (size + 2 * rsize) + held + C * size, "flops": 6 * E}
        # x, residual in, y, h out; their cotangents and h in, both gradients out (one where they are equal)
        one = case["p"] == 0 and size == rsize
        nbytes = E * (2 * size + 2 * rsize) + E * (size + rsize) + E * rsize + (0 if one else E * size)
        nbytes += 2 * held if case["format"] else E * rsize
        return {"bytes": nbytes + 3 * C * size, "flops": E * (16 + (28 if case["p"] else 0))}
    T, D = case["tokens"], case["head_dim"]
    rows = T * (case["heads"] + case["kv_heads"])
    nbytes = 2 * rows * D * size + T * 8 * len(case["sections"].split(","))
    nbytes += min(T, case["context"]) * case["rotary"] * 4
    flops = (8 if case["norm"] else 4) * rows * D
    if case["train"]:  # cotangents in, gradients out; a norm's rows again
        nbytes += (3 if case["norm"] else 2) * rows * D * size
        flops += (14 if case["norm"] else 4) * rows * D
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# The same in 64 bits, gradients by their formulas
# ---------------------------------------------------------------------------

def _exact_scale(case, s):
    """Dropout's factors by the generator's definition, numpy's unsigned numbers."""
    T, C, t = case["rows"], case["hidden"], int(round(case["p"] * 65536))
    per = -(-C // 8)
    key = int(s["seed"].item()) % 2 ** 64
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    ctr = [np.arange(T * per, dtype=np.uint64) & low, np.arange(T * per, dtype=np.uint64) >> half,
           np.uint64(s["offset"] % 2 ** 32), np.uint64(s["offset"] >> 32)]
    k = [key % 2 ** 32, key >> 32]
    for _ in range(10):
        m0, m2 = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
        ctr = [(m2 >> half) ^ ctr[1] ^ np.uint64(k[0]), m2 & low, (m0 >> half) ^ ctr[3] ^ np.uint64(k[1]), m0 & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    u = np.empty((T * per, 8), dtype=np.uint16)
    for e in range(8):
        u[:, e] = (ctr[e // 2] >> np.uint64(16 * (e % 2))).astype(np.uint16)
    keep = torch.from_numpy(u.reshape(T, per * 8)[:, :C] >= t).cuda()
    return keep.double() * (65536 / (65536 - t))


def _exact_pack(x, fmt):
    """(numbers, 2^e) by the definition, fp64."""
    top = 127.0 if fmt == "int8" else 448.0
    b = _blocks(x)
    a = b.abs().amax(-1, keepdim=True)
    _, k = torch.frexp(a / top)
    e = k.double() - 1  # the quotient is rounded: settle the edge by comparing exactly
    e = torch.where(a <= top * torch.exp2(e), e, e + 1)
    e = torch.where(a > 0, e, torch.full_like(e, -100.0)).clamp_min(-100.0)
    v = b * torch.exp2(-e)
    if fmt == "int8":
        return torch.round(v), torch.exp2(e)
    _, kv = torch.frexp(v)
    step = torch.exp2((kv.double() - 1).clamp_min(-6.0) - 3)
    return torch.round(v / step) * step, torch.exp2(e)


def _exact_held(x, fmt):
    if not fmt:
        return x
    q, scale = _exact_pack(x, fmt)
    return (q * scale).reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def _exact_norm_back(x, w, u):
    """Gradients of x / r * w for cotangent u: rows, and the terms of w's."""
    r = torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS)
    dot = (u * w * x).sum(-1, keepdim=True)
    return u * w / r - x * dot / (x.shape[-1] * r ** 3), u * x / r


def _exact_axes(case, s):
    """cos and sin [tokens, 1, rotary / 2], an axis at a time."""
    n, sizes = len(s["sections"]), s["sections"]
    half = s["cos"].shape[1]
    c, sn = (torch.empty(case["tokens"], half, device="cuda", dtype=torch.float64) for _ in range(2))
    start = 0
    for a in range(n):
        if case["dealt"]:
            cols = [p for p in range(half) if (p % n == a and p // n < sizes[a]) or
                    (a == 0 and p // n >= sizes[p % n])]
        else:
            cols = list(range(start, start + sizes[a]))
            start += sizes[a]
        at = s["positions"][a]
        c[:, cols], sn[:, cols] = s["cos"][at][:, cols].double(), s["sin"][at][:, cols].double()
    return c.unsqueeze(1), sn.unsqueeze(1)


def _exact_turn(v, c, sn, interleaved, sign):
    """Rotation of v's pairs by +angle (sign 1) or -angle (sign -1)."""
    half = c.shape[-1]
    i = torch.arange(half, device=v.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    res = v.clone()
    res[..., lo] = v[..., lo] * c - sign * v[..., hi] * sn
    res[..., hi] = v[..., hi] * c + sign * v[..., lo] * sn
    return res


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "dropout":
            f = _exact_scale(case, s)
            return s["x"].detach().double() * f, s["cot"].double() * f
        if kind == "norm":
            f = _exact_scale(case, s) if case["p"] else 1.0
            h = s["residual"].detach().double() + s["x"].detach().double() * f
            stored = h.to(_DTYPES[case["residual"]]).double()  # the sum is the norm's input as it is stored
            w = s["weight"].detach().double()
            y = stored / torch.sqrt(stored.square().mean(-1, keepdim=True) + _EPS) * w
            if not case["train"]:
                q, scale = _exact_pack(y, case["format"])
                v = (q * scale if case["format"] == "int8" else q).reshape(case["rows"], -1)[:, :case["hidden"]]
                return (v, h) if case["format"] == "int8" else (v, scale.squeeze(-1), h)
            back, dw = _exact_norm_back(_exact_held(stored, case["format"]), w, s["cot"][0].double())
            dh = back + s["cot"][1].double()
            return y, h, dh * f, dh, dw.sum(0)
        c, sn = _exact_axes(case, s)
        p = [t.detach().double() for t in s["params"]]
        outs, rows, weights = [], [], []
        for i, key in enumerate(("q", "k")):
            x = s[key].detach().double()
            y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * p[i] if p else x
            outs.append(_exact_turn(y, c, sn, case["interleaved"], 1.0))
            if case["train"]:
                u = _exact_turn(s["cot"][i].double(), c, sn, case["interleaved"], -1.0)
                if p:
                    u, dw = _exact_norm_back(x, p[i], u)
                    weights.append(dw.sum((0, 1)))
                rows.append(u)
        return (*outs, *rows, *weights)
