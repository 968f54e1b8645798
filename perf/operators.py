"""Performance cases of the operators that keep their rows in 8 bits for the
backward pass, and of the per-head norm of queries and keys with its rotation.

Kinds of call:
  pack     rows to an 8-bit checkpoint and back (activation_pack / _unpack)
  rmsnorm  RMSNorm of rows, forward + backward from the checkpoint
  layer    the mHC layer (static or dynamic H), forward + backward from the
           checkpoint of its streams
  qk       per-head RMSNorm of queries and keys and their position rotation:
           a serving step, or forward + backward, with or without a checkpoint

A checkpoint holds blocks of 32 consecutive values of a row (the last one may
be shorter).  With a = max |x| of a block, M = 127 ("int8") or 448 ("e4m3") and
e the least integer with a <= M 2^e, at least -100, it holds x 2^-e rounded to
nearest even in that format.  x^ below is the value it stands for.  A backward
pass is the operator's at x^; the dynamic layer's per-token coefficients stay
the forward's.
"""
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_MAX = {"int8": 127.0, "e4m3": 448.0}
_EPS = 1e-5
_SK_EPS = 1e-8
_ITERS = 20


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # The streams of the paper sweep's smallest training call.
        _pack("pack_small", 1280, 1280, "f32", "e4m3"),
        # The streams of one layer at the benchmark's training size.
        _pack("pack_train", 32768, 4096, "bf16", "int8"),
        # A row length and count with no convenient factor.
        _rmsnorm("rmsnorm_ragged", 2999, 1001, "f32", "e4m3"),
        # The benchmark's RMSNorm rows.
        _rmsnorm("rmsnorm_train", 16384, 4096, "bf16", "int8"),
        # The paper sweep's smallest training call.
        _layer("static_small", 320, 4, 1280, "f32", "int8", False),
        # Training with static H: the benchmark's default workload.
        _layer("static_train", 8192, 4, 4096, "f32", "int8", False),
        # An expansion rate that is no power of two, odd token count.
        _layer("dynamic_n6", 2047, 6, 1040, "bf16", "e4m3", True),
        # Training with dynamic H: the benchmark's dynamic workload.
        _layer("dynamic_train", 8192, 4, 4096, "bf16", "int8", True),
        # A serving step: one new token for each of 16 sequences, far along.
        _qk("qk_decode", 16, 32, 8, 128, 128, "bf16", 131072, False, False, None),
        # Training with grouped heads at the benchmark's width.
        _qk("qk_train", 8192, 32, 8, 128, 128, "bf16", 8192, False, True, None),
        # The same with as many key heads as query heads, rows kept in 8 bits.
        _qk("qk_train_8bit", 16384, 32, 32, 128, 128, "bf16", 4096, False, True, "int8"),
        # Heads of 80 with half of them rotated in neighbouring pairs.
        _qk("qk_ragged", 2999, 13, 13, 80, 40, "f32", 3001, True, True, "e4m3"),
    ]


def _named(c, name):
    if name is not None:
        c["name"] = name
    return c


def _pack(name, rows, hidden, dtype, fmt):
    return _named({"kind": "pack", "rows": rows, "hidden": hidden, "dtype": dtype, "format": fmt}, name)


def _rmsnorm(name, rows, hidden, dtype, fmt):
    return _named({"kind": "rmsnorm", "rows": rows, "hidden": hidden, "dtype": dtype, "format": fmt}, name)


def _layer(name, tokens, n, hidden, dtype, fmt, dynamic):
    return _named({"kind": "layer", "tokens": tokens, "n": n, "hidden": hidden, "dtype": dtype, "format": fmt,
                   "dynamic": dynamic}, name)


def _qk(name, tokens, heads, kv_heads, head_dim, rotary, dtype, context, interleaved, train, fmt):
    return _named({"kind": "qk", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                   "rotary": rotary, "dtype": dtype, "context": context, "interleaved": interleaved, "train": train,
                   "format": fmt or ""}, name)


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(("pack", "rmsnorm", "rmsnorm", "layer", "layer", "layer", "qk", "qk", "qk"))
    dtype = rng.choice(("f32", "bf16"))
    fmt = rng.choice(("int8", "e4m3"))
    if kind in ("pack", "rmsnorm"):
        hidden = _log(rng, 64, 7168)
        if rng.random() < 0.7:  # a transformer's width
            hidden = max(8, hidden // 8 * 8)
        most = min((32768 if kind == "pack" else 16384) * 4096 // hidden, 65536)
        make = _pack if kind == "pack" else _rmsnorm
        return make(None, _log(rng, 16, most), hidden, dtype, fmt)
    if kind == "layer":
        dynamic = rng.random() < 0.5
        n = rng.choice((4, 4, 4, 4, 2, 8, 3, 6, 12))
        hidden = _log(rng, 256, 7168)
        if dynamic:
            hidden = hidden // 32 * 32  # whole k steps of the projection
        elif rng.random() < 0.7:
            hidden = hidden // 8 * 8
        most = min(8192 * 4 * 4096 // (n * hidden), 16384)
        if dynamic:
            most = min(most, 8192 * 4 * 4096 * 24 // (n * hidden * (n * n + 2 * n)))
        if n > 8:
            most = min(most, 1024)
        return _layer(None, _log(rng, 16, max(most, 17)), n, hidden, dtype, fmt, dynamic)
    head_dim = rng.choice((64, 128, 128, 128, 80, 96, 112, 192, 256, 72))
    rotary = rng.choice((head_dim, head_dim, head_dim, head_dim // 2 // 2 * 2))
    kv = rng.choice((1, 2, 4, 8, 8, 13))
    heads = min(kv * rng.choice((1, 4, 5, 8)), 64)
    train = rng.random() < 0.7
    most = 16384 * 64 * 128 // ((heads + kv) * head_dim)
    tokens = _log(rng, 16, min(most, 16384)) if train else _log(rng, 1, 1024)
    return _qk(None, tokens, heads, kv, head_dim, rotary, dtype, _log(rng, 2048, 131072), rng.random() < 0.4, train,
               rng.choice((fmt, "")) if train else "")


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


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    kind = case["kind"]
    s = {"case": case}
    if kind == "pack":
        s["x"] = _rows(g, (case["rows"], case["hidden"]), dt)
        return s
    if kind == "rmsnorm":
        T, C = case["rows"], case["hidden"]
        s["x"] = _rows(g, (T, C), dt).requires_grad_(True)
        s["params"] = [_randn(g, C, std=0.1, mean=1.0).requires_grad_(True)]
        s["cot"] = _randn(g, T, C, dtype=dt)
        return s
    if kind == "layer":
        T, n, C = case["tokens"], case["n"], case["hidden"]
        s["x"] = _rows(g, (T, n, C), dt).requires_grad_(True)
        # the RMSNorm weight as the module keeps it: bf16, or fp32 after .float()
        p = [_randn(g, C, std=0.1, mean=1.0, dtype=dt)]
        if case["dynamic"]:
            p += [_randn(g, n, n * C, std=0.02), _randn(g, n, n * C, std=0.02), _randn(g, n * n, n * C, std=0.02)]
            p += [torch.tensor(0.1, device="cuda") for _ in range(3)]
            p += [_randn(g, n, std=0.3), _randn(g, n, std=0.3), _randn(g, n, n, std=0.3)]
        else:
            p += [_randn(g, n, std=0.5), _randn(g, n, std=0.5), _randn(g, n, n, std=0.5)]
        s["params"] = [t.requires_grad_(True) for t in p]
        s["cot"] = _randn(g, T, n, C)
        return s
    T, H, K, D = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    # queries, keys and values as one projection leaves them
    qkv = _rows(g, (T, H + 2 * K, D), dt)
    s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + K]
    s["params"] = [_randn(g, D, std=0.1, mean=1.0, dtype=dt) for _ in range(2)]
    freq = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"])
    angle = torch.arange(case["context"], device="cuda", dtype=torch.float64).unsqueeze(1) * freq
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["positions"] = torch.randint(case["context"], (T,), device="cuda", generator=g)
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
    kind, fmt = case["kind"], case["format"] or None
    if kind == "pack":
        return mhc.activation_unpack(mhc.activation_pack(s["x"], fmt))
    if kind == "qk":
        call = (s["q"], s["k"], *s["params"], s["cos"], s["sin"], s["positions"])
        if not case["train"]:
            with torch.no_grad():
                return mhc.qk_norm_rope(*call, interleaved=case["interleaved"])
        out = mhc.qk_norm_rope(*call, interleaved=case["interleaved"], checkpoint=fmt)
        grads = torch.autograd.grad(out, [s["q"], s["k"], *s["params"]], s["cot"])
        return (*[o.detach() for o in out], *grads)
    if kind == "rmsnorm":
        out = mhc.rmsnorm(s["x"], *s["params"], checkpoint=fmt)
    elif case["dynamic"]:
        out = mhc.mhc_layer_fused_dynamic_training(s["x"], *s["params"], checkpoint=fmt)
    else:
        out = mhc.mhc_layer_static(s["x"], *s["params"], checkpoint=fmt)
    grads = torch.autograd.grad(out, [s["x"], *s["params"]], s["cot"])
    return (out.detach(), *grads)


# The plain form: 32-bit torch operations, rounded once at the end.

def _blocks(x):
    pad = -x.shape[-1] % 32
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:-1], pad)], -1)
    return x.reshape(*x.shape[:-1], -1, 32)


def _checkpoint(x, fmt):
    """x^ of fp32 x, in bit arithmetic on fp32 numbers."""
    if not fmt:
        return x
    b = _blocks(x)
    a = b.abs().amax(-1, keepdim=True).view(torch.int32)
    # e + 127: the exponent field less that of the format's largest value, one
    # more where the mantissa is past its mantissa (127 = 1.984375 * 2^6, 448 =
    # 1.75 * 2^8)
    past, top = (0x7E0000, 6) if fmt == "int8" else (0x600000, 8)
    e = (((a + (0x7FFFFF - past)) >> 23) - top).clamp_min_(27)
    up = ((254 - e) << 23).view(torch.float32)
    down = (e << 23).view(torch.float32)
    v = b * up
    if fmt == "int8":
        v = v.round()
    else:
        # three mantissa bits, subnormal steps of 2^-9 below 2^-6
        step = (v.view(torch.int32) >> 23 & 255).clamp_min_(121) - 3
        v = (v * ((254 - step) << 23).view(torch.float32)).round() * (step << 23).view(torch.float32)
    v = torch.where(a >= 0x7F800000, float("nan"), v * down)
    return v.reshape(*x.shape[:-1], -1)[..., :x.shape[-1]]


def _norm(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * w


def _sinkhorn(a):
    for _ in range(_ITERS):
        a = a / (a.sum(-1, keepdim=True) + _SK_EPS)
        a = a / (a.sum(-2, keepdim=True) + _SK_EPS)
    return a


def _mix(x, w, h_pre, h_post, m):
    y = _norm((h_pre.unsqueeze(-1) * x).sum(1), w)
    return torch.matmul(m, x) + h_post.unsqueeze(-1) * y.unsqueeze(1)


def _plain_layer(x, held, p, dynamic):
    """The layer on rows x; with `held` the dynamic coefficients' products and
    mean squares take those values, at x's gradient.  The coefficients and the
    sums over tokens of their gradients are in 64 bits: those cancel through
    the normalisations."""
    T, n, C = x.shape
    if not dynamic:
        w, a, b, c = p
        a, b, c = a.double(), b.double(), c.double()
        coefs = (torch.sigmoid(a).expand(T, n), 2 * torch.sigmoid(b).expand(T, n),
                 _sinkhorn(c.exp()).expand(T, n, n))
        return _mix(x, w, *[v.float() for v in coefs])
    w, p_pre, p_post, p_res, a_pre, a_post, a_res, b_pre, b_post, b_res = p
    flat = x.reshape(T, -1)
    prod = flat @ torch.cat([p_pre, p_post, p_res]).t()
    ms = (flat * flat).mean(-1, keepdim=True)
    if held is not None:
        hf = held.reshape(T, -1)
        with torch.no_grad():
            d_prod = hf @ torch.cat([p_pre, p_post, p_res]).t() - prod
            d_ms = (hf * hf).mean(-1, keepdim=True) - ms
        prod, ms = prod + d_prod, ms + d_ms
    t = prod.double() / torch.sqrt(ms + _EPS)
    h_pre = torch.sigmoid(a_pre.double() * t[:, :n] + b_pre.double())
    h_post = 2 * torch.sigmoid(a_post.double() * t[:, n:2 * n] + b_post.double())
    m = _sinkhorn((a_res.double() * t[:, 2 * n:].reshape(T, n, n) + b_res.double()).exp())
    return _mix(x, w, h_pre.float(), h_post.float(), m.float())


def _plain_rope(x, w, cos, sin, interleaved):
    y = _norm(x, w)
    R = 2 * cos.shape[-1]
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    a, b = (y[..., 0:R:2], y[..., 1:R:2]) if interleaved else (y[..., :R // 2], y[..., R // 2:R])
    pair = (a * c - b * s, b * c + a * s)
    rot = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([rot, y[..., R:]], -1)


def _run_plain(s):
    case = s["case"]
    kind, fmt = case["kind"], case["format"]
    dt = _DTYPES[case["dtype"]]
    with torch.no_grad():
        if kind == "pack":
            return _checkpoint(s["x"].float(), fmt).to(dt)
        p32 = [t.float() for t in s["params"]]
        if kind == "qk":
            xs = [s["q"].float(), s["k"].float()]
            cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
            fs = [lambda x, p, i=i: _plain_rope(x, p[i], cos, sin, case["interleaved"]) for i in range(2)]
            cots, out_dt = s.get("cot"), dt
        else:
            xs = [s["x"].float()]
            cots = [s["cot"]]
            if kind == "rmsnorm":
                fs, out_dt = [lambda x, p: _norm(x, p[0])], dt
            else:
                held = xs[0] if case["dynamic"] else None
                fs, out_dt = [lambda x, p: _plain_layer(x, held, p, case["dynamic"])], torch.float32
        outs = [f(x, p32).to(out_dt) for f, x in zip(fs, xs)]
        if cots is None:
            return tuple(outs)
    hats = [_checkpoint(x, fmt).requires_grad_(True) for x in xs]
    ps = [t.detach().requires_grad_(True) for t in p32]
    again = [f(x, ps) for f, x in zip(fs, hats)]
    grads = torch.autograd.grad(again, hats + ps, [c.float() for c in cots])
    types = [dt] * len(hats) + [t.dtype for t in s["params"]]
    return (*outs, *[g.to(t) for g, t in zip(grads, types)])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    """A checkpoint counts once where the forward writes it and once where the
    backward reads it: the rest of the step runs between the two."""
    size = 2 if case["dtype"] == "bf16" else 4
    kind, fmt = case["kind"], case["format"]

    def held(rows, hidden):
        return rows * (hidden + (hidden + 31) // 32)

    if kind == "pack":
        E = case["rows"] * case["hidden"]
        return {"bytes": 2 * E * size + 2 * held(case["rows"], case["hidden"]), "flops": 4 * E}
    if kind == "rmsnorm":
        E = case["rows"] * case["hidden"]
        # x in, out out; cotangent in, gradient out
        return {"bytes": 4 * E * size + 2 * held(case["rows"], case["hidden"]) + 8 * case["hidden"],
                "flops": 16 * E}
    if kind == "layer":
        T, n, C = case["tokens"], case["n"], case["hidden"]
        E, rows = T * n * C, n * n + 2 * n
        nbytes = E * (2 * size + 8) + 2 * held(T * n, C) + 2 * C * size
        flops = 3 * T * C * (2 * n * n + 4 * n)
        if case["dynamic"]:
            nbytes += 2 * rows * n * C * 4
            flops += 3 * 2 * E * rows
        return {"bytes": nbytes, "flops": flops}
    rows, D = case["tokens"] * (case["heads"] + case["kv_heads"]), case["head_dim"]
    nbytes = 2 * rows * D * size + min(case["tokens"], case["context"]) * case["rotary"] * 4
    if case["train"]:
        # cotangent in, gradient out; the rows again, as they were kept
        nbytes += 2 * rows * D * size + (2 * held(rows, D) if fmt else rows * D * size)
    return {"bytes": nbytes, "flops": (22 if case["train"] else 8) * rows * D}


# ---------------------------------------------------------------------------
# The same in 64 bits, gradients by their formulas
# ---------------------------------------------------------------------------

def _exact_held(x, fmt):
    """x^ by its definition, fp64."""
    if not fmt:
        return x
    top = _MAX[fmt]
    b = _blocks(x)
    a = b.abs().amax(-1, keepdim=True)
    # least e with a <= top 2^e: frexp gives a / top = m 2^k with 1/2 <= m < 1,
    # or exactly a power of two at m = 1/2
    m, k = torch.frexp(a / top)
    # a / top is rounded: settle the edge by comparing exactly
    e = k.double() - 1
    e = torch.where(a <= top * torch.exp2(e), e, e + 1)
    e = torch.where(a > 0, e, torch.full_like(e, -100.0)).clamp_min(-100.0)
    v = b * torch.exp2(-e)
    if fmt == "int8":
        q = torch.round(v)
    else:
        _, kv = torch.frexp(v)
        step = torch.exp2((kv.double() - 1).clamp_min(-6.0) - 3)
        q = torch.round(v / step) * step
    q = (q * torch.exp2(e)).reshape(*x.shape[:-1], -1)
    return q[..., :x.shape[-1]]


def _exact_norm_back(x, w, u):
    """Gradients of x / r * w for cotangent u: rows, and the terms of w's."""
    r = torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS)
    dot = (u * w * x).sum(-1, keepdim=True)
    return u * w / r - x * dot / (x.shape[-1] * r ** 3), u * x / r


def _exact_sinkhorn(a):
    steps = []
    for _ in range(_ITERS):
        r = a.sum(2, keepdim=True) + _SK_EPS
        b = a / r
        c = b.sum(1, keepdim=True) + _SK_EPS
        a = b / c
        steps.append((r, b, c, a))
    return a, steps


def _exact_sinkhorn_back(steps, g):
    for r, b, c, a in reversed(steps):
        g = (g - (g * a).sum(1, keepdim=True)) / c
        g = (g - (g * b).sum(2, keepdim=True)) / r
    return g


def _exact_layer(case, s):
    n, C, T = case["n"], case["hidden"], case["tokens"]
    x = s["x"].detach().double()
    xh = _exact_held(x, case["format"])
    p = [t.detach().double() for t in s["params"]]
    g = s["cot"].double()
    w = p[0]
    if case["dynamic"]:
        phi = torch.cat(p[1:4])
        alpha = torch.cat([p[4].expand(n), p[5].expand(n), p[6].expand(n * n)])
        bias = torch.cat([p[7], p[8], p[9].reshape(-1)])
        rh = torch.sqrt(x.reshape(T, -1).square().mean(-1, keepdim=True) + _EPS)
        prod = x.reshape(T, -1) @ phi.t()
        t = alpha * prod / rh + bias
    else:
        t = torch.cat([p[1], p[2], p[3].reshape(-1)]).unsqueeze(0)
    pre, post = torch.sigmoid(t[:, :n]), 2 * torch.sigmoid(t[:, n:2 * n])
    ex = torch.exp(t[:, 2 * n:]).reshape(-1, n, n)
    m, steps = _exact_sinkhorn(ex)

    def rows(v):  # aggregate and its norm
        agg = (pre[..., None] * v).sum(1)
        return agg, torch.sqrt(agg.square().mean(-1, keepdim=True) + _EPS)

    def mixed(mat, v):  # sum_j mat[., i, j] v[., j, :]
        return torch.stack([(mat[:, i, :, None] * v).sum(1) for i in range(n)], 1)

    agg, r = rows(x)
    out = mixed(m, x) + post[..., None] * (agg / r * w).unsqueeze(1)
    del x
    agg, r = rows(xh)
    gy = (post[..., None] * g).sum(1)
    dagg, dw = _exact_norm_back(agg, w, gy)
    dx = mixed(m.transpose(1, 2), g) + pre[..., None] * dagg.unsqueeze(1)
    dm = torch.stack([(g[:, i, None, :] * xh).sum(-1) for i in range(n)], 1)
    dpost = (g * (agg / r * w).unsqueeze(1)).sum(-1)
    dpre = (dagg.unsqueeze(1) * xh).sum(-1)
    if not case["dynamic"]:
        dm, dpost, dpre = (v.sum(0, keepdim=True) for v in (dm, dpost, dpre))
    dt = torch.cat([dpre * pre * (1 - pre), dpost * post * (1 - post / 2),
                    (_exact_sinkhorn_back(steps, dm) * ex).reshape(-1, n * n)], 1)
    dw = dw.sum(0)
    if not case["dynamic"]:
        d = dt[0]
        return out, dx, dw, d[:n], d[n:2 * n], d[2 * n:].reshape(n, n)
    u = dt * alpha
    dprod = u / rh
    drh = -(u * prod).sum(-1, keepdim=True) / rh.square()
    flat = xh.reshape(T, -1)
    dx = dx + (dprod @ phi + drh / (n * C * rh) * flat).reshape(T, n, C)
    dphi = dprod.t() @ flat
    da = (dt * prod / rh).sum(0)
    db = dt.sum(0)
    return (out, dx, dw, dphi[:n], dphi[n:2 * n], dphi[2 * n:], da[:n].sum(), da[n:2 * n].sum(), da[2 * n:].sum(),
            db[:n], db[n:2 * n], db[2 * n:].reshape(n, n))


def _exact_turn(v, cos, sin, interleaved, sign):
    """Rotation of v's pairs by +angle (sign 1) or -angle (sign -1)."""
    R = 2 * cos.shape[-1]
    i = torch.arange(R // 2, device=v.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    c, s = cos.double().unsqueeze(1), sign * sin.double().unsqueeze(1)
    res = v.clone()
    res[..., lo] = v[..., lo] * c - v[..., hi] * s
    res[..., hi] = v[..., hi] * c + v[..., lo] * s
    return res


def exact(case, seed):
    s = prepare(case, seed)
    kind, fmt = case["kind"], case["format"]
    with torch.no_grad():
        if kind == "pack":
            return _exact_held(s["x"].double(), fmt)
        if kind == "layer":
            return _exact_layer(case, s)
        p = [t.detach().double() for t in s["params"]]
        if kind == "rmsnorm":
            x = s["x"].detach().double()
            out = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * p[0]
            dx, dw = _exact_norm_back(_exact_held(x, fmt), p[0], s["cot"].double())
            return out, dx, dw.sum(0)
        cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
        outs, rows, weights = [], [], []
        for i, key in enumerate(("q", "k")):
            x = s[key].detach().double()
            y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * p[i]
            outs.append(_exact_turn(y, cos, sin, case["interleaved"], 1.0))
            if case["train"]:
                u = _exact_turn(s["cot"][i].double(), cos, sin, case["interleaved"], -1.0)
                dx, dw = _exact_norm_back(_exact_held(x, fmt), p[i], u)
                rows.append(dx)
                weights.append(dw.sum((0, 1)))
        return (*outs, *rows, *weights)
