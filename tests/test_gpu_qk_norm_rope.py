"""Per-head norm of queries and keys with the rotation of positions, against
the 64-bit oracle; with a checkpoint, gradients at the values it stands for."""
import pytest
import torch

import mhc_ascend_amd as mhc
from oracle import rows8
from tests.test_gpu_checkpoint import U, _within
from tests.test_gpu_graph import _capture, _replays

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
# Sums over a head take at most 16 values a lane and 6 steps across lanes; a
# rotation, two products and their sum: 48 of 2^-24 on each term.  A weight's
# gradient adds rows one by one within a workgroup (every lane at most rows /
# 64 of them), then 8 + 128 partials.
K_ROW, K_DW = 48, 600


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(T, H, K, D, dtype, seed, w_dtype=None):
    g = _gen(seed)
    q, k = (torch.randn(T, h, D, generator=g).to(dtype) for h in (H, K))
    ws = [(1 + 0.2 * torch.randn(D, generator=g)).to(w_dtype or dtype) for _ in range(2)]
    cots = [torch.randn(T, h, D, generator=g).to(dtype) for h in (H, K)]
    return q, k, ws, cots


def _one(x, w, cot, cos, sin, interleaved, fmt, eps=1e-5):
    """Output at x; gradients at x^ and the magnitudes of their terms."""
    out = rows8.qk_norm_rope(x.double(), w.double(), cos, sin, eps, interleaved)
    xh = rows8.held(x, fmt).requires_grad_(True)
    wd = w.double().requires_grad_(True)
    rows8.qk_norm_rope(xh, wd, cos, sin, eps, interleaved).backward(cot.double())
    D = x.shape[-1]
    with torch.no_grad():
        v = xh.detach()
        r = torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
        # |u|: both products of a pair, |c| and |s| at most 1
        half = cos.shape[-1]
        full = cot.double().abs().clone()
        for p in range(half):
            lo, hi = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
            pair = cot.double()[..., lo].abs() + cot.double()[..., hi].abs()
            full[..., lo] = pair
            full[..., hi] = pair
        mag = (w.double() * full / r).abs() + v.abs() * (full * w.double() * v).abs().sum(-1, keepdim=True) / (D * r ** 3)
        mag_w = (full * v / r).abs().sum((0, 1))
        y = (x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps) * w.double()).abs()
        mag_o = y.clone()
        for p in range(half):
            lo, hi = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
            mag_o[..., lo] = mag_o[..., hi] = y[..., lo] + y[..., hi]
    return out, mag_o, xh.grad, mag, wd.grad, mag_w


def _check(got, inputs, cos, sin, interleaved, fmt):
    q, k, ws, cots = inputs
    dt = q.dtype
    u = U[dt] if dt == torch.bfloat16 else 0.0
    uw = U[torch.bfloat16] if ws[0].dtype == torch.bfloat16 else 0.0
    for i, x in enumerate((q, k)):
        if x.numel() == 0:
            assert got[i].shape == x.shape and got[2 + i].shape == x.shape and bool((got[4 + i] == 0).all())
            continue
        out, mag_o, dx, mag, dw, mag_w = _one(x, ws[i], cots[i], cos, sin, interleaved, fmt)
        assert got[i].dtype == dt and got[2 + i].dtype == dt and got[4 + i].dtype == ws[i].dtype
        assert got[i].is_contiguous()
        _within(got[i], out, K_ROW * 2.0 ** -24 * mag_o + u * out.abs() + 1e-30, f"out {i}")
        _within(got[2 + i], dx, K_ROW * 2.0 ** -24 * mag + u * dx.abs() + 1e-30, f"dx {i}")
        _within(got[4 + i], dw, K_DW * 2.0 ** -24 * mag_w + uw * dw.abs() + 1e-30, f"dw {i}")


def _run(device, inputs, cos, sin, positions, interleaved, fmt, cots=None):
    q, k, ws, c = inputs
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, *ws)]
    out = mhc.qk_norm_rope(*leaves, cos.to(device), sin.to(device), positions, interleaved=interleaved, checkpoint=fmt)
    grads = torch.autograd.grad(out, leaves, cots or [t.to(device) for t in c])
    return [*[o.detach() for o in out], *grads]


SHAPES = [  # tokens, heads, kv heads, D, R
    (1, 1, 1, 2, 2), (3, 2, 1, 6, 4), (5, 4, 4, 64, 64), (130, 5, 2, 64, 32), (33, 13, 3, 72, 72), (17, 3, 3, 80, 40),
    (1, 32, 8, 128, 128), (67, 32, 8, 128, 128), (9, 6, 1, 128, 126), (21, 3, 2, 96, 96), (7, 2, 2, 112, 56),
    (11, 2, 1, 192, 64), (40, 4, 2, 256, 256), (3, 2, 2, 257, 256), (4, 1, 2, 512, 512), (2, 3, 1, 1000, 8),
    (2, 1, 1, 1024, 1024), (700, 3, 1, 64, 64), (2, 5, 0, 64, 64), (0, 4, 2, 64, 64), (1100, 8, 4, 128, 128)]


@pytest.mark.parametrize("T,H,K,D,Rd", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
def test_matches_oracle(device, T, H, K, D, Rd, interleaved, dtype, fmt):
    inputs = _inputs(T, H, K, D, dtype, T + H + D)
    cos, sin = mhc.rope_table(5000, Rd)
    pos = torch.randint(5000, (T,), generator=_gen(T))
    got = _run(device, inputs, cos, sin, pos.to(device), interleaved, fmt)
    _check([g.cpu() for g in got], inputs, cos[pos], sin[pos], interleaved, fmt)


# Few heads and many tokens: several tokens a wave, the last wave's not all there.
@pytest.mark.parametrize("T,H,K,D,Rd", [(4099, 1, 1, 64, 64), (9001, 4, 1, 72, 36), (9003, 2, 2, 80, 80),
                                        (16391, 2, 1, 128, 128), (5003, 5, 0, 64, 32), (4501, 0, 1, 256, 256),
                                        (33001, 1, 1, 32, 32), (20001, 3, 3, 64, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
def test_several_tokens_a_wave(device, T, H, K, D, Rd, interleaved, dtype, fmt):
    test_matches_oracle(device, T, H, K, D, Rd, interleaved, dtype, fmt)


@pytest.mark.parametrize("w_dtype", DTYPES)
def test_weights_of_another_dtype(device, w_dtype):
    dtype = torch.bfloat16 if w_dtype == torch.float32 else torch.float32
    inputs = _inputs(9, 3, 2, 64, dtype, 1, w_dtype)
    cos, sin = mhc.rope_table(16, 64)
    got = _run(device, inputs, cos, sin, None, False, None)
    _check([g.cpu() for g in got], inputs, cos[:9], sin[:9], False, None)


@pytest.mark.parametrize("kind", ["count", "int32", "int64", "strided"])
@pytest.mark.parametrize("shape", ["tokens", "batch"])
def test_positions(device, kind, shape):
    """[tokens, heads, D] and [batch, seq, heads, D], positions counted, per
    token, or one sequence's for every batch."""
    T, S = 24, 8
    inputs = _inputs(T, 3, 2, 64, torch.float32, 2)
    q, k, ws, cots = inputs
    cos, sin = mhc.rope_table(100, 64)
    lead = (T,) if shape == "tokens" else (T // S, S)
    if kind == "count":
        pos, table = None, torch.arange(T) if shape == "tokens" else torch.arange(S).repeat(T // S)
    else:
        n = S if (kind == "int32" and shape == "batch") else T
        p = torch.randint(100, (n,), generator=_gen(3))
        table = p if n == T else p.repeat(T // S)
        pos = p.to(torch.int32 if kind == "int32" else torch.int64).to(device)
        if kind == "strided":
            pos = torch.stack([pos, pos * 0], 1)[:, 0]
        pos = pos.view(lead) if n == T else pos
    leaves = [t.to(device).requires_grad_(True) for t in (q.view(*lead, 3, 64), k.view(*lead, 2, 64), *ws)]
    out = mhc.qk_norm_rope(*leaves, cos.to(device), sin.to(device), pos)
    assert out[0].shape == leaves[0].shape and out[1].shape == leaves[1].shape
    grads = torch.autograd.grad(out, leaves, [c.to(device).view(o.shape) for c, o in zip(cots, out)])
    got = [t.detach().cpu() for t in (*out, *grads)]
    got = [g.reshape(T, *g.shape[-2:]) if g.dim() > 1 else g for g in got]
    _check(got, inputs, cos[table], sin[table], False, None)


@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_views_of_a_joint_projection(device, D, fmt, dtype):
    """q and k as slices of [T, heads, D] and, unaligned, of a flat buffer with
    an odd token stride; cotangents with heads before tokens.  Bit for bit the
    contiguous call's."""
    T, H, K = 37, 6, 2
    inputs = _inputs(T, H, K, D, dtype, 4)
    cos, sin = (t.to(device) for t in mhc.rope_table(64, D))
    want = _run(device, inputs, cos.cpu(), sin.cpu(), None, False, fmt)
    q, k, ws, cots = inputs
    for extra, off in ((D, 0), (3, 1)):
        buf = torch.zeros(T * ((H + K) * D + extra) + 8, dtype=dtype, device=device)
        row = (H + K) * D + extra
        qv = buf.as_strided((T, H, D), (row, D, 1), off)
        kv = buf.as_strided((T, K, D), (row, D, 1), off + H * D)
        qv.copy_(q)
        kv.copy_(k)
        leaves = [t.detach().requires_grad_(True) for t in (qv, kv, *[w.to(device) for w in ws])]
        out = mhc.qk_norm_rope(*leaves, cos, sin, checkpoint=fmt)
        cv = [c.to(device).transpose(0, 1).contiguous().transpose(0, 1) for c in cots]
        got = [*[o.detach() for o in out], *torch.autograd.grad(out, leaves, cv)]
        # sums in another order where the rows cannot be read in whole pieces
        for a, e in zip(got, want):
            assert a.shape == e.shape
        _check([g.cpu() for g in got], inputs, cos.cpu()[:T], sin.cpu()[:T], False, fmt)


def test_expanded_keys(device):
    """Keys repeated to the query heads by expand (head stride 0): their
    gradient is the sum over the repeats."""
    q, k, ws, cots = _inputs(9, 4, 1, 64, torch.float32, 11)
    cos, sin = (t.to(device) for t in mhc.rope_table(9, 64))
    kd = k.to(device).requires_grad_(True)
    leaves = [q.to(device).requires_grad_(True), kd, *[w.to(device).requires_grad_(True) for w in ws]]
    out = mhc.qk_norm_rope(leaves[0], kd.expand(9, 4, 64), *leaves[2:], cos, sin)
    g = [cots[0].to(device), torch.randn(9, 4, 64, generator=_gen(12)).to(device)]
    got = [*[o.detach() for o in out], *torch.autograd.grad(out, leaves, g)]
    # the sum of four rounded rows instead of one row's: four roundings, held by
    # the row bound's 48
    want = (q, k, ws, [cots[0], g[1].cpu().sum(1, keepdim=True)])
    _check([got[0].cpu(), got[1][:, :1].contiguous().cpu(), *[t.cpu() for t in got[2:]]], want, cos.cpu(), sin.cpu(),
           False, None)


def test_expanded_cotangents(device):
    inputs = _inputs(6, 3, 2, 64, torch.float32, 5)
    q, k, ws, _ = inputs
    cos, sin = mhc.rope_table(6, 64)
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, *ws)]
    out = mhc.qk_norm_rope(*leaves, cos.to(device), sin.to(device))
    grads = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves)
    ones = [torch.ones_like(q), torch.ones_like(k)]
    _check([t.detach().cpu() for t in (*out, *grads)], (q, k, ws, ones), cos, sin, False, None)


def test_only_one_output_used(device):
    q, k, ws, cots = _inputs(6, 3, 2, 64, torch.float32, 6)
    cos, sin = (t.to(device) for t in mhc.rope_table(6, 64))
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, *ws)]
    out = mhc.qk_norm_rope(*leaves, cos, sin)
    grads = torch.autograd.grad(out[0], leaves, cots[0].to(device))
    assert bool((grads[1] == 0).all()) and bool((grads[3] == 0).all()) and bool((grads[0] != 0).any())


@pytest.mark.parametrize("D", [64, 66])
def test_positions_outside_the_table_are_nan(device, D):
    """In bounds on the device, loud in the result; the other rows stay."""
    q, k, ws, cots = _inputs(6, 3, 2, D, torch.float32, 7)
    cos, sin = (t.to(device) for t in mhc.rope_table(10, 64))
    pos = torch.tensor([0, 10, 3, -1, 2 ** 40, 9], device=device)
    bad = torch.tensor([False, True, False, True, True, False])
    leaves = [t.to(device).requires_grad_(True) for t in (q, k, *ws)]
    out = mhc.qk_norm_rope(*leaves, cos, sin, pos)
    grads = torch.autograd.grad(out, leaves, [c.to(device) for c in cots])
    for t in (*out, *grads[:2]):
        assert torch.equal(t.detach().cpu().isnan().all(-1).all(-1), bad)
        assert torch.equal(t.detach().cpu().isnan().any(-1).any(-1), bad)
    assert bool(grads[2].isnan().all())


@pytest.mark.parametrize("fmt", [None, "e4m3"])
def test_rows_that_are_not_finite(device, fmt):
    q, k, ws, cots = _inputs(5, 2, 2, 64, torch.float32, 8)
    q[1, 0, 3] = float("nan")
    k[2, 1, 63] = float("inf")
    cos, sin = mhc.rope_table(5, 64)
    got = _run(device, (q, k, ws, cots), cos, sin, None, False, fmt)
    bad_q, bad_k = torch.zeros(5, 2, dtype=torch.bool), torch.zeros(5, 2, dtype=torch.bool)
    bad_q[1, 0] = bad_k[2, 1] = True
    for t, bad in zip(got[2:4], (bad_q, bad_k)):
        assert torch.equal((~t.cpu().isfinite()).any(-1), bad)
    assert torch.equal(got[0].cpu().isnan().any(-1), bad_q)


def test_gradient_against_differences(device):
    """As the norm's (tests/test_gpu_checkpoint.py), through the rotation."""
    g = _gen(9)
    x = mhc.activation_unpack(mhc.activation_pack(torch.randn(16, 4, 64, generator=g).to(device)))
    k = mhc.activation_unpack(mhc.activation_pack(torch.randn(16, 2, 64, generator=g).to(device)))
    ws = [(1 + 0.1 * torch.randn(64, generator=g)).to(device) for _ in range(2)]
    cos, sin = (t.to(device) for t in mhc.rope_table(16, 64))
    cots = [torch.randn(t.shape, generator=g).to(device) for t in (x, k)]
    vals = [x, k, *ws]
    leaves = [v.clone().requires_grad_(True) for v in vals]
    grads = torch.autograd.grad(mhc.qk_norm_rope(*leaves, cos, sin, checkpoint="int8"), leaves, cots)

    def loss(vs):
        return sum(float((o.double() * c.double()).sum()) for o, c in zip(mhc.qk_norm_rope(*vs, cos, sin), cots))

    h = 2.0 ** -6
    noise = 64 * 2.0 ** -24 * sum(float((o * c).double().abs().sum())
                                  for o, c in zip(mhc.qk_norm_rope(*vals, cos, sin), cots)) / h
    for i, v in enumerate(vals):
        d = torch.randn(v.shape, generator=g).to(device)
        hi, lo = list(vals), list(vals)
        hi[i], lo[i] = v + h * d, v - h * d
        diff = (loss(hi) - loss(lo)) / (2 * h)
        want = (grads[i].double() * d.double())
        # third derivatives grow with the norm's 1/r^3 on short rows: 5e-3
        assert abs(diff - float(want.sum())) <= 5e-3 * float(want.abs().sum()) + noise, i


def test_refusals(device):
    q, k = torch.zeros(4, 2, 64, device=device), torch.zeros(4, 1, 64, device=device)
    w = torch.ones(64, device=device)
    cos, sin = (t.to(device) for t in mhc.rope_table(8, 64))
    bad = [((q, k.bfloat16(), w, w, cos, sin), "one floating dtype"), ((q.int(), k.int(), w, w, cos, sin), "dtype"),
           ((q, k, w[:32], w, cos, sin), "weights"), ((q, k, w, w, cos, sin[:4]), "cos and sin"),
           ((q, k, w, w, cos.requires_grad_(True), sin), "no gradient"),
           ((q, k, w, w, cos.detach(), sin, torch.zeros(4, device=device)), "int64 or int32"),
           ((q, k, w, w, cos.detach(), sin, torch.zeros(4, dtype=torch.int64)), "HIP device"),
           ((q, k, w, w, cos.detach().repeat(1, 2), sin.repeat(1, 2)), "rotary_dim"),
           ((q, k, w, w, cos.detach()[:0], sin[:0]), "rows")]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            mhc.qk_norm_rope(*args)
    wide = torch.zeros(1, 1, 1026, device=device)
    with pytest.raises(RuntimeError, match="head_dim"):
        mhc.qk_norm_rope(wide, wide, torch.ones(1026, device=device), torch.ones(1026, device=device), cos.detach(), sin)


@pytest.mark.parametrize("D", [128, 66])
@pytest.mark.parametrize("fmt", [None, "int8"])
def test_offsets_past_32_bits(device, D, fmt):
    """More than 2^32 values of q: the last tokens against a call on them."""
    H, K = 64, 1
    T = (1 << 32) // (H * D) + 70
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device=device).fill_(0.5)
    k = torch.empty(T, K, D, dtype=torch.bfloat16, device=device).fill_(0.5)
    q[-64:] = torch.randn(64, H, D, device=device).bfloat16()
    k[-64:] = torch.randn(64, K, D, device=device).bfloat16()
    w = (torch.rand(D, device=device) + 0.5).bfloat16()
    cos, sin = (t.to(device) for t in mhc.rope_table(1024, 64))
    pos = torch.arange(T, device=device) % 1024
    outs = []
    for a, b, p in ((q, k, pos), (q[-64:].clone(), k[-64:].clone(), pos[-64:])):
        leaves = [t.detach().requires_grad_(True) for t in (a, b)]
        out = mhc.qk_norm_rope(*leaves, w, w, cos, sin, p, checkpoint=fmt)
        grads = torch.autograd.grad(out, leaves, [a, b])
        outs.append([t.detach()[-64:].clone() for t in (*out, *grads)])
        del out, grads, leaves
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_step_replays_in_a_graph(device, fmt):
    T = 40
    q, k = torch.randn(T, 8, 128, device=device), torch.randn(T, 2, 128, device=device)
    ws = [torch.rand(128, device=device) + 0.5 for _ in range(2)]
    cots = [torch.randn_like(q), torch.randn_like(k)]
    pos = torch.arange(T, device=device)
    cos, sin = (t.to(device) for t in mhc.rope_table(512, 128))

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, *ws)]
        out = mhc.qk_norm_rope(*leaves, cos, sin, pos, checkpoint=fmt)
        return [*[o.detach() for o in out], *torch.autograd.grad(out, leaves, cots)]

    graph, outs = _capture(step)
    g = _gen(10)
    feeds = [lambda: q.copy_(torch.randn(q.shape, generator=g)), lambda: pos.add_(300),
             lambda: cots[1].copy_(torch.randn(k.shape, generator=g))]
    _replays(graph, outs, step, feeds)


def test_a_block_as_a_model_runs_it(device):
    """norm -> q, k -> qk_norm_rope -> attention -> hyper-connected residual,
    everything that has rows to keep keeping them in 8 bits; one training step
    against the same step in 64 bits with x^ where a checkpoint is read."""
    torch.manual_seed(3)
    T, C, H, D = 24, 64, 2, 32
    wrap = mhc.MHCResidualWrapper(C, 4, use_dynamic_h=False, checkpoint="int8").to(device)
    nw = (1 + 0.1 * torch.randn(C)).to(device).requires_grad_(True)
    wq, wk, wv = (0.2 * torch.randn(C, H * D) for _ in range(3))
    hw = [(1 + 0.1 * torch.randn(D)) for _ in range(2)]
    x = torch.randn(T, C)
    cos, sin = mhc.rope_table(T, D)
    cot = torch.randn(T, C)

    def block(x, nw, ws, hw, norm, qk, residual):
        h = norm(x, nw)
        q, k, v = ((h @ w).view(T, H, D) for w in ws)
        q, k = qk(q, k, *hw)
        a = torch.softmax(torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / D ** 0.5, -1)
        y = torch.matmul(a, v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(T, H * D)
        return residual(x, y)

    ws_d = [w.to(device).requires_grad_(True) for w in (wq, wk, wv)]
    hw_d = [w.to(device).requires_grad_(True) for w in hw]
    xd = x.to(device).requires_grad_(True)
    out = block(xd, nw, ws_d, hw_d, lambda a, w: mhc.rmsnorm(a, w, checkpoint="int8"),
                lambda q, k, a, b: mhc.qk_norm_rope(q, k, a, b, cos.to(device), sin.to(device), checkpoint="e4m3"),
                wrap)
    leaves = [xd, nw, *ws_d, *hw_d]
    got = torch.autograd.grad(out, leaves, cot.to(device))

    class At(torch.autograd.Function):  # value at x, gradient of f at x^
        @staticmethod
        def forward(ctx, f, fmt, nx, *args):
            ctx.f, ctx.fmt, ctx.nx = f, fmt, nx
            ctx.save_for_backward(*args)
            return f(*args)

        @staticmethod
        def backward(ctx, g):
            args = list(ctx.saved_tensors)
            # the rows are packed as the fp32 path holds them
            args = [rows8.held(a.float(), ctx.fmt) if i < ctx.nx else a for i, a in enumerate(args)]
            args = [a.detach().requires_grad_(True) for a in args]
            with torch.enable_grad():
                return (None, None, None, *torch.autograd.grad(ctx.f(*args), args, g))

    m = wrap.mhc
    pre, post = torch.sigmoid(m.H_pre.detach().cpu().double()), 2 * torch.sigmoid(m.H_post.detach().cpu().double())
    from oracle import reference as R
    mix = R.sinkhorn_knopp(torch.exp(m.H_res.detach().cpu().double()), 20, 1e-8)
    rw = m.rmsnorm_weight.detach().cpu().double()

    def residual(r, b):
        s = torch.stack([r, b, r * 0.1, r * 0.01], 1)
        return R._layer_core(s, rw, pre, post, mix, 1e-5).mean(1)

    def norm(a, w):
        return a / torch.sqrt(a.square().mean(-1, keepdim=True) + 1e-5) * w

    def rot(a, w):
        return rows8.qk_norm_rope(a, w, cos, sin)

    xr = x.double().requires_grad_(True)
    nr = nw.detach().cpu().double().requires_grad_(True)
    ws_r = [w.double().requires_grad_(True) for w in (wq, wk, wv)]
    hw_r = [w.double().requires_grad_(True) for w in hw]
    ref = block(xr, nr, ws_r, hw_r, lambda a, w: At.apply(norm, "int8", 1, a, w),
                lambda q, k, a, b: (At.apply(rot, "e4m3", 1, q, a), At.apply(rot, "e4m3", 1, k, b)),
                lambda r, b: At.apply(residual, "int8", 2, r, b))
    want = torch.autograd.grad(ref, [xr, nr, *ws_r, *hw_r], cot.double())
    # fp32 throughout against 64 bits; a value within fp32 rounding of a half
    # step may be packed one step away, which moves one term of a gradient by a
    # step: 2^-3 of e4m3, 2^-6 of int8 relative to its block's largest.  Norms:
    # one such flip in a row of 64 is below 2e-2 of it, and rare.
    for a, e in zip((out.detach(), *got), (ref.detach(), *want)):
        assert float((a.cpu().double() - e).norm() / e.norm()) <= 2e-2
    ref = ref.detach()
    assert float((out.detach().cpu().double() - ref).norm() / ref.norm()) <= 1e-5


@pytest.mark.parametrize("T,D", [((1 << 24) + 64, 6), ((1 << 26) + 64, 8)])
def test_more_tokens_than_a_launch_takes(device, T, D):
    """2^32 lanes and more: the first and last tokens against calls on them alone."""
    P = 64
    q = torch.randn(P, 1, D, device=device).bfloat16().repeat(T // P, 1, 1).view(T // P, P, 1, D)
    q[-1] = q[-1] * 3 + 1
    k = q.new_empty(T // P, P, 0, D)
    w = torch.rand(D, device=device) + 0.5
    cos, sin = mhc.rope_table(P, D, device=device)
    with torch.no_grad():
        out = mhc.qk_norm_rope(q, k, w, w, cos, sin)[0]
        for at in (0, (1 << 23) // P, 4 * (1 << 23) // P, T // P - 1):
            if at >= T // P:
                continue
            want = mhc.qk_norm_rope(q[at:at + 1], k[at:at + 1], w, w, cos, sin)[0]
            assert torch.equal(out[at:at + 1], want)
        assert torch.equal(out[:-1], out[:1].expand_as(out[:-1]))


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_an_error(device, grad):
    """A tangent on any input is refused, with and without grad mode: a result
    that came back without one would be taken for a constant."""
    q, k, ws, _ = _inputs(5, 2, 1, 64, torch.float32, 3)
    cos, sin = mhc.rope_table(5, 64)
    args = [t.to(device) for t in (q, k, *ws, cos, sin)]
    want = mhc.qk_norm_rope(*args)
    for i in range(len(args)):
        with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad):
            call = [torch.autograd.forward_ad.make_dual(a, torch.ones_like(a)) if j == i else a
                    for j, a in enumerate(args)]
            with pytest.raises(RuntimeError, match="jvp is not implemented" if i < 4 else "no gradient"):
                mhc.qk_norm_rope(*call)
    assert all(torch.equal(a, b) for a, b in zip(mhc.qk_norm_rope(*args), want))
