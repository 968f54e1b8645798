"""8-bit checkpoints of rows and the backward passes that read them, against
the 64-bit oracle.  The format is exact: bytes and values are compared for
equality.  Gradients are those of the operator at the values x^ that a
checkpoint stands for; their tolerances are derived next to them."""
import gc

import pytest
import torch

import mhc_ascend_amd as mhc
from mhc_ascend_amd import ops
from oracle import reference as R
from oracle import rows8
from tests.conftest import assert_close
from tests.test_gpu_dynamic import PARAMS, _check_dyn
from tests.test_gpu_graph import _capture, _replays
from tests.test_gpu_static import _check_static, _oracle_static

pytestmark = pytest.mark.gpu

FORMATS = ["int8", "e4m3"]
DTYPES = [torch.float32, torch.bfloat16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step of one rounding


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(shape, dtype, seed):
    """Rows with a wide range of block maxima, zero blocks and outliers."""
    g = _gen(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-30, 20, (*shape[:-1], 1), generator=g).float())
    x[torch.rand(*shape, generator=g) < 0.01] *= 100
    if x.numel():
        x.view(-1, shape[-1])[::7, :40] = 0
    return x.to(dtype)


def _at(t, device, shift):
    buf = torch.empty(t.numel() + 8, dtype=t.dtype, device=device)
    v = buf[shift:shift + t.numel()].view(t.shape)
    v.copy_(t)
    return v


# ---------------------------------------------------------------------------
# The format
# ---------------------------------------------------------------------------

def _check_packed(x, packed, fmt):
    C = x.shape[-1]
    values, scales = packed.values.cpu(), packed.scales.cpu()
    assert values.shape == (*x.shape[:-1], (C + 15) // 16 * 16) and scales.shape == (*x.shape[:-1], (C + 31) // 32)
    want = (rows8.exponents(x, fmt) + 127).to(torch.uint8)
    assert torch.equal(scales, want)
    held = values.view(torch.int8) if fmt == "int8" else values.view(torch.float8_e4m3fn)
    q = rows8.quantised(x, fmt).flatten(-2)[..., :values.shape[-1]]
    assert torch.equal(held.double(), q), "held numbers"
    for dt in DTYPES:
        assert torch.equal(torch.nan_to_num(mhc.activation_unpack(packed, dt).cpu().double(), nan=12345.0),
                           torch.nan_to_num(rows8.held(x, fmt), nan=12345.0))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,shift", [((5, 1), 0), ((3, 7), 1), ((9, 31), 0), ((9, 32), 1), ((1030, 33), 0), ((4, 72), 0),
                                         ((2, 3, 1001), 3), ((130, 4096), 0), ((3, 96), 0), ((1, 16400), 0), ((0, 64), 0),
                                         ((0, 65), 0), ((64,), 0)])
def test_format(device, fmt, dtype, shape, shift):
    x = _rows(shape, dtype, sum(shape) + shift)
    packed = mhc.activation_pack(_at(x, device, shift), fmt)
    assert packed.format == fmt and packed.hidden == shape[-1] and packed.dtype == dtype
    _check_packed(x, packed, fmt)
    out = mhc.activation_unpack(packed)
    assert out.dtype == dtype and out.shape == x.shape


@pytest.mark.parametrize("fmt", FORMATS)
def test_format_edges(device, fmt):
    """Block maxima at and next to every border of the scale, halves between
    steps, the smallest and largest numbers of fp32."""
    top = rows8.MAX[fmt]
    rows = []
    for e in (-140, -101, -100, -99, -1, 0, 7, 119):
        for a in (top, top * (1 + 2.0 ** -20), top * (1 - 2.0 ** -20), top + 0.5, top * 1.03, top / 2, top / 2 + 0.25):
            m = a * 2.0 ** e
            steps = torch.arange(31, dtype=torch.float64)
            vals = (steps / 2 + 0.5) if fmt == "int8" else (steps / 32 + 1) * 2.0 ** (steps % 17 - 9)
            rows.append(torch.cat([torch.tensor([m], dtype=torch.float64), vals * 2.0 ** e]))
    x = torch.stack(rows)
    x = torch.cat([x, -x]).float()
    x = torch.cat([x, torch.full((1, 32), 3.4028234663852886e38), torch.full((1, 32), 1e-45), torch.zeros(1, 32),
                   -torch.zeros(1, 32)])
    assert x.isfinite().all()
    _check_packed(x, mhc.activation_pack(x.to(device), fmt), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_that_are_not_finite_come_back_as_nan(device, fmt, dtype):
    x = torch.randn(6, 70, generator=_gen(3)).to(dtype)
    x[0, 3] = float("nan")
    x[1, 40] = float("inf")
    x[2, 69] = -float("inf")
    packed = mhc.activation_pack(x.to(device), fmt)
    _check_packed(x, packed, fmt)
    bad = mhc.activation_unpack(packed).cpu().isnan()
    assert bool(bad[0, :32].all()) and bool(bad[1, 32:64].all()) and bool(bad[2, 64:].all())
    assert int(bad.sum()) == 32 + 32 + 6


def test_strided_and_half_inputs(device):
    x = torch.randn(64, 40, generator=_gen(4))
    assert torch.equal(mhc.activation_unpack(mhc.activation_pack(x.to(device).t())).cpu().double(),
                       rows8.held(x.t(), "int8"))
    h = x.half()
    packed = mhc.activation_pack(h.to(device), "e4m3")
    assert packed.dtype == torch.float32
    assert torch.equal(mhc.activation_unpack(packed).cpu().double(), rows8.held(h, "e4m3"))


def test_unpack_refuses_what_does_not_match(device):
    p = mhc.activation_pack(torch.randn(4, 64, device=device))
    for bad in (p._replace(hidden=65), p._replace(scales=p.scales[:3]), p._replace(values=p.values.float())):
        with pytest.raises(RuntimeError, match="checkpoint_unpack"):
            mhc.activation_unpack(bad)
    with pytest.raises(RuntimeError, match="unsupported storage dtype"):
        mhc.activation_unpack(p, torch.float16)
    with pytest.raises(RuntimeError, match="floating"):
        mhc.activation_pack(torch.zeros(4, 64, device=device, dtype=torch.int32))


# ---------------------------------------------------------------------------
# RMSNorm
# ---------------------------------------------------------------------------

def _norm_oracle(x, xh, w, g, eps=1e-5):
    """Output at x; gradients at xh with the magnitudes of their terms."""
    x, w, g = x.double(), w.double(), g.double()
    out = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w
    C = x.shape[-1]
    r = torch.sqrt(xh.square().mean(-1, keepdim=True) + eps)
    dot = (g * w * xh).sum(-1, keepdim=True)
    dx = w * g / r - xh * dot / (C * r ** 3)
    mag = (w * g / r).abs() + xh.abs() * (g * w * xh).abs().sum(-1, keepdim=True) / (C * r ** 3)
    return out, dx, mag, (g * xh / r).sum(0), (g * xh / r).abs().sum(0)


def _within(got, want, bound, what):
    err = (got.detach().cpu().double() - want).abs()
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound"


# Rows are summed by at most 32 values a lane and 10 steps across lanes, and
# every product of sums takes a few roundings more: 64 of 2^-24 on each term
# covers them (the root halves the error of the mean).  A weight's gradient
# adds its rows one by one within a workgroup, then 8 + 128 partials.
K_ROW, K_DW = 64, 400


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C,shift", [(1, 1, 0), (3, 5, 1), (5, 8, 0), (70, 64, 0), (33, 100, 1), (2999, 1001, 0),
                                       (40, 2047, 0), (9, 2048, 0), (600, 4096, 0), (3, 7168, 0), (5, 8200, 0),
                                       (2, 16384, 0), (2, 16379, 2)])
def test_rmsnorm(device, fmt, dtype, B, C, shift):
    x = torch.randn(B, C, generator=_gen(B + C)).to(dtype)
    w = 1 + 0.1 * torch.randn(C, generator=_gen(C))
    g = torch.randn(B, C, generator=_gen(B)).to(dtype)
    xd = _at(x, device, shift).requires_grad_(True)
    wd = _at(w, device, shift).requires_grad_(True)
    out = mhc.rmsnorm(xd, wd, checkpoint=fmt)
    gx, gw = torch.autograd.grad(out, [xd, wd], _at(g, device, shift))
    assert out.dtype == gx.dtype == dtype and gw.dtype == torch.float32
    o, dx, mag, dw, dwmag = _norm_oracle(x, rows8.held(x, fmt), w, g)
    u = U[dtype] if dtype == torch.bfloat16 else 0.0
    _within(out, o, K_ROW * 2.0 ** -24 * o.abs() + u * o.abs() + 1e-30, "out")
    _within(gx, dx, K_ROW * 2.0 ** -24 * mag + u * dx.abs() + 1e-30, "dx")
    _within(gw, dw, K_DW * 2.0 ** -24 * dwmag + 1e-30, "dw")


# Several rows a wave up to 512 values: a lane adds at most 70001 / (4 * 8 * 512)
# + 1 rows of a weight's gradient, then 6 groups, 8 waves and the partials as above.
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C,shift", [(70001, 104, 0), (35003, 100, 1), (35000, 33, 0), (20001, 7, 0), (4097, 256, 0),
                                       (1030, 505, 1), (5, 512, 0), (9, 520, 0), (33, 517, 1), (17, 9, 3)])
def test_rmsnorm_narrow_rows(device, fmt, dtype, B, C, shift):
    test_rmsnorm(device, fmt, dtype, B, C, shift)


def test_rmsnorm_empty_and_refused_rows(device):
    x = torch.empty(0, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    gx, gw = torch.autograd.grad(mhc.rmsnorm(x, w, checkpoint="int8").sum(), [x, w])
    assert gx.shape == (0, 64) and bool((gw == 0).all())
    with pytest.raises(RuntimeError, match="too large"):
        mhc.rmsnorm(torch.randn(2, 16392, device=device, requires_grad=True), torch.ones(16392, device=device),
                    checkpoint="int8")


def test_gradient_against_differences(device):
    """Directional derivatives of the operator itself, at rows that are their
    own checkpoint.  L = sum(cot * out) in 64 bits over fp32 outputs: central
    differences at step h are off by h^2 / 6 times the third derivative (below
    60 times the first for rows of unit size, h = 2^-6: 2.5e-3) and by the
    outputs' rounding, 64 * 2^-24 * sum|cot out| / h."""
    g = _gen(8)
    x = mhc.activation_unpack(mhc.activation_pack(torch.randn(64, 256, generator=g).to(device)))
    w = (1 + 0.1 * torch.randn(256, generator=g)).to(device)
    cot = torch.randn(64, 256, generator=g).to(device)
    xd, wd = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    grads = torch.autograd.grad(mhc.rmsnorm(xd, wd, checkpoint="int8"), [xd, wd], cot)

    def loss(a, b):
        return float((mhc.rmsnorm(a, b).double() * cot.double()).sum())

    h = 2.0 ** -6
    noise = 64 * 2.0 ** -24 * float((mhc.rmsnorm(x, w).double() * cot.double()).abs().sum()) / h
    for i, t in enumerate((x, w)):
        d = torch.randn(t.shape, generator=g).to(device)
        step = [d * h if i == k else 0 for k in range(2)]
        diff = (loss(x + step[0], w + step[1]) - loss(x - step[0], w - step[1])) / (2 * h)
        want = float((grads[i].double() * d.double()).sum())
        scale = float((grads[i].double() * d.double()).abs().sum())
        assert abs(diff - want) <= 2.5e-3 * scale + noise, (i, diff, want)


# ---------------------------------------------------------------------------
# Layers: forward at x, gradients at x^
# ---------------------------------------------------------------------------

LAYER_SHAPES = [(4, 7, 64), (4, 33, 256), (4, 600, 128), (4, 5, 4096), (4, 9, 1001), (4, 3, 7168), (2, 37, 1280),
                (8, 12, 1280), (3, 9, 77), (3, 17, 1040), (6, 17, 256), (5, 4, 320), (1, 7, 100), (12, 5, 130),
                (16, 5, 64)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("n,B,C", LAYER_SHAPES)
def test_static_layer(device, fmt, x_dtype, n, B, C):
    d = R.static_layer_inputs(B, n, C, seed=n * 1000 + B + C, x_dtype=x_dtype)
    x = d["x"].to(device).requires_grad_(True)
    ps = [d[k].to(device).requires_grad_(True) for k in ("weight", "H_pre", "H_post", "H_res")]
    out = mhc.mhc_layer_static(x, *ps, checkpoint=fmt)
    gx, *gp = torch.autograd.grad(out, [x, *ps], d["grad"].to(device))
    want_out = _oracle_static(d)[0]
    _, rgx, rgp = _oracle_static(dict(d, x=rows8.held(d["x"], fmt)))
    _check_static(d, (out, gx, gp), (want_out, rgx, rgp), x_dtype == torch.bfloat16, f"n={n} B={B} C={C}",
                  family_floor=n == 1)


def _oracle_dyn_held(d, fmt, iters=20, eps=1e-5):
    """Output at x; gradients with the streams at x^ and the products with the
    projections and mean squares at their values of x."""
    x, xh = d["x"].double(), rows8.held(d["x"], fmt).requires_grad_(True)
    B, n, C = x.shape
    ps = [d[k].double().requires_grad_(True) for k in PARAMS]
    w, pp, pq, pr, ap, aq, ar, bp, bq, br = ps
    out = R.mhc_layer_dynamic(x, *[p.detach() for p in ps], iters, 1e-8, eps, dtype=torch.float64)
    phi = torch.cat([pp, pq, pr.reshape(n * n, n * C)])
    flat, hflat = x.reshape(B, -1), xh.reshape(B, -1)
    prod, ms = hflat @ phi.t(), hflat.square().mean(-1, keepdim=True)
    prod = prod + (flat @ phi.t() - prod).detach()
    ms = ms + (flat.square().mean(-1, keepdim=True) - ms).detach()
    t = prod / torch.sqrt(ms + eps)
    m = R.sinkhorn_knopp(torch.exp((ar * t[:, 2 * n:] + br.reshape(-1)).reshape(B, n, n)), iters, 1e-8)
    y = R._layer_core(xh, w, torch.sigmoid(ap * t[:, :n] + bp), 2 * torch.sigmoid(aq * t[:, n:2 * n] + bq), m, eps)
    y.backward(d["grad"].double())
    return out, xh.grad, [p.grad for p in ps]


DYN_SHAPES = [(4, 9, 64), (4, 33, 256), (4, 600, 128), (4, 5, 4096), (4, 40, 1024), (2, 37, 256), (8, 12, 1280),
              (3, 9, 160), (6, 17, 1040), (1, 7, 96), (12, 5, 128), (16, 5, 64), (10, 70, 80), (8, 4, 7168), (6, 3, 100 * 16),
              (8, 300, 100), (20, 3, 32), (4, 1090, 136)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("n,B,C", DYN_SHAPES)
def test_dynamic_layer(device, fmt, x_dtype, n, B, C):
    d = R.dynamic_layer_inputs(B, n, C, seed=n * 37 + B + C, x_dtype=x_dtype, alpha=0.2, phi_std=0.03, b_std=0.5)
    x = d["x"].to(device).requires_grad_(True)
    ps = [d[k].to(device).requires_grad_(True) for k in PARAMS]
    out = mhc.mhc_layer_fused_dynamic_training(x, *ps, checkpoint=fmt)
    gx, *gp = torch.autograd.grad(out, [x, *ps], d["grad"].to(device))
    _check_dyn((out, gx, gp), _oracle_dyn_held(d, fmt), x_dtype, f"n={n} B={B} C={C}", family_floor=n == 1)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dynamic,n,C,mode", [(True, 4, 256, "decay"), (True, 8, 64, "zero"), (False, 4, 96, "decay"),
                                              (False, 3, 70, "decay"), (True, 6, 128, "zero")])
def test_wrapper_reads_its_rows_from_the_checkpoint(device, fmt, dynamic, n, C, mode):
    """Forward: that of the wrapper without a checkpoint, bit for bit.
    Backward: with static H the wrapper's at the rows' x^, bit for bit; with
    dynamic H `saved` is the forward's own, so the entry itself is called with
    it on x^."""
    torch.manual_seed(n + C)
    wrap = mhc.MHCResidualWrapper(C, n, residual_mode=mode, use_dynamic_h=dynamic, alpha_init=0.2).to(device)
    rows = [torch.randn(37, C, generator=_gen(k)).to(torch.bfloat16) for k in range(2)]
    cot = torch.randn(37, C, generator=_gen(5)).to(device)
    params = list(wrap.parameters())

    def step(vals):
        leaves = [v.to(device).requires_grad_(True) for v in vals]
        out = wrap(*leaves)
        return out.detach(), torch.autograd.grad(out, leaves + params, cot)

    want_out, _ = step(rows)
    hats = [rows8.held(r, fmt).to(torch.bfloat16) for r in rows]
    wrap.mhc.checkpoint = fmt
    out, grads = step(rows)
    assert torch.equal(out, want_out)
    if not (n == 3 or dynamic):
        wrap.mhc.checkpoint = None
        _, want = step(hats)
        for a, e in zip(grads, want):
            assert torch.equal(a, e)
    elif dynamic:
        m = wrap.mhc
        p = [m.phi_pre, m.phi_post, m.phi_res, m.alpha_pre, m.alpha_post, m.alpha_res]
        _, saved = ops.native.wrapper_dynamic_fwd(*[r.to(device) for r in rows], mode, n, m.rmsnorm_weight, *p, m.b_pre,
                                                  m.b_post, m.b_res)
        want = ops.native.wrapper_dynamic_bwd(cot, *[h.to(device) for h in hats], mode, n, m.rmsnorm_weight, saved, *p,
                                              m.b_res)
        named = dict(zip(["residual", "branch", "rmsnorm_weight", "phi_pre", "phi_post", "phi_res", "alpha_pre",
                          "alpha_post", "alpha_res", "b_pre", "b_post", "b_res"], want))
        order = ["residual", "branch"] + [k for k, _ in m.named_parameters()]
        for k, a in zip(order, grads):
            assert torch.equal(a.flatten(), named[k].flatten()), k


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_stream_operators_read_their_rows_from_the_checkpoint(device, fmt, dtype):
    """The same gradients, bit for bit, as the operators at x^."""
    g = _gen(9)
    B, n, C = 21, 4, 200
    x, y = torch.randn(B, n, C, generator=g).to(dtype), torch.randn(B, C, generator=g).to(dtype)
    h, m = torch.randn(B, n, generator=g), torch.rand(B, n, n, generator=g)
    ca, co = torch.randn(B, C, generator=g).to(dtype).to(device), torch.randn(B, n, C, generator=g).to(device)

    def run(call, vals, cot, **kw):
        leaves = [v.to(device).requires_grad_(True) for v in vals]
        out = call(*leaves, **kw)
        return out.detach(), torch.autograd.grad(out, leaves, cot)

    hat = lambda t: rows8.held(t, fmt).to(dtype)
    out, got = run(mhc.stream_aggregate, [x, h], ca, checkpoint=fmt)
    assert torch.equal(out, run(mhc.stream_aggregate, [x, h], ca)[0])
    assert all(torch.equal(a, b) for a, b in zip(got, run(mhc.stream_aggregate, [hat(x), h], ca)[1]))
    out, got = run(mhc.stream_distribute_mix_add, [y, h, m, x], co, checkpoint=fmt)
    assert torch.equal(out, run(mhc.stream_distribute_mix_add, [y, h, m, x], co)[0])
    want = run(mhc.stream_distribute_mix_add, [hat(y), h, m, hat(x)], co)[1]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# Behaviour around the operators
# ---------------------------------------------------------------------------

def _step(device, dynamic, x, cot, layer):
    x = x.to(device).requires_grad_(True)
    out = layer(x)
    return [out.detach(), *torch.autograd.grad(out, [x, *layer.parameters()], cot.to(device))]


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("n,C", [(4, 256), (6, 96)])
def test_nan_rows_reach_the_gradient(device, dynamic, n, C):
    """A row that is not finite is not hidden by its checkpoint."""
    layer = mhc.MHCLayer(C, n, use_dynamic_h=dynamic, checkpoint="int8").to(device)
    x = torch.randn(20, n, C, generator=_gen(1))
    x[7, 1, 40] = float("nan")
    out, gx, *gp = _step(device, dynamic, x, torch.randn(20, n, C, generator=_gen(2)), layer)
    assert bool(gx[7].isnan().any()) and bool(gx[:7].isfinite().all()) and bool(gx[8:].isfinite().all())
    assert bool(gp[0].float().isnan().any())


@pytest.mark.parametrize("dynamic", [False, True])
def test_empty_batch(device, dynamic):
    layer = mhc.MHCLayer(64, 4, use_dynamic_h=dynamic, checkpoint="e4m3").to(device)
    out, gx, *gp = _step(device, dynamic, torch.empty(0, 4, 64), torch.empty(0, 4, 64), layer)
    assert out.shape == gx.shape == (0, 4, 64) and all(bool((g == 0).all()) for g in gp)


@pytest.mark.parametrize("dynamic", [False, True])
def test_strided_input_and_cotangent(device, dynamic):
    layer = mhc.MHCLayer(64, 4, use_dynamic_h=dynamic, checkpoint="int8").to(device)
    x, cot = torch.randn(9, 4, 64, generator=_gen(3)), torch.randn(9, 4, 64, generator=_gen(4))
    want = _step(device, dynamic, x, cot, layer)
    xs = torch.randn(9, 64, 4, device=device).transpose(1, 2)
    xs.copy_(x)
    cs = torch.randn(9, 64, 4, device=device).transpose(1, 2)
    cs.copy_(cot)
    xs.requires_grad_(True)
    out = layer(xs)
    got = [out.detach(), *torch.autograd.grad(out, [xs, *layer.parameters()], cs)]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_memory_between_forward_and_backward(device):
    """What the pass keeps is the checkpoint: 33/32 bytes a value, not x."""
    T, n, C = 2048, 4, 1024
    layer = mhc.MHCLayer(C, n, use_dynamic_h=False, checkpoint="int8").to(device)
    sizes = {}
    for fmt in (None, "int8"):
        layer.checkpoint = fmt
        gc.collect()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        x = torch.randn(T, n, C, device=device, requires_grad=True)
        out = layer(x * 1.0)  # an activation nobody else holds
        loss = out.sum()
        del out, x
        torch.cuda.synchronize()
        sizes[fmt] = torch.cuda.memory_allocated() - before
        del loss
    E = T * n * C
    # x itself stays with its leaf's gradient edge in neither; the difference is
    # 4 bytes a value against 33/32
    assert abs((sizes[None] - sizes["int8"]) - (4 * E - E * 33 // 32)) <= 1 << 16


def test_no_checkpoint_without_a_backward(device):
    """Nothing is packed where no gradient is wanted: the same result, and a
    width past the packed rows' limit is taken."""
    x = torch.randn(3, 16392, device=device)
    w = torch.ones(16392, device=device)
    assert torch.equal(mhc.rmsnorm(x, w, checkpoint="int8"), mhc.rmsnorm(x, w))
    with torch.no_grad():
        xr = x.clone().requires_grad_(True)
        assert torch.equal(mhc.rmsnorm(xr, w, checkpoint="int8"), mhc.rmsnorm(x, w))


def test_trace_is_refused(device):
    x = torch.randn(4, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device)
    cos, sin = (t.to(device) for t in mhc.rope_table(4, 64))
    h = torch.randn(4, 1, 64, device=device)
    for call in (lambda a: mhc.rmsnorm(a, w, checkpoint="int8"), lambda a: mhc.activation_pack(a).values,
                 lambda a: mhc.qk_norm_rope(a.view(4, 1, 64), h, w, w, cos, sin)):
        with pytest.raises(RuntimeError, match="not recorded by torch.jit.trace"):
            torch.jit.trace(call, (x,), check_trace=False)


@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("n,C,x_dtype", [(4, 256, torch.bfloat16), (4, 256, torch.float32), (6, 96, torch.bfloat16),
                                         (3, 160, torch.float32)])
def test_unaligned_rows(device, dynamic, n, C, x_dtype):
    """x and the cotangent one element past an aligned address: the kernels
    that take any alignment, against the aligned call."""
    layer = mhc.MHCLayer(C, n, use_dynamic_h=dynamic, alpha_init=0.2, checkpoint="int8").to(device)
    x, cot = torch.randn(40, n, C, generator=_gen(1)).to(x_dtype), torch.randn(40, n, C, generator=_gen(2))
    want = _step(device, dynamic, x, cot, layer)
    for sx, sg in ((1, 0), (0, 1), (1, 1)):
        xs = _at(x, device, sx).requires_grad_(True)
        out = layer(xs)
        got = [out.detach(), *torch.autograd.grad(out, [xs, *layer.parameters()], _at(cot, device, sg))]
        for a, e in zip(got, want):
            # the same sums in another order, rounded once to the type
            u = U[a.dtype] if a.dtype == torch.bfloat16 else 0.0
            assert_close(a, e, 2 * u + 1e-4, 2e-5 * float(e.abs().max()) + u * float(e.abs().max()) / 8)


@pytest.mark.parametrize("dynamic", [False, True])
def test_backward_twice_and_inputs_changed_after_the_forward(device, dynamic):
    """The checkpoint is the node's own: changing x afterwards does not reach
    the gradient, and a second backward gives the first one's bits."""
    layer = mhc.MHCLayer(256, 4, use_dynamic_h=dynamic, checkpoint="int8").to(device)
    x, cot = torch.randn(40, 4, 256, generator=_gen(1)), torch.randn(40, 4, 256, generator=_gen(2))
    want = _step(device, dynamic, x, cot, layer)
    leaf = x.to(device).requires_grad_(True)
    rows = leaf * 1.0
    out = layer(rows)
    rows.detach().zero_()
    for _ in range(2):
        got = torch.autograd.grad(out, [leaf, *layer.parameters()], cot.to(device), retain_graph=True)
        assert all(torch.equal(a, e) for a, e in zip(got, want[1:]))


def _tail(t, k):
    return t[-k:].clone()


def test_offsets_past_32_bits(device):
    """More than 2^32 values: the last rows against a call on them alone."""
    C = 4096
    B = (1 << 32) // C + 520
    x = torch.empty(B, C, dtype=torch.bfloat16, device=device)
    x.fill_(0.5)
    x[-512:] = torch.randn(512, C, device=device).bfloat16()
    p = mhc.activation_pack(x, "e4m3")
    assert torch.equal(mhc.activation_unpack(p)[-512:], mhc.activation_unpack(mhc.activation_pack(_tail(x, 512), "e4m3")))
    ragged = x.view(-1)[:(B * C) // 4095 * 4095].view(-1, 4095)
    q = mhc.activation_pack(ragged, "int8")
    want = mhc.activation_pack(_tail(ragged, 300), "int8")
    assert torch.equal(q.values[-300:], want.values) and torch.equal(q.scales[-300:], want.scales)
    assert torch.equal(mhc.activation_unpack(q)[-300:], mhc.activation_unpack(want))
    del p, q, ragged
    w = torch.rand(C, device=device) + 0.5
    outs = []
    for rows in (x, _tail(x, 512)):
        r = rows.detach().requires_grad_(True)
        out = mhc.rmsnorm(r, w, checkpoint="int8")
        gx, = torch.autograd.grad(out, r, rows)
        outs.append((_tail(out.detach(), 512), _tail(gx, 512)))
        del out, gx, r
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("n,C,w_dtype", [(2, 64, torch.float32), (4, 128, torch.bfloat16), (7, 96, torch.float32),
                                         (8, 1280, torch.bfloat16)])
def test_static_layer_in_one_launch_or_two(device, n, C, w_dtype):
    """Few tokens take the coefficients and the rows in one forward launch, many
    in two: the same bits for the same tokens."""
    few, many = 33, 9 * torch.cuda.get_device_properties(device).multi_processor_count
    g = _gen(n)
    x = torch.randn(many, n, C, generator=g).to(device)
    cot = torch.randn(many, n, C, generator=g).to(device)
    params = [torch.randn(C, generator=g).to(device, w_dtype), torch.randn(n, generator=g).to(device),
              torch.randn(n, generator=g).to(device), torch.randn(n, n, generator=g).to(device)]
    outs = []
    for t in (few, many):
        r = x[:t].clone().requires_grad_(True)
        out = mhc.mhc_layer_static(r, *params, checkpoint="int8")
        outs.append((out.detach()[:few], torch.autograd.grad(out, r, cot[:t])[0][:few]))
    # dx sums a row over other lanes where the two batches tile it differently: a
    # value has n products and a term of two row sums, 64 of 2^-24 on each
    assert torch.equal(outs[0][0], outs[1][0])
    scale = float(outs[0][1].abs().max())
    assert float((outs[0][1] - outs[1][1]).abs().max()) <= 64 * 2.0 ** -24 * n * scale


def test_one_row_of_nearly_two_to_the_31(device):
    """The padded row is 2^31 bytes: its last blocks against a short row's."""
    C, tail = (1 << 31) - 1, 32 * 64 - 1
    x = torch.zeros(1, C, dtype=torch.bfloat16, device=device)
    x[:, -tail:] = torch.randn(1, tail, device=device).bfloat16()
    p = mhc.activation_pack(x, "int8")
    want = mhc.activation_pack(x[:, -tail:], "int8")
    assert torch.equal(p.values[:, -want.values.shape[1]:], want.values)
    assert torch.equal(p.scales[:, -want.scales.shape[1]:], want.scales)
    assert not p.values[:, :1024].any() and not p.values[:, C // 2: C // 2 + 1024].any()
    del x
    back = mhc.activation_unpack(p)
    assert torch.equal(back[:, -tail:], mhc.activation_unpack(want)) and not back[:, :1024].any()


@pytest.mark.parametrize("dynamic", [False, True])
def test_layer_offsets_past_32_bits(device, dynamic):
    n, C = 4, 4096
    B = (1 << 32) // (n * C) + 2060
    layer = mhc.MHCLayer(C, n, use_dynamic_h=dynamic, checkpoint="int8").to(device)
    x = torch.empty(B, n, C, dtype=torch.bfloat16, device=device).fill_(0.5)
    x[-2048:] = torch.randn(2048, n, C, device=device).bfloat16()
    cot = torch.zeros(B, n, C, device=device)
    cot[-2048:] = torch.randn(2048, n, C, device=device)
    outs = []
    for rows, g in ((x, cot), (_tail(x, 2048), _tail(cot, 2048))):
        r = rows.detach().requires_grad_(True)
        out = layer(r)
        gx, = torch.autograd.grad(out, r, g)
        outs.append((_tail(out.detach(), 2048), _tail(gx, 2048)))
        del out, gx, r
    # per token; the projection's splits of its sums differ with the batch, and
    # a dx near a border of bf16 may round the other way: one step, 2^-7
    for a, b in zip(*outs):
        scale = float(b.abs().max())
        assert float((a.float() - b.float()).abs().max()) <= (2.0 ** -7 if a.dtype == torch.bfloat16 else 1e-5) * scale


@pytest.mark.parametrize("dynamic", [False, True])
def test_two_runs_and_another_stream_agree(device, dynamic):
    """Fixed-order sums: every run gives the same bits, on any stream, with
    two backward passes in flight at once."""
    layer = mhc.MHCLayer(256, 4, use_dynamic_h=dynamic, checkpoint="e4m3").to(device)
    x, cot = torch.randn(300, 4, 256, generator=_gen(5)), torch.randn(300, 4, 256, generator=_gen(6))
    want = _step(device, dynamic, x, cot, layer)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_step(device, dynamic, x, cot, layer))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("dynamic", [False, True])
def test_step_replays_in_a_graph(device, dynamic):
    """Forward and backward with a checkpoint, captured once."""
    layer = mhc.MHCLayer(256, 4, use_dynamic_h=dynamic, checkpoint="int8").to(device)
    x = torch.randn(48, 4, 256, device=device)
    cot = torch.randn(48, 4, 256, device=device)
    rows = torch.randn(48, 256, device=device)
    w = torch.ones(256, device=device)
    names = PARAMS if dynamic else ["weight", "H_pre", "H_post", "H_res"]
    params = [getattr(layer, "rmsnorm_weight" if k == "weight" else k) for k in names]

    def step():
        # leaves of this call only: none of them lives outside the graph
        xl = x.detach().requires_grad_(True)
        ps = [p.detach().requires_grad_(True) for p in params]
        if dynamic:
            out = mhc.mhc_layer_fused_dynamic_training(xl, *ps, checkpoint="int8")
        else:
            out = mhc.mhc_layer_static(xl, *ps, checkpoint="int8")
        rl, wl = rows.detach().requires_grad_(True), w.detach().requires_grad_(True)
        o2 = mhc.rmsnorm(rl, wl, checkpoint="e4m3")
        grads = torch.autograd.grad([out, o2], [xl, *ps, rl, wl], [cot, rows])
        return [out.detach(), o2.detach(), *grads]

    graph, outs = _capture(step)
    g = _gen(7)
    feeds = [lambda: x.copy_(torch.randn(x.shape, generator=g)), lambda: cot.copy_(torch.randn(x.shape, generator=g)),
             lambda: rows.copy_(torch.randn(rows.shape, generator=g))]
    _replays(graph, outs, step, feeds)


# x^ is exact in bf16 and dP and Phi are not: with 16 bits of each left in their
# products, the part of dx that comes through the projections is 4.3e-6 off in
# the 2-norm.  Roundings of fp32 that are independent add in the 2-norm: 16 *
# 2^-24 allows a chain of 256 of them (fp32 autograd of these inputs, 2-4e-7).
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,B,C", [(4, 40, 1024), (4, 300, 96), (2, 64, 2048), (3, 50, 160), (6, 30, 1040), (8, 24, 512),
                                   (12, 20, 224), (16, 40, 64)])
def test_dx_of_fp32_rows_is_in_fp32(device, fmt, n, B, C):
    """Nearly all of dx is sum_o dP_o Phi_o here: the cotangent is x itself."""
    d = R.dynamic_layer_inputs(B, n, C, seed=n + B, x_dtype=torch.float32, alpha=1.0, phi_std=(n * C) ** -0.5,
                               b_std=0.5)
    d["grad"] = d["x"].clone()
    x = d["x"].to(device).requires_grad_(True)
    ps = [d[k].to(device).requires_grad_(True) for k in PARAMS]
    out = mhc.mhc_layer_fused_dynamic_training(x, *ps, checkpoint=fmt)
    gx, = torch.autograd.grad(out, [x], d["grad"].to(device))
    want = _oracle_dyn_held(d, fmt)[1]
    assert float((gx.cpu().double() - want).norm() / want.norm()) <= 16 * 2.0 ** -24
