"""Dropout without a stored mask and the RMSNorm of a residual's sum, against
the 64-bit oracle.  What is kept is compared for equality with the generator's
definition; tolerances count roundings and are derived next to them."""
import pytest
import torch

import mhc_ascend_amd as mhc
from oracle import branch as B
from oracle import rows8
from tests.test_gpu_checkpoint import _at, _within
from tests.test_gpu_graph import _capture, _replays

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8}  # half a step of one rounding
E32 = 2.0 ** -24
# A row's sums: at most 64 values a lane one after the other (40000 channels over
# 1024 lanes), 6 steps across lanes, 16 waves, so 86 roundings of the terms, half
# of that in 1 / r, which takes 3 more; a value takes 5 products and sums.  dw:
# rows one by one within a workgroup and lane, 8 waves, 32 phases of partials.
K_ROW, K_DW = 100, 600
SEED = 0x9E3779B97F4A7C15  # above 2^63


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(shape, dtype, seed):
    g = _gen(seed)
    x = torch.randn(*shape, generator=g)
    x[torch.rand(*shape, generator=g) < 0.01] *= 20
    return x.to(dtype)


# ---------------------------------------------------------------------------
# Dropout
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,shift", [((1, 1), 0), ((3, 7), 0), ((5, 8), 1), ((129, 33), 3), ((4, 72), 0),
                                         ((2, 3, 1001), 1), ((1030, 4096), 0), ((64,), 0), ((0, 24), 0), ((0, 7), 0),
                                         ((1, 16400), 0)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout_keeps_what_the_numbers_say(device, dtype, shape, shift, p):
    x, g = _rows(shape, dtype, 1), _rows(shape, dtype, 2)
    xd = _at(x, device, shift).requires_grad_(True)
    y = mhc.dropout(xd, p, seed=SEED, offset=5)
    dx, = torch.autograd.grad(y, xd, _at(g, device, shift))
    f = B.factors(shape, p, SEED, 5)
    for got, v in ((y, x), (dx, g)):
        assert got.dtype == dtype and got.shape == x.shape
        want = v.double() * f
        assert torch.equal(got.detach().cpu() != 0, (f != 0) & (v != 0))
        # the scale rounded to fp32, the product, the storage type
        _within(got, want, (2 * E32 + (U[dtype] if dtype == BF16 else 0.0)) * want.abs() * (1 + 2.0 ** -7), "dropout")


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 1.0 - 2.0 ** -18, 1.0])
def test_dropout_at_the_ends(device, p):
    """p under 2^-17 stands for 0, and within 2^-17 of 1 for 1: nothing, or everything."""
    x = _rows((9, 40), F32, 3)
    y = mhc.dropout(x.to(device), p, seed=1).cpu()
    assert torch.equal(y, x if p < 0.5 else torch.zeros_like(x))


def test_dropped_values_are_zero_whatever_they_were(device):
    x = torch.full((64, 100), float("inf"))
    x[::2] = float("nan")
    y = mhc.dropout(x.to(device), 0.5, seed=7).cpu()
    f = B.factors(x.shape, 0.5, 7)
    assert bool((y[f == 0] == 0).all()) and not bool(y[f != 0].isfinite().any())


def test_dropout_numbers_do_not_depend_on_type_or_layout(device):
    x = torch.ones(12, 6, 72, device=device)
    want = mhc.dropout(x, 0.3, seed=11, offset=2)
    assert torch.equal(mhc.dropout(x.bfloat16(), 0.3, seed=11, offset=2) != 0, want != 0)
    assert torch.equal(mhc.dropout(x.half(), 0.3, seed=11, offset=2), want)  # others become fp32
    assert torch.equal(mhc.dropout(x.double(), 0.3, seed=11, offset=2), want)
    assert torch.equal(mhc.dropout(x.view(72, 72), 0.3, seed=11, offset=2), want.view(72, 72))
    strided = torch.ones(72, 6, 12, device=device).permute(2, 1, 0)
    assert torch.equal(mhc.dropout(strided, 0.3, seed=11, offset=2), want)
    assert torch.equal(mhc.dropout(x[:1].expand(12, 6, 72), 0.3, seed=11, offset=2), want)


def test_seeds_and_offsets(device):
    x = torch.ones(64, 128, device=device)
    t = lambda v: torch.tensor([v], device=device)  # noqa: E731
    base = mhc.dropout(x, 0.5, seed=3, offset=1)
    assert torch.equal(mhc.dropout(x, 0.5, seed=t(3), offset=1), base)
    assert torch.equal(mhc.dropout(x, 0.5, seed=t(3).reshape(()), offset=1), base)
    assert torch.equal(mhc.dropout(x, 0.5, seed=-1), mhc.dropout(x, 0.5, seed=2 ** 64 - 1))
    assert torch.equal(mhc.dropout(x, 0.5, seed=t(-1)), mhc.dropout(x, 0.5, seed=2 ** 64 - 1))
    for other in (mhc.dropout(x, 0.5, seed=4, offset=1), mhc.dropout(x, 0.5, seed=3 + 2 ** 32, offset=1),
                  mhc.dropout(x, 0.5, seed=3, offset=2), mhc.dropout(x, 0.5, seed=3, offset=1 + 2 ** 32)):
        # 8192 independent halves: 4096 differ, sigma 45
        assert abs(int((other != base).sum()) - 4096) < 300
    big = mhc.dropout(x, 0.5, seed=9, offset=2 ** 63 - 1).cpu()
    assert torch.equal(big.double(), B.factors(x.shape, 0.5, 9, 2 ** 63 - 1))


def test_a_seed_that_is_not_given_is_torchs(device):
    x = torch.ones(64, 128, device=device, requires_grad=True)
    torch.manual_seed(5)
    a, b = mhc.dropout(x), mhc.dropout(x)
    torch.manual_seed(5)
    c = mhc.dropout(x)
    assert torch.equal(a, c) and not torch.equal(a, b)
    g, = torch.autograd.grad(c, x, torch.ones_like(x))
    assert torch.equal(g, c.detach())  # the backward drops what the forward did


def test_a_seed_changed_before_the_backward_is_an_error(device):
    x = torch.ones(8, 64, device=device, requires_grad=True)
    seed = torch.tensor([3], device=device)
    for call in (lambda: mhc.dropout(x, 0.5, seed=seed),
                 lambda: mhc.rmsnorm_residual(x, x, torch.ones(64, device=device), dropout=0.5, seed=seed)[0]):
        y = call()
        seed.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_dropout_mean_and_shares(device):
    """A million values: shares of each bit of the numbers and of what is kept."""
    x = torch.ones(1024, 1024, device=device)
    for p in (0.05, 0.25, 0.9):
        kept = float((mhc.dropout(x, p, seed=1) != 0).double().mean())
        assert abs(kept - (1 - round(p * 65536) / 65536)) < 6 * (p * (1 - p)) ** 0.5 / 1024


def test_dropout_rows_past_32_bits(device):
    """More than 2^32 values, and more than 2^31 lanes of rows: the last rows."""
    C, seed = 4096, 12
    rows = (1 << 32) // C + 5
    x = torch.ones(rows, C, dtype=BF16, device=device)
    y = mhc.dropout(x, 0.25, seed=seed)
    f = (B.numbers(7, C, seed, 0, rows - 7) >= 16384)
    assert torch.equal(y[-7:].cpu() != 0, f)
    del x, y
    C = 7
    rows = (1 << 30) + 9
    x = torch.ones(rows, C, dtype=BF16, device=device)
    y = mhc.dropout(x, 0.25, seed=seed)
    for at in (0, (1 << 30) - 3, rows - 7):
        f = (B.numbers(7, C, seed, 0, at) >= 16384)
        assert torch.equal(y[at:at + 7].cpu() != 0, f), at


# ---------------------------------------------------------------------------
# RMSNorm of a residual's sum
# ---------------------------------------------------------------------------

# narrow rows, ragged rows, every number of pieces a lane, rows past the registers
SHAPES = [(1, 1), (1, 8), (3, 7), (5, 33), (9, 64), (130, 100), (67, 512), (33, 513), (17, 1001), (40, 1280),
          (1, 4096), (300, 4096), (11, 5003), (5, 8192), (6, 9001), (3, 16384), (3, 16385), (2, 40000), (0, 64),
          (2100, 96), (2600, 1024), (1100, 4096), (550, 5003), (600, 16383), (70001, 33), (3, 256), (9, 257)]
DTYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)]


def _inputs(shape, dtypes, seed, w_dtype=F32):
    xt, rt = dtypes
    x, res = _rows(shape, xt, seed), _rows(shape, rt, seed + 1)
    w = (1 + 0.2 * torch.randn(shape[-1], generator=_gen(seed + 2))).to(w_dtype)
    return x, res, w, [_rows(shape, xt, seed + 3), _rows(shape, rt, seed + 4)]


def _check(got, inputs, p, fmt, seed, offset, eps=1e-5):
    """y, h, dx, dres, dw of a call.  The norm and the gradients are checked at the
    h that came back."""
    x, res, w, (gy, gh) = inputs
    y, h, dx, dres, dw = [t.detach().cpu() for t in got]
    xt, rt = x.dtype, res.dtype
    assert (y.dtype, h.dtype, dx.dtype, dres.dtype, dw.dtype) == (xt, rt, xt, rt, w.dtype)
    if x.numel() == 0:
        assert y.shape == x.shape and dx.shape == x.shape and bool((dw == 0).all())
        return
    C = x.shape[-1]
    f = B.factors(x.shape, p, seed, offset) if p else torch.ones(x.shape, dtype=torch.float64)
    xd = x.double() * f
    want = res.double() + xd
    # the scale, the product and the sum in fp32, the storage type
    _within(h, want, 2 * E32 * xd.abs() + E32 * want.abs() + (U[BF16] * want.abs() * (1 + 2.0 ** -7) if rt == BF16 else 0)
            + 1e-30, "h")
    hd, wd = h.double(), w.double()
    yd = B.rmsnorm(hd, wd, eps)
    _within(y, yd, (K_ROW * E32 + (U[BF16] if xt == BF16 else 0.0)) * yd.abs() + 1e-30, "y")
    hh = rows8.held(h, fmt)
    r = torch.sqrt(hh.square().mean(-1, keepdim=True) + eps)
    u = gy.double() * wd
    dh = gh.double() + u / r - hh * (u * hh).sum(-1, keepdim=True) / (C * r ** 3)
    mag = gh.double().abs() + (u / r).abs() + hh.abs() * (u * hh).abs().sum(-1, keepdim=True) / (C * r ** 3)
    _within(dres, dh, K_ROW * E32 * mag + (U[BF16] * dh.abs() if rt == BF16 else 0.0) + 1e-30, "dres")
    _within(dx, dh * f, (K_ROW + 2) * E32 * mag * f + (U[BF16] * (dh * f).abs() * (1 + 2.0 ** -7) if xt == BF16 else 0.0)
            + 1e-30, "dx")
    assert bool((dx[f == 0] == 0).all())
    terms = gy.double() * hh / r
    _within(dw, terms.flatten(0, -2).sum(0), K_DW * E32 * terms.abs().flatten(0, -2).sum(0)
            + (U[BF16] * terms.flatten(0, -2).sum(0).abs() if w.dtype == BF16 else 0.0) + 1e-30, "dw")


def _run(device, inputs, p, fmt, seed, offset, shift=0):
    x, res, w, cots = inputs
    leaves = [_at(t, device, shift).requires_grad_(True) for t in (x, res)] + [w.to(device).requires_grad_(True)]
    out = mhc.rmsnorm_residual(*leaves, dropout=p, seed=seed, offset=offset, checkpoint=fmt)
    return [*out, *torch.autograd.grad(out, leaves, [_at(t, device, shift) for t in cots])]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtypes", DTYPES)
@pytest.mark.parametrize("p,fmt", [(0.0, None), (0.1, None), (0.0, "int8"), (0.3, "e4m3")])
def test_matches_oracle(device, shape, dtypes, p, fmt):
    inputs = _inputs(shape, dtypes, sum(shape))
    _check(_run(device, inputs, p, fmt, SEED, 3), inputs, p, fmt, SEED, 3)


@pytest.mark.parametrize("dtypes", DTYPES)
@pytest.mark.parametrize("shape", [(7, 64), (9, 1001), (5, 4096), (2, 16390)])
@pytest.mark.parametrize("shift", [1, 3])
def test_rows_at_any_alignment(device, dtypes, shape, shift):
    inputs = _inputs(shape, dtypes, 5, BF16)
    _check(_run(device, inputs, 0.2, None, 4, 0, shift), inputs, 0.2, None, 4, 0)


def test_leading_dimensions_strides_and_broadcasts(device):
    x, res, w, cots = _inputs((4, 6, 96), (BF16, F32), 6)
    want = _run(device, (x, res, w, cots), 0.2, None, 4, 0)
    _check(want, (x, res, w, cots), 0.2, None, 4, 0)
    xs = x.to(device).permute(2, 0, 1).contiguous().permute(1, 2, 0).requires_grad_(True)
    rs = torch.cat([res, res], -1).to(device)[..., :96].requires_grad_(True)
    wd = w.to(device).requires_grad_(True)
    out = mhc.rmsnorm_residual(xs, rs, wd, dropout=0.2, seed=4)
    grads = torch.autograd.grad(out, [xs, rs, wd], [c.to(device).transpose(0, 1).contiguous().transpose(0, 1)
                                                    for c in cots])
    assert all(torch.equal(a, b) for a, b in zip([*out, *grads], want))
    # one residual row for all tokens, one x for the batch: their gradients add up
    x1, r1 = x[:1].to(device).requires_grad_(True), res[:, :1].to(device).requires_grad_(True)
    out = mhc.rmsnorm_residual(x1.expand(4, 6, 96), r1.expand(4, 6, 96), wd)
    g1 = torch.autograd.grad(out, [x1, r1], [c.to(device) for c in cots])
    full = [x1.detach().expand(4, 6, 96).clone().requires_grad_(True),
            r1.detach().expand(4, 6, 96).clone().requires_grad_(True)]
    g2 = torch.autograd.grad(mhc.rmsnorm_residual(*full, wd), full, [c.to(device) for c in cots])
    assert torch.equal(g1[0], g2[0].sum(0, keepdim=True)) and torch.equal(g1[1], g2[1].sum(1, keepdim=True))


def test_is_dropout_then_the_sum_then_the_norm(device):
    """fp32: h and the gradients' parts are those of the calls one after the other."""
    x, res, w, cots = [t.to(device) if torch.is_tensor(t) else t for t in _inputs((50, 1000), (F32, F32), 8)]
    y, h = mhc.rmsnorm_residual(x, res, w, dropout=0.4, seed=21, offset=9)
    assert torch.equal(h, res + mhc.dropout(x, 0.4, seed=21, offset=9))
    assert all(torch.equal(a, b) for a, b in zip((y, h), mhc.rmsnorm_residual(
        mhc.dropout(x, 0.4, seed=21, offset=9), res, w)))


@pytest.mark.parametrize("dtypes", DTYPES)
def test_only_the_wanted_gradients(device, dtypes):
    x, res, w, cots = _inputs((40, 520), dtypes, 9)
    for p in (0.0, 0.2):
        full = _run(device, (x, res, w, cots), p, None, 4, 0)[2:]
        for mask in range(1, 8):
            leaves = [t.to(device).requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, res, w))]
            out = mhc.rmsnorm_residual(*leaves, dropout=p, seed=4)
            want = [i for i in range(3) if mask >> i & 1]
            got = torch.autograd.grad(out, [leaves[i] for i in want], [c.to(device) for c in cots])
            assert all(torch.equal(g, full[i]) for g, i in zip(got, want)), mask


def test_gradients_accumulate(device):
    """.backward() twice, one tensor as x and residual, two calls on one tensor."""
    x, res, w, cots = _inputs((30, 96), (F32, F32), 18)
    cots = [c.to(device) for c in cots]
    for p in (0.0, 0.3):
        _, _, dx, dres, dw = _run(device, (x, res, w, [c.cpu() for c in cots]), p, None, 4, 0)
        leaves = [t.to(device).requires_grad_(True) for t in (x, res, w)]
        for n in (1, 2):
            torch.autograd.backward(mhc.rmsnorm_residual(*leaves, dropout=p, seed=4), cots)
            assert all(torch.equal(a.grad, n * e) for a, e in zip(leaves, (dx, dres, dw)))
        one = x.to(device).requires_grad_(True)
        g, = torch.autograd.grad(mhc.rmsnorm_residual(one, one, w.to(device), dropout=p, seed=4), one, cots)
        _, _, dx, dres, _ = _run(device, (x, x, w, [c.cpu() for c in cots]), p, None, 4, 0)
        assert torch.equal(g, dx + dres)


def test_second_derivatives(device):
    """Dropout is linear: the gradient of its gradient is a dropout with the same
    numbers.  The norm has none, and says so."""
    x = torch.randn(8, 40, device=device, requires_grad=True)
    v = torch.randn(8, 40, device=device, requires_grad=True)
    dx, = torch.autograd.grad(mhc.dropout(x, 0.5, seed=3), x, v, create_graph=True)
    u = torch.randn(8, 40, device=device)
    dv, = torch.autograd.grad(dx, v, u)
    assert torch.equal(dv, mhc.dropout(u, 0.5, seed=3)) and torch.equal(dx.detach(), mhc.dropout(v, 0.5, seed=3).detach())
    y, _ = mhc.rmsnorm_residual(x, x, torch.ones(40, device=device))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(y, x, v, create_graph=True)


@pytest.mark.parametrize("which", [0, 1])
def test_one_output_used(device, which):
    """A cotangent that is not there counts as zeros."""
    x, res, w, cots = _inputs((40, 520), (BF16, F32), 10)
    zero = [torch.zeros_like(c) if i != which else c for i, c in enumerate(cots)]
    want = _run(device, (x, res, w, zero), 0.2, None, 4, 0)[2:]
    leaves = [t.to(device).requires_grad_(True) for t in (x, res, w)]
    out = mhc.rmsnorm_residual(*leaves, dropout=0.2, seed=4)[which]
    got = torch.autograd.grad(out, leaves, cots[which].to(device))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def check_packed(packed, h, w, fmt, eps=1e-5):
    """The exponents and numbers of y rounded once: those of the norm in 64 bits.
    The kernel's y is off by less than 2^-40 of it (its mean square takes 64-bit
    sums, its 1 / r two fp32 parts), so where a number 2^-40 to either side rounds
    differently, either is right."""
    C = h.shape[-1]
    y = B.rmsnorm(h.detach().cpu().double(), w.detach().cpu().double(), eps)
    near = [y * (1 - 2.0 ** -40), y * (1 + 2.0 ** -40)]
    e = packed.scales.cpu().double() - 127
    es = [rows8.exponents(v, fmt) for v in near]
    assert bool(((e == es[0]) | (e == es[1])).all())
    same = (es[0] == es[1]).unsqueeze(-1)
    held = packed.values.cpu().view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).double()
    qs = [torch.where(same, rows8.quantised(v, fmt), 0.0).flatten(-2)[..., :C] for v in near]
    got = torch.where(same.expand(*same.shape[:-1], 32).flatten(-2)[..., :C], held[..., :C], 0.0)
    assert bool(((got == qs[0]) | (got == qs[1])).all())
    assert bool((held[..., C:] == 0).all())


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (9, 64), (5, 33), (16, 4096), (17, 1001), (3, 16384), (2, 40000),
                                   (0, 64), (2, 3, 40), (700, 256), (550, 4096), (4, 9001), (2100, 33)])
@pytest.mark.parametrize("dtypes", DTYPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("w_dtype", [F32, BF16])
def test_output_in_8_bits(device, shape, dtypes, fmt, w_dtype):
    x, res, w, _ = _inputs(shape, dtypes, 11, w_dtype)
    dev = [t.to(device) for t in (x, res, w)]
    packed, h = mhc.rmsnorm_residual(*dev, format=fmt)
    C = shape[-1]
    assert isinstance(packed, mhc.PackedActivation) and packed.format == fmt and packed.hidden == C
    assert packed.dtype == x.dtype and torch.equal(h, mhc.rmsnorm_residual(*dev)[1])
    assert packed.values.shape == (*shape[:-1], (C + 15) // 16 * 16) and packed.scales.shape == (*shape[:-1], (C + 31) // 32)
    if x.numel():
        check_packed(packed, h, w, fmt)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_output_in_8_bits_of_small_and_large_rows(device, fmt):
    """eps = 0.  A mean square past fp32's range is 0 or infinite, as it is for y
    in fp32: y is then infinite (its block NaN), or 0."""
    w = torch.ones(96)
    for size in (1e-10, 1e10, 1e-30, 3e19):
        x = (1 + torch.rand(4, 96, generator=_gen(19))) * size
        z = torch.zeros_like(x).to(device)
        packed, h = mhc.rmsnorm_residual(x.to(device), z, w.to(device), eps=0.0, format=fmt)
        if 1e-18 < size < 1e18:
            check_packed(packed, h, w, fmt, 0.0)
        else:
            y = mhc.rmsnorm_residual(x.to(device), z, w.to(device), eps=0.0)[0].cpu()
            up = mhc.activation_unpack(packed).cpu()
            assert bool(up.isnan().all() and y.isinf().all()) if size < 1 else bool((up == 0).all() and (y == 0).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [96, 1000, 4096, 20000])
@pytest.mark.parametrize("size", [1e-18, 1e-19, 1e-20, 1e-21, 3e-22, 1e16, 1e17, 1e18])
def test_output_in_8_bits_near_the_ends_of_fp32(device, fmt, dtype, C, size):
    """eps = 0, and a mean square that fp32 holds, subnormal for values under
    1e-19 or so and up to 2^121: y is rounded once, as anywhere else."""
    x = ((1 + torch.rand(3, C, generator=_gen(33))) * size).to(dtype)
    w = 1 + torch.rand(C, generator=_gen(34))
    packed, h = mhc.rmsnorm_residual(x.to(device), torch.zeros_like(x).to(device), w.to(device), eps=0.0, format=fmt)
    check_packed(packed, h, w, fmt, 0.0)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("C", [96, 1000, 4096, 20000])
@pytest.mark.parametrize("size", [1.0, 0.25, 1024.0])
def test_output_in_8_bits_takes_ties_to_even(device, fmt, C, size):
    """Rows of +-2^k with eps = 0: y is +-w exactly, and half of int8's numbers (a
    16th of e4m3's) are the middle of two.  What is not lost is not rounded."""
    g = _gen(31)
    x = (2.0 * torch.randint(0, 2, (5, C), generator=g) - 1) * size
    w = 1 + torch.randint(0, 128, (C,), generator=g) / 128
    packed, _ = mhc.rmsnorm_residual(x.to(device), torch.zeros(5, C, device=device), w.to(device), eps=0.0, format=fmt)
    want = mhc.activation_pack((x.sign() * w).to(device), fmt)
    assert torch.equal(packed.scales, want.scales) and torch.equal(packed.values, want.values)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("C", [64, 1024, 32768])
def test_output_in_8_bits_past_fp32(device, fmt, C):
    """A norm past fp32's largest number is infinite, as it is for y in fp32: its
    block unpacks to NaN, the others stay."""
    x = torch.zeros(3, C)
    x[:, 5] = torch.tensor([1.0, -2.0, 4.0])  # y = +-sqrt(C) w there
    w = torch.full((C,), 3e38)
    packed, _ = mhc.rmsnorm_residual(x.to(device), torch.zeros(3, C, device=device), w.to(device), eps=0.0, format=fmt)
    up = mhc.activation_unpack(packed).cpu()
    assert bool(up[:, :32].isnan().all()) and bool((up[:, 32:] == 0).all())


def test_values_that_are_not_finite_stay_in_their_rows(device):
    x, res, w, cots = _inputs((12, 200), (F32, F32), 12)
    x[3, 17] = float("inf")
    res[7, 199] = float("nan")
    got = [t.detach().cpu() for t in _run(device, (x, res, w, cots), 0.0, None, 0, 0)]
    bad = torch.zeros(12, dtype=torch.bool)
    bad[[3, 7]] = True
    for t in (got[0], got[2], got[3]):
        assert torch.equal((~t.isfinite()).any(-1), bad)
    assert not bool(got[4].isfinite().all())
    packed, _ = mhc.rmsnorm_residual(x.to(device), res.to(device), w.to(device), format="e4m3")
    up = mhc.activation_unpack(packed).cpu()
    assert torch.equal((~up.isfinite()).any(-1), bad)
    # a dropped value does not count, finite or not
    f = B.factors((12, 200), 0.5, 2)
    x = torch.where(f == 0, float("nan"), x.nan_to_num(posinf=1.0))
    y, h = mhc.rmsnorm_residual(x.to(device), torch.zeros(12, 200, device=device), w.to(device), dropout=0.5, seed=2)
    assert bool(y.isfinite().all()) and bool((h.cpu()[f == 0] == 0).all())


def test_rows_of_zeros(device):
    z = torch.zeros(4, 96, device=device, requires_grad=True)
    w = torch.ones(96, device=device, requires_grad=True)
    y, h = mhc.rmsnorm_residual(z, z.detach(), w)
    g = torch.autograd.grad([y, h], [z, w], [torch.ones_like(y), torch.ones_like(h)])
    assert bool((y == 0).all()) and bool((g[1] == 0).all())
    want = 1 + 1 / torch.sqrt(torch.tensor(1e-5, dtype=torch.float64))
    assert float((g[0].double().cpu() - want).abs().max()) <= 4 * 2.0 ** -24 * float(want)


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_gradient_against_differences(device, fmt):
    """Directional differences of the operator in fp32: steps of 2^-6 of values
    near 1, the curvature's third-order term below 2e-3 of the gradient's terms."""
    g = _gen(13)
    x = torch.randn(32, 96, generator=g).to(device)
    res = mhc.activation_unpack(mhc.activation_pack(torch.randn(32, 96, generator=g).to(device)))
    f = B.factors((32, 96), 0.25, 6).to(device)
    if fmt:  # h at a checkpoint's values
        x = torch.zeros_like(x)
    w = (1 + 0.1 * torch.randn(96, generator=g)).to(device)
    cots = [torch.randn(32, 96, generator=g).to(device) for _ in range(2)]
    vals = [x, res, w]
    call = lambda vs, c=None: mhc.rmsnorm_residual(*vs, dropout=0.25, seed=6, checkpoint=c)  # noqa: E731
    leaves = [v.clone().requires_grad_(True) for v in vals]
    grads = torch.autograd.grad(call(leaves, fmt), leaves, cots)
    loss = lambda vs: sum(float((o.double() * c.double()).sum()) for o, c in zip(call(vs), cots))  # noqa: E731
    h = 2.0 ** -6
    noise = 64 * E32 * sum(float((o * c).double().abs().sum()) for o, c in zip(call(vals), cots)) / h
    for i, v in enumerate(vals):
        d = torch.randn(v.shape, generator=g).to(device)
        hi, lo = list(vals), list(vals)
        hi[i], lo[i] = v + h * d, v - h * d
        diff = (loss(hi) - loss(lo)) / (2 * h)
        want = grads[i].double() * d.double()
        assert abs(diff - float(want.sum())) <= 5e-3 * float(want.abs().sum()) + noise, i
    assert bool((grads[0][f == 0] == 0).all())


def test_two_calls_are_equal_and_do_not_touch_their_inputs(device):
    inputs = _inputs((3000, 1024), (BF16, BF16), 14)
    a, b = (_run(device, inputs, 0.1, None, 5, 0) for _ in range(2))
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    x = inputs[0].to(device)
    keep = x.clone()
    mhc.rmsnorm_residual(x, x, inputs[2].to(device))
    mhc.dropout(x, 0.5, seed=1)
    assert torch.equal(x, keep)


@pytest.mark.parametrize("C", [96, 1024, 16400])
def test_steps_replay_in_a_graph(device, C):
    """The seed in device memory: each replay drops by its own."""
    x, res, w, cots = [t.to(device) if torch.is_tensor(t) else [c.to(device) for c in t]
                       for t in _inputs((40, C), (BF16, F32), 15)]
    seed = torch.tensor([1], device=device)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, res, w)]
        y, h = mhc.rmsnorm_residual(*leaves, dropout=0.2, seed=seed, checkpoint="int8")
        z = mhc.dropout(y, 0.3, seed=seed, offset=1)
        with torch.no_grad():
            packed, _ = mhc.rmsnorm_residual(x, res, w, format="e4m3")
        return [y.detach(), h.detach(), z.detach(), packed.values, packed.scales,
                *torch.autograd.grad([z, h], leaves, cots)]

    graph, outs = _capture(step)
    g = _gen(16)
    feeds = [lambda: seed.add_(1), lambda: x.copy_(torch.randn(x.shape, generator=g)), lambda: seed.fill_(-5),
             lambda: cots[1].copy_(torch.randn(res.shape, generator=g))]
    _replays(graph, outs, step, feeds)


def test_a_drawn_seed_changes_with_each_replay(device):
    x = torch.ones(64, 256, device=device)
    graph, outs = _capture(lambda: [mhc.dropout(x, 0.5)])
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(outs[0].clone())
        x.add_(0)  # eager work between replays
        torch.cuda.synchronize()
    kept = [s != 0 for s in seen]
    for a in range(3):
        assert abs(int(kept[a].sum()) - 8192) < 400  # 6 sigma of 16384 halves
        for b in range(a):
            assert abs(int((kept[a] != kept[b]).sum()) - 8192) < 400


def test_on_a_stream_of_its_own(device):
    inputs = _inputs((500, 2048), (BF16, BF16), 17)
    want = _run(device, inputs, 0.1, None, 5, 0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(device, inputs, 0.1, None, 5, 0)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtypes,fmt", [((F32, F32), None), ((BF16, F32), None), ((F32, BF16), "int8")])
def test_rows_of_millions(device, dtypes, fmt):
    """The bounds do not grow with the row: every term of its sums has one sign and
    one size, so that roundings of a running sum would add up (2^14 of them a lane,
    fp32: 3000 x 2^-24)."""
    C = (1 << 24) + 5
    row = torch.ones(2, C)
    x = (0.2 * row).to(dtypes[0])
    res = (torch.tensor([[0.7], [0.9]]) * row).to(dtypes[1])
    cots = [(0.9 * row).to(dtypes[0]), (0.3 * row).to(dtypes[1])]
    inputs = (x, res, 1.1 * row[0], cots)
    _check(_run(device, inputs, 0.0, fmt, 0, 0), inputs, 0.0, fmt, 0, 0)


def test_rows_past_32_bits(device):
    """More than 2^32 values: the last rows against a call on them (without
    dropout, whose numbers go by the row)."""
    C = 1024
    T = (1 << 32) // C + 40
    x = torch.empty(T, C, dtype=BF16, device=device).fill_(0.5)
    x[-32:] = torch.randn(32, C, device=device).to(BF16)
    w = (torch.rand(C, device=device) + 0.5).to(BF16)
    outs = []
    for a in (x, x[-32:].clone()):
        leaf = a.detach().requires_grad_(True)
        y, h = mhc.rmsnorm_residual(leaf, a, w)
        dx, = torch.autograd.grad([y, h], [leaf], [a, a])
        outs.append([t.detach()[-32:].clone() for t in (y, h, dx)])
        del y, h, dx, leaf
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_refusals(device):
    x, w = torch.zeros(4, 64, device=device), torch.ones(64, device=device)
    t = torch.tensor([1], device=device)
    for call, text in [
            (lambda: mhc.dropout(x, 1.5), "probability"), (lambda: mhc.dropout(x, -0.1), "probability"),
            (lambda: mhc.dropout(x, float("nan")), "probability"),
            (lambda: mhc.dropout(x, 0.5, seed=1, offset=-1), "offset"),
            (lambda: mhc.dropout(x.int(), 0.5), "floating-point"), (lambda: mhc.dropout(x[0, 0], 0.5), "floating-point"),
            (lambda: mhc.dropout(x[:, :0], 0.5), "channels"),
            (lambda: mhc.dropout(x, 0.5, seed=t.int()), "one int64"),
            (lambda: mhc.dropout(x, 0.5, seed=t.repeat(2)), "one int64"),
            (lambda: mhc.dropout(x, 0.5, seed=t.cpu()), "HIP device"),
            (lambda: mhc.rmsnorm_residual(x, x[:2], w), "one shape"), (lambda: mhc.rmsnorm_residual(x, x.int(), w), "one shape"),
            (lambda: mhc.rmsnorm_residual(x, x, w[:32]), "weight"),
            (lambda: mhc.rmsnorm_residual(x, x, w.view(1, 64)), "weight"),
            (lambda: mhc.rmsnorm_residual(x, x, w, dropout=2.0), "probability"),
            (lambda: mhc.rmsnorm_residual(x, x, w.requires_grad_(True), format="int8"), "no gradient"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_an_error(device, grad):
    x, w = torch.randn(4, 64, device=device), torch.ones(64, device=device)
    fwd = torch.autograd.forward_ad
    for i in range(3):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            args = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate((x, x, w))]
            with pytest.raises(RuntimeError, match="jvp is not implemented"):
                mhc.rmsnorm_residual(*args)
            if i == 0:
                with pytest.raises(RuntimeError, match="jvp is not implemented"):
                    mhc.dropout(args[0], 0.5, seed=1)


# ---------------------------------------------------------------------------
# The residual wrapper's dropout
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("C", [64, 66])
def test_residual_wrapper_drops_its_branch_in_training(device, dynamic, C):
    torch.manual_seed(1)
    kw = {"use_dynamic_h": dynamic and C % 8 == 0}
    wrap = mhc.MHCResidualWrapper(C, 4, dropout=0.3, **kw).to(device)
    plain = mhc.MHCResidualWrapper(C, 4, **kw).to(device)
    plain.load_state_dict(wrap.state_dict())
    r, b = torch.randn(20, C, device=device), torch.randn(20, C, device=device, requires_grad=True)
    torch.manual_seed(2)
    out = wrap(r, b)
    g, = torch.autograd.grad(out.square().sum(), b)
    torch.manual_seed(2)
    dropped = mhc.dropout(b, 0.3)
    want = plain(r, dropped)
    gw, = torch.autograd.grad(want.square().sum(), b)
    assert torch.equal(out, want) and torch.equal(g, gw)
    assert bool((g[dropped == 0] == 0).all()) and bool((dropped == 0).any())
    wrap.eval()
    plain.eval()
    assert torch.equal(wrap(r, b), plain(r, b))


@pytest.mark.parametrize("dtype", [F32, BF16, torch.float16])
@pytest.mark.parametrize("shape", [(6, 64), (2, 5, 64), (3, 1, 64), (0, 64)])
def test_residual_wrapper_takes_what_it_took(device, dtype, shape):
    """Every shape and dtype of the wrapper without dropout, with it."""
    torch.manual_seed(1)
    wrap = mhc.MHCResidualWrapper(64, 4, dropout=0.3, use_dynamic_h=False).to(device)
    plain = mhc.MHCResidualWrapper(64, 4, use_dynamic_h=False).to(device)
    plain.load_state_dict(wrap.state_dict())
    r, b = (torch.randn(*shape, device=device).to(dtype) for _ in range(2))
    torch.manual_seed(2)
    out = wrap(r, b)
    torch.manual_seed(2)
    assert torch.equal(out, plain(r, mhc.dropout(b, 0.3).to(dtype)))
    wrap.dropout = 1.0
    assert torch.equal(wrap(r, b), plain(r, torch.zeros_like(b)))
