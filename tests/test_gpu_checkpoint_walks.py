"""Backward passes over a checkpoint where a workgroup walks several tokens and
a token tile several stages, every gradient against 64 bits; the wrapper whose
streams are the rows that it keeps; weight gradients at the sums they take.

The 64-bit operator runs on the device.  x^ is activation_unpack's, whose bits
tests/test_gpu_checkpoint.py compares with the format's definition.

Tolerances.  Independent roundings of fp32 add in the 2-norm: a chain of N of
them leaves sqrt(N) 2^-24 of the result, where terms of random sign are what it
sums.  Sums over channels, tokens and output rows take under 256 additions in
sequence (16 * 2^-24); the coefficients' adjoint puts 20 Sinkhorn iterations of
some 16 roundings each on top, for the parameters that are one sum over tokens
(32 * 2^-24 of the terms' 2-norm plus the sum, since the terms may cancel)."""
import pytest
import torch

import mhc_ascend_amd as mhc
from oracle import reference as R
from oracle import rows8
from tests.conftest import assert_close_bf16, assert_close_dyn_dx_bf16
from tests.test_gpu_checkpoint import DTYPES, FORMATS, K_ROW, _gen, _norm_oracle, _within

pytestmark = pytest.mark.gpu

NORM, SINGLE = 16 * 2.0 ** -24, 32 * 2.0 ** -24


def _tokens(device, rounds, more):
    return rounds * torch.cuda.get_device_properties(device).multi_processor_count + more


def _inputs(device, B, n, C, dtype, dynamic):
    g = torch.Generator(device=device).manual_seed(B + 10 * n + C)
    rand = lambda *s: torch.randn(*s, device=device, generator=g)
    x, cot = rand(B, n, C).to(dtype), rand(B, n, C)
    ps = [1 + 0.1 * rand(C)]
    if dynamic:
        ps += [rand(r, n * C) * (n * C) ** -0.5 for r in (n, n, n * n)] + [torch.tensor(0.7, device=device) for _ in "abc"]
    ps += [0.5 * rand(n), 0.5 * rand(n), 0.5 * rand(n, n)]
    return x, cot, ps


def _exact(x, xh, ps, cot, dynamic):
    """Output at x, (dx, dw, dPhi) at x^, and the terms [B, ...] of each
    parameter that all tokens share (alphas and biases, or the H)."""
    x, cot, ps = x.double(), cot.double(), [p.double() for p in ps]
    xh = xh.double().requires_grad_(True)
    B, n, C = x.shape
    w = ps[0].requires_grad_(True)
    shared = [p.expand(B, *p.shape).clone().requires_grad_(True) for p in ps[4 if dynamic else 1:]]
    phi = [p.requires_grad_(True) for p in ps[1:4]] if dynamic else []

    def layer(rows):
        if dynamic:
            ap, aq, ar, bp, bq, br = shared
            flat, hflat = x.reshape(B, -1), rows.reshape(B, -1)
            prod, ms = hflat @ torch.cat(phi).t(), hflat.square().mean(-1, keepdim=True)
            prod = prod + (flat @ torch.cat(phi).t() - prod).detach()
            ms = ms + (flat.square().mean(-1, keepdim=True) - ms).detach()
            t = prod / torch.sqrt(ms + 1e-5)
            pre, post = ap[:, None] * t[:, :n] + bp, aq[:, None] * t[:, n:2 * n] + bq
            res = ar[:, None, None] * t[:, 2 * n:].reshape(B, n, n) + br
        else:
            pre, post, res = shared
        return R._layer_core(rows, w, torch.sigmoid(pre), 2 * torch.sigmoid(post),
                             R.sinkhorn_knopp(torch.exp(res), 20, 1e-8), 1e-5)

    with torch.no_grad():
        out = layer(x)
    grads = torch.autograd.grad(layer(xh), [xh, w, *phi, *shared], cot)
    k = 2 + len(phi)
    return out, grads[:k], grads[k:]


def _walk(device, fmt, dtype, B, n, C, dynamic):
    x, cot, ps = _inputs(device, B, n, C, dtype, dynamic)
    leaves = [t.clone().requires_grad_(True) for t in (x, *ps)]
    call = mhc.mhc_layer_fused_dynamic_training if dynamic else mhc.mhc_layer_static
    out = call(*leaves, checkpoint=fmt)
    got = torch.autograd.grad(out, leaves, cot)
    xh = mhc.activation_unpack(mhc.activation_pack(x, fmt), torch.float32)
    want, grads, terms = _exact(x, xh, ps, cot, dynamic)

    def near(a, e, tol, what):
        err = float((a.detach().double() - e).norm() / e.norm())
        assert err <= tol, f"{what}: {err:.3g}, {tol:.3g} allowed"

    near(out, want, NORM, "out")
    if dtype == torch.bfloat16:
        (assert_close_dyn_dx_bf16 if dynamic else assert_close_bf16)(got[0], grads[0], "dx")
    else:
        near(got[0], grads[0], NORM, "dx")
    for i, e in enumerate(grads[1:]):
        near(got[1 + i], e, NORM, f"gradient {1 + i} (the weight and the projections)")
    for a, t in zip(got[1 + len(grads[1:]):], terms):
        bound = SINGLE * (t.square().sum(0).sqrt() + t.sum(0).abs())
        worst = float(((a.double() - t.sum(0)).abs() / bound).max())
        assert worst <= 1.0, f"sums over tokens {tuple(a.shape)}: {worst:.3g} times their bound"


# n, tokens as rounds of the device's CUs and a rest, hidden.  A backward
# workgroup takes the tokens two at a time where it prefetches: two to twenty of
# them here, odd last rounds among them; 512 lanes with two chunks at 4096.
STATIC = [(4, 4, 3, 1024), (2, 5, 1, 2048), (4, 5, 2, 4096), (3, 20, 7, 160), (6, 9, 5, 1040), (8, 9, 5, 512),
          (5, 9, 5, 320), (7, 6, 1, 224), (4, 17, 0, 128), (4, 3, 1, 1001), (12, 3, 1, 96)]
# A projection tile of several stages of 64 tokens, the last one ragged; up to 96
# projection rows in one launch, two and three launches from n = 9 on.
DYNAMIC = [(4, 5, 1, 4096), (4, 5, 3, 2048), (2, 6, 3, 2048), (3, 20, 7, 160), (5, 9, 5, 320), (6, 9, 5, 1040),
           (7, 6, 1, 224), (8, 9, 5, 1280), (4, 20, 7, 136), (12, 20, 1, 224), (16, 20, 1, 64)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rounds,more,C", STATIC)
def test_static_layer_over_many_tokens(device, fmt, dtype, n, rounds, more, C):
    _walk(device, fmt, dtype, _tokens(device, rounds, more), n, C, False)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rounds,more,C", DYNAMIC)
def test_dynamic_layer_over_many_tokens(device, fmt, dtype, n, rounds, more, C):
    _walk(device, fmt, dtype, _tokens(device, rounds, more), n, C, True)


@pytest.mark.parametrize("dynamic,dtype", [(False, torch.float32), (True, torch.bfloat16)])
def test_layers_at_a_training_size(device, dynamic, dtype):
    """[8192, 4, 4096].  The alphas' gradients are one sum of 8192 terms (32768
    and 131072 products) each, that may come out at any part of their 2-norm."""
    _walk(device, "int8", dtype, 8192, 4, 4096, dynamic)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dynamic,n,C,mode", [(False, 3, 70, "decay"), (False, 4, 33, "zero"), (True, 11, 192, "decay")])
def test_wrapper_that_keeps_its_streams(device, fmt, dtype, dynamic, n, C, mode):
    """A shape without a fused wrapper builds the streams and keeps those: the
    gradients are the layer's at their x^, pushed through the construction, bit
    for bit with static H (the layer's own kernels behind an unpack pass)."""
    torch.manual_seed(n + C)
    wrap = mhc.MHCResidualWrapper(C, n, residual_mode=mode, use_dynamic_h=dynamic, alpha_init=0.2,
                                  **({"sinkhorn_eps": 1e-3} if dynamic else {})).to(device)
    rows = [torch.randn(37, C, generator=_gen(k)).to(dtype) for k in range(2)]
    cot = torch.randn(37, C, generator=_gen(5)).to(device)
    params = list(wrap.parameters())

    class AtHeld(torch.autograd.Function):  # the layer's gradient at x^, its output at x
        @staticmethod
        def forward(ctx, X, layer):
            ctx.layer, ctx.hat = layer, rows8.held(X, fmt).to(X.dtype).to(X.device)
            return layer(X)

        @staticmethod
        def backward(ctx, g):
            with torch.enable_grad():
                X = ctx.hat.requires_grad_(True)
                gx, *gp = torch.autograd.grad(ctx.layer(X), [X, *params], g)
            AtHeld.grads = gp
            return gx, None

    def streams(r, b):
        X = torch.zeros(37, n, C, device=device, dtype=dtype)
        X[:, 0], X[:, 1] = r, b
        if mode == "decay":
            for i in range(2, n):
                X[:, i] = r * 0.1 ** (i - 1)
        return X

    leaves = [r.to(device).requires_grad_(True) for r in rows]
    want_out = AtHeld.apply(streams(*leaves), wrap.mhc).mean(1)
    want = [*torch.autograd.grad(want_out, leaves, cot), *AtHeld.grads]
    wrap.mhc.checkpoint = fmt
    leaves = [r.to(device).requires_grad_(True) for r in rows]
    out = wrap(*leaves)
    got = torch.autograd.grad(out, leaves + params, cot)
    assert torch.equal(out, want_out)
    if not dynamic:
        assert all(torch.equal(a, e) for a, e in zip(got, want))
        return
    # The layer at x^ forms its coefficients there, the checkpoint's backward keeps
    # the forward's: they differ by the checkpoint's error, under 2^-4 of a value,
    # through 0.2 and the projection.  The mean gives every stream one cotangent,
    # so dL/dM is the same in every row of a column, and with the columns of M
    # summing to one no change of H_res changes the loss: those gradients are zero
    # but for eps and rounding, and each is held to the largest of its family (pre,
    # post and res of one parameter; residual and branch; the weight).
    names = ["residual", "branch", *(k for k, _ in wrap.named_parameters())]
    family = [k.split("_")[0].split(".")[-1] if k not in ("residual", "branch") else "rows" for k in names]
    for k, a, e in zip(family, got, want):
        scale = max(float(v.double().norm()) for f, v in zip(family, want) if f == k)
        assert float((a.double() - e.double()).norm()) <= 2.0 ** -4 * scale, k


def _rms_adds(device, B, C):
    """Additions in sequence of a weight's gradient: a lane's rows, its groups
    and waves, then 32 phases of the workgroups' partials."""
    cus = torch.cuda.get_device_properties(device).multi_processor_count
    if C <= 512:
        lanes = 4
        while 8 * lanes < C:
            lanes *= 2
        each = 8 * (64 // lanes)
        grid = min(2 * cus, -(-B // each))
        return -(-B // (grid * each)) + 6 + 8 + -(-grid // 32) + 32
    grid = min(2 * cus, B)  # or more workgroups, with 16 rows each at least
    return max(-(-B // grid), 16) + -(-max(grid, 16 * cus) // 32) + 32


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C", [(2999, 1001), (4096, 4096), (20000, 1024), (35003, 100), (20001, 7), (9000, 512), (70, 64)])
def test_rmsnorm_weight_gradient_at_the_sums_it_takes(device, fmt, dtype, B, C):
    x, g = (torch.randn(B, C, generator=_gen(B + C + k)).to(dtype) for k in range(2))
    w = 1 + 0.1 * torch.randn(C, generator=_gen(C))
    leaves = [t.to(device).requires_grad_(True) for t in (x, w)]
    gw = torch.autograd.grad(mhc.rmsnorm(*leaves, checkpoint=fmt), leaves, g.to(device))[1]
    xh = mhc.activation_unpack(mhc.activation_pack(x.to(device), fmt)).cpu().double()
    _, _, _, dw, mag = _norm_oracle(x, xh, w, g)
    _within(gw, dw, (K_ROW + _rms_adds(device, B, C)) * 2.0 ** -24 * mag + 1e-30, "dw")
