"""Autograd functions over the HIP kernels (mirror of src/python/mhc/ops.py).

The autograd nodes of the layers, the wrapper and the stand-alone operators
are C++ (csrc/autograd.cpp); the projection's is a Python Function, and so are
the operators' where a Python one is needed (_NodeFunction).

Public functional ops keep the reference's names, arguments and defaults.
Documented differences from the Ascend implementation (all toward the
PyTorch reference math, which is the contract):
  * arithmetic is fp32 end to end; the Ascend path rounds several
    intermediates to bf16 (ops.py:105-107, 218, 243, 280-281);
  * standalone ops return the dtype of their input instead of bf16;
  * the Sinkhorn backward is the exact gradient (the Ascend kernel's row
    step is approximate, sinkhorn_knopp.cpp:1773-1795);
  * alpha parameters stay on the device (no ``.item()`` host syncs,
    ops.py:362-364, 420-422, 533-535).
"""
from __future__ import annotations

import operator
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib, native

# Projection rows above which the library's dynamic forward streams the fp32
# projections (2n + n^2 > 128: n >= 16) instead of split planes.
_STREAM_PROJ_ROWS = 128


class _NodeFunction(torch.autograd.Function):
    """A stand-alone operator's autograd function.  ``apply`` runs its C++ node;
    under ``torch.jit.trace``, which records Python functions only, and for
    subclasses it runs ``forward`` / ``backward``, over the same entries."""

    @classmethod
    def apply(cls, *args):
        if "node" not in vars(cls) or torch.jit.is_tracing():
            return super().apply(*args)
        return cls.node(*args)


# =============================================================================
# 8-bit checkpoints of saved rows (no counterpart in the reference)
# =============================================================================

_CHECKPOINTS = {None: -1, "int8": _lib.INT8, "e4m3": _lib.E4M3}


def _checkpoint_code(checkpoint: Optional[str]) -> int:
    """The library's code of a ``checkpoint`` argument."""
    try:
        return _CHECKPOINTS[checkpoint]
    except (KeyError, TypeError):
        raise ValueError(f"Unknown checkpoint format: {checkpoint!r} (None, 'int8' or 'e4m3')") from None


def _not_traced(what: str) -> None:
    """torch.jit.trace records Python functions only: a C++ node's result would
    become a constant of the trace."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} is not recorded by torch.jit.trace")


def _operator_checkpoint(checkpoint: Optional[str]) -> int:
    """The same for an operator's call: with a checkpoint torch.jit.trace does
    not record it (the Python functions that it does record save the rows as
    they are)."""
    if checkpoint is None:
        return -1
    code = _checkpoint_code(checkpoint)
    _not_traced("checkpoint=")
    return code


class PackedActivation(NamedTuple):
    """Rows in 8 bits, from :func:`activation_pack`.

    ``values`` [..., ceil16(hidden)] uint8 are int8 or e4m3 numbers (the bytes
    past ``hidden`` are zero), ``scales`` [..., ceil(hidden / 32)] uint8 the
    exponents e + 127 of their blocks of 32: a value stands for q * 2**e, or
    NaN where the byte is 255 (the block held a value that is not finite)."""

    values: torch.Tensor
    scales: torch.Tensor
    format: str
    hidden: int
    dtype: torch.dtype


def activation_pack(x: torch.Tensor, format: str = "int8") -> PackedActivation:
    """Hold x [..., C] in 8 bits, 33/32 bytes a value (rows padded to 16).

    With a = max |x| of a block of 32 and M = 127 ("int8") or 448 ("e4m3"), e
    is the least integer with a <= M 2^e (at least -100); the block holds
    x 2^-e rounded to nearest even.  The error is at most 2^(e-1) ("int8") or
    max(2^-4 |x|, 2^(e-10)) ("e4m3").  No gradient flows through."""
    if format is None:
        raise ValueError("activation_pack: format must be 'int8' or 'e4m3'")
    code = _checkpoint_code(format)
    _not_traced("activation_pack")
    return PackedActivation(*_lib.autograd().checkpoint_pack(x, code), format, x.shape[-1],
                            x.dtype if x.dtype in (torch.float32, torch.bfloat16) else torch.float32)


def activation_unpack(packed: PackedActivation, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values a :class:`PackedActivation` stands for, exactly, in ``dtype``
    (float32 or bfloat16; the packed tensor's storage dtype by default)."""
    if packed.format is None:
        raise ValueError("activation_unpack: format must be 'int8' or 'e4m3'")
    _not_traced("activation_unpack")
    dtype = _lib.dtype_code(packed.dtype if dtype is None else dtype)
    return _lib.autograd().checkpoint_unpack(packed.values, packed.scales, _checkpoint_code(packed.format),
                                             int(packed.hidden), dtype == _lib.BF16)


# =============================================================================
# Sinkhorn-Knopp (ops.py:32-80)
# =============================================================================

class SinkhornKnoppFunction(_NodeFunction):
    """Sinkhorn-Knopp doubly stochastic normalisation of [B, n, n]."""

    @staticmethod
    def forward(ctx, inp: torch.Tensor, num_iters: int = 20, eps: float = 1e-8) -> torch.Tensor:
        out = native.sinkhorn_knopp_fwd(inp, num_iters, eps)
        ctx.save_for_backward(inp, out)
        ctx.num_iters = num_iters
        ctx.eps = eps
        return out

    @staticmethod
    def backward(ctx, grad_out: torch.Tensor):
        inp, out = ctx.saved_tensors
        grad_inp = native.sinkhorn_knopp_bwd(grad_out.float().contiguous(), inp, out, ctx.num_iters, ctx.eps)
        return grad_inp, None, None

    @staticmethod
    def node(inp, num_iters=20, eps=1e-8):
        return _lib.autograd().sinkhorn_knopp(inp, int(num_iters), float(eps))


def sinkhorn_knopp(inp: torch.Tensor, num_iters: int = 20, eps: float = 1e-8) -> torch.Tensor:
    """Apply Sinkhorn-Knopp normalisation to a batch of matrices [B, n, n]."""
    return SinkhornKnoppFunction.apply(inp.float(), num_iters, eps)


# =============================================================================
# RMSNorm (ops.py:87-136)
# =============================================================================

class RMSNormFunction(_NodeFunction):
    """Root Mean Square normalisation of [B, C] rows."""

    @staticmethod
    def forward(ctx, inp: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
        out, rms = native.rmsnorm_fwd(inp, weight, eps)
        ctx.save_for_backward(inp, weight, rms)
        ctx.eps = eps
        return out

    @staticmethod
    def backward(ctx, grad_out: torch.Tensor):
        inp, weight, rms = ctx.saved_tensors
        grad_inp, grad_weight = native.rmsnorm_bwd(grad_out, inp, weight, rms)
        return grad_inp.to(inp.dtype), grad_weight, None

    @staticmethod
    def node(inp, weight, eps=1e-5):
        return _lib.autograd().rmsnorm(inp, weight, float(eps))


def rmsnorm(inp: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
            checkpoint: Optional[str] = None) -> torch.Tensor:
    """RMSNorm of inp [B, C]; the output keeps inp's dtype (fp32 or bf16).

    ``checkpoint`` ("int8" or "e4m3", see :func:`activation_pack`) saves inp in
    8 bits for the backward, which is then RMSNorm's gradient at the values
    that checkpoint stands for (C <= 16384)."""
    code = _operator_checkpoint(checkpoint)
    if code >= 0:
        return _lib.autograd().rmsnorm(inp, weight, float(eps), code)
    return RMSNormFunction.apply(inp, weight, eps)


# =============================================================================
# Stream aggregate (ops.py:143-188)
# =============================================================================

class StreamAggregateFunction(_NodeFunction):
    """out = sum_i sigmoid(H_pre_raw[:, i]) * inp[:, i]."""

    @staticmethod
    def forward(ctx, inp: torch.Tensor, H_pre_raw: torch.Tensor) -> torch.Tensor:
        out, h_act = native.stream_aggregate_fwd(inp, H_pre_raw)
        ctx.save_for_backward(inp, h_act)
        return out

    @staticmethod
    def backward(ctx, grad_out: torch.Tensor):
        inp, h_act = ctx.saved_tensors
        gx, _, graw = native._aggregate_bwd(grad_out, inp, h_act, True)
        return gx.to(inp.dtype), graw

    @staticmethod
    def node(inp, H_pre_raw):
        return _lib.autograd().stream_aggregate(inp, H_pre_raw)


def stream_aggregate(inp: torch.Tensor, H_pre_raw: torch.Tensor, checkpoint: Optional[str] = None) -> torch.Tensor:
    """Aggregate [B, n, C] streams with sigmoid weights H_pre_raw [B, n].
    ``checkpoint`` saves inp in 8 bits for the backward, as :func:`rmsnorm`'s."""
    code = _operator_checkpoint(checkpoint)
    if code >= 0:
        return _lib.autograd().stream_aggregate(inp, H_pre_raw, code)
    return StreamAggregateFunction.apply(inp, H_pre_raw)


# =============================================================================
# Stream distribute-mix-add (ops.py:195-265)
# =============================================================================

class StreamDistributeMixAddFunction(_NodeFunction):
    """out[:, i] = 2 sigmoid(H_post_raw[:, i]) * y_norm + sum_j M[:, i, j] x[:, j]."""

    @staticmethod
    def forward(ctx, y_norm, H_post_raw, M, x_inp):
        out, h_act = native.stream_distribute_mix_add_fwd(y_norm, H_post_raw, M, x_inp)
        ctx.save_for_backward(x_inp, y_norm, M, h_act)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        x_inp, y_norm, M, h_act = ctx.saved_tensors
        gx, gy, gM, _, graw = native._distribute_bwd(grad_out, x_inp, y_norm, M, h_act, True)
        return gy.to(y_norm.dtype), graw, gM, gx.to(x_inp.dtype)

    @staticmethod
    def node(y_norm, H_post_raw, M, x_inp):
        return _lib.autograd().stream_distribute_mix_add(y_norm, H_post_raw, M, x_inp)


def stream_distribute_mix_add(y_norm: torch.Tensor, H_post_raw: torch.Tensor, M: torch.Tensor,
                              x_inp: torch.Tensor, checkpoint: Optional[str] = None) -> torch.Tensor:
    """Distribute y_norm [B, C] to n streams, mix x_inp [B, n, C] with M and add (fp32 out).
    ``checkpoint`` saves y_norm and x_inp in 8 bits for the backward, as :func:`rmsnorm`'s."""
    code = _operator_checkpoint(checkpoint)
    if code >= 0:
        return _lib.autograd().stream_distribute_mix_add(y_norm, H_post_raw, M, x_inp, code)
    return StreamDistributeMixAddFunction.apply(y_norm, H_post_raw, M, x_inp)


stream_distribute = stream_distribute_mix_add


def compute_rms(x_flat: torch.Tensor, eps: float = 1e-8) -> torch.Tensor:
    """Per-row RMS of x_flat [B, K] (ops.py:318-330); no autograd, as in the reference."""
    return native.compute_rms_fwd(x_flat, eps)


# =============================================================================
# Fused static-H layer (layer.py:142-170 as one HBM pass per direction)
# =============================================================================

def mhc_layer_static(x: torch.Tensor, rmsnorm_weight: torch.Tensor, H_pre: torch.Tensor, H_post: torch.Tensor,
                     H_res: torch.Tensor, sinkhorn_iters: int = 20, sinkhorn_eps: float = 1e-8,
                     rmsnorm_eps: float = 1e-5, checkpoint: Optional[str] = None) -> torch.Tensor:
    """Static-H mHC layer on x [B, n, C] -> fp32 [B, n, C]: one fused pass per
    direction (layer.py:142-170), autograd node in C++ (_mhc_autograd.so).

    ``checkpoint`` ("int8" or "e4m3", see :func:`activation_pack`) saves x in 8
    bits for the backward, which is then the layer's gradient at the values
    that checkpoint stands for."""
    return _lib.autograd().static_layer(x, rmsnorm_weight, H_pre, H_post, H_res, int(sinkhorn_iters),
                                        float(sinkhorn_eps), float(rmsnorm_eps), _operator_checkpoint(checkpoint))


# =============================================================================
# Dynamic-H projection (ops.py:272-315)
# =============================================================================

class FusedProjectionFunction(torch.autograd.Function):
    """P = x_flat @ phi_concat^T (fp32), with its backward."""

    @staticmethod
    def forward(ctx, x_flat: torch.Tensor, phi_concat: torch.Tensor) -> torch.Tensor:
        out = native.fused_rmsnorm_matmul_fwd(x_flat, phi_concat)
        ctx.save_for_backward(x_flat, phi_concat)
        return out

    @staticmethod
    def backward(ctx, grad_out: torch.Tensor):
        x_flat, phi_concat = ctx.saved_tensors
        gx, gphi = native.fused_rmsnorm_matmul_bwd(grad_out, x_flat, phi_concat)
        return gx.to(x_flat.dtype), gphi.to(phi_concat.dtype)


def fused_rmsnorm_matmul(x_flat: torch.Tensor, phi_concat: torch.Tensor) -> torch.Tensor:
    """Project x_flat [B, K] with phi_concat [out_dim, K] -> fp32 [B, out_dim]."""
    return FusedProjectionFunction.apply(x_flat, phi_concat)


# =============================================================================
# Dynamic-H layer (ops.py:337-628)
# =============================================================================

def mhc_layer_fused_dynamic_inference(x_expanded, rmsnorm_weight, phi_pre, phi_post, phi_res, alpha_pre,
                                      alpha_post, alpha_res, b_pre, b_post, b_res, sinkhorn_iters: int = 20,
                                      sinkhorn_eps: float = 1e-8, rmsnorm_eps: float = 1e-5,
                                      out_dtype: torch.dtype = torch.float32, packed=None) -> torch.Tensor:
    """Dynamic-H forward without autograd state (ops.py:337-380).

    Extensions (keyword-only in practice, defaults give the reference's
    result): ``out_dtype=torch.bfloat16`` writes the output in bf16;
    ``packed`` (from native.mhc_layer_dynamic_pack on the same weight and
    projections) skips the per-call packing of the parameters."""
    if packed is None:
        if out_dtype == torch.float32 and 2 * phi_pre.shape[0] + phi_res.shape[0] > _STREAM_PROJ_ROWS:
            # More than 128 projection rows: the forward reads the fp32
            # projections directly (no packing pass), and its fp32 output is
            # the packed entry's bit for bit.
            return native.mhc_layer_dynamic_fwd(x_expanded, rmsnorm_weight, phi_pre, phi_post, phi_res, alpha_pre,
                                                alpha_post, alpha_res, b_pre, b_post, b_res, sinkhorn_iters,
                                                sinkhorn_eps, rmsnorm_eps)[0]
        packed = native.mhc_layer_dynamic_pack(rmsnorm_weight, phi_pre, phi_post, phi_res)
    if (out_dtype in (torch.float32, torch.bfloat16) and torch.is_tensor(alpha_pre) and torch.is_tensor(alpha_post)
            and torch.is_tensor(alpha_res)):
        return _lib.autograd().dynamic_infer(x_expanded, packed, alpha_pre, alpha_post, alpha_res, b_pre, b_post,
                                             b_res, int(sinkhorn_iters), float(sinkhorn_eps), float(rmsnorm_eps),
                                             out_dtype == torch.bfloat16)
    return native.mhc_layer_dynamic_infer(x_expanded, packed, alpha_pre, alpha_post, alpha_res, b_pre, b_post, b_res,
                                          sinkhorn_iters, sinkhorn_eps, rmsnorm_eps, out_dtype)


def mhc_layer_fused_dynamic_training(x_expanded, rmsnorm_weight, phi_pre, phi_post, phi_res, alpha_pre, alpha_post,
                                     alpha_res, b_pre, b_post, b_res, sinkhorn_iters: int = 20,
                                     sinkhorn_eps: float = 1e-8, rmsnorm_eps: float = 1e-5,
                                     checkpoint: Optional[str] = None) -> torch.Tensor:
    """Dynamic-H layer with autograd (ops.py:567-628).  Float alphas become
    device tensors; alpha tensors stay on the device (no .item() syncs).

    ``checkpoint`` ("int8" or "e4m3", see :func:`activation_pack`) saves x in 8
    bits: the backward takes the streams from it and keeps the forward's own
    per-token coefficients, projections and their RMS, which it saves as well."""
    dev = phi_pre.device
    if not torch.is_tensor(alpha_pre):
        alpha_pre = torch.tensor(alpha_pre, device=dev, dtype=torch.float32)
    if not torch.is_tensor(alpha_post):
        alpha_post = torch.tensor(alpha_post, device=dev, dtype=torch.float32)
    if not torch.is_tensor(alpha_res):
        alpha_res = torch.tensor(alpha_res, device=dev, dtype=torch.float32)
    return _lib.autograd().dynamic_layer(x_expanded, rmsnorm_weight, phi_pre, phi_post, phi_res, alpha_pre,
                                         alpha_post, alpha_res, b_pre, b_post, b_res, int(sinkhorn_iters),
                                         float(sinkhorn_eps), float(rmsnorm_eps), _operator_checkpoint(checkpoint))


# =============================================================================
# Fused MHCResidualWrapper (layer.py:269-322)
# =============================================================================

def mhc_residual_wrapper(residual: torch.Tensor, branch_output: torch.Tensor, layer, residual_mode: str = "decay"):
    """Fused MHCResidualWrapper on residual / branch_output [tokens, C] for the
    parameters of ``layer`` (an MHCLayer); returns fp32 [tokens, C].  With the
    layer's ``checkpoint`` the saved rows, residual and branch_output (or the
    streams of a shape that is not fused), are kept in 8 bits."""
    checkpoint = _operator_checkpoint(getattr(layer, "checkpoint", None))
    n = layer.expansion_rate
    C = residual.shape[-1]
    # The fused wrapper kernels take 4-channel rows and n = 2..32; with
    # dynamic H also n*C a multiple of the projection's k step of 32, up to
    # 2^22, and past n = 10 (2n + n^2 > 128 projection rows) Sinkhorn
    # settings under which the H_res gradients vanish (at least one
    # iteration, eps <= 1e-6: the defaults).  Other shapes build the n
    # streams with device tensor ops, as layer.py:299-310 does, and run the
    # layer on them (layer.py:313-316).
    fused = 2 <= n <= 32 and C % 4 == 0
    if layer.use_dynamic_h:
        # the library's test, in float32: iters >= 1 and 0 <= eps <= 1e-6f
        eps32 = float(torch.tensor(float(layer.sinkhorn_eps), dtype=torch.float32))
        vanish = int(layer.num_sinkhorn_iters) >= 1 and 0.0 <= eps32 <= float(torch.tensor(1e-6, dtype=torch.float32))
        fused = fused and (n * C) % 32 == 0 and n * C <= 1 << 22 and (n <= 10 or vanish)
    if not fused:
        if n < 2:
            raise RuntimeError("mhc_residual_wrapper: expansion_rate must be >= 2 (stream 1 holds the branch)")
        if residual_mode not in ("zero", "decay"):
            raise ValueError(f"Unknown residual_mode: {residual_mode}")
        X = torch.zeros(residual.shape[0], n, C, device=residual.device, dtype=residual.dtype)
        X[:, 0] = residual
        X[:, 1] = branch_output
        if residual_mode == "decay":
            for i in range(2, n):
                X[:, i] = residual * (0.1 ** (i - 1))
        return layer(X).mean(dim=1)
    iters, sk_eps, rms_eps = int(layer.num_sinkhorn_iters), float(layer.sinkhorn_eps), float(layer.rmsnorm_eps)
    ag = _lib.autograd()
    if layer.use_dynamic_h:
        return ag.dynamic_wrapper(residual, branch_output, layer.rmsnorm_weight, layer.phi_pre, layer.phi_post,
                                  layer.phi_res, layer.alpha_pre, layer.alpha_post, layer.alpha_res, layer.b_pre,
                                  layer.b_post, layer.b_res, residual_mode, n, iters, sk_eps, rms_eps, checkpoint)
    return ag.static_wrapper(residual, branch_output, layer.rmsnorm_weight, layer.H_pre, layer.H_post, layer.H_res,
                             residual_mode, n, iters, sk_eps, rms_eps, checkpoint)


# =============================================================================
# Dropout without a stored mask, RMSNorm of a residual's sum (no counterpart in
# the reference)
# =============================================================================

def _seed(fn: str, seed) -> Tuple[Optional[torch.Tensor], Optional[int]]:
    """A ``seed`` argument as (tensor, None) or (None, the signed 64-bit value);
    (None, None) where it is to be drawn."""
    if seed is None or torch.is_tensor(seed):
        return seed, None
    seed = operator.index(seed)
    if not -2 ** 63 <= seed < 2 ** 64:
        raise ValueError(f"{fn}: seed must fit 64 bits, got {seed}")
    return None, seed - 2 ** 64 if seed >= 2 ** 63 else seed


def dropout(x: torch.Tensor, p: float = 0.5, seed=None, offset: int = 0) -> torch.Tensor:
    """Dropout of x [..., C] whose mask is never stored: forward and backward
    compute it from a counter.

    With t = round(p * 2**16), a value is kept, times 2**16 / (2**16 - t), where
    its 16-bit number is at least t, and 0 elsewhere.  Channels 8 j .. 8 j + 7 of
    row i (rows counted over the leading dimensions) take the numbers of one
    Philox4x32-10 block: counter (i * ceil(C / 8) + j, ``offset``), key ``seed``.

    ``seed`` is an int of 64 bits, or an int64 tensor of one element on x's
    device, read when the call runs: a captured graph that changes it between
    replays drops other values in each.  It has to hold its value until the
    backward.  Without one the call draws a seed from torch's generator of x's
    device.  Call sites that share a seed take an ``offset`` each (0 .. 2**63 - 1).

    fp32 and bf16 keep their dtype; others become fp32."""
    _not_traced("dropout")
    return _lib.autograd().dropout(x, float(p), *_seed("dropout", seed), int(offset))


def rmsnorm_residual(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                     dropout: float = 0.0, seed=None, offset: int = 0, checkpoint: Optional[str] = None,
                     format: Optional[str] = None):
    """(y, h): h = residual + dropout(x), y = RMSNorm of h, in one pass.

    x and residual [..., C] may differ in dtype: y has x's, h residual's (fp32 or
    bf16; others become fp32), and the norm takes h as it is stored.  ``dropout``,
    ``seed`` and ``offset`` are :func:`dropout`'s p, seed and offset; the result
    is that of the two calls one after the other, without x's rounding between
    them.

    ``checkpoint`` ("int8" or "e4m3", see :func:`activation_pack`) saves h in 8
    bits for the backward, which is then the gradient at the values that
    checkpoint stands for; without it the backward reads the h that was returned.

    ``format`` ("int8" or "e4m3") returns y in 8 bits, for a product in 8 bits: a
    :class:`PackedActivation` (its ``dtype`` is x's) whose numbers are rounded
    once, from the norm of h with ``eps`` as an fp32 number.  No gradient flows
    through it: such a call raises where one is wanted."""
    _not_traced("rmsnorm_residual")
    code = _checkpoint_code(checkpoint)
    y_code = -1 if format is None else _checkpoint_code(format)
    out = _lib.autograd().rmsnorm_residual(x, residual, weight, float(eps), float(dropout),
                                           *_seed("rmsnorm_residual", seed), int(offset), code, y_code)
    if y_code < 0:
        return out[0], out[1]
    dtype = x.dtype if x.dtype in (torch.float32, torch.bfloat16) else torch.float32
    return PackedActivation(out[0], out[1], format, x.shape[-1], dtype), out[2]


# =============================================================================
# Per-head norm of queries and keys with the rotation of positions (no
# counterpart in the reference)
# =============================================================================

def _sections(fn: str, sections, rotary_dim: int, dealt: bool) -> list:
    """The pairs of each axis of a ``sections`` argument, checked; [] for None."""
    if sections is None:
        if dealt:
            raise ValueError(f"{fn}: sections_dealt needs sections")
        return []
    sizes = list(map(operator.index, sections))
    n, half = len(sizes), rotary_dim // 2
    if not 1 <= n <= 4 or min(sizes) < 0 or sum(sizes) != half:
        raise ValueError(f"{fn}: sections must name 1 to 4 axes and add up to rotary_dim / 2 = {half}, got {sizes}")
    if dealt:
        for a in range(1, n):
            if sizes[a] and a + n * (sizes[a] - 1) >= half:
                raise ValueError(f"{fn}: sections {sizes} cannot be dealt in turn: past the last pair")
    return sizes


def rope_table(length: int, rotary_dim: int, base: float = 10000.0, device=None,
               sections: Optional[Sequence[int]] = None,
               sections_dealt: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, fp32 [length, rotary_dim / 2], of the angles
    position * base**(-2 p / rotary_dim), formed in 64 bits.

    With ``sections`` (and ``sections_dealt``, as :func:`qk_rope` takes them) the
    pairs of each axis have frequencies of their own: the i-th of an axis with s
    of them turns by position * base**(-i / s).  Without, the axes share one
    table: pair p has the frequency above on whichever axis it is."""
    if length < 1 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rope_table: length must be >= 1 and rotary_dim even and >= 2")
    sizes = _sections("rope_table", sections, rotary_dim, sections_dealt)
    if sizes:
        power = [0.0] * (rotary_dim // 2)
        for a, pairs in enumerate(_axis_pairs(sizes, sections_dealt)):
            for i, p in enumerate(pairs):
                power[p] = -i / sizes[a]
        p = torch.tensor(power, device=device, dtype=torch.float64)
    else:
        p = -torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim
    angle = torch.arange(length, device=device, dtype=torch.float64).unsqueeze(1) * base ** p
    return angle.cos().float(), angle.sin().float()


def _axis_pairs(sizes: list, dealt: bool) -> list:
    """The pairs of each axis, in order."""
    n, half = len(sizes), sum(sizes)
    if not dealt:
        ends = [sum(sizes[:a + 1]) for a in range(n)]
        return [list(range(e - s, e)) for e, s in zip(ends, sizes)]
    rest = [list(range(a, half, n))[:sizes[a]] for a in range(n)]
    taken = {p for a in range(1, n) for p in rest[a]}
    return [[p for p in range(half) if p not in taken]] + rest[1:]


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 cos: torch.Tensor, sin: torch.Tensor, positions: Optional[torch.Tensor] = None, eps: float = 1e-5,
                 interleaved: bool = False, checkpoint: Optional[str] = None,
                 sections: Optional[Sequence[int]] = None,
                 sections_dealt: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm of every head of q and k, then the rotation of its token's
    position, in one pass (no counterpart in the reference).

    q [..., heads, D] and k [..., kv_heads, D] are [tokens, heads, D] or
    [batch, seq, heads, D] in one dtype, D <= 1024; they may be strided views
    (of a joint projection's output, say): rows of D channels next to each
    other are read in place.  Each head row becomes y = x / sqrt(mean x^2 +
    eps) * weight, with q_weight and k_weight [D]; then the first R = 2 *
    cos.shape[1] channels rotate by pairs (p, p + R/2), or (2p, 2p + 1) with
    ``interleaved``: (a, b) -> (a c - b s, b c + a s) with c, s column p of cos
    and sin [positions, R/2] (:func:`rope_table`).

    ``positions`` (int64 or int32) is [tokens], or [batch, seq] or [seq];
    without it they count 0, 1, ... along tokens or seq.  A position outside
    the table makes its rows NaN.  The outputs are contiguous, in q's dtype
    (fp32 or bf16; others become fp32); cos and sin get no gradient.

    ``sections`` gives a token positions on several axes, as :func:`qk_rope`
    describes.

    ``checkpoint`` ("int8" or "e4m3", see :func:`activation_pack`) saves q and
    k in 8 bits for the backward, which is then the gradient at the values that
    checkpoint stands for."""
    code = _checkpoint_code(checkpoint)
    _not_traced("qk_norm_rope")
    sizes = _qk_sections("qk_norm_rope", sections, sections_dealt, cos)
    return _lib.autograd().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, float(eps), bool(interleaved),
                                        code, sizes, bool(sections_dealt))


def _qk_sections(fn: str, sections, dealt, cos: torch.Tensor) -> list:
    if sections is None and not dealt:
        return []
    if cos.dim() != 2:
        raise ValueError(f"{fn}: cos and sin must be [positions, rotary_dim / 2]")
    return _sections(fn, sections, 2 * cos.shape[1], dealt)


def qk_rope(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
            positions: Optional[torch.Tensor] = None, interleaved: bool = False,
            sections: Optional[Sequence[int]] = None,
            sections_dealt: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rotation of q's and k's heads by their tokens' positions alone: q, k,
    cos, sin, ``positions`` and ``interleaved`` are :func:`qk_norm_rope`'s.  Its
    backward is the rotation by the negative angle; no rows are saved.

    ``sections`` gives every token positions on 1 to 4 axes (time, height and
    width of video, say): ``positions`` is then [axes, ...], the axes' positions
    as above one after the other, and pair p turns by column p of the table row
    of its own axis's position.  sections[a] pairs belong to axis a, together
    R/2: consecutive ones, axis 0's first; or, with ``sections_dealt``, dealt to
    the axes in turn (pair p to axis p % axes) until an axis has its number, after
    which its turns go to axis 0.  A position outside the table on any axis makes
    its token's rows NaN."""
    _not_traced("qk_rope")
    sizes = _qk_sections("qk_rope", sections, sections_dealt, cos)
    return _lib.autograd().qk_rope(q, k, cos, sin, positions, bool(interleaved), sizes, bool(sections_dealt))
