"""8-bit checkpoints and qk_norm_rope without a GPU: the oracle's format, the
refusals of the public functions and of the C entries, before any launch."""
import copy
import pickle

import pytest
import torch

import mhc_ascend_amd as mhc
from mhc_ascend_amd import _lib
from oracle import rows8

FORMATS = ["int8", "e4m3"]


@pytest.mark.parametrize("fmt", FORMATS)
def test_oracle_format_bounds(fmt):
    """Half a step of the format, idempotent, exact in bf16."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 100, generator=g) * torch.exp2(torch.randint(-40, 40, (50, 1), generator=g).float())
    h = rows8.held(x, fmt)
    e = rows8.exponents(x, fmt).repeat_interleave(32, -1)[..., :100]
    err = (h - x.double()).abs()
    if fmt == "int8":
        assert bool((err <= torch.exp2(e - 1)).all())
    else:
        assert bool((err <= torch.maximum(x.double().abs() * 2.0 ** -4, torch.exp2(e - 10))).all())
    assert torch.equal(rows8.held(h.float(), fmt), h)
    assert torch.equal(h.to(torch.bfloat16).double(), h)
    # e is least: one less does not hold the block
    a = rows8._split(x).abs().amax(-1)
    ee = rows8.exponents(x, fmt)
    assert bool((a <= rows8.MAX[fmt] * torch.exp2(ee)).all())
    assert bool((a > rows8.MAX[fmt] * torch.exp2(ee - 1)).all())


@pytest.mark.parametrize("bad", ["fp8", "INT8", "", 0, 1.5, ["int8"]])
def test_unknown_formats_are_refused(bad):
    x = torch.zeros(2, 4, 32)
    for call in (lambda: mhc.MHCLayer(32, checkpoint=bad),
                 lambda: mhc.rmsnorm(x[0], torch.ones(32), checkpoint=bad),
                 lambda: mhc.stream_aggregate(x, torch.zeros(2, 4), checkpoint=bad),
                 lambda: mhc.activation_pack(x, bad),
                 lambda: mhc.qk_norm_rope(x, x, torch.ones(32), torch.ones(32), torch.ones(9, 16), torch.ones(9, 16),
                                          checkpoint=bad)):
        with pytest.raises(ValueError, match="Unknown checkpoint format"):
            call()


def test_packing_needs_a_format():
    with pytest.raises(ValueError, match="int8"):
        mhc.activation_pack(torch.zeros(2, 32), None)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 32, requires_grad=True)
    w, t = torch.ones(32), torch.ones(9, 16)
    for call in (lambda: mhc.activation_pack(x), lambda: mhc.rmsnorm(x[0], w, checkpoint="int8"),
                 lambda: mhc.qk_norm_rope(x, x, w, w, t, t),
                 lambda: mhc.mhc_layer_static(x, w, torch.zeros(4), torch.zeros(4), torch.zeros(4, 4),
                                              checkpoint="e4m3")):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_qk_shapes_are_refused():
    w, t = torch.ones(32), torch.ones(9, 16)
    q = torch.zeros(6, 4, 32)
    cases = [(q[0], q[0], None), (q, torch.zeros(5, 2, 32), None), (q, torch.zeros(6, 2, 16), None),
             (q, q.view(2, 3, 4, 32), None), (q, q, torch.zeros(5, dtype=torch.int64)),
             (q.view(2, 3, 4, 32), q.view(2, 3, 4, 32), torch.zeros(3, 2, dtype=torch.int64))]
    for a, b, p in cases:
        with pytest.raises(RuntimeError, match="qk_norm_rope"):
            mhc.qk_norm_rope(a, b, w, w, t, t, p)


def test_rope_table():
    cos, sin = mhc.rope_table(70000, 8, base=500.0)
    assert cos.shape == sin.shape == (70000, 4) and cos.dtype == torch.float32
    angle = 69999.0 * 500.0 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)
    # one rounding of a 64-bit value (which is itself off by 2^-53 of an angle up to 2^17)
    assert float((cos[-1].double() - angle.cos()).abs().max()) <= 2.0 ** -25 + 2.0 ** -34
    assert float((sin[-1].double() - angle.sin()).abs().max()) <= 2.0 ** -25 + 2.0 ** -34
    for bad in ((0, 8), (4, 0), (4, 7)):
        with pytest.raises(ValueError):
            mhc.rope_table(*bad)


def test_modules_carry_the_option():
    layer = mhc.MHCLayer(32, 2, use_dynamic_h=False, checkpoint="e4m3")
    assert layer.checkpoint == "e4m3" and mhc.MHCLayer(32).checkpoint is None
    assert copy.deepcopy(layer).checkpoint == "e4m3"
    assert mhc.create_mhc_layer(32, checkpoint="int8").checkpoint == "int8"
    assert mhc.MHCResidualWrapper(32, checkpoint="int8").mhc.checkpoint == "int8"
    assert set(layer.state_dict()) == set(mhc.MHCLayer(32, 2, use_dynamic_h=False).state_dict())
    old = pickle.loads(pickle.dumps(mhc.MHCLayer(32, 2, use_dynamic_h=False)))
    del old.__dict__["checkpoint"]  # a module saved before the option existed
    assert old.checkpoint is None


def test_sizes_on_host():
    lib = _lib.load()
    assert lib.mhc_checkpoint_values_size(3, 100) == 3 * 112 and lib.mhc_checkpoint_scales_size(3, 100) == 3 * 4
    assert lib.mhc_checkpoint_values_size(1 << 33, 4096) == (1 << 33) * 4096
    assert lib.mhc_checkpoint_values_size(-1, 4) == 0 and lib.mhc_checkpoint_scales_size(1, 0) == 0
    assert lib.mhc_rmsnorm_checkpoint_bwd_workspace_size(4, 16385, 0, 0) == 0
    assert lib.mhc_qk_norm_rope_bwd_workspace_size(4, 1, 1, 1025, 64, 0) == 0


def test_checkpoint_entries_reject_bad_arguments_on_host():
    lib = _lib.load()
    pack, unpack = lib.mhc_checkpoint_pack, lib.mhc_checkpoint_unpack
    assert pack(16, 0, 2, 16, 16, 1, 32, None) == -1 and b"format" in lib.mhc_last_error()
    assert pack(16, 0, -1, 16, 16, 1, 32, None) == -1
    assert pack(16, 3, 0, 16, 16, 1, 32, None) == -1 and b"dtype" in lib.mhc_last_error()
    assert pack(16, 0, 0, 16, 16, -1, 32, None) == -1
    assert pack(16, 0, 0, 16, 16, 1, 0, None) == -1
    assert pack(None, 0, 0, 16, 16, 1, 32, None) == -1 and b"null" in lib.mhc_last_error()
    assert pack(16, 0, 0, 8, 16, 1, 32, None) == -1 and b"aligned" in lib.mhc_last_error()
    assert unpack(8, 16, 0, 16, 0, 1, 32, None) == -1 and b"aligned" in lib.mhc_last_error()
    assert unpack(16, None, 0, 16, 0, 1, 32, None) == -1
    fwd, bwd = lib.mhc_rmsnorm_checkpoint_fwd, lib.mhc_rmsnorm_checkpoint_bwd
    assert fwd(16, 0, 16, 16, 0, 16, 16, 1, 16385, 1e-5, None) == -2 and b"too large" in lib.mhc_last_error()
    assert fwd(16, 0, 16, 16, 0, 16, 16, 1 << 31, 32, 1e-5, None) == -2
    assert fwd(16, 0, 16, 16, 7, 16, 16, 1, 32, 1e-5, None) == -1
    assert bwd(16, 0, 16, 16, 0, 16, 16, 16, None, 0, 4, 64, 1e-5, None) == -3
    assert bwd(16, 0, 16, 16, 0, 16, 16, None, 16, 1 << 30, 4, 64, 1e-5, None) == -1
    sf = lib.mhc_layer_static_checkpoint_fwd
    assert sf(16, 0, 16, 1, 16, 16, 16, 16, 16, 0, 16, None, 4, 4, 64, 20, 1e-8, 1e-5, None) == -1
    assert sf(16, 0, 16, 1, 16, 16, 16, 16, 16, 0, 16, 16, 4, 65, 64, 20, 1e-8, 1e-5, None) == -2
    sb = lib.mhc_layer_static_checkpoint_bwd
    assert sb(16, 16, 16, 0, 0, 1, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 8, 4, 4, 64, 20, 1e-8, 1e-5, None) == -3
    assert sb(16, 16, 16, 5, 0, 1, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 8, 4, 4, 64, 20, 1e-8, 1e-5, None) == -1


def _qk_fwd(lib, **kw):
    a = dict(q=16, qt=128, qh=64, k=16, kt=64, kh=64, dt=0, wq=16, wk=16, wdt=0, cos=16, sin=16, rows=8, pos=None, pb=0,
             period=4, qo=16, ko=16, fmt=-1, qv=None, qs=None, kv=None, ks=None, T=4, H=2, K=1, D=64, R=64, il=0,
             eps=1e-5, st=None)
    a.update(kw)
    return lib.mhc_qk_norm_rope_fwd(*a.values())


@pytest.mark.parametrize("kw", [dict(T=-1), dict(D=1, R=2), dict(R=66), dict(R=3), dict(R=0), dict(dt=2), dict(wdt=5),
                                dict(fmt=2), dict(fmt=-2), dict(pb=3), dict(pb=8), dict(pos=16), dict(period=0),
                                dict(rows=0), dict(wk=None), dict(cos=None), dict(qo=None), dict(q=None),
                                dict(fmt=0), dict(fmt=0, qv=8, qs=8, kv=16, ks=16), dict(H=-1), dict(H=262140)])
def test_qk_entry_rejects_bad_arguments_on_host(kw):
    lib = _lib.load()
    assert _qk_fwd(lib, **kw) == -1 and b"qk_norm_rope_fwd" in lib.mhc_last_error()


def test_qk_entry_rejects_wide_heads_and_small_workspaces_on_host():
    lib = _lib.load()
    assert _qk_fwd(lib, D=1026, R=64) == -2
    bwd = [16, 128, 64, 16, 64, 64, 16, 128, 64, 16, 64, 64, 0, -1, None, None, None, None, 16, 16, 0, 16, 16, 8, None, 0,
           4, 16, 16, 16, 16, 8, 4, 2, 1, 64, 64, 0, 1e-5, None]
    assert lib.mhc_qk_norm_rope_bwd(*bwd) == -3
    bwd[29] = None
    assert lib.mhc_qk_norm_rope_bwd(*bwd) == -1


@pytest.mark.filterwarnings("ignore")
def test_layers_and_wrapper_refuse_to_be_traced_with_a_checkpoint():
    """torch.jit.trace would keep a C++ node's result as a constant."""
    x = torch.zeros(2, 4, 32)
    for dynamic in (False, True):
        layer = mhc.MHCLayer(32, 4, use_dynamic_h=dynamic, checkpoint="int8")
        wrap = mhc.MHCResidualWrapper(32, 4, use_dynamic_h=dynamic)
        wrap.mhc.checkpoint = "e4m3"
        for call in (layer, lambda a: wrap(a[:, 0], a[:, 1]),
                     lambda a: mhc.ops.mhc_residual_wrapper(a[:, 0], a[:, 1], layer)):
            with pytest.raises(RuntimeError, match="not recorded by torch.jit.trace"):
                torch.jit.trace(call, (x,), check_trace=False)
