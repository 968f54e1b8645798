"""Dropout and the RMSNorm of a residual's sum without a GPU: the generator's
published answers, and the refusals of the public functions and of the C entries,
before any launch."""
import copy
import pickle

import pytest
import torch

import mhc_ascend_amd as mhc
from mhc_ascend_amd import _lib
from oracle import branch as B


def test_generator_gives_its_published_answers():
    """Known answers of Philox4x32-10: counter and key of zeros, of ones, and of pi's digits."""
    ones = 2 ** 32 - 1
    for ctr, key, want in [
            ([0] * 4, [0, 0], [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
            ([ones] * 4, [ones] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
            ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0],
             [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])]:
        assert B.philox(ctr, key) == want


def test_numbers_are_the_generators_words():
    n = B.numbers(3, 11, seed=2 ** 40 + 5, offset=2 ** 33 + 1, first_row=2 ** 32)
    for r in range(3):
        for c in range(11):
            block = (2 ** 32 + r) * 2 + c // 8
            w = B.philox([block & B.LOW, block >> 32, 1, 2], [5, 2 ** 8])[c % 8 // 2]
            assert int(n[r, c]) == (w >> 16 if c % 2 else w & 0xFFFF)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 32), torch.ones(32)
    for call in (lambda: mhc.dropout(x, 0.5), lambda: mhc.rmsnorm_residual(x, x, w)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_arguments_are_refused():
    x, w = torch.zeros(4, 32), torch.ones(32)
    for bad in (2 ** 64, -2 ** 63 - 1):
        with pytest.raises(ValueError, match="64 bits"):
            mhc.dropout(x, 0.5, seed=bad)
    with pytest.raises(TypeError):
        mhc.dropout(x, 0.5, seed=1.5)
    for bad in ("fp8", "", 0):
        with pytest.raises(ValueError, match="Unknown checkpoint format"):
            mhc.rmsnorm_residual(x, x, w, format=bad)
        with pytest.raises(ValueError, match="Unknown checkpoint format"):
            mhc.rmsnorm_residual(x, x, w, checkpoint=bad)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="dropout"):
            mhc.MHCResidualWrapper(32, dropout=bad)


def test_calls_are_not_traced():
    x = torch.zeros(4, 32)
    for call in (lambda t: mhc.dropout(t, 0.5, seed=1), lambda t: mhc.rmsnorm_residual(t, t, torch.ones(32))[0]):
        with pytest.raises(RuntimeError, match="not recorded"):
            torch.jit.trace(call, (x,))


def test_wrapper_keeps_its_dropout():
    m = mhc.MHCResidualWrapper(32, dropout=0.25, use_dynamic_h=False)
    assert copy.deepcopy(m).dropout == pickle.loads(pickle.dumps(m)).dropout == 0.25
    assert "dropout=0.25" in repr(m) and "dropout" not in repr(mhc.MHCResidualWrapper(32, use_dynamic_h=False))
    old = mhc.MHCResidualWrapper(32, use_dynamic_h=False)
    del old.__dict__["dropout"]  # as a module pickled before it existed
    assert old.dropout == 0.0
    assert mhc.replace_residual_with_mhc(32, dropout=0.5).dropout == 0.5


def test_c_entries_refuse_on_the_host():
    lib = _lib.load()
    drop = lambda x=64, dt=0, out=64, t=5, seed=None, rows=4, hidden=32: lib.mhc_dropout(  # noqa: E731
        x, dt, out, t, 1, seed, 0, rows, hidden, None)
    for rc, kw in [(-1, {"x": None}), (-1, {"out": None}), (-1, {"dt": 2}), (-1, {"t": -1}), (-1, {"t": 65537}),
                   (-1, {"rows": -1}), (-1, {"hidden": 0}), (-2, {"hidden": 2 ** 30 + 1}), (-1, {"seed": 4})]:
        assert drop(**kw) == rc, kw
        assert lib.mhc_last_error().startswith(b"dropout")

    def fwd(x=64, xd=0, res=64, rd=0, w=64, wd=0, h=64, y=64, yf=-1, yq=None, ys=None, hf=-1, hq=None, hs=None, t=0,
            seed=None, rows=4, hidden=32):
        return lib.mhc_rmsnorm_residual_fwd(x, xd, res, rd, w, wd, h, y, yf, yq, ys, hf, hq, hs, t, 1, seed, 0, rows,
                                            hidden, 1e-5, None)

    for rc, kw in [(-1, {"x": None}), (-1, {"res": None}), (-1, {"w": None}), (-1, {"h": None}), (-1, {"y": None}),
                   (-1, {"xd": 2}), (-1, {"rd": 2}), (-1, {"wd": 2}), (-1, {"yf": 2, "yq": 64, "ys": 64}),
                   (-1, {"yf": 0}), (-1, {"yf": 0, "yq": 8, "ys": 64}), (-1, {"hf": 1, "hq": 64}), (-1, {"hf": -2}),
                   (-1, {"t": 70000}), (-2, {"hidden": 2 ** 30 + 1}), (-2, {"rows": 2 ** 31}), (-1, {"rows": -1}),
                   (-1, {"hidden": 0}), (-1, {"seed": 12})]:
        assert fwd(**kw) == rc, kw
        assert lib.mhc_last_error().startswith(b"rmsnorm_residual_fwd")

    def bwd(gy=64, xd=0, gh=None, rd=0, h=64, hf=-1, hq=None, hs=None, w=64, wd=0, gx=64, gr=64, gw=64, t=0, ws=64,
            wsb=0, rows=4, hidden=32):
        return lib.mhc_rmsnorm_residual_bwd(gy, xd, gh, rd, h, hf, hq, hs, w, wd, gx, gr, gw, t, 1, None, 0, ws, wsb,
                                            rows, hidden, 1e-5, None)

    for rc, kw in [(-1, {"gy": None}), (-1, {"h": None}), (-1, {"w": None}), (-1, {"hf": 0}), (-3, {}),
                   (-3, {"ws": None}), (-1, {"xd": 3}), (-1, {"t": -1})]:
        assert bwd(**kw) == rc, kw
        assert lib.mhc_last_error().startswith(b"rmsnorm_residual_bwd")
    size = lib.mhc_rmsnorm_residual_bwd_workspace_size
    assert size(-1, 32, 0, 0) == size(4, 0, 0, 0) == size(4, 32, 2, 0) == size(4, 2 ** 30 + 1, 0, 0) == 0
