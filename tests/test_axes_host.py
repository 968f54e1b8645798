"""Positions on several axes without a GPU: tables, sections, and the refusals of
the public functions and the C entries before any launch."""
import ctypes

import pytest
import torch

import mhc_ascend_amd as mhc
from mhc_ascend_amd import _lib, ops
from oracle import branch as B


@pytest.mark.parametrize("sections,dealt", [([16, 24, 24], False), ([24, 20, 20], True), ([3, 1], True), ([1, 0, 2, 1], False),
                                            ([5], False), ([5], True), ([0, 4], False), ([22, 21, 21], True)])
def test_pairs_of_an_axis(sections, dealt):
    axes = B.pair_axes(sections, dealt)
    got = ops._axis_pairs(sections, dealt)
    assert [[p for p, a in enumerate(axes) if a == i] for i in range(len(sections))] == got
    assert [len(g) for g in got] == sections


def test_rope_table_of_sections():
    """The i-th pair of an axis with s of them turns by base ** (-i / s)."""
    for sections, dealt in (([4, 2, 2], False), ([4, 2, 2], True)):
        cos, sin = mhc.rope_table(50, 16, base=300.0, sections=sections, sections_dealt=dealt)
        for pairs, s in zip(ops._axis_pairs(sections, dealt), sections):
            for i, p in enumerate(pairs):
                angle = torch.arange(50, dtype=torch.float64) * 300.0 ** (-i / s)
                assert float((cos[:, p].double() - angle.cos()).abs().max()) <= 2.0 ** -24
                assert float((sin[:, p].double() - angle.sin()).abs().max()) <= 2.0 ** -24
    one, two = mhc.rope_table(50, 16), mhc.rope_table(50, 16, sections=[8])
    assert torch.allclose(one[0], two[0], rtol=0, atol=2.0 ** -23)


@pytest.mark.parametrize("sections,dealt", [([], False), ([8, 8], False), ([20, 12, 0, 0, 0], False), ([40, -8], False),
                                            ([15, 17], True), ([10, 11, 11], True), (None, True)])
def test_sections_are_refused(sections, dealt):
    q, w, t = torch.zeros(4, 2, 64), torch.ones(64), torch.ones(9, 32)
    for call in (lambda: mhc.qk_rope(q, q, t, t, sections=sections, sections_dealt=dealt),
                 lambda: mhc.qk_norm_rope(q, q, w, w, t, t, sections=sections, sections_dealt=dealt),
                 lambda: mhc.rope_table(9, 64, sections=sections, sections_dealt=dealt)):
        with pytest.raises(ValueError, match="sections"):
            call()


def test_calls_are_refused_on_the_cpu_and_traced():
    q, t = torch.zeros(4, 2, 64), torch.ones(9, 32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        mhc.qk_rope(q, q, t, t)
    with pytest.raises(RuntimeError, match="not recorded"):
        torch.jit.trace(lambda a: mhc.qk_rope(a, a, t, t)[0], (q,))
    with pytest.raises(ValueError, match="cos and sin"):
        mhc.qk_rope(q, q, t[0], t[0], sections=[16, 16])
    with pytest.raises(TypeError):
        mhc.qk_rope(q, q, t, t, sections=[16.5, 15.5])


def test_c_entries_refuse_on_the_host():
    lib = _lib.load()
    sec = lambda *n: (ctypes.c_int32 * len(n))(*n)  # noqa: E731

    def fwd(axes=2, sections=sec(16, 16), dealt=0, pos=64, nbytes=8, D=64, R=64, q=64, out=64, w=64):
        return lib.mhc_qk_norm_rope_axes_fwd(q, 128, 64, 64, 64, 64, 0, w, 64, 0, 64, 64, 9, pos, nbytes, 4, axes,
                                             sections, dealt, out, 64, -1, None, None, None, None, 4, 2, 1, D, R, 0,
                                             1e-5, None)

    def bwd(axes=2, sections=sec(16, 16), dealt=0, gq=64, ws=None):
        return lib.mhc_qk_norm_rope_axes_bwd(gq, 128, 64, 64, 64, 64, 64, 128, 64, 64, 64, 64, 0, -1, None, None, None,
                                             None, 64, 64, 0, 64, 64, 9, 64, 8, 4, axes, sections, dealt, 64, 64, 64,
                                             ws, 0, 4, 2, 1, 64, 64, 0, 1e-5, None)

    def rope(axes=2, sections=sec(16, 16), dealt=0, pos=64, nbytes=8, D=64, R=64, q=64, out=64, dt=0, cos=64):
        return lib.mhc_qk_rope(q, 128, 64, 64, 64, 64, dt, cos, 64, 9, pos, nbytes, 4, axes, sections, dealt, out, 64,
                               4, 2, 1, D, R, 0, 0, None)

    bad = [{"axes": 5, "sections": sec(16, 16, 0, 0, 0)}, {"axes": -1}, {"sections": None}, {"sections": sec(16, 15)},
           {"sections": sec(33, -1)}, {"sections": sec(15, 17), "dealt": 1}]
    for f, more in ((fwd, [{"axes": 0}, {"pos": None, "nbytes": 0}, {"pos": None}, {"q": None}, {"out": None},
                           {"w": None}, {"R": 66}, {"D": 1}]),
                    (bwd, [{"axes": 0}, {"gq": None}]),
                    (rope, [{"pos": None, "nbytes": 0}, {"pos": None}, {"q": None}, {"out": None}, {"R": 66},
                            {"dt": 2}, {"cos": None}, {"nbytes": 2}])):
        for kw in bad + more:
            assert f(**kw) == -1, (f, kw)
            assert lib.mhc_last_error().startswith(b"qk_")
    assert bwd() == -3
    assert rope(D=1026, R=64, sections=sec(16, 16)) == -2
