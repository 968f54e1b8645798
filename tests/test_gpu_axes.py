"""The rotation of queries and keys by positions on several axes, alone and
after the per-head norm, against the 64-bit oracle."""
import pytest
import torch

import mhc_ascend_amd as mhc
from oracle import branch as B
from oracle import rows8
from tests.test_gpu_checkpoint import U, _within
from tests.test_gpu_graph import _capture, _replays
from tests.test_gpu_qk_norm_rope import _check, _inputs
from tests.test_gpu_residual import check_packed

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
E32 = 2.0 ** -24
L = 700  # table rows


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _split(half, axes, seed):
    """Sections of `half` pairs, which can be dealt too."""
    g = _gen(seed)
    rest = [int(torch.randint(0, half // axes + 1, (1,), generator=g)) for _ in range(axes - 1)]
    return [half - sum(rest)] + rest


def _magnitude(v, half, interleaved):
    """|a| + |b| of the pair that each channel is in."""
    m = v.double().abs()
    out = m.clone()
    for p in range(half):
        lo, hi = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
        out[..., lo] = out[..., hi] = m[..., lo] + m[..., hi]
    return out


def _check_rope(got, inputs, c, s, interleaved):
    """Outputs and gradients of the rotation alone: two products and a sum."""
    q, k, _, cots = inputs
    u = U[q.dtype] if q.dtype == torch.bfloat16 else 0.0
    for i, (x, z) in enumerate(zip((q, k), cots)):
        assert got[i].dtype == q.dtype and got[i].is_contiguous() and got[2 + i].dtype == q.dtype
        if x.numel() == 0:
            continue
        for out, v, sn in ((got[i], x, s), (got[2 + i], z, -s)):
            want = B.rotate(v.double(), c, sn, interleaved)
            _within(out, want, 3 * E32 * _magnitude(v, c.shape[-1], interleaved) + u * want.abs() + 1e-30, f"{i}")
            R = 2 * c.shape[-1]
            assert torch.equal(out[..., R:].cpu(), v[..., R:])


def _run(device, inputs, cos, sin, norm, **how):
    q, k, ws, c = inputs
    leaves = [t.to(device).requires_grad_(True) for t in ((q, k, *ws) if norm else (q, k))]
    tables = cos.to(device), sin.to(device)
    out = mhc.qk_norm_rope(*leaves, *tables, **how) if norm else mhc.qk_rope(*leaves, *tables, **how)
    return [*[o.detach() for o in out], *torch.autograd.grad(out, leaves, [t.to(device) for t in c])]


# tokens, heads, kv heads, D, R: whole pieces of 8 and of 4, ragged pieces, passed
# channels, one head, heads of one side only, several tokens a wave, no tokens
SHAPES = [(1, 1, 1, 2, 2), (3, 2, 1, 6, 4), (5, 4, 4, 64, 64), (130, 5, 2, 64, 32), (33, 13, 3, 72, 72),
          (17, 3, 3, 80, 40), (1, 32, 8, 128, 128), (67, 32, 8, 128, 128), (9, 6, 1, 128, 126), (21, 3, 2, 96, 96),
          (7, 2, 2, 112, 56), (11, 2, 1, 192, 64), (40, 4, 2, 256, 256), (3, 2, 2, 257, 256), (4, 1, 2, 512, 512),
          (2, 3, 1, 1000, 8), (2, 1, 1, 1024, 1024), (700, 3, 1, 64, 64), (2, 5, 0, 64, 64), (0, 4, 2, 64, 64),
          (4099, 1, 1, 64, 64), (9001, 4, 1, 72, 36), (5003, 0, 5, 64, 32), (6, 3, 2, 88, 48), (6, 3, 2, 36, 20)]


@pytest.mark.parametrize("T,H,K,D,R", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("axes,dealt", [(0, False), (1, False), (2, True), (3, False), (3, True), (4, False), (4, True)])
def test_rotation_matches_oracle(device, T, H, K, D, R, interleaved, dtype, axes, dealt):
    inputs = _inputs(T, H, K, D, dtype, T + H + D)
    cos, sin = mhc.rope_table(L, R)
    if axes == 0:
        pos = torch.randint(L, (T,), generator=_gen(T))
        c, s = cos[pos], sin[pos]
        how = {}
    else:
        sections = _split(R // 2, axes, D + axes)
        pos = torch.randint(L, (axes, T), generator=_gen(T))
        c, s = B.columns(cos, sin, pos, sections, dealt)
        how = {"sections": sections, "sections_dealt": dealt}
    got = _run(device, inputs, cos, sin, False, positions=pos.to(device), interleaved=interleaved, **how)
    _check_rope(got, inputs, c, s, interleaved)


@pytest.mark.parametrize("T,H,K,D,R", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("axes,dealt,fmt", [(2, False, None), (3, True, "int8"), (4, False, "e4m3"), (4, True, None)])
def test_norm_and_rotation_match_oracle(device, T, H, K, D, R, interleaved, dtype, axes, dealt, fmt):
    inputs = _inputs(T, H, K, D, dtype, T + H + D)
    cos, sin = mhc.rope_table(L, R)
    sections = _split(R // 2, axes, D + axes)
    pos = torch.randint(L, (axes, T), generator=_gen(T))
    c, s = B.columns(cos, sin, pos, sections, dealt)
    got = _run(device, inputs, cos, sin, True, positions=pos.to(device), interleaved=interleaved, sections=sections,
               sections_dealt=dealt, checkpoint=fmt)
    _check([g.cpu() for g in got], inputs, c, s, interleaved, fmt)


@pytest.mark.parametrize("sections", [[16, 24, 24], [8, 56], [64, 0, 0], [0, 0, 64], [4, 60], [3, 30, 31], [8, 8, 8, 40]])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_blocks_that_end_inside_a_piece_and_not(device, sections, norm, interleaved):
    T = 50
    inputs = _inputs(T, 6, 2, 128, torch.bfloat16, 7)
    cos, sin = mhc.rope_table(L, 128)
    pos = torch.randint(L, (len(sections), T), generator=_gen(8))
    c, s = B.columns(cos, sin, pos, sections)
    got = _run(device, inputs, cos, sin, norm, positions=pos.to(device), interleaved=interleaved, sections=sections)
    if norm:
        _check([g.cpu() for g in got], inputs, c, s, interleaved, None)
    else:
        _check_rope(got, inputs, c, s, interleaved)


@pytest.mark.parametrize("D,R,H", [(128, 128, 8), (72, 36, 3), (80, 40, 13), (64, 64, 1)])
@pytest.mark.parametrize("dealt", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_equal_positions_are_one_axis(device, D, R, H, dealt, norm):
    """Text: the same position on every axis gives the one-axis call's bits."""
    T = 300
    inputs = _inputs(T, H, H, D, torch.bfloat16, 9)
    cos, sin = mhc.rope_table(L, R)
    pos = torch.randint(L, (T,), generator=_gen(1)).to(device)
    one = _run(device, inputs, cos, sin, norm, positions=pos)
    many = _run(device, inputs, cos, sin, norm, positions=pos.expand(3, T), sections=_split(R // 2, 3, 2),
                sections_dealt=dealt)
    assert all(torch.equal(a, b) for a, b in zip(one, many))
    single = _run(device, inputs, cos, sin, norm, positions=pos.view(1, T), sections=[R // 2])
    assert all(torch.equal(a, b) for a, b in zip(one, single))
    counted = _run(device, inputs, cos, sin, norm)
    again = _run(device, inputs, cos, sin, norm, positions=torch.arange(T, device=device))
    assert all(torch.equal(a, b) for a, b in zip(counted, again))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("kind", ["all", "seq", "int32", "strided"])
def test_batches_and_positions(device, norm, kind):
    N, S = 3, 10
    q, k, ws, cots = _inputs(N * S, 3, 2, 64, torch.float32, 2)
    cos, sin = mhc.rope_table(L, 64)
    n = S if kind == "seq" else N * S
    p = torch.randint(L, (3, n), generator=_gen(3))
    full = p if n == N * S else p.repeat(1, N)
    c, s = B.columns(cos, sin, full, [12, 10, 10], True)
    pos = p if kind == "seq" else p.view(3, N, S)
    pos = pos.to(device, torch.int32 if kind == "int32" else torch.int64)
    if kind == "strided":
        pos = torch.stack([pos, pos + 1], -1)[..., 0]
    shaped = (q.view(N, S, 3, 64), k.view(N, S, 2, 64), ws, [cots[0].view(N, S, 3, 64), cots[1].view(N, S, 2, 64)])
    got = _run(device, shaped, cos, sin, norm, positions=pos, sections=[12, 10, 10], sections_dealt=True)
    flat = [g.reshape(N * S, -1, 64) if g.dim() == 4 else g for g in got]
    if norm:
        _check([g.cpu() for g in flat], (q, k, ws, cots), c, s, False, None)
    else:
        _check_rope(flat, (q, k, ws, cots), c, s, False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_cotangents(device, dtype):
    """Views of one projection's output, and cotangents that are views."""
    T, H, K, D = 30, 4, 2, 64
    inputs = _inputs(T, H, K, D, dtype, 4)
    q, k, _, cots = inputs
    cos, sin = (t.to(device) for t in mhc.rope_table(L, D))
    pos = torch.randint(L, (2, T), generator=_gen(5)).to(device)
    how = {"positions": pos, "sections": [20, 12]}
    want = _run(device, inputs, cos, sin, False, **how)
    qkv = torch.cat([q, k, k], 1).to(device).requires_grad_(True)
    out = mhc.qk_rope(qkv[:, :H], qkv[:, H:H + K], cos, sin, **how)
    both = torch.cat([c for c in cots], 1).to(device)
    g, = torch.autograd.grad(out, qkv, [both[:, :H], both[:, H:]])
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert torch.equal(g[:, :H], want[2]) and torch.equal(g[:, H:H + K], want[3]) and bool((g[:, H + K:] == 0).all())
    # one head's row for every token, transposed rows, another dtype
    one = q[:1].to(device).requires_grad_(True)
    out = mhc.qk_rope(one.expand(T, H, D), k.to(device), cos, sin, **how)[0]
    full = mhc.qk_rope(q[:1].to(device).expand(T, H, D).contiguous(), k.to(device), cos, sin, **how)[0]
    assert torch.equal(out, full)
    swapped = q.to(device).transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(mhc.qk_rope(swapped, k.to(device), cos, sin, **how)[0], want[0])
    if dtype == torch.float32:
        got = mhc.qk_rope(q.to(device).double(), k.to(device).double(), cos.double(), sin.double(), **how)
        assert got[0].dtype == torch.float32 and torch.equal(got[0], want[0])


def test_the_backward_turns_back(device):
    """The rotation is orthogonal: <R x, z> = <x, R^T z>, and R^T R x = x to roundings."""
    T, D = 200, 128
    q, k, _, cots = [t.to(device) if torch.is_tensor(t) else [u.to(device) for u in t]
                     for t in _inputs(T, 8, 2, D, torch.float32, 6)]
    cos, sin = (t.to(device) for t in mhc.rope_table(L, D))
    how = {"positions": torch.randint(L, (3, T), generator=_gen(5)).to(device), "sections": [24, 20, 20],
           "sections_dealt": True}
    leaves = [q.requires_grad_(True), k.requires_grad_(True)]
    out = mhc.qk_rope(*leaves, cos, sin, **how)
    grads = torch.autograd.grad(out, leaves, cots, retain_graph=True)
    for o, z, x, g in zip([o.detach() for o in out], cots, [t.detach() for t in leaves], grads):
        terms = (x.double() * g.double()).abs().sum()
        assert abs(float((o.double() * z.double()).sum() - (x.double() * g.double()).sum())) <= 8 * E32 * float(terms)
    back = torch.autograd.grad(out, leaves, [o.detach() for o in out])
    for x, b in zip(leaves, back):
        # a rotation's three roundings twice, and c^2 + s^2 of two rounded table entries
        _within(b, x.detach().cpu().double(), 12 * E32 * _magnitude(x.detach().cpu(), D // 2, False), "back")


def test_second_derivatives_of_the_rotation(device):
    """Linear: the gradient of its gradient turns forward again."""
    q, k, _, cots = _inputs(20, 3, 2, 64, torch.float32, 6)
    q, k, z0, z1 = (t.to(device).requires_grad_(True) for t in (q, k, *cots))
    cos, sin = (t.to(device) for t in mhc.rope_table(L, 64))
    how = {"positions": torch.randint(L, (2, 20), generator=_gen(5)).to(device), "sections": [20, 12]}
    dq, dk = torch.autograd.grad(mhc.qk_rope(q, k, cos, sin, **how), [q, k], [z0, z1], create_graph=True)
    u = [torch.randn_like(t).detach() for t in (q, k)]
    got = torch.autograd.grad([dq, dk], [z0, z1], u)
    assert all(torch.equal(a, b) for a, b in zip(got, mhc.qk_rope(*u, cos, sin, **how)))


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,R", [(128, 128), (66, 64)])
@pytest.mark.parametrize("bad", [-1, L, 2 ** 40, -2 ** 40])
def test_a_position_outside_the_table_on_any_axis(device, norm, D, R, bad):
    T = 12
    inputs = _inputs(T, 4, 2, D, torch.float32, 3)
    cos, sin = mhc.rope_table(L, R)
    pos = torch.randint(L, (3, T), generator=_gen(3))
    for axis, t in enumerate((2, 5, 11)):
        pos[axis, t] = bad
    got = _run(device, inputs, cos, sin, norm, positions=pos.to(device), sections=[R // 2 - 20, 20, 0])
    want = torch.zeros(T, dtype=torch.bool)
    want[[2, 5, 11]] = True
    for g in got[:4]:
        rows = g.cpu().isnan()
        assert torch.equal(rows.all(-1).all(-1), want) and torch.equal(rows.any(-1).any(-1), want)


def test_values_that_are_not_finite_stay_in_their_pairs(device):
    q, k = torch.ones(3, 2, 64, device=device), torch.ones(3, 1, 64, device=device)
    q[1, 0, 3] = float("inf")
    q[2, 1, 50] = float("nan")
    cos, sin = (t.to(device) for t in mhc.rope_table(9, 32))
    out = mhc.qk_rope(q, k, cos, sin)[0].cpu().isfinite()
    want = torch.ones(3, 2, 64, dtype=torch.bool)
    want[1, 0, [3, 19]] = False
    want[2, 1, 50] = False
    assert torch.equal(out, want)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dealt", [False, True])
def test_step_replays_in_a_graph(device, norm, dealt):
    T = 40
    inputs = [t.to(device) if torch.is_tensor(t) else [u.to(device) for u in t]
              for t in _inputs(T, 8, 2, 128, torch.bfloat16, 6)]
    pos = torch.randint(100, (3, T), generator=_gen(5)).to(device)
    cos, sin = (t.to(device) for t in mhc.rope_table(L, 128))

    def step():
        return _run(device, [inputs[0].detach(), inputs[1].detach(), [w.detach() for w in inputs[2]], inputs[3]], cos,
                    sin, norm, positions=pos, sections=[24, 20, 20], sections_dealt=dealt)

    graph, outs = _capture(step)
    g = _gen(10)
    feeds = [lambda: inputs[0].copy_(torch.randn(inputs[0].shape, generator=g)), lambda: pos.add_(300),
             lambda: inputs[3][1].copy_(torch.randn(inputs[3][1].shape, generator=g)), lambda: pos[1].add_(290)]
    _replays(graph, outs, step, feeds)


@pytest.mark.parametrize("D", [128, 66])
def test_offsets_past_32_bits(device, D):
    """More than 2^32 values of q: the last tokens against a call on them."""
    H, K = 64, 1
    T = (1 << 32) // (H * D) + 70
    q = torch.empty(T, H, D, dtype=torch.bfloat16, device=device).fill_(0.5)
    k = torch.empty(T, K, D, dtype=torch.bfloat16, device=device).fill_(0.5)
    q[-64:] = torch.randn(64, H, D, device=device).bfloat16()
    cos, sin = (t.to(device) for t in mhc.rope_table(1024, 64))
    pos = torch.arange(T, device=device) % torch.tensor([[1024], [1000]], device=device)
    outs = []
    for a, b, p in ((q, k, pos), (q[-64:].clone(), k[-64:].clone(), pos[:, -64:])):
        with torch.no_grad():
            out = mhc.qk_rope(a, b, cos, sin, p, sections=[20, 12], sections_dealt=True)
        outs.append([t[-64:].clone() for t in out])
        del out
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_long_tables_past_32_bits(device):
    """A table of more than 2^31 entries: positions at its end."""
    half, rows = 64, (1 << 31) // 64 + 16
    cos, sin = torch.zeros(rows, half, device=device), torch.ones(rows, half, device=device)
    ends = torch.rand(16, half, device=device)
    cos[-16:], sin[-16:] = ends, 1 - ends
    q = torch.randn(8, 4, 128, device=device)
    pos = torch.stack([torch.arange(8) + rows - 16, torch.arange(8) + rows - 8]).to(device)
    small = (q, q[:, :1], ends, 1 - ends)
    for norm in (False, True):
        w = [torch.rand(128, device=device)] * 2 if norm else []
        call = mhc.qk_norm_rope if norm else mhc.qk_rope
        for dealt in (False, True):
            how = {"sections": [32, 32], "sections_dealt": dealt}
            a = call(q, q[:, :1], *w, cos, sin, pos, **how)
            b = call(*small[:2], *w, *small[2:], pos - (rows - 16), **how)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("T,D", [((1 << 24) + 64, 6), ((1 << 26) + 64, 8)])
def test_more_tokens_than_a_launch_takes(device, T, D):
    P = 64
    q = torch.randn(P, 1, D, device=device).bfloat16().repeat(T // P, 1, 1).view(T // P, P, 1, D)
    q[-1] = q[-1] * 3 + 1
    k = q.new_empty(T // P, P, 0, D)
    cos, sin = mhc.rope_table(P, D, device=device)
    pos = torch.stack([torch.arange(P), P - 1 - torch.arange(P)]).to(device)
    how = {"sections": [D // 2 - 1, 1]}
    with torch.no_grad():
        out = mhc.qk_rope(q, k, cos, sin, pos, **how)[0]
        for at in (0, (1 << 23) // P, 4 * (1 << 23) // P, T // P - 1):
            if at >= T // P:
                continue
            assert torch.equal(out[at:at + 1], mhc.qk_rope(q[at:at + 1], k[at:at + 1], cos, sin, pos, **how)[0])
        assert torch.equal(out[:-1], out[:1].expand_as(out[:-1]))


@pytest.mark.parametrize("D,R", [(128, 128), (256, 128), (128, 64), (96, 96), (192, 192)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads", [(13, 4), (0, 16), (17, 0)])
def test_many_rows_are_the_rows_of_smaller_calls(device, D, R, dtype, interleaved, heads):
    """Rows of more than 128 MiB, which some head sizes stream, bit for bit."""
    H, K = heads
    T = (1 << 27) // ((H + K) * D * torch.tensor([], dtype=dtype).element_size()) + 61
    q = torch.randn(T, H, D, device=device).to(dtype)
    k = torch.randn(T, K, D, device=device).to(dtype)
    cos, sin = mhc.rope_table(512, R, device=device)
    pos = torch.randint(512, (3, T), device=device)
    n = R // 2
    for dealt in (False, True):
        how = {"interleaved": interleaved, "sections": [n - 2 * (n // 4), n // 4, n // 4], "sections_dealt": dealt}
        out = mhc.qk_rope(q, k, cos, sin, pos, **how)
        for at in (slice(0, T // 3), slice(T // 3, T // 3 + 300), slice(T // 3 + 300, T)):
            want = mhc.qk_rope(q[at], k[at], cos, sin, pos[:, at], **how)
            assert all(torch.equal(a[at], b) for a, b in zip(out, want))


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_an_error(device, grad):
    q, k, _, _ = _inputs(5, 2, 1, 64, torch.float32, 3)
    cos, sin = mhc.rope_table(5, 64)
    args = [t.to(device) for t in (q, k, cos, sin)]
    fwd = torch.autograd.forward_ad
    for i in range(4):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            call = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
            with pytest.raises(RuntimeError, match="jvp is not implemented" if i < 2 else "no gradient"):
                mhc.qk_rope(*call)


def test_refusals(device):
    q, k = torch.zeros(4, 2, 64, device=device), torch.zeros(4, 1, 64, device=device)
    cos, sin = (t.to(device) for t in mhc.rope_table(8, 64))
    pos = torch.zeros(2, 4, dtype=torch.int64, device=device)
    for call, text in [
            (lambda: mhc.qk_rope(q, k.bfloat16(), cos, sin), "one floating dtype"),
            (lambda: mhc.qk_rope(q, k, cos, sin[:4]), "cos and sin"),
            (lambda: mhc.qk_rope(q, k, cos, sin, sections=[16, 16]), "need positions"),
            (lambda: mhc.qk_rope(q, k, cos, sin, pos[:1], sections=[16, 16]), "one row an axis"),
            (lambda: mhc.qk_rope(q, k, cos, sin, pos[0], sections=[16, 16]), "one row an axis"),
            (lambda: mhc.qk_rope(q, k, cos, sin, pos[:, :3], sections=[16, 16]), "positions must be"),
            (lambda: mhc.qk_rope(q, k, cos, sin, pos), "positions must be"),
            (lambda: mhc.qk_rope(q, k, cos, sin, pos.float(), sections=[16, 16]), "int64 or int32"),
            (lambda: mhc.qk_rope(q, k, cos, sin, pos.cpu(), sections=[16, 16]), "HIP device"),
            (lambda: mhc.qk_rope(q, k, cos[:0], sin[:0]), "rows")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    wide = torch.zeros(1, 1, 1026, device=device)
    with pytest.raises(RuntimeError, match="head_dim"):
        mhc.qk_rope(wide, wide, cos, sin)


def test_a_branch_as_a_model_runs_it(device):
    """Norm, q and k turned on three axes, attention, dropout, the residual's sum
    and the next norm, then the residual wrapper with its dropout: one training
    step against the same step in 64 bits; and the serving form of the norms."""
    torch.manual_seed(4)
    T, C, H, D, p, seed = 24, 64, 2, 32, 0.25, 77
    wrap = mhc.MHCResidualWrapper(C, 4, use_dynamic_h=False, dropout=p).to(device)
    x, b = torch.randn(T, C), torch.randn(T, C)
    n1, n2 = 1 + 0.1 * torch.randn(C), 1 + 0.1 * torch.randn(C)
    ws = [0.2 * torch.randn(C, H * D) for _ in range(3)]
    w2 = 0.2 * torch.randn(C, C)
    hw = [1 + 0.1 * torch.randn(D) for _ in range(2)]
    sections = [6, 5, 5]
    cos, sin = mhc.rope_table(T, D, sections=sections)
    pos = torch.stack([torch.arange(T), torch.arange(T) // 4, torch.arange(T) % 4])
    cots = [torch.randn(T, C), torch.randn(T, C)]

    def block(first, turn, second, out, x, b, n1, n2, ws, w2, hw):
        y, h = first(b, x, n1)
        q, k, v = ((y @ w).view(T, H, D) for w in ws)
        q, k = turn(q, k, *hw)
        a = torch.softmax(torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) / D ** 0.5, -1)
        y = torch.matmul(a, v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(T, C)
        y, h = second(y, h, n2)
        return out(h, y @ w2), y

    leaves = [t.to(device).requires_grad_(True) for t in (x, b, n1, n2, *ws, w2, *hw)]
    args = lambda v: (*v[:4], v[4:7], v[7], v[8:])  # noqa: E731
    how = {"positions": pos.to(device), "sections": sections}
    torch.manual_seed(9)
    drawn = torch.empty(1, dtype=torch.int64, device=device).random_()  # what the wrapper's dropout draws
    torch.manual_seed(9)
    got = block(lambda b, r, w: mhc.rmsnorm_residual(b, r, w),
                lambda q, k, u, v: mhc.qk_norm_rope(q, k, u, v, cos.to(device), sin.to(device), **how),
                lambda y, h, w: mhc.rmsnorm_residual(y, h, w, dropout=p, seed=seed, offset=1),
                wrap, *args(leaves))
    grads = torch.autograd.grad(got, leaves, [c.to(device) for c in cots])

    from oracle import reference as R
    m = wrap.mhc
    pre, post = torch.sigmoid(m.H_pre.detach().cpu().double()), 2 * torch.sigmoid(m.H_post.detach().cpu().double())
    mix = R.sinkhorn_knopp(torch.exp(m.H_res.detach().cpu().double()), 20, 1e-8)
    rw = m.rmsnorm_weight.detach().cpu().double()
    f1, f2 = B.factors((T, C), p, seed, 1), B.factors((T, C), p, int(drawn), 0)
    c, s = B.columns(cos, sin, pos, sections)

    def out64(r, y):
        return R._layer_core(torch.stack([r, y * f2, r * 0.1, r * 0.01], 1), rw, pre, post, mix, 1e-5).mean(1)

    ref_leaves = [t.double().requires_grad_(True) for t in (x, b, n1, n2, *ws, w2, *hw)]
    ref = block(lambda b, r, w: (B.rmsnorm(r + b, w), r + b),
                lambda q, k, u, v: (rows8.qk_norm_rope(q, u, c, s), rows8.qk_norm_rope(k, v, c, s)),
                lambda y, h, w: (B.rmsnorm(h + y * f1, w), h + y * f1), out64, *args(ref_leaves))
    want = torch.autograd.grad(ref, ref_leaves, [t.double() for t in cots])
    # fp32 throughout: a few hundred roundings of 2^-24 (6e-8) on sums that do not cancel far
    for a, e in zip((*got, *grads), (*ref, *want)):
        assert float((a.detach().cpu().double() - e.detach()).norm() / e.detach().norm()) <= 1e-5
    # serving: the same norm's output in 8 bits
    with torch.no_grad():
        packed, h = mhc.rmsnorm_residual(leaves[1], leaves[0], leaves[2], format="int8")
        assert torch.equal(h, mhc.rmsnorm_residual(leaves[1], leaves[0], leaves[2])[1])
    check_packed(packed, h, leaves[2], "int8")
