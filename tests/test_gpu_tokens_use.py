"""-m gpu: the operators on view tokens as programs use them: layouts, masks of any type, streams and graphs, long caches, and all together behind
the regulariser's draws.  Results that only differ in how a tensor lies in memory are equal bit by bit; the rest is measured against 64 bits."""
import math

import pytest
import torch

from mvtn_amd import tokens
from mvtn_amd.regularize import draw_regularization

from gpu_helpers import _dev
from test_gpu_tokens import U32, _attend64, _gen, _norm64, _randn, _rotary64, _tiny, _u
from test_gpu_tokens import test_attention_matches_the_definition as _matches_the_definition

pytestmark = pytest.mark.gpu


def _all(q, k, v, do, keep=None, **kw):
    """(out, dq, dk, dv); the gradients as the leaves' own."""
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = tokens.attend_tokens(*leaves, keep=keep, **kw)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, do))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Lq,Lk,H,E,D,groups,dropped", [
    (2, 100, 130, 4, 2, 64, 0, 0.0),             # shared heads, each with a ragged last tile of queries
    (2, 64, 192, 6, 2, 128, 4, 0.5),             # ... with whole ones
    (1, 63, 65, 4, 1, 64, 0, 0.0),               # ... sharing tiles
    (1, 10, 70, 8, 2, 128, 7, 0.3),
    (1, 257, 64, 2, 2, 32, 0, 0.0),              # rows for one column more than a wide workgroup holds
    (1, 128, 63, 1, 1, 64, 0, 0.0), (1, 129, 65, 1, 1, 64, 0, 0.0),
    (1, 130, 1100, 1, 1, 64, 11, 0.4),           # wide columns and split keys
    (1, 66, 640, 2, 1, 88, 0, 0.0),
    (3, 70, 512, 3, 3, 50, 8, 0.5),              # rows that are not whole chunks, split
])
def test_more_shapes_match_the_definition(dtype, B, Lq, Lk, H, E, D, groups, dropped):
    _matches_the_definition(dtype, B, Lq, Lk, H, E, D, groups, dropped)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,Lk,H,E,D,groups", [(13, 36, 6, 2, 40, 12), (12, 12, 4, 4, 64, 0), (70, 64, 4, 2, 128, 8), (200, 20, 2, 2, 32, 5), (1, 7, 4, 1, 96, 0), (9, 33, 2, 1, 125, 0)])
def test_gradients_over_few_keys_carry_one_rounding(dtype, Lq, Lk, H, E, D, groups):
    """Where all keys lie in one tile P and dS are not rounded to 16 bits: a gradient carries its store's rounding u, what two 16-bit parts leave of P
    and dS (u^2 relative; below 2^-14 of float16 at most 2^-25 each), and 32-bit arithmetic, all against the absolute sums."""
    g = _gen(52)
    q, k, v, do = (_randn(g, *s, dtype=dtype) for s in ((2, Lq, H, D), (2, Lk, E, D), (2, Lk, E, D), (2, Lq, H, D)))
    keep = torch.rand(2, groups, generator=g, device=_dev()) < 0.5 if groups else None
    got = _all(q, k, v, do, keep=keep)
    want, size = _attend64(q, k, v, keep, D ** -0.5, do)
    u = _u(dtype)
    small = 2 * u * u + 2.0 ** -24 * (4 * D + 64)
    low = 2.0 ** -25 * (6 * max(Lk, Lq * (H // E)) + 1) if dtype == torch.float16 else 0.0
    for name, a, w, s in zip(("dq", "dk", "dv"), got[1:], want[1:], size[1:]):
        assert ((a.double() - w).abs() <= u * w.abs() + 2 * small * s + low + 1e-30).all(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,post,gate,views,D", [("rms", False, None, 0, 384), ("rms", False, "channel", 4, 384), ("layer", True, "object", 4, 837), ("rms", True, "channel", 0, 1500)])
def test_norm_gradients_of_16_bit_streams_carry_one_rounding(dtype, kind, post, gate, views, D):
    """y's rounding does not enter the backward: a gradient is off by its own store's u, relative to the tensor's 2-norm, and by 32-bit sums over D and
    over the rows (100 2^-24, as for 32-bit streams)."""
    g = _gen(D + 7)
    B, L = 3, 20
    t = {"residual": _randn(g, B, L, D, dtype=dtype) * 2, "branch": _randn(g, B, L, D, dtype=dtype), "weight": 1 + 0.2 * _randn(g, D, dtype=dtype),
         "post": 1 + 0.2 * _randn(g, D, dtype=dtype) if post else None, "gate": None if gate is None else _randn(g, *((B, D) if gate == "object" else (D,)), dtype=dtype)}
    draws = rows = None
    if views:
        draws = (torch.rand(B, views, generator=g, device=_dev()) >= 0.4).float() / 0.6
        draws[0, 0] = 0.0
        rows = draws.double().repeat_interleave(L // views, 1)[..., None]
    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    dy, dz = _randn(g, B, L, D, dtype=dtype), _randn(g, B, L, D, dtype=dtype)
    out = tokens.add_norm_tokens(leaves["residual"], leaves["branch"], leaves["weight"], post_weight=leaves.get("post"), gate=leaves.get("gate"), scale=draws, kind=kind)
    got = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), (dy, dz))))
    wy, wz, w = _norm64(t, kind, 1e-6, rows)
    want = dict(zip(leaves, torch.autograd.grad((wy, wz), [w[k] for k in leaves], (dy.double(), dz.double()))))
    for k, a in got.items():
        far, norm = (a.double() - want[k]).norm(), want[k].norm()
        assert far <= (_u(dtype) + 100 * U32) * norm + _tiny(dtype) * a.numel() ** 0.5, (k, float(far / norm))


def _unaligned(t):
    """The same values, one element behind an aligned address."""
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


def _heads_first(t):
    return t.transpose(1, 2).contiguous().transpose(1, 2)


def _in_joint(t):
    """A slice of a projection that holds other things beside it."""
    wide = torch.full(t.shape[:2] + (3,) + t.shape[2:], math.nan, dtype=t.dtype, device=t.device)
    wide[:, :, 1] = t
    return wide[:, :, 1]


def _backwards(t):
    """The last dimension strided: taken over a packed copy."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2)


@pytest.mark.parametrize("layout", [_unaligned, _heads_first, _in_joint, _backwards])
@pytest.mark.parametrize("Lq,Lk,H,E,D", [(70, 130, 4, 2, 64), (200, 70, 2, 2, 128), (1, 700, 4, 1, 72), (33, 40, 2, 1, 31)])
def test_layouts_do_not_change_results(layout, Lq, Lk, H, E, D):
    g = _gen(31)
    q, k, v, do = (_randn(g, *s, dtype=torch.bfloat16) for s in ((2, Lq, H, D), (2, Lk, E, D), (2, Lk, E, D), (2, Lq, H, D)))
    want, got = _all(q, k, v, do), _all(layout(q), layout(k), layout(v), layout(do))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_expanded_keys_and_gradients():
    """Keys shared by a batch, and the gradient of a sum (strides of 0 everywhere)."""
    g = _gen(32)
    q, k, v = (_randn(g, *s, dtype=torch.float16) for s in ((3, 50, 2, 64), (1, 90, 2, 64), (1, 90, 2, 64)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(tokens.attend_tokens(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)).sum(), leaves)
    apart = _all(q, k.repeat(3, 1, 1, 1), v.repeat(3, 1, 1, 1), torch.ones_like(q))
    assert torch.equal(got[0], apart[1])
    for a, b in zip(got[1:], apart[2:]):   # three float16 values are summed and rounded once, in torch's order or ours
        assert ((a.double() - b.double().sum(0, keepdim=True)).abs() <= 3 * _u(torch.float16) * b.double().abs().sum(0, keepdim=True) + 2 ** -25).all()


def test_masks_of_any_type():
    g = _gen(33)
    q, k, v, do = (_randn(g, 2, 60, 2, 64, dtype=torch.bfloat16) for _ in range(4))
    keep = torch.tensor([[1, 0, 1, 1], [0, 1, 0, 0]], device=_dev())
    want = _all(q, k, v, do, keep=keep.bool())
    for other in (keep, keep.to(torch.uint8) * 200, keep.float() / 0.75, keep.to(torch.bfloat16) * -3, keep.repeat_interleave(15, 1).bool(),
                  keep.bool().t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(_all(q, k, v, do, keep=other), want))
    gone = (keep == 0).repeat_interleave(15, 1)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(torch.bfloat16).min):
        kb, vb = k.clone(), v.clone()
        kb[gone], vb[gone] = bad, bad
        assert all(torch.equal(a, b) for a, b in zip(_all(q, kb, vb, do, keep=keep), want))


@pytest.mark.parametrize("B,Lq,Lk", [(0, 4, 4), (2, 0, 4), (2, 4, 0)])
def test_empty_sizes(B, Lq, Lk):
    q, k = torch.ones(B, Lq, 2, 16, dtype=torch.float16, device=_dev()), torch.ones(B, Lk, 2, 16, dtype=torch.float16, device=_dev())
    for t, like in zip(_all(q, k, k, q), (q, q, k, k)):
        assert t.shape == like.shape and not t.any()


def test_large_scores_stay_finite():
    """Scores of +-1e5: the maximum moves by more than it may lag, and one key takes all."""
    g = _gen(34)
    q, k, v, do = (_randn(g, 1, n, 1, 64, dtype=torch.bfloat16) for n in (70, 300, 300, 70))
    got = _all(q * 100, k * 100, v, do, scale=1.0)
    best = ((q * 100)[0, :, 0].double() @ (k * 100)[0, :, 0].double().T).topk(2, 1)
    clear = best.values[:, 0] - best.values[:, 1] > 40   # (e^-40 of the second key)
    assert clear.any() and all(torch.isfinite(t).all() for t in got)
    assert torch.equal(got[0][0, clear, 0], v[0, best.indices[clear, 0], 0])


def _cases():
    g = _gen(35)
    for B, Lq, Lk, H, E, D, groups in ((2, 100, 130, 4, 2, 64, 10), (2, 1, 900, 4, 1, 128, 20), (1, 200, 70, 2, 2, 72, 7)):
        yield [_randn(g, *s, dtype=torch.bfloat16) for s in ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D), (B, Lq, H, D))] + [torch.rand(B, groups, generator=g, device=_dev()) < 0.6]


def test_attention_on_another_stream():
    for case in _cases():
        want = _all(*case)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _all(*case)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_in_two_graphs():
    """Forward and backward captured, split keys among them; two graphs replayed in turn with eager calls between."""
    for case in _cases():
        static = [[t.clone() for t in case] for _ in range(2)]
        _all(*static[0])
        torch.cuda.synchronize()
        graphs, outs = [], []
        for s in static:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(_all(*s))
        for turn in range(4):
            now = [[t if t.dtype == torch.bool else _randn(_gen(40 + 2 * turn + k), *t.shape, dtype=t.dtype) for t in case] for k in range(2)]
            for n, s in zip(now, static):
                for a, b in zip(s, n):
                    a.copy_(b)
            for graph in graphs:
                graph.replay()
            eager = [_all(*n) for n in now]
            torch.cuda.synchronize()
            for got, want in zip(outs, eager):
                assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


def test_a_cache_of_more_than_2_31_elements():
    """One query over 2.1 million keys of which the last 1024 are kept: the rest holds whatever the memory held."""
    E, D, per, groups = 8, 128, 1024, 2100
    k, v = (torch.empty(1, per * groups, E, D, dtype=torch.bfloat16, device=_dev()) for _ in range(2))
    assert k.numel() > 2 ** 31
    g = _gen(36)
    q, do = (_randn(g, 1, 1, E, D, dtype=torch.bfloat16) for _ in range(2))
    k[:, -per:], v[:, -per:] = _randn(g, 1, per, E, D, dtype=torch.bfloat16), _randn(g, 1, per, E, D, dtype=torch.bfloat16)
    keep = torch.zeros(1, groups, dtype=torch.bool, device=_dev())
    keep[:, -1] = True
    out, dq, dk, dv = _all(q, k, v, do, keep=keep)
    want, size = _attend64(q, k[:, -per:], v[:, -per:], None, D ** -0.5, do)
    room = (1 + 1 / 32) * _u(torch.bfloat16) + 2 ** -24 * (4 * D + 64)   # one rounding of P and dS each, delta's, and the store's
    for a, w, s, inner in zip((out, dq, dk[:, -per:], dv[:, -per:]), want, size, (1, 2, 2, 1)):
        assert ((a.double() - w).abs() <= room * w.abs() + inner * room * s + 1e-30).all()
    assert not dk[:, :-per].any() and not dv[:, :-per].any()


@pytest.mark.parametrize("stride", [2 ** 24 - 8, 2 ** 25])   # loads of whole chunks at 32-bit offsets in a tile, and rows beyond those
def test_rows_far_apart(stride):
    g = _gen(37)
    q, k, v, do = (_randn(g, 1, n, 1, 64, dtype=torch.bfloat16) for n in (40, 140, 140, 40))
    far = torch.empty(140 * stride, dtype=torch.bfloat16, device=_dev()).as_strided((1, 140, 1, 128), (140 * stride, stride, 128, 1))
    assert 139 * stride > 2 ** 31
    far[..., :64], far[..., 64:] = k, v
    got, want = _all(q, far[..., :64], far[..., 64:], do), _all(q, k, v, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_gradient_against_differences():
    """Central differences of sum(out do) along the gradient's signs.  The difference of the kernel's own outputs is off by the outputs' roundings
    (each output by (2 + 1/16) u of its absolute sum, P's rounding and the store, and by what float16 loses below 2^-14), the gradient along the
    way by its own, and a finite step by what is had in 64 bits."""
    g, u, h = _gen(38), _u(torch.float16), 0.125
    q, k, v, do = (_randn(g, 2, n, 2, 16, dtype=torch.float16) for n in (5, 9, 9, 5))
    keep = torch.tensor([[1, 0, 1], [1, 1, 1]], device=_dev()).bool()
    got = _all(q, k, v, do, keep=keep)
    exact, size = _attend64(q, k, v, keep, 0.25, do)
    lost = 2 ** -25 * (6 * 9 + 1)   # of 9 probabilities, times |v| < 6, and of the store
    for which, t in enumerate((q, k, v)):
        way, ends = exact[1 + which].sign(), []
        for sign in (1, -1):
            args = [q, k, v]
            args[which] = (t.double() + sign * h * way).to(torch.float16)
            o = tokens.attend_tokens(*args, keep=keep).double()
            w, s = _attend64(*args, keep, 0.25, do)
            ends.append(((o * do.double()).sum(), (w[0] * do.double()).sum(), (s[0] * do.double().abs()).sum(), args[which].double()))
        step = ends[0][3] - ends[1][3]   # (as rounded)
        along, along64 = (got[1 + which].double() * step).sum(), (exact[1 + which] * step).sum()
        noise = (2 + 1 / 16) * u * (ends[0][2] + ends[1][2]) + 2 * lost * do.double().abs().sum()
        noise = noise + 4 * u * (size[1 + which] * step.abs()).sum() + 2 * lost * step.abs().sum()
        finite = (ends[0][1] - ends[1][1] - along64).abs()
        assert (ends[0][0] - ends[1][0] - along).abs() <= noise + finite, which
        assert along64 > noise, which   # (the test says something)


def test_all_together():
    """Cameras' positions, rotary queries and keys, attention without the dropped views, the residual kept where a view is dropped: each stage and
    each gradient against 64 bits from that stage's own inputs, down to azimuth and elevation."""
    g = _gen(39)
    B, V, rows, cols, H, D = 2, 6, 5, 3, 4, 32
    L, C, dtype = V * rows * cols, H * D, torch.float16
    azim, elev = (_randn(g, B, V) * 60).requires_grad_(), (_randn(g, B, V) * 20).requires_grad_()
    torch.manual_seed(5)
    scale = draw_regularization(B, V, 8, _dev(), dropout_p=0.4)[0].view(B, V)
    assert 0 < int((scale == 0).sum()) < B * V
    qkv = _randn(g, B, L, 3, H, D, dtype=dtype).requires_grad_()
    x = _randn(g, B, L, C).requires_grad_()
    weight = (_randn(g, C) * 0.1 + 1).requires_grad_()
    rotary = tokens.TokenRotary((4, 4, 4, 4), periods=(360.0, 360.0, None, None))
    positions = tokens.token_positions(azim, elev, rows, cols)
    q, k = rotary(qkv[:, :, 0], positions), rotary(qkv[:, :, 1], positions)
    out = tokens.attend_tokens(q, k, qkv[:, :, 2], keep=scale)
    y, z = tokens.add_norm_tokens(x, out.reshape(B, L, C), weight, scale=scale)
    for t in (positions, q, k, out, y, z):
        t.retain_grad()
    dz = _randn(g, B, L, C, dtype=dtype)
    (z * dz).sum().backward()
    u = _u(dtype)
    keep = scale != 0
    want, size = _attend64(q.detach(), k.detach(), qkv[:, :, 2].detach(), keep, D ** -0.5, out.grad)
    room = (1 + 1 / 32) * u + 2 ** -24 * (4 * D + 64)
    low = 2 ** -25 * 6 * L   # float16 below its normal numbers, in P and dS
    low_grad = low * float(out.grad.abs().max().clamp(min=1))
    for a, w, s, inner, l in zip((out, q.grad, k.grad, qkv.grad[:, :, 2]), want, size, (1, 2, 2, 1), (low, low_grad, low_grad, low_grad)):
        assert ((a.detach().double() - w).abs() <= room * w.abs() + inner * room * s + l).all()
    # dropped views: residual kept to the bit, nothing to their keys and values, nothing from their branch
    gone = (~keep).repeat_interleave(rows * cols, 1)
    assert torch.equal(y[gone], x[gone]) and not k.grad[gone].any() and not qkv.grad[:, :, 2][gone].any() and not out.grad[gone].any()
    y64 = x.detach().double() + out.detach().reshape(B, L, C).double() * scale.double().repeat_interleave(rows * cols, 1)[..., None]
    assert ((y.detach().double() - y64).abs() <= 3 * 2.0 ** -24 * (x.detach().abs().double() + (y64 - x.detach().double()).abs())).all()
    # the rotation, queries' and keys' parts: dx carries its store's rounding, dpos the 32-bit sums of H * 4 pairs' products
    gp = torch.zeros_like(positions, dtype=torch.float64)
    spread = torch.zeros_like(gp)
    for slot, t in ((0, q), (1, k)):
        wy, wdx, wdpos = _rotary64(rotary, qkv.detach()[:, :, slot], positions.detach(), t.grad)[:3]
        assert ((t.detach().double() - wy).abs() <= u * wy.abs() + 2.0 ** -20 * qkv.detach()[:, :, slot].abs().amax(-1, keepdim=True).double() + 2 ** -25).all()
        assert ((qkv.grad[:, :, slot].double() - wdx).abs() <= u * wdx.abs() + 2.0 ** -20 * t.grad.abs().amax(-1, keepdim=True).double() + 2 ** -25).all()
        gp += wdpos
        # |x| |dx| over the axis' pairs, 2 pi turns at most each
        span = (qkv.detach()[:, :, slot].double().abs().amax((-1, -2)) * t.grad.double().abs().amax((-1, -2)) * H * 8)[..., None]
        spread += span * 2 * math.pi * max(rotary.turns)
    assert ((positions.grad.double() - gp).abs() <= 2.0 ** -18 * spread + 2.0 ** -22 * gp.abs()).all()
    per_view = positions.grad.double().view(B, V, rows * cols, 4)
    for axis, camera in ((0, azim), (1, elev)):
        sums = per_view[..., axis].sum(2)
        assert ((camera.grad.double() - sums).abs() <= 2.0 ** -20 * per_view[..., axis].abs().sum(2)).all()
        assert camera.grad.abs().max() > 0


def test_all_together_repeats_in_a_graph():
    """The whole block as one captured step, gradients down to the cameras, several replays against eager runs."""
    B, V, rows, cols, H, D = 2, 4, 3, 5, 2, 64
    L, C = V * rows * cols, H * D
    rotary = tokens.TokenRotary((8, 8, 8, 8), periods=(360.0, 360.0, None, None))
    g = _gen(50)
    weight = _randn(g, C, dtype=torch.bfloat16)

    def step(azim, elev, qkv, scale):
        leaves = [t.detach().requires_grad_() for t in (azim, elev, qkv)]
        positions = tokens.token_positions(leaves[0], leaves[1], rows, cols)
        q, k = rotary(leaves[2][:, :, 0], positions), rotary(leaves[2][:, :, 1], positions)
        out = tokens.attend_tokens(q, k, leaves[2][:, :, 2], keep=scale).reshape(B, L, C)
        y, z = tokens.add_norm_tokens(leaves[2][:, :, 0].reshape(B, L, C), out, weight, post_weight=weight, scale=scale)
        return [y.detach(), z.detach()] + list(torch.autograd.grad((y, z), leaves, (z.detach(), y.detach())))

    def inputs(k):
        g = _gen(60 + k)
        return [_randn(g, B, V) * 90, _randn(g, B, V) * 30, _randn(g, B, L, 3, H, D, dtype=torch.bfloat16), (torch.rand(B, V, generator=g, device=_dev()) < 0.6).float() / 0.6]
    static = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for k in range(1, 5):
        for a, b in zip(static, inputs(k)):
            a.copy_(b)
        graph.replay()
        eager = step(*inputs(k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
