"""-m gpu: the operators on view tokens (mvtn_amd/tokens.py) against their definitions in 64 bits.

Tolerances count roundings.  u(t) is half a step of a type relative to the value: 2^-24 for float32, 2^-11 for float16, 2^-8 for
bfloat16.  A result carries one u(t) of its own from the store, and what its 32-bit arithmetic adds, which is bounded in each test from the
absolute values of the terms that enter."""
import math

import pytest
import torch

from mvtn_amd import tokens

from gpu_helpers import _dev

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half the smallest step of a type: what a store near zero may lose."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=_dev()).to(dtype)


# ---- rotary ----------------------------------------------------------------------------------------------------------

def _rotary64(rotary, x, positions, dy):
    """y, dx, dpos in 64 bits."""
    n = rotary.pairs
    axis = torch.tensor([a for a, s in enumerate(rotary.sections) for _ in range(s)], device=x.device)
    turns = torch.tensor(rotary.turns, dtype=torch.float64, device=x.device)
    ang = (torch.remainder(positions.double()[..., axis] * turns, 1.0) * 2 * math.pi)[:, :, None]
    c, s = ang.cos(), ang.sin()
    one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if rotary.interleaved else (slice(0, n), slice(n, 2 * n))

    def turn(t, s):
        out = t.double().clone()
        out[..., one], out[..., two] = t.double()[..., one] * c - t.double()[..., two] * s, t.double()[..., one] * s + t.double()[..., two] * c
        return out
    y, dx = turn(x, s), turn(dy, -s)
    slope = (x.double()[..., one] * dx[..., two] - x.double()[..., two] * dx[..., one]) * 2 * math.pi * turns
    size = (x.double()[..., one].abs() * dx[..., two].abs() + x.double()[..., two].abs() * dx[..., one].abs()) * 2 * math.pi * turns
    onehot = (axis[:, None] == torch.arange(len(rotary.sections), device=x.device)).double()
    return y, dx, slope.sum(2) @ onehot, size.sum(2) @ onehot


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,L,H,D,sections,periods", [
    (1, 1, 1, 2, (1,), (None,)),                      # the smallest
    (2, 12, 12, 64, (16, 16), (360.0, 360.0)),        # a token per view
    (3, 65, 5, 80, (9, 11, 13), (None, None, 360.0)),    # odd sections, a tail behind the pairs
    (1, 7, 3, 22, (3, 1, 2, 4), (360.0, None, 360.0, None)),   # rows that are not 16-byte aligned
    (2, 33, 24, 128, (64,), (None,)),                  # the whole head, one axis
    (1, 300, 1, 256, (32, 32, 32, 32), (360.0, 360.0, None, None)),   # the widest head
])
def test_rotary_matches_the_definition(dtype, interleaved, B, L, H, D, sections, periods):
    g = _gen(L * D)
    rotary = tokens.TokenRotary(sections, base=100.0, periods=periods, interleaved=interleaved)
    x, dy = _randn(g, B, L, H, D, dtype=dtype).requires_grad_(), _randn(g, B, L, H, D, dtype=dtype)
    pos = ((torch.rand(B, L, len(sections), generator=g, device=_dev()) - 0.5) * 1e5).requires_grad_()
    y = rotary(x, pos)
    dx, dpos = torch.autograd.grad(y, (x, pos), dy)
    wy, wdx, wdpos, size = _rotary64(rotary, x.detach(), pos.detach(), dy)
    # the fraction of a turn is rounded once to 32 bits (|r| <= 1/2: 2^-26 turns = pi 2^-25 rad), sine and cosine are good to 2 u each, then a
    # product, a fused product-sum: 10 u of each element's partner is ample (2 pi / 4 + 2 + 2 < 6)
    n = rotary.pairs
    for got, want, src in ((y, wy, x), (dx, wdx, dy)):
        far = (got.detach().double() - want).abs()
        pair = src.detach().double().abs()
        head = torch.zeros_like(pair)
        a, b = (pair[..., 0:2 * n:2], pair[..., 1:2 * n:2]) if interleaved else (pair[..., :n], pair[..., n:2 * n])
        if interleaved:
            head[..., 0:2 * n:2], head[..., 1:2 * n:2] = a + b, a + b
        else:
            head[..., :n], head[..., n:2 * n] = a + b, a + b
        assert (far <= 10 * U32 * head + (1 + 2 ** -8) * _u(dtype) * want.abs() + _tiny(dtype)).all()
        assert torch.equal(got[..., 2 * n:], src[..., 2 * n:])
    # dpos: terms good to 14 u (two products of a rotated and a given value, the factor), sums of heads and pairs in 32 bits
    assert ((dpos.double() - wdpos).abs() <= (14 + H + n) * U32 * size).all()
    again = torch.autograd.grad(rotary(x, pos), (x, pos), dy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dpos)   # bit-reproducible
    # the positions' gradient against differences of the definition
    i = int(torch.randint(0, L, (1,)).item())
    for axis in range(len(sections)):
        e = torch.zeros_like(pos)
        e[:, i, axis] = 1e-4
        plus, minus = (_rotary64(rotary, x.detach(), pos.detach().double() + s * e.double(), dy)[0] for s in (1, -1))
        slope = ((plus - minus) * dy.double()).sum((1, 2, 3)) / 2e-4
        assert ((slope - dpos[:, i, axis].double()).abs() <= 1e-6 * size[:, i, axis] + (14 + H + n) * U32 * size[:, i, axis]).all()


def test_rotary_periodic_axis_returns_and_far_positions_hold():
    """A period apart is the same place, bit by bit where the positions are exact; a far position keeps its angle."""
    g = _gen(1)
    x = _randn(g, 1, 8, 2, 32)
    cams = tokens.TokenRotary((8, 8), periods=(360.0, 360.0))
    p = torch.tensor([[-180.0, 45.0], [0.0, 0.0], [90.0, -30.0], [10.0, 20.0], [1.0, 2.0], [-7.0, 5.0], [123.0, 60.0], [359.0, 1.0]], device=_dev())
    assert torch.equal(cams(x, p)[:, 1], x[:, 1])
    far = (cams(x, p) - cams(x, p + 360.0)).abs().max()
    assert far <= 16 * U32 * x.abs().max()
    ladder = tokens.TokenRotary((16,), base=10000.0)
    big = torch.full((8, 1), 2.0 ** 24 - 1, device=_dev())
    assert ((ladder(x, big).double() - _rotary64(ladder, x, big[None], x)[0]).abs() <= 10 * U32 * 2 * x.abs().max()).all()


def test_rotary_strides_broadcast_and_empty():
    g = _gen(2)
    B, L, H, D = 2, 9, 3, 16
    rotary = tokens.TokenRotary((3, 2), periods=(360.0, None))
    qkv = _randn(g, B, L, 3 * H, D, dtype=torch.bfloat16).requires_grad_()
    pos = (_randn(g, L, 2) * 50).requires_grad_()
    dy = _randn(g, H, L, B, D, dtype=torch.bfloat16).transpose(0, 2)        # a gradient with other strides
    y = rotary(qkv[:, :, H:2 * H], pos)                                     # heads inside a joint projection, positions of the whole batch
    dq, dp = torch.autograd.grad(y, (qkv, pos), dy)
    x = qkv.detach()[:, :, H:2 * H].contiguous().requires_grad_()
    each = pos.detach().expand(B, L, 2).contiguous().requires_grad_()
    want = rotary(x, each)
    wdx, wdp = torch.autograd.grad(want, (x, each), dy.contiguous())
    assert torch.equal(y, want) and torch.equal(dq[:, :, H:2 * H], wdx) and not dq[:, :, :H].any() and not dq[:, :, 2 * H:].any()
    assert torch.equal(dp, wdp[0] + wdp[1])
    heads_first = _randn(g, B, H, L, D)
    assert torch.equal(rotary(heads_first.transpose(1, 2), pos), rotary(heads_first.transpose(1, 2).contiguous(), pos))
    assert torch.equal(rotary(heads_first.transpose(1, 2), pos.detach().t().contiguous().t()), rotary(heads_first.transpose(1, 2), pos))
    assert torch.equal(rotary(x[:1].expand(B, L, H, D), pos), rotary(x[:1], pos).expand(B, L, H, D))
    assert torch.equal(rotary(x, pos.detach().double()), rotary(x, pos))
    empty = torch.zeros(B, 0, H, D, device=_dev(), requires_grad=True)
    no = torch.zeros(0, 2, device=_dev(), requires_grad=True)
    out = rotary(empty, no)
    assert out.shape == empty.shape
    gx, gp = torch.autograd.grad(out, (empty, no), torch.zeros_like(out))
    assert gx.shape == empty.shape and gp.shape == no.shape
    # only x, only positions
    x1 = x.detach()
    assert torch.equal(torch.autograd.grad(rotary(x1, each), each, dy)[0], wdp)
    assert torch.equal(torch.autograd.grad(rotary(x, each.detach()), x, dy)[0], wdx)


def test_rotary_of_more_than_2_31_elements():
    """Offsets past 32 bits: the last tokens of a tensor of 2.2e9 elements."""
    B, L, H, D = 1, 70000, 248, 128
    x = torch.zeros(B, L, H, D, dtype=torch.bfloat16, device=_dev())
    x[:, -3:] = _randn(_gen(3), B, 3, H, D, dtype=torch.bfloat16)
    pos = torch.arange(L, device=_dev(), dtype=torch.float32)[:, None]
    rotary = tokens.TokenRotary((64,))
    y = rotary(x, pos)
    assert torch.equal(y[:, -3:], rotary(x[:, -3:].contiguous(), pos[-3:])) and not y[:, :1000].any()


# ---- norms around a block --------------------------------------------------------------------------------------------

def _norm64(t, kind, eps, scale_rows):
    """y, z and the gradients of everything by automatic differentiation in 64 bits."""
    t = {k: (v.detach().double().requires_grad_() if torch.is_tensor(v) and k in ("residual", "branch", "weight", "bias", "post", "gate") else v)
         for k, v in t.items()}

    def norm(u):
        u = u - u.mean(-1, keepdim=True) if kind == "layer" else u
        return u / (u.square().mean(-1, keepdim=True) + eps).sqrt()
    branch = t["branch"] if scale_rows is None else torch.where(scale_rows == 0, torch.zeros_like(t["branch"]), t["branch"])
    n = norm(branch) * t["post"] if t.get("post") is not None else branch
    if t.get("gate") is not None:
        gate = t["gate"]
        gate = gate.reshape(gate.shape[0], *([1] * (branch.dim() - 2)), gate.shape[-1]) if gate.dim() > 1 else gate
        n = n * gate
    y = t["residual"] + (n if scale_rows is None else scale_rows * n)
    z = norm(y) * t["weight"] + (t["bias"] if t.get("bias") is not None else 0.0)
    return y, z, t


@pytest.mark.parametrize("types", [("float32",) * 3, ("float16",) * 3, ("bfloat16",) * 3, ("float32", "bfloat16", "float32"), ("float32", "float16", "float32")])
@pytest.mark.parametrize("kind,post,gate,views,D", [
    ("rms", False, None, 0, 1), ("layer", True, "object", 4, 8), ("rms", True, "channel", 0, 65), ("layer", False, "object", 2, 384), ("layer", True, None, 4, 513),
    ("rms", True, "object", 4, 768), ("rms", False, None, 2, 1024), ("layer", True, "channel", 0, 1025), ("layer", True, "object", 4, 2047),
    ("rms", True, "object", 0, 2052), ("layer", True, "channel", 4, 4097), ("rms", True, None, 2, 8192)])
def test_add_norm_matches_the_definition(types, kind, post, gate, views, D):
    r, b, p = (getattr(torch, t) for t in types)
    g = _gen(D)
    B, L = 3, 20
    t = {"residual": _randn(g, B, L, D, dtype=r) * 2 + 0.1, "branch": _randn(g, B, L, D, dtype=b) + 0.1, "weight": 1 + 0.2 * _randn(g, D, dtype=p),
         "bias": 0.2 * _randn(g, D, dtype=p) if kind == "layer" else None, "post": 1 + 0.2 * _randn(g, D, dtype=p) if post else None,
         "gate": None if gate is None else _randn(g, *((B, D) if gate == "object" else (D,)), dtype=p)}
    draws = rows = None
    if views:
        draws = (torch.rand(B, views, generator=g, device=_dev()) >= 0.4).float() / 0.6
        draws[0, 0] = 0.0
        rows = draws.double().repeat_interleave(L // views, 1)[..., None]
    dy, dz = _randn(g, B, L, D, dtype=r), _randn(g, B, L, D, dtype=b)
    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    call = lambda q: tokens.add_norm_tokens(q["residual"], q["branch"], q["weight"], q.get("bias"), post_weight=q.get("post"), gate=q.get("gate"),  # noqa: E731
                                            scale=draws, kind=kind)
    if views:   # whatever a dropped view's branch holds stays out of everything
        with torch.no_grad():
            leaves["branch"].view(B * views, -1)[draws.view(-1) == 0] = math.nan
    y, z = call(leaves)
    names = list(leaves)
    got = dict(zip(names, torch.autograd.grad((y, z), [leaves[k] for k in names], (dy, dz))))
    wy, wz, w = _norm64(t, kind, 1e-6, rows)
    want = dict(zip(names, torch.autograd.grad((wy, wz), [w[k] for k in names], (dy.double(), dz.double()))))
    # relative to a tensor's norm: one rounding of its own; y's rounding, when the stream is kept in 16 bits, enters the backward as yhat and
    # its row means (two more); 32-bit sums over D and over the rows: (D / 8 + 60) u at worst in a chain, in 2-norm far less: 100 u
    ur, ub, up = _u(r), _u(b), _u(p)
    kept = 2 * ur if r != torch.float32 else 0.0
    for name, a, e, own, extra in [("y", y, wy, ur, 0.0), ("z", z, wz, ub, 0.0)] + [
            (k, got[k], want[k], {"residual": ur, "branch": ub}.get(k, up), kept) for k in names]:
        far, norm = (a.detach().double() - e.detach()).norm(), e.detach().norm()
        assert far <= (own + extra + 100 * U32) * norm + _tiny(a.dtype) * a.numel() ** 0.5 + (U32 * 100 if D == 1 else 0.0), (name, float(far / norm))
        # and element by element, in terms of the tensor's own size
        assert ((a.detach().double() - e.detach()).abs() <= (2 * own + 8 * extra + 200 * U32) * (e.detach().abs() + e.detach().abs().max())).all(), name
    if views:
        gone = (draws == 0).repeat_interleave(L // views, 1)
        assert torch.equal(y[gone], t["residual"][gone]) and not got["branch"][gone].any()
    with torch.no_grad():
        y0, z0 = call(leaves)
    assert torch.equal(y0, y) and torch.equal(z0, z)
    y1, z1 = call(leaves)
    again = torch.autograd.grad((y1, z1), [leaves[k] for k in names], (dy, dz))
    assert all(torch.equal(a, got[k]) for k, a in zip(names, again))   # bit-reproducible


def test_add_norm_gradient_against_differences():
    g = _gen(9)
    B, L, D = 2, 3, 24
    t = {"residual": _randn(g, B, L, D), "branch": _randn(g, B, L, D), "weight": 1 + 0.2 * _randn(g, D), "bias": 0.2 * _randn(g, D),
         "post": 1 + 0.2 * _randn(g, D), "gate": _randn(g, B, D)}
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    dy, dz = _randn(g, B, L, D), _randn(g, B, L, D)
    y, z = tokens.add_norm_tokens(leaves["residual"], leaves["branch"], leaves["weight"], leaves["bias"], post_weight=leaves["post"], gate=leaves["gate"],
                                  scale=0.7, kind="layer")
    got = dict(zip(leaves, torch.autograd.grad((y, z), list(leaves.values()), (dy, dz))))
    for name in leaves:
        e = torch.randn_like(t[name]).double()
        vals = []
        for s in (1e-5, -1e-5):
            q = {k: v.detach().double() for k, v in t.items()}
            q[name] = q[name] + s * e
            wy, wz, _ = _norm64(q, "layer", 1e-6, torch.tensor(0.7, device=_dev(), dtype=torch.float64))
            vals.append(float(((wy * dy.double()).sum() + (wz * dz.double()).sum()).detach()))
        slope, mine = (vals[0] - vals[1]) / 2e-5, float((got[name].double() * e).sum())
        # second differences of these smooth rows are O(1e-10) of the terms; 32-bit gradients: 100 u of them
        assert abs(slope - mine) <= (1e-8 + 100 * U32) * float((got[name].double().abs() * e.abs()).sum()), name


def test_add_norm_partial_gradients_strides_and_empty():
    g = _gen(10)
    B, L, D = 2, 5, 40
    x, a, w = _randn(g, B, L, D).requires_grad_(), _randn(g, B, L, D).requires_grad_(), _randn(g, D).requires_grad_()
    gate = _randn(g, B, 1, D).requires_grad_()
    y, z = tokens.add_norm_tokens(x, a, w, gate=gate)
    dy, dz = _randn(g, B, L, D), _randn(g, B, L, D)
    both = torch.autograd.grad((y, z), (x, a, w, gate), (dy, dz), retain_graph=True)
    assert both[3].shape == gate.shape
    only = [torch.autograd.grad(o, (x, a, gate), d, retain_graph=True) for o, d in ((y, dy), (z, dz))]
    for k, i in ((0, 0), (1, 1), (2, 3)):   # the gradient is linear in (dy, dz): two roundings of each part
        assert ((only[0][k] + only[1][k] - both[i]).abs() <= 64 * U32 * (only[0][k].abs() + only[1][k].abs()).max()).all()
    assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], dy)
    assert torch.equal(tokens.add_norm_tokens(x.detach(), a, w.detach(), gate=gate.detach())[0], y)   # some leaves only
    t = _randn(g, L, B, D).transpose(0, 1)
    assert torch.equal(tokens.add_norm_tokens(t, t, w)[1], tokens.add_norm_tokens(t.contiguous(), t.contiguous(), w)[1])
    assert torch.equal(tokens.add_norm_tokens(x, a, w, gate=gate.detach().view(B, D))[1], z)
    e = torch.zeros(0, 5, D, device=_dev(), requires_grad=True)
    ye, ze = tokens.add_norm_tokens(e, e, w)
    ge, gw = torch.autograd.grad((ye, ze), (e, w), (ye, ze))
    assert ye.shape == e.shape and ge.shape == e.shape and not gw.any()


def test_rotary_and_norm_on_another_stream_and_in_a_graph():
    g = _gen(11)
    B, L, H, D = 2, 50, 4, 32
    rotary = tokens.TokenRotary((8, 8))
    x, pos, w = _randn(g, B, L, H, D, dtype=torch.bfloat16), _randn(g, L, 2) * 9, _randn(g, H * D, dtype=torch.bfloat16)
    draws = torch.tensor([[0.0, 2.0], [2.0, 2.0]], device=_dev())

    def step(x):
        x = x.detach().requires_grad_()
        q = rotary(x, pos)
        y, z = tokens.add_norm_tokens(x.reshape(B, L, -1), q.reshape(B, L, -1), w, post_weight=w, scale=draws)
        return (y, z) + torch.autograd.grad((y, z), x, (y.detach(), z.detach()))
    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = x.clone()
    step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for k in range(4):
        xk = _randn(_gen(20 + k), B, L, H, D, dtype=torch.bfloat16)
        static.copy_(xk)
        graph.replay()
        eager = step(xk)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k


# ---- attention -------------------------------------------------------------------------------------------------------

def _attend64(q, k, v, keep, scale, do):
    """o, dq, dk, dv in 64 bits over the kept keys only, and the absolute sums that enter the rounding of P and dS: see the test."""
    B, Lq, H, D = q.shape
    Lk, E = k.shape[1:3]
    out = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, q, k, v)]
    size = [torch.zeros_like(t) for t in out]
    for b in range(B):
        on = torch.ones(Lk, dtype=torch.bool, device=q.device) if keep is None else (keep[b] != 0).repeat_interleave(Lk // keep.shape[1])
        at = on.nonzero()[:, 0]
        if not at.numel():
            continue
        for h in range(H):
            e = h // (H // E)
            Q, G = q[b, :, h].double(), do[b, :, h].double()
            K, V = k[b, at, e].double(), v[b, at, e].double()
            p = torch.softmax(Q @ K.T * scale, -1)
            o, dp = p @ V, G @ V.T
            ds = p * (dp - (G * o).sum(-1, keepdim=True))
            # |dS| with its two parts apart: p |dp| + p |delta|, where delta comes from the stored o
            ads = p * (dp.abs() + (G.abs() * o.abs()).sum(-1, keepdim=True))
            out[0][b, :, h], out[1][b, :, h] = o, ds @ K * scale
            size[0][b, :, h], size[1][b, :, h] = p @ V.abs(), ads @ K.abs() * scale
            out[2][b, at, e] += ds.T @ Q * scale
            out[3][b, at, e] += p.T @ G
            size[2][b, at, e] += ads.T @ Q.abs() * scale
            size[3][b, at, e] += p.T @ G.abs()
    return out, size


ATTENTION = [
    # B, Lq, Lk, H, E, D, groups, dropped
    (1, 1, 1, 1, 1, 1, 0, 0.0),                  # the smallest
    (2, 12, 12, 12, 12, 64, 12, 0.5),            # a token per view
    (3, 31, 33, 2, 2, 32, 0, 0.0),
    (2, 64, 64, 3, 3, 64, 0, 0.0),               # whole tiles
    (2, 65, 127, 4, 2, 40, 0, 0.0),              # ragged tiles, shared heads
    (1, 196, 196, 3, 1, 64, 4, 0.5),             # views of 49 tokens: groups end inside tiles
    (2, 5, 300, 6, 3, 96, 20, 0.3),
    (2, 129, 260, 2, 1, 128, 260, 0.4),          # a mask of single keys
    (2, 1, 1000, 8, 2, 128, 20, 0.25),           # one query: the keys are split
    (1, 1, 4500, 2, 2, 72, 0, 0.0),              # more tiles than a mask chunk
    (1, 3, 9000, 1, 1, 33, 9000, 0.9),           # odd head, most keys gone, three chunks
    (2, 300, 1, 2, 2, 17, 0, 0.0),               # one key
    (1, 700, 50, 4, 1, 104, 2, 0.5),             # many rows over few keys
    (2, 40, 640, 2, 2, 64, 5, 0.99),             # objects with every view dropped
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Lq,Lk,H,E,D,groups,dropped", ATTENTION)
def test_attention_matches_the_definition(dtype, B, Lq, Lk, H, E, D, groups, dropped):
    g = _gen(Lq * 7 + Lk)
    q, k, v, do = (_randn(g, *s, dtype=dtype) for s in ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D), (B, Lq, H, D)))
    keep = None
    if groups:
        keep = torch.rand(B, groups, generator=g, device=_dev()) >= dropped
        if dropped > 0.9:
            keep[-1] = False
    want, size = _attend64(q, k, v, keep, D ** -0.5, do)
    if groups:   # what a dropped key holds stays out
        gone = ~keep.repeat_interleave(Lk // groups, 1)
        k[gone], v[gone] = math.nan, math.inf
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = tokens.attend_tokens(*leaves, keep=keep)
    got = [out.detach()] + list(torch.autograd.grad(out, leaves, do))
    # scores: D products summed in 32 bits, |s log2 e| <= ~ 1.5 |q||k| / sqrt(D): exp2 moves by ln 2 times that error: bounded by 2^-24 (D + 8)
    # times the score's size, far below u(dtype) here.  P and dS are each rounded once (u) against their own absolute size, delta carries the
    # stored output's rounding (u); then the store (u).  1/32 u more for the 32-bit arithmetic (D and Lk sums: at most ~ 1e3 2^-24).
    u = _u(dtype)
    room = (1 + 1 / 32) * u + 2 ** -24 * (4 * D + 64)
    for name, a, w, s, inner in zip(("out", "dq", "dk", "dv"), got, want, size, (1, 2, 2, 1)):
        assert torch.isfinite(a).all(), name
        # subnormal steps of float16 in P and dS: below 2^-14 a value is off by up to 2^-25, times at most Lk or the rows, times |k|, |q|, |do| < 6
        low = 2 ** -25 * 6 * max(Lk, Lq * (H // E)) * D ** -0.5 if dtype == torch.float16 and name in ("dq", "dk") else 2 ** -25 * 6 * max(Lk, Lq * (H // E)) if dtype == torch.float16 else 0.0
        assert ((a.double() - w).abs() <= room * w.abs() + inner * room * s + low + 1e-30).all(), (name, float((a.double() - w).abs().max()))
    if groups:
        assert not got[2][gone].any() and not got[3][gone].any()
        empty = ~keep.any(1)
        assert not got[0][empty].any() and not got[1][empty].any()
    again = torch.autograd.grad(tokens.attend_tokens(*leaves, keep=keep), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(again, got[1:]))   # bit-reproducible
    with torch.no_grad():
        assert torch.equal(tokens.attend_tokens(*leaves, keep=keep), got[0])


def test_gradients_cannot_be_differentiated_again():
    """create_graph gives the gradients; a second differentiation fails where it is asked for, and not silently."""
    g = _gen(12)
    x = _randn(g, 1, 4, 2, 8).requires_grad_()
    pos = _randn(g, 4, 1).requires_grad_()
    h = _randn(g, 1, 4, 2, 8, dtype=torch.bfloat16).requires_grad_()
    rotary = tokens.TokenRotary((4,))
    for out, leaf in ((rotary(x, pos), x), (tokens.attend_tokens(h, h, h), h), (tokens.add_norm_tokens(x, x, _randn(g, 8))[1], x)):
        up = torch.ones_like(out).requires_grad_()
        first, = torch.autograd.grad(out, leaf, up, create_graph=True)
        assert torch.isfinite(first).all()
        with pytest.raises(RuntimeError, match="differentiated"):
            first.float().sum().backward()


def test_saved_tensors_that_were_written_over_are_noticed():
    g = _gen(13)
    x, w = _randn(g, 2, 4, 8).requires_grad_(), _randn(g, 8)
    y, z = tokens.add_norm_tokens(x, x, w)
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
