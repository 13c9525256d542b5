"""-m gpu: how far the attention's results lie from 64 bits, in 2-norm against what its roundings amount to.

A rounding to a type moves a value by a part of it that is spread over +-u (u: half a step), so by u^2 / 3 of its square at most in the mean; roundings of
different values are independent, so that their squares add up.  The store's own part is had by rounding the 64-bit result.  A 2-norm over n
elements strays by about 1 / sqrt(2 n) of itself: below 3 % at the 500 elements and more that are compared here, where the mean of u^2 / 3
leaves 26 % (a value's distance to the next is u to u / 2 of it)."""
import math

import pytest
import torch

from mvtn_amd import tokens

from gpu_helpers import _dev
from test_gpu_tokens import _gen, _randn, _u

pytestmark = pytest.mark.gpu


def _sizes(q, k, v, do, scale, keep=None, stored_out=False):
    """The results in 64 bits and the squares of what roundings in between add to them, elementwise: P where it enters P v and P^T dO, dS where it enters
    dS k and dS^T q, and delta, which P's rounding in the output reaches (a row's sum of dS^2: the sum is taken of the rounded P) and, with stored_out,
    the output's own store and that of the sum."""
    B, Lq, H, D = q.shape
    Lk, E = k.shape[1:3]
    out = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, q, k, v)]
    var = [torch.zeros_like(t) for t in out]
    f = _u(q.dtype) ** 2 / 3
    for b in range(B):
        at = torch.arange(Lk, device=q.device) if keep is None else (keep[b] != 0).repeat_interleave(Lk // keep.shape[1]).nonzero()[:, 0]
        for h in range(H):
            e = h // (H // E)
            Q, G, K, V = q[b, :, h].double(), do[b, :, h].double(), k[b, at, e].double(), v[b, at, e].double()
            p = torch.softmax(Q @ K.T * scale, -1)
            o = p @ V
            ds = p * (G @ V.T - (G * o).sum(-1, keepdim=True))
            # dP and delta are 32-bit sums of D products: D roundings, each of 2^-24 of a partial sum, whose square is in the mean at most that of the whole,
            # the products' squares added up (four times that here).  Nothing beside the rest, but where one key has all of P dP - delta is 0
            r = 4 * D * 2.0 ** -48 / f
            ds2 = ds.square() + p.square() * r * (G.square() @ V.square().T)
            delta = ds.square().sum(-1, keepdim=True) + r * (G * o).square().sum(-1, keepdim=True)
            gain = 0.0
            if stored_out:
                delta = delta + (G * o).square().sum(-1, keepdim=True)
                gain = p.square().sum(-1, keepdim=True)   # of all of a row's P
            pk = p @ K * scale
            out[0][b, :, h], out[1][b, :, h] = o, ds @ K * scale
            out[2][b, at, e] += ds.T @ Q * scale
            out[3][b, at, e] += p.T @ G
            # sum_j p^2 (v - o)^2
            var[0][b, :, h] = f * (p.square() @ V.square() - 2 * (p.square() @ V) * o + p.square().sum(-1, keepdim=True) * o.square())
            var[1][b, :, h] = f * (ds2 @ K.square() * scale ** 2 + delta * pk.square() + gain * (ds @ K * scale).square())
            var[2][b, at, e] += f * ((ds2 + p.square() * delta + gain * ds.square()).T @ Q.square()) * scale ** 2
            var[3][b, at, e] += f * ((1 + gain) * p.square()).T @ G.square()
    return out, var


def _call(q, k, v, do, keep=None, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = tokens.attend_tokens(*leaves, keep=keep, scale=scale)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, do))


def _check(got, want, var, dtype):
    for name, a, w, s in zip(("out", "dq", "dk", "dv"), got, want, var):
        assert torch.isfinite(a).all(), name
        store = (w.to(dtype).double() - w).norm()
        far, room = (a.double() - w).norm(), (store.square() + s.sum()).sqrt()
        assert far <= room + 2.0 ** -16 * w.norm(), (name, float(far / store), float(room / store))   # (32-bit scores, exponentials and sums: some 2^-18)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spread", [1.0, 3.0, 6.0, 10.0])
@pytest.mark.parametrize("B,Lq,Lk,H,E,D,groups", [(1, 512, 1024, 2, 1, 64, 0), (1, 300, 2352, 1, 1, 128, 12), (2, 200, 500, 2, 2, 41, 0), (4, 3, 3000, 8, 2, 64, 20), (4, 2, 3000, 4, 4, 100, 0), (2, 300, 100, 2, 1, 32, 0)])
def test_gradients_of_peaked_probabilities(dtype, spread, B, Lq, Lk, H, E, D, groups):
    """Scores with a deviation of 1 to 10: a few keys take nearly all.  Then dP - delta is a small difference, and neither the output's store nor the rounding
    of the sum may enter it."""
    g = _gen(74)
    q, k, v, do = (_randn(g, *s, dtype=dtype) for s in ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D), (B, Lq, H, D)))
    keep = torch.rand(B, groups, generator=g, device=_dev()) < 0.7 if groups else None
    scale = spread * D ** -0.5
    want, var = _sizes(q, k, v, do, scale, keep)
    _check(_call(q, k, v, do, keep, scale), want, var, dtype)


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("B,Lq,Lk,H,E,D", [(1, 300, 2352, 2, 1, 64), (2, 200, 1500, 1, 1, 128), (4, 1, 3920, 8, 4, 128), (1, 64, 30000, 1, 1, 32), (2, 500, 60, 2, 2, 64), (1, 700, 50, 4, 1, 104)])
def test_float16_gradients_of_any_size(size, B, Lq, Lk, H, E, D):
    """What a loss sends down is small (a mean over tokens), and P over thousands of keys is smaller: neither may fall out of float16's normal numbers."""
    g = _gen(70)
    q, k, v = (_randn(g, *s, dtype=torch.float16) for s in ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D)))
    do = (_randn(g, B, Lq, H, D) * size).to(torch.float16)
    want, var = _sizes(q, k, v, do, D ** -0.5, stored_out=True)
    _check(_call(q, k, v, do), want, var, torch.float16)


@pytest.mark.parametrize("Lk,D", [(40, 64), (40, 128), (200, 64), (200, 128), (3000, 72)])
def test_float16_gradients_beyond_its_largest_number(Lk, D):
    """dP and dS pass 65504 under a loss scale, where the gradients themselves do not."""
    g = _gen(71)
    q, k = (_randn(g, 1, n, 2, D).mul(0.01).to(torch.float16) for n in (70, Lk))
    v, do = _randn(g, 1, Lk, 2, D).mul(300).to(torch.float16), _randn(g, 1, 70, 2, D).mul(300).to(torch.float16)
    want, var = _sizes(q, k, v, do, D ** -0.5, stored_out=True)
    assert (do[0, :, 0].double() @ v[0, :, 0].double().T).abs().max() > 10 * 65504 and want[1].abs().max() < 65504
    got = _call(q, k, v, do)
    got[3], want[3] = got[3][:, :0], want[3][:, :0]   # (dV is large)
    var[3] = var[3][:, :0]
    _check(got, want, var, torch.float16)


@pytest.mark.parametrize("D", [64, 128])
def test_float16_gradients_whose_size_changes_along_the_keys(D):
    """Rows and keys of very different size in one column: the power of two follows them down."""
    g = _gen(72)
    q, k = (_randn(g, 1, 400, 1, D, dtype=torch.float16) for _ in range(2))
    grow = (2.0 ** torch.linspace(-12, 6, 400, device=_dev()))[None, :, None, None]
    v, do = (_randn(g, 1, 400, 1, D) * grow).to(torch.float16), (_randn(g, 1, 400, 1, D) * grow).to(torch.float16)
    want, var = _sizes(q, k, v, do, D ** -0.5, stored_out=True)
    _check(_call(q, k, v, do), want, var, torch.float16)
    _check(_call(q, k.flip(1), v.flip(1), do.flip(1)), *[x for x in _sizes(q, k.flip(1), v.flip(1), do.flip(1), D ** -0.5, stored_out=True)], torch.float16)


@pytest.mark.parametrize("D,Lk", [(64, 300), (128, 300), (64, 40), (128, 40)])
def test_float16_infinite_gradients_stay_where_they_belong(D, Lk):
    """An overflowed row of dO (a loss scale too large) is seen in its own dq, in dk and in dv, and leaves the other rows' dq alone."""
    g = _gen(73)
    q, k, v, do = (_randn(g, 1, n, 1, D, dtype=torch.float16) for n in (90, Lk, Lk, 90))
    clean = _call(q, k, v, do)
    do[0, 33, 0, 5] = math.inf
    got = _call(q, k, v, do)
    assert not torch.isfinite(got[1][0, 33]).any() and not torch.isfinite(got[2]).all() and not torch.isfinite(got[3][..., 5]).any()
    rest = torch.arange(90, device=_dev()) != 33
    assert torch.equal(got[1][:, rest], clean[1][:, rest]) and torch.equal(got[0], clean[0])


MANY_ROWS = [(1, 4000, 12, 4, 1, 128, 0), (1, 4000, 12, 4, 1, 64, 4), (1, 1000, 300, 8, 1, 64, 12), (1, 600, 40, 4, 1, 41, 0), (2, 2100, 65, 2, 2, 72, 0), (1, 40, 200, 64, 1, 64, 0),
             (1, 33, 130, 96, 2, 128, 13), (3, 1111, 1, 2, 1, 32, 0), (1, 2000, 700, 2, 1, 100, 7)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Lq,Lk,H,E,D,groups", MANY_ROWS)
def test_many_rows_over_few_keys(dtype, B, Lq, Lk, H, E, D, groups):
    """dK and dV of few keys: the rows are dealt to several workgroups, and their parts added up."""
    g = _gen(75)
    q, k, v, do = (_randn(g, *s, dtype=dtype) for s in ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D), (B, Lq, H, D)))
    keep = None
    if groups:
        keep = torch.rand(B, groups, generator=g, device=_dev()) < 0.6
        keep[0, 0], keep[0, 1] = True, False
    want, var = _sizes(q, k, v, do, D ** -0.5, keep)
    got = _call(q, k, v, do, keep)
    _check(got, want, var, dtype)
    if groups:
        gone = ~keep.repeat_interleave(Lk // groups, 1)
        assert not got[2][gone].any() and not got[3][gone].any()
    assert all(torch.equal(a, b) for a, b in zip(_call(q, k, v, do, keep), got))   # bit-reproducible


def test_many_rows_over_few_keys_in_graphs():
    """The parts' memory is the graph's own: two graphs replayed in turn, eager calls between."""
    B, Lq, Lk, H, E, D, _ = MANY_ROWS[2]
    shapes = ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D), (B, Lq, H, D))
    inputs = lambda n: [_randn(_gen(n + 100 * k), *s, dtype=torch.bfloat16) for k, s in enumerate(shapes)]  # noqa: E731
    static = [inputs(1), inputs(2)]
    _call(*static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_call(*s))
    for turn in range(3):
        now = [inputs(10 + 2 * turn + k) for k in range(2)]
        for n, s in zip(now, static):
            for a, b in zip(s, n):
                a.copy_(b)
        for graph in graphs:
            graph.replay()
        eager = [_call(*n) for n in now]
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
