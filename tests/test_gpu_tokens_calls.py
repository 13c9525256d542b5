"""-m gpu: calls of the operators on view tokens that programs make now and then: infinities on the way back, gradients of gradients, traced and
replayed calls, sizes and grids past the first round."""
import math

import pytest
import torch

from mvtn_amd import tokens

from gpu_helpers import _dev
from test_gpu_tokens import _gen, _randn

pytestmark = pytest.mark.gpu


def _attention(q, k, v, do, keep=None):
    """(out, dq, dk, dv)"""
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = tokens.attend_tokens(*leaves, keep=keep)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, do))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq,Lk,H,E,D,groups", [(90, 40, 2, 2, 64, 8), (90, 40, 2, 1, 128, 8), (70, 300, 2, 1, 64, 60), (70, 300, 2, 2, 128, 60), (33, 130, 1, 1, 33, 26)])
@pytest.mark.parametrize("which", ["do", "q"])
def test_dropped_keys_get_zero_beside_infinite_rows(dtype, Lq, Lk, H, E, D, groups, which):
    """A loss scale that overflowed, or a broken query: the kept keys' gradients show it, those of left-out keys in the same tile are 0."""
    g = _gen(90)
    q, k, v, do = (_randn(g, *s, dtype=dtype) for s in ((2, Lq, H, D), (2, Lk, E, D), (2, Lk, E, D), (2, Lq, H, D)))
    keep = torch.rand(2, groups, generator=g, device=_dev()) < 0.6
    keep[0, 0], keep[0, 1] = True, False
    t = do if which == "do" else q
    t[0, 7, 0, 3], t[0, 8, 0, 4] = math.inf, math.nan
    gone = ~keep.repeat_interleave(Lk // groups, 1)
    got = _attention(q, k, v, do, keep)
    assert not torch.isfinite(got[2][0][~gone[0]][:, 0]).all() and not torch.isfinite(got[3][0][~gone[0]][:, 0]).all()
    assert not got[2][gone].any() and not got[3][gone].any()   # (any() of a NaN is true)
