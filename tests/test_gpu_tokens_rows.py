"""-m gpu: the norms around a block over as many rows as real batches have, so that every wave and workgroup goes through several (the next row's loads,
its draw and its dropped branch carried along, both LDS buffers in turn), with remainders, and with more gate groups than there are workgroups.

Tolerances, element by element: one rounding of the result's own type, and 32-bit arithmetic against the absolute values that enter it.  With
hats for normed rows, h = |hat| + 1 bounds a hat and what the row's mean and deviation are off by (mean |hat| <= 1): a row's sum is a chain of at
most 32 + 6 + 8 additions, two of them and a square root, division and products make 100 2^-24; the backward's two further means 300 in all.  A column sum adds a
chain of at most 300 rows and partial lines (300 2^-24 of the absolute sum)."""
import pytest
import torch

from mvtn_amd import tokens

from gpu_helpers import _dev
from test_gpu_tokens import U32, _gen, _norm64, _randn, _tiny, _u

pytestmark = pytest.mark.gpu


def _room(t, kind, rows, dy, dz, eps=1e-6):
    """The absolute sums of what enters each result, by name."""
    def of(x):
        x = x - x.mean(-1, keepdim=True) if kind == "layer" else x
        r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        return (x * r).abs() + 1, r
    d = {k: v.detach().double() for k, v in t.items() if torch.is_tensor(v)}
    s = torch.ones((), dtype=torch.float64, device=_dev()) if rows is None else rows
    gate = d["gate"] if d.get("gate") is not None else torch.ones((), dtype=torch.float64, device=_dev())
    gate = (gate[:, None] if gate.dim() == 2 else gate).abs()
    branch = torch.where(s == 0, torch.zeros_like(d["branch"]), d["branch"])
    post = d["post"].abs() if "post" in d else torch.ones((), dtype=torch.float64, device=_dev())
    ha, ra = of(branch) if "post" in d else (branch.abs(), None)
    y = d["residual"].abs() + s * gate * post * ha
    wy, _, _ = _norm64(t, kind, eps, rows)
    hy, ry = of(wy.detach())
    w = d["weight"].abs()
    hz = hy + y * ry
    z = hz * w + (d["bias"].abs() if "bias" in d else 0)
    gz = dz.double().abs() * w
    dyt = dy.double().abs() + ry * (gz + gz.mean(-1, keepdim=True) + hz * (gz * hz).mean(-1, keepdim=True))
    dn = s * gate * dyt
    dp = dn * post
    db = ra * (dp + dp.mean(-1, keepdim=True) + ha * (dp * ha).mean(-1, keepdim=True)) if "post" in d else dp
    every = (0, 1)
    dgate = s * post * ha * dyt
    return dict(y=y, z=z, residual=dyt, branch=torch.where(s == 0, torch.zeros_like(db), db), weight=(dz.double().abs() * hz).sum(every), bias=dz.double().abs().sum(every),
                post=(dn * ha).sum(every), gate=dgate.sum(1) if "gate" in d and d["gate"].dim() == 2 else dgate.sum(every))


TYPES = [("float32",) * 3, ("bfloat16",) * 3, ("float16",) * 3, ("float32", "bfloat16", "float32"), ("float32", "float16", "float32")]
ROWS = [
    # B, L, D, kind, post, gate, views
    (3, 5001, 65, "layer", True, "object", 3), (3, 5001, 513, "rms", True, "channel", 5001), (2, 6007, 768, "layer", True, "object", 0),
    (3, 2000, 1024, "rms", False, "object", 20), (3, 2000, 2052, "layer", True, None, 8), (1, 701, 4097, "rms", True, "channel", 701),
    (2, 350, 8192, "layer", True, "object", 7),
    (1500, 9, 40, "rms", True, "object", 3),      # more gate groups than workgroups, one wave a row
    (1100, 5, 900, "layer", False, "object", 5),  # ... and one workgroup a row
]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("B,L,D,kind,post,gate,views", ROWS)
def test_norms_over_many_rows(types, B, L, D, kind, post, gate, views):
    r, b, p = (getattr(torch, t) for t in types)
    g = _gen(D + L)
    t = {"residual": _randn(g, B, L, D, dtype=r) * 2 + 0.1, "branch": _randn(g, B, L, D, dtype=b) + 0.1, "weight": 1 + 0.2 * _randn(g, D, dtype=p)}
    if kind == "layer":
        t["bias"] = 0.2 * _randn(g, D, dtype=p)
    if post:
        t["post"] = 1 + 0.2 * _randn(g, D, dtype=p)
    if gate:
        t["gate"] = _randn(g, *((B, D) if gate == "object" else (D,)), dtype=p)
    draws = rows = None
    if views:   # dropped and kept views in turn within one wave's rows; what a dropped row's branch holds stays out
        draws = (torch.rand(B, views, generator=g, device=_dev()) >= 0.4).float() / 0.6
        draws[0, 0], draws[-1, -1] = 0.0, 1 / 0.6
        rows = draws.double().repeat_interleave(L // views, 1)[..., None]
    dy, dz = _randn(g, B, L, D, dtype=r), _randn(g, B, L, D, dtype=b)
    wy, wz, w = _norm64(t, kind, 1e-6, rows)
    want = dict(zip(t, torch.autograd.grad((wy, wz), [w[k] for k in t], (dy.double(), dz.double()))))
    want.update(y=wy.detach(), z=wz.detach())
    room = _room(t, kind, rows, dy, dz)
    leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
    if views:
        with torch.no_grad():
            leaves["branch"][(rows == 0)[..., 0]] = float("nan")
    y, z = tokens.add_norm_tokens(leaves["residual"], leaves["branch"], leaves["weight"], leaves.get("bias"), post_weight=leaves.get("post"), gate=leaves.get("gate"),
                                  scale=draws, kind=kind)
    got = dict(zip(t, torch.autograd.grad((y, z), list(leaves.values()), (dy, dz))))
    got.update(y=y.detach(), z=z.detach())
    for name, a in got.items():
        n = 100 if name in "yz" else 300 if name in ("residual", "branch") else 600
        far = (a.double() - want[name]).abs()
        bound = _u(a.dtype) * want[name].abs() + n * U32 * room[name] + _tiny(a.dtype)
        assert (far <= bound).all(), (name, float((far / bound).max()))
    if views:
        gone = (rows == 0)[..., 0]
        assert torch.equal(y[gone], t["residual"][gone]) and not got["branch"][gone].any()
