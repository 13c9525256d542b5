"""The tokens of rendered views: what a network over the views' patches does with them after the renderer and the regulariser, as HIP kernels
with their backward passes (`mvr_rotate_tokens_*`, `mvr_attend_tokens_*`, `mvr_add_norm_tokens_*`, include/mvr.h).

    rotary = TokenRotary((8, 8, 8, 8), periods=(360.0, 360.0, None, None))
    positions = token_positions(azim, elev, 14, 14)             # (B, V*14*14, 4), gradient to the cameras
    q, k = rotary(q, positions), rotary(k, positions)           # (B, L, heads, D)
    out = attend_tokens(q, k, v, keep=scale.view(B, V) != 0)    # views dropped by draw_regularization are left out
    x, h = add_norm_tokens(x, proj(out), weight, scale=scale)   # ... and keep their residual

Tokens are ordered view by view: l = (v * rows + row) * cols + col.  All tensors of a call live on one GPU; the work goes to that GPU's current
stream, memory comes from torch's allocator, nothing synchronises.  Arguments that do not fit raise ValueError, tensors that are not on the GPU
RuntimeError.  Gradients repeat bit by bit; they cannot be differentiated again, and there is no forward mode: both raise.

A step may be captured into a HIP graph, backward included, if its leaves are made (detached) inside the capture or no eager graph of the same leaves
is alive: torch would otherwise hand the capture's gradients to that graph's stream."""
import math

import torch
from torch import nn

from . import _lib


# ---------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------

def token_positions(azim, elev, rows, cols):
    """(B, V * rows * cols, 4) float32 positions of the patches of V views: the view's azimuth and elevation in degrees (as the renderer takes
    them; differentiable), the patch's row and column."""
    if azim.dim() != 2 or azim.shape != elev.shape:
        raise ValueError("azim and elev are (B, V) tensors of one shape")
    B, V = azim.shape
    r = torch.arange(rows, device=azim.device, dtype=torch.float32)[:, None].expand(rows, cols)
    c = torch.arange(cols, device=azim.device, dtype=torch.float32)[None, :].expand(rows, cols)
    views = torch.stack((azim, elev), -1).to(torch.float32)[:, :, None, None, :].expand(B, V, rows, cols, 2)
    patches = torch.stack((r, c), -1).expand(B, V, rows, cols, 2)
    return torch.cat((views, patches), -1).reshape(B, V * rows * cols, 4)


class TokenRotary(nn.Module):
    """Rotary positions with several axes.  `sections`: pairs of each axis (1 to 4 axes; twice their sum at most the head dimension, the rest
    of a head is left as it is).  An axis with a period (cameras' angles: 360 degrees) turns its pairs by whole harmonics — 1, 2, ... turns per
    period, so that positions a period apart are the same place; one without (None or 0) by a geometric ladder of radians per unit,
    base ** (-j / n).  Pairs are (i, i + sum) of a head, or (2 i, 2 i + 1) when `interleaved`.

    `forward(x, positions)`: x (B, L, H, D) float32, float16 or bfloat16, with any strides whose last dimension is contiguous (a slice of a
    joint projection, queries and keys side by side); positions (B, L, axes), (1, L, axes) or (L, axes), taken as float32.  Differentiable
    with respect to both; angles are formed in 64 bits."""

    def __init__(self, sections, base=100.0, periods=None, interleaved=False):
        super().__init__()
        sections = [int(s) for s in sections]
        periods = [None] * len(sections) if periods is None else list(periods)
        if not 1 <= len(sections) <= 4 or min(sections) < 1 or sum(sections) > 128:
            raise ValueError("1 to 4 sections of at least one pair each, 128 pairs at most")
        if len(periods) != len(sections) or any(p is not None and not (p >= 0 and math.isfinite(p)) for p in periods):
            raise ValueError("one period (or None) per section")
        if not (base > 0 and math.isfinite(base)):
            raise ValueError("base must be positive")
        self.sections, self.interleaved, self.pairs = tuple(sections), bool(interleaved), sum(sections)
        turns = []
        for n, p in zip(sections, periods):
            turns += [(j + 1) / p if p else float(base) ** (-j / n) / (2 * math.pi) for j in range(n)]
        self.turns = tuple(turns)   # turns per unit of position, pair by pair

    def extra_repr(self):
        return "sections=%s, interleaved=%s" % (self.sections, self.interleaved)

    def forward(self, x, positions):
        return _lib.token_op().rotate(x, positions, self.turns, self.sections, self.interleaved)


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------

def attend_tokens(q, k, v, keep=None, scale=None):
    """softmax(scale q k^T) v over the kept keys: q (B, Lq, H, D), k and v (B, Lk, Hkv, D) float16 or bfloat16, D at most 128, H a multiple of
    Hkv (consecutive heads share a key/value head); any strides whose last dimension is contiguous.  scale: D ** -0.5 by default.

    keep: (B, G) with G a divisor of Lk, non-zero where the Lk / G consecutive keys of a group stay — one entry per key, or one per view
    (`draw_regularization`'s scale, viewed as (B, V)).  Of keys that are left out nothing enters the output, whatever they hold, and they get
    gradient 0; a query without any key left gets 0.  Returns (B, Lq, H, D), differentiable with respect to q, k and v: the backward recomputes
    the probabilities."""
    return _lib.token_op().attend(q, k, v, keep, scale)


# ---------------------------------------------------------------------------------------------
# norms around a block
# ---------------------------------------------------------------------------------------------

def add_norm_tokens(residual, branch, weight, bias=None, post_weight=None, gate=None, scale=None, kind="rms", eps=1e-6):
    """The end of one block and the norm in front of the next, one pass:

        n = N(branch) * post_weight   (branch itself without post_weight)
        y = residual + scale * gate * n
        z = N(y) * weight + bias

    N divides a row (the last dimension, at most 8192 wide) by sqrt(mean square + eps), with kind "layer" after taking its mean off.
    Returns (y, z): the residual stream, in its own type, and the next block's input, in the branch's.

    residual, branch: one shape (..., D); float32, float16 or bfloat16 alike, or a float32 residual with a 16-bit branch.  weight, bias,
    post_weight: (D,).  gate: (D,), or one row per leading index: (B, D) or (B, 1, D) with residual (B, L, D).  The four share one type.
    scale: a number, or float32 draws for equal runs of rows in memory order — `draw_regularization`'s scale, one per view: a row whose
    scale is 0 keeps its residual, its branch is not read and gets gradient 0.  Differentiable with respect to everything but scale."""
    if kind not in ("rms", "layer"):
        raise ValueError("kind is 'rms' or 'layer'")
    draws, number = (scale, 1.0) if torch.is_tensor(scale) else (None, 1.0 if scale is None else float(scale))
    return tuple(_lib.token_op().add_norm(residual, branch, weight, bias, post_weight, gate, draws, number, kind == "layer", eps))
