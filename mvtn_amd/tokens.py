"""The tokens of rendered views: what a network over the views' patches does with them after the renderer and the regulariser, as HIP kernels
with their backward passes (`mvr_rotate_tokens_*`, `mvr_attend_tokens_*`, `mvr_add_norm_tokens_*`, include/mvr.h).

    rotary = TokenRotary((8, 8, 8, 8), periods=(360.0, 360.0, None, None))
    positions = token_positions(azim, elev, 14, 14)             # (B, V*14*14, 4), gradient to the cameras
    q, k = rotary(q, positions), rotary(k, positions)           # (B, L, heads, D)
    out = attend_tokens(q, k, v, keep=scale.view(B, V) != 0)    # views dropped by draw_regularization are left out
    x, h = add_norm_tokens(x, proj(out), weight, scale=scale)   # ... and keep their residual

Tokens are ordered view by view: l = (v * rows + row) * cols + col.  All tensors live on one GPU; the calls go to its current stream, allocate
through torch and never synchronise."""
import ctypes
import functools
import math

import torch
from torch import nn

from . import _lib
from .functional import _raw_stream, _require_cuda

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # MVR_TYPE_*


def _ptr(t):
    return None if t is None else t.data_ptr()


def _same_device(*ts):
    _require_cuda(*ts)
    dev = ts[0].device
    for t in ts:
        if t is not None and t.device != dev:
            raise RuntimeError("mvtn_amd.tokens: all tensors must be on one GPU (%s and %s)" % (dev, t.device))


def _call(name, device, *args):
    """lib.name(*args, stream) on `device`'s current stream, whichever device is current."""
    fn = getattr(_lib.load(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device.index))
    if rc:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=64)
def _doubles(values):
    return (ctypes.c_double * len(values))(*values)


def _rows_contiguous(t):
    """`t` with its last dimension's elements side by side (a copy only where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


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

    def _params(self, x, grad, positions):
        B, L, H, D = x.shape
        p = _lib.RotaryParams(B, L, H, D, _TYPES[x.dtype], len(self.sections), self.sections, int(self.interleaved), 0)
        p.x_stride[:] = x.stride()[:3]
        if grad is not None:
            p.grad_stride[:] = grad.stride()[:3]
        p.position_stride[:] = positions.stride()[:2]
        return p

    def forward(self, x, positions):
        if x.dim() != 4:
            raise ValueError("x is (B, L, H, D)")
        B, L, H, D = x.shape
        if x.dtype not in _TYPES:
            raise ValueError("x must be float32, float16 or bfloat16, not %s" % x.dtype)
        if 2 * self.pairs > D or D > 256 or (self.interleaved and D % 2):
            raise ValueError("%d pairs do not fit a head of %d (at most 256, even when interleaved)" % (self.pairs, D))
        axes = len(self.sections)
        if positions.dim() not in (2, 3) or positions.shape[-2:] != (L, axes) or (positions.dim() == 3 and positions.shape[0] not in (1, B)):
            raise ValueError("positions are (B, L, axes), (1, L, axes) or (L, axes) with L = %d and %d axes" % (L, axes))
        _same_device(x, positions)
        positions = positions.to(torch.float32).expand(B, L, axes)
        if torch.is_grad_enabled() and (x.requires_grad or positions.requires_grad):
            return _Rotate.apply(x, positions, self)
        return self._run(x, positions)

    def _run(self, x, positions):
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if out.numel():
            x, positions = _rows_contiguous(x), _rows_contiguous(positions)
            _call("mvr_rotate_tokens_forward", x.device, self._params(x, None, positions), _doubles(self.turns), x.data_ptr(), positions.data_ptr(), out.data_ptr())
        return out


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, rotary):
        ctx.rotary = rotary
        ctx.shape, ctx.dtype = x.shape, x.dtype
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, positions)
        return rotary._run(x, positions)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, positions = ctx.saved_tensors
        gx = torch.empty(ctx.shape, dtype=ctx.dtype, device=grad.device)
        gpos = torch.empty(positions.shape, dtype=torch.float32, device=grad.device) if x is not None else None
        if gx.numel():
            grad, positions = _rows_contiguous(grad), _rows_contiguous(positions)
            x = None if x is None else _rows_contiguous(x)
            params = ctx.rotary._params(grad if x is None else x, grad, positions)
            _call("mvr_rotate_tokens_backward", grad.device, params, _doubles(ctx.rotary.turns), _ptr(x), positions.data_ptr(), grad.data_ptr(),
                  gx.data_ptr(), _ptr(gpos))
        elif gpos is not None:
            gpos.zero_()
        return gx, gpos, None


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------

def attend_tokens(q, k, v, keep=None, scale=None):
    """softmax(scale q k^T) v over the kept keys: q (B, Lq, H, D), k and v (B, Lk, Hkv, D) float16 or bfloat16, D at most 128, H a multiple of
    Hkv (consecutive heads share a key/value head); any strides whose last dimension is contiguous.  scale: D ** -0.5 by default.

    keep: (B, G) with G a divisor of Lk, non-zero where the Lk / G consecutive keys of a group stay — one entry per key, or one per view
    (`draw_regularization`'s scale, viewed as (B, V)).  Keys that are left out are not read and get gradient 0; a query without any key
    left gets 0.  Returns (B, Lq, H, D), differentiable with respect to q, k and v: the backward recomputes the probabilities."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q is (B, Lq, H, D), k and v are (B, Lk, Hkv, D)")
    B, Lq, H, D = q.shape
    Lk, E = k.shape[1:3]
    if k.shape[0] != B or k.shape[3] != D or not 1 <= D <= 128:
        raise ValueError("q, k and v share the batch and a head size of 1 to 128")
    if E < 1 or H < 1 or H % E:
        raise ValueError("%d heads are not a multiple of %d key/value heads" % (H, E))
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v share one type of float16, bfloat16")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    if keep is not None:
        if keep.dim() != 2 or keep.shape[0] != B or keep.shape[1] < 1 or Lk % keep.shape[1]:
            raise ValueError("keep is (B, G) with G a divisor of the %d keys" % Lk)
        if keep.requires_grad:
            raise ValueError("keep is a mask: it gets no gradient")
    _same_device(q, k, v, keep)
    if keep is not None:
        keep = (keep if keep.dtype in (torch.bool, torch.uint8) else keep != 0).contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attend.apply(q, k, v, keep, scale)
    return _attend(q, k, v, keep, scale, False)[0]


def _attend_params(q, k, v, keep, scale):
    B, Lq, H, D = q.shape
    p = _lib.AttendParams(B, Lq, k.shape[1], H, k.shape[2], D, _TYPES[q.dtype], 0 if keep is None else keep.shape[1])
    p.q_stride, p.k_stride, p.v_stride, p.scale = q.stride()[:3], k.stride()[:3], v.stride()[:3], scale
    return p


def _attend(q, k, v, keep, scale, training):
    q, k, v = _rows_contiguous(q), _rows_contiguous(k), _rows_contiguous(v)
    B, Lq, H, D = q.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, Lq, dtype=torch.float32, device=q.device) if training else None
    if k.shape[1] == 0:
        out.zero_()
    elif out.numel():
        params = _attend_params(q, k, v, keep, scale)
        size = _lib.load().mvr_attend_tokens_workspace_bytes(params, 0)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _call("mvr_attend_tokens_forward", q.device, params, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(keep), out.data_ptr(), _ptr(lse),
              _ptr(ws), size)
    return out, (q, k, v, keep, out, lse)


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, keep, scale):
        out, kept = _attend(q, k, v, keep, scale, True)
        ctx.scale = scale
        ctx.save_for_backward(*kept)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        q, k, v, keep, out, lse = ctx.saved_tensors
        gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if out.numel() and k.shape[1]:
            grad = _rows_contiguous(grad)
            params = _attend_params(q, k, v, keep, ctx.scale)
            params.grad_stride = grad.stride()[:3]
            size = _lib.load().mvr_attend_tokens_workspace_bytes(params, 1)
            ws = torch.empty(size, dtype=torch.uint8, device=q.device)
            _call("mvr_attend_tokens_backward", q.device, params, q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(keep), out.data_ptr(),
                  lse.data_ptr(), grad.data_ptr(), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), ws.data_ptr(), size)
        else:
            for t in (gq, gk, gv):
                t.zero_()
        return gq, gk, gv, None, None


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
    draw is 0 keeps its residual, its branch is not read and gets gradient 0.  Differentiable with respect to everything but scale."""
    D = residual.shape[-1] if residual.dim() else 0
    if residual.shape != branch.shape or residual.dim() < 2:
        raise ValueError("residual and branch are of one shape (..., D)")
    if not 1 <= D <= 8192:
        raise ValueError("rows of 1 to 8192 elements")
    if residual.dtype not in _TYPES or branch.dtype not in _TYPES or residual.dtype not in (branch.dtype, torch.float32):
        raise ValueError("residual and branch share one type of float32, float16, bfloat16, or the residual is float32")
    if kind not in ("rms", "layer"):
        raise ValueError("kind is 'rms' or 'layer'")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError("eps must not be negative")
    for t in (weight, bias, post_weight):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError("weight, bias and post_weight are (%d,)" % D)
    rows = residual.numel() // D
    groups = 0
    if gate is not None:
        lead = list(gate.shape[:-1])
        while lead and lead[-1] == 1:
            lead.pop()
        if not gate.dim() or gate.shape[-1] != D or lead != list(residual.shape[:len(lead)]) or (len(lead) and len(lead) >= residual.dim() - 1):
            raise ValueError("gate is (D,), or has one row per leading index of the residual ((B, D) or (B, 1, D) for (B, L, D)); a gate of every "
                             "element belongs into the branch")
        groups = math.prod(lead)
        if groups > 65000:
            raise ValueError("at most 65000 rows of gates")
    params = [t for t in (weight, bias, post_weight, gate) if t is not None]
    if any(t.dtype != weight.dtype for t in params) or weight.dtype not in _TYPES:
        raise ValueError("weight, bias, post_weight and gate share one type of float32, float16, bfloat16")
    draws, number = (scale, 1.0) if torch.is_tensor(scale) else (None, 1.0 if scale is None else float(scale))
    if draws is not None:
        if draws.requires_grad:
            raise ValueError("scale holds draws: it gets no gradient (put what is learned into gate)")
        if draws.numel() < 1 or rows % draws.numel():
            raise ValueError("scale has %d draws, which do not divide the %d rows" % (draws.numel(), rows))
        draws = draws.to(torch.float32).contiguous()
    _same_device(residual, branch, draws, *params)
    cfg = _lib.NormParams(rows, D, _TYPES[residual.dtype], _TYPES[branch.dtype], _TYPES[weight.dtype], int(kind == "layer"), 0, groups,
                          0 if draws is None else draws.numel(), number, float(eps))
    if torch.is_grad_enabled() and any(t.requires_grad for t in [residual, branch] + params):
        return _AddNorm.apply(residual, branch, weight, bias, post_weight, gate, draws, cfg)
    return _add_norm(residual, branch, weight, bias, post_weight, gate, draws, cfg, False)[:2]


def _add_norm(residual, branch, weight, bias, post, gate, draws, cfg, training):
    residual, branch = residual.contiguous(), branch.contiguous()
    weight, bias, post, gate = (None if t is None else t.contiguous() for t in (weight, bias, post, gate))
    y, z = torch.empty_like(residual), torch.empty_like(branch)
    stats = torch.empty(cfg.rows, 4, dtype=torch.float32, device=y.device) if training else None
    if cfg.rows:
        _call("mvr_add_norm_tokens_forward", y.device, cfg, residual.data_ptr(), branch.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(post),
              _ptr(gate), _ptr(draws), y.data_ptr(), z.data_ptr(), _ptr(stats))
    return y, z, (y, branch, weight, post, gate, draws, stats)


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, residual, branch, weight, bias, post, gate, draws, cfg):
        y, z, kept = _add_norm(residual, branch, weight, bias, post, gate, draws, cfg, True)
        ctx.set_materialize_grads(False)
        ctx.cfg = cfg
        ctx.save_for_backward(*kept)
        return y, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy, gz):
        y, branch, weight, post, gate, draws, stats = ctx.saved_tensors
        if gy is None and gz is None:
            return (None,) * 8
        cfg, need = ctx.cfg, ctx.needs_input_grad
        gy, gz = (None if t is None else t.contiguous() for t in (gy, gz))
        gr, gb = torch.empty_like(y), torch.empty_like(branch)
        gw, gbias = (torch.empty_like(weight) if n else None for n in need[2:4])
        gpost, ggate = (torch.empty_like(t) if n else None for t, n in ((post, need[4]), (gate, need[5])))
        if cfg.rows:
            ws = None
            if any(need[2:6]):
                ws = torch.empty(_lib.load().mvr_add_norm_tokens_workspace_bytes(cfg), dtype=torch.uint8, device=y.device)
            _call("mvr_add_norm_tokens_backward", y.device, cfg, y.data_ptr(), branch.data_ptr(), weight.data_ptr(), _ptr(post), _ptr(gate),
                  _ptr(draws), stats.data_ptr(), _ptr(gy), _ptr(gz), gr.data_ptr(), gb.data_ptr(), _ptr(gw), _ptr(gbias), _ptr(gpost),
                  _ptr(ggate), _ptr(ws), 0 if ws is None else ws.numel())
        else:
            for t in (gw, gbias, gpost, ggate):
                if t is not None:
                    t.zero_()
        return (gr, gb, gw, gbias, gpost, ggate, None, None)
