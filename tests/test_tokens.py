"""CPU (-m "not gpu"): the operators on view tokens (mvtn_amd/tokens.py) — what they refuse before anything reaches the GPU, through Python
and through the C ABI, and the host-side pieces (positions, frequencies)."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

from mvtn_amd import _lib, tokens


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_token_positions_order_and_gradient():
    B, V, R, C = 2, 3, 4, 5
    azim = torch.arange(6.0).reshape(B, V).requires_grad_()
    elev = (10 + torch.arange(6.0)).reshape(B, V).requires_grad_()
    p = tokens.token_positions(azim, elev, R, C)
    assert p.shape == (B, V * R * C, 4) and p.dtype == torch.float32
    for b, v, r, c in ((0, 0, 0, 0), (1, 2, 3, 4), (0, 1, 2, 3)):
        assert p[b, (v * R + r) * C + c].tolist() == [float(azim[b, v].detach()), float(elev[b, v].detach()), r, c]
    p[..., 0].sum().backward()
    assert (azim.grad == R * C).all()
    expanded = torch.zeros(4).expand(3, 4)   # the selectors' stride-(0, 1) views
    assert tokens.token_positions(expanded, expanded, 2, 2).shape == (3, 16, 4)
    with pytest.raises(ValueError):
        tokens.token_positions(azim, elev[:1], 2, 2)


def test_rotary_frequencies_and_copies():
    r = tokens.TokenRotary((2, 3), base=100.0, periods=(360.0, None))
    want = [1 / 360, 2 / 360] + [100.0 ** (-j / 3) / (2 * math.pi) for j in range(3)]
    assert r.pairs == 5 and max(abs(a - b) for a, b in zip(r.turns, want)) <= 1e-18
    assert pickle.loads(pickle.dumps(copy.deepcopy(r))).turns == r.turns
    assert not list(r.parameters()) and not r.state_dict()


@pytest.mark.parametrize("args", [dict(sections=()), dict(sections=(1, 1, 1, 1, 1)), dict(sections=(0, 2)), dict(sections=(129,)),
                                  dict(sections=(2, 2), periods=(360,)), dict(sections=(2,), periods=(-1,)), dict(sections=(2,), base=0.0),
                                  dict(sections=(2,), periods=(math.inf,))])
def test_rotary_refuses_bad_plans(args):
    with pytest.raises(ValueError):
        tokens.TokenRotary(**args)


def test_rotary_refuses_bad_calls():
    r = tokens.TokenRotary((2, 2))
    pos = _x(3, 2)
    for x, p in ((_x(2, 3, 8), pos), (_x(2, 3, 1, 8, dtype=torch.float64), pos), (_x(2, 3, 1, 6), pos), (_x(2, 3, 1, 300), pos),
                 (_x(2, 3, 1, 8), _x(4, 2)), (_x(2, 3, 1, 8), _x(3, 3)), (_x(2, 3, 1, 8), _x(3, 3, 2)), (_x(2, 3, 1, 8), _x(2))):
        with pytest.raises(ValueError):
            r(x, p)
    with pytest.raises(ValueError):
        tokens.TokenRotary((2, 2), interleaved=True)(_x(2, 3, 1, 9), pos)
    with pytest.raises(RuntimeError, match="GPU"):   # there is no CPU fallback
        r(_x(2, 3, 1, 8), pos)


def test_add_norm_refuses_bad_calls():
    f = tokens.add_norm_tokens
    x, w = _x(2, 6, 8), _x(8)
    half = torch.float16
    for args, kw in (((x, _x(2, 6, 9), w), {}), ((_x(8), _x(8), w), {}), ((x, x, _x(9)), {}), ((x, x, w), dict(bias=_x(1, 8))),
                     ((x, x, w), dict(post_weight=_x(7))), ((x, x, w), dict(kind="batch")), ((x, x, w), dict(eps=-1.0)), ((x, x, w), dict(eps=math.nan)),
                     ((x.to(half), x, w), {}), ((x.to(half), x.to(torch.bfloat16), w), {}), ((x.double(), x.double(), w), {}),
                     ((x, x, w), dict(bias=_x(8, dtype=half))), ((x, x, w.double()), {}),
                     ((x, x, w), dict(gate=_x(3, 8))), ((x, x, w), dict(gate=_x(2, 6, 8))), ((x, x, w), dict(gate=_x(1, 6, 8))), ((x, x, w), dict(gate=_x(2, 7))),
                     ((x, x, w), dict(gate=_x(()))), ((x, x, w), dict(scale=_x(5))), ((x, x, w), dict(scale=_x(0))),
                     ((x, x, w), dict(scale=_x(2).requires_grad_())), ((_x(2, 6, 8193), _x(2, 6, 8193), _x(8193)), {}), ((_x(2, 0), _x(2, 0), _x(0)), {})):
        with pytest.raises(ValueError):
            f(*args, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        f(x, x, w)


def test_c_abi_refuses_before_any_launch():
    lib = _lib.load()
    p = 4096   # never dereferenced: every call below is refused on the host
    turns = (ctypes.c_double * 4)(1, 1, 1, 1)

    def rotary(**kw):
        r = _lib.RotaryParams(2, 3, 1, 8, 0, 2, (2, 2), 0, 0)
        for k, v in kw.items():
            setattr(r, k, v)
        return r
    bad = [dict(batch=0), dict(tokens=-1), dict(heads=0), dict(dim=0), dict(dim=257), dict(dim=6), dict(type=3), dict(axes=0), dict(axes=5),
           dict(sections=(ctypes.c_int32 * 4)(0, 4)), dict(reserved_=1), dict(dim=9, interleaved=1)]
    for kw in bad:
        assert lib.mvr_rotate_tokens_forward(rotary(**kw), turns, p, p, p + 64, None) == 1, kw
        assert lib.mvr_rotate_tokens_backward(rotary(**kw), turns, None, p, p, p + 64, None, None) == 1, kw
        assert b"mvr_rotate_tokens" in lib.mvr_last_error()
    assert lib.mvr_rotate_tokens_forward(rotary(), None, p, p, p + 64, None) == 1
    assert lib.mvr_rotate_tokens_forward(rotary(), turns, p, p, p, None) == 1            # in place
    assert lib.mvr_rotate_tokens_backward(rotary(), turns, p, p, p, p + 64, None, None) == 1   # x without grad_positions
    assert lib.mvr_rotate_tokens_backward(rotary(), turns, None, p, p, p + 64, p, None) == 1

    def norm(**kw):
        n = _lib.NormParams(12, 8, 0, 0, 0, 0, 0, 0, 0, 1.0, 1e-6)
        for k, v in kw.items():
            setattr(n, k, v)
        return n

    def forward(n, gate=None, scale=None, y=p + 64, z=p + 128):
        return lib.mvr_add_norm_tokens_forward(n, p, p + 32, p, None, None, gate, scale, y, z, None, None)

    def backward(n, ws=None, size=0, gate=None, gw=None, gy=p, gg=None, gp=None):
        return lib.mvr_add_norm_tokens_backward(n, p, p, p, None, gate, None, p, gy, None, p, p, gw, None, gp, gg, ws, size, None)
    for kw in (dict(rows=0), dict(dim=0), dict(dim=8193), dict(kind=2), dict(eps=-1.0), dict(gate_groups=5), dict(gate_groups=-1), dict(scale_groups=7),
               dict(param_type=9), dict(residual_type=-1), dict(reserved_=1)):
        assert forward(norm(**kw)) == 1 and lib.mvr_add_norm_tokens_workspace_bytes(norm(**kw)) == 0, kw
    assert forward(norm(residual_type=1)) == 4 and forward(norm(residual_type=1, branch_type=2)) == 4   # 16-bit stream under another type
    assert forward(norm(gate_groups=2)) == 1 and forward(norm(), gate=p) == 1 and forward(norm(scale_groups=2)) == 1 and forward(norm(), scale=p) == 1
    assert forward(norm(), y=p + 32) == 1 and forward(norm(), z=p) == 1 and forward(norm(), y=p + 64, z=p + 64) == 1
    need = lib.mvr_add_norm_tokens_workspace_bytes(norm())
    assert need > 0 and need % (4 * 8 * 4) == 0
    assert backward(norm(), gw=p) == 3 and backward(norm(), gw=p, ws=p, size=need - 1) == 3
    assert backward(norm(), gy=None) == 1 and backward(norm(), gg=p) == 1 and backward(norm(), gp=p) == 1
    assert lib.mvr_add_norm_tokens_forward(None, p, p, p, None, None, None, None, p, p, None, None) == 1


def test_attention_refuses_bad_calls():
    f, half = tokens.attend_tokens, torch.float16
    q = lambda *s, dtype=half: _x(*s, dtype=dtype)  # noqa: E731
    ok = (q(2, 3, 4, 8), q(2, 6, 2, 8), q(2, 6, 2, 8))
    for args, kw in (((q(2, 3, 8),) + ok[1:], {}), ((ok[0], ok[1], q(2, 5, 2, 8)), {}), ((ok[0], q(1, 6, 2, 8), q(1, 6, 2, 8)), {}),
                     ((ok[0], q(2, 6, 3, 8), q(2, 6, 3, 8)), {}), ((q(2, 3, 4, 129), q(2, 6, 2, 129), q(2, 6, 2, 129)), {}),
                     ((ok[0].float(), ok[1].float(), ok[2].float()), {}), ((ok[0], ok[1].bfloat16(), ok[2]), {}), (ok, dict(scale=0.0)), (ok, dict(scale=-1.0)),
                     (ok, dict(scale=math.nan)), (ok, dict(scale=math.inf)), (ok, dict(keep=_x(2, 4))), (ok, dict(keep=_x(1, 6))), (ok, dict(keep=_x(2, 0))),
                     (ok, dict(keep=_x(6))), (ok, dict(keep=_x(2, 6).requires_grad_())), ((q(2, 3, 4, 0), q(2, 6, 2, 0), q(2, 6, 2, 0)), {}),
                     ((ok[0], q(2, 6, 0, 8), q(2, 6, 0, 8)), {})):
        with pytest.raises(ValueError):
            f(*args, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        f(*ok)


def test_attention_c_abi_refuses_before_any_launch():
    lib = _lib.load()
    p = 4096

    def params(**kw):
        r = _lib.AttendParams(2, 3, 6, 4, 2, 8, 1, 0)
        r.scale = 1.0
        for k, v in kw.items():
            setattr(r, k, v)
        return r

    def forward(a, keep=None, out=p + 64, ws=None, size=0):
        return lib.mvr_attend_tokens_forward(a, p, p, p, keep, out, None, ws, size, None)

    def backward(a, ws=p, size=1 << 40, gq=p, keep=None):
        return lib.mvr_attend_tokens_backward(a, p, p, p, keep, p, p, p, gq, p, p, ws, size, None)
    for kw, code in ((dict(batch=0), 1), (dict(queries=0), 1), (dict(keys=-5), 1), (dict(heads=3), 1), (dict(kv_heads=0), 1), (dict(dim=0), 1), (dict(dim=129), 4),
                     (dict(type=0), 4), (dict(type=7), 4), (dict(keep_groups=4), 1), (dict(keep_groups=-1), 1), (dict(scale=0.0), 1), (dict(scale=math.nan), 1),
                     (dict(scale=math.inf), 1), (dict(reserved_=1), 1), (dict(keys=0x7FFFFFFF), 4), (dict(queries=0x7FFFFFFF, heads=4), 4)):
        assert forward(params(**kw)) == code and backward(params(**kw)) == code and lib.mvr_attend_tokens_workspace_bytes(params(**kw), 1) == 0, kw
        assert b"mvr_attend_tokens" in lib.mvr_last_error()
    assert forward(params(keep_groups=2)) == 1 and forward(params(), keep=p) == 1 and backward(params(), keep=p) == 1
    assert forward(params(), out=p) == 1 and backward(params(), gq=None) == 1
    assert backward(params(), ws=None) == 3 and backward(params(), size=lib.mvr_attend_tokens_workspace_bytes(params(), 1) - 1) == 3
    split = params(batch=1, queries=1, keys=4096, heads=2)   # few rows: the keys are split and the parts need room
    need = lib.mvr_attend_tokens_workspace_bytes(split, 0)
    assert need > 0 and forward(split, ws=p, size=need - 1) == 3 and lib.mvr_attend_tokens_workspace_bytes(params(), 0) == 0
