"""-m gpu: calls of the operators on view tokens that programs make now and then: infinities on the way back, gradients of gradients, traced and
replayed calls, sizes and grids past the first round."""
import itertools
import math

import pytest
import torch

from mvtn_amd import _lib, tokens

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


def test_a_penalty_on_gradients_is_noticed():
    """A gradient with create_graph and a constant gradient above it depends on the inputs all the same: its use in a loss fails, it is not a constant."""
    g = _gen(91)
    x, pos = _randn(g, 1, 4, 2, 8).requires_grad_(), _randn(g, 4, 1).requires_grad_()
    h, w = _randn(g, 1, 4, 2, 8, dtype=torch.bfloat16).requires_grad_(), _randn(g, 8).requires_grad_()
    v = _randn(g, 1, 4, 2, 8, dtype=torch.bfloat16).requires_grad_()
    rotary = tokens.TokenRotary((4,))
    for out, leaf in ((rotary(x, pos), x), (rotary(x, pos), pos), (tokens.attend_tokens(h, h, h), h), (tokens.attend_tokens(h.detach(), h, h.detach()), h),
                      (tokens.add_norm_tokens(x, x, w)[1], x), (tokens.add_norm_tokens(x.detach(), x.detach(), w.detach(), gate=w)[0], w)):
        first, = torch.autograd.grad(out.float().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated"):
            (out.float().sum() + first.float().square().sum()).backward()
    # gradients that do not depend on what requires grad are constants, and may be used as such
    for out, leaf in ((rotary(x, pos.detach()), x), (tokens.attend_tokens(h.detach(), h.detach(), v), v), (tokens.add_norm_tokens(x.detach(), x.detach(), w)[1], w)):
        first, = torch.autograd.grad(out.float().sum(), leaf, create_graph=True)
        assert not first.requires_grad
        leaf.grad = None
        (out.float().sum() + first.float().square().sum()).backward()
        assert torch.equal(leaf.grad, first)


def _operators(dtype=torch.bfloat16):
    """(call, inputs): each operator as a function of tensors alone."""
    g = _gen(92)
    rotary = tokens.TokenRotary((4, 4), periods=(360.0, None))
    draws = torch.tensor([[0.0, 2.0, 2.0], [2.0, 0.0, 2.0]], device=_dev())
    keep = torch.tensor([[1, 0, 1], [0, 1, 1]], device=_dev())
    r = lambda *s: _randn(g, *s, dtype=dtype)  # noqa: E731
    return [(rotary, [r(2, 90, 2, 24), _randn(g, 90, 2) * 20]),
            (lambda q, k, v: tokens.attend_tokens(q, k, v, keep=keep), [r(2, 40, 4, 64), r(2, 90, 2, 64), r(2, 90, 2, 64)]),
            (lambda x, a, w, p: tokens.add_norm_tokens(x, a, w, post_weight=p, scale=draws)[1], [r(2, 90, 72), r(2, 90, 72), r(72), r(72)])]


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("which", range(3))
def test_a_traced_call_runs_on_the_replays_stream(which):
    call, inputs = _operators()[which]
    want = call(*inputs)
    traced = torch.jit.trace(call, tuple(inputs), check_trace=False)
    late = torch.zeros_like(inputs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)   # (some 20 ms: a launch on another stream would read the zeros)
        late.copy_(inputs[0])
        got = traced(late, *inputs[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("which", range(3))
def test_a_backward_called_on_another_stream(which):
    """The gradients are computed on the forward's stream, as those of torch's operators, and handed over to the caller's."""
    call, inputs = _operators()[which]
    leaves = [t.requires_grad_() for t in inputs]
    out = call(*leaves)
    up = torch.ones_like(out)
    want = torch.autograd.grad(out, leaves, up, retain_graph=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late = torch.zeros_like(up).copy_(up)
        got = torch.autograd.grad(out, leaves, late)
        got = [t.clone() for t in got]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _step(call):
    """Forward and backward as one function of tensors: what is traced as a training step."""
    def step(up, *inputs):
        leaves = [t.detach().requires_grad_() for t in inputs]
        out = call(*leaves)
        return (out.detach(),) + torch.autograd.grad(out, leaves, up)
    return step


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("which", range(3))
def test_a_recorded_graph_computes(which, mode):
    """make_fx's graph of a call, and of a call with its backward, gives what the call gives, on other inputs than it was recorded with."""
    from torch.fx.experimental.proxy_tensor import make_fx
    call, inputs = _operators()[which]
    other = [t.flip(0) if t.dim() > 1 else t * 2 for t in inputs]
    graph = make_fx(call, tracing_mode=mode, _allow_non_fake_inputs=True)(*inputs)
    assert torch.equal(graph(*other), call(*other))
    up = torch.randn_like(call(*inputs))
    step = make_fx(_step(call), tracing_mode=mode, _allow_non_fake_inputs=True)(up, *inputs)
    assert all(torch.equal(a, b) for a, b in zip(step(up, *other), _step(call)(up, *other)))
    # the graph's inner operators carry gradients themselves
    leaves = [t.detach().requires_grad_() for t in inputs]
    want = torch.autograd.grad(call(*leaves), leaves, up)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(graph(*leaves), leaves, up), want))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("dynamic", [False, True])
@pytest.mark.parametrize("which", range(3))
def test_a_compiled_call_computes(which, dynamic):
    call, inputs = _operators()[which]
    torch._dynamo.reset()
    compiled = torch.compile(call, backend="aot_eager", dynamic=dynamic)
    for args in (inputs, [t.flip(0) if t.dim() > 1 else t * 2 for t in inputs]):
        assert torch.equal(compiled(*args), call(*args))
        leaves = [t.detach().requires_grad_() for t in args]
        out = compiled(*leaves)
        up = torch.randn_like(out)
        want = torch.autograd.grad(call(*leaves), leaves, up)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, up), want))


def test_every_operator_is_registered_whole():
    """torch's own check of a custom operator: schema, autograd, shapes without memory, tracing (of shapes that vary too)."""
    ops = torch.ops.mvr_tokens
    rotary, attend, norm = _operators()
    need = lambda ts: [t.detach().requires_grad_() for t in ts]  # noqa: E731
    x, pos = rotary[1]
    pos = pos.expand(2, 90, 2).contiguous()
    turns, sections = list(rotary[0].turns), list(rotary[0].sections)
    q, k, v = attend[1]
    keep = torch.tensor([[1, 0, 1], [0, 1, 1]], device=_dev()).bool()
    r, a, w, p = norm[1]
    draws = torch.tensor([[0.0, 2.0, 2.0], [2.0, 0.0, 2.0]], device=_dev())
    with torch.no_grad():
        out, rest, lse = ops.attend_training(q, k, v, keep, 0.125)
        stats = ops.add_norm_training(r, a, w, None, p, None, draws, 1.0, False, 1e-6)[2]
    for op, args in ((ops.rotate_forward, (*need((x, pos)), turns, sections, False)), (ops.rotate_backward, (x, x, pos, turns, sections, False)),
                     (ops.attend_forward, (*need((q, k, v)), keep, 0.125)), (ops.attend_training, (q, k, v, keep, 0.125)),
                     (ops.attend_backward, (q, q, k, v, keep, out, rest, lse, 0.125)),
                     (ops.add_norm_forward, (*need((r, a, w)), None, *need((p,)), None, draws, 1.0, False, 1e-6)),
                     (ops.add_norm_training, (r, a, w, None, p, None, draws, 1.0, False, 1e-6)),
                     (ops.add_norm_backward, (r, None, r, a, w, p, None, draws, stats, [1, 0, 1, 0], 1.0, False, 1e-6))):
        torch.library.opcheck(op.default, args)


def test_inner_operators_refuse_what_does_not_fit():
    """A graph that was edited, or a call around mvtn_amd.tokens: every way to the kernels checks shapes, types and devices."""
    ops = torch.ops.mvr_tokens
    (_, (x, pos)), (_, (q, k, v)), (_, (r, a, w, p)) = _operators()
    tokens._lib.token_op()
    pos = pos.expand(2, 90, 2).contiguous()
    keep = torch.ones(2, 3, device=_dev(), dtype=torch.bool)
    out, rest, lse = ops.attend_training(q, k, v, keep, 0.125)
    stats = ops.add_norm_training(r, a, w, None, p, None, None, 1.0, False, 1e-6)[2]
    for op, args in ((ops.rotate_forward, (x, pos[:1], [0.1] * 8, [4, 4], False)), (ops.rotate_forward, (x, pos.double(), [0.1] * 8, [4, 4], False)),
                     (ops.rotate_forward, (x, pos, [0.1] * 7, [4, 4], False)), (ops.rotate_forward, (x, pos, [0.1] * 8, [4, 4, 0], False)),
                     (ops.rotate_backward, (x, x[:1], pos, [0.1] * 8, [4, 4], False)), (ops.attend_forward, (q, k, v, keep.float(), 0.125)),
                     (ops.attend_training, (q, k, v[:, :-1], keep, 0.125)), (ops.attend_backward, (q[:, :-1], q, k, v, keep, out, rest, lse, 0.125)),
                     (ops.attend_backward, (q, q, k, v, keep, out, rest[:0], lse, 0.125)), (ops.attend_backward, (q, q, k, v, keep, out, rest, lse[..., :-1], 0.125)),
                     (ops.attend_backward, (q, q, k, v, keep, out.float(), rest, lse, 0.125)),
                     (ops.add_norm_training, (r, a, w, None, p, None, torch.ones(2, device=_dev(), dtype=torch.float64), 1.0, False, 1e-6)),
                     (ops.add_norm_backward, (r, None, r, a, w, p, None, None, stats[:-1], [1, 0, 1, 0], 1.0, False, 1e-6)),
                     (ops.add_norm_backward, (None, None, r, a, w, p, None, None, stats, [1, 0, 1, 0], 1.0, False, 1e-6)),
                     (ops.add_norm_backward, (r, None, r, a, w, None, None, None, stats, [1, 0, 1, 0], 1.0, False, 1e-6)),
                     (ops.add_norm_backward, (r, None, r, a, w, p, None, None, stats, [1, 0], 1.0, False, 1e-6))):
        with pytest.raises(ValueError):
            op(*args)
    with pytest.raises(RuntimeError, match="one GPU|on the GPU"):
        ops.rotate_forward(x, pos.cpu(), [0.1] * 8, [4, 4], False)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("which", range(3))
def test_vmap_and_function_transforms(which):
    """vmap runs call by call; grad through functorch is refused, and not wrong."""
    call, inputs = _operators()[which]
    stacked = torch.stack([inputs[0], inputs[0].flip(0)])
    got = torch.func.vmap(lambda t: call(t, *inputs[1:]))(stacked)
    assert torch.equal(got, torch.stack([call(t, *inputs[1:]) for t in stacked]))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call(t, *inputs[1:]).float().sum())(inputs[0])
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: call(t, *inputs[1:]), (inputs[0],), (inputs[0],))


def _norm_call(t, scale, kind="rms"):
    return tokens.add_norm_tokens(t["residual"], t["branch"], t["weight"], post_weight=t.get("post"), gate=t.get("gate"), scale=scale, kind=kind)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,post", [(72, False), (72, True), (1500, True)])
def test_a_scale_of_zero_as_a_number_leaves_the_branch_out(dtype, D, post):
    """scale=0.0 for all rows is what draws of 0 for all of them are: the residual stays, whatever the branch holds."""
    g = _gen(93)
    t = {"residual": _randn(g, 2, 6, D, dtype=dtype), "branch": _randn(g, 2, 6, D, dtype=dtype), "weight": _randn(g, D, dtype=dtype), "gate": _randn(g, 2, D, dtype=dtype)}
    if post:
        t["post"] = _randn(g, D, dtype=dtype)
    t["branch"][0, 1, 3], t["branch"][1, 0, 2] = math.nan, math.inf
    results = []
    for scale in (0.0, torch.zeros(2, device=_dev())):
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, z = _norm_call(leaves, scale)
        grads = torch.autograd.grad((y, z), list(leaves.values()), (torch.ones_like(y), torch.ones_like(z)))
        results.append([y.detach(), z.detach()] + list(grads))
        assert torch.equal(y, t["residual"]) and not grads[1].any() and all(torch.isfinite(x).all() for x in results[-1])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [72, 1500])
def test_a_dropped_rows_infinite_gradient_stays_out_of_the_gates(dtype, D):
    """A row whose scale is 0 has no part in n: gate and post_weight get from it nothing, whatever comes down its residual."""
    g = _gen(94)
    t = {"residual": _randn(g, 2, 8, D, dtype=dtype), "branch": _randn(g, 2, 8, D, dtype=dtype), "weight": _randn(g, D, dtype=dtype), "gate": _randn(g, 2, D, dtype=dtype),
         "post": _randn(g, D, dtype=dtype)}
    draws = torch.tensor([[0.0, 2.0], [2.0, 2.0]], device=_dev())
    dy, dz = _randn(g, 2, 8, D, dtype=dtype), _randn(g, 2, 8, D, dtype=dtype)
    results = []
    for bad in (0.0, math.inf):
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        up = dy.clone()
        up[0, 1, 5] = bad
        out = _norm_call(leaves, draws)
        results.append(dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), (up, dz)))))
    clean, got = results
    assert torch.isinf(got["residual"][0, 1, 5]) and not got["branch"][0, :4].any()
    assert all(torch.equal(got[k], clean[k]) for k in ("branch", "gate", "post", "weight"))


def test_a_last_batch_without_objects():
    """The draws of no objects, the mask of no keys: empty results and zero gradients, as without them."""
    g = _gen(95)
    w = _randn(g, 8).requires_grad_()
    x, a = (torch.zeros(0, 12, 8, device=_dev(), requires_grad=True) for _ in range(2))
    gate = torch.zeros(0, 8, device=_dev(), requires_grad=True)
    y, z = tokens.add_norm_tokens(x, a, w, post_weight=w, gate=gate, scale=torch.zeros(0, 3, device=_dev()))
    assert y.shape == x.shape and z.shape == x.shape
    gx, ga, gg, gw = torch.autograd.grad((y, z), (x, a, gate, w), (y.detach(), z.detach()))
    assert gx.shape == x.shape and ga.shape == x.shape and gg.shape == gate.shape and not gw.any()
    h = lambda *s: torch.ones(*s, dtype=torch.float16, device=_dev())  # noqa: E731
    for B, Lq, Lk, keep in ((0, 4, 6, (0, 3)), (2, 4, 0, (2, 0)), (2, 4, 0, (2, 5)), (0, 4, 0, (0, 0))):
        got = _attention(h(B, Lq, 2, 16), h(B, Lk, 2, 16), h(B, Lk, 2, 16), h(B, Lq, 2, 16), torch.zeros(*keep, device=_dev()))
        assert [tuple(t.shape) for t in got] == [(B, Lq, 2, 16)] * 2 + [(B, Lk, 2, 16)] * 2 and not any(t.any() for t in got)


@pytest.mark.parametrize("which", range(3))
def test_some_leaves_only(which):
    """Frozen keys, a learned query, cameras alone: the gradients that are asked for are those of the full backward, bit by bit."""
    call, inputs = _operators()[which]
    leaves = [t.detach().requires_grad_() for t in inputs]
    out = call(*leaves)
    up = torch.randn_like(out)
    full = torch.autograd.grad(out, leaves, up)
    for wanted in itertools.product((False, True), repeat=len(inputs)):
        if not any(wanted):
            continue
        some = [t.detach().requires_grad_(w) for t, w in zip(inputs, wanted)]
        again = call(*some)
        assert torch.equal(again, out)
        got = torch.autograd.grad(again, [t for t, w in zip(some, wanted) if w], up)
        assert all(torch.equal(a, b) for a, b in zip(got, [g for g, w in zip(full, wanted) if w])), wanted


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Lq,Lk,H,E,D", [(2, 150, 300, 4, 2, 64), (1, 2, 3000, 4, 2, 128), (2, 40, 50, 2, 2, 40)])
def test_the_c_abi_without_the_outputs_rest(dtype, B, Lq, Lk, H, E, D):
    """mvr_attend_tokens_forward and _backward, for programs that keep out and lse alone: the same output, gradients that carry out's rounding too."""
    from test_gpu_tokens_accuracy import _check, _sizes
    g = _gen(96)
    q, k, v, do = (_randn(g, *s, dtype=dtype) for s in ((B, Lq, H, D), (B, Lk, E, D), (B, Lk, E, D), (B, Lq, H, D)))
    lib, p = _lib.load(), lambda t: t.data_ptr()  # noqa: E731
    a = _lib.AttendParams(B, Lq, Lk, H, E, D, {torch.float16: 1, torch.bfloat16: 2}[dtype], 0)
    a.scale = D ** -0.5
    for t, s in ((q, a.q_stride), (k, a.k_stride), (v, a.v_stride), (do, a.grad_stride)):
        s[:] = t.stride()[:3]
    room = [torch.empty(max(lib.mvr_attend_tokens_workspace_bytes(a, n), 1), dtype=torch.uint8, device=_dev()) for n in (0, 1)]
    out, lse = torch.empty_like(q), torch.empty(B, H, Lq, device=_dev())
    grads = [torch.empty_like(t) for t in (q, k, v)]
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.mvr_attend_tokens_forward(a, p(q), p(k), p(v), None, p(out), p(lse), p(room[0]), room[0].numel(), stream) == 0
    assert lib.mvr_attend_tokens_backward(a, p(q), p(k), p(v), None, p(out), p(lse), p(do), *map(p, grads), p(room[1]), room[1].numel(), stream) == 0
    want, var = _sizes(q, k, v, do, D ** -0.5, stored_out=True)
    _check([out] + grads, want, var, dtype)
    assert torch.equal(out, tokens.attend_tokens(q, k, v))
    scores = torch.einsum("bqehd,bked->behqk", q.double().view(B, Lq, E, H // E, D), k.double()) * D ** -0.5
    assert torch.allclose(lse.double(), scores.logsumexp(-1).reshape(B, H, Lq) / math.log(2), rtol=0, atol=2.0 ** -16)   # (of numbers below 16: 2^-20 each of score and sum)
