"""CPU (-m "not gpu"): further calls of the operators on view tokens that are refused, or answered, before anything reaches the GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from mvtn_amd import _lib, tokens


def _calls(dtype=torch.float32):
    """(call, inputs that are differentiated) of each operator, on the CPU."""
    r = lambda *s: torch.randn(*s, dtype=dtype)  # noqa: E731
    rotary, h = tokens.TokenRotary((2, 1)), lambda *s: torch.randn(*s).half()  # noqa: E731
    return [(rotary, [r(2, 3, 1, 8), r(3, 2)]), (tokens.attend_tokens, [h(2, 3, 2, 8), h(2, 6, 2, 8), h(2, 6, 2, 8)]),
            (lambda a, b, w, bias, post, gate: tokens.add_norm_tokens(a, b, w, bias, post, gate, kind="layer"),
             [r(2, 6, 8), r(2, 6, 8), r(8), r(8), r(8), r(2, 8)])]


@pytest.mark.parametrize("which", range(3))
def test_forward_mode_is_refused(which):
    """Tangents are not carried on, so they may not be dropped: with any input, whether it requires grad or not, under no_grad too."""
    call, inputs = _calls()[which]
    for k in range(len(inputs)):
        for needs in (False, True):
            with forward_ad.dual_level():
                args = list(inputs)
                args[k] = forward_ad.make_dual(inputs[k].clone().requires_grad_(needs), torch.ones_like(inputs[k]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(call, tuple(inputs), tuple(torch.ones_like(t) for t in inputs))


def test_attention_c_abi_with_the_rest_refuses_before_any_launch():
    lib = _lib.load()
    p = 4096   # never dereferenced: every call below is refused on the host
    a = _lib.AttendParams(2, 3, 6, 4, 2, 8, 1, 0)
    a.scale = 1.0

    def forward(rest, lse=p + 96, out=p + 64):
        return lib.mvr_attend_tokens_forward_rest(a, p, p + 16, p + 32, None, out, rest, lse, None, 0, None)
    assert forward(p + 128, lse=None) == 1 and b"lse" in lib.mvr_last_error()
    for rest in (p, p + 16, p + 32, p + 64):
        assert forward(rest) == 1
    assert lib.mvr_attend_tokens_backward_rest(a, p, p, p, None, p, p, None, p, p, p, p, p, 1 << 40, None) == 1
    assert lib.mvr_attend_tokens_backward_rest(a, p, p, p, None, p, p, p, p, p, p, p, None, 0, None) == 3


def test_a_call_does_not_record_a_stream():
    """A traced call runs on the stream that is current when it is replayed: none of the operators takes a stream's handle as a number."""
    tokens._lib.token_op()
    for name in ("rotate", "attend", "add_norm"):
        schema = getattr(torch.ops.mvr_tokens, name).default._schema
        assert not [a.name for a in schema.arguments if "stream" in a.name], schema


def _on_fake_gpu():
    """(call, inputs) of each operator on tensors that have shapes and a device and no memory."""
    rotary = tokens.TokenRotary((4, 4), periods=(360.0, None))
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
    draws, keep = e(2, 3, dtype=torch.float32), e(2, 3, dtype=torch.float32)
    return [(rotary, [e(2, 90, 2, 24), e(90, 2, dtype=torch.float32)], [(2, 90, 2, 24)]),
            (lambda q, k, v: tokens.attend_tokens(q, k, v, keep=keep), [e(2, 40, 4, 64).transpose(1, 2).contiguous().transpose(1, 2), e(2, 90, 2, 64), e(2, 90, 2, 64)], [(2, 40, 4, 64)]),
            (lambda x, a, w, gate: tokens.add_norm_tokens(x, a, w, gate=gate, scale=draws), [e(2, 90, 72, dtype=torch.float32), e(2, 90, 72), e(72), e(2, 72)], [(2, 90, 72)] * 2)]


@pytest.mark.parametrize("which", range(3))
def test_shapes_without_memory(which):
    """Under a tracer of shapes the operators give tensors of the right shape, type and layout; and what does not fit is refused as ever."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        call, inputs, shapes = _on_fake_gpu()[which]
        out = call(*inputs)
        out = out if isinstance(out, tuple) else (out,)
        assert [tuple(t.shape) for t in out] == shapes and all(t.is_contiguous() and t.device.type == "cuda" for t in out)
        assert [t.dtype for t in out] == ([torch.float32, torch.bfloat16] if which == 2 else [torch.bfloat16])
        out = call(*[t.requires_grad_() for t in inputs])
        assert all(t.requires_grad for t in (out if isinstance(out, tuple) else (out,)))
        with pytest.raises(ValueError):
            call(inputs[0][..., :15], *inputs[1:])


@pytest.mark.parametrize("which", range(3))
def test_a_graph_of_a_call_holds_the_operator(which):
    """What a tracer below autograd records is the operator, not the allocation of its result alone."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode(allow_non_fake_inputs=True):
        call, inputs, _ = _on_fake_gpu()[which]
        graph = make_fx(call)(*inputs).graph
    names = [str(n.target) for n in graph.nodes if n.op == "call_function"]
    assert [n for n in names if n.startswith("mvr_tokens.")] == [("mvr_tokens.rotate_forward.default", "mvr_tokens.attend_forward.default", "mvr_tokens.add_norm_forward.default")[which]], names


def test_empty_masks_and_draws_only_for_empty_tensors():
    h = lambda *s: torch.zeros(*s, dtype=torch.float16)  # noqa: E731
    x, w = torch.zeros(0, 6, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match="GPU"):   # (nothing wrong with the arguments)
        tokens.attend_tokens(h(2, 3, 2, 8), h(2, 0, 2, 8), h(2, 0, 2, 8), keep=torch.zeros(2, 0))
    with pytest.raises(RuntimeError, match="GPU"):
        tokens.add_norm_tokens(x, x, w, scale=torch.zeros(0, 3))
    with pytest.raises(ValueError):
        tokens.attend_tokens(h(2, 3, 2, 8), h(2, 6, 2, 8), h(2, 6, 2, 8), keep=torch.zeros(2, 0))
    with pytest.raises(ValueError):
        tokens.add_norm_tokens(torch.zeros(2, 6, 8), torch.zeros(2, 6, 8), w, scale=torch.zeros(0, 3))
