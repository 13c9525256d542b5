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
