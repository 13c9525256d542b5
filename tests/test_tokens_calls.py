"""CPU (-m "not gpu"): further calls of the operators on view tokens that are refused, or answered, before anything reaches the GPU."""
from mvtn_amd import _lib


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
