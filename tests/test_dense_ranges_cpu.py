"""The ranges of global_attention's and norm_rotary's plain arguments, at the C entry points; no GPU."""
import pytest

from matchattention_b200 import _lib

AT = 4096       # never dereferenced


def forward(scratch=AT, nbytes=1 << 40, **changes):
    a = dict(q=AT, k=AT, v=AT, out=AT, lse=AT, B=1, N=8, M=8, h=4, hk=2, d=16, dtype=1, causal=0, width=1, scale=0.25, cap=0.0)
    a.update(changes)
    for n in ("q_stride", "k_stride", "v_stride"):
        a[n] = (512, 64, 16)
    return _lib.GlobalArgs(**a)


BAD_SCORES = [(1e-39, 0.0), (2.5e38, 0.0), (0.25, 3e38), (0.25, 1e-39), (1e10, 1e-30), (1e-10, 1e30)]


@pytest.mark.parametrize("scale,cap", BAD_SCORES)
def test_scales_and_caps_that_float32_cannot_hold(scale, cap):
    """scale * log2(e), cap * log2(e) and scale / cap have to be normal numbers."""
    args = forward(scale=scale, cap=cap)
    assert _lib.lib.matchattn_global_forward(args, AT, 1 << 40, None) == 2
    assert _lib.lib.matchattn_global_backward(args, AT, AT, AT, AT, AT, 1 << 40, None) == 2
    assert _lib.lib.matchattn_global_scratch_bytes(args, 1) == 0


def test_scales_and_caps_at_the_ends_of_the_range():
    for scale, cap in ((2.0 ** -126, 0.0), (2.3e38, 0.0), (1.0, 8e37), (1.0, 1e-37)):
        assert _lib.lib.matchattn_global_scratch_bytes(forward(scale=scale, cap=cap), 1) > 0
