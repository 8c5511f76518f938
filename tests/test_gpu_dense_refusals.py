"""global_attention and norm_rotary: arguments that are refused, and with which error."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ma():
    import matchattention_b200
    return matchattention_b200


def test_sizes_of_more_than_32_bits():
    """2^32 + 5 items, tokens or heads are not five."""
    many = 2 ** 32 + 5
    one = torch.zeros(1, 1, 1, 1, dtype=torch.float16, device="cuda")
    for shape in ((many, 1, 1, 1), (1, many, 1, 1), (1, 1, many, 1)):
        x = one.expand(shape)
        with pytest.raises(ValueError):
            ma().global_attention(x, x, x)
        with pytest.raises(ValueError):
            ma().norm_rotary(x)
        with pytest.raises(ValueError):
            ma().norm_rotary(x, x)
    with pytest.raises(ValueError):
        ma().global_attention(one, one.expand(1, many, 1, 1), one.expand(1, many, 1, 1))
    with pytest.raises(ValueError):
        ma().global_attention(one, one, one, slopes=torch.ones(1, device="cuda"), width=2 ** 32 + 1)


@pytest.mark.parametrize("scale,cap", [(1e-39, 0.0), (1e-50, 0.0), (2.5e38, 0.0), (0.25, 3e38), (0.25, 1e39), (0.25, 1e-39), (0.25, 1e-50), (1e10, 1e-30),
                                       (1e-10, 1e30)])
def test_scales_and_caps_that_float32_cannot_hold(scale, cap):
    """A cap that float32 rounds to zero is no call without a cap; one whose units overflow gives no NaN."""
    q = torch.zeros(1, 2, 2, 16, device="cuda")
    for x in (q, q.half(), q[:, :1].bfloat16()):
        with pytest.raises(ValueError):
            ma().global_attention(x, x, x, scale=scale, cap=cap)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_largest_cap(dtype):
    q = torch.randn(1, 40, 2, 16, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    for n in (1, 40):
        want = ma().global_attention(q[:, :n], q, q, scale=0.25)
        got = ma().global_attention(q[:, :n], q, q, scale=0.25, cap=2.0 ** 123)
        # c tanh(x / c) is x then, but for an operation or two
        assert torch.allclose(got.float(), want.float(), rtol=2 * torch.finfo(dtype).eps, atol=2.0 ** -12)


def test_arguments_that_are_no_tensors_or_have_no_channels():
    q = torch.zeros(1, 2, 2, 16, device="cuda")
    f = ma().global_attention
    with pytest.raises(TypeError):
        f("q", q, q)
    with pytest.raises(TypeError):
        f(q, None, q)
    with pytest.raises(TypeError):
        f(q, q, q, slopes=[0.5, 0.25])
    for x in (q[..., :0], q[:, :, :0], torch.zeros((), device="cuda")):
        with pytest.raises(ValueError):
            f(x, x, x)
        with pytest.raises(ValueError):
            ma().norm_rotary(x)
