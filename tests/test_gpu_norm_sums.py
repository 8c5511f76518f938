"""norm_rotary: the sums behind the weights' gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [4, 8])
def test_weight_gradients_do_not_lose_to_long_sums(d):
    """Rows of ones (a norm of one, exactly) and equal gradients of 2^23 + 31: sums of 64 of them and more are multiples of 64 in float32, and
    each addition there would lose the 31.  What is rounded: a few rows' sum, a block's and the result, 2^-24 each."""
    import matchattention_b200 as ma
    rows, value = 75000, 2.0 ** 23 + 31
    x = torch.ones(1, rows, 1, d, device="cuda")
    w = torch.ones(d, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(ma.norm_rotary(x, q_weight=w, eps=0.0), w, torch.full_like(x, value))
    assert float((dw.double() / (rows * value) - 1).abs().max()) <= 4 * 2.0 ** -24
