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
