"""global_attention and norm_rotary in torch's autograd: what is formed, and what is refused rather than left out."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ma():
    import matchattention_b200
    return matchattention_b200


def make(*shapes, dtype=torch.float32, seed=51):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=gen).to(dtype).cuda() for s in shapes]


def test_slopes_that_train_elsewhere():
    """Parameters as slopes: constants in inference, refused where a gradient would be expected of them."""
    q, k, v = make((1, 9, 2, 16), (1, 9, 2, 16), (1, 9, 2, 16))
    slopes = torch.tensor([0.5, 0.25], device="cuda", requires_grad=True)
    want = ma().global_attention(q, k, v, slopes=slopes.detach())
    with torch.no_grad():
        assert torch.equal(ma().global_attention(q, k, v, slopes=slopes), want)
        assert torch.equal(ma().global_attention(torch._neg_view(-q), k, v, slopes=slopes), want)
    with torch.inference_mode():
        assert torch.equal(ma().global_attention(q, k, v, slopes=slopes), want)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(NotImplementedError):
            ma().global_attention(x, k, v, slopes=slopes)
