"""global_attention: what a form keeps beyond the bounds that all forms share (_dense.py)."""
import pytest
import torch

import _dense
from _dense import assert_within

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


def ma():
    import matchattention_b200
    return matchattention_b200


def make(seed, B, N, M, h, hk, d, dtype):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=gen).to(dtype).cuda() for shape in ((B, N, h, d), (B, M, hk, d), (B, M, hk, d), (B, N, h, d))]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("N,h,hk", [(1, 8, 8), (1, 8, 2), (3, 4, 1)])
def test_single_tokens_lose_nothing_to_rounded_probabilities(N, h, hk, d, dtype):
    """Probabilities enter the product with v as two terms: float32's bounds, u of the result, and u^2 of the terms of a sum twice."""
    u, last = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    for M in (1, 40, 700, 3000):
        q, k, v, _ = make(41, 2, N, M, h, hk, d, dtype)
        options = dict(lengths=torch.tensor([M, (M + 1) // 2], dtype=torch.int32, device="cuda"))
        got = ma().global_attention(q, k, v, **options)
        (want,), (bound,) = _dense.attention(q.float(), k.float(), v.float(), **options)
        (terms,), _ = _dense.attention(q.float(), k.float(), v.float().abs(), **options)
        assert_within(got, want, bound + u * want.abs() + 2 * u * u * terms + last, f"out over {M} keys")


@pytest.mark.parametrize("dtype", [torch.float32] + HALVES)
@pytest.mark.parametrize("N,h,hk", [(1, 8, 8), (2, 8, 2), (3, 4, 1), (40, 4, 2)])
def test_infinite_values_that_all_see(N, h, hk, dtype):
    """An infinite value stays an infinity of its sign in what it is added to, whatever its weight (a thousandth, or nearly all)."""
    M, d = 300, 64
    q, k, v, _ = make(42, 1, N, M, h, hk, d, dtype)
    k[:, 77] = 0.0
    for at, channel in enumerate(range(0, 48, 3)):
        v[0, 13 * at + 1, at % hk, channel] = float("inf") if at % 2 else float("-inf")
    want, bound = _dense.attention(q, k, v)
    got = ma().global_attention(q, k, v)
    assert int(got.isinf().sum()) >= N * 16
    assert_within(got, want[0], bound[0], "out")
    # one key of weight one: its second term is nothing but the sign
    one = ma().global_attention(q, k[:, 77:78], v[:, 1:2])
    assert torch.equal(one, v[:, 1:2].repeat_interleave(h // hk, 2).expand_as(one))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("N,h,hk,d,options", [(1500, 4, 4, 16, dict(slopes=True, width=40)), (700, 4, 1, 64, dict(causal=True)), (500, 2, 2, 128, dict(causal=True, cap=20.0))],
                         ids=str)
def test_gradients_of_queries_lose_nothing_to_rounded_terms(N, h, hk, d, options, dtype):
    """dS enters the sum over the keys as two terms: what is left beside the rounding of the result itself is what the rounding of the forward's
    probabilities does to delta, a tenth of it (rounded once, dS would put its own error beside the result's: the square root of two)."""
    q, k, v, dout = make(43, 1, N, N, h, hk, d, dtype)
    if "slopes" in options:
        options = dict(options, slopes=(0.5 * 2.0 ** -(8 * torch.arange(h, dtype=torch.float32) / h)).cuda())
    want = _dense.attention(q, k, v, dout=dout, **options)[0][1]
    q.requires_grad_()
    (got,) = torch.autograd.grad(ma().global_attention(q, k, v, **options), q, dout)
    far = (got.double() - want).square().mean().sqrt()
    rounding = (want.to(dtype).double() - want).square().mean().sqrt()
    assert float(far / rounding) <= 1.2
