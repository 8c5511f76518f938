"""global_attention over long caches: many keys of small weight."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def ma():
    import matchattention_b200
    return matchattention_b200


# keys in shares (few blocks: the first key weighs against those of its own share alone) and in one run
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("B,N,h,M,d", [(1, 1, 1, 1 << 20, 64), (1, 20, 1, 1 << 20, 64), (1, 20, 160, 1 << 20, 64), (300, 1, 1, 1 << 16, 8)])
def test_many_small_weights_beside_a_large_one(B, N, h, M, d, train, dtype):
    """Keys that each have exp(-17.75) = 2^-25.6 of the weight of the first one, and make all of the result: of a million 2 % of the sum."""
    ahead = 17.75
    q, k = torch.zeros(B, N, h, d, device="cuda", dtype=dtype), torch.zeros(B, M, 1, d, device="cuda", dtype=dtype)
    v = torch.ones(B, M, 1, d, device="cuda", dtype=dtype)
    q[..., 0], k[:, 0, 0, 0], v[:, 0] = 1.0, ahead, 0.0
    if train:
        q.requires_grad_()
    out = ma().global_attention(q, k, v, scale=1.0)
    rest = (M - 1) * math.exp(-ahead)
    want = rest / (1 + rest)
    # the scores are exact (17.75 has 7 bits).  A weight is rounded by u of it, in float16 held times 2^11 at the least, in steps of 2^-24, by
    # 2^-25 / 2^-14.6 = 2^-10.4; an exponential and a logarithm of 26 in float32 are off by 2^-18; a thread adds 2^15 equal weights at most,
    # by 2^-24 of the sum each: 2^-9, altogether; the result is rounded by u
    u = torch.finfo(dtype).eps / 2
    bound = 2 * u + (2.0 ** -10.4 if dtype == torch.float16 else 0.0) + 2.0 ** -18 + 2.0 ** -9
    assert float((out.detach().double() / want - 1).abs().max()) <= bound
    if train:
        # dq is along the first channel: sum p (v_j - out) . g k_j = ahead p_0 (0 - out) . g, for g = 1: -d ahead p_0 out
        (dq,) = torch.autograd.grad(out, q, torch.ones_like(q))
        slope = -d * ahead / (1 + rest) * want
        assert float((dq.double()[..., 0] / slope - 1).abs().max()) <= 4 * u + bound + 2.0 ** -9
