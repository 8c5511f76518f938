"""global_attention in the forms that large calls and long caches take: blocks of 256 queries whose buffers go round, tiles that one half of a
block sees and the other does not, keys in shares that are joined, 128-row blocks in float32 (bounds in _dense.py)."""
import ctypes

import pytest
import torch

import _dense
from _dense import assert_within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = ("out", "dq", "dk", "dv")


def ma():
    import matchattention_b200
    return matchattention_b200


def make(seed, B, N, M, h, hk, d, dtype):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=gen).to(dtype).cuda() for shape in ((B, N, h, d), (B, M, hk, d), (B, M, hk, d), (B, N, h, d))]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def check(tensors, options, train):
    q, k, v, dout = tensors
    want, bound = _dense.attention(q, k, v, dout=dout if train else None, **options)
    if train:
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = ma().global_attention(*leaves, **options)
        got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    else:
        got = [ma().global_attention(q, k, v, **options)]
    for name, *three in zip(NAMES, got, want, bound):
        assert_within(*three, name)


def options_of(mask, scores, B, N, M, h):
    """Key tiles that only the first, only the second or no tile of a block of 256 queries sees are among them."""
    block = lambda n, size: [i // size for i in range(n)]  # noqa: E731
    far = [(i // 128) % 3 for i in range(M)]
    options = {
        "none": dict(),
        "causal": dict(causal=True),
        "prefix": dict(causal=True, prefix=ints([(b * M) // 4 for b in range(B)])),
        "lengths": dict(lengths=ints([M - 200 * b - 5 for b in range(B)])),
        "lengths_causal": dict(causal=True, lengths=ints([M - 250 * b for b in range(B)])),
        "documents": dict(documents=(ints([block(N, 128)] * B), ints([far] * B))),
        "documents_odd": dict(causal=True, documents=(ints([[(i - 1) // 50 for i in range(N)]] * B), ints([[(i - 7) // 180 for i in range(M)]] * B))),
    }[mask]
    if "cap" in scores:
        options["cap"] = 3.0
    if "map" in scores:
        options.update(slopes=(0.05 * 2.0 ** -(torch.arange(h, dtype=torch.float32) % 8)).cuda(), width=13)
    return options


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scores", ["plain", "cap_map"])
@pytest.mark.parametrize("mask", ["none", "causal", "prefix", "lengths", "lengths_causal", "documents", "documents_odd"])
def test_blocks_of_256_queries(mask, scores, d, dtype):
    B, N, M, h, hk = 5, 300, 1100, 32, 4
    tensors = make(71, B, N, M, h, hk, d, dtype)
    options = options_of(mask, scores, B, N, M, h)
    if mask == "lengths":            # in tiles that are partly hidden: the values of both halves are added term by term
        for b, n in enumerate(options["lengths"].tolist()):
            tensors[1][b, n:], tensors[2][b, n:] = float("nan"), float("inf")
    check(tensors, options, train=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [40, 128])
@pytest.mark.parametrize("mask,scores", [("lengths_causal", "cap"), ("documents_odd", "map"), ("documents", "plain"), ("prefix", "map")])
def test_training_over_many_tiles(mask, scores, d, dtype):
    B, N, M, h, hk = 3, 700, 900, 8, 2
    check(make(72, B, N, M, h, hk, d, dtype), options_of(mask, scores, B, N, M, h), train=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_references_that_move_late_in_a_row(d, dtype):
    """Scores that rise by hundreds along the keys, fall, and jump in single rows, in both tiles of a block."""
    B, N, M, h, hk = 5, 300, 1100, 32, 4
    q, k, v, dout = make(73, B, N, M, h, hk, d, dtype)
    q = (q.float() * 0.1 + 1).to(dtype)
    ramp = torch.linspace(0.0, 400.0 / d, M, device="cuda").view(1, M, 1, 1)
    for way in (ramp, ramp.flip(1), ramp * (torch.arange(M, device="cuda") % 97 == 0).view(1, M, 1, 1)):
        check((q, (k.float() * 0.02 + way).to(dtype), v, dout), dict(scale=1.0), train=False)
    q[:, 200:201] *= 3
    check((q, (k.float() * 0.02 + ramp).to(dtype), v, dout), dict(scale=1.0), train=False)


SHARES = [(1, 20, 1500, 4, 2), (2, 130, 1300, 2, 1), (1, 1, 4000, 8, 2), (3, 4, 2100, 4, 4)]      # B, N, M, h, hk


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("shape", SHARES, ids=str)
def test_keys_in_shares(shape, d, dtype):
    """Forward and backward, which builds on what the join wrote; lengths that leave whole shares, and items, without a key."""
    B, N, M, h, hk = shape
    tensors = make(74, B, N, M, h, hk, d, dtype)
    for options in (dict(), dict(causal=True, cap=4.0), dict(causal=True, lengths=ints([max(N, 150)] + [0] * (B - 1))), dict(lengths=ints([M - 1] + [3] * (B - 1))),
                    options_of("documents_odd", "map", B, N, M, h)):
        check(tensors, options, train=True)


def forward_and_backward(q, k, v, dout, low, **options):
    """Through the C entry points, with or without what the rounding of the output left."""
    from matchattention_b200 import _lib
    B, N, h, d = q.shape
    M, hk = k.shape[1:3]
    out, rest, lse = torch.empty_like(q), torch.full_like(q, float("nan")), torch.empty(B, h, N, device="cuda")
    args = _lib.GlobalArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), out_low=rest.data_ptr() if low else None,
                           lse=lse.data_ptr(), B=B, N=N, M=M, h=h, hk=hk, d=d, q_stride=tuple(q.stride()[:3]), k_stride=tuple(k.stride()[:3]),
                           v_stride=tuple(v.stride()[:3]), dtype=1 if q.dtype == torch.float16 else 2, width=1, scale=d ** -0.5, **options)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    stream = torch.cuda.current_stream().cuda_stream
    for back, call, more in ((0, _lib.lib.matchattn_global_forward, ()),
                             (1, _lib.lib.matchattn_global_backward, [ctypes.c_void_p(t.data_ptr()) for t in (dout, *grads)])):
        size = _lib.lib.matchattn_global_scratch_bytes(args, back)
        scratch = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        assert call(args, *more, scratch.data_ptr(), size, stream) == 0
    torch.cuda.synchronize()
    return out, rest, grads


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("shape", [(1, 600, 600, 4, 2, 64), (5, 300, 300, 32, 4, 128), (1, 20, 1500, 4, 2, 64), (1, 2, 700, 4, 2, 64), (1, 2, 40, 4, 2, 64),
                                   (2, 90, 90, 2, 1, 20)], ids=str)
def test_what_the_rounding_of_the_output_left(shape, dtype):
    """From every forward kernel and from the join: out is out + out_low rounded, and the gradients of q and k gain by it.

    With values around 100 and keys around 1 the rounding of out, u 100 per channel, moves delta by 100 u sqrt(d / 3) and every dS of the row
    by p times that, all to one side, against dS of p sqrt(d) rounded by u: dq and dk are off by tens of times as much without out_low."""
    B, N, M, h, hk, d = shape
    q, k, v, dout = make(75, B, N, M, h, hk, d, dtype)
    k, v = k + 1, v + 100
    out, low, with_low = forward_and_backward(q, k, v, dout, True)
    same, untouched, without = forward_and_backward(q, k, v, dout, False)
    assert bool(untouched.isnan().all())
    assert bool(torch.isfinite(low).all()) and float((low != 0).float().mean()) > 0.9
    # at most half a step, which the type holds exactly: what is rounded to it makes a tie, and no more
    near = (out.double() + low.double()).to(dtype).double()
    assert bool(((near == out.double()) | ((near - out.double()).abs() == 2 * low.double().abs())).all())
    want, _ = _dense.attention(q, k, v, dout=dout)
    far = lambda t, w: float((t.double() - w).square().mean().sqrt())  # noqa: E731
    # out alone is off by its rounding as well, out and out_low together by that of the probabilities
    assert far(out.double() + low.double(), want[0]) < far(out, want[0])
    for i in (0, 1):
        assert 4 * far(with_low[i], want[i + 1]) < far(without[i], want[i + 1]), NAMES[i + 1]
