"""global_attention against its definition in 64 bits (bounds in _dense.py)."""
import pytest
import torch

import _dense
from _dense import assert_within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def ma():
    import matchattention_b200
    return matchattention_b200


def make(seed, B, N, M, h, hk, d, dtype, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(shape, generator=gen) * spread).to(dtype).cuda() for shape in ((B, N, h, d), (B, M, hk, d), (B, M, hk, d), (B, N, h, d))]


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def slopes_of(h, base=0.3):
    return (base * 2.0 ** -torch.arange(h, dtype=torch.float32)).cuda()


def compare(seed, B, N, M, h, hk, d, dtype, train=True, spread=1.0, **options):
    q, k, v, dout = make(seed, B, N, M, h, hk, d, dtype, spread)
    want, bound = _dense.attention(q, k, v, dout=dout if train else None, **options)
    if not train:
        got = [ma().global_attention(q, k, v, **options)]
    else:
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = ma().global_attention(*leaves, **options)
        got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    for name, *three in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert_within(*three, name)
    return got


SHAPES = [  # B, N, M, h, hk, d
    (1, 1, 1, 1, 1, 1), (2, 1, 7, 4, 2, 8), (1, 5, 3, 2, 2, 16), (2, 63, 65, 2, 1, 24), (1, 129, 127, 3, 3, 32), (1, 257, 384, 4, 1, 64),
    (2, 130, 130, 2, 2, 40), (1, 300, 261, 2, 2, 128), (1, 128, 128, 2, 1, 80), (1, 70, 90, 2, 1, 17), (1, 140, 150, 2, 2, 129),
    (1, 33, 200, 2, 1, 256), (1, 513, 640, 1, 1, 96),
    (40, 140, 150, 4, 2, 64), (1, 200, 190, 12, 2, 64), (75, 20, 140, 3, 1, 20),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_shapes(shape, dtype):
    compare(1, *shape, dtype)
    compare(2, *shape, dtype, causal=True)


def masks(B, N, M):
    docs_q = [[(7 * n) // max(N, 1) - (1 if n < N // 9 else 0) for n in range(N)] for _ in range(B)]
    docs_k = [[(7 * m) // max(M, 1) for m in range(M)] for _ in range(B)]
    return {
        "causal": dict(causal=True),
        "prefix": dict(causal=True, prefix=ints([(b * M) // 3 for b in range(B)])),
        "lengths": dict(lengths=ints([max(M - 37 * b - 5, 0) for b in range(B)])),
        "lengths_causal": dict(causal=True, lengths=ints([max(M // (b + 1) - 3, 0) for b in range(B)])),
        "documents": dict(documents=(ints(docs_q), ints(docs_k))),
        "documents_causal_prefix": dict(causal=True, prefix=ints([M // 2] * B), documents=(ints(docs_q), ints(docs_k))),
    }


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scores", ["plain", "cap", "map", "cap_map"])
@pytest.mark.parametrize("mask", ["causal", "prefix", "lengths", "lengths_causal", "documents", "documents_causal_prefix"])
def test_masks_and_scores(mask, scores, dtype):
    for B, N, M, h, hk, d in ((3, 150, 150, 4, 2, 64), (2, 260, 400, 2, 1, 128), (3, 2, 300, 4, 2, 64)):
        options = masks(B, N, M)[mask]
        if "cap" in scores:
            options["cap"] = 3.0
        if "map" in scores:
            options.update(slopes=slopes_of(h), width=13)
        compare(3, B, N, M, h, hk, d, dtype, spread=1.5, **options)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,h,hk", [(1, 1, 1), (1, 8, 1), (1, 12, 4), (2, 8, 2), (3, 5, 5), (4, 16, 2), (7, 14, 2), (16, 4, 2)])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_single_tokens(N, h, hk, d, dtype):
    """New tokens at the end of caches of different fill, an empty one among them."""
    for M in (1, 15, 640, 2500):
        compare(4, 3, N, M, h, hk, d, dtype, train=False, causal=True, lengths=ints([M, M // 2, 0]))
        compare(5, 2, N, M, h, hk, d, dtype, train=False, causal=True, lengths=ints([M, min(M, 3)]), cap=5.0, slopes=slopes_of(h), width=9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing_give_zeros(dtype):
    B, N, M, h, d = 2, 130, 90, 2, 64
    q, k, v, dout = make(6, B, N, M, h, h, d, dtype)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    for options in (dict(lengths=ints([0, M])), dict(documents=(ints([[-1] * N] * B), ints([[-1] * M] * B))), dict(causal=True, lengths=ints([20, 0]))):
        out = ma().global_attention(*leaves, **options)
        want, bound = _dense.attention(q.detach(), k.detach(), v.detach(), dout=dout, **options)
        got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
        for name, *three in zip(("out", "dq", "dk", "dv"), got, want, bound):
            assert_within(*three, name)
        assert bool((got[0][want[0] == 0] == 0).all())


def check(tensors, options, train=True):
    q, k, v, dout = tensors
    want, bound = _dense.attention(q, k, v, dout=dout if train else None, **options)
    if train:
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        out = ma().global_attention(*leaves, **options)
        got = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    else:
        got = [ma().global_attention(q, k, v, **options)]
    for name, *three in zip(("out", "dq", "dk", "dv"), got, want, bound):
        assert_within(*three, name)
    return got, want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 20])
@pytest.mark.parametrize("N", [1, 3, 200])
def test_values_in_masked_places_do_not_matter(N, d, dtype):
    """Infinite and NaN keys and values behind a length and in padding tokens; padding queries and their gradients too."""
    B, M, h, hk = 2, 333, 4, 2
    clean = make(7, B, N, M, h, hk, d, dtype)
    q, k, v, dout = (t.clone() for t in clean)
    k[0, 205:], v[0, 205:] = float("nan"), float("inf")
    for options in (dict(causal=True, lengths=ints([205, 333])), dict(lengths=ints([205, 333])), dict(lengths=ints([205, 333]), cap=3.0),
                    dict(causal=True, lengths=ints([205, 333]), slopes=slopes_of(h), width=11)):
        got, want = check((q, k, v, dout), options)
        assert all(bool(torch.isfinite(w).all()) for w in want)
    q, k, v, dout = (t.clone() for t in clean)
    docs_k = torch.zeros(B, M, dtype=torch.int32, device="cuda")
    docs_k[:, 100:130], docs_k[:, 250:] = -1, 1
    docs_q = torch.zeros(B, N, dtype=torch.int32, device="cuda")
    if N > 3:
        docs_q[:, 150:160], docs_q[:, 160:] = -1, 1
        q[:, 150:160], dout[:, 150:160] = float("nan"), float("-inf")
    k[:, 100:130], v[:, 100:130] = float("inf"), float("nan")
    for options in (dict(), dict(cap=3.0)):
        got, want = check((q, k, v, dout), dict(documents=(docs_q, docs_k), **options))
        assert all(bool(torch.isfinite(w).all()) for w in want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [4, 400])
def test_a_value_reaches_those_that_see_it_and_no_other(N, dtype):
    """A NaN and an infinity in single channels of two tokens of a document: causal rows before them and the other document keep
    their results, and so do the other channels."""
    B, M, h, d = 1, 400, 2, 64
    q, k, v, dout = make(8, B, N, M, h, h, d, dtype)
    docs = torch.zeros(B, M, dtype=torch.int32, device="cuda")
    docs[:, 210:] = 1
    v[0, 170, 1, 5] = float("nan")
    v[0, 180, 0, 7] = float("inf")
    got, want = check((q, k, v, dout), dict(causal=True, documents=(docs[:, M - N:].contiguous(), docs)), train=False)
    if N == M:
        assert int(got[0].isnan().sum()) == 40 and int(got[0].isposinf().sum()) == 30
    v[0, M - 2, 1, 5], v[0, M - 1, 0, 7] = float("nan"), float("-inf")
    got, want = check((q, k, v, dout), dict(causal=True, documents=(docs[:, M - N:].contiguous(), docs)), train=False)
    assert bool(got[0][0, -2:, 1, 5].isnan().all()) and bool(torch.isfinite(got[0][0, -4:-2]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Heads of one projection side by side, tokens first, every second token, a broadcast key head."""
    B, N, h, hk, d = 2, 97, 4, 2, 64
    gen = torch.Generator().manual_seed(9)
    fused = torch.randn(B, N, (h + 2 * hk) * d, generator=gen).to(dtype).cuda()
    q, k, v = (fused[..., a:b].view(B, N, -1, d) for a, b in ((0, h * d), (h * d, (h + hk) * d), ((h + hk) * d, (h + 2 * hk) * d)))
    first = torch.randn(h, B, N, d, generator=gen).to(dtype).cuda().permute(1, 2, 0, 3)
    every = torch.randn(B, 2 * N, hk, d, generator=gen).to(dtype).cuda()[:, ::2]
    shared = torch.randn(B, N, 1, d, generator=gen).to(dtype).cuda().expand(B, N, hk, d)
    columns = torch.randn(B, N, d, hk, generator=gen).to(dtype).cuda().transpose(2, 3)
    odd = torch.randn(B * N * hk * d + 1, generator=gen).to(dtype).cuda()[1:].view(B, N, hk, d)
    wide = torch.randn(B, N, hk, d + 3, generator=gen).to(dtype).cuda()[..., :d]
    for a, b, c in ((q, k, v), (first, every, shared), (q, columns, odd), (first, wide, every)):
        want, bound = _dense.attention(a, b, c, causal=True)
        assert_within(ma().global_attention(a, b, c, causal=True), want[0], bound[0], "out")
        leaves = [t.detach().requires_grad_() for t in (a, b, c)]
        dout = torch.randn(B, N, h, d, generator=gen).to(dtype).cuda()
        want, bound = _dense.attention(a, b, c, causal=True, dout=dout)
        got = torch.autograd.grad(ma().global_attention(*leaves, causal=True), leaves, dout)
        for name, *three in zip(("dq", "dk", "dv"), got, want[1:], bound[1:]):
            assert_within(*three, name)


def test_gradient_against_differences():
    B, N, M, h, hk, d = 1, 9, 12, 2, 1, 6
    q, k, v, dout = make(10, B, N, M, h, hk, d, torch.float32)
    options = dict(causal=True, cap=2.0, slopes=slopes_of(h), width=4)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ma().global_attention(*leaves, **options), leaves, dout)
    for i, t in enumerate((q, k, v)):
        gen = torch.Generator().manual_seed(i)
        way = torch.randn(t.shape, generator=gen).cuda()
        step = 2.0 ** -7
        ends = []
        for sign in (1, -1):
            moved = [x.detach().clone() for x in (q, k, v)]
            moved[i] += sign * step * way
            ends.append((ma().global_attention(*moved, **options).double() * dout.double()).sum())
        slope = float((ends[0] - ends[1]) / (2 * step))
        want = float((grads[i].double() * way.double()).sum())
        # the third derivative times step^2 / 6 (values of order one to a hundred), and 2^-20 of the sum over the step
        assert abs(slope - want) <= 0.02 * max(1.0, abs(want)), (i, slope, want)


def test_gradients_of_broadcast_inputs():
    """A key head that all items and heads share by expand gets the sum of their gradients."""
    B, N, h, d = 2, 50, 4, 32
    q, _, _, dout = make(11, B, N, N, h, h, d, torch.float32)
    k1, v1 = (torch.randn(1, N, 1, d, generator=torch.Generator().manual_seed(s)).cuda().requires_grad_() for s in (1, 2))
    out = ma().global_attention(q, k1.expand(B, N, h, d), v1.expand(B, N, h, d))
    got = torch.autograd.grad(out, (k1, v1), dout)
    want, bound = _dense.attention(q, k1.detach().expand(B, N, h, d), v1.detach().expand(B, N, h, d), dout=dout)
    for g, w, b in zip(got, want[2:], bound[2:]):
        assert_within(g, w.sum((0, 2), keepdim=True), 2 * b.sum((0, 2), keepdim=True), "shared")


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(dtype):
    """Scores of hundreds, growing along the keys and falling, and a scale that makes one probability of a row all."""
    B, N, M, h, d = 1, 140, 700, 2, 64
    q, k, v, dout = make(12, B, N, M, h, h, d, dtype)
    ramp = torch.linspace(0.0, 3.0, M, device="cuda").view(1, M, 1, 1)
    q = (q.float() * 0 + 1).to(dtype)
    for way in (ramp, ramp.flip(1), 30 * ramp):
        kk = (k.float() * 0.02 + way).to(dtype)
        want, bound = _dense.attention(q, kk, v, scale=1.0, dout=dout)
        leaves = [t.detach().requires_grad_() for t in (q, kk, v)]
        out = ma().global_attention(*leaves, scale=1.0)
        for name, *three in zip(("out", "dq", "dk", "dv"), [out.detach(), *torch.autograd.grad(out, leaves, dout)], want, bound):
            assert_within(*three, name)


def test_small_gradients_in_float16():
    """Gradients far below one keep their digits: the products of the backward pass do not fall into the subnormal range."""
    B, N, h, d = 1, 300, 2, 64
    q, k, v, dout = make(13, B, N, N, h, h, d, torch.float16)
    dout = (dout.float() * 2.0 ** -10).half()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(ma().global_attention(*leaves), leaves, dout)
    want, bound = _dense.attention(q.detach(), k.detach(), v.detach(), dout=dout)
    for name, g, w, b in zip(("dq", "dk", "dv"), got, want[1:], bound[1:]):
        # results below 2^-14 are rounded to multiples of 2^-24
        assert_within(g, w, b + 2.0 ** -25, name)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("N", [1, 130])
def test_offsets_beyond_32_bits(N, dtype):
    """A cache of 2^31 values and more: zeros (scores of 0, values of 0) but for its first and last keys, whose share of every
    row is known: 2^24 - 64 exponentials of 0 beside theirs."""
    M, d, n = 2 ** 24, 129 if dtype == torch.float32 else 128, 32
    q = make(22, 1, N, 1, 1, 1, d, dtype)[0]
    k, v = torch.zeros(2, 1, M, 1, d, dtype=dtype, device="cuda")
    ends = make(23, 1, 1, 2 * n, 1, 1, d, dtype)
    for cache, x, by in ((k, ends[1], 4.0), (v, ends[2], 1.0)):
        cache[:, :n], cache[:, -n:] = x[:, :n] * by, x[:, n:] * by
    some = [torch.cat((c[:, :n], c[:, -n:]), 1)[0, :, 0].double() for c in (k, v)]
    x = q[0, :, 0].double() @ some[0].T * d ** -0.5
    top = x.amax(-1, keepdim=True).clamp_min(0)
    p = torch.exp(x - top)
    p = p / (p.sum(-1, keepdim=True) + (M - 2 * n) * torch.exp(-top))
    got = ma().global_attention(q, k, v)[0, :, 0].double()
    want = p @ some[1]
    # probabilities off by u and by their exponents' 2 (d + 16) f |q||k|, the sum of 2^24 of them by 2^24 / 64 steps of 2^-24 at most
    # (a thread adds 64 of a tile before they meet a running sum), and u of the result
    u = torch.finfo(dtype).eps / 2
    far = 2 * (d + 16) * _dense.F * (q[0, :, 0].double().abs() @ some[0].T.abs() * d ** -0.5).amax(-1, keepdim=True)
    bound = (far + u + 2.0 ** -6) * (p @ some[1].abs()) + u * want.abs() + 2.0 ** -24
    assert_within(got, want, bound, "out")


def test_empty_calls():
    for B, N, M in ((0, 4, 4), (2, 0, 5), (2, 3, 0)):
        q, k, v, dout = make(14, B, N, M, 4, 2, 16, torch.float16)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = ma().global_attention(*leaves, causal=True)
        assert out.shape == (B, N, 4, 16) and bool((out == 0).all())
        for g, t in zip(torch.autograd.grad(out, leaves, dout), leaves):
            assert g.shape == t.shape and bool((g == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_calls_give_equal_bits(dtype):
    q, k, v, dout = make(15, 2, 300, 500, 4, 2, 64, dtype)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    runs = []
    for _ in range(3):
        out = ma().global_attention(*leaves, causal=True)
        runs.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


@pytest.mark.parametrize("dtype", DTYPES)
def test_graphs_and_streams(dtype):
    """Captured and replayed with new values, on a side stream, two graphs and an eager call at once, the backward among them, while an
    eager graph of the same leaves lives."""
    B, N, M, h, hk, d = 2, 40, 700, 4, 2, 64
    q, k, v, dout = make(16, B, N, M, h, hk, d, dtype)
    lengths = ints([M, 300])
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        out = ma().global_attention(*leaves, causal=True, lengths=lengths)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    def one():
        with torch.no_grad():
            return ma().global_attention(q[:, :1], k, v, causal=True, lengths=lengths)

    # an eager graph of the same leaves (of the capture's stream: torch refuses the capture of any operator otherwise)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = ma().global_attention(*leaves, causal=True)
        step(), one()
    graphs, held = [], []
    for f in (step, one, one):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held.append(f())
        graphs.append(graph)
    with torch.no_grad():
        for i, t in enumerate((q, k, v)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(40 + i)).to(dtype))
        lengths.copy_(ints([333, M]))
    for graph, stream in zip(graphs[1:], (torch.cuda.Stream(), torch.cuda.Stream())):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph.replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(held[1], one()) and torch.equal(held[2], one())
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held[0], again))
    # (the values under the first graph's saved tensors were changed in place: only that its memory still stands is asked)
    assert alive.shape == q.shape


def test_inputs_of_another_stream_and_profiler_name():
    q, k, v, _ = make(17, 1, 64, 64, 2, 2, 32, torch.float16)
    want = ma().global_attention(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ma().global_attention(q, k, v)
    side.synchronize()
    assert torch.equal(got, want)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        ma().global_attention(q, k, v)
    assert any("global_attention" in e.key for e in prof.key_averages())


def test_custom_op_and_compile():
    import matchattention_b200.ops as ops
    q, k, v, _ = make(18, 2, 64, 64, 4, 2, 32, torch.float16)
    want = ma().global_attention(q, k, v, causal=True, cap=4.0)
    got = torch.ops.matchattn_b200.global_attention_op(q, k, v, 32 ** -0.5, 4.0, None, 1, True, None, None, None, None)
    assert torch.equal(got, want)
    torch.library.opcheck(ops.global_attention_op, (q, k, v, 32 ** -0.5, 4.0, None, 1, True, None, None, None, None),
                          test_utils=("test_schema", "test_faketensor"))


def test_subclasses_and_modes_take_the_python_path():
    from torch.overrides import TorchFunctionMode

    class Mode(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    q, k, v, _ = make(19, 2, 64, 80, 4, 2, 32, torch.float16)
    lengths = ints([70, 10])
    want = ma().global_attention(q, k, v, causal=True, lengths=lengths)
    with Mode():
        assert torch.equal(ma().global_attention(q, k, v, causal=True, lengths=lengths), want)
    negative = torch._neg_view(-q)
    assert torch.equal(ma().global_attention(negative, k, v, causal=True, lengths=lengths), want)


def test_refusals_on_the_device():
    q, k, v, _ = make(20, 2, 8, 8, 4, 2, 16, torch.float16)
    f = ma().global_attention
    with pytest.raises(TypeError):
        f(q, k.float(), v)
    with pytest.raises(ValueError):
        f(q, k[:, :, :, :8], v[:, :, :, :8])
    with pytest.raises(ValueError):
        f(q[:, :, :3], k, v)
    with pytest.raises(ValueError):
        f(q, k, v[:, :4])
    with pytest.raises(ValueError):
        f(q, k, v, prefix=ints([1, 2]))
    with pytest.raises(TypeError):
        f(q, k, v, lengths=torch.ones(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        f(q, k, v, lengths=ints([1, 2, 3]))
    with pytest.raises(RuntimeError):
        f(q, k, v, lengths=torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        f(q, k, v, width=0)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            f(q, k, v, scale=bad)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            f(q, k, v, cap=bad)
    with pytest.raises(NotImplementedError):
        f(q, k, v, slopes=torch.ones(4, device="cuda", requires_grad=True))
    with pytest.raises(ValueError):
        f(q, k, v, documents=(None, ints([[0] * 8] * 2)))
    with pytest.raises(ValueError):
        f(torch.zeros(1, 2, 1, 257, device="cuda"), torch.zeros(1, 2, 1, 257, device="cuda"), torch.zeros(1, 2, 1, 257, device="cuda"))
    with pytest.raises(ValueError):
        f(q[0], k[0], v[0])
    with pytest.raises(RuntimeError):
        f(q.cpu(), k, v)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_another_device_than_the_current_one():
    q, k, v, _ = (t.to("cuda:1") for t in make(21, 1, 64, 64, 2, 2, 32, torch.float16))
    want, bound = _dense.attention(q, k, v)
    assert_within(ma().global_attention(q, k, v), want[0], bound[0], "out")
