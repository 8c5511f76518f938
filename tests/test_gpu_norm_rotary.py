"""norm_rotary against its definition in 64 bits (bounds in _dense.py), and the run of it with global_attention."""
import math

import pytest
import torch

import _dense
from _dense import assert_within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def ma():
    import matchattention_b200
    return matchattention_b200


def angles(positions, rot, axes, theta=10000.0):
    n = rot // 2 // axes
    inv = theta ** (-torch.arange(n, dtype=torch.float64, device="cuda") / max(n, 1))
    at = positions.double()
    at = at[..., None] if axes == 1 else at
    angle = (at[..., None] * inv).flatten(-2)[..., None, :]
    return angle if angle.dim() == 4 else angle[None]


def run(dtype, B, N, h, hk, d, rot, axes=1, weights="same", positions=None, train=True, seed=0, eps=1e-6, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    fused = (draw(B, N, (h + hk) * d) * spread).to(dtype).cuda()
    q, k = fused[..., : h * d].view(B, N, h, d), fused[..., h * d:].view(B, N, hk, d)
    wtype = {"same": dtype, "float": torch.float32, None: None}[weights]
    qw, kw = ((1 + 0.3 * draw(d)).to(wtype).cuda() if weights else None for _ in range(2))
    if positions is None:
        positions = torch.randint(-50, 5000, (B, N) if axes == 1 else (B, N, 2), generator=gen).int().cuda()
    freqs = ma().rotary_frequencies(rot, axes=axes, device="cuda") if rot else None
    angle = angles(positions, rot, axes) if rot else None
    leaves = [t.detach().requires_grad_(train) if t is not None else None for t in (q, k, qw, kw)]
    yq, yk = ma().norm_rotary(leaves[0], leaves[1], freqs, positions if rot else None, q_weight=leaves[2], k_weight=leaves[3], eps=eps)
    dq, dk = (draw(*t.shape).to(dtype).cuda() for t in (q, k))
    if train:
        wanted = [t for t in leaves if t is not None]
        grads = torch.autograd.grad((yq, yk), wanted, (dq, dk))
    for name, x, w, y, dy, i in (("q", q, qw, yq, dq, 0), ("k", k, kw, yk, dk, 1)):
        want, bound = _dense.norm(x, w, freqs, angle, eps, dy if train else None)
        assert_within(y.detach(), want[0], bound[0], name)
        if train:
            assert_within(grads[i], want[1], bound[1], "d" + name)
            if w is not None:
                assert grads[2 + i].dtype == w.dtype
                assert_within(grads[2 + i], want[2], bound[2], "d weight of " + name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot", [(1, 0), (2, 2), (7, 4), (16, 16), (16, 0), (24, 8), (32, 16), (40, 40), (40, 16), (64, 64), (80, 32), (96, 96),
                                   (128, 128), (128, 32), (129, 100), (250, 250), (256, 256), (256, 64)])
def test_widths(d, rot, dtype):
    run(dtype, 2, 19, 3, 2, d, rot)
    if rot % 4 == 0:
        run(dtype, 1, 33, 2, 1, d, rot, axes=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N,h,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (16, 1, 32, 8), (3, 700, 9, 3), (1, 2049, 17, 1), (2, 1, 200, 100)])
@pytest.mark.parametrize("weights", ["same", "float", None])
def test_heads_tokens_and_weights(B, N, h, hk, weights, dtype):
    run(dtype, B, N, h, hk, 64, 64, weights=weights)


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_positions(dtype):
    """Angles stay exact at positions of millions, below zero, beyond 32 bits."""
    N = 40
    for start in (10 ** 6, 2 ** 31 - 64, -10 ** 6):
        run(dtype, 1, N, 2, 1, 64, 64, positions=(start + torch.arange(N)).int().cuda())
    # 64-bit positions: the angle of position p + 2^40 is taken from the table's own exact product
    far = (2 ** 40 + torch.arange(N)).cuda()
    q = torch.randn(1, N, 2, 64, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    freqs = ma().rotary_frequencies(64, device="cuda")
    turns = [[(int(f) % 2 ** 64) * int(p) % 2 ** 64 / 2.0 ** 64 for f in freqs[0].tolist()] for p in far.tolist()]
    angle = 2 * math.pi * torch.tensor(turns, dtype=torch.float64, device="cuda")[None, :, None]
    want, bound = _dense.norm(q, None, freqs, angle, 1e-6)
    assert_within(ma().norm_rotary(q, None, freqs, far), want[0], bound[0], "q")


def test_frequencies():
    table = ma().rotary_frequencies(64, theta=500000.0, axes=2)
    assert table.shape == (2, 16) and table.dtype == torch.int64 and torch.equal(table[0], table[1])
    for j, t in enumerate(table[0].tolist()):
        assert abs((t % 2 ** 64) / 2.0 ** 64 * 2 * math.pi - 500000.0 ** (-j / 16)) < 1e-12


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_for_all_items_and_map(dtype):
    W, H = 13, 9
    column, row = torch.arange(H * W) % W, torch.arange(H * W) // W
    run(dtype, 3, H * W, 4, 2, 32, 32, axes=2, positions=torch.stack((column, row), -1).int().cuda())
    run(dtype, 3, H * W, 4, 2, 32, 32, positions=torch.arange(H * W).cuda())
    run(dtype, 3, H * W, 4, 2, 32, 32, positions=torch.arange(H * W).view(1, -1).cuda())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_zeros_and_of_large_values(dtype):
    run(dtype, 1, 5, 2, 1, 64, 64, spread=0.0)
    run(dtype, 1, 5, 2, 1, 64, 64, spread=2.0 ** 12)
    run(dtype, 1, 5, 2, 1, 64, 64, spread=2.0 ** -9)


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_alone_strides_and_partial_gradients(dtype):
    gen = torch.Generator().manual_seed(5)
    base = torch.randn(4, 2, 31, 64, generator=gen).to(dtype).cuda()
    freqs, at = ma().rotary_frequencies(64, device="cuda"), torch.arange(31).cuda()
    angle = angles(at, 64, 1)
    w = torch.ones(64, device="cuda")
    for q in (base.permute(1, 2, 0, 3), base.permute(1, 2, 0, 3).flip(-1), base.view(2, 31, 4, 64)[:, ::2], base.view(-1)[1:1 + 31 * 64].view(1, 31, 1, 64)):
        a = angle[:, :q.size(1)]
        want, bound = _dense.norm(q, w, freqs, a, 1e-6)
        assert_within(ma().norm_rotary(q, None, freqs, at[:q.size(1)], q_weight=w), want[0], bound[0], "q")
    q = base.permute(1, 2, 0, 3)
    weight = torch.randn(64, generator=gen).cuda().requires_grad_()
    dy = torch.randn(q.shape, generator=gen).to(dtype).cuda()
    want, bound = _dense.norm(q, weight.detach(), freqs, angle, 1e-6, dy)
    (got,) = torch.autograd.grad(ma().norm_rotary(q, None, freqs, at, q_weight=weight), weight, dy)
    assert_within(got, want[2], bound[2], "weight")
    # only k's result is used: q's gradient is zero
    a, b = (t.detach().clone().requires_grad_() for t in (q, q))
    ya, yb = ma().norm_rotary(a, b, freqs, at)
    da, db = torch.autograd.grad(yb, (a, b), dy, allow_unused=True)
    assert da is None or bool((da == 0).all())
    want, bound = _dense.norm(q, None, freqs, angle, 1e-6, dy)
    assert_within(db, want[1], bound[1], "k")


def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(6)
    q = torch.randn(1, 5, 2, 12, generator=gen).cuda().requires_grad_()
    w = (1 + 0.1 * torch.randn(12, generator=gen)).cuda().requires_grad_()
    freqs, at = ma().rotary_frequencies(8, device="cuda"), torch.arange(5).cuda()
    dy = torch.randn(q.shape, generator=gen).cuda()
    f = lambda x, y: (ma().norm_rotary(x, None, freqs, at, q_weight=y).double() * dy.double()).sum()  # noqa: E731
    grads = torch.autograd.grad(f(q, w), (q, w))
    for i, t in enumerate((q, w)):
        way = torch.randn(t.shape, generator=gen).cuda()
        step = 2.0 ** -8
        ends = [f(*[x.detach() + (s * step * way if j == i else 0) for j, x in enumerate((q, w))]) for s in (1, -1)]
        slope, want = float((ends[0] - ends[1]) / (2 * step)), float((grads[i].double() * way.double()).sum())
        # third derivative times step^2 / 6, and float32 roundings (2^-20 of sums of order 100) over the step
        assert abs(slope - want) <= 0.02 * max(1.0, abs(want))


def test_empty_calls():
    freqs = ma().rotary_frequencies(32, device="cuda")
    q = torch.zeros(2, 0, 4, 32, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    y, z = ma().norm_rotary(q, q, freqs, torch.zeros(0, dtype=torch.int32, device="cuda"), q_weight=w)
    assert y.shape == q.shape and z.shape == q.shape
    assert bool((torch.autograd.grad(y.sum(), w)[0] == 0).all())


def test_bits_and_graph():
    freqs = ma().rotary_frequencies(32, device="cuda")
    w = torch.ones(32, device="cuda", requires_grad=True)
    q = torch.randn(2, 300, 4, 32, generator=torch.Generator().manual_seed(1)).half().cuda().requires_grad_()
    at = torch.arange(300).cuda()
    dy = torch.ones_like(q)

    def step():
        out = ma().norm_rotary(q, q, freqs, at, q_weight=w, k_weight=w)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (q, w), (dy, dy))]

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    at.add_(1000)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step())) and not torch.equal(held[0], first[0])


def test_captured_backward_while_an_eager_graph_of_the_leaves_lives():
    gen = torch.Generator().manual_seed(2)
    q, k = (torch.randn(2, 30, h, 32, generator=gen).half().cuda().requires_grad_() for h in (4, 2))
    w = torch.ones(32, device="cuda", requires_grad=True)
    freqs, at = ma().rotary_frequencies(32, device="cuda"), torch.arange(30).cuda()

    def step():
        out = ma().norm_rotary(q, k, freqs, at, q_weight=w)
        return [*(t.detach() for t in out), *torch.autograd.grad(out, (q, k, w), [torch.ones_like(t) for t in out])]

    # an eager graph of another stream makes torch refuse the capture, whatever the operator: this one is of the capture's own
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        alive = ma().norm_rotary(q, k, freqs, at, q_weight=w)
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = step()
    graph.replay()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        again = step()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, again))
    assert torch.equal(alive[0].detach(), held[0])


def test_refusals():
    f, freqs = ma().norm_rotary, ma().rotary_frequencies(32, device="cuda")
    q = torch.zeros(2, 3, 4, 32, device="cuda")
    at = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        f(q, None, freqs, None)
    with pytest.raises(ValueError):
        f(q, None, freqs, at[:2])
    with pytest.raises(TypeError):
        f(q, None, freqs, at.float())
    with pytest.raises(TypeError):
        f(q, q.half(), freqs, at)
    with pytest.raises(ValueError):
        f(q, q[:, :2], freqs, at)
    with pytest.raises(ValueError):
        f(q, None, freqs, at, k_weight=torch.ones(32, device="cuda"))
    with pytest.raises(TypeError):
        f(q.half(), None, freqs, at, q_weight=torch.ones(32, device="cuda").bfloat16())
    with pytest.raises(TypeError):
        f(q.half(), q.half(), freqs, at, q_weight=torch.ones(32, device="cuda").half(), k_weight=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError):
        f(q, None, freqs, at, q_weight=torch.ones(31, device="cuda"))
    with pytest.raises(ValueError):
        f(q, None, ma().rotary_frequencies(64, device="cuda"), at)
    with pytest.raises(ValueError):
        f(q, None, freqs, at, eps=-1.0)
    with pytest.raises(RuntimeError):
        f(q, None, freqs, at.cpu())
    with pytest.raises(ValueError):
        ma().rotary_frequencies(6, axes=2)


def test_custom_op():
    import matchattention_b200.ops as ops
    q = torch.randn(2, 5, 4, 32, generator=torch.Generator().manual_seed(1)).half().cuda()
    freqs, at = ma().rotary_frequencies(32, device="cuda"), torch.arange(5).cuda()
    want = ma().norm_rotary(q, q, freqs, at)
    got = torch.ops.matchattn_b200.norm_rotary_op(q, q, freqs, at, None, None, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.library.opcheck(ops.norm_rotary_op, (q, q, freqs, at, None, None, 1e-6), test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_layer_and_its_new_tokens(dtype):
    """Norm, rotation and attention as a layer runs them, forward and backward; then the same sequence token by token over a cache:
    the last rows agree."""
    B, N, h, hk, d = 2, 150, 4, 2, 64
    gen = torch.Generator().manual_seed(21)
    fused = torch.randn(B, N, (h + 2 * hk) * d, generator=gen).to(dtype).cuda().requires_grad_()
    weight = (1 + 0.1 * torch.randn(d, generator=gen)).cuda().requires_grad_()
    freqs, at = ma().rotary_frequencies(d, device="cuda"), torch.arange(N).cuda()
    dout = torch.randn(B, N, h, d, generator=gen).to(dtype).cuda()

    def layer(x, positions):
        q, k, v = (x[..., a:b].unflatten(-1, (-1, d)) for a, b in ((0, h * d), (h * d, (h + hk) * d), ((h + hk) * d, (h + 2 * hk) * d)))
        q, k = ma().norm_rotary(q, k, freqs, positions, q_weight=weight, k_weight=weight)
        return q, k, v

    q, k, v = layer(fused, at)
    out = ma().global_attention(q, k, v, causal=True, cap=20.0)
    grads = torch.autograd.grad(out, (fused, weight), dout, retain_graph=True)
    # the same in 64 bits from the roundings that the 16-bit tensors between the two take
    want, bound = _dense.attention(q.detach(), k.detach(), v.detach(), causal=True, cap=20.0, dout=dout)
    assert_within(out.detach(), want[0], bound[0], "out")
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    raw = fused.detach()
    angle = angles(at, d, 1)
    far = 0
    for x, dy, a, b in ((raw[..., : h * d], dq, 0, h * d), (raw[..., h * d: (h + hk) * d], dk, h * d, (h + hk) * d)):
        w, bd = _dense.norm(x.unflatten(-1, (-1, d)), weight.detach(), freqs, angle, 1e-6, dy)
        assert_within(grads[0][..., a:b].unflatten(-1, (-1, d)), w[1], bd[1], "fused")
        far = far + w[2]
    assert bool((grads[1].double() - far).abs().max() <= 2.0 ** -15 * far.abs().max())
    assert torch.equal(grads[0][..., (h + hk) * d:].unflatten(-1, (-1, d)), dv)
    with torch.no_grad():
        cache_k, cache_v = (torch.full((B, N + 10, hk, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        cache_k[:, : N - 3], cache_v[:, : N - 3] = k[:, : N - 3], v[:, : N - 3]
        for n in range(N - 3, N):
            qn, kn, vn = layer(fused[:, n: n + 1].detach(), at[n: n + 1])
            assert torch.equal(qn, q[:, n: n + 1]) and torch.equal(kn, k[:, n: n + 1])
            cache_k[:, n], cache_v[:, n] = kn[:, 0], vn[:, 0]
            new = ma().global_attention(qn, cache_k, cache_v, causal=True, cap=20.0, lengths=torch.full((B,), n + 1, dtype=torch.int32, device="cuda"))
            assert_within(new, want[0][:, n: n + 1], bound[0][:, n: n + 1], "token")
