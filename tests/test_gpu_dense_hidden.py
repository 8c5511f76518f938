"""global_attention: what no query sees, and what other items and heads hold, has no say in a result (bounds in _dense.py)."""
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


def step(tensors, options):
    q, k, v, dout = tensors
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = ma().global_attention(*leaves, **options)
    return [out.detach(), *torch.autograd.grad(out, leaves, dout)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("N", [5, 200, 333])
def test_large_finite_values_in_masked_places(N, d, dtype):
    """Keys behind a length, tokens of no document or of one that no query has, queries that see nothing: 6e4 in their places, next to
    small visible values and gradients."""
    B, M, h, hk = 2, 333, 4, 2
    clean = make(31, B, N, M, h, hk, d, dtype)
    clean[2], clean[3] = clean[2] * 0.02, clean[3] * 2.0 ** -6
    q, k, v, dout = (t.clone() for t in clean)
    k[0, 205:], v[0, 205:] = 6e4, -6e4
    for options in (dict(lengths=ints([205, 333])), dict(causal=True, lengths=ints([205, 333])), dict(lengths=ints([205, 333]), cap=20.0)):
        want, bound = _dense.attention(q, k, v, dout=dout, **options)
        for name, *three in zip(NAMES, step((q, k, v, dout), options), want, bound):
            assert_within(*three, name)
    q, k, v, dout = (t.clone() for t in clean)
    docs_k, docs_q = torch.zeros(B, M, dtype=torch.int32), torch.zeros(B, N, dtype=torch.int32)
    docs_k[:, 100:130], docs_k[:, 130:140], docs_k[:, 250:] = -1, 7, 1
    v[:, 100:140], k[:, 100:140] = 6e4, -6e4
    if N > 5:
        docs_q[:, 120:125], docs_q[:, 125:130], docs_q[:, 130:] = -1, 9, 1
        q[:, 120:130], dout[:, 120:130] = 6e4, 6e4
    documents = (docs_q.cuda(), docs_k.cuda())
    for options in (dict(), dict(causal=True), dict(cap=20.0)):
        options = dict(documents=documents, **options)
        want, bound = _dense.attention(q, k, v, dout=dout, **options)
        for name, *three in zip(NAMES, step((q, k, v, dout), options), want, bound):
            assert_within(*three, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_items_and_key_heads_of_unlike_gradients(causal, dtype):
    """Gradients of two items and two key heads that are 2^10 to 2^20 times as large as one another, each within its own bound."""
    B, N, h, hk, d = 2, 300, 4, 2, 64
    q, k, v, dout = make(32, B, N, N, h, hk, d, dtype)
    dout = dout * torch.tensor([2.0 ** 10, 1.0], device="cuda").view(2, 1, 1, 1).to(dtype)
    dout = dout * torch.tensor([2.0 ** -10, 2.0 ** -10, 1.0, 1.0], device="cuda").view(1, 1, 4, 1).to(dtype)
    got = step((q, k, v, dout), dict(causal=causal))
    for b in range(B):
        for kh in range(hk):
            part = lambda t, n: t[b: b + 1, :, kh * n: (kh + 1) * n]  # noqa: E731
            want, bound = _dense.attention(part(q, 2), part(k, 1), part(v, 1), dout=part(dout, 2), causal=causal)
            for name, g, n, w, e in zip(NAMES, got, (2, 2, 1, 1), want, bound):
                assert_within(part(g, n), w, e, f"{name} of item {b}, key head {kh}")


def test_documents_of_unlike_gradients():
    """float16: packed sequences whose gradients are 2^18 times as large as one another's, each within its own bound."""
    N, h, hk, d = 512, 4, 2, 64
    q, k, v, dout = make(33, 1, N, N, h, hk, d, torch.float16)
    dout[:, :256] *= 2.0 ** 8
    dout[:, 256:] *= 2.0 ** -10
    ids = (torch.arange(N) // 256).int().view(1, N).cuda()
    got = step((q, k, v, dout), dict(causal=True, documents=ids))
    for i in range(2):
        part = lambda t: t[:, 256 * i: 256 * (i + 1)]  # noqa: E731
        want, bound = _dense.attention(part(q), part(k), part(v), dout=part(dout), causal=True)
        for name, g, w, e in zip(NAMES, got, want, bound):
            assert_within(part(g), w, e, f"{name} of document {i}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 4, 200])
@pytest.mark.parametrize("cap", [1e6, 1e4, 2.0])
def test_caps_far_above_the_scores(cap, N, dtype):
    """A cap costs no digits of scores below it: c tanh(x / c) is off by a few 2^-24 of x, so the bounds of calls without a cap hold."""
    tensors = make(34, 2, N, 300, 4, 2, 64, dtype)
    want, _ = _dense.attention(*tensors[:3], dout=tensors[3], cap=cap)
    _, bound = _dense.attention(*tensors[:3], dout=tensors[3])
    if cap == 2.0:
        # the slope of the tanh and what it does to the other figures are in the bounds with a cap
        bound[1:] = _dense.attention(*tensors[:3], dout=tensors[3], cap=cap)[1][1:]
    for name, *three in zip(NAMES, step(tensors, dict(cap=cap)), want, bound):
        assert_within(*three, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 4, 200])
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_bits_do_not_depend_on_hidden_keys_or_other_queries(cap, N, dtype):
    q, k, v, dout = make(35, 1, N, 333, 4, 2, 64, dtype)
    q = q * 0.3         # (scores well below the cap, but for those that are changed)
    options = dict(cap=cap, lengths=ints([300]), causal=True)
    first = step((q, k, v, dout), options)
    k2, v2 = k.clone(), v.clone()
    k2[:, 300:], v2[:, 300:] = k[:, 300:] * 50, 1000.0
    again = step((q, k2, v2, dout), options)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    if N > 1:
        q2 = q.clone()
        q2[:, 1] = q[:, 1] * 50
        again = step((q2, k, v, dout), options)
        rest = [n for n in range(N) if n != 1]
        assert all(torch.equal(a[:, rest], b[:, rest]) for a, b in zip(first[:2], again[:2]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [4, 200])
@pytest.mark.parametrize("ahead", [60.0, 400.0])
def test_a_value_that_is_seen_with_hardly_any_weight(ahead, N, dtype):
    """A NaN value reaches all that see it, whatever the weight that the softmax leaves it: exp(-60) and exp(-400) of the largest
    round to zero in float16, and in every type.  The other document stays as it is."""
    M, h, d = 200, 2, 64
    q, k, v, dout = make(36, 1, N, M, h, h, d, dtype)
    documents = torch.zeros(1, M, dtype=torch.int32, device="cuda")
    documents[:, M // 2:] = 1
    if N < M:
        documents[:, :] = 0
    k[..., 0], q[..., 0] = 0.0, 8.0
    k[:, 0, :, 0] = ahead            # with q's 8 and a scale of 1/8: ahead above the others
    v[0, M - 3 if N < M else 5, 1, 3] = float("nan")
    options = dict(causal=True, documents=(documents[:, M - N:].contiguous(), documents), scale=0.125)
    want, bound = _dense.attention(q, k, v, dout=dout, **options)
    got = step((q, k, v, dout), options)
    assert bool(want[0].isnan().any()) and not bool(want[0].isnan().all())
    for name, g, w in zip(NAMES, got, want):
        assert torch.equal(g.isnan(), w.isnan()), name
    assert_within(got[0], want[0], bound[0], "out")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [2, 150])
@pytest.mark.parametrize("options", [dict(), dict(causal=True), dict(slopes=True)], ids=str)
def test_rows_of_scores_of_minus_infinity(options, N, dtype):
    """Scores that overflow: a query that has no other sees nothing, gives zeros and takes part in no gradient."""
    M, h, d = 200, 2, 64
    q, k, v, dout = make(37, 1, N, M, h, h, d, dtype)
    options = dict(options, slopes=torch.ones(h, device="cuda")) if "slopes" in options else options
    q[:], k[:] = 0.0, -100.0
    q[:, ::2] = 100.0
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ma().global_attention(*leaves, scale=1e35, **options)
    grads = torch.autograd.grad(out, leaves, dout)
    assert bool((out[:, ::2] == 0).all()) and bool(torch.isfinite(out).all()) and bool((out[:, 1::2] != 0).any())
    assert bool((grads[0][:, ::2] == 0).all())
    rest = v.detach().clone().requires_grad_()
    (dv,) = torch.autograd.grad(ma().global_attention(q.detach()[:, 1::2], k.detach(), rest, scale=1e35, causal=False), rest, dout[:, 1::2].contiguous())
    if not options:
        assert torch.allclose(grads[2].float(), dv.float(), rtol=4 * torch.finfo(dtype).eps, atol=2.0 ** -10)
