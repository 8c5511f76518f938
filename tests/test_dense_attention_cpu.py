"""What global_attention and norm_rotary refuse, and their 64-bit oracle; no GPU."""
import ctypes

import pytest
import torch

import _dense
import matchattention_b200 as ma
from matchattention_b200 import _lib

AT = 4096       # never dereferenced


def attention_args(**changes):
    a = dict(q=AT, k=AT, v=AT, out=AT, lse=AT, B=1, N=8, M=8, h=4, hk=2, d=16, dtype=1, causal=0, width=1, scale=0.25, cap=0.0)
    a.update(changes)
    for n in ("q_stride", "k_stride", "v_stride"):
        a[n] = a.get(n, (512, 64, 16))
    return _lib.GlobalArgs(**a)


def forward(scratch=AT, nbytes=1 << 30, **changes):
    return _lib.lib.matchattn_global_forward(attention_args(**changes), scratch, nbytes, None)


def test_attention_arguments_are_rejected_on_the_host():
    for name in ("q", "k", "v", "out"):
        assert forward(**{name: None}) == 1
        assert forward(**{name: AT + 1}) == 7
    assert _lib.lib.matchattn_global_forward(None, AT, 1 << 30, None) == 1
    for bad in (dict(B=0), dict(N=0), dict(M=-1), dict(h=0), dict(hk=0), dict(h=3), dict(d=0), dict(d=257), dict(width=0),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(cap=-1.0), dict(cap=float("nan")),
                dict(cap=float("inf")), dict(prefix=AT)):
        assert forward(**bad) == 2, bad
    assert forward(dtype=3) == 4 and forward(dtype=-1) == 4
    assert forward(slopes=AT + 2) == 7 and forward(lengths=AT + 2) == 7 and forward(q_docs=AT + 1, k_docs=AT) == 7
    assert forward(q_docs=AT) == 1 and forward(k_docs=AT) == 1
    assert forward(N=(1 << 24) + 1) == 8 and forward(M=(1 << 24) + 1) == 8 and forward(B=65536) == 8 and forward(h=65536, hk=65536) == 8
    assert forward(N=1 << 24, h=128, hk=1) == 8
    # few queries over many keys: scratch is asked for, and not less
    many = dict(N=1, M=1 << 20)
    need = _lib.lib.matchattn_global_scratch_bytes(attention_args(**many), 0)
    assert need > 0
    assert forward(scratch=None, **many) == 1 and forward(nbytes=need - 1, **many) == 10 and forward(scratch=AT + 4, **many) == 7
    assert _lib.lib.matchattn_global_scratch_bytes(attention_args(d=257), 0) == 0


def test_attention_backward_arguments_are_rejected_on_the_host():
    def backward(dout=AT, dq=AT, dk=AT, dv=AT, scratch=AT, nbytes=1 << 30, **changes):
        return _lib.lib.matchattn_global_backward(attention_args(**changes), dout, dq, dk, dv, scratch, nbytes, None)

    for name in ("dout", "dq", "dk", "dv", "scratch", "lse"):
        assert backward(**{name: None}) == 1, name
    for name in ("dout", "dq", "dk", "dv", "scratch"):
        assert backward(**{name: AT + 1}) == 7, name
    need = _lib.lib.matchattn_global_scratch_bytes(attention_args(), 1)
    assert need > 0 and backward(nbytes=need - 1) == 10
    assert backward(hk=3) == 2


def norm_args(**changes):
    a = dict(q=AT, k=AT, q_weight=AT, k_weight=AT, positions=AT, freqs=AT, axes=1, rot=16, B=1, N=8, h=4, hk=2, d=16, dtype=1, weight_dtype=1,
             eps=1e-6, q_stride=(512, 64, 16), k_stride=(256, 32, 16))
    a.update(changes)
    return _lib.NormArgs(**a)


def test_norm_arguments_are_rejected_on_the_host():
    def forward(q_out=AT, k_out=AT, **changes):
        return _lib.lib.matchattn_norm_rotary_forward(norm_args(**changes), q_out, k_out, None)

    for bad in (dict(q=None), dict(k=None), dict(positions=None), dict(freqs=None), dict(q_out=None), dict(k_out=None)):
        assert forward(**bad) == 1, bad
    for bad in (dict(B=0), dict(N=0), dict(h=0), dict(hk=-1), dict(d=0), dict(d=257), dict(rot=18), dict(rot=15), dict(axes=0), dict(axes=3),
                dict(axes=2, rot=6), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf"))):
        assert forward(**bad) == 2, bad
    assert forward(dtype=5) == 4 and forward(weight_dtype=2) == 4
    assert forward(q=AT + 1) == 7 and forward(k_weight=AT + 1) == 7 and forward(freqs=AT + 4) == 7 and forward(positions=AT + 2) == 7
    assert forward(positions=AT + 4, positions_64=1) == 7
    assert forward(N=1 << 30) == 8

    def backward(gq=AT, gk=AT, dq=AT, dk=AT, dqw=AT, dkw=AT, scratch=AT, nbytes=1 << 30, **changes):
        return _lib.lib.matchattn_norm_rotary_backward(norm_args(**changes), gq, gk, dq, dk, dqw, dkw, scratch, nbytes, None)

    for bad in (dict(gq=None), dict(gk=None), dict(dq=None), dict(dk=None), dict(scratch=None), dict(q_weight=None)):
        assert backward(**bad) == 1, bad
    need = _lib.lib.matchattn_norm_rotary_scratch_bytes(16)
    assert need > 0 and backward(nbytes=need - 1) == 10 and backward(scratch=AT + 2) == 7
    assert _lib.lib.matchattn_norm_rotary_scratch_bytes(0) == 0 and _lib.lib.matchattn_norm_rotary_scratch_bytes(257) == 0


def test_structures_have_the_size_that_the_header_gives_them():
    assert ctypes.sizeof(_lib.GlobalArgs) == 6 * 8 + 9 * 8 + 5 * 8 + 9 * 4 + 2 * 4 + 4
    assert ctypes.sizeof(_lib.NormArgs) == 2 * 8 + 6 * 8 + 4 * 8 + 8 + 10 * 4 + 4 + 4


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 2, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ma.global_attention(q, q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        ma.norm_rotary(q)


def test_frequencies():
    assert ma.rotary_frequencies(0).shape == (1, 0)
    table = ma.rotary_frequencies(8)
    assert table.shape == (1, 4) and (int(table[0, 0]) % 2 ** 64) / 2.0 ** 64 == pytest.approx(0.15915494309189535, abs=1e-15)
    for bad in (dict(rot=3), dict(rot=6, axes=2), dict(rot=4, axes=3), dict(rot=-2), dict(rot=4, theta=0.0)):
        with pytest.raises(ValueError):
            ma.rotary_frequencies(**bad)


def test_oracle_against_autograd():
    """The oracle's formulas against autograd over the plain softmax."""
    gen = torch.Generator().manual_seed(0)
    B, N, M, h, hk, d = 2, 5, 7, 4, 2, 6
    q, k, v, dout = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((B, N, h, d), (B, M, hk, d), (B, M, hk, d), (B, N, h, d)))
    slopes = torch.tensor([0.1, 0.2, 0.3, 0.4])
    want, _ = _dense.attention(q.float(), k.float(), v.float(), cap=2.0, slopes=slopes, width=3, causal=True, prefix=torch.tensor([0, 4]),
                               dout=dout.float())
    leaves = [t.float().double().requires_grad_() for t in (q, k, v)]
    kk, vv = (t.repeat_interleave(2, 2) for t in leaves[1:])
    s = torch.einsum("bnhd,bmhd->bhnm", leaves[0], kk) * d ** -0.5
    s = 2.0 * torch.tanh(s / 2.0)
    at, key = torch.arange(N) + M - N, torch.arange(M)
    far = (at[:, None] % 3 - key % 3).abs() + (at[:, None] // 3 - key // 3).abs()
    s = s - slopes.double()[:, None, None] * far
    seen = (key <= at[:, None]) | (key < torch.tensor([0, 4])[:, None, None])
    p = s.masked_fill(~seen[:, None], float("-inf")).softmax(-1)
    out = torch.einsum("bhnm,bmhd->bnhd", p, vv)
    got = [out, *torch.autograd.grad(out, leaves, dout.float().double())]
    for a, b in zip(want, got):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_norm_oracle_against_autograd():
    gen = torch.Generator().manual_seed(1)
    x, dy, w = torch.randn(2, 3, 2, 8, generator=gen), torch.randn(2, 3, 2, 8, generator=gen), torch.randn(8, generator=gen)
    angle = torch.randn(1, 3, 1, 2, generator=gen, dtype=torch.float64)
    want, _ = _dense.norm(x, w, None, angle, 1e-6, dy)
    a, b = x.double().requires_grad_(), w.double().requires_grad_()
    y = a / (a.square().mean(-1, keepdim=True) + 1e-6).sqrt() * b
    c, s = torch.cos(angle), torch.sin(angle)
    y = torch.cat((y[..., :2] * c - y[..., 2:4] * s, y[..., 2:4] * c + y[..., :2] * s, y[..., 4:]), -1)
    for got, ref in zip([y, *torch.autograd.grad(y, (a, b), dy.double())], want):
        assert torch.allclose(got, ref, rtol=1e-12, atol=1e-12)
