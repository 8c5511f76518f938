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


def test_second_derivatives_are_refused():
    """Gradients with a graph are the same numbers; a second pass through them is an error, also where another term has one."""
    for dtype in (torch.float32, torch.float16):
        q, k, v, dout = (t.requires_grad_() for t in make((1, 40, 2, 16), (1, 50, 2, 16), (1, 50, 2, 16), (1, 40, 2, 16), dtype=dtype))
        w = torch.ones(16, device="cuda", requires_grad=True)
        calls = ((lambda: ma().global_attention(q, k, v), (q, k, v), dout), (lambda: ma().norm_rotary(q, q_weight=w), (q, w), dout))
        for call, leaves, grad in calls:
            want = torch.autograd.grad(call(), leaves, grad.detach())
            got = torch.autograd.grad(call(), leaves, grad, create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(want, got))
            for g in got:
                with pytest.raises(RuntimeError, match="gradients of the gradients"):
                    torch.autograd.grad(g.float().square().sum() + q.float().square().sum(), q, retain_graph=True)
        # a graph that does not lead back through the operator is left alone
        loss = q.float().pow(3).sum()
        (first,) = torch.autograd.grad(loss, q, create_graph=True)
        assert torch.autograd.grad(first.float().sum(), q)[0].shape == q.shape


def test_tangents_are_refused():
    """Forward-mode differentiation has no rule here: a dual tensor is refused, with and without gradients, and not stripped."""
    import torch.autograd.forward_ad as forward_ad
    q, k, v, t = make(*[(1, 9, 2, 16)] * 4)
    w, tw = make((16,), (16,))
    slopes, ts = make((2,), (2,))
    with forward_ad.dual_level():
        for name in ("q", "k", "v", "slopes"):
            args = dict(q=q, k=k, v=v, slopes=slopes)
            args[name] = forward_ad.make_dual(args[name], ts if name == "slopes" else t)
            with pytest.raises(NotImplementedError):
                ma().global_attention(**args)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                ma().global_attention(**args)
        for args in (dict(q=forward_ad.make_dual(q, t)), dict(q=q, k=forward_ad.make_dual(k, t)), dict(q=q, q_weight=forward_ad.make_dual(w, tw))):
            with pytest.raises(NotImplementedError):
                ma().norm_rotary(**args)
        # others that live in a dual level are not concerned
        assert torch.equal(ma().norm_rotary(q), ma().norm_rotary(q.clone()))


def test_transforms_and_modes_refuse_gradients():
    """Under functional transforms and modes a gradient is refused, and inference under a mode gives the same numbers."""
    from torch.overrides import TorchFunctionMode

    class Mode(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    q, k, v = make(*[(1, 9, 2, 16)] * 3)
    want = ma().global_attention(q, k, v)
    with Mode():
        assert torch.equal(ma().global_attention(q, k, v), want)
        with pytest.raises(NotImplementedError):
            ma().global_attention(q.clone().requires_grad_(), k, v)
        with pytest.raises(NotImplementedError):
            ma().norm_rotary(q.clone().requires_grad_())
    for call in (lambda x: ma().global_attention(x, k, v).sum(), lambda x: ma().norm_rotary(x).sum()):
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.grad(call)(q)
