"""global_attention and norm_rotary in 64 bits, and how far a result in a type may lie from them.

Bounds, per element (u: half a step of the type, torch.finfo(t).eps / 2; f = 2^-22: an operation in float32, four times its half
step, which also covers the truncating adders of the matrix units and an approximate exponential):

* a score of absolute terms X = scale * sum |q||k| is off by at most  dx = (d + 16) f (X + cap + |bias|);
* a probability is off by at most  (2 dx + (M + 16) f) p  and, in 16-bit types, by u p more, for the product with v or dout;
* out: that times |v|, summed, and u |out| for the last rounding;
* dP is off by (d + 4) f sum |dout||v|, delta by u sum |dout||out| (out was rounded) plus (d + 4) f of it; dS by its factors' errors
  and, in 16-bit types, u |dS|; dQ, dK, dV by the errors of what is summed, (M + N + 16) f of the absolute sum, and u of the result.

Below the types' normal ranges steps are absolute: a result is off by half the smallest number of its type (float16: 2^-25); an
exponential below 2^-126 may be zero; a float16 probability, held against the largest of its row, by 2^-25, in the backward pass, held
times 2^12 against the row's sum, by 2^-37; a float16 dS, held so that the largest that row norms of dout and v allow, twice their
product, lies between 2^14 and 2^15, by 2^-25 of that: 2^-38 of the product of the norms.
"""
import torch

F = 2.0 ** -22


def _expand(t, g):
    return t.repeat_interleave(g, dim=2) if g > 1 else t


def visible(B, N, M, causal, prefix, lengths, documents, device):
    key = torch.arange(M, device=device)[None, None, :]
    length = torch.full((B, 1, 1), M, device=device) if lengths is None else lengths.clamp(0, M).view(B, 1, 1)
    at = torch.arange(N, device=device)[None, :, None] + length - N
    seen = (key < length).expand(B, N, M)
    if causal:
        open_ = key <= at
        if prefix is not None:
            open_ = open_ | (key < prefix.view(B, 1, 1))
        seen = seen & open_
    if documents is not None:
        qd, kd = documents
        seen = seen & (qd[:, :, None] == kd[:, None, :]) & (qd[:, :, None] >= 0)
    return seen, at


def attention(q, k, v, *, scale=None, cap=0.0, slopes=None, width=1, causal=False, prefix=None, lengths=None, documents=None, dout=None):
    """(results, bounds): [out] or [out, dq, dk, dv] in float64 and the bounds above for q's type."""
    t = q.dtype
    u = torch.finfo(t).eps / 2
    u16 = 0.0 if t == torch.float32 else u
    last = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    half = t == torch.float16
    low, low_back = (2.0 ** -25, 2.0 ** -36) if half else (2.0 ** -125, 2.0 ** -125)
    B, N, h, d = q.shape
    M, hk = k.shape[1:3]
    g = h // hk
    scale = d ** -0.5 if scale is None else scale
    if documents is not None and not isinstance(documents, (tuple, list)):
        documents = (documents, documents)
    seen, at = visible(B, N, M, causal, prefix, lengths, documents, q.device)
    seen = seen[:, None]
    # a key or a query that takes part in no visible pair does not matter, whatever its values
    used_k, used_q = seen.any(2).view(B, M, 1, 1), seen.any(3).view(B, N, 1, 1)
    zero = lambda x, m: torch.where(m, x.double(), torch.zeros((), dtype=torch.float64, device=x.device))  # noqa: E731
    q6 = zero(q, used_q).permute(0, 2, 1, 3)
    k6, v6 = (_expand(zero(x, used_k), g).permute(0, 2, 1, 3) for x in (k, v))
    s = q6 @ k6.transpose(-1, -2) * scale
    X = q6.abs() @ k6.abs().transpose(-1, -2) * scale
    slant = torch.ones_like(s)
    if cap:
        slant = 1 - torch.tanh(s / cap) ** 2
        s = cap * torch.tanh(s / cap)
    bias = torch.zeros((), dtype=torch.float64, device=q.device)
    if slopes is not None:
        key = torch.arange(M, device=q.device)[None, None, :]
        row = lambda p: torch.div(p, width, rounding_mode="floor")  # noqa: E731
        far = (at % width - key % width).abs() + (row(at) - row(key)).abs()
        bias = slopes.double().view(1, h, 1, 1) * far.double()[:, None]
        s = s - bias
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True) if M else s.new_zeros(B, h, N, 1)
    top = torch.where(torch.isneginf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    group = lambda x: back(x.view(B, hk, g, M, d).sum(2))  # noqa: E731
    # a value is multiplied only where its pair is visible
    def safe(w, x):
        if bool(torch.isfinite(x).all()):
            return w @ x
        return (w[..., None] * x[..., None, :, :]).masked_fill(w[..., None] == 0, 0).sum(-2)

    o = safe(p, v6)
    dx = (d + 16) * F * (X + cap + bias.abs())
    rho = 2 * dx.masked_fill(~seen, 0).amax(-1, keepdim=True) + (M + 16) * F if M else torch.zeros_like(total)
    results = [back(o)]
    near = (p * (rho + u16) + low).masked_fill(~seen, 0)
    bounds = [back(safe(near, v6.abs()) + u * o.abs() + last)]
    if dout is None:
        return results, bounds
    do = zero(dout, used_q).permute(0, 2, 1, 3)
    dp = do @ v6.transpose(-1, -2)
    delta = (do * o).sum(-1, keepdim=True)
    ds = (p * (dp - delta) * slant).masked_fill(~seen, 0)
    far_dp = (d + 4) * F * (do.abs() @ v6.abs().transpose(-1, -2))
    far_delta = ((u + (d + 4) * F) * (do * o).abs() + do.abs() * bounds[0].permute(0, 2, 1, 3)).sum(-1, keepdim=True)
    far_slant = 4 * dx / cap if cap else 0.0
    far_ds = (p * slant * (far_dp + far_delta) + (rho + u16) * ds.abs() + p * (dp - delta).abs() * far_slant)
    norms = do.norm(dim=-1).max() * v6.norm(dim=-1).max()
    far_ds = (far_ds + low_back * slant * (dp - delta).abs() + (2.0 ** -38 * norms if half else 0.0)).masked_fill(~seen, 0)
    dq, dk, dv = scale * (ds @ k6), scale * (ds.transpose(-1, -2) @ q6), p.transpose(-1, -2) @ do
    sums = (M + N + 16) * F
    far_dq = scale * ((far_ds + sums * ds.abs()) @ k6.abs()) + u * dq.abs() + last
    far_dk = scale * ((far_ds + sums * ds.abs()).transpose(-1, -2) @ q6.abs())
    far_dv = (p * (rho + u16 + sums) + low_back).masked_fill(~seen, 0).transpose(-1, -2) @ do.abs()
    gk, gv = group(dk), group(dv)
    return results + [back(dq), gk, gv], bounds + [back(far_dq), group(far_dk) + u * gk.abs() + last, group(far_dv) + u * gv.abs() + last]


def norm(x, weight, freqs, angle, eps, dy=None):
    """(results, bounds): [y] or [y, dx, dw].  `angle` [B or 1, N, 1, rot / 2] in float64.  Per element, with n = d + 16 float32 operations
    behind a value: n f of the absolute terms of the rotation, a turn of 2^-24 pi, and u of the result or half the smallest number of its type."""
    u = torch.finfo(x.dtype).eps / 2
    last = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps / 2
    uw = torch.finfo(weight.dtype).eps / 2 if weight is not None else 0.0
    last_w = torch.finfo(weight.dtype).smallest_normal * torch.finfo(weight.dtype).eps / 2 if weight is not None else 0.0
    d = x.size(-1)
    rot = 0 if angle is None else 2 * angle.size(-1)
    x6 = x.double()
    r = (x6.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = x6 * r
    w = torch.ones(d, dtype=torch.float64, device=x.device) if weight is None else weight.double()

    def turn(t, sign, absolute=False):
        if not rot:
            return t.abs() if absolute else t
        a, b, rest = t[..., : rot // 2], t[..., rot // 2: rot], t[..., rot:]
        c, s = torch.cos(angle), sign * torch.sin(angle)
        if absolute:
            return torch.cat((a.abs() + b.abs(), a.abs() + b.abs(), rest.abs()), -1)
        return torch.cat((a * c - b * s, b * c + a * s, rest), -1)

    near = (d + 16) * F
    y = turn(unit * w, 1)
    results, bounds = [y], [near * turn(unit * w, 1, True) + u * y.abs() + last]
    if dy is None:
        return results, bounds
    g = turn(dy.double(), -1)
    far_g = near * turn(dy.double(), -1, True)
    e = g * w
    mean = (e * unit).mean(-1, keepdim=True)
    dx = r * (e - unit * mean)
    far_mean = ((far_g * w.abs() + near * e.abs()) * unit.abs()).mean(-1, keepdim=True)
    far_dx = r * (far_g * w.abs() + near * (e.abs() + (unit * mean).abs()) + unit.abs() * far_mean) + u * dx.abs() + last
    rows = x.numel() // d
    dw = (g * unit).sum((0, 1, 2))
    far_dw = (far_g * unit.abs() + (near + rows * F) * (g * unit).abs()).sum((0, 1, 2)) + uw * dw.abs() + last_w
    return results + [dx, dw], bounds + [far_dx, far_dw]


def assert_within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool((got.isnan() == want.isnan()).all()), f"{what}: NaN in other places"
    assert bool((got.isinf() == want.isinf()).all()), f"{what}: infinities in other places"
    off = (got - want).abs()
    bad = (off > bound) & ~want.isnan() & ~(got == want)
    if bool(bad.any()):
        i = int((off / bound.clamp_min(1e-300)).nan_to_num(0).masked_fill(~bad, 0).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got {got.flatten()[i].item()}, "
                             f"want {want.flatten()[i].item()}, bound {bound.flatten()[i].item()}")
