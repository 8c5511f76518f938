"""Timing cases of the dense attention and of the norm-and-rotation of its queries and keys.

`global_attention`: softmax attention of every query over every key that its masks leave, next to the windowed operator:
scores capped by a tanh, a bias that falls with the distance of the two tokens (in a sequence or on a token map), causal,
prefix, document and length masks, shared key heads; forward, training step, and single tokens over a long cache.
`norm_rotary`: RMS norm of every head of q and k and the rotation by the tokens' positions, in one pass; forward, training
step, single tokens.

With `own` false `run` computes both in plain torch operations in 32 bits (angles in 64); with `own` true it calls the package.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


def _attention(name, dtype, B, N, h, hk, d, *, M=None, train=False, mask="none", cap=0.0, slope=0.0, width=1, docs=1):
    return {"op": "attention", "name": name, "dtype": dtype, "B": B, "N": N, "M": M or N, "h": h, "hk": hk, "d": d,
            "train": train, "mask": mask, "cap": cap, "slope": slope, "width": width, "docs": docs}


def _norm(name, dtype, B, N, h, hk, d, *, rot=None, axes=1, width=1, train=False, weighted=True, far=0):
    return {"op": "norm", "name": name, "dtype": dtype, "B": B, "N": N, "h": h, "hk": hk, "d": d, "rot": d if rot is None else rot,
            "axes": axes, "width": width, "train": train, "weighted": weighted, "far": far}


def listed():
    return [
        # one new token for each of eight requests over caches of different fill, shared key heads
        _attention("decode_b8_8192_h32x128_bf16", "bf16", 8, 1, 32, 8, 128, M=8192, mask="lengths"),
        # one new token of one short request: latency
        _attention("decode_b1_317_h8x64_f16", "f16", 1, 1, 8, 8, 64, M=317, mask="causal"),
        # context over a whole coarse token map (1/32 of 1536 x 1536), two views, scores that fall with the distance on the map
        _attention("map_48x48_b2_h4x32_f16", "f16", 2, 48 * 48, 4, 4, 32, slope=0.25, width=48),
        # a long sequence, causal
        _attention("causal_8192_h32x128_bf16", "bf16", 1, 8192, 32, 8, 128, mask="causal"),
        # documents of odd lengths packed into one row, capped scores
        _attention("packed_5003_h16x64_f16", "f16", 1, 5003, 16, 4, 64, mask="documents", cap=30.0, docs=9),
        # a prefix that all tokens see, in float32
        _attention("prefix_1001_h8x32_f32", "f32", 2, 1001, 8, 8, 32, mask="prefix"),
        # training on a sequence, shared key heads, capped scores
        _attention("train_causal_4096_h16x128_bf16", "bf16", 2, 4096, 16, 4, 128, train=True, mask="causal", cap=50.0),
        # training on a token map with the heads of the matching model, distance bias
        _attention("train_map_68x120_h8x16_f16", "f16", 1, 68 * 120, 8, 8, 16, train=True, slope=0.5, width=120),
        # new tokens of sixteen requests: latency
        _norm("norm_token_b16_h32x128_bf16", "bf16", 16, 1, 32, 8, 128, far=100000),
        # the queries and keys of a token map (1/4 of 1536 x 1536), rotated by column and row
        _norm("norm_map_384x384_h8x16_f16", "f16", 1, 384 * 384, 8, 8, 16, axes=2, width=384),
        # training on a sequence
        _norm("norm_train_16384_h32x128_bf16", "bf16", 1, 16384, 32, 8, 128, train=True),
        # training in float32, odd token map, half of a head's channels rotated
        _norm("norm_train_45x79_h8x40_f32", "f32", 2, 45 * 79, 8, 8, 40, rot=16, axes=2, width=79, train=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "train", "decode", "norm", "norm_train"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind in ("norm", "norm_train"):
        d = rng.choice([16, 32, 40, 64, 80, 128])
        hk = rng.choice([1, 2, 4, 8])
        h = hk * rng.choice([1, 2, 4])
        axes = rng.choice([1, 2])
        B = rng.choice([1, 2, 5])
        N = _log_int(rng, 1, max(1, int(16384 * 40 * 128 / (B * (h + hk) * d))) if kind == "norm" else max(1, int(16384 * 40 * 64 / (B * (h + hk) * d))))
        rot = d if rng.random() < 0.6 else d // 8 * 4
        return _norm(None, dtype, B, N, h, hk, d, rot=rot, axes=axes, width=rng.choice([1, 17, 48, 79]),
                     train=kind == "norm_train", weighted=rng.random() < 0.8, far=rng.choice([0, 5000, 200000]))
    d = rng.choice([16, 32, 40, 64, 80, 128])
    hk = rng.choice([1, 2, 4, 8])
    h = hk * rng.choice([1, 2, 4])
    cap = rng.choice([0.0, 0.0, 30.0])
    slope = rng.choice([0.0, 0.0, 0.25])
    width = rng.choice([1, 48, 79])
    if kind == "decode":
        B, N = rng.choice([1, 3, 8]), rng.choice([1, 1, 2, 4])
        return _attention(None, dtype, B, N, h, hk, d, M=_log_int(rng, 16, 16384), mask=rng.choice(["causal", "lengths"]), cap=cap,
                          slope=slope, width=width)
    B = rng.choice([1, 2, 3])
    most = 8192.0 * 8192 * 32 / (8 if dtype == "f32" else 2) / (4 if kind == "train" else 1)
    mask = rng.choice(["none", "causal", "prefix", "documents", "lengths"])
    longer = 1.0 if mask in ("documents", "prefix") or rng.random() < 0.7 else rng.uniform(1, 2)
    N = _log_int(rng, 1, int(min(8192, math.sqrt(most / (B * h * longer)))))
    M = int(N * longer)
    return _attention(None, dtype, B, N, h, hk, d, M=M, train=kind == "train", mask=mask, cap=cap, slope=slope, width=width,
                      docs=rng.randint(1, 12))


# ---- inputs ------------------------------------------------------------------------------------------------

def _tensor(gen, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * spread).to(dtype)


def prepare(case, seed):
    rs = np.random.RandomState((seed * 7919 + 13) % (1 << 31))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) + 1)
    dtype = DTYPES[case["dtype"]]
    B, N, h, hk, d = (case[n] for n in ("B", "N", "h", "hk", "d"))
    ints = lambda a: torch.from_numpy(np.asarray(a, dtype=np.int32)).cuda()  # noqa: E731
    if case["op"] == "norm":
        # what a projection leaves: queries, keys and values of a token side by side
        fused = _tensor(gen, (B, N, (h + 2 * hk) * d), dtype, 1.5)
        state = {"case": case, "q": fused[..., : h * d].view(B, N, h, d), "k": fused[..., h * d: (h + hk) * d].view(B, N, hk, d)}
        for name in ("q_weight", "k_weight"):
            state[name] = (1 + _tensor(gen, (d,), torch.float32, 0.2)).to(dtype) if case["weighted"] else None
        start = int(rs.randint(0, case["far"] + 1))
        if case["axes"] == 2:
            at = np.stack([np.arange(N) % case["width"], np.arange(N) // case["width"]], -1) + start
            state["positions"] = ints(at)
        else:
            state["positions"] = ints(start + np.arange(N)[None] + rs.randint(0, 1000, size=(B, 1)))
        pairs = case["rot"] // 2 // case["axes"]
        turns = 10000.0 ** (-np.arange(pairs, dtype=np.float64) / max(pairs, 1)) / (2 * np.pi)
        turns = np.broadcast_to(turns, (case["axes"], pairs))
        # turns per position in units of 2^-64
        state["freqs"] = torch.from_numpy((np.rint(turns * 2.0 ** 64)).astype(np.uint64).view(np.int64).copy()).cuda()
        if case["train"]:
            state["dq"], state["dk"] = _tensor(gen, (B, N, h, d), dtype), _tensor(gen, (B, N, hk, d), dtype)
            state["wanted"] = [state[n] for n in ("q", "k", "q_weight", "k_weight") if state[n] is not None]
            for t in state["wanted"]:
                t.requires_grad_()
        return state
    M = case["M"]
    state = {"case": case, "q": _tensor(gen, (B, N, h, d), dtype)}
    if M == N:
        kv = _tensor(gen, (B, M, 2, hk, d), dtype)
        state["k"], state["v"] = kv[:, :, 0], kv[:, :, 1]
    else:
        state["k"], state["v"] = _tensor(gen, (B, M, hk, d), dtype), _tensor(gen, (B, M, hk, d), dtype)
    state["scale"] = d ** -0.5
    state["slopes"] = None
    if case["slope"]:
        # from gentle to steep over the heads
        state["slopes"] = (case["slope"] * 2.0 ** (-8.0 * (torch.arange(h, dtype=torch.float32) + 0.5) / h)).cuda()
    state["prefix"] = state["lengths"] = state["documents"] = None
    if case["mask"] == "prefix":
        state["prefix"] = ints(rs.randint(0, M // 2 + 1, size=B))
    if case["mask"] == "lengths":
        state["lengths"] = ints(rs.randint(max(1, M // 4), M + 1, size=B))
    if case["mask"] == "documents":
        cuts = np.sort(rs.randint(0, N + 1, size=(B, max(case["docs"] - 1, 0))), axis=1)
        state["documents"] = ints((np.arange(N)[None, :, None] >= cuts[:, None, :]).sum(-1))
    if case["train"]:
        state["dout"] = _tensor(gen, (B, N, h, d), dtype)
        for n in ("q", "k", "v"):
            state[n] = state[n].requires_grad_()
    return state


# ---- plain forms -------------------------------------------------------------------------------------------

def _angles(state, rot, pairs, axes):
    inv = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / max(pairs, 1))
    at = state["positions"].double()
    at = at.unsqueeze(-1) if axes == 1 else at
    angle = (at.unsqueeze(-1) * inv).flatten(-2).unsqueeze(-2)          # [B or none, N, 1, rot / 2]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(x, cos, sin, rot):
    a, b, rest = x[..., : rot // 2], x[..., rot // 2: rot], x[..., rot:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)


def _norm_one(x, weight, cos, sin, rot):
    x32 = x.detach().float()
    y = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
    if weight is not None:
        y = y * weight.detach().float()
    return _rotate(y, cos, sin, rot).to(x.dtype)


def _norm_back(x, weight, dy, cos, sin, rot):
    x32 = x.detach().float()
    r = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
    unit = x32 * r
    g = _rotate(dy.float(), cos, -sin, rot)
    dw = None
    if weight is not None:
        dw = (g * unit).double().sum((0, 1, 2)).to(weight.dtype)
        g = g * weight.detach().float()
    return (r * (g - unit * (g * unit).mean(-1, keepdim=True))).to(x.dtype), dw


def _visible(state):
    """[B, 1, 1, N, M] (or less), true where a query may look; None: everywhere."""
    case = state["case"]
    M, N = case["M"], case["N"]
    key = torch.arange(M, device="cuda")
    if case["mask"] == "none":
        return None
    if case["mask"] == "documents":
        ids = state["documents"]
        return ((ids[:, :, None] == ids[:, None, :]) & (key <= key[:, None]))[:, None, None]
    if case["mask"] == "lengths":
        n = state["lengths"][:, None, None]
        at = torch.arange(N, device="cuda")[None, :, None] + n - N
        return ((key < n) & (key <= at))[:, None, None]
    causal = key <= torch.arange(N, device="cuda")[:, None] + M - N
    if case["mask"] == "prefix":
        return (causal | (key < state["prefix"][:, None, None]))[:, None, None]
    return causal


def _distance(state):
    case = state["case"]
    M, N, W = case["M"], case["N"], case["width"]
    key = torch.arange(M, device="cuda")[None]
    last = state["lengths"][:, None] if state["lengths"] is not None else torch.full((1, 1), M, device="cuda")
    at = torch.arange(N, device="cuda")[None] + last - N
    dx = (at % W)[:, :, None] - (key % W)[:, None, :]
    dy = torch.div(at, W, rounding_mode="floor")[:, :, None] - torch.div(key, W, rounding_mode="floor")[:, None, :]
    return (dx.abs() + dy.abs()).float()[:, None, None]


def _plain_attention(state):
    case = state["case"]
    B, N, M, h, hk, d = (case[n] for n in ("B", "N", "M", "h", "hk", "d"))
    g = h // hk
    q = state["q"].detach().float().view(B, N, hk, g, d).permute(0, 2, 3, 1, 4).reshape(B, hk, g * N, d)
    k = state["k"].detach().float().permute(0, 2, 1, 3)
    v = state["v"].detach().float().permute(0, 2, 1, 3)
    s = torch.matmul(q, k.transpose(-1, -2)).view(B, hk, g, N, M)
    s.mul_(state["scale"])
    if case["cap"]:
        s.div_(case["cap"]).tanh_()
        slant = 1 - s * s if case["train"] else None
        s.mul_(case["cap"])
    if state["slopes"] is not None:
        s -= state["slopes"].view(hk, g, 1, 1) * _distance(state)
    visible = _visible(state)
    if visible is not None:
        s.masked_fill_(~visible, float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    p = p.view(B, hk, g * N, M)
    back = lambda t: t.view(B, hk, g, N, d).permute(0, 3, 1, 2, 4).reshape(B, N, h, d).to(state["q"].dtype)  # noqa: E731
    o = torch.matmul(p, v)
    if not case["train"]:
        return back(o)
    do = state["dout"].float().view(B, N, hk, g, d).permute(0, 2, 3, 1, 4).reshape(B, hk, g * N, d)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if case["cap"]:
        ds.mul_(slant.view(B, hk, g * N, M))
    dq = torch.matmul(ds, k).mul_(state["scale"])
    dk = torch.matmul(ds.transpose(-1, -2), q).mul_(state["scale"])
    give = lambda t: t.permute(0, 2, 1, 3).to(state["q"].dtype)  # noqa: E731
    return back(o), back(dq), give(dk), give(dv)


def run(state):
    case = state["case"]
    if case["op"] == "norm":
        if own:
            import matchattention_b200 as ma
            q, k = ma.norm_rotary(state["q"], state["k"], state["freqs"], state["positions"], q_weight=state["q_weight"],
                                  k_weight=state["k_weight"], eps=EPS)
            if not case["train"]:
                return q, k
            return (q.detach(), k.detach(), *torch.autograd.grad((q, k), state["wanted"], (state["dq"], state["dk"])))
        rot = case["rot"]
        cos, sin = _angles(state, rot, rot // 2 // case["axes"], case["axes"])
        q = _norm_one(state["q"], state["q_weight"], cos, sin, rot)
        k = _norm_one(state["k"], state["k_weight"], cos, sin, rot)
        if not case["train"]:
            return q, k
        dq, dqw = _norm_back(state["q"], state["q_weight"], state["dq"], cos, sin, rot)
        dk, dkw = _norm_back(state["k"], state["k_weight"], state["dk"], cos, sin, rot)
        return (q, k, dq, dk) + ((dqw, dkw) if case["weighted"] else ())
    if own:
        import matchattention_b200 as ma
        out = ma.global_attention(state["q"], state["k"], state["v"], scale=state["scale"], cap=case["cap"], slopes=state["slopes"],
                                  width=case["width"], causal=case["mask"] != "none", prefix=state["prefix"],
                                  lengths=state["lengths"], documents=state["documents"])
        if not case["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"]))
    return _plain_attention(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    B, N, h, hk, d = (case[n] for n in ("B", "N", "h", "hk", "d"))
    if case["op"] == "norm":
        rows = B * N * (h + hk)
        # x in, y out; training: dy in and dx out as well
        return {"bytes": rows * d * size * (4 if case["train"] else 2) + 4 * B * N * case["axes"],
                "flops": rows * d * (16 if case["train"] else 6)}
    M = case["M"]
    pairs = B * h * float(N) * M
    if case["mask"] in ("causal", "prefix", "documents", "lengths"):
        pairs = B * h * (N * (M - N) + N * (N + 1) / 2.0)
    keys = float(M)
    if case["mask"] == "lengths":          # caches between a quarter and full
        pairs, keys = pairs * 0.625, M * 0.625
    if case["mask"] == "documents":        # cut at random places: the expected share of pairs in one document
        pairs *= 2.0 / (case["docs"] + 1)
    query, key = B * N * h * d * size, B * keys * hk * d * size
    # forward: q, k, v in, out out; training: also dout in and three gradients out
    return {"bytes": int((2 * query + 2 * key) if not case["train"] else (4 * query + 4 * key)),
            "flops": int(pairs * d * (4 if not case["train"] else 14))}


# ---- the definition in 64 bits -----------------------------------------------------------------------------

def _exact_norm(case, state):
    rot, axes = case["rot"], case["axes"]
    pairs = rot // 2 // axes
    columns = []
    places = state["positions"].to(torch.float64).reshape(-1, case["N"], axes)
    for a in range(axes):
        for j in range(pairs):
            columns.append(places[..., a] * 10000.0 ** (-j / pairs))
    angle = torch.stack(columns, -1)[:, :, None] if columns else None
    results, wanted, upstream = [], [], []
    for x, w in (("q", "q_weight"), ("k", "k_weight")):
        t = state[x].detach().double().requires_grad_()
        wanted.append(t)
        y = t / torch.sqrt(t.square().sum(-1, keepdim=True) / case["d"] + EPS)
        if state[w] is not None:
            y = y * state[w].detach().double().requires_grad_()
        if angle is not None:
            first, second = y[..., : rot // 2], y[..., rot // 2: rot]
            turned = torch.view_as_real(torch.complex(first, second) * torch.polar(torch.ones_like(angle), angle))
            y = torch.cat((turned[..., 0], turned[..., 1], y[..., rot:]), -1)
        results.append(y)
    if not case["train"]:
        return tuple(r.detach() for r in results)
    # the weights' gradients by their own definition: the upstream gradient turned back, times the unit rows
    grads = torch.autograd.grad(results, wanted, (state["dq"].double(), state["dk"].double()))
    weights = []
    if case["weighted"]:
        for t, x in zip(wanted, ("dq", "dk")):
            u = t.detach() / torch.sqrt(t.detach().square().sum(-1, keepdim=True) / case["d"] + EPS)
            d = state[x].double()
            if angle is not None:
                back = torch.view_as_real(torch.complex(d[..., : rot // 2], d[..., rot // 2: rot]) * torch.polar(torch.ones_like(angle), -angle))
                d = torch.cat((back[..., 0], back[..., 1], d[..., rot:]), -1)
            weights.append(torch.einsum("bnhd,bnhd->d", d, u))
    return tuple(r.detach() for r in results) + tuple(grads) + tuple(weights)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, state)
    B, N, M, h, hk, d = (case[n] for n in ("B", "N", "M", "h", "hk", "d"))
    q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if case["train"] else None
    keys = torch.arange(M, device="cuda")
    for b in range(B):
        length = int(state["lengths"][b]) if state["lengths"] is not None else M
        places = torch.arange(length - N, length, device="cuda")
        allowed = torch.ones(N, M, dtype=torch.bool, device="cuda")
        if case["mask"] != "none":
            allowed = keys[None] <= places[:, None]
        if state["prefix"] is not None:
            allowed = allowed | (keys < int(state["prefix"][b]))[None]
        if state["documents"] is not None:
            allowed = allowed & torch.eq(state["documents"][b][:, None], state["documents"][b][None])
        allowed = allowed & (keys < length)[None]
        row = lambda t: torch.div(t, case["width"], rounding_mode="floor")  # noqa: E731
        far = (places - row(places) * case["width"])[:, None] - (keys - row(keys) * case["width"])[None]
        far = (far.abs() + (row(places)[:, None] - row(keys)[None]).abs()).double()
        for i in range(h):
            j = i * hk // h
            qi, ki, vi = q[b, :, i], k[b, :, j], v[b, :, j]
            if case["train"]:
                qi, ki, vi = (t.clone().requires_grad_() for t in (qi, ki, vi))
            s = torch.einsum("nd,md->nm", qi, ki) * state["scale"]
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if state["slopes"] is not None:
                s = s - float(state["slopes"][i]) * far
            weight = torch.softmax(s.masked_fill(~allowed, -1e300), -1).masked_fill(~allowed, 0.0)
            o = weight @ vi
            out[b, :, i] = o.detach()
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, (qi, ki, vi), state["dout"][b, :, i].double())
                grads[0][b, :, i] += dq
                grads[1][b, :, j] += dk
                grads[2][b, :, j] += dv
    return (out, *grads) if case["train"] else out
