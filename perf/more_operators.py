"""Operators of a training step over ternary layers, as cases that can be timed and compared: the gated feed-forward
product with its backward pass, the norm of every query and key head with the rotary embedding and its backward pass,
and an AdamW step over many tensors with states in 32 or in 8 bits.  The first two also in their serving form.

The gated product (kind "glu").  h = act(gate) * up, gate = y[:, :F], up = y[:, F:], y = (codes @ t^T) * a * w: codes the
int8 codes of x's rows (m = max|x|, 1 where m < 1e-6; a = m / 127, code = round_half_even(x * (127 / m))), t the ternary
weights of gate over up (w = mean|W| of each matrix, t = clamp(round_half_even(W / w), -1, 1)), every operation of both
quantisers rounded to fp32.  act is silu or relu squared.  The gradient goes straight through both quantisers:
grad_x = d @ (t * w), grad_W = d^T @ (codes * a), d the gradient at y.  Packed weights: uint8 [2 F, Kp / 4], Kp the
columns rounded up to 128, byte j of a block of 128 columns holding t + 1 of columns j, j + 32, j + 64, j + 96 from the
high bits down.

The norm with the rotation (kind "qk").  y = x / sqrt(mean(x^2) + eps) * weight over the D elements of a head (without
weights: y = x), then pair i of its first R elements turned by the angle of cos / sin [position, i]: pairs (i, i + R / 2)
in the half layout, (2 i, 2 i + 1) in the interleaved one.

AdamW (kind "adamw"), step t, every operation rounded to fp32:
    m = m b1 + g (1 - b1),  v = v b2 + (g g)(1 - b2),  r = sqrt(v)
    p = p (1 - lr wd) - (m (lr / (1 - b1^t))) / (r (1 / sqrt(1 - b2^t)) + eps)
The states of all tensors lie in one flat array each, every tensor from a multiple of 256 on.  In 8 bits, a block of 256
holds a = max|m|, s = max r (0 where below 2^-100) and
    m code c = sign(m) min(127, floor(sqrt(|m| (127^2 / a)) + z)),
    r code u = min(255, floor(sqrt(r (255^2 / s)) + z)), 1 at least where r > 0
standing for m = c |c| (a (1 / 127^2)), r = u u (s (1 / 255^2)), v = r r;
z = ((i 0x9E3779B1 + t 0x6A09E667) mod 2^32 >> 8) 2^-24 for element i of the flat array.

``own`` chooses the package's operators; else ``run`` computes the same with elementary torch operations.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4}
_LR, _B1, _B2, _EPS, _WD = 2e-4, 0.9, 0.95, 1e-8, 0.1
_NORM_EPS = 1e-6
_BLOCK = 256


def listed():
    return [
        # one token of a request in a small batch: latency (BitNet-2B widths, weights packed once)
        {"name": "glu_decode_3", "kind": "glu", "train": False, "tokens": 3, "k": 2560, "f": 6912, "act": "relu2",
         "dtype": "bf16", "wdtype": "fp32"},
        # a prompt through the same layer
        {"name": "glu_prompt_2048", "kind": "glu", "train": False, "tokens": 2048, "k": 2560, "f": 6912, "act": "silu",
         "dtype": "bf16", "wdtype": "fp32"},
        # a training step of a small 32-bit model on a ragged batch (SmolLM2-135M widths)
        {"name": "glu_train_509_small", "kind": "glu", "train": True, "tokens": 509, "k": 576, "f": 1536, "act": "silu",
         "dtype": "fp32", "wdtype": "fp32"},
        # a training step in bf16 over fp32 weights, and one over bf16 weights
        {"name": "glu_train_4096", "kind": "glu", "train": True, "tokens": 4096, "k": 2560, "f": 6912, "act": "relu2",
         "dtype": "bf16", "wdtype": "fp32"},
        {"name": "glu_train_2000_bf16", "kind": "glu", "train": True, "tokens": 2000, "k": 4096, "f": 14336,
         "act": "silu", "dtype": "bf16", "wdtype": "bf16"},
        # one token of each of 8 sequences, far into their contexts: latency
        {"name": "qk_decode_8", "kind": "qk", "train": False, "batch": 8, "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "layout": "half", "norm": True, "far": 100000, "dtype": "bf16"},
        # a batch of prompts behind their projections
        {"name": "qk_prompt_8x2048", "kind": "qk", "train": False, "batch": 8, "tokens": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "rotary": 128, "layout": "half", "norm": True, "far": 0, "dtype": "bf16"},
        # a training step: forward and backward, norms and the interleaved pairs
        {"name": "qk_train_4x2048", "kind": "qk", "train": True, "batch": 4, "tokens": 2048, "heads": 20, "kv_heads": 5,
         "dim": 128, "rotary": 128, "layout": "interleaved", "norm": True, "far": 0, "dtype": "bf16"},
        # a small 32-bit model, an odd number of tokens, half of each head turned
        {"name": "qk_train_3x333_part", "kind": "qk", "train": True, "batch": 3, "tokens": 333, "heads": 9,
         "kv_heads": 3, "dim": 64, "rotary": 32, "layout": "half", "norm": True, "far": 0, "dtype": "fp32"},
        # the norms of a small model alone: many tensors of a few hundred elements, latency
        {"name": "adamw_norms_121", "kind": "adamw", "bits": 32, "layers": 30, "hidden": 576, "kv": 192, "inner": 1536,
         "vocab": 0, "matrices": False, "flat": False, "dtype": "fp32", "gdtype": "fp32", "step": 1000},
        # a whole small model (SmolLM2-135M), states in 32 bits
        {"name": "adamw_model_32", "kind": "adamw", "bits": 32, "layers": 30, "hidden": 576, "kv": 192, "inner": 1536,
         "vocab": 49152, "matrices": True, "flat": False, "dtype": "fp32", "gdtype": "fp32", "step": 1000},
        # two layers of a larger one (BitNet-2B) with bf16 gradients, states in 8 bits
        {"name": "adamw_layers_8", "kind": "adamw", "bits": 8, "layers": 2, "hidden": 2560, "kv": 640, "inner": 6912,
         "vocab": 0, "matrices": True, "flat": False, "dtype": "fp32", "gdtype": "bf16", "step": 300},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["glu", "qk", "adamw"])
    while True:
        c = {"kind": kind}
        if kind == "glu":
            c.update(train=rng.random() < 0.7, tokens=_log(rng, 1, 4096), k=_log(rng, 64, 4096), f=_log(rng, 32, 14336),
                     act=rng.choice(["silu", "relu2"]), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                     wdtype=rng.choice(["bf16", "fp32"]))
            if c["tokens"] * c["k"] * c["f"] <= 4096 * 2560 * 6912:
                return c
        elif kind == "qk":
            kv = rng.choice([1, 2, 3, 5, 8])
            dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
            c.update(train=rng.random() < 0.6, batch=_log(rng, 1, 16), tokens=_log(rng, 1, 8192),
                     heads=kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), kv_heads=kv, dim=dim,
                     rotary=rng.choice([dim, dim, dim // 2, dim // 4]), layout=rng.choice(["half", "interleaved"]),
                     norm=rng.random() < 0.7, far=rng.choice([0, 0, _log(rng, 1, 131000)]),
                     dtype=rng.choice(["bf16", "bf16", "fp32"]))
            if c["batch"] * c["tokens"] * (c["heads"] + kv) * dim <= 8 * 2048 * 40 * 128 // (2 if c["train"] else 1):
                return c
        else:
            c.update(bits=rng.choice([32, 8, 8]), layers=_log(rng, 1, 32), hidden=_log(rng, 32, 4096),
                     kv=_log(rng, 8, 1024), inner=_log(rng, 32, 8192), vocab=rng.choice([0, 0, _log(rng, 100, 50000)]),
                     matrices=rng.random() < 0.8, flat=rng.random() < 0.4, dtype=rng.choice(["fp32", "fp32", "bf16"]),
                     gdtype=rng.choice(["fp32", "bf16"]), step=_log(rng, 1, 100000))
            if sum(a * b for a, b in _shapes(c)) <= 134 << 20:
                return c


def _shapes(c):
    """(rows, columns) of a model's tensors, norms with one row."""
    h, kv, inner = c["hidden"], c["kv"], c["inner"]
    norms = [(1, h), (1, h), (1, h), (1, inner)]
    mats = [(h, h), (kv, h), (kv, h), (h, h), (inner, h), (inner, h), (h, inner)] if c["matrices"] else []
    ends = [(1, h)] + ([(c["vocab"], h)] if c["vocab"] else [])
    return (norms + mats) * c["layers"] + ends


def _up(n, to):
    return (n + to - 1) // to * to


def work(case):
    c = case
    if c["kind"] == "glu":
        e, w, m, k, f = _SIZE[c["dtype"]], _SIZE[c["wdtype"]], c["tokens"], c["k"], c["f"]
        product = 2 * m * k * 2 * f
        if not c["train"]:
            return {"bytes": m * (k + f) * e + 2 * f * _up(k, 128) // 4, "flops": product}
        return {"bytes": m * (2 * k + 2 * f) * e + 2 * 2 * f * k * w, "flops": 3 * product}
    if c["kind"] == "qk":
        n = c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["dim"]
        passes = 4 if c["train"] else 2  # in and out, the gradient in and out
        return {"bytes": passes * n * _SIZE[c["dtype"]], "flops": 10 * passes * n}
    n = sum(a * b for a, b in _shapes(c))
    state = 4 * 8 // 2 if c["bits"] == 32 else 4 + 8  # read and written; in 8 bits also the values it stands for
    return {"bytes": n * (2 * _SIZE[c["dtype"]] + _SIZE[c["gdtype"]] + state), "flops": 16 * n}


# ---- inputs ----------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _prepare_glu(c, g):
    m, k, f, dt = c["tokens"], c["k"], c["f"], _DT[c["dtype"]]
    # a normed hidden state: normal, a few channels larger than the others
    chan = torch.where(torch.rand(k, generator=g, device=DEV) < 0.02, 6.0, 1.0)
    s = {"x": (_randn(g, m, k) * chan).to(dt)}
    weights = [(_randn(g, f, k) * 0.02).to(_DT[c["wdtype"]]) for _ in range(2)]
    if c["train"]:
        return {**s, "gate": weights[0], "up": weights[1], "gh": (_randn(g, m, f) * 1e-3).to(dt)}
    # served from packed weights, laid out once
    t, scales = _ternary(*weights)
    return {**s, "t": t, "scales": scales, "packed": _packed(t)}


def _packed(t):
    n, k = t.shape
    codes = torch.ones((n, _up(k, 128)), dtype=torch.uint8, device=DEV)
    codes[:, :k] = (t + 1).to(torch.uint8)
    a, b, c, d = codes.view(n, -1, 4, 32).unbind(2)
    return ((a << 6) | (b << 4) | (c << 2) | d).reshape(n, -1)


def _prepare_qk(c, g):
    b, t, hq, hk, d, dt = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], _DT[c["dtype"]]
    # q|k|v as one projection gives them
    qkv = (_randn(g, b, t, (hq + 2 * hk) * d) * torch.exp(0.5 * _randn(g, b, t, 1))).to(dt)
    q, k, _ = qkv.split([hq * d, hk * d, hk * d], dim=2)
    table, half = c["far"] + t, c["rotary"] // 2
    ang = torch.arange(table, dtype=torch.float64, device=DEV)[:, None] * 500000.0 ** (
        -torch.arange(half, dtype=torch.float64, device=DEV) / half)[None, :]
    # sequences that stand at different places of their contexts
    first = torch.tensor([c["far"] - c["far"] * i // (2 * b) for i in range(b)], device=DEV)
    s = {"q": q.unflatten(2, (hq, d)), "k": k.unflatten(2, (hk, d)), "cos": ang.cos().float(), "sin": ang.sin().float(),
         "positions": first[:, None] + torch.arange(t, device=DEV), "wq": None, "wk": None}
    if c["norm"]:
        s.update(wq=(1.0 + 0.2 * _randn(g, d)).to(dt), wk=(1.0 + 0.2 * _randn(g, d)).to(dt))
    if c["train"]:
        s.update(gq=_randn(g, b, t, hq, d).to(dt), gk=_randn(g, b, t, hk, d).to(dt))
    return s


def _prepare_adamw(c, g):
    shapes = _shapes(c)
    numels = [a * b for a, b in shapes]
    total = sum(_up(n, _BLOCK) for n in numels)
    dt, gdt = _DT[c["dtype"]], _DT[c["gdtype"]]

    def tensors(scale, dtype):
        """(tensors of a model, the buffer that they lie in): each from a multiple of 64 elements on, as an allocator
        lays them, or one behind the other, wherever they end."""
        sizes = [x for n in numels for x in (n, 0 if c["flat"] else _up(n, 64) - n)]
        buf = (_randn(g, sum(sizes)) * scale).to(dtype)
        return [x.view(s) for x, s in zip(buf.split(sizes)[::2], shapes)], buf

    params, buf = tensors(0.02, dt)
    s = {"params": params, "buf": buf, "grads": tensors(1e-3, gdt)[0], "m_scale": None, "v_scale": None}
    # where each tensor ends short of its last block, the rest of the block is zero
    real = torch.cat([x for n in numels for x in (torch.ones(n, dtype=torch.bool, device=DEV),
                                                 torch.zeros(_up(n, _BLOCK) - n, dtype=torch.bool, device=DEV))])
    s["gaps"] = [torch.zeros(_up(n, _BLOCK) - n, device=DEV) for n in numels]
    if c["bits"] == 32:
        # of a training run under way: gradients of a size that differs from element to element
        r = torch.exp(_randn(g, total) * 0.7) * 1e-3
        return {**s, "m": _randn(g, total) * r * 0.3 * real, "v": (r * r) * real}
    m = (_randn(g, total) * 40.0).round_().clamp_(-127, 127) * real
    v = torch.exp(4.8 + 0.3 * _randn(g, total)).round_().clamp_(1, 255) * real
    scale = torch.exp(0.5 * _randn(g, 2, total // _BLOCK))
    return {**s, "m": m.to(torch.int8), "v": v.to(torch.uint8), "m_scale": scale[0] * 1e-3, "v_scale": scale[1] * 4e-3}


def prepare(case, seed):
    make = {"glu": _prepare_glu, "qk": _prepare_qk, "adamw": _prepare_adamw}[case["kind"]]
    return {"c": case, **make(case, _gen(seed))}


# ---- one pass --------------------------------------------------------------------------------------


def _own(s):
    from __graft_entry__ import load_package

    pkg, c = load_package(), s["c"]
    if c["kind"] == "glu":
        if not c["train"]:
            return pkg.gated_bitlinear(s["x"], act=c["act"], packed=pkg.PackedGated(s["packed"], s["scales"]))
        leaves = [s[n].detach().requires_grad_() for n in ("x", "gate", "up")]
        h = pkg.gated_bitlinear(*leaves, act=c["act"])
        return [h.detach(), *torch.autograd.grad(h, leaves, s["gh"])]
    if c["kind"] == "qk":
        q, k, wq, wk = leaves = [s[n] for n in ("q", "k", "wq", "wk")]
        if c["train"]:
            q, k, wq, wk = leaves = [None if x is None else x.detach().requires_grad_() for x in leaves]
        out = pkg.qk_norm_rope(q, k, s["cos"], s["sin"], s["positions"], wq, wk, eps=_NORM_EPS, layout=c["layout"])
        if not c["train"]:
            return list(out)
        grads = torch.autograd.grad(out, [x for x in leaves if x is not None], [s["gq"], s["gk"]])
        return [*(x.detach() for x in out), *grads]
    state = pkg.AdamWState(s["m"], s["v"], s["m_scale"], s["v_scale"])
    pkg.adamw_step(s["params"], s["grads"], state, c["step"], lr=_LR, betas=(_B1, _B2), eps=_EPS, weight_decay=_WD)
    return [s["buf"], *pkg.adamw_state_values(state)]


def _ternary(gate, up):
    """(t [2 F, K], scales [2]) of the weights in fp32."""
    scales = [w.double().abs().mean().float() for w in (gate, up)]
    scales = [torch.where(x < 1e-8, 1.0, x) for x in scales]
    t = [torch.round(w.float() / x).clamp_(-1, 1) for w, x in zip((gate, up), scales)]
    return torch.cat(t), torch.stack(scales)


def _glu(s):
    c = s["c"]
    x, f = s["x"].float(), c["f"]
    t, scales = _ternary(s["gate"], s["up"]) if c["train"] else (s["t"], s["scales"])
    top = x.abs().amax(1, keepdim=True)
    top = torch.where(top < 1e-6, 1.0, top)
    a = top / 127.0
    codes = torch.round(x * (torch.full_like(top, 127.0) / top)).clamp_(-128, 127)
    wide = scales.repeat_interleave(f)
    gate, up = (torch.matmul(codes, t.t()) * wide * a).split(f, dim=1)
    if c["act"] == "silu":
        sig = 1.0 / (1.0 + torch.exp(-gate))
        act = gate * sig
    else:
        act = gate.clamp(min=0.0).square()
    h = (act * up).to(s["x"].dtype)
    if not c["train"]:
        return h
    slope = sig * (1.0 + gate * (1.0 - sig)) if c["act"] == "silu" else 2.0 * gate.clamp(min=0.0)
    gh = s["gh"].float()
    d = torch.cat([gh * up * slope, gh * act], dim=1)
    gx = torch.matmul(d * wide, t)
    gw = torch.matmul(d.t(), codes * a).to(s["gate"].dtype)
    return [h, gx.to(s["x"].dtype), gw[:f], gw[f:]]


def _pairs(x, r, layout):
    """The first and the second elements of the pairs among the first r."""
    return (x[..., :r // 2], x[..., r // 2:r]) if layout == "half" else (x[..., 0:r:2], x[..., 1:r:2])


def _turn(x, cos, sin, r, layout):
    a, b = _pairs(x, r, layout)
    u, v = a * cos - b * sin, b * cos + a * sin
    head = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([head, x[..., r:]], -1)


def _qk_one(s, x, weight, grad):
    """[output] or [output, grad_x, grad_weight or None] of the queries or the keys."""
    c = s["c"]
    cos, sin = (t[s["positions"]].unsqueeze(2) for t in (s["cos"], s["sin"]))
    xf, how = x.float(), (c["rotary"], c["layout"])
    if weight is not None:
        inv = 1.0 / torch.sqrt(xf.square().mean(-1, keepdim=True) + _NORM_EPS)
        n, w = xf * inv, weight.float()
    y = _turn(xf if weight is None else n * w, cos, sin, *how).to(x.dtype)
    if grad is None:
        return [y]
    g = _turn(grad.float(), cos, -sin, *how)  # turned back
    if weight is None:
        return [y, g.to(x.dtype), None]
    gn = g * w
    gx = inv * (gn - n * (gn * n).mean(-1, keepdim=True))
    return [y, gx.to(x.dtype), (g * n).sum((0, 1, 2)).to(weight.dtype)]


def _qk(s):
    q = _qk_one(s, s["q"], s["wq"], s.get("gq"))
    k = _qk_one(s, s["k"], s["wk"], s.get("gk"))
    return [x for pair in zip(q, k) for x in pair if x is not None]


def _dither(total, step):
    """z of every element of a flat state."""
    i = torch.arange(total, dtype=torch.int64, device=DEV)
    return (((i * 0x9E3779B1 + step * 0x6A09E667) & 0xFFFFFFFF) >> 8).float() * 2.0 ** -24


def _values(s):
    """(m, r) of a state in 8 bits, in fp32."""
    c, u = s["m"].float().view(-1, _BLOCK), s["v"].float().view(-1, _BLOCK)
    m = (c * c.abs()) * (s["m_scale"] * (1.0 / 16129.0))[:, None]
    r = (u * u) * (s["v_scale"] * (1.0 / 65025.0))[:, None]
    return m.view(-1), r.view(-1)


def _codes(x, top, z):
    """(codes, scale) of blocks x >= 0 of a state in 8 bits."""
    x = x.view(-1, _BLOCK)
    scale = x.amax(1)
    scale = torch.where(scale < 2.0 ** -100, 0.0, scale)
    k = torch.full_like(scale, float(top * top)) / torch.where(scale == 0.0, 1.0, scale)
    q = torch.floor(torch.sqrt(x * k[:, None]) + z.view(-1, _BLOCK)).clamp_(max=float(top))
    return torch.where(scale[:, None] == 0.0, 0.0, q).view(-1), scale


def _flat(tensors, gaps):
    """The tensors one behind the other in fp32, each with its gap."""
    return torch.cat([x for t, gap in zip(tensors, gaps) for x in (t.reshape(-1).float(), gap)])


def _adamw(s):
    c = s["c"]
    t = c["step"]
    p, g = _flat(s["params"], s["gaps"]), _flat(s["grads"], s["gaps"])
    if c["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m, r = _values(s)
        v = r * r
    m = m * _B1 + g * (1.0 - _B1)
    v = v * _B2 + (g * g) * (1.0 - _B2)
    r = torch.sqrt(v)
    p = p * (1.0 - _LR * _WD) - (m * (_LR / (1.0 - _B1 ** t))) / (r * (1.0 / math.sqrt(1.0 - _B2 ** t)) + _EPS)
    sizes = [n for x, gap in zip(s["params"], s["gaps"]) for n in (x.numel(), gap.numel())]
    torch._foreach_copy_([x.view(-1) for x in s["params"]], list(p.split(sizes)[::2]))
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return [s["buf"], s["m"], s["v"]]
    z = _dither(m.numel(), t)
    code, scale = _codes(m.abs(), 127, z)
    s["m"].copy_(torch.where(m < 0.0, -code, code))
    s["m_scale"].copy_(scale)
    code, scale = _codes(r, 255, z)
    least = ((r.view(-1, _BLOCK) > 0.0) & (scale[:, None] > 0.0)).view(-1)
    s["v"].copy_(torch.where(least, code.clamp(min=1.0), code))
    s["v_scale"].copy_(scale)
    m, r = _values(s)
    return [s["buf"], m, r * r]


def run(state):
    if own:
        return _own(state)
    return {"glu": _glu, "qk": _qk, "adamw": _adamw}[state["c"]["kind"]](state)


# ---- the definition in 64 bits ----------------------------------------------------------------------


def _f32(x):
    """A 64-bit value rounded to fp32, the precision in which the quantisers are defined."""
    return x.float().double()


def _exact_glu(c, s):
    x, f = s["x"].double(), c["f"]
    if c["train"]:
        mats = []
        for w in (s["gate"], s["up"]):
            scale = float(_f32(w.double().abs().mean()))
            mats.append((_f32(w.double() / scale).round().clamp(-1.0, 1.0), scale))
    else:
        mats = [(s["t"][i * f:(i + 1) * f].double(), float(s["scales"][i])) for i in range(2)]
    top = x.abs().max(dim=1, keepdim=True).values
    top[top < 1e-6] = 1.0
    held = _f32(x * _f32(127.0 / top)).round().clamp(-128.0, 127.0) * _f32(top / 127.0)
    gate, up = (held @ t.t() * scale for t, scale in mats)
    if c["act"] == "silu":
        sig = torch.sigmoid(gate)
        act, slope = gate * sig, sig + gate * sig * (1.0 - sig)
    else:
        act, slope = torch.relu(gate) ** 2, 2.0 * torch.relu(gate)
    if not c["train"]:
        return act * up
    gh = s["gh"].double()
    d = [gh * up * slope, gh * act]
    gx = sum(di @ t * scale for di, (t, scale) in zip(d, mats))
    return [act * up, gx, *(di.t() @ held for di in d)]


def _exact_qk(c, s):
    r, grads = c["rotary"], []
    outs = []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        xd = x.double()
        # the rotation as a matrix of each position: columns of its pairs
        i = torch.arange(r // 2, device=DEV)
        a, b = (i, i + r // 2) if c["layout"] == "half" else (2 * i, 2 * i + 1)
        cos, sin = (t.double()[s["positions"]][:, :, None] for t in (s["cos"], s["sin"]))
        rms = 1.0 if w is None else torch.sqrt((xd * xd).sum(-1, keepdim=True) / c["dim"] + _NORM_EPS)
        wd = 1.0 if w is None else w.double()
        n = xd / rms
        y = n * wd
        z = y.clone()
        z[..., a] = y[..., a] * cos - y[..., b] * sin
        z[..., b] = y[..., a] * sin + y[..., b] * cos
        outs.append(z)
        if g is None:
            continue
        gd = g.double()
        gy = gd.clone()
        gy[..., a] = gd[..., a] * cos + gd[..., b] * sin
        gy[..., b] = gd[..., b] * cos - gd[..., a] * sin
        if w is None:
            grads.append((gy, None))
            continue
        inner = (gy * wd * xd).sum(-1, keepdim=True) / c["dim"]
        grads.append((gy * wd / rms - xd * inner / rms ** 3, (gy * n).sum(0).sum(0).sum(0)))
    outs += [g[0] for g in grads] + [g[1] for g in grads if g[1] is not None]
    return outs


def _exact_adamw(c, s):
    t, step = c["step"], _f32 if c["bits"] == 8 else (lambda x: x)
    f = (lambda v: float(torch.tensor(v, dtype=torch.float32))) if c["bits"] == 8 else float
    numels = [p.numel() for p in s["params"]]
    at = [0]
    for n in numels:
        at.append(at[-1] + _up(n, _BLOCK))
    p, g = (torch.zeros(at[-1], dtype=torch.float64, device=DEV) for _ in range(2))
    for o, n, pt, gt in zip(at, numels, s["params"], s["grads"]):
        p[o:o + n], g[o:o + n] = pt.double().flatten(), gt.double().flatten()
    if c["bits"] == 8:
        code, ucode = s["m"].double(), s["v"].double()
        m = step(code * code.abs() * step(s["m_scale"].double() * f(1.0 / 16129.0)).repeat_interleave(_BLOCK))
        root = step(ucode ** 2 * step(s["v_scale"].double() * f(1.0 / 65025.0)).repeat_interleave(_BLOCK))
        v = step(root * root)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = step(step(m * f(_B1)) + step(g * f(1.0 - _B1)))
    v = step(step(v * f(_B2)) + step(step(g * g) * f(1.0 - _B2)))
    root = step(torch.sqrt(v))
    move = m * f(_LR / (1.0 - _B1 ** t)) / (root * f(1.0 / math.sqrt(1.0 - _B2 ** t)) + f(_EPS))
    p = p * f(1.0 - _LR * _WD) - move
    if c["bits"] == 8:
        z = torch.arange(at[-1], dtype=torch.int64, device=DEV) * 0x9E3779B1 + t * 0x6A09E667
        z = (torch.remainder(z, 1 << 32) // 256).double() / (1 << 24)
        held = []
        for x, top, least in ((m.abs(), 127, 0), (root, 255, 1)):
            big = x.view(-1, _BLOCK).max(dim=1).values
            big[big < 2.0 ** -100] = 0.0
            wide = big.repeat_interleave(_BLOCK)
            q = step(torch.sqrt(step(x * step(top * top / wide.masked_fill(wide == 0, 1.0)))))
            q = step(q + z).floor().clamp(max=top)
            if least:
                q = torch.where(x > 0, q.clamp(min=1.0), q)
            q[wide == 0] = 0.0
            held.append(step(q * q * step(big * f(1.0 / (top * top))).repeat_interleave(_BLOCK)))
        m, v = held[0] * torch.sign(m), step(held[1] * held[1])
    buf = s["buf"].double()
    for o, n, pt in zip(at, numels, s["params"]):
        first = pt.storage_offset()
        buf[first:first + n] = p[o:o + n]
    return [buf, m, v]


def exact(case, seed):
    define = {"glu": _exact_glu, "qk": _exact_qk, "adamw": _exact_adamw}[case["kind"]]
    return define(case, prepare(case, seed))
