"""The operators of an int8 key/value cache, as cases that can be timed and compared: the quantising write of a
chunk's keys and values with the read back, the attention of one decode token per sequence over such a cache, the
causal attention of a prompt chunk over it, and both attentions behind a prefix that the whole batch shares.

The cache.  A (token, kv head) row of D elements is held as int8 codes and one fp32 scale: m = max|x|,
scale = m / 127, code = round_half_even(x * (127 / m)), every operation rounded to fp32; rows with m < 2^-100 have
scale 0 and codes 0.  Keys take the rotary embedding first, in fp32 (rotate half).  Four tensors, a multiple of 64 keys
long: k int8 [batch, kv_heads, cap, D], k_scale fp32 [batch, kv_heads, cap], v int8 [batch, kv_heads, cap / 64, D, 64]
(blocks of 64 keys, transposed), v_scale fp32 [batch, kv_heads, cap].

The attention.  softmax(rope(q) . k~ * D^-1/2) v~ over the values k~, v~ = code * scale that the cache holds, the new
tokens' own among them; token i of a chunk that starts at s sees keys 0 .. s + i, and all keys of the prefix, whose
length is added to the positions that the rotary embedding takes.

``own`` chooses the package's operators; else ``run`` computes the same with elementary torch operations.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4}


def listed():
    return [
        # the write of one decode step of a small model (SmolLM2-135M heads): latency
        {"name": "write_step_4", "kind": "write", "batch": 4, "tokens": 1, "start": 300, "ragged": True, "cap": 512,
         "kv_heads": 3, "heads": 9, "dim": 64, "dtype": "bf16", "prefix": 0},
        # a batch of whole prompts written behind their projections (Llama-3-8B heads)
        {"name": "write_prompt_8x2048", "kind": "write", "batch": 8, "tokens": 2048, "start": 0, "ragged": False,
         "cap": 2304, "kv_heads": 8, "heads": 32, "dim": 128, "dtype": "bf16", "prefix": 0},
        # chunks of sequences of different lengths, each continued where it stands, in a 32-bit model
        {"name": "write_ragged_333", "kind": "write", "batch": 5, "tokens": 333, "start": 700, "ragged": True,
         "cap": 1088, "kv_heads": 5, "heads": 20, "dim": 128, "dtype": "fp32", "prefix": 0},
        # one sequence's decode step of a small 32-bit model: latency
        {"name": "decode_1_300", "kind": "decode", "batch": 1, "tokens": 1, "start": 300, "ragged": True, "cap": 512,
         "kv_heads": 3, "heads": 9, "dim": 64, "dtype": "fp32", "prefix": 0},
        # a serving batch of sequences of 1000 to 4096 tokens
        {"name": "decode_8_4096", "kind": "decode", "batch": 8, "tokens": 1, "start": 4096, "ragged": True, "cap": 4160,
         "kv_heads": 8, "heads": 32, "dim": 128, "dtype": "bf16", "prefix": 0},
        # a larger batch of long documents: gigabytes of cache in a step
        {"name": "decode_16_32768", "kind": "decode", "batch": 16, "tokens": 1, "start": 32768, "ragged": True,
         "cap": 32768 + 64, "kv_heads": 8, "heads": 32, "dim": 128, "dtype": "bf16", "prefix": 0},
        # one very long sequence on few kv heads (BitNet-2B heads)
        {"name": "decode_1_131071", "kind": "decode", "batch": 1, "tokens": 1, "start": 131071, "ragged": True,
         "cap": 131072, "kv_heads": 5, "heads": 20, "dim": 128, "dtype": "bf16", "prefix": 0},
        # a few requests behind a short shared instruction
        {"name": "decode_prefix_4_777", "kind": "decode", "batch": 4, "tokens": 1, "start": 40, "ragged": True,
         "cap": 128, "kv_heads": 3, "heads": 9, "dim": 64, "dtype": "bf16", "prefix": 777},
        # many requests behind a long shared document
        {"name": "decode_prefix_64_8192", "kind": "decode", "batch": 64, "tokens": 1, "start": 500, "ragged": True,
         "cap": 512, "kv_heads": 8, "heads": 32, "dim": 128, "dtype": "bf16", "prefix": 8192},
        # a whole prompt
        {"name": "prompt_1_4096", "kind": "prompt", "batch": 1, "tokens": 4096, "start": 0, "ragged": False,
         "cap": 4096, "kv_heads": 8, "heads": 32, "dim": 128, "dtype": "bf16", "prefix": 0},
        # chunks of different lengths behind older context, small 32-bit model
        {"name": "prompt_ragged_509", "kind": "prompt", "batch": 3, "tokens": 509, "start": 1500, "ragged": True,
         "cap": 2048, "kv_heads": 3, "heads": 9, "dim": 64, "dtype": "fp32", "prefix": 0},
        # short questions behind a shared document: few rows, a long axis
        {"name": "prompt_prefix_8x48", "kind": "prompt", "batch": 8, "tokens": 48, "start": 0, "ragged": False,
         "cap": 128, "kv_heads": 5, "heads": 20, "dim": 128, "dtype": "bf16", "prefix": 4000},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "prompt", "prompt"])
    while True:
        kv = rng.choice([1, 2, 3, 5, 8])
        c = {"kind": kind, "batch": _log(rng, 1, 64 if kind == "decode" else 16), "kv_heads": kv,
             "heads": kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "dim": rng.choice([64, 128, 128]),
             "dtype": rng.choice(["bf16", "bf16", "fp32"]), "prefix": 0, "ragged": rng.random() < 0.5}
        if kind == "decode":
            c.update(tokens=1, start=_log(rng, 1, 131000), ragged=True)
        else:
            c.update(tokens=_log(rng, 1, 4096), start=rng.choice([0, 0, _log(rng, 1, 4096)]))
        if kind != "write" and rng.random() < 0.4:
            c["prefix"] = _log(rng, 1, 16384)
        c["cap"] = (c["start"] + c["tokens"] + 63) // 64 * 64
        rows = c["batch"] * c["tokens"]
        span = c["start"] + c["tokens"]
        cells = c["batch"] * kv * c["dim"] * c["cap"]
        if kind == "write" and rows * kv * c["dim"] <= 8 * 2048 * 8 * 128 and cells <= 64 << 20:
            return c
        if kind == "decode" and cells <= 16 * 8 * 128 * 16384 \
                and rows * c["heads"] * (span + c["prefix"]) <= 32 << 20:
            return c
        if kind == "prompt" and cells <= 64 << 20 and rows * c["heads"] * (span + c["prefix"]) <= 32 * 4096 * 2048:
            return c


def _spread(c):
    """(first position, number of tokens) of every sequence, as lists: a ragged batch spreads its first positions over
    the upper three quarters of ``start`` and its lengths over the upper half of ``tokens``."""
    b, t = c["batch"], c["tokens"]
    if not c["ragged"]:
        return [c["start"]] * b, [t] * b
    return [c["start"] - 3 * c["start"] * i // (4 * b) for i in range(b)], [t - t * i // (2 * b) for i in range(b)]


def work(case):
    c, e = case, _SIZE[case["dtype"]]
    start, lens = _spread(c)
    n, hkv, hq, d = sum(lens), c["kv_heads"], c["heads"], c["dim"]
    new = 2 * hkv * n * (d * e + d + 4)  # keys and values in, codes and scales out
    back = 2 * hkv * n * (d + 4 + 2 * d)  # the written rows read back as bf16
    if c["kind"] == "write":
        return {"bytes": new + back, "flops": 2 * hkv * n * d * 8}
    seen = sum(s + l for s, l in zip(start, lens)) + c["prefix"]
    pairs = sum(l * (c["prefix"] + s) + l * (l + 1) // 2 for s, l in zip(start, lens))
    return {"bytes": new + back + 2 * hkv * seen * (d + 4) + 2 * n * hq * d * e, "flops": 4 * hq * d * pairs}


# ---- inputs ----------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _cache(g, b, hkv, cap, d):
    """A cache in use: codes as rows of normal values have them, scales that differ from token to token."""
    def codes(*shape):
        x = torch.empty(shape, dtype=torch.int8, device=DEV)
        for i in range(shape[0]):
            x[i] = (torch.randn(shape[1:], generator=g, device=DEV) * 40.0).round_().clamp_(-127, 127).to(torch.int8)
        return x

    def scales():
        return 0.024 * torch.exp(0.3 * torch.randn((b, hkv, cap), generator=g, device=DEV))

    return codes(b, hkv, cap, d), scales(), codes(b, hkv, cap // 64, d, 64), scales()


def prepare(case, seed):
    c, g = case, _gen(seed)
    b, t, hq, hkv, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    dt = _DT[c["dtype"]]
    start, lens = _spread(c)
    # q|k|v as one projection gives them, a few channels larger than the others
    width = (hq + 2 * hkv) * d
    chan = torch.where(torch.rand(width, generator=g, device=DEV) < 0.03, 4.0, 1.0)
    qkv = (torch.randn((b * t, width), generator=g, device=DEV) * chan).to(dt)
    q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=1)
    table = c["prefix"] + c["cap"]
    ang = torch.arange(table, dtype=torch.float64, device=DEV)[:, None] * 500000.0 ** (
        -torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)[None, :]
    # which (sequence, token) there is, and at which position: what a scheduler knows of its batch
    seq = torch.tensor([i for i in range(b) for _ in range(lens[i])], device=DEV)
    tok = torch.tensor([j for i in range(b) for j in range(lens[i])], device=DEV)
    first = torch.tensor(start, device=DEV)
    return {"c": c, "q": q, "k": k, "v": v, "cos": ang.cos().float(), "sin": ang.sin().float(),
            "cache": _cache(g, b, hkv, c["cap"], d), "prefix": _cache(g, 1, hkv, (c["prefix"] + 63) // 64 * 64, d),
            "seq": seq, "tok": tok, "at": first[seq] + tok, "first": first,
            "lengths": torch.tensor(lens, device=DEV), "longest": max(s + n for s, n in zip(start, lens))}


# ---- one pass --------------------------------------------------------------------------------------


def _own(s):
    from __graft_entry__ import load_package

    pkg, c = load_package(), s["c"]
    start, lengths = (s["first"], s["lengths"]) if c["ragged"] else (c["start"], None)
    if c["kind"] == "write":
        pkg.kv_cache_write_i8(s["k"], s["v"], s["cache"], start, c["tokens"], s["cos"], s["sin"], lengths=lengths)
        return list(pkg.kv_cache_read_i8(s["cache"], start, c["tokens"]))
    more = {"prefix": s["prefix"], "prefix_len": c["prefix"]} if c["prefix"] else {}
    if c["kind"] == "decode":
        out = pkg.gqa_decode_attention_i8(s["q"], s["k"], s["v"], s["cache"], s["first"], s["cos"], s["sin"], **more)
    else:
        out = pkg.gqa_prefill_attention_i8(s["q"], s["k"], s["v"], s["cache"], start, c["tokens"], s["cos"], s["sin"],
                                           lengths=lengths, **more)
    return [out, *pkg.kv_cache_read_i8(s["cache"], start if c["kind"] == "prompt" else s["first"], c["tokens"])]


def _rotate(x, cos, sin):
    """x [..., heads, D] in fp32 at the positions of cos and sin [..., D / 2]."""
    a, b = x.chunk(2, dim=-1)
    cos, sin = cos.unsqueeze(-2), sin.unsqueeze(-2)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _quantise(x):
    """(codes, scale) of the rows x [..., D] in fp32."""
    m = x.abs().amax(-1, keepdim=True)
    some = m >= 2.0 ** -100
    inv = torch.full_like(m, 127.0) / torch.where(some, m, 1.0)
    codes = torch.round(x * inv).clamp(-127, 127)
    return torch.where(some, codes, 0.0).to(torch.int8), torch.where(some, m / 127.0, 0.0).squeeze(-1)


def _held(cache, n):
    """The first n keys and values [batch, kv_heads, n, D] that a cache stands for, in fp32."""
    k, ks, v, vs = cache
    nb = (n + 63) // 64
    kf = k[:, :, :n].float() * ks[:, :, :n, None]
    vf = v[:, :, :nb].transpose(3, 4).float().reshape(*v.shape[:2], nb * 64, v.shape[3])[:, :, :n]
    return kf, vf * vs[:, :, :n, None]


def _write(s):
    c = s["c"]
    rows = s["seq"] * c["tokens"] + s["tok"]
    k, v = (x[rows].reshape(-1, c["kv_heads"], c["dim"]).float() for x in (s["k"], s["v"]))
    turn = s["at"] + c["prefix"]
    kq, ksc = _quantise(_rotate(k, s["cos"][turn], s["sin"][turn]))
    vq, vsc = _quantise(v)
    kc, ks, vc, vs = s["cache"]
    kc[s["seq"], :, s["at"]] = kq
    ks[s["seq"], :, s["at"]] = ksc
    vc[s["seq"], :, s["at"] // 64, :, s["at"] % 64] = vq
    vs[s["seq"], :, s["at"]] = vsc


def _read(s):
    """The slots of the chunk, read back as bf16 [batch, kv_heads, tokens, D]."""
    c = s["c"]
    at = s["first"][:, None] + torch.arange(c["tokens"], device=DEV)  # [batch, tokens]
    i = torch.arange(c["batch"], device=DEV)[:, None]
    kc, ks, vc, vs = s["cache"]
    k = kc[i, :, at].float() * ks[i, :, at].unsqueeze(-1)
    v = vc[i, :, at // 64, :, at % 64].float() * vs[i, :, at].unsqueeze(-1)
    return [x.transpose(1, 2).to(torch.bfloat16) for x in (k, v)]


def _attend(s):
    c = s["c"]
    b, t, hq, hkv, d, p = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    n, r = s["longest"], hq // hkv
    at = s["first"][:, None] + torch.arange(t, device=DEV)  # [batch, tokens]
    turn = (at + p).clamp(max=s["cos"].shape[0] - 1)
    q = _rotate(s["q"].reshape(b, t, hq, d).float(), s["cos"][turn], s["sin"][turn])
    q = q.reshape(b, t, hkv, r, d).permute(0, 2, 3, 1, 4)  # [b, kv, r, t, d]
    k, v = _held(s["cache"], n)
    sc = torch.matmul(q.reshape(b, hkv, r * t, d), k.transpose(2, 3)) * d ** -0.5
    hidden = torch.arange(n, device=DEV) > at[..., None]  # [b, t, n]
    sc = sc.reshape(b, hkv, r, t, n).masked_fill_(hidden[:, None, None], float("-inf"))
    if p:
        pk, pv = (x[0] for x in _held(s["prefix"], p))  # [kv, p, d]
        qp = q.permute(1, 0, 2, 3, 4).reshape(hkv, b * r * t, d)
        sp = torch.matmul(qp, pk.transpose(1, 2)) * d ** -0.5
        sp = sp.reshape(hkv, b, r, t, p).transpose(0, 1)
        m = torch.maximum(sc.amax(-1, keepdim=True), sp.amax(-1, keepdim=True))
        sp = torch.exp(sp - m)
    else:
        m = sc.amax(-1, keepdim=True)
    sc = sc.sub_(m).exp_()
    total = sc.sum(-1, keepdim=True)
    out = torch.matmul(sc.reshape(b, hkv, r * t, n), v).reshape(b, hkv, r, t, d)
    if p:
        total = total + sp.sum(-1, keepdim=True)
        op = torch.matmul(sp.transpose(0, 1).reshape(hkv, b * r * t, p), pv).reshape(hkv, b, r, t, d)
        out = out + op.transpose(0, 1)
    out = out / total
    out = torch.where((torch.arange(t, device=DEV) < s["lengths"][:, None])[:, None, None, :, None], out, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(b * t, hq * d).to(s["q"].dtype)


def run(state):
    if own:
        return _own(state)
    _write(state)
    back = _read(state)
    return back if state["c"]["kind"] == "write" else [_attend(state), *back]


# ---- the definition in 64 bits ----------------------------------------------------------------------


def _f32(x):
    """A 64-bit value rounded to fp32, the precision in which the cache's quantiser is defined."""
    return x.float().double()


def _exact_row(x):
    """The values [n, D] that quantised rows x stand for, the quantiser's own steps each rounded to fp32."""
    top = x.abs().max(dim=1, keepdim=True).values
    tiny = top < 2.0 ** -100
    top = top.masked_fill(tiny, 1.0)
    codes = _f32(x * _f32(127.0 / top)).round().clamp(-127.0, 127.0)
    return (codes * _f32(top / 127.0)).masked_fill(tiny, 0.0)


def _exact_rope(x, cos, sin, step):
    """Rotary embedding of x [n, D] with cos / sin [n, D / 2], every operation followed by ``step``."""
    h = x.shape[1] // 2
    x1, x2 = x[:, :h].double(), x[:, h:].double()
    c, z = cos.double(), sin.double()
    return torch.cat([step(step(x1 * c) - step(x2 * z)), step(step(x2 * c) + step(x1 * z))], dim=1)


def _exact_cache(cache, i, h, n):
    """(keys, values) [n, D] of sequence i and kv head h in 64 bits."""
    k, ks, v, vs = cache
    kd = k[i, h, :n].double() * ks[i, h, :n, None].double()
    vd = torch.cat(list(v[i, h].unbind(0)), dim=1).t()[:n].double() * vs[i, h, :n, None].double()
    return kd, vd


def exact(case, seed):
    c, s = case, prepare(case, seed)
    b, t, hq, hkv, d, p = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    start, lens = _spread(c)
    r = hq // hkv
    k_back = torch.empty((b, hkv, t, d), dtype=torch.float64, device=DEV)
    v_back = torch.empty_like(k_back)
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device=DEV)
    for i in range(b):
        s0, n, end = start[i], lens[i], start[i] + lens[i]
        cos, sin = (x[p + s0:p + end] for x in (s["cos"], s["sin"]))
        for h in range(hkv):
            keys, values = _exact_cache(s["cache"], i, h, s0 + t)
            rows = slice(i * t, i * t + n)
            keys[s0:end] = _exact_row(_exact_rope(s["k"][rows, h * d:(h + 1) * d], cos, sin, _f32))
            values[s0:end] = _exact_row(s["v"][rows, h * d:(h + 1) * d].double())
            k_back[i, h], v_back[i, h] = keys[s0:], values[s0:]
            if c["kind"] == "write":
                continue
            keys, values = keys[:end], values[:end]
            if p:
                pk, pv = _exact_cache(s["prefix"], 0, h, p)
                keys, values = torch.cat([pk, keys]), torch.cat([pv, values])
            later = torch.arange(p + end, device=DEV)[None, :] - p > s0 + torch.arange(n, device=DEV)[:, None]
            for j in range(h * r, (h + 1) * r):
                q = _exact_rope(s["q"][rows, j * d:(j + 1) * d], cos, sin, lambda x: x)
                prob = torch.softmax((q @ keys.t() / math.sqrt(d)).masked_fill(later, -math.inf), dim=1)
                out[i, :n, j] = prob @ values
    back = [k_back, v_back]
    return back if c["kind"] == "write" else [out.reshape(b * t, hq * d), *back]
