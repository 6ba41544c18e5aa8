"""The int8 key/value cache on the GPU: the quantising write and the read back bit for bit against fp32 torch on the
CPU, and the decode / prompt attentions that read it (with and without a shared prefix) against float64 over the values
that the cache holds.

Tolerances of the attentions, per output element, are sums of what the arithmetic may lose:
  * the output's rounding, half a step of its type (bf16 2^-8, fp32 2^-24 of the value);
  * the query as a fixed-point row of w bits (bf16 16, fp32 24): an element is off by at most 2^-w of its row's largest,
    a score by the sum of that over the key's elements, the output by the weighted sum of (v - out) times that;
  * the weights p * v_scale as fixed-point numbers of w bits, off by at most 2^(2-w) of the largest weight of the row
    (a row's reference may lie up to four times above it), times 127 codes;
  * fp32 scores, exponentials and sums: 2^-20 of sum p |v| (1 + max |s|) covers ten roundings of 2^-24 and the
    exponent's argument;
  * where bf16 rows take fp16 products (prompts, a long prefix of more than 32 rows) and ``half`` asks for it: a half step of
    fp16, 2^-11, of every element of q, and three of them (scale, value, weight) of sum p |v|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _tables(n, d, theta=10000.0):
    inv = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _rope(x, cos, sin):
    """x [..., heads, d], cos / sin [..., d / 2], in x's precision, every operation rounded."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    c, s = cos.unsqueeze(-2).to(x.dtype), sin.unsqueeze(-2).to(x.dtype)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _quantise(x):
    """(codes int8, scale fp32) of fp32 rows, operation by operation."""
    m = x.abs().amax(-1)
    finite = torch.isfinite(x).all(-1)
    some = finite & (m >= 2.0 ** -100)
    ms = torch.where(some, m, torch.ones_like(m))
    codes = torch.round(x * (torch.full_like(ms, 127.0) / ms)[..., None]).clamp(-127, 127)
    codes = torch.where(some[..., None], codes, torch.zeros_like(codes)).to(torch.int8)
    scale = torch.where(some, ms / 127.0, torch.zeros_like(m))
    return codes, torch.where(finite, scale, torch.full_like(m, float("nan")))


class Host:
    """The cache as plain tensors [batch, kv_heads, cap, d] on the CPU."""

    def __init__(self, b, h, cap, d, gen, empty=False):
        self.k, self.v = (torch.randint(-127, 128, (b, h, cap, d), generator=gen, dtype=torch.int8) for _ in range(2))
        self.ks, self.vs = (0.02 * torch.exp(0.4 * torch.randn((b, h, cap), generator=gen)) for _ in range(2))
        if empty:
            for t in (self.k, self.v, self.ks, self.vs):
                t.zero_()

    def to(self, pkg, dev):
        b, h, cap, d = self.k.shape
        v = self.v.reshape(b, h, cap // 64, 64, d).transpose(3, 4).contiguous()
        return pkg.KVCacheI8(*(t.to(dev) for t in (self.k, self.ks, v, self.vs)))

    def write(self, k_new, v_new, start, lens, t, cos, sin, turn=0):
        b, h, _, d = self.k.shape
        for i in range(b):
            s, n = start[i], lens[i]
            k, v = (x[i * t:i * t + n].reshape(n, h, d).float() for x in (k_new, v_new))
            if cos is not None:
                k = _rope(k, cos[turn + s:turn + s + n], sin[turn + s:turn + s + n])
            for x, codes, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                c, sc = _quantise(x)
                codes[i, :, s:s + n], scale[i, :, s:s + n] = c.transpose(0, 1), sc.transpose(0, 1)

    def held(self, i):
        """(keys, values) of sequence i [kv_heads, cap, d] in float64."""
        return (self.k[i].double() * self.ks[i].double()[..., None],
                self.v[i].double() * self.vs[i].double()[..., None])


def _same_cache(cache, host):
    k, ks, v, vs = (t.cpu() for t in cache)
    b, h, cap, d = k.shape
    v = v.transpose(3, 4).reshape(b, h, cap, d)
    for name, got, want in (("k", k, host.k), ("v", v, host.v), ("k_scale", ks, host.ks), ("v_scale", vs, host.vs)):
        if not torch.equal(torch.nan_to_num(got.float(), nan=-7.0), torch.nan_to_num(want.float(), nan=-7.0)):
            bad = (torch.nan_to_num(got.float(), nan=-7.0) != torch.nan_to_num(want.float(), nan=-7.0)).nonzero()
            raise AssertionError(f"{name} differs at {bad[:4].tolist()} ({len(bad)} places)")


def _attention(q, host, start, lens, t, cos, sin, scale, dtype, prefix=None, npre=0, half=False):
    """(out, bound) float64 [b*t, hq*d]: the definition over the host cache as it is after the write."""
    b, h, _, d = host.k.shape
    hq = q.shape[1] // d
    r, bits = hq // h, 24 if dtype == F32 else 16
    out = torch.zeros((b, t, hq, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(b):
        s, n = start[i], lens[i]
        if n == 0:
            continue
        x = q[i * t:i * t + n].reshape(n, hq, d).double()
        if cos is not None:
            x = _rope(x, cos[npre + s:npre + s + n].double(), sin[npre + s:npre + s + n].double())
        keys, vals = (z[:, :s + n] for z in host.held(i))
        vcode = torch.full((h, s + n), 127.0, dtype=torch.float64) * host.vs[i, :, :s + n].double()
        if npre:
            pk, pv = (z[:, :npre] for z in prefix.held(0))
            keys, vals = torch.cat([pk, keys], 1), torch.cat([pv, vals], 1)
            vcode = torch.cat([127.0 * prefix.vs[0, :, :npre].double(), vcode], 1)
        later = torch.arange(npre + s + n)[None, :] - npre > s + torch.arange(n)[:, None]
        for j in range(hq):
            kk, vv, vc = keys[j // r], vals[j // r], vcode[j // r]
            sc = (x[:, j] @ kk.T * scale).masked_fill(later, -math.inf)
            p = torch.softmax(sc, 1)
            o = p @ vv
            out[i, :n, j] = o
            ds = 2.0 ** -bits * x[:, j].abs().amax(1, keepdim=True) * abs(scale) * kk.abs().sum(1)[None, :]
            lost = 0.0
            if half and dtype == BF16:
                ds = ds + 2.0 ** -11 * (x[:, j].abs() @ kk.abs().T) * abs(scale)
                lost = 3 * 2.0 ** -11 * (p @ vv.abs())
            spread = (p * ds) @ vv.abs() + (p * ds).sum(1, keepdim=True) * o.abs()
            w = (p * vc).amax(1) / 127.0
            # a key's weight is off by a step of the fixed-point grid at most, its code by nothing
            fixed = 2.0 ** (2 - bits) * w[:, None] * (kk.shape[0] * 127.0)
            smax = sc.masked_fill(later, 0.0).abs().amax(1, keepdim=True)
            f32 = 2.0 ** -20 * (1.0 + smax) * (p @ vv.abs())
            tol[i, :n, j] = (2.0 ** -8 if dtype == BF16 else 2.0 ** -23) * o.abs() + spread + fixed + f32 + lost
    return out.reshape(b * t, hq * d), tol.reshape(b * t, hq * d)


def _check(got, ref, tol, what=""):
    got = got.cpu().double()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in the wrong rows"
    off = torch.nan_to_num((got - ref).abs() - tol, nan=0.0)
    assert float(off.max()) <= 0.0, f"{what}: {float(off.max())} beyond the bound, at {int(off.argmax())}"


def _qkv(rows, hq, h, d, dtype, gen, chan=True):
    w = (hq + 2 * h) * d
    x = torch.randn((rows, w), generator=gen)
    if chan:
        x = x * torch.where(torch.rand(w, generator=gen) < 0.05, 5.0, 1.0)
    return x.to(dtype)


# ---- write and read ---------------------------------------------------------------------------------

WRITES = [
    # b, hq, hkv, d, cap, starts, lens, t, dtype, rope
    (1, 1, 1, 64, 64, [0], [1], 1, BF16, True),
    (2, 2, 1, 128, 128, [63, 64], [1, 1], 1, F32, True),
    (3, 3, 3, 64, 192, [0, 61, 100], [70, 9, 0], 70, BF16, True),
    (2, 8, 2, 128, 256, [0, 128], [128, 128], 128, BF16, True),
    (2, 5, 5, 128, 320, [3, 190], [257, 130], 257, F32, True),
    (1, 4, 1, 128, 128, [17], [99], 99, F32, False),
    (4, 2, 2, 64, 128, [5, 0, 127, 64], [3, 128, 1, 64], 128, F32, True),
]


@pytest.mark.parametrize("case", WRITES, ids=[f"b{c[0]}_h{c[2]}_d{c[3]}_t{c[7]}_{str(c[8])[6:]}" for c in WRITES])
@pytest.mark.parametrize("rows", ["slices", "odd"])
def test_write_is_the_fp32_definition_bit_for_bit(pkg, dev, case, rows):
    b, hq, h, d, cap, starts, lens, t, dtype, rope = case
    print(f"[kv write] {case} {rows}", flush=True)
    gen = torch.Generator().manual_seed(b * 1000 + t)
    x = _qkv(b * t, hq, h, d, dtype, gen)
    k, v = x[:, hq * d:(hq + h) * d], x[:, (hq + h) * d:]
    cos, sin = _tables(cap + 7, d) if rope else (None, None)
    host = Host(b, h, cap, d, gen)
    cache = host.to(pkg, dev)
    host.write(k, v, starts, lens, t, cos, sin, turn=7 if rope else 0)
    if rows == "slices":
        xd = x.to(dev)
        kd, vd = xd[:, hq * d:(hq + h) * d], xd[:, (hq + h) * d:]
    else:  # rows that do not start on 16 bytes
        pad = torch.cat([x[:, :1], k, v], dim=1).to(dev)
        kd, vd = pad[:, 1:1 + h * d], pad[:, 1 + h * d:]
    tabs = (cos.to(dev), sin.to(dev)) if rope else (None, None)
    pkg.kv_cache_write_i8(kd, vd, cache, torch.tensor(starts, device=dev), t, *tabs,
                          lengths=torch.tensor(lens, device=dev), rope_offset=7 if rope else 0)
    _same_cache(cache, host)
    if len(set(starts)) == 1 and lens == [t] * b:
        again = Host(b, h, cap, d, gen).to(pkg, dev)
        pkg.kv_cache_write_i8(kd, vd, again, starts[0], t, *tabs, rope_offset=7 if rope else 0)
        s = starts[0]
        assert torch.equal(again.k[:, :, s:s + t], cache.k[:, :, s:s + t])


def test_write_rows_of_zeros_tiny_huge_and_not_finite(pkg, dev):
    d, h, t = 128, 1, 8
    gen = torch.Generator().manual_seed(3)
    k = torch.randn((t, d), generator=gen)
    v = torch.randn((t, d), generator=gen)
    k[0] = 0.0
    k[1] *= 1e-38
    k[2] = 3e38 * torch.sign(k[2])
    k[3, 5] = float("nan")
    k[4, 77] = float("inf")
    v[5, 1] = float("-inf")
    v[6] *= 2.0 ** -101 / v[6].abs().max()
    v[7] *= 2.0 ** -99 / v[7].abs().max()
    host = Host(1, h, 64, d, gen)
    cache = host.to(pkg, dev)
    host.write(k, v, [9], [t], t, None, None)
    pkg.kv_cache_write_i8(k.to(dev), v.to(dev), cache, 9, t)
    _same_cache(cache, host)
    kb, vb = pkg.kv_cache_read_i8(cache, 9, t, torch.float32)
    assert torch.isnan(kb[0, 0, 3]).all() and torch.isnan(kb[0, 0, 4]).all() and torch.isnan(vb[0, 0, 5]).all()
    assert not kb[0, 0, :2].any() and not vb[0, 0, 6].any() and vb[0, 0, 7].any()
    assert torch.isfinite(kb[0, 0, 2]).all()
    # a value is off by half a step of its row at most: m / 254, and the roundings of code * scale
    fine = torch.tensor([0, 2, 5, 6, 7])
    lim = k[fine].abs().amax(1, keepdim=True).double() * (1 / 254 + 2.0 ** -20)
    assert ((kb[0, 0].cpu().double()[fine] - k[fine].double()).abs() <= lim).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_read_gives_code_times_scale(pkg, dev, dtype, d):
    b, h, cap = 3, 2, 192
    gen = torch.Generator().manual_seed(d)
    host = Host(b, h, cap, d, gen)
    cache = host.to(pkg, dev)
    starts, n = [-5, 61, 150], 77  # before the cache, across blocks, past its end
    got = pkg.kv_cache_read_i8(cache, torch.tensor(starts, device=dev), n, dtype)
    for codes, scale, x in ((host.k, host.ks, got[0]), (host.v, host.vs, got[1])):
        assert x.shape == (b, h, n, d) and x.dtype == dtype
        for i in range(b):
            want = torch.zeros((h, n, d))
            lo, hi = max(starts[i], 0), min(starts[i] + n, cap)
            want[:, lo - starts[i]:hi - starts[i]] = codes[i, :, lo:hi].float() * scale[i, :, lo:hi, None]
            assert torch.equal(x[i].cpu(), want.to(dtype))
    one = pkg.kv_cache_read_i8(cache, 64, 1, dtype)
    assert torch.equal(one[0][:, :, 0].cpu(), (host.k[:, :, 64].float() * host.ks[:, :, 64, None]).to(dtype))
    far = pkg.kv_cache_read_i8(cache, torch.tensor([2 ** 62, -2 ** 62, 2 ** 63 - 1], device=dev), 2, dtype)
    assert not far[0].any() and not far[1].any()


# ---- decode ------------------------------------------------------------------------------------------

DECODES = [
    # b, hq, hkv, d, cap, positions, dtype, prefix length
    (1, 1, 1, 64, 64, [0], BF16, 0),
    (2, 9, 3, 64, 128, [0, 127], F32, 0),
    (3, 8, 2, 128, 320, [63, 64, 319], BF16, 0),
    (4, 32, 8, 128, 1088, [1087, 255, 256, 700], BF16, 0),
    (2, 20, 5, 128, 2304, [2100, 1], F32, 0),
    (2, 16, 1, 64, 576, [575, 300], BF16, 0),      # 16 query heads on one kv head
    (1, 7, 1, 128, 4160, [4100], BF16, 0),
    (2, 14, 2, 64, 4096, [4095, 2047], F32, 0),
    (3, 9, 3, 64, 128, [0, 77, 127], BF16, 1),     # prefix of one key
    (4, 8, 2, 128, 192, [0, 5, 64, 191], BF16, 65),
    (2, 20, 5, 128, 64, [3, 63], F32, 500),
    (33, 4, 1, 64, 64, list(range(33)), BF16, 130),
    (5, 32, 8, 128, 256, [200, 0, 13, 64, 255], BF16, 1500),
    (2, 12, 1, 128, 192, [190, 64], F32, 0),
    (20, 8, 2, 128, 128, list(range(60, 80)), BF16, 64),   # several workgroups of rows against the prefix, whole blocks
    (20, 8, 2, 128, 64, list(range(20)), F32, 321),
    (17, 33, 3, 64, 64, list(range(17)), F32, 129),
    (45, 16, 2, 64, 64, [63 - i for i in range(45)], BF16, 1790),  # from here the prefix as fp16 products
    (40, 9, 3, 128, 128, list(range(40)), BF16, 3840),
    (15, 64, 4, 64, 64, list(range(15)), F32, 8800),
    (9, 120, 8, 128, 64, list(range(9)), F32, 7300),
]


def _decode(pkg, dev, case, seed=0, stale=True):
    b, hq, h, d, cap, pos, dtype, npre = case
    gen = torch.Generator().manual_seed(seed + cap + b)
    x = _qkv(b, hq, h, d, dtype, gen)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    cos, sin = _tables(cap + npre, d)
    host = Host(b, h, cap, d, gen)
    pre = Host(1, h, (npre + 63) // 64 * 64, d, gen) if npre else None
    if stale:  # what lies behind a sequence must not be met, whatever it is
        for i in range(b):
            host.ks[i, :, pos[i] + 1:] = float("nan")
            host.vs[i, :, pos[i] + 1:] = float("inf")
        if npre:
            pre.ks[:, :, npre:] = float("inf")
            pre.vs[:, :, npre:] = float("nan")
    cache = host.to(pkg, dev)
    pcache = pre.to(pkg, dev) if npre else None
    host.write(k, v, pos, [1] * b, 1, cos, sin, turn=npre)
    ref, tol = _attention(q, host, pos, [1] * b, 1, cos, sin, d ** -0.5, dtype, pre, npre)
    xd = x.to(dev)
    args = (*xd.split([hq * d, h * d, h * d], dim=1), cache, torch.tensor(pos, device=dev), cos.to(dev), sin.to(dev))
    return args, {"prefix": pcache, "prefix_len": npre} if npre else {}, host, ref, tol


@pytest.mark.parametrize("case", DECODES, ids=[f"b{c[0]}_h{c[1]}x{c[2]}_d{c[3]}_cap{c[4]}_p{c[7]}_{str(c[6])[6:]}"
                                               for c in DECODES])
def test_decode_matches_float64_over_the_held_values(pkg, dev, case):
    print(f"[kv decode] {case}", flush=True)
    args, kw, host, ref, tol = _decode(pkg, dev, case)
    out = pkg.gqa_decode_attention_i8(*args, **kw)
    assert out.dtype == case[6]
    _check(out, ref, tol)
    _same_cache(args[3], host)
    # the same call again: the same bits, and an output given
    mine = torch.empty_like(out)
    assert pkg.gqa_decode_attention_i8(*args, out=mine, **kw) is mine
    assert torch.equal(mine, out)


def test_decode_position_outside_the_cache_or_the_tables(pkg, dev):
    case = (4, 8, 2, 64, 128, [3, 3, 3, 3], BF16, 10)
    args, kw, host, ref, tol = _decode(pkg, dev, case)
    good = [t.clone() for t in args[3]]
    pkg.gqa_decode_attention_i8(*args, **kw)
    for bad in (-1, 128, 2 ** 40, -2 ** 63):
        cache = pkg.KVCacheI8(*(t.clone() for t in good))
        before = [t.clone() for t in cache]
        pos = torch.tensor([3, bad, 3, bad], device=dev)
        out = pkg.gqa_decode_attention_i8(*args[:3], cache, pos, *args[5:], **kw)
        assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
        _check(out[::2], ref[::2], tol[::2])
        for t, u in zip(cache, before):  # sequences 1 and 3 are as they were
            assert torch.equal(torch.nan_to_num(t[1::2].float(), nan=-7.0), torch.nan_to_num(u[1::2].float(), nan=-7.0))
    # tables that end before the position (behind the prefix)
    out = pkg.gqa_decode_attention_i8(*args[:3], pkg.KVCacheI8(*(t.clone() for t in good)), args[4], args[5][:13],
                                      args[6][:13], **kw)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_long_uniform_and_outlier_values(pkg, dev, dtype):
    """Equal weights over very many keys of the largest code (no integer sum may wrap), and one value row far larger than
    the others whose key has next to no weight (it must not cost the others their bits)."""
    d, n = 64, 262144
    cache = pkg.kv_cache_i8(1, 1, n, d, dev)
    cache.k[:] = 0
    cache.k_scale[:] = 1.0
    cache.v[:] = 127
    cache.v_scale[:] = 1.0 / 127
    q = torch.ones((1, d), dtype=dtype, device=dev)
    v = torch.ones((1, d), dtype=dtype, device=dev)
    out = pkg.gqa_decode_attention_i8(q, torch.zeros_like(q), v, cache, torch.tensor([n - 1], device=dev))
    assert float((out.float() - 1.0).abs().max()) <= 2.0 ** -8
    own = pkg.kv_cache_i8(2, 1, 64, d, dev)
    q2 = torch.ones((2, d), dtype=dtype, device=dev)
    out = pkg.gqa_decode_attention_i8(q2, torch.zeros_like(q2), v.expand(2, d).contiguous(), own,
                                      torch.tensor([0, 0], device=dev), prefix=cache, prefix_len=n)
    assert float((out.float() - 1.0).abs().max()) <= 2.0 ** -8
    case = (2, 4, 2, 128, 512, [400, 300], dtype, 0)
    gen = torch.Generator().manual_seed(5)
    b, hq, h, d, cap, pos, _, _ = case
    x = _qkv(b, hq, h, d, dtype, gen, chan=False)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    host = Host(b, h, cap, d, gen)
    qm = q.reshape(b, h, hq // h, d).float().mean(2)
    for j in (7, 130):  # keys that point away from the queries
        host.k[:, :, j], host.ks[:, :, j] = _quantise(-30.0 * qm)
        host.vs[:, :, j] *= 1000.0
    cache = host.to(pkg, dev)
    host.write(k, v, pos, [1] * b, 1, None, None)
    ref, tol = _attention(q, host, pos, [1] * b, 1, None, None, d ** -0.5, dtype)
    xd = x.to(dev)
    out = pkg.gqa_decode_attention_i8(*xd.split([hq * d, h * d, h * d], dim=1), cache, torch.tensor(pos, device=dev))
    _check(out, ref, tol)
    assert float(tol.max()) < 0.2 * float(ref.abs().mean())


def test_decode_scales_of_either_sign_and_zero(pkg, dev):
    case = (2, 8, 2, 64, 320, [300, 17], BF16, 70)
    args, kw, host, _, _ = _decode(pkg, dev, case)
    pre = Host(1, 2, 128, 64, torch.Generator().manual_seed(1))
    kw = {"prefix": pre.to(pkg, dev), "prefix_len": 70}
    q = args[0].cpu()
    for scale in (-0.3, 0.0, 1e-30, 4.0):
        out = pkg.gqa_decode_attention_i8(*args, scale=scale, **kw)
        ref, tol = _attention(q, host, case[5], [1, 1], 1, args[5].cpu(), args[6].cpu(), scale, BF16, pre, 70)
        _check(out, ref, tol, f"scale {scale}")


def test_not_finite_rows_reach_what_attends_to_them_only(pkg, dev):
    """A key or value row with a NaN or an infinity makes NaN of every row that sees it, and of no other."""
    b, hq, h, d, t, cap = 2, 4, 2, 64, 90, 128
    gen = torch.Generator().manual_seed(8)
    x = _qkv(b * t, hq, h, d, BF16, gen)
    x[40, hq * d + 3] = float("nan")            # sequence 0, token 40: key of kv head 0
    x[t + 70, (hq + 2 * h) * d - 1] = float("inf")  # sequence 1, token 70: value of kv head 1
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    host = Host(b, h, cap, d, gen)
    cache = host.to(pkg, dev)
    host.write(k, v, [0] * b, [t] * b, t, None, None)
    out = pkg.gqa_prefill_attention_i8(*x.to(dev).split([hq * d, h * d, h * d], dim=1), cache, 0, t)
    got = torch.isnan(out.cpu()).reshape(b, t, hq, d)
    want = torch.zeros((b, t, hq, d), dtype=torch.bool)
    want[0, 40:, :2] = True
    want[1, 70:, 2:] = True
    assert torch.equal(got, want)
    host.ks.nan_to_num_(nan=1.0)
    host.vs.nan_to_num_(nan=1.0)
    ref, tol = _attention(q, host, [0] * b, [t] * b, t, None, None, d ** -0.5, BF16)
    ref[want.reshape(b * t, -1)] = float("nan")
    _check(out, ref, tol)
    step = _qkv(b, hq, h, d, BF16, gen).to(dev).split([hq * d, h * d, h * d], dim=1)
    out = pkg.gqa_decode_attention_i8(*step, cache, torch.tensor([t, t], device=dev)).reshape(b, hq, d)
    assert torch.equal(torch.isnan(out).all(-1).cpu(), torch.tensor([[True, True, False, False], [False, False, True, True]]))
    assert torch.equal(torch.isnan(out).any(-1), torch.isnan(out).all(-1))


# ---- prompt ------------------------------------------------------------------------------------------

PROMPTS = [
    # b, hq, hkv, d, cap, starts, lens, t, dtype, prefix length
    (1, 1, 1, 64, 64, [0], [1], 1, BF16, 0),
    (2, 8, 2, 128, 128, [0, 0], [128, 128], 128, BF16, 0),
    (2, 9, 3, 64, 320, [11, 200], [75, 20], 75, F32, 0),
    (3, 4, 4, 128, 256, [70, 0, 191], [65, 0, 3], 65, BF16, 0),
    (1, 32, 8, 128, 576, [0], [513], 513, BF16, 0),
    (2, 10, 2, 128, 1088, [1000, 63], [33, 66], 66, F32, 0),
    (2, 16, 1, 64, 256, [5, 100], [37, 9], 37, BF16, 0),
    (2, 5, 1, 64, 192, [0, 1], [130, 129], 130, F32, 0),
    (2, 12, 2, 64, 128, [0, 40], [40, 31], 40, BF16, 129),
    (3, 20, 5, 128, 128, [0, 0, 0], [48, 48, 48], 48, BF16, 700),
    (2, 4, 2, 128, 64, [0, 9], [1, 2], 2, F32, 1000),
    (1, 4, 1, 128, 4160, [4000], [100], 100, BF16, 0),  # few rows, a long axis
    (3, 8, 2, 64, 128, [5, 64, 127], [1, 0, 1], 1, BF16, 0),  # one token a sequence, one of them padding
    (2, 33, 3, 128, 192, [100, 0], [41, 90], 90, F32, 64),
    (2, 8, 2, 64, 128, [0, 28], [90, 100], 300, BF16, 0),  # padded to more than the cache holds
    (1, 16, 4, 64, 1024, [700], [200], 200, F32, 0),       # long enough to be split
    (14, 14, 14, 64, 320, [5 * i for i in range(13)] + [0], [257 - i for i in range(13)] + [257], 257, BF16, 0),  # many rows
    (9, 22, 22, 128, 320, list(range(9)), [300] * 9, 300, BF16, 3),
]


@pytest.mark.parametrize("case", PROMPTS, ids=[f"b{c[0]}_h{c[1]}x{c[2]}_d{c[3]}_s{c[5][-1]}_t{c[7]}_p{c[9]}_{str(c[8])[6:]}"
                                               for c in PROMPTS])
def test_prompt_matches_float64_over_the_held_values(pkg, dev, case):
    b, hq, h, d, cap, starts, lens, t, dtype, npre = case
    print(f"[kv prompt] {case}", flush=True)
    gen = torch.Generator().manual_seed(cap + t)
    x = _qkv(b * t, hq, h, d, dtype, gen)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    cos, sin = _tables(cap + npre, d)
    host = Host(b, h, cap, d, gen)
    pre = Host(1, h, (npre + 63) // 64 * 64, d, gen) if npre else None
    for i in range(b):
        host.ks[i, :, starts[i] + lens[i]:] = float("inf")
        host.vs[i, :, starts[i] + lens[i]:] = float("nan")
    cache = host.to(pkg, dev)
    kw = {"prefix": pre.to(pkg, dev), "prefix_len": npre} if npre else {}
    host.write(k, v, starts, lens, t, cos, sin, turn=npre)
    ref, tol = _attention(q, host, starts, lens, t, cos, sin, d ** -0.5, dtype, pre, npre)
    xd = x.to(dev).split([hq * d, h * d, h * d], dim=1)
    tabs = (cos.to(dev), sin.to(dev))
    out = pkg.gqa_prefill_attention_i8(*xd, cache, torch.tensor(starts, device=dev), t, *tabs,
                                       lengths=torch.tensor(lens, device=dev), **kw)
    _check(out, ref, tol)
    _same_cache(cache, host)
    again = pkg.gqa_prefill_attention_i8(*xd, cache, torch.tensor(starts, device=dev), t, *tabs,
                                         lengths=torch.tensor(lens, device=dev), **kw)
    assert torch.equal(again, out)
    if len(set(starts)) == 1 and lens == [t] * b:  # the same as host values, into a wider output
        wide = torch.full((b * t, hq * d + 8), 3.0, dtype=dtype, device=dev)
        pkg.gqa_prefill_attention_i8(*xd, cache, starts[0], t, *tabs, out=wide[:, :hq * d], **kw)
        _check(wide[:, :hq * d], ref, tol)
        assert (wide[:, hq * d:] == 3.0).all()


def test_prompt_sequences_that_do_not_fit(pkg, dev):
    b, hq, h, d, t, cap = 5, 4, 2, 64, 20, 64
    gen = torch.Generator().manual_seed(2)
    x = _qkv(b * t, hq, h, d, BF16, gen)
    cos, sin = _tables(60, d)
    host = Host(b, h, cap, d, gen)
    cache = host.to(pkg, dev)
    before = [c.clone() for c in cache]
    starts, lens = [40, 41, -1, 0, 0], [20, 20, 5, 21, -1]
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    host.write(k, v, [40, 0, 0, 0, 0], [20, 0, 0, 0, 0], t, cos, sin)
    out = pkg.gqa_prefill_attention_i8(*x.to(dev).split([hq * d, h * d, h * d], dim=1), cache,
                                       torch.tensor(starts, device=dev), t, cos.to(dev), sin.to(dev),
                                       lengths=torch.tensor(lens, device=dev))
    assert torch.isnan(out[t:]).all()
    ref, tol = _attention(q, host, [40, 0, 0, 0, 0], [20, 0, 0, 0, 0], t, cos, sin, d ** -0.5, BF16)
    _check(out[:t], ref[:t], tol[:t])
    _same_cache(cache, host)
    for c, u in zip(cache, before):
        assert torch.equal(c[1:], u[1:])


def test_a_prompt_cut_anywhere_and_decoded_onwards_is_the_same(pkg, dev):
    """A sequence as one chunk, as chunks of 1, 62, 70 and 7 tokens and by single steps: the caches agree bit for bit, the
    outputs within their bound; and the first 100 tokens as a prefix shared by two sequences give the rows behind them."""
    hq, h, d, n, cap = 8, 2, 128, 140, 192
    gen = torch.Generator().manual_seed(31)
    x = _qkv(n, hq, h, d, BF16, gen)
    cos, sin = _tables(cap, d)
    tabs = (cos.to(dev), sin.to(dev))
    host = Host(1, h, cap, d, gen, empty=True)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    host.write(k, v, [0], [n], n, cos, sin)
    ref, tol = _attention(q, host, [0], [n], n, cos, sin, d ** -0.5, BF16)
    xd = x.to(dev)

    def rows(a, z):
        return xd[a:z].split([hq * d, h * d, h * d], dim=1)

    whole = pkg.kv_cache_i8(1, h, n, d, dev)
    assert whole.k.shape[2] == cap
    _check(pkg.gqa_prefill_attention_i8(*rows(0, n), whole, 0, n, *tabs), ref, tol, "one chunk")
    _same_cache(whole, host)
    cut = pkg.kv_cache_i8(1, h, n, d, dev)
    outs, at = [], 0
    for t in (1, 62, 70, 7):
        outs.append(pkg.gqa_prefill_attention_i8(*rows(at, at + t), cut, at, t, *tabs))
        at += t
    _check(torch.cat(outs), ref, tol, "chunks")
    _same_cache(cut, host)
    steps = pkg.kv_cache_i8(1, h, n, d, dev)
    outs = [pkg.gqa_decode_attention_i8(*rows(i, i + 1), steps, torch.tensor([i], device=dev), *tabs) for i in range(n)]
    _check(torch.cat(outs), ref, tol, "steps")
    _same_cache(steps, host)
    own = pkg.kv_cache_i8(2, h, 64, d, dev)
    out = pkg.gqa_prefill_attention_i8(*(torch.cat([z, z]) for z in rows(100, 130)), own, 0, 30, *tabs, prefix=whole,
                                       prefix_len=100)
    for i in range(2):
        _check(out[30 * i:30 * i + 30], ref[100:130], tol[100:130], "behind a prefix")
    out = pkg.gqa_decode_attention_i8(*(torch.cat([z, z]) for z in rows(130, 131)), own,
                                      torch.tensor([30, 30], device=dev), *tabs, prefix=whole, prefix_len=100)
    _check(out, ref[[130, 130]], tol[[130, 130]], "a step behind a prefix")


# ---- extremes ------------------------------------------------------------------------------------------

EXTREMES = [
    # b, hq, hkv, d, t, prefix length (t 0: a decode step)
    (3, 8, 2, 64, 0, 0),
    (3, 8, 2, 128, 0, 70),
    (48, 16, 2, 64, 0, 1790),   # bf16: the prefix as fp16 products
    (2, 9, 3, 64, 33, 0),
    (2, 8, 2, 128, 40, 100),
]


def _call(pkg, dev, case, x, cache, pre, base, **kw):
    b, hq, h, d, t, npre = case
    xs = x.to(dev).split([hq * d, h * d, h * d], dim=1)
    if npre:
        kw.update(prefix=pre.to(pkg, dev), prefix_len=npre)
    if t == 0:
        return pkg.gqa_decode_attention_i8(*xs, cache, torch.full((b,), base, device=dev), **kw)
    return pkg.gqa_prefill_attention_i8(*xs, cache, base, t, **kw)


def _made(case, dtype, seed=5):
    b, hq, h, d, t, npre = case
    gen = torch.Generator().manual_seed(seed)
    host = Host(b, h, 192, d, gen)
    pre = Host(1, h, (npre + 63) // 64 * 64, d, gen) if npre else None
    return _qkv(b * max(t, 1), hq, h, d, dtype, gen), host, pre


def _wanted(case, x, host, pre, base, dtype):
    b, hq, h, d, t, npre = case
    t = max(t, 1)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    host.write(k, v, [base] * b, [t] * b, t, None, None)
    return _attention(q, host, [base] * b, [t] * b, t, None, None, d ** -0.5, dtype, pre, npre, half=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", EXTREMES)
def test_a_query_that_is_not_finite_is_its_own_row_only(pkg, dev, case, dtype):
    b, hq, h, d, t, npre = case
    print(f"[kv extremes] {case} {dtype}", flush=True)
    x, host, pre = _made(case, dtype)
    cache = host.to(pkg, dev)
    ref, tol = _wanted(case, x, host, pre, 100, dtype)
    for row, head, bad in ((0, 1, float("nan")), (x.shape[0] - 1, hq - 1, float("-inf")), (1, 0, float("inf"))):
        x[row, head * d + 5] = bad
        ref[row, head * d:(head + 1) * d] = float("nan")
    _check(_call(pkg, dev, case, x, cache, pre, 100), ref, tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", EXTREMES)
def test_large_keys_under_small_queries_and_large_values(pkg, dev, case, dtype):
    b, hq, h, d, t, npre = case
    print(f"[kv extremes] {case} {dtype}", flush=True)
    x, host, pre = _made(case, dtype)
    up, down = 2.0 ** 90, 2.0 ** -90
    x[:, :hq * d] *= down
    x[:, hq * d:(hq + h) * d] *= up
    x[:, (hq + h) * d:] *= up
    for z in (host, pre) if pre else (host,):
        z.ks *= up
        z.vs *= up
    cache = host.to(pkg, dev)
    ref, tol = _wanted(case, x, host, pre, 100, dtype)
    _check(_call(pkg, dev, case, x, cache, pre, 100), ref, tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", EXTREMES)
def test_a_value_far_above_the_others_under_no_weight(pkg, dev, case, dtype):
    """The values that count are 2^-20 of one whose key's weight is nothing."""
    b, hq, h, d, t, npre = case
    print(f"[kv extremes] {case} {dtype}", flush=True)
    x, host, pre = _made(case, dtype)
    x[:, :hq * d] = 2.0 + x[:, :hq * d].abs() / 8
    for z in (host, pre) if pre else (host,):
        z.vs *= 2.0 ** -20
    x[:, (hq + h) * d:] *= 2.0 ** -20
    first = pre if pre else host
    first.k[:, :, 7] = -127
    first.ks[:, :, 7] = 1.0
    first.vs[:, :, 7] *= 2.0 ** 20
    cache = host.to(pkg, dev)
    ref, tol = _wanted(case, x, host, pre, 100, dtype)
    _check(_call(pkg, dev, case, x, cache, pre, 100), ref, tol)
    assert float(ref.abs().max()) < 2.0 ** -10


@pytest.mark.parametrize("case", EXTREMES)
def test_the_output_may_be_the_queries(pkg, dev, case):
    x, host, pre = _made(case, BF16)
    want = _call(pkg, dev, case, x, host.to(pkg, dev), pre, 64)
    b, hq, h, d, t, npre = case
    q = x[:, :hq * d].to(dev).contiguous()
    k, v = (z.to(dev) for z in x[:, hq * d:].split([h * d, h * d], dim=1))
    kw = {"prefix": pre.to(pkg, dev), "prefix_len": npre} if npre else {}
    if t == 0:
        got = pkg.gqa_decode_attention_i8(q, k, v, host.to(pkg, dev), torch.full((b,), 64, device=dev), out=q, **kw)
    else:
        got = pkg.gqa_prefill_attention_i8(q, k, v, host.to(pkg, dev), 64, t, out=q, **kw)
    assert got is q and torch.equal(q, want)


# ---- where and when the calls run ----------------------------------------------------------------------


def test_side_stream_and_unaligned_inputs(pkg, dev):
    case = (3, 8, 2, 128, 320, [63, 64, 319], BF16, 65)
    args, kw, host, ref, tol = _decode(pkg, dev, case)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        out = pkg.gqa_decode_attention_i8(*args, **kw)
        odd = [torch.cat([z[:, :1], z], dim=1)[:, 1:] for z in args[:3]]
        wide = torch.empty((3, 8 * 128 + 1), dtype=BF16, device=dev)
        res = pkg.gqa_decode_attention_i8(*odd, *args[3:], out=wide[:, 1:], **kw)
        col = pkg.gqa_decode_attention_i8(args[0].t().contiguous().t(), *args[1:], **kw)
    s.synchronize()
    _check(out, ref, tol)
    assert torch.equal(res, out) and torch.equal(wide[:, 1:], out) and torch.equal(col, out)


def test_two_streams_at_once(pkg, dev):
    """Calls in flight on two streams, each with a cache and a workspace of its own, over one prefix."""
    cases = [(48, 16, 2, 64, 0, 1790), (2, 9, 3, 64, 33, 0), (3, 8, 2, 128, 0, 0)]
    made = [_made(c, BF16, seed=i) for i, c in enumerate(cases)]
    want = [_call(pkg, dev, c, x, host.to(pkg, dev), pre, 100) for c, (x, host, pre) in zip(cases, made)]
    caches = [[host.to(pkg, dev) for _, host, _ in made] for _ in range(2)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for c, (x, host, pre), own in zip(cases, made, zip(*caches)):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_call(pkg, dev, c, x, own[i], pre, 100))
    torch.cuda.synchronize()
    for i in range(2):
        for g, w in zip(got[i], want):
            assert torch.equal(g, w)


def test_graphs_replayed_as_positions_advance(pkg, dev):
    """Two captured steps (with and without a prefix) replayed in turn while the positions move on, between eager calls:
    every replay is the eager result."""
    b, hq, h, d, cap, npre = 2, 8, 2, 128, 640, 300
    gen = torch.Generator().manual_seed(77)
    cos, sin = (z.to(dev) for z in _tables(cap + npre, d))
    pre = Host(1, h, 320, d, gen).to(pkg, dev)
    host = Host(b, h, cap, d, gen)
    caches = [host.to(pkg, dev) for _ in range(4)]
    x = _qkv(b, hq, h, d, BF16, gen).to(dev)
    pos = torch.tensor([500, 3], device=dev)
    kws = [{}, {"prefix": pre, "prefix_len": npre}]

    def step(cache, kw):
        return pkg.gqa_decode_attention_i8(*x.split([hq * d, h * d, h * d], dim=1), cache, pos, cos, sin, **kw)

    for c, kw in zip(caches, kws):
        step(c, kw)
    graphs, outs = [], []
    for c, kw in zip(caches, kws):
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            outs.append(step(c, kw))
        torch.cuda.current_stream(dev).wait_stream(s)
        graphs.append(g)
    for n in range(6):
        pos.copy_(torch.tensor([500 + 23 * n, 3 + 60 * n], device=dev))
        x.copy_(_qkv(b, hq, h, d, BF16, gen).to(dev))
        for i in (0, 1) if n % 2 else (1, 0):
            graphs[i].replay()
        want = [step(c, kw) for c, kw in zip(caches[2:], kws)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i]), (n, i)
            for t, u in zip(caches[i], caches[2 + i]):
                assert torch.equal(t, u)


def test_prompt_captured_into_a_graph(pkg, dev):
    b, hq, h, d, cap, t = 2, 8, 2, 64, 2112, 40
    gen = torch.Generator().manual_seed(4)
    cos, sin = (z.to(dev) for z in _tables(cap, d))
    host = Host(b, h, cap, d, gen)
    mine, other = host.to(pkg, dev), host.to(pkg, dev)
    x = _qkv(b * t, hq, h, d, BF16, gen).to(dev)
    start, lens = torch.tensor([2000, 1], device=dev), torch.tensor([t, 3], device=dev)

    def call(cache):
        return pkg.gqa_prefill_attention_i8(*x.split([hq * d, h * d, h * d], dim=1), cache, start, t, cos, sin, lengths=lens)

    call(mine)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        out = call(mine)
    torch.cuda.current_stream(dev).wait_stream(s)
    for n in range(4):
        start.copy_(torch.tensor([2000 - 300 * n, 1 + 500 * n], device=dev))
        lens.copy_(torch.tensor([t - 9 * n, 3 + 11 * n], device=dev))
        g.replay()
        want = call(other)
        torch.cuda.synchronize()
        assert torch.equal(out, want), n


def test_cache_past_32_bit_offsets(pkg, dev):
    """The last sequence of a cache of more than 2^31 bytes a tensor."""
    b, hq, h, d, cap = 17, 8, 8, 128, 131072
    assert b * h * cap * d > 2 ** 31
    cache = pkg.kv_cache_i8(b, h, cap, d, dev)
    gen = torch.Generator().manual_seed(6)
    small = Host(1, h, 192, d, gen)
    part = small.to(pkg, dev)
    cache.k[-1, :, :192], cache.k_scale[-1, :, :192] = part.k[0], part.k_scale[0]
    cache.v[-1, :, :3], cache.v_scale[-1, :, :192] = part.v[0], part.v_scale[0]
    x = _qkv(b, hq, h, d, BF16, gen)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    pos = [cap - 1 if i % 2 else 0 for i in range(b)]
    pos[-1] = 150
    out = pkg.gqa_decode_attention_i8(*x.to(dev).split([hq * d, h * d, h * d], dim=1), cache, torch.tensor(pos, device=dev))
    small.write(k[-1:], v[-1:], [150], [1], 1, None, None)
    ref, tol = _attention(q[-1:], small, [150], [1], 1, None, None, d ** -0.5, BF16)
    _check(out[-1:], ref, tol)
    # a sequence of zeros but for its last key: that key's weight is among cap equal ones or more
    k0, v0 = pkg.kv_cache_read_i8(cache, torch.tensor(pos, device=dev), 1, F32)
    want, sc = _quantise(v[15].reshape(h, d).float())
    assert torch.equal(v0[15, :, 0].cpu(), want.float() * sc[:, None])
    t = 70
    x = _qkv(b * t, hq, h, d, BF16, gen)
    q, k, v = x.split([hq * d, h * d, h * d], dim=1)
    starts = [cap - t] * (b - 1) + [100]
    out = pkg.gqa_prefill_attention_i8(*x.to(dev).split([hq * d, h * d, h * d], dim=1), cache,
                                       torch.tensor(starts, device=dev), t)
    small.write(k[-t:], v[-t:], [100], [t], t, None, None)
    ref, tol = _attention(q[-t:], small, [100], [t], t, None, None, d ** -0.5, BF16)
    _check(out[-t:], ref, tol)


def test_empty_calls(pkg, dev):
    cache = pkg.kv_cache_i8(2, 1, 64, 64, dev)
    z = torch.empty((0, 64), dtype=BF16, device=dev)
    assert pkg.gqa_prefill_attention_i8(z, z, z, cache, 0, 0).shape == (0, 64)
    pkg.kv_cache_write_i8(z, z, cache, 0, 0)
    k, v = pkg.kv_cache_read_i8(cache, 0, 0)
    assert k.shape == v.shape == (2, 1, 0, 64)


def test_refusals(pkg, dev):
    b, hq, h, d = 2, 4, 2, 64
    cache = pkg.kv_cache_i8(b, h, 64, d, dev)
    pre = pkg.kv_cache_i8(1, h, 64, d, dev)
    q = torch.zeros((b, hq * d), dtype=BF16, device=dev)
    k = torch.zeros((b, h * d), dtype=BF16, device=dev)
    pos = torch.zeros(b, dtype=torch.int64, device=dev)
    cos, sin = (z.to(dev) for z in _tables(64, d))
    dec, pro = pkg.gqa_decode_attention_i8, pkg.gqa_prefill_attention_i8

    def no(match, fn, *a, **kw):
        with pytest.raises((RuntimeError, ValueError), match=match):
            fn(*a, **kw)

    no("int64", dec, q, k, k, cache, pos.int())
    no("int64", dec, q, k, k, cache, pos[:1])
    no("int64", dec, q, k, k, cache, 3)
    no("int64", dec, q, k, k, cache, torch.zeros(2 * b, dtype=torch.int64, device=dev)[::2])
    no("int64", dec, q, k, k, cache, pos.cpu())
    no("dtype", dec, q.half(), k.half(), k.half(), cache, pos)
    no("elements", dec, q, k.float(), k, cache, pos)
    no("elements", dec, q, k[:1], k, cache, pos)
    no("elements", dec, q.cpu(), k, k, cache, pos)
    no("multiple", dec, q[:, :-1].contiguous(), k, k, cache, pos)
    no("1..16", dec, torch.zeros((b, 3 * d), dtype=BF16, device=dev), k, k, cache, pos)
    no("1..16", dec, torch.zeros((b, 34 * d), dtype=BF16, device=dev), k, k, cache, pos)
    no("rope", dec, q, k, k, cache, pos, cos)
    no("rope", dec, q, k, k, cache, pos, cos, sin[:32])
    no("rope", dec, q, k, k, cache, pos, cos.double(), sin.double())
    no("finite", dec, q, k, k, cache, pos, scale=float("nan"))
    no("out must", dec, q, k, k, cache, pos, out=torch.empty((b, hq * d), device=dev))
    no("prefix", dec, q, k, k, cache, pos, prefix=cache, prefix_len=3)
    no("prefix", dec, q, k, k, cache, pos, prefix_len=3)
    no("lie in the cache", dec, q, k, k, cache, pos, prefix=tuple(c[1:] for c in cache), prefix_len=3)
    no("capacity", dec, q, k, k, cache, pos, prefix=pre, prefix_len=65)
    no("prefix", dec, q, k, k, cache, pos, prefix=pre, prefix_len=-1)
    no("four tensors", dec, q, k, k, cache[:3], pos)
    no("belong", dec, q, k, k, (cache.k, cache.k_scale, cache.k, cache.v_scale), pos)
    no("int8 codes", dec, q, k, k, (cache.k.float(), *cache[1:]), pos)
    no("contiguous", dec, q, k, k, (cache.k.transpose(2, 3).contiguous().transpose(2, 3), *cache[1:]), pos)
    no("HIP device", dec, q, k, k, tuple(c.cpu() for c in cache), pos)
    no("start", pro, q, k, k, cache, 64, 1)
    no("start", pro, q, k, k, cache, -1, 1)
    no("rotary", pro, q, k, k, cache, 0, 1, cos, sin, prefix=pre, prefix_len=64)
    no("lengths", pro, q, k, k, cache, 0, 1, lengths=pos.int())
    no("multiple|elements", pro, q, k, k, cache, 0, 3)
    no("start", pkg.kv_cache_write_i8, k, k, cache, 64, 1)
    no("dtype|expected", pkg.kv_cache_write_i8, k.half(), k.half(), cache, 0, 1)
    no("dtype", pkg.kv_cache_read_i8, cache, 0, 1, torch.float16)
    no("count|negative", pkg.kv_cache_read_i8, cache, 0, -1)
    no("head_dim", pkg.kv_cache_i8, 1, 1, 64, 96, dev)
