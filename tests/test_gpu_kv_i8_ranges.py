"""The attentions over the int8 cache where a number comes near the end of what holds it: value scales that double from
one block of keys to the next, one key that takes nearly all the weight, scores far outside the exponential's range.

Every case runs as a decode step over a sequence's own keys, as a prompt, and as a decode step behind a long prefix that
more than 32 rows share (the matrix-core form of prompts), so each softmax meets it.
"""

import math

import pytest
import torch

from test_gpu_kv_i8 import BF16, F32, Host, _attention, _check

pytestmark = pytest.mark.gpu

D = 64


def _empty(b, h, cap):
    return Host(b, h, cap, D, torch.Generator().manual_seed(0), empty=True)


class Keys:
    """``n`` keys and values, the same for every kv head, met by queries ``q`` [rows, D] in one of three ways; each row sees
    all of them, and new keys of zeros with values of zeros that ``n`` does not count."""

    FORMS = ["step", "prompt", "shared"]

    def __init__(self, form, n, heads, kv_heads, dtype):
        self.form, self.n, self.hq, self.h, self.dtype = form, n, heads, kv_heads, dtype
        # rows of the call: a step and a prompt's last token take one sequence; the prefix is shared by many sequences
        self.b, self.t = {"step": (3, 1), "prompt": (1, 33), "shared": (64, 1)}[form]
        self.cap = (n + self.t + 63) // 64 * 64
        self.held = _empty(1 if form == "shared" else self.b, kv_heads, self.cap)

    def call(self, pkg, dev, q, k_new, scale):
        """Outputs of the rows q [b * t, hq * D] with new keys k_new [b * t, h * D] and values of zeros."""
        own, start, kw = self.held, self.n, {}
        if self.form == "shared":
            own, start = _empty(self.b, self.h, 64), 0
            kw = {"prefix": self.held.to(pkg, dev), "prefix_len": self.n}
        cache = own.to(pkg, dev)
        args = (q.to(dev), k_new.to(dev), torch.zeros_like(k_new, device=dev), cache)
        if self.form == "prompt":
            out = pkg.gqa_prefill_attention_i8(*args, start, self.t, scale=scale, **kw)
        else:
            out = pkg.gqa_decode_attention_i8(*args, torch.full((self.b,), start, device=dev), scale=scale, **kw)
        return out.cpu()

    def run(self, pkg, dev, q, scale, half=True):
        """The outputs under new keys of zeros and the definition with its bound (``half``: with the terms of fp16
        products, where there are any)."""
        b, t, h, n = self.b, self.t, self.h, self.n
        zeros = torch.zeros((b * t, h * D), dtype=self.dtype)
        out = self.call(pkg, dev, q, zeros, scale)
        own, start, pre, npre = (_empty(b, h, 64), 0, self.held, n) if self.form == "shared" else (self.held, n, None, 0)
        own.write(zeros, zeros, [start] * b, [t] * b, t, None, None)
        ref, tol = _attention(q, own, [start] * b, [t] * b, t, None, None, scale, self.dtype, pre, npre,
                              half=half and self.form != "step")
        return out, ref, tol


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", Keys.FORMS)
def test_a_value_scale_that_doubles_under_a_growing_maximum(pkg, dev, form, dtype):
    """Values of scale 1, then one of scale 2 whose key's weight lies just under twice the maximum before it: weight and
    scale at the ends of their ranges at once (scores of 0, then of 0.9990 to 1.0001 in powers of two)."""
    print(f"[kv ranges] doubling {form} {dtype}", flush=True)
    m = Keys(form, 8800, 32, 4, dtype)
    m.held.v[:, :, :m.n] = torch.randint(-127, 128, (1, 4, m.n, D), generator=torch.Generator().manual_seed(1),
                                         dtype=torch.int8)
    m.held.vs[:, :, :m.n] = 1.0
    for j in range(70, m.n, 128):  # in every second block
        m.held.k[:, :, j, 0] = 127
        m.held.ks[:, :, j] = 1.0 / 127
        m.held.v[:, :, j, ::2] = 127
        m.held.vs[:, :, j] = 2.0
    rows = m.b * m.t * 32
    q = torch.zeros((rows, D))
    q[:, 0] = math.log(2.0) * torch.linspace(0.9990, 1.0001, rows)
    out, ref, tol = m.run(pkg, dev, q.reshape(-1, 32 * D).to(dtype), 1.0)
    _check(out, ref, tol, form)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", Keys.FORMS)
def test_keys_far_below_one_that_takes_the_weight(pkg, dev, form, dtype):
    """A key in every 128 with a value of zeros and a score of 10 to 16 above the rest (fp32: 14), whose equal weights make
    the whole output: they are as exact as the large one.  All values are positive, so the output's sum loses nothing and
    an error that the equal weights share shows in full.  The queries are exact in fp16; three roundings of 2^-11 are the
    weight's, the value scale's and the scaled value's."""
    print(f"[kv ranges] sink {form} {dtype}", flush=True)
    m = Keys(form, {"prompt": 500}.get(form, 1790), 32, 4, dtype)
    m.held.v[:, :, :m.n] = torch.randint(64, 128, (1, 4, m.n, D), generator=torch.Generator().manual_seed(2),
                                         dtype=torch.int8)
    m.held.vs[:, :, :m.n] = 1.0 / 127
    sinks = torch.arange(5, m.n, 128)
    m.held.k[:, :, sinks, 0] = 127
    m.held.ks[:, :, sinks] = 1.0 / 127
    m.held.v[:, :, sinks] = 0
    m.held.vs[:, :, sinks] = 0.0
    rows = m.b * m.t * 32
    q = torch.zeros((rows, D))
    q[:, 0] = torch.linspace(10.0, 16.0 if dtype == BF16 else 14.0, rows)
    out, ref, tol = m.run(pkg, dev, q.reshape(-1, 32 * D).to(dtype), 1.0, half=False)
    if dtype == BF16:
        tol = tol + 3 * 2.0 ** -11 * ref.abs()
    assert float(ref.min()) > 0.0 and float((tol / ref).max()) < 0.01
    _check(out, ref, tol, form)


def _one_takes_all(pkg, dev, form, dtype, size, sign):
    """Keys that are multiples of one direction, of elements up to ``size``, under queries of ``size``: the scores lie so
    far apart that the output is the value of the largest, the last key (sign 1) or the first (-1).  Roundings of q turn
    all scores alike; what remains is that of the output, and of fp16 the value's two."""
    print(f"[kv ranges] one takes all {form} {dtype} {size} {sign}", flush=True)
    m = Keys(form, 8800 if form == "shared" else 300, 32, 4, dtype)
    gen = torch.Generator().manual_seed(3)
    m.held.v[:, :, :m.n] = torch.randint(-127, 128, (1, 4, m.n, D), generator=gen, dtype=torch.int8)
    m.held.vs[:, :, :m.n] = 1.0 / 127
    m.held.k[:, :, :m.n] = 127 * sign
    m.held.ks[:, :, :m.n] = size / 127 * torch.arange(1, m.n + 1) / m.n
    rows = m.b * m.t
    q = (size * (1.0 + 0.5 * torch.rand((rows, 32 * D), generator=gen))).to(dtype)
    new = torch.full((rows, 4 * D), -2.0 * size if sign < 0 else 0.0, dtype=dtype)
    out = m.call(pkg, dev, q, new, D ** -0.5).double().reshape(rows, 4, 8, D)
    _, vals = m.held.held(0)
    ref = vals[None, :, None, m.n - 1 if sign > 0 else 0].expand_as(out)
    tol = (2.0 ** -8 + 2 * 2.0 ** -11 if dtype == BF16 else 2.0 ** -20) * ref.abs()
    _check(out, ref, tol, f"{form} {size} {sign}")


@pytest.mark.parametrize("size", [1e3, 2.5e3, 3e3, 4e3, 5e3, 1e4, 1e6, 1e10, 1e14])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", Keys.FORMS)
def test_scores_of_very_large_magnitude(pkg, dev, form, dtype, size):
    """Scores of 1e7 to 1e29, whose rounding alone is many powers of two."""
    for sign in (1, -1):
        _one_takes_all(pkg, dev, form, dtype, size, sign)


@pytest.mark.parametrize("size", [1e15, 1e16, 3e17, 1e18])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", Keys.FORMS)
def test_scores_close_to_the_end_of_fp32(pkg, dev, form, dtype, size):
    """Scores of 10^31 to 10^37 in powers of two, of either sign: a softmax is defined for all that are finite."""
    for sign in (1, -1):
        _one_takes_all(pkg, dev, form, dtype, size, sign)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 2])
@pytest.mark.parametrize("npre", [0, 1])
def test_a_first_key_of_any_score_returns_its_value(pkg, dev, dtype, tokens, npre):
    """The first token of a sequence sees one key (and a prefix of one key that lies further below): its output is that
    key's value whatever the score."""
    print(f"[kv ranges] first key {dtype} {tokens} {npre}", flush=True)
    gen = torch.Generator().manual_seed(4)
    q = torch.full((tokens, 2 * D), 1e16, dtype=dtype)
    v = torch.randn((tokens, D), generator=gen).to(dtype)
    pre = _empty(1, 1, 64)
    pre.k[:, :, 0], pre.ks[:, :, 0], pre.v[:, :, 0], pre.vs[:, :, 0] = -127, 1e20 / 127, 127, 1.0
    kw = {"prefix": pre.to(pkg, dev), "prefix_len": 1} if npre else {}
    for size in (-1e16, -1.0, 0.0, 1e16):
        host = _empty(1, 1, 64)
        cache = host.to(pkg, dev)
        k = torch.full((tokens, D), size, dtype=dtype)
        args = (q.to(dev), k.to(dev), v.to(dev), cache)
        if tokens == 1:
            out = pkg.gqa_decode_attention_i8(*args, torch.zeros(1, dtype=torch.int64, device=dev), **kw)
        else:
            out = pkg.gqa_prefill_attention_i8(*args, 0, tokens, **kw)
        host.write(k, v, [0], [tokens], tokens, None, None)
        ref = host.held(0)[1][0, 0].repeat(2)[None]
        tol = (2.0 ** -8 + 2 * 2.0 ** -11 if dtype == BF16 else 2.0 ** -20) * ref.abs()
        _check(out[:1], ref, tol, f"score of {size}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("form", Keys.FORMS)
def test_values_whose_sum_over_the_keys_is_just_within_fp32(pkg, dev, form, dtype):
    """8800 values of up to 2^113 on a split axis: their sum under weights of one stays below 2^127, and so do the parts
    of a row that are joined."""
    print(f"[kv ranges] large values {form} {dtype}", flush=True)
    m = Keys(form, 8800, 32, 4, dtype)
    gen = torch.Generator().manual_seed(6)
    m.held.v[:, :, :m.n] = torch.randint(64, 128, (1, 4, m.n, D), generator=gen, dtype=torch.int8)
    m.held.vs[:, :, :m.n] = 2.0 ** 106
    m.held.k[:, :, :m.n] = torch.randint(-127, 128, (1, 4, m.n, D), generator=gen, dtype=torch.int8)
    m.held.ks[:, :, :m.n] = 0.01
    q = torch.randn((m.b * m.t, 32 * D), generator=gen).to(dtype)
    out, ref, tol = m.run(pkg, dev, q, D ** -0.5, half=True)
    assert float((tol / ref).max()) < 0.1
    _check(out, ref, tol, form)
