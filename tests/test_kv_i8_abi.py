"""CPU checks of the int8 cache's entry points: arguments that are refused on the host, before any GPU work (the pointers
given are never dereferenced there), the workspace query, and the Python layer's refusals."""

import ctypes

import pytest
import torch

vp = ctypes.c_void_p


def _cache(pkg, cap=128, k=0x1000, ks=0x2000, v=0x3000, vs=0x4000):
    return pkg._lib.KvI8Struct(k, ks, v, vs, cap)


def _write(pkg, cache=None, k=0x1000, v=0x2000, dtype=1, ldk=128, ldv=128, cos=None, sin=None, rope_len=0, turn=0,
           start=0, batch=2, t=3, h=2, d=64):
    c = _cache(pkg) if cache is None else cache
    return pkg._lib.status("wfb_kv_write_i8", vp(k), ldk, vp(v), ldv, dtype, vp(cos) if cos else None,
                           vp(sin) if sin else None, rope_len, turn, ctypes.addressof(c) if c != 0 else None, None, start,
                           None, batch, t, h, d, None)


def test_write_refusals(pkg):
    def no(match, **kw):
        assert _write(pkg, **kw) == -1
        assert match in pkg._lib.last_error(), pkg._lib.last_error()

    no("head_dim", d=96)
    no("num_kv_heads", h=0)
    no("num_kv_heads", h=32768)
    no("batch", batch=65536)
    no("batch", batch=-1)
    no("null cache", cache=0)
    no("capacity", cache=_cache(pkg, cap=100))
    no("capacity", cache=_cache(pkg, cap=0))
    no("capacity", cache=_cache(pkg, cap=1 << 26))
    no("null cache pointer", cache=_cache(pkg, vs=None))
    no("16-byte", cache=_cache(pkg, ks=0x2004))
    no("dtype", dtype=2)
    no("T (", t=-1)
    no("T (", t=(1 << 24) + 1)
    no("strides", ldk=120)
    no("strides", ldv=132)
    no("strides", dtype=0, ldk=130)
    no("both", cos=0x100)
    no("prefix length", turn=-1)
    no("start", start=-1)
    no("start", start=126)
    no("rotary", cos=0x100, sin=0x100, rope_len=2)
    no("rotary", cos=0x100, sin=0x100, rope_len=100, turn=98)
    no("null pointer", k=0)
    no("16-byte", v=0x2008)
    no("16-byte", cos=0x104, sin=0x100, rope_len=100)
    assert _write(pkg, batch=0) == 0 and _write(pkg, t=0, k=0) == 0


def test_read_refusals(pkg):
    def read(cache=None, start=0, batch=1, count=4, h=2, d=64, k=0x1000, v=0x2000, dtype=1):
        c = _cache(pkg) if cache is None else cache
        return pkg._lib.status("wfb_kv_read_i8", ctypes.addressof(c), None, start, batch, count, h, d, vp(k), vp(v), dtype,
                               None)

    for kw, match in ((dict(dtype=2), "dtype"), (dict(count=-1), "count"), (dict(count=1 << 25), "count"),
                      (dict(k=0), "null"), (dict(v=0x2004), "16-byte"), (dict(d=32), "head_dim"),
                      (dict(cache=_cache(pkg, cap=65)), "capacity")):
        assert read(**kw) == -1 and match in pkg._lib.last_error(), (kw, pkg._lib.last_error())
    assert read(count=0, k=0) == 0 and read(batch=0) == 0


def _workspace(pkg, batch, t, hq, h, d, cap, prefix=0):
    n = ctypes.c_int64(-1)
    st = pkg._lib.status("wfb_gqa_attention_i8_workspace", batch, t, hq, h, d, cap, prefix, ctypes.addressof(n))
    return n.value if st == 0 else st


def test_workspace(pkg):
    assert _workspace(pkg, 0, 1, 8, 2, 64, 128) == 0 and _workspace(pkg, 2, 0, 8, 2, 64, 128) == 0
    for bad in ((-1, 1, 8, 2, 64, 128), (1, 1 << 25, 8, 2, 64, 128), (1, 1, 9, 2, 64, 128), (1, 1, 34, 2, 64, 128),
                (1, 1, 8, 2, 64, 100), (1, 1, 8, 2, 80, 128), (1, 1, 8, 2, 64, 128, -1), (1, 1, 8, 0, 64, 128)):
        assert _workspace(pkg, *bad) == -1, bad
    assert pkg._lib.status("wfb_gqa_attention_i8_workspace", 1, 1, 8, 2, 64, 128, 0, None) == -1
    for batch in (1, 7, 64, 300):
        for t in (1, 3, 300):
            for cap in (64, 1024, 1088, 131072):
                for prefix in (0, 1, 5000):
                    n = _workspace(pkg, batch, t, 8, 2, 64, cap, prefix)
                    rows = batch * t * 8 * 66  # outputs, maximum and sum of a part
                    assert n >= 0 and n % rows == 0 and n // rows <= 2 * 1024
                    assert t > 1 or prefix == 0 or n >= 2 * rows  # a prefix is a part of its own


def _attend(pkg, cache=None, prefix=None, prefix_len=0, q=0x1000, out=0x5000, ldq=512, ldo=512, hq=8, h=2, d=64, batch=2,
             t=3, dtype=1, scale=0.125, ws=0x6000, ldk=128, cap=128):
    c = _cache(pkg, cap=cap) if cache is None else cache
    return pkg._lib.status("wfb_gqa_attention_i8", vp(q), ldq, vp(0x2000), ldk, vp(0x3000), ldk, dtype, None, None, 0,
                           ctypes.addressof(c), None, 0, None, ctypes.addressof(prefix) if prefix else None, prefix_len,
                           batch, t, hq, h, d, scale, vp(out), ldo, vp(ws) if ws else None, None)


def test_attention_refusals(pkg):
    def no(match, **kw):
        assert _attend(pkg, **kw) == -1
        assert match in pkg._lib.last_error(), pkg._lib.last_error()

    no("1..16", hq=9)
    no("1..16", hq=34, ldq=34 * 64, ldo=34 * 64)
    no("without a prefix", prefix_len=5)
    no("without a prefix", prefix_len=-1)
    no("capacity", prefix=_cache(pkg), prefix_len=129)
    no("capacity", prefix=_cache(pkg, cap=96), prefix_len=5)
    no("null cache pointer", prefix=_cache(pkg, k=None), prefix_len=5)
    # the cache's codes span 2 * 2 * 128 * 64 bytes from k and v, the prefix's half of that
    far = dict(k=0x100000, v=0x200000)
    no("lie in the cache", prefix=_cache(pkg, k=0x1000, v=0x200000), prefix_len=5)
    no("lie in the cache", prefix=_cache(pkg, k=0x1000 + 4 * 128 * 64 - 16, v=0x200000), prefix_len=5)
    no("lie in the cache", cache=_cache(pkg, k=0x100000, v=0x200000),
       prefix=_cache(pkg, k=0x300000, v=0x200000 - 2 * 128 * 64 + 16), prefix_len=5)
    assert _attend(pkg, cache=_cache(pkg, **far), prefix=_cache(pkg, k=0x100000 + 4 * 128 * 64, v=0x200000 - 2 * 128 * 64),
                   prefix_len=5, t=0) == 0
    no("strides", ldq=500)
    no("strides", ldo=516)
    no("strides", ldk=64)
    no("finite", scale=float("inf"))
    no("finite", scale=float("nan"))
    no("null pointer", q=0)
    no("null pointer", out=0)
    no("16-byte", q=0x1004)
    no("16-byte", ws=0x6004)
    no("workspace", ws=0, batch=1, t=1, cap=4096)
    no("2^30", batch=65535, t=1 << 14, cap=1 << 15)
    no("2^21", batch=65535, hq=64, h=32, ldq=64 * 64, ldo=64 * 64, ldk=32 * 64, t=1)
    assert _attend(pkg, batch=0) == 0 and _attend(pkg, t=0, q=0) == 0


def test_python_layer_needs_device_tensors(pkg):
    c = pkg.kv_cache_i8(2, 2, 100, 64, "cpu")
    assert c.k.shape == (2, 2, 128, 64) and c.v.shape == (2, 2, 2, 64, 64)
    assert c.k_scale.shape == c.v_scale.shape == (2, 2, 128) and c.k_scale.dtype == torch.float32
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.kv_cache_write_i8(x, x, c, 0, 1)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.kv_cache_read_i8(c, 0, 1)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.gqa_decode_attention_i8(x, x, x, c, torch.zeros(2, dtype=torch.int64))
    for bad in (dict(max_len=0), dict(head_dim=80), dict(batch=0), dict(kv_heads=0)):
        with pytest.raises(ValueError):
            pkg.kv_cache_i8(**{**dict(batch=1, kv_heads=1, max_len=64, head_dim=64, device="cpu"), **bad})


def test_model_refuses_what_the_int8_cache_does_not_take(pkg):
    M = pkg.model
    ok = dict(vocab_size=64, hidden_size=128, intermediate_size=128, num_layers=1, num_heads=2, num_kv_heads=1,
              head_dim=64, rope_theta=1e4)
    for cfg, kw in ((ok, dict(kv_cache="int4")), (ok, dict(kv_cache="int8", decode_attention="torch")),
                    (ok, dict(kv_cache="int8", prefill_attention="steps")),
                    (ok, dict(kv_cache="int8", dtype=torch.float16)),
                    (dict(ok, head_dim=32), dict(kv_cache="int8")), (dict(ok, num_heads=17), dict(kv_cache="int8"))):
        with pytest.raises(ValueError, match="kv_cache"):
            M.BitNetDecoder(M.BitNetConfig(**cfg), device="cpu", **kw)


@pytest.mark.parametrize("lengths", [1, 0, [1, 1], (1, 1), 1.0])
def test_lengths_that_are_no_tensor_are_refused(pkg, lengths):
    """A length for the whole batch is not a form of the call: dropped, all t tokens would be written and attended."""
    c = pkg.kv_cache_i8(2, 2, 100, 64, "cpu")
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="lengths"):
        pkg.kv_cache_write_i8(x, x, c, 0, 1, lengths=lengths)
    with pytest.raises(RuntimeError, match="lengths"):
        pkg.gqa_prefill_attention_i8(x, x, x, c, 0, 1, lengths=lengths)


def test_a_prefix_without_its_length_is_refused(pkg):
    """Taken as a length of zero, the prefix would not be attended to at all."""
    c, pre = pkg.kv_cache_i8(2, 2, 100, 64, "cpu"), pkg.kv_cache_i8(1, 2, 100, 64, "cpu")
    x = torch.zeros((2, 128), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="prefix_len"):
        pkg.gqa_decode_attention_i8(x, x, x, c, torch.zeros(2, dtype=torch.int64), prefix=pre)
    with pytest.raises(RuntimeError, match="prefix_len"):
        pkg.gqa_prefill_attention_i8(x, x, x, c, 0, 1, prefix=pre)


def test_share_prefix_takes_one_sequence(pkg):
    """Prompts of several sequences are not joined to one; the prefix that is there stays."""
    model = pkg.model.BitNetDecoder.__new__(pkg.model.BitNetDecoder)
    model.kv_cache, model._prefix, model._prefix_len = "int8", "held", 7
    with pytest.raises(ValueError, match="one sequence"):
        model.share_prefix(torch.zeros((2, 3), dtype=torch.long))
    assert (model._prefix, model._prefix_len) == ("held", 7)
