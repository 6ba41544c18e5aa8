"""CPU checks of the training step's entry points: arguments refused on the host, before any GPU work (the pointers
given are never dereferenced there), the workspace queries, the rotary tables for long contexts and the Python layer's
refusals."""

import ctypes
import math

import pytest
import torch

vp = ctypes.c_void_p


def _no(pkg, match, status):
    assert status == -1 and match in pkg._lib.last_error(), pkg._lib.last_error()


def test_gated_refusals(pkg):
    def fwd(qw=0x1000, f=64, k=256, codes=0x2000, m=4, lda=256, a=0x100, s=0x200, act=1, h=0x3000, hdt=1, gu=0x4000):
        return pkg._lib.status("wfb_gated_i2s", vp(qw), f, k, vp(codes), m, lda, vp(a), vp(s), act, vp(h), hdt, vp(gu), None)

    for match, kw in (("sizes", dict(f=0)), ("sizes", dict(m=-1)), ("2^20", dict(m=1 << 20)), ("2^20", dict(f=1 << 19)),
                      ("multiple", dict(k=200)), ("activation", dict(act=3)), ("dtype", dict(hdt=5)), ("null", dict(qw=None)),
                      ("null", dict(a=None)), ("null", dict(h=None)), ("16-byte", dict(codes=0x2008)),
                      ("16-byte", dict(gu=0x4004)), ("16-byte", dict(h=0x3002)), ("stride", dict(lda=128)),
                      ("stride", dict(lda=264)), ("stride", dict(lda=1 << 25))):
        _no(pkg, match, fwd(**kw))
    assert fwd(m=0, qw=None) == 0

    def pack(g=0x1000, u=0x2000, dt=0, f=64, k=200, s=0x100, q=0x3000, ws=0x4000):
        return pkg._lib.status("wfb_pack_gated", vp(g), vp(u), dt, f, k, vp(s), vp(q), vp(ws), None)

    for match, kw in (("sizes", dict(f=0)), ("sizes", dict(k=0)), ("2^20", dict(k=1 << 20)), ("dtype", dict(dt=3)),
                      ("null", dict(u=None)), ("null", dict(ws=None)), ("misaligned", dict(q=0x3001)),
                      ("misaligned", dict(ws=0x4004))):
        _no(pkg, match, pack(**kw))

    def bwd(gu=0x1000, gh=0x2000, ghdt=1, ldg=64, m=4, f=64, act=1, qw=0x3000, k=200, kp=256, s=0x100, c=0x4000, lda=256,
            a=0x200, gx=0x5000, gxdt=1, gw=0x6000, gwdt=0, work=0x10000):
        return pkg._lib.status("wfb_gated_grad", vp(gu), vp(gh), ghdt, ldg, m, f, act, vp(qw), k, kp, vp(s), vp(c), lda, vp(a),
                               vp(gx), gxdt, vp(gw), gwdt, vp(work), None)

    for match, kw in (("no rows", dict(m=0)), ("activation", dict(act=0)), ("dtype", dict(ghdt=7)), ("dtype", dict(gwdt=-1)),
                      ("null", dict(gu=None)), ("null", dict(gx=None, gw=None)), ("null", dict(work=None)),
                      ("packed rows", dict(kp=128)), ("packed rows", dict(kp=300)), ("packed rows", dict(qw=0x3004)),
                      ("strides", dict(ldg=63)), ("strides", dict(lda=199)), ("aligned", dict(work=0x10010)),
                      ("aligned", dict(gu=0x1004)), ("2^20", dict(k=1 << 20, kp=1 << 20))):
        _no(pkg, match, bwd(**kw))


def test_gated_workspaces(pkg):
    n = ctypes.c_int64(-1)
    at = ctypes.addressof(n)
    sizes = {}
    for want in ((1, 0), (0, 1), (1, 1)):
        assert pkg._lib.status("wfb_gated_grad_workspace", 100, 65, 200, 1, want[0], 0, want[1], at) == 0
        sizes[want] = n.value
    assert 0 < sizes[1, 0] < sizes[1, 1] and 0 < sizes[0, 1] < sizes[1, 1]
    # two planes of d^T, 2 F rows of 128 tokens, and the codes at the least
    assert sizes[0, 1] >= 2 * 2 * 130 * 128 + 2 * 200 * 128
    assert pkg._lib.status("wfb_gated_grad_workspace", 0, 65, 200, 1, 1, 0, 1, at) == 0 and n.value == 0
    _no(pkg, "null", pkg._lib.status("wfb_gated_grad_workspace", 1, 1, 1, 1, 1, 0, 1, None))
    _no(pkg, "dtype", pkg._lib.status("wfb_gated_grad_workspace", 1, 1, 1, 9, 1, 0, 1, at))


def _heads(pkg, x=0x1000, heads=4, out=0x2000, **kw):
    s = pkg._lib.HeadsStruct()
    s.x, s.heads, s.out, s.g = x, heads, out, 0x3000
    s.stride_b, s.stride_t, s.stride_h = 64 * 64, 64 * 4, 64
    s.g_stride_b, s.g_stride_t, s.g_stride_h = 64 * 64, 64 * 4, 64
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _rope(pkg, **kw):
    r = pkg._lib.RopeStruct()
    r.cos, r.sin, r.rope_len, r.rotary_dim = 0x100, 0x200, 32, 64
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def test_qk_refusals(pkg):
    for name in ("wfb_qk_norm_rope", "wfb_qk_norm_rope_grad"):
        grad = name.endswith("grad")

        def call(q=None, k=None, rope=None, dtype=1, b=2, t=8, d=64, work=0x100, null=False):
            q, k, rope = q or _heads(pkg), k or _heads(pkg, heads=2), rope or _rope(pkg)
            args = [None if null else ctypes.addressof(q), ctypes.addressof(k), ctypes.addressof(rope), dtype, b, t, d, 1e-6]
            return pkg._lib.status(name, *args, *([vp(work)] if grad else []), None)

        for match, kw in (("null", dict(null=True)), ("dtype", dict(dtype=3)), ("head_dim", dict(d=63)),
                          ("head_dim", dict(d=258)), ("head_dim", dict(d=0)), ("rotary_dim", dict(rope=_rope(pkg, rotary_dim=66))),
                          ("rotary_dim", dict(rope=_rope(pkg, rotary_dim=31))), ("sizes", dict(b=-1)),
                          ("sizes", dict(q=_heads(pkg, heads=65536))), ("tables", dict(rope=_rope(pkg, cos=None))),
                          ("tables", dict(rope=_rope(pkg, rope_len=0))), ("4-byte", dict(rope=_rope(pkg, sin=0x202))),
                          ("int32 or int64", dict(rope=_rope(pkg, pos=0x100, pos_bytes=2))),
                          ("leave", dict(rope=_rope(pkg, start=25))), ("leave", dict(rope=_rope(pkg, start=-1))),
                          ("weight dtype", dict(q=_heads(pkg, weight=0x100, weight_dtype=4))),
                          ("null pointer", dict(k=_heads(pkg, x=None))), ("aligned", dict(q=_heads(pkg, x=0x1001))),
                          ("without the weight", dict(q=_heads(pkg, grad_weight=0x100))),
                          ("2^31", dict(b=1 << 17, t=1 << 13, rope=_rope(pkg, rope_len=1 << 14)))):
            _no(pkg, match, call(**kw))
        if grad:
            _no(pkg, "workspace", call(q=_heads(pkg, weight=0x100, grad_weight=0x100), work=None))
        else:
            _no(pkg, "null pointer", call(q=_heads(pkg, out=None)))
            assert call(b=0) == 0 and call(t=0) == 0
    n = ctypes.c_int64(-1)
    assert pkg._lib.status("wfb_qk_norm_rope_grad_workspace", 4, 2048, 32, 8, 128, ctypes.addressof(n)) == 0
    assert n.value > 0 and n.value % 256 == 0
    _no(pkg, "null", pkg._lib.status("wfb_qk_norm_rope_grad_workspace", 4, 2048, 32, 8, 128, None))
    _no(pkg, "sizes", pkg._lib.status("wfb_qk_norm_rope_grad_workspace", 4, 2048, 32, 8, 512, ctypes.addressof(n)))


def test_adamw_refusals(pkg):
    def call(rows=((0x1000, 0x2000, 300),), pdt=0, gdt=1, m=0x3000, v=0x4000, ms=0x100, vs=0x200, n=512, bits=8, lr=1e-3,
             b1=0.9, b2=0.99, eps=1e-8, wd=0.0, step=1, step_dev=None, lr_dev=None, scalars=None, tensors=True):
        flat = [x for r in rows for x in r]
        table = (ctypes.c_int64 * max(1, len(flat)))(*flat)
        return pkg._lib.status("wfb_adamw_step", ctypes.addressof(table) if tensors else None, len(rows), pdt, gdt, vp(m), vp(v),
                               vp(ms) if ms else None, vp(vs) if vs else None, n, bits, lr, b1, b2, eps, wd, step,
                               vp(step_dev) if step_dev else None, vp(lr_dev) if lr_dev else None,
                               vp(scalars) if scalars else None, None)

    for match, kw in (("bits", dict(bits=16)), ("multiple", dict(n=500)), ("null state", dict(m=None)),
                      ("null state", dict(ms=None)), ("16-byte", dict(v=0x4008)), ("4-byte", dict(vs=0x202)),
                      ("dtype", dict(pdt=3)), ("dtype", dict(gdt=-1)), ("tensor list", dict(tensors=False)),
                      ("betas", dict(b1=1.0)), ("betas", dict(b2=-0.1)), ("betas", dict(b1=math.nan)),
                      ("negative", dict(lr=-1.0)), ("negative", dict(eps=-1.0)), ("negative", dict(wd=math.nan)),
                      ("steps", dict(step=0)), ("device step", dict(lr_dev=0x100)), ("scalars", dict(step_dev=0x100)),
                      ("leaves the state", dict(rows=((0x1000, 0x2000, 513),))),
                      ("leaves the state", dict(rows=((0x1000, 0x2000, 300), (0x9000, 0x8000, 1)))),
                      ("leaves the state", dict(rows=((0x1000, 0x2000, -1),))),
                      ("elements", dict(rows=((0x1000, 0x2000, 100),))),
                      ("misaligned", dict(rows=((0x1002, 0x2000, 300),))), ("misaligned", dict(rows=((0x1000, 0x2001, 300),))),
                      ("null", dict(rows=((0, 0x2000, 300),)))):
        _no(pkg, match, call(**kw))
    assert call(rows=()) == 0 and call(rows=((0, 0, 0), (0, 0, 300), (0x1000, 0, 0))) == 0

    def values(m=0x1000, n=512, mo=0x3000):
        return pkg._lib.status("wfb_adamw_values", vp(m), vp(0x2000), vp(0x100), vp(0x200), n, vp(mo), vp(0x4000), None)

    _no(pkg, "multiple", values(n=100))
    _no(pkg, "16-byte", values(mo=0x3004))
    _no(pkg, "null state", values(m=None))
    assert values(n=0) == 0


def test_scaled_tables(pkg):
    theta, d, n = 500000.0, 128, 300
    for scaling in (dict(type="linear", factor=8.0),
                    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                         original_max_position_embeddings=8192),
                    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)):
        cos, sin = pkg.rope_tables(theta, d, n, scaling=scaling)
        kind = scaling.get("type", scaling.get("rope_type"))
        for i in range(d // 2):
            f = theta ** (-2 * i / d)
            mscale = 1.0
            if kind == "linear":
                f /= 8.0
            elif kind == "llama3":
                wave = 2 * math.pi / f
                if wave > 8192:
                    f /= 8.0
                elif wave > 8192 / 4:
                    w = (8192 / wave - 1) / 3
                    f = (1 - w) * f / 8 + w * f
            else:
                lo = math.floor(d * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(theta)))
                hi = math.ceil(d * math.log(4096 / (2 * math.pi)) / (2 * math.log(theta)))
                slow = min(1.0, max(0.0, (i - lo) / (hi - lo)))
                f, mscale = f / 4 * slow + f * (1 - slow), 0.1 * math.log(4.0) + 1.0
            for p in (0, 1, 17, n - 1):
                # a frequency from another order of operations: a few roundings of 2^-53 times the position, and fp32's
                assert abs(float(cos[p, i]) - mscale * math.cos(p * f)) <= 2.0 ** -23
                assert abs(float(sin[p, i]) - mscale * math.sin(p * f)) <= 2.0 ** -23
    assert torch.equal(pkg.rope_tables(theta, d, n)[0], pkg.rope_tables(theta, d, n, scaling=dict(type="linear"))[0])
    for bad in (dict(type="dynamic", factor=2.0), dict(type="linear", factor=0.5), dict(type="yarn", factor=2.0),
                dict(type="llama3", factor=2.0, original_max_position_embeddings=100, low_freq_factor=4.0, high_freq_factor=1.0),
                dict(type="yarn", factor=2.0, original_max_position_embeddings=100, beta_fast=1.0, beta_slow=2.0), {}):
        with pytest.raises(ValueError):
            pkg.rope_tables(theta, d, n, scaling=bad)


def test_python_refusals_on_the_cpu(pkg):
    x = torch.zeros(2, 3, 4, 64)
    cos = torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.qk_norm_rope(x, x, cos, cos)
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.gated_bitlinear(torch.zeros(2, 128), torch.zeros(8, 128), torch.zeros(8, 128))
    with pytest.raises(RuntimeError, match="HIP device"):
        pkg.adamw_step([x], [x], pkg.adamw_state([x]), 1)
    with pytest.raises(ValueError, match="no tensors"):
        pkg.adamw_state([])
    with pytest.raises(ValueError, match="act"):
        pkg.GatedBitLinear(8, 8, act="tanh")
    with pytest.raises(RuntimeError, match="bias"):
        pkg.GatedBitLinear.from_linears(torch.nn.Linear(8, 8), torch.nn.Linear(8, 8, bias=False))
    state = pkg.adamw_state([torch.zeros(300), torch.zeros(1)], 8)
    assert state.m.numel() == 768 and state.m_scale.numel() == 3 and state.v.dtype == torch.uint8
