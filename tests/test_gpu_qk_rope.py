"""qk_norm_rope and its gradients against float64.

Bounds: a normed element takes at most 8 fp32 roundings (a mean of squares of up to 256 terms adds a few more to the
shared factor: sqrt(256) / 2 = 8 at most of 2^-24), the rotation three of its two terms: |error| <= 24 roundings of 2^-24 of
|a| + |b|, the pair's magnitudes, and half a step of the type.  Gradients: two such sums, 48 roundings of the row's
largest terms.  A weight's gradient is a sum over N rows: normwise sqrt(N) / 8 + 24 roundings at the most, and half a step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def _tables(dev, n, r):
    ang = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
        -torch.arange(0, r, 2, dtype=torch.float64, device=dev) / max(r, 1))[None, :]
    return ang.cos().float(), ang.sin().float()


def _idx(r, layout, dev):
    i = torch.arange(r // 2, device=dev)
    return (i, i + r // 2) if layout == "half" else (2 * i, 2 * i + 1)


def _turn(y, cos, sin, layout, back=False):
    """The rotation of y [b, t, h, d] in float64 with cos / sin [b, t, 1, r / 2]."""
    a, b = _idx(2 * cos.shape[-1], layout, y.device)
    s = -sin if back else sin
    z = y.clone()
    z[..., a] = y[..., a] * cos - y[..., b] * s
    z[..., b] = y[..., b] * cos + y[..., a] * s
    return z


def _exact(x, w, cos, sin, pos, eps, layout, g=None):
    xd = x.double()
    c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
    if w is None:
        return (_turn(xd, c, s, layout),) if g is None else (_turn(xd, c, s, layout), _turn(g.double(), c, s, layout, True), None)
    r = torch.rsqrt(xd.square().mean(-1, keepdim=True) + eps)
    out = _turn(xd * r * w.double(), c, s, layout)
    if g is None:
        return (out,)
    gy = _turn(g.double(), c, s, layout, True)
    gw = gy * w.double()
    n = xd * r
    return out, r * (gw - n * (gw * n).mean(-1, keepdim=True)), (gy * n).sum((0, 1, 2))


def _check(got, ref, roundings, dtype, what):
    """Elementwise: so many roundings of the row's largest, and half a step."""
    top = ref.abs().amax(-1, keepdim=True)
    lim = roundings * U * top + torch.finfo(dtype).eps / 2 * ref.abs() * 1.001 + torch.finfo(dtype).tiny
    assert got.dtype == dtype and bool(((got.double() - ref).abs() <= lim).all()), (what, float(
        ((got.double() - ref).abs() - lim).max()))


def _inputs(dev, b, t, hq, hk, d, dtype, seed=0, wdtype=None):
    g = torch.Generator(device=dev).manual_seed(seed + b * 1000 + t + d)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    qkv = (rand(b, t, (hq + 2 * hk) * d) * (0.1 + rand(b, t, 1).abs())).to(dtype)
    q, k, _ = qkv.split([hq * d, hk * d, hk * d], 2)
    w = [(1 + 0.3 * rand(d)).to(wdtype or dtype) for _ in range(2)]
    return (q.unflatten(2, (hq, d)), k.unflatten(2, (hk, d)), *w, rand(b, t, hq, d).to(dtype), rand(b, t, hk, d).to(dtype))


def _run(pkg, q, k, cos, sin, pos, wq, wk, gq, gk, layout, eps=1e-6):
    leaves = [None if x is None else x.detach().requires_grad_() for x in (q, k, wq, wk)]
    out = pkg.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3], eps=eps, layout=layout)
    grads = torch.autograd.grad(out, [x for x in leaves if x is not None], [gq, gk])
    return [o.detach() for o in out], list(grads)


# head_dim, rotary: every chunk length and lanes a row, rotated whole, in part and not at all
DIMS = [(128, 128), (64, 64), (256, 256), (64, 32), (128, 32), (192, 96), (96, 96), (80, 20), (80, 80), (32, 8), (2, 2),
        (6, 2), (10, 6), (18, 18), (254, 254), (250, 126), (256, 64), (64, 0), (200, 200), (36, 36)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,r", DIMS)
def test_values_and_gradients(pkg, dev, d, r, layout, dtype):
    b, t, hq, hk = 2, 7, 9, 3
    q, k, wq, wk, gq, gk = _inputs(dev, b, t, hq, hk, d, dtype)
    cos, sin = _tables(dev, 50, r)
    pos = torch.randint(0, 50, (b, t), device=dev, generator=torch.Generator(device=dev).manual_seed(d))
    outs, grads = _run(pkg, q, k, cos, sin, pos, wq, wk, gq, gk, layout)
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        ref, rx, rw = _exact(x, w, cos, sin, pos, 1e-6, layout, g)
        _check(outs[i], ref, 24, dtype, "out")
        _check(grads[i], rx, 96, dtype, "grad_x")
        off = float((grads[2 + i].double() - rw).norm() / rw.norm())
        assert off <= (24 + (b * t * x.shape[2]) ** 0.5) * U + torch.finfo(dtype).eps / 2, off
    with torch.no_grad():
        served = pkg.qk_norm_rope(q, k, cos, sin, pos, wq, wk, layout=layout)
    assert all(torch.equal(a, o) for a, o in zip(served, outs))
    plain, grads = _run(pkg, q, k, cos, sin, pos, None, None, gq, gk, layout)
    for i, (x, g) in enumerate(((q, gq), (k, gk))):
        ref, rx, _ = _exact(x, None, cos, sin, pos, 0, layout, g)
        _check(plain[i], ref, 4, dtype, "turned")
        _check(grads[i], rx, 4, dtype, "turned back")


@pytest.mark.parametrize("b,t,hq,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (3, 333, 9, 3), (8, 1, 20, 5), (1, 2049, 7, 1), (5, 64, 13, 13)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_batches(pkg, dev, b, t, hq, hk, dtype):
    q, k, wq, wk, gq, gk = _inputs(dev, b, t, hq, hk, 64, dtype, wdtype=F32)
    cos, sin = _tables(dev, t + 100, 64)
    outs, grads = _run(pkg, q, k, cos, sin, 77, wq, wk, gq, gk, "half")
    pos = (77 + torch.arange(t, device=dev)).expand(b, t)
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        ref, rx, rw = _exact(x, w, cos, sin, pos, 1e-6, "half", g)
        _check(outs[i], ref, 24, dtype, "out")
        _check(grads[i], rx, 96, dtype, "grad_x")
        assert float((grads[2 + i].double() - rw).norm() / rw.norm()) <= (24 + (b * t * x.shape[2]) ** 0.5) * U + 2.0 ** -24
    for p in (pos, pos.int(), pos[0], pos[0].int(), pos.t().contiguous().t()):
        got = pkg.qk_norm_rope(q, k, cos, sin, p, wq, wk)
        assert all(torch.equal(a, o) for a, o in zip(got, outs))
    flat = pkg.qk_norm_rope(q[0], k[0], cos, sin, pos[0], wq, wk)
    assert all(torch.equal(a, o[0]) for a, o in zip(flat, outs))


def test_one_side_normed_and_wanted(pkg, dev):
    q, k, wq, wk, gq, gk = _inputs(dev, 2, 33, 6, 2, 128, BF16)
    cos, sin = _tables(dev, 40, 128)
    both, gb = _run(pkg, q, k, cos, sin, None, wq, wk, gq, gk, "half")
    bare, ga = _run(pkg, q, k, cos, sin, None, None, None, gq, gk, "half")
    outs, grads = _run(pkg, q, k, cos, sin, None, wq, None, gq, gk, "half")
    assert torch.equal(outs[0], both[0]) and torch.equal(outs[1], bare[1])
    assert torch.equal(grads[0], gb[0]) and torch.equal(grads[1], ga[1]) and torch.equal(grads[2], gb[2])
    leaf = wk.detach().requires_grad_()
    out = pkg.qk_norm_rope(q, k, cos, sin, None, wq, leaf)
    (g,) = torch.autograd.grad(out, [leaf], [gq, gk])
    assert torch.equal(g, gb[3])
    leaf = k.detach().requires_grad_()
    out = pkg.qk_norm_rope(q, leaf, cos, sin, None, wq, wk)
    (g,) = torch.autograd.grad(out[1], [leaf], gk)  # the queries' result unused
    assert torch.equal(g, gb[1])


def test_gradients_against_differences(pkg, dev):
    q, k, wq, wk, gq, gk = _inputs(dev, 1, 5, 2, 1, 16, F32)
    cos, sin = _tables(dev, 9, 8)
    _, grads = _run(pkg, q, k, cos, sin, 3, wq, wk, gq, gk, "interleaved")
    pos = 3 + torch.arange(5, device=dev)[None]
    gen = torch.Generator(device=dev).manual_seed(1)

    def loss(qs, ks, ws, vs):
        c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
        norm = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
        return float((_turn(norm(qs, ws), c, s, "interleaved") * gq).sum() + (_turn(norm(ks, vs), c, s, "interleaved") * gk).sum())

    at = [x.double() for x in (q, k, wq, wk)]
    for i, g in enumerate(grads):
        v = torch.randn(at[i].shape, generator=gen, device=dev).double()
        ends = [loss(*[x + sign * 1e-5 * v if j == i else x for j, x in enumerate(at)]) for sign in (1, -1)]
        # the truncation, step^2 times a third derivative that grows as the smallest row's inverse norm cubed, is below 1e-6
        assert abs((ends[0] - ends[1]) / 2e-5 - float((g.double() * v).sum())) <= 1e-5 * float(g.double().norm() * v.norm())


def test_strides_alignment_and_broadcast(pkg, dev):
    b, t, h, d = 2, 9, 4, 64
    q, k, wq, wk, gq, gk = _inputs(dev, b, t, h, 2, d, BF16)
    cos, sin = _tables(dev, 20, d)
    want, gw = _run(pkg, q, k, cos, sin, None, wq, wk, gq, gk, "half")
    for off in (1, 2, 4):  # rows that start at odd elements, words, half chunks
        buf = torch.zeros(b * t * h * d + off, dtype=BF16, device=dev)
        view = buf[off:].view(b, t, h, d).copy_(q)
        outs, grads = _run(pkg, view, k, cos, sin, None, wq, wk, gq, gk, "half")
        assert torch.equal(outs[0], want[0]) and torch.equal(grads[0], gw[0])
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)  # [b, h, t, d] in memory
    g_first = gq.transpose(1, 2).contiguous().transpose(1, 2)
    outs, grads = _run(pkg, heads_first, k, cos, sin, None, wq, wk, g_first, gk, "half")
    assert torch.equal(outs[0], want[0]) and torch.equal(grads[0], gw[0])
    scattered = q.transpose(2, 3).contiguous().transpose(2, 3)  # no contiguous heads
    outs, grads = _run(pkg, scattered, k, cos, sin, None, wq, wk, gq, gk, "half")
    assert torch.equal(outs[0], want[0]) and torch.equal(grads[0], gw[0])
    leaf = q.detach().requires_grad_()
    a, c = pkg.qk_norm_rope(leaf, k, cos, sin, None, wq, wk)
    (g,) = torch.autograd.grad(a.sum(), [leaf])
    assert torch.equal(g, _run(pkg, q, k, cos, sin, None, wq, wk, torch.ones_like(gq), gk, "half")[1][0])
    one = q[:, :1].expand(b, t, h, d)  # a token for all: stride 0
    assert torch.equal(pkg.qk_norm_rope(one, k, cos, sin, None, wq, wk)[0],
                       pkg.qk_norm_rope(one.contiguous(), k, cos, sin, None, wq, wk)[0])


def test_lazily_negated_operands(pkg, dev):
    q, k, wq, wk, gq, gk = _inputs(dev, 1, 5, 4, 2, 64, F32)
    cos, sin = _tables(dev, 20, 64)
    neg = torch._neg_view
    a, ga = _run(pkg, -q, k, cos, sin, None, wq, wk, -gq, gk, "half")
    b, gb = _run(pkg, neg(q.contiguous()), k, cos, sin, None, wq, wk, neg(gq), gk, "half")
    assert all(torch.equal(x, y) for x, y in zip((*a, *ga), (*b, *(g.resolve_neg() for g in gb))))


def test_offsets_past_32_bits(pkg, dev):
    d = 64
    buf = torch.zeros((1 << 31) + 4096, dtype=BF16, device=dev)
    q = buf.as_strided((1, 2, 1, d), (0, 1 << 31, d, 1))
    k = torch.randn(1, 2, 1, d, device=dev).to(BF16)
    q.copy_(torch.randn(1, 2, 1, d, device=dev))
    cos, sin = _tables(dev, 4, d)
    g = torch.ones(1, 2, 1, d, dtype=BF16, device=dev)
    w = torch.ones(d, dtype=BF16, device=dev)
    a, b = (_run(pkg, x, k, cos, sin, 1, w, w, g, g, "half") for x in (q, q.contiguous()))
    assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[1][0], b[1][0])


def test_positions_outside_the_tables(pkg, dev):
    q, k, wq, wk, gq, gk = _inputs(dev, 1, 6, 3, 2, 64, F32)
    cos, sin = _tables(dev, 10, 32)
    pos = torch.tensor([0, -1, 9, 10, 1 << 40, 5], device=dev)
    outs, grads = _run(pkg, q, k, cos, sin, pos, None, None, gq, gk, "half")
    good = torch.tensor([True, False, True, False, False, True], device=dev)
    fine, gfine = _run(pkg, q, k, cos, sin, torch.where(good, pos, 0), None, None, gq, gk, "half")
    for o, f in zip((*outs, *grads), (*fine, *gfine)):
        assert torch.isnan(o[:, ~good]).all() and torch.equal(o[:, good], f[:, good])
    zero = torch.zeros_like(q)  # rows of zeros: eps decides
    out, _ = pkg.qk_norm_rope(zero, k, cos, sin, 0, wq, wk)
    assert bool((out == 0).all())


def test_empty(pkg, dev):
    cos, sin = _tables(dev, 4, 64)
    w = torch.ones(64, device=dev, requires_grad=True)
    for shape in ((0, 5), (2, 0)):
        q, k = (torch.zeros(*shape, h, 64, device=dev, requires_grad=True) for h in (4, 2))
        a, b = pkg.qk_norm_rope(q, k, cos, sin, None if shape[1] <= 4 else torch.zeros(shape[1], dtype=torch.int64, device=dev), w, w)
        assert a.shape == q.shape and b.shape == k.shape
        g = torch.autograd.grad((a.sum() + b.sum()), [q, w])
        assert g[0].shape == q.shape and bool((g[1] == 0).all())


def test_captured_and_streams(pkg, dev):
    sets = [_inputs(dev, 2, 40, 8, 2, 128, BF16, seed=s) for s in range(3)]
    cos, sin = _tables(dev, 64, 128)
    want = [_run(pkg, s[0], s[1], cos, sin, None, *s[2:], "half") for s in sets]
    state = [x.clone() for x in sets[0]]
    pos = torch.arange(40, device=dev)
    leaves = [x.requires_grad_() for x in state[:4]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(pkg.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3]), leaves, state[4:])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = pkg.qk_norm_rope(leaves[0], leaves[1], cos, sin, pos, leaves[2], leaves[3])
        grads = torch.autograd.grad(outs, leaves, state[4:])
    for _ in range(2):
        for s, (wo, wg) in zip(sets, want):
            with torch.no_grad():
                for dst, src in zip(state, s):
                    dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((*outs, *grads), (*wo, *wg)))


def test_scaled_tables(pkg, dev):
    """Tables for long contexts: closed forms, and the rotation by them."""
    base_c, base_s = pkg.rope_tables(10000.0, 64, 256)
    c, s = pkg.rope_tables(10000.0, 64, 256, scaling={"type": "linear", "factor": 4.0})
    assert torch.equal(c[::4], base_c[:64]) and torch.equal(s[::4], base_s[:64])
    q, k, wq, wk, _, _ = _inputs(dev, 1, 8, 2, 1, 64, F32)
    a = pkg.qk_norm_rope(q, k, c.to(dev), s.to(dev), 4 * torch.arange(8, device=dev), wq, wk)
    b = pkg.qk_norm_rope(q, k, base_c.to(dev), base_s.to(dev), None, wq, wk)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals(pkg, dev):
    q, k, wq, wk, _, _ = _inputs(dev, 2, 5, 4, 2, 64, BF16)
    cos, sin = _tables(dev, 16, 64)
    call = pkg.qk_norm_rope
    for match, err, args, kw in (
            ("layout", ValueError, (q, k, cos, sin), dict(layout="quarters")),
            ("must be \\[batch", RuntimeError, (q[0, 0], k[0, 0], cos, sin), {}),
            ("one type", RuntimeError, (q, k.float(), cos, sin), {}),
            ("one type", RuntimeError, (q.double(), k.double(), cos, sin), {}),
            ("HIP device", RuntimeError, (q.cpu(), k.cpu(), cos.cpu(), sin.cpu()), {}),
            ("different devices", RuntimeError, (q, k, cos.cpu(), sin), {}),
            ("agree", RuntimeError, (q, k[:, :4], cos, sin), {}),
            ("agree", RuntimeError, (q, k[..., :32], cos, sin), {}),
            ("head_dim", ValueError, (q[..., :63], k[..., :63], cos, sin), {}),
            ("cos and sin", RuntimeError, (q, k, cos, sin[:8]), {}),
            ("cos and sin", RuntimeError, (q, k, cos.double(), sin.double()), {}),
            ("cos and sin", RuntimeError, (q[..., :32], k[..., :32], cos, sin), {}),
            ("norm weights", RuntimeError, (q, k, cos, sin, None, wq[:32]), {}),
            ("positions must be", RuntimeError, (q, k, cos, sin, torch.zeros(5, device=dev)), {}),
            ("positions must be", RuntimeError, (q, k, cos, sin, torch.zeros(4, dtype=torch.int64, device=dev)), {}),
            ("leave tables", ValueError, (q, k, cos, sin, 12), {}),
            ("leave tables", ValueError, (q, k, cos, sin, -1), {})):
        with pytest.raises(err, match=match):
            call(*args, **kw)

def _negated_view(t):
    """t's values as a lazily negated, strided view (what .imag of a conjugate is)."""
    return torch.complex(torch.zeros_like(t), -t).conj().imag


def _otherwise(form):
    """An unpack hook that gives float32 tensors back as negated views, or matrices with their last dimensions in other
    memory order."""
    if form == "negated":
        return lambda t: _negated_view(t) if t.dtype == torch.float32 else t
    return lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() >= 2 else t


@pytest.mark.parametrize("form", ["negated", "columns"])
def test_saved_tensor_hooks_may_change_the_form(pkg, dev, form):
    """The same values in other memory, so the same bits."""
    q, k, wq, wk, gq, gk = _inputs(dev, 2, 5, 3, 1, 64, F32)
    (cos, sin), pos = _tables(dev, 64, 32), torch.arange(3, 8, device=dev)
    ins = [x.detach().requires_grad_(True) for x in (q, k, wq, wk)]

    def grads():
        out = pkg.qk_norm_rope(ins[0], ins[1], cos, sin, pos, ins[2], ins[3])
        return lambda: torch.autograd.grad(out, ins, (gq, gk))

    want = grads()()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _otherwise(form)):
        got = grads()
    for x, y in zip(got(), want):
        assert torch.equal(x, y)
