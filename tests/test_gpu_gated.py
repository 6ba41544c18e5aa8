"""The gated feed-forward product (gated_bitlinear, GatedBitLinear) and its gradients against float64.

Bounds, from the arithmetic.  Forward: the sums are exact; gate and up take two fp32 roundings each, relu squared three
more: 8 roundings of 2^-24 in all, and half a step of the result's type.  silu: exp's argument is off by 4 roundings
relative to |g|, so exp by 4 |g|, its polynomial and scaling by 8, and the rest as above: (4 |g| + 16) 2^-24.
Gradients: a term of a product is off by 2^-12 (one fp16 plane, bf16 results) or 2^-23 (two planes) and by the few
roundings of d; the sum over C terms adds at most sqrt(C / 8) roundings of 2^-24; half a step of the result's type comes on
top: 2^-12 + 2^-9 in bf16, 2e-6 in fp32, 2^-11 in fp16.  The terms' errors are independent, so the error of sum_c A_c B_c
has the size u sqrt(sum_c (A_c B_c)^2), whatever the terms cancel to: bounds are relative to that root (for a whole result of
random terms it is the result's own size), over the whole, and three times that over every row and column: the largest of
a few thousand sums of independent errors, each of a spread below the bound by sqrt(3) as errors are spread evenly."""

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
GRAD_BOUND = {F32: 2e-6, BF16: 2.0 ** -12 + 2.0 ** -9, F16: 2e-6 + 2.0 ** -11}


def _case(dev, m, k, f, dtype, wdtype, seed=0, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + 31 * m + 7 * k + f)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    x = (rand(m, k) * (1 + rand(m, 1).abs())).to(dtype)
    return x, (rand(f, k) * 0.05).to(wdtype), (rand(f, k) * 0.03).to(wdtype), (rand(m, f) * scale).to(dtype)


def _exact(pkg, x, gate, up, act, gh=None):
    """(h, gate, (grad_x, root), (grad_gate, root), (grad_up, root)) in float64 from the packs' and the quantiser's own
    codes, with each sum's root of its squared terms."""
    ops = pkg.ops
    k = x.shape[1]
    mats = []
    for w in (gate, up):
        qw, s = ops.pack_ternary_i2s(w, k_pad=(k + 127) // 128 * 128)
        mats.append((ops.unpack_i2s(qw)[:, :k].double(), float(s)))
    q, a = ops.quantize_activations_i8_per_token(x)
    held = q.double() * a.double()[:, None]
    yg, yu = (held @ t.t() * s for t, s in mats)
    if act == "silu":
        sig = torch.sigmoid(yg)
        z, slope = yg * sig, sig * (1 + yg * (1 - sig))
    else:
        z, slope = yg.clamp(min=0) ** 2, 2 * yg.clamp(min=0)
    if gh is None:
        return z * yu, yg
    d = [gh.double() * yu * slope, gh.double() * z]
    gx = sum((di * s) @ t for di, (t, s) in zip(d, mats))
    rx = sum((di * s).square() @ t.square() for di, (t, s) in zip(d, mats)).sqrt()
    out = [(z * yu), yg, (gx, rx)]
    for di in d:
        dt = di.t().contiguous()
        out.append((dt @ held, (dt.square() @ held.square()).sqrt()))
    return out


def _near(got, ref, bound, what):
    """Normwise over the whole, and over every row and column."""
    value, root = ref
    d = got.double() - value
    assert torch.isfinite(got).all(), what
    size = value.abs().maximum(root)
    assert float(d.norm()) <= bound * float(size.norm()), (what, float(d.norm() / size.norm()))
    for dim in (0, 1):
        off, s = d.norm(dim=dim), size.norm(dim=dim)
        # below its normal numbers a type's half step is constant, tiny * eps / 2 (2^-25 in fp16): sqrt(n) of them in a norm
        least = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps / 2 * ref[0].shape[dim] ** 0.5
        assert bool((off <= 3 * bound * s + least).all()), (what, dim, float((off / s).max()))


def _run(pkg, x, gate, up, gh, act, packed=None):
    leaves = [t.detach().clone().requires_grad_() for t in (x, gate, up)]
    h = pkg.gated_bitlinear(*leaves, act=act, packed=packed)
    return (h.detach(), *torch.autograd.grad(h, leaves, gh))


SIZES = [(1, 64, 1), (1, 128, 33), (2, 576, 1536), (3, 2560, 97), (17, 65, 640), (63, 129, 130), (65, 1000, 65),
         (100, 4096, 200), (129, 200, 4097), (257, 384, 256), (300, 577, 1001), (1025, 128, 64)]


@pytest.mark.parametrize("act", ["silu", "relu2"])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_forward_and_gradients(pkg, dev, m, k, f, dtype, wdtype, act):
    x, gate, up, gh = _case(dev, m, k, f, dtype, wdtype)
    h, gx, gg, gu = _run(pkg, x, gate, up, gh, act)
    rh, yg, rx, rg, ru = _exact(pkg, x, gate, up, act, gh)
    roundings = 4 * yg.abs() + 16 if act == "silu" else 8
    assert bool(((h.double() - rh).abs() <= rh.abs() * (roundings * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * 1.001
                 + torch.finfo(dtype).tiny).all())
    assert gx.dtype == dtype and gg.dtype == wdtype and gu.dtype == wdtype
    _near(gx, rx, GRAD_BOUND[dtype], "grad_x")
    _near(gg, rg, GRAD_BOUND[wdtype], "grad_gate")
    _near(gu, ru, GRAD_BOUND[wdtype], "grad_up")
    with torch.no_grad():  # served: the same values, from the pack alone too
        assert torch.equal(pkg.gated_bitlinear(x, gate, up, act=act), h)
        assert torch.equal(pkg.gated_bitlinear(x, act=act, packed=pkg.pack_gated(gate, up)), h)


@pytest.mark.parametrize("m,k,f", [(2000, 640, 1536), (700, 2560, 6912), (4096, 576, 1536), (37, 4096, 14336)])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16)])
def test_large_forms(pkg, dev, m, k, f, dtype, wdtype):
    """Sizes at which the products take their larger tiles, whole and in parts."""
    x, gate, up, gh = _case(dev, m, k, f, dtype, wdtype)
    h, gx, gg, gu = _run(pkg, x, gate, up, gh, "silu")
    rh, yg, rx, rg, ru = _exact(pkg, x, gate, up, "silu", gh)
    assert bool(((h.double() - rh).abs() <= rh.abs() * ((4 * yg.abs() + 16) * 2.0 ** -24 + torch.finfo(dtype).eps / 2)
                 * 1.001 + torch.finfo(dtype).tiny).all())
    _near(gx, rx, GRAD_BOUND[dtype], "grad_x")
    _near(gg, rg, GRAD_BOUND[wdtype], "grad_gate")
    _near(gu, ru, GRAD_BOUND[wdtype], "grad_up")


@pytest.mark.parametrize("act", ["silu", "relu2"])
def test_same_values_as_the_decode_product(pkg, dev, act):
    x, gate, up, _ = _case(dev, 9, 640, 96, F32, F32)
    packed = pkg.pack_gated(gate, up)
    for w, first in ((gate, 0), (up, 96)):
        qw, s = pkg.pack_ternary_i2s(w)
        assert torch.equal(packed.qweight[first:first + 96], qw) and float(packed.scales[first // 96]) == float(s)
    q, a = pkg.quantize_activations_i8_per_token(x)
    ref = pkg.bitnet_linear_glu(packed.qweight, packed.scales, q, act=act, a_scale=a, mid_dtype=F32)
    assert torch.equal(pkg.gated_bitlinear(x, act=act, packed=packed), ref)


def test_gradient_against_differences(pkg, dev):
    """The straight-through gradient is that of the product at the quantised operands: central differences in float64."""
    x, gate, up, gh = _case(dev, 40, 256, 192, F32, F32)
    _, gx, gg, gu = _run(pkg, x, gate, up, gh, "silu")
    ops = pkg.ops
    held = [ops.unpack_i2s(q).double() * float(s) for q, s in (ops.pack_ternary_i2s(w) for w in (gate, up))]
    q, a = ops.quantize_activations_i8_per_token(x)
    held.insert(0, q.double() * a.double()[:, None])

    def loss(xs, gs, us):
        y = xs @ gs.t()
        return float((y * torch.sigmoid(y) * (xs @ us.t()) * gh.double()).sum())

    g = torch.Generator(device=dev).manual_seed(5)
    for i, grad in enumerate((gx, gg, gu)):
        v = torch.randn(held[i].shape, generator=g, device=dev).double()
        step = 1e-5 * held[i].norm() / v.norm()
        ends = [loss(*[t + sign * step * v if j == i else t for j, t in enumerate(held)]) for sign in (1, -1)]
        slope, want = (ends[0] - ends[1]) / (2 * float(step)), float((grad.double() * v).sum())
        # truncation ~ step^2, 1e-10 relative; the gradient's own error 2e-6 of |grad| |v|
        assert abs(slope - want) <= 4e-6 * float(grad.double().norm() * v.norm())


def test_rows_of_any_size(pkg, dev):
    """Every row of d has a scale of its own: gradients of tokens 2^60 apart are each as exact."""
    x, gate, up, gh = _case(dev, 70, 256, 130, F32, F32)
    gh = gh * torch.exp2(torch.arange(70, device=dev, dtype=F32)[:, None] * 3 - 100)
    gh[7] = 0.0
    h, gx, gg, gu = _run(pkg, x, gate, up, gh, "silu")
    _, _, rx, rg, ru = _exact(pkg, x, gate, up, "silu", gh)
    off = (gx.double() - rx[0]).norm(dim=1)
    assert bool((off <= 3 * GRAD_BOUND[F32] * rx[1].norm(dim=1)).all()) and bool((gx[7] == 0).all())
    assert float((gg.double() - rg[0]).norm() / rg[0].norm()) <= GRAD_BOUND[F32]
    assert float((gu.double() - ru[0]).norm() / ru[0].norm()) <= GRAD_BOUND[F32]


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_bad_gradient_stays_in_its_row(pkg, dev, bad, dtype):
    x, gate, up, gh = _case(dev, 66, 256, 130, dtype, dtype)
    clean = _run(pkg, x, gate, up, gh, "silu")
    gh[5, 77] = bad
    h, gx, gg, gu = _run(pkg, x, gate, up, gh, "silu")
    rows = torch.arange(66, device=dev) != 5
    cols = torch.arange(130, device=dev) != 77
    assert not torch.isfinite(gx[5]).any() and torch.equal(gx[rows], clean[1][rows])
    for got, was in ((gg, clean[2]), (gu, clean[3])):
        assert torch.equal(got[cols], was[cols]) and not torch.isfinite(got[77]).all()


def test_zero_and_empty(pkg, dev):
    x, gate, up, gh = _case(dev, 5, 128, 64, BF16, F32)
    for g in _run(pkg, x, gate, up, torch.zeros_like(gh), "relu2")[1:]:
        assert bool((g == 0).all())
    h, gx, gg, gu = _run(pkg, x[:0], gate, up, gh[:0], "silu")
    assert h.shape == (0, 64) and gx.shape == (0, 128) and bool((gg == 0).all()) and bool((gu == 0).all())


def test_wanted_gradients_only(pkg, dev):
    x, gate, up, gh = _case(dev, 33, 320, 96, BF16, F32)
    full = _run(pkg, x, gate, up, gh, "silu")
    for want in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().clone().requires_grad_(i in want) for i, t in enumerate((x, gate, up))]
        h = pkg.gated_bitlinear(*leaves, act="silu")
        got = torch.autograd.grad(h, [leaves[i] for i in want], gh)
        for i, g in zip(want, got):
            assert torch.equal(g, full[1 + i])


def test_strides_and_leading_dimensions(pkg, dev):
    x, gate, up, gh = _case(dev, 24, 200, 72, BF16, BF16)
    full = _run(pkg, x, gate, up, gh, "silu")
    wide = torch.zeros(24, 400, dtype=BF16, device=dev)
    wide[:, 100:300] = x
    leaves = [t.requires_grad_() for t in (wide[:, 100:300].detach().view(4, 6, 200), gate.clone(), up.clone())]
    h = pkg.gated_bitlinear(*leaves, act="silu")
    assert h.shape == (4, 6, 72) and torch.equal(h.detach().view(24, 72), full[0])
    broad = torch.zeros(24, 145, dtype=BF16, device=dev)  # rows of the gradient that start at odd elements
    broad[:, 73:] = gh
    got = torch.autograd.grad(h, leaves, broad[:, 73:].view(4, 6, 72) if broad[:, 73:].is_contiguous() else
                              broad[:, 73:].unflatten(0, (4, 6)), retain_graph=True)
    assert torch.equal(got[0].reshape(24, 200), full[1]) and torch.equal(got[1], full[2]) and torch.equal(got[2], full[3])
    h.sum().backward()  # a broadcast gradient
    ones = _run(pkg, x, gate, up, torch.ones_like(gh), "silu")
    assert torch.equal(leaves[0].grad.reshape(24, 200), ones[1]) and torch.equal(leaves[2].grad, ones[3])


def test_lazily_negated_operands(pkg, dev):
    x, gate, up, gh = _case(dev, 12, 200, 72, F32, F32)
    want = _run(pkg, -x, -gate, up, -gh, "silu")
    neg = torch._neg_view
    leaves = [neg(x).requires_grad_(), neg(gate).requires_grad_(), up.clone().requires_grad_()]
    h = pkg.gated_bitlinear(*leaves, act="silu")
    got = torch.autograd.grad(h, leaves, neg(gh))
    assert torch.equal(h.detach(), want[0])
    assert all(torch.equal(g.resolve_neg(), w) for g, w in zip(got, want[1:]))


def test_another_stream_and_two_at_once(pkg, dev):
    a, b = (_case(dev, 200, 384, 320, BF16, F32, seed=s) for s in (1, 2))
    want = [_run(pkg, *c, "silu") for c in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s, c in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            got.append(_run(pkg, *c, "silu"))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, g))


def test_captured_and_replayed(pkg, dev):
    cases = [_case(dev, 130, 256, 192, BF16, F32, seed=s) for s in range(3)]
    want = [_run(pkg, *c, "silu") for c in cases]
    x, gate, up, gh = (t.clone() for t in cases[0])
    leaves = [t.requires_grad_() for t in (x, gate, up)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(pkg.gated_bitlinear(*leaves, act="silu"), leaves, gh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = pkg.gated_bitlinear(*leaves, act="silu")
        out = (h, *torch.autograd.grad(h, leaves, gh))
    for _ in range(2):
        for c, w in zip(cases, want):
            with torch.no_grad():
                for t, v in zip((x, gate, up, gh), c):
                    t.copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_module(pkg, dev):
    torch.manual_seed(0)
    mod = pkg.GatedBitLinear(200, 96, act="relu2", device=dev)
    assert set(mod.state_dict()) == {"gate_proj.weight", "up_proj.weight"}
    x = torch.randn(7, 200, device=dev)
    first = mod(x)
    assert torch.equal(first, pkg.gated_bitlinear(x, mod.gate_proj.weight, mod.up_proj.weight, act="relu2"))
    pack = mod.packed()
    assert mod.packed() is pack
    with torch.no_grad():
        mod.up_proj.weight.mul_(-1.0)
    assert torch.equal(mod(x), -first) and mod.packed() is not pack
    assert mod.pack() is mod and mod.packed() is not pack and torch.equal(mod(x), -first)
    twin = copy.deepcopy(mod)
    assert torch.equal(twin(x), -first)
    lin = [torch.nn.Linear(200, 96, bias=False, device=dev) for _ in range(2)]
    made = pkg.GatedBitLinear.from_linears(*lin, act="silu")
    made(x).sum().backward()
    assert lin[0].weight.grad is not None and made.gate_proj.weight is lin[0].weight
    made = pkg.GatedBitLinear.from_linears(pkg.BitLinear(200, 96, device=dev), pkg.BitLinear(200, 96, device=dev))
    assert made(x).shape == (7, 96)
    pkg.set_lambda_source(lambda: 0.5)
    try:
        with pytest.raises(RuntimeError, match="lambda"):
            mod(x)
    finally:
        pkg.set_lambda_source(None)


def test_refusals(pkg, dev):
    x, gate, up, gh = _case(dev, 4, 128, 64, BF16, F32)
    call = pkg.gated_bitlinear
    with pytest.raises(ValueError, match="act"):
        call(x, gate, up, act="gelu")
    with pytest.raises(RuntimeError, match="go together"):
        call(x, gate)
    with pytest.raises(RuntimeError, match="needed"):
        call(x)
    with pytest.raises(RuntimeError, match="one shape and type"):
        call(x, gate, up[:32])
    with pytest.raises(RuntimeError, match="one shape and type"):
        call(x, gate, up.to(BF16))
    with pytest.raises(RuntimeError, match="features"):
        call(x[:, :100], gate, up)
    with pytest.raises(RuntimeError, match="x must be"):
        call(x.double(), gate, up)
    with pytest.raises(RuntimeError, match="HIP device"):
        call(x.cpu(), gate.cpu(), up.cpu())
    with pytest.raises(RuntimeError, match="must be on"):
        call(x, gate.cpu(), up.cpu())
    packed = pkg.pack_gated(gate, up)
    with pytest.raises(RuntimeError, match="packed rows"):
        call(torch.cat([x, x], 1), packed=packed)
    with pytest.raises(RuntimeError, match="packed must be"):
        call(x, packed=pkg.PackedGated(packed.qweight[:63], packed.scales))
    with pytest.raises(RuntimeError, match="hidden features"):
        call(x, gate[:32], up[:32], packed=packed)
    with pytest.raises(RuntimeError, match="no float weights"):
        call(x.clone().requires_grad_(), packed=packed)
    leaf, g2 = x.float().requires_grad_(), gh.float().requires_grad_()
    (gx,) = torch.autograd.grad(call(leaf, gate, up), [leaf], g2, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()

def _negated_view(t):
    """t's values as a lazily negated, strided view (what .imag of a conjugate is)."""
    return torch.complex(torch.zeros_like(t), -t).conj().imag


def _otherwise(form):
    """An unpack hook that gives float32 tensors back as negated views, or matrices with their last dimensions in other
    memory order."""
    if form == "negated":
        return lambda t: _negated_view(t) if t.dtype == torch.float32 else t
    return lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() >= 2 else t


@pytest.mark.parametrize("m", [1, 7])
@pytest.mark.parametrize("form", ["negated", "columns"])
def test_saved_tensor_hooks_may_change_the_form(pkg, dev, form, m):
    """The same values in other memory, so the same bits (a single token's scale counts as contiguous in any view)."""
    x = torch.randn(m, 200, device=dev, requires_grad=True)
    g, u = (torch.randn(96, 200, device=dev, requires_grad=True) for _ in range(2))
    gh = torch.randn(m, 96, device=dev)
    want = torch.autograd.grad(pkg.gated_bitlinear(x, g, u), (x, g, u), gh)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _otherwise(form)):
        h = pkg.gated_bitlinear(x, g, u)
    for a, b in zip(torch.autograd.grad(h, (x, g, u), gh), want):
        assert torch.equal(a, b)
