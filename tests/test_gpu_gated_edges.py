"""The gated product and its gradients in the forms that only large calls take, with remainders in every dimension, against
float64.

Bounds: forward, the sums are exact; gate and up take two fp32 roundings each, relu squared three more: 8 of 2^-24, silu
4 |g| + 16, and half a step of the result's type.  Gradients: a term is off by 2^-12 (bf16 results: one fp16 plane) or 2^-23 (two planes) and
by the few roundings of d, their sum by at most sqrt(C / 8) of 2^-24, and half a step of the result's type: relative to the
root of the sum's squared terms, over the whole and three times that over every row and column."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
GRAD_BOUND = {F32: 2e-6, BF16: 2.0 ** -12 + 2.0 ** -9, F16: 2e-6 + 2.0 ** -11}


def _case(dev, m, k, f, dtype, wdtype):
    g = torch.Generator(device=dev).manual_seed(31 * m + 7 * k + f)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    x = (rand(m, k) * (1 + rand(m, 1).abs())).to(dtype)
    return x, (rand(f, k) * 0.05).to(wdtype), (rand(f, k) * 0.03).to(wdtype), rand(m, f).to(dtype)


def _exact(pkg, x, gate, up, act, gh):
    """(h, gate, (grad_x, root), (grad_gate, root), (grad_up, root)) in float64 from the packs' and the quantiser's own codes."""
    k = x.shape[1]
    mats = []
    for w in (gate, up):
        qw, s = pkg.pack_ternary_i2s(w, k_pad=(k + 127) // 128 * 128)
        mats.append((pkg.unpack_i2s(qw)[:, :k].double(), float(s)))
    q, a = pkg.quantize_activations_i8_per_token(x)
    held = q.double() * a.double()[:, None]
    yg, yu = (held @ t.t() * s for t, s in mats)
    if act == "silu":
        sig = torch.sigmoid(yg)
        z, slope = yg * sig, sig * (1 + yg * (1 - sig))
    else:
        z, slope = yg.clamp(min=0) ** 2, 2 * yg.clamp(min=0)
    d = [gh.double() * yu * slope, gh.double() * z]
    gx = sum((di * s) @ t for di, (t, s) in zip(d, mats))
    rx = sum((di * s).square() @ t.square() for di, (t, s) in zip(d, mats)).sqrt()
    out = [z * yu, yg, (gx, rx)]
    for di in d:
        dt = di.t().contiguous()
        out.append((dt @ held, (dt.square() @ held.square()).sqrt()))
    return out


def _near(got, ref, bound, what):
    value, root = ref
    d = got.double() - value
    assert torch.isfinite(got).all(), what
    size = value.abs().maximum(root)
    assert float(d.norm()) <= bound * float(size.norm()), (what, float(d.norm() / size.norm()))
    for dim in (0, 1):
        off, s = d.norm(dim=dim), size.norm(dim=dim)
        # below its normal numbers a type's half step is constant, tiny * eps / 2: sqrt(n) of them in a norm
        least = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps / 2 * value.shape[dim] ** 0.5
        assert bool((off <= 3 * bound * s + least).all()), (what, dim, float((off / s).max()))


def _run(pkg, x, gate, up, gh, act):
    leaves = [t.detach().clone().requires_grad_() for t in (x, gate, up)]
    h = pkg.gated_bitlinear(*leaves, act=act)
    return (h.detach(), *torch.autograd.grad(h, leaves, gh))


# The forward takes its tiles of 128 tokens in each (from 400 of them): one token and two columns past whole tiles, so that no
# row of the output starts aligned; four columns past them; and the gradients' products take their tiles of 128 x 128 in one
# plane (grad_x of the fourth, the weights' of the second), 128 x 256 in two (grad_x of the third) and the ring of 256 x 256 in two
# planes with a part of a tile's columns (the weights' of the second and the third)
@pytest.mark.parametrize("m,k,f", [(2433, 200, 2690), (2500, 640, 2564), (1099, 194, 19764), (4100, 300, 2180)])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("act", ["silu", "relu2"])
def test_forms_of_large_calls(pkg, dev, m, k, f, dtype, wdtype, act):
    x, gate, up, gh = _case(dev, m, k, f, dtype, wdtype)
    if dtype == F16:
        gh = gh * 2.0 ** -10  # (weight gradients within fp16's range)
    h, gx, gg, gu = _run(pkg, x, gate, up, gh, act)
    rh, yg, rx, rg, ru = _exact(pkg, x, gate, up, act, gh)
    roundings = 4 * yg.abs() + 16 if act == "silu" else 8
    assert bool(((h.double() - rh).abs() <= rh.abs() * (roundings * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * 1.001
                 + torch.finfo(dtype).tiny).all())
    _near(gx, rx, GRAD_BOUND[dtype], "grad_x")
    _near(gg, rg, GRAD_BOUND[wdtype], "grad_gate")
    _near(gu, ru, GRAD_BOUND[wdtype], "grad_up")
    with torch.no_grad():
        packed = pkg.pack_gated(gate, up)
        assert torch.equal(pkg.gated_bitlinear(x, act=act, packed=packed), h)
        # the same operations on the same integers in every form: the few-token forms' bits
        for first in (0, 1000, m - 40):
            assert torch.equal(pkg.gated_bitlinear(x[first:first + 40], act=act, packed=packed), h[first:first + 40])
        assert torch.equal(pkg.gated_bitlinear(x[-5:], act=act, packed=packed), h[-5:])


def test_slopes_of_large_gates(pkg, dev):
    """One token, gates from -40 to 40: a weight's gradient is one product d code a, so d itself shows.

    Roundings of 2^-24: exp(-g) 4 (the exponential's ulp counts 2), 1 + exp one, the reciprocal's ulp 2: s has 7, a = g s 8,
    exp(-g) s 12, slope = s + a (exp(-g) s): 7 s + 21 |a exp(-g) s|, and one of the sum.  gh up, its product with the slope, the
    scale of the token, two planes (2), a code's product and the result's rounding: 7 more.  The products kept by the forward have 2
    each (gate's move the slope by 2 |g| |slope'|, up's count as 2)."""
    n = torch.arange(-128, 128, device=dev)
    cols = torch.arange(128, device=dev)
    gate = ((cols[None] < n[:, None].abs()).float() * n[:, None].sign())
    up = torch.ones(256, 128, device=dev)
    w = gate.abs().mean()
    x = torch.full((1, 128), 40.0 / 128.0, device=dev) / w
    gh = torch.randn(1, 256, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    _, gx, gg, gu = _run(pkg, x, gate, up, gh, "silu")
    q, a = pkg.quantize_activations_i8_per_token(x)
    held = float(q[0, 0]) * float(a)
    g = (n.double() * held * float(pkg.pack_gated(gate, up).scales[0]))
    u = 128.0 * held * float(pkg.pack_gated(gate, up).scales[1])
    s = torch.sigmoid(g)
    # (1 - s written so that it keeps its digits)
    rest = torch.sigmoid(-g)
    slope, bend = s * (1 + g * rest), (s * rest * (2 + g * (rest - s))).abs()
    dg, du = gh[0].double() * u * slope, gh[0].double() * g * s
    size = gh[0].double().abs() * u * held
    lim = 2.0 ** -24 * size * (7 * s + 21 * (g * s * rest).abs() + (1 + 7 + 2) * slope.abs() + 2 * g.abs() * bend)
    off = (gg.double() - (dg * held)[:, None]).abs()
    assert float(n.abs().max()) * held * float(pkg.pack_gated(gate, up).scales[0]) > 39.0
    assert bool((off <= 1.001 * lim[:, None]).all()), float((off / lim[:, None]).max())
    # d_up = gh (g s): 8 and the same 6 behind it, 2 of the gate through (g s)'
    lim = 2.0 ** -24 * gh[0].double().abs() * held * ((8 + 6) * (g * s).abs() + 2 * g.abs() * slope.abs())
    off = (gu.double() - (du * held)[:, None]).abs()
    assert bool((off <= 1.001 * lim[:, None]).all()), float((off / lim[:, None].clamp(min=1e-300)).max())


@pytest.mark.parametrize("scale", [90.0, 130.0, 1e4, 3e7, 1e12, 1e18])
def test_gates_of_any_size(pkg, dev, scale):
    """Gates of +- scale: silu's slope is 1 and its value the gate, or both are next to nothing (88 e^-88 of up, below 1e-36)."""
    gate = torch.ones(64, 128, device=dev)
    gate[::2] = -1.0
    up = torch.ones(64, 128, device=dev)
    x = torch.full((2, 128), scale / 128.0, device=dev)
    x[1] = -x[1]
    gh = torch.randn(2, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(2)) * 1e-3
    _, gx, gg, gu = _run(pkg, x, gate, up, gh, "silu")
    q, a = pkg.quantize_activations_i8_per_token(x)
    held = q.double() * a.double()[:, None]
    y = held @ gate.double().t(), held @ up.double().t()
    on = (y[0] > 0).double()
    d = gh.double() * y[1] * on, gh.double() * y[0] * on
    # kept products 2 roundings each, d 8 (slope and value within 8 of 1 and the gate), planes and scales 4, the sum of two tokens
    # or 128 features and the result 3
    for got, ref, size in ((gg, d[0].t() @ held, d[0].abs().t() @ held.abs()), (gu, d[1].t() @ held, d[1].abs().t() @ held.abs()),
                           (gx, d[0] @ gate.double() + d[1] @ up.double(), (d[0].abs() + d[1].abs()) @ up.double())):
        assert torch.isfinite(got).all()
        # (a plane pair holds what is 2^-18 of its row's largest and more to 22 bits, the rest to 2^-40 of it)
        lim = 19 * 2.0 ** -24 * size + 2.0 ** -40 * size.amax(1, keepdim=True) + 1e-36 * scale * scale
        assert bool(((got.double() - ref).abs() <= lim).all())


@pytest.mark.parametrize("m,k,f", [(33, 320, 96), (700, 640, 1536), (2500, 640, 2564)])
@pytest.mark.parametrize("wdtype", [BF16, F32])
def test_wide_gradients(pkg, dev, m, k, f, wdtype):
    """bf16 gradients of operands in 22 bits are the fp32 ones, rounded: the same planes, sums and order."""
    x, gate, up, gh = _case(dev, m, k, f, BF16, wdtype)
    leaves = [t.detach().requires_grad_() for t in (x, gate, up)]
    got = torch.autograd.grad(pkg.gated_bitlinear(*leaves, wide_grads=True), leaves, gh)
    full = _run(pkg, x.float(), gate.float(), up.float(), gh.float(), "silu")[1:]
    for a, b, t in zip(got, full, leaves):
        assert a.dtype == t.dtype and torch.equal(a, b.to(t.dtype))
    mod = pkg.GatedBitLinear.from_linears(*(torch.nn.Linear(k, f, bias=False, device=dev, dtype=wdtype) for _ in range(2)),
                                          wide_grads=True)
    with torch.no_grad():
        mod.gate_proj.weight.copy_(gate)
        mod.up_proj.weight.copy_(up)
    assert torch.equal(torch.autograd.grad(mod(leaves[0]), [leaves[0]], gh)[0], got[0])
