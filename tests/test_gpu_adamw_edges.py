"""AdamW where squares and quotients leave fp32's normal numbers, against IEEE fp32 on the CPU: every operation of a step is one
correctly rounded operation, so the 32-bit results are equal to the bit."""

import math

import numpy
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _plain(p, g, m, v, t, lr, betas, eps, weight_decay):
    """One step in fp32 on the CPU, in place of m and v; the new parameters.  numpy's operations are IEEE's one by one."""
    b1, b2 = betas
    f = numpy.float32
    p, g, mn, vn = (x.numpy() for x in (p, g, m, v))
    with numpy.errstate(all="ignore"):
        mn[:] = mn * f(b1) + g * f(1.0 - b1)
        vn[:] = vn * f(b2) + (g * g) * f(1.0 - b2)
        move = (mn * f(lr / (1.0 - b1 ** t))) / (numpy.sqrt(vn) * f(1.0 / math.sqrt(1.0 - b2 ** t)) + f(eps))
        return torch.from_numpy(p * f(1.0 - lr * weight_decay) - move)


# gradients whose squares overflow, underflow and are subnormal; moments and divisors of every size
@pytest.mark.parametrize("eps", [1e-8, 0.0, 1e-30, 1e30])
@pytest.mark.parametrize("lr", [1e-3, 1e-20])
def test_steps_of_any_size(pkg, dev, eps, lr):
    gen = torch.Generator().manual_seed(7)
    n = 5000
    p = torch.randn(n, generator=gen)
    own, hyper = [p.to(dev)], dict(lr=lr, betas=(0.9, 0.95), eps=eps, weight_decay=0.1)
    state = pkg.adamw_state(own)
    m, v = torch.zeros(n), torch.zeros(n)
    for t in range(1, 4):
        g = torch.randn(n, generator=gen) * torch.exp2(torch.randint(-140, 120, (n,), generator=gen).float())
        g[:50] = 0.0
        p = _plain(p, g, m, v, t, **hyper)
        pkg.adamw_step(own, [g.to(dev)], state, t, **hyper)
        assert torch.equal(state.m[:n].cpu(), m) and torch.equal(state.v[:n].cpu(), v)
        got = own[0].cpu()
        assert torch.equal(got.isnan(), p.isnan()) and torch.equal(got.nan_to_num(nan=0.0), p.nan_to_num(nan=0.0))
        # (zero over zero where eps is 0 is the formula's own NaN)
        assert eps == 0.0 or not p.isnan().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_square_past_fp32_in_8_bits(pkg, dev, dtype):
    gen = torch.Generator(device=dev).manual_seed(3)
    grads = torch.randn(1000, generator=gen, device=dev).to(dtype)
    big = grads.clone()
    big[300] = 1e20
    start = torch.randn(1000, generator=gen, device=dev)
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    a, b = [start.clone()], [start.clone()]
    sa, sb = pkg.adamw_state(a, 8), pkg.adamw_state(b, 8)
    pkg.adamw_step(a, [big], sa, 1, **hyper)
    pkg.adamw_step(b, [grads], sb, 1, **hyper)
    others = torch.arange(1000, device=dev) != 300
    assert torch.equal(a[0][others], b[0][others])
    assert float(a[0][300]) == float(start[300] * torch.tensor(1.0 - 1e-2 * 0.1, device=dev))  # decayed, no more
    block = torch.zeros(1024, dtype=torch.bool, device=dev)
    block[256:512] = True
    assert float(sa.v_scale[1]) == 2.0 ** 63 and int(sa.v[300]) == 255 and int(sa.v[256:300].max()) == 1
    for x, y in zip(pkg.adamw_state_values(sa), pkg.adamw_state_values(sb)):
        assert torch.isfinite(x).all() and torch.equal(x[~block], y[~block])
    for t in range(2, 6):
        before = a[0].clone()
        pkg.adamw_step(a, [grads], sa, t, **hyper)
        pkg.adamw_step(b, [grads], sb, t, **hyper)
        assert torch.equal(a[0][~block[:1000]], b[0][~block[:1000]])
        # the block's moments: m at most 2e19, held to 1 / 127^2 of its largest; r at least 2^63 / 255^2 on its way down
        assert torch.isfinite(a[0]).all()
        assert float((a[0][300] - before[300] * (1.0 - 1e-3)).abs()) <= 1e-2 * 127.0
        assert all(torch.isfinite(x).all() for x in pkg.adamw_state_values(sa))


def test_a_square_that_is_subnormal(pkg, dev):
    """g = 1e-22: v = 5e-46 rounds to a subnormal number or to zero, and the step is the formula's."""
    g = torch.full((512,), 3e-22)
    p, m, v = torch.ones(512), torch.zeros(512), torch.zeros(512)
    hyper = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    own = [p.to(dev)]
    state = pkg.adamw_state(own)
    p = _plain(p, g, m, v, 1, **hyper)
    pkg.adamw_step(own, [g.to(dev)], state, 1, **hyper)
    assert 0.0 < float(v[0]) < torch.finfo(F32).tiny
    assert torch.equal(own[0].cpu(), p) and torch.equal(state.v.cpu(), v)
    eight = pkg.adamw_state(own, 8)
    pkg.adamw_step([torch.ones(512, device=dev)], [g.to(dev)], eight, 1, **hyper)
    assert bool((eight.v == 255).all()) and float(eight.v_scale[0]) == float(v.sqrt()[0])


def test_the_root_of_every_significand(pkg, dev):
    """All 2^24 significands under both parities of the exponent: with m = r, the rounded root of v, the step is r / sqrt(v),
    which is 1 only where the kernel's root is r: one that is an ulp off, a relative 2^-24 at least, gives another quotient
    (an ulp below r a relative step above 2^-24 past 1, an ulp above r a step of 2^-25 at least below it)."""
    v = torch.arange(1 << 24, dtype=torch.int32, device=dev).add_(127 << 23).view(F32)  # [1, 4)
    r = v.double().sqrt().float()  # (53 bits round to 24 as the root itself does)
    p = [torch.zeros(1 << 24, device=dev)]
    # b = 1/2 halves m and v exactly; after 200 steps both corrections are 1
    state = pkg.AdamWState(2.0 * r, 2.0 * v)
    pkg.adamw_step(p, [torch.zeros(1 << 24, device=dev)], state, 200, lr=1.0, betas=(0.5, 0.5), eps=0.0, weight_decay=0.0)
    assert torch.equal(state.v, v) and torch.equal(state.m, r)
    assert bool((p[0] == -1.0).all())


@pytest.mark.parametrize("exponent", [-60, -1, 0, 40])
def test_the_quotient_of_every_divisor(pkg, dev, exponent):
    """Every significand of the divisor under significands of the numerator next to it, at its ends and at random; 64 bits
    round to 24 as the quotient itself does."""
    d = torch.arange(1 << 23, dtype=torch.int32, device=dev).add_(127 << 23).view(F32)  # [1, 2)
    v = d * d
    d = v.double().sqrt().float()
    ulp = 2.0 ** -23
    gen = torch.Generator(device=dev).manual_seed(11)
    tops = [torch.ones_like(d), torch.full_like(d, 2.0 - ulp), (d - ulp).clamp(min=1.0), (d + ulp).clamp(max=2.0 - ulp),
            *(1.0 + torch.randint(1 << 23, d.shape, generator=gen, device=dev).float() * ulp for _ in range(4))]
    for n in tops:
        n = n * 2.0 ** exponent
        p = [torch.zeros_like(d)]
        state = pkg.AdamWState(2.0 * n, 2.0 * v)
        pkg.adamw_step(p, [torch.zeros_like(d)], state, 200, lr=1.0, betas=(0.5, 0.5), eps=0.0, weight_decay=0.0)
        assert torch.equal(p[0], -(n.double() / d.double()).float())
