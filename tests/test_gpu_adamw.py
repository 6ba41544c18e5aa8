"""AdamW over many tensors: its fp32 arithmetic bit for bit against torch's elementary operations, the 8-bit grids against
their definition, and its surfaces.

torch's GPU products, sums, quotients and roots are each correctly rounded, so the moments and the codes have to be equal
bit for bit; a parameter too (its one quotient is correctly rounded on both sides)."""

import copy
import math
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
BLOCK = 256


def _up(n):
    return (n + BLOCK - 1) // BLOCK * BLOCK


def _make(dev, sizes, pdt, gdt, seed=0, offset=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def one(n, scale, dt):
        buf = (torch.randn(n + offset, generator=g, device=dev) * scale).to(dt)
        return buf[offset:]

    return [one(n, 0.1, pdt) for n in sizes], [one(n, 1e-2, gdt) for n in sizes]


class _Plain:
    """The definition with torch's elementary operations in fp32, one tensor at a time."""

    def __init__(self, sizes, bits, dev):
        self.bits = bits
        z = lambda n, dt=F32: torch.zeros(n, dtype=dt, device=dev)  # noqa: E731
        self.first = [sum(_up(n) for n in sizes[:i]) for i in range(len(sizes))]
        self.m, self.v = [z(_up(n)) for n in sizes], [z(_up(n)) for n in sizes]  # v: r in 8 bits
        self.codes = [None] * len(sizes)

    def _grid(self, x, top, z):
        x = x.view(-1, BLOCK)
        big = x.amax(1, keepdim=True)
        big = torch.where(big < 2.0 ** -100, 0.0, big)
        k = torch.full_like(big, float(top * top)) / torch.where(big == 0, 1.0, big)
        q = torch.floor(torch.sqrt(x * k) + z.view(-1, BLOCK)).clamp(max=top)
        return torch.where(big == 0, 0.0, q), big

    def step(self, params, grads, t, lr, betas, eps, weight_decay):
        b1, b2 = betas
        for i, (p, g) in enumerate(zip(params, grads)):
            n = p.numel()
            if g is None or n == 0:
                continue
            gp = torch.zeros_like(self.m[i])
            gp[:n] = g.float().view(-1)
            v = self.v[i] if self.bits == 32 else self.v[i] * self.v[i]
            m = self.m[i] * b1 + gp * (1.0 - b1)
            v = v * b2 + (gp * gp) * (1.0 - b2)
            r = torch.sqrt(v)
            ib2 = 1.0 / math.sqrt(1.0 - b2 ** t)
            new = p.float().view(-1) * (1.0 - lr * weight_decay) - (m[:n] * (lr / (1.0 - b1 ** t))) / (r[:n] * ib2 + eps)
            p.copy_(new.view(p.shape))
            if self.bits == 32:
                self.m[i], self.v[i] = m, v
                continue
            e = torch.arange(m.numel(), dtype=torch.int64, device=p.device) + self.first[i]
            z = (((e * 0x9E3779B1 + t * 0x6A09E667) & 0xFFFFFFFF) >> 8).float() * 2.0 ** -24
            c, a = self._grid(m.abs(), 127, z)
            u, s = self._grid(r, 255, z)
            u = torch.where((r.view(-1, BLOCK) > 0) & (s > 0), u.clamp(min=1), u)
            c = torch.where(m.view(-1, BLOCK) < 0, -c, c)
            self.codes[i] = (c, u, a, s)
            self.m[i] = (c * c.abs() * (a * (1.0 / 16129.0))).view(-1)
            self.v[i] = (u * u * (s * (1.0 / 65025.0))).view(-1)


SIZES = [1, 2, 255, 256, 257, 0, 4095, 4096, 4097, 100, 70000, 3]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdt,gdt", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F32), (F16, F16), (BF16, F32)])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_steps_bit_for_bit(pkg, dev, bits, pdt, gdt, offset):
    params, _ = _make(dev, SIZES, pdt, gdt, offset=offset)
    twins = [p.clone() for p in params]
    state, plain = pkg.adamw_state(params, bits), _Plain(SIZES, bits, dev)
    for t in range(1, 5):
        _, grads = _make(dev, SIZES, pdt, gdt, seed=t, offset=offset)
        grads[4] = grads[4] * 1e-4  # some blocks of another size than the rest
        pkg.adamw_step(params, grads, state, t, **HYPER)
        plain.step(twins, grads, t, **HYPER)
        m, v = pkg.adamw_state_values(state)
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
        assert torch.equal(m, torch.cat(plain.m))
        assert torch.equal(v, torch.cat([x if bits == 32 else x * x for x in plain.v]))
        if bits == 8:
            codes = [c for c in plain.codes if c is not None]
            assert torch.equal(state.m.float(), torch.cat([c[0].view(-1) for c in codes]))
            assert torch.equal(state.v.float(), torch.cat([c[1].view(-1) for c in codes]))


def test_many_tensors_and_missing_gradients(pkg, dev):
    sizes = [1 + 37 * i % 1000 for i in range(200)]
    params, grads = _make(dev, sizes, F32, F32)
    grads = [None if i % 7 == 3 else g for i, g in enumerate(grads)]
    grads[11], params[20] = grads[11].to(BF16), params[20].to(BF16)  # types mixed in one call
    twins = [p.clone() for p in params]
    state, plain = pkg.adamw_state(params), _Plain(sizes, 32, dev)
    pkg.adamw_step(params, grads, state, 1, **HYPER)
    plain.step(twins, grads, 1, **HYPER)
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert torch.equal(state.m, torch.cat(plain.m)) and torch.equal(state.v, torch.cat(plain.v))


def test_against_torch_optimizer(pkg, dev):
    """The same steps as torch.optim.AdamW, whose operations are ordered otherwise: a step differs by a few roundings of
    its own size, 10 steps of at most lr by 10 * 8 * 2^-24 lr and 10 roundings of the parameter."""
    torch.manual_seed(0)
    a = [torch.nn.Parameter(torch.randn(s, device=dev)) for s in ((64, 33), (5,), (1000,))]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ours = pkg.AdamW([{"params": a[:2]}, {"params": a[2:], "lr": 1e-2, "weight_decay": 0.0}], lr=1e-3)
    theirs = torch.optim.AdamW([{"params": b[:2]}, {"params": b[2:], "lr": 1e-2, "weight_decay": 0.0}], lr=1e-3)
    for t in range(10):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, device=dev)
            q.grad = p.grad.clone()
        ours.step()
        theirs.step()
    for p, q in zip(a, b):
        assert float((p - q).abs().max()) <= 10 * (8 * 1e-2 + float(q.detach().abs().max())) * 2.0 ** -24


def test_moments_in_8_bits_follow_the_gradients(pkg, dev):
    """Rounding by the Weyl sequence keeps the average: with b2 = 0.999 a moment moves by less than a code's distance in a
    step, and still arrives.  Gradients of one size: r is that size; halved for 3000 steps (b2^3000 = 0.05, r^2 =
    0.25 + 0.75 * 0.05 of the first) the mean over a block is within 2% of it, an element within two codes at u > 100."""
    p = [torch.zeros(2560, device=dev)]
    state = pkg.adamw_state(p, 8)
    g = torch.where(torch.arange(2560, device=dev) % 3 == 0, 1.0, 0.5)
    for t in range(1, 401):
        pkg.adamw_step(p, [g], state, t, lr=0.0, betas=(0.9, 0.99), weight_decay=0.0)
    # one element of every block keeps its size, so the scale stays
    h = torch.where(torch.arange(2560, device=dev) % 256 == 0, g, 0.5 * g)
    for t in range(401, 3401):
        pkg.adamw_step(p, [h], state, t, lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
    m, v = pkg.adamw_state_values(state)
    moved = torch.arange(2560, device=dev) % 256 != 0
    want = g * g * (0.25 + 0.75 * 0.999 ** 3000)
    ratio = (v / want)[moved].double()
    assert abs(float(ratio.mean()) - 1.0) <= 0.02 and float((ratio - 1).abs().max()) <= 0.2
    assert float((m / h - 1).abs()[moved].max()) <= 0.1


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_bad_gradient_stays_in_its_block(pkg, dev, bad):
    for bits in (32, 8):
        params, grads = _make(dev, [1000, 300], F32, F32)
        clean = [p.clone() for p in params]
        st, sc = pkg.adamw_state(params, bits), pkg.adamw_state(params, bits)
        pkg.adamw_step(clean, grads, sc, 1, **HYPER)
        grads[0][300] = bad
        pkg.adamw_step(params, grads, st, 1, **HYPER)
        m, v = pkg.adamw_state_values(st)
        mc, vc = pkg.adamw_state_values(sc)
        hit = torch.zeros(m.numel(), dtype=torch.bool, device=dev)
        hit[300 if bits == 32 else slice(256, 512)] = True
        assert not torch.isfinite(v[hit]).any() and torch.equal(m[~hit], mc[~hit]) and torch.equal(v[~hit], vc[~hit])
        keep = torch.arange(1000, device=dev) != 300
        assert not torch.isfinite(params[0][300]) and torch.equal(params[0][keep], clean[0][keep])
        assert torch.equal(params[1], clean[1])


def test_tiny_and_zero(pkg, dev):
    for bits in (32, 8):
        p = [torch.ones(512, device=dev)]
        st = pkg.adamw_state(p, bits)
        pkg.adamw_step(p, [torch.zeros(512, device=dev)], st, 1, **HYPER)
        assert torch.equal(p[0], torch.full((512,), 1.0, device=dev) * (1.0 - 3e-3 * 0.1))
        assert not st.m.any() and not st.v.any()
        g = torch.full((512,), 1e-35, device=dev)  # r about 1e-36, below 2^-100 in the 8-bit state: held as zeros
        pkg.adamw_step(p, [g], st, 2, **HYPER)
        assert torch.isfinite(p[0]).all()
        if bits == 8:
            assert not st.m.any() and not st.v.any()


def test_offsets_past_32_bits(pkg, dev):
    """A state of more than 2^31 elements behind a tensor of 2^31."""
    n = (1 << 31) + 512
    p = [torch.zeros(n, dtype=BF16, device=dev), torch.ones(300, device=dev)]
    g = [torch.zeros(n, dtype=BF16, device=dev), torch.ones(300, device=dev)]
    g[0][-1] = 1.0
    st = pkg.adamw_state(p, 8)
    pkg.adamw_step(p, g, st, 1, lr=0.5, weight_decay=0.0)
    assert float(p[0][-1]) == -0.5 and not p[0][:1024].any() and not p[0][1 << 31:-1].any()
    assert bool((p[1] == 0.5).all()) and int(st.m[n - 1]) == 127 and not st.m[:4096].any()
    del p, g, st
    torch.cuda.empty_cache()


def test_captured_steps(pkg, dev):
    sizes = [1000, 257]
    params, grads = _make(dev, sizes, F32, F32)
    twins = [p.clone() for p in params]
    st, tw = pkg.adamw_state(params, 8), pkg.adamw_state(params, 8)
    step, lr = torch.zeros(1, dtype=torch.int64, device=dev), torch.full((1,), 1e-2, device=dev)
    kw = dict(betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step.add_(1)
        pkg.adamw_step(params, grads, st, step, lr=lr, **kw)
    for t in range(1, 6):
        fresh = _make(dev, sizes, F32, F32, seed=t)[1]
        rate = 1e-2 / t
        lr.fill_(rate)
        for g, f in zip(grads, fresh):
            g.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        pkg.adamw_step(twins, fresh, tw, t, lr=float(lr), **kw)
        assert all(torch.equal(a, b) for a, b in zip((*params, *st), (*twins, *tw)))


def test_optimizer_surfaces(pkg, dev):
    torch.manual_seed(1)

    def model():
        torch.manual_seed(2)
        return [torch.nn.Parameter(torch.randn(40, 30, device=dev)), torch.nn.Parameter(torch.randn(30, device=dev))]

    def fill(ps, t):
        g = torch.Generator(device=dev).manual_seed(t)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device=dev)

    for bits in (32, 8):
        for capturable in (False, True):
            a = model()
            oa = pkg.AdamW(a, lr=1e-2, state_bits=bits, capturable=capturable)
            assert oa.group_state() is None
            for t in range(3):
                fill(a, t)
                oa.step()
            b = [torch.nn.Parameter(p.detach().clone()) for p in a]
            ob = pkg.AdamW(b, lr=1.0, state_bits=bits, capturable=capturable)
            ob.load_state_dict(pickle.loads(pickle.dumps(oa.state_dict())))
            assert ob.param_groups[0]["lr"] == 1e-2
            c, oc = copy.deepcopy((a, oa))
            for t in range(3, 6):
                for ps, o in ((a, oa), (b, ob), (c, oc)):
                    fill(ps, t)
                    o.step()
            assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
            assert all(x is None or torch.equal(x, y) for x, y in zip(oa.group_state(), ob.group_state()))
    loss = oa.step(lambda: torch.ones(()))
    assert float(loss) == 1.0
    oa.zero_grad()
    before = [p.detach().clone() for p in a]
    oa.step()
    assert all(torch.equal(x, y) for x, y in zip(a, before))
    oa.add_param_group({"params": [torch.nn.Parameter(torch.ones(3, device=dev))]})
    oa.param_groups[1]["params"][0].grad = torch.ones(3, device=dev)
    oa.step()
    assert oa.group_state(1).m.numel() == 256


def test_a_step_repacks_the_linear(pkg, dev):
    lin = pkg.BitLinear(256, 64, device=dev)
    opt = pkg.AdamW(lin.parameters(), lr=0.05)
    x = torch.randn(8, 256, device=dev)
    lin(x).square().sum().backward()
    packed, version = lin.qweight.clone(), lin.weight._version
    opt.step()
    assert lin.weight._version > version
    lin(x)
    assert not torch.equal(lin.qweight, packed)
    assert torch.equal(lin.qweight, pkg.pack_ternary_i2s(lin.weight.detach())[0])


def test_two_streams(pkg, dev):
    sets = [_make(dev, [5000, 77], F32, F32, seed=s) for s in range(2)]
    twins = [[p.clone() for p in s[0]] for s in sets]
    states = [pkg.adamw_state(s[0], 8) for s in sets]
    refs = [pkg.adamw_state(s[0], 8) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s, (p, g), st in zip(streams, sets, states):
        with torch.cuda.stream(s):
            for t in range(1, 4):
                pkg.adamw_step(p, g, st, t, **HYPER)
    torch.cuda.synchronize()
    for (p, g), tw, st, ref in zip(sets, twins, states, refs):
        for t in range(1, 4):
            pkg.adamw_step(tw, g, ref, t, **HYPER)
        assert all(torch.equal(a, b) for a, b in zip((*p, *st), (*tw, *ref)))


def test_refusals(pkg, dev):
    params, grads = _make(dev, [300, 20], F32, F32)
    state = pkg.adamw_state(params, 8)

    def no(match, *args, err=RuntimeError, **kw):
        with pytest.raises(err, match=match):
            pkg.adamw_step(*args, **kw)

    no("gradients", params, grads[:1], state, 1)
    no("elements", params[:1], grads[:1], state, 1)
    no("shape", params, [grads[1], grads[0]], state, 1)
    no("must be on|both are on", params, [g.cpu() for g in grads], state, 1)
    no("expected float", params, [g.double() for g in grads], state, 1)
    no("contiguous", [torch.randn(20, 30, device=dev).t()[:, :15], params[1]], [torch.randn(30, 15, device=dev), grads[1]],
       pkg.adamw_state([torch.empty(450, device=dev), params[1]]), 1)
    no("twice", [params[0], params[0]], [grads[0], grads[0]], pkg.adamw_state([params[0], params[0]]), 1)
    no("steps count", params, grads, state, 0)
    no("betas", params, grads, state, 1, betas=(1.0, 0.9))
    no("negative", params, grads, state, 1, lr=-1.0)
    no("step tensor", params, grads, state, torch.ones(1, device=dev))
    no("lr tensor", params, grads, state, 1, lr=torch.ones(1, device=dev))
    no("HIP device", params, grads, pkg.AdamWState(*(t.cpu() for t in state)), 1)
    no("scales", params, grads, state._replace(m_scale=state.m_scale[:1]), 1)
    no("a state is", params, grads, state._replace(v=state.v.to(torch.int8)), 1)
    with pytest.raises(ValueError, match="bits"):
        pkg.adamw_state(params, 16)
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(state_bits=4), dict(eps=-1.0), dict(lr=torch.ones(1))):
        with pytest.raises(ValueError):
            pkg.AdamW([torch.nn.Parameter(params[0])], **kw)
