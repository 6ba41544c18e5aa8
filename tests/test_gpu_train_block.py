"""The training operators as a block uses them: projections on BitLinear, qk_norm_rope, attention, the gated product behind
its norm, AdamW on every weight; against the same block with torch's elementary operations in their places.

Both blocks quantise the same way; where their fp32 activations differ in a last bit a code may round to its
neighbour, which moves one element by 1/127 of its row's largest: at most 1 of about 640 (the norm of 256 codes of rms 40)
of the row for each of the four quantisers that a gradient passes, 6.3e-3 were every token hit at each.  Bound 1e-2."""

import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

B, T, H, HQ, HK, D, F = 2, 24, 256, 4, 2, 64, 384


class Block(nn.Module):
    def __init__(self, pkg, dev, kernels):
        super().__init__()
        self.pkg, self.kernels = pkg, kernels
        lin = lambda i, o: pkg.BitLinear(i, o, device=dev)  # noqa: E731
        self.q, self.k, self.v = lin(H, HQ * D), lin(H, HK * D), lin(H, HK * D)
        self.qn, self.kn = (nn.Parameter(torch.ones(D, device=dev)) for _ in range(2))
        self.o = pkg.SubLNBitLinear(HQ * D, H, device=dev)
        self.ffn = pkg.GatedBitLinear(H, F, act="silu", device=dev)
        self.down = pkg.SubLNBitLinear(F, H, device=dev)

    def _rotate(self, x, w, cos, sin):
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = x[..., 0::2], x[..., 1::2]
        c, s = cos[:T, None], sin[:T, None]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)

    def forward(self, x, cos, sin):
        q, k, v = self.q(x).view(B, T, HQ, D), self.k(x).view(B, T, HK, D), self.v(x).view(B, T, HK, D)
        if self.kernels:
            q, k = self.pkg.qk_norm_rope(q, k, cos, sin, None, self.qn, self.kn, layout="interleaved")
        else:
            q, k = self._rotate(q, self.qn, cos, sin), self._rotate(k, self.kn, cos, sin)
        k, v = (t.repeat_interleave(HQ // HK, 2).transpose(1, 2) for t in (k, v))
        s = (q.transpose(1, 2) @ k.transpose(2, 3).contiguous()) / math.sqrt(D)
        s = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device=x.device).triu(1), -math.inf).softmax(-1)
        x = x + self.o((s @ v.contiguous()).transpose(1, 2).reshape(B, T, HQ * D))
        if self.kernels:
            h = self.ffn(x)
        else:
            g = self.ffn.gate_proj(x)
            h = g * torch.sigmoid(g) * self.ffn.up_proj(x)
        return x + self.down(h)


def _blocks(pkg, dev):
    torch.manual_seed(3)
    a = Block(pkg, dev, True)
    b = Block(pkg, dev, False)
    b.load_state_dict(a.state_dict())
    return a, b


def test_a_block_trains(pkg, dev):
    a, b = _blocks(pkg, dev)
    cos, sin = (t.to(dev) for t in pkg.rope_tables(10000.0, D, 64))
    x = torch.randn(B, T, H, device=dev)
    target = torch.randn(B, T, H, device=dev)
    grads = []
    for m in (a, b):
        xi = x.clone().requires_grad_()
        y = m(xi, cos, sin)
        (y * target).sum().backward()
        grads.append([xi.grad] + [p.grad for p in m.parameters()])
    for got, ref in zip(*grads):
        assert float((got - ref).norm()) <= 1e-2 * float(ref.norm())
    # steps of the optimizer: every weight moves, the packs follow, and 8 bits of state stay near 32
    twin = [p.detach().clone().requires_grad_() for p in a.parameters()]
    for p, t in zip(a.parameters(), twin):
        t.grad = p.grad.clone()
    before = [p.detach().clone() for p in a.parameters()]
    packs = (a.ffn.packed().qweight.clone(), a.q.qweight.clone())
    eight, full = pkg.AdamW(a.parameters(), lr=1e-2, state_bits=8), pkg.AdamW(twin, lr=1e-2)
    for _ in range(3):
        eight.step()
        full.step()
    for p, q, t in zip(a.parameters(), before, twin):
        # a constant gradient moves every element by about lr a step, whatever its size.  A moment held in 8 bits is off by
        # up to a code's distance, 2 / c of its value: elements at small codes (below a thousandth of their block's largest)
        # may move by half or by twice lr, and so a tensor by a tenth of its path
        assert not torch.equal(p, q)
        assert float((p - t).detach().norm()) <= 0.1 * float((t - q).detach().norm())
    y = a(x, cos, sin)
    assert torch.isfinite(y).all()
    assert not torch.equal(a.ffn.packed().qweight, packs[0]) and not torch.equal(a.q.qweight, packs[1])


def test_a_block_serves_what_it_trains(pkg, dev):
    a, _ = _blocks(pkg, dev)
    cos, sin = (t.to(dev) for t in pkg.rope_tables(10000.0, D, 64))
    x = torch.randn(B, T, H, device=dev)
    with torch.no_grad():
        served = a(x, cos, sin)
    assert torch.equal(served, a(x, cos, sin).detach())


def test_a_training_step_in_a_graph(pkg, dev):
    """Forward, backward and optimizer captured once; replays on new inputs equal eager steps."""
    a, b = (_blocks(pkg, dev)[0] for _ in range(2))
    cos, sin = (t.to(dev) for t in pkg.rope_tables(10000.0, D, 64))
    xs = [torch.randn(B, T, H, device=dev) for _ in range(4)]
    ys = [torch.randn(B, T, H, device=dev) for _ in range(4)]
    pa, pb = list(a.parameters()), list(b.parameters())
    sa, sb = pkg.adamw_state(pa, 8), pkg.adamw_state(pb, 8)
    x, y = xs[0].clone(), ys[0].clone()
    count = torch.zeros(1, dtype=torch.int64, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad((a(x, cos, sin) * y).sum(), pa)
    torch.cuda.current_stream().wait_stream(side)
    for m in a.modules():  # the packs are made within the step
        for name in ("qweight", "_packed"):
            if getattr(m, name, None) is not None:
                setattr(m, name, None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad((a(x, cos, sin) * y).sum(), pa)
        count.add_(1)
        pkg.adamw_step(pa, grads, sa, count, lr=1e-3)
    for t, (xi, yi) in enumerate(zip(xs, ys), 1):
        x.copy_(xi)
        y.copy_(yi)
        graph.replay()
        torch.cuda.synchronize()
        pkg.adamw_step(pb, torch.autograd.grad((b(xi, cos, sin) * yi).sum(), pb), sb, t, lr=1e-3)
        assert all(torch.equal(p, q) for p, q in zip(pa, pb))
        assert all(torch.equal(p, q) for p, q in zip(sa, sb))
