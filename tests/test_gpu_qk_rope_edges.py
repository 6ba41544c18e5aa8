"""Edges of qk_norm_rope: a norm without an epsilon.

Bounds as for ordinary rows: eps = 0 leaves the formulas as they are wherever a row is not all zeros."""

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def _tables(dev, n, r):
    ang = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * 10000.0 ** (
        -torch.arange(0, r, 2, dtype=torch.float64, device=dev) / max(r, 1))[None, :]
    return ang.cos().float(), ang.sin().float()


def _inputs(dev, b, t, hq, hk, d, dtype):
    g = torch.Generator(device=dev).manual_seed(1000 * b + t + d)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    return (rand(b, t, hq, d).to(dtype), rand(b, t, hk, d).to(dtype), (1 + 0.3 * rand(d)).to(dtype),
            (1 + 0.3 * rand(d)).to(dtype), rand(b, t, hq, d).to(dtype), rand(b, t, hk, d).to(dtype))


def _exact(x, w, cos, sin, g, eps):
    """(out, grad_x, grad_w) of the half layout at positions 0 .. t - 1 in float64."""
    c, s = (y.double()[:x.shape[1], None] for y in (cos, sin))
    r2 = cos.shape[1]

    def turn(y, s):
        a, b = y[..., :r2], y[..., r2:2 * r2]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * r2:]], -1)

    xd, wd = x.double(), w.double()
    r = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
    n, gy = xd * r, turn(g.double(), -s)
    gw = gy * wd
    return turn(n * wd, s), r * (gw - n * (gw * n).mean(-1, keepdim=True)), (gy * n).sum((0, 1, 2))


def _near(got, ref, roundings, what):
    top = ref.abs().amax(-1, keepdim=True)
    lim = roundings * U * top + torch.finfo(got.dtype).eps / 2 * ref.abs() * 1.001 + torch.finfo(got.dtype).tiny
    assert bool(((got.double() - ref).abs() <= lim).all()), what


# heads that are and are not whole groups of four, tokens that leave the last turn of the workgroups unfilled
@pytest.mark.parametrize("b,t,hq,hk,d,r", [(3, 333, 9, 3, 64, 32), (1, 1, 1, 1, 128, 128), (2, 7, 8, 4, 128, 128), (1, 5, 6, 2, 10, 6),
                                           (2, 3, 5, 1, 256, 256), (1, 3000, 4, 4, 64, 64)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_no_epsilon(pkg, dev, b, t, hq, hk, d, r, dtype):
    q, k, wq, wk, gq, gk = _inputs(dev, b, t, hq, hk, d, dtype)
    cos, sin = _tables(dev, t, r)
    leaves = [x.requires_grad_() for x in (q, k, wq, wk)]
    outs = pkg.qk_norm_rope(q, k, cos, sin, None, wq, wk, eps=0.0)
    grads = torch.autograd.grad(outs, leaves, [gq, gk])
    for i, (x, w, g) in enumerate(((q, wq, gq), (k, wk, gk))):
        ref, rx, rw = _exact(x.detach(), w.detach(), cos, sin, g, 0.0)
        _near(outs[i].detach(), ref, 24, "out")
        _near(grads[i], rx, 96, "grad_x")
        # a sum over N rows: sqrt(N) / 8 + 24 roundings at the most, and half a step
        off = float((grads[2 + i].double() - rw).norm() / rw.norm())
        assert off <= (24 + (b * t * x.shape[2]) ** 0.5) * U + torch.finfo(dtype).eps / 2, off


@pytest.mark.parametrize("exponent", [0, -62, -66])
def test_the_inverse_root_is_rounded(pkg, dev, exponent):
    """Heads of two equal elements of 11 bits, no epsilon: the mean of squares and its root are exact, r is off by half a step,
    a r by 2^-24 of 1, and 1 + 2^-24 rounds to 1.  At 2^-62 the squares lie at the least normal numbers, at 2^-66 they are
    subnormal and hold the squares of 8 bits exactly."""
    bits = 11 if exponent > -66 else 8
    a = torch.arange(1, 1 << bits, device=dev).float() * 2.0 ** exponent
    q = torch.stack([a, -a], -1)[None, :, None]  # [1, tokens, 1, 2]
    one = torch.ones(2, device=dev)
    cos, sin = torch.ones(1, 1, device=dev), torch.zeros(1, 1, device=dev)
    pos = torch.zeros(a.numel(), dtype=torch.int64, device=dev)
    out, _ = pkg.qk_norm_rope(q, q, cos, sin, pos, one, one, eps=0.0)
    off = (out.double() - torch.tensor([1.0, -1.0], device=dev, dtype=torch.float64)).abs()
    assert float(off.max()) <= 2.0 ** -24
