"""The training operators under autograd's other modes: what they have no derivative for is refused, not dropped."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._pytree import tree_map

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(4))
def test_tangents_are_refused(pkg, dev, which, grad):
    x, gate, up = torch.randn(5, 128, device=dev), torch.randn(64, 128, device=dev), torch.randn(64, 128, device=dev)
    packed = pkg.pack_gated(gate, up)
    q, k, w = torch.randn(1, 3, 2, 64, device=dev), torch.randn(1, 3, 1, 64, device=dev), torch.ones(64, device=dev)
    cos, sin = (t.to(dev) for t in pkg.rope_tables(1e4, 64, 8))
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.randn_like(t))  # noqa: E731
        with pytest.raises(RuntimeError, match="forward-mode"):
            ins = [x, gate, up]
            if which < 3:
                ins[which] = dual(ins[which])
                pkg.gated_bitlinear(*ins)
            else:
                pkg.gated_bitlinear(dual(x), packed=packed)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ins = [q, k, w, w]
            ins[which] = dual(ins[which])
            pkg.qk_norm_rope(ins[0], ins[1], cos, sin, None, ins[2], ins[3])
        # a level without tangents changes nothing
        inside = (pkg.gated_bitlinear(x, gate, up), *pkg.qk_norm_rope(q, k, cos, sin, None, w, w))
    outside = (pkg.gated_bitlinear(x, gate, up), *pkg.qk_norm_rope(q, k, cos, sin, None, w, w))
    assert all(torch.equal(a, b) for a, b in zip(inside, outside))


def test_lazily_negated_tables_weights_and_states(pkg, dev):
    """A negated view's memory holds the other sign: the value counts, in every operand."""
    neg = torch._neg_view
    q, k = torch.randn(2, 3, 3, 64, device=dev), torch.randn(2, 3, 1, 64, device=dev)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    cos, sin = (t.to(dev) for t in pkg.rope_tables(1e4, 64, 8))
    pos = torch.arange(3, device=dev)
    w = [torch.randn(64, device=dev) for _ in range(2)]

    def run(c, s, p, wq, wk):
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        out = pkg.qk_norm_rope(leaves[0], leaves[1], c, s, p, leaves[2], leaves[3])
        with torch.no_grad():
            served = pkg.qk_norm_rope(q, k, c, s, p, wq, wk)
        return [*(t.detach() for t in out), *served, *(t.resolve_neg() for t in torch.autograd.grad(out, leaves, (gq, gk)))]

    want = run(cos, sin, pos, *w)
    for got in (run(neg(-cos), sin, pos, *w), run(cos, neg(-sin), pos, *w), run(cos, sin, neg(-pos), *w),
                run(cos, sin, pos, neg(-w[0]), w[1]), run(cos, sin, pos, w[0], neg(-w[1]))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, gate, up = torch.randn(5, 128, device=dev), torch.randn(64, 128, device=dev), torch.randn(64, 128, device=dev)
    packed = pkg.pack_gated(gate, up)
    twin = packed._replace(scales=neg(-packed.scales))
    assert torch.equal(pkg.gated_bitlinear(x, packed=packed), pkg.gated_bitlinear(x, packed=twin))
    rows = [torch.randn(300, device=dev)]
    results = []
    for lr, step in ((torch.full((1,), 1e-2, device=dev), torch.ones(1, dtype=torch.int64, device=dev)),
                     (neg(torch.full((1,), -1e-2, device=dev)), neg(-torch.ones(1, dtype=torch.int64, device=dev)))):
        p = [r.clone() for r in rows]
        pkg.adamw_step(p, rows, pkg.adamw_state(p), step, lr=lr)
        results.append(p[0])
    assert torch.equal(*results)
    p, state = [rows[0].clone()], pkg.adamw_state(rows)
    with pytest.raises(RuntimeError, match="state must be contiguous"):
        pkg.adamw_step(p, rows, state._replace(m=neg(state.m)), 1)
    with pytest.raises(RuntimeError, match="state must be contiguous"):
        pkg.adamw_state_values(state._replace(v=neg(state.v)))


class _Wrapped(torch.Tensor):
    """A tensor class whose objects have no memory but that of the tensor they wrap (as distributed tensors are)."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    def __init__(self, t):
        self.inner = t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return func(*tree_map(lambda x: x.inner if isinstance(x, cls) else x, args), **(kwargs or {}))


def test_tensors_without_memory_are_refused(pkg, dev):
    """Their pointer is null, which for a gradient, a norm's weight or positions would mean that there is none."""
    p, g = [torch.randn(300, device=dev), torch.randn(20, device=dev)], [torch.randn(300, device=dev), torch.randn(20, device=dev)]
    before = [t.clone() for t in p]
    for params, grads in ((p, [_Wrapped(g[0]), g[1]]), ([_Wrapped(p[0]), p[1]], g), ([_Wrapped(t) for t in p], [_Wrapped(t) for t in g])):
        with pytest.raises(RuntimeError):
            pkg.adamw_step(params, grads, pkg.adamw_state(p), 1)
    assert all(torch.equal(a, b) for a, b in zip(p, before))
    empty = [torch.randn(300, device=dev), torch.empty(0, device=dev)]  # (no elements, no memory: fine)
    pkg.adamw_step(empty, [g[0], torch.empty(0, device=dev)], pkg.adamw_state(empty), 1)
    q, k, w = torch.randn(1, 3, 2, 64, device=dev), torch.randn(1, 3, 1, 64, device=dev), torch.ones(64, device=dev)
    cos, sin = (t.to(dev) for t in pkg.rope_tables(1e4, 64, 8))
    pos = torch.arange(3, device=dev)
    for args in ((q, k, cos, sin, _Wrapped(pos), w, w), (q, k, cos, sin, pos, _Wrapped(w), w), (q, k, cos, sin, pos, w, _Wrapped(w)),
                 (_Wrapped(q), k, cos, sin, pos, w, w), (q, k, _Wrapped(cos), sin, pos, w, w)):
        with pytest.raises(RuntimeError):
            pkg.qk_norm_rope(*args)
    x, gate, up = torch.randn(5, 128, device=dev), torch.randn(64, 128, device=dev), torch.randn(64, 128, device=dev)
    want = pkg.gated_bitlinear(x, gate, up)
    with pytest.raises(RuntimeError):
        pkg.gated_bitlinear(_Wrapped(x), gate, up)
    for args in ((x, _Wrapped(gate), up), (x, gate, _Wrapped(up))):  # (this class unwraps where its weights are detached)
        assert torch.equal(pkg.gated_bitlinear(*args), want)
