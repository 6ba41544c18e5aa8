"""The training operators under autograd's other modes: what they have no derivative for is refused, not dropped."""

import pytest
import torch
from torch.autograd import forward_ad

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
