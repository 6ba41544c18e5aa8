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
