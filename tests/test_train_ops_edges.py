"""CPU checks of the training operators' refusals at their edges: arguments that the kernels have no meaning for."""

import ctypes
import math

import pytest
import torch

vp = ctypes.c_void_p


def _no(pkg, match, status):
    assert status == -1 and match in pkg._lib.last_error(), pkg._lib.last_error()


@pytest.mark.parametrize("eps", [-1e-6, -math.inf, math.nan])
@pytest.mark.parametrize("grad", [False, True])
def test_epsilon_of_the_head_norm(pkg, eps, grad):
    heads, rope = pkg._lib.HeadsStruct(), pkg._lib.RopeStruct()
    heads.x = heads.g = heads.out = 0x1000
    heads.heads, heads.stride_b, heads.stride_t, heads.stride_h = 2, 1024, 128, 64
    rope.cos, rope.sin, rope.rope_len, rope.rotary_dim = 0x100, 0x200, 32, 64
    at = [ctypes.addressof(s) for s in (heads, heads, rope)]
    name = "wfb_qk_norm_rope_grad" if grad else "wfb_qk_norm_rope"
    _no(pkg, "eps", pkg._lib.status(name, *at, 1, 2, 8, 64, eps, *([vp(0x100)] if grad else []), None))


YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)


@pytest.mark.parametrize("scaling", [
    dict(YARN, mscale=1.0), dict(YARN, mscale_all_dim=0.7), dict(YARN, truncate=False), dict(YARN, low_freq_factor=1.0),
    dict(type="linear", factor=2.0, beta_fast=32.0), dict(type="linear", factor=2.0, atention_factor=1.0),
    dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192, short_factor=[1.0])])
def test_scalings_with_unknown_keys(pkg, scaling):
    with pytest.raises(ValueError, match="does not know"):
        pkg.rope_tables(10000.0, 64, 16, scaling=scaling)


def test_scalings_with_keys_that_are_not_set(pkg):
    plain = pkg.rope_tables(10000.0, 64, 16, scaling=YARN)
    same = pkg.rope_tables(10000.0, 64, 16, scaling=dict(YARN, type="yarn", attention_factor=None, mscale=None, beta_fast=32))
    assert all(torch.equal(a, b) for a, b in zip(plain, same))
    a = pkg.rope_tables(10000.0, 64, 16, scaling=dict(type="linear", factor=2.0))
    b = pkg.rope_tables(10000.0, 64, 16, scaling=dict(type="linear", factor=2.0, original_max_position_embeddings=2048))
    assert torch.equal(a[0], b[0])
    with pytest.raises(ValueError, match="theta"):
        pkg.rope_tables(1.0, 64, 16, scaling=YARN)


def test_workspace_of_wide_gradients(pkg):
    n, wide = ctypes.c_int64(-1), pkg._lib.WFB_GRAD_WIDE
    bf16, f32 = pkg._lib.WFB_BF16, pkg._lib.WFB_F32

    def size(gx, gw):
        assert pkg._lib.status("wfb_gated_grad_workspace", 100, 65, 200, gx, 1, gw, 1, ctypes.addressof(n)) == 0
        return n.value

    assert size(bf16, bf16) < size(bf16 | wide, bf16) < size(bf16 | wide, bf16 | wide) == size(f32, f32) == size(f32 | wide, f32)
    _no(pkg, "dtype", pkg._lib.status("wfb_gated_grad_workspace", 100, 65, 200, 2 * wide, 1, f32, 1, ctypes.addressof(n)))
    _no(pkg, "dtype", pkg._lib.status("wfb_gated_grad_workspace", 100, 65, 200, -1, 1, f32, 1, ctypes.addressof(n)))


def test_a_gated_pair_of_packed_projections(pkg):
    packed = pkg.BitLinear.from_packed(torch.zeros(8, 32, dtype=torch.uint8), torch.ones(1), 128)
    for pair in ((packed, packed), (pkg.BitLinear(128, 8), packed)):
        with pytest.raises(RuntimeError, match="no float weight"):
            pkg.GatedBitLinear.from_linears(*pair)
