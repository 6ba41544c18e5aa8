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
