"""Norm of every query and key head with the rotary embedding, for training attention and for serving.

The rotation of the reference's training attention (WF/models/attention.py:14-64, WF =
packages/training/src/wrinklefree) turns adjacent elements, ``layout="interleaved"``; the stage-1 model's turns the
halves of a head, ``layout="half"``.  Tables come from :func:`rope_tables` or from anywhere else: fp32
[positions, rotary_dim / 2]; a table narrower than half a head turns the head's first elements only.
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import HeadsStruct, RopeStruct, WFB_QK_MAX_DIM
from .ops import _DT, _on, _stream

_LAYOUTS = {"half": 0, "interleaved": 1}
_NAME = "qk_norm_rope"

Positions = Union[None, int, torch.Tensor]


def _side(x: torch.Tensor, weight: Optional[torch.Tensor]) -> HeadsStruct:
    sb, st, sh, _ = x.stride()
    w, wdt = (None, 0) if weight is None else (weight.data_ptr(), _DT[weight.dtype])
    return HeadsStruct(x.data_ptr(), sb, st, sh, None, 0, 0, 0, w, wdt, None, None, x.shape[2])


def _rope(cos: torch.Tensor, sin: torch.Tensor, positions: Positions, layout: str) -> RopeStruct:
    n, half = cos.shape
    if isinstance(positions, torch.Tensor):
        where = (positions.data_ptr(), positions.element_size(), *positions.stride(), 0)
    else:
        where = (None, 0, 0, 0, positions)
    return RopeStruct(cos.data_ptr(), sin.data_ptr(), n, 2 * half, _LAYOUTS[layout], *where)


def _plain(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous heads in its own memory, as the kernels read it."""
    return x if x.stride(-1) == 1 and not x.is_neg() else x.resolve_neg().contiguous()


def _forward(q, k, cos, sin, positions, wq, wk, eps, layout):
    b, t, _, d = q.shape
    out = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k)]
    sq, sk, rope = _side(q, wq), _side(k, wk), _rope(cos, sin, positions, layout)
    sq.out, sk.out = out[0].data_ptr(), out[1].data_ptr()
    with _on(q.device):
        _lib.call("wfb_qk_norm_rope", ctypes.addressof(sq), ctypes.addressof(sk), ctypes.addressof(rope), _DT[q.dtype],
                  b, t, d, eps, _stream(q.device))
    return out


@functools.lru_cache(maxsize=256)
def _grad_workspace(*sizes: int) -> int:
    """Floats that wfb_qk_norm_rope_grad works with at these sizes."""
    n = ctypes.c_int64(0)
    _lib.call("wfb_qk_norm_rope_grad_workspace", *sizes, ctypes.addressof(n))
    return n.value


class _QkNormRope(torch.autograd.Function):
    """The kernel's forward; its backward recomputes the norms from x and turns the gradient back."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, eps, layout):
        ctx.save_for_backward(q, k, wq, wk, cos, sin, positions if isinstance(positions, torch.Tensor) else None)
        ctx.meta = (None if isinstance(positions, torch.Tensor) else positions, eps, layout)
        return tuple(_forward(q, k, cos, sin, positions, wq, wk, eps, layout))

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, wq, wk, cos, sin, pos = ctx.saved_tensors
        start, eps, layout = ctx.meta
        need = ctx.needs_input_grad
        b, t, _, d = q.shape
        dev = q.device
        rope = _rope(cos, sin, pos if pos is not None else start, layout)
        sides, grads, weights = [], [], []
        for x, w, g, need_x, need_w in ((q, wq, gq, need[0], need[2]), (k, wk, gk, need[1], need[3])):
            g = _plain(g)
            s = _side(x, w)
            s.g = g.data_ptr()
            s.g_stride_b, s.g_stride_t, s.g_stride_h = g.stride()[:3]
            gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
            gw = torch.empty_like(w) if w is not None and need_w else None
            s.out = None if gx is None else gx.data_ptr()
            s.grad_weight = None if gw is None else gw.data_ptr()
            sides.append((s, g))
            grads.append(gx)
            weights.append(gw)
        work = None
        if any(w is not None for w in weights):
            work = torch.empty(_grad_workspace(b, t, q.shape[2], k.shape[2], d), dtype=torch.float32, device=dev)
        with _on(dev):
            _lib.call("wfb_qk_norm_rope_grad", ctypes.addressof(sides[0][0]), ctypes.addressof(sides[1][0]),
                      ctypes.addressof(rope), _DT[q.dtype], b, t, d, eps, None if work is None else work.data_ptr(),
                      _stream(dev))
        return (*grads, *weights, None, None, None, None, None)


def qk_norm_rope(
    q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Positions = None,
    q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
    layout: str = "half",
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with their heads normed (x / sqrt(mean(x^2) + eps) * weight over the head's elements; a side
    without a weight is not normed) and turned by their positions' angles, in one pass; differentiable once, by q, k and
    the weights.

    q [batch, tokens, heads, head_dim] and k [batch, tokens, kv_heads, head_dim], or both without the batch dimension,
    fp32, bf16 or fp16 with contiguous heads (slices of one q|k|v projection go as they are); the results are contiguous.
    cos / sin fp32 [positions, rotary_dim / 2].  ``positions``: int32 or int64 [batch, tokens] or [tokens] on the
    device, or the first token's as a number (None: 0).  One of the device's that the tables do not hold gives a row of
    NaN.  layout "half" turns pairs (i, i + rotary_dim / 2) of a head's first rotary_dim elements, "interleaved" pairs
    (2 i, 2 i + 1).  Statistics and rotation are fp32, a result is rounded once."""
    if layout not in _LAYOUTS:
        raise ValueError(f"{_NAME}: layout must be one of {sorted(_LAYOUTS)}")
    if q.dim() not in (3, 4) or k.dim() != q.dim():
        raise RuntimeError(f"{_NAME}: q and k must be [batch, tokens, heads, head_dim] or [tokens, heads, head_dim]")
    if q.dtype not in _DT or k.dtype != q.dtype:
        raise RuntimeError(f"{_NAME}: q and k must be of one type, float32, bfloat16 or float16")
    dev, d = q.device, q.shape[-1]
    if dev.type != "cuda":
        raise RuntimeError(f"{_NAME}: tensors must be on a HIP device (got {dev})")
    for x in (k, cos, sin, q_weight, k_weight) + ((positions,) if isinstance(positions, torch.Tensor) else ()):
        if x is not None and x.device != dev:
            raise RuntimeError(f"{_NAME}: tensors are on different devices ({dev}, {x.device})")
    if k.shape[:-2] != q.shape[:-2] or k.shape[-1] != d:
        raise RuntimeError(f"{_NAME}: q {list(q.shape)} and k {list(k.shape)} must agree in all but their heads")
    if d % 2 or not 2 <= d <= WFB_QK_MAX_DIM:
        raise ValueError(f"{_NAME}: head_dim ({d}) must be even and at most {WFB_QK_MAX_DIM}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or cos.shape != sin.shape \
            or not cos.is_contiguous() or not sin.is_contiguous() or 2 * cos.shape[1] > d:
        raise RuntimeError(f"{_NAME}: cos and sin must be contiguous float32 [positions, at most {d // 2}]")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype not in _DT or w.numel() != d or not w.is_contiguous()):
            raise RuntimeError(f"{_NAME}: norm weights must be contiguous floats of {d} elements")
    flat = q.dim() == 3
    if flat:
        q, k = q.unsqueeze(0), k.unsqueeze(0)
    b, t = q.shape[:2]
    if isinstance(positions, torch.Tensor):
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((t,), (b, t)):
            raise RuntimeError(f"{_NAME}: positions must be int32 or int64 [{t}] or [{b}, {t}]")
        positions = positions.expand(b, t)
    else:
        positions = 0 if positions is None else int(positions)
        if cos.shape[1] and not 0 <= positions <= cos.shape[0] - t:
            raise ValueError(f"{_NAME}: positions {positions}..{positions + t - 1} leave tables of {cos.shape[0]} rows")
    q, k = _plain(q), _plain(k)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, q_weight, k_weight)):
        out = _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), layout)
    else:
        out = _forward(q, k, cos, sin, positions, q_weight, k_weight, float(eps), layout)
    return (out[0].squeeze(0), out[1].squeeze(0)) if flat else (out[0], out[1])
