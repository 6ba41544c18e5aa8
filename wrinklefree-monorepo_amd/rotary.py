"""Norm of every query and key head with the rotary embedding, for training attention and for serving.

The rotation of the reference's training attention (WF/models/attention.py:14-64, WF =
packages/training/src/wrinklefree) turns adjacent elements, ``layout="interleaved"``; the stage-1 model's turns the
halves of a head, ``layout="half"``.  Tables come from :func:`rope_tables` or from anywhere else: fp32
[positions, rotary_dim / 2]; a table narrower than half a head turns the head's first elements only.
"""

from __future__ import annotations

import ctypes
import functools
from array import array
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import HeadsStruct, WFB_QK_MAX_DIM
from .ops import _DT, _no_tangents, _on, _stream

_LAYOUTS = {"half": 0, "interleaved": 1}
_NAME = "qk_norm_rope"

Positions = Union[None, int, torch.Tensor]


# The structs of the C interface (wfb_heads, wfb_rope) are made of 8-byte fields: the calls hand them over as one array of
# integers, which costs a third of three ctypes structures (a single token's call is bound by the host).


def _memory(t: torch.Tensor) -> int:
    """Where t lies, for the operands whose null pointer means that there is none."""
    at = t.data_ptr()
    if not at and t.numel():
        raise RuntimeError(f"{_NAME}: a tensor without memory of its own (of a wrapping class)")
    return at


def _heads(x: torch.Tensor, weight: Optional[torch.Tensor], out: int, g: Optional[torch.Tensor] = None, gw: int = 0) -> tuple:
    """The fields of wfb_heads."""
    w, wdt = (0, 0) if weight is None else (_memory(weight), _DT[weight.dtype])
    gs = (0, 0, 0, 0) if g is None else (g.data_ptr(), *g.stride()[:3])
    return (x.data_ptr(), *x.stride()[:3], *gs, w, wdt, out, gw, x.shape[2])


def _rope(cos: torch.Tensor, sin: torch.Tensor, positions: Union[int, torch.Tensor], layout: str) -> tuple:
    """The fields of wfb_rope."""
    n, half = cos.shape
    if isinstance(positions, torch.Tensor):
        st = positions.stride()
        where = (_memory(positions), positions.element_size(), st[0] if len(st) == 2 else 0, st[-1], 0)
    else:
        where = (0, 0, 0, 0, positions)
    return (cos.data_ptr(), sin.data_ptr(), n, 2 * half, _LAYOUTS[layout], *where)


_K_AT, _ROPE_AT = ctypes.sizeof(HeadsStruct), 2 * ctypes.sizeof(HeadsStruct)


def _plain(x: torch.Tensor) -> torch.Tensor:
    """x with contiguous heads in its own memory, as the kernels read it."""
    return x if x.stride(-1) == 1 and not x.is_neg() else x.resolve_neg().contiguous()


def _forward(q, k, cos, sin, positions, wq, wk, eps, layout):
    b, t, _, d = q.shape
    dev = q.device
    qo, ko = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
    args = array("q", (*_heads(q, wq, qo.data_ptr()), *_heads(k, wk, ko.data_ptr()), *_rope(cos, sin, positions, layout)))
    at = args.buffer_info()[0]
    with _on(dev):
        _lib.call("wfb_qk_norm_rope", at, at + _K_AT, at + _ROPE_AT, _DT[q.dtype], b, t, d, eps, _stream(dev))
    return qo, ko


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
        return _forward(q, k, cos, sin, positions, wq, wk, eps, layout)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        # (a saved-tensor hook may give them back as other views)
        q, k, wq, wk, cos, sin, pos = (t if t is None else t.resolve_neg() for t in ctx.saved_tensors)
        q, k = _plain(q), _plain(k)
        wq, wk, cos, sin = (t if t is None else t.contiguous() for t in (wq, wk, cos, sin))
        start, eps, layout = ctx.meta
        need = ctx.needs_input_grad
        b, t, hq, d = q.shape
        dev = q.device
        gq, gk = _plain(gq), _plain(gk)
        gx = [torch.empty_like(x, memory_format=torch.contiguous_format) if n else None for x, n in ((q, need[0]), (k, need[1]))]
        gw = [torch.empty_like(w) if w is not None and n else None for w, n in ((wq, need[2]), (wk, need[3]))]
        work = 0
        if gw[0] is not None or gw[1] is not None:
            scratch = torch.empty(_grad_workspace(b, t, hq, k.shape[2], d), dtype=torch.float32, device=dev)
            work = scratch.data_ptr()
        p = [0 if x is None else x.data_ptr() for x in (*gx, *gw)]
        args = array("q", (*_heads(q, wq, p[0], gq, p[2]), *_heads(k, wk, p[1], gk, p[3]),
                           *_rope(cos, sin, start if pos is None else pos, layout)))
        at = args.buffer_info()[0]
        with _on(dev):
            _lib.call("wfb_qk_norm_rope_grad", at, at + _K_AT, at + _ROPE_AT, _DT[q.dtype], b, t, d, eps, work, _stream(dev))
        return (*gx, *gw, None, None, None, None, None)


def qk_norm_rope(
    q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: Positions = None,
    q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
    layout: str = "half",
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys with their heads normed (x / sqrt(mean(x^2) + eps) * weight over the head's elements; a side
    without a weight is not normed) and turned by their positions' angles, in one pass; differentiable once, by q, k and
    the weights (in reverse mode; tangents of forward mode are refused).

    q [batch, tokens, heads, head_dim] and k [batch, tokens, kv_heads, head_dim], or both without the batch dimension,
    fp32, bf16 or fp16 with contiguous heads (slices of one q|k|v projection go as they are); the results are contiguous.
    cos / sin fp32 [positions, rotary_dim / 2].  ``positions``: int32 or int64 [batch, tokens] or [tokens] on the
    device, or the first token's as a number (None: 0).  One of the device's that the tables do not hold gives a row of
    NaN.  eps >= 0; layout "half" turns pairs (i, i + rotary_dim / 2) of a head's first rotary_dim elements, "interleaved" pairs
    (2 i, 2 i + 1).  Statistics and rotation are fp32, a result is rounded once."""
    if layout not in _LAYOUTS:
        raise ValueError(f"{_NAME}: layout must be one of {sorted(_LAYOUTS)}")
    shape, kshape = q.shape, k.shape
    if len(shape) not in (3, 4) or len(kshape) != len(shape):
        raise RuntimeError(f"{_NAME}: q and k must be [batch, tokens, heads, head_dim] or [tokens, heads, head_dim]")
    if q.dtype not in _DT or k.dtype != q.dtype:
        raise RuntimeError(f"{_NAME}: q and k must be of one type, float32, bfloat16 or float16")
    if not q.is_cuda:
        raise RuntimeError(f"{_NAME}: tensors must be on a HIP device (got {q.device})")
    at, d, by_tensor = q.get_device(), shape[-1], isinstance(positions, torch.Tensor)
    if k.get_device() != at or cos.get_device() != at or sin.get_device() != at or (by_tensor and positions.get_device() != at):
        raise RuntimeError(f"{_NAME}: tensors are on different devices")
    if kshape[-1] != d or kshape[:-2] != shape[:-2]:
        raise RuntimeError(f"{_NAME}: q {list(shape)} and k {list(kshape)} must agree in all but their heads")
    if d % 2 or not 2 <= d <= WFB_QK_MAX_DIM:
        raise ValueError(f"{_NAME}: head_dim ({d}) must be even and at most {WFB_QK_MAX_DIM}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.dim() != 2 or not cos.is_same_size(sin) \
            or not cos.is_contiguous() or not sin.is_contiguous() or 2 * cos.shape[1] > d:
        raise RuntimeError(f"{_NAME}: cos and sin must be contiguous float32 [positions, at most {d // 2}]")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype not in _DT or w.numel() != d or not w.is_contiguous() or w.get_device() != at):
            raise RuntimeError(f"{_NAME}: norm weights must be contiguous floats of {d} elements on {q.device}")
    flat = len(shape) == 3
    if flat:
        q, k = q.unsqueeze(0), k.unsqueeze(0)
    b, t = (1, shape[0]) if flat else shape[:2]
    if by_tensor:
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((t,), (b, t)):
            raise RuntimeError(f"{_NAME}: positions must be int32 or int64 [{t}] or [{b}, {t}]")
        if positions.is_neg():
            positions = positions.resolve_neg()
    else:
        positions = 0 if positions is None else int(positions)
        if cos.shape[1] and not 0 <= positions <= cos.shape[0] - t:
            raise ValueError(f"{_NAME}: positions {positions}..{positions + t - 1} leave tables of {cos.shape[0]} rows")
    if cos.is_neg() or sin.is_neg() or (q_weight is not None and q_weight.is_neg()) or (k_weight is not None and k_weight.is_neg()):
        cos, sin, q_weight, k_weight = (t if t is None else t.resolve_neg() for t in (cos, sin, q_weight, k_weight))
    if forward_ad._current_level >= 0:
        _no_tangents(_NAME, q, k, q_weight, k_weight, cos, sin)
    q, k = _plain(q), _plain(k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or (q_weight is not None and q_weight.requires_grad)
                                    or (k_weight is not None and k_weight.requires_grad)):
        out = _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, float(eps), layout)
    else:
        out = _forward(q, k, cos, sin, positions, q_weight, k_weight, float(eps), layout)
    return (out[0].squeeze(0), out[1].squeeze(0)) if flat else out
