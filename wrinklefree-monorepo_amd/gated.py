"""The gated feed-forward product of two ternary projections, act(gate(x)) * up(x), with its backward pass.

The float block is the reference's FFN (WF/models/ffn.py:10-45, WF = packages/training/src/wrinklefree); each projection
is a BitLinear (WF/models/bitlinear.py:36-113) under the straight-through estimator at lambda = 1, as
:class:`~.bitlinear.BitLinear` trains it: int8 codes of the tokens, shared by both projections, ternary weights, exact
integer sums.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import WFB_ABSMEAN_WS_DOUBLES, WFB_GRAD_WIDE
from .bitlinear import BitLinear, _check_lambda
from .ops import _ACTS, _DT, QK_I2_S, _capturing, _no_tangents, _on, _p, _require_gpu, _stream

_NAME = "gated_bitlinear"


class PackedGated(NamedTuple):
    """Gate over up as they are multiplied with: I2_S uint8 [2 * hidden, k_pad / 4] and their two fp32 scales."""

    qweight: torch.Tensor
    scales: torch.Tensor


def _check_pair(name: str, gate: torch.Tensor, up: torch.Tensor) -> None:
    if gate.dim() != 2 or gate.shape != up.shape or gate.dtype != up.dtype:
        raise RuntimeError(f"{name}: gate and up must be 2D [hidden, in_features] of one shape and type")
    if gate.dtype not in _DT:
        raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, got {gate.dtype}")


def pack_gated(gate_weight: torch.Tensor, up_weight: torch.Tensor) -> PackedGated:
    """Both matrices [hidden, in_features] ternarised and packed, each with its own absmean scale, as
    :func:`pack_ternary_i2s` packs one; in_features is padded to a multiple of 128 with zero weights."""
    name = "pack_gated"
    _check_pair(name, gate_weight, up_weight)
    gate_weight, up_weight = (w.detach().resolve_neg().contiguous() for w in (gate_weight, up_weight))
    dev = _require_gpu(name, gate_weight, up_weight)
    f, k = gate_weight.shape
    if f == 0 or k == 0:
        raise RuntimeError(f"{name}: empty weights")
    kp = (k + QK_I2_S - 1) // QK_I2_S * QK_I2_S
    dt = _DT[gate_weight.dtype]
    qweight = torch.empty((2 * f, kp // 4), dtype=torch.uint8, device=dev)
    scales = torch.empty(2, dtype=torch.float32, device=dev)
    ws = torch.empty(2 * WFB_ABSMEAN_WS_DOUBLES, dtype=torch.float64, device=dev)
    with _on(dev):
        _lib.call("wfb_pack_gated", _p(gate_weight), _p(up_weight), dt, f, k, _p(scales), _p(qweight), _p(ws), _stream(dev))
    return PackedGated(qweight, scales)


def _forward(x2: torch.Tensor, packed: PackedGated, act: str, keep: bool):
    """(h, gate|up or None, codes, a_scale) of the rows x2."""
    n, kb = packed.qweight.shape
    (m, k), dev, dt = x2.shape, x2.device, _DT[x2.dtype]
    f, kp = n // 2, 4 * kb
    q = torch.empty((m, kp), dtype=torch.int8, device=dev)
    a_scale = torch.empty(m, dtype=torch.float32, device=dev)
    h = torch.empty((m, f), dtype=x2.dtype, device=dev)
    gate_up = torch.empty(2 * m * ((f + 63) // 64 * 64), dtype=torch.float32, device=dev) if keep and m else None
    stream, qp, ap = _stream(dev), q.data_ptr(), a_scale.data_ptr()
    with _on(dev):
        _lib.call("wfb_quantize_act_i8", x2.data_ptr(), dt, m, k, k, qp, kp, kp, ap, stream)
        _lib.call("wfb_gated_i2s", packed.qweight.data_ptr(), f, kp, qp, m, kp, ap, packed.scales.data_ptr(), _ACTS[act],
                  h.data_ptr(), dt, _p(gate_up), stream)
    return h, gate_up, q, a_scale


@functools.lru_cache(maxsize=256)
def _grad_workspace(m: int, f: int, k: int, xdt: int, need_x: bool, wdt: int, need_w: bool) -> int:
    size = ctypes.c_int64(0)
    _lib.call("wfb_gated_grad_workspace", m, f, k, xdt, int(need_x), wdt, int(need_w), ctypes.addressof(size))
    return size.value


class _GatedSTE(torch.autograd.Function):
    """Straight through both quantisers, as BitLinear: the forward's value is the kernels', the backward is the gradient of
    act(x~ gate~^T) * (x~ up~^T) at the quantised operands, from the two products that the forward kept."""

    @staticmethod
    def forward(ctx, x2, gate_weight, up_weight, qweight, scales, act, wide):
        h, gate_up, q, a_scale = _forward(x2, PackedGated(qweight, scales), act, True)
        ctx.save_for_backward(gate_up, q, a_scale, qweight, scales)
        ctx.meta = (act, x2.dtype, gate_weight.dtype, x2.shape[1], WFB_GRAD_WIDE if wide else 0)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, gh):
        # (a saved-tensor hook may give them back as other views; no products of no tokens)
        gate_up, q, a_scale, qweight, scales = (t if t is None else t.resolve_neg().contiguous() for t in ctx.saved_tensors)
        act, xdt, wdt, k, wide = ctx.meta
        need_x, need_gate, need_up = ctx.needs_input_grad[:3]
        f, m, dev = qweight.shape[0] // 2, q.shape[0], q.device
        if gh.stride(-1) != 1 or gh.stride(0) < f or gh.is_neg():
            gh = gh.resolve_neg().contiguous()
        need_w = need_gate or need_up
        gx = torch.empty((m, k), dtype=xdt, device=dev) if need_x else None
        gw = torch.empty((2 * f, k), dtype=wdt, device=dev) if need_w else None
        if m == 0:
            return gx, *([gw[:f].zero_(), gw[f:].zero_()] if need_w else [None, None]), None, None, None, None
        gxdt, gwdt = _DT[xdt] | wide, _DT[wdt] | wide
        work = torch.empty(_grad_workspace(m, f, k, gxdt, need_x, gwdt, need_w), dtype=torch.uint8, device=dev)
        kp = 4 * qweight.shape[1]
        with _on(dev):
            _lib.call("wfb_gated_grad", _p(gate_up), _p(gh), _DT[gh.dtype], gh.stride(0) if m > 1 else f, m, f, _ACTS[act],
                      _p(qweight), k, kp, _p(scales), _p(q), kp, _p(a_scale), _p(gx), gxdt, _p(gw), gwdt, _p(work),
                      _stream(dev))
        return gx, gw[:f] if need_gate else None, gw[f:] if need_up else None, None, None, None, None


def gated_bitlinear(
    x: torch.Tensor, gate_weight: Optional[torch.Tensor] = None, up_weight: Optional[torch.Tensor] = None,
    act: str = "silu", packed: Optional[PackedGated] = None, wide_grads: bool = False,
) -> torch.Tensor:
    """act(gate) * up, [..., hidden] in x's type, of x [..., in_features] (fp32, bf16 or fp16) through two ternary
    projections; ``act`` is "silu" or "relu2" (relu squared).  Products and activation are those of
    :func:`bitnet_linear_glu` with ``mid_dtype=float32``, rounded once.

    ``packed`` (of :func:`pack_gated`) saves packing the float weights; without them the call serves only.  With autograd on
    and x or a weight requiring a gradient, the result is differentiable once, straight through both quantisers (in reverse mode;
    tangents of forward mode are refused), and the products are kept for it (8 bytes per token and hidden feature); x, gate_weight and up_weight get gradients in their
    types.  ``packed`` must then be the weights' own pack.  What the activation's backward pass hands to the products is held in
    22 bits of each row's scale for fp32 and fp16 gradients and in 11 for bf16 ones, an eighth of their own rounding;
    ``wide_grads`` holds it in 22 for those too, at twice their products."""
    if act not in _ACTS:
        raise ValueError(f"{_NAME}: act must be one of {sorted(_ACTS)}")
    if (gate_weight is None) != (up_weight is None):
        raise RuntimeError(f"{_NAME}: gate_weight and up_weight go together")
    if gate_weight is None and packed is None:
        raise RuntimeError(f"{_NAME}: weights or their pack are needed")
    if x.dtype not in _DT or x.dim() < 1:
        raise RuntimeError(f"{_NAME}: x must be float32, bfloat16 or float16 with a feature dimension")
    if not x.is_cuda:
        raise RuntimeError(f"{_NAME}: tensors must be on a HIP device (got {x.device})")
    k = x.shape[-1]
    if gate_weight is not None:
        _check_pair(_NAME, gate_weight, up_weight)
        if gate_weight.shape[1] != k:
            raise RuntimeError(f"{_NAME}: x has {k} features, the weights {gate_weight.shape[1]}")
        if gate_weight.get_device() != x.get_device() or up_weight.get_device() != x.get_device():
            raise RuntimeError(f"{_NAME}: weights must be on {x.device}")
    if packed is None:
        packed = pack_gated(gate_weight, up_weight)
    else:
        if packed.scales.is_neg():
            packed = packed._replace(scales=packed.scales.resolve_neg())
        qw, scales = packed
        _require_gpu(_NAME, qw, scales)
        if qw.dtype != torch.uint8 or qw.dim() != 2 or qw.shape[0] % 2 or qw.shape[0] == 0 \
                or scales.dtype != torch.float32 or scales.numel() != 2 or qw.get_device() != x.get_device():
            raise RuntimeError(f"{_NAME}: packed must be uint8 [2 * hidden, k_pad / 4] and fp32 [2] on {x.device}")
        if 4 * qw.shape[1] != (k + QK_I2_S - 1) // QK_I2_S * QK_I2_S:
            raise RuntimeError(f"{_NAME}: x has {k} features, packed rows hold {4 * qw.shape[1]}")
        if gate_weight is not None and gate_weight.shape[0] != qw.shape[0] // 2:
            raise RuntimeError(f"{_NAME}: packed has {qw.shape[0] // 2} hidden features, the weights {gate_weight.shape[0]}")
    f = packed.qweight.shape[0] // 2
    x2 = x if x.dim() == 2 else x.reshape(-1, k) if k else x.new_empty((0, 0))
    if not x2.is_contiguous() or x2.is_neg():
        x2 = x2.resolve_neg().contiguous()
    if forward_ad._current_level >= 0:
        _no_tangents(_NAME, x2, gate_weight, up_weight)
    if torch.is_grad_enabled() and (
            x2.requires_grad or (gate_weight is not None and (gate_weight.requires_grad or up_weight.requires_grad))):
        if gate_weight is None:
            raise RuntimeError(f"{_NAME}: packed weights alone have no float weights to train")
        h = _GatedSTE.apply(x2, gate_weight, up_weight, packed.qweight, packed.scales, act, wide_grads)
    else:
        h = _forward(x2, packed, act, False)[0]
    return h if x.dim() == 2 else h.view(*x.shape[:-1], f)


class GatedBitLinear(nn.Module):
    """act(gate_proj(x)) * up_proj(x) of two bias-free ternary projections, on one set of activation codes; in front of a
    :class:`SubLNBitLinear` it is the feed-forward block of the converted models
    (packages/training/src/wrinklefree/training/stage1.py:93-166).  ``gate_proj`` and ``up_proj`` hold the float weights under
    the names of the linears that they replace; the pack of both is rebuilt when either has changed, and made anew by every
    replay of a captured call (a graph that serves fixed weights saves that with ``gated_bitlinear(x, packed=mod.packed())``,
    the pack kept as long as the graph)."""

    def __init__(self, in_features: int, hidden_features: int, act: str = "silu", device=None, dtype=None,
                 wide_grads: bool = False):
        super().__init__()
        if act not in _ACTS:
            raise ValueError(f"GatedBitLinear: act must be one of {sorted(_ACTS)}")
        self.act = act
        self.wide_grads = wide_grads
        self.gate_proj = BitLinear(in_features, hidden_features, device=device, dtype=dtype)
        self.up_proj = BitLinear(in_features, hidden_features, device=device, dtype=dtype)
        self._packed: Optional[PackedGated] = None
        self._packed_from = None
        self._packed_on = None

    @classmethod
    def from_linears(cls, gate_proj: nn.Linear, up_proj: nn.Linear, act: str = "silu",
                     wide_grads: bool = False) -> "GatedBitLinear":
        """A module that shares the weights of two linears."""
        if gate_proj.bias is not None or up_proj.bias is not None:
            raise RuntimeError("GatedBitLinear: projections with a bias are not gated in one product")
        if gate_proj.weight is None or up_proj.weight is None:
            raise RuntimeError("GatedBitLinear: a projection built from packed weights has no float weight")
        _check_pair("GatedBitLinear", gate_proj.weight, up_proj.weight)
        mod = cls(gate_proj.in_features, gate_proj.out_features, act, device="meta", dtype=gate_proj.weight.dtype,
                  wide_grads=wide_grads)
        mod.gate_proj.weight, mod.up_proj.weight = gate_proj.weight, up_proj.weight
        return mod

    def packed(self) -> PackedGated:
        """The weights' pack, rebuilt if a weight changed since the last one, and ready for the current stream.  While that
        stream is captured, a new pack that belongs to the graph, whose replays make it of what the weights hold then."""
        gate, up = self.gate_proj.weight, self.up_proj.weight
        if _capturing(gate.device):
            return pack_gated(gate, up)
        stamp = (self.gate_proj._weight_stamp(), self.up_proj._weight_stamp())
        if self._packed is None or self._packed_from != stamp:
            self._packed = pack_gated(gate, up)
            self._packed_from = stamp
            stream = torch.cuda.current_stream(gate.device)
            self._packed_on = (stream.cuda_stream, stream.record_event())
        elif self._packed_on[0] != _stream(gate.device):
            # made on another stream: wait for it there, and keep its memory until this stream has read it
            stream = torch.cuda.current_stream(gate.device)
            stream.wait_event(self._packed_on[1])
            for t in self._packed:
                t.record_stream(stream)
        return self._packed

    def pack(self) -> "GatedBitLinear":
        """Rebuild the pack whether or not the weights show a change (those that a replayed graph steps do not).  Within a
        capture there is nothing to rebuild: its calls pack for themselves."""
        if not _capturing(self.gate_proj.weight.device):
            self._packed = None
            self.packed()
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _check_lambda("GatedBitLinear")
        return gated_bitlinear(x, self.gate_proj.weight, self.up_proj.weight, self.act, self.packed(), self.wide_grads)

    def _apply(self, fn, recurse=True):
        # (a weight that is cast and cast back may lie where it lay, its version counter unmoved)
        self._packed = None
        return super()._apply(fn, recurse)

    def __getstate__(self):
        return {**self.__dict__, "_packed": None, "_packed_from": None, "_packed_on": None}

    def extra_repr(self) -> str:
        return f"act={self.act}"
