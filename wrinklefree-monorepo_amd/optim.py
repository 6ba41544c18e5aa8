"""AdamW over many tensors in one launch, with states in fp32 or in 8 bits.

One kernel walks every tensor of a group, and the states of a group lie in one flat array each, so that a state in 8 bits
(codes and one scale for 256 elements, about a quarter of the bytes) needs no bookkeeping per tensor.  The arithmetic is in
csrc/adamw.hip's first lines.  Weights change in place and their version counters with them, so that a BitLinear over them
repacks.
"""

from __future__ import annotations

from array import array
from itertools import chain
from operator import attrgetter
from typing import Iterable, List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import WFB_ADAMW_BLOCK, WFB_ADAMW_SCALARS
from .ops import _DT, _capturing, _on, _stream


_dtype_of = attrgetter("dtype")


class AdamWState(NamedTuple):
    """The moments of a list of tensors, flat: tensor i starts at a multiple of 256 elements, behind tensor i - 1.  In 32
    bits ``m`` and ``v`` are fp32 and the scales None; in 8 bits int8 and uint8 codes with fp32 scales, one for each 256: a
    moment at code n rises faster and falls slower by 1 / (2 n) of its way (csrc/adamw.hip's first lines).  Elements behind a
    tensor's end are 0."""

    m: torch.Tensor
    v: torch.Tensor
    m_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None


def _blocks(n: int) -> int:
    return (n + WFB_ADAMW_BLOCK - 1) // WFB_ADAMW_BLOCK


def adamw_state(params: Iterable[torch.Tensor], bits: int = 32) -> AdamWState:
    """A zero state in 32 or 8 bits for these tensors, on their device."""
    params = list(params)
    if bits not in (8, 32):
        raise ValueError(f"adamw_state: states have 32 or 8 bits, not {bits}")
    if not params:
        raise ValueError("adamw_state: no tensors")
    blocks, dev = sum(_blocks(p.numel()) for p in params), params[0].device
    n = blocks * WFB_ADAMW_BLOCK
    if bits == 32:
        return AdamWState(*(torch.zeros(n, dtype=torch.float32, device=dev) for _ in range(2)))
    return AdamWState(torch.zeros(n, dtype=torch.int8, device=dev), torch.zeros(n, dtype=torch.uint8, device=dev),
                      *(torch.zeros(blocks, dtype=torch.float32, device=dev) for _ in range(2)))


def _bits_of(name: str, state: AdamWState) -> int:
    """32 or 8, by types and sizes."""
    m, v, ms, vs = state
    n = m.numel()
    if m.dtype == v.dtype == torch.float32 and ms is None and vs is None:
        bits = 32
    elif m.dtype == torch.int8 and v.dtype == torch.uint8 and ms is not None and vs is not None:
        bits = 8
        if ms.dtype != torch.float32 or vs.dtype != torch.float32 or ms.numel() * WFB_ADAMW_BLOCK != n \
                or vs.numel() * WFB_ADAMW_BLOCK != n:
            raise RuntimeError(f"{name}: scales must be fp32, one for each {WFB_ADAMW_BLOCK} elements")
    else:
        raise RuntimeError(f"{name}: a state is fp32 m and v, or int8 m and uint8 v with their scales")
    if v.numel() != n or n % WFB_ADAMW_BLOCK:
        raise RuntimeError(f"{name}: m and v must have as many elements, a multiple of {WFB_ADAMW_BLOCK}")
    return bits


def _check_state(name: str, state: AdamWState) -> Tuple[int, torch.device]:
    """(bits, device) of a state."""
    m = state.m
    if m.device.type != "cuda":
        raise RuntimeError(f"{name}: the state must be on a HIP device (got {m.device})")
    bits = _bits_of(name, state)
    for t in state if bits == 8 else state[:2]:
        if not t.is_contiguous() or t.is_neg() or t.device != m.device:
            raise RuntimeError(f"{name}: the state must be contiguous and on one device")
    return bits, m.device


@torch.no_grad()
def adamw_step(
    params: Sequence[torch.Tensor], grads: Sequence[Optional[torch.Tensor]], state: AdamWState,
    step: Union[int, torch.Tensor], lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8, weight_decay: float = 1e-2,
) -> None:
    """AdamW step number ``step`` (from 1) of every tensor that has a gradient (None: left as it is), in place.

    params fp32, bf16 or fp16 and their gradients, each of any of these types, contiguous, on one device; ``state`` of
    :func:`adamw_state` for the same list.  Decoupled weight decay; arithmetic in fp32, parameters rounded once.
    For a captured graph ``step`` is an int64 device tensor of one element, which the caller counts up, and ``lr`` may be an
    fp32 one; a replay changes no version counters, so packs that modules keep outside the graph are renewed by their
    ``pack()``.  No two tensors may share memory.  A gradient that is not finite spoils its own element, and in 8 bits the
    moments of its block of 256.  One whose square fp32 does not hold (from 1.8e19) has v = infinity: its element only decays
    from then on; in 8 bits sqrt(v) is held as 2^63, and its block takes small steps until that has decayed."""
    name = "adamw_step"
    bits, dev = _check_state(name, state)
    if len(params) != len(grads):
        raise RuntimeError(f"{name}: {len(params)} tensors, {len(grads)} gradients")
    every, have = list(params), list(grads)
    if any([g is None for g in have]):
        pairs = [(p, g) for p, g in zip(every, have) if g is not None]
        live, gs = [p for p, _ in pairs], [g for _, g in pairs]
    else:
        live, gs = every, have
    # (a few calls a tensor are what a step over small tensors costs, so they are made by map over the bound functions: 121
    # norms 138 us with attributes compared one by one, 82 so)
    tensor, at = torch.Tensor, dev.index
    if not all(map(tensor.is_same_size, live, gs)) or not {at}.issuperset(map(tensor.get_device, chain(live, gs))):
        raise RuntimeError(f"{name}: a gradient has its tensor's shape, both are on {dev}")
    if not all(map(tensor.is_contiguous, live)) or any(map(tensor.is_neg, live)):
        raise RuntimeError(f"{name}: tensors must be contiguous")
    if not all(map(tensor.is_contiguous, gs)) or any(map(tensor.is_neg, gs)):
        gs = [g.resolve_neg().contiguous() for g in gs]  # (copies live until the launch)
    kinds = set(zip(map(_dtype_of, live), map(_dtype_of, gs)))
    for pdt, gdt in kinds:
        if pdt not in _DT or gdt not in _DT:
            raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, got {pdt} and {gdt}")
    sizes, ptrs, gptrs = (list(map(f, x)) for f, x in ((tensor.numel, every), (tensor.data_ptr, live), (tensor.data_ptr, gs)))
    if not (all(ptrs) and all(gptrs)) and any(t.numel() and not t.data_ptr() for t in chain(live, gs)):
        raise RuntimeError(f"{name}: a tensor without memory of its own (of a wrapping class): step what it wraps")
    if len(set(ptrs)) != len(ptrs) and len({p for p in ptrs if p}) != sum(p != 0 for p in ptrs):
        raise RuntimeError(f"{name}: a tensor is given twice")
    if len(live) != len(every):  # a null gradient: the tensor is passed over
        it = iter(zip(ptrs, gptrs))
        ptrs, gptrs = zip(*[(0, 0) if g is None else next(it) for g in have])
    tables = []
    for pdt, gdt in kinds:
        wanted = gptrs
        if len(kinds) > 1:
            wanted = [q if g is not None and p.dtype == pdt and g.dtype == gdt else 0 for p, g, q in zip(every, have, gptrs)]
        # rows of wfb_adamw_tensor
        tables.append((_DT[pdt], _DT[gdt], array("q", chain.from_iterable(zip(ptrs, wanted, sizes)))))
    if not kinds and sum(map(_blocks, sizes)) * WFB_ADAMW_BLOCK != state.m.numel():  # (else the C entry's check)
        raise RuntimeError(f"{name}: the state's {state.m.numel()} elements are not these tensors'")
    step_dev = lr_dev = scalars = None
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != dev:
            raise RuntimeError(f"{name}: a step tensor must be one int64 element on {dev}")
        step = step.resolve_neg()
        step_dev = step.data_ptr()
        scalars = torch.empty(WFB_ADAMW_SCALARS, dtype=torch.float32, device=dev)
    if isinstance(lr, torch.Tensor):
        if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != dev or step_dev is None:
            raise RuntimeError(f"{name}: a lr tensor must be one fp32 element on {dev} and goes with a step tensor")
        lr = lr.resolve_neg()
        lr_dev = lr.data_ptr()
    m, v, ms, vs = state
    with _on(dev):
        for pdt, gdt, rows in tables:
            _lib.call("wfb_adamw_step", rows.buffer_info()[0], len(rows) // 3, pdt, gdt, m.data_ptr(),
                      v.data_ptr(), None if ms is None else ms.data_ptr(), None if vs is None else vs.data_ptr(),
                      m.numel(), bits, 0.0 if lr_dev else float(lr), float(betas[0]), float(betas[1]), float(eps),
                      float(weight_decay), 0 if step_dev else int(step), step_dev, lr_dev, None if scalars is None else scalars.data_ptr(), _stream(dev))
    if live:
        torch.autograd.graph.increment_version(live)


def adamw_state_values(state: AdamWState) -> Tuple[torch.Tensor, torch.Tensor]:
    """(m, v) fp32 of a state, flat: of 32 bits its own arrays, of 8 bits new ones with what the codes stand for."""
    name = "adamw_state_values"
    bits, dev = _check_state(name, state)
    if bits == 32:
        return state.m, state.v
    m, v = (torch.empty(state.m.numel(), dtype=torch.float32, device=dev) for _ in range(2))
    with _on(dev):
        _lib.call("wfb_adamw_values", state.m.data_ptr(), state.v.data_ptr(), state.m_scale.data_ptr(),
                  state.v_scale.data_ptr(), m.numel(), m.data_ptr(), v.data_ptr(), _stream(dev))
    return m, v


class AdamW(torch.optim.Optimizer):
    """The step of ``torch.optim.AdamW`` over :func:`adamw_step`, with its ``lr``, ``betas``, ``eps`` and ``weight_decay`` (no
    ``amsgrad``, ``maximize`` or ``foreach``) and states of ``state_bits`` 32 or 8.

    A group has one flat state (:meth:`group_state`; ``state``, torch's dictionary of each parameter's, stays empty); its tensors
    are of one device.  A tensor's steps are counted from its first gradient on and only where it has one, as torch counts
    them; tensors of one count step in one call.  With ``capturable`` the counts lie on the device and :meth:`step` can be
    captured into a graph (``lr`` may then be an fp32 device tensor), behind a step that made the state with gradients for
    the same tensors.  The state dict holds the states as they are."""

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32, capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 32 or 8, not {state_bits}")
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"AdamW: bad lr {lr}")
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("AdamW: a lr tensor needs capturable=True")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"AdamW: bad betas {betas}, eps {eps} or weight_decay {weight_decay}")
        self._flat: List[Optional[dict]] = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        self._flat.append(None)

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "_flat": self._flat}

    def group_state(self, index: int = 0) -> Optional[AdamWState]:
        """The state of a group, None before its first step."""
        return None if self._flat[index] is None else self._flat[index]["state"]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for i, group in enumerate(self.param_groups):
            params = group["params"]
            grads = [p.grad for p in params]
            have = [g is not None for g in grads]
            if not any(have):
                continue
            if any([g is not None and g.is_sparse for g in grads]):
                raise RuntimeError("AdamW: sparse gradients are not supported")
            flat = self._flat[i]
            if _capturing(params[0].device):
                if not group["capturable"]:
                    raise RuntimeError("AdamW: a step that is captured needs capturable=True")
                if flat is None:
                    raise RuntimeError("AdamW: the first step, which makes the state, comes before the capture")
            if flat is None:
                count = torch.zeros(1, dtype=torch.int64, device=params[0].device) if group["capturable"] else 0
                flat = {"state": adamw_state(params, group["state_bits"]), "steps": [(count, list(range(len(params))))]}
            if len(flat["steps"]) > 1 or not all(have):
                flat["steps"] = self._cohorts(flat["steps"], have)
            for k, (count, of) in enumerate(flat["steps"]):
                if not have[of[0]]:
                    continue
                if len(of) < len(params):
                    mine = set(of)
                    wanted = [g if j in mine else None for j, g in enumerate(grads)]
                else:
                    wanted = grads
                args = (group["lr"], group["betas"], group["eps"], group["weight_decay"])
                if group["capturable"]:
                    count += 1
                    try:
                        adamw_step(params, wanted, flat["state"], count, *args)
                    except Exception:
                        count -= 1  # (refused, not stepped)
                        raise
                else:
                    adamw_step(params, wanted, flat["state"], count + 1, *args)
                    flat["steps"][k] = (count + 1, of)
            self._flat[i] = flat
        return loss

    @staticmethod
    def _cohorts(steps, have: List[bool]) -> List[tuple]:
        """(count, tensors) such that the tensors of one count all step now or all do not; equal counts on the host as one."""
        out = []
        for count, of in steps:
            parts = [part for part in ([j for j in of if have[j]], [j for j in of if not have[j]]) if part]
            if len(parts) == 2 and isinstance(count, torch.Tensor) and _capturing(count.device):
                raise RuntimeError("AdamW: a captured step needs gradients for the tensors that stepped together before")
            for n, part in enumerate(parts):
                out.append((count.clone() if n and isinstance(count, torch.Tensor) else count, part))
        if out and not isinstance(out[0][0], torch.Tensor):
            joined: dict = {}
            for count, part in out:
                joined.setdefault((count, have[part[0]]), []).extend(part)
            out = [(count, sorted(part)) for (count, _), part in joined.items()]
        return out

    def state_dict(self) -> dict:
        d = super().state_dict()
        d["flat"] = [None if f is None else {"state": tuple(f["state"]), "steps": [(c, list(of)) for c, of in f["steps"]]}
                     for f in self._flat]
        return d

    def load_state_dict(self, state_dict: dict) -> None:
        flat, groups = state_dict.get("flat"), self.param_groups
        if flat is None or len(flat) != len(groups) or len(state_dict["param_groups"]) != len(groups):
            raise ValueError("AdamW: the state dict is not this optimizer's, with one state for each group")
        made = []
        for group, saved, f in zip(groups, state_dict["param_groups"], flat):  # all of it, before anything changes
            if f is None:
                made.append(None)
                continue
            state, n = AdamWState(*f["state"]), len(group["params"])
            need = sum(_blocks(p.numel()) for p in group["params"]) * WFB_ADAMW_BLOCK
            if state.m.numel() != need:
                raise ValueError(f"AdamW: the state has {state.m.numel()} elements, the group's tensors take {need}")
            if _bits_of("AdamW", state) != saved["state_bits"]:
                raise ValueError(f"AdamW: the state is not one of {saved['state_bits']} bits")
            steps = f["steps"] if "steps" in f else [(f["step"], range(n))]
            if sorted(j for _, of in steps for j in of) != list(range(n)):
                raise ValueError(f"AdamW: the counts of steps are not of {n} tensors")
            dev = group["params"][0].device
            state = AdamWState(*(None if t is None else t.detach().to(dev, copy=True) for t in state))
            counts = [torch.as_tensor(c, dtype=torch.int64).reshape(1).to(dev, copy=True) if saved["capturable"] else int(c)
                      for c, _ in steps]
            made.append({"state": state, "steps": [(c, list(of)) for c, (_, of) in zip(counts, steps)]})
        super().load_state_dict({k: v for k, v in state_dict.items() if k != "flat"})
        self._flat = made
