"""Expert routing: token slots sorted by expert, rows moved there and back.

The sort beside DeviceRadixSort that a mixture-of-experts layer needs (no
reference counterpart).  A layer calls, on one launch and with one plan:

    plan = device_expert_plan(launch, tokens, top_k, experts, align)  # once
    device_expert_sort(launch, expert_ids, plan)            # ids (tokens, top_k)
    device_expert_gather(launch, x, plan, rows)             # into expert order
    ...the experts' products over rows[offsets[e] : offsets[e + 1]]...
    device_expert_combine(launch, expert_out, weights, plan, y)

and, for the gradients, device_expert_combine_backward and
device_expert_gather_backward with the same plan.  All memory is the caller's,
every call is asynchronous on the launch's stream and reads nothing back, so a
step can be captured into a CUDA graph.  Ids outside 0..experts-1 are dropped
slots: they take no row, add nothing and get no gradient.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .cub import ContextMismatch, Launch
from .errors import BadArgument, LengthMismatch, raise_for

REAL_TYPES = {
    torch.float32: _lib.RSORT_F32,
    torch.float16: _lib.RSORT_F16,
    torch.bfloat16: _lib.RSORT_BF16,
}
ID_TYPES = {torch.int32: _lib.RSORT_I32, torch.int64: _lib.RSORT_I64}


def real_code(dtype: torch.dtype) -> int:
    code = REAL_TYPES.get(dtype)
    if code is None:
        raise BadArgument(f"{dtype} is not a row type (float32, float16 or bfloat16)")
    return code


def expert_rows(tokens: int, top_k: int, experts: int, align: int = 1) -> int:
    """Rows that hold every outcome of a sort of tokens x top_k slots."""
    rows = 0
    # what a C size would wrap is out of range too
    sized = (0 <= tokens <= _lib.MAX_EXPERT_SLOTS and 0 <= top_k and
             tokens * top_k <= _lib.MAX_EXPERT_SLOTS and 1 <= experts <= _lib.MAX_EXPERTS and
             1 <= align <= _lib.MAX_EXPERT_ALIGN)
    if sized:
        rows = _lib.lib().rsort_expert_rows(tokens * top_k, experts, align)
    if not sized or (rows == 0 and tokens * top_k):
        raise BadArgument(f"no expert rows for {tokens} x {top_k} slots, {experts} experts "
                          f"(1..{_lib.MAX_EXPERTS}), align {align} (1..{_lib.MAX_EXPERT_ALIGN})")
    return rows


@dataclass(frozen=True, eq=False)
class ExpertPlan:
    """Where every slot goes, filled by device_expert_sort.

    row_of_slot (tokens, top_k): a slot's row, -1 when dropped; slot_of_row
    (rows): a row's slot, -1 in padding; offsets (experts + 1): every expert's
    first row; counts (experts): its slots.  All int32 on the device; scratch is
    the sort's, uint8.  The calls take the arrays' addresses from here, so a
    plan keeps the arrays that it was made with."""
    tokens: int
    top_k: int
    experts: int
    align: int
    rows: int
    row_of_slot: torch.Tensor
    slot_of_row: torch.Tensor
    offsets: torch.Tensor
    counts: torch.Tensor
    scratch: torch.Tensor

    def __post_init__(self):
        for name, t, shape in (("row_of_slot", self.row_of_slot, (self.tokens, self.top_k)),
                               ("slot_of_row", self.slot_of_row, (self.rows,)),
                               ("offsets", self.offsets, (self.experts + 1,)),
                               ("counts", self.counts, (self.experts,))):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise BadArgument(f"expert plan {name} must be contiguous int32")
            if t.shape != shape:
                raise LengthMismatch("expert plan " + name, math.prod(shape), t.numel())
        if self.scratch.dtype != torch.uint8 or not self.scratch.is_contiguous():
            raise BadArgument("expert plan scratch must be contiguous uint8")
        for t in (self.slot_of_row, self.offsets, self.counts, self.scratch):
            if t.device != self.row_of_slot.device:
                raise ContextMismatch(f"expert plan on {self.row_of_slot.device} and {t.device}")
        args = _lib.ExpertPlanArgs(
            self.row_of_slot.data_ptr(), self.offsets.data_ptr(), self.counts.data_ptr(),
            self.tokens, self.top_k, self.experts, self.rows)
        sort_args = (self.tokens * self.top_k, self.experts, self.align,
                     self.row_of_slot.data_ptr(), self.slot_of_row.data_ptr(), self.rows,
                     self.offsets.data_ptr(), self.counts.data_ptr(),
                     self.scratch.data_ptr(), self.scratch.numel())
        for name, value in (("_args", args), ("args", ctypes.byref(args)),
                            ("sort_args", sort_args), ("slots", (self.tokens, self.top_k))):
            object.__setattr__(self, name, value)


def device_expert_plan(launch: Launch, tokens: int, top_k: int, experts: int,
                       align: int = 1) -> ExpertPlan:
    """The plan and the sort's scratch for tokens x top_k slots, with every
    expert's segment padded to a multiple of `align` rows.  Reused from call to
    call, one call at a time."""
    if tokens < 0 or not 1 <= top_k <= _lib.MAX_EXPERTS:
        raise BadArgument(f"{tokens} tokens, top_k {top_k} (1..{_lib.MAX_EXPERTS})")
    rows = expert_rows(tokens, top_k, experts, align)
    lib = _lib.lib()
    nbytes = lib.rsort_expert_sort_scratch_bytes(tokens * top_k, experts)
    # One allocation for all arrays, each on 16 bytes.
    sizes = (nbytes // 4, tokens * top_k, rows, experts + 1, experts)
    starts, end = [], 0
    for n in sizes:
        starts.append(end)
        end += (n + 3) // 4 * 4
    with torch.cuda.stream(launch.stream):
        block = torch.full((end,), -1, dtype=torch.int32, device=launch.device)
    scratch, row_of_slot, *rest = (block[i:i + n] for i, n in zip(starts, sizes))
    return ExpertPlan(tokens, top_k, experts, align, rows, row_of_slot.view(tokens, top_k), *rest,
                      scratch.view(torch.uint8))


def _on(launch: Launch, *tensors: Optional[torch.Tensor]) -> None:
    """Rows may be strided, so only the device is checked here."""
    device = launch.device
    for t in tensors:
        if t is not None and t.device != device:
            raise ContextMismatch(f"tensor on {t.device}, launch on {device}")


def call(launch: Launch, entry, *args) -> None:
    """Calls a C entry on the launch's stream, with the launch's device as the
    current one (kernels launch there)."""
    if torch.cuda.current_device() == launch.device.index:
        status = entry(*args, launch.stream.cuda_stream)
    else:
        with torch.cuda.device(launch.device):
            status = entry(*args, launch.stream.cuda_stream)
    if status:
        raise_for(status)


def _rows(role: str, t: torch.Tensor, count: int, width: int, at_least: bool = False) -> int:
    """Row stride of a (count, width) tensor whose elements of a row are neighbours."""
    shape = t.shape
    if len(shape) == 2 and t.is_contiguous():
        stride = shape[1]
    elif len(shape) == 2 and (t.numel() == 0 or shape[1] == 1 or t.stride(1) == 1):
        stride = t.stride(0)
    else:
        raise BadArgument(f"{role} must be 2-D with neighbouring elements in a row")
    n, w = shape
    if n < count or (n > count and not at_least):
        raise LengthMismatch(role, count, n)
    if w != width:
        raise LengthMismatch(role + " width", width, w)
    return stride


def _slots(role: str, t: torch.Tensor, plan: ExpertPlan) -> None:
    """One entry a slot in the slots' order: (tokens, top_k), with any leading
    dimensions for the tokens, or flat; of any shape when top_k is 1."""
    shape = t.shape
    if shape == plan.slots and t.is_contiguous():
        return
    if t.numel() != plan.tokens * plan.top_k:
        raise LengthMismatch(role, plan.tokens * plan.top_k, t.numel())
    if len(shape) > 1 and shape[-1] != plan.top_k > 1:
        raise LengthMismatch(role + " of a token", plan.top_k, shape[-1])
    if not t.is_contiguous():
        raise BadArgument(f"{role} must be contiguous")


def _weights(t: torch.Tensor, plan: ExpertPlan, role: str = "expert weights") -> int:
    code = real_code(t.dtype)
    _slots(role, t, plan)
    return code


def device_expert_sort(launch: Launch, expert_ids: torch.Tensor, plan: ExpertPlan) -> None:
    """Sort the slots of expert_ids (tokens, top_k; int32 or int64) stably by
    expert into the plan.  Ids and weights may also be (batch, length, top_k) or
    flat, as long as their slots are in that order."""
    _on(launch, expert_ids, plan.row_of_slot)
    code = ID_TYPES.get(expert_ids.dtype)
    if code is None:
        raise BadArgument(f"expert ids of {expert_ids.dtype} (int32 or int64)")
    _slots("expert ids", expert_ids, plan)
    call(launch, _lib.lib().rsort_expert_sort, code, expert_ids.data_ptr(), *plan.sort_args)


def device_expert_gather(launch: Launch, x: torch.Tensor, plan: ExpertPlan, rows: torch.Tensor,
                         zero_padding: bool = True) -> None:
    """rows[plan.row_of_slot[t, k]] = x[t] for every kept slot.  x (tokens,
    width) and rows (at least plan.rows, width) of one dtype, any element type.
    zero_padding: the segments' padding rows become zeros; rows behind the last
    segment are left as they are."""
    _on(launch, x, rows, plan.row_of_slot)
    if x.dtype != rows.dtype:
        raise BadArgument(f"tokens of {x.dtype}, expert rows of {rows.dtype}")
    size = x.element_size()
    x_stride = _rows("tokens", x, plan.tokens, rows.shape[-1])
    rows_stride = _rows("expert rows", rows, plan.rows, rows.shape[-1], at_least=True)
    call(launch, _lib.lib().rsort_expert_gather, plan.args, x.data_ptr(), x_stride * size,
         rows.data_ptr(), rows_stride * size, rows.shape[1] * size, int(zero_padding))


def _combine(launch: Launch, rows, weights, plan: ExpertPlan, out) -> None:
    _on(launch, rows, weights, out, plan.row_of_slot)
    code = real_code(rows.dtype)
    if out.dtype != rows.dtype:
        raise BadArgument(f"expert rows of {rows.dtype}, output of {out.dtype}")
    width = out.shape[-1]
    rows_stride = _rows("expert rows", rows, plan.rows, width, at_least=True)
    out_stride = _rows("expert output", out, plan.tokens, width)
    wcode = code if weights is None else _weights(weights, plan)
    call(launch, _lib.lib().rsort_expert_combine, plan.args, code, rows.data_ptr(), rows_stride,
         None if weights is None else weights.data_ptr(), wcode, out.data_ptr(), out_stride, width)


def device_expert_combine(launch: Launch, rows: torch.Tensor, weights: torch.Tensor,
                          plan: ExpertPlan, out: torch.Tensor) -> None:
    """out[t] = sum over k of weights[t, k] * rows[plan.row_of_slot[t, k]], in
    fp32 in the order of k, rounded once; 0 for a token without kept slots."""
    if weights is None:
        raise BadArgument("expert weights are missing")
    _combine(launch, rows, weights, plan, out)


def device_expert_gather_backward(launch: Launch, grad_rows: torch.Tensor, plan: ExpertPlan,
                                  grad_x: torch.Tensor) -> None:
    """grad_x[t] = sum over k of grad_rows[plan.row_of_slot[t, k]]: the
    gradient of device_expert_gather."""
    _combine(launch, grad_rows, None, plan, grad_x)


def device_expert_combine_backward(launch: Launch, grad_out: torch.Tensor, rows: torch.Tensor,
                                   weights: torch.Tensor, plan: ExpertPlan,
                                   grad_rows: Optional[torch.Tensor],
                                   grad_weights: Optional[torch.Tensor],
                                   zero_padding: bool = True) -> None:
    """The gradients of device_expert_combine from grad_out (tokens, width):
    grad_rows[r] = weight * grad_out[t] at the slot's row (padding rows become
    zeros with zero_padding), grad_weights[t, k] = the dot product of
    grad_out[t] and the slot's row, 0 for dropped slots.  Either output may be
    None; grad_weights has the weights' dtype."""
    _on(launch, grad_out, rows, weights, grad_rows, grad_weights, plan.row_of_slot)
    code = real_code(grad_out.dtype)
    width = grad_out.shape[-1]
    if rows.dtype != grad_out.dtype or (grad_rows is not None and grad_rows.dtype != rows.dtype):
        raise BadArgument("expert rows and gradients differ in type")
    grad_out_stride = _rows("expert output gradient", grad_out, plan.tokens, width)
    rows_stride = _rows("expert rows", rows, plan.rows, width, at_least=True)
    grad_rows_stride = 0
    if grad_rows is not None:
        grad_rows_stride = _rows("expert row gradients", grad_rows, plan.rows, width,
                                 at_least=True)
    wcode = _weights(weights, plan)
    if grad_weights is not None and _weights(grad_weights, plan, "weight gradients") != wcode:
        raise BadArgument("weight gradients differ from the weights in type")
    call(launch, _lib.lib().rsort_expert_combine_backward, plan.args, code, grad_out.data_ptr(),
         grad_out_stride, rows.data_ptr(), rows_stride, weights.data_ptr(), wcode,
         None if grad_rows is None else grad_rows.data_ptr(), grad_rows_stride,
         None if grad_weights is None else grad_weights.data_ptr(), width, int(zero_padding))
