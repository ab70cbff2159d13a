"""CPU tests of the expert routing's sizing and refusals: every call here is
sized or rejected on the host before any device work."""
import ctypes
import dataclasses

import pytest
import torch

from rccl_b200 import _lib, cub, experts
from rccl_b200.errors import BadArgument, LengthMismatch

L = _lib.lib()


class Stream:
    cuda_stream = 0


CPU = cub.Launch(torch.device("cpu"), Stream())  # refused calls never reach a device


def plan_on_cpu(tokens=4, top_k=2, count=3, align=1):
    rows = experts.expert_rows(tokens, top_k, count, align)
    i32 = dict(dtype=torch.int32)
    return experts.ExpertPlan(tokens, top_k, count, align, rows, torch.zeros(tokens, top_k, **i32),
                              torch.zeros(rows, **i32), torch.zeros(count + 1, **i32),
                              torch.zeros(count, **i32), torch.zeros(64, dtype=torch.uint8))


@pytest.mark.parametrize("slots,count,align,rows", [
    (0, 4, 16, 0), (1, 4, 16, 16), (7, 4, 1, 7), (8, 4, 8, 32), (100, 3, 8, 120),
    (2, 1024, 128, 256), (2**31 - 1, 1024, 1, 2**31 - 1)])
def test_rows_hold_every_outcome(slots, count, align, rows):
    assert L.rsort_expert_rows(slots, count, align) == rows


def test_unsupported_sizes_have_no_rows():
    for args in [(8, 0, 1), (8, 1025, 1), (8, 4, 0), (8, 4, 65537), (2**31, 4, 1),
                 (2**31 - 1, 4, 2)]:
        assert L.rsort_expert_rows(*args) == 0
    with pytest.raises(BadArgument):
        experts.expert_rows(4, 2, 0)
    assert L.rsort_expert_sort_scratch_bytes(8, 0) == 0
    assert L.rsort_expert_sort_scratch_bytes(2**31, 8) == 0
    assert L.rsort_expert_sort_scratch_bytes(0, 8) > 0


def sort_status(**kw):
    a = dict(t=_lib.RSORT_I32, ids=0x1000, n=8, count=4, align=1, row=0x2000, slot=0x3000, rows=8,
             offsets=0x4000, counts=0x5000, scratch=0x6000, bytes=1 << 20)
    a.update(kw)
    return L.rsort_expert_sort(a["t"], a["ids"], a["n"], a["count"], a["align"], a["row"],
                               a["slot"], a["rows"], a["offsets"], a["counts"], a["scratch"],
                               a["bytes"], None)


@pytest.mark.parametrize("change,status", [
    (dict(t=_lib.RSORT_U32), _lib.RSORT_BAD_ARGUMENT),
    (dict(count=0), _lib.RSORT_BAD_ARGUMENT),
    (dict(count=1025), _lib.RSORT_BAD_ARGUMENT),
    (dict(align=0), _lib.RSORT_BAD_ARGUMENT),
    (dict(align=65537), _lib.RSORT_BAD_ARGUMENT),
    (dict(n=2**31, rows=2**31), _lib.RSORT_SIZE_OVERFLOW),
    (dict(rows=7), _lib.RSORT_WORKSPACE_TOO_SMALL),
    (dict(align=16, rows=63), _lib.RSORT_WORKSPACE_TOO_SMALL),
    (dict(ids=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(row=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(slot=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(offsets=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(counts=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(scratch=None), _lib.RSORT_WORKSPACE_TOO_SMALL),
    (dict(bytes=8), _lib.RSORT_WORKSPACE_TOO_SMALL),
    (dict(ids=0x1002), _lib.RSORT_BAD_ARGUMENT),
    (dict(t=_lib.RSORT_I64, ids=0x1004), _lib.RSORT_BAD_ARGUMENT),
    (dict(row=0x2001), _lib.RSORT_BAD_ARGUMENT),
    (dict(scratch=0x6002), _lib.RSORT_BAD_ARGUMENT),
    (dict(row=0x1000), _lib.RSORT_BAD_ARGUMENT),           # over the ids
    (dict(slot=0x1010), _lib.RSORT_BAD_ARGUMENT),
    (dict(slot=0x2010), _lib.RSORT_BAD_ARGUMENT),          # over one another
    (dict(counts=0x4008), _lib.RSORT_BAD_ARGUMENT),
    (dict(scratch=0x3010), _lib.RSORT_BAD_ARGUMENT),
    (dict(scratch=0x6008), _lib.RSORT_BAD_ARGUMENT)])
def test_sort_refusals(change, status):
    assert sort_status(**change) == status
    assert _lib.last_error().status == status


def plan_args(**kw):
    a = dict(row_of_slot=0x1000, offsets=0x2000, counts=0x3000, tokens=4, top_k=2, experts=3,
             nrows=8)
    a.update(kw)
    return ctypes.byref(_lib.ExpertPlanArgs(**a))


@pytest.mark.parametrize("change,status", [
    (dict(row_of_slot=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(offsets=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(counts=None), _lib.RSORT_BAD_ARGUMENT),
    (dict(experts=0), _lib.RSORT_BAD_ARGUMENT),
    (dict(experts=1025), _lib.RSORT_BAD_ARGUMENT),
    (dict(top_k=0), _lib.RSORT_BAD_ARGUMENT),
    (dict(top_k=1025), _lib.RSORT_BAD_ARGUMENT),
    (dict(tokens=2**31), _lib.RSORT_SIZE_OVERFLOW),
    (dict(nrows=2**31), _lib.RSORT_SIZE_OVERFLOW),
    (dict(offsets=0x2002), _lib.RSORT_BAD_ARGUMENT)])
def test_plan_refusals(change, status):
    plan = plan_args(**change)
    assert L.rsort_expert_gather(plan, 0x10000, 64, 0x20000, 64, 64, 1, None) == status
    assert L.rsort_expert_combine(plan, _lib.RSORT_F32, 0x10000, 16, 0x20000, _lib.RSORT_F32,
                                  0x30000, 16, 16, None) == status
    assert L.rsort_expert_combine_backward(plan, _lib.RSORT_F32, 0x10000, 16, 0x20000, 16, 0x30000,
                                           _lib.RSORT_F32, 0x40000, 16, 0x50000, 16, 1,
                                           None) == status


def test_null_plan_is_refused():
    assert L.rsort_expert_gather(None, 0x10000, 64, 0x20000, 64, 64, 1,
                                 None) == _lib.RSORT_BAD_ARGUMENT


@pytest.mark.parametrize("args", [
    (None, 64, 0x20000, 64, 64),          # null tokens
    (0x10000, 64, None, 64, 64),          # null rows
    (0x10000, 64, 0x20000, 32, 64),       # output rows would overlap
    (0x10000, 64, 0x10040, 64, 64),       # rows overlap the tokens
    (0x10000, 0, 0x10000 - 7 * 64, 64, 64)])
def test_gather_refusals(args):
    assert L.rsort_expert_gather(plan_args(), *args, 1, None) == _lib.RSORT_BAD_ARGUMENT


def test_gather_sizes_that_wrap_are_refused():
    assert L.rsort_expert_gather(plan_args(), 0x10000, 1 << 62, 0x20000, 64, 64, 1,
                                 None) == _lib.RSORT_SIZE_OVERFLOW
    assert L.rsort_expert_gather(plan_args(), 0x10000, 64, 0x20000, 1 << 62, 64, 1,
                                 None) == _lib.RSORT_SIZE_OVERFLOW


F32, F16 = _lib.RSORT_F32, _lib.RSORT_F16


@pytest.mark.parametrize("args", [
    (_lib.RSORT_F64, 0x10000, 16, 0x20000, F32, 0x30000, 16, 16),   # row type
    (F32, 0x10000, 16, 0x20000, _lib.RSORT_I32, 0x30000, 16, 16),   # weight type
    (F32, None, 16, 0x20000, F32, 0x30000, 16, 16),
    (F32, 0x10000, 16, 0x20000, F32, None, 16, 16),
    (F32, 0x10000, 16, 0x20000, F32, 0x30000, 15, 16),              # rows overlap
    (F32, 0x10002, 16, 0x20000, F32, 0x30000, 16, 16),              # alignment
    (F32, 0x10000, 16, 0x20002, F32, 0x30000, 16, 16),
    (F32, 0x10000, 16, 0x30000, F32, 0x30010, 16, 16),              # output over the weights
    (F16, 0x10000, 16, 0x20000, F32, 0x10010, 16, 16)])             # output over the rows
def test_combine_refusals(args):
    assert L.rsort_expert_combine(plan_args(), *args, None) == _lib.RSORT_BAD_ARGUMENT


@pytest.mark.parametrize("args", [
    (_lib.RSORT_U16, 0x10000, 16, 0x20000, 16, 0x30000, F32, 0x40000, 16, 0x50000, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, _lib.RSORT_U8, 0x40000, 16, 0x50000, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, None, 16, None, 16),   # no output
    (F32, None, 16, 0x20000, 16, 0x30000, F32, 0x40000, 16, 0x50000, 16),
    (F32, 0x10000, 16, None, 16, 0x30000, F32, 0x40000, 16, 0x50000, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, 0x40000, 8, 0x50000, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, 0x40002, 16, 0x50000, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, 0x20000, 16, 0x50000, 16),  # in place
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, 0x40000, 16, 0x30004, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, 0x40000, 16, 0x40010, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, None, 0, 0x20010, 16),
    (F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, None, 0, 0x10010, 16)])
def test_combine_backward_refusals(args):
    assert L.rsort_expert_combine_backward(plan_args(), *args, 1, None) == _lib.RSORT_BAD_ARGUMENT


def test_python_refusals():
    plan = plan_on_cpu()
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(BadArgument):
        experts.device_expert_sort(CPU, ids.to(torch.int16), plan)
    with pytest.raises(LengthMismatch):
        experts.device_expert_sort(CPU, ids[:3], plan)
    with pytest.raises(BadArgument):
        experts.device_expert_sort(CPU, torch.zeros(2, 4, dtype=torch.int32).t(), plan)
    x, rows, w = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(4, 2)
    with pytest.raises(BadArgument):
        experts.device_expert_gather(CPU, x.half(), plan, rows)
    with pytest.raises(BadArgument):
        experts.device_expert_gather(CPU, torch.zeros(8, 4).t(), plan, rows)
    with pytest.raises(BadArgument):  # a broadcast scalar has no rows of elements
        experts.device_expert_gather(CPU, torch.zeros(1, 1).expand(4, 8), plan, rows)
    with pytest.raises(LengthMismatch):
        experts.device_expert_gather(CPU, x[:3], plan, rows)
    with pytest.raises(LengthMismatch):
        experts.device_expert_gather(CPU, x, plan, rows[:7])
    with pytest.raises(LengthMismatch):
        experts.device_expert_gather(CPU, torch.zeros(4, 9), plan, rows)
    with pytest.raises(BadArgument):
        experts.device_expert_combine(CPU, rows.double(), w, plan, x.double())
    with pytest.raises(BadArgument):
        experts.device_expert_combine(CPU, rows, w.double(), plan, x)
    with pytest.raises(BadArgument):
        experts.device_expert_combine(CPU, rows, None, plan, x)
    with pytest.raises(BadArgument):
        experts.device_expert_combine(CPU, rows, w, plan, x.half())
    with pytest.raises(LengthMismatch):
        experts.device_expert_combine(CPU, rows, w[:3], plan, x)
    with pytest.raises(BadArgument):
        experts.device_expert_combine(CPU, rows, torch.zeros(2, 4).t(), plan, x)
    with pytest.raises(BadArgument):
        experts.device_expert_combine_backward(CPU, x, rows, w, plan, rows.half(), w)
    with pytest.raises(BadArgument):
        experts.device_expert_combine_backward(CPU, x, rows, w, plan, rows, w.half())
    with pytest.raises(LengthMismatch):
        experts.device_expert_gather_backward(CPU, rows, plan, x[:2])
    with pytest.raises(cub.ContextMismatch):
        experts.device_expert_gather(cub.Launch(torch.device("cuda:0"), Stream()), x, plan, rows)
    with pytest.raises(BadArgument):
        experts.device_expert_plan(CPU, -1, 2, 4)
    for top_k in (0, 1025):
        with pytest.raises(BadArgument):
            experts.device_expert_plan(CPU, 4, top_k, 4)


@pytest.mark.parametrize("weights,grad_rows,stride", [
    (0x30000, 0x30000, 16), (0x30000, 0x3001c, 16), (0x30000, 0x30000 - 0x1fc, 16),
    # weights in a gap between gradient rows but for their last byte's word
    (0x40000 + 64, 0x40000, 16 + 7)])
def test_gradient_rows_over_the_weights_are_refused(weights, grad_rows, stride):
    """8 weights of 4 bytes; 8 gradient rows of 64 bytes.  CTAs go on reading
    weights while others write rows."""
    for grad_weights in (None, 0x60000):
        assert L.rsort_expert_combine_backward(
            plan_args(), F32, 0x10000, 16, 0x20000, 16, weights, F32, grad_rows, stride,
            grad_weights, 16, 1, None) == _lib.RSORT_BAD_ARGUMENT


# the plan's arrays: 8 slots' rows at 0x1000, 4 offsets at 0x2000, 3 counts at 0x3000
@pytest.mark.parametrize("at", [0x1000, 0x101c, 0x2000, 0x200c, 0x3000, 0x3008])
def test_outputs_over_the_plan_are_refused(at):
    """Whether the output starts there or ends there."""
    for rows, tokens in ((at, at), (at + 4 - 8 * 64, at + 4 - 4 * 64)):
        assert L.rsort_expert_gather(plan_args(), 0x10000, 64, rows, 64, 64, 1,
                                     None) == _lib.RSORT_BAD_ARGUMENT
        for weights in (None, 0x20000):
            assert L.rsort_expert_combine(plan_args(), F32, 0x10000, 16, weights, F32, tokens, 16,
                                          16, None) == _lib.RSORT_BAD_ARGUMENT
        for grad_rows, grad_weights in ((rows, None), (rows, 0x60000), (0x50000, at),
                                        (None, at), (None, at + 4 - 32)):
            assert L.rsort_expert_combine_backward(
                plan_args(), F32, 0x10000, 16, 0x20000, 16, 0x30000, F32, grad_rows, 16,
                grad_weights, 16, 1, None) == _lib.RSORT_BAD_ARGUMENT


def test_ids_and_weights_in_another_order_are_refused():
    """(top_k, tokens) has as many entries, but its slots are in another order."""
    plan = plan_on_cpu(tokens=6, top_k=2)
    x, rows = torch.zeros(6, 8), torch.zeros(plan.rows, 8)
    for shape in ((2, 6), (3, 4), (12, 1), (1, 12), (2, 2, 3)):
        ids, w = torch.zeros(shape, dtype=torch.int64), torch.zeros(shape)
        with pytest.raises(LengthMismatch):
            experts.device_expert_sort(CPU, ids, plan)
        with pytest.raises(LengthMismatch):
            experts.device_expert_combine(CPU, rows, w, plan, x)
        with pytest.raises(LengthMismatch):
            experts.device_expert_combine_backward(CPU, x, rows, w, plan, rows, None)
        with pytest.raises(LengthMismatch):
            experts.device_expert_combine_backward(CPU, x, rows, torch.zeros(6, 2), plan, rows, w)


ARRAYS = ("row_of_slot", "slot_of_row", "offsets", "counts", "scratch")


def test_a_plan_keeps_its_arrays():
    """The calls take the arrays' addresses from the plan once, so none can be
    replaced in place; a plan with another array is another plan."""
    plan = plan_on_cpu()
    for name in ARRAYS:
        other = getattr(plan, name).clone()
        with pytest.raises(dataclasses.FrozenInstanceError):
            setattr(plan, name, other)
        assert getattr(plan, name) is not other
        fresh = dataclasses.replace(plan, **{name: other})
        assert getattr(fresh, name) is other
        where = [getattr(fresh, n).data_ptr() for n in ARRAYS]
        args = fresh._args
        assert [args.row_of_slot, args.offsets, args.counts] == [where[0], where[2], where[3]]
        a = fresh.sort_args
        assert [a[3], a[4], a[6], a[7], a[8]] == where
    with pytest.raises(dataclasses.FrozenInstanceError):
        plan.tokens = 5


@pytest.mark.parametrize("name", ARRAYS)
def test_a_plan_of_wrong_arrays_is_refused(name):
    """The kernels trust the arrays' sizes."""
    plan = plan_on_cpu()
    t = getattr(plan, name)
    wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype)
    bad = [(t.to(torch.int64), BadArgument), (wide[..., ::2], BadArgument)]
    if name != "scratch":  # whose size every sort checks
        bad += [(t[:-1].contiguous(), LengthMismatch), (wide, LengthMismatch)]
    for other, error in bad:
        with pytest.raises(error):
            dataclasses.replace(plan, **{name: other})


@pytest.mark.parametrize("tokens,top_k,count,align", [
    (2**64 + 8, 1, 4, 1), (8, 2**64 + 1, 4, 1), (8, 1, 2**64 + 4, 1), (8, 1, 4, 2**64 + 1),
    (2**31, 1, 4, 1), (-8, -1, 4, 1), (0, 2, 4, 0), (0, 2, 4, 65537), (0, 2, 0, 1), (8, 1, -4, 1)])
def test_plan_sizes_out_of_range_are_refused(tokens, top_k, count, align):
    """Sizes that a 64-bit word would wrap into range, and those of no slots."""
    with pytest.raises(BadArgument):
        experts.expert_rows(tokens, top_k, count, align)
    with pytest.raises(BadArgument):
        experts.device_expert_plan(CPU, tokens, top_k, count, align)
