"""CPU tests of the cache eviction's refusals: every call here is rejected on
the host before any device work."""
import pytest
import torch

from rccl_b200 import _lib, cub, eviction
from rccl_b200.errors import BadArgument, LengthMismatch

L = _lib.lib()
F32 = _lib.RSORT_F32
BAD, OVERFLOW = _lib.RSORT_BAD_ARGUMENT, _lib.RSORT_SIZE_OVERFLOW


class Stream:
    cuda_stream = 0


CPU = cub.Launch(torch.device("cpu"), Stream())  # refused calls never reach a device


def add_status(**kw):
    a = dict(t=F32, w=0x10000, sb=256, sh=64, sq=64, batch=2, heads=2, group=2, queries=1,
             capacity=64, lengths=0x1000, scores=0x20000, score_b=128, score_h=64)
    a.update(kw)
    return L.rsort_attention_weight_add(
        a["t"], a["w"], a["sb"], a["sh"], a["sq"], a["batch"], a["heads"], a["group"],
        a["queries"], a["capacity"], a["lengths"], 1.0, 0, a["scores"], a["score_b"],
        a["score_h"], None)


@pytest.mark.parametrize("change,status", [
    (dict(t=_lib.RSORT_F64), BAD), (dict(t=_lib.RSORT_I32), BAD), (dict(w=None), BAD),
    (dict(scores=None), BAD), (dict(group=0), BAD), (dict(w=0x10002), BAD),
    (dict(t=_lib.RSORT_BF16, w=0x10001), BAD), (dict(scores=0x20002), BAD),
    (dict(lengths=0x1002), BAD), (dict(score_h=63), BAD), (dict(score_b=64), BAD),
    (dict(score_b=0), BAD), (dict(batch=65536), OVERFLOW), (dict(batch=256, heads=256), OVERFLOW),
    (dict(capacity=2**31 - 1), OVERFLOW), (dict(sb=1 << 60), OVERFLOW),
    (dict(queries=2**31), BAD)])
def test_add_refusals(change, status):
    assert add_status(**change) == status
    assert _lib.last_error().status == status


def test_nothing_to_add_is_no_launch():
    for k in ("batch", "heads", "capacity"):
        assert add_status(**{k: 0}) == _lib.RSORT_OK


def select_status(**kw):
    a = dict(scores=0x10000, sb=128, sh=64, lengths=0x1000, batch=2, heads=2, capacity=64,
             budget=16, sinks=2, recent=4, kept=0x2000, kept_lengths=0x3000)
    a.update(kw)
    return L.rsort_cache_select(a["scores"], a["sb"], a["sh"], a["lengths"], a["batch"], a["heads"],
                                a["capacity"], a["budget"], a["sinks"], a["recent"], a["kept"],
                                a["kept_lengths"], None)


@pytest.mark.parametrize("change,status", [
    (dict(scores=None), BAD), (dict(kept=None), BAD), (dict(kept_lengths=None), BAD),
    (dict(budget=0), BAD), (dict(budget=2**31), BAD), (dict(sinks=17), BAD),
    (dict(sinks=13), BAD), (dict(recent=2**64 - 1), BAD), (dict(kept_lengths=0x1000), BAD),
    (dict(kept_lengths=0x1004), BAD), (dict(kept=0x10040), BAD), (dict(kept_lengths=0x10000), BAD),
    (dict(kept=0x0ff8), BAD), (dict(kept_lengths=0x2010), BAD), (dict(scores=0x10002), BAD), (dict(kept=0x2001), BAD),
    (dict(batch=70000), OVERFLOW), (dict(sb=1 << 60), OVERFLOW),
    (dict(capacity=2**31), OVERFLOW)])
def test_select_refusals(change, status):
    assert select_status(**change) == status
    assert _lib.last_error().status == status


def cache(**kw):
    a = dict(src=0x100000, dst=0x200000, row_bytes=64, src_stride_b=128 * 64, src_stride_h=64 * 64,
             src_stride_s=64, dst_stride_b=32 * 64, dst_stride_h=16 * 64, dst_stride_s=64)
    a.update(kw)
    return _lib.CacheRows(**a)


def same(**kw):
    return cache(dst=0x100000, dst_stride_b=128 * 64, dst_stride_h=64 * 64, dst_stride_s=64, **kw)


def compact_status(*rows, kept=0x1000, kept_lengths=0x2000, batch=2, heads=2, budget=16,
                   capacity=64):
    arr = (_lib.CacheRows * max(len(rows), 1))(*rows)
    return L.rsort_cache_compact(arr, len(rows), kept, kept_lengths, batch, heads, budget, capacity,
                                 None)


@pytest.mark.parametrize("rows,status", [
    ([cache()] * 9, BAD),
    ([cache(src=None)], BAD),
    ([cache(dst=None)], BAD),
    ([cache(row_bytes=0)], BAD),
    ([cache(dst_stride_s=32)], BAD),                       # written rows overlap
    ([cache(dst_stride_h=64)], BAD),
    ([cache(dst_stride_b=0)], BAD),
    ([cache(dst=0x100040)], BAD),                          # a dst over its own src
    ([cache(), cache(src=0x300000)], BAD),                 # two dsts in one place
    ([cache(), cache(src=0x200000, dst=0x400000)], BAD),   # a dst over another src
    ([same(), cache(src=0x300000)], BAD),                  # one in place, one not
    ([cache(dst=0x100000)], BAD),                          # in place with other strides
    ([cache(dst=0x1000)], BAD),                            # over the kept positions
    ([cache(src_stride_b=1 << 60)], OVERFLOW)])
def test_compact_refusals(rows, status):
    assert compact_status(*rows) == status
    assert _lib.last_error().status == status


def test_compact_refuses_null_and_misaligned_positions():
    assert compact_status(cache(), kept=None) == BAD
    assert compact_status(cache(), kept_lengths=None) == BAD
    assert compact_status(cache(), kept=0x1001) == BAD
    assert compact_status(cache(), batch=70000) == OVERFLOW
    assert compact_status() == _lib.RSORT_OK
    assert compact_status(cache(), budget=0) == _lib.RSORT_OK


def test_python_refusals():
    w, scores = torch.zeros(2, 4, 1, 8), torch.zeros(2, 2, 8)
    i32 = dict(dtype=torch.int32)
    lens, kept, n = torch.zeros(2, **i32), torch.zeros(2, 2, 4, **i32), torch.zeros(2, **i32)
    add, select = eviction.device_attention_weight_add, eviction.device_cache_select
    compact = eviction.device_cache_compact
    for bad, error in [((w.double(), scores, lens), BadArgument),
                       ((w, scores.half(), lens), BadArgument),
                       ((w, scores, lens.long()), BadArgument),
                       ((w, scores, lens[:1]), LengthMismatch),
                       ((w[:1], scores, lens), LengthMismatch),
                       ((w[:, :3], scores, lens), LengthMismatch),
                       ((w[:, :1], scores, lens), LengthMismatch),
                       ((w[..., :7], scores, lens), LengthMismatch),
                       ((w[..., ::2], scores[..., :4].contiguous(), lens), BadArgument),
                       ((w[0, 0], scores, lens), BadArgument)]:
        with pytest.raises(error):
            add(CPU, *bad)
    for bad, error in [((scores.double(), lens, kept, n), BadArgument),
                       ((scores, lens, kept.long(), n), BadArgument),
                       ((scores, lens, kept[0], n), BadArgument),
                       ((scores, lens, kept[:, :1].contiguous(), n), LengthMismatch),
                       ((scores, lens, kept, n[:1]), LengthMismatch),
                       ((scores, lens, kept, n, -1), BadArgument),
                       ((scores, lens, kept, n, 0, -1), BadArgument)]:
        with pytest.raises(error):
            select(CPU, *bad)
    k = torch.zeros(2, 2, 8, 16)
    for bad, error in [((kept, n, [k], []), LengthMismatch),
                       ((kept, n, [k] * 9), BadArgument),
                       ((kept, n, [k[0]]), LengthMismatch),
                       ((kept, n, [k[:1]]), LengthMismatch),
                       ((kept, n, [k, k[:, :, :7]]), LengthMismatch),
                       ((kept, n, [k], [k.half()]), BadArgument),
                       ((kept, n, [k], [k[:, :, :3]]), LengthMismatch),
                       ((kept, n, [k], [k[..., :8]]), LengthMismatch),
                       ((kept, n, [k.transpose(2, 3)]), BadArgument),
                       ((kept.long(), n, [k]), BadArgument),
                       ((kept, n.long(), [k]), BadArgument)]:
        with pytest.raises(error):
            compact(CPU, *bad)
    with pytest.raises(cub.ContextMismatch):
        compact(cub.Launch(torch.device("cuda:0"), Stream()), kept, n, [k])


def test_rows_of_one_allocation_that_share_a_byte_are_refused():
    """Rows of 64 and 32 bytes in places of 96: apart side by side, refused as
    soon as they share a byte."""
    def view(offset, row_bytes, base):
        return dict(row_bytes=row_bytes, src=base + offset, src_stride_s=96, src_stride_h=64 * 96,
                    src_stride_b=128 * 96)

    def into(offset, base):
        return dict(dst=base + offset, dst_stride_s=96, dst_stride_h=64 * 96, dst_stride_b=128 * 96)

    for offset in (63, 65, 1, 95):
        rows = [cache(**view(0, 64, 0x100000), **into(0, 0x200000)),
                cache(**view(64, 32, 0x100000), **into(offset, 0x200000))]
        assert compact_status(*rows) == BAD
        rows = [cache(**view(0, 64, 0x100000), **into(0, 0x100000)),
                cache(**view(offset, 32, 0x100000), **into(offset, 0x100000))]
        assert compact_status(*rows) == BAD


# float32 weights [2, 4, 1, 64] at 0x10000 take 2 KB, totals [2, 2, 64] 1 KB
@pytest.mark.parametrize("change", [
    dict(scores=0x10000), dict(scores=0x107fc), dict(scores=0x10000 - 0x3fc),
    dict(scores=0x1004 - 0x400), dict(scores=0x1004),        # over the lengths
    dict(lengths=0x20000), dict(lengths=0x203fc),
    # totals between the weights' heads, 96 apart, over the last of 32 weights
    dict(sb=4 * 96, sh=96, scores=0x10000 + 4 * 31, score_b=4 * 96, score_h=96, capacity=32)])
def test_add_refuses_totals_over_what_it_reads(change):
    assert add_status(**change) == BAD
    assert _lib.last_error().status == BAD


@pytest.mark.parametrize("sinks,recent", [(2**64, 0), (0, 2**64), (2**64 + 1, 1), (5, 0), (2, 3),
                                          (0, 5)])
def test_sinks_and_recent_positions_beyond_the_budget_are_refused(sinks, recent):
    i32 = dict(dtype=torch.int32)
    with pytest.raises(BadArgument):
        eviction.device_cache_select(CPU, torch.zeros(2, 2, 8), None, torch.zeros(2, 2, 4, **i32),
                                     torch.zeros(2, **i32), sinks, recent)
