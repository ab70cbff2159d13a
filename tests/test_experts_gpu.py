"""Expert routing on the GPU against a plain 64-bit restatement: the stable
counting sort by expert, the gather into expert order, the weighted combine and
the gradients, with dropped slots, padded segments, strided and misaligned
rows, and buffers whose unused rows hold NaN.

Tolerances: a sum of n terms in fp32 is off by at most n * 2^-24 times the sum
of the terms' magnitudes (products are fused or rounded once each: one more
step), and the result's rounding adds half a step of its type."""
import numpy as np
import pytest
import torch

from rccl_b200 import cub, experts

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
NAN = float("nan")
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def launch():
    return cub.Program.load("cuda:0").on()


def sorted_plan(ids, count, align):
    """The plan of flat ids by its definition."""
    rows = experts.expert_rows(ids.size, 1, count, align) if ids.size else 0
    row_of_slot = np.full(ids.size, -1, np.int64)
    offsets = np.zeros(count + 1, np.int64)
    counts = np.zeros(count, np.int64)
    for e in range(count):
        mine = np.flatnonzero(ids == e)
        counts[e] = mine.size
        row_of_slot[mine] = offsets[e] + np.arange(mine.size)
        offsets[e + 1] = offsets[e] + (mine.size + align - 1) // align * align
    slot_of_row = np.full(rows, -1, np.int64)
    used = row_of_slot >= 0
    slot_of_row[row_of_slot[used]] = np.flatnonzero(used)
    return row_of_slot, slot_of_row, offsets, counts


def make_ids(rng, tokens, top_k, count, kind, dtype):
    n = tokens * top_k
    if kind == "uniform":
        ids = rng.integers(0, count, n)
    elif kind == "skewed":
        ids = np.minimum(rng.geometric(0.3, n) - 1, count - 1)
    elif kind == "one":
        ids = np.full(n, count - 1)
    elif kind == "dropped":
        ids = np.full(n, -1)
    else:  # mixed: every way to be out of range
        ids = rng.integers(0, count, n)
        bad = [-1, count, count + 7, np.iinfo(np.int32).min, np.iinfo(np.int32).max]
        if dtype == torch.int64:
            bad += [2**32, -2**32, 2**62, np.iinfo(np.int64).min]
        hit = rng.random(n) < 0.3
        ids[hit] = rng.choice(np.array(bad, np.int64), int(hit.sum()))
    return torch.from_numpy(ids.reshape(tokens, top_k)).to(dtype)


def sort(ids, count, align):
    lau = launch()
    plan = experts.device_expert_plan(lau, ids.shape[0], ids.shape[1], count, align)
    # what an earlier call left must not matter
    for t in (plan.row_of_slot, plan.slot_of_row, plan.offsets, plan.counts, plan.scratch):
        t.fill_(77)
    experts.device_expert_sort(lau, ids.cuda(), plan)
    return lau, plan


def check_plan(plan, ids, count, align):
    want = sorted_plan(ids.reshape(-1).numpy().astype(np.int64), count, align)
    got = (plan.row_of_slot.view(-1), plan.slot_of_row, plan.offsets, plan.counts)
    for name, w, g in zip(("row_of_slot", "slot_of_row", "offsets", "counts"), want, got):
        assert np.array_equal(g.cpu().numpy().astype(np.int64), w), name


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("kind", ["uniform", "skewed", "one", "dropped", "mixed"])
@pytest.mark.parametrize("tokens,top_k,count,align", [
    (0, 2, 4, 8), (1, 1, 1, 1), (1, 8, 1024, 16), (31, 1, 3, 1), (33, 3, 60, 8), (129, 8, 256, 128),
    (341, 3, 7, 1), (1025, 1, 1000, 4), (8191, 6, 64, 64)])
def test_sort_matches_its_definition(tokens, top_k, count, align, kind, dtype):
    rng = np.random.default_rng(tokens + 7 * top_k + count)
    ids = make_ids(rng, tokens, top_k, count, kind, dtype)
    _, plan = sort(ids, count, align)
    check_plan(plan, ids, count, align)


@pytest.mark.parametrize("tokens,top_k,count,align", [
    (70_001, 4, 1024, 16), (262_144, 8, 256, 128), (1_000_003, 1, 8, 1)])
def test_long_sort_matches_its_definition(tokens, top_k, count, align):
    rng = np.random.default_rng(tokens)
    ids = make_ids(rng, tokens, top_k, count, "mixed", torch.int32)
    _, plan = sort(ids, count, align)
    check_plan(plan, ids, count, align)


def padded(t, stride, offset):
    """t's rows `stride` elements apart, starting `offset` elements into a
    NaN- or 0x77-filled allocation."""
    n, w = t.shape
    flat = torch.empty(offset + max(n, 1) * stride + 1, dtype=t.dtype, device="cuda")
    flat.fill_(float("nan") if t.dtype.is_floating_point else 77)
    v = flat[offset:offset + max(n, 1) * stride].view(max(n, 1), stride)[:n, :w]
    v.copy_(t)
    return v


# width, extra stride, offset of the first element
SHAPES = [(1, 0, 0), (7, 0, 0), (8, 0, 0), (64, 8, 0), (64, 0, 1), (100, 3, 2), (130, 2, 2),
          (1000, 0, 0), (1001, 0, 0), (2056, 8, 8), (4096, 0, 0)]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.float64])
@pytest.mark.parametrize("width,extra,offset", SHAPES)
@pytest.mark.parametrize("zero_padding", [True, False])
def test_gather(dtype, width, extra, offset, zero_padding):
    rng = np.random.default_rng(width)
    tokens, top_k, count, align = 37, 3, 5, 16
    ids = make_ids(rng, tokens, top_k, count, "mixed", torch.int32)
    lau, plan = sort(ids, count, align)
    x = torch.from_numpy(rng.integers(0, 100, (tokens, width))).to(dtype)
    rows = padded(torch.full((plan.rows + 3, width), 55, dtype=dtype), width + extra, offset)
    experts.device_expert_gather(lau, padded(x.cuda(), width + extra, offset), plan, rows,
                                 zero_padding)
    row_of_slot, slot_of_row, offsets, _ = sorted_plan(
        ids.reshape(-1).numpy().astype(np.int64), count, align)
    want = torch.full((plan.rows + 3, width), 55, dtype=dtype)
    if zero_padding:
        want[:offsets[-1]] = 0
    used = np.flatnonzero(slot_of_row >= 0)
    want[used] = x[slot_of_row[used] // top_k]
    assert torch.equal(rows.cpu(), want)


def test_gather_of_a_broadcast_token_and_of_no_tokens():
    lau, plan = sort(torch.tensor([[0, 1], [1, -1], [2, 2]], dtype=torch.int32), 3, 4)
    x = torch.arange(24, dtype=torch.float16, device="cuda").view(1, 24).expand(3, 24)
    rows = torch.full((plan.rows, 24), 9, dtype=torch.float16, device="cuda")
    experts.device_expert_gather(lau, x, plan, rows)
    want = torch.zeros(plan.rows, 24, dtype=torch.float16)
    want[[0, 4, 5, 8, 9]] = x[0].cpu()
    want[12:] = 9
    assert torch.equal(rows.cpu(), want)
    lau, plan = sort(torch.zeros(0, 2, dtype=torch.int64), 3, 4)
    assert plan.rows == 0
    out = torch.zeros(0, 24, device="cuda")
    experts.device_expert_gather(lau, out, plan, out)
    experts.device_expert_combine(lau, out, torch.zeros(0, 2, device="cuda"), plan, out)


class Step:
    """Inputs of one combine and its gradient; rows that no slot uses hold NaN."""

    def __init__(self, seed, tokens, top_k, count, align, width, dtype, wdtype, extra=0, offset=0,
                 kind="mixed"):
        rng = np.random.default_rng(seed)
        self.dtype, self.wdtype, self.top_k = dtype, wdtype, top_k
        ids = make_ids(rng, tokens, top_k, count, kind, torch.int64)
        self.lau, self.plan = sort(ids, count, align)
        self.row_of_slot, self.slot_of_row, self.offsets, _ = sorted_plan(
            ids.reshape(-1).numpy().astype(np.int64), count, align)
        n = self.plan.rows

        def normal(*shape):
            return torch.from_numpy(rng.normal(0, 1, shape)).to(dtype)

        rows = normal(n, width)
        rows[self.slot_of_row < 0] = float("nan")
        self.rows64 = rows.double().numpy()
        self.rows = padded(rows.cuda(), width + extra, offset)
        self.w = torch.from_numpy(rng.normal(0, 1, (tokens, top_k))).to(wdtype).cuda()
        self.w64 = self.w.double().cpu().numpy().reshape(-1)
        grad = normal(tokens, width)
        self.grad64 = grad.double().numpy()
        self.grad = padded(grad.cuda(), width + extra, offset)
        self.tokens, self.width = tokens, width
        self.used = np.flatnonzero(self.row_of_slot >= 0)

    def out(self, n):
        return torch.full((n, self.width), 33, dtype=self.dtype, device="cuda")


def combined(row_of_slot, rows64, w64, tokens, top_k, width):
    """The sums and the sums of magnitudes, by rows."""
    used = np.flatnonzero(row_of_slot >= 0)
    y, mag = np.zeros((2, tokens, width))
    terms = rows64[row_of_slot[used]] * w64[used, None]
    np.add.at(y, used // top_k, terms)
    np.add.at(mag, used // top_k, np.abs(terms))
    return y, mag


def close(got, want, mag, terms, dtype):
    got = got.double().cpu().numpy()
    tol = (terms + 1) * 2.0**-24 * mag
    tol = tol + HALF[dtype] * (np.abs(want) + tol) + TINY[dtype]
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) - tol).max())


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.bfloat16)]
STEPS = [(1, 1, 1, 1), (1, 8, 16, 8), (37, 3, 5, 16), (5, 17, 40, 1), (300, 2, 8, 64)]


@pytest.mark.parametrize("dtype,wdtype", TYPES)
@pytest.mark.parametrize("tokens,top_k,count,align", STEPS)
@pytest.mark.parametrize("width,extra,offset", [(1, 0, 0), (100, 3, 2), (130, 2, 2), (1001, 0, 0),
                                                (2056, 8, 8)])
def test_combine_and_gradients(tokens, top_k, count, align, width, extra, offset, dtype, wdtype):
    s = Step(tokens + width, tokens, top_k, count, align, width, dtype, wdtype, extra, offset)
    y = s.out(tokens)
    experts.device_expert_combine(s.lau, s.rows, s.w, s.plan, y)
    want, mag = combined(s.row_of_slot, s.rows64, s.w64, tokens, top_k, width)
    close(y, want, mag, top_k, dtype)

    grad_x = s.out(tokens)
    experts.device_expert_gather_backward(s.lau, s.rows, s.plan, grad_x)
    want, mag = combined(s.row_of_slot, s.rows64, np.ones(s.w64.size), tokens, top_k, width)
    close(grad_x, want, mag, top_k, dtype)

    grad_rows, grad_w = s.out(s.plan.rows + 2), torch.full_like(s.w, 44)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, grad_rows, grad_w)
    used = s.used
    want = np.full((s.plan.rows + 2, width), 33.0)
    want[:s.offsets[-1]] = 0
    want[s.row_of_slot[used]] = s.grad64[used // top_k] * s.w64[used, None]
    close(grad_rows, want, np.abs(want), 0, dtype)
    assert (grad_rows[s.offsets[-1]:] == 33).all()
    terms = s.grad64[used // top_k] * s.rows64[s.row_of_slot[used]]
    want, mag = np.zeros((2, s.w64.size))
    want[used], mag[used] = terms.sum(1), np.abs(terms).sum(1)
    close(grad_w.view(-1), want, mag, width, wdtype)

    # one of the two alone is the same one
    only_rows, only_w = s.out(s.plan.rows + 2), torch.full_like(s.w, 44)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, only_rows, None)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, None, only_w)
    assert torch.equal(only_rows, grad_rows) and torch.equal(only_w, grad_w)


def test_padding_rows_stay_without_zero_padding():
    s = Step(3, 9, 2, 4, 8, 64, torch.float32, torch.float32)
    grad_rows = s.out(s.plan.rows)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, grad_rows, None,
                                           zero_padding=False)
    assert (grad_rows[s.slot_of_row < 0] == 33).all()


@pytest.mark.parametrize("top_k,width", [(3, 8), (3, 2056), (9, 33)])
def test_dropped_slots_count_for_nothing(top_k, width):
    """Weights of dropped slots are NaN and the gradient is not finite: what is
    dropped stays out of the sums and has the gradient 0."""
    s = Step(21, 40, top_k, 6, 4, width, torch.bfloat16, torch.float32)
    dropped = torch.from_numpy(s.row_of_slot < 0).view(40, top_k).cuda()
    assert dropped.any() and not dropped.all()
    s.w[dropped] = float("nan")
    y = s.out(40)
    experts.device_expert_combine(s.lau, s.rows, s.w, s.plan, y)
    want, mag = combined(s.row_of_slot, s.rows64, s.w64, 40, top_k, width)
    close(y, want, mag, top_k, torch.bfloat16)
    s.grad[:, 0] = float("inf")
    s.grad[:, width - 1] = float("nan")
    grad_w = torch.full_like(s.w, 44)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, None, grad_w)
    assert (grad_w[dropped] == 0).all()
    assert torch.isnan(grad_w[~dropped]).all()


def test_gradients_against_differences():
    """The combine is linear in the weights and in the rows, so a difference
    over any step is the gradient but for roundings: 2 * (top_k + 1) roundings
    of 2^-24 of each side's magnitudes, divided by the step's length 2."""
    s = Step(11, 6, 3, 4, 4, 40, torch.float32, torch.float32, kind="mixed")
    grad_rows, grad_w = s.out(s.plan.rows), torch.zeros_like(s.w)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, grad_rows, grad_w)

    def loss(rows, w):
        y = s.out(6)
        experts.device_expert_combine(s.lau, rows, w, s.plan, y)
        _, mag = combined(s.row_of_slot, rows.double().cpu().numpy(),
                          w.double().cpu().numpy().reshape(-1), 6, 3, 40)
        off = (s.top_k + 1) * 2.0**-24 * (mag * np.abs(s.grad64)).sum()
        return (y.double().cpu().numpy() * s.grad64).sum(), off

    def check(rows_a, w_a, rows_b, w_b, got):
        (la, oa), (lb, ob) = loss(rows_a, w_a), loss(rows_b, w_b)
        # the gradient itself: a dot of 40 or a product, in fp32
        assert abs((la - lb) / 2 - got) <= (oa + ob) / 2 + 41 * 2.0**-24 * 40 * 16

    for slot in range(18):
        d = torch.zeros_like(s.w)
        d.view(-1)[slot] = 1
        check(s.rows, s.w + d, s.rows, s.w - d, float(grad_w.view(-1)[slot]))
    for slot in s.used[::4]:
        for col in (0, 17, 39):
            d = torch.zeros_like(s.rows)
            d[int(s.row_of_slot[slot]), col] = 1
            check(s.rows + d, s.w, s.rows - d, s.w, float(grad_rows[s.row_of_slot[slot], col]))


def layer(lau, plan, ids, x, w, weights_of_experts, rows, expert_out, y):
    experts.device_expert_sort(lau, ids, plan)
    experts.device_expert_gather(lau, x, plan, rows)
    # every expert scales by a number of its own
    per_row = torch.repeat_interleave(weights_of_experts, plan.align)
    torch.mul(rows, per_row[:, None], out=expert_out)
    experts.device_expert_combine(lau, expert_out, w, plan, y)


def test_a_layer_on_a_side_stream_and_captured():
    """Sort, gather, an expert product, combine: eager on a side stream, then
    captured once and replayed on new ids, tokens and weights."""
    tokens, top_k, count, width = 50, 4, 6, 96
    align = tokens * top_k  # one segment an expert, so a row's expert is known
    program = cub.Program.load("cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lau = program.on(side)
        plan = experts.device_expert_plan(lau, tokens, top_k, count, align)
        scale = torch.arange(1, count + 1, dtype=torch.float32, device="cuda")
        state = dict(ids=torch.zeros(tokens, top_k, dtype=torch.int64, device="cuda"),
                     x=torch.zeros(tokens, width, device="cuda"),
                     w=torch.zeros(tokens, top_k, device="cuda"))
        rows = torch.zeros(plan.rows, width, device="cuda")
        expert_out, y = torch.zeros_like(rows), torch.zeros(tokens, width, device="cuda")

    rng = np.random.default_rng(5)

    def fresh():
        # every expert is chosen, so expert e's segment is rows [e, e + 1) * align
        ids = np.stack([rng.permutation(count)[:top_k] for _ in range(tokens)])
        ids[:2] = [[0, 1, 2, 3], [4, 5, 0, -1]]
        new = dict(ids=torch.from_numpy(ids), x=torch.from_numpy(rng.normal(size=(tokens, width))),
                   w=torch.from_numpy(rng.normal(size=(tokens, top_k))))
        with torch.cuda.stream(side):
            for k, v in new.items():
                state[k].copy_(v)
        x, w = state["x"].double().cpu().numpy(), state["w"].double().cpu().numpy()
        f = np.where(ids >= 0, w * (ids + 1), 0)
        return f.sum(1)[:, None] * x, np.abs(f).sum(1)[:, None] * np.abs(x)

    def run():
        layer(lau, plan, state["ids"], state["x"], state["w"], scale, rows, expert_out, y)

    for _ in range(2):
        want, mag = fresh()
        with torch.cuda.stream(side):
            run()
        side.synchronize()
        close(y, want, mag, top_k + 2, torch.float32)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        lau = program.on(torch.cuda.current_stream())
        run()
    for _ in range(3):
        want, mag = fresh()
        y.fill_(7)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        close(y, want, mag, top_k + 2, torch.float32)


def test_calls_count_as_launches_of_this_library():
    lib = experts._lib.lib()
    s = Step(1, 8, 2, 4, 1, 32, torch.bfloat16, torch.float32)
    lib.rsort_launch_count_reset()
    experts.device_expert_combine(s.lau, s.rows, s.w, s.plan, s.out(8))
    assert lib.rsort_launch_count() == 1


def long_ids(seed, tokens, top_k, count):
    """Ids of a sort of more than one cluster, a third of them dropped."""
    return make_ids(np.random.default_rng(seed), tokens, top_k, count, "mixed", torch.int64)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_long_sort_of_ids_that_a_kernel_has_just_written(dtype):
    """The ids' kernel and both kernels of the sort follow one another closely,
    over and over into the same buffers: every plan is that of its own ids."""
    tokens, top_k, count, align = 50_001, 3, 96, 8
    lau = launch()
    plan = experts.device_expert_plan(lau, tokens, top_k, count, align)
    drawn = [long_ids(seed, tokens, top_k, count) for seed in range(8)]
    drawn = [ids.clamp(-1, count).to(dtype) for ids in drawn]
    on_device = [ids.cuda() for ids in drawn]
    ids = torch.full((tokens, top_k), -1, dtype=dtype, device="cuda")
    seen = []
    torch.cuda.synchronize()
    for source in on_device:
        torch.add(source, 0, out=ids)
        experts.device_expert_sort(lau, ids, plan)
        seen.append([t.clone() for t in (plan.row_of_slot, plan.slot_of_row, plan.offsets,
                                         plan.counts)])
    for source, got in zip(drawn, seen):
        want = sorted_plan(source.reshape(-1).numpy().astype(np.int64), count, align)
        for w, g in zip(want, got):
            assert np.array_equal(g.view(-1).cpu().numpy().astype(np.int64), w)


def test_long_sort_captured_behind_the_kernel_of_its_ids():
    """The form of two launches as part of a replayed graph, twice in a row."""
    tokens, top_k, count, align = 40_003, 4, 60, 16
    program = cub.Program.load("cuda:0")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lau = program.on(side)
        plans = [experts.device_expert_plan(lau, tokens, top_k, count, align) for _ in range(2)]
        source = torch.zeros(tokens, top_k, dtype=torch.int64, device="cuda")
        ids = torch.zeros_like(source)

    def run(on):
        torch.add(source, 0, out=ids)
        experts.device_expert_sort(on, ids, plans[0])
        torch.add(source, 1, out=ids)
        experts.device_expert_sort(on, ids, plans[1])

    with torch.cuda.stream(side):
        run(lau)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run(program.on(torch.cuda.current_stream()))
    for seed in range(3):
        drawn = long_ids(seed, tokens, top_k, count).clamp(-2, count)
        with torch.cuda.stream(side):
            source.copy_(drawn)
            graph.replay()
        side.synchronize()
        check_plan(plans[0], drawn, count, align)
        check_plan(plans[1], drawn + 1, count, align)


@pytest.mark.parametrize("dtype,width", [(torch.float32, 24), (torch.bfloat16, 72),
                                         (torch.float16, 7)])
def test_rows_and_outputs_side_by_side_in_one_allocation(dtype, width):
    """Inputs and outputs as columns of one buffer: none shares a byte with
    another, and the columns that no call writes stay."""
    tokens, top_k, count, align = 40, 3, 5, 4
    s = Step(31, tokens, top_k, count, align, width, dtype, torch.float32)
    height = max(s.plan.rows, tokens)

    def columns():
        both = torch.full((height, 2 * width), 9, dtype=dtype, device="cuda")
        return both[:, :width], both[:, width:]

    y = s.out(tokens)
    experts.device_expert_combine(s.lau, s.rows, s.w, s.plan, y)
    left, right = columns()
    left[:s.plan.rows].copy_(s.rows)
    before = left.clone()
    experts.device_expert_combine(s.lau, left, s.w, s.plan, right[:tokens])
    assert torch.equal(right[:tokens], y) and (right[tokens:] == 9).all()
    assert torch.equal(left.nan_to_num(3), before.nan_to_num(3))

    rows = s.out(s.plan.rows)
    experts.device_expert_gather(s.lau, s.grad, s.plan, rows)
    left, right = columns()
    left[:tokens].copy_(s.grad)
    right[:s.plan.rows].fill_(33)
    experts.device_expert_gather(s.lau, left[:tokens], s.plan, right)
    assert torch.equal(right[:s.plan.rows], rows) and torch.equal(left[:tokens], s.grad)

    grad_rows, grad_w = s.out(s.plan.rows), torch.full_like(s.w, 44)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, grad_rows, grad_w)
    left, right = columns()
    left[:s.plan.rows].copy_(s.rows)
    right[:s.plan.rows].fill_(33)
    got_w = torch.full_like(s.w, 44)
    experts.device_expert_combine_backward(s.lau, s.grad, left, s.w, s.plan, right, got_w)
    assert torch.equal(right[:s.plan.rows], grad_rows) and torch.equal(got_w, grad_w)


@pytest.mark.parametrize("top_k", [1, 3])
def test_slots_of_a_batch_of_sequences_and_in_one_row(top_k):
    """Ids and weights (batch, length, top_k), or flat: the slots in order."""
    rng = np.random.default_rng(top_k)
    batch, length, count, width = 4, 5, 6, 16
    ids = make_ids(rng, batch * length, top_k, count, "mixed", torch.int64)
    s = Step(17, batch * length, top_k, count, 1, width, torch.float32, torch.float32)
    flat = [(-1,)] + ([(batch, length), (1, batch * length)] if top_k == 1 else [])
    for shape in [(batch, length, top_k), (batch * length, top_k)] + flat:
        experts.device_expert_sort(s.lau, ids.cuda().view(shape), s.plan)
        check_plan(s.plan, ids, count, 1)
    s = Step(17, batch * length, top_k, count, 1, width, torch.float32, torch.float32)
    want = s.out(s.tokens)
    experts.device_expert_combine(s.lau, s.rows, s.w, s.plan, want)
    for shape in [(batch, length, top_k)] + flat:
        y = s.out(s.tokens)
        experts.device_expert_combine(s.lau, s.rows, s.w.view(shape), s.plan, y)
        assert torch.equal(y, want)


# Tokens for several trips of every CTA of the combine and of its gradient, the
# last one ragged: at most five CTAs of 256 threads an SM stay resident, and a
# token takes from 2 threads (128 tokens a CTA) to 256.
MANY = [(200_003, 1, 8, torch.bfloat16, torch.float32),
        (100_003, 8, 4, torch.float32, torch.float32),
        (60_001, 2, 64, torch.bfloat16, torch.bfloat16),
        (15_001, 3, 33, torch.float32, torch.float32),
        (12_001, 17, 264, torch.bfloat16, torch.float32),
        (13_003, 3, 2056, torch.bfloat16, torch.float32),
        (7_001, 5, 512, torch.bfloat16, torch.float32),
        (4_003, 4, 1024, torch.float16, torch.float16),
        (3_001, 1, 1001, torch.float32, torch.float32),
        (3_001, 2, 1001, torch.float32, torch.bfloat16),
        (3_001, 9, 1001, torch.float32, torch.float32),
        (3_001, 6, 4096, torch.bfloat16, torch.float32),
        (3_001, 8, 2056, torch.float16, torch.float32),
        (3_001, 8, 4096, torch.bfloat16, torch.bfloat16)]


def close_here(got, want, mag, terms, dtype):
    tol = (terms + 1) * 2.0**-24 * mag
    tol = tol + HALF[dtype] * (want.abs() + tol) + TINY[dtype]
    assert torch.isfinite(got).all()
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("tokens,top_k,width,dtype,wdtype", MANY)
def test_combine_and_gradients_of_many_tokens(tokens, top_k, width, dtype, wdtype):
    """CTAs that work on token after token, the next one's slots held while
    this one is summed; rows that no slot uses hold NaN, and two runs are equal
    bit by bit."""
    count, align = 12, 16
    rng = np.random.default_rng(tokens + width)
    ids = make_ids(rng, tokens, top_k, count, "mixed", torch.int64)
    lau, plan = sort(ids, count, align)
    check_plan(plan, ids, count, align)
    g = torch.Generator(device="cuda").manual_seed(width)

    def normal(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    rows, grad = normal(plan.rows, width), normal(tokens, width)
    rows[plan.slot_of_row < 0] = NAN
    w = normal(tokens, top_k, dtype=wdtype)
    w[plan.row_of_slot < 0] = NAN

    slots = torch.nonzero(plan.row_of_slot.view(-1) >= 0).view(-1)
    at, token = plan.row_of_slot.view(-1)[slots].long(), slots // top_k
    w64 = w.double().view(-1)[slots].unsqueeze(1)

    def sums(terms):
        out = torch.zeros(2, tokens, width, dtype=torch.float64, device="cuda")
        return out[0].index_add_(0, token, terms), out[1].index_add_(0, token, terms.abs())

    def twice(make, call):
        """The outputs of a call, which a second one gives again."""
        first, second = make(), make()
        call(*first)
        call(*second)
        for a, b in zip(first, second):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        return first

    def filled(n, like=rows, to=33):
        return torch.full((n, like.shape[1]), to, dtype=like.dtype, device="cuda")

    y, = twice(lambda: [filled(tokens)],
               lambda y: experts.device_expert_combine(lau, rows, w, plan, y))
    close_here(y, *sums(rows[at].double() * w64), top_k, dtype)
    grad_x, = twice(lambda: [filled(tokens)],
                    lambda x: experts.device_expert_gather_backward(lau, rows, plan, x))
    close_here(grad_x, *sums(rows[at].double()), top_k, dtype)

    grad_rows, grad_w = twice(
        lambda: [filled(plan.rows), filled(tokens, w, 44)],
        lambda a, b: experts.device_expert_combine_backward(lau, grad, rows, w, plan, a, b))
    want = torch.full((plan.rows, width), 33.0, dtype=torch.float64, device="cuda")
    want[:int(plan.offsets[-1])] = 0
    want[at] = grad.double()[token] * w64
    close_here(grad_rows, want, want.abs(), 0, dtype)
    terms = grad.double()[token] * rows[at].double()
    dots = torch.zeros(2, tokens * top_k, dtype=torch.float64, device="cuda")
    dots[0, slots], dots[1, slots] = terms.sum(1), terms.abs().sum(1)
    close_here(grad_w.view(-1), dots[0], dots[1], width, wdtype)
    only, = twice(lambda: [filled(tokens, w, 44)],
                  lambda b: experts.device_expert_combine_backward(lau, grad, rows, w, plan, None, b))
    assert torch.equal(only, grad_w)

    moved = filled(plan.rows)
    experts.device_expert_gather(lau, grad, plan, moved)
    want.fill_(33)
    want[:int(plan.offsets[-1])] = 0
    want[at] = grad.double()[token]
    assert torch.equal(moved.double(), want)


@pytest.mark.parametrize("align", [1, 4096])
def test_padding_of_other_alignments(align):
    """No padding at all, and padding rows by the thousand."""
    s = Step(5, 21, 2, 3, align, 40, torch.float16, torch.float32, kind="uniform")
    rows, grad_rows = s.out(s.plan.rows), s.out(s.plan.rows)
    experts.device_expert_gather(s.lau, s.grad, s.plan, rows)
    experts.device_expert_combine_backward(s.lau, s.grad, s.rows, s.w, s.plan, grad_rows, None)
    end = int(s.offsets[-1])
    padding = torch.from_numpy(s.slot_of_row[:end] < 0).cuda()
    for out in (rows, grad_rows):
        assert (out[:end][padding] == 0).all() and (out[end:] == 33).all()
    used = torch.from_numpy(s.row_of_slot[s.used]).cuda()
    assert torch.equal(rows[used], s.grad[torch.from_numpy(s.used // 2).cuda()])
