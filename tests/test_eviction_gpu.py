"""Cache eviction on the GPU against plain restatements: totals of attention
weights in 64 bits, the selection by numpy's lexsort, the compaction by
indexing.  Masked weights and totals behind a sequence's length hold NaN.

Tolerance of a total: a sum of n terms in fp32 is off by at most n * 2^-24
times the sum of the terms' magnitudes, the decayed old total among them."""
import numpy as np
import pytest
import torch

from rccl_b200 import cub, eviction

pytestmark = pytest.mark.gpu
NAN = float("nan")


def launch():
    return cub.Program.load("cuda:0").on()


def lengths_of(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def visible(B, Q, S, lens, causal):
    """(B, Q, S): what query q of sequence b sees."""
    at = np.arange(S)
    end = np.asarray(lens)[:, None, None] + np.zeros((B, Q, 1), np.int64)
    if causal:
        end = end - Q + 1 + np.arange(Q)[None, :, None]
    return at < end


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("H,G,Q,S,lens", [
    (1, 1, 1, 1, [1, 0]), (2, 1, 1, 64, [64, 1, 0, 33]), (2, 4, 1, 257, [257, 256, 8, 9]),
    (1, 8, 5, 100, [100, 3, 5, 4, 99]), (3, 2, 64, 1000, [1000, 64, 63, 1, 0, 500]),
    (2, 2, 130, 4099, [4099, 4098, 131]), (1, 4, 512, 2048, [2048, 700]),
    (1, 1, 0, 16, [16, 3])])
def test_totals(H, G, Q, S, lens, causal, dtype):
    rng = np.random.default_rng(S + Q)
    B = len(lens)
    w = rng.random((B, H * G, Q, S)).astype(np.float32)
    w = torch.from_numpy(w).to(dtype)
    seen = visible(B, Q, S, lens, causal)
    w[torch.from_numpy(~seen)[:, None].expand(w.shape)] = NAN
    old = rng.random((B, H, S)).astype(np.float32)
    live = np.arange(S) < np.asarray(lens)[:, None, None]
    old = np.where(live, old, np.float32(NAN))
    scores = torch.from_numpy(old).cuda()
    eviction.device_attention_weight_add(launch(), w.cuda(), scores, lengths_of(lens), decay=0.75,
                                         causal=causal)
    terms = np.where(seen[:, None], w.double().numpy(), 0).reshape(B, H, G * Q, S)
    want = 0.75 * old.astype(np.float64) + terms.sum(2)
    got = scores.double().cpu().numpy()
    tol = (G * Q + 2) * 2.0**-24 * np.abs(want)
    seen_total = np.broadcast_to(live, want.shape)
    assert (np.abs(got - want)[seen_total] <= tol[seen_total]).all()
    assert np.isnan(got[~seen_total]).all()


def test_totals_without_lengths_strided_and_misaligned():
    """Weights and totals as views of larger, odd allocations; every position
    in use; lengths beyond the capacity and below zero are clamped."""
    rng = np.random.default_rng(2)
    B, H, G, Q, S = 3, 2, 2, 4, 77
    big = torch.from_numpy(rng.random((Q, B, H * G, S + 5)).astype(np.float32)).cuda().bfloat16()
    w = big[..., 3:3 + S].permute(1, 2, 0, 3)
    wide = torch.from_numpy(rng.random((H, B, S + 3)).astype(np.float32)).cuda()
    before = wide.clone()
    scores = wide[..., 1:1 + S].transpose(0, 1)
    want = scores.double() + w.double().view(B, H, G, Q, S).sum((2, 3))
    eviction.device_attention_weight_add(launch(), w, scores)
    assert ((scores.double() - want).abs() <= 18 * 2.0**-24 * want).all()
    assert torch.equal(wide[..., 0], before[..., 0])
    assert torch.equal(wide[..., 1 + S:], before[..., 1 + S:])
    scores = torch.zeros(B, H, S, device="cuda")
    single = w[:, :, 0].float().contiguous()
    eviction.device_attention_weight_add(launch(), single, scores, lengths_of([1000, -3, 5]))
    want = single.double().view(B, H, G, S).sum(2)
    want[1] = 0
    want[2, :, 5:] = 0
    assert ((scores.double() - want).abs() <= 3 * 2.0**-24 * want).all()


def selected(scores, lens, budget, sinks, recent):
    B, H, _ = scores.shape
    kept = np.full((B, H, budget), -1, np.int64)
    for b in range(B):
        n = lens[b]
        for h in range(H):
            if n <= budget:
                kept[b, h, :n] = np.arange(n)
                continue
            part = scores[b, h, sinks:n - recent].astype(np.float64)
            part = np.where(np.isnan(part), -np.inf, part)
            best = np.lexsort((np.arange(part.size), -part))[:budget - sinks - recent] + sinks
            kept[b, h] = np.sort(np.concatenate(
                [np.arange(sinks), best, np.arange(n - recent, n)]))
    return kept, np.minimum(lens, budget)


def make_scores(rng, kind, shape):
    if kind == "heavy":
        x = np.exp(1.5 * rng.normal(size=shape))
        x[rng.random(shape) < 0.05] = 0
    elif kind == "ties":
        x = rng.integers(0, 3, shape).astype(np.float64)
    elif kind == "equal":
        x = np.full(shape, 0.25)
    elif kind == "close":  # neighbouring floats: every bit decides
        x = (np.float32(1).view(np.uint32) + rng.integers(0, 5000, shape).astype(np.uint32)).view(
            np.float32)
    else:  # special values of both signs
        x = rng.normal(size=shape)
        special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38])
        hit = rng.random(shape) < 0.7
        x[hit] = rng.choice(special, int(hit.sum()))
    return x.astype(np.float32)


@pytest.mark.parametrize("kind", ["heavy", "ties", "equal", "close", "special"])
@pytest.mark.parametrize("H,S,budget,sinks,recent,lens", [
    (1, 1, 1, 0, 0, [1, 0]), (2, 2, 1, 0, 0, [2, 1, 0]), (2, 2, 1, 1, 0, [2]),
    (1, 40, 64, 4, 8, [40, 0]),                       # budget above the capacity
    (2, 100, 33, 4, 8, [100, 34, 33, 32, 0]), (2, 100, 12, 4, 8, [100, 13]),
    (3, 1025, 1024, 4, 64, [1025, 1024]), (2, 1025, 1, 0, 1, [1025, 2]),
    (1, 5000, 700, 0, 0, [5000, 4999, 701]), (1, 5000, 4990, 16, 512, [5000, 4991]),
    (2, 20011, 3001, 4, 100, [20011, 8192]), (1, 140_000, 9000, 4, 512, [140_000]),
    (40, 300, 50, 2, 10, [300, 299, 70, 51])])
def test_select(H, S, budget, sinks, recent, lens, kind):
    rng = np.random.default_rng(S + budget)
    B = len(lens)
    scores = make_scores(rng, kind, (B, H, S))
    # what lies behind a sequence must not matter
    scores[np.broadcast_to(np.arange(S) >= np.asarray(lens)[:, None, None], scores.shape)] = np.inf
    wide = torch.full((B, H, S + 2), float("inf"), device="cuda")
    view = wide[..., 1:1 + S]
    view.copy_(torch.from_numpy(scores))
    kept = torch.full((B, H, budget), 99, dtype=torch.int32, device="cuda")
    n = torch.full((B,), 99, dtype=torch.int32, device="cuda")
    eviction.device_cache_select(launch(), view, lengths_of(lens), kept, n, sinks, recent)
    want, want_n = selected(scores, lens, budget, sinks, recent)
    assert np.array_equal(kept.cpu().numpy(), want)
    assert np.array_equal(n.cpu().numpy(), want_n)


@pytest.mark.parametrize("kind", ["ties", "close", "heavy"])
@pytest.mark.parametrize("B,S,budget", [(1, 300_000, 20_000), (170, 9000, 500), (150, 33_000, 32_990)])
def test_select_over_many_pages(B, S, budget, kind):
    """Slices beyond what a CTA holds in registers and in shared memory, and more
    heads than run at once."""
    rng = np.random.default_rng(S)
    scores = make_scores(rng, kind, (B, 1, S))
    lens = [S] + [int(x) for x in rng.integers(budget, S + 1, B - 1)]
    kept = torch.zeros(B, 1, budget, dtype=torch.int32, device="cuda")
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    eviction.device_cache_select(launch(), torch.from_numpy(scores).cuda(), lengths_of(lens), kept,
                                 n, 3, 5)
    want, want_n = selected(scores, lens, budget, 3, 5)
    assert np.array_equal(kept.cpu().numpy(), want)
    assert np.array_equal(n.cpu().numpy(), want_n)


def test_select_without_lengths_and_clamped():
    rng = np.random.default_rng(9)
    scores = make_scores(rng, "heavy", (3, 2, 200))
    t = torch.from_numpy(scores).cuda()
    kept = torch.zeros(3, 2, 50, dtype=torch.int32, device="cuda")
    n = torch.zeros(3, dtype=torch.int32, device="cuda")
    eviction.device_cache_select(launch(), t, None, kept, n)
    assert np.array_equal(kept.cpu().numpy(), selected(scores, [200] * 3, 50, 0, 0)[0])
    eviction.device_cache_select(launch(), t, lengths_of([10**6, -1, 60]), kept, n)
    assert np.array_equal(kept.cpu().numpy(), selected(scores, [200, 0, 60], 50, 0, 0)[0])
    assert n.tolist() == [50, 0, 50]


def random_kept(rng, B, H, S, budget, lens):
    kept = np.full((B, H, budget), -1, np.int32)
    for b in range(B):
        for h in range(H):
            n = min(lens[b], budget)
            kept[b, h, :n] = np.sort(rng.choice(max(lens[b], 1), n, replace=False))
    return kept, np.minimum(lens, budget).astype(np.int32)


def moved(src, kept, n, old):
    want = old.clone()
    for b in range(kept.shape[0]):
        for h in range(kept.shape[1]):
            want[b, h, :n[b]] = src[b, h][torch.from_numpy(kept[b, h, :n[b]]).long()]
    return want


def bits(t):
    return t.contiguous().view(torch.uint8)


def values(rng, shape, dtype):
    return torch.from_numpy(rng.integers(0, 250, shape)).to(dtype)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("layout", ["bhsd", "bshd", "packed"])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float32, 5), (torch.uint8, 3),
                                     (torch.float16, 80), (torch.int64, 1), (torch.bfloat16, 577)])
@pytest.mark.parametrize("H,S,budget,lens", [
    (1, 1, 1, [1, 0]), (2, 50, 17, [50, 17, 3, 0, 18]), (2, 700, 699, [700, 699, 698]),
    (3, 300, 20, [300, 21])])
def test_compact(H, S, budget, lens, dtype, D, layout, in_place):
    rng = np.random.default_rng(S + D)
    B = len(lens)
    kept, n = random_kept(rng, B, H, S, budget, lens)

    def arrays(count):
        """Two (B, H, count, D) views: keys and values."""
        if layout == "packed":
            both = values(rng, (B, count, 2, H, D), dtype).cuda()
            return [both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)]
        shape = (B, H, count, D) if layout == "bhsd" else (B, count, H, D)
        pair = [values(rng, shape, dtype).cuda() for _ in range(2)]
        return pair if layout == "bhsd" else [t.transpose(1, 2) for t in pair]

    src = arrays(S) + [torch.from_numpy(rng.random((B, H, S)).astype(np.float32)).cuda()]
    dst = src if in_place else arrays(budget + 1) + [torch.zeros(B, H, budget + 1, device="cuda")]
    want = [moved(s.cpu(), kept, n, d.cpu()) for s, d in zip(src, dst)]
    kept_d, n_d = torch.from_numpy(kept).cuda(), torch.from_numpy(n).cuda()
    if in_place:
        eviction.device_cache_compact(launch(), kept_d, n_d, src)
    else:
        eviction.device_cache_compact(launch(), kept_d, n_d, src, dst)
    for got, w in zip(dst, want):
        assert torch.equal(bits(got.cpu()), bits(w))


@pytest.mark.parametrize("in_place", [False, True])
def test_compact_long_rows_in_order(in_place):
    """Long moves over many steps: one early position leaves, so nearly every
    row moves down by one."""
    B, H, S, D = 2, 2, 5000, 128
    rng = np.random.default_rng(4)
    k = torch.from_numpy(rng.integers(0, 30000, (B, H, S, D))).to(torch.int16).cuda()
    lens, budget = [S, S - 1], S - 1
    kept, n = random_kept(rng, B, H, S, budget, lens)
    kept[0, 0] = np.delete(np.arange(S), 1)
    want = moved(k.cpu(), kept, n, k.cpu()[:, :, :S] if in_place else torch.zeros(
        B, H, budget, D, dtype=torch.int16))
    dst = k if in_place else torch.zeros(B, H, budget, D, dtype=torch.int16, device="cuda")
    eviction.device_cache_compact(launch(), torch.from_numpy(kept).cuda(),
                                  torch.from_numpy(n).cuda(), [k], [dst])
    assert torch.equal(dst.cpu(), want)


@pytest.mark.parametrize("in_place", [False, True])
def test_positions_out_of_range_are_skipped(in_place):
    kept = torch.tensor([[[0, 2, 9, -5, 2**31 - 1, 7]]], dtype=torch.int32, device="cuda")
    n = torch.tensor([1000], dtype=torch.int32, device="cuda")  # clamped to the budget
    k = torch.arange(8, dtype=torch.float32, device="cuda").view(1, 1, 8, 1) + 1
    dst = k if in_place else torch.full((1, 1, 6, 1), -1.0, device="cuda")
    eviction.device_cache_compact(launch(), kept, n, [k], [dst])
    want = [1, 3, 3, 4, 5, 8, 7, 8] if in_place else [1, 3, -1, -1, -1, 8]
    assert dst.view(-1).tolist() == want


@pytest.mark.parametrize("captured", [False, True])
def test_a_bounded_cache_over_many_tokens(captured):
    """Tokens are appended, their weights added, and the full cache is cut to
    its budget in place, eagerly and as a replayed graph; the same cache kept in
    numpy holds the same positions, totals and rows."""
    B, H, G, S, budget, sinks, recent, D = 2, 2, 2, 48, 32, 2, 8, 16
    rng = np.random.default_rng(8)
    program = cub.Program.load("cuda:0")
    k = torch.zeros(B, H, S, D, device="cuda")
    v = torch.zeros(B, S, H, D, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    scores = torch.zeros(B, H, S, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    kept = torch.zeros(B, H, budget, dtype=torch.int32, device="cuda")
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    w = torch.zeros(B, H * G, S, device="cuda")
    hk, hs, hl = np.zeros((B, H, S, D), np.float32), np.zeros((B, H, S), np.float32), 0

    def evict(lau):
        eviction.device_cache_select(lau, scores, lens, kept, n, sinks, recent)
        eviction.device_cache_compact(lau, kept, n, [k, v, scores])
        lens.copy_(n)

    graph = None
    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            evict(program.on(side))  # lengths are zero: nothing moves
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            evict(program.on(torch.cuda.current_stream()))
    for step in range(100):
        new = rng.normal(size=(B, H, D)).astype(np.float32)
        k[:, :, hl] = torch.from_numpy(new).cuda()
        v[:, :, hl] = torch.from_numpy(new).cuda().bfloat16()
        scores[:, :, hl] = 0
        hk[:, :, hl], hs[:, :, hl] = new, 0
        hl += 1
        lens.fill_(hl)
        # multiples of 2^-10 below 1: their sums are exact in any order
        hw = rng.integers(0, 1024, (B, H * G, S)).astype(np.float32) / 1024
        w.copy_(torch.from_numpy(hw))
        eviction.device_attention_weight_add(program.on(), w, scores, lens)
        hs[:, :, :hl] += hw.reshape(B, H, G, S).sum(2)[:, :, :hl]
        if hl == S:
            graph.replay() if captured else evict(program.on())
            want, _ = selected(hs, [hl] * B, budget, sinks, recent)
            for b in range(B):
                for h in range(H):
                    hk[b, h, :budget] = hk[b, h, want[b, h]]
                    hs[b, h, :budget] = hs[b, h, want[b, h]]
            hl = budget
            assert lens.tolist() == [budget] * B
    assert np.array_equal(k.cpu().numpy()[:, :, :hl], hk[:, :, :hl])
    assert np.array_equal(scores.cpu().numpy()[:, :, :hl], hs[:, :, :hl])
    rounded = torch.from_numpy(hk[:, :, :hl]).bfloat16()
    assert torch.equal(v.cpu()[:, :, :hl], rounded)


def one_allocation(rng, B, S, H, widths):
    """Keys, values (bf16) and totals (f32) of every position side by side in
    one allocation: (B, H, S, width) views of unequal widths and the totals."""
    k_width, v_width = widths
    block = torch.from_numpy(rng.integers(0, 256, (B, S, H, 2 * (k_width + v_width) + 4),
                                          dtype=np.uint8)).cuda()
    k = block[..., :2 * k_width].view(torch.bfloat16).transpose(1, 2)
    v = block[..., 2 * k_width:-4].view(torch.bfloat16).transpose(1, 2)
    scores = block[..., -4:].view(torch.float32)[..., 0].transpose(1, 2)
    return block, [k, v, scores]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("widths", [(64, 8), (16, 48), (5, 3), (2, 2)])
@pytest.mark.parametrize("H", [1, 3])
def test_compact_of_unequal_rows_in_one_allocation(H, widths, in_place):
    """Arrays that interleave without sharing a byte move together, whatever
    their rows' widths; nothing beside the moved rows changes."""
    rng = np.random.default_rng(sum(widths) + H)
    B, S, budget, lens = 2, 90, 31, [90, 40]
    kept, n = random_kept(rng, B, H, S, budget, lens)
    block, src = one_allocation(rng, B, S, H, widths)
    to, dst = (block, src) if in_place else one_allocation(rng, B, budget, H, widths)
    want = to.clone()
    for b in range(B):
        for h in range(H):
            at = torch.from_numpy(kept[b, h, :n[b]]).long().cuda()
            want[b, :n[b], h] = block[b, at, h]
    eviction.device_cache_compact(launch(), torch.from_numpy(kept).cuda(),
                                  torch.from_numpy(n).cuda(), src, None if in_place else dst)
    assert torch.equal(to, want)


def test_totals_beside_the_weights_in_one_allocation():
    rng = np.random.default_rng(12)
    B, H, G, S = 3, 2, 2, 70
    both = torch.from_numpy(rng.random((B, H * G + H, S)).astype(np.float32)).cuda()
    before = both.clone()
    w, scores = both[:, :H * G], both[:, H * G:]
    eviction.device_attention_weight_add(launch(), w, scores, lengths_of([70, 0, 33]))
    want = before.double()
    for b, n in enumerate([70, 0, 33]):
        want[b, H * G:, :n] += before[b, :H * G, :n].double().view(H, G, n).sum(1)
    assert torch.equal(w, before[:, :H * G])
    assert ((both.double() - want).abs() <= 4 * 2.0**-24 * want).all()


@pytest.mark.parametrize("Q,G,S", [(1, 2, 40), (3, 2, 1000), (40, 4, 520), (41, 1, 333)])
def test_unseen_weights_add_nothing_whatever_they_hold(Q, G, S):
    """Infinities of both signs, NaN and the type's largest and lowest values in
    every place that a query does not see give the same bits as zeros."""
    rng = np.random.default_rng(Q)
    B, lens = 3, [S, S // 2 + 1, 2]
    w = torch.from_numpy(rng.random((B, G, Q, S)).astype(np.float32)).bfloat16()
    seen = torch.from_numpy(visible(B, Q, S, lens, True))[:, None].expand(w.shape)
    odd = [float("inf"), -float("inf"), NAN, torch.finfo(w.dtype).max, torch.finfo(w.dtype).min]
    got = []
    for fill in [torch.zeros(w.shape, dtype=w.dtype),
                 torch.tensor(odd, dtype=w.dtype)[torch.randint(5, w.shape)]]:
        scores = torch.ones(B, 1, S, device="cuda")
        eviction.device_attention_weight_add(launch(), torch.where(seen, w, fill).cuda(), scores,
                                             lengths_of(lens), causal=True)
        got.append(scores.cpu())
    assert torch.equal(*got)


@pytest.mark.parametrize("D", [1, 64, 129])
def test_compact_out_of_place_in_any_order_with_repeats(D):
    rng = np.random.default_rng(D)
    B, H, S, budget = 2, 3, 60, 41
    k = torch.from_numpy(rng.normal(size=(B, H, S, D))).half().cuda()
    kept = rng.integers(0, S, (B, H, budget)).astype(np.int32)
    kept[:, :, 1], kept[:, :, 2] = kept[:, :, 0], kept[:, :, 0]
    n = np.array([budget, 7], np.int32)
    dst = torch.full((B, H, budget, D), 5, dtype=k.dtype, device="cuda")
    want = moved(k.cpu(), kept, n, dst.cpu())
    eviction.device_cache_compact(launch(), torch.from_numpy(kept).cuda(),
                                  torch.from_numpy(n).cuda(), [k], [dst])
    assert torch.equal(dst.cpu(), want)


def test_in_place_a_position_below_its_place_does_not_move():
    kept = torch.tensor([[[0, 0, 4, 5, 5, 1]]], dtype=torch.int32, device="cuda")
    k = torch.arange(8, dtype=torch.float32, device="cuda").view(1, 1, 8, 1) + 1
    eviction.device_cache_compact(launch(), kept, lengths_of([6]), [k])
    assert k.view(-1).tolist() == [1, 2, 5, 6, 6, 6, 7, 8]
