"""Operators of the token-routing and cache-eviction modules, as cases.

Expert routing (rccl_b200.experts): token slots sorted by expert, rows gathered
into expert order, expert outputs combined back with their weights, and the
gradients of both.  Cache eviction (rccl_b200.eviction): attention weights
accumulated per cached position, the heaviest positions of every head selected,
and the cache's rows moved together.

A case is a dict of plain values.  `prepare` makes its inputs, `run` one pass,
`exact` the same outputs in 64 bits, `work` the bytes and operations a pass
cannot do without.  With `own` false a pass is elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
IDS = {"i32": torch.int32, "i64": torch.int64}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One decode step of 16 sequences: only the plan, launch latency.
        dict(name="sort_decode", op="sort", T=16, K=8, E=128, align=1, drop=0.0, ids="i32"),
        # A prefill batch of 64 Ki tokens, expert segments padded to GEMM
        # tiles; 2% of the slots belong to padding tokens and are dropped.
        dict(name="sort_prefill", op="sort", T=65536, K=8, E=256, align=128, drop=0.02, ids="i64"),
        # One decode step through a layer: plan, dispatch and combine.
        dict(name="forward_decode", op="forward", T=16, K=8, E=128, H=4096, dtype="bf16",
             weights="f32", align=1, drop=0.0, ids="i32"),
        # A prefill chunk with an odd number of tokens.
        dict(name="forward_prefill", op="forward", T=8191, K=6, E=64, H=2048, dtype="bf16",
             weights="bf16", align=64, drop=0.01, ids="i64"),
        # A small fp32 training step whose rows are 4 bytes short of vectors.
        dict(name="train_f32_odd", op="train", T=1023, K=2, E=8, H=1001, dtype="f32",
             weights="f32", align=1, drop=0.05, ids="i64"),
        # A half-precision training step.
        dict(name="train_f16", op="train", T=4096, K=4, E=32, H=5120, dtype="f16",
             weights="f16", align=16, drop=0.0, ids="i32"),
        # The largest: 16 Ki tokens to 8 of 128 experts with tile padding.
        dict(name="train_bf16_large", op="train", T=16384, K=8, E=128, H=4096, dtype="bf16",
             weights="f32", align=128, drop=0.0, ids="i64"),
        # One generated token per sequence: its weights join the totals.
        dict(name="add_decode", op="add", B=32, Hq=32, Hkv=8, Q=1, S=8192, dtype="bf16",
             causal=False, decay=1.0),
        # The last 256 queries of a prompt vote on its positions.
        dict(name="add_window", op="add", B=2, Hq=32, Hkv=4, Q=256, S=16384, dtype="bf16",
             causal=True, decay=0.9),
        # A long context's heads cut to 4 Ki positions: the selection alone.
        dict(name="select_long", op="select", B=8, H=8, S=65536, budget=4096, sinks=4, recent=512),
        # After a prompt: select, then keys, values and totals into a new cache.
        dict(name="evict_prompt", op="evict", B=8, H=8, S=16384, budget=2048, sinks=4, recent=64,
             D=128, dtype="bf16", layout="bhsd"),
        # During generation: 8 of 4104 positions leave a full cache, in place.
        dict(name="compact_step", op="compact", B=32, H=8, S=4104, budget=4096, D=128,
             dtype="bf16", layout="bhsd", inplace=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "forward", "forward", "train", "train", "add", "add", "select",
                     "evict", "compact"])
    if op in ("sort", "forward", "train"):
        E = rng.choice([4, 8, 16, 60, 64, 128, 160, 256, 384])
        K = rng.choice([k for k in (1, 2, 3, 4, 6, 8) if k <= E])
        T = _log(rng, 8, 65536) if op == "sort" else _log(rng, 1, 16384)
        case = dict(op=op, T=T, K=K, E=E,
                    align=rng.choice([1, 1, 8, 16, 64, 128]),
                    drop=rng.choice([0.0, 0.0, 0.03, 0.3]), ids=rng.choice(["i32", "i64"]))
        if op != "sort":
            H = _log(rng, 64, 8192)
            H = H if rng.random() < 0.25 else max(64, H // 64 * 64)
            case["T"] = max(1, min(case["T"], (3 << 26) // (K * H)))
            if case["T"] * K < E * 16:  # few tokens: no wide padding
                case["align"] = min(case["align"], 8)
            case.update(H=H, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                        weights=rng.choice(["f32", "same"]))
            if case["weights"] == "same":
                case["weights"] = case["dtype"]
        return case
    D = rng.choice([64, 80, 96, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "add":
        S = _log(rng, 16, 32768)
        S = S if rng.random() < 0.3 else max(16, S // 8 * 8)
        G = rng.choice([1, 2, 4, 8])
        Q = rng.choice([1, 1, _log(rng, 2, 512)])
        B = max(1, min(_log(rng, 1, 64), (1 << 28) // (S * G * Q * Hkv)))
        return dict(op=op, B=B, Hq=Hkv * G, Hkv=Hkv, Q=min(Q, S), S=S, dtype=dtype,
                    causal=Q > 1 and rng.random() < 0.7, decay=rng.choice([1.0, 0.99]))
    S = _log(rng, 64, 131072 if op == "select" else 32768)
    limit = 1 << 23 if op == "select" else (1 << 28) // D
    B = max(1, min(_log(rng, 1, 64), limit // (S * Hkv)))
    budget = max(1, int(S * rng.uniform(0.05, 0.999)))
    sinks, recent = min(4, budget // 4), min(_log(rng, 1, 512), budget // 4)
    case = dict(op=op, B=B, H=Hkv, S=S, budget=budget)
    if op != "compact":
        case.update(sinks=sinks, recent=recent)
    if op != "select":
        case.update(D=D, dtype=dtype, layout=rng.choice(["bhsd", "bshd"]))
    if op == "compact":
        case["inplace"] = rng.random() < 0.5
    return case


def _rows(case):
    """Rows that T*K slots can take when every expert's segment is a multiple of align."""
    n, a = case["T"] * case["K"], case["align"]
    return (n + min(case["E"], n) * (a - 1)) // a * a


def work(case):
    op = case["op"]
    if op in ("sort", "forward", "train"):
        n, E = case["T"] * case["K"], case["E"]
        plan = n * (4 if case["ids"] == "i32" else 8) + 4 * n + 4 * _rows(case) + 4 * (2 * E + 1)
        if op == "sort":
            return {"bytes": plan, "flops": 0}
        # Rows that carry a slot; what padding rows cost is left out.
        x = case["T"] * case["H"] * BYTES[case["dtype"]]
        rows = n * case["H"] * BYTES[case["dtype"]]
        w = n * BYTES[case["weights"]]
        total, flops = plan + (x + rows) + (rows + w + x), 2 * n * case["H"]
        if op == "train":
            total += (x + 2 * rows + 2 * w) + (rows + x)
            flops += 4 * n * case["H"]
        return {"bytes": total, "flops": flops}
    if op == "add":
        w = case["B"] * case["Hq"] * case["Q"] * case["S"]
        s = case["B"] * case["Hkv"] * case["S"]
        # Ragged lengths average 3/4 of the capacity (see prepare).
        part = 0.75 if case["B"] > 1 else 1.0
        return {"bytes": part * (w * BYTES[case["dtype"]] + 8 * s), "flops": part * w}
    heads = case["B"] * case["H"]
    part = 0.75 if case["B"] > 1 else 1.0
    select = heads * (4 * case["S"] * part + 4 * case["budget"])
    if op == "select":
        return {"bytes": select, "flops": 0}
    row = 2 * case["D"] * BYTES[case["dtype"]] + 4
    moved = heads * case["budget"] * (2 * row + 4)
    return {"bytes": moved + (select if op == "evict" else 0), "flops": 0}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _lengths(B, S, low, g):
    """Ragged lengths in [low, S]; the first sequence is full."""
    lens = torch.randint(low, S + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = S
    return lens


def _prepare_experts(case, g):
    T, K, E = case["T"], case["K"], case["E"]
    # Router choices: K distinct experts per token, popular ones more often.
    bias = torch.randn(E, generator=g, device="cuda")
    noise = torch.rand(T, E, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
    logits = bias - torch.log(-torch.log(noise))
    top, ids = logits.topk(K, dim=1)
    if case["drop"]:
        gone = torch.rand(T, generator=g, device="cuda") < case["drop"]
        ids[gone] = -1
    s = {"case": case, "ids": ids.to(IDS[case["ids"]]).contiguous()}
    R = _rows(case)
    if case["op"] != "sort":
        H, dt, wt = case["H"], DTYPES[case["dtype"]], DTYPES[case["weights"]]
        s["weights"] = torch.softmax(top, dim=1).to(wt).contiguous()
        s["x"] = torch.randn(T, H, generator=g, device="cuda", dtype=dt)
        s["expert_out"] = torch.randn(R, H, generator=g, device="cuda", dtype=dt)
        s["rows"] = torch.zeros(R, H, device="cuda", dtype=dt)
        s["y"] = torch.zeros(T, H, device="cuda", dtype=dt)
        if case["op"] == "train":
            s["grad_y"] = torch.randn(T, H, generator=g, device="cuda", dtype=dt)
            s["grad_rows"] = torch.randn(R, H, generator=g, device="cuda", dtype=dt)
            s["grad_out"] = torch.zeros(R, H, device="cuda", dtype=dt)
            s["grad_weights"] = torch.zeros(T, K, device="cuda", dtype=wt)
            s["grad_x"] = torch.zeros(T, H, device="cuda", dtype=dt)
    if own:
        from rccl_b200 import cub, experts
        s["launch"] = cub.Program.load("cuda").on()
        s["plan"] = experts.device_expert_plan(s["launch"], T, K, E, case["align"])
    return s


def _prepare_add(case, g):
    B, Hq, Hkv, Q, S = (case[k] for k in ("B", "Hq", "Hkv", "Q", "S"))
    lens = _lengths(B, S, S // 2, g)
    # Attention weights: a softmax over what each query sees, zero elsewhere.
    logits = 2 * torch.randn(B, Hq, Q, S, generator=g, device="cuda")
    at = torch.arange(S, device="cuda")
    end = lens.view(B, 1, 1, 1).long()
    if case["causal"]:
        end = end - Q + 1 + torch.arange(Q, device="cuda").view(1, 1, Q, 1)
    logits = logits.masked_fill_(at >= end, -1e30)
    weights = torch.softmax(logits, dim=-1).masked_fill_(at >= end, 0).to(DTYPES[case["dtype"]])
    s = {"case": case, "weights": weights, "lengths": lens,
         "scores": torch.rand(B, Hkv, S, generator=g, device="cuda")}
    if own:
        from rccl_b200 import cub
        s["launch"] = cub.Program.load("cuda").on()
    return s


def _prepare_cache(case, g):
    B, H, S, budget = (case[k] for k in ("B", "H", "S", "budget"))
    lens = _lengths(B, S, S // 2, g)
    # Totals of attention weights: a heavy tail, some positions never seen.
    scores = torch.exp(1.5 * torch.randn(B, H, S, generator=g, device="cuda"))
    scores.masked_fill_(torch.rand(B, H, S, generator=g, device="cuda") < 0.03, 0)
    s = {"case": case, "scores": scores, "lengths": lens}
    s["kept"] = torch.zeros(B, H, budget, device="cuda", dtype=torch.int32)
    s["kept_lengths"] = torch.zeros(B, device="cuda", dtype=torch.int32)
    if case["op"] != "select":
        shape = (B, H, S, case["D"]) if case["layout"] == "bhsd" else (B, S, H, case["D"])
        dt = DTYPES[case["dtype"]]
        view = (lambda t: t) if case["layout"] == "bhsd" else (lambda t: t.transpose(1, 2))
        s["k"] = view(torch.randn(shape, generator=g, device="cuda", dtype=dt))
        s["v"] = view(torch.randn(shape, generator=g, device="cuda", dtype=dt))
        if not case.get("inplace"):
            new = shape[:2] + (budget, case["D"]) if case["layout"] == "bhsd" else \
                (B, budget, H, case["D"])
            s["new_k"] = view(torch.zeros(new, device="cuda", dtype=dt))
            s["new_v"] = view(torch.zeros(new, device="cuda", dtype=dt))
            s["new_scores"] = torch.zeros(B, H, budget, device="cuda")
    if case["op"] == "compact":
        # Positions kept by an earlier selection: a random ascending subset.
        draws = torch.rand(B, H, S, generator=g, device="cuda")
        draws.masked_fill_(torch.arange(S, device="cuda") >= lens.view(B, 1, 1), -1)
        kept = draws.topk(budget, dim=2).indices.sort(dim=2).values
        n = torch.clamp(lens, max=budget)
        slots = torch.arange(budget, device="cuda")
        short = (lens <= budget).view(B, 1, 1)
        kept = torch.where(short, slots, kept)
        s["kept"] = torch.where(slots < n.view(B, 1, 1), kept, -1).to(torch.int32)
        s["kept_lengths"] = n.to(torch.int32)
    if own:
        from rccl_b200 import cub
        s["launch"] = cub.Program.load("cuda").on()
    return s


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] in ("sort", "forward", "train"):
        return _prepare_experts(case, g)
    return _prepare_add(case, g) if case["op"] == "add" else _prepare_cache(case, g)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op in ("sort", "forward", "train"):
        return _run_experts(state) if own else _plain_experts(state)
    if op == "add":
        return _run_add(state) if own else _plain_add(state)
    return _run_cache(state) if own else _plain_cache(state)


def _run_experts(s):
    from rccl_b200 import experts
    launch, plan, op = s["launch"], s["plan"], s["case"]["op"]
    experts.device_expert_sort(launch, s["ids"], plan)
    out = {"row_of_slot": plan.row_of_slot, "slot_of_row": plan.slot_of_row,
           "offsets": plan.offsets, "counts": plan.counts}
    if op == "sort":
        return out
    experts.device_expert_gather(launch, s["x"], plan, s["rows"])
    experts.device_expert_combine(launch, s["expert_out"], s["weights"], plan, s["y"])
    out.update(rows=s["rows"], y=s["y"])
    if op == "train":
        experts.device_expert_combine_backward(launch, s["grad_y"], s["expert_out"], s["weights"],
                                               plan, s["grad_out"], s["grad_weights"])
        experts.device_expert_gather_backward(launch, s["grad_rows"], plan, s["grad_x"])
        out.update(grad_out=s["grad_out"], grad_weights=s["grad_weights"], grad_x=s["grad_x"])
    return out


def _run_add(s):
    from rccl_b200 import eviction
    eviction.device_attention_weight_add(s["launch"], s["weights"], s["scores"], s["lengths"],
                                         decay=s["case"]["decay"], causal=s["case"]["causal"])
    return s["scores"]


def _run_cache(s):
    from rccl_b200 import eviction
    case, launch = s["case"], s["launch"]
    if case["op"] != "compact":
        eviction.device_cache_select(launch, s["scores"], s["lengths"], s["kept"],
                                     s["kept_lengths"], sinks=case["sinks"],
                                     recent=case["recent"])
        if case["op"] == "select":
            return {"kept": s["kept"], "kept_lengths": s["kept_lengths"]}
    old = [s["k"], s["v"], s["scores"]]
    new = old if case.get("inplace") else [s["new_k"], s["new_v"], s["new_scores"]]
    eviction.device_cache_compact(launch, s["kept"], s["kept_lengths"], old, new)
    out = {"k": new[0], "v": new[1], "scores": new[2]}
    if case["op"] == "evict":
        out.update(kept=s["kept"], kept_lengths=s["kept_lengths"])
    return out


def _plain_sort(case, ids):
    E, a, R, n = case["E"], case["align"], _rows(case), ids.numel()
    flat = ids.reshape(-1).long()
    flat = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(flat, stable=True)
    key = flat[order]
    counts = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    counts.scatter_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(counts, 0) - counts
    padded = (counts + a - 1) // a * a
    start = torch.cumsum(padded, 0) - padded
    row = torch.arange(n, device="cuda") - first[key] + start[key]
    row = torch.where(key < E, row, -1)
    row_of_slot = torch.empty_like(row)
    row_of_slot[order] = row
    slot_of_row = torch.full((R + 1,), -1, dtype=torch.int64, device="cuda")
    slot_of_row[torch.where(row < 0, R, row)] = torch.where(row < 0, -1, order)
    return (row_of_slot.view(ids.shape).int(), slot_of_row[:R].int(), start.int(),
            counts[:E].int())


def _plain_experts(s):
    case = s["case"]
    row_of_slot, slot_of_row, offsets, counts = _plain_sort(case, s["ids"])
    out = {"row_of_slot": row_of_slot, "slot_of_row": slot_of_row, "offsets": offsets,
           "counts": counts}
    if case["op"] == "sort":
        return out
    T, K, H, R = case["T"], case["K"], case["H"], _rows(case)
    dt = DTYPES[case["dtype"]]
    seen = row_of_slot.view(-1, 1) >= 0
    at = row_of_slot.view(-1).long()
    to, at = torch.where(at < 0, R, at), at.clamp(min=0)
    token = torch.arange(T * K, device="cuda") // K

    def scatter(values):  # values of every slot to their rows, zeros elsewhere
        rows = torch.zeros(R + 1, H, dtype=dt, device="cuda")
        rows[to] = values.to(dt)
        return rows[:R]

    w = s["weights"].float().view(T * K, 1)
    picked = torch.where(seen, s["expert_out"][at].float(), 0.0)
    out["rows"] = scatter(s["x"][token])
    out["y"] = (w * picked).view(T, K, H).sum(1).to(dt)
    if case["op"] == "train":
        gy = s["grad_y"].float()[token]
        out["grad_out"] = scatter(w * gy)
        out["grad_weights"] = (gy * picked).sum(1).view(T, K).to(s["weights"].dtype)
        back = torch.where(seen, s["grad_rows"][at].float(), 0.0)
        out["grad_x"] = back.view(T, K, H).sum(1).to(dt)
    return out


def _plain_add(s):
    case, weights, scores = s["case"], s["weights"], s["scores"]
    B, Hq, Q, S = weights.shape
    Hkv = scores.shape[1]
    at = torch.arange(S, device="cuda")
    end = s["lengths"].view(B, 1, 1, 1).long()
    w = weights.float()
    if case["causal"]:
        end = end - Q + 1 + torch.arange(Q, device="cuda").view(1, 1, Q, 1)
        w = torch.where(at < end, w, 0.0)
    total = w.view(B, Hkv, Hq // Hkv * Q, S).sum(2)
    live = at < s["lengths"].view(B, 1, 1)
    scores.copy_(torch.where(live, case["decay"] * scores + total, scores))
    return scores


def _plain_select(case, scores, lengths):
    B, H, S = scores.shape
    budget, sinks, recent = case["budget"], case["sinks"], case["recent"]
    at = torch.arange(S, device="cuda")
    L = lengths.view(B, 1, 1).long()
    key = torch.where(torch.isnan(scores), -math.inf, scores) + 0.0
    order = torch.argsort(key, dim=2, descending=True, stable=True)
    # what always stays first, what is not there last, the scores between
    rank = torch.where((order < sinks) | (order >= L - recent), 0, 1)
    rank = torch.where(order >= L, 2, rank)
    order = order.gather(2, torch.argsort(rank, dim=2, stable=True))[..., :budget]
    n = torch.clamp(L, max=budget)
    slots = torch.arange(budget, device="cuda")
    kept = torch.sort(torch.where(slots < n, order, S), dim=2).values
    kept = torch.where(slots < n, kept, -1)
    return kept.int(), n.view(B).int()


def _plain_cache(s):
    case = s["case"]
    kept, n = s["kept"], s["kept_lengths"]
    if case["op"] != "compact":
        kept, n = _plain_select(case, s["scores"], s["lengths"])
        if case["op"] == "select":
            return {"kept": kept, "kept_lengths": n}
    B, H, budget = kept.shape
    live = torch.arange(budget, device="cuda") < n.view(B, 1, 1)
    at = kept.long().clamp(min=0)

    def moved(src):  # rows of src by kept, in the shape of the new cache
        i = at if src.dim() == 3 else at.unsqueeze(-1).expand(-1, -1, -1, src.shape[3])
        m = live if src.dim() == 3 else live.unsqueeze(-1)
        rows = src.gather(2, i)
        if case.get("inplace"):
            part = src[:, :, :budget]
            part.copy_(torch.where(m, rows, part))
            return src
        return torch.where(m, rows, 0)

    out = {"k": moved(s["k"]), "v": moved(s["v"]), "scores": moved(s["scores"])}
    if case["op"] == "evict":
        out.update(kept=kept, kept_lengths=n)
    return out


# ---------------------------------------------------------------------------
# The same outputs from the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("sort", "forward", "train"):
        return _exact_experts(case, s)
    return _exact_add(case, s) if case["op"] == "add" else _exact_cache(case, s)


def _exact_experts(case, s):
    T, K, E, a, R = case["T"], case["K"], case["E"], case["align"], _rows(case)
    # Counting: a slot's place is the number of earlier slots of its expert.
    ids = s["ids"].cpu().numpy().reshape(-1).astype(np.int64)
    row_of_slot = np.full(T * K, -1, np.int64)
    offsets = np.zeros(E + 1, np.int64)
    counts = np.zeros(E, np.int64)
    for e in range(E):
        mine = np.flatnonzero(ids == e)
        counts[e] = mine.size
        row_of_slot[mine] = offsets[e] + np.arange(mine.size)
        offsets[e + 1] = offsets[e] + -(-mine.size // a) * a
    slot_of_row = np.full(R, -1, np.int64)
    used = np.flatnonzero(row_of_slot >= 0)
    slot_of_row[row_of_slot[used]] = used
    out = {"row_of_slot": row_of_slot.reshape(T, K), "slot_of_row": slot_of_row,
           "offsets": offsets, "counts": counts}
    if case["op"] == "sort":
        return out
    # Row by row: each row adds to its token, so nothing is gathered by slot.
    H = case["H"]
    rows = torch.from_numpy(np.flatnonzero(slot_of_row >= 0)).cuda()
    slots = torch.from_numpy(slot_of_row).cuda()[rows]
    tokens = slots // K
    w = s["weights"].double().view(-1)[slots].unsqueeze(1)

    def placed(values):
        full = torch.zeros(R, H, dtype=torch.float64, device="cuda")
        return full.index_copy_(0, rows, values)

    def added(values):
        total = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        return total.index_add_(0, tokens, values)

    out["rows"] = placed(s["x"].double()[tokens])
    out["y"] = added(s["expert_out"][rows].double() * w)
    if case["op"] == "train":
        gy = s["grad_y"].double()[tokens]
        out["grad_out"] = placed(gy * w)
        dots = torch.zeros(T * K, dtype=torch.float64, device="cuda")
        dots[slots] = torch.linalg.vecdot(gy, s["expert_out"][rows].double())
        out["grad_weights"] = dots.view(T, K)
        out["grad_x"] = added(s["grad_rows"][rows].double())
    return out


def _exact_add(case, s):
    B, Hq, Hkv, Q = (case[k] for k in ("B", "Hq", "Hkv", "Q"))
    total = s["scores"].double()
    lens = s["lengths"].tolist()
    for b in range(B):
        n = lens[b]
        total[b, :, :n] *= case["decay"]
        w = s["weights"][b, :, :, :n].double()
        if case["causal"]:
            w = torch.tril(w, diagonal=n - Q)
        total[b, :, :n] += w.sum(1).view(Hkv, Hq // Hkv, n).sum(1)
    return total


def _exact_cache(case, s):
    if case["op"] == "compact":
        kept = s["kept"].cpu().numpy().astype(np.int64)
        n = s["kept_lengths"].cpu().numpy().astype(np.int64)
    else:
        scores = s["scores"].cpu().numpy().astype(np.float64)
        lens = s["lengths"].cpu().numpy().astype(np.int64)
        B, H, _ = scores.shape
        n = np.minimum(lens, case["budget"])
        kept = np.full((B, H, case["budget"]), -1, np.int64)
        for b in range(B):
            L = int(lens[b])
            for h in range(H):
                if L <= case["budget"]:
                    kept[b, h, :L] = np.arange(L)
                    continue
                lo, hi = case["sinks"], L - case["recent"]
                part = scores[b, h, lo:hi]
                best = np.lexsort((np.arange(hi - lo), -part))
                best = best[:case["budget"] - case["sinks"] - case["recent"]] + lo
                kept[b, h] = np.sort(np.concatenate([np.arange(lo), best, np.arange(hi, L)]))
        if case["op"] == "select":
            return {"kept": kept, "kept_lengths": n}
    out = {}
    for name in ("k", "v", "scores"):
        src = s[name].double()
        old = src if case.get("inplace") else torch.zeros(
            src.shape[:2] + (case["budget"],) + src.shape[3:], dtype=torch.float64, device="cuda")
        new = old.clone()
        for b in range(case["B"]):
            at = torch.from_numpy(kept[b, :, :n[b]]).cuda()
            for h in range(case["H"]):
                new[b, h, :n[b]] = src[b, h].index_select(0, at[h])
        out[name] = new
    if case["op"] == "evict":
        out.update(kept=kept, kept_lengths=n)
    return out
