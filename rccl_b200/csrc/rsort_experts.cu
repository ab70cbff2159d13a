// Expert routing: token slots sorted by expert, rows gathered into expert
// order, expert outputs combined back with their weights, and the gradients.
//
// Slot s = token * top_k + k holds an expert id; ids outside 0..experts-1 are
// dropped.  The sort is a stable counting sort: slot s of expert e goes to row
// offsets[e] + (number of earlier slots of e), with every expert's segment
// padded to a multiple of `align` rows.  The plan stays on the device.
#include <algorithm>
#include <climits>

#include "../../include/rsort_b200.h"
#include "rsort_internal.cuh"
#include "rsort_rows.cuh"

using namespace rsort;

namespace {

// ---------------------------------------------------------------------------
// Counting sort of slots by expert
//
// Bound by latency at every size a router produces (512 Ki slots are 8.5 MB).
// A CTA takes its slots in steps of 32 a warp, SORT_STEPS of them in registers:
// a warp ranks its slots among its own by votes and keeps a counter per expert,
// a scan over the warps and one over the experts turn the counters into rows,
// and every slot adds its rank.  No atomic's order reaches a result.
//   up to SORT_MAX_CLUSTER CTAs: one launch of one cluster; its CTAs read one
//     another's counts through distributed shared memory.
//   longer: a first kernel counts the experts of every CTA's chunk, the second
//     adds up the chunks before its own.  The second comes onto the SMs early,
//     but reads no ids before it has waited itself: that the first has waited
//     for whoever wrote the ids shows them to the first alone.
// 128 slots take 4.1 us, 2 Ki 5.4, 8 Ki 5.5, 32 Ki 9.2, 512 Ki 14.5 (both launches).
// In a full CTA of 4096 slots and 256 experts a quarter of the time goes to the
// votes (33 cycles of the SM for 32 slots) and a quarter to the scattered stores
// of slot_of_row (35 cycles).
// ---------------------------------------------------------------------------
constexpr uint32_t SORT_STEPS = 4;
constexpr uint32_t SORT_MAX_WARPS = 32;
constexpr uint32_t SORT_MAX_CLUSTER = 8;
constexpr uint32_t SORT_MAX_GRID = 1024;  // scratch is sized for this many CTAs

struct SortArgs {
    const void *ids;
    uint32_t n;        // slots
    uint32_t experts;
    uint32_t align;
    uint32_t id_bits;  // of 0..experts
    uint32_t chunk;    // slots per CTA, a multiple of SORT_STEPS * its threads
    uint32_t *counts_of_block;  // [grid][pitch]; null with one cluster
    uint32_t pitch;    // experts rounded up to 4
    int32_t *row_of_slot, *slot_of_row;
    uint32_t rows;     // capacity of slot_of_row
    int32_t *offsets, *counts;
};

// The slot's bucket: its expert, or `experts` for a dropped slot.
template <typename I>
__device__ __forceinline__ uint32_t bucket(const SortArgs &a, uint64_t i) {
    const I id = static_cast<const I *>(a.ids)[i];
    return id >= 0 && id < I(a.experts) ? uint32_t(id) : a.experts;
}

// Every row starts without a slot; the placed ones are overwritten.
__device__ __forceinline__ void clear_rows(const SortArgs &a) {
    for (uint64_t r = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; r < a.rows;
         r += uint64_t(gridDim.x) * blockDim.x)
        a.slot_of_row[r] = -1;
}

template <typename I>
__global__ void __launch_bounds__(SORT_MAX_WARPS * 32) expert_count_kernel(const SortArgs a) {
    extern __shared__ uint32_t hist[];  // experts + 1
    begin_kernel();  // the placing kernel may start: the ids are there
    for (uint32_t e = threadIdx.x; e <= a.experts; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    const uint64_t first = uint64_t(blockIdx.x) * a.chunk;
    const uint64_t last = min(first + a.chunk, uint64_t(a.n));
#pragma unroll 4
    for (uint64_t i = first + threadIdx.x; i < last; i += blockDim.x)
        atomicAdd(&hist[bucket<I>(a, i)], 1u);
    clear_rows(a);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.pitch; e += blockDim.x)
        a.counts_of_block[size_t(blockIdx.x) * a.pitch + e] = e < a.experts ? hist[e] : 0;
}

// Lanes of the warp with the same bucket: one vote a bit of the id (on sm_100
// a vote issues every three cycles and __match_any_sync every sixty).
__device__ __forceinline__ uint32_t same_bucket(uint32_t e, uint32_t bits) {
    uint32_t peers = 0xffffffffu;
    for (uint32_t b = 0; b < bits; ++b) {
        const bool set = (e >> b) & 1u;
        const uint32_t v = __ballot_sync(0xffffffffu, set);
        peers &= set ? v : ~v;
    }
    return peers;
}

// Exclusive scan over one value a thread; *total gets the block's sum.
__device__ __forceinline__ uint32_t sort_scan(uint32_t v, uint32_t *warp_sums, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= uint32_t(off)) inc += y;
    }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    uint32_t sums = lane < (blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, sums, off);
        if (lane >= uint32_t(off)) sums += y;
    }
    *total = __shfl_sync(0xffffffffu, sums, 31);
    const uint32_t lower = __shfl_sync(0xffffffffu, sums, (warp - 1) & 31);
    __syncthreads();  // warp_sums may be written again
    return (warp ? lower : 0) + inc - v;
}

template <typename I>
__global__ void __launch_bounds__(SORT_MAX_WARPS * 32) expert_place_kernel(const SortArgs a) {
    extern __shared__ uint32_t shared[];
    __shared__ uint32_t warp_sums[SORT_MAX_WARPS];
    const uint32_t E = a.experts, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t warps = blockDim.x >> 5, pitch = (E + 2) & ~1u;
    uint32_t *const sub = shared;        // [E] slots of this CTA's current part
    uint32_t *const total = sub + E;     // [E] slots of the expert
    uint32_t *const first = total + E;   // [E] first row of this CTA's slots
    // [warps][pitch] slots of a warp, then of the warps before it
    uint16_t *const base = reinterpret_cast<uint16_t *>(first + E);
    uint16_t *const mine = base + warp * pitch;
    const uint64_t begin = uint64_t(blockIdx.x) * a.chunk;
    const uint64_t end = min(begin + a.chunk, uint64_t(a.n));
    const uint32_t part = SORT_STEPS * blockDim.x;  // slots taken at once

    for (uint64_t p = begin; p == begin || p < end; p += part) {
        const uint64_t slot0 = p + uint64_t(warp) * (SORT_STEPS * 32) + lane;
        uint32_t e[SORT_STEPS], rank[SORT_STEPS];
        for (uint32_t i = tid; i < warps * pitch / 2; i += blockDim.x)
            reinterpret_cast<uint32_t *>(base)[i] = 0;
        if (p == begin) {
            for (uint32_t i = tid; i < E; i += blockDim.x) total[i] = first[i] = 0;
            begin_kernel();
            if (!a.counts_of_block) clear_rows(a);
        }
#pragma unroll
        for (uint32_t k = 0; k < SORT_STEPS; ++k)
            e[k] = slot0 + 32 * k < end ? bucket<I>(a, slot0 + 32 * k) : E;
        __syncthreads();
        // Ranks among the warp's slots: lanes with the same expert in lane
        // order, step after step.
#pragma unroll
        for (uint32_t k = 0; k < SORT_STEPS; ++k) {
            const uint32_t peers = same_bucket(e[k], a.id_bits);
            const uint32_t below = __popc(peers & ((1u << lane) - 1));
            const uint32_t at = mine[e[k]];
            __syncwarp();
            if (below == 0) mine[e[k]] = uint16_t(at + __popc(peers));
            __syncwarp();
            rank[k] = at + below;
        }
        __syncthreads();
        for (uint32_t i = tid; i < E; i += blockDim.x) {
            uint32_t at = 0;
            for (uint32_t w0 = 0; w0 < warps; w0 += 8) {
                uint32_t v[8];
#pragma unroll
                for (uint32_t w = 0; w < 8; ++w)
                    v[w] = w0 + w < warps ? base[(w0 + w) * pitch + i] : 0;
#pragma unroll
                for (uint32_t w = 0; w < 8; ++w) {
                    if (w0 + w < warps) base[(w0 + w) * pitch + i] = uint16_t(at);
                    at += v[w];
                }
            }
            sub[i] = at;
        }
        if (p == begin) {
            // The experts' totals and the slots of the CTAs before this one.
            if (a.counts_of_block) {
                const uint32_t quads = a.pitch / 4, wide = (quads + 31) & ~31u;
                const uint32_t groups = max(blockDim.x / wide, 1u);
                const uint4 *const counts = reinterpret_cast<const uint4 *>(a.counts_of_block);
                for (uint32_t i = tid; i < groups * wide; i += blockDim.x) {
                    const uint32_t q = i % wide;
                    if (q >= quads) continue;
                    uint32_t before[4] = {}, all[4] = {};
#pragma unroll 8
                    for (uint32_t c = i / wide; c < gridDim.x; c += groups) {
                        const uint4 v = counts[size_t(c) * quads + q];
                        const bool b = c < blockIdx.x;
                        all[0] += v.x, all[1] += v.y, all[2] += v.z, all[3] += v.w;
                        before[0] += b ? v.x : 0, before[1] += b ? v.y : 0;
                        before[2] += b ? v.z : 0, before[3] += b ? v.w : 0;
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j) {
                        if (4 * q + j >= E) break;
                        atomicAdd(&total[4 * q + j], all[j]);
                        atomicAdd(&first[4 * q + j], before[j]);
                    }
                }
                __syncthreads();
            } else {
                cluster_sync();  // everyone's `sub`, and the cleared rows
                for (uint32_t i = tid; i < E; i += blockDim.x) {
                    uint32_t before = 0, all = 0;
#pragma unroll
                    for (uint32_t c = 0; c < SORT_MAX_CLUSTER; ++c) {
                        if (c >= gridDim.x) break;
                        const uint32_t v = cluster_read(&sub[i], c);
                        before += c < blockIdx.x ? v : 0;
                        all += v;
                    }
                    total[i] = all;
                    first[i] = before;
                }
                cluster_arrive();  // waited for at the end: `sub` stays until all have read
                __syncthreads();
            }
            // Scan of the padded segment sizes, a block of experts a step.
            uint32_t carry = 0;
            for (uint32_t e0 = 0; e0 < E; e0 += blockDim.x) {
                const uint32_t i = e0 + tid, count = i < E ? total[i] : 0;
                uint32_t sum;
                const uint32_t at =
                    carry + sort_scan((count + a.align - 1) / a.align * a.align, warp_sums, &sum);
                carry += sum;
                if (i < E) {
                    first[i] += at;
                    if (blockIdx.x == 0) {
                        a.offsets[i] = int32_t(at);
                        a.counts[i] = int32_t(count);
                    }
                }
            }
            if (blockIdx.x == 0 && tid == 0) a.offsets[E] = int32_t(carry);
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < SORT_STEPS; ++k) {
            const uint64_t i = slot0 + 32 * k;
            if (i >= end) continue;
            int32_t row = -1;
            if (e[k] < E) {
                row = int32_t(first[e[k]] + mine[e[k]] + rank[k]);
                if (uint32_t(row) < a.rows) a.slot_of_row[row] = int32_t(i);
            }
            a.row_of_slot[i] = row;
        }
        if (p + part < end) {
            __syncthreads();
            for (uint32_t i = tid; i < E; i += blockDim.x) first[i] += sub[i];
            __syncthreads();
        }
    }
    if (!a.counts_of_block) cluster_wait();
}

// Warps of a CTA: an eighth of a short input each (ranking and the scattered
// stores are bound by the SM: 8 Ki slots take 9.3 us on two CTAs of 32 warps,
// 6.0 us on eight of 8), and at most what leaves the counters 48 KB.
uint32_t sort_warps(size_t n, size_t experts) {
    const uint32_t most = experts <= 512 ? 32 : 16;
    const size_t slots = SORT_MAX_CLUSTER * SORT_STEPS * 32, want = (n + slots - 1) / slots;
    return uint32_t(want < 4 ? 4 : want < most ? want : most);
}

uint32_t sort_grid(size_t n, size_t experts, uint32_t sms) {
    const size_t part = size_t(sort_warps(n, experts)) * 32 * SORT_STEPS;
    const size_t want = (n + part - 1) / part;
    return uint32_t(want < 1 ? 1 : want < sms ? want : sms);
}

template <typename I>
cudaError_t launch_sort(SortArgs a, uint32_t grid, uint32_t warps, cudaStream_t s) {
    if (a.counts_of_block) {
        LaunchScope scope(RSORT_KERNEL_EXPERT_SORT, s);
        const cudaError_t e = launch_early(expert_count_kernel<I>, dim3(grid), SORT_MAX_WARPS * 32,
                                           (a.experts + 1) * 4, 1, s, a);
        if (e != cudaSuccess) return e;
    }
    LaunchScope scope(RSORT_KERNEL_EXPERT_SORT, s);
    return launch_early(expert_place_kernel<I>, dim3(grid), warps * 32,
                        size_t(a.experts) * 12 + size_t(warps) * ((a.experts + 2) & ~1u) * 2,
                        a.counts_of_block ? 1 : grid, s, a);
}

// ---------------------------------------------------------------------------
// Rows in and out of expert order
// ---------------------------------------------------------------------------
constexpr int ROW_BLOCK = 256;
constexpr int PAD_BLOCKS = 4;  // CTAs that zero one expert's padding rows

struct Plan {
    const int32_t *row_of_slot, *offsets, *counts;
    uint32_t tokens, top_k, experts, rows;
};

// `lanes` threads (a power of two up to ROW_BLOCK) work on one token.
struct Shape {
    uint32_t lanes, token_blocks, units;
};

Shape shape_of(size_t tokens, size_t units, size_t most_tokens = ROW_BLOCK) {
    Shape s{1, 0, uint32_t(units)};
    while (s.lanes < ROW_BLOCK && (s.lanes < units || ROW_BLOCK / s.lanes > most_tokens))
        s.lanes <<= 1;
    // Half the threads a token where a last, short step would idle many.
    while (s.lanes > 32 && (units + s.lanes - 1) / s.lanes * s.lanes - units > units / 16 &&
           2 * ROW_BLOCK / s.lanes <= most_tokens)
        s.lanes >>= 1;
    const uint32_t per = ROW_BLOCK / s.lanes;
    s.token_blocks = uint32_t((tokens + per - 1) / per);
    return s;
}

// A slot's row, or -1 when it was dropped (or the plan does not fit the rows).
__device__ __forceinline__ int32_t row_at(const Plan &p, uint64_t slot) {
    const int32_t r = p.row_of_slot[slot];
    return uint32_t(r) < p.rows ? r : -1;
}

// Zeros the padding rows of one expert (block b of the padding blocks).
template <typename U>
__device__ __forceinline__ void zero_padding(const Plan &p, uint32_t b, char *rows, size_t stride,
                                             uint32_t units) {
    const uint32_t e = b / PAD_BLOCKS;
    const uint32_t lo = uint32_t(p.offsets[e]) + uint32_t(p.counts[e]);
    const uint32_t hi = min(uint32_t(p.offsets[e + 1]), p.rows);
    for (uint32_t r = lo + b % PAD_BLOCKS; r < hi; r += PAD_BLOCKS) {
        U *row = reinterpret_cast<U *>(rows + size_t(r) * stride);
        for (uint32_t u = threadIdx.x; u < units; u += ROW_BLOCK) row[u] = U{};
    }
}

// rows[row of slot] = x[t]: a token is read once and written to all of its rows,
// so the kernel is bound by the writes (calls in a row: 16 Ki tokens to 8 rows of
// 4096 bf16 and the padding of 128 experts, 1.28 GB, 211 us, 6.0 TB/s; 8191 tokens
// to 6 rows of 2048, 241 MB, 40 us, 6.0 TB/s).
template <typename U>
__global__ void __launch_bounds__(ROW_BLOCK)
    expert_gather_kernel(const Plan p, const Shape s, const char *x, size_t x_stride, char *rows,
                         size_t rows_stride) {
    begin_kernel();
    if (blockIdx.x >= s.token_blocks) {
        zero_padding<U>(p, blockIdx.x - s.token_blocks, rows, rows_stride, s.units);
        return;
    }
    const uint32_t t = blockIdx.x * (ROW_BLOCK / s.lanes) + threadIdx.x / s.lanes;
    if (t >= p.tokens) return;
    const U *src = reinterpret_cast<const U *>(x + size_t(t) * x_stride);
    for (uint32_t u = threadIdx.x % s.lanes; u < s.units; u += s.lanes) {
        const U v = src[u];
        for (uint32_t k = 0; k < p.top_k; ++k) {
            const int32_t r = row_at(p, uint64_t(t) * p.top_k + k);
            if (r >= 0) reinterpret_cast<U *>(rows + size_t(r) * rows_stride)[u] = v;
        }
    }
}

struct Weights {
    const void *w;  // null: every weight is 1
    int type;       // rsort_key_t
};

__device__ __forceinline__ float weight_at(const Weights &w, uint64_t slot) {
    if (!w.w) return 1.0f;
    if (w.type == RSORT_F32) return static_cast<const float *>(w.w)[slot];
    if (w.type == RSORT_F16) return __half2float(static_cast<const __half *>(w.w)[slot]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(w.w)[slot]);
}

__device__ __forceinline__ void store_weight(void *w, int type, uint64_t slot, float v) {
    if (type == RSORT_F32) static_cast<float *>(w)[slot] = v;
    else if (type == RSORT_F16) static_cast<__half *>(w)[slot] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(w)[slot] = __float2bfloat16_rn(v);
}

// Combine and its gradient are bound by reading the rows.  All of a token's
// rows (up to MOST_SLOTS at a time) are read by a thread before it uses the
// first, 16 bytes of each, with no branch between the reads; a CTA stays for
// many tokens, and the next one's slots (rows and weights) come into shared
// memory while it works on this one.
constexpr uint32_t SLOTS_HELD = 1024;  // of a block's tokens
constexpr int MOST_SLOTS = 8;

// Accesses of a row that a thread takes at a time: several where few slots or
// short accesses leave few bytes in flight, as sums of at most eight elements
// (1023 tokens of 2 rows of 1001 f32, 4 bytes an access: combine 4.6 us, 8.0 with
// one at a time; its gradient 6.4 and 9.3 us).
__host__ __device__ constexpr int columns_of(int elements, int slots) {
    int c = 1;
    while (2 * c * slots <= MOST_SLOTS && 2 * c * elements <= 8) c *= 2;
    return c;
}

// CTAs an SM: what the registers of `slots` reads in flight leave room for.  As
// chosen, one instance spills (4 bytes: combine, four f32 packs); with one CTA more,
// 17 do (4 to 188 bytes).  Calls in a row, one CTA fewer / as chosen / one more:
//   16 Ki tokens of 8 rows of 4096 bf16: combine (1.21 GB) 178 / 178 / 184 us
//     (6.8 TB/s), its gradient (2.35 GB) 668 / 418 / 422 us (5.6 TB/s);
//   8191 of 6 rows of 2048 bf16: 47 / 42 / 43 us, 114 / 94 / 92 us;
//   4 Ki of 4 rows of 5120 f16: 38 / 35 / 40 us, 68 / 71 / 76 us.
// Combine took 237 us instead with a branch a row and 196 us with four rows at a
// time.  Rings of asynchronous copies in shared memory were no faster (194 and
// 466 us): they pay for the reads twice in shared memory.
constexpr int combine_ctas(int slots) { return slots <= 4 ? 5 : 4; }
constexpr int backward_ctas(int elements, int slots) {
    return columns_of(elements, slots) > 1 ? 3 : slots <= 4 ? 4 : slots <= 6 ? 3 : 2;
}

// For the CTA's tokens, block by block: work(t, rows, weights, buffer) with the
// token's slots [k0, k0 + count), filled up to a multiple of SLOTS (row -1 and
// weight 0 for what has no row), then, behind a barrier, done(t, buffer).  All
// threads take part, also for tokens behind the last (t >= tokens).
template <int SLOTS, typename Work, typename Done>
__device__ __forceinline__ void each_token(const Plan &p, const Shape &s, const Weights &w,
                                           uint32_t k0, uint32_t count, uint32_t first,
                                           uint32_t stride, Work work, Done done) {
    __shared__ int32_t held_rows[2][SLOTS_HELD];
    __shared__ float held_weights[2][SLOTS_HELD];
    const uint32_t per = ROW_BLOCK / s.lanes, group = threadIdx.x / s.lanes;
    const uint32_t lane = threadIdx.x % s.lanes, filled = (count + SLOTS - 1) / SLOTS * SLOTS;
    const uint32_t at = group * filled;
    auto row_of = [&](uint32_t t, uint32_t k) {
        return t < p.tokens && k < count ? row_at(p, uint64_t(t) * p.top_k + k0 + k) : -1;
    };
    auto weight_of = [&](uint32_t t, uint32_t k, int32_t row) {
        return row >= 0 ? weight_at(w, uint64_t(t) * p.top_k + k0 + k) : 0.0f;
    };
    auto hold = [&](uint32_t buffer, uint32_t t, uint32_t from) {
        for (uint32_t k = from; k < filled; k += s.lanes) {
            const int32_t row = row_of(t, k);
            held_rows[buffer][at + k] = row;
            held_weights[buffer][at + k] = weight_of(t, k, row);
        }
    };
    const uint32_t step = stride * per;
    uint32_t t = first * per + group;
    hold(0, t, lane);
    __syncthreads();
    uint32_t now = 0;
    for (uint32_t b = first; b < s.token_blocks; b += stride, t += step, now ^= 1) {
        int32_t row = -1;
        float weight = 0;
        const bool ahead = b + stride < s.token_blocks && lane < filled;
        if (ahead) {
            row = row_of(t + step, lane);
            weight = weight_of(t + step, lane, row);
        }
        work(t, &held_rows[now][at], &held_weights[now][at], now);
        if (ahead) {
            held_rows[now ^ 1][at + lane] = row;
            held_weights[now ^ 1][at + lane] = weight;
            hold(now ^ 1, t + step, lane + s.lanes);
        }
        __syncthreads();
        done(t, now);
    }
}

// The access u of a row.  A slot without a row reads row 0, whose values
// are dropped (kept_row): no branch parts the reads.
template <typename P, typename T>
__device__ __forceinline__ P read_row(const T *rows, size_t stride, int32_t row, uint32_t u) {
    return reinterpret_cast<const P *>(rows + size_t(max(row, 0)) * stride)[u];
}
template <typename P> __device__ __forceinline__ P kept_row(const P &v, int32_t row) {
    P o = v;
    if constexpr (sizeof(P) >= 4) {
        uint32_t *w = reinterpret_cast<uint32_t *>(&o);
#pragma unroll
        for (int i = 0; i < int(sizeof(P) / 4); ++i) w[i] = row < 0 ? 0u : w[i];
    } else if (row < 0) {
        o = P{};
    }
    return o;
}

// out[t] = sum over k of weight * rows[row of slot], summed in fp32 in the
// order of k and rounded once.
template <typename T, int V, int SLOTS>
__global__ void __launch_bounds__(ROW_BLOCK, combine_ctas(SLOTS))
    expert_combine_kernel(const Plan p, const Shape s, const T *rows, size_t rows_stride,
                          const Weights w, T *out, size_t out_stride) {
    using P = Pack<T, V>;
    constexpr int COLUMNS = columns_of(V, SLOTS);
    begin_kernel();
    each_token<SLOTS>(p, s, w, 0, p.top_k, blockIdx.x, gridDim.x,
               [&](uint32_t t, const int32_t *row, const float *weight, uint32_t) {
        if (t >= p.tokens) return;
        P *const dst = reinterpret_cast<P *>(out + size_t(t) * out_stride);
        const uint32_t wide = gridDim.y * s.lanes;
        for (uint32_t u0 = blockIdx.y * s.lanes + threadIdx.x % s.lanes; u0 < s.units;
             u0 += wide * COLUMNS) {
            float acc[COLUMNS][V] = {};
            for (uint32_t k0 = 0; k0 < (p.rows ? p.top_k : 0); k0 += SLOTS) {
                P v[COLUMNS][SLOTS];
#pragma unroll
                for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
                    for (int k = 0; k < SLOTS; ++k)
                        v[c][k] = read_row<P>(rows, rows_stride, row[k0 + k],
                                              min(u0 + c * wide, s.units - 1));
#pragma unroll
                for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
                    for (int k = 0; k < SLOTS; ++k) {
                        const P kept = kept_row(v[c][k], row[k0 + k]);
                        const float f = weight[k0 + k];
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            acc[c][i] = fmaf(f, to_float(kept.v[i]), acc[c][i]);
                    }
            }
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) {
                if (u0 + c * wide >= s.units) break;
                P o;
#pragma unroll
                for (int i = 0; i < V; ++i) o.v[i] = from_float<T>(acc[c][i]);
                dst[u0 + c * wide] = o;
            }
        }
    }, [](uint32_t, uint32_t) {});
}

// grad_rows[row of slot] = weight * grad_out[t], grad_w[slot] = the dot
// product of grad_out[t] and rows[row of slot] in fp32: one pass over the rows
// serves both.  A launch takes `count` (at most SLOTS) slots of every token
// from k0 on.
template <typename T, int V, int SLOTS>
__global__ void __launch_bounds__(ROW_BLOCK, backward_ctas(V, SLOTS))
    expert_combine_backward_kernel(const Plan p, const Shape s, uint32_t k0, uint32_t count,
                                   const T *grad_out, size_t grad_out_stride, const T *rows,
                                   size_t rows_stride, const Weights w, T *grad_rows,
                                   size_t grad_rows_stride, void *grad_w, uint32_t token_ctas) {
    using P = Pack<T, V>;
    begin_kernel();
    if (blockIdx.x >= token_ctas) {
        zero_padding<P>(p, blockIdx.x - token_ctas, reinterpret_cast<char *>(grad_rows),
                        grad_rows_stride * sizeof(T), s.units);
        return;
    }
    // The warps' sums of a token's dot products; a token of fewer threads than
    // a warp has its sums without them.
    __shared__ float sums[2][ROW_BLOCK / 32][SLOTS];
    constexpr int COLUMNS = columns_of(V, SLOTS);
    const uint32_t lane = threadIdx.x % s.lanes, width = min(s.lanes, 32u);
    each_token<SLOTS>(p, s, w, k0, count, blockIdx.x, token_ctas,
               [&](uint32_t t, const int32_t *row, const float *weight, uint32_t buffer) {
        const bool live = t < p.tokens;
        const P *const g =
            reinterpret_cast<const P *>(grad_out + size_t(live ? t : 0) * grad_out_stride);
        float dot[SLOTS] = {};
        for (uint32_t u0 = lane; live && p.rows && u0 < s.units; u0 += s.lanes * COLUMNS) {
            P gv[COLUMNS], v[COLUMNS][SLOTS];
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) gv[c] = g[min(u0 + c * s.lanes, s.units - 1)];
            if (grad_w) {
#pragma unroll
                for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
                    for (int k = 0; k < SLOTS; ++k)
                        v[c][k] = read_row<P>(rows, rows_stride, row[k],
                                              min(u0 + c * s.lanes, s.units - 1));
            }
#pragma unroll
            for (int c = 0; c < COLUMNS; ++c) {
                const uint32_t u = u0 + c * s.lanes;
                if (u >= s.units) break;
#pragma unroll
                for (int k = 0; grad_rows && k < SLOTS; ++k) {
                    const int32_t r = row[k];
                    const float f = weight[k];
                    P o;
#pragma unroll
                    for (int i = 0; i < V; ++i) o.v[i] = from_float<T>(f * to_float(gv[c].v[i]));
                    if (r >= 0)
                        reinterpret_cast<P *>(grad_rows + size_t(r) * grad_rows_stride)[u] = o;
                }
#pragma unroll
                for (int k = 0; grad_w && k < SLOTS; ++k) {
                    const P kept = kept_row(v[c][k], row[k]);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        dot[k] = fmaf(to_float(gv[c].v[i]), to_float(kept.v[i]), dot[k]);
                }
            }
        }
        if (!grad_w) return;
        // A dropped slot has 0, also where grad_out is not finite.
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) dot[k] = row[k] < 0 ? 0.0f : dot[k];
#pragma unroll
        for (int k = 0; k < SLOTS; ++k)
            for (uint32_t o = width / 2; o > 0; o >>= 1)
                dot[k] += __shfl_down_sync(0xffffffffu, dot[k], o, width);
        if (s.lanes <= 32) {
            if (live && lane == 0)
#pragma unroll
                for (int k = 0; k < SLOTS; ++k)
                    if (uint32_t(k) < count)
                        store_weight(grad_w, w.type, uint64_t(t) * p.top_k + k0 + k, dot[k]);
        } else if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int k = 0; k < SLOTS; ++k) sums[buffer][threadIdx.x >> 5][k] = dot[k];
        }
    }, [&](uint32_t t, uint32_t buffer) {
        if (!grad_w || s.lanes <= 32 || t >= p.tokens || lane >= count) return;
        float total = 0;
        const uint32_t w0 = threadIdx.x / s.lanes * (s.lanes / 32);
        for (uint32_t i = 0; i < s.lanes / 32; ++i) total += sums[buffer][w0 + i][lane];
        store_weight(grad_w, w.type, uint64_t(t) * p.top_k + k0 + lane, total);
    });
}

// Calls f with the reads that a thread has in flight: all of a token's slots,
// up to MOST_SLOTS.  (With eight reads for six slots 8191 tokens of 2048 bf16 take
// 44 us instead of 42, and the gradient, at one CTA an SM less, 129 instead of 94.)
template <typename F> cudaError_t with_slots(uint32_t slots, F f) {
    if (slots <= 1) return f(std::integral_constant<int, 1>{});
    if (slots <= 2) return f(std::integral_constant<int, 2>{});
    if (slots <= 4) return f(std::integral_constant<int, 4>{});
    if (slots <= 6) return f(std::integral_constant<int, 6>{});
    return f(std::integral_constant<int, MOST_SLOTS>{});
}

uint32_t resident(const Shape &shape, int sms, int ctas) {
    const uint32_t most = uint32_t(sms) * uint32_t(ctas);
    return shape.token_blocks < most ? shape.token_blocks : most;
}

// ---------------------------------------------------------------------------
// Argument checks
// ---------------------------------------------------------------------------
size_t rows_bound(size_t nslots, size_t experts, size_t align) {
    const size_t used = experts < nslots ? experts : nslots;
    return (nslots + used * (align - 1)) / align * align;
}

bool sort_shape_ok(size_t nslots, size_t experts, size_t align) {
    return experts >= 1 && experts <= RSORT_MAX_EXPERTS && align >= 1 &&
           align <= RSORT_MAX_EXPERT_ALIGN && nslots <= size_t(INT_MAX) &&
           rows_bound(nslots, experts, align) <= size_t(INT_MAX);
}

rsort_status check_plan(const rsort_expert_plan *p, Plan *out) {
    if (!p) return fail(RSORT_BAD_ARGUMENT, "null expert plan");
    if (p->experts < 1 || p->experts > RSORT_MAX_EXPERTS)
        return fail(RSORT_BAD_ARGUMENT, "expert count", RSORT_MAX_EXPERTS, p->experts);
    if (p->top_k < 1 || p->top_k > RSORT_MAX_EXPERTS)
        return fail(RSORT_BAD_ARGUMENT, "expert plan top_k", RSORT_MAX_EXPERTS, p->top_k);
    if (p->tokens > size_t(INT_MAX) / p->top_k || p->nrows > size_t(INT_MAX))
        return fail(RSORT_SIZE_OVERFLOW, "expert plan (32-bit slots and rows)");
    if (!p->offsets || !p->counts || (p->tokens && !p->row_of_slot))
        return fail(RSORT_BAD_ARGUMENT, "null expert plan array");
    if (check_alignment(addr(p->offsets) | addr(p->counts) | addr(p->row_of_slot), 4,
                        "expert plan alignment") != RSORT_OK)
        return RSORT_BAD_ARGUMENT;
    *out = Plan{p->row_of_slot, p->offsets, p->counts, uint32_t(p->tokens), uint32_t(p->top_k),
                uint32_t(p->experts), uint32_t(p->nrows)};
    return RSORT_OK;
}

// CTAs read the plan while others write.
bool apart_from_plan(const Plan &p, const Strided &out) {
    return apart(out, packed(p.row_of_slot, size_t(p.tokens) * p.top_k * 4)) &&
           apart(out, packed(p.offsets, (size_t(p.experts) + 1) * 4)) &&
           apart(out, packed(p.counts, size_t(p.experts) * 4));
}

}  // namespace

extern "C" {

size_t rsort_expert_rows(size_t nslots, size_t experts, size_t align) {
    return sort_shape_ok(nslots, experts, align) ? rows_bound(nslots, experts, align) : 0;
}

size_t rsort_expert_sort_scratch_bytes(size_t nslots, size_t experts) {
    if (experts < 1 || experts > RSORT_MAX_EXPERTS || nslots > size_t(INT_MAX)) return 0;
    return sort_grid(nslots, experts, SORT_MAX_GRID) * ((experts + 3) & ~size_t(3)) * 4;
}

rsort_status rsort_expert_sort(rsort_key_t id_type, const void *d_ids, size_t nslots,
                               size_t experts, size_t align, int32_t *d_row_of_slot,
                               int32_t *d_slot_of_row, size_t nrows, int32_t *d_offsets,
                               int32_t *d_counts, void *d_scratch, size_t scratch_bytes,
                               rsort_stream_t stream) {
    if (id_type != RSORT_I32 && id_type != RSORT_I64)
        return fail(RSORT_BAD_ARGUMENT, "expert id type (i32 or i64)");
    if (experts < 1 || experts > RSORT_MAX_EXPERTS)
        return fail(RSORT_BAD_ARGUMENT, "expert count", RSORT_MAX_EXPERTS, experts);
    if (align < 1 || align > RSORT_MAX_EXPERT_ALIGN)
        return fail(RSORT_BAD_ARGUMENT, "expert alignment", RSORT_MAX_EXPERT_ALIGN, align);
    if (!sort_shape_ok(nslots, experts, align) || nrows > size_t(INT_MAX))
        return fail(RSORT_SIZE_OVERFLOW, "expert rows (32-bit slots and rows)");
    const size_t need = rows_bound(nslots, experts, align);
    if (nrows < need) return fail(RSORT_WORKSPACE_TOO_SMALL, "expert rows", need, nrows);
    if ((nslots && (!d_ids || !d_row_of_slot)) || (nrows && !d_slot_of_row) || !d_offsets ||
        !d_counts)
        return fail(RSORT_BAD_ARGUMENT, "null buffer");
    const size_t bytes = rsort_expert_sort_scratch_bytes(nslots, experts);
    if (!d_scratch || scratch_bytes < bytes)
        return fail(RSORT_WORKSPACE_TOO_SMALL, "expert sort scratch", bytes, scratch_bytes);
    rsort_status st = check_alignment(addr(d_ids), id_type == RSORT_I64 ? 8 : 4,
                                      "expert ids alignment");
    if (st == RSORT_OK)
        st = check_alignment(addr(d_row_of_slot) | addr(d_slot_of_row) | addr(d_offsets) |
                                 addr(d_counts),
                             4, "expert plan alignment");
    if (st == RSORT_OK) st = check_alignment(addr(d_scratch), 16, "expert sort scratch alignment");
    if (st != RSORT_OK) return st;
    const size_t id_bytes = id_type == RSORT_I64 ? 8 : 4;
    const Strided ids = packed(d_ids, nslots * id_bytes);
    const Strided written[] = {packed(d_row_of_slot, nslots * 4), packed(d_slot_of_row, nrows * 4),
                               packed(d_offsets, (experts + 1) * 4), packed(d_counts, experts * 4),
                               packed(d_scratch, bytes)};
    for (const Strided &w : written) {
        if (!apart(ids, w)) return fail(RSORT_BAD_ARGUMENT, "expert plan overlaps the ids");
        for (const Strided &v : written)
            if (&v != &w && !apart(v, w))
                return fail(RSORT_BAD_ARGUMENT, "expert plan arrays overlap");
    }
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);

    uint32_t grid =
        sort_grid(nslots, experts, uint32_t(sms) < SORT_MAX_GRID ? sms : SORT_MAX_GRID);
    if (grid <= SORT_MAX_CLUSTER)  // clusters of 1, 2, 4 or 8
        while (grid & (grid - 1)) ++grid;
    const uint32_t warps = sort_warps(nslots, experts);
    const size_t part = size_t(warps) * 32 * SORT_STEPS;
    SortArgs a{};
    a.ids = d_ids;
    a.n = uint32_t(nslots);
    a.experts = uint32_t(experts);
    a.align = uint32_t(align);
    while (experts >> a.id_bits) ++a.id_bits;
    a.chunk = uint32_t(((nslots + grid - 1) / grid + part - 1) / part * part);
    a.counts_of_block = grid > SORT_MAX_CLUSTER ? static_cast<uint32_t *>(d_scratch) : nullptr;
    a.pitch = uint32_t((experts + 3) & ~size_t(3));
    a.row_of_slot = d_row_of_slot;
    a.slot_of_row = d_slot_of_row;
    a.rows = uint32_t(nrows);
    a.offsets = d_offsets;
    a.counts = d_counts;
    const cudaError_t e = id_type == RSORT_I32 ? launch_sort<int32_t>(a, grid, warps, s)
                                               : launch_sort<int64_t>(a, grid, warps, s);
    return launched(e, "expert sort launch");
}

rsort_status rsort_expert_gather(const rsort_expert_plan *plan, const void *d_x, size_t x_stride,
                                 void *d_rows, size_t rows_stride, size_t row_bytes,
                                 int zero_padding_rows, rsort_stream_t stream) {
    Plan p{};
    rsort_status st = check_plan(plan, &p);
    if (st != RSORT_OK) return st;
    if (row_bytes > size_t(INT_MAX)) return fail(RSORT_SIZE_OVERFLOW, "expert row bytes");
    if (row_bytes == 0 || p.rows == 0) return RSORT_OK;
    if ((p.tokens && !d_x) || !d_rows) return fail(RSORT_BAD_ARGUMENT, "null buffer");
    if (p.rows > 1 && rows_stride < row_bytes)
        return fail(RSORT_BAD_ARGUMENT, "expert rows stride", row_bytes, rows_stride);
    Strided x, rows;
    if (!strided(d_x, row_bytes, {{p.tokens, x_stride}}, &x) ||
        !strided(d_rows, row_bytes, {{p.rows, rows_stride}}, &rows))
        return fail(RSORT_SIZE_OVERFLOW, "expert rows");
    if (!apart(x, rows))
        return fail(RSORT_BAD_ARGUMENT, "expert rows overlap the tokens");
    if (!apart_from_plan(p, rows)) return fail(RSORT_BAD_ARGUMENT, "expert rows overlap the plan");
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const size_t access =
        access_bytes(addr(d_x) | addr(d_rows) | x_stride | rows_stride | row_bytes, 16);
    const Shape shape = shape_of(p.tokens, row_bytes / access);
    const uint32_t grid = shape.token_blocks + (zero_padding_rows ? p.experts * PAD_BLOCKS : 0);
    if (grid == 0) return RSORT_OK;
    auto go = [&](auto unit) {
        return launch_early(expert_gather_kernel<decltype(unit)>, dim3(grid), ROW_BLOCK, 0, 1, s,
                            p, shape, static_cast<const char *>(d_x), x_stride,
                            static_cast<char *>(d_rows), rows_stride);
    };
    LaunchScope scope(RSORT_KERNEL_EXPERT_ROWS, s);
    return launched(access == 16  ? go(uint4{})
                    : access == 8 ? go(uint2{})
                    : access == 4 ? go(uint32_t{})
                    : access == 2 ? go(uint16_t{})
                                  : go(uint8_t{}),
                    "expert gather launch");
}

rsort_status rsort_expert_combine(const rsort_expert_plan *plan, rsort_key_t type,
                                  const void *d_rows, size_t rows_stride, const void *d_weights,
                                  rsort_key_t weight_type, void *d_out, size_t out_stride,
                                  size_t width, rsort_stream_t stream) {
    Plan p{};
    rsort_status st = check_plan(plan, &p);
    if (st != RSORT_OK) return st;
    const size_t eb = real_bytes(type);
    if (!eb) return fail(RSORT_BAD_ARGUMENT, "expert row type (f32, f16 or bf16)");
    if (d_weights && !real_bytes(weight_type))
        return fail(RSORT_BAD_ARGUMENT, "expert weight type (f32, f16 or bf16)");
    if (width > size_t(INT_MAX)) return fail(RSORT_SIZE_OVERFLOW, "expert row width");
    if (width == 0 || p.tokens == 0) return RSORT_OK;
    if ((p.rows && !d_rows) || !d_out) return fail(RSORT_BAD_ARGUMENT, "null buffer");
    if (p.tokens > 1 && out_stride < width)
        return fail(RSORT_BAD_ARGUMENT, "expert output stride", width, out_stride);
    constexpr size_t most = size_t(1) << 53;
    Strided rows, out;
    if (rows_stride > most || out_stride > most ||
        !strided(d_rows, width * eb, {{p.rows, rows_stride * eb}}, &rows) ||
        !strided(d_out, width * eb, {{p.tokens, out_stride * eb}}, &out))
        return fail(RSORT_SIZE_OVERFLOW, "expert rows");
    st = check_alignment(addr(d_rows) | addr(d_out), eb, "expert rows alignment");
    if (st == RSORT_OK && d_weights)
        st = check_alignment(addr(d_weights), real_bytes(weight_type), "expert weights alignment");
    if (st != RSORT_OK) return st;
    if (!apart(rows, out)) return fail(RSORT_BAD_ARGUMENT, "expert output overlaps the rows");
    const size_t weight_bytes = size_t(p.tokens) * p.top_k * real_bytes(weight_type);
    if (d_weights && !apart(packed(d_weights, weight_bytes), out))
        return fail(RSORT_BAD_ARGUMENT, "expert output overlaps the weights");
    if (!apart_from_plan(p, out))
        return fail(RSORT_BAD_ARGUMENT, "expert output overlaps the plan");
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const size_t access = access_bytes(
        addr(d_rows) | addr(d_out) | rows_stride * eb | out_stride * eb | width * eb, 16);
    const Weights w{d_weights, int(weight_type)};
    LaunchScope scope(RSORT_KERNEL_EXPERT_ROWS, s);
    return launched(with_type(type, access,
                              [&](auto t, auto v) {
                                  using T = decltype(t);
                                  constexpr int V = decltype(v)::value;
                                  const Shape shape =
                                      shape_of(p.tokens, width / V, SLOTS_HELD / ((p.top_k + 7) & ~7u));
                                  // Few tokens: their units on more CTAs.
                                  uint32_t side = 1;
                                  while (side * shape.lanes < shape.units &&
                                         shape.token_blocks * side < uint32_t(sms))
                                      ++side;
                                  return with_slots(p.top_k, [&](auto slots) {
                                      constexpr int S = decltype(slots)::value;
                                      const dim3 grid(resident(shape, sms, combine_ctas(S)), side);
                                      return launch_early(
                                          expert_combine_kernel<T, V, S>, grid, ROW_BLOCK, 0, 1, s,
                                          p, shape, static_cast<const T *>(d_rows), rows_stride, w,
                                          static_cast<T *>(d_out), out_stride);
                                  });
                              }),
                    "expert combine launch");
}

rsort_status rsort_expert_combine_backward(const rsort_expert_plan *plan, rsort_key_t type,
                                           const void *d_grad_out, size_t grad_out_stride,
                                           const void *d_rows, size_t rows_stride,
                                           const void *d_weights, rsort_key_t weight_type,
                                           void *d_grad_rows, size_t grad_rows_stride,
                                           void *d_grad_weights, size_t width,
                                           int zero_padding_rows, rsort_stream_t stream) {
    Plan p{};
    rsort_status st = check_plan(plan, &p);
    if (st != RSORT_OK) return st;
    const size_t eb = real_bytes(type);
    if (!eb) return fail(RSORT_BAD_ARGUMENT, "expert row type (f32, f16 or bf16)");
    const size_t wb = real_bytes(weight_type);
    if (!wb) return fail(RSORT_BAD_ARGUMENT, "expert weight type (f32, f16 or bf16)");
    if (width > size_t(INT_MAX)) return fail(RSORT_SIZE_OVERFLOW, "expert row width");
    if (!d_grad_rows && !d_grad_weights)
        return fail(RSORT_BAD_ARGUMENT, "expert combine gradient without an output");
    if (p.tokens && width && (!d_grad_out || (d_grad_weights && p.rows && !d_rows)))
        return fail(RSORT_BAD_ARGUMENT, "null buffer");
    if (d_grad_rows && p.rows > 1 && grad_rows_stride < width)
        return fail(RSORT_BAD_ARGUMENT, "expert gradient rows stride", width, grad_rows_stride);
    constexpr size_t most = size_t(1) << 53;
    Strided grad_out, rows, grad_rows;
    if (rows_stride > most || grad_out_stride > most || grad_rows_stride > most ||
        !strided(d_rows, width * eb, {{d_rows ? p.rows : 0, rows_stride * eb}}, &rows) ||
        !strided(d_grad_rows, width * eb, {{d_grad_rows ? p.rows : 0, grad_rows_stride * eb}},
                 &grad_rows) ||
        !strided(d_grad_out, width * eb, {{p.tokens, grad_out_stride * eb}}, &grad_out))
        return fail(RSORT_SIZE_OVERFLOW, "expert rows");
    st = check_alignment(addr(d_grad_out) | addr(d_rows) | addr(d_grad_rows), eb,
                         "expert rows alignment");
    if (st == RSORT_OK)
        st = check_alignment(addr(d_weights) | addr(d_grad_weights), wb,
                             "expert weights alignment");
    if (st != RSORT_OK) return st;
    // Without weight gradients the rows are not read.
    const size_t weight_bytes = size_t(p.tokens) * p.top_k * wb;
    const Strided weights = packed(d_weights, d_weights ? weight_bytes : 0);
    if (!apart(grad_rows, grad_out) || !apart(grad_rows, weights) ||
        (d_grad_weights && !apart(grad_rows, rows)) || !apart_from_plan(p, grad_rows))
        return fail(RSORT_BAD_ARGUMENT, "expert gradient rows overlap an input");
    if (d_grad_weights) {
        const Strided out = packed(d_grad_weights, weight_bytes);
        if (!apart(out, grad_out) || !apart(out, rows) || !apart(out, grad_rows) ||
            !apart(out, weights) || !apart_from_plan(p, out))
            return fail(RSORT_BAD_ARGUMENT, "expert weight gradients overlap another buffer");
    }
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    size_t bits = addr(d_grad_out) | grad_out_stride * eb | width * eb;
    if (d_grad_weights) bits |= addr(d_rows) | rows_stride * eb;
    if (d_grad_rows) bits |= addr(d_grad_rows) | grad_rows_stride * eb;
    const size_t access = access_bytes(bits, 16);
    const Weights w{d_weights, int(weight_type)};
    const auto go = [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        cudaError_t e = cudaSuccess;
        for (uint32_t k0 = 0; k0 < p.top_k && e == cudaSuccess; k0 += MOST_SLOTS) {
            const uint32_t count = std::min(p.top_k - k0, uint32_t(MOST_SLOTS));
            const Shape shape = shape_of(p.tokens, width / V, SLOTS_HELD / MOST_SLOTS);
            const uint32_t pad_blocks =
                k0 == 0 && zero_padding_rows && d_grad_rows ? p.experts * PAD_BLOCKS : 0;
            e = with_slots(count, [&](auto slots) {
                constexpr int S = decltype(slots)::value;
                const uint32_t token_ctas = resident(shape, sms, backward_ctas(V, S));
                if (token_ctas + pad_blocks == 0) return cudaSuccess;
                LaunchScope scope(RSORT_KERNEL_EXPERT_ROWS, s);
                return launch_early(
                    expert_combine_backward_kernel<T, V, S>, dim3(token_ctas + pad_blocks),
                    ROW_BLOCK, 0, 1, s, p, shape, k0, count, static_cast<const T *>(d_grad_out),
                    grad_out_stride, static_cast<const T *>(d_rows), rows_stride, w,
                    static_cast<T *>(d_grad_rows), grad_rows_stride, d_grad_weights, token_ctas);
            });
        }
        return e;
    };
    return launched(with_type(type, access, go), "expert combine gradient launch");
}

}  // extern "C"
