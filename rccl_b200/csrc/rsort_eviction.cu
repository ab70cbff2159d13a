// Cache eviction by accumulated attention weight: totals of the attention
// weights per cached position, the heaviest positions of every head, and the
// cache's rows moved together.
//
// A cache holds `capacity` positions for each of batch x heads rows; the first
// lengths[b] of them are in use.
#include <algorithm>
#include <climits>

#include "../../include/rsort_b200.h"
#include "rsort_device.cuh"
#include "rsort_internal.cuh"
#include "rsort_rows.cuh"

using namespace rsort;

namespace {

__device__ __forceinline__ uint32_t length_of(const int32_t *lengths, uint32_t b,
                                              uint32_t capacity) {
    if (!lengths) return capacity;
    const int32_t n = lengths[b];
    return n < 0 ? 0u : min(uint32_t(n), capacity);
}

// ---------------------------------------------------------------------------
// Totals of attention weights
//
// Bound by reading the weights once.  A thread sums V neighbouring positions
// (16 bytes where the rows allow it) down rows = queries x heads of the group.
// One query's few rows are summed by one thread; more rows are dealt out to
// the warps of a CTA and, where the positions alone do not fill the GPU, to the
// CTAs of a cluster, whose sums meet in (distributed) shared memory in a fixed
// order.  Two loads a thread in flight (four where rows are dealt out) at four
// CTAs an SM were best: one query of 64 x 32 heads over 32 Ki positions, bf16
// (201 MB), 33 us with 2, 38 with 4, 42 with 8 (36 us a call in a row, 5.5 TB/s);
// 256 queries of 2 x 32 heads over 16 Ki, causal (490 MB), 80 us with four CTAs an
// SM's worth of work dealt out, 88 and 94 us with 8 and 16 (83 us a call in a row,
// 5.9 TB/s).  At four CTAs an SM the dealt-out form spills 64 to 72 bytes a thread
// in 16-byte packs of two-byte elements.  Tiles that some queries see only in part
// are masked behind the reads: with a branch before each read their CTAs ran twice
// as long as the others (110 us).  Rows that 16 bytes do not divide leave fewer
// bytes in flight: 32 x 32 heads of one query take 7.7 us a call over 8192
// positions, 7.8 over 8188, 13 over 8190 and 17 over 8191.
// ---------------------------------------------------------------------------
constexpr uint32_t ADD_WARPS = 8;
constexpr uint32_t ADD_BLOCK = ADD_WARPS * 32;
constexpr uint32_t ADD_FEW_ROWS = 16;     // summed by one thread
constexpr uint32_t ADD_MAX_CLUSTER = 8;

struct AddArgs {
    const void *weights;
    size_t stride_b, stride_h, stride_q;  // elements
    float *scores;
    size_t score_b, score_h;
    const int32_t *lengths;
    uint32_t heads, group, queries, capacity, cluster;
    float decay;
    uint32_t causal, score_packs;  // score_packs: rows of totals start on 16 bytes
};

// Adds rows first, first + step, ... of the group's heads x queries q0.. to acc.
// SEEN_ALL: every query sees all V positions.  Else query q sees the positions
// below end0 + see_more * q; SEEN_PART: all V lie inside the row and are read,
// without a branch between the reads; SEEN_EDGE: the row may end among them.
enum Seen { SEEN_ALL, SEEN_PART, SEEN_EDGE };
template <typename T, int V, uint32_t DEPTH, Seen SEEN>
__device__ __forceinline__ void add_rows(const AddArgs &a, const T *w, uint32_t s0, uint32_t q0,
                                         uint32_t first, uint32_t step, int32_t end0,
                                         int32_t see_more, float (&acc)[V]) {
    const uint32_t seen = a.queries - q0, rows = a.group * seen;
    const uint32_t step_g = step / seen, step_q = step % seen;
    uint32_t q = first % seen;
    const T *p = w + first / seen * a.stride_h + size_t(q0 + q) * a.stride_q + s0;
    const size_t on = step_g * a.stride_h + step_q * a.stride_q;
    const size_t wrap = a.stride_h - seen * a.stride_q;  // to the next head's first query
    auto load = [&](Pack<T, V> &v, uint32_t &live) {
        if constexpr (SEEN != SEEN_ALL) {
            const int32_t end = end0 + see_more * int32_t(q0 + q);
            live = end <= int32_t(s0) ? 0 : min(uint32_t(end) - s0, uint32_t(V));
        }
        if constexpr (SEEN != SEEN_EDGE) {
            v = *reinterpret_cast<const Pack<T, V> *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (uint32_t(i) < live) v.v[i] = p[i];
        }
        p += on;
        q += step_q;
        if (q >= seen) q -= seen, p += wrap;
    };
    auto add = [&](const Pack<T, V> &v, uint32_t live) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            acc[i] += SEEN == SEEN_ALL || uint32_t(i) < live ? to_float(v.v[i]) : 0.0f;
    };
    uint32_t r = first;
    for (; r + (DEPTH - 1) * step < rows; r += DEPTH * step) {
        Pack<T, V> v[DEPTH];
        uint32_t live[DEPTH];
#pragma unroll
        for (uint32_t k = 0; k < DEPTH; ++k) load(v[k], live[k]);
#pragma unroll
        for (uint32_t k = 0; k < DEPTH; ++k) add(v[k], live[k]);
    }
    Pack<T, V> v[DEPTH - 1];
    uint32_t live[DEPTH - 1];
#pragma unroll
    for (uint32_t k = 0; k < DEPTH - 1; ++k)
        if (r + k * step < rows) load(v[k], live[k]);
#pragma unroll
    for (uint32_t k = 0; k < DEPTH - 1; ++k)
        if (r + k * step < rows) add(v[k], live[k]);
}

// SPLIT: the rows are dealt out to the CTA's warps and to the cluster's CTAs;
// else every thread of the CTA has positions of its own.
template <typename T, int V, bool SPLIT>
__global__ void __launch_bounds__(ADD_BLOCK, 4) weight_add_kernel(const AddArgs a) {
    begin_kernel();
    const uint32_t b = blockIdx.y / a.heads, h = blockIdx.y % a.heads;
    const uint32_t n = length_of(a.lengths, b, a.capacity);
    const uint32_t rank = SPLIT ? blockIdx.x % a.cluster : 0;
    constexpr uint32_t WIDE = SPLIT ? 32 : ADD_BLOCK;  // threads side by side on a row
    const uint32_t tile = (SPLIT ? blockIdx.x / a.cluster : blockIdx.x) * (WIDE * V);
    if (tile >= n) return;  // the whole cluster's tile
    const uint32_t col = threadIdx.x % WIDE, s0 = tile + col * V;
    const T *const w = static_cast<const T *>(a.weights) + b * a.stride_b +
                       size_t(h) * a.group * a.stride_h;
    // Query q sees the positions below n - queries + 1 + q: the first queries
    // see nothing of a late tile.
    const int64_t end0 = a.causal ? int64_t(n) - a.queries + 1 : int64_t(n);
    uint32_t q0 = 0;
    if (a.causal && end0 <= int64_t(tile)) q0 = uint32_t(int64_t(tile) - end0 + 1);
    float acc[V] = {};
    float *const out = a.scores + b * a.score_b + h * a.score_h;
    if (q0 < a.queries) {
        const uint32_t first = SPLIT ? rank * ADD_WARPS + threadIdx.x / WIDE : 0;
        const uint32_t step = SPLIT ? a.cluster * ADD_WARPS : 1;
        const uint32_t last = tile + WIDE * V;
        const auto add = [&](auto seen) {
            add_rows<T, V, SPLIT ? 4 : 2, decltype(seen)::value>(
                a, w, s0, q0, first, step, int32_t(end0), int32_t(a.causal), acc);
        };
        if (end0 + int64_t(a.causal) * q0 >= int64_t(last))
            add(std::integral_constant<Seen, SEEN_ALL>{});
        else if (s0 + V <= a.capacity)
            add(std::integral_constant<Seen, SEEN_PART>{});
        else if (s0 < a.capacity)
            add(std::integral_constant<Seen, SEEN_EDGE>{});
    }
    if constexpr (!SPLIT) {
        using P = Pack<float, V < 4 ? V : 4>;
        if (a.score_packs && s0 + V <= n) {
#pragma unroll
            for (int i = 0; i < V; i += int(sizeof(P) / 4)) {
                P p = *reinterpret_cast<P *>(out + s0 + i);
#pragma unroll
                for (int j = 0; j < int(sizeof(P) / 4); ++j)
                    p.v[j] = fmaf(a.decay, p.v[j], acc[i + j]);
                *reinterpret_cast<P *>(out + s0 + i) = p;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (s0 + i < n) out[s0 + i] = fmaf(a.decay, out[s0 + i], acc[i]);
        }
    } else {
        __shared__ float sums[ADD_WARPS][WIDE * V], part[WIDE * V];
#pragma unroll
        for (int i = 0; i < V; ++i) sums[threadIdx.x / WIDE][i * WIDE + col] = acc[i];
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < WIDE * V; c += ADD_BLOCK) {
            float sum = 0;
#pragma unroll
            for (uint32_t k = 0; k < ADD_WARPS; ++k) sum += sums[k][c];
            part[c] = sum;
        }
        if (a.cluster == 1) __syncthreads();
        else cluster_sync();
        // Each CTA of the cluster finishes its share of the positions; sum c
        // is that of position c % WIDE * V + c / WIDE of the tile.
        for (uint32_t c = threadIdx.x; c < WIDE * V; c += ADD_BLOCK) {
            const uint32_t s = tile + c % WIDE * V + c / WIDE;
            if (c / 8 % a.cluster != rank || s >= n) continue;
            float sum = 0;
            for (uint32_t k = 0; k < a.cluster; ++k)
                sum += __uint_as_float(
                    cluster_read(reinterpret_cast<const uint32_t *>(&part[c]), k));
            out[s] = fmaf(a.decay, out[s], sum);
        }
        if (a.cluster > 1) cluster_sync();  // part stays until all have read it
    }
}

// ---------------------------------------------------------------------------
// Selection
//
// One cluster of CTAs a head.  Each CTA holds the order images of its slice of
// the head's totals in registers and, behind SELECT_PAGE of them, in shared
// memory (only what a slice has beyond three pages is read more than once), and
// radix selection finds the
// smallest kept image in three passes of 11, 11 and 10 bits: a pass counts the
// digits of the images that still match, and every CTA adds up the cluster's
// counts through distributed shared memory: 64 sums of 32 bins first, then the
// one sum's bins (every bin of every CTA took 64 us for 64 heads of 64 Ki
// positions in clusters of eight, bound by that memory; so 25).  Then a count
// of the larger and of the equal images of the CTAs and threads before gives
// every kept position its place, and a page's positions are put in order in shared memory and written
// out together.  When every image of the found bin stays, the passes below are
// left out (22 bits tell most totals apart).  Bound by latency: cluster
// barriers, remote reads and shared-memory atomics of one CTA after another.
// ---------------------------------------------------------------------------
constexpr uint32_t SELECT_BLOCK = 512;
constexpr uint32_t SELECT_WARPS = SELECT_BLOCK / 32;
constexpr uint32_t SELECT_BINS = 4 * SELECT_BLOCK;
constexpr uint32_t SELECT_MAX_CLUSTER = 8;
constexpr uint32_t SELECT_ITEMS = 16;  // images a thread holds
constexpr uint32_t SELECT_PAGE = SELECT_ITEMS * SELECT_BLOCK;
constexpr uint32_t SELECT_KEPT_PAGES = 2;  // in shared memory, at two CTAs an SM

struct SelectArgs {
    const float *scores;
    size_t score_b, score_h;
    const int32_t *lengths;
    uint32_t heads, capacity, budget, sinks, recent, cluster, kept_pages;
    int32_t *kept, *kept_lengths;
};

// Order image of a total: ascending as unsigned, -0 as +0, NaN as -inf.
__device__ __forceinline__ uint32_t score_image(float x) {
    x = x != x ? -INFINITY : x + 0.0f;
    const uint32_t u = __float_as_uint(x);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

// Inclusive sum over the warp.
__device__ __forceinline__ uint32_t warp_scan(uint32_t v) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= uint32_t(off)) v += y;
    }
    return v;
}

// Exclusive sum over the block of one value a thread; *total gets the sum.
__device__ __forceinline__ uint32_t select_scan(uint32_t v, uint32_t *warp_sums, uint32_t *total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t inc = warp_scan(v);
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    const uint32_t sums = warp_scan(lane < SELECT_WARPS ? warp_sums[lane] : 0);
    *total = __shfl_sync(0xffffffffu, sums, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, sums, (warp - 1) & 31);
    return (warp ? before : 0) + inc - v;
}

__global__ void __launch_bounds__(SELECT_BLOCK) cache_select_kernel(const SelectArgs a) {
    begin_kernel();
    // In turn: a page of images on its way from loads by item to runs of
    // SELECT_ITEMS a thread, the three passes' counts, a page of positions.
    __shared__ uint4 shared[(SELECT_PAGE + SELECT_BLOCK) / 4];
    static_assert(SELECT_PAGE + SELECT_BLOCK >= 3 * SELECT_BINS, "the counts fit");
    __shared__ uint32_t groups[3][SELECT_BINS / 32], warp_sums[2][SELECT_WARPS];
    __shared__ uint32_t chosen, left, whole, counts[2];
    uint32_t *const words = reinterpret_cast<uint32_t *>(shared);
    const uint32_t row = blockIdx.x / a.cluster, rank = blockIdx.x % a.cluster;
    const uint32_t b = row / a.heads, h = row % a.heads;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t n = length_of(a.lengths, b, a.capacity);
    int32_t *const kept = a.kept + size_t(row) * a.budget;
    const uint32_t tid_c = rank * SELECT_BLOCK + tid, threads_c = a.cluster * SELECT_BLOCK;
    if (h == 0 && tid_c == 0) a.kept_lengths[b] = int32_t(min(n, a.budget));
    if (n <= a.budget) {
        for (uint32_t j = tid_c; j < a.budget; j += threads_c) kept[j] = j < n ? int32_t(j) : -1;
        return;
    }
    for (uint32_t j = tid_c; j < a.sinks; j += threads_c) kept[j] = int32_t(j);
    for (uint32_t j = tid_c; j < a.recent; j += threads_c)
        kept[a.budget - a.recent + j] = int32_t(n - a.recent + j);
    const uint32_t need = a.budget - a.sinks - a.recent;
    if (need == 0) return;

    // This CTA's slice of the totals between (m is more than need), in pages
    // of SELECT_ITEMS a thread.  No total has the image 0, so places behind
    // the slice match nothing below.
    const float *const scores = a.scores + b * a.score_b + h * a.score_h + a.sinks;
    const uint32_t m = n - a.sinks - a.recent;
    const uint32_t per = (m + a.cluster - 1) / a.cluster;
    const uint32_t lo = min(rank * per, m), len = min(per, m - lo);
    const uint32_t pages = (len + SELECT_PAGE - 1) / SELECT_PAGE;
    using Items = uint32_t[SELECT_ITEMS];
    // Item k: position k * SELECT_BLOCK + tid of the page.  Pages behind the first
    // stay in shared memory, as far as it holds them, each thread's own items.
    extern __shared__ uint32_t select_kept_pages[];
    auto load = [&](uint32_t page, Items &v) {
#pragma unroll
        for (uint32_t k = 0; k < SELECT_ITEMS; ++k) {
            const uint32_t i = page * SELECT_PAGE + k * SELECT_BLOCK + tid;
            v[k] = i < len ? score_image(scores[lo + i]) : 0;
        }
    };
    auto load_again = [&](uint32_t page, Items &v) {
        if (page > a.kept_pages) return load(page, v);
        const uint32_t *const from = select_kept_pages + (page - 1) * SELECT_PAGE + tid;
#pragma unroll
        for (uint32_t k = 0; k < SELECT_ITEMS; ++k) v[k] = from[k * SELECT_BLOCK];
    };
    auto turn = [&](Items &v) {  // item k: position tid * SELECT_ITEMS + k
#pragma unroll
        for (uint32_t k = 0; k < SELECT_ITEMS; ++k) {
            const uint32_t i = k * SELECT_BLOCK + tid;
            words[i + i / SELECT_ITEMS] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < SELECT_ITEMS; ++k) v[k] = words[tid * (SELECT_ITEMS + 1) + k];
        __syncthreads();
    };
    Items held;
    load(0, held);
    turn(held);
#pragma unroll
    for (int p = 0; p < 3; ++p) shared[p * SELECT_BLOCK + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();

    uint32_t prefix = 0, want = need;  // `want` of the images that start with prefix stay
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int above = pass == 1 ? 21 : 10;
        const uint32_t mask = pass == 2 ? 1023 : 2047;
        uint32_t *const hist = words + pass * SELECT_BINS;
        auto count = [&](const Items &v) {
#pragma unroll
            for (uint32_t k = 0; k < SELECT_ITEMS; ++k)
                if (pass == 0 ? v[k] != 0 : v[k] >> above == prefix >> above)
                    atomicAdd(&hist[(v[k] >> shift) & mask], 1u);
        };
        count(held);
        for (uint32_t page = 1; page < pages; ++page) {
            Items v;
            if (pass == 0) {
                load(page, v);
                if (page <= a.kept_pages) {
                    uint32_t *const to = select_kept_pages + (page - 1) * SELECT_PAGE + tid;
#pragma unroll
                    for (uint32_t k = 0; k < SELECT_ITEMS; ++k) to[k * SELECT_BLOCK] = v[k];
                }
            } else {
                load_again(page, v);
            }
            count(v);
        }
        // This CTA's sums of 32 neighbouring bins: eight threads with four
        // bins each.
        __syncthreads();
        const uint4 q = shared[pass * SELECT_BLOCK + tid];
        uint32_t sum = q.x + q.y + q.z + q.w;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        if (lane % 8 == 0) groups[pass][tid / 8] = sum;
        if (a.cluster == 1) __syncthreads();
        else cluster_sync();
        // One warp adds up the cluster's sums and finds, from the highest
        // down, the group and then the bin in which the kept count is reached.
        if (warp == 0) {
            const uint32_t high =
                cluster_sum(&groups[pass][63 - 2 * lane], a.cluster);
            const uint32_t low = cluster_sum(&groups[pass][62 - 2 * lane], a.cluster);
            uint32_t higher = warp_scan(high + low) - high - low;
            const bool second = higher + high < want;
            if (second) higher += high;
            const uint32_t here = __ballot_sync(
                0xffffffffu, higher < want && want <= higher + (second ? low : high));
            const uint32_t from = __ffs(here) - 1;
            const uint32_t group =
                __shfl_sync(0xffffffffu, second ? 62 - 2 * lane : 63 - 2 * lane, from);
            const uint32_t rest = want - __shfl_sync(0xffffffffu, higher, from);
            const uint32_t bin = group * 32 + 31 - lane;
            const uint32_t number = cluster_sum(&hist[bin], a.cluster);
            const uint32_t over = warp_scan(number) - number;
            if (over < rest && rest <= over + number) {
                chosen = bin;
                left = rest - over;
                whole = rest - over == number;
            }
        }
        __syncthreads();
        prefix |= chosen << shift;
        want = left;
        if (whole) {  // every image of the bin stays: the bits below do not matter
            prefix -= 1;
            want = 0;
            break;
        }
    }

    // Images above prefix stay, and `want` of its equals, the lowest positions
    // first.  Both counts in one word: the larger ones in the low half.
    auto tally = [&](const Items &v) {
        uint32_t c = 0;
#pragma unroll
        for (uint32_t k = 0; k < SELECT_ITEMS; ++k)
            c += (v[k] > prefix ? 1u : 0u) + (v[k] == prefix ? 0x10000u : 0u);
        return c;
    };
    uint32_t total, before = select_scan(tally(held), warp_sums[0], &total);
    uint32_t larger = total & 0xffff, equal = total >> 16;  // the CTA's
    for (uint32_t page = 1; page < pages; ++page) {
        Items v;
        load_again(page, v);
        uint32_t sum;
        __syncthreads();
        select_scan(tally(v), warp_sums[1], &sum);
        larger += sum & 0xffff;
        equal += sum >> 16;
    }
    if (a.cluster > 1) {
        if (tid == 0) {
            counts[0] = larger;
            counts[1] = equal;
        }
        cluster_sync();
        larger = equal = 0;
        for (uint32_t c = 0; c < rank; ++c) {
            larger += cluster_read(&counts[0], c);
            equal += cluster_read(&counts[1], c);
        }
        cluster_arrive();
    } else {
        larger = equal = 0;
        __syncthreads();  // the last pass's counts have been read
    }
    // A page's kept positions are put together and then written in order.
    auto place = [&](uint32_t page, const Items &v) {
        const uint32_t first = larger + min(equal, want);
        uint32_t equals = equal + (before >> 16);
        uint32_t at = larger + (before & 0xffff) + min(equals, want) - first;
        const uint32_t i0 = page * SELECT_PAGE + tid * SELECT_ITEMS;
#pragma unroll
        for (uint32_t k = 0; k < SELECT_ITEMS; ++k) {
            const bool is_equal = v[k] == prefix;
            if (v[k] > prefix || (is_equal && equals < want)) words[at++] = a.sinks + lo + i0 + k;
            equals += is_equal;
        }
        larger += total & 0xffff;
        equal += total >> 16;
        __syncthreads();
        const uint32_t number = larger + min(equal, want) - first;
        int32_t *const out = kept + a.sinks + first;
        for (uint32_t j = tid; j < number; j += SELECT_BLOCK) out[j] = int32_t(words[j]);
    };
    place(0, held);
    for (uint32_t page = 1; page < pages; ++page) {
        Items v;
        load_again(page, v);
        __syncthreads();  // the page before has been written
        turn(v);
        before = select_scan(tally(v), warp_sums[0], &total);
        place(page, v);
    }
    if (a.cluster > 1) cluster_wait();
}

// ---------------------------------------------------------------------------
// Moving the cache's rows
//
// Bound by memory: every moved row is read and written once.  A thread takes
// MOVE_UNITS accesses of up to 16 bytes, its neighbours the next ones, and all
// of its reads are in flight before its first write.
// ---------------------------------------------------------------------------
constexpr uint32_t MOVE_BLOCK = 256;
constexpr uint32_t MOVE_UNITS = 8;

struct Rows {
    const char *src;
    char *dst;
    size_t src_b, src_h, src_s, dst_b, dst_h, dst_s;  // bytes
    uint32_t units, access;  // accesses of `access` bytes in a row
    uint32_t slices;         // in place: CTAs that share a row's accesses
    uint32_t first_block;
};

struct MoveArgs {
    Rows rows[RSORT_MAX_CACHES];
    uint32_t count, heads, budget, capacity;
    const int32_t *kept, *kept_lengths;
};

// The accesses of one thread: from the start, every `stride` units of the rows
// laid end to end.
struct Walk {
    uint32_t row, unit, rows_on, units_on, units;
    __device__ __forceinline__ Walk(uint64_t start, uint32_t stride, uint32_t units) : units(units) {
        row = uint32_t(start / units);
        unit = uint32_t(start - uint64_t(row) * units);
        rows_on = stride / units;
        units_on = stride % units;
    }
    __device__ __forceinline__ void next() {
        row += rows_on;
        unit += units_on;
        if (unit >= units) unit -= units, ++row;
    }
};

// Out of place: a CTA moves MOVE_BLOCK * MOVE_UNITS accesses; positions that
// cannot be read do not move.  (64 heads to 2048 rows of 256 bytes, keys and
// values, 139 MB: 18.5 us from a clean L2, which still holds part of the writes at
// the end, 31 us with four accesses a thread and divisions by the row's length for
// each; 24.5 us a call in a row, 5.5 TB/s.)
template <typename U>
__device__ __forceinline__ void move_out(const Rows &r, const int32_t *kept, const char *src,
                                         char *dst, uint32_t n, uint32_t capacity, uint32_t block) {
    const Walk start(uint64_t(block) * (MOVE_BLOCK * MOVE_UNITS) + threadIdx.x, MOVE_BLOCK,
                     r.units);
    int32_t from[MOVE_UNITS];
    U v[MOVE_UNITS];
    Walk at = start;
#pragma unroll
    for (uint32_t k = 0; k < MOVE_UNITS; ++k) {
        from[k] = at.row < n ? kept[at.row] : -1;
        at.next();
    }
    at = start;
#pragma unroll
    for (uint32_t k = 0; k < MOVE_UNITS; ++k) {
        if (uint32_t(from[k]) < capacity)
            v[k] = reinterpret_cast<const U *>(src + size_t(from[k]) * r.src_s)[at.unit];
        at.next();
    }
    at = start;
#pragma unroll
    for (uint32_t k = 0; k < MOVE_UNITS; ++k) {
        if (uint32_t(from[k]) < capacity)
            reinterpret_cast<U *>(dst + size_t(at.row) * r.dst_s)[at.unit] = v[k];
        at.next();
    }
}

// In place: one CTA walks a slice of every row in order, MOVE_BLOCK accesses a
// step.  kept[j] >= j, so a step's reads may run ahead of the writes of any step
// before it, but every read of a step has to come before its writes.  Reads go
// asynchronously into a ring of shared memory, MOVE_UNITS steps ahead, where
// each thread finds its own again; a barrier a step puts the reads first.
// (Without the ring a step waited for its reads: 256 heads of 4096 rows of 256
// bytes, keys and values, took 235 us, and 290 us with the steps of eight CTAs
// joined by a cluster's barrier.)
template <typename U>
__device__ __forceinline__ void move_in_place(const Rows &r, const int32_t *kept, char *rows,
                                              uint32_t n, uint32_t capacity, uint32_t slice,
                                              uint4 *ring_memory) {
    U(*const ring)[MOVE_BLOCK] = reinterpret_cast<U(*)[MOVE_BLOCK]>(ring_memory);
    const uint32_t per = (r.units + r.slices - 1) / r.slices;
    const uint32_t first = slice * per, units = min(per, r.units - min(first, r.units));
    if (units == 0 || n == 0 || kept[n - 1] == int32_t(n - 1)) return;  // nothing moves
    // Rows that stay in front: kept[j] == j up to some row, as positions ascend.
    const uint32_t hop = (n + MOVE_BLOCK - 1) / MOVE_BLOCK, probe = threadIdx.x * hop;
    const uint32_t same = __syncthreads_count(probe < n && kept[probe] == int32_t(probe));
    const uint32_t skip = same ? (same - 1) * hop : 0;
    kept += skip;
    rows += skip * r.src_s + first * sizeof(U);
    n -= skip;
    capacity -= skip;

    const uint32_t slot = uint32_t(__cvta_generic_to_shared(&ring[0][threadIdx.x]));
    constexpr uint32_t SLOTS = sizeof(U) * MOVE_BLOCK;
    Walk look(threadIdx.x, MOVE_BLOCK, units), load = look, store = look;
    int32_t from[MOVE_UNITS], ahead[MOVE_UNITS];
    auto read_kept = [&](int32_t(&f)[MOVE_UNITS]) {
#pragma unroll
        for (uint32_t k = 0; k < MOVE_UNITS; ++k) {
            f[k] = look.row < n ? int32_t(uint32_t(kept[look.row]) - skip) : -1;
            look.next();
        }
    };
    // The read of one access, if it moves; a group of its own either way.
    auto read = [&](uint32_t k, int32_t at) {
        if (uint32_t(at) < capacity && at > int32_t(load.row)) {
            const char *p = rows + size_t(at) * r.src_s + load.unit * sizeof(U);
            if constexpr (sizeof(U) >= 4)
                asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(slot + k * SLOTS),
                             "l"(p), "n"(sizeof(U) < 4 ? 4 : sizeof(U))
                             : "memory");
            else
                ring[k][threadIdx.x] = *reinterpret_cast<const U *>(p);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        load.next();
    };
    read_kept(from);
#pragma unroll
    for (uint32_t k = 0; k < MOVE_UNITS; ++k) read(k, from[k]);
    read_kept(ahead);
    const uint64_t total = uint64_t(n) * units;
    for (uint64_t i = 0; i < total; i += MOVE_BLOCK * MOVE_UNITS) {
        int32_t after[MOVE_UNITS];
        read_kept(after);
#pragma unroll
        for (uint32_t k = 0; k < MOVE_UNITS; ++k) {
            asm volatile("cp.async.wait_group %0;" ::"n"(MOVE_UNITS - 1) : "memory");
            __syncthreads();
            if (uint32_t(from[k]) < capacity && from[k] > int32_t(store.row))
                reinterpret_cast<U *>(rows + size_t(store.row) * r.src_s)[store.unit] =
                    ring[k][threadIdx.x];
            store.next();
            read(k, ahead[k]);
            from[k] = ahead[k];
            ahead[k] = after[k];
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <bool IN_PLACE>
__global__ void __launch_bounds__(MOVE_BLOCK) cache_move_kernel(const __grid_constant__ MoveArgs a) {
    begin_kernel();
    uint32_t t = 0;
    while (t + 1 < a.count && blockIdx.x >= a.rows[t + 1].first_block) ++t;
    const Rows &r = a.rows[t];
    const uint32_t block = blockIdx.x - r.first_block;
    const uint32_t bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads;
    const uint32_t n = min(length_of(a.kept_lengths, b, a.budget), a.capacity);
    const int32_t *const kept = a.kept + size_t(bh) * a.budget;
    const char *const src = r.src + b * r.src_b + h * r.src_h;
    char *const dst = r.dst + b * r.dst_b + h * r.dst_h;
    __shared__ uint4 ring[IN_PLACE ? MOVE_UNITS * MOVE_BLOCK : 1];
    auto go = [&](auto unit) {
        using U = decltype(unit);
        if constexpr (IN_PLACE) move_in_place<U>(r, kept, dst, n, a.capacity, block, ring);
        else move_out<U>(r, kept, src, dst, n, a.capacity, block);
    };
    switch (r.access) {
        case 16: go(uint4{}); break;
        case 8: go(uint2{}); break;
        case 4: go(uint32_t{}); break;
        case 2: go(uint16_t{}); break;
        default: go(uint8_t{}); break;
    }
}

// CTAs of a head: enough to hold its totals in registers, as long as all heads
// run at once (two CTAs an SM).  A CTA costs about 9 us however short its slice:
// 64 heads of 64 Ki positions took 38 / 25 / 25 us on 2 / 4 / 8 CTAs each (eight
// need a second wave; 22.5 us on 4 with the second page in shared memory), 512
// heads of 8 Ki take 17 / 37 / 76 us on 1 / 2 / 4.
uint32_t select_cluster(uint32_t rows, uint32_t capacity, uint32_t sms) {
    uint32_t c = 1;
    while (c < SELECT_MAX_CLUSTER && capacity / c > SELECT_PAGE && rows * c <= sms) c *= 2;
    return c;
}

// batch x heads is a grid dimension of at most 65535.
rsort_status check_grid(size_t batch, size_t heads, size_t capacity) {
    if (batch > 65535 || heads > 65535 || batch * heads > 65535)
        return fail(RSORT_SIZE_OVERFLOW, "cache batch times heads", 65535, batch * heads);
    if (capacity > size_t(INT_MAX) - 1)
        return fail(RSORT_SIZE_OVERFLOW, "cache capacity (32-bit positions)");
    return RSORT_OK;
}

}  // namespace

extern "C" {

rsort_status rsort_attention_weight_add(rsort_key_t type, const void *d_weights, size_t stride_b,
                                        size_t stride_h, size_t stride_q, size_t batch,
                                        size_t heads, size_t group, size_t queries,
                                        size_t capacity, const int32_t *d_lengths, float decay,
                                        int causal, float *d_scores, size_t score_stride_b,
                                        size_t score_stride_h, rsort_stream_t stream) {
    const size_t eb = real_bytes(type);
    if (!eb) return fail(RSORT_BAD_ARGUMENT, "attention weight type (f32, f16 or bf16)");
    rsort_status st = check_grid(batch, heads, capacity);
    if (st != RSORT_OK) return st;
    if (group < 1 || group > size_t(INT_MAX) || queries > size_t(INT_MAX) / group)
        return fail(RSORT_BAD_ARGUMENT, "attention weight heads per cache head or queries");
    if (batch == 0 || heads == 0 || capacity == 0) return RSORT_OK;
    if ((queries && !d_weights) || !d_scores) return fail(RSORT_BAD_ARGUMENT, "null buffer");
    constexpr size_t most = size_t(1) << 50;
    Strided weights, scores;
    if (stride_b > most || stride_h > most || stride_q > most || score_stride_b > most ||
        score_stride_h > most ||
        !strided(d_weights, capacity * eb,
                 {{queries, stride_q * eb}, {heads * group, stride_h * eb}, {batch, stride_b * eb}},
                 &weights))
        return fail(RSORT_SIZE_OVERFLOW, "attention weight strides");
    if (!strided(d_scores, 4,
                 {{capacity, 4}, {heads, score_stride_h * 4}, {batch, score_stride_b * 4}}, &scores))
        return fail(RSORT_SIZE_OVERFLOW, "cache score strides");
    if (!items_apart(scores)) return fail(RSORT_BAD_ARGUMENT, "cache score strides overlap");
    if (!apart(scores, weights))
        return fail(RSORT_BAD_ARGUMENT, "cache scores overlap the weights");
    if (d_lengths && !apart(scores, packed(d_lengths, batch * 4)))
        return fail(RSORT_BAD_ARGUMENT, "cache scores overlap the lengths");
    st = check_alignment(addr(d_weights), eb, "attention weights alignment");
    if (st == RSORT_OK) st = check_alignment(addr(d_scores), 4, "cache scores alignment");
    if (st == RSORT_OK) st = check_alignment(addr(d_lengths), 4, "cache lengths alignment");
    if (st != RSORT_OK) return st;
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;
    AddArgs a{d_weights,         stride_b,       stride_h,        stride_q,
              d_scores,          score_stride_b, score_stride_h,  d_lengths,
              uint32_t(heads),   uint32_t(group), uint32_t(queries), uint32_t(capacity),
              1,                 decay,          causal != 0,
              ((addr(d_scores) | score_stride_b * 4 | score_stride_h * 4) & 15) == 0};
    const size_t access =
        access_bytes(addr(d_weights) | stride_b * eb | stride_h * eb | stride_q * eb, 16);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // Few rows: one thread sums them.
    // More: warps, and CTAs while the positions leave SMs without work.
    const size_t rows = group * queries;
    const bool split = rows > ADD_FEW_ROWS;
    auto go = [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        const size_t per = size_t(split ? 32 : ADD_BLOCK) * V;
        const size_t tiles = (capacity + per - 1) / per;
        if (split)
            while (a.cluster < ADD_MAX_CLUSTER && a.cluster * ADD_WARPS * 4 < rows &&
                   tiles * batch * heads * a.cluster < size_t(sms) * 4)
                a.cluster *= 2;
        const dim3 grid(unsigned(tiles * a.cluster), unsigned(batch * heads));
        return launch_early(split ? weight_add_kernel<T, V, true> : weight_add_kernel<T, V, false>,
                            grid, ADD_BLOCK, 0, a.cluster, s, a);
    };
    LaunchScope scope(RSORT_KERNEL_CACHE, s);
    return launched(with_type(type, access, go), "attention weight add launch");
}

rsort_status rsort_cache_select(const float *d_scores, size_t score_stride_b,
                                size_t score_stride_h, const int32_t *d_lengths, size_t batch,
                                size_t heads, size_t capacity, size_t budget, size_t sinks,
                                size_t recent, int32_t *d_kept, int32_t *d_kept_lengths,
                                rsort_stream_t stream) {
    rsort_status st = check_grid(batch, heads, capacity);
    if (st != RSORT_OK) return st;
    if (budget < 1 || budget > size_t(INT_MAX))
        return fail(RSORT_BAD_ARGUMENT, "cache budget", 1, budget);
    if (sinks > budget || recent > budget - sinks)
        return fail(RSORT_BAD_ARGUMENT, "cache sinks and recent positions exceed the budget",
                    budget, sinks + recent);
    if (batch == 0 || heads == 0) return RSORT_OK;
    if ((capacity && !d_scores) || !d_kept || !d_kept_lengths)
        return fail(RSORT_BAD_ARGUMENT, "null buffer");
    constexpr size_t most = size_t(1) << 50;
    if (score_stride_b > most || score_stride_h > most)
        return fail(RSORT_SIZE_OVERFLOW, "cache score strides");
    st = check_alignment(addr(d_scores) | addr(d_lengths) | addr(d_kept) | addr(d_kept_lengths), 4,
                         "cache selection alignment");
    if (st != RSORT_OK) return st;
    const Strided kept = packed(d_kept, batch * heads * budget * 4);
    const Strided kept_n = packed(d_kept_lengths, batch * 4);
    const Strided lengths = packed(d_lengths, d_lengths ? batch * 4 : 0);
    if (!apart(kept_n, lengths))
        return fail(RSORT_BAD_ARGUMENT, "kept lengths overlap the lengths");
    Strided scores{};
    if (!strided(d_scores, 4,
                 {{capacity, 4}, {heads, score_stride_h * 4}, {batch, score_stride_b * 4}}, &scores))
        return fail(RSORT_SIZE_OVERFLOW, "cache score strides");
    if (!apart(kept, scores) || !apart(kept_n, scores) || !apart(kept, kept_n) ||
        !apart(kept, lengths))
        return fail(RSORT_BAD_ARGUMENT, "kept positions overlap another buffer");
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;
    const uint32_t rows = uint32_t(batch * heads);
    const uint32_t cluster = select_cluster(rows, uint32_t(capacity), uint32_t(sms));
    const uint32_t slice = uint32_t((capacity + cluster - 1) / cluster);
    const uint32_t kept_pages =
        slice <= SELECT_PAGE
            ? 0
            : std::min((slice + SELECT_PAGE - 1) / SELECT_PAGE - 1, SELECT_KEPT_PAGES);
    SelectArgs a{d_scores,           score_stride_b,  score_stride_h,  d_lengths,
                 uint32_t(heads),    uint32_t(capacity), uint32_t(budget), uint32_t(sinks),
                 uint32_t(recent),   cluster,         kept_pages,      d_kept,
                 d_kept_lengths};
    const size_t shared = size_t(kept_pages) * SELECT_PAGE * sizeof(uint32_t);
    if (shared) {
        const cudaError_t e =
            cudaFuncSetAttribute(cache_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(SELECT_KEPT_PAGES * SELECT_PAGE * sizeof(uint32_t)));
        if (e != cudaSuccess) return launched(e, "cache selection shared memory");
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    LaunchScope scope(RSORT_KERNEL_CACHE, s);
    return launched(launch_early(cache_select_kernel, dim3(rows * cluster), SELECT_BLOCK, shared, cluster,
                                 s, a),
                    "cache selection launch");
}

rsort_status rsort_cache_compact(const rsort_cache_rows *caches, size_t ncaches,
                                 const int32_t *d_kept, const int32_t *d_kept_lengths,
                                 size_t batch, size_t heads, size_t budget, size_t capacity,
                                 rsort_stream_t stream) {
    if (ncaches > RSORT_MAX_CACHES)
        return fail(RSORT_BAD_ARGUMENT, "cache count", RSORT_MAX_CACHES, ncaches);
    rsort_status st = check_grid(batch, heads, capacity);
    if (st != RSORT_OK) return st;
    if (budget > size_t(INT_MAX)) return fail(RSORT_SIZE_OVERFLOW, "cache budget");
    if (ncaches == 0 || batch == 0 || heads == 0 || budget == 0 || capacity == 0) return RSORT_OK;
    if (!caches || !d_kept || !d_kept_lengths) return fail(RSORT_BAD_ARGUMENT, "null buffer");
    st = check_alignment(addr(d_kept) | addr(d_kept_lengths), 4, "cache selection alignment");
    if (st != RSORT_OK) return st;
    const size_t bh = batch * heads;
    const Strided kept = packed(d_kept, bh * budget * 4);
    const Strided kept_n = packed(d_kept_lengths, batch * 4);
    Strided in[RSORT_MAX_CACHES], out[RSORT_MAX_CACHES];
    bool in_place = false;
    for (size_t i = 0; i < ncaches; ++i) {
        const rsort_cache_rows &c = caches[i];
        if (c.row_bytes == 0 || c.row_bytes > size_t(INT_MAX))
            return fail(RSORT_BAD_ARGUMENT, "cache row bytes", 1, c.row_bytes);
        if (!c.src || !c.dst) return fail(RSORT_BAD_ARGUMENT, "null buffer");
        const bool same = c.src == c.dst;
        if (i && same != in_place)
            return fail(RSORT_BAD_ARGUMENT, "caches move all in place or all out of place");
        in_place = same;
        if (same && (c.src_stride_b != c.dst_stride_b || c.src_stride_h != c.dst_stride_h ||
                     c.src_stride_s != c.dst_stride_s))
            return fail(RSORT_BAD_ARGUMENT, "cache strides in place");
        const size_t written = same || budget > capacity ? capacity : budget;
        if (!strided(c.src, c.row_bytes,
                     {{capacity, c.src_stride_s}, {heads, c.src_stride_h}, {batch, c.src_stride_b}},
                     &in[i]) ||
            !strided(c.dst, c.row_bytes,
                     {{written, c.dst_stride_s}, {heads, c.dst_stride_h}, {batch, c.dst_stride_b}},
                     &out[i]))
            return fail(RSORT_SIZE_OVERFLOW, "cache strides");
        if (!items_apart(out[i])) return fail(RSORT_BAD_ARGUMENT, "cache strides overlap");
        if (!apart(out[i], kept) || !apart(out[i], kept_n))
            return fail(RSORT_BAD_ARGUMENT, "caches overlap the kept positions");
    }
    for (size_t i = 0; i < ncaches; ++i)
        for (size_t j = 0; j < ncaches; ++j)
            if ((i != j && !apart(out[i], out[j])) ||
                ((i != j || !in_place) && !apart(out[i], in[j])))
                return fail(RSORT_BAD_ARGUMENT, "caches overlap");
    int sms = 0;
    st = current_sm_count(&sms);
    if (st != RSORT_OK) return st;

    MoveArgs a{};
    a.count = uint32_t(ncaches);
    a.heads = uint32_t(heads);
    a.budget = uint32_t(budget);
    a.capacity = uint32_t(capacity);
    a.kept = d_kept;
    a.kept_lengths = d_kept_lengths;
    constexpr uint64_t per = MOVE_BLOCK * MOVE_UNITS;
    uint64_t blocks = 0;
    for (size_t i = 0; i < ncaches; ++i) {
        const rsort_cache_rows &c = caches[i];
        Rows &r = a.rows[i];
        r.src = static_cast<const char *>(c.src);
        r.dst = static_cast<char *>(c.dst);
        r.src_b = c.src_stride_b;
        r.src_h = c.src_stride_h;
        r.src_s = c.src_stride_s;
        r.dst_b = c.dst_stride_b;
        r.dst_h = c.dst_stride_h;
        r.dst_s = c.dst_stride_s;
        r.access = uint32_t(access_bytes(addr(c.src) | addr(c.dst) | r.src_b | r.src_h | r.src_s |
                                             r.dst_b | r.dst_h | r.dst_s | c.row_bytes,
                                         16));
        r.units = uint32_t(c.row_bytes / r.access);
        r.first_block = uint32_t(blocks);
        r.slices = 1;
        if (in_place) {
            // Slices of at least 64 bytes, until there are 16 CTAs an SM: they cost
            // a full batch little (32 x 8 heads of 4096 rows: 175 / 162 / 168 us for
            // 4 / 8 / 16 an SM), and when few heads move they shorten the walk (8
            // heads among 256: 48 / 27 / 17 us).
            while (bh * ncaches * r.slices < size_t(sms) * 16 && c.row_bytes / r.slices >= 128)
                r.slices *= 2;
            blocks += r.slices;
        } else {
            blocks += (uint64_t(budget) * r.units + per - 1) / per;
        }
        if (blocks > uint64_t(INT_MAX)) return fail(RSORT_SIZE_OVERFLOW, "cache rows");
    }
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    LaunchScope scope(RSORT_KERNEL_CACHE, s);
    const dim3 grid{unsigned(blocks), unsigned(bh)};
    if (!in_place)
        return launched(launch_early(cache_move_kernel<false>, grid, MOVE_BLOCK, 0, 1, s, a),
                        "cache compaction launch");
    // Not early: the CTAs of the few heads that move would crowd on the SMs that
    // happen to be free (8 of 256 heads: 23 us against 16).
    cache_move_kernel<true><<<grid, MOVE_BLOCK, 0, s>>>(a);
    return launched(cudaGetLastError(), "cache compaction launch");
}

}  // extern "C"
