// Shared by the operators that move wide rows (expert routing and cache
// eviction): the element types they compute in, packs of elements moved with
// one access, and the argument checks of strided row ranges.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "rsort_internal.cuh"

namespace rsort {

// V elements moved with one access; the address is aligned to the pack.
template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) {
    return __float2half_rn(x);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// The types that rows with arithmetic may have, and their sizes (0: not one).
inline size_t real_bytes(rsort_key_t t) {
    return t == RSORT_F32 ? 4 : (t == RSORT_F16 || t == RSORT_BF16) ? 2 : 0;
}

// Largest power of two (at most `most`) that divides every address and
// stride OR-ed into `bits`: the widest access the rows allow.
inline size_t access_bytes(uintptr_t bits, size_t most) {
    size_t a = most;
    while (a > 1 && (bits & (a - 1)) != 0) a >>= 1;
    return a;
}

// n rows `stride` bytes apart stay below 2^56 bytes, far beyond any device,
// so no offset of theirs wraps.
inline bool rows_fit(size_t n, size_t stride, size_t bytes) {
    constexpr size_t kMost = size_t(1) << 56;
    return bytes <= kMost && (n == 0 || stride <= kMost / n);
}

// An array of `bytes`-wide items along up to four axes, strides in bytes;
// axes of one entry dropped, smallest stride first.  [first, last) spans it
// (nothing without items).
struct Axis {
    size_t count, stride;
};
struct Strided {
    uintptr_t first, last;
    size_t bytes;
    int axes;
    Axis axis[4];
};

// `bytes` next to one another.
inline Strided packed(const void *p, size_t bytes) {
    Strided r;
    r.first = addr(p);
    r.last = r.first + bytes;
    r.bytes = bytes;
    r.axes = 0;
    return r;
}

// False when an offset could wrap.
inline bool strided(const void *p, size_t bytes, std::initializer_list<Axis> axes, Strided *out) {
    Strided &r = *out;
    r = packed(p, bytes);
    bool empty = bytes == 0;
    for (const Axis &x : axes) {
        if (!rows_fit(x.count, x.stride, bytes)) return false;
        empty |= x.count == 0;
        if (x.count <= 1) continue;
        int at = r.axes++;
        for (; at > 0 && r.axis[at - 1].stride > x.stride; --at) r.axis[at] = r.axis[at - 1];
        r.axis[at] = x;
        r.last += (x.count - 1) * x.stride;
    }
    if (empty) r.last = r.first;
    return true;
}

// No two items share a byte (sufficient: every stride spans what lies inside).
inline bool items_apart(const Strided &a) {
    size_t inner = a.bytes;
    for (int i = 0; i < a.axes; ++i) {
        if (a.axis[i].stride < inner) return false;
        inner += (a.axis[i].count - 1) * a.axis[i].stride;
    }
    return true;
}

// Both arrays lie within one interval each modulo some stride s of theirs, and
// these are apart, as keys and values of one allocation are (axes whose strides
// are multiples of s leave an address as it is modulo s).
inline bool side_by_side(const Strided &a, const Strided &b) {
    const auto width = [](const Strided &x, size_t s) {
        size_t w = x.bytes;
        for (int i = 0; i < x.axes; ++i)
            if (x.axis[i].stride % s) w += (x.axis[i].count - 1) * x.axis[i].stride;
        return w;
    };
    const auto within = [&](size_t s) {
        if (s == 0) return false;
        const size_t wa = width(a, s), wb = width(b, s);
        const size_t d = b.first >= a.first ? (b.first - a.first) % s
                                            : (s - (a.first - b.first) % s) % s;
        return wa <= d && wb <= s - d;
    };
    for (int i = 0; i < a.axes; ++i)
        if (within(a.axis[i].stride)) return true;
    for (int i = 0; i < b.axes; ++i)
        if (within(b.axis[i].stride)) return true;
    return false;
}

// No item of one shares a byte with an item of the other (sufficient: their
// spans are apart, or they lie side by side).
inline bool apart(const Strided &a, const Strided &b) {
    return a.first >= b.last || b.first >= a.last || a.first >= a.last || b.first >= b.last ||
           side_by_side(a, b);
}

// Thread-block clusters: a word of CTA `rank`'s shared memory at the same
// place as `p`, and the cluster's barrier in one piece or in two.
__device__ __forceinline__ uint32_t cluster_address(const void *p, uint32_t rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(at)
        : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank));
    return at;
}
__device__ __forceinline__ uint32_t cluster_read(const uint32_t *p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_address(p, rank)));
    return v;
}
// The sum of that word over a cluster of at most eight CTAs, read at once.
__device__ __forceinline__ uint32_t cluster_sum(const uint32_t *p, uint32_t ctas) {
    if (ctas == 1) return *p;
    uint32_t v[8], sum = 0;
#pragma unroll
    for (uint32_t c = 0; c < 8; ++c) v[c] = c < ctas ? cluster_read(p, c) : 0;
#pragma unroll
    for (uint32_t c = 0; c < 8; ++c) sum += v[c];
    return sum;
}
__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}

// Programmatic dependent launch: a kernel of these operators may be brought
// onto the SMs while the one before it on the stream runs out.  Every CTA calls
// begin_kernel before it touches memory that another kernel may write: it waits
// until the kernels before are complete, and lets the next one come.
__device__ __forceinline__ void begin_kernel() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launches a kernel that calls begin_kernel, in clusters of `cluster` CTAs.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, unsigned block, size_t shared,
                         unsigned cluster, cudaStream_t stream, Args &&...args) {
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

inline rsort_status fail(rsort_status s, const char *role, size_t expected = 0,
                         size_t actual = 0) {
    return record_failure(s, role, expected, actual);
}

inline rsort_status launched(cudaError_t e, const char *role) {
    return e == cudaSuccess ? RSORT_OK : fail(RSORT_CUDA_ERROR, role);
}

// Calls f with the element type and the elements of one access.
template <typename F> cudaError_t with_type(rsort_key_t type, size_t access, F f) {
    if (type == RSORT_F32) {
        if (access >= 16) return f(float{}, std::integral_constant<int, 4>{});
        if (access >= 8) return f(float{}, std::integral_constant<int, 2>{});
        return f(float{}, std::integral_constant<int, 1>{});
    }
    auto half = [&](auto t) {
        if (access >= 16) return f(t, std::integral_constant<int, 8>{});
        if (access >= 8) return f(t, std::integral_constant<int, 4>{});
        if (access >= 4) return f(t, std::integral_constant<int, 2>{});
        return f(t, std::integral_constant<int, 1>{});
    };
    return type == RSORT_F16 ? half(__half{}) : half(__nv_bfloat16{});
}

}  // namespace rsort
