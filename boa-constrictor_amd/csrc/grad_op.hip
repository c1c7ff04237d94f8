// The norm of all gradients of a model together, and their clipping by it (boa_grad_norm, boa_clip_grads).
//
//   norm = sqrt(sum over all x of x^2), or the largest |x|;  x *= min(1, max_norm / (norm + 1e-6))
//
// Two launches for up to MOST tensors: squares summed by workgroups that walk blocks of all tensors (their addresses and sizes come
// with the launch, so nothing is copied to the device), then the scaling, whose workgroups add the partial sums themselves.
// Sums and the factor are in 64 bits: squares of large float32 values (and of scaled float16 gradients) stay in range, a norm that
// float32 cannot hold still scales, and it costs nothing beside the memory that bounds both.  Where the factor is 1 nothing is
// written.
//
// Measured: 141 gradients of 32 MB in float32 7 us for the sums (4.4 TB/s) and 12 for the scaling (5.4, from the last-level cache in
// part); 277 of 122 MB in bfloat16, two launches of each, 25 and 51 (4.9 and 4.8 TB/s).  Bound by memory, and below some 100 MB by
// the host, which looks at each gradient: 58 and 111 us.
#include <algorithm>
#include <vector>

#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int WG = 256, WAVES = WG / 64;
constexpr int MOST = 180;        // tensors of a launch: 21 bytes each of the 4 KB that its arguments may take
constexpr int MAX_GROUPS = 1024;  // workgroups of a norm launch, and its partial sums
constexpr int AT_ONCE = 4;        // accesses of 16 bytes that a thread has in flight
constexpr int SPAN = WG * AT_ONCE * 16;  // bytes of a block
constexpr int64_t MOST_BYTES = INT64_C(1) << 39;  // of a tensor

struct Table {
    void* p[MOST];          // down to a multiple of 16 bytes
    int64_t bytes[MOST];    // from there to the tensor's end
    uint32_t first[MOST + 1];  // number of its first block
    uint8_t dtype[MOST];    // and in the upper bits the bytes before the tensor (0 to 15)
    int32_t n;
};
static_assert(sizeof(Table) <= 3900, "");

// Block `k`: calls f with the tensor's type as a constant.
template <class F>
__device__ __forceinline__ void of_block(const Table& t, uint32_t k, F f) {
    int lo = 0, hi = t.n;
    while (hi - lo > 1) {
        const int m = (lo + hi) / 2;
        if (t.first[m] <= k) lo = m;
        else hi = m;
    }
    char* p = static_cast<char*>(t.p[lo]);
    const int64_t at = (int64_t)(k - t.first[lo]) * SPAN, end = t.bytes[lo];
    const int before = t.dtype[lo] >> 4;
    switch (t.dtype[lo] & 15) {
        case DT_F32: return f(std::integral_constant<int, DT_F32>(), p, at, end, before);
        case DT_BF16: return f(std::integral_constant<int, DT_BF16>(), p, at, end, before);
        default: return f(std::integral_constant<int, DT_F16>(), p, at, end, before);
    }
}

// The values of 16 bytes at byte `at` of a tensor; zeros outside of it.
template <int DT>
__device__ __forceinline__ u32x4 load16(const char* p, int64_t at, int64_t end, int before) {
    constexpr int ES = (int)sizeof(typename Elem<DT>::T);
    if (at >= before && at + 16 <= end) return *reinterpret_cast<const u32x4*>(p + at);
    u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 16 / ES; ++e)
        if (at + e * ES >= before && at + e * ES < end) {
            const auto v = *reinterpret_cast<const typename Elem<DT>::T*>(p + at + e * ES);
            if constexpr (ES == 4) r[e] = __float_as_uint(v);
            else r[e / 2] |= (uint32_t)v << (16 * (e & 1));
        }
    return r;
}

struct Square {
    static __device__ __forceinline__ double of(double a, float x) { return __builtin_fma((double)x, (double)x, a); }
    static __device__ __forceinline__ double join(double a, double b) { return a + b; }
    static __device__ __forceinline__ double norm(double a) { return __builtin_sqrt(a); }
};
struct Largest {  // a NaN stays
    static __device__ __forceinline__ double of(double a, float x) { return join(a, (double)fabsf(x)); }
    static __device__ __forceinline__ double join(double a, double b) { return a > b || a != a ? a : b; }
    static __device__ __forceinline__ double norm(double a) { return a; }
};

// Over the workgroup, in a fixed order; every thread gets it.
template <class Op>
__device__ __forceinline__ double over_group(double v) {
    __shared__ double s[WAVES];
    for (int o = 32; o > 0; o >>= 1) v = Op::join(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return Op::join(Op::join(s[0], s[1]), Op::join(s[2], s[3]));
}

template <class Op>
__global__ void __launch_bounds__(WG) k_grad_part(const Table t, double* part) {
    double v = 0.0;
    for (uint32_t k = blockIdx.x; k < t.first[t.n]; k += gridDim.x)
        of_block(t, k, [&](auto dt, const char* p, int64_t at, int64_t end, int before) {
            constexpr int DT = decltype(dt)::value, V = wide<DT>();
            u32x4 r[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) r[i] = load16<DT>(p, at + (i * WG + threadIdx.x) * 16, end, before);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                float x[V];
                Raw<DT, V>::unpack(r[i], x);
#pragma unroll
                for (int e = 0; e < V; ++e) v = Op::of(v, x[e]);
            }
        });
    v = over_group<Op>(v);
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <class Op>
__device__ __forceinline__ double all_parts(const double* part, int n) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += WG) v = Op::join(v, part[i]);
    return over_group<Op>(v);
}

template <class Op>
__global__ void __launch_bounds__(WG) k_grad_norm(const double* part, int n, float* norm) {
    const double v = all_parts<Op>(part, n);
    if (threadIdx.x == 0) *norm = (float)Op::norm(v);
}

template <class Op>
__global__ void __launch_bounds__(WG) k_grad_scale(const Table t, const double* part, int n, double max_norm, float* norm) {
    const double total = Op::norm(all_parts<Op>(part, n));
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    const double f = max_norm / (total + 1e-6);  // NaN where the norm is
    if (f >= 1.0) return;
    for (uint32_t k = blockIdx.x; k < t.first[t.n]; k += gridDim.x)
        of_block(t, k, [&](auto dt, char* p, int64_t at, int64_t end, int before) {
            constexpr int DT = decltype(dt)::value, V = wide<DT>(), ES = 16 / V;
            u32x4 r[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) r[i] = load16<DT>(p, at + (i * WG + threadIdx.x) * 16, end, before);
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int64_t a = at + (i * WG + threadIdx.x) * 16;
                float x[V];
                Raw<DT, V>::unpack(r[i], x);
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = (float)((double)x[e] * f);
                if (a >= before && a + 16 <= end) {
                    *reinterpret_cast<u32x4*>(p + a) = Raw<DT, V>::pack(x);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (a + e * ES >= before && a + e * ES < end)
                            *reinterpret_cast<typename Elem<DT>::T*>(p + a + e * ES) = Elem<DT>::st(x[e]);
                }
            }
        });
}

int element_bytes(int dtype) { return dtype == BOA_DT_F32 ? 4 : 2; }

int check_grads(const char* who, int32_t n, const void* const* grads, const int64_t* counts, const int32_t* dtypes, const void* work,
                int64_t work_bytes) {
    if (n < 0 || (n > 0 && (!grads || !counts || !dtypes))) return boa_fail(BOA_ERR_ARG, "%s: null pointer", who);
    for (int32_t i = 0; i < n; ++i) {
        if (dtypes[i] < BOA_DT_F32 || dtypes[i] > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, dtypes[i]);
        // blocks are counted in 32 bits; no tensor is longer than a device's memory
        if (counts[i] < 0 || counts[i] > MOST_BYTES / element_bytes(dtypes[i]) || (counts[i] > 0 && !grads[i]) || (uintptr_t)grads[i] % element_bytes(dtypes[i]))
            return boa_fail(BOA_ERR_ARG, "%s: tensor %d of %lld values at %p", who, i, (long long)counts[i], grads[i]);
    }
    if (!work || (uintptr_t)work % 8 || work_bytes < boa_grad_norm_work_bytes(n))
        return boa_fail(BOA_ERR_ARG, "%s: workspace of %lld bytes, needs %lld at a multiple of 8", who, (long long)work_bytes,
                        (long long)boa_grad_norm_work_bytes(n));
    return BOA_OK;
}

// Calls f with a table of the next tensors and its number of blocks, until all have been in one.  Empty tensors are left out.
template <class F>
int with_tables(int32_t n, const void* const* grads, const int64_t* counts, const int32_t* dtypes, F f) {
    Table t;
    t.n = 0;
    uint64_t blocks = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (counts[i] == 0) continue;
        const uintptr_t p = (uintptr_t)grads[i];
        const int before = (int)(p % 16);
        const int64_t bytes = before + counts[i] * element_bytes(dtypes[i]);
        const uint64_t mine = (uint64_t)ceil_div(bytes, SPAN);
        if (t.n == MOST || blocks + mine > UINT32_MAX / 2) {
            if (const int rc = f(t, (uint32_t)blocks)) return rc;
            t.n = 0;
            blocks = 0;
        }
        t.p[t.n] = reinterpret_cast<void*>(p - before);
        t.bytes[t.n] = bytes;
        t.dtype[t.n] = (uint8_t)(dtypes[i] | before << 4);
        t.first[t.n++] = (uint32_t)blocks;
        blocks += mine;
        t.first[t.n] = (uint32_t)blocks;
    }
    return t.n > 0 ? f(t, (uint32_t)blocks) : (int)BOA_OK;
}

// Partial sums of all tensors; how many there are.
template <class Op>
int launch_parts(int32_t n, const void* const* grads, const int64_t* counts, const int32_t* dtypes, double* part, int& parts, hipStream_t s) {
    parts = 0;
    return with_tables(n, grads, counts, dtypes, [&](const Table& t, uint32_t blocks) {
        const uint32_t groups = blocks < MAX_GROUPS ? blocks : MAX_GROUPS;
        hipLaunchKernelGGL((k_grad_part<Op>), dim3(groups), dim3(WG), 0, s, t, part + parts);
        BOA_HIP_TRY(hipGetLastError());
        parts += (int)groups;
        return (int)BOA_OK;
    });
}

template <class F>
int with_norm(int largest, F f) {
    return largest ? f(Largest()) : f(Square());
}

}  // namespace

// The partial sums of as many launches as n tensors may take: one for MOST of them, and more where 63 or more of the longest fill
// one (2^25 blocks each of 2^31).
extern "C" int64_t boa_grad_norm_work_bytes(int32_t n) {
    return (n > 0 ? 3 * ceil_div(n, MOST) + 1 : 1) * (int64_t)MAX_GROUPS * (int64_t)sizeof(double);
}

extern "C" int boa_grad_norm(int32_t n, const void* const* d_grads, const int64_t* counts, const int32_t* dtypes, int largest, float* d_norm,
                             void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_grads("boa_grad_norm", n, d_grads, counts, dtypes, d_work, work_bytes);
    if (rc != BOA_OK) return rc;
    if (!d_norm) return boa_fail(BOA_ERR_ARG, "boa_grad_norm: null pointer");
    hipStream_t s = (hipStream_t)stream;
    double* part = static_cast<double*>(d_work);
    return with_norm(largest, [&](auto op) {
        using Op = decltype(op);
        int parts;
        if (const int bad = launch_parts<Op>(n, d_grads, counts, dtypes, part, parts, s)) return bad;
        hipLaunchKernelGGL((k_grad_norm<Op>), dim3(1), dim3(WG), 0, s, part, parts, d_norm);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}

extern "C" int boa_clip_grads(int32_t n, void* const* d_grads, const int64_t* counts, const int32_t* dtypes, int largest, double max_norm,
                              float* d_norm, void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_grads("boa_clip_grads", n, d_grads, counts, dtypes, d_work, work_bytes);
    if (rc != BOA_OK) return rc;
    if (!d_norm) return boa_fail(BOA_ERR_ARG, "boa_clip_grads: null pointer");
    if (!(max_norm >= 0.0)) return boa_fail(BOA_ERR_ARG, "boa_clip_grads: max_norm %g", max_norm);
    // no byte twice: it would be scaled by two workgroups at once
    try {
        std::vector<std::pair<uintptr_t, uintptr_t>> at;
        at.reserve((size_t)n);
        for (int32_t i = 0; i < n; ++i)
            if (counts[i] > 0) at.emplace_back((uintptr_t)d_grads[i], (uintptr_t)d_grads[i] + (uintptr_t)(counts[i] * element_bytes(dtypes[i])));
        std::sort(at.begin(), at.end());
        for (size_t i = 1; i < at.size(); ++i)
            if (at[i].first < at[i - 1].second) return boa_fail(BOA_ERR_ARG, "boa_clip_grads: two tensors share memory");
    } catch (const std::exception& e) {
        return boa_fail(BOA_ERR_ARG, "boa_clip_grads: %s", e.what());
    }
    hipStream_t s = (hipStream_t)stream;
    double* part = static_cast<double*>(d_work);
    return with_norm(largest, [&](auto op) {
        using Op = decltype(op);
        int parts;
        if (const int bad = launch_parts<Op>(n, d_grads, counts, dtypes, part, parts, s)) return bad;
        if (parts == 0) {
            hipLaunchKernelGGL((k_grad_norm<Op>), dim3(1), dim3(WG), 0, s, part, 0, d_norm);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        }
        float* norm = d_norm;
        return with_tables(n, d_grads, counts, dtypes, [&](const Table& t, uint32_t blocks) {
            const uint32_t groups = blocks < 4 * MAX_GROUPS ? blocks : 4 * MAX_GROUPS;
            hipLaunchKernelGGL((k_grad_scale<Op>), dim3(groups), dim3(WG), 0, s, t, part, parts, max_norm, norm);
            BOA_HIP_TRY(hipGetLastError());
            norm = nullptr;
            return (int)BOA_OK;
        });
    });
}
