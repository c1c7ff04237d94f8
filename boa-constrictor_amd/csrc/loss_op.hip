// Cross entropy of rows of logits against the symbol that came (boa_cross_entropy_fwd, boa_cross_entropy_bwd).
//
//   loss_r = log sum_j exp(x_rj - m_r) + (m_r - x_rt),  m_r = max_j x_rj,  t = the row's target
//   dx_rj = (exp(x_rj - m_r) / sum_r - [j = t]) * upstream (divided by the number of rows that count, for the mean)
//
// A wavefront holds a row in registers: the forward pass reads the logits once, the backward pass once more (m_r and
// 1 / sum_r are kept, 8 bytes per row) and writes their gradient.  Both are bound by memory, but for the forward pass in 16
// bits, which has 14 vector instructions per logit to its 2 bytes (the vector units are busy for 0.62 of the cycles).  A row
// whose target is ignore_index counts for nothing (its gradient is 0); one whose target is not a symbol gives NaN, in its loss
// and its gradient.
//
// Measured: 262144 rows of 256 bfloat16, forward 39 us (134 MB: 3.4 TB/s, with the gradient of the pass before still on its way to
// memory; 32 alone), backward 42 (268 MB: 6.4 TB/s, the logits in part still in the last cache); float32 49 (5.5 TB/s) and 112
// (4.8).  8000 rows of 256 float32, 4.5 and 5.4, and 2.6 for the sum.
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int WG = 256, WAVES = WG / 64;
constexpr int MAX_V = BOA_CROSS_ENTROPY_MAX_V;
constexpr int MAX_GROUPS = 4096;  // 262144 rows of 256 bfloat16: 39 us, with 2048 42, with 8192 38 and 0.7 more for their sum

// Rows that a wavefront has in flight, for PER elements per lane.
constexpr int rows_at_once(int per) { return per >= 32 ? 1 : 32 / per; }  // 8, 4, 2 or 1

// Row r's symbol, or what its target is instead of one.
constexpr int NOT_A_SYMBOL = -1, IGNORED = -2;
__device__ __forceinline__ int symbol_at(const void* target, int bytes, int64_t ignore, int V, int64_t r) {
    const int64_t t = bytes == 1 ? (int64_t)static_cast<const uint8_t*>(target)[r]
                      : bytes == 4 ? (int64_t)static_cast<const int32_t*>(target)[r] : static_cast<const int64_t*>(target)[r];
    return t == ignore ? IGNORED : t >= 0 && t < V ? (int)t : NOT_A_SYMBOL;
}

template <int DT, int VEC, int N>
struct Row {
    static constexpr int VECTOR = VEC, COUNT = N, PER = N * VEC;
    using T = typename Elem<DT>::T;
    static __device__ __forceinline__ int col(int i, int lane) { return (i * 64 + lane) * VEC; }
    // a row, `other` behind its end; without branches, so that the loads of several rows go out together (V >= VEC)
    static __device__ __forceinline__ void load(const T* row, int V, int lane, float other, float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = col(i, lane);
            float e[VEC];
            ld_vec<DT, VEC>(row + (c < V ? c : V - VEC), e);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i * VEC + j] = c < V ? e[j] : other;
        }
    }
};

template <int DT, int VEC, int N>
__global__ void __launch_bounds__(WG) k_loss_fwd(const void* xp, int64_t xs, const void* target, int target_bytes,
                                                 int64_t ignore, int64_t rows, int V, float2* stats, float* losses,
                                                 double2* part) {
    using R = Row<DT, VEC, N>;
    constexpr int PER = R::PER, ROWS = rows_at_once(PER);
    __shared__ double2 sum[WAVES];
    const auto* x = static_cast<const typename R::T*>(xp);
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int64_t wave = (int64_t)blockIdx.x * WAVES + wid, waves = (int64_t)gridDim.x * WAVES;
    double total = 0.0, count = 0.0;
    for (int64_t r0 = wave * ROWS; r0 < rows; r0 += waves * ROWS) {
        constexpr int EACH = 64 / ROWS;
        const int64_t my_row = r0 + lane / EACH;  // of the ROWS rows the one whose values this lane ends with
        float v[ROWS][PER];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) R::load(x + min(r0 + r, rows - 1) * xs, V, lane, -__builtin_huge_valf(), v[r]);
        const int symbol = symbol_at(target, target_bytes, ignore, V, min(my_row, rows - 1));
        // Over the lanes all the rows go together (reduce): lane l ends with those of row l / EACH, and takes that row's
        // logarithm.  A NaN is dropped by the maximum but not by the exponentials' sum.
        // the target's logit, by the lanes that will need it (the row is on its way to the cache already)
        const float x_t = Elem<DT>::ld(x[min(my_row, rows - 1) * xs + (symbol >= 0 ? symbol : 0)]);
        float m[ROWS], s[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            m[r] = v[r][0];
#pragma unroll
            for (int i = 1; i < PER; ++i) m[r] = fmaxf(m[r], v[r][i]);
        }
        const float mine = reduce<Max, ROWS>(m, lane);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            m[r] = from_lane(mine, r * EACH);
            s[r] = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) s[r] += hw_exp(v[r][i] - m[r]);  // columns behind the last: -inf
        }
        const float total_s = reduce<Add, ROWS>(s, lane);
        float loss = logf(total_s) + (mine - x_t);
        const bool kept = symbol != IGNORED;
        if (symbol == NOT_A_SYMBOL) loss = __builtin_nanf("");
        if (lane % EACH == 0 && my_row < rows) {
            if (kept) {
                total += (double)loss;
                count += 1.0;
            }
            if (stats != nullptr) stats[my_row] = make_float2(mine, 1.0f / total_s);
            if (losses != nullptr) losses[my_row] = kept ? loss : 0.0f;
        }
    }
    if (part == nullptr) return;
    for (int o = 32; o > 0; o >>= 1) {
        total += __shfl_xor(total, o, 64);
        count += __shfl_xor(count, o, 64);
    }
    if (lane == 0) sum[wid] = make_double2(total, count);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < WAVES; ++k) {
            total += sum[k].x;
            count += sum[k].y;
        }
        part[blockIdx.x] = make_double2(total, count);
    }
}

// The workgroups' sums: their loss (over the count for the mean) and the count.
constexpr int SUM_WG = 1024;
__global__ void __launch_bounds__(SUM_WG) k_loss_sum(const double2* part, int n, int mean, float* loss, float* count) {
    __shared__ double2 s[SUM_WG / 64];
    double2 v = make_double2(0.0, 0.0);
    for (int i = threadIdx.x; i < n; i += SUM_WG) {
        v.x += part[i].x;
        v.y += part[i].y;
    }
    for (int o = 32; o > 0; o >>= 1) {
        v.x += __shfl_xor(v.x, o, 64);
        v.y += __shfl_xor(v.y, o, 64);
    }
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < SUM_WG / 64; ++k) {
            v.x += s[k].x;
            v.y += s[k].y;
        }
        *loss = (float)(mean ? v.x / v.y : v.x);
        *count = (float)v.y;
    }
}

template <int DT, int VEC, int N>
__global__ void __launch_bounds__(WG) k_loss_bwd(const void* xp, int64_t xs, const void* target, int target_bytes,
                                                 int64_t ignore, int64_t rows, int V, const float2* stats, const float* up,
                                                 int up_rows, const float* count, void* dxp, int64_t dxs) {
    using R = Row<DT, VEC, N>;
    constexpr int PER = R::PER, ROWS = rows_at_once(PER);
    const auto* x = static_cast<const typename R::T*>(xp);
    auto* dx = static_cast<typename R::T*>(dxp);
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * WAVES;
    const float all = up_rows ? 0.0f : up[0] / (count != nullptr ? *count : 1.0f);
    for (int64_t r0 = wave * ROWS; r0 < rows; r0 += waves * ROWS) {
        constexpr int EACH = 64 / ROWS;
        float v[ROWS][PER];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) R::load(x + min(r0 + r, rows - 1) * xs, V, lane, 0.0f, v[r]);
        const int64_t my_row = min(r0 + lane / EACH, rows - 1);  // a lane reads one row's values for all
        const int my_symbol = symbol_at(target, target_bytes, ignore, V, my_row);
        const float2 my_stats = stats[my_row];
        const float my_scale = my_symbol == NOT_A_SYMBOL ? __builtin_nanf("") : up_rows ? up[my_row] : all;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (r0 + r >= rows) break;
            const int symbol = __builtin_amdgcn_readlane(my_symbol, r * EACH);
            const float m = from_lane(my_stats.x, r * EACH), inv = from_lane(my_stats.y, r * EACH), k = from_lane(my_scale, r * EACH);
            const bool kept = symbol != IGNORED;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float e[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float p = hw_exp(v[r][i * VEC + j] - m) * inv;
                    const float q = R::col(i, lane) + j == symbol ? p - 1.0f : p;
                    e[j] = kept ? q * k : 0.0f;
                }
                if (R::col(i, lane) < V) st_vec<DT, VEC>(dx + (r0 + r) * dxs + R::col(i, lane), e);
            }
        }
    }
}

// Calls f with the row shape for V symbols: accesses of 16 bytes (8 for 16-bit rows of up to 256 symbols, which then take all
// 64 lanes) where the rows are aligned for them, else single elements.
template <int DT, class F>
int with_row(int d, bool aligned, F f) {
    constexpr int W = wide<DT>();
    if (aligned && d % 4 == 0 && d <= 256) return f(Row<DT, 4, 1>());
    if (aligned && d % W == 0) {
        const int n = (int)ceil_div(d, 64 * W);
        if (n <= 1) return f(Row<DT, W, 1>());
        if (n <= 2) return f(Row<DT, W, 2>());
        if (n <= 4) return f(Row<DT, W, 4>());
        return f(Row<DT, W, 64 / W>());
    }
    const int n = (int)ceil_div(d, 64);
    if (n <= 4) return f(Row<DT, 1, 4>());
    if (n <= 16) return f(Row<DT, 1, 16>());
    return f(Row<DT, 1, 64>());
}

int64_t groups_for(int64_t rows, int per) {
    const int64_t n = ceil_div(rows, WAVES * rows_at_once(per));
    return n < MAX_GROUPS ? n : MAX_GROUPS;
}

int check_loss(const char* who, int dtype, int target_bytes, int64_t rows, int32_t V) {
    if (dtype < BOA_DT_F32 || dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, dtype);
    if (target_bytes != 1 && target_bytes != 4 && target_bytes != 8)
        return boa_fail(BOA_ERR_ARG, "%s: targets of %d bytes (1, 4 or 8)", who, target_bytes);
    if (rows < 0 || V < 1 || V > MAX_V)
        return boa_fail(BOA_ERR_ARG, "%s: need rows >= 0 and 1 <= V <= %d (got %lld, %d)", who, MAX_V, (long long)rows, V);
    return BOA_OK;
}

}  // namespace

extern "C" int64_t boa_cross_entropy_work_bytes(void) { return MAX_GROUPS * (int64_t)sizeof(double2); }

extern "C" int boa_cross_entropy_fwd(int dtype, const void* d_x, int64_t x_stride, const void* d_targets, int target_bytes,
                                     int64_t ignore_index, int64_t rows, int32_t V, int mean, float* d_stats, float* d_losses,
                                     float* d_loss, float* d_count, void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_loss("boa_cross_entropy_fwd", dtype, target_bytes, rows, V);
    if (rc != BOA_OK) return rc;
    if (rows > 0 && (!d_x || !d_targets)) return boa_fail(BOA_ERR_ARG, "boa_cross_entropy_fwd: null pointer");
    if (!d_loss != !d_count) return boa_fail(BOA_ERR_ARG, "boa_cross_entropy_fwd: loss and count go together");
    if (d_loss && (!d_work || work_bytes < boa_cross_entropy_work_bytes()))
        return boa_fail(BOA_ERR_ARG, "boa_cross_entropy_fwd: workspace of %lld bytes, needs %lld", (long long)work_bytes,
                        (long long)boa_cross_entropy_work_bytes());
    hipStream_t s = (hipStream_t)stream;
    double2* part = d_loss ? static_cast<double2*>(d_work) : nullptr;
    int64_t groups = 0;
    if (rows > 0) {
        const int launched = with_dtype(dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            return with_row<DT>(V, aligned16(dtype, d_x, x_stride), [&](auto row) {
                using R = decltype(row);
                groups = groups_for(rows, R::PER);
                hipLaunchKernelGGL((k_loss_fwd<DT, R::VECTOR, R::COUNT>), dim3((uint32_t)groups), dim3(WG), 0, s, d_x, x_stride,
                                   d_targets, target_bytes, ignore_index, rows, V, reinterpret_cast<float2*>(d_stats), d_losses,
                                   part);
                BOA_HIP_TRY(hipGetLastError());
                return (int)BOA_OK;
            });
        });
        if (launched != BOA_OK) return launched;
    }
    if (d_loss) {
        hipLaunchKernelGGL(k_loss_sum, dim3(1), dim3(SUM_WG), 0, s, part, (int)groups, mean, d_loss, d_count);
        BOA_HIP_TRY(hipGetLastError());
    }
    return BOA_OK;
}

extern "C" int boa_cross_entropy_bwd(int dtype, const void* d_x, int64_t x_stride, const void* d_targets, int target_bytes,
                                     int64_t ignore_index, int64_t rows, int32_t V, const float* d_stats, const float* d_up,
                                     int up_rows, const float* d_count, void* d_dx, int64_t dx_stride, void* stream) {
    const int rc = check_loss("boa_cross_entropy_bwd", dtype, target_bytes, rows, V);
    if (rc != BOA_OK) return rc;
    if (rows == 0) return BOA_OK;
    if (!d_x || !d_targets || !d_stats || !d_up || !d_dx) return boa_fail(BOA_ERR_ARG, "boa_cross_entropy_bwd: null pointer");
    return with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return with_row<DT>(V, aligned16(dtype, d_x, x_stride) && aligned16(dtype, d_dx, dx_stride), [&](auto row) {
            using R = decltype(row);
            const int64_t groups = ceil_div(rows, WAVES * rows_at_once(R::PER));
            hipLaunchKernelGGL((k_loss_bwd<DT, R::VECTOR, R::COUNT>), dim3((uint32_t)(groups < 4096 ? groups : 4096)), dim3(WG), 0,
                               (hipStream_t)stream, d_x, x_stride, d_targets, target_bytes, ignore_index, rows, V,
                               reinterpret_cast<const float2*>(d_stats), d_up, up_rows, d_count, d_dx, dx_stride);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
    });
}
