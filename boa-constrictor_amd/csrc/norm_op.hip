// Layer norm over the rows of a matrix with its gradient (boa_layer_norm_fwd, boa_layer_norm_bwd), and the sum of partial
// rows that the operators' parameter gradients end in.
//
//   mean = sum x / d, rstd = 1 / sqrt(sum (x - mean)^2 / d + eps), xh = (x - mean) rstd, y = xh w + b
//   dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w;  dw = sum_rows dy xh, db = sum_rows dy
//
// Both passes are bound by memory.  A wavefront holds a row in registers, so a row is read once per pass, and takes ROWS of
// them at a time to have enough loads in flight.  In the backward pass a wavefront adds its rows' dy xh and dy in registers,
// a workgroup its wavefronts' through LDS, and k_sum_parts the workgroups': no atomics, so the same inputs give the same bits.
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int WG = 256, WAVES = WG / 64;
constexpr int MAX_D = BOA_LAYER_NORM_MAX_D;

// Rows that a wavefront takes at a time, for PER elements per lane: 16 values in flight per lane.
constexpr int rows_at_once(int per) { return per >= 16 ? 1 : 16 / per; }

template <int DT, int VEC, int N>
struct Row {
    static constexpr int VECTOR = VEC, COUNT = N, PER = N * VEC;
    using T = typename Elem<DT>::T;
    static __device__ __forceinline__ int col(int i, int lane) { return (i * 64 + lane) * VEC; }
    // elements beyond d read as 0 (d is a multiple of VEC, so a vector is inside or outside as a whole); without branches, so
    // that the loads of several rows go out together
    static __device__ __forceinline__ void load(const T* row, int d, int lane, float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = col(i, lane);
            float t[VEC];
            ld_vec<DT, VEC>(row + (c < d ? c : d - VEC), t);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i * VEC + j] = c < d ? t[j] : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(T* row, int d, int lane, const float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) t[j] = v[i * VEC + j];
            if (col(i, lane) < d) st_vec<DT, VEC>(row + col(i, lane), t);
        }
    }
    // a float32 parameter row in the same places; `other` beyond d and where there is none
    static __device__ __forceinline__ void param(const float* p, int d, int lane, float other, float (&v)[PER]) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int c = col(i, lane) + j;
                v[i * VEC + j] = (p != nullptr && c < d) ? p[c] : other;
            }
    }
};

template <int DT, int VEC, int N>
__global__ void __launch_bounds__(WG) k_norm_fwd(const void* xp, int64_t xs, const float* w, const float* b, int64_t rows,
                                                 int d, float eps, void* yp, int64_t ys, float2* stats) {
    using R = Row<DT, VEC, N>;
    constexpr int PER = R::PER, ROWS = rows_at_once(PER);
    const auto* x = static_cast<const typename R::T*>(xp);
    auto* y = static_cast<typename R::T*>(yp);
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * WAVES;
    float wv[PER], bv[PER];
    R::param(w, d, lane, 1.0f, wv);
    R::param(b, d, lane, 0.0f, bv);
    const float inv = 1.0f / (float)d;
    for (int64_t r0 = wave * ROWS; r0 < rows; r0 += waves * ROWS) {
        float v[ROWS][PER];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t at = r0 + r < rows ? r0 + r : rows - 1;
            R::load(x + at * xs, d, lane, v[r]);
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) s += v[r][i];
            const float mean = wsum(s) * inv;
            float q = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                // beyond d the difference is not one of the row's
                const float c = R::col(i / VEC, lane) < d ? v[r][i] - mean : 0.0f;
                v[r][i] = c;
                q = __builtin_fmaf(c, c, q);
            }
            const float rstd = 1.0f / sqrtf(wsum(q) * inv + eps);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[r][i] = __builtin_fmaf(v[r][i] * rstd, wv[i], bv[i]);
            if (r0 + r < rows) {
                R::store(y + (r0 + r) * ys, d, lane, v[r]);
                if (stats != nullptr && lane == 0) stats[r0 + r] = make_float2(mean, rstd);
            }
        }
    }
}

template <int DT, int VEC, int N>
__global__ void __launch_bounds__(WG) k_norm_bwd(const void* dyp, int64_t dys, const void* xp, int64_t xs, const float* w,
                                                 const float2* stats, int64_t rows, int d, void* dxp, int64_t dxs,
                                                 float* part) {
    using R = Row<DT, VEC, N>;
    constexpr int PER = R::PER, ROWS = rows_at_once(2 * PER);
    __shared__ float sum[2][64 * PER];
    const auto* x = static_cast<const typename R::T*>(xp);
    const auto* dy = static_cast<const typename R::T*>(dyp);
    auto* dx = static_cast<typename R::T*>(dxp);
    const int lane = threadIdx.x & 63, wv_id = threadIdx.x >> 6;
    const int64_t wave = (int64_t)blockIdx.x * WAVES + wv_id, waves = (int64_t)gridDim.x * WAVES;
    float wv[PER], dw[PER] = {}, db[PER] = {};
    R::param(w, d, lane, 1.0f, wv);
    const float inv = 1.0f / (float)d;
    for (int64_t r0 = wave * ROWS; r0 < rows; r0 += waves * ROWS) {
        float v[ROWS][PER], g[ROWS][PER];
        float2 st[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t at = r0 + r < rows ? r0 + r : rows - 1;
            R::load(x + at * xs, d, lane, v[r]);
            R::load(dy + at * dys, d, lane, g[r]);
            st[r] = stats[at];
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (r0 + r >= rows) break;
            float m1 = 0.0f, m2 = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float xh = (v[r][i] - st[r].x) * st[r].y;  // beyond d: dy is 0 there
                dw[i] = __builtin_fmaf(g[r][i], xh, dw[i]);
                db[i] += g[r][i];
                const float gw = g[r][i] * wv[i];
                m1 += gw;
                m2 = __builtin_fmaf(gw, xh, m2);
                v[r][i] = xh;
                g[r][i] = gw;
            }
            m1 = wsum(m1) * inv;
            m2 = wsum(m2) * inv;
#pragma unroll
            for (int i = 0; i < PER; ++i) v[r][i] = (g[r][i] - m1 - v[r][i] * m2) * st[r].y;
            R::store(dx + (r0 + r) * dxs, d, lane, v[r]);
        }
    }
    if (part == nullptr) return;
    for (int k = 0; k < WAVES; ++k) {
        if (wv_id == k) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = R::col(i / VEC, lane) + i % VEC;
                sum[0][c] = (k ? sum[0][c] : 0.0f) + dw[i];
                sum[1][c] = (k ? sum[1][c] : 0.0f) + db[i];
            }
        }
        __syncthreads();
    }
    float* mine = part + (int64_t)blockIdx.x * 2 * d;
    for (int c = threadIdx.x; c < d; c += WG) {
        mine[c] = sum[0][c];
        mine[d + c] = sum[1][c];
    }
}

constexpr int SUM_GROUPS = 32;
__global__ void __launch_bounds__(SUM_COLS * SUM_GROUPS) k_sum_parts(const float* part, int64_t parts, int64_t width, float* out) {
    sum_parts<SUM_GROUPS>(part, parts, width, out, blockIdx.x);
}

int64_t fwd_groups(int64_t rows, int per) { return ceil_div(rows, WAVES * rows_at_once(per)); }
// Workgroups of the backward pass, each of which leaves a partial row of 2 d sums: four rows or more per wavefront.
int64_t bwd_groups(int64_t rows) {
    const int64_t n = ceil_div(rows, 4 * WAVES);
    return n < 1024 ? n : 1024;
}

// Calls f with the row shape for width d: accesses of 16 bytes (8 for 16-bit rows of up to 256 values, which then take all 64
// lanes) where the rows are aligned for them, else single elements.
template <int DT, class F>
int with_row(int d, bool aligned, F f) {
    constexpr int W = wide<DT>();
    if (aligned && d % 4 == 0 && d <= 256) return f(Row<DT, 4, 1>());
    if (aligned && d % W == 0) {
        const int n = (int)ceil_div(d, 64 * W);
        if (n <= 1) return f(Row<DT, W, 1>());
        if (n <= 2) return f(Row<DT, W, 2>());
        if (n <= 4) return f(Row<DT, W, 4>());
        if (W * n <= 32) return f(Row<DT, W, 32 / W>());
        return f(Row<DT, W, 64 / W>());
    }
    const int n = (int)ceil_div(d, 64);
    if (n <= 4) return f(Row<DT, 1, 4>());
    if (n <= 8) return f(Row<DT, 1, 8>());
    if (n <= 16) return f(Row<DT, 1, 16>());
    if (n <= 32) return f(Row<DT, 1, 32>());
    return f(Row<DT, 1, 64>());
}
int check_norm(const char* who, int dtype, int64_t rows, int32_t d) {
    if (dtype < BOA_DT_F32 || dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, dtype);
    if (rows < 0 || d < 1 || d > MAX_D)
        return boa_fail(BOA_ERR_ARG, "%s: need rows >= 0 and 1 <= d <= %d (got %lld, %d)", who, MAX_D, (long long)rows, d);
    return BOA_OK;
}

}  // namespace

namespace boa {
hipError_t launch_sum_parts(const float* part, int64_t parts, int64_t width, float* out, hipStream_t s) {
    hipLaunchKernelGGL(k_sum_parts, dim3((uint32_t)ceil_div(width, SUM_COLS)), dim3(SUM_COLS * SUM_GROUPS), 0, s, part, parts,
                       width, out);
    return hipGetLastError();
}
}  // namespace boa

extern "C" int boa_layer_norm_fwd(int dtype, const void* d_x, int64_t x_stride, const float* d_w, const float* d_b,
                                  int64_t rows, int32_t d, float eps, void* d_y, int64_t y_stride, float* d_stats,
                                  void* stream) {
    const int rc = check_norm("boa_layer_norm_fwd", dtype, rows, d);
    if (rc != BOA_OK) return rc;
    if (rows == 0) return BOA_OK;
    if (!d_x || !d_y) return boa_fail(BOA_ERR_ARG, "boa_layer_norm_fwd: null pointer");
    const bool al = aligned16(dtype, d_x, x_stride) && aligned16(dtype, d_y, y_stride);
    return with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return with_row<DT>(d, al, [&](auto row) {
            using R = decltype(row);
            const int64_t groups = fwd_groups(rows, R::PER);
            hipLaunchKernelGGL((k_norm_fwd<DT, R::VECTOR, R::COUNT>), dim3((uint32_t)(groups < 4096 ? groups : 4096)), dim3(WG), 0,
                               (hipStream_t)stream, d_x, x_stride, d_w, d_b, rows, d, eps, d_y, y_stride,
                               reinterpret_cast<float2*>(d_stats));
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
    });
}

extern "C" int64_t boa_layer_norm_bwd_work_bytes(int64_t rows, int32_t d) {
    return rows < 1 || d < 1 ? 0 : bwd_groups(rows) * 2 * d * (int64_t)sizeof(float);
}

extern "C" int boa_layer_norm_bwd(int dtype, const void* d_dy, int64_t dy_stride, const void* d_x, int64_t x_stride,
                                  const float* d_w, const float* d_stats, int64_t rows, int32_t d, void* d_dx,
                                  int64_t dx_stride, float* d_dwb, void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_norm("boa_layer_norm_bwd", dtype, rows, d);
    if (rc != BOA_OK) return rc;
    if (d_dwb && work_bytes < boa_layer_norm_bwd_work_bytes(rows, d))
        return boa_fail(BOA_ERR_ARG, "boa_layer_norm_bwd: workspace of %lld bytes, needs %lld", (long long)work_bytes,
                        (long long)boa_layer_norm_bwd_work_bytes(rows, d));
    if (rows > 0 && (!d_dy || !d_x || !d_stats || !d_dx || (d_dwb && !d_work)))
        return boa_fail(BOA_ERR_ARG, "boa_layer_norm_bwd: null pointer");
    hipStream_t s = (hipStream_t)stream;
    float* part = d_dwb ? static_cast<float*>(d_work) : nullptr;
    const int64_t groups = rows > 0 ? bwd_groups(rows) : 0;
    if (rows > 0) {
        const bool al = aligned16(dtype, d_x, x_stride) && aligned16(dtype, d_dy, dy_stride) && aligned16(dtype, d_dx, dx_stride);
        const int launched = with_dtype(dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            return with_row<DT>(d, al, [&](auto row) {
                using R = decltype(row);
                hipLaunchKernelGGL((k_norm_bwd<DT, R::VECTOR, R::COUNT>), dim3((uint32_t)groups), dim3(WG), 0, s, d_dy, dy_stride,
                                   d_x, x_stride, d_w, reinterpret_cast<const float2*>(d_stats), rows, d, d_dx, dx_stride, part);
                BOA_HIP_TRY(hipGetLastError());
                return (int)BOA_OK;
            });
        });
        if (launched != BOA_OK) return launched;
    }
    if (d_dwb) BOA_HIP_TRY(launch_sum_parts(part, groups, 2 * (int64_t)d, d_dwb, s));
    return BOA_OK;
}
