// Layer norm over the rows of a matrix with its gradient (boa_layer_norm_fwd, boa_layer_norm_bwd), and the sum of partial
// rows that the operators' parameter gradients end in.
//
//   mean = sum x / d, rstd = 1 / sqrt(sum (x - mean)^2 / d + eps), xh = (x - mean) rstd, y = xh w + b
//   dx = rstd (g - mean(g) - xh mean(g xh)) with g = dy w;  dw = sum_rows dy xh, db = sum_rows dy
//
// Both passes are bound by memory.  A wavefront (a workgroup for rows of more than 1024 values) holds a row in registers, so a
// row is read once per pass, and takes several of them at a time to have enough loads in flight.  In the backward pass a
// wavefront adds its rows' dy xh and dy in registers, a workgroup its wavefronts' through LDS, and k_sum_parts the workgroups':
// no atomics, so the same inputs give the same bits.
//
// Measured: 262144 rows of 512 bfloat16, forward 99 us (5.4 TB/s), backward 155 and 5 for the parameters' sums (5.0 TB/s; a copy of
// 1 GiB runs at 5.0); 8000 rows of 256 float32, 5 and 10 us.
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int WG = 256, WAVES = WG / 64;
constexpr int MAX_D = BOA_LAYER_NORM_MAX_D;
// Rows up to here are a wavefront's, wider ones a workgroup's.  As a wavefront's, forward and backward, 32768 rows of 2048 float32 take
// 97 and 160 us (as a workgroup's 99 and 161), 16384 of 4096 106 and 316 (97 and 155).
constexpr int WAVE_D = 1024;
static_assert(MAX_D <= 16 * WG, "16 values per thread");

// Rows that a wavefront takes at a time, for PER elements per lane: 16 values in flight per lane.
constexpr int rows_at_once(int per) { return per >= 16 ? 1 : 16 / per; }

// A row over LANES threads (a wavefront, or the workgroup), N accesses of VEC elements each.
template <int DT, int VEC, int N, int LANES_>
struct Row {
    static constexpr int VECTOR = VEC, COUNT = N, PER = N * VEC, LANES = LANES_, TEAMS = WG / LANES;
    using T = typename Elem<DT>::T;
    static __device__ __forceinline__ int col(int i, int lane) { return (i * LANES + lane) * VEC; }
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
    // a float32 parameter row in the same places (16-byte aligned, if the accesses are of several elements); `other` beyond d and
    // where there is none
    static __device__ __forceinline__ void param(const float* p, int d, int lane, float other, float (&v)[PER]) {
        constexpr int PART = VEC == 1 ? 1 : 4;
#pragma unroll
        for (int i = 0; i < PER; i += PART) {
            const int c = col(i / VEC, lane) + i % VEC;
            float t[PART];
            if (p != nullptr && c < d) ld_vec<DT_F32, PART>(p + c, t);
#pragma unroll
            for (int j = 0; j < PART; ++j) v[i + j] = (p != nullptr && c < d) ? t[j] : other;
        }
    }
    // float32 values into such places of a row that begins anywhere
    static __device__ __forceinline__ void put(float* p, int d, int lane, const float (&v)[PER]) {
        constexpr int PART = VEC == 1 ? 1 : 4;
        typedef float Part __attribute__((ext_vector_type(PART), aligned(4)));
#pragma unroll
        for (int i = 0; i < PER; i += PART) {
            const int c = col(i / VEC, lane) + i % VEC;
            Part t;
#pragma unroll
            for (int j = 0; j < PART; ++j) t[j] = v[i + j];
            if (c < d) *reinterpret_cast<Part*>(p + c) = t;
        }
    }
    // K sums over the row's threads
    template <int K>
    static __device__ __forceinline__ void sums(float (&v)[K]) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wsum(v[k]);
        if constexpr (LANES == WG) {
            __shared__ float s[K][WAVES];
            __syncthreads();  // what was here has been read
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int k = 0; k < K; ++k) s[k][threadIdx.x >> 6] = v[k];
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                v[k] = s[k][0];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) v[k] += s[k][w];
            }
        }
    }
};

// And in the backward pass, which reads two arrays and has more registers in use: two rows where one is an access of 8 bytes per
// lane (262144 rows of 256 bfloat16 87 us, 94 one at a time), else one (2 or 4 rows: float32 of 256 and 512 bfloat16 the same, 2048
// bfloat16 99, 103 and 182).
template <class R>
constexpr int bwd_rows_at_once() {
    return R::VECTOR == 4 && R::PER == 4 && sizeof(typename R::T) == 2 ? 2 : 1;
}

template <class R, int DT>
__global__ void __launch_bounds__(WG) k_norm_fwd(const void* xp, int64_t xs, const float* w, const float* b, int64_t rows,
                                                 int d, float eps, void* yp, int64_t ys, float2* stats) {
    constexpr int PER = R::PER, ROWS = rows_at_once(PER), VEC = R::VECTOR;
    const auto* x = static_cast<const typename R::T*>(xp);
    auto* y = static_cast<typename R::T*>(yp);
    const int lane = threadIdx.x % R::LANES;
    const int64_t team = (int64_t)blockIdx.x * R::TEAMS + threadIdx.x / R::LANES, teams = (int64_t)gridDim.x * R::TEAMS;
    float wv[PER], bv[PER];
    R::param(w, d, lane, 1.0f, wv);
    R::param(b, d, lane, 0.0f, bv);
    const float inv = 1.0f / (float)d;
    for (int64_t r0 = team * ROWS; r0 < rows; r0 += teams * ROWS) {
        float v[ROWS][PER];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) R::load(x + min(r0 + r, rows - 1) * xs, d, lane, v[r]);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float s[1] = {0.0f}, q[1] = {0.0f};
#pragma unroll
            for (int i = 0; i < PER; ++i) s[0] += v[r][i];
            R::sums(s);
            const float mean = s[0] * inv;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                // beyond d the difference is not one of the row's
                const float c = R::col(i / VEC, lane) < d ? v[r][i] - mean : 0.0f;
                v[r][i] = c;
                q[0] = __builtin_fmaf(c, c, q[0]);
            }
            R::sums(q);
            const float rstd = 1.0f / sqrtf(q[0] * inv + eps);
#pragma unroll
            for (int i = 0; i < PER; ++i) v[r][i] = __builtin_fmaf(v[r][i] * rstd, wv[i], bv[i]);
            if (r0 + r < rows) {
                R::store(y + (r0 + r) * ys, d, lane, v[r]);
                if (stats != nullptr && lane == 0) stats[r0 + r] = make_float2(mean, rstd);
            }
        }
    }
}

template <class R, int DT>
__global__ void __launch_bounds__(WG) k_norm_bwd(const void* dyp, int64_t dys, const void* xp, int64_t xs, const float* w,
                                                 const float2* stats, int64_t rows, int d, void* dxp, int64_t dxs,
                                                 float* part) {
    constexpr int PER = R::PER, ROWS = bwd_rows_at_once<R>(), VEC = R::VECTOR;
    const auto* x = static_cast<const typename R::T*>(xp);
    const auto* dy = static_cast<const typename R::T*>(dyp);
    auto* dx = static_cast<typename R::T*>(dxp);
    const int lane = threadIdx.x % R::LANES, mine = threadIdx.x / R::LANES;
    const int64_t team = (int64_t)blockIdx.x * R::TEAMS + mine, teams = (int64_t)gridDim.x * R::TEAMS;
    float wv[PER], dw[PER] = {}, db[PER] = {};
    R::param(w, d, lane, 1.0f, wv);
    const float inv = 1.0f / (float)d;
    for (int64_t r0 = team * ROWS; r0 < rows; r0 += teams * ROWS) {
        float v[ROWS][PER], g[ROWS][PER];
        float2 st[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t at = min(r0 + r, rows - 1);
            R::load(x + at * xs, d, lane, v[r]);
            R::load(dy + at * dys, d, lane, g[r]);
            st[r] = stats[at];
        }
        float m[2 * ROWS];  // sums of g, and of g xh
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const bool once = r0 + r < rows;  // the last row is read again behind the end
            m[2 * r] = m[2 * r + 1] = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float xh = (v[r][i] - st[r].x) * st[r].y;  // beyond d: dy is 0 there
                const float gd = once ? g[r][i] : 0.0f;
                dw[i] = __builtin_fmaf(gd, xh, dw[i]);
                db[i] += gd;
                const float gw = gd * wv[i];
                m[2 * r] += gw;
                m[2 * r + 1] = __builtin_fmaf(gw, xh, m[2 * r + 1]);
                v[r][i] = xh;
                g[r][i] = gw;
            }
        }
        R::sums(m);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
#pragma unroll
            for (int i = 0; i < PER; ++i) v[r][i] = (g[r][i] - m[2 * r] * inv - v[r][i] * (m[2 * r + 1] * inv)) * st[r].y;
            if (r0 + r < rows) R::store(dx + (r0 + r) * dxs, d, lane, v[r]);
        }
    }
    if (part == nullptr) return;
    float* out = part + (int64_t)blockIdx.x * 2 * d;
    if constexpr (R::TEAMS == 1) {
        R::put(out, d, lane, dw);
        R::put(out + d, d, lane, db);
    } else {
        __shared__ float sum[2][R::LANES * PER];
        for (int k = 0; k < R::TEAMS; ++k) {
            if (mine == k) {
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int c = R::col(i / VEC, lane) + i % VEC;
                    sum[0][c] = (k ? sum[0][c] : 0.0f) + dw[i];
                    sum[1][c] = (k ? sum[1][c] : 0.0f) + db[i];
                }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < d; c += WG) {
            out[c] = sum[0][c];
            out[d + c] = sum[1][c];
        }
    }
}

constexpr int SUM_GROUPS = 32;
__global__ void __launch_bounds__(SUM_COLS * SUM_GROUPS) k_sum_parts(const float* part, int64_t parts, int64_t width, float* out) {
    sum_parts<SUM_GROUPS>(part, parts, width, out, blockIdx.x);
}

// Workgroups of the backward pass, each of which leaves a partial row of 2 d sums: 4 rows or more per team (1000 rows of 4096
// float32 16 us, with a row per workgroup 20), and no more than run at once; of rows of more than 2048 values half of that, for the
// partial rows' sake (16384 rows of 4096: float32 167 -> 154 us, bfloat16 103 -> 87; of 2048 bfloat16 it would be 90 -> 99).
int64_t bwd_groups(int64_t rows, int d) {
    const int64_t n = ceil_div(rows, d <= WAVE_D ? 4 * WAVES : 4), most = d <= MAX_D / 2 ? 1024 : 512;
    return n < most ? n : most;
}

// Calls f with the row shape for width d: accesses of 16 bytes (8 for 16-bit rows of up to 256 values, which then take all 64
// lanes) where rows and parameters are aligned for them, else single elements; up to 16 values per lane.  Backward and forward,
// 16 bytes and single elements: 174762 rows of 384 bfloat16 129 and 148 us, 131072 of 512 float32 244 and 255.
template <int DT, class F>
int with_row(int d, bool aligned, F f) {
    constexpr int W = wide<DT>();
    if (aligned && d % 4 == 0 && d <= 256) return f(Row<DT, 4, 1, 64>());
    if (aligned && d % W == 0) {
        const bool wave = d <= WAVE_D;
        const int64_t n = ceil_div(d, (wave ? 64 : WG) * W);
        if (n <= 1) return wave ? f(Row<DT, W, 1, 64>()) : f(Row<DT, W, 1, WG>());
        if (n <= 2) return wave ? f(Row<DT, W, 2, 64>()) : f(Row<DT, W, 2, WG>());
        if constexpr (W == 4) {
            if (n <= 3) return wave ? f(Row<DT, W, 3, 64>()) : f(Row<DT, W, 3, WG>());
            return wave ? f(Row<DT, W, 4, 64>()) : f(Row<DT, W, 4, WG>());
        }
    }
    if (d <= 256) return f(Row<DT, 1, 4, 64>());
    if (d <= 512) return f(Row<DT, 1, 8, 64>());
    if (d <= WAVE_D) return f(Row<DT, 1, 16, 64>());
    if (d <= 8 * WG) return f(Row<DT, 1, 8, WG>());
    return f(Row<DT, 1, 16, WG>());
}
bool params_aligned(const float* w, const float* b) { return ((uintptr_t)w | (uintptr_t)b) % 16 == 0; }
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
    const bool al = aligned16(dtype, d_x, x_stride) && aligned16(dtype, d_y, y_stride) && params_aligned(d_w, d_b);
    return with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return with_row<DT>(d, al, [&](auto row) {
            using R = decltype(row);
            const int64_t groups = ceil_div(rows, R::TEAMS * rows_at_once(R::PER));
            hipLaunchKernelGGL((k_norm_fwd<R, DT>), dim3((uint32_t)(groups < 4096 ? groups : 4096)), dim3(WG), 0,
                               (hipStream_t)stream, d_x, x_stride, d_w, d_b, rows, d, eps, d_y, y_stride,
                               reinterpret_cast<float2*>(d_stats));
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
    });
}

extern "C" int64_t boa_layer_norm_bwd_work_bytes(int64_t rows, int32_t d) {
    return rows < 1 || d < 1 ? 0 : bwd_groups(rows, d) * 2 * d * (int64_t)sizeof(float);
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
    const int64_t groups = rows > 0 ? bwd_groups(rows, d) : 0;
    if (rows > 0) {
        const bool al = aligned16(dtype, d_x, x_stride) && aligned16(dtype, d_dy, dy_stride) && aligned16(dtype, d_dx, dx_stride) &&
                        params_aligned(d_w, nullptr);
        const int launched = with_dtype(dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            return with_row<DT>(d, al, [&](auto row) {
                using R = decltype(row);
                hipLaunchKernelGGL((k_norm_bwd<R, DT>), dim3((uint32_t)groups), dim3(WG), 0, s, d_dy, dy_stride,
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
