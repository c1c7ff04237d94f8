// Short causal convolution of every channel over the positions, with SiLU, and its gradient (boa_causal_conv_fwd,
// boa_causal_conv_bwd, boa_causal_conv_step).
//
//   p_t = b + w_0 x_(t-3) + w_1 x_(t-2) + w_2 x_(t-1) + w_3 x_t,  y = p sigmoid(p)
//   gp = dy (sig + p sig (1 - sig));  dx_t = w_3 gp_t + w_2 gp_(t+1) + w_1 gp_(t+2) + w_0 gp_(t+3)
//   dw_k = sum_(batch, t) gp_t x_(t-3+k);  db = sum gp
//
// Bound by memory.  A thread walks a run of positions of its channels with the window in registers, so a value is read once
// per run (and three times more at the runs' borders, from cache).  The backward pass computes p again instead of
// reading it.  Positions before the first come from the state (zeros without one); positions from a sequence's length on are
// not read and are written as zeros.
//
// Measured: 64 x 1500 positions of 512 channels, float32: forward 75 us (393 MB: 5.2 TB/s), backward 130 (590 MB: 4.5; with dy and x
// in part still in the last cache 53 and 91); bfloat16 36 and 77.  One position of 64 x 512, 3 us.
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int TAPS = 4, PAST = TAPS - 1;
constexpr int LANES = 64, RUNS = 4, WG = LANES * RUNS;  // a wavefront: 64 channel vectors of one run
// Positions of a run: of 8, 16 and 32 the case above takes 72, 75 and 83 us forward and 130, 130 and 131 backward, in bfloat16
// 35, 36 and 44, and 87, 77 and 71; a single sequence of 1000 positions 6, 6 and 10, and 11, 12 and 19.
constexpr int RUN = 16;
constexpr int MAX_GROUPS = 1024;                        // workgroups along the runs

struct ConvArgs {
    const void *x, *dy;
    int64_t xb, xr, dyb, dyr;      // element strides of a batch and of a row
    const float *w, *b;            // [C][4], [C] or null
    const void* state_in;          // [batch][3][C] or null
    void* state_out;               // the same, or null
    void *y, *dx;
    int64_t yb, yr, dxb, dxr;
    const int32_t* lens;
    float* part;
    int C, silu;
    int64_t batch, length, runs;   // runs: of one sequence
};

template <int VEC>
__device__ __forceinline__ void load_weights(const ConvArgs& a, int c, float (&w)[TAPS][VEC], float (&bias)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
        for (int k = 0; k < TAPS; ++k) w[k][j] = a.w[(int64_t)(c + j) * TAPS + k];
        bias[j] = a.b != nullptr ? a.b[c + j] : 0.0f;
    }
}

// Row t (>= -3) of [state | x]: zeros before the start without a state and from `end` on.
template <int DT, int VEC>
__device__ __forceinline__ typename Raw<DT, VEC>::V row_at(const ConvArgs& a, int64_t b, int64_t t, int64_t end, int c) {
    using T = typename Elem<DT>::T;
    typename Raw<DT, VEC>::V r = {};
    if (t >= 0) {
        if (t < end) r = Raw<DT, VEC>::load(static_cast<const T*>(a.x) + b * a.xb + t * a.xr + c);
    } else if (a.state_in != nullptr) {
        r = Raw<DT, VEC>::load(static_cast<const T*>(a.state_in) + (b * PAST + t + PAST) * (int64_t)a.C + c);
    }
    return r;
}

__device__ __forceinline__ int64_t end_of(const ConvArgs& a, int64_t b) {
    if (a.lens == nullptr) return a.length;
    const int64_t n = a.lens[b];
    return n < 0 ? 0 : (n < a.length ? n : a.length);
}

template <int DT, int VEC>
__global__ void __launch_bounds__(WG) k_conv_fwd(const ConvArgs a) {
    using T = typename Elem<DT>::T;
    using W = Raw<DT, VEC>;
    const int c = (blockIdx.x * LANES + threadIdx.x) * VEC;
    if (c >= a.C) return;
    float w[TAPS][VEC], bias[VEC];
    load_weights<VEC>(a, c, w, bias);
    for (int64_t k = (int64_t)blockIdx.y * RUNS + threadIdx.y; k < a.batch * a.runs; k += (int64_t)gridDim.y * RUNS) {
        const int64_t b = k / a.runs, t0 = (k % a.runs) * RUN, end = end_of(a, b);
        typename W::V in[RUN + PAST];
#pragma unroll
        for (int i = 0; i < RUN + PAST; ++i) in[i] = row_at<DT, VEC>(a, b, t0 + i - PAST, end, c);
        float win[TAPS][VEC];
#pragma unroll
        for (int i = 0; i < PAST; ++i) W::unpack(in[i], win[i]);
#pragma unroll
        for (int i = 0; i < RUN; ++i) {
            const int64_t t = t0 + i;
            if (t >= a.length) break;
            W::unpack(in[i + PAST], win[PAST]);
            float out[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float p = bias[j];
#pragma unroll
                for (int q = 0; q < TAPS; ++q) p = __builtin_fmaf(w[q][j], win[q][j], p);
                out[j] = t < end ? (a.silu ? hw_silu(p) : p) : 0.0f;
#pragma unroll
                for (int q = 0; q < PAST; ++q) win[q][j] = win[q + 1][j];
            }
            st_vec<DT, VEC>(static_cast<T*>(a.y) + b * a.yb + t * a.yr + c, out);
        }
        if (a.state_out != nullptr && t0 == 0) {
#pragma unroll
            for (int i = 0; i < PAST; ++i) {
                const typename W::V r = row_at<DT, VEC>(a, b, end - PAST + i, end, c);
                *reinterpret_cast<typename W::V*>(static_cast<T*>(a.state_out) + (b * PAST + i) * (int64_t)a.C + c) = r;
            }
        }
    }
}

template <int DT, int VEC>
__global__ void __launch_bounds__(WG) k_conv_bwd(const ConvArgs a) {
    using T = typename Elem<DT>::T;
    using W = Raw<DT, VEC>;
    __shared__ float sum[RUNS][LANES * VEC * (TAPS + 1)];
    const int c = (blockIdx.x * LANES + threadIdx.x) * VEC;
    float w[TAPS][VEC] = {}, bias[VEC] = {}, dw[TAPS][VEC] = {}, db[VEC] = {};
    if (c < a.C) {
        load_weights<VEC>(a, c, w, bias);
        for (int64_t k = (int64_t)blockIdx.y * RUNS + threadIdx.y; k < a.batch * a.runs; k += (int64_t)gridDim.y * RUNS) {
            const int64_t b = k / a.runs, t0 = (k % a.runs) * RUN, end = end_of(a, b);
            float win[TAPS][VEC], g[TAPS][VEC] = {};
#pragma unroll
            for (int i = 0; i < PAST; ++i) W::unpack(row_at<DT, VEC>(a, b, t0 + i - PAST, end, c), win[i]);
            constexpr int AT_ONCE = 4;  // rows in flight
            for (int i0 = 0; i0 < RUN + PAST; i0 += AT_ONCE) {
                typename W::V in[AT_ONCE], din[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int64_t t = t0 + i0 + i;
                    in[i] = row_at<DT, VEC>(a, b, t, end, c);
                    din[i] = typename W::V{};
                    if (t < end) din[i] = W::load(static_cast<const T*>(a.dy) + b * a.dyb + t * a.dyr + c);
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    if (i0 + i >= RUN + PAST) break;
                    const int64_t t = t0 + i0 + i;  // g of this position; dx of the one three before it
                    W::unpack(in[i], win[PAST]);
                    float d[VEC], out[VEC];
                    W::unpack(din[i], d);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float p = bias[j];
#pragma unroll
                        for (int q = 0; q < TAPS; ++q) p = __builtin_fmaf(w[q][j], win[q][j], p);
                        float gp = d[j];
                        if (a.silu) {
                            const float sig = hw_sigmoid(p);
                            gp = d[j] * __builtin_fmaf(p * sig, 1.0f - sig, sig);
                        }
                        gp = t < end ? gp : 0.0f;
                        g[PAST][j] = gp;
                        if (i0 + i < RUN) {
                            db[j] += gp;
#pragma unroll
                            for (int q = 0; q < TAPS; ++q) dw[q][j] = __builtin_fmaf(gp, win[q][j], dw[q][j]);
                        }
                        float s = w[3][j] * g[0][j];
                        s = __builtin_fmaf(w[2][j], g[1][j], s);
                        s = __builtin_fmaf(w[1][j], g[2][j], s);
                        s = __builtin_fmaf(w[0][j], g[3][j], s);
                        out[j] = t - PAST < end ? s : 0.0f;
#pragma unroll
                        for (int q = 0; q < PAST; ++q) {
                            win[q][j] = win[q + 1][j];
                            g[q][j] = g[q + 1][j];
                        }
                    }
                    if (i0 + i >= PAST && t - PAST < a.length)
                        st_vec<DT, VEC>(static_cast<T*>(a.dx) + b * a.dxb + (t - PAST) * a.dxr + c, out);
                }
            }
        }
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
        for (int q = 0; q < TAPS; ++q) sum[threadIdx.y][(j * (TAPS + 1) + q) * LANES + threadIdx.x] = dw[q][j];
        sum[threadIdx.y][(j * (TAPS + 1) + TAPS) * LANES + threadIdx.x] = db[j];
    }
    __syncthreads();
    if (threadIdx.y != 0 || c >= a.C) return;
    float* mine = a.part + (int64_t)blockIdx.y * (TAPS + 1) * a.C;  // [C][4] weights, then [C] bias
#pragma unroll
    for (int j = 0; j < VEC; ++j)
#pragma unroll
        for (int q = 0; q <= TAPS; ++q) {
            float v = 0.0f;
#pragma unroll
            for (int r = 0; r < RUNS; ++r) v += sum[r][(j * (TAPS + 1) + q) * LANES + threadIdx.x];
            mine[q < TAPS ? (int64_t)(c + j) * TAPS + q : (int64_t)a.C * TAPS + c + j] = v;
        }
}

// One position per sequence: state rows shift by one.
template <int DT, int VEC>
__global__ void __launch_bounds__(WG) k_conv_step(const void* xp, int64_t xs, void* statep, const float* w, const float* bias,
                                                  int64_t batch, int C, int silu, void* yp, int64_t ys) {
    using T = typename Elem<DT>::T;
    using W = Raw<DT, VEC>;
    const int cvs = (C + VEC - 1) / VEC;
    const int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x;
    if (i >= batch * cvs) return;
    const int64_t b = i / cvs;
    const int c = (int)(i % cvs) * VEC;
    T* st = static_cast<T*>(statep) + b * PAST * (int64_t)C + c;
    typename W::V r[TAPS];
#pragma unroll
    for (int q = 0; q < PAST; ++q) r[q] = W::load(st + q * (int64_t)C);
    r[PAST] = W::load(static_cast<const T*>(xp) + b * xs + c);
    float v[TAPS][VEC], out[VEC];
#pragma unroll
    for (int q = 0; q < TAPS; ++q) W::unpack(r[q], v[q]);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        float p = bias != nullptr ? bias[c + j] : 0.0f;
#pragma unroll
        for (int q = 0; q < TAPS; ++q) p = __builtin_fmaf(w[(int64_t)(c + j) * TAPS + q], v[q][j], p);
        out[j] = silu ? hw_silu(p) : p;
    }
    st_vec<DT, VEC>(static_cast<T*>(yp) + b * ys + c, out);
#pragma unroll
    for (int q = 0; q < PAST; ++q) *reinterpret_cast<typename W::V*>(st + q * (int64_t)C) = r[q + 1];
}

// Four channels at a time where all rows are aligned for it (else one): the case above, forward and backward, 205 us (208 with
// single ones), in bfloat16 113 (326).  So rows of 510 and 511 channels, or 512 that begin elsewhere, take 356 us in 16 bits, 255 and
// 264 in float32.
bool vec_ok(int dtype, const void* p, int64_t s0, int64_t s1) {
    const int64_t bytes = dtype == BOA_DT_F32 ? 16 : 8;
    return (uintptr_t)p % bytes == 0 && s0 % 4 == 0 && s1 % 4 == 0;
}
template <class F>
int with_vec(int dtype, bool vec, F f) {
    return with_dtype(dtype, [&](auto dt) {
        return vec ? f(dt, std::integral_constant<int, 4>()) : f(dt, std::integral_constant<int, 1>());
    });
}

int64_t bwd_groups(int64_t batch, int64_t length) {
    const int64_t n = ceil_div(batch * ceil_div(length, RUN), RUNS);
    return n < MAX_GROUPS ? n : MAX_GROUPS;
}

int check_conv(const char* who, int dtype, int64_t batch, int64_t length, int32_t C) {
    if (dtype < BOA_DT_F32 || dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, dtype);
    if (batch < 0 || length < 0 || C < 1 || C > BOA_OPS_MAX_CHANNELS)
        return boa_fail(BOA_ERR_ARG, "%s: need batch, length >= 0 and 1 <= channels <= %d (got %lld, %lld, %d)", who,
                        BOA_OPS_MAX_CHANNELS, (long long)batch, (long long)length, C);
    return BOA_OK;
}

}  // namespace

extern "C" int boa_causal_conv_fwd(int dtype, const void* d_x, int64_t x_batch, int64_t x_row, const float* d_w,
                                   const float* d_b, int silu, int64_t batch, int64_t length, int32_t channels,
                                   const int32_t* d_lens, const void* d_state_in, void* d_state_out, void* d_y,
                                   int64_t y_batch, int64_t y_row, void* stream) {
    const int rc = check_conv("boa_causal_conv_fwd", dtype, batch, length, channels);
    if (rc != BOA_OK) return rc;
    if (batch == 0 || (length == 0 && !d_state_out)) return BOA_OK;
    if (!d_w || (length > 0 && (!d_x || !d_y))) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_fwd: null pointer");
    if (d_state_out && d_state_out == d_state_in)
        return boa_fail(BOA_ERR_ARG, "boa_causal_conv_fwd: d_state_out must be another buffer than d_state_in");
    ConvArgs a = {};
    a.x = d_x, a.xb = x_batch, a.xr = x_row, a.w = d_w, a.b = d_b, a.state_in = d_state_in, a.state_out = d_state_out;
    a.y = d_y, a.yb = y_batch, a.yr = y_row, a.lens = d_lens, a.C = channels, a.silu = silu;
    a.batch = batch, a.length = length, a.runs = length > 0 ? ceil_div(length, RUN) : 1;
    const bool vec = channels % 4 == 0 && vec_ok(dtype, d_x, x_batch, x_row) && vec_ok(dtype, d_y, y_batch, y_row) &&
                     vec_ok(dtype, d_state_in, 0, 0) && vec_ok(dtype, d_state_out, 0, 0);
    const int64_t groups = ceil_div(batch * a.runs, RUNS);
    return with_vec(dtype, vec, [&](auto dt, auto v) {
        constexpr int DT = decltype(dt)::value, VEC = decltype(v)::value;
        hipLaunchKernelGGL((k_conv_fwd<DT, VEC>),
                           dim3((uint32_t)ceil_div(channels, LANES * VEC), (uint32_t)(groups < 32768 ? groups : 32768)),
                           dim3(LANES, RUNS), 0, (hipStream_t)stream, a);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}

extern "C" int64_t boa_causal_conv_bwd_work_bytes(int64_t batch, int64_t length, int32_t channels) {
    return batch < 1 || length < 1 || channels < 1 ? 0 : bwd_groups(batch, length) * (TAPS + 1) * channels * (int64_t)sizeof(float);
}

extern "C" int boa_causal_conv_bwd(int dtype, const void* d_dy, int64_t dy_batch, int64_t dy_row, const void* d_x,
                                   int64_t x_batch, int64_t x_row, const float* d_w, const float* d_b, int silu, int64_t batch,
                                   int64_t length, int32_t channels, const int32_t* d_lens, const void* d_state_in, void* d_dx,
                                   int64_t dx_batch, int64_t dx_row, float* d_dwb, void* d_work, int64_t work_bytes,
                                   void* stream) {
    const int rc = check_conv("boa_causal_conv_bwd", dtype, batch, length, channels);
    if (rc != BOA_OK) return rc;
    const int64_t need = boa_causal_conv_bwd_work_bytes(batch, length, channels);
    if (d_dwb && work_bytes < need)
        return boa_fail(BOA_ERR_ARG, "boa_causal_conv_bwd: workspace of %lld bytes, needs %lld", (long long)work_bytes,
                        (long long)need);
    const bool any = batch > 0 && length > 0;
    if (any && (!d_dy || !d_x || !d_w || !d_dx || (d_dwb && !d_work)))
        return boa_fail(BOA_ERR_ARG, "boa_causal_conv_bwd: null pointer");
    hipStream_t s = (hipStream_t)stream;
    const int64_t groups = any ? bwd_groups(batch, length) : 0;
    if (any) {
        ConvArgs a = {};
        a.x = d_x, a.xb = x_batch, a.xr = x_row, a.dy = d_dy, a.dyb = dy_batch, a.dyr = dy_row, a.w = d_w, a.b = d_b;
        a.state_in = d_state_in, a.dx = d_dx, a.dxb = dx_batch, a.dxr = dx_row, a.lens = d_lens, a.C = channels, a.silu = silu;
        a.batch = batch, a.length = length, a.runs = ceil_div(length, RUN);
        a.part = d_dwb ? static_cast<float*>(d_work) : nullptr;
        const bool vec = channels % 4 == 0 && vec_ok(dtype, d_x, x_batch, x_row) && vec_ok(dtype, d_dy, dy_batch, dy_row) &&
                         vec_ok(dtype, d_dx, dx_batch, dx_row) && vec_ok(dtype, d_state_in, 0, 0);
        const int launched = with_vec(dtype, vec, [&](auto dt, auto v) {
            constexpr int DT = decltype(dt)::value, VEC = decltype(v)::value;
            hipLaunchKernelGGL((k_conv_bwd<DT, VEC>), dim3((uint32_t)ceil_div(channels, LANES * VEC), (uint32_t)groups),
                               dim3(LANES, RUNS), 0, s, a);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
        if (launched != BOA_OK) return launched;
    }
    if (d_dwb) BOA_HIP_TRY(launch_sum_parts(static_cast<float*>(d_work), groups, (int64_t)(TAPS + 1) * channels, d_dwb, s));
    return BOA_OK;
}

extern "C" int boa_causal_conv_step(int dtype, const void* d_x, int64_t x_stride, void* d_state, const float* d_w,
                                    const float* d_b, int silu, int64_t batch, int32_t channels, void* d_y, int64_t y_stride,
                                    void* stream) {
    const int rc = check_conv("boa_causal_conv_step", dtype, batch, 1, channels);
    if (rc != BOA_OK) return rc;
    if (batch == 0) return BOA_OK;
    if (!d_x || !d_state || !d_w || !d_y) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_step: null pointer");
    const bool vec = channels % 4 == 0 && vec_ok(dtype, d_x, x_stride, 0) && vec_ok(dtype, d_y, y_stride, 0) &&
                     vec_ok(dtype, d_state, 0, 0);
    return with_vec(dtype, vec, [&](auto dt, auto v) {
        constexpr int DT = decltype(dt)::value, VEC = decltype(v)::value;
        const int64_t groups = ceil_div(batch * ceil_div(channels, VEC), WG);
        if (groups > MAX_BLOCKS) return boa_fail(BOA_ERR_ARG, "boa_causal_conv_step: batch too large");
        hipLaunchKernelGGL((k_conv_step<DT, VEC>), dim3((uint32_t)groups), dim3(WG), 0, (hipStream_t)stream, d_x, x_stride,
                           d_state, d_w, d_b, batch, channels, silu, d_y, y_stride);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}
