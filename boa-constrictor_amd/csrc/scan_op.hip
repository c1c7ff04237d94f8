// Selective state space scan of every channel over the positions, with its gradient, and the same for one position
// (boa_selective_scan_fwd, boa_selective_scan_bwd, boa_selective_scan_step).
//
//   dt = softplus(delta + bias_c);  e_tn = exp(dt A_cn);  h_tn = e_tn h_(t-1)n + dt u B_tn          n < 16 states per channel
//   y0 = sum_n h_tn C_tn + D_c u;  y = y0 z sigmoid(z)
// and with g = dy z sigmoid(z), from the last position to the first:
//   dh_tn = C_tn g_t + e_(t+1)n dh_(t+1)n;  dC_tn = sum_c g h_tn;  dB_tn = sum_c dh_tn dt u;  w_tn = dh_tn e_tn h_(t-1)n
//   du = dt sum_n dh B + D g;  ddelta = sigmoid(delta + bias) (u sum_n dh B + sum_n w A);  dz = dy y0 silu'(z)
//   dA_cn = sum w dt;  dD = sum g u;  dbias = sum ddelta
//
// Work is 16 exponentials (half rate) and some 5 (forward) to 15 (backward) other operations per state for 16 to 28 bytes
// of float32 input and output per (position, channel): the vector units bound it, not memory.
//
// A workgroup is 64 channels of one sequence, lane = channel, and each of its four wavefronts holds 4 of the 16 states: B
// and C of a position are then the same for a whole wavefront (scalar registers), and what is computed per (position,
// channel) is shared out: of SUB = 8 positions a wavefront prepares two (softplus, gate) and finishes two (the sum over
// states, the gate, the stores), through LDS.  The forward pass of a training step leaves the state at every SUB positions
// ("marks", 8 bytes per (position, channel)); the backward pass walks the blocks of SUB positions from the last one,
// computes each forward again from its mark with e and e h in registers, then backward.
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int NS = 16, WAVES = 4, NQ = NS / WAVES;
constexpr int SUB = BOA_SCAN_MARK, MINE = SUB / WAVES;  // positions of a block, and those a wavefront prepares and finishes
constexpr int WG = 64 * WAVES;
static_assert(SUB % WAVES == 0, "");
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

struct Rows {
    const void* p;
    int64_t b, r;  // element strides of a batch and of a row
};
struct ScanArgs {
    Rows u, delta, z, B, C, dy, y, du, ddelta, dz, dB, dC;
    const float *A, *D, *bias, *state_in;
    float *state_out, *marks, *part_bc, *part_par;
    float *local, *dts;           // [batch][chunks][16][channels], [batch][chunks][channels]
    const int32_t* lens;
    int channels, cblocks, chunks;
    int64_t batch, length, subs;  // subs: blocks of SUB positions of a sequence
    int64_t chunk;                // positions of a chunk, a multiple of SUB
};

template <int DT>
__device__ __forceinline__ const typename Elem<DT>::T* row(const Rows& a, int64_t b, int64_t t) {
    return static_cast<const typename Elem<DT>::T*>(a.p) + b * a.b + t * a.r;
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T* row_mut(const Rows& a, int64_t b, int64_t t) {
    return static_cast<typename Elem<DT>::T*>(const_cast<void*>(a.p)) + b * a.b + t * a.r;
}

// Four consecutive values at a uniform address through the scalar cache (constant address space: nothing the kernel
// writes; 16-bit rows are 4-byte aligned, which the entry points check).
template <int DT>
__device__ __forceinline__ void scalar4(const typename Elem<DT>::T* p, float (&v)[NQ]) {
    typedef __attribute__((address_space(4))) const uint32_t CWord;
    CWord* w = (CWord*)p;
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NQ / 2; ++i) {
            const uint32_t x = w[i];
            v[2 * i] = Elem<DT>::ld((uint16_t)(x & 0xFFFFu));
            v[2 * i + 1] = Elem<DT>::ld((uint16_t)(x >> 16));
        }
    }
}

// The same address, which the compiler takes for another: B and C are loaded again for the way back rather than kept (64
// scalar registers per block).
template <class T>
__device__ __forceinline__ const T* again(const T* p) {
    asm volatile("" : "+s"(p));
    return p;
}

__device__ __forceinline__ int64_t end_of(const ScanArgs& a, int64_t b) {
    if (a.lens == nullptr) return a.length;
    const int64_t n = a.lens[b];
    return n < 0 ? 0 : (n < a.length ? n : a.length);
}

// Where a workgroup is: its channels, its sequence, this wavefront's states.
struct Place {
    int lane, q, c, cc;  // cc: c, or the last channel for the lanes past it (which take part with zeros)
    bool live;
    int cb, k;           // block of channels, chunk
    int64_t b;
    // chunks: how many of them this launch has, the first being `first`
    __device__ __forceinline__ Place(const ScanArgs& a, int chunks, int first) {
        lane = threadIdx.x & 63;
        q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        cb = blockIdx.x % a.cblocks;
        k = blockIdx.x / a.cblocks % chunks + first;
        b = blockIdx.x / a.cblocks / chunks;
        c = cb * 64 + lane;
        live = c < a.channels;
        cc = live ? c : a.channels - 1;
    }
    __device__ __forceinline__ void decay(const ScanArgs& a, float (&a2)[NQ]) const {
#pragma unroll
        for (int n = 0; n < NQ; ++n) a2[n] = live ? a.A[(int64_t)cc * NS + q * NQ + n] * LOG2E : 0.0f;
    }
};

// State `n` of this wavefront in an array [rows][16][channels], row r.
__device__ __forceinline__ int64_t state_at(const ScanArgs& a, const Place& p, int64_t r, int n) {
    return (r * NS + p.q * NQ + n) * a.channels + p.cc;
}

// h of this wavefront's states behind chunk j, from h before it.
__device__ __forceinline__ void over_chunk(const ScanArgs& a, const Place& p, int j, const float (&a2)[NQ], float (&h)[NQ]) {
    const int64_t r = p.b * a.chunks + j;
    const float dts = a.dts[r * a.channels + p.cc];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
        h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(dts * a2[n]), h[n], a.local[state_at(a, p, r, n)]);
}

// LOCAL: the state that a chunk alone leaves (from zeros) and its sum of dt, for every chunk but the last; else the chunk's
// outputs, from the state that the chunks before it leave.
template <int DT, bool LOCAL>
__global__ void __launch_bounds__(WG) k_scan_fwd(const ScanArgs a) {
    using E = Elem<DT>;
    __shared__ float2 s_in[2][SUB][64];  // dt, dt u
    __shared__ float s_y[2][LOCAL ? 1 : WAVES][SUB][64];
    const Place p(a, LOCAL ? a.chunks - 1 : a.chunks, 0);
    const int64_t end = end_of(a, p.b), lo = p.k * a.chunk;
    if (LOCAL && lo + a.chunk >= end) return;  // no chunk behind this one reads its state
    const int64_t hi = lo + a.chunk < a.length ? lo + a.chunk : a.length;  // rows to write
    const int n_subs = lo < end ? (int)ceil_div((hi < end ? hi : end) - lo, SUB) : 0;
    const bool gate = !LOCAL && a.z.p != nullptr;
    float a2[NQ], h[NQ];
    p.decay(a, a2);
    const float bias = a.bias != nullptr ? a.bias[p.cc] : 0.0f, D = !LOCAL && a.D != nullptr ? a.D[p.cc] : 0.0f;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
        h[n] = !LOCAL && a.state_in != nullptr && p.live ? a.state_in[state_at(a, p, p.b, n)] : 0.0f;

    // A block's life: fetched (loads issued), prepared (dt and dt u to LDS), computed, finished (sums over the wavefronts'
    // states, gate, stores).  One barrier per block: block i is computed while i - 1 is finished and i + 1 prepared, with
    // two buffers each.
    typename E::T ru[MINE], rd[MINE], rz[MINE];
    auto fetch = [&](int i) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int64_t t = min(lo + i * SUB + p.q * MINE + k, end - 1);
            ru[k] = row<DT>(a.u, p.b, t)[p.cc];
            rd[k] = row<DT>(a.delta, p.b, t)[p.cc];
            if (gate) rz[k] = row<DT>(a.z, p.b, t)[p.cc];
        }
    };
    float u[MINE] = {}, z[MINE] = {}, u_before[MINE], z_before[MINE];
    auto prepare = [&](int i) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = p.q * MINE + k;
            u[k] = E::ld(ru[k]);
            if (gate) z[k] = E::ld(rz[k]);
            float dt = hw_softplus(E::ld(rd[k]) + bias);
            if (lo + i * SUB + at >= end || !p.live) dt = u[k] = 0.0f;  // the state stays as it is
            s_in[i & 1][at][p.lane] = make_float2(dt, dt * u[k]);
        }
    };
    auto finish = [&](int i) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = p.q * MINE + k;
            const int64_t t = lo + i * SUB + at;
            float y = D * u_before[k];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) y += s_y[i & 1][LOCAL ? 0 : w][at][p.lane];
            if (gate) y *= hw_silu(z_before[k]);
            if (p.live && t < hi) row_mut<DT>(a.y, p.b, t)[p.c] = E::st(t < end ? y : 0.0f);
        }
    };
    if (n_subs > 0) {
        fetch(0);
        if (!LOCAL)
            for (int j = 0; j < p.k; ++j) over_chunk(a, p, j, a2, h);
        prepare(0);
        if (n_subs > 1) fetch(1);
    }
    float dts = 0.0f;
    for (int i = 0; i < n_subs; ++i) {
        __syncthreads();
        if (!LOCAL && a.marks != nullptr && p.live)
#pragma unroll
            for (int n = 0; n < NQ; ++n) a.marks[state_at(a, p, p.b * a.subs + lo / SUB + i, n)] = h[n];
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int64_t t = min(lo + i * SUB + s, end - 1);
            float B[NQ], C[NQ];
            scalar4<DT>(row<DT>(a.B, p.b, t) + p.q * NQ, B);
            if constexpr (!LOCAL) scalar4<DT>(row<DT>(a.C, p.b, t) + p.q * NQ, C);
            const float2 in = s_in[i & 1][s][p.lane];
            float y = 0.0f;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(in.x * a2[n]), h[n], B[n] * in.y);
                if constexpr (!LOCAL) y = __builtin_fmaf(h[n], C[n], y);
            }
            if constexpr (LOCAL) dts += in.x;
            else s_y[i & 1][p.q][s][p.lane] = y;
        }
        if (!LOCAL && i > 0) finish(i - 1);
#pragma unroll
        for (int k = 0; k < MINE; ++k) u_before[k] = u[k], z_before[k] = z[k];
        if (i + 1 < n_subs) prepare(i + 1);
        if (i + 2 < n_subs) fetch(i + 2);
    }
    if constexpr (LOCAL) {
        if (!p.live) return;
        const int64_t r = p.b * a.chunks + p.k;
#pragma unroll
        for (int n = 0; n < NQ; ++n) a.local[state_at(a, p, r, n)] = h[n];
        if (p.q == 0) a.dts[r * a.channels + p.c] = dts;
    } else {
        __syncthreads();
        if (n_subs > 0) finish(n_subs - 1);
        if (!p.live) return;
        // the state behind the last position: from the chunk that has it, without positions from the first
        if (a.state_out != nullptr && (end > lo || lo == 0) && end <= lo + a.chunk)
#pragma unroll
            for (int n = 0; n < NQ; ++n) a.state_out[state_at(a, p, p.b, n)] = h[n];
        for (int64_t t = lo + (int64_t)n_subs * SUB + p.q; t < hi; t += WAVES) row_mut<DT>(a.y, p.b, t)[p.c] = E::st(0.0f);
    }
}

// Sums of 8 values over the wavefront; lane l gets the sum of value l / 8.
__device__ __forceinline__ float sum8(float (&v)[8], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        swap32(v[i], v[i + 4]);
        v[i] += v[i + 4];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        swap16(v[i], v[i + 2]);
        v[i] += v[i + 2];
    }
    const bool up = (lane & 8) != 0;
    float keep = up ? v[1] : v[0], give = up ? v[0] : v[1];
    keep += dpp<DPP_ROR8>(give);
    keep += dpp<DPP_HALF_MIRROR>(keep);
    keep += dpp<DPP_XOR2>(keep);
    keep += dpp<DPP_XOR1>(keep);
    return keep;
}

// What the backward pass prepares of a position: loaded, then dt, dt u, g and the factors that finishing it needs.
template <int DT, bool LOCAL>
struct BackIn {
    using E = Elem<DT>;
    typename E::T ru[MINE], rd[MINE], rz[MINE], ry[MINE];
    __device__ __forceinline__ void fetch(const ScanArgs& a, const Place& p, int64_t t0, int64_t end) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int64_t t = min(t0 + p.q * MINE + k, end - 1);
            if constexpr (!LOCAL) ru[k] = row<DT>(a.u, p.b, t)[p.cc];
            rd[k] = row<DT>(a.delta, p.b, t)[p.cc];
            ry[k] = row<DT>(a.dy, p.b, t)[p.cc];
            if (a.z.p != nullptr) rz[k] = row<DT>(a.z, p.b, t)[p.cc];
        }
    }
};

// The adjoint of the state before a chunk that the chunk's own outputs give (dh from zeros behind it), and its sum of dt, for
// every chunk but the first.
template <int DT>
__global__ void __launch_bounds__(WG) k_scan_bwd_local(const ScanArgs a) {
    using E = Elem<DT>;
    __shared__ float2 s_in[2][SUB][64];  // dt, g
    const Place p(a, a.chunks - 1, 1);
    const int64_t end = end_of(a, p.b), lo = p.k * a.chunk;
    if (lo >= end) return;
    const int n_subs = (int)ceil_div(min(lo + a.chunk, end) - lo, SUB);
    float a2[NQ], dh[NQ] = {}, dts = 0.0f;
    p.decay(a, a2);
    const float bias = a.bias != nullptr ? a.bias[p.cc] : 0.0f;
    BackIn<DT, true> in;
    auto prepare = [&](int i) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = p.q * MINE + k;
            float dt = hw_softplus(E::ld(in.rd[k]) + bias), g = E::ld(in.ry[k]);
            if (a.z.p != nullptr) g *= hw_silu(E::ld(in.rz[k]));
            if (lo + i * SUB + at >= end || !p.live) dt = g = 0.0f;
            s_in[i & 1][at][p.lane] = make_float2(dt, g);
        }
    };
    in.fetch(a, p, lo + (n_subs - 1) * SUB, end);
    prepare(n_subs - 1);
    if (n_subs > 1) in.fetch(a, p, lo + (n_subs - 2) * SUB, end);
    for (int i = n_subs - 1; i >= 0; --i) {
        __syncthreads();
#pragma unroll
        for (int s = SUB - 1; s >= 0; --s) {
            const int64_t t = min(lo + i * SUB + s, end - 1);
            float C[NQ];
            scalar4<DT>(row<DT>(a.C, p.b, t) + p.q * NQ, C);
            const float2 x = s_in[i & 1][s][p.lane];
#pragma unroll
            for (int n = 0; n < NQ; ++n) dh[n] = __builtin_fmaf(C[n], x.y, dh[n]) * __builtin_amdgcn_exp2f(x.x * a2[n]);
            dts += x.x;
        }
        if (i > 0) prepare(i - 1);
        if (i > 1) in.fetch(a, p, lo + (i - 2) * SUB, end);
    }
    if (!p.live) return;
    const int64_t r = p.b * a.chunks + p.k;
#pragma unroll
    for (int n = 0; n < NQ; ++n) a.local[state_at(a, p, r, n)] = dh[n];
    if (p.q == 0) a.dts[r * a.channels + p.c] = dts;
}

template <int DT>
__global__ void __launch_bounds__(WG) k_scan_bwd(const ScanArgs a) {
    using E = Elem<DT>;
    __shared__ float2 s_in[SUB][64];  // dt, dt u
    __shared__ float s_g[SUB][64];
    __shared__ float s_y[WAVES][SUB][64], s_s[WAVES][SUB][64], s_w[WAVES][SUB][64];  // partial sums over the states
    const Place p(a, a.chunks, 0);
    const int64_t end = end_of(a, p.b), lo = p.k * a.chunk;
    const int64_t hi = min(lo + a.chunk, a.length);
    const int n_subs = lo < end ? (int)ceil_div(min(hi, end) - lo, SUB) : 0;
    const bool gate = a.z.p != nullptr;
    float a2[NQ], dh[NQ] = {}, dA[NQ] = {}, dA_all[NQ] = {};
    p.decay(a, a2);
    const float bias = a.bias != nullptr ? a.bias[p.cc] : 0.0f, D = a.D != nullptr ? a.D[p.cc] : 0.0f;
    float dD = 0.0f, dbias = 0.0f, mark[NQ] = {};
    BackIn<DT, false> in;
    auto fetch = [&](int i) {
        in.fetch(a, p, lo + i * SUB, end);
#pragma unroll
        for (int n = 0; n < NQ; ++n) mark[n] = p.live ? a.marks[state_at(a, p, p.b * a.subs + lo / SUB + i, n)] : 0.0f;
    };
    if (n_subs > 0) {
        fetch(n_subs - 1);
        for (int j = (int)ceil_div(end, a.chunk) - 1; j > p.k; --j) over_chunk(a, p, j, a2, dh);
    }
    for (int i = n_subs - 1; i >= 0; --i) {
        const int64_t t0 = lo + i * SUB;
        float u[MINE], dt[MINE], g[MINE], sig[MINE], dyz[MINE];
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = p.q * MINE + k;
            u[k] = E::ld(in.ru[k]);
            const float dy = E::ld(in.ry[k]), pre = E::ld(in.rd[k]) + bias;
            dt[k] = hw_softplus(pre);
            sig[k] = hw_sigmoid(pre);
            g[k] = dy;
            dyz[k] = 0.0f;
            if (gate) {
                const float z = E::ld(in.rz[k]), sz = hw_sigmoid(z);
                g[k] = dy * (z * sz);
                dyz[k] = dy * __builtin_fmaf(z * sz, 1.0f - sz, sz);
            }
            if (t0 + at >= end || !p.live) dt[k] = u[k] = g[k] = sig[k] = dyz[k] = 0.0f;
            s_in[at][p.lane] = make_float2(dt[k], dt[k] * u[k]);
            s_g[at][p.lane] = g[k];
        }
        float h[NQ], e[SUB][NQ], eh[SUB][NQ], bc = 0.0f;
#pragma unroll
        for (int n = 0; n < NQ; ++n) h[n] = mark[n];
        if (i > 0) fetch(i - 1);
        __syncthreads();
        float r[8];
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            const int64_t t = min(t0 + s, end - 1);
            float B[NQ], C[NQ];
            scalar4<DT>(row<DT>(a.B, p.b, t) + p.q * NQ, B);
            scalar4<DT>(row<DT>(a.C, p.b, t) + p.q * NQ, C);
            const float2 x = s_in[s][p.lane];
            const float gs = s_g[s][p.lane];
            float y = 0.0f;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                e[s][n] = __builtin_amdgcn_exp2f(x.x * a2[n]);
                eh[s][n] = e[s][n] * h[n];
                h[n] = __builtin_fmaf(B[n], x.y, eh[s][n]);
                y = __builtin_fmaf(h[n], C[n], y);
                r[(s & 1) * NQ + n] = gs * h[n];
            }
            s_y[p.q][s][p.lane] = y;
            if (s & 1) {  // two positions' dC: lane l has the one of position s - 1 + l / 32, state (l / 8) % 4
                const float v = sum8(r, p.lane);
                bc = (p.lane & 7) == s / 2 ? v : bc;
            }
        }
#pragma unroll
        for (int s = SUB - 1; s >= 0; --s) {
            const int64_t t = min(t0 + s, end - 1);
            float B[NQ], C[NQ];
            scalar4<DT>(again(row<DT>(a.B, p.b, t) + p.q * NQ), B);
            scalar4<DT>(again(row<DT>(a.C, p.b, t) + p.q * NQ), C);
            const float2 x = s_in[s][p.lane];
            const float gs = s_g[s][p.lane];
            float sB = 0.0f, sw = 0.0f;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                dh[n] = __builtin_fmaf(C[n], gs, dh[n]);
                sB = __builtin_fmaf(dh[n], B[n], sB);
                r[(s & 1) * NQ + n] = dh[n] * x.y;
                const float w = dh[n] * eh[s][n];
                sw = __builtin_fmaf(w, a2[n], sw);
                dA[n] = __builtin_fmaf(w, x.x, dA[n]);
                dh[n] *= e[s][n];
            }
            s_s[p.q][s][p.lane] = sB;
            s_w[p.q][s][p.lane] = sw;
            if (!(s & 1)) {
                const float v = sum8(r, p.lane);
                bc = (p.lane & 7) == SUB / 2 + s / 2 ? v : bc;
            }
        }
        a.part_bc[(((int64_t)p.cb * a.batch + p.b) * a.subs + lo / SUB + i) * WG + threadIdx.x] = bc;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = p.q * MINE + k;
            const int64_t t = t0 + at;
            float y = D * u[k], sB = 0.0f, sw = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                y += s_y[w][at][p.lane];
                sB += s_s[w][at][p.lane];
                sw += s_w[w][at][p.lane];
            }
            const float ddelta = __builtin_fmaf(u[k], sB, sw * LN2) * sig[k], du = __builtin_fmaf(dt[k], sB, D * g[k]);
            dD = __builtin_fmaf(g[k], u[k], dD);
            dbias += ddelta;
            if (p.live && t < hi) {
                row_mut<DT>(a.du, p.b, t)[p.c] = E::st(t < end ? du : 0.0f);
                row_mut<DT>(a.ddelta, p.b, t)[p.c] = E::st(t < end ? ddelta : 0.0f);
                if (gate) row_mut<DT>(a.dz, p.b, t)[p.c] = E::st(t < end ? dyz[k] * y : 0.0f);
            }
        }
        if (i % 8 == 0)  // sums of 64 positions at a time: a long sum in one register loses digits
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                dA_all[n] += dA[n];
                dA[n] = 0.0f;
            }
        __syncthreads();
    }
    if (p.live)
        for (int64_t t = lo + (int64_t)n_subs * SUB + p.q; t < hi; t += WAVES) {
            row_mut<DT>(a.du, p.b, t)[p.c] = E::st(0.0f);
            row_mut<DT>(a.ddelta, p.b, t)[p.c] = E::st(0.0f);
            if (gate) row_mut<DT>(a.dz, p.b, t)[p.c] = E::st(0.0f);
        }
    // this chunk's sums for the parameters: [channels][16] of A, [channels] of D, [channels] of the bias
    s_s[p.q][0][p.lane] = dD;
    s_s[p.q][1][p.lane] = dbias;
    __syncthreads();
    if (!p.live) return;
    float* mine = a.part_par + (p.b * a.chunks + p.k) * (NS + 2) * a.channels;
#pragma unroll
    for (int n = 0; n < NQ; ++n) mine[(int64_t)p.c * NS + p.q * NQ + n] = dA_all[n];
    if (p.q < 2) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += s_s[w][p.q][p.lane];
        mine[(int64_t)(NS + p.q) * a.channels + p.c] = v;
    }
}

// dB and dC: the sums over the channel blocks, in the activations' type; zeros behind a sequence's end.
template <int DT>
__global__ void __launch_bounds__(WG) k_scan_sum_bc(const ScanArgs a) {
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
    for (int64_t k = blockIdx.x; k < a.batch * a.subs; k += gridDim.x) {
        const int64_t b = k / a.subs, i = k % a.subs;
        const int64_t end = end_of(a, b), t = i * SUB + (lane & 3) * 2 + (lane >> 5);
        if (t >= a.length) continue;
        float v = 0.0f;
        if (t < end)
            for (int cb = 0; cb < a.cblocks; ++cb) v += a.part_bc[(((int64_t)cb * a.batch + b) * a.subs + i) * WG + threadIdx.x];
        row_mut<DT>((lane & 4) ? a.dB : a.dC, b, t)[q * NQ + ((lane >> 3) & 3)] = Elem<DT>::st(v);
    }
}

// One position: a lane has the 16 states of its channel.
template <int DT>
__global__ void __launch_bounds__(WG) k_scan_step(const ScanArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t k = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t b = k / a.cblocks;
    const int c = (int)(k % a.cblocks) * 64 + lane;
    if (b >= a.batch || c >= a.channels) return;
    float B[NS], C[NS];
#pragma unroll
    for (int i = 0; i < NS; i += NQ) {
        float v[NQ];
        scalar4<DT>(row<DT>(a.B, b, 0) + i, v);
#pragma unroll
        for (int j = 0; j < NQ; ++j) B[i + j] = v[j];
        scalar4<DT>(row<DT>(a.C, b, 0) + i, v);
#pragma unroll
        for (int j = 0; j < NQ; ++j) C[i + j] = v[j];
    }
    float* st = a.state_out + b * NS * (int64_t)a.channels + c;
    float h[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = st[n * (int64_t)a.channels];
    const float u = Elem<DT>::ld(row<DT>(a.u, b, 0)[c]);
    const float dt = hw_softplus(Elem<DT>::ld(row<DT>(a.delta, b, 0)[c]) + (a.bias != nullptr ? a.bias[c] : 0.0f));
    const float du = dt * u;
    float y = (a.D != nullptr ? a.D[c] : 0.0f) * u;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const float e = __builtin_amdgcn_exp2f(dt * (a.A[(int64_t)c * NS + n] * LOG2E));
        h[n] = __builtin_fmaf(e, h[n], B[n] * du);
        y = __builtin_fmaf(h[n], C[n], y);
        st[n * (int64_t)a.channels] = h[n];
    }
    if (a.z.p != nullptr) y *= hw_silu(Elem<DT>::ld(row<DT>(a.z, b, 0)[c]));
    row_mut<DT>(a.y, b, 0)[c] = Elem<DT>::st(y);
}

Rows rows(const boa_rows& r) { return {r.p, r.batch_stride, r.row_stride}; }

// The split over the length: chunks of a multiple of SUB positions, as many as give WANT workgroups (4 per CU), at least
// MIN_CHUNK positions each and at most MAX_CHUNKS (each workgroup goes over the chunks before its own).
struct Plan {
    int chunks;
    int64_t chunk;
};
constexpr int64_t WANT = 1024, MIN_CHUNK = 64, MAX_CHUNKS = 64;
Plan plan(const boa_scan* s) {
    const int64_t blocks = s->batch * ceil_div(s->channels, 64);
    int64_t n = ceil_div(WANT, blocks > 0 ? blocks : 1);
    n = n < MAX_CHUNKS ? n : MAX_CHUNKS;
    int64_t chunk = ceil_div(ceil_div(s->length, n), SUB) * SUB;
    chunk = chunk > MIN_CHUNK ? chunk : MIN_CHUNK;
    n = ceil_div(s->length, chunk);
    return {(int)(n > 1 ? n : 1), chunk};
}

// Workspace, in floats: chunk states and sums of dt (more than one chunk), then in the backward pass the partial sums.
struct Work {
    int64_t local, dts, bc, par;
    int64_t bytes() const { return (local + dts + bc + par) * (int64_t)sizeof(float); }
};
Work work_of(const boa_scan* s, bool backward) {
    Work w = {};
    if (s->batch < 1 || s->length < 1) return w;
    const Plan p = plan(s);
    const int64_t c = s->channels;
    if (p.chunks > 1) w.local = s->batch * p.chunks * NS * c, w.dts = s->batch * p.chunks * c;
    if (backward) {
        w.bc = ceil_div(c, 64) * s->batch * ceil_div(s->length, SUB) * WG;
        w.par = s->batch * p.chunks * (NS + 2) * c;
    }
    return w;
}
void lay_out(ScanArgs& a, const Work& w, void* d_work) {
    a.local = static_cast<float*>(d_work);
    a.dts = a.local + w.local;
    a.part_bc = a.dts + w.dts;
    a.part_par = a.part_bc + w.bc;
}

// B and C rows are read four values at a time at uniform addresses, which have to be multiples of 4 bytes.
bool bc_aligned(const boa_scan* s, const boa_rows& r) {
    return s->dtype == BOA_DT_F32 || ((uintptr_t)r.p % 4 == 0 && r.batch_stride % 2 == 0 && r.row_stride % 2 == 0);
}

int check_scan(const char* who, const boa_scan* s, ScanArgs& a) {
    if (!s) return boa_fail(BOA_ERR_ARG, "%s: null arguments", who);
    if (s->dtype < BOA_DT_F32 || s->dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, s->dtype);
    if (s->batch < 0 || s->length < 0 || s->channels < 1 || s->channels > BOA_OPS_MAX_CHANNELS)
        return boa_fail(BOA_ERR_ARG, "%s: need batch, length >= 0 and 1 <= channels <= %d (got %lld, %lld, %d)", who,
                        BOA_OPS_MAX_CHANNELS, (long long)s->batch, (long long)s->length, s->channels);
    if (s->batch > 0 && s->length > 0) {
        if (!s->u.p || !s->delta.p || !s->b.p || !s->c.p || !s->a) return boa_fail(BOA_ERR_ARG, "%s: null pointer", who);
        if (!bc_aligned(s, s->b) || !bc_aligned(s, s->c))
            return boa_fail(BOA_ERR_ARG, "%s: rows of B and C of 16-bit types have to begin at multiples of 4 bytes", who);
    }
    a = ScanArgs{};
    a.u = rows(s->u), a.delta = rows(s->delta), a.z = rows(s->z), a.B = rows(s->b), a.C = rows(s->c), a.y = rows(s->y);
    a.A = s->a, a.D = s->d, a.bias = s->delta_bias, a.lens = s->lens, a.state_in = s->state_in, a.state_out = s->state_out;
    a.marks = s->marks, a.channels = s->channels, a.cblocks = (int)ceil_div(s->channels, 64);
    a.batch = s->batch, a.length = s->length, a.subs = ceil_div(s->length, SUB);
    const Plan pl = plan(s);
    a.chunks = pl.chunks, a.chunk = pl.chunk;
    if (a.batch > MAX_BLOCKS / ((int64_t)a.cblocks * a.chunks))
        return boa_fail(BOA_ERR_ARG, "%s: batch of %lld sequences too large", who, (long long)a.batch);
    return BOA_OK;
}

}  // namespace

extern "C" int64_t boa_selective_scan_work_bytes(const boa_scan* s, int backward) {
    if (!s || s->batch < 1 || s->length < 1 || s->channels < 1) return 0;
    return work_of(s, backward != 0).bytes();
}

extern "C" int boa_selective_scan_fwd(const boa_scan* s, void* d_work, int64_t work_bytes, void* stream) {
    ScanArgs a;
    const int rc = check_scan("boa_selective_scan_fwd", s, a);
    if (rc != BOA_OK) return rc;
    if (a.batch == 0 || (a.length == 0 && !a.state_out)) return BOA_OK;
    if (a.length > 0 && !a.y.p) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_fwd: null pointer");
    const Work w = work_of(s, false);
    if (w.bytes() > 0 && (!d_work || work_bytes < w.bytes()))
        return boa_fail(BOA_ERR_ARG, "boa_selective_scan_fwd: workspace of %lld bytes, needs %lld", (long long)work_bytes,
                        (long long)w.bytes());
    lay_out(a, w, d_work);
    return with_dtype(s->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const uint32_t blocks = (uint32_t)(a.batch * a.cblocks);
        if (a.chunks > 1) {
            hipLaunchKernelGGL((k_scan_fwd<DT, true>), dim3(blocks * (a.chunks - 1)), dim3(WG), 0, (hipStream_t)stream, a);
            BOA_HIP_TRY(hipGetLastError());
        }
        hipLaunchKernelGGL((k_scan_fwd<DT, false>), dim3(blocks * a.chunks), dim3(WG), 0, (hipStream_t)stream, a);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}

extern "C" int boa_selective_scan_bwd(const boa_scan* s, void* d_work, int64_t work_bytes, void* stream) {
    ScanArgs a;
    const int rc = check_scan("boa_selective_scan_bwd", s, a);
    if (rc != BOA_OK) return rc;
    const bool any = a.batch > 0 && a.length > 0;
    if (!s->dpar) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_bwd: null pointer");
    if (any && (!s->dy.p || !s->du.p || !s->ddelta.p || !s->db.p || !s->dc.p || !s->marks || (s->z.p && !s->dz.p)))
        return boa_fail(BOA_ERR_ARG, "boa_selective_scan_bwd: null pointer");
    const Work w = work_of(s, true);
    if (any && (!d_work || work_bytes < w.bytes()))
        return boa_fail(BOA_ERR_ARG, "boa_selective_scan_bwd: workspace of %lld bytes, needs %lld", (long long)work_bytes,
                        (long long)w.bytes());
    hipStream_t st = (hipStream_t)stream;
    lay_out(a, w, d_work);
    if (any) {
        a.dy = rows(s->dy), a.du = rows(s->du), a.ddelta = rows(s->ddelta), a.dz = rows(s->dz), a.dB = rows(s->db), a.dC = rows(s->dc);
        const int launched = with_dtype(s->dtype, [&](auto dt) {
            constexpr int DT = decltype(dt)::value;
            const uint32_t blocks = (uint32_t)(a.batch * a.cblocks);
            if (a.chunks > 1) {
                hipLaunchKernelGGL((k_scan_bwd_local<DT>), dim3(blocks * (a.chunks - 1)), dim3(WG), 0, st, a);
                BOA_HIP_TRY(hipGetLastError());
            }
            hipLaunchKernelGGL((k_scan_bwd<DT>), dim3(blocks * a.chunks), dim3(WG), 0, st, a);
            BOA_HIP_TRY(hipGetLastError());
            hipLaunchKernelGGL((k_scan_sum_bc<DT>), dim3((uint32_t)min(a.batch * a.subs, MAX_BLOCKS)), dim3(WG), 0, st, a);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
        if (launched != BOA_OK) return launched;
    }
    BOA_HIP_TRY(launch_sum_parts(a.part_par, any ? a.batch * a.chunks : 0, (int64_t)(NS + 2) * a.channels, s->dpar, st));
    return BOA_OK;
}

extern "C" int boa_selective_scan_step(const boa_scan* s, void* stream) {
    ScanArgs a;
    const int rc = check_scan("boa_selective_scan_step", s, a);
    if (rc != BOA_OK) return rc;
    if (a.batch == 0) return BOA_OK;
    if (a.length != 1) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_step: one position per sequence (got %lld)", (long long)a.length);
    if (!a.y.p || !a.state_out) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_step: null pointer");
    return with_dtype(s->dtype, [&](auto dt) {
        hipLaunchKernelGGL((k_scan_step<decltype(dt)::value>), dim3((uint32_t)ceil_div(a.batch * a.cblocks, WAVES)), dim3(WG), 0,
                           (hipStream_t)stream, a);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}
