// Linear attention with a decay for each head, with its gradient, and the same for one position (boa_linear_attention_fwd,
// boa_linear_attention_bwd, boa_linear_attention_step).
//
//   S_t = e^(g_t) S_(t-1) + k_t v_t^T;  y_t = scale S_t^T q_t             a state of `key` x `value` values per head
//
// Positions are taken CHUNK = 64 at a time, so that everything is a matrix product.  With G_i the sum of g from a chunk's
// first position up to i, S the state before the chunk, W_ij = scale e^(G_i - G_j) for j <= i and 0 behind:
//   y_i = scale e^(G_i) S^T q_i + sum_j A_ij v_j,  A_ij = W_ij (q_i . k_j)
//   S behind the chunk = e^(G_end) S + sum_j e^(G_end - G_j) k_j v_j^T
// and with dS the gradient of the state behind the chunk, dA_ij = W_ij (dy_i . v_j):
//   dq_i = scale e^(G_i) S dy_i + sum_j dA_ij k_j;  dk_j = e^(G_end - G_j) dS v_j + sum_i dA_ij q_i
//   dv_j = e^(G_end - G_j) dS^T k_j + sum_i A_ij dy_i
//   dS before the chunk = e^(G_end) dS + sum_i scale e^(G_i) q_i dy_i^T
// dg_t is the sum over all pairs that position t lies between (i >= t > j): of this chunk those of M_ij = A_ij (dy_i . v_j),
// from states before it q_i . (far part of dq_i) for i >= t, to positions behind it k_j . (far part of dk_j) for j < t, and what
// passes over the chunk, e^(G_end) <S, dS>.  All of them are sums of what is there; nothing is a difference of sums over the
// whole length, whose rounding would grow with it.
//
// Four kernels: the states before every chunk (one workgroup walks a piece of the length with the state in registers; pieces
// are joined by a small kernel), then every chunk by itself, forward or backward.
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int WG = 256, WAVES = WG / 64;
constexpr int CHUNK = 64;  // positions of a chunk
constexpr int PV = 64;     // values of a head that a workgroup takes
constexpr int MAX_KEY = BOA_ATTENTION_MAX_KEY, MAX_VALUE = BOA_ATTENTION_MAX_VALUE;
constexpr double LOG2E = 1.4426950408889634074;

struct Heads {
    void* p;
    int64_t bs, rs, hs;
};
struct Args {
    Heads q, k, v, g, y, dy, dq, dk, dv;
    const int32_t* lens;
    const float* state_in;
    float* state_out;
    float* marks;   // [batch heads][value tiles][chunks][NP * PV] states before each chunk (backward: dS behind it), of its piece alone
    float* starts;  // [batch heads][value tiles][pieces][NP * PV] what the pieces before leave (pieces > 1)
    float* pre;     // [batch heads][chunks] decay from the start of its piece
    double* fall;   // [batch heads][pieces] log2 of the piece's decay
    const float *fmarks, *fstarts, *fpre;  // backward: the forward's
    float *part_q, *part_k;                // backward: [batch][length][heads * value tiles][key], or null: dq, dk are written
    float* dg;                             // backward: [value tiles][batch][length][heads], or null
    float* dg_sum;                         // backward: [batch * chunks * value tiles][heads], or null
    int64_t batch, length, chunks;
    int32_t heads, share, key, value, tiles, pieces, per_piece;
    float scale;
    uint32_t wide;  // bit per tensor: read or written 16 bytes at a time (W_*)
};
enum { W_Q = 1, W_K = 2, W_V = 4, W_DY = 8, W_Y = 16, W_DQ = 32, W_DK = 64, W_DV = 128 };

// How products of a type run: elements in LDS, parts that a float32 value is split into, K of a step.
//   bfloat16: inputs as they are.  What is computed on the way (A, dA, states) is split into parts of 8 bits each: two for what
//   ends in a result of 16 bits, three (24 bits) for the states and whatever goes into dg, which are float32.  One rounding to 8
//   bits instead would be as large as the result's own rounding.
//   float32, and float16, whose range the parts of a float32 value do not fit: float32 products (v_mfma_f32_16x16x4_f32).
template <int DT> struct Mat {
    using E = float;
    using Frag = f32x4;
    static constexpr int STEP = 16, VEC = 4, TWO = 1, THREE = 1, PAD = 4;
    static __device__ __forceinline__ floatx4 mma(const Frag& a, const Frag& b, floatx4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    // rows of the fragment along K in memory
    static __device__ __forceinline__ Frag row(const E* t, int ld, int row0, int k0, int lane) {
        return *reinterpret_cast<const Frag*>(t + (row0 + (lane & 15)) * ld + k0 + (lane >> 4) * VEC);
    }
    // and across: element [k][row]
    static __device__ __forceinline__ Frag col(const E* t, int ld, int row0, int k0, int lane) {
        const E* p = t + (k0 + (lane >> 4) * VEC) * ld + row0 + (lane & 15);
        return Frag{p[0], p[ld], p[2 * ld], p[3 * ld]};
    }
    static __device__ __forceinline__ float value(E v) { return v; }
    static __device__ __forceinline__ Frag finite(Frag f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __builtin_isfinite(f[i]) ? f[i] : 0.0f;
        return f;
    }
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <> struct Mat<DT_BF16> {
    using E = uint16_t;
    using Frag = bf16x8;
    static constexpr int STEP = 32, VEC = 8, TWO = 2, THREE = 3, PAD = 8;
    static __device__ __forceinline__ floatx4 mma(const Frag& a, const Frag& b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag row(const E* t, int ld, int row0, int k0, int lane) {
        return *reinterpret_cast<const Frag*>(t + (row0 + (lane & 15)) * ld + k0 + (lane >> 4) * VEC);
    }
    // The transposing read: of 16 lanes, lane i gives the address of 4 elements of row i / 4 at column 4 (i % 4) and gets column i of
    // the four rows.
    static __device__ __forceinline__ Frag col(const E* t, int ld, int row0, int k0, int lane) {
        const int l = lane & 15;
        const E* p = t + (k0 + (lane >> 4) * VEC + (l >> 2)) * ld + row0 + (l & 3) * 4;
        using P = __attribute__((address_space(3))) s16x4*;
        struct {
            s16x4 a, b;
        } r = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((P)p), __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + 4 * ld))};
        return __builtin_bit_cast(Frag, r);
    }
    static __device__ __forceinline__ float value(E v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ Frag finite(Frag f) {
        u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] &= ((w[i] & 0x7F80u) != 0x7F80u ? 0xFFFFu : 0u) | ((w[i] & 0x7F800000u) != 0x7F800000u ? 0xFFFF0000u : 0u);
        return __builtin_bit_cast(Frag, w);
    }
};

// acc[ta][tb] += A B over K from k0 to k1: A's rows from a0 on, B's from b0 on (16 each), held along K in memory (false) or across
// (true), in AS and BS parts that are a_part and b_part elements apart (one of the two has a single part).  FINITE: without
// those of A's elements that are infinite or NaN.
template <class M, bool ACOL, bool BCOL, int AS, int BS, bool FINITE = false, int TA, int TB>
__device__ __forceinline__ void product(floatx4 (&acc)[TA][TB], const typename M::E* a, int a_part, int lda, int a0,
                                        const typename M::E* b, int b_part, int ldb, int b0, int k0, int k1, int lane) {
    static_assert(AS == 1 || BS == 1, "");
    for (int k = k0; k < k1; k += M::STEP) {
        typename M::Frag fb[TB][BS];
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int s = 0; s < BS; ++s)
                fb[j][s] = BCOL ? M::col(b + s * b_part, ldb, b0 + 16 * j, k, lane) : M::row(b + s * b_part, ldb, b0 + 16 * j, k, lane);
#pragma unroll
        for (int i = 0; i < TA; ++i) {
            typename M::Frag fa[AS];
#pragma unroll
            for (int s = 0; s < AS; ++s) {
                fa[s] = ACOL ? M::col(a + s * a_part, lda, a0 + 16 * i, k, lane) : M::row(a + s * a_part, lda, a0 + 16 * i, k, lane);
                if constexpr (FINITE) fa[s] = M::finite(fa[s]);
            }
#pragma unroll
            for (int s = 0; s < AS * BS; ++s)
#pragma unroll
                for (int j = 0; j < TB; ++j) acc[i][j] = M::mma(fa[AS > 1 ? s : 0], fb[j][BS > 1 ? s : 0], acc[i][j]);
        }
    }
}

// acc += A B for a B that is zero outside a triangle: with UPTO, B is held along K and k <= column counts, without it across and
// k >= column.  A is held across ([k][row]).  Where A has infinities or NaN, the zeros of B would make NaN of them and a position
// would reach those before it (or behind, backward): they are left out of the matrix product and added element by element, so that
// whatever they do not reach keeps its bits.
template <class M, bool UPTO, int BS, int TA, int TB>
__device__ __forceinline__ void product_within(floatx4 (&acc)[TA][TB], bool finite, const typename M::E* a, int lda, int a0,
                                               const typename M::E* b, int b_part, int ldb, int b0, int lane) {
    const int k0 = UPTO ? 0 : b0, k1 = UPTO ? b0 + 16 * TB : CHUNK;  // b0 is a multiple of M::STEP
    if (finite) {
        product<M, true, !UPTO, 1, BS>(acc, a, 0, lda, a0, b, b_part, ldb, b0, k0, k1, lane);
        return;
    }
    product<M, true, !UPTO, 1, BS, true>(acc, a, 0, lda, a0, b, b_part, ldb, b0, k0, k1, lane);
#pragma unroll
    for (int i = 0; i < TA; ++i)
#pragma unroll
        for (int j = 0; j < TB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = a0 + 16 * i + 4 * (lane >> 4) + r, col = b0 + 16 * j + (lane & 15);
                float v = acc[i][j][r];
#pragma unroll 1
                for (int k = k0; k < k1; ++k) {
                    const float x = M::value(a[k * lda + row]);
                    if (__builtin_isfinite(x) || (UPTO ? k > col : k < col)) continue;
                    float w = 0.0f;
#pragma unroll
                    for (int s = 0; s < BS; ++s) w += M::value(b[s * b_part + (UPTO ? col * ldb + k : k * ldb + col)]);
                    v = __builtin_fmaf(x, w, v);
                }
                acc[i][j][r] = v;
            }
}

// A value that is no infinity minus itself: the parts behind an infinite first one are zero.
__device__ __forceinline__ float rest(float f, float hi) {
    const float r = f - hi;
    return r == r ? r : 0.0f;
}
// Four consecutive values into LDS, in PARTS parts that are `part` elements apart.
template <class M, int PARTS>
__device__ __forceinline__ void put4(typename M::E* p, int part, floatx4 v) {
    if constexpr (sizeof(typename M::E) == 4) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            const u32x2 w = {bf16_pk(v[0], v[1]), bf16_pk(v[2], v[3])};
            *reinterpret_cast<u32x2*>(p + s * part) = w;
            v = floatx4{rest(v[0], __uint_as_float(w[0] << 16)), rest(v[1], __uint_as_float(w[0] & 0xFFFF0000u)),
                        rest(v[2], __uint_as_float(w[1] << 16)), rest(v[3], __uint_as_float(w[1] & 0xFFFF0000u))};
        }
    }
}

// A tile of CHUNK rows and COLS columns on its way from memory to LDS; zeros behind the last row and column.
template <int DT, int COLS>
struct Tile {
    using M = Mat<DT>;
    using T = typename Elem<DT>::T;
    static constexpr int V = wide<DT>(), PER = CHUNK * COLS / (WG * V), ROW = COLS / V, LD = COLS + M::PAD, SIZE = CHUNK * LD;
    u32x4 v[PER];
    // rows from p on, `rows` and `cols` of them
    __device__ __forceinline__ void load(const T* p, int64_t stride, int rows, int cols, bool wide16) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = threadIdx.x + i * WG, r = at / ROW, c = at % ROW * V;
            v[i] = u32x4{0u, 0u, 0u, 0u};
            if (r < rows && c < cols) {
                const T* q = p + r * stride + c;
                if (wide16) {
                    v[i] = *reinterpret_cast<const u32x4*>(q);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (c + e < cols) {
                            if constexpr (sizeof(T) == 4) v[i][e] = __float_as_uint(q[e]);
                            else v[i][e / 2] |= (uint32_t)q[e] << (16 * (e & 1));
                        }
                }
            }
        }
    }
    __device__ __forceinline__ bool finite() const {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (DT == DT_F32) {
                    ok &= (v[i][e] & 0x7F800000u) != 0x7F800000u;
                } else {
                    constexpr uint32_t m = DT == DT_BF16 ? 0x7F80u : 0x7C00u;
                    ok &= (v[i][e] & m) != m && (v[i][e] >> 16 & m) != m;
                }
            }
        return ok;
    }
    __device__ __forceinline__ void unpack(int i, float (&f)[V]) const {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if constexpr (DT == DT_F32) f[e] = __uint_as_float(v[i][e]);
            else f[e] = Elem<DT>::ld((uint16_t)(v[i][e / 2] >> (16 * (e & 1))));
        }
    }
    __device__ __forceinline__ void store(typename M::E* t) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = threadIdx.x + i * WG, r = at / ROW, c = at % ROW * V;
            if constexpr (DT == DT_F16) {
                float f[V];
                unpack(i, f);
#pragma unroll
                for (int e = 0; e < V; e += 4) *reinterpret_cast<f32x4*>(t + r * LD + c + e) = f32x4{f[e], f[e + 1], f[e + 2], f[e + 3]};
            } else {
                *reinterpret_cast<u32x4*>(t + r * LD + c) = v[i];
            }
        }
    }
    // each row times its weight, in three parts (one in float32)
    __device__ __forceinline__ void store_weighted(typename M::E* t, const float* weight) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = threadIdx.x + i * WG, r = at / ROW, c = at % ROW * V;
            const float w = weight[r];
            float f[V];
            unpack(i, f);
#pragma unroll
            for (int e = 0; e < V; e += 4)
                put4<M, M::THREE>(t + r * LD + c + e, SIZE, floatx4{f[e] * w, f[e + 1] * w, f[e + 2] * w, f[e + 3] * w});
        }
    }
};

// log2 of the decay from a chunk's start up to and with each position (lane), summed in 64 bits; a decay of zero (-inf) as
// 2^-200, which is zero in float32 whatever it is multiplied with, so that differences stay numbers.
__device__ __forceinline__ double decays(const Args& a, int64_t b, int h, int64_t t0, int rows, int lane) {
    double g = 0.0;
    if (lane < rows) {
        g = (double)static_cast<const float*>(a.g.p)[b * a.g.bs + (t0 + lane) * a.g.rs + h * a.g.hs] * LOG2E;
        g = g < -200.0 ? -200.0 : g;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(g, o, 64);
        if (lane >= o) g += x;
    }
    return g;
}
__device__ __forceinline__ float2 in_two(double g) {
    const float hi = (float)g;
    return make_float2(hi, (float)(g - (double)hi));
}
// 2^(a - b)
__device__ __forceinline__ float fall_between(float2 a, float2 b) { return __builtin_amdgcn_exp2f((a.x - b.x) + (a.y - b.y)); }

__device__ __forceinline__ int64_t end_of(const Args& a, int64_t b) {
    if (a.lens == nullptr) return a.length;
    const int64_t n = a.lens[b];
    return n < 0 ? 0 : n < a.length ? n : a.length;
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T* row_of(const Heads& x, int64_t b, int64_t t, int h) {
    return static_cast<typename Elem<DT>::T*>(x.p) + b * x.bs + t * x.rs + h * x.hs;
}

// Where a wavefront's values of a state lie: tile [tn][tp], value r of lane l is row n, column p of the state.
template <int NP>
struct State {
    static constexpr int TN = NP / 32, TP = 2, SIZE = NP * PV;
    floatx4 v[TN][TP];
    static __device__ __forceinline__ int n(int tn, int lane, int wave) { return (wave & 1) * (NP / 2) + tn * 16 + 4 * (lane >> 4); }
    static __device__ __forceinline__ int p(int tp, int lane, int wave) { return (wave >> 1) * 32 + tp * 16 + (lane & 15); }
    static __device__ __forceinline__ int at(int tn, int tp, int lane, int wave) { return (((wave * TN + tn) * TP + tp) * 64 + lane) * 4; }
    __device__ __forceinline__ void load(const float* m, int lane, int wave) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TP; ++j) v[i][j] = *reinterpret_cast<const floatx4*>(m + at(i, j, lane, wave));
    }
    __device__ __forceinline__ void add(const float* m, float f, int lane, int wave) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TP; ++j) {
                const floatx4 x = *reinterpret_cast<const floatx4*>(m + at(i, j, lane, wave));
#pragma unroll
                for (int r = 0; r < 4; ++r) v[i][j][r] = __builtin_fmaf(f, x[r], v[i][j][r]);
            }
    }
    __device__ __forceinline__ void store(float* m, int lane, int wave) const {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TP; ++j) *reinterpret_cast<floatx4*>(m + at(i, j, lane, wave)) = v[i][j];
    }
    // Into LDS as rows of a column's values along n, zeros (which what lies behind key and value need not be) behind them.
    template <class M, int PARTS>
    __device__ __forceinline__ void put(typename M::E* t, int key, int value, int lane, int wave) const {
        constexpr int LD = NP + M::PAD;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TP; ++j) {
                floatx4 x = v[i][j];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n(i, lane, wave) + r >= key || p(j, lane, wave) >= value) x[r] = 0.0f;
                put4<M, PARTS>(t + p(j, lane, wave) * LD + n(i, lane, wave), PV * LD, x);
            }
    }
};

// ---- states before every chunk ----------------------------------------------------------------------
// A workgroup walks the chunks of a piece, forward over k v^T, or (BACK) from the last one over scale e^(G_i) q dy^T, and leaves the
// state that it reaches each chunk with.  Where the length is one piece it starts from the caller's state and hands it on.
template <int DT, int NP, bool BACK>
__global__ void __launch_bounds__(WG) k_attn_states(const Args a) {
    using M = Mat<DT>;
    using TX = Tile<DT, NP>;
    using TY = Tile<DT, PV>;
    using S = State<NP>;
    __shared__ __attribute__((aligned(16))) typename M::E tx[TX::SIZE];
    __shared__ __attribute__((aligned(16))) typename M::E ty[M::THREE * TY::SIZE];
    __shared__ float weight[CHUNK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int piece = (int)(blockIdx.x % a.pieces), tile = (int)(blockIdx.x / a.pieces % a.tiles);
    const int64_t bh = blockIdx.x / a.pieces / a.tiles, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t end = end_of(a, b);
    const int64_t c0 = (int64_t)piece * a.per_piece, c1 = min(c0 + a.per_piece, (end + CHUNK - 1) / CHUNK);
    const Heads &X = BACK ? a.q : a.k, &Y = BACK ? a.dy : a.v;
    const bool wx = (a.wide & (BACK ? W_Q : W_K)) != 0, wy = (a.wide & (BACK ? W_DY : W_V)) != 0;
    const int vcols = min(PV, a.value - tile * PV);
    float* marks = a.marks + (bh * a.tiles + tile) * a.chunks * S::SIZE;

    S s;
#pragma unroll
    for (int i = 0; i < S::TN; ++i)
#pragma unroll
        for (int j = 0; j < S::TP; ++j) {
            s.v[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            if (!BACK && a.pieces == 1 && a.state_in != nullptr) {
                const int p = tile * PV + S::p(j, lane, wave);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = S::n(i, lane, wave) + r;
                    if (n < a.key && p < a.value) s.v[i][j][r] = a.state_in[(bh * a.key + n) * a.value + p];
                }
            }
        }
    double passed = 0.0;
    TX x;
    TY y;
    double g = 0.0;
    const auto fetch = [&](int64_t c) {
        const int64_t t0 = c * CHUNK;
        const int rows = (int)min((int64_t)CHUNK, end - t0);
        x.load(row_of<DT>(X, b, t0, h / a.share), X.rs, rows, a.key, wx);
        y.load(row_of<DT>(Y, b, t0, h) + tile * PV, Y.rs, rows, vcols, wy);
        g = decays(a, b, h, t0, rows, lane);
    };
    const int64_t n = c1 - c0;
    if (n > 0) fetch(BACK ? c1 - 1 : c0);
    for (int64_t m = 0; m < n; ++m) {
        const int64_t c = BACK ? c1 - 1 - m : c0 + m;
        s.store(marks + c * S::SIZE, lane, wave);
        if (a.pre != nullptr && tile == 0 && threadIdx.x == 0) a.pre[bh * a.chunks + c] = __builtin_amdgcn_exp2f((float)passed);
        const double all = __shfl(g, 63, 64);
        if (wave == 0) weight[lane] = BACK ? a.scale * __builtin_amdgcn_exp2f((float)g) : __builtin_amdgcn_exp2f((float)(all - g));
        __syncthreads();
        x.store(tx);
        y.store_weighted(ty, weight);
        __syncthreads();
        if (m + 1 < n) fetch(BACK ? c - 1 : c + 1);
        const float f = __builtin_amdgcn_exp2f((float)all);
        passed += all;
#pragma unroll
        for (int i = 0; i < S::TN; ++i)
#pragma unroll
            for (int j = 0; j < S::TP; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) s.v[i][j][r] *= f;
        product<M, true, true, 1, M::THREE>(s.v, tx, 0, TX::LD, (wave & 1) * (NP / 2), ty, TY::SIZE, TY::LD, (wave >> 1) * 32, 0, CHUNK, lane);
        __syncthreads();
    }
    if (a.pieces > 1) {
        s.store(a.starts + ((bh * a.tiles + tile) * a.pieces + piece) * S::SIZE, lane, wave);
        if (tile == 0 && threadIdx.x == 0) a.fall[bh * a.pieces + piece] = passed;
    } else if (!BACK && a.state_out != nullptr) {
#pragma unroll
        for (int i = 0; i < S::TN; ++i)
#pragma unroll
            for (int j = 0; j < S::TP; ++j) {
                const int p = tile * PV + S::p(j, lane, wave);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int k = S::n(i, lane, wave) + r;
                    if (k < a.key && p < a.value) a.state_out[(bh * a.key + k) * a.value + p] = s.v[i][j][r];
                }
            }
    }
}

// What each piece leaves by itself becomes the state that it starts from (backward: the gradient of the state behind it), eight
// pieces' loads at a time.  A thread has four values of a state.
template <int NP, bool BACK>
__global__ void __launch_bounds__(WG) k_attn_join(const Args a) {
    using S = State<NP>;
    constexpr int PER = S::SIZE / (WG * 4), AT_ONCE = 8;
    const int part = (int)(blockIdx.x % PER);
    const int64_t bht = blockIdx.x / PER, bh = bht / a.tiles;
    const int tile = (int)(bht % a.tiles), lane = threadIdx.x & 63;
    const int block = part * (WG / 64) + (threadIdx.x >> 6);  // (wave * TN + tn) * TP + tp
    const int tp = block % S::TP, tn = block / S::TP % S::TN, wave = block / S::TP / S::TN;
    const int n = S::n(tn, lane, wave), p = tile * PV + S::p(tp, lane, wave);
    float* at = a.starts + bht * a.pieces * S::SIZE + block * 256 + lane * 4;
    floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!BACK && a.state_in != nullptr)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < a.key && p < a.value) s[r] = a.state_in[(bh * a.key + n + r) * a.value + p];
    for (int i0 = 0; i0 < a.pieces; i0 += AT_ONCE) {
        floatx4 own[AT_ONCE];
        float f[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int k = min(i0 + i, a.pieces - 1), piece = BACK ? a.pieces - 1 - k : k;
            own[i] = *reinterpret_cast<const floatx4*>(at + (int64_t)piece * S::SIZE);
            f[i] = __builtin_amdgcn_exp2f((float)a.fall[bh * a.pieces + piece]);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (i0 + i >= a.pieces) break;
            const int piece = BACK ? a.pieces - 1 - (i0 + i) : i0 + i;
            *reinterpret_cast<floatx4*>(at + (int64_t)piece * S::SIZE) = s;
#pragma unroll
            for (int r = 0; r < 4; ++r) s[r] = __builtin_fmaf(f[i], s[r], own[i][r]);
        }
    }
    if (!BACK && a.state_out != nullptr)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < a.key && p < a.value) a.state_out[(bh * a.key + n + r) * a.value + p] = s[r];
}

// Four consecutive columns of a row of a result.
template <int DT>
__device__ __forceinline__ void write4(typename Elem<DT>::T* p, int col, int cols, bool wide16, floatx4 v) {
    if (wide16 && col < cols) {
        const float f[4] = {v[0], v[1], v[2], v[3]};
        st_vec<DT, 4>(p + col, f);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (col + r < cols) p[col + r] = Elem<DT>::st(v[r]);
    }
}

struct Place {
    int64_t c, bh, b, t0, end;
    int tile, h, rows, vcols;
    __device__ __forceinline__ Place(const Args& a) {
        c = blockIdx.x % a.chunks;
        tile = (int)(blockIdx.x / a.chunks % a.tiles);
        bh = blockIdx.x / a.chunks / a.tiles;
        b = bh / a.heads;
        h = (int)(bh % a.heads);
        t0 = c * CHUNK;
        end = end_of(a, b);
        rows = (int)max((int64_t)0, min((int64_t)CHUNK, end - t0));  // that hold something
        vcols = min(PV, a.value - tile * PV);
    }
};
// Zeros for the rows of a chunk from `from` on.
template <int DT>
__device__ __forceinline__ void zero_rows(const Args& a, const Place& w, const Heads& x, int h, int col0, int cols, int from) {
    const int last = (int)min((int64_t)CHUNK, a.length - w.t0);
    for (int i = threadIdx.x; i < (last - from) * cols; i += WG)
        row_of<DT>(x, w.b, w.t0 + from + i / cols, h)[col0 + i % cols] = Elem<DT>::st(0.0f);
}

// ---- forward, a chunk ---------------------------------------------------------------------------------
template <int DT, int NP>
__global__ void __launch_bounds__(WG) k_attn_fwd(const Args a) {
    using M = Mat<DT>;
    using E = typename M::E;
    using TN = Tile<DT, NP>;
    using TV = Tile<DT, PV>;
    using S = State<NP>;
    constexpr int SA = CHUNK * (CHUNK + M::PAD), LA = CHUNK + M::PAD;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    E* tq = reinterpret_cast<E*>(lds);
    E* tk = tq + TN::SIZE;
    E* tv = tk + TN::SIZE;
    E* ts = tv + TV::SIZE;                   // [PV][NP] in two parts
    E* ta = ts + M::TWO * PV * TN::LD;       // [CHUNK][CHUNK] in two parts
    __shared__ float2 G[CHUNK];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Place w(a);
    if (w.rows < CHUNK) zero_rows<DT>(a, w, a.y, w.h, w.tile * PV, w.vcols, w.rows);
    if (w.rows == 0) return;
    TN q, k;
    TV v;
    S s;
    const int64_t bht = w.bh * a.tiles + w.tile;
    s.load(a.marks + (bht * a.chunks + w.c) * S::SIZE, lane, wave);
    q.load(row_of<DT>(a.q, w.b, w.t0, w.h / a.share), a.q.rs, w.rows, a.key, a.wide & W_Q);
    k.load(row_of<DT>(a.k, w.b, w.t0, w.h / a.share), a.k.rs, w.rows, a.key, a.wide & W_K);
    v.load(row_of<DT>(a.v, w.b, w.t0, w.h) + w.tile * PV, a.v.rs, w.rows, w.vcols, a.wide & W_V);
    const double g = decays(a, w.b, w.h, w.t0, w.rows, lane);
    if (wave == 0) G[lane] = in_two(g);
    if (a.pieces > 1)
        s.add(a.starts + (bht * a.pieces + w.c / a.per_piece) * S::SIZE, a.pre[w.bh * a.chunks + w.c], lane, wave);
    q.store(tq);
    k.store(tk);
    v.store(tv);
    s.template put<M, M::TWO>(ts, a.key, w.vcols, lane, wave);
    const bool finite = __syncthreads_and(v.finite());
    const int i0 = (wave & 1) * 32, j0 = (wave >> 1) * 32, l15 = lane & 15, row4 = 4 * (lane >> 4);
    // A_ij of 32 x 32 positions (rows j, column i), into LDS along j
    if (j0 <= i0) {
        floatx4 acc[2][2] = {};
        product<M, false, false, 1, 1>(acc, tk, 0, TN::LD, j0, tq, 0, TN::LD, i0, 0, NP, lane);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const int i = i0 + 16 * ti + l15;
            const float2 gi = G[i];
#pragma unroll
            for (int tj = 0; tj < 2; ++tj) {
                const int j = j0 + 16 * tj + row4;
                floatx4 x;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    x[r] = j + r <= i && i < w.rows ? acc[tj][ti][r] * (a.scale * fall_between(gi, G[j + r])) : 0.0f;
                put4<M, M::TWO>(ta + i * LA + j, SA, x);
            }
        }
    }
    // y of 32 positions (columns) and 32 values (rows): what the state gives, then the chunk's own
    const int p0 = j0;
    floatx4 y[2][2] = {};
    product<M, false, false, M::TWO, 1>(y, ts, PV * TN::LD, TN::LD, p0, tq, 0, TN::LD, i0, 0, NP, lane);
#pragma unroll
    for (int ti = 0; ti < 2; ++ti) {
        const float2 gi = G[i0 + 16 * ti + l15];
        const float f = a.scale * __builtin_amdgcn_exp2f(gi.x + gi.y);
#pragma unroll
        for (int tp = 0; tp < 2; ++tp)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[tp][ti][r] *= f;
    }
    __syncthreads();
    product_within<M, true, M::TWO>(y, finite, tv, TV::LD, p0, ta, SA, LA, i0, lane);
#pragma unroll
    for (int ti = 0; ti < 2; ++ti) {
        const int i = i0 + 16 * ti + l15;
        if (i >= w.rows) continue;
        auto* out = row_of<DT>(a.y, w.b, w.t0 + i, w.h) + w.tile * PV;
#pragma unroll
        for (int tp = 0; tp < 2; ++tp) write4<DT>(out, p0 + 16 * tp + row4, w.vcols, a.wide & W_Y, y[tp][ti]);
    }
}
template <int DT, int NP>
constexpr int fwd_lds() {
    using M = Mat<DT>;
    return (int)sizeof(typename M::E) * (2 * Tile<DT, NP>::SIZE + Tile<DT, PV>::SIZE + M::TWO * PV * Tile<DT, NP>::LD +
                                         M::TWO * CHUNK * (CHUNK + M::PAD));
}

// ---- backward, a chunk --------------------------------------------------------------------------------
// The sum of v over the lanes of a tile's column; every lane gets its column's.
__device__ __forceinline__ float over_rows(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// Of the 16 columns of a row of lanes the sum from a lane's own to the last one.
constexpr int DPP_SHL1 = 0x101, DPP_SHL2 = 0x102, DPP_SHL4 = 0x104, DPP_SHL8 = 0x108, DPP_FROM_FIRST = 0x150;
__device__ __forceinline__ float from_here(float v) {
    v += dpp<DPP_SHL1>(v);
    v += dpp<DPP_SHL2>(v);
    v += dpp<DPP_SHL4>(v);
    return v + dpp<DPP_SHL8>(v);
}

template <int DT, int NP>
__global__ void __launch_bounds__(WG) k_attn_bwd(const Args a) {
    using M = Mat<DT>;
    using E = typename M::E;
    using TN = Tile<DT, NP>;
    using TV = Tile<DT, PV>;
    using S = State<NP>;
    constexpr int SA = CHUNK * (CHUNK + M::PAD), LA = CHUNK + M::PAD, SS = PV * TN::LD, NT = NP / 32;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    E* tq = reinterpret_cast<E*>(lds);
    E* tk = tq + TN::SIZE;
    E* tv = tk + TN::SIZE;
    E* td = tv + TV::SIZE;           // dy
    E* ts = td + TV::SIZE;           // [PV][NP] in three parts: S, then dS
    E* ta = ts + M::THREE * SS;      // [CHUNK][CHUNK] in two parts: dA, then A
    __shared__ float2 G[CHUNK];
    __shared__ float pairs[2][CHUNK], over_middle[CHUNK / 2], from_before[2][CHUNK], to_behind[2][CHUNK], through[WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, row4 = 4 * (lane >> 4);
    const Place w(a);
    const int part = w.h * a.tiles + w.tile, parts = a.heads * a.tiles;
    const int present = (int)min((int64_t)CHUNK, a.length - w.t0);
    float* dg = a.dg == nullptr ? nullptr : a.dg + ((w.tile * a.batch + w.b) * a.length + w.t0) * a.heads + w.h;
    float* dg_sum = a.dg_sum == nullptr ? nullptr : a.dg_sum + ((w.b * a.chunks + w.c) * a.tiles + w.tile) * a.heads + w.h;
    const auto part_row = [&](float* p, int i) { return p + ((w.b * a.length + w.t0 + i) * parts + part) * a.key; };
    if (w.rows < CHUNK) {
        zero_rows<DT>(a, w, a.dv, w.h, w.tile * PV, w.vcols, w.rows);
        if (a.part_q == nullptr) {
            zero_rows<DT>(a, w, a.dq, w.h, 0, a.key, w.rows);
            zero_rows<DT>(a, w, a.dk, w.h, 0, a.key, w.rows);
        } else {
            for (int i = threadIdx.x; i < (present - w.rows) * a.key; i += WG) {
                part_row(a.part_q, w.rows + i / a.key)[i % a.key] = 0.0f;
                part_row(a.part_k, w.rows + i / a.key)[i % a.key] = 0.0f;
            }
        }
    }
    if (w.rows == 0) {
        if (dg != nullptr && (int)threadIdx.x < present) dg[(int64_t)threadIdx.x * a.heads] = 0.0f;
        if (dg_sum != nullptr && threadIdx.x == 0) *dg_sum = 0.0f;
        return;
    }
    S s, ds;
    TN q, k;
    TV v, d;
    const int64_t bht = w.bh * a.tiles + w.tile, mark = (bht * a.chunks + w.c) * S::SIZE;
    const int64_t start = (bht * a.pieces + w.c / a.per_piece) * S::SIZE;
    q.load(row_of<DT>(a.q, w.b, w.t0, w.h / a.share), a.q.rs, w.rows, a.key, a.wide & W_Q);
    k.load(row_of<DT>(a.k, w.b, w.t0, w.h / a.share), a.k.rs, w.rows, a.key, a.wide & W_K);
    v.load(row_of<DT>(a.v, w.b, w.t0, w.h) + w.tile * PV, a.v.rs, w.rows, w.vcols, a.wide & W_V);
    d.load(row_of<DT>(a.dy, w.b, w.t0, w.h) + w.tile * PV, a.dy.rs, w.rows, w.vcols, a.wide & W_DY);
    s.load(a.fmarks + mark, lane, wave);
    ds.load(a.marks + mark, lane, wave);
    const double g = decays(a, w.b, w.h, w.t0, w.rows, lane);
    const double all = __shfl(g, 63, 64);
    const float2 g_end = in_two(all);
    if (wave == 0) G[lane] = in_two(g);
    if (a.pieces > 1) {
        s.add(a.fstarts + start, a.fpre[w.bh * a.chunks + w.c], lane, wave);
        ds.add(a.starts + start, a.pre[w.bh * a.chunks + w.c], lane, wave);
    }
    q.store(tq);
    k.store(tk);
    v.store(tv);
    d.store(td);
    s.template put<M, M::THREE>(ts, a.key, w.vcols, lane, wave);
    // what passes over the chunk
    {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < S::TN; ++i)
#pragma unroll
            for (int j = 0; j < S::TP; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (S::n(i, lane, wave) + r < a.key && S::p(j, lane, wave) < w.vcols) x = __builtin_fmaf(s.v[i][j][r], ds.v[i][j][r], x);
        x = wsum(x);
        if (lane == 0) through[wave] = x;
    }
    const bool finite = __syncthreads_and(q.finite() && k.finite() && d.finite());

    // A and dA of 32 x 32 positions (rows j, column i)
    const int i0 = (wave & 1) * 32, j0 = (wave >> 1) * 32;
    floatx4 A[2][2] = {}, dA[2][2] = {};
    if (j0 <= i0) {
        product<M, false, false, 1, 1>(A, tk, 0, TN::LD, j0, tq, 0, TN::LD, i0, 0, NP, lane);
        product<M, false, false, 1, 1>(dA, tv, 0, TV::LD, j0, td, 0, TV::LD, i0, 0, PV, lane);
        floatx4 m[2][2];
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const int i = i0 + 16 * ti + l15;
            const float2 gi = G[i];
#pragma unroll
            for (int tj = 0; tj < 2; ++tj) {
                const int j = j0 + 16 * tj + row4;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = j + r <= i && i < w.rows;
                    const float f = a.scale * fall_between(gi, G[j + r]);
                    A[tj][ti][r] = in ? A[tj][ti][r] * f : 0.0f;
                    m[tj][ti][r] = in ? A[tj][ti][r] * dA[tj][ti][r] : 0.0f;
                    dA[tj][ti][r] = in ? dA[tj][ti][r] * f : 0.0f;
                }
                put4<M, M::TWO>(ta + i * LA + j, SA, dA[tj][ti]);
            }
        }
        // the pairs that a position t (as i) lies between: sums of M_ij over i >= t of these 32, then over j < t
        float at[2] = {0.0f, 0.0f};
#pragma unroll
        for (int tj = 0; tj < 2; ++tj)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float second = from_here(m[tj][1][r]), first = from_here(m[tj][0][r]) + dpp<DPP_FROM_FIRST>(second);
                const int j = j0 + 16 * tj + row4 + r;
                at[0] += j < i0 + l15 ? first : 0.0f;
                at[1] += j < i0 + 16 + l15 ? second : 0.0f;
                if (i0 > j0 && l15 == 0) over_middle[j] = first;
            }
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const float x = over_rows(at[ti]);
            if (lane < 16) pairs[wave >> 1][i0 + 16 * ti + l15] = x;
        }
    } else if (lane < 32) {
        pairs[wave >> 1][i0 + lane] = 0.0f;
    }
    __syncthreads();

    // key halves by the wavefront's second bit here, positions by its first
    const int n0 = (wave >> 1) * (NP / 2);
    {
        floatx4 o[NT][2] = {};
        product<M, true, false, M::THREE, 1>(o, ts, SS, TN::LD, n0, td, 0, TV::LD, i0, 0, PV, lane);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const int i = i0 + 16 * ti + l15;
            const float2 gi = G[i];
            const float f = a.scale * __builtin_amdgcn_exp2f(gi.x + gi.y);
            float x = 0.0f;
#pragma unroll
            for (int tn = 0; tn < NT; ++tn)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    o[tn][ti][r] *= f;
                    x = __builtin_fmaf(o[tn][ti][r], M::value(tq[i * TN::LD + n0 + 16 * tn + row4 + r]), x);
                }
            x = over_rows(x);
            if (lane < 16) from_before[wave >> 1][i] = x;
        }
        product_within<M, true, M::TWO>(o, finite, tk, TN::LD, n0, ta, SA, LA, i0, lane);
#pragma unroll
        for (int ti = 0; ti < 2; ++ti) {
            const int i = i0 + 16 * ti + l15;
            if (i >= w.rows) continue;
#pragma unroll
            for (int tn = 0; tn < NT; ++tn) {
                if (a.part_q == nullptr) write4<DT>(row_of<DT>(a.dq, w.b, w.t0 + i, w.h), n0 + 16 * tn + row4, a.key, a.wide & W_DQ, o[tn][ti]);
                else write4<DT_F32>(part_row(a.part_q, i), n0 + 16 * tn + row4, a.key, a.key % 4 == 0, o[tn][ti]);
            }
        }
    }
    __syncthreads();
    ds.template put<M, M::THREE>(ts, a.key, w.vcols, lane, wave);
    __syncthreads();
    {
        const int c0 = i0;  // the columns are positions j here
        floatx4 o[NT][2] = {};
        product<M, true, false, M::THREE, 1>(o, ts, SS, TN::LD, n0, tv, 0, TV::LD, c0, 0, PV, lane);
#pragma unroll
        for (int tj = 0; tj < 2; ++tj) {
            const int j = c0 + 16 * tj + l15;
            const float f = fall_between(g_end, G[j]);
            float x = 0.0f;
#pragma unroll
            for (int tn = 0; tn < NT; ++tn)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    o[tn][tj][r] *= f;
                    x = __builtin_fmaf(o[tn][tj][r], M::value(tk[j * TN::LD + n0 + 16 * tn + row4 + r]), x);
                }
            x = over_rows(x);
            if (lane < 16) to_behind[wave >> 1][j] = x;
        }
        product_within<M, false, M::TWO>(o, finite, tq, TN::LD, n0, ta, SA, LA, c0, lane);
#pragma unroll
        for (int tj = 0; tj < 2; ++tj) {
            const int j = c0 + 16 * tj + l15;
            if (j >= w.rows) continue;
#pragma unroll
            for (int tn = 0; tn < NT; ++tn) {
                if (a.part_k == nullptr) write4<DT>(row_of<DT>(a.dk, w.b, w.t0 + j, w.h), n0 + 16 * tn + row4, a.key, a.wide & W_DK, o[tn][tj]);
                else write4<DT_F32>(part_row(a.part_k, j), n0 + 16 * tn + row4, a.key, a.key % 4 == 0, o[tn][tj]);
            }
        }
    }
    __syncthreads();
    if (j0 <= i0) {
#pragma unroll
        for (int ti = 0; ti < 2; ++ti)
#pragma unroll
            for (int tj = 0; tj < 2; ++tj) put4<M, M::TWO>(ta + (i0 + 16 * ti + l15) * LA + j0 + 16 * tj + row4, SA, A[tj][ti]);
    }
    __syncthreads();
    {
        const int p0 = j0, c0 = i0;
        floatx4 o[2][2] = {};
        product<M, false, false, M::THREE, 1>(o, ts, SS, TN::LD, p0, tk, 0, TN::LD, c0, 0, NP, lane);
#pragma unroll
        for (int tj = 0; tj < 2; ++tj) {
            const float f = fall_between(g_end, G[c0 + 16 * tj + l15]);
#pragma unroll
            for (int tp = 0; tp < 2; ++tp)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[tp][tj][r] *= f;
        }
        product_within<M, false, M::TWO>(o, finite, td, TV::LD, p0, ta, SA, LA, c0, lane);
#pragma unroll
        for (int tj = 0; tj < 2; ++tj) {
            const int j = c0 + 16 * tj + l15;
            if (j >= w.rows) continue;
            auto* out = row_of<DT>(a.dv, w.b, w.t0 + j, w.h) + w.tile * PV;
#pragma unroll
            for (int tp = 0; tp < 2; ++tp) write4<DT>(out, p0 + 16 * tp + row4, w.vcols, a.wide & W_DV, o[tp][tj]);
        }
    }
    // dg, by one wavefront (lane = position)
    if (wave == 0 && (dg != nullptr || dg_sum != nullptr)) {
        // of the chunk's own pairs those of its second half with its first are missing for the first half's positions
        const double over = ((double)through[0] + (double)through[1] + (double)through[2] + (double)through[3]) * (double)__builtin_amdgcn_exp2f((float)all);
        const bool in = lane < w.rows;
        double behind = in ? (double)to_behind[0][lane] + (double)to_behind[1][lane] : 0.0;
        double middle = lane < CHUNK / 2 ? (double)over_middle[lane] : 0.0;
        double later = in ? (double)from_before[0][lane] + (double)from_before[1][lane] : 0.0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double x = __shfl_up(behind, o, 64), y = __shfl_up(middle, o, 64), z = __shfl_down(later, o, 64);
            if (lane >= o) behind += x, middle += y;
            if (lane + o < 64) later += z;
        }
        behind = __shfl_up(behind, 1, 64), middle = __shfl_up(middle, 1, 64);  // of the positions before
        double x = (double)pairs[0][lane] + (double)pairs[1][lane] + later + over;
        if (lane > 0) x += behind;
        if (lane > 0 && lane < CHUNK / 2) x += middle;
        if (!in) x = 0.0;
        if (dg != nullptr && lane < present) dg[(int64_t)lane * a.heads] = (float)x;
        if (dg_sum != nullptr) {
            double sum = x;
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
            if (lane == 0) *dg_sum = (float)sum;
        }
    }
}
template <int DT, int NP>
constexpr int bwd_lds() {
    using M = Mat<DT>;
    return (int)sizeof(typename M::E) * (2 * Tile<DT, NP>::SIZE + 2 * Tile<DT, PV>::SIZE + M::THREE * PV * Tile<DT, NP>::LD +
                                         M::TWO * CHUNK * (CHUNK + M::PAD));
}

// dq and dk of a group's key from its heads' parts (and those of their value tiles), in their order; dg from its value tiles.
template <int DT>
__global__ void __launch_bounds__(WG) k_attn_sum(const Args a, const float* part, Heads out, int groups) {
    const int64_t n = a.batch * a.length * groups * a.key;
    const int each = a.share * a.tiles;
    for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
        const int col = (int)(i % a.key), gr = (int)(i / a.key % groups);
        const int64_t bt = i / a.key / groups;
        const float* p = part + (bt * groups + gr) * each * a.key + col;
        float v = p[0];
        for (int k = 1; k < each; ++k) v += p[(int64_t)k * a.key];
        row_of<DT>(out, bt / a.length, bt % a.length, gr)[col] = Elem<DT>::st(v);
    }
}
__global__ void __launch_bounds__(WG) k_attn_sum_tiles(const float* part, float* out, int64_t n, int tiles) {
    for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
        float v = part[i];
        for (int k = 1; k < tiles; ++k) v += part[k * n + i];
        out[i] = v;
    }
}

// ---- one position -------------------------------------------------------------------------------------
// A workgroup per head of a sequence: a thread has VEC values of every ROWS-th row of the state, read and written once; the rows'
// products with q are summed over the wavefront's lanes, then through LDS.
template <int DT, int VEC>
__global__ void __launch_bounds__(WG) k_attn_step(const Args a) {
    constexpr int LANES = 64 / VEC, ROWS = WG / LANES, AT_ONCE = 4;  // lanes of a row of PV values, rows at a time
    __shared__ float part[WAVES][PV];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = threadIdx.x % LANES * VEC, row = threadIdx.x / LANES;
    for (int64_t bh = blockIdx.x; bh < a.batch * a.heads; bh += gridDim.x) {
        const int64_t b = bh / a.heads;
        const int h = (int)(bh % a.heads);
        const auto* q = row_of<DT>(a.q, b, 0, h / a.share);
        const auto* k = row_of<DT>(a.k, b, 0, h / a.share);
        const auto* v = row_of<DT>(a.v, b, 0, h);
        const float f = hw_exp(static_cast<const float*>(a.g.p)[b * a.g.bs + h * a.g.hs]);
        for (int p0 = 0; p0 < a.value; p0 += PV) {
            const int p = p0 + col;
            const bool in = p < a.value;
            float* st = a.state_out + bh * a.key * a.value + p;
            float vv[VEC], y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) vv[e] = in ? Elem<DT>::ld(v[p + e]) : 0.0f, y[e] = 0.0f;
            for (int n0 = row; n0 < a.key; n0 += ROWS * AT_ONCE) {
                float s[AT_ONCE][VEC], kn[AT_ONCE], qn[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int n = min(n0 + i * ROWS, a.key - 1);
                    kn[i] = Elem<DT>::ld(k[n]);
                    qn[i] = Elem<DT>::ld(q[n]);
                    if (in) ld_vec<DT_F32, VEC>(st + (int64_t)n * a.value, s[i]);
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int n = n0 + i * ROWS;
                    if (n >= a.key || !in) continue;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        s[i][e] = __builtin_fmaf(f, s[i][e], kn[i] * vv[e]);
                        y[e] = __builtin_fmaf(qn[i], s[i][e], y[e]);
                    }
                    st_vec<DT_F32, VEC>(st + (int64_t)n * a.value, s[i]);
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                for (int o = 32; o >= LANES; o >>= 1) y[e] += __shfl_xor(y[e], o, 64);
            if (lane < LANES)
#pragma unroll
                for (int e = 0; e < VEC; ++e) part[wave][col + e] = y[e];
            __syncthreads();
            if (threadIdx.x < PV && p0 + (int)threadIdx.x < a.value) {
                const int c = threadIdx.x;
                row_of<DT>(a.y, b, 0, h)[p0 + c] = Elem<DT>::st(a.scale * ((part[0][c] + part[1][c]) + (part[2][c] + part[3][c])));
            }
            __syncthreads();
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------
Heads heads_of(const boa_heads& x) { return {x.p, x.batch_stride, x.row_stride, x.head_stride}; }

bool wide_rows(int dtype, const boa_heads& x, int cols) {
    const int64_t es = dtype == DT_F32 ? 4 : 2;
    return ((uintptr_t)x.p | (uintptr_t)(x.batch_stride * es) | (uintptr_t)(x.row_stride * es) | (uintptr_t)(x.head_stride * es) |
            (uintptr_t)(cols * es)) % 16 == 0;
}

// The split: pieces of whole chunks, as many as give the wanted workgroups.
constexpr int64_t WANTED = 1024;
struct Plan {
    int np, tiles;
    int64_t chunks, bh;
    int32_t pieces, per_piece;
    explicit Plan(const boa_attention& s) {
        np = s.key <= 64 ? 64 : 128;
        tiles = (int)ceil_div(s.value, PV);
        chunks = ceil_div(s.length, CHUNK);
        bh = s.batch * s.heads;
        const int64_t each = bh * tiles;
        int64_t n = each > 0 ? ceil_div(WANTED, each) : 1;
        n = n < chunks ? n : chunks;
        per_piece = (int32_t)(n > 1 ? ceil_div(chunks, n) : chunks > 1 ? chunks : 1);
        pieces = (int32_t)(chunks > 1 ? ceil_div(chunks, per_piece) : 1);
    }
    int64_t state() const { return (int64_t)np * PV; }
    int64_t marks() const { return bh * tiles * chunks * state(); }
    int64_t starts() const { return pieces > 1 ? bh * tiles * pieces * state() : 0; }
    int64_t states_bytes() const { return 4 * (marks() + starts()) + (pieces > 1 ? (4 * bh * chunks + 8 * bh * pieces + 15) / 16 * 16 : 0); }
    // [marks][starts][fall][pre] from p on
    void place(Args& a, void* p) const {
        a.marks = static_cast<float*>(p);
        a.starts = a.marks + marks();
        a.fall = reinterpret_cast<double*>(a.starts + starts());
        a.pre = pieces > 1 ? reinterpret_cast<float*>(a.fall + bh * pieces) : nullptr;
    }
};

bool parts_wanted(const boa_attention& s, const Plan& p) { return s.heads / s.groups * p.tiles > 1; }

int64_t bwd_bytes(const boa_attention& s, const Plan& p) {
    int64_t n = p.states_bytes();
    if (parts_wanted(s, p)) n += 2 * 4 * s.batch * s.length * s.heads * p.tiles * s.key;
    if (s.decay_per_head) n += 4 * s.batch * p.chunks * p.tiles * s.heads;
    else if (p.tiles > 1) n += 4 * p.tiles * s.batch * s.length * s.heads;
    return n;
}

int check_sizes(const char* who, const boa_attention* s) {
    if (!s) return boa_fail(BOA_ERR_ARG, "%s: null pointer", who);
    if (s->dtype < BOA_DT_F32 || s->dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, s->dtype);
    if (s->batch < 0 || s->length < 0 || s->heads < 1 || s->groups < 1 || s->heads % s->groups || s->heads > BOA_ATTENTION_MAX_HEADS)
        return boa_fail(BOA_ERR_ARG, "%s: need batch, length >= 0 and heads (up to %d) a multiple of groups (got %lld, %lld, %d, %d)", who,
                        BOA_ATTENTION_MAX_HEADS, (long long)s->batch, (long long)s->length, s->heads, s->groups);
    if (s->key < 1 || s->key > MAX_KEY || s->value < 1 || s->value > MAX_VALUE)
        return boa_fail(BOA_ERR_ARG, "%s: need 1 <= key <= %d and 1 <= value <= %d (got %d, %d)", who, MAX_KEY, MAX_VALUE, s->key, s->value);
    // a launch takes so many workgroups, one for each chunk of a head and 64 of its values
    const int64_t each = ceil_div(s->value, PV) * s->heads;
    if (s->batch > MAX_BLOCKS / each || (s->batch > 0 && ceil_div(s->length, CHUNK) > MAX_BLOCKS / (each * s->batch)))
        return boa_fail(BOA_ERR_ARG, "%s: %lld sequences of %lld positions and %d heads are too many for a launch", who, (long long)s->batch,
                        (long long)s->length, s->heads);
    return BOA_OK;
}

Args args_of(const boa_attention& s, const Plan& p) {
    Args a = {};
    a.q = heads_of(s.q), a.k = heads_of(s.k), a.v = heads_of(s.v), a.y = heads_of(s.y), a.dy = heads_of(s.dy), a.dq = heads_of(s.dq);
    a.dk = heads_of(s.dk), a.dv = heads_of(s.dv);
    a.g = {const_cast<float*>(s.decay), s.decay_per_head ? 0 : s.decay_batch_stride, s.decay_per_head ? 0 : s.decay_row_stride,
           s.decay_per_head ? 1 : s.decay_head_stride};
    a.lens = s.lens, a.state_in = s.state_in, a.state_out = s.state_out;
    a.batch = s.batch, a.length = s.length, a.chunks = p.chunks;
    a.heads = s.heads, a.share = s.heads / s.groups, a.key = s.key, a.value = s.value, a.tiles = p.tiles;
    a.pieces = p.pieces, a.per_piece = p.per_piece, a.scale = s.scale;
    const struct {
        uint32_t bit;
        const boa_heads& x;
        int cols;
    } all[] = {{W_Q, s.q, s.key}, {W_K, s.k, s.key}, {W_V, s.v, s.value}, {W_DY, s.dy, s.value}, {W_Y, s.y, s.value}, {W_DQ, s.dq, s.key},
               {W_DK, s.dk, s.key}, {W_DV, s.dv, s.value}};
    for (const auto& t : all)
        if (wide_rows(s.dtype, t.x, t.cols)) a.wide |= t.bit;
    return a;
}

// Kernels whose LDS passes 64 KB are told so, once per kernel and device (the call is of no stream and may run under capture).
template <class K>
int allow_lds(K* kernel, int bytes) {
    BOA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return BOA_OK;
}

template <class F>
int with_key(int np, F f) {
    return np == 64 ? f(std::integral_constant<int, 64>()) : f(std::integral_constant<int, 128>());
}

// The states before every chunk (backward: their gradients behind it).
template <int DT, int NP, bool BACK>
int launch_states(const Args& a, const Plan& p, hipStream_t s) {
    hipLaunchKernelGGL((k_attn_states<DT, NP, BACK>), dim3((uint32_t)(p.bh * p.tiles * p.pieces)), dim3(WG), 0, s, a);
    BOA_HIP_TRY(hipGetLastError());
    if (p.pieces > 1) {
        hipLaunchKernelGGL((k_attn_join<NP, BACK>), dim3((uint32_t)(p.bh * p.tiles * (State<NP>::SIZE / (WG * 4)))), dim3(WG), 0, s, a);
        BOA_HIP_TRY(hipGetLastError());
    }
    return BOA_OK;
}

}  // namespace

extern "C" int64_t boa_linear_attention_work_bytes(const boa_attention* s, int backward) {
    if (check_sizes("boa_linear_attention_work_bytes", s) != BOA_OK) return -1;
    const Plan p(*s);
    return backward ? bwd_bytes(*s, p) : p.states_bytes();
}

extern "C" int boa_linear_attention_fwd(const boa_attention* s, void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_sizes("boa_linear_attention_fwd", s);
    if (rc != BOA_OK) return rc;
    if (s->batch == 0) return BOA_OK;
    if (!s->decay || (s->length > 0 && (!s->q.p || !s->k.p || !s->v.p || !s->y.p)))
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_fwd: null pointer");
    const Plan p(*s);
    if (p.states_bytes() > 0 && (!d_work || (uintptr_t)d_work % 16 || work_bytes < p.states_bytes()))
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_fwd: workspace of %lld bytes, needs %lld at a multiple of 16", (long long)work_bytes,
                        (long long)p.states_bytes());
    Args a = args_of(*s, p);
    p.place(a, d_work);
    return with_dtype(s->dtype, [&](auto dt) {
        return with_key(p.np, [&](auto np) {
            constexpr int DT = decltype(dt)::value, NP = decltype(np)::value;
            const int done = launch_states<DT, NP, false>(a, p, (hipStream_t)stream);
            if (done != BOA_OK || p.chunks == 0) return done;
            constexpr int LDS = fwd_lds<DT, NP>();
            if (const int no = allow_lds(k_attn_fwd<DT, NP>, LDS)) return no;
            hipLaunchKernelGGL((k_attn_fwd<DT, NP>), dim3((uint32_t)(p.bh * p.tiles * p.chunks)), dim3(WG), LDS, (hipStream_t)stream, a);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
    });
}

extern "C" int boa_linear_attention_bwd(const boa_attention* s, const void* d_fwd_work, int64_t fwd_work_bytes, void* d_work, int64_t work_bytes,
                                        void* stream) {
    const int rc = check_sizes("boa_linear_attention_bwd", s);
    if (rc != BOA_OK) return rc;
    const Plan p(*s);
    if (!s->decay || !s->ddecay) return boa_fail(BOA_ERR_ARG, "boa_linear_attention_bwd: null pointer");
    const int64_t need = bwd_bytes(*s, p);
    hipStream_t st = (hipStream_t)stream;
    if (s->batch == 0 || s->length == 0) {
        if (s->decay_per_head) BOA_HIP_TRY(launch_sum_parts(nullptr, 0, s->heads, s->ddecay, st));
        return BOA_OK;
    }
    if (!s->q.p || !s->k.p || !s->v.p || !s->dy.p || !s->dq.p || !s->dk.p || !s->dv.p)
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_bwd: null pointer");
    if (!d_fwd_work || fwd_work_bytes < p.states_bytes() || !d_work || work_bytes < need || ((uintptr_t)d_fwd_work | (uintptr_t)d_work) % 16)
        return boa_fail(BOA_ERR_ARG,
                        "boa_linear_attention_bwd: workspaces of %lld (the forward's) and %lld bytes, needs %lld and %lld at multiples of 16",
                        (long long)fwd_work_bytes, (long long)work_bytes, (long long)p.states_bytes(), (long long)need);
    Args a = args_of(*s, p);
    p.place(a, const_cast<void*>(d_fwd_work));
    a.fmarks = a.marks, a.fstarts = a.starts, a.fpre = a.pre;
    p.place(a, d_work);
    a.state_in = nullptr, a.state_out = nullptr;
    float* rest = reinterpret_cast<float*>(static_cast<char*>(d_work) + p.states_bytes());
    if (parts_wanted(*s, p)) {
        const int64_t each = s->batch * s->length * s->heads * p.tiles * s->key;
        a.part_q = rest, a.part_k = rest + each;
        rest += 2 * each;
    }
    if (s->decay_per_head) a.dg_sum = rest;
    else a.dg = p.tiles > 1 ? rest : s->ddecay;
    return with_dtype(s->dtype, [&](auto dt) {
        return with_key(p.np, [&](auto np) {
            constexpr int DT = decltype(dt)::value, NP = decltype(np)::value;
            const int done = launch_states<DT, NP, true>(a, p, st);
            if (done != BOA_OK) return done;
            constexpr int LDS = bwd_lds<DT, NP>();
            if (const int no = allow_lds(k_attn_bwd<DT, NP>, LDS)) return no;
            hipLaunchKernelGGL((k_attn_bwd<DT, NP>), dim3((uint32_t)(p.bh * p.tiles * p.chunks)), dim3(WG), LDS, st, a);
            BOA_HIP_TRY(hipGetLastError());
            if (a.part_q != nullptr) {
                const int64_t n = ceil_div(s->batch * s->length * s->groups * s->key, WG);
                const dim3 grid((uint32_t)(n < MAX_BLOCKS ? n : MAX_BLOCKS));
                hipLaunchKernelGGL((k_attn_sum<DT>), grid, dim3(WG), 0, st, a, a.part_q, a.dq, s->groups);
                BOA_HIP_TRY(hipGetLastError());
                hipLaunchKernelGGL((k_attn_sum<DT>), grid, dim3(WG), 0, st, a, a.part_k, a.dk, s->groups);
                BOA_HIP_TRY(hipGetLastError());
            }
            if (a.dg_sum != nullptr) {
                BOA_HIP_TRY(launch_sum_parts(a.dg_sum, s->batch * p.chunks * p.tiles, s->heads, s->ddecay, st));
            } else if (p.tiles > 1) {
                const int64_t n = s->batch * s->length * s->heads, blocks = ceil_div(n, WG);
                hipLaunchKernelGGL(k_attn_sum_tiles, dim3((uint32_t)(blocks < MAX_BLOCKS ? blocks : MAX_BLOCKS)), dim3(WG), 0, st, a.dg, s->ddecay, n,
                                   p.tiles);
                BOA_HIP_TRY(hipGetLastError());
            }
            return (int)BOA_OK;
        });
    });
}

extern "C" int boa_linear_attention_step(const boa_attention* s, void* stream) {
    const int rc = check_sizes("boa_linear_attention_step", s);
    if (rc != BOA_OK) return rc;
    if (s->length != 1) return boa_fail(BOA_ERR_ARG, "boa_linear_attention_step: length %lld (one position)", (long long)s->length);
    if (s->batch == 0) return BOA_OK;
    if (!s->q.p || !s->k.p || !s->v.p || !s->y.p || !s->decay || !s->state_out)
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_step: null pointer");
    const Plan p(*s);
    const Args a = args_of(*s, p);
    const bool vec = s->value % 4 == 0 && (uintptr_t)s->state_out % 16 == 0;
    const dim3 grid((uint32_t)(p.bh < MAX_BLOCKS ? p.bh : MAX_BLOCKS));
    return with_dtype(s->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (vec) hipLaunchKernelGGL((k_attn_step<DT, 4>), grid, dim3(WG), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((k_attn_step<DT, 1>), grid, dim3(WG), 0, (hipStream_t)stream, a);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}
