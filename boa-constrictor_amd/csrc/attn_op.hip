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
// Forward, a workgroup walks a piece of the length with the state in registers; where the length is split, a first kernel finds
// what each piece leaves by itself, and a small one joins them.  Backward, the gradients of the states behind every chunk are laid
// down by a walk from the end, and then every chunk is done by itself.
//
// Everywhere a wavefront has 16 columns of a product's result: its own 16 positions i (or j) in what is made of A and dA, so that
// these stay in its registers, where a result tile (column in the lane, four consecutive rows per lane) is the next product's
// operand as it is; its own 16 of every 64 keys in a state.
//
// Measured with 64 keys and 64 values a head (copies of the sizes moved here reach 5 to 6 TB/s, float32 products of libraries 150
// TFLOP/s), kernels in us; 4 x 4097 positions x 16 heads of 16 groups in bfloat16: states 21, joined 6, forward 59 (136 MB and as
// much of k and v again); 2 x 16384 x 8 heads in float32: forward 38 + 7 + 112, backward 44 + 7 + 219 (539 MB, and 22 GFLOP of
// products that are needed, 149 us at the libraries' rate; 27 are done, with the scores in both orientations and k and v walked
// twice); 32 x up to 500 x 16 heads of 4 groups in bfloat16: forward 44 to 52, backward 18 to 20 + 126; one position of 1000 x 16
// heads: 83 (532 MB, 6.4 TB/s).  What bounds each stands at its kernel.
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
    float* marks;   // [batch heads][value tiles][chunks][NP * PV]: forward (or null) the states before the chunks, backward what lies
                    // behind each chunk of its piece adds to the gradient of the state behind it
    float* starts;  // [batch heads][value tiles][pieces][NP * PV] what each piece leaves, then what it starts from (pieces > 1)
    float* pre;     // backward: [batch heads][chunks] decay from the chunk's end to its piece's
    double* fall;   // [batch heads][pieces] log2 of the piece's decay
    const float* fmarks;     // backward: the forward's
    float *part_q, *part_k;  // backward: [batch][length][groups][parts][key], or null: dq, dk are written
    float* dg;               // backward: [value tiles][batch][length][heads], or null
    float* dg_sum;           // backward: [batch * chunks * value tiles][heads], or null
    int64_t batch, length, chunks;
    int32_t heads, share, parts, key, value, tiles, pieces, per_piece;
    float scale;
};

// How products of a type run: elements in LDS, K of a step, parts that a float32 value is split into.
//   bfloat16: inputs as they are.  What is computed on the way (A, dA, states, decayed keys) is split into three parts of 8 bits
//   each, float32's 24: with two, terms that cancel would leave an error beyond the result's own rounding.
//   float32 and float16: float32 products (v_mfma_f32_16x16x4_f32).  Parts of A, dA and states do not fit float16's range; q . k and
//   dy . v, whose operands are float16, would fit its products but are made like the rest.
// A fragment holds VEC elements along K per lane: `row` of a tile with K along memory, `col` of one with K across; element e of lane
// group g is k = VEC g + e.  `mixed` is `col` in the order of register tiles, k = 16 (e / 4) + 4 g + e % 4: element e of
// `registers` is row 4 g + e % 4 of tile e / 4 of a result.
template <int DT> struct Mat {
    using E = float;
    using Frag = f32x4;
    static constexpr int STEP = 16, VEC = 4, PARTS = 1, PAD = 4;
    static constexpr bool SKIP = true;  // all-zero tiles are left out (2 x 16384 x 8 backward 293 -> 254 us)
    static __device__ __forceinline__ floatx4 mma(const Frag& a, const Frag& b, floatx4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag row(const E* t, int ld, int row0, int k0, int lane) {
        return *reinterpret_cast<const Frag*>(t + (row0 + (lane & 15)) * ld + k0 + (lane >> 4) * VEC);
    }
    static __device__ __forceinline__ Frag col(const E* t, int ld, int row0, int k0, int lane) {
        const E* p = t + (k0 + (lane >> 4) * VEC) * ld + row0 + (lane & 15);
        return Frag{p[0], p[ld], p[2 * ld], p[3 * ld]};
    }
    static __device__ __forceinline__ Frag mixed(const E* t, int ld, int row0, int k0, int lane) { return col(t, ld, row0, k0, lane); }
    static __device__ __forceinline__ void widen(const Frag& f, float (&x)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[i] = f[i];
    }
    static __device__ __forceinline__ void split(const float (&x)[VEC], Frag (&f)[PARTS]) {
        f[0] = Frag{x[0], x[1], x[2], x[3]};
    }
    // An operand times a factor: all of it, or a power of two now and the rest of it (`behind`) times the product.
    static __device__ __forceinline__ Frag scaled(const Frag& f, float by) { return Frag{f[0] * by, f[1] * by, f[2] * by, f[3] * by}; }
    static __device__ __forceinline__ float behind(float) { return 1.0f; }
    static __device__ __forceinline__ floatx4 load4(const E* p) { return *reinterpret_cast<const floatx4*>(p); }
    static __device__ __forceinline__ float value(E v) { return v; }
    // zeros in the place of infinities and NaN
    static __device__ __forceinline__ Frag finite(Frag f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __builtin_isfinite(f[i]) ? f[i] : 0.0f;
        return f;
    }
};
typedef short s16x4 __attribute__((ext_vector_type(4)));
// Parts of float32 values: the upper halves, cut off rather than rounded, so that three of them are the value itself, and finite where it
// is finite.
__device__ __forceinline__ uint32_t uppers(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }
// What is left of f behind its upper half; nothing behind an infinite one.
__device__ __forceinline__ float rest(float f) {
    const float r = f - __uint_as_float(__float_as_uint(f) & 0xFFFF0000u);
    return fabsf(f) == __builtin_inff() ? 0.0f : r;
}
template <> struct Mat<DT_BF16> {
    using E = uint16_t;
    using Frag = bf16x8;
    static constexpr int STEP = 32, VEC = 8, PARTS = 3, PAD = 8;
    static constexpr bool SKIP = false;  // a step is two tiles, and takes an eighth of float32's time a tile
    static __device__ __forceinline__ floatx4 mma(const Frag& a, const Frag& b, floatx4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag row(const E* t, int ld, int row0, int k0, int lane) {
        return *reinterpret_cast<const Frag*>(t + (row0 + (lane & 15)) * ld + k0 + (lane >> 4) * VEC);
    }
    // The transposing read: of 16 lanes, lane i gives the address of 4 elements of row i / 4 at column 4 (i % 4) and gets column i of
    // the four rows.
    static __device__ __forceinline__ Frag across(const E* t, int ld, int row0, int k, int apart, int lane) {
        const int l = lane & 15;
        const E* p = t + (k + (l >> 2)) * ld + row0 + (l & 3) * 4;
        using P = __attribute__((address_space(3))) s16x4*;
        struct {
            s16x4 a, b;
        } r = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((P)p), __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(p + apart * ld))};
        return __builtin_bit_cast(Frag, r);
    }
    static __device__ __forceinline__ Frag col(const E* t, int ld, int row0, int k0, int lane) {
        return across(t, ld, row0, k0 + (lane >> 4) * VEC, 4, lane);
    }
    static __device__ __forceinline__ Frag mixed(const E* t, int ld, int row0, int k0, int lane) {
        return across(t, ld, row0, k0 + (lane >> 4) * 4, 16, lane);
    }
    static __device__ __forceinline__ void widen(const Frag& f, float (&x)[VEC]) { Raw<DT_BF16, VEC>::unpack(__builtin_bit_cast(u32x4, f), x); }
    static __device__ __forceinline__ void split(const float (&x)[VEC], Frag (&f)[PARTS]) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = x[i];
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = uppers(v[2 * i], v[2 * i + 1]);
                v[2 * i] = rest(v[2 * i]);
                v[2 * i + 1] = rest(v[2 * i + 1]);
            }
            f[s] = __builtin_bit_cast(Frag, w);
        }
    }
    // A power of two leaves a bfloat16 value one, down to the smallest ones.
    static __device__ __forceinline__ Frag scaled(const Frag& f, float by) {
        const float two = __uint_as_float(__float_as_uint(by) & 0x7F800000u);
        u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = uppers(__uint_as_float(w[i] << 16) * two, __uint_as_float(w[i] & 0xFFFF0000u) * two);
        return __builtin_bit_cast(Frag, w);
    }
    static __device__ __forceinline__ float behind(float by) {
        return by == by ? __uint_as_float((__float_as_uint(by) & 0x807FFFFFu) | 0x3F800000u) : by;
    }
    static __device__ __forceinline__ floatx4 load4(const E* p) {
        float v[4];
        ld_vec<DT_BF16, 4>(p, v);
        return floatx4{v[0], v[1], v[2], v[3]};
    }
    static __device__ __forceinline__ float value(E v) { return Elem<DT_BF16>::ld(v); }
    static __device__ __forceinline__ Frag finite(const Frag& f) {
        u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] &= ((w[i] & 0x7F80u) != 0x7F80u ? 0xFFFFu : 0u) | ((w[i] & 0x7F800000u) != 0x7F800000u ? 0xFFFF0000u : 0u);
        return __builtin_bit_cast(Frag, w);
    }
};
// Step s of a product over 64 positions whose second operand is in registers, four tiles of 16 rows.
template <class M>
__device__ __forceinline__ void registers(const floatx4 (&t)[4], int s, typename M::Frag (&f)[M::PARTS]) {
    float x[M::VEC];
#pragma unroll
    for (int e = 0; e < M::VEC; ++e) {
        x[e] = t[s * (M::VEC / 4) + e / 4][e % 4];
        if (M::PARTS > 1) asm volatile("" : "+v"(x[e]));  // else the splits of all steps are made ahead, and kept
    }
    M::split(x, f);
}
// Row k (the same for all lanes) of the lane's column of a register operand of four tiles.
__device__ __forceinline__ float row_of_tiles(const floatx4 (&t)[4], int k, int lane) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if ((k >> 4) * 4 + (k & 3) == i) x = t[i / 4][i % 4];
    return __shfl(x, 16 * ((k >> 2) & 3) + (lane & 15), 64);
}

// acc[ta] += A B over 64 positions k: A's rows from 0 on, held across in LDS; B (16 columns) in registers, four tiles of 16 k, of which
// those from `first` to `last` are not all zero.  inside(k) says whether B's k of this lane's column counts; B is zero where it
// does not.  If A has infinities or NaN (it is not `finite`), those times such zeros would be NaN, and a position would reach others
// that it comes behind: they are left out of the product and added one by one, so that whatever they do not reach keeps its bits.
template <class M, int TA, class F>
__device__ __forceinline__ void product_within(floatx4 (&acc)[TA], bool finite, const typename M::E* a, int lda, const floatx4 (&b)[4],
                                               int first, int last, int lane, F inside) {
    const auto all = [&](auto clean) {
#pragma unroll
        for (int s = 0; s < CHUNK / M::STEP; ++s) {
            if (M::SKIP && (s < first || s > last)) continue;  // a step is a tile there
            typename M::Frag fb[M::PARTS];
            registers<M>(b, s, fb);
#pragma unroll
            for (int i = 0; i < TA; ++i) {
                const typename M::Frag fa = clean(M::mixed(a, lda, 16 * i, s * M::STEP, lane));
#pragma unroll
                for (int p = 0; p < M::PARTS; ++p) acc[i] = M::mma(fa, fb[p], acc[i]);
            }
        }
    };
    if (finite) return all([](const typename M::Frag& f) { return f; });
    all([](const typename M::Frag& f) { return M::finite(f); });
#pragma unroll 1
    for (int k = 16 * first; k < 16 * last + 16; ++k) {
        const float w = row_of_tiles(b, k, lane);
        const bool in = inside(k);
#pragma unroll
        for (int i = 0; i < TA; ++i) {
            const floatx4 x = M::load4(a + k * lda + 16 * i + 4 * (lane >> 4));
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][r] = in && !__builtin_isfinite(x[r]) ? __builtin_fmaf(x[r], w, acc[i][r]) : acc[i][r];
        }
    }
}
// The products of 16 columns (rows `own` .. of b) with the tiles from `first` to `last` of a's rows, both held along K.
template <class M, int K>
__device__ __forceinline__ void scores(floatx4 (&acc)[4], const typename M::E* a, const typename M::E* b, int ld, int own, int first, int last,
                                       int lane) {
    typename M::Frag fb[K / M::STEP];
#pragma unroll
    for (int s = 0; s < K / M::STEP; ++s) fb[s] = M::row(b, ld, own, s * M::STEP, lane);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        if (M::SKIP && (t < first || t > last)) continue;
#pragma unroll
        for (int s = 0; s < K / M::STEP; ++s) acc[t] = M::mma(M::row(a, ld, 16 * t, s * M::STEP, lane), fb[s], acc[t]);
    }
}

// Four consecutive values into LDS, in parts that are `part` elements apart.
template <class M>
__device__ __forceinline__ void put4(typename M::E* p, int part, floatx4 v) {
    if constexpr (sizeof(typename M::E) == 4) {
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
        for (int s = 0; s < M::PARTS; ++s) {
            const u32x2 w = {uppers(v[0], v[1]), uppers(v[2], v[3])};
            *reinterpret_cast<u32x2*>(p + s * part) = w;
            v = floatx4{rest(v[0]), rest(v[1]), rest(v[2]), rest(v[3])};
        }
    }
}

// The same number (uniform), which the compiler takes for another one: what is computed from it stays where it is written.  Masks of
// the columns that a head has would otherwise be made before a loop over chunks and be kept, more than there are scalar registers.
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+s"(x));
    return x;
}

// The same for a lane's number: addresses and masks that are made from it.
__device__ __forceinline__ int here_lane(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// 16 bytes at any element's address: the hardware takes them as it takes aligned ones.
typedef u32x4 AnyAt __attribute__((aligned(2)));
// The value without its first n elements of ES bytes (fewer than 16 bytes); zeros behind.
template <int ES>
__device__ __forceinline__ u32x4 shifted(u32x4 v, int n) {
    if (n & (8 / ES)) v = u32x4{v[2], v[3], 0u, 0u};
    if (n & (4 / ES)) v = u32x4{v[1], v[2], v[3], 0u};
    if constexpr (ES == 2)
        if (n & 1)
            v = u32x4{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16),
                      v[3] >> 16};
    return v;
}

// A tile of CHUNK rows and COLS columns on its way from memory to LDS; zeros behind the last row and column.
template <int DT, int COLS>
struct Tile {
    using M = Mat<DT>;
    using T = typename Elem<DT>::T;
    static constexpr int V = wide<DT>(), PER = CHUNK * COLS / (WG * V), ROW = COLS / V;  // accesses of a thread, of a row
    static_assert(WG % ROW == 0, "");
    static constexpr int LD = COLS + M::PAD, SIZE = CHUNK * LD;
    u32x4 v[PER];
    // rows from p on, `rows` and `cols` of them; EVEN: cols are a multiple of V.  A row's last access, where it would pass the row's
    // end, is one that ends there, shifted down.  On the same data (all cases above) that takes 1 to 30% longer than EVEN, and
    // element by element 1.5 to 2.7 times as long.
    template <bool EVEN>
    __device__ __forceinline__ void load(const T* p, int64_t stride, int rows, int cols, int tid) {
        const int r0 = tid / ROW, c = tid % ROW * V;  // WG / ROW rows apart
        p += r0 * stride + c;
        if (EVEN && rows == CHUNK && cols == COLS) {
#pragma unroll
            for (int i = 0; i < PER; ++i) v[i] = *reinterpret_cast<const AnyAt*>(p + i * (WG / ROW * stride));
            return;
        }
        cols = here(cols);
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = u32x4{0u, 0u, 0u, 0u};
        if (c >= cols) return;
        if (EVEN || cols >= V) {
            const int over = EVEN ? 0 : max(c + V - cols, 0);
            p -= over;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (r0 + i * (WG / ROW) < rows) v[i] = *reinterpret_cast<const AnyAt*>(p + i * (WG / ROW * stride));
            if constexpr (!EVEN)
#pragma unroll
                for (int i = 0; i < PER; ++i) v[i] = shifted<sizeof(T)>(v[i], over);
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const T* q = p + i * (WG / ROW * stride);
                if (r0 + i * (WG / ROW) < rows)
#pragma unroll
                    for (int e = 0; e < V - 1; ++e)
                        if (e < cols) {
                            if constexpr (sizeof(T) == 4) v[i][e] = __float_as_uint(q[e]);
                            else v[i][e / 2] |= (uint32_t)q[e] << (16 * (e & 1));
                        }
                __builtin_amdgcn_sched_barrier(0);  // else all elements' loads are on their way at once, in registers of their own
            }
        }
    }
    // An exponent of ones and one more carry into the sign's place.
    __device__ __forceinline__ bool finite() const {
        constexpr uint32_t SIGNS = DT == DT_F32 ? 0x80000000u : 0x80008000u, ONE = DT == DT_F32 ? 0x00800000u : DT == DT_BF16 ? 0x00800080u : 0x04000400u;
        uint32_t any = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= (v[i][e] & ~SIGNS) + ONE;
        return (any & SIGNS) == 0u;
    }
    __device__ __forceinline__ void unpack(int i, float (&f)[V]) const {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if constexpr (DT == DT_F32) f[e] = __uint_as_float(v[i][e]);
            else f[e] = Elem<DT>::ld((uint16_t)(v[i][e / 2] >> (16 * (e & 1))));
        }
    }
    __device__ __forceinline__ void store(typename M::E* t, int tid) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = tid + i * WG, r = at / ROW, c = at % ROW * V;
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
};

// log2 of the decay from a chunk's start up to and with each position (lane), summed in 64 bits; a decay of zero (-inf) as
// 2^-200, which is zero in float32 whatever it is multiplied with, so that differences stay numbers.
__device__ __forceinline__ const float* decays_of(const Args& a, int64_t b, int h) {
    return static_cast<const float*>(a.g.p) + b * a.g.bs + h * a.g.hs;
}
// a position's own, and from it the sum
__device__ __forceinline__ float decay_at(const float* p, int64_t stride, int rows, int lane) { return lane < rows ? p[lane * stride] : 0.0f; }
__device__ __forceinline__ double decays(float own) {
    const double g = (double)own * LOG2E;
    return scan(g < -200.0 ? -200.0 : g);
}
__device__ __forceinline__ float2 in_two(double g) {
    const float hi = (float)g;
    return make_float2(hi, (float)(g - (double)hi));
}
// 2^(a - b)
__device__ __forceinline__ float fall_between(float2 a, float2 b) { return __builtin_amdgcn_exp2f((a.x - b.x) + (a.y - b.y)); }
// The sums of a chunk's logarithms in LDS, in two parts.
struct Falls {
    float x[CHUNK], y[CHUNK];
    __device__ __forceinline__ void put(int i, float2 g) { x[i] = g.x, y[i] = g.y; }
    __device__ __forceinline__ float2 at(int i) const { return make_float2(x[i], y[i]); }
};
// The factors between the own position and the four rows that a lane has of tile t: of the own one behind them, or of them behind it.
template <bool OWN_BEHIND>
__device__ __forceinline__ floatx4 falls(const Falls& g, float2 own, float scale, int lane, int t) {
    const int at = 16 * t + 4 * (lane >> 4);
    const f32x4 x = *reinterpret_cast<const f32x4*>(g.x + at), y = *reinterpret_cast<const f32x4*>(g.y + at);
    floatx4 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float2 o = make_float2(x[r], y[r]);
        f[r] = scale * (OWN_BEHIND ? fall_between(own, o) : fall_between(o, own));
    }
    return f;
}
// Whether all values that the workgroup's threads have are finite, by way of a barrier: each wavefront says so in LDS, of one set of
// values or (in bit 1) of two.
__device__ __forceinline__ void say_finite(int* said, bool finite, int lane, int wave, bool other = true) {
    const int all = (__ballot(!finite) == 0 ? 1 : 0) | (__ballot(!other) == 0 ? 2 : 0);
    if (lane == 0) said[wave] = all;
}
__device__ __forceinline__ int heard(const int* said) { return __builtin_amdgcn_readfirstlane(said[0] & said[1] & said[2] & said[3]); }
__device__ __forceinline__ bool heard_finite(const int* said) { return (heard(said) & 1) != 0; }

// Whether a pair of positions with this decay between them counts.  A score of finite values may pass float32's range and is nothing all
// the same behind a decay of zero; where an infinity or NaN is among the values that scores are made of (not FINITE), it is not.
template <bool FINITE>
__device__ __forceinline__ bool counts(float f) { return !FINITE || f != 0.0f; }
template <class F>
__device__ __forceinline__ void where_finite(bool finite, F f) {
    if (finite) f(std::true_type());
    else f(std::false_type());
}

__device__ __forceinline__ int64_t end_of(const Args& a, int64_t b) {
    if (a.lens == nullptr) return a.length;
    const int64_t n = a.lens[b];
    return n < 0 ? 0 : n < a.length ? n : a.length;
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T* row_of(const Heads& x, int64_t b, int64_t t, int h) {
    return static_cast<typename Elem<DT>::T*>(x.p) + b * x.bs + t * x.rs + h * x.hs;
}

// A state in a wavefront's registers: tile [tp][tn], value r of lane l is value 16 tp + 4 (l / 16) + r of key 64 tn + 16 wave + l % 16.
template <int NP>
struct State {
    static constexpr int TN = NP / 64, TP = PV / 16, SIZE = NP * PV;
    floatx4 v[TP][TN];
    static __device__ __forceinline__ int n(int tn, int lane, int wave) { return 64 * tn + 16 * wave + (lane & 15); }
    static __device__ __forceinline__ int p(int tp, int lane) { return 16 * tp + 4 * (lane >> 4); }
    static __device__ __forceinline__ int at(int tp, int tn, int lane, int wave) { return (((wave * TN + tn) * TP + tp) * 64 + lane) * 4; }
    template <class F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int i = 0; i < TP; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) f(i, j, v[i][j]);
    }
    __device__ __forceinline__ void zero() {
        each([](int, int, floatx4& x) { x = floatx4{0.0f, 0.0f, 0.0f, 0.0f}; });
    }
    __device__ __forceinline__ void load(const float* m, int lane, int wave) {
        each([&](int i, int j, floatx4& x) { x = *reinterpret_cast<const floatx4*>(m + at(i, j, lane, wave)); });
    }
    __device__ __forceinline__ void add(const float* m, float f, int lane, int wave) {
        each([&](int i, int j, floatx4& x) {
            const floatx4 y = *reinterpret_cast<const floatx4*>(m + at(i, j, lane, wave));
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = __builtin_fmaf(f, y[r], x[r]);
        });
    }
    __device__ __forceinline__ void store(float* m, int lane, int wave) {
        each([&](int i, int j, floatx4& x) { *reinterpret_cast<floatx4*>(m + at(i, j, lane, wave)) = x; });
    }
    // the caller's [key][value]
    __device__ __forceinline__ void from_caller(const float* s, int key, int value, int p0, int lane, int wave) {
        each([&](int i, int j, floatx4& x) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n(j, lane, wave) < key && p0 + p(i, lane) + r < value) x[r] = s[n(j, lane, wave) * value + p0 + p(i, lane) + r];
        });
    }
    __device__ __forceinline__ void to_caller(float* s, int key, int value, int p0, int lane, int wave) {
        each([&](int i, int j, floatx4& x) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n(j, lane, wave) < key && p0 + p(i, lane) + r < value) s[n(j, lane, wave) * value + p0 + p(i, lane) + r] = x[r];
        });
    }
    // Into LDS as [key][value], zeros (which what lies behind key and value need not be) behind them.
    template <class M>
    __device__ __forceinline__ void put(typename M::E* t, int key, int value, int lane, int wave) {
        constexpr int LD = PV + M::PAD;
        if (key == NP && value == PV) {
            each([&](int i, int j, floatx4& x) { put4<M>(t + n(j, lane, wave) * LD + p(i, lane), NP * LD, x); });
            return;
        }
        key = here(key), value = here(value);
        each([&](int i, int j, floatx4& x) {
            floatx4 y = x;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (n(j, lane, wave) >= key || p(i, lane) + r >= value) y[r] = 0.0f;
            put4<M>(t + n(j, lane, wave) * LD + p(i, lane), NP * LD, y);
        });
    }
};

// One step of a state's update over STEP positions: s += (y)^T (x weight), y's fragments given; x (tile [position][key]) of the
// wavefront's own keys is weighted in registers.
template <class M, int NP, int LDX>
__device__ __forceinline__ void update(State<NP>& s, const typename M::Frag (&fy)[State<NP>::TP], const typename M::E* tx,
                                       const float* weight, int step, int lane, int wave) {
#pragma unroll
    for (int j = 0; j < State<NP>::TN; ++j) {
        float x[M::VEC];
        M::widen(M::mixed(tx, LDX, 64 * j + 16 * wave, step * M::STEP, lane), x);
#pragma unroll
        for (int e = 0; e < M::VEC; e += 4) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(weight + step * M::STEP + 4 * e + 4 * (lane >> 4));
#pragma unroll
            for (int c = 0; c < 4; ++c) x[e + c] *= w[c];
        }
        typename M::Frag fx[M::PARTS];
        M::split(x, fx);
#pragma unroll
        for (int i = 0; i < State<NP>::TP; ++i)
#pragma unroll
            for (int p = 0; p < M::PARTS; ++p) s.v[i][j] = M::mma(fy[i], fx[p], s.v[i][j]);
    }
}
// What infinities and NaN of y (tile [position][value]) add to it, where x's values are held in parts and zeros among these would make
// NaN of all of them.
template <class M, int NP, int LDX, int LDY>
__device__ __forceinline__ void update_odd(State<NP>& s, const typename M::E* ty, const typename M::E* tx, const float* weight, int lane,
                                           int wave) {
#pragma unroll 1
    for (int k = 0; k < CHUNK; ++k) {
        float w[State<NP>::TN];
#pragma unroll
        for (int j = 0; j < State<NP>::TN; ++j) w[j] = weight[k] * M::value(tx[k * LDX + 64 * j + 16 * wave + (lane & 15)]);
        s.each([&](int i, int j, floatx4& v) {
            const floatx4 y = M::load4(ty + k * LDY + 16 * i + 4 * (lane >> 4));
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = __builtin_isfinite(y[r]) ? v[r] : __builtin_fmaf(y[r], w[j], v[r]);
        });
    }
}
template <int NP>
__device__ __forceinline__ void times(State<NP>& s, float f) {
    s.each([&](int, int, floatx4& x) {
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] *= f;
    });
}

// ---- states by themselves ---------------------------------------------------------------------------
// A workgroup walks the chunks of a piece from a state of zeros, forward over k v^T or (BACK) from the last one over scale e^(G_i)
// q dy^T; leaves what it ends with, and backward also what it reaches each chunk with.  The state stays in registers; two
// workgroups on a CU hide each other's loads.  A chunk takes a workgroup about 2.4 us, of which a product of 64 x 64 x 64 is the
// smallest part: nothing is full (vector 58%, matrix 17%, LDS 24% of the cycles in bfloat16; 18, 47 and 22% in float32), it waits for
// the next chunk's loads and at two barriers (k and v at 3.2 TB/s in bfloat16, 3.5 in float32 over 2 x 16384 x 8).
template <int DT, int NP, bool BACK, bool EVEN>
__global__ void __launch_bounds__(WG, 2) k_attn_states(const Args a) {
    using M = Mat<DT>;
    using TX = Tile<DT, NP>;
    using TY = Tile<DT, PV>;
    using S = State<NP>;
    __shared__ __attribute__((aligned(16))) typename M::E tx[TX::SIZE];
    __shared__ __attribute__((aligned(16))) typename M::E ty[TY::SIZE];
    __shared__ __attribute__((aligned(16))) float weight[CHUNK];
    __shared__ int said[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int piece = (int)(blockIdx.x % a.pieces), tile = (int)(blockIdx.x / a.pieces % a.tiles);
    const int64_t bh = blockIdx.x / a.pieces / a.tiles, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t end = end_of(a, b);
    const int64_t c0 = (int64_t)piece * a.per_piece, c1 = min(c0 + a.per_piece, (end + CHUNK - 1) / CHUNK);
    const Heads &X = BACK ? a.q : a.k, &Y = BACK ? a.dy : a.v;
    const int vcols = min(PV, a.value - tile * PV);
    float* marks = a.marks + (bh * a.tiles + tile) * a.chunks * S::SIZE;

    S s;
    s.zero();
    double passed = 0.0;
    TX x;
    TY y;
    float g_own = 0.0f;
    const auto* xp = row_of<DT>(X, b, 0, h / a.share);
    const auto* yp = row_of<DT>(Y, b, 0, h) + tile * PV;
    const float* gp = decays_of(a, b, h);
    const auto fetch = [&](int64_t c, int tid) {
        const int64_t t0 = c * CHUNK;
        const int rows = (int)min((int64_t)CHUNK, end - t0);
        x.template load<EVEN>(xp + t0 * X.rs, X.rs, rows, a.key, tid);
        y.template load<EVEN>(yp + t0 * Y.rs, Y.rs, rows, vcols, tid);
        g_own = decay_at(gp + t0 * a.g.rs, a.g.rs, rows, tid & 63);
    };
    const int64_t n = c1 - c0;
    if (n > 0) fetch(BACK ? c1 - 1 : c0, threadIdx.x);
    for (int64_t m = 0; m < n; ++m) {
        const int tid = threadIdx.x;
        const int64_t c = BACK ? c1 - 1 - m : c0 + m;
        if constexpr (BACK) {
            s.store(marks + c * S::SIZE, lane, wave);
            if (a.pieces > 1 && tile == 0 && threadIdx.x == 0) a.pre[bh * a.chunks + c] = __builtin_amdgcn_exp2f((float)passed);
        }
        const double g = decays(g_own), all = last_lane(g);
        x.store(tx, tid);
        y.store(ty, tid);
        if (wave == 0) weight[lane] = BACK ? a.scale * __builtin_amdgcn_exp2f((float)g) : __builtin_amdgcn_exp2f((float)(all - g));
        if constexpr (M::PARTS > 1) say_finite(said, y.finite(), lane, wave);
        __syncthreads();
        const bool finite = M::PARTS == 1 || heard_finite(said);
        if (m + 1 < n) fetch(BACK ? c - 1 : c + 1, tid);
        passed += all;
        times(s, __builtin_amdgcn_exp2f((float)all));
        const auto all_steps = [&](auto clean) {
#pragma unroll
            for (int k = 0; k < CHUNK / M::STEP; ++k) {
                typename M::Frag fy[S::TP];
#pragma unroll
                for (int i = 0; i < S::TP; ++i) fy[i] = clean(M::mixed(ty, TY::LD, 16 * i, k * M::STEP, lane));
                update<M, NP, TX::LD>(s, fy, tx, weight, k, lane, wave);
            }
        };
        if (finite) {
            all_steps([](const typename M::Frag& f) { return f; });
        } else {
            all_steps([](const typename M::Frag& f) { return M::finite(f); });
            update_odd<M, NP, TX::LD, TY::LD>(s, ty, tx, weight, lane, wave);
        }
        __syncthreads();
    }
    if (a.pieces > 1) {
        s.store(a.starts + ((bh * a.tiles + tile) * a.pieces + piece) * S::SIZE, lane, wave);
        if (tile == 0 && threadIdx.x == 0) a.fall[bh * a.pieces + piece] = passed;
    }
}

// What each piece leaves by itself becomes the state that it starts from (backward: the gradient of the state behind it), eight
// pieces' loads at a time.  A thread has four values of a state.  Bound by the latency of loads that follow one another: 6 to 7 us
// for the 8 to 32 pieces that fill the card.
template <int NP, bool BACK>
__global__ void __launch_bounds__(WG) k_attn_join(const Args a) {
    using S = State<NP>;
    constexpr int PER = S::SIZE / (WG * 4), AT_ONCE = 8;
    const int part = (int)(blockIdx.x % PER);
    const int64_t bht = blockIdx.x / PER, bh = bht / a.tiles;
    const int tile = (int)(bht % a.tiles), lane = threadIdx.x & 63;
    const int block = part * (WG / 64) + (threadIdx.x >> 6);  // (wave * TN + tn) * TP + tp
    const int tp = block % S::TP, tn = block / S::TP % S::TN, wave = block / S::TP / S::TN;
    const int n = S::n(tn, lane, wave), p = tile * PV + S::p(tp, lane);
    float* at = a.starts + bht * a.pieces * S::SIZE + block * 256 + lane * 4;
    floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!BACK && a.state_in != nullptr)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n < a.key && p + r < a.value) s[r] = a.state_in[(bh * a.key + n) * a.value + p + r];
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
            if (n < a.key && p + r < a.value) a.state_out[(bh * a.key + n) * a.value + p + r] = s[r];
}

// Four consecutive columns of a row of a result.
template <int DT>
__device__ __forceinline__ void write4(typename Elem<DT>::T* p, int col, int cols, floatx4 v) {
    if (col + 4 <= cols) {
        using Any __attribute__((aligned(2))) = typename Raw<DT, 4>::V;
        const float f[4] = {v[0], v[1], v[2], v[3]};
        *reinterpret_cast<Any*>(p + col) = Raw<DT, 4>::pack(f);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (col + r < cols) p[col + r] = Elem<DT>::st(v[r]);
    }
}
// A row of dq or dk, where it is one head's own, or its part of a sum.
template <int DT, int NT>
__device__ __forceinline__ void write_key(float* part, typename Elem<DT>::T* out, int key, int row4, const floatx4 (&v)[NT]) {
    if (part != nullptr) {
#pragma unroll
        for (int n = 0; n < NT; ++n) write4<DT_F32>(part, 16 * n + row4, here(key), v[n]);
    } else if (key == 16 * NT) {
#pragma unroll
        for (int n = 0; n < NT; ++n) write4<DT>(out, 16 * n + row4, 16 * NT, v[n]);
    } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) write4<DT>(out, 16 * n + row4, here(key), v[n]);
    }
}
// Zeros in the columns col0 .. of the rows [from, to).
template <int DT>
__device__ __forceinline__ void zero_rows(const Heads& x, int64_t b, int h, int col0, int cols, int64_t from, int64_t to) {
#pragma unroll 1
    for (int64_t t = from + threadIdx.x / 64; t < to; t += WG / 64)
#pragma unroll 1
        for (int i = threadIdx.x % 64; i < cols; i += 64) row_of<DT>(x, b, t, h)[col0 + i] = Elem<DT>::st(0.0f);
}

// ---- forward ------------------------------------------------------------------------------------------
// A workgroup walks a piece with the state in registers, and lays it into LDS (in parts for bfloat16) for the product
// with q; the next chunk's q, k and v are loaded into registers while this one's products run.  Nothing is full: in bfloat16 (59 us, 2.3
// TB/s of inputs and results) vector work has 64% of the SIMDs' cycles (decays, splits into parts, masks), the matrix cores 19%, LDS
// 34%, 41% of that conflicts; in float32 the matrix cores are busy for 50%: 112 us for 7.0 GFLOP, 62 TFLOP/s.  The rest is waiting,
// at two barriers a chunk with two workgroups on a CU.
template <int DT, int NP>
struct FwdLds {
    using M = Mat<DT>;
    static constexpr int Q = 0, K = Tile<DT, NP>::SIZE, V = 2 * K, S = V + Tile<DT, PV>::SIZE, LDS_STATE = PV + M::PAD, PART = NP * LDS_STATE;
    static constexpr int BYTES = (int)sizeof(typename M::E) * (S + M::PARTS * PART);
};
template <int DT, int NP, bool EVEN>
__global__ void __launch_bounds__(WG, NP == 128 ? 1 : 2) k_attn_fwd(const Args a) {
    using M = Mat<DT>;
    using E = typename M::E;
    using Frag = typename M::Frag;
    using TN = Tile<DT, NP>;
    using TV = Tile<DT, PV>;
    using S = State<NP>;
    using L = FwdLds<DT, NP>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    E* tq = reinterpret_cast<E*>(lds) + L::Q;
    E* tk = reinterpret_cast<E*>(lds) + L::K;
    E* tv = reinterpret_cast<E*>(lds) + L::V;
    E* ts = reinterpret_cast<E*>(lds) + L::S;  // [NP][PV] in parts
    __shared__ __attribute__((aligned(16))) Falls G;
    __shared__ __attribute__((aligned(16))) float weight[CHUNK];
    __shared__ int said[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // a wavefront's own positions i: the later ones have more before them, so workgroups beside each other have them the other way round
    const int own = blockIdx.x & 1 ? WAVES - 1 - wave : wave;
    const int piece = (int)(blockIdx.x % a.pieces), tile = (int)(blockIdx.x / a.pieces % a.tiles);
    const int64_t bh = blockIdx.x / a.pieces / a.tiles, b = bh / a.heads;
    const int h = (int)(bh % a.heads);
    const int64_t end = end_of(a, b), bht = bh * a.tiles + tile;
    const int64_t c0 = (int64_t)piece * a.per_piece, c1 = min(c0 + a.per_piece, (end + CHUNK - 1) / CHUNK);
    const int vcols = min(PV, a.value - tile * PV);
    const int64_t behind = min((c0 + a.per_piece) * CHUNK, a.length);
    if (end < behind) zero_rows<DT>(a.y, b, h, tile * PV, vcols, max(end, c0 * CHUNK), behind);

    S s;
    s.zero();
    if (a.pieces > 1) s.load(a.starts + (bht * a.pieces + piece) * S::SIZE, lane, wave);
    else if (a.state_in != nullptr) s.from_caller(a.state_in + bh * a.key * a.value, a.key, a.value, tile * PV, lane, wave);
    TN q, k;
    TV v;
    float g_own = 0.0f;
    const auto* qp = row_of<DT>(a.q, b, 0, h / a.share);
    const auto* kp = row_of<DT>(a.k, b, 0, h / a.share);
    const auto* vp = row_of<DT>(a.v, b, 0, h) + tile * PV;
    const float* gp = decays_of(a, b, h);
    auto* yp = row_of<DT>(a.y, b, 0, h) + tile * PV;
    float* marks = a.marks == nullptr ? nullptr : a.marks + bht * a.chunks * S::SIZE;
    const auto fetch = [&](int64_t c, int tid) {
        const int64_t t0 = c * CHUNK;
        const int rows = (int)min((int64_t)CHUNK, end - t0);
        q.template load<EVEN>(qp + t0 * a.q.rs, a.q.rs, rows, a.key, tid);
        k.template load<EVEN>(kp + t0 * a.k.rs, a.k.rs, rows, a.key, tid);
        v.template load<EVEN>(vp + t0 * a.v.rs, a.v.rs, rows, vcols, tid);
        g_own = decay_at(gp + t0 * a.g.rs, a.g.rs, rows, tid & 63);
    };
    // a chunk's results are written while the next one is on: what has been stored late would be waited for with the next tiles
    using Out = Raw<DT, 4>;
    typename Out::V done[S::TP];
    const auto write = [&](int64_t t0, int tid) {
        const int row4 = 4 * ((tid & 63) >> 4);
        const int64_t t = t0 + 16 * own + (tid & 15);
        if (t >= end) return;
        auto* out = yp + t * a.y.rs + row4;
        using Any __attribute__((aligned(2))) = typename Out::V;
        if (vcols == PV) {
#pragma unroll
            for (int p = 0; p < S::TP; ++p) *reinterpret_cast<Any*>(out + 16 * p) = done[p];
        } else {
#pragma unroll
            for (int p = 0; p < S::TP; ++p) {
                const int cols = here(vcols) - 16 * p - row4;
                float v[4];
                Out::unpack(done[p], v);
                if (cols >= 4) *reinterpret_cast<Any*>(out + 16 * p) = done[p];
                else
#pragma unroll
                    for (int r = 0; r < 3; ++r)
                        if (r < cols) out[16 * p + r] = Elem<DT>::st(v[r]);
            }
        }
    };
    if (c0 < c1) fetch(c0, threadIdx.x);
    for (int64_t c = c0; c < c1; ++c) {
        const int tid = here_lane(threadIdx.x), lane = tid & 63, l15 = lane & 15, row4 = 4 * (lane >> 4);
        const int64_t t0 = c * CHUNK;
        const int rows = (int)min((int64_t)CHUNK, end - t0);
        const double g = decays(g_own), all = last_lane(g);
        q.store(tq, tid);
        k.store(tk, tid);
        v.store(tv, tid);
        s.template put<M>(ts, a.key, vcols, lane, wave);
        if (wave == 0) {
            G.put(lane, in_two(g));
            weight[lane] = __builtin_amdgcn_exp2f((float)(all - g));
        }
        say_finite(said, v.finite(), lane, wave, k.finite());
        __syncthreads();
        const int all_finite = heard(said);
        const bool finite = (all_finite & 1) != 0, finite_k = (all_finite & 2) != 0;
        if (c > c0) write(t0 - CHUNK, tid);
        if (marks != nullptr) s.store(marks + c * S::SIZE, lane, wave);
        if (c + 1 < c1) fetch(c + 1, tid);

        // q . k of all positions j (rows) and the own ones (columns), and what the state gives
        floatx4 A[4], y[S::TP];
        scores<M, NP>(A, tk, tq, TN::LD, 16 * own, 0, own, lane);
        __builtin_amdgcn_sched_barrier(0);
        const int i = 16 * own + l15;
        const float2 gi = G.at(i);
        const float from_start = a.scale * __builtin_amdgcn_exp2f(gi.x + gi.y);
#pragma unroll
        for (int p = 0; p < S::TP; ++p) y[p] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < NP; n += M::STEP) {
            const Frag fq = M::scaled(M::row(tq, TN::LD, 16 * own, n, lane), from_start);
#pragma unroll
            for (int p = 0; p < S::TP; ++p)
#pragma unroll
                for (int i = 0; i < M::PARTS; ++i) y[p] = M::mma(M::col(ts + i * L::PART, L::LDS_STATE, 16 * p, n, lane), fq, y[p]);
        }
        __builtin_amdgcn_sched_barrier(0);
        where_finite(finite_k, [&](auto clean) {  // a query that is not finite reaches its own position, with no decay
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const floatx4 f = falls<true>(G, gi, a.scale, lane, t);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * t + row4 + r;
                    const float x = A[t][r] * f[r];
                    A[t][r] = j <= i && i < rows && counts<decltype(clean)::value>(f[r]) ? x : 0.0f;
                }
            }
        });
#pragma unroll
        for (int p = 0; p < S::TP; ++p)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[p][r] *= M::behind(from_start);
        __builtin_amdgcn_sched_barrier(0);
        times(s, __builtin_amdgcn_exp2f((float)all));
        if (finite) {
#pragma unroll
            for (int k = 0; k < CHUNK / M::STEP; ++k) {
                Frag fv[S::TP], fa[M::PARTS];
#pragma unroll
                for (int p = 0; p < S::TP; ++p) fv[p] = M::mixed(tv, TV::LD, 16 * p, k * M::STEP, lane);
                if (!M::SKIP || k <= own) {
                    registers<M>(A, k, fa);
#pragma unroll
                    for (int p = 0; p < S::TP; ++p)
#pragma unroll
                        for (int x = 0; x < M::PARTS; ++x) y[p] = M::mma(fv[p], fa[x], y[p]);
                }
                __builtin_amdgcn_sched_barrier(0);
                update<M, NP, TN::LD>(s, fv, tk, weight, k, lane, wave);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            product_within<M>(y, false, tv, TV::LD, A, 0, own, lane, [&](int j) { return j <= i && i < rows; });
#pragma unroll
            for (int k = 0; k < CHUNK / M::STEP; ++k) {
                Frag fv[S::TP];
#pragma unroll
                for (int p = 0; p < S::TP; ++p) {
                    fv[p] = M::mixed(tv, TV::LD, 16 * p, k * M::STEP, lane);
                    if constexpr (M::PARTS > 1) fv[p] = M::finite(fv[p]);
                }
                update<M, NP, TN::LD>(s, fv, tk, weight, k, lane, wave);
            }
            if constexpr (M::PARTS > 1) update_odd<M, NP, TN::LD, TV::LD>(s, tv, tk, weight, lane, wave);
        }
#pragma unroll
        for (int p = 0; p < S::TP; ++p) {
            const float v[4] = {y[p][0], y[p][1], y[p][2], y[p][3]};
            done[p] = Out::pack(v);
        }
        __syncthreads();
    }
    if (c0 < c1) write((c1 - 1) * CHUNK, threadIdx.x);
    if (a.pieces == 1 && a.state_out != nullptr) s.to_caller(a.state_out + bh * a.key * a.value, a.key, a.value, tile * PV, lane, wave);
}

// ---- backward, a chunk --------------------------------------------------------------------------------
// The sum of v over the lanes of a tile's column; every lane gets its column's.
__device__ __forceinline__ float over_rows(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// Of the 16 columns of a row of lanes the sum from a lane's own to the last one.
constexpr int DPP_SHL1 = 0x101, DPP_SHL2 = 0x102, DPP_SHL4 = 0x104, DPP_SHL8 = 0x108;
__device__ __forceinline__ float from_here(float v) {
    v += dpp<DPP_SHL1>(v);
    v += dpp<DPP_SHL2>(v);
    v += dpp<DPP_SHL4>(v);
    return v + dpp<DPP_SHL8>(v);
}

// In LDS: k, v and dy, and in one place after another dS and S, each [NP][PV] in three parts, and q.  SHARED: v's place becomes k's.
template <int DT, int NP, bool SHARED>
struct BwdLds {
    using M = Mat<DT>;
    static constexpr int LDS_STATE = PV + M::PAD, PART = NP * LDS_STATE;
    static constexpr int ONE = M::PARTS * PART > Tile<DT, NP>::SIZE ? M::PARTS * PART : Tile<DT, NP>::SIZE;
    static constexpr int Q = 0, K = ONE, V = SHARED ? K : K + Tile<DT, NP>::SIZE, D = V + Tile<DT, PV>::SIZE;
    static constexpr int BYTES = (int)sizeof(typename M::E) * (D + Tile<DT, PV>::SIZE);
};
// The products of one chunk take no turn behind another's, so there is a workgroup for each and nothing is carried: 4096 of them at
// 2 x 16384 x 8 in float32, 219 us for 16 GFLOP, of which the matrix cores are busy for 58%.  Loads at a chunk's start take a quarter of
// its time, which other workgroups on the CU hide: with up to 64 keys three of them, if what is made of v comes before anything of
// k, so that one place in LDS does for both (four places and two workgroups: 248 us; 2 x 8192 x 16 in bfloat16 128 and 159).  Not in
// turns, which keep k and need more registers, nor in bfloat16 of odd widths.  Walking chunks with the next one's tiles loaded
// ahead needs more registers than there are.  In turn nothing is full (bfloat16: vector 48%, matrix 14%, LDS 31% of the cycles): seven
// barriers a head, and scalar registers for the tensors' addresses that are kept in vector lanes (127 to 180 in turn, 88 to 101 else).
// A workgroup has one chunk of a head, or (TURNS) of all heads of a group one after another: their queries and keys are read once, and
// what the heads give to dq and dk is summed in registers.
template <int DT, int NP, bool TURNS, bool EVEN>
__global__ void __launch_bounds__(WG, NP == 128 ? 1 : TURNS || (DT == DT_BF16 && !EVEN) ? 2 : 3) k_attn_bwd(const Args a) {
    using M = Mat<DT>;
    using E = typename M::E;
    using Frag = typename M::Frag;
    using TN = Tile<DT, NP>;
    using TV = Tile<DT, PV>;
    using S = State<NP>;
    constexpr bool SHARED = !TURNS && NP == PV;
    using L = BwdLds<DT, NP, SHARED>;
    constexpr int NT = NP / 16, LS = L::LDS_STATE;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    E* tq = reinterpret_cast<E*>(lds) + L::Q;
    E* tk = reinterpret_cast<E*>(lds) + L::K;
    E* tv = reinterpret_cast<E*>(lds) + L::V;
    E* td = reinterpret_cast<E*>(lds) + L::D;  // dy
    __shared__ __attribute__((aligned(16))) Falls G;
    __shared__ int said[WAVES];
    __shared__ __attribute__((aligned(16))) float middle[WAVES - 1][CHUNK];
    __shared__ float through[2][WAVES];
    // a position's parts of dg, behind its row of dy
    const auto part_of = [&](int which, int i) -> float& { return reinterpret_cast<float*>(td + i * TV::LD + PV)[which]; };
    enum { PAIRS, FROM_STATE, TO_BEHIND };
    static_assert(M::PAD * sizeof(E) >= 3 * sizeof(float), "");
    const int first_own = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunks = (uint32_t)a.chunks, rest = blockIdx.x / chunks;
    const int64_t c = blockIdx.x - rest * chunks, t0 = c * CHUNK;
    const int tile = (int)(rest % (uint32_t)a.tiles);
    const uint32_t turns = TURNS ? (uint32_t)a.share : 1u, sets = (uint32_t)a.share / turns;  // heads of a workgroup, workgroups of a group
    const uint32_t set = rest / (uint32_t)a.tiles, bg = set / sets;  // bg: a sequence's group
    const uint32_t groups = (uint32_t)(a.heads / a.share);
    const int64_t b = bg / groups;
    const int gr = (int)(bg % groups), h0 = gr * a.share + (int)(set % sets), h1 = h0 + (int)turns;
    const int64_t end = end_of(a, b);
    const int present = (int)min((int64_t)CHUNK, a.length - t0);
    const int all_rows = (int)max((int64_t)0, min((int64_t)CHUNK, end - t0));  // that hold something
    const int vcols = min(PV, a.value - tile * PV);
    const auto part_row = [&](float* p, int64_t i) {
        return p + (((b * a.length + t0 + i) * groups + gr) * sets * a.tiles + (set % sets) * a.tiles + tile) * a.key;
    };
    if (all_rows < present) {
        for (int h = h0; h < h1; ++h) zero_rows<DT>(a.dv, b, h, tile * PV, vcols, t0 + all_rows, t0 + present);
        if (a.part_q == nullptr) {
            zero_rows<DT>(a.dq, b, gr, 0, a.key, t0 + all_rows, t0 + present);
            zero_rows<DT>(a.dk, b, gr, 0, a.key, t0 + all_rows, t0 + present);
        } else {
            for (int i = all_rows + threadIdx.x / 64; i < present; i += WG / 64)
                for (int n = threadIdx.x % 64; n < a.key; n += 64) part_row(a.part_q, i)[n] = 0.0f, part_row(a.part_k, i)[n] = 0.0f;
        }
    }
    const auto dg_of = [&](int h) { return a.dg == nullptr ? nullptr : a.dg + ((tile * a.batch + b) * a.length + t0) * a.heads + h; };
    const auto dg_sum_of = [&](int h) { return a.dg_sum == nullptr ? nullptr : a.dg_sum + ((b * a.chunks + c) * a.tiles + tile) * a.heads + h; };
    if (all_rows == 0) {
        for (int h = h0; h < h1; ++h) {
            if (a.dg != nullptr && (int)threadIdx.x < present) dg_of(h)[(int64_t)threadIdx.x * a.heads] = 0.0f;
            if (a.dg_sum != nullptr && threadIdx.x == 0) *dg_sum_of(h) = 0.0f;
        }
        return;
    }
    floatx4 all_dq[NT] = {}, all_dk[NT] = {};
    bool finite_k = false;
    for (int turn = 0; turn < (TURNS ? a.share : 1); ++turn) {
        const int tid = TURNS ? here_lane(threadIdx.x) : threadIdx.x, lane = tid & 63, own = TURNS ? here(first_own) : first_own;
        const int rows = TURNS ? here(all_rows) : all_rows;
        const int l15 = lane & 15, row4 = 4 * (lane >> 4), me = 16 * own + l15;  // the own position, as i of dq and as j of dk and dv
        const int h = h0 + turn;
        const int64_t bht = (b * a.heads + h) * a.tiles + tile, mark = (bht * a.chunks + c) * S::SIZE;
        S s, ds;
        TN q;
        TV v, d;
        ds.load(a.marks + mark, lane, own);
        v.template load<EVEN>(row_of<DT>(a.v, b, t0, h) + tile * PV, a.v.rs, rows, vcols, tid);
        d.template load<EVEN>(row_of<DT>(a.dy, b, t0, h) + tile * PV, a.dy.rs, rows, vcols, tid);
        s.load(a.fmarks + mark, lane, own);
        const float g_own = decay_at(decays_of(a, b, h) + t0 * a.g.rs, a.g.rs, rows, lane);
        const auto load_q = [&] { q.template load<EVEN>(row_of<DT>(a.q, b, t0, gr), a.q.rs, rows, a.key, tid); };
        if (!SHARED) load_q();
        TN k;
        if (!TURNS || turn == 0) {
            k.template load<EVEN>(row_of<DT>(a.k, b, t0, gr), a.k.rs, rows, a.key, tid);
            if (!SHARED) k.store(tk, tid);
            finite_k = k.finite();
        }
        {
            if (a.pieces > 1)
                ds.add(a.starts + (bht * a.pieces + c / a.per_piece) * S::SIZE, a.pre[(b * a.heads + h) * a.chunks + c], lane, own);
            const double g = decays(g_own);
            if (own == 0) G.put(lane, in_two(g));
            {  // what passes over the chunk; behind key and value there may be anything
                float x = 0.0f;
                const float fall = __builtin_amdgcn_exp2f((float)last_lane(g));
                const bool full = a.key == NP && vcols == PV;
                const int key = here(a.key), value = here(vcols);
                s.each([&](int i, int j, floatx4& y) {
                    if (full) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) x = __builtin_fmaf(y[r] * fall, ds.v[i][j][r], x);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float z = __builtin_fmaf(y[r] * fall, ds.v[i][j][r], x);
                            x = S::n(j, lane, own) < key && S::p(i, lane) + r < value ? z : x;
                        }
                    }
                });
                x = wsum(x);
                if (lane == 0) through[turn & 1][own] = x;
            }
            v.store(tv, tid);
            d.store(td, tid);
            ds.template put<M>(tq, a.key, vcols, lane, own);
            const bool finite_kvd = finite_k && v.finite() && d.finite();
            __syncthreads();
            const float2 mine = G.at(me);
            const float to_end = fall_between(G.at(CHUNK - 1), mine), from_start = a.scale * __builtin_amdgcn_exp2f(mine.x + mine.y);
            floatx4 dq[NT], dk[NT], dv[S::TP], dA_i[4], dA_j[4];  // dy . v with the own positions as i, as j
            // what the positions behind the chunk give to dk and dv, by way of dS
#pragma unroll
            for (int n = 0; n < NT; ++n) dk[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < S::TP; ++p) dv[p] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < PV; p += M::STEP) {
                const Frag f = M::scaled(M::row(tv, TV::LD, 16 * own, p, lane), to_end);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < M::PARTS; ++x) dk[n] = M::mma(M::row(tq + x * L::PART, LS, 16 * n, p, lane), f, dk[n]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (SHARED) {
                scores<M, PV>(dA_i, tv, td, TV::LD, 16 * own, 0, own, lane);
                __builtin_amdgcn_sched_barrier(0);
                scores<M, PV>(dA_j, td, tv, TV::LD, 16 * own, own, 3, lane);
                __syncthreads();
                k.store(tk, tid);
                load_q();
                __syncthreads();
            }
#pragma unroll
            for (int n = 0; n < NP; n += M::STEP) {
                const Frag f = M::scaled(M::row(tk, TN::LD, 16 * own, n, lane), to_end);
#pragma unroll
                for (int p = 0; p < S::TP; ++p)
#pragma unroll
                    for (int x = 0; x < M::PARTS; ++x) dv[p] = M::mma(M::col(tq + x * L::PART, LS, 16 * p, n, lane), f, dv[p]);
                __builtin_amdgcn_sched_barrier(0);
            }
            {
                float x = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const floatx4 f = M::load4(tk + me * TN::LD + 16 * n + row4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        dk[n][r] *= M::behind(to_end);
                        x = __builtin_fmaf(dk[n][r], f[r], x);
                    }
                }
                x = over_rows(x);
                if (lane < 16) part_of(TO_BEHIND, me) = x;
#pragma unroll
                for (int p = 0; p < S::TP; ++p)
#pragma unroll
                    for (int r = 0; r < 4; ++r) dv[p][r] *= M::behind(to_end);
            }
            __syncthreads();
            // and what the state before the chunk gives to dq
            s.template put<M>(tq, a.key, vcols, lane, own);
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NT; ++n) dq[n] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int p = 0; p < PV; p += M::STEP) {
                const Frag f = M::scaled(M::row(td, TV::LD, 16 * own, p, lane), from_start);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int x = 0; x < M::PARTS; ++x) dq[n] = M::mma(M::row(tq + x * L::PART, LS, 16 * n, p, lane), f, dq[n]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __syncthreads();
            q.store(tq, tid);
            say_finite(said, finite_kvd && q.finite(), lane, own);
            __syncthreads();
            const bool finite = heard_finite(said);
            {
                float x = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const floatx4 f = M::load4(tq + me * TN::LD + 16 * n + row4);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        dq[n][r] *= M::behind(from_start);
                        x = __builtin_fmaf(dq[n][r], f[r], x);
                    }
                }
                x = over_rows(x);
                if (lane < 16) part_of(FROM_STATE, me) = x;
            }
            // the own positions as i: rows are positions j before them
            __builtin_amdgcn_sched_barrier(0);
            {
                floatx4 A[4], (&dA)[4] = dA_i;
                scores<M, NP>(A, tk, tq, TN::LD, 16 * own, 0, own, lane);
                __builtin_amdgcn_sched_barrier(0);
                if (!SHARED) scores<M, PV>(dA, tv, td, TV::LD, 16 * own, 0, own, lane);
                __builtin_amdgcn_sched_barrier(0);
                // the pairs that a position t of the own ones lies between: of M_ij the sum over the own i >= t, then over j < t; and all
                // own i for the positions of the tiles before
                float at = 0.0f;
                where_finite(finite, [&](auto clean) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        if (t > own) continue;
                        const floatx4 f = falls<true>(G, mine, a.scale, lane, t);
                        floatx4 sums;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int j = 16 * t + row4 + r;
                            const bool in = j <= me && me < rows && counts<decltype(clean)::value>(f[r]);
                            const float x = dA[t][r] * f[r], m = A[t][r] * x;
                            dA[t][r] = in ? x : 0.0f;
                            sums[r] = from_here(in ? m : 0.0f);
                            at += j < me ? sums[r] : 0.0f;
                        }
                        if (t < own && l15 == 0) *reinterpret_cast<floatx4*>(&middle[own - 1][16 * t + row4]) = sums;
                    }
                });
#pragma unroll
                for (int t = 1; t < 4; ++t)
                    if (t > own) dA[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                at = over_rows(at);
                if (lane < 16) part_of(PAIRS, me) = at;
                product_within<M>(dq, finite, tk, TN::LD, dA, 0, own, lane, [&](int j) { return j <= me && me < rows; });
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) all_dq[n][r] = TURNS ? all_dq[n][r] + dq[n][r] : dq[n][r];
            }
            // the own positions as j: rows are positions i behind them
            __builtin_amdgcn_sched_barrier(0);
            {
                floatx4 A[4], (&dA)[4] = dA_j;
                scores<M, NP>(A, tq, tk, TN::LD, 16 * own, own, 3, lane);
                __builtin_amdgcn_sched_barrier(0);
                if (!SHARED) scores<M, PV>(dA, td, tv, TV::LD, 16 * own, own, 3, lane);
                __builtin_amdgcn_sched_barrier(0);
                where_finite(finite, [&](auto clean) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const floatx4 f = falls<false>(G, mine, a.scale, lane, t);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int i = 16 * t + row4 + r;
                            const bool in = i >= me && i < rows && counts<decltype(clean)::value>(f[r]);
                            const float x = A[t][r] * f[r], y = dA[t][r] * f[r];
                            A[t][r] = in ? x : 0.0f;
                            dA[t][r] = in ? y : 0.0f;
                        }
                    }
                });
                const auto inside = [&](int i) { return i >= me && i < rows; };
                product_within<M>(dk, finite, tq, TN::LD, dA, own, 3, lane, inside);
                __builtin_amdgcn_sched_barrier(0);
                product_within<M>(dv, finite, td, TV::LD, A, own, 3, lane, inside);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) all_dk[n][r] = TURNS ? all_dk[n][r] + dk[n][r] : dk[n][r];
                if (me < rows) {
                    auto* out = row_of<DT>(a.dv, b, t0 + me, h) + tile * PV;
                    if (vcols == PV) {
#pragma unroll
                        for (int p = 0; p < S::TP; ++p) write4<DT>(out, 16 * p + row4, PV, dv[p]);
                    } else {
#pragma unroll
                        for (int p = 0; p < S::TP; ++p) write4<DT>(out, 16 * p + row4, here(vcols), dv[p]);
                    }
                }
            }
            __syncthreads();
            // dg, by one wavefront (lane = position)
            if (own == 0) {
                const float(&over_of)[WAVES] = through[turn & 1];
                const double over = (double)over_of[0] + (double)over_of[1] + (double)over_of[2] + (double)over_of[3];
                const bool in = lane < rows;
                // from the states before: positions i from t on (summed from the last one); to the positions behind the chunk: j before t
                const int last = CHUNK - 1 - lane;
                const double later = __shfl(scan(last < rows ? (double)part_of(FROM_STATE, last) : 0.0), CHUNK - 1 - lane, 64);
                double x = (double)part_of(PAIRS, lane) + later + over;
                const double behind = __shfl_up(scan(in ? (double)part_of(TO_BEHIND, lane) : 0.0), 1, 64);
                if (lane > 0) x += behind;
                // and of the chunk's own pairs those with an i of a later tile than t's
#pragma unroll
                for (int t = 1; t < WAVES; ++t) {
                    const double before = __shfl_up(scan(lane < 16 * t ? (double)middle[t - 1][lane] : 0.0), 1, 64);
                    if (lane > 0 && lane < 16 * t) x += before;
                }
                if (!in) x = 0.0;
                if (a.dg != nullptr && lane < present) dg_of(h)[(int64_t)lane * a.heads] = (float)x;
                if (a.dg_sum != nullptr) {
                    const double sum = last_lane(scan(x));
                    if (lane == 0) *dg_sum_of(h) = (float)sum;
                }
            }
        }
    }
    const int me = 16 * first_own + (threadIdx.x & 15), row4 = 4 * ((threadIdx.x & 63) >> 4);
    if (me < all_rows) {
        write_key<DT>(a.part_q == nullptr ? nullptr : part_row(a.part_q, me), row_of<DT>(a.dq, b, t0 + me, gr), a.key, row4, all_dq);
        write_key<DT>(a.part_k == nullptr ? nullptr : part_row(a.part_k, me), row_of<DT>(a.dk, b, t0 + me, gr), a.key, row4, all_dk);
    }
}

// dq (blockIdx.y 0) and dk of a group's key from its parts, in their order.
template <int DT>
__global__ void __launch_bounds__(WG) k_attn_sum(const Args a, int groups) {
    const float* part = blockIdx.y == 0 ? a.part_q : a.part_k;
    const Heads out = blockIdx.y == 0 ? a.dq : a.dk;
    const int64_t n = a.batch * a.length * groups * a.key;
    const int each = a.parts;
    for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
        const int col = (int)(i % a.key), gr = (int)(i / a.key % groups);
        const int64_t bt = i / a.key / groups;
        const float* p = part + (bt * groups + gr) * each * a.key + col;
        float v = p[0];
        for (int k = 1; k < each; ++k) v += p[(int64_t)k * a.key];
        row_of<DT>(out, bt / a.length, bt % a.length, gr)[col] = Elem<DT>::st(v);
    }
}
// dg from its value tiles.
__global__ void __launch_bounds__(WG) k_attn_sum_tiles(const float* part, float* out, int64_t n, int tiles) {
    for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < n; i += (int64_t)gridDim.x * WG) {
        float v = part[i];
        for (int k = 1; k < tiles; ++k) v += part[k * n + i];
        out[i] = v;
    }
}

// ---- one position -------------------------------------------------------------------------------------
// A workgroup per head of a sequence: a thread has four values of every ROWS-th row of the state, read and written once; the rows'
// products with q are summed over the wavefront's lanes, then through LDS.  Bound by memory: 1000 x 16 heads of 64 x 64 take 83 us
// (6.4 TB/s) with accesses of 16 bytes, 121 with those of 4.  EVEN: values are a multiple of four (63 of them take 9% longer than 64).
template <int DT, bool EVEN>
__global__ void __launch_bounds__(WG) k_attn_step(const Args a) {
    constexpr int VEC = 4, LANES = 64 / VEC, ROWS = WG / LANES, AT_ONCE = 4;  // lanes of a row of PV values, rows at a time
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
            const int have = a.value - p;  // values from p on
            const bool whole = EVEN ? have > 0 : have >= VEC;
            float* st = a.state_out + bh * a.key * a.value + p;
            float vv[VEC], y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) vv[e] = (EVEN ? whole : e < have) ? Elem<DT>::ld(v[p + e]) : 0.0f, y[e] = 0.0f;
            for (int n0 = row; n0 < a.key; n0 += ROWS * AT_ONCE) {
                float s[AT_ONCE][VEC], kn[AT_ONCE], qn[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int n = min(n0 + i * ROWS, a.key - 1);
                    kn[i] = Elem<DT>::ld(k[n]);
                    qn[i] = a.scale * Elem<DT>::ld(q[n]);
                    if (whole) {
                        Raw<DT_F32, VEC>::unpack(*reinterpret_cast<const AnyAt*>(st + (int64_t)n * a.value), s[i]);
                    } else if (!EVEN) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) s[i][e] = e < have ? st[(int64_t)n * a.value + e] : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int n = n0 + i * ROWS;
                    if (n >= a.key || (EVEN && !whole)) continue;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        s[i][e] = __builtin_fmaf(f, s[i][e], kn[i] * vv[e]);
                        y[e] = __builtin_fmaf(qn[i], s[i][e], y[e]);
                    }
                    if (EVEN || whole) {
                        *reinterpret_cast<AnyAt*>(st + (int64_t)n * a.value) = Raw<DT_F32, VEC>::pack(s[i]);
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC - 1; ++e)
                            if (e < have) st[(int64_t)n * a.value + e] = s[i][e];
                    }
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
                row_of<DT>(a.y, b, 0, h)[p0 + c] = Elem<DT>::st((part[0][c] + part[1][c]) + (part[2][c] + part[3][c]));
            }
            __syncthreads();
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------
Heads heads_of(const boa_heads& x) { return {x.p, x.batch_stride, x.row_stride, x.head_stride}; }

// The split: pieces of whole chunks, as many as give the wanted workgroups, two for each CU.  Forward of 4 x 4097 x 16 heads in
// bfloat16 with 256, 512, 768 and 1024 wanted: 109, 86, 88 and 89 us of kernels; of 2 x 16384 x 8 in float32: 194, 158, 192 and 166.
// Backward 1024 and 512 take the same time walking, but joining 13 us against 7.5.  Padding counts as work here and in in_turn: the
// lengths are on the device.
constexpr int64_t WANTED = 512;
struct Plan {
    int np, tiles;
    int64_t chunks, bh;
    int32_t pieces, per_piece;
    bool back;
    Plan(const boa_attention& s, bool backward) : back(backward) {
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
    // [starts][fall][pre], backward behind [marks]
    int64_t bytes() const {
        return (back ? 4 * marks() : 0) + 4 * starts() + (pieces > 1 ? (8 * bh * pieces + (back ? 4 * bh * chunks : 0) + 15) / 16 * 16 : 0);
    }
    void place(Args& a, void* p) const {
        a.starts = static_cast<float*>(p);
        if (back) {
            a.marks = a.starts;
            a.starts += marks();
        }
        a.fall = reinterpret_cast<double*>(a.starts + starts());
        a.pre = reinterpret_cast<float*>(a.fall + bh * pieces);
        a.pieces = pieces, a.per_piece = per_piece;
    }
};

// Whether a workgroup of the backward pass takes the heads of a group in turn: where that leaves two workgroups for each place on a CU
// (two places, with more than 64 keys one), else each head by itself.
// 32 x up to 500 x 16 heads of 4 groups in bfloat16: 127 us so, 112 + 42 for the sums over heads with each head by itself; 2 x 8192 x 16
// heads of 8 groups: 234 in float32 and 160 in bfloat16, each by itself 218 + 66 and 143 + 65; 4 x 4096 x 16 heads of 2 groups and 128
// keys: 454 and 317, each by itself 519 + 90 and 380 + 85.  (A part of a group in turn: forward and backward of 300 x 65 x 8 heads and
// 64 x 500 x 8 heads of one group in bfloat16 247 and 215 us, each by itself 205 and 230.)
bool in_turn(const boa_attention& s, const Plan& p) {
    const int share = s.heads / s.groups;
    return share > 1 && p.bh / share * p.tiles * p.chunks >= (p.np == 64 ? 2 : 1) * WANTED;
}
// Parts of a group's dq and dk, which are then summed.
int group_parts(const boa_attention& s, const Plan& p) { return (in_turn(s, p) ? 1 : s.heads / s.groups) * p.tiles; }

int64_t bwd_bytes(const boa_attention& s, const Plan& p) {
    int64_t n = p.bytes();
    if (group_parts(s, p) > 1) n += 2 * 4 * s.batch * s.length * s.groups * group_parts(s, p) * s.key;
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
    a.heads = s.heads, a.share = s.heads / s.groups, a.key = s.key, a.value = s.value, a.tiles = p.tiles, a.scale = s.scale;
    return a;
}

// Kernels whose LDS passes 64 KB are told so before each launch: it is of the current device, of no stream, and may run under capture.
template <class K>
int allow_lds(K* kernel, int bytes) {
    BOA_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return BOA_OK;
}

// Whether no access of 16 bytes passes a row's end.  Kernels that know it need no shifts, and fewer registers.
bool even(const boa_attention& s) { return (s.key | s.value) % (s.dtype == BOA_DT_F32 ? 4 : 8) == 0; }

// Calls f with the padded key and `even` as constants.
template <class F>
int with_key(int np, bool even, F f) {
    const auto with = [&](auto n) { return even ? f(n, std::true_type()) : f(n, std::false_type()); };
    return np == 64 ? with(std::integral_constant<int, 64>()) : with(std::integral_constant<int, 128>());
}

// What the pieces leave, and backward what every chunk's end is reached with.
template <int DT, int NP, bool BACK, bool EVEN>
int launch_states(const Args& a, const Plan& p, hipStream_t s) {
    hipLaunchKernelGGL((k_attn_states<DT, NP, BACK, EVEN>), dim3((uint32_t)(p.bh * p.tiles * p.pieces)), dim3(WG), 0, s, a);
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
    const Plan p(*s, backward != 0);
    return backward ? bwd_bytes(*s, p) : p.bytes();
}

extern "C" int64_t boa_linear_attention_marks_bytes(const boa_attention* s) {
    if (check_sizes("boa_linear_attention_marks_bytes", s) != BOA_OK) return -1;
    return 4 * Plan(*s, false).marks();
}

extern "C" int boa_linear_attention_fwd(const boa_attention* s, void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_sizes("boa_linear_attention_fwd", s);
    if (rc != BOA_OK) return rc;
    if (s->batch == 0) return BOA_OK;
    if ((s->length > 0 && (!s->decay || !s->q.p || !s->k.p || !s->v.p || !s->y.p)) || (uintptr_t)s->marks % 16)
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_fwd: null pointer, or marks not at a multiple of 16 bytes");
    const Plan p(*s, false);
    if (p.bytes() > 0 && (!d_work || (uintptr_t)d_work % 16 || work_bytes < p.bytes()))
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_fwd: workspace of %lld bytes, needs %lld at a multiple of 16", (long long)work_bytes,
                        (long long)p.bytes());
    Args a = args_of(*s, p);
    p.place(a, d_work);
    a.marks = s->marks;
    hipStream_t st = (hipStream_t)stream;
    return with_dtype(s->dtype, [&](auto dt) {
        return with_key(p.np, even(*s), [&](auto np, auto even) {
            constexpr bool EVEN = decltype(even)::value;
            constexpr int DT = decltype(dt)::value, NP = decltype(np)::value, LDS = FwdLds<DT, NP>::BYTES;
            if (p.pieces > 1)
                if (const int no = launch_states<DT, NP, false, EVEN>(a, p, st)) return no;
            if (const int no = allow_lds(k_attn_fwd<DT, NP, EVEN>, LDS)) return no;
            hipLaunchKernelGGL((k_attn_fwd<DT, NP, EVEN>), dim3((uint32_t)(p.bh * p.tiles * p.pieces)), dim3(WG), LDS, st, a);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
    });
}

extern "C" int boa_linear_attention_bwd(const boa_attention* s, void* d_work, int64_t work_bytes, void* stream) {
    const int rc = check_sizes("boa_linear_attention_bwd", s);
    if (rc != BOA_OK) return rc;
    const Plan p(*s, true);
    const int64_t need = bwd_bytes(*s, p);
    hipStream_t st = (hipStream_t)stream;
    const bool empty = s->batch == 0 || s->length == 0;  // no decay is read, and a gradient for each position has none either
    if ((!empty && !s->decay) || ((!empty || s->decay_per_head) && !s->ddecay))
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_bwd: null pointer");
    if (empty) {
        if (s->decay_per_head) BOA_HIP_TRY(launch_sum_parts(nullptr, 0, s->heads, s->ddecay, st));
        return BOA_OK;
    }
    if (!s->q.p || !s->k.p || !s->v.p || !s->dy.p || !s->dq.p || !s->dk.p || !s->dv.p || !s->marks || (uintptr_t)s->marks % 16)
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_bwd: null pointer, or marks not at a multiple of 16 bytes");
    if (!d_work || work_bytes < need || (uintptr_t)d_work % 16)
        return boa_fail(BOA_ERR_ARG, "boa_linear_attention_bwd: workspace of %lld bytes, needs %lld at a multiple of 16", (long long)work_bytes,
                        (long long)need);
    Args a = args_of(*s, p);
    p.place(a, d_work);
    a.fmarks = s->marks;
    a.state_in = nullptr, a.state_out = nullptr;
    float* rest = reinterpret_cast<float*>(static_cast<char*>(d_work) + p.bytes());
    const bool turns = in_turn(*s, p);
    a.parts = group_parts(*s, p);
    if (a.parts > 1) {
        const int64_t each = s->batch * s->length * s->groups * a.parts * s->key;
        a.part_q = rest, a.part_k = rest + each;
        rest += 2 * each;
    }
    if (s->decay_per_head) a.dg_sum = rest;
    else a.dg = p.tiles > 1 ? rest : s->ddecay;
    return with_dtype(s->dtype, [&](auto dt) {
        return with_key(p.np, even(*s), [&](auto np, auto even) {
            constexpr bool EVEN = decltype(even)::value;
            constexpr int DT = decltype(dt)::value, NP = decltype(np)::value;
            if (const int no = launch_states<DT, NP, true, EVEN>(a, p, st)) return no;
            const dim3 grid((uint32_t)(p.bh / (turns ? a.share : 1) * p.tiles * p.chunks));
            if (turns) {
                constexpr int LDS = BwdLds<DT, NP, false>::BYTES;
                if (const int no = allow_lds(k_attn_bwd<DT, NP, true, EVEN>, LDS)) return no;
                hipLaunchKernelGGL((k_attn_bwd<DT, NP, true, EVEN>), grid, dim3(WG), LDS, st, a);
            } else {
                constexpr int LDS = BwdLds<DT, NP, NP == PV>::BYTES;
                if (const int no = allow_lds(k_attn_bwd<DT, NP, false, EVEN>, LDS)) return no;
                hipLaunchKernelGGL((k_attn_bwd<DT, NP, false, EVEN>), grid, dim3(WG), LDS, st, a);
            }
            BOA_HIP_TRY(hipGetLastError());
            if (a.part_q != nullptr) {
                const int64_t n = ceil_div(s->batch * s->length * s->groups * s->key, WG);
                hipLaunchKernelGGL((k_attn_sum<DT>), dim3((uint32_t)(n < MAX_BLOCKS ? n : MAX_BLOCKS), 2), dim3(WG), 0, st, a, s->groups);
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
    const Plan p(*s, false);
    const Args a = args_of(*s, p);
    const dim3 grid((uint32_t)(p.bh < MAX_BLOCKS ? p.bh : MAX_BLOCKS));
    return with_dtype(s->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (s->value % 4 == 0) hipLaunchKernelGGL((k_attn_step<DT, true>), grid, dim3(WG), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((k_attn_step<DT, false>), grid, dim3(WG), 0, (hipStream_t)stream, a);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}
