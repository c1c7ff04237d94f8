// Shared parts of the training and single-token operators (norm_op.hip, loss_op.hip, conv_op.hip, scan_op.hip): element
// types, row loads and stores, sums over a wavefront without the LDS, and the sum of partial rows.
//
// Every operator takes its activations as float32, bfloat16 or float16 and computes in float32; a result is rounded to the
// activations' type once, when it is stored.  Parameters, their gradients, states and statistics are float32.
#pragma once

#include <type_traits>

#include "boa_common.h"
#include "model_dev.h"

namespace boa {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };  // BOA_DT_*

template <int DT> struct Elem;
template <> struct Elem<DT_F32> {
    using T = float;
    static __device__ __forceinline__ float ld(T v) { return v; }
    static __device__ __forceinline__ T st(float v) { return v; }
};
template <> struct Elem<DT_BF16> {
    using T = uint16_t;
    static __device__ __forceinline__ float ld(T v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ T st(float v) { return (T)bf16_rne(v); }
};
template <> struct Elem<DT_F16> {
    using T = uint16_t;
    static __device__ __forceinline__ float ld(T v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ __forceinline__ T st(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// Elements that one 16-byte access holds.
template <int DT> constexpr int wide() { return 16 / (int)sizeof(typename Elem<DT>::T); }

// VEC consecutive elements as float32, in one access of 16 or 8 bytes (the address a multiple of that) or of one element.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <int DT, int VEC>
struct Raw {
    static constexpr int WORDS = VEC * (int)sizeof(typename Elem<DT>::T) / 4;
    static_assert(VEC == 1 || WORDS == 4 || WORDS == 2, "");
    using V = std::conditional_t<VEC == 1, typename Elem<DT>::T, std::conditional_t<WORDS == 4, u32x4, u32x2>>;
    static __device__ __forceinline__ V load(const typename Elem<DT>::T* p) { return *reinterpret_cast<const V*>(p); }
    static __device__ __forceinline__ void unpack(V r, float (&v)[VEC]) {
        if constexpr (VEC == 1) {
            v[0] = Elem<DT>::ld(r);
        } else {
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                if constexpr (DT == DT_F32) {
                    v[j] = __uint_as_float(r[j]);
                } else {
                    v[2 * j] = Elem<DT>::ld((uint16_t)(r[j] & 0xFFFFu));
                    v[2 * j + 1] = Elem<DT>::ld((uint16_t)(r[j] >> 16));
                }
            }
        }
    }
    static __device__ __forceinline__ V pack(const float (&v)[VEC]) {
        if constexpr (VEC == 1) {
            return Elem<DT>::st(v[0]);
        } else {
            V r;
#pragma unroll
            for (int j = 0; j < WORDS; ++j) {
                if constexpr (DT == DT_F32) r[j] = __float_as_uint(v[j]);
                else if constexpr (DT == DT_BF16) r[j] = bf16_pk(v[2 * j], v[2 * j + 1]);
                else r[j] = (uint32_t)Elem<DT>::st(v[2 * j]) | ((uint32_t)Elem<DT>::st(v[2 * j + 1]) << 16);
            }
            return r;
        }
    }
};
template <int DT, int VEC>
__device__ __forceinline__ void ld_vec(const typename Elem<DT>::T* p, float (&v)[VEC]) {
    Raw<DT, VEC>::unpack(Raw<DT, VEC>::load(p), v);
}
template <int DT, int VEC>
__device__ __forceinline__ void st_vec(typename Elem<DT>::T* p, const float (&v)[VEC]) {
    *reinterpret_cast<typename Raw<DT, VEC>::V*>(p) = Raw<DT, VEC>::pack(v);
}

// ------------------------------------------------------------------------------------------------
// Sums and maxima over a wavefront in registers: DPP permutations inside a row of 16 lanes, permlane swaps across rows.
// Fixed order; every lane gets the result.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_HALF_MIRROR = 0x141, DPP_ROR8 = 0x128;
// (a, b) -> a's low half of the wavefront with b's low half in its high half, and the two high halves likewise
__device__ __forceinline__ void swap32(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
// the same for rows of 16: a gets the even rows of both (b's in its odd rows), b the odd rows of both
__device__ __forceinline__ void swap16(float& a, float& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
}
struct Add {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Max {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
// R values (1, 2, 4 or 8) over the wavefront; lane l gets value l / (64 / R).  While there are several, a step of the butterfly
// halves the values that a lane carries instead of the lanes that differ: 18 instructions for 8 values, 10 for one.
template <int BIT, int CTRL, class Op>
__device__ __forceinline__ float join(float a, float b, int lane) {
    const bool up = (lane & BIT) != 0;
    const float keep = up ? b : a, give = up ? a : b;  // in all lanes: a lane reads what another one gives
    return Op::of(keep, dpp<CTRL>(give));
}
template <class Op, int R>
__device__ __forceinline__ float reduce(const float (&x)[R], int lane) {
    float v[R == 1 ? 2 : R];
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = x[i];
    if constexpr (R == 1) v[1] = v[0];
    constexpr int H = R >= 2 ? R / 2 : 1;  // values left after the step across halves
#pragma unroll
    for (int i = 0; i < H; ++i) {
        swap32(v[i], v[i + H]);
        v[i] = Op::of(v[i], v[i + H]);
    }
    constexpr int Q = R >= 4 ? R / 4 : 1;  // after the step across rows
    if constexpr (R < 4) v[1] = v[0];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        swap16(v[i], v[i + Q]);
        v[i] = Op::of(v[i], v[i + Q]);
    }
    float r;
    if constexpr (R == 8) r = join<8, DPP_ROR8, Op>(v[0], v[1], lane);
    else r = Op::of(v[0], dpp<DPP_ROR8>(v[0]));
    r = Op::of(r, dpp<DPP_HALF_MIRROR>(r));
    r = Op::of(r, dpp<DPP_XOR2>(r));
    return Op::of(r, dpp<DPP_XOR1>(r));
}
__device__ __forceinline__ float wsum(float v) {
    const float x[1] = {v};
    return reduce<Add, 1>(x, 0);
}
// Lane l's value in all lanes (l the same for all).
__device__ __forceinline__ float from_lane(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }

__device__ __forceinline__ float hw_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + hw_exp(-x)); }

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Calls f with the element type as a constant (dtype is one of the three: the entry points check it).
template <class F>
inline int with_dtype(int dtype, F f) {
    switch (dtype) {
        case DT_F32: return f(std::integral_constant<int, DT_F32>());
        case DT_BF16: return f(std::integral_constant<int, DT_BF16>());
        default: return f(std::integral_constant<int, DT_F16>());
    }
}
// whether rows `stride` elements apart from p on can be read 16 bytes at a time
inline bool aligned16(int dtype, const void* p, int64_t stride) {
    const int es = dtype == DT_F32 ? 4 : 2;
    return ((uintptr_t)p | (uintptr_t)(stride * es)) % 16 == 0;
}

// Workgroups of 256 threads that one launch dimension takes (its threads are counted in 32 bits).
constexpr int64_t MAX_BLOCKS = 0xFFFFFF;

// out[j] = sum over p < parts of part[p * width + j] for the SUM_COLS columns j of block `blk`, in a fixed order, by a workgroup of
// SUM_COLS x GROUPS threads: a thread adds every GROUPS-th row, eight loads in flight, and the groups' sums follow one another.
constexpr int SUM_COLS = 32, SUM_AT_ONCE = 8;
template <int GROUPS>
__device__ __forceinline__ void sum_parts(const float* part, int64_t parts, int64_t width, float* out, int64_t blk) {
    __shared__ float s[GROUPS][SUM_COLS + 1];
    const int c = threadIdx.x % SUM_COLS, g = threadIdx.x / SUM_COLS;
    const int64_t j = blk * SUM_COLS + c;
    float v = 0.0f;
    if (j < width)
        for (int64_t p0 = g; p0 < parts; p0 += GROUPS * SUM_AT_ONCE) {
            float t[SUM_AT_ONCE];
#pragma unroll
            for (int i = 0; i < SUM_AT_ONCE; ++i) {
                const int64_t p = p0 + i * GROUPS;
                t[i] = p < parts ? part[p * width + j] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < SUM_AT_ONCE; ++i) v += t[i];
        }
    s[g][c] = v;
    __syncthreads();
    if (g == 0 && j < width) {
        v = s[0][c];
        for (int k = 1; k < GROUPS; ++k) v += s[k][c];
        out[j] = v;
    }
}
// The same as a launch of its own (norm_op.hip).
hipError_t launch_sum_parts(const float* part, int64_t parts, int64_t width, float* out, hipStream_t s);

}  // namespace boa
