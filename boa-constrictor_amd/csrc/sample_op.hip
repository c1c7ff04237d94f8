// Symbols drawn from rows of logits by given random numbers (boa_sample).
//
//   w_i = e^((x_i - max) / temperature), then kept: the top_k largest; of those the fewest largest whose sum reaches top_p of
//   theirs; of those whoever has at least min_p of the largest; drawn: the first i, in the symbols' order, with w_0 + ... + w_i > u sum(w)
//   Among equals the lower index counts as larger.  Temperature 0 takes the largest.
//
// Weights and the sums that decide are in 64 bits, so that which symbol a number falls on does not hang on the order in which 32-bit
// sums are rounded.  A row is held in registers by one wavefront, or by four for more than 1024 symbols.  Nothing is sorted: the
// key of the last symbol that a limit keeps is found bit by bit, by counting (or adding the weights of) the keys above, with the
// logits as unsigned integers of the same order, until one symbol is left that it can be.  The weights are added in 32 bits
// there; whether the symbol found is the one is decided by two sums in 64, and where it is not (a border within 32 bits'
// rounding) the search is done again with those.
//
// Measured with top_k 50 and top_p 0.95: 65536 x 256 float32 122 us, 16384 x 1024 104, 4096 x 4096 139 (0.5 to 0.6 TB/s); a single
// row 6, whose steps follow one another.  Bound by vector work: a search's step is a compare, a count or a sum over the lanes, about
// 30 steps a row; exponentials in 64 bits are the rest.  Above 256 symbols 11 to 62 scalar registers are kept in
// vector lanes (counts of the keys).
#include "ops_common.h"

#include "../../include/boa_hip.h"

using namespace boa;

namespace {

constexpr int WG = 256, WAVES = WG / 64;
constexpr int MAX_V = BOA_SAMPLE_MAX_V;

struct Args {
    const void* x;
    int64_t stride, rows;
    const float* u;
    const float *temperature, *top_p, *min_p;  // per row, or null
    const int32_t* top_k;
    double all_temperature, all_top_p, all_min_p;
    int32_t all_top_k, V;
    int64_t* out;
};

// The largest of all lanes, the same way.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_with(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
    v = max_with<DPP_SHR1, 0xF>(v);
    v = max_with<DPP_SHR2, 0xF>(v);
    v = max_with<DPP_SHR4, 0xF>(v);
    v = max_with<DPP_SHR8, 0xF>(v);
    v = max_with<DPP_BCAST15, 0xA>(v);
    v = max_with<DPP_BCAST31, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Sums over the lanes of a row: of a wavefront, or of four (ROW_WAVES) by way of LDS.
template <int ROW_WAVES>
struct Over {
    double* s;  // [2][WAVES]
    int turn = 0;
    __device__ __forceinline__ explicit Over(double* lds) : s(lds) {}
    template <class F>
    __device__ __forceinline__ double waves(double v, F join) {
        if constexpr (ROW_WAVES == 1) return v;
        double* at = s + (turn ^= 1) * WAVES;  // what the turn before has left may still be read
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        return join(join(at[0], at[1]), join(at[2], at[3]));
    }
    template <class T>
    __device__ __forceinline__ T sum(T v) {
        return (T)waves((double)last_lane(scan(v)), [](double a, double b) { return a + b; });
    }
    __device__ __forceinline__ int count(int of_wave) {
        return ROW_WAVES == 1 ? of_wave : (int)waves((double)of_wave, [](double a, double b) { return a + b; });
    }
    __device__ __forceinline__ uint32_t largest(uint32_t v) {
        v = wave_largest(v);
        return ROW_WAVES == 1 ? v : (uint32_t)waves((double)v, [](double a, double b) { return a > b ? a : b; });
    }
    // of the wavefronts before this one, and of all of them
    __device__ __forceinline__ double before(double of_wave, double& all) {
        if constexpr (ROW_WAVES == 1) {
            all = of_wave;
            return 0.0;
        }
        double* at = s + (turn ^= 1) * WAVES;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) at[wave] = of_wave;
        __syncthreads();
        double v = 0.0, mine = 0.0;
        for (int i = 0; i < WAVES; ++i) {
            if (i == wave) mine = v;
            v += at[i];
        }
        all = v;
        return mine;
    }
};

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }
constexpr uint32_t KEY_OF_NOTHING = 0x007FFFFFu;  // -inf

template <int DT, int VEC, int N, int ROW_WAVES>
__global__ void __launch_bounds__(WG) k_sample(const Args a) {
    constexpr int PER = VEC * N;
    __shared__ double lds[2 * WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = ROW_WAVES == 1 ? 0 : wave;
    Over<ROW_WAVES> over(lds);
    const int64_t walkers = (int64_t)gridDim.x * (WAVES / ROW_WAVES);
    for (int64_t row = (int64_t)blockIdx.x * (WAVES / ROW_WAVES) + (ROW_WAVES == 1 ? wave : 0); row < a.rows; row += walkers) {
        const auto* x = static_cast<const typename Elem<DT>::T*>(a.x) + row * a.stride;
        const auto col = [&](int i) { return ((i * ROW_WAVES + part) * 64 + lane) * VEC; };
        uint32_t key[PER];  // 0 behind the last symbol
        float v[PER];
        bool nan = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = col(i);
            float e[VEC];
            ld_vec<DT, VEC>(x + (c < a.V ? c : a.V - VEC), e);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i * VEC + j] = e[j];
                nan |= c < a.V && e[j] != e[j];
                key[i * VEC + j] = c < a.V ? key_of(e[j]) : 0u;
            }
        }
        const float u = a.u[row];
        const double t = a.temperature != nullptr ? (double)a.temperature[row] : a.all_temperature;
        const double p = a.top_p != nullptr ? (double)a.top_p[row] : a.all_top_p;
        const double least = a.min_p != nullptr ? (double)a.min_p[row] : a.all_min_p;
        const int k = a.top_k != nullptr ? a.top_k[row] : a.all_top_k;

        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) top = max(top, key[i]);
        top = over.largest(top);
        const bool bad = over.count(__popcll(__ballot(nan))) > 0 || top <= KEY_OF_NOTHING || u != u || t != t || p != p || least != least;
        // The largest key of which `enough` holds, where it holds of all smaller ones: bit by bit, from the first in which the keys
        // differ, until one symbol is left between those that are known to be enough and those that are not (bits below a
        // 16-bit logit's last are all the same).
        const auto search = [&](auto enough) {
            constexpr int LAST_BIT = DT == DT_F32 ? 0 : DT == DT_BF16 ? 16 : 13;
            const auto smallest_from = [&](uint32_t c) {  // as the largest complement
                uint32_t found = 0u;
#pragma unroll
                for (int i = 0; i < PER; ++i) found = max(found, key[i] >= c ? ~key[i] : 0u);
                return ~over.largest(found);
            };
            const auto count_from = [&](uint32_t c) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i) n += __popcll(__ballot(key[i] >= c));
                return over.count(n);
            };
            uint32_t last = smallest_from(1u);
            if (last == top) return last;
            const int first_bit = 31 - __clz(last ^ top);
            last &= ~((2u << first_bit) - 1u);
            int with = count_from(max(last, 1u)), above = 0;  // symbols from `last` on, and from the first key known not to be enough on
            for (int bit = first_bit; bit >= LAST_BIT && with - above > 1; --bit) {
                const uint32_t c = last | 1u << bit;
                const int n = count_from(c);
                if (enough(c, n)) last = c, with = n;
                else above = n;
            }
            return smallest_from(max(last, 1u));
        };
        // keeps of the symbols with this key the first n, by their index
        const auto keep_first = [&](uint32_t of, int n) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int lower = 0, all = 0;
                uint64_t mine[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    mine[j] = __ballot(key[i * VEC + j] == of);
                    lower += __builtin_amdgcn_mbcnt_hi((uint32_t)(mine[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mine[j], 0u));
                    all += __popcll(mine[j]);
                }
                double total;
                const int before = (int)over.before((double)all, total);
                lower += before;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (key[i * VEC + j] == of) {
                        if (lower >= n) key[i * VEC + j] = 0u;
                        ++lower;
                    }
                n -= (int)total;
            }
        };
        if (!bad) {
            if (t <= 0.0 || p <= 0.0 || least > 1.0) {
#pragma unroll
                for (int i = 0; i < PER; ++i) key[i] = key[i] == top ? top : 0u;
                keep_first(top, 1);
            } else if (k > 0 && k < a.V) {
                const uint32_t last = search([&](uint32_t, int n) { return n >= k; });
                int above = 0, with = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    above += __popcll(__ballot(key[i] > last));
                    with += __popcll(__ballot(key[i] >= last));
                    if (key[i] < last) key[i] = 0u;
                }
                above = over.count(above);
                with = over.count(with);
                if (with > k) keep_first(last, k - above);
            }
        }
        // weights of what is kept
        const float largest = value_of(top);
        const double by = t > 0.0 ? 1.0 / t : 1.0;
        // an infinity is as large as itself, and infinitely far from all others whatever the temperature
        const auto weight = [&](float x) {
            const double d = (double)x - (double)largest;
            return x == largest ? 1.0 : d == -__builtin_huge_val() ? 0.0 : exp(d * by);
        };
        double w[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) w[i] = key[i] == 0u || bad ? 0.0 : weight(v[i]);
        if (!bad && p > 0.0 && p < 1.0) {
            const auto from = [&](uint32_t c, auto zero) {
                auto sum = zero;
#pragma unroll
                for (int i = 0; i < PER; ++i) sum += key[i] >= c ? (decltype(zero))w[i] : zero;
                return over.sum(sum);
            };
            const double want = p * from(1u, 0.0);
            uint32_t last = search([&](uint32_t c, int) { return from(c, 0.0f) >= (float)want; });
            double above = from(last + 1u, 0.0);
            if (above >= want || from(last, 0.0) < want) {
                last = search([&](uint32_t c, int) { return from(c, 0.0) >= want; });
                above = from(last + 1u, 0.0);
            }
            // of those that are equal to the last as many as it takes
            int equal = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) equal += __popcll(__ballot(key[i] == last));
            equal = over.count(equal);
            int n = 1;
            if (equal > 1) {
                const double one = weight(value_of(last));
                while (n < equal && above + n * one < want) ++n;
            }
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i] < last) key[i] = 0u;
            if (n < equal) keep_first(last, n);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) w[i] = key[i] == 0u || w[i] < least ? 0.0 : w[i];

        // sums up to each symbol, in the symbols' order
        double upto[N], all = 0.0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) s += w[i * VEC + j];
            const double with = scan(s);
            double total;
            const double waves_before = over.before(last_lane(with), total);
            const double lanes_before = __shfl_up(with, 1, 64);
            upto[i] = all + (waves_before + (lane == 0 ? 0.0 : lanes_before));
            all += total;
        }
        const double at = (double)u * all;
        // the first symbol that passes it; the last one of all where rounding lets none
        int first = a.V, end = -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            double s = upto[i];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                s += w[i * VEC + j];
                if (w[i * VEC + j] > 0.0) {
                    if (s > at) first = min(first, col(i) + j);
                    end = col(i) + j;
                }
            }
        }
        const uint32_t far = over.largest((uint32_t)(a.V - first));
        const uint32_t last_of_all = over.largest((uint32_t)(end + 1));
        if (lane == 0 && part == 0) a.out[row] = bad ? -1 : far > 0 ? (int64_t)a.V - far : (int64_t)last_of_all - 1;
    }
}

template <int DT, int VEC, int N, int ROW_WAVES>
int launch(const Args& a, hipStream_t s) {
    const int64_t groups = ceil_div(a.rows, WAVES / ROW_WAVES);
    hipLaunchKernelGGL((k_sample<DT, VEC, N, ROW_WAVES>), dim3((uint32_t)(groups < MAX_BLOCKS ? groups : MAX_BLOCKS)), dim3(WG), 0, s, a);
    BOA_HIP_TRY(hipGetLastError());
    return BOA_OK;
}

}  // namespace

extern "C" int boa_sample(int dtype, const void* d_x, int64_t x_stride, int64_t rows, int32_t V, const float* d_u, double temperature,
                          const float* d_temperature, int32_t top_k, const int32_t* d_top_k, double top_p, const float* d_top_p,
                          double min_p, const float* d_min_p, int64_t* d_out, void* stream) {
    if (dtype < BOA_DT_F32 || dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "boa_sample: unknown type %d", dtype);
    if (rows < 0 || V < 1 || V > MAX_V)
        return boa_fail(BOA_ERR_ARG, "boa_sample: need rows >= 0 and 1 <= V <= %d (got %lld, %d)", MAX_V, (long long)rows, V);
    if ((!d_temperature && !(temperature >= 0.0)) || (!d_top_p && !(top_p >= 0.0)) || (!d_min_p && !(min_p >= 0.0)))
        return boa_fail(BOA_ERR_ARG, "boa_sample: temperature %g, top_p %g, min_p %g", temperature, top_p, min_p);
    if (rows == 0) return BOA_OK;
    if (!d_x || !d_u || !d_out) return boa_fail(BOA_ERR_ARG, "boa_sample: null pointer");
    const Args a = {d_x, x_stride, rows, d_u, d_temperature, d_top_p, d_min_p, d_top_k, temperature, top_p, min_p, top_k, V, d_out};
    hipStream_t s = (hipStream_t)stream;
    return with_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        // Accesses of four values where the rows are aligned for them, else of one (65536 x 256 122 us against 138, 4096 x 4096 139
        // against 367).  One wavefront to a row, whose sums need no LDS, up to 1024 symbols (16384 x 1024: 104 us, with four 187),
        // with fewer registers up to 256; more symbols than that do not fit one wavefront's registers.
        if (V % 4 == 0 && aligned16(dtype, d_x, x_stride)) {
            if (V <= 256) return launch<DT, 4, 1, 1>(a, s);
            if (V <= 1024) return launch<DT, 4, 4, 1>(a, s);
            return launch<DT, 4, 4, 4>(a, s);
        }
        if (V <= 256) return launch<DT, 1, 4, 1>(a, s);
        if (V <= 1024) return launch<DT, 1, 16, 1>(a, s);
        return launch<DT, 1, 16, 4>(a, s);
    });
}
