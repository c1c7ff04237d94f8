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
// computes each forward again from its mark with e and e h in registers, then backward.  Where the batch has too few
// workgroups the length is split into chunks: a first kernel computes what each chunk alone leaves (forward its last state, backward
// the adjoint before it), and the main one goes on from those of the chunks before its own.
//
// Measured, float32 of 2 x 16384 positions and 512 channels: chunks alone 64 us, joined 7, forward 97 (of the vector units' cycles
// 0.74 and 0.68), backward 72 + 7 + 229 (0.71, 0.85) + 13 for the sums, where one pass over the data would take 54 and 94 us of
// memory; 8 x 1000 of 512: 20 + 33 and 20 + 64 + 4; a prompt of 4 x 4097 and 1024 channels in bfloat16: 62 + 90.
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
    bool joined;                  // local holds the states before the chunks (k_scan_join), not those that they leave
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

// An offset that the compiler takes for a new one.  A lane's: an address is then a uniform one and a 32-bit offset that is seen
// where it is used, without arithmetic in the lanes; else the sums are carried through the loop in vector registers, two for each
// array.  A row's: else the address of every row of a block is carried in scalar registers, 32 of them.
__device__ __forceinline__ uint32_t fresh(uint32_t& c) {
    asm volatile("" : "+v"(c));
    return c;
}
__device__ __forceinline__ uint32_t fresh_scalar(uint32_t c) {
    asm volatile("" : "+s"(c));
    return c;
}

// This wavefront's states of B or C in the rows of a block, through the scalar cache (constant address space: nothing the
// kernel writes; 16-bit rows are 4-byte aligned, and a block of rows spans less than 4 GiB, which the entry points check).
// A row's place is a 32-bit offset from the block's first: one scalar multiplication, where 64-bit addresses of single rows
// cost ten scalar instructions, more than the vector work of a row.
template <int DT>
struct ScalarRows {
    static constexpr int WORDS = NQ * (int)sizeof(typename Elem<DT>::T) / 4;
    const char* p;   // the block's first row
    uint32_t bytes;  // of a row
    __device__ __forceinline__ ScalarRows(const Rows& a, int64_t b, int64_t t, int q)
        : p((const char*)(row<DT>(a, b, t) + q * NQ)), bytes((uint32_t)a.r * (uint32_t)sizeof(typename Elem<DT>::T)) {}
    __device__ __forceinline__ void ahead(bool on) { p += on ? bytes * SUB : 0; }
    template <int ROWS = SUB>
    __device__ __forceinline__ void back(bool on) { p -= on ? bytes * ROWS : 0; }
    __device__ __forceinline__ void next_block() { bytes = fresh_scalar(bytes); }
    __device__ __forceinline__ void load(int s, uint32_t (&w)[WORDS]) const {
        typedef __attribute__((address_space(4))) const char CByte;
        typedef __attribute__((address_space(4))) const uint32_t CWord;
        CWord* at = (CWord*)((CByte*)p + (uint32_t)s * bytes);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = at[i];
    }
    static __device__ __forceinline__ float value(const uint32_t (&w)[WORDS], int n) {
        if constexpr (DT == DT_F32) return __uint_as_float(w[n]);
        else return Elem<DT>::ld((uint16_t)(n & 1 ? w[n / 2] >> 16 : w[n / 2] & 0xFFFFu));
    }
};

// G positions of a block as the recurrence reads them: B and C from the scalar cache, what was prepared from LDS.  A group is
// on its way while the one before it is computed, B and C across the blocks' borders too (2 x 16384 positions of 512 channels: forward
// 99 -> 95 us, the chunks alone 70 -> 63).  Both kinds of load return out of order to one counter, so
// a wait is for all that are under way: the group to compute is waited for (here) before the next one is issued.
constexpr int GROUP_ONE = 4, GROUP_TWO = 2;  // where B or C is read, and where both are: 4 spills scalar registers (95, 104 us)
template <int DT, int G>
struct Group {
    using S = ScalarRows<DT>;
    uint32_t B[G][S::WORDS], C[G][S::WORDS];
    float2 in[G];
    float g[G];
    __device__ __forceinline__ void here() {
#pragma unroll
        for (int j = 0; j < G; ++j) asm volatile("" : "+v"(in[j].x), "+v"(in[j].y));
    }
    static __device__ __forceinline__ void words_here(uint32_t (&w)[G][S::WORDS]) {
#pragma unroll
        for (int j = 0; j < G; ++j)
#pragma unroll
            for (int i = 0; i < S::WORDS; ++i) asm volatile("" : "+s"(w[j][i]));
    }
    __device__ __forceinline__ float b(int j, int n) const { return S::value(B[j], n); }
    __device__ __forceinline__ float c(int j, int n) const { return S::value(C[j], n); }
};

// The rows of a block that lanes read or write, each lane its channel: the same 32-bit offsets from the block's first row.
template <int DT>
struct LaneRows {
    using T = typename Elem<DT>::T;
    gmut<char> p;    // the block's first row
    uint32_t bytes;  // of a row
    __device__ __forceinline__ LaneRows(const Rows& a, int64_t b, int64_t t)
        : p((gmut<char>)row_mut<DT>(a, b, t)), bytes((uint32_t)a.r * (uint32_t)sizeof(T)) {}
    __device__ __forceinline__ void ahead(bool on) { p += on ? bytes * SUB : 0; }
    template <int ROWS = SUB>
    __device__ __forceinline__ void back(bool on) { p -= on ? bytes * ROWS : 0; }
    // c: the lane's channel in bytes
    __device__ __forceinline__ gmut<T> at(int s, uint32_t& c) const { return (gmut<T>)(p + (uint32_t)s * bytes + fresh(c)); }
    __device__ __forceinline__ T load(int s, uint32_t& c) const { return *at(s, c); }
    __device__ __forceinline__ void store(int s, uint32_t& c, float v) const { *at(s, c) = Elem<DT>::st(v); }
};

// Element `c4` bytes from p: the same for float32 arrays.
__device__ __forceinline__ gmut<float> lane_at(gmut<float> p, uint32_t& c4) { return (gmut<float>)((gmut<char>)p + fresh(c4)); }
__device__ __forceinline__ gptr<float> lane_at(gptr<float> p, uint32_t& c4) { return (gptr<float>)((gptr<char>)p + fresh(c4)); }

// A loaded value in a register of its own.  Where a float32 value is used later than the next block's load is issued, the
// compiler otherwise takes the loaded register over, loads into another, and waits for that load at the end of the iteration
// to move it into place.
__device__ __forceinline__ float own_register(float v) {
    float r;
    asm volatile("v_mov_b32 %0, %1" : "=v"(r) : "v"(v));
    return r;
}

__device__ __forceinline__ int64_t end_of(const ScanArgs& a, int64_t b) {
    if (a.lens == nullptr) return a.length;
    const int64_t n = a.lens[b];
    return n < 0 ? 0 : (n < a.length ? n : a.length);
}

// Where a workgroup is: its channels, its sequence, this wavefront's states.
struct Place {
    int lane, q, c;
    uint32_t cc;         // c, or the last channel for the lanes past it
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
        cc = (uint32_t)(live ? c : a.channels - 1);
    }
    __device__ __forceinline__ void decay(const ScanArgs& a, float (&a2)[NQ]) const {
#pragma unroll
        for (int n = 0; n < NQ; ++n) a2[n] = a.A[(int64_t)cc * NS + q * NQ + n] * LOG2E;
    }
};

// State `n` of this wavefront in an array [rows][16][channels], row r.
__device__ __forceinline__ int64_t state_at(const ScanArgs& a, const Place& p, int64_t r, int n) {
    return (r * NS + p.q * NQ + n) * a.channels + p.cc;
}

// h of this wavefront's states over the chunks j, j + step .. (n of them), the loads of four chunks in flight.
__device__ __forceinline__ void over_chunks(const ScanArgs& a, const Place& p, int j, int step, int n_chunks, const float (&a2)[NQ],
                                            float (&h)[NQ]) {
    constexpr int AT_ONCE = 4;
    for (int i0 = 0; i0 < n_chunks; i0 += AT_ONCE) {
        float dts[AT_ONCE], l[AT_ONCE][NQ];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int64_t r = p.b * a.chunks + j + step * min(i0 + i, n_chunks - 1);
            dts[i] = (a.dts + r * a.channels)[p.cc];
#pragma unroll
            for (int n = 0; n < NQ; ++n) l[i][n] = (a.local + (r * NS + p.q * NQ + n) * a.channels)[p.cc];
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (i0 + i < n_chunks)
#pragma unroll
                for (int n = 0; n < NQ; ++n) h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(dts[i] * a2[n]), h[n], l[i][n]);
    }
}

// What a wave has to do with memory in a block is the same in every block, without branches: the hardware counts loads and
// stores together in order, and behind a store that may or may not have been issued the compiler waits for all of them (a
// block then takes a store's way to memory and back).  So lanes behind the last channel do what the last one does, a block
// behind the last one is fetched as the last one, and without a gate z is u.
enum { LOCAL, OUT, OUT_MARKS };

// Where there are many chunks, the state before each of them instead: from the ends of the chunks before it (of those behind
// it, from the sequence's end, in the backward pass), in the places of local.  A lane takes one state through 32 chunks with all their
// loads in flight at once, a workgroup has as many wavefronts as that takes, and their ends meet in LDS.
constexpr int JOIN_EACH = 32, MAX_CHUNKS = JOIN_EACH * WAVES;
template <bool BACK>
__global__ void __launch_bounds__(WG) k_scan_join(const ScanArgs a) {
    constexpr int AT_ONCE = JOIN_EACH;
    __shared__ float s_e[WAVES][64], s_h[WAVES][64];
    const int lane = threadIdx.x & 63, q = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t states = (int64_t)NS * a.channels, i0 = (int64_t)blockIdx.x * 64, b0 = i0 / states;  // b0: of the first lane
    // 32 bits are enough in a workgroup: more than two sequences have less than 64 states each
    uint32_t i = (uint32_t)(i0 - b0 * states) + lane, of = i / (uint32_t)states;
    const bool live = b0 + of < a.batch;
    if (!live) of = 0, i = 0;
    const uint32_t in = i % (uint32_t)states, n = in / (uint32_t)a.channels, c = in % (uint32_t)a.channels;
    const int64_t b = b0 + of;
    uint32_t l4 = (uint32_t)((of * a.chunks * states + in) * 4), dts4 = (of * a.chunks * a.channels + c) * 4;  // bytes
    auto chunk = [&](int j) {  // the wavefront's j-th, in the order of the recurrence
        const int at = min(q * AT_ONCE + j, a.chunks - 1);
        return BACK ? a.chunks - 1 - at : at;
    };
    // what is not there (the sums of the last chunk, in the backward pass of the first one, and of those behind the end) is read
    // all the same, but reaches no h that is kept
    float e[AT_ONCE], l[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
        e[j] = *lane_at(G(a.dts) + (b0 * a.chunks + chunk(j)) * a.channels, dts4);
        l[j] = *lane_at(G(a.local) + (b0 * a.chunks + chunk(j)) * states, l4);
    }
    const int chunks = (int)ceil_div(end_of(a, b), a.chunk);  // with positions inside
    const float a2 = a.A[(int64_t)c * NS + n] * LOG2E;
    const float start = !BACK && a.state_in != nullptr ? a.state_in[b * states + in] : 0.0f;
    auto inside = [&](int j) { return q * AT_ONCE + j < a.chunks && chunk(j) < chunks; };
    float h = 0.0f, dts = 0.0f;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
        const float dt = e[j];
        e[j] = __builtin_amdgcn_exp2f(dt * a2);
        if (inside(j)) h = __builtin_fmaf(e[j], h, l[j]), dts += dt;
    }
    s_e[q][lane] = __builtin_amdgcn_exp2f(dts * a2);
    s_h[q][lane] = h;
    __syncthreads();
    h = start;
    for (int w = 0; w < q; ++w) h = __builtin_fmaf(s_e[w][lane], h, s_h[w][lane]);
    if (!live) return;
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
        if (inside(j)) {
            *lane_at(GM(a.local) + (b0 * a.chunks + chunk(j)) * states, l4) = h;
            h = __builtin_fmaf(e[j], h, l[j]);
        }
}

// LOCAL: the state that a chunk alone leaves (from zeros) and its sum of dt, for every chunk but the last; OUT: the chunk's
// outputs, from the state that the chunks before it leave; OUT_MARKS: and the state before every block.
template <int DT, int MODE>
__global__ void __launch_bounds__(WG) k_scan_fwd(const ScanArgs a) {
    using E = Elem<DT>;
    __shared__ float2 s_in[2][SUB][64];  // dt, dt u
    __shared__ float s_y[2][MODE == LOCAL ? 1 : WAVES][SUB][64];
    const Place p(a, MODE == LOCAL ? a.chunks - 1 : a.chunks, 0);
    const int64_t end = end_of(a, p.b), lo = p.k * a.chunk;
    if (MODE == LOCAL && lo + a.chunk >= end) return;  // no chunk behind this one reads its state
    const int64_t hi = lo + a.chunk < a.length ? lo + a.chunk : a.length;  // rows to write
    const int n_subs = lo < end ? (int)ceil_div((hi < end ? hi : end) - lo, SUB) : 0;
    const bool gate = a.z.p != nullptr;
    float a2[NQ], h[NQ];
    p.decay(a, a2);
    const float bias = a.bias != nullptr ? a.bias[p.cc] : 0.0f, D = MODE != LOCAL && a.D != nullptr ? a.D[p.cc] : 0.0f;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
        h[n] = MODE == LOCAL ? 0.0f
               : a.joined && n_subs > 0 ? a.local[state_at(a, p, p.b * a.chunks + p.k, n)]
               : a.state_in != nullptr ? a.state_in[state_at(a, p, p.b, n)] : 0.0f;

    // A block's life: fetched (loads issued), prepared (dt and dt u to LDS), computed, finished (sums over the wavefronts'
    // states, gate, stores).  One barrier per block: block i is computed while i - 1 is finished and i + 1 prepared, with
    // two buffers each.
    const int first = p.q * MINE;  // this wavefront's first position of a block
    uint32_t ce = p.cc * (uint32_t)sizeof(typename E::T), c4 = p.cc * 4;  // the lane's channel in bytes
    LaneRows<DT> xu(a.u, p.b, lo), xd(a.delta, p.b, lo), xz(gate ? a.z : a.u, p.b, lo), xy(a.y, p.b, lo);
    ScalarRows<DT> xB(a.B, p.b, lo, p.q), xC(a.C, p.b, lo, p.q);
    gmut<float> mark = GM(a.marks) + ((p.b * a.subs + lo / SUB) * NS + p.q * NQ) * a.channels;
    const int count = (int)(min(hi, end) - lo), rows_out = (int)(hi - lo);  // positions inside, rows to write
    typename E::T ru[MINE], rd[MINE], rz[MINE];
    auto fetch = [&](int i) {  // i < n_subs
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int s = min(first + k, count - 1 - i * SUB);
            ru[k] = xu.load(s, ce);
            rd[k] = xd.load(s, ce);
            if (MODE != LOCAL) rz[k] = xz.load(s, ce);
        }
    };
    auto prepare = [&](int i, float (&u)[MINE], float (&z)[MINE]) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            u[k] = MODE != LOCAL ? own_register(E::ld(ru[k])) : E::ld(ru[k]);
            if (MODE != LOCAL) z[k] = own_register(E::ld(rz[k]));
            const float dt = hw_softplus(E::ld(rd[k]) + bias);
            // behind the end the state stays as it is
            s_in[i & 1][first + k][p.lane] = i * SUB + first + k < count ? make_float2(dt, dt * u[k]) : make_float2(0.0f, 0.0f);
        }
    };
    // whole: all the block's positions are inside
    auto finish = [&](int i, const float (&u)[MINE], const float (&z)[MINE], bool whole) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = first + k;
            float y = D * u[k];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) y += s_y[i & 1][MODE == LOCAL ? 0 : w][at][p.lane];
            y *= gate ? hw_silu(z[k]) : 1.0f;
            if (whole || i * SUB + at < rows_out) xy.store(at, ce, whole || i * SUB + at < count ? y : 0.0f);
        }
        xy.ahead(true);
    };
    float u[MINE], z[MINE], u_before[MINE], z_before[MINE], u_next[MINE], z_next[MINE], dts = 0.0f;
    if (n_subs > 0) {
        fetch(0);
        if (MODE != LOCAL && !a.joined) over_chunks(a, p, 0, 1, p.k, a2, h);
        prepare(0, u, z);
        const bool more = n_subs > 1;
        xu.ahead(more), xd.ahead(more), xz.ahead(more);
        fetch(more);
    }
    // the first group of a block is on its way before the block begins
    constexpr int G = MODE == LOCAL ? GROUP_ONE : GROUP_TWO;
    Group<DT, G> group[2];
    auto words = [&](int i, int s0, Group<DT, G>& x) {
        xB.next_block(), xC.next_block();
        const int last = min(SUB, count - i * SUB) - 1;  // rows behind the end are read as the last one
#pragma unroll
        for (int j = 0; j < G; ++j) {
            xB.load(min(s0 + j, last), x.B[j]);
            if constexpr (MODE != LOCAL) xC.load(min(s0 + j, last), x.C[j]);
        }
    };
    auto prepared = [&](int i, int s0, Group<DT, G>& x) {
#pragma unroll
        for (int j = 0; j < G; ++j) x.in[j] = s_in[i & 1][s0 + j][p.lane];
    };
    if (n_subs > 0) words(0, 0, group[0]);
    for (int i = 0; i < n_subs; ++i) {
        __syncthreads();
        if constexpr (MODE == OUT_MARKS) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) *lane_at(mark + (uint32_t)(n * a.channels), c4) = h[n];
            mark += NS * a.channels;
        }
        prepared(i, 0, group[0]);
        __builtin_amdgcn_sched_barrier(0);
        if (MODE != LOCAL && i > 0) finish(i - 1, u_before, z_before, true);
#pragma unroll
        for (int s0 = 0; s0 < SUB; s0 += G) {
            Group<DT, G>&x = group[s0 / G % 2], &next = group[s0 / G % 2 ^ 1];
            x.here(), x.words_here(x.B);
            if constexpr (MODE != LOCAL) x.words_here(x.C);
            if (s0 + G < SUB) {
                words(i, s0 + G, next);
                prepared(i, s0 + G, next);
            } else {
                const bool more = i + 1 < n_subs;
                xB.ahead(more), xC.ahead(more);
                words(more ? i + 1 : i, 0, next);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                float y = 0.0f;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(x.in[j].x * a2[n]), h[n], x.b(j, n) * x.in[j].y);
                    if constexpr (MODE != LOCAL) y = __builtin_fmaf(h[n], x.c(j, n), y);
                }
                if constexpr (MODE == LOCAL) dts += x.in[j].x;
                else s_y[i & 1][p.q][s0 + j][p.lane] = y;
            }
        }
        prepare(i + 1, u_next, z_next);
        const bool more = i + 2 < n_subs;
        xu.ahead(more), xd.ahead(more), xz.ahead(more);
        fetch(min(i + 2, n_subs - 1));
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            u_before[k] = u[k], z_before[k] = z[k];
            u[k] = u_next[k], z[k] = z_next[k];
        }
    }
    if constexpr (MODE == LOCAL) {
        if (!p.live) return;
        const int64_t r = p.b * a.chunks + p.k;
#pragma unroll
        for (int n = 0; n < NQ; ++n) a.local[state_at(a, p, r, n)] = h[n];
        if (p.q == 0) a.dts[r * a.channels + p.c] = dts;
    } else {
        __syncthreads();
        if (n_subs > 0) finish(n_subs - 1, u_before, z_before, false);
        if (!p.live) return;
        // the state behind the last position: from the chunk that has it, without positions from the first
        if (a.state_out != nullptr && (end > lo || lo == 0) && end <= lo + a.chunk)
#pragma unroll
            for (int n = 0; n < NQ; ++n) a.state_out[state_at(a, p, p.b, n)] = h[n];
        for (int64_t t = lo + (int64_t)n_subs * SUB + p.q; t < hi; t += WAVES) row_mut<DT>(a.y, p.b, t)[p.c] = E::st(0.0f);
    }
}

// Sums over the wavefront of 8 values (dB or dC of two positions) of four pairs of positions.  A step of the butterfly halves
// the values that a lane carries: where two of them meet, one half of the lanes goes on with one, the other with the other.
// join: lanes with the bit go on with b, the others with a.  sum8: value l / 8 of lane l, still spread over its 8 lanes.
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
    return join<8, DPP_ROR8, Add>(v[0], v[1], lane);
}
// Pairs 0 .. 3 (in this order): lane l gets value l / 8 of pair l / 4 % 2 + 2 (l / 2 % 2), the same in lanes 2 i and 2 i + 1.
__device__ __forceinline__ float join01(float a, float b, int lane) { return join<4, DPP_HALF_MIRROR, Add>(a, b, lane); }
__device__ __forceinline__ float join0123(float a, float b, int lane) {
    const float v = join<2, DPP_XOR2, Add>(a, b, lane);
    return v + dpp<DPP_XOR1>(v);
}

// The same rows, which the compiler takes for others: on the way back B and C are loaded again rather than kept (64 scalar
// registers per block, moved to and from vector registers for want of so many).
template <int DT>
__device__ __forceinline__ ScalarRows<DT> again(ScalarRows<DT> x) {
    asm volatile("" : "+s"(x.p));
    return x;
}

// What the backward pass loads of a block's positions, from the chunk's last block to its first.  Where marks do not set the
// block's size it is twice as long, for half the barriers (2 x 16384 positions of 512 channels: 78 -> 72 us; the forward pass,
// of which more wavefronts run at once, 65 -> 69).
constexpr int LOCAL_SUB = 2 * SUB;
template <int DT, bool LOCAL_>
struct BackIn {
    using E = Elem<DT>;
    static constexpr int BLOCK = LOCAL_ ? LOCAL_SUB : SUB, MINE = BLOCK / WAVES;
    LaneRows<DT> xu, xd, xz, xy;
    typename E::T ru[MINE], rd[MINE], rz[MINE], ry[MINE];
    int first;  // this wavefront's first position of a block
    // t: the first position of the block to start with; without a gate z is dy
    __device__ __forceinline__ BackIn(const ScanArgs& a, const Place& p, int64_t t)
        : xu(a.u, p.b, t), xd(a.delta, p.b, t), xz(a.z.p != nullptr ? a.z : a.dy, p.b, t), xy(a.dy, p.b, t), first(p.q * MINE) {}
    __device__ __forceinline__ void back(bool on) {
        xu.template back<BLOCK>(on), xd.template back<BLOCK>(on), xz.template back<BLOCK>(on), xy.template back<BLOCK>(on);
    }
    // left: positions from the block's first one to the end
    __device__ __forceinline__ void fetch(int left, uint32_t& ce) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int s = min(first + k, left - 1);  // rows behind the end are read as the last one
            if constexpr (!LOCAL_) ru[k] = xu.load(s, ce);
            rd[k] = xd.load(s, ce);
            ry[k] = xy.load(s, ce);
            rz[k] = xz.load(s, ce);
        }
    }
};

// The adjoint of the state before a chunk that the chunk's own outputs give (dh from zeros behind it), and its sum of dt, for
// every chunk but the first.
template <int DT>
__global__ void __launch_bounds__(WG) k_scan_bwd_local(const ScanArgs a) {
    using E = Elem<DT>;
    constexpr int BLOCK = LOCAL_SUB, MINE = BLOCK / WAVES;
    __shared__ float2 s_in[2][BLOCK][64];  // dt, g
    const Place p(a, a.chunks - 1, 1);
    const int64_t end = end_of(a, p.b), lo = p.k * a.chunk;
    if (lo >= end) return;
    const int n_subs = (int)ceil_div(min(lo + a.chunk, end) - lo, BLOCK);
    float a2[NQ], dh[NQ] = {}, dts = 0.0f;
    p.decay(a, a2);
    const float bias = a.bias != nullptr ? a.bias[p.cc] : 0.0f;
    const int count = (int)(min(lo + a.chunk, end) - lo);
    const bool gate = a.z.p != nullptr;
    uint32_t ce = p.cc * (uint32_t)sizeof(typename E::T);
    BackIn<DT, true> in(a, p, lo + (n_subs - 1) * BLOCK);
    ScalarRows<DT> xC(a.C, p.b, lo + (n_subs - 1) * BLOCK, p.q);
    auto prepare = [&](int i) {
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = in.first + k;
            const float dt = hw_softplus(E::ld(in.rd[k]) + bias), g = E::ld(in.ry[k]) * (gate ? hw_silu(E::ld(in.rz[k])) : 1.0f);
            s_in[i & 1][at][p.lane] = i * BLOCK + at < count ? make_float2(dt, g) : make_float2(0.0f, 0.0f);
        }
    };
    in.fetch(count - (n_subs - 1) * BLOCK, ce);
    prepare(n_subs - 1);
    in.back(n_subs > 1);
    in.fetch(n_subs > 1 ? BLOCK : count, ce);
    // the last group of a block, which comes first, is on its way before the block begins
    constexpr int G = GROUP_ONE;
    Group<DT, G> group[2];
    auto words = [&](int i, int s0, Group<DT, G>& x) {
        xC.next_block();
        const int last = min(BLOCK, count - i * BLOCK) - 1;  // rows behind the end are read as the last one
#pragma unroll
        for (int j = 0; j < G; ++j) xC.load(min(s0 + j, last), x.C[j]);
    };
    auto prepared = [&](int i, int s0, Group<DT, G>& x) {
#pragma unroll
        for (int j = 0; j < G; ++j) x.in[j] = s_in[i & 1][s0 + j][p.lane];
    };
    words(n_subs - 1, BLOCK - G, group[0]);
    for (int i = n_subs - 1; i >= 0; --i) {
        __syncthreads();
        prepared(i, BLOCK - G, group[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s0 = BLOCK - G; s0 >= 0; s0 -= G) {
            Group<DT, G>&x = group[(BLOCK - G - s0) / G % 2], &next = group[(BLOCK - s0) / G % 2];
            x.here(), x.words_here(x.C);
            if (s0 > 0) {
                words(i, s0 - G, next);
                prepared(i, s0 - G, next);
            } else {
                xC.template back<BLOCK>(i > 0);
                words(max(i - 1, 0), BLOCK - G, next);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = G - 1; j >= 0; --j) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                    dh[n] = __builtin_fmaf(x.c(j, n), x.in[j].y, dh[n]) * __builtin_amdgcn_exp2f(x.in[j].x * a2[n]);
                dts += x.in[j].x;
            }
        }
        if (i > 0) prepare(i - 1);
        in.back(i > 1);
        in.fetch(min(BLOCK, count), ce);
    }
    if (!p.live) return;
    const int64_t r = p.b * a.chunks + p.k;
#pragma unroll
    for (int n = 0; n < NQ; ++n) a.local[state_at(a, p, r, n)] = dh[n];
    if (p.q == 0) a.dts[r * a.channels + p.c] = dts;
}

// ALL: every lane has a channel (channels a multiple of 64), so the stores need no lane mask (2 x 16384 positions of 512 channels 234 us,
// with the mask 237; 32 x 500 of 1024 bfloat16 139 and 141).  What rows of other widths cost beyond that is their stores, which begin
// and end inside cache lines: the whole backward pass of 511 channels 324 us, of 512 281, of 480 291.
template <int DT, bool ALL>
__global__ void __launch_bounds__(WG, 4) k_scan_bwd(const ScanArgs a) {
    using E = Elem<DT>;
    __shared__ float2 s_in[SUB][64];  // dt, dt u
    __shared__ float s_g[SUB][64];
    __shared__ float s_y[WAVES][SUB][64], s_s[WAVES][SUB][64], s_w[WAVES][SUB][64];  // partial sums over the states
    const Place p(a, a.chunks, 0);
    const bool live = ALL || p.live;
    const int64_t end = end_of(a, p.b), lo = p.k * a.chunk;
    const int64_t hi = min(lo + a.chunk, a.length);
    const int n_subs = lo < end ? (int)ceil_div(min(hi, end) - lo, SUB) : 0;
    const bool gate = a.z.p != nullptr;
    float a2[NQ], dh[NQ] = {}, dA[NQ] = {}, dA_all[NQ] = {};
    p.decay(a, a2);
    const float bias = a.bias != nullptr ? a.bias[p.cc] : 0.0f, D = a.D != nullptr ? a.D[p.cc] : 0.0f;
    float dD = 0.0f, dbias = 0.0f, mark[NQ];
    const int count = (int)(min(hi, end) - lo), rows_out = (int)(hi - lo);
    const int64_t t_last = lo + (int64_t)max(n_subs - 1, 0) * SUB;  // the block to start with
    uint32_t ce = p.cc * (uint32_t)sizeof(typename E::T), c4 = p.cc * 4, tid4 = threadIdx.x * 4;  // the lane's channel in bytes
    BackIn<DT, false> in(a, p, t_last);
    LaneRows<DT> yu(a.du, p.b, t_last), yd(a.ddelta, p.b, t_last), yz(gate ? a.dz : a.du, p.b, t_last);
    ScalarRows<DT> xB(a.B, p.b, t_last, p.q), xC(a.C, p.b, t_last, p.q);
    gptr<float> marks = G(a.marks) + ((p.b * a.subs + t_last / SUB) * NS + p.q * NQ) * a.channels;
    gmut<float> bc_out = GM(a.part_bc) + (((int64_t)p.cb * a.batch + p.b) * a.subs + t_last / SUB) * WG;
    auto fetch = [&](int left) {
        in.fetch(left, ce);
#pragma unroll
        for (int n = 0; n < NQ; ++n) mark[n] = *lane_at(marks + (uint32_t)(n * a.channels), c4);
    };
    // Pairs of positions; a block's first one is on its way (in pair[1]) before the block begins.
    Group<DT, 2> pair[2];
    auto words = [&](int s0, int last, Group<DT, 2>& x, const ScalarRows<DT>& fromB, const ScalarRows<DT>& fromC) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            fromB.load(min(s0 + j, last), x.B[j]);
            fromC.load(min(s0 + j, last), x.C[j]);
        }
    };
    // whole: all the block's positions are inside (all blocks but the first one here)
    auto block = [&](int i, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        xB.next_block(), xC.next_block();
        const int t0 = i * SUB;  // in the chunk
        float u[MINE], sig[MINE], dyz[MINE];
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = in.first + k;
            u[k] = own_register(E::ld(in.ru[k]));
            const float dy = E::ld(in.ry[k]), pre = E::ld(in.rd[k]) + bias, z = E::ld(in.rz[k]), sz = hw_sigmoid(z);
            float dt = hw_softplus(pre), g = dy * (gate ? z * sz : 1.0f);
            sig[k] = hw_sigmoid(pre);
            dyz[k] = dy * __builtin_fmaf(z * sz, 1.0f - sz, sz);
            if ((!WHOLE && t0 + at >= count) || !live) dt = g = u[k] = sig[k] = dyz[k] = 0.0f;
            s_in[at][p.lane] = make_float2(dt, dt * u[k]);
            s_g[at][p.lane] = g;
        }
        float h[NQ], e[SUB][NQ], eh[SUB][NQ], half = 0.0f, low = 0.0f, dC = 0.0f, bc = 0.0f;
        static_assert(SUB == 8, "four pairs");
#pragma unroll
        for (int n = 0; n < NQ; ++n) h[n] = live ? mark[n] : 0.0f;
        __syncthreads();
        const int last = WHOLE ? SUB - 1 : count - t0 - 1;  // rows behind the end are read as the last one
        auto prepared = [&](int s0, Group<DT, 2>& x) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                x.in[j] = s_in[s0 + j][p.lane];
                x.g[j] = s_g[s0 + j][p.lane];
            }
        };
        auto issue = [&](int s0, Group<DT, 2>& x, const ScalarRows<DT>& fromB, const ScalarRows<DT>& fromC) {
            words(s0, last, x, fromB, fromC);
            prepared(s0, x);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto here = [&](Group<DT, 2>& x) {
            x.here(), x.words_here(x.B), x.words_here(x.C);
            asm volatile("" : "+v"(x.g[0]), "+v"(x.g[1]));
        };
        prepared(0, pair[0]);
        pair[1].words_here(pair[1].B), pair[1].words_here(pair[1].C);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int w = 0; w < ScalarRows<DT>::WORDS; ++w) pair[0].B[j][w] = pair[1].B[j][w], pair[0].C[j][w] = pair[1].C[j][w];
        float r[8];
#pragma unroll
        for (int s0 = 0; s0 < SUB; s0 += 2) {
            Group<DT, 2>& x = pair[s0 / 2 % 2];
            here(x);
            if (s0 + 2 < SUB) issue(s0 + 2, pair[s0 / 2 % 2 ^ 1], xB, xC);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int s = s0 + j;
                float y = 0.0f;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    e[s][n] = __builtin_amdgcn_exp2f(x.in[j].x * a2[n]);
                    eh[s][n] = e[s][n] * h[n];
                    h[n] = __builtin_fmaf(x.b(j, n), x.in[j].y, eh[s][n]);
                    y = __builtin_fmaf(h[n], x.c(j, n), y);
                    r[j * NQ + n] = x.g[j] * h[n];
                }
                s_y[p.q][s][p.lane] = y;
            }
            // the two positions' dC: value 4 j + n
            const float v = sum8(r, p.lane);
            if (s0 % 4 == 0) half = v;
            else if (s0 == 2) low = join01(half, v, p.lane);
            else dC = join0123(low, join01(half, v, p.lane), p.lane);
        }
        const ScalarRows<DT> xB2 = again(xB), xC2 = again(xC);
#pragma unroll
        for (int s0 = SUB - 2; s0 >= 0; s0 -= 2) {
            Group<DT, 2>& x = pair[s0 / 2 % 2];  // the last one is still here
            if (s0 < SUB - 2) here(x);
            if (s0 > 0) {
                issue(s0 - 2, pair[s0 / 2 % 2 ^ 1], xB2, xC2);
            } else {
                xB.back(i > 0), xC.back(i > 0);
                words(0, i > 0 ? SUB - 1 : last, pair[1], xB, xC);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int j = 1; j >= 0; --j) {
                const int s = s0 + j;
                float sB = 0.0f, sw = 0.0f;
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    dh[n] = __builtin_fmaf(x.c(j, n), x.g[j], dh[n]);
                    sB = __builtin_fmaf(dh[n], x.b(j, n), sB);
                    r[j * NQ + n] = dh[n] * x.in[j].y;
                    const float w = dh[n] * eh[s][n];
                    sw = __builtin_fmaf(w, a2[n], sw);
                    dA[n] = __builtin_fmaf(w, x.in[j].x, dA[n]);
                    dh[n] *= e[s][n];
                }
                s_s[p.q][s][p.lane] = sB;
                s_w[p.q][s][p.lane] = sw;
            }
            const float v = sum8(r, p.lane);
            if (s0 % 4 != 0) half = v;
            else if (s0 == 4) low = join01(v, half, p.lane);
            else bc = join0123(join01(v, half, p.lane), low, p.lane);
            if (s0 == SUB / 2) {  // the next block's loads, where registers come free
                in.back(i > 0);
                marks -= i > 0 ? NS * a.channels : 0;
                fetch(i > 0 ? SUB : count - t0);
            }
        }
        *lane_at(bc_out, tid4) = (p.lane & 1) ? bc : dC;
        bc_out -= WG;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < MINE; ++k) {
            const int at = in.first + k, t = t0 + at;
            const float dt = s_in[at][p.lane].x, g = s_g[at][p.lane];
            float y = D * u[k], sB = 0.0f, sw = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                y += s_y[w][at][p.lane];
                sB += s_s[w][at][p.lane];
                sw += s_w[w][at][p.lane];
            }
            const float ddelta = __builtin_fmaf(u[k], sB, sw * LN2) * sig[k], du = __builtin_fmaf(dt, sB, D * g);
            dD = __builtin_fmaf(g, u[k], dD);
            dbias += ddelta;
            if (live && (WHOLE || t < rows_out)) {
                const bool inside = WHOLE || t < count;
                yu.store(at, ce, inside ? du : 0.0f);
                yd.store(at, ce, inside ? ddelta : 0.0f);
                yz.store(at, ce, !inside ? 0.0f : gate ? dyz[k] * y : du);  // without a gate du once more
            }
        }
        yu.back(true), yd.back(true), yz.back(true);
        if (i % 8 == 0)  // sums of 64 positions at a time: a long sum in one register loses digits
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                dA_all[n] += dA[n];
                dA[n] = 0.0f;
            }
        __syncthreads();
    };
    if (n_subs > 0) {
        fetch(count - (n_subs - 1) * SUB);
        words(0, count - (n_subs - 1) * SUB - 1, pair[1], xB, xC);
        if (a.joined) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) dh[n] = a.local[state_at(a, p, p.b * a.chunks + p.k, n)];
        } else {
            const int after = (int)ceil_div(end, a.chunk) - 1;
            over_chunks(a, p, after, -1, after - p.k, a2, dh);
        }
        block(n_subs - 1, std::false_type());
        for (int i = n_subs - 2; i >= 0; --i) block(i, std::true_type());
    }
    if (live)
        for (int64_t t = lo + (int64_t)n_subs * SUB + p.q; t < hi; t += WAVES) {
            row_mut<DT>(a.du, p.b, t)[p.c] = E::st(0.0f);
            row_mut<DT>(a.ddelta, p.b, t)[p.c] = E::st(0.0f);
            if (gate) row_mut<DT>(a.dz, p.b, t)[p.c] = E::st(0.0f);
        }
    // this chunk's sums for the parameters: [channels][16] of A, [channels] of D, [channels] of the bias
    s_s[p.q][0][p.lane] = dD;
    s_s[p.q][1][p.lane] = dbias;
    __syncthreads();
    if (!live) return;
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

// What the backward pass leaves in parts: dB and dC, the sums over the channel blocks, in the activations' type (zeros behind a
// sequence's end), by the first bc_blocks workgroups; the parameters' gradients, the sums over the chunks, by the others.
template <int DT>
__global__ void __launch_bounds__(WG) k_scan_sums(const ScanArgs a, int64_t bc_blocks, float* dpar) {
    if (blockIdx.x >= bc_blocks) {
        sum_parts<WG / SUM_COLS>(a.part_par, a.batch * a.chunks, (int64_t)(NS + 2) * a.channels, dpar, blockIdx.x - bc_blocks);
        return;
    }
    const int lane = threadIdx.x & 63, q = threadIdx.x >> 6;
    for (int64_t k = blockIdx.x; k < a.batch * a.subs; k += bc_blocks) {
        const int64_t b = k / a.subs, i = k % a.subs;
        // where k_scan_bwd leaves them: see join01 and join0123
        const int64_t end = end_of(a, b), t = i * SUB + ((lane >> 2 & 1) + (lane & 2)) * 2 + (lane >> 5);
        if (t >= a.length) continue;
        float v = 0.0f;
        if (t < end) {
            constexpr int AT_ONCE = 8;
            const float* part = a.part_bc + k * WG + threadIdx.x;
            const int64_t next = a.batch * a.subs * WG;  // the next block of channels
            for (int cb = 0; cb < a.cblocks; cb += AT_ONCE) {
                float x[AT_ONCE];
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) x[j] = part[min(cb + j, a.cblocks - 1) * next];
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) v += cb + j < a.cblocks ? x[j] : 0.0f;
            }
        }
        row_mut<DT>((lane & 1) ? a.dB : a.dC, b, t)[q * NQ + ((lane >> 3) & 3)] = Elem<DT>::st(v);
    }
}

// One position: a lane has the 16 states of its channel, a wavefront 64 channels of some sequences (A and the parameters are
// read once for all of them).  Bound by the states' way in and out: 1000 x 1024, 23 us (131 MB: 5.7 TB/s); 1 x 512, 3.5 us.
template <int DT>
__global__ void __launch_bounds__(WG) k_scan_step(const ScanArgs a, int64_t walkers) {
    using E = Elem<DT>;
    const int lane = threadIdx.x & 63;
    const int64_t k = (int64_t)blockIdx.x * WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = (int)(k % a.cblocks) * 64 + lane;
    const uint32_t cc = (uint32_t)(c < a.channels ? c : a.channels - 1);
    float a2[NS];
#pragma unroll
    for (int n = 0; n < NS; n += 4) {
        const float4 v = reinterpret_cast<const float4*>(a.A)[cc * (NS / 4) + n / 4];
        a2[n] = v.x * LOG2E, a2[n + 1] = v.y * LOG2E, a2[n + 2] = v.z * LOG2E, a2[n + 3] = v.w * LOG2E;
    }
    const float bias = a.bias != nullptr ? a.bias[cc] : 0.0f, D = a.D != nullptr ? a.D[cc] : 0.0f;
    if (c >= a.channels || k >= walkers * a.cblocks) return;
    for (int64_t b = k / a.cblocks; b < a.batch; b += walkers) {
        uint32_t ce = cc * (uint32_t)sizeof(typename E::T), c4 = cc * 4;
        gmut<float> st = GM(a.state_out) + b * NS * a.channels;
        float h[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = *lane_at(st + (uint32_t)(n * a.channels), c4);
        const float u = E::ld(LaneRows<DT>(a.u, b, 0).load(0, ce));
        const float dt = hw_softplus(E::ld(LaneRows<DT>(a.delta, b, 0).load(0, ce)) + bias);
        const float z = a.z.p != nullptr ? E::ld(LaneRows<DT>(a.z, b, 0).load(0, ce)) : 0.0f;
        float B[NS], C[NS];
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            uint32_t w[ScalarRows<DT>::WORDS], v[ScalarRows<DT>::WORDS];
            ScalarRows<DT>(a.B, b, 0, i).load(0, w);
            ScalarRows<DT>(a.C, b, 0, i).load(0, v);
#pragma unroll
            for (int j = 0; j < NQ; ++j) B[i * NQ + j] = ScalarRows<DT>::value(w, j), C[i * NQ + j] = ScalarRows<DT>::value(v, j);
        }
        const float du = dt * u;
        float y = D * u;
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * a2[n]), h[n], B[n] * du);
            y = __builtin_fmaf(h[n], C[n], y);
            *lane_at(st + (uint32_t)(n * a.channels), c4) = h[n];
        }
        if (a.z.p != nullptr) y *= hw_silu(z);
        LaneRows<DT>(a.y, b, 0).store(0, ce, y);
    }
}

Rows rows(const boa_rows& r) { return {r.p, r.batch_stride, r.row_stride}; }

// The split over the length: chunks of a multiple of SUB positions, as many as give the wanted workgroups, at least MIN_CHUNK
// positions each and at most MAX_CHUNKS.
struct Plan {
    int chunks;
    int64_t chunk;
};
// Workgroups: of sequences as long as the batch, six per CU in the forward pass and four in the backward pass, which is what
// its registers let run at once (2 x 16384 positions of 512 channels: 4 and 6 per CU forward 131 and 129 us, backward 248
// and 273; 4 x 4097 of 1024 in bfloat16 forward 92 and 88).  Where lengths differ, smaller ones even out what the CUs have to do
// (32 sequences of up to 500 positions, 1024 channels, bfloat16: forward 84 us with 1024, 68 with 2048, 64 with 4096; backward
// 194, 161, 142).  The number is reached by rounding up, so a batch that has almost as many by itself is cut in two: 1000 positions
// of 512 channels, float32, forward with 96, 128 and 191 sequences 321, 398 and 571 us (not split 283, 321, 443), backward 696, 876
// and 1270 (684, 830, 1237); up to 500 positions of 1024, bfloat16, 64, 128 and 192 sequences, forward 151, 294, 390 (125, 193,
// 249), backward 327, 638, 891 (296, 510, 692).
int64_t wanted_workgroups(const boa_scan* s, bool backward) { return s->lens ? 4096 : backward ? 1024 : 1536; }
constexpr int64_t MIN_CHUNK = 64;
// From more chunks than this on they are joined by a kernel of its own: to go over the chunks before its own costs a workgroup
// of the last chunk 0.3 us for each, and reads them for every workgroup again (2 x 16384 positions of 512 channels: forward
// kernel 129 us, with k_scan_join 97 + 7; backward, of 64 chunks, 241 and 228 + 7; 24 chunks of the prompt above 89 and 84 + 7; 16 of
// 8 x 1000 forward 32.5 and 28.7 + 6, backward 63.5 and 57.5 + 6).
constexpr int JOIN_FROM = 32;
Plan plan(const boa_scan* s, bool backward) {
    const int64_t blocks = s->batch * ceil_div(s->channels, 64);
    int64_t n = ceil_div(wanted_workgroups(s, backward), blocks > 0 ? blocks : 1);
    n = n < MAX_CHUNKS ? n : MAX_CHUNKS;
    int64_t chunk = ceil_div(ceil_div(s->length, n), SUB) * SUB;
    chunk = chunk > MIN_CHUNK ? chunk : MIN_CHUNK;
    n = ceil_div(s->length, chunk);
    return {(int)(n > 1 ? n : 1), chunk};
}

dim3 join_grid(const ScanArgs& a) { return dim3((uint32_t)ceil_div(a.batch * NS * a.channels, 64)); }
dim3 join_block(const ScanArgs& a) { return dim3(64 * (uint32_t)ceil_div(a.chunks, JOIN_EACH)); }

// Workspace, in floats: chunk states and sums of dt (more than one chunk), then in the backward pass the partial sums.
struct Work {
    int64_t local, dts, bc, par;
    int64_t bytes() const { return (local + dts + bc + par) * (int64_t)sizeof(float); }
};
Work work_of(const boa_scan* s, bool backward) {
    Work w = {};
    if (s->batch < 1 || s->length < 1) return w;
    const Plan p = plan(s, backward);
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

// Rows are read at 32-bit offsets from a block's first; those of B and C four values at a time at uniform addresses, which have
// to be multiples of 4 bytes.
bool stride_ok(const boa_rows& r) { return !r.p || (r.row_stride >= 0 && r.row_stride <= BOA_SCAN_MAX_ROW_STRIDE); }
bool bc_aligned(const boa_scan* s, const boa_rows& r, bool step) {
    return s->dtype == BOA_DT_F32 || ((uintptr_t)r.p % 4 == 0 && r.batch_stride % 2 == 0 && (step || r.row_stride % 2 == 0));
}

// Looks at the members that the call uses: a step has no rows one behind the other, the backward pass no y.
enum Pass { FORWARD, BACKWARD, STEP };
int check_scan(const char* who, const boa_scan* s, ScanArgs& a, Pass pass) {
    if (!s) return boa_fail(BOA_ERR_ARG, "%s: null arguments", who);
    if (s->dtype < BOA_DT_F32 || s->dtype > BOA_DT_F16) return boa_fail(BOA_ERR_ARG, "%s: unknown type %d", who, s->dtype);
    if (s->batch < 0 || s->length < 0 || s->channels < 1 || s->channels > BOA_OPS_MAX_CHANNELS)
        return boa_fail(BOA_ERR_ARG, "%s: need batch, length >= 0 and 1 <= channels <= %d (got %lld, %lld, %d)", who,
                        BOA_OPS_MAX_CHANNELS, (long long)s->batch, (long long)s->length, s->channels);
    if (s->batch > 0 && s->length > 0) {
        if (!s->u.p || !s->delta.p || !s->b.p || !s->c.p || !s->a) return boa_fail(BOA_ERR_ARG, "%s: null pointer", who);
        for (const boa_rows* r : {&s->u, &s->delta, &s->z, &s->b, &s->c, pass == FORWARD ? &s->y : &s->u})
            if (pass != STEP && !stride_ok(*r))
                return boa_fail(BOA_ERR_ARG, "%s: rows have to be 0 to %d values apart", who, BOA_SCAN_MAX_ROW_STRIDE);
        if (!bc_aligned(s, s->b, pass == STEP) || !bc_aligned(s, s->c, pass == STEP))
            return boa_fail(BOA_ERR_ARG, "%s: rows of B and C of 16-bit types have to begin at multiples of 4 bytes", who);
    }
    a = ScanArgs{};
    a.u = rows(s->u), a.delta = rows(s->delta), a.z = rows(s->z), a.B = rows(s->b), a.C = rows(s->c), a.y = rows(s->y);
    a.A = s->a, a.D = s->d, a.bias = s->delta_bias, a.lens = s->lens, a.state_in = s->state_in, a.state_out = s->state_out;
    a.marks = s->marks, a.channels = s->channels, a.cblocks = (int)ceil_div(s->channels, 64);
    a.batch = s->batch, a.length = s->length, a.subs = ceil_div(s->length, SUB);
    const Plan pl = plan(s, pass == BACKWARD);
    a.chunks = pl.chunks, a.chunk = pl.chunk, a.joined = pl.chunks > JOIN_FROM;
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
    const int rc = check_scan("boa_selective_scan_fwd", s, a, FORWARD);
    if (rc != BOA_OK) return rc;
    if (a.batch == 0 || (a.length == 0 && !a.state_out)) return BOA_OK;
    if (!a.A || (a.length > 0 && !a.y.p)) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_fwd: null pointer");
    if (a.state_out && a.state_out == a.state_in)  // read by chunks that run beside the one that writes it
        return boa_fail(BOA_ERR_ARG, "boa_selective_scan_fwd: state_out must be another buffer than state_in");
    const Work w = work_of(s, false);
    if (w.bytes() > 0 && (!d_work || work_bytes < w.bytes()))
        return boa_fail(BOA_ERR_ARG, "boa_selective_scan_fwd: workspace of %lld bytes, needs %lld", (long long)work_bytes,
                        (long long)w.bytes());
    lay_out(a, w, d_work);
    return with_dtype(s->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        const uint32_t blocks = (uint32_t)(a.batch * a.cblocks);
        if (a.chunks > 1) {
            hipLaunchKernelGGL((k_scan_fwd<DT, LOCAL>), dim3(blocks * (a.chunks - 1)), dim3(WG), 0, (hipStream_t)stream, a);
            BOA_HIP_TRY(hipGetLastError());
            if (a.joined) {
                hipLaunchKernelGGL((k_scan_join<false>), join_grid(a), join_block(a), 0, (hipStream_t)stream, a);
                BOA_HIP_TRY(hipGetLastError());
            }
        }
        if (a.marks != nullptr)
            hipLaunchKernelGGL((k_scan_fwd<DT, OUT_MARKS>), dim3(blocks * a.chunks), dim3(WG), 0, (hipStream_t)stream, a);
        else
            hipLaunchKernelGGL((k_scan_fwd<DT, OUT>), dim3(blocks * a.chunks), dim3(WG), 0, (hipStream_t)stream, a);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}

extern "C" int boa_selective_scan_bwd(const boa_scan* s, void* d_work, int64_t work_bytes, void* stream) {
    ScanArgs a;
    const int rc = check_scan("boa_selective_scan_bwd", s, a, BACKWARD);
    if (rc != BOA_OK) return rc;
    const bool any = a.batch > 0 && a.length > 0;
    if (!s->dpar) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_bwd: null pointer");
    if (any && (!s->dy.p || !s->du.p || !s->ddelta.p || !s->db.p || !s->dc.p || !s->marks || (s->z.p && !s->dz.p)))
        return boa_fail(BOA_ERR_ARG, "boa_selective_scan_bwd: null pointer");
    for (const boa_rows* r : {&s->dy, &s->du, &s->ddelta, s->z.p ? &s->dz : &s->du})
        if (any && !stride_ok(*r))
            return boa_fail(BOA_ERR_ARG, "boa_selective_scan_bwd: rows have to be 0 to %d values apart", BOA_SCAN_MAX_ROW_STRIDE);
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
                if (a.joined) {
                    hipLaunchKernelGGL((k_scan_join<true>), join_grid(a), join_block(a), 0, st, a);
                    BOA_HIP_TRY(hipGetLastError());
                }
            }
            if (a.channels % 64 == 0)
                hipLaunchKernelGGL((k_scan_bwd<DT, true>), dim3(blocks * a.chunks), dim3(WG), 0, st, a);
            else
                hipLaunchKernelGGL((k_scan_bwd<DT, false>), dim3(blocks * a.chunks), dim3(WG), 0, st, a);
            BOA_HIP_TRY(hipGetLastError());
            const int64_t bc = min(a.batch * a.subs, MAX_BLOCKS / 2);
            hipLaunchKernelGGL((k_scan_sums<DT>), dim3((uint32_t)(bc + ceil_div((int64_t)(NS + 2) * a.channels, SUM_COLS))), dim3(WG),
                               0, st, a, bc, s->dpar);
            BOA_HIP_TRY(hipGetLastError());
            return (int)BOA_OK;
        });
        if (launched != BOA_OK) return launched;
    } else {
        BOA_HIP_TRY(launch_sum_parts(nullptr, 0, (int64_t)(NS + 2) * a.channels, s->dpar, st));  // zeros
    }
    return BOA_OK;
}

extern "C" int boa_selective_scan_step(const boa_scan* s, void* stream) {
    ScanArgs a;
    const int rc = check_scan("boa_selective_scan_step", s, a, STEP);
    if (rc != BOA_OK) return rc;
    if (a.batch == 0) return BOA_OK;
    if (a.length != 1) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_step: one position per sequence (got %lld)", (long long)a.length);
    if (!a.y.p || !a.state_out) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_step: null pointer");
    if ((uintptr_t)a.A % 16 != 0) return boa_fail(BOA_ERR_ARG, "boa_selective_scan_step: a has to begin at a multiple of 16 bytes");
    // wavefronts for each block of channels: as many as run at once on 256 CUs (8 on each of their SIMDs), or one per sequence
    const int64_t walkers = min(a.batch, ceil_div(8192, a.cblocks));
    return with_dtype(s->dtype, [&](auto dt) {
        hipLaunchKernelGGL((k_scan_step<decltype(dt)::value>), dim3((uint32_t)ceil_div(walkers * a.cblocks, WAVES)), dim3(WG), 0,
                           (hipStream_t)stream, a, walkers);
        BOA_HIP_TRY(hipGetLastError());
        return (int)BOA_OK;
    });
}
