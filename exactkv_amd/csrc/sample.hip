// One token a row from logits, with temperature, top-k, top-p and min-p and given uniform numbers, for
// gfx950 (no counterpart in the reference, whose engine decodes greedily, exactkv/engine.py:93-95).
//
// Of a row's logits l, with M the largest and t the temperature, the weights are w = exp((l - M) / t). Ordered by
// value, equal ones by index, these stay, each time a beginning of the row: those with w >= min_p; of them the first
// top_k; of these the ones before whose weights add up to less than top_p of all. Of what stays, S its sum, the token
// is the first one with which the running sum passes u S.
//
// Every cut is thus a place in one order, the first where a running count or sum passes a bound, and is found without
// a sort of the row: with y = 32 log2(1 / w), weights are counted and added up in bins of one y; the bin in which a bound
// is passed is known from the bins' sums (to a few bins, where the bound depends on a sum that is known to a bin); the
// tokens of these bins alone are collected, sorted and added up one by one. With top_k up to 2,048 all tokens down to the
// k-th's bin are collected at once, and no other weight is computed.
//
// Weights are made in fp64: w = 2^-(i / 32) 2^-(f / 32) with i and f the whole and the rest of y, the second factor a polynomial
// (fifth degree, through 1 at f = 0, to 2^-51). They are rounded to whole multiples of 2^-43 of the largest and added up as
// whole numbers, so that sums do not depend on the order in which they are taken; a bin's factor is applied to its sum. A
// weight in a sum is thus off by up to 2^-44 absolute, and one below 2^-44 is 0: all of a vocabulary of 2^19 together by less
// than 2^-25 of the sum, so that cuts and draws fall where the formula in 64 bits has them but for bounds nearer to a
// running sum than that. The log-probability that is returned takes the token's own y, which is not rounded so.
//
// Rows of up to 8,192 logits take one launch, a workgroup each; longer ones four, cut into pieces: largest, bins, collected,
// taken. 256 rows of 152,064 bf16 logits (78 MB): 19, 33, 25 and 9.4 us, the second bound by its fp64 operations, the first and the
// third by memory (3.1 to 4.1 TB/s); 61 of 50,257 fp32 (12 MB): 4.9, 8.4, 12 and 8.4; one of 128,256: 4.0, 4.9, 6.6
// and 6.4, each a chain of launches, loads and barriers.
//
// A row of which more than kList tokens lie in the bins in question, or more than kLocal of them in one piece, is walked again
// by one workgroup in the last launch: flat rows, and with 1,024 rows or more (a piece each) a top_k of 1,025 to 2,048.
// 64 rows of 128,256: 55 us, at a temperature of 50 (nearly all tokens in a few bins) 314, with top_p 0.9 as well 545; 1,024 of
// 50,257 with top_k 1,500 298 us, 2,049 (by sums) 131.
#include "errors.hpp"
#include "common.hpp"
#include "../../include/exactkv.h"

namespace exkv {

constexpr int kThreads = 1024, kList = 4096;
constexpr int kPerOctave = 32, kReach = 44 * kPerOctave;   // bins of a factor of 2; weights from bin kReach on are 0
constexpr int kBins = 2048;                                // places for them, two a thread
constexpr double kOne = 0x1p43;                            // a weight of 1

struct SampleArgs {
    const void* logits;                // [B, V], row stride in elements
    int64_t stride;
    int B, V;
    const float *u, *t, *p, *m;        // [B]; t, p, m nullptr: the values below
    const int32_t* k;
    float t0, p0, m0;
    int k0;
    int64_t* token;
    float* logprob;                    // may be nullptr
    // rows cut into `pieces` of `per` logits: their maxima [B, pieces] (order << 32 | ~index), a row's bins [B, kReach],
    // what is collected of it [B, kList], and how much [B]
    int pieces, per;
    uint64_t *best, *mass, *list;
    uint32_t *count, *n;
    struct Ranges* ranges;             // what a row's bins say [B]
};

// A logit's place in the order of all; -0 as 0. NaN: 0. kMinusInf: the least that can be drawn is above it.
constexpr uint32_t kMinusInf = ~0xFF800000u;
__device__ inline uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0u : (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}
__device__ inline float of_order(uint32_t k) { return __uint_as_float((k & 0x80000000u) != 0 ? k & 0x7FFFFFFFu : ~k); }
// A token as one number: ascending in the order of the tokens.
__device__ inline uint64_t token_of(float l, int j) { return (uint64_t)~order_of(l) << 32 | (uint32_t)j; }
__device__ inline float logit_of(uint64_t token) { return of_order(~(uint32_t)(token >> 32)); }

enum LogitType { kBf16 = 0, kFp16 = 1, kFp32 = 2 };
template <int TYPE>
struct Logits {
    static constexpr int N = TYPE == kFp32 ? 4 : 8;    // of 16 bytes
    static constexpr int SIZE = TYPE == kFp32 ? 4 : 2;
    __device__ static float one(const uint8_t* p) {
        if constexpr (TYPE == kFp32) return *reinterpret_cast<const float*>(p);
        const uint16_t x = *reinterpret_cast<const uint16_t*>(p);
        if constexpr (TYPE == kBf16) return __uint_as_float((uint32_t)x << 16);
        return (float)__builtin_bit_cast(_Float16, x);
    }
    __device__ static float at(const uint32_t* x, int i) {
        if constexpr (TYPE == kFp32) return __uint_as_float(x[i]);
        const uint32_t d = x[i / 2];
        if constexpr (TYPE == kBf16) return __uint_as_float((i & 1) != 0 ? d & 0xFFFF0000u : d << 16);
        return (float)__builtin_bit_cast(_Float16, (uint16_t)((i & 1) != 0 ? d >> 16 : d));
    }
};

// 2^-(j / 32)
__constant__ double kOctave[kPerOctave] = {
    0x1.0000000000000p+0, 0x1.f50765b6e4540p-1, 0x1.ea4afa2a490dap-1, 0x1.dfc97337b9b5fp-1, 0x1.d5818dcfba487p-1, 0x1.cb720dcef9069p-1,
    0x1.c199bdd85529cp-1, 0x1.b7f76f2fb5e47p-1, 0x1.ae89f995ad3adp-1, 0x1.a5503b23e255dp-1, 0x1.9c49182a3f090p-1, 0x1.93737b0cdc5e5p-1,
    0x1.8ace5422aa0dbp-1, 0x1.82589994cce13p-1, 0x1.7a11473eb0187p-1, 0x1.71f75e8ec5f74p-1, 0x1.6a09e667f3bcdp-1, 0x1.6247eb03a5585p-1,
    0x1.5ab07dd485429p-1, 0x1.5342b569d4f82p-1, 0x1.4bfdad5362a27p-1, 0x1.44e086061892dp-1, 0x1.3dea64c123422p-1, 0x1.371a7373aa9cbp-1,
    0x1.306fe0a31b715p-1, 0x1.29e9df51fdee1p-1, 0x1.2387a6e756238p-1, 0x1.1d4873168b9aap-1, 0x1.172b83c7d517bp-1, 0x1.11301d0125b51p-1,
    0x1.0b5586cf9890fp-1, 0x1.059b0d3158574p-1};

// 2^-(f / 32) for 0 <= f < 1 in multiples of 2^-43: 1 + f q(f), q through (2^-(f / 32) - 1) / f at the five Chebyshev
// nodes of the interval (2^-51.6 off at most). The last step adds 2^52 as well, so that it rounds to a whole number,
// which the low bits then hold.
__device__ inline uint64_t part_of(double f) {
    double x = -0x1.5a647394e5de0p-35 * kOne;
    x = fma(x, f, 0x1.3b27f90273e58p-27 * kOne);
    x = fma(x, f, -0x1.c6b08b7b3d765p-20 * kOne);
    x = fma(x, f, 0x1.ebfbdff7af203p-13 * kOne);
    x = fma(x, f, -0x1.62e42fefa399fp-6 * kOne);
    x = fma(x, f, kOne + 0x1p52);
    return (uint64_t)__double_as_longlong(x) & 0xFFFFFFFFFFFFFull;
}
// The whole and the rest of y, from kBase + y.
constexpr double kBase = 2048.0;
static_assert(kReach < 2048, "y below kBase");
__device__ inline int whole_of(double y) { return (int)((uint32_t)(__double_as_longlong(y) >> 41) & 0x7FFu); }
__device__ inline double rest_of(double y) {
    return __longlong_as_double((__double_as_longlong(y) & 0x1FFFFFFFFFFll) | 0x40A0000000000000ll) - kBase;
}
// A sum of such parts in bin i, in weights.
__device__ inline uint64_t in_bin(uint64_t parts, int i, double octave) {
    return (uint64_t)rint(__builtin_amdgcn_ldexp((double)parts * octave, -(i / kPerOctave)));
}

// A row's settings, and with its largest logit what its weights go by.
struct Settings {
    float t, p, m, u;
    int k;
    __device__ Settings(const SampleArgs& a, int b)
        : t(a.t != nullptr ? a.t[b] : a.t0), p(a.p != nullptr ? a.p[b] : a.p0), m(a.m != nullptr ? a.m[b] : a.m0), u(a.u[b]),
          k(a.k != nullptr ? a.k[b] : a.k0) {}
    __device__ bool few() const { return k > 0 && k <= kList / 2; }     // collected by counts alone
};
struct Row {
    double top, per_bin, limit;        // the largest logit; bins of a logit; the last y that counts
    const double* octave;              // kOctave in LDS
    float top32, p, u0;
    int k;
    bool none, greedy, odd, few;       // odd: the largest is infinite
    __device__ __attribute__((always_inline)) Row(const Settings& set, uint64_t best, const double* table) : octave(table), p(set.p), u0(set.u), k(set.k), few(set.few()) {
        const float t = set.t, m = set.m;
        none = (uint32_t)(best >> 32) <= kMinusInf;
        greedy = none || !(t > 0.f);
        top32 = of_order((uint32_t)(best >> 32));
        odd = top32 == INFINITY;
        top = (double)top32;
        per_bin = kPerOctave * 1.4426950408889634 / (double)t;
        limit = kBase + kReach - 0x1p-40;
        if (!(m <= 0.f)) limit = fmin(limit, m < 1.f ? kBase - (double)kPerOctave * log2((double)m) : kBase);
    }
    __device__ double u() const { return u0 > 0.f ? fmin((double)u0, 1.0 - 0x1p-24) : 0.0; }
    // 2^11 + y, rounded to 41 bits behind the point, so that its bits hold y's whole and its rest: ascends as l falls; not
    // within the limit (NaN too): a weight of 0.
    __device__ double place(float l) const { return fma(top - (double)l, per_bin, kBase); }
    __device__ double any_place(float l) const { return l == top32 ? kBase : place(l); }
    __device__ int bin(float l) const {
        const double y = any_place(l);
        return y <= limit ? whole_of(y) : kReach;
    }
    __device__ uint64_t weight(float l) const {
        const double y = any_place(l);
        if (!(y <= limit)) return 0;
        const int i = whole_of(y);
        return in_bin(part_of(rest_of(y)), i, octave[i & (kPerOctave - 1)]);
    }
};

// Inclusive sums across the lanes of a wavefront, by the steps of wave_incl_scan.
template <int CTRL, int ROWS>
__device__ inline uint64_t moved(uint64_t x) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ inline uint64_t wave_incl_sum(uint64_t x) {
    x += moved<0x111, 0xf>(x);
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);
    x += moved<0x143, 0xc>(x);
    return x;
}
// The first of the wavefronts' lowest values, `none` where a lane has none: to *at, one atomic a wavefront. (A lane's value
// lies below those of the lanes behind it.)
__device__ inline void first_of(int x, int none, int* at) {
    const uint64_t lanes = __ballot(x != none);
    if (lanes == 0) return;
    const int first = __builtin_amdgcn_readlane(x, __builtin_ctzll(lanes));
    if ((threadIdx.x & 63) == 0) atomicMin(at, first);
}

// Shared memory of a row's workgroup.
struct Shared {
    double octave[kPerOctave];
    uint64_t mass[kBins];              // bins, then their running sums
    uint64_t list[kList];              // tokens
    uint32_t count[kBins];
    uint64_t wave_mass[16];
    uint32_t wave_count[16];
    uint64_t lo, hi;                   // tokens
    uint32_t n;
    int found, at[2];
    uint32_t found_count;
    uint64_t found_mass;
};

// Exclusive sums over the workgroup's threads of (c, m).
template <int WAVES>
__device__ inline void block_excl(uint32_t& c, uint64_t& m, uint32_t* sc, uint64_t* sm) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t ci = (uint32_t)wave_incl_scan((int)c);
    const uint64_t mi = wave_incl_sum(m);
    __syncthreads();
    if (lane == 63) {
        sc[w] = ci;
        sm[w] = mi;
    }
    __syncthreads();
    c = ci - c;
    m = mi - m;
    for (int i = 0; i < w; ++i) {
        c += sc[i];
        m += sm[i];
    }
}
template <int WAVES>
__device__ inline uint64_t block_largest(uint64_t best, uint64_t* s) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) best = max(best, s[i]);
    return best;
}

// A bound on the running count or sum, which the first token that satisfies it passes.
struct Bound {
    enum { kRank, kReaches, kPasses } kind;
    uint32_t rank;
    double x;
    __device__ bool passed(uint32_t c, uint64_t m) const {
        return kind == kRank ? c >= rank : kind == kReaches ? (double)m >= x : (double)m > x;
    }
};

// Logits from .. to - 1 of a row, as a workgroup of THREADS looks at them: 16-byte pieces wherever they lie, ascending for a
// thread, what is behind the end as -infinity.
template <int TYPE, int THREADS>
struct MemoryRow {
    static constexpr int N = Logits<TYPE>::N, SIZE = Logits<TYPE>::SIZE, STEP = THREADS * N;
    const uint8_t* p;
    int from, to;
    __device__ MemoryRow(const SampleArgs& a, int b, int f, int t) : p((const uint8_t*)a.logits + b * a.stride * SIZE), from(f), to(t) {}
    __device__ float one(int j) const { return Logits<TYPE>::one(p + (int64_t)j * SIZE); }
    __device__ void load(int j, uint32_t (&x)[4]) const {
        if (j + N <= to) {
            __builtin_memcpy(x, p + (int64_t)j * SIZE, 16);
            return;
        }
        constexpr uint32_t NONE = TYPE == kFp32 ? 0xFF800000u : TYPE == kBf16 ? 0xFF80FF80u : 0xFC00FC00u;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = NONE;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (j + e >= to) continue;
            const uint8_t* at = p + (int64_t)(j + e) * SIZE;
            if constexpr (SIZE == 4) {
                x[e] = *reinterpret_cast<const uint32_t*>(at);
            } else {
                const uint32_t v = *reinterpret_cast<const uint16_t*>(at);
                x[e / 2] = e % 2 != 0 ? (x[e / 2] & 0xFFFFu) | v << 16 : (x[e / 2] & 0xFFFF0000u) | v;
            }
        }
    }
    // f(piece, index of its first logit): U at a time, the next U on their way; the code of f stands here U + 1 times
    template <int U = 2, class F>
    __device__ void pieces(F f) const {
        int j = from + (int)threadIdx.x * N;
        uint32_t x[U][4] = {};
        auto ahead = [&](int at) {
            if (at + (U - 1) * STEP + N <= to)
#pragma unroll
                for (int i = 0; i < U; ++i) __builtin_memcpy(x[i], p + (int64_t)(at + i * STEP) * SIZE, 16);
        };
        ahead(j);
#pragma unroll 1
        for (; j + (U - 1) * STEP + N <= to; j += U * STEP) {
            uint32_t u[U][4];
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int d = 0; d < 4; ++d) u[i][d] = x[i][d];
            ahead(j + U * STEP);
#pragma unroll
            for (int i = 0; i < U; ++i) f(u[i], j + i * STEP);
        }
#pragma unroll 1
        for (; j < to; j += STEP) {
            load(j, x[0]);
            f(x[0], j);
        }
    }
    // f(logit, index): less code
    template <class F>
    __device__ void each(F f) const {
#pragma unroll 1
        for (int j = from + (int)threadIdx.x * N; j < to; j += STEP) {
            uint32_t x[4];
            load(j, x);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (j + e < to) f(Logits<TYPE>::at(x, e), j + e);
        }
    }
    // the largest logit of this thread's and the first place of it: order << 32 | ~index
    __device__ uint64_t largest() const {
        float top = -INFINITY;
        int at = -1;
        pieces<4>([&](const uint32_t (&x)[4], int j) {
            float m = Logits<TYPE>::at(x, 0);
#pragma unroll
            for (int e = 1; e < N; ++e) m = fmaxf(m, Logits<TYPE>::at(x, e));
            if (m > top) {
                top = m;
                at = j;
            }
        });
        if (at < 0) return 0;
        while (!(one(at) == top)) ++at;
        return (uint64_t)order_of(top) << 32 | ~(uint32_t)at;
    }
};

// A row that needs no draw: its largest logit, or nothing to draw at all.
__device__ inline void take_largest(const SampleArgs& a, int b, const Row& row, uint64_t best) {
    if (threadIdx.x != 0) return;
    a.token[b] = row.none ? 0 : (int64_t)~(uint32_t)best;
    if (a.logprob != nullptr) a.logprob[b] = row.none ? -INFINITY : 0.f;
    if (row.none) report_error(kErrLogits);
}
__device__ inline void take(const SampleArgs& a, int b, const Row& row, uint64_t token, uint64_t S) {
    if (threadIdx.x != 0) return;
    a.token[b] = (int64_t)(uint32_t)token;
    // log w - log S, w from its place and not as it is added up: of an unlikely token's few multiples of 2^-43 a logarithm
    // would be off by up to 0.1
    if (a.logprob != nullptr)
        a.logprob[b] = (float)(0.6931471805599453 / kPerOctave * (kBase - row.any_place(logit_of(token))) - log((double)S / kOne));
}

// x of lane ^ D.
template <int D>
__device__ inline uint64_t across(uint64_t x) {
    static_assert(D < 16, "a row of lanes");
    auto half = [](uint32_t v) -> uint32_t {
        if constexpr (D == 4) v = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x1B, 0xf, 0xf, true);   // ^ 3, then ^ 7
        constexpr int CTRL = D == 1 ? 0xB1 : D == 2 ? 0x4E : D == 4 ? 0x141 : 0x128;
        return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
    };
    return (uint64_t)half((uint32_t)(x >> 32)) << 32 | half((uint32_t)x);
}
// The lower (or higher) of a pair of lanes' values, D apart.
template <int D>
__device__ inline uint64_t one_of_pair(uint64_t x, bool lower) {
    uint64_t a = x, b;
    if constexpr (D < 16) {
        b = across<D>(x);
    } else {
        const uint32_t l = (uint32_t)x, h = (uint32_t)(x >> 32);
        const auto pl = D == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false) : __builtin_amdgcn_permlane32_swap(l, l, false, false);
        const auto ph = D == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false) : __builtin_amdgcn_permlane32_swap(h, h, false, false);
        a = (uint64_t)ph[0] << 32 | pl[0];
        b = (uint64_t)ph[1] << 32 | pl[1];
    }
    return (a < b) == lower ? a : b;
}

// The list's n tokens in order. Up to 256: by counting, for each, those before it, a quarter of them a thread. Up to 1,024:
// by a bitonic sort of one token a thread, whose exchanges within a wavefront stay in registers (rows of up to 640:
// 9.4 us in the last launch, with the sort below 19). More: by the same network over LDS, where those within 128 neighbours are one wavefront's own and need no barrier.
__device__ inline void sort_list(Shared& s, int n) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (n <= 256) {                                    // uniform
        uint32_t* before = reinterpret_cast<uint32_t*>(s.list + 1024);
        const int t = tid & 255, part = tid >> 8, per = (n + 3) / 4;
        const uint64_t x = t < n ? s.list[t] : 0;
        uint32_t at = 0;
        const int end = min(n, (part + 1) * per);
        if (t < n)
#pragma unroll 8
            for (int i = part * per; i < end; ++i) at += s.list[i] < x;
        before[tid] = at;
        __syncthreads();
        if (tid < n) s.list[before[tid] + before[tid + 256] + before[tid + 512] + before[tid + 768]] = x;
        __syncthreads();
        return;
    }
    if (n <= kThreads) {                               // uniform
        uint64_t x = tid < n ? s.list[tid] : ~0ull;
        int side = 0;                                  // halves of the list in turn, so that an exchange takes one barrier
        auto merge = [&](auto size) {
            constexpr int K = decltype(size)::value;
            const bool up = (tid & K) == 0;
            auto far = [&](int d) {
                side ^= 1024;
                s.list[side + tid] = x;
                __syncthreads();
                const uint64_t y = s.list[side + (tid ^ d)];
                x = (x < y) == (((tid & d) == 0) == up) ? x : y;
            };
            if constexpr (K >= 1024) far(512);
            if constexpr (K >= 512) far(256);
            if constexpr (K >= 256) far(128);
            if constexpr (K >= 128) far(64);
            if constexpr (K >= 64) x = one_of_pair<32>(x, ((tid & 32) == 0) == up);
            if constexpr (K >= 32) x = one_of_pair<16>(x, ((tid & 16) == 0) == up);
            if constexpr (K >= 16) x = one_of_pair<8>(x, ((tid & 8) == 0) == up);
            if constexpr (K >= 8) x = one_of_pair<4>(x, ((tid & 4) == 0) == up);
            if constexpr (K >= 4) x = one_of_pair<2>(x, ((tid & 2) == 0) == up);
            x = one_of_pair<1>(x, ((tid & 1) == 0) == up);
        };
        merge(std::integral_constant<int, 2>{});
        merge(std::integral_constant<int, 4>{});
        merge(std::integral_constant<int, 8>{});
        merge(std::integral_constant<int, 16>{});
        merge(std::integral_constant<int, 32>{});
        merge(std::integral_constant<int, 64>{});
        merge(std::integral_constant<int, 128>{});
        merge(std::integral_constant<int, 256>{});
        merge(std::integral_constant<int, 512>{});
        if (n > 512) merge(std::integral_constant<int, 1024>{});   // uniform
        __syncthreads();
        s.list[tid] = x;
        __syncthreads();
        return;
    }
    int size = 2048;
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kThreads) s.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int d = k >> 1; d > 0; d >>= 1) {
            for (int i = tid; i < size / 2; i += kThreads) {
                const int a = (i & ~(d - 1)) * 2 + (i & (d - 1)), b = a + d;
                const uint64_t x = s.list[a], y = s.list[b];
                if ((x > y) == ((a & k) == 0)) {
                    s.list[a] = y;
                    s.list[b] = x;
                }
            }
            if (d > 64 || (d == 1 && k >= 128))        // (the next exchange is over more than 128 neighbours, or was)
                __syncthreads();
            else
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    __syncthreads();
}

// ---------------------------------------------------------------- a whole row by one workgroup

// Bins cleared, filled by `fill`, their masses turned into weights by `weigh`, then into running sums. Returns the totals.
template <class F, class G>
__device__ inline void fill_bins(Shared& s, uint32_t& c_all, uint64_t& m_all, F fill, G weigh) {
    const int tid = threadIdx.x;
    __syncthreads();
    s.count[tid] = s.count[tid + kThreads] = 0;
    s.mass[tid] = s.mass[tid + kThreads] = 0;
    __syncthreads();
    fill();
    __syncthreads();
    const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
    const uint64_t m0 = weigh(s.mass[2 * tid], 2 * tid), m1 = weigh(s.mass[2 * tid + 1], 2 * tid + 1);
    uint32_t c = c0 + c1;
    uint64_t m = m0 + m1;
    block_excl<16>(c, m, s.wave_count, s.wave_mass);
    s.count[2 * tid] = c + c0;
    s.count[2 * tid + 1] = c + c0 + c1;
    s.mass[2 * tid] = m + m0;
    s.mass[2 * tid + 1] = m + m0 + m1;
    __syncthreads();
    c_all = s.count[kBins - 1];
    m_all = s.mass[kBins - 1];
}

// The first bin in which `b` is passed (the last one with a token where none is), `c` and `m` being what comes before the
// bins (then before that bin), and its count.
__device__ inline int find_bin(Shared& s, const Bound& b, uint32_t& c, uint64_t& m, uint32_t& in) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid == 0) {
        s.found = kBins;
        s.at[0] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = 2 * tid + i;
        const uint32_t cp = j > 0 ? s.count[j - 1] : 0;
        if (s.count[j] > cp) {
            if (b.passed(c + s.count[j], m + s.mass[j])) atomicMin(&s.found, j);
            if (s.count[j] == s.count[kBins - 1]) s.at[0] = j;
        }
    }
    __syncthreads();
    const int j = s.found < kBins ? s.found : s.at[0];
    const uint32_t cp = j > 0 ? s.count[j - 1] : 0;
    const uint64_t mp = j > 0 ? s.mass[j - 1] : 0;
    in = s.count[j] - cp;
    c += cp;
    m += mp;
    return j;
}

// What a bound finds: the token that passes it, and the sum up to it.
struct Found {
    uint64_t token, mass;
};

// In the sorted list of n tokens, with c and m before it (the last one with a weight where none passes it).
__device__ inline Found find_token(Shared& s, const Row& row, const Bound& b, int n, uint32_t c, uint64_t m) {
    constexpr int E = kList / kThreads;
    const int tid = threadIdx.x;
    uint64_t w[E], sum = 0;
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int j = tid * E + i;
        w[i] = j < n ? row.weight(logit_of(s.list[j])) : 0;
        k += w[i] > 0;
        sum += w[i];
    }
    block_excl<16>(k, sum, s.wave_count, s.wave_mass);
    uint32_t k_all = 0;
    for (int i = 0; i < 16; ++i) k_all += s.wave_count[i];
    k += c;
    sum += m;
    if (tid == 0) {
        s.found = kList;
        s.at[0] = 0;
    }
    __syncthreads();
    int first = kList;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (w[i] == 0) continue;
        ++k;
        w[i] = sum += w[i];
        if (first == kList && b.passed(k, sum)) first = tid * E + i;
        if (k == c + k_all) s.at[0] = tid * E + i;
    }
    first_of(first, kList, &s.found);
    __syncthreads();
    const int found = s.found < kList ? s.found : s.at[0];
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (found == tid * E + i) s.found_mass = w[i];
    __syncthreads();
    const Found f{s.list[found], s.found_mass};
    __syncthreads();
    return f;
}

// A row's bounds one after the other: the bin that each is in, and the token among those of the bin, which are cut further
// by value and then by index while they are more than the list holds.
template <class R>
__device__ inline void sample_row(Shared& s, const SampleArgs& a, const R& r, const Row& row, int b) {
    const int tid = threadIdx.x;
    uint32_t c_all = 0;
    uint64_t m_all = 0, S = 0;
    bool filled = false;
#pragma unroll 1
    for (int step = 0;; ++step) {                      // top_k, top_p, the draw
        if (!filled)
            fill_bins(s, c_all, m_all, [&] {
                r.each([&](float l, int) {
                    if (order_of(l) <= kMinusInf) return;
                    const double y = row.any_place(l);
                    if (!(y <= row.limit)) return;
                    const int i = whole_of(y);
                    atomicAdd(&s.count[i], 1u);
                    atomicAdd((unsigned long long*)&s.mass[i], (unsigned long long)part_of(rest_of(y)));
                });
            }, [&](uint64_t parts, int i) { return parts == 0 ? 0 : in_bin(parts, i, row.octave[i & (kPerOctave - 1)]); });
        filled = true;
        if (step == 0) S = m_all;
        if (step == 0 ? row.k <= 0 || (uint32_t)row.k >= c_all : step == 1 && !(row.p < 1.f)) continue;
        const Bound bound = step == 0   ? Bound{Bound::kRank, (uint32_t)row.k, 0.0}
                            : step == 1 ? Bound{Bound::kReaches, 0, (double)row.p * (double)S}
                                        : Bound{Bound::kPasses, 0, row.u() * (double)S};
        uint32_t c = 0, in;
        uint64_t m = 0, lo = 0, hi = ~0ull;
        const int bin = find_bin(s, bound, c, m, in);
        auto each = [&](auto f) {
            r.each([&](float l, int j) {
                if (order_of(l) <= kMinusInf || row.bin(l) != bin) return;
                const uint64_t x = token_of(l, j);
                if (x >= lo && x <= hi) f(x, l);
            });
        };
        if (in > kList) {                              // uniform
            filled = false;
            if (tid == 0) {
                s.lo = ~0ull;
                s.hi = 0;
            }
            __syncthreads();
            uint64_t x0 = ~0ull, x1 = 0;
            each([&](uint64_t x, float) {
                x0 = min(x0, x);
                x1 = max(x1, x);
            });
            atomicMin((unsigned long long*)&s.lo, (unsigned long long)x0);
            atomicMax((unsigned long long*)&s.hi, (unsigned long long)x1);
            __syncthreads();
            lo = s.lo;
            hi = s.hi;
        }
#pragma unroll 1
        while (in > kList) {                           // each turn narrows hi - lo 1,024 times at least
            const uint64_t span = hi - lo;
            const int shift = span < (uint64_t)kBins ? 0 : 53 - __builtin_clzll(span);
            uint32_t c_in;
            uint64_t m_in;
            fill_bins(s, c_in, m_in, [&] {
                each([&](uint64_t x, float l) {
                    const int i = (int)((x - lo) >> shift);
                    atomicAdd(&s.count[i], 1u);
                    atomicAdd((unsigned long long*)&s.mass[i], (unsigned long long)row.weight(l));
                });
            }, [](uint64_t mass, int) { return mass; });
            const int i = find_bin(s, bound, c, m, in);
            lo += (uint64_t)i << shift;
            hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
        }
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        each([&](uint64_t x, float) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < (uint32_t)kList) s.list[at] = x;
        });
        __syncthreads();
        const int n = min((int)s.n, kList);
        sort_list(s, n);
        const Found f = find_token(s, row, bound, n, c, m);
        if (step == 2) {
            take(a, b, row, f.token, S);
            return;
        }
        S = f.mass;
    }
}

// One launch, a workgroup a row: short rows.
template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_row_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int b = blockIdx.x;
    const MemoryRow<TYPE, kThreads> r(a, b, 0, a.V);
    const Settings set(a, b);
    if (threadIdx.x < kPerOctave) s.octave[threadIdx.x] = kOctave[threadIdx.x];
    const uint64_t best = block_largest<16>(r.largest(), s.wave_mass);
    const Row row(set, best, s.octave);
    __syncthreads();
    if (row.greedy)                                    // uniform
        take_largest(a, b, row, best);
    else
        sample_row(s, a, r, row, b);
}

// ---------------------------------------------------------------- a row in pieces
//
// Four launches, pieces of a row a workgroup for the first three: the largest logit of a piece; the row's bins; the
// tokens of the bins in question; and what they say.
constexpr int kPiece = 256;            // threads of a piece's workgroup
constexpr int kLocal = 1024;           // tokens that a piece collects at most

template <int TYPE>
__global__ void __launch_bounds__(kPiece) sample_largest_kernel(SampleArgs a) {
    __shared__ uint64_t s[kPiece / 64];
    const int b = (int)(blockIdx.x / (unsigned)a.pieces), piece = (int)(blockIdx.x % (unsigned)a.pieces), from = piece * a.per;
    const MemoryRow<TYPE, kPiece> r(a, b, from, min(from + a.per, a.V));
    for (int i = piece * kPiece + (int)threadIdx.x; i < kReach; i += a.pieces * kPiece) {
        a.mass[(int64_t)b * kReach + i] = 0;
        a.count[(int64_t)b * kReach + i] = 0;
    }
    if (piece == 0 && threadIdx.x == 0) a.n[b] = 0;
    const uint64_t best = block_largest<kPiece / 64>(r.largest(), s);
    if (threadIdx.x == 0) a.best[(int64_t)b * a.pieces + piece] = best;
}

// The largest of the row's pieces.
template <int WAVES>
__device__ inline uint64_t row_largest(const SampleArgs& a, int b, uint64_t* s) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.pieces; i += 64 * WAVES) best = max(best, a.best[(int64_t)b * a.pieces + i]);
    return block_largest<WAVES>(best, s);
}

template <int TYPE>
__global__ void __launch_bounds__(kPiece) sample_bins_kernel(SampleArgs a) {
    __shared__ uint64_t mass[kReach];
    __shared__ uint32_t count[kReach];
    __shared__ uint64_t s[kPiece / 64];
    const int b = (int)(blockIdx.x / (unsigned)a.pieces), piece = (int)(blockIdx.x % (unsigned)a.pieces), from = piece * a.per;
    for (int i = threadIdx.x; i < kReach; i += kPiece) {
        mass[i] = 0;
        count[i] = 0;
    }
    const Settings set(a, b);
    const Row row(set, row_largest<kPiece / 64>(a, b, s), nullptr);
    __syncthreads();
    if (row.greedy || row.odd) return;                 // uniform
    const MemoryRow<TYPE, kPiece> r(a, b, from, min(from + a.per, a.V));
    // (a piece's logits side by side, without a branch before the last step)
    constexpr int N = Logits<TYPE>::N;
    if (row.few) {                                     // uniform
        r.pieces([&](const uint32_t (&x)[4], int) {
            double y[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = row.place(Logits<TYPE>::at(x, e));
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (y[e] <= row.limit) atomicAdd(&count[whole_of(y[e])], 1u);
        });
    } else {
        const bool counts = row.k > 0;
        r.pieces([&](const uint32_t (&x)[4], int) {
            double y[N];
            uint64_t part[N];
#pragma unroll
            for (int e = 0; e < N; ++e) y[e] = row.place(Logits<TYPE>::at(x, e));
#pragma unroll
            for (int e = 0; e < N; ++e) part[e] = part_of(rest_of(y[e]));
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (y[e] <= row.limit) atomicAdd((unsigned long long*)&mass[whole_of(y[e])], (unsigned long long)part[e]);
            if (counts)                                // uniform
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (y[e] <= row.limit) atomicAdd(&count[whole_of(y[e])], 1u);
        });
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kReach; i += kPiece) {
        if (mass[i] != 0) atomicAdd((unsigned long long*)&a.mass[(int64_t)b * kReach + i], (unsigned long long)mass[i]);
        if (count[i] != 0) atomicAdd(&a.count[(int64_t)b * kReach + i], count[i]);
    }
}

// Which bins the row's bounds are in: ranges that ascend and lie apart (empty ones: last below first), and the count and
// sum that a token in one has before it less those of the collected tokens before it.
struct Range {
    int first = 1, last = 0;
    uint32_t count = 0;
    uint64_t mass = 0;
};
struct Ranges {
    Range r[3];
    bool cut;                          // top_k cuts
    uint64_t all;                      // the sum of all weights
    uint64_t best;                     // the row's largest logit
    __device__ bool hold(int bin) const {
        bool in = false;
#pragma unroll
        for (int i = 0; i < 3; ++i) in |= bin >= r[i].first && bin <= r[i].last;
        return in;
    }
    __device__ void before(int bin, uint32_t& c, uint64_t& m) const {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (bin >= r[i].first && bin <= r[i].last) {
                c += r[i].count;
                m += r[i].mass;
            }
    }
};

// Logits among which are all that the ranges hold (compared in fp32, with 2^-20 of the row's reach and of the largest logit to
// spare), and few others.
struct Near {
    float low[3], high[3], one_low, one_high;
    int ranges = 0;
    __device__ __attribute__((always_inline)) Near(const Row& row, const Ranges& ranges) {
        const double wide = 1.0 / row.per_bin, spare = 0x1p-20 * (fabs(row.top) + kReach * wide);   // (infinite at t = infinity)
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const Range& q = ranges.r[i];
            const bool none = q.last < q.first;
            low[i] = none ? INFINITY : (float)(row.top - (q.last + 1) * wide - spare);
            high[i] = none ? -INFINITY : q.first == 0 ? row.top32 : (float)(row.top - q.first * wide + spare);
            this->ranges += !none;
        }
        one_low = fminf(low[0], fminf(low[1], low[2]));
        one_high = fmaxf(high[0], fmaxf(high[1], high[2]));
    }
    __device__ bool single() const { return ranges == 1; }
    __device__ bool hold(float l) const {
        return (l >= low[0] && l <= high[0]) | (l >= low[1] && l <= high[1]) | (l >= low[2] && l <= high[2]);
    }
};

// A row's bins as loaded, E neighbouring ones a thread of kBins / E.
template <int E>
struct Bins {
    uint64_t m[E];
    uint32_t c[E];
    __device__ void read(const SampleArgs& a, const Settings& set, int b) {
        const bool masses = !set.few(), counts = set.k > 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = (int)threadIdx.x * E + i;
            m[i] = j < kReach && masses ? a.mass[(int64_t)b * kReach + j] : 0;
            c[i] = j < kReach && counts ? a.count[(int64_t)b * kReach + j] : 0;
        }
    }
};

// The row's bins as running sums in `mass` and `count` [kBins], and the ranges of its bounds; sc, sm, at: scratch. All
// threads get the same.
template <int THREADS>
__device__ inline Ranges find_ranges(const Row& row, const Bins<kBins / THREADS>& bins, uint64_t* mass, uint32_t* count, int* at,
                                     uint32_t* sc, uint64_t* sm) {
    constexpr int E = kBins / THREADS;
    const int j0 = (int)threadIdx.x * E;
    const bool counts = row.k > 0;
    uint64_t m[E], ms = 0;
    uint32_t c[E], cs = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        c[i] = bins.c[i];
        m[i] = bins.m[i] == 0 ? 0 : in_bin(bins.m[i], j0 + i, row.octave[(j0 + i) & (kPerOctave - 1)]);
        ms += m[i];
        cs += c[i];
    }
    block_excl<THREADS / 64>(cs, ms, sc, sm);
    const uint64_t m0 = ms;
    const uint32_t c0 = cs;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        m[i] = mass[j0 + i] = ms += m[i];
        c[i] = count[j0 + i] = cs += c[i];
    }
    // the first bins that satisfy two bounds (the last bin where none does)
    auto find = [&](auto passed0, auto passed1, int& x, int& y) {
        __syncthreads();
        if (threadIdx.x == 0) at[0] = at[1] = kReach - 1;
        __syncthreads();
        uint32_t cb = c0;
        uint64_t mb = m0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            if (passed0(c[i], m[i]) && (j0 + i == 0 || !passed0(cb, mb))) at[0] = j0 + i;
            if (passed1(c[i], m[i]) && (j0 + i == 0 || !passed1(cb, mb))) at[1] = j0 + i;
            cb = c[i];
            mb = m[i];
        }
        __syncthreads();
        x = at[0];
        y = at[1];
    };
    Ranges r;
    __syncthreads();
    r.all = mass[kBins - 1];
    const uint32_t c_all = count[kBins - 1];
    r.cut = counts && (row.few || (uint32_t)row.k < c_all);
    int x, y;
    double s0 = (double)r.all, s1 = s0;                // the sums that are known to a bin, from and to
    if (r.cut) {                                       // uniform
        const uint32_t k = min((uint32_t)row.k, c_all);
        auto reach = [&](uint32_t n, uint64_t) { return n >= k; };
        find(reach, reach, x, y);
        r.r[2].first = row.few ? 0 : x;
        r.r[2].last = x;
        s0 = x > 0 ? (double)mass[x - 1] : 0.0;
        s1 = (double)mass[x];
    }
    if (row.few) return r;
    if (row.p < 1.f) {                                 // uniform
        const double p0 = (double)row.p * s0, p1 = (double)row.p * s1;
        find([&](uint32_t, uint64_t f) { return (double)f >= p0; }, [&](uint32_t, uint64_t f) { return (double)f >= p1; }, x, y);
        r.r[1].first = x;
        r.r[1].last = y;
        s0 = x > 0 ? (double)mass[x - 1] : 0.0;
        s1 = (double)mass[y];
    }
    const double u0 = row.u() * s0, u1 = row.u() * s1;
    find([&](uint32_t, uint64_t f) { return (double)f > u0; }, [&](uint32_t, uint64_t f) { return (double)f > u1; }, x, y);
    r.r[0].first = x;
    r.r[0].last = y;
    // (each bound lies at or before the next range's)
    r.r[1].first = max(r.r[1].first, y + 1);
    r.r[2].first = max(r.r[2].first, max(y, r.r[1].last) + 1);
    uint64_t took_m = 0;
    uint32_t took_c = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (r.r[i].last < r.r[i].first) continue;
        const int f = r.r[i].first;
        const uint64_t before_m = f > 0 ? mass[f - 1] : 0;
        const uint32_t before_c = f > 0 ? count[f - 1] : 0;
        r.r[i].mass = before_m - took_m;
        r.r[i].count = before_c - took_c;
        took_m += mass[r.r[i].last] - before_m;
        took_c += count[r.r[i].last] - before_c;
    }
    return r;
}

template <int TYPE>
__global__ void __launch_bounds__(kPiece) sample_collect_kernel(SampleArgs a) {
    __shared__ uint64_t mass[kBins], list[kLocal];
    __shared__ uint32_t count[kBins];
    __shared__ double octave[kPerOctave];
    __shared__ uint64_t s[kPiece / 64], sm[kPiece / 64];
    __shared__ uint32_t sc[kPiece / 64], n, base;
    __shared__ int at[2];
    const int b = (int)(blockIdx.x / (unsigned)a.pieces), piece = (int)(blockIdx.x % (unsigned)a.pieces), from = piece * a.per;
    const Settings set(a, b);
    if (threadIdx.x < kPerOctave) octave[threadIdx.x] = kOctave[threadIdx.x];
    Bins<kBins / kPiece> bins;
    bins.read(a, set, b);
    const uint64_t best = row_largest<kPiece / 64>(a, b, s);
    const Row row(set, best, octave);
    if (threadIdx.x == 0) n = 0;
    if (row.odd && piece == 0 && threadIdx.x == 0) a.n[b] = kList + 1;
    if (row.greedy || row.odd) {                       // uniform
        if (piece == 0 && threadIdx.x == 0) a.ranges[b].best = best;
        return;
    }
    Ranges ranges = find_ranges<kPiece>(row, bins, mass, count, at, sc, sm);
    ranges.best = best;
    if (piece == 0 && threadIdx.x == 0) a.ranges[b] = ranges;
    const MemoryRow<TYPE, kPiece> r(a, b, from, min(from + a.per, a.V));
    const Near near(row, ranges);
    constexpr int N = Logits<TYPE>::N;
    auto collect = [&](auto hold) {
        r.pieces([&](const uint32_t (&x)[4], int j) {
            uint32_t found = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) found |= (uint32_t)hold(Logits<TYPE>::at(x, e)) << e;
            while (found != 0) {
                const int at = j + __builtin_ctz(found);
                found &= found - 1;
                const float l = r.one(at);
                const double y = row.place(l);
                if (!(y <= row.limit) || !ranges.hold(whole_of(y))) continue;
                const uint32_t i = atomicAdd(&n, 1u);
                if (i < (uint32_t)kLocal) list[i] = token_of(l, at);
            }
        });
    };
    // rows with one range, which most settings have, look at no more
    if (near.single())                                 // uniform
        collect([&](float l) { return l >= near.one_low && l <= near.one_high; });
    else
        collect([&](float l) { return near.hold(l); });
    __syncthreads();
    if (n == 0) return;                                // uniform
    if (threadIdx.x == 0) base = atomicAdd(&a.n[b], n <= (uint32_t)kLocal ? n : (uint32_t)kList + 1);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < min(n, (uint32_t)kLocal); i += kPiece)
        if (base + i < (uint32_t)kList) a.list[(int64_t)b * kList + base + i] = list[i];
}

// The n collected tokens of s.list sorted, and the row's bounds found among them one after the other.
__device__ inline void take_bounds(Shared& s, const SampleArgs& a, const Row& row, const Ranges& ranges, int n, int b) {
    constexpr int E = kList / kThreads;
    const int tid = threadIdx.x;
    sort_list(s, n);
    // each token's running count and sum over the row
    uint64_t w[E], F[E], m = 0;
    uint32_t K[E], c = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int j = tid * E + i;
        w[i] = 0;
        F[i] = 0;
        K[i] = 0;
        if (j < n) {
            const float l = logit_of(s.list[j]);
            w[i] = row.weight(l);
            ranges.before(row.bin(l), K[i], F[i]);
            ++c;
            m += w[i];
        }
    }
    block_excl<16>(c, m, s.wave_count, s.wave_mass);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        F[i] += m += w[i];
        K[i] += ++c;
    }
    // the first token that satisfies a bound, or the last one
    auto find = [&](const Bound& bound) {
        if (tid == 0) s.found = n - 1;
        __syncthreads();
        int first = kList;
#pragma unroll
        for (int i = E - 1; i >= 0; --i)
            if (tid * E + i < n && bound.passed(K[i], F[i])) first = tid * E + i;
        first_of(first, kList, &s.found);
        __syncthreads();
        const int found = s.found;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (found == tid * E + i) s.found_mass = F[i];
        __syncthreads();
        return s.found_mass;
    };
    uint64_t S = ranges.all;
    if (ranges.cut) S = find(Bound{Bound::kRank, (uint32_t)row.k, 0.0});
    if (row.p < 1.f) S = find(Bound{Bound::kReaches, 0, (double)row.p * (double)S});
    find(Bound{Bound::kPasses, 0, row.u() * (double)S});
    take(a, b, row, s.list[s.found], S);
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_take_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int b = blockIdx.x, tid = threadIdx.x;
    const Settings set(a, b);
    const uint32_t n_all = a.n[b];
    const Ranges ranges = a.ranges[b];
    uint64_t early[2];                                 // most rows' tokens, on their way with these
#pragma unroll
    for (int i = 0; i < 2; ++i) early[i] = a.list[(int64_t)b * kList + tid + i * kThreads];
    if (tid < kPerOctave) s.octave[tid] = kOctave[tid];
    const Row row(set, ranges.best, s.octave);
    __syncthreads();
    if (row.greedy) return take_largest(a, b, row, ranges.best);   // uniform
    if (n_all > (uint32_t)kList) {                     // uniform: an infinite largest logit, or more near ones than the list holds
        sample_row(s, a, MemoryRow<TYPE, kThreads>(a, b, 0, a.V), row, b);
        return;
    }
    const int n = (int)n_all;
    if (n == 0) return take_largest(a, b, row, ranges.best);   // uniform (the largest is always near itself)
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (tid + i * kThreads < n) s.list[tid + i * kThreads] = early[i];
    for (int i = tid + 2 * kThreads; i < n; i += kThreads) s.list[i] = a.list[(int64_t)b * kList + i];
    take_bounds(s, a, row, ranges, n, b);
}

hipError_t fetch_errors_sample(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

}  // namespace exkv

using namespace exkv;

// Rows of up to this many logits go by one workgroup each.
constexpr int kShort = 8192;

struct SamplePlan {
    int pieces, per;
    int64_t best, mass, list, ranges, count, n, bytes;   // offsets in the workspace
};
static SamplePlan plan_sample(int64_t B, int64_t V) {
    SamplePlan p{};
    if (V <= kShort || B == 0) return p;
    // pieces of whole 2,048 logits, about 1,024 workgroups in all (256 x 152064, 512 / 1,024 / 2,048: 89.3 / 83.0 / 90.2 us; 128
    // mixed rows, by their inputs, 50 to 60 each), of 4,096 logits at least (61 x 50257, 2,048 / 4,096: 37.4 / 36.0 us), but not
    // so few that CUs stay idle (1 x 128256: 21.4 / 22.2)
    const int64_t least = B * (V / 4096) < 256 ? 2048 : 4096;
    int64_t pieces = (1024 + B - 1) / B;
    if (pieces > V / least) pieces = V / least;
    p.per = (int)(((V + pieces - 1) / pieces + 2047) / 2048 * 2048);
    p.pieces = (int)((V + p.per - 1) / p.per);
    p.mass = B * p.pieces * 8;
    p.list = p.mass + B * kReach * 8;
    p.ranges = p.list + B * kList * 8;
    p.count = p.ranges + B * (int64_t)sizeof(Ranges);
    p.n = p.count + B * kReach * 4;
    p.bytes = p.n + B * 4;
    return p;
}

template <int TYPE>
static void launch_sample(const SampleArgs& a, hipStream_t stream) {
    if (a.pieces == 0) {
        hipLaunchKernelGGL((sample_row_kernel<TYPE>), dim3((unsigned)a.B), dim3(kThreads), 0, stream, a);
        return;
    }
    const dim3 grid((unsigned)((int64_t)a.B * a.pieces)), block(kPiece);
    hipLaunchKernelGGL((sample_largest_kernel<TYPE>), grid, block, 0, stream, a);
    hipLaunchKernelGGL((sample_bins_kernel<TYPE>), grid, block, 0, stream, a);
    hipLaunchKernelGGL((sample_collect_kernel<TYPE>), grid, block, 0, stream, a);
    hipLaunchKernelGGL((sample_take_kernel<TYPE>), dim3((unsigned)a.B), dim3(kThreads), 0, stream, a);
}

extern "C" int64_t exkv_sample_workspace(int32_t B, int32_t V) { return B <= 0 || V <= 0 ? 0 : plan_sample(B, V).bytes; }

extern "C" int exkv_sample(const void* logits, int64_t stride, int32_t type, int32_t B, int32_t V, const float* u, const float* temperature,
                           const int32_t* top_k, const float* top_p, const float* min_p, float temperature0, int32_t top_k0,
                           float top_p0, float min_p0, int64_t* token, float* logprob, void* ws, int64_t ws_bytes, hipStream_t stream) {
    EXKV_REQUIRE(type >= 0 && type <= 2, "sample: logits of type %d", type);
    EXKV_REQUIRE(B >= 0 && V > 0 && V <= (1 << 19) && stride >= 0, "sample: bad shape B=%d V=%d (up to %d)", B, V, 1 << 19);
    if (B == 0) return EXKV_OK;
    const SamplePlan p = plan_sample(B, V);
    EXKV_REQUIRE((int64_t)B * kThreads <= (int64_t)UINT32_MAX && (int64_t)B * p.pieces * kPiece <= (int64_t)UINT32_MAX,
                 "sample: too many rows (%d)", B);
    EXKV_REQUIRE(logits && u && token, "sample: null pointer");
    EXKV_REQUIRE((uintptr_t)logits % (type == kFp32 ? 4 : 2) == 0, "sample: logits must be aligned to their size");
    EXKV_REQUIRE(p.bytes == 0 || (ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= p.bytes), "sample: workspace of %lld bytes, %lld needed",
                 (long long)ws_bytes, (long long)p.bytes);
    uint8_t* w = (uint8_t*)ws;
    const SampleArgs a{logits, stride, B, V, u, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0, token, logprob,
                       p.pieces, p.per, (uint64_t*)w, (uint64_t*)(w + p.mass), (uint64_t*)(w + p.list), (uint32_t*)(w + p.count),
                       (uint32_t*)(w + p.n), (Ranges*)(w + p.ranges)};
    if (type == kBf16)
        launch_sample<kBf16>(a, stream);
    else if (type == kFp16)
        launch_sample<kFp16>(a, stream);
    else
        launch_sample<kFp32>(a, stream);
    return hip_status(hipGetLastError(), "sample");
}
