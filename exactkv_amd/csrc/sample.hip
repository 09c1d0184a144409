// One token a row from logits, with temperature, top-k, top-p and min-p and given uniform numbers, for
// gfx950 (no counterpart in the reference, whose engine decodes greedily, exactkv/engine.py:93-95).
//
// Of a row's logits l, with M the largest and t the temperature, the weights are w = exp((l - M) / t). Ordered by
// value, equal ones by index, these stay, each time a beginning of the row: those with w >= min_p; of them the first
// top_k; of these the ones before whose weights add up to less than top_p of all. Of what stays, S its sum, the token
// is the first one with which the running sum passes u S.
//
// Every cut is thus a place in one order, the first where a running count or sum passes a bound, and is found without
// a sort of the row: weights are counted and added up in 2,048 bins of (M - l) / t, 1/64 wide; the bin in which
// the bound is passed is known from the bins' sums; its tokens alone are collected, sorted and added up one by one.
// With top_k up to 2,048 all tokens down to the k-th's bin are collected at once and no other weight is computed.
//
// Weights are fp64 exponentials rounded to multiples of 2^-43 and held as whole numbers, so sums do not depend on
// the order in which they are taken and a cut falls where the formula in 64 bits has it; weights below 2^-44
// (all of a vocabulary of 2^19 add up to less than 2^-25 of the sum) are 0.
#include "errors.hpp"
#include "common.hpp"
#include "../../include/exactkv.h"

namespace exkv {

constexpr int kThreads = 1024, kBins = 2048, kList = 4096;
constexpr float kPerNat = 64.f;        // bins of width 1 in (M - l) / t
constexpr double kOne = 8796093022208.0;   // 2^43: a weight of 1

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
};

// A logit's place in the order of all; -0 as 0. NaN: 0. kMinusInf: the least that can be drawn is above it.
constexpr uint32_t kMinusInf = ~0xFF800000u;
__device__ inline uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0u : (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}
__device__ inline float of_order(uint32_t k) { return __uint_as_float((k & 0x80000000u) != 0 ? k & 0x7FFFFFFFu : ~k); }

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

// A row's settings and its weights.
struct Row {
    float top, inv_bins;               // M; 64 / t
    double inv_t, min_p;
    __device__ int bin(float l) const {
        const float z = (top - l) * inv_bins;
        return l == top ? 0 : z < (float)(kBins - 1) ? (int)z : kBins - 1;   // (ascends as l falls; NaN: the last)
    }
    // of a logit above -inf
    __device__ uint64_t weight(float l) const {
        if (l == top) return (uint64_t)kOne;
        const double w = exp(((double)l - (double)top) * inv_t);
        return w >= min_p ? (uint64_t)__double2ll_rn(w * kOne) : 0;
    }
};

__device__ inline uint64_t wave_incl_sum(uint64_t x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)x, d);
        if (lane >= d) x += y;
    }
    return x;
}

// Shared memory of a workgroup.
struct Shared {
    uint64_t mass[kBins];              // then inclusive sums
    uint64_t list[kList];              // tokens: ~order << 32 | index, ascending once sorted
    uint32_t count[kBins];
    uint64_t wave_mass[16];
    uint32_t wave_count[16];
    uint64_t lo, hi;                   // composite values
    uint32_t n;
    int found;
    uint32_t found_count;
    uint64_t found_mass;
};

// Exclusive sums over the workgroup's threads of (c, m); totals in the last two.
__device__ inline void block_excl(Shared& s, uint32_t& c, uint64_t& m, uint32_t& c_all, uint64_t& m_all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t ci = (uint32_t)wave_incl_scan((int)c);
    const uint64_t mi = wave_incl_sum(m);
    __syncthreads();
    if (lane == 63) {
        s.wave_count[w] = ci;
        s.wave_mass[w] = mi;
    }
    __syncthreads();
    uint32_t cb = 0;
    uint64_t mb = 0;
    c_all = 0;
    m_all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (i == w) {
            cb = c_all;
            mb = m_all;
        }
        c_all += s.wave_count[i];
        m_all += s.wave_mass[i];
    }
    c = cb + ci - c;
    m = mb + mi - m;
}

// A bound on the running count or sum, which the first element that satisfies it passes.
struct Bound {
    enum { kRank, kReach, kPass } kind;
    uint32_t rank;
    double x;
    __device__ bool passed(uint32_t c, uint64_t m) const {
        return kind == kRank ? c >= rank : kind == kReach ? (double)m >= x : (double)m > x;
    }
};

// The passes over a row: f(logit, index) of every one.
template <int TYPE>
struct MemoryRow {
    const uint8_t* p;
    int V;
    template <class F>
    __device__ void each(F f) const {
        constexpr int N = Logits<TYPE>::N, SIZE = Logits<TYPE>::SIZE;
        for (int j = (int)threadIdx.x * N; j < V; j += kThreads * N) {
            if (j + N <= V) {
                uint32_t x[4];
                __builtin_memcpy(x, p + (int64_t)j * SIZE, 16);
#pragma unroll
                for (int i = 0; i < N; ++i) f(Logits<TYPE>::at(x, i), j + i);
            } else {
                for (int i = j; i < V; ++i) f(Logits<TYPE>::one(p + (int64_t)i * SIZE), i);
            }
        }
    }
};

// Bins cleared, filled by `fill`, turned into running sums (bins ascending). Returns the totals.
template <class F>
__device__ inline void fill_bins(Shared& s, uint32_t& c_all, uint64_t& m_all, F fill) {
    const int tid = threadIdx.x;
    __syncthreads();
    s.count[tid] = s.count[tid + kThreads] = 0;
    s.mass[tid] = s.mass[tid + kThreads] = 0;
    __syncthreads();
    fill();
    __syncthreads();
    const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
    const uint64_t m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
    uint32_t c = c0 + c1;
    uint64_t m = m0 + m1;
    block_excl(s, c, m, c_all, m_all);
    s.count[2 * tid] = c + c0;
    s.count[2 * tid + 1] = c + c0 + c1;
    s.mass[2 * tid] = m + m0;
    s.mass[2 * tid + 1] = m + m0 + m1;
    __syncthreads();
}

// The first bin in which `b` is passed, `c` and `m` being what comes before the bins (then before that bin), and
// its count.
__device__ inline int find_bin(Shared& s, const Bound& b, uint32_t& c, uint64_t& m, uint32_t& in) {
    const int tid = threadIdx.x;
    if (tid == 0) s.found = kBins;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = 2 * tid + i;
        const uint32_t cp = j > 0 ? s.count[j - 1] : 0;
        const uint64_t mp = j > 0 ? s.mass[j - 1] : 0;
        if (s.count[j] > cp && b.passed(c + s.count[j], m + s.mass[j]) && (cp == 0 || !b.passed(c + cp, m + mp))) s.found = j;
    }
    __syncthreads();
    const int j = min(s.found, kBins - 1);
    const uint32_t cp = j > 0 ? s.count[j - 1] : 0;
    const uint64_t mp = j > 0 ? s.mass[j - 1] : 0;
    in = s.count[j] - cp;
    c += cp;
    m += mp;
    return j;
}

// The list's n tokens in order.
__device__ inline void sort_list(Shared& s, int n) {
    const int tid = threadIdx.x;
    int size = 64;
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
            __syncthreads();
        }
}

// What a bound finds: the token that passes it, and the count and sum up to it.
struct Found {
    uint64_t token;                    // ~order << 32 | index
    uint32_t count;
    uint64_t mass;
};

// In the sorted list of n tokens, with c and m before it; weights of tokens past `limit` in all count as none.
__device__ inline Found find_token(Shared& s, const Row& row, const Bound& b, int n, uint32_t c, uint64_t m) {
    constexpr int E = kList / kThreads;
    const int tid = threadIdx.x;
    uint64_t w[E], sum = 0;
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int j = tid * E + i;
        w[i] = j < n ? row.weight(of_order(~(uint32_t)(s.list[j] >> 32))) : 0;
        k += w[i] > 0;
        sum += w[i];
    }
    uint32_t c_all;
    uint64_t m_all;
    block_excl(s, k, sum, c_all, m_all);
    k += c;
    sum += m;
    if (tid == 0) s.found = -1;
    __syncthreads();
    bool before = k > 0 && b.passed(k, sum);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        if (w[i] == 0) continue;
        ++k;
        sum += w[i];
        const bool now = b.passed(k, sum);
        // (the last one where none passes it)
        if ((now && !before) || (!now && k == c + c_all)) {
            s.found = tid * E + i;
            s.found_count = k;
            s.found_mass = sum;
        }
        before = now;
    }
    __syncthreads();
    const Found f{s.list[max(s.found, 0)], s.found_count, s.found_mass};
    __syncthreads();
    return f;
}

// The token that passes `b` among those of z-bin `bin`, c and m before it, `in` of them.
template <class R>
__device__ inline Found find_in_bin(Shared& s, const R& r, const Row& row, const Bound& b, int bin, uint32_t c, uint64_t m,
                                    uint32_t in) {
    const int tid = threadIdx.x;
    uint64_t lo = 0, hi = ~0ull;
    auto each = [&](auto f) {
        r.each([&](float l, int j) {
            const uint32_t o = order_of(l);
            if (o <= kMinusInf || row.bin(l) != bin) return;
            const uint64_t x = (uint64_t)~o << 32 | (uint32_t)j;
            if (x >= lo && x <= hi) f(x, l);
        });
    };
    if (in > kList) {                                  // uniform: cut further, by value and then by index
        if (tid == 0) {
            s.lo = ~0ull;
            s.hi = 0;
        }
        __syncthreads();
        uint64_t a = ~0ull, z = 0;
        each([&](uint64_t x, float l) {
            if (row.weight(l) == 0) return;
            a = min(a, x);
            z = max(z, x);
        });
        atomicMin((unsigned long long*)&s.lo, (unsigned long long)a);
        atomicMax((unsigned long long*)&s.hi, (unsigned long long)z);
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        while (in > kList) {                           // each turn narrows hi - lo 1,024 times at least
            const uint64_t span = hi - lo;
            const int shift = span < (uint64_t)kBins ? 0 : 53 - __builtin_clzll(span);
            uint32_t c_all;
            uint64_t m_all;
            fill_bins(s, c_all, m_all, [&] {
                each([&](uint64_t x, float l) {
                    const uint64_t w = row.weight(l);
                    if (w == 0) return;
                    const int i = (int)((x - lo) >> shift);
                    atomicAdd(&s.count[i], 1u);
                    atomicAdd((unsigned long long*)&s.mass[i], (unsigned long long)w);
                });
            });
            const int i = find_bin(s, b, c, m, in);
            lo += (uint64_t)i << shift;
            hi = min(hi, lo + (((uint64_t)1 << shift) - 1));
        }
    }
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    each([&](uint64_t x, float l) {
        if (row.weight(l) == 0) return;                // (below min_p: not counted either)
        const uint32_t at = atomicAdd(&s.n, 1u);
        if (at < (uint32_t)kList) s.list[at] = x;
    });
    __syncthreads();
    const int n = min((int)s.n, kList);
    sort_list(s, n);
    return find_token(s, row, b, n, c, m);
}

template <class R>
__device__ inline void sample_row(Shared& s, const SampleArgs& a, const R& r, int b) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    // the largest logit, the first of equal ones
    uint64_t best = 0;
    r.each([&](float l, int j) { best = max(best, (uint64_t)order_of(l) << 32 | ~(uint32_t)j); });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) best = max(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
    if (lane == 0) s.wave_mass[w] = best;
    __syncthreads();
    for (int i = 0; i < 16; ++i) best = max(best, s.wave_mass[i]);
    const float t = a.t != nullptr ? a.t[b] : a.t0, p = a.p != nullptr ? a.p[b] : a.p0, m = a.m != nullptr ? a.m[b] : a.m0;
    const int k = a.k != nullptr ? a.k[b] : a.k0;
    const uint32_t top = (uint32_t)(best >> 32);
    if (top <= kMinusInf || !(t > 0.f)) {              // uniform
        if (tid == 0) {
            const bool none = top <= kMinusInf;
            a.token[b] = none ? 0 : (int64_t)~(uint32_t)best;
            if (a.logprob != nullptr) a.logprob[b] = none ? -INFINITY : 0.f;
            if (none) report_error(kErrLogits);
        }
        return;
    }
    Row row;
    row.top = of_order(top);
    row.inv_bins = kPerNat / t;
    row.inv_t = 1.0 / (double)t;
    row.min_p = fmin((double)m, 1.0);
    const float u0 = a.u[b];
    const double u = u0 > 0.f ? fmin((double)u0, 1.0 - 0x1p-24) : 0.0;
    uint32_t c_all;
    uint64_t m_all;
    const bool few = k > 0 && k <= kBins;
    fill_bins(s, c_all, m_all, [&] {
        r.each([&](float l, int) {
            if (order_of(l) <= kMinusInf) return;
            const int i = row.bin(l);
            if (i == kBins - 1) return;                // (weights of 0)
            if (few) {
                atomicAdd(&s.count[i], 1u);
                return;
            }
            const uint64_t x = row.weight(l);
            if (x == 0) return;
            atomicAdd(&s.count[i], 1u);
            atomicAdd((unsigned long long*)&s.mass[i], (unsigned long long)x);
        });
    });
    bool listed = false;
    int n = 0;
    if (few) {                                         // uniform
        const Bound rank{Bound::kRank, min((uint32_t)k, c_all), 0.0};
        uint32_t c = 0, in;
        uint64_t none = 0;
        const int last = find_bin(s, rank, c, none, in);
        listed = c + in <= (uint32_t)kList;
        __syncthreads();
        if (listed) {
            if (tid == 0) s.n = 0;
            __syncthreads();
            r.each([&](float l, int j) {
                const uint32_t o = order_of(l);
                if (o <= kMinusInf || row.bin(l) > last) return;
                const uint32_t at = atomicAdd(&s.n, 1u);
                if (at < (uint32_t)kList) s.list[at] = (uint64_t)~o << 32 | (uint32_t)j;
            });
            __syncthreads();
            n = min((int)s.n, kList);
            sort_list(s, n);
        } else {
            fill_bins(s, c_all, m_all, [&] {
                r.each([&](float l, int) {
                    if (order_of(l) <= kMinusInf) return;
                    const int i = row.bin(l);
                    const uint64_t x = i == kBins - 1 ? 0 : row.weight(l);
                    if (x == 0) return;
                    atomicAdd(&s.count[i], 1u);
                    atomicAdd((unsigned long long*)&s.mass[i], (unsigned long long)x);
                });
            });
        }
    }
    auto find = [&](const Bound& bound) {
        if (listed) return find_token(s, row, bound, n, 0, 0);
        uint32_t c = 0, in;
        uint64_t mass = 0;
        const int bin = find_bin(s, bound, c, mass, in);
        // (the bins are overwritten where a bin is cut further: they are filled again for the next bound)
        return find_in_bin(s, r, row, bound, bin, c, mass, in);
    };
    auto refill = [&] {
        if (listed) return;
        fill_bins(s, c_all, m_all, [&] {
            r.each([&](float l, int) {
                if (order_of(l) <= kMinusInf) return;
                const int i = row.bin(l);
                const uint64_t x = i == kBins - 1 ? 0 : row.weight(l);
                if (x == 0) return;
                atomicAdd(&s.count[i], 1u);
                atomicAdd((unsigned long long*)&s.mass[i], (unsigned long long)x);
            });
        });
    };
    uint64_t S = m_all;
    if (k > 0 && (listed || (uint32_t)k < c_all)) {
        S = find(Bound{Bound::kRank, (uint32_t)k, 0.0}).mass;
        refill();
    }
    if (p < 1.f) {
        S = find(Bound{Bound::kReach, 0, (double)p * (double)S}).mass;
        refill();
    }
    const Found f = find(Bound{Bound::kPass, 0, u * (double)S});
    if (tid == 0) {
        const float l = of_order(~(uint32_t)(f.token >> 32));
        a.token[b] = (int64_t)(uint32_t)f.token;
        if (a.logprob != nullptr) a.logprob[b] = (float)log((double)row.weight(l) / (double)S);
    }
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
    __shared__ Shared s;
    const int b = blockIdx.x;
    const MemoryRow<TYPE> r{(const uint8_t*)a.logits + b * a.stride * Logits<TYPE>::SIZE, a.V};
    sample_row(s, a, r, b);
}

hipError_t fetch_errors_sample(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

}  // namespace exkv

using namespace exkv;

extern "C" int exkv_sample(const void* logits, int64_t stride, int32_t type, int32_t B, int32_t V, const float* u, const float* temperature,
                           const int32_t* top_k, const float* top_p, const float* min_p, float temperature0, int32_t top_k0,
                           float top_p0, float min_p0, int64_t* token, float* logprob, hipStream_t stream) {
    EXKV_REQUIRE(type >= 0 && type <= 2, "sample: logits of type %d", type);
    EXKV_REQUIRE(B >= 0 && V > 0 && V <= (1 << 19) && stride >= 0, "sample: bad shape B=%d V=%d (up to %d)", B, V, 1 << 19);
    EXKV_REQUIRE((int64_t)B * kThreads <= (int64_t)UINT32_MAX, "sample: too many rows (%d)", B);
    if (B == 0) return EXKV_OK;
    EXKV_REQUIRE(logits && u && token, "sample: null pointer");
    EXKV_REQUIRE((uintptr_t)logits % (type == kFp32 ? 4 : 2) == 0, "sample: logits must be aligned to their size");
    const SampleArgs a{logits, stride, B, V, u, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0, token, logprob};
    const dim3 grid((unsigned)B), block(kThreads);
    if (type == kBf16)
        hipLaunchKernelGGL((sample_kernel<kBf16>), grid, block, 0, stream, a);
    else if (type == kFp16)
        hipLaunchKernelGGL((sample_kernel<kFp16>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((sample_kernel<kFp32>), grid, block, 0, stream, a);
    return hip_status(hipGetLastError(), "sample");
}
