// The attention that a packed prompt's keys receive from its queries, for gfx950 (no counterpart in the reference): with
// sequences, positions and visible keys as in prompt attention, for key j of KV head h
//     out[h, j] = sum over the queries t (of each sequence the last `last`, or all) and the query heads g of h of
//                 softmax_j(q[t, g] . k[j, h] / sqrt(D)),
// 0 for keys that no sequence holds.
//
// Two passes over the products, since a weight needs its row's sum first. In both, one side of the product stands in
// registers, the other comes through LDS in two stages of 64 rows (32 at head dim 256), brought by direct loads, and
// S^T = K Q^T is made by v_mfma_f32_32x32x16_bf16 with keys as rows, so that a lane holds one query row (column) of 32
// and 16 keys of each block:
//   rows     a wavefront holds 64 query rows (row r of a sequence is query head r % G of token r / G) and walks the
//            keys they see: each row's sum of 2^(s - m) (s the score in log2 units), m the largest score of the
//            first unit with a visible key. Later scores need no maximum: fp32 holds sums of weights up to 2^100,
//            smaller ones lose nothing, and a sum that leaves the range is made again with a running maximum.
//   columns  a wavefront holds 64 keys and walks the tokens that see them, one query head after the other, adding up
//            2^(s - m) / sum of each key; the 32 lanes of a key are added at the end.
// Both are cut into parts where there are few tiles; parts are joined in order, so a call's bits do not change.
//
// Bound by the exponentials, two for each visible pair: one of 8,192 tokens, 32 query and 8 KV heads of 128, needs
// 2 x 1.07e9 of them and twice 275 GFLOP of products (460 us at the rate of a large library product); the call takes 521 to
// 547 us, by the card, of which under a kernel trace rows 253 and columns 291. Prompts of few rows are bound by the latency of
// their few stages: 64 queries of 32 heads over 16,385 keys 18 + 4 + 24 us (four stages in LDS instead of two do not shorten
// the rows: 19.6 us for then 19, and 8,192 tokens' 267 for 253).
#include "errors.hpp"
#include "prompt_stage.hpp"
#include "../../include/exactkv.h"

namespace exkv {

constexpr float kLowest = -3.402823466e38f;   // a maximum before any key
constexpr float kFar = 0x1p24f;        // log2 units from which on scores are told apart before they are scaled
constexpr float kMost = 0x1p100f;      // a row's sum relative to its first tile's maximum
constexpr int kTile = 256;             // rows, or keys, of a workgroup: 64 a wavefront

struct PromptMassArgs {
    const uint16_t *q, *k;             // rows of D channels, element strides below
    int64_t sq_t, sq_h, sk_t, sk_h;
    const int32_t *cu_q, *cu_k;        // [S + 1]
    int S, N, NK, Hq, Hkv, G, window, last;
    float qk_scale;                    // log2(e) / sqrt(D)
    int row_parts, col_parts;
    float2* part;                      // [row tiles, Hkv, row_parts, kTile]: m, sum
    float2* row;                       // [Hq, N]: m, 1 / sum; infinity and 0 where the row sees no key
    float* sums;                       // [col_parts, Hkv, NK]; out where there is one part
    float* out;                        // [Hkv, NK]
};

// A row's weights are 2^((s - m) scale) over their sum, m one of its scores. Both passes make them alike, so that a
// row's add up to 1 however far from 0 its scores lie: as s scale - M with M = m scale rounded, in one instruction;
// where M's rounding would be a bit of the exponent, from s - m. (With the sum's logarithm in the exponent too, the second
// pass adds where it now multiplies and adds: 8,192 tokens 512 to 532 us for 526 to 545, but five times the error, 2.7e-7.)
__device__ inline float scaled(float m, float scale) {
#pragma clang fp contract(off)
    return m * scale;
}
__device__ inline float weight_of(float s, float m, float scale) {
    const float M = scaled(m, scale);
    return exp2_fast(fabsf(M) > kFar ? (s - m) * scale : fmaf(s, scale, -M));
}
// From sums relative to m to sums relative to `to`.
__device__ inline float rescale(float m, float to, float scale) {
    const float a = scaled(m, scale), b = scaled(to, scale);
    return exp2_fast(fabsf(a) > kFar || fabsf(b) > kFar ? (m - to) * scale : a - b);
}

// Sequence s's queries that count, and its keys.
__device__ inline void counted_sequence(const PromptMassArgs& a, int s, int& q0, int& Lq, int& k0, int& Lk) {
    const bool bad = clip_sequence(a.cu_q[s], a.cu_q[s + 1], s == 0, a.N, q0, Lq);
    const bool bad_k = clip_sequence(a.cu_k[s], a.cu_k[s + 1], s == 0, a.NK, k0, Lk);
    if (bad | bad_k) report_error(kErrOffsets);
    if (a.last > 0 && Lq > a.last) {
        q0 += Lq - a.last;
        Lq = a.last;
    }
}

// The tile to take `t`-th, of kTile rows or keys: sequence by sequence, the tiles with the most to walk first (a
// sequence's last rows, its first keys). row0 counts rows, or keys. False where t is past them all.
template <bool ROWS>
__device__ inline bool tile_at(const PromptMassArgs& a, int t, PromptTile& tile) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
        int q0 = 0, Lq = 0, k0 = 0, Lk = 0;
        if (s0 + lane < a.S) counted_sequence(a, s0 + lane, q0, Lq, k0, Lk);
        const int n = (int)(((ROWS ? (int64_t)Lq * a.G : (int64_t)Lk) + kTile - 1) / kTile);
        const int incl = wave_incl_scan(n), total = __builtin_amdgcn_readlane(incl, 63);
        if (t < total) {
            const int l = max(0, first_lane(__ballot(incl > t)));
            const int end = __builtin_amdgcn_readlane(incl, l), count = __builtin_amdgcn_readlane(n, l);
            const int index = ROWS ? end - 1 - t : t - (end - count);
            tile.q0 = __builtin_amdgcn_readlane(q0, l);
            tile.Lq = __builtin_amdgcn_readlane(Lq, l);
            tile.k0 = __builtin_amdgcn_readlane(k0, l);
            tile.Lk = __builtin_amdgcn_readlane(Lk, l);
            tile.row0 = index * kTile;
            return index >= 0 && index < count;
        }
        t -= total;
    }
    return false;
}

// Every load so far has landed, and every wavefront's LDS reads of the stage loaded into next have returned.
__device__ inline void next_stage() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A stage's geometry: SR rows of D channels.
template <int D>
struct Stage {
    static constexpr int SR = keys_per_tile(D), SB = SR / 32, KS = D / 16, BYTES = SR * 2 * D;
    static constexpr int PIECES = D / 8, RPI = 64 / PIECES, LOADS = BYTES / 1024 / kWaves;
    // lane's byte offsets of the wavefront's loads, row pitch s_t elements
    __device__ static void offsets(int w, int lane, int64_t s_t, uint32_t (&off)[LOADS]) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = (w * LOADS + i) * RPI + lane / PIECES, c = lane % PIECES;
            off[i] = (uint32_t)(r * (int)s_t * 2 + (c ^ key_swizzle<D>(r)) * 16 - i * 1024);
        }
    }
    // the operand piece of block b, k-step s
    __device__ static bf16x8 piece(const uint8_t* lds, int st, int rd, int b, int s) {
        return *(const EXKV_LDS bf16x8*)((const EXKV_LDS uint8_t*)lds + st * BYTES + (rd ^ ((s & 7) << 5)) + (s >> 3) * 256 +
                                         b * 32 * 2 * D);
    }
    __device__ static int read_at(int col, int half) { return col * 2 * D + (half ^ key_swizzle<D>(col)) * 16; }
};

// The second pass's sums as 0, shared by all workgroups of the first: keys that no sequence holds stay so, in front of the
// first one and between offsets that do not ascend as well.
__device__ inline void zero_sums(const PromptMassArgs& a) {
    const int64_t n = (int64_t)a.col_parts * a.Hkv * a.NK;
    for (int64_t i = (int64_t)blockIdx.x * (64 * kWaves) + threadIdx.x; i < n; i += (int64_t)gridDim.x * (64 * kWaves)) a.sums[i] = 0.f;
}

template <int D>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) mass_rows_kernel(PromptMassArgs a) {
    typedef Stage<D> St;
    constexpr int KS = St::KS, SR = St::SR, SB = St::SB;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * St::BYTES];
    __shared__ int s_again;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int hk = (int)(blockIdx.x % (unsigned)a.Hkv), rest = (int)(blockIdx.x / (unsigned)a.Hkv);
    const int part = rest % a.row_parts, index = rest / a.row_parts;
    zero_sums(a);
    PromptTile tile;
    if (!tile_at<true>(a, index, tile)) return;
    const int col = lane & 31, half = lane >> 5, G = a.G, nrows = tile.Lq * G, shift = tile.Lk - tile.Lq;
    const int wrow0 = tile.row0 + 64 * w;
    const bool wave_on = wrow0 < nrows;
    const uint32_t span = a.window > 0 ? (uint32_t)a.window : 0x7FFFFFFFu;
    int tok[2], hq[2], pos[2];
    bf16x8 qf[2][KS];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
        const int row = min(wrow0 + 32 * rb + col, nrows - 1);
        tok[rb] = row / G;
        hq[rb] = hk * G + row % G;
        pos[rb] = tok[rb] + shift;
        const uint16_t* qp = a.q + (int64_t)(tile.q0 + tok[rb]) * a.sq_t + hq[rb] * a.sq_h + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[rb][s] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * s));
    }
    const int w_lo = __builtin_amdgcn_readfirstlane(pos[0]), w_hi = __builtin_amdgcn_readlane(pos[1], 31);
    int first, last;
    {
        const int t_lo = tile.row0 / G, t_hi = min(tile.row0 + kTile - 1, nrows - 1) / G;
        const int k_lo = a.window > 0 ? max(0, t_lo + shift - a.window + 1) : 0, k_hi = t_hi + shift;
        first = k_lo / SR;
        last = k_hi < 0 ? first - 1 : k_hi / SR;
        const int per = (last - first + a.row_parts) / a.row_parts;
        first += part * per;
        last = min(last, first + per - 1);
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(EXKV_LDS uint8_t*)lds) + w * St::LOADS * 1024;
    uint32_t off[St::LOADS];
    St::offsets(w, lane, a.sk_t, off);
    const int rd = St::read_at(col, half);
    float m[2], M[2], l[2];                            // M: m scaled
    // A unit is 32 keys of a stage and the wavefront's 64 rows. The next unit's products go among this one's exponentials,
    // a k-step each (which take 768 cycles a unit at head dim 128, the products 512): a wavefront alone keeps both busy.
    auto walk = [&](auto safe) {
        constexpr bool SAFE = decltype(safe)::value;
        constexpr int AHEAD = 2;                       // k-steps of keys read ahead
        m[0] = m[1] = M[0] = M[1] = kLowest;
        l[0] = l[1] = 0.f;
        if (first > last) return;
        Stream<D, SR> keys(a.k, a.sk_t, hk * a.sk_h, tile, first * SR);
        auto load = [&](int st) {
            each<St::LOADS>([&](auto i) { load_piece<i.value>(keys.buf, off[i.value], lds0 + st * St::BYTES); });
            keys.next();
        };
        auto products = [&](int st, int kb, f32x16 (&sc)[2], auto between) {
            bf16x8 kf[KS];
            each<AHEAD>([&](auto s) { kf[s.value] = St::piece(lds, st, rd, kb, s.value); });
            each<KS>([&](auto step) {
                constexpr int s = decltype(step)::value;
                if constexpr (s + AHEAD < KS) kf[s + AHEAD] = St::piece(lds, st, rd, kb, s + AHEAD);
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
                    if constexpr (s == 0)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sc[rb][i] = 0.f;
                    sc[rb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], qf[rb][s], sc[rb], 0, 0, 0);
                }
                between(step);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        // the maximum that a row's weights are relative to: of its first unit with a visible key (SAFE: so far)
        auto raise = [&](const f32x16 (&sc)[2]) {
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
                if (SAFE || __ballot(m[rb] == kLowest) != 0) {
                    float mx = sc[rb][0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[rb][i]);
                    mx = fmaxf(mx, kLowest);
                    if (SAFE ? mx > m[rb] : m[rb] == kLowest) {
                        if (SAFE) l[rb] *= rescale(m[rb], mx, a.qk_scale);
                        m[rb] = mx;
                        M[rb] = scaled(mx, a.qk_scale);
                    }
                }
        };
        float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
        // (weights are made here, not sunk to the sums' use)
        auto here = [](float (&x)[2]) { asm volatile("" : "+v"(x[0]), "+v"(x[1])); };
        auto weigh = [&](const f32x16 (&sc)[2], int e) {
            sum[e >> 4][e & 1] += SAFE ? weight_of(sc[e >> 4][e & 15], m[e >> 4], a.qk_scale)
                                       : exp2_fast(fmaf(sc[e >> 4][e & 15], a.qk_scale, -M[e >> 4]));
        };
        auto settle = [&] {
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                l[rb] += sum[rb][0] + sum[rb][1];
                sum[rb][0] = sum[rb][1] = 0.f;
            }
        };
        // this unit's weights, of keys j0 on, and the next one's scores: where every row sees all of them, and otherwise
        auto full_step = [&](f32x16 (&cur)[2], f32x16 (&nxt)[2], int st, int kb) {
            products(st, kb, nxt, [&](auto s) {
#pragma unroll
                for (int e = 32 * s.value / KS; e < 32 * (s.value + 1) / KS; ++e) weigh(cur, e);
                here(sum[s.value * 2 / KS]);
            });
        };
        auto part_step = [&](int j0, f32x16 (&cur)[2], f32x16 (&nxt)[2], bool more, int st, int kb) {
            if (more) products(st, kb, nxt, [](auto) {});
            if (j0 > w_hi || (a.window > 0 && j0 + 31 <= w_lo - a.window)) return;   // uniform: none seen
            if (j0 + 31 > w_lo || (a.window > 0 && j0 <= w_hi - a.window)) {   // uniform: not all seen
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
                    const int rel = pos[rb] - j0 - 4 * half;
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if ((uint32_t)(rel - (8 * (i >> 2) + (i & 3))) >= span) cur[rb][i] = -INFINITY;
                }
            }
            raise(cur);
#pragma unroll
            for (int e = 0; e < 32; ++e) weigh(cur, e);
            settle();
        };
        load(0);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[rb][s]));
        f32x16 s0[2], s1[2];
        if constexpr (SAFE) {                          // seldom: unit by unit
            for (int it = first; it <= last; ++it) {
                next_stage();
                if (it < last) load((it - first + 1) & 1);
                if (!wave_on) continue;
#pragma unroll 1
                for (int kb = 0; kb < SB; ++kb) {
                    products((it - first) & 1, kb, s0, [](auto) {});
                    part_step(it * SR + 32 * kb, s0, s1, false, 0, 0);
                }
            }
            return;
        }
        next_stage();
        if (first < last) load(1);
        if (wave_on) products(0, 0, s0, [](auto) {});
        auto part_stage = [&](int it, auto parity, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
            constexpr int st = decltype(parity)::value;
            if constexpr (SB == 2)
                if (wave_on) part_step(it * SR, cur, nxt, true, st, 1);
            const bool more = it < last;
            if (more) next_stage();
            if (it + 1 < last) load(st);
            if (wave_on) {
                if constexpr (SB == 2)
                    part_step(it * SR + 32, nxt, cur, more, st ^ 1, 0);
                else
                    part_step(it * SR, cur, nxt, more, st ^ 1, 0);
            }
        };
        auto full_stage = [&](int it, auto parity, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
            constexpr int st = decltype(parity)::value;
            if constexpr (SB == 2) full_step(cur, nxt, st, 1);
            next_stage();
            if (it + 1 < last) load(st);
            if constexpr (SB == 2)
                full_step(nxt, cur, st ^ 1, 0);
            else
                full_step(cur, nxt, st ^ 1, 0);
            settle();
        };
        constexpr std::integral_constant<int, 0> even{};
        constexpr std::integral_constant<int, 1> odd{};
        // (at two units a stage, a stage ends with the scores where they began; two stages a turn, and the full ones in a loop
        // of their own, so that registers need no copies)
        for (int it = first; it <= last; it += 2) {
            const bool set = __ballot(m[0] == kLowest || m[1] == kLowest) == 0;
            while (set && wave_on && it + 1 < last && (it + 2) * SR - 1 <= w_lo && (a.window == 0 || it * SR > w_hi - a.window)) {
                full_stage(it, even, s0, s1);
                if constexpr (SB == 2)
                    full_stage(it + 1, odd, s0, s1);
                else
                    full_stage(it + 1, odd, s1, s0);
                it += 2;
            }
            part_stage(it, even, s0, s1);
            if (it == last) break;
            if constexpr (SB == 2)
                part_stage(it + 1, odd, s0, s1);
            else
                part_stage(it + 1, odd, s1, s0);
        }
    };
    if (threadIdx.x == 0) s_again = 0;
    walk(std::false_type{});
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
        if (!(l[rb] < kMost) || (m[rb] != kLowest && fabsf(M[rb]) > kFar)) s_again = 1;
    __syncthreads();
    if (s_again != 0) walk(std::true_type{});          // uniform
    if (!wave_on) return;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
        const float m2 = __shfl_xor(m[rb], 32), l2 = __shfl_xor(l[rb], 32), top = fmaxf(m[rb], m2);
        const float sum = l[rb] * rescale(m[rb], top, a.qk_scale) + l2 * rescale(m2, top, a.qk_scale);
        if (half != 0 || wrow0 + 32 * rb + col >= nrows) continue;
        if (a.row_parts > 1)
            a.part[(((int64_t)index * a.Hkv + hk) * a.row_parts + part) * kTile + 64 * w + 32 * rb + col] = make_float2(top, sum);
        else
            a.row[(int64_t)hq[rb] * a.N + tile.q0 + tok[rb]] = sum == 0.f ? make_float2(INFINITY, 0.f) : make_float2(top, 1.f / sum);
    }
}

// The parts of 64 of a tile's rows joined: a thread a row and wavefront, with four parts or less each.
constexpr int kPartsEach = 4;
__global__ void __launch_bounds__(1024) mass_rows_join_kernel(PromptMassArgs a) {
    __shared__ float2 s[16][64];
    constexpr int QUARTERS = kTile / 64;
    const int hk = (int)(blockIdx.x % (unsigned)a.Hkv), rest = (int)(blockIdx.x / (unsigned)a.Hkv), index = rest / QUARTERS;
    const int r = threadIdx.x % 64, w = threadIdx.x / 64, waves = blockDim.x / 64, at = rest % QUARTERS * 64 + r;
    const float2* part = a.part + ((int64_t)index * a.Hkv + hk) * a.row_parts * kTile + at;
    float2 x[kPartsEach];                              // on their way while the tile is found
#pragma unroll
    for (int i = 0; i < kPartsEach; ++i)
        x[i] = w + waves * i < a.row_parts ? part[(int64_t)(w + waves * i) * kTile] : make_float2(kLowest, 0.f);
    PromptTile tile;
    if (!tile_at<true>(a, index, tile)) return;
    const int row = tile.row0 + at;
    const bool real = row < tile.Lq * a.G;             // (behind them parts were not written)
    float m = kLowest, l = 0.f;
#pragma unroll
    for (int i = 0; i < kPartsEach; ++i)
        if (real) {
            const float top = fmaxf(m, x[i].x);
            l = l * rescale(m, top, a.qk_scale) + x[i].y * rescale(x[i].x, top, a.qk_scale);
            m = top;
        }
    s[w][r] = make_float2(m, l);
    __syncthreads();
    if (w != 0 || !real) return;
    float2 all[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) all[i] = i < waves ? s[i][r] : make_float2(kLowest, 0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, all[i].x);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) l += all[i].y * rescale(all[i].x, m, a.qk_scale);
    a.row[(int64_t)(hk * a.G + row % a.G) * a.N + tile.q0 + row / a.G] = l == 0.f ? make_float2(INFINITY, 0.f) : make_float2(m, 1.f / l);
}

template <int D>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) mass_columns_kernel(PromptMassArgs a) {
    typedef Stage<D> St;
    constexpr int KS = St::KS, SR = St::SR, SB = St::SB;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * St::BYTES];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int hk = (int)(blockIdx.x % (unsigned)a.Hkv), rest = (int)(blockIdx.x / (unsigned)a.Hkv);
    const int part = rest % a.col_parts;
    PromptTile tile;
    if (!tile_at<false>(a, rest / a.col_parts, tile)) return;
    const int col = lane & 31, half = lane >> 5, G = a.G, shift = tile.Lk - tile.Lq;
    const int key0 = tile.row0, wkey0 = key0 + 64 * w;
    const bool wave_on = wkey0 < tile.Lk;
    const uint32_t span = a.window > 0 ? (uint32_t)a.window : 0x7FFFFFFFu;
    bf16x8 kf[2][KS];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const uint16_t* kp = a.k + (int64_t)(tile.k0 + min(wkey0 + 32 * kb + col, tile.Lk - 1)) * a.sk_t + hk * a.sk_h + 8 * half;
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[kb][s] = __builtin_bit_cast(bf16x8, ld16(kp + 16 * s));
    }
    // tokens that see one of the workgroup's keys, in tiles of SR
    const int key_hi = min(key0 + kTile, tile.Lk) - 1;
    const int t_lo = max(0, key0 - shift), t_hi = a.window > 0 ? (int)min((int64_t)tile.Lq - 1, (int64_t)key_hi - shift + a.window - 1) : tile.Lq - 1;
    const int first = t_lo / SR, tiles = t_hi < t_lo ? 0 : t_hi / SR - first + 1;
    const int64_t steps = (int64_t)G * tiles, per = (steps + a.col_parts - 1) / a.col_parts;
    const int64_t begin = min(steps, part * per), end = min(steps, begin + per);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(EXKV_LDS uint8_t*)lds) + w * St::LOADS * 1024;
    uint32_t off[St::LOADS];
    St::offsets(w, lane, a.sq_t, off);
    const int rd = St::read_at(col, half);
    f32x16 acc[2];
    // rows are tokens of one query head at a time: a "sequence" of Lq rows at the head's channels
    PromptTile rows = tile;
    rows.k0 = tile.q0;
    rows.Lk = tile.Lq;
    auto walk = [&](auto safe) {                       // the largest M of the rows
        constexpr bool SAFE = decltype(safe)::value;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[kb][i] = 0.f;
        int g = tiles > 0 ? (int)(begin / tiles) : 0, t = tiles > 0 ? (int)(begin % tiles) : 0;
        float2 row[SB], next_row[SB];                      // m, 1 / sum
        float far = 0.f;                                   // the largest M so far
        int gl = g, tl = t;                                // of the loads
        auto load = [&](int st) {
            Stream<D, SR> s(a.q, a.sq_t, (hk * G + gl) * a.sq_h, rows, (first + tl) * SR);
            each<St::LOADS>([&](auto i) { load_piece<i.value>(s.buf, off[i.value], lds0 + st * St::BYTES); });
#pragma unroll
            for (int rb = 0; rb < SB; ++rb) {
                const int tok = (first + tl) * SR + 32 * rb + col;
                next_row[rb] = tok < tile.Lq ? a.row[(int64_t)(hk * G + gl) * a.N + tile.q0 + tok] : make_float2(INFINITY, 0.f);
            }
            if (++tl == tiles) {
                tl = 0;
                ++gl;
            }
        };
        auto take = [&](int rb) {                          // the rows of the stage that has landed
            row[rb] = next_row[rb];
            const float M = scaled(row[rb].x, a.qk_scale);
            far = fmaxf(far, fabsf(M) < INFINITY ? fabsf(M) : 0.f);
            if (!SAFE) row[rb].x = M;
        };
        // A unit is 32 tokens of a stage and the wavefront's 64 keys, walked as the other pass walks its units.
        constexpr int AHEAD = 2;
        auto products = [&](int st, int rb, f32x16 (&sc)[2], auto between) {
            bf16x8 qf[KS];
            each<AHEAD>([&](auto s) { qf[s.value] = St::piece(lds, st, rd, rb, s.value); });
            each<KS>([&](auto step) {
                constexpr int s = decltype(step)::value;
                if constexpr (s + AHEAD < KS) qf[s + AHEAD] = St::piece(lds, st, rd, rb, s + AHEAD);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    if constexpr (s == 0)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sc[kb][i] = 0.f;
                    sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kb][s], qf[s], sc[kb], 0, 0, 0);
                }
                between(step);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        auto here = [](float x) {                          // made here, not sunk to its use
            asm volatile("" : "+v"(x));
            return x;
        };
        // this unit's weights, of tokens standing at p0 on, and the next one's scores: where all of them see every key, and otherwise
        auto full_step = [&](float2 row, f32x16 (&cur)[2], f32x16 (&nxt)[2], int st, int rb) {
            products(st, rb, nxt, [&](auto s) {
#pragma unroll
                for (int e = 32 * s.value / KS; e < 32 * (s.value + 1) / KS; ++e) {
                    acc[e >> 4][e & 15] = here(fmaf(exp2_fast(fmaf(cur[e >> 4][e & 15], a.qk_scale, -row.x)), row.y, acc[e >> 4][e & 15]));
                }
            });
        };
        auto part_step = [&](int p0, float2 row, f32x16 (&cur)[2], f32x16 (&nxt)[2], bool more, int st, int rb) {
            if (more) products(st, rb, nxt, [](auto) {});
            if (p0 + 31 < wkey0 || (a.window > 0 && p0 - (wkey0 + 63) >= a.window)) return;   // uniform: none sees
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                // (rows behind the last token are zeros, and zeros times an infinite key are no weight of 0: none of them sees a key)
                const int rel = p0 + col < tile.Lk ? p0 + col - wkey0 - 4 * half : -1;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = SAFE ? weight_of(cur[kb][i], row.x, a.qk_scale) : exp2_fast(fmaf(cur[kb][i], a.qk_scale, -row.x));
                    // (after the product: a row's sum may be NaN)
                    acc[kb][i] += (uint32_t)(rel - (kb * 32 + 8 * (i >> 2) + (i & 3))) < span ? x * row.y : 0.f;
                }
            }
        };
        const int count = (int)(end - begin);
        if (count > 0) {
            load(0);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(kf[kb][s]));
            next_stage();
#pragma unroll
            for (int rb = 0; rb < SB; ++rb) take(rb);
            if (count > 1) load(1);
            f32x16 s0[2], s1[2];
            if constexpr (SAFE) {                          // seldom: unit by unit
#pragma unroll 1
                for (int it = 0; it < count; ++it) {
                    if (it > 0) {
                        next_stage();
#pragma unroll
                        for (int rb = 0; rb < SB; ++rb) take(rb);
                        if (it + 1 < count) load((it + 1) & 1);
                    }
                    if (wave_on)
#pragma unroll 1
                        for (int rb = 0; rb < SB; ++rb) {
                            products(it & 1, rb, s0, [](auto) {});
                            part_step((first + t) * SR + shift + 32 * rb, rb == 0 ? row[0] : row[SB - 1], s0, s1, false, 0, 0);
                        }
                    if (++t == tiles) t = 0;
                }
                return far;
            }
            if (wave_on) products(0, 0, s0, [](auto) {});
            auto advance = [&] {
                if (++t == tiles) t = 0;
            };
            auto part_stage = [&](int it, auto parity, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
                constexpr int st = decltype(parity)::value;
                const int p0 = (first + t) * SR + shift;
                if constexpr (SB == 2)
                    if (wave_on) part_step(p0, row[0], cur, nxt, true, st, 1);
                const bool more = it + 1 < count;
                const float2 last_row = row[SB - 1];
                if (more) {
                    next_stage();
#pragma unroll
                    for (int rb = 0; rb < SB; ++rb) take(rb);
                }
                if (it + 2 < count) load(st);
                if (wave_on) {
                    if constexpr (SB == 2)
                        part_step(p0 + 32, last_row, nxt, cur, more, st ^ 1, 0);
                    else
                        part_step(p0, last_row, cur, nxt, more, st ^ 1, 0);
                }
                advance();
            };
            auto full_stage = [&](int it, auto parity, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
                constexpr int st = decltype(parity)::value;
                if constexpr (SB == 2) full_step(row[0], cur, nxt, st, 1);
                const float2 last_row = row[SB - 1];
                next_stage();
#pragma unroll
                for (int rb = 0; rb < SB; ++rb) take(rb);
                if (it + 2 < count) load(st);
                if constexpr (SB == 2)
                    full_step(last_row, nxt, cur, st ^ 1, 0);
                else
                    full_step(last_row, cur, nxt, st ^ 1, 0);
                advance();
            };
            // whether the tile of tokens `at` is whole, and all of them see every key of the wavefront
            auto full = [&](int at) {
                const int p0 = (first + at) * SR + shift;
                return p0 >= wkey0 + 63 && p0 + SR <= tile.Lk && (a.window == 0 || p0 + SR - 1 - wkey0 < a.window);
            };
            constexpr std::integral_constant<int, 0> even{};
            constexpr std::integral_constant<int, 1> odd{};
            for (int it = 0; it < count; it += 2) {
                while (wave_on && it + 2 < count && full(t) && full(t + 1 == tiles ? 0 : t + 1)) {
                    full_stage(it, even, s0, s1);
                    if constexpr (SB == 2)
                        full_stage(it + 1, odd, s0, s1);
                    else
                        full_stage(it + 1, odd, s1, s0);
                    it += 2;
                }
                part_stage(it, even, s0, s1);
                if (it + 1 == count) break;
                if constexpr (SB == 2)
                    part_stage(it + 1, odd, s0, s1);
                else
                    part_stage(it + 1, odd, s1, s0);
            }
        }
        return far;
    };
    if (__syncthreads_or(walk(std::false_type{}) > kFar)) walk(std::true_type{});
    if (!wave_on) return;
    // over the 32 lanes of a key: halving the values with the lanes, so that lane c of a half ends up with value
    // c >> 1 of a block, which is key 8 (c >> 3) + 4 half + (c >> 1 & 3)
    float* out = a.sums + ((int64_t)part * a.Hkv + hk) * a.NK + tile.k0;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = acc[kb][i];
#pragma unroll
        for (int n = 8, d = 16; n > 0; n >>= 1, d >>= 1) {
            const bool upper = (lane & d) != 0;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const float low = v[i], high = v[i + n];
                v[i] = (upper ? high : low) + __shfl_xor(upper ? low : high, d);
            }
        }
        v[0] += __shfl_xor(v[0], 1);
        const int i = col >> 1, key = wkey0 + 32 * kb + 8 * (i >> 2) + 4 * half + (i & 3);
        if ((col & 1) == 0 && key < tile.Lk) out[key] = v[0];
    }
}

// The parts of every key added up; 0 where the call has no query.
__global__ void __launch_bounds__(256) mass_columns_join_kernel(PromptMassArgs a) {
    const int64_t n = (int64_t)a.Hkv * a.NK, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= n) return;
    float sum = 0.f;
    if (a.S > 0)
#pragma unroll 8
        for (int i = 0; i < a.col_parts; ++i) sum += a.sums[i * n + at];
    a.out[at] = sum;
}

hipError_t fetch_errors_prompt_mass(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

// How a call is laid out: tiles at most (every sequence's last may be partial), and the parts of each, so that there
// are about 1,024 workgroups with a few steps each.
struct MassPlan {
    int64_t row_tiles, col_tiles;
    int row_parts, col_parts;
    int64_t part_bytes, row_bytes, sum_bytes;
};
static MassPlan plan_mass(int64_t S, int64_t N, int64_t NK, int64_t Hq, int64_t Hkv, int D, int64_t window, int64_t last) {
    MassPlan p{};
    const int64_t G = Hq / Hkv, SR = keys_per_tile(D);
    const int64_t rows = last > 0 && S < N / last + 1 && S * last < N ? S * last : N;
    p.row_tiles = (rows * G + S * (kTile - 1)) / kTile;
    p.col_tiles = (NK + S * (kTile - 1)) / kTile;
    const int64_t reach = window > 0 && window + kTile < NK ? window + kTile : NK;
    auto cut = [&](int64_t units, int64_t steps) {
        int64_t parts = units > 0 ? 1024 / units : 1;
        if (parts > steps / 4) parts = steps / 4;
        if (parts > 64) parts = 64;                    // (four for each of a workgroup's wavefronts in the rows' join)
        return (int)(parts < 1 ? 1 : parts);
    };
    p.row_parts = cut(p.row_tiles * Hkv, (reach + SR - 1) / SR);
    const int64_t most = last > 0 && last < N ? last : N, seen = window > 0 && window + kTile < most ? window + kTile : most;
    p.col_parts = cut(p.col_tiles * Hkv, (seen + SR - 1) / SR * G);
    p.part_bytes = p.row_parts > 1 ? p.row_tiles * Hkv * p.row_parts * kTile * 8 : 0;
    p.row_bytes = (Hq * N * 8 + 15) / 16 * 16;
    p.sum_bytes = p.col_parts > 1 ? (p.col_parts * Hkv * NK * 4 + 15) / 16 * 16 : 0;
    return p;
}

template <int D>
static void launch_prompt_mass(const PromptMassArgs& a, const MassPlan& p, hipStream_t stream) {
    const dim3 block(64 * kWaves);
    hipLaunchKernelGGL((mass_rows_kernel<D>), dim3((unsigned)(p.row_tiles * a.Hkv * a.row_parts)), block, 0, stream, a);
    if (a.row_parts > 1)
        hipLaunchKernelGGL(mass_rows_join_kernel, dim3((unsigned)(p.row_tiles * a.Hkv * (kTile / 64))), dim3(64 * ((a.row_parts + kPartsEach - 1) / kPartsEach)),
                           0, stream, a);
    hipLaunchKernelGGL((mass_columns_kernel<D>), dim3((unsigned)(p.col_tiles * a.Hkv * a.col_parts)), block, 0, stream, a);
}

}  // namespace exkv

using namespace exkv;

static bool rows_ok(const void* p, int64_t s_t, int64_t s_h) {
    return (uintptr_t)p % 16 == 0 && s_t % 8 == 0 && s_h % 8 == 0 && s_t >= 0 && s_h >= 0;
}

extern "C" int64_t exkv_prompt_mass_workspace(int32_t S, int32_t N, int32_t NK, int32_t Hq, int32_t Hkv, int32_t D, int32_t window,
                                              int32_t last) {
    if (!head_dim_ok(D) || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || S < 0 || N <= 0 || NK <= 0 || window < 0 || last < 0) return 0;
    const MassPlan p = plan_mass(S, N, NK, Hq, Hkv, D, window, last);
    return p.part_bytes + p.row_bytes + p.sum_bytes;
}

extern "C" int exkv_prompt_mass(const void* q, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t, int64_t sk_h,
                                const int32_t* cu_q, const int32_t* cu_k, int32_t S, int32_t N, int32_t NK, int32_t Hq, int32_t Hkv,
                                int32_t D, int32_t window, int32_t last, float qk_scale, float* out, void* ws, int64_t ws_bytes,
                                hipStream_t stream) {
    EXKV_REQUIRE(head_dim_ok(D), "prompt_mass: head dim must be 64, 128 or 256 (got %d)", D);
    EXKV_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "prompt_mass: %d query heads over %d KV heads", Hq, Hkv);
    EXKV_REQUIRE(S >= 0 && N >= 0 && NK >= 0 && window >= 0 && last >= 0, "prompt_mass: bad shape S=%d N=%d NK=%d window=%d last=%d", S, N,
                 NK, window, last);
    if (NK == 0) return EXKV_OK;
    EXKV_REQUIRE(out && cu_q && cu_k && k && (q || N == 0), "prompt_mass: null pointer");
    EXKV_REQUIRE((N == 0 || rows_ok(q, sq_t, sq_h)) && rows_ok(k, sk_t, sk_h),
                 "prompt_mass: rows must be 16-byte aligned, with strides of whole 16 bytes");
    // a stage of rows is one 32-bit window whose rows lie at least a row apart
    EXKV_REQUIRE(sk_t >= D && sk_t <= (1 << 23) && (N == 0 || (sq_t >= D && sq_t <= (1 << 23))),
                 "prompt_mass: query and key rows must lie %d to %d elements apart", D, 1 << 23);
    const int64_t G = Hq / Hkv;
    if (window > NK) window = NK;                      // no sequence is longer; sums of positions stay in 32 bits
    if (last > N) last = N;
    EXKV_REQUIRE(((int64_t)N + 1) * G < INT32_MAX - 1024 && (int64_t)N + 2 * (int64_t)NK < INT32_MAX - 1024,
                 "prompt_mass: too many rows (N=%d, NK=%d, %d heads per KV head)", N, NK, (int)G);
    const MassPlan p = plan_mass(S, N, NK, Hq, Hkv, D, window, last);
    EXKV_REQUIRE(p.row_tiles * p.row_parts * Hkv * 64 * kWaves <= (int64_t)UINT32_MAX && p.row_tiles * Hkv * (kTile / 64) * 1024 <= (int64_t)UINT32_MAX &&
                     p.col_tiles * p.col_parts * Hkv * 64 * kWaves <= (int64_t)UINT32_MAX &&
                     (int64_t)Hq * N <= (int64_t)UINT32_MAX && (int64_t)Hkv * NK <= (int64_t)UINT32_MAX,
                 "prompt_mass: too many rows (N=%d, NK=%d, %d query heads, %d KV heads, S=%d)", N, NK, Hq, Hkv, S);
    PromptMassArgs a{(const uint16_t*)q, (const uint16_t*)k, sq_t, sq_h, sk_t, sk_h, cu_q, cu_k, S, N, NK, Hq, Hkv, (int)G, window, last,
                     qk_scale, p.row_parts, p.col_parts, nullptr, nullptr, nullptr, out};
    if (N > 0 && S > 0) {
        const int64_t need = p.part_bytes + p.row_bytes + p.sum_bytes;
        EXKV_REQUIRE(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "prompt_mass: workspace of %lld bytes, %lld needed",
                     (long long)ws_bytes, (long long)need);
        a.row = (float2*)ws;
        a.sums = p.col_parts > 1 ? (float*)((uint8_t*)ws + p.row_bytes) : out;
        a.part = (float2*)((uint8_t*)ws + p.row_bytes + p.sum_bytes);
        if (D == 64)
            launch_prompt_mass<64>(a, p, stream);
        else if (D == 128)
            launch_prompt_mass<128>(a, p, stream);
        else
            launch_prompt_mass<256>(a, p, stream);
        if (p.col_parts == 1) return hip_status(hipGetLastError(), "prompt_mass");
    } else {
        a.S = 0;                                       // no query: zeros
    }
    hipLaunchKernelGGL(mass_columns_join_kernel, dim3((unsigned)(((int64_t)Hkv * NK + 255) / 256)), dim3(256), 0, stream, a);
    return hip_status(hipGetLastError(), "prompt_mass");
}
