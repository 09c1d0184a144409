// Causal attention of whole prompts, packed one behind the other, for gfx950: the prefill
// counterpart of decode attention (no kernel of the reference: its prefill runs in the model's
// own modules, exactkv/engine.py:42-49).
//
// Sequence s holds query rows cu_q[s] .. cu_q[s + 1] - 1 and key rows cu_k[s] .. cu_k[s + 1] - 1;
// its queries are its last tokens, so query t stands at key position p = t + Lk - Lq and attends
// to the keys j of its own sequence with p - window < j <= p (window 0: j <= p):
//     out[t, h] = sum_j softmax_j(q[t, h] . k[j, h / G] / sqrt(D)) v[j, h / G],
// and 0 where no key is visible.
//
// One workgroup of four wavefronts takes 128 rows of one sequence and KV head, where row r is query
// head r % G of token r / G: the G query heads of a KV head share its key and value tiles, and a tile
// of rows spans few tokens, so little of it lies beyond the causal edge, at any G. Each wavefront owns
// 32 rows and walks the visible keys 64 at a time (32 at head dim 256, whose registers then hold two
// wavefronts a SIMD: 8K tokens at 16q/4kv 491 to 508 us):
//   S^T = K Q^T   v_mfma_f32_32x32x16_bf16, keys as rows, the wavefront's rows as columns, so a
//                 lane holds one column (row of the tile) and half of its 64 scores: maximum and
//                 sum are in-lane plus one exchange between the two halves of the wavefront;
//   O^T += V^T P^T  the score registers, rounded to bf16, are P^T's operand as they stand: eight
//                 of a lane's scores are the keys 16 s + 4 half + {0 .. 3, 8 .. 11}, and V^T is
//                 read from the value rows in the same key order (ds_read_b64_tr_b16: four keys
//                 of one channel per lane and read).
// Key and value tiles arrive in LDS by direct loads (buffer_load ... lds, 16 bytes a lane; rows
// past the sequence's end read as zeros), two stages, one barrier per tile. The 16-byte pieces of
// a row are XOR-swizzled so that the reads of one piece over 16 or 32 rows hit every bank (no bank
// conflict counted).
//
// What bounds it: at 8K tokens, 32q/8kv, head dim 128, 485 to 501 us on several cards = 1,100 to 1,130
// TFLOP/s, 0.83 to 0.86 of what a large library product reaches here; both are held by power (1.76 GHz; the
// same call on zeros takes 359 us).
// Two workgroups a CU (four at head dim 64) overlap one's matrix products with the other's
// exponentials; one of eight wavefronts does so less (mixed prompts 79 / 68 us), three stages of keys
// with a second barrier a tile cost more than they hide (continued prompts 78 / 93). A workgroup alone
// on its CU needs 0.92 us a tile, of which the matrix products are 0.43.
//
// Numbers: scores, maxima, sums and the accumulator are fp32; the weights are rounded to bf16 for
// the matrix product (half a step, at most 2^-8 of each weight, as the bf16 output's own rounding).
// Weights are taken relative to a running maximum that is raised only when some score passes it
// by 2^8 (the accumulator is then rescaled), so they stay below 256.
//
// Values that a row does not attend to must not reach it, also where they are infinite or NaN,
// but the matrix product multiplies them by a weight of zero. And the accumulator, which is divided by the
// sum at the end only, overflows where values are finite but large (from about 2^128 / 2^8 / keys on).
// A wavefront whose result is not finite, or large, therefore looks through the values of its tiles, and where one that
// some of its rows do not see is not finite, or one is that large, computes the rows in question again over
// their visible keys alone (careful_rows; of split keys the part looks and the join computes); so do rows
// whose weights are all zero. What the formula gives then stands; other results pay for none of it.
#include "errors.hpp"
#include "prompt_stage.hpp"
#include "../../include/exactkv.h"

namespace exkv {

constexpr float kLowest = -1e30f;      // the running maximum before any key, in log2 units
constexpr float kRaise = 8.f;          // a score this far above the running maximum raises it
constexpr float kLarge = 0x1p120f;     // results from here on are looked at again: the weights' rounding, or a sum of
                                       // parts, may leave the range

struct PromptArgs {
    const uint16_t *q, *k, *v;         // rows of D channels, element strides below
    uint16_t* out;                     // [N, Hq, D]
    int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;
    const int32_t *cu_q, *cu_k;        // [S + 1]
    int S, N, NK, Hq, Hkv, G, window, zero_tail;
    float qk_scale;                    // log2(e) / sqrt(D)
    // keys split into up to `split` parts a tile, of about the tiles that fill `slots` workgroups: partial results
    int split, slots;
    int turn;                          // tiles from here on are taken in reverse
    float* part_o;                     // [split, N * Hq, D]
    float2* part_ml;                   // [split, N * Hq]: running maximum (log2 units), sum (or its negative)
    int32_t* part_n;                   // [N * Hq]: the row's parts
};

// Begin and length of sequence s's queries and keys; offsets that do not ascend from 0 are reported (once
// both are read: they arrive together).
__device__ inline void sequence_of(const PromptArgs& a, int s, int& q0, int& Lq, int& k0, int& Lk) {
    const bool bad = clip_sequence(a.cu_q[s], a.cu_q[s + 1], s == 0, a.N, q0, Lq);
    const bool bad_k = clip_sequence(a.cu_k[s], a.cu_k[s + 1], s == 0, a.NK, k0, Lk);
    if (bad | bad_k) report_error(kErrOffsets);
}

// The tile to take `t`-th: every wavefront finds it by itself from the offsets. The tiles with the most
// keys come first, over up to 64 sequences (a lane each); beyond, sequence by sequence, each one's last
// tile first. The longest tiles must not start last: twelve prompts of 0 to
// 1,500 tokens at 28q/4kv in their order / ordered 64.3 / 61.5 us, three at 14q/2kv with head dim 64
// and a window of 1,024 34.9 / 31.6. False where t is past the tiles of all sequences.
template <int KEYS>
__device__ inline bool find_tile(const PromptArgs& a, int t, PromptTile& tile) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
        int begin = 0, len = 0, begin_k = 0, len_k = 0;
        if (s0 + lane < a.S) sequence_of(a, s0 + lane, begin, len, begin_k, len_k);
        const int n = row_tiles(len, a.G), incl = wave_incl_scan(n), total = __builtin_amdgcn_readlane(incl, 63);
        if (t < total) {
            int l, index;
            if (!nth_tile<KEYS>(DeviceWave(), a.S, a.G, a.NK, t, len, len_k, n, incl, l, index)) {
                report_error(kErrOffsets);
                return false;
            }
            tile.q0 = __builtin_amdgcn_readlane(begin, l);
            tile.Lq = __builtin_amdgcn_readlane(len, l);
            tile.row0 = index * kRows;
            tile.k0 = __builtin_amdgcn_readlane(begin_k, l);
            tile.Lk = __builtin_amdgcn_readlane(len_k, l);
            return true;
        }
        t -= total;
    }
    return false;
}

// Of the key tiles first .. last that rows standing at keys p_lo .. p_hi walk: whether a value that some of
// these rows does not see is infinite or NaN, or any value so large that finite ones overflow a row's
// accumulator (N < 2^31 keys with weights up to 2^8: from 2^88 on). Otherwise a result that is not finite is
// what the formula gives (2,048 such tokens at 8q/8kv, head dim 128: 53 us, 32 else).
constexpr uint32_t kLargeBits = (127 + 88) << 7;
template <int D, int KEYS>
__device__ inline bool values_suspect(const PromptArgs& a, const PromptTile& tile, int hk, int p_lo, int p_hi, int first, int last) {
    constexpr int PIECES = D / 8, BATCH = 8;           // 16-byte pieces of a row; loads in flight
    const int lane = threadIdx.x & 63, from = first * KEYS;
    const int64_t n = (int64_t)(min((last + 1) * KEYS, tile.Lk) - from) * PIECES;
    // the largest exponent field + 1 of either half of a dword, where bit 15 says infinite or NaN
    u16x2 top = {0, 0};
    for (int64_t i0 = lane; i0 < n; i0 += 64 * BATCH) {
        uint4 x[BATCH];
        int j[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int64_t i = min(i0 + 64 * u, n - 1);  // the last piece once more where there is none
            j[u] = from + (int)(i / PIECES);
            x[u] = ld16(a.v + (int64_t)(tile.k0 + j[u]) * a.sv_t + hk * a.sv_h + i % PIECES * 8);
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const uint32_t keep = j[u] > p_lo || (a.window > 0 && j[u] <= p_hi - a.window) ? ~0u : 0x7FFF7FFFu;
            const uint32_t xs[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, ((xs[c] & 0x7F807F80u) + 0x00800080u) & keep));
        }
    }
    return __ballot(max(top.x, top.y) >= kLargeBits + 0x80) != 0;
}

// Rows (bit c of `rows`: row wrow0 + c) computed again from their visible keys alone, one row at a
// time: 64 scores at once, a lane each, for the maximum, again for the sum and again for the weights, which
// are divided by the sum first, so that finite values cannot overflow; then the values with D / 64 channels
// a lane. 2,048 tokens at 8q/8kv, head dim 128, every row so: 10 ms (32 us else).
template <int D>
__device__ __attribute__((always_inline)) inline void careful_rows(const PromptArgs& a, const PromptTile& tile, int wrow0, int hk,
                                                                   uint32_t rows) {
    constexpr int C = D / 64;
    const int lane = threadIdx.x & 63;
    while (rows != 0) {                                // uniform
        const int r = wrow0 + __builtin_ctz(rows);
        rows &= rows - 1;
        const int t = r / a.G, h = hk * a.G + r % a.G, p = t + tile.Lk - tile.Lq;
        const uint16_t* q = a.q + (int64_t)(tile.q0 + t) * a.sq_t + h * a.sq_h;
        const int first = a.window > 0 ? max(0, p - a.window + 1) : 0;
        auto score = [&](int j) {                      // of key j, in log2 units
            const uint16_t* k = a.k + (int64_t)(tile.k0 + j) * a.sk_t + hk * a.sk_h;
            float s = 0.f;
#pragma unroll 2
            for (int c = 0; c < D; c += 8) {
                const uint4 x = ld16(q + c), y = ld16(k + c);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s = fmaf(__uint_as_float(xs[i] << 16), __uint_as_float(ys[i] << 16), s);
                    s = fmaf(__uint_as_float(xs[i] & 0xFFFF0000u), __uint_as_float(ys[i] & 0xFFFF0000u), s);
                }
            }
            return s * a.qk_scale;
        };
        float m = -INFINITY, l = 0.f, o[C];
        bool nan = false;
        for (int j0 = first; j0 <= p; j0 += 64) {
            const float s = score(min(j0 + lane, p));  // the last key once more where there is none
            nan |= s != s;
            m = fmaxf(m, s);
        }
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        if (__ballot(nan) != 0) m = NAN;
        for (int c = 0; c < C; ++c) o[c] = 0.f;
        // (every weight is NaN where a score is: the first keys say so)
        const int end = m != m ? first : p;
        auto weight = [&](int j) { return j <= p ? exp2_fast(score(min(j, p)) - m) : 0.f; };
        for (int j0 = first; j0 <= end; j0 += 64) l += weight(j0 + lane);
        for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
        const float inv = 1.f / l;
        for (int j0 = first; j0 <= end; j0 += 64) {
            const int n = min(64, p - j0 + 1);
            const float w = weight(j0 + lane) * inv;
            const uint16_t* v = a.v + (int64_t)(tile.k0 + j0) * a.sv_t + hk * a.sv_h + C * lane;
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const float wi = __shfl(w, i);
                for (int c = 0; c < C; ++c) o[c] = fmaf(wi, bf16_float(v[i * a.sv_t + c]), o[c]);
            }
        }
        uint16_t* out = a.out + ((int64_t)(tile.q0 + t) * a.Hq + h) * D + C * lane;
        for (int c = 0; c < C; ++c) out[c] = __builtin_bit_cast(uint16_t, (__bf16)o[c]);
    }
}

// Rows that no sequence holds, from row `end` on, shared by `parts` workgroups.
template <int D, int THREADS>
__device__ inline void zero_rows(const PromptArgs& a, int64_t end, int part, int parts) {
    const int64_t per = (int64_t)a.Hq * D / 8, n = (a.N - end) * per;
    uint4* out = reinterpret_cast<uint4*>(a.out) + end * per;
    for (int64_t i = (int64_t)part * THREADS + threadIdx.x; i < n; i += (int64_t)parts * THREADS)
        out[i] = make_uint4(0, 0, 0, 0);
}

// Which row tile and part of its keys a workgroup takes where the keys are split (t: the workgroup's
// number of its KV head). Of the ways to cut the longest row tile into 1 to `split` parts it takes the
// one that a model of the time finds best, and `most` are then the key tiles of a part; a row tile of n
// key tiles has ceil(n / most). Lane k - 1 models k parts, in steps of one key tile (1.07 us with one
// workgroup on a CU): with r workgroups on every CU a step takes 0.8 r; parts that find no place at once
// wait for half a part on average; a part's results, written and read, cost 0.02 and 0.02 more per 128
// channels, and the second launch 3. The tiles' lengths ascend evenly within a sequence, from n0 to n1,
// so its tiles have on average (F(n1 / most) - F(n0 / most)) / (n1 / most - n0 / most) parts, F the
// integral of ceil. Every wavefront computes this from the offsets. Parts are then handed out without gaps
// (nth_part), since workgroups that have nothing to do take every second CU's place, or half the XCDs, from
// those that do (128 tokens on 8K keys 37.7 us with gaps, 31.5 so).
// Measured without / with split (us), 32q/8kv, head dim 128: 17 tokens on 32K keys 489 / 36, 512 on
// 16K 255 / 141, 128 on 8K 128 / 31.5.
__device__ inline float ceil_integral(float x) {
    const float f = floorf(x);
    return 0.5f * f * (f + 1.f) + (x - f) * (f + 1.f);
}
template <int N>
__device__ inline float ror(float x) {                 // lane i of a 16-lane row: lane (i - N) % 16 of it
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + N, 0xf, 0xf, false));
}
__device__ inline float wave_least(float x) {
    x = fminf(x, ror<8>(x));
    x = fminf(x, ror<4>(x));
    x = fminf(x, ror<2>(x));
    x = fminf(x, ror<1>(x));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fminf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fminf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <int D, int KEYS>
__device__ inline bool find_part(const PromptArgs& a, int limit, int& t, int& part, int& most) {
    const int lane = threadIdx.x & 63, k = lane + 1;
    // the lane's sequence (there are at most 64): its row tiles, key tiles of the first and of the last one
    int q0, k0, Lq = 0, Lk = 0;
    if (lane < a.S) sequence_of(a, lane, q0, Lq, k0, Lk);
    const int tiles = row_tiles(Lq, a.G);
    const int n0 = key_tiles_most<KEYS>(min((kRows - 1) / a.G, Lq - 1), Lq, Lk, a.G, a.window);
    const int n1 = key_tiles_most<KEYS>(Lq - 1, Lq, Lk, a.G, a.window);
    const float far = -wave_least(-(tiles > 0 ? (float)max(1, max(n0, n1)) : 1.f));
    const int longest = __builtin_amdgcn_readfirstlane((int)far);
    most = (longest + k - 1) / k;
    const float per = 1.f / (float)most;
    float model = 0.f, steps = 0.f;
    for (int i = 0; i < a.S; ++i) {
        const int n = __builtin_amdgcn_readlane(tiles, i), m0 = __builtin_amdgcn_readlane(n0, i), m1 = __builtin_amdgcn_readlane(n1, i);
        const float x0 = (float)min(m0, m1) * per, x1 = (float)max(m0, m1) * per;
        steps += 0.5f * (float)n * (float)(m0 + m1);
        model += (float)n * (x1 - x0 < 0.01f ? ceilf(x1 - 1e-4f) : (ceil_integral(x1) - ceil_integral(x0)) / (x1 - x0));
    }
    model = ceilf(model - 0.01f) * (float)a.Hkv;
    const float slots = (float)a.slots, side = ceilf(fminf(model, slots) * (1.f / 256.f));
    float time = (float)most;
    if (model > slots + 1.f) time = fmaxf(time, steps * (float)a.Hkv / slots + 0.5f * time);
    time *= side <= 1.f ? 1.07f : 0.8f * side;
    if (k > 1) time += 3.f + (0.02f + 0.02f / 128.f * D) * model;
    if (k > a.split || (k > 1 && model > (float)(limit * a.Hkv))) time = INFINITY;
    most = __builtin_amdgcn_readlane(most, max(0, first_lane(__ballot(time == wave_least(time)))));
    return nth_part<KEYS>(DeviceWave(), a.S, a.G, a.window, longest, limit, tiles, Lq, Lk, t, part, most);
}

template <int D, int KEYS, int WPE, bool PIPE>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
prompt_kernel(PromptArgs a, int tiles) {
    constexpr bool CUTS = D < 256 || PIPE;                       // (the other instance never splits keys)
    constexpr int KB = KEYS / 32;                                // 32-key blocks of a tile
    constexpr int NW = kWaves, KS = D / 16, NB = D / 32;         // wavefronts, score k-steps, 32-channel blocks
    constexpr int PIECES = D / 8, RPI = 64 / PIECES;             // 16-byte pieces of a row, rows per load
    constexpr int TILE = KEYS * 2 * D, LOADS = TILE / 1024 / NW;
    static_assert(TILE % (1024 * NW) == 0, "whole loads");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TILE];     // two key stages, then two value stages
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int hk = (int)blockIdx.x % a.Hkv;
    int t = (int)blockIdx.x / a.Hkv, part = 0, most = 0;
    bool found = true;
    if (CUTS && a.split > 1)                           // uniform
        found = find_part<D, KEYS>(a, (int)gridDim.x / a.Hkv, t, part, most);
    else if (t >= a.turn)
        t = tiles - 1 - (t - a.turn);
    PromptTile tile;
    found = found && find_tile<KEYS>(a, t, tile);
    if (a.zero_tail) {
        const int end = a.S > 0 ? min(max(a.cu_q[a.S], 0), a.N) : 0;
        if (end < a.N) zero_rows<D, 64 * NW>(a, end, (int)blockIdx.x, (int)gridDim.x);
    }
    if (!found) return;
    // the lane's row
    const int col = lane & 31, half = lane >> 5, G = a.G, nrows = tile.Lq * G;
    const int wrow0 = tile.row0 + 32 * w, row = min(wrow0 + col, nrows - 1);
    const int tok = row / G, hq = hk * G + row % G;
    const int shift = tile.Lk - tile.Lq, pos = tok + shift;      // the key it stands at; < 0: none visible
    // keys that the wavefront's first and last row, and the workgroup's, see
    const int w_lo = __builtin_amdgcn_readfirstlane(pos), w_hi = __builtin_amdgcn_readlane(pos, 31);
    const bool wave_on = wrow0 < nrows;
    const uint32_t span = a.window > 0 ? (uint32_t)a.window : 0x7FFFFFFFu;
    int first, last;
    key_tiles<KEYS>(tile, G, a.window, first, last);
    const int parts = CUTS && a.split > 1 ? parts_of(first, last, most) : 1;
    if (part >= parts) return;
    if (CUTS && a.split > 1 && part == 0 && half == 0 && wrow0 + col < nrows) a.part_n[(int64_t)(tile.q0 + tok) * a.Hq + hq] = parts;
    if (parts > 1) part_tiles(part, parts, first, last);

    bf16x8 qf[KS];
    const uint16_t* qp = a.q + (int64_t)(tile.q0 + tok) * a.sq_t + hq * a.sq_h + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * s));
    // waited for here, once (`settled`, behind the first tile's loads): the compiler would otherwise
    // wait for them at every use in the loop, and so for the next tiles' loads in flight
    auto settled = [&] {
#pragma unroll
        for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
    };

    // Loads: a wavefront brings LOADS KiB of a tile, one after the other, so that the instruction's
    // offset moves both addresses and M0 is written once a tile (the offset is taken off the lane's:
    // rows lie at least a row apart, so that stays >= 0). A tile's descriptor is the last one's, a
    // tile further; rows past the sequence's end lie past its size.
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(EXKV_LDS uint8_t*)lds) + w * LOADS * 1024;
    uint32_t k_off[LOADS], v_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (w * LOADS + i) * RPI + lane / PIECES, c = lane % PIECES;
        k_off[i] = (uint32_t)(r * (int)a.sk_t * 2 + (c ^ key_swizzle<D>(r)) * 16 - i * 1024);
        v_off[i] = (uint32_t)(r * (int)a.sv_t * 2 + (c ^ value_swizzle<D>(r)) * 16 - i * 1024);
    }
    Stream<D, KEYS> keys(a.k, a.sk_t, hk * a.sk_h, tile, first * KEYS), vals(a.v, a.sv_t, hk * a.sv_h, tile, first * KEYS);
    auto load_keys = [&](int st) {
        each<LOADS>([&](auto i) { load_piece<i.value>(keys.buf, k_off[i.value], lds0 + st * TILE); });
        keys.next();
    };
    auto load_values = [&](int st) {
        each<LOADS>([&](auto i) { load_piece<i.value>(vals.buf, v_off[i.value], lds0 + (2 + st) * TILE); });
        vals.next();
    };

    // reads: K piece 2 s + half of row 32 kb + col; V four keys x 16 channels per 16 lanes
    const int k_rd = col * 2 * D + (half ^ key_swizzle<D>(col)) * 16;
    const int vi = lane & 15, v_row = 4 * half + (vi >> 2);
    const int v_piece = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
    constexpr int VA = NB < 4 ? NB : 4;                // the swizzle turns two bits of a block's index
    int v_rd[VA];
#pragma unroll
    for (int nb = 0; nb < VA; ++nb)
        v_rd[nb] = v_row * 2 * D + ((4 * nb + v_piece) ^ value_swizzle<D>(v_row)) * 16 + (vi & 1) * 8;

    f32x16 o[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nb][i] = 0.f;
    float m = kLowest, l = 0.f;

    // the 16-byte K pieces of block kb, k-step s in K stage st, as the scores' operand
    auto key_piece = [&](int st, int kb, int s) {
        return *(const EXKV_LDS bf16x8*)((const EXKV_LDS uint8_t*)lds + st * TILE + (k_rd ^ ((s & 7) << 5)) + (s >> 3) * 256 + kb * 32 * 2 * D);
    };
    auto value_piece = [&](int st, int s, int nb) {
        const EXKV_LDS uint8_t* p = (const EXKV_LDS uint8_t*)lds + (2 + st) * TILE + v_rd[nb % VA] + nb / VA * 256 + 16 * s * 2 * D;
        union {
            s16x4 q[2];
            bf16x8 v;
        } u;
        u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EXKV_LDS s16x4*)p);
        u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EXKV_LDS s16x4*)(p + 8 * 2 * D));
        return u.v;
    };
    auto hide = [&](f32x16 (&sc)[KB], int it) {
        const int j0 = it * KEYS;
        if (j0 + KEYS - 1 <= w_lo && (a.window == 0 || j0 > w_hi - a.window)) return;   // uniform: all seen
        const int rel = pos - j0 - 4 * half;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((uint32_t)(rel - (kb * 32 + 8 * (i >> 2) + (i & 3))) >= span) sc[kb][i] = -INFINITY;
    };
    auto top = [&](const f32x16 (&sc)[KB]) {
        float mx = sc[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][i]);
        return halves_max(mx) * a.qk_scale;
    };
    auto raise = [&](float mx) {
        if (__ballot(mx > m + kRaise) == 0) return;    // uniform
        const float mn = fmaxf(m, mx), alpha = exp2_fast(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[nb][i] *= alpha;
    };
    auto scores = [&](int st, f32x16 (&sc)[KB]) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(key_piece(st, kb, s), qf[s], sc[kb], 0, 0, 0);
    };
    // weights of scores 2 i, 2 i + 1 of the operand's order: dword i % 4 of operand piece i / 4
    auto weigh = [&](const f32x16 (&sc)[KB], uint32_t (&pw)[8 * KB], int i) {
        const int r = 8 * (i >> 2 & 1) + 2 * (i & 3);
        const float p0 = exp2_fast(fmaf(sc[i >> 3][r], a.qk_scale, -m)), p1 = exp2_fast(fmaf(sc[i >> 3][r + 1], a.qk_scale, -m));
        l += p0;
        l += p1;
        pw[i] = pack_bf16(p0, p1);
    };
    auto weight_piece = [&](const uint32_t (&pw)[8 * KB], int s) {
        const u32x4 u = {pw[4 * s], pw[4 * s + 1], pw[4 * s + 2], pw[4 * s + 3]};
        return __builtin_bit_cast(bf16x8, u);
    };
    // every load so far has landed, and every wavefront is done with the stages loaded into next: its LDS
    // reads have returned (the products that use them may be placed behind the barrier, and the wait for
    // a read with them)
    auto next_stage = [&] {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    if constexpr (PIPE) {
        // One tile a step: its scores `cur` become weights and meet the values while the next tile's
        // scores `nxt` are made, and what one wavefront waits for is issued before other work: the
        // scores' products (512 of a step's 1,024 matrix cycles) go two at a time with a piece of the
        // loads of the tiles after (their issue costs 350 cycles on their own), half of the weights,
        // and the first value pieces, which the products after the maximum need. A step of a
        // workgroup alone on its CU takes 0.92 us so, 0.97 with the compiler's order.
        constexpr int EARLY = 4 * KB, AHEAD = 2;       // weight pairs among the scores; key k-steps read ahead
        auto step = [&](int it, auto stage, f32x16 (&cur)[KB], f32x16 (&nxt)[KB]) {
            constexpr int st = decltype(stage)::value;
            const bool more = it < last;               // uniform
            next_stage();
            if (!wave_on) {
                if (more) {
                    load_keys(st);
                    load_values(st ^ 1);
                }
                return;
            }
            uint32_t pw[8 * KB];
            float mx = kLowest;
            bf16x8 vf[2][NB];
            if (more) {
                bf16x8 kf[KS][KB];
                each<AHEAD>([&](auto s) {
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) kf[s.value][kb] = key_piece(st ^ 1, kb, s.value);
                });
                each<KS>([&](auto step) {
                    constexpr int s = decltype(step)::value;
                    if constexpr (s + AHEAD < KS)
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb) kf[s + AHEAD][kb] = key_piece(st ^ 1, kb, s + AHEAD);
                    if constexpr (s >= KS - 2)
#pragma unroll
                        for (int nb = NB / 2 * (s - KS + 2); nb < NB / 2 * (s - KS + 3); ++nb) vf[0][nb] = value_piece(st, 0, nb);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) {
                        if constexpr (s == 0)
#pragma unroll
                            for (int i = 0; i < 16; ++i) nxt[kb][i] = 0.f;
                        nxt[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s][kb], qf[s], nxt[kb], 0, 0, 0);
                    }
                    // (past the last tile: loads of no bytes, zeros to a stage that nothing reads)
                    if constexpr (s < LOADS) load_piece<s>(keys.buf, k_off[s], lds0 + st * TILE);
                    if constexpr (s == LOADS - 1) keys.next();
                    if constexpr (s >= KS - LOADS)
                        load_piece<s - (KS - LOADS)>(vals.buf, v_off[s - (KS - LOADS)], lds0 + (2 + (st ^ 1)) * TILE);
                    if constexpr (s == KS - 1) vals.next();
#pragma unroll
                    for (int i = EARLY * s / KS; i < EARLY * (s + 1) / KS; ++i) {
                        weigh(cur, pw, i);
                        asm volatile("" : "+v"(pw[i]), "+v"(l));     // here, not sunk to its use
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                hide(nxt, it + 1);
                mx = top(nxt);
            } else {
#pragma unroll
                for (int i = 0; i < EARLY; ++i) weigh(cur, pw, i);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) vf[0][nb] = value_piece(st, 0, nb);
            }
#pragma unroll
            for (int s = 0; s < 2 * KB; ++s) {
                if (s + 1 < 2 * KB)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) vf[(s + 1) & 1][nb] = value_piece(st, s + 1, nb);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[s & 1][nb], weight_piece(pw, s), o[nb], 0, 0, 0);
                if (s + 1 < 2 * KB)
#pragma unroll
                    for (int i = 4 * (s + 1); i < 4 * (s + 2); ++i)
                        if (i >= EARLY) weigh(cur, pw, i);
            }
            raise(mx);
        };
        if (first <= last) {
            f32x16 s0[KB], s1[KB];
            load_keys(0);
            load_values(0);
            settled();
            next_stage();
            if (first < last) load_keys(1);
            if (wave_on) {
                scores(0, s0);
                hide(s0, first);
                m = fmaxf(m, top(s0));
            }
            for (int it = first; it <= last; it += 2) {
                step(it, std::integral_constant<int, 0>{}, s0, s1);
                if (it == last) break;
                step(it + 1, std::integral_constant<int, 1>{}, s1, s0);
            }
        }
    } else {
        if (first <= last) {
            load_keys(0);
            load_values(0);
        }
        settled();
        for (int it = first; it <= last; ++it) {
            const int st = (it - first) & 1;
            next_stage();
            if (it < last) {
                load_keys(st ^ 1);
                load_values(st ^ 1);
            }
            const int j0 = it * KEYS;
            if (!wave_on || j0 > w_hi || (a.window > 0 && j0 + KEYS - 1 <= w_lo - a.window)) continue;   // uniform: none seen
            f32x16 sc[KB];
            uint32_t pw[8 * KB];
            scores(st, sc);
            hide(sc, it);
            raise(top(sc));
#pragma unroll
            for (int i = 0; i < 8 * KB; ++i) weigh(sc, pw, i);
#pragma unroll
            for (int s = 0; s < 2 * KB; ++s)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(value_piece(st, s, nb), weight_piece(pw, s), o[nb], 0, 0, 0);
        }
    }

    if (!wave_on) return;
    l = halves_sum(l);
    const bool live = wrow0 + col < nrows, seen = pos >= 0;
    if (parts > 1) {
        const int64_t row_out = (int64_t)part * a.N * a.Hq + (int64_t)(tile.q0 + tok) * a.Hq + hq;
        // the join adds up to 64 parts; what it cannot see, suspect values among this part's, is the sum's sign
        float size = 0.f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) size += fabsf(o[nb][i]);
        const bool suspect = __ballot(live && l == l && !(size < kLarge)) != 0 &&
                             values_suspect<D, KEYS>(a, tile, hk, w_lo, w_hi, first, last);
        if (!live) return;
        if (half == 0) a.part_ml[row_out] = make_float2(m, suspect ? -l : l);
        float* op = a.part_o + row_out * D + 4 * half;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4*>(op + 32 * nb + 2 * i) = make_float4(o[nb][i], o[nb][i + 1], o[nb][i + 2], o[nb][i + 3]);
        return;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    float size = 0.f;                                  // not below kLarge once a value is not, or not finite
    uint16_t* op = a.out + ((int64_t)(tile.q0 + tok) * a.Hq + hq) * D + 4 * half;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = l == 0.f ? 0.f : o[nb][i + j] * inv;     // no key seen: 0, whatever the hidden values are
                size += fabsf(x[j]);
            }
            if (live) *reinterpret_cast<uint2*>(op + 32 * nb + 2 * i) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        }
    // (l is NaN where a score the row sees is infinite or NaN: so is the row)
    const uint64_t empty = __ballot(live && seen && l == 0.f), odd = __ballot(live && seen && l == l && !(size < kLarge));
    uint64_t again = empty;
    if (odd != 0 && values_suspect<D, KEYS>(a, tile, hk, w_lo, w_hi, first, last)) again |= odd;
    if (again != 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // these rows' stores come first
        careful_rows<D>(a, tile, wrow0, hk, (uint32_t)again | (uint32_t)(again >> 32));
    }
}

// The parts of a split joined: with M the largest of a row's maxima m_i,
//     out = sum_i o_i 2^(m_i - M) / sum_i l_i 2^(m_i - M).
// D / 4 lanes hold a row, four channels each, and at first a part's maximum and sum each (hence no more
// parts than that); then every part's factor goes to all of them, and the parts' loads do not wait for
// one another. Rows of one part are done. Bound by the parts' reads, which the other launch has just
// written: 813 tokens of two continued prompts 7.0 us (joined by a workgroup per four rows of a tile,
// a row after the other, 12.5).
template <int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(PromptArgs a) {
    constexpr int LPR = D / 4, RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j = lane % LPR;
    const int rows = min(max(a.cu_q[a.S], 0), a.N) * a.Hq;       // of sequences
    const int row = ((int)blockIdx.x * 4 + w) * RPW + lane / LPR, at = min(row, rows - 1);
    const int parts = row < rows ? min(a.part_n[at], a.split) : 0;
    if (__ballot(parts > 1) == 0) return;
    const int64_t stride = (int64_t)a.N * a.Hq;
    const float2 ml = j < parts ? a.part_ml[j * stride + at] : make_float2(kLowest, 0.f);
    float M = ml.x;
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
    const float f = exp2_fast(ml.x - M);
    const uint64_t suspect = __ballot(__float_as_int(ml.y) < 0);
    float l = fabsf(ml.y) * f;
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) l += __shfl_xor(l, d);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* po = a.part_o + (int64_t)at * D + 4 * j;
#pragma unroll 8
    for (int i = 0; i < parts; ++i) {                  // the lanes of a row stay together
        const float4 x = *reinterpret_cast<const float4*>(po + i * stride * D);
        const float fi = __shfl(f, i, LPR);
        o.x = fmaf(x.x, fi, o.x);
        o.y = fmaf(x.y, fi, o.y);
        o.z = fmaf(x.z, fi, o.z);
        o.w = fmaf(x.w, fi, o.w);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
    if (l == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);  // no key seen: 0, whatever the hidden values are
    const float size = fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w);
    if (parts > 1)
        *reinterpret_cast<uint2*>(a.out + (int64_t)at * D + 4 * j) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
    uint64_t odd = __ballot(parts > 1 && l == l && (!(size < kLarge) || l == 0.f));
    if (odd == 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    for (int i = 0; i < RPW; ++i) {                    // rows to compute again, one by one (uniform)
        const uint64_t lanes = (LPR == 64 ? ~0ull : (1ull << LPR) - 1ull) << (i * LPR);
        const bool none = __builtin_amdgcn_readlane(__float_as_int(l), i * LPR) == 0;
        if ((odd & lanes) == 0 || (!none && (suspect & lanes) == 0)) continue;
        const int r = __builtin_amdgcn_readlane(at, i * LPR), t = r / a.Hq, hq = r % a.Hq, hk = hq / a.G;
        int s = 0;                                     // the sequence that holds row t
        while (s + 1 < a.S && a.cu_q[s + 1] <= t) ++s;
        PromptTile tile{};
        sequence_of(a, s, tile.q0, tile.Lq, tile.k0, tile.Lk);
        const int tok = t - tile.q0, p = tok + tile.Lk - tile.Lq, own = tok * a.G + hq % a.G;
        if (tok < 0 || tok >= tile.Lq || p < 0) continue;
        careful_rows<D>(a, tile, own, hk, 1u);
    }
}

static int64_t workspace_bytes(const PromptPlan& p, int64_t N, int64_t Hq, int64_t D) {
    return (p.split * (D + 2) + 1) * N * Hq * 4;
}

// WPE wavefronts a SIMD, PIPE the next tile's scores beside this tile's weights. At head dim 64 four and
// no PIPE (8K tokens, 32q/8kv: 287 us; two and no PIPE 330), at 128 the registers of the second scores
// leave two (500 us; without PIPE 533), at 256 one (PromptPlan).
template <int D, int WPE, bool PIPE>
static void launch_prompt(const PromptArgs& a, const PromptPlan& p, hipStream_t stream) {
    constexpr int KEYS = keys_per_tile(D);
    const int64_t blocks = a.split > 1 ? p.blocks : p.tiles;
    hipLaunchKernelGGL((prompt_kernel<D, KEYS, WPE, PIPE>), dim3((unsigned)(blocks * a.Hkv)), dim3(64 * kWaves), 0, stream, a,
                       (int)p.tiles);
    if (a.split > 1)
        hipLaunchKernelGGL((prompt_merge_kernel<D>), dim3((unsigned)(((int64_t)a.N * a.Hq * (D / 4) + 255) / 256)), dim3(256),
                           0, stream, a);
}

hipError_t fetch_errors_prompt(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

}  // namespace exkv

using namespace exkv;

static bool rows_ok(const void* p, int64_t s_t, int64_t s_h) {
    return (uintptr_t)p % 16 == 0 && s_t % 8 == 0 && s_h % 8 == 0 && s_t >= 0 && s_h >= 0;
}

extern "C" int64_t exkv_prompt_workspace(int32_t S, int32_t N, int32_t NK, int32_t Hq, int32_t Hkv, int32_t D, int32_t window) {
    if (!head_dim_ok(D) || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || S < 0 || N <= 0 || NK <= 0 || window < 0) return 0;
    const PromptPlan p = plan_prompt(N, NK, S, Hq, Hkv, D, window);
    return p.split > 1 ? workspace_bytes(p, N, Hq, D) : 0;
}

extern "C" int exkv_prompt_attention(const void* q, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t, int64_t sk_h,
                                     const void* v, int64_t sv_t, int64_t sv_h, void* out, const int32_t* cu_q,
                                     const int32_t* cu_k, int32_t S, int32_t N, int32_t NK, int32_t Hq, int32_t Hkv,
                                     int32_t D, int32_t window, int32_t zero_tail, float qk_scale, void* ws, int64_t ws_bytes,
                                     hipStream_t stream) {
    EXKV_REQUIRE(head_dim_ok(D), "prompt_attention: head dim must be 64, 128 or 256 (got %d)", D);
    EXKV_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "prompt_attention: %d query heads over %d KV heads", Hq, Hkv);
    EXKV_REQUIRE(S >= 0 && N >= 0 && NK >= 0 && window >= 0, "prompt_attention: bad shape S=%d N=%d NK=%d window=%d", S, N,
                 NK, window);
    if (N == 0) return EXKV_OK;
    EXKV_REQUIRE(q && out && cu_q && cu_k && ((k && v) || NK == 0), "prompt_attention: null pointer");
    EXKV_REQUIRE(rows_ok(q, sq_t, sq_h) && (NK == 0 || (rows_ok(k, sk_t, sk_h) && rows_ok(v, sv_t, sv_h))) &&
                     (uintptr_t)out % 16 == 0,
                 "prompt_attention: rows must be 16-byte aligned, with strides of whole 16 bytes");
    // a tile of keys is one 32-bit window whose rows lie at least a row apart
    EXKV_REQUIRE(NK == 0 || (sk_t >= D && sv_t >= D && sk_t <= (1 << 23) && sv_t <= (1 << 23)),
                 "prompt_attention: key and value rows must lie %d to %d elements apart", D, 1 << 23);
    const int64_t G = Hq / Hkv;
    if (window > NK) window = NK;                      // no sequence is longer; sums of positions stay in 32 bits
    EXKV_REQUIRE(((int64_t)N + 1) * G < INT32_MAX - 1024 && (int64_t)N + 2 * (int64_t)NK < INT32_MAX - 1024 &&
                     ((int64_t)N * G / kRows + S + 1) * Hkv * 64 * kWaves <= (int64_t)UINT32_MAX,
                 "prompt_attention: too many rows (N=%d, NK=%d, %d heads per KV head, %d KV heads, S=%d)", N, NK, (int)G, Hkv, S);
    PromptArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)out, sq_t, sq_h, sk_t, sk_h,
                 sv_t, sv_h, cu_q, cu_k, S, N, NK, Hq, Hkv, (int)G, window, zero_tail, qk_scale, 1, 0, INT32_MAX, nullptr, nullptr, nullptr};
    PromptPlan p = plan_prompt(N, NK, S, Hq, Hkv, D, window);
    if (ws != nullptr && p.split > 1) {
        const int64_t rows = (int64_t)p.split * N * Hq, need = workspace_bytes(p, N, Hq, D);
        EXKV_REQUIRE((uintptr_t)ws % 16 == 0 && ws_bytes >= need, "prompt_attention: workspace of %lld bytes, %lld needed",
                     (long long)ws_bytes, (long long)need);
        a.split = p.split;
        a.slots = p.slots;
        a.part_o = (float*)ws;
        a.part_ml = (float2*)((float*)ws + rows * D);
        a.part_n = (int32_t*)(a.part_ml + rows);
    }
    a.turn = p.turn;
    if (D == 64)
        launch_prompt<64, 4, false>(a, p, stream);
    else if (D == 128)
        launch_prompt<128, 2, true>(a, p, stream);
    else if (p.alone)
        launch_prompt<256, 1, true>(a, p, stream);
    else
        launch_prompt<256, 2, false>(a, p, stream);
    return hip_status(hipGetLastError(), "prompt_attention");
}
