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
// One workgroup takes 32 NW rows of one sequence and KV head, where row r is query head r % G of
// token r / G: the G query heads of a KV head share its key and value tiles, and a tile of rows
// spans few tokens, so little of it lies beyond the causal edge, at any G. Each wavefront owns
// 32 rows and walks the visible keys 64 at a time:
//   S^T = K Q^T   v_mfma_f32_32x32x16_bf16, keys as rows, the wavefront's rows as columns, so a
//                 lane holds one column (row of the tile) and half of its 64 scores: maximum and
//                 sum are in-lane plus one exchange between the two halves of the wavefront;
//   O^T += V^T P^T  the score registers, rounded to bf16, are P^T's operand as they stand: eight
//                 of a lane's scores are the keys 16 s + 4 half + {0 .. 3, 8 .. 11}, and V^T is
//                 read from the value rows in the same key order (ds_read_b64_tr_b16: four keys
//                 of one channel per lane and read).
// Key and value tiles arrive in LDS by direct loads (buffer_load ... lds, 16 bytes a lane; rows
// past the sequence's end read as zeros), two stages, one barrier per tile. The 16-byte pieces of
// a row are XOR-swizzled so that the reads of one piece over 16 or 32 rows hit every bank.
//
// Numbers: scores, maxima, sums and the accumulator are fp32; the weights are rounded to bf16 for
// the matrix product (half a step, 2^-9 of each weight, no more than the bf16 output loses).
// Weights are taken relative to a running maximum that is raised only when some score passes it
// by 2^8 (the accumulator is then rescaled), so they stay below 256.
//
// Values that a row does not attend to must not reach it, also where they are infinite or NaN,
// but the matrix product multiplies them by a weight of zero. A wavefront whose result is not
// finite therefore computes the rows in question again, key by key over their visible keys
// (careful_rows): what the formula gives then stands, and finite inputs never pay for it.
#include "errors.hpp"
#include "tile.hpp"
#include "../../include/exactkv.h"

namespace exkv {

#define EXKV_LDS __attribute__((address_space(3)))

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -1e30f;      // the running maximum before any key, in log2 units
constexpr float kRaise = 8.f;          // a score this far above the running maximum raises it

struct PromptArgs {
    const uint16_t *q, *k, *v;         // rows of D channels, element strides below
    uint16_t* out;                     // [N, Hq, D]
    int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;
    const int32_t *cu_q, *cu_k;        // [S + 1]
    int S, N, NK, Hq, Hkv, G, window, zero_tail;
    float qk_scale;                    // log2(e) / sqrt(D)
};

// Two values to bf16 (nearest even): one v_cvt_pk_bf16_f32. Converted one by one they take three
// more instructions a pair.
__device__ inline uint32_t pack_bf16(float a, float b) {
    const f32x2 x = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
}
__device__ inline float bf16_float(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Over the two halves of a wavefront (lanes l and l ^ 32).
__device__ inline float halves_max(float x) {
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(c[0]), __uint_as_float(c[1]));
}
__device__ inline float halves_sum(float x) {
    const auto c = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(c[0]) + __uint_as_float(c[1]);
}

// A buffer descriptor over `bytes` bytes from p: loads past them return zeros.
__device__ inline u32x4 buffer_of(const void* p, uint32_t bytes) {
    const uint64_t a = (uint64_t)(uintptr_t)p;
    u32x4 b;
    b.x = __builtin_amdgcn_readfirstlane((uint32_t)a);
    b.y = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xFFFFu);
    b.z = __builtin_amdgcn_readfirstlane(bytes);
    b.w = 0x00020000u;
    return b;
}
// Direct-to-LDS load of 16 bytes a lane (lane l's land at lds + 16 l), ordered by the kernel's own
// s_waitcnt: inline, since the compiler would wait for every such load before each LDS read.
__device__ inline void load_lds16(u32x4 buf, uint32_t off, uint32_t lds) {
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(buf), "{m0}"(lds) : "memory");
}

// Which piece of a row's 16-byte pieces lies where: piece c of key row r at c ^ swizzle(r). Keys are
// read one piece over 16 rows at a time (16 pieces or 16 rows cover the 256 bytes of all banks),
// values four pieces over four rows.
template <int D>
__host__ __device__ constexpr int key_swizzle(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
template <int D>
__host__ __device__ constexpr int value_swizzle(int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }

// One sequence's share of a workgroup: rows row0 .. of its Lq * G, key rows k0 .. k0 + Lk - 1.
struct PromptTile {
    int q0, Lq, k0, Lk, row0;
};

// The offsets of sequence s, made fit for use where they are not: 0 <= begin <= end <= rows.
__device__ inline void sequence_of(const int32_t* cu, int s, int rows, int& begin, int& len, bool& bad) {
    const int a = cu[s], b = cu[s + 1];
    begin = min(max(a, 0), rows);
    const int end = min(max(b, begin), rows);
    len = end - begin;
    bad = begin != a || end != b || (s == 0 && a != 0);
}

// Tile t of the packed rows, each sequence's last tile first (the longest work of it): every wavefront
// finds it by itself, 64 sequences at a time. `before`: the tiles of all sequences, where t is past
// them (then false).
template <int ROWS>
__device__ inline bool find_tile(const PromptArgs& a, int t, PromptTile& tile, int& before, int& end) {
    const int lane = threadIdx.x & 63;
    before = 0;
    end = 0;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
        int begin = 0, len = 0;
        bool bad = false;
        if (s0 + lane < a.S) sequence_of(a.cu_q, s0 + lane, a.N, begin, len, bad);
        if (bad) report_error(kErrOffsets);
        const int n = (int)(((int64_t)len * a.G + ROWS - 1) / ROWS);
        const int incl = wave_incl_scan(n);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (t < before + total) {
            const int l = __builtin_ctzll(__ballot(incl > t - before));
            const int last = __builtin_amdgcn_readlane(incl, l) - 1 - (t - before);     // tile of the sequence
            tile.q0 = __builtin_amdgcn_readlane(begin, l);
            tile.Lq = __builtin_amdgcn_readlane(len, l);
            tile.row0 = last * ROWS;
            bool bad_k = false;
            sequence_of(a.cu_k, s0 + l, a.NK, tile.k0, tile.Lk, bad_k);
            if (bad_k) report_error(kErrOffsets);
            tile.k0 = __builtin_amdgcn_readfirstlane(tile.k0);
            tile.Lk = __builtin_amdgcn_readfirstlane(tile.Lk);
            return true;
        }
        before += total;
        end = __builtin_amdgcn_readlane(begin + len, min(63, a.S - 1 - s0));
    }
    return false;
}

// Rows (bit c of `rows`: the wavefront's row c) computed again from their visible keys alone, one row
// at a time with D / 64 channels a lane: the maximum first, then the sum.
template <int D>
__device__ __attribute__((always_inline)) inline void careful_rows(const PromptArgs& a, const PromptTile& tile, int wrow0, int hk,
                                                       uint32_t rows) {
    constexpr int C = D / 64;
    const int lane = threadIdx.x & 63;
    while (rows != 0) {
        const int r = wrow0 + __builtin_ctz(rows);
        rows &= rows - 1;
        const int t = r / a.G, h = hk * a.G + r % a.G, p = t + tile.Lk - tile.Lq;
        const uint16_t* q = a.q + (int64_t)(tile.q0 + t) * a.sq_t + h * a.sq_h + C * lane;
        const int first = a.window > 0 ? max(0, p - a.window + 1) : 0;
        float m = -INFINITY, l = 0.f, o[C];
        for (int c = 0; c < C; ++c) o[c] = 0.f;
        for (int pass = 0; pass < 2; ++pass)
            for (int j = first; j <= p; ++j) {
                const uint16_t* k = a.k + (int64_t)(tile.k0 + j) * a.sk_t + hk * a.sk_h + C * lane;
                float s = 0.f;
                for (int c = 0; c < C; ++c) s = fmaf(bf16_float(q[c]), bf16_float(k[c]), s);
                for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
                s *= a.qk_scale;
                if (pass == 0) {
                    m = s != s ? s : (m != m ? m : fmaxf(m, s));           // a NaN stays
                } else {
                    const uint16_t* v = a.v + (int64_t)(tile.k0 + j) * a.sv_t + hk * a.sv_h + C * lane;
                    const float w = exp2_fast(s - m);
                    l += w;
                    for (int c = 0; c < C; ++c) o[c] = fmaf(w, bf16_float(v[c]), o[c]);
                }
            }
        uint16_t* out = a.out + ((int64_t)(tile.q0 + t) * a.Hq + h) * D + C * lane;
        for (int c = 0; c < C; ++c) out[c] = __builtin_bit_cast(uint16_t, (__bf16)(p < first ? 0.f : o[c] / l));
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

template <int D, int NW, int KEYS, int WPE>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(WPE, WPE)))
prompt_kernel(PromptArgs a, int tiles) {
    constexpr int KB = KEYS / 32;                                // 32-key blocks of a tile
    constexpr int ROWS = 32 * NW, KS = D / 16, NB = D / 32;      // rows, score k-steps, 32-channel blocks
    constexpr int PIECES = D / 8, RPI = 64 / PIECES;             // 16-byte pieces of a row, rows per load
    constexpr int TILE = KEYS * 2 * D, LOADS = TILE / 1024 / NW;
    static_assert(TILE % (1024 * NW) == 0, "whole loads");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * TILE];     // K, V of stage 0, K, V of stage 1
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int hk = (int)blockIdx.x % a.Hkv, t = (int)blockIdx.x / a.Hkv;
    PromptTile tile;
    int before, end;
    if (!find_tile<ROWS>(a, t, tile, before, end)) {
        if (a.zero_tail && end < a.N)
            zero_rows<D, 64 * NW>(a, end, (t - before) * a.Hkv + hk, (tiles - before) * a.Hkv);
        return;
    }
    // the lane's row
    const int col = lane & 31, half = lane >> 5, G = a.G, nrows = tile.Lq * G;
    const int wrow0 = tile.row0 + 32 * w, row = min(wrow0 + col, nrows - 1);
    const int tok = row / G, hq = hk * G + row % G;
    const int shift = tile.Lk - tile.Lq, pos = tok + shift;      // the key it stands at; < 0: none visible
    // keys that the workgroup's and the wavefront's rows see
    const int t_lo = tile.row0 / G, t_hi = min(tile.row0 + ROWS - 1, nrows - 1) / G;
    const int k_lo = a.window > 0 ? max(0, t_lo + shift - a.window + 1) : 0, k_hi = t_hi + shift;
    const int w_lo = __builtin_amdgcn_readfirstlane(pos), w_hi = __builtin_amdgcn_readlane(pos, 31);
    const bool wave_on = wrow0 < nrows;
    const uint32_t span = a.window > 0 ? (uint32_t)a.window : 0x7FFFFFFFu;
    const int first = k_lo / KEYS, last = k_hi < 0 ? first - 1 : k_hi / KEYS;

    bf16x8 qf[KS];
    const uint16_t* qp = a.q + (int64_t)(tile.q0 + tok) * a.sq_t + hq * a.sq_h + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * s));

    // loads: the wavefront's pieces of a tile
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(EXKV_LDS uint8_t*)lds);
    uint32_t k_off[LOADS], v_off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (i * NW + w) * RPI + lane / PIECES, c = lane % PIECES;
        k_off[i] = (uint32_t)(r * (int)a.sk_t * 2 + (c ^ key_swizzle<D>(r)) * 16);
        v_off[i] = (uint32_t)(r * (int)a.sv_t * 2 + (c ^ value_swizzle<D>(r)) * 16);
    }
    auto load_tile = [&](int it, int stage) {
        const int j0 = it * KEYS, n = min(KEYS, tile.Lk - j0);
        const u32x4 kb = buffer_of(a.k + (int64_t)(tile.k0 + j0) * a.sk_t + hk * a.sk_h, (uint32_t)(((n - 1) * (int)a.sk_t + D) * 2));
        const u32x4 vb = buffer_of(a.v + (int64_t)(tile.k0 + j0) * a.sv_t + hk * a.sv_h, (uint32_t)(((n - 1) * (int)a.sv_t + D) * 2));
        const uint32_t at = lds0 + stage * 2 * TILE + w * 1024;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load_lds16(kb, k_off[i], at + i * NW * 1024);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) load_lds16(vb, v_off[i], at + TILE + i * NW * 1024);
    };

    // reads: K piece 2 s + half of row 32 kb + col; V four keys x 16 channels per 16 lanes
    const int k_rd = col * 2 * D + (half ^ key_swizzle<D>(col)) * 16;
    const int vi = lane & 15, v_row = 4 * half + (vi >> 2);
    const int v_piece = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1);
    int v_rd[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
        v_rd[nb] = v_row * 2 * D + ((4 * nb + v_piece) ^ value_swizzle<D>(v_row)) * 16 + (vi & 1) * 8;

    f32x16 o[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[nb][i] = 0.f;
    float m = kLowest, l = 0.f;

    auto tile_step = [&](int it, int stage) {
        const int j0 = it * KEYS;
        if (!wave_on || j0 > w_hi || (a.window > 0 && j0 + KEYS - 1 <= w_lo - a.window)) return;   // uniform: none visible
        const EXKV_LDS uint8_t* ks = (const EXKV_LDS uint8_t*)lds + stage * 2 * TILE;
        const EXKV_LDS uint8_t* vs = ks + TILE;
        f32x16 sc[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const bf16x8 kf = *(const EXKV_LDS bf16x8*)(ks + (k_rd ^ (s << 5)) + kb * 32 * 2 * D);
                sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[s], sc[kb], 0, 0, 0);
            }
        if (!(j0 + KEYS - 1 <= w_lo && (a.window == 0 || j0 > w_hi - a.window))) {     // uniform: some hidden
            asm volatile("");                          // a branch, not selects in every tile
            const int rel = pos - j0 - 4 * half;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if ((uint32_t)(rel - (kb * 32 + 8 * (i >> 2) + (i & 3))) >= span) sc[kb][i] = -INFINITY;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][i]);
        mx = halves_max(mx) * a.qk_scale;
        if (__ballot(mx > m + kRaise) != 0) {
            const float mn = fmaxf(m, mx), alpha = exp2_fast(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[nb][i] *= alpha;
        }
        bf16x8 pf[2 * KB];
#pragma unroll
        for (int s = 0; s < 2 * KB; ++s) {
            float p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = exp2_fast(fmaf(sc[s >> 1][8 * (s & 1) + i], a.qk_scale, -m));
                l += p[i];
            }
            const u32x4 u = {pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]), pack_bf16(p[4], p[5]), pack_bf16(p[6], p[7])};
            pf[s] = __builtin_bit_cast(bf16x8, u);
        }
#pragma unroll
        for (int s = 0; s < 2 * KB; ++s)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                union {
                    s16x4 q[2];
                    bf16x8 v;
                } u;
                u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EXKV_LDS s16x4*)(vs + v_rd[nb] + (16 * s) * 2 * D));
                u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((EXKV_LDS s16x4*)(vs + v_rd[nb] + (16 * s + 8) * 2 * D));
                o[nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u.v, pf[s], o[nb], 0, 0, 0);
            }
    };

    if (first <= last) load_tile(first, 0);
    for (int it = first; it <= last; ++it) {
        const int stage = (it - first) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                  // tile `it` is whole, and every wavefront is done with the one before
        asm volatile("" ::: "memory");
        if (it < last) load_tile(it + 1, stage ^ 1);
        tile_step(it, stage);
    }

    if (!wave_on) return;
    l = halves_sum(l);
    const bool live = wrow0 + col < nrows, seen = pos >= 0;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    float finite = 0.f;                                // NaN once a value is not finite
    uint16_t* op = a.out + ((int64_t)(tile.q0 + tok) * a.Hq + hq) * D + 4 * half;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = o[nb][i + j] * inv;
                finite = fmaf(x[j], 0.f, finite);
            }
            if (live) *reinterpret_cast<uint2*>(op + 32 * nb + 2 * i) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        }
    const uint64_t again = __ballot(live && seen && (finite != finite || !(l > 0.f && l < INFINITY)));
    if (again != 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // these rows' stores come first
        careful_rows<D>(a, tile, wrow0, hk, (uint32_t)again | (uint32_t)(again >> 32));
    }
}

template <int D, int NW, int KEYS, int WPE>
static void launch_prompt(const PromptArgs& a, hipStream_t stream) {
    // every sequence's last tile may be partial, and one more for rows behind the last sequence
    const int64_t tiles = (int64_t)a.N * a.G / (32 * NW) + a.S + 1;
    hipLaunchKernelGGL((prompt_kernel<D, NW, KEYS, WPE>), dim3((unsigned)(tiles * a.Hkv)), dim3(64 * NW), 0, stream, a, (int)tiles);
}

hipError_t fetch_errors_prompt(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

}  // namespace exkv

using namespace exkv;

static bool rows_ok(const void* p, int64_t s_t, int64_t s_h) {
    return (uintptr_t)p % 16 == 0 && s_t % 8 == 0 && s_h % 8 == 0 && s_t >= 0 && s_h >= 0;
}

extern "C" int exkv_prompt_attention(const void* q, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t, int64_t sk_h,
                                     const void* v, int64_t sv_t, int64_t sv_h, void* out, const int32_t* cu_q,
                                     const int32_t* cu_k, int32_t S, int32_t N, int32_t NK, int32_t Hq, int32_t Hkv,
                                     int32_t D, int32_t window, int32_t zero_tail, float qk_scale, hipStream_t stream) {
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
    EXKV_REQUIRE(((int64_t)N + 1) * G < INT32_MAX - 1024 &&
                     ((int64_t)N * G / 128 + S + 1) * Hkv * 512 <= (int64_t)UINT32_MAX,
                 "prompt_attention: too many rows (N=%d, %d heads per KV head, %d KV heads, S=%d)", N, (int)G, Hkv, S);
    const PromptArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)out, sq_t, sq_h, sk_t, sk_h,
                       sv_t, sv_h, cu_q, cu_k, S, N, NK, Hq, Hkv, (int)G, window, zero_tail, qk_scale};
    if (D == 64)
        launch_prompt<64, 4, 64, 4>(a, stream);
    else if (D == 128)
        launch_prompt<128, 4, 64, 2>(a, stream);
    else
        launch_prompt<256, 4, 32, 2>(a, stream);
    return hip_status(hipGetLastError(), "prompt_attention");
}
