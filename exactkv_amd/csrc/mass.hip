// The attention that cached tokens receive, for gfx950 (no counterpart in the reference): for one new query token of
// each sequence and KV head h, over its visible keys j,
//     out[b, h, j] = mass[b, h, j] + sum over the query heads g of h of softmax_j(q[b, g] . k[b, j, h] / sqrt(D)).
//
// Two launches. The first reads the keys once: a wavefront takes one KV head and a run of 16-token pages, rebuilds a page
// in registers in the A layout of v_mfma_f32_16x16x32_bf16 (tokens as rows, the head's query heads as columns), writes the
// scores (fp32, log2 units) to a workspace and keeps each column's running maximum and sum. The second joins the runs'
// maxima and sums and adds up the weights token by token. Scores go through memory because a weight needs its row's sum:
// 4 bytes a query head and key, of which the keys' own bytes are 1.5 D a KV head (4 heads of 128: 16 to 192).
//
// Bound by the keys' bytes where there are many (8 sequences of 8,192 compressed tokens, 8 KV heads: 105 MB of keys in
// 24 us, 4.4 TB/s, and 5.4 us for the join; 61 of up to 4,339 in pages, 4 KV heads: 144 MB in 34 us, 4.2 TB/s, and 8.5), by the
// host's 12 us a call where there are few (one of 997 tokens: 4.0 and 4.2 us).
#include "errors.hpp"
#include "tile.hpp"
#include "../../include/exactkv.h"

namespace exkv {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLowest = -3.402823466e38f;   // a running maximum before any key, in log2 units

struct MassArgs {
    const uint16_t* q;                 // [B, Hq, D]
    CSrc k;
    const uint16_t* kb;                // bf16 [B, TS, Hkv, D], or pages of it
    const int32_t* table;              // as in decode attention; nullptr: contiguous
    int64_t table_stride, pool_pages;
    const int32_t* lens;
    int64_t lens_stride;
    int B, Hq, Hkv, G, T, TS, window, runs;
    float qk_scale;                    // log2(e) / sqrt(D)
    float* score;                      // [B * Hq, tsw]
    int64_t tsw;                       // T (with lens TS, as a sequence may have so many) rounded up to 16
    float2* part;                      // [B * Hq, runs]: maximum, sum
    const float* mass;                 // [B, Hkv, TS], or nullptr
    float* out;
    int fresh;                         // out's entries behind a sequence's tokens are written too (0)
};

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline int tokens_of(const MassArgs& a, int b) {
    return min(max(a.lens != nullptr ? a.lens[b * a.lens_stride] : a.T, 0), a.TS);
}

// A page's rows as loaded, before they are rebuilt.
template <int D, bool COMPRESSED>
struct PageIn;
template <int D>
struct PageIn<D, true> {
    PageBytesD<D> bytes;
    uint32_t mask;
    int32_t off;
};
template <int D>
struct PageIn<D, false> {
    uint32_t x[Run<D>::V];
};

template <int D, bool COMPRESSED>
__global__ void __launch_bounds__(256) mass_score_kernel(MassArgs a) {
    constexpr int R = Run<D>::R, KB = D / 32;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int groups = (a.G + 15) / 16;
    int64_t id = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int h = (int)(id % a.Hkv);
    id /= a.Hkv;
    const int run = (int)(id % a.runs);
    id /= a.runs;
    const int group = (int)(id % groups);
    const int64_t b = id / groups;
    if (b >= a.B) return;
    const int n = tokens_of(a, (int)b), low = a.window > 0 ? max(0, n - a.window) : 0;
    const int col = group * 16 + r, hq = h * a.G + col;
    const bool real = col < a.G;
    const int p0 = low / kPage, pages = (n + kPage - 1) / kPage - p0, per = (pages + a.runs - 1) / a.runs;
    const int first = p0 + run * per, last = min(first + per, p0 + pages);
    bf16x8 qf[KB];
#pragma unroll
    for (int s = 0; s < KB; ++s) {
        const int ch = 8 * s < R ? g * R + 8 * s : D / 2 + g * R + 8 * s - R;
        const uint4 x = real ? ld16(a.q + (b * a.Hq + hq) * D + ch) : make_uint4(0, 0, 0, 0);
        qf[s] = __builtin_bit_cast(bf16x8, x);
    }
    // the run's pool pages, a lane each, 64 at a time: read one by one, each would hold up its page's loads
    int pool = 0;
    auto table = [&](int p) {
        if (a.table != nullptr) pool = a.table[b * a.table_stride + min(p + lane, last - 1)];
    };
    auto load = [&](int p, PageIn<D, COMPRESSED>& in) {
        int64_t page = p;
        if (a.table != nullptr) {                      // uniform
            if (p > first && (p - first) % 64 == 0) table(p);
            page = min(max((int64_t)__builtin_amdgcn_readlane(pool, (p - first) % 64), (int64_t)0), a.pool_pages - 1);
        }
        if constexpr (COMPRESSED) {
            if (a.table == nullptr) page += b * (a.TS / kPage);
            const int64_t unit = page * a.Hkv + h;
            load_page_d<D>(a.k, (page * kPage + r) * a.Hkv + h, unit, g, in.bytes);
            in.mask = (uint32_t)a.k.rowmask[unit];
            in.off = a.k.rowoff[unit];
        } else {                                       // (a contiguous cache's rows may end inside a page)
            const int64_t row = a.table == nullptr ? b * a.TS + min(p * kPage + r, n - 1) : page * kPage + r;
            load_row_values_d<D>(a.kb + (row * a.Hkv + h) * D, g, in.x);
        }
    };
    float m = kLowest, l = 0.f;
    PageIn<D, COMPRESSED> in;
    if (first < last) {
        table(first);
        load(first, in);
    }
    for (int p = first; p < last; ++p) {
        uint32_t x[Run<D>::V];
        if constexpr (COMPRESSED)
            rebuild_page_d<D>(a.k, in.bytes, in.mask, in.off, r, g, x);
        else
#pragma unroll
            for (int i = 0; i < Run<D>::V; ++i) x[i] = in.x[i];
        if (p + 1 < last) load(p + 1, in);
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            const u32x4 u = {x[4 * kb], x[4 * kb + 1], x[4 * kb + 2], x[4 * kb + 3]};
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u), qf[kb], s, 0, 0, 0);
        }
        const int j = p * kPage + 4 * g;               // the lane's four tokens
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] *= a.qk_scale;
            if (j + i >= n || j + i < low) s[i] = -INFINITY;
        }
        const float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        if (mx > m) {
            l *= exp2_fast(m - mx);
            m = mx;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) l += exp2_fast(s[i] - m);
        if (real) *reinterpret_cast<f32x4*>(a.score + (b * a.Hq + hq) * a.tsw + j) = s;
    }
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) {
        const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d), M = fmaxf(m, m2);
        l = l * exp2_fast(m - M) + l2 * exp2_fast(m2 - M);
        m = M;
    }
    if (g == 0 && real) a.part[(b * a.Hq + hq) * a.runs + run] = make_float2(m, l);
}

// One workgroup: 1,024 tokens of one sequence and KV head, four neighbouring ones a thread.
__global__ void __launch_bounds__(256) mass_join_kernel(MassArgs a, int tiles) {
    extern __shared__ float2 s_head[];                 // [G]: each query head's maximum, 1 / sum (apart, as far scores need it)
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t unit = blockIdx.x / (unsigned)tiles, b = unit / a.Hkv;
    const int h = (int)(unit % a.Hkv), tile = (int)(blockIdx.x % (unsigned)tiles);
    const int n = tokens_of(a, (int)b), low = a.window > 0 ? max(0, n - a.window) : 0;
    const int j = (tile * 256 + (int)threadIdx.x) * 4;
    if (tile * 1024 >= n && a.fresh == 0) return;
    const int64_t head = b * a.Hq + h * a.G;
    // scores and masses are on their way while the sums are joined
    constexpr int FIRST = 8;
    const bool some = j < n && j + 3 >= low;
    const int64_t at = unit * a.TS;
    f32x4 score[FIRST];
    float before[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < FIRST; ++g)
        if (some && g < a.G) score[g] = *reinterpret_cast<const f32x4*>(a.score + (head + g) * a.tsw + j);
    if (a.mass != nullptr)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (j + i < n) before[i] = a.mass[at + j + i];
    for (int g = w; g < a.G; g += 4) {
        const float2* part = a.part + (head + g) * a.runs;
        float m = kLowest, l = 0.f;
        for (int i = lane; i < a.runs; i += 64) {
            const float2 x = part[i];
            const float M = fmaxf(m, x.x);
            l = l * exp2_fast(m - M) + x.y * exp2_fast(x.x - M);
            m = M;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d), M = fmaxf(m, m2);
            l = l * exp2_fast(m - M) + l2 * exp2_fast(m2 - M);
            m = M;
        }
        if (lane == 0) s_head[g] = make_float2(m, 1.f / l);
    }
    __syncthreads();
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    if (some) {
#pragma unroll
        for (int g = 0; g < FIRST; ++g)
            if (g < a.G)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[i] = fmaf(exp2_fast(score[g][i] - s_head[g].x), s_head[g].y, sum[i]);
        for (int g = FIRST; g < a.G; ++g) {
            const f32x4 s = *reinterpret_cast<const f32x4*>(a.score + (head + g) * a.tsw + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = fmaf(exp2_fast(s[i] - s_head[g].x), s_head[g].y, sum[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (j + i >= (a.fresh != 0 ? a.TS : n)) break;
        const bool seen = j + i >= low && j + i < n;
        a.out[at + j + i] = seen ? before[i] + sum[i] : before[i];
    }
}

hipError_t fetch_errors_mass(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

// Runs of pages that each (sequence, KV head) is cut into: about 8,192 wavefronts in all (new data each call, 4,096 / 6,144 /
// 8,192 / 12,288: 8 x 8192 34.9 / 39.0 / 33.8 / 35.5 us, 61 x 4339 over a pool 57.3 / 56.3 / 53.3 / 51.4).
static int mass_runs(int64_t B, int64_t Hq, int64_t Hkv, int64_t reach) {
    const int64_t G = Hq / Hkv, units = B * Hkv * ((G + 15) / 16), pages = (reach + kPage - 1) / kPage;
    int64_t runs = 8192 / units;
    if (runs > 256) runs = 256;
    if (runs > pages) runs = pages;
    return runs < 1 ? 1 : (int)runs;
}
static int64_t score_row(int64_t T) { return (T + kPage - 1) / kPage * kPage; }
static int64_t reach_of(int64_t T, int64_t window) { return window > 0 && window + kPage - 1 < T ? window + kPage - 1 : T; }

template <bool COMPRESSED>
static int launch_mass(MassArgs a, int32_t D, void* ws, int64_t ws_bytes, hipStream_t stream) {
    EXKV_REQUIRE(head_dim_ok(D), "attention_mass: head dim must be 64, 128 or 256 (got %d)", D);
    EXKV_REQUIRE(a.Hkv > 0 && a.Hq > 0 && a.Hq % a.Hkv == 0, "attention_mass: %d query heads over %d KV heads", a.Hq, a.Hkv);
    EXKV_REQUIRE(a.B >= 0 && a.TS >= 0 && a.T >= 0 && a.T <= a.TS && a.window >= 0, "attention_mass: bad shape B=%d TS=%d T=%d window=%d",
                 a.B, a.TS, a.T, a.window);
    EXKV_REQUIRE(a.lens_stride >= 0, "attention_mass: negative stride");
    if (a.B == 0 || a.TS == 0) return EXKV_OK;
    EXKV_REQUIRE(a.q && a.out && ws, "attention_mass: null pointer");
    EXKV_REQUIRE(a.table == nullptr || (a.pool_pages > 0 && a.table_stride >= (a.TS + kPage - 1) / kPage), "attention_mass: bad page table");
    EXKV_REQUIRE((COMPRESSED || a.table) ? a.TS % kPage == 0 : true, "attention_mass: TS=%d is no multiple of %d", a.TS, kPage);
    EXKV_REQUIRE(a.TS <= (1 << 30) && a.Hq <= 8192, "attention_mass: TS=%d, %d query heads", a.TS, a.Hq);
    a.G = a.Hq / a.Hkv;
    const int64_t reach = reach_of(a.lens != nullptr ? a.TS : a.T, a.window), rows = (int64_t)a.B * a.Hq;
    a.runs = mass_runs(a.B, a.Hq, a.Hkv, reach);
    a.tsw = score_row(a.lens != nullptr ? a.TS : a.T);
    const int64_t need = rows * (a.tsw * 4 + a.runs * 8);
    EXKV_REQUIRE((uintptr_t)ws % 16 == 0 && ws_bytes >= need, "attention_mass: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
                 (long long)need);
    a.score = (float*)ws;
    a.part = (float2*)(a.score + rows * a.tsw);
    const int64_t waves = (int64_t)a.B * a.Hkv * ((a.G + 15) / 16) * a.runs, blocks = (waves + 3) / 4;
    const int64_t most = a.fresh != 0 || a.lens != nullptr ? a.TS : a.T, tiles = (most + 1023) / 1024;
    EXKV_REQUIRE(blocks * 256 <= (int64_t)UINT32_MAX && tiles * a.B * a.Hkv * 256 <= (int64_t)UINT32_MAX,
                 "attention_mass: too many workgroups (B=%d, %d KV heads, TS=%d)", a.B, a.Hkv, a.TS);
    const dim3 grid((unsigned)blocks), block(256);
    if (D == 64)
        hipLaunchKernelGGL((mass_score_kernel<64, COMPRESSED>), grid, block, 0, stream, a);
    else if (D == 128)
        hipLaunchKernelGGL((mass_score_kernel<128, COMPRESSED>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((mass_score_kernel<256, COMPRESSED>), grid, block, 0, stream, a);
    if (tiles > 0) hipLaunchKernelGGL(mass_join_kernel, dim3((unsigned)(tiles * a.B * a.Hkv)), block, a.G * 8, stream, a, (int)tiles);
    return hip_status(hipGetLastError(), "attention_mass");
}

}  // namespace exkv

using namespace exkv;

extern "C" int64_t exkv_mass_workspace(int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t TS, int32_t has_lens, int32_t window) {
    if (B <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || TS < 0 || T < 0 || window < 0) return 0;
    const int64_t most = has_lens != 0 ? TS : T;
    return (int64_t)B * Hq * (score_row(most) * 4 + mass_runs(B, Hq, Hkv, reach_of(most, window)) * 8);
}

extern "C" int exkv_attention_mass(const void* q, const void* sm, const void* code, const void* base, const int32_t* rowmask,
                                   const int32_t* rowoff, const void* raw, int64_t raw_rows, const int32_t* block_table,
                                   int64_t table_stride, int64_t pool_pages, int32_t B, int32_t Hq, int32_t Hkv, int32_t D,
                                   int32_t T, int32_t TS, const int32_t* lens, int64_t lens_stride, int32_t window, float qk_scale,
                                   const float* mass, float* out, int32_t fresh, void* ws, int64_t ws_bytes, hipStream_t stream) {
    EXKV_REQUIRE(B <= 0 || TS <= 0 || (sm && code && base && rowmask && rowoff && raw && raw_rows > 0), "attention_mass: null pointer");
    MassArgs a{};
    a.q = (const uint16_t*)q;
    a.k = CSrc{(const uint8_t*)sm, (const uint8_t*)code, (const uint8_t*)base, rowmask, rowoff, (const uint16_t*)raw, raw_rows};
    a.table = block_table;
    a.table_stride = table_stride;
    a.pool_pages = pool_pages;
    a.lens = lens;
    a.lens_stride = lens_stride;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.T = T;
    a.TS = TS;
    a.window = window;
    a.qk_scale = qk_scale;
    a.mass = mass;
    a.out = out;
    a.fresh = fresh;
    return launch_mass<true>(a, D, ws, ws_bytes, stream);
}

extern "C" int exkv_attention_mass_bf16(const void* q, const void* k, const int32_t* block_table, int64_t table_stride,
                                        int64_t pool_pages, int32_t B, int32_t Hq, int32_t Hkv, int32_t D, int32_t T, int32_t TS,
                                        const int32_t* lens, int64_t lens_stride, int32_t window, float qk_scale, const float* mass,
                                        float* out, int32_t fresh, void* ws, int64_t ws_bytes, hipStream_t stream) {
    EXKV_REQUIRE(B <= 0 || TS <= 0 || k, "attention_mass: null pointer");
    MassArgs a{};
    a.q = (const uint16_t*)q;
    a.kb = (const uint16_t*)k;
    a.table = block_table;
    a.table_stride = table_stride;
    a.pool_pages = pool_pages;
    a.lens = lens;
    a.lens_stride = lens_stride;
    a.B = B;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.T = T;
    a.TS = TS;
    a.window = window;
    a.qk_scale = qk_scale;
    a.mass = mass;
    a.out = out;
    a.fresh = fresh;
    return launch_mass<false>(a, D, ws, ws_bytes, stream);
}
