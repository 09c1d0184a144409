// Eviction from a cache by gathered attention weight, for gfx950 (no counterpart in the reference,
// whose caches keep every token): which tokens of each KV head a budget keeps, and their rows out of
// the cache.
//
// select: of the n tokens of a (sequence, KV head), `keep` stay: the first `sinks`, the last `recent`,
// and of those between the ones with the most mass, of equal ones the first. All of them where n <= keep.
// gather: out[b, i, h] = row index[b, h, i] of head h, zeros where the index is -1.
#include "errors.hpp"
#include "tile.hpp"
#include "../../include/exactkv.h"

namespace exkv {

// A value's place in the order of all: whole numbers that ascend with it; -0 as 0, NaN before all others.
__device__ inline uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0u : (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}

struct SelectArgs {
    const float* mass;                 // [B, H, TS], element strides s_b, s_h
    int64_t s_b, s_h;
    const int32_t* lens;               // tokens of sequence b: lens[b * lens_stride], or T
    int64_t lens_stride;
    int T, H, TS, keep, sinks, recent;
    int32_t* index;                    // [B, H, keep]
    float* kept;
};

constexpr int kBins = 2048, kNear = 512;

// One workgroup a row. A thread holds E neighbouring tokens, of longer rows (WHOLE false) one piece of
// 1024 E tokens after the other, read anew by every pass. The r-th largest is found by cutting the interval of the keys
// into 2,048 bins of one width, counting, and going on with the bin that holds it while that has more than 512 tokens;
// among these it is the one with r - 1 before it. Keys that are all equal go by index. The tokens that stay are then
// written in order by a scan. Bound by its steps, each a barrier or two: 64 rows of 8,192 tokens 9.6 us, 8 rows of 2,048 tokens 6.6 us.
template <int E, bool WHOLE>
__global__ void __launch_bounds__(1024) select_kernel(SelectArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint64_t near[kNear], s_border;
    __shared__ uint32_t s_lo, s_hi, s_need, s_in, s_near;
    const int tid = threadIdx.x, row = blockIdx.x, b = row / a.H, h = row % a.H;
    const float* mass = a.mass + b * a.s_b + h * a.s_h;
    int32_t* index = a.index + (int64_t)row * a.keep;
    float* kept = a.kept + (int64_t)row * a.keep;
    const int n = min(max(a.lens != nullptr ? a.lens[b * a.lens_stride] : a.T, 0), a.TS);
    if (n <= a.keep) {
        for (int j = tid; j < a.keep; j += 1024) {
            index[j] = j < n ? j : -1;
            kept[j] = j < n ? mass[j] : 0.f;
        }
        return;
    }
    constexpr int PIECE = 1024 * E;
    const int pieces = WHOLE ? 1 : (n + PIECE - 1) / PIECE;
    const int from = a.sinks, to = n - a.recent;       // those between; from <= to, as keep < n
    const bool aligned = ((uintptr_t)mass & 15) == 0;
    uint32_t key[E];
    float val[E];
    auto load = [&](int p) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const int j = p * PIECE + tid * E + i;
            float x[4];
            if (aligned && j + 4 <= n) {
                const float4 v = *reinterpret_cast<const float4*>(mass + j);
                x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] = j + c < n ? mass[j + c] : 0.f;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                val[i + c] = x[c];
                key[i + c] = order_of(x[c]);
            }
        }
    };
    auto between = [&](int p, int i) {
        const int j = p * PIECE + tid * E + i;
        return j >= from && j < to;
    };
    if (tid == 0) {
        s_lo = ~0u;
        s_hi = 0u;
    }
    __syncthreads();
    uint32_t lo = ~0u, hi = 0u;
    for (int p = 0; p < pieces; ++p) {
        load(p);
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (between(p, i)) {
                lo = min(lo, key[i]);
                hi = max(hi, key[i]);
            }
    }
    for (int d = 1; d < 64; d <<= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, d));
        hi = max(hi, (uint32_t)__shfl_xor((int)hi, d));
    }
    if ((tid & 63) == 0) {
        atomicMin(&s_lo, lo);
        atomicMax(&s_hi, hi);
    }
    __syncthreads();
    lo = s_lo;
    hi = s_hi;
    uint32_t need = (uint32_t)(a.keep - a.sinks - a.recent), ties = 0;
    // a token in the order of all: those up to `border` stay; where equal keys are many, those with keys above `level` and
    // the first `ties` at it
    auto place = [&](int p, int i) { return (uint64_t)~key[i] << 32 | (uint32_t)(p * PIECE + tid * E + i); };
    uint64_t border = 0;
    uint32_t level = 0;
    bool stop = need == 0;
    while (!stop) {                                    // uniform; each turn narrows hi - lo 1,024 times at least
        const uint32_t span = hi - lo;
        const int shift = span < (uint32_t)kBins ? 0 : 21 - __builtin_clz(span);
        hist[tid] = 0;
        hist[tid + 1024] = 0;
        if (tid == 0) s_near = 0;
        __syncthreads();
        for (int p = 0; p < pieces; ++p) {
            if (!WHOLE) load(p);
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (between(p, i) && key[i] >= lo && key[i] <= hi) atomicAdd(&hist[(key[i] - lo) >> shift], 1u);
        }
        __syncthreads();
        // from the last bin on
        const int c0 = (int)hist[kBins - 1 - 2 * tid], c1 = (int)hist[kBins - 2 - 2 * tid];
        int total;
        const int before = block_excl_scan(c0 + c1, total);
        if (before < (int)need && before + c0 + c1 >= (int)need) {
            const bool second = before + c0 < (int)need;
            const int bin = kBins - 1 - 2 * tid - second;
            s_lo = lo + ((uint32_t)bin << shift);
            s_hi = min(hi, s_lo + ((1u << shift) - 1u));
            s_need = need - (uint32_t)(second ? before + c0 : before);
            s_in = (uint32_t)(second ? c1 : c0);
        }
        __syncthreads();
        lo = s_lo;
        hi = s_hi;
        need = s_need;
        const uint32_t in = s_in;
        if (in == need) {                              // the whole bin
            border = (uint64_t)~lo << 32 | 0xFFFFFFFFu;
            stop = true;
        } else if (in <= (uint32_t)kNear) {
            for (int p = 0; p < pieces; ++p) {
                if (!WHOLE) load(p);
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (between(p, i) && key[i] >= lo && key[i] <= hi) near[atomicAdd(&s_near, 1u)] = place(p, i);
            }
            __syncthreads();
            if (tid < (int)in) {
                const uint64_t x = near[tid];
                uint32_t r = 0;
#pragma unroll 8
                for (uint32_t i = 0; i < in; ++i) r += near[i] < x;
                if (r == need - 1) s_border = x;
            }
            __syncthreads();
            border = s_border;
            stop = true;
        } else if (lo == hi) {                         // equal keys
            level = lo;
            ties = need;
            stop = true;
        }
        __syncthreads();
    }
    int done = 0, tied = 0;
    for (int p = 0; p < pieces; ++p) {
        if (!WHOLE) load(p);
        uint32_t stays = 0, equal = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int j = p * PIECE + tid * E + i;
            if (j >= n) continue;
            if (j < from || j >= to || (ties > 0 ? key[i] > level : a.keep > a.sinks + a.recent && place(p, i) <= border))
                stays |= 1u << i;
            else if (ties > 0 && key[i] == level)
                equal |= 1u << i;
        }
        if (ties > 0) {
            int total, at = tied + block_excl_scan(__builtin_popcount(equal), total);
            tied += total;
#pragma unroll
            for (int i = 0; i < E; ++i)
                if ((equal >> i) & 1u) stays |= (uint32_t)(at++ < (int)ties) << i;
        }
        int total, at = done + block_excl_scan(__builtin_popcount(stays), total);
        done += total;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (((stays >> i) & 1u) && at < a.keep) {
                index[at] = p * PIECE + tid * E + i;
                kept[at++] = val[i];
            }
    }
}

struct GatherArgs {
    CSrc k, v;                         // compressed: pages of H heads
    const uint16_t *kb, *vb;           // bf16 [B, TS, H, D]
    const int32_t* table;              // pool page of sequence b's page p: table[b * table_stride + p]; nullptr: contiguous
    int64_t table_stride;
    int64_t pool_pages;
    int H, TS, keep;
    int64_t rows;                      // B * H * keep
    const int32_t* index;              // [B, H, keep]
    uint16_t *ko, *vo;                 // [B, keep, H, D]
};

// One head row: D / 16 lanes, lane c with channels 8 c .. and D / 2 + 8 c .., whose codes share eight bytes.
template <int D>
__device__ inline void gather_row(const CSrc& s, int64_t row, int64_t unit, int r, int c, uint4& lo, uint4& hi) {
    const uint2 slo = *reinterpret_cast<const uint2*>(s.sm + row * D + 8 * c);
    const uint2 shi = *reinterpret_cast<const uint2*>(s.sm + row * D + D / 2 + 8 * c);
    const uint2 code = *reinterpret_cast<const uint2*>(s.code + row * (D / 2) + 8 * c);
    const uint2 blo = *reinterpret_cast<const uint2*>(s.base + unit * D + 8 * c);
    const uint2 bhi = *reinterpret_cast<const uint2*>(s.base + unit * D + D / 2 + 8 * c);
    const uint32_t mask = (uint32_t)s.rowmask[unit];
    rebuild4<true>(slo.x, code.x & 0x0F0F0F0Fu, blo.x, lo.x, lo.y);
    rebuild4<true>(slo.y, code.y & 0x0F0F0F0Fu, blo.y, lo.z, lo.w);
    rebuild4<true>(shi.x, (code.x >> 4) & 0x0F0F0F0Fu, bhi.x, hi.x, hi.y);
    rebuild4<true>(shi.y, (code.y >> 4) & 0x0F0F0F0Fu, bhi.y, hi.z, hi.w);
    if ((mask >> r) & 1u) {
        const uint16_t* raw = s.raw + raw_slot(mask, s.rowoff[unit], r, s.raw_rows) * D;
        lo = ld16(raw + 8 * c);
        hi = ld16(raw + D / 2 + 8 * c);
    }
}

// A head row of both caches by D / 16 lanes, 16 bytes of each half at a time. Bound by memory: rows of one head lie H rows
// apart, so a compressed one is read in pieces of 64 and 128 bytes. 64 heads' 2,048 rows of 8,192 tokens, head dim 128
// (keys and values, compressed): 122 MB read and written in 22.8 us, 5.3 TB/s, what a copy reaches.
template <int D, bool COMPRESSED>
__global__ void __launch_bounds__(256) gather_kernel(GatherArgs a) {
    constexpr int L = D / 16, ROWS = 256 / L;
    const int64_t at = (int64_t)blockIdx.x * ROWS + threadIdx.x / L;
    const int c = threadIdx.x % L;
    if (at >= a.rows) return;
    const int i = (int)(at % a.keep);
    const int64_t unit = at / a.keep, b = unit / a.H;
    const int h = (int)(unit % a.H);
    const int j = a.index[at];
    uint4 klo = make_uint4(0, 0, 0, 0), khi = klo, vlo = klo, vhi = klo;
    if (j >= 0 && j < a.TS) {
        int64_t page = j / kPage;
        if (a.table != nullptr)
            page = min(max((int64_t)a.table[b * a.table_stride + page], (int64_t)0), a.pool_pages - 1);
        else
            page += b * (a.TS / kPage);
        const int r = j % kPage;
        const int64_t row = a.table == nullptr && !COMPRESSED ? (b * a.TS + j) * a.H + h : (page * kPage + r) * a.H + h;
        if constexpr (COMPRESSED) {
            gather_row<D>(a.k, row, page * a.H + h, r, c, klo, khi);
            gather_row<D>(a.v, row, page * a.H + h, r, c, vlo, vhi);
        } else {
            klo = ld16(a.kb + row * D + 8 * c);
            khi = ld16(a.kb + row * D + D / 2 + 8 * c);
            vlo = ld16(a.vb + row * D + 8 * c);
            vhi = ld16(a.vb + row * D + D / 2 + 8 * c);
        }
    } else if (j != -1) {
        report_error(kErrIndex);
    }
    const int64_t out = ((b * a.keep + i) * a.H + h) * D;
    *reinterpret_cast<uint4*>(a.ko + out + 8 * c) = klo;
    *reinterpret_cast<uint4*>(a.ko + out + D / 2 + 8 * c) = khi;
    *reinterpret_cast<uint4*>(a.vo + out + 8 * c) = vlo;
    *reinterpret_cast<uint4*>(a.vo + out + D / 2 + 8 * c) = vhi;
}

hipError_t fetch_errors_evict(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

template <bool COMPRESSED>
static void launch_gather(const GatherArgs& a, int D, hipStream_t stream) {
    const unsigned blocks = (unsigned)((a.rows * (D / 16) + 255) / 256);
    if (D == 64)
        hipLaunchKernelGGL((gather_kernel<64, COMPRESSED>), dim3(blocks), dim3(256), 0, stream, a);
    else if (D == 128)
        hipLaunchKernelGGL((gather_kernel<128, COMPRESSED>), dim3(blocks), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((gather_kernel<256, COMPRESSED>), dim3(blocks), dim3(256), 0, stream, a);
}

static int gather_check(const GatherArgs& a, int32_t B, int32_t D) {
    EXKV_REQUIRE(head_dim_ok(D), "gather_tokens: head dim must be 64, 128 or 256 (got %d)", D);
    EXKV_REQUIRE(B >= 0 && a.H > 0 && a.TS >= 0 && a.keep >= 0 && a.table_stride >= 0, "gather_tokens: bad shape B=%d H=%d TS=%d keep=%d",
                 B, a.H, a.TS, a.keep);
    EXKV_REQUIRE(a.table == nullptr || (a.pool_pages > 0 && a.table_stride >= a.TS / kPage), "gather_tokens: bad page table");
    EXKV_REQUIRE(a.rows == 0 || (a.index && a.ko && a.vo), "gather_tokens: null pointer");
    EXKV_REQUIRE((a.rows * (D / 16) + 255) / 256 * 256 <= (int64_t)UINT32_MAX, "gather_tokens: too many rows (%lld)",
                 (long long)a.rows);
    return EXKV_OK;
}

}  // namespace exkv

using namespace exkv;

extern "C" int exkv_select_tokens(const float* mass, int64_t s_b, int64_t s_h, const int32_t* lens, int64_t lens_stride,
                                  int32_t T, int32_t B, int32_t H, int32_t TS, int32_t keep, int32_t sinks, int32_t recent,
                                  int32_t* index, float* kept, hipStream_t stream) {
    EXKV_REQUIRE(B >= 0 && H > 0 && TS >= 0 && T >= 0 && T <= TS, "select_tokens: bad shape B=%d H=%d TS=%d T=%d", B, H, TS, T);
    EXKV_REQUIRE(keep >= 0 && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= keep,
                 "select_tokens: %d first and %d latest tokens of %d kept", sinks, recent, keep);
    EXKV_REQUIRE((int64_t)B * H * 1024 <= (int64_t)UINT32_MAX, "select_tokens: too many rows (B=%d, H=%d)", B, H);
    EXKV_REQUIRE(s_b >= 0 && s_h >= 0 && lens_stride >= 0, "select_tokens: negative stride");
    if (B == 0 || keep == 0) return EXKV_OK;
    EXKV_REQUIRE((mass || TS == 0) && index && kept, "select_tokens: null pointer");
    EXKV_REQUIRE(TS <= (1 << 30), "select_tokens: TS=%d", TS);
    const SelectArgs a{mass, s_b, s_h, lens, lens_stride, T, H, TS, keep, sinks, recent, index, kept};
    const dim3 grid((unsigned)(B * H)), block(1024);
    const int most = lens != nullptr ? TS : T;
    if (most <= 4096)
        hipLaunchKernelGGL((select_kernel<4, true>), grid, block, 0, stream, a);
    else if (most <= 8192)
        hipLaunchKernelGGL((select_kernel<8, true>), grid, block, 0, stream, a);
    else if (most <= 16384)
        hipLaunchKernelGGL((select_kernel<16, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((select_kernel<16, false>), grid, block, 0, stream, a);
    return hip_status(hipGetLastError(), "select_tokens");
}

extern "C" int exkv_gather_tokens(const void* k_sm, const void* k_code, const void* k_base, const int32_t* k_rowmask,
                                  const int32_t* k_rowoff, const void* k_raw, int64_t k_raw_rows, const void* v_sm,
                                  const void* v_code, const void* v_base, const int32_t* v_rowmask, const int32_t* v_rowoff,
                                  const void* v_raw, int64_t v_raw_rows, const int32_t* block_table, int64_t table_stride,
                                  int64_t pool_pages, int32_t B, int32_t H, int32_t TS, int32_t D, const int32_t* index,
                                  int32_t keep, void* k_out, void* v_out, hipStream_t stream) {
    GatherArgs a{};
    a.k = CSrc{(const uint8_t*)k_sm, (const uint8_t*)k_code, (const uint8_t*)k_base, k_rowmask, k_rowoff, (const uint16_t*)k_raw, k_raw_rows};
    a.v = CSrc{(const uint8_t*)v_sm, (const uint8_t*)v_code, (const uint8_t*)v_base, v_rowmask, v_rowoff, (const uint16_t*)v_raw, v_raw_rows};
    a.table = block_table;
    a.table_stride = table_stride;
    a.pool_pages = pool_pages;
    a.H = H;
    a.TS = TS;
    a.keep = keep;
    a.rows = (int64_t)B * H * keep;
    a.index = index;
    a.ko = (uint16_t*)k_out;
    a.vo = (uint16_t*)v_out;
    if (const int rc = gather_check(a, B, D)) return rc;
    if (a.rows == 0) return EXKV_OK;
    EXKV_REQUIRE(k_sm && k_code && k_base && k_rowmask && k_rowoff && k_raw && v_sm && v_code && v_base && v_rowmask && v_rowoff && v_raw,
                 "gather_tokens: null pointer");
    EXKV_REQUIRE(TS % kPage == 0 && k_raw_rows > 0 && v_raw_rows > 0, "gather_tokens: TS=%d, raw rows %lld and %lld", TS,
                 (long long)k_raw_rows, (long long)v_raw_rows);
    launch_gather<true>(a, D, stream);
    return hip_status(hipGetLastError(), "gather_tokens");
}

extern "C" int exkv_gather_tokens_bf16(const void* k, const void* v, const int32_t* block_table, int64_t table_stride,
                                       int64_t pool_pages, int32_t B, int32_t H, int32_t TS, int32_t D, const int32_t* index,
                                       int32_t keep, void* k_out, void* v_out, hipStream_t stream) {
    GatherArgs a{};
    a.kb = (const uint16_t*)k;
    a.vb = (const uint16_t*)v;
    a.table = block_table;
    a.table_stride = table_stride;
    a.pool_pages = pool_pages;
    a.H = H;
    a.TS = TS;
    a.keep = keep;
    a.rows = (int64_t)B * H * keep;
    a.index = index;
    a.ko = (uint16_t*)k_out;
    a.vo = (uint16_t*)v_out;
    if (const int rc = gather_check(a, B, D)) return rc;
    if (a.rows == 0) return EXKV_OK;
    EXKV_REQUIRE(k && v, "gather_tokens: null pointer");
    launch_gather<false>(a, D, stream);
    return hip_status(hipGetLastError(), "gather_tokens");
}
