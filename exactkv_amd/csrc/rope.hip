// The rotation of a packed prompt's queries and keys (rope.hpp), for prompt attention and the
// caches' prefill. No kernel of the reference (its model's own modules rotate, engine.py:42-49).
//
// Bound by HBM: a row is read and written once (8K tokens, 32q/8kv, head dim 128: 27.7 us, 6.1 TB/s;
// 97 tokens 3.0). D / 16 lanes take one row and its table row, which the caches hold for a token's
// other heads; lanes that walk four heads with one table row in registers take 28.3 and 4.2 us.
#include "rope.hpp"
#include "../../include/exactkv.h"

namespace exkv {

struct RotateArgs {
    RopeRows r;                        // v unused; n rows in all
    uint16_t* k_out;                   // [n, Hkv, D]
    const int32_t* cu;                 // [S + 1]
    const int32_t* start;              // [S] first positions, or nullptr: 0
    int S;
};

// The sequence that holds row t, by bisection: the last s with cu[s] <= t; S where t is behind
// the last one. Offsets that do not ascend are reported by the rows that meet them.
__device__ inline int sequence_at(const int32_t* cu, int S, int t) {
    if (S == 0 || t >= cu[S]) return S;
    int lo = 0, hi = S - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int D, bool V16>
__global__ void __launch_bounds__(256) rotate_kernel(RotateArgs a) {
    constexpr int GL = D / 16;
    const int g = threadIdx.x % GL;
    const int64_t row = (int64_t)blockIdx.x * (256 / GL) + threadIdx.x / GL;
    const int heads = a.r.Hq + a.r.Hkv, t = (int)(row / heads), h = (int)(row % heads);
    if (t >= a.r.n) return;
    const int s = sequence_at(a.cu, a.S, t);
    const bool isq = h < a.r.Hq;
    uint32_t u[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (s < a.S) {
        const int first = a.cu[s];
        if (first < 0 || first > t || a.cu[s + 1] <= t || a.cu[0] != 0) report_error(kErrOffsets);
        load_row16<D, V16>(isq ? a.r.q + t * a.r.sq_n + h * a.r.sq_h : a.r.k + t * a.r.sk_n + (h - a.r.Hq) * a.r.sk_h, g, u);
        float c[8], sn[8];
        const int64_t at = (int64_t)table_row(a.r.t, t - first + (a.start ? a.start[s] : 0)) * (D / 2) + 8 * g;
        load_angles(a.r.t.cos + at, c);
        load_angles(a.r.t.sin + at, sn);
        turn_row<D>(u, isq ? a.r.q_norm : a.r.k_norm, a.r.eps, c, sn, g);
    }
    store_row16<D>(isq ? a.r.q_out + ((int64_t)t * a.r.Hq + h) * D : a.k_out + ((int64_t)t * a.r.Hkv + h - a.r.Hq) * D, g, u);
}

template <int D>
static void launch_rotate(const RotateArgs& a, bool v16, hipStream_t stream) {
    const int64_t per = 256 / (D / 16), blocks = ((int64_t)a.r.n * (a.r.Hq + a.r.Hkv) + per - 1) / per;
    if (v16)
        hipLaunchKernelGGL((rotate_kernel<D, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((rotate_kernel<D, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

hipError_t fetch_errors_rope(uint32_t* out, int first, int clear, hipStream_t stream) {
    return fetch_file_errors(out, first, clear, stream);
}

}  // namespace exkv

using namespace exkv;

static bool row_align(const void* p, int64_t s_n, int64_t s_h, int bytes) {
    return ((uintptr_t)p | (uintptr_t)(2 * s_n) | (uintptr_t)(2 * s_h)) % bytes == 0;
}

extern "C" int exkv_rotate_prompt(const void* q, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_t, int64_t sk_h,
                                  const float* cos, const float* sin, int32_t table_rows, const void* q_norm,
                                  const void* k_norm, float eps, void* q_out, void* k_out, const int32_t* cu,
                                  const int32_t* start, int32_t S, int32_t N, int32_t Hq, int32_t Hkv, int32_t D,
                                  hipStream_t stream) {
    EXKV_REQUIRE(head_dim_ok(D), "rotate_prompt: head dim must be 64, 128 or 256 (got %d)", D);
    EXKV_REQUIRE(S >= 0 && N >= 0 && Hq > 0 && Hkv > 0 && table_rows > 0,
                 "rotate_prompt: bad shape S=%d N=%d Hq=%d Hkv=%d table rows=%d", S, N, Hq, Hkv, table_rows);
    if (N == 0) return EXKV_OK;
    EXKV_REQUIRE(q && k && cos && sin && q_out && k_out && cu, "rotate_prompt: null pointer");
    EXKV_REQUIRE(row_align(q, sq_t, sq_h, 4) && row_align(k, sk_t, sk_h, 4),
                 "rotate_prompt: rows must start at even elements (4-byte aligned)");
    EXKV_REQUIRE(((uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_norm |
                  (uintptr_t)k_norm) % 16 == 0, "rotate_prompt: tables, norms and outputs must be 16-byte aligned");
    EXKV_REQUIRE(((int64_t)N * ((int64_t)Hq + Hkv) * (D / 16) + 255) / 256 <= UINT32_MAX / 256, "rotate_prompt: too many rows (N=%d)", N);
    const RotateArgs a{{(const uint16_t*)q, (const uint16_t*)k, nullptr, sq_t, sq_h, sk_t, sk_h, 0, 0, {cos, sin, table_rows},
                        (const uint16_t*)q_norm, (const uint16_t*)k_norm, eps, (uint16_t*)q_out, N, Hq, Hkv},
                       (uint16_t*)k_out, cu, start, S};
    const bool v16 = row_align(q, sq_t, sq_h, 16) && row_align(k, sk_t, sk_h, 16);
    if (D == 64)
        launch_rotate<64>(a, v16, stream);
    else if (D == 128)
        launch_rotate<128>(a, v16, stream);
    else
        launch_rotate<256>(a, v16, stream);
    return hip_status(hipGetLastError(), "rotate_prompt");
}
