// The residual stream between two blocks of a decoder layer, for gfx950: a block's output x
// (normed, gated, scaled, each where asked for) added to the stream r, and the norm that feeds the
// next block:
//     u = x                         or  x rsqrt(mean(x^2) + eps) post_w
//     u = u gate                    (where a gate is given)
//     h = r + scale u               (without r: scale u)
//     y = h rsqrt(mean(h^2) + eps) w.
// bf16 rows in and out, fp32 between; h and y are rounded once each (y from the unrounded h).
// No kernel of the reference (its model's own modules do this, engine.py:75-91).
//
// Bound by HBM: x, r and a row-wise gate are read once, h and y written once (8191 rows of 3584 with a
// norm behind the block and a gate as large: 56 us, 5.2 TB/s; 8191 of 4,096 with neither 40 us, 6.7 TB/s;
// 621 4.9; one 2.7, which is the launch and one round trip).
// One workgroup of 64 WAVES threads holds a row in registers, eight channels a thread and piece, CH
// pieces; the two sums go through the wavefront's lanes and, with several wavefronts, through LDS.
// Rows that do not lie at whole 16 bytes (V16 false) go by the same pieces wherever they lie, as the
// hardware allows, but for a partial last one: 8191 rows of 4,096 41 us (channel by channel 134), of
// 4,095 57.
#include "rope.hpp"
#include "../../include/exactkv.h"

namespace exkv {

struct NormArgs {
    const uint16_t *x, *r, *w, *post_w, *gate;     // r, post_w, gate may be nullptr
    int64_t sx, sr, sg;                            // row strides in elements (sg 0: one gate row for all)
    uint16_t *h, *y;                               // [N, C]; h may be nullptr
    float eps, scale;
    int N, C;
};

__device__ inline float wave_total(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    return x;
}
template <int WAVES>
__device__ inline float block_total(float x, float* s) {
    x = wave_total(x);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) x += s[i];
    }
    return x;
}

// Eight channels of a row from channel c0 on: one 16-byte piece, which need not lie at 16 bytes unless
// V16; then a row's last piece may be partial as well, and goes one by one, channels past C as zeros.
template <bool V16>
__device__ inline void load8(const uint16_t* row, int c0, int C, float (&v)[8]) {
    if (V16 || c0 + 8 <= C) {
        uint32_t u[4];
        if constexpr (V16)
            ld_words<4>(row + c0, u);
        else
            __builtin_memcpy(u, row + c0, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = lo_float(u[i]);
            v[2 * i + 1] = hi_float(u[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i < C ? lo_float(row[c0 + i]) : 0.f;
    }
}
template <bool V16>
__device__ inline void store8(uint16_t* row, int c0, int C, const float (&v)[8]) {
    if (V16 || c0 + 8 <= C) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
        if constexpr (V16)
            st_words<4>(row + c0, u);
        else
            __builtin_memcpy(row + c0, u, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < C) row[c0 + i] = (uint16_t)bf16_pair(v[i], 0.f);
    }
}

template <int WAVES, int CH, bool V16>
__global__ void __launch_bounds__(64 * WAVES) norm_kernel(NormArgs a) {
    __shared__ float s_sum[2][WAVES];
    const int64_t row = blockIdx.x;
    const uint16_t *x = a.x + row * a.sx, *r = a.r + row * a.sr, *gate = a.gate + row * a.sg;
    const float inv_c = 1.f / (float)a.C;
    float v[CH][8];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c0 = (i * 64 * WAVES + (int)threadIdx.x) * 8;
        if (c0 < a.C)
            load8<V16>(x, c0, a.C, v[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
    float k = a.scale;
    if (a.post_w != nullptr) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(v[i][j], v[i][j], sq);
        k *= rsqrtf(fmaf(block_total<WAVES>(sq, s_sum[0]), inv_c, a.eps));
        sq = 0.f;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c0 = (i * 64 * WAVES + (int)threadIdx.x) * 8;
        if (c0 < a.C) {
            float f[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= k;
            if (a.post_w != nullptr) {
                load8<V16>(a.post_w, c0, a.C, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] *= f[j];
            }
            if (a.gate != nullptr) {
                load8<V16>(gate, c0, a.C, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] *= f[j];
            }
            if (a.r != nullptr) {
                load8<V16>(r, c0, a.C, f);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] += f[j];
            }
            if (a.h != nullptr) store8<V16>(a.h + row * a.C, c0, a.C, v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) sq = fmaf(v[i][j], v[i][j], sq);
        }
    }
    const float rs = rsqrtf(fmaf(block_total<WAVES>(sq, s_sum[1]), inv_c, a.eps));
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c0 = (i * 64 * WAVES + (int)threadIdx.x) * 8;
        if (c0 < a.C) {
            float f[8];
            load8<V16>(a.w, c0, a.C, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= rs * f[j];
            store8<V16>(a.y + row * a.C, c0, a.C, v[i]);
        }
    }
}

// A grid holds fewer than 2^32 threads: as many rows a launch.
template <int WAVES, int CH>
static void launch_norm(NormArgs a, bool v16, hipStream_t stream) {
    constexpr int kMost = UINT32_MAX / (64 * WAVES);
    for (int left = a.N; left > 0; left -= kMost) {
        a.N = left < kMost ? left : kMost;
        if (v16)
            hipLaunchKernelGGL((norm_kernel<WAVES, CH, true>), dim3((unsigned)a.N), dim3(64 * WAVES), 0, stream, a);
        else
            hipLaunchKernelGGL((norm_kernel<WAVES, CH, false>), dim3((unsigned)a.N), dim3(64 * WAVES), 0, stream, a);
        a.x += a.N * a.sx;
        if (a.r) a.r += a.N * a.sr;
        if (a.gate) a.gate += a.N * a.sg;
        if (a.h) a.h += (int64_t)a.N * a.C;
        a.y += (int64_t)a.N * a.C;
    }
}

}  // namespace exkv

using namespace exkv;

extern "C" int exkv_add_norm(const void* x, int64_t sx, const void* r, int64_t sr, const void* w, const void* post_w,
                             const void* gate, int64_t sg, float scale, float eps, void* h, void* y, int32_t N, int32_t C,
                             hipStream_t stream) {
    EXKV_REQUIRE(N >= 0 && C > 0 && C <= 16384, "add_norm: 1 to 16384 channels (got %d, N=%d)", C, N);
    if (N == 0) return EXKV_OK;
    EXKV_REQUIRE(x && w && y, "add_norm: null pointer");
    EXKV_REQUIRE(sx >= 0 && sr >= 0 && sg >= 0, "add_norm: negative row stride");
    EXKV_REQUIRE(((uintptr_t)x | (uintptr_t)r | (uintptr_t)w | (uintptr_t)post_w | (uintptr_t)gate | (uintptr_t)h |
                  (uintptr_t)y) % 2 == 0, "add_norm: unaligned bf16 pointer");
    const NormArgs a{(const uint16_t*)x, (const uint16_t*)r, (const uint16_t*)w, (const uint16_t*)post_w,
                     (const uint16_t*)gate, sx, r ? sr : 0, gate ? sg : 0, (uint16_t*)h, (uint16_t*)y, eps, scale, N, C};
    const bool v16 = (((uintptr_t)x | (uintptr_t)r | (uintptr_t)w | (uintptr_t)post_w | (uintptr_t)gate | (uintptr_t)h |
                       (uintptr_t)y) % 16 == 0) && C % 8 == 0 && sx % 8 == 0 && a.sr % 8 == 0 && a.sg % 8 == 0;
    // one piece a thread while a workgroup's 1024 threads can hold the row so; us for 1, 621 and 8191
    // rows, this / half the wavefronts with two pieces: 1,024 channels 2.1, 2.7, 11.9 / 2.6, 3.3, 10.7;
    // 4,096 2.3, 4.6, 39.5 / 2.9, 5.0, 40.4; 8,192 2.6, 7.7, 91.0 / 3.1, 7.3, 94.7; 16,384 (two pieces
    // / four) 3.6, 14.3, 182 / 4.4, 13.9, 197
    if (C <= 512)
        launch_norm<1, 1>(a, v16, stream);
    else if (C <= 1024)
        launch_norm<2, 1>(a, v16, stream);
    else if (C <= 2048)
        launch_norm<4, 1>(a, v16, stream);
    else if (C <= 4096)
        launch_norm<8, 1>(a, v16, stream);
    else if (C <= 8192)
        launch_norm<16, 1>(a, v16, stream);
    else
        launch_norm<16, 2>(a, v16, stream);
    return hip_status(hipGetLastError(), "add_norm");
}
