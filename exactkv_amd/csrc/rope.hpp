// The rotation of query and key rows, shared by the prompt's kernel and the appends'.
//
// Half-split rotary embedding (the one of Llama and Qwen): with c_i, s_i the cosine and sine of
// channel pair i at the row's position (fp32 tables [positions, D / 2]),
//     y_i = x_i c_i - x_{i + D/2} s_i,    y_{i + D/2} = x_{i + D/2} c_i + x_i s_i,
// after x <- x w rsqrt(mean(x^2) + eps) where a norm's weights w are given (the per-head norms of
// Qwen3). All of it in fp32 from the bf16 row; the only rounding is the store's.
//
// D / 16 lanes hold a row, lane g the channels 8 g .. 8 g + 7 and D/2 + 8 g .. : both halves of
// its pairs, in two 16-byte loads.
#pragma once

#include "errors.hpp"
#include "tile.hpp"

namespace exkv {

struct RopeTables {
    const float *cos, *sin;            // [rows, D / 2]
    int rows;
};

// Rows of n tokens' heads, and where the rotated queries go.
struct RopeRows {
    const uint16_t *q, *k, *v;
    int64_t sq_n, sq_h, sk_n, sk_h, sv_n, sv_h;   // elements
    RopeTables t;
    const uint16_t *q_norm, *k_norm;   // [D] or nullptr
    float eps;
    uint16_t* q_out;                   // [n, Hq, D]
    int n, Hq, Hkv;
};

// A position within the tables; others are clamped and reported.
__device__ inline int table_row(const RopeTables& t, int pos) {
    const int p = min(max(pos, 0), t.rows - 1);
    if (p != pos) report_error(kErrPosition);
    return p;
}

__device__ inline float lo_float(uint32_t u) { return __uint_as_float(u << 16); }
__device__ inline float hi_float(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }
__device__ inline uint32_t bf16_pair(float a, float b) {
    const __bf16 lo = (__bf16)a, hi = (__bf16)b;
    return (uint32_t)__builtin_bit_cast(uint16_t, lo) | ((uint32_t)__builtin_bit_cast(uint16_t, hi) << 16);
}

// The lane's 16 values of a row: u[0..3] the low run, u[4..7] the high one. V16: rows of 16-byte
// pieces, else of 4-byte ones.
template <int D, bool V16>
__device__ inline void load_row16(const uint16_t* row, int g, uint32_t (&u)[8]) {
    const uint16_t *a = row + 8 * g, *b = a + D / 2;
    if constexpr (V16) {
        ld_words<4>(a, u);
        ld_words<4>(b, u + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = reinterpret_cast<const uint32_t*>(a)[i];
            u[4 + i] = reinterpret_cast<const uint32_t*>(b)[i];
        }
    }
}
template <int D>
__device__ inline void store_row16(uint16_t* row, int g, const uint32_t (&u)[8]) {
    st_words<4>(row + 8 * g, u);
    st_words<4>(row + D / 2 + 8 * g, u + 4);
}

// Eight fp32 values of a table row.
__device__ inline void load_angles(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// Sum over the D / 16 lanes of a row (all of them call it).
template <int D>
__device__ inline float row_sum(float x) {
#pragma unroll
    for (int d = 1; d < D / 16; d <<= 1) x += __shfl_xor(x, d);
    return x;
}

// The lane's values normed with w (may be nullptr; uniform) and rotated.
template <int D>
__device__ inline void turn_row(uint32_t (&u)[8], const uint16_t* w, float eps, const float (&c)[8], const float (&s)[8], int g) {
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[2 * i] = lo_float(u[i]);
        a[2 * i + 1] = hi_float(u[i]);
        b[2 * i] = lo_float(u[4 + i]);
        b[2 * i + 1] = hi_float(u[4 + i]);
    }
    if (w != nullptr) {
        uint32_t wu[8];
        load_row16<D, true>(w, g, wu);
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq = fmaf(a[i], a[i], fmaf(b[i], b[i], sq));
        const float r = rsqrtf(fmaf(row_sum<D>(sq), 1.f / D, eps));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[2 * i] *= r * lo_float(wu[i]);
            a[2 * i + 1] *= r * hi_float(wu[i]);
            b[2 * i] *= r * lo_float(wu[4 + i]);
            b[2 * i + 1] *= r * hi_float(wu[4 + i]);
        }
    }
    float y[8], z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = fmaf(a[i], c[i], -(b[i] * s[i]));
        z[i] = fmaf(b[i], c[i], a[i] * s[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u[i] = bf16_pair(y[2 * i], y[2 * i + 1]);
        u[4 + i] = bf16_pair(z[2 * i], z[2 * i + 1]);
    }
}

}  // namespace exkv
