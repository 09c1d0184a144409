// What the kernels over packed prompts share: rows of queries, keys and values brought to LDS by direct loads, and
// the exchange between a wavefront's halves.
#pragma once

#include "prompt_tiles.hpp"
#include "tile.hpp"

namespace exkv {

#define EXKV_LDS __attribute__((address_space(3)))

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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

// f(0), .. f(N - 1) with constants.
template <int N, class F, int... I>
__device__ inline void each_of(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ inline void each(F f) { each_of<N>(f, std::make_integer_sequence<int, N>{}); }

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
// Piece I of a wavefront's share of a tile straight to LDS: 16 bytes a lane, lane l's to lds + 1024 I
// + 16 l. Inline, since the compiler would wait for every such load before each LDS read; no memory
// clobber either, so that LDS reads of other stages may move past it: the wait and the barrier
// before a stage is read, and the barrier before it is loaded again, order them.
template <int I>
__device__ inline void load_piece(u32x4 buf, uint32_t off, uint32_t lds) {
    if constexpr (I == 0)                              // M0 may have been written just before
        asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(buf), "{m0}"(lds));
    else
        asm volatile("buffer_load_dwordx4 %0, %1, 0 offen offset:%3 lds" ::"v"(off), "s"(buf), "{m0}"(lds), "n"(1024 * I));
}

// Which piece of a row's 16-byte pieces lies where: piece c of key row r at c ^ swizzle(r). Keys are
// read one piece over 16 rows at a time (16 pieces or 16 rows cover the 256 bytes of all banks),
// values four pieces over four rows.
template <int D>
__host__ __device__ constexpr int key_swizzle(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
template <int D>
__host__ __device__ constexpr int value_swizzle(int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }

// The descriptor of a tile of KEYS key or value rows of one sequence and head (wave-uniform), and of
// the next ones. Rows behind the sequence's end lie past its size.
template <int D, int KEYS>
struct Stream {
    u32x4 buf;
    int left;                          // rows from the tile on
    uint32_t pitch, step;              // bytes between rows; of a tile
    __device__ Stream(const uint16_t* p, int64_t s_t, int64_t at_head, const PromptTile& t, int key)
        : left(t.Lk - key), pitch((uint32_t)s_t * 2) {
        buf = buffer_of(p + (int64_t)(t.k0 + key) * s_t + at_head, 0);
        step = KEYS * pitch;
        size();
    }
    __device__ void size() { buf.z = left > 0 ? (min(left, KEYS) - 1) * pitch + 2 * D : 0; }
    __device__ void next() {
        const uint64_t a = (((uint64_t)buf.y << 32) | buf.x) + step;
        buf.x = (uint32_t)a;
        buf.y = (uint32_t)(a >> 32);
        left -= KEYS;
        size();
    }
};

// A wavefront's lane operations, for the searches.
struct DeviceWave {
    typedef int Int;
    template <class F, class... X>
    __device__ auto map(F f, X... x) const { return f(x...); }
    __device__ int lane() const { return threadIdx.x & 63; }
    __device__ int scan(int x) const { return wave_incl_scan(x); }
    __device__ int read(int x, int lane) const { return __builtin_amdgcn_readlane(x, lane); }
    __device__ uint64_t ballot(int x) const { return __ballot(x); }
};

}  // namespace exkv
