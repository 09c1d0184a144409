// Prompt attention's row tiles and the key tiles they walk: how a call is laid out, and which row tile and
// part of its keys a workgroup takes. All of it is integer arithmetic over the sequences' lengths, and what
// it finds goes into the addresses of reads, so it builds for the host as well (tests/native/tiles_check.cpp
// counts every tile and part there).
//
// The searches run in a wavefront, a lane a sequence. They are templates on the wavefront `w`, which gives
// the kernel's lane operations, or those of 64 lanes in host memory: Int (a value per lane), map(f, x, ..)
// (f lane by lane), scan (inclusive sums), read(x, lane), ballot.
#pragma once

#include "common.hpp"

namespace exkv {

constexpr int kRows = 128, kWaves = 4;   // query rows and wavefronts of a workgroup

// One sequence's share of a workgroup: rows row0 .. of its Lq * G, key rows k0 .. k0 + Lk - 1.
struct PromptTile {
    int q0, Lq, k0, Lk, row0;
};

__host__ __device__ inline int least_of(int a, int b) { return a < b ? a : b; }
__host__ __device__ inline int most_of(int a, int b) { return a > b ? a : b; }

// The offsets a, b of a sequence (`first`: the call's first), made fit for use where they are not:
// 0 <= begin <= end <= rows. True where they were not.
__host__ __device__ inline bool clip_sequence(int a, int b, bool first, int rows, int& begin, int& len) {
    begin = least_of(most_of(a, 0), rows);
    const int end = least_of(most_of(b, begin), rows);
    len = end - begin;
    return begin != a || end != b || (first && a != 0);
}

__host__ __device__ inline int row_tiles(int Lq, int G) { return (int)(((int64_t)Lq * G + kRows - 1) / kRows); }

// Of a sequence's n row tiles those whose last row is `row` or behind it.
__host__ __device__ inline int tiles_from(int64_t row, int Lq, int n, int G) {
    return row >= (int64_t)Lq * G ? 0 : n - (row > 0 ? (int)((uint32_t)row / kRows) : 0);
}

// Those that walk at least x key tiles: row r does if its token's key, r / G + Lk - Lq, is at least
// (x - 1) KEYS, and a tile if its last row does; all walk 0 (tokens may stand far before the first key).
template <int KEYS>
__host__ __device__ inline int tiles_walking(int x, int Lq, int Lk, int n, int G) {
    return x == 0 ? n : tiles_from((int64_t)((x - 1) * KEYS - (Lk - Lq)) * G, Lq, n, G);
}

// Key tiles that row tile `row0` of a sequence walks: first .. last.
template <int KEYS>
__host__ __device__ inline void key_tiles(const PromptTile& tile, int G, int window, int& first, int& last) {
    const int shift = tile.Lk - tile.Lq, nrows = tile.Lq * G;
    const int t_lo = tile.row0 / G, t_hi = least_of(tile.row0 + kRows - 1, nrows - 1) / G;
    const int k_lo = window > 0 ? most_of(0, t_lo + shift - window + 1) : 0, k_hi = t_hi + shift;
    first = k_lo / KEYS;
    last = k_hi < 0 ? first - 1 : k_hi / KEYS;
}

// Key tiles, at most, of a row tile whose last token is t_hi: a row tile's tokens, which may begin and end
// within a group, are up to `span` apart, and c keys in a row, which may begin and end within a tile, lie in
// (c - 2) / KEYS + 2.
template <int KEYS>
__host__ __device__ inline int key_tiles_most(int t_hi, int Lq, int Lk, int G, int window) {
    const int span = (kRows - 1 + G - 1) / G;
    const int keys = most_of(0, t_hi + Lk - Lq + 1), n = (keys + KEYS - 1) / KEYS;
    return window > 0 ? least_of(n, (window + span + 2 * KEYS - 2) / KEYS) : n;
}

// Parts of a row tile whose keys are cut into parts of up to `most` tiles, and the tiles of one of them.
__host__ __device__ inline int parts_of(int first, int last, int most) { return most_of(1, (last - first + most) / most); }
__host__ __device__ inline void part_tiles(int part, int parts, int& first, int& last) {
    const int per = (last - first + parts) / parts;
    first += part * per;
    last = least_of(last, first + per - 1);
}

__host__ __device__ inline int first_lane(uint64_t lanes) { return lanes != 0 ? __builtin_ctzll(lanes) : -1; }

// The tile to take `t`-th of up to 64 sequences (of S) with n row tiles, incl up to and with theirs: lane
// `l`'s row tile `index`. The tiles with the most keys come first where these are all sequences; else
// sequence by sequence, each one's last tile first. False where none is found, which the counts rule out:
// what is read follows from l and index, so they are checked rather than trusted.
template <int KEYS, class W>
__host__ __device__ inline bool nth_tile(const W& w, int S, int G, int NK, int t, typename W::Int Lq, typename W::Int Lk,
                                         typename W::Int n, typename W::Int incl, int& l, int& index) {
    if (S > 1 && S <= 64) {
        auto walking = [&](int x) {
            return w.map([=](int lq, int lk, int tiles) { return tiles_walking<KEYS>(x, lq, lk, tiles, G); }, Lq, Lk, n);
        };
        // the most key tiles that more than t tiles walk at least
        int lo = 0, hi = NK / KEYS + 2;                // all tiles walk 0; none walks hi
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            const int c = w.read(w.scan(walking(mid)), 63);
            if (c > t) lo = mid; else hi = mid;
        }
        const auto more = walking(lo + 1);
        const auto same = w.map([](int a, int b) { return a - b; }, walking(lo), more);
        const int rank = t - w.read(w.scan(more), 63);
        const auto upto = w.scan(same);
        l = first_lane(w.ballot(w.map([=](int u) { return (int)(u > rank); }, upto)));
        if (l < 0) return false;
        index = w.read(n, l) - w.read(more, l) - 1 - (rank - (w.read(upto, l) - w.read(same, l)));
    } else {
        l = first_lane(w.ballot(w.map([=](int u) { return (int)(u > t); }, incl)));
        if (l < 0) return false;
        index = w.read(incl, l) - 1 - t;
    }
    return index >= 0 && index < w.read(n, l);
}

// Which part of a row tile workgroup t takes, and the number t of that tile among those that have such a
// part (nth_tile's), where parts have up to `most` key tiles and no row tile more than `longest`. Lane p
// counts the row tiles that have a part p, exactly: all first parts come first, then all second ones and so
// on, without gaps. Where these would be more than `limit` no tile is cut (most becomes longest). With a
// window all tiles have a place for every part where any has; some are then empty. False: no part is left.
template <int KEYS, class W>
__host__ __device__ inline bool nth_part(const W& w, int S, int G, int window, int longest, int limit, typename W::Int n,
                                         typename W::Int Lq, typename W::Int Lk, int& t, int& part, int& most) {
    int all = 0;
    const int64_t keys = (int64_t)most * KEYS;
    typename W::Int count = w.map([](int) { return 0; }, w.lane());
    for (int i = 0; i < S; ++i) {
        const int tiles = w.read(n, i), lq = w.read(Lq, i), lk = w.read(Lk, i);
        count = w.map([=](int c, int lane) { return c + tiles_from(((int64_t)lane * keys - (lk - lq)) * G, lq, tiles, G); },
                      count, w.lane());
        all += tiles;
    }
    const int places = window > 0 ? (longest + most - 1) / most : 1;     // that all tiles have
    count = w.map([=](int c, int lane) { return lane < places ? all : window > 0 ? 0 : c; }, count, w.lane());
    typename W::Int upto = w.scan(count);
    if (w.read(upto, 63) > limit) {                    // more than the model thought: no split
        most = longest;
        count = w.map([=](int lane) { return lane == 0 ? all : 0; }, w.lane());
        upto = w.map([=](int) { return all; }, w.lane());
    }
    const int at = t;
    part = first_lane(w.ballot(w.map([=](int u) { return (int)(u > at); }, upto)));
    if (part < 0) return false;
    t -= w.read(upto, part) - w.read(count, part);
    return true;
}

// How a call is laid out. `slots` workgroups run at a time: two a CU (four at head dim 64). Keys are
// split where the row tiles leave CUs free and are long enough for what the parts' results cost.
//
// Head dim 256 has two instances: one workgroup a CU, with the next tile's scores beside this tile's
// weights (1.05 us a step), and two without (1.35 us alone, 0.96 together). The former where no CU gets
// more than two: one / two a CU, 16q/4kv, 2K tokens 72 / 92 us, 3,000 101 / 131, 4K 155 / 190, but 6,000
// 337 / 312, 8K 563 / 491.
__host__ __device__ constexpr int keys_per_tile(int D) { return D == 256 ? 32 : 64; }
constexpr int kLeast = 8;              // key tiles of the longest row tile, per part, at least
struct PromptPlan {
    int64_t tiles;                     // row tiles, at most
    int split, slots;
    int turn;                          // two workgroups a CU in one go: the second ones in reverse, so that a
                                       // CU's two tiles add up to about the same (one prompt of 1,500
                                       // tokens 32.7 us without, 31.4 so; of 2,048 no difference)
    bool alone;                        // head dim 256: one workgroup a CU
    int64_t blocks;                    // workgroups of a KV head
};
inline PromptPlan plan_prompt(int64_t N, int64_t NK, int64_t S, int64_t Hq, int64_t Hkv, int D, int64_t window) {
    // every sequence's last tile may be partial
    const int64_t tiles = (N * (Hq / Hkv) + S * (kRows - 1)) / kRows, units = (tiles > 0 ? tiles : 1) * Hkv;
    PromptPlan p{units / Hkv, 1, D == 64 ? 1024 : 512, INT32_MAX, D == 256 && units <= 512, units / Hkv};
    if (p.alone) p.slots = 256;
    const int64_t reach = window > 0 && window + kRows < NK ? window + kRows : NK;
    const int64_t keys = (reach + keys_per_tile(D) - 1) / keys_per_tile(D), few = D == 64 ? 512 : 256;
    if (units >= few || S > 64 || S == 0 || 25 * keys < 150 + units * D / 64) {
        if (!p.alone && units > 256 && units <= 512) p.turn = (int)((256 + Hkv - 1) / Hkv);
        return p;
    }
    int64_t split = 4 * few / units;
    if (split > D / 4) split = D / 4;
    if (split > keys / kLeast) split = keys / kLeast;
    if (split > 1) {
        const int64_t most = (p.slots + p.slots / (p.alone ? 2 : 8)) / Hkv;
        p.split = (int)split;
        p.blocks = p.tiles * split < most ? p.tiles * split : most > p.tiles ? most : p.tiles;
    }
    return p;
}

}  // namespace exkv
