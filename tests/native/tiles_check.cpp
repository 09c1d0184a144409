// CPU check of prompt attention's layout and searches (exactkv_amd/csrc/prompt_tiles.hpp), the kernel's own
// code over 64 lanes in host memory: for random packed prompts -- empty sequences, fewer or far more keys than
// queries, windows, query heads per KV head that do not divide a row tile -- every row tile and part of its
// keys is taken by exactly one workgroup, the parts hold the tile's keys without gap or overlap, for every
// number of parts that the kernel may choose; and with offsets that do not ascend, nothing outside the rows
// is named.
#include "../../exactkv_amd/csrc/prompt_tiles.hpp"
#include <cstdio>
#include <cstdlib>
#include <map>
#include <utility>
#include <vector>

using namespace exkv;

struct Lanes {
    int v[64];
};
struct HostWave {
    typedef Lanes Int;
    template <class F, class... X>
    Lanes map(F f, const X&... x) const {
        Lanes r;
        for (int i = 0; i < 64; ++i) r.v[i] = f(x.v[i]...);
        return r;
    }
    Lanes lane() const {
        Lanes r;
        for (int i = 0; i < 64; ++i) r.v[i] = i;
        return r;
    }
    Lanes scan(const Lanes& x) const {
        Lanes r;
        for (int i = 0, sum = 0; i < 64; ++i) r.v[i] = sum += x.v[i];
        return r;
    }
    int read(const Lanes& x, int lane) const {
        if (lane < 0 || lane > 63) abort();
        return x.v[lane];
    }
    uint64_t ballot(const Lanes& x) const {
        uint64_t r = 0;
        for (int i = 0; i < 64; ++i) r |= (uint64_t)(x.v[i] != 0) << i;
        return r;
    }
};

static uint64_t state = 0x9E3779B97F4A7C15ull;
static int pick(int lo, int hi) {      // lo .. hi
    state ^= state << 13; state ^= state >> 7; state ^= state << 17;
    return lo + (int)(state % (uint64_t)(hi - lo + 1));
}

struct Call {
    int S, N, NK, G, Hkv, D, window;
    std::vector<int> cq, ck;
    bool sound;
};
static long checks = 0, failures = 0;
static void check(bool ok, const char* what, const Call& c, int t) {
    ++checks;
    if (ok) return;
    if (++failures > 10) return;
    printf("FAIL %s: t %d S %d N %d NK %d G %d Hkv %d D %d window %d sound %d; cq", what, t, c.S, c.N, c.NK, c.G, c.Hkv, c.D,
           c.window, (int)c.sound);
    for (int x : c.cq) printf(" %d", x);
    printf("; ck");
    for (int x : c.ck) printf(" %d", x);
    printf("\n");
}

// find_tile: the block of 64 sequences that holds tile t, then its search.
template <int KEYS>
static bool find_tile(const Call& c, int t, PromptTile& tile, int& seq) {
    const HostWave w;
    for (int s0 = 0; s0 < c.S; s0 += 64) {
        Lanes begin{}, len{}, begin_k{}, len_k{}, n{};
        for (int i = 0; i < 64 && s0 + i < c.S; ++i) {
            clip_sequence(c.cq[s0 + i], c.cq[s0 + i + 1], s0 + i == 0, c.N, begin.v[i], len.v[i]);
            clip_sequence(c.ck[s0 + i], c.ck[s0 + i + 1], s0 + i == 0, c.NK, begin_k.v[i], len_k.v[i]);
            n.v[i] = row_tiles(len.v[i], c.G);
        }
        const Lanes incl = w.scan(n);
        if (t < incl.v[63]) {
            int l, index;
            const bool found = nth_tile<KEYS>(w, c.S, c.G, c.NK, t, len, len_k, n, incl, l, index);
            check(found, "a tile within the count is found", c, t);
            if (!found) return false;
            tile = PromptTile{begin.v[l], len.v[l], begin_k.v[l], len_k.v[l], index * kRows};
            seq = s0 + l;
            return true;
        }
        t -= incl.v[63];
    }
    return false;
}

// The tile's rows and keys lie within the call's.
static void check_bounds(const Call& c, int t, const PromptTile& x, int first, int last, int KEYS) {
    check(x.row0 >= 0 && x.row0 < x.Lq * c.G, "rows within the sequence", c, t);
    check(x.q0 >= 0 && x.q0 + x.Lq <= c.N && x.k0 >= 0 && x.Lk >= 0 && x.k0 + x.Lk <= c.NK, "sequence within the rows", c, t);
    check(first >= 0 && (last < first || last * KEYS < x.Lk), "key tiles within the sequence", c, t);
}

template <int KEYS>
static void run(const Call& c) {
    const HostWave w;
    const PromptPlan p = plan_prompt(c.N, c.NK, c.S, (int64_t)c.G * c.Hkv, c.Hkv, c.D, c.window);
    std::vector<int> Lq(c.S), Lk(c.S);
    int all = 0, begin;
    for (int s = 0; s < c.S; ++s) {
        clip_sequence(c.cq[s], c.cq[s + 1], s == 0, c.N, begin, Lq[s]);
        clip_sequence(c.ck[s], c.ck[s + 1], s == 0, c.NK, begin, Lk[s]);
        all += row_tiles(Lq[s], c.G);
    }
    if (c.sound) check(all <= p.tiles, "a workgroup for every row tile", c, all);
    typedef std::pair<int, int> Key;                   // sequence, row tile
    // whole tiles
    std::map<Key, int> seen;
    PromptTile x;
    int seq, first, last;
    for (int64_t b = 0; b < p.tiles; ++b) {
        const int t = b >= p.turn ? (int)(p.tiles - 1 - (b - p.turn)) : (int)b;
        if (!find_tile<KEYS>(c, t, x, seq)) continue;
        key_tiles<KEYS>(x, c.G, c.window, first, last);
        check_bounds(c, t, x, first, last, KEYS);
        ++seen[Key(seq, x.row0)];
    }
    if (c.sound) {
        check((int)seen.size() == all, "every tile taken", c, (int)seen.size());
        for (auto& s : seen) check(s.second == 1, "a tile taken once", c, s.first.second);
    }
    if (p.split <= 1) return;
    // cut keys: every number of parts that may be chosen
    Lanes lq{}, lk{}, n{};
    int longest = 1;
    for (int s = 0; s < c.S; ++s) {
        lq.v[s] = Lq[s];
        lk.v[s] = Lk[s];
        n.v[s] = row_tiles(Lq[s], c.G);
        if (n.v[s] == 0) continue;
        longest = most_of(longest, key_tiles_most<KEYS>(least_of((kRows - 1) / c.G, Lq[s] - 1), Lq[s], Lk[s], c.G, c.window));
        longest = most_of(longest, key_tiles_most<KEYS>(Lq[s] - 1, Lq[s], Lk[s], c.G, c.window));
    }
    for (int k = 1; k <= p.split; ++k) {
        std::map<Key, std::vector<Key>> parts_seen;    // of a tile: first and last key tile of each part
        for (int64_t b = 0; b < p.blocks; ++b) {
            int t = (int)b, part = 0, most = (longest + k - 1) / k;
            if (!nth_part<KEYS>(w, c.S, c.G, c.window, longest, (int)p.blocks, n, lq, lk, t, part, most)) continue;
            if (!find_tile<KEYS>(c, t, x, seq)) {
                check(false, "a part has a tile", c, t);
                continue;
            }
            key_tiles<KEYS>(x, c.G, c.window, first, last);
            check_bounds(c, t, x, first, last, KEYS);
            check(last - first + 1 <= longest, "no tile is longer than the longest", c, t);
            const int parts = parts_of(first, last, most);
            if (c.sound) check(parts <= p.split, "no more parts than the workspace holds", c, parts);
            if (part >= parts) continue;
            if (parts > 1) part_tiles(part, parts, first, last);
            check_bounds(c, t, x, first, last, KEYS);
            check(parts == 1 || first <= last, "no part is empty", c, t);
            parts_seen[Key(seq, x.row0)].push_back(Key(first, last));
        }
        if (!c.sound) continue;
        check((int)parts_seen.size() == all, "every tile taken, cut", c, k);
        for (auto& s : parts_seen) {
            x = PromptTile{0, Lq[s.first.first], 0, Lk[s.first.first], s.first.second};
            key_tiles<KEYS>(x, c.G, c.window, first, last);
            for (auto& q : s.second) {                 // ascending: all first parts come first
                check(q.first == first, "parts join", c, k);
                first = q.second + 1;
            }
            check(first == last + 1, "parts hold all keys", c, k);
        }
    }
}

int main() {
    const int groups[] = {1, 2, 3, 4, 5, 7, 8, 16, 17, 130}, dims[] = {64, 128, 256}, counts[] = {1, 1, 2, 3, 5, 20, 64, 70};
    int split = 0;
    for (int it = 0; it < 1500; ++it) {
        Call c;
        c.S = counts[pick(0, 7)];
        c.G = groups[pick(0, 9)];
        c.D = dims[pick(0, 2)];
        c.Hkv = 1 << pick(0, 3);
        c.cq.assign(1, 0);
        c.ck.assign(1, 0);
        for (int s = 0; s < c.S; ++s) {
            const int few = c.S < 10 ? 400 : 30;
            const int l = pick(0, 3) == 0 ? pick(0, 1) : pick(0, few);
            const int kind = pick(0, 4), k = kind == 0 ? l : kind == 1 ? pick(0, most_of(1, l)) : kind == 2 ? 0 : l + pick(0, 6000);
            c.cq.push_back(c.cq.back() + l);
            c.ck.push_back(c.ck.back() + k);
        }
        c.N = c.cq.back() + (pick(0, 2) == 0 ? 5 : 0);
        c.NK = c.ck.back();
        c.window = pick(0, 2) == 0 ? pick(1, 3000) : 0;
        c.sound = pick(0, 4) != 0;
        if (!c.sound)
            for (int i = 0; i < 2; ++i) {
                c.cq[pick(0, c.S)] += pick(-500, 500);
                c.ck[pick(0, c.S)] += pick(-5000, 5000);
            }
        if (c.N == 0) continue;
        if (c.window > c.NK) c.window = c.NK;
        split += plan_prompt(c.N, c.NK, c.S, (int64_t)c.G * c.Hkv, c.Hkv, c.D, c.window).split > 1;
        if (c.D == 256) run<32>(c); else run<64>(c);
    }
    // row tiles that begin and end within a token's heads, and windows that reach one tile further with one
    // token more, at every place of a key tile
    for (int G : {3, 5, 7, 17})
        for (int D : dims) {
            const int K = keys_per_tile(D), span = (127 + G - 1) / G, window = 1024 + (K + 2 - span % K) % K;
            for (int keys = 2700; keys < 2700 + K; ++keys) {
                const Call c{1, 280, keys, G, 1, D, window, {0, 280}, {0, keys}, true};
                ++split;
                if (D == 256) run<32>(c); else run<64>(c);
            }
        }
    printf("%ld checks, %d split calls, %ld failures\n", checks, split, failures);
    return failures != 0;
}
