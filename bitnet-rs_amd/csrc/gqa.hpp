// gqa.hpp -- what the attention of shared keys and values has in common whatever its caches hold (kernels_gqa.hip, kernels_kv8.hip): the keys that a
// position sees, the records they are cut into, rotation, distance penalty, gates and convolutions.
#pragma once

#include <algorithm>
#include <type_traits>

#include "dense.hpp"

namespace bitnet_hip {

constexpr float kLog2e = 1.44269504088896f;

// the first key a query at this position sees
__host__ __device__ __forceinline__ int gqa_first(const Gqa &p, int pos) {
    const int first = p.chunk ? pos - (int)((unsigned)pos % (unsigned)p.chunk) : 0;
    return p.window && pos - (int)p.window + 1 > first ? pos - (int)p.window + 1 : first;
}

// The records of a query at `pos`: tiles of keys from `base` (the tile that holds its first key) on, `per` tiles each.
struct GqaRange {
    int first, base, per, used;
};
__device__ __forceinline__ GqaRange gqa_range(const Gqa &p, int pos) {
    GqaRange r;
    r.first = gqa_first(p, pos);
    r.base = r.first & ~(kGqaTile - 1);
    const int tiles = (pos + 1 - r.base + kGqaTile - 1) / kGqaTile;
    r.per = (tiles + kGqaSplits - 1) / kGqaSplits;
    r.used = (tiles + r.per - 1) / r.per;
    return r;
}
// records a launch has to provide for
static int gqa_records(const Gqa &g) {
    size_t keys = g.capacity;
    if (g.chunk && g.chunk + kGqaTile < keys) keys = g.chunk + kGqaTile;  // (a chunk may start inside a tile)
    if (g.window && g.window + kGqaTile < keys) keys = g.window + kGqaTile;
    return (int)min((size_t)kGqaSplits, (keys + kGqaTile - 1) / kGqaTile);
}

// element i of a head at a position, v being its own and the lane's neighbour holding the other element of the pair; cs, sn: the tables' row
__device__ __forceinline__ float turn_neighbours(float v, int i, const float *cs, const float *sn, int dims) {
    const float o = dpp<0xb1>(v);  // quad_perm [1,0,3,2]
    if (i >= dims) return v;
    const float c = cs[i >> 1], s = sn[i >> 1];
    return (i & 1) ? v * c + o * s : v * c - o * s;
}
// what a head's gate (or that of a column of it) is the sigmoid of
__device__ __forceinline__ float gate_logit(const Gqa &p, int row, int h, int column) {
    const size_t i = (size_t)row * p.ldgate + (p.gate_columns ? (size_t)h * p.vdimp + column : (size_t)h);
    return p.gate_f32 ? ((const float *)p.gate)[i] : bf2f(((const uint16_t *)p.gate)[i]);
}
// a head's distance penalty: what is taken off the natural score is weight * log2(1 + rate * distance)
struct FarPenalty {
    float weight, rate;
};
__device__ __forceinline__ FarPenalty far_penalty(const Gqa &p, int h) {
    FarPenalty f{0.f, 0.f};
    if (p.far_weight) f.weight = p.far_weight[h] * 0.69314718055994531f, f.rate = p.far_rate[h];
    return f;
}
__device__ __forceinline__ float nearer(float score, const FarPenalty &f, int distance) { return fmaf(-f.weight, __log2f(fmaf(f.rate, (float)distance, 1.0f)), score); }
// columns of a row of projections that a convolution covers
__host__ __device__ __forceinline__ int gqa_channels(const Gqa &p) {
    if (p.queries_only) return (int)(p.heads * p.maps * p.dimp);
    return (int)((p.heads + p.kv_heads) * p.maps * p.dimp + (p.values_are_keys ? 0 : p.kv_heads * p.vdimp));
}
// column c of the row of projections t (negative: an earlier portion's; zero ahead of the sequence)
template <class TR>
__device__ __forceinline__ float raw_value(const Gqa &p, const TR *rows, size_t ld, int pos0, int t, int c, int channels) {
    if (t >= 0) return ld_act(rows + (size_t)t * ld, c);
    const int at = pos0 + t;
    return at >= 0 ? p.ring[(size_t)(at % (int)p.taps) * channels + c] : 0.f;
}

// ---- how a prompt's launch is shared out -----------------------------------------------------------------------------
// Two groups fill a CU, and halve its walks; of one group two workgroups fit.  They pay while the launch is as long as its longest walk: with four tiles or more in it, a CU's
// share of all tiles not much above it, and no second round behind walks that are all long (the shortest walk of the first round and the longest of the second one in turn).
// Heads count as a multiple of eight, as the launch deals them to the XCDs (20 heads take what 24 do).  us with two / with one: 24 heads, 2600 tokens
// 80 / 90 (share / walk 1.05), 32 heads, 2048 63 / 75 (1.06), 40 heads, 1664 63 / 62 (1.09), 24 heads, 3000 105 / 105 (1.19), 3328 124 / 121 (1.27), 4096 173 / 153 (1.55); two maps,
// 24 heads, 1280 39 / 44, 1531 57 / 53, 2048 88 / 75; five tiles 13.1 / 13.9, four 13.0 / 12.4.
inline bool two_groups(const Gqa &g, int rows, int n_ctx, int nq) {
    const int at_once = 256, pos0 = n_ctx - nq, heads = ((int)g.heads + 7) / 8 * 8, blocks = (nq + rows - 1) / rows, all_tiles = (n_ctx + 63) / 64;
    long longest = 0, total = 0, second = 0;
    for (int qb = blocks - 1, done = 0; qb >= 0 && total <= 2l * at_once * all_tiles; --qb, done += heads) {
        const int q0 = qb * rows, tiles = (std::min(n_ctx, pos0 + q0 + rows) + 63) / 64 - (gqa_first(g, pos0 + q0) >> 6);
        longest = std::max<long>(longest, tiles), total += (long)heads * tiles;
        for (int i : {at_once - 1, at_once})
            if ((long)heads * blocks > at_once && done <= i && i < done + heads) second += tiles;
    }
    return longest >= 4 && 16 * total <= 17 * at_once * longest && 10 * second <= 11 * longest;
}

// Few queries behind many keys: a launch whose blocks leave CUs without a workgroup lasts as long as its longest walk, so a block's tiles are cut into stretches, of two tiles (a step of two
// groups) at least and no more of them than there are CUs for (heads count as a multiple of eight, as the launch deals them to the XCDs: 12 heads in 21 stretches take 32 us where 15 take 24).
// A step of a walk that is saved is worth 2.7 us (7 of one group); the launch that puts the records together costs 5 and 0.7 ns for each query's head, 1.4 for each of a head's two maps.
// us without / with, heads, keys, queries: 12, 2090, 90 51 / 18; 24, 2090, 90 52 / 22; 12, 600, 20 18.3 / 11.1; 12, 1000, 200 28.7 / 18.9; 12, 450, 130 17.7 / 14.5; 12, 8000, 30 168 / 27;
// 24 of two maps, 2090, 90 49 / 28; 2 of 256 columns, 2000, 50 131 / 22; 8, 2000, 2000 50 / 40.  What stays whole: 12, 400, 400 15.9 / 18.1; 16, 512, 512 18.6 / 21.2; 24 of two maps,
// 600, 100 18.3 / 20.6; 12, 100, 3 8.4.
inline int gqa_prefill_parts(const Gqa &g, int n_ctx, int nq) {
    const int rows = g.maps == 2 ? 64 : 128, blocks = (nq + rows - 1) / rows, heads = ((int)g.heads + 7) / 8 * 8;
    const int tiles = (n_ctx + 63) / 64 - (gqa_first(g, n_ctx - nq + (blocks - 1) * rows) >> 6), most = std::min<long>(256 / ((long)heads * blocks), 32);
    if (most < 2) return 1;
    const int each = ((tiles + most - 1) / most + 1) & ~1, saved = (tiles + 1) / 2 - each / 2;
    return 2.7 * saved > 5.0 + (g.maps == 2 ? 1.4e-3 : 7e-4) * (double)nq * (double)(g.heads * g.maps) ? (tiles + each - 1) / each : 1;
}

}  // namespace bitnet_hip
