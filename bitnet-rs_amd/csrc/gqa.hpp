// gqa.hpp -- what the attention of shared keys and values has in common whatever its caches hold (kernels_gqa.hip, kernels_kv8.hip): the keys that a
// position sees, the records they are cut into, rotation, distance penalty, gates, convolutions and the rows of query and key heads.
#pragma once

#include <algorithm>
#include <cfloat>
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
// How a vector of an 8-bit cache is held: whole numbers -127 .. 127 and one scale.  The scale stays 32 bits wide.  What is smaller than 1.5e-36 throughout counts as zero (its scale would
// have no full mantissa), and a vector with a value that is not finite has a scale that is not a number, so that whoever sees it gets NaN.
struct Kv8Scale {
    float scale, factor;
};
__device__ __forceinline__ Kv8Scale kv8_scale(float largest, bool finite) {
    if (!finite) return {__builtin_nanf(""), 0.f};
    if (!(largest >= 1.5e-36f)) return {0.f, 0.f};
    return {largest / 127.0f, 127.0f / largest};
}
__device__ __forceinline__ int kv8_number(float v, const Kv8Scale &s) { return s.factor == 0.f ? 0 : (int)rintf(v * s.factor); }
__device__ __forceinline__ bool is_finite(float v) { return fabsf(v) <= FLT_MAX; }

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

constexpr int kRowTokens = 16, kRowCols = 32;

// Four tokens of a query or key head of up to 128 NJ columns: a lane holds neighbouring elements, so that a pair turns within it.  TAPS: those of the convolution
// (0: none, -1: any number).  TC int8_t: a key's numbers, and its scale by position in `scales`.
template <class TR, class TC, int NJ, int TAPS>
__device__ __forceinline__ void head_rows(const Gqa &p, const TR *rows, size_t ld, int pos0, int t0, int n, int y, bool key, TC *cache, TR *queries, size_t ldq, float *scales = nullptr) {
    constexpr int U = kRowTokens / 4;
    constexpr bool CONV = TAPS != 0;
    const int lane = threadIdx.x & 63, dim = (int)p.dim, dimp = (int)p.dimp, turned = (int)p.rot_dims, half = turned >> 1;
    const float *w = key ? p.k_weight : p.q_weight;
    float v[U][NJ][2], cs[U][NJ], sn[U][NJ], factor[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int t = min(t0 + u, n - 1);
        const TR *row = rows + (size_t)t * ld + (size_t)y * dimp;
        factor[u] = key ? 1.0f : p.q_factor[pos0 + t];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int i = min(2 * lane + 128 * j, dimp - 2);
            if (CONV)
                v[u][j][0] = v[u][j][1] = 0.f;
            else
                v[u][j][0] = ld_act(row, i), v[u][j][1] = ld_act(row, i + 1);
            cs[u][j] = 1.0f, sn[u][j] = 0.f;
            if (turned && 2 * lane + 128 * j < turned) {
                const size_t at = (size_t)(pos0 + t) * half + lane + 64 * j;
                cs[u][j] = p.rope_cos[at], sn[u][j] = p.rope_sin[at];
            }
        }
    }
    if (TAPS > 0) {  // the tokens and those ahead of them once, in registers
        constexpr int T = TAPS > 0 ? TAPS : 1;
        const int channels = gqa_channels(p);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int c = y * dimp + min(2 * lane + 128 * j, dimp - 2);
            float f[T][2], raw[U + T - 1][2];
#pragma unroll
            for (int k = 0; k < T; ++k) f[k][0] = p.conv[(size_t)k * channels + c], f[k][1] = p.conv[(size_t)k * channels + c + 1];
            if (t0 >= T - 1) {
#pragma unroll
                for (int k = 0; k < U + T - 1; ++k) {
                    const TR *row = rows + (size_t)min(t0 - (T - 1) + k, n - 1) * ld;
                    raw[k][0] = ld_act(row, c), raw[k][1] = ld_act(row, c + 1);
                }
            } else {
#pragma unroll
                for (int k = 0; k < U + T - 1; ++k) {
                    const int t = min(t0 - (T - 1) + k, n - 1);
                    raw[k][0] = raw_value(p, rows, ld, pos0, t, c, channels), raw[k][1] = raw_value(p, rows, ld, pos0, t, c + 1, channels);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < T; ++k) v[u][j][0] += f[k][0] * raw[u + k][0], v[u][j][1] += f[k][1] * raw[u + k][1];
        }
    } else if (CONV) {
        const int taps = (int)p.taps, channels = gqa_channels(p);
        for (int k = 0; k < taps; ++k)
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int c = y * dimp + min(2 * lane + 128 * j, dimp - 2);
                const float f0 = p.conv[(size_t)k * channels + c], f1 = p.conv[(size_t)k * channels + c + 1];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int t = min(t0 + u, n - 1) - (taps - 1) + k;
                    v[u][j][0] += f0 * raw_value(p, rows, ld, pos0, t, c, channels), v[u][j][1] += f1 * raw_value(p, rows, ld, pos0, t, c + 1, channels);
                }
            }
    }
    float wv[NJ][2];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) wv[j][e] = w && 2 * lane + 128 * j + e < dim ? w[2 * lane + 128 * j + e] : 1.0f;  // (padding columns hold zeros)
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (w || p.unit_norm) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j) ss += 2 * lane + 128 * j < dimp ? v[u][j][0] * v[u][j][0] + v[u][j][1] * v[u][j][1] : 0.f;
            factor[u] *= 1.0f / sqrtf(wave_sum(ss) / (float)dim + p.eps);
        }
        if (t0 + u >= n) continue;
        TR *row = queries + (size_t)(t0 + u) * ldq + (size_t)y * dimp;
        if constexpr (std::is_same_v<TC, int8_t>) {
            if (key) {
                float x[NJ][2], largest = 0.f;
                bool finite = true;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const float a = v[u][j][0] * factor[u] * wv[j][0], b = v[u][j][1] * factor[u] * wv[j][1];
                    x[j][0] = a * cs[u][j] - b * sn[u][j], x[j][1] = b * cs[u][j] + a * sn[u][j];
                    if (2 * lane + 128 * j < dimp) largest = fmaxf(largest, fmaxf(fabsf(x[j][0]), fabsf(x[j][1]))), finite = finite && is_finite(x[j][0]) && is_finite(x[j][1]);
                }
                const Kv8Scale s = kv8_scale(rows_max(row_max(largest)), __all(finite));
                int8_t *dst = cache + (size_t)(pos0 + t0 + u) * dimp;
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    if (2 * lane + 128 * j < dimp)
                        *reinterpret_cast<uint16_t *>(dst + 2 * lane + 128 * j) = (uint16_t)((kv8_number(x[j][0], s) & 0xff) | (kv8_number(x[j][1], s) & 0xff) << 8);
                if (lane == 0) scales[pos0 + t0 + u] = s.scale;
                continue;
            }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int i = 2 * lane + 128 * j;
            if (i >= dimp) continue;
            const float a = v[u][j][0] * factor[u] * wv[j][0], b = v[u][j][1] * factor[u] * wv[j][1];
            const float x = a * cs[u][j] - b * sn[u][j], z = b * cs[u][j] + a * sn[u][j];
            if constexpr (!std::is_same_v<TC, int8_t>) {
                if (key) {
                    TC *dst = cache + (size_t)(pos0 + t0 + u) * dimp;
                    st_act(dst, i, x), st_act(dst, i + 1, z);
                    continue;
                }
            }
            st_act(row, i, x), st_act(row, i + 1, z);
        }
    }
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
