// gqa.hpp -- what the attention of shared keys and values has in common whatever its caches hold (kernels_gqa.hip, kernels_kv8.hip): the keys that a
// position sees, the records that a launch has to provide for, distance penalty, gates and convolutions.
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

// records a launch has to provide for
static int gqa_records(const Gqa &g) {
    size_t keys = g.capacity;
    if (g.chunk && g.chunk + kGqaTile < keys) keys = g.chunk + kGqaTile;  // (a chunk may start inside a tile)
    if (g.window && g.window + kGqaTile < keys) keys = g.window + kGqaTile;
    return (int)min((size_t)kGqaSplits, (keys + kGqaTile - 1) / kGqaTile);
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

}  // namespace bitnet_hip
