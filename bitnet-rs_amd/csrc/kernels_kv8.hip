// kernels_kv8.hip -- the attention of kernels_gqa.hip over caches of 8 bits (gfx950).
//
// A head's key (of one map) and a head's value at a position are whole numbers -127 .. 127 with one f32 scale each: value = number * scale (kv8_scale).  One scale
// per position, not per block of them: an append touches nothing that is written, and the cache is a function of the tokens alone, whatever portions they came in.
// Keys int8 [kv head][map][capacity][dimp]; values int8 [kv head][capacity / 32][vdimp / 32][16][4][2][8]: column c at position p lies at [p / 32][c / 32][c % 16]
// [p % 32 / 8][c % 32 / 16][p % 8], so that 32 keys by 32 columns are 1 KiB in the order in which the matrix cores take them, and 32 keys of a head are one piece.
//   k_kv8_rows     rows of projections: convolution, norms, rotation, then 8 bits
//   k_kv8_read     positions back as bf16 or f32
//   k_kv8_step     the decode step, records as k_gqa_step leaves them
//   k_kv8_prefill  a prompt's portion
// A step's scores are whole: a query is cut into three balanced digits of 8 bits with one scale (23 bits), the products with the keys' numbers are exact in 32-bit integers, and
// the scales come behind them; a weight times its value's scale meets the values' numbers, which f16 holds exactly, as a (high, low) pair of f16.  A prompt's queries are bf16 and
// so are its outputs: f16 throughout (see there).
#include <cfloat>

#include "gqa.hpp"
#include "kv8_schedule.hpp"

namespace bitnet_hip {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// four int8 -> four f16: 0x6400 | u is 1024 + u, u = number + 128
__device__ __forceinline__ void four_f16(uint32_t numbers, uint32_t &lo, uint32_t &hi) {
    const uint32_t u = numbers ^ 0x80808080u;
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
}
__device__ __forceinline__ f16x8 eight_f16(uint32_t a, uint32_t b) {
    u32x4 v;
    uint32_t x, y;
    four_f16(a, x, y), v.x = x, v.y = y;
    four_f16(b, x, y), v.z = x, v.w = y;
    return __builtin_bit_cast(f16x8, v);
}
// the same plus 1152: what a sum of them is too much by is taken off elsewhere
__device__ __forceinline__ f16x8 eight_raised(uint32_t a, uint32_t b) {
    const uint32_t u = a ^ 0x80808080u, v = b ^ 0x80808080u;
    return __builtin_bit_cast(f16x8, u32x4{__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u),
                                           __builtin_amdgcn_perm(0x64646464u, v, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, v, 0x04030402u)});
}
// the largest of three (an instruction by name: fmaxf would first make every operand canonical)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
// the least E with |v| < 2^E (v = 0: `least`, which is the least it gives)
__device__ __forceinline__ int exponent_above(float v, int least) { return v > 0.f ? max(__builtin_amdgcn_frexp_expf(v), least) : least; }
__device__ __forceinline__ float power2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// Shares.  What a value brings to an output is its numbers times a share: its weight, exp2(score - m), times its scale.  Shares meet the numbers in f16, so a scale goes without the power of
// two that the largest one so far needs (its factor, below 1), and m follows a query's largest share (score plus the factor's exponent) instead of its largest score: whatever else is larger,
// unseen or without weight, a query's shares lie where f16 holds them.  (A weight alone, of a small value, may be above 1: sums are f32.)  A factor's exponent counts as kBelow at least, which
// keeps sums finite; and where a larger scale makes all factors smaller by 2^less, m moves down with them as far as the sum has room.
constexpr int kLeast = -126, kBelow = -64;  // of scales, of factors
// (of a factor that is held times 2^up)
__device__ __forceinline__ float factor_exponent(float v, int up) { return (float)max((int)(__builtin_bit_cast(uint32_t, v) >> 23) - 126 - up, kBelow); }
__device__ __forceinline__ int room_for(float sum, int less) { return sum > 0.f ? min(less, max(100 - __builtin_amdgcn_frexp_expf(sum), 0)) : min(less, 100); }

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

// What a portion and a step do to a key alike, operation by operation, so that both write the same bytes (but for the order of a norm's sum): what a norm multiplies with, and an element of a
// turned pair, `other` with its sign.
// (the instruction's root and one of Newton's steps: to a unit in the last place; 16384 rows of 25 heads 47 us, by 1 / sqrtf(sum / dim + eps) 52)
__device__ __forceinline__ float norm_factor(float sum, float per_dim, float eps) {
    const float a = fmaf(sum, per_dim, eps), y = __builtin_amdgcn_rsqf(a), off = fmaf(-(a * y), y, 1.0f);
    return off == off ? fmaf(0.5f * y, off, y) : y;  // (zero and infinity)
}
__device__ __forceinline__ float turned(float own, float other, float c, float s) { return fmaf(own, c, other * s); }

// where column c of a kv head's values at position pos lies
__device__ __forceinline__ size_t kv8_value_at(int vdimp, int pos, int c) {
    return (size_t)(pos >> 5) * (vdimp * 32) + (c >> 5) * 1024 + (c & 15) * 64 + (pos >> 3 & 3) * 16 + (c >> 4 & 1) * 8 + (pos & 7);
}

// ---- rows of projections ----------------------------------------------------------------------------------------------
// Bound by memory: 16384 tokens of 20 heads on 5 of 128 columns, bf16, half of them turned, are 232 MB in 53 us (4.4 TB/s; a copy reaches 5.3 to 5.5).  By heads first and pairs of columns it
// was 80, whole rows at a time 64; a wave's heads in turn, with the rotation and the next columns in registers, took the rest.  One token 3.7, 1531 of two maps of 64 / 128 7.2.
// A lane holds eight neighbouring columns, KL or VL lanes a head's row: pairs turn within a lane, and a wave takes 64 / KL tokens at a time, R times.  Workgroups: four waves'
// tokens and a part of the heads (query heads x maps, key heads x maps; one after the other, the next one's columns on their way), then values, eight or 32
// positions a wave, through LDS into the cache's order.

template <int L>
__device__ __forceinline__ float lanes_max(float v) {
    v = fmaxf(v, dpp<0xb1>(v));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp<0x4e>(v));   // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp<0x141>(v));  // row_half_mirror
    if (L >= 16) v = fmaxf(v, dpp<0x140>(v));  // row_mirror
    if (L >= 32) {
        float w = v;
        swap_rows16(v, w);
        v = fmaxf(v, w);
    }
    return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
    v += dpp<0xb1>(v);
    v += dpp<0x4e>(v);
    v += dpp<0x141>(v);
    if (L >= 16) v += dpp<0x140>(v);
    if (L >= 32) {
        float w = v;
        swap_rows16(v, w);
        v += w;
    }
    return v;
}
struct Eight {
    float v[8];
};
__device__ __forceinline__ Eight load8(const float *p) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
    return {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ Eight load8(const uint16_t *p) {
    const u32x4 a = *reinterpret_cast<const u32x4 *>(p);
    Eight r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = bf2f(a[i >> 1] >> (16 * (i & 1)) & 0xffffu);
    return r;
}
__device__ __forceinline__ void store8(float *p, const Eight &x) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{x.v[0], x.v[1], x.v[2], x.v[3]};
    *reinterpret_cast<f32x4 *>(p + 4) = f32x4{x.v[4], x.v[5], x.v[6], x.v[7]};
}
__device__ __forceinline__ void store8(uint16_t *p, const Eight &x) {
    bf16x8 b;
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = (__bf16)x.v[i];
    *reinterpret_cast<bf16x8 *>(p) = b;
}
// eight columns of the row of projections t from column c on, convolved
template <class TR, int TAPS>
__device__ __forceinline__ Eight row8(const Gqa &p, const TR *rows, size_t ld, int pos0, int t, int c, int channels) {
    if (TAPS == 0) return load8(rows + (size_t)t * ld + c);
    Eight r{};
    const int taps = TAPS > 0 ? TAPS : (int)p.taps;
#pragma unroll TAPS > 0 ? TAPS : 1
    for (int k = 0; k < taps; ++k) {
        const int at = t - (taps - 1) + k;
        const Eight f = load8(p.conv + (size_t)k * channels + c);
        Eight x;
        if (at >= 0)
            x = load8(rows + (size_t)at * ld + c);
        else
            for (int i = 0; i < 8; ++i) x.v[i] = raw_value(p, rows, ld, pos0, at, c + i, channels);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = fmaf(f.v[i], x.v[i], r.v[i]);
    }
    return r;
}
// the lane's eight numbers of a vector that L lanes share
template <int L>
__device__ __forceinline__ Kv8Scale eight_numbers(const Eight &x, bool live, u32x2 &numbers) {
    float largest = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = fmaxf(largest, live ? (is_finite(x.v[i]) ? fabsf(x.v[i]) : INFINITY) : 0.f);
    largest = lanes_max<L>(largest);
    const Kv8Scale s = kv8_scale(largest, is_finite(largest));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= (uint32_t)(kv8_number(x.v[4 * h + i], s) & 0xff) << (8 * i);
        numbers[h] = w;
    }
    return s;
}

template <class TR, int KL, int VL, int TAPS, int R, int VP>
__global__ __launch_bounds__(256) void k_kv8_rows(Kv8 c, const TR *rows, size_t ld, const int *pos_ptr, int n, TR *queries, size_t ldq, int blocks, int chunks) {
    constexpr int PITCH = VL * 8 + 4;
    __shared__ uint32_t turned_round[4][VP][PITCH / 4];
    const Gqa &p = c.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pos0 = *pos_ptr, channels = gqa_channels(p);
    const int nq = (int)(p.heads * p.maps), nk = (int)(p.kv_heads * p.maps), dim = (int)p.dim, dimp = (int)p.dimp, vdimp = (int)p.vdimp, heads = p.queries_only ? nq : nq + nk;
    if ((int)blockIdx.x < blocks * chunks) {
        constexpr int AT_ONCE = 64 / KL;
        // (the wave's first token is one for all lanes: places are its own and 32 bits for the lane)
        const int block = blockIdx.x / chunks, chunk = blockIdx.x - block * chunks, h0 = heads * chunk / chunks, h1 = heads * (chunk + 1) / chunks;
        const int col = lane % KL * 8, half = (int)p.rot_dims >> 1, first = (block * 4 + wave) * AT_ONCE * R, left = n - 1 - first, mine = lane / KL;
        const bool live = col < dimp, fours = half % 4 == 0 && (((uintptr_t)p.rope_cos | (uintptr_t)p.rope_sin) & 15) == 0;
        const int at = min(col, dimp - 8);
        if (left < 0) return;
        const TR *src = rows + (size_t)first * ld;
        const float per_dim = 1.0f / (float)dim, *ct = p.rope_cos + (size_t)(pos0 + first) * half, *st = p.rope_sin + (size_t)(pos0 + first) * half, *fac = p.q_factor + pos0 + first;
        Eight x[R], next[R], wv;
        auto fetch = [&](int y) {
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int t = min(mine + u * AT_ONCE, left);
                if (TAPS == 0)
                    next[u] = load8(src + (unsigned)(t * (int)ld + y * dimp + at));
                else
                    next[u] = row8<TR, TAPS>(p, rows, ld, pos0, first + t, y * dimp + at, channels);
            }
        };
        auto weights = [&](const float *w) {
#pragma unroll
            for (int i = 0; i < 8; ++i) wv.v[i] = w && at + i < dim ? w[at + i] : 1.0f;
        };
        fetch(h0);
        weights(h0 < nq ? p.q_weight : p.k_weight);
        f32x4 cs[R], sn[R];
        float factor[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int t = min(mine + u * AT_ONCE, left);
            factor[u] = fac[(unsigned)t];
            if (half) {
                if (fours) {
                    const int pair = t * half + min(at >> 1, half - 4);
                    cs[u] = *reinterpret_cast<const f32x4 *>(ct + (unsigned)pair), sn[u] = *reinterpret_cast<const f32x4 *>(st + (unsigned)pair);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) cs[u][e] = ct[(unsigned)(t * half + min((at >> 1) + e, half - 1))], sn[u][e] = st[(unsigned)(t * half + min((at >> 1) + e, half - 1))];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)  // (pairs past the turned ones: by nothing)
                    if ((at >> 1) + e >= half) cs[u][e] = 1.0f, sn[u][e] = 0.f;
            }
        }
        for (int y = h0; y < h1; ++y) {
            const bool key = y >= nq;
#pragma unroll
            for (int u = 0; u < R; ++u) x[u] = next[u];
            if (y == nq && y > h0) weights(p.k_weight);
            if (y + 1 < h1) fetch(y + 1);
            TR *out = queries + (size_t)first * ldq + (size_t)y * dimp;
            const size_t row0 = (size_t)(y - nq) * p.capacity + pos0 + first;  // (keys)
            int8_t *cache = (int8_t *)p.kcache + row0 * dimp;
            float *scales = c.k_scale + row0;
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const int t = mine + u * AT_ONCE;
                float f = key ? 1.0f : factor[u];
                if ((key ? p.k_weight : p.q_weight) || p.unit_norm) {
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) ss = fmaf(x[u].v[i], x[u].v[i], ss);
                    f *= norm_factor(lanes_sum<KL>(live ? ss : 0.f), per_dim, p.eps);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u].v[i] *= f * wv.v[i];
                if (half)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = x[u].v[2 * e], b = x[u].v[2 * e + 1];
                        x[u].v[2 * e] = turned(a, -b, cs[u][e], sn[u][e]), x[u].v[2 * e + 1] = turned(b, a, cs[u][e], sn[u][e]);
                    }
                if (!key) {
                    if (live && t <= left) store8(out + (unsigned)(t * (int)ldq + col), x[u]);
                    continue;
                }
                u32x2 numbers;
                const Kv8Scale s = eight_numbers<KL>(x[u], live, numbers);
                if (live && t <= left) *reinterpret_cast<u32x2 *>(cache + (unsigned)(t * dimp + col)) = numbers;
                if (col == 0 && t <= left) scales[(unsigned)t] = s.scale;
            }
        }
        return;
    }
    constexpr int AT_ONCE = 64 / VL, ROUNDS = VP / AT_ONCE;
    const int at_block = (int)blockIdx.x - blocks * chunks, block = at_block / (int)p.kv_heads, kv = at_block - block * (int)p.kv_heads, tile = (pos0 / VP + block * 4 + wave) * VP, col = lane % VL * 8, column = (p.values_are_keys ? nq : nq + nk) * dimp + kv * vdimp;
    const bool live = col < vdimp;
    const int at = min(col, vdimp - 8);
    if (tile < pos0 + n) {
        Eight x[ROUNDS];
#pragma unroll
        for (int u = 0; u < ROUNDS; ++u) x[u] = row8<TR, TAPS>(p, rows, ld, pos0, min(max(tile + u * AT_ONCE + lane / VL - pos0, 0), n - 1), column + at, channels);
#pragma unroll
        for (int u = 0; u < ROUNDS; ++u) {
            const int row = u * AT_ONCE + lane / VL, t = tile + row - pos0;
            if (tile + (u + 1) * AT_ONCE <= pos0 || tile + u * AT_ONCE >= pos0 + n) continue;  // (no token of these)
            u32x2 numbers;
            const Kv8Scale s = eight_numbers<VL>(x[u], live, numbers);
            if (col == 0 && t >= 0 && t < n) c.v_scale[(size_t)kv * p.capacity + tile + row] = s.scale;
            turned_round[wave][row][(col >> 2)] = numbers.x, turned_round[wave][row][(col >> 2) + 1] = numbers.y;
        }
    }
    __syncthreads();
    if (tile >= pos0 + n) return;
    uint8_t *dst = (uint8_t *)p.vcache + (size_t)kv * vdimp * p.capacity + (size_t)(tile >> 5) * (32 * vdimp);
    // four columns and the four 16 further on, eight positions: two blocks of four by four bytes each, turned
    for (int i = lane; i < (vdimp >> 3) * (VP / 8); i += 64) {
        const int p8 = i % (VP / 8) * 8, c = i / (VP / 8), c4 = c & 3, c32 = c >> 2, t8 = tile + p8 - pos0;
        uint32_t out[4][4];  // [column][16 bytes: eight positions of it, eight of the one 16 further on]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                uint32_t a[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = turned_round[wave][p8 + 4 * q + e][c32 * 8 + h * 4 + c4];
                const uint32_t l0 = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), l1 = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u);  // (columns 0 and 1 of two positions)
                const uint32_t h0 = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u), h1 = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);  // (2 and 3)
                out[0][2 * h + q] = __builtin_amdgcn_perm(l1, l0, 0x05040100u), out[1][2 * h + q] = __builtin_amdgcn_perm(l1, l0, 0x07060302u);
                out[2][2 * h + q] = __builtin_amdgcn_perm(h1, h0, 0x05040100u), out[3][2 * h + q] = __builtin_amdgcn_perm(h1, h0, 0x07060302u);
            }
        uint8_t *to = dst + (c32 * 16 + c4 * 4) * 64 + ((tile + p8) >> 3 & 3) * 16;
        if (t8 >= 0 && t8 + 8 <= n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<u32x4 *>(to + e * 64) = u32x4{out[e][0], out[e][1], out[e][2], out[e][3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (t8 + (k & 7) >= 0 && t8 + (k & 7) < n) to[e * 64 + k] = (uint8_t)(out[e][k >> 2] >> (8 * (k & 3)));
        }
    }
}

template <class TR, int KL, int VL, int TAPS>
static hipError_t rows_launch(const Kv8 &c, const void *rows, size_t ld, const int *pos, int n, void *q, size_t ldq, hipStream_t s) {
    const Gqa &g = c.g;
    const int heads = (int)(g.heads * g.maps + (g.queries_only ? 0 : g.kv_heads * g.maps)), at_once = 4 * 64 / KL;
    const bool few = n <= at_once;  // (a wave takes its tokens at once, else four times as many in turn)
    const int each = few ? at_once : 4 * at_once, blocks = (n + each - 1) / each;
    const int chunks = std::min(heads, std::max({1, (heads + 7) / 8, 1280 / blocks}));  // (of heads: all of them where the tokens alone fill the chip, up to eight by a wave in turn)
    // values: a wave takes 32 positions where that fills the chip (us of 16384 tokens, by 32 / by eights: 8 heads on 8 of 64 20.9 / 24.3, 12 on 3 of 64 18.6 / 18.1, 20 on 5 of 128 42.5 / 41.7;
    // 1531 tokens of two maps 9.1 / 7.0), else eight
    auto groups = [&](int vp) { return g.queries_only ? 0 : ((n + 2 * vp - 2) / vp + 3) / 4 * (int)g.kv_heads; };  // (n tokens reach into (n + 2 vp - 2) / vp such pieces at most)
    const bool many = !few && groups(32) >= 512;
    // three taps: unrolled for few tokens (us of one, unrolled / looped: 20 heads on 5 of 128 4.3 / 4.7, 16 on 2 of 256 5.2 / 6.0), looped for more (1531: 21 / 16, 27 / 21; 16384: 179 / 145, 276 / 240)
    auto fn = few ? (TAPS < 0 && g.taps == 3 ? k_kv8_rows<TR, KL, VL, TAPS < 0 ? 3 : TAPS, 1, 8> : k_kv8_rows<TR, KL, VL, TAPS, 1, 8>) : many ? k_kv8_rows<TR, KL, VL, TAPS, 4, 32> : k_kv8_rows<TR, KL, VL, TAPS, 4, 8>;
    hipLaunchKernelGGL(fn, dim3((size_t)blocks * chunks + groups(many ? 32 : 8)), dim3(256), 0, s, c, (const TR *)rows, ld, pos, n, (TR *)q, ldq, blocks, chunks);
    return hipGetLastError();
}
// Lanes of a row by its columns (us of 16384 tokens, this / as for wider heads: 64 columns 20.9 / 25.1 with sixteen lanes for the values and 30.7 for both; 64 / 128 of two maps 26.9 / 37.6)
template <class TR, int TAPS>
static hipError_t rows_go(const Kv8 &c, const void *rows, size_t ld, const int *pos, int n, void *q, size_t ldq, hipStream_t s) {
    if (c.g.dimp > 128 || c.g.vdimp > 128) return rows_launch<TR, 32, 32, TAPS>(c, rows, ld, pos, n, q, ldq, s);
    if (c.g.dimp > 64) return rows_launch<TR, 16, 16, TAPS>(c, rows, ld, pos, n, q, ldq, s);
    return c.g.vdimp > 64 ? rows_launch<TR, 8, 16, TAPS>(c, rows, ld, pos, n, q, ldq, s) : rows_launch<TR, 8, 8, TAPS>(c, rows, ld, pos, n, q, ldq, s);
}
template <class TR>
static hipError_t rows_taps(const Kv8 &c, const void *rows, size_t ld, const int *pos, int n, void *q, size_t ldq, hipStream_t s) {
    return c.g.taps == 0 ? rows_go<TR, 0>(c, rows, ld, pos, n, q, ldq, s) : rows_go<TR, -1>(c, rows, ld, pos, n, q, ldq, s);
}
hipError_t launch_kv8_rows(const Kv8 &c, const void *rows, size_t ld, int rows_f32, const int *pos, int n, void *q, size_t ldq, hipStream_t s) {
    return rows_f32 ? rows_taps<float>(c, rows, ld, pos, n, q, ldq, s) : rows_taps<uint16_t>(c, rows, ld, pos, n, q, ldq, s);
}

// ---- positions read back ----------------------------------------------------------------------------------------------
// blockIdx.y: key heads x maps (16 bytes a thread), then value heads (a tile of 32 positions a workgroup, turned round in LDS).
// Bound by memory: 131072 positions of 8 heads of 128 columns as bf16 are 814 MB in 148 us (5.5 TB/s; a copy of as much 5.3, writing alone 6.9); 300 of 3 heads of 80 as f32 3.0.
template <class TO>
__device__ __forceinline__ void store_numbers(TO *dst, uint32_t numbers, float scale) {  // four of them
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)((int)(numbers << (24 - 8 * e)) >> 24) * scale;
    if constexpr (sizeof(TO) == 4)
        *reinterpret_cast<f32x4 *>(dst) = v;
    else
        *reinterpret_cast<bf16x4 *>(dst) = bf16x4{(__bf16)v.x, (__bf16)v.y, (__bf16)v.z, (__bf16)v.w};
}

template <class TO>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8 c, int first, int n, TO *keys, TO *values) {
    __shared__ __attribute__((aligned(16))) uint8_t tile[256 * 32];
    const Gqa &p = c.g;
    const int tid = threadIdx.x, nk = keys ? (int)(p.kv_heads * p.maps) : 0, dimp = (int)p.dimp, vdimp = (int)p.vdimp;
    if ((int)blockIdx.y < nk) {
        const int pieces = dimp >> 4, t_here = tid / pieces, at = (tid - t_here * pieces) * 16, t = (int)blockIdx.x * (256 / pieces) + t_here;  // (whole rows: pieces of all of them may be more than 2^31)
        if (t_here >= 256 / pieces || t >= n) return;
        const size_t row = (size_t)blockIdx.y * p.capacity + first + t;
        const u32x4 v = *reinterpret_cast<const u32x4 *>((const int8_t *)p.kcache + row * dimp + at);
        const float s = c.k_scale[row];
        TO *dst = keys + ((size_t)blockIdx.y * n + t) * dimp + at;
#pragma unroll
        for (int e = 0; e < 4; ++e) store_numbers(dst + 4 * e, v[e], s);
        return;
    }
    const int kv = blockIdx.y - nk, p0 = ((first >> 5) + (int)blockIdx.x) * 32;
    if (p0 >= first + n) return;
    const uint8_t *src = (const uint8_t *)p.vcache + (size_t)kv * vdimp * p.capacity + (size_t)p0 * vdimp;
    for (int i = tid; i < vdimp * 2; i += 256) *reinterpret_cast<u32x4 *>(tile + i * 16) = *reinterpret_cast<const u32x4 *>(src + i * 16);
    __syncthreads();
    const int at = tid >> 3, part = tid & 7, t = p0 + at - first;
    if (t < 0 || t >= n) return;
    const float s = c.v_scale[(size_t)kv * p.capacity + p0 + at];
    TO *dst = values + ((size_t)kv * n + t) * vdimp;
    for (int c0 = 4 * part; c0 < vdimp; c0 += 32) {
        uint32_t v = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) v |= (uint32_t)tile[kv8_value_at(vdimp, at, c0 + e)] << (8 * e);
        store_numbers(dst + c0, v, s);
    }
}

hipError_t launch_kv8_read(const Kv8 &c, int first, int n, void *keys, void *values, int f32, hipStream_t s) {
    const Gqa &g = c.g;
    const int rows = (int)((keys ? g.kv_heads * g.maps : 0) + (values ? g.kv_heads : 0));
    const size_t each = 256 / (g.dimp / 16), blocks = std::max(keys ? (n + each - 1) / each : (size_t)1, values ? ((size_t)n + 62) / 32 : (size_t)1);
    if (f32)
        hipLaunchKernelGGL(k_kv8_read<float>, dim3(blocks, rows), dim3(256), 0, s, c, first, n, (float *)keys, (float *)values);
    else
        hipLaunchKernelGGL(k_kv8_read<uint16_t>, dim3(blocks, rows), dim3(256), 0, s, c, first, n, (uint16_t *)keys, (uint16_t *)values);
    return hipGetLastError();
}

// ---- decode step ------------------------------------------------------------------------------------------------------
// One workgroup per (record, kv head and 16 of its query heads), four waves; a wave takes every fourth block of 32 keys by itself, with maximum, sum and output of its own, and
// the four meet at the end.  S^T = K Q^T on whole numbers: row 4 g + e of score tile t is key 8 g + 4 t + e of the block, so that a lane's weights of both tiles are the eight
// consecutive keys 8 g .. 8 g + 7 which it needs as an operand of O^T = V^T P^T.
// Shares are at most 2^14 (o is held times 2^(14 - above)), in pairs of f16.
// Bound by memory behind many keys: 131072 of 32 heads on 8 of 128 columns are 277 MB in 49 us (5.7 TB/s; reading alone reaches 7.0).  From 63.5 on: neighbouring records joined where a
// launch has more of them than the chip holds workgroups, which saves a second preparation of the queries, 53.4; loads past the caches 47.6 (shares instead of weights under the maximum 1 more).  By latency behind few: 200 keys of 20 heads on 5
// 7.0 us, 2090 of 12 on 3 with two maps of 64 / 128 8.0, 4096 in a window of 16 on 2 of 256 10.5.  A launch is a chain of arguments, position, rows, norms, digits, keys, records: every
// argument is asked for at once and what does not hang on the position ahead of it (7.5, 8.2 and 11.6 without).
struct Kv8StepK {
    const float *row, *q_weight, *k_weight, *q_factor, *rope_cos, *rope_sin, *far_weight, *far_rate;
    const int *pos;
    int8_t *K, *V;
    float *k_scale, *v_scale, *scratch, eps;
    int heads, group, dim, dimp, vdimp, capacity, turned, chunk, window, normed, append, k_at, v_at;  // normed: 1 queries, 2 keys
};
constexpr float kStepDigits = 8355000.0f;  // below 127 (2^16 + 2^8 + 1): three balanced digits

// a load that leaves no copy in the caches on its way, where kPast holds: a cache read once.  131072 keys of one map: 53.4 -> 48.0 us; in the forms that keep one block (two maps,
// heads above 128) 8.0 -> 8.4 and 10.5 -> 11.5
template <bool kPast, class T>
__device__ __forceinline__ T once(const T *p) {
    return kPast ? __builtin_nontemporal_load(p) : *p;
}
constexpr int step_held(int nk, int nv, int maps) { return nv > 8 || nk * maps >= 4 ? 1 : 2; }  // workgroups a compute unit has registers for

template <int NK, int NV, int MAPS>
__global__ __launch_bounds__(256, step_held(NK, NV, MAPS)) void k_kv8_step(Kv8StepK p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t area[];  // digits of the queries [maps][3][16][QS]; then the waves' outputs
    __shared__ float sm[4][MAPS][16], sl[4][MAPS][16], qscale[MAPS][16], news[MAPS + 1];
    __shared__ __attribute__((aligned(16))) int8_t newk[MAPS][NK * 64], newv[NV * 16];
    constexpr int QS = NK * 64 + 32, J = NK, JV = (NV * 16 + 63) / 64, QR = NK > 2 ? 1 : 4;  // QR: rows of a wave at a time
    // (every argument at once: read where they are used they are a chain of scalar loads)
    asm volatile("" ::"s"(p.row), "s"(p.q_weight), "s"(p.k_weight), "s"(p.q_factor), "s"(p.rope_cos), "s"(p.rope_sin), "s"(p.far_weight), "s"(p.far_rate), "s"(p.pos), "s"(p.K), "s"(p.V),
                 "s"(p.k_scale), "s"(p.v_scale), "s"(p.scratch), "s"(p.eps), "s"(p.heads), "s"(p.group), "s"(p.dim), "s"(p.dimp), "s"(p.vdimp), "s"(p.capacity), "s"(p.turned), "s"(p.chunk),
                 "s"(p.window), "s"(p.normed), "s"(p.append), "s"(p.k_at), "s"(p.v_at));
    const int posv = *p.pos;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int kv = blockIdx.x, first_head = blockIdx.y * 16, h0 = kv * p.group + first_head, nh = min(16, p.group - first_head), dimp = p.dimp, vdimp = p.vdimp;
    // What does not hang on the position: rows of queries (head, map), a wave every fourth; the new key of map 3 - wave; the new value, wave 0.
    float x[QR][J], wq[J], wk[J], own[J > JV ? J : JV];
    auto row_of = [&](int i0) {
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const float *src = p.row + (size_t)(h0 * MAPS + min(wave + 4 * (i0 + i), nh * MAPS - 1)) * dimp;
#pragma unroll
            for (int j = 0; j < J; ++j) x[i][j] = lane + 64 * j < dimp ? src[lane + 64 * j] : 0.f;
        }
    };
    row_of(0);
    const bool writes_key = p.append && 3 - wave < MAPS, writes_value = p.append && wave == 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int at = min(lane + 64 * j, p.dim - 1);
        wq[j] = wk[j] = 1.0f;
        if (p.q_weight) wq[j] = p.q_weight[at];
        if (p.k_weight) wk[j] = p.k_weight[at];
    }
    if (writes_value) {
#pragma unroll
        for (int j = 0; j < JV; ++j) own[j] = lane + 64 * j < vdimp ? p.row[p.v_at + kv * vdimp + lane + 64 * j] : 0.f;
    } else if (writes_key) {
#pragma unroll
        for (int j = 0; j < J; ++j) own[j] = lane + 64 * j < dimp ? p.row[p.k_at + (kv * MAPS + 3 - wave) * dimp + lane + 64 * j] : 0.f;
    }
    const int pos = __builtin_amdgcn_readfirstlane(posv), n_keys = pos + 1;
    int first = p.chunk ? pos - (int)((unsigned)pos % (unsigned)p.chunk) : 0;  // gqa_range
    if (p.window && pos - p.window + 1 > first) first = pos - p.window + 1;
    const int base = first & ~(kGqaTile - 1), tiles = (n_keys - base + kGqaTile - 1) / kGqaTile, per = (tiles + kGqaSplits - 1) / kGqaSplits, used = per == 1 ? tiles : (tiles + per - 1) / per;
    // More workgroups than the chip holds at once would each pay for the queries again: neighbouring records become one, and those behind it empty.
    constexpr int kHeld = 256 * step_held(NK, NV, MAPS);
    const int wide = (int)(gridDim.x * gridDim.y) * used, take = wide > 2 * kHeld ? 4 : wide > kHeld ? 2 : 1, record = blockIdx.z * take;
    if (record >= used) return;
    const int k0 = base + record * per * kGqaTile, k1 = min(k0 + take * per * kGqaTile, n_keys);
    int8_t *K = p.K + (size_t)kv * MAPS * p.capacity * dimp, *V = p.V + (size_t)kv * vdimp * p.capacity;
    float *KS = p.k_scale + (size_t)kv * MAPS * p.capacity, *VS = p.v_scale + (size_t)kv * p.capacity;
    // the next block on its way while this one is worked on, where registers allow it; else from the last use of the registers on
    constexpr bool kTwo = NK <= 2 && NV * MAPS <= 8;
    struct Block {
        i32x4 k[2][MAPS][NK];
        u32x4 v[NV / 2];
        f32x4 sk[MAPS][2], sv[2];
    };
    auto fetch_keys = [&](Block &b, int kb) {  // (blocks lie below the capacity, a multiple of 128)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
#pragma unroll
                for (int kk = 0; kk < NK; ++kk)
                    b.k[t][j][kk] = once<kTwo>(reinterpret_cast<const i32x4 *>(K + ((size_t)j * p.capacity + kb + (r16 >> 2) * 8 + t * 4 + (r16 & 3)) * dimp + min(kk * 64 + g * 16, dimp - 16)));
                b.sk[j][t] = *reinterpret_cast<const f32x4 *>(KS + (size_t)j * p.capacity + kb + g * 8 + t * 4);
            }
    };
    auto fetch_values = [&](Block &b, int kb) {
#pragma unroll
        for (int v = 0; v < NV / 2; ++v) b.v[v] = once<kTwo>(reinterpret_cast<const u32x4 *>(V + (size_t)kb * vdimp + min(v, (vdimp >> 5) - 1) * 1024 + r16 * 64 + g * 16));
#pragma unroll
        for (int t = 0; t < 2; ++t) b.sv[t] = *reinterpret_cast<const f32x4 *>(VS + kb + g * 8 + t * 4);
    };
    Block blocks[kTwo ? 2 : 1];
    if (k0 + wave * 32 < k1) fetch_keys(blocks[0], k0 + wave * 32), fetch_values(blocks[0], k0 + wave * 32);
    float cs[J], sn[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        cs[j] = 1.0f, sn[j] = 0.f;
        if (p.turned && 64 * j < p.turned) {
            const size_t at = (size_t)pos * (p.turned >> 1) + (min(lane + 64 * j, p.turned - 1) >> 1);
            cs[j] = p.rope_cos[at], sn[j] = p.rope_sin[at];
        }
    }
    const float factor = p.q_factor[pos];
    // a row of a head, elements lane + 64 j: norm, weight, rotation by pairs of neighbours; the largest of them, INFINITY if one is not finite
    auto finished = [&](float (&x)[J], const float (&weight)[J], bool normed, float factor) {
        float ss = 0.f, largest = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) ss += x[j] * x[j];
        if (normed) factor *= norm_factor(wave_sum(ss), 1.0f / (float)p.dim, p.eps);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = lane + 64 * j;
            x[j] *= factor * (i < p.dim ? weight[j] : 1.0f);
            if (p.turned) {
                const float o = dpp<0xb1>(x[j]);  // quad_perm [1,0,3,2]
                if (i < p.turned) x[j] = turned(x[j], (i & 1) ? o : -o, cs[j], sn[j]);
            }
            largest = fmaxf(largest, is_finite(x[j]) ? fabsf(x[j]) : INFINITY);
        }
        return rows_max(row_max(largest));
    };
    const bool owner = k1 == n_keys && p.append;
    if (owner && writes_value) {
        float largest = 0.f;
#pragma unroll
        for (int i = 0; i < JV; ++i) largest = fmaxf(largest, is_finite(own[i]) ? fabsf(own[i]) : INFINITY);
        largest = rows_max(row_max(largest));
        const Kv8Scale s = kv8_scale(largest, is_finite(largest));
#pragma unroll
        for (int i = 0; i < JV; ++i)
            if (lane + 64 * i < vdimp) {
                const int8_t b = (int8_t)kv8_number(own[i], s);
                V[kv8_value_at(vdimp, pos, lane + 64 * i)] = b;
                newv[lane + 64 * i] = b;
            }
        if (lane == 0) VS[pos] = s.scale, news[MAPS] = s.scale;
    } else if (owner && writes_key) {  // the record that holds the new position appends it (and puts it into its own fragments below)
        const int j = 3 - wave;
        float key[J];
#pragma unroll
        for (int i = 0; i < J; ++i) key[i] = own[i];
        const float largest = finished(key, wk, p.normed & 2, 1.0f);
        const Kv8Scale s = kv8_scale(largest, is_finite(largest));
#pragma unroll
        for (int i = 0; i < J; ++i)
            if (lane + 64 * i < dimp) {
                const int8_t b = (int8_t)kv8_number(key[i], s);
                K[((size_t)j * p.capacity + pos) * dimp + lane + 64 * i] = b;
                newk[j][lane + 64 * i] = b;
            }
        if (lane == 0) KS[(size_t)j * p.capacity + pos] = s.scale, news[j] = s.scale;
    }
    for (int i0 = 0; wave + 4 * i0 < nh * MAPS; i0 += QR) {
        if (i0) row_of(i0);
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const int at = wave + 4 * (i0 + i), hh = at / MAPS, j = at - hh * MAPS;  // (head, map)
            if (at >= nh * MAPS) continue;
            const float largest = finished(x[i], wq, p.normed & 1, factor);
            const bool live = largest >= 1e-30f && is_finite(largest);
            const float to = live ? kStepDigits / largest : 0.f;
            uint8_t *dst = area + (size_t)(j * 3 * 16 + hh) * QS;
#pragma unroll
            for (int e = 0; e < J; ++e) {
                const int v = live ? (int)rintf(x[i][e] * to) : 0, d0 = (int)(int8_t)v, v1 = (v - d0) >> 8, d1 = (int)(int8_t)v1, d2 = (v1 - d1) >> 8;
                dst[lane + 64 * e] = (uint8_t)d0, dst[16 * QS + lane + 64 * e] = (uint8_t)d1, dst[32 * QS + lane + 64 * e] = (uint8_t)d2;
            }
            if (lane == 0) qscale[j][hh] = is_finite(largest) ? largest * (kLog2e / kStepDigits) : __builtin_nanf("");
        }
    }
    __syncthreads();
    constexpr bool kInLds = NK * MAPS > 4;  // (two maps of the largest heads: their queries stay there)
    auto digits = [&](int j, int d, int kk) { return *reinterpret_cast<const i32x4 *>(area + (size_t)((j * 3 + d) * 16 + r16) * QS + kk * 64 + g * 16); };
    i32x4 q[MAPS][3][NK];  // (lanes past the last head: whatever lies there; a column of the products is a head of its own)
    float qs[MAPS];
#pragma unroll
    for (int j = 0; j < MAPS; ++j) {
        qs[j] = qscale[j][r16];
#pragma unroll
        for (int d = 0; d < 3; ++d)
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) q[j][d][kk] = kInLds ? i32x4{0, 0, 0, 0} : digits(j, d, kk);
    }
    FarPenalty far{0.f, 0.f};
    if (p.far_weight) far.weight = p.far_weight[min(h0 + r16, p.heads - 1)], far.rate = p.far_rate[min(h0 + r16, p.heads - 1)];
    f32x4 o[NV][MAPS];
    float m[MAPS], l[MAPS];
#pragma unroll
    for (int j = 0; j < MAPS; ++j) {
        m[j] = -INFINITY, l[j] = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int above = kLeast;
    auto work = [&](int kb, Block &now, Block &then) __attribute__((always_inline)) {
        const bool more = kb + 128 < k1;
        if (kTwo && more) fetch_keys(then, kb + 128), fetch_values(then, kb + 128);
        if (kb + 32 <= first) {  // (another chunk's keys)
            if (!kTwo && more) fetch_keys(then, kb + 128), fetch_values(then, kb + 128);
            return;
        }
        auto &kf = now.k;
        auto &vf = now.v;
        auto &sk = now.sk;
        auto &sv = now.sv;
        if (owner && pos - kb < 32) {  // the new position, which memory need not show yet
            const int at = pos - kb, t = (at >> 2) & 1;
            const bool mine = r16 == (at >> 3) * 4 + (at & 3);
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
#pragma unroll
                for (int kk = 0; kk < NK; ++kk) {
                    const i32x4 k = *reinterpret_cast<const i32x4 *>(&newk[j][min(kk * 64 + g * 16, dimp - 16)]);
                    if (mine && t == 0) kf[0][j][kk] = k;
                    if (mine && t == 1) kf[1][j][kk] = k;
                }
            }
            if (g == at >> 3) {
                const uint32_t sh = (at & 3) * 8, keep = ~(0xffu << sh);
#pragma unroll
                for (int v = 0; v < NV / 2; ++v)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t b = (uint32_t)(uint8_t)newv[min(v * 32 + half * 16 + r16, vdimp - 16 + r16)] << sh;
                        if ((at >> 2 & 1) == 0) vf[v][2 * half] = (vf[v][2 * half] & keep) | b;
                        if ((at >> 2 & 1) == 1) vf[v][2 * half + 1] = (vf[v][2 * half + 1] & keep) | b;
                    }
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e == (at & 7)) {
#pragma unroll
                        for (int j = 0; j < MAPS; ++j) sk[j][e >> 2][e & 3] = news[j];
                        sv[e >> 2][e & 3] = news[MAPS];
                    }
            }
        }
        const bool whole = kb >= first && kb + 32 <= k1;
        auto seen = [&](int t, int e) { return kb + g * 8 + t * 4 + e < k1 && kb + g * 8 + t * 4 + e >= first; };
        if (!whole)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) sv[t][e] = seen(t, e) ? sv[t][e] : 0.f;
        const float largest = fmaxf(fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[0][2], sv[0][3])), fmaxf(fmaxf(sv[1][0], sv[1][1]), fmaxf(sv[1][2], sv[1][3])));
        const int need = __builtin_amdgcn_readfirstlane(exponent_above(rows_max(largest), kLeast));
        if (need > above) {
            const int less = need - above;
            above = need;
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
                const int moved = room_for(rows_sum(l[j]), less);
                const float down = power2(moved - less);
                m[j] -= (float)moved, l[j] *= power2(moved);
#pragma unroll
                for (int v = 0; v < NV; ++v) o[v][j] *= down;
            }
        }
        f32x4 factor[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) factor[t][e] = __builtin_amdgcn_ldexpf(sv[t][e], 14 - above);
        f16x8 hi[MAPS], lo[MAPS];
#pragma unroll
        for (int j = 0; j < MAPS; ++j) {
            f32x4 s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                i32x4 a[3];
#pragma unroll
                for (int d = 0; d < 3; ++d) {
                    a[d] = i32x4{0, 0, 0, 0};
#pragma unroll
                    for (int kk = 0; kk < NK; ++kk) a[d] = mfma_i8(kf[t][j][kk], kInLds ? digits(j, d, kk) : q[j][d][kk], a[d]);  // (columns past dimp: the query is zero there)
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] = fmaf((float)a[2][e], 65536.0f, fmaf((float)a[1][e], 256.0f, (float)a[0][e])) * (sk[j][t][e] * qs[j]);  // (qs holds log2(e))
                    if (MAPS == 1 && p.far_weight) s[t][e] = nearer(s[t][e], far, pos - (kb + g * 8 + t * 4 + e));
                }
            }
            if (!whole)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][e] = seen(t, e) ? s[t][e] : -INFINITY;
            float mx = -INFINITY;  // (of shares)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[t][e] + factor_exponent(factor[t][e], 14));
            mx = fmaxf(m[j], rows_max(mx));
            if (__any(mx > m[j] || mx == -INFINITY)) {
                if (mx == -INFINITY) mx = 0.f;  // (no score is a number: neither is the sum)
                const float al = __builtin_amdgcn_exp2f(m[j] - mx);
                m[j] = mx;
                l[j] *= al;
#pragma unroll
                for (int v = 0; v < NV; ++v) o[v][j] *= al;
            }
            f32x4 w[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[t][e] = __builtin_amdgcn_exp2f(s[t][e] - mx);
            l[j] += ((w[0][0] + w[0][1]) + (w[0][2] + w[0][3])) + ((w[1][0] + w[1][1]) + (w[1][2] + w[1][3]));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float x = w[t][e] * factor[t][e], y = w[t][e + 1] * factor[t][e + 1];
                    // (an instruction by name: left to itself the compiler rounds the product once for the products and another time for what is left of it)
                    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
                    hi[j][4 * t + e] = h.x, hi[j][4 * t + e + 1] = h.y;
                    lo[j][4 * t + e] = (_Float16)(x - (float)h.x), lo[j][4 * t + e + 1] = (_Float16)(y - (float)h.y);
                }
        }
        if (!kTwo && more) fetch_keys(then, kb + 128);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const f16x8 a = eight_f16(vf[v / 2][2 * (v & 1)], vf[v / 2][2 * (v & 1) + 1]);
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
                o[v][j] = mfma_f16(a, hi[j], o[v][j]);
                o[v][j] = mfma_f16(a, lo[j], o[v][j]);
            }
        }
        if (!kTwo && more) fetch_values(then, kb + 128);
    };
    for (int kb = k0 + wave * 32; kb < k1; kb += kTwo ? 256 : 128) {
        work(kb, blocks[0], blocks[kTwo ? 1 : 0]);
        if (kTwo && kb + 128 < k1) work(kb + 128, blocks[kTwo ? 1 : 0], blocks[0]);
    }
#pragma unroll
    for (int j = 0; j < MAPS; ++j) {
        const float t = rows_sum(l[j]);
        if (g == 0) sm[wave][j][r16] = m[j], sl[wave][j][r16] = t;
    }
    __syncthreads();
    float *outs = reinterpret_cast<float *>(area);
#pragma unroll
    for (int j = 0; j < MAPS; ++j) {
        const float M = fmaxf(fmaxf(sm[0][j][r16], sm[1][j][r16]), fmaxf(sm[2][j][r16], sm[3][j][r16]));
        const float w = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[j] - M);
        if (r16 < nh)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (v * 16 < vdimp) {
                    f32x4 t;
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_ldexpf(o[v][j][e], above - 14) * w;
                    *reinterpret_cast<f32x4 *>(outs + ((size_t)(wave * MAPS + j) * nh + r16) * vdimp + v * 16 + g * 4) = t;
                }
    }
    __syncthreads();
    const int n_rows = MAPS * nh;
    for (int r = tid >> 5; r < n_rows; r += 8) {
        const int j = MAPS == 2 && r >= nh ? 1 : 0, hh = r - j * nh;
        float *rec = p.scratch + ((size_t)((h0 + hh) * MAPS + j) * kGqaSplits + record) * (kGqaRecHead + vdimp);
        for (int e = 1; e < min(take, used - record); ++e) {
            float *empty = rec + (size_t)e * (kGqaRecHead + vdimp);
            for (int c = (tid & 31) * 4; c < vdimp; c += 128) *reinterpret_cast<f32x4 *>(empty + kGqaRecHead + c) = f32x4{0.f, 0.f, 0.f, 0.f};
            if ((tid & 31) == 0) empty[0] = -INFINITY, empty[1] = 0.f;
        }
        for (int c = (tid & 31) * 4; c < vdimp; c += 128) {
            const float *src = outs + (size_t)r * vdimp + c;
            const size_t step = (size_t)n_rows * vdimp;
            *reinterpret_cast<f32x4 *>(rec + kGqaRecHead + c) = (*reinterpret_cast<const f32x4 *>(src) + *reinterpret_cast<const f32x4 *>(src + step)) +
                                                                (*reinterpret_cast<const f32x4 *>(src + 2 * step) + *reinterpret_cast<const f32x4 *>(src + 3 * step));
        }
        if ((tid & 31) == 0) {
            const float M = fmaxf(fmaxf(sm[0][j][hh], sm[1][j][hh]), fmaxf(sm[2][j][hh], sm[3][j][hh]));
            float L = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) L += sm[w][j][hh] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[w][j][hh] - M) * sl[w][j][hh];
            rec[0] = M, rec[1] = L;
        }
    }
}

template <int NK, int NV>
static hipError_t step_go(const Kv8 &c, const GqaStep &a, hipStream_t s) {
    const Gqa &g = c.g;
    const int splits = gqa_records(g), group = (int)(g.heads / g.kv_heads), nh = min(16, group);
    const size_t queries = g.maps * 3 * 16 * (NK * 64 + 32), outs = 4 * g.maps * nh * g.vdimp * sizeof(float), lds = queries > outs ? queries : outs;
    auto fn = g.maps == 2 ? k_kv8_step<NK, NV, 2> : k_kv8_step<NK, NV, 1>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    Kv8StepK k;
    k.row = a.row, k.q_weight = g.q_weight, k.k_weight = g.k_weight, k.q_factor = g.q_factor, k.rope_cos = g.rope_cos, k.rope_sin = g.rope_sin, k.far_weight = g.far_weight;
    k.far_rate = g.far_rate, k.pos = a.pos, k.K = (int8_t *)g.kcache, k.V = (int8_t *)g.vcache, k.k_scale = c.k_scale, k.v_scale = c.v_scale, k.scratch = a.scratch, k.eps = g.eps;
    k.heads = (int)g.heads, k.group = group, k.dim = (int)g.dim, k.dimp = (int)g.dimp, k.vdimp = (int)g.vdimp, k.capacity = (int)g.capacity, k.turned = (int)g.rot_dims;
    k.append = !g.queries_only;
    k.chunk = g.chunk < g.capacity ? (int)g.chunk : 0, k.window = g.window < g.capacity ? (int)g.window : 0;  // (as large as the cache: no position has keys outside)
    k.normed = (g.q_weight || g.unit_norm ? 1 : 0) | (g.k_weight || g.unit_norm ? 2 : 0);
    k.k_at = (int)(g.heads * g.maps * g.dimp), k.v_at = g.values_are_keys ? k.k_at : (int)((g.heads + g.kv_heads) * g.maps * g.dimp);
    hipLaunchKernelGGL(fn, dim3(g.kv_heads, (group + 15) / 16, splits), dim3(256), lds, s, k);
    return hipGetLastError();
}

hipError_t launch_kv8_step(const Kv8 &c, const GqaStep &a, hipStream_t s) {
    const Gqa &g = c.g;
    if (!gqa_supported((int)g.dimp, (int)g.vdimp)) return hipErrorInvalidValue;
    if (g.dimp <= 64 && g.vdimp <= 64) return step_go<1, 4>(c, a, s);
    if (g.dimp <= 64 && g.vdimp <= 128) return step_go<1, 8>(c, a, s);
    if (g.dimp <= 128 && g.vdimp <= 128) return step_go<2, 8>(c, a, s);
    return step_go<4, 16>(c, a, s);
}

// ---- prompt -----------------------------------------------------------------------------------------------------------
constexpr int kv8_tile_bytes(int nk, int nv, int maps) { return maps * 64 * (nk * 128 + 32) + nv * 16 * (64 * 2 + 32); }
// Weights are exp2(score - m) times 2^kWeightUp, and m follows the largest share once that may be kLazy above it: shares are at most 2^14, and a query's largest is 2^5 or more, so that an f16
// holds 11 bits of all that are 2^-19 of it.
constexpr float kWeightUp = 6.0f, kLazy = 8.0f, kLittle = 2.0f;

// One workgroup: the rows of W waves, a row being a query of one head; the heads that share keys and values are neighbours among the rows (row r: query r / group, head r % group of
// the kv head).  A wave holds two slots of 16 rows: both maps of one set of rows, or two sets of the only map.  Key tiles of 64 (every map's) and the values of a tile are staged
// through registers into LDS.  G = 2: two such groups of W waves share the keys of the same rows, tile by tile in turn, and meet in LDS at the end.  records: gridDim.y workgroups
// share a block's tiles of keys, in stretches (launch_gqa_merge_parts).  MAPS = 1 with two maps, whose keys together find no room in LDS: gridDim.z is the map, with records.
// In LDS keys are their numbers + 1152 as f16 (exact; a row's sum times 1152 is what its scores start from), and so is a query of bf16 times a power of two: scores are exact but
// for the f32 sums (partial sums up to ten times the size that the numbers alone would have, 2^-20 of it together), a key's scale meets them in f32.  Values are their numbers (exact in f16), and a weight times its value's factor is rounded to f16 once, to the nearest
// (2^-11 of it at most, 1.5e-4 of an output that is rounded to 2^-8 afterwards; f16 pairs would double these products).
// The products of a SIMD's two waves and their vector instructions take about the same time, and as phases of their own they add up: hence the next tile's scores are made among
// this tile's exponentials, and this tile's outputs among the staging of the tiles to come.
// Bound by both pipes of a SIMD: 8192 tokens of 20 heads on 5 of 128 columns, 344 GFLOP, take 422 us (0.82 PFLOP/s, a large product of f16 reaches 1.35; over a cache of bf16 k_gqa_prefill
// takes 530); 509 tokens behind 20011 of 12 heads on 3 with two maps of 64 / 128 149 us (0.64), 130 tokens of 12 heads 12.5.  Phases one behind the other, two groups of four waves: 515,
// 226, 11.5.
// One barrier a tile: what is read and written between two of them is in kv8_schedule.hpp.
// Wave 0 makes the values' factors a tile ahead, wave 1 the keys' scales two.  A value without a scale takes its key's away instead, so that only queries that see it lose theirs.
// LDS of a tile: keys [maps][64][KS], values [columns][VS]; the 32 bytes behind a row of values hold the keys' scales (rows 16 s + 8 map .., s = 0
// and 1 in turn), the factors (32 ..) and their exponents (40).
// FAR: with a distance penalty, gates per column, or both.
template <int NK, int NV, int MAPS, bool FAR, int G, int W>
__global__ __launch_bounds__(64 * W * G, NV > 8 || NK > 2 || (NK == 2 && MAPS == 2 && W == 4) ? 1 : 2) void k_kv8_prefill(Kv8 c, const uint16_t *Q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, int n_qb, float *records) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int SLOTS = 2, QW = 16 * SLOTS / MAPS, KK = 2 * NK, KS = NK * 128 + 32, VS = 64 * 2 + 32, T = 64 * W, KC = NK * 4, KR = T / KC, NKL = (MAPS * 64 + KR - 1) / KR, NVL = (NV * 64 + T - 1) / T;
    constexpr int KB = MAPS * 64 * KS, TILE = kv8_tile_bytes(NK, NV, MAPS), PAD = KB + 128;
    const Gqa &p = c.g;
    const int grp = G == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x / T) : 0, tid = threadIdx.x & (T - 1), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    uint8_t *lk = lds + grp * 2 * TILE;
    const int heads = (int)p.heads, kv_heads = (int)p.kv_heads, group = heads / kv_heads, dimp = (int)p.dimp, vdimp = (int)p.vdimp;
    // longest blocks first; consecutive workgroups go to the eight XCDs in turn
    const int level = blockIdx.x / kv_heads, kv = blockIdx.x - level * kv_heads, qb = n_qb - 1 - level, maps = MAPS == 1 ? (int)p.maps : MAPS, alone = MAPS == 1 ? (int)blockIdx.z : 0;
    const int pos0 = n_ctx - nq, row0 = qb * W * QW, rw = row0 + wave * QW, last = nq - 1;
    const int q_lo = min(rw / group, last), q_hi = min((rw + QW - 1) / group, last), q_first = row0 / group, q_last = min((row0 + W * QW - 1) / group, last);
    f16x8 qf[SLOTS][KK];
    float qs[SLOTS], raised[SLOTS], m[SLOTS], l[SLOTS];
    FarPenalty far[SLOTS / MAPS];
    int qpos[SLOTS], qfirst[SLOTS], head[SLOTS / MAPS];
    f32x4 o[NV][SLOTS];
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) {
        const int at = rw + t / MAPS * 16 + r16, qi = min(at / group, last), h = kv * group + at % group, map = alone + t % MAPS;
        head[t / MAPS] = h, qpos[t] = pos0 + qi, qfirst[t] = gqa_first(p, qpos[t]);
        const uint16_t *q = Q + (size_t)qi * ldq + (size_t)(h * maps + map) * dimp;
        float largest = 0.f, total = 0.f, v[KK][8];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const u32x4 raw = kk * 32 < dimp ? *reinterpret_cast<const u32x4 *>(q + kk * 32 + g * 8) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[kk][i] = bf2f(raw[i >> 1] >> (16 * (i & 1)) & 0xffffu);
                largest = fmaxf(largest, is_finite(v[kk][i]) ? fabsf(v[kk][i]) : INFINITY);
            }
        }
        largest = rows_max(largest);
        const int e = exponent_above(largest, -100);
        qs[t] = is_finite(largest) ? kLog2e * power2(e - 12) : __builtin_nanf("");
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                qf[t][kk][i] = (_Float16)(is_finite(largest) ? __builtin_amdgcn_ldexpf(v[kk][i], 12 - e) : 0.f);
                total += (float)qf[t][kk][i];
            }
        raised[t] = -1152.0f * rows_sum(total);
        // (finite: with chunks a tile may hold no key that a query sees)
        m[t] = -1e30f;
        if (FAR && MAPS == 1) far[t] = far_penalty(p, h), far[t].weight *= kLog2e;
        l[t] = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int8_t *K = (const int8_t *)p.kcache + (size_t)(kv * maps + alone) * p.capacity * dimp, *V = (const int8_t *)p.vcache + (size_t)kv * vdimp * p.capacity;
    const float *KSC = c.k_scale + (size_t)(kv * maps + alone) * p.capacity, *VSC = c.v_scale + (size_t)kv * p.capacity;
    // keys: a row of the tile by KC neighbouring threads; row p of 32 in LDS is key 8 (p >> 2 & 3) + 4 (p >> 4) + (p & 3)
    u32x4 kreg[NKL], vreg[NVL];
    float kscale[MAPS], vscale = 0.f, vnan = 0.f;
    int kw[NKL], vw[NVL], voff[NVL];
    unsigned koff[NKL];
#pragma unroll
    for (int j = 0; j < NKL; ++j) {
        const int at = min(tid / KC + j * KR, MAPS * 64 - 1), key = at & 63, mp = at >> 6, row = (key & 32) + (key >> 2 & 1) * 16 + (key >> 3 & 3) * 4 + (key & 3);
        kw[j] = (mp * 64 + row) * KS + (tid % KC) * 32;
        koff[j] = (unsigned)(key * dimp + min((tid % KC) * 16, dimp - 16));
    }
#pragma unroll
    for (int j = 0; j < NVL; ++j) {  // sixteen bytes: eight keys of two columns, 16 apart; columns past vdimp are zero
        const int i = tid + T * j, half = i / (NV * 32) & 1, rem = i % (NV * 32), key = half * 32 + (rem & 3) * 8;
        vw[j] = KB + ((rem >> 6) * 32 + (rem >> 2 & 15)) * VS + key * 2;
        voff[j] = (rem >> 6) * 32 < vdimp ? half * vdimp * 32 + rem * 16 : -1;
        vreg[j] = u32x4{0u, 0u, 0u, 0u};
    }
    int t_first = gqa_first(p, pos0 + q_first) >> 6, n_tiles = (pos0 + q_last) / 64 + 1;
    const int w_last = gqa_first(p, pos0 + q_hi);
    if (records) {
        const int each = (n_tiles - t_first + (int)gridDim.y - 1) / (int)gridDim.y;
        t_first = min(t_first + (int)blockIdx.y * each, n_tiles), n_tiles = min(t_first + each, n_tiles);
    }
    const int end = n_tiles * 64 - 1;
    // The group's i-th tile; what lies past the last one is read from the last one, and all of it hidden.
    auto first_key = [&](int i) { return max(min(t_first + grp + G * i, n_tiles - 1), 0) * 64; };
    constexpr bool whole_keys = NKL * KR == MAPS * 64, whole_values = NVL * T == NV * 64;
    // which half of a tile a wave's j-th piece of the keys belongs to
    auto half_of = [&](int j) { return (KR < 64 ? j * KR : wave * (64 / KC)) >> 5 & 1; };
    constexpr Kv8Schedule ahead_by = kKv8Schedule;
    auto keys_ahead = [&](int j) { return half_of(j) ? ahead_by.keys[1] : ahead_by.keys[0]; };
    auto fetch_keys = [&](int i, int j) {  // (whole tiles: the capacity is a multiple of 64)
        const int mp = MAPS == 1 ? 0 : (tid / KC + j * KR) >> 6 & 1;
        if (whole_keys || tid / KC + j * KR < MAPS * 64) kreg[j] = *reinterpret_cast<const u32x4 *>(K + ((size_t)mp * p.capacity + first_key(i)) * dimp + koff[j]);
    };
    auto fetch_scales = [&](int i) {
        const int key0 = first_key(i);
        if (wave == 1) {
            const bool in = key0 + lane < n_ctx;  // (a position past the portion may hold anything)
#pragma unroll
            for (int mp = 0; mp < MAPS; ++mp) kscale[mp] = in ? KSC[(size_t)mp * p.capacity + key0 + lane] : 0.f;
            vnan = in ? VSC[key0 + lane] : 0.f;
        }
    };
    auto fetch_values = [&](int i) {
        const int8_t *vb = V + (size_t)first_key(i) * vdimp;
#pragma unroll
        for (int j = 0; j < NVL; ++j)
            if (voff[j] >= 0 && (whole_values || tid + T * j < NV * 64)) vreg[j] = *reinterpret_cast<const u32x4 *>(vb + voff[j]);
    };
    auto fetch_factors = [&](int i) {
        if (wave == 0) {
            const int key0 = first_key(i);
            vscale = key0 + lane < n_ctx ? VSC[key0 + lane] : 0.f;
        }
    };
    int highest = kLeast;
    auto publish = [&](int i) {  // the factors of tile i, the exponent that they are without, and how far below it they all are
        if (wave == 0) {
            const float v = fmaxf(vscale, 0.f);
            const int here = __builtin_amdgcn_readfirstlane(exponent_above(rows_max(row_max(v)), kLeast));
            highest = max(highest, here);
            uint8_t *dst = lk + (i & 1) * TILE + PAD + 32 * VS;
            *reinterpret_cast<float *>(dst + (lane >> 3) * VS + (lane & 7) * 4) = __builtin_amdgcn_ldexpf(v, -highest);
            if (lane == 0) *reinterpret_cast<int2 *>(dst + 8 * VS) = int2{highest, max(here - highest, kBelow)};
        }
    };
    // stores go by pieces of eight numbers a thread, 2 NKL and 2 NVL of them
    auto store_keys = [&](int i, int u) {
        uint8_t *dst = lk + (i & 1) * TILE;
        const int j = u >> 1;
        if (whole_keys || tid / KC + j * KR < MAPS * 64)
            *reinterpret_cast<f16x8 *>(dst + kw[j] + (u & 1) * 16) = u & 1 ? eight_raised(kreg[j].z, kreg[j].w) : eight_raised(kreg[j].x, kreg[j].y);
    };
    auto store_scales = [&](int i) {
        uint8_t *dst = lk + (i & 1) * TILE;
        if (wave == 1)
#pragma unroll
            for (int mp = 0; mp < MAPS; ++mp)
                *reinterpret_cast<float *>(dst + PAD + ((i >> 1 & 1) * 16 + 8 * mp + (lane >> 3)) * VS + (lane & 7) * 4) = vnan == vnan ? kscale[mp] : vnan;
    };
    auto store_values = [&](int i, int u) {
        const int j = u >> 1;
        if (whole_values || tid + T * j < NV * 64)
            *reinterpret_cast<f16x8 *>(lk + (i & 1) * TILE + vw[j] + (u & 1) * 16 * VS) = u & 1 ? eight_f16(vreg[j].z, vreg[j].w) : eight_f16(vreg[j].x, vreg[j].y);
    };
    const int steps = (n_tiles - t_first + G - 1) / G;
    // what the first iteration finds: keys 0 .. 31 of tiles 0 and 1 and 32 .. 63 of tile 0, their tiles' scales, values and factors of tile 0
    static_assert(ahead_by.keys[0] == 2 && ahead_by.keys[1] == 1 && ahead_by.scales == 2 && ahead_by.values == 1 && ahead_by.factors == 1 && ahead_by.slots == 2, "what the prologue leaves");
#pragma unroll
    for (int j = 0; j < NKL; ++j) fetch_keys(0, j);
    fetch_scales(0), fetch_values(0), fetch_factors(0);
    publish(0);
    fetch_factors(1);
#pragma unroll
    for (int u = 0; u < 2 * NKL; ++u) store_keys(0, u);
    store_scales(0);
#pragma unroll
    for (int j = 0; j < NKL; ++j) fetch_keys(1, j);
    fetch_scales(1);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2 * NVL; ++u) store_values(0, u);
    fetch_values(1);
#pragma unroll
    for (int u = 0; u < 2 * NKL; ++u)
        if (half_of(u >> 1) == 0) store_keys(1, u);
    store_scales(1);
#pragma unroll
    for (int j = 0; j < NKL; ++j)
        if (half_of(j) == 0) fetch_keys(2, j);
    fetch_scales(2);
    // Scores go by halves of a tile (32 keys): of the half at hand and of the next one, times their keys' scales, in units of qs, which holds log2(e).
    f32x4 s0[2][SLOTS], s1[2][SLOTS];
    float mx[SLOTS];  // the largest of the lane's
    constexpr int KREADS = 2 * KK * MAPS, AHEAD = 4;
    // operand j of a half's scores, and what it is multiplied with
    auto key_operand = [&](const uint8_t *tile, int half, int j) {
        const int kk = j / (2 * MAPS), kt = j / MAPS % 2, mp = j % MAPS;
        return *reinterpret_cast<const f16x8 *>(tile + (mp * 64 + half * 32 + kt * 16 + r16) * KS + kk * 64 + g * 16);
    };
    auto key_products = [&](const f16x8 &k, int j, f32x4 (&to)[2][SLOTS]) {
        const int kk = j / (2 * MAPS), kt = j / MAPS % 2, mp = j % MAPS;
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            if (MAPS == 2 && t != mp) continue;
            if (kk == 0) to[kt][t] = f32x4{raised[t], raised[t], raised[t], raised[t]};
            to[kt][t] = mfma_f16(k, qf[t][kk], to[kt][t]);
        }
    };
    auto value_operand = [&](const uint8_t *tile, int half, int j) { return *reinterpret_cast<const f16x8 *>(tile + KB + (j * 16 + r16) * VS + half * 64 + g * 16); };
    // the j-th quarter of a half's scores: their keys' scales and the largest
    auto scaled = [&](const uint8_t *tile, int i, int half, int j, f32x4 (&of)[2][SLOTS]) {
        const int kt = j / SLOTS, t = j % SLOTS;
        of[kt][t] *= *reinterpret_cast<const f32x4 *>(tile + PAD + ((i >> 1 & 1) * 16 + 8 * (t % MAPS) + half * 4 + g) * VS + kt * 16);
        mx[t] = kt == 0 ? max3(of[kt][t][0], of[kt][t][1], of[kt][t][2]) : max3(mx[t], of[kt][t][0], of[kt][t][1]);
        mx[t] = kt == 0 ? max3(mx[t], of[kt][t][3], of[kt][t][3]) : max3(mx[t], of[kt][t][2], of[kt][t][3]);
    };
#pragma unroll
    for (int j = 0; j < KREADS; ++j) key_products(key_operand(lk, 0, j), j, s0);
#pragma unroll
    for (int j = 0; j < 4; ++j) scaled(lk, 0, 0, j, s0);
    int above = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int *>(lk + PAD + 40 * VS));
    // half `half` of tile i, its scores in s; the half behind it, of tile ni, into ahead
    auto step = [&](int i, int half, int2 need, f32x4 (&s)[2][SLOTS], f32x4 (&ahead)[2][SLOTS]) __attribute__((always_inline)) {
        const int key0 = (t_first + grp + G * i) * 64 + half * 32, ni = i + half, other = half ^ 1;
        const uint8_t *here = lk + (i & 1) * TILE, *next = lk + (ni & 1) * TILE;
        if (key0 + 31 > min(pos0 + q_lo, end) || key0 < w_last || (FAR && p.far_weight))  // (the diagonal or what lies past the last tile; an earlier chunk of some of the queries)
#pragma unroll
            for (int t = 0; t < SLOTS; ++t) {
                mx[t] = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + g * 8 + kt * 4 + e;
                        float v = s[kt][t][e];
                        if (FAR && p.far_weight) v = nearer(v * qs[t], far[t / MAPS], max(qpos[t] - key, 0));
                        s[kt][t][e] = v = key > min(qpos[t], end) || key < qfirst[t] ? -INFINITY : v;
                        mx[t] = fmaxf(mx[t], v);
                    }
            }
        float c2[SLOTS];
        auto factors = [&](int kt) { return *reinterpret_cast<const f32x4 *>(here + PAD + (32 + half * 4 + g) * VS + kt * 16); };
        bool grows = need.x > above;
        const float most = kLazy - (float)need.y;
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            c2[t] = FAR && p.far_weight ? 1.0f : qs[t];
            grows = grows || mx[t] * c2[t] > m[t] + most;
        }
        if (__any(grows)) {
            const int less = max(need.x - above, 0);  // (factors from here on are 2^-less of what they would have been)
            above = max(above, need.x);
            float e[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) e[kt][i] = factor_exponent(factors(kt)[i], 0);
#pragma unroll
            for (int t = 0; t < SLOTS; ++t) {
                float largest = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) largest = fmaxf(largest, fmaf(s[kt][t][i], c2[t], e[kt][i]));
                largest = rows_max(largest);
                const int moved = room_for(rows_sum(l[t]), less);
                const float from = m[t] - (float)moved, to = largest > from + kLittle ? largest : from, al = __builtin_amdgcn_exp2f(from - to), down = power2(moved - less);
                m[t] = to;
                l[t] *= al * power2(moved);
#pragma unroll
                for (int v = 0; v < NV; ++v) o[v][t] *= al * down;
            }
        }
        u32x4 w[SLOTS];
        {
            // (scores in place and factors read again: what the compiler would keep of both across the branch costs up to 160 registers)
            asm volatile("" : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1])::"memory");
            const f32x4 vs[2] = {factors(0), factors(1)};
            f16x8 k[KREADS];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) k[j] = key_operand(next, other, j);
#pragma unroll
            for (int j = 0; j < KREADS; ++j) {
                __builtin_amdgcn_sched_barrier(0);
                if (j + AHEAD < KREADS) k[j + AHEAD] = key_operand(next, other, j + AHEAD);
                key_products(k[j], j, ahead);
#pragma unroll
                for (int u = j * 8 / KREADS; u < (j + 1) * 8 / KREADS; ++u) {  // two weights
                    const int t = u % SLOTS, e = u / SLOTS;
                    const float off = kWeightUp - m[t];
                    const float a = __builtin_amdgcn_exp2f(fmaf(s[e >> 1][t][2 * e & 3], c2[t], off)), b = __builtin_amdgcn_exp2f(fmaf(s[e >> 1][t][(2 * e & 3) + 1], c2[t], off));
                    l[t] += a + b;
                    w[t][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a * vs[e >> 1][2 * e & 3], b * vs[e >> 1][(2 * e & 3) + 1]}), f16x2));
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        {
            f16x8 v[NV];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) v[j] = value_operand(here, half, j);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                __builtin_amdgcn_sched_barrier(0);
                if (j + AHEAD < NV) v[j + AHEAD] = value_operand(here, half, j + AHEAD);
#pragma unroll
                for (int t = 0; t < SLOTS; ++t) o[j][t] = mfma_f16(v[j], __builtin_bit_cast(f16x8, w[t]), o[j][t]);
#pragma unroll
                for (int u = j * 4 / NV; u < (j + 1) * 4 / NV; ++u) scaled(next, ni, other, u, ahead);
                constexpr int VP = 2 * NVL, KP = 2 * NKL;
#pragma unroll
                for (int u = j * VP / NV; half == 0 && u < (j + 1) * VP / NV; ++u) store_values(i + ahead_by.values, u);
#pragma unroll
                for (int u = j * KP / NV; half == 1 && u < (j + 1) * KP / NV; ++u) store_keys(i + keys_ahead(u >> 1), u);
            }
            if (half == 0) {
                fetch_values(i + ahead_by.values + 1);
            } else {
                store_scales(i + ahead_by.scales);
#pragma unroll
                for (int u = 0; u < NKL; ++u) fetch_keys(i + keys_ahead(u) + 1, u);
                fetch_scales(i + ahead_by.scales + 1);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    for (int i = 0; i < steps; ++i) {
        __syncthreads();
        publish(i + ahead_by.factors);
        fetch_factors(i + ahead_by.factors + 1);
        const int2 both = *reinterpret_cast<const int2 *>(lk + (i & 1) * TILE + PAD + 40 * VS);
        const int2 need{__builtin_amdgcn_readfirstlane(both.x), __builtin_amdgcn_readfirstlane(both.y)};
        step(i, 0, need, s0, s1);
        step(i, 1, need, s1, s0);
    }
    float sum[SLOTS];
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) {
        const float back = power2(above - (int)kWeightUp);
        sum[t] = rows_sum(l[t]) * power2(-(int)kWeightUp);
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v][t] *= back;
    }
    if (G == 2) {
        f32x4 *po = reinterpret_cast<f32x4 *>(lds);                                       // [wave][slot][NV][lane]
        float2 *pm = reinterpret_cast<float2 *>(lds + (size_t)W * SLOTS * NV * 64 * 16);  // [wave][slot][lane]
        __syncthreads();
        if (grp == 1) {
#pragma unroll
            for (int t = 0; t < SLOTS; ++t) {
#pragma unroll
                for (int v = 0; v < NV; ++v) po[((wave * SLOTS + t) * NV + v) * 64 + lane] = o[v][t];
                pm[(wave * SLOTS + t) * 64 + lane] = float2{m[t], sum[t]};
            }
        }
        __syncthreads();
        if (grp == 1) return;
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            const float2 b = pm[(wave * SLOTS + t) * 64 + lane];
            const float mx = fmaxf(m[t], b.x), wa = __builtin_amdgcn_exp2f(m[t] - mx), wb = __builtin_amdgcn_exp2f(b.x - mx);
            m[t] = mx, sum[t] = sum[t] * wa + b.y * wb;
#pragma unroll
            for (int v = 0; v < NV; ++v) o[v][t] = o[v][t] * wa + po[((wave * SLOTS + t) * NV + v) * 64 + lane] * wb;
        }
    }
    if (records) {
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            const int at = rw + t / MAPS * 16 + r16;
            if (at >= nq * group) continue;
            float *rec = records + ((((size_t)(at / group) * heads + head[t / MAPS]) * maps + alone + t % MAPS) * gridDim.y + blockIdx.y) * (kGqaRecHead + vdimp);
            if (g == 0) rec[0] = m[t], rec[1] = sum[t];
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (v * 16 < vdimp) *reinterpret_cast<f32x4 *>(rec + kGqaRecHead + v * 16 + g * 4) = o[v][t];
        }
        return;
    }
    float inv[SLOTS];
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) {
        inv[t] = 1.0f / sum[t];
        if (MAPS == 1 && p.sink) {  // (behind the keys: as their first maximum one far above them would leave their weights no bits)
            const float z = p.sink[head[t / MAPS]] * kLog2e, M = fmaxf(m[t], z), w = __builtin_amdgcn_exp2f(m[t] - M);
            inv[t] = w / (sum[t] * w + __builtin_amdgcn_exp2f(z - M));
        }
    }
    if (MAPS == 2) {
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            o[v][0] = o[v][0] * inv[0] - (p.lambda * inv[1]) * o[v][1];
            ss += (o[v][0].x * o[v][0].x + o[v][0].y * o[v][0].y) + (o[v][0].z * o[v][0].z + o[v][0].w * o[v][0].w);
        }
        inv[0] = p.out_scale / sqrtf(rows_sum(ss) / (float)p.vdim + p.eps);
    }
#pragma unroll
    for (int t = 0; t < SLOTS / MAPS; ++t) {
        const int at = rw + t * 16 + r16, qi = at / group, h = head[t];
        if (at >= nq * group) continue;
        if (p.gate && !(FAR && p.gate_columns)) inv[t] *= activate(gate_logit(p, qi, h, 0), BITNET_HIP_ACT_SIGMOID);
        uint16_t *dst = out + (size_t)qi * ldo + (size_t)h * vdimp + g * 4;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v * 16 < vdimp) {
                f32x4 q = o[v][t] * inv[t];
                if (FAR && p.gate_columns)
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[i] *= activate(gate_logit(p, qi, h, v * 16 + g * 4 + i), BITNET_HIP_ACT_SIGMOID);
                *reinterpret_cast<bf16x4 *>(dst + v * 16) = bf16x4{(__bf16)q.x, (__bf16)q.y, (__bf16)q.z, (__bf16)q.w};
            }
    }
}

// two maps whose keys find no room together: each by itself, put together from records
static bool maps_apart(const Gqa &g) { return g.maps == 2 && (g.dimp > 128 || g.vdimp > 128); }
bool kv8_prefill_wants_records(const Gqa &g) { return maps_apart(g); }

// Waves that share a tile, groups of them that share the rows, and stretches of the keys.  us of a step of a walk that the rule counts with (128 columns; measured last 1.77, 2.5, 2.15 for 1.72, 2.44, 1.98, which
// chooses no better: over eight shapes and eight lengths the forms taken are 2 % above the best on average, 20 % at most): four waves 1.72, with two such workgroups on a compute unit
// 2.4; two groups of four waves 2.44 for two tiles; eight waves (twice the rows) 1.98; heads of more than 128 columns 3.3, one workgroup on a compute unit; two maps of 65 to 128 columns 2.4
// whatever the waves, one workgroup.  A launch lasts as long as its longest walk, or as its share of all of them with what workgroups of unequal length leave idle (an eighth; more where few
// long ones share a compute unit's time).  Records cost 5 us and their bytes, 0.23 ns for 132 floats.
// Heads of up to 64 columns go by the same figures: they take three quarters of the time in every form.
// us, what this rule takes / four waves / two groups / eight waves, and in stretches where that is best:
//   20 heads on 5 of 128: 130 tokens 13 / 13 / 14 / 16; 600 23 / 26 / 23 / 30; 2000 53 / 70 / 53 / 78; 4000 130 / 130 / 141 / 149; 8192 428 / 407 / 459 / 428; 30 behind 7970 28 (157 whole)
//   32 on 8 of 128: 4000 174 / 186 / 208 / 174; 8192 610 / 626 / 709 / 609; 509 behind 20011 232 (384 whole, 214 in four)
//   20 on 5 of 64: 4000 101 / 101 / 106 / 116; 8192 338 / 306 / 355 / 335.  8 on 8 of 64: 4000 78 / 95 / 68 / 111 (65); 8192 147 / 189 / 145 / 222
//   two maps, 12 on 3 of 64 / 128: 4000 131 / 128 / 152 / 139; 509 behind 20011 177 (367 whole).  12 on 3 of 128: 600 32 / 32 / - / 33; 2000 88 / 88 / - / 86 (73); 4000 167 / 273 / - / 167
thread_local Kv8Form g_last_kv8_form{0, 0, 0};
static Kv8Form prefill_form(const Gqa &g, int n_ctx, int nq, bool room) {
    const int group = (int)(g.heads / g.kv_heads), maps = maps_apart(g) ? 1 : (int)g.maps, longest = n_ctx / 64 + 1 - (gqa_first(g, n_ctx - 1) >> 6);
    const double shortest = (n_ctx - nq) / 64 + 1 - (gqa_first(g, n_ctx - nq) >> 6), record = 0.23e-3 * (kGqaRecHead + g.vdimp) / 132 * nq * g.heads * g.maps;
    const bool wide = g.dimp > 128 || g.vdimp > 128, both = maps == 2 && g.dimp > 64;  // (keys of both maps: LDS has room for one workgroup)
    Kv8Form best{1, 4, 1};
    double least = 1e30;
    for (const Kv8Form f : {Kv8Form{1, 4, 1}, Kv8Form{2, 4, 1}, Kv8Form{1, 8, 1}}) {
        if ((wide && (f.groups == 2 || f.waves == 8)) || (f.groups == 2 && both)) continue;
        const int rows = 32 * f.waves / maps;
        const double workgroups = (double)g.kv_heads * ((nq * (size_t)group + rows - 1) / rows) * (maps_apart(g) ? 2 : 1);
        for (int parts = 1; parts <= (room ? 32 : 1) && (parts == 1 || (2 * parts <= longest && workgroups * parts <= 512)); ++parts) {
            const double at_once = workgroups * parts, stretch = ((longest + f.groups - 1) / f.groups + parts - 1) / parts, all = workgroups * 0.5 * (longest + shortest) / f.groups;
            const double walk = parts > 1 && at_once > 256 ? 2 * stretch : stretch;  // (stretches are all long: two rounds of them)
            double us;
            if (wide)
                us = 3.3 * std::max(walk, 1.12 * all / 256);
            else if (both)
                us = (f.waves == 8 ? 2.5 : 0.0) + 2.4 * std::max(walk, 1.12 * all / 256);
            else if (f.groups == 2)
                us = 2.0 + 2.44 * std::max(walk, 1.4 * all / 256);
            else if (f.waves == 8)
                us = 2.5 + 1.98 * std::max(walk, 1.12 * all / 256);
            else
                us = at_once <= 256 ? 1.72 * stretch : std::max((parts > 1 ? 2.4 : 1.9) * stretch, 2.4 * 1.12 * all / 512);
            if (parts > 1) us += 5.0 + record * parts;
            if (us < least) least = us, best = Kv8Form{f.groups, f.waves, parts};
        }
    }
    return best;
}
size_t kv8_prefill_floats(const Gqa &g, int n_ctx, int nq) {
    const int parts = prefill_form(g, n_ctx, nq, true).parts;
    return parts > 1 || maps_apart(g) ? (size_t)nq * g.heads * g.maps * parts * (kGqaRecHead + g.vdimp) : 0;
}

template <int NK, int NV, int G, int W>
static hipError_t prefill_go(const Kv8 &c, const uint16_t *q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, float *records, int parts, hipStream_t s) {
    const Gqa &g = c.g;
    const bool apart = maps_apart(g);
    const int maps = apart ? 1 : (int)g.maps, rows = 32 * W / maps, n_qb = (int)((nq * (g.heads / g.kv_heads) + rows - 1) / rows);
    const size_t tiles = (size_t)2 * G * kv8_tile_bytes(NK, NV, maps), sums = G == 2 ? (size_t)W * 2 * 64 * (NV * 16 + 8) : 0;
    const size_t lds = tiles > sums ? tiles : sums;
    auto fn = k_kv8_prefill<NK, NV, 1, false, G, W>;
    if (g.far_weight || g.gate_columns) fn = k_kv8_prefill<NK, NV, 1, true, G, W>;
    if constexpr (NK <= 2 && NV <= 8 && 2 * G * kv8_tile_bytes(NK, NV, 2) <= 163840)
        if (maps == 2) fn = k_kv8_prefill<NK, NV, 2, false, G, W>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const bool leaves = parts > 1 || apart;
    hipLaunchKernelGGL(fn, dim3(g.kv_heads * n_qb, parts, apart ? 2 : 1), dim3(64 * W * G), lds, s, c, q, ldq, n_ctx, nq, out, ldo, n_qb, leaves ? records : nullptr);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || !leaves ? e : launch_gqa_merge_parts(g, records, parts, nq, out, ldo, s);
}

template <int NK, int NV>
static hipError_t prefill_pick(const Kv8 &c, const uint16_t *q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, float *records, hipStream_t s) {
    const Kv8Form f = g_last_kv8_form = prefill_form(c.g, n_ctx, nq, records != nullptr);
    if constexpr (NV <= 8) {
        if (f.groups == 2) return prefill_go<NK, NV, 2, 4>(c, q, ldq, n_ctx, nq, out, ldo, records, f.parts, s);
        if (f.waves == 8) return prefill_go<NK, NV, 1, 8>(c, q, ldq, n_ctx, nq, out, ldo, records, f.parts, s);
    }
    return prefill_go<NK, NV, 1, 4>(c, q, ldq, n_ctx, nq, out, ldo, records, f.parts, s);
}

// records: kv8_prefill_floats(g, n_ctx, nq) of them, or none where a block's keys stay together (not with maps apart)
hipError_t launch_kv8_prefill(const Kv8 &c, const uint16_t *q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, float *records, hipStream_t s) {
    const Gqa &g = c.g;
    if (!gqa_supported((int)g.dimp, (int)g.vdimp) || (maps_apart(g) && !records)) return hipErrorInvalidValue;
    if (g.dimp <= 64 && g.vdimp <= 64) return prefill_pick<1, 4>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
    if (g.dimp <= 64 && g.vdimp <= 128) return prefill_pick<1, 8>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
    if (g.dimp <= 128 && g.vdimp <= 128) return prefill_pick<2, 8>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
    return prefill_pick<4, 16>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
}

}  // namespace bitnet_hip
