// kernels_kv8.hip -- the attention of kernels_gqa.hip over caches of 8 bits (gfx950).
//
// A head's key (of one map) and a head's value at a position are whole numbers -127 .. 127 with one f32 scale each: value = number * scale (kv8_scale, gqa.hpp).  One scale
// per position, not per block of them: an append touches nothing that is written, and the cache is a function of the tokens alone, however they came in.
// Keys int8 [kv head][map][capacity][dimp]; values int8 [kv head][capacity / 32][vdimp / 32][16][4][2][8]: column c at position p lies at [p / 32][c / 32][c % 16]
// [p % 32 / 8][c % 32 / 16][p % 8], so that 32 keys by 32 columns are 1 KiB in the order in which the matrix cores take them, and 32 keys of a head are one piece.
//   k_kv8_rows     rows of projections: convolution, norms, rotation, then 8 bits
//   k_kv8_read     positions back as bf16 or f32
//   k_kv8_step     the decode step, records as k_gqa_step leaves them
//   k_kv8_prefill  a prompt's portion
// Scores are whole: a query is cut into balanced digits of 8 bits with one scale (23 bits in a step, 15 in a prompt, whose queries are bf16), the products with the keys'
// numbers are exact in 32-bit integers, and the scales come behind them.  A weight times its value's scale meets the values' numbers as f16, which holds them exactly: a
// (high, low) pair in a step, one f16 in a prompt (2^-12 against the 2^-9 of its bf16 output).
#include "gqa.hpp"

namespace bitnet_hip {

typedef int i32x4 __attribute__((ext_vector_type(4)));
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
// the least E with |v| < 2^E (v = 0: -100)
__device__ __forceinline__ int exponent_above(float v) { return v > 0.f ? max(__builtin_amdgcn_frexp_expf(v), -100) : -100; }
__device__ __forceinline__ float power2(int e) { return __builtin_amdgcn_ldexpf(1.0f, e); }

// a product in which zero times anything is zero
__device__ __forceinline__ float mul_zero(float a, float b) {
    float r;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// where column c of a kv head's values at position pos lies
__device__ __forceinline__ size_t kv8_value_at(int vdimp, int pos, int c) {
    return (size_t)(pos >> 5) * (vdimp * 32) + (c >> 5) * 1024 + (c & 15) * 64 + (pos >> 3 & 3) * 16 + (c >> 4 & 1) * 8 + (pos & 7);
}

// ---- rows of projections ----------------------------------------------------------------------------------------------
// blockIdx.y: query heads x maps and key heads x maps (sixteen tokens per workgroup), then value heads: 32 positions of whole tiles, eight threads a token.
template <class TR, int NJ, int TAPS>
__global__ __launch_bounds__(256) void k_kv8_rows(Kv8 c, const TR *rows, size_t ld, const int *pos_ptr, int n, TR *queries, size_t ldq) {
    __shared__ __attribute__((aligned(16))) uint8_t tile[256 * 32];
    const Gqa &p = c.g;
    const int tid = threadIdx.x, wave = tid >> 6, pos0 = *pos_ptr;
    const int nq = (int)(p.heads * p.maps), nk = (int)(p.kv_heads * p.maps), dimp = (int)p.dimp, vdimp = (int)p.vdimp, y = blockIdx.y;
    if (y < nq + nk) {
        const bool key = y >= nq;
        const int t0 = blockIdx.x * kRowTokens + wave * (kRowTokens / 4);
        if (t0 >= n) return;
        int8_t *cache = key ? (int8_t *)p.kcache + (size_t)(y - nq) * p.capacity * dimp : nullptr;
        head_rows<TR, int8_t, NJ, TAPS>(p, rows, ld, pos0, t0, n, y, key, cache, queries, ldq, key ? c.k_scale + (size_t)(y - nq) * p.capacity : nullptr);
        return;
    }
    const int kv = y - nq - nk, first = ((pos0 >> 5) + (int)blockIdx.x) * 32;
    if (first >= pos0 + n) return;
    const int at = tid >> 3, part = tid & 7, t = first + at - pos0, column = (p.values_are_keys ? nq : nq + nk) * dimp + kv * vdimp;
    const bool live = t >= 0 && t < n;
    const int taps = TAPS > 0 ? TAPS : TAPS < 0 ? (int)p.taps : 1, channels = gqa_channels(p);
    f32x4 v[8];
    float largest = 0.f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (!live || 32 * j >= vdimp) continue;
        const int at_col = column + 32 * j + 4 * part;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (TAPS != 0)
                for (int k = 0; k < taps; ++k) v[j][e] += p.conv[(size_t)k * channels + at_col + e] * raw_value(p, rows, ld, pos0, t - (taps - 1) + k, at_col + e, channels);
            else
                v[j][e] = ld_act(rows + (size_t)t * ld, at_col + e);
            largest = fmaxf(largest, fabsf(v[j][e])), finite = finite && is_finite(v[j][e]);
        }
    }
    if (!finite) largest = INFINITY;  // (no finite value is)
#pragma unroll
    for (int d = 1; d < 8; d *= 2) largest = fmaxf(largest, __shfl_xor(largest, d, 64));
    const Kv8Scale s = kv8_scale(largest, is_finite(largest));
    if (live && part == 0) c.v_scale[(size_t)kv * p.capacity + first + at] = s.scale;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (32 * j < vdimp)
#pragma unroll
            for (int e = 0; e < 4; ++e) tile[kv8_value_at(vdimp, at, 32 * j + 4 * part + e)] = (uint8_t)kv8_number(v[j][e], s);
    __syncthreads();
    uint8_t *dst = (uint8_t *)p.vcache + (size_t)kv * vdimp * p.capacity + (size_t)first * vdimp;
    for (int i = tid; i < vdimp * 2; i += 256) {  // sixteen bytes: eight positions of two columns
        const int t8 = first + (i & 3) * 8 - pos0;
        if (t8 >= 0 && t8 + 8 <= n) {
            *reinterpret_cast<u32x4 *>(dst + i * 16) = *reinterpret_cast<const u32x4 *>(tile + i * 16);
        } else {
            for (int e = 0; e < 16; ++e)
                if (t8 + (e & 7) >= 0 && t8 + (e & 7) < n) dst[i * 16 + e] = tile[i * 16 + e];
        }
    }
}

template <class TR>
static hipError_t rows_go(const Kv8 &c, const void *rows, size_t ld, const int *pos, int n, void *q, size_t ldq, hipStream_t s) {
    const Gqa &g = c.g;
    const int keys = g.queries_only ? 0 : (int)(g.kv_heads * g.maps + g.kv_heads);
    // (n tokens from anywhere in a tile of 32 on reach into (n + 62) / 32 of them at most)
    const dim3 grid(std::max((n + kRowTokens - 1) / kRowTokens, (n + 62) / 32), (int)(g.heads * g.maps) + keys);
    auto pick = [&](auto narrow, auto wide) { return g.dimp <= 128 ? narrow : wide; };
    auto fn = g.taps == 0   ? pick(k_kv8_rows<TR, 1, 0>, k_kv8_rows<TR, 2, 0>)
              : g.taps == 3 ? pick(k_kv8_rows<TR, 1, 3>, k_kv8_rows<TR, 2, 3>)
                            : pick(k_kv8_rows<TR, 1, -1>, k_kv8_rows<TR, 2, -1>);
    hipLaunchKernelGGL(fn, grid, dim3(256), 0, s, c, (const TR *)rows, ld, pos, n, (TR *)q, ldq);
    return hipGetLastError();
}
hipError_t launch_kv8_rows(const Kv8 &c, const void *rows, size_t ld, int rows_f32, const int *pos, int n, void *q, size_t ldq, hipStream_t s) {
    return rows_f32 ? rows_go<float>(c, rows, ld, pos, n, q, ldq, s) : rows_go<uint16_t>(c, rows, ld, pos, n, q, ldq, s);
}

// ---- positions read back ----------------------------------------------------------------------------------------------
// blockIdx.y: key heads x maps (16 bytes a thread), then value heads (a tile of 32 positions a workgroup, turned round in LDS).
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
        const int pieces = dimp >> 4, i = blockIdx.x * 256 + tid, t = i / pieces;
        if (t >= n) return;
        const size_t row = (size_t)blockIdx.y * p.capacity + first + t;
        const int at = (i - t * pieces) * 16;
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
    const size_t blocks = std::max(keys ? ((size_t)n * (g.dimp / 16) + 255) / 256 : (size_t)1, values ? ((size_t)n + 62) / 32 : (size_t)1);
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
// A weight times its value's scale is brought to at most 2^14 by a power of two that the wave keeps (o is held times 2^(14 - above)).
struct Kv8StepK {
    const float *row, *q_weight, *k_weight, *q_factor, *rope_cos, *rope_sin, *far_weight, *far_rate;
    const int *pos;
    int8_t *K, *V;
    float *k_scale, *v_scale, *scratch, eps;
    int heads, group, dim, dimp, vdimp, capacity, turned, chunk, window, normed, append, k_at, v_at;  // normed: 1 queries, 2 keys
};
constexpr float kStepDigits = 8355000.0f;   // below 127 (2^16 + 2^8 + 1): three balanced digits
constexpr float kPromptDigits = 32600.0f;   // below 127 (2^8 + 1): two

template <int NK, int NV, int MAPS>
__global__ __launch_bounds__(256, NV > 8 || NK * MAPS >= 4 ? 1 : 2) void k_kv8_step(Kv8StepK p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t area[];  // digits of the queries [maps][3][16][QS]; then the waves' outputs
    __shared__ float sm[4][MAPS][16], sl[4][MAPS][16], qscale[MAPS][16], news[MAPS + 1];
    __shared__ __attribute__((aligned(16))) int8_t newk[MAPS][NK * 64], newv[NV * 16];
    constexpr int QS = NK * 64 + 32, J = NK, JV = (NV * 16 + 63) / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    const int kv = blockIdx.x, first_head = blockIdx.y * 16, h0 = kv * p.group + first_head, nh = min(16, p.group - first_head);
    const int dimp = p.dimp, vdimp = p.vdimp, pos = __builtin_amdgcn_readfirstlane(*p.pos), n_keys = pos + 1;
    int first = p.chunk ? pos - (int)((unsigned)pos % (unsigned)p.chunk) : 0;  // gqa_range
    if (p.window && pos - p.window + 1 > first) first = pos - p.window + 1;
    const int base = first & ~(kGqaTile - 1), tiles = (n_keys - base + kGqaTile - 1) / kGqaTile, per = (tiles + kGqaSplits - 1) / kGqaSplits, used = (tiles + per - 1) / per;
    if ((int)blockIdx.z >= used) return;
    const int k0 = base + blockIdx.z * per * kGqaTile, k1 = min(k0 + per * kGqaTile, n_keys);
    int8_t *K = p.K + (size_t)kv * MAPS * p.capacity * dimp, *V = p.V + (size_t)kv * vdimp * p.capacity;
    float *KS = p.k_scale + (size_t)kv * MAPS * p.capacity, *VS = p.v_scale + (size_t)kv * p.capacity;
    i32x4 kf[2][MAPS][NK];
    u32x4 vf[NV / 2];
    f32x4 sk[MAPS][2], sv[2];
    auto fetch_keys = [&](int kb) {  // (blocks lie below the capacity, a multiple of 128)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
#pragma unroll
                for (int kk = 0; kk < NK; ++kk)
                    kf[t][j][kk] = *reinterpret_cast<const i32x4 *>(K + ((size_t)j * p.capacity + kb + (r16 >> 2) * 8 + t * 4 + (r16 & 3)) * dimp + min(kk * 64 + g * 16, dimp - 16));
                sk[j][t] = *reinterpret_cast<const f32x4 *>(KS + (size_t)j * p.capacity + kb + g * 8 + t * 4);
            }
    };
    auto fetch_values = [&](int kb) {
#pragma unroll
        for (int v = 0; v < NV / 2; ++v) vf[v] = *reinterpret_cast<const u32x4 *>(V + (size_t)kb * vdimp + min(v, (vdimp >> 5) - 1) * 1024 + r16 * 64 + g * 16);
#pragma unroll
        for (int t = 0; t < 2; ++t) sv[t] = *reinterpret_cast<const f32x4 *>(VS + kb + g * 8 + t * 4);
    };
    if (k0 + wave * 32 < k1) fetch_keys(k0 + wave * 32), fetch_values(k0 + wave * 32);
    float cs[J], sn[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        cs[j] = 1.0f, sn[j] = 0.f;
        if (p.turned && 64 * j < p.turned) {
            const size_t at = (size_t)pos * (p.turned >> 1) + (min(lane + 64 * j, p.turned - 1) >> 1);
            cs[j] = p.rope_cos[at], sn[j] = p.rope_sin[at];
        }
    }
    // a row of a head, elements lane + 64 j: norm, weight, rotation by pairs of neighbours; the largest of them, INFINITY if one is not finite
    auto finished = [&](const float *src, const float *weight, bool normed, float factor, float (&x)[J]) {
        float ss = 0.f, largest = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            x[j] = lane + 64 * j < dimp ? src[lane + 64 * j] : 0.f;
            ss += x[j] * x[j];
        }
        if (normed) factor *= 1.0f / sqrtf(wave_sum(ss) / (float)p.dim + p.eps);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int i = lane + 64 * j;
            x[j] *= factor * (weight && i < p.dim ? weight[i] : 1.0f);
            if (p.turned) {
                const float o = dpp<0xb1>(x[j]);  // quad_perm [1,0,3,2]
                if (i < p.turned) x[j] = (i & 1) ? x[j] * cs[j] + o * sn[j] : x[j] * cs[j] - o * sn[j];
            }
            largest = fmaxf(largest, is_finite(x[j]) ? fabsf(x[j]) : INFINITY);
        }
        return rows_max(row_max(largest));
    };
    const bool owner = k1 == n_keys && p.append;
    if (owner && 3 - wave < MAPS) {  // the record that holds the new position appends it (and puts it into its own fragments below)
        const int j = 3 - wave;
        float x[J];
        const float largest = finished(p.row + p.k_at + (kv * MAPS + j) * dimp, p.k_weight, p.normed & 2, 1.0f, x);
        const Kv8Scale s = kv8_scale(largest, is_finite(largest));
#pragma unroll
        for (int i = 0; i < J; ++i)
            if (lane + 64 * i < dimp) {
                const int8_t b = (int8_t)kv8_number(x[i], s);
                K[((size_t)j * p.capacity + pos) * dimp + lane + 64 * i] = b;
                newk[j][lane + 64 * i] = b;
            }
        if (lane == 0) KS[(size_t)j * p.capacity + pos] = s.scale, news[j] = s.scale;
    }
    if (owner && wave == 0) {
        float x[JV], largest = 0.f;
#pragma unroll
        for (int i = 0; i < JV; ++i) {
            x[i] = lane + 64 * i < vdimp ? p.row[p.v_at + kv * vdimp + lane + 64 * i] : 0.f;
            largest = fmaxf(largest, is_finite(x[i]) ? fabsf(x[i]) : INFINITY);
        }
        largest = rows_max(row_max(largest));
        const Kv8Scale s = kv8_scale(largest, is_finite(largest));
#pragma unroll
        for (int i = 0; i < JV; ++i)
            if (lane + 64 * i < vdimp) {
                const int8_t b = (int8_t)kv8_number(x[i], s);
                V[kv8_value_at(vdimp, pos, lane + 64 * i)] = b;
                newv[lane + 64 * i] = b;
            }
        if (lane == 0) VS[pos] = s.scale, news[MAPS] = s.scale;
    }
    const float factor = p.q_factor[pos];
    for (int r = wave; r < nh * MAPS; r += 4) {  // (head, map)
        const int hh = r / MAPS, j = r - hh * MAPS;
        float x[J];
        const float largest = finished(p.row + ((size_t)(h0 + hh) * MAPS + j) * dimp, p.q_weight, p.normed & 1, factor, x);
        const bool live = largest >= 1e-30f && is_finite(largest);
        const float to = live ? kStepDigits / largest : 0.f;
        uint8_t *dst = area + (size_t)(j * 3 * 16 + hh) * QS;
#pragma unroll
        for (int i = 0; i < J; ++i) {
            const int v = live ? (int)rintf(x[i] * to) : 0, d0 = (int)(int8_t)v, v1 = (v - d0) >> 8, d1 = (int)(int8_t)v1, d2 = (v1 - d1) >> 8;
            dst[lane + 64 * i] = (uint8_t)d0, dst[16 * QS + lane + 64 * i] = (uint8_t)d1, dst[32 * QS + lane + 64 * i] = (uint8_t)d2;
        }
        if (lane == 0) qscale[j][hh] = is_finite(largest) ? largest / kStepDigits : __builtin_nanf("");
    }
    __syncthreads();
    i32x4 q[MAPS][3][NK];  // (lanes past the last head: whatever lies there; a column of the products is a head of its own)
    float qs[MAPS];
#pragma unroll
    for (int j = 0; j < MAPS; ++j) {
        qs[j] = qscale[j][r16];
#pragma unroll
        for (int d = 0; d < 3; ++d)
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) q[j][d][kk] = *reinterpret_cast<const i32x4 *>(area + (size_t)((j * 3 + d) * 16 + r16) * QS + kk * 64 + g * 16);
    }
    FarPenalty far{0.f, 0.f};
    if (p.far_weight) far.weight = p.far_weight[min(h0 + r16, p.heads - 1)] * 0.69314718055994531f, far.rate = p.far_rate[min(h0 + r16, p.heads - 1)];
    f32x4 o[NV][MAPS];
    float m[MAPS], l[MAPS];
#pragma unroll
    for (int j = 0; j < MAPS; ++j) {
        m[j] = -INFINITY, l[j] = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int above = -100;
    for (int kb = k0 + wave * 32; kb < k1; kb += 128) {
        const bool more = kb + 128 < k1;
        if (kb + 32 <= first) {  // (another chunk's keys)
            if (more) fetch_keys(kb + 128), fetch_values(kb + 128);
            continue;
        }
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
        float largest = 0.f;
        bool seen[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = kb + g * 8 + t * 4 + e;
                seen[t][e] = key < k1 && key >= first;
                sv[t][e] = seen[t][e] ? sv[t][e] : 0.f;
                largest = fmaxf(largest, sv[t][e]);
            }
        const int need = __builtin_amdgcn_readfirstlane(exponent_above(rows_max(largest)));
        if (need > above) {
            const float down = power2(max(above - need, -140));
#pragma unroll
            for (int j = 0; j < MAPS; ++j)
#pragma unroll
                for (int v = 0; v < NV; ++v) o[v][j] *= down;
            above = need;
        }
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
                    for (int kk = 0; kk < NK; ++kk) a[d] = mfma_i8(kf[t][j][kk], q[j][d][kk], a[d]);  // (columns past dimp: the query is zero there)
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] = fmaf((float)a[2][e], 65536.0f, fmaf((float)a[1][e], 256.0f, (float)a[0][e])) * (sk[j][t][e] * qs[j]);
                    if (MAPS == 1 && p.far_weight) s[t][e] = nearer(s[t][e], far, pos - (kb + g * 8 + t * 4 + e));
                    s[t][e] = seen[t][e] ? s[t][e] * kLog2e : -INFINITY;
                }
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            mx = fmaxf(m[j], rows_max(mx));
            if (mx == -INFINITY) mx = 0.f;  // (no score is a number: neither is the sum)
            const float al = __builtin_amdgcn_exp2f(m[j] - mx);
            m[j] = mx;
            f32x4 w[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[t][e] = __builtin_amdgcn_exp2f(s[t][e] - mx);
            l[j] = l[j] * al + ((w[0][0] + w[0][1]) + (w[0][2] + w[0][3])) + ((w[1][0] + w[1][1]) + (w[1][2] + w[1][3]));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float x = w[t][e] * __builtin_amdgcn_ldexpf(sv[t][e], 14 - above), y = w[t][e + 1] * __builtin_amdgcn_ldexpf(sv[t][e + 1], 14 - above);
                    // (an instruction by name: left to itself the compiler rounds the product once for the products and another time for what is left of it)
                    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
                    hi[j][4 * t + e] = h.x, hi[j][4 * t + e + 1] = h.y;
                    lo[j][4 * t + e] = (_Float16)(x - (float)h.x), lo[j][4 * t + e + 1] = (_Float16)(y - (float)h.y);
                }
#pragma unroll
            for (int v = 0; v < NV; ++v) o[v][j] *= al;
        }
        if (more) fetch_keys(kb + 128);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const f16x8 a = eight_f16(vf[v / 2][2 * (v & 1)], vf[v / 2][2 * (v & 1) + 1]);
#pragma unroll
            for (int j = 0; j < MAPS; ++j) {
                o[v][j] = mfma_f16(a, hi[j], o[v][j]);
                o[v][j] = mfma_f16(a, lo[j], o[v][j]);
            }
        }
        if (more) fetch_values(kb + 128);
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
        float *rec = p.scratch + ((size_t)((h0 + hh) * MAPS + j) * kGqaSplits + blockIdx.z) * (kGqaRecHead + vdimp);
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
// buffers of a tile in LDS: two where the tiles that are under way on a compute unit leave room
constexpr int kv8_tile_bytes(int nk, int nv, int maps) { return maps * 64 * (nk * 64 + 32) + nv * 16 * (64 * 2 + 32) + (maps + 1) * 256 + 16; }
constexpr int kv8_buffers(int nk, int nv, int maps) { return (nv > 8 || nk > 2 ? 2 : 4) * kv8_tile_bytes(nk, nv, maps) <= 163840 ? 2 : 1; }

// One workgroup: one head, four waves; a wave holds two slots of 16 queries: both maps of one query tile, or two tiles of the only map.  Key tiles of 64 (every map's) and the
// values of the tile staged through registers into LDS one step ahead, the values as f16.  G = 2: two such groups of four waves share the keys of the same queries, tile by tile
// in turn, and meet in LDS at the end.  records: gridDim.y workgroups share a block's tiles of keys, in stretches (launch_gqa_merge_parts).
// A query of bf16 is two digits of 8 bits, 15 bits of its largest element.  l and o are held times 2^(14 - above), above being the exponent of the largest value scale so far.
// FAR: with a distance penalty, gates per column, or both.
template <int NK, int NV, int MAPS, bool FAR, int G>
__global__ __launch_bounds__(256 * G, NV > 8 || NK > 2 ? 1 : 2) void k_kv8_prefill(Kv8 c, const uint16_t *Q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, int n_qb, float *records) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int SLOTS = 2, QW = 16 * SLOTS / MAPS, KS = NK * 64 + 32, VS = 64 * 2 + 32, NVL = NV / 4;
    const Gqa &p = c.g;
    const int grp = G == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0, tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g = lane >> 4;
    constexpr int KB = MAPS * 64 * KS, SB = KB + NV * 16 * VS, TILE = kv8_tile_bytes(NK, NV, MAPS), BUFS = kv8_buffers(NK, NV, MAPS);
    uint8_t *lk = lds + grp * BUFS * TILE;
    const int heads = (int)p.heads, dimp = (int)p.dimp, vdimp = (int)p.vdimp;
    // (the order of k_gqa_prefill's workgroups)
    const int x = blockIdx.x & 7, rest = blockIdx.x >> 3, own = heads >> 3, left = heads & 7, per = own + (left ? 1 : 0);
    const int level = rest / per, slot = rest - level * per, r = (x + 8 * left - (level % 8) * left) & 7;
    if (slot == own && r >= left) return;
    const int h = slot < own ? x * own + slot : 8 * own + r, qb = n_qb - 1 - level;
    const int kv = h / (int)(p.heads / p.kv_heads), q0 = qb * 4 * QW, pos0 = n_ctx - nq, qw = q0 + wave * QW;
    i32x4 qd[SLOTS][2][NK];  // digits: low, high
    float qs[SLOTS];
    int qpos[SLOTS], qfirst[SLOTS];
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) {
        const int tile = t / MAPS, map = t % MAPS, qi = min(qw + tile * 16 + r16, nq - 1);
        qpos[t] = pos0 + qw + tile * 16 + r16;
        qfirst[t] = gqa_first(p, qpos[t]);
        const uint16_t *q = Q + (size_t)qi * ldq + (size_t)(h * MAPS + map) * dimp;
        float largest = 0.f;
        u32x4 raw[NK][2];
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                raw[kk][e] = kk * 64 + g * 16 < dimp ? *reinterpret_cast<const u32x4 *>(q + kk * 64 + g * 16 + e * 8) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = bf2f(raw[kk][e][i >> 1] >> (16 * (i & 1)) & 0xffffu);
                    largest = fmaxf(largest, is_finite(v) ? fabsf(v) : INFINITY);
                }
            }
        largest = rows_max(largest);
        const bool live = largest >= 1e-30f && is_finite(largest);
        const float to = live ? kPromptDigits / largest : 0.f;
        qs[t] = live ? largest * (kLog2e / kPromptDigits) : is_finite(largest) ? 1.0f : __builtin_nanf("");
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t lo = 0, hi = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 4 * i + e;
                    const float v = bf2f(raw[kk][at >> 3][(at & 7) >> 1] >> (16 * (at & 1)) & 0xffffu);
                    const int n = live ? (int)rintf(v * to) : 0, d0 = (int)(int8_t)n, d1 = (n - d0) >> 8;
                    lo |= (uint32_t)(d0 & 0xff) << (8 * e), hi |= (uint32_t)(d1 & 0xff) << (8 * e);
                }
                qd[t][0][kk][i] = (int)lo, qd[t][1][kk][i] = (int)hi;
            }
    }
    f32x4 o[NV][SLOTS];
    float m[SLOTS], l[SLOTS];
    int above = -80;
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) {
        // (finite: with chunks a tile may hold no key that a query sees; the sink counts once per query, four lanes share one)
        const bool sink = MAPS == 1 && p.sink && grp == 0 && !records;
        m[t] = sink ? p.sink[h] * kLog2e : -1e30f, l[t] = sink && g == 0 ? power2(14 - above) : 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) o[v][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int8_t *K = (const int8_t *)p.kcache + (size_t)kv * MAPS * p.capacity * dimp, *V = (const int8_t *)p.vcache + (size_t)kv * vdimp * p.capacity;
    const float *KSC = c.k_scale + (size_t)kv * MAPS * p.capacity, *VSC = c.v_scale + (size_t)kv * p.capacity;
    // keys: a row of the tile by KC neighbouring threads; row p of 32 in LDS is key 8 (p >> 2 & 3) + 4 (p >> 4) + (p & 3)
    constexpr int KC = NK * 4, KR = 256 / KC;
    u32x4 kreg[MAPS][NK], vreg[NVL];
    float sreg[MAPS + 1];
    const unsigned koff = (unsigned)((tid / KC) * dimp + min((tid % KC) * 16, dimp - 16));
    int kw[NK], vw[NVL], voff[NVL];
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        const int key = tid / KC + j * KR, row = (key & 32) + (key >> 2 & 1) * 16 + (key >> 3 & 3) * 4 + (key & 3);
        kw[j] = row * KS + (tid % KC) * 16;
    }
#pragma unroll
    for (int j = 0; j < NVL; ++j) {  // sixteen bytes: eight keys of two columns, 16 apart; columns past vdimp are zero
        const int i = tid + 256 * j, half = i / (NV * 32), rem = i % (NV * 32);
        vw[j] = KB + ((rem >> 6) * 32 + (rem >> 2 & 15)) * VS + half * 64 + (rem & 3) * 16;
        voff[j] = (rem >> 6) * 32 < vdimp ? half * vdimp * 32 + rem * 16 : -1;
        vreg[j] = u32x4{0u, 0u, 0u, 0u};
    }
    auto fetch = [&](int key0) {  // (whole tiles: the capacity is a multiple of 64)
#pragma unroll
        for (int mp = 0; mp < MAPS; ++mp) {
            const int8_t *kb = K + ((size_t)mp * p.capacity + key0) * dimp;
#pragma unroll
            for (int j = 0; j < NK; ++j) kreg[mp][j] = *reinterpret_cast<const u32x4 *>(kb + (size_t)(j * KR) * dimp + koff);
        }
        const int8_t *vb = V + (size_t)key0 * vdimp;
#pragma unroll
        for (int j = 0; j < NVL; ++j)
            if (voff[j] >= 0) vreg[j] = *reinterpret_cast<const u32x4 *>(vb + voff[j]);
        if (wave == 0) {  // (a position past the portion may hold anything)
            const bool in = key0 + lane < n_ctx;
#pragma unroll
            for (int mp = 0; mp < MAPS; ++mp) sreg[mp] = in ? KSC[(size_t)mp * p.capacity + key0 + lane] : 0.f;
            sreg[MAPS] = in ? VSC[key0 + lane] : 0.f;
        }
    };
    auto store = [&](int at) {
#pragma unroll
        for (int mp = 0; mp < MAPS; ++mp)
#pragma unroll
            for (int j = 0; j < NK; ++j) *reinterpret_cast<u32x4 *>(lk + at + kw[j] + mp * 64 * KS) = kreg[mp][j];
#pragma unroll
        for (int j = 0; j < NVL; ++j) {
            *reinterpret_cast<f16x8 *>(lk + at + vw[j]) = eight_f16(vreg[j].x, vreg[j].y);
            *reinterpret_cast<f16x8 *>(lk + at + vw[j] + 16 * VS) = eight_f16(vreg[j].z, vreg[j].w);
        }
        if (wave == 0) {
            float *sc = reinterpret_cast<float *>(lk + at + SB);
#pragma unroll
            for (int mp = 0; mp <= MAPS; ++mp) sc[mp * 64 + lane] = sreg[mp];
            const int e = min(exponent_above(rows_max(row_max(fmaxf(sreg[MAPS], 0.f)))), 126);
            if (lane == 0) reinterpret_cast<int *>(sc)[(MAPS + 1) * 64] = e;
        }
    };
    int n_tiles = (min(n_ctx, pos0 + q0 + 4 * QW) + 63) / 64;
    const FarPenalty far = far_penalty(p, h);
    // tiles from the first key of the workgroup's first query on; a wave leaves out what lies ahead of its own first key
    int t_first = gqa_first(p, pos0 + q0) >> 6;
    const int w_first = gqa_first(p, pos0 + qw), w_last = gqa_first(p, pos0 + qw + QW - 1);
    if (records) {
        const int each = (n_tiles - t_first + (int)gridDim.y - 1) / (int)gridDim.y;
        t_first = min(t_first + (int)blockIdx.y * each, n_tiles), n_tiles = min(t_first + each, n_tiles);
    }
    fetch(max(min(t_first + grp, n_tiles - 1), 0) * 64);
    if (BUFS == 2) {
        store(0);
        if (t_first + grp + G < n_tiles) fetch((t_first + grp + G) * 64);
    }
    int at = 0;  // the tile's buffer
    for (int t0 = t_first; t0 < n_tiles; t0 += G) {
        const int kt0 = t0 + grp, key0 = kt0 * 64;
        __syncthreads();
        if (BUFS == 1) {
            store(0);
            __syncthreads();
            if (kt0 + G < n_tiles) fetch(key0 + G * 64);
        }
        const bool seen = !(key0 > pos0 + qw + QW - 1 || key0 + 63 < w_first || (G == 2 && kt0 >= n_tiles));  // (else: no key of the tile is seen by this wave's queries)
        const uint8_t *kt_ = lk + at;
        f16x8 pf[2][SLOTS];
        if (seen) {
            const float *sc = reinterpret_cast<const float *>(kt_ + SB);
            const int need = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int *>(sc)[(MAPS + 1) * 64]);
            if (need > above) {
                const float down = power2(above - need);
#pragma unroll
                for (int t = 0; t < SLOTS; ++t) {
                    l[t] *= down;
#pragma unroll
                    for (int v = 0; v < NV; ++v) o[v][t] *= down;
                }
                above = need;
            }
            f32x4 s[4][SLOTS];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                i32x4 a[SLOTS][2];
#pragma unroll
                for (int t = 0; t < SLOTS; ++t) a[t][0] = a[t][1] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                    for (int t = 0; t < SLOTS; ++t) {
                        const i32x4 k = *reinterpret_cast<const i32x4 *>(kt_ + ((t % MAPS) * 64 + kt * 16 + r16) * KS + kk * 64 + g * 16);
                        a[t][0] = mfma_i8(k, qd[t][0][kk], a[t][0]);
                        a[t][1] = mfma_i8(k, qd[t][1][kk], a[t][1]);
                    }
#pragma unroll
                for (int t = 0; t < SLOTS; ++t) {
                    const f32x4 ks = *reinterpret_cast<const f32x4 *>(sc + (t % MAPS) * 64 + (kt >> 1) * 32 + g * 8 + (kt & 1) * 4);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[kt][t][i] = (float)(a[t][1][i] * 256 + a[t][0][i]) * ks[i];
                }
            }
            // (from here on a score is times qs, which holds log2(e))
            if (FAR && p.far_weight)
#pragma unroll
                for (int t = 0; t < SLOTS; ++t)
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[kt][t][i] = nearer(s[kt][t][i] * qs[t], FarPenalty{far.weight * kLog2e, far.rate}, qpos[t] - (key0 + (kt >> 1) * 32 + g * 8 + (kt & 1) * 4 + i));
            if (key0 + 63 > pos0 + qw)  // the diagonal
#pragma unroll
                for (int t = 0; t < SLOTS; ++t)
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kt][t][i] = key0 + (kt >> 1) * 32 + g * 8 + (kt & 1) * 4 + i > qpos[t] ? -INFINITY : s[kt][t][i];
            if (key0 < w_last)  // an earlier chunk of some of the queries
#pragma unroll
                for (int t = 0; t < SLOTS; ++t)
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[kt][t][i] = key0 + (kt >> 1) * 32 + g * 8 + (kt & 1) * 4 + i < qfirst[t] ? -INFINITY : s[kt][t][i];
            float mn[SLOTS], c2[SLOTS];
            bool grows = false;
#pragma unroll
            for (int t = 0; t < SLOTS; ++t) {
                c2[t] = FAR && p.far_weight ? 1.0f : qs[t];
                float mx = fmaxf(fmaxf(s[0][t][0], s[0][t][1]), fmaxf(s[0][t][2], s[0][t][3]));
#pragma unroll
                for (int kt = 1; kt < 4; ++kt) mx = fmaxf(mx, fmaxf(fmaxf(s[kt][t][0], s[kt][t][1]), fmaxf(s[kt][t][2], s[kt][t][3])));
                mn[t] = fmaxf(m[t], rows_max(mx) * c2[t]);
                grows = grows || mn[t] > m[t];
            }
            if (__any(grows)) {
#pragma unroll
                for (int t = 0; t < SLOTS; ++t) {
                    const float al = __builtin_amdgcn_exp2f(m[t] - mn[t]);
                    m[t] = mn[t];
                    l[t] *= al;
#pragma unroll
                    for (int v = 0; v < NV; ++v) o[v][t] *= al;
                }
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                f32x4 vs[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) vs[j] = *reinterpret_cast<const f32x4 *>(sc + MAPS * 64 + ks * 32 + g * 8 + j * 4);
#pragma unroll
                for (int t = 0; t < SLOTS; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f32x4 w;
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(s[2 * ks + j][t][i], c2[t], (float)(14 - above) - m[t]));
                        l[t] += (w[0] + w[1]) + (w[2] + w[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) pf[ks][t][4 * j + i] = (_Float16)mul_zero(w[i], vs[j][i]);  // (a value that the mask hides may have no number for a scale)
                    }
            }
        }
        if (BUFS == 2) {
            at ^= TILE;
            if (kt0 + G < n_tiles) store(at);
            if (kt0 + 2 * G < n_tiles) fetch(key0 + 2 * G * 64);
        }
        if (seen)
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const f16x8 a = *reinterpret_cast<const f16x8 *>(kt_ + KB + (v * 16 + r16) * VS + ks * 64 + g * 16);
#pragma unroll
                    for (int t = 0; t < SLOTS; ++t) o[v][t] = mfma_f16(a, pf[ks][t], o[v][t]);
                }
    }
    {
        const float back = power2(above - 14);
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            l[t] *= back;
#pragma unroll
            for (int v = 0; v < NV; ++v) o[v][t] *= back;
        }
    }
    if (G == 2) {
        f32x4 *po = reinterpret_cast<f32x4 *>(lds);                                       // [wave][slot][NV][lane]
        float2 *pm = reinterpret_cast<float2 *>(lds + (size_t)4 * SLOTS * NV * 64 * 16);  // [wave][slot][lane]
        __syncthreads();
        if (grp == 1) {
#pragma unroll
            for (int t = 0; t < SLOTS; ++t) {
#pragma unroll
                for (int v = 0; v < NV; ++v) po[((wave * SLOTS + t) * NV + v) * 64 + lane] = o[v][t];
                pm[(wave * SLOTS + t) * 64 + lane] = float2{m[t], l[t]};
            }
        }
        __syncthreads();
        if (grp == 1) return;
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            const float2 b = pm[(wave * SLOTS + t) * 64 + lane];
            const float mx = fmaxf(m[t], b.x), wa = __builtin_amdgcn_exp2f(m[t] - mx), wb = __builtin_amdgcn_exp2f(b.x - mx);
            m[t] = mx, l[t] = l[t] * wa + b.y * wb;
#pragma unroll
            for (int v = 0; v < NV; ++v) o[v][t] = o[v][t] * wa + po[((wave * SLOTS + t) * NV + v) * 64 + lane] * wb;
        }
    }
    if (records) {
#pragma unroll
        for (int t = 0; t < SLOTS; ++t) {
            const int qi = qw + t / MAPS * 16 + r16;
            const float sum = rows_sum(l[t]);
            if (qi >= nq) continue;
            float *rec = records + ((((size_t)qi * heads + h) * MAPS + t % MAPS) * gridDim.y + blockIdx.y) * (kGqaRecHead + vdimp);
            if (g == 0) rec[0] = m[t], rec[1] = sum;
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (v * 16 < vdimp) *reinterpret_cast<f32x4 *>(rec + kGqaRecHead + v * 16 + g * 4) = o[v][t];
        }
        return;
    }
    float inv[SLOTS], gate[SLOTS / MAPS];
#pragma unroll
    for (int t = 0; t < SLOTS / MAPS; ++t) gate[t] = 1.0f;
#pragma unroll
    for (int t = 0; t < SLOTS; ++t) inv[t] = 1.0f / rows_sum(l[t]);
    if (p.gate && !(FAR && p.gate_columns))
#pragma unroll
        for (int t = 0; t < SLOTS / MAPS; ++t) gate[t] = activate(gate_logit(p, min(qw + t * 16 + r16, nq - 1), h, 0), BITNET_HIP_ACT_SIGMOID);
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
        const int qi = qw + t * 16 + r16;
        if (qi >= nq) continue;
        uint16_t *dst = out + (size_t)qi * ldo + (size_t)h * vdimp + g * 4;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (v * 16 < vdimp) {
                f32x4 q = o[v][t] * (inv[t] * gate[t]);
                if (FAR && p.gate_columns)
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[i] *= activate(gate_logit(p, qi, h, v * 16 + g * 4 + i), BITNET_HIP_ACT_SIGMOID);
                *reinterpret_cast<bf16x4 *>(dst + v * 16) = bf16x4{(__bf16)q.x, (__bf16)q.y, (__bf16)q.z, (__bf16)q.w};
            }
    }
}

size_t kv8_prefill_floats(const Gqa &g, int n_ctx, int nq) {
    const int parts = gqa_prefill_parts(g, n_ctx, nq);
    return parts > 1 ? (size_t)nq * g.heads * g.maps * parts * (kGqaRecHead + g.vdimp) : 0;
}

template <int NK, int NV, int G>
static hipError_t prefill_go(const Kv8 &c, const uint16_t *q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, float *records, hipStream_t s) {
    const Gqa &g = c.g;
    const int rows = g.maps == 2 ? 64 : 128, n_qb = (nq + rows - 1) / rows, parts = records ? gqa_prefill_parts(g, n_ctx, nq) : 1;
    if constexpr (G == 2)
        if (parts == 1 && !two_groups(g, rows, n_ctx, nq)) return prefill_go<NK, NV, 1>(c, q, ldq, n_ctx, nq, out, ldo, nullptr, s);
    const size_t tiles = (size_t)G * kv8_buffers(NK, NV, (int)g.maps) * kv8_tile_bytes(NK, NV, (int)g.maps), sums = G == 2 ? (size_t)4 * 2 * 64 * (NV * 16 + 8) : 0;
    const size_t lds = tiles > sums ? tiles : sums;
    auto fn = g.maps == 2 ? k_kv8_prefill<NK, NV, 2, false, G> : g.far_weight || g.gate_columns ? k_kv8_prefill<NK, NV, 1, true, G> : k_kv8_prefill<NK, NV, 1, false, G>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(fn, dim3(8 * ((g.heads + 7) / 8) * n_qb, parts), dim3(256 * G), lds, s, c, q, ldq, n_ctx, nq, out, ldo, n_qb, parts > 1 ? records : nullptr);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || parts == 1 ? e : launch_gqa_merge_parts(g, records, parts, nq, out, ldo, s);
}

// records: kv8_prefill_floats(g, n_ctx, nq) of them, or none where a block's keys stay together
hipError_t launch_kv8_prefill(const Kv8 &c, const uint16_t *q, size_t ldq, int n_ctx, int nq, uint16_t *out, size_t ldo, float *records, hipStream_t s) {
    const Gqa &g = c.g;
    if (!gqa_supported((int)g.dimp, (int)g.vdimp)) return hipErrorInvalidValue;
    if (g.dimp <= 64 && g.vdimp <= 64) return prefill_go<1, 4, 2>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
    if (g.dimp <= 64 && g.vdimp <= 128) return prefill_go<1, 8, 2>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
    if (g.dimp <= 128 && g.vdimp <= 128) return prefill_go<2, 8, 2>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
    return prefill_go<4, 16, 1>(c, q, ldq, n_ctx, nq, out, ldo, records, s);
}

}  // namespace bitnet_hip
