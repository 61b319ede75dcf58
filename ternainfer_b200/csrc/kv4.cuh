// A key / value cache held in 4 bits, for sm_100a: writing new tokens (with their rotation) and reading them back.
//
// Each group of 32 values along a head shares one scale.  With m the group's value of largest magnitude (the positive one of
// two), scale = fp16(m / -8) and code = clamp(rint(x / scale) + 8, 0, 15), so that m itself has code 0 and a value stands for
// scale * (code - 8): 4.5 bits a value, for normally distributed groups a step 6 % smaller than that of 16 levels between
// minimum and maximum, which would also cost a second number per group.  A group of zeros has scale 0 and codes 8.
//
// Codes are kept in the order in which the lanes of the attention kernel take them (D / 32 groups of 16 bytes in natural order,
// two codes a byte, even element low): a key row holds word t of every group, t = 0 .. 3 - lane t of an MMA fragment reads its
// words of all groups with one load -, a value row halfword g of every group, g = 0 .. 7.
#pragma once
#include "attn_decode.cuh"
#include "rotary.cuh"

namespace tsp {

constexpr int kKv4Group = 32;
constexpr int kKv4Tile = 64;               // capacity of a cache is a multiple of this

struct Kv4Cache {
    uint8_t *k_codes, *v_codes;            // [B][Hkv][L][D / 2]
    __half *k_scales, *v_scales;           // [B][Hkv][L][D / 32]
    int kv_heads, max_len;
};

struct Kv4Side {
    const __nv_bfloat16* x;
    long long sb, st, sh;
};

struct Kv4AppendParams {
    Kv4Cache c;
    Kv4Side q, k, v;                       // q.x may be null
    __nv_bfloat16* q_out;                  // [B][T][heads][D]
    const float *cos_tab, *sin_tab;        // null: no rotation
    const long long *start, *counts;       // position of the first new token; new tokens (null: all)
    int start_stride;                      // 0: the same for every sequence
    FastDiv head_groups, tokens;
    int heads, rotary, half, table_len;
    int tables_16, rows_16;                // whether every table row, and every row of q, k and v, starts on 16 bytes
    int* status;
};

// Whether the `count` tokens of a sequence from position `start` on lie in the cache.
__device__ __forceinline__ bool kv4_fits(long long start, long long count, int tokens, int max_len) {
    return start >= 0 && count >= 0 && count <= tokens && start <= max_len && start + count <= max_len;
}

// Where 8 consecutive values of a row of codes lie, `u` the unit of 8: one word of a key row, two halfwords of a value row.
template <int D>
__device__ __forceinline__ void kv4_put_codes(uint8_t* row, bool key, int u, uint32_t codes) {
    constexpr int G = D / kKv4Group;
    const int i = u >> 2, t = u & 3;
    if (key) {
        *reinterpret_cast<uint32_t*>(row + (t * G + i) * 4) = codes;
    } else {
        *reinterpret_cast<uint16_t*>(row + (2 * t * G + i) * 2) = (uint16_t)codes;
        *reinterpret_cast<uint16_t*>(row + ((2 * t + 1) * G + i) * 2) = (uint16_t)(codes >> 16);
    }
}
template <int D>
__device__ __forceinline__ uint32_t kv4_get_codes(const uint8_t* row, bool key, int u) {
    constexpr int G = D / kKv4Group;
    const int i = u >> 2, t = u & 3;
    if (key) return *reinterpret_cast<const uint32_t*>(row + (t * G + i) * 4);
    return (uint32_t)*reinterpret_cast<const uint16_t*>(row + (2 * t * G + i) * 2) |
           (uint32_t)*reinterpret_cast<const uint16_t*>(row + ((2 * t + 1) * G + i) * 2) << 16;
}

constexpr int kKv4Heads = 4;               // rows of a token that a thread of the reading kernel takes a unit of

// A thread takes 8 consecutive values in HEADS heads of a token - queries (rotated into q_out), keys (rotated, quantised), values
// (quantised) -, all of them on their way before the first is used; four lanes share a group's scale.  Three prompts of 1,226 tokens, 20 + 2 x 5 heads
// of 128, rotation included, and the reading back of what was written: 26.5 us for 60 MB, of which 9.3 are the bytes; what bounds it is the
// instructions of a value (pair, maximum, quotient, packing, some 12): 68 % of the issue slots at 38 % of the warps.  A step of 8 tokens 5.9 us, two chains of
// latencies.
template <int D, int HEADS>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p, uint32_t items) {
    constexpr int U = D / 8, G = D / kKv4Group;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    const bool live = item < items;                                // (all lanes take part in the shuffles)
    const int u = item % U, e = u * 8, kv = p.c.kv_heads;
    uint32_t hg, t;
    const uint32_t bt = p.head_groups.div(live ? item / U : 0u, hg), b = p.tokens.div(bt, t);
    const long long start = p.start[(long long)b * p.start_stride], count = p.counts ? p.counts[b] : (long long)p.tokens.d;
    // a sequence is refused as a whole where one of its tokens lies outside of the cache or of the table: not written, its queries NaN
    const bool fits = kv4_fits(start, count, (int)p.tokens.d, p.c.max_len) && (!p.cos_tab || count == 0 || start + count <= p.table_len);
    if (!fits && live) *p.status = 1;
    const long long pos = start + t;
    const int half = p.rotary / 2;
    // (a padded query behind the table takes NaN as well, and is nobody's concern)
    const bool turns = p.cos_tab && e < p.rotary, pos_ok = fits && pos < p.table_len;
    // pairs of 8 values whose other halves are 8 values too, or neighbours: whole vectors
    const bool whole = p.half ? half % 8 == 0 : p.rotary % 8 == 0, second = p.half && e >= half;
    uint4 x[HEADS], y[HEADS];
    int kind[HEADS], head[HEADS];                          // 0 query, 1 key, 2 value
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = (int)hg * HEADS + i;
        kind[i] = h < p.heads ? 0 : h < p.heads + kv ? 1 : h < p.heads + 2 * kv ? 2 : 3;
        head[i] = kind[i] == 0 ? h : kind[i] == 1 ? h - p.heads : h - p.heads - kv;
        x[i] = y[i] = make_uint4(0, 0, 0, 0);
        if (!live || kind[i] == 3) continue;
        const Kv4Side& sd = kind[i] == 0 ? p.q : kind[i] == 1 ? p.k : p.v;
        const __nv_bfloat16* src = sd.x + (long long)b * sd.sb + (long long)t * sd.st + (long long)head[i] * sd.sh;
        if (p.rows_16) {
            x[i] = ld_cg_128(src + e);
            if (turns && p.half && whole && kind[i] < 2) y[i] = ld_cg_128(src + (second ? e - half : e + half));
        } else {
            const uint2 lo = *reinterpret_cast<const uint2*>(src + e), hi = *reinterpret_cast<const uint2*>(src + e + 4);
            x[i] = make_uint4(lo.x, lo.y, hi.x, hi.y);
            if (turns && p.half && whole && kind[i] < 2) {
                const __nv_bfloat16* o = src + (second ? e - half : e + half);
                const uint2 olo = *reinterpret_cast<const uint2*>(o), ohi = *reinterpret_cast<const uint2*>(o + 4);
                y[i] = make_uint4(olo.x, olo.y, ohi.x, ohi.y);
            }
        }
    }
    float c[8], s[8];
    if (turns && whole) {
        const long long row = (pos_ok ? pos : 0) * half;
        if (p.half) {
            table_values(p.cos_tab + row + (second ? e - half : e), p.tables_16, c);
            table_values(p.sin_tab + row + (second ? e - half : e), p.tables_16, s);
        } else {
            float c4[4], s4[4];
            table_values(p.cos_tab + row + e / 2, p.tables_16, c4);
            table_values(p.sin_tab + row + e / 2, p.tables_16, s4);
#pragma unroll
            for (int j = 0; j < 4; ++j) c[j] = c4[j], s[j] = s4[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = pos_ok ? c[j] : __int_as_float(0x7fffffff);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        float v[8];
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = bf16_lo(w[j]), v[2 * j + 1] = bf16_hi(w[j]);
        if (turns && kind[i] < 2 && live) {
            float r[8];
            if (whole && p.half) {
                const uint32_t o[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float other = j & 1 ? bf16_hi(o[j >> 1]) : bf16_lo(o[j >> 1]);
                    r[j] = second ? rot_b(other, v[j], c[j], s[j]) : rot_a(v[j], other, c[j], s[j]);
                }
            } else if (whole) {
#pragma unroll
                for (int j = 0; j < 4; ++j) r[2 * j] = rot_a(v[2 * j], v[2 * j + 1], c[j], s[j]), r[2 * j + 1] = rot_b(v[2 * j], v[2 * j + 1], c[j], s[j]);
            } else {                                               // the rotated part ends, or changes sides, inside of the 8 values
                const Kv4Side& sd = kind[i] == 0 ? p.q : p.k;
                const __nv_bfloat16* src = sd.x + (long long)b * sd.sb + (long long)t * sd.st + (long long)head[i] * sd.sh;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int d = e + j;
                    r[j] = v[j];
                    if (d >= p.rotary) continue;
                    const bool first = p.half ? d < half : !(d & 1);   // of its pair
                    const int pair = p.half ? (first ? d : d - half) : d >> 1;
                    const float other = p.half ? __bfloat162float(src[first ? d + half : d - half]) : v[j ^ 1];
                    const float cc = pos_ok ? p.cos_tab[pos * half + pair] : __int_as_float(0x7fffffff), ss = pos_ok ? p.sin_tab[pos * half + pair] : cc;
                    r[j] = first ? rot_a(v[j], other, cc, ss) : rot_b(other, v[j], cc, ss);
                }
            }
            x[i] = make_uint4(bf16_pack(r[0], r[1]), bf16_pack(r[2], r[3]), bf16_pack(r[4], r[5]), bf16_pack(r[6], r[7]));   // rounded as the activations are
            const uint32_t z[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) v[2 * j] = bf16_lo(z[j]), v[2 * j + 1] = bf16_hi(z[j]);
        }
        if (kind[i] == 0 && live) *reinterpret_cast<uint4*>(p.q_out + ((long long)bt * p.heads + head[i]) * D + e) = x[i];
        // (a half-warp or quarter has one head: its lanes go the same way up to here but for `live`)
        float hi = v[0], lo = v[0];
        bool nan = v[0] != v[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) hi = fmaxf(hi, v[j]), lo = fminf(lo, v[j]), nan |= v[j] != v[j];
#pragma unroll
        for (int m = 1; m < 4; m <<= 1) {
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
            nan |= __shfl_xor_sync(0xffffffffu, (int)nan, m) != 0;
        }
        if (!live || kind[i] == 0 || kind[i] == 3 || !fits || t >= count) continue;
        const __half scale = nan ? __ushort_as_half(0x7fff) : __float2half_rn((hi >= -lo ? hi : lo) * -0.125f);   // (a NaN stays one)
        const float sc = __half2float(scale), inv = __frcp_rn(sc);
        uint32_t code = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // a product with the reciprocal is within 2^-19 of the quotient; where that may matter the quotient decides
            const float t = v[j] * inv;
            float q = rintf(t);
            if (fabsf(t - q) > 0.4999f) q = rintf(__fdiv_rn(v[j], sc));
            q = sc == 0.f ? 8.f : fminf(fmaxf(q + 8.f, 0.f), 15.f);
            code |= (uint32_t)q << (4 * j);
        }
        const size_t row = ((size_t)b * kv + head[i]) * p.c.max_len + pos;
        kv4_put_codes<D>((kind[i] == 1 ? p.c.k_codes : p.c.v_codes) + row * (D / 2), kind[i] == 1, u, code);
        if ((u & 3) == 0) (kind[i] == 1 ? p.c.k_scales : p.c.v_scales)[row * G + (u >> 2)] = scale;
    }
}

struct Kv4ReadParams {
    Kv4Cache c;
    __nv_bfloat16 *k_out, *v_out;          // [B][T][Hkv][D]
    const long long *start, *counts;
    int start_stride;
    FastDiv head_groups, tokens;
    int* status;
};

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p, uint32_t items) {
    constexpr int U = D / 8, G = D / kKv4Group;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    if (item >= items) return;
    const int u = item % U, kv = p.c.kv_heads;
    uint32_t hg, t;
    const uint32_t bt = p.head_groups.div(item / U, hg), b = p.tokens.div(bt, t);
    const long long start = p.start[(long long)b * p.start_stride], count = p.counts ? p.counts[b] : (long long)p.tokens.d;
    const bool fits = kv4_fits(start, count, (int)p.tokens.d, p.c.max_len);
    if (!fits) *p.status = 1;
    uint32_t code[kKv4Heads];
    float scale[kKv4Heads];
#pragma unroll
    for (int i = 0; i < kKv4Heads; ++i) {
        const int h = (int)hg * kKv4Heads + i;
        const bool key = h < kv;
        code[i] = 0x88888888u, scale[i] = fits ? 0.f : __int_as_float(0x7fffffff);
        if (h >= 2 * kv || !fits || t >= count) continue;
        const size_t row = ((size_t)b * kv + (key ? h : h - kv)) * p.c.max_len + start + t;
        code[i] = kv4_get_codes<D>((key ? p.c.k_codes : p.c.v_codes) + row * (D / 2), key, u);
        scale[i] = __half2float((key ? p.c.k_scales : p.c.v_scales)[row * G + (u >> 2)]);
    }
#pragma unroll
    for (int i = 0; i < kKv4Heads; ++i) {
        const int h = (int)hg * kKv4Heads + i;
        if (h >= 2 * kv) continue;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = scale[i] * ((float)(code[i] >> (4 * j) & 15u) - 8.f);
        if (!(t < count)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = fits ? 0.f : scale[i];
        }
        __nv_bfloat16* dst = h < kv ? p.k_out + ((long long)bt * kv + h) * D : p.v_out + ((long long)bt * kv + h - kv) * D;
        *reinterpret_cast<uint4*>(dst + u * 8) = make_uint4(bf16_pack(x[0], x[1]), bf16_pack(x[2], x[3]), bf16_pack(x[4], x[5]), bf16_pack(x[6], x[7]));
    }
}

}  // namespace tsp
