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
    int tokens, heads, rotary, half, table_len;
    int* status;
};

// Whether the `count` tokens of a sequence from position `start` on lie in the cache.
__device__ __forceinline__ bool kv4_fits(long long start, long long count, int tokens, int max_len) {
    return start >= 0 && count >= 0 && count <= tokens && start <= max_len && start + count <= max_len;
}

// One row (head of a token) per D / 4 lanes, 4 values a lane.  Rows: queries (rotated into q_out), keys (rotated, quantised),
// values (quantised).
template <int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p, long long rows) {
    constexpr int LANES = D / 4;
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES, e = lane * 4;
    const bool live = r < rows;                                    // (all lanes take part in the shuffles)
    const int kv = p.c.kv_heads, per_token = (p.q.x ? p.heads : 0) + 2 * kv;
    const long long bt = live ? r / per_token : 0, b = bt / p.tokens, t = bt - b * p.tokens;
    int h = live ? (int)(r - bt * per_token) : 0;
    const bool is_q = p.q.x && h < p.heads;
    if (!is_q && p.q.x) h -= p.heads;
    const bool is_k = !is_q && h < kv;
    if (!is_q && !is_k) h -= kv;
    const Kv4Side& sd = is_q ? p.q : is_k ? p.k : p.v;
    const __nv_bfloat16* src = sd.x + b * sd.sb + t * sd.st + h * sd.sh;
    const long long start = p.start[b * p.start_stride], count = p.counts ? p.counts[b] : p.tokens;
    const bool fits = kv4_fits(start, count, p.tokens, p.c.max_len);
    const long long pos = start + t;
    if (!fits && live) *p.status = 1;

    const uint2 raw = *reinterpret_cast<const uint2*>(src + e);
    float x[4] = {bf16_lo(raw.x), bf16_hi(raw.x), bf16_lo(raw.y), bf16_hi(raw.y)};
    if (p.cos_tab && (is_q || is_k)) {
        const int half = p.rotary / 2;
        const bool ok = pos >= 0 && pos < p.table_len;
        // a padded query lies behind the table at most where the cache ends: it takes NaN, and is nobody's concern
        if (live && fits && t < count && !ok) *p.status = 1;
        const float* ct = p.cos_tab + (ok ? pos : 0) * half;
        const float* st = p.sin_tab + (ok ? pos : 0) * half;
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = e + i;
            y[i] = x[i];
            if (d >= p.rotary) continue;
            const bool first = p.half ? d < half : !(d & 1);       // of its pair
            const int pair = p.half ? (first ? d : d - half) : d >> 1;
            const float other = p.half ? __bfloat162float(src[first ? d + half : d - half]) : x[i ^ 1];
            const float c = ok ? ct[pair] : __int_as_float(0x7fffffff), s = ok ? st[pair] : c;
            y[i] = first ? rot_a(x[i], other, c, s) : rot_b(other, x[i], c, s);
        }
        const uint32_t lo = bf16_pack(y[0], y[1]), hi = bf16_pack(y[2], y[3]);   // rounded as the activations are
        x[0] = bf16_lo(lo), x[1] = bf16_hi(lo), x[2] = bf16_lo(hi), x[3] = bf16_hi(hi);
    }
    if (is_q) {
        if (live) *reinterpret_cast<uint2*>(p.q_out + (bt * p.heads + h) * D + e) = make_uint2(bf16_pack(x[0], x[1]), bf16_pack(x[2], x[3]));
    }
    float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
    bool nan = x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3];
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        nan |= __shfl_xor_sync(0xffffffffu, (int)nan, m) != 0;
    }
    if (!live || is_q || !fits || t >= count) return;
    const __half scale = nan ? __ushort_as_half(0x7fff) : __float2half_rn((hi >= -lo ? hi : lo) * -0.125f);   // (a NaN stays one)
    const float s = __half2float(scale);
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float c = s == 0.f ? 8.f : fminf(fmaxf(rintf(__fdiv_rn(x[i], s)) + 8.f, 0.f), 15.f);
        code |= (uint32_t)c << (4 * i);
    }
    constexpr int G = D / kKv4Group;
    const int i = lane >> 3, g = lane & 7;
    const size_t row = ((size_t)b * kv + h) * p.c.max_len + pos;
    uint8_t* codes = (is_k ? p.c.k_codes : p.c.v_codes) + row * (D / 2);
    const int at = is_k ? ((g >> 1) * G + i) * 4 + (g & 1) * 2 : (g * G + i) * 2;
    *reinterpret_cast<uint16_t*>(codes + at) = (uint16_t)code;
    if (g == 0) (is_k ? p.c.k_scales : p.c.v_scales)[row * G + i] = scale;
}

struct Kv4ReadParams {
    Kv4Cache c;
    __nv_bfloat16 *k_out, *v_out;          // [B][T][Hkv][D]
    const long long *start, *counts;
    int start_stride, tokens;
    int* status;
};

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p, long long rows) {
    constexpr int LANES = D / 4, G = D / kKv4Group;
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
    if (r >= rows) return;
    const int lane = threadIdx.x % LANES, kv = p.c.kv_heads, hk = (int)(r % (2 * kv)), i = lane >> 3, g = lane & 7;
    const long long bt = r / (2 * kv), b = bt / p.tokens, t = bt - b * p.tokens;
    const bool is_k = hk < kv;
    const int h = is_k ? hk : hk - kv;
    const long long start = p.start[b * p.start_stride], count = p.counts ? p.counts[b] : p.tokens;
    const bool fits = kv4_fits(start, count, p.tokens, p.c.max_len);
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (!fits) {
        x[0] = x[1] = x[2] = x[3] = __int_as_float(0x7fffffff);
        *p.status = 1;
    } else if (t < count) {
        const size_t row = ((size_t)b * kv + h) * p.c.max_len + start + t;
        const int at = is_k ? ((g >> 1) * G + i) * 4 + (g & 1) * 2 : (g * G + i) * 2;
        const uint32_t code = *reinterpret_cast<const uint16_t*>((is_k ? p.c.k_codes : p.c.v_codes) + row * (D / 2) + at);
        const float s = __half2float((is_k ? p.c.k_scales : p.c.v_scales)[row * G + i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s * ((float)(code >> (4 * j) & 15u) - 8.f);
    }
    *reinterpret_cast<uint2*>((is_k ? p.k_out : p.v_out) + (bt * kv + h) * D + lane * 4) = make_uint2(bf16_pack(x[0], x[1]), bf16_pack(x[2], x[3]));
}

}  // namespace tsp
