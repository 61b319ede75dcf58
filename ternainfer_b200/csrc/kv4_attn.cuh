// Attention of new tokens over a 4-bit cache (kv4.cuh), for sm_100a.
//
// out = softmax(scale q k^T) v with k = ks (kc - 8), v = vs (vc - 8) per group of 32 dimensions.  Nothing is dequantised: the codes
// are the MMAs' operands.  A code of 0 .. 15 in the low bits of an fp16 is the subnormal code * 2^-24, exactly; masked in place
// by 0x000f000f or 0x00f000f0 (sixteen times that) a word of eight codes needs one shift and four ANDs.  For q k^T the query
// is fp16, scaled per row by a power of two (a sixteenth where the codes count sixteen times), so its products are exact; a
// group's accumulator starts at -8 times the sum of the query over the group, and is multiplied by the key's scale at the end.
// For p v the probabilities take the value's scale with them, one A operand per group, and one more MMA per group against a
// constant of 8 gives what the offset has to take off.  p is relative to the running maximum and to the largest power of two
// among the values' scales so far, so that p * vs stays below 2 and within fp16's normal range wherever it matters.
#pragma once
#include "kv4.cuh"

namespace tsp {

struct Kv4AttnParams {
    Kv4Side q;                             // [B][T][heads][D]
    Kv4Cache c;
    const long long *start, *counts;
    int start_stride;
    __nv_bfloat16* out;                    // [B][T][heads][D]
    float* part_o;                         // [item][split][rows][D], where there is more than one split
    float2* part_ml;                       // [item][split][rows]: reference of the exponents, sum
    int tokens, heads, window, splits, row_tiles;
    float scale_log2;                      // log2(e) * softmax scale
    int* status;
};

constexpr int kKv4Warps = 4;
constexpr float kTwo24 = 16777216.f;

// D(16x8) += A(16x16) * B(16x8), fp16 in, fp32 out
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t f16_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16_lo(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v & 0xffffu))); }
__device__ __forceinline__ float f16_hi(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }

// What the rows of one CTA see: row i of the tile is query token (r0 + i) / G of query head kv * G + (r0 + i) % G.
struct Kv4Range {
    long long first_pos;                   // of row 0's token
    long long limit;                       // keys below it exist
    int lo, hi;                            // keys that some row may see
    bool ok;
};
__device__ __forceinline__ Kv4Range kv4_range(const long long* start_p, const long long* counts, int start_stride, int b, int tokens, int window,
                                              int max_len, int t_first, int t_last) {
    Kv4Range r;
    const long long start = start_p[b * start_stride], count = counts ? counts[b] : tokens;
    r.ok = kv4_fits(start, count, tokens, max_len);
    r.first_pos = start + t_first;
    r.limit = r.ok ? start + count : 0;
    const long long hi = min(start + t_last + 1, r.limit), lo = window > 0 ? max(start + t_first - window + 1, 0ll) : 0ll;
    r.hi = r.ok ? (int)hi : 0;
    r.lo = r.ok ? (int)min(lo, hi) : 0;
    return r;
}

// ROWS: rows of the tile, 8 or 16.  A warp takes groups of 16 keys by itself; the warps of a CTA merge through shared memory, the
// splits of an item through the workspace.
template <int D, int ROWS>
__global__ void __launch_bounds__(kKv4Warps * 32) kv4_attn_kernel(const Kv4AttnParams p) {
    constexpr int G = D / kKv4Group, KW = G, NT = D / 8;           // groups; words of a key row per lane; tiles of 8 dimensions
    constexpr int HALVES = ROWS / 8;
    __shared__ __align__(16) float os[kKv4Warps][ROWS][D];
    __shared__ float2 ml[kKv4Warps][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
    const int b = blockIdx.y, split = blockIdx.x % p.splits, item = blockIdx.x / p.splits;
    const int hk = item / p.row_tiles, tile = item % p.row_tiles;
    const int per_kv = p.heads / p.c.kv_heads, rows_all = p.tokens * per_kv, r0 = tile * ROWS, r_last = min(r0 + ROWS, rows_all) - 1;
    const Kv4Range rg = kv4_range(p.start, p.counts, p.start_stride, b, p.tokens, p.window, p.c.max_len, r0 / per_kv, r_last / per_kv);
    const int t_first = r0 / per_kv;

    // ---- the query as A fragments
    uint32_t a[G][2][4];
    float init[G][4], row_f[2];                                    // row_f: what a raw score is multiplied by
    int row_pos[2];                                                // position of the row's token (clamped: below 2^31)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int r = r0 + g + 8 * e;
        const bool has = e < HALVES && r < rows_all;
        const int t = has ? r / per_kv : 0, h = has ? hk * per_kv + r % per_kv : 0;
        row_pos[e] = (int)min(rg.first_pos - t_first + t, 0x7fffffffll);
        const __nv_bfloat16* src = p.q.x + b * p.q.sb + t * p.q.st + h * p.q.sh;
        uint4 raw[G];                                              // elements 32 i + 8 q .. + 7
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            raw[i] = has ? *reinterpret_cast<const uint4*>(src + 32 * i + 8 * q) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[j])), fabsf(bf16_hi(w[j]))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^(14 - exponent of the largest): that one becomes 2^14 .. 2^15
        const int ex = min(max((int)(__float_as_uint(amax) >> 23), 30), 240) - 127;
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        row_f[e] = p.scale_log2 * __uint_as_float((uint32_t)(127 + 10 + ex) << 23);   // 2^24 / up
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float x[8], sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[2 * j] = bf16_lo(w[j]) * up, x[2 * j + 1] = bf16_hi(w[j]) * up;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += x[j];
            // B's halves are codes j of the low halfword and 4 + j of the high one
            a[i][0][e] = f16_pack(x[0], x[4]), a[i][0][2 + e] = f16_pack(x[1] * 0.0625f, x[5] * 0.0625f);
            a[i][1][e] = f16_pack(x[2], x[6]), a[i][1][2 + e] = f16_pack(x[3] * 0.0625f, x[7] * 0.0625f);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            init[i][2 * e] = init[i][2 * e + 1] = sum * (-8.f / kTwo24);
        }
    }

    float o[NT][4], on[G][4], base[2] = {-INFINITY, -INFINITY}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int vexp = -24;                                                // exponent of the largest value scale so far
#pragma unroll
    for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) on[i][0] = on[i][1] = on[i][2] = on[i][3] = 0.f;

    const size_t row0 = ((size_t)b * p.c.kv_heads + hk) * p.c.max_len;
    const uint8_t *kc = p.c.k_codes + row0 * (D / 2) + q * (KW * 4), *vc = p.c.v_codes + row0 * (D / 2) + g * (G * 2);
    const __half *ks = p.c.k_scales + row0 * G, *vs = p.c.v_scales + row0 * G;
    const int lo16 = rg.lo & ~15, groups = (rg.hi - lo16 + 15) >> 4, stride = p.splits * kKv4Warps;
    const bool plain_rows = rg.ok;

    uint32_t kf[2][KW], vf[4][G / 2], ksf[2][G], vsf[2][G];        // (scales: two tokens' G halves = G words)
    auto load = [&](int grp) {
        const size_t key = (size_t)lo16 + (size_t)grp * 16;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint8_t* src = kc + (key + 8 * t + g) * (D / 2);
            const __half *s1 = ks + (key + 8 * t + 2 * q) * G, *s2 = vs + (key + 8 * t + 2 * q) * G;
            if constexpr (D == 128) {
                const uint4 w = ldg_128(src), x = ldg_128(s1), y = ldg_128(s2);
                kf[t][0] = w.x, kf[t][1] = w.y, kf[t][2] = w.z, kf[t][3] = w.w;
                ksf[t][0] = x.x, ksf[t][1] = x.y, ksf[t][2] = x.z, ksf[t][3] = x.w;
                vsf[t][0] = y.x, vsf[t][1] = y.y, vsf[t][2] = y.z, vsf[t][3] = y.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(src), x = *reinterpret_cast<const uint2*>(s1), y = *reinterpret_cast<const uint2*>(s2);
                kf[t][0] = w.x, kf[t][1] = w.y, ksf[t][0] = x.x, ksf[t][1] = x.y, vsf[t][0] = y.x, vsf[t][1] = y.y;
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint8_t* src = vc + (key + 2 * q + (t & 1) + 8 * (t >> 1)) * (D / 2);
            if constexpr (D == 128) {
                const uint2 w = *reinterpret_cast<const uint2*>(src);
                vf[t][0] = w.x, vf[t][1] = w.y;
            } else {
                vf[t][0] = *reinterpret_cast<const uint32_t*>(src);
            }
        }
    };
    // scale of group i of token 2 q + n of tile t
    auto scale_of = [](const uint32_t (&f)[2][G], int t, int n, int i) {
        const uint32_t w = f[t][n * (G / 2) + i / 2];
        return i & 1 ? f16_hi(w) : f16_lo(w);
    };

    int grp = split * kKv4Warps + warp;
    if (plain_rows && grp < groups) load(grp);
#pragma unroll 1
    for (; plain_rows && grp < groups; grp += stride) {
        const int key0 = lo16 + grp * 16;
        // ---- scores: 16 keys
        float s[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const uint32_t w = kf[t][i], w8 = w >> 8;
                float d[4];
                mma_f16(d, a[i][0], w & 0x000f000fu, w & 0x00f000f0u, init[i]);
                mma_f16(d, a[i][1], w8 & 0x000f000fu, w8 & 0x00f000f0u, d);
                const float s0 = scale_of(ksf, t, 0, i), s1 = scale_of(ksf, t, 1, i);
                s[t][0] += d[0] * s0, s[t][1] += d[1] * s1;
                if (HALVES > 1) s[t][2] += d[2] * s0, s[t][3] += d[3] * s1;
            }
        }
        uint32_t big = 0;
        float vsc[2][2][G];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < G; ++i) vsc[t][n][i] = scale_of(vsf, t, n, i);
        // ---- keys that some row does not see
        const bool part = key0 + 16 > rg.limit || key0 + 15 > rg.first_pos || (p.window > 0 && key0 <= rg.first_pos + (r_last / per_kv - t_first) - p.window);
        bool hide[2][4];
        if (part) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + 8 * t + 2 * q + (e & 1), pos = row_pos[e >> 1];
                    hide[t][e] = key > pos || key >= rg.limit || (p.window > 0 && key <= pos - p.window);
                    if (hide[t][e]) s[t][e] = -INFINITY;
                }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int n = 0; n < 2; ++n)                        // rows without a token hold anything
                    if (key0 + 8 * t + 2 * q + n >= rg.limit)
#pragma unroll
                        for (int i = 0; i < G; ++i) vsc[t][n][i] = 0.f;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < G; ++i) big = max(big, __float_as_uint(fabsf(vsc[t][n][i])));
        // ---- running maximum
        float mx[2];
#pragma unroll
        for (int e = 0; e < HALVES; ++e) {
            mx[e] = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
            mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2)) * row_f[e];
        }
        int big_exp = (int)(big >> 23) - 127;
        const bool grown = mx[0] > m[0] || (HALVES > 1 && mx[HALVES - 1] > m[HALVES - 1]) || big_exp > vexp;
        if (__any_sync(0xffffffffu, grown)) {
            if (big_exp == 128) {                                  // an infinite or NaN scale is the matter of the rows that see it alone
                big = 0;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int i = 0; i < G; ++i)
                            if (fabsf(vsc[t][n][i]) < INFINITY) big = max(big, __float_as_uint(fabsf(vsc[t][n][i])));
                big_exp = (int)(big >> 23) - 127;
            }
            vexp = max(vexp, __reduce_max_sync(0xffffffffu, big_exp));
#pragma unroll
            for (int e = 0; e < HALVES; ++e) {
                m[e] = fmaxf(m[e], mx[e]);
                const float to = m[e] + (float)vexp;               // (-inf until the row has seen a key)
                const float r = base[e] == -INFINITY ? 0.f : ex2_approx(base[e] - to);
                base[e] = to;
                l[e] *= r;
#pragma unroll
                for (int j = 0; j < NT; ++j) o[j][2 * e] *= r, o[j][2 * e + 1] *= r;
#pragma unroll
                for (int i = 0; i < G; ++i) on[i][2 * e] *= r, on[i][2 * e + 1] *= r;
            }
        }
        // ---- probabilities
#pragma unroll
        for (int e = 0; e < 2 * HALVES; ++e) {
            const float bs = base[e >> 1] == -INFINITY ? 0.f : base[e >> 1];
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t][e] = ex2_approx(fmaf(s[t][e], row_f[e >> 1], -bs)), l[e >> 1] += s[t][e];
        }
        // ---- values
#pragma unroll
        for (int i = 0; i < G; ++i) {
            uint32_t pa[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < HALVES; ++e) {
                    float x = s[t][2 * e] * vsc[t][0][i], y = s[t][2 * e + 1] * vsc[t][1][i];
                    if (part) x = hide[t][2 * e] ? 0.f : x, y = hide[t][2 * e + 1] ? 0.f : y;   // (a hidden value may be NaN)
                    pa[2 * t + e] = f16_pack(x, y);
                }
            const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
            const uint32_t x = __byte_perm(vf[0][i / 2], vf[1][i / 2], sel), y = __byte_perm(vf[2][i / 2], vf[3][i / 2], sel);
            const uint32_t x8 = x >> 8, y8 = y >> 8;
            mma_f16(o[4 * i], pa, x & 0x000f000fu, y & 0x000f000fu, o[4 * i]);
            mma_f16(o[4 * i + 1], pa, x & 0x00f000f0u, y & 0x00f000f0u, o[4 * i + 1]);
            mma_f16(o[4 * i + 2], pa, x8 & 0x000f000fu, y8 & 0x000f000fu, o[4 * i + 2]);
            mma_f16(o[4 * i + 3], pa, x8 & 0x00f000f0u, y8 & 0x00f000f0u, o[4 * i + 3]);
            mma_f16(on[i], pa, 0x00080008u, 0x00080008u, on[i]);
        }
        if (grp + stride < groups) load(grp + stride);
    }
    // ---- merge of the warps
#pragma unroll
    for (int e = 0; e < HALVES; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (q == 0) ml[warp][g + 8 * e] = make_float2(base[e], l[e]);
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int n = 0; n < 2; ++n) {                          // dimensions 32 i + 8 q + 4 n .. + 3
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = (o[4 * i + j][2 * e + n] * (j & 1 ? 0.0625f : 1.f) - on[i][2 * e + n]) * kTwo24;
                *reinterpret_cast<float4*>(&os[warp][g + 8 * e][32 * i + 8 * q + 4 * n]) = make_float4(v[0], v[1], v[2], v[3]);
            }
    }
    __syncthreads();
    if (!rg.ok && threadIdx.x == 0) *p.status = 1;
    for (int x = threadIdx.x; x < ROWS * D; x += kKv4Warps * 32) {
        const int r = x / D, d = x % D;
        if (r0 + r >= rows_all) break;
        float top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
        for (int w = 0; w < kKv4Warps; ++w) top = fmaxf(top, ml[w][r].x);
#pragma unroll
        for (int w = 0; w < kKv4Warps; ++w) {
            const float f = ml[w][r].x == -INFINITY ? 0.f : ex2_approx(ml[w][r].x - top);
            sum += f * ml[w][r].y;
            if (f != 0.f) val += f * os[w][r][d];
        }
        if (p.splits > 1) {
            const size_t at = ((size_t)((size_t)b * p.c.kv_heads * p.row_tiles + item) * p.splits + split) * ROWS + r;
            p.part_o[at * D + d] = val;
            if (d == 0) p.part_ml[at] = make_float2(top, sum);
        } else {
            const int t = (r0 + r) / per_kv, h = hk * per_kv + (r0 + r) % per_kv;
            const float out = !rg.ok ? __int_as_float(0x7fffffff) : sum == 0.f ? 0.f : val / sum;   // (a row that sees no key is zero)
            p.out[(((size_t)b * p.tokens + t) * p.heads + h) * D + d] = __float2bfloat16_rn(out);
        }
    }
}

// Joins the splits: a CTA per row.
template <int D, int ROWS>
__global__ void __launch_bounds__(D) kv4_attn_join_kernel(const Kv4AttnParams p) {
    const int d = threadIdx.x, b = blockIdx.y, r = blockIdx.x % ROWS, item = blockIdx.x / ROWS;
    const int hk = item / p.row_tiles, tile = item % p.row_tiles, per_kv = p.heads / p.c.kv_heads, rr = tile * ROWS + r;
    if (rr >= p.tokens * per_kv) return;
    const size_t at = (size_t)((size_t)b * p.c.kv_heads * p.row_tiles + item) * p.splits;
    float top = -INFINITY, sum = 0.f, val = 0.f;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_ml[(at + s) * ROWS + r].x);
    for (int s = 0; s < p.splits; ++s) {
        const float2 st = p.part_ml[(at + s) * ROWS + r];
        const float f = st.x == -INFINITY ? 0.f : ex2_approx(st.x - top);
        sum += f * st.y;
        if (f != 0.f) val += f * p.part_o[((at + s) * ROWS + r) * D + d];
    }
    const long long start = p.start[b * p.start_stride], count = p.counts ? p.counts[b] : p.tokens;
    const float out = !kv4_fits(start, count, p.tokens, p.c.max_len) ? __int_as_float(0x7fffffff) : sum == 0.f ? 0.f : val / sum;
    p.out[(((size_t)b * p.tokens + rr / per_kv) * p.heads + hk * per_kv + rr % per_kv) * D + d] = __float2bfloat16_rn(out);
}

}  // namespace tsp
