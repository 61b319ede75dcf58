// Attention of new tokens over a 4-bit cache (kv4.cuh), for sm_100a.
//
// out = softmax(scale q k^T) v with k = ks (kc - 8), v = vs (vc - 8) per group of 32 dimensions.  Nothing is dequantised: the codes
// are the MMAs' A operands.  A code of 0 .. 15 in the low bits of an fp16 is the subnormal code * 2^-24, exactly; masked in place
// by 0x000f000f or 0x00f000f0 (sixteen times that) a word of eight codes needs one shift and four ANDs.  For k q^T (keys are the
// MMA's 16 rows, query rows its 8 columns) the query is fp16, scaled per row by a power of two (a sixteenth where the codes count sixteen
// times), so its products are exact; a group's accumulator starts at -8 times the sum of the query over the group, and is
// multiplied by the key's scale at the end.  For v^T p^T (dimensions are the rows) the probabilities, transposed in registers, take the value's
// scale with them, one B operand per group, and one more MMA per group against a constant of 8 gives what the offset has to
// take off.  p is relative to the running maximum and, where all values' scales are small, to the largest power of two among them, so
// that p * vs lies in fp16's normal range wherever it matters.
//
// A warp takes 32 tokens at a time by itself: their codes and scales, four contiguous pieces of memory, arrive by cp.async.bulk in a ring of
// three places that is the warp's own, and are read from there in the order in which the fragments want them.
#pragma once
#include "kv4.cuh"
#include "w2_tile.cuh"

namespace tsp {

struct Kv4AttnParams {
    Kv4Side q;                             // [B][T][heads][D]
    Kv4Cache c;
    const long long *start, *counts;
    int start_stride;
    __nv_bfloat16* out;                    // [B][T][heads][D]
    float* part_o;                         // [item][split][rows][D], where there is more than one split
    float2* part_ml;                       // [item][split][rows]: reference of the exponents, sum
    int tokens, heads, window, splits, row_tiles, row_bytes;   // row_bytes: of a row's codes, D / 2
    float scale_log2;                      // log2(e) * softmax scale
    int* status;
};

constexpr int kKv4Warps = 4, kKv4Stages = 3;
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

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
template <bool V> struct Kv4Const { static constexpr bool value = V; };

// Four dimensions of a query row: val / sum as bf16; zero for a row that saw no key, NaN for a sequence outside of the cache.
__device__ __forceinline__ void kv4_store(const Kv4AttnParams& p, bool ok, int b, int hk, int per_kv, int row, int d, float4 val, float sum) {
    const int dim = 2 * (int)p.row_bytes;
    const float inv = sum == 0.f ? 0.f : 1.f / sum, nan = __int_as_float(0x7fffffff);
    const uint2 w = ok ? make_uint2(bf16_pack(val.x * inv, val.y * inv), bf16_pack(val.z * inv, val.w * inv)) : make_uint2(bf16_pack(nan, nan), bf16_pack(nan, nan));
    *reinterpret_cast<uint2*>(p.out + (((size_t)b * p.tokens + row / per_kv) * p.heads + hk * per_kv + row % per_kv) * dim + d) = w;
}

template <int D>
struct Kv4Stage {                          // 32 tokens of a head
    static constexpr int G = D / kKv4Group;
    static constexpr int codes = 32 * D / 2, scales = 32 * G * 2;
    static constexpr int vc = codes, ks = 2 * codes, vs = 2 * codes + scales, bytes = 2 * (codes + scales);
    static constexpr int ring = kKv4Stages * bytes;
};
constexpr int kKv4BarBytes = kKv4Warps * kKv4Stages * 8;

template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 4) {
        const uint4 v = lds128(addr);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (WORDS == 2) {
        const uint2 v = lds64(addr);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = lds32(addr);
    }
}
__device__ __forceinline__ uint32_t transposed_8x8(uint32_t v) {       // of b16: row g, columns 2q, 2q + 1 -> row 2q, 2q + 1, column g
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void fma2(float& d0, float& d1, float a0, float a1, float b) {
    const float2 r = f32x2_fma(make_float2(a0, a1), make_float2(b, b), make_float2(d0, d1));
    d0 = r.x, d1 = r.y;
}

// NT tiles of 8 query rows.  The warps of a CTA merge through shared memory; the splits of an item through distributed shared
// memory, where they are a cluster, or through the workspace.
template <int D, int NT, bool CLUSTER>
__global__ void __launch_bounds__(kKv4Warps * 32, NT == 1 ? 4 : 2) kv4_attn_kernel(const Kv4AttnParams p) {
    using St = Kv4Stage<D>;
    constexpr int G = St::G, ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];               // rings of the warps, then their barriers; the partial results at the end
    const uint32_t base_s = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int b = blockIdx.y, split = blockIdx.x % p.splits, item = blockIdx.x / p.splits;
    const int hk = item / p.row_tiles, tile = item % p.row_tiles;
    const int per_kv = p.heads / p.c.kv_heads, rows_all = p.tokens * per_kv, r0 = tile * ROWS, r_last = min(r0 + ROWS, rows_all) - 1;
    const int t_first = r0 / per_kv, t_last = r_last / per_kv;
    const Kv4Range rg = kv4_range(p.start, p.counts, p.start_stride, b, p.tokens, p.window, p.c.max_len, t_first, t_last);
    griddep_launch_dependents();

    const uint32_t ring = base_s + warp * St::ring, bars = base_s + kKv4Warps * St::ring + warp * kKv4Stages * 8;
    const size_t row0 = ((size_t)b * p.c.kv_heads + hk) * p.c.max_len;
    const int lo32 = rg.lo & ~31, blocks = (rg.hi - lo32 + 31) >> 5, stride = p.splits * kKv4Warps, first = split * kKv4Warps + warp;
    if (lane == 0) {
        for (int i = 0; i < kKv4Stages; ++i) mbar_init(bars + 8 * i, 1);
        mbar_fence_init();
    }
    auto fetch = [&](int block, int place) {
        if (lane == 0 && block < blocks) {
            const size_t row = row0 + lo32 + (size_t)block * 32;
            const uint32_t dst = ring + place * St::bytes, bar = bars + 8 * place;
            mbar_arrive_expect_tx(bar, St::bytes);
            bulk_load(dst, p.c.k_codes + row * (D / 2), St::codes, bar);
            bulk_load(dst + St::ks, p.c.k_scales + row * G, St::scales, bar);
            bulk_load(dst + St::vc, p.c.v_codes + row * (D / 2), St::codes, bar);
            bulk_load(dst + St::vs, p.c.v_scales + row * G, St::scales, bar);
        }
    };
#pragma unroll
    for (int i = 0; i < kKv4Stages; ++i) fetch(first + i * stride, i);
    __syncwarp();

    // ---- the query as B fragments: lane (g, q) has elements 8 q .. + 7 of every group of row 8 nt + g
    uint32_t qb[NT][G][2][2];
    float init[NT][G][2], row_f[NT][2];                            // of rows 2 q, 2 q + 1; row_f: what a raw score is multiplied by
    int row_pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + 8 * nt + g;
        const bool has = r < rows_all;
        const int t = has ? r / per_kv : 0, h = has ? hk * per_kv + r % per_kv : 0;
        const __nv_bfloat16* src = p.q.x + b * p.q.sb + t * p.q.st + h * p.q.sh;
        uint4 raw[G];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            raw[i] = has ? ld_cg_128(src + 32 * i + 8 * q) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[j])), fabsf(bf16_hi(w[j]))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^(14 - exponent of the largest): that one becomes 2^14 .. 2^15
        const int ex = min(max((int)(__float_as_uint(amax) >> 23), 30), 240) - 127;
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        const float f = p.scale_log2 * __uint_as_float((uint32_t)(127 + 10 + ex) << 23);   // 2^24 / up
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            row_f[nt][n] = __shfl_sync(0xffffffffu, f, (2 * q + n) * 4);
            row_pos[nt][n] = (int)min(rg.first_pos - t_first + (r0 + 8 * nt + 2 * q + n) / per_kv, 0x7fffffffll);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            float x[8], sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[2 * j] = bf16_lo(w[j]) * up, x[2 * j + 1] = bf16_hi(w[j]) * up;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += x[j];
            // A's halves are codes j of the low halfword and 4 + j of the high one
            qb[nt][i][0][0] = f16_pack(x[0], x[4]), qb[nt][i][0][1] = f16_pack(x[1] * 0.0625f, x[5] * 0.0625f);
            qb[nt][i][1][0] = f16_pack(x[2], x[6]), qb[nt][i][1][1] = f16_pack(x[3] * 0.0625f, x[7] * 0.0625f);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= -8.f / kTwo24;
#pragma unroll
            for (int n = 0; n < 2; ++n) init[nt][i][n] = __shfl_sync(0xffffffffu, sum, (2 * q + n) * 4);
        }
    }

    float o[NT][G][2][4], on[NT][G][4], m[NT][2], nb[NT][2], l[NT][2];   // m: running maximum of raw scores, nb: -(m row_f + vexp)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY, nb[nt][0] = nb[nt][1] = l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][i][0][e] = o[nt][i][1][e] = on[nt][i][e] = 0.f;
    }
    auto rescale = [&](int nt, float f0, float f1) {
        l[nt][0] *= f0, l[nt][1] *= f1;
#pragma unroll
        for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) o[nt][i][jj][0] *= f0, o[nt][i][jj][1] *= f1, o[nt][i][jj][2] *= f0, o[nt][i][jj][3] *= f1;
            on[nt][i][0] *= f0, on[nt][i][1] *= f1;
        }
    };
    int vexp = -14;                                                // exponent of the largest value scale so far, within -14 .. 0
    uint32_t vlimit = 2u << 10;                                    // fp16 bits of 2^(vexp + 1)

    // 16 keys, the first of them key0, in the half `u` of a place.  PART: some row does not see some of them.
    auto group = [&](uint32_t at, int u, int key0, auto part) {
        constexpr bool PART = decltype(part)::value;
        uint32_t k0[G], k1[G], s0w[G / 2], s1w[G / 2];
        lds_words(at + (u * 16 + g) * (D / 2) + q * (G * 4), k0);
        lds_words(at + (u * 16 + g + 8) * (D / 2) + q * (G * 4), k1);
        lds_words(at + St::ks + (u * 16 + g) * (G * 2), s0w);
        lds_words(at + St::ks + (u * 16 + g + 8) * (G * 2), s1w);
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint32_t a0[4] = {k0[i] & 0x000f000fu, k1[i] & 0x000f000fu, k0[i] & 0x00f000f0u, k1[i] & 0x00f000f0u};
            const uint32_t x = k0[i] >> 8, y = k1[i] >> 8;
            const uint32_t a1[4] = {x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u};
            const float f0 = i & 1 ? f16_hi(s0w[i / 2]) : f16_lo(s0w[i / 2]), f1 = i & 1 ? f16_hi(s1w[i / 2]) : f16_lo(s1w[i / 2]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float c[4] = {init[nt][i][0], init[nt][i][1], init[nt][i][0], init[nt][i][1]};
                float d[4];
                mma_f16(d, a0, qb[nt][i][0][0], qb[nt][i][0][1], c);
                mma_f16(d, a1, qb[nt][i][1][0], qb[nt][i][1][1], d);
                fma2(s[nt][0], s[nt][1], d[0], d[1], f0);
                fma2(s[nt][2], s[nt][3], d[2], d[3], f1);
            }
        }
        if constexpr (PART) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + g + 8 * (e >> 1), pos = row_pos[nt][e & 1];
                    if (key > pos || key >= rg.limit || (p.window > 0 && key <= pos - p.window)) s[nt][e] = -INFINITY;
                }
        }
        // ---- running maximum: the lanes of a row compare by themselves and confer only where one has more
        bool grown = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) grown |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] || fmaxf(s[nt][1], s[nt][3]) > m[nt][1];
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float f[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float mx = fmaxf(m[nt][n], fmaxf(s[nt][n], s[nt][2 + n]));
#pragma unroll
                    for (int j = 4; j < 32; j <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, j));
                    const float to = mx == -INFINITY ? 0.f : -(mx * row_f[nt][n] + (float)vexp);
                    f[n] = m[nt][n] == -INFINITY ? 0.f : ex2_approx(to - nb[nt][n]);
                    m[nt][n] = mx, nb[nt][n] = to;
                }
                rescale(nt, f[0], f[1]);
            }
        }
        // ---- probabilities, transposed to the B operand of the second product
        uint32_t pt[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = ex2_approx(fmaf(s[nt][e], row_f[nt][e & 1], nb[nt][e & 1]));
            l[nt][0] += s[nt][0] + s[nt][2], l[nt][1] += s[nt][1] + s[nt][3];
            pt[nt][0] = transposed_8x8(f16_pack(s[nt][0], s[nt][1]));
            pt[nt][1] = transposed_8x8(f16_pack(s[nt][2], s[nt][3]));
        }
        // ---- values
        uint32_t v[4][G / 2], w0[G], w1[G];
#pragma unroll
        for (int t = 0; t < 4; ++t) lds_words(at + St::vc + (u * 16 + 2 * q + (t & 1) + 8 * (t >> 1)) * (D / 2) + g * (G * 2), v[t]);
        lds_words(at + St::vs + (u * 16 + 2 * q) * (G * 2), w0);
        lds_words(at + St::vs + (u * 16 + 2 * q + 8) * (G * 2), w1);
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
            const uint32_t x = __byte_perm(v[0][i / 2], v[1][i / 2], sel), y = __byte_perm(v[2][i / 2], v[3][i / 2], sel), x8 = x >> 8, y8 = y >> 8;
            const uint32_t a0[4] = {x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};       // rows g: code 0, rows g + 8: code 1
            const uint32_t a1[4] = {x8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x000f000fu, y8 & 0x00f000f0u};   // codes 2, 3
            const uint32_t eight[4] = {0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u};
            const uint32_t f0 = __byte_perm(w0[i / 2], w0[G / 2 + i / 2], sel), f1 = __byte_perm(w1[i / 2], w1[G / 2 + i / 2], sel);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                uint32_t b0 = f16x2_mul(pt[nt][0], f0), b1 = f16x2_mul(pt[nt][1], f1);
                if constexpr (PART) {                              // a value that is not seen may be NaN
                    b0 &= __vcmpne2(pt[nt][0], 0u), b1 &= __vcmpne2(pt[nt][1], 0u);
                }
                mma_f16(o[nt][i][0], a0, b0, b1, o[nt][i][0]);
                mma_f16(o[nt][i][1], a1, b0, b1, o[nt][i][1]);
                mma_f16(on[nt][i], eight, b0, b1, on[nt][i]);
            }
        }
    };

    bool ok = true;
    int issued = first + kKv4Stages * stride;                      // next block to fetch
    int place = 0;
    uint32_t parity = 0;
#pragma unroll 1
    for (int block = first; block < blocks; block += stride) {
        if (!mbar_wait_bounded(bars + 8 * place, parity)) {
            ok = false;
            break;
        }
        const uint32_t at = ring + place * St::bytes;
        const int key0 = lo32 + block * 32;
        // ---- a value scale beyond the limit: lane = token
        uint32_t vw[G / 2], big = 0;
        lds_words(at + St::vs + lane * (G * 2), vw);
        const bool part = key0 + 32 > rg.limit || key0 + 31 > rg.first_pos || (p.window > 0 && key0 <= rg.first_pos + (t_last - t_first) - p.window);
        if (!part || (key0 + lane >= rg.lo && key0 + lane < rg.hi)) {
#pragma unroll
            for (int i = 0; i < G / 2; ++i) {
                uint32_t a = vw[i] & 0x7fffu, c = vw[i] >> 16 & 0x7fffu;
                a = a >= 0x7c00u ? 0u : a, c = c >= 0x7c00u ? 0u : c;   // (an infinite or NaN scale is the matter of the rows that see it)
                big = max(big, max(a, c));
            }
        }
        if (__any_sync(0xffffffffu, big >= vlimit)) {
            const int to = min((int)(__reduce_max_sync(0xffffffffu, big) >> 10) - 15, 0);
            const float f = __uint_as_float((uint32_t)(127 + vexp - to) << 23);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                rescale(nt, f, f);
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    if (m[nt][n] != -INFINITY) nb[nt][n] -= (float)(to - vexp);
            }
            vexp = to;
            vlimit = to == 0 ? 0x8000u : (uint32_t)(to + 16) << 10;
        }
        if (!part) {
            group(at, 0, key0, Kv4Const<false>());
            group(at, 1, key0 + 16, Kv4Const<false>());
        } else {
            group(at, 0, key0, Kv4Const<true>());
            if (key0 + 16 < rg.hi) group(at, 1, key0 + 16, Kv4Const<true>());
        }
        __syncwarp();                                              // the place may be filled again
        fetch(issued, place);
        issued += stride;
        if (++place == kKv4Stages) place = 0, parity ^= 1;
    }
    if (!ok) {                                                     // (no copy may land in memory that is used for something else)
        for (int i = 0; i < kKv4Stages; ++i) mbar_wait_bounded(bars + 8 * i, parity ^ (i < place ? 1u : 0u));
        if (lane == 0) atomicExch(p.status, ST_WAIT_TIMEOUT);
    }

    // ---- merge of the warps
    float(*os)[ROWS][D] = reinterpret_cast<float(*)[ROWS][D]>(smem);
    __shared__ float2 ml[kKv4Warps][ROWS], cta_ml[ROWS];
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float sum = l[nt][n];
#pragma unroll
            for (int j = 4; j < 32; j <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, j);
            const int r = 8 * nt + 2 * q + n;
            if (g == 0) ml[warp][r] = make_float2(m[nt][n] == -INFINITY ? -INFINITY : -nb[nt][n], ok ? sum : __int_as_float(0x7fffffff));
#pragma unroll
            for (int i = 0; i < G; ++i)
                *reinterpret_cast<float4*>(&os[warp][r][32 * i + 4 * g]) =
                    make_float4((o[nt][i][0][n] - on[nt][i][n]) * kTwo24, (o[nt][i][0][2 + n] * 0.0625f - on[nt][i][n]) * kTwo24,
                                (o[nt][i][1][n] - on[nt][i][n]) * kTwo24, (o[nt][i][1][2 + n] * 0.0625f - on[nt][i][n]) * kTwo24);
        }
    __syncthreads();
    if (!rg.ok && tid == 0) *p.status = 1;
    const size_t part0 = ((size_t)((size_t)b * p.c.kv_heads * p.row_tiles + item) * p.splits + split) * ROWS;
    constexpr int VECS = ROWS * D / 4;
#pragma unroll 1
    for (int x = tid; x < VECS; x += kKv4Warps * 32) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        float top = -INFINITY, sum = 0.f;
        float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kKv4Warps; ++w) top = fmaxf(top, ml[w][r].x);
#pragma unroll
        for (int w = 0; w < kKv4Warps; ++w) {
            const float f = ml[w][r].x == -INFINITY ? 0.f : ex2_approx(ml[w][r].x - top);
            sum += f * ml[w][r].y;
            if (f != 0.f) {
                const float4 y = *reinterpret_cast<const float4*>(&os[w][r][d]);
                val.x += f * y.x, val.y += f * y.y, val.z += f * y.z, val.w += f * y.w;
            }
        }
        if (CLUSTER) {                                             // (each thread reads and writes its own place of warp 0's part)
            *reinterpret_cast<float4*>(&os[0][r][d]) = val;
            if (d == 0) cta_ml[r] = make_float2(top, sum);
        } else if (p.splits > 1) {
            if (r0 + r >= rows_all) break;
            *reinterpret_cast<float4*>(p.part_o + (part0 + r) * D + d) = val;
            if (d == 0) p.part_ml[part0 + r] = make_float2(top, sum);
        } else {
            if (r0 + r >= rows_all) break;
            kv4_store(p, rg.ok, b, hk, per_kv, r0 + r, d, val, sum);
        }
    }
    if constexpr (CLUSTER) {
        cluster_arrive();
        cluster_wait();
        const uint32_t os_s = base_s, ml_s = smem_u32(cta_ml);
#pragma unroll 1
        for (int x = split * kKv4Warps * 32 + tid; x < VECS; x += p.splits * kKv4Warps * 32) {
            const int r = x / (D / 4), d = x % (D / 4) * 4;
            if (r0 + r >= rows_all) break;
            float2 st[8];
            float4 y[8];
            float top = -INFINITY, sum = 0.f;
            float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.splits) {
                    st[c] = ld_cluster_f2(map_to_rank(ml_s + r * 8, c));
                    y[c] = ld_cluster_f4(map_to_rank(os_s + (r * D + d) * 4, c));
                    top = fmaxf(top, st[c].x);
                }
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.splits) {
                    const float f = st[c].x == -INFINITY ? 0.f : ex2_approx(st[c].x - top);
                    sum += f * st[c].y;
                    if (f != 0.f) val.x += f * y[c].x, val.y += f * y[c].y, val.z += f * y[c].z, val.w += f * y[c].w;
                }
            kv4_store(p, rg.ok, b, hk, per_kv, r0 + r, d, val, sum);
        }
        cluster_arrive();                                          // nobody leaves while its results are read
        cluster_wait();
    }
}

// Joins the splits: a CTA per row.
template <int D, int NT>
__global__ void __launch_bounds__(D) kv4_attn_join_kernel(const Kv4AttnParams p) {
    constexpr int ROWS = 8 * NT;
    __shared__ float weight[1024];
    __shared__ float red[2][D / 32];
    const int d = threadIdx.x, b = blockIdx.y, r = blockIdx.x % ROWS, item = blockIdx.x / ROWS;
    const int hk = item / p.row_tiles, tile = item % p.row_tiles, per_kv = p.heads / p.c.kv_heads, rr = tile * ROWS + r;
    griddep_wait();
    if (rr >= p.tokens * per_kv) return;
    const size_t at = (size_t)((size_t)b * p.c.kv_heads * p.row_tiles + item) * p.splits;
    float top = -INFINITY, sum = 0.f, val = 0.f;
    for (int s = d; s < p.splits; s += D) top = fmaxf(top, p.part_ml[(at + s) * ROWS + r].x);
#pragma unroll
    for (int j = 16; j; j >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, j));
    if ((d & 31) == 0) red[0][d >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < D / 32; ++w) top = fmaxf(top, red[0][w]);
    for (int s = d; s < p.splits; s += D) {
        const float2 st = p.part_ml[(at + s) * ROWS + r];
        const float f = st.x == -INFINITY ? 0.f : ex2_approx(st.x - top);
        weight[s] = f;
        sum += f * st.y;
    }
#pragma unroll
    for (int j = 16; j; j >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, j);
    if ((d & 31) == 0) red[1][d >> 5] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) sum += red[1][w];
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) {
        const float f = weight[s], y = p.part_o[((at + s) * ROWS + r) * D + d];
        val += f != 0.f ? f * y : 0.f;
    }
    const long long start = p.start[b * p.start_stride], count = p.counts ? p.counts[b] : p.tokens;
    const float out = !kv4_fits(start, count, p.tokens, p.c.max_len) ? __int_as_float(0x7fffffff) : sum == 0.f ? 0.f : val / sum;
    p.out[(((size_t)b * p.tokens + rr / per_kv) * p.heads + hk * per_kv + rr % per_kv) * D + d] = __float2bfloat16_rn(out);
}

}  // namespace tsp
