// Attention of new tokens over a 4-bit cache (kv4.cuh), for sm_100a.
//
// out = softmax(scale q k^T) v with k = ks (kc - 8), v = vs (vc - 8) per group of 32 dimensions.  Nothing is dequantised: the codes
// are the MMAs' A operands.  A code of 0 .. 15 in the low bits of an fp16 is the subnormal code * 2^-24, exactly; masked in place
// by 0x000f000f or 0x00f000f0 (sixteen times that) a word of eight codes needs one shift and four ANDs.  For k q^T (keys are the
// MMA's 16 rows, query rows its 8 columns) the query is fp16, scaled per row by a power of two (a sixteenth where the codes count sixteen
// times), so its products are exact; a group's accumulator is multiplied by the key's scale at the end, and one MMA per 16 keys, of their scales
// against -8 times the sums of the query over the groups (in two fp16 parts), takes the offset off.  For v^T p^T (dimensions are the rows) the probabilities, transposed in registers, take the value's
// scale with them, one B operand per group, and one more MMA per group against a constant of 8 gives what the offset has to
// take off.  p is relative to the running maximum and to the largest power of two among the values' scales, so that p and p * vs lie in
// fp16's normal range wherever it matters: down to values of 3e-6, where a scale is two of fp16's last places.
// Probabilities, and their products with the value scales, are rounded to fp16 because that is what the MMA takes; the errors of the results against 64 bits
// go from 1.66e-3 (their own rounding to bf16) to 1.67e-3.  The MMA lines subnormal operands up as if they were 2^-14, and cuts sums off at some 2^-14 of p vs,
// an eighth of what that rounding leaves in a value of one step: a value of 0 under one key that has all of the weight comes out as some 2^-17 of the largest.
//
// A warp takes 32 tokens at a time by itself: their codes and scales, four contiguous pieces of memory, arrive by cp.async in a ring of
// three places that is the warp's own, and are read from there in the order in which the fragments want them.  (Bulk copies of 256 bytes to
// 2 KB, four to a block, came at 1.7 TB/s: the copy engine takes them one by one.)
//
// What bounds it is a block's instructions: some 300 for 32 keys of 128 and 8 query rows, of which the MMAs are a fifth of the tensor pipe, at 16 warps
// an SM and 1.7 instructions a clock.  32 sequences of 8,000 keys, 64 heads over 8: 62 us, 3.6 TB/s of 6.46; 131,000 keys, 20 heads over 5: 33.6 us, 2.8
// TB/s, the join included; 600 keys 6.5 us, a chain of latencies.
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
    float* part_o;                         // KV4_STREAM: [CTA][first, last item][rows][D]; kv4_prefill_kernel in parts: [CTA][rows][D]
    float2* part_ml;                       // the same without [D]: reference of the exponents, sum
    int batch, tokens, heads, window;
    int cluster, row_tiles, row_bytes;     // CTAs of a cluster (kv4_prefill_kernel: for a tile); tiles of rows per key / value head; D / 2
    float scale_log2;                      // log2(e) * softmax scale
    int* status;
};

constexpr int kKv4Warps = 4, kKv4Stages = 3, kKv4JoinWarps = 32;
constexpr float kTwo24 = 16777216.f;
// Probabilities are at most 2^(kKv4Slack - kKv4MinExp) = 2^14, and products with a scale 2^(kKv4Slack + 1), or what the largest scale is where
// that is above 2^kKv4MaxExp: fp16 holds them.
constexpr int kKv4Slack = 8, kKv4MinExp = -6, kKv4MaxExp = 8;

// D(16x8) += A(16x16) * B(16x8), fp16 in, fp32 out
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// D = A * B
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// D(16x8) = A(16x8) * B(8x8)
__device__ __forceinline__ void mma_f16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
__device__ __forceinline__ uint32_t f16_pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16_lo(uint32_t v) {
    float r;
    asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, lo; }" : "=f"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float f16_hi(uint32_t v) {
    float r;
    asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %1; cvt.f32.f16 %0, hi; }" : "=f"(r) : "r"(v));
    return r;
}

// What the rows of one CTA see: row i of the tile is query token (r0 + i) / G of query head kv * G + (r0 + i) % G.
struct Kv4Range {
    int first_pos;                         // of row 0's token
    int limit;                             // keys below it exist
    int lo, hi;                            // keys that some row may see
    bool ok;
};
__device__ __forceinline__ Kv4Range kv4_range(const long long* start_p, const long long* counts, int start_stride, int b, int tokens, int window,
                                              int max_len, int t_first, int t_last) {
    Kv4Range r;
    const long long start = start_p[b * start_stride], count = counts ? counts[b] : tokens;
    r.ok = kv4_fits(start, count, tokens, max_len);
    if (!r.ok) {
        r.first_pos = r.limit = r.lo = r.hi = 0;
        return r;
    }
    r.first_pos = (int)start + t_first;    // (below 2^30 + 2^30)
    r.limit = (int)(start + count);
    r.hi = min((int)start + t_last + 1, r.limit);
    r.lo = window > 0 ? min(max(r.first_pos - window + 1, 0), r.hi) : 0;
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

// Whether a query at `pos` sees a key at all.
__device__ __forceinline__ bool kv4_sees(const Kv4Range& r, int pos, int window) { return min(pos, r.limit - 1) >= (window > 0 ? max(pos - window + 1, 0) : 0); }

// Four dimensions of a query row at position `pos`: val / sum as bf16; zero for a row that sees no key, NaN for one that sees keys but has a sum of 0 (every
// score is -inf: infinite keys or queries), and for a sequence outside of the cache.
__device__ __forceinline__ void kv4_store(const Kv4AttnParams& p, const Kv4Range& r, int pos, int b, int hk, int per_kv, int row, int d, float4 val, float sum) {
    const int dim = 2 * (int)p.row_bytes;
    const float nan = __int_as_float(0x7fffffff), inv = sum == 0.f ? (kv4_sees(r, pos, p.window) ? nan : 0.f) : 1.f / sum;
    const uint2 w = r.ok ? make_uint2(bf16_pack(val.x * inv, val.y * inv), bf16_pack(val.z * inv, val.w * inv)) : make_uint2(bf16_pack(nan, nan), bf16_pack(nan, nan));
    *reinterpret_cast<uint2*>(p.out + (((size_t)b * p.tokens + row / per_kv) * p.heads + hk * per_kv + row % per_kv) * dim + d) = w;
}

// What a row's raw scores are multiplied by, kept from 0 and infinity (the product of a tiny or huge scale and query): -inf, of a key that is not
// seen, and 0 must stay what they are.  Raw scores are below 2^45 (queries 2^15, codes less 8, scales 2^16, 128 of them), so what the lower
// border changes is far below a rounding of 1; at the upper one a score that is not 0 is beyond what a difference of 1 can be told from.
__device__ __forceinline__ float kv4_row_factor(float f) { return fminf(fmaxf(f, 0x1p-100f), 0x1p127f); }

template <int D>
struct Kv4Stage {                          // 32 tokens of a head
    static constexpr int G = D / kKv4Group;
    static constexpr int codes = 32 * D / 2, scales = 32 * G * 2;
    static constexpr int ks = codes, vc = codes + scales, vs = vc + ks, bytes = 2 * vc;
    static constexpr int ring = kKv4Stages * bytes;
    static constexpr int frags(int tiles) { return tiles * G * 512; }   // query fragments: 16 bytes a lane
};

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
// Blocks of 32 keys that some row of the tile sees.
__device__ __forceinline__ int kv4_blocks(const Kv4Range& r) { return (r.hi - (r.lo & ~31) + 31) >> 5; }

// Sum of what(i) over i < n, for all threads of the CTA of WARPS warps.
template <int WARPS, typename F>
__device__ __forceinline__ long long kv4_cta_sum(long long* part, int n, F what) {
    long long x = 0;
    for (int i = threadIdx.x; i < n; i += WARPS * 32) x += what(i);
#pragma unroll
    for (int j = 16; j; j >>= 1) x += __shfl_xor_sync(0xffffffffu, x, j);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) x += part[w];
    return x;
}

// How the keys of an item (a tile of query rows over a key / value head) are spread:
//   KV4_CLUSTER  a cluster of CTAs takes an item, every CTA an equal part, and merges through distributed shared memory
//   KV4_STREAM   one CTA for each place on the SMs; the blocks of all items, one behind the other, are cut into equal parts, whatever the
//                lengths of the sequences.  A CTA finishes the items that it has as a whole, and leaves its part of the first and of the last
//                one in the workspace, for kv4_attn_join_kernel.
enum Kv4Mode : int { KV4_CLUSTER = 0, KV4_STREAM = 1 };

// NT tiles of 8 query rows.  The warps of a CTA take every fourth block of its part, and merge through shared memory.
template <int D, int NT, int MODE>
__global__ void __launch_bounds__(kKv4Warps * 32, NT == 1 ? 4 : 2) kv4_attn_kernel(const Kv4AttnParams p) {
    using St = Kv4Stage<D>;
    constexpr int G = St::G, ROWS = 8 * NT, VECS = ROWS * D / 4;
    // rings of the warps, where their partial results come at the end; behind them the query's fragments, then the results' statistics
    extern __shared__ __align__(128) uint8_t smem[];
    float2(*ml)[ROWS] = reinterpret_cast<float2(*)[ROWS]>(smem + kKv4Warps * St::ring);
    float2* cta_ml = reinterpret_cast<float2*>(smem + kKv4Warps * St::ring + kKv4Warps * ROWS * 8);
    const uint32_t base_s = smem_u32(smem), frag_s = base_s + kKv4Warps * St::ring;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
    const int per_kv = p.heads / p.c.kv_heads, rows_all = p.tokens * per_kv;
    griddep_launch_dependents();
    auto range = [&](int b, int t_first, int t_last) {
        return kv4_range(p.start, p.counts, p.start_stride, b, p.tokens, p.window, p.c.max_len, t_first, t_last);
    };
    int b, hk, tile = 0, begin, end;                               // blocks begin .. end - 1 of the item
    long long left = 0;                                            // KV4_STREAM: blocks of this CTA from there on
    const int rank = MODE == KV4_CLUSTER ? blockIdx.x % p.cluster : 0;
    if constexpr (MODE == KV4_CLUSTER) {
        const int item = blockIdx.x / p.cluster;
        b = blockIdx.y, hk = item / p.row_tiles, tile = item % p.row_tiles;
        const int r0 = tile * ROWS;
        const int n = kv4_blocks(range(b, r0 / per_kv, (min(r0 + ROWS, rows_all) - 1) / per_kv));
        begin = (int)((long long)n * rank / p.cluster), end = (int)((long long)n * (rank + 1) / p.cluster);
    } else {
        auto blocks_of = [&](int i) { return kv4_blocks(range(i, 0, p.tokens - 1)); };
        const long long all = kv4_cta_sum<kKv4Warps>(reinterpret_cast<long long*>(cta_ml), p.batch, blocks_of) * p.c.kv_heads;
        long long at = all * blockIdx.x / gridDim.x;
        left = all * (blockIdx.x + 1) / gridDim.x - at;
        if (left == 0) return;
        // the sequence, head and block where this CTA's part begins: every warp finds them, by shuffles (shared memory that carried them from one
        // warp to the others would have to outlive their reading, and all of it belongs to the rings and the query's fragments from here on)
        b = hk = begin = 0;
        long long before = 0;
        for (int b0 = 0; b0 < p.batch; b0 += 32) {
            const int n = b0 + lane < p.batch ? blocks_of(b0 + lane) : 0;
            long long upto = (long long)n * p.c.kv_heads;
#pragma unroll
            for (int j = 1; j < 32; j <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, upto, j);
                if (lane >= j) upto += y;
            }
            const unsigned has = __ballot_sync(0xffffffffu, before + upto > at);
            if (has) {
                const int src = __ffs(has) - 1, blocks = __shfl_sync(0xffffffffu, n, src);
                const long long in = at - (before + __shfl_sync(0xffffffffu, upto, src) - (long long)blocks * p.c.kv_heads);
                b = b0 + src, hk = (int)(in / blocks), begin = (int)(in % blocks);
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        __syncthreads();                                           // (the query's fragments come where kv4_cta_sum's parts are)
    }
#pragma unroll 1
    for (bool first_part = true;; first_part = false) {
    const int r0 = tile * ROWS, r_last = min(r0 + ROWS, rows_all) - 1, t_first = r0 / per_kv, t_last = r_last / per_kv;
    const Kv4Range rg = range(b, t_first, t_last);
    if constexpr (MODE == KV4_STREAM) {
        const int n = kv4_blocks(rg);
        if (begin >= n) {                                          // on to the next head or sequence
            begin = 0;
            if (++hk == p.c.kv_heads) hk = 0, ++b;
            continue;
        }
        end = (int)min((long long)n, begin + left);
    }
    const uint32_t ring = base_s + warp * St::ring;
    const size_t row0 = ((size_t)b * p.c.kv_heads + hk) * p.c.max_len;
    const int lo32 = rg.lo & ~31, first = begin + warp;
    // 16 bytes a lane at a time: a block's codes of keys and of values, then (D = 128: lanes 0 .. 15 and 16 .. 31, D = 64: half as many) their scales
    constexpr int CHUNKS = St::codes / 512, SCALE_LANES = St::scales / 16;
    const size_t block0 = row0 + lo32 + (size_t)first * 32;
    const uint8_t *f_k = p.c.k_codes + block0 * (D / 2) + lane * 16, *f_v = p.c.v_codes + block0 * (D / 2) + lane * 16;
    const uint8_t* f_s = reinterpret_cast<const uint8_t*>(lane < SCALE_LANES ? p.c.k_scales : p.c.v_scales) + block0 * (G * 2) + lane % SCALE_LANES * 16;
    const uint32_t f_sd = ring + (lane < SCALE_LANES ? St::ks : St::vs) + lane % SCALE_LANES * 16;
    int issued = first;                                            // next block to fetch
    auto fetch = [&](int place) {
        if (issued < end) {
            const uint32_t dst = ring + place * St::bytes + lane * 16;
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i) cp_async_16(dst + i * 512, f_k + i * 512), cp_async_16(dst + St::vc + i * 512, f_v + i * 512);
            if (lane < 2 * SCALE_LANES) cp_async_16(f_sd + place * St::bytes, f_s);
            f_k += kKv4Warps * St::codes, f_v += kKv4Warps * St::codes, f_s += kKv4Warps * St::scales;
        }
        cp_async_commit();
        issued += kKv4Warps;
    };
#pragma unroll
    for (int i = 0; i < kKv4Stages; ++i) fetch(i);

    // ---- the query as B fragments, made once for the CTA: lane (g, q) of warp i has elements 8 q .. + 7 of group i of row 8 nt + g
    uint32_t off[NT];                                              // B operand of the offsets' product: -8 times the sums over the groups
    float row_f[NT][2];                                            // of rows 2 q, 2 q + 1: what a raw score is multiplied by
    int row_pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = r0 + 8 * nt + g;
        const bool has = r < rows_all;
        const int t = has ? r / per_kv : 0, h = has ? hk * per_kv + r % per_kv : 0;
        const __nv_bfloat16* src = p.q.x + b * p.q.sb + t * p.q.st + h * p.q.sh;
        uint4 mine = make_uint4(0, 0, 0, 0);
        float amax = 0.f, sums[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const uint4 raw = has ? ldg_128(src + 32 * i + 8 * q) : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo(w[j])), fabsf(bf16_hi(w[j]))));
            sums[i] = ((bf16_lo(w[0]) + bf16_hi(w[0])) + (bf16_lo(w[1]) + bf16_hi(w[1]))) + ((bf16_lo(w[2]) + bf16_hi(w[2])) + (bf16_lo(w[3]) + bf16_hi(w[3])));
            sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], 1);
            sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], 2);
            if (i == warp) mine = raw;
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^(14 - exponent of the largest): that one becomes 2^14 .. 2^15
        const int ex = min(max((int)(__float_as_uint(amax) >> 23), 30), 240) - 127;
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        const float f = kv4_row_factor(p.scale_log2 * __uint_as_float((uint32_t)(127 + 10 + ex) << 23));   // 2^24 / up
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            row_f[nt][n] = __shfl_sync(0xffffffffu, f, (2 * q + n) * 4);
            row_pos[nt][n] = rg.first_pos - t_first + (r0 + 8 * nt + 2 * q + n) / per_kv;
        }
        if (warp < G) {
            const uint32_t w[4] = {mine.x, mine.y, mine.z, mine.w};
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[2 * j] = bf16_lo(w[j]) * up, x[2 * j + 1] = bf16_hi(w[j]) * up;
            // A's halves are codes j of the low halfword and 4 + j of the high one
            sts128(frag_s + (uint32_t)((nt * G + warp) * 512 + lane * 16),
                   make_uint4(f16_pack(x[0], x[4]), f16_pack(x[1] * 0.0625f, x[5] * 0.0625f), f16_pack(x[2], x[6]), f16_pack(x[3] * 0.0625f, x[7] * 0.0625f)));
        }
        // groups 2 (q & 1), 2 (q & 1) + 1: rounded to fp16 in the lanes q = 0, 1, what the rounding left in the lanes 2, 3
        const float c8 = up * (-8.f / kTwo24), e0 = (G == 4 && (q & 1) ? sums[G - 2] : sums[0]) * c8, e1 = (G == 4 && (q & 1) ? sums[G - 1] : sums[1]) * c8;
        const uint32_t hi = f16_pack(e0, e1);
        off[nt] = q < 2 ? hi : f16_pack(e0 - f16_lo(hi), e1 - f16_hi(hi));
        if (G == 2 && (q & 1)) off[nt] = 0u;
    }
    __syncthreads();

    // top: the raw score above which a row's reference follows, -inf before its first key; nb: minus the reference of its exponents
    float o[NT][G][2][4], on[NT][G / 2][4], top[NT][2], nb[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = top[nt][1] = -INFINITY, nb[nt][0] = nb[nt][1] = l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][i][0][e] = o[nt][i][1][e] = on[nt][i / 2][e] = 0.f;
    }
    auto rescale = [&](int nt, float f0, float f1) {
        l[nt][0] *= f0, l[nt][1] *= f1;
#pragma unroll
        for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) o[nt][i][jj][0] *= f0, o[nt][i][jj][1] *= f1, o[nt][i][jj][2] *= f0, o[nt][i][jj][3] *= f1;
            on[nt][i / 2][i % 2 * 2] *= f0, on[nt][i / 2][i % 2 * 2 + 1] *= f1;
        }
    };
    int vexp = kKv4MinExp;                                         // exponent of the largest value scale so far, within kKv4MinExp .. kKv4MaxExp
    uint32_t vlimit = (uint32_t)(kKv4MinExp + 16) << 10;           // fp16 bits of 2^(vexp + 1)

    // The 32 keys of a place, the first of them key0, as two groups of 16.  PART: some row does not see some of them.
    auto keys32 = [&](uint32_t at, int key0, auto part) {
        constexpr bool PART = decltype(part)::value;
        float s[2][NT][4];
        {
            uint32_t k0[2][G], k1[2][G], s0w[2][G / 2], s1w[2][G / 2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                lds_words(at + (u * 16 + g) * (D / 2) + q * (G * 4), k0[u]);
                lds_words(at + (u * 16 + g + 8) * (D / 2) + q * (G * 4), k1[u]);
                lds_words(at + St::ks + (u * 16 + g) * (G * 2), s0w[u]);
                lds_words(at + St::ks + (u * 16 + g + 8) * (G * 2), s1w[u]);
                // the offsets: scales of groups 2 (q & 1), + 1 of the two keys
                const uint32_t sa = at + St::ks + (u * 16 + g) * (G * 2) + (G == 4 ? (q & 1) * 4 : 0), a0 = lds32(sa), a1 = lds32(sa + 16 * G);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_f16_k8(s[u][nt], a0, a1, off[nt]);
            }
#pragma unroll
            for (int i = 0; i < G; ++i) {
                uint32_t f[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) lds_words(frag_s + (nt * G + i) * 512 + lane * 16, f[nt]);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t a0[4] = {k0[u][i] & 0x000f000fu, k1[u][i] & 0x000f000fu, k0[u][i] & 0x00f000f0u, k1[u][i] & 0x00f000f0u};
                    const uint32_t x = k0[u][i] >> 8, y = k1[u][i] >> 8;
                    const uint32_t a1[4] = {x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u};
                    const float f0 = i & 1 ? f16_hi(s0w[u][i / 2]) : f16_lo(s0w[u][i / 2]), f1 = i & 1 ? f16_hi(s1w[u][i / 2]) : f16_lo(s1w[u][i / 2]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float d[4];
                        mma_f16_first(d, a0, f[nt][0], f[nt][1]);
                        mma_f16(d, a1, f[nt][2], f[nt][3]);
                        s[u][nt][0] = fmaf(d[0], f0, s[u][nt][0]), s[u][nt][1] = fmaf(d[1], f0, s[u][nt][1]);
                        s[u][nt][2] = fmaf(d[2], f1, s[u][nt][2]), s[u][nt][3] = fmaf(d[3], f1, s[u][nt][3]);
                    }
                }
            }
        }
        if constexpr (PART) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + 16 * u + g + 8 * (e >> 1), pos = row_pos[nt][e & 1];
                        if (key > pos || key >= rg.limit || (p.window > 0 && key <= pos - p.window)) s[u][nt][e] = -INFINITY;
                    }
        }
        // ---- the reference follows the maximum only where that has left it by more than 2^kKv4Slack: the lanes of a row compare by themselves,
        // and confer where one has more
        bool grown = false;
        float mx[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                mx[nt][n] = fmaxf(fmaxf(s[0][nt][n], s[0][nt][2 + n]), fmaxf(s[1][nt][n], s[1][nt][2 + n]));
                grown |= mx[nt][n] > top[nt][n];
            }
        if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float f[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float x = mx[nt][n];
#pragma unroll
                    for (int j = 4; j < 32; j <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, j));
                    f[n] = 1.f;
                    if (x > top[nt][n]) {
                        const float to = -fmaf(x, row_f[nt][n], (float)vexp);
                        f[n] = top[nt][n] == -INFINITY ? 0.f : ex2_approx(to - nb[nt][n]);
                        nb[nt][n] = to;
                        top[nt][n] = x + kKv4Slack / row_f[nt][n];
                    }
                }
                rescale(nt, f[0], f[1]);
            }
        }
        // ---- probabilities, transposed to the B operand of the second product
        uint32_t pt[2][NT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[u][nt][e] = ex2_approx(fmaf(s[u][nt][e], row_f[nt][e & 1], nb[nt][e & 1]));
                l[nt][0] += s[u][nt][0] + s[u][nt][2], l[nt][1] += s[u][nt][1] + s[u][nt][3];
                pt[u][nt][0] = transposed_8x8(f16_pack(s[u][nt][0], s[u][nt][1]));
                pt[u][nt][1] = transposed_8x8(f16_pack(s[u][nt][2], s[u][nt][3]));
            }
        // ---- values
#pragma unroll
        for (int u = 0; u < 2; ++u) {
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
                // sums times 8: of an even group in the rows g, of an odd one in the rows g + 8
                const uint32_t eight[4] = {i & 1 ? 0u : 0x00080008u, i & 1 ? 0x00080008u : 0u, i & 1 ? 0u : 0x00080008u, i & 1 ? 0x00080008u : 0u};
                const uint32_t f0 = __byte_perm(w0[i / 2], w0[G / 2 + i / 2], sel), f1 = __byte_perm(w1[i / 2], w1[G / 2 + i / 2], sel);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t b0 = f16x2_mul(pt[u][nt][0], f0), b1 = f16x2_mul(pt[u][nt][1], f1);
                    if constexpr (PART) {                          // a value that is not seen may be NaN
                        b0 &= __vcmpne2(pt[u][nt][0], 0u), b1 &= __vcmpne2(pt[u][nt][1], 0u);
                    }
                    mma_f16(o[nt][i][0], a0, b0, b1);
                    mma_f16(o[nt][i][1], a1, b0, b1);
                    mma_f16(on[nt][i / 2], eight, b0, b1);
                }
            }
        }
    };

    int place = 0;
#pragma unroll 1
    for (int block = first; block < end; block += kKv4Warps) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kKv4Stages - 1) : "memory");
        __syncwarp();
        const uint32_t at = ring + place * St::bytes;
        const int key0 = lo32 + block * 32;
        // ---- a value scale beyond the limit: lane = token
        uint32_t vw[G / 2], big = 0;
        lds_words(at + St::vs + lane * (G * 2), vw);
        const bool part = key0 + 32 > rg.limit || key0 + 31 > rg.first_pos || (p.window > 0 && key0 <= rg.first_pos + (t_last - t_first) - p.window);
        if (!part || (key0 + lane >= rg.lo && key0 + lane < rg.hi)) {
            uint32_t x = vw[0] & 0x7fff7fffu;
            if (G == 4) x = __vmaxu2(x, vw[G / 2 - 1] & 0x7fff7fffu);
            big = max(x & 0xffffu, x >> 16);
        }
        if (__any_sync(0xffffffffu, big >= vlimit)) {
            if (big >= 0x7c00u) {                                  // an infinite or NaN scale is the matter of the rows that see it alone
                big = 0;
#pragma unroll
                for (int i = 0; i < G / 2; ++i) {
                    const uint32_t a = vw[i] & 0x7fffu, c = vw[i] >> 16 & 0x7fffu;
                    big = max(big, max(a < 0x7c00u ? a : 0u, c < 0x7c00u ? c : 0u));
                }
            }
            const int to = max(min((int)(__reduce_max_sync(0xffffffffu, big) >> 10) - 15, kKv4MaxExp), vexp);
            const float f = __uint_as_float((uint32_t)(127 + vexp - to) << 23);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                rescale(nt, f, f);
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    if (top[nt][n] != -INFINITY) nb[nt][n] -= (float)(to - vexp);
            }
            vexp = to;
            vlimit = to == kKv4MaxExp ? 0x8000u : (uint32_t)(to + 16) << 10;
        }
        if (!part) keys32(at, key0, Kv4Const<false>());
        else keys32(at, key0, Kv4Const<true>());
        __syncwarp();                                              // the place may be filled again
        fetch(place);
        if (++place == kKv4Stages) place = 0;
    }
    cp_async_wait_all();

    // ---- merge of the warps
    float(*os)[ROWS][D] = reinterpret_cast<float(*)[ROWS][D]>(smem);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float sum = l[nt][n];
#pragma unroll
            for (int j = 4; j < 32; j <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, j);
            const int r = 8 * nt + 2 * q + n;
            if (g == 0) ml[warp][r] = make_float2(top[nt][n] == -INFINITY ? -INFINITY : -nb[nt][n], sum);
#pragma unroll
            for (int i = 0; i < G; ++i)
                *reinterpret_cast<float4*>(&os[warp][r][32 * i + 4 * g]) =
                    make_float4((o[nt][i][0][n] - on[nt][i / 2][i % 2 * 2 + n]) * kTwo24, (o[nt][i][0][2 + n] * 0.0625f - on[nt][i / 2][i % 2 * 2 + n]) * kTwo24,
                                (o[nt][i][1][n] - on[nt][i / 2][i % 2 * 2 + n]) * kTwo24, (o[nt][i][1][2 + n] * 0.0625f - on[nt][i / 2][i % 2 * 2 + n]) * kTwo24);
        }
    __syncthreads();
    if (!rg.ok && tid == 0) *p.status = 1;
    const bool whole = MODE == KV4_CLUSTER || end - begin == kv4_blocks(rg);
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
        if (MODE == KV4_CLUSTER && p.cluster > 1) {                // (each thread reads and writes its own place of warp 0's part)
            *reinterpret_cast<float4*>(&os[0][r][d]) = val;
            if (d == 0) cta_ml[r] = make_float2(top, sum);
        } else if (r0 + r < rows_all) {
            if (whole) {
                kv4_store(p, rg, rg.first_pos - t_first + (r0 + r) / per_kv, b, hk, per_kv, r0 + r, d, val, sum);
            } else {
                const size_t at = (size_t)(2 * blockIdx.x + (first_part ? 0 : 1)) * ROWS + r;
                *reinterpret_cast<float4*>(p.part_o + at * D + d) = val;
                if (d == 0) p.part_ml[at] = make_float2(top, sum);
            }
        }
    }
    if constexpr (MODE == KV4_CLUSTER) {
        if (p.cluster == 1) return;
        cluster_arrive();
        cluster_wait();
        const uint32_t ml_s = smem_u32(cta_ml);
#pragma unroll 1
        for (int x = rank * kKv4Warps * 32 + tid; x < VECS; x += p.cluster * kKv4Warps * 32) {
            const int r = x / (D / 4), d = x % (D / 4) * 4;
            if (r0 + r >= rows_all) break;
            float2 st[8];
            float4 y[8];
            float top = -INFINITY, sum = 0.f;
            float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.cluster) {
                    st[c] = ld_cluster_f2(map_to_rank(ml_s + r * 8, c));
                    y[c] = ld_cluster_f4(map_to_rank(base_s + (r * D + d) * 4, c));
                    top = fmaxf(top, st[c].x);
                }
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (c < p.cluster) {
                    const float f = st[c].x == -INFINITY ? 0.f : ex2_approx(st[c].x - top);
                    sum += f * st[c].y;
                    if (f != 0.f) val.x += f * y[c].x, val.y += f * y[c].y, val.z += f * y[c].z, val.w += f * y[c].w;
                }
            kv4_store(p, rg, rg.first_pos - t_first + (r0 + r) / per_kv, b, hk, per_kv, r0 + r, d, val, sum);
        }
        cluster_arrive();                                          // nobody leaves while its results are read
        cluster_wait();
        return;
    } else {
        left -= end - begin;
        if (left == 0) return;
        begin = end;
        __syncthreads();                                           // the rings may be filled again
    }
    }
}

// KV4_STREAM: joins what several CTAs have found for an item, and writes the items that no CTA had a key for.  A CTA takes `rows_here`
// rows of an item, its warps spread over the rows and, within a row, over the parts.
template <int D, int NT>
__global__ void __launch_bounds__(kKv4JoinWarps * 32) kv4_attn_join_kernel(const Kv4AttnParams p, int ctas, int rows_here) {
    constexpr int ROWS = 8 * NT, DEEP = 4;                         // parts of a warp on their way at once
    __shared__ float4 os[kKv4JoinWarps][D / 4];
    __shared__ float2 ml[kKv4JoinWarps];
    __shared__ long long part[kKv4JoinWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y, hk = blockIdx.x % p.c.kv_heads, per_kv = p.heads / p.c.kv_heads, rows = p.tokens * per_kv;
    long long upto = 0;
    auto blocks_of = [&](int i) {
        return kv4_blocks(kv4_range(p.start, p.counts, p.start_stride, i, p.tokens, p.window, p.c.max_len, 0, p.tokens - 1));
    };
    const long long all = kv4_cta_sum<kKv4JoinWarps>(part, p.batch, [&](int i) {
        const int m = blocks_of(i);
        if (i < b) upto += m;
        return m;
    }) * p.c.kv_heads;
    const int n = blocks_of(b);
    const long long from = kv4_cta_sum<kKv4JoinWarps>(part, kKv4JoinWarps * 32, [&](int) { return upto; }) * p.c.kv_heads + (long long)hk * n;
    // CTA c has the blocks all * c / ctas .. all * (c + 1) / ctas - 1; the last one that begins at or before block x has it
    auto holder = [&](long long x) { return (int)(((x + 1) * ctas - 1) / all); };
    const int c0 = n ? holder(from) : 0, c1 = n ? holder(from + n - 1) : -1;
    griddep_wait();                                                // (also where nothing is left to do: what follows waits for this kernel alone)
    if (n && c0 == c1) return;                                     // finished by that CTA
    const int per_row = kKv4JoinWarps / rows_here, sub = warp % per_row;
    const int r = warp < per_row * rows_here ? blockIdx.x / p.c.kv_heads * rows_here + warp / per_row : rows;
    float top = -INFINITY, sum = 0.f;
    float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = r < rows ? c0 + sub : c1 + 1; c <= c1; c += per_row * DEEP) {
        float2 st[DEEP];
        float4 y[DEEP];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            const int cc = c + j * per_row;
            const long long s = all * cc / ctas;
            st[j] = make_float2(-INFINITY, 0.f);
            if (cc <= c1 && all * (cc + 1) / ctas > s) {           // (with fewer blocks than CTAs some have none)
                const size_t at = (size_t)(2 * cc + (s >= from ? 0 : 1)) * ROWS + r;
                st[j] = p.part_ml[at];
                if (lane < D / 4) y[j] = *reinterpret_cast<const float4*>(p.part_o + at * D + lane * 4);
            }
        }
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            if (st[j].x == -INFINITY) {
                sum += st[j].y;                                    // (zero, or NaN)
                continue;
            }
            const float to = fmaxf(top, st[j].x), f = top == -INFINITY ? 0.f : ex2_approx(top - to), h = ex2_approx(st[j].x - to);
            top = to, sum = sum * f + st[j].y * h;
            val.x = val.x * f + y[j].x * h, val.y = val.y * f + y[j].y * h, val.z = val.z * f + y[j].z * h, val.w = val.w * f + y[j].w * h;
        }
    }
    if (lane < D / 4) os[warp][lane] = val;
    if (lane == 0) ml[warp] = make_float2(top, sum);
    __syncthreads();
    if (r >= rows || sub || lane >= D / 4) return;
    top = -INFINITY, sum = 0.f, val = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = warp; w < warp + per_row; ++w) top = fmaxf(top, ml[w].x);
    for (int w = warp; w < warp + per_row; ++w) {
        const float f = ml[w].x == -INFINITY ? 0.f : ex2_approx(ml[w].x - top);
        sum += ml[w].x == -INFINITY ? ml[w].y : f * ml[w].y;
        if (f != 0.f) val.x += f * os[w][lane].x, val.y += f * os[w][lane].y, val.z += f * os[w][lane].z, val.w += f * os[w][lane].w;
    }
    const Kv4Range rg = kv4_range(p.start, p.counts, p.start_stride, b, p.tokens, p.window, p.c.max_len, 0, p.tokens - 1);
    if (!rg.ok && lane == 0) *p.status = 1;
    kv4_store(p, rg, rg.first_pos + r / per_kv, b, hk, per_kv, r, lane * 4, val, sum);
}

}  // namespace tsp
