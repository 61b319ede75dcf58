// Attention of many new tokens over a 4-bit cache (kv4.cuh), for sm_100a: flash attention on tcgen05.
//
// A CTA takes 128 query rows - tokens times the query heads of a key / value head - and goes over the keys in tiles of 64; two CTAs share
// an SM, so that one's products run beside the other's exponentials.  Its warps:
//   0-3  a row per thread: the query into shared memory as fp16 (scaled by a power of two per row, exact), then for every tile the scores
//        from tensor memory, the running maximum, exponentials, probabilities as fp16 back into tensor memory where the scores were
//   4-7  expand codes to fp16 in the operands' swizzled layouts: two warps keys (a key per thread), two warps values (16 dimensions of 8 keys
//        per thread: the operand wants the keys of a dimension behind each other)
//   8    one thread issues the products: S = Q K^T of the next tile, then O += P V of this one, P from tensor memory
// A code c becomes 1024 + c (or 1024 + 16 c) by one AND-OR, c - 8 exactly by one addition (or FMA), and is rounded once, in the
// product with its scale.  The order of dimensions within 8 of keys and queries is the one in which codes come out of their words.
// O stays in tensor memory; it is rescaled only where a row's maximum has left its reference by 2^8.
// A product takes P = 0 times a value for keys that a row does not see.  So values that are not finite as fp16 (a NaN or infinite scale, or more than
// 65504) are left out, and the rows that see one of them get NaN in that group of dimensions at the end.
// Where there are few tiles of rows the keys are cut into parts (`cluster` CTAs to a tile, kv4_prefill_join_kernel).
//
// 2,048 tokens of 20 heads over 5 after 2,048: 140 to 144 us for 64 GFLOP, 450 TFLOP/s; the floor of the products is 38 us.  A tile of 64 keys takes two CTAs of an
// SM 3,500 cycles: a softmax warp works through them all (600 to load the scores, 300 for the maximum, 1,750 for exponentials, sums and packing, beside the
// other CTA's), and so does the thread that issues (1,600 in the queue of MMAs and commits, four of them then, two now; 1,000 waiting for probabilities).  Without the expansion
// of keys and values - wrong results - it took 115 us, without exponentials as well 113: no single part is the bound.
#pragma once
#include "kv4_attn.cuh"

namespace tsp {

constexpr int kKvpRows = 128, kKvpKeys = 64, kKvpThreads = 288;

template <int D>
struct KvpSmem {
    static constexpr int q = 0, q_block = kKvpRows * 128, q_bytes = D / 64 * q_block;
    static constexpr int k = q + q_bytes, k_block = kKvpKeys * 128, k_bytes = D / 64 * k_block;   // two stages
    static constexpr int v = k + 2 * k_bytes, v_bytes = D * 128;                                   // two stages: a row per dimension
    static constexpr int bars = v + 2 * v_bytes;                   // q; keys, values, scores, probabilities and O of a tile there (2 each)
    static constexpr int slot = bars + 16 * 8, abort_flag = slot + 4, bad = slot + 16;             // bad: first key of each group that is not finite
    static constexpr int total = 1024 + bad + 32;
    static constexpr uint32_t columns = 256;                       // O: D, S: two buffers of 64
};

// D[tmem] (+)= A * B, fp16 operands, fp32 accumulators
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
          "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]),
          "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
// (names the registers: nothing that reads them may move ahead of the wait)
__device__ __forceinline__ void tmem_ld32_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]),
                   "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]),
                   "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]),
                   "+f"(v[31])::"memory");
}
__device__ __forceinline__ uint32_t f16x2_add(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// The codes in bits 0 .. 3 (16 .. 19) and 4 .. 7 (20 .. 23) of x, less 8, times the scales
__device__ __forceinline__ uint32_t kvp_low(uint32_t x, uint32_t scales) { return f16x2_mul(f16x2_add((x & 0x000f000fu) | 0x64006400u, 0xe408e408u), scales); }   // - 1032
__device__ __forceinline__ uint32_t kvp_high(uint32_t x, uint32_t scales) {
    return f16x2_mul(f16x2_fma((x & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, 0xd480d480u), scales);   // / 16 - 72
}

template <int WORDS>
__device__ __forceinline__ void ldg_words(const void* src, uint32_t (&w)[WORDS]) {
    if constexpr (WORDS == 2) {
        const uint2 v = *static_cast<const uint2*>(src);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *static_cast<const uint32_t*>(src);
    }
}
// One arrival for a warp, after all of its lanes' writes (64 and 128 arrivals of single threads on one barrier took as long as a product).
__device__ __forceinline__ void kvp_arrive(uint32_t bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}
__device__ __forceinline__ bool kvp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
        if (mbar_test(bar, parity)) return true;
    return wait_longer(bar, parity, abort_flag);
}
__device__ __forceinline__ bool kvp_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) { return __all_sync(0xffffffffu, kvp_wait(bar, parity, abort_flag)); }

template <int D>
__global__ void __launch_bounds__(kKvpThreads, 2) kv4_prefill_kernel(const Kv4AttnParams p) {
    using Sm = KvpSmem<D>;
    constexpr int G = D / kKv4Group;
    extern __shared__ __align__(16) uint8_t raw_smem[];
    uint8_t* smem = raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023);
    const uint32_t sb = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t b_q = sb + Sm::bars, b_kf = b_q + 8, b_vf = b_kf + 16, b_s = b_vf + 16, b_p = b_s + 16, b_o = b_p + 16;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Sm::abort_flag);
    int* bad = reinterpret_cast<int*>(smem + Sm::bad);
    // the longest rows first
    const int part = blockIdx.x % p.cluster, item = blockIdx.x / p.cluster, tile = p.row_tiles - 1 - item / p.c.kv_heads, hk = item % p.c.kv_heads, b = blockIdx.y;
    const int per_kv = p.heads / p.c.kv_heads, rows_all = p.tokens * per_kv, r0 = tile * kKvpRows, r_last = min(r0 + kKvpRows, rows_all) - 1;
    const int t_first = r0 / per_kv;
    const Kv4Range rg = kv4_range(p.start, p.counts, p.start_stride, b, p.tokens, p.window, p.c.max_len, t_first, r_last / per_kv);
    // key tiles of this CTA: its part of those that some row sees; `base`, the first
    const int j_lo = rg.lo / kKvpKeys, j_all = (rg.hi + kKvpKeys - 1) / kKvpKeys - j_lo;
    const int j0 = (int)((long long)j_all * part / p.cluster), tiles = (int)((long long)j_all * (part + 1) / p.cluster) - j0, base = (j_lo + j0) * kKvpKeys;
    if (tid == 0) {
        mbar_init(b_q, 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_kf + 8 * i, 2), mbar_init(b_vf + 8 * i, 2);
            mbar_init(b_s + 8 * i, 1), mbar_init(b_p + 8 * i, 4), mbar_init(b_o + 8 * i, 1);
        }
        mbar_fence_init();
        *abort_flag = 0;
        for (int i = 0; i < G; ++i) bad[i] = 0x7fffffff;
        if (!rg.ok) *p.status = 1;
    }
    if (warp == 8) tmem_alloc(sb + Sm::slot, Sm::columns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + Sm::slot), t_o = tmem, t_s = tmem + 128;
    const size_t row0 = ((size_t)b * p.c.kv_heads + hk) * p.c.max_len + base;
    // warps 0 .. 3: this thread's row, its sum and whether all went well
    const int row = r0 + min(tid, kKvpRows - 1), t = min(row, rows_all - 1) / per_kv, h = hk * per_kv + min(row, rows_all - 1) % per_kv;
    const int pos = rg.first_pos - t_first + t, seen_from = p.window ? max(pos - p.window + 1, 0) : 0, seen_to = min(pos, rg.limit - 1);
    const uint32_t mine = (uint32_t)(warp * 32) << 16;
    float l = 0.f, nb = 0.f;                                       // sum, minus the reference of the exponents
    bool ok = true;

    if (warp < 4) {
        float row_f;
        {
            const __nv_bfloat16* src = p.q.x + (long long)b * p.q.sb + (long long)t * p.q.st + (long long)h * p.q.sh;
            float amax = 0.f;
#pragma unroll 4
            for (int i = 0; i < D / 8; ++i) {
                const uint4 w = ldg_128(src + 8 * i);
                amax = fmaxf(amax, fmaxf(fmaxf(fmaxf(fabsf(bf16_lo(w.x)), fabsf(bf16_hi(w.x))), fmaxf(fabsf(bf16_lo(w.y)), fabsf(bf16_hi(w.y)))),
                                         fmaxf(fmaxf(fabsf(bf16_lo(w.z)), fabsf(bf16_hi(w.z))), fmaxf(fabsf(bf16_lo(w.w)), fabsf(bf16_hi(w.w))))));
            }
            const int ex = min(max((int)(__float_as_uint(amax) >> 23), 30), 240) - 127;      // the largest becomes 2^14 .. 2^15
            const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
            row_f = kv4_row_factor(p.scale_log2 * __uint_as_float((uint32_t)(127 - 14 + ex) << 23));
#pragma unroll 4
            for (int i = 0; i < D / 8; ++i) {
                const uint4 w = ldg_128(src + 8 * i);
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[2 * j] = bf16_lo(x[j]) * up, f[2 * j + 1] = bf16_hi(x[j]) * up;
                sts128(sb + Sm::q + (uint32_t)((i >> 3) * Sm::q_block + tid * 128 + (((i & 7) ^ (tid & 7)) << 4)),
                       make_uint4(f16_pack(f[0], f[4]), f16_pack(f[1], f[5]), f16_pack(f[2], f[6]), f16_pack(f[3], f[7])));
            }
        }
        fence_proxy_async_smem();
        kvp_arrive(b_q, lane);
        float top = -INFINITY;                                     // as in kv4_attn_kernel
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
            const int buf = j & 1;
            ok = kvp_wait_warp(b_s + 8 * buf, (j >> 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t ts = t_s + mine + buf * 64;
            float s[2][32];
            tmem_ld32(ts, s[0]);
            tmem_ld32(ts + 32, s[1]);
            tmem_ld32_wait(s[0]);
            tmem_ld32_wait(s[1]);
            const int key0 = base + j * kKvpKeys;
            if (key0 + kKvpKeys - 1 > rg.first_pos || key0 + kKvpKeys > rg.limit) {
                const int sees = seen_to - key0;                   // the last key of the tile that the row sees
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i > sees) s[i >> 5][i & 31] = -INFINITY;
            }
            if (__any_sync(0xffffffffu, seen_from > key0)) {
                const int from = seen_from - key0;                 // the first one
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i < from) s[i >> 5][i & 31] = -INFINITY;
            }
            float m4[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};   // (four chains: one would take as long as the exponentials)
#pragma unroll
            for (int i = 4; i < 64; ++i) m4[i & 3] = fmaxf(m4[i & 3], s[i >> 5][i & 31]);
            const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            const bool grown = mx > top;
            if (__any_sync(0xffffffffu, grown)) {
                float f = 1.f;
                if (grown) {
                    const float to = -mx * row_f;
                    f = top == -INFINITY ? 0.f : ex2_approx(to - nb);
                    nb = to, top = mx + kKv4Slack / row_f;
                }
                l *= f;
                if (j > 0) {                                       // O is complete up to tile j - 1 before it is touched
                    ok = kvp_wait_warp(b_o + 8 * (buf ^ 1), ((j - 1) >> 1) & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        tmem_ld32(t_o + mine + c, o);
                        tmem_ld32_wait(o);
                        uint32_t w[16];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(o[16 * half + i] * f);
                            tmem_st16(t_o + mine + c + 16 * half, w);
                        }
                    }
                    tmem_st_wait();
                }
            }
            float l2[2] = {0.f, 0.f};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = ex2_approx(fmaf(s[half][2 * i], row_f, nb)), y = ex2_approx(fmaf(s[half][2 * i + 1], row_f, nb));
                    l2[i & 1] += x + y;
                    w[i] = f16_pack(x, y);
                }
                tmem_st16(ts + 16 * half, w);
            }
            l += l2[0] + l2[1];
            tmem_st_wait();
            tc_fence_before();
            kvp_arrive(b_p + 8 * buf, lane);
        }
        if (ok && tiles > 0) ok = kvp_wait_warp(b_o + 8 * ((tiles - 1) & 1), ((tiles - 1) >> 1) & 1, abort_flag);
    } else if (warp < 6) {                                         // ---- keys: one per thread
        const int key = tid - 128;
        const uint8_t* kc = p.c.k_codes + (row0 + key) * (D / 2);
        const __half* ks = p.c.k_scales + (row0 + key) * G;
        uint4 w[D / 32];
        uint32_t sc[G / 2];
        auto load = [&](int j, uint4 (&w)[D / 32], uint32_t (&sc)[G / 2]) {
            const uint8_t* src = kc + (size_t)j * kKvpKeys * (D / 2);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) w[i] = ldg_128(src + 16 * i);
            ldg_words(ks + (size_t)j * kKvpKeys * G, sc);
        };
        if (tiles > 0) load(0, w, sc);
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
            const int st = j & 1;
            if (j >= 2 && !kvp_wait_warp(b_s + 8 * st, ((j >> 1) - 1) & 1, abort_flag)) break;
            const uint32_t dst = sb + Sm::k + st * Sm::k_bytes + key * 128;
            // 16 bytes t of a row hold word t of every group (64 dimensions: 8 bytes)
            uint32_t words[4 * G];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) words[4 * i] = w[i].x, words[4 * i + 1] = w[i].y, words[4 * i + 2] = w[i].z, words[4 * i + 3] = w[i].w;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const uint32_t f = __byte_perm(sc[i / 2], 0, i & 1 ? 0x3232 : 0x1010);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t x = words[t * G + i], x8 = x >> 8;
                    const int c = 4 * i + t;                       // chunk of 8 dimensions
                    sts128(dst + (c >> 3) * Sm::k_block + (((c & 7) ^ (key & 7)) << 4), make_uint4(kvp_low(x, f), kvp_high(x, f), kvp_low(x8, f), kvp_high(x8, f)));
                }
            }
            fence_proxy_async_smem();
            kvp_arrive(b_kf + 8 * st, lane);
            if (j + 1 < tiles) load(j + 1, w, sc);                 // (arrives while the place for it is waited for)
        }
    } else if (warp < 8) {                                         // ---- values: 16 dimensions of 8 keys per thread
        const int oct = tid & 7, g = (tid - 192) >> 3;             // keys 8 oct .. + 7, halfword g of every group
        const uint8_t* vc = p.c.v_codes + (row0 + 8 * oct) * (D / 2) + g * (G * 2);
        const __half* vs = p.c.v_scales + (row0 + 8 * oct) * G;
        uint32_t w[8][G / 2], sc[8][G / 2];
        auto load = [&](int j, uint32_t (&w)[8][G / 2], uint32_t (&sc)[8][G / 2]) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                ldg_words(vc + ((size_t)j * kKvpKeys + k) * (D / 2), w[k]);
                ldg_words(vs + ((size_t)j * kKvpKeys + k) * G, sc[k]);
            }
        };
        if (tiles > 0) load(0, w, sc);
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
            const int st = j & 1, key0 = base + j * kKvpKeys + 8 * oct;
            if (j >= 2 && !kvp_wait_warp(b_o + 8 * st, ((j >> 1) - 1) & 1, abort_flag)) break;
            const uint32_t dst = sb + Sm::v + st * Sm::v_bytes;
            // keys behind the last one hold anything; scales beyond 8188 (0x6fff) make values that fp16 does not hold
            uint32_t big = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int i = 0; i < G / 2; ++i) big = __vmaxu2(big, sc[k][i] & 0x7fff7fffu);
            if (base + (j + 1) * kKvpKeys > rg.hi || __vcmpgtu2(big, 0x6fff6fffu)) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int i = 0; i < G / 2; ++i) {
                        if (key0 + k >= rg.hi) sc[k][i] = 0u;
                        if ((sc[k][i] & 0x7fffu) > 0x6fffu) atomicMin(&bad[2 * i], key0 + k), sc[k][i] &= 0xffff0000u;
                        if ((sc[k][i] >> 16 & 0x7fffu) > 0x6fffu) atomicMin(&bad[2 * i + 1], key0 + k), sc[k][i] &= 0x0000ffffu;
                    }
            }
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
                uint32_t out[4][4];                                // [code][two keys each]
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t x = __byte_perm(w[2 * k][i / 2], w[2 * k + 1][i / 2], sel), f = __byte_perm(sc[2 * k][i / 2], sc[2 * k + 1][i / 2], sel), x8 = x >> 8;
                    out[0][k] = kvp_low(x, f), out[1][k] = kvp_high(x, f), out[2][k] = kvp_low(x8, f), out[3][k] = kvp_high(x8, f);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int d = 32 * i + 4 * g + n;
                    sts128(dst + d * 128 + ((oct ^ (d & 7)) << 4), make_uint4(out[n][0], out[n][1], out[n][2], out[n][3]));
                }
            }
            fence_proxy_async_smem();
            kvp_arrive(b_vf + 8 * st, lane);
            if (j + 1 < tiles) load(j + 1, w, sc);                 // (arrives while the place for it is waited for)
        }
    } else if (lane == 0) {                                        // ---- products
        const uint32_t id_s = (1u << 4) | ((uint32_t)(kKvpKeys >> 3) << 17) | ((uint32_t)(kKvpRows >> 4) << 24);
        const uint32_t id_o = (1u << 4) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kKvpRows >> 4) << 24);
        ok = tiles == 0 || kvp_wait(b_q, 0, abort_flag);
        auto scores = [&](int j) {
            const int st = j & 1;
            if (!kvp_wait(b_kf + 8 * st, (j >> 1) & 1, abort_flag)) return false;
            tc_fence_after();
            const uint32_t k = sb + Sm::k + st * Sm::k_bytes;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                umma_f16(t_s + st * 64, umma_desc_sw128(sb + Sm::q + (i >> 2) * Sm::q_block + (i & 3) * 32),
                         umma_desc_sw128(k + (i >> 2) * Sm::k_block + (i & 3) * 32), id_s, i > 0);
            umma_commit(b_s + 8 * st);                             // (the scores are there, and the keys' place is free)
            return true;
        };
        if (ok && tiles > 0) ok = scores(0);
        for (int j = 0; ok && j < tiles; ++j) {
            const int st = j & 1;
            // the buffer that the scores of tile j + 1 go to is the one that the product of tile j - 1 with V reads
            if (j + 1 < tiles) ok = (j == 0 || kvp_wait(b_o + 8 * (st ^ 1), ((j - 1) >> 1) & 1, abort_flag)) && scores(j + 1);
            ok = ok && kvp_wait(b_vf + 8 * st, (j >> 1) & 1, abort_flag) && kvp_wait(b_p + 8 * st, (j >> 1) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t v = sb + Sm::v + st * Sm::v_bytes;
#pragma unroll
            for (int i = 0; i < kKvpKeys / 16; ++i) umma_f16_ts(t_o, t_s + st * 64 + i * 8, umma_desc_sw128(v + i * 32), id_o, j > 0 || i > 0);
            umma_commit(b_o + 8 * st);
        }
    }
    __syncwarp();
    __syncthreads();                                               // (`bad` is complete)
    if (warp < 4) {
        tc_fence_after();
        const float nan = __int_as_float(0x7fffffff);
        const bool whole = p.cluster == 1;
        const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;
        const bool none = whole && l == 0.f && kv4_sees(rg, pos, p.window);   // keys, but no score above -inf (as in kv4_store)
        const size_t at = ((size_t)b * gridDim.x + blockIdx.x) * kKvpRows + tid;
        __nv_bfloat16* dst = p.out + (((size_t)b * p.tokens + t) * p.heads + h) * D;
        if (!whole) p.part_ml[at] = make_float2(-nb, ok ? l : nan);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            float o[32];
            if (tiles > 0) {
                tmem_ld32(t_o + mine + c, o);
                tmem_ld32_wait(o);
            }
            bool lost = !ok || !rg.ok || none || seen_to >= bad[c / 32];
            if (p.window && ok && rg.ok && !none && lost) {                 // (`bad` is the first such key: is there one that this row sees?)
                lost = false;
                const __half* vs = p.c.v_scales + (row0 - base) * G + c / 32;
                for (int key = max(seen_from, base); key <= min(seen_to, base + tiles * kKvpKeys - 1); ++key)
                    lost |= (__half_as_ushort(vs[(size_t)key * G]) & 0x7fff) > 0x6fff;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = lost ? nan : l == 0.f ? 0.f : o[i] * inv;
            if (!whole) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(p.part_o + at * D + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            } else if (row < rows_all) {
#pragma unroll
                for (int i = 0; i < 32; i += 8)
                    stg_128(dst + c + i, make_uint4(bf16_pack(o[i], o[i + 1]), bf16_pack(o[i + 2], o[i + 3]), bf16_pack(o[i + 4], o[i + 5]), bf16_pack(o[i + 6], o[i + 7])));
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (*abort_flag && tid == 0) atomicExch(p.status, ST_WAIT_TIMEOUT);
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, Sm::columns);
    }
}

// Joins the parts of a row, a warp per row.  One that saw no key has sum 0 and stays out; NaN of a part's values or sum goes to the row.
constexpr int kKvpJoinWarps = 8;
template <int D>
__global__ void __launch_bounds__(kKvpJoinWarps * 32) kv4_prefill_join_kernel(const Kv4AttnParams p) {
    constexpr int DEEP = 8;                                        // parts on their way at once
    const int lane = threadIdx.x & 31, per_kv = p.heads / p.c.kv_heads, rows = p.tokens * per_kv, b = blockIdx.y;
    const long long at = (long long)blockIdx.x * kKvpJoinWarps + (threadIdx.x >> 5);
    griddep_wait();
    if (at >= (long long)rows * p.c.kv_heads) return;
    const int hk = (int)(at / rows), row = (int)(at % rows);
    const int item = (p.row_tiles - 1 - row / kKvpRows) * p.c.kv_heads + hk;
    const size_t first = ((size_t)b * p.row_tiles * p.c.kv_heads + item) * p.cluster * kKvpRows + row % kKvpRows;
    float top = -INFINITY, sum = 0.f;
    float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < p.cluster; c += DEEP) {
        float2 ml[DEEP];
        float4 y[DEEP];
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            ml[j] = make_float2(0.f, 0.f);
            if (c + j >= p.cluster) continue;
            const size_t from = first + (size_t)(c + j) * kKvpRows;
            ml[j] = p.part_ml[from];
            if (lane < D / 4) y[j] = *reinterpret_cast<const float4*>(p.part_o + from * D + lane * 4);
        }
#pragma unroll
        for (int j = 0; j < DEEP; ++j) {
            if (ml[j].y == 0.f) continue;
            const float to = fmaxf(top, ml[j].x), f = top == -INFINITY ? 0.f : ex2_approx(top - to), g = ex2_approx(ml[j].x - to);
            top = to, sum = sum * f + ml[j].y * g;
            val.x = val.x * f + y[j].x * g, val.y = val.y * f + y[j].y * g, val.z = val.z * f + y[j].z * g, val.w = val.w * f + y[j].w * g;
        }
    }
    const Kv4Range rg = kv4_range(p.start, p.counts, p.start_stride, b, p.tokens, p.window, p.c.max_len, 0, 0);
    if (lane < D / 4) kv4_store(p, rg, rg.first_pos + row / per_kv, b, hk, per_kv, row, lane * 4, val, sum);
}

}  // namespace tsp
