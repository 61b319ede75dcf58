// Log probabilities of given tokens for sm_100a: per row of logits the log probability of one token, the entropy of the
// distribution and the most probable tokens, from one pass over the row; and the gradient of the first two.
//
// With a reference r and t = x log2(e) - r,  l = sum 2^t and w = sum 2^t t:  lse = ln(2) (r + log2 l), H = ln(2) (log2 l - w / l).
// Rows are cut into parts of 32 KB, which a fixed number of CTAs take in turn, the next one on its way to shared memory
// (cp.async) while one is worked on: so the load is even whatever the number of rows, and three parts per SM are always in flight.  A warp takes
// the maximum of its share first - from shared memory, two 16-bit values at a time - and then the sums against it, so nothing
// is ever rescaled.  For the alternatives a CTA takes up to eight parts of a row in turn: the k-th largest of the maxima of 32 groups of 8
// threads is a bound that at least k elements of the first one reach, and few more do (k = 20: 31 on average); they and what exceeds the bound in the
// other parts are collected, and ranked by counting.  A second kernel, a warp per row, joins the sums and merges the lists.
#pragma once
#include "rotary.cuh"
#include "w2_tile.cuh"

namespace tsp {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 8;                                        // 16-byte vectors of a thread and part
constexpr int kLpPartBytes = kLpThreads * kLpVecs * 16;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxVocab = 1 << 20;
constexpr int kLpCandidates = 512;
constexpr int kLpCtasPerSm = 3;

struct LogprobParams {
    const void* logits;
    long long ld;                          // elements between two rows
    const long long* targets;
    float *logprob, *entropy, *lse;
    float* top_logprob;                    // [rows][top]
    long long* top_token;
    float* sums;                           // [rows][parts][warps]: r, l, w and the warp's maximum
    unsigned long long* keys;              // [rows][lists][top], largest first, 0 where there are fewer elements
    int rows, vocab, top, parts;
    int run, lists;                        // parts that a CTA takes in turn; such runs of a row
    int* status;
};

// Order of the values as unsigned numbers: NaN above all, +0 and -0 alike; nothing is 0.
__device__ __forceinline__ uint32_t lp_order(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) {
    return o == 0xffffffffu ? __int_as_float(0x7fffffff) : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// larger value first, then the lower index
__device__ __forceinline__ unsigned long long lp_key(float x, int i) { return (unsigned long long)lp_order(x) << 32 | (0xffffffffu - (uint32_t)i); }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 16 bytes of logits
template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static constexpr uint32_t none = 0xff800000u;                 // -inf
    uint4 w;
    __device__ __forceinline__ float max() const { return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w))); }
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w); }
    __device__ __forceinline__ LpVec floored() const {            // no value below -1e37 (but NaN stays)
        LpVec r;
        const uint32_t* a = &w.x;
        uint32_t* d = &r.w.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float y;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(__uint_as_float(a[i])), "f"(-1e37f));
            d[i] = __float_as_uint(y);
        }
        return r;
    }
};
#define TSP_LP_VEC16(T, TYPE, NONE, FLOOR, LO, HI)                                                                                        \
    template <> struct LpVec<T> {                                                                                                         \
        static constexpr int N = 8;                                                                                                       \
        static constexpr uint32_t none = NONE;                                                                                            \
        uint4 w;                                                                                                                          \
        static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {                                                         \
            uint32_t r;                                                                                                                   \
            asm("max." TYPE " %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));                                                                   \
            return r;                                                                                                                     \
        }                                                                                                                                 \
        static __device__ __forceinline__ uint32_t floor2(uint32_t a) {                                                                   \
            uint32_t r;                                                                                                                   \
            asm("max.NaN." TYPE " %0, %1, %2;" : "=r"(r) : "r"(a), "r"(FLOOR));                                                           \
            return r;                                                                                                                     \
        }                                                                                                                                 \
        __device__ __forceinline__ float max() const {                                                                                    \
            const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));                                                                      \
            return fmaxf(LO(m), HI(m));                                                                                                   \
        }                                                                                                                                 \
        __device__ __forceinline__ void get(float (&x)[8]) const {                                                                        \
            x[0] = LO(w.x), x[1] = HI(w.x), x[2] = LO(w.y), x[3] = HI(w.y), x[4] = LO(w.z), x[5] = HI(w.z), x[6] = LO(w.w), x[7] = HI(w.w); \
        }                                                                                                                                 \
        __device__ __forceinline__ LpVec floored() const { return {make_uint4(floor2(w.x), floor2(w.y), floor2(w.z), floor2(w.w))}; }     \
    }
__device__ __forceinline__ float lp_f16_lo(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)v)); }
__device__ __forceinline__ float lp_f16_hi(uint32_t v) { return __half2float(__ushort_as_half((unsigned short)(v >> 16))); }
TSP_LP_VEC16(__nv_bfloat16, "bf16x2", 0xff80ff80u, 0xfe80fe80u, bf16_lo, bf16_hi);   // floor -2^126
TSP_LP_VEC16(__half, "f16x2", 0xfc00fc00u, 0xfbfffbffu, lp_f16_lo, lp_f16_hi);      // floor -65504
#undef TSP_LP_VEC16

// Whether a maximum is neither so large or low that log2(e) could take logits out of fp32's range, nor so low that the floor that -inf is
// raised to (for the sake of 0 * -inf) would weigh anything beside it.
template <typename T>
__device__ __forceinline__ bool lp_near(float m) {
    return fabsf(m) < 1e36f && (sizeof(T) == 4 || LpVec<T>::none != 0xfc00fc00u || m > -6e4f);
}

__device__ __forceinline__ float2 f32x2_add(float2 a, float2 b) {
    unsigned long long r;
    float2 o;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f32x2(a.x, a.y)), "l"(f32x2(b.x, b.y)));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
    return o;
}

// Where part `part` of row `r` lies: vectors first .. of the row's 16-byte aligned middle; up to 15 elements of its edges go with the first and
// the last part, one to a thread.
template <typename T>
struct LpPart {
    const T* row;
    int head, vecs, first, part, parts, vocab;
    __device__ __forceinline__ LpPart(const LogprobParams& p, long long item) {
        constexpr int V = LpVec<T>::N;
        const long long r = item / p.parts;
        part = (int)(item - r * p.parts), parts = p.parts, vocab = p.vocab;
        row = static_cast<const T*>(p.logits) + r * p.ld;
        head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
        vecs = (vocab - head) / V, first = part * kLpThreads * kLpVecs;
    }
    __device__ __forceinline__ int index(int j, int tid) const { return head + (first + j * kLpThreads + tid) * LpVec<T>::N; }   // of a vector's first element
    __device__ __forceinline__ bool has(int j, int tid) const { return first + j * kLpThreads + tid < vecs; }
    __device__ __forceinline__ int edge(int tid) const {          // index of this thread's element of the edges, or -1
        if (part == 0 && tid < head) return tid;
        const int rest = head + vecs * LpVec<T>::N + tid - 8;
        return part == parts - 1 && tid >= 8 && rest < vocab && tid < 16 ? rest : -1;
    }
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) logprob_kernel(const LogprobParams p) {
    using Vec16 = LpVec<T>;
    constexpr int V = Vec16::N;
    extern __shared__ __align__(128) uint8_t smem[];              // two parts
    __shared__ unsigned long long cand[kLpCandidates], best[kLpWarps];
    __shared__ uint32_t groups[32];
    __shared__ int n_cand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t mine = smem_u32(smem) + tid * 16;
    // run `c` of the launch is parts first .. first + count - 1 (of all rows, one behind the other)
    const long long runs = (long long)p.rows * p.lists;
    auto run_first = [&](long long c) { return c / p.lists * p.parts + c % p.lists * p.run; };
    auto run_count = [&](long long c) { return min(p.run, p.parts - (int)(c % p.lists) * p.run); };
    griddep_launch_dependents();
    auto fetch = [&](long long item, int buf) {
        const LpPart<T> at(p, item);
#pragma unroll
        for (int j = 0; j < kLpVecs; ++j) {
            const uint32_t dst = mine + buf * kLpPartBytes + j * (kLpThreads * 16);
            if (at.has(j, tid)) cp_async_16(dst, at.row + at.index(j, tid));
            else sts128(dst, make_uint4(Vec16::none, Vec16::none, Vec16::none, Vec16::none));
        }
    };
    if (tid == 0) n_cand = 0;
    if (blockIdx.x < runs) fetch(run_first(blockIdx.x), 0);
    cp_async_commit();
    uint32_t bound = 0;
    int buf = 0;
#pragma unroll 1
    for (long long run = blockIdx.x; run < runs; run += gridDim.x) {
    const long long first = run_first(run);
    const int count = run_count(run);
    bool full = false;
#pragma unroll 1
    for (int k = 0; k < count; ++k, buf ^= 1) {
        const long long item = first + k;
        if (k + 1 < count) fetch(item + 1, buf ^ 1);
        else if (run + gridDim.x < runs) fetch(run_first(run + gridDim.x), buf ^ 1);
        cp_async_commit();
        const LpPart<T> at(p, item);
        const int edge = at.edge(tid);
        const float xe = edge >= 0 ? Elem<T>::get(at.row[edge]) : -INFINITY;
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        const uint32_t src = mine + buf * kLpPartBytes;
        float tm = xe;                                             // this thread's maximum (NaN aside)
        uint32_t hits = 0;                                         // vectors with an element above the bound of the parts before
        const float above = k > 0 ? lp_value(bound) : INFINITY;
#pragma unroll
        for (int j = 0; j < kLpVecs; ++j) {
            const float vm = Vec16{lds128(src + j * (kLpThreads * 16))}.max();
            tm = fmaxf(tm, vm);
            if (vm > above) hits |= 1u << j;
        }
        float m = tm;
#pragma unroll
        for (int j = 16; j; j >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, j));
        float2 l = make_float2(0.f, 0.f), w = l;
        float r = 0.f;
        if (lp_near<T>(m)) {
            r = m * kLog2e;
            const float2 e2 = make_float2(kLog2e, kLog2e), nr = make_float2(-r, -r);
#pragma unroll
            for (int j = 0; j < kLpVecs; ++j) {
                float x[V];
                Vec16{lds128(src + j * (kLpThreads * 16))}.floored().get(x);
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 t = f32x2_fma(make_float2(x[i], x[i + 1]), e2, nr), e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
                    l = f32x2_add(l, e), w = f32x2_fma(e, t, w);
                }
            }
            if (edge >= 0) {
                const float t = fmaf(xe < -1e37f ? -1e37f : xe, kLog2e, -r), e = ex2_approx(t);
                l.x += e, w.x = fmaf(e, t, w.x);
            }
        } else {                                                   // a maximum of the type's largest or lowest order, or infinite: differences first
            auto add = [&](float x) {
                const float t = fmaxf((x - m) * kLog2e, -200.f), e = x == -INFINITY ? 0.f : ex2_approx((x - m) * kLog2e);
                l.x += e, w.x = fmaf(e, t, w.x);
            };
#pragma unroll 1
            for (int j = 0; j < kLpVecs; ++j) {
                float x[V];
                Vec16{lds128(src + j * (kLpThreads * 16))}.get(x);
#pragma unroll
                for (int i = 0; i < V; ++i) add(x[i]);
            }
            if (edge >= 0) add(xe);
        }
        l.x += l.y, w.x += w.y;
        const float own = l.x;
#pragma unroll
        for (int j = 16; j; j >>= 1) l.x += __shfl_xor_sync(0xffffffffu, l.x, j), w.x += __shfl_xor_sync(0xffffffffu, w.x, j);
        if (lane == 0) *reinterpret_cast<float4*>(p.sums + (item * kLpWarps + warp) * 4) = make_float4(r, l.x, w.x, m);
        if (p.top == 0) continue;

        // ---- candidates for the most probable tokens
        const bool odd = own != own;                               // NaN or +inf among this thread's elements: which, the sum does not tell
        if (k == 0) {
            uint32_t u = lp_order(tm);
            if (odd) {
                u = lp_order(xe);
#pragma unroll 1
                for (int j = 0; j < kLpVecs; ++j) {
                    float x[V];
                    Vec16{lds128(src + j * (kLpThreads * 16))}.get(x);
#pragma unroll
                    for (int i = 0; i < V; ++i) u = max(u, lp_order(x[i]));
                }
            }
            uint32_t gm = u;
#pragma unroll
            for (int j = 1; j < 8; j <<= 1) gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, j));
            if ((lane & 7) == 0) groups[warp * 4 + (lane >> 3)] = gm;
            __syncthreads();
            const uint32_t v = groups[lane];
            bound = 0;
#pragma unroll 1
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1)       // the largest that p.top of the groups reach
                if (__popc(__ballot_sync(0xffffffffu, v >= (bound | bit))) >= p.top) bound |= bit;
            if (u >= bound) {
                const float bf = lp_value(bound);
#pragma unroll
                for (int j = 0; j < kLpVecs; ++j)
                    if (!(Vec16{lds128(src + j * (kLpThreads * 16))}.max() < bf)) hits |= 1u << j;
            }
        }
        if (odd && bound != 0xffffffffu) hits = (1u << kLpVecs) - 1;
        // (an element of a later part that equals the bound has a higher index than the p.top elements that reach it)
        const uint32_t least = bound + (k > 0 ? 1u : 0u);
        const float bf = lp_value(least);
        auto push = [&](float x, int i) {
            if (lp_order(x) >= least) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < kLpCandidates) cand[at] = lp_key(x, i);
            }
        };
        if (bound == 0xffffffffu && k > 0) hits = 0;               // (nothing is above p.top times NaN, or the run is past keeping candidates)
        while (hits) {
            const int j = __ffs(hits) - 1;
            hits &= hits - 1;
            if (!at.has(j, tid)) continue;
            float x[V];
            Vec16{lds128(src + j * (kLpThreads * 16))}.get(x);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!(x[i] < bf)) push(x[i], at.index(j, tid) + i);
        }
        if (edge >= 0 && !(bound == 0xffffffffu && k > 0)) push(xe, edge);
        // ---- after the parts 1, 2, 4 of a run and its last one the best are kept, in their order, and the bound follows
        if (k == 0 || k == 1 || k == 3 || k == count - 1) {
            __syncthreads();
            const int n = n_cand;
            if (n > kLpCandidates) {                               // many elements at the bound or above it: found at the end
                full = true, bound = 0xffffffffu;
            } else {
                unsigned long long key[kLpCandidates / kLpThreads];
                int rank[kLpCandidates / kLpThreads];
#pragma unroll
                for (int i = 0; i < kLpCandidates / kLpThreads; ++i) {
                    key[i] = tid + i * kLpThreads < n ? cand[tid + i * kLpThreads] : 0ull, rank[i] = 0;
                    if (key[i])
                        for (int j = 0; j < n; ++j) rank[i] += cand[j] > key[i];
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kLpCandidates / kLpThreads; ++i)
                    if (key[i] && rank[i] < p.top) cand[rank[i]] = key[i];
                if (tid == 0) n_cand = min(n, p.top);
                __syncthreads();
                if (n >= p.top) bound = (uint32_t)(cand[p.top - 1] >> 32);
            }
        }
    }
    if (p.top == 0) continue;
    unsigned long long* keys = p.keys + run * p.top;
    if (!full) {
        if (tid < p.top) keys[tid] = tid < n_cand ? cand[tid] : 0ull;
    } else {                                                       // a pass over the run for each place
        unsigned long long last = ~0ull;
        for (int place = 0; place < p.top; ++place) {
            unsigned long long key = 0;
            auto look = [&](float x, int i) {
                const unsigned long long y = lp_key(x, i);
                if (y < last && y > key) key = y;
            };
#pragma unroll 1
            for (int k = 0; k < count; ++k) {
                const LpPart<T> at(p, first + k);
#pragma unroll 1
                for (int j = 0; j < kLpVecs; ++j) {
                    if (!at.has(j, tid)) continue;
                    float x[V];
                    Vec16{ldg_128(at.row + at.index(j, tid))}.get(x);
#pragma unroll
                    for (int i = 0; i < V; ++i) look(x[i], at.index(j, tid) + i);
                }
                const int edge = at.edge(tid);
                if (edge >= 0) look(Elem<T>::get(at.row[edge]), edge);
            }
#pragma unroll
            for (int i = 16; i; i >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, i);
                key = other > key ? other : key;
            }
            __syncthreads();
            if (lane == 0) best[warp] = key;
            __syncthreads();
            key = best[0];
            for (int i = 1; i < kLpWarps; ++i) key = best[i] > key ? best[i] : key;
            last = key;
            if (tid == 0) keys[place] = key;
        }
    }
    __syncthreads();
    if (tid == 0) n_cand = 0;                                      // (seen by all at the next run's first barrier)
    }
}

// Log probability; rounding does not take it above 0.
__device__ __forceinline__ float lp_least(float x, float m, float ln) {
    const float lp = (x - m) - ln;
    return lp > 0.f ? 0.f : lp;
}

// Joins a row's parts: a warp per row.
template <typename T>
__global__ void __launch_bounds__(32) logprob_join_kernel(const LogprobParams p) {
    extern __shared__ unsigned long long lists[];                 // [lists][top], then the places reached in them
    const int lane = threadIdx.x;
    const long long r = blockIdx.x;
    const T* row = static_cast<const T*>(p.logits) + r * p.ld;
    const long long target = p.targets[r];
    const float xt = target >= 0 && target < p.vocab ? Elem<T>::get(row[target]) : 0.f;
    griddep_wait();
    const float4* s = reinterpret_cast<const float4*>(p.sums) + r * p.parts * kLpWarps;
    const int n = p.parts * kLpWarps;
    int* place = reinterpret_cast<int*>(lists + p.lists * p.top);
    for (int i = lane; i < p.lists * p.top; i += 32) lists[i] = p.keys[r * p.lists * p.top + i];
    for (int i = lane; i < p.lists; i += 32) place[i] = 0;
    float m = -INFINITY, l = 0.f, w = 0.f;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, s[i].w);
#pragma unroll
    for (int j = 16; j; j >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, j));
    // the warps' sums are relative to r = m log2(e) as rounded, or to m itself where that is far out
    const bool far = !lp_near<T>(m);
    const float ref = far ? 0.f : m * kLog2e;
    for (int i = lane; i < n; i += 32) {
        const float4 a = s[i];
        // exponent that takes the warp's sums to the row's reference
        const float d = a.w == -INFINITY ? (a.y != a.y ? 0.f : -INFINITY) : far ? (a.w - m) * kLog2e : lp_near<T>(a.w) ? a.x - ref : fmaf(a.w, kLog2e, -ref);
        const float f = ex2_approx(d);
        l += a.y * f, w += (a.z + a.y * fmaxf(d, -200.f)) * f;
    }
#pragma unroll
    for (int j = 16; j; j >>= 1) l += __shfl_xor_sync(0xffffffffu, l, j), w += __shfl_xor_sync(0xffffffffu, w, j);
    const float ll = log2f(l);
    // ln of the sum of exp(x - m); m log2(e) was rounded
    const float ln = m == -INFINITY ? __int_as_float(0x7fffffff) : far ? ll * kLn2 : (ll - fmaf(m, kLog2e, -ref)) * kLn2;
    if (lane == 0) {
        float lp = lp_least(xt, m, ln);
        if (target < 0) lp = 0.f;                                  // no token
        if (target >= p.vocab) {
            lp = __int_as_float(0x7fffffff);
            *p.status = 1;
        }
        p.logprob[r] = lp;
        const float h = (ll - w / l) * kLn2;
        p.entropy[r] = ln != ln ? ln : h < 0.f ? 0.f : h;
        p.lse[r] = m + ln;
    }
    __syncwarp();
    for (int k = 0; k < p.top; ++k) {                              // the lists' heads against each other
        unsigned long long key = 0;
        int from = 0;
        for (int i = lane; i < p.lists; i += 32) {
            const unsigned long long head = place[i] < p.top ? lists[i * p.top + place[i]] : 0ull;
            if (head > key) key = head, from = i;
        }
        unsigned long long top = key;
#pragma unroll
        for (int j = 16; j; j >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, j);
            top = other > top ? other : top;
        }
        if (key == top) {                                          // (keys differ: one lane; top <= vocab: none is 0)
            ++place[from];
            p.top_logprob[r * p.top + k] = lp_least(lp_value((uint32_t)(key >> 32)), m, ln);
            p.top_token[r * p.top + k] = 0xffffffffu - (uint32_t)key;
        }
        __syncwarp();
    }
}

struct LogprobGradParams {
    const void* logits;
    long long ld;
    const long long* targets;
    const float *lse, *entropy, *g_logprob, *g_entropy;            // either gradient may be null
    void* grad;                                                    // contiguous [rows][vocab]
    int vocab;
};

// d/dx_j = g (delta_jt - p_j) - h p_j (log p_j + H).  One CTA per row and part of it.
template <typename T>
__global__ void __launch_bounds__(256) logprob_grad_kernel(const LogprobGradParams p, int parts) {
    constexpr int V = 16 / sizeof(T);
    const size_t r = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    const T* row = static_cast<const T*>(p.logits) + (long long)r * p.ld;
    T* out = static_cast<T*>(p.grad) + r * (size_t)p.vocab;
    const long long t = p.targets[r];
    const float g = p.g_logprob && t >= 0 ? p.g_logprob[r] : 0.f, h = p.g_entropy ? p.g_entropy[r] : 0.f;
    const float lse = p.lse[r], ent = p.entropy[r];
    auto one = [&](int j, float x) {
        const float lp = x - lse, e = ex2_approx(lp * kLog2e);
        const float d = -e * fmaf(h, fmaxf(lp, -200.f) + ent, g);
        return j == t ? d + g : d;
    };
    const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int head = same ? min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T)) : 0;
    const int vecs = same ? (p.vocab - head) / V : 0;
    const int tid = part * 256 + threadIdx.x, all = parts * 256;
    for (int i = tid; i < vecs; i += all) {
        const int j0 = head + i * V;
        const Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(row + j0);
        Vec<T, V> y;
#pragma unroll
        for (int j = 0; j < V; ++j) y.v[j] = Elem<T>::put(one(j0 + j, Elem<T>::get(x.v[j])));
        *reinterpret_cast<Vec<T, V>*>(out + j0) = y;
    }
    for (int i = tid; i < p.vocab - vecs * V; i += all) {
        const int j = i < head ? i : i + vecs * V;
        out[j] = Elem<T>::put(one(j, Elem<T>::get(row[j])));
    }
}

}  // namespace tsp
