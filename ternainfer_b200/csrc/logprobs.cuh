// Log probabilities of given tokens for sm_100a: per row of logits the log probability of one token, the entropy of the
// distribution and the most probable tokens, from one pass over the row; and the gradient of the first two.
//
// With a reference r and t = x log2(e) - r,  l = sum 2^t and w = sum 2^t t:  lse = ln(2) (r + log2 l), H = ln(2) (log2 l - w / l).  fp32 has room
// for sums of elements far above the reference, so that the maximum of a run's first part serves for all of it but in the rarest cases.
// Rows are cut into parts of 32 KB, which a fixed number of CTAs take in turn, a warp's 4 KB of the next one on their way to
// shared memory (one bulk copy) while it works on one: so the load is even whatever the number of rows, and three parts per SM are always in flight.  A warp takes
// the maximum of its share first - two 16-bit values at a time - and then the sums against it, so nothing
// is ever rescaled.  For the alternatives a CTA takes up to eight parts of a row in turn: the k-th largest of the maxima of 32 groups of 8
// threads is a bound that at least k elements of the first one reach, and few more do (k = 20: 31 on average); they and what exceeds the bound in the
// other parts are collected, and ranked by counting.  A second kernel, a warp per row, joins the sums and merges the lists.
//
// 1,226 rows of 128,256 bf16: 62 us, 5.1 TB/s of 6.46, bound by the exponentials (two 16-bit logits a lane take two of them) at 24 warps an SM; with 20
// alternatives 106 us: two to four barriers of the CTA and a ranking per run of parts.  3 rows of fp32 with 5 alternatives 9.4 us, two launches' latencies.
#pragma once
#include "rotary.cuh"
#include "w2_tile.cuh"

namespace tsp {

constexpr int kLpThreads = 256, kLpWarps = kLpThreads / 32;
constexpr int kLpVecs = 8;                                        // 16-byte vectors of a thread and part
constexpr int kLpPartBytes = kLpThreads * kLpVecs * 16, kLpWarpBytes = kLpPartBytes / kLpWarps;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxVocab = 1 << 19;
constexpr int kLpCandidates = 512;
constexpr int kLpCtasPerSm = 3;

struct LpSums {                            // l and w relative to 2^ref
    double ref;
    float l, w;
};

struct LogprobParams {
    const void* logits;
    long long ld;                          // elements between two rows
    const long long* targets;
    float *logprob, *entropy, *lse;
    float* top_logprob;                    // [rows][top]
    long long* top_token;
    LpSums* sums;                          // [rows][lists][warps]
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
// larger value first, then the lower index; neither 0 nor the largest number
__device__ __forceinline__ unsigned long long lp_key(float x, int i) { return (unsigned long long)lp_order(x) << 32 | (0xfffffffeu - (uint32_t)i); }
__device__ __forceinline__ long long lp_token(unsigned long long key) { return 0xfffffffeu - (uint32_t)key; }

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr double kOverLog2e = 1.0 / kLog2e;                       // (of the rounded one: divisions in 64 bits took as long as a short row's sums)

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
    __device__ __forceinline__ LpPart(const LogprobParams& p, unsigned r, int which) {
        constexpr int V = LpVec<T>::N;
        part = which, parts = p.parts, vocab = p.vocab;
        row = static_cast<const T*>(p.logits) + r * p.ld;
        head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
        vecs = (vocab - head) / V, first = part * kLpThreads * kLpVecs;
    }
    // a warp has 256 vectors behind each other, a lane every 32nd of them
    __device__ __forceinline__ int vec(int j, int tid) const { return first + (tid >> 5) * (32 * kLpVecs) + j * 32 + (tid & 31); }
    __device__ __forceinline__ int index(int j, int tid) const { return head + vec(j, tid) * LpVec<T>::N; }   // of a vector's first element
    __device__ __forceinline__ bool has(int j, int tid) const { return vec(j, tid) < vecs; }
    __device__ __forceinline__ int edge(int tid) const { return edge(tid, part == 0, part == parts - 1); }
    __device__ __forceinline__ int edge(int tid, bool front, bool back) const {   // index of this thread's element of the edges, or -1
        if (front && tid < head) return tid;
        const int rest = head + vecs * LpVec<T>::N + tid - 8;
        return back && tid >= 8 && rest < vocab && tid < 16 ? rest : -1;
    }
};

// A warp's sums over a run of elements: l, w of every lane's, relative to 2^ref; `near`: ref is a float that takes the short way, up to elements of `limit`.
template <typename T>
struct LpRun {
    double ref = -INFINITY;
    float2 l = make_float2(0.f, 0.f), w = l;
    bool near = false;
    float limit = 0.f;

    // Adds the first n vectors of x16 and, where edge >= 0, xe; tm is the largest of them (NaN aside).  pl: the lane's own l, NaN where one of its
    // elements is NaN or +inf; again(j) reads vector j once more.
    template <typename F>
    __device__ __forceinline__ void add(const LpVec<T> (&x16)[kLpVecs], int n, float tm, int edge, float xe, float2& pl, float2& pw, F again) {
        constexpr int V = LpVec<T>::N;
        auto add_all = [&](float r, float2& sl, float2& sw) {      // t = x log2(e) - r
            const float2 e2 = make_float2(kLog2e, kLog2e), nr = make_float2(-r, -r);
#pragma unroll
            for (int j = 0; j < kLpVecs; ++j) {
                if (j >= n) break;
                float x[V];
                x16[j].floored().get(x);
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 t = f32x2_fma(make_float2(x[i], x[i + 1]), e2, nr), e = make_float2(ex2_approx(t.x), ex2_approx(t.y));
                    sl = f32x2_add(sl, e), sw = f32x2_fma(e, t, sw);
                }
            }
            if (edge >= 0) {
                const float t = fmaf(xe < -1e37f ? -1e37f : xe, kLog2e, -r), e = ex2_approx(t);
                sl.x += e, sw.x = fmaf(e, t, sw.x);
            }
        };
        if (near && !__any_sync(0xffffffffu, tm > limit)) {
            add_all((float)ref, pl, pw);
            l = f32x2_add(l, pl), w = f32x2_add(w, pw);
        } else {                                                   // the first part of a run, or one with much larger elements
            float m = tm;
#pragma unroll
            for (int j = 16; j; j >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, j));
            double part_ref = (double)m * kLog2e;
            if (lp_near<T>(m)) {
                part_ref = m * kLog2e;                             // (as rounded to fp32)
                add_all((float)part_ref, pl, pw);
            } else {                                               // a maximum of the type's largest or lowest order, or infinite: differences first
                auto far = [&](float x) {
                    const float t = fmaxf((x - m) * kLog2e, -200.f), e = x == -INFINITY ? 0.f : ex2_approx((x - m) * kLog2e);
                    pl.x += e, pw.x = fmaf(e, t, pw.x);
                };
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    float x[V];
                    again(j).get(x);
#pragma unroll
                    for (int i = 0; i < V; ++i) far(x[i]);
                }
                if (edge >= 0) far(xe);
            }
            // (part_ref of -inf: nothing but -inf and NaN)
            const double to = fmax(ref, part_ref);
            const float ds = ref == -INFINITY ? 0.f : (float)(ref - to), dp = part_ref == -INFINITY ? 0.f : (float)(part_ref - to);
            const float fs = ex2_approx(ds), fp = ex2_approx(dp), cs = fmaxf(ds, -200.f), cp = fmaxf(dp, -200.f);
            w.x = (w.x + w.y + (l.x + l.y) * cs) * fs + (pw.x + pw.y + (pl.x + pl.y) * cp) * fp, w.y = 0.f;
            l.x = (l.x + l.y) * fs + (pl.x + pl.y) * fp, l.y = 0.f;
            ref = to;
            near = fabs(ref) < 1.4e36 && lp_near<T>((float)(ref * 0.69314718)) && (double)(float)ref == ref;
            limit = (float)((ref + 60) * 0.69314718);              // (2^60 times as many elements as a row has fit into fp32)
        }
    }
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int j = 16; j; j >>= 1) x += __shfl_xor_sync(0xffffffffu, x, j);
    return x;
}

// Log probability of x beside a sum of 2^(ref + ll) (differences first: ll is nothing beside the reference of a row of the type's lowest value);
// rounding does not take it above 0.
__device__ __forceinline__ float lp_of(float x, double ref, float ll) {
    const float lp = (float)((((double)x * (double)kLog2e - ref) - ll) * kOverLog2e);
    return lp > 0.f ? 0.f : lp;
}
// A row's results but for the alternatives.
__device__ __forceinline__ void lp_finish(const LogprobParams& p, long long r, long long target, float xt, double ref, float ll, float l, float w) {
    float lp = lp_of(xt, ref, ll);
    if (target < 0) lp = 0.f;                                      // no token
    if (target >= p.vocab) {
        lp = __int_as_float(0x7fffffff);
        *p.status = 1;
    }
    p.logprob[r] = lp;
    const float h = (ll - w / l) * kLn2;
    p.entropy[r] = h < 0.f ? 0.f : h;
    // in two parts, for the gradient
    const float hi = (float)(ref * kOverLog2e);
    p.lse[2 * r] = hi, p.lse[2 * r + 1] = (float)(((ref - (double)hi * (double)kLog2e) + ll) * kOverLog2e);
}
// Of `mine` of all lanes, the k-th largest (k <= 32).
__device__ __forceinline__ uint32_t lp_kth(uint32_t mine, int k, int lane) {
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const uint32_t other = __shfl_sync(0xffffffffu, mine, j);
        rank += other > mine || (other == mine && j < lane);
    }
    return __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, rank == k - 1)) - 1);
}

// The same of two of every lane.
__device__ __forceinline__ uint32_t lp_kth_of_64(uint32_t a, uint32_t b, int k, int lane) {
    int rank_a = a < b, rank_b = a >= b;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const uint32_t x = __shfl_sync(0xffffffffu, a, j), y = __shfl_sync(0xffffffffu, b, j);
        if (j == lane) continue;
        rank_a += (x > a || (x == a && j < lane)) + (y > a || (y == a && j < lane));
        rank_b += (x > b || (x == b && j < lane)) + (y > b || (y == b && j < lane));
    }
    const uint32_t in_a = __ballot_sync(0xffffffffu, rank_a == k - 1), in_b = __ballot_sync(0xffffffffu, rank_b == k - 1);   // (one lane, one of its two)
    return __shfl_sync(0xffffffffu, in_a ? a : b, __ffs(in_a ? in_a : in_b) - 1);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) logprob_kernel(const LogprobParams p) {
    using Vec16 = LpVec<T>;
    constexpr int V = Vec16::N;
    extern __shared__ __align__(128) uint8_t smem[];              // two parts
    __shared__ unsigned long long cand[kLpCandidates], best[kLpWarps];
    __shared__ uint32_t groups[32];
    __shared__ int n_cand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    __shared__ __align__(8) unsigned long long bars[kLpWarps][2];
    const uint32_t mine = smem_u32(smem) + warp * (2 * kLpWarpBytes) + lane * 16, bar = smem_u32(bars[warp]);
    // run c of the launch: row c / lists, parts from c % lists * run on (32 bits: divisions of 64 were half of the instructions)
    const unsigned runs = (unsigned)p.rows * (unsigned)p.lists;
    griddep_launch_dependents();
    if (lane == 0) {
        mbar_init(bar, 1), mbar_init(bar + 8, 1);
        mbar_fence_init();
    }
    __syncwarp();
    // a warp's share of a part in one bulk copy; vectors behind the row's last one are filled in
    auto fetch = [&](const LpPart<T>& at, int buf) {
        const int from = at.vec(0, tid) - lane, n = min(max(at.vecs - from, 0), 32 * kLpVecs);
        if (n < 32 * kLpVecs) {
#pragma unroll 1
            for (int j = 0; j < kLpVecs; ++j)
                if (j * 32 + lane >= n) sts128(mine + buf * kLpWarpBytes + j * 512, make_uint4(Vec16::none, Vec16::none, Vec16::none, Vec16::none));
            fence_proxy_async_smem();                              // (a later copy may write there)
            __syncwarp();
        }
        if (lane == 0) {
            mbar_arrive_expect_tx(bar + 8 * buf, n * 16);
            if (n) bulk_load(mine + buf * kLpWarpBytes, at.row + at.index(0, tid), n * 16, bar + 8 * buf);
        }
    };
    if (tid == 0) n_cand = 0;
    if (blockIdx.x < runs) fetch(LpPart<T>(p, blockIdx.x / p.lists, blockIdx.x % p.lists * p.run), 0);
    uint32_t phases = 0;                                           // of the two barriers
    bool ok = true;
    uint32_t bound = 0;
    int buf = 0;
#pragma unroll 1
    for (unsigned run = blockIdx.x; run < runs; run += gridDim.x) {
    const unsigned r_now = run / p.lists, next = run + gridDim.x;
    const int first = (int)(run - r_now * p.lists) * p.run, count = min(p.run, p.parts - first);
    bool full = false;
    LpRun<T> sums;
    LpPart<T> at(p, r_now, first);
#pragma unroll 1
    for (int k = 0; k < count; ++k, buf ^= 1, ++at.part, at.first += kLpThreads * kLpVecs) {
        __syncwarp();                                              // (every lane has read what lay there)
        if (k + 1 < count) {
            LpPart<T> then = at;
            ++then.part, then.first += kLpThreads * kLpVecs;
            fetch(then, buf ^ 1);
        } else if (next < runs) {
            fetch(LpPart<T>(p, next / p.lists, next % p.lists * p.run), buf ^ 1);
        }
        const int edge = at.edge(tid);
        const float xe = edge >= 0 ? Elem<T>::get(at.row[edge]) : -INFINITY;
        ok = mbar_wait_bounded(bar + 8 * buf, phases >> buf & 1u) && ok;
        phases ^= 1u << buf;
        const uint32_t src = mine + buf * kLpWarpBytes;
        Vec16 x16[kLpVecs];
        float tm = xe;                                             // this thread's maximum (NaN aside)
        uint32_t hits = 0;                                         // vectors with an element above the bound of the parts before
        const float above = k > 0 ? lp_value(bound) : INFINITY;
#pragma unroll
        for (int j = 0; j < kLpVecs; ++j) x16[j].w = lds128(src + j * 512);
#pragma unroll
        for (int j = 0; j < kLpVecs; ++j) {
            const float vm = x16[j].max();
            tm = fmaxf(tm, vm);
            if (vm > above) hits |= 1u << j;
        }
        float2 pl = make_float2(0.f, 0.f), pw = pl;
        sums.add(x16, kLpVecs, tm, edge, xe, pl, pw, [&](int j) { return Vec16{lds128(src + j * 512)}; });
        if (p.top == 0) continue;

        // ---- candidates for the most probable tokens
        const float own = pl.x + pl.y;
        const bool odd = own != own;                               // NaN or +inf among this thread's elements: which, the sum does not tell
        if (k == 0) {
            uint32_t u = lp_order(tm);
            if (odd) {
                u = lp_order(xe);
#pragma unroll 1
                for (int j = 0; j < kLpVecs; ++j) {
                    float x[V];
                    Vec16{lds128(src + j * 512)}.get(x);
#pragma unroll
                    for (int i = 0; i < V; ++i) u = max(u, lp_order(x[i]));
                }
            }
            uint32_t gm = u;
#pragma unroll
            for (int j = 1; j < 8; j <<= 1) gm = max(gm, __shfl_xor_sync(0xffffffffu, gm, j));
            if ((lane & 7) == 0) groups[warp * 4 + (lane >> 3)] = gm;
            __syncthreads();
            bound = lp_kth(groups[lane], p.top, lane);             // that p.top of the groups reach
            if (u >= bound) {
                const float bf = lp_value(bound);
#pragma unroll
                for (int j = 0; j < kLpVecs; ++j)
                    if (!(x16[j].max() < bf)) hits |= 1u << j;
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
            Vec16{lds128(src + j * 512)}.get(x);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!(x[i] < bf)) push(x[i], at.index(j, tid) + i);
        }
        if (edge >= 0 && !(bound == 0xffffffffu && k > 0)) push(xe, edge);
        // ---- after the parts 1 and 3 of a run and its last one the best are kept, in their order, and the bound follows
        if (k == 0 || k == 2 || k == count - 1) {
            __syncthreads();
            const int n = n_cand;
            if (n > kLpCandidates) {                               // many elements at the bound or above it: found at the end
                full = true, bound = 0xffffffffu;
            } else {
                constexpr int PER = kLpThreads / 4;                // four threads to a candidate
                unsigned long long key[kLpCandidates / PER];
                int rank[kLpCandidates / PER];
#pragma unroll
                for (int i = 0; i < kLpCandidates / PER; ++i) {
                    const int c = i * PER + (tid >> 2);
                    key[i] = 0ull, rank[i] = 0;
                    if (i * PER >= n) continue;                    // (the same for all threads)
                    key[i] = c < n ? cand[c] : 0ull;
                    for (int j = tid & 3; j < n; j += 4) rank[i] += cand[j] > key[i];
                    rank[i] += __shfl_xor_sync(0xffffffffu, rank[i], 1);
                    rank[i] += __shfl_xor_sync(0xffffffffu, rank[i], 2);
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kLpCandidates / PER; ++i)
                    if ((tid & 3) == 0 && key[i] && rank[i] < p.top) cand[rank[i]] = key[i];
                if (tid == 0) n_cand = min(n, p.top);
                __syncthreads();
                if (n >= p.top) bound = (uint32_t)(cand[p.top - 1] >> 32);
            }
        }
    }
    {
        const float sl = warp_sum(sums.l.x + sums.l.y), sw = warp_sum(sums.w.x + sums.w.y);
        if (lane == 0) p.sums[(size_t)run * kLpWarps + warp] = {sums.ref, ok ? sl : __int_as_float(0x7fffffff), sw};
    }
    if (p.top == 0) continue;
    unsigned long long* keys = p.keys + (size_t)run * p.top;
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
                const LpPart<T> at(p, r_now, first + k);
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
    if (!ok && lane == 0) atomicExch(p.status, ST_WAIT_TIMEOUT);
}

// Short rows, a warp each and nothing between the warps: 100,000 rows of 300 fp32 logits take 89 us (1.3 TB/s; 754 with a CTA for each, which left
// most of it idle), 8,000 of 5,000 bf16 28 us (2.8 TB/s).  What bounds the shortest is the chain of loads, sums and logarithm of a row, 24 of
// them at work on an SM.  A warp has up to 4 KB of its row in registers at a time.  The k-th largest of the lanes' maxima is the bound for the
// alternatives of the first 4 KB, the k-th largest element so far that for the next ones.  Above the least of 32 maxima (k = 32) one row in a
// hundred has more than 256 elements, and takes ten times as long; so for many alternatives a lane has two groups, its even and its odd vectors:
// 44 elements on average are above the 32nd of 64 (300 rows of 4,000: 104 -> 19 us; with k = 5 the 64 cost 12.2 us and the 32 10.4).
constexpr int kLpRowCandidates = 256, kLpRanked = 64;
template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtasPerSm) logprob_rows_kernel(const LogprobParams p) {
    using Vec16 = LpVec<T>;
    constexpr int V = Vec16::N;
    __shared__ unsigned long long lists[kLpWarps][kLpRowCandidates];
    __shared__ int counts[kLpWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned r = blockIdx.x * kLpWarps + warp;
    if (r >= (unsigned)p.rows) return;                             // (no barrier of the CTA below)
    unsigned long long* cand = lists[warp];
    LpPart<T> at(p, r, 0);
    const long long target = p.targets[r];
    const float xt = target >= 0 && target < p.vocab ? Elem<T>::get(at.row[target]) : 0.f;
    if (lane == 0) counts[warp] = 0;
    LpRun<T> sums;
    uint32_t bound = 0;
    bool full = false;
#pragma unroll 1
    for (int k = 0; k == 0 || at.first < at.vecs; ++k, at.first += 32 * kLpVecs) {
        // (of the edges the row's last elements go with its last 4 KB, as ids ascend)
        const int edge = at.edge(lane, k == 0, at.first + 32 * kLpVecs >= at.vecs), n = min(kLpVecs, (at.vecs - at.first + 31) / 32);
        auto again = [&](int j) { return at.has(j, lane) ? Vec16{ldg_128(at.row + at.index(j, lane))} : Vec16{make_uint4(Vec16::none, Vec16::none, Vec16::none, Vec16::none)}; };
        Vec16 x16[kLpVecs];
#pragma unroll
        for (int j = 0; j < kLpVecs; ++j)
            if (j < n) x16[j] = again(j);
        const float xe = edge >= 0 ? Elem<T>::get(at.row[edge]) : -INFINITY;
        float tm2[2] = {xe, -INFINITY};                            // the maxima of this lane's groups (NaN aside)
        uint32_t hits = 0;                                         // vectors with an element above the bound so far
        const float above = k > 0 ? lp_value(bound) : INFINITY;
#pragma unroll
        for (int j = 0; j < kLpVecs; ++j) {
            if (j >= n) break;
            const float vm = x16[j].max();
            tm2[j & 1] = fmaxf(tm2[j & 1], vm);
            if (vm > above) hits |= 1u << j;
        }
        const float tm = fmaxf(tm2[0], tm2[1]);
        float2 pl = make_float2(0.f, 0.f), pw = pl;
        sums.add(x16, n, tm, edge, xe, pl, pw, again);
        if (p.top == 0 || full) continue;

        const float own = pl.x + pl.y;
        const bool odd = own != own;                               // NaN or +inf among this lane's elements: which, the sum does not tell
        if (k == 0) {
            uint32_t u = lp_order(tm2[0]), u1 = lp_order(tm2[1]);
            if (odd) {                                             // (its largest speaks for the lane)
                u = lp_order(xe), u1 = lp_order(-INFINITY);
#pragma unroll 1
                for (int j = 0; j < n; ++j) {
                    float x[V];
                    again(j).get(x);
#pragma unroll
                    for (int i = 0; i < V; ++i) u = max(u, lp_order(x[i]));
                }
            }
            bound = p.top > 24 ? lp_kth_of_64(u, u1, p.top, lane) : lp_kth(max(u, u1), p.top, lane);
            if (max(u, u1) >= bound) {
                const float bf = lp_value(bound);
#pragma unroll
                for (int j = 0; j < kLpVecs; ++j)
                    if (j < n && !(x16[j].max() < bf)) hits |= 1u << j;
            }
        }
        if (odd && bound != 0xffffffffu) hits = (1u << n) - 1;
        const uint32_t least = bound + (k > 0 ? 1u : 0u);          // (as in logprob_kernel)
        const float bf = lp_value(least);
        auto push = [&](float x, int i) {
            if (lp_order(x) >= least) {
                const int to = atomicAdd(&counts[warp], 1);
                if (to < kLpRowCandidates) cand[to] = lp_key(x, i);
            }
        };
        __syncwarp();
        if (bound == 0xffffffffu && k > 0) hits = 0;               // (nothing is above p.top times NaN)
        while (hits) {
            const int j = __ffs(hits) - 1;
            hits &= hits - 1;
            if (!at.has(j, lane)) continue;
            float x[V];
            again(j).get(x);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!(x[i] < bf)) push(x[i], at.index(j, lane) + i);
        }
        if (edge >= 0 && !(bound == 0xffffffffu && k > 0)) push(xe, edge);
        __syncwarp();
        int c = counts[warp];
        if (c > kLpRowCandidates) {                                // many elements at the bound or above it: found at the end
            full = true;
            continue;
        }
        if (c > kLpRanked) {                                       // a border that leaves p.top .. kLpRanked of them, by halving: keys differ
            unsigned long long key[kLpRowCandidates / 32], lo = 0ull, hi = ~0ull;
#pragma unroll
            for (int i = 0; i < kLpRowCandidates / 32; ++i) key[i] = i * 32 + lane < c ? cand[i * 32 + lane] : 0ull;
            if (least) lo = ((unsigned long long)least << 32) - 1; // (all are above it)
            int over = c;
#pragma unroll 1
            for (int step = 0; step < 64 && (over > kLpRanked || over < p.top); ++step) {
                const unsigned long long mid = lo + (hi - lo) / 2;
                int mine = 0;
#pragma unroll
                for (int i = 0; i < kLpRowCandidates / 32; ++i) mine += key[i] > mid;
                over = __reduce_add_sync(0xffffffffu, mine);
                if (over > kLpRanked) lo = mid;
                else hi = mid;                                     // (the border itself, if this ends it)
            }
            __syncwarp();
            c = 0;
#pragma unroll
            for (int i = 0; i < kLpRowCandidates / 32; ++i) {
                const uint32_t kept = __ballot_sync(0xffffffffu, key[i] > hi);
                if (key[i] > hi) cand[c + __popc(kept & ((1u << lane) - 1))] = key[i];
                c += __popc(kept);
            }
            __syncwarp();
        }
        const unsigned long long k0 = lane < c ? cand[lane] : 0ull, k1 = lane + 32 < c ? cand[lane + 32] : 0ull;
        int rank0 = 0, rank1 = 0;
        for (int i = 0; i < c; ++i) rank0 += cand[i] > k0, rank1 += cand[i] > k1;
        __syncwarp();
        if (k0 && rank0 < p.top) cand[rank0] = k0;
        if (k1 && rank1 < p.top) cand[rank1] = k1;
        if (lane == 0) counts[warp] = min(c, p.top);
        __syncwarp();
        if (c >= p.top) bound = (uint32_t)(cand[p.top - 1] >> 32);
    }
    double ref = sums.ref;                                         // (the same in all lanes)
    const float l = warp_sum(sums.l.x + sums.l.y), w = warp_sum(sums.w.x + sums.w.y);
    const float ll = ref == -INFINITY ? __int_as_float(0x7fffffff) : log2f(l);
    if (lane == 0) lp_finish(p, r, target, xt, ref, ll, l, w);
    if (p.top == 0) return;
    unsigned long long key = lane < p.top ? cand[lane] : 0ull;
    if (full) {                                                    // a pass over the row for each place
        unsigned long long last = ~0ull;
        for (int place = 0; place < p.top; ++place) {
            unsigned long long top = 0;
            for (int i = lane; i < p.vocab; i += 32) {
                const unsigned long long y = lp_key(Elem<T>::get(at.row[i]), i);
                if (y < last && y > top) top = y;
            }
#pragma unroll
            for (int j = 16; j; j >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, j);
                top = other > top ? other : top;
            }
            last = top;
            if (lane == place) key = top;
        }
    }
    if (lane < p.top) {
        p.top_logprob[(size_t)r * p.top + lane] = lp_of(lp_value((uint32_t)(key >> 32)), ref, ll);
        p.top_token[(size_t)r * p.top + lane] = lp_token(key);
    }
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
    const LpSums* s = p.sums + r * p.lists * kLpWarps;
    const int n = p.lists * kLpWarps;
    int* place = reinterpret_cast<int*>(lists + p.lists * p.top);
    for (int i = lane; i < p.lists * p.top; i += 32) lists[i] = p.keys[r * p.lists * p.top + i];
    for (int i = lane; i < p.lists; i += 32) place[i] = 0;
    double ref = -INFINITY;
    float l = 0.f, w = 0.f;
    for (int i = lane; i < n; i += 32) ref = fmax(ref, s[i].ref);
#pragma unroll
    for (int j = 16; j; j >>= 1) ref = fmax(ref, __shfl_xor_sync(0xffffffffu, ref, j));
    for (int i = lane; i < n; i += 32) {
        const LpSums a = s[i];
        const float d = a.ref == -INFINITY ? 0.f : (float)(a.ref - ref), f = ex2_approx(d);   // (-inf: l is 0 or NaN)
        l += a.l * f, w += (a.w + a.l * fmaxf(d, -200.f)) * f;
    }
#pragma unroll
    for (int j = 16; j; j >>= 1) l += __shfl_xor_sync(0xffffffffu, l, j), w += __shfl_xor_sync(0xffffffffu, w, j);
    // log2 of the sum of 2^(x log2(e)); the units are those of log2(e) as rounded to fp32.  Without a finite logit it is NaN
    const float ll = ref == -INFINITY ? __int_as_float(0x7fffffff) : log2f(l);
    if (lane == 0) lp_finish(p, r, target, xt, ref, ll, l, w);
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
            p.top_logprob[r * p.top + k] = lp_of(lp_value((uint32_t)(key >> 32)), ref, ll);
            p.top_token[r * p.top + k] = lp_token(key);
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
    int rows, vocab;
};

// d/dx_j = g (delta_jt - p_j) - h p_j (log p_j + H).  A CTA per row and part of it, or 256 / threads rows of one part: up
// to 2,048 tokens a warp (100,000 rows of 300: 64 us against 143).  512 rows of 128,256 fp32 after the forward pass: 149 us together, 5.3 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) logprob_grad_kernel(const LogprobGradParams p, int parts, int threads) {
    constexpr int V = 16 / sizeof(T);
    const size_t r = blockIdx.x / parts * (256u / threads) + threadIdx.x / threads;
    if (r >= (size_t)p.rows) return;
    const int part = blockIdx.x % parts;
    const T* row = static_cast<const T*>(p.logits) + (long long)r * p.ld;
    T* out = static_cast<T*>(p.grad) + r * (size_t)p.vocab;
    const long long t = p.targets[r];
    // (a token outside of the vocabulary has log probability NaN, and so has the gradient that comes through it)
    const float given = p.g_logprob && t >= 0 ? p.g_logprob[r] : 0.f, g = t >= p.vocab && given != 0.f ? __int_as_float(0x7fffffff) : given;
    const float h = p.g_entropy ? p.g_entropy[r] : 0.f;
    const float hi = p.lse[2 * r], lo = p.lse[2 * r + 1], ent = p.entropy[r];
    auto one = [&](int j, float x) {
        const float lp = (x - hi) - lo, e = ex2_approx(lp * kLog2e);
        const float d = -e * fmaf(h, fmaxf(lp, -200.f) + ent, g);
        return j == t ? d + g : d;
    };
    const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int head = same ? min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T)) : 0;
    const int vecs = same ? (p.vocab - head) / V : 0;
    const int tid = part * 256 + threadIdx.x % threads, all = parts * threads;
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
