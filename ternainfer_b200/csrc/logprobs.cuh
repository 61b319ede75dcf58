// Log probabilities of given tokens for sm_100a: per row of logits the log probability of one token, the entropy of the
// distribution and the most probable tokens, from one pass over the row; and the gradient of the first two.
//
// With m the running maximum, l = sum exp(x - m) and w = sum exp(x - m) (x - m):  lse = m + log l, log p_t = x_t - m - log l,
// H = log l - w / l.  Each thread keeps its own (m, l, w), joined at the end.  For the alternatives a thread's m is all that
// the pass has to keep: the k-th largest of the threads' maxima is a bound that at least k elements reach, and only the k threads
// or so that reach it have such elements.  They look through their own part of the row again, which is in L2 by then.
#pragma once
#include "rotary.cuh"

namespace tsp {

constexpr int kLpThreads = 512;
constexpr int kLpMaxTop = 32;
constexpr int kLpCandidates = 2048;

struct LogprobParams {
    const void* logits;
    long long ld;                          // elements between two rows
    const long long* targets;
    float *logprob, *entropy, *lse;
    float* top_logprob;                    // [rows][top]
    long long* top_token;
    int vocab, top;
    int* status;
};

struct LpSum { float m, l, w; };

__device__ __forceinline__ float ln_to_2(float x) { return x * 1.4426950408889634f; }

// (m, l, w) of two disjoint parts
__device__ __forceinline__ LpSum lp_join(const LpSum& a, const LpSum& b) {
    LpSum r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m == r.m ? 0.f : a.m - r.m, db = b.m == r.m ? 0.f : b.m - r.m;
    const float fa = ex2_approx(ln_to_2(da)), fb = ex2_approx(ln_to_2(db));
    r.l = a.l * fa + b.l * fb;
    r.w = (a.w + a.l * fmaxf(da, -200.f)) * fa + (b.w + b.l * fmaxf(db, -200.f)) * fb;
    return r;
}

// Order of the values as unsigned numbers: NaN above all, +0 and -0 alike.
__device__ __forceinline__ uint32_t lp_order(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) {
    return o == 0xffffffffu ? __int_as_float(0x7fffffff) : __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Calls f(index, value) for this thread's part of a row: every kLpThreads-th vector of the 16-byte aligned middle, and single
// elements of the edges.
template <typename T, typename F>
__device__ __forceinline__ void lp_visit(const T* row, int vocab, int tid, F f) {
    constexpr int V = 16 / sizeof(T);
    const int head = min(vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
    const int vecs = (vocab - head) / V;
    for (int i = tid; i < vecs; i += kLpThreads) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + head + (size_t)i * V);
        const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < V; ++j) f(head + i * V + j, Elem<T>::get(x[j]));
    }
    if (tid < head) f(tid, Elem<T>::get(row[tid]));
    const int rest = head + vecs * V + tid;
    if (rest < vocab) f(rest, Elem<T>::get(row[rest]));
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprob_kernel(const LogprobParams p) {
    constexpr int V = 16 / sizeof(T), WARPS = kLpThreads / 32;
    __shared__ LpSum sums[WARPS];
    __shared__ LpSum total;
    __shared__ unsigned long long cand[kLpCandidates];
    __shared__ unsigned long long best[WARPS];
    __shared__ int n_cand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t r = blockIdx.x;
    const T* row = static_cast<const T*>(p.logits) + (long long)r * p.ld;

    LpSum a = {-INFINITY, 0.f, 0.f};
    float ref = 0.f;                                               // m, or 0 while that is -inf
    auto take = [&](const float* x, int n) {
        float vm = x[0];
#pragma unroll
        for (int j = 1; j < n; ++j) vm = fmaxf(vm, x[j]);
        if (vm > a.m) {
            if (a.m != -INFINITY) {
                const float d = a.m - vm, f = ex2_approx(ln_to_2(d));
                a.w = (a.w + a.l * fmaxf(d, -200.f)) * f, a.l *= f;
            }
            a.m = ref = vm;
        }
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const float d = x[j] - ref, e = ex2_approx(ln_to_2(d));
            a.l += e, a.w = fmaf(e, fmaxf(d, -200.f), a.w);        // (exp(-inf) * -inf counts as nothing)
        }
    };
    const int head = min(p.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
    const int vecs = (p.vocab - head) / V;
#pragma unroll 4
    for (int i = tid; i < vecs; i += kLpThreads) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + head + (size_t)i * V);
        const T* x = reinterpret_cast<const T*>(&raw);
        float f[V];
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = Elem<T>::get(x[j]);
        take(f, V);
    }
    if (tid < head) {
        const float f = Elem<T>::get(row[tid]);
        take(&f, 1);
    }
    if (head + vecs * V + tid < p.vocab) {
        const float f = Elem<T>::get(row[head + vecs * V + tid]);
        take(&f, 1);
    }
    LpSum s = a;
#pragma unroll
    for (int i = 16; i; i >>= 1) {
        const LpSum b = {__shfl_xor_sync(0xffffffffu, s.m, i), __shfl_xor_sync(0xffffffffu, s.l, i), __shfl_xor_sync(0xffffffffu, s.w, i)};
        s = lp_join(s, b);
    }
    if (lane == 0) sums[warp] = s;
    if (tid == 0) n_cand = 0;
    __syncthreads();
    if (tid == 0) {
        s = sums[0];
        for (int i = 1; i < WARPS; ++i) s = lp_join(s, sums[i]);
        total = s;
        const float ln = logf(s.l);
        const long long t = p.targets[r];
        float lp;
        if (t < 0) {
            lp = 0.f;                                              // no token
        } else if (t >= p.vocab) {
            lp = __int_as_float(0x7fffffff);
            *p.status = 1;
        } else {
            lp = (Elem<T>::get(row[t]) - s.m) - ln;
        }
        p.logprob[r] = lp;
        p.entropy[r] = ln - s.w / s.l;
        p.lse[r] = s.m + ln;
    }
    if (p.top == 0) return;
    __syncthreads();

    // ---- the most probable tokens
    uint32_t bound = 0;
    if (p.vocab > kLpThreads) {                                    // (so that more threads than `top` have elements)
        uint32_t mine = lp_order(a.m);
        if (a.l != a.l) {                                          // NaN or +inf among the elements: which, the sums do not tell
            mine = 0;
            lp_visit(row, p.vocab, tid, [&](int, float x) { mine = max(mine, lp_order(x)); });
        }
        // the largest bound that top threads reach, or a smaller one that few more do
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
            const int n = __syncthreads_count(mine >= (bound | bit));
            if (n >= p.top) bound |= bit;
            if (n >= p.top && n <= p.top + 8) break;
        }
        if (mine >= bound)
            lp_visit(row, p.vocab, tid, [&](int i, float x) {
                const uint32_t u = lp_order(x);
                if (u >= bound) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < kLpCandidates) cand[at] = (unsigned long long)u << 32 | (0xffffffffu - (uint32_t)i);
                }
            });
    } else {
        for (int i = tid; i < p.vocab; i += kLpThreads) cand[i] = (unsigned long long)lp_order(Elem<T>::get(row[i])) << 32 | (0xffffffffu - (uint32_t)i);
        if (tid == 0) n_cand = p.vocab;
    }
    __syncthreads();
    const float lm = total.m, ln = logf(total.l);
    const int n = n_cand;
    auto put = [&](int rank, unsigned long long key) {
        p.top_logprob[r * p.top + rank] = (lp_value((uint32_t)(key >> 32)) - lm) - ln;
        p.top_token[r * p.top + rank] = 0xffffffffu - (uint32_t)key;
    };
    if (n <= kLpCandidates) {
        for (int i = tid; i < n; i += kLpThreads) {
            const unsigned long long key = cand[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += cand[j] > key;
            if (rank < p.top) put(rank, key);
        }
        return;
    }
    // many equal elements at the bound: one pass over the row for each place
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long mine = 0;
        lp_visit(row, p.vocab, tid, [&](int i, float x) {
            const unsigned long long key = (unsigned long long)lp_order(x) << 32 | (0xffffffffu - (uint32_t)i);
            if (key < last && key > mine) mine = key;
        });
#pragma unroll
        for (int i = 16; i; i >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, i);
            mine = other > mine ? other : mine;
        }
        __syncthreads();
        if (lane == 0) best[warp] = mine;
        __syncthreads();
        mine = best[0];
        for (int i = 1; i < WARPS; ++i) mine = best[i] > mine ? best[i] : mine;
        last = mine;
        if (tid == 0) put(k, mine);
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
        const float lp = x - lse, e = ex2_approx(ln_to_2(lp));
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
