// Rotary positions for sm_100a: queries and keys of a step, a prompt or a training batch, turned by the angles of their
// positions in one launch.  A pair (a, b) of a head - neighbours (2i, 2i+1), or (i, i + rotary/2) in the half layout -
// becomes (a c - b s, a s + b c); what lies behind the rotated part is copied.  The gradient is the same with -s.  Cosines and
// sines come from fp32 tables (angles of far positions need 64 bits, rotary.py), products are rounded one by one as torch's are.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx_sm100.cuh"

namespace tsp {

struct RotateSide {                        // queries or keys
    const void* x;
    void* y;                               // contiguous [B][T][heads][D]
    long long sb, st, sh;                  // elements between two sequences, tokens, heads of x
    int heads;
};

struct RotateParams {
    RotateSide q, k;                       // k.heads may be 0
    const float *cos_tab, *sin_tab;        // [table_len][rotary / 2]
    const long long* pos;
    long long pos_sb, pos_st;
    long long tokens_all;                  // batch * tokens
    int tokens, dim, rotary, table_len;
    float sign;                            // of the sines
    int* status;
};

__device__ __forceinline__ float rot_a(float a, float b, float c, float s) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)); }
__device__ __forceinline__ float rot_b(float a, float b, float c, float s) { return __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c)); }

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Elem<float> {
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec { T v[N]; };

// A thread takes one unit of a token - V pairs of the half layout, V / 2 of the other, or V copied values - in HEADS heads, so that
// cosines and sines are read once for all of them.
template <typename T, int V, bool HALF, int HEADS>
__global__ void __launch_bounds__(256) rotate_kernel(const RotateParams p, int units, int head_groups, long long items) {
    using VT = Vec<T, V>;
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    if (item >= items) return;
    const int u = (int)(item % units);
    const long long r = item / units;
    const int hg = (int)(r % head_groups);
    const long long bt = r / head_groups, b = bt / p.tokens, t = bt - b * p.tokens;
    const int half = p.rotary / 2, turned = HALF ? half / V : p.rotary / V;
    constexpr int PAIRS = HALF ? V : (V > 1 ? V / 2 : 1);
    const bool copies = u >= turned;
    const int e = HALF && copies ? p.rotary + (u - turned) * V : u * V;   // first element
    float c[PAIRS], s[PAIRS];
    if (!copies) {
        const long long pos = p.pos[b * p.pos_sb + t * p.pos_st];
        const bool ok = pos >= 0 && pos < p.table_len;
        const long long row = (ok ? pos : 0) * half + (HALF ? e : e / 2);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) c[i] = p.cos_tab[row + i], s[i] = p.sign * p.sin_tab[row + i];
        if (!ok) {                                                 // a position outside of the table
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
            *p.status = 1;
        }
    }
    VT x[HEADS], y[HEADS];
    const T* src[HEADS];
    T* dst[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = hg * HEADS + i;
        const bool is_q = h < p.q.heads;
        const RotateSide& sd = is_q ? p.q : p.k;
        const int hh = is_q ? h : h - p.q.heads;
        src[i] = hh < sd.heads ? static_cast<const T*>(sd.x) + b * sd.sb + t * sd.st + hh * sd.sh + e : nullptr;
        dst[i] = static_cast<T*>(sd.y) + (bt * sd.heads + hh) * p.dim + e;
        if (!src[i]) continue;
        x[i] = *reinterpret_cast<const VT*>(src[i]);
        if (HALF && !copies) y[i] = *reinterpret_cast<const VT*>(src[i] + half);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        if (!src[i]) continue;
        if (!copies) {
            if (HALF) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float a = Elem<T>::get(x[i].v[j]), bb = Elem<T>::get(y[i].v[j]);
                    x[i].v[j] = Elem<T>::put(rot_a(a, bb, c[j], s[j])), y[i].v[j] = Elem<T>::put(rot_b(a, bb, c[j], s[j]));
                }
                *reinterpret_cast<VT*>(dst[i] + half) = y[i];
            } else {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float a = Elem<T>::get(x[i].v[2 * j]), bb = Elem<T>::get(x[i].v[2 * j + 1]);
                    x[i].v[2 * j] = Elem<T>::put(rot_a(a, bb, c[j], s[j])), x[i].v[2 * j + 1] = Elem<T>::put(rot_b(a, bb, c[j], s[j]));
                }
            }
        }
        *reinterpret_cast<VT*>(dst[i]) = x[i];
    }
}

}  // namespace tsp
