// Rotary positions for sm_100a: queries and keys of a step, a prompt or a training batch, turned by the angles of their
// positions in one launch.  A pair (a, b) of a head - neighbours (2i, 2i+1), or (i, i + rotary/2) in the half layout -
// becomes (a c - b s, a s + b c); what lies behind the rotated part is copied.  The gradient is the same with -s.  Cosines and
// sines come from fp32 tables (angles of far positions need 64 bits, rotary.py), products are rounded one by one as torch's are.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx_sm100.cuh"

namespace tsp {

// Division of 0 <= n < 2^31 by a number that the launch knows.
struct FastDiv {
    uint32_t d = 1, mul = 1, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t by) : d(by) {
        while (shift < 31 && (1u << shift) < d) ++shift;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
    __device__ __forceinline__ uint32_t div(uint32_t n, uint32_t& rest) const {
        const uint32_t q = div(n);
        rest = n - q * d;
        return q;
    }
};

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
    FastDiv units, head_groups, tokens;
    int dim, rotary, table_len;
    int tables_16;                         // whether every table row starts on 16 bytes
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

// N consecutive values of a table row.
template <int N>
__device__ __forceinline__ void table_values(const float* t, int by_16, float (&x)[N]) {
    if (N % 4 == 0 && by_16) {
#pragma unroll
        for (int i = 0; i + 3 < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(t + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = t[i];
    }
}

// A thread takes one unit of a token - V pairs of the half layout, V / 2 of the other, or V copied values - in HEADS heads, so that
// cosines and sines are read once for all of them.  Memory is the bound: what matters is that all loads of a thread are on their way
// before the first is used, and that the index arithmetic (divisions by multiplication, 32 bits) stays small beside them.  Two prompts of 2,048
// tokens, 64 + 8 heads of 128 in bf16, half layout: 37.7 us, 4.06 TB/s of 6.46 (51 us with a head per thread and divisions); 8 single tokens 1.9 us.
template <typename T, int V, bool HALF, int HEADS>
__global__ void __launch_bounds__(256, 4) rotate_kernel(const RotateParams p, uint32_t items) {
    using VT = Vec<T, V>;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x;
    if (item >= items) return;
    uint32_t u, hg, t;
    const uint32_t bt = p.head_groups.div(p.units.div(item, u), hg), b = p.tokens.div(bt, t);
    const int half = p.rotary / 2, turned = HALF ? half / V : p.rotary / V;
    constexpr int PAIRS = HALF ? V : (V > 1 ? V / 2 : 1);
    const bool copies = (int)u >= turned;
    const int e = HALF && copies ? p.rotary + ((int)u - turned) * V : (int)u * V;   // first element
    VT x[HEADS], y[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = (int)hg * HEADS + i, hk = h - p.q.heads;
        const RotateSide& sd = hk < 0 ? p.q : p.k;
        const int hh = hk < 0 ? h : hk;
        if (hh >= sd.heads) continue;
        const T* src = static_cast<const T*>(sd.x) + (long long)b * sd.sb + (long long)t * sd.st + (long long)hh * sd.sh + e;
        x[i] = *reinterpret_cast<const VT*>(src);
        if (HALF && !copies) y[i] = *reinterpret_cast<const VT*>(src + half);
    }
    float c[PAIRS], s[PAIRS];
    if (!copies) {
        const long long pos = p.pos[b * p.pos_sb + t * p.pos_st];
        const bool ok = pos >= 0 && pos < p.table_len;
        const long long row = (ok ? pos : 0) * half + (HALF ? e : e / 2);
        table_values(p.cos_tab + row, p.tables_16, c);
        table_values(p.sin_tab + row, p.tables_16, s);
        if (!ok) *p.status = 1;                                    // a position outside of the table
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) c[i] = ok ? c[i] : __int_as_float(0x7fffffff), s[i] *= p.sign;
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int h = (int)hg * HEADS + i, hk = h - p.q.heads;
        const RotateSide& sd = hk < 0 ? p.q : p.k;
        const int hh = hk < 0 ? h : hk;
        if (hh >= sd.heads) continue;
        T* dst = static_cast<T*>(sd.y) + ((long long)bt * sd.heads + hh) * p.dim + e;
        if (!copies) {
            if (HALF) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float a = Elem<T>::get(x[i].v[j]), bb = Elem<T>::get(y[i].v[j]);
                    x[i].v[j] = Elem<T>::put(rot_a(a, bb, c[j], s[j])), y[i].v[j] = Elem<T>::put(rot_b(a, bb, c[j], s[j]));
                }
                *reinterpret_cast<VT*>(dst + half) = y[i];
            } else {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) {
                    const float a = Elem<T>::get(x[i].v[2 * j]), bb = Elem<T>::get(x[i].v[2 * j + 1]);
                    x[i].v[2 * j] = Elem<T>::put(rot_a(a, bb, c[j], s[j])), x[i].v[2 * j + 1] = Elem<T>::put(rot_b(a, bb, c[j], s[j]));
                }
            }
        }
        *reinterpret_cast<VT*>(dst) = x[i];
    }
}

}  // namespace tsp
