// Shared by the sequence-layer kernels (causal_conv.hip, state_scan*.hip, linear.hip, grad_clip.hip): element types, the
// non-linearities of the state-space layer and the column sums that end their parameter gradients.
#pragma once

#include "afd_common.h"
#include "../../include/afd_hip.h"

namespace afd {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }  // round to nearest even

constexpr long kMaxGroups = 0xffffff;  // workgroups of 256 threads: a launch holds less than 2^32 threads

inline size_t dtype_bytes(int dtype) { return dtype == AFD_T_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == AFD_T_F32 || dtype == AFD_T_BF16 || dtype == AFD_T_F16; }

constexpr float kLog2e = 1.44269504088896340736f;

// 1 / (1 + exp(-x)): the hardware's base-2 exponential and reciprocal, 1 ulp each, and the rounding of the exponent's product,
// 2^-24 |x| of the result for x << 0 (5e-6 at x = -80).  exp overflows to inf for x < -88 and the reciprocal of that is 0, which
// is the limit.
__device__ __forceinline__ float sigmoid_f32(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-kLog2e * x));
}

// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1].  The step widths of a state-space layer start at
// 1e-3 .. 1e-1, where log(1 + e) taken at face value has lost ten bits: log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, and
// 2 atanh(s) / s as a polynomial in s^2 on [0, 1/9], fitted for the least relative error (8e-9, an eighth of a rounding).
__device__ __forceinline__ float softplus_f32(float x) {
    const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.f + e);
    const float q = s * s;
    float p = 0.28178325f;
    p = fmaf(p, q, 0.27960604f);
    p = fmaf(p, q, 0.40024909f);
    p = fmaf(p, q, 0.66666317f);
    p = fmaf(p, q, 2.f);
    return fmaf(s, p, fmaxf(x, 0.f));  // (NaN comes in through e)
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes from or to any element's address: global memory takes them on every alignment, aligned ones fastest
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
template <typename T, int V> struct Pack { T v[V]; };

template <typename T, int V> __device__ __forceinline__ void load_row(const T* p, float (&r)[V]) {
    if constexpr (V == 1) {
        r[0] = to_f32(*p);
    } else {
        static_assert(V * sizeof(T) == 16 || V * sizeof(T) == 8, "vector rows");
        Pack<T, V> k;
        if constexpr (V * sizeof(T) == 16) k = __builtin_bit_cast(Pack<T, V>, (u32x4)*reinterpret_cast<const u32x4_any*>(p));
        else k = __builtin_bit_cast(Pack<T, V>, (u32x2)*reinterpret_cast<const u32x2_any*>(p));
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = to_f32(k.v[i]);
    }
}

template <typename T, int V> __device__ __forceinline__ void store_row(T* p, const float (&r)[V]) {
    if constexpr (V == 1) {
        *p = from_f32<T>(r[0]);
    } else {
        Pack<T, V> k;
#pragma unroll
        for (int i = 0; i < V; ++i) k.v[i] = from_f32<T>(r[i]);
        if constexpr (V * sizeof(T) == 16) *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, k);
        else *reinterpret_cast<u32x2_any*>(p) = __builtin_bit_cast(u32x2, k);
    }
}

// Sums of the columns of part[rows][cols]: each workgroup takes 64 columns, its 16 waves take every 16th row and meet in LDS.
// Column c goes to the output that owns it (fixed order: no atomics, the same bits every time).  The partial rows are
// written just before by the same stream: L2-resident in most cases, a tenth or less of the main kernel's bytes.
struct ColumnOut {
    void* out;        // NULL: dropped
    int begin, end;   // the columns [begin, end) of a row belong to this output
    int width, keep;  // inside it, column i = (g, j) = (i / width, i % width) is kept where j < keep
    int gs, js;       // ... and goes to g gs + j js
    int dtype;
};
struct ColumnOuts {
    ColumnOut o[4];
    int n;
};
int launch_column_sums(const float* part, long rows, int cols, const ColumnOuts& outs, hipStream_t s);

}  // namespace afd
