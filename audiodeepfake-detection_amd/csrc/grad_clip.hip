// Global norm of a list of tensors, and the scaling of gradients to a largest norm.
//
//   norm = sqrt(sum_k sum_i t_k[i]^2)  (or the largest |t_k[i]|),   factor = min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: one read for the norm, one read and one write for the scaling.  The tensors of a call go to the kernels as
// tables of (pointer, length) in the argument block, cut into pieces of 16 Ki elements, one workgroup per piece, so a list
// of many small tensors is one launch and a large one is spread over the card.  Squares are summed in 64 bits: a square
// of an fp32 or bf16 gradient can leave the range of 32 bits either way.  Every piece has a slot of its own for its sum and
// one workgroup adds the slots in order: the same bits every time.
// Measured on 200 bf16 tensors of 300 M elements together: norm 132 us in two launches (4.5 TB/s), scaling 215 us in three
// (5.6 TB/s).  On 48 small tensors the kernels take 14 us of a call's 70, the rest is the host's.
// The scaling pass walks the tensors from the last piece to the first, so it starts on what the norm pass read last, which
// the 256 MB memory-side cache still holds.
#include "seq_common.h"

#include <cmath>

namespace {

using namespace afd;

constexpr int kT = 256;
constexpr int kPiece = 16384;  // elements per workgroup
constexpr int kNormTable = 128, kScaleTable = 96;

struct NormTable {
    const void* src[kNormTable];
    long count[kNormTable];
    int first[kNormTable + 1];  // first piece of tensor k; first[n] = pieces of the launch
    unsigned char dtype[kNormTable];
    int n;
};
struct ScaleTable {
    const void* src[kScaleTable];
    void* dst[kScaleTable];
    long count[kScaleTable];
    int first[kScaleTable + 1];
    unsigned char dtype[kScaleTable];
    int n;
};

// the tensor a piece belongs to: binary search in `first` (uniform over the workgroup)
template <typename Table> __device__ __forceinline__ int owner(const Table& t, int piece) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= piece) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// NaN stays: fmax would drop it.
__device__ __forceinline__ double larger(double a, double b) { return (a > b || a != a) ? a : b; }

template <typename T, bool MAX> __device__ double piece_sum(const T* p, int n) {
    constexpr int V = 16 / (int)sizeof(T);
    double acc[4] = {0, 0, 0, 0};
    auto add = [&](double& s, T v) {
        const double d = (double)to_f32(v);
        if constexpr (MAX) s = larger(fabs(d), s);
        else s = fma(d, d, s);
    };
    int head = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
    head = head < n ? head : n;
    if ((int)threadIdx.x < head) add(acc[0], p[threadIdx.x]);
    const int nv = (n - head) / V;
    const u32x4* q = reinterpret_cast<const u32x4*>(p + head);
    int i = threadIdx.x;
    for (; i + 3 * kT < nv; i += 4 * kT) {
        u32x4 r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) r[u] = q[i + u * kT];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            struct { T v[V]; } k = __builtin_bit_cast(decltype(k), r[u]);
#pragma unroll
            for (int j = 0; j < V; ++j) add(acc[j & 3], k.v[j]);
        }
    }
    for (; i < nv; i += kT) {
        const u32x4 r = q[i];
        struct { T v[V]; } k = __builtin_bit_cast(decltype(k), r);
#pragma unroll
        for (int j = 0; j < V; ++j) add(acc[j & 3], k.v[j]);
    }
    const int done = head + nv * V;
    if (done + (int)threadIdx.x < n) add(acc[0], p[done + threadIdx.x]);
    if constexpr (MAX) return larger(larger(acc[0], acc[1]), larger(acc[2], acc[3]));
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// sum (or maximum) over the workgroup, in thread 0
template <bool MAX> __device__ double block_sum(double v) {
    __shared__ double lds[kT / 64];
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const double o = __shfl_xor(v, m);
        v = MAX ? larger(v, o) : v + o;
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < kT / 64; ++i) v = MAX ? larger(v, lds[i]) : v + lds[i];
    return v;
}

template <bool MAX>
__global__ void __launch_bounds__(kT) norm_pieces_kernel(const NormTable t, double* __restrict__ part) {
    const int piece = blockIdx.x, k = owner(t, piece);
    const long at = (long)(piece - t.first[k]) * kPiece;
    const long left = t.count[k] - at;
    const int n = left < kPiece ? (int)left : kPiece;
    double v;
    if (t.dtype[k] == AFD_T_F32) v = piece_sum<float, MAX>(static_cast<const float*>(t.src[k]) + at, n);
    else if (t.dtype[k] == AFD_T_BF16) v = piece_sum<bf16_t, MAX>(static_cast<const bf16_t*>(t.src[k]) + at, n);
    else v = piece_sum<f16_t, MAX>(static_cast<const f16_t*>(t.src[k]) + at, n);
    v = block_sum<MAX>(v);
    if (threadIdx.x == 0) part[piece] = v;
}

// out[0] = norm, out[1] = factor (times `scale`, by which the gradients are still to be multiplied)
template <bool MAX>
__global__ void __launch_bounds__(kT) norm_finish_kernel(const double* __restrict__ part, long n, float max_norm, float scale,
                                                         float* __restrict__ out) {
    double a[4] = {0, 0, 0, 0};
    long i = threadIdx.x;
    for (; i + 3 * kT < n; i += 4 * kT) {
#pragma unroll
        for (int u = 0; u < 4; ++u) a[u] = MAX ? larger(a[u], part[i + u * kT]) : a[u] + part[i + u * kT];
    }
    for (; i < n; i += kT) a[0] = MAX ? larger(a[0], part[i]) : a[0] + part[i];
    double v = MAX ? larger(larger(a[0], a[1]), larger(a[2], a[3])) : (a[0] + a[1]) + (a[2] + a[3]);
    v = block_sum<MAX>(v);
    if (threadIdx.x == 0) {
        const double norm = (MAX ? v : sqrt(v)) * (double)fabsf(scale);
        out[0] = (float)norm;
        const double f = (double)max_norm / (norm + 1e-6);
        out[1] = scale * (float)(f > 1.0 ? 1.0 : f);  // (NaN stays NaN)
    }
}

// 16 bytes at a time, on the destination's 16-byte boundaries (the source may lie anywhere: gradients go into an arena, one
// behind the other; element by element such a pair ran at 3.0 TB/s).
template <typename T> __device__ void piece_scale(const T* p, T* o, int n, float f) {
    constexpr int V = 16 / (int)sizeof(T);
    int head = (int)(((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / sizeof(T));
    head = head < n ? head : n;
    if ((int)threadIdx.x < head) o[threadIdx.x] = from_f32<T>(to_f32(p[threadIdx.x]) * f);
    const int nv = (n - head) / V;
    const T* q = p + head;
    u32x4* w = reinterpret_cast<u32x4*>(o + head);
    auto get = [&](int i) { return (u32x4)*reinterpret_cast<const u32x4_any*>(q + (size_t)i * V); };
    auto one = [&](u32x4 r) {
        Pack<T, V> k = __builtin_bit_cast(Pack<T, V>, r);
#pragma unroll
        for (int j = 0; j < V; ++j) k.v[j] = from_f32<T>(to_f32(k.v[j]) * f);
        return __builtin_bit_cast(u32x4, k);
    };
    int i = threadIdx.x;
    for (; i + 3 * kT < nv; i += 4 * kT) {
        u32x4 r[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) r[u] = get(i + u * kT);
#pragma unroll
        for (int u = 0; u < 4; ++u) w[i + u * kT] = one(r[u]);
    }
    for (; i < nv; i += kT) w[i] = one(get(i));
    const int done = head + nv * V;
    if (done + (int)threadIdx.x < n) o[done + threadIdx.x] = from_f32<T>(to_f32(p[done + threadIdx.x]) * f);
}

__global__ void __launch_bounds__(kT) scale_pieces_kernel(const ScaleTable t, const float* __restrict__ stats) {
    const int piece = t.first[t.n] - 1 - (int)blockIdx.x, k = owner(t, piece);
    const float f = stats[1];
    if (f == 1.f && t.src[k] == t.dst[k]) return;  // in place and nothing to clip
    const long at = (long)(piece - t.first[k]) * kPiece;
    const long left = t.count[k] - at;
    const int n = left < kPiece ? (int)left : kPiece;
    if (t.dtype[k] == AFD_T_F32)
        piece_scale(static_cast<const float*>(t.src[k]) + at, static_cast<float*>(t.dst[k]) + at, n, f);
    else if (t.dtype[k] == AFD_T_BF16)
        piece_scale(static_cast<const bf16_t*>(t.src[k]) + at, static_cast<bf16_t*>(t.dst[k]) + at, n, f);
    else
        piece_scale(static_cast<const f16_t*>(t.src[k]) + at, static_cast<f16_t*>(t.dst[k]) + at, n, f);
}

long pieces(long n) { return (n + kPiece - 1) / kPiece; }

int check(const char* what, const void* const* src, const long* counts, const int* dtypes, int n) {
    if (n < 0 || (n > 0 && (!src || !counts || !dtypes))) return fail(AFD_ERR_ARG, "%s: bad argument", what);
    long total = 0;
    for (int k = 0; k < n; ++k) {
        if (counts[k] < 0 || (counts[k] > 0 && !src[k]) || !dtype_ok(dtypes[k]))
            return fail(AFD_ERR_ARG, "%s: tensor %d: count %ld, dtype %d", what, k, counts[k], dtypes[k]);
        total += pieces(counts[k]);
        if (total > 0x7fffffffL) return fail(AFD_ERR_UNSUPPORTED, "%s: too many elements", what);
    }
    return AFD_OK;
}

}  // namespace

extern "C" size_t afd_global_norm_workspace_bytes(const long* counts, int n) {
    long total = 0;
    for (int k = 0; k < n; ++k) total += counts[k] > 0 ? pieces(counts[k]) : 0;
    return (size_t)(total > 0 ? total : 1) * sizeof(double);
}

extern "C" int afd_global_norm(const void* const* src, const long* counts, const int* dtypes, int n, int maximum,
                               float max_norm, float scale, float* stats, void* ws, size_t ws_bytes, afd_stream_t stream) {
    if (!stats) return fail(AFD_ERR_ARG, "global norm: no output");
    if (int rc = check("global norm", src, counts, dtypes, n)) return rc;
    if (!ws || ws_bytes < afd_global_norm_workspace_bytes(counts, n))
        return fail(AFD_ERR_WORKSPACE, "global norm: workspace of %zu bytes is too small", ws_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    double bytes = 0.0;
    for (int k = 0; k < n; ++k) bytes += (double)counts[k] * dtype_bytes(dtypes[k]);
    ScopedBytes timing(AFD_K_SEQUENCE, bytes, s);
    double* part = static_cast<double*>(ws);
    long done = 0;
    for (int k = 0; k < n;) {
        NormTable t{};
        int at = 0;
        while (k < n && t.n < kNormTable) {
            if (counts[k] > 0) {
                t.src[t.n] = src[k];
                t.count[t.n] = counts[k];
                t.dtype[t.n] = (unsigned char)dtypes[k];
                t.first[t.n] = at;
                at += (int)pieces(counts[k]);
                ++t.n;
            }
            ++k;
        }
        t.first[t.n] = at;
        if (at == 0) continue;
        if (maximum) hipLaunchKernelGGL(norm_pieces_kernel<true>, dim3((unsigned)at), dim3(kT), 0, s, t, part + done);
        else hipLaunchKernelGGL(norm_pieces_kernel<false>, dim3((unsigned)at), dim3(kT), 0, s, t, part + done);
        done += at;
    }
    if (maximum) hipLaunchKernelGGL(norm_finish_kernel<true>, dim3(1), dim3(kT), 0, s, part, done, max_norm, scale, stats);
    else hipLaunchKernelGGL(norm_finish_kernel<false>, dim3(1), dim3(kT), 0, s, part, done, max_norm, scale, stats);
    return check_launch("global norm");
}

extern "C" int afd_multi_scale(const void* const* src, void* const* dst, const long* counts, const int* dtypes, int n,
                               const float* stats, afd_stream_t stream) {
    if (!stats || (n > 0 && !dst)) return fail(AFD_ERR_ARG, "multi scale: bad argument");
    if (int rc = check("multi scale", src, counts, dtypes, n)) return rc;
    for (int k = 0; k < n; ++k)
        if (counts[k] > 0 && !dst[k]) return fail(AFD_ERR_ARG, "multi scale: tensor %d has no destination", k);
    hipStream_t s = static_cast<hipStream_t>(stream);
    double bytes = 0.0;
    for (int k = 0; k < n; ++k) bytes += 2.0 * (double)counts[k] * dtype_bytes(dtypes[k]);
    ScopedBytes timing(AFD_K_SEQUENCE, bytes, s);
    for (int k = n; k > 0;) {  // from the last tensor to the first, as inside a launch
        ScaleTable t{};
        int lo = k;
        while (lo > 0 && k - lo < kScaleTable) --lo;
        int at = 0;
        for (int i = lo; i < k; ++i) {
            if (counts[i] <= 0) continue;
            t.src[t.n] = src[i];
            t.dst[t.n] = dst[i];
            t.count[t.n] = counts[i];
            t.dtype[t.n] = (unsigned char)dtypes[i];
            t.first[t.n] = at;
            at += (int)pieces(counts[i]);
            ++t.n;
        }
        t.first[t.n] = at;
        k = lo;
        if (at > 0) hipLaunchKernelGGL(scale_pieces_kernel, dim3((unsigned)at), dim3(kT), 0, s, t, stats);
    }
    return check_launch("multi scale");
}
