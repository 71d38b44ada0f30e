// Short causal depthwise convolution over [batch, time, channels] tensors, with SiLU in its epilogue: forward, backward
// and the single-token form.
//
//   z[t][c] = bias[c] + sum_j w[c][j] x[t - (W - 1) + j][c],    y = z  or  z sigmoid(z)
//
// Rows before the first are the `state` (the last W - 1 rows of an earlier part, oldest first) or zero.  Bound by memory:
// 2 W + 6 flops against one element read and one written, so every element is loaded once: a thread owns V neighbouring
// channels (16 bytes where alignment allows, so a wave's load is one 1 KB run of a row) and walks over consecutive rows with
// the W taps' window in registers; rows are loaded several at a time ahead of the window.
#include "seq_common.h"

namespace {

constexpr int kT = 256;
constexpr int kMaxW = 8;

struct ConvArgs {
    const void* x;
    long xb, xl;  // batch / row strides of x in elements (channels are contiguous)
    const void* w;
    const void* bias;  // NULL: none
    int w_f32;         // taps and bias are fp32 whatever T is (else T)
    const void* state;
    const int* lengths;
    void* y;
    void* state_out;
    int B, L, D, act;
    int tile, ntiles, groups;  // rows per thread, row tiles, channel groups of V
    // backward only
    const void* dy;
    long dyb, dyl;
    const void* dstate_out;
    void* dx;
    void* dstate;
    float* part;  // [B * ntiles][D * W + D]
};

template <typename T, int V> struct Pack { T v[V]; };

template <typename T, int V> __device__ __forceinline__ void load_row(const T* p, float (&r)[V]) {
    if constexpr (V == 1) {
        r[0] = afd::to_f32(*p);
    } else {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 raw = *reinterpret_cast<const u32x4*>(p);
        const Pack<T, V> k = __builtin_bit_cast(Pack<T, V>, raw);
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = afd::to_f32(k.v[i]);
    }
}

template <typename T, int V> __device__ __forceinline__ void store_row(T* p, const float (&r)[V]) {
    if constexpr (V == 1) {
        *p = afd::from_f32<T>(r[0]);
    } else {
        typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
        Pack<T, V> k;
#pragma unroll
        for (int i = 0; i < V; ++i) k.v[i] = afd::from_f32<T>(r[i]);
        *reinterpret_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, k);
    }
}

template <typename T> __device__ __forceinline__ float param(const void* p, size_t i, int f32) {
    return f32 ? static_cast<const float*>(p)[i] : afd::to_f32(static_cast<const T*>(p)[i]);
}

__device__ __forceinline__ int row_count(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > L ? L : n);
}

// Row t of the padded sequence: x for 0 <= t < n, the state for t < 0, zero elsewhere.
template <typename T, int W, int V>
__device__ __forceinline__ void padded_row(const ConvArgs& p, const T* x, int b, int c, int t, int n, float (&r)[V]) {
    if (t >= 0 && t < n) {
        load_row<T, V>(x + (size_t)t * p.xl, r);
    } else if (t < 0 && p.state) {
        load_row<T, V>(static_cast<const T*>(p.state) + ((size_t)b * (W - 1) + (t + W - 1)) * p.D + c, r);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = 0.f;
    }
}

template <typename T, int W, int V>
__device__ __forceinline__ void load_taps(const ConvArgs& p, int c, float (&w)[V][W], float (&bias)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = p.bias ? param<T>(p.bias, c + i, p.w_f32) : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = param<T>(p.w, (size_t)(c + i) * W + j, p.w_f32);
    }
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(kT) conv_fwd_kernel(const ConvArgs p) {
    const size_t id = (size_t)blockIdx.x * kT + threadIdx.x;
    const size_t per_b = (size_t)p.ntiles * p.groups;
    if (id >= per_b * p.B) return;
    const int b = (int)(id / per_b);
    const int rest = (int)(id - b * per_b);
    const int tile = rest / p.groups;
    const int c = (rest - tile * p.groups) * V;
    const int n = row_count(p.lengths, b, p.L);
    const T* x = static_cast<const T*>(p.x) + (size_t)b * p.xb + c;
    T* y = static_cast<T*>(p.y) + (size_t)b * p.L * p.D + c;
    const int t0 = tile * p.tile, t1 = min(t0 + p.tile, p.L);
    // the tile that holds row 0 (the only one there is when L = 0 is refused) also leaves the state behind row n
    if (p.state_out && tile == 0) {
        T* so = static_cast<T*>(p.state_out) + (size_t)b * (W - 1) * p.D + c;
        for (int k = 0; k < W - 1; ++k) {
            float r[V];
            padded_row<T, W, V>(p, x, b, c, n - (W - 1) + k, n, r);
            store_row<T, V>(so + (size_t)k * p.D, r);
        }
    }
    float zero[V];
#pragma unroll
    for (int i = 0; i < V; ++i) zero[i] = 0.f;
    int t = t0;
    if (t < n) {
        float w[V][W], bias[V], win[W][V];
        load_taps<T, W, V>(p, c, w, bias);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) padded_row<T, W, V>(p, x, b, c, t0 - (W - 1) + j, n, win[j]);
        constexpr int U = 8;
        const int tn = min(t1, n);
        for (; t < tn; t += U) {
            float in[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u < tn) load_row<T, V>(x + (size_t)(t + u) * p.xl, in[u]);
                else {
#pragma unroll
                    for (int i = 0; i < V; ++i) in[u][i] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u < tn) {
                    float z[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        win[W - 1][i] = in[u][i];
                        z[i] = bias[i];
#pragma unroll
                        for (int j = 0; j < W; ++j) z[i] = fmaf(w[i][j], win[j][i], z[i]);
                        if (p.act) z[i] *= afd::sigmoid_f32(z[i]);
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
                    }
                    store_row<T, V>(y + (size_t)(t + u) * p.D, z);
                }
            }
        }
        t = tn;
    }
    for (; t < t1; ++t) store_row<T, V>(y + (size_t)t * p.D, zero);
}

// Backward.  A thread walks over its rows [t0, t1) once: dz[t] = dy[t] act'(z[t]) from the x window, and with the last W
// values of dz in a second window the gradient of row t - (W - 1) is complete.  It starts at t0 (the rows before t0 get
// the rest of their gradient from the neighbour, which walks W - 1 rows past its end for that), so x and dy are read once
// but for W - 1 rows per tile.  dw and dbias are summed in registers over the tile and leave as one partial row.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kT) conv_bwd_kernel(const ConvArgs p) {
    const size_t id = (size_t)blockIdx.x * kT + threadIdx.x;
    const size_t per_b = (size_t)p.ntiles * p.groups;
    if (id >= per_b * p.B) return;
    const int b = (int)(id / per_b);
    const int rest = (int)(id - b * per_b);
    const int tile = rest / p.groups;
    const int c = (rest - tile * p.groups) * V;
    const int n = row_count(p.lengths, b, p.L);
    const T* x = static_cast<const T*>(p.x) + (size_t)b * p.xb + c;
    const T* dy = static_cast<const T*>(p.dy) + (size_t)b * p.dyb + c;
    const int t0 = tile * p.tile, t1 = min(t0 + p.tile, p.L);
    float w[V][W], bias[V], win[W][V], dzw[W][V], dw[V][W], db[V];
    load_taps<T, W, V>(p, c, w, bias);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        db[i] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) dw[i][j] = dzw[j][i] = 0.f;
    }
    // positions whose gradient this thread owns: its rows, and for the first tile the W - 1 rows of the state
    const int first = tile == 0 ? -(W - 1) : t0;
    if (t0 < n || tile == 0) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) padded_row<T, W, V>(p, x, b, c, t0 - (W - 1) + j, n, win[j]);
        constexpr int U = 4;
        for (int t = t0; t < t1 + W - 1; t += U) {
            float in[U][V], g[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool live = t + u < n && t + u < t1 + W - 1;
                if (live) {
                    load_row<T, V>(x + (size_t)(t + u) * p.xl, in[u]);
                    load_row<T, V>(dy + (size_t)(t + u) * p.dyl, g[u]);
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) in[u][i] = g[u][i] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (t + u < t1 + W - 1) {
                    const bool live = t + u < n, own = t + u < t1;
                    float out[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        win[W - 1][i] = in[u][i];
                        float dz = g[u][i];
                        if (p.act) {
                            float z = bias[i];
#pragma unroll
                            for (int j = 0; j < W; ++j) z = fmaf(w[i][j], win[j][i], z);
                            const float s = afd::sigmoid_f32(z);
                            dz *= s * (1.f + z * (1.f - s));
                        }
                        dz = live ? dz : 0.f;
                        if (own) {
                            db[i] += dz;
#pragma unroll
                            for (int j = 0; j < W; ++j) dw[i][j] = fmaf(dz, win[j][i], dw[i][j]);
                        }
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) {
                            win[j][i] = win[j + 1][i];
                            dzw[j][i] = dzw[j + 1][i];
                        }
                        dzw[W - 1][i] = dz;
                        // position q = t + u - (W - 1) feeds dz[q + W - 1 - j] through tap j
                        out[i] = 0.f;
#pragma unroll
                        for (int j = 0; j < W; ++j) out[i] = fmaf(w[i][j], dzw[W - 1 - j][i], out[i]);
                    }
                    const int q = t + u - (W - 1);
                    if (q >= first && q < t1) {
                        if (p.dstate_out && q < n && q >= n - (W - 1)) {
                            float e[V];
                            load_row<T, V>(static_cast<const T*>(p.dstate_out) +
                                               ((size_t)b * (W - 1) + (q - n + W - 1)) * p.D + c, e);
#pragma unroll
                            for (int i = 0; i < V; ++i) out[i] += e[i];
                        }
                        if (q >= 0) {
                            store_row<T, V>(static_cast<T*>(p.dx) + ((size_t)b * p.L + q) * p.D + c, out);
                        } else if (p.dstate) {
                            store_row<T, V>(static_cast<T*>(p.dstate) + ((size_t)b * (W - 1) + q + W - 1) * p.D + c, out);
                        }
                    }
                }
            }
        }
    } else {
        float zero[V];
#pragma unroll
        for (int i = 0; i < V; ++i) zero[i] = 0.f;
        for (int t = t0; t < t1; ++t) store_row<T, V>(static_cast<T*>(p.dx) + ((size_t)b * p.L + t) * p.D + c, zero);
    }
    float* row = p.part + (size_t)(b * p.ntiles + tile) * ((size_t)p.D * (W + 1));
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) row[(size_t)(c + i) * W + j] = dw[i][j];
        row[(size_t)p.D * W + c + i] = db[i];
    }
}

// One token: a thread reads the W - 1 state rows of its channels before it writes any, so state_out may be the state.
template <typename T, int W, int V>
__global__ void __launch_bounds__(kT) conv_step_kernel(const ConvArgs p) {
    const size_t id = (size_t)blockIdx.x * kT + threadIdx.x;
    if (id >= (size_t)p.B * p.groups) return;
    const int b = (int)(id / p.groups);
    const int c = (int)(id - (size_t)b * p.groups) * V;
    const T* st = static_cast<const T*>(p.state) + (size_t)b * (W - 1) * p.D + c;
    T* so = static_cast<T*>(p.state_out) + (size_t)b * (W - 1) * p.D + c;
    float w[V][W], bias[V], win[W][V];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) load_row<T, V>(st + (size_t)j * p.D, win[j]);
    load_row<T, V>(static_cast<const T*>(p.x) + (size_t)b * p.xb + c, win[W - 1]);
    load_taps<T, W, V>(p, c, w, bias);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        z[i] = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) z[i] = fmaf(w[i][j], win[j][i], z[i]);
        if (p.act) z[i] *= afd::sigmoid_f32(z[i]);
    }
    store_row<T, V>(static_cast<T*>(p.y) + (size_t)b * p.D + c, z);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<T, V>(so + (size_t)j * p.D, win[j + 1]);
}

enum Kind { kFwd, kBwd, kStep };

template <typename T, int W, int V> void launch_t(Kind kind, const ConvArgs& p, unsigned grid, hipStream_t s) {
    if (kind == kFwd) hipLaunchKernelGGL((conv_fwd_kernel<T, W, V>), dim3(grid), dim3(kT), 0, s, p);
    else if (kind == kBwd) hipLaunchKernelGGL((conv_bwd_kernel<T, W, V>), dim3(grid), dim3(kT), 0, s, p);
    else hipLaunchKernelGGL((conv_step_kernel<T, W, V>), dim3(grid), dim3(kT), 0, s, p);
}

template <typename T, int V> void launch_w(Kind kind, int W, const ConvArgs& p, unsigned grid, hipStream_t s) {
    switch (W) {
        case 2: return launch_t<T, 2, V>(kind, p, grid, s);
        case 3: return launch_t<T, 3, V>(kind, p, grid, s);
        case 4: return launch_t<T, 4, V>(kind, p, grid, s);
        case 5: return launch_t<T, 5, V>(kind, p, grid, s);
        case 6: return launch_t<T, 6, V>(kind, p, grid, s);
        case 7: return launch_t<T, 7, V>(kind, p, grid, s);
        default: return launch_t<T, 8, V>(kind, p, grid, s);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 16-byte accesses need every row of every tensor on a 16-byte boundary; single elements otherwise.
int vector_width(const ConvArgs& p, int dtype) {
    const int v = (int)(16 / afd::dtype_bytes(dtype));
    const bool ok = p.D % v == 0 && p.xb % v == 0 && p.xl % v == 0 && p.dyb % v == 0 && p.dyl % v == 0 && aligned16(p.x) &&
                    aligned16(p.y) && aligned16(p.state) && aligned16(p.state_out) && aligned16(p.dy) && aligned16(p.dx) &&
                    aligned16(p.dstate) && aligned16(p.dstate_out);
    return ok ? v : 1;
}

int run(Kind kind, ConvArgs& p, int W, int dtype, hipStream_t s) {
    const int v = vector_width(p, dtype);
    p.groups = (p.D + v - 1) / v;
    const size_t threads = (size_t)p.B * p.ntiles * p.groups;
    const size_t grid = (threads + kT - 1) / kT;
    if (grid > 0x7fffffffu) return afd::fail(AFD_ERR_UNSUPPORTED, "causal conv: %zu workgroups", grid);
    if (dtype == AFD_T_F32) {
        if (v > 1) launch_w<float, 4>(kind, W, p, (unsigned)grid, s);
        else launch_w<float, 1>(kind, W, p, (unsigned)grid, s);
    } else if (dtype == AFD_T_BF16) {
        if (v > 1) launch_w<afd::bf16_t, 8>(kind, W, p, (unsigned)grid, s);
        else launch_w<afd::bf16_t, 1>(kind, W, p, (unsigned)grid, s);
    } else {
        if (v > 1) launch_w<afd::f16_t, 8>(kind, W, p, (unsigned)grid, s);
        else launch_w<afd::f16_t, 1>(kind, W, p, (unsigned)grid, s);
    }
    return afd::check_launch("causal_conv kernel");
}

// Rows per thread.
constexpr int kFwdTile = 16, kBwdTile = 64;

int check(const char* what, int B, int L, int D, int W, int act, int dtype) {
    if (B < 1 || L < 1 || D < 1 || W < 2 || W > kMaxW || act < 0 || act > 1 || !afd::dtype_ok(dtype))
        return afd::fail(AFD_ERR_ARG, "%s: B=%d L=%d D=%d W=%d (2..%d) act=%d dtype=%d", what, B, L, D, W, kMaxW, act, dtype);
    if ((long)B * afd::ceil_div(L, kFwdTile) > 0x7fffffffL)
        return afd::fail(AFD_ERR_UNSUPPORTED, "%s: B=%d L=%d has too many row tiles", what, B, L);
    return AFD_OK;
}

}  // namespace

extern "C" int afd_causal_conv_forward(const void* x, long long xb, long long xl, const void* w, const void* bias, int w_f32,
                                       const void* state, const int* lengths, void* y, void* state_out, int B, int L, int D,
                                       int W, int act, int dtype, afd_stream_t stream) {
    if (!x || !w || !y) return afd::fail(AFD_ERR_ARG, "causal conv: missing tensor");
    if (int rc = check("causal conv", B, L, D, W, act, dtype)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ConvArgs p{};
    p.x = x; p.xb = xb; p.xl = xl; p.w = w; p.bias = bias; p.w_f32 = w_f32; p.state = state; p.lengths = lengths;
    p.y = y; p.state_out = state_out; p.B = B; p.L = L; p.D = D; p.act = act;
    p.tile = kFwdTile;
    p.ntiles = afd::ceil_div(L, p.tile);
    afd::ScopedBytes timing(AFD_K_SEQUENCE, 2.0 * afd::dtype_bytes(dtype) * B * L * D, s);
    return run(kFwd, p, W, dtype, s);
}

extern "C" size_t afd_causal_conv_backward_workspace_bytes(int B, int L, int D, int W) {
    return (size_t)B * afd::ceil_div(L, kBwdTile) * D * (W + 1) * sizeof(float);
}

extern "C" int afd_causal_conv_backward(const void* x, long long xb, long long xl, const void* w, const void* bias, int w_f32,
                                        const void* state, const int* lengths, const void* dy, long long dyb, long long dyl,
                                        const void* dstate_out, void* dx, void* dw, void* dbias, void* dstate, int B, int L,
                                        int D, int W, int act, int dtype, void* ws, size_t ws_bytes, afd_stream_t stream) {
    if (!x || !w || !dy || !dx || !dw) return afd::fail(AFD_ERR_ARG, "causal conv backward: missing tensor");
    if (int rc = check("causal conv backward", B, L, D, W, act, dtype)) return rc;
    if (!ws || ws_bytes < afd_causal_conv_backward_workspace_bytes(B, L, D, W))
        return afd::fail(AFD_ERR_WORKSPACE, "causal conv backward: workspace of %zu bytes is too small", ws_bytes);
    if ((long)D * (W + 1) > 0x7fffffc0L) return afd::fail(AFD_ERR_UNSUPPORTED, "causal conv backward: D=%d", D);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ConvArgs p{};
    p.x = x; p.xb = xb; p.xl = xl; p.w = w; p.bias = bias; p.w_f32 = w_f32; p.state = state; p.lengths = lengths;
    p.dy = dy; p.dyb = dyb; p.dyl = dyl; p.dstate_out = dstate_out; p.dx = dx; p.dstate = dstate;
    p.B = B; p.L = L; p.D = D; p.act = act;
    p.part = static_cast<float*>(ws);
    p.tile = kBwdTile;
    p.ntiles = afd::ceil_div(L, p.tile);
    afd::ScopedBytes timing(AFD_K_SEQUENCE, 3.0 * afd::dtype_bytes(dtype) * B * L * D, s);
    if (int rc = run(kBwd, p, W, dtype, s)) return rc;
    const int pt = w_f32 ? AFD_T_F32 : dtype;
    afd::ColumnOuts o{};
    o.n = 2;
    o.o[0] = {dw, 0, D * W, W, W, pt};
    o.o[1] = {dbias, D * W, D * W + D, 1, 1, pt};
    return afd::launch_column_sums(p.part, (long)B * p.ntiles, D * (W + 1), o, s);
}

extern "C" int afd_causal_conv_step(const void* x, long long xb, const void* w, const void* bias, int w_f32,
                                    const void* state, void* y, void* state_out, int B, int D, int W, int act, int dtype,
                                    afd_stream_t stream) {
    if (!x || !w || !y || !state || !state_out) return afd::fail(AFD_ERR_ARG, "causal conv step: missing tensor");
    if (int rc = check("causal conv step", B, 1, D, W, act, dtype)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ConvArgs p{};
    p.x = x; p.xb = xb; p.w = w; p.bias = bias; p.w_f32 = w_f32; p.state = state; p.y = y; p.state_out = state_out;
    p.B = B; p.L = 1; p.D = D; p.act = act; p.tile = 1; p.ntiles = 1;
    afd::ScopedBytes timing(AFD_K_SEQUENCE, 2.0 * afd::dtype_bytes(dtype) * B * D * W, s);
    return run(kStep, p, W, dtype, s);
}
