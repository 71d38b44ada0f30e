// Short causal depthwise convolution over [batch, time, channels] tensors, with SiLU in its epilogue: forward, backward
// and the single-token form.
//
//   z[t][c] = bias[c] + sum_j w[c][j] x[t - (W - 1) + j][c],    y = z  or  z sigmoid(z)
//
// Rows before the first are the `state` (the last W - 1 rows of an earlier part, oldest first) or zero.  Bound by memory:
// 2 W + 6 flops against one element read and one written, so every element is loaded once: a thread owns V neighbouring
// channels (16 bytes; 4 in the backward) and walks over consecutive rows with the W taps' window in registers; rows are
// loaded several at a time ahead of the window.  The taps come through LDS: 16-byte reads of [channel][tap] rows, one per
// lane, touched a cache line per lane and made up half of the line traffic.
// Measured at 4 x 4096 x 2048 bf16, 4 taps: forward 32 us (4.2 TB/s of what it has to move; a large copy runs at 4.9), backward
// 56 us (3.6 TB/s): every 32 rows the W - 1 behind them are walked again, 9 % of its bytes, and no loads are under way while a
// trip's rows are computed and stored.
#include "seq_common.h"

namespace {

using namespace afd;

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
    int tile, ntiles;  // rows per thread, row tiles
    int groups, gx;    // channel groups of V; groups per workgroup (8 .. 64; the other factor of 256 is tiles)
    int gblocks;       // workgroups over a row's groups
    // backward only
    const void* dy;
    long dyb, dyl;
    const void* dstate_out;
    void* dx;
    void* dstate;
    float* part;  // [B * ntiles][W + 1][D]: dw by tap, dbias
};

template <typename T> __device__ __forceinline__ float param(const void* p, size_t i, int f32) {
    return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const T*>(p)[i]);
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

// Where a thread works: channels c .. c + V of rows [t0, t1) of sequence b.  Where V does not divide D the last group is moved
// back to end with the row: its first channels are computed twice, with the same result.
struct Place {
    int b, tile, c, n, t0, t1, lane_group;
    bool live;
};
template <int V> __device__ __forceinline__ Place place(const ConvArgs& p) {
    Place w;
    w.lane_group = threadIdx.x & (p.gx - 1);
    const int gb = blockIdx.x % p.gblocks;
    const long rows = (long)(blockIdx.x / p.gblocks) * (kT / p.gx) + threadIdx.x / p.gx;
    const int g = gb * p.gx + w.lane_group;
    w.live = g < p.groups && rows < (long)p.B * p.ntiles;
    w.b = (int)(rows / p.ntiles);
    w.tile = (int)(rows - (long)w.b * p.ntiles);
    w.c = min(g * V, p.D - V);
    w.n = w.live ? row_count(p.lengths, w.b, p.L) : 0;
    w.t0 = w.tile * p.tile;
    w.t1 = min(w.t0 + p.tile, p.L);
    return w;
}

// The taps and biases of the workgroup's channels, through LDS: [tap i of V][tap j or bias][group].
template <typename T, int W, int V>
__device__ __forceinline__ void load_taps(const ConvArgs& p, const Place& q, float* lds, float (&w)[V][W], float (&bias)[V]) {
    const int g0 = (int)(blockIdx.x % p.gblocks) * p.gx, gn = min(p.gx, p.groups - g0);
    for (int e = threadIdx.x; e < gn * V * W; e += kT) {
        const int g = e / (V * W), r = e - g * (V * W);
        lds[((r / W) * (W + 1) + r % W) * p.gx + g] = param<T>(p.w, (size_t)min((g0 + g) * V, p.D - V) * W + r, p.w_f32);
    }
    for (int e = threadIdx.x; e < gn * V; e += kT) {
        const int g = e / V, i = e - g * V;
        lds[(i * (W + 1) + W) * p.gx + g] = p.bias ? param<T>(p.bias, min((g0 + g) * V, p.D - V) + i, p.w_f32) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = lds[(i * (W + 1) + j) * p.gx + q.lane_group];
        bias[i] = lds[(i * (W + 1) + W) * p.gx + q.lane_group];
    }
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(kT) conv_fwd_kernel(const ConvArgs p) {
    extern __shared__ float taps[];
    const Place q = place<V>(p);
    float w[V][W], bias[V], win[W][V];
    load_taps<T, W, V>(p, q, taps, w, bias);
    if (!q.live) return;
    const int b = q.b, c = q.c, n = q.n, t0 = q.t0, t1 = q.t1, tile = q.tile;
    const T* x = static_cast<const T*>(p.x) + (size_t)b * p.xb + c;
    T* y = static_cast<T*>(p.y) + (size_t)b * p.L * p.D + c;
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
#pragma unroll
        for (int j = 0; j < W - 1; ++j) padded_row<T, W, V>(p, x, b, c, t0 - (W - 1) + j, n, win[j]);
        constexpr int U = 4;
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
                float z[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    win[W - 1][i] = in[u][i];
                    z[i] = bias[i];
#pragma unroll
                    for (int j = 0; j < W; ++j) z[i] = fmaf(w[i][j], win[j][i], z[i]);
                    if (p.act) z[i] *= sigmoid_f32(z[i]);
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
                }
                if (t + u < tn) store_row<T, V>(y + (size_t)(t + u) * p.D, z);
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
    extern __shared__ float taps[];
    const Place q = place<V>(p);
    float w[V][W], bias[V], win[W][V], dzw[W][V], dw[V][W], db[V];
    load_taps<T, W, V>(p, q, taps, w, bias);
    if (!q.live) return;
    const int b = q.b, c = q.c, n = q.n, t0 = q.t0, t1 = q.t1, tile = q.tile;
    const T* x = static_cast<const T*>(p.x) + (size_t)b * p.xb + c;
    const T* dy = static_cast<const T*>(p.dy) + (size_t)b * p.dyb + c;
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
        constexpr int U = 2;
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
                // (steps behind the last row only move zeros: a condition around them would keep the windows from being
                // renamed instead of moved)
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
                        const float s = sigmoid_f32(z);
                        dz *= s * (1.f + z * (1.f - s));
                    }
                    dz = live ? dz : 0.f;
                    const float dzo = own ? dz : 0.f;
                    db[i] += dzo;
#pragma unroll
                    for (int j = 0; j < W; ++j) dw[i][j] = fmaf(dzo, win[j][i], dw[i][j]);
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) {
                        win[j][i] = win[j + 1][i];
                        dzw[j][i] = dzw[j + 1][i];
                    }
                    dzw[W - 1][i] = dz;
                    // position `at` = t + u - (W - 1) feeds dz[at + W - 1 - j] through tap j
                    out[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < W; ++j) out[i] = fmaf(w[i][j], dzw[W - 1 - j][i], out[i]);
                }
                const int at = t + u - (W - 1);
                if (at >= first && at < t1) {
                    if (p.dstate_out && at < n && at >= n - (W - 1)) {
                        float e[V];
                        load_row<T, V>(static_cast<const T*>(p.dstate_out) +
                                           ((size_t)b * (W - 1) + (at - n + W - 1)) * p.D + c, e);
#pragma unroll
                        for (int i = 0; i < V; ++i) out[i] += e[i];
                    }
                    if (at >= n) {  // (no product of zeros: a tap need not be finite)
#pragma unroll
                        for (int i = 0; i < V; ++i) out[i] = 0.f;
                    }
                    if (at >= 0) {
                        store_row<T, V>(static_cast<T*>(p.dx) + ((size_t)b * p.L + at) * p.D + c, out);
                    } else if (p.dstate) {
                        store_row<T, V>(static_cast<T*>(p.dstate) + ((size_t)b * (W - 1) + at + W - 1) * p.D + c, out);
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
    float* row = p.part + (size_t)(b * p.ntiles + tile) * ((size_t)p.D * (W + 1)) + c;
#pragma unroll
    for (int j = 0; j < W; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) row[(size_t)j * p.D + i] = dw[i][j];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) row[(size_t)W * p.D + i] = db[i];
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
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = p.bias ? param<T>(p.bias, c + i, p.w_f32) : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[i][j] = param<T>(p.w, (size_t)(c + i) * W + j, p.w_f32);
    }
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        z[i] = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) z[i] = fmaf(w[i][j], win[j][i], z[i]);
        if (p.act) z[i] *= sigmoid_f32(z[i]);
    }
    store_row<T, V>(static_cast<T*>(p.y) + (size_t)b * p.D + c, z);
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_row<T, V>(so + (size_t)j * p.D, win[j + 1]);
}

enum Kind { kFwd, kBwd, kStep };

template <typename T, int W, int V> void launch_t(Kind kind, const ConvArgs& p, unsigned grid, hipStream_t s) {
    const unsigned lds = (unsigned)(p.gx * V * (W + 1) * sizeof(float));
    constexpr bool kWide = V == 1 || V * sizeof(T) == 16;
    if constexpr (V <= 4)
        if (kind == kBwd) hipLaunchKernelGGL((conv_bwd_kernel<T, W, V>), dim3(grid), dim3(kT), lds, s, p);
    if constexpr (kWide) {
        if (kind == kFwd) hipLaunchKernelGGL((conv_fwd_kernel<T, W, V>), dim3(grid), dim3(kT), lds, s, p);
        if (kind == kStep) hipLaunchKernelGGL((conv_step_kernel<T, W, V>), dim3(grid), dim3(kT), 0, s, p);
    }
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

int run(Kind kind, ConvArgs& p, int W, int dtype, hipStream_t s) {
    // Whole sequences take 16 bytes of channels per thread from the width of one such group on; backward four channels (with
    // eight of a 16-bit type its registers leave two waves per SIMD: 63 us against 56 at 4 x 4096 x 2048 bf16).  The step form
    // writes its state in place, so no channel may be computed twice there: single channels where V does not divide D.
    int v = kind == kBwd ? 4 : (int)(16 / dtype_bytes(dtype));
    if (kind == kStep ? p.D % v != 0 : p.D < v) v = 1;
    p.groups = (p.D + v - 1) / v;
    size_t grid;
    if (kind == kStep) {
        grid = ((size_t)p.B * p.groups + kT - 1) / kT;
    } else {
        // the widest workgroup that leaves at most an eighth of its lanes without a channel
        p.gx = 64;
        while (p.gx > 8 && (p.groups + p.gx - 1) / p.gx * p.gx * 8 > p.groups * 9) p.gx /= 2;
        p.gblocks = (p.groups + p.gx - 1) / p.gx;
        const int per = kT / p.gx;
        grid = (((size_t)p.B * p.ntiles + per - 1) / per) * p.gblocks;
    }
    if (grid > (size_t)kMaxGroups) return fail(AFD_ERR_UNSUPPORTED, "causal conv: %zu workgroups", grid);
    if (dtype == AFD_T_F32) {
        if (v > 1) launch_w<float, 4>(kind, W, p, (unsigned)grid, s);
        else launch_w<float, 1>(kind, W, p, (unsigned)grid, s);
    } else if (dtype == AFD_T_BF16) {
        if (v == 8) launch_w<bf16_t, 8>(kind, W, p, (unsigned)grid, s);
        else if (v == 4) launch_w<bf16_t, 4>(kind, W, p, (unsigned)grid, s);
        else launch_w<bf16_t, 1>(kind, W, p, (unsigned)grid, s);
    } else {
        if (v == 8) launch_w<f16_t, 8>(kind, W, p, (unsigned)grid, s);
        else if (v == 4) launch_w<f16_t, 4>(kind, W, p, (unsigned)grid, s);
        else launch_w<f16_t, 1>(kind, W, p, (unsigned)grid, s);
    }
    return check_launch("causal_conv kernel");
}

// Rows per thread: long tiles repeat fewer rows at their ends (W - 1, both ends backward) and load fewer taps, short ones
// make more waves.  The longest up to 32 that leaves two waves per SIMD, counted at 8 channels per thread.  4 x 4096 x 2048
// bf16: backward and the sums behind it 56 + 5 / 66 + 5 / 73 + 4 us with 32 / 48 / 64 rows, forward 33 / 32 us with 16 / 32;
// 16 x 777 x 1024: forward 17.1 / 19.2 us with 8 / 16 rows.
int tile_rows(int B, int L, int D, int shortest) {
    const double waves = (double)B * L * D / (8 * 64);
    int tile = 32;
    while (tile > shortest && waves / tile < 2048) tile /= 2;
    return tile;
}
constexpr int kFwdShortest = 8, kBwdShortest = 16;

int check(const char* what, int B, int L, int D, int W, int act, int dtype) {
    if (B < 1 || L < 1 || D < 1 || W < 2 || W > kMaxW || act < 0 || act > 1 || !dtype_ok(dtype))
        return fail(AFD_ERR_ARG, "%s: B=%d L=%d D=%d W=%d (2..%d) act=%d dtype=%d", what, B, L, D, W, kMaxW, act, dtype);
    if ((long)B * ceil_div(L, kFwdShortest) > 0x7fffffffL)
        return fail(AFD_ERR_UNSUPPORTED, "%s: B=%d L=%d has too many row tiles", what, B, L);
    return AFD_OK;
}

}  // namespace

extern "C" int afd_causal_conv_forward(const void* x, long long xb, long long xl, const void* w, const void* bias, int w_f32,
                                       const void* state, const int* lengths, void* y, void* state_out, int B, int L, int D,
                                       int W, int act, int dtype, afd_stream_t stream) {
    if (!x || !w || !y) return fail(AFD_ERR_ARG, "causal conv: missing tensor");
    if (int rc = check("causal conv", B, L, D, W, act, dtype)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ConvArgs p{};
    p.x = x; p.xb = xb; p.xl = xl; p.w = w; p.bias = bias; p.w_f32 = w_f32; p.state = state; p.lengths = lengths;
    p.y = y; p.state_out = state_out; p.B = B; p.L = L; p.D = D; p.act = act;
    p.tile = tile_rows(B, L, D, kFwdShortest);
    p.ntiles = ceil_div(L, p.tile);
    ScopedBytes timing(AFD_K_SEQUENCE, 2.0 * dtype_bytes(dtype) * B * L * D, s);
    return run(kFwd, p, W, dtype, s);
}

extern "C" size_t afd_causal_conv_backward_workspace_bytes(int B, int L, int D, int W) {
    if (B < 1 || L < 1 || D < 1) return 0;
    return (size_t)B * ceil_div(L, tile_rows(B, L, D, kBwdShortest)) * D * (W + 1) * sizeof(float);
}

extern "C" int afd_causal_conv_backward(const void* x, long long xb, long long xl, const void* w, const void* bias, int w_f32,
                                        const void* state, const int* lengths, const void* dy, long long dyb, long long dyl,
                                        const void* dstate_out, void* dx, void* dw, void* dbias, void* dstate, int B, int L,
                                        int D, int W, int act, int dtype, void* ws, size_t ws_bytes, afd_stream_t stream) {
    if (!x || !w || !dy || !dx || !dw) return fail(AFD_ERR_ARG, "causal conv backward: missing tensor");
    if (int rc = check("causal conv backward", B, L, D, W, act, dtype)) return rc;
    if (!ws || ws_bytes < afd_causal_conv_backward_workspace_bytes(B, L, D, W))
        return fail(AFD_ERR_WORKSPACE, "causal conv backward: workspace of %zu bytes is too small", ws_bytes);
    if ((long)D * (W + 1) > 0x7fffffc0L) return fail(AFD_ERR_UNSUPPORTED, "causal conv backward: D=%d", D);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ConvArgs p{};
    p.x = x; p.xb = xb; p.xl = xl; p.w = w; p.bias = bias; p.w_f32 = w_f32; p.state = state; p.lengths = lengths;
    p.dy = dy; p.dyb = dyb; p.dyl = dyl; p.dstate_out = dstate_out; p.dx = dx; p.dstate = dstate;
    p.B = B; p.L = L; p.D = D; p.act = act;
    p.part = static_cast<float*>(ws);
    p.tile = tile_rows(B, L, D, kBwdShortest);
    p.ntiles = ceil_div(L, p.tile);
    ScopedBytes timing(AFD_K_SEQUENCE, 3.0 * dtype_bytes(dtype) * B * L * D, s);
    if (int rc = run(kBwd, p, W, dtype, s)) return rc;
    const int pt = w_f32 ? AFD_T_F32 : dtype;
    ColumnOuts o{};
    o.n = 2;
    o.o[0] = {dw, 0, D * W, D, D, 1, W, pt};
    o.o[1] = {dbias, D * W, D * W + D, 1, 1, 1, 0, pt};
    return launch_column_sums(p.part, (long)B * p.ntiles, D * (W + 1), o, s);
}

extern "C" int afd_causal_conv_step(const void* x, long long xb, const void* w, const void* bias, int w_f32,
                                    const void* state, void* y, void* state_out, int B, int D, int W, int act, int dtype,
                                    afd_stream_t stream) {
    if (!x || !w || !y || !state || !state_out) return fail(AFD_ERR_ARG, "causal conv step: missing tensor");
    if (int rc = check("causal conv step", B, 1, D, W, act, dtype)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ConvArgs p{};
    p.x = x; p.xb = xb; p.w = w; p.bias = bias; p.w_f32 = w_f32; p.state = state; p.y = y; p.state_out = state_out;
    p.B = B; p.L = 1; p.D = D; p.act = act; p.tile = 1; p.ntiles = 1;
    ScopedBytes timing(AFD_K_SEQUENCE, 2.0 * dtype_bytes(dtype) * B * D * W, s);
    return run(kStep, p, W, dtype, s);
}
