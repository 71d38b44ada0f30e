// Forward of the selective state-space scan (see state_scan.h for the formulas and the lane layout).
// Bound by vector instruction issue: per token, channel and state one exponential (two issue slots), two products and two
// multiply-adds, 6 slots, against 8 bytes per token and channel.  Measured, 16 states: 128 x 101 x 1024 fp32 82 us, vector
// issue 93 % of the time; 4 x 4096 x 2048 bf16 in 8 time segments 120 + 180 us, 96 and 93 %; 1 x 16384 x 1024 62 + 90 us.
#include "state_scan.h"

namespace {

using namespace afd;

// LOCAL: the walk of a time segment from a zero state, leaving only its end state and its sum of delta (the decay over the
// whole segment is exp(a sum delta)).  Otherwise the full walk; with more than one segment it first carries the state
// over the segments in front of it, one exponential and one multiply-add per state and segment.
template <typename T, int Q, int NS, bool LOCAL>
__global__ void __launch_bounds__(kScanT) scan_fwd_kernel(const ScanArgs p) {
    constexpr int NP = Q * NS, R = kTokF / Q;
    __shared__ __attribute__((aligned(16))) float lds[2][kTokF * 2 * NP];
    const ScanPlace w = scan_place<Q, NS>(p);
    const int start = w.s * p.seg;
    const int end = min(start + p.seg, w.n);  // tokens [start, end) are this segment's
    if (LOCAL && end >= w.n) return;  // the last segment with tokens (and all behind it): nobody asks
    const size_t seg = ((size_t)w.b * p.S + w.s) * p.D + w.cl;

    float a2[NS], h[NS];
    load_states<NS>(p.a + (size_t)w.cl * p.N, w.n0, p.N, true, a2);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        a2[k] = log2_decay(a2[k]);
        h[k] = 0.f;
    }
    if (!LOCAL) {
        load_states<NS>(p.state ? p.state + ((size_t)w.b * p.D + w.cl) * p.N : nullptr, w.n0, p.N, true, h);
        if (start < w.n) {
            for (int s = 0; s < w.s; ++s) {
                const size_t at = ((size_t)w.b * p.S + s) * p.D + w.cl;
                float e[NS];
                load_vec<NS>(p.seg_h + at * NP + w.n0, e);
                carry<NS>(a2, p.seg_d[at], e, h);
            }
        }
    }
    const float bias = p.dt_bias ? p.dt_bias[w.cl] : 0.f;
    const float dskip = (!LOCAL && p.d) ? p.d[w.cl] : 0.f;
    const bool gated = !LOCAL && p.gate;
    const T* xb = static_cast<const T*>(p.x) + (size_t)w.b * p.xb;
    const T* tb = static_cast<const T*>(p.dt) + (size_t)w.b * p.tb;
    const T* gb = gated ? static_cast<const T*>(p.gate) + (size_t)w.b * p.gb : nullptr;
    const T* br = static_cast<const T*>(p.b) + (size_t)w.b * p.bb;
    const T* cr = static_cast<const T*>(p.c) + (size_t)w.b * p.cb;
    T* yb = LOCAL ? nullptr : static_cast<T*>(p.y) + (size_t)w.b * p.L * p.D;
    const unsigned chan = (unsigned)w.cl * sizeof(T);
    const unsigned xo = chan + (unsigned)(w.q * p.xl * sizeof(T)), to = chan + (unsigned)(w.q * p.tl * sizeof(T));
    const unsigned go = gated ? chan + (unsigned)(w.q * p.gl * sizeof(T)) : 0u;
    const unsigned yo = chan + (unsigned)(w.q * p.D * sizeof(T));
    float sum_delta = 0.f;

    BcStage<T, NP, kTokF> bc;
    TokLoad<T, Q, kTokF> nx, nt, ng;
    auto fetch = [&](int t0) {
        bc.fetch(p, br, cr, t0, w.n);
        const int left = w.n - t0;
        if (left >= kTokF) {
            nx.full(xb + (size_t)t0 * p.xl, p.xl, xo);
            nt.full(tb + (size_t)t0 * p.tl, p.tl, to);
            if (gated) ng.full(gb + (size_t)t0 * p.gl, p.gl, go);
        } else {
            nx.tail(xb + (size_t)t0 * p.xl, p.xl, left, w.q, chan);
            nt.tail(tb + (size_t)t0 * p.tl, p.tl, left, w.q, chan);
            if (gated) ng.tail(gb + (size_t)t0 * p.gl, p.gl, left, w.q, chan);
        }
    };
    if (start < end) {
        fetch(start);
        bc.put(lds[0], start, w.n, p.N);
    }
    __syncthreads();
    int turn = 0;
    for (int t0 = start; t0 < end; t0 += kTokF, turn ^= 1) {
        const float* row = lds[turn] + w.n0;
        float dl[R], dx[R], xv[R], gv[R], yv[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            xv[i] = to_f32(nx.v[i]);
            const float raw = to_f32(nt.v[i]) + bias;
            dl[i] = p.softplus ? softplus_f32(raw) : raw;
            dx[i] = dl[i] * xv[i];
            if (gated) gv[i] = to_f32(ng.v[i]);
        }
        if (t0 + kTokF > w.n) {  // exp(0) = 1 and nothing added: the state holds behind row n
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool in = t0 + i * Q + w.q < w.n;
                dl[i] = in ? dl[i] : 0.f;
                dx[i] = in ? dx[i] : 0.f;
            }
        }
        if (LOCAL) {
#pragma unroll
            for (int i = 0; i < R; ++i) sum_delta += dl[i];
        }
        if (t0 + kTokF < end) fetch(t0 + kTokF);
        // The steps go first at the SIMD, in front of what other waves do between their blocks: waves then take turns instead of
        // moving in step (190 to 182 us at 4 x 4096 x 2048 bf16, 54 to 49 at 16 x 777 x 771 fp16).
        __builtin_amdgcn_s_setprio(1);
        float part[Q], nb[NS], nc[NS];  // nb, nc: the next token's rows, asked for one token ahead
        load_vec<NS>(row, nb);
        if (!LOCAL) load_vec<NS>(row + NP, nc);
#pragma unroll
        for (int j = 0; j < kTokF; ++j) {
            if (!LOCAL && j % kCkpt == 0 && p.ckpt && w.live && t0 + j < w.n)
                store_vec<NS>(p.ckpt + (((size_t)w.b * ((p.L + kCkpt - 1) / kCkpt) + (t0 + j) / kCkpt) * p.D + w.ch) * NP + w.n0, h);
            const int i = j / Q, ql = j % Q;
            const float de = from_lane<Q>(dl[i], ql), dxj = from_lane<Q>(dx[i], ql);
            float bv[NS], cv[NS], y = 0.f;
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                bv[k] = nb[k];
                if (!LOCAL) cv[k] = nc[k];
            }
            if (j + 1 < kTokF) {
                load_vec<NS>(row + (j + 1) * 2 * NP, nb);
                if (!LOCAL) load_vec<NS>(row + (j + 1) * 2 * NP + NP, nc);
                hold_lds();
            }
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const float e = __builtin_amdgcn_exp2f(de * a2[k]);
                h[k] = fmaf(e, h[k], dxj * bv[k]);
                if (!LOCAL) y = fmaf(cv[k], h[k], y);
            }
            if (!LOCAL) {
                part[ql] = y;
                if (ql == Q - 1) yv[i] = scatter_lanes<Q>(part);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (!LOCAL) {
            loads_arrived();
            T out[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                float y = fmaf(dskip, xv[i], yv[i]);
                if (gated) y *= gv[i] * sigmoid_f32(gv[i]);
                out[i] = from_f32<T>(y);
            }
            T* yt = yb + (size_t)t0 * p.D;
            if (t0 + kTokF <= w.n) {
                if (w.live) {
#pragma unroll
                    for (int i = 0; i < R; ++i)
                        *reinterpret_cast<T*>(reinterpret_cast<char*>(yt + (size_t)(i * Q) * p.D) + yo) = out[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int t = t0 + i * Q + w.q;
                    if (w.live && t < p.L) yb[(size_t)t * p.D + w.ch] = t < w.n ? out[i] : from_f32<T>(0.f);
                }
            }
        }
        if (t0 + kTokF < end) bc.put(lds[turn ^ 1], t0 + kTokF, w.n, p.N);
        __syncthreads();
    }
    if (LOCAL) {
        sum_delta = sum_lanes<Q>(sum_delta);
        if (w.live) {
            store_vec<NS>(p.seg_h + seg * NP + w.n0, h);
            if (w.q == 0) p.seg_d[seg] = sum_delta;
        }
        return;
    }
    // rows behind the last token, and the state behind it (by the segment that holds it, or the first if there is none)
    const int done = start < end ? start + (end - start + kTokF - 1) / kTokF * kTokF : start;
    const int stop = min(start + p.seg, p.L);
    for (int t = done + w.q; t < stop; t += Q)
        if (w.live) yb[(size_t)t * p.D + w.ch] = from_f32<T>(0.f);
    const int last = w.n > 0 ? (w.n - 1) / p.seg : 0;
    if (p.state_out && w.s == last)
        store_states<NS>(p.state_out + ((size_t)w.b * p.D + w.cl) * p.N, w.n0, p.N, w.live, h);
}

template <typename T, int Q, int NS> int launch(const ScanArgs& p, hipStream_t s) {
    const unsigned grid = (unsigned)((long)p.B * p.S * p.nb);
    if (p.S > 1) hipLaunchKernelGGL((scan_fwd_kernel<T, Q, NS, true>), dim3(grid), dim3(kScanT), 0, s, p);
    hipLaunchKernelGGL((scan_fwd_kernel<T, Q, NS, false>), dim3(grid), dim3(kScanT), 0, s, p);
    return check_launch("scan_fwd_kernel");
}

template <typename T> int launch_n(const ScanArgs& p, hipStream_t s) {
    const ScanShape g = scan_shape(p.N);
    if (g.NP == 4) return launch<T, 4, 1>(p, s);
    if (g.NP == 8) return launch<T, 4, 2>(p, s);
    if (g.NP == 16) return launch<T, 4, 4>(p, s);
    if (g.NP == 32) return launch<T, 8, 4>(p, s);
    return launch<T, 16, 4>(p, s);
}

// NS neighbouring elements, in one load where there are 8 or 16 bytes of them
template <typename T, int NS> __device__ __forceinline__ void load_few(const T* p, float (&r)[NS]) {
    if constexpr (NS * sizeof(T) >= 8) load_row<T, NS>(p, r);
    else {
#pragma unroll
        for (int k = 0; k < NS; ++k) r[k] = to_f32(p[k]);
    }
}

// One token for RB rows of the batch at a time.  Bound by the state, 8 bytes read and written per channel and state:
// 512 x 2048 x 16 in 23.7 us, 6.0 TB/s.  With
// RB = 4 a channel's lanes share the rows' per-token work as they share a sequence's tokens (lane q: softplus and gate of
// row q), a is loaded once and four state loads are under way per lane; RB = 1 where there are too few rows for that to
// fill the card.  Every lane reads its states before it writes them: state_out may be the state.
template <typename T, int Q, int NS, int RB>
__global__ void __launch_bounds__(kScanT) scan_step_kernel(const ScanArgs p) {
    const int cb = blockIdx.x % p.nb, b0 = (int)(blockIdx.x / p.nb) * RB;
    const int q = threadIdx.x & (Q - 1), ch = cb * (kScanT / Q) + (int)threadIdx.x / Q, n0 = q * NS;
    if (ch >= p.D) return;  // (whole channels: the Q lanes that meet below are all there or all gone)
    const bool vec = p.N == Q * NS && p.seg;  // unpadded rows on 16-byte boundaries (seg: what the host found)
    const int r = RB > 1 ? q & (RB - 1) : 0, own = min(b0 + r, p.B - 1);
    const float x = to_f32(static_cast<const T*>(p.x)[(size_t)own * p.xb + ch]);
    const float raw = to_f32(static_cast<const T*>(p.dt)[(size_t)own * p.tb + ch]) + (p.dt_bias ? p.dt_bias[ch] : 0.f);
    const float gt = p.gate ? to_f32(static_cast<const T*>(p.gate)[(size_t)own * p.gb + ch]) : 0.f;
    float a2[NS], h[RB][NS], bv[RB][NS], cv[RB][NS];
    if (vec) load_vec<NS>(p.a + (size_t)ch * p.N + n0, a2);
    else load_states<NS>(p.a + (size_t)ch * p.N, n0, p.N, true, a2);
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        const int b = min(b0 + j, p.B - 1);
        const float* st = p.state + ((size_t)b * p.D + ch) * p.N;
        const T* br = static_cast<const T*>(p.b) + (size_t)b * p.bb;
        const T* cr = static_cast<const T*>(p.c) + (size_t)b * p.cb;
        if (vec) {
            load_vec<NS>(st + n0, h[j]);
            load_few<T, NS>(br + n0, bv[j]);
            load_few<T, NS>(cr + n0, cv[j]);
        } else {
            load_states<NS>(st, n0, p.N, true, h[j]);
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                bv[j][k] = n0 + k < p.N ? to_f32(br[n0 + k]) : 0.f;
                cv[j][k] = n0 + k < p.N ? to_f32(cr[n0 + k]) : 0.f;
            }
        }
    }
    const float de = p.softplus ? softplus_f32(raw) : raw, dx = de * x;
    float yown = 0.f;
#pragma unroll
    for (int j = 0; j < RB; ++j) {
        const float dej = RB > 1 ? from_lane<Q>(de, j) : de, dxj = RB > 1 ? from_lane<Q>(dx, j) : dx;
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            h[j][k] = fmaf(__builtin_amdgcn_exp2f(dej * (a2[k] * kLog2e)), h[j][k], dxj * bv[j][k]);
            y = fmaf(cv[j][k], h[j][k], y);
        }
        y = sum_lanes<Q>(y);
        yown = r == j ? y : yown;
        if (b0 + j < p.B) {
            float* so = p.state_out + ((size_t)(b0 + j) * p.D + ch) * p.N;
            if (vec) store_vec<NS>(so + n0, h[j]);
            else store_states<NS>(so, n0, p.N, true, h[j]);
        }
    }
    if (q < RB && b0 + q < p.B) {
        float y = fmaf(p.d ? p.d[ch] : 0.f, x, yown);
        if (p.gate) y *= gt * sigmoid_f32(gt);
        static_cast<T*>(p.y)[(size_t)(b0 + q) * p.D + ch] = from_f32<T>(y);
    }
}

// Four rows at a time from 8 workgroups per CU on.
template <typename T, int Q, int NS> int step(const ScanArgs& p, hipStream_t s) {
    const long one = (long)p.B * p.nb;
    if (one >= 2048)
        hipLaunchKernelGGL((scan_step_kernel<T, Q, NS, 4>), dim3((unsigned)((long)((p.B + 3) / 4) * p.nb)), dim3(kScanT), 0, s, p);
    else
        hipLaunchKernelGGL((scan_step_kernel<T, Q, NS, 1>), dim3((unsigned)one), dim3(kScanT), 0, s, p);
    return check_launch("scan_step_kernel");
}
template <typename T> int step_n(const ScanArgs& p, hipStream_t s) {
    const ScanShape g = scan_shape(p.N);
    if (g.NP == 4) return step<T, 4, 1>(p, s);
    if (g.NP == 8) return step<T, 4, 2>(p, s);
    if (g.NP == 16) return step<T, 4, 4>(p, s);
    if (g.NP == 32) return step<T, 8, 4>(p, s);
    return step<T, 16, 4>(p, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Time segments: batch and channels give `have` workgroups.  From one per CU on the axis is walked in one piece; below that
// it is split into about 4 workgroups per CU, in segments of at least 128 tokens, which costs a second, lighter walk.
// 4 x 4096 x 2048 bf16, 128 workgroups, forward (both walks) / backward (both): 422 / 1011 us in 2 segments, 328 / 629 in 4,
// 299 / 619 in 8, 297 / 637 in 16; one walk alone at 256 workgroups takes 125 ns a token (backward 385) whatever the split
// would make of it: 512 us for 4096 tokens against 610 in 4 segments.
int segments(int B, int nb, int nblk) {
    const long have = (long)B * nb;
    if (have >= 256 || nblk < 16) return 1;
    const long want = (1024 + have - 1) / have, most = nblk / 8;
    return (int)(want < most ? want : most);
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct ScanPlan {
    ScanShape g;
    int nb, S, seg;
    size_t seg_h, seg_d, part_bc, part_p;  // bytes
};
ScanPlan scan_plan(int B, int L, int D, int N, bool backward) {
    ScanPlan q;
    q.g = scan_shape(N);
    q.nb = ceil_div(D, kScanT / q.g.Q);
    const int nblk = ceil_div(L, kTokF);
    q.seg = ceil_div(nblk, segments(B, q.nb, nblk)) * kTokF;
    q.S = ceil_div(L, q.seg);
    q.seg_h = q.S > 1 ? align256((size_t)B * q.S * D * q.g.NP * 4) : 0;
    q.seg_d = q.S > 1 ? align256((size_t)B * q.S * D * 4) : 0;
    q.part_bc = backward ? align256((size_t)q.nb * B * L * 2 * q.g.NP * 4) : 0;
    q.part_p = backward ? align256((size_t)B * q.S * D * (q.g.NP + 2) * 4) : 0;
    return q;
}

int check(const char* what, int B, int L, int D, int N, int dtype) {
    if (B < 1 || L < 1 || D < 1 || N < 1 || N > 64 || !dtype_ok(dtype))
        return fail(AFD_ERR_ARG, "%s: B=%d L=%d D=%d N=%d (1..64) dtype=%d", what, B, L, D, N, dtype);
    const ScanPlan q = scan_plan(B, L, D, N, false);
    if ((long)B * q.S * q.nb > kMaxGroups || (long)D * (q.g.NP + 2) > 0x3fffffffL || L > 0x7fff0000 ||
        (long)D * kTokF * 4 > 0x7fffffffL)
        return fail(AFD_ERR_UNSUPPORTED, "%s: B=%d L=%d D=%d is too large", what, B, L, D);
    return AFD_OK;
}

// the lanes' offsets inside a block of tokens are 32-bit: 2^24 elements of 4 bytes between rows at most
int check_rows(const char* what, const long long* st, int n, int dtype) {
    for (int i = 1; i < n; i += 2)
        if (st[i] < 0 || st[i] * kTokF * (long long)dtype_bytes(dtype) > 0x40000000LL)
            return fail(AFD_ERR_UNSUPPORTED, "%s: row stride %lld", what, st[i]);
    return AFD_OK;
}

void set_inputs(ScanArgs& p, const void* x, const void* dt, const void* b, const void* c, const void* gate,
                const long long* st) {
    p.x = x; p.dt = dt; p.b = b; p.c = c; p.gate = gate;
    p.xb = st[0]; p.xl = st[1]; p.tb = st[2]; p.tl = st[3]; p.bb = st[4]; p.bl = st[5]; p.cb = st[6]; p.cl = st[7];
    p.gb = st[8]; p.gl = st[9];
}

}  // namespace

int afd::scan_forward_launch(const ScanArgs& p, int dtype, hipStream_t s) {
    if (dtype == AFD_T_F32) return launch_n<float>(p, s);
    if (dtype == AFD_T_BF16) return launch_n<bf16_t>(p, s);
    return launch_n<f16_t>(p, s);
}

extern "C" size_t afd_state_scan_workspace_bytes(int B, int L, int D, int N, int backward) {
    if (B < 1 || L < 1 || D < 1 || N < 1 || N > 64) return 0;
    const ScanPlan q = scan_plan(B, L, D, N, backward != 0);
    return q.seg_h + q.seg_d + q.part_bc + q.part_p;
}

extern "C" size_t afd_state_scan_checkpoint_floats(int B, int L, int D, int N) {
    if (B < 1 || L < 1 || D < 1 || N < 1 || N > 64) return 0;
    return (size_t)B * ceil_div(L, kCkpt) * D * scan_shape(N).NP;
}

extern "C" int afd_state_scan_forward(const void* x, const void* dt, const void* b, const void* c, const void* gate,
                                      const long long* strides, const float* a, const float* d, const float* dt_bias,
                                      const float* state, const int* lengths, void* y, float* state_out, float* checkpoints,
                                      int B, int L, int D, int N, int softplus, int dtype, void* ws, size_t ws_bytes,
                                      afd_stream_t stream) {
    if (!x || !dt || !b || !c || !a || !y || !strides) return fail(AFD_ERR_ARG, "state scan: missing tensor");
    if (int rc = check("state scan", B, L, D, N, dtype)) return rc;
    if (int rc = check_rows("state scan", strides, 10, dtype)) return rc;
    const ScanPlan q = scan_plan(B, L, D, N, false);
    if (q.seg_h + q.seg_d > 0 && (!ws || ws_bytes < q.seg_h + q.seg_d))
        return fail(AFD_ERR_WORKSPACE, "state scan: workspace of %zu bytes, %zu needed", ws_bytes, q.seg_h + q.seg_d);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ScanArgs p{};
    set_inputs(p, x, dt, b, c, gate, strides);
    p.a = a; p.d = d; p.dt_bias = dt_bias; p.state = state; p.lengths = lengths; p.y = y; p.state_out = state_out;
    p.ckpt = checkpoints;
    p.B = B; p.L = L; p.D = D; p.N = N; p.softplus = softplus; p.S = q.S; p.seg = q.seg; p.nb = q.nb;
    p.seg_h = static_cast<float*>(ws);
    p.seg_d = reinterpret_cast<float*>(static_cast<char*>(ws) + q.seg_h);
    ScopedBytes timing(AFD_K_SEQUENCE, dtype_bytes(dtype) * (gate ? 4.0 : 3.0) * B * L * D, s);
    return scan_forward_launch(p, dtype, s);
}

extern "C" int afd_state_scan_step(const void* x, const void* dt, const void* b, const void* c, const void* gate,
                                   const long long* strides, const float* a, const float* d, const float* dt_bias,
                                   const float* state, void* y, float* state_out, int B, int D, int N, int softplus, int dtype,
                                   afd_stream_t stream) {
    if (!x || !dt || !b || !c || !a || !y || !state || !state_out || !strides)
        return fail(AFD_ERR_ARG, "state scan step: missing tensor");
    if (int rc = check("state scan step", B, 1, D, N, dtype)) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    ScanArgs p{};
    const long long st[10] = {strides[0], 0, strides[1], 0, strides[2], 0, strides[3], 0, strides[4], 0};
    set_inputs(p, x, dt, b, c, gate, st);
    p.a = a; p.d = d; p.dt_bias = dt_bias; p.state = state; p.y = y; p.state_out = state_out;
    p.B = B; p.L = 1; p.D = D; p.N = N; p.softplus = softplus;
    const ScanShape g = scan_shape(N);
    p.nb = ceil_div(D, kScanT / g.Q);
    p.S = 1;
    p.seg = aligned16(a) && aligned16(state) && aligned16(state_out);
    ScopedBytes timing(AFD_K_SEQUENCE, 8.0 * B * D * N, s);
    if (dtype == AFD_T_F32) return step_n<float>(p, s);
    if (dtype == AFD_T_BF16) return step_n<bf16_t>(p, s);
    return step_n<f16_t>(p, s);
}

extern "C" int afd_state_scan_backward(const void* x, const void* dt, const void* b, const void* c, const void* gate,
                                       const void* dy, const long long* strides, const float* a, const float* d,
                                       const float* dt_bias, const int* lengths, const float* checkpoints,
                                       const float* dstate_out, void* dx, void* ddt, void* db, void* dc, void* dgate, float* da,
                                       float* dd, float* ddt_bias, float* dstate, int B, int L, int D, int N, int softplus,
                                       int dtype, void* ws, size_t ws_bytes, afd_stream_t stream) {
    if (!x || !dt || !b || !c || !a || !dy || !strides || !checkpoints || !dx || !ddt || !db || !dc || !da || (gate && !dgate))
        return fail(AFD_ERR_ARG, "state scan backward: missing tensor");
    if (int rc = check("state scan backward", B, L, D, N, dtype)) return rc;
    if (int rc = check_rows("state scan backward", strides, 12, dtype)) return rc;
    const ScanPlan q = scan_plan(B, L, D, N, true);
    const size_t need = q.seg_h + q.seg_d + q.part_bc + q.part_p;
    if (!ws || ws_bytes < need)
        return fail(AFD_ERR_WORKSPACE, "state scan backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ScanArgs p{};
    set_inputs(p, x, dt, b, c, gate, strides);
    p.dy = dy; p.yb = strides[10]; p.yl = strides[11];
    p.a = a; p.d = d; p.dt_bias = dt_bias; p.lengths = lengths; p.ckpt = const_cast<float*>(checkpoints);
    p.dstate_out = dstate_out; p.dx = dx; p.ddt = ddt; p.dgate = dgate; p.dstate = dstate;
    p.B = B; p.L = L; p.D = D; p.N = N; p.softplus = softplus; p.S = q.S; p.seg = q.seg; p.nb = q.nb;
    char* at = static_cast<char*>(ws);
    p.seg_h = reinterpret_cast<float*>(at);
    p.seg_d = reinterpret_cast<float*>(at + q.seg_h);
    p.part_bc = reinterpret_cast<float*>(at + q.seg_h + q.seg_d);
    p.part_p = reinterpret_cast<float*>(at + q.seg_h + q.seg_d + q.part_bc);
    ScopedBytes timing(AFD_K_SEQUENCE, dtype_bytes(dtype) * (gate ? 6.0 : 4.0) * B * L * D, s);
    if (int rc = scan_backward_launch(p, dtype, s)) return rc;
    if (int rc = scan_bc_gradients(p, db, dc, dtype, s)) return rc;
    ColumnOuts o{};
    o.n = 3;
    o.o[0] = {da, 0, D * q.g.NP, q.g.NP, N, N, 1, AFD_T_F32};
    o.o[1] = {dd, D * q.g.NP, D * q.g.NP + D, 1, 1, 1, 0, AFD_T_F32};
    o.o[2] = {ddt_bias, D * q.g.NP + D, D * q.g.NP + 2 * D, 1, 1, 1, 0, AFD_T_F32};
    return launch_column_sums(p.part_p, (long)B * q.S, D * (q.g.NP + 2), o, s);
}
