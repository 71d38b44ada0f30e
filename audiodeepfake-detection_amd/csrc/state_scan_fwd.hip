// Forward of the selective state-space scan (see state_scan.h for the formulas and the lane layout).
#include "state_scan.h"

namespace {

using namespace afd;

// LOCAL: the walk of a time segment from a zero state, leaving only its end state and its sum of delta (the decay over the
// whole segment is exp(a sum delta)).  Otherwise the full walk; with more than one segment it first carries the state
// over the segments in front of it, S fused multiply-adds per state.
template <typename T, int Q, int NS, bool LOCAL>
__global__ void __launch_bounds__(kScanT) scan_fwd_kernel(const ScanArgs p) {
    constexpr int NP = Q * NS, R = kTok / Q;
    __shared__ float lds[2][kTok * 2 * NP];
    const ScanPlace w = scan_place<Q, NS>(p);
    const int nblk = (w.n + kTok - 1) / kTok;
    const int blk0 = w.s * p.seg_blocks;
    const int blk1 = min(blk0 + p.seg_blocks, nblk);
    if (LOCAL && blk1 * kTok >= w.n) return;  // the last segment with tokens (and all behind it): nobody asks
    const size_t seg = ((size_t)w.b * p.S + w.s) * p.D + w.ch;

    float a2[NS], h[NS];
    load_states<NS>(p.a + (size_t)w.ch * p.N, w.n0, p.N, w.live, a2);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        a2[k] *= kLog2e;
        h[k] = 0.f;
    }
    if (!LOCAL) {
        load_states<NS>(p.state ? p.state + ((size_t)w.b * p.D + w.ch) * p.N : nullptr, w.n0, p.N, w.live, h);
        if (w.live && blk0 < nblk) {
            for (int s = 0; s < w.s; ++s) {
                const size_t at = ((size_t)w.b * p.S + s) * p.D + w.ch;
                float e[NS];
                load_vec<NS>(p.seg_h + at * NP + w.n0, e);
                const float sd = p.seg_d[at];
#pragma unroll
                for (int k = 0; k < NS; ++k) h[k] = fmaf(__builtin_amdgcn_exp2f(a2[k] * sd), h[k], e[k]);
            }
        }
    }
    const float bias = (p.dt_bias && w.live) ? p.dt_bias[w.ch] : 0.f;
    const float dskip = (!LOCAL && p.d && w.live) ? p.d[w.ch] : 0.f;
    const T* xc = static_cast<const T*>(p.x) + (size_t)w.b * p.xb + w.ch;
    const T* tc = static_cast<const T*>(p.dt) + (size_t)w.b * p.tb + w.ch;
    const T* gc = p.gate ? static_cast<const T*>(p.gate) + (size_t)w.b * p.gb + w.ch : nullptr;
    const T* br = static_cast<const T*>(p.b) + (size_t)w.b * p.bb;
    const T* cr = static_cast<const T*>(p.c) + (size_t)w.b * p.cb;
    T* yc = LOCAL ? nullptr : static_cast<T*>(p.y) + (size_t)w.b * p.L * p.D + w.ch;
    float sum_delta = 0.f;

    BcStage<T, NP> bc;
    TokLoad<T, Q> nx, nt, ng;
    if (blk0 < blk1) {
        bc.fetch(p, br, cr, blk0 * kTok, w.n);
        nx.fetch(xc, p.xl, blk0 * kTok, w.q, w.n, w.live);
        nt.fetch(tc, p.tl, blk0 * kTok, w.q, w.n, w.live);
        if (!LOCAL && gc) ng.fetch(gc, p.gl, blk0 * kTok, w.q, w.n, w.live);
        bc.put(lds[0]);
    }
    __syncthreads();
    for (int blk = blk0; blk < blk1; ++blk) {
        const int t0 = blk * kTok;
        const float* row = lds[(blk - blk0) & 1] + w.n0;
        float dl[R], dx[R], xv[R], gv[R], yv[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool in = t0 + i * Q + w.q < w.n;
            xv[i] = to_f32(nx.v[i]);
            const float raw = to_f32(nt.v[i]) + bias;
            const float de = p.softplus ? softplus_f32(raw) : raw;
            dl[i] = in ? de : 0.f;  // exp(0) = 1 and nothing added: the state holds behind row n
            dx[i] = dl[i] * xv[i];
            sum_delta += dl[i];
            yv[i] = 0.f;
            if (!LOCAL && gc) gv[i] = to_f32(ng.v[i]);
        }
        if (blk + 1 < blk1) {
            bc.fetch(p, br, cr, t0 + kTok, w.n);
            nx.fetch(xc, p.xl, t0 + kTok, w.q, w.n, w.live);
            nt.fetch(tc, p.tl, t0 + kTok, w.q, w.n, w.live);
            if (!LOCAL && gc) ng.fetch(gc, p.gl, t0 + kTok, w.q, w.n, w.live);
        }
        if (!LOCAL && p.ckpt && w.live)
            store_vec<NS>(p.ckpt + (((size_t)w.b * ((p.L + kTok - 1) / kTok) + blk) * p.D + w.ch) * NP + w.n0, h);
#pragma unroll
        for (int j = 0; j < kTok; ++j) {
            const int i = j / Q, ql = j % Q;
            const float de = from_lane<Q>(dl[i], ql), dxj = from_lane<Q>(dx[i], ql);
            float bv[NS], cv[NS], y = 0.f;
            load_vec<NS>(row + j * 2 * NP, bv);
            if (!LOCAL) load_vec<NS>(row + j * 2 * NP + NP, cv);
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const float e = __builtin_amdgcn_exp2f(de * a2[k]);
                h[k] = fmaf(e, h[k], dxj * bv[k]);
                if (!LOCAL) y = fmaf(cv[k], h[k], y);
            }
            if (!LOCAL) {
                y = sum_lanes<Q>(y);
                yv[i] = w.q == ql ? y : yv[i];
            }
        }
        if (!LOCAL) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int t = t0 + i * Q + w.q;
                float y = fmaf(dskip, xv[i], yv[i]);
                if (gc) y *= gv[i] * sigmoid_f32(gv[i]);
                if (w.live && t < p.L) yc[(size_t)t * p.D] = from_f32<T>(t < w.n ? y : 0.f);
            }
        }
        if (blk + 1 < blk1) bc.put(lds[(blk + 1 - blk0) & 1]);
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
    const int tail0 = max(blk0, blk1) * kTok, tail1 = min((blk0 + p.seg_blocks) * kTok, p.L);
    for (int t = tail0 + w.q; t < tail1; t += Q)
        if (w.live) yc[(size_t)t * p.D] = from_f32<T>(0.f);
    const int last = nblk > 0 ? (nblk - 1) / p.seg_blocks : 0;
    if (p.state_out && w.s == last)
        store_states<NS>(p.state_out + ((size_t)w.b * p.D + w.ch) * p.N, w.n0, p.N, w.live, h);
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

// One token.  Every lane reads its NS states before it writes them: state_out may be the state.
template <typename T, int Q, int NS>
__global__ void __launch_bounds__(kScanT) scan_step_kernel(const ScanArgs p) {
    const ScanPlace w = scan_place<Q, NS>(p);
    if (!w.live) return;  // (whole channels: the Q lanes that meet below are all there or all gone)
    const size_t st = ((size_t)w.b * p.D + w.ch) * p.N;
    float a2[NS], h[NS], bv[NS], cv[NS];
    const T* br = static_cast<const T*>(p.b) + (size_t)w.b * p.bb;
    const T* cr = static_cast<const T*>(p.c) + (size_t)w.b * p.cb;
    if (p.N == Q * NS && p.seg_blocks) {  // unpadded rows on 16-byte boundaries (seg_blocks: what the host found)
        load_vec<NS>(p.state + st + w.n0, h);
        load_vec<NS>(p.a + (size_t)w.ch * p.N + w.n0, a2);
    } else {
        load_states<NS>(p.state + st, w.n0, p.N, true, h);
        load_states<NS>(p.a + (size_t)w.ch * p.N, w.n0, p.N, true, a2);
    }
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        bv[k] = w.n0 + k < p.N ? to_f32(br[w.n0 + k]) : 0.f;
        cv[k] = w.n0 + k < p.N ? to_f32(cr[w.n0 + k]) : 0.f;
    }
    const float x = to_f32(static_cast<const T*>(p.x)[(size_t)w.b * p.xb + w.ch]);
    const float raw = to_f32(static_cast<const T*>(p.dt)[(size_t)w.b * p.tb + w.ch]) + (p.dt_bias ? p.dt_bias[w.ch] : 0.f);
    const float de = p.softplus ? softplus_f32(raw) : raw;
    float y = 0.f;
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        h[k] = fmaf(__builtin_amdgcn_exp2f(de * (a2[k] * kLog2e)), h[k], de * x * bv[k]);
        y = fmaf(cv[k], h[k], y);
    }
    y = sum_lanes<Q>(y);
    if (p.N == Q * NS && p.seg_blocks) store_vec<NS>(p.state_out + st + w.n0, h);
    else store_states<NS>(p.state_out + st, w.n0, p.N, true, h);
    if (w.q == 0) {
        y = fmaf(p.d ? p.d[w.ch] : 0.f, x, y);
        if (p.gate) {
            const float g = to_f32(static_cast<const T*>(p.gate)[(size_t)w.b * p.gb + w.ch]);
            y *= g * sigmoid_f32(g);
        }
        static_cast<T*>(p.y)[(size_t)w.b * p.D + w.ch] = from_f32<T>(y);
    }
}

template <typename T, int Q, int NS> int step(const ScanArgs& p, hipStream_t s) {
    hipLaunchKernelGGL((scan_step_kernel<T, Q, NS>), dim3((unsigned)((long)p.B * p.nb)), dim3(kScanT), 0, s, p);
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

// Time segments: batch and channels give B nb workgroups; below two per CU the time axis is split until there are
// about that many, in segments of at least 8 blocks (each costs a second, lighter walk over its tokens).
int segments(int B, int nb, int nblk) {
    const long have = (long)B * nb;
    if (have >= 256 || nblk < 16) return 1;
    long want = (512 + have - 1) / have;
    const long most = nblk / 8;
    return (int)(want < most ? want : most);
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

struct ScanPlan {
    ScanShape g;
    int nb, nblk, S, seg_blocks;
    size_t seg_h, seg_d, part_bc, part_p;  // bytes
};
ScanPlan scan_plan(int B, int L, int D, int N, bool backward) {
    ScanPlan q;
    q.g = scan_shape(N);
    q.nb = ceil_div(D, kScanT / q.g.Q);
    q.nblk = ceil_div(L, kTok);
    const int want = segments(B, q.nb, q.nblk);
    q.seg_blocks = ceil_div(q.nblk, want);
    q.S = ceil_div(q.nblk, q.seg_blocks);
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
    if ((long)B * q.S * q.nb > 0x7fffffffL || (long)D * (q.g.NP + 2) > 0x7fffffc0L || L > 0x7fffff00)
        return fail(AFD_ERR_UNSUPPORTED, "%s: B=%d L=%d D=%d is too large", what, B, L, D);
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
    return (size_t)B * ceil_div(L, kTok) * D * scan_shape(N).NP;
}

extern "C" int afd_state_scan_forward(const void* x, const void* dt, const void* b, const void* c, const void* gate,
                                      const long long* strides, const float* a, const float* d, const float* dt_bias,
                                      const float* state, const int* lengths, void* y, float* state_out, float* checkpoints,
                                      int B, int L, int D, int N, int softplus, int dtype, void* ws, size_t ws_bytes,
                                      afd_stream_t stream) {
    if (!x || !dt || !b || !c || !a || !y || !strides) return fail(AFD_ERR_ARG, "state scan: missing tensor");
    if (int rc = check("state scan", B, L, D, N, dtype)) return rc;
    const ScanPlan q = scan_plan(B, L, D, N, false);
    if (q.seg_h + q.seg_d > 0 && (!ws || ws_bytes < q.seg_h + q.seg_d))
        return fail(AFD_ERR_WORKSPACE, "state scan: workspace of %zu bytes, %zu needed", ws_bytes, q.seg_h + q.seg_d);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ScanArgs p{};
    set_inputs(p, x, dt, b, c, gate, strides);
    p.a = a; p.d = d; p.dt_bias = dt_bias; p.state = state; p.lengths = lengths; p.y = y; p.state_out = state_out;
    p.ckpt = checkpoints;
    p.B = B; p.L = L; p.D = D; p.N = N; p.softplus = softplus; p.S = q.S; p.seg_blocks = q.seg_blocks; p.nb = q.nb;
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
    p.seg_blocks = aligned16(a) && aligned16(state) && aligned16(state_out);
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
    p.B = B; p.L = L; p.D = D; p.N = N; p.softplus = softplus; p.S = q.S; p.seg_blocks = q.seg_blocks; p.nb = q.nb;
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
    o.o[0] = {da, 0, D * q.g.NP, q.g.NP, N, AFD_T_F32};
    o.o[1] = {dd, D * q.g.NP, D * q.g.NP + D, 1, 1, AFD_T_F32};
    o.o[2] = {ddt_bias, D * q.g.NP + D, D * q.g.NP + 2 * D, 1, 1, AFD_T_F32};
    return launch_column_sums(p.part_p, (long)B * q.S, D * (q.g.NP + 2), o, s);
}
