// Backward of the selective state-space scan (state_scan.h: forward formulas and lane layout).
//
//   g = dy silu(gate)  (or dy);   dgate = dy y0 silu'(gate)
//   G[t][c][n] = c[t][n] g[t][c] + X,   X = exp(delta[t+1] a) G[t+1]     (the gradient of h[t], walking backwards)
//   s1 = sum_n G b[t],   W = G exp(delta a) h[t-1],   s2 = sum_n W a
//   dx = g d + delta s1;   ddt = (s2 + x s1) softplus'(.);   da = sum_t W delta;   dd = sum g x;   ddt_bias = sum ddt
//   db[t][n] = sum_c G delta x;   dc[t][n] = sum_c h[t] g
//
// A workgroup walks its channels' blocks of 8 tokens from the last to the first.  The states inside a block come from the
// checkpoint the forward left in front of it: 8 steps forward, with every state and decay kept in registers (2 x 8 NS per
// lane), then 8 steps back.  Checkpoints every 8 tokens cost 8 bytes per token and channel at 16 states (x is 2 or 4); with
// 16 tokens the history alone took half the register file, two waves per SIMD were left and three quarters of the time went
// into waiting (1.13 ms at 4 x 4096 x 2048 bf16).  Walking h backwards instead would divide by decays that go to zero, and
// recomputing from farther apart costs another exponential per state.  The sums over channels behind db and dc are a
// reduce-scatter over the wave: v_permlane32_swap and v_permlane16_swap fold two values into one register per add, so 8
// values per lane over 16 channels take 17 instructions instead of 32; the 4 waves meet in LDS, the workgroups in a second
// small kernel.
// Bound by vector instruction issue: 25 instructions per token, channel and state, 16 of them the formulas above, the rest
// broadcasts and sums over lanes.  Measured, 16 states: 128 x 101 x 1024 fp32 227 us (issue 81 % of the time); 4 x 4096 x 2048
// bf16 in 8 time segments 136 + 490 us (95 and 89 %) + 13 for the workgroups' db and dc + 5 for the parameters' sums.
#include "state_scan.h"

namespace {

using namespace afd;

constexpr int kBwdWaves = 2;  // waves per SIMD the registers are cut for

// (In assembly: hipcc 7.2 hands out the first result of __builtin_amdgcn_permlane32_swap / 16_swap for both, and does not form
// additions that write some banks of lanes only.  Swaps and DPP reads may follow a vector instruction that wrote their source
// after two wait states at the earliest, which the compiler cannot see to: s_nop 1 in front of each group.)
__device__ __forceinline__ float fold32(float a, float b) {  // lanes 0..31: a's sum over the halves, lanes 32..63: b's
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}
__device__ __forceinline__ float fold16(float a, float b) {  // even rows of 16 lanes: a's sum over row pairs, odd rows: b's
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}
// lanes 0..7 of a row: lo[i]'s sum over the row's halves, lanes 8..15: hi[i]'s
__device__ __forceinline__ void fold8(const float* lo, const float* hi, float (&r)[4]) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %2, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %3, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
        : "v"(lo[0]), "v"(lo[1]), "v"(lo[2]), "v"(lo[3]), "v"(hi[0]), "v"(hi[1]), "v"(hi[2]), "v"(hi[3]));
}
// fold32 of two pairs
__device__ __forceinline__ void fold32x2(float a, float b, float c, float d, float& r0, float& r1) {
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_permlane32_swap_b32 %2, %3" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
    r0 = a + b;
    r1 = c + d;
}

// Sums v[0 .. 2 NS) over the wave's 64 / Q channels and stores them: value i of lane group q goes to
// out[(i / NS) NP + q NS + i % NS].
template <int Q, int NS> __device__ __forceinline__ void channel_sums(const float (&v)[2 * NS], float* out, int q) {
    constexpr int NP = Q * NS;
    const int lane = threadIdx.x & 63;
    const int b5 = lane >> 5, b4 = (lane >> 4) & 1, b3 = (lane >> 3) & 1;
    if constexpr (NS == 4) {
        const int k = b5 + 2 * b4;
        float r0, r1;
        if constexpr (Q == 16) {
            float p0, p1;
            fold32x2(v[0], v[1], v[2], v[3], r0, r1);
            fold32x2(v[4], v[5], v[6], v[7], p0, p1);
            out[q * NS + k] = fold16(r0, r1);
            out[NP + q * NS + k] = fold16(p0, p1);
        } else {
            float f[4];
            fold8(v, v + 4, f);  // lower half rows: b's sums, upper: c's
            fold32x2(f[0], f[1], f[2], f[3], r0, r1);
            float r = fold16(r0, r1);
            if constexpr (Q == 4) r += dpp<0x1b>(dpp<0x141>(r));  // lane ^ 4 = half mirror, then quad_perm [3, 2, 1, 0]
            out[b3 * NP + q * NS + k] = r;
        }
    } else if constexpr (NS == 2) {
        static_assert(NS != 2 || Q == 4, "lanes per channel");
        float r = fold16(fold32(v[0], v[1]), fold32(v[2], v[3]));
        r += dpp<0x128>(r);
        r += dpp<0x1b>(dpp<0x141>(r));
        out[b4 * NP + q * NS + b5] = r;
    } else {
        static_assert(NS != 1 || Q == 4, "lanes per channel");
        float r = fold32(v[0], v[1]);
        r = fold16(r, r);
        r += dpp<0x128>(r);
        r += dpp<0x1b>(dpp<0x141>(r));
        out[b5 * NP + q] = r;
    }
}

// The lane's own token's sum over the channel's lanes, tokens arriving one by one (upwards; down: downwards): collected
// and reduced Q at a time where a block holds Q tokens, one by one where it does not (Q = 16).
template <int Q> __device__ __forceinline__ void own_sum(float v, int ql, float (&part)[Q], float& own) {
    if constexpr (Q > kTokB) {
        v = sum_lanes<Q>(v);
        own = (int)(threadIdx.x & (Q - 1)) == ql ? v : own;
    } else {
        part[ql] = v;
        if (ql == Q - 1) own = scatter_lanes<Q>(part);
    }
}
template <int Q> __device__ __forceinline__ void own_sum_down(float v, int ql, float (&part)[Q], float& own) {
    if constexpr (Q > kTokB) {
        v = sum_lanes<Q>(v);
        own = (int)(threadIdx.x & (Q - 1)) == ql ? v : own;
    } else {
        part[ql] = v;
        if (ql == 0) own = scatter_lanes<Q>(part);
    }
}

// LOCAL: the gradient X that a time segment hands to the one in front of it when nothing comes from behind, and the
// segment's sum of delta.  Otherwise the full walk.
template <typename T, int Q, int NS, bool LOCAL>
__global__ void __launch_bounds__(kScanT, LOCAL ? 4 : kBwdWaves) scan_bwd_kernel(const ScanArgs p) {
    constexpr int NP = Q * NS, TB = kTokB, R = TB > Q ? TB / Q : 1;
    constexpr int TS = 2 * TB;  // tokens between barriers: b and c rows come, and sums over channels go, for TS at a time
    __shared__ __attribute__((aligned(16))) float lds[2][TS * 2 * NP];
    __shared__ float red[LOCAL ? 1 : 2][LOCAL ? 1 : 4 * TS * 2 * NP];
    const ScanPlace w = scan_place<Q, NS>(p);
    const int wave = threadIdx.x >> 6;
    const int start = w.s * p.seg;
    const int end = min(start + p.seg, w.n);
    const size_t seg = ((size_t)w.b * p.S + w.s) * p.D + w.cl;
    if (LOCAL && (w.s == 0 || start >= end)) return;  // nobody is in front, or nothing happens here

    float a2[NS], X[NS], da[NS];
    load_states<NS>(p.a + (size_t)w.cl * p.N, w.n0, p.N, true, a2);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        a2[k] = log2_decay(a2[k]);
        X[k] = da[k] = 0.f;
    }
    const int last = w.n > 0 ? (w.n - 1) / p.seg : 0;  // the segment with the last token
    if (!LOCAL && w.s <= last) {
        load_states<NS>(p.dstate_out ? p.dstate_out + ((size_t)w.b * p.D + w.cl) * p.N : nullptr, w.n0, p.N, w.live, X);
        for (int s = last; s > w.s; --s) {
            const size_t at = ((size_t)w.b * p.S + s) * p.D + w.cl;
            float e[NS];
            load_vec<NS>(p.seg_h + at * NP + w.n0, e);
            carry<NS>(a2, p.seg_d[at], e, X);
        }
        if (!w.live) {  // lanes behind the last channel add nothing to db and dc
#pragma unroll
            for (int k = 0; k < NS; ++k) X[k] = 0.f;
        }
    }
    const float bias = p.dt_bias ? p.dt_bias[w.cl] : 0.f;
    const float dskip = p.d ? p.d[w.cl] : 0.f;
    const bool gated = p.gate;
    const T* xb = static_cast<const T*>(p.x) + (size_t)w.b * p.xb;
    const T* tb = static_cast<const T*>(p.dt) + (size_t)w.b * p.tb;
    const T* gb = gated ? static_cast<const T*>(p.gate) + (size_t)w.b * p.gb : nullptr;
    const T* yb = static_cast<const T*>(p.dy) + (size_t)w.b * p.yb;
    const T* br = static_cast<const T*>(p.b) + (size_t)w.b * p.bb;
    const T* cr = static_cast<const T*>(p.c) + (size_t)w.b * p.cb;
    const int tq = min(w.q, TB - 1);  // (16 lanes per channel, 8 tokens: the upper lanes have none of their own)
    const unsigned chan = (unsigned)w.cl * sizeof(T);
    const unsigned xo = chan + (unsigned)(tq * p.xl * sizeof(T)), to = chan + (unsigned)(tq * p.tl * sizeof(T));
    const unsigned yo = chan + (unsigned)(tq * p.yl * sizeof(T));
    const unsigned go = gated ? chan + (unsigned)(tq * p.gl * sizeof(T)) : 0u;
    const unsigned oo = chan + (unsigned)(tq * p.D * sizeof(T));
    T* dxb = static_cast<T*>(p.dx) + (size_t)w.b * p.L * p.D;
    T* dtb = static_cast<T*>(p.ddt) + (size_t)w.b * p.L * p.D;
    T* dgb = gated ? static_cast<T*>(p.dgate) + (size_t)w.b * p.L * p.D : nullptr;
    float sum_delta = 0.f, sum_d = 0.f, sum_bias = 0.f;

    BcStage<T, NP, TS> bc;
    TokLoad<T, Q, TB> nx, nt, ng, ny;
    float nh[NS];
    const float* ck = p.ckpt + (size_t)w.b * ((p.L + kCkpt - 1) / kCkpt) * p.D * NP;
    const unsigned co = (unsigned)(w.cl * NP + w.n0) * 4u;
    auto fetch = [&](int t0) {
        const int left = w.n - t0;
        if (left >= TB) {
            nt.full(tb + (size_t)t0 * p.tl, p.tl, to);
            ny.full(yb + (size_t)t0 * p.yl, p.yl, yo);
            if (gated) ng.full(gb + (size_t)t0 * p.gl, p.gl, go);
            if (!LOCAL) nx.full(xb + (size_t)t0 * p.xl, p.xl, xo);
        } else {
            nt.tail(tb + (size_t)t0 * p.tl, p.tl, left, w.q, chan);
            ny.tail(yb + (size_t)t0 * p.yl, p.yl, left, w.q, chan);
            if (gated) ng.tail(gb + (size_t)t0 * p.gl, p.gl, left, w.q, chan);
            if (!LOCAL) nx.tail(xb + (size_t)t0 * p.xl, p.xl, left, w.q, chan);
        }
        if (!LOCAL) load_vec<NS>(reinterpret_cast<const float*>(reinterpret_cast<const char*>(ck + (size_t)(t0 / kCkpt) * p.D * NP) + co), nh);
    };
    const int top = start < end ? start + (end - 1 - start) / TB * TB : start - TB;  // the last block's first token
    if (start < end) {  // (start is a multiple of TS)
        const int ts = top / TS * TS;
        bc.fetch(p, br, cr, ts, w.n);
        fetch(top);
        bc.put(lds[0], ts, w.n, p.N);
    }
    __syncthreads();
    int turn = 0;
    for (int t0 = top; t0 >= start; t0 -= TB) {
        const int half = t0 % TS;  // 0 or TB
        const float* row = lds[turn] + half * 2 * NP + w.n0;
        if (half == 0 && t0 > start) bc.fetch(p, br, cr, t0 - TS, w.n);
        float dl[R], dx[R], g[R], xv[R], gt[R], dyv[R], sp[R], yv[R], s1v[R], s2v[R], h0[NS];
        const bool whole = t0 + TB <= w.n;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float raw = to_f32(nt.v[i]) + bias;
            dl[i] = p.softplus ? softplus_f32(raw) : raw;
            dyv[i] = to_f32(ny.v[i]);
            gt[i] = gated ? to_f32(ng.v[i]) : 0.f;
            g[i] = gated ? dyv[i] * gt[i] * sigmoid_f32(gt[i]) : dyv[i];
            if (!LOCAL) {
                sp[i] = p.softplus ? sigmoid_f32(raw) : 1.f;
                xv[i] = to_f32(nx.v[i]);
                dx[i] = dl[i] * xv[i];
                yv[i] = s1v[i] = s2v[i] = 0.f;
            }
        }
        if (!whole || !w.live || Q > TB) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const bool in = w.live && i * Q + w.q < TB && t0 + i * Q + w.q < w.n;
                dl[i] = in ? dl[i] : 0.f;
                g[i] = in ? g[i] : 0.f;
                if (!LOCAL) {
                    dx[i] = in ? dx[i] : 0.f;
                    xv[i] = in ? xv[i] : 0.f;
                }
            }
        }
        if (LOCAL) {
#pragma unroll
            for (int i = 0; i < R; ++i) sum_delta += dl[i];
        } else {
#pragma unroll
            for (int k = 0; k < NS; ++k) h0[k] = w.live ? nh[k] : 0.f;
        }
        if (t0 > start) fetch(t0 - TB);
        if constexpr (LOCAL) {
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = TB - 1; j >= 0; --j) {
                const int i = j / Q, ql = j % Q;
                const float de = from_lane<Q>(dl[i], ql), gj = from_lane<Q>(g[i], ql);
                float cv[NS];
                load_vec<NS>(row + j * 2 * NP + NP, cv);
#pragma unroll
                for (int k = 0; k < NS; ++k) X[k] = __builtin_amdgcn_exp2f(de * a2[k]) * fmaf(cv[k], gj, X[k]);
            }
            __builtin_amdgcn_s_setprio(0);
        } else {
            // The steps go first at the SIMD, in front of what other waves do between their blocks, and the steps back in front of
            // those forward: waves take turns instead of moving in step.  545 to 490 us at 4 x 4096 x 2048 bf16; steps back alone
            // 494, all alike 515.
            __builtin_amdgcn_s_setprio(1);
            float e[TB][NS], hs[TB][NS], part1[Q], part2[Q];
            float nb[NS], nc[NS];  // the next token's rows, asked for one token ahead
            load_vec<NS>(row, nb);
            load_vec<NS>(row + NP, nc);
#pragma unroll
            for (int j = 0; j < TB; ++j) {
                const int i = j / Q, ql = j % Q;
                const float de = from_lane<Q>(dl[i], ql), dxj = from_lane<Q>(dx[i], ql);
                float bv[NS], cv[NS];
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    bv[k] = nb[k];
                    cv[k] = nc[k];
                }
                const int ahead = j + 1 < TB ? j + 1 : TB - 1;
                load_vec<NS>(row + ahead * 2 * NP, nb);
                load_vec<NS>(row + ahead * 2 * NP + NP, nc);
                hold_lds();
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    e[j][k] = __builtin_amdgcn_exp2f(de * a2[k]);
                    hs[j][k] = fmaf(e[j][k], j ? hs[j ? j - 1 : 0][k] : h0[k], dxj * bv[k]);
                }
                if (gated) {
                    float y = 0.f;
#pragma unroll
                    for (int k = 0; k < NS; ++k) y = fmaf(cv[k], hs[j][k], y);
                    own_sum<Q>(y, ql, part1, yv[i]);
                }
            }
            __builtin_amdgcn_s_setprio(2);
#pragma unroll
            for (int j = TB - 1; j >= 0; --j) {
                const int i = j / Q, ql = j % Q;
                const float de = from_lane<Q>(dl[i], ql), dxj = from_lane<Q>(dx[i], ql), gj = from_lane<Q>(g[i], ql);
                float bv[NS], cv[NS], v[2 * NS], s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    bv[k] = nb[k];
                    cv[k] = nc[k];
                }
                if (j > 0) {
                    load_vec<NS>(row + (j - 1) * 2 * NP, nb);
                    load_vec<NS>(row + (j - 1) * 2 * NP + NP, nc);
                }
                hold_lds();
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    const float G = fmaf(cv[k], gj, X[k]);
                    X[k] = e[j][k] * G;
                    const float W = X[k] * (j ? hs[j ? j - 1 : 0][k] : h0[k]);
                    s1 = fmaf(G, bv[k], s1);
                    s2 = fmaf(W, a2[k], s2);
                    da[k] = fmaf(W, de, da[k]);
                    v[k] = G * dxj;
                    v[NS + k] = hs[j][k] * gj;
                }
                own_sum_down<Q>(s1, ql, part1, s1v[i]);
                own_sum_down<Q>(s2, ql, part2, s2v[i]);
                channel_sums<Q, NS>(v, &red[turn][(wave * TS + half + j) * 2 * NP], w.q);
            }
            __builtin_amdgcn_s_setprio(0);
            loads_arrived();
            T odx[R], odt[R], odg[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                // (a2 carries log2 e, which s2 does not want)
                const float ddt = fmaf(xv[i], s1v[i], s2v[i] * (1.f / kLog2e)) * sp[i];
                odt[i] = from_f32<T>(ddt);
                odx[i] = from_f32<T>(fmaf(g[i], dskip, dl[i] * s1v[i]));
                sum_d = fmaf(g[i], xv[i], sum_d);
                if (gated) {
                    const float s = sigmoid_f32(gt[i]), y0 = fmaf(dskip, xv[i], yv[i]);
                    odg[i] = from_f32<T>(dyv[i] * y0 * s * (1.f + gt[i] * (1.f - s)));
                }
                if ((whole && Q <= TB) || (i * Q + w.q < TB && t0 + i * Q + w.q < w.n)) sum_bias += ddt;
            }
            if (whole) {
                if (w.live && (Q <= TB || w.q < TB)) {
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const size_t at = (size_t)(t0 + i * Q) * p.D;
                        *reinterpret_cast<T*>(reinterpret_cast<char*>(dxb + at) + oo) = odx[i];
                        *reinterpret_cast<T*>(reinterpret_cast<char*>(dtb + at) + oo) = odt[i];
                        if (gated) *reinterpret_cast<T*>(reinterpret_cast<char*>(dgb + at) + oo) = odg[i];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int t = t0 + i * Q + w.q;
                    if (w.live && i * Q + w.q < TB && t < p.L) {
                        const size_t at = (size_t)t * p.D + w.ch;
                        const bool in = t < w.n;
                        dxb[at] = in ? odx[i] : from_f32<T>(0.f);
                        dtb[at] = in ? odt[i] : from_f32<T>(0.f);
                        if (gated) dgb[at] = in ? odg[i] : from_f32<T>(0.f);
                    }
                }
            }
        }
        if (half != 0) continue;
        if (t0 > start) bc.put(lds[turn ^ 1], t0 - TS, w.n, p.N);
        __syncthreads();
        if constexpr (!LOCAL) {
            // the 4 waves' sums over their channels; the other half of `red` is the next tokens'
            float* dst = p.part_bc + (((size_t)w.cb * p.B + w.b) * p.L + t0) * 2 * NP;
            for (int i = threadIdx.x; i < TS * 2 * NP; i += kScanT) {
                if (t0 + TS <= w.n || t0 + i / (2 * NP) < w.n) {
                    const float* r = red[turn] + i;
                    constexpr int kW = TS * 2 * NP;
                    dst[i] = (r[0] + r[kW]) + (r[2 * kW] + r[3 * kW]);
                }
            }
        }
        turn ^= 1;
    }
    if constexpr (LOCAL) {
        sum_delta = sum_lanes<Q>(sum_delta);
        if (w.live) {
            store_vec<NS>(p.seg_h + seg * NP + w.n0, X);
            if (w.q == 0) p.seg_d[seg] = sum_delta;
        }
    } else {
        const int done = start < end ? top + TB : start, stop = min(start + p.seg, p.L);
        const T zero = from_f32<T>(0.f);
        for (int t = done + w.q; t < stop; t += Q) {
            if (w.live) {
                const size_t at = (size_t)t * p.D + w.ch;
                dxb[at] = zero;
                dtb[at] = zero;
                if (gated) dgb[at] = zero;
            }
        }
        sum_d = sum_lanes<Q>(sum_d);
        sum_bias = sum_lanes<Q>(sum_bias);
        if (w.live) {
            float* part = p.part_p + ((size_t)w.b * p.S + w.s) * ((size_t)p.D * (NP + 2));
#pragma unroll
            for (int k = 0; k < NS; ++k) part[(size_t)w.ch * NP + w.n0 + k] = da[k];
            if (w.q == 0) {
                part[(size_t)p.D * NP + w.ch] = sum_d;
                part[(size_t)p.D * (NP + 1) + w.ch] = sum_bias;
            }
        }
        if (p.dstate && w.s == 0)
            store_states<NS>(p.dstate + ((size_t)w.b * p.D + w.cl) * p.N, w.n0, p.N, w.live, X);
    }
}

// db, dc [B][L][N]: the sums over the workgroups of a row, zero behind the last token.
template <typename T>
__global__ void __launch_bounds__(256) scan_bc_kernel(const ScanArgs p, T* __restrict__ db, T* __restrict__ dc, int NP) {
    const size_t rows = (size_t)p.B * p.L, all = rows * 2 * NP;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (size_t)gridDim.x * 256) {
        const size_t r = i / (2 * NP);
        const int col = (int)(i - r * 2 * NP), n = col < NP ? col : col - NP;
        if (n >= p.N) continue;
        const int b = (int)(r / p.L), t = (int)(r - (size_t)b * p.L);
        float v = 0.f;
        if (t < scan_rows(p.lengths, b, p.L)) {
            int k = 0;
            float u[4] = {0.f, 0.f, 0.f, 0.f};
            for (; k + 4 <= p.nb; k += 4) {
#pragma unroll
                for (int m = 0; m < 4; ++m) u[m] += p.part_bc[(size_t)(k + m) * all + i];
            }
            for (; k < p.nb; ++k) u[0] += p.part_bc[(size_t)k * all + i];
            v = (u[0] + u[1]) + (u[2] + u[3]);
        }
        (col < NP ? db : dc)[r * p.N + n] = from_f32<T>(v);
    }
}

template <typename T, int Q, int NS> int launch(const ScanArgs& p, hipStream_t s) {
    const unsigned grid = (unsigned)((long)p.B * p.S * p.nb);
    if (p.S > 1) hipLaunchKernelGGL((scan_bwd_kernel<T, Q, NS, true>), dim3(grid), dim3(kScanT), 0, s, p);
    hipLaunchKernelGGL((scan_bwd_kernel<T, Q, NS, false>), dim3(grid), dim3(kScanT), 0, s, p);
    return check_launch("scan_bwd_kernel");
}
template <typename T> int launch_n(const ScanArgs& p, hipStream_t s) {
    const ScanShape g = scan_shape(p.N);
    if (g.NP == 4) return launch<T, 4, 1>(p, s);
    if (g.NP == 8) return launch<T, 4, 2>(p, s);
    if (g.NP == 16) return launch<T, 4, 4>(p, s);
    if (g.NP == 32) return launch<T, 8, 4>(p, s);
    return launch<T, 16, 4>(p, s);
}
template <typename T> int bc(const ScanArgs& p, void* db, void* dc, hipStream_t s) {
    const int NP = scan_shape(p.N).NP;
    const size_t all = (size_t)p.B * p.L * 2 * NP;
    const size_t grid = (all + 255) / 256;
    hipLaunchKernelGGL(scan_bc_kernel<T>, dim3((unsigned)(grid < 65536 ? grid : 65536)), dim3(256), 0, s, p,
                       static_cast<T*>(db), static_cast<T*>(dc), NP);
    return check_launch("scan_bc_kernel");
}

}  // namespace

int afd::scan_backward_launch(const ScanArgs& p, int dtype, hipStream_t s) {
    if (dtype == AFD_T_F32) return launch_n<float>(p, s);
    if (dtype == AFD_T_BF16) return launch_n<bf16_t>(p, s);
    return launch_n<f16_t>(p, s);
}

int afd::scan_bc_gradients(const ScanArgs& p, void* db, void* dc, int dtype, hipStream_t s) {
    if (dtype == AFD_T_F32) return bc<float>(p, db, dc, s);
    if (dtype == AFD_T_BF16) return bc<bf16_t>(p, db, dc, s);
    return bc<f16_t>(p, db, dc, s);
}
