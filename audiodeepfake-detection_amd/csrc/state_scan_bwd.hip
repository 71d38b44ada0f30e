// Backward of the selective state-space scan (state_scan.h: forward formulas and lane layout).
//
//   g = dy silu(gate)  (or dy);   dgate = dy y0 silu'(gate)
//   G[t][c][n] = c[t][n] g[t][c] + X,   X = exp(delta[t+1] a) G[t+1]     (the gradient of h[t], walking backwards)
//   s1 = sum_n G b[t],   W = G exp(delta a) h[t-1],   s2 = sum_n W a
//   dx = g d + delta s1;   ddt = (s2 + x s1) softplus'(.);   da = sum_t W delta;   dd = sum g x;   ddt_bias = sum ddt
//   db[t][n] = sum_c G delta x;   dc[t][n] = sum_c h[t] g
//
// A workgroup walks its channels' blocks of 16 tokens from the last to the first.  The states inside a block come from the
// checkpoint the forward left in front of it: 16 steps forward, with every state and decay kept in registers (2 x 16 NS per
// lane), then 16 steps back.  Checkpoints every 16 tokens cost 4 bytes per token and channel at 16 states (x is 2 or 4);
// walking h backwards instead would divide by decays that go to zero, and recomputing from farther apart costs another
// exponential per state.  The sums over channels behind db and dc are a reduce-scatter over the wave: v_permlane32_swap
// and v_permlane16_swap fold two values into one register per add, so 8 values per lane over 16 channels take 17 instructions
// instead of 32; the 4 waves meet in LDS, the workgroups in a second small kernel.
#include "state_scan.h"

namespace {

using namespace afd;

// (In assembly: hipcc 7.2 hands out the first result of __builtin_amdgcn_permlane32_swap / 16_swap for both.  A swap may read
// what a vector instruction wrote two wait states before at the earliest, which the compiler cannot see to: s_nop 1.)
__device__ __forceinline__ float fold32(float a, float b) {  // lanes 0..31: a's sum over the halves, lanes 32..63: b's
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}
__device__ __forceinline__ float fold16(float a, float b) {  // even rows of 16 lanes: a's sum over row pairs, odd rows: b's
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return a + b;
}

// Sums v[0 .. 2 NS) over the wave's 64 / Q channels and stores them: value i of lane group q goes to
// out[(i / NS) NP + q NS + i % NS].
template <int Q, int NS> __device__ __forceinline__ void channel_sums(const float (&v)[2 * NS], float* out, int q) {
    constexpr int NP = Q * NS;
    const int lane = threadIdx.x & 63;
    const int b5 = lane >> 5, b4 = (lane >> 4) & 1, b3 = (lane >> 3) & 1;
    if constexpr (NS == 4) {
        const float p0 = fold32(v[0], v[1]), p1 = fold32(v[2], v[3]), p2 = fold32(v[4], v[5]), p3 = fold32(v[6], v[7]);
        const float r0 = fold16(p0, p1), r1 = fold16(p2, p3);  // state b5 + 2 b4 of b (r0) and c (r1)
        const int k = b5 + 2 * b4;
        if constexpr (Q == 16) {
            out[q * NS + k] = r0;
            out[NP + q * NS + k] = r1;
        } else {
            float r = (b3 ? r1 : r0) + dpp<0x128>(b3 ? r0 : r1);  // row_ror:8
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

// LOCAL: the gradient X that a time segment hands to the one in front of it when nothing comes from behind, and the
// segment's sum of delta.  Otherwise the full walk.
template <typename T, int Q, int NS, bool LOCAL>
__global__ void __launch_bounds__(kScanT, LOCAL ? 1 : 2) scan_bwd_kernel(const ScanArgs p) {
    constexpr int NP = Q * NS, R = kTok / Q;
    __shared__ float lds[2][kTok * 2 * NP];
    __shared__ float red[LOCAL ? 1 : 2][LOCAL ? 1 : 4 * kTok * 2 * NP];
    const ScanPlace w = scan_place<Q, NS>(p);
    const int wave = threadIdx.x >> 6;
    const int nblk = (w.n + kTok - 1) / kTok, nblk_all = (p.L + kTok - 1) / kTok;
    const int blk0 = w.s * p.seg_blocks;
    const int blk1 = min(blk0 + p.seg_blocks, nblk);
    const size_t seg = ((size_t)w.b * p.S + w.s) * p.D + w.ch;
    if (LOCAL && (w.s == 0 || blk0 >= blk1)) return;  // nobody is in front, or nothing happens here

    float a2[NS], X[NS], da[NS];
    load_states<NS>(p.a + (size_t)w.ch * p.N, w.n0, p.N, w.live, a2);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        a2[k] *= kLog2e;
        X[k] = da[k] = 0.f;
    }
    const int last = nblk > 0 ? (nblk - 1) / p.seg_blocks : 0;  // the segment with the last token
    if (!LOCAL && w.s <= last) {
        load_states<NS>(p.dstate_out ? p.dstate_out + ((size_t)w.b * p.D + w.ch) * p.N : nullptr, w.n0, p.N, w.live, X);
        if (w.live) {
            for (int s = last; s > w.s; --s) {
                const size_t at = ((size_t)w.b * p.S + s) * p.D + w.ch;
                float e[NS];
                load_vec<NS>(p.seg_h + at * NP + w.n0, e);
                const float sd = p.seg_d[at];
#pragma unroll
                for (int k = 0; k < NS; ++k) X[k] = fmaf(__builtin_amdgcn_exp2f(a2[k] * sd), X[k], e[k]);
            }
        }
    }
    const float bias = (p.dt_bias && w.live) ? p.dt_bias[w.ch] : 0.f;
    const float dskip = (p.d && w.live) ? p.d[w.ch] : 0.f;
    const T* xc = static_cast<const T*>(p.x) + (size_t)w.b * p.xb + w.ch;
    const T* tc = static_cast<const T*>(p.dt) + (size_t)w.b * p.tb + w.ch;
    const T* gc = p.gate ? static_cast<const T*>(p.gate) + (size_t)w.b * p.gb + w.ch : nullptr;
    const T* yc = static_cast<const T*>(p.dy) + (size_t)w.b * p.yb + w.ch;
    const T* br = static_cast<const T*>(p.b) + (size_t)w.b * p.bb;
    const T* cr = static_cast<const T*>(p.c) + (size_t)w.b * p.cb;
    const size_t out0 = (size_t)w.b * p.L * p.D + w.ch;
    T* dxc = static_cast<T*>(p.dx) + out0;
    T* dtc = static_cast<T*>(p.ddt) + out0;
    T* dgc = gc ? static_cast<T*>(p.dgate) + out0 : nullptr;
    float sum_delta = 0.f, sum_d = 0.f, sum_bias = 0.f;

    BcStage<T, NP> bc;
    TokLoad<T, Q> nx, nt, ng, ny;
    float nh[NS];
    const float* ck = p.ckpt + ((size_t)w.b * nblk_all * p.D + w.ch) * NP + w.n0;
    const size_t ck_row = (size_t)p.D * NP;
    auto fetch = [&](int blk) {
        const int t0 = blk * kTok;
        bc.fetch(p, br, cr, t0, w.n);
        nt.fetch(tc, p.tl, t0, w.q, w.n, w.live);
        ny.fetch(yc, p.yl, t0, w.q, w.n, w.live);
        if (gc) ng.fetch(gc, p.gl, t0, w.q, w.n, w.live);
        if (!LOCAL) {
            nx.fetch(xc, p.xl, t0, w.q, w.n, w.live);
            if (w.live) load_vec<NS>(ck + (size_t)blk * ck_row, nh);
            else {
#pragma unroll
                for (int k = 0; k < NS; ++k) nh[k] = 0.f;
            }
        }
    };
    if (blk0 < blk1) {
        fetch(blk1 - 1);
        bc.put(lds[0]);
    }
    __syncthreads();
    for (int blk = blk1 - 1; blk >= blk0; --blk) {
        const int t0 = blk * kTok, turn = (blk1 - 1 - blk) & 1;
        const float* row = lds[turn] + w.n0;
        float dl[R], dx[R], g[R], xv[R], gt[R], dyv[R], sp[R], yv[R], s1v[R], s2v[R], h0[NS];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool in = t0 + i * Q + w.q < w.n;
            const float raw = to_f32(nt.v[i]) + bias;
            dl[i] = in ? (p.softplus ? softplus_f32(raw) : raw) : 0.f;
            dyv[i] = to_f32(ny.v[i]);
            gt[i] = gc ? to_f32(ng.v[i]) : 0.f;
            g[i] = gc ? dyv[i] * gt[i] * sigmoid_f32(gt[i]) : dyv[i];
            if (!LOCAL) {
                sp[i] = p.softplus ? sigmoid_f32(raw) : 1.f;
                xv[i] = to_f32(nx.v[i]);
                dx[i] = dl[i] * xv[i];
                yv[i] = s1v[i] = s2v[i] = 0.f;
            } else {
                sum_delta += dl[i];
            }
        }
        if (!LOCAL) {
#pragma unroll
            for (int k = 0; k < NS; ++k) h0[k] = nh[k];
        }
        if (blk > blk0) fetch(blk - 1);
        if constexpr (LOCAL) {
#pragma unroll
            for (int j = kTok - 1; j >= 0; --j) {
                const int i = j / Q, ql = j % Q;
                const float de = from_lane<Q>(dl[i], ql), gj = from_lane<Q>(g[i], ql);
                float cv[NS];
                load_vec<NS>(row + j * 2 * NP + NP, cv);
#pragma unroll
                for (int k = 0; k < NS; ++k) X[k] = __builtin_amdgcn_exp2f(de * a2[k]) * fmaf(cv[k], gj, X[k]);
            }
        } else {
            float e[kTok][NS], hs[kTok][NS];
#pragma unroll
            for (int j = 0; j < kTok; ++j) {
                const int i = j / Q, ql = j % Q;
                const float de = from_lane<Q>(dl[i], ql), dxj = from_lane<Q>(dx[i], ql);
                float bv[NS];
                load_vec<NS>(row + j * 2 * NP, bv);
#pragma unroll
                for (int k = 0; k < NS; ++k) {
                    e[j][k] = __builtin_amdgcn_exp2f(de * a2[k]);
                    hs[j][k] = fmaf(e[j][k], j ? hs[j ? j - 1 : 0][k] : h0[k], dxj * bv[k]);
                }
                if (gc) {
                    float cv[NS], y = 0.f;
                    load_vec<NS>(row + j * 2 * NP + NP, cv);
#pragma unroll
                    for (int k = 0; k < NS; ++k) y = fmaf(cv[k], hs[j][k], y);
                    y = sum_lanes<Q>(y);
                    yv[i] = w.q == ql ? y : yv[i];
                }
            }
#pragma unroll
            for (int j = kTok - 1; j >= 0; --j) {
                const int i = j / Q, ql = j % Q;
                const float de = from_lane<Q>(dl[i], ql), dxj = from_lane<Q>(dx[i], ql), gj = from_lane<Q>(g[i], ql);
                float bv[NS], cv[NS], v[2 * NS], s1 = 0.f, s2 = 0.f;
                load_vec<NS>(row + j * 2 * NP, bv);
                load_vec<NS>(row + j * 2 * NP + NP, cv);
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
                s1 = sum_lanes<Q>(s1);
                s2 = sum_lanes<Q>(s2);
                s1v[i] = w.q == ql ? s1 : s1v[i];
                s2v[i] = w.q == ql ? s2 : s2v[i];
                channel_sums<Q, NS>(v, &red[turn][(wave * kTok + j) * 2 * NP], w.q);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int t = t0 + i * Q + w.q;
                const bool in = t < w.n;
                // (a2 carries log2 e, which s2 does not want)
                const float ddt = in ? fmaf(xv[i], s1v[i], s2v[i] * (1.f / kLog2e)) * sp[i] : 0.f;
                sum_bias += ddt;
                sum_d = fmaf(g[i], xv[i], sum_d);
                if (w.live && t < p.L) {
                    dxc[(size_t)t * p.D] = from_f32<T>(in ? fmaf(g[i], dskip, dl[i] * s1v[i]) : 0.f);
                    dtc[(size_t)t * p.D] = from_f32<T>(ddt);
                    if (gc) {
                        const float s = sigmoid_f32(gt[i]), y0 = fmaf(dskip, xv[i], yv[i]);
                        dgc[(size_t)t * p.D] = from_f32<T>(in ? dyv[i] * y0 * s * (1.f + gt[i] * (1.f - s)) : 0.f);
                    }
                }
            }
        }
        if (blk > blk0) bc.put(lds[turn ^ 1]);
        __syncthreads();
        if constexpr (!LOCAL) {
            // the 4 waves' sums over their channels; the other half of `red` is the next block's
            float* dst = p.part_bc + (((size_t)w.cb * p.B + w.b) * p.L + t0) * 2 * NP;
            for (int i = threadIdx.x; i < kTok * 2 * NP; i += kScanT) {
                if (t0 + i / (2 * NP) < w.n) {
                    const float* r = red[turn] + i;
                    constexpr int kW = kTok * 2 * NP;
                    dst[i] = (r[0] + r[kW]) + (r[2 * kW] + r[3 * kW]);
                }
            }
        }
    }
    if constexpr (LOCAL) {
        sum_delta = sum_lanes<Q>(sum_delta);
        if (w.live) {
            store_vec<NS>(p.seg_h + seg * NP + w.n0, X);
            if (w.q == 0) p.seg_d[seg] = sum_delta;
        }
    } else {
        const int tail0 = max(blk0, blk1) * kTok, tail1 = min((blk0 + p.seg_blocks) * kTok, p.L);
        const T zero = from_f32<T>(0.f);
        for (int t = tail0 + w.q; t < tail1; t += Q) {
            if (w.live) {
                dxc[(size_t)t * p.D] = zero;
                dtc[(size_t)t * p.D] = zero;
                if (gc) dgc[(size_t)t * p.D] = zero;
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
            store_states<NS>(p.dstate + ((size_t)w.b * p.D + w.ch) * p.N, w.n0, p.N, w.live, X);
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
