// Selective state-space scan: argument block and device helpers shared by state_scan_fwd.hip and state_scan_bwd.hip.
//
//   delta = softplus(dt + dt_bias)  (or dt + dt_bias)
//   h[t][c][n] = exp(delta[t][c] a[c][n]) h[t-1][c][n] + delta[t][c] b[t][n] x[t][c]
//   y0[t][c]   = sum_n c[t][n] h[t][c][n] + d[c] x[t][c],      y = y0  or  y0 silu(gate)
//
// Lane layout (both directions): a lane owns NS (<= 4) states of one channel, Q neighbouring lanes own the channel, so a wave
// holds 64 / Q channels and the states live in registers for the whole walk over time.  The Q lanes of a channel also
// share its per-token work: time advances in blocks of 16 tokens, lane q of a channel loads tokens q, q + Q, ... and
// computes their softplus / gate ONCE, and the value a token needs is broadcast to the channel's lanes by a DPP move.  Against
// one lane per channel this quarters the transcendental work that is not exp(delta a), and it gives 4 x the waves from
// the same rows, which is what a scan lacks: its only parallel axes are batch and channel.
// The b and c rows are the same for every channel: a workgroup (4 waves) stages a block's rows in LDS as fp32, double
// buffered, and each lane reads its own NS of them as one vector.
#pragma once

#include "seq_common.h"

namespace afd {

constexpr int kTokF = 16;      // tokens per block, forward
constexpr int kTokB = 8;       // ... and backward, where a block's states and decays stay in registers
constexpr int kCkpt = kTokB;   // tokens between the states that the forward keeps for the backward
constexpr int kScanT = 256;    // threads per workgroup: 4 waves

struct ScanArgs {
    const void *x, *dt, *b, *c, *gate, *dy;
    long xb, xl, tb, tl, bb, bl, cb, cl, gb, gl, yb, yl;  // batch / row strides in elements; the last axis is contiguous
    const float *a, *d, *dt_bias, *state;
    const int* lengths;
    void* y;
    float* state_out;
    float* ckpt;  // [B][ceil(L / kCkpt)][D][NP]: the state in front of every kCkpt tokens (written for training)
    float* seg_h;  // [B][S][D][NP]: what a time segment leaves on its own (forward: state, backward: gradient)
    float* seg_d;  // [B][S][D]: the segment's sum of delta
    int B, L, D, N, softplus;
    int S, seg;  // time segments and tokens per segment (a multiple of kTokF)
    int nb;             // workgroups per row of channels
    // backward only
    const float* dstate_out;
    void *dx, *ddt, *dgate;
    float* dstate;
    float* part_bc;  // [nb][B][L][2 NP]
    float* part_p;   // [B S][D NP + 2 D]: da, dd, ddt_bias
};

// Everything below is device code.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// the value that lane j of the channel's Q lanes holds, to all of them (j is a constant once the callers are unrolled)
template <int Q> __device__ __forceinline__ float from_lane(float v, int j) {
    if constexpr (Q == 4) {
        switch (j) {  // quad_perm [j, j, j, j]
            case 0: return dpp<0x00>(v);
            case 1: return dpp<0x55>(v);
            case 2: return dpp<0xaa>(v);
            default: return dpp<0xff>(v);
        }
    } else if constexpr (Q == 16) {
        switch (j) {  // row_newbcast:j
            case 0: return dpp<0x150>(v);
            case 1: return dpp<0x151>(v);
            case 2: return dpp<0x152>(v);
            case 3: return dpp<0x153>(v);
            case 4: return dpp<0x154>(v);
            case 5: return dpp<0x155>(v);
            case 6: return dpp<0x156>(v);
            case 7: return dpp<0x157>(v);
            case 8: return dpp<0x158>(v);
            case 9: return dpp<0x159>(v);
            case 10: return dpp<0x15a>(v);
            case 11: return dpp<0x15b>(v);
            case 12: return dpp<0x15c>(v);
            case 13: return dpp<0x15d>(v);
            case 14: return dpp<0x15e>(v);
            default: return dpp<0x15f>(v);
        }
    } else {
        static_assert(Q == 8, "lanes per channel");
        float lo, hi;  // the two channels of a row of 16 lanes
        switch (j) {
            case 0: lo = dpp<0x150>(v); hi = dpp<0x158>(v); break;
            case 1: lo = dpp<0x151>(v); hi = dpp<0x159>(v); break;
            case 2: lo = dpp<0x152>(v); hi = dpp<0x15a>(v); break;
            case 3: lo = dpp<0x153>(v); hi = dpp<0x15b>(v); break;
            case 4: lo = dpp<0x154>(v); hi = dpp<0x15c>(v); break;
            case 5: lo = dpp<0x155>(v); hi = dpp<0x15d>(v); break;
            case 6: lo = dpp<0x156>(v); hi = dpp<0x15e>(v); break;
            default: lo = dpp<0x157>(v); hi = dpp<0x15f>(v); break;
        }
        return (threadIdx.x & 8) ? hi : lo;
    }
}

// sum over the Q lanes of a channel, in all of them
template <int Q> __device__ __forceinline__ float sum_lanes(float v) {
    v += dpp<0xb1>(v);  // quad_perm [1, 0, 3, 2]
    v += dpp<0x4e>(v);  // quad_perm [2, 3, 0, 1]
    if constexpr (Q >= 8) v += dpp<0x141>(v);   // row_half_mirror: the quads are uniform by now
    if constexpr (Q >= 16) v += dpp<0x140>(v);  // row_mirror
    return v;
}

// Sums of v[0 .. Q) over the Q lanes of a channel; lane q gets that of v[q].  Every step halves the values, so it takes
// 3 (Q - 1) instructions where summing each in full and picking one's own takes Q (log2 Q + 1).
template <int Q> __device__ __forceinline__ float scatter_lanes(float (&v)[Q]) {
    const int q = threadIdx.x & (Q - 1);
    if constexpr (Q == 16) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // row_mirror: lane q meets lane 15 - q
            const float lo = v[i] + dpp<0x140>(v[i]), hi = v[i + 8] + dpp<0x140>(v[i + 8]);
            v[i] = (q & 8) ? hi : lo;
        }
    }
    if constexpr (Q >= 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // row_half_mirror: q meets 7 - q
            const float lo = v[i] + dpp<0x141>(v[i]), hi = v[i + 4] + dpp<0x141>(v[i + 4]);
            v[i] = (q & 4) ? hi : lo;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // quad_perm [2, 3, 0, 1]
        const float lo = v[i] + dpp<0x4e>(v[i]), hi = v[i + 2] + dpp<0x4e>(v[i + 2]);
        v[i] = (q & 2) ? hi : lo;
    }
    const float lo = v[0] + dpp<0xb1>(v[0]), hi = v[1] + dpp<0xb1>(v[1]);  // quad_perm [1, 0, 3, 2]
    return (q & 1) ? hi : lo;
}

template <int NS> struct Vec;
template <> struct Vec<1> { typedef float type; };
template <> struct Vec<2> { typedef float type __attribute__((ext_vector_type(2))); };
template <> struct Vec<4> { typedef float type __attribute__((ext_vector_type(4))); };

template <int NS> __device__ __forceinline__ void load_vec(const float* p, float (&r)[NS]) {
    const typename Vec<NS>::type v = *reinterpret_cast<const typename Vec<NS>::type*>(p);
    if constexpr (NS == 1) r[0] = v;
    else {
#pragma unroll
        for (int k = 0; k < NS; ++k) r[k] = v[k];
    }
}
template <int NS> __device__ __forceinline__ void store_vec(float* p, const float (&r)[NS]) {
    typename Vec<NS>::type v;
    if constexpr (NS == 1) v = r[0];
    else {
#pragma unroll
        for (int k = 0; k < NS; ++k) v[k] = r[k];
    }
    *reinterpret_cast<typename Vec<NS>::type*>(p) = v;
}

// rows of N floats that need not be aligned or padded (the caller's state, a): n0 = this lane's first state
template <int NS> __device__ __forceinline__ void load_states(const float* p, int n0, int N, bool live, float (&r)[NS]) {
#pragma unroll
    for (int k = 0; k < NS; ++k) r[k] = (live && p && n0 + k < N) ? p[n0 + k] : 0.f;
}
template <int NS> __device__ __forceinline__ void store_states(float* p, int n0, int N, bool live, const float (&r)[NS]) {
#pragma unroll
    for (int k = 0; k < NS; ++k)
        if (live && n0 + k < N) p[n0 + k] = r[k];
}

// a log2 e, finite from below: a of -inf forgets the state at every token, and tokens that only hold it (padding in the last block,
// lanes behind the last channel: delta = 0) would make 0 x inf of it.
__device__ __forceinline__ float log2_decay(float a) {
    const float v = a * kLog2e;
    return v < -3.402823466e38f ? -3.402823466e38f : v;
}

// The carry over a time segment: v exp(a sum delta) + e, a2 = a log2 e.  A whole segment's decay leaves the range of fp32 where
// the value that it multiplies does not (growing decays over a stretch of zeros, a large state that fades): half of it is
// applied at a time, and no half is infinite, so that zero stays zero as it does token by token.
template <int NS> __device__ __forceinline__ void carry(const float (&a2)[NS], float sum_delta, const float (&e)[NS], float (&v)[NS]) {
#pragma unroll
    for (int k = 0; k < NS; ++k) {
        const float f = __builtin_amdgcn_exp2f(fminf(0.5f * a2[k] * sum_delta, 127.f));  // (NaN comes in through e)
        v[k] = fmaf(f, f * v[k], e[k]);
    }
}

__device__ __forceinline__ int scan_rows(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > L ? L : n);
}

// Loads go to a uniform base (advanced by scalar instructions) plus a 32-bit byte offset of the lane that never changes, so
// an element costs one instruction.  A full block reads without looking; in the last block of a sequence rows behind it are
// replaced by its last row, and the caller puts zeros in the place of what they give.
template <typename T> __device__ __forceinline__ T load_at(const T* base, unsigned off) {
    return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off);
}

// The b and c rows of one block on their way into LDS: E values per thread, fetched early and written late.
template <typename T, int NP, int TOK> struct BcStage {
    static constexpr int kAll = TOK * 2 * NP;
    static constexpr int E = (kAll + kScanT - 1) / kScanT;
    T v[E];
    // thread's element e: token (e kScanT + tid) / (2 NP), column of [b | c] the rest
    static __device__ __forceinline__ int tok(int e) { return (e * kScanT + (int)threadIdx.x) / (2 * NP); }
    static __device__ __forceinline__ int col() { return (int)threadIdx.x % (2 * NP); }  // 2 NP divides kScanT
    __device__ __forceinline__ void fetch(const ScanArgs& p, const T* brow, const T* crow, int t0, int n) {
        const bool is_c = col() >= NP;
        const int s = min(is_c ? col() - NP : col(), p.N - 1);
        const T* base = is_c ? crow : brow;
        const long row = is_c ? p.cl : p.bl;
        if (t0 + TOK <= n) {
            base += (size_t)t0 * row;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = base[(unsigned)min(tok(e), TOK - 1) * (unsigned)row + (unsigned)s];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int t = min(t0 + min(tok(e), TOK - 1), n - 1);
                v[e] = base[(size_t)t * row + s];
            }
        }
    }
    __device__ __forceinline__ void put(float* lds, int t0, int n, int N) const {
        const int s = col() >= NP ? col() - NP : col();
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = e * kScanT + (int)threadIdx.x;
            if (kAll % kScanT == 0 || i < kAll) lds[i] = (s < N && t0 + tok(e) < n) ? to_f32(v[e]) : 0.f;
        }
    }
};

// Tokens q, q + Q, ... of a block for this lane's channel.
template <typename T, int Q, int TOK> struct TokLoad {
    static constexpr int R = TOK > Q ? TOK / Q : 1;
    T v[R];
    // col: the row of token t0 (uniform); off: byte offset of (token q, channel); qr = the lane's token, row = row stride
    __device__ __forceinline__ void full(const T* base, long row, unsigned off) {
#pragma unroll
        for (int i = 0; i < R; ++i) v[i] = load_at(base + (size_t)(i * Q) * row, off);
    }
    __device__ __forceinline__ void tail(const T* base, long row, int left, int q, unsigned chan) {
#pragma unroll
        for (int i = 0; i < R; ++i) v[i] = load_at(base + (size_t)min(i * Q + q, left - 1) * row, chan);
    }
};

// The loads under way have arrived.  Stores count with loads and complete in order: a block that starts right behind the
// stores of the one before it would wait for those too when it takes its loaded values, so the wait comes in front of them.
__device__ __forceinline__ void loads_arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

// No instruction moves across, LDS accesses among them, which is what it is for: left to itself the compiler puts each token's
// rows right in front of their use and waits for them there, once or twice a token.  It also keeps the next token's
// exponentials, which do not depend on the state, behind this token's chain.
__device__ __forceinline__ void hold_lds() { __builtin_amdgcn_sched_barrier(0); }

struct ScanPlace {
    int b, s, cb, ch, cl, q, n0, n;  // cl: the channel, or the last one for lanes behind it (they load and compute along)
    bool live;
};
// workgroup id -> (row of the batch, time segment, block of channels), channel blocks fastest
template <int Q, int NS> __device__ __forceinline__ ScanPlace scan_place(const ScanArgs& p) {
    ScanPlace w;
    const int id = blockIdx.x;
    w.cb = id % p.nb;
    const int r = id / p.nb;
    w.s = r % p.S;
    w.b = r / p.S;
    w.q = threadIdx.x & (Q - 1);
    w.ch = w.cb * (kScanT / Q) + (int)threadIdx.x / Q;
    w.live = w.ch < p.D;
    w.cl = min(w.ch, p.D - 1);
    w.n0 = w.q * NS;
    w.n = scan_rows(p.lengths, w.b, p.L);
    return w;
}

struct ScanShape {
    int Q, NS, NP;  // lanes per channel, states per lane, Q NS
};
// The smallest padded state count that holds N; 4 lanes per channel up to 16 states, then 4 states per lane.
inline ScanShape scan_shape(int N) {
    if (N <= 4) return {4, 1, 4};
    if (N <= 8) return {4, 2, 8};
    if (N <= 16) return {4, 4, 16};
    if (N <= 32) return {8, 4, 32};
    return {16, 4, 64};
}

int scan_forward_launch(const ScanArgs& p, int dtype, hipStream_t s);
int scan_backward_launch(const ScanArgs& p, int dtype, hipStream_t s);
// db and dc [B][L][N] from the workgroups' partial sums
int scan_bc_gradients(const ScanArgs& p, void* db, void* dc, int dtype, hipStream_t s);

}  // namespace afd
