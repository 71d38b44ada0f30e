// y = act(x w^T + bias) + residual and its backward, on the matrix cores: fp32 (v_mfma_f32_32x32x2_f32, exact products),
// bf16 and fp16 (32x32x16, sums in fp32).
//
// One kernel computes C[m][n] = sum_k A[m][k] B[n][k] for operands whose rows are contiguous along k: the forward as it
// stands, dx with w transposed, dw with dz and x transposed (prepare_kernel; operands of the forward whose rows do not start
// or end on 16-byte boundaries are copied by pad_kernel).  A workgroup owns a TM x TN tile; 128 bytes of k per row
// are staged in LDS, double buffered, one barrier per slab, and a slab's global loads are under way for the whole slab in
// front of it.  Both operands of a lane are 16-byte reads: lane l holds row l % 32 and the (2 s + l / 32)-th 16 bytes of its
// slab, which are 8 bf16 (one 32x32x16 product) or 4 fp32 (four 32x32x2 products, whose k order does not matter as long as
// both operands agree).  Chunks are XORed with the row, so 8 rows' reads of one chunk number spread over all banks.
// Few tiles: the k axis is split over workgroups, which leave fp32 partial tiles for a second kernel with the same epilogue.
//
// Bound by the matrix instructions and what keeps them waiting.  Measured, with the library's product of the same sizes in
// brackets: bf16 8192 x 8192 x 8192 1255 (1555) TFLOP/s, 16384 x 2048 x 2048 1124 (1402), where the matrix units are busy
// three fifths of the time (128 KB of LDS leave one workgroup per CU, and two waves per SIMD do not cover each other's barriers);
// fp32 16384 x 2048 x 2048 135 (147), 12928 x 1024 x 512 111 (108).  Before the waves' priorities, at 1172:
// staging 2 or 3 slabs ahead 1164, one wave per SIMD with 128 x 128 each 958, two workgroups of 128 x 256 per CU 958.  A forward with
// GELU, residual and the fp32 z takes 208 us at 16384 x 2048 x 2048, its input gradient 146: 201 MB more to move and 24 us of
// arithmetic, which no other workgroup of the CU covers.
#include "seq_common.h"

namespace {

using namespace afd;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kSlab = 128;  // bytes of k per row and slab

enum Act { kNone, kRelu, kSilu, kGelu };

// The normal distribution's Phi.  fp32: the library's erf.  16-bit results: 1 - Phi(a) = exp(-a^2 / 2) t P(t) for a = |z| and
// t = 1 / (1 + k a), the degree of P and k chosen for the least RELATIVE error over all a (7e-7 of the tail itself, 3e-6 with the
// float32 evaluation at a = 8; half a step is 5e-4 in fp16, 4e-3 in bf16): GELU of a negative z is z times that tail, and a fit
// with a small absolute error alone, 1.5e-7, is off by several half steps from z = -4 on.  No branch and a fifth of the library's
// instructions (its erf took 50 us of a 16384 x 2048 forward's epilogue).
__device__ __forceinline__ float gauss(float z) { return __builtin_amdgcn_exp2f(-0.5f * kLog2e * z * z); }  // exp(-z^2 / 2)
template <typename T> __device__ __forceinline__ float phi(float z) {
    if constexpr (sizeof(T) == 4) return 0.5f * (1.f + erff(z * 0.70710678118654752f));
    const float t = __builtin_amdgcn_rcpf(fmaf(0.261629522f, fabsf(z), 1.f));
    float p = -0.0712759495f;
    p = fmaf(p, t, 0.217830449f);
    p = fmaf(p, t, -0.0932164118f);
    p = fmaf(p, t, 0.158703104f);
    p = fmaf(p, t, 0.0763278529f);
    p = fmaf(p, t, 0.107441373f);
    p = fmaf(p, t, 0.10418994f);
    const float tail = p * t * gauss(z);  // 1 - Phi(|z|)
    return z < 0.f ? tail : 1.f - tail;
}

template <typename T> __device__ __forceinline__ float activate(float z, int act) {
    if (act == kRelu) return z < 0.f ? 0.f : z;  // (NaN stays)
    if (act == kSilu) return z * sigmoid_f32(z);
    if (act == kGelu) return z * phi<T>(z);
    return z;
}
template <typename T> __device__ __forceinline__ float activate_slope(float z, int act) {
    if (act == kRelu) return z > 0.f ? 1.f : 0.f;
    if (act == kSilu) {
        const float s = sigmoid_f32(z);
        return s * (1.f + z * (1.f - s));
    }
    if (act == kGelu) return phi<T>(z) + z * 0.39894228040143268f * gauss(z);
    return 1.f;
}

struct Epi {
    const void* bias;  // [N], NULL: none
    int bias_f32;
    const void* residual;  // rows of ldr elements, NULL: none
    long ldr;
    void* out;  // rows of ldo elements
    long ldo;
    float* z;  // pre-activation, rows of N elements, NULL: not kept
    int act;
};

struct Gemm {
    const void *a, *b;
    long lda, ldb;
    int M, N, K;
    Epi e;
    float* part;  // split k: [S][M][ldp] partial sums
    long ldp;
    int S, ksplit;  // splits and slabs per split
    int tm, tn;     // tiles
};

// One element.
template <typename T> __device__ __forceinline__ void finish_one(const Epi& e, int m, int n, int N, float z) {
    if (e.z) e.z[(size_t)m * N + n] = z;
    float o = activate<T>(z, e.act);
    if (e.residual) o += to_f32(static_cast<const T*>(e.residual)[(size_t)m * e.ldr + n]);
    static_cast<T*>(e.out)[(size_t)m * e.ldo + n] = from_f32<T>(o);
}

// (Compact on purpose: every workgroup walks through its epilogue once, and with the activation chosen element by element
// and all passes unrolled it was 90 KB of code that missed the instruction cache: 9 us for a product of a single slab.)
template <typename T> __device__ __forceinline__ void activate8(float (&v)[8], int act) {
    if (act == kRelu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activate<T>(v[i], kRelu);
    } else if (act == kSilu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activate<T>(v[i], kSilu);
    } else if (act == kGelu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activate<T>(v[i], kGelu);
    }
}

// Eight columns n .. n + 8 of a residual's row, asked for ahead (zeros where there is none or the row ends inside).
template <typename T> struct Ahead { u32x4 v[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Ahead<T> ask_residual(const Epi& e, int m, int n, int M, int N) {
    Ahead<T> r{};
    if (e.residual && m < M && n + 8 <= N) {
        const T* p = static_cast<const T*>(e.residual) + (size_t)m * e.ldr + n;
#pragma unroll
        for (int g = 0; g < (int)sizeof(T) / 2; ++g) r.v[g] = *reinterpret_cast<const u32x4_any*>(p + g * (16 / (int)sizeof(T)));
    }
    return r;
}

// Eight columns of row m.  The pre-activation is kept in fp32 whatever the tensors' type: the bias gradient is a sum of dy
// times its slope and an fp32 parameter's; at a z rounded to bf16 it was off by 2e-3.
template <typename T>
__device__ __forceinline__ void finish(const Epi& e, int m, int n, int N, float (&v)[8], const float (&bias)[8], const Ahead<T>& r) {
    T* out = static_cast<T*>(e.out) + (size_t)m * e.ldo + n;
    constexpr int W = 16 / (int)sizeof(T);
    const bool whole = n + 8 <= N;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += bias[i];
    if (e.z) {
        float* z = e.z + (size_t)m * N + n;
        if (whole) {
            store_row<float, 4>(z, *reinterpret_cast<float(*)[4]>(&v[0]));
            store_row<float, 4>(z + 4, *reinterpret_cast<float(*)[4]>(&v[4]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (n + i < N) z[i] = v[i];
        }
    }
    activate8<T>(v, e.act);
    if (whole) {
        if (e.residual) {
            const Pack<T, 8> k = __builtin_bit_cast(Pack<T, 8>, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += to_f32(k.v[i]);
        }
#pragma unroll
        for (int g = 0; g < 8; g += W) store_row<T, W>(out + g, *reinterpret_cast<float(*)[W]>(&v[g]));
    } else {
        const T* res = static_cast<const T*>(e.residual) + (size_t)m * e.ldr + n;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (n + i < N) out[i] = from_f32<T>(e.residual ? v[i] + to_f32(res[i]) : v[i]);
    }
}

template <typename T, int V> __device__ __forceinline__ void load_bias(const Epi& e, int n, int N, float (&b)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        b[i] = 0.f;
        if (e.bias && n + i < N)
            b[i] = e.bias_f32 ? static_cast<const float*>(e.bias)[n + i] : to_f32(static_cast<const T*>(e.bias)[n + i]);
    }
}

template <typename T> __device__ __forceinline__ void mma(const u32x4& a, const u32x4& b, f32x16& c) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    } else if constexpr (__is_same(T, bf16_t)) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// Where a chunk of 16 bytes sits in its 128-byte row: 16 lanes read one chunk number of 16 rows at a time, and two rows span
// the 64 banks, so every other row has to turn to another place.
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// Tile of this workgroup.  Workgroups go to the 8 XCDs in turn; each XCD takes a contiguous run of tiles, in groups of 8 tile
// rows walked column by column, so the rows of A and B that its workgroups share stay in its L2.
__device__ __forceinline__ void tile_of(const Gemm& g, int id, int& tm, int& tn) {
    const int total = g.tm * g.tn, each = total / 8, left = total % 8;
    const int x = id % 8, i = id / 8;
    const int t = x * each + min(x, left) + i;
    const int per = 8 * g.tn, grp = t / per, in = t - grp * per;
    const int rows = min(8, g.tm - grp * 8);
    tm = grp * 8 + in % rows;
    tn = in / rows;
}

template <int N> struct Const { static constexpr int value = N; };

template <typename T, int TM, int TN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) gemm_kernel(const Gemm g) {
    constexpr int kThreads = 64 * WM * WN, MI = TM / WM / 32, NI = TN / WN / 32;
    constexpr int EPC = 16 / (int)sizeof(T), KS = kSlab / (int)sizeof(T);  // elements per chunk and per slab
    constexpr int CA = TM * 8 / kThreads, CB = TN * 8 / kThreads;          // chunks a thread stages
    constexpr int kBuf = (TM + TN) * kSlab;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tm, tn;
    tile_of(g, blockIdx.x, tm, tn);
    const int m0 = tm * TM, n0 = tn * TN;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave % WM, wn = wave / WM, l31 = lane & 31, half = lane >> 5;
    const int kbeg = blockIdx.y * g.ksplit * KS, kend = min(kbeg + g.ksplit * KS, g.K);

    // operands: a uniform base that moves along k plus a fixed 32-bit offset per chunk; rows behind the matrix repeat its last
    const T* ab = static_cast<const T*>(g.a) + (size_t)m0 * g.lda + kbeg;
    const T* bb = static_cast<const T*>(g.b) + (size_t)n0 * g.ldb + kbeg;
    unsigned oa[CA], ob[CB], la[CA], lb[CB];
    int chunk[CA > CB ? CA : CB];
#pragma unroll
    for (int e = 0; e < (CA > CB ? CA : CB); ++e) chunk[e] = (e * kThreads + tid) & 7;
#pragma unroll
    for (int e = 0; e < CA; ++e) {
        const int row = (e * kThreads + tid) >> 3;
        oa[e] = (unsigned)((size_t)min(row, g.M - 1 - m0) * g.lda * sizeof(T)) + chunk[e] * 16;
        la[e] = row * kSlab + ((chunk[e] ^ swizzle(row)) * 16);
    }
#pragma unroll
    for (int e = 0; e < CB; ++e) {
        const int row = (e * kThreads + tid) >> 3;
        ob[e] = (unsigned)((size_t)min(row, g.N - 1 - n0) * g.ldb * sizeof(T)) + chunk[e] * 16;
        lb[e] = TM * kSlab + row * kSlab + ((chunk[e] ^ swizzle(row)) * 16);
    }
    u32x4 ra[CA], rb[CB];
    auto fetch = [&](int k) {
        const T* pa = ab + (k - kbeg);
        const T* pb = bb + (k - kbeg);
        auto at = [](const T* p, unsigned off) { return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p) + off); };
        if (k + KS <= kend) {
#pragma unroll
            for (int e = 0; e < CA; ++e) ra[e] = at(pa, oa[e]);
#pragma unroll
            for (int e = 0; e < CB; ++e) rb[e] = at(pb, ob[e]);
        } else {  // (kend is a multiple of a chunk; for chunks behind it the row's first, then zeros: one wait for all)
#pragma unroll
            for (int e = 0; e < CA; ++e) ra[e] = at(pa, k + chunk[e] * EPC < kend ? oa[e] : oa[e] - chunk[e] * 16);
#pragma unroll
            for (int e = 0; e < CB; ++e) rb[e] = at(pb, k + chunk[e] * EPC < kend ? ob[e] : ob[e] - chunk[e] * 16);
#pragma unroll
            for (int e = 0; e < CA; ++e) ra[e] = k + chunk[e] * EPC < kend ? ra[e] : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < CB; ++e) rb[e] = k + chunk[e] * EPC < kend ? rb[e] : u32x4{0, 0, 0, 0};
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int e = 0; e < CA; ++e) *reinterpret_cast<u32x4*>(lds + buf * kBuf + la[e]) = ra[e];
#pragma unroll
        for (int e = 0; e < CB; ++e) *reinterpret_cast<u32x4*>(lds + buf * kBuf + lb[e]) = rb[e];
    };

    f32x16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int arow = wm * (TM / WM) + l31, brow = wn * (TN / WN) + l31;
    // One slab: four steps of 32 bytes of k.  A step's fragments are read while the step before it is multiplied.  The next
    // slab's registers go to LDS between the first three steps' products, each loaded anew at once, so every load has a whole
    // slab's time to arrive (written in the third step and loaded behind it: 981 TFLOP/s at 16384 x 2048 x 2048 bf16 where this had
    // 1037); the barrier is passed in front of the last step, whose products cover the next slab's first reads.
    u32x4 fa[2][MI], fb[2][NI];
    auto read = [&](int buf, int st, int to) {
        const char* base = lds + buf * kBuf;
        const int c = ((2 * st + half) ^ swizzle(l31)) * 16;
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[to][i] = *reinterpret_cast<const u32x4*>(base + (arow + i * 32) * kSlab + c);
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[to][j] = *reinterpret_cast<const u32x4*>(base + TM * kSlab + (brow + j * 32) * kSlab + c);
    };
    // 16-bit: the products go first at the SIMD while they last, so that two waves take turns instead of waiting for the same
    // thing (1061 to 1124 TFLOP/s at 16384 x 2048 x 2048); the four times longer fp32 products only get in each other's way (135
    // to 121).
    constexpr bool kFirst = sizeof(T) == 2;
    auto multiply = [&](int from) {
        if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) mma<T>(fa[from][i], fb[from][j], acc[i][j]);
        if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
    };
    // reads, writes and products of a step take turns
    constexpr int kMma = MI * NI * (sizeof(T) == 4 ? 4 : 1);
    auto weave = [&](auto writes) {
        constexpr int kReads = MI + NI, kWrites = decltype(writes)::value, kAll = kReads + kWrites;
        constexpr int kEach = kMma / kAll > 0 ? kMma / kAll : 1;
#pragma unroll
        for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
        }
#pragma unroll
        for (int i = 0; i < kWrites; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
        }
    };
    // part P of three of the next slab's writes, each register loaded anew (from a whole slab) as soon as it is written
    constexpr int kStaged = CA + CB;
    auto turn_over = [&](auto part, int to, int k) {
        constexpr int lo = kStaged * decltype(part)::value / 3, hi = kStaged * (decltype(part)::value + 1) / 3;
        const char* pa = reinterpret_cast<const char*>(ab + (k - kbeg));
        const char* pb = reinterpret_cast<const char*>(bb + (k - kbeg));
        auto one = [&](u32x4& r, unsigned at, const char* next) {
            *reinterpret_cast<u32x4*>(lds + to * kBuf + at) = r;
            r = *reinterpret_cast<const u32x4*>(next);
        };
#pragma unroll
        for (int e = lo; e < hi; ++e) {
            if (e < CA) one(ra[e < CA ? e : 0], la[e < CA ? e : 0], pa + oa[e < CA ? e : 0]);
            else one(rb[e < CA ? 0 : e - CA], lb[e < CA ? 0 : e - CA], pb + ob[e < CA ? 0 : e - CA]);
        }
    };
    auto weave_turn = [&](auto part) {
        constexpr int kReads = MI + NI, kW = kStaged * (decltype(part)::value + 1) / 3 - kStaged * decltype(part)::value / 3;
        constexpr int kEach = kMma / (kReads + kW) > 0 ? kMma / (kReads + kW) : 1;
#pragma unroll
        for (int i = 0; i < kReads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            if (i < kW) {
                __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
        }
    };
    constexpr Const<0> none;
    constexpr Const<CA + CB> all;
    const int slabs = (kend - kbeg + KS - 1) / KS;
    if (slabs > 0) {
        fetch(kbeg);
        put(0);
        if (slabs > 1) fetch(kbeg + KS);
    }
    __syncthreads();
    read(0, 0, 0);
    int buf = 0;
    const int whole = (kend - kbeg) / KS;
    int i = 1;
    for (; i + 1 < whole; ++i, buf ^= 1) {
        const int k = kbeg + (i + 1) * KS;
        read(buf, 1, 1);
        turn_over(Const<0>{}, buf ^ 1, k);
        multiply(0);
        weave_turn(Const<0>{});
        read(buf, 2, 0);
        turn_over(Const<1>{}, buf ^ 1, k);
        multiply(1);
        weave_turn(Const<1>{});
        read(buf, 3, 1);
        turn_over(Const<2>{}, buf ^ 1, k);
        multiply(0);
        weave_turn(Const<2>{});
        __syncthreads();
        read(buf ^ 1, 0, 0);
        multiply(1);
        weave(none);
    }
    for (; i < slabs; ++i, buf ^= 1) {  // the last slabs: nothing, or only a part of one, is left to load
        read(buf, 1, 1);
        multiply(0);
        weave(none);
        read(buf, 2, 0);
        multiply(1);
        weave(none);
        read(buf, 3, 1);
        put(buf ^ 1);
        multiply(0);
        weave(all);
        if (i + 1 < slabs) fetch(kbeg + (i + 1) * KS);
        __syncthreads();
        read(buf ^ 1, 0, 0);
        multiply(1);
        weave(none);
    }
    read(buf, 1, 1);
    multiply(0);
    weave(none);
    read(buf, 2, 0);
    multiply(1);
    weave(none);
    read(buf, 3, 1);
    multiply(0);
    multiply(1);
    __syncthreads();

    // Epilogue, wave by wave through LDS (nobody reads the slabs any more): 32 rows of the wave's columns at a time, then
    // 8 columns per lane in row order.
    constexpr int WC = NI * 32, kPitch = WC + 4;
    float* tile = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
    constexpr int LPR = WC / 8, RPP = 64 / LPR;  // lanes per row, rows per pass
    const int col = (lane % LPR) * 8, n = n0 + wn * WC + col;
    float bias[8];
    auto row_of = [&](int i, int r) { return m0 + wm * (TM / WM) + i * 32 + r; };
    Ahead<T> next{};
    if (g.S == 1) {
        load_bias<T, 8>(g.e, n, g.N, bias);
        next = ask_residual<T>(g.e, row_of(0, lane / LPR), n, g.M, g.N);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) tile[((r & 3) + 8 * (r >> 2) + 4 * half) * kPitch + j * 32 + l31] = acc[i][j][r];
        __builtin_amdgcn_wave_barrier();
        if (g.S > 1) {  // 16 bytes per lane, in the order of memory (ldp is a multiple of 8)
            constexpr int L4 = WC / 4;
            const int c4 = (lane % L4) * 4, n4 = n0 + wn * WC + c4;
            float* dst = g.part + ((size_t)blockIdx.y * g.M + row_of(i, lane / L4)) * g.ldp + n4;
#pragma unroll 4
            for (int p = lane / L4; p < 32; p += 64 / L4) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(tile + p * kPitch + c4);
                if (row_of(i, p) < g.M && n4 < g.N) *reinterpret_cast<f32x4*>(dst) = v;
                dst += (64 / L4) * g.ldp;
            }
        } else {
#pragma unroll 1
            for (int p = lane / LPR; p < 32; p += RPP) {
                const int m = row_of(i, p);
                float v[8];
                const f32x4 lo = *reinterpret_cast<const f32x4*>(tile + p * kPitch + col);
                const f32x4 hi = *reinterpret_cast<const f32x4*>(tile + p * kPitch + col + 4);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    v[c] = lo[c];
                    v[4 + c] = hi[c];
                }
                const Ahead<T> res = next;
                next = ask_residual<T>(g.e, p + RPP < 32 ? m + RPP : row_of(i + 1, lane / LPR), n, g.M, g.N);
                if (m < g.M && n < g.N) finish<T>(g.e, m, n, g.N, v, bias, res);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Up to 16 MT rows: B's rows (the weights) are what is read, each once, straight into the operand registers of 16-column
// products, and x comes out of the L2.  A workgroup owns 16 columns and its 8 waves take every eighth slab of 128 bytes
// of k, four at a time, so K = 2048 in bf16 is one batch of loads per wave; the waves meet in LDS, in a fixed order.
constexpr int kFewWaves = 8, kFewBatch = 4;
template <typename T> __device__ __forceinline__ void mma16(const u32x4& a, const u32x4& b, f32x4& c) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
    } else if constexpr (__is_same(T, bf16_t)) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}
template <typename T, int MT, int NT> __global__ void __launch_bounds__(64 * kFewWaves, 2) few_rows_kernel(const Gemm g) {
    constexpr int EPC = 16 / (int)sizeof(T), KS = kSlab / (int)sizeof(T), kStep = kFewWaves * KS, U = kFewBatch;
    constexpr int kCols = NT * 16, kPitch = kCols + 4;  // (rows 0, 4, 8 and 12 of a tile on different banks)
    __shared__ float red[kFewWaves][MT * 16][kPitch];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * kCols;
    const int kbeg = blockIdx.y * g.ksplit * KS, kend = min(kbeg + g.ksplit * KS, g.K);
    const T *ap[MT], *bp[NT];
    f32x4 acc[MT][NT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        ap[t] = static_cast<const T*>(g.a) + (size_t)min(t * 16 + l15, g.M - 1) * g.lda;
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) bp[j] = static_cast<const T*>(g.b) + (size_t)min(n0 + j * 16 + l15, g.N - 1) * g.ldb;
    const u32x4 zero{0, 0, 0, 0};
    for (int k0 = kbeg + wave * KS; k0 < kend; k0 += U * kStep) {
        u32x4 ra[U][MT][2], rb[U][NT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int ku = k0 + u * kStep;
            const bool whole = ku + KS <= kend;  // (the same for the wave)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int k = ku + (s * 4 + quad) * EPC;
                if (whole) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) rb[u][j][s] = *reinterpret_cast<const u32x4*>(bp[j] + k);
#pragma unroll
                    for (int t = 0; t < MT; ++t) ra[u][t][s] = *reinterpret_cast<const u32x4*>(ap[t] + k);
                } else {
#pragma unroll
                    for (int j = 0; j < NT; ++j) rb[u][j][s] = k < kend ? *reinterpret_cast<const u32x4*>(bp[j] + k) : zero;
#pragma unroll
                    for (int t = 0; t < MT; ++t) ra[u][t][s] = k < kend ? *reinterpret_cast<const u32x4*>(ap[t] + k) : zero;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int j = 0; j < NT; ++j) mma16<T>(ra[u][t][s], rb[u][j][s], acc[t][j]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave][t * 16 + quad * 4 + r][j * 16 + l15] = acc[t][j][r];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 16 * kCols; i += 64 * kFewWaves) {
        const int m = i / kCols, c = i % kCols, n = n0 + c;
        if (m >= g.M || n >= g.N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) v += red[w][m][c];
        if (g.S > 1) {
            g.part[((size_t)blockIdx.y * g.M + m) * g.ldp + n] = v;
        } else {
            float bias[1];
            load_bias<T, 1>(g.e, n, g.N, bias);
            finish_one<T>(g.e, m, n, g.N, v + bias[0]);
        }
    }
}

// Sum of the k splits' partial tiles, and the epilogue.
template <typename T> __global__ void __launch_bounds__(256) join_kernel(const Gemm g) {
    const long groups = g.ldp / 8, all = (long)g.M * groups;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        const int m = (int)(i / groups), n = (int)(i - (long)m * groups) * 8;
        if (n >= g.N) continue;
        float v[8], bias[8];
        load_bias<T, 8>(g.e, n, g.N, bias);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = 0.f;
#pragma unroll 8
        for (int s = 0; s < g.S; ++s) {
            const float* src = g.part + ((size_t)s * g.M + m) * g.ldp + n;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(src), hi = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c] += lo[c];
                v[4 + c] += hi[c];
            }
        }
        finish<T>(g.e, m, n, g.N, v, bias, ask_residual<T>(g.e, m, n, g.M, g.N));
    }
}

// 64 x 64 tiles of the two transposing passes: a thread reads 8 columns of rows y and y + 32, and writes 8 rows of columns y
// and y + 32 (x8 its first column or row); 16-byte accesses inside the matrix, single elements at its edges.
template <typename T> __device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
    constexpr int W = 16 / (int)sizeof(T);
    if (left >= 8) {
#pragma unroll
        for (int g = 0; g < 8; g += W) load_row<T, W>(p + g, *reinterpret_cast<float(*)[W]>(&v[g]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32(p[i]) : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int left, const float (&v)[8]) {
    constexpr int W = 16 / (int)sizeof(T);
    if (left >= 8) {
#pragma unroll
        for (int g = 0; g < 8; g += W) store_row<T, W>(p + g, *reinterpret_cast<const float(*)[W]>(&v[g]));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = from_f32<T>(v[i]);
    }
}

// dst[c][r] = src[r][c] for R x C elements, rows of dst padded with zeros to ldd (a multiple of 16 bytes); `tiles` along r.
struct TurnJob {
    const void* src;
    void* dst;
    long ld, ldd;
    int R, C, tiles, groups;  // groups: workgroups, 0: nothing to turn
};
template <typename T> __device__ __forceinline__ void turn_tile(const TurnJob& j, int id, float (&t)[64][65]) {
    const int r0 = id % j.tiles * 64, c0 = id / j.tiles * 64;
    const int x8 = (threadIdx.x & 7) * 8, y = threadIdx.x >> 3;
    const T* src = static_cast<const T*>(j.src);
    T* dst = static_cast<T*>(j.dst);
#pragma unroll
    for (int i = y; i < 64; i += 32) {
        float v[8];
        load8<T>(src + (size_t)min(r0 + i, j.R - 1) * j.ld + c0 + x8, r0 + i < j.R ? j.C - c0 - x8 : 0, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) t[i][x8 + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int i = y; i < 64; i += 32) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = t[x8 + k][i];
        if (c0 + i < j.C) store8<T>(dst + (size_t)(c0 + i) * j.ldd + r0 + x8, (int)min(j.ldd - r0 - x8, 8L), v);
    }
}

// Rows of C elements copied to rows of ldd (whole 16-byte chunks, zeros behind C): one or two matrices in one launch, a wave
// per row.
struct PadJob {
    const void* src;
    void* dst;
    long ld;
    int rows;
};
template <typename T> __global__ void __launch_bounds__(256) pad_kernel(const PadJob a, const PadJob b, int C, int ldd) {
    const PadJob j = blockIdx.y ? b : a;
    const int lane8 = (threadIdx.x & 63) * 8;
    for (long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6); r < j.rows; r += (long)gridDim.x * 4) {
        const T* src = static_cast<const T*>(j.src) + (size_t)r * j.ld;
        T* dst = static_cast<T*>(j.dst) + (size_t)r * ldd;
        for (int c = lane8; c < ldd; c += 512) {
            float v[8];
            load8<T>(src + c, C - c, v);
            store8<T>(dst + c, ldd - c, v);
        }
    }
}

// dz = dy act'(z) as rows (ldz, zeros behind N) and turned (ldt, zeros behind M), and its column sums over the tile's rows;
// NULL: not wanted.  The rows are rounded to T: the matrix instructions take 16-bit operands, and two of them for one dz (its
// rounding's remainder as the second) would double both products, 255 of 533 us at 16384 x 2048 x 2048 bf16.  It is the rounding that an
// activation's gradient has wherever it is a tensor of its own; dx and dw of that case are off by 2.35e-3 (root mean
// square) with it, by 1.66e-3, their own rounding, without.  The column sums are of the unrounded dz.
struct DzJob {
    const void* dy;
    const float* z;
    void *dz, *turned;
    float* sums;
    long ldy, ldz, ldt;
    int act, M, N, tiles, groups;
};
template <typename T> __device__ __forceinline__ void dz_tile(const DzJob& j, int id, float (&t)[64][65], float (&red)[4][64]) {
    const int m0 = id % j.tiles * 64, n0 = id / j.tiles * 64;
    const int x8 = (threadIdx.x & 7) * 8, y = threadIdx.x >> 3;
    const T* dy = static_cast<const T*>(j.dy);
    T *dz = static_cast<T*>(j.dz), *turned = static_cast<T*>(j.turned);
#pragma unroll
    for (int i = y; i < 64; i += 32) {
        const int m = m0 + i, n = n0 + x8, left = m < j.M ? j.N - n : 0;
        float v[8], zv[8];
        load8<T>(dy + (size_t)min(m, j.M - 1) * j.ldy + n, left, v);
        if (j.act != kNone) {
            load8<float>(j.z + (size_t)min(m, j.M - 1) * j.N + n, left, zv);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = k < left ? v[k] * activate_slope<T>(zv[k], j.act) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) t[i][x8 + k] = v[k];
        if (dz && m < j.M) store8<T>(dz + (size_t)m * j.ldz + n, (int)min(j.ldz - n, 8L), v);
    }
    __syncthreads();
    if (turned) {
#pragma unroll
        for (int i = y; i < 64; i += 32) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = t[x8 + k][i];
            if (n0 + i < j.N) store8<T>(turned + (size_t)(n0 + i) * j.ldt + m0 + x8, (int)min(j.ldt - m0 - x8, 8L), v);
        }
    }
    if (!j.sums) return;
    const int col = threadIdx.x & 63, part = threadIdx.x >> 6;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += t[part * 16 + i][col];
    red[part][col] = s;
    __syncthreads();
    if (part == 0 && n0 + col < j.N)
        j.sums[(size_t)(id % j.tiles) * j.N + n0 + col] = (red[0][col] + red[1][col]) + (red[2][col] + red[3][col]);
}

// What the two products of a backward pass read, in one launch: the workgroups share themselves out over the three jobs.
// Bound by memory: 485 MB in 93 us (5.2 TB/s) at 16384 x 2048 x 2048 bf16 with an activation; three launches took 102.
template <typename T> __global__ void __launch_bounds__(256) prepare_kernel(const DzJob d, const TurnJob w, const TurnJob x) {
    __shared__ float t[64][65];
    __shared__ float red[4][64];
    const int id = blockIdx.x;
    if (id < d.groups) dz_tile<T>(d, id, t, red);
    else if (id < d.groups + w.groups) turn_tile<T>(w, id - d.groups, t);
    else turn_tile<T>(x, id - d.groups - w.groups, t);
}

// ---- host side -------------------------------------------------------------------------------------------------------
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
long pad_to(long n, long k) { return (n + k - 1) / k * k; }

// Tiles by what they took, us (M x N x K; `/` separates the tiles or splits compared).
//   256 x 256, 16-bit, from 16 slabs of work per CU on: bf16 16384 x 2048 x 2048 and its two gradients 220 171 162, with
//   128 x 128 263 211 186 (half the operand traffic per product).
//   Below, the largest tile that leaves 1.5 workgroups per CU (of 128 x 128, 128 x 64, 64 x 64), splits of a long k counted:
//   bf16 12928 x 512 x 1024 23 / 27 / 28, 2048 x 2048 x 2048 34 / 27 / 31, 4096 x 512 x 512 10.3 / 7.9 / 7.4, 1000 x 1000 x
//   1000 13.6 / 10.4 / 8.0; fp32 (no 128 x 128: a fifth of the card idles at the end) 2048 x 2048 x 2048 - / 136 / 159,
//   300 x 300 x 300 - / 15.2 / 9.6.
//   k is split until every CU has a workgroup, into 4 slabs at least: the partial tiles cost their traffic and a second
//   launch, and splitting on for two workgroups per CU took 14.2 against 8.3 at 1000 x 1000 x 1000 and 39 against 24 at
//   12928 x 512 x 1024; but splits of 32 slabs and more are worth it, 33 against 46 at 1024 x 512 x 12928.
// Up to 32 rows the weights are what is read (us here, and with one 32 x 128 tile row split along k and joined):
//   bf16 1 / 16 / 32 x 2048 x 2048: 4.9 / 6.2 / 8.1, 8.9 / 10.3 / 10.8; 32 x 8192 x 2048: 12.9 with 32 columns per workgroup,
//   15.8 with 16, 13.8; fp32 1 / 16 x 2048 x 2048: 7.9 / 11.1, 12.5 / 13.8; 4 x 10000 x 1024: 11.7 with 16 columns, 16.8 with
//   32, 17.0; but 32 rows of fp32 re-read x too often for large weights: 29 against 21.6 at 8192 x 2048, 13.8 against 16.2 at
//   2048 x 2048.
struct Shape {
    int kind;
    int tm, tn, S, ksplit;
    size_t part;
    double issued;  // flops with the tiles' padding
};
enum { kFew16, kFew32, kTile32x128, kTile64, kTile128x64, kTile128, kTile256 };
constexpr int kLong = 32;                         // slabs of a split that its workgroup's prologue and the joining are small against
constexpr int kFewLoad = kFewWaves * kFewBatch;  // slabs of one batch of a workgroup's loads
Shape gemm_shape(int M, int N, int K, int dtype) {
    Shape s;
    const int slabs = ceil_div(K, kSlab / (int)dtype_bytes(dtype));
    int rows = 64, cols = 64, least = 4, fill = 1024;  // slabs of a split at least; workgroups that a long k is split into
    const int longs = slabs / kLong > 1 ? slabs / kLong : 1;
    s.kind = kTile64;
    auto tiles = [&](int r, int c) { return (long)ceil_div(M, r) * ceil_div(N, c); };
    if (M <= 16 || (M <= 32 && (dtype != AFD_T_F32 || (long)N * K <= 1 << 22))) {
        const long loads = slabs / kFewLoad > 1 ? slabs / kFewLoad : 1;
        const bool wide = M > 16 && ceil_div(N, 32) * loads >= 256;
        s.kind = wide ? kFew32 : kFew16;
        rows = 32;
        cols = wide ? 32 : 16;
        least = kFewLoad;
    } else if (M <= 32) {
        s.kind = kTile32x128;
        rows = 32;
        cols = 128;
        least = 2;
    } else if (dtype != AFD_T_F32 && tiles(256, 256) * slabs >= 256 * 16) {  // 16 slabs for every CU
        s.kind = kTile256;
        rows = cols = fill = 256;
    } else if (dtype != AFD_T_F32 && M > 64 && N > 64 && tiles(128, 128) * longs >= 400) {
        s.kind = kTile128;
        rows = cols = 128;
        fill = 512;
    } else if (M > 64 && tiles(128, 64) * longs >= 400) {
        s.kind = kTile128x64;
        rows = 128;
        fill = 768;
    }
    s.tm = ceil_div(M, rows);
    s.tn = ceil_div(N, cols);
    // k is split for a workgroup on every CU, and for all that fit where the splits stay long
    const long all = (long)s.tm * s.tn;
    auto split = [&](long to, int slabs_each) {
        const long want = (to + all - 1) / all, most = slabs / slabs_each;
        return (int)(want < most ? want : most);
    };
    int want = split(256, least);
    if (want < split(fill, kLong)) want = split(fill, kLong);
    if (want < 1) want = 1;
    s.ksplit = ceil_div(slabs, want);
    s.S = ceil_div(slabs, s.ksplit);
    s.part = s.S > 1 ? align256((size_t)s.S * M * pad_to(N, 8) * 4) : 0;
    s.issued = 2.0 * s.tm * (s.kind == kFew16 && M <= 16 ? 16 : rows) * s.tn * cols * slabs * (kSlab / (int)dtype_bytes(dtype));
    return s;
}

template <typename T, int TM, int TN, int WM, int WN> int launch_tile(const Gemm& g, hipStream_t s) {
    constexpr int kBuf = 2 * (TM + TN) * kSlab, kEpi = WM * WN * 32 * (TN / WN + 4) * 4;
    constexpr unsigned lds = kBuf > kEpi ? kBuf : kEpi;
    if constexpr (lds > 64 * 1024) {
        static PerDeviceOnce once;
        if (!once.done()) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_kernel<T, TM, TN, WM, WN>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return fail(AFD_ERR_HIP, "linear: %s", hipGetErrorString(e));
            once.mark();
        }
    }
    hipLaunchKernelGGL((gemm_kernel<T, TM, TN, WM, WN>), dim3((unsigned)(g.tm * g.tn), (unsigned)g.S), dim3(64 * WM * WN), lds, s, g);
    return AFD_OK;
}

template <typename T, int MT, int NT> int launch_few(const Gemm& g, hipStream_t s) {
    hipLaunchKernelGGL((few_rows_kernel<T, MT, NT>), dim3((unsigned)g.tn, (unsigned)g.S), dim3(64 * kFewWaves), 0, s, g);
    return AFD_OK;
}

template <typename T> int gemm_t(const Gemm& g, int kind, hipStream_t s) {
    int rc;
    if (kind == kFew32) rc = launch_few<T, 2, 2>(g, s);
    else if (kind == kFew16) rc = g.M <= 16 ? launch_few<T, 1, 1>(g, s) : launch_few<T, 2, 1>(g, s);
    else if (kind == kTile64) rc = launch_tile<T, 64, 64, 2, 2>(g, s);
    else if (kind == kTile128x64) rc = launch_tile<T, 128, 64, 2, 2>(g, s);
    else if constexpr (sizeof(T) == 4) rc = launch_tile<T, 32, 128, 1, 4>(g, s);
    else if (kind == kTile256) rc = launch_tile<T, 256, 256, 2, 4>(g, s);
    else rc = launch_tile<T, 128, 128, 2, 2>(g, s);
    if (rc) return rc;
    if (g.S > 1) {
        const long all = (long)g.M * (g.ldp / 8), grid = (all + 255) / 256;
        hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, s, g);
    }
    return check_launch("gemm_kernel");
}

// C = A B^T with the epilogue; operands on 16-byte boundaries, K a multiple of 16 bytes.
int gemm(const void* a, long lda, const void* b, long ldb, int M, int N, int K, const Epi& e, int dtype, float* part, hipStream_t s) {
    const Shape q = gemm_shape(M, N, K, dtype);
    Gemm g{};
    g.a = a; g.b = b; g.lda = lda; g.ldb = ldb; g.M = M; g.N = N; g.K = K; g.e = e; g.part = part; g.ldp = pad_to(N, 8);
    g.S = q.S; g.ksplit = q.ksplit; g.tm = q.tm; g.tn = q.tn;
    if (dtype == AFD_T_F32) return gemm_t<float>(g, q.kind, s);
    if (dtype == AFD_T_BF16) return gemm_t<bf16_t>(g, q.kind, s);
    return gemm_t<f16_t>(g, q.kind, s);
}

TurnJob turn_job(const void* src, long ld, int R, int C, void* dst, long ldd) {
    const int tiles = ceil_div(ldd, 64);
    return {src, dst, ld, ldd, R, C, tiles, tiles * ceil_div(C, 64)};
}
int pad(const PadJob* jobs, int n, int C, long ldd, int dtype, hipStream_t s) {
    const PadJob &a = jobs[0], &b = jobs[n - 1];
    const long most = a.rows > b.rows ? a.rows : b.rows, grid = (most + 3) / 4;
    const dim3 d((unsigned)(grid < 65536 ? grid : 65536), (unsigned)n);
    if (dtype == AFD_T_F32) hipLaunchKernelGGL(pad_kernel<float>, d, dim3(256), 0, s, a, b, C, (int)ldd);
    else if (dtype == AFD_T_BF16) hipLaunchKernelGGL(pad_kernel<bf16_t>, d, dim3(256), 0, s, a, b, C, (int)ldd);
    else hipLaunchKernelGGL(pad_kernel<f16_t>, d, dim3(256), 0, s, a, b, C, (int)ldd);
    return check_launch("pad_kernel");
}

// May the product's kernel read these rows as they are?
bool direct(const void* p, long ld, int K, int dtype) {
    const long epc = 16 / (long)dtype_bytes(dtype);
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % epc == 0 && K % epc == 0 && ld <= (1 << 20);
}

int check(const char* what, long M, int N, int K, int act, int dtype) {
    if (M < 1 || N < 1 || K < 1 || act < 0 || act > 3 || !dtype_ok(dtype))
        return fail(AFD_ERR_ARG, "%s: M=%ld N=%d K=%d act=%d dtype=%d", what, M, N, K, act, dtype);
    if (M > 0x7fffff00L || N > (1 << 20) - 64 || K > (1 << 20) - 64 || (long)ceil_div(M, 128) * ceil_div(N, 64) > kMaxGroups)
        return fail(AFD_ERR_UNSUPPORTED, "%s: M=%ld N=%d K=%d is too large", what, M, N, K);
    return AFD_OK;
}

struct Arena {
    char* base;
    size_t at;
    void* take(size_t n) {
        void* p = base + at;
        at += align256(n);
        return p;
    }
};

}  // namespace

extern "C" size_t afd_linear_workspace_bytes(const void* x, long long ldx, const void* w, long long ldw, long long M, int N, int K,
                                             int dtype) {
    if (M < 1 || M > 0x7fffff00L || N < 1 || K < 1 || !dtype_ok(dtype)) return 0;
    const size_t e = dtype_bytes(dtype);
    const long kp = pad_to(K, 16 / (long)e);
    return (direct(x, ldx, K, dtype) ? 0 : align256((size_t)M * kp * e)) +
           (direct(w, ldw, K, dtype) ? 0 : align256((size_t)N * kp * e)) + gemm_shape((int)M, N, (int)kp, dtype).part;
}

extern "C" int afd_linear_forward(const void* x, long long ldx, const void* w, long long ldw, const void* bias, int bias_f32,
                                  const void* residual, long long ldr, void* y, float* z, long long M, int N, int K, int act,
                                  int dtype, void* ws, size_t ws_bytes, afd_stream_t stream) {
    if (!x || !w || !y) return fail(AFD_ERR_ARG, "linear: missing tensor");
    if (int rc = check("linear", M, N, K, act, dtype)) return rc;
    const size_t e = dtype_bytes(dtype);
    const long kp = pad_to(K, 16 / (long)e);
    const bool dx = direct(x, ldx, K, dtype), dw = direct(w, ldw, K, dtype);
    const size_t need = afd_linear_workspace_bytes(x, ldx, w, ldw, M, N, K, dtype);
    if (need > 0 && (!ws || ws_bytes < need)) return fail(AFD_ERR_WORKSPACE, "linear: workspace of %zu bytes, %zu needed", ws_bytes, need);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ScopedTiming timing(AFD_K_LINEAR, 2.0 * (double)M * N * K, s);
    timing.issued(gemm_shape((int)M, N, (int)kp, dtype).issued);
    timing.bytes((double)e * ((double)M * K + (double)N * K + (double)M * N * (residual ? 2 : 1)) + (z ? 4.0 * M * N : 0.0));
    Arena ar{static_cast<char*>(ws), 0};
    PadJob jobs[2];
    int n = 0;
    if (!dx) {
        jobs[n++] = {x, ar.take((size_t)M * kp * e), (long)ldx, (int)M};
        x = jobs[n - 1].dst;
        ldx = kp;
    }
    if (!dw) {
        jobs[n++] = {w, ar.take((size_t)N * kp * e), (long)ldw, N};
        w = jobs[n - 1].dst;
        ldw = kp;
    }
    if (n > 0)
        if (int rc = pad(jobs, n, K, kp, dtype, s)) return rc;
    Epi ep{bias, bias_f32, residual, ldr, y, N, z, act};
    return gemm(x, ldx, w, ldw, (int)M, N, (int)kp, ep, dtype, reinterpret_cast<float*>(ar.base + ar.at), s);
}

namespace {
struct BackPlan {
    long mp, np;  // padded lengths of the k axes
    size_t dz, dzt, xt, wt, sums, part, total;
};
BackPlan back_plan(long M, int N, int K, int dtype) {
    BackPlan b;
    const size_t e = dtype_bytes(dtype);
    const long epc = 16 / (long)e;
    b.mp = pad_to(M, epc);
    b.np = pad_to(N, epc);
    b.dz = align256((size_t)M * b.np * e);
    b.dzt = align256((size_t)N * b.mp * e);
    b.xt = align256((size_t)K * b.mp * e);
    b.wt = align256((size_t)K * b.np * e);
    b.sums = align256((size_t)ceil_div(b.mp, 64) * N * 4);
    const size_t p1 = gemm_shape((int)M, K, (int)b.np, dtype).part, p2 = gemm_shape(N, K, (int)b.mp, dtype).part;
    b.part = p1 > p2 ? p1 : p2;
    b.total = b.dz + b.dzt + b.xt + b.wt + b.sums + b.part;
    return b;
}
}  // namespace

extern "C" size_t afd_linear_backward_workspace_bytes(long long M, int N, int K, int dtype) {
    if (M < 1 || N < 1 || K < 1 || !dtype_ok(dtype)) return 0;
    return back_plan(M, N, K, dtype).total;
}

extern "C" int afd_linear_backward(const void* x, long long ldx, const void* w, long long ldw, const float* z, const void* dy,
                                   long long ldy, void* dx, void* dw, void* dbias, int bias_f32, long long M, int N, int K,
                                   int act, int dtype, void* ws, size_t ws_bytes, afd_stream_t stream) {
    if (!x || !w || !dy || (act != kNone && !z)) return fail(AFD_ERR_ARG, "linear backward: missing tensor");
    if (int rc = check("linear backward", M, N, K, act, dtype)) return rc;
    // (a tile's rows of the turned operands have to be within a 32-bit offset of each other)
    if (M > 8000000) return fail(AFD_ERR_UNSUPPORTED, "linear backward: M=%lld, at most 8000000 rows", M);
    const long mt = ceil_div(M + 8, 64), nt = ceil_div(N + 8, 64), kt = ceil_div(K, 64);
    if (mt * nt + mt * kt + nt * kt > kMaxGroups) return fail(AFD_ERR_UNSUPPORTED, "linear backward: M=%lld N=%d K=%d", M, N, K);
    const BackPlan b = back_plan(M, N, K, dtype);
    if (!ws || ws_bytes < b.total)
        return fail(AFD_ERR_WORKSPACE, "linear backward: workspace of %zu bytes, %zu needed", ws_bytes, b.total);
    hipStream_t s = static_cast<hipStream_t>(stream);
    ScopedTiming timing(AFD_K_LINEAR, 2.0 * (double)M * N * K * ((dx != nullptr) + (dw != nullptr)), s);
    timing.issued((dx ? gemm_shape((int)M, K, (int)b.np, dtype).issued : 0.0) + (dw ? gemm_shape(N, K, (int)b.mp, dtype).issued : 0.0));
    timing.bytes((double)dtype_bytes(dtype) * ((double)M * N + (dx ? (double)N * K + (double)M * K : 0.0) +
                                               (dw ? (double)M * K + (double)N * K : 0.0)) + (act != kNone ? 4.0 * M * N : 0.0));
    Arena ar{static_cast<char*>(ws), 0};
    void* dz = ar.take(b.dz);
    void* dzt = ar.take(b.dzt);
    void* xt = ar.take(b.xt);
    void* wt = ar.take(b.wt);
    float* sums = static_cast<float*>(ar.take(b.sums));
    float* part = reinterpret_cast<float*>(ar.base + ar.at);
    // without an activation dy is dz, and can be read as it is where its rows allow
    const bool rows = act != kNone || !direct(dy, ldy, N, dtype);
    DzJob jd{dy, z, dx && rows ? dz : nullptr, dw ? dzt : nullptr, dbias ? sums : nullptr, ldy, b.np, b.mp, act, (int)M, N, 0, 0};
    if (jd.dz || jd.turned || jd.sums) {
        jd.tiles = ceil_div(b.mp, 64);
        jd.groups = jd.tiles * ceil_div(b.np, 64);
    }
    const TurnJob jw = dx ? turn_job(w, ldw, N, K, wt, b.np) : TurnJob{}, jx = dw ? turn_job(x, ldx, (int)M, K, xt, b.mp) : TurnJob{};
    const dim3 grid((unsigned)(jd.groups + jw.groups + jx.groups));
    if (grid.x == 0) return AFD_OK;
    if (dtype == AFD_T_F32) hipLaunchKernelGGL(prepare_kernel<float>, grid, dim3(256), 0, s, jd, jw, jx);
    else if (dtype == AFD_T_BF16) hipLaunchKernelGGL(prepare_kernel<bf16_t>, grid, dim3(256), 0, s, jd, jw, jx);
    else hipLaunchKernelGGL(prepare_kernel<f16_t>, grid, dim3(256), 0, s, jd, jw, jx);
    if (int rc = check_launch("prepare_kernel")) return rc;
    if (dbias) {
        ColumnOuts o{};
        o.n = 1;
        o.o[0] = {dbias, 0, N, 1, 1, 1, 0, bias_f32 ? AFD_T_F32 : dtype};
        if (int r = launch_column_sums(sums, ceil_div(b.mp, 64), N, o, s)) return r;
    }
    if (dx) {
        Epi e{nullptr, 0, nullptr, 0, dx, K, nullptr, kNone};
        if (int r = gemm(rows ? dz : dy, rows ? b.np : ldy, wt, b.np, (int)M, K, (int)b.np, e, dtype, part, s)) return r;
    }
    if (dw) {
        Epi e{nullptr, 0, nullptr, 0, dw, K, nullptr, kNone};
        if (int r = gemm(dzt, b.mp, xt, b.mp, N, K, (int)b.mp, e, dtype, part, s)) return r;
    }
    return AFD_OK;
}
