// Products of 8-bit rows: c[m, n] = (sum_k A[m, k] B[n, k]) sa[m] sb[n] (+ bias[n]), A [M, K]
// and B [N, K] int8 with a float32 scale for each row (a token, an output channel), and what
// closes a layer, in the same launch:
//
//   C[m, n] = act(c[m, n]) (+ R[m, n])
//   C[m, n] = act(c[m, n]) c[m, N + n] (+ R[m, n])    gated: B [2 N, K], the gate's rows first
//
// The sum is exact (int32: K <= 131071 keeps it below 2^31 for any bytes), so how it is cut
// over work-groups, wavefronts and k ranges never changes a bit of the result; the epilogue
// rounds it to float32 once, multiplies by the two scales in turn and adds the bias; all after
// that is float32 too, rounded to C's type at the end.
//
// The kernels are instantiated by kind (gemm_int8.hip: the product alone, gemm_int8_epilogue.hip:
// with an activation or a residual, gemm_int8_gated.hip).
//
// Three kernels:
//   gemm_int8_kernel     tiles through LDS on v_mfma_i32_32x32x32_i8, bound by the matrix
//                        cores (and the loads that feed them) for large M
//   rows_int8_kernel     few rows: bound by streaming B once; a work-group takes 16 rows of B,
//                        its wavefronts split K, operands go straight to registers
//   rows_int8_kernel with x in float: the same for up to three rows (fused_rows), x quantised by
//                        every work-group (x is small and in L2): one launch instead of two
#pragma once

#include "gemm_direct.h"
#include "int8_common.h"

namespace migemm {

// What a kernel computes beside the product: nothing; an activation and a residual; the product of
// a gate's activation and the other half.
enum Int8Kind { kProduct, kEpilogue, kGated };

int launch_product_epilogue(hipStream_t stream, const Int8Product &p);
int launch_product_gated(hipStream_t stream, const Int8Product &p);
int launch_linear_epilogue(hipStream_t stream, const void *X, int64_t ldx, int cols,
                           const Int8Product &p);
int launch_linear_gated(hipStream_t stream, const void *X, int64_t ldx, int cols,
                        const Int8Product &p);

namespace {

constexpr int BK = 32;  // words of four values of K in a stage

struct Int8Args {
    TiledArgs t;  // A, B, lda, ldb, K in units of four bytes; the tile mapping
    const float *sa, *sb, *bias;
    void *C;
    int64_t ldc;
    int32_t *partial;  // [splits][M][N] when splits > 1
    // kGated: t.N counts the columns of the tiles, in which 16 of the gate and the 16 of the other
    // half that belong to them take turns; outputs counts those of C
    int outputs, act;
    const void *residual;
    int64_t ldr;
};

template <typename T>
__device__ __forceinline__ void put(T *c, int sum, float sa, float sb, float bias) {
    *c = from_f32<T>((float)sum * sa * sb + bias);
}

// The activations, each a function of float32. relu keeps NaN (a maximum would not).
struct Identity {
    __device__ __forceinline__ float operator()(float x) const { return x; }
};
struct Relu {
    __device__ __forceinline__ float operator()(float x) const { return x < 0.f ? 0.f : x; }
};
// x / (1 + exp(-x (a + b x^2))): silu with a = 1, b = 0, and gelu_tanh, as 1 + tanh(u) = 2 / (1 +
// exp(-2 u)), with a = 2 sqrt(2 / pi), b = 0.044715 a. log2(e) is folded into the constants, and
// exponential and reciprocal are the hardware's (each within 1 ulp; about 45 cycles a wavefront
// against 130 by division and a library exponential, on values that no product hides): off by
// less than (4 + 1.5 |x (a + b x^2)|) 2^-23 of the value (the exponent's three roundings, then one
// of each step), and 0 where the reciprocal is less than 2^-126.
template <bool CUBIC>
struct Sigmoid {
    float a, b;
    __device__ __forceinline__ float operator()(float x) const {
#pragma clang fp contract(off)
        const float z = x * (CUBIC ? __builtin_fmaf(x * x, b, a) : a);
        return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z));
    }
};
// x (1 + erf(x / sqrt 2)) / 2 = x P(x), P the normal distribution: P(-a) = exp(-a^2 / 2) u q(u) for a
// = |x| and u = 1 / (1 + 0.39 a), q of degree 9 through the Chebyshev nodes of u for 0 <= a <= 13.3
// (off by 2^-26.7), and P(a) = 1 - P(-a). Off by less than (10 + 1.5 x^2 / 2) 2^-23 of the value,
// the small ones of negative x too (in 2^-24: 6 of u, 7 of q, 5 of the other steps, 3 x^2 / 2 of the
// exponent; 1 + erf moves in steps of 2^-24, and at -5 is off by a tenth), and 0 where the
// exponential is less than 2^-126 (beyond 13.2).
struct Gelu {
    __device__ __forceinline__ float operator()(float x) const {
#pragma clang fp contract(off)
        const float a = fabsf(x);
        float p = 0.f;
        if (a < 13.3f) {  // (a branch also keeps the values of a thread apart, so registers suffice)
            const float u = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.39f, 1.f));
            float q = 0.0300211515f;
            q = __builtin_fmaf(q, u, -0.172886625f);
            q = __builtin_fmaf(q, u, 0.398460865f);
            q = __builtin_fmaf(q, u, -0.432662934f);
            q = __builtin_fmaf(q, u, 0.184471577f);
            q = __builtin_fmaf(q, u, -0.0497388989f);
            q = __builtin_fmaf(q, u, 0.101456709f);
            q = __builtin_fmaf(q, u, 0.129514083f);
            q = __builtin_fmaf(q, u, 0.155783504f);
            q = __builtin_fmaf(q, u, 0.155580565f);
            p = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170368f) * (u * q);
        }
        return x * (x < 0.f ? p : 1.f - p);
    }
};
constexpr float kLog2e = 1.44269504088896340736f, kGeluA = 1.59576912160573071176f;

// Calls f with the activation: one branch a work-group, not one a value.
template <typename F>
__device__ __forceinline__ void with_activation(int act, const F &f) {
    switch (act) {
        case MIGEMM_ACT_RELU: f(Relu{}); break;
        case MIGEMM_ACT_SILU: f(Sigmoid<false>{-kLog2e, 0.f}); break;
        case MIGEMM_ACT_GELU: f(Gelu{}); break;
        case MIGEMM_ACT_GELU_TANH:
            f(Sigmoid<true>{-kLog2e * kGeluA, -kLog2e * kGeluA * 0.044715f});
            break;
        default: f(Identity{}); break;
    }
}

// One output from its sum (and the other half's), with the residual where there is one. Every
// rounding is written out (the compiler joins no product and sum of its own), so that a result has
// the same bits whichever kernel computes it.
__device__ __forceinline__ float scaled(int sum, float sa, float sb, float bias) {
    return __builtin_fmaf((float)sum * sa, sb, bias);
}
template <typename T, typename Act>
__device__ __forceinline__ void put_act(T *c, const Act &act, int sum, float sa, float sb,
                                        float bias, float res) {
#pragma clang fp contract(off)
    const float y = act(scaled(sum, sa, sb, bias));
    *c = from_f32<T>(y + res);
}
template <typename T, typename Act>
__device__ __forceinline__ void put_gated(T *c, const Act &act, int sum, int up, float sa,
                                          float sb, float bias, float sb_up, float bias_up,
                                          float res) {
#pragma clang fp contract(off)
    const float g = act(scaled(sum, sa, sb, bias));
    const float y = g * scaled(up, sa, sb_up, bias_up);
    *c = from_f32<T>(y + res);
}

// B's tile of a gated product: tile row r is output o0 + 16 (r / 32) + r % 16 of the gate
// (r % 32 < 16) or of the other half, which begins `outputs` rows on. A load instruction
// fills 8 rows of the tile, so each is wholly of one half: its base is uniform (and kept in scalar
// registers) and its lanes' offsets stay within the tile's rows.
__device__ __forceinline__ const char *uniform(const char *p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)x);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32));
    return reinterpret_cast<const char *>((uint64_t)hi << 32 | lo);
}
template <typename Op>
struct GatedOperand : Op {
    const char *from[Op::NS];

    __device__ __forceinline__ void init(const float *op, int64_t ld, int o0, int outputs,
                                         int wave, int lane) {
        static_assert(Op::FPI == 8 * BK, "a load instruction fills 8 rows");
        this->q0 = wave * Op::NS;
#pragma unroll
        for (int j = 0; j < Op::NS; ++j) {
            const int f = Op::FPI * (this->q0 + j) + 4 * lane;
            const int r = f / BK, pos = f % BK;
            const int k = 4 * ((pos / 4) ^ kc_swz<BK>(r)) + pos % 4;
            const int o = min(o0 + 16 * (r >> 5) + (r & 15), outputs - 1);
            this->kk[j] = k;
            this->voff[j] = (uint32_t)(((o - o0) * (uint32_t)ld + k) * 4);
            const int64_t first = o0 + (((this->q0 + j) >> 1) & 1 ? (int64_t)outputs : 0);
            from[j] = uniform(reinterpret_cast<const char *>(op + first * ld));
        }
    }
    __device__ __forceinline__ void issue(float *stage, int kt, int64_t) const {
#pragma unroll
        for (int j = 0; j < Op::NS; ++j)
            dma16(from[j] + (int64_t)kt * BK * 4, this->voff[j], stage + this->lds_off(j));
    }
};
template <int NT, int T>
__device__ __forceinline__ const char *base_of(const DlOperand<NT, true, 32, T, 4> &op, int) {
    return op.base;
}
template <typename Op>
__device__ __forceinline__ const char *base_of(const GatedOperand<Op> &op, int j) {
    return op.from[j];
}

// This lane's 16 bytes of each load of the tail tile kt, zero at k >= K. K is a multiple of 16
// bytes, so each is wholly inside or outside; all loads are made (outside: at the row's start)
// and fly together.
template <typename Op>
__device__ __forceinline__ void fetch_tail(const Op &op, typename Op::Tail &t, int kt, int K) {
#pragma unroll
    for (int j = 0; j < Op::NS; ++j) {
        const bool in = kt * BK + op.kk[j] < K;
        const char *row = base_of(op, j) + (op.voff[j] - 4 * op.kk[j]);
        t.v[j] = *reinterpret_cast<const f4 *>(in ? row + ((int64_t)kt * BK + op.kk[j]) * 4 : row);
        if (!in) t.v[j] = f4{0.f, 0.f, 0.f, 0.f};
    }
}

// The epilogue of a wavefront's tiles. Registers hold a block of 32 x 32 sums by columns, and a
// gate's sum and the one that it multiplies lie 16 lanes apart, so a block goes through 4 KB of
// LDS (the operands' stages, which are free then) and comes back with four neighbouring outputs a
// lane: residual and results move in wide accesses, and the code of five activations is there once
// a block, not once a register. A block's residual is read before its sums are
// exchanged, all of it at once. (From the registers, one value a lane and access, the 256 x 256
// tiles keep 428 values in scratch.) Row r of a block stands at r with bits 0 and 2 exchanged: the
// two half-wavefronts that write rows r and r + 4 then meet different banks. 4096 x 4096 to
// 11008 outputs and their gates takes 360 to 371 us (as many plain products, 8192 x 4096 to 11008, 362;
// bound by the matrix cores as those are); 1000 x 777 to gelu of 3000 12.9 (silu 11.7).
// The 256 x 256 tiles keep up to 9 registers in scratch here (of a gated product none).
__device__ __forceinline__ int block_row(int r) {
    return (r & ~5) | ((r >> 2) & 1) | ((r & 1) << 2);
}

// The scales and bias of a tile's rows and columns, one value a thread: loaded as the kernel
// begins, kept in a register and put into LDS for its end (read from memory as they are used, each
// block waits for them: 27 us more). By place: the rows' scales, the columns' (of a
// gated tile the gate's outputs, then the other half's), the columns' bias.
template <int KIND, int BM, int BN>
__device__ __forceinline__ float closing_value(const Int8Args &p, int m0, int n0, int i) {
    if (i < BM) return p.sa[min(m0 + i, p.t.M - 1)];
    const int c = (i - BM) % BN;
    const float *from = i < BM + BN ? p.sb : p.bias;
    if (i >= BM + 2 * BN || from == nullptr) return 0.f;
    if (KIND != kGated) return from[min(n0 + c, p.outputs - 1)];
    return from[(c < BN / 2 ? 0 : p.outputs) + min(n0 / 2 + c % (BN / 2), p.outputs - 1)];
}

// block: this wavefront's 4 KB; held: the closing values. r0, c0: its place in the tile.
template <typename T, int KIND, int BM, int BN, int FM, int FN>
__device__ __forceinline__ void store_closed(const Int8Args &p, int32_t *block, const float *held,
                                             int m0, int n0, int r0, int c0, int lane,
                                             const v16i (&acc)[FM][FN]) {
    constexpr bool GATED = KIND == kGated;
    constexpr int COLS = GATED ? 16 : 32;     // outputs of a block's row
    constexpr int LANES = COLS / 4;           // lanes that take a row
    constexpr int ROWS = 64 / LANES;          // rows a pass
    constexpr int PASSES = 32 / ROWS;
    const int lo = lane & 31, hi = lane >> 5;
    const int from = lane % LANES * 4, at = lane / LANES;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int local = (GATED ? c0 / 2 : c0) + j * COLS + from;
        const int out = (GATED ? n0 / 2 : n0) + local;
        const int left = p.outputs - out, o = left > 0 ? out : 0;
        const float *columns = held + BM + local;
        const v4f sb = *reinterpret_cast<const v4f *>(columns);
        const v4f bias = *reinterpret_cast<const v4f *>(columns + BN);
        v4f sb_up = sb, bias_up = bias;
        if (GATED) {
            sb_up = *reinterpret_cast<const v4f *>(columns + BN / 2);
            bias_up = *reinterpret_cast<const v4f *>(columns + BN + BN / 2);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            float sa[PASSES], add[PASSES][4];
#pragma unroll
            for (int s = 0; s < PASSES; ++s) {
                const int row = r0 + i * 32 + block_row(s * ROWS + at);
                sa[s] = held[row];
                load_f32<T, 4>(static_cast<const T *>(p.residual) +
                                   (int64_t)min(m0 + row, p.t.M - 1) * p.ldr + o,
                               p.residual != nullptr ? left : 0, add[s]);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int r = 0; r < 16; ++r)
                block[block_row(8 * (r >> 2) + 4 * hi + (r & 3)) * 32 + lo] = acc[i][j][r];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int s = 0; s < PASSES; ++s) {
                const int row = m0 + r0 + i * 32 + block_row(s * ROWS + at);
                const int32_t *sums = block + (s * ROWS + at) * 32 + from;
                const v4i sum = *reinterpret_cast<const v4i *>(sums);
                v4i up = sum;
                if (GATED) up = *reinterpret_cast<const v4i *>(sums + 16);
                struct Raw {
                    T v[4];
                } y;
                with_activation(p.act, [&](auto act) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (GATED)
                            put_gated(&y.v[e], act, sum[e], up[e], sa[s], sb[e], bias[e], sb_up[e],
                                      bias_up[e], add[s][e]);
                        else
                            put_act(&y.v[e], act, sum[e], sa[s], sb[e], bias[e], add[s][e]);
                    }
                });
                if (row < p.t.M) {
                    T *c = static_cast<T *>(p.C) + (int64_t)row * p.ldc + out;
                    if (left >= 4) {
                        store_any(c, y);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (e < left) c[e] = y.v[e];
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// ---------------------------------------------------------------------------- large tiles
// BM x BN tiles, 128 bytes of K a stage, loaded straight into LDS (DlOperand, whose unit of
// four bytes holds four values of K here) and swizzled by 16-byte chunks; a fragment read of
// 16 bytes a lane is one operand of v_mfma_i32_32x32x32_i8. The order of waits, barrier and
// loads is gemm_direct_kernel's: a tile's loads run D tiles ahead, and every fragment read of
// a stage is issued before the barrier that frees it. 256 x 256 tiles have 16 wavefronts of
// 32 x 128, four on a SIMD, so that one's fragment reads and waits pass under the others'
// products (8 wavefronts of 64 x 128: 401 us, 16: 348 at 8192 x 11008 x 4096); K in stages of 64
// bytes and four of them: 376. Bound by the matrix cores and their clock, which follows the data:
// random bytes 471 us at 8192^3 (2.33 POP/s; a library's product 447) and 362 at 8192 x 11008 x
// 4096 (2.04; 340), zeros 305 (3.60; 307) and 263 (263), on one card.
template <typename T, int KIND, int BM, int BN, int WM, int WN, int S, int D, int OCC>
__global__ void __launch_bounds__(WM *WN * 64) __attribute__((amdgpu_waves_per_eu(OCC)))
gemm_int8_kernel(Int8Args p) {
    constexpr int NT = WM * WN * 64;
    constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
    constexpr int G = BK / 8;
    typedef DlOperand<NT, true, BK, BM, 4> OpA;
    typedef DlOperand<NT, true, BK, BN, 4> PlainB;
    typedef typename std::conditional<KIND == kGated, GatedOperand<PlainB>, PlainB>::type OpB;
    constexpr int A_FL = OpA::FLOATS, B_FL = OpB::FLOATS;
    constexpr int LPT = OpA::NS + OpB::NS;
    static_assert(S >= 2 && S <= 4 && D >= 2 && D <= S, "the loop below takes S steps of 2..4");
    __shared__ __attribute__((aligned(16))) float lds[S * (A_FL + B_FL)];
    float *const lds_a = lds, *const lds_b = lds + S * A_FL;

    static_assert(NT >= BM + 2 * BN, "a closing value a thread");
    __shared__ __attribute__((aligned(16))) float closing[KIND == kProduct ? 4 : BM + 2 * BN];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    TileCoord tc = tile_coord<BM, BN>(p.t, blockIdx.x);
    tc.split = __builtin_amdgcn_readfirstlane(tc.split);
    tc.m0 = __builtin_amdgcn_readfirstlane(tc.m0);
    tc.n0 = __builtin_amdgcn_readfirstlane(tc.n0);
    OpA opa;
    OpB opb;
    opa.init(p.t.A, p.t.lda, tc.m0, p.t.M, wave, lane);
    if constexpr (KIND == kGated)
        opb.init(p.t.B, p.t.ldb, tc.n0 / 2, p.outputs, wave, lane);
    else
        opb.init(p.t.B, p.t.ldb, tc.n0, p.t.N, wave, lane);

    float mine = 0.f;
    if (KIND != kProduct)
        mine = closing_value<KIND, BM, BN>(p, tc.m0, tc.n0, threadIdx.x);
    v16i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    const int K = p.t.K;
    const int kt0 = tc.split * p.t.kt_per_split;
    const int kt1 = min((K + BK - 1) / BK, kt0 + p.t.kt_per_split);
    const int kf = min(kt1, K / BK);

    auto issue = [&](int kt, int st) {
        opa.issue(lds_a + st * A_FL, kt, p.t.lda);
        opb.issue(lds_b + st * B_FL, kt, p.t.ldb);
    };
    auto frags = [&](int st, int g, f4(&fa)[FM], f4(&fb)[FN]) {
        dl_frags<true, BK, BM, FM>(lds_a + st * A_FL, wm * (BM / WM), g, lane, fa);
        dl_frags<true, BK, BN, FN>(lds_b + st * B_FL, wn * (BN / WN), g, lane, fb);
    };
    auto mfmas = [&](const f4(&fa)[FM], const f4(&fb)[FN]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                    __builtin_bit_cast(v4i, fa[i]), __builtin_bit_cast(v4i, fb[j]), acc[i][j], 0,
                    0, 0);
    };
    auto step = [&](int kt, auto st) {
        constexpr int ST = decltype(st)::value;
        f4 fa[2][FM], fb[2][FN];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            frags(ST, g, fa[g & 1], fb[g & 1]);
            if (g > 0) mfmas(fa[(g - 1) & 1], fb[(g - 1) & 1]);
        }
        if constexpr (D > 2) {
            if (kt + D - 1 < kf)
                wait_vmcnt<(D - 2) * LPT>();
            else
                wait_vmcnt<0>();
        } else {
            wait_vmcnt<0>();
        }
        __syncthreads();
        if (kt + D < kf) issue(kt + D, (ST + D) % S);
        mfmas(fa[(G - 1) & 1], fb[(G - 1) & 1]);
    };

    // The tail tile's loads are issued first where registers allow (a short k loop does not
    // hide their latency at its end); being the oldest, every wait below covers them.
    constexpr bool EARLY = OpA::NS + OpB::NS <= 4 && BM * BN < 256 * 256;
    typename OpA::Tail ta;
    typename OpB::Tail tb;
    if (EARLY && kf < kt1) {
        fetch_tail(opa, ta, kf, K);
        fetch_tail(opb, tb, kf, K);
    }

    int kt = kt0;
    if (kt0 < kf) {
#pragma unroll
        for (int t = 0; t < D; ++t)
            if (kt0 + t < kf) issue(kt0 + t, t);
        if (kt0 + D - 1 < kf)
            wait_vmcnt<(D - 1) * LPT>();
        else
            wait_vmcnt<0>();
        __syncthreads();
        for (; kt + S - 1 < kf; kt += S) {
            step(kt, std::integral_constant<int, 0>{});
            step(kt + 1, std::integral_constant<int, 1 % S>{});
            if constexpr (S > 2) step(kt + 2, std::integral_constant<int, 2 % S>{});
            if constexpr (S > 3) step(kt + 3, std::integral_constant<int, 3 % S>{});
        }
        if (kt < kf) step(kt++, std::integral_constant<int, 0>{});
        if constexpr (S > 2)
            if (kt < kf) step(kt++, std::integral_constant<int, 1 % S>{});
        if constexpr (S > 3)
            if (kt < kf) step(kt++, std::integral_constant<int, 2 % S>{});
    }
    wait_vmcnt<0>();
    if (kt < kt1) {  // the tail tile: k >= K zero in both operands
        if (!EARLY) {
            fetch_tail(opa, ta, kt, K);
            fetch_tail(opb, tb, kt, K);
        }
        __syncthreads();
        opa.tail_put(ta, lds_a, lane);
        opb.tail_put(tb, lds_b, lane);
        __syncthreads();
        const int groups = (K - kt * BK + 7) / 8;
        f4 fa[FM], fb[FN];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (g < groups) {
                frags(0, g, fa, fb);
                mfmas(fa, fb);
            }
        }
    }

    const int lo = lane & 31, hi = lane >> 5;
    const int r0 = tc.m0 + wm * (BM / WM), c0 = tc.n0 + wn * (BN / WN);
    if (p.t.splits > 1) {
        const int ld = (p.t.N + 3) & ~3;
        int32_t *out = p.partial + (int64_t)tc.split * p.t.M * ld;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = r0 + i * 32 + 8 * (r >> 2) + 4 * hi + (r & 3);
                    const int col = c0 + j * 32 + lo;
                    if (row < p.t.M && col < p.t.N)
                        out[(int64_t)row * ld + col] = acc[i][j][r];
                }
        return;
    }
    T *C = static_cast<T *>(p.C);
    if constexpr (KIND != kProduct) {
        static_assert(S * (A_FL + B_FL) >= WM * WN * 1024, "4 KB of LDS a wavefront");
        if ((int)threadIdx.x < BM + 2 * BN) closing[threadIdx.x] = mine;
        __syncthreads();  // (and every wavefront has read its last operands)
        store_closed<T, KIND, BM, BN, FM, FN>(p, reinterpret_cast<int32_t *>(lds) + wave * 1024,
                                              closing, tc.m0, tc.n0, wm * (BM / WM),
                                              wn * (BN / WN), lane, acc);
        return;
    }
    float sb[FN], bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int col = min(c0 + j * 32 + lo, p.t.N - 1);
        sb[j] = p.sb[col];
        bias[j] = p.bias != nullptr ? p.bias[col] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = r0 + i * 32 + 8 * (r >> 2) + 4 * hi + (r & 3);
            if (row < p.t.M) {
                const float sa = p.sa[row];
                T *c = C + (int64_t)row * p.ldc + c0 + lo;
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    if (c0 + j * 32 + lo < p.t.N) put(c + j * 32, acc[i][j][r], sa, sb[j], bias[j]);
            }
        }
}

// The k ranges' sums added (exactly) and finished: four neighbouring outputs a thread.
template <typename T, int KIND>
__global__ void __launch_bounds__(256) join_int8_kernel(Int8Args p, int64_t plane, FastDiv quads) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    const int row = (int)fast_div(i, quads), col = (int)(i - row * quads.d) * 4;
    if (row >= p.t.M) return;
    const int N = KIND == kGated ? p.outputs : p.t.N;
    const int n = min(4, N - col);
    const int64_t ld = (p.t.N + 3) & ~3;  // (rows padded to 4)
    const int32_t *from =
        p.partial + row * ld + (KIND == kGated ? 2 * (col & ~15) + (col & 15) : col);
    int sum[4] = {0, 0, 0, 0}, up[4] = {0, 0, 0, 0};
    for (int s = 0; s < p.t.splits; ++s) {
        const v4i x = *reinterpret_cast<const v4i *>(from + s * plane);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += x[e];
        if constexpr (KIND == kGated) {
            const v4i y = *reinterpret_cast<const v4i *>(from + s * plane + 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) up[e] += y[e];
        }
    }
    const float a = p.sa[row];
    T *c = static_cast<T *>(p.C) + (int64_t)row * p.ldc + col;
    const float *bias = p.bias;
    if constexpr (KIND == kProduct) {
        for (int e = 0; e < n; ++e)
            put(c + e, sum[e], a, p.sb[col + e], bias != nullptr ? bias[col + e] : 0.f);
    } else {
        const T *res = p.residual != nullptr
                           ? static_cast<const T *>(p.residual) + (int64_t)row * p.ldr + col
                           : nullptr;
        with_activation(p.act, [&](auto act) {
            for (int e = 0; e < n; ++e) {
                const float add = res != nullptr ? to_f32(res[e]) : 0.f;
                const float b = bias != nullptr ? bias[col + e] : 0.f;
                if constexpr (KIND == kGated)
                    put_gated(c + e, act, sum[e], up[e], a, p.sb[col + e], b,
                              p.sb[N + col + e], bias != nullptr ? bias[N + col + e] : 0.f, add);
                else
                    put_act(c + e, act, sum[e], a, p.sb[col + e], b, add);
            }
        });
    }
}

// The tiles' columns: of a gated product each 16 outputs take 32.
template <int KIND>
int tile_columns(int N) {
    return KIND == kGated ? (N + 15) / 16 * 32 : N;
}

template <typename T, int KIND, int BM, int BN, int WM, int WN, int S, int D, int OCC>
int launch_tiles(hipStream_t stream, const Int8Product &p, int splits) {
    Int8Args a{};
    TiledArgs &t = a.t;
    t.A = reinterpret_cast<const float *>(p.A);
    t.B = reinterpret_cast<const float *>(p.B);
    t.lda = p.lda / 4;
    t.ldb = p.ldb / 4;
    t.M = p.M;
    t.N = tile_columns<KIND>(p.N);
    t.K = p.K / 4;
    t.batch = 1;
    t.tiles_m = (p.M + BM - 1) / BM;
    t.tiles_n = (t.N + BN - 1) / BN;
    const int nk = (t.K + BK - 1) / BK;
    const int want = splits < nk ? splits : nk;
    t.kt_per_split = (nk + want - 1) / want;
    t.splits = (nk + t.kt_per_split - 1) / t.kt_per_split;
    const int64_t total = (int64_t)t.tiles_m * t.tiles_n * t.splits;
    if (total > INT32_MAX)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "matmul_int8: %lld tiles exceed one launch",
                         (long long)total);
    t.total = (int)total;
    set_tile_divisors(t);
    a.sa = p.sa;
    a.sb = p.sb;
    a.bias = p.bias;
    a.C = p.C;
    a.ldc = p.ldc;
    a.outputs = p.N;
    a.act = p.act;
    a.residual = p.residual;
    a.ldr = p.ldr;
    const uint32_t quads = (uint32_t)(p.N + 3) / 4;
    const int64_t plane = (int64_t)p.M * ((t.N + 3) / 4 * 4);
    if (t.splits > 1) {
        int rc = MIGEMM_OK;
        a.partial = static_cast<int32_t *>(
            workspace(stream, (size_t)t.splits * plane * sizeof(int32_t), &rc, 0));
        if (a.partial == nullptr) return rc;
    }
    MIGEMM_LAUNCH((gemm_int8_kernel<T, KIND, BM, BN, WM, WN, S, D, OCC>), dim3(t.total),
                  dim3(WM * WN * 64), 0, stream, a);
    if (const int rc = launch_status("gemm_int8_kernel launch")) return rc;
    if (t.splits > 1) {
        const int64_t blocks = ((int64_t)p.M * quads + 255) / 256;
        MIGEMM_LAUNCH((join_int8_kernel<T, KIND>), dim3((unsigned)blocks), dim3(256), 0, stream, a,
                      plane, make_fastdiv(quads));
        if (const int rc = launch_status("join_int8_kernel launch")) return rc;
    }
    record_plan(PlanRecord{"int8-tiles", BM, BN, t.splits, 16, p.M, p.N, p.K, 1, false, true});
    return MIGEMM_OK;
}

// ------------------------------------------------------------------------------- few rows
// A work-group of NW wavefronts takes 16 rows of B (output columns) and all M <= 16 MT rows
// of A; its wavefronts take 128-byte pieces of K in turn. Both operands of
// v_mfma_i32_16x16x64_i8 hold 16 bytes of one row a lane, in any order of k that is the same
// for both: lane group g = lane / 16 takes bytes 32 g .. 32 g + 31 of a piece, so a piece of a
// row is one whole 128-byte line and two instructions. Bound by streaming B: 1 x 4096 to 11008
// (45 MB, quantising its row) 10.2 us a call, 4.4 TB/s; 24 x 2048 to 4096 5.5 us; gated, 1 x 4096
// to 11008 of 22016 (90 MB) 17 us, 5.3 TB/s.
// X != void: A is not given but x [M, K] in X, and each work-group quantises it into LDS
// itself (its first loads of B are on their way meanwhile).
constexpr int kKeep = 3;  // steps of x (NW * 512 values each) that stay in registers
struct RowsArgs {
    const int8_t *A, *B;
    const void *X;
    int64_t lda, ldb, ldx, ldc;
    const float *sa, *sb, *bias;
    void *C;
    int M, N, K, cols;  // K: cols rounded up to 16
    int act;
    const void *residual;
    int64_t ldr;
};

template <typename T, int KIND, typename X, int MT, int NW>
__global__ void __launch_bounds__(NW * 64) rows_int8_kernel(RowsArgs p) {
    constexpr bool FUSED = !std::is_same<X, void>::value;
    constexpr int U = 4;  // pieces in flight
    const int tid = threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const int row = lane & 15, g = lane >> 4;
    // gated: 8 rows of the gate, then the 8 of the other half that belong to them
    constexpr int COLS = KIND == kGated ? 8 : 16;
    const int n0 = blockIdx.x * COLS;
    const int n = min(n0 + (row & (COLS - 1)), p.N - 1);
    const int8_t *b =
        p.B + ((int64_t)n + (KIND == kGated && row >= 8 ? p.N : 0)) * p.ldb + 32 * g;
    const int pieces = (p.K + 127) / 128;

    extern __shared__ __attribute__((aligned(16))) char lds[];
    int32_t *sums = reinterpret_cast<int32_t *>(lds);  // [NW][16 MT][16]
    int8_t *held = reinterpret_cast<int8_t *>(lds + NW * MT * 1024);  // FUSED: [M][K + 16]
    __shared__ uint32_t most[kKeep];
    __shared__ float scales[kKeep];

    v4i rb[U][2];
    auto load_b = [&](int u, int piece) {
        const int k = piece * 128 + 32 * g;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            rb[u][h] = k + 16 * h < p.K
                           ? *reinterpret_cast<const v4i *>(b + (int64_t)piece * 128 + 16 * h)
                           : v4i{0, 0, 0, 0};
    };
    if constexpr (!FUSED) {
#pragma unroll
        for (int u = 0; u < U; ++u) load_b(u, wave + u * NW);
    } else {
        typedef typename std::conditional<FUSED, X, float>::type Xt;
        constexpr int STEP = NW * 64 * 8;  // values that the work-group takes at a time
        const int per_row = (p.K + STEP - 1) / STEP;
        float v[kKeep][8];
        auto at = [&](int c, int &m, int &k) {  // step c: row m, this thread's first column k
            m = c / per_row;
            k = (c - m * per_row) * STEP + tid * 8;
        };
        // x first: loads come back in order, and x is in L2
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            int m, k;
            at(c, m, k);
            if (m < p.M)
                load_f32<Xt, 8>(static_cast<const Xt *>(p.X) + (int64_t)m * p.ldx + k,
                                p.cols - k, v[c]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) load_b(u, wave + u * NW);
        if (tid < kKeep) most[tid] = 0;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            int m, k;
            at(c, m, k);
            if (m < p.M) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t bits = __float_as_uint(v[c][i]) & 0x7fffffffu;
                    top = bits > top ? bits : top;
                }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    const uint32_t other = __shfl_xor(top, o);
                    top = other > top ? other : top;
                }
                if (lane == 0) atomicMax(&most[m], top);  // (a maximum: in any order the same)
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kKeep; ++c) {
            int m, k;
            at(c, m, k);
            if (m < p.M && k < p.K) {
                const float inv = inverse_scale(scale_of(most[m]));
                uint2 q;
                q.x = pack4(held_byte(v[c][0], inv), held_byte(v[c][1], inv),
                            held_byte(v[c][2], inv), held_byte(v[c][3], inv));
                q.y = pack4(held_byte(v[c][4], inv), held_byte(v[c][5], inv),
                            held_byte(v[c][6], inv), held_byte(v[c][7], inv));
                *reinterpret_cast<uint2 *>(held + (int64_t)m * (p.K + 16) + k) = q;
            }
        }
        if (tid < p.M) scales[tid] = scale_of(most[tid]);
        __syncthreads();
    }

    v4i acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = v4i{0, 0, 0, 0};
    const int8_t *a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = min(16 * i + row, p.M - 1);
        if constexpr (FUSED)
            a[i] = held + m * (p.K + 16);
        else
            a[i] = p.A + (int64_t)m * p.lda;
    }
    for (int piece = wave; piece < pieces; piece += U * NW) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = piece + u * NW;
            if (at < pieces) {
                v4i ra[MT][2];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int k = at * 128 + 32 * g + 16 * h;
                        ra[i][h] = k < p.K ? *reinterpret_cast<const v4i *>(a[i] + k)
                                           : v4i{0, 0, 0, 0};
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ra[i][h], rb[u][h],
                                                                       acc[i], 0, 0, 0);
                load_b(u, at + U * NW);
            }
        }
    }
    // Lane: column lane % 16 (a row of B), rows 4 g + 0..3 of each block of 16.
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            sums[((wave * MT + i) * 16 + 4 * g + r) * 16 + row] = acc[i][r];
    __syncthreads();
    for (int e = tid; e < MT * 256; e += NW * 64) {
        const int m = e >> 4, c = n0 + (e & 15);
        if (m >= p.M || c >= p.N || (e & 15) >= COLS) continue;
        int sum = 0, up = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += sums[w * MT * 256 + e];
        if constexpr (KIND == kGated) {
#pragma unroll
            for (int w = 0; w < NW; ++w) up += sums[w * MT * 256 + e + 8];
        }
        const float sa = FUSED ? scales[m] : p.sa[m];
        const float sb = p.sb[c], bias = p.bias != nullptr ? p.bias[c] : 0.f;
        T *out = static_cast<T *>(p.C) + (int64_t)m * p.ldc + c;
        if constexpr (KIND == kProduct) {
            put(out, sum, sa, sb, bias);
        } else {
            const float add =
                p.residual != nullptr
                    ? to_f32(static_cast<const T *>(p.residual)[(int64_t)m * p.ldr + c])
                    : 0.f;
            with_activation(p.act, [&](auto act) {
                if constexpr (KIND == kGated)
                    put_gated(out, act, sum, up, sa, sb, bias, p.sb[p.N + c],
                              p.bias != nullptr ? p.bias[p.N + c] : 0.f, add);
                else
                    put_act(out, act, sum, sa, sb, bias, add);
            });
        }
    }
}

template <typename T, int KIND, typename X, int MT, int NW>
int launch_rows(hipStream_t stream, const RowsArgs &a) {
    const size_t lds = (size_t)NW * MT * 1024 +
                       (std::is_same<X, void>::value ? 0 : (size_t)a.M * (a.K + 16));
    constexpr int COLS = KIND == kGated ? 8 : 16;
    MIGEMM_LAUNCH((rows_int8_kernel<T, KIND, X, MT, NW>), dim3((a.N + COLS - 1) / COLS),
                  dim3(NW * 64), lds, stream, a);
    record_plan(PlanRecord{std::is_same<X, void>::value ? "int8-rows" : "int8-rows-fused",
                           16 * MT, 16, NW, 16, a.M, a.N, a.K, 1, false, true});
    return launch_status("rows_int8_kernel launch");
}

RowsArgs rows_args(const Int8Product &p) {
    RowsArgs a{};
    a.A = p.A;
    a.B = p.B;
    a.lda = p.lda;
    a.ldb = p.ldb;
    a.ldc = p.ldc;
    a.sa = p.sa;
    a.sb = p.sb;
    a.bias = p.bias;
    a.C = p.C;
    a.M = p.M;
    a.N = p.N;
    a.K = a.cols = p.K;
    a.act = p.act;
    a.residual = p.residual;
    a.ldr = p.ldr;
    return a;
}

// What a choice costs, in work of one CU at the best tiles' rate: rounds of work-groups over
// the 256 CUs, a tile's products over the rate that its shape reaches. Rates measured against
// 256 x 256 (at 8192^3): 128 x 256 0.88, 128 x 128 0.84, 64 x 128 0.70, 64 x 64 0.55. (Where a
// round is not full the choice hardly matters: 1000 x 3000 x 784 takes 12.5 us in 128 x 128, 12.8 in
// 64 x 128, 12.6 in 64 x 64, 17.3 in 128 x 256.)
struct TileChoice {
    int bm, bn;
    float rate;
};
constexpr TileChoice kTiles[] = {
    {256, 256, 1.f}, {128, 256, 0.88f}, {128, 128, 0.84f}, {64, 128, 0.70f}, {64, 64, 0.55f}};

template <typename T, int KIND>
int launch_product(hipStream_t stream, const Int8Product &p) {
    const int N = tile_columns<KIND>(p.N);  // (what is said of N goes by the rows of B)
    // Few rows: 16 columns a work-group (24 x 4096 x 2048: 4.2 us, tiles 6.8; with the quantising
    // before it 16 x 4096 x 4096 10.2, 12.5; 16 x 8192 x 8192 23.2, 29.7). Not where many columns
    // read A, each work-group all of it: there the tiles stream B as well and read A once for 64
    // columns (16 x 11008 x 4096: 18.4, 17.6; 16 x 32000 x 4096 35.5, 25.9; 24 x 4096 x 11008
    // 22.4, 20.5). And not over long K of few columns, as a work-group's time grows with K (alone, up
    // to a work-group a CU) and tiles cut it in ranges: M <= 16 8.1 us at 512 x 8192 (tiles 9.9), 9.7
    // (10.4) at 10240, 11.0 (11.1) at 12288, 13.7 (11.4) at 16384, 64.7 (22.7) at 64 x 131056; M <=
    // 32 9.1 (10.7) at 512 x 5120, 10.3 (10.3) at 6144, 11.6 (10.2) at 8192.
    if ((p.M <= 32 && (int64_t)N * p.K <= (int64_t)12 << 20 &&
         p.K <= (p.M <= 16 ? 10240 : 6144)) ||
        (p.M <= 16 && N >= 2048 && N <= 8192)) {
        const RowsArgs a = rows_args(p);
        return p.M <= 16 ? launch_rows<T, KIND, void, 1, 8>(stream, a)
                         : launch_rows<T, KIND, void, 2, 8>(stream, a);
    }
    auto tiles = [&](const TileChoice &c) {
        return (int64_t)((p.M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    };
    int best = 0;
    float least = INFINITY;
    for (int i = 0; i < 5; ++i) {
        const TileChoice &c = kTiles[i];
        const float cost = (float)((tiles(c) + 255) / 256) * (float)(c.bm * c.bn) / c.rate;
        if (cost < least) {
            least = cost;
            best = i;
        }
    }
    switch (best) {
        case 0: return launch_tiles<T, KIND, 256, 256, 8, 2, 2, 2, 4>(stream, p, 1);
        case 1: return launch_tiles<T, KIND, 128, 256, 4, 4, 3, 3, 4>(stream, p, 1);
        case 2: return launch_tiles<T, KIND, 128, 128, 4, 4, 2, 2, 4>(stream, p, 1);
        case 3: return launch_tiles<T, KIND, 64, 128, 2, 4, 3, 3, 4>(stream, p, 1);
    }
    // Too few of the smallest tiles for the CUs: k ranges, each of 16 stages at least (they
    // cost a second launch), until there is a work-group for each CU (128 x 4096 x 11008 in two:
    // 27 us, 37 whole; with two for each CU 64 x 4096 x 11008 takes 24.6 instead of 20.9, 256 x
    // 4096 x 4096 18.9 instead of 16.4).
    const int64_t n = tiles(kTiles[4]);
    const int splits = n > 256 ? 1 : (int)(256 / n);
    const int most = p.K / 2048 > 1 ? p.K / 2048 : 1;
    return launch_tiles<T, KIND, 64, 64, 2, 2, 3, 3, 3>(stream, p, splits < most ? splits : most);
}

// Up to three rows that a work-group of 8 wavefronts holds in its registers: quantised by each
// (1 x 4096 to 11008, weights from HBM: 10.4 us, against 3 and 10.5 by two launches; 2 x 4096
// to 4096: 5.9, and 3 and 5.0; 3 x 4096 to 11008 13.1 and 17.0 together, 1 x 11008 to 4096 12.9
// and 17.1). Room for a fourth step costs a wavefront a SIMD (1 x 4096 to 11008: 12.5).
bool fused_rows(int M, int K) { return M <= kKeep && M * ((K + 4095) / 4096) <= kKeep; }

template <int KIND>
int product_int8(hipStream_t stream, const Int8Product &p) {
    return p.type == MIGEMM_FLOAT32 ? launch_product<float, KIND>(stream, p)
                                    : launch_product<Bf16, KIND>(stream, p);
}

template <int KIND>
int linear_int8(hipStream_t stream, const void *X, int64_t ldx, int cols, const Int8Product &q) {
    Int8Product p = q;
    if (fused_rows(p.M, p.K)) {
        RowsArgs a = rows_args(p);
        a.X = X;
        a.ldx = ldx;
        a.cols = cols;
        return p.type == MIGEMM_FLOAT32 ? launch_rows<float, KIND, float, 1, 8>(stream, a)
                                        : launch_rows<Bf16, KIND, Bf16, 1, 8>(stream, a);
    }
    // the quantised rows and their scales: staged operands (the products' partial sums are in
    // the stream's other buffer)
    int rc = MIGEMM_OK;
    const size_t bytes = (size_t)p.M * p.K;
    char *ws = static_cast<char *>(
        workspace(stream, bytes + (size_t)p.M * sizeof(float) + 16, &rc, 1));
    if (ws == nullptr) return rc;
    int8_t *held = reinterpret_cast<int8_t *>(ws);
    float *scales = reinterpret_cast<float *>(ws + ((bytes + 15) & ~(size_t)15));
    rc = launch_quantize_rows(stream, X, p.type, ldx, held, p.K, scales, p.M, cols);
    if (rc != MIGEMM_OK) return rc;
    p.A = held;
    p.lda = p.K;
    p.sa = scales;
    return product_int8<KIND>(stream, p);
}
}  // namespace
}  // namespace migemm
