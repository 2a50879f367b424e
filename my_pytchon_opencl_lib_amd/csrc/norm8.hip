// Rows after a residual's addition and their root-mean-square norm, in 8 bits with a float32
// scale for each row, as the 8-bit products take them:
//
//   t[r, k] = x[r, k] + res[r, k], rounded to the activations' type (the residual stream goes on
//             with it, so it is what is normed)
//   q[r]    = fl(1 / sqrt(mean_k t[r, k]^2 + eps))
//   y[r, k] = fl(fl(t[r, k] * q[r]) * w[k])
//   s[r]    = fl(max_k |y[r, k]| / 127),  v[r, k] = rint(fl(y[r, k] * fl(1 / s[r])))
//
// Squares and their sum are in 64 bits and q is rounded to 32 once: its bits then do not depend on
// the order of the sum (but where the 64-bit value lies within some 2^-50 of a tie), every later
// step is one correctly rounded float32 operation, and rows are checked bit for bit. The 64-bit
// operations, two a value, pass under the loads.
//
// One pass over the data: a row stays in registers between its sum of squares, its maximum and the
// rounding, so x and the residual are read once and the sum and a byte a value written: bound by
// memory. 8192 x 4096 in bfloat16 with a residual take 47-49 us, 4.9 TB/s read and written, where
// a large copy reaches 5.1; 1 x 4096 takes 3.5 us and 1000 x 777 in float32 5.3 us, a launch and
// the latency of its loads. The weight is loaded with the row, so that its latency passes under
// the sum of squares (loaded where it is used, 4096 x 777 in bfloat16 took 11.4 us and now 9.0).
//
// A wavefront takes a row of up to 2048 values (four rows a work-group, no barrier); longer ones
// take a work-group. What a thread keeps of a row decides how many rows are in flight: at 4096
// rows of 8192 in bfloat16, 512 threads with 16 values each take 46 us, 256 with 32 48 us and 256
// with 64 93 us; 2048 rows of 16384 take 48 us in 512 threads with 32 values, 56 in 1024 with 16.
// Up to 4096 values 256 threads with 16 are ahead of 512 with 8 by 5 % in bfloat16 with many rows
// (24.2 us against 25.4) and behind by 4 % in float32. What is beyond 16384 values is read three
// times, from L2 (1024 x 20000: 35 us).
#include "int8_common.h"

namespace migemm {
namespace {

// Eight neighbouring sums, rounded to T; those at and after `left` are 0.
template <typename T, bool RES>
__device__ __forceinline__ void load_sum(const T *x, const T *res, int left, float (&v)[8]) {
    load_f32<T, 8>(x, left, v);
    if constexpr (RES) {
        float a[8];
        load_f32<T, 8>(res, left, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(from_f32<T>(v[i] + a[i]));
    }
}

template <typename T>
__device__ __forceinline__ void store_sum(T *out, int left, const float (&v)[8]) {
    struct Raw {
        T t[8];
    } r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.t[i] = from_f32<T>(v[i]);
    if (left >= 8) {
        store_any(out, r);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) out[i] = r.t[i];
    }
}

// (Times a weight of 1 nothing is rounded.)
__device__ __forceinline__ void load_weight(const float *w, int k, int cols, float (&a)[8]) {
    if (w != nullptr) {
        load_f32<float, 8>(w + k, cols - k, a);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = 1.f;
    }
}
__device__ __forceinline__ void normed(float (&v)[8], float q, const float (&a)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * q * a[i];
}

__device__ __forceinline__ uint32_t magnitude(const float (&v)[8], uint32_t most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
        most = b > most ? b : most;
    }
    return most;
}

__device__ __forceinline__ void store_bytes(int8_t *out, const float (&v)[8], float inv) {
    uint2 q;
    q.x = pack4(held_byte(v[0], inv), held_byte(v[1], inv), held_byte(v[2], inv),
                held_byte(v[3], inv));
    q.y = pack4(held_byte(v[4], inv), held_byte(v[5], inv), held_byte(v[6], inv),
                held_byte(v[7], inv));
    *reinterpret_cast<uint2 *>(out) = q;
}

// TPR threads a row, each CH chunks of 8 neighbouring values in registers.
template <typename T, bool RES, int TPR, int CH>
__global__ void __launch_bounds__(TPR == 64 ? 256 : TPR) norm_int8_kernel(NormInt8 p) {
    constexpr int RPB = TPR == 64 ? 4 : 1;
    const int t = threadIdx.x % TPR;
    const int r = blockIdx.x * RPB + threadIdx.x / TPR;
    __shared__ double part[TPR / 64];
    __shared__ uint32_t tops[TPR / 64];
    if (TPR == 64 && r >= p.rows) return;  // (a wavefront of its own; a work-group has its row)
    const T *x = static_cast<const T *>(p.X) + (int64_t)r * p.ldx;
    const T *res = RES ? static_cast<const T *>(p.R) + (int64_t)r * p.ldr : nullptr;
    T *sum = RES && p.S != nullptr ? static_cast<T *>(p.S) + (int64_t)r * p.lds : nullptr;
    const int cols = p.cols;
    float v[CH][8], weight[CH][8];  // (the weight is on its way while squares are summed)
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int k = (c * TPR + t) * 8;
        load_sum<T, RES>(x + k, res + k, cols - k, v[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) load_weight(p.weight, (c * TPR + t) * 8, cols, weight[c]);
    double squares = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int k = (c * TPR + t) * 8;
        if (RES && sum != nullptr) store_sum<T>(sum + k, cols - k, v[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            squares = __builtin_fma((double)v[c][i], (double)v[c][i], squares);
    }
    for (int k = (CH * TPR + t) * 8; k < cols; k += TPR * 8) {
        float a[8];
        load_sum<T, RES>(x + k, res + k, cols - k, a);
        if (RES && sum != nullptr) store_sum<T>(sum + k, cols - k, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) squares = __builtin_fma((double)a[i], (double)a[i], squares);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) squares += __shfl_xor(squares, o);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = squares;
        __syncthreads();
        squares = part[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) squares += part[i];
    }
    const float q = (float)(1.0 / __builtin_sqrt(squares / (double)cols + (double)p.eps));

    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        normed(v[c], q, weight[c]);
        most = magnitude(v[c], most);
    }
    for (int k = (CH * TPR + t) * 8; k < cols; k += TPR * 8) {
        float a[8], b[8];
        load_sum<T, RES>(x + k, res + k, cols - k, a);
        load_weight(p.weight, k, cols, b);
        normed(a, q, b);
        most = magnitude(a, most);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor(most, o);
        most = b > most ? b : most;
    }
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TPR / 64; ++i) most = tops[i] > most ? tops[i] : most;
    }
    const float s = scale_of(most);
    const float inv = inverse_scale(s);
    if (t == 0) p.scales[r] = s;
    int8_t *out = p.values + (int64_t)r * p.ldv;
    const int padded = (cols + 15) & ~15;  // the columns that are added are zeros
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int k = (c * TPR + t) * 8;
        if (k < padded) store_bytes(out + k, v[c], inv);
    }
    for (int k = (CH * TPR + t) * 8; k < padded; k += TPR * 8) {
        float a[8], b[8];
        load_sum<T, RES>(x + k, res + k, cols - k, a);
        load_weight(p.weight, k, cols, b);
        normed(a, q, b);
        store_bytes(out + k, a, inv);
    }
}

template <typename T, bool RES>
void launch(hipStream_t stream, const NormInt8 &p) {
    const dim3 waves((p.rows + 3) / 4), groups(p.rows), block(norm_int8_threads(p.cols));
    if (p.cols <= 512)
        MIGEMM_LAUNCH((norm_int8_kernel<T, RES, 64, 1>), waves, block, 0, stream, p);
    else if (p.cols <= 1024)
        MIGEMM_LAUNCH((norm_int8_kernel<T, RES, 64, 2>), waves, block, 0, stream, p);
    else if (p.cols <= 2048)
        MIGEMM_LAUNCH((norm_int8_kernel<T, RES, 64, 4>), waves, block, 0, stream, p);
    else if (p.cols <= 4096)
        MIGEMM_LAUNCH((norm_int8_kernel<T, RES, 256, 2>), groups, block, 0, stream, p);
    else if (p.cols <= 8192)
        MIGEMM_LAUNCH((norm_int8_kernel<T, RES, 512, 2>), groups, block, 0, stream, p);
    else
        MIGEMM_LAUNCH((norm_int8_kernel<T, RES, 512, 4>), groups, block, 0, stream, p);
}
}  // namespace

int launch_norm_int8(hipStream_t stream, const NormInt8 &p) {
    if (p.type == MIGEMM_FLOAT32)
        p.R != nullptr ? launch<float, true>(stream, p) : launch<float, false>(stream, p);
    else
        p.R != nullptr ? launch<Bf16, true>(stream, p) : launch<Bf16, false>(stream, p);
    return launch_status("norm_int8_kernel launch");
}

}  // namespace migemm
