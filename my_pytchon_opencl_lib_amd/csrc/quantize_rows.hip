// Rows of activations or weights in 8 bits, with a float32 scale for each row.
//
//   s[r] = fl(max_k |x[r, k]| / 127),  v[r, k] = rint(fl(x[r, k] * fl(1 / s[r])))
//
// (scale_of, held_byte). One pass over the data: a row stays in registers between the
// maximum and the rounding, so x is read once and a byte a value written: bound by memory
// (8192 x 4096 bfloat16: 22 us, 4.5 TB/s; 1000 x 777 float32: 3.0 to 4.0 us, a launch's latency).
// A wavefront takes a row of up to 2048 values (four rows a work-group, no barrier); longer
// ones take a work-group of 256 threads, which keeps 16384 values and reads what is beyond
// them twice (from L2).
#include "int8_common.h"

namespace migemm {
namespace {

// TPR threads a row, each CH chunks of 8 neighbouring values in registers.
template <typename T, int TPR, int CH>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T *X, int64_t ldx, int8_t *V, int64_t ldv, float *S, int rows,
                     int cols) {
    constexpr int RPB = 256 / TPR;
    const int t = threadIdx.x % TPR;
    const int r = blockIdx.x * RPB + threadIdx.x / TPR;
    __shared__ uint32_t part[4];
    if (TPR == 64 && r >= rows) return;  // (a wavefront of its own; TPR 256 has a row always)
    const T *x = X + (int64_t)r * ldx;
    float v[CH][8];
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int k = (c * TPR + t) * 8;
        load_f32<T, 8>(x + k, cols - k, v[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = __float_as_uint(v[c][i]) & 0x7fffffffu;
            most = b > most ? b : most;
        }
    for (int k = (CH * TPR + t) * 8; k < cols; k += TPR * 8) {
        float w[8];
        load_f32<T, 8>(x + k, cols - k, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = __float_as_uint(w[i]) & 0x7fffffffu;
            most = b > most ? b : most;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor(most, o);
        most = b > most ? b : most;
    }
    if constexpr (TPR == 256) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) most = part[i] > most ? part[i] : most;
    }
    const float s = scale_of(most);
    const float inv = inverse_scale(s);
    if (t == 0) S[r] = s;
    int8_t *out = V + (int64_t)r * ldv;
    const int padded = (cols + 15) & ~15;  // the columns that are added are zeros
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int k = (c * TPR + t) * 8;
        uint2 q;
        q.x = pack4(held_byte(v[c][0], inv), held_byte(v[c][1], inv), held_byte(v[c][2], inv),
                    held_byte(v[c][3], inv));
        q.y = pack4(held_byte(v[c][4], inv), held_byte(v[c][5], inv), held_byte(v[c][6], inv),
                    held_byte(v[c][7], inv));
        if (k < padded) *reinterpret_cast<uint2 *>(out + k) = q;
    }
    for (int k = (CH * TPR + t) * 8; k < padded; k += TPR * 8) {
        float w[8];
        load_f32<T, 8>(x + k, cols - k, w);
        uint2 q;
        q.x = pack4(held_byte(w[0], inv), held_byte(w[1], inv), held_byte(w[2], inv),
                    held_byte(w[3], inv));
        q.y = pack4(held_byte(w[4], inv), held_byte(w[5], inv), held_byte(w[6], inv),
                    held_byte(w[7], inv));
        *reinterpret_cast<uint2 *>(out + k) = q;
    }
}

template <typename T>
void launch(hipStream_t stream, const T *X, int64_t ldx, int8_t *V, int64_t ldv, float *S,
            int rows, int cols) {
    if (cols <= 512)
        MIGEMM_LAUNCH((quantize_rows_kernel<T, 64, 1>), dim3((rows + 3) / 4), dim3(256), 0,
                      stream, X, ldx, V, ldv, S, rows, cols);
    else if (cols <= 2048)
        MIGEMM_LAUNCH((quantize_rows_kernel<T, 64, 4>), dim3((rows + 3) / 4), dim3(256), 0,
                      stream, X, ldx, V, ldv, S, rows, cols);
    else if (cols <= 4096)
        MIGEMM_LAUNCH((quantize_rows_kernel<T, 256, 2>), dim3(rows), dim3(256), 0, stream, X,
                      ldx, V, ldv, S, rows, cols);
    else
        MIGEMM_LAUNCH((quantize_rows_kernel<T, 256, 8>), dim3(rows), dim3(256), 0, stream, X,
                      ldx, V, ldv, S, rows, cols);
}
}  // namespace

int launch_quantize_rows(hipStream_t stream, const void *X, int type, int64_t ldx,
                         int8_t *values, int64_t ldv, float *scales, int rows, int cols) {
    if (type == MIGEMM_FLOAT32)
        launch(stream, static_cast<const float *>(X), ldx, values, ldv, scales, rows, cols);
    else
        launch(stream, static_cast<const Bf16 *>(X), ldx, values, ldv, scales, rows, cols);
    return launch_status("quantize_rows_kernel launch");
}

}  // namespace migemm
