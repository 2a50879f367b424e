// Shared by the 8-bit operators (quantised rows and products, the 8-bit paged cache and the
// attention that reads it): activation types, the quantisation rule, and int8 -> bf16.
#pragma once

#include "migemm_internal.h"

namespace migemm {

// ---- launchers (validated arguments; they only enqueue work) ----------------------------
struct Int8Product {
    const int8_t *A, *B;  // [M, K], [N, K], rows lda / ldb bytes apart
    const float *sa, *sb, *bias;
    void *C;
    int64_t lda, ldb, ldc;
    int M, N, K, type;
};
int launch_quantize_rows(hipStream_t stream, const void *X, int type, int64_t ldx,
                         int8_t *values, int64_t ldv, float *scales, int rows, int cols);
int launch_product_int8(hipStream_t stream, const Int8Product &p);
// The layer: x quantised by rows, then the product (one launch for a few rows).
int launch_linear_int8(hipStream_t stream, const void *X, int64_t ldx, int cols,
                       const Int8Product &p);

struct TablesArgs {
    const int *lengths, *counts;
    int requests;
    int *table;
    int max_pages, page_size;
    const int *free_pages, *free_count;  // null: slots of the pages that the table holds
    int free_capacity;
    int *slots, *positions, *starts, *new_lengths, *new_free;
    int tokens;
};
int launch_cache_tables(hipStream_t stream, const TablesArgs &a);
int launch_cache_release(hipStream_t stream, const int *finished, int *lengths, int requests,
                         int *table, int max_pages, int page_size, int *free_pages, int pages,
                         int *free_count);

struct Cache8 {
    int8_t *keys;    // [pages, heads, page_size, width]
    int8_t *values;  // [pages, heads, width, page_size]
    float *key_scales, *value_scales;  // [pages, heads]
    int pages, heads, dim, width, page_size;
};
int launch_cache_append(hipStream_t stream, const void *K, const void *V, int type,
                        int64_t ldk, int64_t ldv, const int *slots, int tokens,
                        const Cache8 &c);
int launch_cache_read(hipStream_t stream, const Cache8 &c, const int *slots, int tokens,
                      void *K, void *V, int type);

struct CacheAttention {
    const void *Q;
    void *O;
    int type;
    int64_t ldq;
    Cache8 c;
    const int *table, *starts, *positions;
    int max_pages, requests, tokens, heads;  // heads: of queries
    float scale;
    int max_count, max_length;  // what the launch is shaped for; any call is computed right
};
int launch_cache_attention(hipStream_t stream, const CacheAttention &a);

#ifdef __HIPCC__
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));

// Loads and stores of any alignment (a row may begin at any element; the hardware takes
// unaligned vector accesses to global memory).
template <typename V>
__device__ __forceinline__ V load_any(const void *p) {
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <typename V>
__device__ __forceinline__ void store_any(void *p, const V &v) {
    __builtin_memcpy(p, &v, sizeof(V));
}

// Activation types: float32 and bfloat16 (kept as its 16 bits, rounded to nearest even).
struct Bf16 {
    uint16_t b;
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(Bf16 x) { return __uint_as_float((uint32_t)x.b << 16); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ Bf16 from_f32<Bf16>(float x) {
    __bf16 h = (__bf16)x;
    Bf16 r;
    __builtin_memcpy(&r, &h, 2);
    return r;
}

// N neighbouring values as float32; those at and after `left` are 0 and not read.
template <typename T, int N>
__device__ __forceinline__ void load_f32(const T *p, int left, float (&x)[N]) {
    if (left >= N) {
        struct Raw {
            T t[N];
        };
        Raw r;
        __builtin_memcpy(&r, p, sizeof(r));
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_f32(r.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? to_f32(p[i]) : 0.f;
    }
}

// The scale of a row (or of a page and head) whose largest magnitude has the bits `most`
// (magnitudes of floats order as their bits do, infinities and NaN above every number):
// fl(a / 127); 0 where that is subnormal, as its reciprocal would lose bits; NaN where a
// value is not finite, so that what is computed from it is NaN and never silently finite.
__device__ __forceinline__ float scale_of(uint32_t most) {
    if (most >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    const float s = __uint_as_float(most) / 127.0f;
    return s < 1.17549435e-38f ? 0.0f : s;
}
// fl(1 / s), 0 for a scale of 0 or NaN (the values are then 0).
__device__ __forceinline__ float inverse_scale(float s) { return s > 0.0f ? 1.0f / s : 0.0f; }

// rint(fl(x * inv)) as the low byte. |x * inv| <= 127 (1 + 2^-22), and adding 1.5 * 2^23
// rounds to integers, half to even, in the adder; the product is rounded first (a fused
// multiply-add would not, and a tie would then go by bits that the rule drops).
__device__ __forceinline__ uint32_t held_byte(float x, float inv) {
#pragma clang fp contract(off)
    const float y = x * inv;
    return __float_as_uint(y + 12582912.0f);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return lo | (hi << 16);
}

// What a loop loaded a round ahead, at its use: keeps the compiler from unpacking it where it was
// loaded (which waits for the load there, and spills).
__device__ __forceinline__ void pin(v4i &x) { asm volatile("" : "+v"(x)); }

// Four signed bytes as bf16: exact (|v| <= 127 has 7 significant bits), so only the upper
// half of each float is kept.
__device__ __forceinline__ void bytes_to_bf16(uint32_t v, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __float_as_uint((float)(int8_t)(v));
    const uint32_t b = __float_as_uint((float)(int8_t)(v >> 8));
    const uint32_t c = __float_as_uint((float)(int8_t)(v >> 16));
    const uint32_t d = __float_as_uint((float)(int8_t)(v >> 24));
    lo = __builtin_amdgcn_perm(b, a, 0x07060302u);
    hi = __builtin_amdgcn_perm(d, c, 0x07060302u);
}
__device__ __forceinline__ v8bf bytes8_to_bf16(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        v8bf v;
    } r;
    bytes_to_bf16(a, r.u[0], r.u[1]);
    bytes_to_bf16(b, r.u[2], r.u[3]);
    return r.v;
}
// Four signed bytes as f16, exact: byte + 128 as the low bits of 1024 + x, less 1152.
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void bytes_to_f16(uint32_t v, uint32_t &lo, uint32_t &hi) {
    const uint32_t x = v ^ 0x80808080u;
    const v2h less = {(_Float16)-1152.f, (_Float16)-1152.f};
    const v2h a = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(x, 0x64646464u, 0x00050004u));
    const v2h b = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(x, 0x64646464u, 0x00070006u));
    lo = __builtin_bit_cast(uint32_t, a + less);
    hi = __builtin_bit_cast(uint32_t, b + less);
}
__device__ __forceinline__ v8h bytes8_to_f16(uint32_t a, uint32_t b) {
    union {
        uint32_t u[4];
        v8h v;
    } r;
    bytes_to_f16(a, r.u[0], r.u[1]);
    bytes_to_f16(b, r.u[2], r.u[3]);
    return r.v;
}
// Two floats as two bf16, rounded to nearest even.
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2bf));
}
// The same as two f16.
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2h));
}
__device__ __forceinline__ float bf16_low(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_high(uint32_t u) {
    return __uint_as_float(u & 0xffff0000u);
}
#endif

}  // namespace migemm
