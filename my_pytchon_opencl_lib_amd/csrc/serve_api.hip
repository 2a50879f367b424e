// C ABI of the 8-bit serving operators (include/migemm.h, 6): argument validation before any
// HIP call, and the shape of the attention's launches.
#include <algorithm>
#include <initializer_list>

#include "cache_attention.h"

namespace migemm {
namespace {

struct Range {
    const void *p;
    int64_t bytes;
};

bool overlap(const Range &a, const Range &b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return a.bytes > 0 && b.bytes > 0 && x < y + (uintptr_t)b.bytes &&
           y < x + (uintptr_t)a.bytes;
}

// Outputs may overlap neither inputs nor each other.
int check_alias(const char *what, std::initializer_list<Range> outs,
                std::initializer_list<Range> ins) {
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        for (const Range &i : ins)
            if (overlap(*o, i))
                return set_error(MIGEMM_ERR_ALIAS, "%s: an output overlaps an input", what);
        for (auto q = outs.begin(); q != o; ++q)
            if (overlap(*o, *q))
                return set_error(MIGEMM_ERR_ALIAS, "%s: two outputs overlap", what);
    }
    return MIGEMM_OK;
}

int check_pointers(const char *what, std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (p == nullptr)
            return set_error(MIGEMM_ERR_INVALID_ARG, "%s: null pointer", what);
    return MIGEMM_OK;
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int type_size(int type) { return type == MIGEMM_FLOAT32 ? 4 : 2; }

int check_type(const char *what, int type) {
    if (type != MIGEMM_FLOAT32 && type != MIGEMM_BFLOAT16)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: type %d is neither MIGEMM_FLOAT32 nor "
                         "MIGEMM_BFLOAT16", what, type);
    return MIGEMM_OK;
}

// A launch holds fewer than 2^32 threads.
int check_grid(const char *what, int64_t blocks, int threads) {
    if (blocks * threads >= (int64_t)1 << 32)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: %lld work-groups of %d threads exceed one "
                         "launch", what, (long long)blocks, threads);
    return MIGEMM_OK;
}

constexpr int64_t kMaxStride = (int64_t)1 << 28;  // elements: rows * stride cannot overflow

int64_t rows_bytes(int64_t rows, int64_t ld, int64_t cols, int size) {
    return rows < 1 ? 0 : ((rows - 1) * ld + cols) * size;
}

int check_ld(const char *what, const char *name, int64_t ld, int64_t cols) {
    if (ld < cols || ld > kMaxStride)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: %s=%lld, must be %lld..2^28", what, name,
                         (long long)ld, (long long)cols);
    return MIGEMM_OK;
}

#define MIGEMM_TRY(x)                      \
    do {                                   \
        const int _rc = (x);               \
        if (_rc != MIGEMM_OK) return _rc;  \
    } while (0)

int check_product(const char *what, int M, int N, int K) {
    if (M < 1 || N < 1 || K < 1)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: sizes must be >= 1 (M=%d N=%d K=%d)", what,
                         M, N, K);
    if (K > 131071)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: K=%d, int32 sums hold K <= 131071", what,
                         K);
    // the largest grid of the kernels: one work-group of 512 threads for 16 columns, or for a
    // tile of 64 x 64 at least
    MIGEMM_TRY(check_grid(what, ((int64_t)N + 15) / 16, 512));
    return check_grid(what, (((int64_t)M + 63) / 64) * (((int64_t)N + 63) / 64), 256);
}

int check_int8_rows(const char *what, const char *name, const int8_t *p, int64_t ld, int K) {
    if (ld < K || ld % 16 != 0 || ld > (int64_t)1 << 23)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: ld%s=%lld, must be a multiple of 16 in "
                         "%d..2^23", what, name, (long long)ld, K);
    if (!aligned(p, 16))
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: %s must be 16-byte aligned", what, name);
    return MIGEMM_OK;
}

int check_cache(const char *what, const Cache8 &c) {
    MIGEMM_TRY(check_pointers(what, {c.keys, c.values, c.key_scales, c.value_scales}));
    if (c.pages < 1 || c.heads < 1 || c.heads > 65535)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: pages=%d must be >= 1, kv_heads=%d in "
                         "1..65535", what, c.pages, c.heads);
    if (c.dim < 8 || c.dim > 256 || c.dim % 8 != 0)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: head_dim=%d, must be a multiple of 8 in "
                         "8..256", what, c.dim);
    if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: page_size=%d, must be 16, 32, 64 or 128",
                         what, c.page_size);
    if ((int64_t)c.pages * c.page_size > INT32_MAX)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: %d pages of %d tokens exceed the int32 "
                         "slots", what, c.pages, c.page_size);
    if (!aligned(c.keys, 16) || !aligned(c.values, 16) || !aligned(c.key_scales, 4) ||
        !aligned(c.value_scales, 4))
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: keys and values must be 16-byte aligned, "
                         "scales 4-byte", what);
    return MIGEMM_OK;
}

int width_of(int dim) { return dim <= 128 ? (dim + 31) / 32 * 32 : (dim + 63) / 64 * 64; }

Cache8 make_cache(const int8_t *keys, const int8_t *values, const float *ks, const float *vs,
                  int pages, int heads, int dim, int page_size) {
    Cache8 c{};
    c.keys = const_cast<int8_t *>(keys);
    c.values = const_cast<int8_t *>(values);
    c.key_scales = const_cast<float *>(ks);
    c.value_scales = const_cast<float *>(vs);
    c.pages = pages;
    c.heads = heads;
    c.dim = dim;
    c.width = width_of(dim);
    c.page_size = page_size;
    return c;
}

int64_t cache_bytes(const Cache8 &c) {
    return (int64_t)c.pages * c.page_size * c.heads * c.width;
}
int64_t scale_bytes(const Cache8 &c) { return (int64_t)c.pages * c.heads * 4; }

int check_table(const char *what, int requests, int max_pages, int page_size, int tokens) {
    if (requests < 1 || requests > 1 << 24)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: requests=%d, must be 1..2^24", what,
                         requests);
    if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: page_size=%d, must be 16, 32, 64 or 128",
                         what, page_size);
    if (max_pages < 1 || (int64_t)max_pages * page_size > 1 << 30)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: max_pages=%d, must be >= 1 and hold at "
                         "most 2^30 tokens", what, max_pages);
    if (tokens < 0 || tokens > 1 << 30)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: tokens=%d, must be 0..2^30", what, tokens);
    return MIGEMM_OK;
}

}  // namespace
}  // namespace migemm

using namespace migemm;

extern "C" {

int migemm_quantize_rows(void *stream, const void *X, int type, int64_t ldx, int8_t *values,
                         int64_t ldv, float *scales, int rows, int cols) {
    const char *w = "quantize_rows";
    clear_error();
    MIGEMM_TRY(check_pointers(w, {X, values, scales}));
    MIGEMM_TRY(check_type(w, type));
    if (rows < 1 || cols < 1 || cols > INT32_MAX - 65536)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: sizes must be >= 1 (rows=%d cols=%d)", w,
                         rows, cols);
    const int64_t padded = ((int64_t)cols + 15) / 16 * 16;
    MIGEMM_TRY(check_ld(w, "ldx", ldx, cols));
    MIGEMM_TRY(check_ld(w, "ldv", ldv, padded));
    if (ldv % 16 != 0 || !aligned(values, 16))
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: values must be 16-byte aligned and ldv=%lld "
                         "a multiple of 16", w, (long long)ldv);
    MIGEMM_TRY(check_grid(w, rows, 256));
    MIGEMM_TRY(check_alias(w, {{values, rows_bytes(rows, ldv, padded, 1)},
                               {scales, (int64_t)rows * 4}},
                           {{X, rows_bytes(rows, ldx, cols, type_size(type))}}));
    return launch_quantize_rows((hipStream_t)stream, X, type, ldx, values, ldv, scales, rows,
                                cols);
}

int migemm_matmul_int8(void *stream, const int8_t *A, int64_t lda, const float *a_scales,
                       const int8_t *B, int64_t ldb, const float *b_scales, const float *bias,
                       void *C, int type, int64_t ldc, int M, int N, int K) {
    const char *w = "matmul_int8";
    clear_error();
    MIGEMM_TRY(check_pointers(w, {A, a_scales, B, b_scales, C}));
    MIGEMM_TRY(check_type(w, type));
    MIGEMM_TRY(check_product(w, M, N, K));
    if (K % 16 != 0)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: K=%d must be a multiple of 16 (rows padded "
                         "with zeros, as quantize_rows leaves them)", w, K);
    MIGEMM_TRY(check_int8_rows(w, "a", A, lda, K));
    MIGEMM_TRY(check_int8_rows(w, "b", B, ldb, K));
    MIGEMM_TRY(check_ld(w, "ldc", ldc, N));
    MIGEMM_TRY(check_alias(w, {{C, rows_bytes(M, ldc, N, type_size(type))}},
                           {{A, rows_bytes(M, lda, K, 1)}, {B, rows_bytes(N, ldb, K, 1)},
                            {a_scales, (int64_t)M * 4}, {b_scales, (int64_t)N * 4},
                            {bias, bias != nullptr ? (int64_t)N * 4 : 0}}));
    Int8Product p{};
    p.A = A;
    p.B = B;
    p.sa = a_scales;
    p.sb = b_scales;
    p.bias = bias;
    p.C = C;
    p.lda = lda;
    p.ldb = ldb;
    p.ldc = ldc;
    p.M = M;
    p.N = N;
    p.K = K;
    p.type = type;
    return launch_product_int8((hipStream_t)stream, p);
}

int migemm_linear_int8(void *stream, const void *X, int type, int64_t ldx, const int8_t *W,
                       int64_t ldw, const float *w_scales, const float *bias, void *Y,
                       int64_t ldy, int M, int N, int cols) {
    const char *w = "linear_int8";
    clear_error();
    MIGEMM_TRY(check_pointers(w, {X, W, w_scales, Y}));
    MIGEMM_TRY(check_type(w, type));
    MIGEMM_TRY(check_product(w, M, N, cols));
    const int K = (cols + 15) / 16 * 16;
    if (K > 131071)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: K=%d, int32 sums hold K <= 131071", w, K);
    MIGEMM_TRY(check_ld(w, "ldx", ldx, cols));
    MIGEMM_TRY(check_int8_rows(w, "w", W, ldw, K));
    MIGEMM_TRY(check_ld(w, "ldy", ldy, N));
    MIGEMM_TRY(check_grid(w, M, 256));
    MIGEMM_TRY(check_alias(w, {{Y, rows_bytes(M, ldy, N, type_size(type))}},
                           {{X, rows_bytes(M, ldx, cols, type_size(type))},
                            {W, rows_bytes(N, ldw, K, 1)}, {w_scales, (int64_t)N * 4},
                            {bias, bias != nullptr ? (int64_t)N * 4 : 0}}));
    Int8Product p{};
    p.B = W;
    p.sb = w_scales;
    p.bias = bias;
    p.C = Y;
    p.ldb = ldw;
    p.ldc = ldy;
    p.M = M;
    p.N = N;
    p.K = K;
    p.type = type;
    return launch_linear_int8((hipStream_t)stream, X, ldx, cols, p);
}

int migemm_cache_tables(void *stream, const int *lengths, const int *counts, int requests,
                        int *table, int max_pages, int page_size, const int *free_pages,
                        const int *free_count, int free_capacity, int *slots,
                        int *positions, int *starts, int *new_lengths, int *new_free,
                        int tokens) {
    const char *w = "cache_tables";
    clear_error();
    MIGEMM_TRY(check_pointers(w, {lengths, counts, table, free_pages, free_count, starts,
                                  new_lengths, new_free}));
    MIGEMM_TRY(check_table(w, requests, max_pages, page_size, tokens));
    if (tokens > 0) MIGEMM_TRY(check_pointers(w, {slots, positions}));
    if (free_capacity < 1)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: free_capacity=%d must be >= 1", w,
                         free_capacity);
    const int64_t r4 = (int64_t)requests * 4, t4 = (int64_t)tokens * 4;
    MIGEMM_TRY(check_alias(w, {{table, r4 * max_pages}, {slots, t4}, {positions, t4},
                               {starts, r4 + 4}, {new_lengths, r4}, {new_free, 4}},
                           {{lengths, r4}, {counts, r4},
                            {free_pages, (int64_t)free_capacity * 4},
                            {free_count, 4}}));
    TablesArgs a{};
    a.lengths = lengths;
    a.counts = counts;
    a.requests = requests;
    a.table = table;
    a.max_pages = max_pages;
    a.page_size = page_size;
    a.free_pages = free_pages;
    a.free_count = free_count;
    a.free_capacity = free_capacity;
    a.slots = slots;
    a.positions = positions;
    a.starts = starts;
    a.new_lengths = new_lengths;
    a.new_free = new_free;
    a.tokens = tokens;
    return launch_cache_tables((hipStream_t)stream, a);
}

int migemm_cache_slots(void *stream, const int *lengths, const int *counts, int requests,
                       const int *table, int max_pages, int page_size, int *slots,
                       int *positions, int *starts, int tokens) {
    const char *w = "cache_slots";
    clear_error();
    MIGEMM_TRY(check_pointers(w, {lengths, counts, table, starts}));
    MIGEMM_TRY(check_table(w, requests, max_pages, page_size, tokens));
    if (tokens > 0) MIGEMM_TRY(check_pointers(w, {slots, positions}));
    const int64_t r4 = (int64_t)requests * 4, t4 = (int64_t)tokens * 4;
    MIGEMM_TRY(check_alias(w, {{slots, t4}, {positions, t4}, {starts, r4 + 4}},
                           {{lengths, r4}, {counts, r4}, {table, r4 * max_pages}}));
    TablesArgs a{};
    a.lengths = lengths;
    a.counts = counts;
    a.requests = requests;
    a.table = const_cast<int *>(table);  // (only read: no free pages)
    a.max_pages = max_pages;
    a.page_size = page_size;
    a.slots = slots;
    a.positions = positions;
    a.starts = starts;
    a.tokens = tokens;
    return launch_cache_tables((hipStream_t)stream, a);
}

int migemm_cache_release(void *stream, const int *finished, int *lengths, int requests,
                         int *table, int max_pages, int page_size, int *free_pages, int pages,
                         int *free_count) {
    const char *w = "cache_release";
    clear_error();
    MIGEMM_TRY(check_pointers(w, {finished, lengths, table, free_pages, free_count}));
    MIGEMM_TRY(check_table(w, requests, max_pages, page_size, 0));
    if (pages < 1)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: pages=%d must be >= 1", w, pages);
    const int64_t r4 = (int64_t)requests * 4;
    MIGEMM_TRY(check_alias(w, {{lengths, r4}, {table, r4 * max_pages},
                               {free_pages, (int64_t)pages * 4}, {free_count, 4}},
                           {{finished, r4}}));
    return launch_cache_release((hipStream_t)stream, finished, lengths, requests, table,
                                max_pages, page_size, free_pages, pages, free_count);
}

int migemm_cache_append(void *stream, const void *K, const void *V, int type, int64_t ldk,
                        int64_t ldv, const int *slots, int tokens, int8_t *keys,
                        int8_t *values, float *key_scales, float *value_scales, int pages,
                        int kv_heads, int head_dim, int page_size) {
    const char *w = "cache_append";
    clear_error();
    const Cache8 c = make_cache(keys, values, key_scales, value_scales, pages, kv_heads,
                                head_dim, page_size);
    MIGEMM_TRY(check_cache(w, c));
    MIGEMM_TRY(check_type(w, type));
    if (tokens < 0 || tokens > 1 << 30)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: tokens=%d, must be 0..2^30", w, tokens);
    if (tokens == 0) return MIGEMM_OK;
    MIGEMM_TRY(check_pointers(w, {K, V, slots}));
    const int64_t row = (int64_t)kv_heads * head_dim;
    MIGEMM_TRY(check_ld(w, "ldk", ldk, row));
    MIGEMM_TRY(check_ld(w, "ldv", ldv, row));
    MIGEMM_TRY(check_grid(w, tokens, 256));
    MIGEMM_TRY(check_alias(w, {{keys, cache_bytes(c)}, {values, cache_bytes(c)},
                               {key_scales, scale_bytes(c)}, {value_scales, scale_bytes(c)}},
                           {{K, rows_bytes(tokens, ldk, row, type_size(type))},
                            {V, rows_bytes(tokens, ldv, row, type_size(type))},
                            {slots, (int64_t)tokens * 4}}));
    return launch_cache_append((hipStream_t)stream, K, V, type, ldk, ldv, slots, tokens, c);
}

int migemm_cache_read(void *stream, const int8_t *keys, const int8_t *values,
                      const float *key_scales, const float *value_scales, int pages,
                      int kv_heads, int head_dim, int page_size, const int *slots, int tokens,
                      void *K, void *V, int type) {
    const char *w = "cache_read";
    clear_error();
    const Cache8 c = make_cache(keys, values, key_scales, value_scales, pages, kv_heads,
                                head_dim, page_size);
    MIGEMM_TRY(check_cache(w, c));
    MIGEMM_TRY(check_type(w, type));
    if (tokens < 0 || tokens > 1 << 30)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: tokens=%d, must be 0..2^30", w, tokens);
    if (tokens == 0) return MIGEMM_OK;
    MIGEMM_TRY(check_pointers(w, {K, V, slots}));
    const int64_t out = (int64_t)tokens * kv_heads * head_dim * type_size(type);
    MIGEMM_TRY(check_grid(w, (tokens + 63) / 64, 256));
    MIGEMM_TRY(check_alias(w, {{K, out}, {V, out}},
                           {{keys, cache_bytes(c)}, {values, cache_bytes(c)},
                            {key_scales, scale_bytes(c)}, {value_scales, scale_bytes(c)},
                            {slots, (int64_t)tokens * 4}}));
    return launch_cache_read((hipStream_t)stream, c, slots, tokens, K, V, type);
}

int migemm_cache_attention(void *stream, const void *Q, int type, int64_t ldq,
                           const int8_t *keys, const int8_t *values, const float *key_scales,
                           const float *value_scales, int pages, int kv_heads, int head_dim,
                           int page_size, const int *table, int max_pages, const int *starts,
                           const int *positions, int requests, int tokens, int heads,
                           float scale, int max_count, int max_length, void *O) {
    const char *w = "cache_attention";
    clear_error();
    CacheAttention a{};
    a.c = make_cache(keys, values, key_scales, value_scales, pages, kv_heads, head_dim,
                     page_size);
    MIGEMM_TRY(check_cache(w, a.c));
    MIGEMM_TRY(check_type(w, type));
    MIGEMM_TRY(check_pointers(w, {table, starts}));
    MIGEMM_TRY(check_table(w, requests, max_pages, page_size, tokens));
    if (heads < 1 || heads % kv_heads != 0)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: heads=%d must be a multiple of "
                         "kv_heads=%d", w, heads, kv_heads);
    if (!(scale >= 0.f && scale <= 3.4e38f))
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: scale=%g must be finite and not negative",
                         w, (double)scale);
    if (max_count < 0 || max_length < 0)
        return set_error(MIGEMM_ERR_INVALID_ARG, "%s: max_count=%d and max_length=%d must not be "
                         "negative", w, max_count, max_length);
    if (tokens == 0) return MIGEMM_OK;
    MIGEMM_TRY(check_pointers(w, {Q, positions, O}));
    const int64_t row = (int64_t)heads * head_dim;
    MIGEMM_TRY(check_ld(w, "ldq", ldq, row));
    if ((int64_t)tokens * heads > INT32_MAX)
        return set_error(MIGEMM_ERR_UNSUPPORTED, "%s: %d tokens of %d heads exceed int32", w,
                         tokens, heads);
    const int64_t r4 = (int64_t)requests * 4;
    MIGEMM_TRY(check_alias(w, {{O, (int64_t)tokens * row * type_size(type)}},
                           {{Q, rows_bytes(tokens, ldq, row, type_size(type))},
                            {keys, cache_bytes(a.c)}, {values, cache_bytes(a.c)},
                            {key_scales, scale_bytes(a.c)}, {value_scales, scale_bytes(a.c)},
                            {table, r4 * max_pages}, {starts, r4 + 4},
                            {positions, (int64_t)tokens * 4}}));
    a.Q = Q;
    a.O = O;
    a.type = type;
    a.ldq = ldq;
    a.table = table;
    a.starts = starts;
    a.positions = positions;
    a.max_pages = max_pages;
    a.requests = requests;
    a.tokens = tokens;
    a.heads = heads;
    a.scale = scale;
    a.max_count = max_count;
    a.max_length = max_length;
    return launch_cache_attention((hipStream_t)stream, a);
}

}  // extern "C"

namespace migemm {

int launch_cache_attention(hipStream_t stream, const CacheAttention &a) {
    AttnArgs p{};
    p.a = a;
    p.shift = __builtin_ctz((unsigned)a.c.page_size);
    p.group = a.heads / a.c.heads;
    p.cap = a.max_pages * a.c.page_size;
    p.c = a.scale * 1.44269504088896340736f;
    const int64_t count = a.max_count > 0 && a.max_count < a.tokens ? a.max_count : a.tokens;
    const int64_t length =
        a.max_length > 0 && a.max_length < p.cap ? a.max_length : p.cap;
    const int64_t count_rows = count * p.group;
    // Single tokens in even shares, two work-groups a CU (one where a head's registers allow no
    // more): int32 holds the number of tiles, and their scan is kept on the chip. Short contexts
    // in ranges, without the scan (8 requests of 200 tokens: 6.5 us, 9.4 in shares; 32 of 500: 15.5,
    // 17.5; 32 of 1000: 23.0, 22.3).
    const int64_t tiles = ((int64_t)a.tokens * p.group / 16 + a.requests + kNoRequest) *
                          ((p.cap + 63) / 64);
    const bool even = length > 512 && a.requests <= kShareRequests &&
                      tiles * a.c.heads < (int64_t)1 << 30;
    // Requests of at most 16 rows are computed one way, others another; where one request may
    // bring more, one launch holds both ways. Up to 32 float32 rows go the first way twice, in
    // shares (32 requests of 4096 tokens, 20 rows each, 8 kv heads of 128: 95 us, 183 the other
    // way, whose work-groups hold 128; 48 rows: 154 and 198, 64: 198 and 213; bfloat16 20 rows 92
    // and 71).
    const bool many = count_rows > (even && a.type == MIGEMM_FLOAT32 ? 2 * kFewRows : kFewRows);
    p.both = many;
    if (!many && even) {
        p.shares = a.c.width <= 128 ? 512 : 256;
        p.tiles = (int)tiles;
        MIGEMM_TRY(check_grid("cache_attention", (int64_t)a.requests * a.heads, 256));
        const size_t parts = (size_t)p.shares * 2 * 16;
        const size_t scan = ((size_t)a.requests + kNoRequest + 1) * 2 * sizeof(int);
        int rc = MIGEMM_OK;
        p.part_o = static_cast<float *>(workspace(
            stream, parts * (a.c.width + 2) * sizeof(float) + scan, &rc, 0));
        if (p.part_o == nullptr) return rc;
        p.part_ml = p.part_o + parts * a.c.width;
        p.firsts = reinterpret_cast<int *>(p.part_ml + parts * 2);
        return a.type == MIGEMM_FLOAT32 ? launch_attention_f32(stream, p)
                                        : launch_attention_bf16(stream, p);
    }
    const int64_t units = (int64_t)a.tokens * p.group / kManyRows + a.requests + kNoRequest;
    p.units = (int)units;
    // Contexts are cut in ranges (of whole rounds of a few-rows work-group, 256 tokens) where the
    // requests, tiles and kv heads alone make too few work-groups: single tokens until there are
    // about 1024 (they wait for memory), more rows until there is one for each CU, or two where
    // the registers hold two (bfloat16, heads up to 128) and the rows are fewer than the keys
    // (their partial results, four bytes a feature and row and range, cost more otherwise). 32
    // requests of 4096 tokens, 20 rows each, 8 kv heads of 128: 115 us with one, 70 with two; 8
    // of 8192, 512 rows: 221 and 198; float32 with two: 375 and 411.
    const int64_t base =
        std::max<int64_t>(a.requests, many ? (int64_t)a.tokens * p.group / kManyRows : 0) *
        a.c.heads;
    const bool two = a.type == MIGEMM_BFLOAT16 && a.c.width <= 128 &&
                     (int64_t)a.tokens * p.group <= a.requests * length;
    const int64_t fill = two ? 512 : 256;
    const int64_t want = many ? (base < fill ? fill / base : 1) : (1024 + base - 1) / base;
    int64_t chunk = (length + want - 1) / want;
    chunk = (chunk + 255) / 256 * 256;
    p.chunk = (int)chunk;
    p.splits = (int)((length + chunk - 1) / chunk);
    const int64_t rows = (int64_t)a.tokens * a.heads;
    MIGEMM_TRY(check_grid("cache_attention", (int64_t)p.splits * a.c.heads *
                                                  (a.requests + kNoRequest + (many ? units : 0)), 512));
    if (p.splits > 1) {
        MIGEMM_TRY(check_grid("cache_attention", rows, 256));
        const size_t parts = (size_t)rows * p.splits;
        int rc = MIGEMM_OK;
        p.part_o = static_cast<float *>(
            workspace(stream, parts * (a.c.width + 2) * sizeof(float), &rc, 0));
        if (p.part_o == nullptr) return rc;
        p.part_ml = p.part_o + parts * a.c.width;
    }
    return a.type == MIGEMM_FLOAT32 ? launch_attention_f32(stream, p)
                                    : launch_attention_bf16(stream, p);
}

}  // namespace migemm
