// Causal attention over the 8-bit paged cache: the kernels, instantiated by
// cache_attention_f32.hip and cache_attention_bf16.hip.
//
// For a row (a query token and head) with n keys: S = c (q . k8) ks, p = 2^(S - max S),
// O = sum p vs v8 / sum p, with c = scale log2 e, k8 and v8 the bytes, ks and vs the scales
// of their page and head; one pass over the keys with the running maximum and sum, in fp32.
//
// The bytes are exact in bf16 (7 bits), so products run on the bf16 matrix cores with the
// cache's side exact. A bf16 query is exact too. A float32 query, and p vs, are cut into bf16
// parts whose products add up in the fp32 accumulator: three parts (24 bits) for float32
// calls, so that they are as exact as float32 arithmetic. For bf16 calls p vs is one f16 number
// (11 bits, an eighth of the result's own rounding; the bytes of V are exact in f16 too). f16's
// range is small, so weights have a running maximum of their own, over score + log2 vs, in whose
// unit they and the sums of weights times V are held (Weights, below): a row's weights come to
// at most 2^14, whatever its pages' scales, and what f16 rounds as subnormal is below 2^-20 of the
// row's largest. The denominator is summed over the rounded weights where a tile's scales are not far
// below the row's, else over the exponentials. (With one bf16 number, 8 bits, results were 2.3e-3 off
// the formula in norm; the result's own rounding is 1.7e-3, and so are they now. Single tokens take
// the same time, prompts 2 % more: 4 x 4096 tokens 636 and 652 us.)
//
// The transposed products S^T = K Q^T and O^T = V^T P^T keep everything in registers: a lane
// holds keys of one row, the exponentials come out where the second product wants them, and
// since the sum over tokens may run in any order, the tokens are dealt to the rows of the
// first product such that a lane's bytes of V are neighbours in the (transposed) page.
//
// Keys at and after a row's limit, or in pages outside the pool, are masked by selection
// after the scale (so a page's NaN scale reaches only the rows that may see the page).
#pragma once

#include <type_traits>

#include "int8_common.h"

namespace migemm {

struct AttnArgs {
    CacheAttention a;
    int shift;          // log2 page_size
    int group;          // query heads a kv head
    int cap;            // tokens a table row holds
    float c;            // scale * log2 e
    int chunk, splits;  // keys of a range (the last takes the rest), ranges
    int both;           // few and many rows in one launch, each part takes its requests
    int units;          // many rows: tiles of rows that the grid covers
    int shares;         // work-groups of few_shares (0: ranges)
    int tiles;          // its bound of one kv head's tiles
    int *firsts;        // [2][requests + kNoRequest + 1]: its scan, for the join
    float *part_o;      // [tokens * heads][splits][width], or [2 shares][16][width]
    float *part_ml;     // likewise, 2 (the largest score, the sum)
};

constexpr int kFewRows = 16;
constexpr int kShareRequests = 1022;  // few_shares keeps a scan of the requests in LDS
constexpr int kSnap = 2;              // (its cuts)
constexpr int kManyRows = 128;        // of a many-rows work-group
constexpr float kLag = 8.f;  // (weights stay below 2^8)

namespace {

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Tokens [s0, s1) of request r. Two more "requests", without keys, have the tokens that belong to
// none: r == requests those past the last one's, r == requests + 1 those before the first one's.
constexpr int kNoRequest = 2;
__device__ __forceinline__ void request_tokens(const CacheAttention &a, int r, int &s0,
                                               int &s1) {
    const bool leading = r > a.requests;
    const int at = clamp_int(a.starts[leading ? 0 : r], 0, a.tokens);
    const int next = a.starts[min(r + 1, a.requests)];
    s0 = leading ? 0 : at;
    s1 = leading ? at : r < a.requests ? clamp_int(next, s0, a.tokens) : a.tokens;
}

// Keys that a row sees: its position's and those before it.
__device__ __forceinline__ int keys_of(int position, int cap) {
    return clamp_int(position, -1, cap - 1) + 1;
}

// N parts of x, largest first: x = sum of the parts up to 2^-8N.
template <int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&out)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        out[i] = pack_bf16(x, y);
        if (i + 1 < N) {
            x -= bf16_low(out[i]);
            y -= bf16_high(out[i]);
        }
    }
}

union Frag {
    uint32_t u[4];
    v8bf v;
    v8h h;
};

// bf16 calls: a row's weights, in units of 2^(top - kUnit). top follows score + log2 vs as m
// follows the scores, and whenever m does, so that over = top - m is log2 of a scale that the row
// saw. Rows that saw no key: over = -inf; nothing but zeros: inf.
constexpr float kUnit = 6.f;
constexpr float kFar = -5.f;  // scales below 2^kFar of the row's: the denominator from exponentials
struct Weights {
    float top = -INFINITY, over = -INFINITY;
    __device__ __forceinline__ float unit() const {
        return (top == -INFINITY ? 0.f : top) - kUnit;
    }
    // Returns what the sums are multiplied with.
    __device__ __forceinline__ float follow(float now, float m) {
        now = fmaxf(top, now);
        const float alpha = __builtin_amdgcn_exp2f(top - (now == -INFINITY ? 0.f : now));
        top = now;
        over = top == -INFINITY ? (m == -INFINITY ? -INFINITY : INFINITY) : top - m;
        return alpha;
    }
    // What brings a sum of weights over vs to units of 2^m.
    __device__ __forceinline__ float to_m() const { return __builtin_amdgcn_exp2f(over - kUnit); }
    // What brings the sums to units of 2^m, times 2^kUnit (2^over alone stays a normal number).
    __device__ __forceinline__ float natural() const {
        return over == INFINITY ? 0.f : __builtin_amdgcn_exp2f(over);
    }
};

// Eight neighbouring values of a query row as float32 (head sizes are multiples of 8: all of
// them are there or none, which reads `row` itself and gives zeros; no branch waits for a load).
template <typename T>
__device__ __forceinline__ void query_values(const T *row, int d, bool there, float (&x)[8]) {
    struct Raw {
        T t[8];
    };
    const Raw v = load_any<Raw>(row + (there ? d : 0));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = there ? to_f32(v.t[i]) : 0.f;
}

// The same in N parts.
template <typename T, int N>
__device__ __forceinline__ void query_frag(const T *row, int d, bool there, Frag (&f)[N]) {
    if constexpr (std::is_same<T, Bf16>::value && N == 1) {
        f[0] = load_any<Frag>(row + (there ? d : 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) f[0].u[i] = there ? f[0].u[i] : 0u;
    } else {
        float x[8];
        query_values(row, d, there, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t part[N];
            split_pair<N>(x[2 * i], x[2 * i + 1], part);
#pragma unroll
            for (int n = 0; n < N; ++n) f[n].u[i] = part[n];
        }
    }
}

// A float32 query that is not finite has parts that are NaN, and with them all scores of its row.
// A bf16 one is held as it is, and against keys of one sign an infinity would give scores that
// are all -inf, as of a row without keys: where one of a lane's values is not finite (times 0 it is
// NaN), its first ones become NaN.
template <int N>
__device__ __forceinline__ void spoil(Frag (&q)[N][1]) {
    float odd[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            odd[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, q[s][0].u[i]),
                                                         v2bf{(__bf16)0.f, (__bf16)0.f},
                                                         odd[i & 1], false);
    const float sum = odd[0] + odd[1];
    q[0][0].u[0] = sum != sum ? 0x7fc07fc0u : q[0][0].u[0];
}

// The largest of three, NaN if one is (fmaxf would make each operand canonical first, an
// instruction of its own).
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// Rows that are whole after range 0 are written by it; others leave a part for each range.
__device__ __forceinline__ bool row_is_whole(const AttnArgs &p, int limit) {
    return p.splits == 1 || limit <= p.chunk;
}

// ------------------------------------------------------------------------- few rows
// Up to 16 rows (queries x heads that share a kv head): decoding. Bound by reading the cache
// once, if little enough is done for each byte. A work-group takes one request, kv head and
// range of keys; its four wavefronts take tiles of 64 tokens in turn, straight from memory to registers
// (K of the next tile flies from the first product on, V from the second).
//
// v_mfma_f32_16x16x32_bf16: row m of subtile u is token 16 (m / 4) + 4 u + m % 4 of the tile, so
// that lane group g ends up with the scores of tokens 16 g .. 16 g + 15, whose bytes of V^T are
// 16 neighbours: one load a row of V. Of K a lane's 16 bytes are two steps' operands.
template <int W>
struct FewLds {
    alignas(16) float o[4 * 16 * (W + 4)];
    float m[4][16], l[4][16];
};

// 16 rows from row0 on of request r (tokens from s0 on) and kv head h, over its keys lo .. end - 1
// (as far as a row sees them). part: kWhole (all its keys: the result), a place for a part, or
// -2 - range where rows go by row_is_whole.
constexpr int kWhole = -1;

template <typename T, int W>
__device__ __forceinline__ void few_segment(const AttnArgs &p, int r, int s0, int rows, int h,
                                            int row0, int lo, int end, int part,
                                            FewLds<W> &lds) {
    constexpr int STEP = 256;  // tokens that the work-group takes at a time
    constexpr int PP = std::is_same<T, float>::value ? 3 : 1;  // parts of q and of the weights
    constexpr int SK = (W + 63) / 64;  // pairs of steps of 32 features of the first product
    constexpr bool HALF = W % 64 != 0; // of the last one only 32 are there: lane groups 2 and 3
                                       // take 0 and 1's bytes of K, and zeros of q
    constexpr int DT = W / 16;         // blocks of the second product
    constexpr int OS = W + 4;          // LDS row
    float *const o_lds = lds.o;
    auto &m_lds = lds.m;
    auto &l_lds = lds.l;

    const CacheAttention &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int P = a.c.page_size;
    const int *table = a.table + (int64_t)(r < a.requests ? r : 0) * a.max_pages;
    const int64_t page_bytes = (int64_t)P * W;
    const int split = part < kWhole ? -2 - part : 0;

    const int j = row0 + col;
    const int tok = j < rows ? s0 + j / p.group : min(s0, a.tokens - 1);
    const int head = h * p.group + j % p.group;

    v4i kb[4][SK];
    v4i vb[DT];
    float ks = 0.f, vs = 0.f;
    int page = -1;
    // The table's entry for lane group g's 16 tokens: as it stands, and looked at only where
    // the tile is loaded. (A check here would wait for the entry, and as loads come back in
    // order, for every load before it.)
    auto find = [&](int t0) { return table[min(t0 + 16 * g, p.cap - 1) >> p.shift]; };
    // (not live: behind the last tile, where every lane reads the same few bytes)
    auto load_k = [&](int t0, int entry, bool live) {
        const int pg = entry >= 0 && entry < a.c.pages ? entry : -1;
        page = pg;
        const int64_t mine = (int64_t)max(pg, 0) * a.c.heads + h;
        ks = a.c.key_scales[mine];
        vs = a.c.value_scales[mine];
        const int kpage = max(__shfl(pg, (col >> 2) * 16), 0);
        const int64_t at = ((int64_t)kpage * a.c.heads + h) * page_bytes +
                           ((t0 + 16 * (col >> 2) + (col & 3)) & (P - 1)) * W;
        const int8_t *kp = a.c.keys + (live ? at : 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int i = 0; i < SK; ++i) {
                const int group = HALF && i == SK - 1 ? g & 1 : g;
                kb[u][i] = __builtin_nontemporal_load(
                    reinterpret_cast<const v4i *>(kp + u * 4 * W + 64 * i + 16 * group));
            }
        }
    };
    auto load_v = [&](int t0, bool live) {  // (of the pages of the last load_k)
        const int64_t at = ((int64_t)max(page, 0) * a.c.heads + h) * page_bytes + col * P +
                           ((t0 + 16 * g) & (P - 1));
        const int8_t *vp = a.c.values + (live ? at : 0);
#pragma unroll
        for (int d = 0; d < DT; ++d)
            vb[d] = __builtin_nontemporal_load(reinterpret_cast<const v4i *>(vp + d * 16 * P));
    };
    // What the first tile needs is asked for at once, before it is known whether a row sees it
    // (a segment begins with loads that wait for each other).
    int t0 = lo + 64 * wave;
    const int entry = find(t0);
    int next = find(t0 + STEP);
    const int position = a.positions[tok];
    load_k(t0, entry, t0 < end);
    load_v(t0, t0 < end);

    // q: lane (col, g) holds features 64 i + 16 g .. + 15, eight a step
    Frag q[2 * SK][PP];
    {
        const T *qp = static_cast<const T *>(a.Q) +
                      (j < rows ? (int64_t)tok * a.ldq + (int64_t)head * a.c.dim : 0);
#pragma unroll
        for (int i = 0; i < 2 * SK; ++i) {
            const int d = 64 * (i / 2) + 16 * g + 8 * (i % 2);
            query_frag<T, PP>(qp, d, j < rows && d < a.c.dim, q[i]);
        }
        if constexpr (PP == 1) spoil(q);
    }

    const int limit = j < rows && r < a.requests ? keys_of(position, p.cap) : 0;
    int most = limit;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o));
    most = __builtin_amdgcn_readfirstlane(most);
    const int hi = min(most, end);
    if (split > 0 && lo >= most) return;  // (the same for the whole work-group)

    float m = -INFINITY, l = 0.f;
    Weights weights;
    v4f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};

    for (; t0 < hi; t0 += STEP) {
        v4f s[4];
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u) s[u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2 * SK; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (i % 2 == 0) pin(kb[u][i / 2]);
                const v8bf k =
                    bytes8_to_bf16(kb[u][i / 2][i % 2 * 2], kb[u][i / 2][i % 2 * 2 + 1]);
#pragma unroll
                for (int n = PP - 1; n >= 0; --n)
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[i][n].v, s[u], 0, 0, 0);
            }
        float sc = ks * p.c;
        const float vscale = vs;
        const int seen = page < 0 ? 0 : limit - t0 - 16 * g;  // of this lane's 16 tokens
        // The next tile's loads, behind the last one too: loads in a branch would make every
        // wait below one for all loads.
        const bool more = t0 + STEP < hi;
        load_k(t0 + STEP, next, more);
        next = find(t0 + 2 * STEP);
        // Scores are s * sc: scaled at once only where some are masked.
        if (__ballot(seen < 16) == 0) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, s[u][i]);
            top *= sc;
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[u][i] = 4 * u + i < seen ? s[u][i] * sc : -INFINITY;
                    top = fmaxf(top, s[u][i]);
                }
            sc = 1.f;
        }
        // m is any number near the largest score: it follows only where it would be left
        // behind by more than kLag, so the sums are rarely scaled anew
        const float lg = __builtin_amdgcn_logf(vscale);  // (log2)
        float big = PP == 1 ? top + lg : 0.f;
        if (__ballot(top > m + kLag || (PP == 1 && big > weights.top + kLag)) != 0) {
#pragma unroll
            for (int x = 16; x < 64; x <<= 1) {
                top = fmaxf(top, __shfl_xor(top, x));
                if constexpr (PP == 1) big = fmaxf(big, __shfl_xor(big, x));
            }
            const float now = fmaxf(m, top);
            const float alpha = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.f : now));
            l *= alpha;
            m = now;
            const float by = PP == 1 ? weights.follow(big, m) : alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][i] *= by;
        }
        Frag w[2][PP];
        const float less = lg - weights.unit();
        if (PP == 1 && __ballot(!(vscale >= 0x1p-90f) || lg - weights.over < kFar) == 0) {
            // the sum is taken over the rounded weights, so that numerator and denominator round
            // alike (a row that sees one key gives its value, whatever the scale's bits)
            float sum = 0.f;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t e =
                        pack_f16(__builtin_amdgcn_exp2f(fmaf(s[u][2 * i], sc, less)),
                                 __builtin_amdgcn_exp2f(fmaf(s[u][2 * i + 1], sc, less)));
                    w[u / 2][0].u[2 * (u & 1) + i] = e;
                    sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, e),
                                                 v2h{(_Float16)1.f, (_Float16)1.f}, sum, false);
                }
            l = fmaf(sum, __builtin_amdgcn_rcpf(vscale) * weights.to_m(), l);
        } else {  // (a scale of 0, a tiny one, NaN, one far below the row's, or float32)
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float z = fmaf(s[u][2 * i + k], sc, -base);
                        e[k] = __builtin_amdgcn_exp2f(z);
                        l += e[k];
                        if constexpr (PP == 1)
                            e[k] = __builtin_amdgcn_exp2f(z + (less + base));
                        else
                            e[k] *= vscale;
                        e[k] = z != -INFINITY ? e[k] : 0.f;
                    }
                    if constexpr (PP == 1) {
                        w[u / 2][0].u[2 * (u & 1) + i] = pack_f16(e[0], e[1]);
                    } else {
                        uint32_t part[PP];
                        split_pair<PP>(e[0], e[1], part);
#pragma unroll
                        for (int n = 0; n < PP; ++n)
                            w[u / 2][n].u[2 * (u & 1) + i] = part[n];
                    }
                }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            pin(vb[d]);
            if constexpr (PP == 1) {
                const v8h x = bytes8_to_f16(vb[d][0], vb[d][1]);
                const v8h y = bytes8_to_f16(vb[d][2], vb[d][3]);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w[0][0].h, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, w[1][0].h, o[d], 0, 0, 0);
            } else {
                const v8bf x = bytes8_to_bf16(vb[d][0], vb[d][1]);
                const v8bf y = bytes8_to_bf16(vb[d][2], vb[d][3]);
#pragma unroll
                for (int n = PP - 1; n >= 0; --n) {
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w[0][n].v, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, w[1][n].v, o[d], 0, 0, 0);
                }
            }
        }
        load_v(t0 + STEP, more);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the wavefronts' results under their common maximum, added in order
    if (g == 0) {
        m_lds[wave][col] = m;
        l_lds[wave][col] = l;
    }
    __syncthreads();
    float top = m_lds[0][col];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, m_lds[w][col]);
    const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - top);
    const float natural = PP == 1 ? weights.natural() : 1.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        v4f x = o[d];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = (PP == 1 ? x[i] * 0x1p-6f * natural : x[i]) * f;  // (2^-kUnit)
        *reinterpret_cast<v4f *>(o_lds + (wave * 16 + col) * OS + d * 16 + 4 * g) = x;
    }
    __syncthreads();
    if (lane < 16 && wave == 0) {  // (m_lds, l_lds: now the joined ones)
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = m_lds[w][col], lw = l_lds[w][col];
            sum += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f(mw - top);
        }
        m_lds[0][col] = top;
        l_lds[0][col] = sum;
    }
    __syncthreads();
    for (int e = tid; e < 16 * (W / 4); e += STEP) {
        const int c = e / (W / 4), d = (e - c * (W / 4)) * 4;
        const int jj = row0 + c;
        if (jj >= rows) continue;
        v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const v4f y = *reinterpret_cast<const v4f *>(o_lds + (w * 16 + c) * OS + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += y[i];
        }
        const int tk = s0 + jj / p.group;
        const int64_t row = (int64_t)tk * a.heads + h * p.group + jj % p.group;
        bool whole = part == kWhole;
        int64_t at = (int64_t)part * 16 + c;
        if (part < kWhole) {
            const int lim = r < a.requests ? keys_of(a.positions[tk], p.cap) : 0;
            whole = row_is_whole(p, lim);
            if (whole && split > 0) continue;
            at = row * p.splits + split;
        }
        const float sum = l_lds[0][c];
        if (whole) {
            if (d < a.c.dim) {
                struct {
                    T t[4];
                } y;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int i = 0; i < 4; ++i) y.t[i] = from_f32<T>(x[i] * inv);
                store_any(static_cast<T *>(a.O) + row * a.c.dim + d, y);
            }
        } else {
            *reinterpret_cast<v4f *>(p.part_o + at * W + d) = x;
            if (d == 0) {
                p.part_ml[at * 2] = m_lds[0][c];
                p.part_ml[at * 2 + 1] = sum;
            }
        }
    }
    __syncthreads();
}

// One request, kv head and range of its keys, all its rows.
template <typename T, int W>
__device__ __forceinline__ void few_rows(const AttnArgs &p, int id, FewLds<W> &lds) {
    const CacheAttention &a = p.a;
    const int split = id % p.splits;
    id /= p.splits;
    const int h = id % a.c.heads;
    const int r = id / a.c.heads;
    int s0, s1;
    request_tokens(a, r, s0, s1);
    const int rows = (s1 - s0) * p.group;
    if (p.both && rows > kFewRows) return;
    const int lo = split * p.chunk;
    for (int row0 = 0; row0 < rows; row0 += 16)
        few_segment<T, W>(p, r, s0, rows, h, row0, lo,
                          split == p.splits - 1 ? p.cap : lo + p.chunk, -2 - split, lds);
}

// Single tokens in even shares: the tiles (of 64 tokens) of all requests and kv heads in one
// line, cut into p.shares equal pieces, one a work-group, all of which run at once; a decoding
// batch's contexts differ, and work-groups of whole ranges would leave CUs idle at the end.
// 32 requests of up to 4096 tokens, 8 kv heads of 128: 38.4 us (172 MB, 4.5 TB/s; 41.8 in ranges), 2
// of up to 131072: 74 us (415 MB, 5.6 TB/s). float32 queries 41.6 and 77.6. Where all contexts
// have one length ranges are as good (32 x 4096: bfloat16 50.9 us in shares and 49.1 in ranges with
// the join, float32 54.3 and 49.1).
// A unit is one request, kv head and 16 rows (its rows beyond 16 are further units, and a unit
// without keys has one tile, which writes its zeros). Cuts within two tiles of a unit's end
// are moved there. A unit that is cut is joined afterwards (attention_share_join_kernel, which
// finds the same cuts): a share has at most one unit that began before it (part 2 w) and one
// that goes on after it (part 2 w + 1).
struct Shares {
    int total, each;  // tiles of all units, of a share
};
__device__ __forceinline__ Shares shares_of(const AttnArgs &p, int tiles) {
    const int total = tiles * p.a.c.heads;
    return {total, max(4, (total + p.shares - 1) / p.shares)};
}

struct ShareLds {
    int first[kShareRequests + kNoRequest + 1];  // tiles of one head of the requests before r
    int units[kShareRequests + kNoRequest];      // tiles of a unit of r
    int token[kShareRequests + kNoRequest];      // r's first token
    int rows[kShareRequests + kNoRequest];
};

template <typename T, int W>
__device__ __forceinline__ void few_shares(const AttnArgs &p, FewLds<W> &lds,
                                           ShareLds &scan) {
    const CacheAttention &a = p.a;
    auto &first = scan.first;
    auto &units = scan.units;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto &sums = lds.m[0];
    const int all_requests = a.requests + kNoRequest;
    // (Sums end at p.tiles, which starts that do not descend never reach: no index below leaves its
    // array, and no int32 overflows, whatever the device's memory holds.)
    int before = 0;
    for (int base = 0; base < all_requests; base += 256) {
        const int r = base + tid;
        int n = 0, unit = 1;
        if (r < all_requests) {
            int s0, s1, most = 0;
            request_tokens(a, r, s0, s1);
            if (r < a.requests)
                for (int t = s0; t < s1; ++t) most = max(most, keys_of(a.positions[t], p.cap));
            unit = max(1, (most + 63) / 64);
            n = ((s1 - s0) * p.group + 15) / 16 * unit;
            units[r] = unit;
            scan.token[r] = s0;
            scan.rows[r] = (s1 - s0) * p.group;
        }
        int upto = min(n, p.tiles);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(upto, o);
            if (lane >= o) upto = min(upto + u, p.tiles);
        }
        if (lane == 63) sums[wave] = __int_as_float(upto);
        __syncthreads();
        int all = before;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w == wave) upto = min(upto + all, p.tiles);
            all = min(all + __float_as_int(sums[w]), p.tiles);
        }
        if (r < all_requests) first[r + 1] = upto;
        before = all;
        __syncthreads();
    }
    if (tid == 0) first[0] = 0;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = tid; i <= all_requests; i += 256) {
            p.firsts[i] = first[i];
            p.firsts[all_requests + 1 + i] = i < all_requests ? units[i] : 1;
        }
    const Shares s = shares_of(p, before);
    auto request_at = [&](int tile) {  // the last request that begins at or before the tile
        int r = -1;
        for (int base = 0; base < all_requests; base += 64)
            r += __builtin_popcountll(__ballot(
                base + lane < all_requests && first[min(base + lane, all_requests)] *
                                                      a.c.heads <= tile));
        return r;
    };
    auto cut = [&](int w) {
        const int64_t at = (int64_t)w * s.each;
        if (at >= s.total) return s.total;
        const int r = request_at((int)at);
        const int in = ((int)at - first[r] * a.c.heads) % units[r];
        if (in <= kSnap) return (int)at - in;
        return units[r] - in <= kSnap ? min((int)at + units[r] - in, s.total) : (int)at;
    };
    const int w = blockIdx.x;
    int at = __builtin_amdgcn_readfirstlane(cut(w));
    const int stop = __builtin_amdgcn_readfirstlane(cut(w + 1));
    while (at < stop) {
        const int r = request_at(at);
        const int unit = __builtin_amdgcn_readfirstlane(units[r]);
        const int n = __builtin_amdgcn_readfirstlane(first[r + 1] - first[r]);
        const int in = at - __builtin_amdgcn_readfirstlane(first[r]) * a.c.heads;
        const int h = in / n;
        const int block = (in - h * n) / unit;
        const int tile = in - h * n - block * unit;
        const int last = min(unit, tile + stop - at);
        const bool ends = last == unit;
        const int s0 = __builtin_amdgcn_readfirstlane(scan.token[r]);
        const int rows = __builtin_amdgcn_readfirstlane(scan.rows[r]);
        few_segment<T, W>(p, r, s0, rows, h, block * 16, tile * 64, last * 64,
                          tile == 0 && ends ? kWhole : 2 * w + (tile == 0 ? 1 : 0), lds);
        at += last - tile;
    }
}

// ------------------------------------------------------------------------ many rows
// Prompts: 32 rows (queries x heads that share a kv head) a wavefront, four wavefronts, on
// v_mfma_f32_32x32x16_bf16 (bf16 calls' second product: _f16). Tiles of 64 tokens are read as
// bytes, turned into 16 bits once for the work-group and shared in LDS (two buffers: the next
// tile's bytes fly during a tile's work, one barrier a tile). LDS rows are padded by 16 bytes: the
// 16 lanes of a read phase fall on different banks.
//
// 4 x 4096 tokens, 32 heads on 8 of 128: 637 to 660 us, 0.85 PFLOP/s; 16 x 1024: 228 us. Of a
// wavefront's 2900 cycles a tile the matrix cores have 1024, the vector instructions (softmax
// 110, maxima 35, conversions 96, exponentials at a quarter of the rate) about 1350, and the
// LDS reads, a kilobyte an instruction, as long as the matrix cores have: each has a half of
// the time, and the two work-groups of a CU overlap them in part. Tried and slower: eight
// wavefronts, two on a SIMD a phase apart (690); 64 rows a wavefront, which halves the LDS
// reads, with a SIMD to itself (1420: the registers do not hold it).
template <int W>
struct ManyLds {
    static constexpr int KR = W + 8, VR = 64 + 8;  // LDS rows, in 16-bit values
    alignas(16) uint16_t k[2][64 * KR];
    alignas(16) uint16_t v[2][W * VR];
    // of the tile's four groups of 16 tokens: ks c, vs, log2 vs and 1 / vs
    v4f scales[2][4];
    // (1: the page is outside the pool, 2: vs is a plain number)
    alignas(4) uint8_t flags[2][4];
    int most[4];
};

// A work-group's share: request r's rows from tile * kManyRows on, of kv head h, and a range of
// keys.
struct ManyTile {
    int r, tile, s0, rows, h, split;
};
__device__ __forceinline__ bool many_tile(const AttnArgs &p, int id, ManyTile &x) {
    const CacheAttention &a = p.a;
    const int lane = threadIdx.x & 63;
    x.h = id % a.c.heads;
    id /= a.c.heads;
    x.split = id % p.splits;
    id /= p.splits;
    // which request's tile: requests in order (tiles that run together share keys in L2), 64 at
    // a time
    int r = -1, tile = 0, s0 = 0, s1 = 0;
    for (int base = 0, before = 0; base < a.requests + kNoRequest; base += 64) {
        int x0 = 0, x1 = 0, n = 0;
        if (base + lane < a.requests + kNoRequest) {
            request_tokens(a, base + lane, x0, x1);
            const int rows = (x1 - x0) * p.group;
            n = rows > kFewRows ? (rows + kManyRows - 1) / kManyRows : 0;
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(upto, o);
            if (lane >= o) upto += u;
        }
        const uint64_t mine = __ballot(before + upto > id);
        if (mine != 0) {
            const int w = __builtin_ctzll(mine);
            r = base + w;
            s0 = __shfl(x0, w);
            s1 = __shfl(x1, w);
            tile = before + __shfl(upto, w) - 1 - id;  // the last tiles, the longest, first
            break;
        }
        before += __shfl(upto, 63);
    }
    x.r = __builtin_amdgcn_readfirstlane(r);
    x.s0 = __builtin_amdgcn_readfirstlane(s0);
    x.rows = (__builtin_amdgcn_readfirstlane(s1) - x.s0) * p.group;
    x.tile = __builtin_amdgcn_readfirstlane(tile);
    return r >= 0;
}

// How a work-group of four wavefronts brings tiles of 64 tokens into LDS. A wavefront moves 16
// tokens' rows of K, so that their page is one for the wavefront and its address scalar; of V it
// moves the same tokens of all features or, where a page holds whole tiles, a quarter of the
// features of all 64 (rows of 64 neighbouring bytes). A thread's place in the page never changes.
template <int W, bool F16>  // (V in f16, or bf16)
struct ManyStage {
    static constexpr int CH = W / 16;          // units of 16 bytes in a row of K
    static constexpr int MU = (W + 63) / 64;   // units of K, and of V, that a thread moves
    static constexpr bool EVEN = W % 64 == 0;  // (as many for every thread)
    static constexpr int KR = ManyLds<W>::KR, VR = ManyLds<W>::VR;
    const AttnArgs &p;
    ManyLds<W> &lds;
    const int *table;
    int lane, wave, h, P, vrow, vgroup;
    bool whole, gone = false;
    uint32_t zero;
    v4i kb[MU], vb[MU];
    int entry = -1;
    int64_t block = 0;  // of the tile whose K was loaded last
    float ks = 0.f, vs = 0.f;

    __device__ __forceinline__ ManyStage(const AttnArgs &args, ManyLds<W> &l, int r, int head)
        : p(args), lds(l) {
        const CacheAttention &a = p.a;
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        h = head;
        P = a.c.page_size;
        table = a.table + (int64_t)(r < a.requests ? r : 0) * a.max_pages;
        whole = P >= 64;
        vrow = whole ? threadIdx.x >> 2 : lane;  // and vrow + 64, ...
        vgroup = whole ? threadIdx.x & 3 : wave;
        // (keeps the loads below vector loads: scalar ones return out of order)
        asm("v_mov_b32 %0, 0" : "=v"(zero));
    }
    template <typename X>
    __device__ __forceinline__ X at(const X *x, int64_t i) const {
        return *reinterpret_cast<const X *>(reinterpret_cast<const char *>(x + i) + zero);
    }
    __device__ __forceinline__ int clip(int u) const { return EVEN ? u : min(u, W - 1); }
    // A tile's table entry is read a tile before its bytes, and looked at only then (a check at
    // once would wait for it, and as loads come back in order, for every load before).
    __device__ __forceinline__ void find(int t) {
        entry = at(table, min(t + 16 * wave, p.cap - 1) >> p.shift);
    }
    __device__ __forceinline__ void load_k(int t) {
        const CacheAttention &a = p.a;
        const int page = __builtin_amdgcn_readfirstlane(entry);
        gone = page < 0 || page >= a.c.pages;
        block = (int64_t)(gone ? 0 : page) * a.c.heads + h;
        const int8_t *kp =
            a.c.keys + block * P * W + ((t + 16 * wave) & (P - 1)) * W;
#pragma unroll
        for (int i = 0; i < MU; ++i)
            kb[i] = *reinterpret_cast<const v4i *>(kp + (uint32_t)(clip(lane + 64 * i) * 16));
        ks = at(a.c.key_scales, block);
        vs = at(a.c.value_scales, block);
    }
    // (of the tile whose K was loaded last)
    __device__ __forceinline__ void load_v(int t) {
        const int8_t *vp = p.a.c.values + block * P * W + ((whole ? t : t + 16 * wave) & (P - 1));
#pragma unroll
        for (int i = 0; i < MU; ++i)
            vb[i] = *reinterpret_cast<const v4i *>(
                vp + (uint32_t)(clip(vrow + 64 * i) * P + (whole ? vgroup * 16 : 0)));
    }
    // Half n of 2 MU of K, then of V.
    __device__ __forceinline__ void put_k(int b, int n) {
        const int i = n >> 1, half = n & 1, unit = lane + 64 * i;
        if (EVEN || unit < W) {
            uint16_t *kp =
                lds.k[b] + (16 * wave + unit / CH) * KR + unit % CH * 16 + 8 * half;
            *reinterpret_cast<v8bf *>(kp) = bytes8_to_bf16(kb[i][2 * half], kb[i][2 * half + 1]);
        }
    }
    // a half-wavefront's eight tokens of each 16 are neighbours: 0-3, 8-11 and 4-7, 12-15, as
    // the rows of the first product fall
    __device__ __forceinline__ void put_v(int b, int n) {
        const int i = n >> 1, half = n & 1, row = vrow + 64 * i;
        if (EVEN || row < W) {
            uint16_t *vp = lds.v[b] + row * VR + vgroup * 16 + 8 * half;
            if constexpr (F16)
                *reinterpret_cast<v8h *>(vp) = bytes8_to_f16(vb[i][half], vb[i][half + 2]);
            else
                *reinterpret_cast<v8bf *>(vp) = bytes8_to_bf16(vb[i][half], vb[i][half + 2]);
        }
    }
    __device__ __forceinline__ void put_scales(int b) {
        if (lane == 0) {
            lds.scales[b][wave] = v4f{ks * p.c, vs, __builtin_amdgcn_logf(vs),
                                      __builtin_amdgcn_rcpf(vs)};
            lds.flags[b][wave] = (uint8_t)((gone ? 1 : 0) | (vs >= 0x1p-90f ? 2 : 0));
        }
    }
    __device__ __forceinline__ void pin_k() {
#pragma unroll
        for (int i = 0; i < MU; ++i) pin(kb[i]);
    }
    __device__ __forceinline__ void pin_v() {
#pragma unroll
        for (int i = 0; i < MU; ++i) pin(vb[i]);
    }
    __device__ __forceinline__ void stage_k(int b) {
        pin_k();
#pragma unroll
        for (int n = 0; n < 2 * MU; ++n) put_k(b, n);
        put_scales(b);
    }
    __device__ __forceinline__ void stage_v(int b) {
        pin_v();
#pragma unroll
        for (int n = 0; n < 2 * MU; ++n) put_v(b, n);
    }
};

template <typename T, int W>
__device__ __forceinline__ void many_rows(const AttnArgs &p, int id, ManyLds<W> &lds) {
    constexpr int QP = std::is_same<T, float>::value ? 3 : 1;
    constexpr int PP = QP;
    constexpr int ST = W / 16;       // steps of the first product
    constexpr int DT = W / 32;       // blocks of the second product
    constexpr int VA = W <= 128 && QP == 1 ? 2 : 1;  // groups of 16 tokens read ahead
    constexpr int KR = ManyLds<W>::KR, VR = ManyLds<W>::VR;
    auto &k_lds = lds.k;
    auto &v_lds = lds.v;
    auto &scale_lds = lds.scales;
    auto &flags_lds = lds.flags;
    auto &most_lds = lds.most;

    const CacheAttention &a = p.a;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lo32 = lane & 31, hi32 = lane >> 5;
    ManyTile x;
    if (!many_tile(p, id, x)) return;
    const int r = x.r, tile = x.tile, s0 = x.s0, rows = x.rows, h = x.h, split = x.split;
    ManyStage<W, QP == 1> st(p, lds, r, h);

    const int j = tile * kManyRows + wave * 32 + lo32;
    const int tok = j < rows ? s0 + j / p.group : s0;
    const int head = j < rows ? h * p.group + j % p.group : 0;
    // What the first tile needs is asked for at once, before it is known whether any row sees it
    // (a work-group's beginning is a chain of loads that wait for each other).
    const int lo = split * p.chunk;
    auto load = [&](int t) {
        st.load_k(t);
        st.load_v(t);
    };
    auto stage = [&](int b) {
        st.stage_k(b);
        st.stage_v(b);
    };

    st.find(lo);
    const int position = j < rows && r < a.requests ? a.positions[tok] : -1;
    Frag q[ST][QP];
    {
        const T *qp = static_cast<const T *>(a.Q) + (int64_t)tok * a.ldq +
                      (int64_t)head * a.c.dim;
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            const int d = 16 * s + 8 * hi32;
            query_frag<T, QP>(qp, d, j < rows && d < a.c.dim, q[s]);
        }
    }
    load(lo);
    st.find(lo + 64);
    if constexpr (QP == 1) spoil(q);  // (behind the loads: it waits for q)
    const int limit = keys_of(position, p.cap);
    // the work-group's longest row, this wavefront's and its shortest
    int most = limit, least = j < rows ? limit : INT32_MAX;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        most = max(most, __shfl_xor(most, o));
        least = min(least, __shfl_xor(least, o));
    }
    least = __builtin_amdgcn_readfirstlane(least);
    const int mine = __builtin_amdgcn_readfirstlane(most);
    if (lane == 0) most_lds[wave] = most;
    stage(0);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) most = max(most, most_lds[w]);
    most = __builtin_amdgcn_readfirstlane(most);
    const int hi = split == p.splits - 1 ? most : min(most, lo + p.chunk);
    if (split > 0 && lo >= most) return;

    float m = -INFINITY, l = 0.f;
    Weights weights;
    v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += 64, buf ^= 1) {
        const bool more = t0 + 64 < hi;
        if (more) load(t0 + 64);
        st.find(t0 + 128);  // (always: a value that only a branch loads is copied, and waited for)
        if (t0 < mine) {  // (else none of this wavefront's rows sees the tile)
        const uint32_t flags = __builtin_amdgcn_readfirstlane(
            *reinterpret_cast<const uint32_t *>(flags_lds[buf]));
        const uint32_t lost = flags & 0x01010101u;

        // The products' operands are read from LDS several steps ahead (a read takes longer than
        // a step's instructions); the accumulators of neighbouring instructions are different
        // ones.
        constexpr int KA = ST < 4 ? ST : 4;  // steps ahead
        v16f s[2];
        const v16f none = {};
        const uint16_t *kp = k_lds[buf] + lo32 * KR + 8 * hi32;
        v8bf kf[KA][2];
        auto read_k = [&](int i) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
                kf[i % KA][b] = *reinterpret_cast<const v8bf *>(kp + 32 * b * KR + 16 * i);
        };
#pragma unroll
        for (int i = 0; i < KA; ++i) read_k(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < ST; ++i) {
#pragma unroll
            for (int n = QP - 1; n >= 0; --n)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        kf[i % KA][b], q[i][n].v, i == 0 && n == QP - 1 ? none : s[b], 0, 0,
                        0);
            if (i + KA < ST) read_k(i + KA);
        }
        const uint16_t *vp = v_lds[buf] + lo32 * VR + 8 * hi32;
        v8bf vf[VA][DT];
        auto read_v = [&](int x) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
                vf[x % VA][d] = *reinterpret_cast<const v8bf *>(vp + 32 * d * VR + 16 * x);
        };
#pragma unroll
        for (int x = 0; x < VA; ++x) read_v(x);
        __builtin_amdgcn_sched_barrier(0);
        float ks[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) ks[w] = scale_lds[buf][w][0];
        // Scores are s * ks. Where some are masked, a ks that -inf could not be multiplied with
        // (0, tiny, NaN) is multiplied first.
        if (t0 + 64 > least || lost != 0) {  // the same for the wavefront
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int seen = lost >> 8 * w & 1 ? 0 : limit - t0 - 16 * w - 4 * hi32;
                const bool odd = !(ks[w] >= 0x1p-100f);
                const float by = odd ? ks[w] : 1.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = s[w >> 1][8 * (w & 1) + i] * by;
                    s[w >> 1][8 * (w & 1) + i] = 8 * (i >> 2) + (i & 3) < seen ? x : -INFINITY;
                }
                ks[w] = odd ? 1.f : ks[w];
            }
        }
        float top = -INFINITY, big = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const v16f &x = s[w >> 1];
            const int i = 8 * (w & 1);
            const float most = max3(max3(max3(x[i], x[i + 1], x[i + 2]), x[i + 3], x[i + 4]),
                                    x[i + 5], max3(x[i + 6], x[i + 7], x[i])) * ks[w];
            top = fmaxf(top, most);
            if constexpr (PP == 1) big = fmaxf(big, most + scale_lds[buf][w][2]);
        }
        // m is any number near the largest score: it follows only where it would be left behind
        // by more than kLag, so the sums are rarely scaled anew
        if (__ballot(top > m + kLag || (PP == 1 && big > weights.top + kLag)) != 0) {
            top = fmaxf(top, __shfl_xor(top, 32));
            const float now = fmaxf(m, top);
            const float alpha = __builtin_amdgcn_exp2f(m - (now == -INFINITY ? 0.f : now));
            l *= alpha;
            m = now;
            float by = alpha;
            if constexpr (PP == 1) by = weights.follow(fmaxf(big, __shfl_xor(big, 32)), m);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= by;
        }
        Frag w[4][PP];
        const float unit = weights.unit();
        bool near = false;
        if constexpr (PP == 1) {
            const float low = fminf(fminf(scale_lds[buf][0][2], scale_lds[buf][1][2]),
                                    fminf(scale_lds[buf][2][2], scale_lds[buf][3][2]));
            near = (flags & 0x02020202u) == 0x02020202u &&
                   __ballot(low - weights.over < kFar) == 0;
        }
        if (near) {
            // the sum is taken over the rounded weights, so that numerator and denominator round
            // alike (a row that sees one key gives its value, whatever the scale's bits)
            const float to_m = weights.to_m();
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float less = scale_lds[buf][x][2] - unit;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        e[k] = __builtin_amdgcn_exp2f(
                            fmaf(s[x >> 1][8 * (x & 1) + 2 * i + k], ks[x], less));
                    w[x][0].u[i] = pack_f16(e[0], e[1]);
                    sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w[x][0].u[i]),
                                                 v2h{(_Float16)1.f, (_Float16)1.f}, sum, false);
                }
                l = fmaf(sum, scale_lds[buf][x][3] * to_m, l);
            }
        } else {  // (a scale of 0, a tiny one, NaN, one far below a row's, or float32)
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float z = fmaf(s[x >> 1][8 * (x & 1) + 2 * i + k], ks[x], -base);
                        e[k] = __builtin_amdgcn_exp2f(z);
                        l += e[k];
                        if constexpr (PP == 1)
                            e[k] = __builtin_amdgcn_exp2f(z + (scale_lds[buf][x][2] + base - unit));
                        else
                            e[k] *= scale_lds[buf][x][1];
                        e[k] = z != -INFINITY ? e[k] : 0.f;
                    }
                    if constexpr (PP == 1) {
                        w[x][0].u[i] = pack_f16(e[0], e[1]);
                    } else {
                        uint32_t part[PP];
                        split_pair<PP>(e[0], e[1], part);
#pragma unroll
                        for (int n = 0; n < PP; ++n) w[x][n].u[i] = part[n];
                    }
                }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int n = PP - 1; n >= 0; --n)
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    if constexpr (PP == 1)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            __builtin_bit_cast(v8h, vf[x % VA][d]), w[x][n].h, o[d], 0, 0, 0);
                    else
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[x % VA][d], w[x][n].v,
                                                                       o[d], 0, 0, 0);
                }
            if (x + VA < 4) read_v(x + VA);
        }
        }
        if (more) stage(buf ^ 1);
        __syncthreads();
    }
    l += __shfl_xor(l, 32);
    if constexpr (PP == 1) {
        const float natural = weights.natural();
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * 0x1p-6f * natural;  // (2^-kUnit)
    }

    if (j < rows) {
        const int64_t row = (int64_t)tok * a.heads + head;
        const bool direct = row_is_whole(p, limit);
        if (direct && split > 0) return;
        const int64_t at = row * p.splits + split;
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (!direct && hi32 == 0) {
            p.part_ml[at * 2] = m;
            p.part_ml[at * 2 + 1] = l;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int dd = 32 * d + 8 * i + 4 * hi32;
                v4f x;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = o[d][4 * i + k];
                if (!direct) {
                    *reinterpret_cast<v4f *>(p.part_o + at * W + dd) = x;
                } else if (dd < a.c.dim) {
                    struct {
                        T t[4];
                    } y;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        y.t[k] = from_f32<T>(x[k] * inv);
                    store_any(static_cast<T *>(a.O) + row * a.c.dim + dd, y);
                }
            }
    }
}

// --------------------------------------------------------------------------- join
// A work-group joins the ranges of one row, in order within each of its thread groups and
// over them, under their common maximum.
template <typename T, int W>
__global__ void __launch_bounds__(256) attention_join_kernel(AttnArgs p) {
    constexpr int Q = W / 4;        // threads that hold a row of O
    constexpr int N = 256 / Q;      // ranges at a time
    __shared__ __attribute__((aligned(16))) float o_lds[N][W + 4];
    __shared__ float l_lds[N];
    const CacheAttention &a = p.a;
    const int64_t row = blockIdx.x;
    const int tok = (int)(row / a.heads);
    if (tok < a.starts[0] || tok >= clamp_int(a.starts[a.requests], 0, a.tokens)) return;
    const int limit = keys_of(a.positions[tok], p.cap);
    if (row_is_whole(p, limit)) return;
    const int n = min(p.splits, (limit + p.chunk - 1) / p.chunk);
    const int g = threadIdx.x / Q, d = threadIdx.x % Q * 4;
    const float *ml = p.part_ml + row * p.splits * 2;
    const float *po = p.part_o + row * p.splits * W;
    float top = -INFINITY;
    for (int s = threadIdx.x & 63; s < n; s += 64) top = fmaxf(top, ml[2 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (g < N) {
        float l = 0.f;
        v4f x = {0.f, 0.f, 0.f, 0.f};
        for (int s = g; s < n; s += N) {
            const float ms = ml[2 * s], ls = ml[2 * s + 1];
            // (a range whose scores were all NaN has sum NaN and no maximum)
            const float f = ms == -INFINITY ? (ls == 0.f ? 0.f : 1.f)
                                            : __builtin_amdgcn_exp2f(ms - top);
            const v4f y = *reinterpret_cast<const v4f *>(po + (int64_t)s * W + d);
            l += ls * f;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += y[i] * f;
        }
        *reinterpret_cast<v4f *>(&o_lds[g][d]) = x;
        if (d == 0) l_lds[g] = l;
    }
    __syncthreads();
    if (threadIdx.x < Q && d < a.c.dim) {
        float l = 0.f;
        v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < N; ++k) {
            l += l_lds[k];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] += o_lds[k][d + i];
        }
        struct {
            T t[4];
        } y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.t[i] = from_f32<T>(l == 0.f ? 0.f : x[i] / l);
        store_any(static_cast<T *>(a.O) + row * a.c.dim + d, y);
    }
}

// Joins what few_shares cut: one request and query head a work-group (a row of each token),
// parts side by side over its thread groups and in order within them, under their common
// maximum.
template <typename T, int W>
__global__ void __launch_bounds__(256) attention_share_join_kernel(AttnArgs p) {
    constexpr int Q = W / 4;    // threads that hold a row of O
    constexpr int N = 256 / Q;  // parts at a time
    __shared__ __attribute__((aligned(16))) float o_lds[N][W + 4];
    __shared__ float l_lds[N];
    const CacheAttention &a = p.a;
    const int r = blockIdx.x / a.heads, head = blockIdx.x % a.heads;
    const int h = head / p.group;
    const int before = p.firsts[r], n = p.firsts[r + 1] - before;
    const int all_requests = a.requests + kNoRequest;
    const int tiles = p.firsts[all_requests], unit = p.firsts[all_requests + 1 + r];
    if (n == 0 || unit <= 2 * kSnap) return;
    const Shares s = shares_of(p, tiles);
    int s0, s1;
    request_tokens(a, r, s0, s1);
    const int g = threadIdx.x / Q, d = threadIdx.x % Q * 4;
    for (int tok = s0; tok < s1; ++tok) {
        const int j = (tok - s0) * p.group + head % p.group;
        const int begin = before * a.c.heads + h * n + j / 16 * unit;
        const int cut0 = (begin + kSnap) / s.each + 1;         // the first cut inside
        const int cut1 = min(begin + unit - kSnap, s.total) - 1;
        const int parts = cut1 / s.each - cut0 + 2;            // (to the last one)
        if (parts < 2) continue;
        auto place = [&](int k) {
            return (int64_t)(k == 0 ? 2 * (cut0 - 1) + 1 : 2 * (cut0 + k - 1)) * 16 + j % 16;
        };
        float top = -INFINITY;
        for (int k = threadIdx.x & 63; k < parts; k += 64)
            top = fmaxf(top, p.part_ml[place(k) * 2]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if (g < N) {
            float l = 0.f;
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int k = g; k < parts; k += N) {
                const int64_t at = place(k);
                const float ms = p.part_ml[at * 2], ls = p.part_ml[at * 2 + 1];
                // (a part whose scores were all NaN has sum NaN and no maximum)
                const float f = ms == -INFINITY ? (ls == 0.f ? 0.f : 1.f)
                                                : __builtin_amdgcn_exp2f(ms - top);
                const v4f y = *reinterpret_cast<const v4f *>(p.part_o + at * W + d);
                l += ls * f;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += y[i] * f;
            }
            *reinterpret_cast<v4f *>(&o_lds[g][d]) = x;
            if (d == 0) l_lds[g] = l;
        }
        __syncthreads();
        if (threadIdx.x < Q && d < a.c.dim) {
            float l = 0.f;
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < N; ++k) {
                l += l_lds[k];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] += o_lds[k][d + i];
            }
            struct {
                T t[4];
            } y;
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int i = 0; i < 4; ++i) y.t[i] = from_f32<T>(x[i] * inv);
            store_any(static_cast<T *>(a.O) + ((int64_t)tok * a.heads + head) * a.c.dim + d, y);
        }
        __syncthreads();
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(W <= 128 ? 2 : 1)))
attention_share_kernel(AttnArgs p) {
    __shared__ FewLds<W> lds;
    __shared__ ShareLds scan;
    few_shares<T, W>(p, lds, scan);
}

template <typename T, int W>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(W <= 128 ? 2 : 1)))
attention_few_kernel(AttnArgs p) {
    __shared__ FewLds<W> lds;
    few_rows<T, W>(p, blockIdx.x, lds);
}

// Both in one launch, each request's rows where they belong: the few-rows work-groups first.
template <typename T, int W>
__global__ void __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 || W > 128 ? 1 : 2)))
attention_both_kernel(AttnArgs p, int few) {
    __shared__ union {
        FewLds<W> few;
        ManyLds<W> many;
    } lds;
    if ((int)blockIdx.x < few) {
        few_rows<T, W>(p, blockIdx.x, lds.few);
    } else {
        many_rows<T, W>(p, blockIdx.x - few, lds.many);
    }
}

template <typename T, int W>
int launch_width(hipStream_t stream, const AttnArgs &p) {
    if (p.shares != 0) {
        MIGEMM_LAUNCH((attention_share_kernel<T, W>), dim3((unsigned)p.shares), dim3(256), 0,
                      stream, p);
        if (const int rc = launch_status("attention kernel launch")) return rc;
        if (p.cap <= 64 * (2 * kSnap + 1)) return MIGEMM_OK;  // (no unit is long enough to cut)
        MIGEMM_LAUNCH((attention_share_join_kernel<T, W>),
                      dim3((unsigned)(p.a.requests * p.a.heads)), dim3(256), 0, stream, p);
        return launch_status("attention_share_join_kernel launch");
    }
    const int few = p.splits * p.a.c.heads * (p.a.requests + kNoRequest);
    if (p.both)
        MIGEMM_LAUNCH((attention_both_kernel<T, W>),
                      dim3((unsigned)(few + p.units * p.splits * p.a.c.heads)), dim3(256),
                      0, stream, p, few);
    else
        MIGEMM_LAUNCH((attention_few_kernel<T, W>), dim3((unsigned)few), dim3(256), 0, stream,
                      p);
    if (const int rc = launch_status("attention kernel launch")) return rc;
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.a.tokens * p.a.heads;
        MIGEMM_LAUNCH((attention_join_kernel<T, W>), dim3((unsigned)rows), dim3(256), 0, stream,
                      p);
        if (const int rc = launch_status("attention_join_kernel launch")) return rc;
    }
    return MIGEMM_OK;
}

template <typename T>
int launch_widths(hipStream_t stream, const AttnArgs &p) {
    switch (p.a.c.width) {
        case 32: return launch_width<T, 32>(stream, p);
        case 64: return launch_width<T, 64>(stream, p);
        case 96: return launch_width<T, 96>(stream, p);
        case 128: return launch_width<T, 128>(stream, p);
        case 192: return launch_width<T, 192>(stream, p);
        default: return launch_width<T, 256>(stream, p);
    }
}
}  // namespace

int launch_attention_f32(hipStream_t stream, const AttnArgs &p);
int launch_attention_bf16(hipStream_t stream, const AttnArgs &p);

}  // namespace migemm
