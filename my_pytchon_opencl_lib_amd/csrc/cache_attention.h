// Causal attention over the 8-bit paged cache: the kernels, instantiated by
// cache_attention_f32.hip and cache_attention_bf16.hip.
//
// For a row (a query token and head) with n keys: S = c (q . k8) ks, p = 2^(S - max S),
// O = sum p vs v8 / sum p, with c = scale log2 e, k8 and v8 the bytes, ks and vs the scales
// of their page and head; one pass over the keys with the running maximum and sum, in fp32.
//
// The bytes are exact in bf16 (7 bits), so both products run on the bf16 matrix cores with
// the cache's side exact. A bf16 query is exact too. A float32 query, and p vs, are cut into
// bf16 parts whose products add up in the fp32 accumulator: three parts (24 bits) for float32
// calls, so that they are as exact as float32 arithmetic; for bf16 calls two in the few-rows
// kernel (it waits for memory) and one in the many-rows kernel, which sums the rounded weights
// for the denominator too: their roundings average over the keys and stay below the result's.
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
    int both;           // few- and many-rows kernels run, each takes its requests
    int units;          // many-rows kernel: tiles of rows that the grid covers
    float *part_o;      // [tokens * heads][splits][width]
    float *part_ml;     // [tokens * heads][splits][2]
};

constexpr int kFewRows = 16;
constexpr int kManyRows = 128;

namespace {

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Tokens [s0, s1) of request r; r == requests: the tokens past the last request's, without
// keys.
__device__ __forceinline__ void request_tokens(const CacheAttention &a, int r, int &s0,
                                               int &s1) {
    s0 = clamp_int(a.starts[r], 0, a.tokens);
    s1 = r < a.requests ? clamp_int(a.starts[r + 1], s0, a.tokens) : a.tokens;
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
};

// Eight neighbouring values of a query row from d on (0 at and after `left`), in N parts.
template <typename T, int N>
__device__ __forceinline__ void query_frag(const T *q, int left, Frag (&f)[N]) {
    float x[8];
    load_f32<T, 8>(q, left, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t part[N];
        split_pair<N>(x[2 * i], x[2 * i + 1], part);
#pragma unroll
        for (int n = 0; n < N; ++n) f[n].u[i] = part[n];
    }
}

// Rows that are whole after range 0 are written by it; others leave a part for each range.
__device__ __forceinline__ bool row_is_whole(const AttnArgs &p, int limit) {
    return p.splits == 1 || limit <= p.chunk;
}

// ------------------------------------------------------------------------- few rows
// Up to 16 rows (queries x heads that share a kv head): decoding. Bound by reading the cache
// once. A work-group takes one request, kv head and range of keys; its four wavefronts take
// tiles of 64 tokens in turn, straight from memory to registers (the next tile's loads fly
// while one is computed), on v_mfma_f32_16x16x32_bf16. Row m of subtile u is token
// 16 (m / 4) + 4 u + m % 4 of the tile, so that lane group g ends up with the scores of
// tokens 16 g .. 16 g + 15, whose bytes of V^T are 16 neighbours: one load a row of V.
template <typename T, int W>
__global__ void __launch_bounds__(256) attention_few_kernel(AttnArgs p) {
    constexpr int QP = std::is_same<T, float>::value ? 3 : 1;
    constexpr int PP = std::is_same<T, float>::value ? 3 : 2;
    constexpr int ST = W / 32;   // steps of the first product
    constexpr int KD = W / 16;   // dwords of a K row that a lane takes
    constexpr int DT = W / 16;   // blocks of the second product
    constexpr int OS = W + 4;    // LDS row
    __shared__ __attribute__((aligned(16))) float o_lds[4 * 16 * OS];
    __shared__ float m_lds[4][16], l_lds[4][16];

    const CacheAttention &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    int id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int h = id % a.c.heads;
    const int r = id / a.c.heads;
    int s0, s1;
    request_tokens(a, r, s0, s1);
    const int rows = (s1 - s0) * p.group;
    if (p.both && rows > kFewRows) return;
    const int P = a.c.page_size;
    const int *table = a.table + (int64_t)(r < a.requests ? r : 0) * a.max_pages;
    const int64_t page_bytes = (int64_t)P * W;

    for (int row0 = 0; row0 < rows; row0 += 16) {
        const int j = row0 + col;
        const int tok = s0 + j / p.group;
        const int head = h * p.group + j % p.group;
        const int limit = j < rows && r < a.requests
                              ? keys_of(a.positions[tok], p.cap)
                              : 0;
        int most = limit;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o));
        most = __builtin_amdgcn_readfirstlane(most);
        const int lo = split * p.chunk;
        const int hi = split == p.splits - 1 ? most : min(most, lo + p.chunk);
        if (split > 0 && lo >= most) continue;  // (the same for the whole work-group)

        Frag q[ST][QP];
        {
            const T *qp = static_cast<const T *>(a.Q) + (int64_t)(j < rows ? tok : s0) * a.ldq +
                          (int64_t)head * a.c.dim;
            if (j >= rows) qp = static_cast<const T *>(a.Q) + (int64_t)s0 * a.ldq;
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                const int d = g * (W / 4) + 8 * s;
                query_frag<T, QP>(qp + d, j < rows ? a.c.dim - d : 0, q[s]);
            }
        }

        uint32_t kb[4][KD];
        v4i vb[DT];
        float ks = 0.f, vs = 0.f;
        int page = -1;
        auto find = [&](int t0) {  // the page of lane group g's 16 tokens
            const int t = t0 + 16 * g;
            const int pg = t < hi ? table[t >> p.shift] : -1;
            return pg >= 0 && pg < a.c.pages ? pg : -1;
        };
        auto load = [&](int t0, int pg) {
            page = pg;
            const int64_t mine = (int64_t)max(pg, 0) * a.c.heads + h;
            ks = a.c.key_scales[mine];
            vs = a.c.value_scales[mine];
            const int kpage = max(__shfl(pg, (col >> 2) * 16), 0);
            const int8_t *kp = a.c.keys + ((int64_t)kpage * a.c.heads + h) * page_bytes +
                               ((t0 + 16 * (col >> 2) + (col & 3)) & (P - 1)) * W + g * (W / 4);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (W / 4 >= 16) {
#pragma unroll
                    for (int i = 0; i < W / 64; ++i) {
                        const v4i x = *reinterpret_cast<const v4i *>(kp + u * 4 * W + 16 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) kb[u][4 * i + e] = x[e];
                    }
                }
                if constexpr (W % 64 != 0) {
                    const uint2 x =
                        *reinterpret_cast<const uint2 *>(kp + u * 4 * W + W / 64 * 16);
                    kb[u][W / 64 * 4] = x.x;
                    kb[u][W / 64 * 4 + 1] = x.y;
                }
            }
            const int8_t *vp = a.c.values + mine * page_bytes + col * P + ((t0 + 16 * g) & (P - 1));
#pragma unroll
            for (int d = 0; d < DT; ++d)
                vb[d] = *reinterpret_cast<const v4i *>(vp + d * 16 * P);
        };

        float m = -INFINITY, l = 0.f;
        v4f o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};

        int t0 = lo + 64 * wave;
        int next = -1;
        if (t0 < hi) {
            load(t0, find(t0));
            if (t0 + 256 < hi) next = find(t0 + 256);
        }
        for (; t0 < hi; t0 += 256) {
            // first product, then this tile's K registers are free for the next tile
            v4f s[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                s[u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < ST; ++st) {
                    const v8bf k = bytes8_to_bf16(kb[u][2 * st], kb[u][2 * st + 1]);
#pragma unroll
                    for (int n = QP - 1; n >= 0; --n)
                        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[st][n].v, s[u], 0, 0,
                                                                       0);
                }
            }
            const float sc = ks * p.c;
            const float vscale = vs;
            const int seen = page < 0 ? 0 : limit - t0 - 16 * g;  // of this lane's 16 tokens
            v4i v[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) v[d] = vb[d];
            if (t0 + 256 < hi) {
                load(t0 + 256, next);
                if (t0 + 512 < hi) next = find(t0 + 512);
            }
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[u][i] = 4 * u + i < seen ? s[u][i] * sc : -INFINITY;
                    top = fmaxf(top, s[u][i]);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float now = fmaxf(m, top);
            const float base = now == -INFINITY ? 0.f : now;
            if (__ballot(now != m) != 0) {
                const float alpha = __builtin_amdgcn_exp2f(m - base);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
                m = now;
            }
            Frag w[2][PP];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = __builtin_amdgcn_exp2f(s[u][i] - base);
                    l += e[i];
                    e[i] = 4 * u + i < seen ? e[i] * vscale : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t part[PP];
                    split_pair<PP>(e[2 * i], e[2 * i + 1], part);
#pragma unroll
                    for (int n = 0; n < PP; ++n) w[u / 2][n].u[2 * (u & 1) + i] = part[n];
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const v8bf x = bytes8_to_bf16(v[d][0], v[d][1]);
                const v8bf y = bytes8_to_bf16(v[d][2], v[d][3]);
#pragma unroll
                for (int n = PP - 1; n >= 0; --n) {
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w[0][n].v, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y, w[1][n].v, o[d], 0, 0, 0);
                }
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);

        // the four wavefronts' results under their common maximum, added in order
        if (g == 0) {
            m_lds[wave][col] = m;
            l_lds[wave][col] = l;
        }
        __syncthreads();
        float top = m_lds[0][col];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, m_lds[w][col]);
        const float f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            v4f x = o[d];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] *= f;
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
        for (int e = tid; e < 16 * (W / 4); e += 256) {
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
            const int lim = r < a.requests ? keys_of(a.positions[tk], p.cap) : 0;
            const float sum = l_lds[0][c];
            if (row_is_whole(p, lim)) {
                if (split == 0 && d < a.c.dim) {
                    struct {
                        T t[4];
                    } y;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        y.t[i] = from_f32<T>(sum == 0.f ? 0.f : x[i] / sum);
                    store_any(static_cast<T *>(a.O) + row * a.c.dim + d, y);
                }
            } else {
                const int64_t at = row * p.splits + split;
                *reinterpret_cast<v4f *>(p.part_o + at * W + d) = x;
                if (d == 0) {
                    p.part_ml[at * 2] = m_lds[0][c];
                    p.part_ml[at * 2 + 1] = sum;
                }
            }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------ many rows
// Prompts: 128 rows (queries x heads that share a kv head) a work-group, 32 a wavefront, on
// v_mfma_f32_32x32x16_bf16. Tiles of 64 tokens are read as bytes, turned into bf16 once for
// the work-group and shared in LDS (two buffers: the next tile's bytes fly during a tile's
// work, one barrier a tile). Bound by the matrix cores and by the exponentials and
// conversions beside them. LDS rows are padded by 16 bytes: the 16 lanes of a read phase fall
// on different banks.
template <typename T, int W>
__global__ void __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(std::is_same<T, float>::value || W > 128 ? 1 : 2)))
attention_many_kernel(AttnArgs p) {
    constexpr int QP = std::is_same<T, float>::value ? 3 : 1;
    constexpr int PP = QP;
    constexpr int ST = W / 16;       // steps of the first product
    constexpr int DT = W / 32;       // blocks of the second product
    constexpr int KR = W + 8;        // LDS rows, in bf16
    constexpr int VR = 64 + 8;
    constexpr int KD = W / 16;       // dwords of K a thread moves
    constexpr int VU = (W * 4 + 255) / 256;  // units of 16 bytes of V a thread moves
    __shared__ __attribute__((aligned(16))) uint16_t k_lds[2][64 * KR];
    __shared__ __attribute__((aligned(16))) uint16_t v_lds[2][W * VR];
    __shared__ float scale_lds[2][8];  // ks c of the tile's four groups of 16 tokens, then vs
    __shared__ uint32_t lost_lds[2];

    const CacheAttention &a = p.a;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lo32 = lane & 31, hi32 = lane >> 5;

    int id = blockIdx.x;
    const int h = id % a.c.heads;
    id /= a.c.heads;
    const int split = id % p.splits;
    id /= p.splits;
    // which request's tile: requests in order, 64 at a time
    int r = -1, tile = 0, s0 = 0, s1 = 0;
    for (int base = 0, before = 0; base <= a.requests; base += 64) {
        int x0 = 0, x1 = 0, n = 0;
        if (base + lane <= a.requests) {
            request_tokens(a, base + lane, x0, x1);
            const int rows = (x1 - x0) * p.group;
            n = rows > kFewRows || !p.both ? (rows + kManyRows - 1) / kManyRows : 0;
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
    if (r < 0) return;
    r = __builtin_amdgcn_readfirstlane(r);
    s0 = __builtin_amdgcn_readfirstlane(s0);
    s1 = __builtin_amdgcn_readfirstlane(s1);
    tile = __builtin_amdgcn_readfirstlane(tile);
    const int rows = (s1 - s0) * p.group;
    const int P = a.c.page_size;
    const int *table = a.table + (int64_t)(r < a.requests ? r : 0) * a.max_pages;
    const int64_t page_bytes = (int64_t)P * W;

    const int j = tile * kManyRows + wave * 32 + lo32;
    const int tok = j < rows ? s0 + j / p.group : s0;
    const int head = j < rows ? h * p.group + j % p.group : 0;
    const int limit =
        j < rows && r < a.requests ? keys_of(a.positions[tok], p.cap) : 0;
    // the work-group's longest row, and this wavefront's shortest
    __shared__ int most_lds[4];
    int most = limit, least = j < rows ? limit : INT32_MAX;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        most = max(most, __shfl_xor(most, o));
        least = min(least, __shfl_xor(least, o));
    }
    least = __builtin_amdgcn_readfirstlane(least);
    if (lane == 0) most_lds[wave] = most;
    __syncthreads();
    most = max(max(most_lds[0], most_lds[1]), max(most_lds[2], most_lds[3]));
    most = __builtin_amdgcn_readfirstlane(most);
    const int lo = split * p.chunk;
    const int hi = split == p.splits - 1 ? most : min(most, lo + p.chunk);
    if (split > 0 && lo >= most) return;

    Frag q[ST][QP];
    {
        const T *qp = static_cast<const T *>(a.Q) + (int64_t)tok * a.ldq +
                      (int64_t)head * a.c.dim;
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            const int d = 16 * s + 8 * hi32;
            query_frag<T, QP>(qp + d, j < rows ? a.c.dim - d : 0, q[s]);
        }
    }

    // this thread's part of a tile: a quarter row of K (token tid / 4: group = wave), units of
    // 16 bytes of V (row d = unit / 4, group unit % 4)
    uint32_t kb[KD];
    v4i vb[VU];
    float sc = 0.f;
    auto page_at = [&](int t) {
        const int pg = t < hi ? table[t >> p.shift] : -1;
        return pg >= 0 && pg < a.c.pages ? pg : -1;
    };
    // (the pages of a tile are looked up a tile before its bytes are loaded)
    int kpage = -1, vpage = -1;
    auto find = [&](int t0) {
        kpage = page_at(t0 + 16 * wave);
        vpage = page_at(t0 + 16 * (tid & 3));
    };
    uint32_t gone = 0;
    auto load = [&](int t0) {
        gone = (uint32_t)__ballot(lane < 4 && t0 + 16 * lane < hi && vpage < 0);
        const int8_t *kp = a.c.keys + ((int64_t)max(kpage, 0) * a.c.heads + h) * page_bytes +
                           ((t0 + (tid >> 2)) & (P - 1)) * W + (tid & 3) * (W / 4);
        if constexpr (W / 4 >= 16) {
#pragma unroll
            for (int i = 0; i < W / 64; ++i) {
                const v4i x = *reinterpret_cast<const v4i *>(kp + 16 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) kb[4 * i + e] = x[e];
            }
        }
        if constexpr (W % 64 != 0) {
            const uint2 x = *reinterpret_cast<const uint2 *>(kp + W / 64 * 16);
            kb[W / 64 * 4] = x.x;
            kb[W / 64 * 4 + 1] = x.y;
        }
        const int8_t *vp = a.c.values + ((int64_t)max(vpage, 0) * a.c.heads + h) * page_bytes +
                           ((t0 + 16 * (tid & 3)) & (P - 1));
#pragma unroll
        for (int i = 0; i < VU; ++i) {
            const int d = (tid + 256 * i) >> 2;
            vb[i] = *reinterpret_cast<const v4i *>(vp + min(d, W - 1) * P);
        }
        if (tid < 8) {  // tid & 3: the group
            const int64_t at = (int64_t)max(vpage, 0) * a.c.heads + h;
            sc = tid < 4 ? a.c.key_scales[at] * p.c : a.c.value_scales[at];
        }
    };
    auto stage = [&](int b) {
        uint16_t *kp = k_lds[b] + (tid >> 2) * KR + (tid & 3) * (W / 4);
#pragma unroll
        for (int i = 0; i < KD / 2; ++i)
            *reinterpret_cast<v8bf *>(kp + 8 * i) = bytes8_to_bf16(kb[2 * i], kb[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < VU; ++i) {
            const int d = (tid + 256 * i) >> 2;
            if (W * 4 % 256 == 0 || d < W) {
                // a half-wavefront's eight tokens of each 16 are neighbours: 0-3, 8-11 and
                // 4-7, 12-15, as the rows of the first product fall
                uint16_t *vp = v_lds[b] + d * VR + (tid & 3) * 16;
                *reinterpret_cast<v8bf *>(vp) = bytes8_to_bf16(vb[i][0], vb[i][2]);
                *reinterpret_cast<v8bf *>(vp + 8) = bytes8_to_bf16(vb[i][1], vb[i][3]);
            }
        }
        if (tid < 8) scale_lds[b][tid] = sc;
        if (tid == 0) lost_lds[b] = gone;
    };

    float m = -INFINITY, l = 0.f;
    v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

    if (lo < hi) {
        find(lo);
        load(lo);
        find(lo + 64);
        stage(0);
    }
    __syncthreads();
    int buf = 0;
    for (int t0 = lo; t0 < hi; t0 += 64, buf ^= 1) {
        const bool more = t0 + 64 < hi;
        if (more) {
            load(t0 + 64);
            find(t0 + 128);
        }
        // pages of the tile that are outside the pool (one bit for each group of 16 tokens)
        const uint32_t lost = lost_lds[buf];

        v16f s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                const v8bf k = *reinterpret_cast<const v8bf *>(
                    k_lds[buf] + (32 * b + lo32) * KR + 16 * st + 8 * hi32);
#pragma unroll
                for (int n = QP - 1; n >= 0; --n)
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[st][n].v, s[b], 0, 0, 0);
            }
        }
        float ks[4], vs[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ks[w] = scale_lds[buf][w];
            vs[w] = scale_lds[buf][4 + w];
        }
        const bool whole = t0 + 64 <= least && lost == 0;  // the same for the wavefront
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = s[w >> 1][8 * (w & 1) + i] * ks[w];
                if (!whole) {
                    const int t = t0 + 16 * w + 8 * (i >> 2) + 4 * hi32 + (i & 3);
                    x = t < limit && !(lost >> w & 1) ? x : -INFINITY;
                }
                s[w >> 1][8 * (w & 1) + i] = x;
                top = fmaxf(top, x);
            }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float now = fmaxf(m, top);
        const float base = now == -INFINITY ? 0.f : now;
        if (__ballot(now != m) != 0) {
            const float alpha = __builtin_amdgcn_exp2f(m - base);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
            m = now;
        }
        Frag w[4][PP];
        const bool plain_scales = vs[0] >= 0x1p-90f && vs[1] >= 0x1p-90f &&
                                  vs[2] >= 0x1p-90f && vs[3] >= 0x1p-90f;
        if (PP == 1 && plain_scales) {
            // one part: the sum is taken over the rounded weights, so that numerator and
            // denominator round alike (a row that sees one key gives its value, whatever the
            // scale's bits; p vs alone would be off by the same 2^-9 in all of a page)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        e[k] = __builtin_amdgcn_exp2f(s[x >> 1][8 * (x & 1) + 2 * i + k] -
                                                      base) * vs[x];
                    w[x][0].u[i] = pack_bf16(e[0], e[1]);
                    sum += bf16_low(w[x][0].u[i]) + bf16_high(w[x][0].u[i]);
                }
                l += sum * __builtin_amdgcn_rcpf(vs[x]);
            }
        } else {  // (a scale of 0, a tiny one, NaN, or float32)
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float z = s[x >> 1][8 * (x & 1) + 2 * i + k];
                        e[k] = __builtin_amdgcn_exp2f(z - base);
                        l += e[k];
                        e[k] = whole || z != -INFINITY ? e[k] * vs[x] : 0.f;
                    }
                    uint32_t part[PP];
                    split_pair<PP>(e[0], e[1], part);
#pragma unroll
                    for (int n = 0; n < PP; ++n) w[x][n].u[i] = part[n];
                }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const v8bf v = *reinterpret_cast<const v8bf *>(
                    v_lds[buf] + (32 * d + lo32) * VR + 16 * x + 8 * hi32);
#pragma unroll
                for (int n = PP - 1; n >= 0; --n)
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, w[x][n].v, o[d], 0, 0, 0);
            }
        if (more) stage(buf ^ 1);
        __syncthreads();
    }
    l += __shfl_xor(l, 32);

    if (j < rows) {
        const int64_t row = (int64_t)tok * a.heads + head;
        const bool direct = row_is_whole(p, limit);
        if (direct && split > 0) return;
        const int64_t at = row * p.splits + split;
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
                        y.t[k] = from_f32<T>(l == 0.f ? 0.f : x[k] / l);
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
    if (tok >= clamp_int(a.starts[a.requests], 0, a.tokens)) return;
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

// few, many: which kernels the call runs.
template <typename T, int W>
int launch_width(hipStream_t stream, const AttnArgs &p, bool few, bool many) {
    if (many) {
        const int64_t blocks = (int64_t)p.units * p.splits * p.a.c.heads;
        MIGEMM_LAUNCH((attention_many_kernel<T, W>), dim3((unsigned)blocks), dim3(256), 0,
                      stream, p);
        if (const int rc = launch_status("attention_many_kernel launch")) return rc;
    }
    if (few) {
        const int64_t blocks = (int64_t)p.splits * p.a.c.heads * (p.a.requests + 1);
        MIGEMM_LAUNCH((attention_few_kernel<T, W>), dim3((unsigned)blocks), dim3(256), 0, stream,
                      p);
        if (const int rc = launch_status("attention_few_kernel launch")) return rc;
    }
    if (p.splits > 1) {
        const int64_t rows = (int64_t)p.a.tokens * p.a.heads;
        MIGEMM_LAUNCH((attention_join_kernel<T, W>), dim3((unsigned)rows), dim3(256), 0, stream,
                      p);
        if (const int rc = launch_status("attention_join_kernel launch")) return rc;
    }
    return MIGEMM_OK;
}

template <typename T>
int launch_widths(hipStream_t stream, const AttnArgs &p, bool few, bool many) {
    switch (p.a.c.width) {
        case 32: return launch_width<T, 32>(stream, p, few, many);
        case 64: return launch_width<T, 64>(stream, p, few, many);
        case 96: return launch_width<T, 96>(stream, p, few, many);
        case 128: return launch_width<T, 128>(stream, p, few, many);
        case 192: return launch_width<T, 192>(stream, p, few, many);
        default: return launch_width<T, 256>(stream, p, few, many);
    }
}
}  // namespace

int launch_attention_f32(hipStream_t stream, const AttnArgs &p, bool few, bool many);
int launch_attention_bf16(hipStream_t stream, const AttnArgs &p, bool few, bool many);

}  // namespace migemm
