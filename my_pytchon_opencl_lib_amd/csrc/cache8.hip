// The 8-bit paged cache: its tables and slots, and the kernels that write and read tokens.
// The layouts and rules are those of include/migemm.h (6).
#include "int8_common.h"

namespace migemm {
namespace {

// ---------------------------------------------------------------------- tables and slots
constexpr int TW = 1024;  // threads of a work-group, and tokens that one fills

// Inclusive scan over the work-group (part: 16 ints of LDS, free again on return).
template <typename F>
__device__ __forceinline__ int scan_block(int v, int *part, F op) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o);
        if (lane >= o) v = op(u, v);
    }
    if (lane == 63) part[wave] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TW / 64; ++w)
        if (w < wave) v = op(part[w], v);
    __syncthreads();
    return v;
}

// One launch, no work-group waits for another: each runs over all requests (a scan of the
// counts for the tokens' places, a scan of the pages asked for their pages; 8 bytes a request
// from L2) and keeps, in LDS, what the requests that own tokens of its window of 1024 tokens
// need; then one thread a token. Bound by latency: a step of a few hundred requests is one
// round of loads, two scans and one more dependent load (32 requests, a token each: 4.9 us; 512
// requests with 180000 tokens: 7.5 us). The token at a new page's first
// place writes that page to the table, so each entry has one writer; tokens in new pages take
// them from the free list and never read an entry that another work-group may be writing.
// GROW false: slots of the pages that the table already names, nothing is allocated.
template <bool GROW>
__global__ void __launch_bounds__(TW) cache_tables_kernel(TablesArgs a, int shift) {
    __shared__ int part[TW / 64];
    __shared__ int owner[TW], place[TW], ends[TW], first[TW], rank[TW];
    __shared__ int taken;
    const int tid = threadIdx.x;
    const int w0 = blockIdx.x * TW;
    const int cap = a.tokens + 1;  // places are added up to this: no sum overflows
    const int mask = (1 << shift) - 1;
    const int held = GROW ? min(max(*a.free_count, 0), a.free_capacity) : 0;
    owner[tid] = -1;
    if (tid == 0) taken = 0;
    auto capped = [cap](int x, int y) { return min(x + y, cap); };
    auto plus = [](int x, int y) { return x + y; };
    int end0 = 0, asks0 = 0;  // sums over the requests of earlier rounds
    __syncthreads();
    for (int base = 0; base < a.requests; base += TW) {
        const int r = base + tid;
        const bool is = r < a.requests;
        const int n = is ? max(a.lengths[r], 0) : 0;
        const int count = is ? max(a.counts[r], 0) : 0;
        const int c = min(count, cap);
        const int end = min(scan_block(c, part, capped) + end0, cap);
        const int start = end - c;
        const bool fits = is && (int64_t)n + count <= ((int64_t)a.max_pages << shift) &&
                          end <= a.tokens;  // (end is exact where it is below the cap)
        const int have = GROW ? (int)(((int64_t)n + mask) >> shift) : a.max_pages;
        const int asks = GROW && fits ? ((n + count + mask) >> shift) - have : 0;
        int upto = 0;
        if constexpr (GROW) upto = scan_block(asks, part, plus) + asks0;
        const bool ok = fits && (asks == 0 || upto <= held);
        if (is && blockIdx.x == 0) {
            a.starts[r + 1] = min(end, a.tokens);
            if (r == 0) a.starts[0] = 0;
            if constexpr (GROW) {
                a.new_lengths[r] = ok ? n + count : n;
                if (ok && asks > 0) atomicMax(&taken, upto);
            }
        }
        if (ok && c > 0 && end > w0 && start < w0 + TW) {
            const int at = max(start - w0, 0);
            owner[at] = r;
            place[at] = n - start;
            ends[at] = end;
            first[at] = have;
            rank[at] = upto - asks;
        }
        // carries: the last thread's sums
        __syncthreads();
        if (tid == TW - 1) {
            part[0] = end;
            part[1] = upto;
        }
        __syncthreads();
        end0 = part[0];
        asks0 = part[1];
        __syncthreads();
    }
    __syncthreads();
    if (GROW && blockIdx.x == 0 && tid == 0) *a.new_free = held - taken;
    const int own = scan_block(owner[tid] >= 0 ? tid : -1, part,
                               [](int x, int y) { return max(x, y); });
    const int t = w0 + tid;
    if (t >= a.tokens) return;
    int slot = -1, pos = -1;
    if (own >= 0 && t < ends[own]) {
        const int r = owner[own];
        const int p = place[own] + t;
        const int j = p >> shift;
        int *entry = a.table + (int64_t)r * a.max_pages + j;
        int page;
        if (GROW && j >= first[own]) {
            page = a.free_pages[held - 1 - (rank[own] + j - first[own])];
            if ((p & mask) == 0) *entry = page;
        } else {
            page = *entry;
        }
        if (page >= 0 && page <= INT32_MAX >> shift) {  // (else no page, or no int32 slot)
            slot = (page << shift) + (p & mask);
            pos = p;
        }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
}

// One work-group: a scheduler frees a few requests at a time, in order. It looks at one request
// after the other, a load that is waited for each: 512 requests with one finished take 45 us, with 8
// of 64 pages 53, with all 631.
__global__ void __launch_bounds__(TW)
cache_release_kernel(const int *finished, int *lengths, int requests, int *table, int max_pages,
                     int shift, int *free_pages, int pages, int *free_count) {
    __shared__ int part[TW / 64];
    __shared__ int last;
    const int tid = threadIdx.x;
    const int mask = (1 << shift) - 1;
    int count = min(max(*free_count, 0), pages);
    for (int r = 0; r < requests; ++r) {
        if (finished[r] == 0) continue;  // the same for every thread
        const int n = (int)min(((int64_t)max(lengths[r], 0) + mask) >> shift,
                               (int64_t)max_pages);
        for (int base = 0; base < n; base += TW) {
            const int j = base + tid;
            int *entry = table + (int64_t)r * max_pages + j;
            const int page = j < n ? *entry : -1;
            const int is = page >= 0 && page < pages;
            const int upto = scan_block(is, part, [](int x, int y) { return x + y; });
            if (is && count + upto <= pages) free_pages[count + upto - 1] = page;
            if (j < n) *entry = -1;
            if (tid == TW - 1) last = upto;
            __syncthreads();
            count = min(count + last, pages);
            __syncthreads();
        }
        __syncthreads();
        if (tid == 0) lengths[r] = 0;
    }
    __syncthreads();
    if (tid == 0) *free_count = count;
}

// ------------------------------------------------------------------------------ append
__device__ __forceinline__ int page_of(int slot, int shift, int pages) {
    const int page = slot >> shift;
    return slot >= 0 && page < pages ? page : -1;
}

struct AppendArgs {
    const void *x[2];  // K, V
    int64_t ld[2];
    const int *slots;
    int tokens, chunk;
    Cache8 c;
    int shift;
    FastDiv d8;  // head_dim / 8
};

// The slot of token t, -1 past the call's tokens or where it is outside the pool: skipped.
__device__ __forceinline__ int slot_at(const AppendArgs &a, int t) {
    const int slot = a.slots[min(max(t, 0), a.tokens - 1)];
    return t >= 0 && t < a.tokens && page_of(slot, a.shift, a.c.pages) >= 0 ? slot : -1;
}

// The slot of the last token before `end` that is not skipped, -1 if there is none; 256 tokens at
// a time (a wavefront's work, the same in each).
__device__ __forceinline__ int last_slot(const AppendArgs &a, int end) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int hi = end; hi > 0; hi -= 256) {
        int slot[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) slot[j] = slot_at(a, hi - 1 - lane - 64 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t is = __ballot(slot[j] >= 0);
            if (is != 0) return __shfl(slot[j], __builtin_ctzll(is));
        }
    }
    return -1;
}

// The first token from `begin` on that is not skipped, a.tokens if there is none.
__device__ __forceinline__ int next_token(const AppendArgs &a, int begin) {
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int lo = begin; lo < a.tokens; lo += 256) {
        int slot[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) slot[j] = slot_at(a, lo + lane + 64 * j);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t is = __ballot(slot[j] >= 0);
            if (is != 0) return lo + 64 * j + __builtin_ctzll(is);
        }
    }
    return a.tokens;
}

// A work-group takes the pages that begin (in the order of tokens) in its chunk of tokens, for
// one head and one of K and V, one after the other, so that each page and head has one owner:
// no atomics, and the scale, the rounding anew and the new tokens follow each other behind
// barriers. Skipped tokens neither begin nor end a page, however many lie between two of its
// tokens: both searches look past them, beyond the window only where it holds nothing else (256
// of them cost a load). New tokens stay in registers between the maximum and the rounding (up to 8192
// values; what is beyond is read again). Values are transposed through LDS so that a page's rows
// are written in whole words. Bound by memory for prompts; for single tokens by latency: two
// loads that wait for each other (slots; tokens and scale). A page is rounded anew only where
// its scale grew, a third load that waits for the first two and the bytes of the page, read and
// written. 63 tokens, 8 heads of 128, pages of 64: 6.7 us where no scale grows, 8.7 where all do;
// 8767 float32 tokens in pages of 32 (90 MB): 28 and 30.6 us, 3.2 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(5)))
cache_append_kernel(AppendArgs a) {
    constexpr int KEEP = 4;  // items of 8 values that a thread keeps
    __shared__ uint32_t most_part[4];
    __shared__ int token_at[128];
    __shared__ int window[256];  // slots of tokens c0 - 1 ..: -1 where skipped
    __shared__ int run_token[128];  // the run's tokens (after its first), and their places in the
    __shared__ int run_off[128];    // page
    extern __shared__ __attribute__((aligned(16))) int8_t tile[];  // values: [page_size][W + 4]
    const int tid = threadIdx.x, lane = tid & 63;
    const int h = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const T *x = static_cast<const T *>(a.x[is_v]) + (int64_t)h * a.c.dim;
    const int64_t ld = a.ld[is_v];
    const int P = a.c.page_size, W = a.c.width, D = a.c.dim, d8 = D / 8;
    // item i: eight features from 8 e on of token t of the run
    auto split = [&](int i, int &t, int &e) {
        t = (int)fast_div((uint32_t)i, a.d8);
        e = i - t * d8;
    };
    const int c0 = blockIdx.x * a.chunk;
    window[tid] = slot_at(a, c0 - 1 + tid);  // (chunk <= 64 and a page's 128 tokens: 193 without
    __syncthreads();                         // skipped ones)
    // which tokens of the chunk begin a page: those whose last token before that is not skipped
    // is in another one, or is not there (every wavefront finds the same; -1 has the page -1)
    const int its = lane < a.chunk ? window[lane + 1] : -1;
    const uint64_t held = __ballot(its >= 0);
    if (held == 0) return;
    const uint64_t before = held & ((1ull << lane) - 1);
    int prior = window[0];
    if (prior < 0) prior = last_slot(a, c0 - 1);
    if (before != 0) prior = window[64 - __builtin_clzll(before)];
    uint64_t todo = __ballot(its >= 0 && prior >> a.shift != its >> a.shift);
#pragma unroll 1
    while (todo != 0) {
        const int at = __builtin_ctzll(todo) + 1;  // the page's first token in the window
        todo &= todo - 1;
        const int t0 = c0 + at - 1;
        const int page = window[at] >> a.shift;
        const int64_t ph = (int64_t)page * a.c.heads + h;
        float *scale = (is_v ? a.c.value_scales : a.c.key_scales) + ph;
        const float was = *scale;
        // the run: the tokens from t0 on, past skipped ones, until one is in another page; at
        // most as many as the page holds (every wavefront finds the same)
        int n = 0;
        bool fresh = false, dense = true;  // dense: neighbours
#pragma unroll 1
        for (int base = at;;) {
            const int i = base + lane;
            const int slot = base + 63 < 256 ? window[i] : slot_at(a, c0 - 1 + i);
            const uint64_t in = __ballot(slot >= 0 && slot >> a.shift == page);
            const uint64_t other = __ballot(slot >= 0 && slot >> a.shift != page);
            const uint64_t run = other == 0 ? in : in & ((other & -other) - 1);
            const int place = n + __builtin_popcountll(run & ((1ull << lane) - 1));
            const bool here = (run >> lane & 1) != 0 && place < P;
            const int off = slot & (P - 1);
            if (here && tid < 64) {
                run_token[place] = i - at;
                run_off[place] = off;
            }
            fresh = fresh || __ballot(here && off == 0) != 0;
            dense = dense && __ballot(here && place != i - at) == 0;
            n = min(n + __builtin_popcountll(run), P);
            base += 64;
            if (other != 0 || n == P || c0 - 1 + base >= a.tokens) break;
            if (base + 63 >= 256) {
                const int t = next_token(a, c0 - 1 + base);
                if (t >= a.tokens) break;
                base = t - (c0 - 1);
            }
        }
        const int items = n * d8;
        // the first items' tokens (past the run: its first item again, so that no register of
        // the loads depends on a branch)
        int from[KEEP], feature[KEEP];
#pragma unroll
        for (int k = 0; k < KEEP; ++k) {
            const int i = tid + 256 * k;
            split(i < items ? i : 0, from[k], feature[k]);
        }
        if (!dense) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < KEEP; ++k) from[k] = run_token[from[k]];
        }
        float v[KEEP][8];
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            load_f32<T, 8>(x + (int64_t)(t0 + from[k]) * ld + feature[k] * 8, 8, v[k]);
        auto token = [&](int t) { return t0 + (dense ? t : run_token[t]); };
        if (tid < P) token_at[tid] = -1;
        uint32_t most = 0;
        auto largest = [&most](const float(&y)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = __float_as_uint(y[j]) & 0x7fffffffu;
                most = b > most ? b : most;
            }
        };
#pragma unroll
        for (int k = 0; k < KEEP; ++k) largest(v[k]);
#pragma unroll 1
        for (int i = tid + 256 * KEEP; i < items; i += 256) {
            int t, e;
            split(i, t, e);
            float y[8];
            load_f32<T, 8>(x + (int64_t)token(t) * ld + e * 8, 8, y);
            largest(y);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint32_t b = __shfl_xor(most, o);
            most = b > most ? b : most;
        }
        if (lane == 0) most_part[tid >> 6] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) most = most_part[w] > most ? most_part[w] : most;
        if (tid < n) atomicMax(&token_at[run_off[tid]], tid);
        const float old = fresh ? 0.0f : was;
        const float mine = scale_of(most);
        // the larger; NaN where either is
        const float now = old != old ? old : (mine != mine || mine > old ? mine : old);
        if (tid == 0) *scale = now;
        int8_t *base = (is_v ? a.c.values : a.c.keys) + ph * P * W;
        if (!fresh && now > old) {  // (not where now is NaN: the bytes hold nothing then)
            const float ratio = old / now;
#pragma unroll 1
            for (int i = tid; i < P * W / 16; i += 256) {
                uint4 q = reinterpret_cast<uint4 *>(base)[i];
                uint32_t *w = reinterpret_cast<uint32_t *>(&q);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t b[4];
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        b[m] = held_byte((float)(int8_t)(w[k] >> (8 * m)), ratio);
                    w[k] = pack4(b[0], b[1], b[2], b[3]);
                }
                reinterpret_cast<uint4 *>(base)[i] = q;
            }
        }
        __syncthreads();
        const float inv = inverse_scale(now);
        auto put = [&](const float(&y)[8], int i) {
            int t, e;
            split(i, t, e);
            const int off = run_off[t];
            if (token_at[off] != t) return;
            uint2 q;
            q.x = pack4(held_byte(y[0], inv), held_byte(y[1], inv), held_byte(y[2], inv),
                        held_byte(y[3], inv));
            q.y = pack4(held_byte(y[4], inv), held_byte(y[5], inv), held_byte(y[6], inv),
                        held_byte(y[7], inv));
            if (!is_v) {
                *reinterpret_cast<uint2 *>(base + off * W + e * 8) = q;
            } else {
                *reinterpret_cast<uint32_t *>(tile + off * (W + 4) + e * 8) = q.x;
                *reinterpret_cast<uint32_t *>(tile + off * (W + 4) + e * 8 + 4) = q.y;
            }
        };
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            if (tid + 256 * k < items) put(v[k], tid + 256 * k);
#pragma unroll 1
        for (int i = tid + 256 * KEEP; i < items; i += 256) {
            int t, e;
            split(i, t, e);
            float y[8];
            load_f32<T, 8>(x + (int64_t)token(t) * ld + e * 8, 8, y);
            put(y, i);
        }
        if (is_v) __syncthreads();
        if (is_v && n == 1) {  // (a single token's bytes lie apart)
            const int off = run_off[0];
#pragma unroll 1
            for (int d = tid; d < D; d += 256) base[(int64_t)d * P + off] = tile[off * (W + 4) + d];
        } else if (is_v) {
            const int groups = P / 4, per = a.shift - 2;  // groups of four neighbouring offsets
#pragma unroll 1
            for (int i = tid; i < D * groups; i += 256) {
                const int d = i >> per, off = (i & (groups - 1)) * 4;
                uint32_t b[4];
                int here = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    b[k] = (uint8_t)tile[(off + k) * (W + 4) + d];
                    here |= (token_at[off + k] >= 0) << k;
                }
                int8_t *out = base + (int64_t)d * P + off;
                if (here == 15)
                    *reinterpret_cast<uint32_t *>(out) = pack4(b[0], b[1], b[2], b[3]);
                else if (here != 0) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (here >> k & 1) out[k] = (int8_t)b[k];
                }
            }
        }
        __syncthreads();
    }
}

// -------------------------------------------------------------------------------- read
// 64 tokens of one head, of K or of V: a thread takes four tokens' eight features at a time.
// Values are read along a page's tokens, four neighbouring slots a load (wherever they begin),
// and turned in registers. Two loads that wait for each other (slots; bytes and scales), then
// 16 bytes or more a store: bound by memory (8972 float32 tokens, 92 MB: 22.8 us, 4.0 TB/s).
// A step's 64 pages of 64 tokens, bfloat16 (25 MB): 8.2 us.
template <typename T>
__global__ void __launch_bounds__(256)
cache_read_kernel(Cache8 c, const int *slots, int tokens, T *K, T *V, int shift) {
    const int tid = threadIdx.x;
    const int h = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int t0 = blockIdx.x * 64 + (tid & 15) * 4;
    if (t0 >= tokens) return;
    const int n = min(4, tokens - t0);
    const int P = c.page_size, W = c.width, D = c.dim;
    // Outside the pool: page 0's bytes, and the scale 0. All loads are made (in branches each
    // would be waited for).
    int64_t at[4];
    float scale[4];
    int slot[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) slot[j] = slots[min(t0 + j, tokens - 1)];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int page = page_of(slot[j], shift, c.pages);
        const int64_t ph = (int64_t)max(page, 0) * c.heads + h;
        const int off = slot[j] & (P - 1);
        at[j] = ph * P * W + (is_v ? off : off * W);
        const float s = (is_v ? c.value_scales : c.key_scales)[ph];
        scale[j] = page < 0 ? 0.f : s;
    }
    const bool four = slot[1] == slot[0] + 1 && slot[2] == slot[0] + 2 &&
                      slot[3] == slot[0] + 3 && (slot[0] & (P - 1)) + 3 < P;
    T *out = (is_v ? V : K) + ((int64_t)t0 * c.heads + h) * D;
    for (int e = (tid >> 4) * 8; e < D; e += 128) {
        uint32_t w[4][2];  // eight bytes of each token
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint2 x = load_any<uint2>(c.keys + at[j] + e);
                w[j][0] = x.x;
                w[j][1] = x.y;
            }
        } else {
            uint32_t f[8];  // four tokens of each feature
            const int8_t *from = c.values + (int64_t)e * P;
            if (four) {
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] = load_any<uint32_t>(from + at[0] + k * P);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    f[k] = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        f[k] |= (uint32_t)(uint8_t)from[at[j] + k * P] << (8 * j);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t *g = f + 4 * half;
                // bytes (0, 0', 1, 1'), (2, 2', 3, 3') of two features, then of four
                const uint32_t a = __builtin_amdgcn_perm(g[1], g[0], 0x05010400u);
                const uint32_t b = __builtin_amdgcn_perm(g[1], g[0], 0x07030602u);
                const uint32_t x = __builtin_amdgcn_perm(g[3], g[2], 0x05010400u);
                const uint32_t y = __builtin_amdgcn_perm(g[3], g[2], 0x07030602u);
                w[0][half] = __builtin_amdgcn_perm(x, a, 0x05040100u);
                w[1][half] = __builtin_amdgcn_perm(x, a, 0x07060302u);
                w[2][half] = __builtin_amdgcn_perm(y, b, 0x05040100u);
                w[3][half] = __builtin_amdgcn_perm(y, b, 0x07060302u);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            struct {
                T t[8];
            } r;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                r.t[k] =
                    from_f32<T>((float)(int8_t)(w[j][k / 4] >> (8 * (k & 3))) * scale[j]);
            if (j < n) store_any(out + (int64_t)j * c.heads * D + e, r);
        }
    }
}

int shift_of(int page_size) { return __builtin_ctz((unsigned)page_size); }
}  // namespace

int launch_cache_tables(hipStream_t stream, const TablesArgs &a) {
    const unsigned blocks = a.tokens > 0 ? (unsigned)((a.tokens + TW - 1) / TW) : 1u;
    const int shift = shift_of(a.page_size);
    if (a.free_pages != nullptr)
        MIGEMM_LAUNCH((cache_tables_kernel<true>), dim3(blocks), dim3(TW), 0, stream, a, shift);
    else
        MIGEMM_LAUNCH((cache_tables_kernel<false>), dim3(blocks), dim3(TW), 0, stream, a, shift);
    return launch_status("cache_tables_kernel launch");
}

int launch_cache_release(hipStream_t stream, const int *finished, int *lengths, int requests,
                         int *table, int max_pages, int page_size, int *free_pages, int pages,
                         int *free_count) {
    MIGEMM_LAUNCH(cache_release_kernel, dim3(1), dim3(TW), 0, stream, finished, lengths,
                  requests, table, max_pages, shift_of(page_size), free_pages, pages,
                  free_count);
    return launch_status("cache_release_kernel launch");
}

int launch_cache_append(hipStream_t stream, const void *K, const void *V, int type,
                        int64_t ldk, int64_t ldv, const int *slots, int tokens,
                        const Cache8 &c) {
    AppendArgs a{};
    a.x[0] = K;
    a.x[1] = V;
    a.ld[0] = ldk;
    a.ld[1] = ldv;
    a.slots = slots;
    a.tokens = tokens;
    a.c = c;
    a.shift = shift_of(c.page_size);
    a.d8 = make_fastdiv((uint32_t)c.dim / 8);
    // work-groups for each CU several times over before one takes more than one page's tokens
    const int64_t want = (int64_t)tokens * c.heads * 2 / 2048;
    a.chunk = 1;
    while (a.chunk < 64 && a.chunk < c.page_size && a.chunk < want) a.chunk *= 2;
    const dim3 grid((tokens + a.chunk - 1) / a.chunk, c.heads, 2);
    const size_t lds = (size_t)c.page_size * (c.width + 4);
    if (type == MIGEMM_FLOAT32)
        MIGEMM_LAUNCH((cache_append_kernel<float>), grid, dim3(256), lds, stream, a);
    else
        MIGEMM_LAUNCH((cache_append_kernel<Bf16>), grid, dim3(256), lds, stream, a);
    return launch_status("cache_append_kernel launch");
}

int launch_cache_read(hipStream_t stream, const Cache8 &c, const int *slots, int tokens,
                      void *K, void *V, int type) {
    const dim3 grid((tokens + 63) / 64, c.heads, 2);
    const int shift = shift_of(c.page_size);
    if (type == MIGEMM_FLOAT32)
        MIGEMM_LAUNCH((cache_read_kernel<float>), grid, dim3(256), 0, stream, c, slots, tokens,
                      static_cast<float *>(K), static_cast<float *>(V), shift);
    else
        MIGEMM_LAUNCH((cache_read_kernel<Bf16>), grid, dim3(256), 0, stream, c, slots, tokens,
                      static_cast<Bf16 *>(K), static_cast<Bf16 *>(V), shift);
    return launch_status("cache_read_kernel launch");
}

}  // namespace migemm
