// A token for each row of logits: temperature, min-p, top-k, top-p, and a given random number.
//
// Tokens are ordered by logit, largest first, equal ones by index. A token's weight is w =
// exp((l - top) / T), 0 where w < min_p, 0 beyond the first top_k; of the others the fewest are
// kept that hold top_p of their sum, and the token is the first whose weights up to its own are
// more than u times the kept ones' sum. So every step asks one question: where in the order does a
// running count or sum cross a value? It is answered without sorting the row:
//
//   * A histogram of the row, in bins of equal width in (top - l), a monotone function of the logit
//     in float32. Its running sums name the bin that a value falls in. With top_k it holds counts
//     (the few tokens that are left get their weights later), otherwise weights.
//   * The tokens of that bin, or of all bins up to it where they are few, are collected into LDS
//     and sorted there by logit and index; the running sums over them name the token. A bin of more
//     tokens than the list holds (equal logits, mostly) is cut again by bits of logit and index
//     until few are left.
//
// Weights come from 64-bit arithmetic, because a sum of 10^5 float32 weights is off by more than a
// token's share, and are summed as integers: exactly, in any order (atomics among them), so that a
// result does not depend on how a row was walked. Within a bin's width of at most 0.023 in log2 w
// a token's weight over its bin's middle one is a polynomial of degree 5 (off by 2^-50); these are
// summed with 43 fractional bits, and a bin's sum is multiplied by its middle weight once, to 42 bits
// below the point or more (62 - log2(vocabulary), at most 46). Tokens that weigh less than half of
// the last bit are left out.
//
#include "int8_common.h"

namespace migemm {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2 * kThreads;
constexpr int kList = 2 * kThreads;
constexpr int kWhole = 512;     // all bins up to the one in question are sorted together up to here
constexpr int kIndexBits = 20;  // of a token, below the bits of its logit in an order's key
constexpr int kFraction = 43;   // bits of a weight over its bin's middle one (2^20 of them fit)
constexpr double kOne = (double)((u64)1 << kFraction);
constexpr float kMost = 3.402823466e38f;

struct Shared {
    u64 mass[kBins];        // running weight (or count) over the row's bins
    uint32_t count[kBins];  // running number of tokens, or a bound of it
    union {
        struct {
            u64 list[kList], upto[kList];  // keys in order, and the running weight over them
        };
        struct {
            u64 part_mass[kBins];  // the same over the parts of a bin
            uint32_t part_count[kBins];
        };
    };
    u64 wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float high[kWaves], low[kWaves];
    int bad;
    uint32_t listed, found;
};

// Ascending keys: largest logit first, then lowest index.
__device__ __forceinline__ uint32_t order_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);  // (-0 as 0)
    return b & 0x80000000u ? b : b ^ 0x7fffffffu;
}
__device__ __forceinline__ float logit_of(u64 key) {
    const uint32_t order = (uint32_t)(key >> kIndexBits);
    return __uint_as_float(order & 0x80000000u ? order : order ^ 0x7fffffffu);
}
__device__ __forceinline__ u64 key_of(float l, uint32_t index) {
    return (u64)order_of(l) << kIndexBits | index;
}
// inf counts as the largest number.
__device__ __forceinline__ float bounded(float l) {
    return __builtin_amdgcn_fmed3f(l, -INFINITY, kMost);
}

// 2^x for x > -1000. 2^f for |f| <= 1/2 is 1 + f q(f), q of degree 9 through the Chebyshev nodes of
// (2^f - 1) / f: off by 2^-50.
__device__ __forceinline__ double power(double x) {
    const double t = x + 6755399441055744.0;  // (1.5 2^52: rounds x, its low bits are the integer)
    const double f = x - (t - 6755399441055744.0);
    double q = 7.070978550292061e-09;
    q = __builtin_fma(q, f, 1.0205905583190955e-07);
    q = __builtin_fma(q, f, 1.3215451631397446e-06);
    q = __builtin_fma(q, f, 1.5252672924085807e-05);
    q = __builtin_fma(q, f, 0.00015403530424773178);
    q = __builtin_fma(q, f, 0.0013333558200795622);
    q = __builtin_fma(q, f, 0.009618129107618677);
    q = __builtin_fma(q, f, 0.05550410866465167);
    q = __builtin_fma(q, f, 0.24022650695910075);
    q = __builtin_fma(q, f, 0.6931471805599462);
    q = __builtin_fma(q, f, 1.0);
    return __longlong_as_double(
        (long long)((u64)__double_as_longlong(q) + ((u64)__double_as_longlong(t) << 52)));
}
// A number in [0, 2^52) rounded to an integer, in the adder.
__device__ __forceinline__ u64 rounded(double x, double unit) {
    const double y = __builtin_fma(x, unit, 4503599627370496.0);
    return (u64)__double_as_longlong(y) & (((u64)1 << 52) - 1);
}

// What a row's logits weigh, and its bins.
struct Weights {
    float scale, top;  // the largest logit times the scale
    float bins;        // bins a unit of (top - l) scale
    double top64;
    double rate;     // log2(e) / T
    double width;    // of a bin, in log2 of the weight
    double cut;      // l - top below which a token weighs nothing
    float least;     // the smallest logit that is not below it
    double unit;     // 2^bits

    __device__ __forceinline__ void init(const SampleArgs &p, float high, float low,
                                         float temperature, float min_p) {
        top64 = high;
        rate = 1.4426950408889634074 / (double)temperature;
        unit = p.unit;
        // bins over the logits that weigh something, or over all of them where that is less
        const double spread = top64 - (double)low;
        double span = (double)(p.bits + 1) / rate;
        span = spread < span ? spread : span;
        cut = -span;
        if (min_p > 0.f) {
            const double least = min_p < 1.f ? log2((double)min_p) / rate : 0.0;
            cut = least > cut ? least : cut;
        }
        // (the float32 coordinate of a token at the cut stays below kBins - 1)
        double per = span > 0.0 ? (kBins - 2) / span : 0.0;
        // Halves, so that the difference of the largest numbers is one too. Spans that are too
        // small for float32's range of bins a unit: logits that are small as well are scaled up,
        // larger ones have no neighbour within such a span.
        scale = 0.5f;
        if (per > 1e30) {
            if (fabsf(high) < 1.f)
                scale = 0x1p100f;
            else
                per = 0.0;
        }
        top = high * scale;
        bins = (float)(per / (double)scale);
        width = bins > 0.f ? rate / ((double)bins * (double)scale) : 0.0;
        least = smallest(kBins - 1);
    }
    // The smallest logit of bins 0 .. b, by all lanes of a wavefront: bin and cut go by the order
    // of logits, so 64 of them at a time narrow it down.
    __device__ __forceinline__ float smallest(uint32_t b) const {
        uint32_t lo = order_of((float)top64), hi = order_of(-kMost);
        while (hi > lo) {
            const uint32_t step = (hi - lo) / 64 + 1;
            const u64 at = lo + (u64)step * (threadIdx.x & 63);
            const float l = logit_of((at < hi ? at : hi) << kIndexBits);
            const int in = __popcll(__ballot(at <= hi && bin(l) <= b && below(l) >= cut));
            lo += step * (in - 1);
            hi = (u64)lo + step - 1 < hi ? lo + step - 1 : hi;
        }
        return logit_of((u64)lo << kIndexBits);
    }
    __device__ __forceinline__ double below(float l) const { return (double)l - top64; }
    // (two roundings, each of which keeps the order)
    __device__ __forceinline__ uint32_t bin(float l) const {
        return (uint32_t)fminf(__builtin_fmaf(-scale, l, top) * bins, (float)(kBins - 1));
    }
    // 2^(log2 w + width (b + 1/2)) with kFraction bits: the weight over the middle one of its bin
    __device__ __forceinline__ u64 over_middle(double d, uint32_t b) const {
        const double f = __builtin_fma(d, rate, __builtin_fma((double)b, width, 0.5 * width));
        double q = 0.0013333558146428443;  // ln2^k / k!
        q = __builtin_fma(q, f, 0.009618129107628477);
        q = __builtin_fma(q, f, 0.05550410866482158);
        q = __builtin_fma(q, f, 0.24022650695910072);
        q = __builtin_fma(q, f, 0.6931471805599453);
        q = __builtin_fma(q, f, 1.0);
        return rounded(q, kOne);
    }
    __device__ __forceinline__ double middle(int b) const {
        return power(-width * ((double)b + 0.5));
    }
    __device__ __forceinline__ double share(float l) const {
        const double y = below(l) * rate;
        return y > -64.0 ? power(y) : 0.0;
    }
    __device__ __forceinline__ u64 mass(float l) const { return rounded(share(l), unit); }
};

// What a row asks for.
struct Asked {
    float temperature, top_p, min_p, uniform;
    int top_k;
    bool valid;

    __device__ __forceinline__ Asked(const SampleArgs &p, int r) {
        temperature = p.temperatures != nullptr ? p.temperatures[r] : p.temperature;
        top_k = p.top_ks != nullptr ? p.top_ks[r] : p.top_k;
        top_p = p.top_ps != nullptr ? p.top_ps[r] : p.top_p;
        min_p = p.min_ps != nullptr ? p.min_ps[r] : p.min_p;
        uniform = p.uniforms[r];
        valid = temperature >= 0.f && temperature < INFINITY && top_p == top_p &&
                min_p == min_p && uniform == uniform;
    }
    __device__ __forceinline__ bool wide() const { return temperature > 2.f; }
    __device__ __forceinline__ bool greedy() const { return temperature == 0.f || top_k == 1; }
    // Whether the row's histogram holds numbers: top-k comes first.
    __device__ __forceinline__ bool counted(int n) const { return top_k > 0 && top_k < n; }
    // The running weight that ends the tokens that top-p keeps of a sum, and the one to draw.
    __device__ __forceinline__ u64 kept(u64 total) const {
        const u64 t = (u64)ceil((double)fmaxf(top_p, 0.f) * (double)total);
        return t < 1 ? 1 : t > total ? total : t;
    }
    __device__ __forceinline__ u64 drawn(u64 total) const {
        const double u = uniform < 0.f ? 0.0 : uniform > 1.f ? 1.0 : (double)uniform;
        const u64 t = (u64)(u * (double)total) + 1;
        return t > total ? total : t;
    }
};

// Calls f(logit, index) for the logits first .. end of a row, those of a thread in ascending order.
template <int THREADS, typename T, typename F>
__device__ __forceinline__ void each(const T *row, int first, int end, const F &f) {
    constexpr int V = 16 / sizeof(T), U = sizeof(T) == 4 ? 4 : 2;
    for (int part = first; part < end; part += THREADS * V * U) {
        const int at = part + threadIdx.x * V;
        float x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u)
            load_f32<T, V>(row + at + u * THREADS * V, end - at - u * THREADS * V, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = at + u * THREADS * V + e;
                if (i < end) f(x[u][e], i);
            }
    }
}

// The largest logit of a range and whether one is NaN, in every lane, and with `wide` the smallest
// above -inf (otherwise it is -inf). At low temperatures the logits that weigh something span
// less than all of them, so the smallest does not matter, and costs half of the pass.
template <int THREADS, typename T>
__device__ __forceinline__ void extremes(const T *row, int first, int end, bool wide, float &high,
                                         float &low, bool &nan) {
    high = -INFINITY;
    low = wide ? INFINITY : -INFINITY;
    nan = false;
    if (wide)
        each<THREADS>(row, first, end, [&](float x, int) {
            nan |= x != x;
            high = fmaxf(high, x);
            low = x > -INFINITY ? fminf(low, x) : low;
        });
    else
        each<THREADS>(row, first, end, [&](float x, int) {
            nan |= x != x;
            high = fmaxf(high, x);
        });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        high = fmaxf(high, __shfl_xor(high, o));
        low = fminf(low, __shfl_xor(low, o));
    }
    high = bounded(high);
    low = fminf(low, kMost);
    nan = __ballot(nan) != 0;
}

// The tokens first .. end into the histogram: their weights, or with COUNT their number. Keys past
// `limit` are left out.
template <bool COUNT, typename T>
__device__ __forceinline__ void fill(u64 *mass, const T *row, int first, int end, const Weights &w,
                                     u64 limit) {
    each<kThreads>(row, first, end, [&](float x, int i) {
        if (!(x >= w.least)) return;
        const float l = bounded(x);
        if (limit != ~(u64)0 && key_of(l, i) > limit) return;
        const uint32_t b = w.bin(l);
        atomicAdd(&mass[b], COUNT ? (u64)1 : w.over_middle(w.below(l), b));
    });
}

// Running sums over a wavefront's lanes (within rows of 16, then over the rows).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 x) {
    return (u64)moved<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)x);
}
template <typename N>
__device__ __forceinline__ N run_up_lanes(N x) {
    x += moved<0x111, 0xf>(x);
    x += moved<0x112, 0xf>(x);
    x += moved<0x114, 0xf>(x);
    x += moved<0x118, 0xf>(x);
    x += moved<0x142, 0xa>(x);
    x += moved<0x143, 0xc>(x);
    return x;
}

// Running sums of 2 * kThreads masses (and counts), in place. Ends with a barrier.
template <bool COUNTS>
__device__ __forceinline__ void run_up(Shared &s, u64 *mass, uint32_t *count) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64 m1 = mass[2 * tid + 1];
    u64 m = run_up_lanes(mass[2 * tid] + m1);
    uint32_t c = 0, c1 = 0;
    if (COUNTS) {
        c1 = count[2 * tid + 1];
        c = run_up_lanes(count[2 * tid] + c1);
    }
    if (lane == 63) {
        s.wave_mass[wave] = m;
        s.wave_count[wave] = c;
    }
    __syncthreads();
    // the sums of the wavefronts before: each lane of a row of 16 takes one
    const u64 wm = run_up_lanes(lane < wave ? s.wave_mass[lane & (kWaves - 1)] : 0);
    m += __shfl(wm, kWaves - 1);
    if (COUNTS) {
        const uint32_t wc = run_up_lanes(lane < wave ? s.wave_count[lane & (kWaves - 1)] : 0);
        c += __shfl(wc, kWaves - 1);
    }
    mass[2 * tid] = m - m1;
    mass[2 * tid + 1] = m;
    if (COUNTS) {
        count[2 * tid] = c - c1;
        count[2 * tid + 1] = c;
    }
    __syncthreads();
}

// A filled histogram becomes its running sums. A bin's weight is its sum times its middle one; its
// number of tokens is at most the sum over the least that a token adds to it (2^-0.012).
template <bool COUNT>
__device__ __forceinline__ void finish(Shared &s, const Weights &w) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        const u64 m = s.mass[b];
        if (COUNT) {
            s.count[b] = (uint32_t)m;
        } else {
            s.count[b] = m ? (uint32_t)((double)m * (1.01 / kOne)) + 1 : 0;
            s.mass[b] = m ? (u64)((double)m * (w.middle(b) * (w.unit / kOne)) + 0.5) : 0;
        }
    }
    __syncthreads();
    run_up<true>(s, s.mass, s.count);
}

// The first place whose running sum reaches target (the last one's does, or the last is returned).
template <typename N>
__device__ __forceinline__ int reach(Shared &s, const N *sums, int n, N target) {
    const N last = sums[n - 1];
    target = target < last ? target : last;
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (sums[i] >= target && (i == 0 || sums[i - 1] < target)) s.found = i;
    __syncthreads();
    const int i = s.found;
    __syncthreads();
    return i;
}

// Sorts the first `size` (a power of two, at least 2) keys of the list. A wavefront's threads
// exchange within its own 128 keys while their distance is at most 64: those steps need no barrier.
__device__ __forceinline__ void sort(Shared &s, int size) {
    const int tid = threadIdx.x;
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            if (j > 64) __syncthreads();
            if (tid < size / 2) {
                const int x = 2 * tid - (tid & (j - 1)), y = x + j;
                const u64 p = s.list[x], q = s.list[y];
                if ((p > q) == ((x & k) == 0)) {
                    s.list[x] = q;
                    s.list[y] = p;
                }
            }
            if (j > 64)
                __syncthreads();
            else
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    __syncthreads();
}

// Bins whose tokens a row's answer may need, as far as the histogram tells: all up to one of them,
// or single ones. `listed`: they are few enough for a list.
struct Plan {
    bool whole, listed;
    int kept, first, last;  // the bin where top-k or top-p ends (-1: none does), those to draw from

    __device__ __forceinline__ bool has(int b) const {
        return whole ? b <= kept : b == kept || (first <= b && b <= last);
    }
};

// Of the tokens of bins a .. b.
__device__ __forceinline__ uint32_t count_in(const Shared &s, int a, int b) {
    return s.count[b] - (a ? s.count[a - 1] : 0);
}

__device__ __forceinline__ Plan plan_of(Shared &s, const Asked &q, bool counted) {
    Plan g{true, true, kBins - 1, 0, -1};
    const u64 total = s.mass[kBins - 1];
    if (counted) {
        g.kept = reach(s, s.mass, kBins, (u64)q.top_k);
        g.listed = s.count[g.kept] <= kList;
        return g;
    }
    u64 low = total, high = total;
    if (q.top_p < 1.f) {
        g.kept = reach(s, s.mass, kBins, q.kept(total));
        low = g.kept ? s.mass[g.kept - 1] : 1;
        high = s.mass[g.kept];
    }
    if (s.count[g.kept] <= kWhole) return g;
    g.whole = false;
    g.first = reach(s, s.mass, kBins, q.drawn(low));
    g.last = reach(s, s.mass, kBins, q.drawn(high));
    uint32_t n = count_in(s, g.first, g.last);
    if (q.top_p < 1.f) {
        if (g.kept > g.last) n += count_in(s, g.kept, g.kept);
    } else {
        g.kept = -1;
    }
    g.listed = n <= kList;
    return g;
}

// A row and what is known of it. Its tokens come from its logits, or (given) from keys that an
// earlier kernel gathered. The list holds those of bins first .. last.
template <typename T>
struct Row {
    Shared &s;
    const T *logits;
    int n;
    const u64 *given;
    int gathered;
    Weights w;
    u64 limit;   // keys past it are out (top-k)
    bool whole;  // the list holds all tokens that may be kept
    int first, last;
    u64 base;    // what runs up to the list

    // The tokens of bins a .. b with keys lo .. hi (at most kList), sorted, and their running weights.
    __device__ __forceinline__ void collect(int a, int b, u64 lo, u64 hi) {
        const int tid = threadIdx.x;
        hi = hi < limit ? hi : limit;
        if (tid == 0) s.listed = 0;
        __syncthreads();
        const auto take = [&](u64 key) {
            if (key < lo || key > hi) return;
            const uint32_t place = atomicAdd(&s.listed, 1u);
            if (place < kList) s.list[place] = key;
        };
        if (given != nullptr) {
            for (int i = tid; i < gathered; i += kThreads) {
                const int at = (int)w.bin(logit_of(given[i]));
                if (at >= a && at <= b) take(given[i]);
            }
        } else {
            const float from = w.smallest(b);
            const float below = a ? w.smallest(a - 1) : INFINITY;
            each<kThreads>(logits, 0, n, [&](float x, int i) {
                if (x >= from && (x < below || a == 0)) take(key_of(bounded(x), i));
            });
        }
        __syncthreads();
        const int found = min((int)s.listed, kList);
        int size = 2;
        while (size < found) size *= 2;
        for (int i = tid; i < kList; i += kThreads)
            if (i >= found) s.list[i] = ~(u64)0;
        __syncthreads();
        sort(s, size);
        for (int i = tid; i < kList; i += kThreads)
            s.upto[i] = i < found ? w.mass(logit_of(s.list[i])) : 0;
        __syncthreads();
        run_up<false>(s, s.upto, nullptr);
    }

    __device__ __forceinline__ void collect_up_to(int b) {
        whole = true;
        base = 0;
        collect(0, b, 0, ~(u64)0);
    }

    // The list comes to hold the token of bin b whose running weight (COUNT: number) reaches target.
    template <bool COUNT>
    __device__ __forceinline__ void hold(int b, u64 target) {
        if (first <= b && b <= last) return;
        base = b ? s.mass[b - 1] : 0;
        uint32_t left = count_in(s, b, b);
        u64 lo = 0, hi = ((u64)1 << (32 + kIndexBits)) - 1;
        first = last = b;
        while (left > kList) {  // cut by the keys' bits; a range of one key holds one token
            first = 1;
            last = 0;  // (not the whole bin: for this target alone)
            const int bits = 64 - __clzll(hi - lo);
            const int shift = bits > 11 ? bits - 11 : 0;
            for (int i = threadIdx.x; i < kBins; i += kThreads) {
                s.part_count[i] = 0;
                s.part_mass[i] = 0;
            }
            __syncthreads();
            each<kThreads>(logits, 0, n, [&](float x, int i) {
                const float l = bounded(x);
                if ((int)w.bin(l) != b || !(l >= w.least)) return;
                const u64 key = key_of(l, i);
                if (key < lo || key > hi || key > limit) return;
                const int at = (int)((key - lo) >> shift);
                atomicAdd(&s.part_count[at], 1u);
                if (!COUNT) atomicAdd(&s.part_mass[at], w.mass(l));
            });
            __syncthreads();
            if (COUNT) {
                for (int i = threadIdx.x; i < kBins; i += kThreads)
                    s.part_mass[i] = s.part_count[i];
                __syncthreads();
            }
            run_up<true>(s, s.part_mass, s.part_count);
            const int at = reach(s, s.part_mass, kBins, target - base);
            left = count_parts(at);
            base += at ? s.part_mass[at - 1] : 0;
            lo += (u64)at << shift;
            const u64 end = lo + (((u64)1 << shift) - 1);
            hi = end < hi ? end : hi;
            __syncthreads();
        }
        collect(b, b, lo, hi);
    }
    __device__ __forceinline__ uint32_t count_parts(int at) const {
        return s.part_count[at] - (at ? s.part_count[at - 1] : 0);
    }

    // The place in the list of the token whose running weight reaches target.
    __device__ __forceinline__ int by_mass(u64 target) {
        hold<false>(reach(s, s.mass, kBins, target), target);
        return reach(s, s.upto, kList, target - base);
    }

    // The row's token, from its histogram's running sums.
    __device__ __forceinline__ void answer(const SampleArgs &p, int r, const Asked &q, bool counted,
                                           const Plan &plan) {
        u64 total = s.mass[kBins - 1];
        if (counted) {
            const u64 k = (u64)q.top_k < total ? (u64)q.top_k : total;
            if (plan.listed) {
                collect_up_to(plan.kept);
                total = s.upto[k - 1];
            } else {  // so many that their weights need a histogram too
                hold<true>(plan.kept, k);
                limit = s.list[k - base - 1];
                __syncthreads();
                for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0;
                __syncthreads();
                fill<false>(s.mass, logits, 0, n, w, limit);
                __syncthreads();
                finish<false>(s, w);
                total = s.mass[kBins - 1];
                first = 1;
                last = 0;  // (its list went by numbers)
            }
        } else if (plan.whole) {
            collect_up_to(plan.kept);
        }
        if (whole) {
            if (q.top_p < 1.f)
                total = s.upto[reach(s, s.upto, kList, q.kept(total))];
            else if (!counted)
                total = s.upto[kList - 1];
        } else if (q.top_p < 1.f) {
            const u64 target = q.kept(total);
            const u64 most = s.mass[reach(s, s.mass, kBins, target)];
            const int i = by_mass(target);
            // (roundings of the bin's weight and of its tokens' must not reach into the next bin)
            total = base + s.upto[i] < most ? base + s.upto[i] : most;
        }
        const u64 target = q.drawn(total);
        const int i = whole ? reach(s, s.upto, kList, target) : by_mass(target);
        if (threadIdx.x == 0) {
            const u64 key = s.list[i];
            p.tokens[r] = (int)(key & (((u64)1 << kIndexBits) - 1));
            p.probabilities[r] = (float)(w.share(logit_of(key)) * p.unit / (double)total);
        }
    }
};

__device__ __forceinline__ void nothing(const SampleArgs &p, int r) {
    if (threadIdx.x == 0) {
        p.tokens[r] = -1;
        p.probabilities[r] = 0.f;
    }
}

// ------------------------------------------------------------- a row in one work-group
template <typename T>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4)))
sample_row_kernel(SampleArgs p) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x, n = p.vocab;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const Asked q(p, r);
    float high, low;
    bool nan;
    if (tid == 0) {
        s.bad = 0;
        s.found = n;
    }
    extremes<kThreads>(logits, 0, n, q.wide(), high, low, nan);
    if (lane == 0) {
        s.high[wave] = high;
        s.low[wave] = low;
    }
    for (int i = tid; i < kBins; i += kThreads) s.mass[i] = 0;
    __syncthreads();
    if (nan) s.bad = 1;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
        high = fmaxf(high, s.high[w]);
        low = fminf(low, s.low[w]);
    }
    if (!q.valid || s.bad || !(high > -INFINITY)) return nothing(p, r);
    if (q.greedy()) {
        uint32_t best = n;
        each<kThreads>(logits, 0, n, [&](float x, int i) {
            best = bounded(x) == high && (uint32_t)i < best ? i : best;
        });
        if (best < (uint32_t)n) atomicMin(&s.found, best);
        __syncthreads();
        if (tid == 0) {
            p.tokens[r] = (int)s.found;
            p.probabilities[r] = 1.f;
        }
        return;
    }
    Weights w;
    w.init(p, high, low, q.temperature, q.min_p);
    const bool counted = q.counted(n);
    if (counted)
        fill<true>(s.mass, logits, 0, n, w, ~(u64)0);
    else
        fill<false>(s.mass, logits, 0, n, w, ~(u64)0);
    __syncthreads();
    if (counted)
        finish<true>(s, w);
    else
        finish<false>(s, w);
    Row<T> row{s, logits, n, nullptr, 0, w, ~(u64)0, false, 1, 0, 0};
    row.answer(p, r, q, counted, plan_of(s, q, counted));
}
// ------------------------------------------------------------- rows cut over work-groups
// Four launches: the largest logit of each part of a row; the parts' histograms, added up; the tokens
// of the bins that the answer may need; and the answer, from the histogram and those tokens. Each
// work-group of the last two reads the whole histogram and plans the same. A row that the list does
// not hold is walked by the last kernel's work-group alone.
struct SplitArgs {
    SampleArgs p;
    int splits, chunk;  // parts of a row, tokens of a part
    u64 *mass;          // [rows][kBins]
    u64 *list;          // [rows][kList]
    float4 *parts;      // [rows][splits]: largest, smallest, whether one is NaN
    uint32_t *listed;   // [rows]
    uint32_t *best;     // [rows]: where the largest logit stands first
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_top_kernel(SplitArgs a) {
    __shared__ float highs[kWaves], lows[kWaves];
    __shared__ int bad;
    const SampleArgs &p = a.p;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    for (int i = part * kThreads + tid; i < kBins; i += a.splits * kThreads)
        a.mass[(int64_t)r * kBins + i] = 0;
    if (part == 0 && tid == 0) {
        a.listed[r] = 0;
        a.best[r] = ~0u;
    }
    if (tid == 0) bad = 0;
    const int first = part * a.chunk, end = min(first + a.chunk, p.vocab);
    float high, low;
    bool nan;
    extremes<kThreads>(logits, first, end, Asked(p, r).wide(), high, low, nan);
    if ((tid & 63) == 0) {
        highs[tid >> 6] = high;
        lows[tid >> 6] = low;
    }
    __syncthreads();
    if (nan) bad = 1;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kWaves; ++w) {
            high = fmaxf(high, highs[w]);
            low = fminf(low, lows[w]);
        }
        a.parts[(int64_t)r * a.splits + part] = make_float4(high, low, bad ? 1.f : 0.f, 0.f);
    }
}

// A row's extremes from its parts', in every lane; false where there is nothing to choose from.
__device__ __forceinline__ bool joined(const SplitArgs &a, int r, const Asked &q, float &high,
                                       float &low) {
    const int lane = threadIdx.x & 63;
    float4 x = make_float4(-INFINITY, INFINITY, 0.f, 0.f);
    if (lane < a.splits) x = a.parts[(int64_t)r * a.splits + lane];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        x.x = fmaxf(x.x, __shfl_xor(x.x, o));
        x.y = fminf(x.y, __shfl_xor(x.y, o));
    }
    high = x.x;
    low = x.y;
    return q.valid && __ballot(x.z != 0.f) == 0 && high > -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_bins_kernel(SplitArgs a) {
    __shared__ u64 mass[kBins];
    const SampleArgs &p = a.p;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const Asked q(p, r);
    float high, low;
    if (!joined(a, r, q, high, low) || q.greedy()) return;
    Weights w;
    w.init(p, high, low, q.temperature, q.min_p);
    for (int i = tid; i < kBins; i += kThreads) mass[i] = 0;
    __syncthreads();
    const int first = part * a.chunk, end = min(first + a.chunk, p.vocab);
    if (q.counted(p.vocab))
        fill<true>(mass, logits, first, end, w, ~(u64)0);
    else
        fill<false>(mass, logits, first, end, w, ~(u64)0);
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads)
        if (mass[i] != 0) atomicAdd(&a.mass[(int64_t)r * kBins + i], mass[i]);
}

// The running sums of a row's histogram.
__device__ __forceinline__ void load_bins(Shared &s, const SplitArgs &a, int r, const Weights &w,
                                          bool counted) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = a.mass[(int64_t)r * kBins + i];
    if (counted)
        finish<true>(s, w);
    else
        finish<false>(s, w);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_gather_kernel(SplitArgs a) {
    __shared__ Shared s;
    const SampleArgs &p = a.p;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const Asked q(p, r);
    float high, low;
    if (!joined(a, r, q, high, low)) return;
    const int first = part * a.chunk, end = min(first + a.chunk, p.vocab);
    const float mine = a.parts[(int64_t)r * a.splits + part].x;
    if (q.greedy()) {
        if (mine != high) return;
        uint32_t best = ~0u;
        each<kThreads>(logits, first, end, [&](float x, int i) {
            best = bounded(x) == high && (uint32_t)i < best ? i : best;
        });
        if (best != ~0u) atomicMin(&a.best[r], best);
        return;
    }
    Weights w;
    w.init(p, high, low, q.temperature, q.min_p);
    const bool counted = q.counted(p.vocab);
    load_bins(s, a, r, w, counted);
    const Plan plan = plan_of(s, q, counted);
    if (!plan.listed) return;
    // the bins to draw from, and the one where top-p ends, which is not before them
    const int lowest = plan.whole || plan.kept >= plan.last ? plan.kept : plan.last;
    const float from = w.smallest(lowest);
    if (!(mine >= from)) return;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    each<kThreads>(logits, first, end, [&](float x, int i) {
        if (!(x >= from)) return;
        const float l = bounded(x);
        if (!plan.has((int)w.bin(l))) return;
        const uint32_t place = atomicAdd(&s.listed, 1u);
        if (place < kList) s.list[place] = key_of(l, i);
    });
    __syncthreads();
    const uint32_t found = min(s.listed, (uint32_t)kList);
    if (found == 0) return;
    if (tid == 0) s.found = atomicAdd(&a.listed[r], found);
    __syncthreads();
    const uint32_t to = s.found;
    for (uint32_t i = tid; i < found && to + i < kList; i += kThreads)
        a.list[(int64_t)r * kList + to + i] = s.list[i];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_pick_kernel(SplitArgs a) {
    __shared__ Shared s;
    const SampleArgs &p = a.p;
    const int r = blockIdx.x;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const Asked q(p, r);
    float high, low;
    if (!joined(a, r, q, high, low)) return nothing(p, r);
    if (q.greedy()) {
        if (threadIdx.x == 0) {
            p.tokens[r] = (int)a.best[r];
            p.probabilities[r] = 1.f;
        }
        return;
    }
    Weights w;
    w.init(p, high, low, q.temperature, q.min_p);
    const bool counted = q.counted(p.vocab);
    load_bins(s, a, r, w, counted);
    const Plan plan = plan_of(s, q, counted);
    const u64 *given = plan.listed ? a.list + (int64_t)r * kList : nullptr;
    const int gathered = plan.listed ? (int)min(a.listed[r], (uint32_t)kList) : 0;
    Row<T> row{s, logits, p.vocab, given, gathered, w, ~(u64)0, false, 1, 0, 0};
    row.answer(p, r, q, counted, plan);
}

template <typename T>
int launch_split(hipStream_t stream, SplitArgs a) {
    const SampleArgs &p = a.p;
    const size_t row = (kBins + kList) * sizeof(u64) + a.splits * sizeof(float4) + 8;
    int rc = MIGEMM_OK;
    a.mass = static_cast<u64 *>(workspace(stream, p.rows * row, &rc, 0));
    if (a.mass == nullptr) return rc;
    a.list = a.mass + (int64_t)p.rows * kBins;
    a.parts = reinterpret_cast<float4 *>(a.list + (int64_t)p.rows * kList);
    a.listed = reinterpret_cast<uint32_t *>(a.parts + (int64_t)p.rows * a.splits);
    a.best = a.listed + p.rows;
    const dim3 grid(a.splits, p.rows), block(kThreads);
    MIGEMM_LAUNCH((sample_top_kernel<T>), grid, block, 0, stream, a);
    MIGEMM_LAUNCH((sample_bins_kernel<T>), grid, block, 0, stream, a);
    MIGEMM_LAUNCH((sample_gather_kernel<T>), grid, block, 0, stream, a);
    MIGEMM_LAUNCH((sample_pick_kernel<T>), dim3(p.rows), block, 0, stream, a);
    return launch_status("sample_pick_kernel launch");
}

template <typename T>
int launch(hipStream_t stream, const SampleArgs &p) {
    SplitArgs a{};
    a.p = p;
    const int most = p.vocab / 4096 < 64 ? p.vocab / 4096 : 64;
    a.splits = 512 / p.rows < most ? 512 / p.rows : most;
    if (a.splits >= 2) {
        // (whole vectors: a part begins at a multiple of 8 tokens)
        a.chunk = ((p.vocab + a.splits - 1) / a.splits + 7) / 8 * 8;
        a.splits = (p.vocab + a.chunk - 1) / a.chunk;
        return launch_split<T>(stream, a);
    }
    MIGEMM_LAUNCH((sample_row_kernel<T>), dim3(p.rows), dim3(kThreads), 0, stream, p);
    return launch_status("sample_row_kernel launch");
}
}  // namespace

int launch_sample(hipStream_t stream, const SampleArgs &a) {
    SampleArgs p = a;
    int log2 = 0;
    while (((int64_t)1 << log2) < p.vocab) ++log2;
    p.bits = 62 - log2 < 46 ? 62 - log2 : 46;
    p.unit = (double)((uint64_t)1 << p.bits);
    return p.type == MIGEMM_FLOAT32 ? launch<float>(stream, p) : launch<Bf16>(stream, p);
}

}  // namespace migemm
