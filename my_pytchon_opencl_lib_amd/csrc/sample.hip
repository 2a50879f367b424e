// A token for each row of logits: temperature, min-p, top-k, top-p, and a given random number.
//
// Tokens are ordered by logit, largest first, equal ones by index. A token's weight is w =
// exp((l - max) / T), 0 where w < min_p, 0 beyond the first top_k; of the others the fewest are
// kept that hold top_p of their sum, and the token is the first whose weights up to its own are
// more than u times the kept ones' sum. So every step asks one question: where in the order does a
// running count or sum cross a value? It is answered without sorting the row.
//
//   * Weights are integers, rint(w 2^bits): sums are exact, in any order (atomics among them), and
//     a result never depends on how the row was walked. w itself comes from 64-bit arithmetic (its
//     logarithm is exact, the power off by 2^-50), because a sum of 10^5 float32 weights is off by
//     more than the share of a token. With bits = 62 - log2(vocabulary), at most 46, a weight is
//     rounded by 2^-47 or less of the largest one; tokens below half of that weigh nothing.
//   * A histogram of the row in 2048 bins of equal width in (max - l), a monotone function of the
//     logit in float32, holds each bin's count and weight; their running sums name the bin that a
//     value falls in.
//   * The tokens of that bin (with all bins before it where that is few) are collected into LDS and
//     sorted there by logit and index, and the running sums over them name the token. A bin
//     of more tokens than the list holds (equal logits, mostly) is cut again by bits of logit
//     and index until few are left.
//
// One work-group a row, which reads it a few times (from L2 after the first).
#include "int8_common.h"

namespace migemm {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2 * kThreads;
constexpr int kList = 2 * kThreads;
constexpr int kIndexBits = 20;  // of a token, below the bits of its logit in an order's key

struct Shared {
    uint32_t count[kBins], part_count[kBins];  // running over the row's bins, over a bin's parts
    u64 mass[kBins], part_mass[kBins];
    u64 list[kList], upto[kList];  // keys in order, and the running weight over them
    u64 wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float high[kWaves], low[kWaves];
    int bad;
    uint32_t listed, found;
};

// Ascending keys: largest logit first, then lowest index.
__device__ __forceinline__ uint32_t order_of(float l) {
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? b : b ^ 0x7fffffffu;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order : order ^ 0x7fffffffu);
}
__device__ __forceinline__ u64 key_of(float l, uint32_t index) {
    return (u64)order_of(l) << kIndexBits | index;
}

struct Weights {
    float top;     // the row's largest logit
    float bins;    // bins a unit of (top - l)
    double rate;   // log2(e) / T
    double least;  // min-p
    double unit;   // 2^bits

    __device__ __forceinline__ int bin(float l) const {
        const float d = l == top ? 0.f : top - l;
        return (int)fminf(d * bins, (float)(kBins - 1));
    }
    // exp((l - top) / T), 0 below 2^-60. 2^f for |f| <= 1/2 is 1 + f q(f), q of degree 9 through the
    // Chebyshev nodes of (2^f - 1) / f: off by 2^-50.
    __device__ __forceinline__ double share(float l) const {
        const double y = ((double)l - (double)top) * rate;
        const double t = y + 6755399441055744.0;  // (1.5 2^52: rounds y, its low word is the integer)
        const double f = y - (t - 6755399441055744.0);
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
        const u64 n = (u64)__double_as_longlong(t) << 52;
        const double w = __longlong_as_double((long long)((u64)__double_as_longlong(q) + n));
        return l == top ? 1.0 : y > -60.0 ? w : 0.0;
    }
    __device__ __forceinline__ u64 mass(float l) const {
        const double w = share(l);
        const double x = __builtin_fma(w, unit, 4503599627370496.0);  // (2^52: rounds to integers)
        const u64 m = (u64)__double_as_longlong(x) & (((u64)1 << 52) - 1);
        return w < least ? 0 : m;
    }
};

// Calls f(logit, index) for a row's logits (-0 as 0), those of a thread in ascending order.
template <typename T, typename F>
__device__ __forceinline__ void each(const T *row, int n, const F &f) {
    constexpr int V = 16 / sizeof(T), U = 4;
    for (int first = 0; first < n; first += kThreads * V * U) {
        const int at = first + threadIdx.x * V;
        float x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u)
            load_f32<T, V>(row + at + u * kThreads * V, n - at - u * kThreads * V, x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = at + u * kThreads * V + e;
                if (i < n) f(x[u][e] + 0.f, i);
            }
    }
}

// Running sums of 2 * kThreads masses (and counts), in place. Ends with a barrier.
template <bool COUNTS>
__device__ __forceinline__ void run_up(Shared &s, u64 *mass, uint32_t *count) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64 m0 = mass[2 * tid], m1 = mass[2 * tid + 1];
    u64 m = m0 + m1;
    uint32_t c0 = 0, c1 = 0;
    if (COUNTS) {
        c0 = count[2 * tid];
        c1 = count[2 * tid + 1];
    }
    uint32_t c = c0 + c1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 pm = __shfl_up(m, o);
        if (lane >= o) m += pm;
        if (COUNTS) {
            const uint32_t pc = __shfl_up(c, o);
            if (lane >= o) c += pc;
        }
    }
    if (lane == 63) {
        s.wave_mass[wave] = m;
        s.wave_count[wave] = c;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        m += s.wave_mass[w];
        c += s.wave_count[w];
    }
    mass[2 * tid] = m - m1;
    mass[2 * tid + 1] = m;
    if (COUNTS) {
        count[2 * tid] = c - c1;
        count[2 * tid + 1] = c;
    }
    __syncthreads();
}

// The first place whose running sum reaches 1 <= target <= the last one's.
template <typename N>
__device__ __forceinline__ int reach(Shared &s, const N *sums, int n, N target) {
    for (int i = threadIdx.x; i < n; i += kThreads)
        if (sums[i] >= target && (i == 0 || sums[i - 1] < target)) s.found = i;
    __syncthreads();
    const int i = s.found;
    __syncthreads();
    return i;
}

// A row and what is known of it: the list holds bins first .. last.
template <typename T>
struct Row {
    Shared &s;
    const T *logits;
    int n;
    Weights w;
    int first, last;
    u64 base_mass;        // before the list
    uint32_t base_count;

    __device__ __forceinline__ u64 mass_before(int b) const { return b ? s.mass[b - 1] : 0; }
    __device__ __forceinline__ uint32_t count_before(int b) const {
        return b ? s.count[b - 1] : 0;
    }

    // The tokens of bins a .. b with keys lo .. hi that weigh something (at most kList), sorted, and
    // their running weights.
    __device__ __forceinline__ void collect(int a, int b, u64 lo, u64 hi) {
        const int tid = threadIdx.x;
        if (tid == 0) s.listed = 0;
        __syncthreads();
        each(logits, n, [&](float l, int i) {
            const int at = w.bin(l);
            if (at < a || at > b) return;
            const u64 key = key_of(l, i);
            if (key < lo || key > hi || w.mass(l) == 0) return;
            const uint32_t place = atomicAdd(&s.listed, 1u);
            if (place < kList) s.list[place] = key;
        });
        __syncthreads();
        const int found = min((int)s.listed, kList);
        int size = 2;
        while (size < found) size *= 2;
        for (int i = tid; i < kList; i += kThreads)
            if (i >= found) s.list[i] = ~(u64)0;
        __syncthreads();
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                if (tid < size / 2) {
                    const int x = 2 * tid - (tid & (j - 1)), y = x + j;
                    const u64 p = s.list[x], q = s.list[y];
                    if ((p > q) == ((x & k) == 0)) {
                        s.list[x] = q;
                        s.list[y] = p;
                    }
                }
                __syncthreads();
            }
        for (int i = tid; i < kList; i += kThreads)
            s.upto[i] = i < found ? w.mass(logit_of((uint32_t)(s.list[i] >> kIndexBits))) : 0;
        __syncthreads();
        run_up<false>(s, s.upto, nullptr);
    }

    // The list comes to hold the token of bin b whose running weight (COUNT: number) reaches target.
    template <bool COUNT>
    __device__ __forceinline__ void hold(int b, u64 target) {
        if (first <= b && b <= last) return;
        if (s.count[b] <= kList) {
            first = 0;
            last = b;
            base_mass = 0;
            base_count = 0;
            collect(0, b, 0, ~(u64)0);
            return;
        }
        base_mass = mass_before(b);
        base_count = count_before(b);
        uint32_t left = s.count[b] - base_count;
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
            each(logits, n, [&](float l, int i) {
                if (w.bin(l) != b) return;
                const u64 key = key_of(l, i);
                if (key < lo || key > hi) return;
                const u64 m = w.mass(l);
                if (m == 0) return;
                const int at = (int)((key - lo) >> shift);
                atomicAdd(&s.part_count[at], 1u);
                atomicAdd(&s.part_mass[at], m);
            });
            __syncthreads();
            run_up<true>(s, s.part_mass, s.part_count);
            const int at =
                COUNT ? reach(s, s.part_count, kBins, (uint32_t)target - base_count)
                      : reach(s, s.part_mass, kBins, target - base_mass);
            const uint32_t before = at ? s.part_count[at - 1] : 0;
            left = s.part_count[at] - before;
            base_count += before;
            base_mass += at ? s.part_mass[at - 1] : 0;
            lo += (u64)at << shift;
            const u64 end = lo + (((u64)1 << shift) - 1);
            hi = end < hi ? end : hi;
            __syncthreads();
        }
        collect(b, b, lo, hi);
    }

    // The place in the list of the token whose running weight (number) reaches target.
    __device__ __forceinline__ int by_mass(u64 target) {
        hold<false>(reach(s, s.mass, kBins, target), target);
        return reach(s, s.upto, kList, target - base_mass);
    }
    __device__ __forceinline__ int by_count(uint32_t target) {
        hold<true>(reach(s, s.count, kBins, target), target);
        return (int)(target - base_count) - 1;
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs p) {
    __shared__ Shared s;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x;
    const int n = p.vocab;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const float temperature = p.temperatures != nullptr ? p.temperatures[r] : p.temperature;
    const int top_k = p.top_ks != nullptr ? p.top_ks[r] : p.top_k;
    const float top_p = p.top_ps != nullptr ? p.top_ps[r] : p.top_p;
    const float min_p = p.min_ps != nullptr ? p.min_ps[r] : p.min_p;
    const float uniform = p.uniforms[r];

    // The largest logit, the smallest finite one, and whether any is NaN.
    if (tid == 0) s.bad = 0;
    float high = -INFINITY, low = INFINITY;
    bool nan = false;
    each(logits, n, [&](float l, int) {
        nan |= l != l;
        high = fmaxf(high, l);
        low = l > -INFINITY ? fminf(low, l) : low;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        high = fmaxf(high, __shfl_xor(high, o));
        low = fminf(low, __shfl_xor(low, o));
    }
    if (lane == 0) {
        s.high[wave] = high;
        s.low[wave] = low;
    }
    for (int i = tid; i < kBins; i += kThreads) {
        s.count[i] = 0;
        s.mass[i] = 0;
    }
    __syncthreads();
    if (nan) s.bad = 1;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
        high = fmaxf(high, s.high[w]);
        low = fminf(low, s.low[w]);
    }
    const bool valid = temperature >= 0.f && temperature < INFINITY && top_p == top_p &&
                       min_p == min_p && uniform == uniform;
    if (!valid || s.bad || !(high > -INFINITY)) {  // nothing to choose from
        if (tid == 0) {
            p.tokens[r] = -1;
            p.probabilities[r] = 0.f;
        }
        return;
    }
    if (temperature == 0.f || top_k == 1) {
        if (tid == 0) s.found = n;
        __syncthreads();
        uint32_t best = n;
        each(logits, n, [&](float l, int i) { best = l == high && (uint32_t)i < best ? i : best; });
        if (best < (uint32_t)n) atomicMin(&s.found, best);
        __syncthreads();
        if (tid == 0) {
            p.tokens[r] = (int)s.found;
            p.probabilities[r] = 1.f;
        }
        return;
    }

    Weights w;
    w.top = high;
    w.rate = 1.4426950408889634074 / (double)temperature;
    w.least = min_p < 1.f ? (double)min_p : 1.0;
    w.unit = p.unit;
    // bins over the logits that weigh something, or over all of them where that is less
    const float reach_of = (float)(p.bits + 1) * 0.6931472f * temperature * 1.001f;
    const float span = fminf(reach_of, high - low);
    w.bins = span > 0.f && span < INFINITY ? fminf((float)(kBins - 1) / span, 3e38f) : 0.f;
    each(logits, n, [&](float l, int) {
        const u64 m = w.mass(l);
        if (m == 0) return;
        const int b = w.bin(l);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], m);
    });
    __syncthreads();
    run_up<true>(s, s.mass, s.count);

    Row<T> row{s, logits, n, w, 1, 0, 0, 0};
    u64 total = s.mass[kBins - 1];
    if (top_k > 0 && (uint32_t)top_k < s.count[kBins - 1]) {
        const int i = row.by_count(top_k);
        total = row.base_mass + s.upto[i];
    }
    if (top_p < 1.f) {
        const double t = ceil((double)fmaxf(top_p, 0.f) * (double)total);
        u64 target = (u64)t;
        target = target < 1 ? 1 : target > total ? total : target;
        const int i = row.by_mass(target);
        total = row.base_mass + s.upto[i];
    }
    const double u = uniform < 0.f ? 0.0 : uniform > 1.f ? 1.0 : (double)uniform;
    u64 target = (u64)(u * (double)total) + 1;
    target = target > total ? total : target;
    const int i = row.by_mass(target);
    if (tid == 0) {
        const u64 key = s.list[i];
        p.tokens[r] = (int)(key & (((u64)1 << kIndexBits) - 1));
        p.probabilities[r] =
            (float)(w.share(logit_of((uint32_t)(key >> kIndexBits))) * p.unit / (double)total);
    }
}
}  // namespace

int launch_sample(hipStream_t stream, const SampleArgs &a) {
    SampleArgs p = a;
    int log2 = 0;
    while (((int64_t)1 << log2) < p.vocab) ++log2;
    p.bits = 62 - log2 < 46 ? 62 - log2 : 46;
    p.unit = (double)((uint64_t)1 << p.bits);
    if (p.type == MIGEMM_FLOAT32)
        MIGEMM_LAUNCH((sample_kernel<float>), dim3(p.rows), dim3(kThreads), 0, stream, p);
    else
        MIGEMM_LAUNCH((sample_kernel<Bf16>), dim3(p.rows), dim3(kThreads), 0, stream, p);
    return launch_status("sample_kernel launch");
}

}  // namespace migemm
