// A token for each row of logits: temperature, min-p, top-k, top-p, and a given random number.
//
// Tokens are ordered by logit, largest first, equal ones by index. A token's weight is w =
// exp((l - top) / T), 0 where w < min_p, 0 beyond the first top_k; of the others the fewest are
// kept that hold top_p of their sum, and the token is the first whose weights up to its own are
// more than u times the kept ones' sum. So every step asks one question: where in the order does a
// running count or sum cross a value? It is answered without sorting the row:
//
//   * A histogram of the row, in bins of equal width in (top - l). Its running sums name the bin
//     that a value falls in. With top_k it holds counts (the few tokens that are left get their
//     weights later), otherwise weights.
//   * The tokens of the bins in question are gathered, those that can matter are sorted by logit
//     and index, and the running sums over them name the token. A bin of more tokens than are
//     sorted at once (equal logits, mostly) is first cut by bits of logit and index until few are
//     left.
//
// Weights come from 64-bit arithmetic, because a sum of 10^5 float32 weights is off by more than a
// token's share, and are summed as integers: exactly, in any order (atomics among them), so that a
// result does not depend on how a row was walked. Within a bin's width of at most 2^-5 in log2 w
// a token's weight over its bin's middle one is a polynomial of degree 4 (off by 2^-40 at most);
// these are summed with 43 fractional bits, and a bin's sum is multiplied by its middle weight
// once, to 42 bits below the point or more (62 - log2(vocabulary), at most 46). Tokens that weigh
// less than half of the last bit are left out.
//
// Logits are read three times: for the largest, for the histogram, for the gathering. One
// work-group a row, two of them a CU, is bound by these reads (512 x 65536 float32: 73 us, of
// which 20, 15 and 15 to 18 for 134 MB each; one read at a streaming read's rate gives 19) and,
// with fewer rows than CUs, by the 64-bit steps of the histogram (half of the float32 rate: 11 us
// for 65536 tokens) and by what waits for what: 18 us for 1 x 32000, 4.5 of them the histogram.
// Few rows of many tokens are cut over work-groups, in three launches (1 x 131072: 19 us with
// top-k 50, 35 with top-p 0.9 and no top-k, against 41 and 79 in one work-group).
//
// Where more than 2048 tokens are in question (any top-k above that; rows so flat, or so alike, that
// a bin holds as many) the row's logits are walked again for each cut and sum, one a thread and
// step, by one work-group, so this costs most where rows are few. 1 x 131072, gaussian logits
// of deviation 2: top-k 2500 163 us, with top-p 0.95 212 (top-k 2000: 37); of deviation 0.5, top-p
// 0.9 245 (without 28); of 0.02 337 (150); 64 x 131072 of 0.5 428. Elementary torch operations: 340
// to 390, 1980 for the 64 rows.
#include "int8_common.h"

namespace migemm {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kGather = kBins;  // tokens that are taken out of a row
constexpr int kSort = 256;      // tokens that are sorted at once
constexpr int kIndexBits = 20;  // of a token, below the bits of its logit in an order's key
constexpr int kFraction = 43;   // bits of a weight over its bin's middle one (2^20 of them fit)
constexpr double kOne = (double)((u64)1 << kFraction);
constexpr float kMost = 3.402823466e38f;

struct Shared {
    u64 mass[kBins];        // running weight (or count) over the row's bins
    uint32_t count[kBins];  // running number of tokens, or a bound of it
    union {
        struct {
            u64 list[kSort], upto[kSort];  // keys in order, and the running weight over them
        };
        struct {
            u64 part_mass[kBins];  // the same over the parts of a bin
            uint32_t part_count[kBins];
        };
    };
    u64 gathered[kGather];  // keys of the bins that the answer may need, in any order
    u64 wave_mass[kWaves];
    uint32_t wave_count[kWaves];
    float high[kWaves], low[kWaves];
    int bad;
    // Tokens of the list (set to 0 again only behind a barrier that follows its last reading), and
    // of `gathered`, set once a row: the list begins while some still read the other.
    uint32_t listed, taken;
    uint32_t found;
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
    float r;
    asm("v_min_f32 %0, %1, %2" : "=v"(r) : "s"(kMost), "v"(l));  // (one step: no NaN comes here)
    return r;
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
// a b + c with c in scalar registers (the compiler's form copies c for each use).
__device__ __forceinline__ double step(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}
// A number in [0, 2^52) rounded to an integer, in the adder.
__device__ __forceinline__ u64 rounded(double x, double unit) {
    const double y = __builtin_fma(x, unit, 4503599627370496.0);
    return (u64)__double_as_longlong(y) & (((u64)1 << 52) - 1);
}

// What a row's logits weigh, and its bins: 2^j of them a unit of log2 of the weight, each around
// its middle, a multiple of 2^-j.
struct Weights {
    float least;   // the smallest logit that weighs something
    double top;    // the largest
    double rate;   // log2(e) / T
    double cut;    // how far below the top the smallest weight is
    double magic;  // 1.5 2^(52 - j): adding it rounds to multiples of 2^-j
    double width;  // 2^-j
    double unit;   // 2^bits

    __device__ __forceinline__ void init(const SampleArgs &p, float high, float low,
                                         float temperature, float min_p) {
        top = high;
        rate = 1.4426950408889634074 / (double)temperature;
        unit = p.unit;
        // bins over the logits that weigh something, or over all of them where that is less
        const double spread = top - (double)low;
        cut = (double)(p.bits + 1) * 0.69314718055994530942 * (double)temperature;
        cut = spread < cut ? spread : cut;
        // cut rate = m 2^e with 1 <= m < 2: 1024 to 2047 bins of 2^(e - 10)
        const int e = (int)((u64)__double_as_longlong(cut * rate * 1.001) >> 52) - 1023;
        const int j = 10 - e < 900 ? 10 - e : 900;  // (no spread at all)
        width = ldexp(1.0, -j);
        magic = 6755399441055744.0 * width;
        if (min_p > 0.f) {
            const double most = min_p < 1.f ? -log2((double)min_p) / rate : 0.0;
            cut = most < cut ? most : cut;
        }
        least = smallest(kBins - 1);
    }
    // The smallest logit of bins 0 .. b, by all lanes of a wavefront: bin and cut go by the order
    // of logits, so 64 of them at a time narrow it down.
    __device__ __forceinline__ float smallest(uint32_t b) const {
        uint32_t lo = order_of((float)top), hi = order_of(-kMost);
        while (hi > lo) {
            const uint32_t step = (hi - lo) / 64 + 1;
            const u64 at = lo + (u64)step * (threadIdx.x & 63);
            const float l = logit_of((at < hi ? at : hi) << kIndexBits);
            const int in = __popcll(__ballot(at <= hi && bin(l) <= b && below(l) <= cut));
            lo += step * (in - 1);
            hi = (u64)lo + step - 1 < hi ? lo + step - 1 : hi;
        }
        return logit_of((u64)lo << kIndexBits);
    }
    // How far a logit is below the top.
    __device__ __forceinline__ double below(float l) const { return top - (double)l; }
    // The bin whose middle is nearest is in the low bits of d rate + magic. (For logits beyond the
    // cut they are any.)
    __device__ __forceinline__ double placed(double d) const {
        return __builtin_fma(d, rate, magic);
    }
    static __device__ __forceinline__ uint32_t index(double t) {
        return (uint32_t)__double_as_longlong(t) & (kBins - 1);
    }
    __device__ __forceinline__ uint32_t bin(float l) const {
        const double d = below(l);
        return index(placed(d < cut ? d : cut));
    }
    // The weight over the middle one of its bin, 2^f for |f| <= width / 2, with kFraction bits: 1
    // + f q(f), q of degree 3 through the Chebyshev nodes of (2^f - 1) / f (off by 2^-40 at the
    // bin's ends). Eight 64-bit steps: the middle comes from adding and taking off `magic`, and
    // the last step of the polynomial rounds to an integer, too.
    __device__ __forceinline__ u64 over_middle(double d, uint32_t &b) const {
        const double t = placed(d);
        b = index(t);
        const double f = __builtin_fma(-d, rate, t - magic);
        double q = step(0.00961821489950097 * kOne, f, 0.05550485129481622 * kOne);
        q = step(q, f, 0.24022650695312786 * kOne);
        q = step(q, f, 0.6931471805082434 * kOne);
        const double y = step(q, f, kOne + 4503599627370496.0);  // (2^52: rounds to integers)
        return (u64)__double_as_longlong(y) & (((u64)1 << 52) - 1);
    }
    __device__ __forceinline__ double middle(int b) const { return power(-width * (double)b); }
    __device__ __forceinline__ double share(float l) const {
        const double y = below(l) * rate;
        return y < 64.0 ? power(-y) : 0.0;
    }
    // (A token that is not beyond the cut weighs something.)
    __device__ __forceinline__ u64 mass(float l) const {
        const u64 m = rounded(share(l), unit);
        return m < 1 ? 1 : m;
    }
};

// What a row asks for.
struct Asked {
    float temperature, top_p, min_p, uniform;
    int top_k;
    bool valid;

    __device__ __forceinline__ Asked(const SampleArgs &p, int r) {
        // (loaded whether there or not, from somewhere that is: five loads that fly together)
        uniform = p.uniforms[r];
        const float t = (p.temperatures != nullptr ? p.temperatures : p.uniforms)[r];
        const float tp = (p.top_ps != nullptr ? p.top_ps : p.uniforms)[r];
        const float mp = (p.min_ps != nullptr ? p.min_ps : p.uniforms)[r];
        const int k = (p.top_ks != nullptr ? p.top_ks
                                           : reinterpret_cast<const int *>(p.uniforms))[r];
        temperature = p.temperatures != nullptr ? t : p.temperature;
        top_p = p.top_ps != nullptr ? tp : p.top_p;
        min_p = p.min_ps != nullptr ? mp : p.min_p;
        top_k = p.top_ks != nullptr ? k : p.top_k;
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

// The 16 bytes of logits of a row from place `at`; those at and after `end` are -inf.
template <typename T>
__device__ __forceinline__ uint4 load_logits(const T *row, int at, int end) {
    constexpr int V = 16 / sizeof(T);
    uint4 raw;
    if (at + V <= end) {
        __builtin_memcpy(&raw, row + at, sizeof(raw));
        return raw;
    }
    T x[V];
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = at + e < end ? row[at + e] : from_f32<T>(-INFINITY);
    __builtin_memcpy(&raw, x, sizeof(raw));
    return raw;
}
// Calls f(logits, place of the first) with their float32 values.
template <typename T, typename F>
__device__ __forceinline__ void of_logits(const uint4 &raw, int at, const F &f) {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    constexpr int V = 16 / sizeof(T);
    float x[V];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (V == 4) {
            x[e] = __uint_as_float(u[e]);
        } else {
            x[2 * e] = bf16_low(u[e]);
            x[2 * e + 1] = bf16_high(u[e]);
        }
    }
    f(x, at);
}

// Calls f(logits, place of the first) for the logits first .. end of a row, 16 bytes at a time,
// those of a thread in ascending order (and with -inf for places behind the end). The first HELD
// vectors of a thread stay in registers from start() on, for as many walks as there are; what is
// beyond comes in parts of four vectors, each on its way while the one before is looked at.
template <typename T, int HELD>
struct Walk {
    static constexpr int V = 16 / sizeof(T), STEP = kThreads * V, U = 4;
    const T *row;
    int first, end;
    uint4 held[HELD];

    __device__ __forceinline__ int place(int vector) const {
        return first + vector * STEP + threadIdx.x * V;
    }
    __device__ __forceinline__ void start(const T *r, int a, int b) {
        row = r;
        first = a;
        end = b;
#pragma unroll
        for (int u = 0; u < HELD; u += 2)
            if (first + u * STEP < end) {
                held[u] = load_logits<T>(row, place(u), end);
                held[u + 1] = load_logits<T>(row, place(u + 1), end);
            }
    }
    template <typename F>
    __device__ __forceinline__ void go(const F &f) const {
#pragma unroll
        for (int u = 0; u < HELD; u += 2) {
            const uint4 a = held[u], b = held[u + 1];
            if (first + u * STEP < end) {  // (two at a time: more to do while one waits)
                of_logits<T>(a, place(u), f);
                of_logits<T>(b, place(u + 1), f);
            }
        }
        if (first + HELD * STEP < end) rest(HELD, f);
    }
    template <typename F>
    __device__ __forceinline__ void rest(int vector, const F &f) const {
        uint4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load_logits<T>(row, place(vector + u), end);
        for (; first + vector * STEP < end; vector += U) {
            uint4 y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) y[u] = x[u];
            if (first + (vector + U) * STEP < end) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    x[u] = load_logits<T>(row, place(vector + U + u), end);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) of_logits<T>(y[u], place(vector + u), f);
        }
    }
};
// The largest logit of a range and whether one is NaN, in every lane, and with `wide` the smallest
// above -inf (otherwise it is -inf). At low temperatures the logits that weigh something span
// less than all of them, so the smallest does not matter, and costs half of the pass.
template <typename W>
__device__ __forceinline__ void extremes(const W &walk, bool wide, float &high,
                                         float &low, bool &nan) {
    high = -INFINITY;
    low = wide ? INFINITY : -INFINITY;
    nan = false;
    constexpr int V = W::V;
    if (wide)
        walk.go([&](const auto &x, int) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                nan |= x[e] != x[e];
                high = fmaxf(high, x[e]);
                low = x[e] > -INFINITY ? fminf(low, x[e]) : low;
            }
        });
    else
        walk.go([&](const auto &x, int) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                nan |= x[e] != x[e];
                high = fmaxf(high, x[e]);
            }
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

// The tokens first .. end into the histogram: their weights, or with COUNT their number.
template <bool COUNT, typename W>
__device__ __forceinline__ void fill(u64 *mass, const W &walk, const Weights &w) {
    walk.go([&](const auto &x, int) {
        constexpr int V = W::V;
        u64 m[V];
        uint32_t b[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const double d = w.below(bounded(x[e]));
            m[e] = COUNT ? 1 : w.over_middle(d, b[e]);
            if (COUNT) b[e] = w.index(w.placed(d));
        }
        // (here all are known: left alone, the compiler moves each token's chain of dependent steps
        // behind its comparison, and none runs beside another)
#pragma unroll
        for (int e = 0; e < V; ++e) asm volatile("" : "+v"(m[e]), "+v"(b[e]));
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (x[e] >= w.least) atomicAdd(&mass[b[e]], m[e]);
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

// Running sums of kBins masses (and counts), in place. Ends with a barrier.
template <bool COUNTS>
__device__ __forceinline__ void run_up(Shared &s, u64 *mass, uint32_t *count) {
    constexpr int PER = kBins / kThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    u64 m[PER];
    uint32_t c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        m[i] = mass[PER * tid + i] + (i ? m[i - 1] : 0);
        if (COUNTS) c[i] = count[PER * tid + i] + (i ? c[i - 1] : 0);
    }
    const u64 lanes_m = run_up_lanes(m[PER - 1]);
    const uint32_t lanes_c = COUNTS ? run_up_lanes(c[PER - 1]) : 0;
    if (lane == 63) {
        s.wave_mass[wave] = lanes_m;
        s.wave_count[wave] = lanes_c;
    }
    __syncthreads();
    // the sums of the wavefronts before: the lanes of a row of 16 take one each
    u64 before_m = run_up_lanes(lane < wave ? s.wave_mass[lane & (kWaves - 1)] : 0);
    before_m = __shfl(before_m, kWaves - 1) + lanes_m - m[PER - 1];
    uint32_t before_c = 0;
    if (COUNTS) {
        before_c = run_up_lanes(lane < wave ? s.wave_count[lane & (kWaves - 1)] : 0);
        before_c = __shfl(before_c, kWaves - 1) + lanes_c - c[PER - 1];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        mass[PER * tid + i] = before_m + m[i];
        if (COUNTS) count[PER * tid + i] = before_c + c[i];
    }
    __syncthreads();
}

// A filled histogram becomes its running sums. A bin's weight is its sum times its middle one; its
// number of tokens is at most the sum over the least that a token adds to it (2^-0.016, 1 / 1.011).
template <bool COUNT>
__device__ __forceinline__ void finish(Shared &s, const Weights &w) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        const u64 m = s.mass[b];
        if (COUNT) {
            s.count[b] = (uint32_t)m;
        } else {
            s.count[b] = m ? (uint32_t)((double)m * (1.02 / kOne)) + 1 : 0;
            s.mass[b] = m ? (u64)((double)m * (w.middle(b) * (w.unit / kOne)) + 0.5) : 0;
        }
    }
    __syncthreads();
    run_up<true>(s, s.mass, s.count);
}

// The first place whose running sum reaches target (the last one's does, or the last sum is taken
// for it). Every wavefront looks for itself: at every N / 64-th sum, then at those between.
template <int N>
__device__ __forceinline__ int reach(const u64 *sums, u64 target) {
    constexpr int STEP = N / 64;
    static_assert(STEP >= 1 && STEP <= 64 && STEP * 64 == N, "two looks");
    const int lane = threadIdx.x & 63;
    const u64 last = sums[N - 1];
    target = target < last ? target : last;
    const u64 far = __ballot(sums[STEP * lane + STEP - 1] >= target);
    const int from = STEP * (__ffsll(far) - 1);
    const u64 near = __ballot(sums[from + (lane < STEP ? lane : STEP - 1)] >= target);
    return from + __ffsll(near) - 1;
}

// Sorts the first n keys of the list, with `upto` as room: each finds its place by counting the
// smaller ones, two threads or more a key. (64 keys: 0.3 us, 3.0 by exchanges, each of whose steps
// waits for the one before.)
__device__ __forceinline__ void sort(Shared &s, int n) {
    const int tid = threadIdx.x;
    int per = kThreads / kSort;  // threads a key
    while (per < 32 && n * per * 2 <= kThreads) per *= 2;
    const int i = tid / per, part = tid & (per - 1);
    u64 key = 0;
    uint32_t less = 0;
    if (i < n) {
        key = s.list[i];
        int j = part;
        for (; j + 7 * per < n; j += 8 * per) {  // (eight reads fly together)
            u64 x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = s.list[j + k * per];
#pragma unroll
            for (int k = 0; k < 8; ++k) less += x[k] < key;
        }
        for (; j < n; j += per) less += s.list[j] < key;
    }
    for (int o = 1; o < per; o *= 2) less += __shfl_xor(less, o);
    if (i < n && part == 0) s.upto[less] = key;
    __syncthreads();
    if (tid < n) s.list[tid] = s.upto[tid];
    __syncthreads();
}

// Bins whose tokens a row's answer may need, as far as the histogram tells: all up to one of them
// that can be sorted at once (whole), or single ones. `listed`: they are few enough to be
// gathered.
struct Plan {
    bool whole, listed;
    int kept, first, last;  // the bin where top-k or top-p ends (-1: none does), those to draw from
};

// Of the tokens of bins a .. b.
__device__ __forceinline__ uint32_t count_in(const Shared &s, int a, int b) {
    return s.count[b] - (a ? s.count[a - 1] : 0);
}

__device__ __forceinline__ Plan plan_of(Shared &s, const Asked &q, bool counted) {
    Plan g{true, true, kBins - 1, 0, -1};
    const u64 total = s.mass[kBins - 1];
    u64 low = total, high = total;
    if (counted) {
        g.kept = reach<kBins>(s.mass, (u64)q.top_k);
    } else if (q.top_p < 1.f) {
        g.kept = reach<kBins>(s.mass, q.kept(total));
        low = g.kept ? s.mass[g.kept - 1] : 1;
        high = s.mass[g.kept];
    }
    if (s.count[g.kept] <= kSort) return g;
    g.whole = false;
    if (counted) {
        g.last = g.kept;
        g.listed = s.count[g.kept] <= kGather;
        return g;
    }
    g.first = reach<kBins>(s.mass, q.drawn(low));
    g.last = reach<kBins>(s.mass, q.drawn(high));
    uint32_t n = count_in(s, g.first, g.last);
    if (q.top_p < 1.f) {
        if (g.kept > g.last) n += count_in(s, g.kept, g.kept);
    } else {
        g.kept = -1;
    }
    g.listed = n <= kGather;
    return g;
}

// The logits of bins a .. b: from the smallest one's up to, but not with, the one that ends the bin
// before (NaN: there is none).
struct Span {
    float from, end;

    __device__ __forceinline__ Span(const Weights &w, int a, int b)
        : from(w.smallest(b)), end(a > 0 ? w.smallest(a - 1) : __uint_as_float(0x7fc00000u)) {}
    __device__ __forceinline__ bool has(float x) const { return x >= from && !(x >= end); }
};

// The keys of the plan's tokens into s.gathered; returns their number. Top-p's bin and those to
// draw from are two spans of logits, so no token's bin is computed.
template <typename W>
__device__ __forceinline__ int gather(Shared &s, const W &walk, const Weights &w,
                                      const Plan &plan) {
    constexpr int V = W::V;
    const Span draw = plan.whole ? Span(w, 0, plan.kept) : Span(w, plan.first, plan.last);
    const bool apart = !plan.whole && plan.kept > plan.last;
    Span kept = draw;
    if (apart) kept = Span(w, plan.kept, plan.kept);
    if (threadIdx.x == 0) s.taken = 0;
    __syncthreads();
    walk.go([&](const auto &x, int i) {
        float most = x[0];  // (few are taken: one question for all of them)
#pragma unroll
        for (int e = 1; e < V; ++e) most = fmaxf(most, x[e]);
        if (!(most >= kept.from)) return;  // (kept is not before draw)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            if (!(draw.has(x[e]) || kept.has(x[e]))) continue;
            const uint32_t place = atomicAdd(&s.taken, 1u);
            if (place < kGather) s.gathered[place] = key_of(bounded(x[e]), i + e);
        }
    });
    __syncthreads();
    return min((int)s.taken, kGather);
}

// A row and what is known of it. Its tokens come from keys that were gathered, or (keys null; a
// row of too many, and walked simply, so that this case takes no registers from the other) its
// logits.
template <typename T>
struct Row {
    Shared &s;
    const T *logits;
    int n;
    const u64 *keys;
    int gathered;
    const Weights &w;
    u64 limit;  // keys past it are out (top-k)
    u64 base;   // what runs up to the list

    // Calls f(key) for the tokens with keys lo .. hi.
    template <typename F>
    __device__ __forceinline__ void tokens(u64 lo, u64 hi, const F &f) const {
        hi = hi < limit ? hi : limit;
        if (keys != nullptr) {
            for (int i = threadIdx.x; i < gathered; i += kThreads)
                if (keys[i] >= lo && keys[i] <= hi) f(keys[i]);
            return;
        }
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 key = key_of(bounded(to_f32(logits[i])), i);
            if (key >= lo && key <= hi) f(key);
        }
    }
    // The keys of bins a .. b lie within these.
    __device__ __forceinline__ u64 first_key(int a) const {
        return a ? ((u64)order_of(w.smallest(a - 1)) + 1) << kIndexBits : 0;
    }
    __device__ __forceinline__ u64 last_key(int b) const {
        return (((u64)order_of(w.smallest(b)) + 1) << kIndexBits) - 1;
    }

    // The list: the tokens with keys lo .. hi (at most kSort), sorted, and their running weights.
    __device__ __forceinline__ void collect(u64 lo, u64 hi) {
        const int tid = threadIdx.x;
        if (tid == 0) s.listed = 0;
        __syncthreads();
        tokens(lo, hi, [&](u64 key) {
            const uint32_t place = atomicAdd(&s.listed, 1u);
            if (place < kSort) s.list[place] = key;
        });
        __syncthreads();
        const int n = min((int)s.listed, kSort);
        sort(s, n);
        if (tid < kSort) {
            const u64 m = run_up_lanes(tid < n ? w.mass(logit_of(s.list[tid])) : 0);
            s.upto[tid] = m;
            if ((tid & 63) == 63) s.wave_mass[tid >> 6] = m;
        }
        __syncthreads();
        if (tid < kSort) {
            u64 m = s.upto[tid];
            for (int k = 0; k < tid >> 6; ++k) m += s.wave_mass[k];
            s.upto[tid] = m;
        }
        __syncthreads();
    }

    // The list comes to hold the token of bin b whose running weight (COUNT: number) reaches
    // target.
    template <bool COUNT>
    __device__ __forceinline__ void hold(int b, u64 target) {
        base = b ? s.mass[b - 1] : 0;
        u64 lo = first_key(b), hi = last_key(b);
        uint32_t left;
        if (keys != nullptr) {
            if (threadIdx.x == 0) s.listed = 0;
            __syncthreads();
            tokens(lo, hi, [&](u64) { atomicAdd(&s.listed, 1u); });
            __syncthreads();
            left = s.listed;
            __syncthreads();
        } else {
            left = count_in(s, b, b);
        }
        while (left > kSort) {  // cut by the keys' bits; a range of one key holds one token
            const int bits = 64 - __clzll(hi - lo);
            const int shift = bits > 11 ? bits - 11 : 0;
            __syncthreads();
            for (int i = threadIdx.x; i < kBins; i += kThreads) {
                s.part_count[i] = 0;
                s.part_mass[i] = 0;
            }
            __syncthreads();
            tokens(lo, hi, [&](u64 key) {
                const int at = (int)((key - lo) >> shift);
                atomicAdd(&s.part_count[at], 1u);
                atomicAdd(&s.part_mass[at], COUNT ? (u64)1 : w.mass(logit_of(key)));
            });
            __syncthreads();
            run_up<true>(s, s.part_mass, s.part_count);
            const int at = reach<kBins>(s.part_mass, target - base);
            left = s.part_count[at] - (at ? s.part_count[at - 1] : 0);
            base += at ? s.part_mass[at - 1] : 0;
            lo += (u64)at << shift;
            const u64 end = lo + (((u64)1 << shift) - 1);
            hi = end < hi ? end : hi;
            __syncthreads();
        }
        collect(lo, hi);
    }

    // The place in the list of the token whose running weight reaches target.
    __device__ __forceinline__ int by_mass(u64 target) {
        hold<false>(reach<kBins>(s.mass, target), target);
        return reach<kSort>(s.upto, target - base);
    }

    // The row's token, from its histogram's running sums.
    __device__ __forceinline__ void answer(const SampleArgs &p, int r, const Asked &q, bool counted,
                                           const Plan &plan, u64 total) {
        int i;
        if (plan.whole) {  // the list holds all tokens that may be kept
            collect(0, last_key(plan.kept));
            if (counted)
                total = s.upto[q.top_k < kSort ? q.top_k - 1 : kSort - 1];
            else if (!(q.top_p < 1.f))
                total = s.upto[kSort - 1];
            if (q.top_p < 1.f) total = s.upto[reach<kSort>(s.upto, q.kept(total))];
            i = reach<kSort>(s.upto, q.drawn(total));
        } else {
            if (counted) {  // the tokens that top-k leaves get their weights
                const u64 k = (u64)q.top_k < total ? (u64)q.top_k : total;
                hold<true>(plan.kept, k);
                limit = s.list[k - base - 1];
                __syncthreads();
                for (int b = threadIdx.x; b < kBins; b += kThreads) s.mass[b] = 0;
                __syncthreads();
                tokens(0, limit, [&](u64 key) {
                    uint32_t b;
                    const u64 m = w.over_middle(w.below(logit_of(key)), b);
                    atomicAdd(&s.mass[b], m);
                });
                __syncthreads();
                finish<false>(s, w);
                total = s.mass[kBins - 1];
            }
            if (q.top_p < 1.f) {
                const u64 target = q.kept(total);
                const u64 most = s.mass[reach<kBins>(s.mass, target)];
                const int at = by_mass(target);
                // (roundings of the bin's weight and of its tokens' must not reach into the next)
                total = base + s.upto[at] < most ? base + s.upto[at] : most;
            }
            i = by_mass(q.drawn(total));
        }
        if (threadIdx.x == 0) {
            const u64 key = s.list[i];
            p.tokens[r] = min((int)(key & (((u64)1 << kIndexBits) - 1)), p.vocab - 1);
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
    Walk<T, 4> walk;
    walk.start(logits, 0, n);
    extremes(walk, q.wide(), high, low, nan);
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
        walk.go([&](const auto &x, int i) {
#pragma unroll
            for (int e = 0; e < 16 / (int)sizeof(T); ++e)
                best = bounded(x[e]) == high && (uint32_t)(i + e) < best ? i + e : best;
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
        fill<true>(s.mass, walk, w);
    else
        fill<false>(s.mass, walk, w);
    __syncthreads();
    if (counted)
        finish<true>(s, w);
    else
        finish<false>(s, w);
    const Plan plan = plan_of(s, q, counted);
    const u64 total = s.mass[kBins - 1];
    const int gathered = plan.listed ? gather(s, walk, w, plan) : 0;
    Row<T> row{s, logits, n, plan.listed ? s.gathered : nullptr, gathered, w, ~(u64)0, 0};
    row.answer(p, r, q, counted, plan, total);
}
// ------------------------------------------------------------- rows cut over work-groups
// Three launches: the largest logit of each part of a row; the parts' histograms, added up; and the
// tokens of the bins that the answer may need, and from them the answer. Each part of the third
// reads the whole histogram and plans the same, and the one that comes to its end last (no other is
// waited for) goes on to the answer, with the running sums still in LDS. A row whose tokens
// the list does not hold is walked by that work-group alone. What waits for memory is loaded as a
// kernel begins.
enum RowKind { kNothing, kGreedy, kDraw };
struct RowState {
    Weights w;         // these two of the second kernel's first part
    int kind;
    uint32_t listed;   // tokens gathered
    uint32_t arrived;  // parts that have gathered theirs
    uint32_t best;     // where the largest logit stands first (kGreedy)
};
struct SplitArgs {
    SampleArgs p;
    int splits, chunk;  // parts of a row, tokens of a part
    u64 *mass;          // [rows][kBins]
    u64 *list;          // [rows][kGather]
    float4 *parts;      // [rows][splits]: largest, smallest, whether one is NaN
    RowState *state;    // [rows]
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_top_kernel(SplitArgs a) {
    __shared__ float highs[kWaves], lows[kWaves];
    __shared__ int bad;
    const SampleArgs &p = a.p;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const int first = part * a.chunk, end = min(first + a.chunk, p.vocab);
    Walk<T, 4> walk;
    walk.start(logits, first, end);
    const Asked q(p, r);
    for (int i = part * kThreads + tid; i < kBins; i += a.splits * kThreads)
        a.mass[(int64_t)r * kBins + i] = 0;
    if (part == 0 && tid == 0) {
        a.state[r].listed = 0;
        a.state[r].arrived = 0;
        a.state[r].best = ~0u;
    }
    if (tid == 0) bad = 0;
    float high, low;
    bool nan;
    extremes(walk, q.wide(), high, low, nan);
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

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_bins_kernel(SplitArgs a) {
    __shared__ u64 mass[kBins];
    const SampleArgs &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, part = blockIdx.x, r = blockIdx.y;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const int first = part * a.chunk, end = min(first + a.chunk, p.vocab);
    float4 x = make_float4(-INFINITY, INFINITY, 0.f, 0.f);
    if (lane < a.splits) x = a.parts[(int64_t)r * a.splits + lane];
    const Asked q(p, r);
    Walk<T, 4> walk;
    walk.start(logits, first, end);
    for (int i = tid; i < kBins; i += kThreads) mass[i] = 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        x.x = fmaxf(x.x, __shfl_xor(x.x, o));
        x.y = fminf(x.y, __shfl_xor(x.y, o));
    }
    const bool some = q.valid && __ballot(x.z != 0.f) == 0 && x.x > -INFINITY;
    const int kind = !some ? kNothing : q.greedy() ? kGreedy : kDraw;
    Weights w{};
    w.top = x.x;
    if (kind == kDraw) w.init(p, x.x, x.y, q.temperature, q.min_p);
    if (part == 0 && tid == 0) {
        a.state[r].w = w;
        a.state[r].kind = kind;
    }
    if (kind != kDraw) return;
    __syncthreads();
    if (q.counted(p.vocab))
        fill<true>(mass, walk, w);
    else
        fill<false>(mass, walk, w);
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads)
        if (mass[i] != 0) atomicAdd(&a.mass[(int64_t)r * kBins + i], mass[i]);
}

// What a row's parts tell each other within a launch goes to memory and comes from there, past the
// caches that they do not share.
template <typename N>
__device__ __forceinline__ void write_now(N *to, N x) {
    __hip_atomic_store(to, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename N>
__device__ __forceinline__ N read_now(const N *x) {
    return __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this work-group is the last of its row's parts to come here: all that the others wrote is
// then there to be read. This rests on the chip's order, not on the language's release and acquire:
// stores and loads of agent scope go past the L2s that work-groups do not share (sc1), a
// wavefront's wait ends when its stores have got there, and a work-group is counted behind the
// barrier that its threads come to after that wait. (A fence, which would say it in the language,
// writes back and invalidates a whole L2, in every work-group: 64 x 131072 73 us.)
__device__ __forceinline__ bool last_part(Shared &s, RowState &state, int parts) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // (no write moves behind the wait)
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) s.found = atomicAdd(&state.arrived, 1u);
    __syncthreads();
    return s.found == (uint32_t)parts - 1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_answer_kernel(SplitArgs a) {
    __shared__ Shared s;
    const SampleArgs &p = a.p;
    const int tid = threadIdx.x, part = blockIdx.x, r = blockIdx.y;
    const T *logits = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    const int first = part * a.chunk, end = min(first + a.chunk, p.vocab);
    RowState &state = a.state[r];
    for (int i = tid; i < kBins; i += kThreads) s.mass[i] = a.mass[(int64_t)r * kBins + i];
    const float mine = a.parts[(int64_t)r * a.splits + part].x;
    const Asked q(p, r);
    const int kind = state.kind;
    const Weights w = state.w;
    Walk<T, 4> walk;
    walk.start(logits, first, end);
    if (kind == kNothing) {
        if (part == 0) nothing(p, r);
        return;
    }
    if (kind == kGreedy) {
        const float high = (float)w.top;
        if (mine == high) {
            uint32_t best = ~0u;
            walk.go([&](const auto &x, int i) {
#pragma unroll
                for (int e = 0; e < 16 / (int)sizeof(T); ++e)
                    best = bounded(x[e]) == high && (uint32_t)(i + e) < best ? i + e : best;
            });
            if (best != ~0u) atomicMin(&state.best, best);
        }
        if (last_part(s, state, a.splits) && tid == 0) {
            p.tokens[r] = (int)read_now(&state.best);
            p.probabilities[r] = 1.f;
        }
        return;
    }
    const bool counted = q.counted(p.vocab);
    if (counted)
        finish<true>(s, w);
    else
        finish<false>(s, w);
    const Plan plan = plan_of(s, q, counted);
    u64 *list = a.list + (int64_t)r * kGather;
    if (plan.listed && mine >= w.smallest(plan.kept > plan.last ? plan.kept : plan.last)) {
        const int found = gather(s, walk, w, plan);
        if (tid == 0 && found) s.found = atomicAdd(&state.listed, (uint32_t)found);
        __syncthreads();
        const int to = s.found;
        for (int i = tid; i < found && to + i < kGather; i += kThreads)
            write_now(list + to + i, s.gathered[i]);
    }
    if (!last_part(s, state, a.splits)) return;
    const int gathered = min(read_now(&state.listed), (uint32_t)kGather);
    if (plan.listed) {
        for (int i = tid; i < gathered; i += kThreads) s.gathered[i] = read_now(list + i);
        __syncthreads();
    }
    const u64 total = s.mass[kBins - 1];
    Row<T> row{s, logits, p.vocab, plan.listed ? s.gathered : nullptr, gathered, w, ~(u64)0, 0};
    row.answer(p, r, q, counted, plan, total);
}

template <typename T>
int launch_split(hipStream_t stream, SplitArgs a) {
    const SampleArgs &p = a.p;
    const size_t row = (kBins + kGather) * sizeof(u64) + a.splits * sizeof(float4) +
                       sizeof(RowState);
    int rc = MIGEMM_OK;
    a.mass = static_cast<u64 *>(workspace(stream, p.rows * row, &rc, 0));
    if (a.mass == nullptr) return rc;
    a.list = a.mass + (int64_t)p.rows * kBins;
    a.parts = reinterpret_cast<float4 *>(a.list + (int64_t)p.rows * kGather);
    a.state = reinterpret_cast<RowState *>(a.parts + (int64_t)p.rows * a.splits);
    const dim3 grid(a.splits, p.rows), block(kThreads);
    MIGEMM_LAUNCH((sample_top_kernel<T>), grid, block, 0, stream, a);
    MIGEMM_LAUNCH((sample_bins_kernel<T>), grid, block, 0, stream, a);
    MIGEMM_LAUNCH((sample_answer_kernel<T>), grid, block, 0, stream, a);
    return launch_status("sample_answer_kernel launch");
}

template <typename T>
int launch(hipStream_t stream, const SampleArgs &p) {
    // In parts or a work-group a row, us on a graph with top-k 50 and top-p 0.95 / with top-p 0.9
    // alone, rows of gaussian float32 logits (deviation 2): 1 x 32000 20.4 / 31.6 in parts, 18.9 /
    // 33.7 whole; 1 x 40960 19.1 / 31.1 and 20.5 / 37.7; 40 x 40960 24.3 / 37.1 and 21.6 / 40.2;
    // 64 x 40960 28.5 / 41.6 and 23.3 / 41.6; 1 x 65536 19.0 / 33.0 and 26.3 / 50.3; 64 x 65536
    // 28.8 / 45.4 and 29.7 / 55.4; 128 x 65536 34.0 / 54.2 and 30.4 / 56.9; 1 x 131072 19.1 / 35.0
    // and 40.8 / 78.6; 128 x 131072 48.9 / 76.0 and 48.3 / 90.3. 256 parts in all (one a CU) of at
    // least 4096 tokens: with 512 or 1024 each reads and writes more of the histogram than it
    // saves (1 to 4 us more). A row in two parts at least, so 128 rows at most.
    SplitArgs a{};
    a.p = p;
    const int most = p.vocab / 4096 < 64 ? p.vocab / 4096 : 64;
    a.splits = 256 / p.rows < most ? 256 / p.rows : most;
    if (p.vocab >= 40960 && p.rows <= p.vocab / 1024 && a.splits > 1) {
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
