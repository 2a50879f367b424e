// What a kernel of this library needs of HIP, for a CPU: a work-group's threads are fibers of one
// thread. A wavefront runs until all of its lanes are at a barrier, before the next wavefront does
// anything, in an order that the caller gives: what one wavefront does between two barriers must
// not depend on whether another has done so yet, so every order has to give the same results. Lanes
// run one after another from one cross-lane operation to the next.
#pragma once
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#define __HIPCC__ 1
#define __global__
#define __device__
#define __host__
#define __forceinline__ inline
#define __shared__ static
#define __launch_bounds__(...)
#define amdgpu_waves_per_eu(x)

typedef void *hipStream_t;
enum hipError_t { hipSuccess = 0 };
inline hipError_t hipGetLastError() { return hipSuccess; }

struct dim3 {
    unsigned x, y, z;
    dim3(unsigned a = 1, unsigned b = 1, unsigned c = 1) : x(a), y(b), z(c) {}
};
struct float4 {
    float x, y, z, w;
};
struct uint4 {
    uint32_t x, y, z, w;
};
struct uint2 {
    uint32_t x, y;
};
inline float4 make_float4(float x, float y, float z, float w) { return float4{x, y, z, w}; }

namespace cpu {
enum State { kReady, kLanes, kBarrier, kDone };  // (kLanes: waits for its wavefront's other lanes)
struct Fiber {
    ucontext_t context;
    char *stack;
    State state;
    unsigned operations;
};
constexpr int kMost = 1024;
static Fiber fibers[kMost];
static ucontext_t scheduler;
static int current, threads;
static uint64_t slots[2][kMost];  // (two, as a lane may be one operation ahead of another)
static int order;                 // of wavefronts: 0 ascending, 1 descending, others shuffled
static void (*call)(const void *);
static const void *argument;

inline void yield(State s) {
    Fiber &f = fibers[current];
    f.state = s;
    swapcontext(&f.context, &scheduler);
}
// The values of this wavefront's lanes.
inline const uint64_t *exchange(uint64_t x) {
    Fiber &f = fibers[current];
    uint64_t *s = slots[f.operations++ & 1];
    s[current] = x;
    yield(kLanes);
    return s + (current & ~63);
}
inline void body() {
    call(argument);
    yield(kDone);
}
}  // namespace cpu

static dim3 blockIdx, threadIdx;

namespace cpu {
inline void run_wavefront(int w) {
    for (;;) {
        int waiting = 0, stopped = 0;
        for (int i = 64 * w; i < 64 * w + 64; ++i) {
            if (fibers[i].state == kReady) {
                current = i;
                threadIdx = dim3(i, 0, 0);
                swapcontext(&scheduler, &fibers[i].context);
            }
            waiting += fibers[i].state == kLanes;
            stopped += fibers[i].state == kBarrier;
        }
        if (waiting == 0) return;
        if (stopped != 0) {
            fprintf(stderr, "lanes of a wavefront wait for different things\n");
            abort();
        }
        for (int i = 64 * w; i < 64 * w + 64; ++i)
            if (fibers[i].state == kLanes) fibers[i].state = kReady;
    }
}
inline void run_group(uint32_t &seed) {
    for (int i = 0; i < threads; ++i) {
        Fiber &f = fibers[i];
        if (f.stack == nullptr) f.stack = static_cast<char *>(malloc(128 << 10));
        getcontext(&f.context);
        f.context.uc_stack.ss_sp = f.stack;
        f.context.uc_stack.ss_size = 128 << 10;
        f.context.uc_link = nullptr;
        makecontext(&f.context, body, 0);
        f.state = kReady;
        f.operations = 0;
    }
    const int waves = threads / 64;
    for (bool left = true; left;) {
        int turn[kMost / 64];
        for (int w = 0; w < waves; ++w) turn[w] = order == 1 ? waves - 1 - w : w;
        if (order > 1)
            for (int w = waves - 1; w > 0; --w) {
                seed = seed * 1664525u + 1013904223u;
                const int o = (seed >> 16) % (w + 1), t = turn[w];
                turn[w] = turn[o];
                turn[o] = t;
            }
        for (int w = 0; w < waves; ++w) run_wavefront(turn[w]);
        left = false;
        for (int i = 0; i < threads; ++i)
            if (fibers[i].state == kBarrier) {
                fibers[i].state = kReady;
                left = true;
            }
    }
}
template <typename F>
void launch(dim3 grid, dim3 block, const F &f) {
    threads = (int)block.x;
    if (threads % 64 != 0 || threads > kMost) abort();
    call = [](const void *p) { (*static_cast<const F *>(p))(); };
    argument = &f;
    uint32_t seed = order;
    const unsigned n = grid.x * grid.y;
    for (unsigned g = 0; g < n; ++g) {
        const unsigned at = order == 1 ? n - 1 - g : g;  // (work-groups in either order, too)
        blockIdx = dim3(at % grid.x, at / grid.x, 0);
        run_group(seed);
    }
}
}  // namespace cpu
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
    cpu::launch(grid, block, [&]() { kernel(__VA_ARGS__); })

inline void __syncthreads() { cpu::yield(cpu::kBarrier); }
inline unsigned long long __ballot(bool x) {
    const uint64_t *s = cpu::exchange(x);
    unsigned long long r = 0;
    for (int i = 0; i < 64; ++i) r |= (unsigned long long)(s[i] & 1) << i;
    return r;
}
template <typename T>
T __shfl(T x, int lane) {
    uint64_t bits = 0;
    memcpy(&bits, &x, sizeof(T));
    bits = cpu::exchange(bits)[lane & 63];
    memcpy(&x, &bits, sizeof(T));
    return x;
}
template <typename T>
T __shfl_xor(T x, int mask) {
    return __shfl(x, (cpu::current & 63) ^ mask);
}
// Moves within rows of 16 lanes (0x111 .. 0x11f) and from the last lane of a row (0x142) or of two
// (0x143) to the rows behind it; `old` where a lane gets nothing.
inline int __builtin_amdgcn_update_dpp(int old, int x, int control, int rows, int, bool) {
    const int lane = cpu::current & 63, row = lane / 16;
    const uint64_t *s = cpu::exchange((uint32_t)x);
    int from;
    if (control > 0x110 && control < 0x120)
        from = lane % 16 - (control - 0x110) >= 0 ? lane - (control - 0x110) : -1;
    else if (control == 0x142)
        from = row > 0 ? 16 * row - 1 : -1;
    else if (control == 0x143)
        from = row > 1 ? 31 : -1;
    else
        abort();
    return from >= 0 && (rows >> row & 1) ? (int)(uint32_t)s[from] : old;
}
template <typename T>
T atomicAdd(T *p, T x) {
    const T old = *p;
    *p += x;
    return old;
}
inline uint32_t atomicMin(uint32_t *p, uint32_t x) {
    const uint32_t old = *p;
    if (x < old) *p = x;
    return old;
}
#define __hip_atomic_store(p, x, ...) (*(p) = (x))
#define __hip_atomic_load(p, ...) (*(p))
#define __HIP_MEMORY_SCOPE_AGENT 0
#define __builtin_amdgcn_fence(...)
#define __builtin_amdgcn_s_waitcnt(x)
#define __builtin_amdgcn_perm(a, b, c) 0u

template <typename To, typename From>
To bits_as(From x) {
    To r;
    memcpy(&r, &x, sizeof(r));
    return r;
}
inline uint32_t __float_as_uint(float x) { return bits_as<uint32_t>(x); }
inline float __uint_as_float(uint32_t x) { return bits_as<float>(x); }
inline long long __double_as_longlong(double x) { return bits_as<long long>(x); }
inline double __longlong_as_double(long long x) { return bits_as<double>(x); }
inline uint32_t __umulhi(uint32_t a, uint32_t b) { return (uint32_t)((uint64_t)a * b >> 32); }
inline int __popcll(unsigned long long x) { return __builtin_popcountll(x); }
inline int __ffsll(unsigned long long x) { return __builtin_ffsll((long long)x); }
inline int __clzll(unsigned long long x) { return x ? __builtin_clzll(x) : 64; }
inline int min(int a, int b) { return a < b ? a : b; }
inline uint32_t min(uint32_t a, uint32_t b) { return a < b ? a : b; }
