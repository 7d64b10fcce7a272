// The host stand-in of tests/host_requests with cross-lane operations that give their values:
// a block's threads run in turns, a barrier is passed once all of the block's (a cross-lane
// operation's: of the wave's) threads have come to it.  Results are the kernels' own.
#pragma once
#include "../../host_requests/hip/hip_runtime.h"
#include <stdint.h>

// Saves the callee's registers (x86-64) on this stack, whose top goes to *from, and goes on
// where `to` was saved.  (swapcontext asks the kernel for the signals' mask each time: five
// times slower here.)
extern "C" void host_switch(void **from, void *to);
asm(R"(
.text
.weak host_switch
host_switch:
    push %rbp
    push %rbx
    push %r12
    push %r13
    push %r14
    push %r15
    mov %rsp, (%rdi)
    mov %rsi, %rsp
    pop %r15
    pop %r14
    pop %r13
    pop %r12
    pop %rbx
    pop %rbp
    ret
)");
struct HostTurns {
    static constexpr size_t kStack = 64 << 10;
    void *main, *top[1024];
    bool over[1024];
    char *stack = (char *)aligned_alloc(64, 1024 * kStack);
    void (*call)(void *);
    void *argument;
    unsigned now;
    static HostTurns &get() {
        static HostTurns t;
        return t;
    }
    static void enter() {
        HostTurns &t = get();
        t.call(t.argument);
        t.over[t.now] = true;
        t.wait();
    }
    void wait() { host_switch(&top[now], main); }
    void run(unsigned n) {
        for (unsigned i = 0; i < n; ++i) {
            void **p = (void **)(stack + (i + 1) * kStack) - 2;      // (enter begins as a call leaves the stack)
            *p = (void *)&HostTurns::enter;
            top[i] = p - 6;
            over[i] = false;
        }
        for (bool any = true; any;) {
            any = false;
            for (unsigned i = 0; i < n; ++i) {
                if (over[i]) continue;
                any = true;
                now = i;
                threadIdx = dim3(i, 0, 0);
                host_switch(&main, top[i]);
            }
        }
    }
};

struct HostMeeting {
    unsigned live = 0, there = 0, times = 0;
    uint64_t slot[2][64];
    bool over() {
        if (there < live) return false;
        there = 0;
        ++times;
        return true;
    }
    void meet() {
        const unsigned was = times;
        ++there;
        while (times == was && !over()) HostTurns::get().wait();
    }
};
inline HostMeeting host_block, host_wave[16];
inline void host_sync() { host_block.meet(); }
// the slots of a wave's lanes, each with the lane's v
inline const uint64_t *host_lanes(uint64_t v) {
    HostMeeting &w = host_wave[threadIdx.x >> 6];
    uint64_t *slot = w.slot[w.times & 1];      // (the last ones may still be read)
    slot[threadIdx.x & 63] = v;
    w.meet();
    return slot;
}
inline int host_shfl(int v, int lane) { return (int)host_lanes((uint32_t)v)[lane & 63]; }
inline int host_shfl_xor(int v, int o) { const int at = threadIdx.x & 63; return (int)host_lanes((uint32_t)v)[at ^ o]; }
inline int host_shfl_up(int v, int o) {
    const int at = threadIdx.x & 63;
    return (int)host_lanes((uint32_t)v)[at >= o ? at - o : at];
}
inline uint64_t host_ballot(bool v) {
    const uint64_t *slot = host_lanes(v);
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= slot[i] << i;
    return r;
}
template <class T> T atomicMin(T *p, T v) { T o = *p; if (v < o) *p = v; return o; }
inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
#undef __syncthreads
#define __syncthreads host_sync
#define __shfl host_shfl
#define __shfl_xor host_shfl_xor
#define __shfl_up host_shfl_up
#define __ballot host_ballot

template <class... P, class... A> void host_grid(const char *name, void (*f)(P...), dim3 g, dim3 b, A... a) {
    host_kernel = name;
    gridDim = g; blockDim = b;
    auto one = [&] {
        const unsigned wave = threadIdx.x >> 6;
        f(static_cast<P>(a)...);
        --host_block.live;
        --host_wave[wave].live;
    };
    HostTurns &t = HostTurns::get();
    t.call = [](void *p) { (*static_cast<decltype(one) *>(p))(); };
    t.argument = &one;
    for (unsigned z = 0; z < g.z; ++z) for (unsigned y = 0; y < g.y; ++y) for (unsigned x = 0; x < g.x; ++x) {
        blockIdx = dim3(x, y, z);
        host_block = HostMeeting{b.x};
        for (unsigned w = 0; w < b.x / 64; ++w) host_wave[w] = HostMeeting{64};
        t.run(b.x);
    }
}
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(k, g, b, s, st, ...) ((void)(st), host_grid(#k, k, g, b, __VA_ARGS__))
