// The host stand-in of tests/host_float with what the gated recurrence's and the adapters'
// kernels use beside it.  Here a block's threads run in turns from barrier to barrier (each
// has a stack of its own), since a block takes its tiles through LDS.  Blocks run one after
// another, so a word that a block waits for has to be there.
#pragma once
#include "../../host_float/hip/hip_runtime.h"
#include <ucontext.h>
#include <vector>
#define __HIP_MEMORY_SCOPE_AGENT 4
inline void __builtin_amdgcn_s_sleep(int) { host_die("a wait for a word that no block before has written", 0, 0); }
inline float __builtin_amdgcn_rsqf(float v) { return 1.0f / sqrtf(v); }

struct HostThreads {
    static constexpr size_t kStack = 128 << 10;
    ucontext_t main;
    std::vector<ucontext_t> thread;
    std::vector<char> stack;
    std::vector<bool> over;
    void (*call)(void *);
    void *argument;
    unsigned now;
    static HostThreads &get() {
        static HostThreads t;
        return t;
    }
    static void enter() {
        HostThreads &t = get();
        t.call(t.argument);
        t.over[t.now] = true;
        swapcontext(&t.thread[t.now], &t.main);
    }
    void barrier() { swapcontext(&thread[now], &main); }
    void run(unsigned n) {
        thread.resize(n);
        over.assign(n, false);
        if (stack.size() < n * kStack) stack.resize(n * kStack);
        for (unsigned i = 0; i < n; ++i) {
            getcontext(&thread[i]);
            thread[i].uc_stack.ss_sp = &stack[i * kStack];
            thread[i].uc_stack.ss_size = kStack;
            thread[i].uc_link = nullptr;
            makecontext(&thread[i], &HostThreads::enter, 0);
        }
        for (bool any = true; any;) {
            any = false;
            for (unsigned i = 0; i < n; ++i) {
                if (over[i]) continue;
                any = true;
                now = i;
                threadIdx = dim3(i, 0, 0);
                swapcontext(&main, &thread[i]);
            }
        }
    }
};
inline void host_barrier() { HostThreads::get().barrier(); }
#define __syncthreads host_barrier

template <class... P, class... A> void host_blocks(const char *name, void (*f)(P...), dim3 g, dim3 b, A... a) {
    host_kernel = name;
    gridDim = g; blockDim = b;
    if (host_dry) {
        if (!g.x || (uint64_t)g.x * b.x >> 32 || !g.y || g.y > 65535 || !g.z || g.z > 65535) host_error = hipErrorInvalidValue;
        return;
    }
    auto one = [&] { f(static_cast<P>(a)...); };
    HostThreads &t = HostThreads::get();
    t.call = [](void *p) { (*static_cast<decltype(one) *>(p))(); };
    t.argument = &one;
    for (unsigned z = 0; z < g.z; ++z) for (unsigned y = 0; y < g.y; ++y) for (unsigned x = 0; x < g.x; ++x) {
        blockIdx = dim3(x, y, z);
        t.run(b.x);
    }
}
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(k, g, b, s, st, ...) ((void)(st), host_blocks(#k, k, g, b, __VA_ARGS__))
