// Element types, argument checks and float formulas of the float operators
// (norm.hip, conv.hip, selective_scan.hip, w4.hip).
#pragma once

#include "mi_common.hpp"

namespace mi {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

inline bool known_type(int t) { return t == MI_F32 || t == MI_BF16 || t == MI_F16; }

// Calls f with a value of the element type's C++ type.
template <class F>
void with_type(int type, F &&f) {
    if (type == MI_F32)
        f(float{});
    else if (type == MI_BF16)
        f(bf16_t{});
    else
        f(f16_t{});
}

// V elements with any alignment of the type's own (global memory takes wide loads
// and stores at every element's address).
template <class T, int V>
struct __attribute__((packed)) Packed {
    T v[V];
};
template <int V, class T>
__device__ __forceinline__ Packed<T, V> load_packed(const T *p) {
    return *reinterpret_cast<const Packed<T, V> *>(p);
}
template <int V, class T>
__device__ __forceinline__ void store_packed(T *p, const Packed<T, V> &v) {
    *reinterpret_cast<Packed<T, V> *>(p) = v;
}

// A tensor of rows [batch, len, dim]: the address of row (b, t).
template <class T>
struct Rows {
    T *p;
    int64_t ld, bs;   // elements from a row to the next, from a sequence to the next
    __device__ __forceinline__ T *row(int64_t b, int64_t t) const { return p + b * bs + t * ld; }
};

// v / (1 + exp(-v)); -0 where exp(-v) overflows (the value is below 1e-36 there).
__device__ __forceinline__ float silu(float v) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}

}  // namespace mi
