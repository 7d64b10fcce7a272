// The host stand-in of tests/host_kernels with what the float operators' kernels use
// beside it.  Results mean nothing; addresses are the kernels' own.
#pragma once
#include "../../host_kernels/hip/hip_runtime.h"
#include <algorithm>
struct float2 { float x, y; } __attribute__((aligned(8)));
typedef float host_v4f __attribute__((ext_vector_type(4)));
typedef __bf16 host_v8b __attribute__((ext_vector_type(8)));
typedef _Float16 host_v8h __attribute__((ext_vector_type(8)));
inline float __builtin_amdgcn_exp2f(float v) { return exp2f(v); }
inline float __builtin_amdgcn_logf(float v) { return log2f(v); }
inline host_v4f __builtin_amdgcn_mfma_f32_16x16x32_bf16(host_v8b, host_v8b, host_v4f c, int, int, int) { return c; }
inline host_v4f __builtin_amdgcn_mfma_f32_16x16x32_f16(host_v8h, host_v8h, host_v4f c, int, int, int) { return c; }
