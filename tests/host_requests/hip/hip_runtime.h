// The host stand-in of tests/host_float with what the gated recurrence's and the adapters'
// kernels use beside it.  Blocks run one after another, so a word that a block waits for has
// been written by then.
#pragma once
#include "../../host_float/hip/hip_runtime.h"
#define __HIP_MEMORY_SCOPE_AGENT 4
inline void __builtin_amdgcn_s_sleep(int) { host_die("a wait for a word that no block before has written", 0, 0); }
inline float __builtin_amdgcn_rsqf(float v) { return 1.0f / sqrtf(v); }
