// The host stand-in of tests/host_requests with matrix products that may give NaN (what is done
// about an infinity then has addresses of its own).
#pragma once
#include "../../host_requests/hip/hip_runtime.h"
extern int host_nan;      // one product in so many, 0: none
inline host_v4f host_product(host_v4f c) {
    static unsigned n;
    if (host_nan && ++n % (unsigned)host_nan == 0) c[n / 7 % 4] = __builtin_nanf("");
    return c;
}
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, x, y, z) host_product(c)
