// Selective state space scan of float rows, over prompts and single tokens:
//
//   d = softplus(dt[b,t,c] + dt_bias[c])
//   h[n] = exp(d * a[c,n]) * h[n] + d * u[b,t,c] * B[b,t,g,n]
//   y[b,t,c] = (sum_n C[b,t,g,n] * h[n] + d_skip[c] * u[b,t,c]) * silu(z[b,t,c])
//
// with g = c / (dim / groups) and h in 32 bits.
#include "float_ops.hpp"

namespace mi {

constexpr int kScanMaxStates = 256;

template <class T>
struct ScanArgs {
    Rows<const T> u, dt, b, c, z;
    const float *a, *d_skip, *dt_bias, *h_in;
    float *h_out;
    const int32_t *lens;
    Rows<T> y;
    int softplus, batch, len, dim, nstate, groups;
};

__device__ __forceinline__ int scan_len(const int32_t *lens, int64_t b, int len) {
    return lens ? min(max(lens[b], 0), len) : len;
}

// log(1 + exp(v)) = max(v, 0) + log(w) + (e - (w - 1)) with e = exp(-|v|), w = 1 + e
// rounded: the last term is what the rounding of w lost (1 / w of it, and w = 1
// wherever it matters), so small steps keep their relative precision.
__device__ __forceinline__ float softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(v));
    const float w = 1.0f + e;
    const float s = 0.693147181f * __builtin_amdgcn_logf(w) + (e - (w - 1.0f));
    return v > 0.0f ? v + s : (v <= 0.0f ? s : v);
}

// LANES lanes of a wave hold a channel, four states each (adjacent: 16-byte loads
// of the state, of A and of B and C's rows where N % 4 == 0); step after step.
template <class T, int LANES, bool QUADS>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs<T> a) {
    const uint32_t id = (blockIdx.x * 256 + threadIdx.x) / LANES, all = (uint32_t)a.batch * (uint32_t)a.dim;
    const int lane = threadIdx.x % LANES, N = a.nstate, n0 = 4 * lane;
    const bool on = id < all;
    const uint32_t ch = on ? id : all - 1;
    const uint32_t b = ch / (uint32_t)a.dim;
    const int c = (int)(ch - b * (uint32_t)a.dim);
    const int64_t g0 = (int64_t)(c / (a.dim / a.groups)) * N + n0;
    const int len = scan_len(a.lens, b, a.len);
    // four values from p on, those of states past N as zero
    auto four = [&](auto *p, float (&o)[4]) {
        if (QUADS) {
            if (n0 < N) {
                const auto v = load_packed<4>(p);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = (float)v.v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + i < N) o[i] = (float)p[i];
        }
    };
    float h[4] = {}, am[4] = {};
    four(a.a + (int64_t)c * N + n0, am);
    if (a.h_in) four(a.h_in + (int64_t)ch * N + n0, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) am[i] *= 1.44269504f;
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f, skip = a.d_skip ? a.d_skip[c] : 0.0f;
    for (int t = 0; t < len; ++t) {
        float bn[4] = {}, cn[4] = {};
        four(a.b.row(b, t) + g0, bn);
        four(a.c.row(b, t) + g0, cn);
        const float u = (float)a.u.row(b, t)[c];
        float dt = (float)a.dt.row(b, t)[c] + bias;
        if (a.softplus) dt = softplus(dt);
        const float du = dt * u;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * am[i]), h[i], du * bn[i]);
            if (n0 + i < N) y = __builtin_fmaf(cn[i], h[i], y);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) y += __shfl_xor(y, o);
        y = __builtin_fmaf(skip, u, y);
        if (a.z.p) y *= silu((float)a.z.row(b, t)[c]);
        if (on && lane == 0) a.y.row(b, t)[c] = (T)y;
    }
    if (!on) return;
    if (lane == 0)
        for (int t = len; t < a.len; ++t) a.y.row(b, t)[c] = (T)0.0f;
    if (!a.h_out) return;
    float *h_out = a.h_out + (int64_t)ch * N + n0;
    if (QUADS) {
        if (n0 < N) store_packed<4>(h_out, Packed<float, 4>{{h[0], h[1], h[2], h[3]}});
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < N) h_out[i] = h[i];
    }
}

template <class T, int LANES>
void launch_scan_step(const ScanArgs<T> &a, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.batch * a.dim * LANES + 255) / 256));
    if (a.nstate % 4 == 0)
        hipLaunchKernelGGL((scan_step_kernel<T, LANES, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((scan_step_kernel<T, LANES, false>), grid, dim3(256), 0, st, a);
}

template <class T>
void launch_scan(const ScanArgs<T> &a, hipStream_t st) {
    if (a.nstate <= 4)
        launch_scan_step<T, 1>(a, st);
    else if (a.nstate <= 8)
        launch_scan_step<T, 2>(a, st);
    else if (a.nstate <= 16)
        launch_scan_step<T, 4>(a, st);
    else if (a.nstate <= 32)
        launch_scan_step<T, 8>(a, st);
    else if (a.nstate <= 64)
        launch_scan_step<T, 16>(a, st);
    else if (a.nstate <= 128)
        launch_scan_step<T, 32>(a, st);
    else
        launch_scan_step<T, 64>(a, st);
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_selective_scan_workspace_size(int batch, int len, int dim, int nstate, size_t *bytes) {
    clear_error();
    MI_REQUIRE(bytes, MI_ERR_NULL_POINTER, "mi_selective_scan_workspace_size: bytes is required");
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0 && nstate >= 1 && nstate <= kScanMaxStates, MI_ERR_BAD_DIM,
               "mi_selective_scan_workspace_size: a size is negative, or nstate=%d not in [1, %d]", nstate, kScanMaxStates);
    *bytes = 0;
    return MI_OK;
}

extern "C" mi_status mi_selective_scan(const void *u, int64_t ldu, int64_t bsu, const void *dt, int64_t ldt, int64_t bst,
                                       const float *a, const void *b, int64_t ldb, int64_t bsb, const void *c,
                                       int64_t ldc, int64_t bsc, const float *d_skip, const void *z, int64_t ldz,
                                       int64_t bsz, const float *dt_bias, int dt_softplus, const float *h_in,
                                       float *h_out, const int32_t *lens, void *y, int64_t ldy, int64_t bsy, int type,
                                       int batch, int len, int dim, int nstate, int groups, void *workspace,
                                       size_t workspace_bytes, void *stream) {
    clear_error();
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0, MI_ERR_BAD_DIM, "mi_selective_scan: negative size");
    MI_REQUIRE(nstate >= 1 && nstate <= kScanMaxStates, MI_ERR_BAD_DIM, "mi_selective_scan: nstate=%d must be in [1, %d]",
               nstate, kScanMaxStates);
    MI_REQUIRE(groups >= 1 && dim % groups == 0, MI_ERR_BAD_DIM, "mi_selective_scan: groups=%d must divide dim=%d", groups,
               dim);
    MI_REQUIRE(known_type(type), MI_ERR_BAD_ARG, "mi_selective_scan: unknown element type %d", type);
    MI_REQUIRE(ldu >= 0 && ldt >= 0 && ldb >= 0 && ldc >= 0 && ldz >= 0 && bsu >= 0 && bst >= 0 && bsb >= 0 && bsc >= 0 &&
                   bsz >= 0 && ldy >= dim && bsy >= 0,
               MI_ERR_BAD_DIM, "mi_selective_scan: a stride is negative, or ldy is less than dim");
    MI_REQUIRE((int64_t)batch * dim <= ((int64_t)1 << 25), MI_ERR_BAD_DIM,
               "mi_selective_scan: batch * dim must be at most 2^25");
    if (batch == 0 || dim == 0) return MI_OK;
    MI_REQUIRE(a && (len == 0 || (u && dt && b && c && y)), MI_ERR_NULL_POINTER,
               "mi_selective_scan: u, dt, a, b, c and y are required");
    size_t need = 0;
    mi_selective_scan_workspace_size(batch, len, dim, nstate, &need);
    MI_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG,
               "mi_selective_scan: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
    const hipStream_t st = as_stream(stream);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto in = [](const void *p, int64_t ld, int64_t bs) { return Rows<const T>{static_cast<const T *>(p), ld, bs}; };
        launch_scan<T>({in(u, ldu, bsu), in(dt, ldt, bst), in(b, ldb, bsb), in(c, ldc, bsc), in(z, ldz, bsz), a, d_skip,
                        dt_bias, h_in, h_out, lens, {static_cast<T *>(y), ldy, bsy}, dt_softplus, batch, len, dim, nstate,
                        groups},
                       st);
    });
    return check_launch("mi_selective_scan");
}
