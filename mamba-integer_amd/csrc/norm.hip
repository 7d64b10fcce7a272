// Residual addition and root-mean-square norm of float rows, with a float
// output, an 8-bit one with a scale a row, or both.
//
//   s = residual + x,  r = s in the residual's type,  y = s / sqrt(mean(s^2) + eps) * w
//   scale = max(max |y|, 1e-8) / 127,  q = round(y * 127 / max(max |y|, 1e-8))
//
// The row is read once: s stays in registers in 32 bits (unrounded, whatever
// the residual's type) between the sum of squares, the maximum and the outputs.
#include "float_ops.hpp"

namespace mi {

constexpr int kNormMaxDim = 16384;

struct NormArgs {
    const void *x, *res;
    const float *w;
    void *y, *res_out;
    int8_t *q;
    float *scale;
    int64_t ldx, ldr, ldy, ldq, ldro;
    int64_t rows;
    int dim;
    float eps;
};

// Over the block's threads: the sum of v, or the maximum of v as unsigned
// (the bits of |y| order as the values do, with inf and NaN on top, so a NaN
// of any element reaches the scale).
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float *red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (THREADS == 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < THREADS / 64; ++i) s += red[i];
    return s;
}
template <int THREADS>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t *red) {
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    if (THREADS == 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t s = 0;
    for (int i = 0; i < THREADS / 64; ++i) s = max(s, red[i]);
    return s;
}

// One block a row, one element a thread and step.
template <class T, class R, int THREADS, int E>
__global__ __launch_bounds__(THREADS) void add_rms_norm_kernel(NormArgs a) {
    __shared__ float red_s[THREADS / 64];
    __shared__ uint32_t red_m[THREADS / 64];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const R *res = a.res ? static_cast<const R *>(a.res) + row * a.ldr : nullptr;
    float v[E], ss = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int i = tid + j * THREADS;
        v[j] = 0.0f;
        if (i < a.dim) {
            v[j] = (float)x[i];
            if (res) v[j] = (float)res[i] + v[j];
            ss += v[j] * v[j];
        }
    }
    const float inv = 1.0f / sqrtf(block_sum<THREADS>(ss, red_s) / (float)a.dim + a.eps);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int i = tid + j * THREADS;
        if (i >= a.dim) break;
        if (a.res_out) static_cast<R *>(a.res_out)[row * a.ldro + i] = (R)v[j];
        v[j] = v[j] * inv * a.w[i];
        if (a.y) static_cast<T *>(a.y)[row * a.ldy + i] = (T)v[j];
        m = max(m, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
    }
    if (!a.q) return;
    m = block_max<THREADS>(m, red_m);
    const float amax = __builtin_bit_cast(float, m);
    const float top = amax < 1e-8f ? 1e-8f : amax;
    const float mul = 127.0f / top;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int i = tid + j * THREADS;
        if (i < a.dim)
            a.q[row * a.ldq + i] = (int8_t)fminf(fmaxf(rintf(v[j] * mul), -127.0f), 127.0f);
        else if (i < a.ldq)
            a.q[row * a.ldq + i] = 0;
    }
    for (int64_t i = tid + E * THREADS; i < a.ldq; i += THREADS) a.q[row * a.ldq + i] = 0;
    if (tid == 0) a.scale[row] = top / 127.0f;
}

template <class T, class R>
void launch_add_rms_norm(const NormArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.rows);
    if (a.dim <= 2048)
        hipLaunchKernelGGL((add_rms_norm_kernel<T, R, 256, 8>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((add_rms_norm_kernel<T, R, 1024, 16>), grid, dim3(1024), 0, st, a);
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_add_rms_norm(const void *x, int x_type, int64_t ldx, const void *residual, int res_type,
                                     int64_t ldr, const float *weight, float eps, void *y, int64_t ldy, int8_t *q,
                                     int64_t ldq, float *scale, void *res_out, int64_t ldro, int tokens, int dim,
                                     void *stream) {
    clear_error();
    MI_REQUIRE(tokens >= 0, MI_ERR_BAD_DIM, "mi_add_rms_norm: negative tokens");
    MI_REQUIRE(dim >= 1 && dim <= kNormMaxDim, MI_ERR_BAD_DIM, "mi_add_rms_norm: dim=%d must be in [1, %d]", dim,
               kNormMaxDim);
    MI_REQUIRE(known_type(x_type) && known_type(res_type), MI_ERR_BAD_ARG, "mi_add_rms_norm: unknown element type");
    MI_REQUIRE(res_type == x_type || res_type == MI_F32, MI_ERR_BAD_ARG,
               "mi_add_rms_norm: the residual has x's type or MI_F32");
    MI_REQUIRE(eps >= 0.0f, MI_ERR_BAD_ARG, "mi_add_rms_norm: eps must not be negative");
    MI_REQUIRE(ldx >= 0 && ldr >= 0 && (!y || ldy >= dim) && (!res_out || ldro >= dim), MI_ERR_BAD_DIM,
               "mi_add_rms_norm: a row stride is negative, or an output's is less than dim");
    MI_REQUIRE(!q || (ldq >= dim && ldq <= 2 * kNormMaxDim), MI_ERR_BAD_DIM, "mi_add_rms_norm: ldq must be in [dim, %d]",
               2 * kNormMaxDim);
    MI_REQUIRE(tokens < (1 << 22), MI_ERR_BAD_DIM, "mi_add_rms_norm: tokens=%d must be below %d", tokens, 1 << 22);
    if (tokens == 0) return MI_OK;
    MI_REQUIRE(x && weight && (y || q), MI_ERR_NULL_POINTER, "mi_add_rms_norm: x, weight and y or q are required");
    MI_REQUIRE(!q || scale, MI_ERR_NULL_POINTER, "mi_add_rms_norm: q needs scale");
    const NormArgs a{x, residual, weight, y, res_out, q, scale, ldx, ldr, ldy, ldq, ldro, tokens, dim, eps};
    const hipStream_t st = as_stream(stream);
    with_type(x_type, [&](auto t) {
        using T = decltype(t);
        if (res_type == MI_F32)
            launch_add_rms_norm<T, float>(a, st);
        else
            launch_add_rms_norm<T, T>(a, st);
    });
    return check_launch("mi_add_rms_norm");
}
