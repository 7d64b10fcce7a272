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

constexpr int kNormMaxDim = 16384;   // 8 vectors of 16 bits a thread, 16 of 32 bits

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

// The row's 8-bit values and their scale from max |y| (its bits): y * 127 / max
// plus 1.5 * 2^23 has the value, rounded half to even, in its low byte.  (No clamp:
// |y| <= max, so the product rounds to 127 at most.)
struct NormQuant {
    float mul, scale;
    __device__ __forceinline__ explicit NormQuant(uint32_t bits) {
        const float amax = __builtin_bit_cast(float, bits);
        const float top = amax < 1e-8f ? 1e-8f : amax;
        mul = __fdiv_rn(127.0f, top);
        scale = __fdiv_rn(top, 127.0f);
    }
    __device__ __forceinline__ int8_t operator()(float y) const {
        return (int8_t)__builtin_bit_cast(int32_t, __fadd_rn(__fmul_rn(y, mul), 12582912.0f));
    }
};

// TPR threads a row, E times V adjacent elements each: every load is issued
// before the sum.  Rows of V elements at least; the last V of a row whose width
// V does not divide start at dim - V (elements of two threads are summed once and
// stored twice with one value).
template <class T, class R, int TPR, int E>
__global__ __launch_bounds__(256) void add_rms_norm_kernel(NormArgs a) {
    constexpr int V = 16 / sizeof(T);
    __shared__ float red_s[TPR / 64];
    __shared__ uint32_t red_m[TPR / 64];
    const int64_t row = TPR == 64 ? (int64_t)blockIdx.x * 4 + wave_id() : (int64_t)blockIdx.x;
    const int tid = TPR == 64 ? threadIdx.x & 63 : threadIdx.x;
    if (row >= a.rows) return;
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    const int dim = a.dim;
    int at[E];
    Packed<T, V> xv[E];
    Packed<R, V> rv[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
        at[j] = min((tid + j * TPR) * V, dim - V);
        xv[j] = load_packed<V>(x + at[j]);
    }
    if (a.res) {
        const R *res = static_cast<const R *>(a.res) + row * a.ldr;
#pragma unroll
        for (int j = 0; j < E; ++j) rv[j] = load_packed<V>(res + at[j]);
    }
    float v[E][V], ss = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int first = (tid + j * TPR) * V;   // elements below it belong to another thread
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[j][i] = (float)xv[j].v[i];
            if (a.res) v[j][i] += (float)rv[j].v[i];
            ss += at[j] + i >= first ? v[j][i] * v[j][i] : 0.0f;
        }
    }
    const float inv = 1.0f / sqrtf(block_sum<TPR>(ss, red_s) / (float)dim + a.eps);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        if ((tid + j * TPR) * V >= dim) break;
        if (a.res_out) {
            Packed<R, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = (R)v[j][i];
            store_packed<V>(static_cast<R *>(a.res_out) + row * a.ldro + at[j], o);
        }
        const Packed<float, V> w = load_packed<V>(a.w + at[j]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[j][i] = v[j][i] * inv * w.v[i];
            m = max(m, __builtin_bit_cast(uint32_t, v[j][i]) & 0x7fffffffu);
        }
        if (a.y) {
            Packed<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) o.v[i] = (T)v[j][i];
            store_packed<V>(static_cast<T *>(a.y) + row * a.ldy + at[j], o);
        }
    }
    if (!a.q) return;
    const NormQuant quant(block_max<TPR>(m, red_m));
    int8_t *q = a.q + row * a.ldq;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        if ((tid + j * TPR) * V >= dim) break;
        Packed<int8_t, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = quant(v[j][i]);
        store_packed<V>(q + at[j], o);
    }
    for (int64_t i = dim + tid; i < a.ldq; i += TPR) q[i] = 0;
    if (tid == 0) a.scale[row] = quant.scale;
}

// Rows narrower than one thread's vector: one thread a row.
template <class T, class R>
__global__ __launch_bounds__(64) void add_rms_norm_narrow_kernel(NormArgs a) {
    const int64_t row = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (row >= a.rows) return;
    float v[8], ss = 0.0f;
    for (int i = 0; i < a.dim; ++i) {
        v[i] = (float)static_cast<const T *>(a.x)[row * a.ldx + i];
        if (a.res) v[i] += (float)static_cast<const R *>(a.res)[row * a.ldr + i];
        ss += v[i] * v[i];
    }
    const float inv = 1.0f / sqrtf(ss / (float)a.dim + a.eps);
    uint32_t m = 0;
    for (int i = 0; i < a.dim; ++i) {
        if (a.res_out) static_cast<R *>(a.res_out)[row * a.ldro + i] = (R)v[i];
        v[i] = v[i] * inv * a.w[i];
        m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
        if (a.y) static_cast<T *>(a.y)[row * a.ldy + i] = (T)v[i];
    }
    if (!a.q) return;
    const NormQuant quant(m);
    for (int64_t i = 0; i < a.ldq; ++i) a.q[row * a.ldq + i] = i < a.dim ? quant(v[i]) : (int8_t)0;
    a.scale[row] = quant.scale;
}

template <class T, class R, int TPR, int E>
void launch_rows(const NormArgs &a, hipStream_t st) {
    const int64_t blocks = TPR == 64 ? (a.rows + 3) / 4 : a.rows;
    hipLaunchKernelGGL((add_rms_norm_kernel<T, R, TPR, E>), dim3((unsigned)blocks), dim3(256), 0, st, a);
}

// A wave a row while a lane holds at most 32 elements, then a block a row (up to 64 a thread).
template <class T, class R>
void launch_add_rms_norm(const NormArgs &a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int e = (a.dim + 64 * V - 1) / (64 * V);
    if (a.dim < V)
        hipLaunchKernelGGL((add_rms_norm_narrow_kernel<T, R>), dim3((unsigned)((a.rows + 63) / 64)), dim3(64), 0, st, a);
    else if (e <= 1)
        launch_rows<T, R, 64, 1>(a, st);
    else if (e <= 2)
        launch_rows<T, R, 64, 2>(a, st);
    else if (e <= 3)
        launch_rows<T, R, 64, 3>(a, st);
    else if (e <= 4)
        launch_rows<T, R, 64, 4>(a, st);
    else if (e <= 8)
        launch_rows<T, R, V == 4 ? 64 : 256, V == 4 ? 8 : 2>(a, st);
    else if (e <= 16)
        launch_rows<T, R, 256, 4>(a, st);
    else if (V == 8 || e <= 32)
        launch_rows<T, R, 256, 8>(a, st);
    else if constexpr (V == 4)
        launch_rows<T, R, 256, 16>(a, st);
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
