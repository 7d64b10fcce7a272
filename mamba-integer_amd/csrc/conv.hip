// Short depthwise causal convolution of float rows, over prompts and single
// tokens, with the last inputs carried as a state.
//
//   y[b,t,c] = act(bias[c] + sum_j w[c,j] * x[b, t - width + 1 + j, c])
//
// x before the sequence comes from state_in (zeros without one).
#include "float_ops.hpp"

namespace mi {

constexpr int kConvMaxWidth = 8;

template <class T>
struct ConvArgs {
    Rows<const T> x;
    const float *w, *bias;
    const T *state_in;
    T *state_out;
    const int32_t *lens;
    Rows<T> y;
    int width, silu, batch, len, dim;
};

template <class T>
__device__ __forceinline__ int seq_len(const int32_t *lens, int64_t b, int len) {
    return lens ? min(max(lens[b], 0), len) : len;
}

// One thread a (sequence, channel), step after step.
template <class T>
__global__ __launch_bounds__(64) void causal_conv_kernel(ConvArgs<T> a) {
    const int64_t id = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (id >= (int64_t)a.batch * a.dim) return;
    const int64_t b = id / a.dim;
    const int c = (int)(id - b * a.dim), W = a.width;
    const int n = seq_len<T>(a.lens, b, a.len);
    float win[kConvMaxWidth];
    for (int j = 0; j < W - 1; ++j) win[j] = a.state_in ? (float)a.state_in[(b * (W - 1) + j) * a.dim + c] : 0.0f;
    const float bias = a.bias ? a.bias[c] : 0.0f;
    for (int t = 0; t < n; ++t) {
        win[W - 1] = (float)a.x.row(b, t)[c];
        float s = bias;
        for (int j = 0; j < W; ++j) s = __builtin_fmaf(a.w[(int64_t)c * W + j], win[j], s);
        a.y.row(b, t)[c] = (T)(a.silu ? silu(s) : s);
        for (int j = 0; j < W - 1; ++j) win[j] = win[j + 1];
    }
    for (int t = n; t < a.len; ++t) a.y.row(b, t)[c] = (T)0.0f;
    if (a.state_out)
        for (int j = 0; j < W - 1; ++j) a.state_out[(b * (W - 1) + j) * a.dim + c] = (T)win[j];
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_causal_conv(const void *x, int64_t ldx, int64_t bsx, int type, const float *w, const float *bias,
                                    int width, int silu, const void *state_in, void *state_out, const int32_t *lens,
                                    void *y, int64_t ldy, int64_t bsy, int batch, int len, int dim, void *stream) {
    clear_error();
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0, MI_ERR_BAD_DIM, "mi_causal_conv: negative size");
    MI_REQUIRE(width >= 1 && width <= kConvMaxWidth, MI_ERR_BAD_ARG, "mi_causal_conv: width=%d must be in [1, %d]", width,
               kConvMaxWidth);
    MI_REQUIRE(known_type(type), MI_ERR_BAD_ARG, "mi_causal_conv: unknown element type %d", type);
    MI_REQUIRE(ldx >= 0 && bsx >= 0 && ldy >= dim && bsy >= 0, MI_ERR_BAD_DIM,
               "mi_causal_conv: a stride is negative, or ldy is less than dim");
    MI_REQUIRE((int64_t)batch * dim < ((int64_t)1 << 31), MI_ERR_BAD_DIM, "mi_causal_conv: batch * dim must be below 2^31");
    if (batch == 0 || dim == 0) return MI_OK;
    MI_REQUIRE(w && (len == 0 || (x && y)), MI_ERR_NULL_POINTER, "mi_causal_conv: x, w and y are required");
    const hipStream_t st = as_stream(stream);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const ConvArgs<T> a{{static_cast<const T *>(x), ldx, bsx}, w, bias, static_cast<const T *>(state_in),
                            static_cast<T *>(state_out), lens, {static_cast<T *>(y), ldy, bsy}, width, silu, batch, len,
                            dim};
        const int64_t n = (int64_t)batch * dim;
        hipLaunchKernelGGL(causal_conv_kernel<T>, dim3((unsigned)((n + 63) / 64)), dim3(64), 0, st, a);
    });
    return check_launch("mi_causal_conv");
}
