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

// The rows [t0, t1) of V channels of a sequence: W - 1 rows before them, then a
// step for each, kSteps rows loaded ahead.  The first `skip` channels belong to the
// thread before (the last V of a row whose width V does not divide): read and computed
// with the others (their state may be overwritten meanwhile), not stored.  NARROW: rows
// of fewer than V channels, element by element.
template <class T, int W, int V, bool NARROW>
__device__ __forceinline__ void conv_rows(const ConvArgs<T> &a, int64_t b, int c, int skip, int t0, int t1, int n) {
    constexpr int kSteps = 4;
    auto load = [&](const T *p) {
        Packed<T, V> v;
        if (!NARROW) {
            v = load_packed<V>(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = i < a.dim ? p[i] : (T)0.0f;
        }
        return v;
    };
    auto store = [&](T *p, const Packed<T, V> &v) {
        if (!NARROW && skip == 0) {
            store_packed<V>(p, v);
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i >= skip && (!NARROW || i < a.dim)) p[i] = v.v[i];
    };
    // row t of the sequence, the state in front of it
    auto row = [&](int t) {
        Packed<T, V> v;
        if (t >= 0) {
            v = load(a.x.row(b, t) + c);
        } else if (a.state_in) {
            v = load(a.state_in + (b * (W - 1) + (W - 1 + t)) * a.dim + c);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = (T)0.0f;
        }
        return v;
    };
    float w[W][V], bias[V], win[W][V];
    if (!NARROW) {
        // the channels' taps are adjacent: one run of 16-byte loads
        const Packed<float, V * W> wp = load_packed<V * W>(a.w + (int64_t)c * W);
        Packed<float, V> bp;
        if (a.bias) bp = load_packed<V>(a.bias + c);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            bias[i] = a.bias ? bp.v[i] : 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = wp.v[i * W + j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int ci = min(i, a.dim - 1);
            bias[i] = a.bias ? a.bias[ci] : 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = a.w[(int64_t)ci * W + j];
        }
    }
    const int end = min(t1, n);
    Packed<T, V> next[kSteps];
    if (t0 < end) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const Packed<T, V> r = row(t0 - (W - 1) + j);
#pragma unroll
            for (int i = 0; i < V; ++i) win[j][i] = (float)r.v[i];
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) next[s] = row(min(t0 + s, end - 1));
    }
    if (t0 == 0 && a.state_out) {
        // the thread that read state_in writes state_out, so the two may be one
        Packed<T, V> last[W];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) last[j] = row(n - (W - 1) + j);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store(a.state_out + (b * (W - 1) + j) * a.dim + c, last[j]);
    }
    for (int t = t0; t < end; t += kSteps) {
        Packed<T, V> now[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) now[s] = next[s];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) next[s] = load(a.x.row(b, min(t + kSteps + s, end - 1)) + c);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            Packed<T, V> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                win[W - 1][i] = (float)now[s].v[i];
                float y = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) y = __builtin_fmaf(w[j][i], win[j][i], y);
                o.v[i] = (T)(a.silu ? silu(y) : y);
#pragma unroll
                for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
            }
            if (t + s < end) store(a.y.row(b, t + s) + c, o);
        }
    }
    Packed<T, V> none;
#pragma unroll
    for (int i = 0; i < V; ++i) none.v[i] = (T)0.0f;
    for (int t = max(t0, n); t < t1; ++t) store(a.y.row(b, t) + c, none);
}

// One thread V channels (16 bytes) of `steps` rows of a sequence.
template <class T, int W, bool NARROW>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvArgs<T> a, int steps, int tiles, int64_t threads) {
    constexpr int V = 16 / sizeof(T);
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= threads) return;
    const int cols = (a.dim + V - 1) / V;
    const int64_t tile = id / cols;
    const int first = (int)(id - tile * cols) * V, c = NARROW ? 0 : min(first, a.dim - V);
    const int64_t b = tile / tiles;
    const int t0 = (int)(tile - b * tiles) * steps, t1 = min(a.len, t0 + steps);
    const int n = a.lens ? min(max(a.lens[b], 0), a.len) : a.len;
    conv_rows<T, W, V, NARROW>(a, b, c, first - c, t0, t1, n);
}

template <class T, int W>
mi_status launch_conv(const ConvArgs<T> &a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int64_t cols = (a.dim + V - 1) / V, rows = (int64_t)a.batch * cols;
    // rows a thread: the W - 1 in front of them are read twice, so as many as leave
    // four waves a SIMD; at least W - 1, so that only the first rows' thread, which writes
    // state_out, reads state_in
    int steps = 32;
    while (steps > (W <= 5 ? 4 : 8) && rows * ((a.len + steps - 1) / steps) < (int64_t)device_cus() * 4 * 4 * 64) steps /= 2;
    const int tiles = a.len > 0 ? (a.len + steps - 1) / steps : 1;
    const int64_t threads = rows * tiles;
    MI_REQUIRE(threads < ((int64_t)1 << 32) - 256, MI_ERR_BAD_DIM, "mi_causal_conv: batch * len * dim is too large");
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (a.dim < V)
        hipLaunchKernelGGL((causal_conv_kernel<T, W, true>), grid, dim3(256), 0, st, a, steps, tiles, threads);
    else
        hipLaunchKernelGGL((causal_conv_kernel<T, W, false>), grid, dim3(256), 0, st, a, steps, tiles, threads);
    return MI_OK;
}

template <class T>
mi_status launch_width(const ConvArgs<T> &a, hipStream_t st) {
    switch (a.width) {
        case 1: return launch_conv<T, 1>(a, st);
        case 2: return launch_conv<T, 2>(a, st);
        case 3: return launch_conv<T, 3>(a, st);
        case 4: return launch_conv<T, 4>(a, st);
        case 5: return launch_conv<T, 5>(a, st);
        case 6: return launch_conv<T, 6>(a, st);
        case 7: return launch_conv<T, 7>(a, st);
        default: return launch_conv<T, 8>(a, st);
    }
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
    MI_REQUIRE((int64_t)batch * dim < ((int64_t)1 << 31) && len <= 1 << 30, MI_ERR_BAD_DIM,
               "mi_causal_conv: batch * dim must be below 2^31, and len at most 2^30");
    if (batch == 0 || dim == 0) return MI_OK;
    MI_REQUIRE(w && (len == 0 || (x && y)), MI_ERR_NULL_POINTER, "mi_causal_conv: x, w and y are required");
    const hipStream_t st = as_stream(stream);
    mi_status status = MI_OK;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        const ConvArgs<T> a{{static_cast<const T *>(x), ldx, bsx}, w, bias, static_cast<const T *>(state_in),
                            static_cast<T *>(state_out), lens, {static_cast<T *>(y), ldy, bsy}, width, silu, batch, len,
                            dim};
        status = launch_width(a, st);
    });
    return status != MI_OK ? status : check_launch("mi_causal_conv");
}
