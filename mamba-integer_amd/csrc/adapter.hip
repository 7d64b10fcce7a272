// Low-rank adapters beside a shared projection, each sequence with its own of a bank:
//
//   out[b,t,:] = y[b,t,:] + scale[id] * x_scale[b,t] * (x[b,t,:] A[id]^T) B[id]^T,  id = ids[b]
//
// in two kernels: t = x A^T in 32 bits into the workspace, then out = y + t B^T, the sum
// rounded once to out's type.
#include "float_ops.hpp"

namespace mi {

constexpr int kAdapterMaxRank = 128;

struct AdapterArgs {
    const void *x, *y;
    void *out;
    int64_t ldx, bsx, ldy, bsy, ldo, bso;
    const float *x_scale;      // [batch, len]
    const void *a, *b;         // [bank, rank, k], [bank, n, rank]
    const float *scales;       // [bank]
    const int32_t *ids, *lens;
    float *t;                  // [batch, len, rank]
    int batch, len, k, n, rank, bank;
};

// The adapter of a sequence, -1 for none; tokens of it.
__device__ __forceinline__ int adapter_of(const AdapterArgs &a, int b) {
    const int id = a.ids[b];
    return (unsigned)id < (unsigned)a.bank ? id : -1;
}
__device__ __forceinline__ int tokens_of(const AdapterArgs &a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.len) : a.len;
}

// A wave a (row, rank): the row's products with one row of A.
template <class X, class W>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a) {
    const int64_t row = blockIdx.x;
    const int b = (int)(row / a.len), t = (int)(row % a.len), lane = threadIdx.x & 63;
    const int id = adapter_of(a, b);
    if (id < 0 || t >= tokens_of(a, b)) return;
    const X *x = static_cast<const X *>(a.x) + b * a.bsx + t * a.ldx;
    for (int j = wave_id(); j < a.rank; j += 4) {
        const W *w = static_cast<const W *>(a.a) + ((int64_t)id * a.rank + j) * a.k;
        float s = 0.0f;
        for (int i = lane; i < a.k; i += 64) s = __builtin_fmaf((float)x[i], (float)w[i], s);
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (a.scales) s *= a.scales[id];
        if (a.x_scale) s *= a.x_scale[row];
        if (lane == 0) a.t[row * a.rank + j] = s;
    }
}

// A thread an output.
template <class Y, class W>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a) {
    const int64_t row = blockIdx.x;
    const int b = (int)(row / a.len), t = (int)(row % a.len);
    const int id = adapter_of(a, b);
    const bool on = id >= 0 && t < tokens_of(a, b);
    if (!on && a.out == a.y) return;
    const Y *y = static_cast<const Y *>(a.y) + b * a.bsy + t * a.ldy;
    Y *out = static_cast<Y *>(a.out) + b * a.bso + t * a.ldo;
    const int n = blockIdx.y * 256 + threadIdx.x;
    if (n >= a.n) return;
    if (!on) {
        out[n] = y[n];
        return;
    }
    const W *w = static_cast<const W *>(a.b) + ((int64_t)id * a.n + n) * a.rank;
    float s = (float)y[n];
    float d = 0.0f;
    for (int j = 0; j < a.rank; ++j) d = __builtin_fmaf(a.t[row * a.rank + j], (float)w[j], d);
    out[n] = (Y)(s + d);
}

// Calls f with values of the types of x, of y and of the weights.
template <class F>
void with_adapter_types(int x_type, int y_type, int w_type, F &&f) {
    with_type(w_type, [&](auto w) {
        if (x_type == MI_I8)
            with_type(y_type, [&](auto y) { f(int8_t{}, y, w); });
        else
            with_type(x_type, [&](auto x) { f(x, x, w); });
    });
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_adapter_workspace_size(int batch, int len, int rank, size_t *bytes) {
    clear_error();
    MI_REQUIRE(bytes, MI_ERR_NULL_POINTER, "mi_adapter_workspace_size: bytes is required");
    MI_REQUIRE(batch >= 0 && len >= 0 && rank >= 0 && rank <= kAdapterMaxRank, MI_ERR_BAD_DIM,
               "mi_adapter_workspace_size: a size is negative, or rank=%d above %d", rank, kAdapterMaxRank);
    MI_REQUIRE((int64_t)batch * len < (1 << 22), MI_ERR_BAD_DIM, "mi_adapter_workspace_size: batch * len must be below %d", 1 << 22);
    *bytes = ((size_t)batch * len * rank * sizeof(float) + 15) / 16 * 16;
    return MI_OK;
}

extern "C" mi_status mi_adapter_add(const void *x, int x_type, int64_t ldx, int64_t bsx, const float *x_scale, const void *a,
                                    const void *b, int weight_type, const float *scales, const int32_t *ids,
                                    const int32_t *lens, const void *y, int64_t ldy, int64_t bsy, void *out, int64_t ldo,
                                    int64_t bso, int type, int batch, int len, int k, int n, int rank, int bank,
                                    void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    MI_REQUIRE(batch >= 0 && len >= 0 && n >= 0, MI_ERR_BAD_DIM, "mi_adapter_add: a size is negative");
    MI_REQUIRE(k >= 0 && k <= (1 << 23) && n <= (1 << 23), MI_ERR_BAD_DIM, "mi_adapter_add: k=%d and n=%d must be in [0, %d]", k, n,
               1 << 23);
    MI_REQUIRE(rank >= 0 && rank <= kAdapterMaxRank, MI_ERR_BAD_DIM, "mi_adapter_add: rank=%d must be in [0, %d]", rank,
               kAdapterMaxRank);
    MI_REQUIRE(bank >= 0, MI_ERR_BAD_DIM, "mi_adapter_add: negative bank");
    MI_REQUIRE((int64_t)batch * len < (1 << 22), MI_ERR_BAD_DIM, "mi_adapter_add: batch * len must be below %d", 1 << 22);
    MI_REQUIRE(known_type(type) && known_type(weight_type) && (x_type == MI_I8 || x_type == type), MI_ERR_BAD_ARG,
               "mi_adapter_add: unknown element type, or x neither MI_I8 nor y's");
    MI_REQUIRE((x_type == MI_I8) == (x_scale != nullptr), MI_ERR_BAD_ARG, "mi_adapter_add: x_scale goes with 8-bit rows");
    MI_REQUIRE(ldx >= 0 && bsx >= 0 && ldy >= 0 && bsy >= 0, MI_ERR_BAD_DIM, "mi_adapter_add: a stride is negative");
    MI_REQUIRE(ldo >= n && bso >= 0, MI_ERR_BAD_DIM, "mi_adapter_add: ldo=%lld must be at least n", (long long)ldo);
    if (batch == 0 || len == 0 || n == 0) return MI_OK;
    MI_REQUIRE(y && out && ids, MI_ERR_NULL_POINTER, "mi_adapter_add: y, out and ids are required");
    MI_REQUIRE(out != y || (ldo == ldy && bso == bsy), MI_ERR_BAD_ARG, "mi_adapter_add: in place, out has y's strides");
    const AdapterArgs args{x, y, out, ldx, bsx, ldy, bsy, ldo, bso, x_scale, a, b, scales, ids, lens,
                           static_cast<float *>(workspace), batch, len, k, n, k ? rank : 0, bank};
    const bool work = args.rank && bank;
    if (!work && out == y) return MI_OK;
    MI_REQUIRE(!work || (x && a && b), MI_ERR_NULL_POINTER, "mi_adapter_add: x, a and b are required");
    size_t need = 0;
    mi_adapter_workspace_size(batch, len, args.rank, &need);
    MI_REQUIRE(!work || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG, "mi_adapter_add: the workspace has %zu bytes, %zu are needed",
               workspace_bytes, need);
    MI_REQUIRE(!work || aligned(workspace, 16), MI_ERR_BAD_ALIGNMENT, "mi_adapter_add: the workspace must be 16-byte aligned");
    const hipStream_t st = as_stream(stream);
    const unsigned rows = (unsigned)(batch * len);
    with_adapter_types(x_type, type, weight_type, [&](auto xt, auto yt, auto wt) {
        using X = decltype(xt);
        using Y = decltype(yt);
        using W = decltype(wt);
        if (work) hipLaunchKernelGGL((adapter_down_kernel<X, W>), dim3(rows), dim3(256), 0, st, args);
        hipLaunchKernelGGL((adapter_up_kernel<Y, W>), dim3(rows, (unsigned)((n + 255) / 256)), dim3(256), 0, st, args);
    });
    return check_launch("mi_adapter_add");
}
