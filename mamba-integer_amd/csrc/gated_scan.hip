// Gated linear recurrence of float rows, over prompts and single tokens, and its backward
// pass:
//
//   s = sigmoid(r),  q = sigmoid(i),  a = exp(-rate * softplus(decay[c]) * s)
//   h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) q[t] x[t],  y[t] = h[t] silu(z[t])
//
// with h in 32 bits.  Backwards, with n = rate softplus(decay) s = -log a and
// m = sqrt(1 - a^2):
//
//   g[t] = dy[t] silu(z[t]) + a[t+1] g[t+1]
//   dx = g m q,  di = g m q x (1 - q),  dz = dy h silu'(z),  dh[-1] = a[0] g[0]
//   p = n dn = g (q x a^2 n / m - n a h[t-1]),  dr = p (1 - s)
//   ddecay = sigmoid(decay) / softplus(decay) * sum over b, t of p
#include "float_ops.hpp"

namespace mi {

constexpr int kGatedChunk = 16;   // steps between the states that a forward pass keeps for its backward pass

struct GatedRows {
    void *p;
    int64_t ld, bs;
    template <class T>
    __device__ __forceinline__ T *row(int64_t b, int64_t t) const { return static_cast<T *>(p) + b * bs + t * ld; }
};

struct GatedArgs {
    GatedRows x, r, i, z, y;             // y: dy in a backward pass
    GatedRows dx, dr, di, dz;
    const float *decay, *h_in;
    float *h_out, *saved;                // saved [batch, chunks, dim]: the state in front of each chunk
    float *dh_in, *sums;                 // sums [batch, dim]: of p over the steps
    const int32_t *lens;
    float rate;
    int batch, len, dim, chunks;
};

__device__ __forceinline__ int gated_len(const GatedArgs &a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.len) : a.len;
}
// log(1 + exp(v)), with the relative precision of exp(v) for low v
__device__ __forceinline__ float gated_softplus(float v) { return v > 20.0f ? v : log1pf(expf(v)); }
__device__ __forceinline__ float sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}
// 1 - exp(-2 n) for n >= 0 and a = exp(-n): by its series where the difference would cancel
__device__ __forceinline__ float one_minus_square(float n, float a) {
    const float v = 2.0f * n;
    // v - v^2/2 + v^3/6 - ...: the term after the last is below 2^-24 of the sum at v = 0.5
    float s = __builtin_fmaf(v, -1.0f / 40320.0f, 1.0f / 5040.0f);
    s = __builtin_fmaf(v, -s, 1.0f / 720.0f);
    s = __builtin_fmaf(v, -s, 1.0f / 120.0f);
    s = __builtin_fmaf(v, -s, 1.0f / 24.0f);
    s = __builtin_fmaf(v, -s, 1.0f / 6.0f);
    s = __builtin_fmaf(v, -s, 0.5f);
    s = __builtin_fmaf(v, -s, 1.0f);
    return v < 0.5f ? v * s : __builtin_fmaf(-a, a, 1.0f);
}

// One step's decay and input.
struct GatedStep {
    float s, q, n, a, m2, b;
    __device__ __forceinline__ GatedStep(float k, float x, float r, float i) {
        s = sigmoid(r);
        q = sigmoid(i);
        n = k * s;
        a = __builtin_amdgcn_exp2f(-1.44269504f * n);
        m2 = one_minus_square(n, a);
        b = __builtin_amdgcn_sqrtf(m2) * q * x;
    }
};

// A thread a channel, step by step.
template <class T>
__global__ __launch_bounds__(64) void gated_scan_kernel(GatedArgs a) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= a.dim) return;
    const int len = gated_len(a, b);
    const int64_t at = (int64_t)b * a.dim + c;
    const float k = a.rate * gated_softplus(a.decay[c]);
    float h = a.h_in ? a.h_in[at] : 0.0f;
    for (int t = 0; t < a.len; ++t) {
        if (a.saved && t % kGatedChunk == 0) a.saved[((int64_t)b * a.chunks + t / kGatedChunk) * a.dim + c] = h;
        float y = 0.0f;
        if (t < len) {
            const GatedStep g(k, (float)a.x.row<const T>(b, t)[c], (float)a.r.row<const T>(b, t)[c], (float)a.i.row<const T>(b, t)[c]);
            h = __builtin_fmaf(g.a, h, g.b);
            y = a.z.p ? h * silu((float)a.z.row<const T>(b, t)[c]) : h;
        }
        a.y.row<T>(b, t)[c] = (T)y;
    }
    if (a.h_out) a.h_out[at] = h;
}

template <class T>
__global__ __launch_bounds__(64) void gated_scan_backward_kernel(GatedArgs a) {
    const int c = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (c >= a.dim) return;
    const int len = gated_len(a, b);
    const int64_t at = (int64_t)b * a.dim + c;
    const float k = a.rate * gated_softplus(a.decay[c]);
    float carry = 0.0f, sum = 0.0f;      // a g of the step after
    for (int chunk = a.chunks - 1; chunk >= 0; --chunk) {
        const int t0 = chunk * kGatedChunk;
        float h[kGatedChunk + 1];
        h[0] = a.saved[((int64_t)b * a.chunks + chunk) * a.dim + c];
#pragma unroll
        for (int j = 0; j < kGatedChunk; ++j) {
            h[j + 1] = h[j];
            if (t0 + j < len) {
                const GatedStep g(k, (float)a.x.row<const T>(b, t0 + j)[c], (float)a.r.row<const T>(b, t0 + j)[c],
                                  (float)a.i.row<const T>(b, t0 + j)[c]);
                h[j + 1] = __builtin_fmaf(g.a, h[j], g.b);
            }
        }
#pragma unroll
        for (int j = kGatedChunk - 1; j >= 0; --j) {
            const int t = t0 + j;
            if (t >= a.len) continue;
            float dx = 0.0f, dr = 0.0f, di = 0.0f, dz = 0.0f;
            if (t < len) {
                const float x = (float)a.x.row<const T>(b, t)[c];
                const GatedStep st(k, x, (float)a.r.row<const T>(b, t)[c], (float)a.i.row<const T>(b, t)[c]);
                float dh = (float)a.y.row<const T>(b, t)[c];
                if (a.z.p) {
                    const float z = (float)a.z.row<const T>(b, t)[c], sz = sigmoid(z), act = z * sz;
                    dz = dh * h[j + 1] * __builtin_fmaf(act, 1.0f - sz, sz);
                    dh *= act;
                }
                const float g = dh + carry;
                // (the hardware root takes a subnormal for 0, its reciprocal is infinite there)
                const float inv = st.m2 >= 0x1p-126f ? __builtin_amdgcn_rsqf(st.m2) : 0.0f, m = st.m2 * inv;
                const float p = g * (st.q * x * st.a * st.a * (st.n * inv) - st.n * st.a * h[j]);
                dx = g * m * st.q;
                di = g * st.b * (1.0f - st.q);
                dr = p * (1.0f - st.s);
                sum += p;
                carry = st.a * g;
            }
            if (a.dx.p) a.dx.row<T>(b, t)[c] = (T)dx;
            if (a.dr.p) a.dr.row<T>(b, t)[c] = (T)dr;
            if (a.di.p) a.di.row<T>(b, t)[c] = (T)di;
            if (a.dz.p) a.dz.row<T>(b, t)[c] = (T)dz;
        }
    }
    if (a.dh_in) a.dh_in[at] = carry;
    if (a.sums) a.sums[at] = sum;
}

// ddecay from the sums of p.
__global__ __launch_bounds__(64) void gated_decay_kernel(const float *sums, const float *decay, float *out, int rows, int dim) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= dim) return;
    float s = 0.0f;
    for (int j = 0; j < rows; ++j) s += sums[(int64_t)j * dim + c];
    // sigmoid / softplus: 1 - e/2 + ... of e = exp(v) for low v
    const float v = decay[c], e = expf(v);
    const float ratio = v < -9.0f ? 1.0f - 0.5f * e : 1.0f / (1.0f + expf(-v)) / gated_softplus(v);
    out[c] = s * ratio;
}

mi_status gated_dims(const char *fn, int batch, int len, int dim) {
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0, MI_ERR_BAD_DIM, "%s: a size is negative", fn);
    MI_REQUIRE(batch <= 65535, MI_ERR_BAD_DIM, "%s: batch=%d must be at most 65535", fn, batch);
    MI_REQUIRE(dim <= (1 << 24), MI_ERR_BAD_DIM, "%s: dim=%d must be at most 2^24", fn, dim);
    MI_REQUIRE(len <= (1 << 30), MI_ERR_BAD_DIM, "%s: len=%d must be at most 2^30", fn, len);
    return MI_OK;
}

inline int gated_chunks(int len) { return (len + kGatedChunk - 1) / kGatedChunk; }

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_gated_scan_sizes(int batch, int len, int dim, size_t *forward_bytes, size_t *backward_bytes,
                                         size_t *saved_bytes) {
    clear_error();
    MI_REQUIRE(forward_bytes && backward_bytes && saved_bytes, MI_ERR_NULL_POINTER, "mi_gated_scan_sizes: the sizes are required");
    if (const mi_status st = gated_dims("mi_gated_scan_sizes", batch, len, dim)) return st;
    *forward_bytes = 0;
    *backward_bytes = (size_t)batch * dim * sizeof(float);
    *saved_bytes = (size_t)batch * gated_chunks(len) * dim * sizeof(float);
    return MI_OK;
}

extern "C" mi_status mi_gated_scan(const void *x, int64_t ldx, int64_t bsx, const void *r, int64_t ldr, int64_t bsr,
                                   const void *i, int64_t ldi, int64_t bsi, const float *decay, float rate, const void *z,
                                   int64_t ldz, int64_t bsz, const float *h_in, float *h_out, const int32_t *lens, void *y,
                                   int64_t ldy, int64_t bsy, float *saved, int type, int batch, int len, int dim,
                                   void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    if (const mi_status st = gated_dims("mi_gated_scan", batch, len, dim)) return st;
    MI_REQUIRE(known_type(type), MI_ERR_BAD_ARG, "mi_gated_scan: unknown element type");
    MI_REQUIRE(rate >= 0.0f && rate <= 1e30f, MI_ERR_BAD_ARG, "mi_gated_scan: rate must be in [0, 1e30]");
    MI_REQUIRE(ldx >= 0 && bsx >= 0 && ldr >= 0 && bsr >= 0 && ldi >= 0 && bsi >= 0 && ldz >= 0 && bsz >= 0, MI_ERR_BAD_DIM,
               "mi_gated_scan: a stride is negative");
    MI_REQUIRE(ldy >= dim && bsy >= 0, MI_ERR_BAD_DIM, "mi_gated_scan: ldy=%lld must be at least dim", (long long)ldy);
    if (batch == 0 || dim == 0) return MI_OK;
    MI_REQUIRE(decay && (len == 0 || (x && r && i && y)), MI_ERR_NULL_POINTER, "mi_gated_scan: x, r, i, decay and y are required");
    const auto in = [](const void *p, int64_t ld, int64_t bs) { return GatedRows{const_cast<void *>(p), ld, bs}; };
    GatedArgs a{};
    a.x = in(x, ldx, bsx), a.r = in(r, ldr, bsr), a.i = in(i, ldi, bsi), a.z = in(z, ldz, bsz), a.y = {y, ldy, bsy};
    a.decay = decay, a.h_in = h_in, a.h_out = h_out, a.saved = saved, a.lens = lens, a.rate = rate;
    a.batch = batch, a.len = len, a.dim = dim, a.chunks = gated_chunks(len);
    const hipStream_t st = as_stream(stream);
    with_type(type, [&](auto t) {
        hipLaunchKernelGGL((gated_scan_kernel<decltype(t)>), dim3((unsigned)((dim + 63) / 64), (unsigned)batch), dim3(64), 0, st, a);
    });
    return check_launch("mi_gated_scan");
}

extern "C" mi_status mi_gated_scan_backward(const void *dy, int64_t ldy, int64_t bsy, const void *x, int64_t ldx, int64_t bsx,
                                            const void *r, int64_t ldr, int64_t bsr, const void *i, int64_t ldi, int64_t bsi,
                                            const float *decay, float rate, const void *z, int64_t ldz, int64_t bsz,
                                            const int32_t *lens, const float *saved, void *dx, void *dr, void *di, void *dz,
                                            float *ddecay, float *dh_in, int type, int batch, int len, int dim, void *workspace,
                                            size_t workspace_bytes, void *stream) {
    clear_error();
    if (const mi_status st = gated_dims("mi_gated_scan_backward", batch, len, dim)) return st;
    MI_REQUIRE(known_type(type), MI_ERR_BAD_ARG, "mi_gated_scan_backward: unknown element type");
    MI_REQUIRE(rate >= 0.0f && rate <= 1e30f, MI_ERR_BAD_ARG, "mi_gated_scan_backward: rate must be in [0, 1e30]");
    MI_REQUIRE(ldx >= 0 && bsx >= 0 && ldr >= 0 && bsr >= 0 && ldi >= 0 && bsi >= 0 && ldz >= 0 && bsz >= 0 && ldy >= 0 && bsy >= 0,
               MI_ERR_BAD_DIM, "mi_gated_scan_backward: a stride is negative");
    MI_REQUIRE(!dz || z, MI_ERR_BAD_ARG, "mi_gated_scan_backward: dz without z");
    if (dim == 0) return MI_OK;
    MI_REQUIRE(decay, MI_ERR_NULL_POINTER, "mi_gated_scan_backward: decay is required");
    MI_REQUIRE(batch == 0 || len == 0 || (dy && x && r && i && saved), MI_ERR_NULL_POINTER,
               "mi_gated_scan_backward: dy, x, r, i and saved are required");
    size_t forward = 0, need = 0, keep = 0;
    mi_gated_scan_sizes(batch, len, dim, &forward, &need, &keep);
    MI_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG,
               "mi_gated_scan_backward: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    MI_REQUIRE(aligned(workspace, 16), MI_ERR_BAD_ALIGNMENT, "mi_gated_scan_backward: the workspace must be 16-byte aligned");
    const auto in = [](const void *p, int64_t ld, int64_t bs) { return GatedRows{const_cast<void *>(p), ld, bs}; };
    const int64_t bs = (int64_t)len * dim;
    GatedArgs a{};
    a.x = in(x, ldx, bsx), a.r = in(r, ldr, bsr), a.i = in(i, ldi, bsi), a.z = in(z, ldz, bsz), a.y = in(dy, ldy, bsy);
    a.dx = {dx, dim, bs}, a.dr = {dr, dim, bs}, a.di = {di, dim, bs}, a.dz = {dz, dim, bs};
    a.decay = decay, a.saved = const_cast<float *>(saved), a.dh_in = dh_in, a.sums = static_cast<float *>(workspace), a.lens = lens;
    a.rate = rate, a.batch = batch, a.len = len, a.dim = dim, a.chunks = gated_chunks(len);
    const hipStream_t st = as_stream(stream);
    if (batch > 0)
        with_type(type, [&](auto t) {
            hipLaunchKernelGGL((gated_scan_backward_kernel<decltype(t)>), dim3((unsigned)((dim + 63) / 64), (unsigned)batch), dim3(64),
                               0, st, a);
        });
    if (ddecay)
        hipLaunchKernelGGL(gated_decay_kernel, dim3((unsigned)((dim + 63) / 64)), dim3(64), 0, st, a.sums, decay, ddecay, batch, dim);
    return check_launch("mi_gated_scan_backward");
}
