// Selective state space scan of float rows, over prompts and single tokens:
//
//   d = softplus(dt[b,t,c] + dt_bias[c])
//   h[n] = exp(d * a[c,n]) * h[n] + d * u[b,t,c] * B[b,t,g,n]
//   y[b,t,c] = (sum_n C[b,t,g,n] * h[n] + d_skip[c] * u[b,t,c]) * silu(z[b,t,c])
//
// with g = c / (dim / groups) and h in 32 bits.
#include <type_traits>
#include <utility>

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

// ------------------------------------------------------------- prompts
// A block holds 64 channels of a sequence (a lane each) and NW * S states (S a
// wave), and walks the steps in tiles of TT.  Per state and step: the decay's
// product, its exponential, its product with h, and two matrix instructions of
// 4 x 1 by 1 x 4 in 16 blocks (block = four channels): one adds the outer product
// of four states' B with the channels' d * u to four states, one adds C * h of a
// state to the channels' y.  They take their B and C from any one lane group of a
// register (cbsz 4, abid), so a register holds 64 values of B, or 16 of C, and no
// lane moves a value to another.  (The other three rows of y's product are not
// used: a row of its own for each of four steps would carry a NaN of a later step
// into an earlier one.)
//
// The decays are kept in log2: d is softplus in units of log 2, so exp(d a) is one
// exp2 of the product with a as it is.
typedef float v4f __attribute__((ext_vector_type(4)));

template <int ABID>
__device__ __forceinline__ v4f outer(float a, float b, v4f c) {
    return __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, c, 4, ABID, 0);
}

// Calls f with integral_constant 0 .. N - 1.
template <class F, int... I>
__device__ __forceinline__ void static_for_seq(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F &&f) {
    static_for_seq(f, std::make_integer_sequence<int, N>{});
}

// The steps of a sequence in `chunks` parts of `chunk` steps: kWhole is one part;
// kEnds computes each part's last state from zero and its sum of d (into ends,
// [batch, chunks, nstate + 1, dim]); kParts starts each part from the states in
// front of it, joined from those.
enum ScanPass { kWhole, kEnds, kParts };

struct ScanSplit {
    float *ends;
    int chunks, chunk, blocks;   // blocks: of 64 channels, a group
};

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f, kMaxFloat = 3.402823466e38f;

template <class T, int S, int NW, int TT, int PASS>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2))) void scan_tile_kernel(ScanArgs<T> a, ScanSplit sp) {
    constexpr int kRows = TT / NW;               // of a tile, a wave's share
    constexpr int kB = TT * S / 64, kC = TT * S / 16;
    static_assert(kRows * NW == TT && kB * 64 == TT * S, "tile");
    constexpr bool kShare = NW > 1, kY = PASS != kEnds;
    __shared__ float2 steps[kShare ? TT : 1][64];
    __shared__ float parts[kShare && kY ? NW : 1][kShare && kY ? TT : 1][64];
    const int wave = NW > 1 ? wave_id() : 0, lane = threadIdx.x & 63;
    const int group_dim = a.dim / a.groups, N = a.nstate;
    const int64_t b = blockIdx.x / (a.groups * sp.blocks);
    const int rest = blockIdx.x % (a.groups * sp.blocks), g = rest / sp.blocks;
    const int in_group = rest % sp.blocks * 64 + lane;
    const bool on = in_group < group_dim;
    const int c = g * group_dim + min(in_group, group_dim - 1);
    const int n0 = wave * S, k = PASS == kWhole ? 0 : blockIdx.y;
    const int len = scan_len(a.lens, b, a.len);
    const int from = k * sp.chunk, to = PASS == kWhole ? a.len : min(a.len, from + sp.chunk);
    const int end = min(to, len);                // steps of this part that are computed

    float am[S];
    v4f h[S / 4];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int n = n0 + i;
        float v = n < N ? a.a[(int64_t)c * N + n] : 0.0f;
        am[i] = v < -kMaxFloat ? -kMaxFloat : v;  // (a step of 0 then keeps the state whatever a is)
        h[i / 4][i % 4] = PASS != kEnds && a.h_in && n < N ? a.h_in[(b * a.dim + c) * N + n] : 0.0f;
    }
    if (PASS == kParts) {
        const float *e = sp.ends + b * sp.chunks * (N + 1) * a.dim + c;
        for (int j = 0; j < k; ++j, e += (int64_t)(N + 1) * a.dim) {
            const float sum = e[(int64_t)N * a.dim];
#pragma unroll
            for (int i = 0; i < S; ++i) {
                const float last = n0 + i < N ? e[(int64_t)(n0 + i) * a.dim] : 0.0f, was = h[i / 4][i % 4];
                h[i / 4][i % 4] = was != 0.0f ? __builtin_fmaf(__builtin_amdgcn_exp2f(am[i] * sum), was, last) : last;
            }
        }
    }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f, skip = a.d_skip ? a.d_skip[c] : 0.0f;
    const bool gate = kY && a.z.p != nullptr;

    // the rows of the tile at t: this wave's share of dt, u and z, and B and C of its states
    T dt_next[kRows], u_next[kRows], z_next[kRows], b_next[kB], c_next[kC];
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int row = min(t + wave * kRows + i, end - 1);
            dt_next[i] = a.dt.row(b, row)[c];
            u_next[i] = a.u.row(b, row)[c];
            if (gate) z_next[i] = a.z.row(b, row)[c];
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int at = i * 64 + lane;
            b_next[i] = a.b.row(b, min(t + at / S, end - 1))[(int64_t)g * N + min(n0 + at % S, N - 1)];
        }
        if (kY) {
#pragma unroll
            for (int i = 0; i < kC; ++i) {
                const int at = i * 16 + lane / 4;
                c_next[i] = a.c.row(b, min(t + at / S, end - 1))[(int64_t)g * N + min(n0 + at % S, N - 1)];
            }
        }
    };

    float sum = 0.0f;
    if (from < end) load(from);
    for (int t = from; t < end; t += TT) {
        float u[kRows], z[kRows], bv[kB], cv[kC], d[kRows], du[kRows], y[kShare ? 1 : TT];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const bool in = t + wave * kRows + i < end;
            u[i] = (float)u_next[i];
            z[i] = gate ? (float)z_next[i] : 0.0f;
            const float raw = (float)dt_next[i] + bias;
            float s = kLog2e * raw, v = raw * u[i];
            if (a.softplus) {
                const float e = __builtin_amdgcn_exp2f(-fabsf(s)), w = 1.0f + e;
                const float low = __builtin_amdgcn_logf(w) + kLog2e * (e - (w - 1.0f));
                s = s > 0.0f ? s + low : (s <= 0.0f ? low : s);
                v = s * (kLn2 * u[i]);
            }
            d[i] = in ? s : 0.0f;
            du[i] = in ? v : 0.0f;
            if (kShare) steps[wave * kRows + i][lane] = float2{d[i], du[i]};
        }
#pragma unroll
        for (int i = 0; i < kB; ++i) {
            const int at = i * 64 + lane;
            bv[i] = t + at / S < end && n0 + at % S < N ? (float)b_next[i] : 0.0f;
        }
        if (kY) {
#pragma unroll
            for (int i = 0; i < kC; ++i) cv[i] = n0 + (i * 16 + lane / 4) % S < N ? (float)c_next[i] : 0.0f;
        }
        if (t + TT < end) load(t + TT);
        if (kShare) __syncthreads();
        static_for<TT>([&](auto step) {
            constexpr int s = decltype(step)::value;
            float ds, dus;
            if constexpr (kShare) {
                const float2 v = steps[s][lane];
                ds = v.x;
                dus = v.y;
            } else {
                ds = d[s];
                dus = du[s];
            }
            if (PASS == kEnds) sum += ds;
            v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
            static_for<S / 4>([&](auto quad) {
                constexpr int q = decltype(quad)::value, at = s * S + 4 * q;
                v4f p;
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(am[4 * q + i] * ds) * h[q][i];
                h[q] = outer<at % 64 / 4>(bv[at / 64], dus, p);
                if constexpr (kY)
                    static_for<4>([&](auto state) {
                        constexpr int n = at + decltype(state)::value;
                        acc = outer<n % 16>(cv[n / 16], h[q][decltype(state)::value], acc);
                    });
            });
            if constexpr (kY) {
                if constexpr (kShare)
                    parts[wave][s][lane] = acc[0];
                else
                    y[s] = acc[0];
            }
        });
        if (kShare) __syncthreads();
        if (kY) {
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
                const int s = wave * kRows + i;
                float v = skip * u[i];
                if (kShare) {
#pragma unroll
                    for (int w = 0; w < NW; ++w) v += parts[w][s][lane];
                } else {
                    v += y[i];
                }
                if (gate) v *= silu(z[i]);
                if (on && t + s < end) a.y.row(b, t + s)[c] = (T)v;
            }
        }
    }
    if (kY)
        for (int t = max(from, end) + wave; t < to; t += NW)
            if (on) a.y.row(b, t)[c] = (T)0.0f;
    if (!on) return;
    if (PASS == kEnds) {
        float *e = sp.ends + (b * sp.chunks + k) * (N + 1) * a.dim + c;
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (n0 + i < N) e[(int64_t)(n0 + i) * a.dim] = h[i / 4][i % 4];
        if (wave == 0) e[(int64_t)N * a.dim] = sum;
    } else if (a.h_out && (PASS == kWhole || k == sp.chunks - 1)) {
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (n0 + i < N) a.h_out[(b * a.dim + c) * N + n0 + i] = h[i / 4][i % 4];
    }
}

// How a scan is split: states a wave, waves a block, parts of the sequence (0: the
// step kernel).
struct ScanPlan {
    int states, waves, chunks, chunk, blocks;
};

inline ScanPlan scan_plan(int batch, int len, int dim, int nstate, int groups) {
    ScanPlan p{};
    if (len <= 4) return p;
    p.blocks = (dim / groups + 63) / 64;
    const int64_t blocks = (int64_t)batch * groups * p.blocks;
    const int64_t simds = (int64_t)device_cus() * 4;
    p.states = nstate > 64 || blocks >= 2 * simds ? 16 : 4;
    p.waves = 1;
    while (p.waves * p.states < nstate) p.waves *= 2;
    // a second pass over the sequence costs as much as the first one saves until the
    // waves are few
    int64_t chunks = 1;
    if (blocks * p.waves * 2 <= simds) chunks = 2 * simds / (blocks * p.waves);
    const int64_t most = (len + 63) / 64;
    if (chunks > most) chunks = most;
    if (chunks > 64) chunks = 64;
    if (chunks < 3) chunks = 1;
    p.chunk = (int)(((len + chunks - 1) / chunks + 15) / 16 * 16);
    p.chunks = (len + p.chunk - 1) / p.chunk;
    return p;
}

template <class T, int S, int NW, int TT>
void launch_scan_tiles(const ScanArgs<T> &a, const ScanPlan &p, float *ends, hipStream_t st) {
    const ScanSplit sp{ends, p.chunks, p.chunk, p.blocks};
    const dim3 grid((unsigned)(a.batch * a.groups * p.blocks), (unsigned)p.chunks);
    if (p.chunks == 1) {
        hipLaunchKernelGGL((scan_tile_kernel<T, S, NW, TT, kWhole>), grid, dim3(64 * NW), 0, st, a, sp);
    } else {
        hipLaunchKernelGGL((scan_tile_kernel<T, S, NW, TT, kEnds>), dim3(grid.x, grid.y - 1), dim3(64 * NW), 0, st, a, sp);
        hipLaunchKernelGGL((scan_tile_kernel<T, S, NW, TT, kParts>), grid, dim3(64 * NW), 0, st, a, sp);
    }
}

template <class T>
void launch_scan_steps(const ScanArgs<T> &a, hipStream_t st) {
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

template <class T>
void launch_scan(const ScanArgs<T> &a, const ScanPlan &p, float *ends, hipStream_t st) {
    if (p.chunks == 0) return launch_scan_steps(a, st);
    switch (p.states * 100 + p.waves) {
        case 401: return launch_scan_tiles<T, 4, 1, 16>(a, p, ends, st);
        case 402: return launch_scan_tiles<T, 4, 2, 16>(a, p, ends, st);
        case 404: return launch_scan_tiles<T, 4, 4, 16>(a, p, ends, st);
        case 408: return launch_scan_tiles<T, 4, 8, 16>(a, p, ends, st);
        case 416: return launch_scan_tiles<T, 4, 16, 16>(a, p, ends, st);
        case 1601: return launch_scan_tiles<T, 16, 1, 8>(a, p, ends, st);
        case 1602: return launch_scan_tiles<T, 16, 2, 16>(a, p, ends, st);
        case 1604: return launch_scan_tiles<T, 16, 4, 16>(a, p, ends, st);
        case 1608: return launch_scan_tiles<T, 16, 8, 16>(a, p, ends, st);
        default: return launch_scan_tiles<T, 16, 16, 16>(a, p, ends, st);
    }
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_selective_scan_workspace_size(int batch, int len, int dim, int nstate, int groups, size_t *bytes) {
    clear_error();
    MI_REQUIRE(bytes, MI_ERR_NULL_POINTER, "mi_selective_scan_workspace_size: bytes is required");
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0 && nstate >= 1 && nstate <= kScanMaxStates, MI_ERR_BAD_DIM,
               "mi_selective_scan_workspace_size: a size is negative, or nstate=%d not in [1, %d]", nstate, kScanMaxStates);
    MI_REQUIRE(groups >= 1 && dim % groups == 0, MI_ERR_BAD_DIM, "mi_selective_scan_workspace_size: groups=%d must divide dim=%d",
               groups, dim);
    *bytes = 0;
    if (batch == 0 || dim == 0) return MI_OK;
    const ScanPlan p = scan_plan(batch, len, dim, nstate, groups);
    if (p.chunks > 1) *bytes = (size_t)batch * p.chunks * (nstate + 1) * dim * sizeof(float);
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
    const ScanPlan plan = scan_plan(batch, len, dim, nstate, groups);
    MI_REQUIRE((int64_t)batch * groups * plan.blocks * plan.waves * 64 < ((int64_t)1 << 32), MI_ERR_BAD_DIM,
               "mi_selective_scan: too many groups of few channels for one launch");
    const size_t need = plan.chunks > 1 ? (size_t)batch * plan.chunks * (nstate + 1) * dim * sizeof(float) : 0;
    MI_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG,
               "mi_selective_scan: workspace of %zu bytes, %zu are needed", workspace ? workspace_bytes : 0, need);
    MI_REQUIRE(need == 0 || aligned(workspace, 16), MI_ERR_BAD_ALIGNMENT, "mi_selective_scan: workspace must be 16-byte aligned");
    const hipStream_t st = as_stream(stream);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto in = [](const void *p, int64_t ld, int64_t bs) { return Rows<const T>{static_cast<const T *>(p), ld, bs}; };
        launch_scan<T>({in(u, ldu, bsu), in(dt, ldt, bst), in(b, ldb, bsb), in(c, ldc, bsc), in(z, ldz, bsz), a, d_skip,
                        dt_bias, h_in, h_out, lens, {static_cast<T *>(y), ldy, bsy}, dt_softplus, batch, len, dim, nstate,
                        groups},
                       plan, static_cast<float *>(workspace), st);
    });
    return check_launch("mi_selective_scan");
}
