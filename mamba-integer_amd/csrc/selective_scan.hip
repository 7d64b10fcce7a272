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
// Up to these steps a lane walks them with their loads, a memory latency each.  Kernel
// times in us, that and the tiles below, of 2, 4 and 8 steps: 1 x 1536 channels 4.1, 5.0, 8.2
// and 4.4, 4.5, 4.6; 64 x 4096 13.9, 20.4, 32.4 and 25.8, 25.6, 26.2.  (The tiles are ahead
// from 4 and 6 steps on; the host covers the difference where channels are few.)
constexpr int kScanStepLen = 8;
constexpr int64_t kScanMaxLd = (int64_t)1 << 25;   // 16 rows' offsets in 32 bits

constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147181f, kMaxFloat = 3.402823466e38f;

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

// A decay of -inf is the lowest float's: a step of 0 then keeps the state whatever a is.
// (The maximum that keeps a NaN, one instruction.)
__device__ __forceinline__ float finite_decay(float a) { return __builtin_elementwise_maximum(a, -kMaxFloat); }

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
#pragma unroll
    for (int i = 0; i < 4; ++i) am[i] = finite_decay(am[i]);
    if (a.h_in) four(a.h_in + (int64_t)ch * N + n0, h);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f, skip = a.d_skip ? a.d_skip[c] : 0.0f;
    for (int t = 0; t < len; ++t) {
        float bn[4] = {}, cn[4] = {};
        four(a.b.row(b, t) + g0, bn);
        four(a.c.row(b, t) + g0, cn);
        const float u = (float)a.u.row(b, t)[c];
        float dt = (float)a.dt.row(b, t)[c] + bias;
        if (a.softplus) dt = softplus(dt);
        const float du = dt * u, dl = kLog2e * dt;             // (kLog2e * am may be infinite, and the step 0)
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(dl * am[i]), h[i], du * bn[i]);
            if (n0 + i < N) y = __builtin_fmaf(cn[i], h[i], y);
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) y += __shfl_xor(y, o);
        if (a.d_skip) y = __builtin_fmaf(skip, u, y);          // (0 * inf without it)
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

// One token: as above, over kSeqs sequences a thread, which share the channel's A, bias
// and skip, and whose states' loads are all in flight together.  Bound by the states,
// read and written once.
constexpr int kSeqs = 2;

template <class T, int LANES>
__global__ __launch_bounds__(256) void scan_token_kernel(ScanArgs<T> a) {
    const uint32_t id = (blockIdx.x * 256 + threadIdx.x) / LANES, all = (uint32_t)a.dim * (uint32_t)((a.batch + kSeqs - 1) / kSeqs);
    const int lane = threadIdx.x % LANES, N = a.nstate, n0 = min(4 * lane, N - 4);
    const bool on = id < all, mine = 4 * lane < N;
    const uint32_t ch = on ? id : all - 1;
    const uint32_t b0 = ch / (uint32_t)a.dim * kSeqs;
    const int c = (int)(ch % (uint32_t)a.dim);
    const int64_t g0 = (int64_t)(c / (a.dim / a.groups)) * N + n0;
    Packed<float, 4> h[kSeqs];
    Packed<T, 4> bn[kSeqs], cn[kSeqs];
    T u[kSeqs], dt[kSeqs], z[kSeqs];
    int64_t b[kSeqs], at[kSeqs];
#pragma unroll
    for (int s = 0; s < kSeqs; ++s) {
        b[s] = min((int)b0 + s, a.batch - 1);
        at[s] = (b[s] * a.dim + c) * N + n0;
        if (a.h_in) h[s] = load_packed<4>(a.h_in + at[s]);
        u[s] = a.u.row(b[s], 0)[c];
        dt[s] = a.dt.row(b[s], 0)[c];
        bn[s] = load_packed<4>(a.b.row(b[s], 0) + g0);
        cn[s] = load_packed<4>(a.c.row(b[s], 0) + g0);
        if (a.z.p) z[s] = a.z.row(b[s], 0)[c];
    }
    Packed<float, 4> am = load_packed<4>(a.a + (int64_t)c * N + n0);
#pragma unroll
    for (int i = 0; i < 4; ++i) am.v[i] = finite_decay(am.v[i]);
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f, skip = a.d_skip ? a.d_skip[c] : 0.0f;
#pragma unroll
    for (int s = 0; s < kSeqs; ++s) {
        const bool run = scan_len(a.lens, b[s], 1) != 0;
        const float uf = (float)u[s];
        float d = (float)dt[s] + bias;
        if (a.softplus) d = softplus(d);
        const float du = d * uf, dl = kLog2e * d;
        float y = 0.0f;
        Packed<float, 4> next;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float was = a.h_in ? h[s].v[i] : 0.0f;
            const float now = __builtin_fmaf(__builtin_amdgcn_exp2f(dl * am.v[i]), was, du * (float)bn[s].v[i]);
            y = __builtin_fmaf((float)cn[s].v[i], now, y);
            next.v[i] = run ? now : was;
        }
        if (!mine) y = 0.0f;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) y += __shfl_xor(y, o);
        if (!on || (int)b0 + s >= a.batch) continue;
        if (a.h_out && mine) store_packed<4>(a.h_out + at[s], next);
        if (lane == 0) {
            if (a.d_skip) y = __builtin_fmaf(skip, uf, y);
            if (a.z.p) y *= silu((float)z[s]);
            a.y.row(b[s], 0)[c] = (T)(run ? y : 0.0f);
        }
    }
}

template <class T, int LANES>
void launch_scan_step(const ScanArgs<T> &a, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)a.batch * a.dim * LANES + 255) / 256));
    if (a.len == 1 && a.nstate % 4 == 0)
        hipLaunchKernelGGL((scan_token_kernel<T, LANES>),
                           dim3((unsigned)(((int64_t)((a.batch + kSeqs - 1) / kSeqs) * a.dim * LANES + 255) / 256)), dim3(256), 0, st, a);
    else if (a.nstate % 4 == 0)
        hipLaunchKernelGGL((scan_step_kernel<T, LANES, true>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((scan_step_kernel<T, LANES, false>), grid, dim3(256), 0, st, a);
}

// ------------------------------------------------------------- prompts
// A block holds 64 channels of a sequence (a lane each) and NW * S states (S a
// wave), and walks the steps in tiles of TT.  Per state and step: the decay's
// product, its exponential (two issue slots), d u B, the multiply-add of h and that
// of y.  B and C are the same for all lanes: a register holds 16 of their values in
// each row of 16 lanes, and the multiplications read one of them by a DPP row
// broadcast, so they cost no instruction, no LDS and no scalar load of their own.
// (Both products on 4x4x1 matrix instructions, with the same broadcast by cbsz and
// abid: one takes 9 to 12 issue cycles and blocks the SIMD meanwhile, a
// multiply-add 4; 8 x 2048 x 1536 x 16 took 319 us.)
//
// The decays are kept in log2: d is softplus in units of log 2, so exp(d a) is one
// exp2 of the product with a as it is.
template <int LANE>
__device__ __forceinline__ float bcast(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + LANE, 0xf, 0xf, true));
}

// One step of four states: p = a * next (the next step's exponents), h = e * h + x,
// y += C * h with C in lanes LANE .. + 3 of every row of c.  In assembly, since the
// compiler does not fold a broadcast into a multiply-add.  The four products in
// front are the wait states that a broadcast of a register just written, and the
// use of an exponential just taken, ask for.
template <int LANE>
__device__ __forceinline__ void scan_quad(const float (&a)[4], float next, const float (&e)[4], float (&x)[4], float c,
                                          float (&p)[4], float (&h)[4], float &y) {
    asm("v_mul_f32 %0, %9, %13\n\tv_mul_f32 %1, %10, %13\n\tv_mul_f32 %2, %11, %13\n\tv_mul_f32 %3, %12, %13\n\t"
        "v_fmac_f32 %4, %14, %18\n\tv_fmac_f32 %5, %15, %19\n\tv_fmac_f32 %6, %16, %20\n\tv_fmac_f32 %7, %17, %21\n\t"
        "v_fmac_f32_dpp %8, %22, %4 row_newbcast:%23 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %8, %22, %5 row_newbcast:%24 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %8, %22, %6 row_newbcast:%25 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %8, %22, %7 row_newbcast:%26 row_mask:0xf bank_mask:0xf"
        : "=&v"(p[0]), "=&v"(p[1]), "=&v"(p[2]), "=&v"(p[3]), "+&v"(x[0]), "+&v"(x[1]), "+&v"(x[2]), "+&v"(x[3]), "+&v"(y)
        : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(next), "v"(e[0]), "v"(e[1]), "v"(e[2]), "v"(e[3]), "v"(h[0]),
          "v"(h[1]), "v"(h[2]), "v"(h[3]), "v"(c), "n"(LANE), "n"(LANE + 1), "n"(LANE + 2), "n"(LANE + 3));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = x[i];
}

// A barrier for what the block shares through LDS: __syncthreads would also wait for
// the next tile's loads.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
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
// [batch, chunks, nstate + 1, dim], the last part's place holding the sequence's first
// state); kParts starts each part from the states in front of it, joined from those.
enum ScanPass { kWhole, kEnds, kParts };

// The state that a place of a block's holds.  The N states do not always fill the places
// (at most 2 N, or 4): one past N holds a second copy of a state, and a state's copies
// share its C in equal parts, halves or quarters, which are exact.  (Zeros there would
// make 0 * inf of an infinite input or step, a NaN in the channel's sum.)
__device__ __forceinline__ int place_state(int place, int N) { return place < N ? place : N > 1 ? place - N : 0; }
__device__ __forceinline__ float place_share(int place, int N, int places) {
    return N == 1 ? 1.0f / places : place_state(place, N) + N < places ? 0.5f : 1.0f;
}

struct ScanSplit {
    float *ends;
    int chunks, chunk, blocks;   // blocks: of 64 channels, a group
};

// 16 bytes at any float's address
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

// kHelpers waves of a block turn rows into a tile's d, d u, B and C in LDS and the
// recurring waves' parts of y into output rows, one tile ahead and one behind.
constexpr int kHelpers = 4;

template <class T, int S, int NW, int TT, int PASS>
__global__ __launch_bounds__(64 * (NW + kHelpers)) __attribute__((amdgpu_waves_per_eu(S <= 8 ? 4 : 2))) void
scan_tile_kernel(ScanArgs<T> a, ScanSplit sp) {
    constexpr bool kY = PASS != kEnds;
    constexpr int kStates = S * NW, kRows = TT / kHelpers;     // a helper wave's rows of a tile
    constexpr int kBC = TT * S / 16;                           // registers of B, and of C, of a tile
    constexpr int kLoadBC = (TT * kStates + 64 * kHelpers - 1) / (64 * kHelpers);
    static_assert(kRows * kHelpers == TT && kBC * 16 == TT * S, "tile");
    __shared__ float2 steps[2][TT][64];                        // d, d u
    __shared__ float parts[2][kY ? NW : 1][kY ? TT : 1][64];
    __shared__ float bs[2][TT * kStates], cs[2][kY ? TT * kStates : 1];
    const int wave = wave_id(), lane = threadIdx.x & 63;
    const int group_dim = a.dim / a.groups, N = a.nstate;
    const int64_t b = blockIdx.x / (a.groups * sp.blocks);
    const int rest = blockIdx.x % (a.groups * sp.blocks), g = rest / sp.blocks;
    const int in_group = rest % sp.blocks * 64 + lane;
    const bool on = in_group < group_dim;
    const int c = g * group_dim + min(in_group, group_dim - 1);
    const int k = PASS == kWhole ? 0 : blockIdx.y;
    const int len = scan_len(a.lens, b, a.len);
    const int from = k * sp.chunk, to = PASS == kWhole ? a.len : min(a.len, from + sp.chunk);
    const int end = min(to, len);                              // steps of this part that are computed

    if (wave < NW) {
        // ---- the recurrence: the states n0 .. + S - 1
        const int n0 = wave * S;
        float am[S / 4][4], h[S / 4][4];
        // a channel's values from n0 on of rows of N states: four at once where N % 4 == 0
        // (3 x 701 x 1000 x 64 49.1 us instead of 54.6; 8 x 2048 x 1536 x 16 the same)
        auto states = [&](const float *p, float (&o)[S / 4][4]) {
#pragma unroll
            for (int q = 0; q < S / 4; ++q) {
                if (N % 4 == 0) {
                    // (a vector: four floats of a struct are merged with the loads below)
                    const v4f_any v = *reinterpret_cast<const v4f_any *>(p + place_state(n0 + 4 * q, N));
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[q][i] = v[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[q][i] = p[place_state(n0 + 4 * q + i, N)];
                }
            }
        };
        states(a.a + (int64_t)c * N, am);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            float &v = am[i / 4][i % 4];
            v = finite_decay(v);
            h[i / 4][i % 4] = 0.0f;
        }
        if (PASS != kParts && k == 0 && a.h_in) states(a.h_in + (b * a.dim + c) * N, h);
        if (PASS == kEnds && k == 0) {
            // the second pass reads the first state here: h_out, which it writes, may be h_in
            float *e = sp.ends + (b * sp.chunks + sp.chunks - 1) * (N + 1) * a.dim + c;
#pragma unroll
            for (int i = 0; i < S; ++i) {
                if (on && n0 + i < N) e[(int64_t)(n0 + i) * a.dim] = h[i / 4][i % 4];
                h[i / 4][i % 4] = 0.0f;
            }
        }
        if (PASS == kParts) {
            const float *e = sp.ends + b * sp.chunks * (N + 1) * a.dim + c;
            const float *first = e + (int64_t)(sp.chunks - 1) * (N + 1) * a.dim;
#pragma unroll
            for (int i = 0; i < S; ++i) h[i / 4][i % 4] = first[(int64_t)place_state(n0 + i, N) * a.dim];
            // A part's decay in two equal factors, each held at 2^-126 where it would be
            // flushed to zero: one exponential of the whole loses a state of up to 2^128 that
            // has not decayed yet, and makes a NaN of an infinite one.  (An infinite step's is 0.)
            for (int j = 0; j < k; ++j, e += (int64_t)(N + 1) * a.dim) {
                const float sum = 0.5f * e[(int64_t)N * a.dim];
                const float least = fabsf(sum) <= kMaxFloat ? -126.0f : -__builtin_inff();
#pragma unroll
                for (int i = 0; i < S; ++i) {
                    const float last = e[(int64_t)place_state(n0 + i, N) * a.dim];
                    float &hi = h[i / 4][i % 4];
                    const float decay = __builtin_amdgcn_exp2f(fmaxf(am[i / 4][i % 4] * sum, least));
                    hi = hi != 0.0f ? __builtin_fmaf(decay, decay * hi, last) : last;
                }
            }
        }
        float sum = 0.0f;
        int buf = 0;
        if (from < end) lds_barrier();
        for (int t = from; t < end; t += TT, buf ^= 1) {
            float bv[kBC], cv[kBC];
#pragma unroll
            for (int i = 0; i < kBC; ++i) {
                const int e = i * 16 + (lane & 15), at = e / S * kStates + n0 + e % S;
                bv[i] = bs[buf][at];
                cv[i] = kY ? cs[buf][at] : 0.0f;
            }
            float2 dx[TT];
#pragma unroll
            for (int s = 0; s < TT; ++s) dx[s] = steps[buf][s][lane];
            float p[S / 4][4];
#pragma unroll
            for (int i = 0; i < S; ++i) p[i / 4][i % 4] = am[i / 4][i % 4] * dx[0].x;
            static_for<TT>([&](auto step) {
                constexpr int s = decltype(step)::value;
                const float next = dx[s + 1 < TT ? s + 1 : s].x;
                if (PASS == kEnds) sum += dx[s].x;
                float acc = 0.0f;
                static_for<S / 4>([&](auto quad) {
                    constexpr int q = decltype(quad)::value, k0 = s * S + 4 * q;
                    float e[4], x[4];
                    static_for<4>([&](auto state) {
                        constexpr int i = decltype(state)::value;
                        e[i] = __builtin_amdgcn_exp2f(p[q][i]);
                        x[i] = bcast<(k0 + i) % 16>(bv[k0 / 16]) * dx[s].y;
                    });
                    if constexpr (kY) {
                        scan_quad<k0 % 16>(am[q], next, e, x, cv[k0 / 16], p[q], h[q], acc);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            h[q][i] = __builtin_fmaf(e[i], h[q][i], x[i]);
                            p[q][i] = am[q][i] * next;
                        }
                    }
                });
                if (kY) parts[buf][wave][s][lane] = acc;
            });
            lds_barrier();
        }
        if (!on) return;
        if (PASS == kEnds) {
            float *e = sp.ends + (b * sp.chunks + k) * (N + 1) * a.dim + c;
#pragma unroll
            for (int i = 0; i < S; ++i)
                if (n0 + i < N) e[(int64_t)(n0 + i) * a.dim] = h[i / 4][i % 4];
            if (wave == 0) e[(int64_t)N * a.dim] = sum;
        } else if (a.h_out && (PASS == kWhole || k == sp.chunks - 1)) {
            float *o = a.h_out + (b * a.dim + c) * N + n0;
#pragma unroll
            for (int q = 0; q < S / 4; ++q) {
                if (N % 4 == 0) {
                    if (n0 + 4 * q < N) store_packed<4>(o + 4 * q, Packed<float, 4>{{h[q][0], h[q][1], h[q][2], h[q][3]}});
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n0 + 4 * q + i < N) o[4 * q + i] = h[q][i];
                }
            }
        }
        return;
    }

    // ---- a helper wave, in front of the others: they wait for it at the barrier
    // (151 us instead of 156 at 8 x 2048 x 1536 x 16)
    __builtin_amdgcn_s_setprio(2);
    const int hw = wave - NW, r0 = hw * kRows, tid = hw * 64 + lane;
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.0f, skip = a.d_skip ? a.d_skip[c] : 0.0f;
    const bool gate = kY && a.z.p != nullptr;
    static_assert(64 * kHelpers % kStates == 0, "a thread stages one place's C");
    const float share = place_share(min(tid, TT * kStates - 1) % kStates, N, kStates);
    // Rows are read from the tile's first row, whose address every lane shares, by
    // 32-bit offsets that stay the same from tile to tile.
    uint32_t dt_off[kRows], u_off[kRows], z_off[kRows], y_off[kRows], b_off[kLoadBC], c_off[kLoadBC];
    auto offsets = [&](int last) {                             // last: the last row of the tile that is read
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const uint32_t row = min(r0 + i, last);
            dt_off[i] = (row * (uint32_t)a.dt.ld + c) * sizeof(T);
            u_off[i] = (row * (uint32_t)a.u.ld + c) * sizeof(T);
            z_off[i] = gate ? (row * (uint32_t)a.z.ld + c) * sizeof(T) : u_off[i];
            y_off[i] = ((r0 + i) * (uint32_t)a.y.ld + c) * sizeof(T);
        }
#pragma unroll
        for (int i = 0; i < kLoadBC; ++i) {
            const int e = min(tid + i * 64 * kHelpers, TT * kStates - 1);
            const uint32_t row = min(e / kStates, last), col = g * N + place_state(e % kStates, N);
            b_off[i] = (row * (uint32_t)a.b.ld + col) * sizeof(T);
            c_off[i] = (row * (uint32_t)a.c.ld + col) * sizeof(T);
        }
    };
    auto at = [](const T *base, uint32_t off) {
        return *reinterpret_cast<const T *>(reinterpret_cast<const char *>(base) + off);
    };
    const T *dt_p = a.dt.row(b, from), *u_p = a.u.row(b, from), *z_p = gate ? a.z.row(b, from) : u_p;
    const T *b_p = a.b.row(b, from), *c_p = a.c.row(b, from);
    const int64_t z_ld = gate ? a.z.ld : a.u.ld;
    T *y_p = kY ? a.y.row(b, from) : nullptr;
    T dt_next[kRows], u_next[kRows], z_next[kRows], b_next[kLoadBC], c_next[kLoadBC];
    auto load = [&]() {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            dt_next[i] = at(dt_p, dt_off[i]);
            u_next[i] = at(u_p, u_off[i]);
            if (kY) z_next[i] = at(z_p, z_off[i]);
        }
#pragma unroll
        for (int i = 0; i < kLoadBC; ++i) {
            b_next[i] = at(b_p, b_off[i]);
            if (kY) c_next[i] = at(c_p, c_off[i]);
        }
    };
    // the loads of the tile at t, the one after the last that was loaded
    auto fetch = [&](int t) {
        if (t >= end) return;
        if (end - t < TT) offsets(end - t - 1);
        dt_p += TT * a.dt.ld;
        u_p += TT * a.u.ld;
        z_p += TT * z_ld;
        b_p += TT * a.b.ld;
        c_p += TT * a.c.ld;
        load();
    };
    float u[3][kRows], z[3][kRows];                            // of the tile staged, the one before it, ...
    auto stage = [&](int t, int buf) {
        const int rows = end - t;                              // steps past the end: a step of 0 that adds nothing
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            u[2][i] = u[1][i];
            z[2][i] = z[1][i];
            u[1][i] = u[0][i];
            z[1][i] = z[0][i];
            u[0][i] = (float)u_next[i];
            z[0][i] = kY ? (float)z_next[i] : 0.0f;
            const float raw = (float)dt_next[i] + bias;
            float d = kLog2e * raw, du = raw * u[0][i];
            if (a.softplus) {
                const float e = __builtin_amdgcn_exp2f(-fabsf(d)), w = 1.0f + e;
                d = fmaxf(d, 0.0f) + (__builtin_amdgcn_logf(w) + kLog2e * (e - (w - 1.0f)));
                du = d * (kLn2 * u[0][i]);
            }
            steps[buf][r0 + i][lane] = r0 + i < rows ? float2{d, du} : float2{0.0f, 0.0f};
        }
#pragma unroll
        for (int i = 0; i < kLoadBC; ++i) {
            const int e = min(tid + i * 64 * kHelpers, TT * kStates - 1);
            bs[buf][e] = e / kStates < rows ? (float)b_next[i] : 0.0f;
            if (kY) cs[buf][e] = share * (float)c_next[i];
        }
    };
    auto finish = [&](int t, int buf, const float (&uf)[kRows], const float (&zf)[kRows]) {
        float v[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) v[i] = parts[buf][0][r0 + i][lane];
        if (a.d_skip) {                                        // (0 * inf without it)
#pragma unroll
            for (int i = 0; i < kRows; ++i) v[i] = __builtin_fmaf(skip, uf[i], v[i]);
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
#pragma unroll
            for (int w = 1; w < NW; ++w) v[i] += parts[buf][w][r0 + i][lane];
            const float gated = v[i] * silu(zf[i]);
            if (on && t + r0 + i < end)
                *reinterpret_cast<T *>(reinterpret_cast<char *>(y_p) + y_off[i]) = (T)(gate ? gated : v[i]);
        }
        y_p += TT * a.y.ld;
    };
    if (from < end) {
        offsets(min(TT, end - from) - 1);
        load();
        stage(from, 0);
        fetch(from + TT);
        lds_barrier();
        int buf = 0, t = from;
        for (; t + TT < end; t += TT, buf ^= 1) {
            stage(t + TT, buf ^ 1);
            fetch(t + 2 * TT);
            if (kY && t > from) finish(t - TT, buf ^ 1, u[2], z[2]);
            lds_barrier();
        }
        if (kY && t > from) finish(t - TT, buf ^ 1, u[1], z[1]);
        lds_barrier();
        if (kY) finish(t, buf, u[0], z[0]);
    }
    if (kY && on)
        for (int t = max(from, end) + hw; t < to; t += kHelpers) a.y.row(b, t)[c] = (T)0.0f;
}

// How a scan is split: states a wave, waves a block, parts of the sequence (0: the
// step kernel).
struct ScanPlan {
    int states, waves, chunks, chunk, blocks;
};

inline ScanPlan scan_plan(int batch, int len, int dim, int nstate, int groups) {
    ScanPlan p{};
    if (len <= kScanStepLen) return p;
    p.blocks = (dim / groups + 63) / 64;
    // four waves of the states where that is 4 to 16 a wave (64 states, 256 blocks of 512
    // steps: 16 x 4 110 us, 8 x 8 120; 32 states: 8 x 4 67, 4 x 8 75)
    p.states = nstate <= 16 ? 4 : nstate <= 32 ? 8 : nstate <= 128 ? 16 : 32;
    p.waves = nstate <= 4 ? 1 : nstate <= 8 ? 2 : nstate <= 64 ? 4 : 8;
    // Parts: a first pass over them costs about two thirds of the second, so only where
    // blocks are few, and then about three blocks a CU; and parts of 2 sqrt(len) steps
    // at least, since each walks over those in front of it.  16 states, one part and the
    // split in us: 4096 steps, 24 blocks 283 and 63; 96 blocks 284 and 176; 128 blocks 284
    // and 229; 192 blocks 290 and 331.  256 steps: 24 blocks 22 and 14, 128 blocks 23 and 26.
    const int64_t blocks = (int64_t)batch * groups * p.blocks;
    const int cus = device_cus();
    int64_t chunks = 1;
    if (blocks <= (len < 512 ? cus * 3 / 8 : cus / 2)) {
        chunks = 3 * cus / blocks;
        while (chunks * chunks * 4 > len) --chunks;
    }
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
        hipLaunchKernelGGL((scan_tile_kernel<T, S, NW, TT, kWhole>), grid, dim3(64 * (NW + kHelpers)), 0, st, a, sp);
    } else {
        hipLaunchKernelGGL((scan_tile_kernel<T, S, NW, TT, kEnds>), dim3(grid.x, grid.y - 1), dim3(64 * (NW + kHelpers)), 0, st, a, sp);
        hipLaunchKernelGGL((scan_tile_kernel<T, S, NW, TT, kParts>), grid, dim3(64 * (NW + kHelpers)), 0, st, a, sp);
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
        case 804: return launch_scan_tiles<T, 8, 4, 16>(a, p, ends, st);
        case 1604: return launch_scan_tiles<T, 16, 4, 16>(a, p, ends, st);
        case 1608: return launch_scan_tiles<T, 16, 8, 8>(a, p, ends, st);
        default: return launch_scan_tiles<T, 32, 8, 8>(a, p, ends, st);
    }
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_selective_scan_workspace_size(int batch, int len, int dim, int nstate, int groups, size_t *bytes) {
    clear_error();
    MI_REQUIRE(bytes, MI_ERR_NULL_POINTER, "mi_selective_scan_workspace_size: bytes is required");
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0 && nstate >= 1 && nstate <= kScanMaxStates, MI_ERR_BAD_DIM,
               "mi_selective_scan_workspace_size: a size is negative, or nstate=%d not in [1, %d]", nstate, kScanMaxStates);
    MI_REQUIRE(len <= 1 << 30, MI_ERR_BAD_DIM, "mi_selective_scan_workspace_size: len must be at most 2^30");
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
    MI_REQUIRE(len <= 1 << 30 && (int64_t)groups * nstate <= kScanMaxLd, MI_ERR_BAD_DIM,
               "mi_selective_scan: len must be at most 2^30, groups * nstate at most %lld", (long long)kScanMaxLd);
    if (batch == 0 || dim == 0) return MI_OK;
    MI_REQUIRE(a && (len == 0 || (u && dt && b && c && y)), MI_ERR_NULL_POINTER,
               "mi_selective_scan: u, dt, a, b, c and y are required");
    const ScanPlan plan = scan_plan(batch, len, dim, nstate, groups);
    MI_REQUIRE((int64_t)batch * groups * plan.blocks * (plan.waves + kHelpers) * 64 < ((int64_t)1 << 32), MI_ERR_BAD_DIM,
               "mi_selective_scan: too many groups of few channels for one launch");
    MI_REQUIRE(plan.chunks == 0 || (ldu <= kScanMaxLd && ldt <= kScanMaxLd && ldb <= kScanMaxLd && ldc <= kScanMaxLd &&
                                    ldz <= kScanMaxLd && ldy <= kScanMaxLd),
               MI_ERR_BAD_DIM, "mi_selective_scan: a row stride is above %lld", (long long)kScanMaxLd);
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
