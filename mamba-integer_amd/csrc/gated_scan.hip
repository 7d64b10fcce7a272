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

constexpr int kWaves = 8;                     // of a block with a whole chunk
constexpr int kSteps = 16;                    // of a wave
constexpr int kGatedChunk = kWaves * kSteps;  // steps of a block, and between the saved states
constexpr int kJoin = 8;                      // chunks between the states that are passed on as such

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
    float *dh_in, *sums;                 // sums [batch, chunks, dim]: of p over a chunk's steps
    const int32_t *lens;
    uint32_t *ticket;                    // what the blocks pass on, 0 at first (GatedWords)
    uint64_t *words;
    float rate;
    int batch, len, dim, chunks, groups;
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

// ---------------------------------------------------------------- chunks
// A block has a chunk of a sequence's steps (16 a wave) and 64 C channels, C in a lane
// (4 bytes of a row).  A wave keeps its rows in registers, sums its steps up as one step
// h -> A h + H, and starts from the state in front of it, which comes from the waves
// before it through LDS, and from the chunks before through memory: every block passes
// its chunk's (A, H) on as soon as it has them, and every kJoin-th chunk the state behind
// it.  A block reads at most the last such state and kJoin - 1 sums, so the rows are read
// once, and only every kJoin-th chunk waits for a state; which values are joined in which
// order depends on the chunk alone, not on who was first.
//
// No block waits for one that may not run: a block takes its chunk by a ticket, so those
// in front of it in its sequence were taken before, by blocks that run, and the one with
// the lowest ticket waits for none.  A word holds a value and a mark beside it, so it
// needs no other memory to be seen in order.
struct GatedWords {
    uint64_t *p;
    int64_t seq, dim;      // words of a sequence's chunk, channels
    int batch;

    __device__ __forceinline__ explicit GatedWords(const GatedArgs &a)
        : p(a.words), seq((int64_t)a.dim * 2), dim(a.dim), batch(a.batch) {}
    // the sums of chunk k of the order, and the state behind it for every last one of kJoin
    __device__ __forceinline__ uint64_t *sums(int b, int k) const { return p + ((int64_t)k * batch + b) * seq; }
    __device__ __forceinline__ uint64_t *state(int b, int k, int chunks) const {
        return p + (int64_t)chunks * batch * seq + ((int64_t)(k / kJoin) * batch + b) * dim;
    }
    static size_t count(int64_t batch, int64_t dim, int64_t chunks) {
        return (size_t)(batch * dim * (2 * chunks + chunks / kJoin));
    }
};
__device__ __forceinline__ void pass_on(uint64_t *p, float v) {
    __hip_atomic_store(p, (uint64_t)1 << 32 | __builtin_bit_cast(uint32_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// (bounded, so that a fault elsewhere ends in NaN and not in a hang)
__device__ __forceinline__ float wait_for(const uint64_t *p) {
    for (int n = 0; n < (1 << 22); ++n) {
        const uint64_t v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (v >> 32) return __builtin_bit_cast(float, (uint32_t)v);
        __builtin_amdgcn_s_sleep(1);
    }
    return __builtin_nanf("");
}

__global__ __launch_bounds__(256) void gated_clear_kernel(uint64_t *p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

// What a block works on.
struct GatedBlock {
    int chunk, b, group;
};
template <bool MANY>
__device__ __forceinline__ GatedBlock gated_block(const GatedArgs &a, uint32_t *lds) {
    uint32_t at = blockIdx.x;
    if constexpr (MANY) {
        if (threadIdx.x == 0) *lds = atomicAdd(a.ticket, 1u);
        __syncthreads();
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)*lds);
    }
    const uint32_t per = (uint32_t)a.groups * (uint32_t)a.batch, rest = at % per;
    return {(int)(at / per), (int)(rest / (uint32_t)a.groups), (int)(rest % (uint32_t)a.groups)};
}

// C channels of a row from the lane's first one on.  FULL: every lane of the wave has them.
template <int C, bool FULL, class T>
__device__ __forceinline__ Packed<T, C> load_channels(const T *row, int c, int dim) {
    if constexpr (FULL) return load_packed<C>(row + c);
    Packed<T, C> v;
#pragma unroll
    for (int j = 0; j < C; ++j) v.v[j] = c + j < dim ? row[c + j] : T(0);
    return v;
}
template <int C, bool FULL, class T>
__device__ __forceinline__ void store_channels(T *row, int c, int dim, const Packed<T, C> &v) {
    if constexpr (FULL)
        store_packed<C>(row + c, v);
    else {
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c + j < dim) row[c + j] = v.v[j];
    }
}

// The sums of the block's waves, and of the chunks in front of it.
template <int C, int WAVES, bool MANY>
struct GatedLds {
    static constexpr int kBefore = MANY ? kJoin : 1;
    float a[WAVES][64 * C], h[WAVES][64 * C], first[64 * C];
    float before_a[kBefore][64 * C], before_h[kBefore][64 * C];
};
template <int C>
struct GatedLds<C, 1, false> {};

// The state in front of chunk `at` > 0 of the order, from what the chunks before passed on;
// this block's (A, H) are passed on first.  Chunk 0 passes the state behind it on, from
// `first`, which is its own.  Every wave; LDS holds the waves' sums.  `behind`: whether
// chunks follow.  BACKWARDS: the waves' order.
template <int C, int WAVES, bool BACKWARDS>
__device__ __forceinline__ void join_chunks(const GatedArgs &a, GatedLds<C, WAVES, true> &s, int b, int at, bool behind, int c,
                                            const float *first, float *carry) {
    static_assert(WAVES >= kJoin, "a wave for each chunk that is read");
    const int lane = threadIdx.x & 63, wave = wave_id();
    const GatedWords words(a);
    float A[C], H[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        carry[j] = first[j];
        A[j] = 1.0f;
        H[j] = at == 0 ? first[j] : 0.0f;
    }
    if (wave == 0 && behind) {
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int v = BACKWARDS ? WAVES - 1 - w : w;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                H[j] = __builtin_fmaf(s.a[v][lane * C + j], H[j], s.h[v][lane * C + j]);
                A[j] *= s.a[v][lane * C + j];
            }
        }
        uint64_t *p = words.sums(b, at);
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c + j < a.dim) {
                pass_on(p + c + j, H[j]);
                if (at > 0) pass_on(p + a.dim + c + j, A[j]);
            }
    }
    if (at == 0) return;
    const int base = at / kJoin * kJoin;
    // wave w < kJoin - 1 reads the sums of chunk base + w, wave kJoin - 1 the state in front of base
    if (wave < kJoin - 1 ? base + wave < at : wave == kJoin - 1 && base > 0) {
        const uint64_t *p = wave < kJoin - 1 ? words.sums(b, base + wave) : words.state(b, base - 1, a.chunks);
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c + j < a.dim) {
                s.before_h[wave][lane * C + j] = wait_for(p + c + j);
                if (wave < kJoin - 1 && base + wave > 0) s.before_a[wave][lane * C + j] = wait_for(p + a.dim + c + j);
            }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C; ++j) {
        float h = base > 0 ? s.before_h[kJoin - 1][lane * C + j] : s.before_h[0][lane * C + j];
        for (int w = base > 0 ? 0 : 1; base + w < at; ++w)
            h = __builtin_fmaf(s.before_a[w][lane * C + j], h, s.before_h[w][lane * C + j]);
        carry[j] = h;
    }
    if (wave == 0 && at % kJoin == kJoin - 1 && behind) {
        uint64_t *p = words.state(b, at, a.chunks);
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c + j < a.dim) pass_on(p + c + j, __builtin_fmaf(A[j], carry[j], H[j]));
    }
}

template <class T, int C, int STEPS, int WAVES, bool MANY, bool FULL>
__device__ __forceinline__ void gated_forward(const GatedArgs &a, GatedLds<C, WAVES, MANY> &s, const GatedBlock &at) {
    const int lane = threadIdx.x & 63, wave = wave_id(), b = at.b;
    const int c = (at.group * 64 + lane) * C, len = gated_len(a, b);
    const int start = at.chunk * STEPS * WAVES, t0 = start + wave * STEPS;
    Packed<T, C> zero;
#pragma unroll
    for (int j = 0; j < C; ++j) zero.v[j] = T(0);
    if (start >= len && at.chunk > 0) {      // past the sequence: zeros
#pragma unroll
        for (int t = 0; t < STEPS; ++t)
            if (t0 + t < a.len) store_channels<C, FULL>(a.y.row<T>(b, t0 + t), c, a.dim, zero);
        return;
    }
    float av[STEPS][C], bv[STEPS][C], A[C], H[C];
    Packed<T, C> z[STEPS];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        A[j] = 1.0f;
        H[j] = 0.0f;
    }
    if (t0 < len) {
        Packed<T, C> x[STEPS], r[STEPS], i[STEPS];
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int row = min(t0 + t, len - 1);
            r[t] = load_channels<C, FULL>(a.r.row<const T>(b, row), c, a.dim);
            i[t] = load_channels<C, FULL>(a.i.row<const T>(b, row), c, a.dim);
            x[t] = load_channels<C, FULL>(a.x.row<const T>(b, row), c, a.dim);
            if (a.z.p) z[t] = load_channels<C, FULL>(a.z.row<const T>(b, row), c, a.dim);
        }
        float k[C];
#pragma unroll
        for (int j = 0; j < C; ++j) k[j] = FULL || c + j < a.dim ? a.rate * gated_softplus(a.decay[c + j]) : 0.0f;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const GatedStep g(k[j], (float)x[t].v[j], (float)r[t].v[j], (float)i[t].v[j]);
                av[t][j] = t0 + t < len ? g.a : 1.0f;
                bv[t][j] = t0 + t < len ? g.b : 0.0f;
                H[j] = __builtin_fmaf(av[t][j], H[j], bv[t][j]);
                A[j] *= av[t][j];
            }
        }
    }
    const int64_t state = (int64_t)b * a.dim + c;
    float h[C];
    // (one wave reads h_in, so that it has been read before a later chunk, or wave, writes
    // h_out in its place)
#pragma unroll
    for (int j = 0; j < C; ++j) h[j] = a.h_in && wave == 0 && at.chunk == 0 && (FULL || c + j < a.dim) ? a.h_in[state + j] : 0.0f;
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            s.a[wave][lane * C + j] = A[j];
            s.h[wave][lane * C + j] = H[j];
            if (wave == 0) s.first[lane * C + j] = h[j];
        }
        __syncthreads();
        float first[C];
#pragma unroll
        for (int j = 0; j < C; ++j) h[j] = first[j] = s.first[lane * C + j];
        if constexpr (MANY) join_chunks<C, WAVES, false>(a, s, b, at.chunk, len - start > STEPS * WAVES, c, first, h);
    }
    if (a.saved && wave == 0) {
        float *p = a.saved + ((int64_t)b * a.chunks + at.chunk) * a.dim;
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (FULL || c + j < a.dim) p[c + j] = h[j];
    }
    if constexpr (WAVES > 1)
        for (int w = 0; w < wave; ++w) {
#pragma unroll
            for (int j = 0; j < C; ++j) h[j] = __builtin_fmaf(s.a[w][lane * C + j], h[j], s.h[w][lane * C + j]);
        }
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
        if (t0 + t >= a.len) break;
        Packed<T, C> y = zero;
        if (t0 + t < len) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                h[j] = __builtin_fmaf(av[t][j], h[j], bv[t][j]);
                y.v[j] = (T)(a.z.p ? h[j] * silu((float)z[t].v[j]) : h[j]);
            }
        }
        store_channels<C, FULL>(a.y.row<T>(b, t0 + t), c, a.dim, y);
    }
    if (a.h_out && wave == WAVES - 1 && start + STEPS * WAVES >= len) {
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (FULL || c + j < a.dim) a.h_out[state + j] = h[j];
    }
}

template <class T, int C, int STEPS, int WAVES, bool MANY>
__global__ __launch_bounds__(WAVES * 64) void gated_scan_kernel(GatedArgs a) {
    __shared__ GatedLds<C, WAVES, MANY> s;
    __shared__ uint32_t ticket;
    const GatedBlock at = gated_block<MANY>(a, &ticket);
    if ((at.group + 1) * 64 * C <= a.dim)
        gated_forward<T, C, STEPS, WAVES, MANY, true>(a, s, at);
    else
        gated_forward<T, C, STEPS, WAVES, MANY, false>(a, s, at);
}

template <class T, int C, int STEPS, int WAVES, bool MANY, bool FULL>
__device__ __forceinline__ void gated_backward(const GatedArgs &a, GatedLds<C, WAVES, MANY> &s, GatedBlock at) {
    const int lane = threadIdx.x & 63, wave = wave_id(), b = at.b;
    at.chunk = a.chunks - 1 - at.chunk;      // from the last one
    const int c = (at.group * 64 + lane) * C, len = gated_len(a, b);
    const int start = at.chunk * STEPS * WAVES, t0 = start + wave * STEPS;
    const int64_t kept = ((int64_t)b * a.chunks + at.chunk) * a.dim;
    Packed<T, C> zero;
#pragma unroll
    for (int j = 0; j < C; ++j) zero.v[j] = T(0);
    const auto store = [&](const GatedRows &to, int t, const Packed<T, C> &v) {
        if (to.p) store_channels<C, FULL>(to.row<T>(b, t), c, a.dim, v);
    };
    if (start >= len) {      // past the sequence: zeros
#pragma unroll
        for (int t = 0; t < STEPS; ++t)
            if (t0 + t < a.len) {
                store(a.dx, t0 + t, zero);
                store(a.dr, t0 + t, zero);
                store(a.di, t0 + t, zero);
                store(a.dz, t0 + t, zero);
            }
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (wave == 0 && (FULL || c + j < a.dim)) {
                a.sums[kept + c + j] = 0.0f;
                if (a.dh_in && at.chunk == 0) a.dh_in[(int64_t)b * a.dim + c + j] = 0.0f;
            }
        return;
    }
    const int last = (len - 1) / (STEPS * WAVES);
    Packed<T, C> x[STEPS], r[STEPS], i[STEPS], z[STEPS], dy[STEPS];
    float av[STEPS][C], hv[STEPS][C], A[C], H[C], G[C], k[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        A[j] = 1.0f;
        H[j] = 0.0f;
        G[j] = 0.0f;
        k[j] = FULL || c + j < a.dim ? a.rate * gated_softplus(a.decay[c + j]) : 0.0f;
    }
    if (t0 < len) {
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const int row = min(t0 + t, len - 1);
            r[t] = load_channels<C, FULL>(a.r.row<const T>(b, row), c, a.dim);
            i[t] = load_channels<C, FULL>(a.i.row<const T>(b, row), c, a.dim);
            x[t] = load_channels<C, FULL>(a.x.row<const T>(b, row), c, a.dim);
            dy[t] = load_channels<C, FULL>(a.y.row<const T>(b, row), c, a.dim);
            if (a.z.p) z[t] = load_channels<C, FULL>(a.z.row<const T>(b, row), c, a.dim);
        }
        // hv: the state behind each step, from 0 in front of the wave
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const GatedStep g(k[j], (float)x[t].v[j], (float)r[t].v[j], (float)i[t].v[j]);
                av[t][j] = t0 + t < len ? g.a : 1.0f;
                hv[t][j] = t0 + t < len ? g.b : 0.0f;       // (the input until the state in front is known)
                H[j] = __builtin_fmaf(av[t][j], H[j], hv[t][j]);
                A[j] *= av[t][j];
            }
        }
        // G: a g of the wave's first step, from 0 behind it
#pragma unroll
        for (int t = STEPS - 1; t >= 0; --t) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                float dh = (float)dy[t].v[j];
                if (a.z.p) dh *= silu((float)z[t].v[j]);
                G[j] = t0 + t < len ? av[t][j] * (dh + G[j]) : G[j];
            }
        }
    }
    float h[C], carry[C];
    if constexpr (WAVES > 1) {
        // the states in front of the waves, then the gradients behind them
#pragma unroll
        for (int j = 0; j < C; ++j) {
            s.a[wave][lane * C + j] = A[j];
            s.h[wave][lane * C + j] = H[j];
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
        carry[j] = 0.0f;
        h[j] = FULL || c + j < a.dim ? a.saved[kept + c + j] : 0.0f;
    }
    if constexpr (WAVES > 1) {
        for (int w = 0; w < wave; ++w) {
#pragma unroll
            for (int j = 0; j < C; ++j) h[j] = __builtin_fmaf(s.a[w][lane * C + j], h[j], s.h[w][lane * C + j]);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C; ++j) s.h[wave][lane * C + j] = G[j];
        __syncthreads();
        const float none[C] = {};
        if constexpr (MANY) join_chunks<C, WAVES, true>(a, s, b, last - at.chunk, at.chunk > 0, c, none, carry);
        for (int w = WAVES - 1; w > wave; --w) {
#pragma unroll
            for (int j = 0; j < C; ++j) carry[j] = __builtin_fmaf(s.a[w][lane * C + j], carry[j], s.h[w][lane * C + j]);
        }
    }
    float sum[C];
#pragma unroll
    for (int j = 0; j < C; ++j) sum[j] = 0.0f;
    if (t0 < len) {
        // hv: the state in front of each step
        float behind[C];
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float was = h[j];
                h[j] = __builtin_fmaf(av[t][j], h[j], hv[t][j]);
                hv[t][j] = was;
            }
        }
#pragma unroll
        for (int j = 0; j < C; ++j) behind[j] = h[j];
#pragma unroll
        for (int t = STEPS - 1; t >= 0; --t) {
            if (t0 + t >= a.len) continue;
            Packed<T, C> dx = zero, dr = zero, di = zero, dz = zero;
            if (t0 + t < len) {
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    const float xf = (float)x[t].v[j];
                    const GatedStep st(k[j], xf, (float)r[t].v[j], (float)i[t].v[j]);
                    float dh = (float)dy[t].v[j];
                    if (a.z.p) {
                        const float zf = (float)z[t].v[j], sz = sigmoid(zf), act = silu(zf);
                        dz.v[j] = (T)(dh * behind[j] * __builtin_fmaf(act, 1.0f - sz, sz));
                        dh *= act;
                    }
                    const float g = dh + carry[j];
                    // (the hardware root takes a subnormal for 0, its reciprocal is infinite there)
                    const float inv = st.m2 >= 0x1p-126f ? __builtin_amdgcn_rsqf(st.m2) : 0.0f, m = st.m2 * inv;
                    const float p = g * (st.q * xf * st.a * st.a * (st.n * inv) - st.n * st.a * hv[t][j]);
                    dx.v[j] = (T)(g * m * st.q);
                    di.v[j] = (T)(g * st.b * (1.0f - st.q));
                    dr.v[j] = (T)(p * (1.0f - st.s));
                    sum[j] += p;
                    carry[j] = st.a * g;
                    behind[j] = hv[t][j];
                }
            }
            store(a.dx, t0 + t, dx);
            store(a.dr, t0 + t, dr);
            store(a.di, t0 + t, di);
            store(a.dz, t0 + t, dz);
        }
    } else {
#pragma unroll
        for (int t = 0; t < STEPS; ++t)
            if (t0 + t < a.len) {
                store(a.dx, t0 + t, zero);
                store(a.dr, t0 + t, zero);
                store(a.di, t0 + t, zero);
                store(a.dz, t0 + t, zero);
            }
    }
    if constexpr (WAVES > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C; ++j) s.h[wave][lane * C + j] = sum[j];
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        if constexpr (WAVES > 1)
            for (int w = 1; w < WAVES; ++w) sum[j] += s.h[w][lane * C + j];
        if (FULL || c + j < a.dim) {
            a.sums[kept + c + j] = sum[j];
            if (a.dh_in && at.chunk == 0) a.dh_in[(int64_t)b * a.dim + c + j] = carry[j];
        }
    }
}

template <class T, int C, int STEPS, int WAVES, bool MANY>
__global__ __launch_bounds__(WAVES * 64) void gated_scan_backward_kernel(GatedArgs a) {
    __shared__ GatedLds<C, WAVES, MANY> s;
    __shared__ uint32_t ticket;
    const GatedBlock at = gated_block<MANY>(a, &ticket);
    if ((at.group + 1) * 64 * C <= a.dim)
        gated_backward<T, C, STEPS, WAVES, MANY, true>(a, s, at);
    else
        gated_backward<T, C, STEPS, WAVES, MANY, false>(a, s, at);
}

// ddecay from the sums of p over the chunks: 16 waves share them.
__global__ __launch_bounds__(1024) void gated_decay_kernel(const float *sums, const float *decay, float *out, int64_t rows, int dim) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = wave_id(), c = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < dim)
        for (int64_t j = wave; j < rows; j += 16) s += sums[j * dim + c];
    part[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || c >= dim) return;
    for (int w = 1; w < 16; ++w) s += part[w][lane];
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
    MI_REQUIRE(((int64_t)len + kGatedChunk - 1) / kGatedChunk * batch * (((int64_t)dim + 63) / 64) < (1 << 23), MI_ERR_BAD_DIM,
               "%s: ceil(len / %d) * batch * ceil(dim / 64) must be below 2^23", fn, kGatedChunk);
    return MI_OK;
}

inline int gated_chunks(int len) { return max(1, (len + kGatedChunk - 1) / kGatedChunk); }
// bytes of the words and the ticket in front of them, none for one chunk
inline size_t gated_word_bytes(int batch, int len, int dim) {
    const int chunks = gated_chunks(len);
    return chunks > 1 ? 16 + GatedWords::count(batch, dim, chunks) * sizeof(uint64_t) : 0;
}

// Launches F<T, C, STEPS, WAVES, MANY>: one wave with as many steps as there are up to 16,
// blocks of 8 waves beyond.
template <template <class, int, int, int, bool> class F, class T>
void launch_gated(GatedArgs a, void *workspace, hipStream_t st) {
    constexpr int C = 4 / sizeof(T);
    a.groups = (a.dim + 64 * C - 1) / (64 * C);
    const auto launch = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)a.groups * (unsigned)a.batch * (unsigned)a.chunks), dim3(waves * 64), 0, st, a);
    };
    if (a.chunks > 1) {
        const int64_t n = 2 + (int64_t)GatedWords::count(a.batch, a.dim, a.chunks);
        a.ticket = static_cast<uint32_t *>(workspace);
        a.words = static_cast<uint64_t *>(workspace) + 2;
        hipLaunchKernelGGL(gated_clear_kernel, dim3((unsigned)min((n + 1023) / 1024, (int64_t)2048)), dim3(256), 0, st,
                           static_cast<uint64_t *>(workspace), n);
        launch(F<T, C, kSteps, kWaves, true>::kernel, kWaves);
    } else if (a.len <= 1) {
        launch(F<T, C, 1, 1, false>::kernel, 1);
    } else if (a.len <= 4) {
        launch(F<T, C, 4, 1, false>::kernel, 1);
    } else if (a.len <= kSteps) {
        launch(F<T, C, kSteps, 1, false>::kernel, 1);
    } else if (a.len <= 4 * kSteps) {
        launch(F<T, C, kSteps, 4, false>::kernel, 4);
    } else {
        launch(F<T, C, kSteps, kWaves, false>::kernel, kWaves);
    }
}
template <class T, int C, int STEPS, int WAVES, bool MANY>
struct Forward {
    static constexpr auto kernel = gated_scan_kernel<T, C, STEPS, WAVES, MANY>;
};
template <class T, int C, int STEPS, int WAVES, bool MANY>
struct Backward {
    static constexpr auto kernel = gated_scan_backward_kernel<T, C, STEPS, WAVES, MANY>;
};

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_gated_scan_sizes(int batch, int len, int dim, size_t *forward_bytes, size_t *backward_bytes,
                                         size_t *saved_bytes) {
    clear_error();
    MI_REQUIRE(forward_bytes && backward_bytes && saved_bytes, MI_ERR_NULL_POINTER, "mi_gated_scan_sizes: the sizes are required");
    if (const mi_status st = gated_dims("mi_gated_scan_sizes", batch, len, dim)) return st;
    *forward_bytes = gated_word_bytes(batch, len, dim);
    *backward_bytes = gated_word_bytes(batch, len, dim) + (size_t)batch * gated_chunks(len) * dim * sizeof(float);
    *saved_bytes = len ? (size_t)batch * gated_chunks(len) * dim * sizeof(float) : 0;
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
    a.decay = decay, a.h_in = h_in, a.h_out = h_out, a.saved = len ? saved : nullptr, a.lens = lens, a.rate = rate;
    a.batch = batch, a.len = len, a.dim = dim, a.chunks = gated_chunks(len);
    const size_t need = gated_word_bytes(batch, len, dim);
    MI_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG,
               "mi_gated_scan: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    MI_REQUIRE(need == 0 || aligned(workspace, 16), MI_ERR_BAD_ALIGNMENT, "mi_gated_scan: the workspace must be 16-byte aligned");
    with_type(type, [&](auto t) { launch_gated<Forward, decltype(t)>(a, workspace, as_stream(stream)); });
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
    a.decay = decay, a.saved = const_cast<float *>(saved), a.dh_in = dh_in, a.lens = lens;
    a.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + gated_word_bytes(batch, len, dim));
    a.rate = rate, a.batch = batch, a.len = len, a.dim = dim, a.chunks = gated_chunks(len);
    const hipStream_t st = as_stream(stream);
    if (batch > 0) with_type(type, [&](auto t) { launch_gated<Backward, decltype(t)>(a, workspace, st); });
    if (ddecay)
        hipLaunchKernelGGL(gated_decay_kernel, dim3((unsigned)((dim + 63) / 64)), dim3(1024), 0, st, a.sums, decay, ddecay,
                           (int64_t)batch * a.chunks, dim);
    return check_launch("mi_gated_scan_backward");
}
