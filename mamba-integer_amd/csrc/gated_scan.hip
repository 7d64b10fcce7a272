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
#include <algorithm>
#include <type_traits>

#include "float_ops.hpp"

namespace mi {

// Steps of a wave and waves of a block with a whole chunk.  Forwards 16 x 16: 8 x 2048 x 1536 in
// bf16 68.6 us, 1 x 16384 x 1536 in float32 86.6; 8 waves 69.7 and 88.3, 4 waves 93 and 111, waves
// of 8 steps with two channels a lane 78 and 101.  A wave takes 73 registers, so a CU has one
// block; held to 64 for two of them it spills: 77.6 and 90.5.  What bounds it is that block's
// chain of load, join and store (the vector units work in 38 us), in float32 HBM (4.8 TB/s).  Backwards 4 waves of 16, since a wave there
// takes 160 registers and a block of 8 leaves no room for a second one: 133 us against 166.
constexpr int kSteps = 16, kWaves = 16;
constexpr int kStepsBack = 16, kWavesBack = 4;
constexpr int kChunk = kSteps * kWaves, kChunkBack = kStepsBack * kWavesBack;
static_assert(kChunkBack % kSteps == 0, "a wave of the forward pass saves the state in front of it");

struct GatedRows {
    void *p;
    int64_t ld, bs;
    template <class T>
    __device__ __forceinline__ T *row(int64_t b, int64_t t) const {
        return static_cast<T *>(p) + (b * bs + t * ld);
    }
};

struct GatedArgs {
    GatedRows x, r, i, z, y;             // y: dy in a backward pass
    GatedRows dx, dr, di, dz;
    const float *decay, *h_in;
    float *h_out, *saved;                // saved [batch, kept, dim]: the state in front of each chunk of the backward pass
    float *dh_in, *sums;                 // sums [batch, chunks, dim]: of p over a chunk's steps
    const int32_t *lens;
    uint32_t *ticket;                    // what the blocks pass on, 0 at first (GatedWords)
    uint64_t *words;
    float rate;
    int batch, len, dim, chunks, kept, groups;
};

__device__ __forceinline__ int gated_len(const GatedArgs &a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.len) : a.len;
}
// log(1 + exp(v)) = max(v, 0) + log(w) + (e - (w - 1)) / w, e = exp(-|v|), w = 1 + e rounded: the
// last term is what the rounding of w lost (w = 1 wherever it matters).  The exponent's
// product with log2 e is kept in two parts, so a low v, whose value is e, has e's precision.
// (The maximum that keeps a NaN: past -1e4 e is 0, and the parts of an infinite product none.)
__device__ __forceinline__ float gated_softplus(float v) {
    const float u = __builtin_elementwise_maximum(-fabsf(v), -1e4f), p = u * 1.44269504f;
    const float e = __builtin_amdgcn_exp2f(p);
    const float lost = __builtin_fmaf(u, 1.44269504f, -p) + u * 1.925963033e-8f;      // log2 e's next bits
    const float f = __builtin_fmaf(e, lost * 0.693147181f, e), w = 1.0f + f;
    return fmaxf(v, 0.0f) + __builtin_fmaf(__builtin_amdgcn_logf(w), 0.693147181f, f - (w - 1.0f));
}
__device__ __forceinline__ float sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}
// 1 - exp(-2 n) for n >= 0 and a = exp(-n).  Where the difference would cancel, v times a
// polynomial of (1 - exp(-v)) / v, v = 2 n: of the six coefficients that leave the least
// relative error on [0, 0.5], 0.12 * 2^-24.
__device__ __forceinline__ float one_minus_square(float n, float a) {
    const float v = 2.0f * n;
    float s = __builtin_fmaf(v, -0.0011216348502784967f, 0.008187386207282543f);
    s = __builtin_fmaf(v, s, -0.041629090905189514f);
    s = __builtin_fmaf(v, s, 0.16666224598884583f);
    s = __builtin_fmaf(v, s, -0.4999998211860657f);
    s = __builtin_fmaf(v, s, 1.0f) * v;
    asm("" : "+v"(s));      // (selected, not branched over)
    return v < 0.5f ? s : __builtin_fmaf(-a, a, 1.0f);
}

// The decay of many steps goes as its root r = exp(-sum of n / 2), held at 2^-126 where it would
// be flushed to zero: a product of the decays themselves loses a state of up to 2^128 that has
// not decayed yet, and makes a NaN of an infinite one.  (A NaN among the n is in the sum beside.)
constexpr float kLeastRoot = 0x1p-126f;
__device__ __forceinline__ float decay_root(float n) { return fmaxf(__builtin_amdgcn_exp2f(-0.72134752f * n), kLeastRoot); }
__device__ __forceinline__ float after_steps(float root, float h, float sum) { return __builtin_fmaf(root, root * h, sum); }

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
// A block has a chunk of a sequence's steps (16 a wave) and 64 C channels, C in a lane.  A
// wave keeps its rows in registers, sums its steps up as one step
// h -> A^2 h + H, and starts from the state in front of it, which comes from the waves
// before it through LDS, and from the chunks before through memory: every block passes
// its chunk's (A, H) on as soon as it has them, and every kJoin-th chunk the state behind
// it.  A block reads at most the last such state and JOIN - 1 sums, so the rows are read
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
    // the sums of chunk k of the order, and the state behind it for every last one of JOIN
    __device__ __forceinline__ uint64_t *sums(int b, int k) const { return p + ((int64_t)k * batch + b) * seq; }
    template <int JOIN>
    __device__ __forceinline__ uint64_t *state(int b, int k, int chunks) const {
        return p + (int64_t)chunks * batch * seq + ((int64_t)(k / JOIN) * batch + b) * dim;
    }
    static size_t count(int64_t batch, int64_t dim, int64_t chunks, int join) {
        return (size_t)(batch * dim * (2 * chunks + chunks / join));
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

// What a block works on: a chunk of a sequence and a group of channels.
struct GatedTile {
    int b, chunk, group, len, start;
    bool full;      // every lane has its channels, and the sequence fills the chunk

    // BACKWARDS: the last chunk first
    template <int C, int CHUNK, bool BACKWARDS, bool MANY, class Lds>
    static __device__ __forceinline__ GatedTile take(const GatedArgs &a, Lds &s) {
        uint32_t at = blockIdx.x;
        if constexpr (MANY) {
            if (threadIdx.x == 0) s.ticket = atomicAdd(a.ticket, 1u);
            __syncthreads();
            at = (uint32_t)__builtin_amdgcn_readfirstlane((int)s.ticket);
        }
        const uint32_t per = (uint32_t)a.groups * (uint32_t)a.batch, rest = at % per;
        GatedTile t;
        t.chunk = BACKWARDS ? a.chunks - 1 - (int)(at / per) : (int)(at / per);
        t.b = (int)(rest / (uint32_t)a.groups);
        t.group = (int)(rest % (uint32_t)a.groups);
        t.len = gated_len(a, t.b);
        t.start = t.chunk * CHUNK;
        t.full = (t.group + 1) * 64 * C <= a.dim && t.start + CHUNK <= t.len;
        return t;
    }
};

// Rows of a tensor from row (b, t) on, and C channels of each from the lane's first one on.
// The row's address is the wave's, the channel's offset the lane's, which keeps a row's
// access to one instruction.  FULL: every lane of the wave has its channels.
template <class T>
struct Cursor {
    T *p;
    int64_t step;
    __device__ __forceinline__ Cursor(const GatedRows &r, int b, int t) : p(r.row<T>(b, t)), step(r.ld) {}
    __device__ __forceinline__ void next(bool more = true) { p += more ? step : 0; }
    __device__ __forceinline__ void back() { p -= step; }

    template <int C, bool FULL>
    __device__ __forceinline__ Packed<std::remove_const_t<T>, C> load(uint32_t c, int dim) const {
        if constexpr (FULL) return load_packed<C>(p + c);
        Packed<std::remove_const_t<T>, C> v;
#pragma unroll
        for (int j = 0; j < C; ++j) v.v[j] = (int)c + j < dim ? p[c + j] : T(0);
        return v;
    }
    template <int C, bool FULL>
    __device__ __forceinline__ void store(uint32_t c, int dim, const Packed<T, C> &v) const {
        if constexpr (FULL)
            store_packed<C>(p + c, v);
        else {
#pragma unroll
            for (int j = 0; j < C; ++j)
                if ((int)c + j < dim) p[c + j] = v.v[j];
        }
    }
};

// The sums of the block's waves, and of the chunks in front of it.
template <int C, int WAVES, bool MANY>
struct GatedLds {
    static constexpr int kBefore = MANY ? WAVES : 1;
    float a[WAVES][64 * C], h[WAVES][64 * C], first[64 * C];
    float before_a[kBefore][64 * C], before_h[kBefore][64 * C];
    uint32_t ticket;
};
template <int C>
struct GatedLds<C, 1, false> {};

// The state in front of chunk `at` > 0 of the order, from what the chunks before passed on;
// this block's (A, H) are passed on first.  Chunk 0 passes the state behind it on, from
// `first`, which is its s.  Every wave; LDS holds the waves' sums.  `behind`: whether
// chunks follow.  BACKWARDS: the waves' order.
template <int C, int WAVES, bool BACKWARDS>
__device__ __forceinline__ void join_chunks(const GatedArgs &a, GatedLds<C, WAVES, true> &s, int b, int at, bool behind, int c,
                                            const float *first, float *carry) {
    constexpr int JOIN = WAVES;      // a wave for each chunk that is read, and one for the state
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
                H[j] = after_steps(s.a[v][lane * C + j], H[j], s.h[v][lane * C + j]);
                A[j] = fmaxf(A[j] * s.a[v][lane * C + j], kLeastRoot);
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
    const int base = at / JOIN * JOIN;
    // wave w < JOIN - 1 reads the sums of chunk base + w, wave JOIN - 1 the state in front of base
    if (wave < JOIN - 1 ? base + wave < at : wave == JOIN - 1 && base > 0) {
        const uint64_t *p = wave < JOIN - 1 ? words.sums(b, base + wave) : words.template state<JOIN>(b, base - 1, a.chunks);
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c + j < a.dim) {
                s.before_h[wave][lane * C + j] = wait_for(p + c + j);
                if (wave < JOIN - 1 && base + wave > 0) s.before_a[wave][lane * C + j] = wait_for(p + a.dim + c + j);
            }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C; ++j) {
        float h = base > 0 ? s.before_h[JOIN - 1][lane * C + j] : s.before_h[0][lane * C + j];
        for (int w = base > 0 ? 0 : 1; base + w < at; ++w)
            h = after_steps(s.before_a[w][lane * C + j], h, s.before_h[w][lane * C + j]);
        carry[j] = h;
    }
    if (wave == 0 && at % JOIN == JOIN - 1 && behind) {
        uint64_t *p = words.template state<JOIN>(b, at, a.chunks);
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (c + j < a.dim) pass_on(p + c + j, after_steps(A[j], carry[j], H[j]));
    }
}

// A wave's rows in registers.  FULL: the tile is.  (Past the sequence the last row again.)
template <class T, int C, int STEPS>
struct GatedInputs {
    Packed<T, C> x[STEPS], r[STEPS], i[STEPS];

    template <bool FULL>
    __device__ __forceinline__ void load(const GatedArgs &a, const GatedTile &at, int t0, uint32_t c) {
        if (!FULL && t0 >= at.len) return;
        Cursor<const T> xp(a.x, at.b, t0), rp(a.r, at.b, t0), ip(a.i, at.b, t0);
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            r[t] = rp.template load<C, FULL>(c, a.dim);
            i[t] = ip.template load<C, FULL>(c, a.dim);
            x[t] = xp.template load<C, FULL>(c, a.dim);
            const bool more = FULL || t0 + t + 1 < at.len;
            rp.next(more), ip.next(more), xp.next(more);
        }
    }
    template <bool FULL>
    static __device__ __forceinline__ void load_one(Packed<T, C> *to, const GatedArgs &a, const GatedRows &rows, const GatedTile &at,
                                                    int t0, uint32_t c) {
        if (!FULL && t0 >= at.len) return;
        Cursor<const T> p(rows, at.b, t0);
#pragma unroll
        for (int t = 0; t < STEPS; ++t, p.next(FULL || t0 + t < at.len)) to[t] = p.template load<C, FULL>(c, a.dim);
    }
    // Each step's decay and input, and the wave's steps as one: h -> A^2 h + H.
    template <bool FULL>
    __device__ __forceinline__ void steps(const GatedArgs &a, const GatedTile &at, int t0, const float *k, float (*av)[C], float (*bv)[C],
                                          float *A, float *H, float (*m2)[C] = nullptr) const {
        float n[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            n[j] = 0.0f;
            A[j] = 1.0f;
            H[j] = 0.0f;
        }
        if (!FULL && t0 >= at.len) return;
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
            const bool on = FULL || t0 + t < at.len;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const GatedStep g(k[j], (float)x[t].v[j], (float)r[t].v[j], (float)i[t].v[j]);
                av[t][j] = on ? g.a : 1.0f;
                bv[t][j] = on ? g.b : 0.0f;
                if (m2) m2[t][j] = g.m2;
                H[j] = __builtin_fmaf(av[t][j], H[j], bv[t][j]);
                n[j] += on ? g.n : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < C; ++j) A[j] = decay_root(n[j]);
    }
};

template <int C>
__device__ __forceinline__ uint32_t first_channel(const GatedTile &at) {
    return (uint32_t)(at.group * 64 + (int)(threadIdx.x & 63)) * C;
}
// rate softplus(decay), the largest float where that is infinite: a closed gate then keeps the
// state whatever the decay is.
template <int C, bool FULL>
__device__ __forceinline__ void decays(const GatedArgs &a, uint32_t c, float *k) {
    constexpr float kMost = 0x1.fffffep127f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
        const float soft = FULL || (int)c + j < a.dim ? __builtin_elementwise_minimum(gated_softplus(a.decay[c + j]), kMost) : 0.0f;
        k[j] = __builtin_elementwise_minimum(a.rate * soft, kMost);
    }
}

template <class T, int C, int STEPS, int WAVES, bool MANY>
__global__ __launch_bounds__(WAVES * 64) void gated_scan_kernel(GatedArgs a) {
    using Inputs = GatedInputs<T, C, STEPS>;
    constexpr int CHUNK = STEPS * WAVES;
    __shared__ GatedLds<C, WAVES, MANY> s;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const GatedTile at = GatedTile::take<C, CHUNK, false, MANY>(a, s);
    Inputs in;
    const int b = at.b, t0 = at.start + wave * STEPS;
    const uint32_t c = first_channel<C>(at);
    const auto has = [&](int j) { return (int)c + j < a.dim; };
    // (chunks past the sequence pass nothing on, and nothing reads them)
    const bool work = at.start < at.len || at.chunk == 0;
    float av[STEPS][C], bv[STEPS][C], A[C], H[C], h[C], k[C];
    Packed<T, C> z[STEPS];
    if (at.full) {
        in.template load<true>(a, at, t0, c);
        decays<C, true>(a, c, k);
        in.template steps<true>(a, at, t0, k, av, bv, A, H);
        // (they arrive while the block waits for the state in front of it)
        if (a.z.p) Inputs::template load_one<true>(z, a, a.z, at, t0, c);
    } else {
        in.template load<false>(a, at, t0, c);
        decays<C, false>(a, c, k);
        in.template steps<false>(a, at, t0, k, av, bv, A, H);
        if (a.z.p) Inputs::template load_one<false>(z, a, a.z, at, t0, c);
    }
    const int64_t state = (int64_t)b * a.dim + c;
    // (one wave reads h_in, so that it has been read before a later chunk, or wave, writes
    // h_out in its place)
#pragma unroll
    for (int j = 0; j < C; ++j) h[j] = a.h_in && wave == 0 && at.chunk == 0 && has(j) ? a.h_in[state + j] : 0.0f;
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
        if constexpr (MANY)
            if (work) join_chunks<C, WAVES, false>(a, s, b, at.chunk, at.len - at.start > CHUNK, (int)c, first, h);
    }
    if constexpr (WAVES > 1)
        for (int w = 0; w < wave; ++w) {
#pragma unroll
            for (int j = 0; j < C; ++j) h[j] = after_steps(s.a[w][lane * C + j], h[j], s.h[w][lane * C + j]);
        }
    if (a.saved && t0 % kChunkBack == 0 && t0 < a.len) {
        float *p = a.saved + ((int64_t)b * a.kept + t0 / kChunkBack) * a.dim;
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (has(j)) p[c + j] = h[j];
    }
    Cursor<T> to(a.y, b, t0);
    const auto step = [&](int t) {
        Packed<T, C> y;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            h[j] = __builtin_fmaf(av[t][j], h[j], bv[t][j]);
            y.v[j] = (T)(a.z.p ? h[j] * silu((float)z[t].v[j]) : h[j]);
        }
        return y;
    };
    if (at.full) {
#pragma unroll
        for (int t = 0; t < STEPS; ++t, to.next()) to.template store<C, true>(c, a.dim, step(t));
    } else {
#pragma unroll
        for (int t = 0; t < STEPS; ++t, to.next()) {
            if (t0 + t >= a.len) break;
            Packed<T, C> y;
#pragma unroll
            for (int j = 0; j < C; ++j) y.v[j] = T(0);
            if (t0 + t < at.len) y = step(t);
            to.template store<C, false>(c, a.dim, y);
        }
    }
    if (a.h_out && wave == WAVES - 1 && work && at.start + CHUNK >= at.len) {
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (has(j)) a.h_out[state + j] = h[j];
    }
}

template <class T, int C, int STEPS, int WAVES, bool MANY>
__global__ __launch_bounds__(WAVES * 64) void gated_scan_backward_kernel(GatedArgs a) {
    using Inputs = GatedInputs<T, C, STEPS>;
    constexpr int CHUNK = STEPS * WAVES;
    __shared__ GatedLds<C, WAVES, MANY> s;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const GatedTile at = GatedTile::take<C, CHUNK, true, MANY>(a, s);
    const int b = at.b, t0 = at.start + wave * STEPS;
    const uint32_t c = first_channel<C>(at);
    const auto has = [&](int j) { return (int)c + j < a.dim; };
    const bool work = at.start < at.len;
    float av[STEPS][C], hv[STEPS][C], m2[STEPS][C], A[C], H[C], G[C], k[C], h[C], carry[C], sum[C];
    Inputs in;
    Packed<T, C> z[STEPS], dy[STEPS];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        G[j] = 0.0f;
        carry[j] = 0.0f;
        sum[j] = 0.0f;
        h[j] = work && has(j) ? a.saved[((int64_t)b * a.chunks + at.chunk) * a.dim + c + j] : 0.0f;
    }
    // hv: what a step adds, first; G: a g of the wave's first step, from 0 behind the wave
    const auto load = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        in.template load<FULL>(a, at, t0, c);
        Inputs::template load_one<FULL>(dy, a, a.y, at, t0, c);
        if (a.z.p) Inputs::template load_one<FULL>(z, a, a.z, at, t0, c);
        decays<C, FULL>(a, c, k);
        in.template steps<FULL>(a, at, t0, k, av, hv, A, H, m2);
        if (!FULL && t0 >= at.len) return;
#pragma unroll
        for (int t = STEPS - 1; t >= 0; --t) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                float dh = (float)dy[t].v[j];
                if (a.z.p) dh *= silu((float)z[t].v[j]);
                G[j] = FULL || t0 + t < at.len ? av[t][j] * (dh + G[j]) : G[j];
            }
        }
    };
    if (at.full)
        load(std::true_type{});
    else
        load(std::false_type{});
    if constexpr (WAVES > 1) {
        // the states in front of the waves, then the gradients behind them
#pragma unroll
        for (int j = 0; j < C; ++j) {
            s.a[wave][lane * C + j] = A[j];
            s.h[wave][lane * C + j] = H[j];
        }
        __syncthreads();
        for (int w = 0; w < wave; ++w) {
#pragma unroll
            for (int j = 0; j < C; ++j) h[j] = after_steps(s.a[w][lane * C + j], h[j], s.h[w][lane * C + j]);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C; ++j) s.h[wave][lane * C + j] = G[j];
        __syncthreads();
        const float none[C] = {};
        if constexpr (MANY)
            if (work) join_chunks<C, WAVES, true>(a, s, b, (at.len - 1) / CHUNK - at.chunk, at.chunk > 0, (int)c, none, carry);
        for (int w = WAVES - 1; w > wave; --w) {
#pragma unroll
            for (int j = 0; j < C; ++j) carry[j] = after_steps(s.a[w][lane * C + j], carry[j], s.h[w][lane * C + j]);
        }
    }
    const auto finish = [&](auto full) {
        constexpr bool FULL = decltype(full)::value;
        if (!FULL && t0 >= at.len) return;
        // hv: the state in front of each step; h: behind the last
#pragma unroll
        for (int t = 0; t < STEPS; ++t) {
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float was = h[j];
                h[j] = __builtin_fmaf(av[t][j], h[j], hv[t][j]);
                hv[t][j] = was;
            }
        }
        Cursor<T> xo(a.dx, b, t0 + STEPS - 1), ro(a.dr, b, t0 + STEPS - 1), io(a.di, b, t0 + STEPS - 1), zo(a.dz, b, t0 + STEPS - 1);
#pragma unroll
        for (int t = STEPS - 1; t >= 0; --t, xo.back(), ro.back(), io.back(), zo.back()) {
            if (!FULL && t0 + t >= at.len) continue;
            Packed<T, C> dx, dr, di, dz;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const float xf = (float)in.x[t].v[j], sr = sigmoid((float)in.r[t].v[j]), si = sigmoid((float)in.i[t].v[j]);
                const float n = k[j] * sr, av_ = av[t][j];
                float dh = (float)dy[t].v[j];
                if (a.z.p) {
                    const float zf = (float)z[t].v[j], sz = sigmoid(zf), act = zf * sz;
                    dz.v[j] = (T)(dh * h[j] * __builtin_fmaf(act, 1.0f - sz, sz));
                    dh *= act;
                }
                const float g = dh + carry[j];
                // (the hardware root takes a subnormal for 0, its reciprocal is infinite there)
                const float inv = m2[t][j] >= 0x1p-126f ? __builtin_amdgcn_rsqf(m2[t][j]) : 0.0f, gx = g * m2[t][j] * inv * si;
                // (n may be the largest float, beside decays of 0)
                const float p = g * (n * (si * xf * av_ * av_ * inv - av_ * hv[t][j]));
                dx.v[j] = (T)gx;
                di.v[j] = (T)(gx * xf * (1.0f - si));
                dr.v[j] = (T)(p * (1.0f - sr));
                sum[j] += p;
                carry[j] = av_ * g;
                h[j] = hv[t][j];
            }
            if (a.dx.p) xo.template store<C, FULL>(c, a.dim, dx);
            if (a.dr.p) ro.template store<C, FULL>(c, a.dim, dr);
            if (a.di.p) io.template store<C, FULL>(c, a.dim, di);
            if (a.dz.p) zo.template store<C, FULL>(c, a.dim, dz);
        }
    };
    if (at.full)
        finish(std::true_type{});
    else {
        finish(std::false_type{});
        // zeros past the sequence
        Packed<T, C> zero;
#pragma unroll
        for (int j = 0; j < C; ++j) zero.v[j] = T(0);
        for (int t = max(at.len - t0, 0); t < STEPS && t0 + t < a.len; ++t)
            for (const GatedRows &to : {a.dx, a.dr, a.di, a.dz})
                if (to.p) Cursor<T>(to, b, t0 + t).template store<C, false>(c, a.dim, zero);
    }
    if constexpr (WAVES > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < C; ++j) s.h[wave][lane * C + j] = sum[j];
        __syncthreads();
    }
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            if constexpr (WAVES > 1)
                for (int w = 1; w < WAVES; ++w) sum[j] += s.h[w][lane * C + j];
            if (has(j)) {
                a.sums[((int64_t)b * a.chunks + at.chunk) * a.dim + c + j] = sum[j];
                if (a.dh_in && at.chunk == 0) a.dh_in[(int64_t)b * a.dim + c + j] = carry[j];
            }
        }
    }
}

// ddecay from the sums of p over the chunks: 16 waves share them, in 64 bits (sequences and
// chunks may cancel, and there may be any number of them).
__global__ __launch_bounds__(1024) void gated_decay_kernel(const float *sums, const float *decay, float *out, int64_t rows, int dim) {
    __shared__ double part[16][64];
    const int lane = threadIdx.x & 63, wave = wave_id(), c = blockIdx.x * 64 + lane;
    double s = 0.0;
    if (c < dim) {
        int64_t j = wave;
        for (; j + 7 * 16 < rows; j += 8 * 16) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = sums[(j + i * 16) * dim + c];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; j < rows; j += 16) s += sums[j * dim + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || c >= dim) return;
    for (int w = 1; w < 16; ++w) s += part[w][lane];
    // sigmoid / softplus: 1 - e/2 + ... of e = exp(v) for low v
    const float v = decay[c], e = expf(v);
    const float ratio = v < -9.0f ? 1.0f - 0.5f * e : 1.0f / (1.0f + expf(-v)) / gated_softplus(v);
    out[c] = (float)(s * ratio);
}

mi_status gated_dims(const char *fn, int batch, int len, int dim) {
    MI_REQUIRE(batch >= 0 && len >= 0 && dim >= 0, MI_ERR_BAD_DIM, "%s: a size is negative", fn);
    MI_REQUIRE(batch <= 65535, MI_ERR_BAD_DIM, "%s: batch=%d must be at most 65535", fn, batch);
    MI_REQUIRE(dim <= (1 << 24), MI_ERR_BAD_DIM, "%s: dim=%d must be at most 2^24", fn, dim);
    MI_REQUIRE(len <= (1 << 30), MI_ERR_BAD_DIM, "%s: len=%d must be at most 2^30", fn, len);
    MI_REQUIRE(((int64_t)len + 63) / 64 * batch * (((int64_t)dim + 63) / 64) < (1 << 23), MI_ERR_BAD_DIM,
               "%s: ceil(len / 64) * batch * ceil(dim / 64) must be below 2^23", fn);
    return MI_OK;
}

inline int gated_chunks(int len, int chunk) { return std::max(1, (len + chunk - 1) / chunk); }
// bytes of the words and the ticket in front of them, none for one chunk
inline size_t gated_word_bytes(int batch, int len, int dim, int chunk, int join) {
    const int chunks = gated_chunks(len, chunk);
    return chunks > 1 ? 16 + GatedWords::count(batch, dim, chunks, join) * sizeof(uint64_t) : 0;
}

// Launches F<T, C, STEPS, WAVES, MANY>: one wave with as many steps as there are up to 16,
// blocks of more waves beyond.
template <template <class, int, int, int, bool> class F, class T>
void launch_gated(GatedArgs a, void *workspace, hipStream_t st) {
    using K = F<T, 0, 0, 0, false>;
    constexpr int C = 1;      // channels of a lane (two of 16 bits: the registers of twice the steps, 93 us)
    a.chunks = gated_chunks(a.len, K::kAll);
    a.kept = gated_chunks(a.len, kChunkBack);
    a.groups = (a.dim + 64 * C - 1) / (64 * C);
    const unsigned tiles = (unsigned)a.groups * (unsigned)a.batch * (unsigned)a.chunks;
    const auto launch = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, dim3(tiles), dim3(waves * 64), 0, st, a); };
    if (a.chunks > 1) {
        const int64_t n = 2 + (int64_t)GatedWords::count(a.batch, a.dim, a.chunks, K::kLast);
        a.ticket = static_cast<uint32_t *>(workspace);
        a.words = static_cast<uint64_t *>(workspace) + 2;
        // (std::min: the runtime's own on the host takes ints)
        hipLaunchKernelGGL(gated_clear_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 4096)), dim3(256), 0, st,
                           static_cast<uint64_t *>(workspace), n);
        launch(F<T, C, K::kEach, K::kLast, true>::kernel, K::kLast);
    } else if (a.len <= 1) {
        launch(F<T, C, 1, 1, false>::kernel, 1);
    } else if (a.len <= 4) {
        launch(F<T, C, 4, 1, false>::kernel, 1);
    } else if (a.len <= 16) {
        launch(F<T, C, 16, 1, false>::kernel, 1);
    } else if (K::kLast > 4 && a.len <= 64) {
        launch(F<T, C, 16, 4, false>::kernel, 4);
    } else {
        launch(F<T, C, K::kEach, K::kLast, false>::kernel, K::kLast);
    }
}
template <class T, int C, int STEPS, int WAVES, bool MANY>
struct Forward {
    static constexpr int kEach = kSteps, kLast = kWaves, kAll = kChunk;
    static constexpr auto kernel = gated_scan_kernel<T, C, STEPS, WAVES, MANY>;
};
template <class T, int C, int STEPS, int WAVES, bool MANY>
struct Backward {
    static constexpr int kEach = kStepsBack, kLast = kWavesBack, kAll = kChunkBack;
    static constexpr auto kernel = gated_scan_backward_kernel<T, C, STEPS, WAVES, MANY>;
};
// (the sizes alone)
template <class T>
struct Forward<T, 0, 0, 0, false> {
    static constexpr int kEach = kSteps, kLast = kWaves, kAll = kChunk;
};
template <class T>
struct Backward<T, 0, 0, 0, false> {
    static constexpr int kEach = kStepsBack, kLast = kWavesBack, kAll = kChunkBack;
};

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_gated_scan_sizes(int batch, int len, int dim, size_t *forward_bytes, size_t *backward_bytes,
                                         size_t *saved_bytes) {
    clear_error();
    MI_REQUIRE(forward_bytes && backward_bytes && saved_bytes, MI_ERR_NULL_POINTER, "mi_gated_scan_sizes: the sizes are required");
    if (const mi_status st = gated_dims("mi_gated_scan_sizes", batch, len, dim)) return st;
    const size_t rows = (size_t)batch * gated_chunks(len, kChunkBack) * dim * sizeof(float);
    *forward_bytes = gated_word_bytes(batch, len, dim, kChunk, kWaves);
    *backward_bytes = gated_word_bytes(batch, len, dim, kChunkBack, kWavesBack) + rows;
    *saved_bytes = len ? rows : 0;
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
    a.batch = batch, a.len = len, a.dim = dim;
    const size_t need = gated_word_bytes(batch, len, dim, kChunk, kWaves);
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
    a.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + gated_word_bytes(batch, len, dim, kChunkBack, kWavesBack));
    a.rate = rate, a.batch = batch, a.len = len, a.dim = dim;
    const hipStream_t st = as_stream(stream);
    if (batch > 0) with_type(type, [&](auto t) { launch_gated<Backward, decltype(t)>(a, workspace, st); });
    if (ddecay)
        hipLaunchKernelGGL(gated_decay_kernel, dim3((unsigned)((dim + 63) / 64)), dim3(1024), 0, st, a.sums, decay, ddecay,
                           (int64_t)batch * gated_chunks(len, kChunkBack), dim);
    return check_launch("mi_gated_scan_backward");
}
