// The next token of every row of logits, drawn with a given random number:
//
//   l = logit * scale,  e_i = exp((l_i - max l) / temperature)
//   order: larger l first, of equal ones the lower token
//   keep the first top_k of the order, of those the shortest beginning whose mass is at
//   least top_p of theirs, of those the ones with e >= min_p (the first always)
//   the token: the first one, in the vocabulary's order, at which the kept mass up to and
//   with it exceeds u * (the kept mass)
//
// A draw compares sums of many small masses, and a sum that rounds by its order would
// move the border between two tokens: e is a double, and a mass is e * 2^bits as an
// integer, so every sum is exact, in any order.  The kept tokens are a beginning of the
// order, so one 64-bit number (the key of l above the token's complement) tells them
// from the rest.
//
// Rows in slices, a launch each for the first of the order, the bins, the candidates and the
// draw.  1 x 32000 takes 24 us, 64 x 131072 in bf16 76 (first 7, bins 18, candidates 24, draw
// 29), where its bytes take 3: what bounds it is the chain of loads, barriers and sums over
// lanes in each launch, and the exponentials (11 us of the bins).  Where more than 8192 tokens
// are candidates (flat logits, a large top_k) a block goes over the whole row: 64 x 32000 within
// 0.01 of each other 102 us with top_k 50, 164 by top_p.
#include <algorithm>
#include <type_traits>

#include "float_ops.hpp"

namespace mi {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048;
constexpr int kSampleNear = 256;            // candidates whose ranks are counted pairwise
constexpr int kSampleList = 8192;           // candidates of a row that are listed
constexpr int kSampleSlices = 64;           // of a row, at most
constexpr int kSampleBlocks = 512;          // of the slices of all rows, at most
constexpr int kSampleMaxVocab = 1 << 24;
constexpr double kSampleRange = 40.0;       // e^-40 * 2^51 rounds to a mass of 0

struct SampleArgs {
    const void *logits;
    int64_t ld;
    double scale;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    float temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    int64_t *ids;
    float *logprob;
    int vocab, bits;
    int slices, slice;      // of a row, and tokens of one
    char *workspace;
    size_t row_bytes;       // of it
};

// What the kernels of a row pass on, in the workspace; behind it the masses of each slice's bins
// (top_p alone).
struct SampleShared {
    uint64_t best[kSampleSlices];            // the first of the order in a slice
    uint64_t slice_mass[kSampleSlices];      // the mass of a slice that is surely kept
    uint64_t mass[kSampleBins];
    uint32_t count[kSampleBins];
    uint32_t found, unused[63];      // (256 bytes)
    uint64_t list[kSampleList];              // places of candidates
    __device__ __forceinline__ uint64_t *slice_bins(int slice) { return reinterpret_cast<uint64_t *>(this + 1) + slice * kSampleBins; }
    static size_t bytes(int slices) { return sizeof(SampleShared) + (size_t)slices * kSampleBins * sizeof(uint64_t); }
};

// A logit's place in the order: larger for larger logits, 0 and -0 alike.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint32_t order_key(int32_t v) { return (uint32_t)v ^ 0x80000000u; }
__device__ __forceinline__ bool drawable(float v) { return v > -__builtin_inff(); }   // (a NaN is not)
__device__ __forceinline__ bool drawable(int32_t) { return true; }
template <class T>
using Logit = std::conditional_t<std::is_same<T, int32_t>::value, int32_t, float>;

// The key above the token's complement: larger is earlier in the order; never 0.
__device__ __forceinline__ uint64_t order_of(uint32_t key, int token) { return (uint64_t)key << 32 | (uint32_t)~token; }
__device__ __forceinline__ int token_of(uint64_t place) { return (int)~(uint32_t)place; }
// The logit of a key.
template <class L>
__device__ __forceinline__ L value_of(uint32_t key) {
    if constexpr (std::is_same<L, int32_t>::value)
        return (int32_t)(key ^ 0x80000000u);
    else
        return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// 2^(j / 64).
__constant__ const double kExpTable[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

struct alignas(16) Candidate {
    uint64_t place, mass;
};

struct SampleLds {
    double table[64];
    uint32_t count[kSampleBins];
    uint64_t mass[kSampleBins];
    Candidate near[kSampleNear];
    uint64_t wave_mass[kSampleWaves], lo, hi, above_mass, last;
    uint32_t wave_count[kSampleWaves], above_count, found;
    int bin;
};

// (of two 64-bit types that differ in name, min and max are those of 32 bits)
__device__ __forceinline__ uint64_t less(uint64_t a, uint64_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t more(uint64_t a, uint64_t b) { return a < b ? b : a; }
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, o);
}
__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_up((int)(v >> 32), o) << 32 | (uint32_t)__shfl_up((int)(uint32_t)v, o);
}
__device__ __forceinline__ uint64_t block_sum(SampleLds &s, uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
    if ((threadIdx.x & 63) == 0) s.wave_mass[wave_id()] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < kSampleWaves; ++w) v += s.wave_mass[w];
    __syncthreads();
    return v;
}

// One row's logits and what its passes share.
template <class T>
struct SampleRow {
    const T *p;
    const double *table;
    double top, factor, unit;      // the largest logit; scale / temperature; 2^bits
    int begin, end;                // the tokens that the passes go over

    // l - max l over the temperature: 0 for the largest (an infinite one too), -inf or NaN far below
    __device__ __forceinline__ double below(Logit<T> v) const { return (double)v == top ? 0.0 : ((double)v - top) * factor; }
    // exp(d) of d in (-40, 0] to 2 of its last places, 0 below: 2^(n / 64) exp(r) with |r| < ln 2 / 128
    __device__ __forceinline__ double e(double d) const {
        const double n = __builtin_rint(d * 0x1.71547652b82fep+6);
        const double r = __builtin_fma(n, -0x1.9ef35793c7673p-47, __builtin_fma(n, -0x1.62e42fefa2000p-7, d));
        double q = __builtin_fma(r, 1.0 / 120.0, 1.0 / 24.0);
        q = __builtin_fma(r, q, 1.0 / 6.0);
        q = __builtin_fma(r, q, 0.5);
        q = __builtin_fma(r * r, q, r);
        const int k = d > -kSampleRange ? (int)n : 0;
        const double t = table[k & 63];
        return d > -kSampleRange ? __builtin_ldexp(__builtin_fma(t, q, t), k >> 6) : 0.0;
    }
    // e * 2^bits as an integer (bits <= 51): the mantissa of its sum with 2^52
    __device__ __forceinline__ uint64_t mass(double e) const {
        return __builtin_bit_cast(uint64_t, __builtin_fma(e, unit, 0x1p52)) - __builtin_bit_cast(uint64_t, 0x1p52);
    }
    __device__ __forceinline__ static int bin(double d) {
        return d > -kSampleRange ? min((int)(d * (-kSampleBins / kSampleRange)), kSampleBins - 1) : kSampleBins - 1;
    }
};

// 16 bytes of a row from token i on, zeros from `end` on.
template <class T, int N = 16 / sizeof(T)>
__device__ __forceinline__ Packed<T, N> load_logits(const T *p, int i, int end) {
    if (i + N <= end) return load_packed<N>(p + i);
    Packed<T, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = i + e < end ? p[i + e] : T(0);
    return v;
}

// Calls f(logit, token) for every token that may be drawn, by all threads, in no order.
template <class T, class F>
__device__ __forceinline__ void each_logit(const SampleRow<T> &r, F &&f) {
    constexpr int N = 16 / sizeof(T), STEP = kSampleThreads * N;
    int i = r.begin + (int)threadIdx.x * N;
    Packed<T, N> next;
    if (i < r.end) next = load_logits(r.p, i, r.end);
    for (; i < r.end; i += STEP) {
        const Packed<T, N> now = next;
        if (i + STEP < r.end) next = load_logits(r.p, i + STEP, r.end);
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (i + e < r.end && drawable((Logit<T>)now.v[e])) f((Logit<T>)now.v[e], i + e);
    }
}

// Calls f(logits, first token, how many of them) over a wave's share of the row, in the order of
// tokens, N adjacent ones a lane, with all lanes active, until f says true (the same for all).
template <class T, class F>
__device__ __forceinline__ void wave_share(const SampleRow<T> &r, int wave, F &&f) {
    constexpr int N = 16 / sizeof(T), STEP = 64 * N;
    const int share = (r.end - r.begin + kSampleWaves * STEP - 1) / (kSampleWaves * STEP) * STEP;
    const int end = min(r.begin + (wave + 1) * share, r.end), lane = (int)threadIdx.x & 63;
    Packed<T, N> next;
    int base = r.begin + wave * share;
    if (base < end) next = load_logits(r.p, base + lane * N, end);
    for (; base < end; base += STEP) {
        const Packed<T, N> now = next;
        if (base + STEP < end) next = load_logits(r.p, base + STEP + lane * N, end);
        const int i = base + lane * N;
        if (f(now, i, min(max(end - i, 0), N))) break;
    }
}

__device__ __forceinline__ void clear_bins(SampleLds &s) {
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) {
        s.count[i] = 0;
        s.mass[i] = 0;
    }
}

// The first of the bins, from 0 on, at which the counts reach `count` or the masses reach
// `mass`, and what lies in the bins before it; the last bin if none.  All threads.
__device__ __forceinline__ void cut_bin(SampleLds &s, uint32_t count, uint64_t mass) {
    constexpr int PER = kSampleBins / kSampleThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    uint32_t c[PER], cs = 0;
    uint64_t m[PER], ms = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        c[i] = s.count[tid * PER + i];
        m[i] = s.mass[tid * PER + i];
        cs += c[i];
        ms += m[i];
    }
    uint32_t ci = cs;
    uint64_t mi_ = ms;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cu = (uint32_t)__shfl_up((int)ci, o);
        const uint64_t mu = shfl_up64(mi_, o);
        if (lane >= o) {
            ci += cu;
            mi_ += mu;
        }
    }
    if (lane == 63) {
        s.wave_count[wave] = ci;
        s.wave_mass[wave] = mi_;
    }
    if (tid == 0) s.bin = kSampleBins - 1;
    __syncthreads();
    uint32_t cb = ci - cs;
    uint64_t mb = mi_ - ms;
    for (int w = 0; w < wave; ++w) {
        cb += s.wave_count[w];
        mb += s.wave_mass[w];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        // one bin of one thread: not reached before it, reached with it
        if (cb < count && mb < mass && (cb + c[i] >= count || mb + m[i] >= mass)) {
            s.bin = tid * PER + i;
            s.above_count = cb;
            s.above_mass = mb;
        }
        cb += c[i];
        mb += m[i];
    }
    __syncthreads();
}

// How many of the n candidates in LDS have a larger place than `mine`, and their mass.
__device__ __forceinline__ void in_front(const SampleLds &s, int n, uint64_t mine, uint32_t &c, uint64_t &m) {
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
        const Candidate o = s.near[j];
        const bool earlier = o.place > mine;
        c += earlier ? 1u : 0u;
        m += earlier ? o.mass : 0ull;
    }
}

// Of n candidates in the order of their places, larger first: the place of the last one that
// has fewer than `count` and less than `mass` in front of it (there is one: neither is 0).
// visit(f) calls f(place, d) for each candidate, by all threads, in any order; no two places
// are alike.  Too many candidates are parted by place until few enough share a part.  All
// threads.
template <class T, class V>
__device__ __forceinline__ uint64_t cut_among(const SampleRow<T> &r, SampleLds &s, uint32_t n, uint32_t count, uint64_t mass, V &&visit) {
    const int tid = threadIdx.x;
    const bool by_mass = mass != ~0ull;
    uint64_t lo = 0, hi = ~0ull;
    __syncthreads();
    if (tid == 0) {
        s.lo = ~0ull;
        s.hi = 0;
        s.found = 0;
        s.last = ~0ull;
    }
    if (n > kSampleNear) {
        __syncthreads();
        uint64_t least = ~0ull, most = 0;
        visit([&](uint64_t place, double) {
            least = less(least, place);
            most = more(most, place);
        });
        for (int o = 32; o > 0; o >>= 1) {
            least = less(least, shfl_xor64(least, o));
            most = more(most, shfl_xor64(most, o));
        }
        if ((tid & 63) == 0) {
            atomicMin((unsigned long long *)&s.lo, (unsigned long long)least);
            atomicMax((unsigned long long *)&s.hi, (unsigned long long)most);
        }
        __syncthreads();
        lo = s.lo;
        hi = s.hi;
        while (n > kSampleNear) {
            const int shift = max(0, 64 - __builtin_clzll((hi - lo) | 1) - 11);      // (hi - lo) >> shift is a bin
            clear_bins(s);
            __syncthreads();
            visit([&](uint64_t place, double d) {
                if (place < lo || place > hi) return;
                const int at = (int)((hi - place) >> shift);
                atomicAdd(&s.count[at], 1u);
                if (by_mass) atomicAdd((unsigned long long *)&s.mass[at], (unsigned long long)r.mass(r.e(d)));
            });
            __syncthreads();
            cut_bin(s, count, mass);
            n = s.count[s.bin];
            count -= s.above_count;
            if (by_mass) mass -= s.above_mass;
            hi -= (uint64_t)s.bin << shift;
            // (the last part is cut off at lo, which may be nearer to 0 than a part is wide)
            const uint64_t width = ((uint64_t)1 << shift) - 1;
            if (hi - lo > width) lo = hi - width;
            __syncthreads();
        }
    }
    __syncthreads();
    visit([&](uint64_t place, double d) {
        if (place < lo || place > hi) return;
        const uint32_t at = atomicAdd(&s.found, 1u);
        if (at < kSampleNear) {
            s.near[at] = {place, by_mass ? r.mass(r.e(d)) : 0};
        }
    });
    __syncthreads();
    if (tid < (int)n) {
        const uint64_t mine = s.near[tid].place;
        uint32_t c = 0;
        uint64_t m = 0;
        in_front(s, (int)n, mine, c, m);
        if (c < count && m < mass) atomicMin((unsigned long long *)&s.last, (unsigned long long)mine);
    }
    __syncthreads();
    return s.last;
}

// The first of the order among the row's tokens in [begin, end), by all threads.
template <class T>
__device__ __forceinline__ uint64_t first_of(const SampleRow<T> &r, SampleLds &s) {
    Logit<T> most{};
    int first = -1;
    each_logit(r, [&](Logit<T> v, int i) {
        if (first < 0 || v > most) {
            most = v;
            first = i;
        }
    });
    uint64_t best = first < 0 ? 0 : order_of(order_key(most), first);
    for (int o = 32; o > 0; o >>= 1) best = more(best, shfl_xor64(best, o));
    if ((threadIdx.x & 63) == 0) s.wave_mass[wave_id()] = best;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; ++w) best = more(best, s.wave_mass[w]);
    return best;
}

// A row's parameters.
struct SampleFilters {
    float temperature, p, least;
    int32_t k;
    bool by_k, by_p;
    __device__ __forceinline__ SampleFilters(const SampleArgs &a, int64_t row) {
        temperature = a.temperature ? a.temperature[row] : a.temperature_all;
        k = a.top_k ? a.top_k[row] : a.top_k_all;
        p = a.top_p ? a.top_p[row] : a.top_p_all;
        least = a.min_p ? a.min_p[row] : a.min_p_all;
        by_k = k > 0 && k < a.vocab;
        by_p = p < 1.0f;
    }
    // the least mass that top_p keeps of `sum`
    __device__ __forceinline__ uint64_t mass_of(uint64_t sum) const {
        return more(p > 0.0f ? (uint64_t)ceil((double)p * (double)sum) : 1, 1);
    }
};
template <class T>
__device__ __forceinline__ SampleRow<T> sample_row(const SampleArgs &a, const SampleLds &s, int64_t row, int begin, int end) {
    SampleRow<T> r;
    r.p = static_cast<const T *>(a.logits) + row * a.ld;
    r.table = s.table;
    r.begin = begin;
    r.end = end;
    return r;
}
template <class T>
__device__ __forceinline__ void scale_by(SampleRow<T> &r, const SampleArgs &a, uint64_t best, float temperature) {
    r.top = (double)(Logit<T>)r.p[token_of(best)];
    r.factor = a.scale / (double)temperature;
    r.unit = (double)(1ull << a.bits);
}

// ------------------------------------------------------------------ slices
// Few rows of many tokens: a row's passes are shared by `slices` blocks, in a kernel each
// (the first of the order; the bins; what the bins leave), and the last kernel draws.
__device__ __forceinline__ SampleShared &shared_of(const SampleArgs &a, int64_t row) {
    return *reinterpret_cast<SampleShared *>(a.workspace + row * a.row_bytes);
}
// (a slice's a lane: one after the other they took a load's latency each)
__device__ __forceinline__ uint64_t best_of(const SampleArgs &a, const SampleShared &g) {
    const int lane = threadIdx.x & 63;
    uint64_t best = lane < a.slices ? g.best[lane] : 0;
    for (int o = 32; o > 0; o >>= 1) best = more(best, shfl_xor64(best, o));
    return best;
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_first_kernel(SampleArgs a) {
    __shared__ SampleLds s;
    const int64_t row = blockIdx.y;
    const int slice = blockIdx.x;
    SampleShared &g = shared_of(a, row);
    for (int i = slice * kSampleThreads + (int)threadIdx.x; i < kSampleBins; i += a.slices * kSampleThreads) {
        g.count[i] = 0;
        g.mass[i] = 0;
    }
    const SampleRow<T> r = sample_row<T>(a, s, row, slice * a.slice, min((slice + 1) * a.slice, a.vocab));
    const uint64_t best = first_of(r, s);
    if (threadIdx.x == 0) {
        g.best[slice] = best;
        if (slice == 0) g.found = 0;
    }
}

// Counts, for top_k, or masses, for top_p alone, added to the row's bins.
template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_bins_kernel(SampleArgs a) {
    __shared__ SampleLds s;
    const int64_t row = blockIdx.y;
    const int slice = blockIdx.x, tid = threadIdx.x;
    SampleShared &g = shared_of(a, row);
    const SampleFilters f(a, row);
    const uint64_t best = best_of(a, g);
    if (best == 0 || !(f.temperature > 0.0f) || !(f.by_k || f.by_p)) return;
    SampleRow<T> r = sample_row<T>(a, s, row, slice * a.slice, min((slice + 1) * a.slice, a.vocab));
    scale_by(r, a, best, f.temperature);
    if (tid < 64) s.table[tid] = kExpTable[tid];
    clear_bins(s);
    __syncthreads();
    if (f.by_k)
        each_logit(r, [&](Logit<T> v, int) {
            const int at = SampleRow<T>::bin(r.below(v));
            if (at != kSampleBins - 1) atomicAdd(&s.count[at], 1u);
        });
    else
        each_logit(r, [&](Logit<T> v, int) {
            const double d = r.below(v);
            const int at = SampleRow<T>::bin(d);
            const uint64_t m = r.mass(r.e(d));
            if (m == 0) return;
            atomicAdd(&s.count[at], 1u);
            atomicAdd((unsigned long long *)&s.mass[at], (unsigned long long)m);
        });
    __syncthreads();
    for (int i = tid; i < kSampleBins; i += kSampleThreads) {
        if (s.count[i]) atomicAdd(&g.count[i], s.count[i]);
        if (f.by_k) continue;
        if (s.mass[i]) atomicAdd((unsigned long long *)&g.mass[i], (unsigned long long)s.mass[i]);
        g.slice_bins(slice)[i] = s.mass[i];
    }
}

// What the bins say: the bin in which the first filter cuts, how many tokens are candidates
// (top_k: all that it may keep; top_p alone: those of the bin), or that the row has to be gone
// over as a whole.  LDS has the row's bins then.  All threads.
struct SampleCut {
    bool whole;
    int bin;
    uint32_t listed;
    uint64_t mass;      // top_p alone: what is kept of the bin's mass, at least
};
__device__ __forceinline__ SampleCut cut_row(const SampleShared &g, SampleLds &s, const SampleFilters &f) {
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) {
        s.count[i] = g.count[i];
        s.mass[i] = g.mass[i];
    }
    __syncthreads();
    SampleCut c{};
    if (f.by_k) {
        cut_bin(s, (uint32_t)f.k, ~0ull);
        c.bin = s.bin;
        c.listed = c.bin == kSampleBins - 1 ? 0 : s.above_count + s.count[c.bin];
        c.whole = c.bin == kSampleBins - 1 || c.listed > kSampleList;
    } else {
        uint64_t sum = 0;
        for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) sum += s.mass[i];
        const uint64_t mass = f.mass_of(block_sum(s, sum));
        cut_bin(s, ~0u, mass);
        c.bin = s.bin;
        c.listed = s.count[c.bin];
        c.whole = c.listed > kSampleList;
        c.mass = mass - s.above_mass;
    }
    return c;
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_gather_kernel(SampleArgs a) {
    __shared__ SampleLds s;
    __shared__ uint64_t own[kSampleList];      // the slice's candidates (a global counter for each: 64 rows of 131072 in 52 us instead of 24)
    const int64_t row = blockIdx.y;
    const int slice = blockIdx.x, tid = threadIdx.x;
    SampleShared &g = shared_of(a, row);
    const SampleFilters f(a, row);
    const uint64_t best = best_of(a, g);
    if (best == 0 || !(f.temperature > 0.0f)) return;
    SampleCut c{};
    c.bin = kSampleBins;      // (without top_k and top_p every token is surely kept)
    if (f.by_k || f.by_p) c = cut_row(g, s, f);
    if (c.whole) return;
    SampleRow<T> r = sample_row<T>(a, s, row, slice * a.slice, min((slice + 1) * a.slice, a.vocab));
    scale_by(r, a, best, f.temperature);
    if (tid < 64) s.table[tid] = kExpTable[tid];
    if (tid == 0) s.found = 0;
    __syncthreads();
    uint64_t sum = 0;
    const auto list = [&](Logit<T> v, int i) {
        const uint32_t at = atomicAdd(&s.found, 1u);
        if (at < kSampleList) own[at] = order_of(order_key(v), i);
    };
    if (f.by_k)
        each_logit(r, [&](Logit<T> v, int i) {
            if (SampleRow<T>::bin(r.below(v)) <= c.bin) list(v, i);
        });
    else if (f.by_p && !(f.least > 0.0f)) {
        // (the bins in front of the cut are kept as they are)
        for (int i = tid; i < c.bin; i += kSampleThreads) sum += g.slice_bins(slice)[i];
        each_logit(r, [&](Logit<T> v, int i) {
            const double d = r.below(v);
            if (SampleRow<T>::bin(d) == c.bin) list(v, i);
        });
    } else
        each_logit(r, [&](Logit<T> v, int i) {
            const double d = r.below(v);
            const int at = SampleRow<T>::bin(d);
            if (at > c.bin) return;
            const double e = r.e(d);
            if (at == c.bin) {
                list(v, i);
            } else if (e >= (double)f.least || !(f.least > 0.0f) || order_of(order_key(v), i) == best) {
                sum += r.mass(e);
            }
        });
    sum = block_sum(s, sum);
    const uint32_t n = s.found;
    if (tid == 0) {
        g.slice_mass[slice] = sum;
        s.above_count = n ? atomicAdd(&g.found, n) : 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kSampleThreads)
        if (i < kSampleList && s.above_count + i < kSampleList) g.list[s.above_count + i] = own[i];
}

// The draw from the few candidates of a top_k, a thread each: its place among them and the
// mass in front of it by looking at them all, in the order and then by token.
template <class T>
__device__ __forceinline__ void draw_listed(const SampleArgs &a, const SampleRow<T> &r, SampleLds &s, const SampleFilters &f, int64_t row,
                                            const uint64_t *list, int n) {
    const int tid = threadIdx.x;
    uint64_t place = 0, mass = 0;
    double d = 0.0, e = 0.0;
    if (tid < n) {
        place = list[tid];
        d = r.below(value_of<Logit<T>>((uint32_t)(place >> 32)));
        e = r.e(d);
        mass = r.mass(e);
        s.near[tid] = {place, mass};
    }
    __syncthreads();
    uint32_t c = 0;
    uint64_t m = 0;
    if (tid < n) in_front(s, n, place, c, m);
    const bool in_k = tid < n && c < (uint32_t)f.k;
    const uint64_t sum = block_sum(s, in_k ? mass : 0);
    const bool keep = in_k && (!f.by_p || m < f.mass_of(sum)) && (e >= (double)f.least || c == 0 || !(f.least > 0.0f));
    if (!keep) mass = 0;
    if (tid < n) s.near[tid] = {(uint64_t)(uint32_t)place, mass};      // (the complement of the token)
    const uint64_t total = block_sum(s, mass);
    const double at = (double)a.u[row] * (double)total;
    const uint64_t target = at > 0.0 ? less((uint64_t)fmin(at, 9e18), total - 1) : (uint64_t)0;
    m = 0;
    if (tid < n) in_front(s, n, (uint64_t)(uint32_t)place, c, m);
    if (m <= target && target < m + mass) {
        a.ids[row] = token_of(place);
        if (a.logprob) a.logprob[row] = (float)(d - log((double)total / r.unit));
    }
}

// A block a row: all of it, or after the kernels above.
template <class T, bool SLICES>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
    __shared__ SampleLds s;
    constexpr int N = 16 / sizeof(T);
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int64_t row = blockIdx.x;
    SampleRow<T> r = sample_row<T>(a, s, row, 0, a.vocab);
    SampleShared &g = shared_of(a, row);
    const SampleFilters f(a, row);
    const uint64_t best = SLICES ? best_of(a, g) : first_of(r, s);
    if (tid < 64) s.table[tid] = kExpTable[tid];
    clear_bins(s);
    if (best == 0 || !(f.temperature > 0.0f)) {     // nothing to draw from, or the first
        if (tid == 0) {
            a.ids[row] = best ? (int64_t)token_of(best) : -1;
            if (a.logprob) a.logprob[row] = best ? 0.0f : -__builtin_inff();
        }
        return;
    }
    scale_by(r, a, best, f.temperature);
    uint64_t threshold = 0;
    const uint64_t *listed = nullptr;      // tokens that may be left, if they are few
    uint32_t n_listed = 0;
    const auto in_list = [&](auto &&fn) {
        for (uint32_t i = tid; i < n_listed; i += kSampleThreads) fn(listed[i], r.below(value_of<Logit<T>>((uint32_t)(listed[i] >> 32))));
    };
    const auto in_row = [&](auto &&fn) { each_logit(r, [&](Logit<T> v, int i) { fn(order_of(order_key(v), i), r.below(v)); }); };
    const auto left = [&](auto &&fn) {      // the tokens that the filters so far have left
        const auto one = [&](uint64_t place, double d) {
            if (place >= threshold) fn(place, d);
        };
        if (SLICES && listed)
            in_list(one);
        else
            in_row(one);
    };
    const auto of_bin = [&](int bin) {
        return [&, bin](auto &&fn) {
            left([&](uint64_t place, double d) {
                if (SampleRow<T>::bin(d) == bin && r.mass(r.e(d)) != 0) fn(place, d);
            });
        };
    };
    const auto cut_mass = [&] {      // top_p of what is left
        __syncthreads();
        clear_bins(s);
        __syncthreads();
        uint64_t sum = 0;
        left([&](uint64_t, double d) {
            const int at = SampleRow<T>::bin(d);
            const uint64_t m = r.mass(r.e(d));
            if (m == 0) return;
            atomicAdd(&s.count[at], 1u);
            atomicAdd((unsigned long long *)&s.mass[at], (unsigned long long)m);
            sum += m;
        });
        const uint64_t mass = f.mass_of(block_sum(s, sum));
        cut_bin(s, ~0u, mass);
        const int bin = s.bin;
        const uint32_t n = s.count[bin];
        const uint64_t before = s.above_mass;
        threshold = more(threshold, cut_among(r, s, n, ~0u, mass - before, of_bin(bin)));
    };
    __syncthreads();
    bool by_slices = SLICES;       // the row's mass is known by slices, but for the listed tokens
    if (SLICES && (f.by_k || f.by_p)) {
        const SampleCut c = cut_row(g, s, f);
        // (top_p's bin is listed with the tokens in it that have no mass, which the bins do not count)
        const uint32_t found = f.by_k ? c.listed : g.found;
        const bool whole = c.whole || found > kSampleList;
        by_slices = !whole && !f.by_k;
        if (!whole) {
            listed = g.list;
            n_listed = found;
            if (f.by_k && n_listed <= kSampleNear) {
                draw_listed(a, r, s, f, row, g.list, (int)n_listed);
                return;
            }
            if (f.by_k) {
                const uint32_t n = s.count[c.bin];
                threshold = cut_among(r, s, n, (uint32_t)f.k - (c.listed - n), ~0ull, [&](auto &&fn) {
                    in_list([&](uint64_t place, double d) {
                        if (SampleRow<T>::bin(d) == c.bin) fn(place, d);
                    });
                });
                if (f.by_p) cut_mass();
            } else {
                threshold = cut_among(r, s, c.listed, ~0u, c.mass, [&](auto &&fn) {
                    in_list([&](uint64_t place, double d) {
                        if (r.mass(r.e(d)) != 0) fn(place, d);
                    });
                });
            }
        }
    }
    if (!listed && !by_slices) {
        if (f.by_k) {
            __syncthreads();
            clear_bins(s);
            __syncthreads();
            each_logit(r, [&](Logit<T> v, int) {
                const int at = SampleRow<T>::bin(r.below(v));
                if (at != kSampleBins - 1) atomicAdd(&s.count[at], 1u);
            });
            __syncthreads();
            cut_bin(s, (uint32_t)f.k, ~0ull);
            const int bin = s.bin;
            // (the last bin has no mass: a cut in it takes nothing away)
            if (bin != kSampleBins - 1) {
                const uint32_t above = s.above_count, n = s.count[bin];
                threshold = cut_among(r, s, n, (uint32_t)f.k - above, ~0ull, [&](auto &&fn) {
                    in_row([&](uint64_t place, double d) {
                        if (SampleRow<T>::bin(d) == bin) fn(place, d);
                    });
                });
            }
        }
        if (f.by_p) cut_mass();
    }

    // a token's mass, 0 for one that is not kept
    const auto kept = [&](uint64_t place, double d) -> uint64_t {
        if (place < threshold) return 0;
        const double e = r.e(d);
        return e >= (double)f.least || place == best || !(f.least > 0.0f) ? r.mass(e) : 0;
    };
    const auto target_of = [&](uint64_t total) {
        const double at = (double)a.u[row] * (double)total;
        return at > 0.0 ? less((uint64_t)fmin(at, 9e18), total - 1) : (uint64_t)0;
    };
    const auto write = [&](int token, uint64_t total) {
        a.ids[row] = token;
        if (a.logprob) a.logprob[row] = (float)(r.below((Logit<T>)r.p[token]) - log((double)total / r.unit));
    };
    uint64_t total = 0, before = 0, target = 0;
    if (SLICES && listed && f.by_k) {
        // of the kept ones by token, the last one with no more than the target in front of it
        uint64_t sum = 0, n = 0;
        in_list([&](uint64_t place, double d) {
            const uint64_t m = kept(place, d);
            sum += m;
            n += m != 0 ? 1 : 0;
        });
        sum = block_sum(s, sum);
        n = block_sum(s, n);
        const uint64_t at = cut_among(r, s, (uint32_t)n, ~0u, target_of(sum) + 1, [&](auto &&fn) {
            in_list([&](uint64_t place, double d) {
                if (kept(place, d) != 0) fn((uint64_t)(uint32_t)place, d);
            });
        });
        if (tid == 0) write(token_of(at), sum);
        return;
    }
    if (SLICES && by_slices) {
        // the slices' kept masses, and the slice that the target lies in
        __syncthreads();
        for (int i = tid; i < a.slices; i += kSampleThreads) s.mass[i] = g.slice_mass[i];
        __syncthreads();
        in_list([&](uint64_t place, double d) {
            const uint64_t m = kept(place, d);
            if (m) atomicAdd((unsigned long long *)&s.mass[token_of(place) / a.slice], (unsigned long long)m);
        });
        __syncthreads();
        for (int i = 0; i < a.slices; ++i) total += s.mass[i];
        target = target_of(total);
        int slice = 0;
        for (; slice + 1 < a.slices && before + s.mass[slice] <= target; ++slice) before += s.mass[slice];
        r.begin = slice * a.slice;
        r.end = min(r.begin + a.slice, a.vocab);
    }
    // the kept mass of each wave's share of the row, or slice, in the order of tokens
    const auto masses = [&](const Packed<T, N> &v, int i, int n, uint64_t *m) {
        uint64_t sum = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const Logit<T> l = (Logit<T>)v.v[e];
            m[e] = e < n && drawable(l) ? kept(order_of(order_key(l), i + e), r.below(l)) : 0;
            sum += m[e];
        }
        return sum;
    };
    uint64_t sum = 0;
    wave_share(r, wave, [&](const Packed<T, N> &v, int i, int n) {
        uint64_t m[N];
        sum += masses(v, i, n, m);
        return false;
    });
    for (int o = 32; o > 0; o >>= 1) sum += shfl_xor64(sum, o);
    __syncthreads();
    if (lane == 0) s.wave_mass[wave] = sum;
    __syncthreads();
    for (int w = 0; w < wave; ++w) before += s.wave_mass[w];
    if (!(SLICES && by_slices)) {
        for (int w = 0; w < kSampleWaves; ++w) total += s.wave_mass[w];
        target = target_of(total);
    }
    if (!(before <= target && target < before + sum)) return;
    wave_share(r, wave, [&](const Packed<T, N> &v, int i, int n) {
        uint64_t m[N], run = masses(v, i, n, m);
        const uint64_t mine = run;
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t up = shfl_up64(run, o);
            if (lane >= o) run += up;
        }
        const uint64_t votes = __ballot(before + run > target);
        if (votes != 0) {
            if (lane == __ffsll((unsigned long long)votes) - 1) {
                uint64_t at = before + run - mine;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    if (at <= target && target < at + m[e]) write(i + e, total);
                    at += m[e];
                }
            }
            return true;
        }
        before += (uint64_t)(uint32_t)__shfl((int)(run >> 32), 63) << 32 | (uint32_t)__shfl((int)(uint32_t)run, 63);
        return false;
    });
}

// Slices of a row: of 8192 tokens or so (each block has the row's bins to read first: 64 rows
// of 32000 in slices of 4000 49 us, of 8000 42), 512 blocks at most.  So from 257 rows on a block
// has a whole row: of 32000 with top_k 50 and top_p 0.9 79 us instead of the 44 of 256 rows, by
// top_p alone 101 and 74; of 131072 269 and 91, 438 and 161.
inline int sample_slices(int rows, int vocab) {
    const int n = std::min((vocab + 8191) / 8192, kSampleSlices);
    return std::max(1, std::min(n, kSampleBlocks / std::max(rows, 1)));
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_sample_workspace_size(int rows, int vocab, size_t *bytes) {
    clear_error();
    MI_REQUIRE(bytes, MI_ERR_NULL_POINTER, "mi_sample_workspace_size: bytes is required");
    MI_REQUIRE(rows >= 0 && rows < (1 << 22), MI_ERR_BAD_DIM, "mi_sample_workspace_size: rows=%d must be in [0, %d)", rows, 1 << 22);
    MI_REQUIRE(vocab >= 1 && vocab <= kSampleMaxVocab, MI_ERR_BAD_DIM, "mi_sample_workspace_size: vocab=%d must be in [1, %d]", vocab,
               kSampleMaxVocab);
    const int slices = sample_slices(rows, vocab);
    *bytes = slices > 1 ? rows * SampleShared::bytes(slices) : 0;
    return MI_OK;
}

extern "C" mi_status mi_sample_tokens(const void *logits, int type, int64_t ld, double scale, const float *u,
                                      const float *temperature, float temperature_all, const int32_t *top_k, int top_k_all,
                                      const float *top_p, float top_p_all, const float *min_p, float min_p_all, int64_t *ids,
                                      float *logprob, int rows, int vocab, void *workspace, size_t workspace_bytes,
                                      void *stream) {
    clear_error();
    MI_REQUIRE(rows >= 0, MI_ERR_BAD_DIM, "mi_sample_tokens: negative rows");
    MI_REQUIRE(rows < (1 << 22), MI_ERR_BAD_DIM, "mi_sample_tokens: rows=%d must be below %d", rows, 1 << 22);
    MI_REQUIRE(vocab >= 1 && vocab <= kSampleMaxVocab, MI_ERR_BAD_DIM, "mi_sample_tokens: vocab=%d must be in [1, %d]", vocab,
               kSampleMaxVocab);
    MI_REQUIRE(known_type(type) || type == MI_I32, MI_ERR_BAD_ARG, "mi_sample_tokens: unknown element type");
    MI_REQUIRE(ld >= 0, MI_ERR_BAD_DIM, "mi_sample_tokens: the row stride is negative");
    MI_REQUIRE(scale > 0.0 && scale <= 1e30, MI_ERR_BAD_ARG, "mi_sample_tokens: scale must be in (0, 1e30]");
    MI_REQUIRE(temperature || temperature_all == temperature_all, MI_ERR_BAD_ARG, "mi_sample_tokens: temperature is not a number");
    MI_REQUIRE((top_p || top_p_all == top_p_all) && (min_p || min_p_all == min_p_all), MI_ERR_BAD_ARG,
               "mi_sample_tokens: top_p or min_p is not a number");
    if (rows == 0) return MI_OK;
    MI_REQUIRE(logits && u && ids, MI_ERR_NULL_POINTER, "mi_sample_tokens: logits, u and ids are required");
    const int slices = sample_slices(rows, vocab);
    const size_t need = slices > 1 ? rows * SampleShared::bytes(slices) : 0;
    MI_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG,
               "mi_sample_tokens: the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
    MI_REQUIRE(need == 0 || aligned(workspace, 16), MI_ERR_BAD_ALIGNMENT, "mi_sample_tokens: the workspace must be 16-byte aligned");
    int log2v = 0;
    while ((1 << log2v) < vocab) ++log2v;
    // the masses of a row sum to 2^62 at most; a slice has whole vectors of 16 bytes
    SampleArgs a{logits, ld, scale, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all,
                 ids, logprob, vocab, std::min(51, 62 - log2v), slices, ((vocab + slices - 1) / slices + 7) / 8 * 8,
                 static_cast<char *>(workspace), SampleShared::bytes(slices)};
    a.slices = (vocab + a.slice - 1) / a.slice;      // (none without tokens)
    const hipStream_t st = as_stream(stream);
    const auto launch = [&](auto t) {
        using T = decltype(t);
        const dim3 each((unsigned)a.slices, (unsigned)rows), block(kSampleThreads);
        if (need == 0) {
            hipLaunchKernelGGL((sample_kernel<T, false>), dim3((unsigned)rows), block, 0, st, a);
            return;
        }
        hipLaunchKernelGGL((sample_first_kernel<T>), each, block, 0, st, a);
        // (without the filters there is nothing to bin)
        if (top_k || top_p || (top_k_all > 0 && top_k_all < vocab) || top_p_all < 1.0f)
            hipLaunchKernelGGL((sample_bins_kernel<T>), each, block, 0, st, a);
        hipLaunchKernelGGL((sample_gather_kernel<T>), each, block, 0, st, a);
        hipLaunchKernelGGL((sample_kernel<T, true>), dim3((unsigned)rows), block, 0, st, a);
    };
    if (type == MI_I32)
        launch(int32_t{});
    else
        with_type(type, launch);
    return check_launch("mi_sample_tokens");
}
