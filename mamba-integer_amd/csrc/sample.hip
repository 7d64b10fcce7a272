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
#include "float_ops.hpp"

namespace mi {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 1024;           // candidates whose ranks are counted pairwise
constexpr int kSampleMaxVocab = 1 << 24;
constexpr double kSampleRange = 40.0;       // e^-40 * 2^52 rounds to a mass of 0

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

struct SampleLds {
    uint32_t count[kSampleBins];
    uint64_t mass[kSampleBins];
    uint64_t list[kSampleList], list_mass[kSampleList];
    uint64_t wave_mass[kSampleWaves], threshold;
    uint32_t wave_count[kSampleWaves], found, lo, hi;
    uint64_t above_mass;
    uint32_t above_count;
    int bin, token;
};

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, o);
}
__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_up((int)(v >> 32), o) << 32 | (uint32_t)__shfl_up((int)(uint32_t)v, o);
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
    return v;
}

// One row's logits and what its passes share.
template <class T>
struct SampleRow {
    const T *p;
    double scale, top, inv_t, unit;
    uint32_t top_key;
    int vocab;

    // 0 for the largest logit (an infinite one too), below 0 for others, -inf or NaN far below
    __device__ __forceinline__ double below(Logit<T> v) const {
        return order_key(v) == top_key ? 0.0 : ((double)v * scale - top) * inv_t;
    }
    __device__ __forceinline__ static double e(double d) { return d > -kSampleRange ? exp(d) : 0.0; }
    __device__ __forceinline__ uint64_t mass(double e) const { return (uint64_t)__builtin_rint(e * unit); }
    __device__ __forceinline__ static int bin(double d) {
        return d > -kSampleRange ? min((int)(d * (-kSampleBins / kSampleRange)), kSampleBins - 1) : kSampleBins - 1;
    }
};

// The first of the bins, from 0 on, at which the counts reach `count` or the masses reach
// `mass`, and what lies in the bins before it.  All threads; the bins hold them by then.
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

// Calls f(logit, token, on) over a wave's share of the row, in the order of tokens, 64 at a time,
// with all lanes active (`on`: the lane has a token), until f says true (the same for all lanes).
template <class T, class F>
__device__ __forceinline__ void wave_share(const SampleRow<T> &r, int wave, F &&f) {
    const int share = ((r.vocab + kSampleWaves - 1) / kSampleWaves + 63) / 64 * 64;
    const int end = min((wave + 1) * share, r.vocab);
    for (int base = wave * share; base < end; base += 64) {
        const int i = base + (threadIdx.x & 63);
        const Logit<T> v = i < end ? (Logit<T>)r.p[i] : Logit<T>(0);
        if (f(v, i, i < end && drawable(v))) break;
    }
}

// Of the tokens in bin s.bin (by `below`) whose place in the order is at least `from`:
// keeps the first ones while fewer than `count` of them and less than `mass` lie before.
// Returns the last kept one's place.  All threads; the bins count these tokens.
template <class T>
__device__ uint64_t cut_in_bin(const SampleRow<T> &r, SampleLds &s, uint64_t from, uint32_t count, uint64_t mass) {
    const int tid = threadIdx.x, bin = s.bin;
    uint32_t n = s.count[bin];
    __syncthreads();
    if (tid == 0) {
        s.lo = 0xffffffffu;
        s.hi = 0;
        s.found = 0;
        s.threshold = ~0ull;
    }
    __syncthreads();
    {
        uint32_t lo = 0xffffffffu, hi = 0;
        for (int i = tid; i < r.vocab; i += kSampleThreads) {
            const Logit<T> v = (Logit<T>)r.p[i];
            if (!drawable(v) || order_of(order_key(v), i) < from) continue;
            const double d = r.below(v);
            if (SampleRow<T>::bin(d) != bin) continue;
            lo = min(lo, order_key(v));
            hi = max(hi, order_key(v));
        }
        if (lo <= hi) {
            atomicMin(&s.lo, lo);
            atomicMax(&s.hi, hi);
        }
    }
    __syncthreads();
    uint32_t lo = s.lo, hi = s.hi;
    // The keys in [lo, hi] are the candidates: too many are parted by key.
    while (n > kSampleList && lo != hi) {
        const uint64_t span = (uint64_t)hi - lo + 1;
        for (int i = tid; i < kSampleBins; i += kSampleThreads) {
            s.count[i] = 0;
            s.mass[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < r.vocab; i += kSampleThreads) {
            const Logit<T> v = (Logit<T>)r.p[i];
            const uint32_t key = order_key(v);
            if (!drawable(v) || key < lo || key > hi || order_of(key, i) < from) continue;
            const int at = (int)((uint64_t)(hi - key) * kSampleBins / span);
            atomicAdd(&s.count[at], 1u);
            atomicAdd((unsigned long long *)&s.mass[at], (unsigned long long)r.mass(r.e(r.below(v))));
        }
        __syncthreads();
        cut_bin(s, count, mass);
        const uint64_t at = (uint64_t)s.bin;
        // hi - key in [ceil(at * span / bins), ceil((at + 1) * span / bins))
        const uint64_t first = (at * span + kSampleBins - 1) / kSampleBins, end = ((at + 1) * span + kSampleBins - 1) / kSampleBins;
        n = s.count[s.bin];
        count -= s.above_count;
        mass -= s.above_mass;
        lo = hi - (uint32_t)(end - 1);
        hi = hi - (uint32_t)first;
        __syncthreads();
    }
    if (n <= kSampleList) {
        for (int i = tid; i < r.vocab; i += kSampleThreads) {
            const Logit<T> v = (Logit<T>)r.p[i];
            const uint32_t key = order_key(v);
            if (!drawable(v) || key < lo || key > hi || order_of(key, i) < from) continue;
            const uint32_t at = atomicAdd(&s.found, 1u);
            if (at < kSampleList) {
                s.list[at] = order_of(key, i);
                s.list_mass[at] = r.mass(r.e(r.below(v)));
            }
        }
        __syncthreads();
        if (tid < (int)n) {
            const uint64_t mine = s.list[tid];
            uint32_t c = 0;
            uint64_t m = 0;
            for (int j = 0; j < (int)n; ++j) {
                const bool earlier = s.list[j] > mine;
                c += earlier ? 1u : 0u;
                m += earlier ? s.list_mass[j] : 0ull;
            }
            if (c < count && m < mass) atomicMin((unsigned long long *)&s.threshold, (unsigned long long)mine);
        }
    } else {
        // one key: the first tokens of it, in their order
        const int wave = wave_id(), lane = tid & 63;
        uint64_t each = 0;
        uint32_t mine = 0;
        wave_share(r, wave, [&](Logit<T> v, int i, bool on) {
            mine += __popcll(__ballot(on && order_key(v) == lo && order_of(lo, i) >= from));
            return false;
        });
        if (lane == 0) s.wave_count[wave] = mine;
        wave_share(r, wave, [&](Logit<T> v, int, bool on) {     // the mass that each has
            const bool is = on && order_key(v) == lo;
            if (is) s.list_mass[0] = r.mass(r.e(r.below(v)));
            return __any(is) != 0;
        });
        __syncthreads();
        each = s.list_mass[0];
        uint64_t keep = min((uint64_t)count, (uint64_t)n);
        if (each != 0) keep = min(keep, (mass - 1) / each + 1);
        uint32_t seen = 0;
        for (int w = 0; w < wave; ++w) seen += s.wave_count[w];
        if (seen < keep && seen + mine >= keep)
            wave_share(r, wave, [&](Logit<T> v, int i, bool on) {
                const bool is = on && order_key(v) == lo && order_of(lo, i) >= from;
                const uint64_t votes = __ballot(is);
                const uint32_t rank = seen + __popcll(votes & ((1ull << lane) - 1));
                if (is && rank + 1 == keep) s.threshold = order_of(lo, i);
                seen += __popcll(votes);
                return seen >= keep;
            });
    }
    __syncthreads();
    return s.threshold;
}

template <class T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
    __shared__ SampleLds s;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int64_t row = blockIdx.x;
    SampleRow<T> r;
    r.p = static_cast<const T *>(a.logits) + row * a.ld;
    r.vocab = a.vocab;
    r.scale = a.scale;

    // the first of the order
    uint64_t best = 0;
    for (int i = tid; i < r.vocab; i += kSampleThreads) {
        const Logit<T> v = (Logit<T>)r.p[i];
        if (drawable(v)) best = max(best, order_of(order_key(v), i));
    }
    for (int o = 32; o > 0; o >>= 1) best = max(best, shfl_xor64(best, o));
    if (lane == 0) s.wave_mass[wave] = best;
    for (int i = tid; i < kSampleBins; i += kSampleThreads) {
        s.count[i] = 0;
        s.mass[i] = 0;
    }
    __syncthreads();
    for (int w = 0; w < kSampleWaves; ++w) best = max(best, s.wave_mass[w]);
    const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
    if (best == 0 || !(temperature > 0.0f)) {     // nothing to draw from, or the first
        if (tid == 0) {
            a.ids[row] = best ? (int64_t)(uint32_t)~(uint32_t)best : -1;
            if (a.logprob) a.logprob[row] = best ? 0.0f : -__builtin_inff();
        }
        return;
    }
    r.top_key = (uint32_t)(best >> 32);
    r.top = (double)(Logit<T>)r.p[(uint32_t)~(uint32_t)best] * a.scale;
    r.inv_t = 1.0 / (double)temperature;
    r.unit = (double)(1ull << a.bits);

    const int32_t k = a.top_k ? a.top_k[row] : a.top_k_all;
    const float p = a.top_p ? a.top_p[row] : a.top_p_all, least = a.min_p ? a.min_p[row] : a.min_p_all;
    const bool by_k = k > 0 && k < r.vocab, by_p = p < 1.0f;
    uint64_t threshold = 0;
    __syncthreads();
    if (by_k || by_p) {
        for (int i = tid; i < r.vocab; i += kSampleThreads) {
            const Logit<T> v = (Logit<T>)r.p[i];
            if (!drawable(v)) continue;
            const double d = r.below(v);
            const int at = SampleRow<T>::bin(d);
            atomicAdd(&s.count[at], 1u);
            if (by_p) {
                const uint64_t m = r.mass(r.e(d));
                if (m) atomicAdd((unsigned long long *)&s.mass[at], (unsigned long long)m);
            }
        }
        __syncthreads();
        if (by_k) {
            cut_bin(s, (uint32_t)k, ~0ull);
            // (the last bin has no mass: a cut in it takes nothing away)
            if (s.bin != kSampleBins - 1) threshold = cut_in_bin(r, s, 0, (uint32_t)k - s.above_count, ~0ull);
        }
        if (by_p) {
            // the bins again, of what top_k left: its cut has used them
            for (int i = tid; i < kSampleBins; i += kSampleThreads) {
                s.count[i] = 0;
                s.mass[i] = 0;
            }
            __syncthreads();
            uint64_t sum = 0;
            for (int i = tid; i < r.vocab; i += kSampleThreads) {
                const Logit<T> v = (Logit<T>)r.p[i];
                if (!drawable(v) || order_of(order_key(v), i) < threshold) continue;
                const double d = r.below(v);
                const uint64_t m = r.mass(r.e(d));
                atomicAdd(&s.count[SampleRow<T>::bin(d)], 1u);
                atomicAdd((unsigned long long *)&s.mass[SampleRow<T>::bin(d)], (unsigned long long)m);
                sum += m;
            }
            sum = wave_sum64(sum);
            if (lane == 0) s.wave_mass[wave] = sum;
            __syncthreads();
            sum = 0;
            for (int w = 0; w < kSampleWaves; ++w) sum += s.wave_mass[w];
            __syncthreads();
            uint64_t mass = p > 0.0f ? (uint64_t)ceil((double)p * (double)sum) : 1;
            mass = max(mass, (uint64_t)1);
            cut_bin(s, ~0u, mass);
            threshold = max(threshold, cut_in_bin(r, s, threshold, ~0u, mass - s.above_mass));
        }
    }

    // the kept mass of each wave's share of the row, in the order of tokens
    auto kept = [&](Logit<T> v, int i, bool on) -> uint64_t {
        if (!on) return 0;
        const uint64_t at = order_of(order_key(v), i);
        if (at < threshold) return 0;
        const double e = r.e(r.below(v));
        return e >= (double)least || at == best || !(least > 0.0f) ? r.mass(e) : 0;
    };
    uint64_t sum = 0;
    wave_share(r, wave, [&](Logit<T> v, int i, bool on) {
        sum += kept(v, i, on);
        return false;
    });
    sum = wave_sum64(sum);
    if (lane == 0) s.wave_mass[wave] = sum;
    __syncthreads();
    uint64_t total = 0, before = 0;
    for (int w = 0; w < kSampleWaves; ++w) {
        before += w < wave ? s.wave_mass[w] : 0;
        total += s.wave_mass[w];
    }
    const float u = a.u[row];
    const double at = (double)u * (double)total;
    const uint64_t target = at > 0.0 ? min((uint64_t)fmin(at, 9e18), total - 1) : 0;
    if (!(before <= target && target < before + sum)) return;
    wave_share(r, wave, [&](Logit<T> v, int i, bool on) {
        const uint64_t m = kept(v, i, on);
        uint64_t run = m;
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t up = shfl_up64(run, o);
            if (lane >= o) run += up;
        }
        const uint64_t votes = __ballot(before + run > target);
        if (votes != 0) {
            if (lane == __ffsll((unsigned long long)votes) - 1) {
                a.ids[row] = i;
                if (a.logprob) a.logprob[row] = (float)(r.below(v) - log((double)total / r.unit));
            }
            return true;
        }
        before += (uint64_t)(uint32_t)__shfl((int)(run >> 32), 63) << 32 | (uint32_t)__shfl((int)(uint32_t)run, 63);
        return false;
    });
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_sample_tokens(const void *logits, int type, int64_t ld, double scale, const float *u,
                                      const float *temperature, float temperature_all, const int32_t *top_k, int top_k_all,
                                      const float *top_p, float top_p_all, const float *min_p, float min_p_all, int64_t *ids,
                                      float *logprob, int rows, int vocab, void *stream) {
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
    int log2v = 0;
    while ((1 << log2v) < vocab) ++log2v;
    // the masses of a row sum to 2^62 at most
    const SampleArgs a{logits, ld, scale, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all,
                       ids, logprob, vocab, min(52, 62 - log2v)};
    const hipStream_t st = as_stream(stream);
    const auto launch = [&](auto t) {
        hipLaunchKernelGGL((sample_kernel<decltype(t)>), dim3((unsigned)rows), dim3(kSampleThreads), 0, st, a);
    };
    if (type == MI_I32)
        launch(int32_t{});
    else
        with_type(type, launch);
    return check_launch("mi_sample_tokens");
}
