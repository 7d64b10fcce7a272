// Low-rank adapters beside a shared projection, each sequence with its own of a bank:
//
//   out[b,t,:] = y[b,t,:] + scale[id] * x_scale[b,t] * (x[b,t,:] A[id]^T) B[id]^T,  id = ids[b]
//
// in two kernels: t = x A^T (with the scales) into the workspace, then out = y + t B^T, the
// sum rounded once to out's type.  Sequences of up to 7 tokens (decode steps) go row by row
// on the vector units, where the adapters' bytes are the work; longer ones in tiles of 16
// tokens on the matrix units, where x and y are.  16384 x 4096 -> 2048 of rank 32 in bf16: 40.1
// and 37.5 us, 3.3 and 3.6 TB/s, bound by HBM (31.4 and 33.2 where the same rows come again and
// the last-level cache has some of them); 64 x 1 x 2048 -> 8192 of rank 16: 4.2 and 4.8 us, the
// second's B at 3.5 TB/s, and a call 10 us with its host side.
#include <algorithm>
#include <type_traits>

#include "float_ops.hpp"

namespace mi {

constexpr int kAdapterMaxRank = 128;
constexpr int kAdapterTileLen = 8;       // the shortest sequence that goes in tiles

struct AdapterArgs {
    const void *x, *y;
    void *out;
    int64_t ldx, bsx, ldy, bsy, ldo, bso;
    const float *x_scale;      // [batch, len]
    const void *a, *b;         // [bank, rank, k], [bank, n, rank]
    const float *scales;       // [bank]
    const int32_t *ids, *lens;
    void *t;                   // rows: float [rows, rank]; tiles: bf16 [3, rows, ranks]
    int batch, len, k, n, rank, ranks, bank;
    int up_tokens;             // of a block of the second kernel, a multiple of 16 UT
};

// The adapter of a sequence, -1 for none; tokens of it.
__device__ __forceinline__ int adapter_of(const AdapterArgs &a, int b) {
    const int id = a.ids[b];
    return (unsigned)id < (unsigned)a.bank ? id : -1;
}
__device__ __forceinline__ int tokens_of(const AdapterArgs &a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.len) : a.len;
}

// --------------------------------------------------------------- few tokens
// A wave a (row, rank): the row's products with one row of A.
template <class X, class W>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a) {
    constexpr int V = 16 / (sizeof(X) > sizeof(W) ? sizeof(X) : sizeof(W));
    const int64_t row = blockIdx.x;
    const int b = (int)(row / a.len), t = (int)(row % a.len), lane = threadIdx.x & 63;
    const int j = (int)blockIdx.y * 4 + wave_id();
    const int id = adapter_of(a, b);
    if (j >= a.rank || id < 0 || t >= tokens_of(a, b)) return;
    const X *x = static_cast<const X *>(a.x) + (b * a.bsx + t * a.ldx);
    const W *w = static_cast<const W *>(a.a) + ((int64_t)id * a.rank + j) * a.k;
    float s = 0.0f;
    int i = lane * V;
#pragma unroll 4
    for (; i + V <= a.k; i += 64 * V) {
        const auto xv = load_packed<V>(x + i);
        const auto wv = load_packed<V>(w + i);
#pragma unroll
        for (int v = 0; v < V; ++v) s = __builtin_fmaf((float)xv.v[v], (float)wv.v[v], s);
    }
    for (; i < a.k; ++i) s = __builtin_fmaf((float)x[i], (float)w[i], s);      // (one lane's)
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (a.scales) s *= a.scales[id];
    if (a.x_scale) s *= a.x_scale[row];
    if (lane == 0) static_cast<float *>(a.t)[row * a.rank + j] = s;
}

// A thread an output: its row of B is rank adjacent elements.
template <class Y, class W>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a) {
    constexpr int V = 16 / sizeof(W);
    __shared__ float t_row[kAdapterMaxRank];
    const int64_t row = blockIdx.x;
    const int b = (int)(row / a.len), t = (int)(row % a.len);
    const int id = adapter_of(a, b);
    const bool on = id >= 0 && t < tokens_of(a, b);
    if (!on && a.out == a.y) return;
    if (on)
        for (int j = threadIdx.x; j < a.rank; j += 256) t_row[j] = static_cast<const float *>(a.t)[row * a.rank + j];
    __syncthreads();
    const int n = (int)blockIdx.y * 256 + (int)threadIdx.x;
    if (n >= a.n) return;
    const Y y = (static_cast<const Y *>(a.y) + (b * a.bsy + t * a.ldy))[n];
    Y &out = (static_cast<Y *>(a.out) + (b * a.bso + t * a.ldo))[n];
    if (!on) {
        out = y;
        return;
    }
    const W *w = static_cast<const W *>(a.b) + ((int64_t)id * a.n + n) * a.rank;
    float d = 0.0f;
    int j = 0;
    for (; j + V <= a.rank; j += V) {
        const auto wv = load_packed<V>(w + j);
#pragma unroll
        for (int v = 0; v < V; ++v) d = __builtin_fmaf(t_row[j + v], (float)wv.v[v], d);
    }
    for (; j < a.rank; ++j) d = __builtin_fmaf(t_row[j], (float)w[j], d);
    out = (Y)((float)y + d);
}

// -------------------------------------------------------------------- tiles
// Matrix instructions on bf16: a float of more bits goes as the sum of bf16 parts, cut off
// one after the other, which hold all its bits (float32 in three, float16 in two, bf16 and
// int8 in one), and a product as the sum of the parts' products (those of parts whose
// numbers sum to 4 are below 2^-28 of the product and left out).  Sums are in 32 bits.
// (A matrix instruction of float32 has a sixteenth of this one's rate.)
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

template <class T>
constexpr int parts_of() {
    return std::is_same<T, float>::value ? 3 : std::is_same<T, f16_t>::value ? 2 : 1;
}
__device__ __forceinline__ v4f mfma_bf16(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Eight values as operands: the first bf16 of each, and the rest as the next part's.
template <int P>
struct Parts {
    v8b v[P];
};
template <class T>
__device__ __forceinline__ Parts<parts_of<T>()> parts(const Packed<T, 8> &in) {
    constexpr int P = parts_of<T>();
    Parts<P> out;
    if constexpr (std::is_same<T, bf16_t>::value) {
        out.v[0] = __builtin_bit_cast(v8b, in);
    } else {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (float)in.v[i];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = __builtin_bit_cast(uint32_t, f[2 * i]), hi = __builtin_bit_cast(uint32_t, f[2 * i + 1]);
                w[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);      // the upper halves
                if (p + 1 < P) {
                    f[2 * i] -= __builtin_bit_cast(float, lo & 0xffff0000u);
                    f[2 * i + 1] -= __builtin_bit_cast(float, hi & 0xffff0000u);
                }
            }
            out.v[p] = __builtin_bit_cast(v8b, w);
        }
    }
    return out;
}
// Eight adjacent values from column c on, zeros from column n on.
template <class T>
__device__ __forceinline__ Packed<T, 8> load8(const T *p, int c, int n) {
    if (c + 8 <= n) return load_packed<8>(p + c);
    Packed<T, 8> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.v[i] = c + i < n ? p[c + i] : T(0);
    return v;
}
// What the parts leave of an infinity is inf - inf, and 0 * inf with another's parts.  So a sum
// that came out as a NaN is computed again from the values, one by one until it is one itself.
template <class F>
__device__ __forceinline__ float sum_again(int n, F &&term) {
    float s = 0.0f;
    for (int i = 0; i < n && s == s; ++i) s = term(i, s);
    return s;
}
template <int P, int Q>
__device__ __forceinline__ v4f product(const Parts<P> &a, const Parts<Q> &b, v4f d) {
    // the small ones first
#pragma unroll
    for (int s = P + Q - 2; s >= 0; --s) {
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (s < 4 && s - p >= 0 && s - p < Q) d = mfma_bf16(a.v[p], b.v[s - p], d);
    }
    return d;
}

// t of 16 MT tokens: 8 waves share the columns, 64 at a time (a line
// of 16-bit x; 32 where that takes too many registers), and join in LDS.  Operands as
// the instruction takes them: lane 16 g + r has columns 8 g .. + 7 of row r, of A for the
// result's rows (ranks), of x for its columns (tokens), so a lane gets four adjacent ranks of
// a token.  Every load is 16 bytes (32 of float32) of one row.
constexpr int kDownWaves = 8;
template <class X, class W, int MT, int NT>
__global__ __launch_bounds__(kDownWaves * 64) void adapter_down_tiles_kernel(AdapterArgs a) {
    constexpr int S = sizeof(X) == 4 || NT * sizeof(W) > 8 ? 1 : 2;
    __shared__ v4f sums[kDownWaves / 2][MT * NT][64];
    const int b = blockIdx.y, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = wave_id();
    const int id = adapter_of(a, b), tokens = tokens_of(a, b), t0 = (int)blockIdx.x * 16 * MT;
    if (id < 0 || t0 >= tokens) return;
    const X *x[MT];
    const W *w[NT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = static_cast<const X *>(a.x) + (b * a.bsx + min(t0 + 16 * m + r, tokens - 1) * a.ldx);
#pragma unroll
    for (int n = 0; n < NT; ++n) w[n] = static_cast<const W *>(a.a) + ((int64_t)id * a.rank + min(16 * n + r, a.rank - 1)) * a.k;
    v4f d[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) d[m][n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // a turn's operands: S times 32 columns
    struct Turn {
        Packed<X, 8> x[S][MT];
        Packed<W, 8> w[S][NT];
    } turn[2];
    const auto load = [&](int c, Turn &to, auto with) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
#pragma unroll
            for (int m = 0; m < MT; ++m) to.x[s][m] = with(x[m], c + 32 * s + 8 * g);
#pragma unroll
            for (int n = 0; n < NT; ++n) to.w[s][n] = with(w[n], c + 32 * s + 8 * g);
        }
    };
    const auto whole = [](const auto *p, int at) { return load_packed<8>(p + at); };
    const auto add = [&](const Turn &of) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            Parts<parts_of<X>()> xp[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) xp[m] = parts(of.x[s][m]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const auto wp = parts(of.w[s][n]);
#pragma unroll
                for (int m = 0; m < MT; ++m) d[m][n] = product(wp, xp[m], d[m][n]);
            }
        }
    };
    // whole turns, the next one's loads in flight over the products
    constexpr int kStride = kDownWaves * 32 * S;
    int c = wave * 32 * S, turns = (a.k - c) / (32 * S) > 0 ? ((a.k - c) / (32 * S) + kDownWaves - 1) / kDownWaves : 0;
    if (turns > 0) load(c, turn[0], whole);
    for (int i = 0; i < turns; i += 2) {
        if (i + 1 < turns) load(c + kStride, turn[1], whole);
        add(turn[0]);
        if (i + 2 < turns) load(c + 2 * kStride, turn[0], whole);
        if (i + 1 < turns) add(turn[1]);
        c += 2 * kStride;
    }
    c = wave * 32 * S + turns * kStride;
    if (c < a.k) {
        load(c, turn[0], [&](const auto *p, int at) { return load8(p, at, a.k); });
        add(turn[0]);
    }
    // the second half of the waves to the first, then those
    constexpr int HALF = kDownWaves / 2;
    const auto put = [&](int at) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) sums[at][m * NT + n][lane] = d[m][n];
    };
    if (wave >= HALF) put(wave - HALF);
    __syncthreads();
    if (wave < HALF) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) d[m][n] += sums[wave][m * NT + n][lane];
        put(wave);
    }
    __syncthreads();
    for (int tile = wave; tile < MT * NT; tile += kDownWaves) {
        v4f s = sums[0][tile][lane];
#pragma unroll
        for (int v = 1; v < HALF; ++v) s += sums[v][tile][lane];
        const int token = t0 + tile / NT * 16 + r, rank = tile % NT * 16 + 4 * g;
        if (token >= tokens) continue;
        if constexpr (parts_of<X>() > 1 || parts_of<W>() > 1) {
            const X *xp = static_cast<const X *>(a.x) + (b * a.bsx + token * a.ldx);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (s[i] == s[i] || rank + i >= a.rank) continue;
                const W *wp = static_cast<const W *>(a.a) + ((int64_t)id * a.rank + rank + i) * a.k;
                s[i] = sum_again(a.k, [&](int c, float v) { return __builtin_fmaf((float)xp[c], (float)wp[c], v); });
            }
        }
        const int64_t row = (int64_t)b * a.len + token;
        float f = a.scales ? a.scales[id] : 1.0f;
        if (a.x_scale) f *= a.x_scale[row];
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = rank + i < a.rank ? s[i] * f : 0.0f;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            uint32_t o[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t lo = __builtin_bit_cast(uint32_t, v[2 * i]), hi = __builtin_bit_cast(uint32_t, v[2 * i + 1]);
                o[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
                // (an infinity is its first part alone)
                v[2 * i] = fabsf(v[2 * i]) == __builtin_inff() ? 0.0f : v[2 * i] - __builtin_bit_cast(float, lo & 0xffff0000u);
                v[2 * i + 1] = fabsf(v[2 * i + 1]) == __builtin_inff() ? 0.0f : v[2 * i + 1] - __builtin_bit_cast(float, hi & 0xffff0000u);
            }
            *reinterpret_cast<uint2 *>(static_cast<bf16_t *>(a.t) + (p * (int64_t)a.batch * a.len + row) * a.ranks + rank) =
                make_uint2(o[0], o[1]);
        }
        if (NT == 1)      // 32 ranks are read
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<uint2 *>(static_cast<bf16_t *>(a.t) + (p * (int64_t)a.batch * a.len + row) * a.ranks + rank + 16) =
                    make_uint2(0, 0);
    }
}

// out of up_tokens tokens and 16 NT columns a wave, 4 waves side by side.  B's operands stay in
// registers, 16 UT tokens after the other bring t's three parts and y (a turn ahead).  A lane gets
// four adjacent columns of a token from a tile of the result, so B's rows go to tiles such
// that the lane's tiles (two of them for 16-bit y) are 16 adjacent bytes.
template <class Y, class W, int KS, int NT, int UT>
__global__ __launch_bounds__(256, KS == 1 && parts_of<W>() == 1 ? 4 : 1) void adapter_up_tiles_kernel(AdapterArgs a) {
    constexpr int PAIR = sizeof(Y) == 4 ? 1 : 2, V = 4 * PAIR;
    const int b = blockIdx.z, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int id = adapter_of(a, b), tokens = id < 0 || a.rank == 0 ? 0 : tokens_of(a, b), t0 = (int)blockIdx.y * a.up_tokens;
    const int n0 = ((int)blockIdx.x * 4 + wave_id()) * 16 * NT;
    const bool in_place = a.out == a.y;
    if (n0 >= a.n || (in_place && t0 >= tokens)) return;
    const int end = min(t0 + a.up_tokens, in_place ? tokens : a.len);
    const bool whole = n0 + 16 * NT <= a.n;
    // the column of element i of this lane's vector h
    const auto column = [&](int h) { return n0 + h * 16 * PAIR + g * V; };
    Parts<parts_of<W>()> w[NT][KS];
    if (t0 < tokens) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // row r of tile n: of the four lanes' vectors, the one of lane group r / 4
            const int col = n0 + n / PAIR * 16 * PAIR + (r >> 2) * V + n % PAIR * 4 + (r & 3);
            const W *p = static_cast<const W *>(a.b) + ((int64_t)id * a.n + min(col, a.n - 1)) * a.rank;
#pragma unroll
            for (int s = 0; s < KS; ++s) w[n][s] = parts(load8(p, 32 * s + 8 * g, a.rank));
        }
    }
    Packed<Y, V> y[2][UT][NT / PAIR];
    const auto load_y = [&](int t, Packed<Y, V> *to) {
        const Y *p = static_cast<const Y *>(a.y) + (b * a.bsy + min(t + r, a.len - 1) * a.ldy);
#pragma unroll
        for (int h = 0; h < NT / PAIR; ++h) {
            if (whole)
                to[h] = load_packed<V>(p + column(h));
            else {
#pragma unroll
                for (int i = 0; i < V; ++i) to[h].v[i] = column(h) + i < a.n ? p[column(h) + i] : Y(0);
            }
        }
    };
    uint32_t again = 0;      // tiles in which the lane has a NaN, left for later
    const auto tile = [&](int t, const Packed<Y, V> *yv) {
        v4f d[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) d[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (t < tokens) {
            const int64_t row = (int64_t)b * a.len + min(t + r, tokens - 1);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                Parts<3> tp;
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    tp.v[p] = *reinterpret_cast<const v8b *>(static_cast<const bf16_t *>(a.t) +
                                                             (p * (int64_t)a.batch * a.len + row) * a.ranks + 32 * s + 8 * g);
#pragma unroll
                for (int n = 0; n < NT; ++n) d[n] = product(w[n][s], tp, d[n]);
            }
        }
        const bool on = t + r < tokens;
        if (t + r >= (in_place ? tokens : a.len)) return;
        bool odd = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) odd |= __builtin_isunordered(d[n][0], d[n][1]) || __builtin_isunordered(d[n][2], d[n][3]);
        if (on && odd) {
            again |= 1u << (t - t0) / 16;
            return;
        }
        Y *p = static_cast<Y *>(a.out) + (b * a.bso + (t + r) * a.ldo);
#pragma unroll
        for (int h = 0; h < NT / PAIR; ++h) {
            Packed<Y, V> o = yv[h];
            if (on) {
#pragma unroll
                for (int i = 0; i < V; ++i) o.v[i] = (Y)((float)yv[h].v[i] + d[h * PAIR + i / 4][i % 4]);
            }
            if (whole)
                store_packed<V>(p + column(h), o);
            else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (column(h) + i < a.n) p[column(h) + i] = o.v[i];
            }
        }
    };
    const auto load = [&](int t, auto &to) {
#pragma unroll
        for (int u = 0; u < UT; ++u)
            if (t + 16 * u < end) load_y(t + 16 * u, to[u]);
    };
    const auto turn = [&](int t, const auto &yv) {
#pragma unroll
        for (int u = 0; u < UT; ++u)
            if (t + 16 * u < end) tile(t + 16 * u, yv[u]);
    };
    load(t0, y[0]);
    for (int t = t0; t < end; t += 32 * UT) {
        load(t + 16 * UT, y[1]);
        turn(t, y[0]);
        load(t + 32 * UT, y[0]);
        turn(t + 16 * UT, y[1]);
    }
    // (in the loop above it took 31 to 50 registers more)
    const int64_t part = (int64_t)a.batch * a.len * a.ranks;
    for (; again; again &= again - 1) {
        const int t = t0 + 16 * __builtin_ctz(again) + r;
        const bf16_t *tr = static_cast<const bf16_t *>(a.t) + ((int64_t)b * a.len + t) * a.ranks;
#pragma unroll 1
        for (int e = 0; e < 4 * NT; ++e) {
            const int col = column(e / V) + e % V;
            if (col >= a.n) continue;
            const W *wp = static_cast<const W *>(a.b) + ((int64_t)id * a.n + col) * a.rank;
            const float sum = sum_again(a.rank, [&](int j, float v) {
                return __builtin_fmaf((float)tr[j] + (float)tr[j + part] + (float)tr[j + 2 * part], (float)wp[j], v);
            });
            const Y yv = (static_cast<const Y *>(a.y) + (b * a.bsy + t * a.ldy))[col];
            (static_cast<Y *>(a.out) + (b * a.bso + t * a.ldo))[col] = (Y)((float)yv + sum);
        }
    }
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

// Ranks of a row of t in tiles: what the instructions read.
inline int adapter_ranks(int rank) { return rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

template <class X, class Y, class W>
void launch_adapter_rows(const AdapterArgs &a, bool work, hipStream_t st) {
    const unsigned rows = (unsigned)(a.batch * a.len);
    if (work) hipLaunchKernelGGL((adapter_down_kernel<X, W>), dim3(rows, (unsigned)((a.rank + 3) / 4)), dim3(256), 0, st, a);
    hipLaunchKernelGGL((adapter_up_kernel<Y, W>), dim3(rows, (unsigned)((a.n + 255) / 256)), dim3(256), 0, st, a);
}

// The first kernel's tiles have 64 tokens (A is read once for them: 16384 x 4096 of rank 32 in
// bf16 31 us, with 32 tokens 40, with 16 51; a row maximum of the same x 30) where that leaves a
// block for every CU, else 16.
template <class X, class Y, class W>
void launch_adapter_tiles(const AdapterArgs &a, bool work, hipStream_t st) {
    const bool many = (int64_t)((a.len + 63) / 64) * a.batch >= device_cus();
    const auto down = [&](auto kernel, int mt) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((a.len + 16 * mt - 1) / (16 * mt)), (unsigned)a.batch), dim3(kDownWaves * 64), 0, st, a);
    };
    const auto up = [&](auto kernel, int nt, int ut) {
        AdapterArgs b = a;
        const int64_t columns = (a.n + 64 * nt - 1) / (64 * nt);
        // as many tokens a block as leave 1024 blocks, 64 at most while the grid has room (8 x 2048
        // -> 2048 in bf16: 33.8 us, 128 tokens 35.5; 8 tiles of columns a wave 44)
        b.up_tokens = a.len <= 64 * 65535 ? 64 : 128;
        while (b.up_tokens > 16 * ut && columns * a.batch * ((a.len + b.up_tokens - 1) / b.up_tokens) < 1024) b.up_tokens /= 2;
        hipLaunchKernelGGL(kernel, dim3((unsigned)columns, (unsigned)((a.len + b.up_tokens - 1) / b.up_tokens), (unsigned)a.batch),
                           dim3(256), 0, st, b);
    };
    if (work) {
        const auto ranks = [&](auto nt) {
            constexpr int NT = decltype(nt)::value, P = std::max(parts_of<X>(), parts_of<W>());
            constexpr int MT = NT < 4 ? 4 : NT == 4 ? (P == 1 ? 4 : 2) : P == 1 ? 2 : 1;      // (registers)
            if (many)
                down(adapter_down_tiles_kernel<X, W, MT, NT>, MT);
            else
                down(adapter_down_tiles_kernel<X, W, 1, NT>, 1);
        };
        if (a.rank <= 16)
            ranks(std::integral_constant<int, 1>{});
        else if (a.rank <= 32)
            ranks(std::integral_constant<int, 2>{});
        else if (a.rank <= 64)
            ranks(std::integral_constant<int, 4>{});
        else
            ranks(std::integral_constant<int, 8>{});
    }
    // B's parts in registers: 16 a tile of columns for 32 ranks and part
    constexpr int P = parts_of<W>(), UT = sizeof(Y) == 4 ? 1 : 2;
    if (a.rank <= 32)
        up(adapter_up_tiles_kernel<Y, W, 1, 4, UT>, 4, UT);
    else if (a.rank <= 64)
        up(adapter_up_tiles_kernel<Y, W, 2, P < 3 ? 4 : 2, UT>, P < 3 ? 4 : 2, UT);
    else
        up(adapter_up_tiles_kernel<Y, W, 4, P < 2 ? 4 : 2, 1>, P < 2 ? 4 : 2, 1);
}

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_adapter_workspace_size(int batch, int len, int rank, size_t *bytes) {
    clear_error();
    MI_REQUIRE(bytes, MI_ERR_NULL_POINTER, "mi_adapter_workspace_size: bytes is required");
    MI_REQUIRE(batch >= 0 && len >= 0 && rank >= 0 && rank <= kAdapterMaxRank, MI_ERR_BAD_DIM,
               "mi_adapter_workspace_size: a size is negative, or rank=%d above %d", rank, kAdapterMaxRank);
    MI_REQUIRE((int64_t)batch * len < (1 << 22), MI_ERR_BAD_DIM, "mi_adapter_workspace_size: batch * len must be below %d", 1 << 22);
    const size_t rows = (size_t)batch * len;
    *bytes = len < kAdapterTileLen ? (rows * rank * sizeof(float) + 15) / 16 * 16 : rank ? rows * adapter_ranks(rank) * 3 * 2 : 0;
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
    MI_REQUIRE(len < kAdapterTileLen || batch <= 65535, MI_ERR_BAD_DIM, "mi_adapter_add: batch=%d of %d tokens and more must be at most 65535",
               batch, kAdapterTileLen);
    MI_REQUIRE(known_type(type) && known_type(weight_type) && (x_type == MI_I8 || x_type == type), MI_ERR_BAD_ARG,
               "mi_adapter_add: unknown element type, or x neither MI_I8 nor y's");
    MI_REQUIRE((x_type == MI_I8) == (x_scale != nullptr), MI_ERR_BAD_ARG, "mi_adapter_add: x_scale goes with 8-bit rows");
    MI_REQUIRE(ldx >= 0 && bsx >= 0 && ldy >= 0 && bsy >= 0, MI_ERR_BAD_DIM, "mi_adapter_add: a stride is negative");
    MI_REQUIRE(ldo >= n && bso >= 0, MI_ERR_BAD_DIM, "mi_adapter_add: ldo=%lld must be at least n", (long long)ldo);
    if (batch == 0 || len == 0 || n == 0) return MI_OK;
    MI_REQUIRE(y && out && ids, MI_ERR_NULL_POINTER, "mi_adapter_add: y, out and ids are required");
    MI_REQUIRE(out != y || (ldo == ldy && bso == bsy), MI_ERR_BAD_ARG, "mi_adapter_add: in place, out has y's strides");
    const AdapterArgs args{x, y, out, ldx, bsx, ldy, bsy, ldo, bso, x_scale, a, b, scales, ids, lens,
                           workspace, batch, len, k, n, k ? rank : 0, adapter_ranks(rank), bank, 0};
    const bool work = args.rank && bank;
    if (!work && out == y) return MI_OK;
    MI_REQUIRE(!work || (x && a && b), MI_ERR_NULL_POINTER, "mi_adapter_add: x, a and b are required");
    size_t need = 0;
    mi_adapter_workspace_size(batch, len, args.rank, &need);
    MI_REQUIRE(!work || (workspace && workspace_bytes >= need), MI_ERR_BAD_ARG, "mi_adapter_add: the workspace has %zu bytes, %zu are needed",
               workspace_bytes, need);
    MI_REQUIRE(!work || aligned(workspace, 16), MI_ERR_BAD_ALIGNMENT, "mi_adapter_add: the workspace must be 16-byte aligned");
    const hipStream_t st = as_stream(stream);
    with_adapter_types(x_type, type, weight_type, [&](auto xt, auto yt, auto wt) {
        if (len < kAdapterTileLen)
            launch_adapter_rows<decltype(xt), decltype(yt), decltype(wt)>(args, work, st);
        else
            launch_adapter_tiles<decltype(xt), decltype(yt), decltype(wt)>(args, work, st);
    });
    return check_launch("mi_adapter_add");
}
