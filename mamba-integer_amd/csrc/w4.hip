// Products of a few float rows with 4-bit weights and group scales:
//
//   y[m,n] = bias[n] + sum_k x[m,k] * (q[n,k] - zero[n,k/group]) * scale[n,k/group]
//
// Packed weights: blocks of 16 rows x 128 columns, 1024 contiguous bytes each,
// so that a wave reads a block in one 16-byte load a lane and every lane's words
// are matrix-instruction operands as they are.  In a block, the 32-bit word
// 4 * (16 * g + r) + j holds columns 32 j + 8 g .. + 7 of row r: column c of the
// eight in bits 4 (c / 2) for an even c, 16 + 4 (c / 2) for an odd one (the two
// columns of a 16-bit pair lie 16 bits apart).  Scales and zero points lie as
// [row block, group, 16].
#include <type_traits>

#include "float_ops.hpp"

namespace mi {

constexpr int kW4Rows = 16, kW4Cols = 128;

__device__ __forceinline__ int w4_shift(int c) { return 4 * (c >> 1) + 16 * (c & 1); }

template <class S>
__global__ __launch_bounds__(256) void pack_w4_kernel(const uint8_t *codes, const S *scales, const uint8_t *zeros,
                                                      uint32_t *packed, S *scales_out, uint8_t *zeros_out, int n, int k,
                                                      int ng, int ng_pad, int64_t words, int64_t vals) {
    const int kb = (k + kW4Cols - 1) / kW4Cols;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id < words) {
        const int64_t blk = id / 256;
        const int w = (int)(id % 256), j = w & 3, r = (w >> 2) & 15, g = w >> 6;
        const int64_t row = blk / kb * kW4Rows + r;
        const int64_t col = blk % kb * kW4Cols + 32 * j + 8 * g;
        uint32_t v = 0;
        for (int c = 0; c < 8; ++c)
            if (row < n && col + c < k) v |= (uint32_t)(codes[row * k + col + c] & 15) << w4_shift(c);
        packed[id] = v;
    }
    if (id < vals) {
        const int r = (int)(id % kW4Rows);
        const int64_t gi = id / kW4Rows % ng_pad, row = id / kW4Rows / ng_pad * kW4Rows + r;
        const bool in = row < n && gi < ng;
        scales_out[id] = in ? scales[row * ng + gi] : (S)0.0f;
        if (zeros_out) zeros_out[id] = in ? zeros[row * ng + gi] : (uint8_t)0;
    }
}

template <class T, class S>
struct W4Args {
    const T *x;
    int64_t ldx;
    const uint32_t *packed;
    const S *scales;
    const uint8_t *zeros;   // without zero points any readable bytes, `zeroed` false
    const float *bias;
    T *y;
    int64_t ldy;
    int m, n, k, group, ng, zeroed;
};

typedef float v4f __attribute__((ext_vector_type(4)));
typedef bf16_t v8b __attribute__((ext_vector_type(8)));
typedef f16_t v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4f mfma(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Operands of the matrix instruction by the type of x.  A weight is made as 16 + q,
// exact in 16 bits by a shift and a bit select for two of them (q are the top bits of
// the mantissa of 2^4).  f16 then takes 16 + zero off in one packed addition of two,
// exactly; bf16 has none, so the product is made with 16 + q and 16 + zero times the
// row's sum of x is taken off it (its 2^-8 rounding of y hides the bits this costs);
// float32 rows, which keep theirs, enter as three bf16 parts whose sum is the value,
// and their weights are subtracted one by one.
template <class T>
struct W4Type;
template <>
struct W4Type<bf16_t> {
    typedef v8b Vec;
    static constexpr int kParts = 1;
    static constexpr bool kOffset = true;
    static __device__ __forceinline__ v4u pairs(uint32_t w) {
        return v4u{((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                   ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u};
    }
    static __device__ __forceinline__ Vec weights(uint32_t w, float) { return __builtin_bit_cast(Vec, pairs(w)); }
    static __device__ __forceinline__ void split(const Packed<bf16_t, 8> &x, Vec (&o)[1]) {
        o[0] = __builtin_bit_cast(Vec, x);
    }
};
template <>
struct W4Type<f16_t> {
    typedef v8h Vec;
    static constexpr int kParts = 1;
    static constexpr bool kOffset = false;
    static __device__ __forceinline__ Vec weights(uint32_t w, float zero) {
        const v4u r = {((w << 6) & 0x03c003c0u) | 0x4c004c00u, ((w << 2) & 0x03c003c0u) | 0x4c004c00u,
                       ((w >> 2) & 0x03c003c0u) | 0x4c004c00u, ((w >> 6) & 0x03c003c0u) | 0x4c004c00u};
        typedef f16_t v2h __attribute__((ext_vector_type(2)));
        const v2h off = (f16_t)(-16.0f - zero);
        v4u o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t pair = r[i];   // (bit_cast of a vector's element itself takes element 0)
            o[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, pair) + off);
        }
        return __builtin_bit_cast(Vec, o);
    }
    static __device__ __forceinline__ void split(const Packed<f16_t, 8> &x, Vec (&o)[1]) {
        o[0] = __builtin_bit_cast(Vec, x);
    }
};
template <>
struct W4Type<float> {
    typedef v8b Vec;
    static constexpr int kParts = 3;
    static constexpr bool kOffset = false;
    // bf16 is the upper half of float32, and q - zero needs no bits below it
    static __device__ __forceinline__ Vec weights(uint32_t w, float zero) {
        v4u r = W4Type<bf16_t>::pairs(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lo = __builtin_bit_cast(float, r[i] << 16) - (16.0f + zero);
            const float hi = __builtin_bit_cast(float, r[i] & 0xffff0000u) - (16.0f + zero);
            r[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
        }
        return __builtin_bit_cast(Vec, r);
    }
    // each part the leading 8 bits of what the ones before it leave (cut off, not
    // rounded: no part overflows, and the third holds the rest exactly)
    static __device__ __forceinline__ void split(const Packed<float, 8> &x, Vec (&o)[3]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v = x.v[i];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const uint32_t top = __builtin_bit_cast(uint32_t, v) >> 16;
                o[p][i] = __builtin_bit_cast(bf16_t, (uint16_t)top);
                v -= __builtin_bit_cast(float, top << 16);
            }
        }
    }
};

// A block: NT x 16 weight rows and MT x 16 rows of x; its KS waves take every KS-th
// column block and join their sums in LDS, so the block reads each of its weights and
// its rows of x once and no wave waits for another before the end: a call is a few
// memory latencies long.  In the matrix instruction x is operand A (lane: row
// l & 15, columns 8 (l >> 4) .. + 7 of 32) and the weights B (lane: weight row l & 15),
// so a lane's results belong to one weight row and its scale.  Row sums of x (bf16)
// come from a product with ones.
// The loads of a whole column block stand in no branch (one in a branch is waited for
// where it ends), though where its products are many the compiler issues some of x's
// among them (three of the eight with 16-bit rows, MT 2, NT 4 and groups of 32); the
// columns past the whole blocks are a last step of their own.
template <class T, class S, int MT, int NT, int KS, int PER>
__global__ __launch_bounds__(64 * KS) void w4_kernel(W4Args<T, S> a) {
    using W = W4Type<T>;
    using Vec = typename W::Vec;
    constexpr int P = W::kParts;
    const v4u kOnes = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};    // 1 in bf16
    __shared__ v4f part[KS][MT * NT][64];
    const int wave = wave_id(), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int nb_all = (a.n + kW4Rows - 1) / kW4Rows, kb_all = (a.k + kW4Cols - 1) / kW4Cols, kb_whole = a.k / kW4Cols;
    const int m0 = blockIdx.y * 16 * MT;
    const int each = PER > 1 ? 1 : a.group / kW4Cols;                      // column blocks of a group
    const v4u *words[NT];
    const S *scales[NT];
    const uint8_t *zeros[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int64_t nb = min((int)blockIdx.x * NT + nt, nb_all - 1);     // past the last: not stored
        words[nt] = reinterpret_cast<const v4u *>(a.packed) + nb * kb_all * 64 + lane;
        // a lane loads one of the column block's (group, row) values, and gets those it needs from other lanes
        const int64_t at = nb * a.ng * kW4Rows + (lane & (16 * PER - 1));
        scales[nt] = a.scales + at;
        zeros[nt] = a.zeros + at;
    }
    const T *x[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) x[mt] = a.x + (int64_t)min(m0 + 16 * mt + r, a.m - 1) * a.ldx + 8 * g;
    v4f acc[MT][NT] = {};
    auto compute = [&](const v4u (&w)[NT], const Packed<T, 8> (&xv)[MT][4], const float (&s)[NT], const float (&z)[NT]) {
        v4f d[MT][NT], sx[MT];                   // of the group so far; sx: the rows' sums of x
        float sj[NT], zj[NT];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j % (4 / PER) == 0) {
                const int from = 16 * (j * PER / 4) + r;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    sj[nt] = PER == 1 ? s[nt] : __shfl(s[nt], from);
                    zj[nt] = PER == 1 ? z[nt] : __shfl(z[nt], from);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    sx[mt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) d[mt][nt] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                }
            }
            Vec wj[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) wj[nt] = W::weights(w[nt][j], zj[nt]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                Vec parts[P];
                W::split(xv[mt][j], parts);
#pragma unroll
                for (int p = P - 1; p >= 0; --p) {
                    if constexpr (W::kOffset) sx[mt] = mfma(parts[p], __builtin_bit_cast(Vec, kOnes), sx[mt]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) d[mt][nt] = mfma(parts[p], wj[nt], d[mt][nt]);
                }
            }
            if ((j + 1) % (4 / PER) == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
                        acc[mt][nt] += sj[nt] * (W::kOffset ? d[mt][nt] - (16.0f + zj[nt]) * sx[mt] : d[mt][nt]);
            }
        }
    };
    auto zero_of = [&](uint8_t z) { return a.zeroed ? (float)z : 8.0f; };
    for (int kb = wave; kb < kb_whole; kb += KS) {
        v4u w[NT];
        S s[NT];
        uint8_t z[NT];
        Packed<T, 8> xv[MT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            w[nt] = words[nt][(int64_t)kb * 64];
            s[nt] = scales[nt][(int64_t)(kb / each) * (16 * PER)];
            z[nt] = zeros[nt][(int64_t)(kb / each) * (16 * PER)];
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j) xv[mt][j] = load_packed<8>(x[mt] + kb * kW4Cols + 32 * j);
        float sf[NT], zf[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            sf[nt] = (float)s[nt];
            zf[nt] = zero_of(z[nt]);
        }
        compute(w, xv, sf, zf);
    }
    if (kb_whole < kb_all && wave == kb_whole % KS) {
        v4u w[NT];
        float s[NT], z[NT];
        Packed<T, 8> xv[MT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            w[nt] = words[nt][(int64_t)kb_whole * 64];
            s[nt] = (float)scales[nt][(int64_t)(kb_whole / each) * (16 * PER)];
            z[nt] = zero_of(zeros[nt][(int64_t)(kb_whole / each) * (16 * PER)]);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = kb_whole * kW4Cols + 32 * j + i;
                    xv[mt][j].v[i] = k + 8 * g < a.k ? x[mt][k] : (T)0.0f;
                }
        compute(w, xv, s, z);
    }
#pragma unroll
    for (int i = 0; i < MT * NT; ++i) part[wave][i][lane] = acc[i / NT][i % NT];
    __syncthreads();
    for (int i = wave; i < MT * NT; i += KS) {
        v4f sum = part[0][i][lane];
#pragma unroll
        for (int w = 1; w < KS; ++w) sum += part[w][i][lane];
        const int n = (int)(blockIdx.x * NT + i % NT) * kW4Rows + r;
        if (n >= a.n) continue;
        const float bias = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int m = m0 + 16 * (i / NT) + 4 * g + e;
            if (m < a.m) a.y[(int64_t)m * a.ldy + n] = (T)(sum[e] + bias);
        }
    }
}

// PER: groups of a column block (1 for a group of 128 columns and more).
template <class T, class S, int MT, int NT, int KS>
void launch_w4(const W4Args<T, S> &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.n + 16 * NT - 1) / (16 * NT)), (unsigned)((a.m + 16 * MT - 1) / (16 * MT)));
    if (a.group == 32)
        hipLaunchKernelGGL((w4_kernel<T, S, MT, NT, KS, 4>), grid, dim3(64 * KS), 0, st, a);
    else if (a.group == 64)
        hipLaunchKernelGGL((w4_kernel<T, S, MT, NT, KS, 2>), grid, dim3(64 * KS), 0, st, a);
    else
        hipLaunchKernelGGL((w4_kernel<T, S, MT, NT, KS, 1>), grid, dim3(64 * KS), 0, st, a);
}

// More weight rows a block read x fewer times; fewer leave more blocks.  Kernel times in
// us (traced, weights of three sets in turn), bf16 rows and groups of 128 unless named.
// One tile of 16 rows of x, NT 4, 2 and 1: 1 x 2048 -> 32000 8.1, 9.6, 8.9; 8 x 2048 ->
// 32000 10.1, 10.9, 13.7; 1 x 2048 -> 8192 5.2, 3.9, 4.1; 1 x 2048 -> 2048 4.7, 3.4, 3.1.
// Two tiles, NT 4 and 2: 64 x 2048 -> 8192 8.3 and 11.1, f16 with groups of 32 9.3 and 12.0;
// 64 x 2048 -> 2048 7.5 and 7.2.  64 rows as one block of four tiles, 64 x 2048 -> 8192: 13.2,
// as two of two tiles, which read the weights twice, 8.3.  Four waves and eight where column
// blocks are fewer than those: 64 x 768 -> 32000 14.8 and 17.7 (float32 rows, groups of 64:
// 35.1 and 30.6).  One tile a block is faster than the two taken for 17 to 32 rows (32 x 2048
// -> 8192, NT 4: 6.2, two tiles and NT 2 8.0) and for few row blocks (64 x 2048 -> 2048, NT 2:
// 5.0 and 7.2).
template <class T, class S>
void launch_w4_shape(const W4Args<T, S> &a, hipStream_t st) {
    const int nb = (a.n + kW4Rows - 1) / kW4Rows, kb = (a.k + kW4Cols - 1) / kW4Cols, cus = device_cus();
    if (a.m <= 16) {
        if (nb >= 4 * cus)
            launch_w4<T, S, 1, 4, 8>(a, st);
        else if (nb >= 2 * cus)
            launch_w4<T, S, 1, 2, 8>(a, st);
        else
            launch_w4<T, S, 1, 1, 8>(a, st);
    } else if (a.m <= 32 || nb < 2 * cus) {
        launch_w4<T, S, 2, 2, 8>(a, st);
    } else if (kb < 8) {
        launch_w4<T, S, 2, 4, 4>(a, st);
    } else {
        launch_w4<T, S, 2, 4, 8>(a, st);
    }
}

// Scales of a row (a group may be any number of columns above k: no sum with it).
inline int w4_scales(int k, int group) { return k / group + (k % group != 0); }
// Groups of one packed row block: whole column blocks of them.
inline int w4_groups(int k, int group) {
    const int kp = (k + kW4Cols - 1) / kW4Cols * kW4Cols;
    return group < kW4Cols ? kp / group : w4_scales(k, group);
}
inline bool w4_group_ok(int group) { return group == 32 || group == 64 || (group > 0 && group % kW4Cols == 0); }

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_pack_w4(const uint8_t *codes, const void *scales, int scale_type, const uint8_t *zeros,
                                uint8_t *packed, void *scales_out, uint8_t *zeros_out, int n, int k, int group,
                                void *stream) {
    clear_error();
    MI_REQUIRE(n >= 0 && k >= 0, MI_ERR_BAD_DIM, "mi_pack_w4: negative size");
    MI_REQUIRE(n <= 1 << 28 && k <= 1 << 30, MI_ERR_BAD_DIM, "mi_pack_w4: n must be at most 2^28, k at most 2^30");
    MI_REQUIRE(w4_group_ok(group), MI_ERR_BAD_ARG, "mi_pack_w4: group=%d must be 32, 64 or a multiple of 128", group);
    MI_REQUIRE(scale_type == MI_F32 || scale_type == MI_F16, MI_ERR_BAD_ARG, "mi_pack_w4: scales are MI_F32 or MI_F16");
    if (n == 0 || k == 0) return MI_OK;
    MI_REQUIRE(codes && scales && packed && scales_out, MI_ERR_NULL_POINTER,
               "mi_pack_w4: codes, scales, packed and scales_out are required");
    MI_REQUIRE(!zeros == !zeros_out, MI_ERR_NULL_POINTER, "mi_pack_w4: zeros and zeros_out go together");
    MI_REQUIRE(aligned(packed, 16), MI_ERR_BAD_ALIGNMENT, "mi_pack_w4: packed must be 16-byte aligned");
    const int64_t nb = (n + kW4Rows - 1) / kW4Rows, kb = (k + kW4Cols - 1) / kW4Cols;
    const int ng = w4_scales(k, group), ng_pad = w4_groups(k, group);
    const int64_t words = nb * kb * 256, vals = nb * ng_pad * kW4Rows;
    MI_REQUIRE(words < ((int64_t)1 << 32), MI_ERR_BAD_DIM, "mi_pack_w4: n * k is too large");
    const int64_t ids = words > vals ? words : vals;
    const dim3 grid((unsigned)((ids + 255) / 256));
    auto go = [&](auto s) {
        using S = decltype(s);
        hipLaunchKernelGGL(pack_w4_kernel<S>, grid, dim3(256), 0, as_stream(stream), codes, static_cast<const S *>(scales),
                           zeros, reinterpret_cast<uint32_t *>(packed), static_cast<S *>(scales_out), zeros_out, n, k, ng,
                           ng_pad, words, vals);
    };
    if (scale_type == MI_F32)
        go(float{});
    else
        go(f16_t{});
    return check_launch("mi_pack_w4");
}

extern "C" mi_status mi_w4_matvec(const void *x, int64_t ldx, int type, const uint8_t *packed, const void *scales,
                                  int scale_type, const uint8_t *zeros, const float *bias, void *y, int64_t ldy, int m,
                                  int n, int k, int group, void *stream) {
    clear_error();
    MI_REQUIRE(m >= 0 && n >= 0 && k >= 1, MI_ERR_BAD_DIM, "mi_w4_matvec: a size is negative, or k=%d not positive", k);
    MI_REQUIRE(k <= 1 << 30, MI_ERR_BAD_DIM, "mi_w4_matvec: k must be at most 2^30");
    MI_REQUIRE(w4_group_ok(group), MI_ERR_BAD_ARG, "mi_w4_matvec: group=%d must be 32, 64 or a multiple of 128", group);
    MI_REQUIRE(known_type(type), MI_ERR_BAD_ARG, "mi_w4_matvec: unknown element type %d", type);
    MI_REQUIRE(scale_type == MI_F32 || scale_type == MI_F16, MI_ERR_BAD_ARG, "mi_w4_matvec: scales are MI_F32 or MI_F16");
    MI_REQUIRE(ldx >= 0 && ldy >= n, MI_ERR_BAD_DIM, "mi_w4_matvec: ldx is negative, or ldy less than n");
    if (m == 0 || n == 0) return MI_OK;
    MI_REQUIRE(x && packed && scales && y, MI_ERR_NULL_POINTER, "mi_w4_matvec: x, packed, scales and y are required");
    MI_REQUIRE(aligned(packed, 16), MI_ERR_BAD_ALIGNMENT, "mi_w4_matvec: packed must be 16-byte aligned");
    MI_REQUIRE((int64_t)m * n < ((int64_t)1 << 31) && m <= 32 * 65535 && n <= 1 << 28, MI_ERR_BAD_DIM,
               "mi_w4_matvec: m * n must be below 2^31, m at most 32 * 65535 and n at most 2^28");
    const hipStream_t st = as_stream(stream);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto s) {
            using S = decltype(s);
            const W4Args<T, S> a{static_cast<const T *>(x), ldx, reinterpret_cast<const uint32_t *>(packed),
                                 static_cast<const S *>(scales),
                                 zeros ? zeros : static_cast<const uint8_t *>(scales), bias, static_cast<T *>(y), ldy, m, n,
                                 k, group, w4_groups(k, group), zeros != nullptr};
            launch_w4_shape<T, S>(a, st);
        };
        if (scale_type == MI_F32)
            go(float{});
        else
            go(f16_t{});
    });
    return check_launch("mi_w4_matvec");
}
