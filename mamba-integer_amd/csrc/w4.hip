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
    const uint8_t *zeros;
    const float *bias;
    T *y;
    int64_t ldy;
    int m, n, k, group, ng;
};

// One thread an output.
template <class T, class S>
__global__ __launch_bounds__(64) void w4_kernel(W4Args<T, S> a) {
    const int64_t id = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (id >= (int64_t)a.m * a.n) return;
    const int64_t m = id / a.n;
    const int n = (int)(id - m * a.n), r = n % kW4Rows;
    const int64_t nb = n / kW4Rows;
    const int kb = (a.k + kW4Cols - 1) / kW4Cols;
    float acc = 0.0f;
    for (int k = 0; k < a.k; ++k) {
        const int in = k % kW4Cols, c = in & 7;
        const uint32_t w = a.packed[(nb * kb + k / kW4Cols) * 256 + 4 * (16 * ((in & 31) >> 3) + r) + (in >> 5)];
        const int64_t at = (nb * a.ng + k / a.group) * kW4Rows + r;
        const int zero = a.zeros ? a.zeros[at] : 8;
        acc += (float)a.x[m * a.ldx + k] * ((float)((int)((w >> w4_shift(c)) & 15) - zero) * (float)a.scales[at]);
    }
    a.y[m * a.ldy + n] = (T)(acc + (a.bias ? a.bias[n] : 0.0f));
}

// Groups of one packed row block: whole column blocks of them.
inline int w4_groups(int k, int group) {
    const int kp = (k + kW4Cols - 1) / kW4Cols * kW4Cols;
    return group < kW4Cols ? kp / group : (k + group - 1) / group;
}
inline bool w4_group_ok(int group) { return group == 32 || group == 64 || (group > 0 && group % kW4Cols == 0); }

}  // namespace mi

using namespace mi;

extern "C" mi_status mi_pack_w4(const uint8_t *codes, const void *scales, int scale_type, const uint8_t *zeros,
                                uint8_t *packed, void *scales_out, uint8_t *zeros_out, int n, int k, int group,
                                void *stream) {
    clear_error();
    MI_REQUIRE(n >= 0 && k >= 0, MI_ERR_BAD_DIM, "mi_pack_w4: negative size");
    MI_REQUIRE(w4_group_ok(group), MI_ERR_BAD_ARG, "mi_pack_w4: group=%d must be 32, 64 or a multiple of 128", group);
    MI_REQUIRE(scale_type == MI_F32 || scale_type == MI_F16, MI_ERR_BAD_ARG, "mi_pack_w4: scales are MI_F32 or MI_F16");
    if (n == 0 || k == 0) return MI_OK;
    MI_REQUIRE(codes && scales && packed && scales_out, MI_ERR_NULL_POINTER,
               "mi_pack_w4: codes, scales, packed and scales_out are required");
    MI_REQUIRE(!zeros == !zeros_out, MI_ERR_NULL_POINTER, "mi_pack_w4: zeros and zeros_out go together");
    MI_REQUIRE(aligned(packed, 16), MI_ERR_BAD_ALIGNMENT, "mi_pack_w4: packed must be 16-byte aligned");
    const int64_t nb = (n + kW4Rows - 1) / kW4Rows, kb = (k + kW4Cols - 1) / kW4Cols;
    const int ng = (k + group - 1) / group, ng_pad = w4_groups(k, group);
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
    MI_REQUIRE(w4_group_ok(group), MI_ERR_BAD_ARG, "mi_w4_matvec: group=%d must be 32, 64 or a multiple of 128", group);
    MI_REQUIRE(known_type(type), MI_ERR_BAD_ARG, "mi_w4_matvec: unknown element type %d", type);
    MI_REQUIRE(scale_type == MI_F32 || scale_type == MI_F16, MI_ERR_BAD_ARG, "mi_w4_matvec: scales are MI_F32 or MI_F16");
    MI_REQUIRE(ldx >= 0 && ldy >= n, MI_ERR_BAD_DIM, "mi_w4_matvec: ldx is negative, or ldy less than n");
    if (m == 0 || n == 0) return MI_OK;
    MI_REQUIRE(x && packed && scales && y, MI_ERR_NULL_POINTER, "mi_w4_matvec: x, packed, scales and y are required");
    MI_REQUIRE(aligned(packed, 16), MI_ERR_BAD_ALIGNMENT, "mi_w4_matvec: packed must be 16-byte aligned");
    MI_REQUIRE((int64_t)m * n < ((int64_t)1 << 31), MI_ERR_BAD_DIM, "mi_w4_matvec: m * n must be below 2^31");
    const hipStream_t st = as_stream(stream);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto s) {
            using S = decltype(s);
            const W4Args<T, S> a{static_cast<const T *>(x), ldx, reinterpret_cast<const uint32_t *>(packed),
                                 static_cast<const S *>(scales), zeros, bias, static_cast<T *>(y), ldy, m, n, k, group,
                                 w4_groups(k, group)};
            hipLaunchKernelGGL((w4_kernel<T, S>), dim3((unsigned)(((int64_t)m * n + 63) / 64)), dim3(64), 0, st, a);
        };
        if (scale_type == MI_F32)
            go(float{});
        else
            go(f16_t{});
    });
    return check_launch("mi_w4_matvec");
}
