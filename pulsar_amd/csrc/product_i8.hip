// product_i8.hip - pulsar_matmul_i8: the product of int8 rows with a scale a token and
// a channel.
#include "pk_i8.h"

namespace pk {

// ------------------------------------------------------------ lane kernel --
// A wave is one channel and up to T tokens: lane l takes 16 bytes of each 1024 of the
// row, four dot instructions a token.
template <uint32_t TYPE, uint32_t T>
__global__ __launch_bounds__(256) void i8_lane_kernel(I8Args a) {
    const uint32_t lane = threadIdx.x & 63u, r = blockIdx.x * 4u + (threadIdx.x >> 6), t0 = blockIdx.y * T;
    if (r >= a.out_dim) return;  // wave-uniform
    const uint32_t nt = a.n_tok - t0 < T ? a.n_tok - t0 : T;
    const uint8_t *w = a.w + r * a.w_stride, *x = a.x + t0 * a.x_stride;
    int32_t acc[T] = {};
    for (uint32_t k = 16u * lane; k < a.in_dim; k += 1024u) {
        const uint4 wv = ld_i8(w + k, a.in_dim - k);
#pragma unroll
        for (uint32_t t = 0; t < T; t++)
            if (t < nt) acc[t] = dot16(wv, ld_i8(x + t * a.x_stride + k, a.in_dim - k), acc[t]);
    }
#pragma unroll
    for (uint32_t t = 0; t < T; t++) {
        acc[t] = group_sum<64>(acc[t]);
        if (t < nt && lane == t) i8_put<TYPE>(a, t0 + t, r, acc[t]);
    }
}

template <uint32_t TYPE>
static int launch_i8(const I8Args &a) {
    const dim3 grid((a.out_dim + 3u) / 4u, (a.n_tok + 3u) / 4u);
    if (grid.y > 65535u) return reject("matmul_i8");
    hipLaunchKernelGGL((i8_lane_kernel<TYPE, 4>), grid, dim3(256), 0, pk::stream(), a);
    return launch_ok("matmul_i8 launch");
}

}  // namespace pk

extern "C" int pulsar_matmul_i8(void *out, const void *w, const void *w_scales, const void *x, const void *x_scales,
                                const void *bias, const void *residual, uint32_t in_dim, uint32_t out_dim,
                                uint32_t n_tok, uint32_t act, uint32_t type, uint64_t w_stride, uint64_t x_stride,
                                uint64_t out_stride, uint64_t res_stride) {
    using namespace pk;
    if (w_stride == 0) w_stride = in_dim;
    if (x_stride == 0) x_stride = in_dim;
    if (out_stride == 0) out_stride = out_dim;
    if (res_stride == 0) res_stride = out_dim;
    if (!out || !w || !w_scales || !x || !x_scales || in_dim == 0 || in_dim > 131071u || out_dim == 0 || n_tok == 0 ||
        out_dim > 0x7fffffffu || n_tok > 0x7fffffffu || act > PULSAR_EPI_SIGMOID || type > PULSAR_TYPE_BF16)
        return reject("matmul_i8");
    if (w_stride < in_dim || x_stride < in_dim || out_stride < out_dim || (residual && res_stride < out_dim) ||
        w_stride > 1u << 23 || x_stride > 1u << 23 || (out_stride | res_stride) >> 32)
        return reject("matmul_i8 (stride)");
    const uint32_t size = elem_bytes(type);
    const u128 on = size * ((u128)(n_tok - 1u) * out_stride + out_dim);
    if (on >> 62 ||
        (residual && !rows_allow(out, out_stride, residual, res_stride, out_dim, n_tok, size)) ||
        overlap(out, on, x, (u128)(n_tok - 1u) * x_stride + in_dim) ||
        overlap(out, on, w, (u128)(out_dim - 1u) * w_stride + in_dim) || overlap(out, on, w_scales, 4 * (u128)out_dim) ||
        overlap(out, on, x_scales, 4 * (u128)n_tok) || (bias && overlap(out, on, bias, 4 * (u128)out_dim)))
        return reject("matmul_i8 (overlap)");
    const I8Args a = {(const uint8_t *)w, (const uint8_t *)x, (const float *)w_scales, (const float *)x_scales,
                      (const float *)bias, residual, out, w_stride, x_stride, out_stride, res_stride, in_dim, out_dim,
                      n_tok, act};
    switch (type) {
    case PULSAR_TYPE_F32: return launch_i8<PULSAR_TYPE_F32>(a);
    case PULSAR_TYPE_F16: return launch_i8<PULSAR_TYPE_F16>(a);
    default: return launch_i8<PULSAR_TYPE_BF16>(a);
    }
}
