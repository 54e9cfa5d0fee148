// product_i8.hip - pulsar_matmul_i8: the product of int8 rows with a scale a token and
// a channel. Its kernels: pk_i8_launch.h.
#include "pk_i8.h"

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
    // no tile that a product takes counts more than these: finer ones are for up to 64 tokens
    // or 256 tiles
    if ((((uint64_t)n_tok + 127u) / 128u * (((uint64_t)out_dim + 127u) / 128u)) >> 31) return reject("matmul_i8 (size)");
    const I8Args a = {(const uint8_t *)w, (const uint8_t *)x, (const float *)w_scales, (const float *)x_scales,
                      (const float *)bias, residual, out, w_stride, x_stride, out_stride, res_stride, in_dim, out_dim,
                      n_tok, act};
    switch (type) {
    case PULSAR_TYPE_F32: return launch_i8<PULSAR_TYPE_F32>(a);
    case PULSAR_TYPE_F16: return launch_i8<PULSAR_TYPE_F16>(a);
    default: return launch_i8<PULSAR_TYPE_BF16>(a);
    }
}
