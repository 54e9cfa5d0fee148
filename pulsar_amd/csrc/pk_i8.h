// pk_i8.h - what the kernels of pulsar_matmul_i8 share: its arrays, loads of int8 rows
// at any byte, and how a finished sum is written.
#pragma once

#include "pk_elem.h"
#include "pk_epilogue.h"

namespace pk {

struct I8Args {
    const uint8_t *w, *x;
    const float *w_scales, *x_scales, *bias;  // bias NULL: none
    const void *residual;                     // NULL: none
    void *out;
    uint64_t w_stride, x_stride, out_stride, res_stride;
    uint32_t in_dim, out_dim, n_tok, act;
};

// 16 bytes at p, of which the first n (16 and more: all) are there; 0 for the others
PK_DEV uint4 ld_i8(const uint8_t *p, uint32_t n) {
    if (n >= 16u) return ldw128(p);
    uint32_t w[4] = {};
#pragma unroll
    for (uint32_t j = 0; j < 16u; j++)
        if (j < n) w[j >> 2] |= ldw8(p + j) << (8u * (j & 3u));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

PK_DEV int32_t dot16(uint4 a, uint4 b, int32_t c) {
    return dot4(a.w, b.w, dot4(a.z, b.z, dot4(a.y, b.y, dot4(a.x, b.x, c))));
}

// N sums of the same token and channels r, r + step, ...: act(x_scale w_scale sum +
// bias) + residual, in f32, rounded to the rows' type at the end
template <uint32_t TYPE, uint32_t N>
PK_DEV void i8_values(const I8Args &a, const int32_t (&sum)[N], float x_scale, const float (&w_scale)[N],
                      const float (&bias)[N], const float (&res)[N], typename Elem<TYPE>::raw (&out)[N]) {
    float v[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i++) v[i] = (float)sum[i] * x_scale * w_scale[i];
    if (a.bias) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) v[i] += bias[i];
    }
    const FusedOut e = {nullptr, nullptr, 0, 0, a.act};
    e.activate(v);
    if (a.residual) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) v[i] += res[i];
    }
#pragma unroll
    for (uint32_t i = 0; i < N; i++) out[i] = Elem<TYPE>::down(v[i]);
}

// One finished sum
template <uint32_t TYPE>
PK_DEV void i8_put(const I8Args &a, uint32_t t, uint32_t r, int32_t sum) {
    typedef typename Elem<TYPE>::raw raw;
    const int32_t s[1] = {sum};
    const float ws[1] = {a.w_scales[r]}, b[1] = {a.bias ? a.bias[r] : 0.0f};
    const float res[1] = {a.residual ? Elem<TYPE>::up(((const raw *)a.residual)[t * a.res_stride + r]) : 0.0f};
    raw o[1];
    i8_values<TYPE, 1>(a, s, a.x_scales[t], ws, b, res, o);
    ((raw *)a.out)[t * a.out_stride + r] = o[0];
}

}  // namespace pk
