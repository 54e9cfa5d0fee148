// pk_i8.h - what the kernels of pulsar_matmul_i8 share: its arrays and how a finished sum
// is written.
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

PK_DEV int32_t dot16(uint4 a, uint4 b, int32_t c) {
    return dot4(a.w, b.w, dot4(a.z, b.z, dot4(a.y, b.y, dot4(a.x, b.x, c))));
}

template <uint32_t N>
PK_DEV void i8_activate(const I8Args &a, float (&v)[N]) {
    const FusedOut e = {nullptr, nullptr, 0, 0, a.act};
    e.activate(v);
}

// One finished sum: act(x_scale w_scale sum + bias) + residual, in f32, rounded to the
// rows' type at the end
template <uint32_t TYPE>
PK_DEV void i8_put(const I8Args &a, uint32_t t, uint32_t r, int32_t sum) {
    typedef typename Elem<TYPE>::raw raw;
    float v[1] = {(float)sum * a.x_scales[t] * a.w_scales[r]};
    if (a.bias) v[0] += a.bias[r];
    i8_activate(a, v);
    if (a.residual) v[0] += Elem<TYPE>::up(((const raw *)a.residual)[t * a.res_stride + r]);
    ((raw *)a.out)[t * a.out_stride + r] = Elem<TYPE>::down(v[0]);
}

template <uint32_t TYPE>
int launch_i8(const I8Args &a);  // for the three types, a translation unit each

}  // namespace pk
