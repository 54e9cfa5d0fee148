// pk_epilogue.h - how the dense product kernels write a finished sum.
//
//   PlainOut: out[t][r] = v
//   FusedOut: out[t][r] = act(v + bias[r]) + residual[t][r], rows of both
//             arrays at a stride of their own
//
// What an epilogue adds is fetched (bias, residual) before the sum it belongs to
// is complete, so that its loads run beside the weights'; put finishes the sum.
// What a call leaves out is read from a spare address, at offset 0, and not
// used: no branch around a load, which would make the compiler wait for every
// load before it.
#pragma once

#include "pk_common.h"

namespace pk {

// exp(x) within 2 units in the last place. The argument in units of ln 2 is x
// log2(e) = p + lo, lo the rounding of the product and the constant's own, so
// that far from 0 the error does not grow with x as exp2(x log2(e)) alone would;
// 2^lo = 1 + lo ln 2. lo is bounded where p is past exp2's range.
PK_DEV float exp_near(float x) {
    constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f;
    const float p = x * kHi;
    const float lo = __builtin_fmaf(x, kLo, __builtin_fmaf(x, kHi, -p));
    return __builtin_amdgcn_exp2f(p) *
           __builtin_fmaf(__builtin_amdgcn_fmed3f(lo, -0.5f, 0.5f), 0.693147181f, 1.0f);
}
PK_DEV float sigmoid_near(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_near(-x)); }

struct PlainOut {
    PK_DEV float bias_of(uint32_t) const { return 0.0f; }
    PK_DEV float residual_of(uint32_t, uint32_t) const { return 0.0f; }
    PK_DEV void put(float *out, uint32_t out_dim, uint32_t t, uint32_t row, float v, float, float) const {
        out[(uint64_t)t * out_dim + row] = v;
    }
};

struct FusedOut {
    const float *bias, *residual;  // a spare address where left out
    uint64_t out_stride, res_stride;
    uint32_t act;
    uint32_t with_bias, with_residual;  // 1 or 0

    PK_DEV float bias_of(uint32_t row) const {
        return __uint_as_float(ldw32((const uint8_t *)(bias + with_bias * row)));
    }
    PK_DEV float residual_of(uint32_t t, uint32_t row) const {
        return __uint_as_float(ldw32((const uint8_t *)(residual + with_residual * (t * res_stride + row))));
    }
    PK_DEV void put(float *out, uint32_t, uint32_t t, uint32_t row, float v, float b, float r) const {
        v = activate(v + (with_bias ? b : 0.0f));
        out[t * out_stride + row] = with_residual ? v + r : v;
    }
    PK_DEV float activate(float v) const {
        switch (act) {
        case PULSAR_EPI_NONE: return v;
        case PULSAR_EPI_SILU: return v * sigmoid_near(v);
        case PULSAR_EPI_GELU:  // v/2 (1 + tanh z) = v / (1 + exp(-2 z)), 2 z = sqrt(8 / pi) (v + 0.044715 v^3)
            return v * sigmoid_near(1.5957691216057308f * (v + 0.044715f * v * v * v));
        case PULSAR_EPI_RELU: return v > 0.0f ? v : v != v ? v : 0.0f;
        default: return sigmoid_near(v);  // PULSAR_EPI_SIGMOID
        }
    }
};

}  // namespace pk
