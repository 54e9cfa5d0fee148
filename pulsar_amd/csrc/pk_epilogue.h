// pk_epilogue.h - how the dense product kernels write a finished sum.
//
//   PlainOut: out[t][r] = v
//   FusedOut: out[t][r] = act(v + bias[r]) + residual[t][r], rows of both
//             arrays at a stride of their own
//
// Where a kernel has registers for what an epilogue adds (Term), it fetches it ahead
// of the sum it belongs to, and ahead of the loads that the sum waits for: behind a
// branch that leaves a fetch out, the compiler can only count what was requested
// after it. matvec_kernel and ksplit_kernel do; matvec_wide_kernel (rows of more than
// 32768 values), the 16-row kernel and the wide tile fetch at their end.
#pragma once

#include "pk_common.h"

namespace pk {

// exp(x) within 2 units in the last place. The argument in units of ln 2 is x
// log2(e) = p + lo, lo the rounding of the product and the constant's own, so
// that far from 0 the error does not grow with x as exp2(x log2(e)) alone would;
// 2^lo = 1 + lo ln 2. lo is bounded where p is past exp2's range.
PK_DEV float exp_near(float x) {
    constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f;  // log2(e)
    const float p = x * kHi;
    const float lo = __builtin_fmaf(x, kLo, __builtin_fmaf(x, kHi, -p));
    return __builtin_amdgcn_exp2f(p) *
           __builtin_fmaf(__builtin_amdgcn_fmed3f(lo, -0.5f, 0.5f), 0.693147181f, 1.0f);
}
// 1 / (1 + e^-x) within 4 units (0 below 2^-126): e^-x's 2, the sum's half, the
// reciprocal instruction's 1. expf and a division are within 2, and cost a product
// of 14336 x 4096 with 512 tokens and SiLU 3 of 93 us; its dots are off by more
PK_DEV float sigmoid_near(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_near(-x)); }

struct PlainOut {
    struct Term {};
    PK_DEV Term fetch(uint32_t, uint32_t) const { return {}; }
    PK_DEV void put(float *out, uint32_t out_dim, uint32_t t, uint32_t row, float v, Term) const {
        out[(uint64_t)t * out_dim + row] = v;
    }
};

struct FusedOut {
    const float *bias, *residual;  // NULL: none
    uint64_t out_stride, res_stride;
    uint32_t act;

    struct Term {
        float b, r;
    };
    PK_DEV Term fetch(uint32_t t, uint32_t row) const {  // an element inside the matrix
        Term g = {0.0f, 0.0f};
        if (bias) g.b = bias[row];
        if (residual) g.r = residual[t * res_stride + row];
        return g;
    }
    PK_DEV void put(float *out, uint32_t, uint32_t t, uint32_t row, float v, Term g) const {
        float y[1] = {bias ? v + g.b : v};
        activate(y);
        out[t * out_stride + row] = residual ? y[0] + g.r : y[0];
    }
    // N values at once: one choice of the activation for all
    template <uint32_t N>
    PK_DEV void activate(float (&v)[N]) const {
        switch (act) {
        case PULSAR_EPI_NONE: break;
        case PULSAR_EPI_SILU:
#pragma unroll
            for (uint32_t i = 0; i < N; i++) v[i] *= sigmoid_near(v[i]);
            break;
        case PULSAR_EPI_GELU:  // v/2 (1 + tanh z) = v / (1 + exp(-2 z)), 2 z = sqrt(8 / pi) (v + 0.044715 v^3)
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
                v[i] *= sigmoid_near(1.5957691216057308f * (v[i] + 0.044715f * v[i] * v[i] * v[i]));
            break;
        case PULSAR_EPI_RELU:
#pragma unroll
            for (uint32_t i = 0; i < N; i++) v[i] = v[i] < 0.0f ? 0.0f : v[i];  // NaN stays
            break;
        default:  // PULSAR_EPI_SIGMOID
#pragma unroll
            for (uint32_t i = 0; i < N; i++) v[i] = sigmoid_near(v[i]);
        }
    }
};

}  // namespace pk
