// pk_epilogue.h - how the dense product kernels write a finished sum.
//
//   PlainOut: out[t][r] = v
//   FusedOut: out[t][r] = act(v + bias[r]) + residual[t][r], rows of both
//             arrays at a stride of their own
//
// An epilogue is fetched before the sum it belongs to is complete (get), so
// that its loads run beside the weights', and applied to it (put). What a call
// leaves out is read from a spare address, at offset 0, and not used: no branch
// around a load, which would make the compiler wait for every load before it.
#pragma once

#include "pk_common.h"

namespace pk {

struct PlainOut {
    struct Got {};
    PK_DEV Got get(uint32_t, uint32_t) const { return {}; }
    PK_DEV void put(float *out, uint32_t out_dim, uint32_t t, uint32_t row, float v, Got) const {
        out[(uint64_t)t * out_dim + row] = v;
    }
};

struct FusedOut {
    const float *bias, *residual;  // a spare address where left out
    uint64_t out_stride, res_stride;
    uint32_t act;
    uint32_t with_bias, with_residual;  // 1 or 0

    struct Got {
        float bias, residual;
    };
    PK_DEV Got get(uint32_t t, uint32_t row) const {
        Got g;
        g.bias = __uint_as_float(ldw32((const uint8_t *)(bias + with_bias * row)));
        g.residual = __uint_as_float(ldw32((const uint8_t *)(residual + with_residual * (t * res_stride + row))));
        return g;
    }
    PK_DEV void put(float *out, uint32_t, uint32_t t, uint32_t row, float v, Got g) const {
        if (with_bias) v += g.bias;
        if (act != PULSAR_EPI_NONE) v = activate(v);
        if (with_residual) v += g.residual;
        out[t * out_stride + row] = v;
    }
    PK_DEV float activate(float v) const {
        switch (act) {
        case PULSAR_EPI_SILU: return v / (1.0f + expf(-v));
        case PULSAR_EPI_GELU: {
            // v/2 (1 + tanh(z)) = v / (1 + exp(-2 z)), z = sqrt(2/pi) (v + 0.044715 v^3)
            const float z = 0.7978845608028654f * (v + 0.044715f * v * v * v);
            return v / (1.0f + expf(-2.0f * z));
        }
        case PULSAR_EPI_RELU: return v > 0.0f ? v : v != v ? v : 0.0f;
        default: return 1.0f / (1.0f + expf(-v));  // PULSAR_EPI_SIGMOID
        }
    }
};

}  // namespace pk
