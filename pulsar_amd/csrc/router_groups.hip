// router_groups.hip - routing with expert groups (pulsar_router_select_groups):
// scores, a selection bias, the best groups of experts, the top-k of their
// experts, and the winners' weights.
//
//   s_e = 1 / (1 + exp(-l_e))  or  exp(l_e - m) / sum exp(l - m)
//   c_e = s_e + b_e, a group's score the sum of its group_top largest c
//   the topk_group best groups; the k_used largest c of their experts
//   w = s, over its sum where renorm, times weight_scale
//
// Which experts win is decided as the scores stand in 64 bits: two scores that
// f32 rounds to one value, or swaps, are told apart, so the ids do not depend
// on a rounding; equal scores go to the lower id.
#include "pk_route.h"

namespace pk {

constexpr uint32_t kMaxGroups = 64;

struct GroupRoute {
    const float *logits, *bias;
    int32_t *selected;
    float *weights;
    uint32_t n_expert, k_used, n_group, topk_group, group_top, softmax, renorm, n_tok;
    float scale;
};

// A logit of the finite f32 range; NaN stays NaN, so that it is never a candidate
PK_DEV float finite_logit(float l) { return fabsf(l) > 3.402823466e38f ? copysignf(3.402823466e38f, l) : l; }

PK_DEV bool candidate(float l, float b) { return l > -INFINITY && b > -INFINITY; }

PK_DEV uint64_t order_key(double v) {  // larger value <=> larger key, every non-NaN value >= 1
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);  // -0 -> +0
    return (u >> 63 ? ~u : u | 0x8000000000000000ull) + 1ull;
}

template <typename T>
PK_DEV T lane_bcast(T v, uint32_t lane) {
    uint32_t w[sizeof(T) / 4u];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T) / 4u; i++) w[i] = (uint32_t)__builtin_amdgcn_readlane((int)w[i], (int)lane);
    __builtin_memcpy(&v, w, sizeof(T));
    return v;
}

PK_DEV double wave_sum(double v) {
#pragma unroll
    for (uint32_t m = 1; m < 64; m <<= 1) v += __shfl_xor(v, (int)m, 64);
    return v;
}
PK_DEV uint64_t wave_max_u64(uint64_t v) {
#pragma unroll
    for (uint32_t m = 1; m < 64; m <<= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)v, (int)m, 64);
        v = v > o ? v : o;
    }
    return v;
}

// One token by one wave, everything in 64 bits: lane l holds experts lJ .. lJ
// + J - 1, so a lower lane means a lower id. c_l: n_expert doubles of LDS of
// the wave's own (read where there are groups).
template <uint32_t J>
PK_DEV void route_token_f64(const GroupRoute &r, uint32_t token, double *c_l) {
    const uint32_t lane = threadIdx.x & 63u, E = r.n_expert;
    const float *lg = r.logits + (uint64_t)token * E;
    float l[J];
    double b[J], s[J];
    bool ok[J];
#pragma unroll
    for (uint32_t j = 0; j < J; j++) {
        const uint32_t e = lane * J + j, ec = e < E ? e : E - 1u;
        const float bias = r.bias ? r.bias[ec] : 0.0f;
        l[j] = lg[ec];
        b[j] = (double)bias;
        ok[j] = e < E && candidate(l[j], bias);
        // a masked logit has no part in the softmax either
        if (e >= E || !(l[j] > -INFINITY)) l[j] = -INFINITY;
        else l[j] = finite_logit(l[j]);
    }
    if (r.softmax) {
        float m = -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < J; j++) m = fmaxf(m, l[j]);
        m = wave_max(m);
        double z = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < J; j++) {
            s[j] = l[j] > -INFINITY ? exp((double)l[j] - (double)m) : 0.0;
            z += s[j];
        }
        z = wave_sum(z);
#pragma unroll
        for (uint32_t j = 0; j < J; j++) s[j] /= z;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < J; j++) {
            const double e = exp(-fabs((double)l[j]));
            s[j] = (l[j] >= 0.0f ? 1.0 : e) / (1.0 + e);
        }
    }
    uint64_t key[J];
#pragma unroll
    for (uint32_t j = 0; j < J; j++) key[j] = ok[j] ? order_key(s[j] + b[j]) : 0ull;
    if (r.n_group > 1u) {
        const uint32_t size = E / r.n_group;
#pragma unroll
        for (uint32_t j = 0; j < J; j++)
            if (lane * J + j < E) c_l[lane * J + j] = ok[j] ? s[j] + b[j] : -INFINITY;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // lane g: group g's two largest, then its rank among the groups
        double c0 = -INFINITY, c1 = -INFINITY;
        if (lane < r.n_group)
            for (uint32_t i = 0; i < size; i++) {
                const double v = c_l[lane * size + i];
                c1 = fmax(c1, fmin(c0, v));
                c0 = fmax(c0, v);
            }
        // a group of one candidate stands with that one, a group of none behind all
        const double gs = r.group_top == 2u && c1 > -INFINITY ? c0 + c1 : c0;
        const uint64_t gk = c0 > -INFINITY ? order_key(gs) : 0ull;
        uint32_t rank = 0;
        for (uint32_t h = 0; h < r.n_group; h++) {
            const uint64_t o = lane_bcast(gk, h);
            rank += o > gk || (o == gk && h < lane) ? 1u : 0u;
        }
        const uint64_t kept = __ballot(lane < r.n_group && rank < r.topk_group);
#pragma unroll
        for (uint32_t j = 0; j < J; j++) {
            const uint32_t g = (lane * J + j) / size;
            if (g >= 64u || !(kept >> g & 1u)) key[j] = 0ull;
        }
        __builtin_amdgcn_wave_barrier();  // c_l is read before the wave's next token writes it
    }
    int32_t id = -1;
    double ws = 0.0, sum = 0.0;
    for (uint32_t k = 0; k < r.k_used; k++) {
        uint64_t bk = 0ull;
        uint32_t bj = 0u;
        double bs = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < J; j++)
            if (key[j] > bk) {
                bk = key[j];
                bj = j;
                bs = s[j];
            }
        const uint64_t m = wave_max_u64(bk);
        if (m == 0ull) break;  // no candidate left: the other slots stay -1 with weight 0
        const uint32_t f = (uint32_t)__builtin_ctzll(__ballot(bk == m));
        const int32_t e = (int32_t)lane_bcast(lane * J + bj, f);
        const double p = lane_bcast(bs, f);
#pragma unroll
        for (uint32_t j = 0; j < J; j++)
            if (lane == f && j == bj) key[j] = 0ull;
        if (lane == k) {
            id = e;
            ws = p;
        }
        sum += p;
    }
    if (r.renorm) {
        const double d = r.softmax ? sum : fmax(sum, 6.103515625e-5);
        ws = d > 0.0 ? ws / d : 0.0;
    }
    if (lane < r.k_used) {
        r.selected[(uint64_t)token * r.k_used + lane] = id;
        r.weights[(uint64_t)token * r.k_used + lane] = (float)(ws * (double)r.scale);
    }
}

template <uint32_t J>
__global__ __launch_bounds__(256) void route_groups_f64_kernel(GroupRoute r) {
    __shared__ double c_l[4][64u * J];
    const uint32_t wave = threadIdx.x >> 6, token = blockIdx.x * 4u + wave;
    if (token >= r.n_tok) return;  // whole wave
    route_token_f64<J>(r, token, c_l[wave]);
}

}  // namespace pk

extern "C" int pulsar_router_select_groups(void *selected, void *weights, const void *logits, const void *bias,
                                           uint32_t n_expert, uint32_t k_used, uint32_t n_group, uint32_t topk_group,
                                           uint32_t group_top, uint32_t score, uint32_t renorm, float weight_scale,
                                           uint32_t n_tok) {
    if (!selected || !weights || !logits || n_tok == 0 || n_expert == 0 || n_expert > 64u * pk::kMaxPerLane ||
        n_group == 0 || n_group > pk::kMaxGroups || n_expert % n_group != 0 || topk_group == 0 ||
        topk_group > n_group || group_top == 0 || group_top > 2u || k_used == 0 || k_used > 64u ||
        k_used > n_expert / n_group * topk_group || score > 1u)
        return pk::reject("router select groups");
    const pk::GroupRoute r = {(const float *)logits, (const float *)bias, (int32_t *)selected, (float *)weights,
                              n_expert, k_used, n_group, topk_group, group_top, score, renorm, n_tok, weight_scale};
    const dim3 grid((n_tok + 3u) / 4u);
#define PK_RG64(J) hipLaunchKernelGGL(pk::route_groups_f64_kernel<J>, grid, dim3(256), 0, pk::stream(), r)
    if (n_expert <= 64u)
        PK_RG64(1);
    else if (n_expert <= 128u)
        PK_RG64(2);
    else if (n_expert <= 256u)
        PK_RG64(4);
    else if (n_expert <= 512u)
        PK_RG64(8);
    else
        PK_RG64(16);
#undef PK_RG64
    return pk::launch_ok("router select groups launch");
}
