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
//
// What a token costs is its order, not its bytes: 16384 tokens of 256 experts in 8
// groups, 8 winners, take 8.7 us, 3.5 of them a launch of that many blocks, where
// their logits pass at 4.8 TB/s in 3.7 us; by route_token_f64 alone, a wave a token,
// 37.6. One token: 3.9 us; 4096 tokens of 128 experts, softmax: 3.6.
#include "pk_route.h"

namespace pk {

constexpr uint32_t kMaxGroups = 64;
constexpr uint32_t kMaxTokens = 1u << 25;  // a launch has below 2^32 threads, 64 a token at most

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
PK_DEV uint64_t wave_max_u64(uint64_t v) {  // the largest high word, then of those the largest low one
    const uint32_t hi = wave_max_u32((uint32_t)(v >> 32));
    const uint32_t lo = wave_max_u32((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
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
        // `of` lanes a group (a power of two), each the two largest of its share
        uint32_t of = 64u / r.n_group;
        of = 1u << (31 - __builtin_clz(of));
        const uint32_t g = lane / of, first = lane % of;
        double c0 = -INFINITY, c1 = -INFINITY;
        if (g < r.n_group)
            for (uint32_t i = first; i < size; i += of) {
                const double v = c_l[g * size + i];
                c1 = fmax(c1, fmin(c0, v));
                c0 = fmax(c0, v);
            }
        for (uint32_t m = 1; m < of; m <<= 1) {
            const double o0 = __shfl_xor(c0, (int)m, 64), o1 = __shfl_xor(c1, (int)m, 64);
            c1 = fmax(fmax(c1, o1), fmin(c0, o0));
            c0 = fmax(c0, o0);
        }
        // a group of one candidate stands with that one, a group of none behind all
        const double gs = r.group_top == 2u && c1 > -INFINITY ? c0 + c1 : c0;
        const uint64_t gk = c0 > -INFINITY ? order_key(gs) : 0ull;
        uint32_t rank = 0;
        for (uint32_t h = 0; h < r.n_group; h++) {
            const uint64_t o = lane_bcast(gk, h * of);
            rank += o > gk || (o == gk && h < g) ? 1u : 0u;
        }
        const uint64_t kept = __ballot(g < r.n_group && rank < r.topk_group);  // bit g of: group g
#pragma unroll
        for (uint32_t j = 0; j < J; j++) {
            const uint32_t at = (lane * J + j) / size * of;
            if (at >= 64u || !(kept >> at & 1u)) key[j] = 0ull;
        }
        // c_l is read before the wave's next token writes it
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
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
        r.weights[(uint64_t)token * r.k_used + lane] = id < 0 ? 0.0f : (float)(ws * (double)r.scale);
    }
}

template <uint32_t J>
__global__ __launch_bounds__(256) void route_groups_f64_kernel(GroupRoute r) {
    __shared__ double c_l[4][64u * J];
    const uint32_t wave = threadIdx.x >> 6, token = blockIdx.x * 4u + wave;
    if (token >= r.n_tok) return;  // whole wave
    route_token_f64<J>(r, token, c_l[wave]);
}


// ---- four tokens a wave, in f32 with a proof of the order -----------------
//
// 16 lanes a token (a DPP row, so that every exchange is a DPP move). A group has
// `of` of them (a power of two), each per_lane of its experts in their order, so
// a lower (lane, place) is a lower id. The choice c is taken in f32 and scaled
// to a 23-bit integer q over a window below the row's best; q, the lane and the
// expert's place in it make one unique 32-bit key, so that sorting keys is
// single max / min operations. The error of q is bounded (err), so keys whose q
// lie `gap` apart are in the order of the 64-bit scores. That settles which
// groups stay, but for a row with two at the border closer than that, whose
// groups' best are scored in 64 bits, and which experts win; the winners, and the
// one behind them if it is close, are then put to the test by their 64-bit
// scores. A row that fails one (ties, an order that f32 swapped), that has
// infinite scores or runs out of candidates or of the window, is done again by
// route_token_f64: a row of many ties, a trained router's hardly ever.

constexpr uint32_t kQShift = 9;  // below q: 15 - kk in 4 bits, 31 - j in 5
constexpr float kSteps = 8384000.0f;  // q < 2^23, with room for 4600 steps of rounding

// v as an integer, 0 where it is negative or NaN (as the instruction has it)
PK_DEV uint32_t steps_of(float v) {
    uint32_t q;
    asm("v_cvt_u32_f32 %0, %1" : "=v"(q) : "v"(v));
    return q;
}

template <uint32_t N>
struct SortPairs {  // Batcher's odd-even merge sort of N (a power of two)
    uint32_t n = 0;
    uint8_t a[N * 8] = {}, b[N * 8] = {};
    constexpr SortPairs() {
        for (uint32_t p = 1; p < N; p *= 2)
            for (uint32_t k = p; k >= 1; k /= 2)
                for (uint32_t j = k % p; j + k < N; j += 2 * k)
                    for (uint32_t i = 0; i < k && i + j + k < N; i++)
                        if ((i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                            a[n] = (uint8_t)(i + j);
                            b[n++] = (uint8_t)(i + j + k);
                        }
    }
};

PK_DEV uint32_t max_u(uint32_t a, uint32_t b) { return a > b ? a : b; }
PK_DEV uint32_t min_u(uint32_t a, uint32_t b) { return a < b ? a : b; }
PK_DEV void falling(uint32_t &a, uint32_t &b) {
    const uint32_t x = max_u(a, b);
    b = min_u(a, b);
    a = x;
}

template <uint32_t N>
PK_DEV void sort_falling(uint32_t (&v)[N]) {
    constexpr SortPairs<N> net;
#pragma unroll
    for (uint32_t i = 0; i < net.n; i++) falling(v[net.a[i]], v[net.b[i]]);
}

// a: the N largest of two falling lists, falling (theirs in place, other(i)
// element i of the second): the larger ends of the two, one against the other's
// reverse, are those N, rising then falling; log N steps of exchanges sort them
template <uint32_t N, typename Other>
PK_DEV void merge_falling(uint32_t (&a)[N], Other other) {
    uint32_t o[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i++) o[i] = other(i);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) a[i] = max_u(a[i], o[N - 1u - i]);
#pragma unroll
    for (uint32_t d = N / 2u; d >= 1u; d /= 2u)
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            if (!(i & d)) falling(a[i], a[i + d]);
}

// Reductions over the 16 lanes of a row, the result in all of them
template <typename T, typename F>
PK_DEV T row_reduce(T v, F f) {
#pragma unroll
    for (uint32_t m = 1; m < 16; m <<= 1)
        v = f(v, __builtin_bit_cast(T, partner(__builtin_bit_cast(int32_t, v), m)));
    return v;
}
PK_DEV float row_max_f(float v) {
    return row_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
template <typename F>
PK_DEV double halves(double v, F f) {  // f of both words
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)f((uint32_t)(u >> 32)) << 32 | f((uint32_t)u));
}
PK_DEV double partner_f64(double v, uint32_t m) {
    return halves(v, [m](uint32_t h) { return (uint32_t)partner((int32_t)h, m); });
}
template <typename F>
PK_DEV double row_reduce_f64(double v, F f) {
#pragma unroll
    for (uint32_t m = 1; m < 16; m <<= 1) v = f(v, partner_f64(v, m));
    return v;
}
PK_DEV double row_sum(double v) {
    return row_reduce_f64(v, [](double a, double b) { return a + b; });
}
// lane i gets lane i - 1 of its row, the first one 0
PK_DEV uint32_t row_before(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);
}
// lane i gets lane i + 1 of its row
PK_DEV uint32_t row_behind(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x101, 0xF, 0xF, true);
}
PK_DEV double row_behind(double v) {
    return halves(v, [](uint32_t h) { return row_behind(h); });
}
// lane i gets lane (i - N) % 16 of its row
template <uint32_t N>
PK_DEV uint32_t row_turn(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xF, 0xF, false);
}
template <uint32_t N>
PK_DEV double row_turn(double v) {
    return halves(v, [](uint32_t h) { return row_turn<N>(h); });
}

// e^(l - m) for finite l <= m, within 2^-33 of itself: y = (l - m) log2(e) = n + f,
// 2^f = 1 + f g(f), g the polynomial through (2^f - 1) / f at the 7 Chebyshev
// points of |f| <= 1/2. 0, to any sum with e^0 in it, where l is NaN or far below m
PK_DEV double exp_below(float l, double m) {
    constexpr double g[7] = {0.69314718055994495,   0.2402265092228883,    0.055504108839093055,  0.0096180566785164946,
                             0.0013333502386613757, 0.00015461444699823332, 1.5297323668109702e-05};
    const double y = fmax(((double)l - m) * 1.4426950408889634, -1020.0), n = __builtin_rint(y), f = y - n;
    double p = g[6];
#pragma unroll
    for (int i = 5; i >= 0; i--) p = __builtin_fma(p, f, g[i]);
    const uint64_t power = (uint64_t)((int32_t)n + 1023) << 52;  // 2^n, n in [-1020, 0]
    return __builtin_fma(p, f, 1.0) * __builtin_bit_cast(double, power);
}

// how many of the row's other groups, of G lanes each, have a larger v
template <uint32_t G, uint32_t N = G, typename T>
PK_DEV uint32_t groups_ahead_of(T v) {
    if constexpr (N >= 16u)
        return 0u;
    else
        return (row_turn<N>(v) > v ? 1u : 0u) + groups_ahead_of<G, N + G>(v);
}
template <typename T>
PK_DEV uint32_t groups_ahead(T v, uint32_t of) {  // `of` is uniform
    return of == 1u   ? groups_ahead_of<1>(v)
           : of == 2u ? groups_ahead_of<2>(v)
           : of == 4u ? groups_ahead_of<4>(v)
                      : groups_ahead_of<8>(v);
}

// Blocks start at about one in 4 ns, but of 8 or 16 waves they leave CUs idle
// where they are not a multiple of the 256: 20000 tokens of 256 experts 9.5 us,
// 10.9 and 16.6; 16384 8.2, 8.3 and 9.0.
constexpr uint32_t kRouteWaves = 4;

struct GroupLanes {
    uint32_t size, of_log2, of, per_lane;  // experts and lanes of a group, experts of a lane
    uint32_t by_size, by_lane;  // 2^20 / size and / per_lane, rounded up

    // where a row of `pitch` floats a lane has expert e; e < 512, so the quotients are exact
    PK_DEV uint32_t at(uint32_t e, uint32_t pitch) const {
        const uint32_t g = e * by_size >> 20, i = e - g * size, l = i * by_lane >> 20;
        return (g * of + l) * pitch + i - l * per_lane;
    }
};

// J: experts a lane has room for; K: k_used <= K. n_group <= 16.
template <uint32_t J, uint32_t K>
__global__ __launch_bounds__(64 * kRouteWaves) void route_groups_kernel(GroupRoute r, GroupLanes g) {
    constexpr uint32_t W = kRouteWaves, kJ64 = J < 4u ? 1u : J / 4u;
    // A lane's experts in LDS: rows are read from memory as they lie, 16 lanes
    // that read J floats each then find them on distinct banks
    constexpr uint32_t kPitch = J + 4u, kRow = 16u * kPitch;
    static_assert(4u * kRow * 4u >= 64u * kJ64 * 8u, "route_token_f64's doubles take the rows' place");
    __shared__ __align__(16) float rows_l[W][4u * kRow];
    __shared__ __align__(16) float bias_l[kRow];
    const uint32_t lane = threadIdx.x & 63u, kk = lane & 15u, E = r.n_expert;
    const uint32_t token0 = (blockIdx.x * W + (threadIdx.x >> 6)) * 4u;
    float *mine_l = rows_l[threadIdx.x >> 6];
    if (J >= 4u && E == 16u * J && g.of * r.n_group == 16u) {  // rows of whole 16-byte pieces, one after the other
#pragma unroll
        for (uint32_t i = 0; i < J / 4u; i++) {
            const uint32_t f = (lane + 64u * i) * 4u, t = f / (16u * J), e = f % (16u * J);
            const uint32_t token = token0 + t < r.n_tok ? token0 + t : r.n_tok - 1u;
            *(uint4 *)(mine_l + t * kRow + e / J * kPitch + e % J) =
                    ld128((const uint8_t *)(r.logits + (uint64_t)token * E + e));
        }
    } else {
        constexpr uint32_t P = J < 4u ? 1u : J / 4u;  // 64 P >= E
        float v[P][4];  // all requested before the first is waited for
#pragma unroll
        for (uint32_t p = 0; p < P; p++)
#pragma unroll
            for (uint32_t t = 0; t < 4u; t++) {
                const uint32_t token = token0 + t < r.n_tok ? token0 + t : r.n_tok - 1u;
                v[p][t] = r.logits[(uint64_t)token * E + min_u(lane + 64u * p, E - 1u)];
            }
        for (uint32_t i = lane; i < 4u * kRow; i += 64u) mine_l[i] = __builtin_nanf("");  // no expert there
        __builtin_amdgcn_wave_barrier();  // a wave's LDS writes land in order
#pragma unroll
        for (uint32_t p = 0; p < P; p++) {
            const uint32_t e = lane + 64u * p, at = g.at(e < E ? e : 0u, kPitch);
#pragma unroll
            for (uint32_t t = 0; t < 4u; t++)
                if (e < E) mine_l[t * kRow + at] = v[p][t];
        }
    }
    if (r.bias)
        for (uint32_t e = threadIdx.x; e < E; e += 64u * W) bias_l[g.at(e, kPitch)] = r.bias[e];
    __syncthreads();
    if (token0 >= r.n_tok) return;  // whole wave, behind the block's only barrier
    const uint32_t token = token0 + (lane >> 4);
    const float *row_l = mine_l + (lane >> 4) * kRow;
    // c; NaN or -inf for an expert that is no candidate. err: how far c may be
    // from the exact one, in steps of 2^-24
    float c[J], err, window;
    float m = 0.0f, z = 1.0f;
    double total = 1.0;
    bool unsure = false;
    constexpr float kLog2e = 1.4426950408889634f;
    const bool by_logit = r.softmax && !r.bias && (r.n_group == 1u || r.group_top == 1u);
#pragma unroll
    for (uint32_t j = 0; j < J; j++) {
        const float l = row_l[kk * kPitch + j];
        c[j] = l > -INFINITY ? l : __builtin_nanf("");
    }
    if (r.softmax) {
        m = -INFINITY;
#pragma unroll
        for (uint32_t j = 0; j < J; j++) m = fmaxf(m, c[j]);
        m = row_max_f(m);
        unsure = !(fabsf(m) < INFINITY);
        float x[J];
        if (!r.renorm) {
            // total divides the weights, and f32's sum of exps is off by more than the
            // half step that rounds them. 16384 tokens of 256 experts: 11.0 us, in 8
            // groups 12.4, by f32's sum 9.3 and 10.8
            total = 0.0;
#pragma unroll
            for (uint32_t j = 0; j < J; j++) {
                const double term = exp_below(c[j], (double)m);
                total += term;
                x[j] = __builtin_fmaf(c[j], 0.0f, (float)term);  // NaN stays
            }
            total = row_sum(total);
            z = (float)total;
        } else if (!by_logit) {
            float sum[J];
#pragma unroll
            for (uint32_t j = 0; j < J; j++) {
                x[j] = __builtin_amdgcn_exp2f((c[j] - m) * kLog2e);
                sum[j] = fmaxf(x[j], 0.0f);  // NaN: none
            }
#pragma unroll
            for (uint32_t d = J / 2u; d >= 1u; d /= 2u)
#pragma unroll
                for (uint32_t j = 0; j < d; j++) sum[j] += sum[j + d];
            z = row_reduce(sum[0], [](float a, float b) { return a + b; });
        }
        if (by_logit) {  // the softmax keeps their order
            err = 0.0f;
            window = 16.0f;
        } else {
            // a term e^-x is off by (3 x + 2) steps of itself, at most 2.2 of the
            // largest, z by the terms' mean of that, at most 3 ln 512 + 2 = 20.7,
            // and by the 9 additions of a sum; the quotient and the product 2
            const float rz = 1.0f / z;
#pragma unroll
            for (uint32_t j = 0; j < J; j++) c[j] = x[j] * rz;
            err = 34.0f * rz;
            window = r.bias ? 2.0f : rz;
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < J; j++)
            // e^-l off by (2 |l| + 2) steps of itself, which moves s by at most 2;
            // the sum, the reciprocal and its rounding 4
            c[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(c[j] * -kLog2e));
        err = 8.0f;
        window = r.bias ? 2.0f : 1.0f;
    }
    if (r.bias) {
#pragma unroll
        for (uint32_t j = 0; j < J; j++) c[j] += bias_l[kk * kPitch + j];
    }
    // The score in 64 bits of the expert at `at` of the row, a softmax's without
    // its sum; the choice of it, a softmax's but for z's error, at most zerr of the
    // score (as f32's above: 20.7 + 9 steps)
    constexpr double zerr = 33.0 * 0x1p-24;
    const double rz = r.softmax && !by_logit ? 1.0 / (double)z : 1.0;
    auto score = [&](uint32_t at) {
        const double raw = (double)row_l[at];
        const double e = exp(r.softmax ? raw - (double)m : -fabs(raw));
        return r.softmax ? e : (raw >= 0.0 ? 1.0 : e) / (1.0 + e);
    };
    auto choice = [&](double s, uint32_t at) { return s * rz + (r.bias ? (double)bias_l[at] : 0.0); };
    float hi = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < J; j++) hi = fmaxf(hi, c[j]);
    hi = row_max_f(hi);
    unsure |= !(fabsf(hi) < INFINITY);
    // q = 0: no candidate, or one below the window (a row that needs it is unsure)
    const float scale = kSteps / window, shift = 2.0f - (hi - window) * scale;
    if (!by_logit) err += fabsf(hi) + window;
    unsure |= !(fabsf(shift) < 6e10f);  // its rounding is the whole row's, below 3600 steps
    // on both sides the error of c, two roundings of a step of q each and its floor
    const float gap_f = 2.0f * err * 0x1p-24f * scale + 8.0f;
    const uint32_t gap = gap_f < kSteps ? (uint32_t)gap_f : 1u << 23;
    constexpr uint32_t N = J < K ? J : K, L = J / N;  // L falling lists of N
    uint32_t s[L][N];
#pragma unroll
    for (uint32_t j = 0; j < J; j++)
        s[j / N][j % N] = steps_of(__builtin_fmaf(c[j], scale, shift)) << kQShift | (31u - j);
    uint32_t top[K];
#pragma unroll
    for (uint32_t i = 0; i < L; i++) {
        sort_falling(s[i]);
        if (i > 0u) merge_falling(s[0], [&](uint32_t k) { return s[i][k]; });
    }
#pragma unroll
    for (uint32_t k = 0; k < K; k++) top[k] = k < N ? s[0][k < N ? k : 0u] | (15u - kk) << 5 : 0u;
    if (r.n_group > 1u) {
        uint32_t g0 = top[0], g1 = K > 1u ? top[K > 1u ? 1 : 0] : 0u;
#pragma unroll
        for (uint32_t st = 1; st < 16u; st <<= 1)
            if (st < g.of) {  // uniform
                const uint32_t o0 = (uint32_t)partner((int32_t)g0, st), o1 = (uint32_t)partner((int32_t)g1, st);
                g1 = max_u(max_u(g1, o1), min_u(g0, o0));
                g0 = max_u(g0, o0);
            }
        const bool two = r.group_top == 2u && E > r.n_group;  // a group of one expert is that one
        const uint32_t q0 = g0 >> kQShift, q1 = g1 >> kQShift, stand = q0 + (two ? q1 : 0u);
        const bool real = kk < r.n_group * g.of;
        // a group that stands with one, or with what the window cut, has no sum here
        unsure |= real && two && q1 == 0u;
        const uint32_t rank = groups_ahead(stand, g.of);  // by all lanes: they read one another
        bool kept = real && rank < r.topk_group;
        const uint32_t last = row_reduce(kept ? stand : UINT32_MAX, min_u), next = row_reduce(kept ? 0u : stand, max_u);
        auto lanes_of = [&](bool b) {  // lanes of the row that say b
            return (uint32_t)__builtin_popcount((uint32_t)(__ballot(b) >> (lane & 48u)) & 0xffffu);
        };
        const bool doubt = lanes_of(kept) != r.topk_group * g.of ||  // equal ones
                           (r.topk_group < r.n_group && last < next + 2u * gap);
        if (__any(doubt)) {
            // a group's two best are among those whose q is within the gap of the second
            const uint32_t second = two ? q1 : q0;
            double c0 = -INFINITY, c1 = -INFINITY;
            bool more = doubt && real;
            unsure |= more && second < gap;
#pragma unroll 1
            for (uint32_t i = 0; i < N; i++) {
                uint32_t key = top[0];
#pragma unroll
                for (uint32_t k = 1; k < N; k++) key = i == k ? top[k] : key;
                more &= (key >> kQShift) + gap > second;
                if (!__any(more)) break;
                const uint32_t at = min_u(kk * kPitch + 31u - (key & 31u), kRow - 1u);
                const double v = more ? choice(score(at), at) : -INFINITY;
                c1 = fmax(c1, fmin(c0, v));
                c0 = fmax(c0, v);
            }
            if constexpr (L > 1u) unsure |= more;  // there may be one behind the list
#pragma unroll
            for (uint32_t st = 1; st < 16u; st <<= 1)
                if (st < g.of) {
                    const double o0 = partner_f64(c0, st), o1 = partner_f64(c1, st);
                    c1 = fmax(fmax(c1, o1), fmin(c0, o0));
                    c0 = fmax(c0, o0);
                }
            const double full = !real ? -INFINITY : two ? c0 + c1 : c0;
            const uint32_t place = groups_ahead(full, g.of);
            const bool stays = real && place < r.topk_group;
            auto least = [](double a, double b) { return fmin(a, b); };
            const double low = row_reduce_f64(stays ? full : INFINITY, least);
            const double high = -row_reduce_f64(stays ? INFINITY : -full, least);
            // z's error of two scores of at most rz (without a bias one factor on all), and what 64 bits round
            const double off = r.softmax && r.bias ? 2.0 * zerr * rz : 0.0;
            unsure |= doubt && !(low - high > off + 1e-15 * (1.0 + fabs(low)));
            kept = doubt ? stays : kept;
        }
        unsure |= lanes_of(kept) != r.topk_group * g.of;
#pragma unroll
        for (uint32_t k = 0; k < K; k++) top[k] = kept ? top[k] : 0u;
    }
    // the lane's best are kept to see what is left behind the row's
    uint32_t own[N];
#pragma unroll
    for (uint32_t k = 0; k < N; k++) own[k] = top[k];
#pragma unroll
    for (uint32_t st = 1; st < 16u; st <<= 1)
        merge_falling(top, [&](uint32_t k) { return (uint32_t)partner((int32_t)top[k], st); });
    // winner k to lane k, the last one to all
    uint32_t won = 0u, last = 0u;
#pragma unroll
    for (uint32_t k = 0; k < K; k++) {
        won = kk == k ? top[k] : won;
        last = k + 1u == r.k_used ? top[k] : last;  // scalar compare
    }
    // the best two keys behind the winners; a lane whose whole list is ahead of
    // them may hold a better one behind it
    uint32_t next = 0u, then = 0u;
#pragma unroll
    for (uint32_t k = 0; k < N; k++) next = max_u(next, own[k] < last ? own[k] : 0u);
    next = row_reduce(next, max_u);
#pragma unroll
    for (uint32_t k = 0; k < N; k++) then = max_u(then, own[k] < next ? own[k] : 0u);
    then = row_reduce(then, max_u);
    unsure |= last >> kQShift == 0u;
    if constexpr (L > 1u) unsure |= own[N - 1u] >= next && own[N - 1u] != 0u;
    const bool close = (last >> kQShift) - (next >> kQShift) < gap;
    const bool crowd = (last >> kQShift) - (then >> kQShift) < gap;
    // The winners are known but for `next`, if it is close to the last of them;
    // lane k_used takes it. Then the order by 64-bit scores, which the weights
    // take anyway
    won = kk == r.k_used ? next : won;
    const bool here = kk < r.k_used, seen = kk <= r.k_used;
    const bool pair = kk + 1u < r.k_used || (close && kk + 1u == r.k_used && kk < 15u);  // with the lane behind
    uint32_t id;
    double w, chosen;
    // by how much a choice has to be ahead of that of a score v: what z's error
    // moves them by, as much of both scores, and what 64 bits round
    auto margin = [&](double v) {
        const double off = r.softmax && r.bias ? fabs(w - v) * (rz * zerr) : 0.0;
        return off + 1e-15 * (r.bias ? fabs(chosen) + w * rz : fabs(chosen));
    };
#pragma unroll 1
    for (uint32_t pass = 0;; pass++) {
        // (a key of 0, no expert's, is an unsure row's)
        const uint32_t from = 15u - (won >> 5 & 15u), nth = 31u - (won & 31u);
        id = (from >> g.of_log2) * g.size + (from & (g.of - 1u)) * g.per_lane + nth;
        const uint32_t at = seen ? min_u(from * kPitch + nth, kRow - 1u) : 0u;
        w = score(at);
        chosen = choice(w, at);
        // equal ones, of equal logits and biases, lie in the order of their keys, their ids'
        const uint32_t logit = __float_as_uint(row_l[at]), bias = r.bias ? __float_as_uint(bias_l[at]) : 0u;
        // (what lanes read of one another is read by all, ahead of any choice)
        const double ahead = chosen - row_behind(chosen), off = margin(row_behind(w));
        const uint32_t apart = (logit ^ row_behind(logit)) | (bias ^ row_behind(bias));
        const bool wrong = pair && !(ahead > off || apart == 0u);
        const uint32_t swap = wrong && ahead < -off ? 1u : 0u;
        if (pass == 3u || !__any(swap != 0u)) {
            unsure |= wrong;
            break;
        }
        // two that f32 has in the wrong order change places
        const uint32_t after = row_behind(won), before = row_before(won);
        const uint32_t down = swap & ~row_before(swap), up = row_before(down);
        won = down ? after : up ? before : won;
    }
    unsure |= close && crowd;
    if (r.k_used == 16u && __any(close)) {  // no lane behind the last one: the two once more
        const uint32_t at2 = min_u((15u - (next >> 5 & 15u)) * kPitch + 31u - (next & 31u), kRow - 1u);
        const double w2 = score(at2);
        unsure |= close && kk == 15u && !(chosen - choice(w2, at2) > margin(w2));
    }
    w = here ? w : 0.0;
    if (r.softmax) {
        if (r.renorm) total = row_sum(w);
        w = total > 0.0 ? w / total : 0.0;  // as far below the row's best as 64 bits reach: 0
    } else if (r.renorm) {
        w /= fmax(row_sum(w), 6.103515625e-5);
    }
    const uint64_t slow = __ballot(unsure);
    if (token < r.n_tok && here && ((slow >> (lane & 48u)) & 0xffffu) == 0u) {
        r.selected[(uint64_t)token * r.k_used + kk] = (int32_t)id;
        r.weights[(uint64_t)token * r.k_used + kk] = (float)(w * (double)r.scale);
    }
    if (slow == 0ull) return;
    // the rows are read before doubles take their place
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (uint32_t i = 0; i < 4u && token0 + i < r.n_tok; i++)  // wave-uniform
        if ((slow >> (16u * i)) & 0xffffu) route_token_f64<kJ64>(r, token0 + i, (double *)mine_l);
}

}  // namespace pk

extern "C" int pulsar_router_select_groups(void *selected, void *weights, const void *logits, const void *bias,
                                           uint32_t n_expert, uint32_t k_used, uint32_t n_group, uint32_t topk_group,
                                           uint32_t group_top, uint32_t score, uint32_t renorm, float weight_scale,
                                           uint32_t n_tok) {
    if (!selected || !weights || !logits || n_tok == 0 || n_tok > pk::kMaxTokens || n_expert == 0 || n_expert > 64u * pk::kMaxPerLane ||
        n_group == 0 || n_group > pk::kMaxGroups || n_expert % n_group != 0 || topk_group == 0 ||
        topk_group > n_group || group_top == 0 || group_top > 2u || k_used == 0 || k_used > 64u ||
        k_used > n_expert / n_group * topk_group || score > 1u)
        return pk::reject("router select groups");
    // other tokens' logits and the bias are still read as a token's results are written
    const pk::u128 out_bytes = 4 * (pk::u128)n_tok * k_used, in_bytes = 4 * (pk::u128)n_tok * n_expert;
    bool over = pk::overlap(selected, out_bytes, weights, out_bytes);
    for (const void *out : {selected, weights})
        over |= pk::overlap(out, out_bytes, logits, in_bytes) ||
                (bias && pk::overlap(out, out_bytes, bias, 4 * (pk::u128)n_expert));
    if (over) return pk::reject("router select groups (overlap)");
    const pk::GroupRoute r = {(const float *)logits, (const float *)bias, (int32_t *)selected, (float *)weights,
                              n_expert, k_used, n_group, topk_group, group_top, score, renorm, n_tok, weight_scale};
    // the f32 kernel: of the 16 lanes of a token, as many to a group as a power of two allows
    uint32_t of_log2 = 4u;
    while (of_log2 > 0u && n_group << of_log2 > 16u) of_log2--;
    const uint32_t of = 1u << of_log2, size = n_expert / n_group;
    const uint32_t per_lane = (size + of - 1u) / of;
    if (n_group <= 16u && per_lane <= 32u && n_expert <= 512u && k_used <= 16u) {
        const pk::GroupLanes lanes = {size, of_log2, of, per_lane, (1u << 20) / size + 1u, (1u << 20) / per_lane + 1u};
        constexpr uint32_t W = pk::kRouteWaves;
#define PK_RGFK(J, K)                                                                                        \
    hipLaunchKernelGGL((pk::route_groups_kernel<J, K>), dim3((n_tok + 4u * W - 1u) / (4u * W)), dim3(64u * W), 0, \
                       pk::stream(), r, lanes)
#define PK_RGF(J)          \
    do {                   \
        if (k_used <= 8u)  \
            PK_RGFK(J, 8); \
        else               \
            PK_RGFK(J, 16); \
    } while (0)
        if (per_lane <= 1u)
            PK_RGF(1);
        else if (per_lane <= 2u)
            PK_RGF(2);
        else if (per_lane <= 4u)
            PK_RGF(4);
        else if (per_lane <= 8u)
            PK_RGF(8);
        else if (per_lane <= 16u)
            PK_RGF(16);
        else
            PK_RGF(32);
#undef PK_RGF
#undef PK_RGFK
        return pk::launch_ok("router select groups launch");
    }
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
