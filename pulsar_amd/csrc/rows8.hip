// rows8.hip - rows in 8 bits: the norm with the residual's addition
// (pulsar_rms_norm_q8) and the quantizer behind a gated combine
// (pulsar_quantize_i8).
//
// A row is one block's: a lane holds 16 bytes of a chunk (a q8_K block of f32 values, two
// of 16-bit ones), a wave up to eight chunks, so that the row is read once, stays in
// registers and is written once. The norm needs one exchange between the waves: its root
// divides every value of the row alike, so codes and the largest size are those of s *
// gain, known without it. Sums, products and codes in 64 bits cost about what the bytes
// do: a value of a norm is 7 to 17 bytes of traffic and 35 instructions, most of them at the
// rate of f32's. Measured (GB/s of what has to move; inputs from HBM, calls one behind the
// other in a replayed graph, here and below): norm with the residual of 8192 rows of 4096 bf16
// values to int8 56 to 59 us (4100), to q8_K with y 68 (4520), of 2048 rows of f32 to q8_K
// with y 34 (4190); 8192 rows of bf16 quantized as they are 23 (4370), combined by glu first
// 43 (3910).
#include "pk_elem.h"
#include "pk_epilogue.h"

namespace pk {

// Largest sizes and sums over a block of up to 16 waves: one exchange through LDS
struct RowStats {
    double sum[16];
    uint64_t top[16];
};
PK_DEV void block_stats(RowStats &lds, double &sum, uint64_t &top) {
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    if (waves == 1u) return;  // block-uniform
    if (lane == 0u) {
        lds.sum[wave] = sum;
        lds.top[wave] = top;
    }
    __syncthreads();
    sum = 0.0;
    top = 0u;
    for (uint32_t k = 0; k < waves; k++) {
        sum += lds.sum[k];
        top = max_bits(top, lds.top[k]);
    }
}

// A lane's values of a chunk: 16 bytes of the rows' type. A chunk is 64 lanes' worth: one
// q8_K block of f32 values, two of 16-bit ones
template <uint32_t TYPE>
constexpr uint32_t kLane = TYPE == PULSAR_TYPE_F32 ? 4u : 8u;

// The lane's values as int8 codes, packed, and the sum of the codes
template <uint32_t V>
PK_DEV int32_t codes_of(const double (&v)[V], double factor, int8_t (&q)[V]) {
    int32_t sum = 0;
#pragma unroll
    for (uint32_t j = 0; j < V; j++) {
        const int32_t c = code_of(v[j], factor);
        sum += c;
        q[j] = (int8_t)c;
    }
    return sum;
}

// How many of the V values from c0 on are in the row
template <uint32_t V>
PK_DEV uint32_t inside(uint32_t c0, uint32_t dim) {
    return c0 < dim ? (dim - c0 < V ? dim - c0 : V) : 0u;
}

// ------------------------------------------------------------------ norm --

template <uint32_t TYPE>
struct NormArgs {
    typedef typename Elem<TYPE>::raw raw;
    uint8_t *q;
    float *scales;
    raw *y, *sum;
    const raw *x, *residual;
    const float *gain;
    uint64_t x_stride, res_stride, sum_stride, q_stride;
    uint32_t dim, n_rows, format;
    float eps;
};

// s of V values: x + residual, rounded to the rows' type. n: constant where a chunk is whole
template <uint32_t TYPE, uint32_t V>
PK_DEV void norm_load(const NormArgs<TYPE> &a, uint64_t row, uint32_t c0, uint32_t n, float (&s)[V]) {
    load_row<TYPE>(a.x + row * a.x_stride + c0, n, s);
    if (!a.residual) return;
    float r[V];
    load_row<TYPE>(a.residual + row * a.res_stride + c0, n, r);
#pragma unroll
    for (uint32_t j = 0; j < V; j++) s[j] = Elem<TYPE>::up(Elem<TYPE>::down(s[j] + r[j]));
}
template <uint32_t TYPE, uint32_t V>
PK_DEV void norm_put_sum(const NormArgs<TYPE> &a, uint64_t row, uint32_t c0, uint32_t n, const float (&s)[V]) {
    typename Elem<TYPE>::raw w[V];
#pragma unroll
    for (uint32_t j = 0; j < V; j++) w[j] = Elem<TYPE>::down(s[j]);  // exact
    store_row(a.sum + row * a.sum_stride + c0, n, w);
}
// p = s * gain (exact), the squares of s added to ss, the largest |p|, as bits
template <uint32_t TYPE, uint32_t V>
PK_DEV uint64_t norm_products(const NormArgs<TYPE> &a, uint32_t c0, uint32_t n, const float (&s)[V], double (&p)[V],
                              double &ss) {
    float g[V];
    load_row<PULSAR_TYPE_F32>(a.gain + c0, n, g);
    double top = 0.0, poison = 0.0;  // a maximum passes over a NaN
#pragma unroll
    for (uint32_t j = 0; j < V; j++) {
        const double v = s[j];
        ss = __builtin_fma(v, v, ss);
        p[j] = v * (double)g[j];
        top = __builtin_fmax(top, __builtin_fabs(p[j]));
        poison = __builtin_fma(p[j], 0.0, poison);
    }
    return size_bits(poison != poison && top < __builtin_inf() ? poison : top);
}
PK_DEV double norm_root(double sum, uint32_t dim, float eps) {
    const double m = sum / (double)dim + (double)eps;
    return m == 0.0 ? 0.0 : 1.0 / __builtin_sqrt(m);
}
// y and codes of a lane's share of a chunk. top: the largest |p| of what shares a scale
template <uint32_t TYPE, uint32_t V>
PK_DEV void norm_put(const NormArgs<TYPE> &a, uint64_t row, uint32_t c0, uint32_t n, const double (&p)[V], double root,
                     uint64_t top, double factor) {
    if (a.y) {
        typename Elem<TYPE>::raw w[V];
#pragma unroll
        for (uint32_t j = 0; j < V; j++) w[j] = Elem<TYPE>::down((float)(p[j] * root));
        store_row(a.y + row * a.dim + c0, n, w);
    }
    if (!a.q) return;
    int8_t q[V];
    int32_t sum = codes_of(p, factor, q);
    if (a.format == PULSAR_ROWS_I8) {
        store_row((int8_t *)a.q + row * a.q_stride + c0, n, q);
        return;
    }
    sum = group_sum<16u / V>(sum);
    if (c0 >= ((a.dim + 255u) & ~255u)) return;  // the second block of a chunk may not be there
    uint8_t *ob = a.q + (row * ((a.dim + 255u) / 256u) + c0 / 256u) * 292u;
    const uint32_t at = c0 % 256u;
    __builtin_memcpy(ob + 4u + at, q, V);
    if (at % 16u == 0u) {
        const int16_t s16 = (int16_t)sum;
        __builtin_memcpy(ob + 260u + at / 8u, &s16, 2);
    }
    if (at == 0u) {
        const float d = (float)(__builtin_bit_cast(double, top) * root * (1.0 / 127.0));
        __builtin_memcpy(ob, &d, 4);
    }
}

template <uint32_t TYPE, uint32_t NB>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs<TYPE> a) {
    constexpr uint32_t V = kLane<TYPE>;
    typedef typename Elem<TYPE>::raw raw;
    __shared__ RowStats lds;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t row = block_index();
    if (row >= a.n_rows) return;  // block-uniform
    const bool blocks = a.format == PULSAR_ROWS_Q8_K;
    auto first = [&](uint32_t j) { return V * (64u * (wave + waves * j) + lane); };
    // f of how many of the lane's values of chunk j are there: a constant where all lanes'
    // are, whose loads then need no masks (2048 rows of 14336 f32 values to int8 97 us against
    // 106)
    auto with_count = [&](uint32_t j, auto f) {
        if (64u * V * (wave + waves * j + 1u) <= a.dim)  // wave-uniform
            f(V);
        else
            f(inside<V>(first(j), a.dim));
    };
    double ss = 0.0;
    uint64_t top[NB], row_top = 0u;
    // held over the exchange in the rows' type, a quarter of the products' registers: two
    // blocks of a row of 14336 values fit a CU, and the products cost 5 operations again
    raw held[NB][V];
    {
        float s[NB][V];
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) with_count(j, [&](uint32_t n) { norm_load(a, row, first(j), n, s[j]); });
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) {
            with_count(j, [&](uint32_t n) {
                double p[V];
#pragma unroll
                for (uint32_t k = 0; k < V; k++) held[j][k] = Elem<TYPE>::down(s[j][k]);  // exact
                if (a.sum) store_row(a.sum + row * a.sum_stride + first(j), n, held[j]);
                top[j] = norm_products(a, first(j), n, s[j], p, ss);
            });
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        if (blocks)
            top[j] = group_max64<256u / V>(top[j]);
        else
            row_top = max_bits(row_top, top[j]);
    }
    if (!blocks) row_top = group_max64<64>(row_top);
    ss = wave_sum64(ss);
    block_stats(lds, ss, row_top);
    const double root = norm_root(ss, a.dim, a.eps);
    const double row_factor = code_factor(__builtin_bit_cast(double, row_top));
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        if (64u * V * (wave + waves * j) >= a.dim) break;  // wave-uniform
        with_count(j, [&](uint32_t n) {
            float g[V];
            double p[V];
            load_row<PULSAR_TYPE_F32>(a.gain + first(j), n, g);
#pragma unroll
            for (uint32_t k = 0; k < V; k++) p[k] = (double)Elem<TYPE>::up(held[j][k]) * (double)g[k];
            norm_put(a, row, first(j), n, p, root, blocks ? top[j] : row_top,
                     blocks ? code_factor(__builtin_bit_cast(double, top[j])) : row_factor);
        });
    }
    if (a.scales && threadIdx.x == 0u)
        a.scales[row] = (float)(__builtin_bit_cast(double, row_top) * root * (1.0 / 127.0));
}

// Rows of more values than a block holds: read twice, the second time from sum where it
// is written (x and residual may be gone by then)
template <uint32_t TYPE>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs<TYPE> a) {
    constexpr uint32_t V = kLane<TYPE>;
    __shared__ RowStats lds;
    const uint32_t step = V * blockDim.x;
    const uint64_t row = block_index();
    if (row >= a.n_rows) return;  // block-uniform
    const bool blocks = a.format == PULSAR_ROWS_Q8_K;
    double ss = 0.0, p[V];
    uint64_t row_top = 0u;
    float s[V];
    for (uint32_t c0 = V * threadIdx.x; c0 < a.dim; c0 += step) {
        const uint32_t n = inside<V>(c0, a.dim);
        norm_load(a, row, c0, n, s);
        if (a.sum) norm_put_sum(a, row, c0, n, s);
        row_top = max_bits(row_top, norm_products(a, c0, n, s, p, ss));
    }
    ss = wave_sum64(ss);
    row_top = group_max64<64>(row_top);
    block_stats(lds, ss, row_top);
    const double root = norm_root(ss, a.dim, a.eps);
    const double row_factor = code_factor(__builtin_bit_cast(double, row_top));
    const uint32_t chunks = (a.dim + 64u * V - 1u) / (64u * V);  // whole waves: lanes exchange
    for (uint32_t c0 = V * threadIdx.x; c0 / (64u * V) < chunks; c0 += step) {
        const uint32_t n = inside<V>(c0, a.dim);
        if (a.sum)
            load_row<TYPE>(a.sum + row * a.sum_stride + c0, n, s);  // this lane's own stores
        else
            norm_load(a, row, c0, n, s);
        double unused = 0.0;
        uint64_t top = norm_products(a, c0, n, s, p, unused);
        top = blocks ? group_max64<256u / V>(top) : row_top;
        norm_put(a, row, c0, n, p, root, top, blocks ? code_factor(__builtin_bit_cast(double, top)) : row_factor);
    }
    if (a.scales && threadIdx.x == 0u)
        a.scales[row] = (float)(__builtin_bit_cast(double, row_top) * root * (1.0 / 127.0));
}

// ------------------------------------------------------------- quantizer --

// 1 / (1 + e^-z) in 64 bits, within some units in the last place. With E = e^-|z| in
// (0, 1] it is E^(z < 0) / (1 + E), where nothing overflows. e^-|z| = 2^n e^r, r within
// ln 2 / 2 (ln 2 in two parts), by the series to r^12 (what is left: 2^-52); the
// reciprocal of 1 .. 2 from the instruction's 2^-24 in two Newton steps. Of z < 0 it is
// 2^LIFT times as large.
template <int32_t LIFT = 0>
PK_DEV double sigmoid64(double z) {
    const double x = __builtin_fmax(-__builtin_fabs(z), -800.0 - 2 * LIFT);  // E is 0 from -745 - 0.7 LIFT on
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0.6931471805599453, x);  // ln 2 rounded, and what is left of it
    r = __builtin_fma(n, -2.3190468138462996e-17, r);
    double e = 1.0 / 479001600.0;
    constexpr double c[] = {1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                            1.0 / 120.0,      1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
#pragma unroll
    for (int k = 0; k < 12; k++) e = __builtin_fma(e, r, c[k]);
    const double d = 1.0 + __builtin_ldexp(e, (int)n);
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return (z < 0.0 ? __builtin_ldexp(e, (int)n + LIFT) : 1.0) * y;
}
// The gated combine of pk::glu in 64 bits; 2^LIFT times it where the gate is below 0
template <int32_t LIFT = 0>
PK_DEV double glu64(float g, float u, uint32_t op) {
    double v = g, w = u;
    if (op == PULSAR_ACT_SWIGLU_OAI) {
        v = v > 7.0 ? 7.0 : v;  // NaN stays
        w = (w > 7.0 ? 7.0 : w < -7.0 ? -7.0 : w) + 1.0;
        return v * sigmoid64<LIFT>(1.702 * v) * w;
    }
    return v * sigmoid64<LIFT>(v) * w;
}

template <uint32_t TYPE>
struct QuantArgs {
    typedef typename Elem<TYPE>::raw raw;
    uint8_t *q;
    float *scales;
    const raw *x, *up;  // up NULL: x as it is
    uint64_t x_stride, up_stride, q_stride;
    uint32_t dim, n_rows, act_op;
};

template <int32_t LIFT, uint32_t TYPE, uint32_t V>
PK_DEV void quant_values(const QuantArgs<TYPE> &a, uint64_t row, uint32_t c0, uint32_t n, double (&v)[V]) {
    float g[V], u[V];
    load_row<TYPE>(a.x + row * a.x_stride + c0, n, g);
    if (a.up) {
        load_row<TYPE>(a.up + row * a.up_stride + c0, n, u);
#pragma unroll
        for (uint32_t k = 0; k < V; k++) v[k] = glu64<LIFT>(g[k], u[k], a.act_op);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < V; k++) v[k] = g[k];
    }
}
// A row of any length and values, read twice and combined in 64 bits. Where E leaves the
// normal numbers, gates below -708, values are below 2^-884 (E 2^-1022, the gate 2^10, up
// 2^128) and short of bits, and 127 / A overflows for A < 2^-1017. So a row whose largest
// is below 2^-800 is looked at again with 2^600 times its values: they have all their bits
// then. Its gates that are not below 0 have values of 0 (others are above 2^-300).
template <int32_t LIFT = 0, uint32_t TYPE>
PK_DEV void quantize_row(const QuantArgs<TYPE> &a, RowStats &lds) {
    constexpr uint32_t V = kLane<TYPE>;
    const uint32_t step = V * blockDim.x;
    const uint64_t row = block_index();
    double v[V], none = 0.0;
    uint64_t top = 0u;
    for (uint32_t c0 = V * threadIdx.x; c0 < a.dim; c0 += step) {
        quant_values<LIFT>(a, row, c0, inside<V>(c0, a.dim), v);
#pragma unroll
        for (uint32_t k = 0; k < V; k++) top = max_bits(top, size_bits(v[k]));
    }
    top = group_max64<64>(top);
    block_stats(lds, none, top);
    const double largest = __builtin_bit_cast(double, top), factor = code_factor(largest);
    if constexpr (LIFT == 0) {
        if (largest > 0.0 && largest < 0x1p-800) {  // block-uniform
            __syncthreads();  // lds is read
            quantize_row<600>(a, lds);
            return;
        }
    }
    for (uint32_t c0 = V * threadIdx.x; c0 < a.dim; c0 += step) {
        const uint32_t n = inside<V>(c0, a.dim);
        quant_values<LIFT>(a, row, c0, n, v);
        int8_t q[V];
        codes_of(v, factor, q);
        store_row((int8_t *)a.q + row * a.q_stride + c0, n, q);
    }
    if (threadIdx.x == 0u) a.scales[row] = LIFT ? 0.0f : (float)(largest * (1.0 / 127.0));
}
template <uint32_t TYPE>
__global__ __launch_bounds__(1024) void quantize_i8_long_kernel(QuantArgs<TYPE> a) {
    __shared__ RowStats lds;
    if (block_index() >= a.n_rows) return;  // block-uniform
    quantize_row(a, lds);
}

// x as it is
template <uint32_t TYPE, uint32_t NB>
__global__ __launch_bounds__(1024) void quantize_i8_kernel(QuantArgs<TYPE> a) {
    constexpr uint32_t V = kLane<TYPE>;
    __shared__ RowStats lds;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t row = block_index();
    if (row >= a.n_rows) return;  // block-uniform
    auto first = [&](uint32_t j) { return V * (64u * (wave + waves * j) + lane); };
    float x[NB][V];
    double none = 0.0;
    uint32_t top32 = 0u;
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        load_row<TYPE>(a.x + row * a.x_stride + first(j), inside<V>(first(j), a.dim), x[j]);
#pragma unroll
        for (uint32_t k = 0; k < V; k++) {
            const uint32_t w = __float_as_uint(x[j][k]) & 0x7fffffffu;
            top32 = top32 > w ? top32 : w;
        }
    }
    uint64_t top = group_max64<64>(__builtin_bit_cast(uint64_t, (double)__uint_as_float(top32)));
    block_stats(lds, none, top);
    const double largest = __builtin_bit_cast(double, top), factor = code_factor(largest);
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        double v[V];
        int8_t q[V];
#pragma unroll
        for (uint32_t k = 0; k < V; k++) v[k] = x[j][k];
        codes_of(v, factor, q);
        store_row((int8_t *)a.q + row * a.q_stride + first(j), inside<V>(first(j), a.dim), q);
    }
    if (threadIdx.x == 0u) a.scales[row] = (float)(largest * (1.0 / 127.0));
}

// The gated combine in f32, of relative error below 2^-20 (or a step of f32's least
// numbers): the sigmoid's 4 units and the exponent's part that z's rounding leaves (below
// 2^-21 together), 5 roundings. Where the sigmoid's argument z is below kFar it is nearly
// out of f32's range, and the value no use. g u comes first: g of f32's least numbers
// would lose its bits to the sigmoid, and a large u would bring the loss up.
constexpr float kFar = -85.0f;
PK_DEV float glu32(float g, float u, uint32_t op, float &z) {
    if (op == PULSAR_ACT_SWIGLU_OAI) {
        constexpr float kHi = 1.702f, kLo = (float)(1.702 - (double)1.702f);
        g = g > 7.0f ? 7.0f : g;  // NaN stays
        u = (u > 7.0f ? 7.0f : u < -7.0f ? -7.0f : u) + 1.0f;
        z = kHi * g;
        const float lo = __builtin_fmaf(kLo, g, __builtin_fmaf(kHi, g, -z)), e = exp_near(-z);
        return g * __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e, -lo, e)) * u;
    }
    z = g;
    return g * u * sigmoid_near(g);
}
// What passes NaN on: one instruction for three values
PK_DEV float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }
PK_DEV float min3(float a, float b, float c) { return __builtin_elementwise_minimum(__builtin_elementwise_minimum(a, b), c); }

// glu(x, up): 64 bits decide the codes, but few of them need 64 bits. Of the f32 values,
// off by 2^-20, those that may be the row's largest are combined again in 64 bits, and
// those whose code argument (up to 127: off by 2^-13) lies within 2^-12 of a half, one in
// 2000. The common way only asks a lane's largest and its nearest to a half; a lane with
// some looks for which. 4096 rows of 14336 bf16 values take 84 us, 3490 GB/s (175 with
// every value combined in 64 bits); the vector pipes are busy 54% of it, with 31
// instructions a value, two of them transcendental; waves wait 63% of their time for
// memory or one another. 8192 rows of 4096: 43 us, 3900 GB/s.
template <uint32_t TYPE, uint32_t NB>
__global__ __launch_bounds__(1024) void glu_i8_kernel(QuantArgs<TYPE> a) {
    constexpr uint32_t V = kLane<TYPE>;
    typedef typename Elem<TYPE>::raw raw;
    __shared__ RowStats lds, lds64;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t row = block_index();
    if (row >= a.n_rows) return;  // block-uniform
    auto first = [&](uint32_t j) { return V * (64u * (wave + waves * j) + lane); };
    auto whole = [&](uint32_t j) { return 64u * V * (wave + waves * j + 1u) <= a.dim; };  // wave-uniform
    const raw *x = a.x + row * a.x_stride, *up = a.up + row * a.up_stride;
    // value i of the lane (of chunk i / V) in 64 bits
    auto again = [&](uint32_t i, uint32_t &c) {
        c = V * (64u * (wave + waves * (i / V)) + lane) + i % V;
        return glu64(Elem<TYPE>::up(x[c]), Elem<TYPE>::up(up[c]), a.act_op);
    };
    float v[NB][V], most = 0.0f, lowest = 0.0f;  // the lane's largest, and its least z
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        float g[V], u[V], z[V];
        if (whole(j)) {
            load_row<TYPE>(x + first(j), V, g);
            load_row<TYPE>(up + first(j), V, u);
        } else {
            load_row<TYPE>(x + first(j), inside<V>(first(j), a.dim), g);
            load_row<TYPE>(up + first(j), inside<V>(first(j), a.dim), u);
        }
#pragma unroll
        for (uint32_t k = 0; k < V; k++) v[j][k] = glu32(g[k], u[k], a.act_op, z[k]);
#pragma unroll
        for (uint32_t k = 0; k < V; k += 2u) {
            most = max3(most, __builtin_fabsf(v[j][k]), __builtin_fabsf(v[j][k + 1u]));
            lowest = min3(lowest, z[k], z[k + 1u]);
        }
    }
    double none = 0.0;
    uint64_t top = group_max64<64>(__float_as_uint(most) & 0x7fffffffu);
    block_stats(lds, none, top);
    // zeros, values at the ends of f32's range, infinity, NaN
    const float about = __uint_as_float((uint32_t)top);
    if (!(about >= 1e-30f && about <= 1e30f)) {  // block-uniform
        __syncthreads();
        quantize_row(a, lds);
        return;
    }
    uint32_t far = 0u;  // a bit a value: all of a lane's in the row, where one is far
    if (!(lowest >= kFar)) {
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) far |= ((1u << inside<V>(first(j), a.dim)) - 1u) << (j * V);
    }
    uint32_t todo = far;
    const float least = about * (1.0f - 0x1p-18f);
    if (most >= least) {
#pragma unroll
        for (uint32_t i = 0; i < NB * V; i++)
            if (__builtin_fabsf(v[i / V][i % V]) >= least) todo |= 1u << i;
    }
    top = 0u;
    uint32_t c;
    for (; todo; todo &= todo - 1u) top = max_bits(top, size_bits(again(__builtin_ctz(todo), c)));
    top = group_max64<64>(top);
    block_stats(lds64, none, top);
    const double largest = __builtin_bit_cast(double, top), factor = code_factor(largest);
    const float factor32 = (float)factor;
    // code + 128 as an unsigned byte, rounded by the conversion
    auto argument = [&](uint32_t i) { return __builtin_fmaf(v[i / V][i % V], factor32, 128.0f); };
    auto off_half = [&](uint32_t i) { return __builtin_amdgcn_fractf(argument(i)) - 0.5f; };
    float nearest = 1.0f;
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        uint32_t words[V / 4u] = {};
        int8_t q[V];
#pragma unroll
        for (uint32_t k = 0; k < V; k++)
            words[k / 4u] = __builtin_amdgcn_cvt_pk_u8_f32(argument(j * V + k), k % 4u, words[k / 4u]);
#pragma unroll
        for (uint32_t k = 0; k < V; k += 2u)
            nearest = min3(nearest, __builtin_fabsf(off_half(j * V + k)), __builtin_fabsf(off_half(j * V + k + 1u)));
#pragma unroll
        for (uint32_t k = 0; k < V / 4u; k++) words[k] ^= 0x80808080u;
        __builtin_memcpy(q, words, V);
        int8_t *to = (int8_t *)a.q + row * a.q_stride + first(j);
        if (whole(j))
            store_row(to, V, q);
        else
            store_row(to, inside<V>(first(j), a.dim), q);
    }
    todo = far;
    if (nearest < 0x1p-12f) {
#pragma unroll
        for (uint32_t i = 0; i < NB * V; i++)
            if (__builtin_fabsf(off_half(i)) < 0x1p-12f) todo |= 1u << i;
    }
    for (; todo; todo &= todo - 1u) {
        const double w = again(__builtin_ctz(todo), c);
        *(volatile PK_GLOBAL int8_t *)(a.q + row * a.q_stride + c) = (int8_t)code_of(w, factor);
    }
    if (threadIdx.x == 0u) a.scales[row] = (float)(largest * (1.0 / 127.0));
}

// ---------------------------------------------------------------- launch --

// Waves and chunks of a wave for rows of n_chunk chunks; 0 chunks: more than a block holds
struct RowShape {
    uint32_t waves, chunks;
};
// Few rows take as many waves as there are chunks (norm of one row of 4096 bf16 values
// 4.2 us, with two chunks a wave 4.5). Many rows want fewer waves to start and more of a
// row on its way in each: two chunks (8192 rows of 4096 bf16 values, combined: 43 us, one
// chunk 59; normed to int8 56 / 61), and twice as many where a row would take more than 12
// waves, so that a CU has room for a second (4096 rows of 14336 bf16 values combined 84
// against 113, quantized as they are 41 / 49; of 11264, 11 waves, combined 78 against 75). A
// norm has gained nothing by the latter since its whole chunks have no masks (4096 rows of
// 8192 f32 values to int8 87 / 85, to q8_K with y 114 / 111).
static RowShape row_shape(uint32_t n_chunk, uint32_t n_rows, uint32_t most) {
    uint32_t nb = 1u;
    const bool few = n_rows < 256u || n_chunk == 1u;
    if (!few) nb = 2u;
    while (nb < most && n_chunk > (few ? 16u : 12u) * nb) nb <<= 1;
    if (n_chunk > 16u * nb) return {16u, 0u};
    return {(n_chunk + nb - 1u) / nb, nb};
}
// Chunks of a wave at most: 16 values a lane in a norm, whose products are of 64 bits, 32 in
// the quantizers. With masks on its loads a norm was slower with 32 (2048 rows of 14336 f32
// values 151 us against 133); since whole chunks have none, 32 takes 3% less (to int8 93 / 97,
// to q8_K with y 120 / 124)
template <uint32_t TYPE>
constexpr uint32_t kNormChunks = 16u / kLane<TYPE>;
template <uint32_t TYPE>
constexpr uint32_t kQuantChunks = 32u / kLane<TYPE>;

// Rows that may be written while those of `in` are read: the same rows
static bool same_rows(const void *out, uint64_t out_stride, const void *in, uint64_t in_stride) {
    return out == in && out_stride == in_stride;
}

template <uint32_t TYPE>
static int launch_norm(void *q, void *scales, void *y, void *sum, const void *x, const void *residual,
                       const void *gain, uint32_t dim, uint32_t n_rows, float eps, uint32_t format,
                       uint64_t x_stride, uint64_t res_stride, uint64_t sum_stride, uint64_t q_stride) {
    typedef typename Elem<TYPE>::raw raw;
    const NormArgs<TYPE> a = {(uint8_t *)q, (float *)scales, (raw *)y, (raw *)sum, (const raw *)x,
                              (const raw *)residual, (const float *)gain, x_stride, res_stride, sum_stride, q_stride,
                              dim, n_rows, format, eps};
    const RowShape s = row_shape((dim + 64u * kLane<TYPE> - 1u) / (64u * kLane<TYPE>), n_rows, kNormChunks<TYPE>);
    const dim3 grid = grid_of(n_rows), block(64u * s.waves);
    if (s.chunks == 1u)
        hipLaunchKernelGGL((norm_kernel<TYPE, 1>), grid, block, 0, pk::stream(), a);
    else if (s.chunks == 2u)
        hipLaunchKernelGGL((norm_kernel<TYPE, 2>), grid, block, 0, pk::stream(), a);
    else if (s.chunks != 0u)
        hipLaunchKernelGGL((norm_kernel<TYPE, kNormChunks<TYPE>>), grid, block, 0, pk::stream(), a);
    else
        hipLaunchKernelGGL((norm_long_kernel<TYPE>), grid, block, 0, pk::stream(), a);
    return launch_ok("rms_norm_q8 launch");
}

template <uint32_t TYPE>
static int launch_quantize(void *q, void *scales, const void *x, const void *up, uint32_t dim, uint32_t n_rows,
                           uint32_t act_op, uint64_t x_stride, uint64_t up_stride, uint64_t q_stride) {
    typedef typename Elem<TYPE>::raw raw;
    const QuantArgs<TYPE> a = {(uint8_t *)q, (float *)scales, (const raw *)x, (const raw *)up, x_stride, up_stride,
                               q_stride, dim, n_rows, act_op};
    const RowShape s = row_shape((dim + 64u * kLane<TYPE> - 1u) / (64u * kLane<TYPE>), n_rows, kQuantChunks<TYPE>);
    const dim3 grid = grid_of(n_rows), block(64u * s.waves);
#define PK_QUANT_NB(NB)                                                                        \
    do {                                                                                       \
        if (up)                                                                                \
            hipLaunchKernelGGL((glu_i8_kernel<TYPE, NB>), grid, block, 0, pk::stream(), a);      \
        else                                                                                   \
            hipLaunchKernelGGL((quantize_i8_kernel<TYPE, NB>), grid, block, 0, pk::stream(), a); \
    } while (0)
    if (s.chunks == 1u)
        PK_QUANT_NB(1);
    else if (s.chunks == 2u)
        PK_QUANT_NB(2);
    else if (s.chunks == 4u)
        PK_QUANT_NB(4);
    else if (s.chunks != 0u)
        PK_QUANT_NB(kQuantChunks<TYPE>);
    else
        hipLaunchKernelGGL((quantize_i8_long_kernel<TYPE>), grid, block, 0, pk::stream(), a);
#undef PK_QUANT_NB
    return launch_ok("quantize_i8 launch");
}

// Bytes from the first to the last of n rows
static u128 span(uint32_t n, uint64_t stride, uint64_t dim, uint32_t size) {
    return size * ((u128)(n - 1u) * stride + dim);
}

}  // namespace pk

extern "C" int pulsar_rms_norm_q8(void *q, void *scales, void *y, void *sum, const void *x, const void *residual,
                                  const void *gain, uint32_t dim, uint32_t n_rows, float eps, uint32_t type,
                                  uint32_t format, uint64_t x_stride, uint64_t res_stride, uint64_t sum_stride,
                                  uint64_t q_stride) {
    using namespace pk;
    const bool blocks = format == PULSAR_ROWS_Q8_K;
    if (!x || !gain || (!y && !q) || dim == 0 || dim > 1u << 24 || n_rows == 0 || n_rows > 0x7fffffffu ||
        !(eps >= 0.0f) || eps > 3.4028235e38f || type > PULSAR_TYPE_BF16 || format > PULSAR_ROWS_I8 ||
        (blocks && (scales || q_stride)) || (!blocks && !q != !scales) || (!q && q_stride))
        return reject("rms_norm_q8");
    if (x_stride == 0) x_stride = dim;
    if (res_stride == 0) res_stride = dim;
    if (sum_stride == 0) sum_stride = dim;
    if (q_stride == 0) q_stride = dim;
    if (x_stride < dim || res_stride < dim || sum_stride < dim || q_stride < dim ||
        (x_stride | res_stride | sum_stride | q_stride) >> 32)
        return reject("rms_norm_q8 (stride)");
    // arrays that the call reads and writes, with their bytes
    const uint32_t size = elem_bytes(type);
    const struct {
        const void *p;
        u128 n;
    } in[] = {{x, span(n_rows, x_stride, dim, size)},
              {residual, span(n_rows, res_stride, dim, size)},
              {gain, 4 * (u128)dim}},
      out[] = {{sum, span(n_rows, sum_stride, dim, size)},
               {y, span(n_rows, dim, dim, size)},
               {q, blocks ? (u128)n_rows * ((dim + 255u) / 256u) * 292u : span(n_rows, q_stride, dim, 1u)},
               {scales, 4 * (u128)n_rows}};
    for (uint32_t i = 0; i < 4; i++) {
        if (!out[i].p) continue;
        for (uint32_t j = 0; j < 3; j++) {
            if (!in[j].p || !overlap(out[i].p, out[i].n, in[j].p, in[j].n)) continue;
            if (i != 0u || j > 1u || !same_rows(sum, sum_stride, in[j].p, j ? res_stride : x_stride))
                return reject("rms_norm_q8 (overlap)");
        }
        for (uint32_t j = 0; j < i; j++)
            if (out[j].p && overlap(out[i].p, out[i].n, out[j].p, out[j].n)) return reject("rms_norm_q8 (overlap)");
    }
    switch (type) {
#define PK_NORM(T)                                                                                              \
    case T:                                                                                                     \
        return launch_norm<T>(q, scales, y, sum, x, residual, gain, dim, n_rows, eps, format, x_stride, res_stride, \
                              sum_stride, q_stride);
        PK_NORM(PULSAR_TYPE_F32)
        PK_NORM(PULSAR_TYPE_F16)
    default:
        PK_NORM(PULSAR_TYPE_BF16)
#undef PK_NORM
    }
}

extern "C" int pulsar_quantize_i8(void *q, void *scales, const void *x, const void *up, uint32_t dim, uint32_t n_rows,
                                  uint32_t act_op, uint32_t type, uint64_t x_stride, uint64_t up_stride,
                                  uint64_t q_stride) {
    using namespace pk;
    if (!q || !scales || !x || dim == 0 || dim > 1u << 24 || n_rows == 0 || n_rows > 0x7fffffffu ||
        type > PULSAR_TYPE_BF16 ||
        (up ? act_op != PULSAR_ACT_SILU && act_op != PULSAR_ACT_SWIGLU_OAI : act_op != 0u))
        return reject("quantize_i8");
    if (x_stride == 0) x_stride = dim;
    if (up_stride == 0) up_stride = dim;
    if (q_stride == 0) q_stride = dim;
    if (x_stride < dim || up_stride < dim || q_stride < dim || (x_stride | up_stride | q_stride) >> 32)
        return reject("quantize_i8 (stride)");
    const uint32_t size = elem_bytes(type);
    const u128 qn = span(n_rows, q_stride, dim, 1u), sn = 4 * (u128)n_rows, xn = span(n_rows, x_stride, dim, size),
               un = span(n_rows, up_stride, dim, size);
    if (overlap(q, qn, scales, sn) || overlap(q, qn, x, xn) || overlap(scales, sn, x, xn) ||
        (up && (overlap(q, qn, up, un) || overlap(scales, sn, up, un))))
        return reject("quantize_i8 (overlap)");
    switch (type) {
#define PK_QUANT(T) \
    case T: return launch_quantize<T>(q, scales, x, up, dim, n_rows, act_op, x_stride, up_stride, q_stride);
        PK_QUANT(PULSAR_TYPE_F32)
        PK_QUANT(PULSAR_TYPE_F16)
    default:
        PK_QUANT(PULSAR_TYPE_BF16)
#undef PK_QUANT
    }
}
