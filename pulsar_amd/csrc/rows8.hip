// rows8.hip - rows in 8 bits: the norm with the residual's addition
// (pulsar_rms_norm_q8) and the quantizer behind a gated combine
// (pulsar_quantize_i8).
//
// A row is one block's: lane l of a wave holds values 4 l .. 4 l + 3 of a chunk of 256
// (a q8_K block), a wave NB chunks, so that the row is read once, stays in registers as
// 64-bit products and is written once. The norm needs one exchange between the waves: its root
// divides every value of the row alike, so codes and the largest size are those of s *
// gain, known without it. 64 bits cost no time that the bytes do not: a value is 10 to 13
// bytes of traffic and about 10 operations at the rate of f32's.
#include "pk_elem.h"

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

// The lane's 4 values as int8 codes, packed, and the sum of the codes
PK_DEV uint32_t codes4(const double (&v)[4], double factor, int32_t &sum) {
    uint32_t packed = 0;
    sum = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int32_t q = code_of(v[j], factor);
        sum += q;
        packed |= ((uint32_t)q & 0xffu) << (8 * j);
    }
    return packed;
}
PK_DEV void store_codes(uint8_t *p, uint32_t n, uint32_t packed) {
    if (n >= 4u)
        __builtin_memcpy(p, &packed, 4);
    else {
#pragma unroll
        for (uint32_t j = 0; j < 3u; j++)
            if (j < n) *(volatile PK_GLOBAL uint8_t *)(p + j) = (uint8_t)(packed >> (8 * j));
    }
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
    uint32_t dim, format;
    float eps;
};

// s of 4 values: x + residual, rounded to the rows' type
template <uint32_t TYPE>
PK_DEV void norm_load(const NormArgs<TYPE> &a, const typename Elem<TYPE>::raw *x,
                      const typename Elem<TYPE>::raw *res, uint32_t n, float (&s)[4]) {
    load_row4<TYPE>(x, n, s);
    if (!a.residual) return;
    float r[4];
    load_row4<TYPE>(res, n, r);
#pragma unroll
    for (int j = 0; j < 4; j++) s[j] = Elem<TYPE>::up(Elem<TYPE>::down(s[j] + r[j]));
}
template <uint32_t TYPE>
PK_DEV void norm_put_sum(typename Elem<TYPE>::raw *sum, uint32_t n, const float (&s)[4]) {
    typename Elem<TYPE>::raw w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = Elem<TYPE>::down(s[j]);  // exact
    store_row4<TYPE>(sum, n, w);
}
PK_DEV double norm_root(double sum, uint32_t dim, float eps) {
    const double m = sum / (double)dim + (double)eps;
    return m == 0.0 ? 0.0 : 1.0 / __builtin_sqrt(m);
}
// y and codes of one chunk. top: the largest |p| of what shares a scale
template <uint32_t TYPE>
PK_DEV void norm_put(const NormArgs<TYPE> &a, uint64_t row, uint32_t b, uint32_t n, const double (&p)[4], double root,
                     uint64_t top, double factor) {
    const uint32_t lane = threadIdx.x & 63u, c0 = 256u * b + 4u * lane;
    if (a.y) {
        typename Elem<TYPE>::raw w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = Elem<TYPE>::down((float)(p[j] * root));
        store_row4<TYPE>(a.y + row * a.dim + c0, n, w);
    }
    if (!a.q) return;
    int32_t sum;
    const uint32_t packed = codes4(p, factor, sum);
    if (a.format == PULSAR_ROWS_Q8_K) {
        uint8_t *ob = a.q + (row * ((a.dim + 255u) / 256u) + b) * 292u;
        sum = group_sum<4>(sum);
        __builtin_memcpy(ob + 4u + 4u * lane, &packed, 4);
        if ((lane & 3u) == 0u) {
            const int16_t s16 = (int16_t)sum;
            __builtin_memcpy(ob + 260u + 2u * (lane >> 2), &s16, 2);
        }
        if (lane == 0u) {
            const float d = (float)(__builtin_bit_cast(double, top) * root * (1.0 / 127.0));
            __builtin_memcpy(ob, &d, 4);
        }
    } else {
        store_codes(a.q + row * a.q_stride + c0, n, packed);
    }
}

// How many of the 4 values from c0 on are in the row
PK_DEV uint32_t inside(uint32_t c0, uint32_t dim) { return c0 < dim ? (dim - c0 < 4u ? dim - c0 : 4u) : 0u; }

template <uint32_t TYPE, uint32_t NB>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs<TYPE> a) {
    __shared__ RowStats lds;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_chunk = (a.dim + 255u) / 256u;
    const uint64_t row = blockIdx.x;
    double p[NB][4], ss = 0.0;
    uint64_t top[NB];
    float s[NB][4];
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        const uint32_t b = wave + waves * j, c0 = 256u * b + 4u * lane;
        norm_load<TYPE>(a, a.x + row * a.x_stride + c0, a.residual + row * a.res_stride + c0, inside(c0, a.dim), s[j]);
    }
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        const uint32_t b = wave + waves * j, c0 = 256u * b + 4u * lane, n = inside(c0, a.dim);
        if (a.sum) norm_put_sum<TYPE>(a.sum + row * a.sum_stride + c0, n, s[j]);
        float g[4];
        load_row4<PULSAR_TYPE_F32>(a.gain + c0, n, g);
        top[j] = 0u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double v = s[j][k];
            ss = __builtin_fma(v, v, ss);
            p[j][k] = v * (double)g[k];
            top[j] = max_bits(top[j], size_bits(p[j][k]));
        }
    }
    uint64_t row_top = 0u;
    if (a.format == PULSAR_ROWS_Q8_K) {
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) top[j] = wave_max64(top[j]);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) row_top = max_bits(row_top, top[j]);
        row_top = wave_max64(row_top);
    }
    ss = wave_sum64(ss);
    block_stats(lds, ss, row_top);
    const double root = norm_root(ss, a.dim, a.eps);
    const double row_factor = code_factor(__builtin_bit_cast(double, row_top));
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        const uint32_t b = wave + waves * j, c0 = 256u * b + 4u * lane;
        if (b >= n_chunk) break;  // wave-uniform
        const bool blocks = a.format == PULSAR_ROWS_Q8_K;
        norm_put<TYPE>(a, row, b, inside(c0, a.dim), p[j], root, blocks ? top[j] : row_top,
                       blocks ? code_factor(__builtin_bit_cast(double, top[j])) : row_factor);
    }
    if (a.scales && threadIdx.x == 0u)
        a.scales[row] = (float)(__builtin_bit_cast(double, row_top) * root * (1.0 / 127.0));
}

// Rows of more values than a block holds: read twice, the second time from sum where it
// is written (x and residual may be gone by then)
template <uint32_t TYPE>
__global__ __launch_bounds__(1024) void norm_long_kernel(NormArgs<TYPE> a) {
    __shared__ RowStats lds;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_chunk = (a.dim + 255u) / 256u;
    const uint64_t row = blockIdx.x;
    const typename Elem<TYPE>::raw *x = a.x + row * a.x_stride, *res = a.residual + row * a.res_stride;
    double ss = 0.0;
    uint64_t row_top = 0u;
    for (uint32_t b = wave; b < n_chunk; b += waves) {
        const uint32_t c0 = 256u * b + 4u * lane, n = inside(c0, a.dim);
        float s[4], g[4];
        norm_load<TYPE>(a, x + c0, res + c0, n, s);
        if (a.sum) norm_put_sum<TYPE>(a.sum + row * a.sum_stride + c0, n, s);
        load_row4<PULSAR_TYPE_F32>(a.gain + c0, n, g);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const double v = s[k];
            ss = __builtin_fma(v, v, ss);
            row_top = max_bits(row_top, size_bits(v * (double)g[k]));
        }
    }
    ss = wave_sum64(ss);
    row_top = wave_max64(row_top);
    block_stats(lds, ss, row_top);
    const double root = norm_root(ss, a.dim, a.eps);
    const double row_factor = code_factor(__builtin_bit_cast(double, row_top));
    for (uint32_t b = wave; b < n_chunk; b += waves) {
        const uint32_t c0 = 256u * b + 4u * lane, n = inside(c0, a.dim);
        float s[4], g[4];
        if (a.sum)
            load_row4<TYPE>(a.sum + row * a.sum_stride + c0, n, s);  // this lane's own stores
        else
            norm_load<TYPE>(a, x + c0, res + c0, n, s);
        load_row4<PULSAR_TYPE_F32>(a.gain + c0, n, g);
        double p[4];
        uint64_t top = 0u;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            p[k] = (double)s[k] * (double)g[k];
            top = max_bits(top, size_bits(p[k]));
        }
        const bool blocks = a.format == PULSAR_ROWS_Q8_K;
        top = blocks ? wave_max64(top) : row_top;
        norm_put<TYPE>(a, row, b, n, p, root, top,
                       blocks ? code_factor(__builtin_bit_cast(double, top)) : row_factor);
    }
    if (a.scales && threadIdx.x == 0u)
        a.scales[row] = (float)(__builtin_bit_cast(double, row_top) * root * (1.0 / 127.0));
}

// ------------------------------------------------------------- quantizer --

// 1 / (1 + e^-z) in 64 bits, within some units in the last place. With E = e^-|z| in
// (0, 1] it is E^(z < 0) / (1 + E), where nothing overflows. e^-|z| = 2^n e^r, r within
// ln 2 / 2 (ln 2 in two parts), by the series to r^12 (what is left: 2^-52); the
// reciprocal of 1 .. 2 from the instruction's 2^-24 in two Newton steps.
PK_DEV double sigmoid64(double z) {
    const double x = __builtin_fmax(-__builtin_fabs(z), -800.0);  // E is 0 from -745 on
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0.6931471805599453, x);  // ln 2 rounded, and what is left of it
    r = __builtin_fma(n, -2.3190468138462996e-17, r);
    double e = 1.0 / 479001600.0;
    constexpr double c[] = {1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                            1.0 / 120.0,      1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
#pragma unroll
    for (int k = 0; k < 12; k++) e = __builtin_fma(e, r, c[k]);
    e = __builtin_ldexp(e, (int)n);
    const double d = 1.0 + e;
    double y = __builtin_amdgcn_rcp(d);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    y = __builtin_fma(__builtin_fma(-d, y, 1.0), y, y);
    return (z < 0.0 ? e : 1.0) * y;
}
// The gated combine of pk::glu in 64 bits
PK_DEV double glu64(float g, float u, uint32_t op) {
    double v = g, w = u;
    if (op == PULSAR_ACT_SWIGLU_OAI) {
        v = v > 7.0 ? 7.0 : v;  // NaN stays
        w = (w > 7.0 ? 7.0 : w < -7.0 ? -7.0 : w) + 1.0;
        return v * sigmoid64(1.702 * v) * w;
    }
    return v * sigmoid64(v) * w;
}

template <uint32_t TYPE>
struct QuantArgs {
    typedef typename Elem<TYPE>::raw raw;
    uint8_t *q;
    float *scales;
    const raw *x, *up;  // up NULL: x as it is
    uint64_t x_stride, up_stride, q_stride;
    uint32_t dim, act_op;
};

template <uint32_t TYPE>
PK_DEV void quant_values(const QuantArgs<TYPE> &a, const typename Elem<TYPE>::raw *x,
                         const typename Elem<TYPE>::raw *up, uint32_t n, double (&v)[4]) {
    float g[4], u[4];
    load_row4<TYPE>(x, n, g);
    if (a.up) {
        load_row4<TYPE>(up, n, u);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = glu64(g[k], u[k], a.act_op);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = g[k];
    }
}

template <uint32_t TYPE, uint32_t NB>
__global__ __launch_bounds__(1024) void quantize_i8_kernel(QuantArgs<TYPE> a) {
    __shared__ RowStats lds;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t row = blockIdx.x;
    double v[NB][4], none = 0.0;
    uint64_t top = 0u;
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        const uint32_t c0 = 256u * (wave + waves * j) + 4u * lane;
        quant_values<TYPE>(a, a.x + row * a.x_stride + c0, a.up + row * a.up_stride + c0, inside(c0, a.dim), v[j]);
#pragma unroll
        for (int k = 0; k < 4; k++) top = max_bits(top, size_bits(v[j][k]));
    }
    top = wave_max64(top);
    block_stats(lds, none, top);
    const double largest = __builtin_bit_cast(double, top), factor = code_factor(largest);
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
        const uint32_t c0 = 256u * (wave + waves * j) + 4u * lane;
        int32_t sum;
        store_codes(a.q + row * a.q_stride + c0, inside(c0, a.dim), codes4(v[j], factor, sum));
    }
    if (threadIdx.x == 0u) a.scales[row] = (float)(largest * (1.0 / 127.0));
}

// Rows of more values than a block holds: read and combined twice
template <uint32_t TYPE>
__global__ __launch_bounds__(1024) void quantize_i8_long_kernel(QuantArgs<TYPE> a) {
    __shared__ RowStats lds;
    const uint32_t waves = blockDim.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n_chunk = (a.dim + 255u) / 256u;
    const uint64_t row = blockIdx.x;
    const typename Elem<TYPE>::raw *x = a.x + row * a.x_stride, *up = a.up + row * a.up_stride;
    double v[4], none = 0.0;
    uint64_t top = 0u;
    for (uint32_t b = wave; b < n_chunk; b += waves) {
        const uint32_t c0 = 256u * b + 4u * lane;
        quant_values<TYPE>(a, x + c0, up + c0, inside(c0, a.dim), v);
#pragma unroll
        for (int k = 0; k < 4; k++) top = max_bits(top, size_bits(v[k]));
    }
    top = wave_max64(top);
    block_stats(lds, none, top);
    const double largest = __builtin_bit_cast(double, top), factor = code_factor(largest);
    for (uint32_t b = wave; b < n_chunk; b += waves) {
        const uint32_t c0 = 256u * b + 4u * lane, n = inside(c0, a.dim);
        quant_values<TYPE>(a, x + c0, up + c0, n, v);
        int32_t sum;
        store_codes(a.q + row * a.q_stride + c0, n, codes4(v, factor, sum));
    }
    if (threadIdx.x == 0u) a.scales[row] = (float)(largest * (1.0 / 127.0));
}

// ---------------------------------------------------------------- launch --

// Waves and chunks of a wave for rows of n_chunk chunks; 0: the row is too long
struct RowShape {
    uint32_t waves, chunks;
};
static RowShape row_shape(uint32_t n_chunk) {
    for (uint32_t nb = 1; nb <= 4u; nb <<= 1)
        if (n_chunk <= 16u * nb) return {(n_chunk + nb - 1u) / nb, nb};
    return {16u, 0u};
}

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
                              dim, format, eps};
    const RowShape s = row_shape((dim + 255u) / 256u);
    const dim3 grid(n_rows), block(64u * s.waves);
    switch (s.chunks) {
    case 1: hipLaunchKernelGGL((norm_kernel<TYPE, 1>), grid, block, 0, pk::stream(), a); break;
    case 2: hipLaunchKernelGGL((norm_kernel<TYPE, 2>), grid, block, 0, pk::stream(), a); break;
    case 4: hipLaunchKernelGGL((norm_kernel<TYPE, 4>), grid, block, 0, pk::stream(), a); break;
    default: hipLaunchKernelGGL((norm_long_kernel<TYPE>), grid, block, 0, pk::stream(), a);
    }
    return launch_ok("rms_norm_q8 launch");
}

template <uint32_t TYPE>
static int launch_quantize(void *q, void *scales, const void *x, const void *up, uint32_t dim, uint32_t n_rows,
                           uint32_t act_op, uint64_t x_stride, uint64_t up_stride, uint64_t q_stride) {
    typedef typename Elem<TYPE>::raw raw;
    const QuantArgs<TYPE> a = {(uint8_t *)q, (float *)scales, (const raw *)x, (const raw *)up, x_stride, up_stride,
                               q_stride, dim, act_op};
    const RowShape s = row_shape((dim + 255u) / 256u);
    const dim3 grid(n_rows), block(64u * s.waves);
    switch (s.chunks) {
    case 1: hipLaunchKernelGGL((quantize_i8_kernel<TYPE, 1>), grid, block, 0, pk::stream(), a); break;
    case 2: hipLaunchKernelGGL((quantize_i8_kernel<TYPE, 2>), grid, block, 0, pk::stream(), a); break;
    case 4: hipLaunchKernelGGL((quantize_i8_kernel<TYPE, 4>), grid, block, 0, pk::stream(), a); break;
    default: hipLaunchKernelGGL((quantize_i8_long_kernel<TYPE>), grid, block, 0, pk::stream(), a);
    }
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
