// pk_elem.h - rows of f32, f16 or bf16 values (PULSAR_TYPE_*), four values at a time.
#pragma once

#include "pk_common.h"

namespace pk {

template <uint32_t TYPE>
struct Elem;

template <>
struct Elem<PULSAR_TYPE_F32> {
    typedef float raw;
    PK_DEV static float up(raw v) { return v; }
    PK_DEV static raw down(float v) { return v; }
};
template <>
struct Elem<PULSAR_TYPE_F16> {
    typedef _Float16 raw;
    PK_DEV static float up(raw v) { return (float)v; }
    PK_DEV static raw down(float v) { return (raw)v; }  // to the nearest, ties to even
};
template <>
struct Elem<PULSAR_TYPE_BF16> {
    typedef __bf16 raw;
    PK_DEV static float up(raw v) { return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16); }
    PK_DEV static raw down(float v) { return (raw)v; }  // to the nearest, ties to even
};

static inline uint32_t elem_bytes(uint32_t type) { return type == PULSAR_TYPE_F32 ? 4u : 2u; }

// Values p[0 .. V - 1], of which the first n (V and more: all, one load) are there; 0 for
// the others. Rows may start at any element: global loads and stores take any alignment.
// Single values are volatile so that the compiler leaves them apart from the whole: where
// it joins the last of either in one store, lanes that write all of them write one twice
// (seen behind a branch that is uniform on one side).
template <uint32_t TYPE, uint32_t V>
PK_DEV void load_row(const typename Elem<TYPE>::raw *p, uint32_t n, float (&v)[V]) {
    typedef typename Elem<TYPE>::raw raw;
    raw w[V] = {};
    if (n >= V)
        __builtin_memcpy(w, p, sizeof(w));
    else {
#pragma unroll
        for (uint32_t j = 0; j + 1u < V; j++)
            if (j < n) w[j] = *(const volatile PK_GLOBAL raw *)(p + j);
    }
#pragma unroll
    for (uint32_t j = 0; j < V; j++) v[j] = Elem<TYPE>::up(w[j]);
}
template <typename raw, uint32_t V>
PK_DEV void store_row(raw *p, uint32_t n, const raw (&w)[V]) {
    if (n >= V)
        __builtin_memcpy(p, w, sizeof(w));
    else {
#pragma unroll
        for (uint32_t j = 0; j + 1u < V; j++)
            if (j < n) *(volatile PK_GLOBAL raw *)(p + j) = w[j];
    }
}
template <uint32_t TYPE>
PK_DEV void load_row4(const typename Elem<TYPE>::raw *p, uint32_t n, float (&v)[4]) {
    load_row<TYPE, 4>(p, n, v);
}
template <uint32_t TYPE>
PK_DEV void store_row4(typename Elem<TYPE>::raw *p, uint32_t n, const typename Elem<TYPE>::raw (&w)[4]) {
    store_row(p, n, w);
}

// ------------------------------------------------- 8-bit codes of 64-bit values --
// Sizes |v| in the order of their bits: a NaN is above infinity, so the largest of a
// row that holds one is a NaN, and so is the row's scale.
PK_DEV uint64_t size_bits(double v) { return __builtin_bit_cast(uint64_t, v) & 0x7fffffffffffffffull; }
PK_DEV uint64_t max_bits(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <typename F>
PK_DEV uint64_t wave_step64(uint64_t v, F &&lane32) {
    return (uint64_t)(uint32_t)lane32((int32_t)(v >> 32)) << 32 | (uint32_t)lane32((int32_t)v);
}
PK_DEV uint64_t partner64(uint64_t v, uint32_t s) {
    return wave_step64(v, [&](int32_t w) { return partner(w, s); });
}
// Largest of aligned groups of G lanes, in every lane
template <uint32_t G>
PK_DEV uint64_t group_max64(uint64_t v) {
#pragma unroll
    for (uint32_t s = 1; s < G; s <<= 1) v = max_bits(v, partner64(v, s));
    return v;
}
PK_DEV double wave_sum64(double v) {
#pragma unroll
    for (uint32_t s = 1; s < 64; s <<= 1)
        v += __builtin_bit_cast(double, partner64(__builtin_bit_cast(uint64_t, v), s));
    return v;
}

// 127 / largest, 0 where the largest is 0 (every code is 0 then; infinity and NaN
// give 0 and NaN, and NaN converts to 0)
PK_DEV double code_factor(double largest) { return largest > 0.0 || largest != largest ? 127.0 / largest : 0.0; }
// The integer nearest to v * factor, halves away from 0. What is nearer to a half
// than 2^-40 counts as on it: the product's own rounding is below 2^-44, so a value
// of exactly half the largest is decided alike whatever the rounding of 127 / largest
PK_DEV int32_t code_of(double v, double factor) {
    const double t = v * factor;
    return (int32_t)(t + __builtin_copysign(0.5 + 0x1p-40, t));
}

}  // namespace pk
