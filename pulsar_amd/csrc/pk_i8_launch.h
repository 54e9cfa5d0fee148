// pk_i8_launch.h - which kernel takes a product of int8 rows: the lane kernel for one or
// two tokens, else a tile of pk_i8_tile.h.
#pragma once

#include "pk_i8_tile.h"

namespace pk {

// A wave is one channel and T tokens: lane l takes 16 bytes of each 1024 of the row, four
// dot instructions a token, two pieces of the row on their way at once (with one and four
// it is as fast or 3% slower).
template <uint32_t TYPE, uint32_t T>
__global__ __launch_bounds__(256) void i8_lane_kernel(I8Args a) {
    const uint32_t lane = threadIdx.x & 63u, r = block_index() * 4u + (threadIdx.x >> 6);
    if (r >= a.out_dim) return;  // wave-uniform
    const uint8_t *w = a.w + r * a.w_stride;
    int32_t acc[T] = {};
    auto dot = [&](uint32_t t, uint4 wv, uint32_t k) { acc[t] = dot16(wv, ldw128(a.x + t * a.x_stride + k), acc[t]); };
    uint32_t k = 16u * lane;
    for (uint32_t n = a.in_dim / 2048u; n > 0u; n--, k += 2048u) {
        const uint4 w0 = ldw128(w + k), w1 = ldw128(w + k + 1024u);
#pragma unroll
        for (uint32_t t = 0; t < T; t++) {
            dot(t, w0, k);
            dot(t, w1, k + 1024u);
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < 2u; j++, k += 1024u)
        if (k + 16u <= a.in_dim) {
            const uint4 wv = ldw128(w + k);
#pragma unroll
            for (uint32_t t = 0; t < T; t++) dot(t, wv, k);
        }
    const uint32_t last = (a.in_dim & ~15u) + lane;  // a byte a lane behind the last whole piece
    if (last < a.in_dim) {
#pragma unroll
        for (uint32_t t = 0; t < T; t++)
            acc[t] += (int32_t)(int8_t)ldw8(w + last) * (int32_t)(int8_t)ldw8(a.x + t * a.x_stride + last);
    }
#pragma unroll
    for (uint32_t t = 0; t < T; t++) {
        acc[t] = group_sum<64>(acc[t]);
        if (lane == t) i8_put<TYPE>(a, t, r, acc[t]);
    }
}
template <uint32_t TYPE, uint32_t T>
static int launch_i8_lane(const I8Args &a) {
    hipLaunchKernelGGL((i8_lane_kernel<TYPE, T>), grid_of((a.out_dim + 3u) / 4u), dim3(256), 0, pk::stream(), a);
    return launch_ok("matmul_i8 launch");
}

// One block a CU: where a shape's tiles are no more than this, all are in flight at once
constexpr uint64_t kI8Slots = 256;

template <uint32_t TYPE>
int launch_i8(const I8Args &a) {
    // All times here: bf16 rows out, no epilogue, weights from HBM, calls one behind the other
    // in a replayed graph, both sides in turn.
    // The lane kernel has no start and end to pay for; a matrix-core tile has room for more
    // tokens (4096 x 4096, lane / tile: 1 token 5.1 / 5.8 us, 2 tokens 5.5 / 5.9, 4 tokens
    // 6.3 / 6.0; 1024 x 1024, 2 tokens 2.6 / 3.4). The border is not the best one everywhere: with
    // few channels a third token is still faster there (384 x 10400 5.2 / 6.4), with many short ones
    // the second no more (23840 x 1744 13.1 / 10.6, 21424 x 3328 17.8 / 15.6)
    if (a.n_tok == 1u) return launch_i8_lane<TYPE, 1>(a);
    if (a.n_tok == 2u) return launch_i8_lane<TYPE, 2>(a);
    // The finest tile whose blocks are all in flight at once, else the widest: a block's
    // time grows with its tokens and channels, and a tile's reads for each product fall
    // with them. Of 411 shapes (1 to 8192 tokens, 64 to 28672 rows and 64 to 16384 columns)
    // the rule as it stands here misses the fastest of 11 tiles by 1.0% on average, by more than
    // 10% in 12; with lane kernels of up to 4 tokens among the choices by 1.3%, in 18. Of 193
    // shapes of rows at any byte and 8 tiles 1.2%, 7; with lane kernels 2.5%, 15.
    // us of 32 x 32, 32 x 64, 64 x 64, 64 x 128, 128 x 128, 128 x 256, 256 x 256, 4096 channels,
    // 4096 values: 16 tokens 6.4 / 7.1 / 9.1 / 11.0 / 14 / 22 / 46 (16 x 16: 6.0); 256 tokens 20 /
    // 13.5 / 10.4 / 12.0 / 14.8 / 22 / 47; 1024 tokens 32 x 64 on 49 / 31 / 26 / 23 / 26 / 48; 4096
    // tokens of 14336 values 64 x 128 on 364 / 263 / 216 / 204
#define PK_I8_TRY(...)                                    \
    do {                                                  \
        using T = I8Tile<__VA_ARGS__>;                    \
        if (i8_items<T>(a) <= kI8Slots) return launch_i8_tile<TYPE, T>(a); \
    } while (0)
    const bool whole = (((uintptr_t)a.x | (uintptr_t)a.w | a.x_stride | a.w_stride | a.in_dim) & 15u) == 0u;
    // 8 groups of the finest tile split K: below 8 steps some of them have none, and a
    // wider tile takes as long
    const bool split = a.in_dim > 7u * 128u;
    if (!whole) {
        // rows at any byte: the words of a step go through registers, which costs 1.4 to
        // 1.8 times the time (16 tokens 4095 x 4090 against 4096 x 4096: 8.6 / 6.0 us; 130 tokens
        // 5001 x 2047 / 5008 x 2048: 10.0 / 6.9; 1023 tokens 4095 x 4090 / 4096 x 4096: 34 / 23;
        // 4095 tokens 126 / 69). Two groups of 32 x 32, and 16 waves for one round of tiles of
        // 128 x 128, 8 for more (40 tokens 2881 x 2049 6.9 us, 4 groups 8.3; 1023 tokens 4095 x
        // 4090 34, 8 waves 45; 4095 tokens 126, 16 waves 148). Up to 64 tokens rounds of 64 x
        // 128, not of 128 x 128 (8 tokens 151935 x 4095 139 / 160; 64 tokens 60001 x 2047 42 / 43)
        if (split) PK_I8_TRY(16, 16, 16, 1, 1, 8, 128, 2, false);
        PK_I8_TRY(16, 32, 32, 2, 2, 2, 128, 4, false);
        PK_I8_TRY(16, 32, 64, 2, 2, 2, 128, 4, false);
        PK_I8_TRY(16, 64, 64, 2, 4, 1, 128, 4, false);
        using Wide = I8Tile<16, 64, 128, 2, 4, 1, 128, 4, false>;
        if (i8_items<Wide>(a) <= kI8Slots || a.n_tok <= 64u) return launch_i8_tile<TYPE, Wide>(a);
        PK_I8_TRY(16, 128, 128, 4, 4, 1, 128, 4, false);
        return launch_i8_tile<TYPE, I8Tile<32, 128, 128, 4, 2, 1, 128, 2, false>>(a);
    }
    if (split) PK_I8_TRY(16, 16, 16, 1, 1, 8, 128, 4, true);
    // two of 32 x 32: of long rows four groups take a part each (4096 channels, 48 tokens of
    // 4096 values 6.7 against 8.6 us), for short ones joining them costs more (992: 4.5 / 4.3)
    if (a.in_dim > 1024u)
        PK_I8_TRY(16, 32, 32, 2, 1, 4, 128, 4, true);
    else
        PK_I8_TRY(16, 32, 32, 2, 2, 1, 128, 4, true);
    PK_I8_TRY(16, 32, 64, 2, 2, 2, 128, 4, true);
    // many channels of few tokens: rounds of a tile without room for many more tokens (16
    // tokens of 4096 values, 151936 channels 129 us, 128 x 256 151; 64 tokens 139 / 159)
    if (a.n_tok <= 32u) return launch_i8_tile<TYPE, I8Tile<16, 32, 32, 2, 2, 1, 128, 4, true>>(a);
    // 64 x 64, one round: two groups for rows of more than 2048 values (4096 channels of 4096, 192
    // tokens 9.3 us against 9.9, 256 tokens 10.3 / 10.4, of 14336 36 / 38; of 992 6.0 / 5.6)
    if (a.in_dim > 2048u) PK_I8_TRY(32, 64, 64, 2, 2, 2, 128, 4, true);
    using Square = I8Tile<32, 64, 64, 2, 2, 1, 128, 4, true>;
    if (i8_items<Square>(a) <= kI8Slots) return launch_i8_tile<TYPE, Square>(a);
    PK_I8_TRY(16, 64, 128, 2, 4, 1, 128, 4, true);
    if (a.n_tok <= 64u) return launch_i8_tile<TYPE, Square>(a);
    PK_I8_TRY(16, 128, 128, 4, 2, 1, 128, 4, true);
    using Half = I8Tile<32, 128, 256, 2, 4, 1, 128, 3, true>;
    using Widest = I8Tile<16, 256, 256, 2, 4, 1, 64, 4, true>;
    // past that, rounds of blocks count, a round of the half tile being 0.55 of one of the
    // widest (28672 x 4096, 768 tokens: 3 rounds 104 us, 2 rounds 122)
    auto rounds = [](uint64_t items) { return (items + kI8Slots - 1u) / kI8Slots; };
    if (rounds(i8_items<Half>(a)) * 11u < rounds(i8_items<Widest>(a)) * 20u) return launch_i8_tile<TYPE, Half>(a);
    return launch_i8_tile<TYPE, Widest>(a);
#undef PK_I8_TRY
}

}  // namespace pk
