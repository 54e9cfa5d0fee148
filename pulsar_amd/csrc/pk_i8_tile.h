// pk_i8_tile.h - the matrix-core tile of pulsar_matmul_i8: BM tokens x BN channels, sums
// exact in int32 on v_mfma_i32_32x32x32_i8 or 16x16x64.
//
// Operands are 16 bytes a lane, lane l the row l % MF and the l / MF-th 16 bytes of the
// step, of tokens (A) and channels (B) alike; D has channel l % MF in lane l. Both come
// through LDS in steps of 128 values: 16-byte piece c of row r lies in slot c ^ r / 2 % 8.
// A cycle serves 16 lanes, 0-3, 12-15 and 20-27 or 4-11, 16-19 and 28-31 and the same 32
// on, from 64 banks, two rows wide: their pairs of r % 2 and slot all differ (with slot
// c ^ r % 8 half of the LDS time of 32 x 32 was conflicts), and 8 lanes copy a row's 128
// bytes in one piece. S steps are on their way at once. A step's last operands are
// read before its wait, so the wait, the barrier and the next step's first reads are
// behind MFMAs that need nothing of them.
//
// WM x WN waves share a step's tokens and channels; WK such groups split the steps among
// them, for sizes whose tiles would leave much of the chip idle, and add their sums in
// LDS at the end.
//
// Measured: 4096 tokens through 4096 x 14336, bias and residual, bf16, 209 us, 2300 T
// operations a second; 8192 tokens of 8192 x 8192 457 us, 2400. What bounds them is power:
// with random bytes the card runs at 1.76 GHz, with zeros at 2.46 and takes 168 of the 200 us
// without an epilogue; the MFMAs alone, their operands in registers, reach 3500 to 4000 T on random
// bytes. Start and end of a block take some 10 us. 16 tokens of 8192 x 4096 read 34 MB in 8.4
// us, 4.1 TB/s: a launch and HBM.
#pragma once

#include "pk_i8.h"

namespace pk {

typedef int32_t i8v4 __attribute__((ext_vector_type(4)));
typedef int32_t i8v16 __attribute__((ext_vector_type(16)));

template <uint32_t MF>
struct I8Mfma;
template <>
struct I8Mfma<32> {
    typedef i8v16 acc;
    static constexpr uint32_t kElem = 16;
    PK_DEV static acc run(uint4 a, uint4 b, acc c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i8v4, a), __builtin_bit_cast(i8v4, b), c, 0, 0, 0);
    }
    // token of element e
    PK_DEV static uint32_t token(uint32_t e, uint32_t lane) { return 8u * (e >> 2) + 4u * (lane >> 5) + (e & 3u); }
};
template <>
struct I8Mfma<16> {
    typedef i8v4 acc;
    static constexpr uint32_t kElem = 4;
    PK_DEV static acc run(uint4 a, uint4 b, acc c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i8v4, a), __builtin_bit_cast(i8v4, b), c, 0, 0, 0);
    }
    PK_DEV static uint32_t token(uint32_t e, uint32_t lane) { return 4u * (lane >> 4) + e; }
};

// DMA: rows of x and w on 16-byte boundaries, of whole 16-byte pieces, copied to LDS
// without a register; else through registers, rows at any byte and of any length
template <uint32_t MF_, uint32_t BM_, uint32_t BN_, uint32_t WM_, uint32_t WN_, uint32_t WK_, uint32_t KB_, uint32_t S_, bool DMA_>
struct I8Tile {
    static constexpr uint32_t MF = MF_, BM = BM_, BN = BN_, WM = WM_, WN = WN_, WK = WK_, KB = KB_, S = S_;
    static constexpr bool DMA = DMA_;
    static constexpr uint32_t kGroup = WM * WN, kWaves = kGroup * WK, kThreads = 64u * kWaves;
    static constexpr uint32_t kStage = (BM + BN) * KB;               // bytes of a group's step
    static constexpr uint32_t kRows = 1024u / KB, kX = BM / kRows / kGroup, kW = BN / kRows / kGroup;  // a wave's copies
    static constexpr uint32_t MT = BM / WM / MF, NT = BN / WN / MF, kCols = NT * MF;
    static constexpr uint32_t kSub = KB * MF / 1024u;                // K slices of a step, of 32 (MF 32) or 64 (MF 16)
    // tokens whose sums a wave's share of a step's buffer holds at once
    static constexpr uint32_t kRoom = kStage / kGroup / (kCols * 4u);
    static constexpr uint32_t kSliceTok = kRoom >= MF ? MF : kRoom >= MF / 2u ? MF / 2u : MF / 4u;
    static_assert(MF == 32u || kSliceTok == MF, "16 tokens are in every element");
    static constexpr uint32_t kSlice = kSliceTok * kCols * 4u;
    static_assert(kX * kRows * kGroup == BM && kW * kRows * kGroup == BN, "whole copies");
    static_assert(S * kSub % 2u == 0u, "the operands' two places in turn");
    static_assert(kSlice <= kStage / kGroup, "a wave's sums fit its share of a step's buffer");
    static_assert(DMA ? S >= 3u && S <= 5u : S % 2u == 0u, "a copy has S - 2 steps to land, or S in registers");
    static constexpr uint32_t kBuffers = DMA ? S : 2u;  // in LDS
    static_assert((S - 1u) * (kX + kW) <= 63u, "the counter of loads");
};

// The slot of piece 0 of a row in LDS; piece c lies in slot c ^ this
template <uint32_t KB>
PK_DEV uint32_t i8_slot_of(uint32_t row) {
    static_assert(KB == 64u || KB == 128u, "bytes of a row in a step");
    return KB == 128u ? row >> 1 & 7u : 0x78u >> 2u * (row >> 2 & 3u) & 3u;
}

// 16 of 20 bytes, from byte n < 4 on
PK_DEV uint4 shifted(uint4 lo, uint32_t hi, uint32_t n) {
    return make_uint4(__builtin_amdgcn_alignbyte(lo.y, lo.x, n), __builtin_amdgcn_alignbyte(lo.z, lo.y, n),
                      __builtin_amdgcn_alignbyte(lo.w, lo.z, n), __builtin_amdgcn_alignbyte(hi, lo.w, n));
}
// the first n bytes, 0 for the others
PK_DEV uint4 first_bytes(uint4 v, uint32_t n) {
    auto keep = [&](uint32_t w, uint32_t i) { return n >= i + 4u ? w : n <= i ? 0u : w & ((1u << 8u * (n - i)) - 1u); };
    return make_uint4(keep(v.x, 0u), keep(v.y, 4u), keep(v.z, 8u), keep(v.w, 12u));
}

PK_DEV void wait_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); }
template <uint32_t N>
PK_DEV void wait_loads_lds() {  // at most N loads of the wave are on their way, no LDS read
    __builtin_amdgcn_s_waitcnt((N & 15u) | (N >> 4) << 14 | 7u << 4);
}

// 16 bytes a lane of a buffer, from byte `offset` on, to LDS from `to` on (uniform; lane
// l's to to + 16 l); 0 where they are behind the buffer's end. As the builtin does, but that
// the compiler waits for a copy into one array ahead of reads of another there: these
// copies are waited for by wait_loads_lds, and every read is ordered behind them by it.
typedef uint32_t rsrc_t __attribute__((ext_vector_type(4)));
PK_DEV rsrc_t buffer_of(const uint8_t *base, uint32_t bytes) {
    const uint64_t at = (uint64_t)(uintptr_t)base;
    return rsrc_t{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, bytes, 0x00027000u};
}
PK_DEV uint32_t lds_address(uint8_t *p) { return (uint32_t)(uintptr_t)(PK_LDS uint8_t *)p; }
PK_DEV void copy_to_lds(rsrc_t from, uint32_t offset, uint32_t to) {
    // The instruction takes the address from m0. The compiler reserves that register and
    // refuses it as a clobber; so that none of its own uses gets an asm between its write and
    // its read, these kernels must have none (tests/test_tile_assembly.py; to put m0 back
    // behind each copy took 1.3% at 4096 tokens through 4096 x 14336)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(to), "v"(offset), "s"(from)
                 : "memory");
}

template <uint32_t TYPE, typename T>
__global__ __launch_bounds__(T::kThreads) void i8_tile_kernel(I8Args a, uint32_t n_tt, uint32_t n_rt, uint32_t n_item) {
    using M = I8Mfma<T::MF>;
    constexpr uint32_t S = T::S, kBuf = T::WK * T::kStage;
    __shared__ __align__(16) uint8_t buf0[kBuf];
    __shared__ __align__(16) uint8_t buf1[kBuf];
    __shared__ __align__(16) uint8_t buf2[T::kBuffers > 2u ? kBuf : 16u];
    __shared__ __align__(16) uint8_t buf3[T::kBuffers > 3u ? kBuf : 16u];
    __shared__ __align__(16) uint8_t buf4[T::kBuffers > 4u ? kBuf : 16u];
    auto buf_of = [&](uint32_t s) { return s == 0u ? buf0 : s == 1u ? buf1 : s == 2u ? buf2 : s == 3u ? buf3 : buf4; };
    auto address_of = [&](uint32_t s) {
        return s == 0u   ? lds_address(buf0)
               : s == 1u ? lds_address(buf1)
               : s == 2u ? lds_address(buf2)
               : s == 3u ? lds_address(buf3)
                         : lds_address(buf4);
    };
    // XCD x (blocks x, x + 8, ...) takes the x-th eighth of the items; 4 channel tiles by
    // all token tiles are one run of them, channels first: what an XCD works on at a time
    // is about as many tokens as channels
    const uint32_t block = block_index(), item = (block & 7u) * (gridDim.x * gridDim.y >> 3) + (block >> 3);
    if (item >= n_item) return;  // block-uniform
    const uint32_t panel = item / (4u * n_tt), in_panel = item - panel * 4u * n_tt;
    const uint32_t width = n_rt - 4u * panel < 4u ? n_rt - 4u * panel : 4u;
    const uint32_t t0 = in_panel / width * T::BM, r0 = (4u * panel + in_panel % width) * T::BN;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t group = wave / T::kGroup, in_group = wave % T::kGroup;
    const uint32_t wm = in_group / T::WN, wn = in_group % T::WN;

    // ------------------------------------------------------------ copies --
    const uint32_t nx = a.n_tok - t0 < T::BM ? a.n_tok - t0 : T::BM, nw = a.out_dim - r0 < T::BN ? a.out_dim - r0 : T::BN;
    const uint8_t *xb = a.x + t0 * a.x_stride, *wb = a.w + r0 * a.w_stride;
    const uint32_t xs = (uint32_t)a.x_stride, ws = (uint32_t)a.w_stride;  // at most 2^23: offsets of a tile fit 32 bits
    const uint32_t x_bytes = (nx - 1u) * xs + a.in_dim, w_bytes = (nw - 1u) * ws + a.in_dim;
    // the byte of a step that the lane copies of the row of copy j: with DMA, whose lanes
    // land side by side, of the piece that belongs there; else a row's pieces in order
    constexpr uint32_t kPieces = T::KB / 16u;
    auto slot_of = [&](uint32_t j) { return i8_slot_of<T::KB>(T::kRows * (in_group + T::kGroup * j) + lane / kPieces); };
    auto piece_of = [&](uint32_t j) { return 16u * ((lane % kPieces) ^ (T::DMA ? slot_of(j) : 0u)); };
    // a copy's row; without bounds of their own (!DMA) rows behind the last are the last
    auto row_of = [&](uint32_t j, uint32_t n) {
        const uint32_t row = T::kRows * (in_group + T::kGroup * j) + lane / kPieces;
        return T::DMA || row < n ? row : n - 1u;
    };
    constexpr uint32_t kCopies = T::kX + T::kW;
    uint32_t from[kCopies];
#pragma unroll
    for (uint32_t j = 0; j < kCopies; j++)
        from[j] = j < T::kX ? row_of(j, nx) * xs + piece_of(j) : row_of(j - T::kX, nw) * ws + piece_of(j - T::kX);
    // where copy j lands in its group's part of a step's buffer
    auto to_of = [&](uint32_t j) {
        return group * T::kStage + (in_group + T::kGroup * j) * 1024u;  // the channels' behind the tokens'
    };
    // Step `it` of the group. Pieces and steps behind a row's end count 0: by the buffers'
    // bounds, and where a piece behind the end of one row is inside the next, of the tokens
    // alone (0 times what the channels' row has there). Rows behind the last token or
    // channel are 0 or the last one's, and nothing is made of them
    struct Step {
        rsrc_t x, w;
        uint32_t k, outside[2];
    };
    auto step_of = [&](uint32_t it) {
        Step st;
        st.k = T::KB * (it * T::WK + group);
        st.x = buffer_of(xb, st.k < a.in_dim ? x_bytes : 0u);
        st.w = buffer_of(wb, st.k < a.in_dim ? w_bytes : 0u);
#pragma unroll
        for (uint32_t j = 0; j < 2u; j++) {
            st.outside[j] = st.k + piece_of(j) < a.in_dim ? 0u : 0xfffffff0u;
            asm volatile("" : "+v"(st.outside[j]));  // masks, no branches
        }
        return st;
    };
    auto copy = [&](const Step &st, uint32_t buffer, uint32_t j) {
        if (j < T::kX)
            copy_to_lds(st.x, (from[j] + st.k) | st.outside[j & 1u], buffer + to_of(j));
        else
            copy_to_lds(st.w, from[j] + st.k, buffer + to_of(j));
    };
    // Without DMA: a step's pieces as the words that each starts in, which the lane shifts:
    // loads at odd bytes take the memory pipe longer. What a piece has in the word behind
    // its four is the next lane's first, for the last piece that of the row's next step,
    // and a group's steps follow one another for that (130 tokens 5001 x 2047: 9.6 us, with
    // loads of those words 11.1). The buffers start and end with the words of the tile's first and
    // last byte, so nothing is read but words that the rows are in, and a load needs no
    // condition of its own
    const uint32_t n_it = ((a.in_dim + T::KB - 1u) / T::KB + T::WK - 1u) / T::WK;
    uint4 words[T::DMA ? 1u : S][kCopies];
    const uint32_t x_odd = (uint32_t)(uintptr_t)xb & 3u, w_odd = (uint32_t)(uintptr_t)wb & 3u;
    const auto x_words = __builtin_amdgcn_make_buffer_rsrc((void *)(xb - x_odd), 0, (int)((x_bytes + x_odd + 3u) & ~3u), 0x00027000);
    const auto w_words = __builtin_amdgcn_make_buffer_rsrc((void *)(wb - w_odd), 0, (int)((w_bytes + w_odd + 3u) & ~3u), 0x00027000);
    auto step_at = [&](uint32_t it) { return T::KB * (group * n_it + it); };
    auto fetch = [&](uint32_t h, uint32_t it) {
#pragma unroll
        for (uint32_t j = 0; j < kCopies; j++) {
            const uint32_t at = (from[j] + (j < T::kX ? x_odd : w_odd) + step_at(it)) & ~3u;
            words[h][j] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(j < T::kX ? x_words : w_words, at, 0, 0));
        }
    };
    auto put = [&](uint8_t *buf, uint32_t h, uint32_t it) {
        static_assert(T::DMA || kPieces == 8u, "lanes of a row");
        const uint32_t k = step_at(it);
#pragma unroll
        for (uint32_t j = 0; j < kCopies; j++) {
            const uint32_t beside = __builtin_amdgcn_update_dpp(0, (int)words[h][j].x, 0x101, 0xf, 0xf, true);  // lane + 1's
            const uint32_t after = __builtin_amdgcn_update_dpp(0, (int)words[(h + 1u) % S][j].x, 0x117, 0xf, 0xf, true);  // lane - 7's
            uint4 v = shifted(words[h][j], lane % 8u == 7u ? after : beside, (from[j] + (j < T::kX ? x_odd : w_odd)) & 3u);
            if (j < T::kX && k + T::KB > a.in_dim) {  // uniform; of the tokens alone, as above
                const uint32_t at = k + piece_of(j);
                v = first_bytes(v, at < a.in_dim ? a.in_dim - at : 0u);
            }
            const uint32_t slot = (lane & ~7u) | ((lane & 7u) ^ slot_of(j < T::kX ? j : j - T::kX));
            *(uint4 *)(buf + to_of(j) + 16u * slot) = v;
        }
    };
    auto barrier = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // ------------------------------------------------------------- steps --
    typename M::acc acc[T::MT][T::NT];
#pragma unroll
    for (uint32_t m = 0; m < T::MT; m++)
#pragma unroll
        for (uint32_t n = 0; n < T::NT; n++)
#pragma unroll
            for (uint32_t e = 0; e < M::kElem; e++) acc[m][n][e] = 0;
    uint4 av[2][T::MT], bv[2][T::NT];
    const uint32_t own = (lane % T::MF) * T::KB + 16u * ((lane / T::MF) ^ i8_slot_of<T::KB>(lane % T::MF));
    const uint32_t a_at = group * T::kStage + wm * (T::BM / T::WM) * T::KB + own;
    const uint32_t b_at = group * T::kStage + (T::BM + wn * (T::BN / T::WN)) * T::KB + own;
    constexpr uint32_t kSubBytes = T::KB / T::kSub, kMfmas = T::MT * T::NT, kSlots = kMfmas * T::kSub;
    auto read = [&](const uint8_t *buf, uint32_t sub, uint32_t to) {
#pragma unroll
        for (uint32_t n = 0; n < T::NT; n++) bv[to][n] = *(const uint4 *)(buf + (b_at ^ (kSubBytes * sub)) + n * T::MF * T::KB);
#pragma unroll
        for (uint32_t m = 0; m < T::MT; m++) av[to][m] = *(const uint4 *)(buf + (a_at ^ (kSubBytes * sub)) + m * T::MF * T::KB);
    };
    // a slice's MFMAs, the copies of a later step spread among them: a wave that issues
    // its copies one behind the other waits for the memory pipe of all waves meanwhile
    auto multiply = [&](uint32_t of, uint32_t sub, const Step &st, uint32_t buffer) {
#pragma unroll
        for (uint32_t i = 0; i < kMfmas; i++) {
            const uint32_t m = i / T::NT, n = i % T::NT;
            acc[m][n] = M::run(av[of][m], bv[of][n], acc[m][n]);
            if constexpr (T::DMA) {
#pragma unroll
                for (uint32_t j = 0; j < kCopies; j++)
                    if (j * kSlots / kCopies == sub * kMfmas + i) {
                        copy(st, buffer, j);
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
    };
    // copies of a step that are issued behind its wait, among the last slice's MFMAs
    constexpr uint32_t kBehind = kCopies - (((T::kSub - 1u) * kMfmas * kCopies + kSlots - 1u) / kSlots);
    if constexpr (T::DMA) {
#pragma unroll
        for (uint32_t s = 0; s + 1u < S; s++) {
            const Step st = step_of(s);
#pragma unroll
            for (uint32_t j = 0; j < kCopies; j++) copy(st, address_of(s), j);
        }
        wait_loads_lds<(S - 2u) * kCopies>();
    } else {
#pragma unroll
        for (uint32_t s = 0; s < S; s++) fetch(s, s);
        put(buf0, 0u, 0u);
        fetch(0u, S);
        wait_lds();
    }
    if constexpr (T::kWaves > 1u) barrier();
    read(buf0, 0u, 0u);
    for (uint32_t it = 0; it < n_it; it += S) {
#pragma unroll
        for (uint32_t s = 0; s < S; s++) {
            if (s > 0u && it + s >= n_it) break;  // uniform
            uint8_t *const buf = buf_of(s % T::kBuffers), *const next = buf_of((s + 1u) % T::kBuffers);
            // the buffer of the step before this one is free: every wave has read its last
            // operands of it and passed the barrier
            const uint32_t buffer = address_of((s + S - 1u) % S);
            Step st = {};
            if constexpr (T::DMA) st = step_of(it + s + S - 1u);
#pragma unroll
            for (uint32_t sub = 0; sub < T::kSub; sub++) {
                const uint32_t of = (s * T::kSub + sub) & 1u;
                if (sub + 1u < T::kSub) {
                    read(buf, sub + 1u, of ^ 1u);
                } else {
                    if constexpr (T::DMA) {
                        wait_loads_lds<(S - 2u) * kCopies - kBehind>();
                    } else {
                        put(next, (s + 1u) % S, it + s + 1u);
                        wait_lds();
                    }
                    if constexpr (T::kGroup > 1u) barrier();
                    read(next, 0u, of ^ 1u);
                    if constexpr (!T::DMA) fetch((s + 1u) % S, it + s + 1u + S);
                }
                __builtin_amdgcn_sched_barrier(0);
                multiply(of, sub, st, buffer);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // the copies behind the last step have landed
    barrier();

    // -------------------------------------------------------------- sums --
    // some tokens of the wave's channels at a time through LDS, so that a lane finishes 4
    // neighbouring channels and a token's stores lie side by side
    constexpr uint32_t kLanes = T::kCols / 4u, kTok = 64u / kLanes, kParts = T::kSliceTok / kTok;
    constexpr uint32_t kSlices = T::MF / T::kSliceTok, kElem = M::kElem / kSlices;
    typedef typename Elem<TYPE>::raw raw;
    uint8_t *const mine = buf0 + group * T::kStage + in_group * T::kSlice;
    const uint32_t r = r0 + wn * T::kCols + 4u * (lane % kLanes), nr = r < a.out_dim ? (a.out_dim - r < 4u ? a.out_dim - r : 4u) : 0u;
    // what the sums meet is requested before the first of them is touched, the residual a
    // slice at a time: one wait for memory each, not one a store
    constexpr uint32_t kOwn = (kParts + T::WK - 1u) / T::WK, kAll = T::MT * kSlices;
    const uint32_t t_own = t0 + wm * (T::BM / T::WM) + group * kTok + lane / kLanes;
    auto token_of = [&](uint32_t p, uint32_t i) { return t_own + p * T::kSliceTok + i * T::WK * kTok; };
    auto any = [&](uint32_t i) { return kParts % T::WK == 0u || group + i * T::WK < kParts; };  // uniform
    const bool whole = nx == T::BM && nw == T::BN;                                             // uniform
    float scale[4], bias[4] = {}, x_scale[kAll][kOwn];
#pragma unroll
    for (uint32_t p = 0; p < kAll; p++)
#pragma unroll
        for (uint32_t i = 0; i < kOwn; i++) {
            const uint32_t t = token_of(p, i);
            x_scale[p][i] = a.x_scales[t < a.n_tok ? t : a.n_tok - 1u];
        }
    load_row4<PULSAR_TYPE_F32>(a.w_scales + r, nr, scale);
    if (a.bias) load_row4<PULSAR_TYPE_F32>(a.bias + r, nr, bias);
    raw *out = (raw *)a.out + t_own * a.out_stride + r;
    const raw *residual = (const raw *)a.residual + t_own * a.res_stride + r;
#pragma unroll
    for (uint32_t p = 0; p < kAll; p++) {
        const uint32_t m = p / kSlices, part = p % kSlices;
        float res[kOwn][4] = {}, v[4u * kOwn];
        if (a.residual) {
#pragma unroll
            for (uint32_t i = 0; i < kOwn; i++) {
                if (!any(i)) continue;  // tokens behind the tile's, and behind the array's end
                const raw *from_row = residual + (p * T::kSliceTok + i * T::WK * kTok) * a.res_stride;
                if (whole)
                    load_row4<TYPE>(from_row, 4u, res[i]);
                else
                    load_row4<TYPE>(from_row, token_of(p, i) < a.n_tok ? nr : 0u, res[i]);
            }
        }
        if (p > 0u && T::WK > 1u) __syncthreads();
#pragma unroll
        for (uint32_t n = 0; n < T::NT; n++)
#pragma unroll
            for (uint32_t e = 0; e < kElem; e++)
                *(int32_t *)(mine + (M::token(e, lane) * T::kCols + n * T::MF + lane % T::MF) * 4u) =
                    acc[m][n][part * kElem + e];
        if (T::WK > 1u)
            __syncthreads();
        else
            __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t i = 0; i < kOwn; i++) {
            i8v4 sum = {};
            if (any(i)) {
                const uint32_t tw = (group + i * T::WK) * kTok + lane / kLanes;
#pragma unroll
                for (uint32_t g = 0; g < T::WK; g++)
                    sum += *(const i8v4 *)(buf0 + g * T::kStage + in_group * T::kSlice + (tw * T::kCols + 4u * (lane % kLanes)) * 4u);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) v[4u * i + j] = (float)sum[j] * x_scale[p][i] * scale[j];
        }
        if (a.bias) {
#pragma unroll
            for (uint32_t i = 0; i < 4u * kOwn; i++) v[i] += bias[i % 4u];
        }
        i8_activate(a, v);
        if (a.residual) {
#pragma unroll
            for (uint32_t i = 0; i < 4u * kOwn; i++) v[i] += res[i / 4u][i % 4u];
        }
#pragma unroll
        for (uint32_t i = 0; i < kOwn; i++) {
            raw o[4];
#pragma unroll
            for (uint32_t j = 0; j < 4u; j++) o[j] = Elem<TYPE>::down(v[4u * i + j]);
            raw *to_row = out + (p * T::kSliceTok + i * T::WK * kTok) * a.out_stride;
            if (!any(i)) continue;
            if (whole)
                store_row4<TYPE>(to_row, 4u, o);
            else if (token_of(p, i) < a.n_tok)
                store_row4<TYPE>(to_row, nr, o);
        }
        if (T::WK == 1u) __builtin_amdgcn_wave_barrier();
    }
}

// Tiles of the shape
template <typename T>
static uint64_t i8_items(const I8Args &a) {
    return (uint64_t)((a.n_tok + T::BM - 1u) / T::BM) * ((a.out_dim + T::BN - 1u) / T::BN);
}
template <uint32_t TYPE, typename T>
static int launch_i8_tile(const I8Args &a) {
    const uint64_t n = i8_items<T>(a);  // below 2^31: the entry point refuses more
    hipLaunchKernelGGL((i8_tile_kernel<TYPE, T>), grid_of(n, 8u), dim3(T::kThreads), 0, pk::stream(), a,
                       (a.n_tok + T::BM - 1u) / T::BM, (a.out_dim + T::BN - 1u) / T::BN, (uint32_t)n);
    return launch_ok("matmul_i8 tile launch");
}

}  // namespace pk
