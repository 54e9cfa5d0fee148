// ksplit.hip - the dense product of a short chunk: a block's waves split K.
//
// A chunk of a few to some hundred tokens over a matrix of a few thousand rows is
// bound by neither bytes nor matrix instructions but by latency and by the decode
// of its weights, so what counts is how much of the chip works on it at once. A
// block is 16 rows x 16 NS tokens, its W waves take every W-th super-block each,
// with no wait for another wave before the end: the weights straight from memory,
// decoded as the wide tile decodes them (TileFmt, pk_tile.h), the tokens' q8 values
// from L2 through a piece of LDS of the wave's own. At the end the W sums of an
// element are added in wave order.
#include "pk_epilogue.h"
#include "pk_tile.h"

namespace pk {

template <uint32_t Q, uint32_t NS>
struct KTokens {  // what a super-block needs of the tokens
    uint4 a[NS][4];
    uint2 bs[NS];
    float d[NS];
};

template <uint32_t Q, uint32_t NS, uint32_t W, typename E>
__global__ __launch_bounds__(64 * W) void ksplit_kernel(float *__restrict__ out, const uint8_t *__restrict__ w,
                                                        const pulsar_block_q8_K *__restrict__ xq, uint32_t nb,
                                                        uint32_t out_dim, uint32_t n_tok, uint64_t row_bytes,
                                                        uint32_t n_tt, uint32_t n_item, E epi) {
    using F = TileFmt<Q>;
    constexpr uint32_t kElem = NS * 4u * 64u, kOwn = (kElem + 64u * W - 1u) / (64u * W);
    // a wave's own: the tokens' q8 values of a step, at the end its sums
    __shared__ __align__(16) uint8_t lds[W][NS * 4096u];
    PK_FMT_LUT(Q)
    // XCD x (blocks x, x + 8, ...) takes the x-th eighth of the items, token tiles
    // fastest: a row tile's weights come into one L2
    const uint32_t item = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (item >= n_item) return;  // block-uniform
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t i = lane & 15u, q = lane >> 4;
    const uint32_t t0 = item % n_tt * (16u * NS), row0 = item / n_tt * 16u;
    // the elements this thread finishes: e = tid, tid + 64 W, ...: element e / 64 % 4 of slice e / 256
    typename E::Term term[kOwn];
    auto token_of = [&](uint32_t e) { return t0 + 16u * (e >> 8) + 4u * (e >> 4 & 3u) + (e >> 6 & 3u); };
#pragma unroll
    for (uint32_t k = 0; k < kOwn; k++) {
        const uint32_t e = tid + 64u * W * k, t = token_of(e < kElem ? e : 0u), row = row0 + (e & 15u);
        term[k] = epi.fetch(t < n_tok ? t : n_tok - 1u, row < out_dim ? row : out_dim - 1u);
    }
    const uint8_t *wr = w + (uint64_t)(row0 + i < out_dim ? row0 + i : out_dim - 1u) * row_bytes;
    // byte offset of a token's row from the tile's first (host: below 2^32)
    const uint8_t *xb = (const uint8_t *)(xq + (uint64_t)t0 * nb);
    auto token_at = [&](uint32_t t) { return (t0 + t < n_tok ? t : n_tok - 1u - t0) * (nb * 292u); };
    // A row's 256 q8 values lie in one piece: 16 lanes load them (tokens 4 m + l / 16)
    // and the wave's LDS turns them to the lanes that multiply them; by the lanes
    // themselves, 16 bytes of each row at a time, they take the memory pipeline 4
    // times as long. Piece p of token t goes to slot p ^ t % 16, on distinct banks
    uint32_t xo[NS][4], xt[NS];
#pragma unroll
    for (uint32_t n = 0; n < NS; n++) {
#pragma unroll
        for (uint32_t m = 0; m < 4; m++) xo[n][m] = token_at(16u * n + 4u * m + q) + 4u + 16u * i;
        xt[n] = token_at(16u * n + i);
    }
    uint8_t *mine = lds[wave];
    auto weights = [&](uint32_t sb) { return F::load(wr + (uint64_t)sb * F::kSb, q); };
    auto tokens = [&](uint32_t sb) {
        KTokens<Q, NS> k;
        const uint8_t *x = xb + (uint64_t)sb * 292u;  // uniform
#pragma unroll
        for (uint32_t n = 0; n < NS; n++) {
#pragma unroll
            for (uint32_t m = 0; m < 4; m++) k.a[n][m] = ldw128(x + xo[n][m]);
            if (F::kMin) k.bs[n] = ldw64(x + xt[n] + 260u + 8u * q);
            k.d[n] = __uint_as_float(ldw32(x + xt[n]));
        }
        return k;
    };
    float acc[NS][4];
#pragma unroll
    for (uint32_t n = 0; n < NS; n++)
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) acc[n][r] = 0.0f;
    auto step = [&](const typename F::Raw &raw, const KTokens<Q, NS> &k) {
        TileW tw;
        F::decode(raw, q, lut, tw);
#pragma unroll
        for (uint32_t n = 0; n < NS; n++)
#pragma unroll
            for (uint32_t m = 0; m < 4; m++)
                *(uint4 *)(mine + 4096u * n + 256u * (4u * m + q) + 16u * (i ^ (4u * m + q))) = k.a[n][m];
        wave_lds_sync();
#pragma unroll
        for (uint32_t n = 0; n < NS; n++) {
            v4i_t dl = {}, dh = {};
#pragma unroll
            for (uint32_t s = 0; s < 4; s++) {
                const uint4 a = *(const uint4 *)(mine + 4096u * n + 256u * i + 16u * (F::piece(s, q) ^ i));
                dl = mfma64(a, tw.lo[s], dl);
                if (F::kHi) dh = mfma64(a, tw.hi[s], dh);
            }
            v4f_t ms;
            if constexpr (F::kMin) ms = mfma16_f16(make_uint2(f16_of_i16(k.bs[n].x), f16_of_i16(k.bs[n].y)), tw.mins);
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                // as the wide tile: the super-block's value from exact integers
                const int32_t sum = F::kHi ? (int32_t)((uint32_t)dh[r] << F::kShift) + dl[r] : dl[r];
                float v = (F::kNeg ? -tw.xd : tw.xd) * (float)sum;
                if constexpr (F::kMin) v = __builtin_fmaf(-tw.xmin, ms[r], v);
                acc[n][r] = __builtin_fmaf(__shfl(k.d[n], (int)(4u * q + r), 64), v, acc[n][r]);
            }
        }
        wave_lds_sync();  // read before the next step's values take their place
    };
    // The weights come from HBM and are requested a step ahead, the tokens from L2,
    // under the decode
    if (wave < nb) {
        typename F::Raw raw = weights(wave);
        uint32_t sb = wave;
        for (; sb + W < nb; sb += W) {
            const KTokens<Q, NS> k = tokens(sb);
            const typename F::Raw next = weights(sb + W);
            step(raw, k);
            raw = next;
        }
        step(raw, tokens(sb));
    }
#pragma unroll
    for (uint32_t n = 0; n < NS; n++)
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) ((float *)mine)[(4u * n + r) * 64u + lane] = acc[n][r];
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kOwn; k++) {
        const uint32_t e = tid + 64u * W * k, t = token_of(e), row = row0 + (e & 15u);
        if (e >= kElem || t >= n_tok || row >= out_dim) continue;
        float v = ((const float *)lds[0])[e];
#pragma unroll
        for (uint32_t x = 1; x < W; x++) v += ((const float *)lds[x])[e];
        epi.put(out, out_dim, t, row, v, term[k]);
    }
}

template <uint32_t Q, uint32_t NS, uint32_t W, typename E>
static int launch_ksplit_n(float *out, const uint8_t *w, const pulsar_block_q8_K *xq, uint32_t nb, uint32_t out_dim,
                           uint32_t n_tok, uint64_t row_bytes, const E &epi) {
    const uint32_t n_tt = (n_tok + 16u * NS - 1u) / (16u * NS);
    const uint64_t n_item = (uint64_t)n_tt * ((out_dim + 15u) / 16u);
    if (n_item > 0x7ffffff0ull) return -1;
    hipLaunchKernelGGL((ksplit_kernel<Q, NS, W, E>), dim3((uint32_t)((n_item + 7u) & ~7ull)), dim3(64 * W), 0,
                       pk::stream(), out, w, xq, nb, out_dim, n_tok, row_bytes, n_tt, (uint32_t)n_item, epi);
    return launch_ok("matmul_kq_fused K split launch");
}

static uint64_t ksplit_tiles(uint32_t out_dim, uint32_t n_tok) {  // of 16 rows x 16 tokens
    return (uint64_t)((n_tok + 15u) / 16u) * ((out_dim + 15u) / 16u);
}

// The token tile with the shortest time, which goes by the rounds its blocks take:
// a CU holds two blocks of one slice at once, one of more (registers). Time of a
// round as measured, in hundredths of one of two slices (Q4_K 4096 x 4096: 4.9 us).
struct KPlan {
    uint32_t ns;
    uint64_t cost;
};
static KPlan ksplit_plan(uint32_t out_dim, uint32_t n_tok) {
    const uint64_t slices = (n_tok + 15u) / 16u, row_tiles = (out_dim + 15u) / 16u;
    KPlan best = {1u, slices * row_tiles <= 256u ? 70u : (slices * row_tiles + 511u) / 512u * 106u};
    const uint64_t round[3] = {100u, 140u, 162u};
    for (uint32_t ns = 2; ns <= 4u && ns <= slices; ns++) {
        const uint64_t cost = ((slices + ns - 1u) / ns * row_tiles + 255u) / 256u * round[ns - 2u];
        if (cost <= best.cost) best = {ns, cost};
    }
    return best;
}

template <uint32_t Q, typename E>
static int launch_ksplit_q(float *out, const uint8_t *w, const pulsar_block_q8_K *xq, uint32_t nb, uint32_t out_dim,
                           uint32_t n_tok, uint64_t row_bytes, const E &epi) {
    const uint32_t ns = ksplit_plan(out_dim, n_tok).ns;
    const uint64_t tiles = ksplit_tiles(out_dim, n_tok);
#define PK_KS(NS, W) return launch_ksplit_n<Q, NS, W>(out, w, xq, nb, out_dim, n_tok, row_bytes, epi)
    if (ns == 1u && nb >= 16u && tiles <= 128u) PK_KS(1, 16);
    if (ns == 1u) PK_KS(1, 8);
    if (ns == 2u) PK_KS(2, 8);
    if (ns == 3u) PK_KS(3, 8);
    PK_KS(4, 8);
#undef PK_KS
}

// Where this kernel was the faster one: a fit by format, rows, row length and tokens
// to timed shapes, weights from HBM. Of 3000 other shapes (48 to 16384 rows, 1 to 56
// super-blocks, 2 to 500 tokens, 7 formats) it takes 2255 and is there 1.36 times as
// fast as the kernels behind it; 54 of them are more than a tenth slower than those.
// It is ahead as long as its blocks take few rounds, more for formats of a longer
// decode (`most`, in the plan's cost): then the wide tile or, up to 16 tokens, the
// 16-row kernel has the whole chip at work too and shares a decoded row among more
// tokens (Q4_K 4096 x 4096: 33 tokens 8.5 against 11.0 us, 100 tokens 18.9 against
// 15.2). Below `least` tiles of long rows its blocks leave most CUs idle, and
// kernels that spread rows further are ahead: the lane kernels, a wave per row
// (Q3_K 83 x 12032, 2 tokens: 14.7 against 4.4 us), and for Q6_K, whose decode is
// the longest, the 16-row kernel.
static bool ksplit_wins(uint32_t quant, uint32_t nb, uint32_t out_dim, uint32_t n_tok) {
    if (n_tok == 1u) return false;
    const uint64_t tiles = ksplit_tiles(out_dim, n_tok);
    const bool q45 = quant == PULSAR_QUANT_Q4_K || quant == PULSAR_QUANT_Q5_K, q2 = quant == PULSAR_QUANT_Q2_K;
    const bool q6 = quant == PULSAR_QUANT_Q6_K, iq = quant == PULSAR_QUANT_IQ4_XS || quant == PULSAR_QUANT_IQ2_XXS;
    uint32_t least = 0u, most = 212u;
    if (n_tok <= 4u) {
        if (q6 && nb > 8u && (n_tok == 2u || (nb <= 16u && tiles > 256u))) return false;
        if (iq && n_tok == 2u) most = 106u;
        least = q6 || (n_tok == 2u && !q45 && !q2) ? 129u : 65u;
    } else if (n_tok <= 32u) {
        if (q6 && nb > 32u && n_tok <= 16u) return false;
        least = q45 || (q6 && nb <= 16u) ? 0u : q6 ? (nb <= 32u ? 257u : 513u) : 33u;
        if (n_tok > 16u && (q6 || quant == PULSAR_QUANT_Q3_K)) most = 300u;
    } else {
        least = n_tok > 64u || q45 || q6 ? 0u : 17u;
        most = q6 || iq || quant == PULSAR_QUANT_Q3_K ? 300u : n_tok > 128u && !q45 ? 162u : 212u;
    }
    return ksplit_plan(out_dim, n_tok).cost <= most && (nb <= 8u || tiles >= least);
}

// -1: no such kernel for the format, or another one is as fast
template <typename E>
int launch_ksplit(uint32_t quant, float *out, const uint8_t *w, const pulsar_block_q8_K *xq, uint32_t in_dim,
                  uint32_t out_dim, uint32_t n_tok, uint64_t row_bytes, const E &epi) {
    const uint32_t nb = in_dim / 256u;
    if (nb > 65536u) return -1;  // a tile's activation offsets are 32 bits
    if (!ksplit_wins(quant, nb, out_dim, n_tok)) return -1;
#define PK_KQ(Q) \
    case Q: return launch_ksplit_q<Q>(out, w, xq, nb, out_dim, n_tok, row_bytes, epi);
    switch (quant) {
        PK_KQ(PULSAR_QUANT_Q4_K)
        PK_KQ(PULSAR_QUANT_Q5_K)
        PK_KQ(PULSAR_QUANT_Q6_K)
        PK_KQ(PULSAR_QUANT_Q2_K)
        PK_KQ(PULSAR_QUANT_Q3_K)
        PK_KQ(PULSAR_QUANT_IQ4_XS)
        PK_KQ(PULSAR_QUANT_IQ2_XXS)
    default: return -1;
    }
#undef PK_KQ
}
template int launch_ksplit(uint32_t, float *, const uint8_t *, const pulsar_block_q8_K *, uint32_t, uint32_t, uint32_t,
                           uint64_t, const FusedOut &);

}  // namespace pk
