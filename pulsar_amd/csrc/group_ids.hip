// group_ids.hip - the CSR by expert of a chunk of any length, from the router's
// ids (pulsar_moe_group_ids).
//
// Up to 65536 ids: a block per group. Block e scans every id: those below e (and
// not negative) count into the group's start, a ballot per 64 ids marks those
// equal to e, and the marks, in order, are the group's pairs. No workspace, no
// atomics, one launch, and the pairs of a group come out in (token, slot) order.
// The blocks read the same ids, from L2, which bounds them (64 bytes a clock and
// CU); a mark stays in the registers of one lane (strip i of a wave in lane i), so
// that the lanes unpack them side by side. 32768 ids of 256 experts: 5.5 us, about
// 3.5 of them a launch. Longer chunks: a counting sort in two launches, below.
#include "pk_route.h"

namespace pk {

// v with lane `lane` replaced by x (both uniform); there is no builtin for it. A
// select by the lane in its place makes the compiler do it for every strip: 301
// tokens of 256 experts 5.0 -> 6.2 us, 2048 of 1024 9.0 -> 12.0
__device__ int32_t write_lane(int32_t x, int32_t lane, int32_t v) __asm("llvm.amdgcn.writelane.i32");

constexpr uint32_t kGidThreads = 1024, kGidWaves = kGidThreads / 64u;
struct GroupIds {
    pulsar_expert_ptrs *gptrs;
    uint32_t *starts, *pairs;
    float *slot_w;
    const int32_t *sel;
    const float *router_w;
    pulsar_expert_bank bank;
    SharedSlots shared;
    uint32_t n_expert, n_shared, n_tok, k_used;
};

// the sum of v over the lanes up to this one
PK_DEV uint32_t wave_scan(uint32_t v) {
    int32_t x = (int32_t)v;
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
    return (uint32_t)x;
}

// the slots' weights, i of them by thread i: the router's, then ones
PK_DEV void copy_weights(const GroupIds &a, uint64_t i) {
    const uint32_t slots = a.k_used + a.n_shared;
    if (i >= (uint64_t)a.n_tok * slots) return;
    const uint32_t t = (uint32_t)(i / slots), s = (uint32_t)(i % slots);
    a.slot_w[i] = s < a.k_used ? a.router_w[(uint64_t)t * a.k_used + s] : 1.0f;
}

// Blocks [0, n_expert + n_shared): the groups; the blocks after them copy the
// router's weights next to the shared slots' ones.
__global__ __launch_bounds__(kGidThreads) void group_ids_kernel(GroupIds a) {
    __shared__ uint32_t below_l[kGidWaves], equal_l[kGidWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t g = blockIdx.x, n = a.n_tok * a.k_used, n_group = a.n_expert + a.n_shared;
    if (g >= n_group) return copy_weights(a, (uint64_t)(g - n_group) * kGidThreads + tid);
    const uint32_t e = g < a.n_expert ? g : a.n_expert;
    // wave w takes the 64-id strips [w per, (w + 1) per)
    const uint32_t strips = (n + 63u) / 64u, per = (strips + kGidWaves - 1u) / kGidWaves;
    const uint32_t p0 = wave * per < strips ? wave * per : strips, p1 = p0 + per < strips ? p0 + per : strips;
    constexpr uint32_t U = 16;  // strips requested at a time, a batch ahead of their use
    struct Ids {
        int32_t v[U];
    };
    auto ids_of = [&](uint32_t p) {
        Ids id;
        if ((p + U) * 64u <= n) {
            const int32_t *at = a.sel + (uint64_t)p * 64u + lane;
#pragma unroll
            for (uint32_t u = 0; u < U; u++) id.v[u] = at[64u * u];
        } else {
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint64_t i = (uint64_t)(p + u) * 64u + lane;
                const int32_t v = a.sel[i < n ? i : n - 1u];
                id.v[u] = i < n ? v : -1;  // no expert
            }
        }
        return id;
    };
    // strip p0 + i's marks in lane i (at most 64 strips a wave)
    uint32_t below = 0, equal = 0;
    int32_t lo = 0, hi = 0;
    auto strip = [&](int32_t id, uint32_t i) {
        below += (uint32_t)__builtin_popcountll(__ballot((uint32_t)id < e));
        const uint64_t eq = __ballot(id == (int32_t)e);
        if (eq) {  // uniform; of many experts few strips
            equal += (uint32_t)__builtin_popcountll(eq);
            lo = write_lane((int32_t)(uint32_t)eq, (int32_t)i, lo);
            hi = write_lane((int32_t)(eq >> 32), (int32_t)i, hi);
        }
    };
    Ids id = ids_of(p0 < p1 ? p0 : 0u);
    for (uint32_t q = p0; q < p1; q += U) {
        const Ids now = id;
        id = ids_of(q + U < p1 ? q + U : q);
        if (q + U <= p1) {
#pragma unroll
            for (uint32_t u = 0; u < U; u++) strip(now.v[u], q + u - p0);
        } else {
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                if (q + u < p1) strip(now.v[u], q + u - p0);
        }
    }
    uint64_t mark = (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
    if (lane == 0) {
        below_l[wave] = below;
        equal_l[wave] = equal;
    }
    __syncthreads();
    uint32_t start = 0, at = 0, count = 0;
#pragma unroll
    for (uint32_t w = 0; w < kGidWaves; w++) {
        start += below_l[w];
        at += w < wave ? equal_l[w] : 0u;
        count += equal_l[w];
    }
    if (g >= a.n_expert) {  // a shared slot: every token, behind the routed pairs
        const uint32_t i = g - a.n_expert;
        start += i * a.n_tok;
        for (uint32_t t = tid; t < a.n_tok; t += kGidThreads) a.pairs[start + t] = (t << 4) | (a.k_used + i);
        count = a.n_tok;
    } else {
        // each lane the pairs of its mark, behind those of the lanes below it
        const uint32_t own = (uint32_t)__builtin_popcountll(mark);
        uint32_t q = start + at + wave_scan(own) - own;
        const uint32_t i0 = (p0 + lane) * 64u;
        while (mark) {
            const uint32_t i = i0 + (uint32_t)__builtin_ctzll(mark), t = i / a.k_used;
            a.pairs[q++] = (t << 4) | (i - t * a.k_used);
            mark &= mark - 1ull;
        }
    }
    if (tid == 0) {
        a.starts[g] = start;
        if (g == n_group - 1u) a.starts[n_group] = start + count;
        a.gptrs[g] = g < a.n_expert ? bank_ptrs(a.bank, a.n_expert, (int32_t)g) : a.shared.p[g - a.n_expert];
    }
}

// ---- long chunks: a counting sort in two launches --------------------------
//
// count: 12 blocks, each the ids of one twelfth per expert, into the 12 words of
// the expert's record in gptrs, which nothing else holds yet. place: a block per
// part of a twelfth turns the counts into the place of its first pair of every
// expert, counts the twelfth's ids before its part, and puts its pairs where they
// belong, 64 ids of a wave at a time: the lanes with the same expert find each
// other by ballots of the id's bits, so their order is the ids' order. The last
// block to have read the counts (an arrival count in starts' last word, which the
// first launch cleared) writes the records and starts over them.
constexpr uint32_t kSeg = sizeof(pulsar_expert_ptrs) / 4u;  // 12
constexpr uint32_t kMostExperts = 64u * kMaxPerLane;
static_assert(kMostExperts <= kGidThreads, "a thread per expert");

// adds the ids of [i0, i1) to count, by the whole block
PK_DEV void count_ids(uint32_t *count, const int32_t *sel, uint32_t i0, uint32_t i1, uint32_t n_expert) {
    constexpr uint32_t U = 8;
    for (uint64_t at = i0 + threadIdx.x; at < i1; at += U * kGidThreads) {
        int32_t id[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint64_t i = at + u * kGidThreads;
            id[u] = sel[i < i1 ? i : i1 - 1u];
            id[u] = i < i1 ? id[u] : -1;
        }
#pragma unroll
        for (uint32_t u = 0; u < U; u++)
            if ((uint32_t)id[u] < n_expert) atomicAdd(&count[id[u]], 1u);
    }
}

__global__ __launch_bounds__(kGidThreads) void group_count_kernel(GroupIds a, uint32_t seg_len) {
    __shared__ uint32_t count[kMostExperts];
    const uint32_t tid = threadIdx.x, n = a.n_tok * a.k_used, seg = blockIdx.x;
    if (seg >= kSeg) return copy_weights(a, (uint64_t)(seg - kSeg) * kGidThreads + tid);
    for (uint32_t e = tid; e < a.n_expert; e += kGidThreads) count[e] = 0u;
    if (seg == 0u && tid == 0u) a.starts[a.n_expert + a.n_shared] = 0u;
    __syncthreads();
    const uint64_t i0 = (uint64_t)seg * seg_len, i1 = i0 + seg_len;
    if (i0 < n) count_ids(count, a.sel, (uint32_t)i0, i1 < n ? (uint32_t)i1 : n, a.n_expert);
    __syncthreads();
    for (uint32_t e = tid; e < a.n_expert; e += kGidThreads) ((uint32_t *)a.gptrs)[e * kSeg + seg] = count[e];
}

// blocks seg * parts + part, then one per 1024 tokens and shared slot
__global__ __launch_bounds__(kGidThreads) void group_place_kernel(GroupIds a, uint32_t seg_len, uint32_t part_len,
                                                                  uint32_t parts) {
    __shared__ uint32_t at_l[kGidWaves][kMostExperts];  // where a wave's next pair of an expert goes
    __shared__ uint32_t before_l[kMostExperts];
    __shared__ uint32_t sums[kGidWaves], last_l;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t E = a.n_expert, n_group = E + a.n_shared, n = a.n_tok * a.k_used;
    const uint32_t seg = blockIdx.x / parts, part = blockIdx.x % parts;  // seg >= kSeg: a shared slot's block
    // thread e: the ids of expert e, and those in the twelfths before this one
    uint32_t total = 0u, before = 0u;
    if (tid < E) {
        uint32_t c[kSeg];
        __builtin_memcpy(c, (const uint32_t *)a.gptrs + tid * kSeg, sizeof c);
#pragma unroll
        for (uint32_t s = 0; s < kSeg; s++) {
            total += c[s];
            before += s < seg ? c[s] : 0u;
        }
    }
    const uint32_t upto = wave_scan(total);
    if (lane == 63u) sums[wave] = upto;
    for (uint32_t e = lane; e < E; e += 64u) at_l[wave][e] = 0u;
    if (tid < E) before_l[tid] = 0u;
    __syncthreads();  // every count is read
    uint32_t start = upto - total, routed = 0u;
#pragma unroll
    for (uint32_t w = 0; w < kGidWaves; w++) {
        start += w < wave ? sums[w] : 0u;
        routed += sums[w];
    }
    // nothing that this block wrote is handed over, so the arrival needs no fence
    if (tid == 0u) last_l = atomicAdd(&a.starts[n_group], 1u) == gridDim.x - 1u ? 1u : 0u;
    if (seg >= kSeg) {
        const uint32_t b = blockIdx.x - kSeg * parts, i = b % a.n_shared, t = b / a.n_shared * kGidThreads + tid;
        if (t < a.n_tok) a.pairs[routed + i * a.n_tok + t] = (t << 4) | (a.k_used + i);
    } else {
        const uint64_t s0 = (uint64_t)seg * seg_len, s1 = s0 + seg_len < n ? s0 + seg_len : n;
        const uint64_t p0 = s0 + (uint64_t)part * part_len, p1 = p0 + part_len < s1 ? p0 + part_len : s1;
        if (p0 < p1) {  // block-uniform
            count_ids(before_l, a.sel, (uint32_t)s0, (uint32_t)p0, E);
            // wave w: strips of 64 ids [w per, (w + 1) per) of the part
            const uint32_t strips = ((uint32_t)(p1 - p0) + 63u) / 64u, per = (strips + kGidWaves - 1u) / kGidWaves;
            auto id_of = [&](uint32_t strip) {
                const uint64_t i = p0 + strip * 64u + lane;
                const int32_t v = a.sel[i < p1 ? i : p1 - 1u];
                return i < p1 && strip < strips ? v : -1;
            };
            for (uint32_t k = 0; k < per; k++) {
                const int32_t id = id_of(wave * per + k);
                if ((uint32_t)id < E) atomicAdd(&at_l[wave][id], 1u);
            }
            __syncthreads();
            if (tid < E) {
                uint32_t at = start + before + before_l[tid];
#pragma unroll
                for (uint32_t w = 0; w < kGidWaves; w++) {
                    const uint32_t c = at_l[w][tid];
                    at_l[w][tid] = at;
                    at += c;
                }
            }
            __syncthreads();
            const uint32_t bits = 32u - (uint32_t)__builtin_clz(E);  // of the ids
            const uint64_t lower = (1ull << lane) - 1ull;
            for (uint32_t k = 0; k < per; k++) {
                const uint32_t strip = wave * per + k;
                const int32_t id = id_of(strip);
                const bool real = (uint32_t)id < E;
                uint64_t same = __ballot(real);
                for (uint32_t b = 0; b < bits; b++) {
                    const bool set = (uint32_t)id >> b & 1u;
                    const uint64_t m = __ballot(set);
                    same &= set ? m : ~m;
                }
                const uint32_t rank = (uint32_t)__builtin_popcountll(same & lower);
                uint32_t at = 0u;
                if (real) at = at_l[wave][id];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (real && rank == 0u) at_l[wave][id] = at + (uint32_t)__builtin_popcountll(same);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if (real) {
                    const uint32_t i = (uint32_t)p0 + strip * 64u + lane, t = i / a.k_used;
                    a.pairs[at + rank] = (t << 4) | (i - t * a.k_used);
                }
            }
        }
    }
    __syncthreads();
    if (last_l == 0u) return;
    if (tid < E) a.starts[tid] = start;
    for (uint32_t g = tid; g < n_group; g += kGidThreads)
        a.gptrs[g] = g < E ? bank_ptrs(a.bank, E, (int32_t)g) : a.shared.p[g - E];
    if (tid <= a.n_shared) a.starts[E + tid] = routed + tid * a.n_tok;
}

}  // namespace pk

extern "C" int pulsar_moe_group_ids(void *gptrs, void *starts, void *pairs, void *slot_weights, const void *selected,
                                    const void *router_weights, const pulsar_expert_bank *bank, uint32_t n_expert,
                                    const pulsar_expert_ptrs *shared, uint32_t n_shared, uint32_t n_tok,
                                    uint32_t k_used) {
    const uint64_t n_slot = (uint64_t)n_tok * ((uint64_t)k_used + n_shared);
    if (!gptrs || !starts || !pairs || !selected || !bank || (slot_weights && !router_weights) || n_expert == 0 ||
        n_expert > 64u * pk::kMaxPerLane || n_shared > pk::kMaxShared || (n_shared && !shared) || n_tok == 0 ||
        n_tok > 1u << 28 || k_used == 0 || k_used > 16u || k_used + n_shared > 16u || n_slot > 0x7fffffffull)
        return pk::reject("moe group ids");
    // Blocks still read the ids and weights as others write, and hand their counts
    // over in gptrs and starts. Weights copied onto themselves are each read and
    // written by one thread
    struct {
        const void *at;
        pk::u128 bytes;
    } const out[4] = {{gptrs, sizeof(pulsar_expert_ptrs) * (pk::u128)(n_expert + n_shared)},
                      {starts, 4 * (pk::u128)(n_expert + n_shared + 1u)},
                      {pairs, 4 * (pk::u128)n_slot},
                      {slot_weights, slot_weights ? 4 * (pk::u128)n_slot : 0}};
    const pk::u128 in_bytes = 4 * (pk::u128)n_tok * k_used;
    for (uint32_t i = 0; i < (slot_weights ? 4u : 3u); i++) {
        bool over = pk::overlap(out[i].at, out[i].bytes, selected, in_bytes);
        if (slot_weights && !(i == 3u && slot_weights == router_weights && n_shared == 0u))
            over |= pk::overlap(out[i].at, out[i].bytes, router_weights, in_bytes);
        for (uint32_t j = 0; j < i; j++) over |= pk::overlap(out[i].at, out[i].bytes, out[j].at, out[j].bytes);
        if (over) return pk::reject("moe group ids (overlap)");
    }
    pk::GroupIds a = {(pulsar_expert_ptrs *)gptrs, (uint32_t *)starts, (uint32_t *)pairs, (float *)slot_weights,
                      (const int32_t *)selected, (const float *)router_weights, *bank, {}, n_expert, n_shared, n_tok,
                      k_used};
    for (uint32_t i = 0; i < n_shared; i++) a.shared.p[i] = shared[i];
    const uint32_t n = n_tok * k_used;
    const uint32_t copies = slot_weights ? (uint32_t)((n_slot + pk::kGidThreads - 1u) / pk::kGidThreads) : 0u;
    const dim3 block(pk::kGidThreads);
    // Both sides timed, 8 ids a token: of 256 experts 65536 ids 7.4 against 8.7 us,
    // 98304 10.5 against 9.4; of 512 32768 7.5 against 9.1, 65536 10.2 against 9.4;
    // of 1024 16384 8.6 against 10.1, 32768 11.6 against 10.6. The scan has room
    // for the marks of 65536 ids
    if (n <= 65536u && (uint64_t)n * n_expert <= 24u << 20) {
        hipLaunchKernelGGL(pk::group_ids_kernel, dim3(n_expert + n_shared + copies), block, 0, pk::stream(), a);
    } else {
        const uint32_t seg_len = (n / pk::kSeg / 64u + 1u) * 64u;  // kSeg of them hold n
        const uint32_t want = (seg_len + pk::kGidThreads - 1u) / pk::kGidThreads, parts = want < 16u ? want : 16u;
        const uint32_t part_len = (seg_len / parts / 64u + 1u) * 64u;
        const uint32_t tokens = (n_tok + pk::kGidThreads - 1u) / pk::kGidThreads;  // blocks of a shared slot
        hipLaunchKernelGGL(pk::group_count_kernel, dim3(pk::kSeg + copies), block, 0, pk::stream(), a, seg_len);
        hipLaunchKernelGGL(pk::group_place_kernel, dim3(pk::kSeg * parts + tokens * n_shared), block, 0, pk::stream(),
                           a, seg_len, part_len, parts);
    }
    return pk::launch_ok("moe group ids launch");
}
