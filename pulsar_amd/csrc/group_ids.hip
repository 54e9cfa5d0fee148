// group_ids.hip - the CSR by expert of a chunk of any length, from the router's
// ids (pulsar_moe_group_ids).
//
// A block per group. Block e scans every id: those below e (and not negative)
// count into the group's start, a ballot marks those equal to e, and the marks,
// in order, are the group's pairs. No workspace, no atomics, one launch, and the
// pairs of a group come out in (token, slot) order. The blocks read the same
// ids, from L2: n ids cost each block n / 16 wave loads.
#include "pk_route.h"

namespace pk {

constexpr uint32_t kGidThreads = 1024, kGidWaves = kGidThreads / 64u;
constexpr uint32_t kGidMarked = 1u << 18;  // ids whose marks fit 32 KiB of LDS

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

// Blocks [0, n_expert + n_shared): the groups; the blocks after them copy the
// router's weights next to the shared slots' ones.
__global__ __launch_bounds__(kGidThreads) void group_ids_kernel(GroupIds a) {
    extern __shared__ uint64_t mark[];  // 4 ballots per 256 ids
    __shared__ uint32_t below_l[kGidWaves], equal_l[kGidWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t g = blockIdx.x, n = a.n_tok * a.k_used, n_group = a.n_expert + a.n_shared;
    const uint32_t slots = a.k_used + a.n_shared;
    if (g >= n_group) {
        const uint64_t i = (uint64_t)(g - n_group) * kGidThreads + tid;
        if (i < (uint64_t)a.n_tok * slots) {
            const uint32_t t = (uint32_t)(i / slots), s = (uint32_t)(i % slots);
            a.slot_w[i] = s < a.k_used ? a.router_w[(uint64_t)t * a.k_used + s] : 1.0f;
        }
        return;
    }
    const uint32_t e = g < a.n_expert ? g : a.n_expert;
    // wave w takes the 256-id pieces [w per, (w + 1) per)
    const uint32_t pieces = (n + 255u) / 256u, per = (pieces + kGidWaves - 1u) / kGidWaves;
    const uint32_t p0 = wave * per, p1 = p0 + per < pieces ? p0 + per : pieces;
    const bool marked = n <= kGidMarked;
    // the ids of a piece: lane l those at 4 l .. 4 l + 3; past the end -1, which is no expert
    auto ids_of = [&](uint32_t p, int32_t (&id)[4]) {
        const uint32_t at = p * 256u + 4u * lane;
        if (p * 256u + 256u <= n) {
            const uint4 v = ld128((const uint8_t *)(a.sel + at));
            id[0] = (int32_t)v.x, id[1] = (int32_t)v.y, id[2] = (int32_t)v.z, id[3] = (int32_t)v.w;
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) id[j] = at + j < n ? a.sel[at + j] : -1;
        }
    };
    uint32_t below = 0, equal = 0;
    for (uint32_t p = p0; p < p1; p++) {
        int32_t id[4];
        ids_of(p, id);
        uint64_t m[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            below += (uint32_t)id[j] < e ? 1u : 0u;
            m[j] = __ballot(g < a.n_expert && id[j] == (int32_t)e);
            equal += (uint32_t)__builtin_popcountll(m[j]);
        }
        if (marked && lane < 4u) mark[4u * p + lane] = lane == 0u ? m[0] : lane == 1u ? m[1] : lane == 2u ? m[2] : m[3];
    }
    below = (uint32_t)group_sum<64>((int32_t)below);
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
        at += start;
        for (uint32_t p = p0; p < p1; p++) {
            uint64_t m[4];
            if (marked) {
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) m[j] = mark[4u * p + j];
            } else {
                int32_t id[4];
                ids_of(p, id);
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) m[j] = __ballot(id[j] == (int32_t)e);
            }
            if ((m[0] | m[1] | m[2] | m[3]) == 0ull) continue;
            const uint64_t lower = (1ull << lane) - 1ull;
            uint32_t q = at;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) q += (uint32_t)__builtin_popcountll(m[j] & lower);
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                if (m[j] >> lane & 1u) {
                    const uint32_t i = p * 256u + 4u * lane + j, t = i / a.k_used;
                    a.pairs[q++] = (t << 4) | (i - t * a.k_used);
                }
                at += (uint32_t)__builtin_popcountll(m[j]);
            }
        }
    }
    if (tid == 0) {
        a.starts[g] = start;
        if (g == n_group - 1u) a.starts[n_group] = start + count;
        a.gptrs[g] = g < a.n_expert ? bank_ptrs(a.bank, a.n_expert, (int32_t)g) : a.shared.p[g - a.n_expert];
    }
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
    pk::GroupIds a = {(pulsar_expert_ptrs *)gptrs, (uint32_t *)starts, (uint32_t *)pairs, (float *)slot_weights,
                      (const int32_t *)selected, (const float *)router_weights, *bank, {}, n_expert, n_shared, n_tok,
                      k_used};
    for (uint32_t i = 0; i < n_shared; i++) a.shared.p[i] = shared[i];
    const uint32_t n = n_tok * k_used, copies = slot_weights ? (uint32_t)((n_slot + pk::kGidThreads - 1u) / pk::kGidThreads) : 0u;
    const uint32_t lds = n <= pk::kGidMarked ? (n + 255u) / 256u * 32u : 0u;
    hipLaunchKernelGGL(pk::group_ids_kernel, dim3(n_expert + n_shared + copies), dim3(pk::kGidThreads), lds,
                       pk::stream(), a);
    return pk::launch_ok("moe group ids launch");
}
