// group_ids.hip - the CSR by expert of a chunk of any length, from the router's
// ids (pulsar_moe_group_ids).
//
// A block per group. Block e scans every id: those below e (and not negative)
// count into the group's start, a ballot per 64 ids marks those equal to e, and
// the marks, in order, are the group's pairs. No workspace, no atomics, one
// launch, and the pairs of a group come out in (token, slot) order. The blocks
// read the same ids, from L2; a mark stays in the registers of one lane (ballot
// i of a wave in lane i % 64), so that the lanes unpack them side by side.
#include "pk_route.h"

namespace pk {

constexpr uint32_t kGidThreads = 1024, kGidWaves = kGidThreads / 64u;
struct GroupIds {
    pulsar_expert_ptrs *gptrs;
    uint32_t *starts, *pairs;
    float *slot_w;
    const int32_t *sel;
    const float *router_w;
    pulsar_expert_bank bank;
    SharedSlots shared;
    uint32_t n_expert, n_shared, n_tok, k_used, kept;
};

// Blocks [0, n_expert + n_shared): the groups; the blocks after them copy the
// router's weights next to the shared slots' ones.
// R: 64-bit marks a lane keeps, for up to 65536 R ids; where there are more,
// a.kept is 0 and the blocks read the ids twice.
template <uint32_t R>
__global__ __launch_bounds__(kGidThreads) void group_ids_kernel(GroupIds a) {
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
    // wave w takes the 64-id strips [w per, (w + 1) per), eight at a time
    const uint32_t strips = (n + 63u) / 64u, per = (strips + kGidWaves - 1u) / kGidWaves;
    const uint32_t p0 = wave * per < strips ? wave * per : strips, p1 = p0 + per < strips ? p0 + per : strips;
    constexpr uint32_t U = 8;
    auto ids_of = [&](uint32_t p, int32_t (&id)[U]) {
        if ((p + U) * 64u <= n) {
            const int32_t *at = a.sel + (uint64_t)p * 64u + lane;
#pragma unroll
            for (uint32_t u = 0; u < U; u++) id[u] = at[64u * u];
        } else {
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint64_t i = (uint64_t)(p + u) * 64u + lane;
                const int32_t v = a.sel[i < n ? i : n - 1u];
                id[u] = i < n ? v : -1;  // no expert
            }
        }
    };
    uint64_t mark[R];
#pragma unroll
    for (uint32_t q = 0; q < R; q++) mark[q] = 0ull;
    // the marks of strips p .. of one register, strips past p1 none
    auto marks_of = [&](uint32_t p, uint32_t &below, uint32_t &equal) {
        uint64_t mk = 0ull;
        const uint32_t end = p + 64u < p1 ? p + 64u : p1;
        for (uint32_t q = p; q < end; q += U) {
            int32_t id[U];
            ids_of(q, id);
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                if (q + u >= end) break;  // uniform
                below += (uint32_t)__builtin_popcountll(__ballot((uint32_t)id[u] < e));
                const uint64_t eq = __ballot(id[u] == (int32_t)e);
                equal += (uint32_t)__builtin_popcountll(eq);
                mk = lane == q + u - p ? eq : mk;
            }
        }
        return mk;
    };
    uint32_t below = 0, equal = 0;
    if (a.kept) {
#pragma unroll
        for (uint32_t q = 0; q < R; q++)
            if (p0 + 64u * q < p1) mark[q] = marks_of(p0 + 64u * q, below, equal);
    } else {
        for (uint32_t p = p0; p < p1; p += 64u) marks_of(p, below, equal);
    }
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
        // each lane the pairs of its mark, behind those of the lanes below it
        auto unpack = [&](uint32_t p, uint64_t mk) {
            const uint32_t own = (uint32_t)__builtin_popcountll(mk);
            int32_t x = (int32_t)own;  // inclusive scan over the wave
            x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
            x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
            x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
            x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
            x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
            x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
            uint32_t q = at + (uint32_t)x - own;
            const uint32_t i0 = (p + lane) * 64u;
            while (mk) {
                const uint32_t i = i0 + (uint32_t)__builtin_ctzll(mk), t = i / a.k_used;
                a.pairs[q++] = (t << 4) | (i - t * a.k_used);
                mk &= mk - 1ull;
            }
            at += (uint32_t)__builtin_amdgcn_readlane(x, 63);
        };
        if (a.kept) {
#pragma unroll
            for (uint32_t q = 0; q < R; q++)
                if (p0 + 64u * q < p1) unpack(p0 + 64u * q, mark[q]);
        } else {
            for (uint32_t p = p0; p < p1; p += 64u) {
                uint32_t b = 0, c = 0;
                unpack(p, marks_of(p, b, c));
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
                      k_used, 1u};
    for (uint32_t i = 0; i < n_shared; i++) a.shared.p[i] = shared[i];
    const uint32_t n = n_tok * k_used;
    const uint32_t copies = slot_weights ? (uint32_t)((n_slot + pk::kGidThreads - 1u) / pk::kGidThreads) : 0u;
    const dim3 grid(n_expert + n_shared + copies), block(pk::kGidThreads);
    if (n <= 65536u) {
        hipLaunchKernelGGL(pk::group_ids_kernel<1>, grid, block, 0, pk::stream(), a);
    } else {
        a.kept = n <= 8u * 65536u ? 1u : 0u;
        hipLaunchKernelGGL(pk::group_ids_kernel<8>, grid, block, 0, pk::stream(), a);
    }
    return pk::launch_ok("moe group ids launch");
}
