// Verification of drafted tokens against the target's candidates, from given
// uniform numbers: rejection sampling down a tree.
//
// With p the target's distribution and q the draft's, accepting a token t
// drawn from q with probability min(1, p(t)/q(t)) and otherwise drawing from
// (p − q)₊ normalized gives draws of p. Siblings drawn without replacement
// repeat this with r = that residual in p's place and q without the tokens
// refused. r is nothing outside the target's 64 candidates, so it lives in
// one warp's registers, two candidates a lane in the list's order.
//
// Bound: latency, a chain of warp reductions a visited node. Two warps a
// sequence: one walks and makes the target's distributions, the other makes
// the draft's of the same node; every node's lists are on their way to shared
// memory from the start, so no visited node waits for its own. The draft's
// probabilities of the target's candidates (64 by 64 comparisons) are found
// only where a child is refused. A chain of 6 greedy drafts 3.1 us; 256 trees of
// 48 nodes with a draft's lists 20.0 us, the longest walk's ten nodes at 2 us
// each (34 us in the first form, one warp a sequence).
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "cache.cuh"
#include "kernels.h"
#include "numerics.cuh"
#include "tma.cuh"

namespace cb {

namespace {

constexpr uint32_t kList = 64;
constexpr uint32_t kAbsent = 0xFFFFFFFFu;
constexpr uint32_t kAll = 0xFFFFFFFFu;

struct VerifyArgs {
    cb_verify v;
    float target_log_min_p, draft_log_min_p;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) v += __shfl_xor_sync(kAll, v, k);
    return v;
}

// Two sums, whose steps go beside one another.
__device__ __forceinline__ float2 warp_sums(float a, float b) {
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
        const float x = __shfl_xor_sync(kAll, a, k), y = __shfl_xor_sync(kAll, b, k);
        a += x;
        b += y;
    }
    return make_float2(a, b);
}

// Sum of the values before this lane's pair (a, b), in list order.
__device__ __forceinline__ float sum_before(float a, float b, uint32_t lane) {
    float run = a + b;
#pragma unroll
    for (uint32_t k = 1; k < 32u; k <<= 1) {
        const float o = __shfl_up_sync(kAll, run, k);
        if (lane >= k) run += o;
    }
    const float before = __shfl_up_sync(kAll, run, 1);
    return lane ? before : 0.0f;
}

// A list's entries 2·lane and 2·lane + 1: tokens and their probabilities.
struct List {
    uint32_t token[2];
    float p[2];
};

// The draw's distribution over a list (select.cu, draw_candidates: the
// prefix top_k, top_p and min_p leave, weighed at the temperature). False
// when its first candidate is not finite.
__device__ bool distribution(const uint32_t* pairs, const cb_sampling& s, float log_min_p, uint32_t lane, List& out) {
    const uint4 w = reinterpret_cast<const uint4*>(pairs)[lane];
    const uint32_t bits[2] = {w.x, w.z};
    out.token[0] = w.y;
    out.token[1] = w.w;
    const uint32_t first_bits = __shfl_sync(kAll, bits[0], 0);
    const float first = __uint_as_float(first_bits);
    const uint32_t k = min(max(s.top_k, 1u), kList);
    bool kept[2];
    float gap[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const float logit = __uint_as_float(bits[c]);
        gap[c] = logit - first;
        kept[c] = 2u * lane + c < k && out.token[c] != kAbsent && bits[c] != 0xFF800000u;
    }
    if (s.top_p < 1.0f) {
        const float a = kept[0] ? exp_nonpositive(gap[0]) : 0.0f, b = kept[1] ? exp_nonpositive(gap[1]) : 0.0f;
        const float before = sum_before(a, b, lane);
        const float scale = 1.0f / __shfl_sync(kAll, before + a + b, 31);
        kept[0] = kept[0] && (lane == 0 || before * scale < s.top_p);   // the first stays, whatever top_p is
        kept[1] = kept[1] && (before + a) * scale < s.top_p;
    }
    if (s.min_p != 0.0f) {
        const uint32_t m0 = __ballot_sync(kAll, lane > 0 && !(__uint_as_float(bits[0]) >= first + log_min_p));
        const uint32_t m1 = __ballot_sync(kAll, !(__uint_as_float(bits[1]) >= first + log_min_p));
        const uint32_t below = min(m0 ? 2u * (__ffs(m0) - 1u) : kList, m1 ? 2u * (__ffs(m1) - 1u) + 1u : kList);
        kept[0] = kept[0] && 2u * lane < below;
        kept[1] = kept[1] && 2u * lane + 1u < below;
    }
    if (s.temperature > 0.0f) {
        const float a = kept[0] ? exp_nonpositive(gap[0] / s.temperature) : 0.0f;
        const float b = kept[1] ? exp_nonpositive(gap[1] / s.temperature) : 0.0f;
        const float scale = 1.0f / warp_sum(a + b);
        out.p[0] = a * scale;
        out.p[1] = b * scale;
    } else {
        out.p[0] = lane == 0 ? 1.0f : 0.0f;
        out.p[1] = 0.0f;
    }
    return (first_bits & 0x7F800000u) != 0x7F800000u;
}

// The list's probability of a token (0 where it is not there).
__device__ __forceinline__ float of_token(const List& l, uint32_t token) {
    const uint32_t m0 = __ballot_sync(kAll, l.token[0] == token), m1 = __ballot_sync(kAll, l.token[1] == token);
    if (m0) return __shfl_sync(kAll, l.p[0], __ffs(m0) - 1);
    if (m1) return __shfl_sync(kAll, l.p[1], __ffs(m1) - 1);
    return 0.0f;
}

__device__ __forceinline__ void forget(List& l, uint32_t token) {
    if (l.token[0] == token) l.p[0] = 0.0f;
    if (l.token[1] == token) l.p[1] = 0.0f;
}

// Two warps a sequence (one without a draft's lists).
__global__ void __launch_bounds__(64) verify_kernel(const VerifyArgs args) {
    const cb_verify& a = args.v;
    extern __shared__ __align__(16) uint32_t lists[];   // [tokens][64][2] of the target, then of the draft
    __shared__ uint2 draft_list[kList];                 // the current node's draft tokens and probabilities
    __shared__ uint32_t visited;                        // the node to make a draft distribution of; kAbsent: none
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t s = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const size_t row0 = static_cast<size_t>(s) * a.tokens;
    const uint32_t n = a.nodes ? min(a.nodes[s], a.tokens) : a.tokens;
    if (n == 0) {
        if (warp == 0) {
            for (uint32_t i = lane; i < a.tokens; i += 32u) a.path[row0 + i] = kAbsent;
            if (lane < 4) a.sampled[4u * s + lane] = 0u;
            if (lane == 0) a.kept[s] = 0u;
        }
        return;
    }
    // Each warp brings its own lists: lane by lane what the lane will read, a
    // node at a time, so a warp waits for its own copies alone.
    uint32_t* const own = lists + warp * a.tokens * (2u * kList);
    const uint32_t* const source = (warp ? a.draft_candidates : a.candidates) + row0 * 2u * kList;
    for (uint32_t i = 0; i < n; ++i) cp_async16(own + i * 2u * kList + 4u * lane, source + i * 2u * kList + 4u * lane);
    if (warp == 1) {
        cp_async_wait_all();
        for (;;) {
            __syncthreads();   // the walker has named a node
            const uint32_t at = visited;
            if (at == kAbsent) return;
            List q;
            if (!distribution(own + at * 2u * kList, a.draft, args.draft_log_min_p, lane, q))
                q.p[0] = q.p[1] = 0.0f;   // no distribution: its children are refused
            draft_list[2u * lane] = make_uint2(q.token[0], __float_as_uint(q.p[0]));
            draft_list[2u * lane + 1u] = make_uint2(q.token[1], __float_as_uint(q.p[1]));
            __syncthreads();   // it is there
        }
    }
    const bool have = a.draft_candidates != nullptr;
    for (uint32_t i = lane; i < a.tokens; i += 32u) a.path[row0 + i] = i == 0 ? 0u : kAbsent;
    __syncwarp();
    // Lane i holds nodes i and i + 32: token, uniform number, parent (the
    // latest ancestor; a later one or none at all: not a node of the walk).
    uint32_t id[2], parent[2];
    float u[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint32_t i = lane + 32u * c;
        id[c] = 0;
        u[c] = 0.0f;
        parent[c] = kAbsent;
        if (i < n) {
            id[c] = a.ids[row0 + i];
            u[c] = a.uniforms[row0 + i];
            if (i > 0) {
                if (a.ancestors) {
                    const uint64_t mask = a.ancestors[row0 + i] & ((1ull << i) - 1ull);
                    if (mask) parent[c] = 63u - __clzll(mask);
                } else {
                    parent[c] = i - 1u;
                }
            }
        }
    }
    cp_async_wait_all();
    uint32_t at = 0, kept = 1;
    List r, q;
    bool failed;
    for (;;) {
        const uint32_t c0 = __ballot_sync(kAll, parent[0] == at), c1 = __ballot_sync(kAll, parent[1] == at);
        uint64_t children = (static_cast<uint64_t>(c1) << 32) | c0;
        const bool ask = have && children;
        if (ask) {
            if (lane == 0) visited = at;
            __syncthreads();
        }
        failed = !distribution(own + at * 2u * kList, a.target, args.target_log_min_p, lane, r);
        if (ask) {
            __syncthreads();
            const uint4 e = reinterpret_cast<const uint4*>(draft_list)[lane];
            q.token[0] = e.x;
            q.p[0] = __uint_as_float(e.y);
            q.token[1] = e.z;
            q.p[1] = __uint_as_float(e.w);
        }
        if (failed || !children) break;
        float mass = 1.0f;
        float on_target[2] = {0.0f, 0.0f};   // the draft's probability of this lane's target candidates
        bool matched = false;
        uint32_t next = kAbsent;
        while (children) {
            const uint32_t i = __ffsll(children) - 1u;
            children &= children - 1ull;
            const uint32_t t = __shfl_sync(kAll, i < 32u ? id[0] : id[1], i & 31u);
            const float draw = __shfl_sync(kAll, i < 32u ? u[0] : u[1], i & 31u);
            const float p = of_token(r, t);
            float q_of = 1.0f;
            if (have) {
                q_of = of_token(q, t);
                if (!(q_of > 0.0f)) continue;
                q_of /= mass;
            }
            if (draw * q_of < p) {
                next = i;
                break;
            }
            float rest[2];
            if (have) {
                if (!matched) {   // by the distribution as it was: what has been refused since is forgotten below
                    matched = true;
#pragma unroll 8
                    for (uint32_t j = 0; j < kList; j += 2u) {
                        const uint4 e = reinterpret_cast<const uint4*>(draft_list)[j / 2u];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (e.x == r.token[c]) on_target[c] = __uint_as_float(e.y);
                            if (e.z == r.token[c]) on_target[c] = __uint_as_float(e.w);
                        }
                    }
                }
                const float scale = 1.0f / mass;
                float given[2] = {on_target[0] * scale, on_target[1] * scale};
                if (!(scale < __builtin_huge_valf())) {   // a subnormal mass
                    given[0] = on_target[0] / mass;
                    given[1] = on_target[1] / mass;
                }
                rest[0] = fmaxf(r.p[0] - given[0], 0.0f);
                rest[1] = fmaxf(r.p[1] - given[1], 0.0f);
            } else {
                rest[0] = r.token[0] == t ? 0.0f : r.p[0];
                rest[1] = r.token[1] == t ? 0.0f : r.p[1];
            }
            float total;
            if (have) {
                // What is left of q, summed and not one less what is gone: a draft
                // sure of its first token leaves its siblings 1e-8 and less, which
                // that difference rounds away. Nothing left: every later sibling's
                // probability is 0, and it is refused.
                forget(q, t);
                const float2 both = warp_sums(rest[0] + rest[1], q.p[0] + q.p[1]);
                total = both.x;
                mass = both.y;
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    if (r.token[c] == t) on_target[c] = 0.0f;
            } else {
                total = warp_sum(rest[0] + rest[1]);
            }
            if (total > 0.0f) {
                const float scale = 1.0f / total;
                r.p[0] = rest[0] * scale;
                r.p[1] = rest[1] * scale;
            }
        }
        if (next == kAbsent) break;
        at = next;
        if (lane == 0) a.path[row0 + kept] = at;
        ++kept;
    }
    if (have) {   // lets the other warp go
        if (lane == 0) visited = kAbsent;
        __syncthreads();
    }
    const float u0 = __shfl_sync(kAll, u[0], 0);
    uint32_t token = 0;
    if (!failed) {
        const float before = sum_before(r.p[0], r.p[1], lane);
        const float run0 = before + r.p[0], run1 = run0 + r.p[1];
        const float goal = u0 * __shfl_sync(kAll, run1, 31);
        const uint32_t m0 = __ballot_sync(kAll, run0 > goal && r.p[0] > 0.0f);
        const uint32_t m1 = __ballot_sync(kAll, run1 > goal && r.p[1] > 0.0f);
        uint32_t chosen = min(m0 ? 2u * (__ffs(m0) - 1u) : kList, m1 ? 2u * (__ffs(m1) - 1u) + 1u : kList);
        if (chosen == kList) {   // rounding left the goal at the total: the last candidate with weight
            const uint32_t w0 = __ballot_sync(kAll, r.p[0] > 0.0f), w1 = __ballot_sync(kAll, r.p[1] > 0.0f);
            chosen = max(w0 ? 2u * (31u - __clz(w0)) : 0u, w1 ? 2u * (31u - __clz(w1)) + 1u : 0u);
        }
        token = __shfl_sync(kAll, chosen & 1u ? r.token[1] : r.token[0], chosen >> 1);
    }
    if (lane == 0) {
        a.kept[s] = kept;
        a.sampled[4u * s] = token;
        a.sampled[4u * s + 1u] = failed ? 1u : 0u;
        a.sampled[4u * s + 2u] = __float_as_uint(u0);
        a.sampled[4u * s + 3u] = 0u;
    }
}

}  // namespace

cudaError_t verify_run(const cb_verify& v, cudaStream_t stream, bool pdl) {
    static bool configured[64] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device >= 64) return cudaErrorInvalidDevice;
    if (!configured[device]) {
        e = cudaFuncSetAttribute(verify_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(2u * kTreeRows * kList * 8u));
        if (e != cudaSuccess) return e;
        configured[device] = true;
    }
    VerifyArgs a{v, 0.0f, 0.0f};
    if (v.target.min_p > 0.0f) a.target_log_min_p = std::log(v.target.min_p);
    if (v.draft.min_p > 0.0f) a.draft_log_min_p = std::log(v.draft.min_p);
    cudaLaunchConfig_t cfg = {};
    const uint32_t warps = v.draft_candidates ? 2u : 1u;
    cfg.gridDim = dim3(v.sequences);
    cfg.blockDim = dim3(32u * warps);
    cfg.dynamicSmemBytes = static_cast<size_t>(warps) * v.tokens * kList * 8u;   // 64 KB at most
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, verify_kernel, a);
}

}  // namespace cb
