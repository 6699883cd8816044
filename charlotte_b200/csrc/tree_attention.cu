// Attention of drafted trees over a cache (cb_tree_attention_run): each row
// of a step attends the committed entries its window reaches and the nodes
// of its ancestor mask; a step of one row a sequence is plain decode.
//
// Mathematics. For a row's query q and the visible keys j,
//   s_j = scale_log2e · q·k_j,  p_j = 2^(s_j − m),  out = Σ p_j v_j / Σ p_j,
// m a running maximum (one pass over the cache). The products run on the
// tensor cores in f16 with f32 sums, without giving up f32 accuracy: a cache
// value is exact in f16 (an f16 row as it is, an 8-bit row as its code), and
// the f32 operand beside it is given in two f16 terms, x = hi + lo with hi
// the nearest f16 and lo the nearest f16 of what is left (22 bits of x), each
// multiplied by the same cache values. A query row is first scaled by the
// power of two that brings its largest magnitude into [2^14, 2^15), so
// neither term leaves f16's range; a row's scale is applied to the finished
// score, once a key. Weights take the value's scale: w_j = p_j·scale_j,
// scaled by the power of two that brings the largest of them that the row has
// seen to 2^14 (it is kept like the running maximum, and the sums with it). It
// is not the largest scale's: a key of large values and no weight would leave
// the others few bits, or none.
//
// A masked key's weight is a chosen zero, never 0 times something, and its
// score a chosen −∞: what it holds does not reach the row. In an 8-bit cache
// every code is finite, so that is enough; an f16 value that is not finite
// would still meet the zero weight in the product (0·∞), so a warp whose sums
// come out not finite runs its keys again with scalar sums over the visible
// keys alone.
//
// Split. A step is bounded by reading the cache (for few rows) and has one
// to a few hundred (sequence, kv head) pairs, so a pair's keys are divided
// among CTAs until the GPU is full, and a CTA's among its warps, a tile of 16
// keys at a time; a warp works alone through the whole loop (copies,
// scores, softmax, sums) with no barrier, and the states (m, Σp, Σpv) meet at
// the end, over shared memory and then over the workspace, where the last
// CTA of a pair to finish adds them in part order (the result does not
// depend on which that is). All G query heads of a kv head and all rows of
// the tree share the keys' fragments.
//
// Bound. A batch's decode is bound by instructions issued (two a cycle; the
// copies, codes to f16 and two terms for every product, of whose 16 rows a step
// of 8 rows or fewer leaves half empty): 64 sequences of one row over 2k to 4k
// keys of 128 values, 8-bit, 132 us (3.0 TB/s), of 64 values 95 us, of 256
// values in one head 47 us (2.1 TB/s); f16 rows of 128, 16 sequences over 2,000,
// 29 us (3.0 TB/s); 32 sequences of 16 rows over 8k to 16k 242 us (3.2 TB/s). A small step
// is latency: one row over 2,000 keys 9.2 us, 16 sequences of 52 rows over a
// window of 512 (256 values) 16.8 us.
//
// Fragments (mma.sync m16n8k16). The contraction order over d is free, so a
// lane takes keys as 16-byte pieces of a row, four steps a piece; the columns
// of P·V are free too, so a lane takes its key's values as d/8 consecutive
// ones. Codes become f16 in two instructions for two values: the byte is
// placed under the exponent of 1,024 (1024 + code) and 1,152 is subtracted.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "api_common.h"
#include "cache.cuh"
#include "kernels.h"
#include "tma.cuh"
#include "tree_attention.cuh"

namespace cb {

namespace {

constexpr uint32_t kKeys = 16;   // keys a tile
constexpr float kLeastUnit = 0x1p-111f;   // 2^14 over it is a normal number
constexpr uint32_t kAll = kAllLanes;

__device__ __forceinline__ void mma(float (&c)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// The sizes of one form: head dimension D, 8-bit or f16 rows, MT row tiles
// of 16, W warps a CTA, S stages of copies a warp.
template <uint32_t D_, bool Q8_, uint32_t MT_, uint32_t W_, uint32_t S_>
struct Form {
    static constexpr uint32_t D = D_, MT = MT_, W = W_, S = S_;
    static constexpr bool Q8 = Q8_;
    static constexpr uint32_t kRows = 16 * MT;
    static constexpr uint32_t kRowBytes = Q8 ? D : 2 * D;
    static constexpr uint32_t kPieces = kRowBytes / 16;                    // 16-byte pieces of a row
    static constexpr uint32_t kTileBytes = kKeys * kRowBytes;
    static constexpr uint32_t kStage = 2 * kTileBytes + (Q8 ? 128 : 0);    // keys, values, 16 + 16 scales
    static constexpr uint32_t kSteps = D / 16;
    static constexpr uint32_t kResident = MT == 1 && D <= 128 ? 2 : 1;     // CTAs an SM the registers are held to
    static constexpr uint32_t kQuery = MT * kSteps * 2 * 512;              // fragments, hi and lo
    static constexpr uint32_t kMergeRow = D + (D == 256 ? 4 : D == 128 ? 16 : 8);   // floats (see merge_piece)
    static constexpr uint32_t kMerge = W * 16 * (kMergeRow + 3) * 4;
    static constexpr uint32_t kWork = W * S * kStage > kMerge ? W * S * kStage : kMerge;
    // per row: the mask, first visible entry, score factor
    static constexpr uint32_t kRowInfo = kRows * 16;
    static constexpr uint32_t kSmem = kWork + kQuery + kRowInfo;
};

// Where piece c of tile row r is kept, so that the lanes that read together
// fall on distinct banks.
template <class F>
__device__ __forceinline__ uint32_t key_piece(uint32_t r, uint32_t c) {
    return F::kRowBytes >= 128 ? c ^ ((r & 1u) << 2) : c;
}
template <class F>
__device__ __forceinline__ uint32_t value_piece(uint32_t r, uint32_t c) {
    return F::kRowBytes >= 128 ? c ^ (r & 6u) : c ^ (r & 2u);
}

// Where 16-byte piece c of a row's outputs is kept while the warps' states
// meet: a lane's run of D/32 pieces in an order of its own, so that the eight
// lanes (two rows by four runs) that store together fall on distinct banks.
template <class F>
__device__ __forceinline__ uint32_t merge_piece(uint32_t c) {
    constexpr uint32_t kRun = F::D / 32;
    return c ^ (c / kRun >> (F::D == 256 ? 0 : F::D == 128 ? 1 : 2));
}

struct TreeArgs {
    cb_tree_attention a;
    uint32_t groups;        // query heads a kv head
    uint32_t row_groups;    // CTAs' worth of rows a (sequence, kv head)
    uint32_t parts;         // most parts a pair's keys are divided into
    unsigned int* tickets;
    float* partials;        // [sequence][kv head][row group][part][rows][D + 2]
};

template <class F>
__global__ void __launch_bounds__(F::W * 32, F::kResident) tree_attention_kernel(const TreeArgs args) {
    constexpr uint32_t D = F::D, MT = F::MT, W = F::W;
    extern __shared__ __align__(128) char smem[];
    const cb_tree_attention& a = args.a;
    const cb_cache& c = a.cache;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t g = lane >> 2, q = lane & 3u;
    const uint32_t h = blockIdx.y % c.kv_heads, rg = blockIdx.y / c.kv_heads;
    const uint32_t s = blockIdx.z, part = blockIdx.x;
    const uint32_t G = args.groups;

    grid_dependency_wait();
    grid_dependents_launch();
    const Step step = step_of(a, s);
    const uint32_t keys = step.end - step.first;
    const uint32_t tiles = (keys + kKeys - 1u) / kKeys;
    // a part takes at least a tile a warp, so a short sequence takes fewer parts
    const uint32_t part_tiles = max((tiles + args.parts - 1u) / args.parts, W);
    const uint32_t parts = max((tiles + part_tiles - 1u) / part_tiles, 1u);
    if (part >= parts) return;
    const uint32_t tile0 = part * part_tiles, tile1 = min(tile0 + part_tiles, tiles);

    uint64_t* row_mask = reinterpret_cast<uint64_t*>(smem + F::kWork + F::kQuery);
    uint32_t* row_first = reinterpret_cast<uint32_t*>(row_mask + F::kRows);
    float* row_factor = reinterpret_cast<float*>(row_first + F::kRows);
    uint4* query = reinterpret_cast<uint4*>(smem + F::kWork);
    char* ring = smem + warp * F::S * F::kStage;

    // ---- copies: a tile's rows into stage `st` of this warp's ring --------------
    const size_t sequence_at = s * cache_sequence_stride(c);
    constexpr uint32_t kElement = F::Q8 ? 1u : 2u;
    const char* key_rows = static_cast<const char*>(c.key) + (sequence_at + static_cast<size_t>(h) * D) * kElement;
    const char* value_rows = static_cast<const char*>(c.value) + (sequence_at + static_cast<size_t>(h) * D) * kElement;
    const size_t entry_bytes = static_cast<size_t>(c.kv_heads) * D * kElement;
    const size_t scale_at = F::Q8 ? s * cache_scale_stride(c) + static_cast<size_t>(h) * c.slots : 0u;
    const uint32_t first_slot = step.first % c.slots;   // entries first .. end − 1 span at most `slots`
    auto copy_tile = [&](uint32_t tile, uint32_t st) {
        char* to = ring + st * F::kStage;
        const uint32_t i0 = tile * kKeys;
        constexpr uint32_t kRowsPass = 32u / F::kPieces > 0 ? 32u / F::kPieces : 1u;
        if (F::kPieces <= 32u) {
            const uint32_t piece = lane % F::kPieces, r0 = lane / F::kPieces;
#pragma unroll
            for (uint32_t r = r0; r < kKeys; r += kRowsPass) {
                const uint32_t i = i0 + r;
                const bool there = i < keys;
                uint32_t slot = first_slot + (there ? i : 0u);
                if (slot >= c.slots) slot -= c.slots;
                const size_t at = slot * entry_bytes + piece * 16u;
                copy16(to + r * F::kRowBytes + key_piece<F>(r, piece) * 16u, key_rows + at, there);
                copy16(to + F::kTileBytes + r * F::kRowBytes + value_piece<F>(r, piece) * 16u, value_rows + at, there);
            }
        }
        if (F::Q8) {
            const uint32_t i = i0 + (lane & 15u);
            const bool there = i < keys;
            uint32_t slot = first_slot + (there ? i : 0u);
            if (slot >= c.slots) slot -= c.slots;
            copy4(to + 2 * F::kTileBytes + lane * 4u, (lane < 16u ? c.key_scale : c.value_scale) + scale_at + slot, there);
        }
    };
#pragma unroll
    for (uint32_t i = 0; i + 1u < F::S; ++i) {
        const uint32_t t = tile0 + warp + W * i;
        if (t < tile1) copy_tile(t, i);
        copies_commit();
    }

    // ---- the rows: masks, first entries, and query fragments. A warp has its
    // rows' loads on their way together -----------------------------------------
    {
        constexpr uint32_t kMine = F::kRows / W, kVecs = (D + 127u) / 128u;
        static_assert(F::kRows % W == 0u && kMine <= 32u, "every warp has as many rows");
        auto node_of = [&](uint32_t r) { return (rg * F::kRows + r) / G; };
        float4 x[kMine][kVecs];
#pragma unroll
        for (uint32_t k = 0; k < kMine; ++k) {
            const uint32_t r = warp + k * W, node = node_of(r);
            const float* src = a.query + (static_cast<size_t>(s) * a.tokens + node) * (a.query_stride ? a.query_stride : a.query_heads * D) +
                               (static_cast<size_t>(h) * G + (rg * F::kRows + r) % G) * D;
#pragma unroll
            for (uint32_t i = 0; i < kVecs; ++i) {
                x[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (node < step.nodes && lane + 32u * i < D / 4u) x[k][i] = reinterpret_cast<const float4*>(src)[lane + 32u * i];
            }
        }
        if (lane < kMine) {
            const uint32_t r = warp + lane * W, node = node_of(r);
            uint64_t mask = 0;
            uint32_t first = 0;   // a row past the step's is computed as any other and written as zeros
            if (node < step.nodes) row_sight(a, step, s, node, mask, first);
            row_mask[r] = mask;
            row_first[r] = first;
        }
#pragma unroll
        for (uint32_t k = 0; k < kMine; ++k) {
            const uint32_t r = warp + k * W;
            uint32_t top = 0;
#pragma unroll
            for (uint32_t i = 0; i < kVecs; ++i)
                top = max(max(max(top, __float_as_uint(x[k][i].x) & 0x7FFFFFFFu), __float_as_uint(x[k][i].y) & 0x7FFFFFFFu),
                          max(__float_as_uint(x[k][i].z) & 0x7FFFFFFFu, __float_as_uint(x[k][i].w) & 0x7FFFFFFFu));
            const float up = row_power(__reduce_max_sync(kAll, top));
            if (lane == 0) row_factor[r] = a.scale_log2e / up;
            // step k's elements of lane column qq: piece j·4 + qq, word w
            const uint32_t mt = r / 16u, rr = r % 16u;
            uint32_t* frag = reinterpret_cast<uint32_t*>(query + mt * F::kSteps * 2u * 32u);
#pragma unroll
            for (uint32_t i = 0; i < kVecs; ++i) {
                const uint32_t e = lane + 32u * i;   // four consecutive elements, 4·e ..
                if (e >= D / 4u) break;
                constexpr uint32_t kWords = F::Q8 ? 4u : 2u;   // steps a 16-byte piece
                const uint32_t piece = e / kWords, w = e % kWords;
                const uint32_t step_k = piece / 4u * kWords + w, qq = piece % 4u;
                uint32_t h0, l0, h1, l1;
                split2(x[k][i].x * up, x[k][i].y * up, h0, l0);
                split2(x[k][i].z * up, x[k][i].w * up, h1, l1);
                const uint32_t to = ((step_k * 2u) * 32u + (rr % 8u) * 4u + qq) * 4u + rr / 8u;
                frag[to] = h0;
                frag[to + 2u] = h1;
                frag[to + 128u] = l0;
                frag[to + 130u] = l1;
            }
        }
    }
    __syncthreads();

    // This lane's rows: g and g + 8 of each row tile.
    uint64_t mask[MT][2];
    uint32_t first[MT][2];
    float factor[MT][2];
    uint32_t latest = 0;   // the latest first entry of the CTA's rows that attend any
#pragma unroll
    for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            mask[m][k] = row_mask[m * 16u + g + 8u * k];
            first[m][k] = row_first[m * 16u + g + 8u * k];
            factor[m][k] = row_factor[m * 16u + g + 8u * k];
            latest = max(latest, first[m][k]);
        }
    latest = __reduce_max_sync(kAll, latest);
    const uint32_t context = min(step.length, step.end);

    float o[MT][D / 8][4];
    float top[MT][2], sum[MT][2];
    float unit[MT][2];   // Q8: the power of two a row's p·scale are held against
    const uint32_t mine = tile0 + warp < tile1 ? (tile1 - tile0 - warp + W - 1u) / W : 0u;

    auto pass = [&](const bool scalar) {
#pragma unroll
        for (uint32_t m = 0; m < MT; ++m) {
#pragma unroll
            for (uint32_t n = 0; n < D / 8; ++n) o[m][n][0] = o[m][n][1] = o[m][n][2] = o[m][n][3] = 0.0f;
            top[m][0] = top[m][1] = kNegInf;
            unit[m][0] = unit[m][1] = kLeastUnit;
            sum[m][0] = sum[m][1] = 0.0f;
        }
        for (uint32_t it = 0; it < mine; ++it) {
            copies_wait<F::S - 2>();
            __syncwarp();
            {
                const uint32_t ahead = it + F::S - 1u, t = tile0 + warp + W * ahead;
                if (t < tile1) copy_tile(t, ahead % F::S);
                copies_commit();
            }
            const char* keys_at = ring + (it % F::S) * F::kStage;
            const char* values_at = keys_at + F::kTileBytes;
            const float* scales = reinterpret_cast<const float*>(keys_at + 2 * F::kTileBytes);
            const uint32_t e0 = step.first + (tile0 + warp + W * it) * kKeys;   // the tile's first entry

            // ---- scores: rows × 16 keys, key 8·n + 2q + {0, 1} a lane ------------
            float sc[MT][2][4], sl[MT][2][4];   // of the hi and the lo terms: chains half as long, and small sums added to small
#pragma unroll
            for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n) {
                    sc[m][n][0] = sc[m][n][1] = sc[m][n][2] = sc[m][n][3] = 0.0f;
                    sl[m][n][0] = sl[m][n][1] = sl[m][n][2] = sl[m][n][3] = 0.0f;
                }
#pragma unroll
            for (uint32_t j = 0; j < F::kPieces / 4u; ++j) {
                uint4 kw[2];
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n) {
                    const uint32_t r = 8u * n + g;
                    kw[n] = *reinterpret_cast<const uint4*>(keys_at + r * F::kRowBytes + key_piece<F>(r, j * 4u + q) * 16u);
                }
                constexpr uint32_t kWords = F::Q8 ? 4u : 2u;
#pragma unroll
                for (uint32_t w = 0; w < kWords; ++w) {
                    uint32_t b[2][2];
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n) {
                        const uint32_t words[4] = {kw[n].x, kw[n].y, kw[n].z, kw[n].w};
                        if (F::Q8) {
                            b[n][0] = codes2<0x4140>(words[w]);
                            b[n][1] = codes2<0x4342>(words[w]);
                        } else {
                            b[n][0] = words[2u * w];
                            b[n][1] = words[2u * w + 1u];
                        }
                    }
                    const uint32_t k = j * kWords + w;
#pragma unroll
                    for (uint32_t m = 0; m < MT; ++m) {
                        const uint4 hi = query[(m * F::kSteps + k) * 64u + lane];
                        const uint4 lo = query[(m * F::kSteps + k) * 64u + 32u + lane];
#pragma unroll
                        for (uint32_t n = 0; n < 2; ++n) {
                            mma(sc[m][n], hi, b[n][0], b[n][1]);
                            mma(sl[m][n], lo, b[n][0], b[n][1]);
                        }
                    }
                }
            }

            // ---- softmax: masks, running maxima, weights -------------------------
            const bool plain = e0 >= latest && e0 + kKeys <= context;   // every row sees every key
            float vs[2][2] = {{1.0f, 1.0f}, {1.0f, 1.0f}};
            float most = 0.0f;
            if (F::Q8) {
                const float2 v0 = *reinterpret_cast<const float2*>(scales + 16 + 2u * q);
                const float2 v1 = *reinterpret_cast<const float2*>(scales + 24 + 2u * q);
                vs[0][0] = v0.x; vs[0][1] = v0.y; vs[1][0] = v1.x; vs[1][1] = v1.y;
                most = fmaxf(fmaxf(v0.x, v0.y), fmaxf(v1.x, v1.y));
            }
            float ks[2][2] = {{1.0f, 1.0f}, {1.0f, 1.0f}};
            if (F::Q8) {
                const float2 k0 = *reinterpret_cast<const float2*>(scales + 2u * q);
                const float2 k1 = *reinterpret_cast<const float2*>(scales + 8 + 2u * q);
                ks[0][0] = k0.x; ks[0][1] = k0.y; ks[1][0] = k1.x; ks[1][1] = k1.y;
            }
            uint4 phi[MT], plo[MT];
            float alpha[MT][2];
#pragma unroll
            for (uint32_t m = 0; m < MT; ++m) {
                float p[2][4];
                uint32_t hidden = 0;
                // p is at most 1, so no p·scale can pass a unit that no scale passes
                // (the weights have room for twice it): seen before the scores are
                const bool wide = F::Q8 && __any_sync(kAll, most > 2.0f * fminf(unit[m][0], unit[m][1]));
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t k = i >> 1, x = i & 1u;
                        float v = (sc[m][n][i] + sl[m][n][i]) * factor[m][k] * ks[n][x];
                        if (!plain) {
                            const uint32_t e = e0 + 8u * n + 2u * q + x;
                            const bool ok = e < step.end && (e < step.length ? e >= first[m][k]
                                                                             : (mask[m][k] >> (e - step.length) & 1ull));
                            if (!ok) {
                                v = kNegInf;
                                hidden |= 1u << (4u * n + i);
                            }
                        }
                        p[n][i] = v;
                    }
                bool risen = false;
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                    float t = fmaxf(fmaxf(p[0][2 * k], p[0][2 * k + 1]), fmaxf(p[1][2 * k], p[1][2 * k + 1]));
                    t = fmaxf(t, __shfl_xor_sync(kAll, t, 1));
                    t = fmaxf(t, __shfl_xor_sync(kAll, t, 2));
                    const float was = top[m][k], now = fmaxf(was, t);
                    risen |= now > was;
                    top[m][k] = now;
                    alpha[m][k] = now == kNegInf ? 1.0f : ex2(was - now);
                }
                // p, added to its row's sum, then p·scale
                const float base[2] = {top[m][0] == kNegInf ? 0.0f : top[m][0], top[m][1] == kNegInf ? 0.0f : top[m][1]};
                float add[2] = {0.0f, 0.0f};
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t k = i >> 1, x = i & 1u;
                        const float w = ex2(p[n][i] - base[k]);
                        add[k] += w;
                        p[n][i] = F::Q8 ? w * vs[n][x] : w;
                    }
                if (!plain) {   // a hidden key's scale may be anything
#pragma unroll
                    for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            if (hidden >> (4u * n + i) & 1u) p[n][i] = 0.0f;
                }
                // The unit falls with the sums when the maximum rises, and is
                // raised where some p·scale passes it; what both make of the
                // outputs so far:
                float keep[2] = {alpha[m][0], alpha[m][1]};
                bool moved = __any_sync(kAll, risen);
                if (F::Q8 && (moved || wide)) {
                    float big[2];
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        big[k] = fmaxf(fmaxf(p[0][2 * k], p[0][2 * k + 1]), fmaxf(p[1][2 * k], p[1][2 * k + 1]));
                        if (!(big[k] < __builtin_huge_valf())) big[k] = 0.0f;
                    }
                    moved = moved || __any_sync(kAll, big[0] > 2.0f * unit[m][0] || big[1] > 2.0f * unit[m][1]);
                    if (moved) {
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) {
                            float b = fmaxf(big[k], __shfl_xor_sync(kAll, big[k], 1));
                            b = fmaxf(b, __shfl_xor_sync(kAll, b, 2));
                            b = fmaxf(fmaxf(b, unit[m][k] * alpha[m][k]), kLeastUnit);
                            // the power of two at or above it, kept where 2^14 over it is a normal number
                            const uint32_t now = min((__float_as_uint(b) + 0x007FFFFFu) >> 23, 253u);   // its exponent
                            // unit over now, at most 1 / alpha where alpha is not 0
                            const int over = static_cast<int>((__float_as_uint(unit[m][k]) >> 23) - now) + 127;
                            keep[k] *= __uint_as_float(static_cast<uint32_t>(min(max(over, 0), 254)) << 23);
                            unit[m][k] = __uint_as_float(now << 23);
                        }
                    }
                }
                // 2^14 over the units, by their exponents
                const float down[2] = {F::Q8 ? __uint_as_float((268u - (__float_as_uint(unit[m][0]) >> 23)) << 23) : 16384.0f,
                                       F::Q8 ? __uint_as_float((268u - (__float_as_uint(unit[m][1]) >> 23)) << 23) : 16384.0f};
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) p[n][i] *= down[i >> 1];
                sum[m][0] = fmaf(sum[m][0], alpha[m][0], add[0]);
                sum[m][1] = fmaf(sum[m][1], alpha[m][1], add[1]);
                split2(p[0][0], p[0][1], phi[m].x, plo[m].x);
                split2(p[0][2], p[0][3], phi[m].y, plo[m].y);
                split2(p[1][0], p[1][1], phi[m].z, plo[m].z);
                split2(p[1][2], p[1][3], phi[m].w, plo[m].w);
                if (moved) {
#pragma unroll
                    for (uint32_t n = 0; n < D / 8; ++n) {
                        o[m][n][0] *= keep[0];
                        o[m][n][1] *= keep[0];
                        o[m][n][2] *= keep[1];
                        o[m][n][3] *= keep[1];
                    }
                }
                if (!F::Q8 && scalar) {
                    // Sums over the visible keys alone, each lane its own rows and
                    // columns: the weights of a row's 16 keys lie in its four lanes.
                    for (uint32_t j = 0; j < kKeys; ++j) {
                        const uint32_t from = (lane & 28u) | (j % 8u) / 2u;
                        float w[2];
                        bool off[2];
#pragma unroll
                        for (uint32_t k = 0; k < 2; ++k) {
                            float v = 0.0f;
                            uint32_t hid = 0;
#pragma unroll
                            for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
                                for (uint32_t x = 0; x < 2; ++x)
                                    if (n == j / 8u && x == j % 2u) {
                                        v = p[n][2 * k + x];
                                        hid = hidden >> (4u * n + 2u * k + x) & 1u;
                                    }
                            w[k] = __shfl_sync(kAll, v, from);
                            off[k] = __shfl_sync(kAll, hid, from) != 0u;
                        }
#pragma unroll
                        for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                            for (uint32_t n = 0; n < D / 8; ++n) {
                                const uint32_t d = (2u * q + x) * (D / 8u) + n;
                                const uint32_t at = j * F::kRowBytes + value_piece<F>(j, d / 8u) * 16u + (d % 8u) * 2u;
                                const float v = __half2float(*reinterpret_cast<const __half*>(values_at + at));
                                if (!off[0]) o[m][n][x] = fmaf(w[0], v, o[m][n][x]);
                                if (!off[1]) o[m][n][2 + x] = fmaf(w[1], v, o[m][n][2 + x]);
                            }
                    }
                }
            }
            if (!F::Q8 && scalar) continue;

            // ---- weights × values: keys 2q, 2q+1, 2q+8, 2q+9; d/8 columns a lane --
            constexpr uint32_t kLaneBytes = F::kRowBytes / 8u;   // this lane's values of a row
            const uint32_t kr[4] = {2u * q, 2u * q + 1u, 2u * q + 8u, 2u * q + 9u};
            constexpr uint32_t kWordsPass = kLaneBytes >= 16u ? 4u : 2u;
#pragma unroll
            for (uint32_t j = 0; j < kLaneBytes / (4u * kWordsPass); ++j) {
                uint32_t vw[4][4];
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t r = kr[k];
                    if (kWordsPass == 4u) {
                        const uint32_t piece = g * (kLaneBytes / 16u) + j;
                        const uint4 v = *reinterpret_cast<const uint4*>(values_at + r * F::kRowBytes +
                                                                        value_piece<F>(r, piece) * 16u);
                        vw[k][0] = v.x; vw[k][1] = v.y; vw[k][2] = v.z; vw[k][3] = v.w;
                    } else {
                        const uint32_t byte = g * 8u;
                        const uint2 v = *reinterpret_cast<const uint2*>(
                            values_at + r * F::kRowBytes + value_piece<F>(r, byte / 16u) * 16u + byte % 16u);
                        vw[k][0] = v.x; vw[k][1] = v.y;
                    }
                }
#pragma unroll
                for (uint32_t w = 0; w < kWordsPass; ++w) {
                    constexpr uint32_t kPer = F::Q8 ? 4u : 2u;   // columns a word
                    const uint32_t n0 = (j * kWordsPass + w) * kPer;
                    uint32_t b[4][2];
                    if (F::Q8) {
                        const uint32_t x0 = __byte_perm(vw[0][w], vw[1][w], 0x5140), y0 = __byte_perm(vw[0][w], vw[1][w], 0x7362);
                        const uint32_t x1 = __byte_perm(vw[2][w], vw[3][w], 0x5140), y1 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
                        b[0][0] = codes2<0x4140>(x0); b[0][1] = codes2<0x4140>(x1);
                        b[1][0] = codes2<0x4342>(x0); b[1][1] = codes2<0x4342>(x1);
                        b[2][0] = codes2<0x4140>(y0); b[2][1] = codes2<0x4140>(y1);
                        b[3][0] = codes2<0x4342>(y0); b[3][1] = codes2<0x4342>(y1);
                    } else {
                        b[0][0] = __byte_perm(vw[0][w], vw[1][w], 0x5410); b[0][1] = __byte_perm(vw[2][w], vw[3][w], 0x5410);
                        b[1][0] = __byte_perm(vw[0][w], vw[1][w], 0x7632); b[1][1] = __byte_perm(vw[2][w], vw[3][w], 0x7632);
                        b[2][0] = b[2][1] = b[3][0] = b[3][1] = 0u;
                    }
#pragma unroll
                    for (uint32_t n = 0; n < kPer; ++n)
#pragma unroll
                        for (uint32_t m = 0; m < MT; ++m) {
                            mma(o[m][n0 + n], phi[m], b[n][0], b[n][1]);
                            mma(o[m][n0 + n], plo[m], b[n][0], b[n][1]);
                        }
                }
            }
        }
    };
    pass(false);
    if (!F::Q8) {
        bool fine = true;
#pragma unroll
        for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
            for (uint32_t n = 0; n < D / 8; ++n)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) fine &= fabsf(o[m][n][i]) < __builtin_huge_valf();
        if (!__all_sync(kAll, fine)) {
            copies_wait<0>();
            __syncwarp();
#pragma unroll
            for (uint32_t i = 0; i + 1u < F::S; ++i) {
                const uint32_t t = tile0 + warp + W * i;
                if (t < tile1) copy_tile(t, i);
                copies_commit();
            }
            pass(true);
        }
    }
    copies_wait<0>();

    // ---- the warps' states meet, a row tile at a time ------------------------------
    float* merge = reinterpret_cast<float*>(smem);
    float* merge_top = merge + W * 16u * F::kMergeRow;
    float* merge_sum = merge_top + W * 16u;
    float* merge_factor = merge_sum + W * 16u;
    const size_t pair = (static_cast<size_t>(s) * c.kv_heads + h) * args.row_groups + rg;
    float* partial = args.partials + (pair * args.parts + part) * F::kRows * (D + 2u);
    const bool whole = parts == 1u;
    const uint32_t rows = a.tokens * G;
#pragma unroll
    for (uint32_t m = 0; m < MT; ++m) {
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < 2; ++k) {
            const uint32_t r = warp * 16u + g + 8u * k;
            const float down = F::Q8 ? unit[m][k] / 16384.0f : 1.0f / 16384.0f;
            float t = sum[m][k];
            t += __shfl_xor_sync(kAll, t, 1);
            t += __shfl_xor_sync(kAll, t, 2);
            if (q == 0) {
                merge_top[r] = top[m][k];
                merge_sum[r] = t;
            }
            if (rg * F::kRows + m * 16u + g + 8u * k < rows)
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                for (uint32_t n = 0; n < D / 8; n += 4)
                    *reinterpret_cast<float4*>(merge + r * F::kMergeRow + 4u * merge_piece<F>((2u * q + x) * (D / 32u) + n / 4u)) =
                        make_float4(o[m][n][2 * k + x] * down, o[m][n + 1][2 * k + x] * down,
                                    o[m][n + 2][2 * k + x] * down, o[m][n + 3][2 * k + x] * down);
        }
        __syncthreads();
        const uint32_t row0 = rg * F::kRows + m * 16u, live = rows > row0 ? min(rows - row0, 16u) : 0u;   // rows of this tile
        if (threadIdx.x < W * 16u) {   // what a warp's state counts for in its row
            const uint32_t r = threadIdx.x % 16u;
            float t = kNegInf;
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) t = fmaxf(t, merge_top[w * 16u + r]);
            const float wt = merge_top[threadIdx.x], f = wt == kNegInf ? 0.0f : ex2(wt - t);
            // a warp that saw no visible key adds nothing, whatever it holds
            merge_factor[threadIdx.x] = wt == kNegInf && merge_sum[threadIdx.x] == 0.0f ? -1.0f : f;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < live * (D / 4u); i += W * 32u) {
            const uint32_t r = i / (D / 4u), col = i % (D / 4u);
            float l = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (uint32_t w = 0; w < W; ++w) {
                const float f = merge_factor[w * 16u + r];
                if (f < 0.0f) continue;
                const float4 v = *reinterpret_cast<const float4*>(merge + (w * 16u + r) * F::kMergeRow + 4u * merge_piece<F>(col));
                l = fmaf(merge_sum[w * 16u + r], f, l);
                acc.x = fmaf(v.x, f, acc.x);
                acc.y = fmaf(v.y, f, acc.y);
                acc.z = fmaf(v.z, f, acc.z);
                acc.w = fmaf(v.w, f, acc.w);
            }
            if (whole) {
                write_row(a, step, s, h, G, row0 + r, 4u * col, acc, l);
            } else {
                float* to = partial + (m * 16u + r) * D + 4u * col;
                __stcg(reinterpret_cast<float4*>(to), acc);
                if (col == 0) {
                    float t = kNegInf;
#pragma unroll
                    for (uint32_t w = 0; w < W; ++w) t = fmaxf(t, merge_top[w * 16u + r]);
                    __stcg(partial + F::kRows * D + m * 16u + r, t);
                    __stcg(partial + F::kRows * (D + 1u) + m * 16u + r, l);
                }
            }
        }
    }
    if (whole) return;

    // ---- the parts' states meet, in part order, in the last CTA to finish ----------
    __shared__ uint32_t is_last;
    __syncthreads();
    if (threadIdx.x == 0) {   // one thread's fences, for what the barriers order before and after them
        __threadfence();
        const unsigned int seen = atomicAdd(args.tickets + pair, 1u);
        is_last = seen == parts - 1u;
        if (is_last) {
            args.tickets[pair] = 0u;
            __threadfence();
        }
    }
    __syncthreads();
    if (!is_last) return;
    // Each part's factor for each row, then every output's sum over the parts:
    // by as many groups of threads as the outputs leave idle, each a run of the
    // parts, whose sums are added in run order. The first outputs are on their
    // way while the factors are found.
    const float* all = args.partials + pair * args.parts * F::kRows * (D + 2u);
    constexpr size_t kPart = F::kRows * (D + 2u);
    constexpr uint32_t kThreads = W * 32u, kAhead = 8;
    const uint32_t live = min(rows - rg * F::kRows, F::kRows), outputs = live * (D / 4u);
    float* weight = merge;                       // [parts][kRows], then the sums alike
    float* totals = weight + 2u * args.parts * F::kRows;
    float4* sums = reinterpret_cast<float4*>(totals + F::kRows);   // the runs' sums
    const uint32_t runs = max(min(kThreads / outputs, min(parts, 8u)), 1u), run = (parts + runs - 1u) / runs;
    const uint32_t mine_outputs = (runs * outputs + kThreads - 1u - threadIdx.x) / kThreads, items = mine_outputs * run;
    for (uint32_t i = threadIdx.x; i < parts * live; i += kThreads) {
        const uint32_t k = i / live, r = i % live;
        weight[k * F::kRows + r] = __ldcg(all + k * kPart + F::kRows * D + r);
        weight[(args.parts + k) * F::kRows + r] = __ldcg(all + k * kPart + F::kRows * (D + 1u) + r);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    // the next item: an output, and a part of its run. A thread has several
    // outputs only where there is one run
    const uint32_t part0 = threadIdx.x / outputs * run;
    uint32_t at_output = threadIdx.x % outputs, at_part = 0;
    for (uint32_t b = 0; b == 0 || b < items; b += kAhead) {
        float4 v[kAhead];
        uint32_t o_ = at_output, j = at_part;
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
            if (b + u < items && part0 + j < parts)
                v[u] = __ldcg(reinterpret_cast<const float4*>(all + (part0 + j) * kPart + 4u * o_));
            if (++j == run) {
                j = 0;
                o_ += kThreads;
            }
        }
        if (b == 0) {
            __syncthreads();
            for (uint32_t r = warp; r < live; r += W) {   // a warp a row, lanes its parts
                float t = kNegInf, l = 0.0f;
                for (uint32_t k = lane; k < parts; k += 32u) t = fmaxf(t, weight[k * F::kRows + r]);
#pragma unroll
                for (uint32_t x = 16; x > 0; x >>= 1) t = fmaxf(t, __shfl_xor_sync(kAll, t, x));
                for (uint32_t k = lane; k < parts; k += 32u) {
                    const float kt = weight[k * F::kRows + r], kl = weight[(args.parts + k) * F::kRows + r];
                    const bool none = kt == kNegInf && kl == 0.0f;   // a part that saw nothing of the row adds nothing
                    const float f = kt == kNegInf ? 0.0f : ex2(kt - t);
                    if (!none) l = fmaf(kl, f, l);
                    weight[k * F::kRows + r] = none ? -1.0f : f;
                }
#pragma unroll
                for (uint32_t x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(kAll, l, x);
                if (lane == 0) totals[r] = l;
            }
            __syncthreads();
        }
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
            if (b + u >= items) break;
            const uint32_t k = part0 + at_part, r = at_output / (D / 4u);
            if (k < parts) {
                const float f = weight[k * F::kRows + r];
                if (!(f < 0.0f)) {
                    acc.x = fmaf(v[u].x, f, acc.x);
                    acc.y = fmaf(v[u].y, f, acc.y);
                    acc.z = fmaf(v[u].z, f, acc.z);
                    acc.w = fmaf(v[u].w, f, acc.w);
                }
            }
            if (++at_part == run) {
                if (runs == 1u) write_row(a, step, s, h, G, rg * F::kRows + r, 4u * (at_output % (D / 4u)), acc, totals[r]);
                else sums[threadIdx.x] = acc;
                acc = make_float4(0.f, 0.f, 0.f, 0.f);
                at_part = 0;
                at_output += kThreads;
            }
        }
    }
    if (runs == 1u) return;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < outputs; i += W * 32u) {
        float4 total = sums[i];
        for (uint32_t k = 1; k < runs; ++k) {
            const float4 v = sums[k * outputs + i];
            total = make_float4(total.x + v.x, total.y + v.y, total.z + v.z, total.w + v.w);
        }
        write_row(a, step, s, h, G, rg * F::kRows + i / (D / 4u), 4u * (i % (D / 4u)), total, totals[i / (D / 4u)]);
    }
}

struct Shape {
    uint32_t row_groups, parts;
    uint64_t pairs, bytes;
};

template <class F>
Shape shape_of(const cb_tree_attention& a, uint32_t resident) {
    Shape x;
    const uint32_t rows = a.tokens * (a.query_heads / a.cache.kv_heads);
    x.row_groups = (rows + F::kRows - 1u) / F::kRows;
    x.pairs = static_cast<uint64_t>(a.sequences) * a.cache.kv_heads * x.row_groups;
    // as many parts as one wave holds, each of at least a tile a warp; or, of
    // long caches, so many that four waves even out sequences of different
    // lengths, each of at least eight tiles a warp
    uint64_t keys = a.max_keys < a.cache.slots ? a.max_keys : a.cache.slots;
    if (a.window && keys > static_cast<uint64_t>(a.window) + a.tokens) keys = static_cast<uint64_t>(a.window) + a.tokens;
    const uint64_t most = (keys + kKeys * F::W - 1u) / (kKeys * F::W);
    uint64_t parts = (resident < kTreeTickets ? resident : kTreeTickets) / x.pairs;
    if (parts > most) parts = most;
    uint64_t even = x.pairs <= kTreeTickets ? (4u * static_cast<uint64_t>(resident) + x.pairs - 1u) / x.pairs : 1u;
    if (even > most / 8u) even = most / 8u;
    if (parts < even) parts = even;
    const uint64_t room = (F::kWork - 16384u) / (F::kRows * 8u);   // the parts' factors and sums at the end
    if (parts > room) parts = room;
    // a few tiles a warp end before parts could meet (300 keys of 128 values 8.6
    // us against 9.2, 500 of 64 7.5 against 8.4; 600 of 128 12.5 against 12.0)
    if (most * F::D <= 512u) parts = 1;
    x.parts = parts ? static_cast<uint32_t>(parts) : 1u;
    x.bytes = kTreeTickets * 4ull + (x.parts > 1 ? x.pairs * x.parts * F::kRows * (F::D + 2u) * sizeof(float) : 0u);
    return x;
}

template <class F>
int resident_ctas() {   // on the whole current device, of this form; 0 on an error
    constexpr int kDevices = 64;
    static int count[kDevices] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= kDevices) return 0;
    if (count[device] == 0) {
        auto kernel = tree_attention_kernel<F>;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(F::kSmem)) != cudaSuccess)
            return 0;
        int per = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, F::W * 32, F::kSmem) != cudaSuccess) return 0;
        const int sms = sm_count();
        count[device] = per * (sms > 0 ? sms : 0);
    }
    return count[device];
}

template <class F>
cudaError_t launch_form(const cb_tree_attention& a, cudaStream_t stream, bool pdl) {
    const int resident = resident_ctas<F>();
    if (resident <= 0) return cudaErrorInvalidConfiguration;
    const Shape x = shape_of<F>(a, static_cast<uint32_t>(resident));
    TreeArgs args{a, a.query_heads / a.cache.kv_heads, x.row_groups, x.parts,
                  static_cast<unsigned int*>(a.workspace),
                  reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kTreeTickets * 4u)};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(x.parts, a.cache.kv_heads * x.row_groups, a.sequences);
    cfg.blockDim = dim3(F::W * 32);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, tree_attention_kernel<F>, args);
}

// Calls f with the form of these sizes.
template <class Fn>
auto with_form(const cb_tree_attention& a, Fn&& f) {
    const bool q8 = a.cache.format == CB_CACHE_Q8;
    const uint32_t rows = a.tokens * (a.query_heads / a.cache.kv_heads);
    switch (a.cache.head_dim) {
        case 64:
            if (q8) return rows <= 16 ? f(Form<64, true, 1, 8, 4>{}) : f(Form<64, true, 2, 8, 4>{});
            return rows <= 16 ? f(Form<64, false, 1, 8, 3>{}) : f(Form<64, false, 2, 8, 3>{});
        case 128:
            if (q8) return rows <= 16 ? f(Form<128, true, 1, 8, 3>{}) : f(Form<128, true, 2, 8, 3>{});
            return rows <= 16 ? f(Form<128, false, 1, 4, 3>{}) : f(Form<128, false, 2, 4, 3>{});
        default:
            return q8 ? f(Form<256, true, 1, 8, 3>{}) : f(Form<256, false, 1, 4, 3>{});
    }
}

}  // namespace

uint64_t tree_attention_bytes(const cb_tree_attention& a) {   // of either form
    const uint64_t own = with_form(a, [&](auto form) -> uint64_t {
        using F = decltype(form);
        const int resident = resident_ctas<F>();
        return resident > 0 ? shape_of<F>(a, static_cast<uint32_t>(resident)).bytes : 0u;
    });
    const uint64_t tensor = own && tree_attention_tensor_fits(a) ? tree_attention_tensor_bytes(a) : 0u;
    return own > tensor ? own : tensor;
}

cudaError_t tree_attention_run(const cb_tree_attention& a, cudaStream_t stream, bool pdl, bool tensor) {
    if (tree_attention_tensor_fits(a) && (tensor || tree_attention_tensor_pays(a))) return tree_attention_tensor_run(a, stream, pdl);
    return with_form(a, [&](auto form) { return launch_form<decltype(form)>(a, stream, pdl); });
}

}  // namespace cb
