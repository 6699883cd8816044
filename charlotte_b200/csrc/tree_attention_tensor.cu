// Tree attention on the 5th-generation tensor cores: the form for large steps
// of many rows a kv head (tree_attention.cu states the mathematics and has the
// form for the others).
//
// Products. A tile is 128 keys. S^T = K·Q^T puts a key on each of the 128
// accumulator lanes and a row in each column; the queries' lo terms are
// multiplied first and the hi terms added to them, in the same columns. O = P·V
// puts the rows on the lanes (hi terms in lanes 0–63, lo terms in lanes 64–127)
// and the head dimension in the columns; its two halves are added once, at the
// end. Both products are 128 lanes wide whatever the row count, so rows up to
// 64 fill what a 128-lane product computes anyway.
//
// A key being a lane, its scale is a number of the thread that holds it, and
// a row's maximum runs across lanes. It is not found for every tile: the
// weights are taken against a base, and their products with the scales
// against a unit, that only have to keep them in f16's range, and both are
// raised (with the sums) when some p passes the base, or some p·scale the
// unit, by 2^8.
// Otherwise a tile costs one barrier-with-or of the eight warps of each half
// of the rows.
//
// Work. Every CTA stays resident (one an SM) and takes an equal share of all
// (sequence, kv head, row group) pairs' tiles laid end to end, whatever the
// sequences' lengths; a pair that falls to several CTAs is added up in CTA
// order by the last to finish. S of the next two tiles runs under a tile's
// softmax. An f16 cache's whole tiles are copied straight into the operands;
// codes land in a ring and are made f16 by warps of their own.
//
// Bound. 32 trees of 32 nodes (64 rows a kv head of 128 values) over 8-bit
// contexts of 16k to 32k keys: 620 to 710 us as the clocks go, that is 1.58
// GB at 2.2 to 2.5 TB/s and 377 GFLOP of both terms at 530 to 610 TFLOP/s, 2 us a
// tile. Nothing is full: the issue slots half, the tensor pipe a quarter, and
// shared memory, whose 320 KB a tile (160 that the products read, 64 rows being
// few for keys that are read once a term, 32 of weights, 128 for codes to
// arrive and become f16) are 2,500 cycles at 128 bytes, 1.3 us of the 2. The rest
// is a chain that waits: with one stage of operands a tile's codes become f16
// only once the products of the tile before are done with theirs, and the
// softmax's warps all stand at one tile and its vote.
// With f16 rows of 64 values (8 trees of 96 rows over 4k to 8k keys, 83 to 87 us) a tile is the
// softmax's own chain, 1.5 us of waits, conversions and stores, and beginning
// and ending a share takes 15 us.
// Measured and not kept: the two terms side by side in S's columns (a sum more
// a score); the two halves of the rows taking turns (5 % slower); the vote on
// raising the bases read after the weights, which are made again when it
// comes (-2 to +8 %: registers spill).
//
// Shared-memory operands. A key row's d values lie in 64-value pieces, eight
// keys a 1,024-byte swizzle atom, atoms of the same piece along the keys: read
// along d (K-major) they are K·Q^T's A, read along the keys (MN-major) P·V's
// B. P is written key by key, a lane its key's weights: MN-major A.
//
// Every wait is bounded: one that runs out sets the fault word (which
// cb_fault_check reports) and `abort`, after which the other waits run out too
// and the kernel runs to its end with whatever it has.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "api_common.h"
#include "cache.cuh"
#include "kernels.h"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "tree_attention.cuh"

namespace cb {

namespace {

constexpr uint32_t kTile = 128;                 // keys
// Warps: of softmax (four to each group of rows), of loading (half of them
// keys, half values, so that neither waits for the other's space), and one that
// issues the products. Little of a role's loop may spill: the shared memory
// taken leaves the L1 little, and a spilled word may come back from L2 (600
// cycles). 800 threads leave each 72 registers: the softmax keeps 4 to 28 bytes
// in local memory, for 64 rows over f16 rows of 64 values 80, of 128 values 148.
constexpr uint32_t kSoftWarps = 16, kLoadWarps = 8, kThreads = 32 * (kSoftWarps + kLoadWarps + 1);
constexpr uint32_t kGroups = kSoftWarps / 4, kHalfThreads = kSoftWarps * 16, kColumnParts = kGroups / 2;
constexpr uint32_t kPrefetch = 2;               // tiles brought to L2 ahead of the loads
// Tiles whose products are summed in one accumulator. The tensor cores cut each
// of a tile's eight sums short instead of rounding it, always towards zero: over
// 300 tiles 4e-6 of the result. In runs of kFold tiles, added up in f32, it is
// 5e-7 (in runs of 8 3e-7, of 24 7e-7, of 48 1.3e-6; four times that where few
// keys have most of the weight); a run's end takes 1.3 us.
constexpr uint32_t kFold = 16;
constexpr uint32_t kBegin = 6;                  // tiles' time that beginning a pair takes, for the shares
constexpr uint32_t kPiece = kTile * 128;        // bytes of a tile's 64-value piece
constexpr uint32_t kMostSequences = 1024;
constexpr uint32_t kScaleTiles = 8;             // tiles whose scales are held: copies run at most six ahead of the softmax
constexpr uint32_t kPolls = 1u << 20;           // of a wait: a large fraction of a second at least
constexpr float kRise = 8.0f;                   // log2 units a weight may pass its base by
constexpr float kWeightTop = 128.0f;            // 2^15 / 2^kRise: a weight whose p·scale is its row's unit
constexpr float kLeastUnit = -100.0f;           // log2

template <uint32_t D_, bool Q8_, uint32_t RT_>
struct Form {
    static constexpr uint32_t D = D_, RT = RT_;
    static constexpr bool Q8 = Q8_;
    static constexpr uint32_t N = 2 * RT;                       // query rows held: the hi terms, then the lo
    static constexpr uint32_t RH = RT / kGroups;                // rows of a group's softmax warps
    // Eight-bit rows wait in a ring of whole tiles (head dimension 256 has no
    // room for one: its codes wait in registers); the operands they become then
    // need one buffer each, an f16 cache's own copies two.
    static constexpr uint32_t kRing = Q8 && D <= 128 ? 2 : 0;   // tiles
    static constexpr uint32_t kStages = D == 256 || (Q8 && D == 128) ? 1 : 2;   // of keys, of values
    static constexpr uint32_t kWeights = D == 64 ? 2 : 1;         // P buffers
    // TMEM columns: S's two buffers, O, and what has been folded out of O: as wide
    // as O, or for 256 values half as wide, columns 128 .. on the lanes 16 .. that
    // rows of 16 a quadrant leave.
    static constexpr uint32_t kSumsAt = 256, kFoldedAt = D == 256 ? 64 : 256 + D, kFoldedWide = D == 256 ? 128 : D;
    static_assert(kFoldedAt + kFoldedWide <= (D == 256 ? 256 : 512) && 2 * RT <= (D == 256 ? kFoldedAt : 256), "columns");
    static_assert(D < 256 || RT == 32, "the upper lanes are free");
    static constexpr uint32_t kOperand = kTile * D * 2;         // a tile's keys or values as f16
    static constexpr uint32_t kQuery = N * D * 2;
    static constexpr uint32_t kP = 2 * kPiece;
    static constexpr uint32_t kKeysAt = kQuery, kValuesAt = kKeysAt + kStages * kOperand;
    static constexpr uint32_t kPAt = kValuesAt + kStages * kOperand;
    static constexpr uint32_t kRingAt = kPAt + kWeights * kP;
    static constexpr uint32_t kInfoAt = kRingAt + kRing * 2 * kTile * D;
    static constexpr uint32_t kOut = D + 4;                     // floats of an output row on its way out
    // At a stretch's end its output rows pass through the operands' space, and
    // after them lie the factors of a pair's parts, one a CTA at most.
    static constexpr uint32_t kFactorAt = kKeysAt + (RT * kOut * 4 + 127) / 128 * 128;
    static constexpr uint32_t kMostCtas = (kInfoAt - kFactorAt) / (RT * 4);
};

// A stretch of one pair's tiles, as the roles need it.
struct Stretch {
    const char* keys_rows;     // the head's rows of the sequence
    const char* values;
    const float* key_scales;
    const float* value_scales;
    size_t entry;              // bytes from an entry's row to the next's
    uint32_t slots, first_slot, first, length, keys;
    uint32_t tile0, n;         // tiles tile0 .. tile0 + n − 1
    uint32_t done;             // tiles this CTA has put through before: every role counts the same
    const CUtensorMap* keys_map;   // of the caches' rows; NULL: none
    const CUtensorMap* values_map;
    uint32_t s, h;
};

struct Info {
    Stretch on;
    unsigned int* fault;
    __align__(16) float factor[64], base[64];   // a row's score factor, and its base, negated
    __align__(16) float weight[64];             // its weight factor (0: no row of the step)
    uint32_t top[64];          // its query's largest magnitude (bits)
    bool even_factor, even_weight[2];   // every row's (of a half) is the same
    uint64_t mask[64];
    uint32_t first[64];
    float unit[64];            // log2 of the power of two the row's p·scale are held against
    __align__(8) float shift[64], sums[64];   // what a raised base adds to scores, makes of sums
    float outs[64];                           // and of outputs
    int found[4][64];          // a quadrant's largest score, ordered as an integer
    int weighty[4][64];        // and its largest log2 of p·scale, likewise
    float total[4][64];
    uint32_t unset[2];         // a half's live rows that have seen no key yet
    float least_unit[2];       // of the rows that have (log2)
    uint32_t latest, context;  // tiles from one to before the other are seen whole by every row
    uint32_t last, abort, polls, tmem;
    uint32_t first_cta, last_cta;   // of a divided pair
    bool begins;                    // whether its tiles begin inside the first one's share
    float2 scales[kScaleTiles][kTile];   // an 8-bit tile's key and value scales
    uint32_t before[kMostSequences + 1];   // tiles of all pairs of the sequences before
    uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], sempty[2], pfull[2], pempty[2];
    uint64_t rfull[2][2], rempty[2][2];   // the rings of codes, of keys and of values
};

struct TensorArgs {
    cb_tree_attention a;
    uint32_t groups, row_groups;
    unsigned int* tickets;     // a word for each CTA that begins a divided pair
    float* partials;           // two a CTA: [RT][D], then [RT] bases, [RT] sums
    unsigned int* fault;
    uint32_t maps;             // whether the maps are given
};

__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {   // MN-major, 128-byte swizzle, 64-value atoms a piece apart
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(kPiece >> 4) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// 128 rows of a head (from column x) by one copy, completing on `bar`.
__device__ __forceinline__ void copy_tile(void* to, const CUtensorMap* map, uint32_t x, uint32_t h, uint32_t slot, uint32_t s, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(to)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(h), "r"(slot), "r"(s), "r"(smem_addr(bar))
        : "memory");
}

// Byte of 16-byte chunk `c` (8 values) of row `r` within a piece.
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c) {
    return (r >> 3) * 1024u + (r & 7u) * 128u + ((c ^ (r & 7u)) << 4);
}

// 8 or 16 f32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[8]) {
    uint32_t r[8];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const float (&v)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n\t"
        "tcgen05.wait::st.sync.aligned;" ::"r"(taddr),
        "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
        : "memory");
}

// The softmax warps of a half of the rows: a barrier, and one that
// tells whether any thread said so.
__device__ __forceinline__ void half_sync(uint32_t half) { asm volatile("bar.sync %0, %1;" ::"r"(1u + half), "n"(kHalfThreads) : "memory"); }
__device__ __forceinline__ bool half_any(uint32_t half, bool p) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(p)), "r"(1u + half), "n"(kHalfThreads)
        : "memory");
    return r != 0;
}

// A wait never changes where a thread goes next, so that the barriers of whole
// warps stay matched whatever runs out. It is looked at (`sound`) before the
// arrivals that stand on it: those on a barrier that counts a copy's bytes,
// which must not come before its phase is done, and the commits that let the
// loaders on.
__device__ __forceinline__ void ran_out(Info& info) {
    *reinterpret_cast<volatile uint32_t*>(&info.abort) = 1u;
    if (info.fault) atomicOr(info.fault, kFaultTimeout);
}
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, Info& info) {
#pragma unroll 1
    for (uint32_t i = 0; i < kPolls; ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if (i % 16u == 15u) {
            if (*reinterpret_cast<volatile uint32_t*>(&info.abort)) return;
            if (i >= info.polls) break;
        }
    }
    ran_out(info);
}
// Whether every wait of the CTA was met so far, this thread's own among them.
__device__ __forceinline__ bool sound(const Info& info) { return *reinterpret_cast<const volatile uint32_t*>(&info.abort) == 0u; }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ int ordered(float v) {   // −∞ and NaN lowest
    const int b = __float_as_int(v);
    return v == v ? b ^ ((b >> 31) & 0x7FFFFFFF) : static_cast<int>(0x80000000u);
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7FFFFFFF)); }

// Where row r's hi-term weights lie on the output's lanes (its lo-term's: 64
// on): each half of the rows in a quadrant of its own.
template <class F>
__device__ __forceinline__ uint32_t output_lane(uint32_t r) { return r / (F::RT / 2) * 32u + r % (F::RT / 2); }

// The rows that see entry e (bit r).
template <class F>
__device__ __noinline__ uint64_t sight_of(const Info& info, uint32_t e) {
    const uint32_t length = info.on.length;
    uint64_t sight = 0;
    if (e < info.on.first + info.on.keys) {
        if (e < length) {
#pragma unroll 4
            for (uint32_t r = 0; r < F::RT; ++r) sight |= static_cast<uint64_t>(e >= info.first[r]) << r;
        } else {
#pragma unroll 4
            for (uint32_t r = 0; r < F::RT; ++r) sight |= (info.mask[r] >> (e - length) & 1ull) << r;
        }
    }
    return sight;
}

// 2^x of a whole number up to 127; 0 below −126.
__device__ __forceinline__ float exp2i(float x) { return __uint_as_float(static_cast<uint32_t>(max(static_cast<int>(x), -127) + 127) << 23); }
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One warp of a half: from the tile's largest scores and p·scale, each row's
// new base and unit, and what they make of what it has (info.shift, sums,
// outs). A lane a row.
template <class F>
__device__ __forceinline__ void raise_bases(Info& info, uint32_t half, uint32_t lane) {
    constexpr uint32_t kRows = F::RT / 2;
    const uint32_t r = half * kRows + lane % kRows;
    const bool mine = lane < kRows;
    int v = info.found[0][r], w = F::Q8 ? info.weighty[0][r] : 0;
#pragma unroll
    for (int k = 1; k < 4; ++k) {
        v = max(v, info.found[k][r]);
        if (F::Q8) w = max(w, info.weighty[k][r]);
    }
    const float top = unordered(v);   // relative to the base; ordered(NaN) is below −∞'s
    const bool unset = info.unset[half] >> (lane % kRows) & 1u;
    float shift = 0.0f, keep = 1.0f;
    if (top > kNegInf && (unset || top > 0.0f)) {
        shift = top;
        if (!unset) keep = ex2(-top);
    }
    const bool set = mine && info.weight[r] != 0.0f && (!unset || top > kNegInf);
    const float was = info.unit[r];
    float now = 0.0f;
    bool even = true;
    if (F::Q8) {
        // The unit falls with the sums when the base rises, and is raised to the tile's largest p·scale.
        const float heaviest = unordered(w) - shift;
        now = unset ? kLeastUnit : fmaxf(ceilf(was - shift), kLeastUnit);
        if (heaviest > now) now = fminf(ceilf(heaviest), 126.0f);   // kWeightTop over it stays a normal number
        // one unit for all rows where theirs are within 2^6 of each other
        const int most = __reduce_max_sync(kAllLanes, set ? static_cast<int>(now) : -1000);
        const int least = __reduce_min_sync(kAllLanes, set ? static_cast<int>(now) : 1000);
        even = most - least <= 6;   // or no row is set
        if (even && most > -1000) now = static_cast<float>(most);
        if (lane == 0) info.least_unit[half] = static_cast<float>(most == -1000 ? static_cast<int>(kLeastUnit) : even ? most : least);
    }
    const uint32_t now_set = __ballot_sync(kAllLanes, set);
    if (mine) {
        info.shift[r] = -shift;
        info.sums[r] = keep;
        info.base[r] -= shift;
        // nothing was summed of an unset row; else now >= was − shift, so that this is at most 1
        info.outs[r] = F::Q8 ? (unset || keep == 0.0f ? keep : keep * exp2i(was - now)) : keep;
        info.unit[r] = now;
        if (F::Q8 && info.weight[r] != 0.0f) info.weight[r] = kWeightTop * exp2i(-now);
    }
    __syncwarp();
    if (lane == 0) {
        info.unset[half] &= ~now_set;
        info.even_weight[half] = even;
    }
}

// New bases for the rows of a half, by all its warps: each row's largest score
// and p·scale of the tile, then scores, sums and the outputs so far moved
// to the new bases and units. `it`: the tile's number, `after` whether the
// stretch has products before it. In line and without a call, so that what
// the loop holds stays in registers.
template <class F>
__device__ __forceinline__ void raise_all(Info& info, float (&e)[F::RH], float (&sum)[F::RH], float scale, uint32_t it,
                                          bool after, bool folded, uint32_t lanes) {
    constexpr uint32_t D = F::D, RT = F::RT, RH = F::RH;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, group = warp >> 2, quad = warp & 3u, half = group / kColumnParts;
    const uint32_t r0 = group * RH;
    const float log_scale = F::Q8 && scale > 0.0f && scale < __builtin_huge_valf() ? lg2(scale) : kNegInf;
#pragma unroll
    for (uint32_t i = 0; i < RH; ++i) {
        const int v = __reduce_max_sync(kAllLanes, ordered(e[i]));
        if (lane == 0) info.found[quad][r0 + i] = v;
        if (F::Q8) {
            const int w = __reduce_max_sync(kAllLanes, ordered(e[i] + log_scale));
            if (lane == 0) info.weighty[quad][r0 + i] = w;
        }
    }
    half_sync(half);
    if (warp % (kSoftWarps / 2u) == 0) raise_bases<F>(info, half, lane);
    half_sync(half);
#pragma unroll
    for (uint32_t i = 0; i < RH; ++i) {
        e[i] += info.shift[r0 + i];
        sum[i] *= info.sums[r0 + i];
    }
    if (!after) return;
    // the outputs so far, once the last product into them is done
    wait(&info.pempty[(it - 1u) % F::kWeights], (it - 1u) / F::kWeights & 1u, info);
    tc_fence_after();
    // this half's rows lie in two of the four quadrants (`output_lane`)
    if (quad % 2u == half) {
        const float f = info.outs[half * (RT / 2) + lane % (RT / 2)];
#pragma unroll 1
        for (uint32_t d = 0; d < D / kColumnParts; d += 8u) {
            float v[8];
            tmem_ld(lanes + F::kSumsAt + group % kColumnParts * (D / kColumnParts) + d, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= f;
            tmem_st(lanes + F::kSumsAt + group % kColumnParts * (D / kColumnParts) + d, v);
        }
        if (folded) {
            constexpr uint32_t kWide = F::kFoldedWide / kColumnParts;
#pragma unroll 1
            for (uint32_t d = 0; d < kWide; d += 8u) {
                float v[8];
                tmem_ld(lanes + F::kFoldedAt + group % kColumnParts * kWide + d, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= f;
                tmem_st(lanes + F::kFoldedAt + group % kColumnParts * kWide + d, v);
            }
        }
    }
    tc_fence_before();
}

// The products of the tiles before number `it`, added to those folded before
// them (`more`: there are some) by the same warps that raise_all moves them
// with; the next tile's product begins at zero.
template <class F>
__device__ __forceinline__ void fold(Info& info, uint32_t it, bool more, uint32_t lanes) {
    constexpr uint32_t kWide = F::kFoldedWide / kColumnParts;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, group = warp >> 2, quad = warp & 3u, half = group / kColumnParts;
    wait(&info.pempty[(it - 1u) % F::kWeights], (it - 1u) / F::kWeights & 1u, info);
    tc_fence_after();
    if (quad % 2u == half) {
#pragma unroll 1
        for (uint32_t d = group % kColumnParts * kWide; d < (group % kColumnParts + 1u) * kWide; d += 8u) {
            float v[8], m[8];
            tmem_ld(lanes + F::kSumsAt + d, v);
            if constexpr (F::D == 256) {
                tmem_ld(lanes + F::kSumsAt + 128u + d, m);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float high = __shfl_xor_sync(kAllLanes, m[j], 16);
                    if (lane >= 16u) v[j] = high;
                }
            }
            if (more) {
                tmem_ld(lanes + F::kFoldedAt + d, m);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += m[j];
            }
            tmem_st(lanes + F::kFoldedAt + d, v);
        }
    }
    tc_fence_before();
}

// S of tile number `it` of this CTA, and its P·V, issued by one warp: each
// waits for what it reads, and for the space it writes.
template <class F>
__device__ __forceinline__ void issue_scores(Info& info, uint32_t base, uint32_t tmem, uint32_t it, uint32_t lane) {
    const uint32_t st = it % F::kStages, sb = it & 1u;
    wait(&info.kfull[st], it / F::kStages & 1u, info);
    wait(&info.sempty[sb], (it >> 1 & 1u) ^ 1u, info);
    tc_fence_after();
    if (lane == 0) {
        const bool go = sound(info);
        asm volatile("" : "+r"(base));   // descriptors are made here, not kept in registers through the softmax
        const uint64_t da = umma_desc_sw128(base + F::kKeysAt + st * F::kOperand), db = umma_desc_sw128(base);
#pragma unroll
        for (uint32_t term = 0; term < 2; ++term)   // lo first: its small sums take the roundings
#pragma unroll
            for (uint32_t k = 0; k < F::D / 16u; ++k)
                umma_f16(tmem + sb * F::RT, da + k / 4u * (kPiece >> 4) + k % 4u * 2u,
                         db + (1u - term) * (F::RT * 128u >> 4) + k / 4u * (F::N * 128u >> 4) + k % 4u * 2u,
                         umma_idesc_f16(kTile, F::RT), term + k > 0);
        if (go) {
            umma_commit(&info.kempty[st]);
            umma_commit(&info.sfull[sb]);
        }
    }
    __syncwarp();
}
template <class F>
__device__ __forceinline__ void issue_sums(Info& info, uint32_t base, uint32_t tmem, uint32_t it, uint32_t first, uint32_t lane) {
    constexpr uint32_t kBothMn = 1u << 15 | 1u << 16;   // both operands MN-major
    const uint32_t st = it % F::kStages, pb = it % F::kWeights;
    wait(&info.vfull[st], it / F::kStages & 1u, info);
    wait(&info.pfull[pb], it / F::kWeights & 1u, info);
    tc_fence_after();
    if (lane == 0) {
        const bool go = sound(info);
        asm volatile("" : "+r"(base));
        const uint64_t da = desc_mn(base + F::kPAt + pb * F::kP), db = desc_mn(base + F::kValuesAt + st * F::kOperand);
#pragma unroll
        for (uint32_t k = 0; k < kTile / 16u; ++k)
            umma_f16(tmem + F::kSumsAt, da + k * (2048u >> 4), db + k * (2048u >> 4), umma_idesc_f16(128, F::D) | kBothMn,
                     (it - first) % kFold != 0 || k > 0);
        if (go) {
            umma_commit(&info.vempty[st]);
            umma_commit(&info.pempty[pb]);
        }
    }
    __syncwarp();
}

// The softmax warps' part of a stretch: thread = key lane; each group's
// warps take the rows r0 .. r0 + RH − 1. The two halves of the rows meet only
// in P·V: each has its own bases.
template <class F>
__device__ __noinline__ void soften(Info& info, char* smem, uint32_t tmem) {
    constexpr uint32_t D = F::D, RT = F::RT, RH = F::RH;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, group = warp >> 2, quad = warp & 3u, half = group / kColumnParts,
                   key = quad * 32u + lane, r0 = group * RH;
    const uint32_t lanes = tmem + ((quad * 32u) << 16);
    const Stretch& on = info.on;
    const uint32_t n = on.n, done = on.done, first = on.first + on.tile0 * kTile;
    const bool even_factor = info.even_factor;
    float sum[RH];
#pragma unroll
    for (uint32_t i = 0; i < RH; ++i) sum[i] = 0.0f;
    for (uint32_t t = 0; t < n; ++t) {
        const uint32_t it = done + t, sb = it & 1u;
        const uint32_t e0 = first + t * kTile;
        const bool plain = e0 >= info.latest && e0 + kTile <= info.context;
        const uint64_t sight = plain ? ~0ull : sight_of<F>(info, e0 + key);   // the rows that see this thread's key
        const uint32_t mine = static_cast<uint32_t>(sight >> r0);   // this group's rows
        if (t > 0 && t % kFold == 0) fold<F>(info, it, t > kFold, lanes);
        wait(&info.sfull[sb], it >> 1 & 1u, info);
        tc_fence_after();
        const float2 scale = F::Q8 ? info.scales[it % kScaleTiles][key] : make_float2(1.0f, 1.0f);
        float e[RH];   // scores less their bases
        tmem_ld(lanes + sb * RT + r0, e);
        const float both = scale.x * info.factor[0];
#pragma unroll
        for (uint32_t j = 0; j < RH; j += 4) {
            const float4 base = *reinterpret_cast<const float4*>(&info.base[r0 + j]);
            float4 f = make_float4(both, both, both, both);
            if (!even_factor) {
                f = *reinterpret_cast<const float4*>(&info.factor[r0 + j]);
                f = make_float4(scale.x * f.x, scale.x * f.y, scale.x * f.z, scale.x * f.w);
            }
            e[j] = fmaf(e[j], f.x, base.x);
            e[j + 1] = fmaf(e[j + 1], f.y, base.y);
            e[j + 2] = fmaf(e[j + 2], f.z, base.z);
            e[j + 3] = fmaf(e[j + 3], f.w, base.w);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&info.sempty[sb]);
        if (!plain) {
#pragma unroll
            for (uint32_t j = 0; j < RH; ++j)
                if (!(mine >> j & 1u)) e[j] = kNegInf;
        }
        const uint32_t half_sight = static_cast<uint32_t>(sight >> (half * (RT / 2)));
        float most[2] = {kNegInf, kNegInf};
#pragma unroll
        for (uint32_t j = 0; j < RH; j += 2) most[j / 2 % 2] = max3(most[j / 2 % 2], e[j], e[j + 1]);
        // p may pass its base, and p·scale its row's unit, by 2^kRise
        float past = 0.0f;   // log2 of the scale over the least unit
        if (F::Q8 && scale.y < __builtin_huge_valf()) past = fmaxf(lg2(scale.y) - info.least_unit[half], 0.0f);
        bool raise = fmaxf(most[0], most[1]) + past > kRise;
        raise |= (info.unset[half] & half_sight) != 0;
        if (half_any(half, raise)) raise_all<F>(info, e, sum, scale.y, it, t > 0, t >= kFold, lanes);   // rare
        const uint32_t pb = it % F::kWeights;
        wait(&info.pempty[pb], (it / F::kWeights & 1u) ^ 1u, info);
        char* to = smem + F::kPAt + pb * F::kP;
        // p = 2^e, added to its row's sum; its weight p·scale·factor in two terms.
        const float down = scale.y * info.weight[half * (RT / 2)];
        // every key seen, one weight factor, and one that does not pass f32's range where p·scale does not
        const bool simple = plain && info.even_weight[half] && (!F::Q8 || down < __builtin_huge_valf());
#pragma unroll
        for (uint32_t i = 0; i < RH; i += 8) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (uint32_t j = 0; j < 8; j += 2) {
                float w[2];
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                    const float p = ex2(e[i + j + k]);
                    sum[i + j + k] += p;
                    w[k] = p * down;
                    if (!simple) {
                        w[k] = p * scale.y * info.weight[r0 + i + j + k];
                        if (!(mine >> (i + j + k) & 1u)) w[k] = 0.0f;   // a hidden key's scale may be anything
                    }
                }
                split2(w[0], w[1], hi[j / 2], lo[j / 2]);
            }
            const uint32_t chunk = swizzled(key, output_lane<F>(r0 + i) / 8u);
            *reinterpret_cast<uint4*>(to + chunk) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(to + kPiece + chunk) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&info.pfull[pb]);
    }
    // ---- the sums: a row's 128 lanes to one -------------------------------
#pragma unroll
    for (uint32_t w = 16; w >= RH; w >>= 1) {
#pragma unroll
        for (uint32_t i = 0; i < RH; ++i) sum[i] += __shfl_xor_sync(kAllLanes, sum[i], w);
    }
#pragma unroll
    for (uint32_t w = RH / 2u; w > 0; w >>= 1) {
#pragma unroll
        for (uint32_t i = 0; i < w; ++i) {
            const bool up = lane & w;
            const float keep = up ? sum[i + w] : sum[i], send = up ? sum[i] : sum[i + w];
            sum[i] = keep + __shfl_xor_sync(kAllLanes, send, w);
        }
    }
    if (lane < RH) info.total[quad][r0 + lane] = sum[0];
}

// The issuing warp's part: S runs two tiles ahead, each in the buffer of the
// tile two before, which its softmax frees before it has its weights.
template <class F>
__device__ __noinline__ void multiply(Info& info, char* smem, uint32_t tmem) {
    const uint32_t lane = threadIdx.x & 31u, base = smem_addr(smem), n = info.on.n, done = info.on.done;
    if (info.polls == 0u) ran_out(info);   // a wait given no poll at all
    for (uint32_t t = 0; t < n; ++t) {
        issue_scores<F>(info, base, tmem, done + t, lane);
        if (t > 1u) issue_sums<F>(info, base, tmem, done + t - 2u, done, lane);
    }
    if (n > 1u) issue_sums<F>(info, base, tmem, done + n - 2u, done, lane);
    issue_sums<F>(info, base, tmem, done + n - 1u, done, lane);
}

// The loading warps': the tiles' keys (the first half of the warps) and
// values (the second) as f16 operands.
template <class F>
__device__ __noinline__ void bring(Info& info, char* smem) {
    constexpr uint32_t D = F::D;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    // ---- the tiles' keys, or values, as f16 operands ----------------------
    constexpr uint32_t kWarps = kLoadWarps / 2u;
    const uint32_t w = (warp - kSoftWarps) % kWarps;
    const bool value = warp - kSoftWarps >= kWarps;
    uint64_t* const full = value ? info.vfull : info.kfull;
    uint64_t* const empty = value ? info.vempty : info.kempty;
    char* const operand = smem + (value ? F::kValuesAt : F::kKeysAt);
    const Stretch& on = info.on;
    const uint32_t n = on.n, done = on.done, keys = on.keys, slots = on.slots, first_slot = on.first_slot, at0 = on.tile0 * kTile;
    constexpr uint32_t kElement = F::Q8 ? 1u : 2u;
    const size_t entry = on.entry;
    const char* const head_rows = value ? on.values : on.keys_rows;
    // Eight keys by four 16-byte pieces of a row a warp instruction:
    // 64 consecutive bytes a key, and swizzled chunks of eight keys on
    // distinct banks.
    const uint32_t sub = lane & 7u, piece4 = lane >> 3;
    constexpr uint32_t kQuads = D * kElement / 64u;   // 64-byte pieces of a row
    static_assert(16u * kQuads % kWarps == 0u, "every warp loads as much");
    constexpr uint32_t kEach = 16u * kQuads / kWarps;                                 // warp loads of a tile, of this warp
    constexpr uint32_t kSub = kQuads > kWarps ? kQuads / kWarps : 1u;                 // to a group of eight keys
    constexpr uint32_t kStep = kQuads > kWarps ? 8u : 8u * kWarps / kQuads;           // keys from one group to the next
    const uint32_t key0 = (kQuads > kWarps ? 0u : w / kQuads * 8u) + sub, piece0 = w % kQuads * 4u + piece4;
    auto place = [&](uint32_t i, uint32_t& key, uint32_t& piece) {
        key = key0 + i / kSub * kStep;
        piece = piece0 + i % kSub * (4u * kWarps);
    };
    // A tile that is whole and does not wrap comes by one copy; any other's
    // rows in turn: f(i, source, there).
    const CUtensorMap* const map = value ? on.values_map : on.keys_map;
    auto slot_at = [&](uint32_t i) {
        const uint32_t slot = first_slot + i;
        return slot >= slots ? slot - slots : slot;
    };
    auto whole = [&](uint32_t t) {
        const uint32_t k0 = at0 + t * kTile, slot = first_slot + k0;
        return map && k0 + kTile <= keys && (slot >= slots || slot + kTile <= slots);
    };
    auto each = [&](uint32_t t, uint32_t i0, uint32_t count, auto&& f) {
#pragma unroll
        for (uint32_t i = 0; i < count; ++i) {
            uint32_t key, piece;
            place(i0 + i, key, piece);
            const uint32_t k = at0 + t * kTile + key;
            const bool there = t < n && k < keys;
            f(i, head_rows + slot_at(there ? k : 0u) * entry + piece * 16u, there);
        }
    };
    auto prefetch = [&](uint32_t t) {
        constexpr uint32_t kLines = D * kElement <= 128u ? 1u : D * kElement / 128u;
        const uint32_t k0 = at0 + t * kTile;
        if (t >= n) return;
        for (uint32_t l = w * 32u + lane; l < kLines * kTile; l += kWarps * 32u) {
            const uint32_t i = k0 + l / kLines;
            if (i >= keys) break;
            uint32_t slot = first_slot + i;
            if (slot >= slots) slot -= slots;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(head_rows + slot * entry + l % kLines * 128u));
        }
    };
    auto landed = [&](uint32_t st) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && (F::Q8 || sound(info))) mbar_arrive(&full[st]);   // codes' copies count on barriers of their own
    };
    if constexpr (F::Q8) {
        // A tile's codes as f16 values, in the operand's swizzle.
        auto store = [&](char* to, uint32_t i, const uint4& x) {
            uint32_t key, piece;
            place(i, key, piece);
            char* at16 = to + piece / 4u * kPiece;
            const uint32_t chunk = piece % 4u * 2u;
            *reinterpret_cast<uint4*>(at16 + swizzled(key, chunk)) =
                make_uint4(codes2<0x4140>(x.x), codes2<0x4342>(x.x), codes2<0x4140>(x.y), codes2<0x4342>(x.y));
            *reinterpret_cast<uint4*>(at16 + swizzled(key, chunk + 1u)) =
                make_uint4(codes2<0x4140>(x.z), codes2<0x4342>(x.z), codes2<0x4140>(x.w), codes2<0x4342>(x.w));
        };
        // With the keys come the tile's scales; a key past the last has the
        // last one's (every row's weight of it is zero).
        auto copy_scales = [&](uint32_t t) {
#pragma unroll
            for (uint32_t key = w * 32u + lane; key < kTile; key += kWarps * 32u) {
                uint32_t slot = first_slot + min(at0 + t * kTile + key, keys - 1u);
                if (slot >= slots) slot -= slots;
                float2* to = &info.scales[(done + t) % kScaleTiles][key];
                copy4(&to->x, on.key_scales + slot, true);
                copy4(&to->y, on.value_scales + slot, true);
            }
        };
        if constexpr (F::kRing > 0) {
            // Two tiles of keys and of values are on their way at any time. A
            // thread converts its own 16-byte pieces of every row it takes, and
            // a tile that does not come by one copy it also copies piece by piece.
            constexpr uint32_t kSwap = D == 128 ? 7u : 3u;   // the copy's swizzle: chunk c of row r at c ^ (r or r/2)
            const uint32_t kind = value ? 1u : 0u;
            char* const ring = smem + F::kRingAt + kind * (F::kRing * kTile * D);
            const uint32_t own = key0 * D + ((piece0 ^ ((D == 128 ? sub : sub / 2u) & kSwap)) << 4);
            static_assert(kSub == 1, "a thread's piece is the same of all its rows");
            // rfull has one arrival a tile, the first warp's, which is made only
            // once every warp is done with the slot's tile before, however this
            // one comes: so the barrier is never two phases ahead of a warp that
            // is still at that tile (it would take the parity of the later phase
            // for one not yet done), and no copy lands on codes still unread.
            auto fetch = [&](uint32_t t) {
                if (t < n) {
                    const uint32_t it = done + t, r = it % F::kRing;
                    if (w == 0 && lane == 0) wait(&info.rempty[kind][r], (it / F::kRing & 1u) ^ 1u, info);
                    if (whole(t)) {
                        if (w == 0 && lane == 0 && sound(info)) {
                            mbar_arrive_expect_tx(&info.rfull[kind][r], kTile * D);
                            copy_tile(ring + r * kTile * D, map, 0, on.h, slot_at(at0 + t * kTile), on.s, &info.rfull[kind][r]);
                        }
                        __syncwarp();
                    } else {
                        each(t, 0, kEach, [&](uint32_t i, const char* src, bool there) {
                            copy16(ring + r * kTile * D + own + i * (kStep * D), src, there);
                        });
                        if (w == 0 && lane == 0 && sound(info)) mbar_arrive(&info.rfull[kind][r]);
                    }
                    if (!value) copy_scales(t);
                }
                copies_commit();
            };
#pragma unroll
            for (uint32_t k = 0; k < F::kRing; ++k) fetch(k);
            for (uint32_t t = 0; t < n; ++t) {
                const uint32_t it = done + t, st = it % F::kStages, r = it % F::kRing;
                copies_wait<F::kRing - 1>();
                wait(&info.rfull[kind][r], it / F::kRing & 1u, info);
                wait(&empty[st], (it / F::kStages & 1u) ^ 1u, info);
                char* to = operand + st * F::kOperand;
                const char* from = ring + r * kTile * D + own;
#pragma unroll
                for (uint32_t i = 0; i < kEach; ++i) store(to, i, *reinterpret_cast<const uint4*>(from + i * (kStep * D)));
                landed(st);
                if (lane == 0) mbar_arrive(&info.rempty[kind][r]);
                fetch(t + F::kRing);
            }
            copies_wait<0>();
        } else {
            // The next quarter of a tile's codes waits in registers.
            constexpr uint32_t kBatch = 4, kBatches = kEach / kBatch;
            static_assert(kEach % kBatch == 0u && kBatches % 2u == 0u, "the two sets of codes take turns");
            uint4 codes[2][kBatch];
            auto load = [&](uint32_t t, uint32_t b, uint4 (&x)[kBatch]) {
                each(t, b * kBatch, kBatch, [&](uint32_t i, const char* src, bool there) {
                    x[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (there) x[i] = __ldg(reinterpret_cast<const uint4*>(src));
                });
            };
            load(0, 0, codes[0]);
            for (uint32_t t = 0; t < n; ++t) {
                const uint32_t it = done + t, st = it % F::kStages;
                if (!value) copy_scales(t);
                copies_commit();
                wait(&empty[st], (it / F::kStages & 1u) ^ 1u, info);
                char* to = operand + st * F::kOperand;
#pragma unroll
                for (uint32_t b = 0; b < kBatches; ++b) {
                    load(b + 1u < kBatches ? t : t + 1u, (b + 1u) % kBatches, codes[(b + 1u) % 2u]);
#pragma unroll
                    for (uint32_t i = 0; i < kBatch; ++i) store(to, b * kBatch + i, codes[b % 2u][i]);
                }
                copies_wait<0>();
                landed(st);
                prefetch(t + 1u + kPrefetch);
            }
        }
    } else {
        for (uint32_t t = 0; t < n; ++t) {
            const uint32_t it = done + t, st = it % F::kStages;
            wait(&empty[st], (it / F::kStages & 1u) ^ 1u, info);
            char* to = operand + st * F::kOperand;
            if (whole(t)) {   // straight into the operand's layout
                const bool arrives = lane == 0 && sound(info);
                if (w == 0 && arrives) {
                    mbar_arrive_expect_tx(&full[st], F::kOperand);
#pragma unroll
                    for (uint32_t d = 0; d < D / 64u; ++d)
                        copy_tile(to + d * kPiece, map, d * 64u, on.h, slot_at(at0 + t * kTile), on.s, &full[st]);
                } else if (arrives) {
                    mbar_arrive(&full[st]);
                }
                __syncwarp();
            } else {
                each(t, 0, kEach, [&](uint32_t i, const char* src, bool there) {
                    uint32_t key, piece;
                    place(i, key, piece);
                    copy16(to + piece / 8u * kPiece + swizzled(key, piece % 8u), src, there);
                });
                copies_commit();
                copies_wait<0>();
                landed(st);
            }
        }
    }
}

// Rows first .. of a stretch of entries by plain loops, for the stretch that
// holds a value that is not finite: a masked one must not touch the others.
template <class F>
__device__ void plain_rows(const TensorArgs& args, const Step& step, uint32_t s, uint32_t h, uint32_t rg, uint32_t from,
                           uint32_t to, float* out, float* base, float* sum, float* scratch) {
    const cb_tree_attention& a = args.a;
    const cb_cache& c = a.cache;
    const uint32_t G = args.groups, rows = a.tokens * G, tid = threadIdx.x;
    const __half* keys = static_cast<const __half*>(c.key) + s * cache_sequence_stride(c) + static_cast<size_t>(h) * F::D;
    const __half* values = static_cast<const __half*>(c.value) + s * cache_sequence_stride(c) + static_cast<size_t>(h) * F::D;
    const size_t entry = static_cast<size_t>(c.kv_heads) * F::D;
    constexpr uint32_t kChunk = 512;   // scores in `scratch`; NaN marks none
    for (uint32_t r = 0; r < F::RT; ++r) {
        const uint32_t row = rg * F::RT + r, node = row / G;
        float top = kNegInf, total = 0.0f, acc = 0.0f;
        if (row < rows && node < step.nodes) {
            uint64_t mask;
            uint32_t first;
            row_sight(a, step, s, node, mask, first);
            const float* q = a.query + (static_cast<size_t>(s) * a.tokens + node) * (a.query_stride ? a.query_stride : a.query_heads * F::D) +
                             (static_cast<size_t>(h) * G + row % G) * F::D;
            auto seen = [&](uint32_t e) { return e < step.length ? e >= first : (mask >> (e - step.length) & 1ull) != 0; };
            for (uint32_t e0 = from; e0 < to; e0 += kChunk) {
                const uint32_t count = min(kChunk, to - e0);
                __syncthreads();
                for (uint32_t i = tid; i < count; i += kThreads) {
                    float v = kNegInf;
                    if (seen(e0 + i)) {
                        const __half* k = keys + ((e0 + i) % c.slots) * entry;
                        v = 0.0f;
                        for (uint32_t d = 0; d < F::D; ++d) v = fmaf(q[d], __half2float(k[d]), v);
                        v *= a.scale_log2e;
                    }
                    scratch[i] = v;
                }
                __syncthreads();
                float most = top;
                for (uint32_t i = 0; i < count; ++i) most = fmaxf(most, scratch[i]);
                const float ground = most == kNegInf ? 0.0f : most, keep = top == kNegInf ? 0.0f : ex2(top - most);
                total *= keep;
                acc *= keep;
                for (uint32_t i = 0; i < count; ++i) {
                    if (!seen(e0 + i)) continue;
                    const float p = ex2(scratch[i] - ground);
                    total += p;
                    if (tid < F::D) acc = fmaf(p, __half2float(values[((e0 + i) % c.slots) * entry + tid]), acc);
                }
                top = most;
            }
        }
        if (tid < F::D) out[r * F::kOut + tid] = acc;
        if (tid == 0) {
            base[r] = top;
            sum[r] = total;
        }
    }
    __syncthreads();
}

template <class F>
__global__ void __launch_bounds__(kThreads, 1) tree_attention_tensor_kernel(const TensorArgs args, const __grid_constant__ CUtensorMap keys_map,
                                                                              const __grid_constant__ CUtensorMap values_map) {
    constexpr uint32_t D = F::D, RT = F::RT, N = F::N;
    extern __shared__ __align__(1024) char smem_raw[];
    char* smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    Info& info = *reinterpret_cast<Info*>(smem + F::kInfoAt);
    const cb_tree_attention& a = args.a;
    const cb_cache& c = a.cache;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t G = args.groups, pairs = c.kv_heads * args.row_groups;   // a sequence's

    grid_dependency_wait();
    grid_dependents_launch();

    // ---- the share of this CTA: units mine0 .. mine1 − 1 of all pairs'. A pair is
    // kBegin units (its beginning) and then one a tile ------------------------------
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&info.kfull[i], kLoadWarps / 2u);
            mbar_init(&info.vfull[i], kLoadWarps / 2u);
            mbar_init(&info.kempty[i], 1);
            mbar_init(&info.vempty[i], 1);
            mbar_init(&info.sfull[i], 1);
            mbar_init(&info.sempty[i], kSoftWarps);
            mbar_init(&info.pfull[i], kSoftWarps);
            mbar_init(&info.pempty[i], 1);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                mbar_init(&info.rfull[i][k], 1);
                mbar_init(&info.rempty[i][k], kLoadWarps / 2u);
            }
        }
        info.abort = 0;
        info.polls = min(spin_limit_of(args.fault), kPolls);
        info.fault = args.fault;
        fence_barrier_init();
    }
    if (warp == 0) {
        tmem_alloc(&info.tmem, 512);
        tmem_relinquish();
    }
    for (uint32_t i = tid; i < a.sequences; i += kThreads) {
        const Step t = step_of(a, i);
        info.before[i + 1] = (kBegin + (t.end - t.first + kTile - 1u) / kTile) * pairs;
    }
    if (tid == 0) info.before[0] = 0;
    __syncthreads();
    if (warp == 0) {   // running sums, 32 at a time
        uint32_t carry = 0;
        for (uint32_t i0 = 1; i0 <= a.sequences; i0 += 32u) {
            uint32_t v = i0 + lane <= a.sequences ? info.before[i0 + lane] : 0u;
#pragma unroll
            for (uint32_t k = 1; k < 32u; k <<= 1) {
                const uint32_t o = __shfl_up_sync(kAllLanes, v, k);
                if (lane >= k) v += o;
            }
            v += carry;
            if (i0 + lane <= a.sequences) info.before[i0 + lane] = v;
            carry = __shfl_sync(kAllLanes, v, 31);
        }
    }
    __syncthreads();
    const uint32_t tmem = info.tmem;
    const uint32_t all = info.before[a.sequences], ctas = min(gridDim.x, all);   // no CTA among these without a unit
    auto share = [&](uint32_t cta) { return static_cast<uint32_t>(static_cast<uint64_t>(all) * cta / ctas); };
    const uint32_t mine0 = blockIdx.x < ctas ? share(blockIdx.x) : 0u, mine1 = blockIdx.x < ctas ? share(blockIdx.x + 1u) : 0u;
    auto owner = [&](uint32_t unit) {   // the CTA whose share holds a unit
        uint32_t o = static_cast<uint32_t>(static_cast<uint64_t>(unit) * ctas / all);
        while (share(o + 1u) <= unit) ++o;
        while (share(o) > unit) --o;
        return o;
    };

    uint32_t done = 0;   // tiles this CTA has put through its pipeline: every role counts the same
    for (uint32_t at = mine0; at < mine1;) {
        // ---- a stretch of one pair's tiles --------------------------------------
        uint32_t s = 0;
        {
            uint32_t hi = a.sequences;   // before[s] ≤ at < before[s + 1]
            while (hi - s > 1u) {
                const uint32_t mid = (s + hi) >> 1;
                if (info.before[mid] <= at) s = mid; else hi = mid;
            }
        }
        const uint32_t units = (info.before[s + 1] - info.before[s]) / pairs, tiles = units - kBegin;
        const uint32_t pair = (at - info.before[s]) / units, pair0 = info.before[s] + pair * units;
        const uint32_t unit1 = min(pair0 + units, mine1) - pair0;   // within the pair
        const uint32_t tile0 = at - pair0 > kBegin ? at - pair0 - kBegin : 0u;
        const uint32_t n = unit1 > kBegin ? unit1 - kBegin - tile0 : 0u;
        at = pair0 + unit1;
        const uint32_t h = pair % c.kv_heads, rg = pair / c.kv_heads;
        const Step step = step_of(a, s);
        const uint32_t keys = step.end - step.first;
        const uint32_t rows = a.tokens * G;
        if (tid == 0) {
            constexpr uint32_t kElement = F::Q8 ? 1u : 2u;
            const size_t head = (s * cache_sequence_stride(c) + static_cast<size_t>(h) * D) * kElement;
            const size_t scales = s * cache_scale_stride(c) + static_cast<size_t>(h) * c.slots;
            info.on = Stretch{static_cast<const char*>(c.key) + head, static_cast<const char*>(c.value) + head,
                              c.key_scale + (F::Q8 ? scales : 0u), c.value_scale + (F::Q8 ? scales : 0u),
                              static_cast<size_t>(c.kv_heads) * D * kElement, c.slots, step.first % c.slots, step.first,
                              step.length, keys, tile0, n, done, args.maps ? &keys_map : nullptr,
                              args.maps ? &values_map : nullptr, s, h};
        }
        if (n == 0) {
            if (tiles == 0 && unit1 == units)   // a pair without keys: its last unit's CTA writes its zeros
                for (uint32_t i = tid; i < RT * (D / 4u); i += kThreads) {
                    const uint32_t row = rg * RT + i / (D / 4u);
                    if (row < rows) write_row(a, step, s, h, G, row, 4u * (i % (D / 4u)), make_float4(0.f, 0.f, 0.f, 0.f), 0.0f);
                }
            continue;
        }

        // ---- its rows: masks, factors, and the two query terms -------------------
        if (tid < RT) {
            const uint32_t r = tid, row = rg * RT + r, node = row / G;
            const bool live = row < rows && node < step.nodes;
            uint64_t mask = 0;
            uint32_t first = 0xFFFFFFFFu;
            if (live) row_sight(a, step, s, node, mask, first);
            info.mask[r] = mask;
            info.first[r] = first;
            info.unit[r] = kLeastUnit;
            info.base[r] = 0.0f;
            info.weight[r] = live ? (F::Q8 ? kWeightTop * 0x1p100f : kWeightTop) : 0.0f;
        }
        {
            // A warp a row, four values a lane (D = 256: two such pieces);
            // all of the warp's rows on their way at once.
            constexpr uint32_t kWarps = kThreads / 32u, kEach = D == 256 ? 2 : 1, kMine = (RT + kWarps - 1u) / kWarps;
            float4 x[kMine][kEach];
#pragma unroll
            for (uint32_t k = 0; k < kMine; ++k) {
                const uint32_t r = warp + k * kWarps, row = rg * RT + r, node = row / G;
                const bool live = r < RT && row < rows && node < step.nodes;
                const float* src = a.query + (live ? static_cast<size_t>(s) * a.tokens + node : 0u) * (a.query_stride ? a.query_stride : a.query_heads * D) +
                                   (static_cast<size_t>(h) * G + row % G) * D;
#pragma unroll
                for (uint32_t i = 0; i < kEach; ++i)
                    x[k][i] = live && 4u * lane < D ? reinterpret_cast<const float4*>(src)[32u * i + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (uint32_t k = 0; k < kMine; ++k) {
                const uint32_t r = warp + k * kWarps;
                uint32_t top = 0;
#pragma unroll
                for (uint32_t i = 0; i < kEach; ++i)
                    top = max(max(max(top, __float_as_uint(x[k][i].x) & 0x7FFFFFFFu), max(__float_as_uint(x[k][i].y) & 0x7FFFFFFFu, __float_as_uint(x[k][i].z) & 0x7FFFFFFFu)),
                              __float_as_uint(x[k][i].w) & 0x7FFFFFFFu);
                top = __reduce_max_sync(kAllLanes, top);
                if (lane == 0 && r < RT) info.top[r] = top;
            }
            __syncthreads();
            // One power of two for all rows where their sizes are within 2^6
            // of each other (rows of zeros and rows that are not finite aside),
            // else one for each.
            uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
            for (uint32_t r = lane; r < RT; r += 32u) {
                const uint32_t top = info.top[r];
                if (top != 0u && top < 0x7F800000u) {
                    most = max(most, top);
                    least = min(least, top);
                }
            }
            most = __reduce_max_sync(kAllLanes, most);
            least = __reduce_min_sync(kAllLanes, least);
            const bool even = most == 0u || (most >> 23) - (least >> 23) <= 6u;
            if (tid == 0) {
                info.even_factor = even;
                info.even_weight[0] = info.even_weight[1] = true;
            }
#pragma unroll
            for (uint32_t k = 0; k < kMine; ++k) {
                const uint32_t r = warp + k * kWarps;
                if (r >= RT) break;
                const float up = row_power(even ? most : info.top[r]);
#pragma unroll
                for (uint32_t i = 0; i < kEach; ++i) {
                    const uint32_t d = 128u * i + 4u * lane;
                    if (4u * lane >= D) break;
                    uint2 hi, lo;
                    split2(x[k][i].x * up, x[k][i].y * up, hi.x, lo.x);
                    split2(x[k][i].z * up, x[k][i].w * up, hi.y, lo.y);
                    char* piece = smem + d / 64u * (N * 128u);
                    *reinterpret_cast<uint2*>(piece + swizzled(r, d % 64u / 8u) + d % 8u * 2u) = hi;
                    *reinterpret_cast<uint2*>(piece + swizzled(RT + r, d % 64u / 8u) + d % 8u * 2u) = lo;
                }
                if (lane == 0) info.factor[r] = a.scale_log2e / up;   // a dead row's products are 0
            }
        }
        fence_proxy_async();
        __syncthreads();
        if (warp == 0) {
            uint32_t late = 0;
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
                const uint32_t first = lane < RT / 2 ? info.first[half * (RT / 2) + lane] : 0xFFFFFFFFu;
                const bool live = first != 0xFFFFFFFFu;
                if (live) late = max(late, first);
                const uint32_t unset = __ballot_sync(kAllLanes, live);
                if (lane == 0) {
                    info.unset[half] = unset;
                    info.least_unit[half] = kLeastUnit;
                }
            }
            late = __reduce_max_sync(kAllLanes, late);
            if (lane == 0) {
                info.latest = late;
                info.context = min(step.length, step.end);
            }
        }
        __syncthreads();

        if (warp < kSoftWarps) soften<F>(info, smem, tmem);
        else if (warp < kSoftWarps + kLoadWarps) {
            bring<F>(info, smem);
            // A loader is done first: it finds who shares the pair.
            if (n != tiles && tid == 32u * (kSoftWarps + kLoadWarps - 1u)) {
                const uint32_t unit0 = pair0 + kBegin, c0 = owner(unit0);
                info.first_cta = c0;
                info.last_cta = owner(unit0 + tiles - 1u);
                info.begins = share(c0) < unit0;
            }
        } else multiply<F>(info, smem, tmem);

        // ---- the stretch's outputs: the two terms' halves added ---------------------
        float* out = reinterpret_cast<float*>(smem + F::kKeysAt);
        const uint32_t last = done + n - 1u;
        wait(&info.pempty[last % F::kWeights], last / F::kWeights & 1u, info);
        __syncthreads();
        if (warp < kSoftWarps) {
            const uint32_t group = warp >> 2, quad = warp & 3u, r = quad % 2u * (RT / 2) + lane;   // output_lane's row
            const uint32_t lanes = tmem + ((quad * 32u) << 16) + F::kSumsAt + group * (D / kGroups);
            tc_fence_after();
            const bool mine = lane < RT / 2;
            const float weight = mine ? info.weight[r] : 0.0f, back = weight != 0.0f ? 1.0f / weight : 0.0f;
            float* to = out + r * F::kOut + group * (D / kGroups);
            auto sums_at = [&](uint32_t d, float (&v)[16]) {   // with what was folded
                tmem_ld(lanes + d, v);
                if (n <= kFold) return;
                constexpr bool kPacked = D == 256;
                const bool upper = kPacked && group >= kGroups / 2u;
                float m[16];
                tmem_ld(tmem + ((quad * 32u) << 16) + F::kFoldedAt + (upper ? group - kGroups / 2u : group) * (D / kGroups) + d, m);
#pragma unroll
                for (uint32_t j = 0; j < 16; ++j) {
                    if (kPacked) {
                        const float high = __shfl_xor_sync(kAllLanes, m[j], 16);
                        if (upper) m[j] = high;
                    }
                    v[j] += m[j];
                }
            };
            if (quad >= 2u) {
#pragma unroll
                for (uint32_t d = 0; d < D / kGroups; d += 16u) {
                    float v[16];
                    sums_at(d, v);
                    if (mine)
#pragma unroll
                        for (uint32_t j = 0; j < 16; j += 4)
                            *reinterpret_cast<float4*>(to + d + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kSoftWarps * 32u) : "memory");
            if (quad < 2u) {
#pragma unroll
                for (uint32_t d = 0; d < D / kGroups; d += 16u) {
                    float v[16];
                    sums_at(d, v);
                    if (mine)
#pragma unroll
                        for (uint32_t j = 0; j < 16; j += 4) {
                            const float4 lo = *reinterpret_cast<const float4*>(to + d + j);
                            *reinterpret_cast<float4*>(to + d + j) =
                                make_float4((v[j] + lo.x) * back, (v[j + 1] + lo.y) * back, (v[j + 2] + lo.z) * back, (v[j + 3] + lo.w) * back);
                        }
                }
            }
            if (tid < RT) {   // the row's base and sum (a row that saw nothing: none)
                info.shift[tid] = info.unset[tid / (RT / 2)] >> tid % (RT / 2) & 1u ? kNegInf : -info.base[tid];
                info.sums[tid] = ((info.total[0][tid] + info.total[1][tid]) + info.total[2][tid]) + info.total[3][tid];
            }
            tc_fence_before();
        }
        __syncthreads();
        if constexpr (!F::Q8) {
            bool odd = false;
            for (uint32_t i = tid; i < RT * D; i += kThreads) {
                const uint32_t r = i / D, row = rg * RT + r;
                odd |= row < rows && row / G < step.nodes && !(fabsf(out[r * F::kOut + i % D]) < __builtin_huge_valf());
            }
            if (__syncthreads_or(odd))
                plain_rows<F>(args, step, s, h, rg, step.first + tile0 * kTile, min(step.first + (tile0 + n) * kTile, step.end), out,
                              info.shift, info.sums, reinterpret_cast<float*>(smem + F::kPAt));
        }

        if (n == tiles) {
            for (uint32_t i = tid; i < RT * (D / 4u); i += kThreads) {
                const uint32_t r = i / (D / 4u), col = 4u * (i % (D / 4u)), row = rg * RT + r;
                if (row < rows) write_row(a, step, s, h, G, row, col, *reinterpret_cast<const float4*>(out + r * F::kOut + col), info.sums[r]);
            }
        } else {
            // A CTA's stretch of a pair is its first (slot 0) unless the pair's tiles begin inside its share.
            constexpr size_t kSlot = RT * (D + 2u);
            const uint32_t c0 = info.first_cta, c1 = info.last_cta;
            const bool begins = info.begins;
            auto slot_of = [&](uint32_t k) { return args.partials + (2u * k + (k == c0 && begins ? 1u : 0u)) * kSlot; };
            float* slot = slot_of(blockIdx.x);
            for (uint32_t i = tid; i < RT * (D / 4u); i += kThreads) {
                const uint32_t r = i / (D / 4u), col = 4u * (i % (D / 4u));
                __stcg(reinterpret_cast<float4*>(slot + r * D + col), *reinterpret_cast<const float4*>(out + r * F::kOut + col));
            }
            if (tid < RT) {
                __stcg(slot + RT * D + tid, info.shift[tid]);
                __stcg(slot + RT * (D + 1u) + tid, info.sums[tid]);
            }
            __syncthreads();
            if (tid == 0) {   // one thread's fences, for what the barriers order before and after them
                __threadfence();
                const unsigned int arrived = atomicAdd(args.tickets + c0, 1u);
                info.last = arrived == c1 - c0;
                if (info.last) {
                    args.tickets[c0] = 0u;
                    __threadfence();
                }
            }
            __syncthreads();
            if (info.last) {
                // Each part's factor for each row, then every output adds the
                // parts with their loads together.
                float* factor = reinterpret_cast<float*>(smem + F::kFactorAt);
                const uint32_t parts = c1 - c0 + 1u;
                for (uint32_t i = tid; i < parts * RT; i += kThreads) factor[i] = __ldcg(slot_of(c0 + i / RT) + RT * D + i % RT);
                __syncthreads();
                if (tid < RT) {
                    float top = kNegInf, total = 0.0f;
                    for (uint32_t k = 0; k < parts; ++k) top = fmaxf(top, factor[k * RT + tid]);
                    for (uint32_t k = 0; k < parts; ++k) {
                        const float kt = factor[k * RT + tid], kl = __ldcg(slot_of(c0 + k) + RT * (D + 1u) + tid);
                        // a part that saw nothing of the row adds nothing
                        const float f = kt == kNegInf ? 0.0f : ex2(kt - top);
                        total = kt == kNegInf && kl == 0.0f ? total : fmaf(kl, f, total);
                        factor[k * RT + tid] = kt == kNegInf && kl == 0.0f ? -1.0f : f;
                    }
                    info.sums[tid] = total;
                }
                __syncthreads();
                for (uint32_t i = tid; i < RT * (D / 4u); i += kThreads) {
                    const uint32_t r = i / (D / 4u), col = 4u * (i % (D / 4u)), row = rg * RT + r;
                    if (row >= rows) break;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (uint32_t k = 0; k < parts; ++k) {
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(slot_of(c0 + k) + r * D + col));
                        const float f = factor[k * RT + r];
                        if (f >= 0.0f || f != f) {
                            acc.x = fmaf(v.x, f, acc.x);
                            acc.y = fmaf(v.y, f, acc.y);
                            acc.z = fmaf(v.z, f, acc.z);
                            acc.w = fmaf(v.w, f, acc.w);
                        }
                    }
                    write_row(a, step, s, h, G, row, col, acc, info.sums[r]);
                }
            }
        }
        done += n;
        __syncthreads();   // the operands' space, the queries and `info` are free again
    }
    if (info.abort && tid == 0)   // a wait ran out: give copies still on their way a millisecond to land
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

// The map of a cache's rows for copies of 128 slots of a head: as they lie
// (codes, in a swizzle that spreads the threads' pieces over the banks), or in
// 64-value pieces in the operands' swizzle. False where it cannot be made; the
// kernel then copies rows piece by piece.
template <class F>
bool encode_map(CUtensorMap* map, const cb_cache& c, uint32_t sequences, const void* rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    if (!encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess || !fn)
            return false;
        encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
    const cuuint64_t element = F::Q8 ? 1u : 2u, entry = static_cast<cuuint64_t>(c.kv_heads) * F::D * element;
    const cuuint64_t dims[4] = {F::D, c.kv_heads, c.slots, sequences};
    const cuuint64_t strides[3] = {F::D * element, entry, cache_sequence_stride(c) * element};
    const cuuint32_t box[4] = {F::Q8 ? F::D : 64u, 1, kTile, 1}, elem[4] = {1, 1, 1, 1};
    return encode(map, F::Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(rows), dims,
                  strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  F::Q8 && F::D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class F>
constexpr size_t smem_bytes() { return F::kInfoAt + sizeof(Info) + 1024; }

template <class F>
cudaError_t launch_form(const cb_tree_attention& a, cudaStream_t stream, bool pdl) {
    auto kernel = tree_attention_tensor_kernel<F>;
    static_assert(smem_bytes<F>() <= 227 * 1024, "shared memory");
    static bool configured[64] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device >= 64) return cudaErrorInvalidDevice;
    if (!configured[device]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem_bytes<F>()));
        if (e != cudaSuccess) return e;
        configured[device] = true;
    }
    const uint32_t G = a.query_heads / a.cache.kv_heads, row_groups = (a.tokens * G + F::RT - 1u) / F::RT;
    TensorArgs args{a, G, row_groups, static_cast<unsigned int*>(a.workspace),
                    reinterpret_cast<float*>(static_cast<char*>(a.workspace) + kTreeTickets * 4u), fault_word(), 0};
    CUtensorMap keys_map = {}, values_map = {};
    // head dimension 256's codes go through registers; fewer slots than a tile hold no whole one
    if ((!F::Q8 || F::kRing > 0) && a.cache.slots >= kTile)
        args.maps = encode_map<F>(&keys_map, a.cache, a.sequences, a.cache.key) && encode_map<F>(&values_map, a.cache, a.sequences, a.cache.value);
    const uint32_t sms = static_cast<uint32_t>(sm_count());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms < F::kMostCtas ? sms : F::kMostCtas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem_bytes<F>();
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args, keys_map, values_map);
}

uint32_t row_tile(const cb_tree_attention& a) {
    const uint32_t rows = a.tokens * (a.query_heads / a.cache.kv_heads);
    return a.cache.head_dim == 256 || rows <= 32 ? 32u : 64u;
}

}  // namespace

// Whether the form can take a step: its tiles are counted in 32 bits, and
// each CTA lists every sequence.
bool tree_attention_tensor_fits(const cb_tree_attention& a) {
    if (a.sequences > kMostSequences) return false;
    const uint32_t rows = a.tokens * (a.query_heads / a.cache.kv_heads);
    const uint64_t keys = a.max_keys < a.cache.slots ? a.max_keys : a.cache.slots;
    const uint64_t tiles = static_cast<uint64_t>(a.sequences) * a.cache.kv_heads * ((rows + 31u) / 32u) * (keys / kTile + 1u + kBegin);
    return tiles < 0x7FFFFFFFull;
}

// Whether it should: 16 rows or fewer fill one row tile of the other form,
// and a small step ends before this one's pipelines fill (about 20 us). The
// sides cross near 120,000 (key, 32 rows) products. This form against the other,
// in us: 64 values in f16, 8 sequences of 2k to 4k keys (65,000) 24.1 / 23.9, of
// twice that 29.8 / 37.5; 128 in 8 bits, 4 of 2k (65,000) 27.0 / 25.4, 4 of 4k 30.8 /
// 35.4, but 16 of 1,000 36.9 / 28.7, 16 of 2,000 45.9 / 58.9; 256 in 8 bits, 16 of 4k
// (64,000) 36.9 / 31.0, of 8k 50.9 / 55.1.
bool tree_attention_tensor_pays(const cb_tree_attention& a) {
    const uint32_t rows = a.tokens * (a.query_heads / a.cache.kv_heads);
    if (rows <= 16) return false;
    uint64_t keys = a.max_keys < a.cache.slots ? a.max_keys : a.cache.slots;
    if (a.window && keys > static_cast<uint64_t>(a.window) + a.tokens) keys = static_cast<uint64_t>(a.window) + a.tokens;
    return static_cast<uint64_t>(a.sequences) * a.cache.kv_heads * ((rows + 31u) / 32u) * keys >= 120000ull;
}

uint64_t tree_attention_tensor_bytes(const cb_tree_attention& a) {
    const int sms = sm_count();
    if (sms <= 0) return 0;
    return kTreeTickets * 4ull + 2ull * sms * row_tile(a) * (a.cache.head_dim + 2u) * sizeof(float);
}

cudaError_t tree_attention_tensor_run(const cb_tree_attention& a, cudaStream_t stream, bool pdl) {
    const bool q8 = a.cache.format == CB_CACHE_Q8, wide = row_tile(a) == 64u;
    switch (a.cache.head_dim) {
        case 64:
            if (q8) return wide ? launch_form<Form<64, true, 64>>(a, stream, pdl) : launch_form<Form<64, true, 32>>(a, stream, pdl);
            return wide ? launch_form<Form<64, false, 64>>(a, stream, pdl) : launch_form<Form<64, false, 32>>(a, stream, pdl);
        case 128:
            if (q8) return wide ? launch_form<Form<128, true, 64>>(a, stream, pdl) : launch_form<Form<128, true, 32>>(a, stream, pdl);
            return wide ? launch_form<Form<128, false, 64>>(a, stream, pdl) : launch_form<Form<128, false, 32>>(a, stream, pdl);
        default:
            return q8 ? launch_form<Form<256, true, 32>>(a, stream, pdl) : launch_form<Form<256, false, 32>>(a, stream, pdl);
    }
}

}  // namespace cb
