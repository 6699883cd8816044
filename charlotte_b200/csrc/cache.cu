// A cache of f16 or 8-bit rows: writing a step's keys and values (with the
// QK-norm and RoPE before them), reading entries back, and moving a drafted
// tree's accepted rows together. The arithmetic of the norm and the turns is
// rope.cu's (rope_math.cuh).
//
// The 8-bit form keeps one scale a head row, m/127 of its largest magnitude
// m: a score is then (q·codes)·scale and a weighted value (p·scale)·codes,
// so attention multiplies by the scale once a key, outside its products. A
// scale a 32-value block would follow outliers more closely but would have to
// enter between the products' steps.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "api_common.h"
#include "cache.cuh"
#include "kernels.h"
#include "numerics.cuh"
#include "rope_math.cuh"
#include "tma.cuh"

namespace cb {

namespace {

// ---- write ------------------------------------------------------------------

// A CTA takes R rows of a sequence; d/8 lanes a head, lane i holding its vec4s
// i and i + d/8 as in rope_kernel. The rows' angles are found once into shared
// memory while their queries, keys and values are on their way. Bound: latency
// (load, angles, norm, store, one after the other) while the rows fill the GPU
// less than once: eight trees of 16 rows, 16 + 2·8 heads of 128, 3.8 to 4.2 us. Past
// that, latency of two waves and L2, which holds that much: a 2,047-row prompt of
// 32 + 2·8 heads of 64, 44 MB, 10.4 to 11.1 us (4.1 TB/s).
// Two rows a CTA have their loads and angles together, which helps once the
// rows are more than the CTAs that fit at a time (that prompt 12.2 us with one
// row) and costs a row's arithmetic before (those trees 5.0 us with two).
template <uint32_t R>
__global__ void __launch_bounds__(512, 2) cache_write_kernel(const cb_cache_write a) {
    extern __shared__ float angles[];   // a row's cosines then sines, d/2 each
    grid_dependency_wait();
    const uint32_t d = a.cache.head_dim, lanes = d / 8u;
    const uint32_t s = blockIdx.y, i0 = blockIdx.x * R;
    const uint32_t n = a.nodes ? min(a.nodes[s], a.tokens) : a.tokens;
    if (i0 >= n) return;
    const uint32_t length = a.lengths ? a.lengths[s] : a.position0;
    const size_t row0 = static_cast<size_t>(s) * a.tokens + i0;
    const uint32_t hq = a.query_heads, hkv = a.cache.kv_heads;
    const uint32_t total = (hq + 2u * hkv) * lanes;
    for (uint32_t base = 0; base < total; base += blockDim.x) {
        const uint32_t item = base + threadIdx.x;
        const bool in_row = item < total;   // dead lanes only take part in the shuffles
        const uint32_t head = in_row ? item / lanes : 0u, lane = item % lanes;
        const bool is_query = head < hq, is_value = head >= hq + hkv;
        const uint32_t h = is_query ? head : is_value ? head - hq - hkv : head - hq;
        const size_t stride = is_query ? (a.query_stride ? a.query_stride : hq * d)
                              : is_value ? (a.value_stride ? a.value_stride : hkv * d)
                                         : (a.key_stride ? a.key_stride : hkv * d);
        const float* src = (is_query ? a.query : is_value ? a.value : a.key) + row0 * stride + static_cast<size_t>(h) * d;
        float4 in0[R], in1[R];
#pragma unroll
        for (uint32_t r = 0; r < R; ++r) {
            in0[r] = in1[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (in_row && i0 + r < n) {
                in0[r] = reinterpret_cast<const float4*>(src + r * stride)[lane];
                in1[r] = reinterpret_cast<const float4*>(src + r * stride)[lane + lanes];
            }
        }
        if (base == 0) {   // the angles, while the first rows are on their way
            if (a.turns) {
                const uint32_t share = blockDim.x / R, r = min(threadIdx.x / share, R - 1u), i = i0 + r;
                if (i < n && threadIdx.x < share * R) {
                    const uint32_t p = length + (a.ancestors ? mask_depth(a.ancestors[row0 + r]) : i);
                    rope_angles(p, a.turns, a.factors, d, angles + r * d, angles + r * d + d / 2u, threadIdx.x - r * share, share);
                }
            }
            __syncthreads();
            grid_dependents_launch();
        }
#pragma unroll
        for (uint32_t r = 0; r < R; ++r) {
            const uint32_t i = i0 + r;
            const bool live = in_row && i < n;
            const size_t row = row0 + r;
            const uint32_t slot = (length + i) % a.cache.slots;
            const bool stored = i + a.cache.slots >= n;   // no later row of the step takes the slot
            float4 x0 = in0[r], x1 = in1[r];
            if (a.key_gain) {
                const float rms = head_norm_factor(x0, x1, lanes, d, a.epsilon);
                if (live && !is_value) {
                    const float4* g = reinterpret_cast<const float4*>(is_query ? a.query_gain : a.key_gain);
                    const float4 g0 = g[lane], g1 = g[lane + lanes];
                    x0 = make_float4((x0.x * rms) * g0.x, (x0.y * rms) * g0.y, (x0.z * rms) * g0.z, (x0.w * rms) * g0.w);
                    x1 = make_float4((x1.x * rms) * g1.x, (x1.y * rms) * g1.y, (x1.z * rms) * g1.z, (x1.w * rms) * g1.w);
                }
            }
            if (a.turns && !is_value)
                rope_head(x0, x1, lane, lanes, d, false, a.epsilon, nullptr, true, a.halves != 0, angles + r * d, angles + r * d + d / 2u);

            float inverse = 0.0f, scale = 0.0f;
            if (a.cache.format == CB_CACHE_Q8) {
                // The largest magnitude by its bits: a NaN's are above an
                // infinity's, so either reaches the scale.
                uint32_t m = 0;
                const float e[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
                for (int c = 0; c < 8; ++c) m = max(m, __float_as_uint(e[c]) & 0x7FFFFFFFu);
                for (uint32_t k = lanes / 2u; k > 0; k >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, k));
                const float top = __uint_as_float(m);
                scale = top / 127.0f;
                inverse = 127.0f / top;
                if (inverse > 3.402823466e+38f) inverse = 3.402823466e+38f;   // a NaN stays
            }
            if (!live) continue;
            if (is_query) {
                float4* dst = reinterpret_cast<float4*>(a.query_out + (row * hq + h) * d);
                dst[lane] = x0;
                dst[lane + lanes] = x1;
                continue;
            }
            if (!stored) continue;
            const size_t at = s * cache_sequence_stride(a.cache) + (static_cast<size_t>(slot) * hkv + h) * d;
            void* cache = is_value ? a.cache.value : a.cache.key;
            if (a.cache.format == CB_CACHE_F16) {
                uint16_t* dst = static_cast<uint16_t*>(cache) + at;
                store_f16x4(dst + 4u * lane, x0);
                store_f16x4(dst + 4u * (lane + lanes), x1);
            } else {
                auto code = [&](float v) -> uint32_t {   // a NaN's is 128: its row's scale is not finite
                    const float t = rintf(v * inverse);
                    return t == t ? static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(t, -127.0f), 127.0f)) + 128) : 128u;
                };
                uint8_t* dst = static_cast<uint8_t*>(cache) + at;
                *reinterpret_cast<uint32_t*>(dst + 4u * lane) =
                    code(x0.x) | code(x0.y) << 8 | code(x0.z) << 16 | code(x0.w) << 24;
                *reinterpret_cast<uint32_t*>(dst + 4u * (lane + lanes)) =
                    code(x1.x) | code(x1.y) << 8 | code(x1.z) << 16 | code(x1.w) << 24;
                if (lane == 0)
                    (is_value ? a.cache.value_scale
                              : a.cache.key_scale)[s * cache_scale_stride(a.cache) +
                                                   static_cast<size_t>(h) * a.cache.slots + slot] = scale;
            }
        }
    }
}

// ---- read -------------------------------------------------------------------

// A thread takes the values that make one 16-byte store (4 f32 or 8 f16), so
// that a warp's stores are whole lines whatever the formats: the same piece of
// kReadUnroll entries, their loads together, with the entry's slot stepped and
// not divided out: with the divisions a store, one 16-code unit a thread, the
// figures below were 7.1 and 27.8 us. Bound: launch and one dependent load, then
// L2 and HBM. Called again on the same cache, whose codes then wait in L2: a
// 4,096-entry ring of 8 heads of 128 codes to f16 6.4 us, 64 times 777 entries of
// a head of 256 to f32 23.4 us (128 MB read and written, 5.5 TB/s); on caches that
// do not, 8.2 and 28.7 us. The same entries of an f16 cache, waiting in L2: to f16
// 5.4 and 12.1 us, to f32 7.4 and 24.4.
constexpr uint32_t kReadUnroll = 8;

template <bool Q8, bool F32>
__global__ void __launch_bounds__(256) cache_read_kernel(const cb_cache_read a, uint32_t entries_a_pass) {
    constexpr uint32_t kValues = F32 ? 4 : 8;
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t d = a.cache.head_dim, hkv = a.cache.kv_heads, slots = a.cache.slots;
    const uint32_t s = blockIdx.y;
    const bool value = blockIdx.z & 1u;
    char* out = static_cast<char*>(value ? a.out_value : a.out_key);
    if (!out) return;
    const uint32_t shift = (d == 64 ? 6u : d == 128 ? 7u : 8u) - (F32 ? 2u : 3u), row_units = hkv << shift;   // stores an entry
    // This thread's entry of each pass and its piece of it (wide entries take several CTAs).
    const uint32_t local = row_units <= 256u ? threadIdx.x / row_units : 0u;
    const uint32_t unit = row_units <= 256u ? threadIdx.x - local * row_units : (blockIdx.z >> 1) * 256u + threadIdx.x;
    if (local >= entries_a_pass || unit >= row_units) return;
    const uint32_t h = unit >> shift, piece = unit & ((1u << shift) - 1u);
    const uint32_t i0 = blockIdx.x * (entries_a_pass * kReadUnroll) + local;
    const uint32_t start = a.starts ? a.starts[s] : a.start0;
    const uint32_t length = a.lengths ? a.lengths[s] : 0u;
    constexpr uint32_t kElement = Q8 ? 1u : 2u;
    const size_t entry = static_cast<size_t>(hkv) * d * kElement;
    const char* rows = static_cast<const char*>(value ? a.cache.value : a.cache.key) +
                       (s * cache_sequence_stride(a.cache) + static_cast<size_t>(h) * d + piece * kValues) * kElement;
    const float* scales = (value ? a.cache.value_scale : a.cache.key_scale) + (Q8 ? s * cache_scale_stride(a.cache) + static_cast<size_t>(h) * slots : 0u);
    uint32_t words[kReadUnroll][4];
    float scale[kReadUnroll];
    bool held[kReadUnroll];
    uint32_t slot = (start + i0) % slots;
#pragma unroll
    for (uint32_t u = 0; u < kReadUnroll; ++u) {
        const uint32_t i = i0 + u * entries_a_pass, e = start + i;
        held[u] = i < a.tokens && (!a.lengths || (e < length && length - e <= slots));
        if (held[u]) {
            const char* src = rows + slot * entry;
            if (Q8) scale[u] = __ldg(scales + slot);
            if (Q8 && F32) {
                words[u][0] = __ldg(reinterpret_cast<const uint32_t*>(src));
            } else if (Q8 || F32) {
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(src));
                words[u][0] = w.x;
                words[u][1] = w.y;
            } else {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(src));
                words[u][0] = w.x;
                words[u][1] = w.y;
                words[u][2] = w.z;
                words[u][3] = w.w;
            }
        }
        slot += entries_a_pass;
        if (slot >= slots) slot %= slots;
    }
#pragma unroll
    for (uint32_t u = 0; u < kReadUnroll; ++u) {
        const uint32_t i = i0 + u * entries_a_pass;
        if (i >= a.tokens) return;
        uint4 to = make_uint4(0u, 0u, 0u, 0u);
        if (held[u]) {
            if (!Q8 && !F32) {
                to = make_uint4(words[u][0], words[u][1], words[u][2], words[u][3]);
            } else {
                float v[kValues];
#pragma unroll
                for (uint32_t c = 0; c < kValues; ++c)
                    v[c] = Q8 ? (static_cast<float>((words[u][c / 4] >> (8 * (c % 4))) & 0xFFu) - 128.0f) * scale[u]
                              : fp16_bits_to_f32(static_cast<uint16_t>(words[u][c / 2] >> (16 * (c % 2))));
                if (F32) {
                    to = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                } else {
                    uint32_t h2[4];
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c) {
                        const __half2 p = __floats2half2_rn(v[(2 * c) % kValues], v[(2 * c + 1) % kValues]);
                        h2[c] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    to = make_uint4(h2[0], h2[1], h2[2], h2[3]);
                }
            }
        }
        __stcs(reinterpret_cast<uint4*>(out + ((static_cast<size_t>(s) * a.tokens + i) * row_units + unit) * 16u), to);
    }
}

// ---- keep -------------------------------------------------------------------

// A CTA a sequence, layer and one of keys and values. Each thread owns a
// 16-byte column of the entry (or one head's scale) and moves it along the
// whole path, in order: row d's source lies at or after it (path ascends, so
// path[d] ≥ d), and no earlier move of the same column has written it. Eight
// rows' loads go before their stores. Bound: for one layer latency (path, rows
// and stores one after the other; eight sequences 3.2 us, 4.5 with keys and
// values in one CTA); for a batch's layers HBM (64 sequences of 28 layers, of 32
// rows 11.7 moved, read and written 171 MB, 28.7 us: 6.0 TB/s; 4 or 16 rows ahead
// take 28 and 29 us).
__global__ void __launch_bounds__(256) cache_keep_kernel(const cb_cache_keep a) {
    __shared__ uint32_t path[kTreeRows];
    grid_dependency_wait();
    const uint32_t s = blockIdx.x, layer = blockIdx.y;
    const bool value = blockIdx.z != 0;
    const uint32_t kept = min(a.kept[s], a.tokens);
    const uint32_t length = a.lengths ? a.lengths[s] : a.position0;
    if (layer == 0 && !value && threadIdx.x == 0 && a.new_lengths) a.new_lengths[s] = length + kept;
    for (uint32_t i = threadIdx.x; i < kept; i += blockDim.x) path[i] = a.path[static_cast<size_t>(s) * a.tokens + i];
    __syncthreads();
    grid_dependents_launch();
    const cb_cache& c = a.cache;
    const uint32_t bytes = c.kv_heads * c.head_dim * (c.format == CB_CACHE_F16 ? 2u : 1u);   // an entry's keys
    const uint32_t columns = bytes / 16u;
    const uint32_t scales = c.format == CB_CACHE_Q8 ? c.kv_heads : 0u;
    const size_t data0 = (layer * a.layer_stride + s * cache_sequence_stride(c)) * (c.format == CB_CACHE_F16 ? 2u : 1u);
    const size_t scale0 = layer * a.scale_layer_stride + s * cache_scale_stride(c);
    const uint32_t first = length % c.slots;   // tokens ≤ slots: one wrap at most
    auto slot = [&](uint32_t row) -> size_t { return first + row >= c.slots ? first + row - c.slots : first + row; };
    auto moves = [&](uint32_t d) { return path[d] != d && path[d] < a.tokens; };
    for (uint32_t w = threadIdx.x; w < columns + scales; w += blockDim.x) {
        if (w < columns) {
            char* base = static_cast<char*>(value ? c.value : c.key) + data0 + w * 16u;
            constexpr uint32_t kBatch = 8;   // a row's source lies after every row moved before it: loads go ahead of stores
            for (uint32_t d0 = 1; d0 < kept; d0 += kBatch) {
                uint4 row[kBatch];
#pragma unroll
                for (uint32_t k = 0; k < kBatch; ++k)
                    if (d0 + k < kept && moves(d0 + k)) row[k] = *reinterpret_cast<const uint4*>(base + slot(path[d0 + k]) * bytes);
#pragma unroll
                for (uint32_t k = 0; k < kBatch; ++k)
                    if (d0 + k < kept && moves(d0 + k)) *reinterpret_cast<uint4*>(base + slot(d0 + k) * bytes) = row[k];
            }
        } else {
            float* base = (value ? c.value_scale : c.key_scale) + scale0 + static_cast<size_t>(w - columns) * c.slots;
            for (uint32_t d = 1; d < kept; ++d)
                if (moves(d)) base[slot(d)] = base[slot(path[d])];
        }
    }
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, dim3 grid, uint32_t threads, size_t smem, cudaStream_t stream, bool pdl, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace

cudaError_t cache_write_run(const cb_cache_write& a, cudaStream_t stream, bool pdl) {
    const uint32_t lanes = (a.query_heads + 2u * a.cache.kv_heads) * (a.cache.head_dim / 8u);
    const uint32_t threads = lanes < 512u ? (lanes + 31u) / 32u * 32u : 512u;
    const size_t smem = a.cache.head_dim * sizeof(float);
    const int sms = sm_count();
    if (sms <= 0) return cudaErrorNoDevice;
    if (static_cast<uint64_t>(a.tokens) * a.sequences <= static_cast<uint32_t>(sms) * (2048u / threads))
        return launch(cache_write_kernel<1>, dim3(a.tokens, a.sequences), threads, smem, stream, pdl, a);
    return launch(cache_write_kernel<2>, dim3((a.tokens - 1u) / 2u + 1u, a.sequences), threads, 2u * smem, stream, pdl, a);
}

cudaError_t cache_read_run(const cb_cache_read& a, cudaStream_t stream, bool pdl) {
    const bool q8 = a.cache.format == CB_CACHE_Q8, f32 = a.out_format == CB_F32;
    const uint32_t row_units = a.cache.kv_heads * (a.cache.head_dim / (f32 ? 4u : 8u));
    const uint32_t pass = row_units < 256u ? 256u / row_units : 1u, wide = (row_units + 255u) / 256u;
    const dim3 grid((a.tokens + pass * kReadUnroll - 1u) / (pass * kReadUnroll), a.sequences, 2u * wide);
    if (q8) return f32 ? launch(cache_read_kernel<true, true>, grid, 256, 0, stream, pdl, a, pass)
                       : launch(cache_read_kernel<true, false>, grid, 256, 0, stream, pdl, a, pass);
    return f32 ? launch(cache_read_kernel<false, true>, grid, 256, 0, stream, pdl, a, pass)
               : launch(cache_read_kernel<false, false>, grid, 256, 0, stream, pdl, a, pass);
}

cudaError_t cache_keep_run(const cb_cache_keep& a, cudaStream_t stream, bool pdl) {
    const uint32_t columns = a.cache.kv_heads * a.cache.head_dim / (a.cache.format == CB_CACHE_F16 ? 8u : 16u);
    const uint32_t lanes = columns + (a.cache.format == CB_CACHE_Q8 ? a.cache.kv_heads : 0u);
    const uint32_t threads = lanes < 256u ? (lanes + 31u) / 32u * 32u : 256u;
    return launch(cache_keep_kernel, dim3(a.sequences, a.layers, 2), threads, 0, stream, pdl, a);
}

}  // namespace cb
