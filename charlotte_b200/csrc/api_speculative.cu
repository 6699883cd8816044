// C ABI entry points of speculative decoding over a quantised cache: the
// cache's write, read and keep, tree attention and verification. A bad
// argument is CB_ERROR_INVALID before anything runs.
#include <cuda_runtime.h>

#include <cmath>

#include "api_common.h"
#include "cache.cuh"
#include "charlotte_b200.h"
#include "kernels.h"

using namespace cb;

namespace {

int launched(cudaError_t e, const char* what) { return e == cudaSuccess ? CB_OK : fail_cuda(e, what); }

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// A cache's preconditions. `pointers`: its buffers are given (a size query
// has none).
int cache_arguments(const cb_cache& c, uint32_t sequences, const char* who, bool pointers) {
    if (c.format != CB_CACHE_F16 && c.format != CB_CACHE_Q8)
        return fail(CB_ERROR_INVALID, "%s: cache format %u", who, c.format);
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
        return fail(CB_ERROR_INVALID, "%s: head dimension %u", who, c.head_dim);
    if (c.slots == 0 || c.slots > 0x7FFFFFFFu) return fail(CB_ERROR_INVALID, "%s: %u slots (1 to 2^31 - 1)", who, c.slots);
    if (c.kv_heads == 0 || c.kv_heads > 1024) return fail(CB_ERROR_INVALID, "%s: %u kv heads (1 to 1024)", who, c.kv_heads);
    if (sequences > 65535) return fail(CB_ERROR_INVALID, "%s: %u sequences (at most 65,535)", who, sequences);
    if (c.sequence_stride % 16 != 0)
        return fail(CB_ERROR_INVALID, "%s: a sequence stride that is not a multiple of 16 elements", who);
    const uint64_t entries = static_cast<uint64_t>(c.slots) * c.kv_heads;
    if (sequences > 1 && cache_sequence_stride(c) < entries * c.head_dim)
        return fail(CB_ERROR_INVALID, "%s: sequences' caches overlap (stride below one cache)", who);
    if (sequences > 1 && c.format == CB_CACHE_Q8 && cache_scale_stride(c) < entries)
        return fail(CB_ERROR_INVALID, "%s: sequences' scales overlap (stride below one cache's)", who);
    if (!pointers) return CB_OK;
    if (!c.key || !c.value) return fail(CB_ERROR_INVALID, "%s: a cache without keys or values", who);
    if (!aligned16(c.key) || !aligned16(c.value))
        return fail(CB_ERROR_INVALID, "%s: cache rows must be 16-byte aligned", who);
    if (c.format == CB_CACHE_Q8 && (!c.key_scale || !c.value_scale || !aligned4(c.key_scale) || !aligned4(c.value_scale)))
        return fail(CB_ERROR_INVALID, "%s: an 8-bit cache without its scales", who);
    return CB_OK;
}

// A step's: rows, masks, positions.
int step_arguments(const uint32_t* lengths, const uint32_t* nodes, const uint64_t* ancestors, uint32_t position0,
                   uint32_t tokens, bool tree, const char* who) {
    if (tokens > kTreeRows && (tree || ancestors))
        return fail(CB_ERROR_INVALID, "%s: %u rows a sequence (at most %u)", who, tokens, kTreeRows);
    if (!lengths && static_cast<uint64_t>(position0) + tokens > 0x7FFFFFFFull)
        return fail(CB_ERROR_INVALID, "%s: positions past 2^31 - 1", who);
    if (!aligned4(lengths) || !aligned4(nodes) || !aligned8(ancestors))
        return fail(CB_ERROR_INVALID, "%s: unaligned lengths, nodes or ancestors", who);
    return CB_OK;
}

// A row stride in floats (0: packed) for heads of `width` floats together.
bool stride_ok(uint32_t stride, uint64_t width) { return stride == 0 || (stride >= width && stride % 4 == 0); }

int tree_attention_arguments(const cb_tree_attention* a, bool pointers) {
    const char* who = pointers ? "cb_tree_attention_run" : "cb_tree_attention_bytes";
    if (!a) return fail(CB_ERROR_INVALID, "%s: null argument", who);
    if (int rc = cache_arguments(a->cache, a->sequences, who, pointers)) return rc;
    if (a->query_heads == 0 || a->query_heads % a->cache.kv_heads != 0 || a->query_heads / a->cache.kv_heads > 16)
        return fail(CB_ERROR_INVALID, "%s: %u query heads over %u kv heads", who, a->query_heads, a->cache.kv_heads);
    if (int rc = step_arguments(a->lengths, a->nodes, a->ancestors, a->position0, a->tokens, true, who)) return rc;
    if (!stride_ok(a->query_stride, static_cast<uint64_t>(a->query_heads) * a->cache.head_dim))
        return fail(CB_ERROR_INVALID, "%s: a query stride of %u floats", who, a->query_stride);
    if (!(std::fabs(a->scale_log2e) <= 3.0e38f)) return fail(CB_ERROR_INVALID, "%s: a scale that is not finite", who);
    if (a->max_keys == 0) return fail(CB_ERROR_INVALID, "%s: max_keys is 0", who);
    if (!pointers) return CB_OK;
    if (!a->query || !a->out || !a->workspace) return fail(CB_ERROR_INVALID, "%s: null argument", who);
    if (!aligned16(a->query) || !aligned16(a->out) || !aligned8(a->out16) || !aligned16(a->workspace))
        return fail(CB_ERROR_INVALID, "%s: unaligned queries, outputs or workspace", who);
    return CB_OK;
}

int sampling_arguments(const cb_sampling& s, const char* which) {
    if (!(s.temperature >= 0.0f && s.temperature <= 3.0e38f) || !(s.min_p >= 0.0f && s.min_p <= 1.0f) || !(s.top_p >= 0.0f))
        return fail(CB_ERROR_INVALID, "cb_verify_run: the %s's temperature, top_p or min_p", which);
    return CB_OK;
}

}  // namespace

extern "C" {

int cb_cache_write_run(const cb_cache_write* w, uint32_t flags, void* stream) {
    const char* who = "cb_cache_write_run";
    if (!w || !w->key || !w->value) return fail(CB_ERROR_INVALID, "%s: null argument", who);
    if (int rc = cache_arguments(w->cache, w->sequences, who, true)) return rc;
    if (int rc = step_arguments(w->lengths, w->nodes, w->ancestors, w->position0, w->tokens, false, who)) return rc;
    if ((w->query == nullptr) != (w->query_out == nullptr) || (w->query == nullptr) != (w->query_heads == 0))
        return fail(CB_ERROR_INVALID, "%s: queries, their output and their heads come together", who);
    if (w->query_heads > 16384) return fail(CB_ERROR_INVALID, "%s: %u query heads", who, w->query_heads);
    if (w->query && (w->query_gain == nullptr) != (w->key_gain == nullptr))
        return fail(CB_ERROR_INVALID, "%s: QK-norm on queries or keys alone", who);
    if (w->factors && !w->turns) return fail(CB_ERROR_INVALID, "%s: factors without turns", who);
    const uint64_t d = w->cache.head_dim;
    if (!stride_ok(w->query_stride, w->query_heads * d) || !stride_ok(w->key_stride, w->cache.kv_heads * d) ||
        !stride_ok(w->value_stride, w->cache.kv_heads * d))
        return fail(CB_ERROR_INVALID, "%s: a row stride below the row or not a multiple of 4", who);
    if (w->query && w->query_out == w->query && w->query_stride && w->query_stride != w->query_heads * d)
        return fail(CB_ERROR_INVALID, "%s: queries written in place are packed", who);
    if (!aligned16(w->query) || !aligned16(w->query_out) || !aligned16(w->key) || !aligned16(w->value) ||
        !aligned16(w->query_gain) || !aligned16(w->key_gain))
        return fail(CB_ERROR_INVALID, "%s: rows and gains must be 16-byte aligned", who);
    if (!aligned4(w->turns) || !aligned4(w->factors)) return fail(CB_ERROR_INVALID, "%s: unaligned turns or factors", who);
    if (w->tokens == 0 || w->sequences == 0) return CB_OK;
    return launched(cache_write_run(*w, static_cast<cudaStream_t>(stream), flags & CB_RUN_PDL), who);
}

int cb_cache_read_run(const cb_cache_read* r, uint32_t flags, void* stream) {
    const char* who = "cb_cache_read_run";
    if (!r) return fail(CB_ERROR_INVALID, "%s: null argument", who);
    if (int rc = cache_arguments(r->cache, r->sequences, who, true)) return rc;
    if (r->out_format != CB_F32 && r->out_format != CB_F16)
        return fail(CB_ERROR_INVALID, "%s: output format %u", who, r->out_format);
    if (!aligned16(r->out_key) || !aligned16(r->out_value))
        return fail(CB_ERROR_INVALID, "%s: outputs must be 16-byte aligned", who);
    if (int rc = step_arguments(r->lengths, r->starts, nullptr, r->start0, r->tokens, false, who)) return rc;
    if (r->tokens == 0 || r->sequences == 0 || (!r->out_key && !r->out_value)) return CB_OK;
    return launched(cache_read_run(*r, static_cast<cudaStream_t>(stream), flags & CB_RUN_PDL), who);
}

uint64_t cb_tree_attention_bytes(const cb_tree_attention* a) {
    if (tree_attention_arguments(a, false)) return 0;
    if (a->tokens == 0 || a->sequences == 0) return 16;
    const uint64_t n = tree_attention_bytes(*a);
    if (n == 0) fail(CB_ERROR_STEP, "cb_tree_attention_bytes: no device");
    return n;
}

int cb_tree_attention_run(const cb_tree_attention* a, uint32_t flags, void* stream) {
    if (int rc = tree_attention_arguments(a, true)) return rc;
    if (a->tokens == 0 || a->sequences == 0) return CB_OK;
    const uint64_t need = tree_attention_bytes(*a);
    if (need && a->workspace_bytes < need)
        return fail(CB_ERROR_INVALID, "cb_tree_attention_run: a workspace of %llu bytes (needs %llu)",
                    static_cast<unsigned long long>(a->workspace_bytes), static_cast<unsigned long long>(need));
    return launched(tree_attention_run(*a, static_cast<cudaStream_t>(stream), flags & CB_RUN_PDL, flags & CB_RUN_TENSOR),
                    "cb_tree_attention_run");
}

int cb_verify_run(const cb_verify* v, uint32_t flags, void* stream) {
    const char* who = "cb_verify_run";
    if (!v || !v->candidates || !v->ids || !v->uniforms || !v->path || !v->kept || !v->sampled)
        return fail(CB_ERROR_INVALID, "%s: null argument", who);
    if (v->sequences > 0x7FFFFFFFu) return fail(CB_ERROR_INVALID, "%s: %u sequences", who, v->sequences);
    if (int rc = step_arguments(v->nodes, v->nodes, v->ancestors, 0, v->tokens, true, who)) return rc;
    if (!aligned16(v->candidates) || !aligned16(v->draft_candidates))
        return fail(CB_ERROR_INVALID, "%s: candidate lists must be 16-byte aligned", who);
    if (!aligned4(v->ids) || !aligned4(v->uniforms) || !aligned4(v->path) || !aligned4(v->kept) || !aligned4(v->sampled))
        return fail(CB_ERROR_INVALID, "%s: unaligned ids, uniforms or outputs", who);
    if (int rc = sampling_arguments(v->target, "target")) return rc;
    if (v->draft_candidates)
        if (int rc = sampling_arguments(v->draft, "draft")) return rc;
    if (v->tokens == 0 || v->sequences == 0) return CB_OK;
    return launched(verify_run(*v, static_cast<cudaStream_t>(stream), flags & CB_RUN_PDL), who);
}

int cb_cache_keep_run(const cb_cache_keep* k, uint32_t flags, void* stream) {
    const char* who = "cb_cache_keep_run";
    if (!k || !k->path || !k->kept) return fail(CB_ERROR_INVALID, "%s: null argument", who);
    if (int rc = cache_arguments(k->cache, k->sequences, who, true)) return rc;
    if (int rc = step_arguments(k->lengths, k->kept, nullptr, k->position0, k->tokens, true, who)) return rc;
    if (k->tokens > k->cache.slots)
        return fail(CB_ERROR_INVALID, "%s: %u rows in %u slots", who, k->tokens, k->cache.slots);
    if (!aligned4(k->path) || !aligned4(k->new_lengths)) return fail(CB_ERROR_INVALID, "%s: unaligned path or new lengths", who);
    if (k->new_lengths && k->new_lengths == k->lengths)
        return fail(CB_ERROR_INVALID, "%s: lengths updated in place", who);
    if (k->layers > 65535) return fail(CB_ERROR_INVALID, "%s: %u layers", who, k->layers);
    const uint64_t span = k->sequences * cache_sequence_stride(k->cache);
    if (k->layers > 1 && (k->layer_stride < span || k->layer_stride % 16 != 0 ||
                          (k->cache.format == CB_CACHE_Q8 &&
                           k->scale_layer_stride < k->sequences * cache_scale_stride(k->cache))))
        return fail(CB_ERROR_INVALID, "%s: layers' caches overlap or are not 16-byte aligned", who);
    if (k->tokens == 0 || k->sequences == 0 || k->layers == 0) return CB_OK;
    return launched(cache_keep_run(*k, static_cast<cudaStream_t>(stream), flags & CB_RUN_PDL), who);
}

}  // extern "C"
