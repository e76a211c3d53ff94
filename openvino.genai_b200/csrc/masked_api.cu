// Entry points of include/masked_b200.h: argument checks, scratch, launch sequence of a masked step and of the acceptance of drafts.
#include <algorithm>
#include <climits>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "pa_handle.h"
#include "tensor_map.h"

namespace {

int fail(int code, const char* msg) {
    pa::set_last_error(msg);
    return code;
}

int fail_cuda(const char* what, cudaError_t e) {
    cudaGetLastError();   // (told to this caller, not to whoever asks the runtime next)
    pa::set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
    return PA_ERR_CUDA;
}

#define MASKED_CUDA(expr)                                   \
    do {                                                    \
        const cudaError_t _e = (expr);                      \
        if (_e != cudaSuccess) return fail_cuda(#expr, _e); \
    } while (0)

// The body of an entry point: what it throws (the text of an error may not find memory) ends here.
template <class F>
int guarded(F&& body) {
    try {
        return body();
    } catch (...) {
        return PA_ERR_CUDA;
    }
}

// The caller's current device is put back when the call returns.
struct DeviceScope {
    int before = -1;
    cudaError_t error;
    explicit DeviceScope(int device) {
        error = cudaGetDevice(&before);
        if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Scratch of a masked step.  No part falls where tokens or sequences grow, so what is reserved for the largest step holds every smaller one.
struct Scratch {
    size_t header, tile_prefix, ptile_prefix, worker_start, stream_done, decode_o, decode_ml, tree_words, tree_depth, redo, items, item_prefix, starts, cuts, part_o, part_ml, total;
};
// Steps of single tokens go without a plan where a stream has few tiles (under a short window, or by its block table): the plan is a launch's chain in front
// of a kernel that is not much longer.  Longer streams are better off in the plan's slices, which know how many tiles each has.  us, with | without a plan, 8 kv
// heads of 128, L2 flushed, contexts of 9001 (a window of 1984 makes 64 tiles):
//   window          256        1000        1984        4000        8000
//   1 row, bf16   26 | 17     30 | 23     32 | 26     54 | 44     65 | 38
//   32, bf16      30 | 26     52 | 46     79 | 73    118 | 114   194 | 190
//   128, bf16     60 | 56    122 | 119   198 | 196   351 | 351   650 | 656
//   8, u8         28 | 22     32 | 28     36 | 40     54 | 48     69 | 65
//   32, u8        32 | 28     48 | 42     63 | 60     91 | 89    140 | 140
//   128, u8       52 | 50     93 | 93    138 | 145   228 | 243   396 | 429
// The line lies where many rows over a u8 cache begin to lose; single rows would gain beyond it.
constexpr int kDirectTiles = 64;

// The partial results of the tensor-core kernel's CTAs, by far the largest part (39 MB at a head size of 128), come last and are there where it is launched: not in
// `rows_only`, a step of as many tokens as sequences.
Scratch plan_scratch(const pa_handle* h, int tokens, int sequences, bool rows_only) {
    const pa::CacheGeom& g = h->g;
    const int G = g.Hq / g.Hkv, HK = g.Hkv * ((G + 15) / 16), RT = std::min(G, 16);
    Scratch s{};
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += (bytes + 255) / 256 * 256; return at; };
    const size_t B = (size_t)sequences, workers = (size_t)pa::decode_max_workers(h->sm_count), slots = B * HK + workers;
    s.header = take(sizeof(pa::PlanHeader));
    s.tile_prefix = take((B + 1) * sizeof(int));
    s.ptile_prefix = take((B + 1) * sizeof(int));
    s.worker_start = take(workers * sizeof(pa::WorkerStart));
    s.stream_done = take(std::max<size_t>(B, 1) * HK * sizeof(int));
    s.decode_o = take(slots * RT * g.D * sizeof(float));
    s.decode_ml = take(slots * RT * 2 * sizeof(float));
    s.tree_words = take((size_t)tokens * pa::kTreeWords * sizeof(uint32_t));
    s.tree_depth = take((size_t)tokens * sizeof(int));
    s.redo = take((size_t)tokens * g.Hq * sizeof(int));
    const size_t q_tiles = (size_t)tokens * G / pa::kPrefillItemRows + B, pieces = 2 * (size_t)h->sm_count;
    s.items = take(q_tiles * sizeof(pa::MaskItem));
    s.item_prefix = take((q_tiles + 1) * sizeof(long long));
    s.starts = take(((size_t)h->sm_count + 1) * sizeof(pa::MaskStart));
    s.cuts = take((size_t)h->sm_count * sizeof(pa::MaskCut));
    if (!rows_only && tokens > 1 && pa::prefill_tc_supported(g)) {
        s.part_o = take(pieces * pa::kPrefillItemRows * g.D * sizeof(float));
        s.part_ml = take(pieces * pa::kPrefillItemRows * sizeof(float2));
    }
    s.total = off;
    return s;
}

int ensure_scratch(pa_handle* h, size_t bytes, cudaStream_t stream) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (stream) MASKED_CUDA(cudaStreamIsCapturing(stream, &capture));
    const bool capturing = capture != cudaStreamCaptureStatusNone;
    if (bytes <= h->mws_bytes) {
        h->mws_captured |= capturing;
        return PA_OK;
    }
    if (capturing) return fail(PA_ERR_TOO_LARGE, "the scratch would have to grow inside a stream capture: pa_b200_masked_reserve for the step beforehand");
    if (h->mws_captured) h->mws_retired.push_back(h->mws);
    else if (h->mws) MASKED_CUDA(cudaFree(h->mws));   // (waits for the work that uses it)
    h->mws = nullptr; h->mws_bytes = 0; h->mws_captured = false;
    const size_t want = (bytes + bytes / 4 + (1 << 20) - 1) >> 20 << 20;
    MASKED_CUDA(cudaMalloc((void**)&h->mws, want));
    h->mws_bytes = want;
    return PA_OK;
}

int validate_masked(const pa_handle* h, const pa_forward_args* a, const pa_mask_args* m, bool host) {
    const int rc = pa::validate_forward_args(h, a);
    if (rc != PA_OK) return rc;
    if (!m || m->struct_size != sizeof(pa_mask_args)) return fail(PA_ERR_INVALID_ARG, "pa_mask_args: NULL or struct_size mismatch");
    if (m->sliding_window < 0 || m->sink_tokens < 0) return fail(PA_ERR_INVALID_ARG, "negative sliding_window or sink_tokens");
    if (a->scores) return fail(PA_ERR_UNSUPPORTED, "a masked step has no score output");
    if (!(a->scale >= 0.f) || a->scale > 3.0e38f) return fail(PA_ERR_INVALID_ARG, "scale is negative or not finite");
    if (a->num_tokens == 0 || a->num_sequences == 0) return PA_OK;
    if (a->num_blocks == 0) return fail(PA_ERR_INVALID_ARG, "the cache has no blocks");
    if (!aligned(a->key_cache) || !aligned(a->value_cache)) return fail(PA_ERR_UNSUPPORTED, "a cache is not 16-byte aligned");
    if (!host && (!aligned(a->query) || !aligned(a->output))) return fail(PA_ERR_UNSUPPORTED, "query or output is not 16-byte aligned");
    if ((long long)a->num_tokens * h->g.Hq > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 query rows in one call");
    if ((long long)a->num_blocks * h->g.Hkv > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 blocks of heads in one cache");
    if ((long long)a->num_block_indices * h->g.bs > INT_MAX - 4096) return fail(PA_ERR_TOO_LARGE, "more than 2^31 tokens of context in one call");
    const int G = h->g.Hq / h->g.Hkv;   // (the decode kernel numbers the tiles of all its streams)
    if (((long long)a->num_block_indices * h->g.bs / 32 + a->num_sequences + 1) * h->g.Hkv * ((G + 15) / 16) > INT_MAX)
        return fail(PA_ERR_TOO_LARGE, "more than 2^31 tiles of 32 tokens of all kv heads in one call");
    return PA_OK;
}

}  // namespace

namespace pa {

int forward_masked(pa_handle* h, const pa_forward_args* a, const pa_mask_args& mask, cudaStream_t stream) {
    if (a->num_sequences == 0 || a->num_tokens == 0) return PA_OK;
    const Scratch s = plan_scratch(h, a->num_tokens, a->num_sequences, /*rows_only=*/a->num_tokens == a->num_sequences);
    const int rc = ensure_scratch(h, s.total, stream);
    if (rc != PA_OK) return rc;
    const int G = h->g.Hq / h->g.Hkv, HK = h->g.Hkv * ((G + 15) / 16);
    KernelArgs k;
    std::memset(&k, 0, sizeof(k));
    k.g = h->g;
    k.query = a->query; k.key = a->key; k.value = a->value; k.output = a->output;
    k.num_tokens = a->num_tokens;
    k.key_cache = a->key_cache; k.value_cache = a->value_cache; k.num_blocks = a->num_blocks;
    k.past_lens = a->past_lens; k.subsequence_begins = a->subsequence_begins;
    k.block_indices = a->block_indices; k.block_indices_begins = a->block_indices_begins;
    k.num_block_indices = a->num_block_indices;
    k.num_sequences = a->num_sequences; k.max_context_len = a->max_context_len;
    k.scale = a->scale;
    k.rotated_block_indices = a->rotated_block_indices; k.rotation_deltas = a->rotation_deltas;
    k.num_rotated_blocks = a->num_rotated_blocks;
    k.rotation_trig_lut = a->rotation_trig_lut; k.rotation_lut_rows = a->rotation_lut_rows;
    k.status = h->status;
    uint8_t* const ws = h->mws;
    k.plan = (PlanHeader*)(ws + s.header);
    k.tile_prefix = (int*)(ws + s.tile_prefix);
    k.ptile_prefix = (int*)(ws + s.ptile_prefix);
    k.worker_start = (WorkerStart*)(ws + s.worker_start);
    k.stream_done = (int*)(ws + s.stream_done);
    k.part_o = (float*)(ws + s.decode_o);
    k.part_ml = (float*)(ws + s.decode_ml);
    k.rows_per_tile = std::min(G, 16);
    // upper bounds of the tiles of rows with one new token: all tiles of their block tables, or what their windows leave
    const long long table_tiles = (long long)a->num_block_indices * h->g.bs / 32 + 1;
    long long row_tiles = table_tiles;
    if (mask.sliding_window > 0) row_tiles = std::min(row_tiles, ((long long)mask.sliding_window + 31) / 32 + ((long long)mask.sink_tokens + 31) / 32 + 1);
    k.max_tiles = std::min(table_tiles + a->num_sequences, row_tiles * a->num_sequences) * HK;
    MaskParams& m = k.m;
    m.on = 1;
    m.window = mask.sliding_window;
    m.sinks = mask.sink_tokens;
    m.parents = mask.tree_parents;
    m.tree_words = (uint32_t*)(ws + s.tree_words);
    m.tree_depth = (int*)(ws + s.tree_depth);
    m.tree_blocks = mask.tree_parents ? a->num_sequences : 0;
    m.sm_count = h->sm_count;
    m.items = (MaskItem*)(ws + s.items);
    m.item_prefix = (long long*)(ws + s.item_prefix);
    m.starts = (MaskStart*)(ws + s.starts);
    m.cuts = (MaskCut*)(ws + s.cuts);
    m.redo = (int*)(ws + s.redo);
    // As many tokens as sequences: single tokens, almost always, and no launches for chunks; what of them there is beside sequences without
    // tokens, the device finds out
    m.rows_in_decode = a->num_tokens > 1 && a->num_tokens == a->num_sequences;
    if (a->num_tokens == a->num_sequences && row_tiles <= kDirectTiles && row_tiles * a->num_sequences * HK <= INT_MAX / 2) {
        m.direct_tiles = (int)row_tiles;
        k.release_early = 1;
    }
    m.part_o = s.part_o ? (float*)(ws + s.part_o) : nullptr;
    m.part_ml = s.part_o ? (float2*)(ws + s.part_ml) : nullptr;
    if (m.direct_tiles == 0) k.decode_all_workers = decode_launch_workers(k, h->sm_count);
    int launches = 0;
    if (a->num_rotated_blocks > 0) { MASKED_CUDA(launch_rotate(k, stream)); ++launches; }
    MASKED_CUDA(launch_write_kv(k, stream, /*with_plan=*/true)); ++launches;
    // (always: among the tokens that no sequence has, even a step of one sequence may hold a single token)
    MASKED_CUDA(launch_decode(k, stream, h->sm_count, &launches));
    h->last_prefill_kernel = PA_PREFILL_NONE;
    if (a->num_tokens > 1 && !m.rows_in_decode) {
        h->last_prefill_kernel = prefill_tc_supported(h->g) ? PA_PREFILL_TCGEN05 : PA_PREFILL_GENERIC;
        if (prefill_tc_supported(h->g)) {
            if (h->g.cache != PA_DTYPE_U8) {
                const long long size[3] = {h->g.D, h->g.bs, (long long)a->num_blocks * h->g.Hkv}, stride[2] = {h->g.D, (long long)h->g.bs * h->g.D};
                const int box[3] = {64, h->g.bs, 1};
                if (!make_map(&m.map_k, h->g.cache, a->key_cache, 3, size, stride, box) || !make_map(&m.map_v, h->g.cache, a->value_cache, 3, size, stride, box))
                    return fail(PA_ERR_CUDA, "a tensor map could not be made");
            }
            MASKED_CUDA(launch_prefill_tc(k, stream, h->sm_count, /*max_items=*/h->sm_count, &launches));
            MASKED_CUDA(launch_masked_join(k, stream, &launches));
        } else {
            MASKED_CUDA(launch_masked_rows(k, stream, &launches));
        }
    }
    h->launches += launches;
    return PA_OK;
}

}  // namespace pa

extern "C" {

int pa_b200_forward_masked(pa_handle* h, const pa_forward_args* a, const pa_mask_args* mask) {
    return guarded([&] {
        const int rc = validate_masked(h, a, mask, /*host=*/false);
        if (rc != PA_OK) return rc;
        DeviceScope scope(h->device);
        MASKED_CUDA(scope.error);
        return pa::forward_masked(h, a, *mask, a->stream ? (cudaStream_t)a->stream : h->stream);
    });
}

int pa_b200_forward_masked_host(pa_handle* h, const pa_forward_args* a, const pa_mask_args* mask) {
    return guarded([&] {
        const int rc = validate_masked(h, a, mask, /*host=*/true);
        if (rc != PA_OK) return rc;
        DeviceScope scope(h->device);
        MASKED_CUDA(scope.error);
        return pa::forward_host(h, a, mask);
    });
}

int pa_b200_masked_reserve(pa_handle* h, int32_t num_tokens, int32_t num_sequences, int32_t num_block_indices) {
    return guarded([&] {
        if (!h) return fail(PA_ERR_INVALID_ARG, "NULL handle");
        if (num_tokens < 0 || num_sequences < 0 || num_block_indices < 0) return fail(PA_ERR_INVALID_ARG, "negative size");
        if (num_sequences > 65535) return fail(PA_ERR_TOO_LARGE, "more than 65535 sequences in one call");
        DeviceScope scope(h->device);
        MASKED_CUDA(scope.error);
        return ensure_scratch(h, plan_scratch(h, num_tokens, num_sequences, /*rows_only=*/false).total, nullptr);
    });
}

int pa_b200_tree_accept(pa_handle* h, const pa_tree_accept_args* a) {
    return guarded([&] {
        if (!h) return fail(PA_ERR_INVALID_ARG, "NULL handle");
        if (!a || a->struct_size != sizeof(pa_tree_accept_args)) return fail(PA_ERR_INVALID_ARG, "pa_tree_accept_args: NULL or struct_size mismatch");
        if (a->num_tokens < 0 || a->num_sequences < 0 || a->num_block_indices < 0 || a->num_blocks < 0 || a->num_layers < 0)
            return fail(PA_ERR_INVALID_ARG, "negative size");
        if (a->num_sequences > 65535) return fail(PA_ERR_TOO_LARGE, "more than 65535 sequences in one call");
        if (a->num_sequences == 0) return (int)PA_OK;
        if (a->max_path < 1 || a->max_path > PA_TREE_MAX_TOKENS) return fail(PA_ERR_INVALID_ARG, "max_path must be 1 to 256");
        if (!a->past_lens || !a->subsequence_begins || !a->block_indices_begins || !a->path || !a->num_accepted || !a->next_token)
            return fail(PA_ERR_INVALID_ARG, "NULL metadata or output pointer");
        if (a->num_tokens > 0 && (!a->tree_parents || !a->draft_tokens || !a->sampled_tokens)) return fail(PA_ERR_INVALID_ARG, "NULL token pointer");
        if (a->num_block_indices > 0 && !a->block_indices) return fail(PA_ERR_INVALID_ARG, "NULL block_indices");
        if ((long long)a->num_block_indices * h->g.bs > INT_MAX - 4096) return fail(PA_ERR_TOO_LARGE, "more than 2^31 tokens of context in one call");
        if ((long long)a->num_blocks * h->g.bs > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 tokens of cache");
        if (a->num_layers > 0 && (!a->key_caches || !a->value_caches)) return fail(PA_ERR_INVALID_ARG, "NULL array of caches");
        if (a->num_layers > 0 && a->num_blocks == 0) return fail(PA_ERR_INVALID_ARG, "the cache has no blocks");
        for (int i = 0; i < a->num_layers; ++i) {
            if (!a->key_caches[i] || !a->value_caches[i]) return fail(PA_ERR_INVALID_ARG, "NULL cache pointer");
            if (!aligned(a->key_caches[i]) || !aligned(a->value_caches[i])) return fail(PA_ERR_UNSUPPORTED, "a cache is not 16-byte aligned");
        }
        // bytes that two caches share would be moved by two blocks at once
        std::vector<const void*> caches(a->key_caches, a->key_caches + a->num_layers);
        caches.insert(caches.end(), a->value_caches, a->value_caches + a->num_layers);
        std::sort(caches.begin(), caches.end(), std::less<>());
        const uintptr_t bytes = (uintptr_t)a->num_blocks * (uintptr_t)h->g.block_bytes;
        const auto shared = std::adjacent_find(caches.begin(), caches.end(), [&](const void* x, const void* y) { return (uintptr_t)y - (uintptr_t)x < bytes; });
        if (shared != caches.end()) return fail(PA_ERR_INVALID_ARG, shared[0] == shared[1] ? "a cache is among the layers' twice" : "two of the layers' caches overlap");
        DeviceScope scope(h->device);
        MASKED_CUDA(scope.error);
        const pa::TreeAcceptArgs t{h->g, a->tree_parents, a->draft_tokens, a->sampled_tokens, a->past_lens, a->subsequence_begins, a->block_indices,
                                   a->block_indices_begins, a->num_tokens, a->num_sequences, a->num_block_indices, a->num_blocks, a->max_path,
                                   a->path, a->num_accepted, a->next_token, a->new_past_lens, h->status};
        int launches = 0;
        MASKED_CUDA(pa::launch_tree_accept(t, a->key_caches, a->value_caches, a->num_layers, a->stream ? (cudaStream_t)a->stream : h->stream, &launches));
        h->launches += launches;
        return (int)PA_OK;
    });
}

}  // extern "C"
