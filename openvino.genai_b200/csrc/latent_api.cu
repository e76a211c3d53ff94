// C ABI of latent attention (include/latent_b200.h): argument checking, scratch and launch sequencing.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <new>
#include <string>
#include <vector>

#include "latent_kernels.h"

namespace pa {
void set_last_error(const std::string& msg);
}

struct pa_latent_handle {
    pa_latent_desc desc;
    int device = 0;
    int sm_count = 148;
    cudaStream_t stream = nullptr;
    uint32_t* status = nullptr;   // device status word
    uint8_t* ws = nullptr;        // kernel scratch
    size_t ws_bytes = 0;
    bool captured = false;        // a stream capture has named the scratch
    std::vector<uint8_t*> retired;   // scratch of captures, outgrown since: their graphs may still run
    int64_t launches = 0;
    uint32_t wait_polls = latent::kWaitPolls;   // env PA_B200_LATENT_TEST_WAIT_POLLS: the kernels' bounded waits are made to run out
};

namespace {

int fail(int code, const char* msg) {
    pa::set_last_error(msg);
    return code;
}

int fail_cuda(const char* what, cudaError_t e) {
    cudaGetLastError();      // (told to this caller, not to whoever asks the runtime next)
    pa::set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
    return PA_ERR_CUDA;
}

#define LATENT_CUDA(expr)                                                  \
    do {                                                                   \
        const cudaError_t _e = (expr);                                     \
        if (_e != cudaSuccess) return fail_cuda(#expr, _e);                \
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

int validate_desc(const pa_latent_desc* d) {
    if (!d || d->struct_size != sizeof(pa_latent_desc)) return fail(PA_ERR_INVALID_ARG, "pa_latent_desc: NULL or struct_size mismatch");
    if (d->num_heads < 1 || d->num_heads > 1024) return fail(PA_ERR_INVALID_ARG, "num_heads must be 1 to 1024");
    if (d->latent_size != 256 && d->latent_size != 512) return fail(PA_ERR_UNSUPPORTED, "latent_size must be 256 or 512");
    if (d->rope_size != 32 && d->rope_size != 64) return fail(PA_ERR_UNSUPPORTED, "rope_size must be 32 or 64");
    if (d->nope_size != 64 && d->nope_size != 128) return fail(PA_ERR_UNSUPPORTED, "nope_size must be 64 or 128");
    if (d->value_size != 64 && d->value_size != 128) return fail(PA_ERR_UNSUPPORTED, "value_size must be 64 or 128");
    if (d->block_size != 16 && d->block_size != 32 && d->block_size != 64) return fail(PA_ERR_UNSUPPORTED, "block_size must be 16, 32 or 64");
    if (d->dtype != PA_DTYPE_F16 && d->dtype != PA_DTYPE_BF16) return fail(PA_ERR_UNSUPPORTED, "dtype must be f16 or bf16");
    return PA_OK;
}

const char kBadStride[] = "a stride is not positive or not a multiple of 8 elements";

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool strided(int64_t s) { return s > 0 && (s & 7) == 0; }
// A stride that is never stepped along may be anything: it is replaced.
int64_t used_stride(int64_t s, int64_t extent, int64_t instead) { return extent > 1 ? s : instead; }

size_t align_up(size_t x) { return (x + 1023) / 1024 * 1024; }

// ---- tensor maps ------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? (EncodeTiled)p : (EncodeTiled) nullptr;
    }();
    return fn;
}

// A map of 16-bit elements whose boxes are 64 elements wide and land 128-byte-swizzled; elements outside the tensor read as zero.
// sizes and box in elements, innermost first; strides in elements, of the dimensions behind the first.
bool make_map(CUtensorMap* map, int dtype, const void* base, int rank, const long long* sizes, const long long* strides, const int* box) {
    cuuint64_t dims[4], pitch[3];
    cuuint32_t b[4], one[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) { dims[i] = (cuuint64_t)sizes[i]; b[i] = (cuuint32_t)box[i]; }
    for (int i = 0; i + 1 < rank; ++i) pitch[i] = (cuuint64_t)strides[i] * 2;
    const EncodeTiled encode = encode_tiled();
    return encode && encode(map, dtype == PA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
                            dims, pitch, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// ---- scratch ------------------------------------------------------------------------------------------------------------

// Expanded keys and values of as many heads as fit this are made at a time.
constexpr size_t kExpandBytes = (size_t)1 << 30;

struct Scratch {
    int row_tiles, groups;
    long long part_rows;
    size_t unit_prefix, block_prefix, token_prefix, starts, q_abs, part_o, part_ml, row_part;
    int heads, passes;       // expanded: heads of a pass
    long long rows;
    size_t tile_prefix, query_prefix, order, heads_per_item, counter, arrived, split_o, split_ml, k, v, k_rope;
    int part_slots;
    size_t total;
};

// The scratch of a step.  `total` does not fall where tokens, sequences or block indices grow (what goes by the number of heads in a pass, which falls,
// takes its upper bound), so that the scratch of the largest step holds every smaller one of its form.
Scratch plan_scratch(const pa_latent_handle* h, int tokens, int sequences, int block_indices, int form) {
    const pa_latent_desc& d = h->desc;
    Scratch s{};
    // Two row tiles of a sequence read the same context: two CTAs walk it side by side, so that one of them finds it in the L2 cache
    s.row_tiles = d.num_heads > latent::kTile ? 2 : 1;
    s.groups = h->sm_count / s.row_tiles;
    size_t off = 0;
    auto take = [&](size_t bytes) { const size_t at = off; off += align_up(bytes); return at; };
    if (form != PA_LATENT_EXPANDED) {
        const size_t rows = (size_t)tokens * d.num_heads;
        // in an AUTO step only the short sequences' rows have partial results
        const int most = form == PA_LATENT_AUTO ? (int)std::min<long long>(tokens, (long long)sequences * latent::kAutoMaxNew) : tokens;
        s.part_rows = latent::absorbed_slots(most, sequences, d.num_heads, s.groups, s.row_tiles) * latent::kTile;
        s.unit_prefix = take(((size_t)sequences + 1) * sizeof(long long));
        s.block_prefix = take(((size_t)sequences + 1) * sizeof(int));
        s.token_prefix = take(((size_t)sequences + 1) * sizeof(int));
        s.starts = take(s.groups * sizeof(latent::SliceStart));
        s.q_abs = take(rows * (d.latent_size + d.rope_size) * 2);
        s.row_part = take(rows * sizeof(int2));
        s.part_ml = take((size_t)s.part_rows * sizeof(float2));
        s.part_o = take((size_t)s.part_rows * d.latent_size * sizeof(float));
    }
    if (form == PA_LATENT_EXPANDED || (form == PA_LATENT_AUTO && tokens > latent::kAutoFewNew)) {
        const int served = form == PA_LATENT_AUTO ? std::min(sequences, tokens / (latent::kAutoFewNew + 1)) : sequences;
        s.rows = ((long long)block_indices * d.block_size / latent::kExpandTile + served) * latent::kExpandTile;
        const size_t head = (size_t)s.rows * (d.nope_size + d.value_size) * 2;
        s.heads = (int)std::max<size_t>(1, std::min<size_t>(d.num_heads, kExpandBytes / std::max<size_t>(1, head)));
        s.passes = (d.num_heads + s.heads - 1) / s.heads;
        s.tile_prefix = take(((size_t)sequences + 1) * sizeof(int));
        s.query_prefix = take(((size_t)sequences + 1) * sizeof(int));
        s.part_slots = 2 * h->sm_count / s.heads * s.heads;      // (a pass of so many heads as CTAs cuts no context)
        if (s.heads >= h->sm_count) s.part_slots = 0;
        const size_t most_slots = 2 * (size_t)h->sm_count;
        s.order = take(((size_t)tokens / latent::kQueryTile + served + most_slots) * sizeof(latent::PieceOfQuery));
        s.arrived = take((size_t)s.passes * most_slots * 8 * sizeof(int));
        s.split_o = take(most_slots * latent::kQueryTile * d.value_size * sizeof(float));
        s.split_ml = take(most_slots * latent::kQueryTile * sizeof(float2));
        s.heads_per_item = take(2 * sizeof(int));
        s.counter = take((size_t)s.passes * sizeof(int));
        s.k_rope = take((size_t)s.rows * 64 * 2);
        // keys and values: all heads', or as much as a pass may take
        s.k = take(std::min(d.num_heads * head, std::max(kExpandBytes, head)) + align_up(1));
        s.v = s.k + align_up((size_t)s.heads * s.rows * d.nope_size * 2);
    }
    s.total = off;
    return s;
}

// What a reserve makes room for: an AUTO step's, and that of the same step in either form (the absorbed form by itself has partial results of all
// rows, the expanded one tiles of every sequence).
size_t reserved_bytes(const pa_latent_handle* h, int tokens, int sequences, int block_indices, int form) {
    size_t bytes = plan_scratch(h, tokens, sequences, block_indices, form).total;
    if (form == PA_LATENT_AUTO)
        for (int narrower : {PA_LATENT_ABSORBED, PA_LATENT_EXPANDED}) bytes = std::max(bytes, plan_scratch(h, tokens, sequences, block_indices, narrower).total);
    return bytes;
}

int ensure_ws(pa_latent_handle* h, size_t bytes, bool capturing) {
    if (bytes <= h->ws_bytes) {
        h->captured |= capturing;
        return PA_OK;
    }
    if (capturing) return fail(PA_ERR_TOO_LARGE, "the scratch would have to grow inside a stream capture: pa_b200_latent_reserve for the step beforehand");
    if (h->captured) h->retired.push_back(h->ws);
    else if (h->ws) LATENT_CUDA(cudaFree(h->ws));   // (waits for the work that uses it)
    h->ws = nullptr; h->ws_bytes = 0; h->captured = false;
    const size_t want = (bytes + bytes / 4 + (1 << 20) - 1) >> 20 << 20;
    LATENT_CUDA(cudaMalloc((void**)&h->ws, want));
    h->ws_bytes = want;
    return PA_OK;
}

// What both calls share.
template <class Args>
int validate_step(const Args* a) {
    if (a->num_tokens < 0 || a->num_sequences < 0 || a->num_blocks < 0 || a->num_block_indices < 0) return fail(PA_ERR_INVALID_ARG, "negative size");
    if (a->num_sequences > 65535) return fail(PA_ERR_TOO_LARGE, "more than 65535 sequences in one call");
    if (a->num_tokens == 0 || a->num_sequences == 0) return PA_OK;
    if (!a->past_lens || !a->subsequence_begins || !a->block_indices_begins || !a->cache) return fail(PA_ERR_INVALID_ARG, "NULL metadata or cache pointer");
    if (a->num_block_indices > 0 && !a->block_indices) return fail(PA_ERR_INVALID_ARG, "NULL block_indices");
    if (a->num_blocks == 0) return fail(PA_ERR_INVALID_ARG, "the cache has no blocks");
    if (!aligned(a->cache)) return fail(PA_ERR_UNSUPPORTED, "cache is not 16-byte aligned");
    return PA_OK;
}

template <class Args>
latent::Step make_step(const pa_latent_handle* h, const Args* a) {
    const pa_latent_desc& d = h->desc;
    return latent::Step{d.num_heads, d.latent_size, d.rope_size, d.nope_size, d.value_size, d.block_size,
                        a->num_tokens, a->num_sequences, a->num_block_indices, a->num_blocks,
                        a->past_lens, a->subsequence_begins, a->block_indices, a->block_indices_begins, h->status, PA_LATENT_AUTO, h->wait_polls};
}

int append(pa_latent_handle* h, const pa_latent_append_args* a) {
    if (!h) return fail(PA_ERR_INVALID_ARG, "NULL handle");
    if (!a || a->struct_size != sizeof(pa_latent_append_args)) return fail(PA_ERR_INVALID_ARG, "pa_latent_append_args: NULL or struct_size mismatch");
    const int rc = validate_step(a);
    if (rc != PA_OK) return rc;
    if (a->num_tokens == 0 || a->num_sequences == 0) return PA_OK;
    if (!a->latent || !a->rope_table) return fail(PA_ERR_INVALID_ARG, "NULL latent or rope_table");
    if (a->rope_table_rows <= 0) return fail(PA_ERR_INVALID_ARG, "rope_table has no rows");
    if ((a->query_rope != nullptr) != (a->query_rope_out != nullptr)) return fail(PA_ERR_INVALID_ARG, "query_rope and query_rope_out must be given together");
    if (!aligned(a->latent) || !aligned(a->norm_weight) || !aligned(a->query_rope) || !aligned(a->query_rope_out) || !aligned(a->rope_table))
        return fail(PA_ERR_UNSUPPORTED, "a tensor is not 16-byte aligned");
    const int T = a->num_tokens, H = h->desc.num_heads, P = h->desc.rope_size;
    const int64_t ls = used_stride(a->latent_stride, T, h->desc.latent_size + P);
    const int64_t qt = used_stride(a->query_rope_token_stride, T, H * P), qh = used_stride(a->query_rope_head_stride, H, P);
    const int64_t ot = used_stride(a->query_rope_out_token_stride, T, H * P), oh = used_stride(a->query_rope_out_head_stride, H, P);
    if (!strided(ls) || (a->query_rope && (!strided(qt) || !strided(qh) || !strided(ot) || !strided(oh))))
        return fail(PA_ERR_UNSUPPORTED, kBadStride);
    DeviceScope scope(h->device);
    LATENT_CUDA(scope.error);
    latent::AppendArgs k{make_step(h, a), a->latent, ls, a->norm_weight, a->norm_eps, a->query_rope, qt, qh, a->query_rope_out, ot, oh, a->rope_table,
                         a->rope_table_rows, a->interleaved, a->positions, a->cache};
    int launches = 0;
    LATENT_CUDA(latent::launch_append(k, h->desc.dtype, a->stream ? (cudaStream_t)a->stream : h->stream, &launches));
    h->launches += launches;
    return PA_OK;
}

int attention(pa_latent_handle* h, const pa_latent_attention_args* a) {
    if (!h) return fail(PA_ERR_INVALID_ARG, "NULL handle");
    if (!a || a->struct_size != sizeof(pa_latent_attention_args)) return fail(PA_ERR_INVALID_ARG, "pa_latent_attention_args: NULL or struct_size mismatch");
    if (a->form != PA_LATENT_AUTO && a->form != PA_LATENT_ABSORBED && a->form != PA_LATENT_EXPANDED) return fail(PA_ERR_INVALID_ARG, "unknown form");
    int rc = validate_step(a);
    if (rc != PA_OK) return rc;
    if (a->num_tokens == 0 || a->num_sequences == 0) return PA_OK;
    if (!a->query_nope || !a->query_rope || !a->key_up || !a->value_up || !a->output) return fail(PA_ERR_INVALID_ARG, "NULL query, weight or output pointer");
    if (!aligned(a->query_nope) || !aligned(a->query_rope) || !aligned(a->key_up) || !aligned(a->value_up) || !aligned(a->output))
        return fail(PA_ERR_UNSUPPORTED, "a tensor is not 16-byte aligned");
    const pa_latent_desc& d = h->desc;
    const int T = a->num_tokens, H = d.num_heads, R = d.latent_size, P = d.rope_size;
    const int64_t nt = used_stride(a->query_nope_token_stride, T, H * d.nope_size), nh = used_stride(a->query_nope_head_stride, H, d.nope_size);
    const int64_t rt = used_stride(a->query_rope_token_stride, T, H * P), rh = used_stride(a->query_rope_head_stride, H, P);
    const int64_t kh = used_stride(a->key_up_head_stride, H, (int64_t)d.nope_size * R), vh = used_stride(a->value_up_head_stride, H, (int64_t)d.value_size * R);
    if (!strided(nt) || !strided(nh) || !strided(rt) || !strided(rh) || !strided(kh) || !strided(vh)) return fail(PA_ERR_UNSUPPORTED, kBadStride);
    if (!(a->scale >= 0.f) || std::isinf(a->scale)) return fail(PA_ERR_INVALID_ARG, "scale is negative or not finite");
    if ((long long)T * H > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 query rows in one call");
    if ((long long)a->num_blocks * d.block_size > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 tokens of cache");
    DeviceScope scope(h->device);
    LATENT_CUDA(scope.error);
    const cudaStream_t stream = a->stream ? (cudaStream_t)a->stream : h->stream;
    const float scale = a->scale != 0.f ? a->scale : 1.f / sqrtf((float)(d.nope_size + P));
    const Scratch s = plan_scratch(h, T, a->num_sequences, a->num_block_indices, a->form);
    cudaStreamCaptureStatus capture;
    LATENT_CUDA(cudaStreamIsCapturing(stream, &capture));
    rc = ensure_ws(h, s.total, capture != cudaStreamCaptureStatusNone);
    if (rc != PA_OK) return rc;
    int launches = 0;
    if (a->form != PA_LATENT_EXPANDED) {
        latent::AbsorbedArgs k{};
        k.m = make_step(h, a);
        k.m.form = a->form;
        k.groups = s.groups; k.row_tiles = s.row_tiles;
        k.unit_prefix = (long long*)(h->ws + s.unit_prefix);
        k.block_prefix = (int*)(h->ws + s.block_prefix);
        k.token_prefix = (int*)(h->ws + s.token_prefix);
        k.starts = (latent::SliceStart*)(h->ws + s.starts);
        k.q_rope = a->query_rope; k.qr_token = rt; k.qr_head = rh;
        k.q_abs = h->ws + s.q_abs;
        k.part_o = (float*)(h->ws + s.part_o);
        k.part_ml = (float2*)(h->ws + s.part_ml);
        k.row_part = (int2*)(h->ws + s.row_part);
        k.part_rows = s.part_rows;
        k.output = a->output;
        k.scale_log2 = scale * 1.4426950408889634f;
        const int W = R + P;
        const long long qn_size[3] = {d.nope_size, H, T}, qn_stride[2] = {nh, nt};
        const long long ku_size[3] = {R, d.nope_size, H}, ku_stride[2] = {R, kh};
        const long long vu_size[3] = {R, d.value_size, H}, vu_stride[2] = {R, vh};
        // rows of latents in groups of eight, every 64-element chunk of a group 1024 bytes in shared memory; the rotated part by itself
        const long long groups = (long long)a->num_blocks * d.block_size / 8;
        const long long ca_size[4] = {64, 8, R / 64, groups}, ca_stride[3] = {W, 64, 8 * W}, cr_size[3] = {P, 8, groups}, cr_stride[2] = {W, 8 * W};
        const long long qa_size[3] = {64, (long long)T * H, R / 64}, qa_stride[2] = {W, 64}, qr_size[2] = {P, (long long)T * H}, qr_stride[1] = {W};
        const int box_tokens[3] = {64, 1, latent::kTile}, box_ku[3] = {64, d.nope_size, 1}, box_vu[3] = {64, d.value_size, 1};
        const int box_q[3] = {64, latent::kTile, R / 64}, box_qr[2] = {64, latent::kTile}, box_c[4] = {64, 8, R / 64, std::min(d.block_size, latent::kTokens / 2) / 8}, box_cr[3] = {64, 8, box_c[3]}, box_cp[4] = {64, 8, 2, box_c[3]};
        if (!make_map(&k.map_qn, d.dtype, a->query_nope, 3, qn_size, qn_stride, box_tokens) || !make_map(&k.map_key_up, d.dtype, a->key_up, 3, ku_size, ku_stride, box_ku) ||
            !make_map(&k.map_value_up, d.dtype, a->value_up, 3, vu_size, vu_stride, box_vu) || !make_map(&k.map_q_abs, d.dtype, k.q_abs, 3, qa_size, qa_stride, box_q) ||
            !make_map(&k.map_q_abs_rope, d.dtype, (const uint16_t*)k.q_abs + R, 2, qr_size, qr_stride, box_qr) ||
            !make_map(&k.map_cache, d.dtype, a->cache, 4, ca_size, ca_stride, box_c) || !make_map(&k.map_cache_part, d.dtype, a->cache, 4, ca_size, ca_stride, box_cp) || !make_map(&k.map_cache_rope, d.dtype, (const uint16_t*)a->cache + R, 3, cr_size, cr_stride, box_cr))
            return fail(PA_ERR_CUDA, "a tensor map could not be made");
        LATENT_CUDA(latent::launch_absorbed(k, d.dtype, stream, &launches));
    }
    if (s.passes > 0) {
        if (s.heads * s.rows > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 rows of expanded keys");
        latent::ExpandedArgs k{};
        k.m = make_step(h, a);
        k.m.form = a->form;
        k.rows = s.rows;
        k.tile_prefix = (int*)(h->ws + s.tile_prefix);
        k.query_prefix = (int*)(h->ws + s.query_prefix);
        k.order = (latent::PieceOfQuery*)(h->ws + s.order);
        k.items = (int*)(h->ws + s.heads_per_item) + 1;
        k.arrived = (int*)(h->ws + s.arrived);
        k.part_slots = s.part_slots;
        k.part_o = (float*)(h->ws + s.split_o);
        k.part_ml = (float2*)(h->ws + s.split_ml);
        k.counter = (int*)(h->ws + s.counter);
        k.heads_per_item = (int*)(h->ws + s.heads_per_item);
        k.passes = s.passes; k.ctas = h->sm_count; k.heads = s.heads;
        k.cache = a->cache;
        k.k_rope = h->ws + s.k_rope;
        k.output = a->output;
        k.scale_log2 = scale * 1.4426950408889634f;
        const int W = R + P;
        const long long ca_size[2] = {W, (long long)a->num_blocks * d.block_size}, ca_stride[1] = {W};
        const long long ku_size[3] = {R, d.nope_size, H}, ku_stride[2] = {R, kh}, vu_size[3] = {R, d.value_size, H}, vu_stride[2] = {R, vh};
        const long long qn_size[3] = {d.nope_size, H, T}, qn_stride[2] = {nh, nt}, qr_size[3] = {P, H, T}, qr_stride[2] = {rh, rt};
        const long long k_size[2] = {d.nope_size, s.heads * s.rows}, k_stride[1] = {d.nope_size}, v_size[2] = {d.value_size, s.heads * s.rows}, v_stride[1] = {d.value_size};
        const long long r_size[2] = {64, s.rows}, r_stride[1] = {64};
        const int box_c[2] = {64, d.block_size}, box_ku[3] = {64, d.nope_size, 1}, box_vu[3] = {64, d.value_size, 1}, box_q[3] = {64, 1, 128};
        const int box_out[2] = {64, 32}, box_k[2] = {64, latent::kExpandTile}, box_v[2] = {64, 64};
        if (!make_map(&k.map_cache, d.dtype, a->cache, 2, ca_size, ca_stride, box_c) || !make_map(&k.map_key_up, d.dtype, a->key_up, 3, ku_size, ku_stride, box_ku) ||
            !make_map(&k.map_value_up, d.dtype, a->value_up, 3, vu_size, vu_stride, box_vu) || !make_map(&k.map_k_out, d.dtype, h->ws + s.k, 2, k_size, k_stride, box_out) ||
            !make_map(&k.map_v_out, d.dtype, h->ws + s.v, 2, v_size, v_stride, box_out) || !make_map(&k.map_k, d.dtype, h->ws + s.k, 2, k_size, k_stride, box_k) ||
            !make_map(&k.map_v, d.dtype, h->ws + s.v, 2, v_size, v_stride, box_v) || !make_map(&k.map_k_rope, d.dtype, k.k_rope, 2, r_size, r_stride, box_k) ||
            !make_map(&k.map_qn, d.dtype, a->query_nope, 3, qn_size, qn_stride, box_q) || !make_map(&k.map_qr, d.dtype, a->query_rope, 3, qr_size, qr_stride, box_q))
            return fail(PA_ERR_CUDA, "a tensor map could not be made");
        LATENT_CUDA(latent::launch_expanded_plan(k, stream, &launches));
        for (k.pass = 0; k.pass < s.passes; ++k.pass) {
            k.h0 = k.pass * s.heads;
            k.heads = std::min(s.heads, H - k.h0);
            LATENT_CUDA(latent::launch_expanded(k, d.dtype, h->sm_count, stream, &launches));
        }
    }
    h->launches += launches;
    return PA_OK;
}

}  // namespace

extern "C" {

int pa_b200_latent_create(const pa_latent_desc* desc, int device, pa_latent_handle** out) {
    return guarded([&] {
        const int rc = validate_desc(desc);
        if (rc != PA_OK) return rc;
        if (!out) return fail(PA_ERR_INVALID_ARG, "NULL out pointer");
        int count = 0;
        if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) return fail(PA_ERR_NO_DEVICE, "no CUDA device");
        if (device < 0 || device >= count) return fail(PA_ERR_INVALID_ARG, "device ordinal out of range");
        cudaDeviceProp prop;
        LATENT_CUDA(cudaGetDeviceProperties(&prop, device));
        if (prop.major != 10) return fail(PA_ERR_NO_DEVICE, "this library is built for sm_100a only");
        DeviceScope scope(device);
        LATENT_CUDA(scope.error);
        pa_latent_handle* h = new (std::nothrow) pa_latent_handle();
        if (!h) return fail(PA_ERR_TOO_LARGE, "out of host memory");
        h->desc = *desc;
        h->device = device;
        h->sm_count = prop.multiProcessorCount;
        if (const char* e = std::getenv("PA_B200_LATENT_TEST_WAIT_POLLS")) h->wait_polls = (uint32_t)std::max(0, std::min(std::atoi(e), (int)latent::kWaitPolls));
        cudaError_t e = cudaStreamCreateWithFlags(&h->stream, cudaStreamNonBlocking);
        if (e == cudaSuccess) e = cudaMalloc((void**)&h->status, 256);
        if (e == cudaSuccess) e = cudaMemset(h->status, 0, 256);
        latent::Step sizes{};
        sizes.H = desc->num_heads; sizes.R = desc->latent_size; sizes.P = desc->rope_size; sizes.Dn = desc->nope_size; sizes.Dv = desc->value_size;
        if (e == cudaSuccess) e = latent::prepare_absorbed(sizes, desc->dtype);
        if (e == cudaSuccess) e = latent::prepare_expanded(sizes, desc->dtype);
        if (e != cudaSuccess) {
            pa_b200_latent_destroy(h);
            return fail_cuda("pa_b200_latent_create", e);
        }
        *out = h;
        return (int)PA_OK;
    });
}

int pa_b200_latent_destroy(pa_latent_handle* h) {
    if (!h) return PA_OK;
    DeviceScope scope(h->device);
    if (h->stream) cudaStreamSynchronize(h->stream);
    if (h->ws) cudaFree(h->ws);   // (waits for the work that uses it)
    for (uint8_t* p : h->retired) cudaFree(p);
    if (h->status) cudaFree(h->status);
    if (h->stream) cudaStreamDestroy(h->stream);
    delete h;
    return PA_OK;
}

int pa_b200_latent_append(pa_latent_handle* h, const pa_latent_append_args* a) {
    return guarded([&] { return append(h, a); });
}

int pa_b200_latent_attention(pa_latent_handle* h, const pa_latent_attention_args* a) {
    return guarded([&] { return attention(h, a); });
}

int pa_b200_latent_reserve(pa_latent_handle* h, int32_t num_tokens, int32_t num_sequences, int32_t num_block_indices, int32_t form) {
    return guarded([&] {
        if (!h) return fail(PA_ERR_INVALID_ARG, "NULL handle");
        if (num_tokens < 0 || num_sequences < 0 || num_block_indices < 0) return fail(PA_ERR_INVALID_ARG, "negative size");
        if (form != PA_LATENT_AUTO && form != PA_LATENT_ABSORBED && form != PA_LATENT_EXPANDED) return fail(PA_ERR_INVALID_ARG, "unknown form");
        DeviceScope scope(h->device);
        LATENT_CUDA(scope.error);
        return ensure_ws(h, reserved_bytes(h, num_tokens, num_sequences, num_block_indices, form), false);
    });
}

int pa_b200_latent_last_device_status(pa_latent_handle* h, uint32_t* status_bits) {
    return guarded([&] {
        if (!h || !status_bits) return fail(PA_ERR_INVALID_ARG, "NULL argument");
        DeviceScope scope(h->device);
        LATENT_CUDA(scope.error);
        LATENT_CUDA(cudaDeviceSynchronize());   // the calls may have gone to any stream
        LATENT_CUDA(cudaMemcpy(status_bits, h->status, 4, cudaMemcpyDeviceToHost));
        if (*status_bits) LATENT_CUDA(cudaMemset(h->status, 0, 4));
        return (int)PA_OK;
    });
}

int64_t pa_b200_latent_launch_count(const pa_latent_handle* h) { return h ? h->launches : -1; }

}  // extern "C"
