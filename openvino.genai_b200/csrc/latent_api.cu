// C ABI of latent attention (include/latent_b200.h): argument checking, scratch and launch sequencing.
#include <cuda_runtime.h>

#include <climits>
#include <new>
#include <string>

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
    int64_t launches = 0;
};

namespace {

int fail(int code, const char* msg) {
    pa::set_last_error(msg);
    return code;
}

int fail_cuda(const char* what, cudaError_t e) {
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

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool strided(int64_t s) { return s >= 0 && (s & 7) == 0; }

// What both calls share.
template <class Args>
int validate_step(const Args* a) {
    if (a->num_tokens < 0 || a->num_sequences < 0 || a->num_blocks < 0 || a->num_block_indices < 0) return fail(PA_ERR_INVALID_ARG, "negative size");
    if (a->num_sequences > 65535) return fail(PA_ERR_TOO_LARGE, "more than 65535 sequences in one call");
    if (a->num_tokens == 0 || a->num_sequences == 0) return PA_OK;
    if (!a->past_lens || !a->subsequence_begins || !a->block_indices_begins || !a->cache) return fail(PA_ERR_INVALID_ARG, "NULL metadata or cache pointer");
    if (a->num_block_indices > 0 && !a->block_indices) return fail(PA_ERR_INVALID_ARG, "NULL block_indices");
    if (!aligned(a->cache)) return fail(PA_ERR_UNSUPPORTED, "cache is not 16-byte aligned");
    return PA_OK;
}

template <class Args>
latent::Step make_step(const pa_latent_handle* h, const Args* a) {
    const pa_latent_desc& d = h->desc;
    return latent::Step{d.num_heads, d.latent_size, d.rope_size, d.nope_size, d.value_size, d.block_size,
                        a->num_tokens, a->num_sequences, a->num_block_indices, a->num_blocks,
                        a->past_lens, a->subsequence_begins, a->block_indices, a->block_indices_begins, h->status};
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
    if (!strided(a->latent_stride) || !strided(a->query_rope_token_stride) || !strided(a->query_rope_head_stride) ||
        !strided(a->query_rope_out_token_stride) || !strided(a->query_rope_out_head_stride))
        return fail(PA_ERR_UNSUPPORTED, "a stride is negative or not a multiple of 8 elements");
    DeviceScope scope(h->device);
    LATENT_CUDA(scope.error);
    latent::AppendArgs k{make_step(h, a), a->latent, a->latent_stride, a->norm_weight, a->norm_eps,
                         a->query_rope, a->query_rope_token_stride, a->query_rope_head_stride,
                         a->query_rope_out, a->query_rope_out_token_stride, a->query_rope_out_head_stride,
                         a->rope_table, a->rope_table_rows, a->interleaved, a->positions, a->cache};
    int launches = 0;
    LATENT_CUDA(latent::launch_append(k, h->desc.dtype, a->stream ? (cudaStream_t)a->stream : h->stream, &launches));
    h->launches += launches;
    return PA_OK;
}

int attention(pa_latent_handle* h, const pa_latent_attention_args* a) {
    if (!h) return fail(PA_ERR_INVALID_ARG, "NULL handle");
    if (!a || a->struct_size != sizeof(pa_latent_attention_args)) return fail(PA_ERR_INVALID_ARG, "pa_latent_attention_args: NULL or struct_size mismatch");
    if (a->form != PA_LATENT_AUTO && a->form != PA_LATENT_ABSORBED && a->form != PA_LATENT_EXPANDED) return fail(PA_ERR_INVALID_ARG, "unknown form");
    const int rc = validate_step(a);
    if (rc != PA_OK) return rc;
    if (a->num_tokens == 0 || a->num_sequences == 0) return PA_OK;
    if (!a->query_nope || !a->query_rope || !a->key_up || !a->value_up || !a->output) return fail(PA_ERR_INVALID_ARG, "NULL query, weight or output pointer");
    if (!aligned(a->query_nope) || !aligned(a->query_rope) || !aligned(a->key_up) || !aligned(a->value_up) || !aligned(a->output))
        return fail(PA_ERR_UNSUPPORTED, "a tensor is not 16-byte aligned");
    if (!strided(a->query_nope_token_stride) || !strided(a->query_nope_head_stride) || !strided(a->query_rope_token_stride) ||
        !strided(a->query_rope_head_stride) || !strided(a->key_up_head_stride) || !strided(a->value_up_head_stride))
        return fail(PA_ERR_UNSUPPORTED, "a stride is negative or not a multiple of 8 elements");
    if ((long long)a->num_tokens * h->desc.num_heads > INT_MAX) return fail(PA_ERR_TOO_LARGE, "more than 2^31 query rows in one call");
    DeviceScope scope(h->device);
    LATENT_CUDA(scope.error);
    const float scale = a->scale != 0.f ? a->scale : 1.f / sqrtf((float)(h->desc.nope_size + h->desc.rope_size));
    latent::AttentionArgs k{make_step(h, a), a->query_nope, a->query_nope_token_stride, a->query_nope_head_stride,
                            a->query_rope, a->query_rope_token_stride, a->query_rope_head_stride, a->key_up, a->key_up_head_stride,
                            a->value_up, a->value_up_head_stride, a->output, a->cache, scale};
    int launches = 0;
    LATENT_CUDA(latent::launch_attention_simple(k, h->desc.dtype, a->stream ? (cudaStream_t)a->stream : h->stream, &launches));
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
        cudaError_t e = cudaStreamCreateWithFlags(&h->stream, cudaStreamNonBlocking);
        if (e == cudaSuccess) e = cudaMalloc((void**)&h->status, 256);
        if (e == cudaSuccess) e = cudaMemset(h->status, 0, 256);
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
