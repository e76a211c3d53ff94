/*
 * latent_b200.h - C ABI of latent attention on the B200 (sm_100a): attention whose keys and values all come from one
 * cached vector a token.
 *
 * A token's cache row is [ c (latent_size) | k_r (rope_size) ], shared by every head.  With the layer's up-projections
 * key_up[h] (nope_size x latent_size) and value_up[h] (value_size x latent_size) the logit of query row (t, h) and context
 * position j <= position of t is
 *     s = scale * ( query_nope[t,h] . (key_up[h] c_j) + query_rope[t,h] . k_r,j ),
 * and the output row is value_up[h] * sum_j softmax_j(s) c_j.  The products may be grouped in two ways:
 *     absorbed   q~ = key_up[h]^T query_nope, o~ = sum_j p_j c_j, output = value_up[h] o~.  Per (row, position) pair
 *                2 (2 latent_size + rope_size) operations, and the cache is read as it is: decode rows, a few drafted tokens.
 *     expanded   k_j = key_up[h] c_j and v_j = value_up[h] c_j for the whole context once, then attention per head.  Per pair
 *                2 (nope_size + rope_size + value_size) operations: prompts.
 *
 * Conventions are those of pa_b200.h: plain C, status codes (pa_status), no exceptions across the boundary, the text of
 * the last error of this thread from pa_b200_last_error(), a device status word (PA_DEV_*) in place of faults, one engine thread
 * per handle, calls on one handle ordered on one stream.  Metadata tensors have the names, types and meaning that
 * pa_b200_forward gives them.
 */
#ifndef LATENT_B200_H
#define LATENT_B200_H

#include "pa_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Device status bit, beside those of pa_b200.h: a bounded wait of an attention kernel ran out; the step's output is incomplete. */
#define PA_DEV_WAIT_TIMEOUT_LATENT 0x10000000u

/* Static attributes of a layer.  Layers of the same attributes share a handle, whose scratch (gigabytes for long prompts by many heads) then serves them in
 * turn: every call brings its own weights, cache and metadata. */
typedef struct pa_latent_desc {
    uint32_t struct_size; /* sizeof(pa_latent_desc)                                               */
    int32_t num_heads;    /* 1 .. 1024                                                            */
    int32_t latent_size;  /* 256 or 512                                                           */
    int32_t rope_size;    /* 32 or 64                                                             */
    int32_t nope_size;    /* unrotated query / key elements per head: 64 or 128                   */
    int32_t value_size;   /* value elements per head: 64 or 128                                   */
    int32_t block_size;   /* tokens per physical block: 16, 32 or 64                              */
    int32_t dtype;        /* pa_dtype of activations, weights and cache: F16 or BF16              */
} pa_latent_desc;

/* Every data pointer below is 16-byte aligned, and every stride is a multiple of 8 elements (PA_ERR_UNSUPPORTED
 * otherwise).  Strides count elements; the innermost dimension is contiguous. */

/* Writes the new tokens' rows into the paged cache, normalised and rotated, and rotates the queries' part:
 *   cache row = [ latent[:R] * rsqrt(mean(latent[:R]^2) + norm_eps) * norm_weight | rotate(latent[R:], pos) ]
 *   query_rope_out[t,h] = rotate(query_rope[t,h], pos)
 * in f32, rounded once.  pos is past_len + index in the chunk, or positions[t].  rotate pairs element j with j + P/2, or,
 * interleaved, 2j with 2j + 1:  (a, b) -> (a cos - b sin, b cos + a sin). */
typedef struct pa_latent_append_args {
    uint32_t struct_size;
    const void* latent;            /* [num_tokens, latent_size + rope_size]                                     */
    int64_t latent_stride;         /* elements from one token to the next                                       */
    const void* norm_weight;       /* [latent_size], or NULL: the latent is written as it is                    */
    float norm_eps;
    const void* query_rope;        /* [num_tokens, num_heads, rope_size], or NULL: no queries to rotate         */
    int64_t query_rope_token_stride, query_rope_head_stride;
    void* query_rope_out;          /* may be query_rope itself                                                  */
    int64_t query_rope_out_token_stride, query_rope_out_head_stride;
    const float* rope_table;       /* [rope_table_rows, rope_size]: cos of the P/2 angles, then their sin       */
    int32_t rope_table_rows;       /* a position outside the table sets PA_DEV_BAD_ROTATION, its token is skipped */
    int32_t interleaved;
    const int32_t* positions;      /* [num_tokens] or NULL                                                      */
    int32_t num_tokens;
    void* cache;                   /* [num_blocks, block_size, latent_size + rope_size]                         */
    int32_t num_blocks;
    const int32_t* past_lens;            /* [num_sequences]     */
    const int32_t* subsequence_begins;   /* [num_sequences + 1] */
    const int32_t* block_indices;        /* [num_block_indices] */
    const int32_t* block_indices_begins; /* [num_sequences + 1] */
    int32_t num_sequences;
    int32_t num_block_indices;
    void* stream;                  /* cudaStream_t, NULL => the handle's stream */
} pa_latent_append_args;

enum pa_latent_form {
    /* Every sequence in the form that suits its number of new tokens.  Which that is, is known on the device only: the expanded form's scratch and passes
     * go by the block tables of the whole step, and both forms' kernels are launched as soon as there are more than 16 tokens.  A step that the
     * caller knows to hold single tokens and drafts only, or prompts only, is served faster and in less scratch by its form's name. */
    PA_LATENT_AUTO = 0,
    PA_LATENT_ABSORBED = 1,
    PA_LATENT_EXPANDED = 2
};

/* Attention of the new tokens over the cache, which holds their own rows already (pa_b200_latent_append first).
 * A row whose logits hold not-a-number or plus infinity has no softmax and its output is not finite, whichever form serves it; nor is that of one whose
 * intermediates leave the type (with F16: key_up[h]^T query_nope beyond 65504 in the absorbed form, keys and values beyond it in the expanded one). */
typedef struct pa_latent_attention_args {
    uint32_t struct_size;
    const void* query_nope;        /* [num_tokens, num_heads, nope_size] */
    int64_t query_nope_token_stride, query_nope_head_stride;
    const void* query_rope;        /* [num_tokens, num_heads, rope_size], rotated */
    int64_t query_rope_token_stride, query_rope_head_stride;
    const void* key_up;            /* [num_heads, nope_size, latent_size], rows contiguous */
    int64_t key_up_head_stride;
    const void* value_up;          /* [num_heads, value_size, latent_size], rows contiguous */
    int64_t value_up_head_stride;
    void* output;                  /* [num_tokens, num_heads * value_size] */
    int32_t num_tokens;
    const void* cache;
    int32_t num_blocks;
    const int32_t* past_lens;
    const int32_t* subsequence_begins;
    const int32_t* block_indices;
    const int32_t* block_indices_begins;
    int32_t num_sequences;
    int32_t num_block_indices;
    float scale;                   /* 0 => 1/sqrt(nope_size + rope_size) */
    int32_t form;                  /* pa_latent_form */
    void* stream;
} pa_latent_attention_args;

typedef struct pa_latent_handle pa_latent_handle;

int pa_b200_latent_create(const pa_latent_desc* desc, int device, pa_latent_handle** out);
int pa_b200_latent_destroy(pa_latent_handle* h);
int pa_b200_latent_append(pa_latent_handle* h, const pa_latent_append_args* args);
int pa_b200_latent_attention(pa_latent_handle* h, const pa_latent_attention_args* args);

/* The handle's scratch grows when a call needs more (cudaMalloc; inside a stream capture such a call is PA_ERR_TOO_LARGE).  After reserve, attention
 * calls of no more tokens, sequences and block indices, in the same form or, behind an AUTO reserve, in any, do not allocate.  A graph names the scratch
 * of its capture, which the handle keeps until it is destroyed, whatever grows since; replays and calls of one handle stay ordered on one stream. */
int pa_b200_latent_reserve(pa_latent_handle* h, int32_t num_tokens, int32_t num_sequences, int32_t num_block_indices, int32_t form);

/* Reads (and clears) the device status word; synchronises the device's work on it. */
int pa_b200_latent_last_device_status(pa_latent_handle* h, uint32_t* status_bits);
/* Kernels launched by this handle since its creation. */
int64_t pa_b200_latent_launch_count(const pa_latent_handle* h);

#ifdef __cplusplus
}
#endif
#endif /* LATENT_B200_H */
