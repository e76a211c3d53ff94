/*
 * masked_b200.h - C ABI of attention over the paged cache under masks other than the causal one, on the B200 (sm_100a), and of
 * what a speculative step does with the cache once its drafts are judged.
 *
 * pa_b200_forward_masked is pa_b200_forward (same handle, same caches, same metadata; the new tokens' keys and values are written
 * first) with a narrower set of visible positions.  Per query row, with `position` its place in the context:
 *
 *   sliding window W, sinks S    the cached positions j with  j < S  or  j > position - W   (W = 0: all of them)
 *   no tree                      position = past_len + index in the chunk; every token of the chunk in front of the row, by the same rule
 *   a tree of drafted tokens     position = past_len + depth in the tree; of the chunk only the row's ancestors and itself, by the same rule
 *                                with their own positions
 *
 * Blocks that no row of the step sees are neither looked up nor read: their entries of block_indices may hold anything, so that a cache
 * manager may give blocks back once the window has left them behind.  Positions that a row does not see take no part in it, whatever their bytes
 * are, not-a-number and infinities included: a row of a chunk whose result is not finite is computed again by a slow path, so that a step of which
 * most rows rightly are not finite takes far longer than another.  So are the rows of chunks that see a token of a u8 cache whose step is 511 or more.
 *
 * Conventions are those of pa_b200.h: plain C, status codes, the text of the last error of this thread from pa_b200_last_error(), a
 * device status word (PA_DEV_*) in place of faults.  The caller's current device is left as it was.
 */
#ifndef MASKED_B200_H
#define MASKED_B200_H

#include "pa_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Device status bit, beside those of pa_b200.h: a parent that is not in front of its child, or a tree of too many tokens. */
#define PA_DEV_BAD_TREE 0x10u

/* Tokens of one sequence's tree, at most.  A sequence that brings more is skipped: its keys and values are written, its output rows are not. */
#define PA_TREE_MAX_TOKENS 256

/* tree_parents of a sequence's first token that has no tree: its tokens follow one another (a prompt, a single token). */
#define PA_TREE_NONE (-2)

typedef struct pa_mask_args {
    uint32_t struct_size;        /* sizeof(pa_mask_args) */
    int32_t sliding_window;      /* W >= 0; 0: no window */
    int32_t sink_tokens;         /* S >= 0 */
    /* [num_tokens], device memory, or NULL: no sequence has a tree.  The index of the token's parent among its sequence's new tokens,
     * smaller than its own; -1: it follows the last cached token; PA_TREE_NONE at a sequence's first token: no tree.  A
     * parent out of range sets PA_DEV_BAD_TREE and counts as -1. */
    const int32_t* tree_parents;
} pa_mask_args;

/* The operator: every pointer in `args` and `mask` is device memory, query, output and the caches 16-byte aligned (PA_ERR_UNSUPPORTED
 * otherwise); args->sliding_window is 0, the mask has it.  No score output (PA_ERR_UNSUPPORTED): scores are those of causal rows.  Asynchronous on
 * the stream.  The handle's scratch grows when a call needs more; inside a stream capture such a call is PA_ERR_TOO_LARGE.  Graphs name the scratch
 * of their capture, which the handle keeps until it is destroyed; replays and calls of one handle stay ordered on one stream.
 * pa_b200_last_prefill_kernel tells of masked steps too (row by row: PA_PREFILL_GENERIC; PA_PREFILL_NONE of as many tokens as sequences), the kernel
 * timing of pa_b200.h of causal ones only.
 * Two kinds of chunks are served row by row, far from the tensor cores' pace: those over a bf16 cache under f16 or f32 activations, and those of a step with
 * exactly as many tokens as sequences (some of them without tokens), which is taken for one of single tokens. */
int pa_b200_forward_masked(pa_handle* h, const pa_forward_args* args, const pa_mask_args* mask);

/* The same for host tensors, as pa_b200_forward_host takes them (the caches stay device memory). */
int pa_b200_forward_masked_host(pa_handle* h, const pa_forward_args* args, const pa_mask_args* mask);

/* Grows the scratch for masked calls of up to so many tokens, sequences and block indices (which take none), which then do not allocate.  From two tokens on it holds
 * what chunks take, 39 MB for the tensor cores' partial results at a head size of 128; a handle whose steps are all of single tokens does not take them
 * by itself.  Layers of one geometry whose steps follow one another on one stream can share a handle. */
int pa_b200_masked_reserve(pa_handle* h, int32_t num_tokens, int32_t num_sequences, int32_t num_block_indices);

/* Judges trees of drafts and makes the accepted ones the cache's newest tokens.
 *
 * A sequence's first new token is certain (its id was sampled before the step).  From an accepted token a, the step goes on to
 * its first child c with draft_tokens[c] == sampled_tokens[a], where sampled_tokens[a] is what the sampler gave for the logits of a, until
 * there is none, or the path is max_path long.  The keys and values of the k-th accepted token are then moved from position
 * past_len + path[k] to past_len + k in every layer's caches, so that the next step's past_len is past_len + num_accepted.
 * A sequence without a tree (PA_TREE_NONE) keeps all of its tokens where they are.  All pointers are device memory but the two
 * arrays of cache pointers; asynchronous on the stream; no scratch. */
typedef struct pa_tree_accept_args {
    uint32_t struct_size;
    const int32_t* tree_parents;         /* [num_tokens] as above                                                  */
    const int64_t* draft_tokens;         /* [num_tokens] ids of the new tokens                                      */
    const int64_t* sampled_tokens;       /* [num_tokens] ids sampled behind them                                    */
    const int32_t* past_lens;            /* [num_sequences]     */
    const int32_t* subsequence_begins;   /* [num_sequences + 1] */
    const int32_t* block_indices;        /* [num_block_indices] */
    const int32_t* block_indices_begins; /* [num_sequences + 1] */
    int32_t num_tokens;
    int32_t num_sequences;
    int32_t num_block_indices;
    int32_t num_blocks;                  /* physical blocks in each cache tensor                                    */
    int32_t max_path;                    /* 1 .. PA_TREE_MAX_TOKENS: row length of `path`, the longest path taken   */
    int32_t num_layers;                  /* 0: nothing is moved                                                     */
    void* const* key_caches;             /* [num_layers] host array of device pointers, 16-byte aligned; no two overlap */
    void* const* value_caches;
    int32_t* path;                       /* out [num_sequences][max_path] accepted tokens, ascending; -1 behind them, and everywhere
                                          * for a sequence without a tree                                           */
    int32_t* num_accepted;               /* out [num_sequences]; all tokens of a sequence without a tree; 0: the sequence has no tokens, or metadata
                                          * or a tree that set the status word: too many tokens, or any parent out of range (of which the attention
                                          * makes a follower of the cache; here nothing of such a tree is accepted or moved) */
    int64_t* next_token;                 /* out [num_sequences] id sampled behind the last accepted token, -1: none */
    int32_t* new_past_lens;              /* out [num_sequences] past_len + num_accepted, or NULL; may be past_lens  */
    void* stream;                        /* cudaStream_t, NULL => the handle's stream */
} pa_tree_accept_args;
int pa_b200_tree_accept(pa_handle* h, const pa_tree_accept_args* args);

#ifdef __cplusplus
}
#endif
#endif /* MASKED_B200_H */
