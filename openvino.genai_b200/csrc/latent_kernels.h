// Internal launch interface of latent attention, between the C ABI (latent_api.cu) and the kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/latent_b200.h"
#include "pa_common.cuh"

namespace latent {

// The step's paged metadata and the layer's sizes, passed by value.  All pointers are device memory.
struct Step {
    int H, R, P, Dn, Dv, bs;
    int num_tokens, num_sequences, num_block_indices, num_blocks;
    const int32_t* past_lens;
    const int32_t* subsequence_begins;
    const int32_t* block_indices;
    const int32_t* block_indices_begins;
    uint32_t* status;
    int form;        // pa_latent_form
    uint32_t wait_polls;   // looks at a barrier before a wait on it gives up
};
constexpr uint32_t kWaitPolls = 1u << 22;

// Form of a sequence in an AUTO step.  With n new tokens over L tokens of context the absorbed form costs a n L and the expanded one b n L + c L, so the
// number of new tokens decides: with 4 sequences of 2000 cached tokens by 64 heads, 64 new tokens each took 158 us absorbed and 220
// expanded, 96 took 225 and 222, 128 299 and 219 (with 16 sequences 622 and 898, 913 and 889, 1229 and 884).  Short contexts leave the absorbed form with
// more results than work (16 sequences of 64 tokens by 16 heads 62 and 35 us).
// The rule runs on the device, so the host lays out and launches the expanded form for whatever the whole step's block tables allow: 64 rows over
// 259,540 tokens by 128 heads take 137 us, 3 launches and 60 MiB in the absorbed form and 211 us, 36 launches (33 find no work) and 1424 MiB under AUTO; 4
// prompts by 32 heads 450 us expanded and 547 under AUTO, whose query projection loads before it knows that no token is its own.
constexpr int kAutoMaxNew = 80, kAutoFewNew = 16, kAutoContext = 8;

struct AppendArgs {
    Step m;
    const void* latent;
    long long latent_stride;
    const void* norm_weight;
    float norm_eps;
    const void* q_in;
    long long q_in_token, q_in_head;
    void* q_out;
    long long q_out_token, q_out_head;
    const float* rope_table;
    int rope_rows;
    int interleaved;
    const int32_t* positions;
    void* cache;
};

// The absorbed form.  Its unit of work is a tile of 64 context tokens for a block of `row_tiles` tiles of 64 query rows (new token, head) of one
// sequence; sequence s has block_prefix[s + 1] - block_prefix[s] such blocks, every one of the same number of tiles.  Units are
// numbered by sequence, block and tile, and group w of `row_tiles` CTAs takes the w-th of equal slices; a block leaves one partial result
// for every group that has a part of it, in slot (block + group) * row_tiles + row tile.
constexpr int kTile = 64;      // query rows of a row tile, new tokens of a projection's tile
constexpr int kTokens = 64;    // context tokens of a tile

// Where a group's slice begins: sequence (-1: no units) and what there is to know of it, row block of the sequence, context tile of the block; and
// the slice's units.
struct __align__(16) SliceStart {
    int s, block, first, units;
    int t0, n, past, tb;            // of the sequence (SeqView)
    int blocks, tiles;              // its row blocks, and context tiles of each
    int block0;                     // row blocks of the sequences before
    int per;                        // units of a whole slice
};

struct AbsorbedArgs {
    Step m;
    int groups, row_tiles;
    long long* unit_prefix;     // [num_sequences + 1]
    int* block_prefix;          // [num_sequences + 1]
    int* token_prefix;          // [num_sequences + 1], tokens of the sequences of this form
    SliceStart* starts;         // [groups]
    const void* q_rope;
    long long qr_token, qr_head;
    void* q_abs;                // [num_tokens * H][R + P] absorbed query rows
    float* part_o;              // [slot][64][R]
    float2* part_ml;            // [slot][64] maximum (base 2, scaled) and sum
    int2* row_part;             // [num_tokens * H] a row's first partial result (slot * 64 + row of the tile) and how many it has
    long long part_rows;        // rows of part_o and part_ml
    void* output;
    float scale_log2;           // softmax scale * log2(e)
    CUtensorMap map_qn, map_key_up, map_q_abs, map_q_abs_rope, map_cache, map_cache_part, map_cache_rope, map_value_up;
};
// A row's record as the join may follow it: its `part.y` partial results lie `step` rows apart among the `rows` of the scratch.  A record that the
// attention left unwritten, because a wait of its CTA ran out, is whatever an earlier call had there: one that leads outside has no results.
__host__ __device__ inline int2 checked_part(int2 part, int step, long long rows) {
    const bool inside = part.x >= 0 && part.y > 0 && part.x + (part.y - 1LL) * step < rows;
    return inside ? part : make_int2(0, 0);
}
// Largest number of slots a step can need.
long long absorbed_slots(int tokens, int sequences, int heads, int groups, int row_tiles);
cudaError_t launch_absorbed(const AbsorbedArgs& a, int dtype, cudaStream_t stream, int* launches);

// The expanded form.  Keys and values of the context are made per head in scratch, whose rows are the contexts of the served sequences one
// after another, each in whole tiles of 128 tokens (rows behind a context are zero); then every (256 new tokens, head) attends over them.
constexpr int kExpandTile = 128;   // context tokens of a tile
constexpr int kQueryTile = 256;    // new tokens of a work item, in two halves

// A query tile's piece of context: `length` tiles from number piece * length.
struct PieceOfQuery {
    int s, tile, piece, length;
    int slot;                   // of the tile's first piece, -1: the only one
};

struct ExpandedArgs {
    Step m;
    int h0, heads;              // heads of this pass
    long long rows;             // rows of a head's scratch
    int* tile_prefix;           // [num_sequences + 1] context tiles
    int* query_prefix;          // [num_sequences + 1] query tiles
    PieceOfQuery* order;        // the longest first
    int* items;                 // their number
    int* arrived;               // [passes][part_slots][8] pieces done, of every 32 rows
    int part_slots;             // (pieces, heads) of query tiles with more than one piece
    float* part_o;              // [part_slots][value / 4][kQueryTile][4] their sums
    float2* part_ml;            // [part_slots][kQueryTile] maximum and denominator
    int* heads_per_item;        // heads that a CTA makes keys and values of for one context tile
    int* counter;               // [passes] work counters
    int pass, passes, ctas;
    const void* cache;
    void* k_rope;               // [rows][64] rotated key part (the same for every head)
    void* output;
    float scale_log2;           // softmax scale * log2(e)
    // k, v: the scratch [heads * rows][Dn] and [heads * rows][Dv], written 32 rows and read 128 (k) or 64 (v) rows at a time
    CUtensorMap map_cache, map_key_up, map_value_up, map_k_out, map_v_out, map_k, map_v, map_k_rope, map_qn, map_qr;
};
cudaError_t launch_expanded_plan(const ExpandedArgs& a, cudaStream_t stream, int* launches);
cudaError_t launch_expanded(const ExpandedArgs& a, int dtype, int sm_count, cudaStream_t stream, int* launches);

// What a kernel's launches need once on every device.
cudaError_t prepare_absorbed(const Step& m, int dtype);
cudaError_t prepare_expanded(const Step& m, int dtype);

cudaError_t launch_append(const AppendArgs& a, int dtype, cudaStream_t stream, int* launches);

#ifdef __CUDACC__
// One sequence's slice of the metadata, checked before anything is indexed with it: begins monotone and inside the arrays they
// index, past_len >= 0, and a block table long enough for past_len + new tokens.  A sequence that fails sets its status bit
// and gets no work.
struct SeqView {
    int t0, n;      // its new tokens
    int past;
    int tb;         // its block table inside block_indices
};
__device__ __forceinline__ bool seq_view(const Step& m, int s, SeqView& v) {
    const int t0 = m.subsequence_begins[s], t1 = m.subsequence_begins[s + 1];
    const int tb = m.block_indices_begins[s], te = m.block_indices_begins[s + 1];
    const int past = m.past_lens[s];
    v = SeqView{0, 0, 0, 0};
    if (t0 < 0 || t1 < t0 || t1 > m.num_tokens || tb < 0 || te < tb || te > m.num_block_indices) {
        atomicOr(m.status, PA_DEV_BAD_BEGINS);
        return false;
    }
    if (past < 0 || (long long)(te - tb) * m.bs < (long long)past + (t1 - t0)) {
        atomicOr(m.status, PA_DEV_BAD_PAST_LEN);
        return false;
    }
    v = SeqView{t0, t1 - t0, past, tb};
    return true;
}

__device__ __forceinline__ bool takes_absorbed(const Step& m, const SeqView& v) {
    if (m.form != PA_LATENT_AUTO) return m.form == PA_LATENT_ABSORBED;
    return v.n <= kAutoFewNew || (v.n <= kAutoMaxNew && (long long)v.n * kAutoContext <= (long long)v.past + v.n);
}

// The sequence that owns token t.  In a step of one token each that is sequence t, which two loads show; else a binary search.
__device__ __forceinline__ int find_sequence(const Step& m, int t) {
    if (t < m.num_sequences && m.subsequence_begins[t] == t && m.subsequence_begins[t + 1] == t + 1) return t;
    int lo = 0, hi = m.num_sequences;   // begins[lo] <= t < begins[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (m.subsequence_begins[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

// Sequence and checked view of token t; false (with the status bit set) where the prefix sums leave it out.
__device__ __forceinline__ bool token_view(const Step& m, int t, SeqView& v) {
    if (!seq_view(m, find_sequence(m, t), v)) return false;
    if (t < v.t0 || t >= v.t0 + v.n) {
        atomicOr(m.status, PA_DEV_BAD_BEGINS);
        return false;
    }
    return true;
}
#endif

}  // namespace latent
