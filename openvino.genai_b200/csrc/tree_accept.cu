// Acceptance of drafted trees (include/masked_b200.h): the walk down every tree by the sampled tokens, and the accepted tokens'
// keys and values moved to where the next step's context begins.
//
// Nothing is computed, so the bound is launches and chains of loads: a walk is one block per sequence that looks at all of its tokens at once, per
// step of the path one comparison a thread and one barrier; a moved row is read and written once, all of a path's rows in flight together.
#include "pa_common.cuh"
#include "pa_kernels.h"

#include "../../include/masked_b200.h"

namespace pa {

namespace {

static_assert(kTreeMax == PA_TREE_MAX_TOKENS && kTreeNone == PA_TREE_NONE, "as the header says");

// One sequence's metadata, checked before anything is indexed with it.
__device__ __forceinline__ bool accept_view(const TreeAcceptArgs& a, int s, SeqView& v, bool report) {
    const int t0 = a.subsequence_begins[s], t1 = a.subsequence_begins[s + 1], tb = a.block_indices_begins[s], te = a.block_indices_begins[s + 1];
    const int past = a.past_lens[s];
    uint32_t bad = 0;
    if (t0 < 0 || t1 < t0 || t1 > a.num_tokens || tb < 0 || te < tb || te > a.num_block_indices) bad = PA_DEV_BAD_BEGINS;
    else if (past < 0 || (long long)(te - tb) * a.g.bs < (long long)past + (t1 - t0)) bad = PA_DEV_BAD_PAST_LEN;
    if (bad && report) atomicOr(a.status, bad);
    v = bad ? SeqView{0, 0, 0, 0, 0} : SeqView{t0, t1 - t0, past, tb, te - tb};
    return bad == 0;
}

__global__ void __launch_bounds__(kTreeMax) tree_walk_kernel(TreeAcceptArgs a) {
    __shared__ int sh_next[3];   // a turn's offers, taken from three in turn: one is offered to and read, the next one is cleared, the last one may still be read
    grid_wait();
    const int s = blockIdx.x, i = threadIdx.x;
    SeqView v;
    accept_view(a, s, v, i == 0);
    const bool tree = v.n > 0 && a.parents[v.t0] != kTreeNone;
    int parent = -1;
    int64_t draft = 0;
    bool bad = tree && v.n > kTreeMax;
    if (tree && !bad && i < v.n) {
        parent = a.parents[v.t0 + i];
        draft = a.draft[v.t0 + i];
        bad = parent < -1 || parent >= i;
    }
    // one parent that is none: who knows what the drafts were judged by, so none of them is accepted and nothing is moved
    bad = __syncthreads_or(bad) != 0;
    if (bad && i == 0) atomicOr(a.status, PA_DEV_BAD_TREE);
    const bool walk = tree && !bad;
    int32_t* path = a.path + (long long)s * a.max_path;
    int at = walk ? 0 : -1, count = 0;
    if (i == 0) sh_next[0] = kTreeMax;   // (turn 0's)
    // one step of the path a turn: the children that carry the sampled token offer themselves, the first one is it
    while (at >= 0) {
        int* const next = &sh_next[count % 3];
        if (i == 0) { path[count] = at; sh_next[(count + 1) % 3] = kTreeMax; }
        ++count;
        __syncthreads();
        if (count == a.max_path) break;
        if (walk && i < v.n && i > 0 && parent == at && draft == a.sampled[v.t0 + at]) atomicMin(next, i);
        __syncthreads();
        const int n = *next;
        if (n == kTreeMax) break;
        at = n;
    }
    for (int k = count + i; k < a.max_path; k += kTreeMax) path[k] = -1;
    if (i == 0) {
        const int accepted = walk ? count : tree ? 0 : v.n;
        const int last = walk ? at : accepted - 1;
        a.num_accepted[s] = accepted;
        a.next_token[s] = accepted > 0 ? a.sampled[v.t0 + last] : -1;
        if (a.new_past_lens) a.new_past_lens[s] = a.past_lens[s] + accepted;
    }
}

// The accepted rows of one sequence, a block for the keys or the values of a layer at a time.  A row moves from past + path[k] to past + k, never
// up: a later row's place is not overwritten by an earlier one's move, so a thread that owns the same bytes of every row and goes along the path reads each of
// them in time.  Token-minor u8 values are single bytes out of 32-byte sectors: what bounds the move of a batch of trees (64 trees, 32 layers: 26 MB of
// rows in some 300 MB of sectors, 0.05 ms of HBM).  kMoveBatch rows' loads are under way before the first store; more of them, or several pieces a thread,
// cost registers and so blocks beside one another (54 | 75 us).
constexpr int kMoveBatch = 4;
constexpr int kMoveThreads = 256;

// Unit u of `units` of every row: unit(u) is where a row's unit lies in slot 0 of block 0, slot(x) the offset of slot x.
template <class T, class Unit, class Slot>
__device__ __forceinline__ void move_rows(uint8_t* cache, int units, int count, const int* src, const int* dst, int bs, long long block_bytes, Unit&& unit, Slot&& slot) {
    for (int u = threadIdx.x; u < units; u += kMoveThreads) {
        uint8_t* const base = cache + unit(u);
        for (int k0 = 0; k0 < count; k0 += kMoveBatch) {
            T w[kMoveBatch];
#pragma unroll
            for (int k = 0; k < kMoveBatch; ++k)
                if (k0 + k < count) w[k] = *reinterpret_cast<const T*>(base + (long long)(src[k0 + k] / bs) * block_bytes + slot(src[k0 + k] % bs));
#pragma unroll
            for (int k = 0; k < kMoveBatch; ++k)
                if (k0 + k < count) *reinterpret_cast<T*>(base + (long long)(dst[k0 + k] / bs) * block_bytes + slot(dst[k0 + k] % bs)) = w[k];
        }
    }
}

template <int D, int BS>
__global__ void __launch_bounds__(kMoveThreads) tree_move_kernel(const __grid_constant__ TreeMoveArgs m) {
    const TreeAcceptArgs& a = m.t;
    __shared__ int sh_src[kTreeMax], sh_dst[kTreeMax];   // slots (block * BS + slot) of the rows that move
    __shared__ int sh_moves[kTreeMax / 32];
    grid_wait();
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kMoveWarps = kMoveThreads / 32;
    static_assert(kMoveThreads == kTreeMax, "a thread per place of a path");
    const int tb = a.block_indices_begins[s], pages = a.block_indices_begins[s + 1] - tb, count = a.num_accepted[s];
    const int from = tid < a.max_path ? a.path[(long long)s * a.max_path + tid] : -1;   // (-1 everywhere without a tree, and where the metadata are bad)
    const int past = a.past_lens[s] - (a.new_past_lens == a.past_lens ? count : 0);     // (the walk has written the new ones)
    int src = -1, dst = -1;
    if (from >= 0 && from != tid) {
        const int p0 = past + from, p1 = past + tid;
        const bool inside = past >= 0 && from < kTreeMax && p0 / BS < pages && p1 / BS < pages;   // (as the walk has checked, if its outputs are still its own)
        const int b0 = inside ? a.block_indices[tb + p0 / BS] : -1, b1 = inside ? a.block_indices[tb + p1 / BS] : -1;
        if (b0 < 0 || b0 >= a.num_blocks || b1 < 0 || b1 >= a.num_blocks) {
            if (blockIdx.y == 0) atomicOr(a.status, PA_DEV_BAD_BLOCK_INDEX);
        } else {
            src = b0 * BS + p0 % BS;
            dst = b1 * BS + p1 % BS;
        }
    }
    // the list of moves, in the order of the path
    const uint32_t mine = __ballot_sync(0xffffffffu, src >= 0);
    if (lane == 0) sh_moves[warp] = __popc(mine);
    __syncthreads();
    int at = __popc(mine & ((1u << lane) - 1u)), moves = 0;
    for (int w = 0; w < kMoveWarps; ++w) {
        if (w < warp) at += sh_moves[w];
        moves += sh_moves[w];
    }
    if (src >= 0) { sh_src[at] = src; sh_dst[at] = dst; }
    if (moves == 0) return;
    __syncthreads();
    const bool u8 = a.g.cache == PA_DTYPE_U8;
    const int heads = a.g.Hkv;
    const long long hb = a.g.head_bytes, bb = a.g.block_bytes;
    uint8_t* const cache = m.cache[blockIdx.y & 1][blockIdx.y >> 1];
    const bool value = (blockIdx.y & 1) != 0;
    if (!u8) {
        constexpr int CH = D / 8;   // 16-byte pieces of a row
        move_rows<uint4>(cache, heads * CH, moves, sh_src, sh_dst, BS, bb, [&](int u) { return (u / CH) * hb + 16 * (u % CH); }, [](int x) { return x * D * 2; });
        return;
    }
    if (!value) {
        constexpr int CH = D / 16;
        move_rows<uint4>(cache, heads * CH, moves, sh_src, sh_dst, BS, bb, [&](int u) { return (u / CH) * hb + 16 * (u % CH); }, [](int x) { return x * D; });
    } else {
        move_rows<uint8_t>(cache, heads * D, moves, sh_src, sh_dst, BS, bb, [&](int u) { return (u / D) * hb + (u % D) * BS; }, [](int x) { return x; });
    }
    // scales and zero-points
    move_rows<uint32_t>(cache, heads * 2, moves, sh_src, sh_dst, BS, bb, [&](int u) { return (u >> 1) * hb + BS * D + (u & 1) * BS * 4; }, [](int x) { return 4 * x; });
}

}  // namespace

cudaError_t launch_tree_accept(const TreeAcceptArgs& a, void* const* key_caches, void* const* value_caches, int num_layers, cudaStream_t stream, int* launches) {
    if (a.num_sequences <= 0) return cudaSuccess;
    cudaError_t e = launch_dependent(tree_walk_kernel, dim3(a.num_sequences), dim3(kTreeMax), 0, stream, a);
    if (e != cudaSuccess) return e;
    ++*launches;
    for (int l0 = 0; l0 < num_layers; l0 += kMoveLayers) {
        TreeMoveArgs m{};
        m.t = a;
        m.num_layers = num_layers - l0 < kMoveLayers ? num_layers - l0 : kMoveLayers;
        for (int i = 0; i < m.num_layers; ++i) {
            m.cache[0][i] = (uint8_t*)key_caches[l0 + i];
            m.cache[1][i] = (uint8_t*)value_caches[l0 + i];
        }
        const dim3 grid(a.num_sequences, 2 * m.num_layers);   // a block per layer's keys or values
        auto launch = [&](auto kernel) { return launch_dependent(kernel, grid, dim3(kMoveThreads), 0, stream, m); };
        if (a.g.D == 128) e = a.g.bs == 32 ? launch(tree_move_kernel<128, 32>) : launch(tree_move_kernel<128, 16>);
        else e = a.g.bs == 32 ? launch(tree_move_kernel<64, 32>) : launch(tree_move_kernel<64, 16>);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    return cudaSuccess;
}

}  // namespace pa
