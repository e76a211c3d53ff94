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
    const bool walk = tree && v.n <= kTreeMax;
    if (tree && !walk && i == 0) atomicOr(a.status, PA_DEV_BAD_TREE);
    int parent = -1;
    int64_t draft = 0;
    if (walk && i < v.n) {
        parent = a.parents[v.t0 + i];
        draft = a.draft[v.t0 + i];
        if (parent < -1 || parent >= i) { atomicOr(a.status, PA_DEV_BAD_TREE); parent = -1; }
    }
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
    }
}

// Rows of one (sequence, layer, keys or values) per block.  A row moves from past + path[k] to past + k <= past + path[k]: nothing that a later move
// reads is written by an earlier one, but a row may be both read and written, so all rows of a head are read before the first is written.
template <int D>
__global__ void __launch_bounds__(256) tree_move_kernel(const __grid_constant__ TreeMoveArgs m) {
    const TreeAcceptArgs& a = m.t;
    __shared__ int sh_src[kTreeMax], sh_dst[kTreeMax];   // slots (block * bs + slot), -1: stays
    grid_wait();
    const int s = blockIdx.x, layer = blockIdx.y >> 1, value = blockIdx.y & 1, tid = threadIdx.x;
    SeqView v;
    accept_view(a, s, v, false);
    const bool walk = v.n > 0 && v.n <= kTreeMax && a.parents[v.t0] != kTreeNone;
    const int count = walk ? min(a.num_accepted[s], a.max_path) : 0;
    bool moves = false;
    if (tid < count) {
        const int from = a.path[(long long)s * a.max_path + tid];
        int src = -1, dst = -1;
        if (from != tid) {
            const int p0 = v.past + from, p1 = v.past + tid;
            const int b0 = a.block_indices[v.tb + p0 / a.g.bs], b1 = a.block_indices[v.tb + p1 / a.g.bs];
            if (b0 < 0 || b0 >= a.num_blocks || b1 < 0 || b1 >= a.num_blocks) atomicOr(a.status, PA_DEV_BAD_BLOCK_INDEX);
            else { src = b0 * a.g.bs + p0 % a.g.bs; dst = b1 * a.g.bs + p1 % a.g.bs; moves = true; }
        }
        sh_src[tid] = src;
        sh_dst[tid] = dst;
    }
    if (!__syncthreads_or(moves)) return;
    uint8_t* const cache = m.cache[value][layer];
    const int bs = a.g.bs;
    // a thread's own elements of every row: no two threads touch the same bytes, so a thread that goes along the path in order reads
    // each of them before it is overwritten
    if (a.g.cache != PA_DTYPE_U8) {
        constexpr int CH = D / 8;   // 16-byte chunks of a row
        for (int u = tid; u < a.g.Hkv * CH; u += 256) {
            uint8_t* const head = cache + (long long)(u / CH) * a.g.head_bytes + 16 * (u % CH);
            for (int k = 0; k < count; ++k) {
                if (sh_src[k] < 0) continue;
                const uint4 w = *reinterpret_cast<const uint4*>(head + (long long)(sh_src[k] / bs) * a.g.block_bytes + (long long)(sh_src[k] % bs) * D * 2);
                *reinterpret_cast<uint4*>(head + (long long)(sh_dst[k] / bs) * a.g.block_bytes + (long long)(sh_dst[k] % bs) * D * 2) = w;
            }
        }
        return;
    }
    if (!value) {
        constexpr int CH = D / 16;
        for (int u = tid; u < a.g.Hkv * CH; u += 256) {
            uint8_t* const head = cache + (long long)(u / CH) * a.g.head_bytes + 16 * (u % CH);
            for (int k = 0; k < count; ++k) {
                if (sh_src[k] < 0) continue;
                const uint4 w = *reinterpret_cast<const uint4*>(head + (long long)(sh_src[k] / bs) * a.g.block_bytes + (long long)(sh_src[k] % bs) * D);
                *reinterpret_cast<uint4*>(head + (long long)(sh_dst[k] / bs) * a.g.block_bytes + (long long)(sh_dst[k] % bs) * D) = w;
            }
        }
    } else {   // value bytes are token-minor: [D][bs]
        for (int u = tid; u < a.g.Hkv * D; u += 256) {
            uint8_t* const head = cache + (long long)(u / D) * a.g.head_bytes + (long long)(u % D) * bs;
            for (int k = 0; k < count; ++k) {
                if (sh_src[k] < 0) continue;
                const uint8_t b = head[(long long)(sh_src[k] / bs) * a.g.block_bytes + sh_src[k] % bs];
                head[(long long)(sh_dst[k] / bs) * a.g.block_bytes + sh_dst[k] % bs] = b;
            }
        }
    }
    for (int u = tid; u < a.g.Hkv * 2; u += 256) {   // scales and zero-points
        uint8_t* const head = cache + (long long)(u >> 1) * a.g.head_bytes + (long long)bs * D + (long long)(u & 1) * bs * 4;
        for (int k = 0; k < count; ++k) {
            if (sh_src[k] < 0) continue;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(head + (long long)(sh_src[k] / bs) * a.g.block_bytes + 4 * (sh_src[k] % bs));
            *reinterpret_cast<uint32_t*>(head + (long long)(sh_dst[k] / bs) * a.g.block_bytes + 4 * (sh_dst[k] % bs)) = w;
        }
    }
}

// new_past_lens comes last: it may be past_lens, which the moves read.
__global__ void __launch_bounds__(256) tree_past_kernel(TreeAcceptArgs a) {
    grid_wait();
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s < a.num_sequences) a.new_past_lens[s] = a.past_lens[s] + a.num_accepted[s];
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
        const dim3 grid(a.num_sequences, 2 * m.num_layers);
        e = a.g.D == 128 ? launch_dependent(tree_move_kernel<128>, grid, dim3(256), 0, stream, m) : launch_dependent(tree_move_kernel<64>, grid, dim3(256), 0, stream, m);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    if (a.new_past_lens) {
        e = launch_dependent(tree_past_kernel, dim3((a.num_sequences + 255) / 256), dim3(256), 0, stream, a);
        if (e != cudaSuccess) return e;
        ++*launches;
    }
    return cudaSuccess;
}

}  // namespace pa
