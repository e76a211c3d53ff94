// What the kernels of a masked step (include/masked_b200.h) share: which context positions a query row sees, as tiles of
// the context and as words of bits.
//
// A row sees the "causal part" j < ctx of its context, of that  j < sinks  or  j >= lo,  and, with a tree, bits of its chunk:
//   no tree:  ctx = past + index + 1,  lo = max(0, ctx - W)
//   a tree:   ctx = past,              lo = max(0, past + depth + 1 - W),  bits = its ancestors and itself (those the window leaves)
#pragma once

#include "../../include/masked_b200.h"
#include "pa_kernels.h"

namespace pa {

// The tiles of T tokens that rows with lo and a context of ctx tokens touch: [0, split) and [split + gap, split + gap + rest), listed one behind
// the other.
struct VisTiles {
    int split, gap, count;
    __host__ __device__ __forceinline__ int tile(int i) const { return i < split ? i : i + gap; }
};
template <int T>
__host__ __device__ __forceinline__ VisTiles vis_tiles(int ctx, int lo, int sinks) {
    const int total = (ctx + T - 1) / T, ts = ((sinks < ctx ? sinks : ctx) + T - 1) / T, tw = lo / T;
    const int gap = tw > ts ? tw - ts : 0;
    return VisTiles{ts, gap, total - gap};
}

__host__ __device__ __forceinline__ int window_lo(const MaskParams& m, int ctx) { return m.window > 0 && ctx > m.window ? ctx - m.window : 0; }

// n lowest bits
__host__ __device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }
__host__ __device__ __forceinline__ uint32_t low_bits32(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// Bit c: position pos0 + c belongs to the causal part of a row.
__host__ __device__ __forceinline__ uint64_t causal_bits(int pos0, int ctx, int lo, int sinks) {
    return low_bits(ctx - pos0) & ~(low_bits(lo - pos0) & ~low_bits(sinks - pos0));
}
__host__ __device__ __forceinline__ uint32_t causal_bits32(int pos0, int ctx, int lo, int sinks) {
    return low_bits32(ctx - pos0) & ~(low_bits32(lo - pos0) & ~low_bits32(sinks - pos0));
}

// Bit c: token o + c of the chunk is among `words` (a row's ancestors and itself); o may be negative.
__host__ __device__ __forceinline__ uint32_t tree_bits32(const uint32_t* words, int o) {
    if (o <= -32 || o >= kTreeMax) return 0u;
    if (o < 0) return words[0] << -o;
    const int w = o >> 5;
    const uint32_t lo = words[w], hi = w + 1 < kTreeWords ? words[w + 1] : 0u;
    return (uint32_t)(((uint64_t)hi << 32 | lo) >> (o & 31));
}
__host__ __device__ __forceinline__ uint64_t tree_bits64(const uint32_t* words, int o) {
    return (uint64_t)tree_bits32(words, o) | (uint64_t)tree_bits32(words, o + 32) << 32;
}

// What one row sees.
struct RowMask {
    int ctx, lo;
    const uint32_t* words;   // null: no tree
    int past;
};
__device__ __forceinline__ RowMask row_mask(const KernelArgs& a, int t0, int past, int tok, bool tree) {
    if (!tree) return RowMask{past + tok + 1, window_lo(a.m, past + tok + 1), nullptr, past};
    const int t = t0 + tok;
    return RowMask{past, window_lo(a.m, past + __ldcg(a.m.tree_depth + t) + 1), a.m.tree_words + (long long)t * kTreeWords, past};
}
__host__ __device__ __forceinline__ uint32_t row_bits32(const MaskParams& m, const RowMask& r, int pos0) {
    uint32_t w = causal_bits32(pos0, r.ctx, r.lo, m.sinks);
    if (r.words && pos0 + 32 > r.past) w |= tree_bits32(r.words, pos0 - r.past);
    return w;
}
// The same of a row of a chunk of n tokens, none behind it: the words of a token that two sequences claim may be the other one's, and positions behind the
// chunk have no pages.
__host__ __device__ __forceinline__ uint32_t row_bits32(const MaskParams& m, const RowMask& r, int n, int pos0) {
    return row_bits32(m, r, pos0) & low_bits32(r.past + n - pos0);
}
// The tiles that one row of a chunk of n tokens goes through.  A tree's whole chunk is among them, however far the row's window has come: its tokens are seen by
// their positions, and an ancestor whose position is below the sinks may lie anywhere in the chunk.
template <int T>
__host__ __device__ __forceinline__ VisTiles row_tiles(const MaskParams& m, const RowMask& r, int n) {
    return r.words ? vis_tiles<T>(r.past + n, r.lo < r.past ? r.lo : r.past, m.sinks) : vis_tiles<T>(r.ctx, r.lo, m.sinks);
}

__device__ __forceinline__ bool has_tree(const KernelArgs& a, int t0, int n) { return a.m.parents && n > 0 && a.m.parents[t0] != kTreeNone; }

// The tiles of 64 tokens that the 256 rows of a q tile touch: rows row0 .. of a sequence, (token, head) pairs in order.
struct QTile {
    VisTiles v;
    int lo;           // smallest lo of the rows
    int cnt[2];       // tiles of the list that each half of 128 rows reaches (a prefix; 0: the half has no rows)
    int ctx_hi[2];    // context that the last row of each half sees
};
__host__ __device__ __forceinline__ QTile q_tile(const MaskParams& m, int past, int n, int G, int row0, bool tree) {
    QTile q;
    q.lo = window_lo(m, tree ? past + 1 : past + row0 / G + 1);
    int top = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int r0 = row0 + 128 * x;
        q.ctx_hi[x] = r0 >= n * G ? 0 : tree || (r0 + 127) / G >= n ? past + n : past + (r0 + 127) / G + 1;
        top = q.ctx_hi[x] > top ? q.ctx_hi[x] : top;
    }
    q.v = vis_tiles<64>(top, q.lo, m.sinks);
#pragma unroll
    for (int x = 0; x < 2; ++x) q.cnt[x] = q.ctx_hi[x] > 0 ? vis_tiles<64>(q.ctx_hi[x], q.lo, m.sinks).count : 0;
    return q;
}

// One query row on CUDA cores, by one warp: lane l owns dims {l + 32 i}, online softmax over the positions that the row sees, read back from the paged
// cache; what it does not see is not read.  Any cache type, head size and mask: for rows that no other kernel serves, and for those
// whose tile held something that is not finite and that they do not see (0 times it is not 0 in a product).
template <int D>
static __device__ __noinline__ void masked_row(const KernelArgs& a, int t, int hq) {
    constexpr int PER = D / 32;
    const int lane = threadIdx.x & 31, hk = hq / (a.g.Hq / a.g.Hkv), bs = a.g.bs;
    int lo = 0, hi = a.num_sequences;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.subsequence_begins[mid] <= t) lo = mid; else hi = mid;
    }
    SeqView sv;
    if (!seq_view(a, lo, sv) || sv.n <= 1 || t < sv.t0 || t >= sv.t0 + sv.n) return;
    const bool tree = has_tree(a, sv.t0, sv.n);
    if (tree && sv.n > kTreeMax) { atomicOr(a.status, PA_DEV_BAD_TREE); return; }
    const RowMask rm = row_mask(a, sv.t0, sv.past, t - sv.t0, tree);
    const float scale = (a.scale != 0.f ? a.scale : rsqrtf((float)D)) * 1.4426950408889634f;
    float q[PER], acc[PER];
    const long long row = (long long)t * a.g.Hq + hq;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        q[i] = load_act(a.query, row * D + lane + 32 * i, a.g.act) * scale;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const VisTiles v = row_tiles<32>(a.m, rm, sv.n);
    for (int i = 0; i < v.count; ++i) {
        const int pos0 = 32 * v.tile(i);
        for (uint32_t w = row_bits32(a.m, rm, sv.n, pos0); w; w &= w - 1) {
            const int pos = pos0 + __ffs(w) - 1;
            const int blk = a.block_indices[sv.tb + pos / bs];
            if (blk < 0 || blk >= a.num_blocks) {
                atomicOr(a.status, PA_DEV_BAD_BLOCK_INDEX);
                continue;
            }
            const long long rec = (long long)blk * a.g.block_bytes + (long long)hk * a.g.head_bytes;
            const int slot = pos % bs;
            const uint8_t* kr = (const uint8_t*)a.key_cache + rec;
            const uint8_t* vr = (const uint8_t*)a.value_cache + rec;
            float s = 0.f, val[PER];
            if (a.g.cache == PA_DTYPE_U8) {
                const float* kp = (const float*)(kr + (long long)bs * D);
                const float* vp = (const float*)(vr + (long long)bs * D);
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const int d = lane + 32 * e;
                    s += q[e] * dequant_one(kr[(long long)slot * D + d], kp[slot], kp[bs + slot]);
                    val[e] = dequant_one(vr[(long long)d * bs + slot], vp[slot], vp[bs + slot]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const long long at = (long long)slot * D + lane + 32 * e;
                    s += q[e] * load_act(kr, at, a.g.cache);
                    val[e] = load_act(vr, at, a.g.cache);
                }
            }
            s = warp_sum(s);
            const float m_new = fmaxf(m, s);
            const float f = m_new == -INFINITY ? 1.f : exp2f(m - m_new), p = s == -INFINITY ? 0.f : exp2f(s - m_new);   // (an s that is not a number stays one)
            l = l * f + p;
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = acc[e] * f + p * val[e];
            m = m_new;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) store_act(a.output, row * D + lane + 32 * i, a.g.act, acc[i] / l);
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

}  // namespace pa
