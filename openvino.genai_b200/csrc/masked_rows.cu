// Masked attention, rows one by one on CUDA cores: one warp per (new token, q head), lane l owns dims {l + 32 i}, online softmax over the
// positions that the row sees (masked.cuh), read back from the paged cache.  Any cache type, head size and mask; what a row does not see is not read.
#include "masked.cuh"
#include "pa_common.cuh"
#include "pa_kernels.h"

namespace pa {

namespace {

template <int D>
__global__ void __launch_bounds__(256) masked_rows_kernel(KernelArgs a) {
    constexpr int PER = D / 32;
    grid_wait();
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (warp >= (long long)a.num_tokens * a.g.Hq) return;
    const int t = (int)(warp / a.g.Hq), hq = (int)(warp % a.g.Hq), hk = hq / (a.g.Hq / a.g.Hkv), bs = a.g.bs;
    int lo = 0, hi = a.num_sequences;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.subsequence_begins[mid] <= t) lo = mid; else hi = mid;
    }
    SeqView sv;
    if (!seq_view(a, lo, sv) || t < sv.t0 || t >= sv.t0 + sv.n) return;
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
    const VisTiles v = vis_tiles<32>(tree ? sv.past + sv.n : rm.ctx, rm.lo, a.m.sinks);
    for (int i = 0; i < v.count; ++i) {
        const int pos0 = 32 * v.tile(i);
        for (uint32_t w = row_bits32(a, rm, pos0); w; w &= w - 1) {
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
            const float f = m_new == -INFINITY ? 1.f : exp2f(m - m_new), p = m_new == -INFINITY ? 0.f : exp2f(s - m_new);
            l = l * f + p;
#pragma unroll
            for (int e = 0; e < PER; ++e) acc[e] = acc[e] * f + p * val[e];
            m = m_new;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) store_act(a.output, row * D + lane + 32 * i, a.g.act, acc[i] / l);
}

}  // namespace

cudaError_t launch_masked_rows(const KernelArgs& a, cudaStream_t stream, int* launches) {
    if (a.num_tokens <= 0) return cudaSuccess;
    const long long blocks = ((long long)a.num_tokens * a.g.Hq + 7) / 8;
    const cudaError_t e = a.g.D == 128 ? launch_dependent(masked_rows_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, stream, a)
                                       : launch_dependent(masked_rows_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace pa
