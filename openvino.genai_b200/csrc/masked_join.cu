// Joins the pieces of q tiles that a masked step cut along their context (build_mask_items): a row's result is
// sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over its pieces, M the largest m_i.  A warp per row, a lane per D / 32 neighbouring elements, in the order of
// the pieces, so that the result does not depend on who ended first.  Bound by the chain plan -> records -> maxima -> results, with up to eight
// pieces' loads in flight.  Rows whose result is not finite are computed again by themselves (masked_row): what they do not see may have been the cause.
#include "masked.cuh"
#include "pa_common.cuh"
#include "pa_kernels.h"

namespace pa {

namespace {

constexpr int kJoinWarps = 8;
constexpr int kJoinBatch = 8;

template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) masked_join_kernel(const __grid_constant__ KernelArgs a) {
    constexpr int PER = D / 32;
    grid_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.g.Hq / a.g.Hkv, Hkv = a.g.Hkv;
    constexpr int kChunks = kPrefillItemRows / kJoinWarps;
    const long long units = (long long)a.plan->total_splits * Hkv * kChunks;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const MaskSplit& sp = a.m.splits[u / (Hkv * kChunks)];
        const int hk = (int)(u / kChunks % Hkv), r = (int)(u % kChunks) * kJoinWarps + warp;
        const int pair = sp.row0 + r;
        if (pair >= sp.n_new * G) continue;
        const QTile q = q_tile(a.m, sp.past, sp.n_new, G, sp.row0, sp.tree);
        const int pieces = min(sp.pieces, (q.cnt[r >> 7] + sp.len - 1) / sp.len);   // those that the row's half has tiles in
        const long long row0 = ((long long)sp.first_part + hk) * kPrefillItemRows + r, step = (long long)Hkv * kPrefillItemRows;
        float m = -INFINITY;
        for (int i = lane; i < pieces; i += 32) m = fmaxf(m, __ldcg(a.m.part_ml + row0 + i * step).x);
        m = warp_max(m);
        float l = 0.f, o[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = 0.f;
        for (int i0 = 0; i0 < pieces; i0 += kJoinBatch) {
            float2 ml[kJoinBatch];
            float v[kJoinBatch][PER];
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) {
                const long long at = row0 + min(i0 + k, pieces - 1) * step;
                ml[k] = __ldcg(a.m.part_ml + at);
                if constexpr (PER == 4) {
                    const float4 w = __ldcg(reinterpret_cast<const float4*>(a.m.part_o + at * D + lane * PER));
                    v[k][0] = w.x; v[k][1] = w.y; v[k][2] = w.z; v[k][3] = w.w;
                } else {
                    const float2 w = __ldcg(reinterpret_cast<const float2*>(a.m.part_o + at * D + lane * PER));
                    v[k][0] = w.x; v[k][1] = w.y;
                }
            }
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) {
                // a piece of which the row sees nothing has no maximum and no weight
                const float f = i0 + k < pieces && ml[k].x > -INFINITY ? exp2f(ml[k].x - m) : 0.f;
                l += f * ml[k].y;
#pragma unroll
                for (int e = 0; e < PER; ++e) o[e] += f != 0.f ? f * v[k][e] : 0.f;
            }
        }
        const long long out = (((long long)sp.t0 + pair / G) * a.g.Hq + hk * G + pair % G) * D + lane * PER;
        const float inv = 1.f / l;
        bool finite = true;
#pragma unroll
        for (int e = 0; e < PER; ++e) finite = finite && !not_finite(o[e] * inv);
        if (!__all_sync(0xffffffffu, finite)) {
            masked_row<D>(a, sp.t0 + pair / G, hk * G + pair % G);
            continue;
        }
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
            if (a.g.act == PA_DTYPE_F32) *reinterpret_cast<float2*>((float*)a.output + out + e) = make_float2(o[e] * inv, o[e + 1] * inv);
            else *reinterpret_cast<uint32_t*>((uint16_t*)a.output + out + e) = a.g.act == PA_DTYPE_F16 ? pack_h2(o[e] * inv, o[e + 1] * inv) : pack_bf2(o[e] * inv, o[e + 1] * inv);
        }
    }
    // rows of whole q tiles that are not finite: once more, by themselves
    const int redo = min(a.plan->total_redo, a.num_tokens * a.g.Hq);
    for (int i = blockIdx.x * kJoinWarps + warp; i < redo; i += gridDim.x * kJoinWarps) {
        const int row = a.m.redo[i];
        masked_row<D>(a, row / a.g.Hq, row % a.g.Hq);
    }
}

}  // namespace

cudaError_t launch_masked_join(const KernelArgs& a, cudaStream_t stream, int* launches) {
    const dim3 grid(2 * a.m.sm_count), block(kJoinWarps * 32);
    const cudaError_t e = a.g.D == 128 ? launch_dependent(masked_join_kernel<128>, grid, block, 0, stream, a) : launch_dependent(masked_join_kernel<64>, grid, block, 0, stream, a);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace pa
