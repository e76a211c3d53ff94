// Joins the pieces of lists that a masked step cut between CTAs (build_mask_items): a row's result is
// sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over its pieces, M the largest m_i.  A warp per row, a lane per D / 32 neighbouring elements, in the order of
// the pieces, so that the result does not depend on who ended first.  Bound by the chain plan -> record -> pieces and by the kernel's own code, which every SM
// has to fetch: this short loop over rows, dealt out one by one over all warps, takes 8 us for 864 rows of nine pieces, 15 us for 37,000 of two, where blocks of
// 32 rows with their loads unrolled took 20 and 17.  Rows whose result is not finite are computed again by themselves (masked_row): what they do not
// see may have been the cause.
#include "masked.cuh"
#include "pa_common.cuh"
#include "pa_kernels.h"

namespace pa {

namespace {

constexpr int kJoinWarps = 8;
constexpr int kJoinBatch = 4;   // pieces under way

template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32, 4) masked_join_kernel(const __grid_constant__ KernelArgs a) {
    constexpr int PER = D / 32;
    grid_wait();
    const int lane = threadIdx.x & 31, G = a.g.Hq / a.g.Hkv;
    const int warp = blockIdx.x * kJoinWarps + (threadIdx.x >> 5), warps = gridDim.x * kJoinWarps;
    const int units = __ldcg(&a.plan->total_cuts) * kPrefillItemRows, redo = min(__ldcg(&a.plan->total_redo), a.num_tokens * a.g.Hq);
    int again = -1;   // a row of this warp's to compute again
    for (int u = warp; u < units; u += warps) {
        const MaskCut c = a.m.cuts[u / kPrefillItemRows];
        const int r = u % kPrefillItemRows;
        if (r >= c.rows) continue;
        const int pieces = c.pieces[r >> 7], row = (c.t0 + (c.row0 + r) / G) * a.g.Hq + c.hk * G + (c.row0 + r) % G;
        float m = -INFINITY, l = 0.f, o[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = 0.f;
#pragma unroll 1
        for (int i0 = 0; i0 < pieces; i0 += kJoinBatch) {
            float2 ml[kJoinBatch];
            float v[kJoinBatch][PER];
#pragma unroll
            for (int i = 0; i < kJoinBatch; ++i) {
                const int piece = min(i0 + i, pieces - 1);
                const long long at = (long long)(2 * (c.w + piece) + (piece == 0 ? 1 : 0)) * kPrefillItemRows + r;   // CTA w's last list, the others' first
                ml[i] = __ldcg(a.m.part_ml + at);
                const float* const src = a.m.part_o + at * D + lane * PER;
                if constexpr (PER == 4) {
                    const float4 w = __ldcg(reinterpret_cast<const float4*>(src));
                    v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
                } else {
                    const float2 w = __ldcg(reinterpret_cast<const float2*>(src));
                    v[i][0] = w.x; v[i][1] = w.y;
                }
                if (i0 + i >= pieces) ml[i] = make_float2(-INFINITY, 0.f);
            }
            float top = m;
#pragma unroll
            for (int i = 0; i < kJoinBatch; ++i) top = fmaxf(top, ml[i].x);
            const float keep = m > -INFINITY ? exp2f(m - top) : 0.f;
            m = top;
            l *= keep;
#pragma unroll
            for (int e = 0; e < PER; ++e) o[e] *= keep;
#pragma unroll
            for (int i = 0; i < kJoinBatch; ++i) {
                if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;   // a piece of which the row sees nothing (a sum that is not a number: it saw only such)
                const float f = exp2f(ml[i].x - top);
                l += f * ml[i].y;
#pragma unroll
                for (int e = 0; e < PER; ++e) o[e] += f * v[i][e];
            }
        }
        const float inv = 1.f / l;
        bool finite = true;
#pragma unroll
        for (int e = 0; e < PER; ++e) finite = finite && !not_finite(o[e] * inv);
        if (!__all_sync(0xffffffffu, finite)) {
            if (again >= 0) masked_row<D>(a, again / a.g.Hq, again % a.g.Hq);
            again = row;
            continue;
        }
        const long long out = (long long)row * D + lane * PER;
#pragma unroll
        for (int e = 0; e < PER; e += 2) {
            if (a.g.act == PA_DTYPE_F32) *reinterpret_cast<float2*>((float*)a.output + out + e) = make_float2(o[e] * inv, o[e + 1] * inv);
            else *reinterpret_cast<uint32_t*>((uint16_t*)a.output + out + e) = a.g.act == PA_DTYPE_F16 ? pack_h2(o[e] * inv, o[e + 1] * inv) : pack_bf2(o[e] * inv, o[e + 1] * inv);
        }
    }
    // and rows of whole lists that are not finite
    for (int i = warp; i < redo || again >= 0; i += warps) {
        const int row = again >= 0 ? again : a.m.redo[i];
        if (again >= 0) { again = -1; i -= warps; }
        masked_row<D>(a, row / a.g.Hq, row % a.g.Hq);
    }
}

}  // namespace

cudaError_t launch_masked_join(const KernelArgs& a, cudaStream_t stream, int* launches) {
    const dim3 grid(4 * a.m.sm_count), block(kJoinWarps * 32);
    const cudaError_t e = a.g.D == 128 ? launch_dependent(masked_join_kernel<128>, grid, block, 0, stream, a) : launch_dependent(masked_join_kernel<64>, grid, block, 0, stream, a);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace pa
