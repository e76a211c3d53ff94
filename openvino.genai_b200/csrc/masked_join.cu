// Joins the pieces of lists that a masked step cut between CTAs (build_mask_items): a row's result is
// sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over its pieces, M the largest m_i.  A lane has D / 32 neighbouring elements of a row, pieces are taken in
// order, so that the result does not depend on who ended first.  Bound by the chain starts -> q tile -> pieces, so a block looks its list up once for 32
// rows, and eight or sixteen loads of a warp are under way: two pieces of four rows, or eight of two.  Rows whose result is not finite are computed again by themselves (masked_row): what they do not see may have been the cause.
#include <type_traits>

#include "masked.cuh"
#include "pa_common.cuh"
#include "pa_kernels.h"

namespace pa {

namespace {

constexpr int kJoinWarps = 8;
constexpr int kJoinRows = 32;   // rows of a block
constexpr int kJoinParts = kPrefillItemRows / kJoinRows;

// Joins R rows of a warp, P pieces' loads of each under way at a time.  row_of(i, k): where piece i of row k lies; pieces[k]: its pieces, 0: no row.
template <int D, int R, int P, class RowOf, class Done>
__device__ __forceinline__ void join_rows(const KernelArgs& a, const int (&pieces)[R], RowOf&& row_of, Done&& done) {
    constexpr int PER = D / 32;
    const int lane = threadIdx.x & 31;
    float m[R], l[R], o[R][PER];
    int most = 0;
#pragma unroll
    for (int k = 0; k < R; ++k) {
        m[k] = -INFINITY; l[k] = 0.f;
        most = max(most, pieces[k]);
#pragma unroll
        for (int e = 0; e < PER; ++e) o[k][e] = 0.f;
    }
    for (int i0 = 0; i0 < most; i0 += P) {
        float2 ml[R][P];
        float v[R][P][PER];
#pragma unroll
        for (int k = 0; k < R; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                ml[k][i] = make_float2(-INFINITY, 0.f);
                if (i0 + i >= pieces[k]) continue;
                const long long row = row_of(i0 + i, k);
                ml[k][i] = __ldcg(a.m.part_ml + row);
                if constexpr (PER == 4) {
                    const float4 w = __ldcg(reinterpret_cast<const float4*>(a.m.part_o + row * D + lane * PER));
                    v[k][i][0] = w.x; v[k][i][1] = w.y; v[k][i][2] = w.z; v[k][i][3] = w.w;
                } else {
                    const float2 w = __ldcg(reinterpret_cast<const float2*>(a.m.part_o + row * D + lane * PER));
                    v[k][i][0] = w.x; v[k][i][1] = w.y;
                }
            }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            float top = m[k];
#pragma unroll
            for (int i = 0; i < P; ++i) top = fmaxf(top, ml[k][i].x);
            // a piece of which the row sees nothing has no maximum and no weight
            const float f0 = m[k] > -INFINITY ? exp2f(m[k] - top) : 0.f;
            m[k] = top;
            l[k] *= f0;
#pragma unroll
            for (int e = 0; e < PER; ++e) o[k][e] *= f0;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float f = ml[k][i].x > -INFINITY ? exp2f(ml[k][i].x - top) : 0.f;
                if (f != 0.f) {   // (not-a-number is different from zero)
                    l[k] += f * ml[k][i].y;
#pragma unroll
                    for (int e = 0; e < PER; ++e) o[k][e] += f * v[k][i][e];
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < R; ++k)
        if (pieces[k] > 0) done(k, l[k], o[k]);
}

template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) masked_join_kernel(const __grid_constant__ KernelArgs a) {
    constexpr int PER = D / 32;
    grid_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.g.Hq / a.g.Hkv, ctas = a.m.sm_count;
    // a block per 32 rows of the list that CTA w is the first to take over in its middle
    const int w = blockIdx.x / kJoinParts + 1, r0 = blockIdx.x % kJoinParts * kJoinRows;
    const MaskStart at = a.m.starts[min(w, ctas)], before = a.m.starts[min(w, ctas) - 1];
    if (w < ctas && at.j > 0 && !(before.q == at.q && before.hk == at.hk && before.j > 0)) {
        const MaskItem it = a.m.items[at.q];
        const int hk = at.hk, rows = it.n_new * G - it.row0;
        if (r0 < rows) {
            // its pieces: CTA w - 1's last list, then the first ones of those from w on that begin in it; a half's rows have those that begin in its tiles
            const QTile q = q_tile(a.m, it.past, it.n_new, G, it.row0, it.tree);
            const int reach = q.cnt[r0 >> 7];
            int all = 1;
            for (int v0 = w; v0 < ctas; v0 += 32) {
                bool in = false;
                if (v0 + lane < ctas) {
                    const MaskStart st = a.m.starts[v0 + lane];
                    in = st.q == at.q && st.hk == hk && st.j > 0 && st.j < reach;
                }
                const uint32_t out = ~__ballot_sync(0xffffffffu, in);
                all += out ? __ffs(out) - 1 : 32;
                if (out) break;
            }
            auto done = [&](int r, float l, const float (&o)[PER]) {
                const int pair = it.row0 + r;
                const float inv = 1.f / l;
                bool finite = true;
#pragma unroll
                for (int e = 0; e < PER; ++e) finite = finite && !not_finite(o[e] * inv);
                if (!__all_sync(0xffffffffu, finite)) {
                    masked_row<D>(a, it.t0 + pair / G, hk * G + pair % G);
                    return;
                }
                const long long out = (((long long)it.t0 + pair / G) * a.g.Hq + hk * G + pair % G) * D + lane * PER;
#pragma unroll
                for (int e = 0; e < PER; e += 2) {
                    if (a.g.act == PA_DTYPE_F32) *reinterpret_cast<float2*>((float*)a.output + out + e) = make_float2(o[e] * inv, o[e + 1] * inv);
                    else *reinterpret_cast<uint32_t*>((uint16_t*)a.output + out + e) = a.g.act == PA_DTYPE_F16 ? pack_h2(o[e] * inv, o[e + 1] * inv) : pack_bf2(o[e] * inv, o[e + 1] * inv);
                }
            };
            auto slot = [&](int i) { return (long long)(i == 0 ? 2 * (w - 1) + 1 : 2 * (w + i - 1)) * kPrefillItemRows; };
            const int first = r0 + warp * (kJoinRows / kJoinWarps);
            auto join = [&](auto rows_at_once, auto pieces_at_once) {
                constexpr int R = decltype(rows_at_once)::value, P = decltype(pieces_at_once)::value;
#pragma unroll 1
                for (int r = first; r < first + kJoinRows / kJoinWarps; r += R) {
                    int pieces[R];
#pragma unroll
                    for (int k = 0; k < R; ++k) pieces[k] = r + k < rows ? all : 0;
                    join_rows<D, R, P>(a, pieces, [&](int i, int k) { return slot(i) + r + k; }, [&](int k, float l, const float (&o)[PER]) { done(r + k, l, o); });
                }
            };
            if (all <= 2) join(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
            else join(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
        }
    }
    // rows of whole q tiles that are not finite: once more, by themselves
    const int redo = min(a.plan->total_redo, a.num_tokens * a.g.Hq);
    for (int i = (int)blockIdx.x * kJoinWarps + warp; i < redo; i += gridDim.x * kJoinWarps) {
        const int row = a.m.redo[i];
        masked_row<D>(a, row / a.g.Hq, row % a.g.Hq);
    }
}

}  // namespace

cudaError_t launch_masked_join(const KernelArgs& a, cudaStream_t stream, int* launches) {
    const dim3 grid((a.m.sm_count - 1) * kJoinParts), block(kJoinWarps * 32);
    const cudaError_t e = a.g.D == 128 ? launch_dependent(masked_join_kernel<128>, grid, block, 0, stream, a) : launch_dependent(masked_join_kernel<64>, grid, block, 0, stream, a);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace pa
