// Latent attention, straight from the formulas: one CTA per (new token, head), everything in f32.
#include "latent_kernels.h"

namespace latent {

namespace {

constexpr int kWarps = 8;

// A warp takes every eighth position; lane l holds elements l, l + 32, .. of the absorbed query and of its sum of latents.
template <class T, int NR>
__global__ void __launch_bounds__(kWarps * 32) simple_kernel(AttentionArgs a) {
    constexpr int R = 32 * NR;
    __shared__ float sh_q[R + 64];
    __shared__ float sh_o[kWarps][R];
    __shared__ float sh_m[kWarps], sh_l[kWarps];
    const Step& m = a.m;
    const int t = blockIdx.x / m.H, h = blockIdx.x % m.H, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    SeqView v;
    if (!token_view(m, t, v) || v.n < a.min_new) return;
    const T* qn = (const T*)a.q_nope + t * a.qn_token + h * a.qn_head;
    const T* qr = (const T*)a.q_rope + t * a.qr_token + h * a.qr_head;
    const T* up = (const T*)a.key_up + h * a.key_up_head;
    for (int r = tid; r < R; r += blockDim.x) {
        float s = 0.f;
        for (int d = 0; d < m.Dn; ++d) s += pa::to_float(qn[d]) * pa::to_float(up[(long long)d * R + r]);
        sh_q[r] = s;
    }
    if (tid < 64) sh_q[R + tid] = tid < m.P ? pa::to_float(qr[tid]) : 0.f;
    __syncthreads();
    const int ctx = v.past + (t - v.t0) + 1;
    float o[NR], mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) o[i] = 0.f;
    for (int j = warp; j < ctx; j += kWarps) {
        int page = m.block_indices[v.tb + j / m.bs];
        if (page < 0 || page >= m.num_blocks) {
            if (lane == 0) atomicOr(m.status, PA_DEV_BAD_BLOCK_INDEX);
            page = 0;
        }
        const T* row = (const T*)a.cache + ((long long)page * m.bs + j % m.bs) * (R + m.P);
        float c[NR], s = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            c[i] = pa::to_float(row[32 * i + lane]);
            s += c[i] * sh_q[32 * i + lane];
        }
        for (int i = lane; i < m.P; i += 32) s += pa::to_float(row[R + i]) * sh_q[R + i];
        s = pa::warp_sum(s) * a.scale;
        const float top = fmaxf(mx, s), keep = expf(mx - top), p = expf(s - top);
        mx = top;
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < NR; ++i) o[i] = o[i] * keep + p * c[i];
    }
    if (lane == 0) { sh_m[warp] = mx; sh_l[warp] = l; }
#pragma unroll
    for (int i = 0; i < NR; ++i) sh_o[warp][32 * i + lane] = o[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sh_m[w]);
    for (int w = 0; w < kWarps; ++w) sum += sh_l[w] * expf(sh_m[w] - top);
    for (int r = tid; r < R; r += blockDim.x) {
        float x = 0.f;
        for (int w = 0; w < kWarps; ++w) x += sh_o[w][r] * expf(sh_m[w] - top);
        sh_q[r] = x / sum;
    }
    __syncthreads();
    const T* vu = (const T*)a.value_up + h * a.value_up_head;
    for (int d = warp; d < m.Dv; d += kWarps) {
        float s = 0.f;
        for (int r = lane; r < R; r += 32) s += sh_q[r] * pa::to_float(vu[(long long)d * R + r]);
        s = pa::warp_sum(s);
        if (lane == 0) pa::from_float(((T*)a.output)[((long long)t * m.H + h) * m.Dv + d], s);
    }
}

}  // namespace

cudaError_t launch_attention_simple(const AttentionArgs& a, int dtype, cudaStream_t stream, int* launches) {
    const unsigned grid = (unsigned)(a.m.num_tokens * a.m.H);
    if (dtype == PA_DTYPE_BF16) {
        if (a.m.R == 512) simple_kernel<__nv_bfloat16, 16><<<grid, kWarps * 32, 0, stream>>>(a);
        else simple_kernel<__nv_bfloat16, 8><<<grid, kWarps * 32, 0, stream>>>(a);
    } else {
        if (a.m.R == 512) simple_kernel<__half, 16><<<grid, kWarps * 32, 0, stream>>>(a);
        else simple_kernel<__half, 8><<<grid, kWarps * 32, 0, stream>>>(a);
    }
    ++*launches;
    return cudaGetLastError();
}

}  // namespace latent
