// Writing a step's latent rows into their paged cache: norm of the latent, rotation of the shared key part, and the rotation of the
// queries' part in the same launch (include/latent_b200.h: pa_b200_latent_append).
#include "latent_kernels.h"

namespace latent {

namespace {

// Eight 16-bit elements and their values.
template <bool BF>
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (BF) {
            x[2 * k] = __uint_as_float(u[k] << 16);
            x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
            x[2 * k] = f.x; x[2 * k + 1] = f.y;
        }
    }
}
template <bool BF>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) u[k] = BF ? pa::pack_bf2(x[2 * k], x[2 * k + 1]) : pa::pack_h2(x[2 * k], x[2 * k + 1]);
    return make_uint4(u[0], u[1], u[2], u[3]);
}

// Eight pairs of one row: l-th piece of sixteen elements.  `src` and `dst` are the row's P elements.
template <bool BF>
__device__ __forceinline__ void rotate16(const uint16_t* src, uint16_t* dst, const float* table, int P, int l, bool interleaved) {
    const int at0 = interleaved ? 16 * l : 8 * l, at1 = interleaved ? 16 * l + 8 : P / 2 + 8 * l;
    const uint4 w0 = *reinterpret_cast<const uint4*>(src + at0), w1 = *reinterpret_cast<const uint4*>(src + at1);
    float c[8], s[8];
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
        const float4 c4 = *reinterpret_cast<const float4*>(table + 8 * l + k), s4 = *reinterpret_cast<const float4*>(table + P / 2 + 8 * l + k);
        c[k] = c4.x; c[k + 1] = c4.y; c[k + 2] = c4.z; c[k + 3] = c4.w;
        s[k] = s4.x; s[k + 1] = s4.y; s[k + 2] = s4.z; s[k + 3] = s4.w;
    }
    float x0[8], x1[8], y0[8], y1[8];
    unpack8<BF>(w0, x0);
    unpack8<BF>(w1, x1);
    if (interleaved) {
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            y0[k] = x0[k] * c[k / 2] - x0[k + 1] * s[k / 2];
            y0[k + 1] = x0[k + 1] * c[k / 2] + x0[k] * s[k / 2];
            y1[k] = x1[k] * c[4 + k / 2] - x1[k + 1] * s[4 + k / 2];
            y1[k + 1] = x1[k + 1] * c[4 + k / 2] + x1[k] * s[4 + k / 2];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            y0[k] = x0[k] * c[k] - x1[k] * s[k];
            y1[k] = x1[k] * c[k] + x0[k] * s[k];
        }
    }
    *reinterpret_cast<uint4*>(dst + at0) = pack8<BF>(y0);
    *reinterpret_cast<uint4*>(dst + at1) = pack8<BF>(y1);
}

// A warp takes a token's latent row, or 32 pieces (sixteen elements each) of its heads' query rows.
template <bool BF>
__global__ void __launch_bounds__(256) append_kernel(AppendArgs a) {
    pa::grid_wait();
    pa::grid_release();
    const Step& m = a.m;
    const int lane = threadIdx.x & 31;
    const int pieces = m.P / 16;                                            // lanes of one row's rotation
    const int per_token = 1 + (a.q_in ? (m.H * pieces + 31) / 32 : 0);     // warps
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int t = (int)(warp / per_token), part = (int)(warp % per_token);
    if (t >= m.num_tokens) return;
    SeqView v;
    if (!token_view(m, t, v)) return;
    const int at = v.past + (t - v.t0), pos = a.positions ? a.positions[t] : at;
    if (pos < 0 || pos >= a.rope_rows) {
        if (lane == 0) atomicOr(m.status, PA_DEV_BAD_ROTATION);
        return;
    }
    const float* table = a.rope_table + (long long)pos * m.P;
    if (part > 0) {
        const int u = (part - 1) * 32 + lane, h = u / pieces;
        if (h < m.H)
            rotate16<BF>((const uint16_t*)a.q_in + t * a.q_in_token + h * a.q_in_head, (uint16_t*)a.q_out + t * a.q_out_token + h * a.q_out_head,
                         table, m.P, u % pieces, a.interleaved != 0);
        return;
    }
    const int page = m.block_indices[v.tb + at / m.bs];
    if (page < 0 || page >= m.num_blocks) {
        if (lane == 0) atomicOr(m.status, PA_DEV_BAD_BLOCK_INDEX);
        return;
    }
    const uint16_t* src = (const uint16_t*)a.latent + t * a.latent_stride;
    uint16_t* dst = (uint16_t*)a.cache + ((long long)page * m.bs + at % m.bs) * (m.R + m.P);
    uint4 raw[2];
    const int nv = m.R / 256;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (i < nv) {
            raw[i] = *reinterpret_cast<const uint4*>(src + 256 * i + 8 * lane);
            float x[8];
            unpack8<BF>(raw[i], x);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += x[k] * x[k];
        }
    }
    const float inv = a.norm_weight ? rsqrtf(pa::warp_sum(sum) / (float)m.R + a.norm_eps) : 1.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (i < nv) {
            if (a.norm_weight) {
                float x[8], w[8];
                unpack8<BF>(raw[i], x);
                unpack8<BF>(*reinterpret_cast<const uint4*>((const uint16_t*)a.norm_weight + 256 * i + 8 * lane), w);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = x[k] * inv * w[k];
                raw[i] = pack8<BF>(x);
            }
            *reinterpret_cast<uint4*>(dst + 256 * i + 8 * lane) = raw[i];
        }
    }
    if (lane < pieces) rotate16<BF>(src + m.R, dst + m.R, table, m.P, lane, a.interleaved != 0);
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, int dtype, cudaStream_t stream, int* launches) {
    const long long warps = (long long)a.m.num_tokens * (1 + (a.q_in ? (a.m.H * (a.m.P / 16) + 31) / 32 : 0));
    const unsigned blocks = (unsigned)((warps + 7) / 8);
    ++*launches;
    return pa::launch_dependent(dtype == PA_DTYPE_BF16 ? append_kernel<true> : append_kernel<false>, blocks, 256, 0, stream, a);
}

}  // namespace latent
