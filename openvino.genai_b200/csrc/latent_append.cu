// Writing a step's latent rows into their paged cache: norm of the latent, rotation of the shared key part, and the rotation of the
// queries' part in the same launch (include/latent_b200.h: pa_b200_latent_append).
#include "latent_kernels.h"

#include <algorithm>

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

// Eight pairs of one row: its l-th piece of sixteen elements, in two loads that are under way until they are turned.
struct Piece {
    uint4 w0, w1;
    __device__ __forceinline__ void load(const uint16_t* src, int P, int l, bool interleaved) {
        w0 = *reinterpret_cast<const uint4*>(src + (interleaved ? 16 * l : 8 * l));
        w1 = *reinterpret_cast<const uint4*>(src + (interleaved ? 16 * l + 8 : P / 2 + 8 * l));
    }
    template <bool BF>
    __device__ __forceinline__ void store(uint16_t* dst, const float* table, int P, int l, bool interleaved) const {
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
        *reinterpret_cast<uint4*>(dst + (interleaved ? 16 * l : 8 * l)) = pack8<BF>(y0);
        *reinterpret_cast<uint4*>(dst + (interleaved ? 16 * l + 8 : P / 2 + 8 * l)) = pack8<BF>(y1);
    }
};

constexpr int kQueryWarps = 8;

// A block takes a token: warp 0 its latent row, the others its heads' query rows in pieces of sixteen elements, two to a lane at a time.  The
// kernel is bound by HBM; what it reads does not depend on where the token belongs, so the rows are under way before the search for the token's
// sequence begins (five dependent loads for 32 sequences, one more for the position and one for the page): 17,411 tokens of ragged
// prompts by 32 heads of 64 elements, 187 MB, 50.7 -> 42.1 us with one piece to a lane, 35.3 us with two (5.3 TB/s); 36.2 us with a second round of
// two.  256 tokens by 128 heads 4.6 -> 4.1 us.
template <bool BF>
__global__ void __launch_bounds__(32 + 32 * kQueryWarps, 4) append_kernel(AppendArgs a) {
    pa::grid_wait();
    pa::grid_release();
    const Step& m = a.m;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x;
    const int per_row = m.P / 16;                         // pieces (2 or 4)
    const int shift = per_row >> 1;                       // and their log2
    const bool interleaved = a.interleaved != 0;
    const int total = m.H * per_row, step = blockDim.x - 32;
    const uint16_t* q = (const uint16_t*)a.q_in + t * a.q_in_token;
    const uint16_t* src = (const uint16_t*)a.latent + t * a.latent_stride;
    const int nv = m.R / 256;
    uint4 raw[2];
    Piece piece[2];
    int u = (int)threadIdx.x - 32;
    if (warp > 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (u + i * step < total) piece[i].load(q + ((u + i * step) >> shift) * a.q_in_head, m.P, (u + i * step) & (per_row - 1), interleaved);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < nv) raw[i] = *reinterpret_cast<const uint4*>(src + 256 * i + 8 * lane);
        if (lane < per_row) piece[0].load(src + m.R, m.P, lane, interleaved);
    }
    SeqView v;
    if (!token_view(m, t, v)) return;
    const int at = v.past + (t - v.t0), pos = a.positions ? a.positions[t] : at;
    if (pos < 0 || pos >= a.rope_rows) {
        if (threadIdx.x == 0) atomicOr(m.status, PA_DEV_BAD_ROTATION);
        return;
    }
    const float* table = a.rope_table + (long long)pos * m.P;
    if (warp > 0) {
        uint16_t* out = (uint16_t*)a.q_out + t * a.q_out_token;
        for (;;) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (u + i * step < total)
                    piece[i].store<BF>(out + ((u + i * step) >> shift) * a.q_out_head, table, m.P, (u + i * step) & (per_row - 1), interleaved);
            u += 2 * step;
            if (u >= total) return;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (u + i * step < total) piece[i].load(q + ((u + i * step) >> shift) * a.q_in_head, m.P, (u + i * step) & (per_row - 1), interleaved);
        }
    }
    const int page = m.block_indices[v.tb + at / m.bs];
    if (page < 0 || page >= m.num_blocks) {
        if (lane == 0) atomicOr(m.status, PA_DEV_BAD_BLOCK_INDEX);
        return;
    }
    uint16_t* dst = (uint16_t*)a.cache + ((long long)page * m.bs + at % m.bs) * (m.R + m.P);
    float inv = 1.f;
    if (a.norm_weight) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < nv) {
                float x[8];
                unpack8<BF>(raw[i], x);
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += x[k] * x[k];
            }
        inv = rsqrtf(pa::warp_sum(sum) / (float)m.R + a.norm_eps);
    }
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
    if (lane < per_row) piece[0].store<BF>(dst + m.R, table, m.P, lane, interleaved);
}

}  // namespace

cudaError_t launch_append(const AppendArgs& a, int dtype, cudaStream_t stream, int* launches) {
    const int warps = a.q_in ? std::min(kQueryWarps, (a.m.H * (a.m.P / 16) + 63) / 64) : 0;      // two pieces to a lane
    ++*launches;
    return pa::launch_dependent(dtype == PA_DTYPE_BF16 ? append_kernel<true> : append_kernel<false>, a.m.num_tokens, 32 + 32 * warps, 0, stream, a);
}

}  // namespace latent
