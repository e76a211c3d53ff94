// Masked attention of chunks and trees, rows one by one (masked_row): for caches and activations that the tensor-core kernel does not take.
#include "masked.cuh"
#include "pa_common.cuh"
#include "pa_kernels.h"

namespace pa {

namespace {

template <int D>
__global__ void __launch_bounds__(256) masked_rows_kernel(const __grid_constant__ KernelArgs a) {
    grid_wait();
    const long long warp = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (warp >= (long long)a.num_tokens * a.g.Hq) return;
    masked_row<D>(a, (int)(warp / a.g.Hq), (int)(warp % a.g.Hq));
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
