// Translation unit of the fp8 x fp8 kernels with block-wise scales (wq_gemm_f8f8.h).
#include <hip/hip_runtime.h>

#include "wqgemm.h"
#include "wq_gemm_f8f8.h"

namespace wq {

int launch_f8f8(int kernel, const F8F8Params& p, int k_batch, hipStream_t s)
{
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)k_batch);
    (void)kernel;
    hipLaunchKernelGGL(wq_gemm_f8f8_any, grid, dim3(256), 0, s, p);
    return WQ_OK;
}

void launch_reduce_f8f8(const float* slabs, int k_batch, int ld_part, const F8F8Params& p, hipStream_t s)
{
    const long blocks = ((long)p.M * (ld_part / 4) + 255) / 256;
    hipLaunchKernelGGL(wq_reduce_f8f8, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, slabs, k_batch, ld_part, p);
}

} // namespace wq
