// Translation unit of the fp8 x fp8 kernels with block-wise scales (wq_gemm_f8f8.h).
#include <hip/hip_runtime.h>
#include <atomic>

#include "wqgemm.h"
#include "wq_gemm_f8f8.h"

namespace wq {

namespace {

// more than 64 KiB of dynamic LDS must be opted into once per device
template <class T, void (*kernel)(const F8F8Params)>
int launch_tile(const F8F8Params& p, dim3 grid, hipStream_t s)
{
    static std::atomic<bool> opted_in[64];
    int dev = 0;
    if(hipGetDevice(&dev) != hipSuccess)
        return WQ_ERR_HIP;
    if(dev < 0 || dev >= 64 || !opted_in[dev])
    {
        if(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS_BYTES) != hipSuccess)
            return WQ_ERR_HIP;
        if(dev >= 0 && dev < 64)
            opted_in[dev] = true;
    }
    hipLaunchKernelGGL(kernel, grid, dim3(T::THREADS), T::LDS_BYTES, s, p);
    return WQ_OK;
}

} // namespace

int launch_f8f8(int kernel, const F8F8Params& p, int k_batch, hipStream_t s)
{
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)k_batch);
    const bool tail = (p.k_end - p.k_begin) % 128 != 0; // (slices between are whole K tiles)
    switch(kernel)
    {
    case F8F8_256:
        return tail ? launch_tile<F8F8Tile<8, 4, 2, 4>, wq_gemm_f8f8_256<true>>(p, grid, s) : launch_tile<F8F8Tile<8, 4, 2, 4>, wq_gemm_f8f8_256<false>>(p, grid, s);
    case F8F8_128:
        return tail ? launch_tile<F8F8Tile<4, 4, 2, 2>, wq_gemm_f8f8_128<true>>(p, grid, s) : launch_tile<F8F8Tile<4, 4, 2, 2>, wq_gemm_f8f8_128<false>>(p, grid, s);
    default: hipLaunchKernelGGL(wq_gemm_f8f8_any, grid, dim3(256), 0, s, p); return WQ_OK;
    }
}

void launch_reduce_f8f8(const float* slabs, int k_batch, int ld_part, const F8F8Params& p, hipStream_t s)
{
    const long blocks = ((long)p.M * (ld_part / 4) + 255) / 256;
    hipLaunchKernelGGL(wq_reduce_f8f8, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, slabs, k_batch, ld_part, p);
}

} // namespace wq
