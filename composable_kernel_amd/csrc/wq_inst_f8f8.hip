// Translation unit of the fp8 x fp8 kernels with block-wise scales (wq_gemm_f8f8.h).
#include <hip/hip_runtime.h>
#include <algorithm>
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

int launch_f8f8(int kernel, const F8F8Params& p, hipStream_t s)
{
    const bool tail = (p.k_end - p.k_begin) % 128 != 0; // (slices between are whole K tiles)
    const int kind  = p.epi.kind;
    const bool stream = !p.partial && p.N % 8 == 0 && p.ldc % 8 == 0 && p.ldc <= 1 << 22 && (uintptr_t)p.c % 16 == 0 &&
                        (kind == WQ_EPI_PASSTHROUGH || kind == WQ_EPI_FASTGELU || kind == WQ_EPI_CONVERT_BF16_RTN ||
                         ((kind == WQ_EPI_ADD || kind == WQ_EPI_ADD_FASTGELU) && p.epi.ldd0 == 0));
    // (streaming workgroups walk the tiles: one resident grid on the 256 CUs)
    const long units = (long)p.tiles_m * p.tiles_n * p.slices;
    const dim3 strips((unsigned)p.tiles_n, (unsigned)p.slices); // small-M kernels: strips of columns
    // (the last argument: workgroups that the chip holds at a time)
#define F8F8_TILE_CASE(KIND, TILE, KERNEL, RESIDENT)                                                                             \
    case KIND:                                                                                                                   \
        return stream ? tail ? launch_tile<TILE, KERNEL<true, true>>(p, dim3((unsigned)std::min(units, (long)RESIDENT)), s)      \
                             : launch_tile<TILE, KERNEL<false, true>>(p, dim3((unsigned)std::min(units, (long)RESIDENT)), s)     \
               : tail ? launch_tile<TILE, KERNEL<true, false>>(p, dim3((unsigned)units), s)                                      \
                      : launch_tile<TILE, KERNEL<false, false>>(p, dim3((unsigned)units), s);
    switch(kernel)
    {
        F8F8_TILE_CASE(F8F8_256, F8F8Tile256, wq_gemm_f8f8_256, 256)
        F8F8_TILE_CASE(F8F8_128X256, F8F8Tile128x256, wq_gemm_f8f8_128x256, 256)
        F8F8_TILE_CASE(F8F8_128, F8F8Tile128, wq_gemm_f8f8_128, 512)
        F8F8_TILE_CASE(F8F8_128_W8, F8F8Tile128W8, wq_gemm_f8f8_128_w8, 256)
        F8F8_TILE_CASE(F8F8_64, F8F8Tile64, wq_gemm_f8f8_64, 512)
        F8F8_TILE_CASE(F8F8_64X64, F8F8Tile64x64, wq_gemm_f8f8_64x64, 768)
#undef F8F8_TILE_CASE
    case F8F8_SKINNY_DIRECT: hipLaunchKernelGGL((wq_gemm_f8f8_skinny_direct<16, 2>), strips, dim3(1024), 0, s, p); return WQ_OK;
    case F8F8_SKINNY_16: return launch_tile<F8F8Skinny<1, 1, 8, 2>, wq_gemm_f8f8_skinny<1, 1, 8, 2>>(p, strips, s);
    case F8F8_SKINNY_16X64: return launch_tile<F8F8Skinny<1, 4, 4, 2>, wq_gemm_f8f8_skinny<1, 4, 4, 2>>(p, strips, s);
    case F8F8_SKINNY_16X32: return launch_tile<F8F8Skinny<1, 2, 8, 1>, wq_gemm_f8f8_skinny<1, 2, 8, 1>>(p, strips, s);
    case F8F8_SKINNY_32X32: return launch_tile<F8F8Skinny<2, 2, 8, 1>, wq_gemm_f8f8_skinny<2, 2, 8, 1>>(p, strips, s);
    case F8F8_SKINNY_32: return launch_tile<F8F8Skinny<2, 1, 8, 1>, wq_gemm_f8f8_skinny<2, 1, 8, 1>>(p, strips, s);
    default:
        hipLaunchKernelGGL(wq_gemm_f8f8_any, dim3((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)p.slices), dim3(256), 0, s, p);
        return WQ_OK;
    }
}

void launch_pad_f8(const wqgemm_problem* p, uint8_t* rows, hipStream_t s)
{
    hipLaunchKernelGGL(wq_pad_rows_f8, dim3((unsigned)std::min(((long)p->M + p->N + 3) / 4, 1L << 16)), dim3(256), 0, s, (const uint8_t*)p->a, (long)p->lda, p->M,
                       (const uint8_t*)p->b, (long)p->ldb, p->N, p->K, rows);
}

void launch_reduce_f8f8(const float* slabs, int k_batch, int ld_part, const F8F8Params& p, hipStream_t s)
{
    const long blocks = ((long)p.M * (ld_part / 4) + 255) / 256;
    hipLaunchKernelGGL(wq_reduce_f8f8, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, slabs, k_batch, ld_part, p);
}

} // namespace wq
