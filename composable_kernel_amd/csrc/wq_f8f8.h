// Parameters and launch functions of the fp8 x fp8 kernels (wq_gemm_f8f8.h, compiled in wq_inst_f8f8.hip).
#pragma once

#include "wq_device.h"

namespace wq {

enum F8F8Kernel
{
    F8F8_ANY = 0, // 128 x 128, any alignment and K
    F8F8_64X64,   // 64 x 64, four waves, three workgroups per CU
    F8F8_64,      // 64 x 128, four waves, two workgroups per CU
    F8F8_128,     // 128 x 128, four waves, two workgroups per CU
    F8F8_128_W8,  // 128 x 128, eight waves, one workgroup per CU
    F8F8_128X256, // 128 x 256, eight waves
    F8F8_256,     // 256 x 256, eight waves
    F8F8_SKINNY_DIRECT, // M <= 16 (used up to 4): 16 columns, sixteen waves, weights straight to registers
    F8F8_SKINNY_16,     // M <= 16: 16 columns, eight waves
    F8F8_SKINNY_16X32,  // M <= 16: 32 columns, eight waves
    F8F8_SKINNY_16X64,  // M <= 16: 64 columns, four waves
    F8F8_SKINNY_32,     // M <= 32: 16 columns, eight waves
    F8F8_SKINNY_32X32   // M <= 32: 32 columns, eight waves
};
// K of operands copied to aligned rows
inline int f8f8_padded_k(int K) { return (K + 15) & ~15; }
constexpr int f8f8_bm(int kernel) { return kernel == F8F8_256 ? 256 : kernel == F8F8_64 || kernel == F8F8_64X64 ? 64 : 128; }
constexpr int f8f8_bn(int kernel)
{
    return kernel == F8F8_64X64 ? 64 : kernel <= F8F8_128_W8 ? 128 : kernel <= F8F8_256 ? 256 : kernel == F8F8_SKINNY_16X64 ? 64 : kernel == F8F8_SKINNY_16X32 || kernel == F8F8_SKINNY_32X32 ? 32 : 16;
}

struct F8F8Params
{
    const uint8_t* a;
    const uint8_t* b;
    const float* sa;
    const float* sb;
    void* c; // fp32 slabs [z][M][ldc] when partial
    int M, N, K;
    int lda, ldb, ldc;
    int bm, bn, ld_sa, ld_sb;
    int k_begin, k_end, k_per_z; // slices start on multiples of 128
    int partial;
    int slices;                  // K slices (split-K)
    int tiles_m, tiles_n, group_m;
    float fnuz; // 2^-(number of FNUZ operands)
    int bf16_rtn; // bf16 outputs rounded to nearest even under every epilogue (else truncated, as everywhere in this engine)
    EpilogueArgs epi;
};

int launch_f8f8(int kernel, const F8F8Params& p, hipStream_t s);
void launch_pad_f8(const wqgemm_problem* p, uint8_t* rows, hipStream_t s);
void launch_reduce_f8f8(const float* slabs, int k_batch, int ld_part, const F8F8Params& p, hipStream_t s);

} // namespace wq
