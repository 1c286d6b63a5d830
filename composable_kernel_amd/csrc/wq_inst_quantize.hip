// Translation unit of the row quantisers (wq_quantize.h): kernel selection and launch.
#include <hip/hip_runtime.h>
#include <algorithm>

#include "wqgemm.h"
#include "wq_quantize.h"

namespace wq {

namespace {

template <int OP, bool BF16>
void launch_groups(const QuantParams& p, hipStream_t s)
{
    const int chunks  = (p.K + 511) / 512;
    const long waves  = (long)p.M * chunks;
    const long blocks = (waves + 3) / 4;
    // (a grid of four rounds walks what is left: 8192 x 8192 37.7 us; of one 39.3, a workgroup for every four waves 40.2)
    hipLaunchKernelGGL((wq_quantize_groups<OP, BF16>), dim3((unsigned)std::min(blocks, 256L * 32)), dim3(256), 0, s, p, chunks);
}

template <int OP, bool BF16, bool GROUPED>
void launch_row(QuantParams p, hipStream_t s)
{
    // (a launch holds fewer than 2^32 work items: more rows than that go in several)
    constexpr int MOST = 1 << 21;
    for(; p.M > MOST; p.M -= MOST)
    {
        QuantParams part = p;
        part.M           = MOST;
        launch_row<OP, BF16, GROUPED>(part, s);
        p.x     = (const uint16_t*)p.x + MOST * p.ldx;
        p.x2    = p.x2 ? (const uint16_t*)p.x2 + MOST * p.ldx2 : nullptr;
        p.q     = p.q + MOST * p.ldq;
        p.scale = p.scale + MOST * p.ld_scale;
        p.residual_out = p.residual_out ? (uint16_t*)p.residual_out + MOST * p.ld_res : nullptr;
    }
    // Threads: 512 with up to two pieces each in registers (norm of 4096 x 8192: 51.8 us = 4.5 TB/s; 256 threads 60, 1024 54), 1024
    // for longer rows, and while there are few rows, where the latency of one counts (64 x 8192: 3.9 us, 512 threads 4.3).  The norm's
    // sums do not see which: only T = 512 with two pieces stands for another T, and wq_quantize_row sums those two apart.
    const long pieces = ((long)p.K + 7) / 8;
    int T             = p.M >= 512 ? 512 : 1024;
    while(T > 64 && pieces <= T / 2)
        T >>= 1;
    if(pieces > 2L * T)
        T = 1024;
    const long r = (pieces + T - 1) / T;
    const dim3 grid((unsigned)p.M), block((unsigned)T);
    if(r <= 1)
        hipLaunchKernelGGL((wq_quantize_row<OP, BF16, GROUPED, 1>), grid, block, 0, s, p);
    else if(r <= 2)
        hipLaunchKernelGGL((wq_quantize_row<OP, BF16, GROUPED, 2>), grid, block, 0, s, p);
    else if(r <= 4)
        hipLaunchKernelGGL((wq_quantize_row<OP, BF16, GROUPED, 4>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((wq_quantize_row<OP, BF16, GROUPED, 0>), grid, block, 0, s, p);
}

template <bool BF16>
void launch_typed(const QuantParams& p, int op, bool grouped, hipStream_t s)
{
    if(op == WQ_QUANT_RMSNORM)
        grouped ? launch_row<1, BF16, true>(p, s) : launch_row<1, BF16, false>(p, s);
    else if(op == WQ_QUANT_GATED)
        grouped ? launch_groups<2, BF16>(p, s) : launch_row<2, BF16, false>(p, s);
    else
        grouped ? launch_groups<0, BF16>(p, s) : launch_row<0, BF16, false>(p, s);
}

} // namespace

void launch_quantize(const wqgemm_quant* d, hipStream_t s)
{
    QuantParams p;
    p.x = d->x, p.x2 = d->x2, p.weight = d->weight, p.q = (uint8_t*)d->q, p.scale = d->scale, p.residual_out = d->residual_out;
    p.M = d->M, p.K = d->K;
    p.ldx = d->ldx, p.ldx2 = d->ldx2, p.ld_res = d->ld_residual_out, p.ldq = d->ldq, p.ld_scale = d->ld_scale;
    p.weight_f32 = d->weight_dtype == WQ_F32;
    p.act        = d->activation;
    p.eps        = d->eps;
    const bool grouped = d->group_k > 0;
    d->dtype == WQ_BF16 ? launch_typed<true>(p, d->op, grouped, s) : launch_typed<false>(p, d->op, grouped, s);
}

} // namespace wq
