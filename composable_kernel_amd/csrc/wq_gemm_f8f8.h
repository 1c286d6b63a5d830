// fp8 x fp8 GEMM with block-wise scales of both operands (gfx950).
//
//   C[m, n] = epilogue( sum_kb sa[m / bm, kb] * sb[kb, n / bn] * ( sum_{k in kb} a[m, k] * b[k, n] ) ),   kb = k / 128
//
// a: e4m3 bytes, K contiguous per row; b: e4m3 bytes, K contiguous per column; sa, sb: fp32.  One scale block along K is
// one K step of v_mfma_f32_16x16x128_f8f6f4, so the sum of a block is one instruction from a zero accumulator and the
// scales are applied once per block and output, acc = fma(sum, sa * sb, acc), in fp32.
// FNUZ bytes decode as twice their value (see wq_gemm_256_f8.h); the factor 1/2 per FNUZ operand rides on sb.
#pragma once

#include "wq_f8f8.h"
#include "wq_gemm_256_f8.h"

namespace wq {

__device__ __forceinline__ uint16_t f8f8_cvt16(const F8F8Params& p, float v)
{
    if(p.epi.c_dtype == 1 /*WQ_BF16*/ && p.bf16_rtn)
        v = convert_bf16_rtn_bits(v);
    return cvt_out16(v, p.epi.c_dtype);
}

// Four consecutive outputs (n .. n+3) of row m: epilogue, conversion, store; columns at and past N are left alone.
// (the kind is resolved at run time: this runs once per four outputs, outside the unrolled fragment loops)
__device__ __forceinline__ void f8f8_store4(const F8F8Params& p, f4_t v, int m, int n)
{
    if(m >= p.M || n >= p.N)
        return;
    const int cols = min(p.N - n, 4);
    if(p.partial)
    {
        float* c = (float*)p.c + ((size_t)blockIdx.z * p.M + m) * (size_t)p.ldc + n;
        if(cols == 4)
            __builtin_memcpy(c, &v, 16);
        else
            for(int j = 0; j < cols; ++j)
                c[j] = v[j];
        return;
    }
    uint16_t o[4];
#pragma unroll
    for(int j = 0; j < 4; ++j)
        o[j] = j < cols ? f8f8_cvt16(p, apply_epilogue(p.epi, v[j], m, n + j)) : (uint16_t)0;
    uint16_t* c = (uint16_t*)p.c + (size_t)m * (size_t)p.ldc + n;
    if(cols == 4)
        __builtin_memcpy(c, o, 8);
    else
        for(int j = 0; j < cols; ++j)
            c[j] = o[j];
}

// 16 bytes of an operand row from k, bytes at and past `end` as zeros; no alignment assumption
__device__ __forceinline__ u4_t f8f8_load16(const uint8_t* row, int k, int end)
{
    u4_t v = {0, 0, 0, 0};
    if(k + 16 <= end)
        __builtin_memcpy(&v, row + k, 16);
    else
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            if(k + j < end)
                v[j >> 2] |= (uint32_t)row[k + j] << (8 * (j & 3));
    }
    return v;
}

__device__ __forceinline__ i8v_t f8f8_frag(u4_t lo, u4_t hi)
{
    return i8v_t{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// ---------------------------------------------------------------------------------------------
// 128 x 128 tile, four waves of 32 columns, for operands of any alignment and any K: global loads with per-byte tails,
// activations through one LDS buffer (the next tile's bytes wait in registers), weights straight to registers.
// ---------------------------------------------------------------------------------------------
struct F8F8Any
{
    static constexpr int BM = 128, BN = 128, BK = 128, MT = 8, NT = 2;
    static constexpr int A_PITCH = 144; // 128 bytes + 16: 16 rows of a fragment read start in different banks
    static constexpr int C_PITCH = 132; // floats
};

__global__ __launch_bounds__(256) void wq_gemm_f8f8_any(const F8F8Params p)
{
    using T = F8F8Any;
    constexpr int MT = T::MT, NT = T::NT;
    __shared__ __attribute__((aligned(16))) uint8_t lds_a[T::BM * T::A_PITCH];
    __shared__ float lds_s[T::BM];
    __shared__ __attribute__((aligned(16))) float lds_c[32 * T::C_PITCH];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 15, fq = lane >> 4;
    int tm, tn;
    tile_coords(xcd_remap(blockIdx.x, p.tiles_m * p.tiles_n), p.tiles_m, p.tiles_n, p.group_m, tm, tn);
    const int m0 = tm * T::BM, n0 = tn * T::BN, nw = n0 + wave * 32;
    const int k0 = p.k_begin + blockIdx.z * p.k_per_z, k1 = min(p.k_end, k0 + p.k_per_z);

    // rows and columns past the edge repeat the last one: their results are not stored
    const uint8_t* a_row[4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
        a_row[i] = p.a + (size_t)min(m0 + i * 32 + (int)(threadIdx.x >> 3), p.M - 1) * (size_t)p.lda;
    const int a_k = (threadIdx.x & 7) * 16;
    const uint8_t* b_col[NT];
#pragma unroll
    for(int nt = 0; nt < NT; ++nt)
        b_col[nt] = p.b + (size_t)min(nw + nt * 16 + fr, p.N - 1) * (size_t)p.ldb;
    const float* sa_row = p.sa + (size_t)(min(m0 + (int)(threadIdx.x & 127), p.M - 1) / p.bm) * (size_t)p.ld_sa;
    const float* sb_col = p.sb + (size_t)(min(nw, p.N - 1) / p.bn) * (size_t)p.ld_sb; // (bn is a multiple of 32: one block per wave)

    f4_t acc[NT][MT];
#pragma unroll
    for(int nt = 0; nt < NT; ++nt)
#pragma unroll
        for(int mt = 0; mt < MT; ++mt)
            acc[nt][mt] = f4_t{0.f, 0.f, 0.f, 0.f};

    u4_t ra[4], rb[NT][2];
    float rs = 0.f;
    auto load = [&](int k) __attribute__((always_inline)) {
#pragma unroll
        for(int i = 0; i < 4; ++i)
            ra[i] = f8f8_load16(a_row[i], k + a_k, k1);
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
#pragma unroll
            for(int h = 0; h < 2; ++h)
                rb[nt][h] = f8f8_load16(b_col[nt], k + fq * 32 + h * 16, k1);
        rs = sa_row[k >> 7];
    };
    if(k0 < k1)
        load(k0);
    for(int k = k0; k < k1; k += T::BK)
    {
#pragma unroll
        for(int i = 0; i < 4; ++i)
            *(u4_t*)(lds_a + (i * 32 + (threadIdx.x >> 3)) * T::A_PITCH + a_k) = ra[i];
        if(threadIdx.x < T::BM)
            lds_s[threadIdx.x] = rs;
        i8v_t bf[NT];
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
            bf[nt] = f8f8_frag(rb[nt][0], rb[nt][1]);
        const float sb = sb_col[k >> 7] * p.fnuz;
        __syncthreads();
        if(k + T::BK < k1)
            load(k + T::BK);
#pragma unroll
        for(int mt = 0; mt < MT; ++mt)
        {
            const uint8_t* s = lds_a + (mt * 16 + fr) * T::A_PITCH + fq * 32;
            const i8v_t af   = f8f8_frag(*(const u4_t*)s, *(const u4_t*)(s + 16));
            const float sc   = lds_s[mt * 16 + fr] * sb;
#pragma unroll
            for(int nt = 0; nt < NT; ++nt)
            {
                const f4_t zero = {0.f, 0.f, 0.f, 0.f};
                const f4_t sum  = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[nt], af, zero, 0, 0, 0, 0, 0, 0);
                acc[nt][mt]     = __builtin_elementwise_fma(sum, f4_t{sc, sc, sc, sc}, acc[nt][mt]);
            }
        }
        __syncthreads();
    }

    // out through LDS, 32 rows at a time, so that the epilogue and the edge handling stand in one rolled loop
#pragma unroll
    for(int ph = 0; ph < MT / 2; ++ph)
    {
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
#pragma unroll
            for(int mi = 0; mi < 2; ++mi)
                *(f4_t*)(lds_c + (mi * 16 + fr) * T::C_PITCH + wave * 32 + nt * 16 + fq * 4) = acc[nt][ph * 2 + mi];
        __syncthreads();
#pragma unroll 1
        for(int i = 0; i < 4; ++i)
        {
            const int r = i * 8 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * 4;
            f8f8_store4(p, *(const f4_t*)(lds_c + r * T::C_PITCH + c), m0 + ph * 32 + r, n0 + c);
        }
        __syncthreads();
    }
}

// Split-K: out[m, n] = epilogue(sum_z slab[z][m][n]), z ascending, for any N (ld_part is N rounded up to 4).
__global__ __launch_bounds__(256) void wq_reduce_f8f8(const float* __restrict__ slabs, int k_batch, int ld_part, F8F8Params p)
{
    const int n4     = ld_part >> 2;
    const long total = (long)p.M * n4;
    for(long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256)
    {
        const int m = (int)(i / n4), n = (int)(i % n4) * 4;
        f4_t s = *(const f4_t*)(slabs + (size_t)m * ld_part + n);
        for(int z = 1; z < k_batch; ++z)
            s += *(const f4_t*)(slabs + ((size_t)z * p.M + m) * (size_t)ld_part + n);
        f8f8_store4(p, s, m, n);
    }
}

} // namespace wq
