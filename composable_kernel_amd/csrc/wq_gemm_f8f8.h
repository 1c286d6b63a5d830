// fp8 x fp8 GEMM with block-wise scales of both operands (gfx950).
//
//   C[m, n] = epilogue( sum_kb sa[m / bm, kb] * sb[kb, n / bn] * ( sum_{k in kb} a[m, k] * b[k, n] ) ),   kb = k / 128
//
// a: e4m3 bytes, K contiguous per row; b: e4m3 bytes, K contiguous per column; sa, sb: fp32.  One scale block along K is
// one K step of v_mfma_f32_16x16x128_f8f6f4, so the sum of a block is one instruction from a zero accumulator and the
// scales are applied once per block and output, acc = fma(sum, sa * sb, acc), in fp32.
// Inside the instruction 8 consecutive k share an exponent: what lies below 2^-13 of the largest of their products is dropped
// (2^16 + 2^3 survives, 2^16 + 2^2 does not; 8 k apart 2^16 + 2^-7 does), an error of less than 7 * 2^-13 of sum |a b|.  Taken
// because it is small beside what the operands lost in 8 bits: on normal data 1.4e-5 of the outputs' root mean square, fp16
// rounding 2e-4, the operands' own roundings 3e-2; wq_gemm_generic sums in fp32 throughout.
// FNUZ bytes decode as twice their value (see wq_gemm_256_f8.h); the factor 1/2 per FNUZ operand rides on sb.
#pragma once

#include <utility>

#include "wq_f8f8.h"
#include "wq_f8f8_walk.h"
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
__device__ __forceinline__ void f8f8_store4(const F8F8Params& p, f4_t v, int m, int n, int z)
{
    if(m >= p.M || n >= p.N)
        return;
    const int cols = min(p.N - n, 4);
    if(p.partial)
    {
        float* c = (float*)p.c + ((size_t)z * p.M + m) * (size_t)p.ldc + n;
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
            f8f8_store4(p, *(const f4_t*)(lds_c + r * T::C_PITCH + c), m0 + ph * 32 + r, n0 + c, blockIdx.z);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// BM x BN tile for 16-byte aligned operands: WR x WC waves, each MT row blocks x NT column blocks of 16.
//
// Bound by the matrix core with one fused multiply-add per output and K tile beside it: in registers alone 3440 TFLOP/s on random
// bits (4080 without the folds).  256 x 256 reaches 2100 (4096 x 4096 x 4096 65 us, 4096 x 11008 x 4096 175; 145 on zeros, where the
// clock holds): MFMAs take 63 % of a busy CU's cycles, 5.4 vector instructions go with each, LDS is busy 36 % of them.
//
// Both operands pass through LDS (LDS-DMA, 8 rows of 128 bytes per piece).  Weights fetched straight into the registers of the
// MFMA were slower: a wave's load then touches 16 rows, and the vector cache takes one access per lane instead of one per 64
// bytes, 2048 cycles per 256 x 256 x 128 step, as long as its MFMAs (205 us at 4096 x 11008 x 4096 with 32 columns a wave, 222
// with 64, two workgroups per CU).
//   * two LDS slots of a whole K tile; each half of a tile's rows has a barrier of its own, in front of the row block that first
//     reads the next half, and refills what the half before it has freed: every piece is issued at least a K tile's time before
//     its barrier.  Weights live in registers for a K tile: read at its end, each column block behind the last MFMA that needs
//     the old one, so that their slot is free for most of it.  Activations are read LEAD row blocks ahead;
//   * scales: once per four K tiles the row scales of those four travel as one 16-byte LDS-DMA piece per row (every row's scales
//     lie in a cache line of their own, so fetching them tile by tile would move a line per row and tile, as much as the
//     activations themselves), and the column blocks' the same way.  A table row of fewer than four scales (K <= 384) is copied by
//     ordinary loads instead, to the end of the same 16 bytes;
//   * a block sum is one MFMA from a zero accumulator.  The sums of a row block are folded into the accumulators,
//     acc = fma(sum, sa * sb, acc), each just in front of the next row block's MFMA that overwrites it: NT MFMAs after it was
//     issued, so that neither waits for the other.
// VMEM bookkeeping (in-order completion, counted waits).  Behind barrier(t, 0), in front of row block MT / 2 - LEAD of tile t:
// A(t + 2) first half, B(t + 2), one scale piece [group (t, 0)]; behind barrier(t, 1), in front of row block MT - LEAD: A(t + 2)
// second half [group (t, 1)].  barrier(t, 0) needs group (t - 2, 1) = A(t) second half, barrier(t, 1) needs group (t - 1, 0) =
// A(t + 1) first half, B(t + 1), scales: two groups, one of each kind, were issued behind either.  Each wave also waits for its
// own LDS reads in front of a barrier: what the pieces behind it overwrite has been read by everybody.  (The tile body has no
// branch: the compiler would sink the fused multiply-adds behind it and keep every block sum alive.)
// STREAM (epilogues with at most a bias per column and a FastGelu): a workgroup walks tiles blockIdx.x, + gridDim.x, ... and
// issues the next tile's first loads before this one's outputs leave.
// Tiles past the last one are loaded through a resource of zero records: no memory access.  TAIL: the last K tile is partial
// (K a multiple of 16): its 16-byte pieces past the end are sent out of range, which reads as zeros.
// ---------------------------------------------------------------------------------------------
template <int MT_, int NT_, int WR_, int WC_, int LEAD_>
struct F8F8Tile
{
    static constexpr int MT = MT_, NT = NT_, WR = WR_, WC = WC_, WAVES = WR * WC, LEAD = LEAD_, WIN = LEAD + 1;
    static constexpr int BM = WR * MT * 16, BN = WC * NT * 16, BK = 128, THREADS = WAVES * 64;
    static constexpr int A_TILE  = BM * BK, B_TILE = BN * BK;
    static constexpr int SLOT    = A_TILE + B_TILE <= 16384 ? 16384 : A_TILE + B_TILE <= 32768 ? 32768 : 65536; // (a power of two: slots change by an exclusive or)
    static constexpr int A_DMA   = BM / 16 / WAVES; // pieces per wave and half of A
    static constexpr int B_DMA   = BN / 8 / WAVES;
    static constexpr int S_ROWS  = BM * 16;       // four K tiles of row scales
    static constexpr int S_SLOT  = S_ROWS + 1024; // + one piece for the column blocks (lanes 0 .. BN / 32 - 1)
    static constexpr int S_OFF   = 2 * SLOT;
    static constexpr int S_DUMP  = S_OFF + 2 * S_SLOT;
    static constexpr int ST_PITCH = NT * 32 + 16;  // a wave's own 16-bit image of one row block
    static constexpr int ST_OFF   = S_DUMP + 1024;
    static constexpr int F_PITCH  = BN * 4 + 16;   // fp32 image of half the tile
    static constexpr int LDS_MAIN = ST_OFF + WAVES * 16 * ST_PITCH;
    static constexpr int LDS_BYTES = LDS_MAIN > BM / 2 * F_PITCH ? LDS_MAIN : BM / 2 * F_PITCH;
    static_assert(BM / 64 < WAVES, "one scale piece per 64 rows and one for the columns, a wave each");
    static_assert(MT % 2 == 0 && NT % 2 == 0 && MT % WIN == 0 && LEAD < MT / 2 + 1 && A_DMA * 16 * WAVES == BM && B_DMA * 8 * WAVES == BN, "whole pieces");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS");
};

// Epilogues with at most a bias per column and a FastGelu: every wave turns one row block at a time into whole lines through a
// piece of LDS of its own, so that neither the slots nor a barrier are needed and the next tile's loads run underneath.
// (N and ldc multiples of 8, C 16-byte aligned: whole 16-byte pieces; pieces past M or N fall out of the buffer resource.)
enum F8F8Out { F8F8_F16, F8F8_BF16_TRUNC, F8F8_BF16_RTN };

template <class T, F8F8Out OUTK>
__device__ __forceinline__ void f8f8_stream_rows(const f4_t (&acc)[T::NT][T::MT], uint8_t* st, const __amdgpu_buffer_rsrc_t& rsrc, uint32_t voff,
                                                 uint32_t row_bytes, int lane)
{
    constexpr int CH = T::NT * 2, RPI = 64 / CH; // 16-byte pieces of a row, rows per store instruction
    uint8_t* w       = st + (lane & 15) * T::ST_PITCH + (lane >> 4) * 8;
    const uint8_t* r = st + lane / CH * T::ST_PITCH + lane % CH * 16;
#pragma unroll
    for(int mt = 0; mt < T::MT; ++mt)
    {
#pragma unroll
        for(int nt = 0; nt < T::NT; ++nt)
        {
            f4_t v = acc[nt][mt];
            if constexpr(OUTK == F8F8_BF16_RTN)
                v = f4_t{convert_bf16_rtn_bits(v[0]), convert_bf16_rtn_bits(v[1]), convert_bf16_rtn_bits(v[2]), convert_bf16_rtn_bits(v[3])};
            *(u2_t*)(w + nt * 32) = pack_out4<OUTK != F8F8_F16>(v);
        }
        // (a wave's LDS operations are executed in order: no barrier between its own writes, reads and the next block's writes)
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for(int i = 0; i < 16 / RPI; ++i)
        {
            const u4_t v = *(const u4_t*)(r + i * RPI * T::ST_PITCH);
            __builtin_amdgcn_raw_buffer_store_b128(v, rsrc, voff, (uint32_t)(mt * 16 + i * RPI) * row_bytes, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <class T>
__device__ __forceinline__ void f8f8_epilogue_stream(const F8F8Params& p, f4_t (&acc)[T::NT][T::MT], uint8_t* lds, int m0, int n0, int wave,
                                                     int lane)
{
    constexpr int MT = T::MT, NT = T::NT;
    const int mw = m0 + wave / T::WC * (MT * 16), nw = n0 + wave % T::WC * (NT * 16);
    const int kind = p.epi.kind;
    if(kind == 6 || kind == 7)
    {
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
        {
            f4_t d;
#pragma unroll
            for(int j = 0; j < 4; ++j)
                d[j] = load_d_as_f32(p.epi.d0, min(nw + nt * 16 + (lane >> 4) * 4 + j, p.N - 1), p.epi.c_dtype);
#pragma unroll
            for(int mt = 0; mt < MT; ++mt)
                acc[nt][mt] = acc[nt][mt] + d;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if(kind == 1 || kind == 7)
    {
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
#pragma unroll
            for(int mt = 0; mt < MT; ++mt)
            {
                const f4_t v = acc[nt][mt];
                acc[nt][mt]  = f4_t{fast_gelu(v[0]), fast_gelu(v[1]), fast_gelu(v[2]), fast_gelu(v[3])};
                __builtin_amdgcn_sched_barrier(0);
            }
    }
    if(mw >= p.M || nw >= p.N)
        return;
    constexpr int CH = NT * 2;
    const uint32_t row_bytes = (uint32_t)p.ldc * 2;
    const long bytes         = ((long)(p.M - mw - 1) * p.ldc + (p.N - nw)) * 2;
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc((uint16_t*)p.c + (size_t)mw * (size_t)p.ldc + nw, 0, (int)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF), 0x00020000);
    const uint32_t voff = nw + lane % CH * 8 < p.N ? (uint32_t)(lane / CH) * row_bytes + lane % CH * 16 : 0x80000000u;
    uint8_t* st         = lds + T::ST_OFF + wave * (16 * T::ST_PITCH);
    if(p.epi.c_dtype != 1 /*WQ_BF16*/)
        f8f8_stream_rows<T, F8F8_F16>(acc, st, rsrc, voff, row_bytes, lane);
    else if(p.bf16_rtn || kind == 14)
        f8f8_stream_rows<T, F8F8_BF16_RTN>(acc, st, rsrc, voff, row_bytes, lane);
    else
        f8f8_stream_rows<T, F8F8_BF16_TRUNC>(acc, st, rsrc, voff, row_bytes, lane);
}

// Every epilogue, and fp32 slabs: half of every wave's rows at a time as fp32 through the slots, epilogue and edges in one rolled loop.
template <class T>
__device__ __forceinline__ void f8f8_epilogue_any(const F8F8Params& p, const f4_t (&acc)[T::NT][T::MT], uint8_t* lds, int m0, int n0, int z,
                                                  int wave, int lane)
{
    constexpr int MT = T::MT, NT = T::NT;
    const int fr = lane & 15, fq = lane >> 4, col = wave % T::WC * (NT * 16) + fq * 4, row = wave / T::WC * (MT * 8) + fr;
#pragma unroll
    for(int ph = 0; ph < 2; ++ph)
    {
        if(ph)
            __syncthreads();
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
#pragma unroll
            for(int mi = 0; mi < MT / 2; ++mi)
                *(f4_t*)(lds + (row + mi * 16) * T::F_PITCH + (col + nt * 16) * 4) = acc[nt][ph * (MT / 2) + mi];
        __syncthreads();
#pragma unroll 2
        for(int i = threadIdx.x; i < T::BM / 2 * (T::BN / 4); i += T::THREADS)
        {
            const int r = i / (T::BN / 4), n = (i % (T::BN / 4)) * 4;
            const int m = r / (MT * 8) * (MT * 16) + ph * (MT * 8) + r % (MT * 8);
            f8f8_store4(p, *(const f4_t*)(lds + r * T::F_PITCH + n * 4), m0 + m, n0 + n, z);
        }
    }
}

template <class F, int... I>
__device__ __forceinline__ void for_each_constant(F& f, std::integer_sequence<int, I...>)
{
    (f(std::integral_constant<int, I>{}), ...);
}

template <class T, bool TAIL, bool STREAM>
__device__ __forceinline__ void f8f8_tile_body(const F8F8Params& p)
{
    constexpr int MT = T::MT, NT = T::NT, MH = MT / 2, LEAD = T::LEAD, WIN = T::WIN;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave / T::WC, wc = wave % T::WC;
    const int fr = lane & 15, fq = lane >> 4;
    auto resource = [](const void* base, long bytes) __attribute__((always_inline)) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF), 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t null_rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)p.a, 0, 0, 0x00020000);
    constexpr uint32_t OUT = 0x80000000u; // an offset past every resource

    // A piece: 8 rows of 128 bytes, a row's 16-byte chunks permuted on the source side (f8_a_swz) so that the fragment reads are
    // free of bank conflicts (the kernel for few rows makes the same reads and counts none).  What the counters show here, 16 cycles
    // a wave and K tile beside 132 of LDS work, is two for each of the eight reads of a row block's scales, 16 bytes apart; 192 more
    // per wave go to the outputs' way through LDS.  Half h of A: row blocks h * MH .. of every wave row.
    const int chunk       = ((lane & 7) ^ f8_a_swz(lane >> 3)) << 4;
    const uint32_t a_lane = (uint32_t)(lane >> 3) * (uint32_t)p.lda + chunk;
    const uint32_t b_lane = (uint32_t)(lane >> 3) * (uint32_t)p.ldb + chunk;
    auto a_row = [&](int h, int i) __attribute__((always_inline)) {
        const int q = wave * T::A_DMA + i;
        return q / MT * (MT * 16) + h * (MT * 8) + q % MT * 8;
    };
    // Scale pieces: waves 0 .. BM / 64 - 1 fetch the scales of 64 rows each, the others all the same piece with the column
    // blocks' (one lane per 32 columns); four consecutive K tiles per lane, 16 bytes from a 4-byte aligned address.
    const bool s_is_row = wave < T::BM / 64;
    const int kblocks   = (p.K + T::BK - 1) / T::BK;

    // ---- the unit of work at hand: a tile, or a K slice of one ----
    const int tiles = p.tiles_m * p.tiles_n, units = tiles * p.slices;
    int m0, n0, z, ntiles, kt0, s_end;
    __amdgpu_buffer_rsrc_t a_rsrc, b_rsrc, s_rsrc;
    uint32_t a_run[2][T::A_DMA], b_run[T::B_DMA], s_lane;
    const float* s_table; // this lane's table row, and its place in LDS
    int s_at;
    bool past;
    auto set_unit = [&](int unit) __attribute__((always_inline)) {
        int tm, tn;
        z = unit / tiles;
        tile_coords(xcd_remap(unit - z * tiles, tiles), p.tiles_m, p.tiles_n, p.group_m, tm, tn);
        m0 = tm * T::BM, n0 = tn * T::BN;
        const int k0 = p.k_begin + z * p.k_per_z, k1 = min(p.k_end, k0 + p.k_per_z);
        ntiles = max(0, (k1 - k0 + T::BK - 1) / T::BK);
        kt0    = k0 / T::BK;
        s_end  = kblocks - kt0 - 4;
        past   = chunk >= k1 - k0 - (ntiles - 1) * T::BK; // this lane's chunk of the last K tile lies past its end
        // Resources start at the tile's first row / column (the distance from there fits 32 bits: lda, ldb <= 2^22 is checked
        // on the host) and end with the last byte of the last one: what lies past M or N reads as zeros.
        a_rsrc = resource(p.a + (size_t)m0 * (size_t)p.lda, (long)(p.M - m0 - 1) * p.lda + p.K);
        b_rsrc = resource(p.b + (size_t)n0 * (size_t)p.ldb, (long)(p.N - n0 - 1) * p.ldb + p.K);
#pragma unroll
        for(int i = 0; i < T::A_DMA; ++i)
#pragma unroll
            for(int h = 0; h < 2; ++h)
                a_run[h][i] = (uint32_t)a_row(h, i) * (uint32_t)p.lda + k0;
#pragma unroll
        for(int i = 0; i < T::B_DMA; ++i)
            b_run[i] = (uint32_t)((wave * T::B_DMA + i) * 8) * (uint32_t)p.ldb + k0;
        // (scale tables relative to the tile's first table row; rows past M repeat the last one, columns past N the last block)
        const int ra = m0 / p.bm, ra_last = (p.M - 1) / p.bm, rb = n0 / p.bn, rb_last = (p.N - 1) / p.bn;
        const __amdgpu_buffer_rsrc_t sa = resource(p.sa + (size_t)ra * (size_t)p.ld_sa, ((long)(ra_last - ra) * p.ld_sa + kblocks) * 4);
        const __amdgpu_buffer_rsrc_t sb = resource(p.sb + (size_t)rb * (size_t)p.ld_sb, ((long)(rb_last - rb) * p.ld_sb + kblocks) * 4);
        s_rsrc = s_is_row ? sa : sb;
        const int row = min(m0 + (s_is_row ? wave : 0) * 64 + lane, p.M - 1) / p.bm - ra;
        const int blk = min(n0 + lane * 32, p.N - 1) / p.bn - rb;
        s_lane = s_is_row ? (uint32_t)row * (uint32_t)p.ld_sa * 4u : lane < T::BN / 32 ? (uint32_t)blk * (uint32_t)p.ld_sb * 4u : OUT;
        // (the waves behind the row pieces all fetch the same piece: one of them writes by hand)
        s_table = s_is_row ? p.sa + (size_t)(ra + row) * (size_t)p.ld_sa : p.sb + (size_t)(rb + blk) * (size_t)p.ld_sb;
        s_at    = s_is_row ? T::S_OFF + (wave * 64 + lane) * 16 : wave == T::BM / 64 && lane < T::BN / 32 ? T::S_OFF + T::S_ROWS + lane * 16 : -1;
    };
    auto lds_at = [&](int at) __attribute__((always_inline)) { return (__attribute__((address_space(3))) void*)(lds + at); };
    auto dma_a = [&](const __amdgpu_buffer_rsrc_t& rsrc, int slot, int h, int i, bool last) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, lds_at(slot * T::SLOT + a_row(h, i) * 128), 16, TAIL && last && past ? OUT : a_lane,
                                                 a_run[h][i], 0, 0);
        a_run[h][i] += T::BK;
    };
    auto dma_b = [&](const __amdgpu_buffer_rsrc_t& rsrc, int slot, int i, bool last) __attribute__((always_inline)) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, lds_at(slot * T::SLOT + T::A_TILE + (wave * T::B_DMA + i) * 1024), 16,
                                                 TAIL && last && past ? OUT : b_lane, b_run[i], 0, 0);
        b_run[i] += T::BK;
    };
    // the four scales of tile `tile`'s group: from 4 (tile / 4), or the last four of the table row
    auto s_first = [&](int tile) __attribute__((always_inline)) { return min(tile & ~3, s_end); };
    // (not due: a piece of zeros into a place nobody reads, so that every tile issues the same number of pieces)
    auto dma_s = [&](int tile, bool due) __attribute__((always_inline)) {
        const int at = due ? T::S_OFF + ((tile >> 2) & 1) * T::S_SLOT + (s_is_row ? wave * 1024 : T::S_ROWS) : T::S_DUMP;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(due ? s_rsrc : null_rsrc, lds_at(at), 16, s_lane, (uint32_t)(kt0 + s_first(tile)) * 4u, 0, 0);
    };

    // This lane's two 16-byte chunks of row fr of a 16-row block (swizzled position inside the 128-byte row): LDS addresses of the
    // wave's first row block and first column block, in the slot that is read next (they change slots by an exclusive or).
    const int f_lo = fr * 128 + (((2 * fq) ^ f8_a_swz(fr)) << 4), f_hi = fr * 128 + (((2 * fq + 1) ^ f8_a_swz(fr)) << 4);
    static_assert((T::SLOT & (T::SLOT - 1)) == 0 && T::A_TILE + T::B_TILE <= T::SLOT, "slots change by an exclusive or");
    uint32_t a_lo, a_hi, b_lo, b_hi;
    i8v_t af[WIN], bf[NT]; // fragments of row blocks mt .. mt + LEAD; weights of the tile
    auto read_frag = [&](uint32_t lo, uint32_t hi, int block) __attribute__((always_inline)) {
        return f8f8_frag(*(const u4_t*)(lds + lo + block * 2048), *(const u4_t*)(lds + hi + block * 2048));
    };
    // pieces [first, last) of a tile's group 0 (scales, first half of A, B) and group 1 (second half of A)
    auto group0 = [&](int tile, bool s_due, int slot, int first, int last) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t ra = tile < ntiles ? a_rsrc : null_rsrc, rb = tile < ntiles ? b_rsrc : null_rsrc;
#pragma unroll
        for(int i = first; i < last; ++i)
            if(i == 0)
                dma_s(tile, s_due && tile < ntiles);
            else if(i <= T::A_DMA)
                dma_a(ra, slot, 0, i - 1, tile == ntiles - 1);
            else
                dma_b(rb, slot, i - 1 - T::A_DMA, tile == ntiles - 1);
    };
    auto group1 = [&](int tile, int slot, int first, int last) __attribute__((always_inline)) {
        const __amdgpu_buffer_rsrc_t ra = tile < ntiles ? a_rsrc : null_rsrc;
#pragma unroll
        for(int i = first; i < last; ++i)
            dma_a(ra, slot, 1, i, tile == ntiles - 1);
    };
    constexpr int G0 = 1 + T::A_DMA + T::B_DMA, G1 = T::A_DMA;

    auto prologue = [&]() __attribute__((always_inline)) {
        const bool wide = kblocks >= 4;
        if(!wide && s_at >= 0)
            for(int i = 0; i < kblocks; ++i)
                *(float*)(lds + s_at + (4 - kblocks + i) * 4) = s_table[i];
        __builtin_amdgcn_sched_barrier(0); // (issue order is part of the vmcnt arithmetic)
        group0(0, wide, 0, 0, G0);
        __builtin_amdgcn_sched_barrier(0);
        group1(0, 0, 0, G1);
        __builtin_amdgcn_sched_barrier(0);
        group0(1, false, 1, 0, G0);
        __builtin_amdgcn_sched_barrier(0);
        group1(1, 1, 0, G1);
        __builtin_amdgcn_sched_barrier(0);
    };

    f4_t acc[NT][MT];
    f4_t pend[NT];        // block sums not yet folded in: of the previous row block
    float s_fold[NT / 2]; // and their factors, per 32 columns
    int t;
    auto tile_body = [&]() __attribute__((always_inline)) {
        const int slot    = t & 1;
        const uint8_t* sp = lds + T::S_OFF + ((t >> 2) & 1) * T::S_SLOT + (t - s_first(t)) * 4;
        const float* row_s = (const float*)(sp + (wr * MT * 16 + fr) * 16); // row 16 mt + fr at [64 mt]
        float sb[NT / 2];
#pragma unroll
        for(int h = 0; h < NT / 2; ++h)
            sb[h] = *(const float*)(sp + T::S_ROWS + (wc * (NT / 2) + h) * 16) * p.fnuz;
        float s_row = row_s[0];

        auto row_block = [&](auto mt_c) __attribute__((always_inline)) {
            constexpr int mt = decltype(mt_c)::value, prev = (mt + MT - 1) % MT;
            if constexpr(mt == MH - LEAD || mt == MT - LEAD)
            {
                wait_vmcnt<G0 + G1>();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr(mt == MT - LEAD)
                a_lo ^= T::SLOT, a_hi ^= T::SLOT; // (from here on the next tile's)
            af[(mt + LEAD) % WIN] = read_frag(a_lo, a_hi, (mt + LEAD) % MT);
            float s_now[NT / 2];
#pragma unroll
            for(int h = 0; h < NT / 2; ++h)
                s_now[h] = s_row * sb[h];
            if constexpr(mt + 1 < MT)
                s_row = row_s[64 * (mt + 1)];
            // (a piece or two per row block: issued at once they hold the wave up behind everybody else's)
            if constexpr(mt >= MH - LEAD && mt < MT - LEAD)
            {
                constexpr int PER = (G0 + MH - 1) / MH, i = (mt - (MH - LEAD)) * PER;
                group0(t + 2, (t & 3) == 2, slot, i, i + PER < G0 ? i + PER : G0); // (scale slot: of tiles t - 6 .. t - 3)
            }
            if constexpr(mt >= MT - LEAD)
            {
                constexpr int PER = (G1 + LEAD - 1) / LEAD, i = (mt - (MT - LEAD)) * PER;
                group1(t + 2, slot, i, i + PER < G1 ? i + PER : G1);
            }
            const f4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for(int nt = 0; nt < NT; ++nt)
            {
                const float f  = s_fold[nt / 2];
                acc[nt][prev] = __builtin_elementwise_fma(pend[nt], f4_t{f, f, f, f}, acc[nt][prev]);
                pend[nt]      = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[nt], af[mt % WIN], zero, 0, 0, 0, 0, 0, 0);
                if constexpr(mt == MT - 1)
                    bf[nt] = read_frag(b_lo, b_hi, nt);
            }
#pragma unroll
            for(int h = 0; h < NT / 2; ++h)
                s_fold[h] = s_now[h];
            // order: a fold and an MFMA in turn, the fragment reads behind the first MFMA (as early as they can hide behind one)
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, mt == MT - 1 ? 5 : 3, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
#pragma unroll
            for(int nt = 1; nt < NT; ++nt)
            {
                __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if constexpr(mt == MT - 1)
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        for_each_constant(row_block, std::make_integer_sequence<int, MT>{});
        b_lo ^= T::SLOT, b_hi ^= T::SLOT;
    };
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
        {
            pend[nt] = f4_t{0.f, 0.f, 0.f, 0.f}, s_fold[nt / 2] = 0.f;
#pragma unroll
            for(int mt = 0; mt < MT; ++mt)
                acc[nt][mt] = f4_t{0.f, 0.f, 0.f, 0.f};
        }
    };
    // the K loop of the unit whose first loads are in flight (ntiles > 0); every wave is done with the slots at its end
    auto multiply = [&]() __attribute__((always_inline)) {
        wait_vmcnt<G0 + 2 * G1>(); // group (0, 0) done (the stores of the tile before are younger: they only add to the wait)
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // (scales copied by hand)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        a_lo = f_lo + wr * (MT * 2048), a_hi = f_hi + wr * (MT * 2048);
        b_lo = f_lo + T::A_TILE + wc * (NT * 2048), b_hi = f_hi + T::A_TILE + wc * (NT * 2048);
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
            bf[nt] = read_frag(b_lo, b_hi, nt);
#pragma unroll
        for(int i = 0; i < LEAD; ++i)
            af[i] = read_frag(a_lo, a_hi, i);
        b_lo ^= T::SLOT, b_hi ^= T::SLOT;
        __builtin_amdgcn_sched_barrier(0);
        t = 0;
        do
            tile_body();
        while(++t < ntiles);
#pragma unroll
        for(int nt = 0; nt < NT; ++nt)
        {
            const float f   = s_fold[nt / 2];
            acc[nt][MT - 1] = __builtin_elementwise_fma(pend[nt], f4_t{f, f, f, f}, acc[nt][MT - 1]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    };

    int unit = blockIdx.x;
    set_unit(unit);
    if constexpr(STREAM)
    {
        prologue();
        for(;;)
        {
            clear();
            multiply();
            const int m = m0, n = n0;
            unit += gridDim.x;
            if(unit < units)
            {
                set_unit(unit);
                prologue(); // (the next tile's first loads fly while this one leaves)
            }
            f8f8_epilogue_stream<T>(p, acc, lds, m, n, wave, lane);
            if(unit >= units)
                break;
        }
        wait_vmcnt<0>();
    }
    else
    {
        clear();
        if(ntiles > 0)
        {
            prologue();
            multiply();
            wait_vmcnt<0>(); // (null-resource pieces of tiles past the end write zeros into the slots)
            __syncthreads();
        }
        f8f8_epilogue_any<T>(p, acc, lds, m0, n0, z, wave, lane);
    }
}

// The smaller tiles are for grids that leave the chip empty: what a K tile costs is then the time from one barrier to the next, not
// its bytes or MFMAs (a ring of four K tiles instead of two: 128 x 128 0.75 us a K tile against 0.62), and it shrinks with the tile:
// 256 x 256 1.6 us, 128 x 256 0.98, 128 x 128 with eight waves 0.6, with four 0.55, 64 x 128 0.37, 64 x 64 0.3.  Eight waves on
// 128 x 128 hide each other's waits where there is one workgroup per CU (777 x 4096 x 4096: 23.5 us against 24.8), two workgroups of
// four waves do it better where there are two (512 x 11008 x 4096: 36.6 against 43.5).
using F8F8Tile256 = F8F8Tile<8, 4, 2, 4, 3>;
using F8F8Tile128 = F8F8Tile<4, 4, 2, 2, 1>;
using F8F8Tile128W8 = F8F8Tile<4, 2, 2, 4, 1>;
using F8F8Tile64 = F8F8Tile<2, 4, 2, 2, 1>;
using F8F8Tile64x64 = F8F8Tile<2, 2, 2, 2, 1>;
using F8F8Tile128x256 = F8F8Tile<4, 4, 2, 4, 1>;
template <bool TAIL, bool STREAM>
__global__ __launch_bounds__(512, 2) void wq_gemm_f8f8_256(const F8F8Params p) { f8f8_tile_body<F8F8Tile256, TAIL, STREAM>(p); }
template <bool TAIL, bool STREAM>
__global__ __launch_bounds__(512, 2) void wq_gemm_f8f8_128x256(const F8F8Params p) { f8f8_tile_body<F8F8Tile128x256, TAIL, STREAM>(p); }
template <bool TAIL, bool STREAM>
__global__ __launch_bounds__(256, 2) void wq_gemm_f8f8_128(const F8F8Params p) { f8f8_tile_body<F8F8Tile128, TAIL, STREAM>(p); }

template <bool TAIL, bool STREAM>
__global__ __launch_bounds__(512, 2) void wq_gemm_f8f8_128_w8(const F8F8Params p) { f8f8_tile_body<F8F8Tile128W8, TAIL, STREAM>(p); }
template <bool TAIL, bool STREAM>
__global__ __launch_bounds__(256, 3) void wq_gemm_f8f8_64x64(const F8F8Params p) { f8f8_tile_body<F8F8Tile64x64, TAIL, STREAM>(p); }
template <bool TAIL, bool STREAM>
__global__ __launch_bounds__(256, 2) void wq_gemm_f8f8_64(const F8F8Params p) { f8f8_tile_body<F8F8Tile64, TAIL, STREAM>(p); }

// ---------------------------------------------------------------------------------------------
// Few rows (M <= 16 MT): one pass over the weights, bound by their stream.  A workgroup owns 16 NB columns; its waves deal the K
// tiles among themselves (tile i WAVES + wave: the workgroup reads runs of WAVES cache lines of every column) and add their sums
// through LDS at the end, in the order of the waves: no second kernel, no workspace.  Workgroups start at different K tiles: all of
// them at the same k of columns a power of two apart ask few of the memory's channels at a time (8192 x 8192 at M = 16 with 32
// columns a workgroup 20.7 us, turned 14.8; 4096 x 11008 15.5 and 13.5).  Rows past M and columns past N lie outside the resources and
// read as zeros without memory accesses, and so does what lies past the end of the last K tile (K a multiple of 16).  Two forms:
//   * _direct: operands straight to the registers of the MFMA, P tiles at a time.  The vector cache takes such fragment-shaped
//     loads at one access of 16 bytes per lane: 16 bytes a cycle and CU, 8.6 TB/s on the chip, more than HBM delivers, but
//     activations of 16 rows double the accesses.  Least latency: 4096 x 4096 at M = 1 6.5 us (6.9 through LDS), 28672 x 8192
//     38.3 us = 6.1 TB/s (43.1).  Turned only where a workgroup has a CU of its own (4096 x 11008 14.0 -> 11.8; 28672 x 8192
//     would be 39.8);
//   * through LDS: LDS-DMA takes 64 bytes an access; every wave fills a ring of its own, D tiles ahead, so there is no barrier in
//     the loop.  At M = 16: 4096 x 4096 7.8 us (direct 8.4); 28672 x 8192, 64 columns a workgroup, 44.5 (68.7).
// (Weights not in the last-level cache: several copies in turn.)
// ---------------------------------------------------------------------------------------------
constexpr unsigned kF8F8Turn = 11; // (3, 5, 13 and 21 within 3 % of it)

template <int WAVES, int P>
__global__ __launch_bounds__(WAVES * 64) void wq_gemm_f8f8_skinny_direct(const F8F8Params p)
{
    __shared__ __attribute__((aligned(16))) f4_t sums[WAVES][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 15, fq = lane >> 4;
    const int n0 = blockIdx.x * 16, z = blockIdx.y;
    const int k0 = p.k_begin + z * p.k_per_z, k1 = min(p.k_end, k0 + p.k_per_z);
    const int ntiles = (k1 - k0 + 127) >> 7; // (empty slices: <= 0)
    const F8F8Walk walk(ntiles, gridDim.x <= 256 ? blockIdx.x * kF8F8Turn : 0);
    constexpr uint32_t OUT = 0x80000000u;

    const long a_bytes = (long)(p.M - 1) * p.lda + p.K, b_bytes = (long)(p.N - n0 - 1) * p.ldb + p.K;
    const __amdgpu_buffer_rsrc_t a_rsrc =
        __builtin_amdgcn_make_buffer_rsrc((void*)p.a, 0, (int)(a_bytes < 0x7FFFFFFF ? a_bytes : 0x7FFFFFFF), 0x00020000);
    const __amdgpu_buffer_rsrc_t b_rsrc =
        __builtin_amdgcn_make_buffer_rsrc((void*)(p.b + (size_t)n0 * (size_t)p.ldb), 0, (int)(b_bytes < 0x7FFFFFFF ? b_bytes : 0x7FFFFFFF), 0x00020000);
    const uint32_t a_lane = (uint32_t)fr * (uint32_t)p.lda + fq * 32, b_lane = (uint32_t)fr * (uint32_t)p.ldb + fq * 32;
    const int k_last      = k1 - k0 - (ntiles - 1) * 128;
    const uint32_t bad_lo = fq * 32 < k_last ? 0u : OUT, bad_hi = fq * 32 + 16 < k_last ? 0u : OUT;
    const int kt0   = k0 >> 7;
    const float* sa = p.sa + (size_t)(min(fr, p.M - 1) / p.bm) * (size_t)p.ld_sa + kt0; // (rows past M repeat the last one: their results are not stored)
    const float* sb = p.sb + (size_t)(n0 / p.bn) * (size_t)p.ld_sb + kt0;

    f4_t acc  = {0.f, 0.f, 0.f, 0.f};
    auto load = [&](const __amdgpu_buffer_rsrc_t& rsrc, uint32_t off, int tile) __attribute__((always_inline)) {
        const bool last     = tile == ntiles - 1;
        const uint32_t soff = k0 + tile * 128;
        const u4_t lo = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, last ? off | bad_lo : off, soff, 0));
        const u4_t hi = __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(rsrc, last ? off | bad_hi : off, soff + 16, 0));
        return f8f8_frag(lo, hi);
    };
    auto step = [&](int first, int tiles) __attribute__((always_inline)) {
        i8v_t w[P], a[P];
        float ra[P];
#pragma unroll
        for(int i = 0; i < P; ++i)
            if(i < tiles)
            {
                const int tile = walk.tile(first + i * WAVES);
                w[i]  = load(b_rsrc, b_lane, tile);
                a[i]  = load(a_rsrc, a_lane, tile);
                ra[i] = sa[tile];
            }
#pragma unroll
        for(int i = 0; i < P; ++i)
            if(i < tiles)
            {
                const float cs  = sb[walk.tile(first + i * WAVES)] * p.fnuz, s = ra[i] * cs;
                const f4_t zero = {0.f, 0.f, 0.f, 0.f};
                const f4_t sum  = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i], a[i], zero, 0, 0, 0, 0, 0, 0);
                acc             = __builtin_elementwise_fma(sum, f4_t{s, s, s, s}, acc);
            }
    };
    int tile = wave;
    for(; tile + (P - 1) * WAVES < ntiles; tile += P * WAVES)
        step(tile, P);
    for(; tile < ntiles; tile += WAVES)
        step(tile, 1);

    sums[wave][lane] = acc;
    __syncthreads();
    if(wave == 0)
    {
        f4_t v = sums[0][lane];
#pragma unroll
        for(int w = 1; w < WAVES; ++w)
            v += sums[w][lane];
        f8f8_store4(p, v, fr, n0 + fq * 4, z);
    }
}

// One wave's ring: D tiles of 16 NB columns' weights and 16 MT rows of activations, in LDS-DMA pieces of 8 rows.  OPS: what a tile
// adds to vmcnt, its pieces and its row scales.
template <int MT, int NB, int WAVES, int D>
struct F8F8Skinny
{
    static constexpr int THREADS = WAVES * 64, SLOT = (NB + MT) * 2048, LDS_BYTES = WAVES * D * SLOT, OPS = 2 * (NB + MT) + MT;
    static_assert(LDS_BYTES >= WAVES * MT * NB * 1024 && LDS_BYTES <= 160 * 1024, "the sums reuse the ring");
};

template <int MT, int NB, int WAVES, int D>
__global__ __launch_bounds__(WAVES * 64) void wq_gemm_f8f8_skinny(const F8F8Params p)
{
    using T = F8F8Skinny<MT, NB, WAVES, D>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fr = lane & 15, fq = lane >> 4;
    const int n0 = blockIdx.x * (NB * 16), z = blockIdx.y;
    const int k0 = p.k_begin + z * p.k_per_z, k1 = min(p.k_end, k0 + p.k_per_z);
    const int ntiles = (k1 - k0 + 127) >> 7; // (empty slices: <= 0)
    const int mine   = ntiles > wave ? (ntiles - wave + WAVES - 1) / WAVES : 0;
    const F8F8Walk walk(ntiles, blockIdx.x * kF8F8Turn);
    constexpr uint32_t OUT = 0x80000000u;

    auto resource = [](const void* base, long bytes) __attribute__((always_inline)) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF), 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t a_rsrc    = resource(p.a, (long)(p.M - 1) * p.lda + p.K);
    const __amdgpu_buffer_rsrc_t b_rsrc    = resource(p.b + (size_t)n0 * (size_t)p.ldb, (long)(p.N - n0 - 1) * p.ldb + p.K);
    const __amdgpu_buffer_rsrc_t null_rsrc = resource(p.a, 0);
    const int chunk       = ((lane & 7) ^ f8_a_swz(lane >> 3)) << 4;
    const uint32_t a_lane = (uint32_t)(lane >> 3) * (uint32_t)p.lda + chunk, b_lane = (uint32_t)(lane >> 3) * (uint32_t)p.ldb + chunk;
    const bool past       = chunk >= k1 - k0 - (ntiles - 1) * 128;
    const int kt0 = k0 >> 7;
    const float* sa[MT]; // (rows past M repeat the last one: their results are not stored)
    const float* sb[NB];
#pragma unroll
    for(int mt = 0; mt < MT; ++mt)
        sa[mt] = p.sa + (size_t)(min(mt * 16 + fr, p.M - 1) / p.bm) * (size_t)p.ld_sa + kt0;
#pragma unroll
    for(int nb = 0; nb < NB; ++nb)
        sb[nb] = p.sb + (size_t)(min(n0 + nb * 16, p.N - 1) / p.bn) * (size_t)p.ld_sb + kt0;

    f4_t acc[MT][NB];
#pragma unroll
    for(int mt = 0; mt < MT; ++mt)
#pragma unroll
        for(int nb = 0; nb < NB; ++nb)
            acc[mt][nb] = f4_t{0.f, 0.f, 0.f, 0.f};
    float ra[D][MT];
    uint8_t* ring = lds + wave * (D * T::SLOT);
    // (tiles past the wave's last one: scales of its last, pieces of zeros without a memory access)
    auto fetch = [&](int i, int j) __attribute__((always_inline)) {
        const int step = wave + j * WAVES, tile = walk.tile(step), known = walk.scales(step);
#pragma unroll
        for(int mt = 0; mt < MT; ++mt)
            ra[i][mt] = sa[mt][known];
        __builtin_amdgcn_sched_barrier(0); // (issue order is part of the vmcnt arithmetic)
        const bool last = tile == ntiles - 1, there = step < ntiles;
        const __amdgpu_buffer_rsrc_t wr = there ? b_rsrc : null_rsrc, ar = there ? a_rsrc : null_rsrc;
        const uint32_t w_off = last && past ? OUT : b_lane, x_off = last && past ? OUT : a_lane, soff = (uint32_t)(k0 + tile * 128);
#pragma unroll
        for(int h = 0; h < 2 * NB; ++h)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (__attribute__((address_space(3))) void*)(ring + i * T::SLOT + h * 1024), 16, w_off,
                                                     soff + (uint32_t)(h * 8) * (uint32_t)p.ldb, 0, 0);
#pragma unroll
        for(int h = 0; h < 2 * MT; ++h)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ar, (__attribute__((address_space(3))) void*)(ring + i * T::SLOT + (2 * NB + h) * 1024), 16,
                                                     x_off, soff + (uint32_t)(h * 8) * (uint32_t)p.lda, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    const int f_lo = fr * 128 + (((2 * fq) ^ f8_a_swz(fr)) << 4), f_hi = fr * 128 + (((2 * fq + 1) ^ f8_a_swz(fr)) << 4);

    if(!walk.empty())
#pragma unroll
        for(int i = 0; i < D; ++i)
            fetch(i, i);
    for(int j = 0; j < mine; j += D)
    {
#pragma unroll
        for(int i = 0; i < D; ++i)
            if(j + i < mine)
            {
                const int tile = walk.tile(wave + (j + i) * WAVES);
                wait_vmcnt<(D - 1) * T::OPS>();
                __builtin_amdgcn_sched_barrier(0);
                i8v_t w[NB], a[MT];
                float s[MT];
                const uint8_t* st = ring + i * T::SLOT;
#pragma unroll
                for(int nb = 0; nb < NB; ++nb)
                    w[nb] = f8f8_frag(*(const u4_t*)(st + nb * 2048 + f_lo), *(const u4_t*)(st + nb * 2048 + f_hi));
#pragma unroll
                for(int mt = 0; mt < MT; ++mt)
                {
                    a[mt] = f8f8_frag(*(const u4_t*)(st + (NB + mt) * 2048 + f_lo), *(const u4_t*)(st + (NB + mt) * 2048 + f_hi));
                    s[mt] = ra[i][mt];
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // read: the slot may be filled again
                __builtin_amdgcn_sched_barrier(0);
                fetch(i, j + i + D);
#pragma unroll
                for(int nb = 0; nb < NB; ++nb)
                {
                    const float cs = sb[nb][tile] * p.fnuz;
#pragma unroll
                    for(int mt = 0; mt < MT; ++mt)
                    {
                        const float f   = s[mt] * cs;
                        const f4_t zero = {0.f, 0.f, 0.f, 0.f};
                        const f4_t sum  = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[nb], a[mt], zero, 0, 0, 0, 0, 0, 0);
                        acc[mt][nb]     = __builtin_elementwise_fma(sum, f4_t{f, f, f, f}, acc[mt][nb]);
                    }
                }
            }
    }
    wait_vmcnt<0>(); // (pieces of zeros still write)
    __syncthreads();
    f4_t* sums = (f4_t*)lds;
#pragma unroll
    for(int mt = 0; mt < MT; ++mt)
#pragma unroll
        for(int nb = 0; nb < NB; ++nb)
            sums[(wave * (MT * NB) + mt * NB + nb) * 64 + lane] = acc[mt][nb];
    __syncthreads();
    for(int u = threadIdx.x; u < MT * NB * 64; u += WAVES * 64)
    {
        const int block = u >> 6, l = u & 63;
        f4_t v = sums[u];
#pragma unroll
        for(int w = 1; w < WAVES; ++w)
            v += sums[w * (MT * NB * 64) + u];
        f8f8_store4(p, v, block / NB * 16 + (l & 15), n0 + block % NB * 16 + (l >> 4) * 4, z);
    }
}

// Rows of both operands, of any alignment, to rows of whole 16-byte pieces, zeros behind their last byte; a wave per row.
__global__ __launch_bounds__(256) void wq_pad_rows_f8(const uint8_t* __restrict__ a, long lda, int M, const uint8_t* __restrict__ b, long ldb, int N, int K,
                                                      uint8_t* __restrict__ rows)
{
    const int pieces = (K + 15) >> 4;
    for(long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < (long)M + N; row += (long)gridDim.x * 4)
    {
        const uint8_t* src = row < M ? a + row * lda : b + (row - M) * ldb;
        for(int i = threadIdx.x & 63; i < pieces; i += 64)
            *(u4_t*)(rows + (row * pieces + i) * 16) = f8f8_load16(src, i * 16, K);
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
        f8f8_store4(p, s, m, n, 0);
    }
}

} // namespace wq
