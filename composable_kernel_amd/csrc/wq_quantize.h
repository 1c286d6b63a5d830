// Quantisation of 16-bit rows to e4m3fn with fp32 scales (gfx950), plain or behind a function that is fused into the
// same pass: the gated activation act(gate) * up, or the root-mean-square norm of x (+ residual).
//
//   y[m, k]  = x                                              WQ_QUANT_ROWS
//            = act(x) * x2                                    WQ_QUANT_GATED
//            = h / sqrt(mean_k(h^2) + eps) * weight[k]        WQ_QUANT_RMSNORM, h = x (+ x2), residual_out = h
//   scale[m, g] = max(max_{k in group g} |y|, 1e-12) / 448,   q[m, k] = e4m3(y / scale[m, g])
//
// All of it in fp32 from the 16-bit operands; h, y and the sums are never rounded to 16 bits on the way (only
// residual_out is, once, to nearest even).  The largest magnitude is found on the bits of |y| as unsigned integers, an
// order in which a NaN is larger than every number: a group with a NaN gets a NaN scale and NaN bytes, and so poisons
// the products that read it instead of vanishing in a maximum.
//
// The traffic is the bound (one read of each operand, one write of each result), so every operand passes through
// registers exactly once: a lane owns 8 consecutive elements (one 16-byte load, one 8-byte store of q), 16 lanes own a
// group of 128 and exchange their maximum with DPP moves inside the row of 16.  Loads and stores carry no alignment
// assumption (gfx950 handles unaligned vector accesses), so that odd widths and odd row pitches take the same path; only
// the lane that holds a row's last K % 8 elements goes element by element.
#pragma once

#include <type_traits>

#include "wq_device.h"

namespace wq {

struct QuantParams
{
    const void* x;
    const void* x2; // residual or up operand, may be null for the norm
    const void* weight;
    uint8_t* q;
    float* scale;
    void* residual_out;
    int M, K;
    long ldx, ldx2, ld_res, ldq, ld_scale;
    int weight_f32; // weight holds floats instead of x's 16-bit type
    int act;        // wq_activation
    float eps;
};

constexpr float kF8Max     = 448.f;  // largest finite e4m3fn
constexpr float kAmaxFloor = 1e-12f; // keeps 448 / amax finite for groups of zeros

// 8 consecutive 16-bit values; elements at and past `valid` read as zero
template <bool BF16>
__device__ __forceinline__ u4_t quant_load16(const void* base, long at, int valid)
{
    const uint16_t* p = (const uint16_t*)base + at;
    u4_t v            = {0, 0, 0, 0};
    if(valid >= 8)
        __builtin_memcpy(&v, p, 16);
    else
    {
#pragma unroll
        for(int j = 0; j < 8; ++j)
            if(j < valid)
                v[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
    }
    return v;
}

template <bool BF16>
__device__ __forceinline__ void widen8(u4_t b, float (&v)[8])
{
#pragma unroll
    for(int j = 0; j < 8; ++j)
    {
        const uint16_t h = (uint16_t)(b[j >> 1] >> (16 * (j & 1)));
        v[j]             = BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
    }
}

template <bool BF16>
__device__ __forceinline__ void quant_load8(const void* base, long at, int valid, float (&v)[8])
{
    widen8<BF16>(quant_load16<BF16>(base, at, valid), v);
}

__device__ __forceinline__ void quant_load8_f32(const float* p, int valid, float (&v)[8])
{
    if(valid >= 8)
        __builtin_memcpy(v, p, 32);
    else
    {
#pragma unroll
        for(int j = 0; j < 8; ++j)
            v[j] = j < valid ? p[j] : 0.f;
    }
}

template <bool BF16>
__device__ __forceinline__ void quant_store8_16(void* base, long at, int valid, const float (&v)[8])
{
    uint16_t* p = (uint16_t*)base + at;
    uint16_t b[8];
#pragma unroll
    for(int j = 0; j < 8; ++j)
        b[j] = BF16 ? (uint16_t)(__builtin_bit_cast(uint32_t, convert_bf16_rtn_bits(v[j])) >> 16) : __builtin_bit_cast(uint16_t, (_Float16)v[j]);
    if(valid >= 8)
        __builtin_memcpy(p, b, 16);
    else
    {
#pragma unroll
        for(int j = 0; j < 8; ++j)
            if(j < valid)
                p[j] = b[j];
    }
}

// 8 values, already divided by their scale, to e4m3fn (the gfx950 conversion rounds to nearest even; |v| <= 448 up to
// rounding, which stays below the 464 where the format would overflow)
__device__ __forceinline__ void quant_store8_f8(uint8_t* p, int valid, const float (&v)[8])
{
    uint32_t w[2];
#pragma unroll
    for(int h = 0; h < 2; ++h)
    {
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
        w[h]  = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], t, true);
    }
    if(valid >= 8)
        __builtin_memcpy(p, w, 8);
    else
    {
#pragma unroll
        for(int j = 0; j < 8; ++j)
            if(j < valid)
                p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

__device__ __forceinline__ uint32_t amax8(const float (&v)[8])
{
    uint32_t m = abs_bits(v[0]);
#pragma unroll
    for(int j = 1; j < 8; ++j)
        m = max(m, abs_bits(v[j]));
    return m;
}

// maximum over the 16 lanes of a DPP row, in all of them: quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror
__device__ __forceinline__ uint32_t row16_max(uint32_t m)
{
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, true));
    return m;
}

// Scale of a group from the bits of its largest magnitude, and what the quotients are made with: the reciprocal, and the scale
// again for the correction (0 if it is infinite: the finite values of such a group become 0, not NaN).
struct GroupScale
{
    float s, inv, fix;
    __device__ __forceinline__ explicit GroupScale(uint32_t bits)
    {
        float a = __builtin_bit_cast(float, bits);
        a       = a < kAmaxFloor ? kAmaxFloor : a; // (a NaN passes through)
        s       = a / kF8Max;
        inv     = 1.f / s;
        fix     = __builtin_isinf(s) ? 0.f : s;
    }
    // y / s as a division gives it: the product with the reciprocal, corrected by what it leaves over.  (The product alone rounds
    // exact ties of the 8-bit format, frequent with 16-bit inputs, either way.)
    __device__ __forceinline__ float quotient(float y) const
    {
        const float q = y * inv;
        return __builtin_fmaf(__builtin_fmaf(-q, fix, y), inv, q);
    }
};

__device__ __forceinline__ float silu(float g) { return g * __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

template <bool BF16>
__device__ __forceinline__ void gated8(const QuantParams& p, long row, int k, int valid, float (&y)[8])
{
    float g[8], u[8];
    quant_load8<BF16>(p.x, row * p.ldx + k, valid, g);
    quant_load8<BF16>(p.x2, row * p.ldx2 + k, valid, u);
#pragma unroll
    for(int j = 0; j < 8; ++j)
        y[j] = (p.act == 1 /*WQ_ACT_FASTGELU*/ ? fast_gelu(g[j]) : silu(g[j])) * u[j];
}

// ---------------------------------------------------------------------------------------------
// Groups of 128, no statistic over the row: every wave takes 512 consecutive elements (four groups) of a row at a time.
// ---------------------------------------------------------------------------------------------
template <int OP, bool BF16>
__global__ __launch_bounds__(256) void wq_quantize_groups(const QuantParams p, int chunks)
{
    const int lane   = threadIdx.x & 63;
    const long total = (long)p.M * chunks;
    const long wave  = (long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for(long t = wave; t < total; t += (long)gridDim.x * 4)
    {
        const long row  = t / chunks;
        const int k     = (int)(t - row * chunks) * 512 + lane * 8;
        const int valid = min(p.K - k, 8);
        float y[8];
        if constexpr(OP == 2)
            gated8<BF16>(p, row, k, valid, y);
        else
            quant_load8<BF16>(p.x, row * p.ldx + k, valid, y);
        const GroupScale g(row16_max(amax8(y)));
#pragma unroll
        for(int j = 0; j < 8; ++j)
            y[j] = g.quotient(y[j]);
        quant_store8_f8(p.q + row * p.ldq + k, valid, y);
        if((lane & 15) == 0 && valid > 0)
            p.scale[row * p.ld_scale + (k >> 7)] = g.s;
    }
}

// ---------------------------------------------------------------------------------------------
// One workgroup per row: the norm, and one scale per row.  R 8-element pieces per thread stay in registers between the
// statistics and the conversion (R = 0: any width, the operands are read again).
// ---------------------------------------------------------------------------------------------
// Sums over the wave: of a in the lanes of its lower half, of b in those of its upper half.  Halves, rows of 16, then inside a row
// lanes 8, 4, 2, 1 apart (row_ror: once both halves of a row are equal, a rotation by 4 is an exchange of lanes 4 apart, and so on).
// The exchange of the halves brings both sums into one register; six exchanges through LDS for each sum made the norm of
// 4096 x 8192 2 % longer, two sums one beside the other that of 777 x 5000 per token (6.7 us).
__device__ __forceinline__ float wave_sums(float a, float b)
{
    const auto add = [](auto two) __attribute__((always_inline)) {
        return __builtin_bit_cast(float, (uint32_t)two[0]) + __builtin_bit_cast(float, (uint32_t)two[1]);
    };
    const auto ror = [](float x, auto dpp) __attribute__((always_inline)) {
        return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(dpp)::value, 0xF, 0xF, true));
    };
    float v = add(__builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false));
    v       = add(__builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false));
    v = ror(v, std::integral_constant<int, 0x128>{});
    v = ror(v, std::integral_constant<int, 0x124>{});
    v = ror(v, std::integral_constant<int, 0x122>{});
    return ror(v, std::integral_constant<int, 0x121>{});
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = row16_max(v);
    v = max(v, (uint32_t)__shfl_xor((int)v, 16));
    return max(v, (uint32_t)__shfl_xor((int)v, 32));
}

template <int OP, bool BF16>
__device__ __forceinline__ void row_value8(const QuantParams& p, long row, int k, int valid, float (&y)[8])
{
    if constexpr(OP == 2)
        gated8<BF16>(p, row, k, valid, y);
    else
    {
        quant_load8<BF16>(p.x, row * p.ldx + k, valid, y);
        if constexpr(OP == 1)
            if(p.x2)
            {
                float r[8];
                quant_load8<BF16>(p.x2, row * p.ldx2 + k, valid, r);
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    y[j] += r[j];
            }
    }
}

template <int OP, bool BF16, bool GROUPED, int R>
__global__ void wq_quantize_row(const QuantParams p)
{
    __shared__ float part[16];
    __shared__ uint32_t partm[16];
    const long row  = blockIdx.x;
    const int T     = blockDim.x;
    const int waves = T >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int RR = R > 0 ? R : 1;
    float y[RR][8];
    u4_t w16[RR];

    float rinv = 1.f;
    if constexpr(OP == 1)
    {
        // The sum of squares: a chain over a thread's elements, a tree over a wave, the waves in order.  Rows of 4097 to 8192 elements
        // take 1024 threads of one piece or 512 of two, by M (launch_row): the two pieces are summed apart there, as the other half of
        // 1024 threads sums the second, so that a row's result is the same in every batch.
        const bool apart = R == 2 && T == 512;
        float ss = 0.f, first = 0.f;
        if constexpr(R > 0)
        {
#pragma unroll
            for(int r = 0; r < RR; ++r)
            {
                const int k = (r * T + (int)threadIdx.x) * 8;
                row_value8<OP, BF16>(p, row, k, min(p.K - k, 8), y[r]);
            }
            // (the weights' loads fly while the row's sum is made)
            if(!p.weight_f32)
#pragma unroll
                for(int r = 0; r < RR; ++r)
                {
                    const int k = (r * T + (int)threadIdx.x) * 8;
                    w16[r]      = quant_load16<BF16>(p.weight, k, min(p.K - k, 8));
                }
#pragma unroll
            for(int r = 0; r < RR; ++r)
            {
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    ss = __builtin_fmaf(y[r][j], y[r][j], ss);
                if(R == 2 && r == 0 && apart)
                    first = ss, ss = 0.f;
            }
        }
        else
            for(int k = threadIdx.x * 8; k < p.K; k += T * 8)
            {
                row_value8<OP, BF16>(p, row, k, min(p.K - k, 8), y[0]);
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    ss = __builtin_fmaf(y[0][j], y[0][j], ss);
            }
        ss = wave_sums(R == 2 ? first : ss, ss);
        if(lane == 32)
            part[apart ? 8 + wave : wave] = ss;
        if(lane == 0 && apart)
            part[wave] = ss;
        __syncthreads();
        ss = 0.f;
        for(int w = 0; w < (apart ? 16 : waves); ++w)
            ss += part[w];
        rinv = 1.f / sqrtf(ss / (float)p.K + p.eps);
    }
    else if constexpr(R > 0)
    {
#pragma unroll
        for(int r = 0; r < RR; ++r)
        {
            const int k = (r * T + (int)threadIdx.x) * 8;
            row_value8<OP, BF16>(p, row, k, min(p.K - k, 8), y[r]);
        }
    }

    // the final values of piece r (k, valid): the norm's factor and weight, and h written out on the way
    auto finish = [&](float (&v)[8], int k, int valid, bool write_h, int r = -1) __attribute__((always_inline)) {
        if constexpr(OP == 1)
        {
            if(write_h && p.residual_out && valid > 0)
                quant_store8_16<BF16>(p.residual_out, row * p.ld_res + k, valid, v);
            float w[8];
            if(p.weight_f32)
                quant_load8_f32((const float*)p.weight + k, valid, w);
            else
                widen8<BF16>(r >= 0 ? w16[r] : quant_load16<BF16>(p.weight, k, valid), w);
#pragma unroll
            for(int j = 0; j < 8; ++j)
                v[j] = v[j] * rinv * w[j];
        }
    };
    auto emit = [&](float (&v)[8], int k, int valid, const GroupScale& g) __attribute__((always_inline)) {
#pragma unroll
        for(int j = 0; j < 8; ++j)
            v[j] = g.quotient(v[j]);
        if(valid > 0)
            quant_store8_f8(p.q + row * p.ldq + k, valid, v);
    };

    if constexpr(GROUPED)
    {
        // (16 lanes hold one group; lanes past the row's end hold zeros)
        auto one = [&](float (&v)[8], int k, int r) __attribute__((always_inline)) {
            const int valid = min(p.K - k, 8);
            finish(v, k, valid, true, r);
            const GroupScale g(row16_max(amax8(v)));
            emit(v, k, valid, g);
            if((lane & 15) == 0 && valid > 0)
                p.scale[row * p.ld_scale + (k >> 7)] = g.s;
        };
        if constexpr(R > 0)
        {
#pragma unroll
            for(int r = 0; r < RR; ++r)
                one(y[r], (r * T + (int)threadIdx.x) * 8, r);
        }
        else
            for(int k0 = 0; k0 < p.K; k0 += T * 8)
            {
                const int k = k0 + threadIdx.x * 8;
                row_value8<OP, BF16>(p, row, k, min(p.K - k, 8), y[0]);
                one(y[0], k, -1);
            }
    }
    else
    {
        uint32_t m = 0;
        if constexpr(R > 0)
        {
#pragma unroll
            for(int r = 0; r < RR; ++r)
            {
                const int k = (r * T + (int)threadIdx.x) * 8;
                finish(y[r], k, min(p.K - k, 8), true, r);
                m = max(m, amax8(y[r]));
            }
        }
        else
            for(int k = threadIdx.x * 8; k < p.K; k += T * 8)
            {
                row_value8<OP, BF16>(p, row, k, min(p.K - k, 8), y[0]);
                finish(y[0], k, min(p.K - k, 8), false);
                m = max(m, amax8(y[0]));
            }
        m = wave_max(m);
        if(lane == 0)
            partm[wave] = m;
        __syncthreads();
        m = 0;
        for(int w = 0; w < waves; ++w)
            m = max(m, partm[w]);
        const GroupScale g(m);
        if(threadIdx.x == 0)
            p.scale[row * p.ld_scale] = g.s;
        if constexpr(R > 0)
        {
#pragma unroll
            for(int r = 0; r < RR; ++r)
            {
                const int k = (r * T + (int)threadIdx.x) * 8;
                emit(y[r], k, min(p.K - k, 8), g);
            }
        }
        else
            for(int k = threadIdx.x * 8; k < p.K; k += T * 8)
            {
                const int valid = min(p.K - k, 8);
                row_value8<OP, BF16>(p, row, k, valid, y[0]);
                finish(y[0], k, valid, true);
                emit(y[0], k, valid, g);
            }
    }
}

} // namespace wq
