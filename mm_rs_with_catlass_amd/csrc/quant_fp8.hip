// Quantizer: rows of 16- or 32-bit values to e4m3 with one fp32 scale per 128 values of a row, or per 128x128 block.
//
// scale = max(largest magnitude, 2^-40) / 448, code = value / scale rounded to nearest even: both divisions are the correctly rounded ones.  A block's values share their
// divisor, so a quotient takes three operations instead of a division's ten: with r the correctly rounded 1 / s, q = x r and the remainder
// x - q s (exact in one fused operation), fma(remainder, r, q) is the correctly rounded x / s (Markstein, IBM J. Res. Dev. 34, 1990).  It needs a remainder that is
// representable, which the scale's floor sees to: a value whose code is not 0 is at least 2^-59.
//
// Bound by memory where there are many rows: 16384 rows of 1792 gated values, bf16, 30.4 us, 4.8 TB/s (a copy reaches 4.9), 39.6 us with a division a value and four rows a wave; blocks of
// 4096x4096 bf16 10.4 us; 16 rows of 1024 5.6 us, the launch.
#include <hip/hip_runtime.h>

#include "ragged.h"

namespace catcoc {

namespace {

struct Eight {
    float v[8];
};

// Values [at, at + 8) of a row of `size`; zeros past its end.
template <uint32_t DT>
__device__ __forceinline__ Eight load8(const void *x, size_t row, uint32_t pitch, uint32_t at, uint32_t size)
{
    constexpr uint32_t ES = DT == 0 ? 4u : 2u;
    const unsigned char *p = (const unsigned char *)x + (row * pitch + at) * ES;
    uint32_t raw[ES * 2];
    if (at + 8u <= size) {
        __builtin_memcpy(raw, p, sizeof raw);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < ES * 2u; ++i) raw[i] = 0;
#pragma unroll
        for (uint32_t i = 0; i < 7u; ++i) {
            if (at + i >= size) continue;
            if constexpr (DT == 0) __builtin_memcpy(&raw[i], p + 4u * i, 4);
            else {
                unsigned short h;
                __builtin_memcpy(&h, p + 2u * i, 2);
                raw[i >> 1] |= (uint32_t)h << (16u * (i & 1u));
            }
        }
    }
    Eight e;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        if constexpr (DT == 0) e.v[i] = __builtin_bit_cast(float, raw[i]);
        else {
            const uint32_t h = (raw[i >> 1] >> (16u * (i & 1u))) & 0xffffu;
            if constexpr (DT == DT_BF16) e.v[i] = __builtin_bit_cast(float, h << 16);
            else e.v[i] = (float)__builtin_bit_cast(_Float16, (unsigned short)h);
        }
    }
    return e;
}

// silu(g) * u = g / (1 + e^-g) * u, where e^-g and its reciprocal are far inside fp32's range.  e^-g = 2^t e^r, t = -g log2 e and r what its rounding leaves: it would
// else cost the result 2^-18.
__device__ __forceinline__ float silu_times(float g, float u)
{
    const float t = g * -1.44269504f, r = __builtin_fmaf(t, -0.693147181f, -g), e = __builtin_amdgcn_exp2f(t);
    return g * __builtin_amdgcn_rcpf(1.f + __builtin_fmaf(e, r, e)) * u;
}

// The same for any gate, as g u / (1 + h^2) with h = e^(-|g|/2), times h^2 where g < 0, one h before u and one behind it: g h is below 1 and nothing leaves fp32's
// range that the result does not leave (e^-g does from g = -88 on, where a large u still makes something of silu).  From |g| = 175 on h is 0.
__device__ __forceinline__ float silu_times_far(float g, float u)
{
    const float a = __builtin_amdgcn_fmed3f(__builtin_fabsf(g), 0.f, 200.f);   // (an infinity would leave no remainder; a NaN is in g still)
    const float t = a * -0.721347520f, r = __builtin_fmaf(t, -0.693147181f, a * -0.5f), h0 = __builtin_amdgcn_exp2f(t), h = __builtin_fmaf(h0, r, h0);
    const float s = __builtin_amdgcn_rcpf(__builtin_fmaf(h, h, 1.f)), f = g < 0.f ? h : 1.f;
    return g * (f * s) * u * f;
}

__device__ __forceinline__ void silu_times8(Eight &g, const Eight &u)
{
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_fmaxf(top, __builtin_fabsf(g.v[i]));   // (a NaN stays one on either way)
    // 16384 rows of 1792 in bf16: 30.4 us with the choice, 31.8 with the second form for all gates; instructions bound it as much as memory does
    if (top < 64.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g.v[i] = silu_times(g.v[i], u.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) g.v[i] = silu_times_far(g.v[i], u.v[i]);
    }
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }   // (as an integer: a NaN is the largest)

__device__ __forceinline__ float scale_of(uint32_t top)
{
    const float t = __builtin_bit_cast(float, top);
    return (t < kScaleFloor ? kScaleFloor : t) / kE4m3Top;   // (NaN stays)
}

__device__ __forceinline__ v2i codes8(const Eight &e, float scale)
{
    float q[8];
    const float r = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = e.v[i] * r;
        q[i] = __builtin_fmaf(__builtin_fmaf(-t, scale, e.v[i]), r, t);
    }
    if (!__builtin_isfinite(scale)) {   // (zeros and NaN)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = e.v[i] / scale;
    }
    int a = 0, b = 0;
    a = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], a, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], a, true);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], b, false);
    b = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], b, true);
    return v2i{a, b};
}

__device__ __forceinline__ void store8(unsigned char *q, size_t row, uint32_t pitch, uint32_t at, uint32_t size, v2i v)
{
    unsigned char *p = q + row * pitch + at;
    if (at + 8u <= size) {
        __builtin_memcpy(p, &v, 8);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 7u; ++i)
            if (at + i < size) p[i] = (unsigned char)((uint32_t)v[i >> 2] >> (8u * (i & 3u)));
    }
}

// The largest of 16 consecutive lanes' values, in all of them.
__device__ __forceinline__ uint32_t max16(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));   // row_ror:8, 4, 2, 1
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
    return v;
}

}  // namespace

// One scale per 128 values of a row: 16 lanes share a block; a wave takes the same block of 4 QUADS consecutive rows, whose loads all go out first.
template <uint32_t DT, bool GATED, int QUADS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs args)
{
    const uint32_t lane = threadIdx.x & 63u, blocks = (args.cols + kScaleBlock - 1u) / kScaleBlock;
    const uint32_t groups = (args.rows + 4u * QUADS - 1u) / (4u * QUADS);
    const uint32_t at = workgroup() * 4u + (threadIdx.x >> 6);   // (fewer than 2^31 blocks of four rows, the host sees to it)
    const uint32_t group = at / blocks, block = at - group * blocks;
    if (group >= groups) return;
    const uint32_t row0 = 4u * QUADS * group + (lane >> 4), col = block * kScaleBlock + (lane & 15u) * 8u;
    const uint32_t pitch = GATED ? 2u * args.cols : args.cols;
    // (the upper half's values lie `cols` further on; where fewer than eight are left nothing is read)
    const void *const up = (const unsigned char *)args.x + (GATED ? (size_t)args.cols * (DT == 0 ? 4u : 2u) : (size_t)0);
    Eight e[QUADS], u[GATED ? QUADS : 1];
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        const uint32_t row = umin(row0 + 4u * j, args.rows - 1u);   // (rows past the last one repeat it and are not stored)
        e[j] = load8<DT>(args.x, row, pitch, col, args.cols);
        if constexpr (GATED) u[j] = load8<DT>(up, row, pitch, col, args.cols);
    }
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        const uint32_t row = row0 + 4u * j;
        if constexpr (GATED) silu_times8(e[j], u[j]);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, magnitude(e[j].v[i]));
        const float scale = scale_of(max16(top));
        if (row >= args.rows) continue;
        if ((lane & 15u) == 0) args.scale[(size_t)block * args.rows + row] = scale;
        if (col < args.cols) store8(args.q, row, args.cols, col, args.cols, codes8(e[j], scale));
    }
}

// One scale per 128x128 block: a workgroup holds the block in registers.
template <uint32_t DT>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const QuantArgs args)
{
    __shared__ uint32_t tops[4];
    const uint32_t at = workgroup(), blocks = (args.cols + kScaleBlock - 1u) / kScaleBlock, rb = at / blocks, cb = at - rb * blocks;
    if (rb >= (args.rows + kScaleBlock - 1u) / kScaleBlock) return;
    const uint32_t col = cb * kScaleBlock + (threadIdx.x & 15u) * 8u, row0 = rb * kScaleBlock + (threadIdx.x >> 4);
    Eight e[8];
    uint32_t top = 0;
#pragma unroll
    for (uint32_t j = 0; j < 8u; ++j) {
        if (row0 + 16u * j < args.rows) e[j] = load8<DT>(args.x, row0 + 16u * j, args.cols, col, args.cols);
        else e[j] = Eight{};
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, magnitude(e[j].v[i]));
    }
    top = max16(top);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    if ((threadIdx.x & 63u) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    const float scale = scale_of(max(max(tops[0], tops[1]), max(tops[2], tops[3])));
    if (threadIdx.x == 0) args.scale[at] = scale;
    if (col >= args.cols) return;
#pragma unroll
    for (uint32_t j = 0; j < 8u; ++j)
        if (row0 + 16u * j < args.rows) store8(args.q, row0 + 16u * j, args.cols, col, args.cols, codes8(e[j], scale));
}

template <uint32_t DT>
static int launch_dt(const QuantArgs &a, bool blocks, bool gated, hipStream_t stream)
{
    const uint64_t cb = (a.cols + kScaleBlock - 1u) / kScaleBlock;
    if (blocks) {
        hipLaunchKernelGGL((quantize_blocks_kernel<DT>), grid_of((a.rows + kScaleBlock - 1u) / kScaleBlock * cb, 256), dim3(256), 0, stream, a);
    } else {
        // four rows a wave where that leaves a CU fewer than 32 waves, else sixteen
        const uint64_t fours = (a.rows + 3ull) / 4u * cb;
        const bool many = fours >= 4u * 8192u;
        const dim3 grid = grid_of(((many ? (a.rows + 15ull) / 16u * cb : fours) + 3u) / 4u, 256);
        if (gated && many) hipLaunchKernelGGL((quantize_rows_kernel<DT, true, 4>), grid, dim3(256), 0, stream, a);
        else if (gated) hipLaunchKernelGGL((quantize_rows_kernel<DT, true, 1>), grid, dim3(256), 0, stream, a);
        else if (many) hipLaunchKernelGGL((quantize_rows_kernel<DT, false, 4>), grid, dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((quantize_rows_kernel<DT, false, 1>), grid, dim3(256), 0, stream, a);
    }
    return (int)hipGetLastError();
}

int launch_quantize(uint32_t dtype, const QuantArgs &a, bool blocks, bool gated, void *stream)
{
    if (dtype == DT_F16) return launch_dt<DT_F16>(a, blocks, gated, (hipStream_t)stream);
    if (dtype == DT_BF16) return launch_dt<DT_BF16>(a, blocks, gated, (hipStream_t)stream);
    return launch_dt<0>(a, blocks, gated, (hipStream_t)stream);
}

}  // namespace catcoc
