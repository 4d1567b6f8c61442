// Device code that the kernels over rows share (the quantizer, norms, routing, rows to experts and back): eight values of a row at any alignment, sums and
// maxima over lanes, e4m3 codes and their scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "launch_grid.h"
#include "ragged_args.h"

namespace catcoc {

typedef int v2i __attribute__((ext_vector_type(2)));

// One dimension of a launch holds fewer than 2^32 threads: workgroups past that go on in the second one, in rows of kGridRow (launch_grid.h).  Those past the last one
// asked for have to find nothing to do.  For the checked kernel, the quantizer, norms, router and rows; in the small tiles' kernel the second index costs a call of 18.5 us
// 0.46 of them.
inline dim3 grid_of(uint64_t wgs, uint32_t threads)
{
    const LaunchGrid g = launch_grid(wgs, threads);
    return dim3(g.x, g.y);
}
__device__ __forceinline__ uint32_t workgroup() { return (blockIdx.y << kGridRowLog) + blockIdx.x; }

struct Eight {
    float v[8];
};

// Eight values as they lie in memory; DT 0: fp32.
template <uint32_t DT>
struct Raw8 {
    uint32_t w[DT == 0 ? 8 : 4];
};

// Values [at, at + 8) of a row of `size`; zeros past its end.
template <uint32_t DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void *x, size_t row, uint32_t pitch, uint32_t at, uint32_t size)
{
    constexpr uint32_t ES = DT == 0 ? 4u : 2u;
    const unsigned char *p = (const unsigned char *)x + (row * pitch + at) * ES;
    Raw8<DT> raw;
    if (at + 8u <= size) {
        __builtin_memcpy(raw.w, p, sizeof raw.w);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < ES * 2u; ++i) raw.w[i] = 0;
#pragma unroll
        for (uint32_t i = 0; i < 7u; ++i) {
            if (at + i >= size) continue;
            if constexpr (DT == 0) __builtin_memcpy(&raw.w[i], p + 4u * i, 4);
            else {
                unsigned short h;
                __builtin_memcpy(&h, p + 2u * i, 2);
                raw.w[i >> 1] |= (uint32_t)h << (16u * (i & 1u));
            }
        }
    }
    return raw;
}

template <uint32_t DT>
__device__ __forceinline__ Eight widen8(const Raw8<DT> &raw)
{
    Eight e;
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        if constexpr (DT == 0) e.v[i] = __builtin_bit_cast(float, raw.w[i]);
        else {
            const uint32_t h = (raw.w[i >> 1] >> (16u * (i & 1u))) & 0xffffu;
            if constexpr (DT == DT_BF16) e.v[i] = __builtin_bit_cast(float, h << 16);
            else e.v[i] = (float)__builtin_bit_cast(_Float16, (unsigned short)h);
        }
    }
    return e;
}

template <uint32_t DT>
__device__ __forceinline__ Eight load8(const void *x, size_t row, uint32_t pitch, uint32_t at, uint32_t size)
{
    return widen8<DT>(load_raw8<DT>(x, row, pitch, at, size));
}

// Rounded to nearest even.
template <uint32_t DT>
__device__ __forceinline__ Raw8<DT> round8(const Eight &e)
{
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    Raw8<DT> raw;
    if constexpr (DT == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw.w[i] = __builtin_bit_cast(uint32_t, e.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == DT_BF16) raw.w[i] = __builtin_bit_cast(uint32_t, v2bf{(__bf16)e.v[2 * i], (__bf16)e.v[2 * i + 1]});
            else raw.w[i] = __builtin_bit_cast(uint32_t, v2h{(_Float16)e.v[2 * i], (_Float16)e.v[2 * i + 1]});
        }
    }
    return raw;
}

// LATER: past the caches, for what is not read again soon.
template <uint32_t DT, bool LATER = false>
__device__ __forceinline__ void store_raw8(void *x, size_t row, uint32_t pitch, uint32_t at, uint32_t size, const Raw8<DT> &raw)
{
    constexpr uint32_t ES = DT == 0 ? 4u : 2u;
    unsigned char *p = (unsigned char *)x + (row * pitch + at) * ES;
    if (at + 8u <= size) {
        if constexpr (LATER) {
            typedef uint32_t v4u __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
            for (uint32_t i = 0; i < ES * 2u; i += 4u) __builtin_nontemporal_store(v4u{raw.w[i], raw.w[i + 1u], raw.w[i + 2u], raw.w[i + 3u]}, (v4u *)(p + 4u * i));
        } else {
            __builtin_memcpy(p, raw.w, sizeof raw.w);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 7u; ++i) {
            if (at + i >= size) continue;
            if constexpr (DT == 0) __builtin_memcpy(p + 4u * i, &raw.w[i], 4);
            else {
                const unsigned short h = (unsigned short)(raw.w[i >> 1] >> (16u * (i & 1u)));
                __builtin_memcpy(p + 2u * i, &h, 2);
            }
        }
    }
}

// The sum of a wave's lanes, in all of them; the order is always the same.
__device__ __forceinline__ float wave_sum(float v)
{
    auto lanes = [](float f, auto turn) { return f + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, f), decltype(turn)::value, 0xf, 0xf, false)); };
    v = lanes(v, std::integral_constant<int, 0x128>{});   // row_ror:8, 4, 2, 1
    v = lanes(v, std::integral_constant<int, 0x124>{});
    v = lanes(v, std::integral_constant<int, 0x122>{});
    v = lanes(v, std::integral_constant<int, 0x121>{});
    auto at = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
    return (at(0) + at(16)) + (at(32) + at(48));
}

// Inclusive sums over the lanes of a wave.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v)
{
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false);   // row_shr:1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);   // row_bcast:15 and 31
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
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

}  // namespace catcoc
