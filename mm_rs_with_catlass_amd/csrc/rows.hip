// Rows to their experts and back: every token's row at the places of its choices (with e4m3 scales), the choices' rows summed at their tokens by share, and that sum's
// gradients.
//
//   spread: out[back[t,j]] = x[t];  gather: out[t] = sum over j of share[t,j] y[back[t,j]], in fp32 and in the order of j, rounded once;
//   backward: dy[back[t,j]] = share[t,j] dout[t], dshare[t,j] = <dout[t], y[back[t,j]]>.
//
// Memory bounds all three.  Work is cut by token, not by place: a token's row is read once for all of its choices.  A place outside the rows (a choice without a row: -1)
// is neither read nor written.
#include <hip/hip_runtime.h>

#include "layer_args.h"
#include "rows_device.h"

namespace catcoc {

typedef int v4i __attribute__((ext_vector_type(4)));

// 16 bytes at any address, or what is left of a row of `size` bytes in whole values of ES.
template <uint32_t ES>
__device__ __forceinline__ v4i load16(const unsigned char *row, uint64_t at, uint64_t size)
{
    v4i v = {0, 0, 0, 0};
    if (at + 16u <= size) {
        __builtin_memcpy(&v, row + at, 16);
    } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < 16u; i += ES) {
            if (at + i >= size) continue;
            if constexpr (ES == 4) __builtin_memcpy(&w[i >> 2], row + at + i, 4);
            else if constexpr (ES == 2) {
                unsigned short h;
                __builtin_memcpy(&h, row + at + i, 2);
                w[i >> 2] |= (uint32_t)h << (8u * (i & 3u));
            } else {
                w[i >> 2] |= (uint32_t)row[at + i] << (8u * (i & 3u));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (int)w[i];
    }
    return v;
}

template <uint32_t ES>
__device__ __forceinline__ void store16(unsigned char *row, uint64_t at, uint64_t size, v4i v)
{
    if (at + 16u <= size) {
        __builtin_memcpy(row + at, &v, 16);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16u; i += ES) {
            if (at + i >= size) continue;
            const uint32_t w = (uint32_t)v[i >> 2] >> (8u * (i & 3u));
            __builtin_memcpy(row + at + i, &w, ES);
        }
    }
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// A wave takes SEG KiB of a token's row.  ES: bytes of a value.
template <uint32_t ES, int SEG>
__global__ void __launch_bounds__(256) spread_rows_kernel(const RowsArgs args)
{
    const uint64_t size = (uint64_t)args.cols * ES, rows = (uint64_t)args.tokens * args.top;
    const uint32_t segs = (uint32_t)((size + SEG * 1024u - 1u) / (SEG * 1024u)), lane = threadIdx.x & 63u;
    const uint32_t wave = uniform(workgroup() * 4u + (threadIdx.x >> 6));
    const uint32_t token = wave / segs, seg = wave - token * segs;
    if (token >= args.tokens) return;
    const unsigned char *const from = (const unsigned char *)args.x + token * size;
    const uint64_t at = (uint64_t)seg * SEG * 1024u + lane * 16u;
    v4i v[SEG];
#pragma unroll
    for (int i = 0; i < SEG; ++i) v[i] = load16<ES>(from, at + i * 1024u, size);
    const int32_t *const back = args.back + (uint64_t)token * args.top;
    for (uint32_t j = 0; j < args.top; ++j) {
        const uint32_t to = uniform((uint32_t)back[j]);
        if (to >= rows) continue;
        unsigned char *const row = (unsigned char *)args.out + to * size;
#pragma unroll
        for (int i = 0; i < SEG; ++i)
            if (at + i * 1024u < size) store16<ES>(row, at + i * 1024u, size, v[i]);
    }
    if (args.scale != nullptr && seg == 0) {
        const uint32_t blocks = (args.cols + kScaleBlock - 1u) / kScaleBlock;
        for (uint32_t b = lane; b < blocks; b += 64u) {
            const float s = args.scale[(uint64_t)b * args.tokens + token];
            for (uint32_t j = 0; j < args.top; ++j) {
                const uint32_t to = uniform((uint32_t)back[j]);
                if (to < rows) args.outScale[b * rows + to] = s;
            }
        }
    }
}

// A wave takes SEG times 512 values of a token's sum; four choices' rows are asked for together.
template <uint32_t DT, int SEG>
__global__ void __launch_bounds__(256) gather_rows_kernel(const RowsArgs args)
{
    const uint64_t rows = (uint64_t)args.tokens * args.top;
    const uint32_t segs = (args.cols + SEG * 512u - 1u) / (SEG * 512u), lane = threadIdx.x & 63u;
    const uint32_t wave = uniform(workgroup() * 4u + (threadIdx.x >> 6));
    const uint32_t token = wave / segs, col = (wave - token * segs) * SEG * 512u + lane * 8u;
    if (token >= args.tokens) return;
    const int32_t *const back = args.back + (uint64_t)token * args.top;
    const float *const share = args.share ? args.share + (uint64_t)token * args.top : nullptr;
    Eight sum[SEG] = {};
    constexpr int BATCH = SEG > 1 ? 4 : 8;
    for (uint32_t first = 0; first < args.top; first += BATCH) {
        Raw8<DT> raw[BATCH][SEG];
        bool on[BATCH];
#pragma unroll
        for (uint32_t j = 0; j < (uint32_t)BATCH; ++j) {
            const uint32_t at = first + j < args.top ? uniform((uint32_t)back[first + j]) : 0xffffffffu;
            on[j] = at < rows;
            if (!on[j]) continue;
#pragma unroll
            for (int i = 0; i < SEG; ++i) raw[j][i] = load_raw8<DT>(args.y, at, args.cols, col + i * 512u, args.cols);
        }
#pragma unroll
        for (uint32_t j = 0; j < (uint32_t)BATCH; ++j) {
            if (!on[j]) continue;
            const float s = share ? share[first + j] : 1.f;
#pragma unroll
            for (int i = 0; i < SEG; ++i) {
                const Eight v = widen8<DT>(raw[j][i]);
#pragma unroll
                for (int k = 0; k < 8; ++k) sum[i].v[k] = __builtin_fmaf(s, v.v[k], sum[i].v[k]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < SEG; ++i)
        if (col + i * 512u < args.cols) store_raw8<DT>(args.out, token, args.cols, col + i * 512u, args.cols, round8<DT>(sum[i]));
}

// T threads take a choice's row, one after the other a token's.
template <uint32_t DT, int T>
__global__ void __launch_bounds__(256) gather_rows_backward_kernel(const RowsArgs args)
{
    constexpr uint32_t W = T / 64;
    __shared__ float parts[2][W];
    const uint64_t rows = (uint64_t)args.tokens * args.top;
    const uint32_t t = threadIdx.x % T;
    const uint64_t token = T < 256 ? (uint64_t)workgroup() * (256u / T) + uniform(threadIdx.x / T) : workgroup();
    if (token >= args.tokens) return;
    for (uint32_t j = 0; j < args.top; ++j) {
        const uint64_t i = token * args.top + j;
        const uint32_t at = uniform((uint32_t)args.back[i]);
        const float share = args.share[i];
        float dot = 0.f;
        if (at < rows) {
            for (uint32_t col = t * 8u; col < args.cols; col += T * 16u) {
                const uint32_t next = col + T * 8u;   // (two pieces of both rows are asked for together)
                const Raw8<DT> rd = load_raw8<DT>(args.x, token, args.cols, col, args.cols), ry = load_raw8<DT>(args.y, at, args.cols, col, args.cols);
                Raw8<DT> rd2 = {}, ry2 = {};
                if (next < args.cols) {
                    rd2 = load_raw8<DT>(args.x, token, args.cols, next, args.cols);
                    ry2 = load_raw8<DT>(args.y, at, args.cols, next, args.cols);
                }
                Eight d = widen8<DT>(rd), y = widen8<DT>(ry);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    dot = __builtin_fmaf(d.v[k], y.v[k], dot);
                    d.v[k] *= share;
                }
                store_raw8<DT>(args.out, at, args.cols, col, args.cols, round8<DT>(d));
                if (next < args.cols) {
                    d = widen8<DT>(rd2), y = widen8<DT>(ry2);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        dot = __builtin_fmaf(d.v[k], y.v[k], dot);
                        d.v[k] *= share;
                    }
                    store_raw8<DT>(args.out, at, args.cols, next, args.cols, round8<DT>(d));
                }
            }
        }
        dot = wave_sum(dot);
        if constexpr (W > 1) {
            if ((t & 63u) == 0) parts[j & 1u][t >> 6] = dot;
            __syncthreads();
            dot = parts[j & 1u][0];
#pragma unroll
            for (uint32_t k = 1; k < W; ++k) dot += parts[j & 1u][k];
        }
        if (t == 0) args.dshare[i] = dot;
    }
}

// Fewer segments a wave where there would else be fewer than 16 waves a CU.
constexpr uint64_t kManyWaves = 4096;

template <uint32_t ES>
static int launch_spread_size(const RowsArgs &a, hipStream_t stream)
{
    const uint64_t size = (uint64_t)a.cols * ES, fours = a.tokens * ((size + 4095) / 4096), ones = a.tokens * ((size + 1023) / 1024);
    if (fours >= kManyWaves) hipLaunchKernelGGL((spread_rows_kernel<ES, 4>), grid_of((fours + 3) / 4, 256), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((spread_rows_kernel<ES, 1>), grid_of((ones + 3) / 4, 256), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int launch_spread_rows(uint32_t valueBytes, const RowsArgs &a, void *stream)
{
    if (valueBytes == 1) return launch_spread_size<1>(a, (hipStream_t)stream);
    if (valueBytes == 2) return launch_spread_size<2>(a, (hipStream_t)stream);
    return launch_spread_size<4>(a, (hipStream_t)stream);
}

template <uint32_t DT>
static int launch_gather_type(const RowsArgs &a, hipStream_t stream)
{
    const uint64_t twos = a.tokens * (uint64_t)((a.cols + 1023u) / 1024u), ones = a.tokens * (uint64_t)((a.cols + 511u) / 512u);
    if (twos >= kManyWaves) hipLaunchKernelGGL((gather_rows_kernel<DT, 2>), grid_of((twos + 3) / 4, 256), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((gather_rows_kernel<DT, 1>), grid_of((ones + 3) / 4, 256), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int launch_gather_rows(uint32_t type, const RowsArgs &a, void *stream)
{
    if (type == DT_F16) return launch_gather_type<DT_F16>(a, (hipStream_t)stream);
    if (type == DT_BF16) return launch_gather_type<DT_BF16>(a, (hipStream_t)stream);
    return launch_gather_type<0>(a, (hipStream_t)stream);
}

template <uint32_t DT>
static int launch_gather_backward_type(const RowsArgs &a, hipStream_t stream)
{
    if (a.cols <= 1024) hipLaunchKernelGGL((gather_rows_backward_kernel<DT, 64>), grid_of((a.tokens + 3ull) / 4, 256), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((gather_rows_backward_kernel<DT, 256>), grid_of(a.tokens, 256), dim3(256), 0, stream, a);
    return (int)hipGetLastError();
}

int launch_gather_rows_backward(uint32_t type, const RowsArgs &a, void *stream)
{
    if (type == DT_F16) return launch_gather_backward_type<DT_F16>(a, (hipStream_t)stream);
    if (type == DT_BF16) return launch_gather_backward_type<DT_BF16>(a, (hipStream_t)stream);
    return launch_gather_backward_type<0>(a, (hipStream_t)stream);
}

}  // namespace catcoc
