// Rows to their experts and back: every token's row at the places of its choices (with e4m3 scales), the choices' rows summed at their tokens by share, and that sum's
// gradients.
//
//   spread: out[back[t,j]] = x[t];  gather: out[t] = sum over j of share[t,j] y[back[t,j]], in fp32 and in the order of j, rounded once;
//   backward: dy[back[t,j]] = share[t,j] dout[t], dshare[t,j] = <dout[t], y[back[t,j]]>.
//
// Memory bounds all three.  Work is cut by token, not by place: a token's row is read once for all of its choices.  A place outside the rows (a choice without a row: -1)
// is neither read nor written.
//
// us a call, six sets of operands and results in turn, so that they come from memory: 2048 tokens of 4096 bf16 values with eight places each: spread 30.5, 4.9 TB/s (e4m3 with
// scales 17.4, 4.5; 14.5 where every call's results go to one place, half of which the 256 MB cache holds), gather 33.5, 4.5, backward 57, 5.0, its rows alone 40; 32 tokens 3.6, 3.8 and 3.6.
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

// A wave takes a KiB of a token's row (four were slower: 8192 tokens' 4096 e4m3 values to eight places 81.6 us, 76.8 with one; 16384 rows of 256 values to two 13 and 7.3).
// Scales, if any, are the first `scaleWgs` workgroups': a thread takes a choice's of up to eight blocks, all asked for before the first is stored (2048 tokens of 4096 to
// eight places 17.4 us, 15.2 without scales; with a row's scales behind its values 2.3 more, one token 1.2 more).  ES: bytes of a value.
constexpr uint32_t kScaleRows = 256, kScaleBlocks = 8;

template <uint32_t ES>
__global__ void __launch_bounds__(256) spread_rows_kernel(const RowsArgs args)
{
    const uint64_t rows = (uint64_t)args.tokens * args.top;
    uint32_t wg = workgroup();
    if constexpr (ES == 1) {
        if (wg < args.scaleWgs) {
            const uint32_t blocks = (args.cols + kScaleBlock - 1u) / kScaleBlock, parts = (blocks + kScaleBlocks - 1u) / kScaleBlocks;
            const uint32_t group = wg / parts, first = (wg - group * parts) * kScaleBlocks;
            const uint64_t at = (uint64_t)group * kScaleRows + threadIdx.x;
            if (at >= rows) return;
            const uint32_t to = (uint32_t)args.back[at], token = (uint32_t)at / args.top;
            if (to >= rows) return;
            float s[kScaleBlocks];
#pragma unroll
            for (uint32_t i = 0; i < kScaleBlocks; ++i) s[i] = args.scale[(uint64_t)umin(first + i, blocks - 1u) * args.tokens + token];
#pragma unroll
            for (uint32_t i = 0; i < kScaleBlocks; ++i)
                if (first + i < blocks) args.outScale[(first + i) * rows + to] = s[i];
            return;
        }
        wg -= args.scaleWgs;
    }
    const uint64_t size = (uint64_t)args.cols * ES;
    const uint32_t segs = (uint32_t)((size + 1023u) / 1024u), lane = threadIdx.x & 63u;
    const uint32_t wave = uniform(wg * 4u + (threadIdx.x >> 6));
    const uint32_t token = wave / segs;
    if (token >= args.tokens) return;
    const uint64_t at = (uint64_t)(wave - token * segs) * 1024u + lane * 16u;
    if (at >= size) return;
    const v4i v = load16<ES>((const unsigned char *)args.x + token * size, at, size);
    const int32_t *const back = args.back + (uint64_t)token * args.top;
    for (uint32_t j = 0; j < args.top; ++j) {
        const uint32_t to = uniform((uint32_t)back[j]);
        if (to < rows) store16<ES>((unsigned char *)args.out + to * size, at, size, v);
    }
}

// A wave takes 512 values of a token's sum (1024 were slower: 2048 tokens of eight rows of 4096 37.1 us, 34.9 with 512); eight choices' rows are asked for together.
template <uint32_t DT>
__global__ void __launch_bounds__(256) gather_rows_kernel(const RowsArgs args)
{
    const uint64_t rows = (uint64_t)args.tokens * args.top;
    const uint32_t segs = (args.cols + 511u) / 512u, lane = threadIdx.x & 63u;
    const uint32_t wave = uniform(workgroup() * 4u + (threadIdx.x >> 6));
    const uint32_t token = wave / segs, col = (wave - token * segs) * 512u + lane * 8u;
    if (token >= args.tokens) return;
    const int32_t *const back = args.back + (uint64_t)token * args.top;
    const float *const share = args.share ? args.share + (uint64_t)token * args.top : nullptr;
    Eight sum = {};
    constexpr uint32_t BATCH = 8;
    for (uint32_t first = 0; first < args.top; first += BATCH) {
        Raw8<DT> raw[BATCH];
        bool on[BATCH];
#pragma unroll
        for (uint32_t j = 0; j < BATCH; ++j) {
            const uint32_t at = first + j < args.top ? uniform((uint32_t)back[first + j]) : 0xffffffffu;
            on[j] = at < rows;
            if (on[j]) raw[j] = load_raw8<DT>(args.y, at, args.cols, col, args.cols);
        }
#pragma unroll
        for (uint32_t j = 0; j < BATCH; ++j) {
            if (!on[j]) continue;
            const float s = share ? share[first + j] : 1.f;
            const Eight v = widen8<DT>(raw[j]);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum.v[k] = __builtin_fmaf(s, v.v[k], sum.v[k]);
        }
    }
    if (col < args.cols) store_raw8<DT>(args.out, token, args.cols, col, args.cols, round8<DT>(sum));
}

// T threads take a choice's row.  The choices of a token follow each other on one XCD, whose L2 then has the token's gradient for all but the first (us, with one workgroup
// for all of a token's choices / with these: 2048 tokens of eight rows of 4096 64 / 57, 32 of them 8.6 / 3.6).
// DY, DSHARE: which of the two gradients is wanted; y is not read for dy alone.
template <uint32_t DT, int T, bool DY, bool DSHARE>
__global__ void __launch_bounds__(256) gather_rows_backward_kernel(const RowsArgs args)
{
    constexpr uint32_t W = T / 64, EACH = 256 / T;
    __shared__ float parts[W];
    const uint64_t rows = (uint64_t)args.tokens * args.top;
    const uint32_t t = threadIdx.x % T, wg = workgroup(), turn = wg >> 3;
    const uint64_t token = ((uint64_t)(turn / args.top) * 8u + (wg & 7u)) * EACH + uniform(threadIdx.x / T);
    if (token >= args.tokens) return;   // (a wave's or a workgroup's)
    const uint64_t i = token * args.top + turn % args.top;
    const uint32_t at = uniform((uint32_t)args.back[i]);
    float dot = 0.f;
    if (at < rows) {
        const float share = DY ? args.share[i] : 0.f;
        auto piece = [&](uint32_t col, Raw8<DT> &d, Raw8<DT> &y) {
            d = load_raw8<DT>(args.x, token, args.cols, col, args.cols);
            if constexpr (DSHARE) y = load_raw8<DT>(args.y, at, args.cols, col, args.cols);
        };
        auto done = [&](uint32_t col, const Raw8<DT> &rd, const Raw8<DT> &ry) {
            Eight d = widen8<DT>(rd);
            if constexpr (DSHARE) {
                const Eight y = widen8<DT>(ry);
#pragma unroll
                for (int k = 0; k < 8; ++k) dot = __builtin_fmaf(d.v[k], y.v[k], dot);
            }
            if constexpr (DY) {
#pragma unroll
                for (int k = 0; k < 8; ++k) d.v[k] *= share;
                store_raw8<DT>(args.out, at, args.cols, col, args.cols, round8<DT>(d));
            }
        };
        for (uint32_t col = t * 8u; col < args.cols; col += T * 16u) {
            const uint32_t next = col + T * 8u;   // (two pieces of both rows are asked for together)
            Raw8<DT> d = {}, y = {}, d2 = {}, y2 = {};
            piece(col, d, y);
            if (next < args.cols) piece(next, d2, y2);
            done(col, d, y);
            if (next < args.cols) done(next, d2, y2);
        }
    }
    if constexpr (DSHARE) {
        dot = wave_sum(dot);
        if constexpr (W > 1) {
            if ((t & 63u) == 0) parts[t >> 6] = dot;
            __syncthreads();
            dot = parts[0];
#pragma unroll
            for (uint32_t k = 1; k < W; ++k) dot += parts[k];
        }
        if (t == 0) args.dshare[i] = dot;
    }
}

template <uint32_t ES>
static int launch_spread_size(RowsArgs a, hipStream_t stream)
{
    const uint64_t waves = a.tokens * (((uint64_t)a.cols * ES + 1023) / 1024);
    if (a.scale != nullptr) {
        const uint64_t blocks = (a.cols + kScaleBlock - 1u) / kScaleBlock, rows = (uint64_t)a.tokens * a.top;
        a.scaleWgs = (uint32_t)((rows + kScaleRows - 1) / kScaleRows * ((blocks + kScaleBlocks - 1) / kScaleBlocks));
    }
    hipLaunchKernelGGL((spread_rows_kernel<ES>), grid_of(a.scaleWgs + (waves + 3) / 4, 256), dim3(256), 0, stream, a);
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
    const uint64_t waves = a.tokens * (uint64_t)((a.cols + 511u) / 512u);
    hipLaunchKernelGGL((gather_rows_kernel<DT>), grid_of((waves + 3) / 4, 256), dim3(256), 0, stream, a);
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
    const uint32_t each = a.cols <= 1024 ? 4 : 1;   // tokens a workgroup
    const uint64_t wgs = (a.tokens + 8ull * each - 1) / (8ull * each) * 8 * a.top;
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid_of(wgs, 256), dim3(256), 0, stream, a);
        return (int)hipGetLastError();
    };
    if (a.dshare == nullptr) return each == 4 ? go(gather_rows_backward_kernel<DT, 64, true, false>) : go(gather_rows_backward_kernel<DT, 256, true, false>);
    if (a.out == nullptr) return each == 4 ? go(gather_rows_backward_kernel<DT, 64, false, true>) : go(gather_rows_backward_kernel<DT, 256, false, true>);
    return each == 4 ? go(gather_rows_backward_kernel<DT, 64, true, true>) : go(gather_rows_backward_kernel<DT, 256, true, true>);
}

int launch_gather_rows_backward(uint32_t type, const RowsArgs &a, void *stream)
{
    if (type == DT_F16) return launch_gather_backward_type<DT_F16>(a, (hipStream_t)stream);
    if (type == DT_BF16) return launch_gather_backward_type<DT_BF16>(a, (hipStream_t)stream);
    return launch_gather_backward_type<0>(a, (hipStream_t)stream);
}

}  // namespace catcoc
