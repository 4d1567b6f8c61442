// Root-mean-square norm of rows with the residual's addition in front and e4m3 codes behind, and its backward pass.
//
//   s = x + residual, y = s r w with r = 1 / sqrt(mean(s^2) + eps); codes and scales of y as the quantizer's.
//   With n = s r and g = dy w: ds = r (g - n mean(g n)) + dsum, dw = sum over the rows of dy n.
//
// The sum is rounded to the residual's type, in which it is kept, and what is kept is normalised: so the backward pass, which has only that, takes the gradient of
// what the forward pass computed.  y is rounded once, from fp32, to each of the forms it is wanted in: codes are not codes of the 16-bit y.  A code's quotient does not depend on the
// root, so that products of 16-bit values often lie on the very middle of two codes: there fp32's last bit decides, and of 65536 codes up to nine are a step from those of another
// order of the same operations.
//
// Memory bounds both.  A row stays in the registers of the threads that share it between its one read and its writes: 64, 256 or 1024 threads with eight to 32 values each.
// y is what the next operator reads, the sum is read after a whole layer: it is stored past the caches, which leaves them to y (us, a norm and a quantizer of its y, without /
// with it: 3000 rows of 4096 26.3 / 23.7, 16384 140 / 128; where the sum is read at once 37.3 / 40.1 and 185 / 185).  Loops of resident workgroups with the next row's loads ahead
// were 7 to 10 % slower, as were loads past the caches.
//
// us a call, three or more sets of operands in turn: 16384 rows of 4096 in bf16 with a residual 91, 5.9 TB/s (a copy of as many bytes 104); 4099 rows of 1808 to e4m3 with an fp32 residual 15.8, 5.2 TB/s; 16 rows 3.6 on the GPU.  The
// backward pass of 8192 rows of 4096 54 us, 5.0 TB/s: 47 its rows, 4 the sum of the weight gradient's parts.
#include <hip/hip_runtime.h>

#include "layer_args.h"
#include "rows_device.h"

namespace catcoc {

// The sum over the T threads of a row, in all of them; `parts`: a place of LDS for each wave of the workgroup.
template <int T>
__device__ __forceinline__ float row_sum(float v, float *parts)
{
    v = wave_sum(v);
    if constexpr (T > 64) {
        if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = v;
        __syncthreads();
        const float *const mine = parts + threadIdx.x / T * (T / 64);
        v = mine[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v += mine[i];
    }
    return v;
}

// Workgroup `wg` of a launch, which go round-robin to the eight XCDs, as the place of its rows: every XCD gets runs of kRun consecutive ones, whose scales lie in one
// line (4099 rows of 1808 to e4m3 with an fp32 residual 16.7 us without, 15.9 with it, 4096 of 8192 with one 42.7 and 40.8, without one 24.6 and 23.7; not where few workgroups would share few XCDs, nor without scales, where it costs up to a
// tenth).
constexpr uint32_t kRun = 16;
__device__ __forceinline__ uint32_t run_place(uint32_t wg)
{
    const uint32_t at = wg >> 3;
    return (at / kRun * 8u + (wg & 7u)) * kRun + at % kRun;
}

// DT: type of x and y; RT: of the residual and the sum, DT_NONE: there is none.  T threads a row, CH times eight values each.
template <uint32_t DT, uint32_t RT, int T, int CH>
__global__ void __launch_bounds__(T < 256 ? 256 : T) rms_norm_kernel(const NormArgs args)
{
    constexpr bool SUM = RT != DT_NONE;
    constexpr uint32_t ST = SUM ? RT : DT;
    __shared__ float parts[T < 256 ? 4 : T / 64];
    const uint32_t t = threadIdx.x % T, wgs = T < 256 ? (args.rows + 256u / T - 1u) / (256u / T) : args.rows, wg = args.runs ? run_place(workgroup()) : workgroup();
    if (wg >= wgs) return;
    const uint64_t at = T < 256 ? (uint64_t)wg * (256u / T) + threadIdx.x / T : wg;
    const bool mine = T >= 256 || at < args.rows;
    const uint64_t row = mine ? at : args.rows - 1u;   // (the last one once more, for nothing)
    Raw8<DT> x[CH], w[CH];
    Raw8<ST> s[CH];
    Raw8<0> wide[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) x[c] = load_raw8<DT>(args.x, row, args.cols, (c * T + t) * 8u, args.cols);
    if constexpr (SUM) {
#pragma unroll
        for (int c = 0; c < CH; ++c) s[c] = load_raw8<RT>(args.residual, row, args.cols, (c * T + t) * 8u, args.cols);
    }
    if (args.weightType == DT) {
#pragma unroll
        for (int c = 0; c < CH; ++c) w[c] = load_raw8<DT>(args.weight, 0, 0, (c * T + t) * 8u, args.cols);
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c) wide[c] = load_raw8<0>(args.weight, 0, 0, (c * T + t) * 8u, args.cols);
    }
    Eight v[CH];
    float squares = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        v[c] = widen8<DT>(x[c]);
        if constexpr (SUM) {
            const Eight r = widen8<RT>(s[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c].v[i] += r.v[i];
            s[c] = round8<RT>(v[c]);
            v[c] = widen8<RT>(s[c]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) squares = __builtin_fmaf(v[c].v[i], v[c].v[i], squares);
    }
    const float r = 1.f / sqrtf(row_sum<T>(squares, parts) / (float)args.cols + args.eps);
    if (!mine) return;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t col = (c * T + t) * 8u;
        if constexpr (SUM) {
            if (col < args.cols) store_raw8<RT, true>(args.sum, row, args.cols, col, args.cols, s[c]);
        }
        const Eight g = args.weightType == DT ? widen8<DT>(w[c]) : widen8<0>(wide[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c].v[i] = v[c].v[i] * r * g.v[i];
        if (args.out != nullptr && col < args.cols) store_raw8<DT>(args.out, row, args.cols, col, args.cols, round8<DT>(v[c]));
        if (args.q != nullptr) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[c].v[i]));
            const float scale = scale_of(max16(top));
            if (col < args.cols) {
                if ((t & 15u) == 0) args.scale[(size_t)(col / kScaleBlock) * args.rows + row] = scale;
                store8(args.q, row, args.cols, col, args.cols, codes8(v[c], scale));
            }
        }
    }
}

// dx, and this workgroup's part of dw: WG / T rows at a time, whose columns' sums stay in the threads' registers.  DT: type of dy; ST: of x, dsum and dx.
template <uint32_t DT, uint32_t ST, int T, int WG>
__global__ void __launch_bounds__(WG) rms_norm_backward_kernel(const NormBackwardArgs args)
{
    constexpr int CH = 2, G = WG / T, W = T / 64;
    __shared__ float parts[2][G][W][2];
    __shared__ float sums[G > 1 ? T * CH * 8 : 1];
    const uint32_t t = threadIdx.x % T, g = threadIdx.x / T;
    Eight w[CH], dw[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t col = (c * T + t) * 8u;
        if (args.weightType == DT) w[c] = load8<DT>(args.weight, 0, 0, col, args.cols);
        else w[c] = load8<0>(args.weight, 0, 0, col, args.cols);
        dw[c] = Eight{};
    }
    uint32_t turn = 0;
    for (uint64_t base = (uint64_t)blockIdx.x * G; base < args.rows; base += (uint64_t)gridDim.x * G, turn ^= 1u) {
        const bool mine = base + g < args.rows;
        const uint64_t row = mine ? base + g : args.rows - 1u;   // (the last row once more, for nothing)
        Raw8<ST> rx[CH], rs[CH];
        Raw8<DT> rd[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t col = (c * T + t) * 8u;
            rx[c] = load_raw8<ST>(args.x, row, args.cols, col, args.cols);
            rd[c] = load_raw8<DT>(args.dy, row, args.cols, col, args.cols);
        }
        if (args.dsum != nullptr) {
#pragma unroll
            for (int c = 0; c < CH; ++c) rs[c] = load_raw8<ST>(args.dsum, row, args.cols, (c * T + t) * 8u, args.cols);
        }
        float squares = 0.f, dot = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const Eight s = widen8<ST>(rx[c]), d = widen8<DT>(rd[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                squares = __builtin_fmaf(s.v[i], s.v[i], squares);
                dot = __builtin_fmaf(s.v[i] * w[c].v[i], d.v[i], dot);
            }
        }
        squares = wave_sum(squares);
        dot = wave_sum(dot);
        if constexpr (W > 1) {   // (two sets of places in turn: who is behind the next row's barrier has read this row's)
            float(&p)[W][2] = parts[turn][g];
            if ((t & 63u) == 0) p[t >> 6][0] = squares, p[t >> 6][1] = dot;
            __syncthreads();
            squares = p[0][0], dot = p[0][1];
#pragma unroll
            for (int i = 1; i < W; ++i) squares += p[i][0], dot += p[i][1];
        }
        if (!mine) continue;
        const float r = 1.f / sqrtf(squares / (float)args.cols + args.eps), m = dot * r / (float)args.cols;   // (m: the mean of g n)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t col = (c * T + t) * 8u;
            const Eight s = widen8<ST>(rx[c]), d = widen8<DT>(rd[c]);
            Eight more = {}, dx;
            if (args.dsum != nullptr) more = widen8<ST>(rs[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = s.v[i] * r;
                dw[c].v[i] = __builtin_fmaf(d.v[i], n, dw[c].v[i]);
                dx.v[i] = __builtin_fmaf(__builtin_fmaf(-n, m, d.v[i] * w[c].v[i]), r, more.v[i]);
            }
            if (col < args.cols) store_raw8<ST>(args.dx, row, args.cols, col, args.cols, round8<ST>(dx));
        }
    }
    if constexpr (G > 1) {   // the groups' sums one after the other
#pragma unroll
        for (int k = 0; k < G; ++k) {
            if (g == (uint32_t)k) {
#pragma unroll
                for (int c = 0; c < CH; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float &at = sums[(c * 8 + i) * T + t];
                        if (k > 0) dw[c].v[i] += at;
                        if (k < G - 1) at = dw[c].v[i];
                    }
            }
            if (k < G - 1) __syncthreads();
        }
        if (g != G - 1u) return;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const uint32_t col = (c * T + t) * 8u;
        if (col < args.cols) store_raw8<0>(args.part, blockIdx.x, args.cols, col, args.cols, round8<0>(dw[c]));
    }
}

// dw: the parts' sums.  32 columns a workgroup, 32 threads for each.
template <uint32_t DT>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const NormBackwardArgs args)
{
    __shared__ float sums[32][33];
    const uint32_t c = threadIdx.x & 31u, p = threadIdx.x >> 5, col = blockIdx.x * 32u + c;
    float v = 0.f;
    if (col < args.cols) {
#pragma unroll 8
        for (uint32_t i = p; i < args.parts; i += 32u) v += args.part[(size_t)i * args.cols + col];
    }
    sums[p][c] = v;
    __syncthreads();
    v = sums[c][p];   // (lane c: part c of column p)
#pragma unroll
    for (int by = 16; by > 0; by >>= 1) v += __shfl_xor(v, by, 32);
    const uint32_t at = blockIdx.x * 32u + p;
    if (c != 0 || at >= args.cols) return;
    if (args.weightType != DT) ((float *)args.dw)[at] = v;
    else if constexpr (DT == 0) ((float *)args.dw)[at] = v;
    else if constexpr (DT == DT_BF16) ((__bf16 *)args.dw)[at] = (__bf16)v;
    else ((_Float16 *)args.dw)[at] = (_Float16)v;
}

template <uint32_t DT, uint32_t RT>
static int launch_norm_types(const NormArgs &args, hipStream_t stream)
{
    NormArgs a = args;
    const uint64_t rows = a.rows;
    auto go = [&](auto kernel, uint64_t wgs, uint32_t threads) {
        a.runs = a.q != nullptr && wgs >= 1024;
        if (a.runs) wgs = (wgs + 8 * kRun - 1) / (8 * kRun) * (8 * kRun);
        hipLaunchKernelGGL(kernel, grid_of(wgs, threads), dim3(threads), 0, stream, a);
        return (int)hipGetLastError();
    };
    if (a.cols <= 512) return go(rms_norm_kernel<DT, RT, 64, 1>, (rows + 3) / 4, 256);
    if (a.cols <= 1024) return go(rms_norm_kernel<DT, RT, 64, 2>, (rows + 3) / 4, 256);
    if (a.cols <= 2048) return go(rms_norm_kernel<DT, RT, 256, 1>, rows, 256);
    if (a.cols <= 4096) return go(rms_norm_kernel<DT, RT, 256, 2>, rows, 256);
    if (a.cols <= 8192) return go(rms_norm_kernel<DT, RT, 256, 4>, rows, 256);
    return go(rms_norm_kernel<DT, RT, 1024, 2>, rows, 1024);
}

template <uint32_t DT>
static int launch_norm_type(const NormArgs &a, uint32_t residualType, hipStream_t stream)
{
    if (residualType == DT_NONE) return launch_norm_types<DT, DT_NONE>(a, stream);
    if (residualType == DT) return launch_norm_types<DT, DT>(a, stream);
    return launch_norm_types<DT, 0>(a, stream);
}

// residualType: DT_NONE, type or 0
int launch_norm(uint32_t type, uint32_t residualType, const NormArgs &a, void *stream)
{
    if (type == DT_F16) return launch_norm_type<DT_F16>(a, residualType, (hipStream_t)stream);
    if (type == DT_BF16) return launch_norm_type<DT_BF16>(a, residualType, (hipStream_t)stream);
    return launch_norm_type<0>(a, residualType, (hipStream_t)stream);
}

// Threads of a row and of a workgroup, and how many workgroups share the rows, each with a part of dw of its own: 512 of 512 threads, two to a CU; 256 of 1024, whose rows'
// sums meet in LDS before they are a part, where there are many long rows (us: 8192 rows of 8192 110 / 106, 16384 of 4096 107 / 104; 32 of 4096 6.3 / 7.6, 8192 of 2048 31 / 33).
struct BackwardShape {
    uint32_t row, wg, parts;
};
static BackwardShape backward_shape(uint32_t rows, uint32_t cols)
{
    const uint32_t row = cols <= 1024 ? 64u : cols <= 2048 ? 128u : cols <= 4096 ? 256u : cols <= 8192 ? 512u : 1024u;
    const uint32_t wg = cols > 8192 || (cols > 2048 && rows >= 2048) ? 1024u : 512u, each = wg / row, most = 262144u / wg, turns = rows / each + (rows % each != 0);
    return {row, wg, turns < most ? turns : most};
}

uint32_t norm_backward_parts(uint32_t rows, uint32_t cols) { return backward_shape(rows, cols).parts; }

template <uint32_t DT, uint32_t ST>
static int launch_backward_types(const NormBackwardArgs &a, hipStream_t stream)
{
    if (a.parts) {
        auto go = [&](auto kernel, uint32_t threads) { hipLaunchKernelGGL(kernel, dim3(a.parts), dim3(threads), 0, stream, a); };
        const BackwardShape s = backward_shape(a.rows, a.cols);
        if (s.row == 64) go(rms_norm_backward_kernel<DT, ST, 64, 512>, 512);
        else if (s.row == 128) go(rms_norm_backward_kernel<DT, ST, 128, 512>, 512);
        else if (s.row == 256 && s.wg == 512) go(rms_norm_backward_kernel<DT, ST, 256, 512>, 512);
        else if (s.row == 256) go(rms_norm_backward_kernel<DT, ST, 256, 1024>, 1024);
        else if (s.row == 512 && s.wg == 512) go(rms_norm_backward_kernel<DT, ST, 512, 512>, 512);
        else if (s.row == 512) go(rms_norm_backward_kernel<DT, ST, 512, 1024>, 1024);
        else go(rms_norm_backward_kernel<DT, ST, 1024, 1024>, 1024);
        const int e = (int)hipGetLastError();
        if (e) return e;
    }
    hipLaunchKernelGGL((rms_norm_dw_kernel<DT>), dim3((a.cols + 31u) / 32u), dim3(1024), 0, stream, a);
    return (int)hipGetLastError();
}

template <uint32_t DT>
static int launch_backward_type(const NormBackwardArgs &a, bool wide, hipStream_t stream)
{
    return wide ? launch_backward_types<DT, 0>(a, stream) : launch_backward_types<DT, DT>(a, stream);
}

// type: of dy; wide: x, dsum and dx are fp32 all the same
int launch_norm_backward(uint32_t type, bool wide, const NormBackwardArgs &a, void *stream)
{
    if (type == DT_F16) return launch_backward_type<DT_F16>(a, wide, (hipStream_t)stream);
    if (type == DT_BF16) return launch_backward_type<DT_BF16>(a, wide, (hipStream_t)stream);
    return launch_backward_type<0>(a, true, (hipStream_t)stream);
}

}  // namespace catcoc
