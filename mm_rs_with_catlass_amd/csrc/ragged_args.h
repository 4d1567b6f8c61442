// Arguments of the products whose rows come in groups (one matrix per group), of those in 8-bit floating point with block scales, and of the quantizer
// in front of them; what their kernels and the host share.
#pragma once
#include <stdint.h>

#include "gemm_args.h"

namespace catcoc {

enum : uint32_t { DT_F8 = 36 };   // e4m3 (finite values and NaN), beside gemm_args.h's codes; a type of 0 is fp32

constexpr uint32_t kScaleBlock = 128;        // values of k that share a scale, and columns of a weight matrix that do
constexpr float kE4m3Top = 448.f;            // largest e4m3 value
constexpr float kScaleFloor = 0x1p-40f;      // a block's largest magnitude counts as at least this: no scale is zero or denormal

// y[i] = x[i] w[group of i] (+ peers), or dw[group] = sum over its rows of x[i]^T dy[i].  Group e holds rows [ends[e-1], ends[e]) of x.
struct RaggedArgs {
    const void *x;             // [rows, k]
    const void *w;             // [groups, n, k] or, kn, [groups, k, n]; weight gradient: dy [rows, n]
    void *out;                 // [rows, n]; weight gradient: [groups, k, n]
    const float *sx;           // e4m3: [k blocks, rows]
    const float *sw;           //       [groups, n blocks, k blocks]
    const int32_t *ends;       // [groups] on the GPU; NULL: one group of all rows
    const float *peers[kMaxRanks];
    int64_t peerLd;
    uint32_t nPeers;
    uint32_t rows, k, n, groups;
    uint32_t outType;          // 0 (fp32), DT_F16, DT_BF16
    uint32_t dealt;            // groups' tiles are dealt out to the XCDs (dealt_group), not a run of them to each
    uint32_t tileRows;         // large tiles: at most so many rows each, a multiple of 32 and no more than the kernel's
};

struct QuantArgs {
    const void *x;             // [rows, cols], or [rows, 2 cols] where gated
    unsigned char *q;          // [rows, cols]
    float *scale;              // [k blocks, rows]; blocks of 128 rows: [row blocks, k blocks]
    uint32_t rows, cols;
};

}  // namespace catcoc
