// Arguments of the kernels around a layer of experts: the norm in front of it, the router, the rows' way to their experts and back.
#pragma once
#include <stdint.h>

#include "ragged_args.h"

namespace catcoc {

constexpr uint32_t kMostNormCols = 16384;     // of a norm's rows: a row is held in registers
constexpr uint32_t kMostExperts = 1024, kMostTop = 64;
constexpr uint32_t DT_NONE = 0xffffffffu;     // no residual

struct NormArgs {
    const void *x, *residual, *weight;
    void *out;                   // NULL: not wanted
    void *sum;                   // x + residual, of the residual's type
    unsigned char *q;            // NULL: not wanted
    float *scale;                // [column blocks, rows]
    uint32_t rows, cols;
    float eps;
    uint32_t weightType;         // 0 (fp32), or the type of x
    uint32_t runs;               // workgroups are dealt out in runs (run_place)
};

struct NormBackwardArgs {
    const void *dy, *x, *weight, *dsum;   // dsum: NULL or a gradient that is added to dx
    void *dx, *dw;
    float *part;                 // [parts, cols] sums of the weight gradient
    uint32_t rows, cols, parts;
    float eps;
    uint32_t weightType;         // 0 (fp32), or the type of dy
};

struct RouteArgs {
    const void *logits;          // [tokens, experts]
    const float *bias;           // [experts] or NULL
    int32_t *choice;             // [tokens, top]
    float *share;
    const float *dshare;         // backward
    const int32_t *chosen;
    void *dlogits;
    uint32_t tokens, experts, top, type;
    uint32_t sigmoid, groups, topGroups, groupTop, renormalize;
    float scale;
    uint32_t groupLanes;         // lanes of a group's experts, a power of two
};

struct SortArgs {
    const void *choice;          // [rows], 32 or 64 bits
    int32_t *order, *back, *ends;
    uint32_t *part;              // [blocks, experts] how many rows of a block go to each expert; NULL: each block counts for itself
    uint32_t rows, experts, blocks, perBlock;
};

struct RowsArgs {
    const void *x;               // [tokens, cols]; backward: the gradient that comes in
    const void *y;               // [tokens * top, cols]; backward: NULL without dshare
    const float *scale;          // spread: [column blocks, tokens] or NULL
    const float *share;          // [tokens, top] or NULL (ones)
    const int32_t *back;         // [tokens, top]
    void *out;                   // spread, backward: [tokens * top, cols], backward NULL where it is not wanted; gather: [tokens, cols]
    float *outScale;             // spread: [column blocks, tokens * top]
    float *dshare;               // backward: [tokens, top], NULL where it is not wanted
    uint32_t tokens, top, cols;
    uint32_t scaleWgs;           // spread: how many workgroups are the scales'
};

}  // namespace catcoc
