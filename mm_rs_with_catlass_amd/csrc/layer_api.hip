// C ABI of the operators around a layer of experts (norms, the router, rows to their experts and back): checks of arguments.
#include <hip/hip_runtime.h>

#include <math.h>

#include <initializer_list>

#include "api_status.h"
#include "layer_args.h"

namespace catcoc {
int launch_norm(uint32_t type, uint32_t residualType, const NormArgs &a, void *stream);
uint32_t norm_backward_parts(uint32_t rows, uint32_t cols);
int launch_norm_backward(uint32_t type, bool wide, const NormBackwardArgs &a, void *stream);
bool can_route(uint32_t experts, uint32_t top, uint32_t groups);
int launch_route(const RouteArgs &a, void *stream);
int launch_route_backward(const RouteArgs &a, void *stream);
bool sort_counts_first(uint32_t rows, uint32_t experts);
uint32_t sort_blocks(uint32_t rows, uint32_t experts);
int launch_sort(uint32_t choiceBits, SortArgs a, void *stream);
int launch_spread_rows(uint32_t valueBytes, const RowsArgs &a, void *stream);
int launch_gather_rows(uint32_t type, const RowsArgs &a, void *stream);
int launch_gather_rows_backward(uint32_t type, const RowsArgs &a, void *stream);
}

using namespace catcoc;

namespace {

constexpr uint32_t kMostRows = 0x7fffffffu, kMaxWidth = 1u << 22;
constexpr uint64_t kMaxWgs = 1ull << 29;   // of four waves: their number fits 32 bits

bool is16(uint32_t dt) { return dt == FP16 || dt == BF16; }
bool is_float(uint32_t dt) { return dt == 0 || is16(dt); }

int check_norm(uint32_t rows, uint32_t cols, uint32_t type, uint32_t otherType, uint32_t weightType, const char *other)
{
    if (!is_float(type)) return api_fail(E_DTYPE, "dataType %u must be 0 (fp32), FP16 or BF16", type);
    if (otherType != 0 && otherType != type) return api_fail(E_DTYPE, "%s %u must be 0 (fp32) or dataType", other, otherType);
    if (weightType != 0 && weightType != type) return api_fail(E_DTYPE, "weightType %u must be 0 (fp32) or dataType", weightType);
    if (cols == 0 || cols > kMostNormCols) return api_fail(E_SHAPE, "%u columns out of range 1..%u", cols, kMostNormCols);
    if (rows > kMostRows) return api_fail(E_SHAPE, "%u rows: fewer than 2^31 are supported", rows);
    return 0;
}

int check_route(const CatcocRouting *how, uint32_t tokens, uint32_t experts, uint32_t top, uint32_t type)
{
    if (how == nullptr) return api_fail(E_NULL, "how must be non-NULL");
    if (!is_float(type)) return api_fail(E_DTYPE, "dataType %u must be 0 (fp32), FP16 or BF16", type);
    if (tokens > kMostRows) return api_fail(E_SHAPE, "%u tokens: fewer than 2^31 are supported", tokens);
    if (experts == 0 || experts > kMostExperts) return api_fail(E_SHAPE, "%u experts out of range 1..%u", experts, kMostExperts);
    if (top == 0 || top > kMostTop || top > experts) return api_fail(E_SHAPE, "top %u out of range 1..%u, and of %u experts", top, kMostTop, experts);
    if (how->score > CATCOC_SCORE_SIGMOID) return api_fail(E_SHAPE, "score %u must be CATCOC_SCORE_SOFTMAX (0) or CATCOC_SCORE_SIGMOID (1)", how->score);
    if (!isfinite(how->scale)) return api_fail(E_SHAPE, "scale must be finite");
    return 0;
}

int check_rows(uint32_t tokens, uint32_t top, uint32_t cols)
{
    if (cols == 0 || cols >= kMaxWidth) return api_fail(E_SHAPE, "%u columns out of range 1..%u", cols, kMaxWidth - 1u);
    if (top == 0 || top > kMostTop) return api_fail(E_SHAPE, "top %u out of range 1..%u", top, kMostTop);
    if ((uint64_t)tokens * top > kMostRows) return api_fail(E_SHAPE, "%u tokens with %u choices each: fewer than 2^31 rows are supported", tokens, top);
    return 0;
}

// An operand's memory.
struct Memory {
    const char *name;
    const void *at;
    uint64_t bytes;
    int like = 0;   // an output may take the place of an operand that has this number too, the same rows of values of one size: who writes a row has read it before, and nobody else does
};

int check_apart(std::initializer_list<Memory> outs, std::initializer_list<Memory> ins)
{
    auto overlap = [](const Memory &a, const Memory &b) {
        const uintptr_t x = (uintptr_t)a.at, y = (uintptr_t)b.at;
        return a.at && b.at && a.bytes && b.bytes && x < y + b.bytes && y < x + a.bytes;
    };
    for (const Memory *o = outs.begin(); o != outs.end(); ++o) {
        for (const Memory &i : ins)
            if (overlap(*o, i) && !(o->like && o->like == i.like && o->at == i.at && o->bytes == i.bytes)) return api_fail(E_SHAPE, "%s lies in the memory of %s", o->name, i.name);
        for (const Memory *p = outs.begin(); p != o; ++p)
            if (overlap(*o, *p)) return api_fail(E_SHAPE, "%s lies in the memory of %s", o->name, p->name);
    }
    return 0;
}

uint64_t bytes_of(uint32_t dt) { return dt ? 2u : 4u; }

// The most workgroups that a launch can have: a wave for each KiB of a row.
int check_pieces(uint32_t tokens, uint64_t rowBytes)
{
    if ((tokens * ((rowBytes + 1023u) / 1024u) + 3u) / 4u > kMaxWgs) return api_fail(E_SHAPE, "%u tokens of %llu bytes are more than one launch holds", tokens, (unsigned long long)rowBytes);
    return 0;
}

}  // namespace

extern "C" {

void catcoc_rms_norm(void *stream, const void *x, const void *residual, const void *weight, void *out, void *sum, uint8_t *q, float *scale, uint32_t rows,
                     uint32_t cols, float eps, uint32_t dataType, uint32_t residualType, uint32_t weightType)
{
    if (check_norm(rows, cols, dataType, residual ? residualType : dataType, weightType, "residualType")) return;
    if (!(eps >= 0) || !isfinite(eps)) { api_fail(E_SHAPE, "eps must be finite and not negative"); return; }
    if (rows == 0) { api_launched(0); return; }   // (before the pointers: those of nothing may be NULL)
    if (!out && !q) { api_fail(E_NULL, "out or q must be non-NULL"); return; }
    if (!q != !scale) { api_fail(E_NULL, "q and scale come together"); return; }
    if (!residual != !sum) { api_fail(E_NULL, "residual and sum come together"); return; }
    if (!x || !weight) { api_fail(E_NULL, "x and weight must be non-NULL"); return; }
    if ((cols <= 1024 ? (rows + 3ull) / 4 : rows) > 2 * kMaxWgs) { api_fail(E_SHAPE, "%u rows of %u columns are more than one launch holds", rows, cols); return; }
    const uint64_t values = (uint64_t)rows * cols;
    if (check_apart({{"out", out, values * bytes_of(dataType), 1}, {"sum", sum, values * bytes_of(residualType), 1}, {"q", q, values}, {"scale", scale, (cols + 127ull) / 128u * rows * 4u}},
                    {{"x", x, values * bytes_of(dataType), 1}, {"residual", residual, values * bytes_of(residualType), 1}, {"weight", weight, cols * bytes_of(weightType)}}))
        return;
    NormArgs a{x, residual, weight, out, sum, q, scale, rows, cols, eps, weightType, 0};
    api_launched(launch_norm(dataType, residual ? residualType : DT_NONE, a, stream));
}

uint64_t catcoc_rms_norm_backward_workspace_size(uint32_t rows, uint32_t cols)
{
    return cols == 0 || cols > kMostNormCols ? 0 : (uint64_t)norm_backward_parts(rows, cols) * cols * 4u;
}

void catcoc_rms_norm_backward(void *stream, const void *dy, const void *x, const void *weight, const void *dsum, void *dx, void *dw, void *workspace,
                              uint64_t workspaceBytes, uint32_t rows, uint32_t cols, float eps, uint32_t dataType, uint32_t sumType, uint32_t weightType)
{
    if (check_norm(rows, cols, dataType, sumType, weightType, "sumType")) return;
    if (!(eps >= 0) || !isfinite(eps)) { api_fail(E_SHAPE, "eps must be finite and not negative"); return; }
    if (!dw || (rows != 0 && (!dy || !x || !weight || !dx || !workspace))) { api_fail(E_NULL, "dy, x, weight, dx, dw and workspace must be non-NULL"); return; }
    if (workspaceBytes < catcoc_rms_norm_backward_workspace_size(rows, cols)) {
        api_fail(E_WORKSPACE, "workspace holds %llu bytes, the launch needs %llu", (unsigned long long)workspaceBytes,
                 (unsigned long long)catcoc_rms_norm_backward_workspace_size(rows, cols));
        return;
    }
    if ((uintptr_t)workspace % 4 != 0) { api_fail(E_WORKSPACE, "workspace must be 4-byte aligned"); return; }
    const uint64_t values = (uint64_t)rows * cols;
    if (check_apart({{"dx", dx, values * bytes_of(sumType), 1}, {"dw", dw, cols * bytes_of(weightType), 2}, {"workspace", workspace, catcoc_rms_norm_backward_workspace_size(rows, cols)}},
                    {{"dy", dy, values * bytes_of(dataType), 1}, {"x", x, values * bytes_of(sumType), 1}, {"weight", weight, cols * bytes_of(weightType), 2},
                     {"dsum", dsum, values * bytes_of(sumType), 1}}))
        return;
    NormBackwardArgs a{dy, x, weight, dsum, dx, dw, (float *)workspace, rows, cols, norm_backward_parts(rows, cols), eps, weightType};
    api_launched(launch_norm_backward(dataType, sumType == 0, a, stream));
}

void catcoc_route(void *stream, const void *logits, const float *bias, int32_t *choice, float *share, const CatcocRouting *how, uint32_t tokens,
                  uint32_t experts, uint32_t top, uint32_t dataType)
{
    if (check_route(how, tokens, experts, top, dataType)) return;
    const uint32_t groups = how->groups ? how->groups : 1u, topGroups = how->topGroups ? how->topGroups : groups, groupTop = how->groupTop ? how->groupTop : 1u;
    if (groups > experts || experts % groups != 0) { api_fail(E_SHAPE, "%u experts do not come in %u groups of one size", experts, groups); return; }
    if (topGroups > groups) { api_fail(E_SHAPE, "topGroups %u out of range 1..%u", topGroups, groups); return; }
    if (groupTop > 2) { api_fail(E_SHAPE, "groupTop %u must be 1 or 2", groupTop); return; }
    if ((uint64_t)topGroups * (experts / groups) < top) { api_fail(E_SHAPE, "%u groups of %u experts have fewer than top %u", topGroups, experts / groups, top); return; }
    const uint32_t laid = topGroups < groups ? groups : 1u;   // (all groups are taken: there might as well be none)
    if (!can_route(experts, top, laid)) { api_fail(E_SHAPE, "%u groups: at most 64 are supported", groups); return; }
    if (tokens == 0) { api_launched(0); return; }
    if (!logits || !choice || !share) { api_fail(E_NULL, "logits, choice and share must be non-NULL"); return; }
    const uint64_t scores = (uint64_t)tokens * experts, choices = (uint64_t)tokens * top;
    if (check_apart({{"choice", choice, choices * 4u}, {"share", share, choices * 4u}}, {{"logits", logits, scores * bytes_of(dataType)}, {"bias", bias, experts * 4ull}})) return;
    RouteArgs a{};
    a.logits = logits;
    a.bias = bias;
    a.choice = choice;
    a.share = share;
    a.tokens = tokens;
    a.experts = experts;
    a.top = top;
    a.type = dataType;
    a.sigmoid = how->score == CATCOC_SCORE_SIGMOID;
    a.groups = laid;
    a.topGroups = laid == 1 ? 1 : topGroups;
    a.groupTop = laid == 1 ? 1 : groupTop;
    a.renormalize = how->renormalize != 0;
    a.scale = how->scale;
    api_launched(launch_route(a, stream));
}

void catcoc_route_backward(void *stream, const float *dshare, const void *logits, const int32_t *choice, void *dlogits, const CatcocRouting *how, uint32_t tokens,
                           uint32_t experts, uint32_t top, uint32_t dataType)
{
    if (check_route(how, tokens, experts, top, dataType)) return;
    if (tokens == 0) { api_launched(0); return; }
    if (!dshare || !logits || !choice || !dlogits) { api_fail(E_NULL, "dshare, logits, choice and dlogits must be non-NULL"); return; }
    const uint64_t bytes = (uint64_t)tokens * experts * bytes_of(dataType), choices = (uint64_t)tokens * top;
    if (check_apart({{"dlogits", dlogits, bytes, 1}}, {{"logits", logits, bytes, 1}, {"dshare", dshare, choices * 4u}, {"choice", choice, choices * 4u}})) return;
    RouteArgs a{};
    a.logits = logits;
    a.dshare = dshare;
    a.chosen = choice;
    a.dlogits = dlogits;
    a.tokens = tokens;
    a.experts = experts;
    a.top = top;
    a.type = dataType;
    a.sigmoid = how->score == CATCOC_SCORE_SIGMOID;
    a.renormalize = how->renormalize != 0;
    a.scale = how->scale;
    api_launched(launch_route_backward(a, stream));
}

uint64_t catcoc_sort_by_expert_workspace_size(uint32_t rows, uint32_t experts)
{
    return sort_counts_first(rows, experts) ? (uint64_t)sort_blocks(rows, experts) * experts * 4u : 0u;
}

void catcoc_sort_by_expert(void *stream, const void *choice, int32_t *order, int32_t *back, int32_t *ends, void *workspace, uint64_t workspaceBytes, uint32_t rows,
                           uint32_t experts, uint32_t choiceBits)
{
    if (choiceBits != 32 && choiceBits != 64) { api_fail(E_DTYPE, "choiceBits %u must be 32 or 64", choiceBits); return; }
    if (rows > kMostRows) { api_fail(E_SHAPE, "%u rows: fewer than 2^31 are supported", rows); return; }
    if (experts == 0 || experts > kMostExperts) { api_fail(E_SHAPE, "%u experts out of range 1..%u", experts, kMostExperts); return; }
    if (!ends || (rows != 0 && (!choice || !order || !back))) { api_fail(E_NULL, "choice, order, back and ends must be non-NULL"); return; }
    const uint64_t need = catcoc_sort_by_expert_workspace_size(rows, experts);
    if (need && (!workspace || workspaceBytes < need)) {
        api_fail(E_WORKSPACE, "workspace holds %llu bytes, the launch needs %llu", (unsigned long long)(workspace ? workspaceBytes : 0), (unsigned long long)need);
        return;
    }
    if ((uintptr_t)workspace % 4 != 0) { api_fail(E_WORKSPACE, "workspace must be 4-byte aligned"); return; }
    if (check_apart({{"order", order, rows * 4ull}, {"back", back, rows * 4ull}, {"ends", ends, experts * 4ull}, {"workspace", workspace, need}},
                    {{"choice", choice, (uint64_t)rows * (choiceBits / 8u)}}))
        return;
    SortArgs a{};
    a.choice = choice;
    a.order = order;
    a.back = back;
    a.ends = ends;
    a.part = (uint32_t *)workspace;
    a.rows = rows;
    a.experts = experts;
    api_launched(launch_sort(choiceBits, a, stream));
}

void catcoc_spread_rows(void *stream, const void *x, const float *scale, const int32_t *back, void *out, float *outScale, uint32_t tokens, uint32_t top, uint32_t cols,
                        uint32_t valueBytes)
{
    if (valueBytes != 1 && valueBytes != 2 && valueBytes != 4) { api_fail(E_DTYPE, "valueBytes %u must be 1, 2 or 4", valueBytes); return; }
    if (check_rows(tokens, top, cols) || check_pieces(tokens, (uint64_t)cols * valueBytes)) return;
    if (tokens == 0) { api_launched(0); return; }
    if (!scale != !outScale) { api_fail(E_NULL, "scale and outScale come together"); return; }
    if (scale && valueBytes != 1) { api_fail(E_DTYPE, "scales come with values of 1 byte (got %u)", valueBytes); return; }
    if (!x || !back || !out) { api_fail(E_NULL, "x, back and out must be non-NULL"); return; }
    const uint64_t rows = (uint64_t)tokens * top, blocks = (cols + 127u) / 128u;
    if (check_apart({{"out", out, rows * cols * valueBytes}, {"outScale", outScale, rows * blocks * 4u}},
                    {{"x", x, (uint64_t)tokens * cols * valueBytes}, {"scale", scale, tokens * blocks * 4u}, {"back", back, rows * 4u}}))
        return;
    RowsArgs a{};
    a.x = x;
    a.scale = scale;
    a.back = back;
    a.out = out;
    a.outScale = outScale;
    a.tokens = tokens;
    a.top = top;
    a.cols = cols;
    api_launched(launch_spread_rows(valueBytes, a, stream));
}

void catcoc_gather_rows(void *stream, const void *y, const int32_t *back, const float *share, void *out, uint32_t tokens, uint32_t top, uint32_t cols,
                        uint32_t dataType)
{
    if (!is_float(dataType)) { api_fail(E_DTYPE, "dataType %u must be 0 (fp32), FP16 or BF16", dataType); return; }
    if (check_rows(tokens, top, cols) || check_pieces(tokens, cols * 2ull)) return;
    if (tokens == 0) { api_launched(0); return; }
    if (!y || !back || !out) { api_fail(E_NULL, "y, back and out must be non-NULL"); return; }
    const uint64_t rows = (uint64_t)tokens * top;
    if (check_apart({{"out", out, (uint64_t)tokens * cols * bytes_of(dataType)}}, {{"y", y, rows * cols * bytes_of(dataType)}, {"back", back, rows * 4u}, {"share", share, rows * 4u}})) return;
    RowsArgs a{};
    a.y = y;
    a.back = back;
    a.share = share;
    a.out = out;
    a.tokens = tokens;
    a.top = top;
    a.cols = cols;
    api_launched(launch_gather_rows(dataType, a, stream));
}

void catcoc_gather_rows_backward(void *stream, const void *dout, const void *y, const int32_t *back, const float *share, void *dy, float *dshare, uint32_t tokens,
                                 uint32_t top, uint32_t cols, uint32_t dataType)
{
    if (!is_float(dataType)) { api_fail(E_DTYPE, "dataType %u must be 0 (fp32), FP16 or BF16", dataType); return; }
    if (check_rows(tokens, top, cols) || check_pieces(tokens, 1024)) return;
    if (tokens == 0) { api_launched(0); return; }
    if (!dout || !back || !share) { api_fail(E_NULL, "dout, back and share must be non-NULL"); return; }
    if (!dy && !dshare) { api_fail(E_NULL, "dy or dshare must be non-NULL"); return; }
    if (!y != !dshare) { api_fail(E_NULL, "y and dshare come together"); return; }
    const uint64_t rows = (uint64_t)tokens * top;
    if (check_apart({{"dy", dy, rows * cols * bytes_of(dataType), 1}, {"dshare", dshare, rows * 4u, 2}},
                    {{"dout", dout, (uint64_t)tokens * cols * bytes_of(dataType)}, {"y", y, rows * cols * bytes_of(dataType), 1}, {"back", back, rows * 4u}, {"share", share, rows * 4u, 2}}))
        return;
    RowsArgs a{};
    a.x = dout;
    a.y = y;
    a.back = back;
    a.share = share;
    a.out = dy;
    a.dshare = dshare;
    a.tokens = tokens;
    a.top = top;
    a.cols = cols;
    api_launched(launch_gather_rows_backward(dataType, a, stream));
}

}  // extern "C"
