// C ABI of the products in 8-bit floating point with block scales, of those whose rows come in groups, and of the quantizer: checks of arguments and the
// choice of kernel.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "api_status.h"
#include "ragged_args.h"

namespace catcoc {
int launch_quantize(uint32_t dtype, const QuantArgs &a, bool blocks, bool gated, void *stream);
int launch_ragged_tile(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, uint32_t wgs, void *stream);
int launch_ragged_checked(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, uint32_t wgs, void *stream);
}

using namespace catcoc;

namespace {

constexpr uint32_t kMaxWidth = 1u << 22;   // a tile's rows are addressed with 32-bit byte offsets
constexpr uint64_t kMaxWgs = 0x7fffffffull;

uint64_t cdiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Most row tiles of height bx that `groups` groups of together `rows` rows can have, whatever their ends (rows past the last group count as one more).
uint64_t most_row_tiles(const RaggedArgs &a, uint64_t bx)
{
    if (a.ends == nullptr) return cdiv(a.rows, bx);
    const uint64_t some = a.rows < a.groups + 1ull ? a.rows : a.groups + 1ull;
    return (a.rows - some) / bx + some;
}

int check_sizes(uint64_t rows, uint32_t k, uint32_t n, uint32_t groups)
{
    if (k == 0 || n == 0) return api_fail(E_SHAPE, "empty problem n=%u k=%u", n, k);
    if (k >= kMaxWidth || n >= kMaxWidth) return api_fail(E_SHAPE, "n=%u and k=%u must be below %u", n, k, kMaxWidth);
    if (rows > 0x7fffffffull) return api_fail(E_SHAPE, "%llu rows: fewer than 2^31 are supported", (unsigned long long)rows);
    if (groups == 0 || groups > 65536u) return api_fail(E_SHAPE, "%u groups out of range 1..65536", groups);
    return 0;
}

bool is16(uint32_t dt) { return dt == FP16 || dt == BF16; }

// Rows of both operands start on 4 bytes, as the copies that go straight to LDS need it.
bool rows_on_words(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw)
{
    const uint64_t es = dtype == DT_F8 ? 1 : 2;
    return ((uintptr_t)a.x | (uintptr_t)a.w) % 4 == 0 && a.k * es % 4 == 0 && ((!kn && !dw) || a.n * es % 4 == 0);
}

void run(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, void *stream)
{
    const bool tile = rows_on_words(dtype, a, kn, dw) && (dw || a.rows > 32ull * a.groups);
    const uint64_t bx = tile ? 256 : 64, nt = cdiv(a.n, bx);
    // weight gradient on large tiles: eighths of every group's tiles, dealt out to one workgroup a CU
    const uint64_t wgs = dw && tile ? std::min<uint64_t>(256, a.groups * cdiv(cdiv(a.k, bx) * nt, 8) * 8) : dw ? a.groups * cdiv(a.k, bx) * nt : most_row_tiles(a, bx) * nt;
    if (wgs > kMaxWgs) { api_fail(E_SHAPE, "%llu tiles are more than one launch holds", (unsigned long long)wgs); return; }
    api_launch_info({tile ? (uint32_t)CATCOC_KERNEL_RAGGED : (uint32_t)CATCOC_KERNEL_RAGGED_CHECKED, (uint32_t)bx, (uint32_t)bx, 1, 0, 0});
    api_launched((tile ? launch_ragged_tile : launch_ragged_checked)(dtype, a, kn, dw, (uint32_t)wgs, stream));
}

}  // namespace

extern "C" {

void catcoc_quantize_fp8(void *stream, const void *x, uint8_t *q, float *scale, uint32_t rows, uint32_t cols, uint32_t blockRows, uint32_t gated,
                         uint32_t dataType)
{
    if (dataType != 0 && !is16(dataType)) { api_fail(E_DTYPE, "dataType %u must be 0 (fp32), FP16 or BF16", dataType); return; }
    if (blockRows != 1 && blockRows != kScaleBlock) { api_fail(E_SHAPE, "blockRows %u must be 1 or %u", blockRows, kScaleBlock); return; }
    if (gated && blockRows != 1) { api_fail(E_SHAPE, "gated rows are quantized with blockRows 1"); return; }
    if (check_sizes(rows, cols, 1, 1)) return;
    if (rows == 0) { api_launched(0); return; }
    if (!x || !q || !scale) { api_fail(E_NULL, "x, q and scale must be non-NULL"); return; }
    QuantArgs a{x, q, scale, rows, cols};
    if (cdiv(rows, 4) * cdiv(cols, kScaleBlock) > kMaxWgs) { api_fail(E_SHAPE, "%u x %u are more blocks than one launch holds", rows, cols); return; }
    api_launched(launch_quantize(dataType, a, blockRows != 1, gated != 0, stream));
}

void catcoc_fp8_matmul_allreduce(void *stream, const uint8_t *x1, const uint8_t *x2, const float *scale_x1, const float *scale_x2, void *c,
                                 uint8_t *symmetricPtr, uint32_t m, uint32_t n, uint32_t k, uint32_t outDataType)
{
    if (!is16(outDataType)) { api_fail(E_DTYPE, "outDataType %u must be FP16 (1) or BF16 (27)", outDataType); return; }
    if (check_sizes(m, k, n, 1)) return;
    RaggedArgs a{};
    if (const auto *d = (const CatcocSymmetricDesc *)symmetricPtr) {
        if (d->magic != CATCOC_DESC_MAGIC) { api_fail(E_DESC, "symmetricPtr does not point at a CatcocSymmetricDesc (bad magic)"); return; }
        if (d->rankSize == 0 || d->rankSize > CATCOC_MAX_RANKS || d->rankIdx >= d->rankSize) {
            api_fail(E_RANK, "rankIdx %u / rankSize %u out of range (1..%d ranks)", d->rankIdx, d->rankSize, CATCOC_MAX_RANKS);
            return;
        }
        a.nPeers = d->rankSize - 1u;
        a.peerLd = d->peerLd;
        if (a.nPeers && d->peerLd < (int64_t)n) { api_fail(E_DESC, "peerLd %lld < n %u", (long long)d->peerLd, n); return; }
        if (d->peerRowOffset < 0) { api_fail(E_DESC, "peerRowOffset must be >= 0"); return; }
        for (uint32_t s = 0; s < a.nPeers; ++s) {
            if (d->peers[s] == nullptr && m != 0) { api_fail(E_NULL, "reduce needs %u staged peer partials; peers[%u] is NULL", a.nPeers, s); return; }
            a.peers[s] = (const float *)d->peers[s] + d->peerRowOffset * d->peerLd;
        }
    }
    if (m == 0) { api_launched(0); return; }
    if (!x1 || !x2 || !scale_x1 || !scale_x2 || !c) { api_fail(E_NULL, "x1, x2, scale_x1, scale_x2 and c must be non-NULL"); return; }
    a.x = x1;
    a.w = x2;
    a.out = c;
    a.sx = scale_x1;
    a.sw = scale_x2;
    a.rows = m;
    a.k = k;
    a.n = n;
    a.groups = 1;
    a.outType = outDataType;
    run(DT_F8, a, false, false, stream);
}

void catcoc_grouped_matmul(void *stream, uint32_t dataType, const void *x, const void *w, const int32_t *groupEnds, void *out, uint32_t rows, uint32_t n,
                           uint32_t k, uint32_t groups, uint32_t transB)
{
    if (!is16(dataType)) { api_fail(E_DTYPE, "dataType %u must be FP16 (1) or BF16 (27)", dataType); return; }
    if (check_sizes(rows, k, n, groups)) return;
    if (rows == 0) { api_launched(0); return; }
    if (!x || !w || !groupEnds || !out) { api_fail(E_NULL, "x, w, groupEnds and out must be non-NULL"); return; }
    RaggedArgs a{};
    a.x = x;
    a.w = w;
    a.out = out;
    a.ends = groupEnds;
    a.rows = rows;
    a.k = k;
    a.n = n;
    a.groups = groups;
    a.outType = dataType;
    run(dataType, a, transB == 0, false, stream);
}

void catcoc_grouped_matmul_dw(void *stream, uint32_t dataType, const void *x, const void *dy, const int32_t *groupEnds, void *dw, uint32_t rows, uint32_t n,
                              uint32_t k, uint32_t groups, uint32_t transB, uint32_t outDataType)
{
    if (!is16(dataType)) { api_fail(E_DTYPE, "dataType %u must be FP16 (1) or BF16 (27)", dataType); return; }
    if (outDataType != 0 && !is16(outDataType)) { api_fail(E_DTYPE, "outDataType %u must be 0 (fp32), FP16 or BF16", outDataType); return; }
    if (check_sizes(rows, k, n, groups)) return;
    if (((!x || !dy) && rows != 0) || !groupEnds || !dw) { api_fail(E_NULL, "x, dy, groupEnds and dw must be non-NULL"); return; }
    RaggedArgs a{};
    a.x = transB ? dy : x;      // dw^T is the same sum with its operands' places changed
    a.w = transB ? x : dy;
    a.out = dw;
    a.ends = groupEnds;
    a.rows = rows;
    a.k = transB ? n : k;
    a.n = transB ? k : n;
    a.groups = groups;
    a.outType = outDataType;
    run(dataType, a, false, true, stream);
}

void catcoc_grouped_fp8_matmul(void *stream, const uint8_t *x, const uint8_t *w, const float *scale_x, const float *scale_w, const int32_t *groupEnds,
                               void *out, uint32_t rows, uint32_t n, uint32_t k, uint32_t groups, uint32_t outDataType)
{
    if (!is16(outDataType)) { api_fail(E_DTYPE, "outDataType %u must be FP16 (1) or BF16 (27)", outDataType); return; }
    if (check_sizes(rows, k, n, groups)) return;
    if (rows == 0) { api_launched(0); return; }
    if (!x || !w || !scale_x || !scale_w || !groupEnds || !out) { api_fail(E_NULL, "x, w, scale_x, scale_w, groupEnds and out must be non-NULL"); return; }
    RaggedArgs a{};
    a.x = x;
    a.w = w;
    a.out = out;
    a.sx = scale_x;
    a.sw = scale_w;
    a.ends = groupEnds;
    a.rows = rows;
    a.k = k;
    a.n = n;
    a.groups = groups;
    a.outType = outDataType;
    run(DT_F8, a, false, false, stream);
}

}  // extern "C"
