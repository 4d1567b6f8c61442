// C ABI of the products in 8-bit floating point with block scales, of those whose rows come in groups, and of the quantizer: checks of arguments and the
// choice of kernel.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "api_status.h"
#include "ragged_args.h"

namespace catcoc {
int launch_quantize(uint32_t dtype, const QuantArgs &a, bool blocks, bool gated, void *stream);
int launch_ragged_tile(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, uint32_t cols, uint32_t teams, uint32_t wgs, void *stream);
int launch_ragged_small(uint32_t dtype, const RaggedArgs &a, bool kn, uint32_t rows, uint32_t wgs, void *stream);
int launch_ragged_checked(uint32_t dtype, const RaggedArgs &a, bool kn, bool dw, uint32_t wgs, void *stream);
}

using namespace catcoc;

namespace {

constexpr uint32_t kMaxWidth = 1u << 22;   // a tile's rows are addressed with 32-bit byte offsets
constexpr uint64_t kMaxWgs = 0x7fffffffull;       // of a launch in two dimensions (checked products, the quantizer)

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

// The kernels that a product can run on: their tiles, and how many teams of a workgroup's waves share a tile's steps of k.
struct Choice {
    enum Kind { SMALL, TILE, CHECKED } kind;
    uint32_t rows, cols, teams;
};
constexpr Choice kChecked{Choice::CHECKED, 64, 64, 1};
constexpr Choice kSmallNk[] = {{Choice::SMALL, 16, 32, 4}, {Choice::SMALL, 32, 32, 4}};
constexpr Choice kSmallKn[] = {{Choice::SMALL, 16, 64, 4}, {Choice::SMALL, 32, 64, 4}, {Choice::SMALL, 64, 64, 4}};
constexpr Choice kTeams64{Choice::TILE, 64, 128, 2}, kTeams128{Choice::TILE, 128, 128, 2}, kTile128{Choice::TILE, 128, 128, 1}, kTile256{Choice::TILE, 256, 256, 1};
constexpr uint32_t kLeastRows = 96;   // tiles of 256 columns: 96 to 256 rows in steps of 32

// Most workgroups of a launch on kernel c: its tiles other than the checked ones lie in one dimension, which holds fewer than 2^32 threads.
uint64_t most_wgs(const Choice &c) { return c.kind == Choice::CHECKED ? kMaxWgs : 0xffffffffull / (c.kind == Choice::TILE && (c.cols == 256 || c.teams == 2) ? 512 : 256); }

// Whether each group's tiles are dealt out to all XCDs, the highest first, or every XCD gets a run of all tiles: dealt out they end together, but every XCD reads
// every group's rows, which has to be less than the matrices; runs of many groups end together by themselves.  Measured (us, run / dealt, tiles of at most 256
// rows, 16 bits): 15 groups of together 4099 rows, 3584x4096, 192 / 173; 16 of 4096, 4096x3584, 177 / 160; 24 of 6000, 4096x3584, 251 / 224; 48 of 12000, 2048x2048,
// 164 / 147; 62 of 16384, 4096x3584, 575 / 581 (160 rows); and where the rows are more than the matrices 16 of 12000, 4096x1792, 197 / 210 and 8 of 4096 59 / 65 (128 rows).
bool deal(const RaggedArgs &a) { return a.ends && a.groups <= 48 && 8ull * a.rows <= (uint64_t)std::min(a.groups, a.rows) * a.n; }

// Workgroups of a product on kernel c.
uint64_t count_wgs(const RaggedArgs &a, const Choice &c)
{
    const uint64_t wgs = most_row_tiles(a, c.rows) * cdiv(a.n, c.cols);
    return c.kind == Choice::TILE && deal(a) ? cdiv(wgs, 8) * 8 + 8 : wgs;   // (dealt out, an XCD's eighths of the groups and of the rows behind them are rounded by themselves)
}

// By what a launch is estimated to take, in us: the larger of what memory needs for each byte once (5.7 GB/ms; `reach`: over what a kernel reaches of it in several rounds) and of its
// rounds of workgroups, a quarter of the smaller, and a start.  A round costs its steps of 128 bytes of k, `step` us each with the GPU full, `few` of that with
// at most one workgroup a CU.  Fitted to, and compared on, 84 sizes that ran on all of these kernels (1 to 8192 rows of e4m3 against 2048 to 8192 columns and
// k; 64 to 16384 rows in 1 to 128 groups of 1792 to 4096 by 1792 to 8192, uneven, 16 bits either way and e4m3): for 74 of them the choice is within 7 % of the
// fastest, the worst 1.17 of it.  The constants have no other reason than that fit.  Of 48 sizes that it has not seen (1 to 12000 rows, 1 to 128 groups, k and n 512 to 6000)
// the choice is within 7 % of the fastest for 41.  The others are e4m3 with few rows a group, the further off the shorter k is, as a small tile's start counts for more than
// the estimate has it (453 rows in 128 groups of 4480x512 130 us on 16x32, 67 on 128x128; 257 in 48 of 2688x512 24.5 and 16.6; 91 in 128 of 5376x1408 128 and 104), and 16 bits with k = 512
// (11096 rows in 48 groups of 1792x512 46.6 us on 128x256, 36.3 on 256x256).  Heights: 4096 rows in 16 groups of 4096x3584 take 195 us in tiles of at most 256 rows, 177 of 192, 153 of 160, 181 of 128;
// 2400 in 8 groups of 2048x4096 49, 43, 65 and 57 (16 bits).
Choice choose(uint32_t dtype, const RaggedArgs &a, bool kn)
{
    const bool f8 = dtype == DT_F8;
    const double es = f8 ? 1 : 2, steps = (double)cdiv(a.k * (uint64_t)es, 128);
    const double active = a.ends ? std::min(a.groups, a.rows) : 1, mean = a.rows / active;
    const double mem = (active * a.k * a.n * es + a.rows * (double)a.k * es + a.rows * (double)a.n * (2.0 + 4.0 * a.nPeers)) / 5.7e6;
    const bool dealt = deal(a);
    Choice best = kChecked;   // (whose launches hold more tiles than the others')
    double least = 0;
    const bool many = (a.rows / 16.0 + a.groups + 2) * (a.n / 32.0 + 1) > 4e6;   // more tiles of 16x32 than this: each kernel's own are counted
    // Groups are taken to have 0.4, 0.6 .. 1.6 of the mean: how many tiles of at most `rows` that makes, and how high they are, in 32 rows (no less than two).
    auto row_tiles = [&](uint32_t rows, double *height) {
        double tiles = 0, high = 0;
        for (int i = a.ends ? 2 : 5; i <= (a.ends ? 8 : 5); ++i) {
            const double group = mean * i / 5, t = std::max(1.0, std::ceil(group / rows));
            tiles += t;
            high += t * std::max(2.0, std::ceil(group / t / 32));
        }
        if (height) *height = a.ends && !dealt ? 0.8 * high / tiles + 0.2 * std::min(rows / 32.0, std::max(2.0, std::ceil(mean * 1.6 / 32))) : high / tiles;   // (a round ends with its highest)
        return a.ends ? active * tiles / 7 : tiles;
    };
    auto offer = [&](const Choice &c, double start, double slots, double step, double few, double reach) {
        if (many && count_wgs(a, c) > most_wgs(c)) return;
        const double tiles = row_tiles(c.rows, nullptr) * (double)cdiv(a.n, c.cols);
        double rounds = tiles / slots;
        rounds = rounds > 4 ? rounds + 0.3 : std::ceil(rounds);
        const double work = (tiles <= 256 ? few : 1.0) * step * steps * rounds, m = mem * (tiles <= slots ? std::min(reach, 1.0) : reach);
        const double t = start + std::max(m, work) + 0.25 * std::min(m, work);
        if (least == 0 || t < least) { least = t; best = c; }
    };
    if (kn) {
        offer(kSmallKn[0], 5, 512, 0.2, 1, 1.12);
        offer(kSmallKn[1], 5, 256, 0.17, 1, 1.12);
        offer(kSmallKn[2], 5, 256, 0.24, 1, 1.12);
    } else {
        offer(kSmallNk[0], 5, 512, f8 ? 0.156 : 0.106, 0.83, 1);
        offer(kSmallNk[1], 5, 512, f8 ? 0.21 : 0.16, 0.7, 1);
    }
    offer(kTeams64, 6, 256, f8 ? 0.43 : 0.41, f8 ? 1 : 0.85, 1.2);
    offer(kTeams128, 6, 256, f8 ? 0.6 : 0.55, f8 ? 1 : 0.85, 1.2);
    offer(kTile128, 6, 512, f8 ? 1.05 : 1.09, 0.65, f8 ? 1.15 : 1.05);
    for (uint32_t rows = kLeastRows; rows <= kTile256.rows; rows += 32) {
        double height;   // above five two stages instead of three
        row_tiles(rows, &height);
        offer({Choice::TILE, rows, 256, 1}, 8, 256, f8 ? 0.35 + 0.19 * height + (height > 5 ? 0.05 : 0) : height > 5 ? 0.65 + 0.11 * height : 0.45 + 0.115 * height, 1,
              (f8 ? 1.15 : 0.98) + (rows > 160 && !dealt ? 0.05 : 0));
    }
    return best;
}

// Weight gradients: rounds of 256 (512) workgroups, each a start and its steps.  Measured (us, fp32 results, 256x256 / 128x128 tiles): 8 groups of 512 rows,
// 512x512 22.5 / 10.4; 64 of 256, 512x512 38.9 / 27.9; 8 of 128, 2048x2048 38.0 / 34.6; 16 of 256, 1024x1024 25.5 / 25.4; 8 of 2048, 1024x2048 71 / 78;
// 16 of 512, 4096x1792 227 / 273; one of 4096, 4096x4096 117 / 156.
Choice choose_dw(const RaggedArgs &a)
{
    const double steps = std::ceil((double)a.rows / a.groups / 64);
    const double large = std::ceil(a.groups * (double)(cdiv(a.k, 256) * cdiv(a.n, 256)) / 256) * (9 + 1.5 * steps);
    const double small = std::ceil(a.groups * (double)(cdiv(a.k, 128) * cdiv(a.n, 128)) / 512) * (3.5 + steps);
    return small < large ? kTile128 : kTile256;
}

// Whether a product can run on what the caller asks for.
bool can_run(const Choice &asked, bool kn, bool dw, bool words)
{
    auto is = [&](const Choice &c) { return c.rows == asked.rows && c.cols == asked.cols && c.teams == asked.teams; };
    if (!words) return false;
    if (is(kTile256) || is(kTile128)) return true;
    if (dw) return false;
    if (is(kTeams64) || is(kTeams128)) return true;
    if (asked.cols == 256 && asked.teams == 1) return asked.rows >= kLeastRows && asked.rows <= kTile256.rows && asked.rows % 32 == 0;
    if (kn) return std::any_of(std::begin(kSmallKn), std::end(kSmallKn), is);
    return std::any_of(std::begin(kSmallNk), std::end(kSmallNk), is);
}

void run(uint32_t dtype, const RaggedArgs &args, bool kn, bool dw, const CatcocTile *tile, void *stream)
{
    RaggedArgs a = args;
    const bool words = rows_on_words(dtype, a, kn, dw);
    Choice c = kChecked;
    if (tile != nullptr && (tile->rows || tile->cols || tile->teams)) {
        c = {tile->teams == 4 ? Choice::SMALL : Choice::TILE, tile->rows, tile->cols, tile->teams};
        if (c.rows == kChecked.rows && c.cols == kChecked.cols && c.teams == kChecked.teams) {
            c = kChecked;
        } else if (!can_run(c, kn, dw, words)) {
            api_fail(E_TILING, "no kernel of %ux%u tiles and %u team(s) for this product%s", tile->rows, tile->cols, tile->teams, words ? "" : " (rows that do not start on 4 bytes run 64x64 tiles, 1 team)");
            return;
        }
    } else if (words) {
        c = dw ? choose_dw(a) : choose(dtype, a, kn);
    }
    a.tileRows = c.rows;
    a.dealt = c.kind == Choice::TILE && !dw && deal(a);
    uint64_t wgs;
    if (!dw) {
        wgs = count_wgs(a, c);
    } else {
        const uint64_t tiles = cdiv(a.k, c.rows) * cdiv(a.n, c.cols);
        wgs = a.groups * tiles;
        if (c.kind == Choice::TILE)   // eighths of every group's tiles, dealt out to one workgroup a CU (two of 128 columns)
            wgs = std::min<uint64_t>(65536 / c.cols, a.groups * cdiv(tiles, 8) * 8);
    }
    if (wgs > most_wgs(c)) { api_fail(E_SHAPE, "%llu tiles are more than one launch holds", (unsigned long long)wgs); return; }
    api_launch_info({c.kind == Choice::CHECKED ? (uint32_t)CATCOC_KERNEL_RAGGED_CHECKED : (uint32_t)CATCOC_KERNEL_RAGGED, c.rows, c.cols, c.teams, 0, 0});
    if (c.kind == Choice::SMALL) api_launched(launch_ragged_small(dtype, a, kn, c.rows, (uint32_t)wgs, stream));
    else if (c.kind == Choice::TILE) api_launched(launch_ragged_tile(dtype, a, kn, dw, c.cols, c.teams, (uint32_t)wgs, stream));
    else api_launched(launch_ragged_checked(dtype, a, kn, dw, (uint32_t)wgs, stream));
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
                                 uint8_t *symmetricPtr, uint32_t m, uint32_t n, uint32_t k, uint32_t outDataType, const CatcocTile *tile)
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
    run(DT_F8, a, false, false, tile, stream);
}

void catcoc_grouped_matmul(void *stream, uint32_t dataType, const void *x, const void *w, const int32_t *groupEnds, void *out, uint32_t rows, uint32_t n,
                           uint32_t k, uint32_t groups, uint32_t transB, const CatcocTile *tile)
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
    run(dataType, a, transB == 0, false, tile, stream);
}

void catcoc_grouped_matmul_dw(void *stream, uint32_t dataType, const void *x, const void *dy, const int32_t *groupEnds, void *dw, uint32_t rows, uint32_t n,
                              uint32_t k, uint32_t groups, uint32_t transB, uint32_t outDataType,
                              const CatcocTile *tile)
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
    run(dataType, a, false, true, tile, stream);
}

void catcoc_grouped_fp8_matmul(void *stream, const uint8_t *x, const uint8_t *w, const float *scale_x, const float *scale_w, const int32_t *groupEnds,
                               void *out, uint32_t rows, uint32_t n, uint32_t k, uint32_t groups, uint32_t outDataType,
                               const CatcocTile *tile)
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
    run(DT_F8, a, false, false, tile, stream);
}

}  // extern "C"
