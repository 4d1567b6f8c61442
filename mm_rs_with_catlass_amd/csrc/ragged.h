// Device code that the kernels of ragged products share: which tile a workgroup computes, the MFMAs of one step of k, rounding and stores.
//
// A step is 128 BYTES of k (64 values of 16 bits, 128 of e4m3: one scale block).  The first MFMA operand is the matrix (its columns become the result's
// registers), the second the rows: a lane then holds four consecutive columns, 4 * (lane >> 4) + r of a 16-column block, of ONE row, lane & 15.  So a
// row's scale is one value per lane, and a lane's results are 8 or 16 consecutive bytes of the output.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemm_dma_kernel.h"
#include "ragged_args.h"

namespace catcoc {

typedef int v8i __attribute__((ext_vector_type(8)));

// One dimension of a launch holds fewer than 2^32 threads: workgroups past that go on in the second one, in rows of kGridRow.  Those past the last one asked for
// have to find nothing to do.  For the checked kernel and the quantizer; in the small tiles' kernel the second index costs a call of 18.5 us 0.46 of them.
constexpr uint32_t kGridRowLog = 22, kGridRow = 1u << kGridRowLog;
inline dim3 grid_of(uint64_t wgs, uint32_t threads)
{
    return wgs * threads < (1ull << 32) ? dim3((uint32_t)wgs) : dim3(kGridRow, (uint32_t)((wgs + kGridRow - 1u) >> kGridRowLog));
}
__device__ __forceinline__ uint32_t workgroup() { return (blockIdx.y << kGridRowLog) + blockIdx.x; }

// A read of 16 bytes at any address.
__device__ __forceinline__ v4i load16_any(const unsigned char *p)
{
    v4i v;
    __builtin_memcpy(&v, p, 16);
    return v;
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

// Position `wg` of a launch of `total` tiles that go round-robin to the eight XCDs: each of them gets a run of consecutive tiles, which share rows and
// matrices in its L2.  Returns total or more past the end.
__device__ __forceinline__ uint32_t xcd_run(uint32_t wg, uint32_t total)
{
    const uint32_t x = wg & 7u, at = wg >> 3, each = total >> 3, rest = total & 7u;
    return at < each + (x < rest ? 1u : 0u) ? x * each + umin(x, rest) + at : 0xffffffffu;
}

// Rows of group e, kept inside [0, rows) and never of negative length whatever `ends` says; e == groups: the rows past the last group, whose results
// are zero.
__device__ __forceinline__ void group_rows(const RaggedArgs &args, uint32_t e, uint32_t &begin, uint32_t &end)
{
    if (args.ends == nullptr) {
        begin = e == 0 ? 0u : args.rows;
        end = args.rows;
        return;
    }
    const int32_t b = e == 0 ? 0 : args.ends[umin(e, args.groups) - 1u];
    const int32_t t = e < args.groups ? args.ends[e] : (int32_t)args.rows;
    begin = (uint32_t)min(max(b, 0), (int32_t)args.rows);
    end = (uint32_t)max(min(t, (int32_t)args.rows), (int32_t)begin);
}

// A tile of y: `rows` rows from `row` on, all of `group` (group == args.groups: zeros), column tile `colTile`.
struct RaggedTile {
    uint32_t group, row, rows, colTile;
};

// Which of up to 64 groups (or the rows past the last one) workgroup `wg` works for where every XCD gets an eighth of each group's tiles, the highest first;
// count: the group's row tiles, local: which of its tiles.  False: none.
__device__ __forceinline__ bool dealt_group(const RaggedArgs &args, uint32_t wg, uint32_t bx, uint32_t nt, uint32_t &group, uint32_t &begin, uint32_t &end, uint32_t &count, uint32_t &local)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t b, e;
    group_rows(args, umin(lane, args.groups - 1u), b, e);
    const uint32_t mine = lane < args.groups ? (e - b + bx - 1u) / bx : 0u, height = mine ? (e - b + 32u * mine - 1u) / (32u * mine) : 0u;
    uint32_t rank = 0, before = 0;   // by height, at most 256 / 32
#pragma unroll
    for (uint32_t h = 9; h-- > 0u;) {
        const uint64_t same = __ballot(height == h);
        if (height == h) rank = before + (uint32_t)__builtin_popcountll(same & ((1ull << lane) - 1ull));
        before += (uint32_t)__builtin_popcountll(same);
    }
    const uint32_t order = (uint32_t)__builtin_amdgcn_ds_permute((int)(rank * 4u), (int)lane);
    // lane i: the i-th group's tiles, and those of them that this XCD gets; what is left of a division by eight goes to the XCDs in turn
    const uint32_t tiles = (uint32_t)__builtin_amdgcn_ds_permute((int)(rank * 4u), (int)(mine * nt)), each = tiles >> 3, rest = tiles & 7u;
    const uint32_t place = (wg - (wave_prefix(rest) - rest)) & 7u, part = each + (place < rest ? 1u : 0u), upTo = wave_prefix(part), j = wg >> 3;
    const uint64_t past = __ballot(upTo > j);
    if (past == 0) {   // rows past the last group
        group = args.groups;
        begin = (uint32_t)__builtin_amdgcn_readlane((int)e, 63);
        end = args.rows;
        count = (end - begin + bx - 1u) / bx;
        local = 8u * (j - (uint32_t)__builtin_amdgcn_readlane((int)upTo, 63)) + (wg & 7u);
        return local < count * nt;
    }
    const int l = __builtin_ctzll(past);
    local = (uint32_t)__builtin_amdgcn_readlane((int)(place * each + umin(place, rest) + j + part - upTo), l);
    group = (uint32_t)__builtin_amdgcn_readlane((int)order, l);
    begin = (uint32_t)__builtin_amdgcn_readlane((int)b, (int)group);
    end = (uint32_t)__builtin_amdgcn_readlane((int)e, (int)group);
    count = (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)group);
    return true;
}

// Tile of workgroup `wg` where a group's rows are cut into tiles of at most bx rows of about the same height (whole `unit`s), nt column tiles.  A group's tiles follow each
// other, eight row tiles to a band and column by column within it: the tiles that run on an XCD at a time share few rows and columns.  Every wave
// works it out by itself, 64 groups at a time.  False: no tile left.
__device__ __forceinline__ bool ragged_tile(const RaggedArgs &args, uint32_t wg, uint32_t bx, uint32_t nt, uint32_t unit, RaggedTile &t)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t first = 0, count, begin, end, local;   // the group's first row tile and how many it has
    if (args.ends == nullptr) {
        count = (args.rows + bx - 1u) / bx;
        local = xcd_run(wg, count * nt);
        if (local >= count * nt) return false;
        t.group = 0;
        begin = 0;
        end = args.rows;
    } else if (args.dealt) {
        if (!dealt_group(args, wg, bx, nt, t.group, begin, end, count, local)) return false;
    } else {
        uint32_t total = 0, b = 0, e = 0, tiles = 0, upTo = 0;
        const uint32_t chunks = args.groups / 64u + 1u;   // (one group more than there are: the rows past the last one)
        for (uint32_t c = 0; c < chunks; ++c) {
            const uint32_t g = c * 64u + lane;
            group_rows(args, umin(g, args.groups), b, e);
            tiles = g <= args.groups ? (e - b + bx - 1u) / bx : 0u;
            upTo = wave_prefix(tiles);
            total += (uint32_t)__builtin_amdgcn_readlane((int)upTo, 63);
        }
        const uint32_t at = xcd_run(wg, total * nt);
        if (at >= total * nt) return false;
        uint32_t before = 0;
        for (uint32_t c = 0;; ++c) {
            if (chunks > 1u) {
                const uint32_t g = c * 64u + lane;
                group_rows(args, umin(g, args.groups), b, e);
                tiles = g <= args.groups ? (e - b + bx - 1u) / bx : 0u;
                upTo = wave_prefix(tiles);
            }
            const uint64_t past = __ballot((before + upTo) * nt > at);
            if (past != 0 || c + 1u == chunks) {
                const int l = past != 0 ? __builtin_ctzll(past) : 63;
                t.group = c * 64u + (uint32_t)l;
                begin = (uint32_t)__builtin_amdgcn_readlane((int)b, l);
                end = (uint32_t)__builtin_amdgcn_readlane((int)e, l);
                count = (uint32_t)__builtin_amdgcn_readlane((int)tiles, l);
                first = before + (uint32_t)__builtin_amdgcn_readlane((int)upTo, l) - count;
                break;
            }
            before += (uint32_t)__builtin_amdgcn_readlane((int)upTo, 63);
        }
        local = at - first * nt;
    }
    const uint32_t band = local / (8u * nt), in = local - band * 8u * nt, wide = umin(8u, count - 8u * band);
    t.colTile = in / wide;
    const uint32_t r = 8u * band + in - t.colTile * wide;
    const uint32_t units = (end - begin + unit - 1u) / unit, each = units / count, rest = units - each * count;
    const uint32_t u0 = r * each + umin(r, rest);
    t.row = begin + u0 * unit;
    t.rows = umin((each + (r < rest ? 1u : 0u)) * unit, end - t.row);
    t.group = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.group);
    t.row = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.row);
    t.rows = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.rows);
    t.colTile = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.colTile);
    return true;
}

// A step's 128 bytes of k of 16 rows or columns: the lane's two 16-byte pieces.
struct Frag {
    v4i lo, hi;
};

// A step's product of e4m3 values, before its scale.  The instruction is no exact fp32 sum: of up to eight adjacent products it keeps 13 bits below the largest's
// leading one (rms error at 128 values 2.1e-6 of the sum of magnitudes, 1/2000 of what the values' own rounding to e4m3 is).  The exact alternative, 16-bit MFMAs
// on widened values, has half the rate; sums over steps are fp32.
__device__ __forceinline__ v4f step_mfma_f8(const Frag &w, const Frag &x)
{
    const v8i a = __builtin_shufflevector(w.lo, w.hi, 0, 1, 2, 3, 4, 5, 6, 7), b = __builtin_shufflevector(x.lo, x.hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// acc += w x over a step.  e4m3: one MFMA over the whole step from zero, then acc += s * its result in fp32: the scales of a block are outside its sum.
template <uint32_t DT>
__device__ __forceinline__ void step_mfma(const Frag &w, const Frag &x, v4f &acc, float s)
{
    if constexpr (DT == DT_F8) {
        const v4f d = step_mfma_f8(w, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(s, d[r], acc[r]);
    } else {
        acc = mfma16<DT>(w.lo, x.lo, acc);
        acc = mfma16<DT>(w.hi, x.hi, acc);
    }
}

// Two values rounded to the output's 16-bit type, to nearest even.
__device__ __forceinline__ uint32_t round2(float a, float b, uint32_t type)
{
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    if (type == DT_BF16) return __builtin_bit_cast(uint32_t, v2bf{(__bf16)a, (__bf16)b});
    return __builtin_bit_cast(uint32_t, v2h{(_Float16)a, (_Float16)b});
}

// Four consecutive values of one output row, `have` of them inside it.
__device__ __forceinline__ void store4(const RaggedArgs &args, size_t at, v4f v, uint32_t have)
{
    if (args.outType == 0) {
        float *p = (float *)args.out + at;
        if (have >= 4u) __builtin_memcpy(p, &v, 16);
        else {
#pragma unroll
            for (uint32_t r = 0; r < 3u; ++r)
                if (r < have) p[r] = v[r];
        }
    } else {
        unsigned short *p = (unsigned short *)args.out + at;
        const v2i u = {(int)round2(v[0], v[1], args.outType), (int)round2(v[2], v[3], args.outType)};
        if (have >= 4u) __builtin_memcpy(p, &u, 8);
        else {
#pragma unroll
            for (uint32_t r = 0; r < 3u; ++r)
                if (r < have) p[r] = (unsigned short)((uint32_t)u[r >> 1] >> (16u * (r & 1u)));
        }
    }
}

// Eight consecutive values in 16 bits.
__device__ __forceinline__ void store8_16bit(const RaggedArgs &args, size_t at, v4i v, uint32_t have)
{
    unsigned short *p = (unsigned short *)args.out + at;
    if (have >= 8u) {
        __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll
        for (uint32_t r = 0; r < 7u; ++r)
            if (r < have) p[r] = (unsigned short)((uint32_t)v[r >> 1] >> (16u * (r & 1u)));
    }
}

// The other ranks' partials of four consecutive values of a row: `BATCH` of them from slot `first` on, asked for together ...
template <int BATCH>
__device__ __forceinline__ void load_peers4(const RaggedArgs &args, uint32_t first, uint32_t row, uint32_t col, uint32_t have, v4f (&u)[BATCH])
{
#pragma unroll
    for (uint32_t p = 0; p < (uint32_t)BATCH; ++p) {
        u[p] = v4f{0.f, 0.f, 0.f, 0.f};
        if (first + p >= args.nPeers || have == 0u) continue;
        const float *q = args.peers[first + p] + (int64_t)row * args.peerLd + col;
        if (have >= 4u) {
            __builtin_memcpy(&u[p], q, 16);
        } else {
#pragma unroll
            for (uint32_t r = 0; r < 3u; ++r)
                if (r < have) u[p][r] = q[r];
        }
    }
}

// ... and all of them added in slot order, the first `BATCH` from `u`.
template <int BATCH>
__device__ __forceinline__ void add_peers4(const RaggedArgs &args, uint32_t row, uint32_t col, v4f &v, uint32_t have, v4f (&u)[BATCH])
{
    for (uint32_t first = 0; first < args.nPeers; first += BATCH) {
        if (first != 0) load_peers4<BATCH>(args, first, row, col, have, u);
#pragma unroll
        for (uint32_t p = 0; p < (uint32_t)BATCH; ++p)
            if (first + p < args.nPeers) {
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] += u[p][r];
            }
    }
}

// The same where nothing was asked for yet.
__device__ __forceinline__ void add_peers4(const RaggedArgs &args, uint32_t row, uint32_t col, v4f &v, uint32_t have)
{
    if (args.nPeers == 0) return;
    v4f u[4];
    load_peers4<4>(args, 0, row, col, have, u);
    add_peers4<4>(args, row, col, v, have, u);
}

}  // namespace catcoc
