// Ragged products on 64x64 tiles whose every load is checked: any width, any alignment.
//
// Four waves of 32x32; a step's pieces of both operands are fetched into registers while the one before is multiplied, and written to the other half of
// a double buffer in LDS.  A piece is 16 bytes wherever that many belong to its row, read at whatever address it has, else its values one by one and
// zeros behind them.  It serves rows that do not start on 4 bytes (the copies that go straight to LDS need that).
// Bound by its small tile's loads through registers: 4096 rows in 16 groups of 4096x3584, bf16, 279 us against 148 on the tiles of aligned rows; e4m3 512x4096x4096 24
// against 20.
#pragma once
#include "ragged.h"

namespace catcoc {

// Bytes [at, at + 16) of a row of `size` bytes; zeros past its end.
__device__ __forceinline__ v4i load16_within(const unsigned char *row, uint32_t at, uint32_t size)
{
    if (at + 16u <= size) return load16_any(row + at);
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 15u; ++i)
        if (at + i < size) v[i >> 2] |= (uint32_t)row[at + i] << (8u * (i & 3u));
    return v4i{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
}

// A 64-column (or 64-row) operand of one step in LDS, as the tile kernels lay it out for 128-byte rows.
//   k contiguous: 64 rows of 128 bytes of k; piece c of row r at slot c ^ ((r >> 1) & 7): a fragment read's 16 lanes meet all banks once.
//   else:         64 rows of k, 64 columns of 2 bytes each; piece q of row r at slot q ^ k_major64_slot(r), for the transposing reads.
__device__ __forceinline__ uint32_t k_rows_slot(uint32_t row) { return (row >> 1) & 7u; }
__device__ __forceinline__ uint32_t k_major64_slot(uint32_t row) { return (((row >> 1) & 1u) << 1) | (((row >> 3) & 1u) << 2); }

// LDS offsets of a lane's pieces in an operand of one step, and the reads.
//   k contiguous: the lane's row `row`; 16 rows on is 2048 bytes on.
//   else:         rows of `pitch` bytes, columns [col0, +16), col0 a multiple of 16; SLOT: where piece q of a row lies.  16 i columns on (i < 8, inside the same
//                 aligned 128 or, SLOT's values below 8, 64 columns) is this ^ 32 i.  TURNED: the column quads in the order 0, 2, 1, 3.
__device__ __forceinline__ uint32_t at_k_rows(uint32_t row, uint32_t lane) { return row * 128u + ((lane >> 4) ^ k_rows_slot(row)) * 16u; }

template <bool TURNED, typename SLOT>
__device__ __forceinline__ uint32_t at_k_major(uint32_t pitch, uint32_t col0, uint32_t lane, SLOT slot)
{
    const uint32_t i = lane & 15u, q = col0 / 8u + (TURNED ? i & 1u : (i >> 1) & 1u), half = TURNED ? (i >> 1) & 1u : i & 1u;
    const uint32_t row = 8u * (lane >> 4) + (i >> 2);   // (slot(row) is that of row + 4, row + 32 and row + 36 too)
    return row * pitch + (q ^ slot(row)) * 16u + half * 8u;
}

__device__ __forceinline__ Frag frag_k_rows(const unsigned char *smem, uint32_t at)
{
    return {*(const v4i *)(smem + at), *(const v4i *)(smem + (at ^ 64u))};
}

template <uint32_t PITCH>
__device__ __forceinline__ Frag frag_k_major(const unsigned char *smem, uint32_t at)
{
    v4s16 v[4];
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u)
        v[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CATCOC_LDS v4s16 *)(smem + at + (32u * (u >> 1) + 4u * (u & 1u)) * PITCH));
    Frag f;
    f.lo = __builtin_bit_cast(v4i, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
    f.hi = __builtin_bit_cast(v4i, __builtin_shufflevector(v[2], v[3], 0, 1, 2, 3, 4, 5, 6, 7));
    return f;
}

// KN: w is [k, n].  DW: the weight gradient; x [rows, k] and dy [rows, n] are both rows of columns, the sum runs over a group's rows.
template <uint32_t DT, bool KN, bool DW>
__global__ void __launch_bounds__(256, 2) ragged_checked_kernel(const RaggedArgs args)
{
    constexpr uint32_t ES = DT == DT_F8 ? 1u : 2u, KE = 128u / ES;
    constexpr bool XK = DW, WK = KN || DW;   // operands whose rows are rows of k
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * 8192];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, w = tid >> 6;
    const uint32_t nt = (args.n + 63u) / 64u;
    RaggedTile t;
    uint32_t K, xCols = 0;
    const unsigned char *X, *W;
    uint32_t group = 0;
    if constexpr (DW) {
        const uint32_t pt = (args.k + 63u) / 64u, total = args.groups * pt * nt, at = xcd_run(workgroup(), total);
        if (at >= total) return;
        group = at / (pt * nt);
        const uint32_t in = at - group * (pt * nt);
        t.colTile = in / pt;
        const uint32_t p = in - t.colTile * pt;
        uint32_t b, e;
        group_rows(args, group, b, e);
        K = e - b;
        t.row = 64u * p;
        t.rows = umin(64u, args.k - t.row);
        xCols = args.k - t.row;
        X = (const unsigned char *)args.x + ((size_t)b * args.k + t.row) * 2u;
        W = (const unsigned char *)args.w + ((size_t)b * args.n + 64u * t.colTile) * 2u;
    } else {
        if (!ragged_tile(args, workgroup(), 64u, nt, 64u, t)) return;
        group = t.group;
        K = group < args.groups ? args.k : 0u;
        X = (const unsigned char *)args.x + (size_t)t.row * args.k * ES;
        W = (const unsigned char *)args.w + (size_t)umin(group, args.groups - 1u) * args.n * args.k * ES + (size_t)(64u * t.colTile) * (KN ? ES : args.k * ES);
    }
    const uint32_t col0 = 64u * t.colTile, cols = umin(64u, args.n - col0), steps = (K + KE - 1u) / KE;

    // a thread's two pieces of each operand
    v4i px[2], pw[2];
    float sx = 0.f, sw = 0.f;   // e4m3: scales of the step whose pieces are in registers, of row lane & 15 (+ 16) of the wave's rows
    float sx1 = 0.f;
    const uint32_t kb = (args.k + kScaleBlock - 1u) / kScaleBlock, wr = (w >> 1) * 32u, wc = (w & 1u) * 32u;
    auto fetch = [&](uint32_t s) {
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
            const uint32_t r = 32u * j + (tid >> 3), c = tid & 7u;
            if constexpr (XK) px[j] = s * 64u + r < K ? load16_within(X + (size_t)(s * 64u + r) * args.k * 2u, c * 16u, xCols * 2u) : v4i{0, 0, 0, 0};
            else px[j] = load16_within(X + (size_t)umin(r, t.rows - 1u) * args.k * ES, s * 128u + c * 16u, K * ES);
            if constexpr (WK) pw[j] = s * 64u + r < K ? load16_within(W + (size_t)(s * 64u + r) * args.n * 2u, c * 16u, (args.n - col0) * 2u) : v4i{0, 0, 0, 0};
            else pw[j] = load16_within(W + (size_t)umin(r, cols - 1u) * args.k * ES, s * 128u + c * 16u, K * ES);
        }
        if constexpr (DT == DT_F8) {
            const float *p = args.sx + (size_t)s * args.rows + t.row;
            sx = p[umin(wr + (lane & 15u), t.rows - 1u)];
            sx1 = p[umin(wr + 16u + (lane & 15u), t.rows - 1u)];
            sw = args.sw[((size_t)umin(group, args.groups - 1u) * ((args.n + kScaleBlock - 1u) / kScaleBlock) + col0 / kScaleBlock) * kb + s];
        }
    };
    auto put = [&](uint32_t s) {
        unsigned char *p = smem + (s & 1u) * 16384u;
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
            const uint32_t r = 32u * j + (tid >> 3), c = tid & 7u;
            *(v4i *)(p + r * 128u + (c ^ (XK ? k_major64_slot(r) : k_rows_slot(r))) * 16u) = px[j];
            *(v4i *)(p + 8192u + r * 128u + (c ^ (WK ? k_major64_slot(r) : k_rows_slot(r))) * 16u) = pw[j];
        }
    };

    v4f acc[2][2];   // [16 rows][16 columns]
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = v4f{0.f, 0.f, 0.f, 0.f};
    if (steps != 0) fetch(0);
    for (uint32_t s = 0; s < steps; ++s) {
        put(s);
        const float s0 = sx * sw, s1 = sx1 * sw;
        if (s + 1u < steps) fetch(s + 1u);
        __syncthreads();   // (the other half was last read before the barrier of the step before this one)
        const unsigned char *p = smem + (s & 1u) * 16384u;
        Frag fx[2], fw[2];
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
            if constexpr (XK) fx[i] = frag_k_major<128>(p, at_k_major<false>(128u, wr + 16u * i, lane, k_major64_slot));
            else fx[i] = frag_k_rows(p, at_k_rows(wr + 16u * i + (lane & 15u), lane));
            if constexpr (WK) fw[i] = frag_k_major<128>(p + 8192u, at_k_major<false>(128u, wc + 16u * i, lane, k_major64_slot));
            else fw[i] = frag_k_rows(p + 8192u, at_k_rows(wc + 16u * i + (lane & 15u), lane));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) step_mfma<DT>(fw[j], fx[i], acc[i][j], i == 0 ? s0 : s1);
    }
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i)
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j) {
            const uint32_t r = wr + 16u * i + (lane & 15u), c = wc + 16u * j + 4u * (lane >> 4);
            if (r >= t.rows || c >= cols) continue;
            const uint32_t have = umin(4u, cols - c);
            v4f v = acc[i][j];
            if constexpr (DT == DT_F8) add_peers4(args, t.row + r, col0 + c, v, have);
            store4(args, ((size_t)(DW ? (size_t)group * args.k : (size_t)0) + t.row + r) * args.n + col0 + c, v, have);
        }
}

}  // namespace catcoc
