// Ragged products on tiles of few rows, as decode batches have them: the matrix is streamed once, from memory.
#pragma once
#include "ragged_tile.h"

namespace catcoc {

// A tile of 16 NI rows and 16 NJ columns on four waves that deal a tile's steps of 128 bytes of k out among themselves: wave w multiplies steps w, w + 4, ...
// through a ring of its own in LDS, NS stages deep, and meets nobody until the four sums are added, in the order of the waves.  So no wave ever waits for another
// one's copies, and what is in flight per CU (two workgroups, where their rings fit) is 64 KiB and more, what memory needs to stream.
// Bound by the matrix's bytes: one row of e4m3 times 8192x8192 and seven peers 12.2 us (5.5 TB/s), 16 rows in 14 of 64 groups of 4096x3584 in bf16 72 us (5.7 TB/s),
// 256 rows in 60 of them in e4m3 148 us (5.9 TB/s), where reads alone reach 6.1 TB/s.  Narrow tiles, since a decode launch has no more columns to fill 256 CUs with:
// on 128x128 tiles the first takes 40 us.
template <uint32_t DT, bool KN, int NI, int NJ, int NS>
struct RaggedSmall {
    static constexpr uint32_t ES = DT == DT_F8 ? 1u : 2u, KE = 128u / ES, WAVES = 4u;
    static constexpr uint32_t XB = NI * 2048u, WB = NJ * 2048u, STAGE = XB + WB + (DT == DT_F8 ? 256u : 0u);
    static constexpr uint32_t WAVE = NS * STAGE > NI * NJ * 1024u ? NS * STAGE : NI * NJ * 1024u;   // (the sums meet where the rings were)
    static constexpr int PER = 2 * NI + 2 * NJ + (DT == DT_F8 ? 1 : 0);                             // copies of a step
    static_assert(!KN || NJ == 4, "a matrix as [k, n]: rows of 128 bytes");
};

template <uint32_t DT, bool KN, int NI, int NJ, int NS>
__global__ void __launch_bounds__(256, 2) ragged_small_kernel(const RaggedArgs args)
{
    using S = RaggedSmall<DT, KN, NI, NJ, NS>;
    constexpr uint32_t ES = S::ES, KE = S::KE, BX = 16u * NI, BY = 16u * NJ;
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * S::WAVE];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    RaggedTile t;
    if (!ragged_tile(args, blockIdx.x, BX, (args.n + BY - 1u) / BY, 16u, t)) return;
    const uint32_t g = umin(t.group, args.groups - 1u), K = t.group < args.groups ? args.k : 0u;
    const uint32_t col0 = BY * t.colTile, cols = umin(BY, args.n - col0), steps = (K + KE - 1u) / KE;
    const uint32_t mine = steps > wave ? (steps - wave + 3u) / 4u : 0u;   // steps of this wave
    const bool partLast = K % KE != 0 || (KN && args.n % 8u != 0);

    // The other ranks' partials of the four columns that a thread will store: asked for before anything else.
    constexpr int VECS = (NI * NJ + 3) / 4, BATCH = VECS == 1 ? 8 : 4;
    v4f peer[VECS][BATCH];
    uint32_t vr[VECS], vc[VECS], have[VECS];
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        const uint32_t f = wave + 4u * v;
        vr[v] = 16u * (f / NJ) + (lane & 15u);
        vc[v] = 16u * (f % NJ) + 4u * (lane >> 4);
        have[v] = f < (uint32_t)(NI * NJ) && vr[v] < t.rows && vc[v] < cols ? umin(4u, cols - vc[v]) : 0u;
        if constexpr (DT == DT_F8) load_peers4<BATCH>(args, 0, t.row + vr[v], col0 + vc[v], have[v], peer[v]);
    }

    // ---- this wave's copies
    unsigned char *const ring = smem + wave * S::WAVE;
    const uint32_t ring0 = (uint32_t)(uintptr_t)(CATCOC_LDS unsigned char *)smem + wave * S::WAVE;
    const unsigned char *const X = uniform_ptr((const unsigned char *)args.x + (size_t)t.row * args.k * ES);
    const uint32_t xPitch = args.k * ES, wPitch = KN ? args.n * 2u : args.k * ES;
    const unsigned char *const W = uniform_ptr((const unsigned char *)args.w + (size_t)g * args.n * args.k * ES + (size_t)col0 * (KN ? 2u : wPitch));
    uint32_t xo[2 * NI], wo[2 * NJ];
#pragma unroll
    for (uint32_t j = 0; j < 2u * NI; ++j) {
        const uint32_t row = 8u * j + (lane >> 3);
        xo[j] = umin(row, t.rows - 1u) * xPitch + ((lane & 7u) ^ k_rows_slot(row)) * 16u;
    }
#pragma unroll
    for (uint32_t j = 0; j < 2u * NJ; ++j) {
        const uint32_t row = 8u * j + (lane >> 3);
        if constexpr (KN) wo[j] = row * wPitch + umin((lane & 7u) ^ k_major64_slot(row), (cols - 1u) / 8u) * 16u;
        else wo[j] = umin(row, cols - 1u) * wPitch + ((lane & 7u) ^ k_rows_slot(row)) * 16u;
    }
    const uint32_t kb = (args.k + kScaleBlock - 1u) / kScaleBlock;
    const float *const SX = DT == DT_F8 ? uniform_ptr(args.sx + t.row) : nullptr;
    const float *const SW = DT == DT_F8 ? uniform_ptr(args.sw + ((size_t)g * ((args.n + kScaleBlock - 1u) / kScaleBlock) + col0 / kScaleBlock) * kb) : nullptr;
    auto issue = [&](uint32_t i, uint32_t stage) {   // this wave's step i into stage `stage` (its offset)
        const uint32_t s = wave + 4u * i;
        const unsigned char *const x = X + (size_t)s * 128u, *const w = W + (size_t)s * (KN ? 64u * wPitch : 128u);
        if (partLast && s + 1u == steps) {
            // what is there of the last step, 4 bytes at a time, and zeros
            const uint32_t left = (K - s * KE) * ES;
#pragma unroll 1
            for (uint32_t c = 0; c < (S::XB + S::WB) / 256u; ++c) {
                const bool isX = c < S::XB / 256u;
                const uint32_t at = c * 64u + lane - (isX ? 0u : S::XB / 4u), row = at / 32u, slot = at % 32u / 4u;
                const bool km = KN && !isX;
                const uint32_t byte = (slot ^ (km ? k_major64_slot(row) : k_rows_slot(row))) * 16u + at % 4u * 4u;
                const bool there = km ? row < K - s * KE && byte < (args.n - col0) * 2u : byte < left;
                const uint32_t from = byte + (km ? row : umin(row, (isX ? t.rows : cols) - 1u)) * (isX ? xPitch : wPitch);
                if (there) copy4(isX ? x : w, from, ring0 + stage + c * 256u);
                else *(uint32_t *)(ring + stage + c * 256u + lane * 4u) = 0u;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2 * NJ; ++j) copy16(w, wo[j], ring0 + stage + S::XB + j * 1024u);
#pragma unroll
            for (int j = 0; j < 2 * NI; ++j) copy16(x, xo[j], ring0 + stage + j * 1024u);
        }
        if constexpr (DT == DT_F8) copy4((const unsigned char *)(SX + (size_t)s * args.rows), umin(lane, t.rows - 1u) * 4u, ring0 + stage + S::XB + S::WB);
    };

    v4f acc[NI][NJ];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)NS; ++i)
        if (i < mine) issue(i, i * S::STAGE);
    const uint32_t xa = at_k_rows(lane & 15u, lane), wa = S::XB + (KN ? at_k_major<false>(128u, 0, lane, k_major64_slot) : at_k_rows(lane & 15u, lane));
    // steps that as many whole ones follow that only the last NS - 1 steps' copies may be under way
    const uint32_t whole = steps - (partLast ? 1u : 0u), wholeMine = whole > wave ? (whole - wave + 3u) / 4u : 0u;
    uint32_t stage = 0;
    float sw = 0.f;
    if constexpr (DT == DT_F8) sw = mine ? load_uniform(SW + wave) : 0.f;
#pragma unroll 1
    for (uint32_t i = 0; i < mine; ++i) {
        float swNext = 0.f;
        if constexpr (DT == DT_F8) swNext = load_uniform(SW + umin(wave + 4u * (i + 1u), steps - 1u));
        if (i + NS <= wholeMine) CATCOC_WAIT_VMCNT((NS - 1) * S::PER);
        else CATCOC_WAIT_VMCNT(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (zeros of a last step)
        Frag fx[NI], fw[NJ];
        float sc[NI];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            if constexpr (KN) fw[j] = frag_k_major<128>(ring, (stage + wa) ^ (32u * j));
            else fw[j] = frag_k_rows(ring, stage + wa + 2048u * j);
        }
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            fx[n] = frag_k_rows(ring, stage + xa + 2048u * n);
            sc[n] = DT == DT_F8 ? *(const float *)(ring + stage + S::XB + S::WB + (16u * n + (lane & 15u)) * 4u) * sw : 0.f;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the stage may be overwritten)
        if (i + NS < mine) issue(i + NS, stage);
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int j = 0; j < NJ; ++j) step_mfma<DT>(fw[j], fx[n], acc[n][j], sc[n]);
        stage = stage == (NS - 1u) * S::STAGE ? 0u : stage + S::STAGE;
        sw = swNext;
    }

    // ---- the four waves' sums
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int j = 0; j < NJ; ++j) *(v4f *)(ring + (n * NJ + j) * 1024u + lane * 16u) = acc[n][j];
    __syncthreads();
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        const uint32_t f = wave + 4u * v;
        if (have[v] == 0) continue;
        v4f sum = *(const v4f *)(smem + f * 1024u + lane * 16u);
#pragma unroll
        for (uint32_t u = 1; u < 4u; ++u) {
            const v4f part = *(const v4f *)(smem + u * S::WAVE + f * 1024u + lane * 16u);
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[r] += part[r];
        }
        if constexpr (DT == DT_F8) add_peers4<BATCH>(args, t.row + vr[v], col0 + vc[v], sum, have[v], peer[v]);
        store4(args, (size_t)(t.row + vr[v]) * args.n + col0 + vc[v], sum, have[v]);
    }
}

}  // namespace catcoc
