// Ragged products on large tiles fed by copies that go straight to LDS.
//
// What bounds them: a step of a 256x256 tile multiplies 64 KiB that come from the L2 at 56 to 72 GB/s a CU, about as long as its MFMAs take in 16 bits and e4m3
// alike (a step is 128 bytes of k).  So tiles are as large as registers allow, and a copy has a whole step or two to arrive.  Measured: e4m3 8192x27392x4096 750 us
// (2.45 PFLOP/s; a library product of 8192^3 reaches 2.73), 16384 rows in 62 groups of 4096x3584 in 16 bits 570 us (840 TFLOP/s, 3.6 TB/s), in e4m3 320 us (1.5
// PFLOP/s), weight gradients of 8 uneven groups of together 16384 rows, 4096x1792, 226 us (1.07 PFLOP/s; 240 with the groups in their own order).
#pragma once
#include "ragged_checked.h"

namespace catcoc {

// 16 (4) bytes per lane to LDS: lane l lands at ldsAddr + 16 l (4 l).  A scalar base and 32-bit lane offsets: no 64-bit address per copy to keep and to advance.
__device__ __forceinline__ void copy16(const unsigned char *base, uint32_t off, uint32_t ldsAddr)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(ldsAddr) : "memory", "m0");
}
__device__ __forceinline__ void copy4(const unsigned char *base, uint32_t off, uint32_t ldsAddr)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "s"(ldsAddr) : "memory", "m0");
}

// Scalar loads: the address is the same for every lane, the memory is not written while the kernel runs.
__device__ __forceinline__ float load_uniform(const float *p) { return *(const __attribute__((address_space(4))) float *)p; }

template <typename T>
__device__ __forceinline__ T *uniform_ptr(T *p)
{
    const uint64_t u = (uint64_t)p;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
    return (T *)(((uint64_t)hi << 32) | lo);
}

// Where an operand's pieces of one step lie, in memory and in LDS, in sub-stages of 16 KiB: 128 rows of 128 bytes of k, or (KM) 64 rows of k of 128 columns.
//   KM = false: piece p of row r at slot p ^ k_rows_slot(r).   KM = true: piece p of row r at slot p ^ b16_slot<2>(r).
// A sub-stage's two halves of 64 rows (columns) are `apart` rows (columns) of the tile apart.  Rows and columns past the tile's last one repeat it.
template <bool KM, uint32_t SUBS, uint32_t ES, uint32_t WAVES>
struct TileOperand {
    static constexpr uint32_t COPIES = 16u / WAVES;   // of a wave and sub-stage, 1 KiB each
    const unsigned char *base;   // the tile's first row and column, first step
    uint32_t pitch, have, apart;
    bool packed;                 // of the second sub-stage only 16 rows of either half are there, 4 KiB
    uint32_t off[SUBS][COPIES];

    // The row (column) of the tile that row (column) q of sub-stage h holds.
    __device__ __forceinline__ uint32_t of_tile(uint32_t h, uint32_t q) const
    {
        const uint32_t log = !KM && h == 1u && packed ? 4u : 6u;
        return (q >> log) * apart + 64u * h + (q & ((1u << log) - 1u));
    }
    // Copies between a wave's first and second of a sub-stage.
    __device__ __forceinline__ uint32_t stride(uint32_t h) const { return !KM && h == 1u && packed ? 2u : WAVES; }
    // Byte of the tile's step that byte `in` of the 16-byte slot `slot` of LDS row `row` holds.
    __device__ __forceinline__ uint32_t source(uint32_t h, uint32_t row, uint32_t slot, uint32_t in) const
    {
        if constexpr (KM) {
            const uint32_t piece = of_tile(h, (slot ^ b16_slot<2>(row)) * 8u) / 8u;
            return row * pitch + umin(piece, (have - 1u) / 8u) * 16u + in;
        } else {
            return umin(of_tile(h, row), have - 1u) * pitch + (slot ^ k_rows_slot(row)) * 16u + in;
        }
    }
    __device__ __forceinline__ void init(const unsigned char *p, uint32_t pitch_, uint32_t have_, uint32_t apart_, bool packed_, uint32_t wave, uint32_t lane)
    {
        base = uniform_ptr(p);
        pitch = pitch_;
        have = have_;
        apart = apart_;
        packed = packed_;
#pragma unroll
        for (uint32_t h = 0; h < SUBS; ++h)
#pragma unroll
            for (uint32_t j = 0; j < COPIES; ++j) {
                const uint32_t at = (wave + stride(h) * j) * 64u + lane;
                off[h][j] = source(h, KM ? at >> 4 : at >> 3, KM ? at & 15u : at & 7u, 0);
            }
    }
    __device__ __forceinline__ const unsigned char *at_step(uint32_t s) const { return base + (size_t)s * (KM ? 64u * pitch : 128u); }
    // (rows: sixteen of them that no wave reads are left out; eight waves only, where that is all of a wave's copies or none)
    static __device__ __forceinline__ bool wanted(uint32_t h, uint32_t ni, uint32_t wave) { return KM || WAVES != 8u || 4u * h + (wave >> 1) < ni; }
    __device__ __forceinline__ void issue(uint32_t h, uint32_t s, uint32_t lds, uint32_t wave) const
    {
        const unsigned char *const p = at_step(s);
#pragma unroll
        for (uint32_t j = 0; j < COPIES; ++j) copy16(p, off[h][j], lds + (wave + stride(h) * j) * 1024u);
    }
    // The last step where it ends inside its 128 bytes of k or 64 rows of k, or where pieces of 16 bytes would end behind the matrix: copies of what is there (4
    // bytes at a time where a row ends inside a piece), and zeros.  inRow: bytes of a row that are there, from the step's first (KM: the tile's first column) on;
    // rows: rows of k (KM).
    __device__ __forceinline__ void issue_part(uint32_t h, uint32_t s, unsigned char *stage, uint32_t lds, uint32_t inRow, uint32_t rows, uint32_t wave, uint32_t lane) const
    {
        if (inRow % 16u == 0) part<16>(h, s, stage, lds, inRow, rows, wave, lane);
        else part<4>(h, s, stage, lds, inRow, rows, wave, lane);
    }
    template <uint32_t BYTES>
    __device__ __forceinline__ void part(uint32_t h, uint32_t s, unsigned char *stage, uint32_t lds, uint32_t inRow, uint32_t rows, uint32_t wave, uint32_t lane) const
    {
        constexpr uint32_t PER = (KM ? 256u : 128u) / BYTES;   // copied pieces of a row
        const unsigned char *const p = at_step(s);
#pragma unroll 1
        for (uint32_t c = wave; c < (!KM && h == 1u && packed ? 64u : 256u) / BYTES; c += WAVES) {
            const uint32_t at = c * 64u + lane, row = at / PER, slot = (at % PER) * BYTES / 16u, in = at * BYTES % 16u;
            const uint32_t byte = KM ? of_tile(h, (slot ^ b16_slot<2>(row)) * 8u) * 2u + in : (slot ^ k_rows_slot(row)) * 16u + in;
            const bool there = byte < inRow && (!KM || row < rows);
            if (there) {
                if constexpr (BYTES == 16u) copy16(p, source(h, row, slot, in), lds + c * 1024u);
                else copy4(p, source(h, row, slot, in), lds + c * 256u);
            } else if constexpr (BYTES == 16u) {
                *(v4i *)(stage + at * 16u) = v4i{0, 0, 0, 0};
            } else {
                *(uint32_t *)(stage + at * 4u) = 0u;
            }
        }
    }
};

// Which column of its 16 a matrix fragment's lane m holds: 0-3, 8-11, 4-7, 12-15.  The results of lane groups 0 and 2 (1 and 3) are then eight consecutive
// columns, and one exchange of half waves between two column blocks gives every lane 16 bytes of output.
__device__ __forceinline__ uint32_t result_col(uint32_t m) { return ((m >> 2) & 1u) * 8u + ((m >> 3) & 1u) * 4u + (m & 3u); }

// A tile of 32 NIMAX rows and 64 WY columns: 2 WY waves, two by WY, of up to 16 NIMAX rows and 64 columns each (NI row fragments, as many as the tile's rows
// need; four of columns).  A wave keeps a step's column fragments in registers and streams its row fragments, two ahead of the MFMAs.
//
// Two stages of 128 bytes of k, three with eight waves and at most five row fragments each (their stages are smaller).  When the last read of a step is out, the
// wave waits for the next stage's copies (issued a whole step before, or several) and for its own reads; the barrier behind that says both that the next stage
// is complete and that this one may be overwritten: its next copies start there.  The last two row fragments' MFMAs then cover the first reads of the next
// step, whose column fragments take the registers of those just used.
//
// KG = 2: two teams of 2 WY waves multiply every other step of the same tile, each through stages of its own, and add their sums at the end (team 0's first).
// A launch of at most one tile per CU else has one wave on a SIMD, which pays for barrier, LDS and issue one after the other (512 rows of e4m3 times 8192x8192:
// 128x128 with one team 60 us, with two 52; 4096x4096 25 and 20 on 64x128).
template <uint32_t DT, bool XK, bool WK, int WY, int NIMAX, int KG>
struct RaggedTileLoop {
    static constexpr uint32_t ES = DT == DT_F8 ? 1u : 2u, KE = 128u / ES;
    static constexpr uint32_t WAVES = 2u * WY, BX = 32u * NIMAX, BY = 64u * WY, SUB = 16384u;
    static constexpr uint32_t XSUBS = BX / 128u, WSUBS = BY / 128u;
    static constexpr bool PACK = NIMAX == 8 && !XK;   // five row fragments a wave: the fifth ones packed, so that three stages fit
    static constexpr uint32_t stages(int ni) { return NIMAX == 8 && ni <= (PACK ? 5 : 4) ? 3u : 2u; }
    static constexpr uint32_t x_bytes(int ni) { return ni <= 4 ? SUB : PACK && ni == 5 ? SUB + 4096u : 2u * SUB; }
    static constexpr uint32_t stage_bytes(int ni) { return x_bytes(ni) + WSUBS * SUB; }
    static constexpr uint32_t SX = NIMAX == 8 ? (XK ? 2u * stage_bytes(8) : 3u * stage_bytes(5)) : 2u * stage_bytes(4);   // e4m3: row scales behind the stages
    static constexpr uint32_t SXB = BX * 4u, SXN = NIMAX == 8 ? 3u : 2u;
    static constexpr uint32_t LDS = SX + (DT == DT_F8 ? SXN * SXB : 0u);   // of a team
    static_assert(KG == 1 || (KG == 2 && NIMAX * WAVES * 2048u <= SX), "two teams: half of a team's sums fit its stages");
    TileOperand<XK, XSUBS, ES, WAVES> x;
    TileOperand<WK, WSUBS, ES, WAVES> w;
    v4f acc[NIMAX][4];

    struct Problem {
        uint32_t K, steps;          // values of k, this team's steps of them
        uint32_t rounds, team;      // steps of the team that has most; which one this is
        uint32_t rows, cols;        // of the tile
        uint32_t ni;                // row fragments of a wave
        uint32_t xLeft, wLeft;      // columns of the matrix from the tile's first on (operands that are rows of k)
        bool partLast;              // the last step is no whole one (issue_part)
        const float *sx, *sw;       // e4m3: scales of the tile's first row, and of this wave's block of columns
        uint32_t sxPitch;
    };

    static __device__ __forceinline__ uint32_t of_all(const Problem &p, uint32_t s) { return KG * s + (KG > 1 ? p.team : 0u); }

    // Copies of the team's step s into `stage`.
    template <int NI>
    __device__ __forceinline__ void issue(const Problem &p, unsigned char *smem, uint32_t stage, uint32_t s, uint32_t wave, uint32_t lane)
    {
        const uint32_t lds0 = (uint32_t)(uintptr_t)(CATCOC_LDS unsigned char *)smem, ws = stage + x_bytes(NI);
        constexpr bool TWO = NI > 4;
        if (p.partLast && s + 1u == p.steps) {
            const uint32_t left = p.K - of_all(p, s) * KE;
#pragma unroll 1
            for (uint32_t h = 0; h < WSUBS; ++h) w.issue_part(h, of_all(p, s), smem + ws + h * SUB, lds0 + ws + h * SUB, WK ? p.wLeft * 2u : left * ES, left, wave, lane);
#pragma unroll 1
            for (uint32_t h = 0; h < (TWO ? 2u : 1u); ++h) x.issue_part(h, of_all(p, s), smem + stage + h * SUB, lds0 + stage + h * SUB, XK ? p.xLeft * 2u : left * ES, left, wave, lane);
        } else {
#pragma unroll
            for (uint32_t h = 0; h < WSUBS; ++h) w.issue(h, of_all(p, s), lds0 + ws + h * SUB, wave);
#pragma unroll
            for (uint32_t h = 0; h < (TWO ? 2u : 1u); ++h)
                if (x.wanted(h, p.ni, wave)) x.issue(h, of_all(p, s), lds0 + stage + h * SUB, wave);
        }
        if constexpr (DT == DT_F8) {   // 64 rows' scales a wave (several waves fetch the same ones)
            const uint32_t q = wave % (BX / 64u);
            copy4((const unsigned char *)(p.sx + (size_t)of_all(p, s) * p.sxPitch), umin(64u * q + lane, p.rows - 1u) * 4u, lds0 + SX + s % SXN * SXB + q * 256u);
        }
    }

    // A tile's first copies.
    template <int NI>
    __device__ __forceinline__ void first(const Problem &p, unsigned char *smem, uint32_t wave, uint32_t lane)
    {
#pragma unroll 1
        for (uint32_t s = 0; s < stages(NI) && s < p.steps; ++s) issue<NI>(p, smem, s * stage_bytes(NI), s, wave, lane);
    }
    __device__ __forceinline__ void begin(const Problem &p, unsigned char *smem, uint32_t wave, uint32_t lane)
    {
        if constexpr (NIMAX == 8) {
            if (p.ni > 5u) return first<8>(p, smem, wave, lane);
            if (p.ni == 5u) return first<5>(p, smem, wave, lane);
        }
        first<4>(p, smem, wave, lane);
    }

    // All but this wave's copies of the last N steps are there where `whole` steps follow, else all; then everybody's are, and everybody's reads are done.
    template <int N>
    __device__ __forceinline__ void meet(bool whole, bool first, bool second)
    {
        constexpr int C = (int)(16u / WAVES), W = N * (C * (int)WSUBS + (DT == DT_F8 ? 1 : 0));
        if (N == 0 || !whole) CATCOC_WAIT_VMCNT(0);
        else if (second) CATCOC_WAIT_VMCNT(W + 2 * N * C);
        else if (first) CATCOC_WAIT_VMCNT(W + N * C);
        else CATCOC_WAIT_VMCNT(W);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        barrier_keep_vmem();
    }

    template <int NI>
    __device__ __forceinline__ void run(const Problem &p, unsigned char *smem, uint32_t wave, uint32_t lane)
    {
        static_assert(NI >= 2 && NI <= NIMAX, "row fragments of a wave");
        constexpr bool TWO = NI > 4;   // (row fragments in two sub-stages)
        constexpr uint32_t STAGES = stages(NI), STAGE = stage_bytes(NI);
        const uint32_t wr = wave / WY, wc = wave % WY;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        if (p.rounds == 0) return;
        const uint32_t full = p.steps - (p.partLast ? 1u : 0u);   // whole steps
        const bool first = TWO || x.wanted(0, NI, wave), second = TWO && x.wanted(1, NI, wave);
        meet<(int)STAGES - 1>(full >= STAGES, first, second);

        const uint32_t xa = XK ? at_k_major<false>(256u, 64u * wr, lane, b16_slot<2>) : at_k_rows(64u * wr + (lane & 15u), lane);
        const uint32_t x4 = SUB + at_k_rows(16u * wr + (lane & 15u), lane);   // (packed: the fifth row fragment)
        const uint32_t wh = WSUBS == 2u ? wc % 2u : 0u, w64 = 64u * (WSUBS == 2u ? wc / 2u : wc);   // the wave's columns: sub-stage, half of it
        uint32_t wa = x_bytes(NI) + wh * SUB + (WK ? at_k_major<true>(256u, w64, lane, b16_slot<2>) : at_k_rows(w64 + result_col(lane & 15u), lane));
        // Two teams: team 1 has its column blocks in the order 2, 3, 0, 1, so that 0 and 1 are those that either team stores.
        if (KG > 1 && p.team) wa ^= WK ? 64u : 4096u;
        auto read_x = [&](uint32_t stage, uint32_t i) {
            if constexpr (XK) return frag_k_major<256>(smem, ((stage + xa) ^ (32u * (i & 3u))) + (i >> 2) * SUB);
            else if (PACK && NI == 5 && i == 4u) return frag_k_rows(smem, stage + x4);
            else return frag_k_rows(smem, stage + xa + 2048u * (i & 3u) + (i >> 2) * SUB);
        };
        auto read_w = [&](uint32_t stage, uint32_t j) {
            if constexpr (WK) return frag_k_major<256>(smem, (stage + wa) ^ (32u * j));
            else if constexpr (KG > 1) return frag_k_rows(smem, ((stage + wa) ^ (j / 2u * 4096u)) + 2048u * (j % 2u));
            else return frag_k_rows(smem, stage + wa + 2048u * j);
        };
        const uint32_t sa = SX + (wr * 16u * NI + (lane & 15u)) * 4u;
        auto row_scale = [&](uint32_t s, int i) { return *(const float *)(smem + sa + s % SXN * SXB + 64u * i); };

        // Row fragments' registers: the first two of a step have their own, which are free when the last two run.
        constexpr int SLOTS = NI == 8 ? 4 : NI >= 4 ? 5 : NI;
        auto slot = [](int i) { return NI == 8 ? i & 3 : i < 2 || NI < 4 ? i : 2 + (i - 2) % 3; };
        Frag fx[SLOTS], fw[4], ahead[2];
        float fs[SLOTS], aheadS[2], sw = 0.f;   // e4m3: the fragments' row scales, the columns' scale
        constexpr int LAG = 3;   // e4m3: a result is scaled and added while the MFMAs behind it run
        v4f late[LAG];
        float lateS[LAG];
        int li[LAG], lj[LAG], queued = 0;
        auto settle = [&](int q) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[li[q]][lj[q]][r] = __builtin_fmaf(lateS[q], late[q][r], acc[li[q]][lj[q]][r]);
            asm volatile("" : "+v"(acc[li[q]][lj[q]]));   // (here, and not all of them together behind the next branch)
        };
        auto multiply = [&](int i, int j, const Frag &f, float scale) {
            if constexpr (DT == DT_F8) {
                const v4f d = step_mfma_f8(fw[j], f);
                if (queued >= LAG) settle(queued % LAG);
                late[queued % LAG] = d;
                lateS[queued % LAG] = scale;
                li[queued % LAG] = i;
                lj[queued % LAG] = j;
                ++queued;
                __builtin_amdgcn_sched_barrier(0);
            } else {
                step_mfma<DT>(fw[j], f, acc[i][j], 0.f);
            }
        };
#pragma unroll
        for (int j = 0; j < 4; ++j) fw[j] = read_w(0, j);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fx[i] = read_x(0, i);
            if constexpr (DT == DT_F8) fs[i] = row_scale(0, i);
        }
        if constexpr (DT == DT_F8) sw = load_uniform(p.sw + (KG > 1 ? min(p.team, (p.K - 1u) / KE) : 0u));
        // Of the two waves on a SIMD one starts its copies behind the barrier, the other at the next step's start: while copies wait for their issue the other one
        // multiplies (e4m3 8192x27392x4096 817 -> 750 us).
        const bool early = WAVES != 8u || wave < WAVES / 2u;
        uint32_t cur = 0;   // this step's stage
#pragma unroll 1
        for (uint32_t s = 0; s < p.rounds; ++s) {
            if (KG > 1 && s >= p.steps) {   // (the other team has one more)
                meet<0>(false, first, second);
                break;
            }
            const uint32_t next = cur == (STAGES - 1u) * STAGE ? 0u : cur + STAGE;
            queued = 0;
            if (!early && s > 0u && s + STAGES - 1u < p.steps) issue<NI>(p, smem, cur == 0u ? (STAGES - 1u) * STAGE : cur - STAGE, s + STAGES - 1u, wave, lane);
            float swNext = 0.f;
            if constexpr (DT == DT_F8) {   // (asked for here: its wait is the one for the step's reads)
                swNext = load_uniform(p.sw + umin(of_all(p, s + 1u), (p.K - 1u) / KE));
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < NI - 2; ++i) {
                fx[slot(i + 2)] = read_x(cur, i + 2);
                if constexpr (DT == DT_F8) fs[slot(i + 2)] = row_scale(s, i + 2);
                const float scale = DT == DT_F8 ? fs[slot(i)] * sw : 0.f;
#pragma unroll
                for (int jj = 0; jj < 4; ++jj) multiply(i, snake16(i, jj, 4), fx[slot(i)], scale);
                __builtin_amdgcn_sched_barrier(0);
            }
            meet<(int)STAGES - 2>(s + STAGES <= full, first, second);
            if (early && s + STAGES < p.steps) issue<NI>(p, smem, cur, s + STAGES, wave, lane);
            // (behind the last step nobody looks at what is read here)
            const float s0 = DT == DT_F8 ? fs[slot(NI - 2)] * sw : 0.f, s1 = DT == DT_F8 ? fs[slot(NI - 1)] * sw : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                Frag &to = NI >= 4 ? fx[i] : ahead[i];
                to = read_x(next, i);
                if constexpr (DT == DT_F8) (NI >= 4 ? fs[i] : aheadS[i]) = row_scale(s + 1u, i);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                multiply(NI - 2, j, fx[slot(NI - 2)], s0);
                multiply(NI - 1, j, fx[slot(NI - 1)], s1);
                fw[j] = read_w(next, j);
            }
            if constexpr (DT == DT_F8) {
#pragma unroll
                for (int q = 0; q < LAG; ++q) settle((queued + q) % LAG);
                sw = swNext;
            }
            if constexpr (NI < 4) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    fx[i] = ahead[i];
                    if constexpr (DT == DT_F8) fs[i] = aheadS[i];
                }
            }
            cur = next;
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Two teams: each gets the other's sums of the columns that it stores.
    __device__ __forceinline__ void join(const Problem &p, unsigned char *all, uint32_t wave, uint32_t lane)
    {
        // (all reads of the stages were before the last barrier)
        unsigned char *const to = all + p.team * LDS + wave * (NIMAX * 2048u) + lane * 16u, *const from = all + (1u - p.team) * LDS + wave * (NIMAX * 2048u) + lane * 16u;
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)NIMAX; ++i)
            if (i < p.ni) {
                *(v4f *)(to + 2048u * i) = acc[i][2];
                *(v4f *)(to + 2048u * i + 1024u) = acc[i][3];
            }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)NIMAX; ++i)
            if (i < p.ni) {
                const v4f a = *(const v4f *)(from + 2048u * i), b = *(const v4f *)(from + 2048u * i + 1024u);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    acc[i][0][r] += a[r];
                    acc[i][1][r] += b[r];
                }
            }
    }

    template <int NI = NIMAX>
    __device__ __forceinline__ void run_rows(const Problem &p, unsigned char *smem, uint32_t wave, uint32_t lane)
    {
        if (p.ni == (uint32_t)NI || NI == 2) run<NI>(p, smem, wave, lane);
        else if constexpr (NI > 2) run_rows<NI - 1>(p, smem, wave, lane);
    }
};

// DW: x and w are rows of k (the group's rows), the result is the group's [k, n] matrix.  KN: w is [k, n].
// A weight gradient's workgroups walk several tiles: few rows make few steps, and a tile's first copies are on their way while the one before is stored.
// 4099 rows in 16 groups (one without rows), 4096x3584 in fp32, 327 us: 150 without the stores, and the stores alone take 178 in this order (940 MB, 5.3 TB/s).
// They hardly overlap: vmcnt counts copies and stores in their order, so the wait for a tile's first step, whose copies are older than the stores, lets 24 of a
// wave's 32 stores finish too, and directly behind it five of the 11 registers that this kernel spills come back one after the other, each behind all that is under way.
// 128x256 tiles that store a tile piece by piece between the next one's steps took 373 us, five stages of 32 rows that leave 2.5 us of work in LDS 326 (and
// the long sums of 8 groups of 2048 rows 271 instead of 240).
template <uint32_t DT, bool KN, bool DW, int WY, int NIMAX, int KG>
__global__ void __launch_bounds__(128 * WY * KG, 2) ragged_tile_kernel(const RaggedArgs args)
{
    using Loop = RaggedTileLoop<DT, DW, KN || DW, WY, NIMAX, KG>;
    constexpr uint32_t ES = Loop::ES, BX = Loop::BX, BY = Loop::BY;
    static_assert(!DW || KG == 1, "a weight gradient's tiles have one team");
    __shared__ __attribute__((aligned(16))) unsigned char lds[KG * Loop::LDS];

    const uint32_t tid = threadIdx.x, lane = tid & 63u, waves = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const uint32_t wave = waves % Loop::WAVES, team = waves / Loop::WAVES;
    unsigned char *const smem = lds + team * Loop::LDS;
    const uint32_t nt = (args.n + BY - 1u) / BY;
    Loop loop;
    typename Loop::Problem p;

    uint32_t order = 0;   // DW: lane i's group is the i-th of up to 64, those with most rows first
    if constexpr (DW) {
        if (args.groups <= 64u) {
            uint32_t b = 0, e = 0, rank = lane;
            if (lane < args.groups) group_rows(args, lane, b, e);
            if (lane < args.groups) rank = 0;
            for (uint32_t g = 0; g < args.groups; ++g) {
                const uint32_t rows = (uint32_t)__builtin_amdgcn_readlane((int)(e - b), (int)g);
                if (lane < args.groups) rank += rows > e - b || (rows == e - b && g < lane) ? 1u : 0u;
            }
            order = (uint32_t)__builtin_amdgcn_ds_permute((int)(rank * 4u), (int)lane);
        }
    }
    // Tile `at` of this launch; DW: t.group's rows are the sum, t.row and t.rows rows of the result.
    uint32_t sumBegin = 0, sumEnd = 0;
    auto find = [&](uint32_t &at, RaggedTile &t) {
        if constexpr (DW) {
            // every XCD gets an eighth of each group's tiles: they cost what the group has rows; its workgroups take them in turns, forth and back
            const uint32_t pt = (args.k + BX - 1u) / BX, tiles = pt * nt, share = (tiles + 7u) / 8u;
            uint32_t in;
            do {
                const uint32_t per = gridDim.x >> 3, turn = (at >> 3) / per, place = (at >> 3) - turn * per, j = turn * per + (turn & 1u ? per - 1u - place : place);
                if (j >= args.groups * share) return false;
                t.group = j / share;
                in = ((at + t.group) & 7u) * share + j - t.group * share;
                if (args.groups <= 64u) t.group = (uint32_t)__builtin_amdgcn_readlane((int)order, (int)__builtin_amdgcn_readfirstlane((int)t.group));
                if (in >= tiles) at += gridDim.x;
            } while (in >= tiles);
            t.colTile = in / pt;
            t.row = BX * (in - t.colTile * pt);
            t.rows = umin(BX, args.k - t.row);
            t.group = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.group);
            t.colTile = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.colTile);
            t.row = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.row);
            t.rows = (uint32_t)__builtin_amdgcn_readfirstlane((int)t.rows);
            group_rows(args, t.group, sumBegin, sumEnd);
            sumBegin = (uint32_t)__builtin_amdgcn_readfirstlane((int)sumBegin);
            sumEnd = (uint32_t)__builtin_amdgcn_readfirstlane((int)sumEnd);
            return true;
        } else {
            return ragged_tile(args, at, args.tileRows, nt, 32u, t);
        }
    };
    auto set = [&](const RaggedTile &t) {
        const uint32_t col0 = BY * t.colTile;
        p.wLeft = args.n - col0;
        p.rows = t.rows;
        p.cols = umin(BY, p.wLeft);
        p.ni = DW ? (uint32_t)NIMAX : max((t.rows + 31u) / 32u, 2u);
        if constexpr (DW) {
            p.K = sumEnd - sumBegin;
            p.xLeft = args.k - t.row;
            p.partLast = p.K % 64u != 0 || args.k % 8u != 0 || args.n % 8u != 0;
            loop.x.init((const unsigned char *)args.x + ((size_t)sumBegin * args.k + t.row) * 2u, args.k * 2u, t.rows, 16u * NIMAX, false, wave, lane);
            loop.w.init((const unsigned char *)args.w + ((size_t)sumBegin * args.n + col0) * 2u, args.n * 2u, p.cols, BY / 2u, false, wave, lane);
        } else {
            const uint32_t g = umin(t.group, args.groups - 1u);
            p.K = t.group < args.groups ? args.k : 0u;
            const uint32_t wPitch = KN ? args.n * ES : args.k * ES;
            p.xLeft = 0;
            p.partLast = p.K % Loop::KE != 0 || (KN && args.n % 8u != 0);
            loop.x.init((const unsigned char *)args.x + (size_t)t.row * args.k * ES, args.k * ES, t.rows, 16u * p.ni, Loop::PACK && p.ni == 5u, wave, lane);
            loop.w.init((const unsigned char *)args.w + (size_t)g * args.n * args.k * ES + (size_t)col0 * (KN ? ES : wPitch), wPitch, p.cols, BY / 2u, false, wave, lane);
            if constexpr (DT == DT_F8) {
                const uint32_t kb = (args.k + kScaleBlock - 1u) / kScaleBlock, nb = (args.n + kScaleBlock - 1u) / kScaleBlock;
                p.sx = uniform_ptr(args.sx + t.row);
                p.sxPitch = args.rows;
                p.sw = uniform_ptr(args.sw + ((size_t)g * nb + umin((col0 + (wave % WY) * 64u) / kScaleBlock, nb - 1u)) * kb);
            }
        }
        p.steps = (p.K + Loop::KE - 1u) / Loop::KE;
        p.rounds = (p.steps + KG - 1u) / KG;
        p.team = team;
        if constexpr (KG > 1) {
            p.partLast = p.partLast && (p.steps - 1u) % KG == team;
            p.steps = p.steps > team ? (p.steps - team + KG - 1u) / KG : 0u;
        }
    };

    uint32_t at = blockIdx.x;
    RaggedTile t;
    if (!find(at, t)) return;
    set(t);
    loop.begin(p, smem, wave, lane);
    for (;;) {
        // DW: a workgroup's next tile is looked up while this one's first copies are on their way, and its own start before this one's results are stored
        RaggedTile after;
        bool more = false;
        const size_t outRow = (DW ? (size_t)t.group * args.k : (size_t)0) + t.row;
        const uint32_t ni = p.ni;
        if constexpr (DW) {
            at += gridDim.x;
            more = find(at, after);
            loop.template run<NIMAX>(p, smem, wave, lane);
        } else {
            loop.run_rows(p, smem, wave, lane);
            if constexpr (KG > 1) loop.join(p, lds, wave, lane);
        }
        const uint32_t rows = t.rows, row0 = t.row, col0 = BY * t.colTile, cols = p.cols;
        if (more) {
            t = after;
            set(t);
            loop.begin(p, smem, wave, lane);
        }

        // ---- output: rows [wr, +16 ni) and columns [wc, +64) of the tile are this wave's (two teams: half of the columns each)
        constexpr uint32_t NJ = KG == 1 ? 4u : 2u;   // column blocks that this wave stores
        const uint32_t wr = (wave / WY) * 16u * ni, wc = (wave % WY) * 64u + 32u * team, lr = lane & 15u;
        if (DW && args.outType == 0) {
#pragma unroll
            for (uint32_t i = 0; i < (uint32_t)NIMAX; ++i) {
                const uint32_t r = wr + 16u * i + lr;
                if (i >= ni || r >= rows) continue;
#pragma unroll
                for (uint32_t j = 0; j < NJ; ++j) {
                    const uint32_t c = wc + 16u * j + result_col((lane >> 4) * 4u);
                    if (c < cols) store4(args, (outRow + r) * args.n + col0 + c, loop.acc[i][j], umin(4u, cols - c));
                }
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < (uint32_t)NIMAX; ++i) {
                const uint32_t r = wr + 16u * i + lr;
                if (i >= ni) continue;
                if constexpr (DT == DT_F8) {
                    if (args.nPeers && r < rows) {
#pragma unroll
                        for (uint32_t j = 0; j < NJ; ++j) {
                            const uint32_t c = wc + 16u * j + result_col((lane >> 4) * 4u);
                            if (c < cols) add_peers4(args, row0 + r, col0 + c, loop.acc[i][j], umin(4u, cols - c));
                        }
                    }
                }
#pragma unroll
                for (uint32_t j = 0; j < NJ; j += 2u) {   // lanes 0-31: block j, lanes 32-63: block j + 1, eight columns each
                    const v4f a = loop.acc[i][j], b = loop.acc[i][j + 1u];
                    const auto lo = __builtin_amdgcn_permlane32_swap(round2(a[0], a[1], args.outType), round2(b[0], b[1], args.outType), false, false);
                    const auto hi = __builtin_amdgcn_permlane32_swap(round2(a[2], a[3], args.outType), round2(b[2], b[3], args.outType), false, false);
                    const uint32_t c = wc + 16u * (j + (lane >> 5)) + 8u * ((lane >> 4) & 1u);
                    if (r < rows && c < cols) store8_16bit(args, (outRow + r) * args.n + col0 + c, v4i{(int)lo[0], (int)hi[0], (int)lo[1], (int)hi[1]}, umin(8u, cols - c));
                }
            }
        }
        if (!more) return;
    }
}

}  // namespace catcoc
