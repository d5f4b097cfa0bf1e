// az_tile.hpp -- the matrix tile that the int8 products (az_int8.hip) and the split-fp16 products (az_ortho.hip) share.
//
// D[m][n] = sum_k P[m][k] Q[n][k]: both operands run along their rows, 64 bytes of a row per step (TILE_KB): 64 int8 values,
// or 16 values as 16 fp16 high halves and their 16 low halves.  A step's BM + BN rows go from memory straight into LDS
// (buffer_load ... lds, 16 bytes a lane: no registers, no address arithmetic but one scalar add) into a ring of STAGES buffers,
// STAGES - 1 steps ahead of the products.  A wave computes FM x FN blocks of 32 x 32.
//
// In LDS a row is 4 pieces of 16 bytes (one lane's operand of a 32x32 MFMA); piece p of row r sits at p ^ ((r >> 2) & 3): 16 rows
// read at one p then touch all 64 banks once (rows are 64 bytes = 16 banks apart, so r & 3 picks the quarter and r >> 2 the
// piece).  The loads write LDS in lane order, so the exchange is made in the address they read from.
#pragma once
#include "az_ops.hpp"

namespace az {

constexpr int TILE_KB = 64;
__device__ inline int tile_off(int row, int piece) { return row * TILE_KB + ((piece ^ ((row >> 2) & 3)) << 4); }
// 32x32 MFMA result: lane holds column (lane & 31) and, in register r, row
__device__ inline int acc_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

typedef __attribute__((address_space(3))) void lds_void;

// one operand: rows `ld` bytes apart, a step's 64 bytes of them `kstep` bytes behind those of the step before.  Rows of the caller
// (int8): ld is the row, kstep 64.  Operands of our own are kept in panels, a step's 64 bytes of all rows together: ld is 64 and
// a step's tile one run of memory (rows a power of two apart crowd into a few channels of L2).
// Reads behind `bytes` from a step's first row on give zeros.
// PAIRS: of every 64 rows the even ones come first, then the odd ones.  A wave with two blocks of 32 columns then holds columns
// 2 c and 2 c + 1 in lane c, and stores them together.
template <bool PAIRS>
struct TileSrc {
    const u8* base;
    u64 kstep;
    u32 bytes, ld, voff, piece;   // this lane's row and piece inside a group of 16 rows
    __device__ TileSrc(const void* base_, u64 kstep_, u32 ld_, u32 bytes_, int lane)
        : base((const u8*)base_), kstep(kstep_), bytes(bytes_), ld(ld_) {
        piece = (u32)(((lane & 3) ^ (lane >> 4)) << 4);
        voff = (u32)(lane >> 2) * (PAIRS ? 2 : 1) * ld + piece;
    }
    // first row of the 16 that go to the tile's rows row..row + 15
    __device__ static u32 source_row(u32 row) { return PAIRS ? (row & ~63u) + 2 * (row & 31) + (row >> 5 & 1) : row; }
};

// ROWS rows x 64 bytes of step `step` into `tile`; pieces at or behind byte `kend` (a multiple of 16) of the rows become zeros
template <int ROWS, int WAVES, bool PAIRS>
__device__ inline void tile_load(const TileSrc<PAIRS>& s, u32 step, u32 kend, u8* tile, int wave) {
    static_assert(ROWS % (16 * WAVES) == 0, "every wave loads whole groups of 16 rows");
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<u8*>(s.base + step * s.kstep), 0, (int)s.bytes, 0x00020000);
    const u32 voff = step * TILE_KB + s.piece < kend ? s.voff : 0x7ffffff0u;   // out of range: the buffer gives zeros
#pragma unroll
    for (int i = 0; i < ROWS / (16 * WAVES); i++) {
        const u32 row = (u32)(i * WAVES + wave) * 16;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(tile + row * TILE_KB), 16, (int)voff,
                                                 (int)(s.source_row(row) * s.ld), 0, 0);
    }
}

// One k-slice of a step in registers: KS slices make up a step; read() asks LDS for slice ks of the wave's FM + FN blocks of 32
// rows (from row wm of tile P, wn of tile Q), mul() multiplies it.  READS per block of rows, MULS per block of the result.
struct KindI8 {
    typedef i32x16 acc_t;
    static constexpr int KS = 2, READS = 1, MULS = 1;   // 32 values each
    template <int FM, int FN>
    struct Slice {
        i32x4 a[FM], b[FN];
        __device__ inline void read(const u8* tp, const u8* tq, int wm, int wn, int ks, int lane) {
            const int r = lane & 31, piece = 2 * ks + (lane >> 5);
#pragma unroll
            for (int f = 0; f < FM; f++) a[f] = *(const i32x4*)(tp + tile_off(wm + 32 * f + r, piece));
#pragma unroll
            for (int f = 0; f < FN; f++) b[f] = *(const i32x4*)(tq + tile_off(wn + 32 * f + r, piece));
        }
        __device__ inline void mul(i32x16 (&acc)[FM][FN]) const {
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    };
};
struct KindSplit {
    typedef f32x16 acc_t;
    static constexpr int KS = 1, READS = 2, MULS = 3;   // 16 values: high halves in pieces 0, 1, low halves in 2, 3
    template <int FM, int FN>
    struct Slice {
        f16x8 ah[FM], al[FM], bh[FN], bl[FN];
        __device__ inline void read(const u8* tp, const u8* tq, int wm, int wn, int, int lane) {
            const int r = lane & 31, piece = lane >> 5;
#pragma unroll
            for (int f = 0; f < FM; f++) {
                ah[f] = *(const f16x8*)(tp + tile_off(wm + 32 * f + r, piece));
                al[f] = *(const f16x8*)(tp + tile_off(wm + 32 * f + r, piece + 2));
            }
#pragma unroll
            for (int f = 0; f < FN; f++) {
                bh[f] = *(const f16x8*)(tq + tile_off(wn + 32 * f + r, piece));
                bl[f] = *(const f16x8*)(tq + tile_off(wn + 32 * f + r, piece + 2));
            }
        }
        // the small products first; blocks in turn, so that no MFMA waits for the one before
        __device__ inline void mul(f32x16 (&acc)[FM][FN]) const {
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[i], bh[j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bl[j], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < FM; i++)
#pragma unroll
                for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[i], bh[j], acc[i][j], 0, 0, 0);
        }
    };
};

// this wave's loads into LDS but the LATER last ones have landed and its reads of LDS have returned; and everybody else's
template <int LATER>
__device__ inline void step_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LATER) : "memory");
}

// a workgroup's tile: BM x BN outputs, WM x WN waves, STAGES buffers of GROUP steps each (a barrier every GROUP steps)
template <int BM_, int BN_, int WM_, int WN_, int STAGES_, int GROUP_>
struct TileShape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, WAVES = WM * WN, THREADS = 64 * WAVES, STAGES = STAGES_, GROUP = GROUP_;
    static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
    static constexpr bool PAIRS = FN % 2 == 0;   // lane c of blocks 2 j and 2 j + 1: columns 64 j + 2 c, 64 j + 2 c + 1
    static constexpr int STEP_BYTES = (BM + BN) * TILE_KB, STAGE_BYTES = GROUP * STEP_BYTES, LDS = STAGES * STAGE_BYTES;
    static_assert(LDS <= 160 * 1024 && STAGES >= 2, "the ring fits LDS");
};

// GROUP steps from `step` on into the buffer at `stage`
template <class S>
__device__ inline void stage_load(const TileSrc<false>& p, const TileSrc<S::PAIRS>& q, u32 step, u32 kend, u8* stage, int wave) {
#pragma unroll
    for (int g = 0; g < S::GROUP; g++) {
        tile_load<S::BM, S::WAVES, false>(p, step + g, kend, stage + g * S::STEP_BYTES, wave);
        tile_load<S::BN, S::WAVES, S::PAIRS>(q, step + g, kend, stage + g * S::STEP_BYTES + S::BM * TILE_KB, wave);
    }
}

// The order of a slice's instructions: its reads spread over its MFMAs from the first one on (left alone, the compiler moves the
// reads back to where the next slice uses them).
template <int READS, int MULS>
__device__ inline void spread_reads() {
#pragma unroll
    for (int i = 0; i < MULS; i++) {
        constexpr int PER = (READS + MULS - 1) / MULS;
        if (i * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
}

// The steps from `at` up to byte kend of the rows, kend a multiple of 16 (whole groups are read, with zeros behind kend).
// One barrier a group of steps: it says that the next group's tiles have landed and that everybody holds this group's last slice
// in registers.  That slice is multiplied behind it, while the next group's first slice is on its way from LDS and the group STAGES
// ahead (into the buffer that has just become free) on its way from memory.  Behind the last step the loads ask for nothing
// (zeros) and the slice read is nobody's: no branch in the loop, and the count of loads in flight stays what the barrier waits for.
template <class Kind, class S>
__device__ inline void tile_product(Kind, const TileSrc<false>& p, const TileSrc<S::PAIRS>& q, u32 at, u32 kend, u8* lds, int wave,
                                    int lane, typename Kind::acc_t (&acc)[S::FM][S::FN]) {
    const int wm = wave / S::WN * (S::FM * 32), wn = wave % S::WN * (S::FN * 32);
    constexpr int LOADS = S::GROUP * (S::BM + S::BN) / (16 * S::WAVES), KS = Kind::KS, Q = S::BM * TILE_KB, SL = S::GROUP * KS;
    static_assert((S::STAGES - 1) * LOADS < 64, "vmcnt counts to 63");
    typedef typename Kind::template Slice<S::FM, S::FN> Slice;
#pragma unroll
    for (int s = 0; s < S::STAGES; s++) stage_load<S>(p, q, at + s * S::GROUP, kend, lds + s * S::STAGE_BYTES, wave);
    step_barrier<(S::STAGES - 1) * LOADS>();
    Slice f0, f1;
    f0.read(lds, lds + Q, wm, wn, 0, lane);
    u8* cur = lds;
    auto group = [&](Slice& even, Slice& odd) {   // even: holds slice 0; odd is free
        u8* nxt = cur + S::STAGE_BYTES < lds + S::LDS ? cur + S::STAGE_BYTES : lds;
#pragma unroll
        for (int sl = 0; sl + 1 < SL; sl++) {
            u8* step = cur + (sl + 1) / KS * S::STEP_BYTES;
            (sl & 1 ? even : odd).read(step, step + Q, wm, wn, (sl + 1) % KS, lane);
            (sl & 1 ? odd : even).mul(acc);
            spread_reads<Kind::READS * (S::FM + S::FN), Kind::MULS * S::FM * S::FN>();
            __builtin_amdgcn_sched_barrier(0);
        }
        step_barrier<(S::STAGES - 2) * LOADS>();
        (SL & 1 ? odd : even).read(nxt, nxt + Q, wm, wn, 0, lane);
        stage_load<S>(p, q, at + S::STAGES * S::GROUP, kend, cur, wave);
        (SL & 1 ? even : odd).mul(acc);
        __builtin_amdgcn_sched_barrier(0);
        cur = nxt;
        at += S::GROUP;
    };
    const u32 end = (kend + TILE_KB - 1) / TILE_KB;
    if constexpr (SL % 2 == 0) {
        while (at < end) group(f0, f1);
    } else {
        while (at < end) {   // a group behind the last multiplies zeros (leaving in the middle would copy the accumulators)
            group(f0, f1);
            group(f1, f0);
        }
    }
    step_barrier<0>();   // nothing is on its way into LDS any more
}

// Which tile a workgroup computes.  Workgroups go to the 8 XCDs in turn and every XCD has its own L2: each XCD gets a
// contiguous run of tiles, and runs go through the tiles in bands of 8 tile rows, column by column, so that the tiles in
// flight on an XCD share few rows of P and Q.
__host__ __device__ inline u32 xcd_run(u32 block, u32 total) {
    const u32 per = total / 8, rest = total % 8, x = block & 7, i = block >> 3;
    return x * per + (x < rest ? x : rest) + i;   // XCD x has `per` tiles, one more if x < rest
}
__device__ inline void tile_place(u32 block, u32 tiles_m, u32 tiles_n, u32& tm, u32& tn) {
    const u32 t = xcd_run(block, tiles_m * tiles_n);
    const u32 band = t / (8 * tiles_n), first = band * 8, rows = tiles_m - first < 8 ? tiles_m - first : 8, in = t - band * 8 * tiles_n;
    tm = first + in % rows;
    tn = in / rows;
}

// The same for the tiles of a symmetric matrix that touch its lower triangle: rows of bm = `per` bn, row i has the first
// min(per (i + 1), cols) tiles.  Bands of 4 rows, column by column.
__host__ __device__ inline u32 symmetric_row(u32 i, u32 per, u32 cols) { return per * (i + 1) < cols ? per * (i + 1) : cols; }
__host__ __device__ inline u32 symmetric_total(u32 rows, u32 per, u32 cols) {
    return per * (rows - 1) * rows / 2 + symmetric_row(rows - 1, per, cols);
}
__host__ __device__ inline void symmetric_place(u32 block, u32 rows, u32 per, u32 cols, u32& tm, u32& tn) {
    u32 t = xcd_run(block, symmetric_total(rows, per, cols));
    for (u32 r0 = 0;; r0 += 4) {
        const u32 nr = rows - r0 < 4 ? rows - r0 : 4;
        u32 from = 0;   // columns before row r0 + k's own: rows r0 + k .. r0 + nr - 1 have them
        for (u32 k = 0; k < nr; k++) {
            const u32 to = symmetric_row(r0 + k, per, cols), n = (nr - k) * (to - from);
            if (t < n) {
                tm = r0 + k + t % (nr - k);
                tn = from + t / (nr - k);
                return;
            }
            t -= n;
            from = to;
        }
    }
}

}  // namespace az
