// az_ortho.hip -- orthogonalisation of matrices by Newton-Schulz products, and the weight update around it.
//
//   X = G / (||G||_F + eps);   `steps` times:  A = X X^T,  B = a I + b A + c A^2,  X <- B X      (s x l, s <= l: G or G^T)
//
// Products are fp32-accurate on the fp16 matrix pipe: every operand is kept as hi + lo, two fp16 halves of the value times a
// fixed power of two (X 2^14, A 2^12, B 2^11), and a product is hi hi + hi lo + lo hi with fp32 accumulation; the dropped
// lo lo is 2^-22 of a product.  Singular values stay below 2 (the host checks the coefficients), so |X| <= 2, |A| <= 4 and
// |B| <= 16 and no high half leaves fp16's range.  The fp32 pipe would be exact to 2^-24 and run at a sixteenth of the rate, 3
// products at a third; one fp16 product (2^-11) is not enough: the iteration multiplies the rounding of X's small singular
// directions by a^steps = 485.
//
// X is kept in both orientations, X [sp][lp] and T = X^T [lp][sp] (sp, lp: padded with zeros), because all three products
// then read both operands along their rows:  A = X X^T,  A^2 = A A^T,  T <- T B  (A and B are symmetric).
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#include "az_tile.hpp"

namespace az {

constexpr int OT = 64;             // padding of s and l
constexpr int MAX_JOBS = 16;       // matrices per set of launches (their table travels as a kernel argument)
constexpr int MAX_PARTS = 512;     // partial sums of a norm
constexpr i64 ORTHO_MAX_DIM = 32768;

struct Job {
    const void* g;   // gradient / input, [rows][cols]
    float* m;        // momentum or null
    void* w;         // weights (update) or output
    i32 rows, cols, s, l, sp, lp, n_part;
    float kappa;
    double* part;
    u8 *x, *t0, *t1, *a, *b, *c, *d;   // split operands in panels: 16 values of every row (16 hi, 16 lo: 64 bytes), then the next 16
    // short side <= 128 (see "Narrow matrices"): T in MFMA order in t, partial Gram matrices in gram
    float* gram;
    u8* image;
    i32 nb, groups, per_group;
};
struct Jobs {
    Job j[MAX_JOBS];
    i32 first[MAX_JOBS + 1];   // first block of every job in this launch
    i32 n;
};
struct Hyper {
    float mu, one_mu, decay, lr, a, b, c;
    double eps;
    int nesterov, update;   // update: the weight update; else out <- O(g)
};

__device__ inline int find_job(const Jobs& js, int block) {
    int j = 0;
    while (j + 1 < js.n && block >= js.first[j + 1]) j++;
    return j;
}
// what is orthogonalised, after k_ortho_norm has updated m: N values a thread, at `at` (where `in`; else zeros)
template <class T, int N>
__device__ inline void update_values(const Job& J, const Hyper& h, const i32 (&at)[N], const bool (&in)[N], float (&v)[N]) {
    T g[N];
    float m[N];
#pragma unroll
    for (int k = 0; k < N; k++) g[k] = ((const T*)J.g)[in[k] ? at[k] : 0];
    if (h.update)
#pragma unroll
        for (int k = 0; k < N; k++) m[k] = J.m[in[k] ? at[k] : 0];
    loads_first();
#pragma unroll
    for (int k = 0; k < N; k++) {
        v[k] = to_f32(g[k]);
        if (h.update) v[k] = h.nesterov ? h.mu * m[k] + h.one_mu * v[k] : m[k];
        if (!in[k]) v[k] = 0;
    }
}
// 2^14 / (norm + eps) as two factors to be multiplied one after the other.  The first is 1, or a power of two where the quotient
// could leave float32's normal range: of an infinite factor even the zeros would become NaN.  Below 2^-150, half of the smallest
// float32, the norm is 0 and so is every value; no factor needs to be larger for an eps that is.
__device__ inline void norm_factors(double sum, double eps, float& first, float& second) {
    double d = sqrt(sum) + eps;
    if (d < 0x1p-150) d = 0x1p-150;   // a NaN stays one
    first = d < 0x1p-100 ? 0x1p100f : d > 0x1p100 ? 0x1p-100f : 1.0f;
    second = (float)(16384.0 / (d * first));
}
__device__ inline i64 split_off(i64 row, i64 rows, i64 k) { return ((k >> 4) * rows + row) * TILE_KB + (k & 15) * 2; }

// eight values of a row from a multiple of eight on: their halves, 16 bytes each
__device__ inline void split_store8(u8* p, const float (&v)[8]) {
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        hi[e] = (f16)v[e];
        lo[e] = (f16)(v[e] - (float)hi[e]);
    }
    *(f16x8*)p = hi;
    *(f16x8*)(p + 32) = lo;
}
__device__ inline void split_load8(const u8* p, float (&v)[8]) {
    const f16x8 hi = *(const f16x8*)p, lo = *(const f16x8*)(p + 32);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (float)hi[e] + (float)lo[e];
}

// momentum (in place) and partial sums of squares of the update, in float64: the squares of float32 values can leave float32.
// 10.5 M values (g in bf16, momentum read and written: 105 MB): 20 us, 5.2 TB/s, a copy's rate.
template <class T>
__global__ __launch_bounds__(256) void k_ortho_norm(Jobs js, Hyper h) {
    __shared__ double red[4];
    const int ji = find_job(js, blockIdx.x);
    const Job J = js.j[ji];
    const int part = blockIdx.x - js.first[ji];
    const i64 n = (i64)J.rows * J.cols, per = (n + J.n_part - 1) / J.n_part, lo = part * per;
    const i64 hi = lo + per < n ? lo + per : n;
    double sum = 0;
    constexpr int U = 8;   // loads in flight
    for (i64 i0 = lo + threadIdx.x; i0 < hi; i0 += 256 * U) {
        float g[U], m[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const i64 i = i0 + 256 * k < hi ? i0 + 256 * k : hi - 1;
            g[k] = to_f32(((const T*)J.g)[i]);
            m[k] = h.update ? J.m[i] : 0.0f;
        }
        loads_first();
#pragma unroll
        for (int k = 0; k < U; k++) {
            const i64 i = i0 + 256 * k;
            if (i >= hi) break;
            float u = g[k];
            if (h.update) {
                const float n = h.mu * m[k] + h.one_mu * u;
                J.m[i] = n;
                u = h.nesterov ? h.mu * n + h.one_mu * u : n;
            }
            sum += (double)u * u;
        }
    }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) J.part[part] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X and T from the update, padding included: one 64 x 64 tile per workgroup.  10.5 M values (147 MB): 29 us, 5.0 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_ortho_init(Jobs js, Hyper h) {
    __shared__ float tile[OT][OT + 1];   // [short index][long index]
    __shared__ double red[4];
    const int ji = find_job(js, blockIdx.x), tid = threadIdx.x;
    const Job J = js.j[ji];
    const int nl = J.lp / OT, tl = blockIdx.x - js.first[ji], i0 = tl / nl * OT, j0 = tl % nl * OT;
    double sum = 0;
    for (int i = tid; i < J.n_part; i += 256) sum += J.part[i];
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    float f1, f2;
    norm_factors((red[0] + red[1]) + (red[2] + red[3]), h.eps, f1, f2);
    const bool flip = J.rows > J.cols;
    constexpr int U = 16;   // values a thread, all on their way at once
    float v[U];
    i32 at[U];   // rows * cols <= 2^30
    bool in[U];
#pragma unroll
    for (int k = 0; k < U; k++) {
        const int e = tid + 256 * k, slow = e / OT, fast = e % OT;   // fast runs along the matrix's rows in memory
        const int i = flip ? fast : slow, j = flip ? slow : fast;
        in[k] = i0 + i < J.s && j0 + j < J.l;
        at[k] = flip ? (j0 + j) * J.cols + i0 + i : (i0 + i) * J.cols + j0 + j;
    }
    update_values<T>(J, h, at, in, v);
#pragma unroll
    for (int k = 0; k < U; k++) {
        const int e = tid + 256 * k, slow = e / OT, fast = e % OT;
        tile[flip ? fast : slow][flip ? slow : fast] = v[k] * f1 * f2;
    }
    __syncthreads();
    for (int u = tid; u < OT * OT / 8; u += 256) {   // pairs of lanes: 16 values of a row, 64 bytes
        const int r = u / 2 % OT, c = (u % 2 + u / (2 * OT) * 2) * 8;
        float a[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            a[e] = tile[r][c + e];
            b[e] = tile[c + e][r];
        }
        split_store8(J.x + split_off(i0 + r, J.sp, j0 + c), a);
        split_store8(J.t0 + split_off(j0 + r, J.lp, i0 + c), b);
    }
}

enum { GRAM = 0, POLY = 1, SQUARE = 2, STEP = 3, LAST = 4 };
// GRAM: A = X X^T     POLY: B = a I + b A + c A A^T     SQUARE: a product of two of the s x s matrices     STEP: T <- T B (and X)
// LAST: the output, in its own orientation.
// The s x s matrices are polynomials of A: symmetric, and they commute.  Their launches compute the tiles that touch the lower
// triangle and store them twice.
//
// Several steps at once.  A step on X costs 2.4 s^2 l multiplications and 0.8 s^3 (a symmetric product takes 0.8 of a whole one's
// time).  Two or three can be made on the s x s side alone, A <- B A B and P <- B P, with X <- P X at their end: the default's five
// steps cost 3.6 s^2 l + 11.2 s^3 as 2 + 3 against 9 s^2 l + 4 s^3 one by one, less from l = 1.33 s on.  All five at once would
// not do: P's coefficients grow by (a^2)^k, and with them A's rounding (4.6e-5 where step by step has 1.3e-6).  2 + 3 keeps A's rounding
// from step to step too, where step by step makes A anew from X: that costs accuracy in float32, more or less by the matrix's singular
// values (relative error, 2 + 3 | step by step | plain float32: 1024 x 1024 5.2e-6 | 2.2e-6 | 1.0e-6, 300 x 300 5.2e-6 | 1.3e-6 | 1.1e-6,
// 512 x 2048 2.3e-6 | 2.2e-6 | 1.4e-6; six strong directions in noise, 512 x 4096 4.4e-6 | 2.0e-6 | 2.5e-6).  So results in float32 go step by
// step, whatever the sizes; a result in 16 bits is rounded by up to 4.9e-4 (fp16) or 3.9e-3 of itself, a hundred times that, and takes
// what is faster.

// what a launch multiplies: s x s matrices 0..3 (a, b, c, d), and the power of two from its sums to what it stores
struct Op {
    int p, q, out;
    float unit;
};
__device__ inline u8* square(const Job& J, int i) { return i == 0 ? J.a : i == 1 ? J.b : i == 2 ? J.c : J.d; }
__host__ __device__ constexpr bool symmetric(int mode) { return mode == GRAM || mode == POLY || mode == SQUARE; }

// rows and columns of a launch's result (padded)
__host__ __device__ inline void product_dims(int mode, const Job& J, int& rows, int& cols) {
    const bool flip = J.rows > J.cols;
    rows = symmetric(mode) ? J.sp : (mode == STEP || flip ? J.lp : J.sp);
    cols = mode == LAST && !flip ? J.lp : J.sp;
}
// the tile's result passes through LDS as float32, so that rows leave it 16 bytes a lane
template <class S>
struct Staged {
    static constexpr int PITCH = S::BN + 4;   // floats; rows stay 16-byte aligned and start 4 banks apart
    static constexpr int BYTES = S::BM * PITCH * 4;
    static constexpr int LDS = BYTES > S::LDS ? BYTES : S::LDS;
};

// 2048 x 2048: Gram 46 us (0.56 PFLOP/s of fp16 products, the lower triangle's counted), polynomial 48, step 57 (0.90), last 54; a
// library's fp16 product reaches 1.38 at 8192^3, this one 1.03 over whole calls at 4096 x 4096.  Neither pipe is full: of the Gram launch's
// cycles the matrix pipe works in 37 %, of a step's in 55 %, LDS in 20 %.  272 or 256 tiles on 256 CUs leave one wave a SIMD on most of them,
// which no other covers while it waits: 22 % of its cycles at loads and barriers (one a step), 32 % for the pipe it needs next.  272 symmetric
// tiles cost 12 us more than 240 (1920 x 1920: 36), but 64 x 64 tiles, longer and shorter rings and 8 waves each came out between 0 and
// 20 % slower over the whole call.  384 x 384 of two matrices: 7.6 us, latency.
template <int MODE, class S, class T>
__global__ __launch_bounds__(S::THREADS) void k_ortho_product(Jobs js, Hyper h, int cur, Op op) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    const int ji = find_job(js, blockIdx.x), tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job J = js.j[ji];
    const bool flip = J.rows > J.cols;
    constexpr bool SYM = symmetric(MODE);
    u8 *const t_cur = cur ? J.t1 : J.t0, *const t_next = cur ? J.t0 : J.t1;
    const u8 *P, *Q;
    int kp, rows, cols;
    product_dims(MODE, J, rows, cols);
    if (MODE == GRAM) { P = Q = J.x; kp = J.lp; }
    else if (MODE == POLY) { P = Q = J.a; kp = J.sp; }
    else if (MODE == SQUARE) { P = square(J, op.p); Q = square(J, op.q); kp = J.sp; }
    else if (MODE == STEP || flip) { P = t_cur; Q = square(J, op.q); kp = J.sp; }
    else { P = square(J, op.q); Q = t_cur; kp = J.sp; }
    u32 tm, tn;
    const int block = blockIdx.x - js.first[ji];
    if (SYM) symmetric_place(block, (rows + S::BM - 1) / S::BM, S::BM / S::BN, (cols + S::BN - 1) / S::BN, tm, tn);
    else tile_place(block, (rows + S::BM - 1) / S::BM, (cols + S::BN - 1) / S::BN, tm, tn);
    const int m0 = tm * S::BM, n0 = tn * S::BN;
    const int mrows = rows - m0 < S::BM ? rows - m0 : S::BM, ncols = cols - n0 < S::BN ? cols - n0 : S::BN;
    const TileSrc<false> p(P + m0 * TILE_KB, (u64)rows * TILE_KB, TILE_KB, mrows * TILE_KB, lane);
    const TileSrc<S::PAIRS> q(Q + n0 * TILE_KB, (u64)cols * TILE_KB, TILE_KB, ncols * TILE_KB, lane);
    f32x16 acc[S::FM][S::FN] = {};
    tile_product<KindSplit, S>(KindSplit(), p, q, 0, kp * 4, lds, wave, lane, acc);

    constexpr int W = S::PAIRS ? 2 : 1, PITCH = Staged<S>::PITCH;
    float* tile = (float*)lds;
#pragma unroll
    for (int i = 0; i < S::FM; i++)
#pragma unroll
        for (int j = 0; j < S::FN; j += W)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float* d = tile + (wave / S::WN * (S::FM * 32) + 32 * i + acc_row(r, lane)) * PITCH + wave % S::WN * (S::FN * 32) +
                           32 * j + W * (lane & 31);
                d[0] = acc[i][j][r] * op.unit;
                if (W == 2) d[1] = acc[i][j + W - 1][r] * op.unit;
            }
    __syncthreads();
    if (MODE != LAST) {   // mrows and ncols are multiples of 64 here
        u8* out = MODE == GRAM ? J.a : SYM ? square(J, op.out) : t_next;
        // 32 lanes store 16 values of 16 rows, 1 KB in a run: 16 lanes the first eight, 16 the others (16 rows read from LDS at
        // one column are on different banks)
#pragma unroll 2
        for (int u = tid; u < S::BM * S::BN / 8; u += S::THREADS) {
            const int at = u % (2 * S::BM), r = at / 32 * 16 + at % 16, c = u / (2 * S::BM) * 16 + at / 16 % 2 * 8, m = m0 + r, n = n0 + c;
            if (r >= mrows || c >= ncols || (SYM && n / OT > m / OT)) continue;
            float v[8];
            float* d = tile + r * PITCH + c;
            *(f32x4*)v = *(const f32x4*)d;
            *(f32x4*)(v + 4) = *(const f32x4*)(d + 4);
            if (MODE == POLY) {
                float A[8];
                split_load8(J.a + split_off(m, J.sp, n), A);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[e] = (h.c * v[e] + h.b * (A[e] * 0x1p-12f) + (m == n + e ? h.a : 0.0f)) * 0x1p11f;
                    d[e] = v[e];
                }
            }
            split_store8(out + split_off(m, rows, n), v);
        }
        // transposed: X for STEP, the mirrored blocks for A and B.  Of the 64 x 64 blocks those on the diagonal cover both sides
        // themselves (a mirrored value could differ from the computed one in its last bit, and both would be written); those above it
        // are the ones below, mirrored.  So it is with tiles of either size, and a matrix's bits do not depend on which its list takes.
        if (SYM && n0 + OT > m0 + S::BM - OT) return;
        if (MODE == POLY) __syncthreads();
        u8* outT = MODE == STEP ? J.x : out;
#pragma unroll 2
        for (int u = tid; u < S::BM * S::BN / 8; u += S::THREADS) {
            const int c = u / 2 % S::BN, r = (u % 2 + u / (2 * S::BN) * 2) * 8;
            if (r >= mrows || c >= ncols || (SYM && (n0 + c) / OT >= (m0 + r) / OT)) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = tile[(r + e) * PITCH + c];
            split_store8(outT + split_off(n0 + c, cols, m0 + r), v);
        }
    } else {
        // four neighbouring columns a thread; whole and aligned where the matrix's rows are
        struct __attribute__((aligned(4 * sizeof(T)))) Four { T v[4]; };
        const bool whole = J.cols % 4 == 0 && ((uintptr_t)J.w & (4 * sizeof(T) - 1)) == 0;
#pragma unroll 4
        for (int u = tid; u < S::BM * S::BN / 4; u += S::THREADS) {
            const int r = u / (S::BN / 4), c = u % (S::BN / 4) * 4;
            if (m0 + r >= J.rows || n0 + c >= J.cols) continue;
            const f32x4 o = *(const f32x4*)(tile + r * PITCH + c);
            T* w = (T*)J.w + (i64)(m0 + r) * J.cols + n0 + c;
            if (whole) {
                Four f;
                if (h.update) f = *(const Four*)w;
#pragma unroll
                for (int e = 0; e < 4; e++) f.v[e] = from_f32<T>(h.update ? to_f32(f.v[e]) * h.decay - o[e] * (h.lr * J.kappa) : o[e]);
                *(Four*)w = f;
            } else {
                for (int e = 0; e < 4 && n0 + c + e < J.cols; e++)
                    w[e] = from_f32<T>(h.update ? to_f32(w[e]) * h.decay - o[e] * (h.lr * J.kappa) : o[e]);
            }
        }
    }
}

using OTile128 = TileShape<128, 128, 2, 2, 4, 1>;
using OTile128s = TileShape<128, 64, 2, 2, 4, 1>;   // symmetric results
using OTile64 = TileShape<64, 64, 2, 2, 3, 4>;   // few tiles: what counts is the way from step to step, so few barriers

// ---------------------------------------------------------------------------------------------------- Narrow matrices
// Short side s <= 128: two launches a step.  B (s x s) fits LDS, and so does a panel of 128 values of the long index.  The first
// launch adds up the panels' parts of A = X X^T (in order, so the sum is the same every time); in the second every workgroup owns
// some panels and
//   1. takes A into LDS,
//   2. makes B = a I + b A + c A A^T for itself, and where the result has 16 bits the next step's as well, of B A B (two steps a launch),
//   3. multiplies its panels by it, keeping T for the next launch, and adds up their part of the next Gram matrix.
// What bounds it is latency: 5 steps of a 128 x 1152 matrix are 0.4 GFLOP, but 15 products one after the other; between launches,
// each product would start on cold operands.  Seven float32 matrices up to 128 x 1152 in one call: norm 6 us, init 12, sums 4.5 a
// launch, a step 15, the last 12: 105 us in all.  Two steps a launch take 24 us (2.5 for each of the four products more, which read 512 KB
// of LDS); 16-bit results are made so (us, two steps a launch | one: 128 x 1152 83 | 98, 128 x 32768 174 | 233, 4 x 100 x 5000 107 |
// 136, 16 x 64 x 64 54 | 74), float32 ones are not: the second step's A keeps the first one's rounding (relative error, two | one | plain
// float32: 32 x 32 1.5e-6 | 0.7e-6 | 0.8e-6, 128 x 128 1.4e-6 | 0.8e-6 | 1.3e-6, 128 x 1152 1.15e-6 | 1.14e-6 | 1.43e-6).  The wide matrices'
// launches instead of these: the seven 136 us, 128 x 128 76.
//
// T goes through memory in the order in which the MFMA of 3. takes it and the one before leaves it.  D = B T^T leaves lane
// (h = lane / 32, j = lane % 32) rows i = 8 (r / 4) + 4 h + r % 4 of column j: eight registers are eight values of k for lane (h, j) of the
// next product, if its k runs in the order that swaps bits 2 and 3 of i.  Columns of A and B in LDS are kept in that order.
constexpr int NARROW = 128, NPANEL = 128, NTHREADS = 1024, NWAVES = 16;
constexpr int NBUF = NARROW * 512;   // a row: 128 high halves, 128 low halves
constexpr int NSTEP_LDS = 2 * NBUF + 32 * 1024;
constexpr int MAX_GROUPS = 64;       // workgroups a matrix: so many parts of the Gram matrix are added up

__device__ inline int swap23(int i) { return (i & ~12) | ((i & 4) << 1) | ((i & 8) >> 1); }
// byte of value k of a row; pieces of 16 bytes are exchanged by row & 15, so that 16 rows read at one k use all banks
__device__ inline int nar_off(int row, int k, int low) {
    const int piece = low * 16 + (k >> 3);
    return row * 512 + ((piece ^ (row & 15)) << 4) + (k & 7) * 2;
}
__device__ inline f16x8 nar_frag(const u8* buf, int row, int step, int h, int low) {
    const int piece = low * 16 + 2 * step + h;
    return *(const f16x8*)(buf + row * 512 + ((piece ^ (row & 15)) << 4));
}
__device__ inline void nar_put(u8* buf, int row, int k, float v) {
    const f16 hi = (f16)v;
    *(f16*)(buf + nar_off(row, k, 0)) = hi;
    *(f16*)(buf + nar_off(row, k, 1)) = (f16)(v - (float)hi);
}
// block b of the lower triangle of 32 x 32 blocks
__device__ inline void lower_block(int b, int& bi, int& bj) {
    bi = b >= 6 ? 3 : b >= 3 ? 2 : b >= 1 ? 1 : 0;
    bj = b - bi * (bi + 1) / 2;
}
__device__ inline void mul3(f32x16& acc, f32x16& cross, f16x8 ah, f16x8 al, f16x8 bh, f16x8 bl) {
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, cross, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, acc, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, cross, 0, 0, 0);
}
// rows p.. of one buffer times rows q.. of another, over `steps` * 16 values
__device__ inline void nar_block(const u8* P, int p, const u8* Q, int q, int steps, int lane, f32x16& acc) {
    const int r = lane & 31, h = lane >> 5;
    f32x16 cross = {};
#pragma unroll 1
    for (int c = 0; c < steps; c++)
        mul3(acc, cross, nar_frag(P, p + r, c, h, 0), nar_frag(P, p + r, c, h, 1), nar_frag(Q, q + r, c, h, 0),
             nar_frag(Q, q + r, c, h, 1));
    acc += cross;
}
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
// rows m..m + 3 (a multiple of four on) of column n of a symmetric matrix, as row n, columns m..m + 3: they stay together there
__device__ inline void nar_put4(u8* buf, int m, int n, const float (&v)[4]) {
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        hi[e] = (f16)v[e];
        lo[e] = (f16)(v[e] - (float)hi[e]);
    }
    *(f16x4*)(buf + nar_off(n, swap23(m), 0)) = hi;
    *(f16x4*)(buf + nar_off(n, swap23(m), 1)) = lo;
}
__device__ inline void nar_get4(const u8* buf, int m, int n, float (&v)[4]) {
    const f16x4 hi = *(const f16x4*)(buf + nar_off(n, swap23(m), 0)), lo = *(const f16x4*)(buf + nar_off(n, swap23(m), 1));
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = (float)hi[e] + (float)lo[e];
}
__device__ inline int nar_blocks(const Job& J) { return J.nb * (J.nb + 1) / 2; }
// this wave's block of the panel's Gram matrix (10 at most); the panel is in buf as [short index][long index]
__device__ inline void nar_gram(const Job& J, const u8* buf, int wave, int lane, f32x16& acc) {
    if (wave >= nar_blocks(J)) return;
    int bi, bj;
    lower_block(wave, bi, bj);
    nar_block(buf, bi * 32, buf, bj * 32, NPANEL / 16, lane, acc);
}
__device__ inline void nar_gram_store(const Job& J, int group, int wave, int lane, const f32x16& acc) {
    if (wave >= nar_blocks(J)) return;
    float* d = J.gram + ((i64)(group * nar_blocks(J) + wave) * 64 + lane) * 16;
#pragma unroll
    for (int g = 0; g < 4; g++) *(f32x4*)(d + 4 * g) = f32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
}
// T of panel p, long-index block jb (32 values), k step c: 64 lanes x 16 bytes
__device__ inline u8* nar_t(u8* t, int p, int jb, int c, int low) { return t + ((((i64)p * 4 + jb) * 8 + c) * 2 + low) * 1024; }

template <class T>
__global__ __launch_bounds__(NTHREADS) void k_narrow_init(Jobs js, Hyper h) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    __shared__ double red[NWAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job J = js.j[blockIdx.y];
    const int group = blockIdx.x;
    if (group >= J.groups) return;
    const int panels = (J.l + NPANEL - 1) / NPANEL, height = J.nb * 32;
    const bool flip = J.rows > J.cols;
    double sum = 0;
    for (int i = tid; i < J.n_part; i += NTHREADS) sum += J.part[i];
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int i = 0; i < NWAVES; i++) sum += red[i];
    float f1, f2;
    norm_factors(sum, h.eps, f1, f2);
    f32x16 acc = {};
    for (int p = group * J.per_group; p < panels && p < (group + 1) * J.per_group; p++) {
        const int j0 = p * NPANEL;
        // consecutive threads along the matrix's rows in memory; 8 values a thread on their way at once
        constexpr int U = 8;
        static_assert(NARROW * NPANEL % (NTHREADS * U) == 0, "whole rounds");
#pragma unroll 1
        for (int e0 = tid; e0 < NARROW * NPANEL; e0 += NTHREADS * U) {
            float v[U];
            i32 at[U];   // rows * cols <= 2^30
            bool in[U];
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int e = e0 + NTHREADS * k, i = flip ? e % NARROW : e / NPANEL, j = flip ? e / NARROW : e % NPANEL;
                in[k] = i < J.s && j0 + j < J.l;
                at[k] = flip ? (j0 + j) * J.cols + i : i * J.cols + j0 + j;
            }
            update_values<T>(J, h, at, in, v);
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int e = e0 + NTHREADS * k, i = flip ? e % NARROW : e / NPANEL, j = flip ? e / NARROW : e % NPANEL;
                if (i < height) nar_put(lds, i, j, v[k] * f1 * f2);
            }
        }
        __syncthreads();
        const int jb = wave & 3, hh = lane >> 5, j = jb * 32 + (lane & 31);
        for (int c = (wave >> 2) * 2; c < (wave >> 2) * 2 + 2 && c < 2 * J.nb; c++)
            for (int low = 0; low < 2; low++) {
                f16x8 f;
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = *(const f16*)(lds + nar_off(16 * c + swap23(8 * hh + e), j, low));
                *(f16x8*)(nar_t(J.t0, p, jb, c, low) + lane * 16) = f;
            }
        nar_gram(J, lds, wave, lane, acc);
        __syncthreads();
    }
    nar_gram_store(J, group, wave, lane, acc);
}

// A = sum of the groups' parts (in order), as the image that k_narrow_step takes into LDS: a block a workgroup.  A launch of its
// own: every workgroup of k_narrow_step adding up 40 KB from each of 9 others took 11 of its 24 us.
__global__ __launch_bounds__(256) void k_narrow_sum(Jobs js) {
    const Job J = js.j[blockIdx.y];
    const int blocks = nar_blocks(J), b = blockIdx.x, lane = threadIdx.x & 63, g4 = threadIdx.x >> 6;
    if (b >= blocks) return;
    const float* d = J.gram + ((i64)b * 64 + lane) * 16 + 4 * g4;
    constexpr int AHEAD = 16;
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll 1
    for (int g0 = 0; g0 < J.groups; g0 += AHEAD) {
        f32x4 y[AHEAD];
#pragma unroll
        for (int g = 0; g < AHEAD; g++) y[g] = *(const f32x4*)(d + (i64)(g0 + g < J.groups ? g0 + g : 0) * blocks * 1024);
        loads_first();
#pragma unroll
        for (int g = 0; g < AHEAD; g++)
            if (g0 + g < J.groups) sum += y[g];
    }
    int bi, bj;
    lower_block(b, bi, bj);
    const int m = bi * 32 + acc_row(4 * g4, lane), n = bj * 32 + (lane & 31);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = sum[e] * 0x1p-16f;
    nar_put4(J.image, m, n, v);
    if (bi != bj)
#pragma unroll
        for (int e = 0; e < 4; e++) nar_put(J.image, m + e, swap23(n), v[e]);
}

// TWO: two steps.  The powers of two from the sums to P, and from P X to X (to the output in the last launch)
struct Narrow {
    float p_unit, x_unit;
};
// 128 registers a wave (16 of them share a CU) are not enough: the compiler keeps 28 to 48 bytes a lane in scratch, by the form.
template <class T, bool LASTSTEP, bool TWO>
__global__ __launch_bounds__(NTHREADS) void k_narrow_step(Jobs js, Hyper h, int cur, Narrow pass) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    u8 *const bufA = lds, *const bufB = lds + NBUF;   // A, then the new panel; B
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Job J = js.j[blockIdx.y];   // no search: what a launch waits for first is its arguments, one line after the other
    if ((int)blockIdx.x >= J.groups) return;
    u8 *const t_cur = cur ? J.t1 : J.t0, *const t_next = cur ? J.t0 : J.t1;
    const int group = blockIdx.x, panels = (J.l + NPANEL - 1) / NPANEL, steps = 2 * J.nb;
    const int first = group * J.per_group, end = first + J.per_group < panels ? first + J.per_group : panels;
    const bool flip = J.rows > J.cols;
    const int jb = wave & 3, ib = wave >> 2;   // this wave: 32 of the panel's long index, a block of the short one
    // 1. A
    {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(J.image, 0, J.nb * 32 * 512, 0x00020000);
#pragma unroll
        for (int i = 0; i < NBUF / 1024 / NWAVES; i++) {   // rows behind nb blocks: zeros
            const int at = (i * NWAVES + wave) * 1024;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(bufA + at), 16, lane * 16, at, 0, 0);
        }
    }
    // T of a panel: k steps 0..3 in registers, 4..7 through LDS (64 registers more than a wave has)
    u8* const bufT = lds + 2 * NBUF;
    f16x8 t[4][2];
    auto fetch = [&](int p) {
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int low = 0; low < 2; low++) t[c][low] = *(const f16x8*)(nar_t(t_cur, p, jb, c < steps ? c : 0, low) + lane * 16);
    };
    auto fetch_high = [&](int p) {   // waves of one jb: a k step each
        if (4 + ib >= steps) return;
        const u8* src = nar_t(t_cur, p, jb, 4 + ib, 0);
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<u8*>(src), 0, 2048, 0x00020000);
#pragma unroll
        for (int low = 0; low < 2; low++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(bufT + ((jb * 4 + ib) * 2 + low) * 1024), 16, lane * 16, low * 1024, 0, 0);
    };
    fetch_high(first);
    if (!TWO) fetch(first);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    // 2. B, every block of it
    if (wave < J.nb * J.nb) {
        const int bi = wave / J.nb, bj = wave - bi * J.nb, n = bj * 32 + (lane & 31);
        f32x16 acc = {};
        nar_block(bufA, bi * 32, bufA, bj * 32, steps, lane, acc);
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int m = bi * 32 + acc_row(4 * g, lane);
            float v[4];
            nar_get4(bufA, m, n, v);
#pragma unroll
            for (int e = 0; e < 4; e++)
                v[e] = (h.c * (acc[4 * g + e] * 0x1p-24f) + h.b * (v[e] * 0x1p-12f) + (m + e == n ? h.a : 0.0f)) * 0x1p11f;
            nar_put4(bufB, m, n, v);
        }
    }
    __syncthreads();
    if constexpr (TWO) {   // P = B2 B instead of B, with B2 = f(B A B)
        const bool on = wave < J.nb * J.nb;
        const int bi = wave / J.nb * 32, bj = (wave - wave / J.nb * J.nb) * 32, n = bj + (lane & 31);
        // a product of two of these symmetric, commuting matrices, into a buffer that it reads itself
        auto times = [&](const u8* P, const u8* Q, u8* out, float unit, bool poly) {
            f32x16 acc = {};
            if (on) {
                nar_block(P, bi, Q, bj, steps, lane, acc);
                acc *= unit;
                if (poly)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const int m = bi + acc_row(4 * g, lane);
                        float v[4];
                        nar_get4(P, m, n, v);
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            acc[4 * g + e] = (h.c * acc[4 * g + e] + h.b * (v[e] * 0x1p-12f) + (m + e == n ? h.a : 0.0f)) * 0x1p11f;
                    }
            }
            __syncthreads();
            if (on)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const float v[4] = {acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
                    nar_put4(out, bi + acc_row(4 * g, lane), n, v);
                }
            __syncthreads();
        };
        times(bufA, bufB, bufA, 0x1p-11f, false);
        times(bufA, bufB, bufA, 0x1p-11f, false);
        times(bufA, bufA, bufA, 0x1p-24f, true);
        fetch(first);   // not earlier: its 32 registers would spill more
        times(bufA, bufB, bufB, pass.p_unit, false);
    }
    // 3. the panels
    f32x16 gram = {};
    for (int p = first; p < end; p++) {
        if (ib < J.nb) {
            const int i0 = ib * 32, hh = lane >> 5;
            f32x16 acc = {}, cross = {};
            const bool across = LASTSTEP && flip;   // the output's rows are the long index: lanes along the short one
#pragma unroll
            for (int c = 0; c < 8; c++) {
                if (c >= steps) continue;
                const f16x8 bh = nar_frag(bufB, i0 + (lane & 31), c, hh, 0), bl = nar_frag(bufB, i0 + (lane & 31), c, hh, 1);
                f16x8 th, tl;
                if (c < 4) {
                    th = t[c & 3][0];
                    tl = t[c & 3][1];
                } else {
                    th = *(const f16x8*)(bufT + ((jb * 4 + c - 4) * 2) * 1024 + lane * 16);
                    tl = *(const f16x8*)(bufT + ((jb * 4 + c - 4) * 2 + 1) * 1024 + lane * 16);
                }
                if (across) mul3(acc, cross, th, tl, bh, bl);
                else mul3(acc, cross, bh, bl, th, tl);
                if (c & 1) __builtin_amdgcn_sched_barrier(0);   // 128 registers a wave: not all of B's reads at once
            }
            acc += cross;
            if (!LASTSTEP) {
                acc *= pass.x_unit;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    f16x8 hi, lo;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float v = acc[8 * half + e];
                        hi[e] = (f16)v;
                        lo[e] = (f16)(v - (float)hi[e]);
                        const int i = i0 + acc_row(8 * half + e, lane), j = jb * 32 + (lane & 31);
                        *(f16*)(bufA + nar_off(i, j, 0)) = hi[e];
                        *(f16*)(bufA + nar_off(i, j, 1)) = lo[e];
                    }
                    const int c = 2 * ib + half;
                    *(f16x8*)(nar_t(t_next, p, jb, c, 0) + lane * 16) = hi;
                    *(f16x8*)(nar_t(t_next, p, jb, c, 1) + lane * 16) = lo;
                }
            } else {
                const int col = (across ? i0 : p * NPANEL + jb * 32) + (lane & 31), row0 = across ? p * NPANEL + jb * 32 : i0;
                float old[16];
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int row = row0 + acc_row(r, lane);
                    const bool in = row < J.rows && col < J.cols;
                    old[r] = to_f32(((const T*)J.w)[in && h.update ? (i64)row * J.cols + col : 0]);
                }
                loads_first();
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int row = row0 + acc_row(r, lane);
                    if (row >= J.rows || col >= J.cols) continue;
                    float o = acc[r] * pass.x_unit;
                    if (h.update) o = old[r] * h.decay - o * (h.lr * J.kappa);
                    ((T*)J.w)[(i64)row * J.cols + col] = from_f32<T>(o);
                }
            }
        }
        if (LASTSTEP && p + 1 == end) break;
        __syncthreads();   // bufT has been read; bufA holds the new panel
        if (p + 1 < end) {
            fetch_high(p + 1);
            fetch(p + 1);
        }
        if (!LASTSTEP) nar_gram(J, bufA, wave, lane, gram);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    if (!LASTSTEP) nar_gram_store(J, group, wave, lane, gram);
}

// ---------------------------------------------------------------------------------------------------- host side
static i64 pad(i64 n) { return (n + OT - 1) / OT * OT; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static bool dims_ok(i64 rows, i64 cols) { return rows >= 1 && cols >= 1 && rows <= ORTHO_MAX_DIM && cols <= ORTHO_MAX_DIM; }

// lays a job's workspace out from `p` on (null: only counts) and returns its bytes
static size_t plan(Job& J, i64 rows, i64 cols, char* p) {
    J.rows = (i32)rows;
    J.cols = (i32)cols;
    J.s = (i32)(rows < cols ? rows : cols);
    J.l = (i32)(rows < cols ? cols : rows);
    J.sp = (i32)pad(J.s);
    J.lp = (i32)pad(J.l);
    const i64 parts = (rows * cols + 4095) / 4096;
    J.n_part = (i32)(parts < MAX_PARTS ? parts : MAX_PARTS);
    J.kappa = (float)sqrt(rows > cols ? (double)rows / (double)cols : 1.0);
    size_t off = 0;
    auto take = [&](size_t n) {
        char* r = p ? p + off : nullptr;
        off += up256(n);
        return (u8*)r;
    };
    J.part = (double*)take(J.n_part * sizeof(double));
    J.nb = (J.s + 31) / 32;
    if (J.s <= NARROW) {
        const int panels = (J.l + NPANEL - 1) / NPANEL;
        J.per_group = (panels + MAX_GROUPS - 1) / MAX_GROUPS;
        J.groups = (panels + J.per_group - 1) / J.per_group;
        J.t0 = take((size_t)panels * NPANEL * NARROW * 4);
        J.t1 = take((size_t)panels * NPANEL * NARROW * 4);
        J.gram = (float*)take((size_t)J.groups * (J.nb * (J.nb + 1) / 2) * 4096);
        J.image = take(NBUF);
        J.x = J.a = J.b = J.c = J.d = nullptr;
        return off;
    }
    J.gram = nullptr;
    J.image = nullptr;
    J.groups = J.per_group = 0;
    J.x = take((size_t)J.sp * J.lp * 4);
    J.t0 = take((size_t)J.sp * J.lp * 4);
    J.t1 = take((size_t)J.sp * J.lp * 4);
    J.a = take((size_t)J.sp * J.sp * 4);
    J.b = take((size_t)J.sp * J.sp * 4);
    J.c = take((size_t)J.sp * J.sp * 4);
    J.d = take((size_t)J.sp * J.sp * 4);
    return off;
}

// Which coefficients keep the halves in range: follows the largest singular value through the steps on a grid.  (The limits below
// leave a factor of two to where a high half would overflow: room for what lies between the grid's points.)
static bool coeffs_ok(int steps, const double* k) {
    if (!k || !isfinite(k[0]) || !isfinite(k[1]) || !isfinite(k[2])) return false;
    double top = 1.0;
    for (int it = 0; it < steps; it++) {
        double next = 0;
        for (int i = 0; i <= 256; i++) {
            const double x = top * i / 256, x2 = x * x, poly = k[0] + k[1] * x2 + k[2] * x2 * x2;
            if (fabs(poly) > 15.9 || fabs(poly - k[0]) > 15.9) return false;
            next = fmax(next, fabs(poly * x));
        }
        top = next * 1.01;
        if (top > 1.99) return false;
    }
    return true;
}

static double step_poly(const Hyper& h, double x2) { return h.a + h.b * x2 + h.c * x2 * x2; }
// the largest singular value after a step, from the largest before it
static double top_after(const Hyper& h, double top) {
    double next = 0;
    for (int i = 0; i <= 256; i++) next = fmax(next, fabs(step_poly(h, top * i / 256 * (top * i / 256)) * top * i / 256));
    return next * 1.01;
}

// how much a step A <- B A B can enlarge an error of A: the largest slope of y p(y)^2 (a^2 = 12 for the default coefficients)
static double steepest(const Hyper& h, int steps) {
    double top = 1.0, most = 0;
    for (int it = 0; it < steps; it++, top = top_after(h, top))
        for (int i = 0; i <= 256; i++) {
            const double y = top * top * i / 256, p = step_poly(h, y);
            most = fmax(most, fabs(p * p + 2 * y * p * (h.b + 2 * h.c * y)));
        }
    return most;
}

// the power of two that keeps the product of `n` steps' B, from step `first` on, inside fp16's range
static int product_exponent(const Hyper& h, int first, int n) {
    double top = 1.0, most = 1.0;
    for (int it = 0; it < first; it++) top = top_after(h, top);
    for (int i = 0; i <= 256; i++) {
        double x = top * i / 256, product = 1.0;
        for (int k = 0; k < n; k++) {
            const double p = step_poly(h, x * x);
            product *= p;
            x *= p;
            most = fmax(most, fabs(product));
        }
    }
    int e = 11;
    while (ldexp(most, e) > 32000.0) e--;   // a factor of two for what lies between the grid's points
    return e;
}

template <class F>
static void each_first(Jobs& js, F blocks) {
    js.first[0] = 0;
    for (int i = 0; i < js.n; i++) js.first[i + 1] = js.first[i] + (i32)blocks(js.j[i]);
}

template <int MODE, class S>
static int product_blocks(Jobs& js) {   // fills js.first
    each_first(js, [](const Job& J) {
        int rows, cols;
        product_dims(MODE, J, rows, cols);
        if (symmetric(MODE))
            return (i64)symmetric_total((rows + S::BM - 1) / S::BM, S::BM / S::BN, (cols + S::BN - 1) / S::BN);
        return (i64)((rows + S::BM - 1) / S::BM) * ((cols + S::BN - 1) / S::BN);
    });
    return js.first[js.n];
}
template <int MODE, class T>
static void product(Jobs& js, const Hyper& h, int cur, const Op& op, hipStream_t st) {
    // The larger tile reads half as much per product; it needs enough tiles to fill the chip (us, from 80 tiles on | from 160 on:
    // 1500 x 1500, 144 and 156 tiles, 392 | 512; 800 x 2000, 112 tiles, 248 | 241).
    constexpr int ENOUGH = 120;
    if constexpr (symmetric(MODE)) {
        const int n = product_blocks<MODE, OTile128s>(js);
        if (n >= ENOUGH) {
            k_ortho_product<MODE, OTile128s, T><<<dim3((u32)n), dim3(OTile128s::THREADS), Staged<OTile128s>::LDS, st>>>(js, h, cur, op);
            return;
        }
    } else {
        const int n = product_blocks<MODE, OTile128>(js);
        if (n >= ENOUGH) {
            k_ortho_product<MODE, OTile128, T><<<dim3((u32)n), dim3(OTile128::THREADS), Staged<OTile128>::LDS, st>>>(js, h, cur, op);
            return;
        }
    }
    const int n = product_blocks<MODE, OTile64>(js);
    k_ortho_product<MODE, OTile64, T><<<dim3((u32)n), dim3(OTile64::THREADS), Staged<OTile64>::LDS, st>>>(js, h, cur, op);
}

static int run_narrow(Jobs& js, const Hyper& h, int steps, int dtype, hipStream_t st) {
    each_first(js, [](const Job& J) { return J.n_part; });
    AZ_DISPATCH_DTYPE(dtype, k_ortho_norm<T><<<dim3(js.first[js.n]), dim3(256), 0, st>>>(js, h));
    int most = 0;
    for (int i = 0; i < js.n; i++) most = js.j[i].groups > most ? js.j[i].groups : most;
    const dim3 grid(most, js.n), block(NTHREADS);
    AZ_DISPATCH_DTYPE(dtype, k_narrow_init<T><<<grid, block, NBUF, st>>>(js, h));
    const dim3 grid_sum(10, js.n);   // blocks of a 128 x 128 matrix's lower triangle
    const bool pairs = dtype != AZ_F32 && steepest(h, steps) <= 16.0;   // (see above)
    int cur = 0;
    for (int done = 0; done < steps; cur ^= 1) {
        const bool two = pairs && done + 2 <= steps;
        const int e = two ? product_exponent(h, done, 2) : 11;
        done += two ? 2 : 1;
        const bool last = done == steps;
        const Narrow pass = {ldexpf(1.0f, e - 22), ldexpf(1.0f, last ? -14 - e : -e)};
        k_narrow_sum<<<grid_sum, dim3(256), 0, st>>>(js);
        if (last && two) {
            if (dtype == AZ_F16) k_narrow_step<f16, true, true><<<grid, block, NSTEP_LDS, st>>>(js, h, cur, pass);
            else k_narrow_step<bf16, true, true><<<grid, block, NSTEP_LDS, st>>>(js, h, cur, pass);
        } else if (last) {
            AZ_DISPATCH_DTYPE(dtype, k_narrow_step<T, true, false><<<grid, block, NSTEP_LDS, st>>>(js, h, cur, pass));
        } else if (two) {
            k_narrow_step<float, false, true><<<grid, block, NSTEP_LDS, st>>>(js, h, cur, pass);
        } else {
            k_narrow_step<float, false, false><<<grid, block, NSTEP_LDS, st>>>(js, h, cur, pass);
        }
    }
    return launch_status("az_orthogonalize");
}

static int run_jobs(Jobs& all, const Hyper& h, int steps, int dtype, hipStream_t st) {
    Jobs js;
    js.n = 0;
    for (int i = 0; i < all.n; i++)
        if (all.j[i].s <= NARROW) js.j[js.n++] = all.j[i];
    if (js.n) {
        const int rc = run_narrow(js, h, steps, dtype, st);
        if (rc != AZ_OK || js.n == all.n) return rc;
    }
    js.n = 0;
    for (int i = 0; i < all.n; i++)
        if (all.j[i].s > NARROW) js.j[js.n++] = all.j[i];
    each_first(js, [](const Job& J) { return J.n_part; });
    AZ_DISPATCH_DTYPE(dtype, k_ortho_norm<T><<<dim3(js.first[js.n]), dim3(256), 0, st>>>(js, h));
    each_first(js, [](const Job& J) { return (i64)(J.sp / OT) * (J.lp / OT); });
    AZ_DISPATCH_DTYPE(dtype, k_ortho_init<T><<<dim3(js.first[js.n]), dim3(256), 0, st>>>(js, h));
    // Steps on the s x s side where the result has 16 bits (see above) and that should take less time for the list as a whole: launches
    // are shared, and a second set of them for some of its matrices would cost more than it saves (1024 x 4096, 4096 x 1024 and two of
    // 1024 x 1024, bf16: together 703 us, the squares step by step in launches of their own 833, all step by step 843).
    // A launch costs 5 us and its work at 0.9 PFLOP/s, or 0.1 us for every 16 values of the sums of its longest tile (both as measured, a
    // symmetric product as 0.8 of a whole one).  2 + 3 | one by one, us: 2 x 333 x 1027 155 | 151, 2 x 400 x 800 158 | 147, 1024 x 1536
    // 251 | 247, 1024 x 2048 265 | 275, 300 x 2000 153 | 170, 512 x 4096 213 | 274, 1024 x 4096 323 | 394
    int len[16], n = 0, left = steps, squares = 0;
    while (left > 0) {
        len[n] = n == 0 ? (left < 2 ? left : 2) : (left < 3 ? left : 3);
        squares += len[n] == 1 ? 0 : len[n] == 2 ? 3 : 6;
        left -= len[n++];
    }
    double s2l = 0, s3 = 0, longest_l = 0, longest_s = 0;
    for (int i = 0; i < js.n; i++) {
        const double s = js.j[i].sp, l = js.j[i].lp;
        s2l += s * s * l;
        s3 += s * s * s;
        longest_l = fmax(longest_l, l);
        longest_s = fmax(longest_s, s);
    }
    auto launch = [](double products, double k) { return 5.0 + fmax(6 * products / 0.9e9, 0.1 * k / 16); };
    const double on_x = launch(0.8 * s2l, longest_l) + launch(s2l, longest_s), on_a = launch(0.8 * s3, longest_s);
    if (dtype == AZ_F32 || n * on_x + (steps + squares) * on_a > steps * (on_x + on_a) || steepest(h, steps) > 16.0)
        for (n = 0; n < steps; n++) len[n] = 1;
    const Op gram = {0, 0, 0, 0x1p-16f};                                  // 2^14 2^14 -> 2^12
    auto poly = [](int out) { return Op{0, 0, out, 0x1p-24f}; };           // 2^12 2^12 -> 1, then 2^11
    auto to_a = [](int p, int q, int out) { return Op{p, q, out, 0x1p-11f}; };   // 2^11 2^12 -> 2^12
    int cur = 0, done = 0;
    for (int k = 0; k < n; k++) {
        product<GRAM, float>(js, h, cur, gram, st);
        product<POLY, float>(js, h, cur, poly(1), st);
        int by = 1, e = 11;   // X is multiplied by matrix `by`, kept times 2^e
        if (len[k] > 1) {
            e = product_exponent(h, done, len[k]);
            product<SQUARE, float>(js, h, cur, to_a(1, 0, 2), st);          // c = B A
            product<SQUARE, float>(js, h, cur, to_a(2, 1, 0), st);          // a = B A B: the next step's A
            product<POLY, float>(js, h, cur, poly(3), st);                  // d: the next step's B
            product<SQUARE, float>(js, h, cur, Op{3, 1, 2, ldexpf(1.0f, e - 22)}, st);   // c = P of two steps
            by = 2;
        }
        if (len[k] > 2) {
            product<SQUARE, float>(js, h, cur, to_a(3, 0, 1), st);
            product<SQUARE, float>(js, h, cur, to_a(1, 3, 0), st);
            product<POLY, float>(js, h, cur, poly(3), st);
            product<SQUARE, float>(js, h, cur, Op{3, 2, 1, 0x1p-11f}, st);  // b = P of three: 2^11 2^e -> 2^e
            by = 1;
        }
        if (k + 1 < n) {
            product<STEP, float>(js, h, cur, Op{0, by, 0, ldexpf(1.0f, -e)}, st);
        } else {
            AZ_DISPATCH_DTYPE(dtype, product<LAST, T>(js, h, cur, Op{0, by, 0, ldexpf(1.0f, -14 - e)}, st));
        }
        cur ^= 1;
        done += len[k];
    }
    return launch_status("az_orthogonalize");
}

}  // namespace az

using namespace az;

extern "C" {

size_t az_orthogonalize_ws(int64_t batch, int64_t rows, int64_t cols) {
    if (batch < 1 || !dims_ok(rows, cols)) return 0;
    Job J;
    return plan(J, rows, cols, nullptr) * (size_t)(batch < MAX_JOBS ? batch : MAX_JOBS);
}

static int ortho_check(int dtype, int steps, const double* coeffs, double eps) {
    if (!dtype_ok(dtype)) return refuse("az_orthogonalize: unknown dtype");
    if (steps < 1 || steps > 16) return refuse("az_orthogonalize: steps is 1..16");
    if (!(eps > 0) || !isfinite(eps)) return refuse("az_orthogonalize: eps must be positive and finite");
    if (!coeffs_ok(steps, coeffs)) return refuse("az_orthogonalize: these coefficients leave the range of the products");
    return AZ_OK;
}
static int ws_check(const void* ws, size_t ws_bytes, size_t need) {
    if (ws_bytes < need || (need && (!ws || ((uintptr_t)ws & 255))))
        return refuse("az_orthogonalize: workspace too small or not aligned to 256 bytes");
    return AZ_OK;
}

int az_orthogonalize_dev(int device, int dtype, int64_t batch, int64_t rows, int64_t cols, const void* g_dev, void* out_dev,
                         int steps, const double* coeffs, double eps, void* ws_dev, size_t ws_bytes, void* stream) {
    if (batch < 0 || batch > (i64)1 << 31 || !dims_ok(rows, cols))
        return refuse("az_orthogonalize: bad shape (rows and cols are 1..32768)");
    int rc = ortho_check(dtype, steps, coeffs, eps);
    if (rc == AZ_OK) rc = ws_check(ws_dev, ws_bytes, az_orthogonalize_ws(batch, rows, cols));
    if (rc != AZ_OK) return rc;
    if (batch > 0 && (!g_dev || !out_dev)) return refuse("az_orthogonalize: null pointer");
    const size_t all = (size_t)batch * rows * cols * dtype_size(dtype);
    if (g_dev != out_dev && overlap(g_dev, all, out_dev, all)) return refuse("az_orthogonalize: out overlaps g without being it");
    DeviceScope dev(device);
    if (dev.rc != AZ_OK || batch == 0) return dev.rc;
    Hyper h = {};
    h.a = (float)coeffs[0];
    h.b = (float)coeffs[1];
    h.c = (float)coeffs[2];
    h.eps = eps;
    const size_t bytes = (size_t)rows * cols * dtype_size(dtype);
    for (int64_t lo = 0; lo < batch; lo += MAX_JOBS) {
        Jobs js;
        js.n = (i32)(batch - lo < MAX_JOBS ? batch - lo : MAX_JOBS);
        size_t off = 0;
        for (int i = 0; i < js.n; i++) {
            Job& J = js.j[i];
            off += plan(J, rows, cols, (char*)ws_dev + off);
            J.g = (const char*)g_dev + (lo + i) * bytes;
            J.w = (char*)out_dev + (lo + i) * bytes;
            J.m = nullptr;
        }
        rc = run_jobs(js, h, steps, dtype, (hipStream_t)stream);
        if (rc != AZ_OK) return rc;
    }
    return AZ_OK;
}

// what is written (w, m) overlaps nothing else: all of them in the order of their addresses, each held against the farthest end so far
static bool items_apart(const az_muon_item* items, i64 n, size_t es) {
    struct Range { uintptr_t from, to; bool written; };
    std::vector<Range> all;
    all.reserve((size_t)n * 3);
    for (i64 i = 0; i < n; i++) {
        const size_t count = (size_t)items[i].rows * items[i].cols;
        const uintptr_t w = (uintptr_t)items[i].w_dev, g = (uintptr_t)items[i].g_dev, m = (uintptr_t)items[i].m_dev;
        all.push_back({w, w + count * es, true});
        all.push_back({g, g + count * es, false});
        all.push_back({m, m + count * 4, true});
    }
    std::sort(all.begin(), all.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t end = 0, written = 0;   // of all, of those written
    for (const Range& r : all) {
        if (r.from < (r.written ? end : written)) return false;
        end = r.to > end ? r.to : end;
        if (r.written && r.to > written) written = r.to;
    }
    return true;
}

size_t az_muon_step_ws(const az_muon_item* items, int64_t n) {
    size_t most = 0;
    if (!items) return 0;
    for (int64_t lo = 0; lo < n; lo += MAX_JOBS) {
        size_t sum = 0;
        for (int64_t i = lo; i < n && i < lo + MAX_JOBS; i++) {
            Job J;
            if (!dims_ok(items[i].rows, items[i].cols)) return 0;
            sum += plan(J, items[i].rows, items[i].cols, nullptr);
        }
        most = sum > most ? sum : most;
    }
    return most;
}

int az_muon_step_check(int dtype, const az_muon_item* items, int64_t n, double lr, double momentum, double weight_decay, int steps,
                       const double* coeffs, double eps) {
    if (n < 0 || n > 65536 || (n > 0 && !items)) return refuse("az_muon_step: bad item list");
    if (!dtype_ok(dtype)) return refuse("az_muon_step: unknown dtype");
    for (int64_t i = 0; i < n; i++) {
        if (!dims_ok(items[i].rows, items[i].cols)) return refuse("az_muon_step: bad shape (rows and cols are 1..32768)");
        if (!items[i].w_dev || !items[i].g_dev || !items[i].m_dev) return refuse("az_muon_step: null pointer");
    }
    bool apart = false;
    try {
        apart = items_apart(items, n, dtype_size(dtype));
    } catch (const std::bad_alloc&) {
        return refuse("az_muon_step: out of host memory");
    }
    if (!apart) return refuse("az_muon_step: weights and momenta must not overlap each other or a gradient");
    if (!isfinite(lr) || !isfinite(weight_decay) || !(momentum >= 0 && momentum < 1))
        return refuse("az_muon_step: bad lr, weight_decay or momentum (0 <= momentum < 1)");
    return ortho_check(dtype, steps, coeffs, eps);
}

int az_muon_step_dev(int device, int dtype, const az_muon_item* items, int64_t n, double lr, double momentum, int nesterov,
                     double weight_decay, int steps, const double* coeffs, double eps, void* ws_dev, size_t ws_bytes,
                     void* stream) {
    int rc = az_muon_step_check(dtype, items, n, lr, momentum, weight_decay, steps, coeffs, eps);
    if (rc == AZ_OK) rc = ws_check(ws_dev, ws_bytes, az_muon_step_ws(items, n));
    if (rc != AZ_OK) return rc;
    DeviceScope dev(device);
    if (dev.rc != AZ_OK || n == 0) return dev.rc;
    Hyper h = {};
    h.mu = (float)momentum;
    h.one_mu = (float)(1.0 - momentum);
    h.decay = (float)(1.0 - lr * weight_decay);
    h.lr = (float)lr;
    h.a = (float)coeffs[0];
    h.b = (float)coeffs[1];
    h.c = (float)coeffs[2];
    h.eps = eps;
    h.nesterov = nesterov != 0;
    h.update = 1;
    for (int64_t lo = 0; lo < n; lo += MAX_JOBS) {
        Jobs js;
        js.n = (i32)(n - lo < MAX_JOBS ? n - lo : MAX_JOBS);
        size_t off = 0;
        for (int i = 0; i < js.n; i++) {
            const az_muon_item& it = items[lo + i];
            Job& J = js.j[i];
            off += plan(J, it.rows, it.cols, (char*)ws_dev + off);
            J.g = it.g_dev;
            J.w = it.w_dev;
            J.m = it.m_dev;
        }
        rc = run_jobs(js, h, steps, dtype, (hipStream_t)stream);
        if (rc != AZ_OK) return rc;
    }
    return AZ_OK;
}

}  // extern "C"
