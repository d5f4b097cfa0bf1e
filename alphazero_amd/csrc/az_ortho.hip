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
    u8 *x, *t[2], *a, *b;   // split operands in panels: 16 values of every row (16 hi, 16 lo: 64 bytes), then the next 16
    // short side <= 128 (see "Narrow matrices"): T in MFMA order in t, partial Gram matrices in gram
    float* gram[2];
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
template <class T>
__device__ inline float update_value(const Job& J, const Hyper& h, i64 i) {   // after k_ortho_norm has updated m
    const float g = to_f32(((const T*)J.g)[i]);
    if (!h.update) return g;
    const float m = J.m[i];
    return h.nesterov ? h.mu * m + h.one_mu * g : m;
}
__device__ inline void split_store(u8* p, float v) {   // p: the high half's place
    const f16 hi = (f16)v;
    *(f16*)p = hi;
    *(f16*)(p + 32) = (f16)(v - (float)hi);
}
__device__ inline i64 split_off(i64 row, i64 rows, i64 k) { return ((k >> 4) * rows + row) * TILE_KB + (k & 15) * 2; }

// momentum (in place) and partial sums of squares of the update, in float64: the squares of float32 values can leave float32
template <class T>
__global__ __launch_bounds__(256) void k_ortho_norm(Jobs js, Hyper h) {
    __shared__ double red[4];
    const int ji = find_job(js, blockIdx.x);
    const Job& J = js.j[ji];
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

// X and T from the update, padding included: one 64 x 64 tile per workgroup
template <class T>
__global__ __launch_bounds__(256) void k_ortho_init(Jobs js, Hyper h) {
    __shared__ float tile[OT][OT + 1];   // [short index][long index]
    __shared__ double red[4];
    const int ji = find_job(js, blockIdx.x), tid = threadIdx.x;
    const Job& J = js.j[ji];
    const int nl = J.lp / OT, tl = blockIdx.x - js.first[ji], i0 = tl / nl * OT, j0 = tl % nl * OT;
    double sum = 0;
    for (int i = tid; i < J.n_part; i += 256) sum += J.part[i];
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((tid & 63) == 0) red[tid >> 6] = sum;
    __syncthreads();
    const float scale = (float)(16384.0 / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + h.eps));
    const bool flip = J.rows > J.cols;
    for (int e = tid; e < OT * OT; e += 256) {
        const int hi_ = e / OT, lo_ = e % OT;           // lo_ runs along the matrix's rows in memory
        const int i = flip ? lo_ : hi_, j = flip ? hi_ : lo_;
        float v = 0;
        if (i0 + i < J.s && j0 + j < J.l)
            v = update_value<T>(J, h, flip ? (i64)(j0 + j) * J.cols + i0 + i : (i64)(i0 + i) * J.cols + j0 + j) * scale;
        tile[i][j] = v;
    }
    __syncthreads();
    for (int e = tid; e < OT * OT; e += 256) {
        const int r = e / OT, c = e % OT;
        split_store(J.x + split_off(i0 + r, J.sp, j0 + c), tile[r][c]);
        split_store(J.t[0] + split_off(j0 + r, J.lp, i0 + c), tile[c][r]);
    }
}

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

enum { GRAM = 0, POLY = 1, STEP = 2, LAST = 3 };
// GRAM: A = X X^T     POLY: B = a I + b A + c A A^T     STEP: T <- T B (and X)     LAST: the output, in its own orientation
// A and B are symmetric: their launches compute the tiles that touch the lower triangle and store them twice.

// rows and columns of a launch's result (padded)
__host__ __device__ inline void product_dims(int mode, const Job& J, int& rows, int& cols) {
    const bool flip = J.rows > J.cols;
    rows = mode == GRAM || mode == POLY ? J.sp : (mode == STEP || flip ? J.lp : J.sp);
    cols = mode == LAST && !flip ? J.lp : J.sp;
}
// tiles of a symmetric launch: tile row i covers rows from bm i on and has the tiles whose first column is not behind its last
// row: (i + 1) bm / bn of them, but for the last row, which ends with the matrix
__host__ __device__ inline int symmetric_tiles(int n, int bm, int bn) {
    const int full = n / bm, per = bm / bn;
    return per * full * (full + 1) / 2 + (n % bm ? (n + bn - 1) / bn : 0);
}

// the tile's result passes through LDS as float32, so that rows leave it 16 bytes a lane
template <class S>
struct Staged {
    static constexpr int PITCH = S::BN + 4;   // floats; rows stay 16-byte aligned and start 4 banks apart
    static constexpr int BYTES = S::BM * PITCH * 4;
    static constexpr int LDS = BYTES > S::LDS ? BYTES : S::LDS;
};

template <int MODE, class S, class T>
__global__ __launch_bounds__(S::THREADS) void k_ortho_product(Jobs js, Hyper h, int cur) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    const int ji = find_job(js, blockIdx.x), tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job& J = js.j[ji];
    const bool flip = J.rows > J.cols;
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    const u8 *P, *Q;
    int kp, rows, cols;
    product_dims(MODE, J, rows, cols);
    if (MODE == GRAM) { P = Q = J.x; kp = J.lp; }
    else if (MODE == POLY) { P = Q = J.a; kp = J.sp; }
    else if (MODE == STEP || flip) { P = J.t[cur]; Q = J.b; kp = J.sp; }
    else { P = J.b; Q = J.t[cur]; kp = J.sp; }
    u32 tm, tn;
    const int block = blockIdx.x - js.first[ji];
    if (SYM) {
        constexpr int PER = S::BM / S::BN;
        tm = (u32)((sqrtf(8.0f * (float)(block / PER) + 1.0f) - 1.0f) * 0.5f);   // the row i with PER i (i + 1) / 2 <= block
        while (PER * tm * (tm + 1) / 2 > (u32)block) tm--;
        while (PER * (tm + 1) * (tm + 2) / 2 <= (u32)block) tm++;
        tn = block - PER * tm * (tm + 1) / 2;
    } else {
        tile_place(block, (rows + S::BM - 1) / S::BM, (cols + S::BN - 1) / S::BN, tm, tn);
    }
    const int m0 = tm * S::BM, n0 = tn * S::BN;
    const int mrows = rows - m0 < S::BM ? rows - m0 : S::BM, ncols = cols - n0 < S::BN ? cols - n0 : S::BN;
    const TileSrc<false> p(P + m0 * TILE_KB, (u64)rows * TILE_KB, TILE_KB, mrows * TILE_KB, lane);
    const TileSrc<S::PAIRS> q(Q + n0 * TILE_KB, (u64)cols * TILE_KB, TILE_KB, ncols * TILE_KB, lane);
    f32x16 acc[S::FM][S::FN] = {};
    tile_product<KindSplit, S>(KindSplit(), p, q, 0, kp * 4, lds, wave, lane, acc);

    constexpr int W = S::PAIRS ? 2 : 1, PITCH = Staged<S>::PITCH;
    constexpr float UNIT = MODE == GRAM ? 0x1p-16f : MODE == POLY ? 0x1p-24f : MODE == STEP ? 0x1p-11f : 0x1p-25f;
    float* tile = (float*)lds;
#pragma unroll
    for (int i = 0; i < S::FM; i++)
#pragma unroll
        for (int j = 0; j < S::FN; j += W)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                float* d = tile + (wave / S::WN * (S::FM * 32) + 32 * i + acc_row(r, lane)) * PITCH + wave % S::WN * (S::FN * 32) +
                           32 * j + W * (lane & 31);
                d[0] = acc[i][j][r] * UNIT;
                if (W == 2) d[1] = acc[i][j + W - 1][r] * UNIT;
            }
    __syncthreads();
    if (MODE != LAST) {   // mrows and ncols are multiples of 64 here
        u8* out = MODE == GRAM ? J.a : MODE == POLY ? J.b : J.t[cur ^ 1];
        // pairs of lanes store 16 values of a row, 64 bytes; the next pair those of the next row, right behind them
        for (int u = tid; u < S::BM * S::BN / 8; u += S::THREADS) {
            const int r = u / 2 % S::BM, c = (u % 2 + u / (2 * S::BM) * 2) * 8, m = m0 + r, n = n0 + c;
            if (r >= mrows || c >= ncols) continue;
            float v[8];
            float* d = tile + r * PITCH + c;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = d[e];
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
        // transposed: X for STEP, the mirrored tile for A and B.  The tiles across the diagonal cover both sides themselves: a
        // mirrored value could differ from the computed one in its last bit, and both would be written.
        if (SYM && n0 + S::BN > m0) return;
        if (MODE == POLY) __syncthreads();
        u8* outT = MODE == STEP ? J.x : out;
        for (int u = tid; u < S::BM * S::BN / 8; u += S::THREADS) {
            const int c = u / 2 % S::BN, r = (u % 2 + u / (2 * S::BN) * 2) * 8;
            if (r >= mrows || c >= ncols) continue;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = tile[(r + e) * PITCH + c];
            split_store8(outT + split_off(n0 + c, cols, m0 + r), v);
        }
    } else {
        for (int u = tid; u < S::BM * S::BN; u += S::THREADS) {
            const int r = u / S::BN, c = u % S::BN;
            if (m0 + r >= J.rows || n0 + c >= J.cols) continue;
            float o = tile[r * PITCH + c];
            T* w = (T*)J.w + (i64)(m0 + r) * J.cols + n0 + c;
            if (h.update) o = to_f32(*w) * h.decay - o * (h.lr * J.kappa);
            *w = from_f32<T>(o);
        }
    }
}

using OTile128 = TileShape<128, 128, 2, 2, 4>;
using OTile128s = TileShape<128, 64, 2, 2, 4>;   // symmetric results
using OTile64 = TileShape<64, 64, 2, 2, 4>;

// ---------------------------------------------------------------------------------------------------- Narrow matrices
// Short side s <= 128: a launch a step.  B (s x s) fits LDS, and so does a panel of 128 values of the long index; every workgroup
// owns some panels and
//   1. adds the panels' partial Gram matrices that the launch before left (in order, so the sum is the same every time),
//   2. makes B = a I + b A + c A A^T for itself,
//   3. multiplies its panels by it, keeping T for the next launch, and adds up their part of the next Gram matrix.
// What bounds it is latency: 5 steps of a 128 x 1152 matrix are 0.4 GFLOP, but 15 products one after the other; between launches,
// each product would start on cold operands.
//
// T goes through memory in the order in which the MFMA of 3. takes it and the one before leaves it.  D = B T^T leaves lane
// (h = lane / 32, j = lane % 32) rows i = 8 (r / 4) + 4 h + r % 4 of column j: eight registers are eight values of k for lane (h, j) of the
// next product, if its k runs in the order that swaps bits 2 and 3 of i.  Columns of A and B in LDS are kept in that order.
constexpr int NARROW = 128, NPANEL = 128, NTHREADS = 512, NWAVES = 8;
constexpr int NBUF = NARROW * 512;   // a row: 128 high halves, 128 low halves
constexpr int MAX_GROUPS = 16;       // workgroups a matrix: each adds up that many partial Gram matrices

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
__device__ inline float nar_get(const u8* buf, int row, int k) {
    return (float)*(const f16*)(buf + nar_off(row, k, 0)) + (float)*(const f16*)(buf + nar_off(row, k, 1));
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
#pragma unroll 4
    for (int c = 0; c < steps; c++)
        mul3(acc, cross, nar_frag(P, p + r, c, h, 0), nar_frag(P, p + r, c, h, 1), nar_frag(Q, q + r, c, h, 0),
             nar_frag(Q, q + r, c, h, 1));
    acc += cross;
}
// a block of a symmetric matrix, both ways
__device__ inline void nar_put_symmetric(u8* buf, int bi, int bj, int lane, const f32x16& v) {
    const int n = bj * 32 + (lane & 31);
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const int m = bi * 32 + acc_row(4 * g, lane);
        typedef f16 f16x4 __attribute__((ext_vector_type(4)));
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x = v[4 * g + e];
            hi[e] = (f16)x;
            lo[e] = (f16)(x - (float)hi[e]);
            *(f16*)(buf + nar_off(m + e, swap23(n), 0)) = hi[e];
            *(f16*)(buf + nar_off(m + e, swap23(n), 1)) = lo[e];
        }
        if (bi != bj) {   // four rows from a multiple of four on stay together
            *(f16x4*)(buf + nar_off(n, swap23(m), 0)) = hi;
            *(f16x4*)(buf + nar_off(n, swap23(m), 1)) = lo;
        }
    }
}
__device__ inline int nar_blocks(const Job& J) { return J.nb * (J.nb + 1) / 2; }
// this wave's blocks (wave, wave + 8) of the panel's Gram matrix; the panel is in buf as [short index][long index]
__device__ inline void nar_gram(const Job& J, const u8* buf, int wave, int lane, f32x16 (&acc)[2]) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int b = wave + NWAVES * x;
        if (b >= nar_blocks(J)) continue;
        int bi, bj;
        lower_block(b, bi, bj);
        nar_block(buf, bi * 32, buf, bj * 32, NPANEL / 16, lane, acc[x]);
    }
}
__device__ inline void nar_gram_store(const Job& J, float* gram, int group, int wave, int lane, const f32x16 (&acc)[2]) {
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int b = wave + NWAVES * x;
        if (b >= nar_blocks(J)) continue;
        float* d = gram + ((i64)(group * nar_blocks(J) + b) * 64 + lane) * 16;
#pragma unroll
        for (int g = 0; g < 4; g++) *(f32x4*)(d + 4 * g) = f32x4{acc[x][4 * g], acc[x][4 * g + 1], acc[x][4 * g + 2], acc[x][4 * g + 3]};
    }
}
// T of panel p, long-index block jb (32 values), k step c: 64 lanes x 16 bytes
__device__ inline u8* nar_t(u8* t, int p, int jb, int c, int low) { return t + ((((i64)p * 4 + jb) * 8 + c) * 2 + low) * 1024; }

template <class T>
__global__ __launch_bounds__(NTHREADS) void k_narrow_init(Jobs js, Hyper h) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    __shared__ double red[NWAVES];
    const int ji = find_job(js, blockIdx.x), tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Job& J = js.j[ji];
    const int group = blockIdx.x - js.first[ji], panels = (J.l + NPANEL - 1) / NPANEL, height = J.nb * 32;
    const bool flip = J.rows > J.cols;
    double sum = 0;
    for (int i = tid; i < J.n_part; i += NTHREADS) sum += J.part[i];
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) red[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int i = 0; i < NWAVES; i++) sum += red[i];
    const float scale = (float)(16384.0 / (sqrt(sum) + h.eps));
    f32x16 acc[2] = {};
    for (int p = group * J.per_group; p < panels && p < (group + 1) * J.per_group; p++) {
        const int j0 = p * NPANEL;
#pragma unroll 8
        for (int e = tid; e < height * NPANEL; e += NTHREADS) {   // consecutive threads along the matrix's rows in memory
            const int i = flip ? e % height : e / NPANEL, j = flip ? e / height : e % NPANEL;
            float v = 0;
            if (i < J.s && j0 + j < J.l)
                v = update_value<T>(J, h, flip ? (i64)(j0 + j) * J.cols + i : (i64)i * J.cols + j0 + j) * scale;
            nar_put(lds, i, j, v);
        }
        __syncthreads();
        const int jb = wave & 3, hh = lane >> 5, j = jb * 32 + (lane & 31);
        for (int c = (wave >> 2) * 4; c < (wave >> 2) * 4 + 4 && c < 2 * J.nb; c++)
            for (int low = 0; low < 2; low++) {
                f16x8 f;
#pragma unroll
                for (int e = 0; e < 8; e++) f[e] = *(const f16*)(lds + nar_off(16 * c + swap23(8 * hh + e), j, low));
                *(f16x8*)(nar_t(J.t[0], p, jb, c, low) + lane * 16) = f;
            }
        nar_gram(J, lds, wave, lane, acc);
        __syncthreads();
    }
    nar_gram_store(J, J.gram[0], group, wave, lane, acc);
}

template <class T, bool LASTSTEP>
__global__ __launch_bounds__(NTHREADS) void k_narrow_step(Jobs js, Hyper h, int cur) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    u8 *const bufA = lds, *const bufB = lds + NBUF;   // A, then the new panel; B
    const int ji = find_job(js, blockIdx.x), lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Job& J = js.j[ji];
    const int group = blockIdx.x - js.first[ji], panels = (J.l + NPANEL - 1) / NPANEL, blocks = nar_blocks(J), steps = 2 * J.nb;
    const int first = group * J.per_group, end = first + J.per_group < panels ? first + J.per_group : panels;
    const bool flip = J.rows > J.cols;
    const int jb = wave & 3, ib = (wave >> 2) * 2;   // this wave: 32 of the panel's long index, short-index blocks ib, ib + 1
    f16x8 t[8][2];
    auto fetch = [&](int p) {
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (c < steps)
#pragma unroll
                for (int low = 0; low < 2; low++) t[c][low] = *(const f16x8*)(nar_t(J.t[cur], p, jb, c, low) + lane * 16);
    };
    if (first < end) fetch(first);
    // 1. A = sum of the groups' parts
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int b = wave + NWAVES * x;
        if (b >= blocks) continue;
        f32x16 v = {};
        for (int g = 0; g < J.groups; g++) {
            const f32x4* d = (const f32x4*)(J.gram[cur] + ((i64)(g * blocks + b) * 64 + lane) * 16);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const f32x4 y = d[k];
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * k + e] += y[e];
            }
        }
        int bi, bj;
        lower_block(b, bi, bj);
        nar_put_symmetric(bufA, bi, bj, lane, v * 0x1p-16f);
    }
    __syncthreads();
    // 2. B
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int b = wave + NWAVES * x;
        if (b >= blocks) continue;
        int bi, bj;
        lower_block(b, bi, bj);
        f32x16 acc = {};
        nar_block(bufA, bi * 32, bufA, bj * 32, steps, lane, acc);
        const int n = bj * 32 + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int m = bi * 32 + acc_row(r, lane);
            const float A = nar_get(bufA, m, swap23(n)) * 0x1p-12f;
            acc[r] = (h.c * (acc[r] * 0x1p-24f) + h.b * A + (m == n ? h.a : 0.0f)) * 0x1p11f;
        }
        nar_put_symmetric(bufB, bi, bj, lane, acc);
    }
    __syncthreads();
    // 3. the panels
    f32x16 gram[2] = {};
    for (int p = first; p < end; p++) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            if (ib + x >= J.nb) continue;
            const int i0 = (ib + x) * 32, hh = lane >> 5;
            f32x16 acc = {}, cross = {};
            const bool across = LASTSTEP && flip;   // the output's rows are the long index: lanes along the short one
#pragma unroll
            for (int c = 0; c < 8; c++) {
                if (c >= steps) continue;
                const f16x8 bh = nar_frag(bufB, i0 + (lane & 31), c, hh, 0), bl = nar_frag(bufB, i0 + (lane & 31), c, hh, 1);
                if (across) mul3(acc, cross, t[c][0], t[c][1], bh, bl);
                else mul3(acc, cross, bh, bl, t[c][0], t[c][1]);
            }
            acc += cross;
            if (!LASTSTEP) {
                acc *= 0x1p-11f;
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
                    const int c = 2 * (ib + x) + half;
                    *(f16x8*)(nar_t(J.t[cur ^ 1], p, jb, c, 0) + lane * 16) = hi;
                    *(f16x8*)(nar_t(J.t[cur ^ 1], p, jb, c, 1) + lane * 16) = lo;
                }
            } else {
                const int col = (across ? i0 : p * NPANEL + jb * 32) + (lane & 31), row0 = across ? p * NPANEL + jb * 32 : i0;
                float old[16];
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int row = row0 + acc_row(r, lane);
                    old[r] = h.update && row < J.rows && col < J.cols ? to_f32(((const T*)J.w)[(i64)row * J.cols + col]) : 0.0f;
                }
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int row = row0 + acc_row(r, lane);
                    if (row >= J.rows || col >= J.cols) continue;
                    float o = acc[r] * 0x1p-25f;
                    if (h.update) o = old[r] * h.decay - o * (h.lr * J.kappa);
                    ((T*)J.w)[(i64)row * J.cols + col] = from_f32<T>(o);
                }
            }
        }
        if (p + 1 < end) fetch(p + 1);
        if (!LASTSTEP) {
            __syncthreads();
            nar_gram(J, bufA, wave, lane, gram);
            __syncthreads();
        }
    }
    if (!LASTSTEP) nar_gram_store(J, J.gram[cur ^ 1], group, wave, lane, gram);
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
        for (int i = 0; i < 2; i++) {
            J.t[i] = take((size_t)panels * NPANEL * NARROW * 4);
            J.gram[i] = (float*)take((size_t)J.groups * (J.nb * (J.nb + 1) / 2) * 4096);
        }
        J.x = J.a = J.b = nullptr;
        return off;
    }
    J.gram[0] = J.gram[1] = nullptr;
    J.groups = J.per_group = 0;
    J.x = take((size_t)J.sp * J.lp * 4);
    J.t[0] = take((size_t)J.sp * J.lp * 4);
    J.t[1] = take((size_t)J.sp * J.lp * 4);
    J.a = take((size_t)J.sp * J.sp * 4);
    J.b = take((size_t)J.sp * J.sp * 4);
    return off;
}

// Which coefficients keep the halves in range: follows the largest singular value through the steps on a fine grid.
static bool coeffs_ok(int steps, const double* k) {
    if (!k || !isfinite(k[0]) || !isfinite(k[1]) || !isfinite(k[2])) return false;
    double top = 1.0;
    for (int it = 0; it < steps; it++) {
        double next = 0;
        for (int i = 0; i <= 4096; i++) {
            const double x = top * i / 4096, x2 = x * x, poly = k[0] + k[1] * x2 + k[2] * x2 * x2;
            if (fabs(poly) > 15.9 || fabs(poly - k[0]) > 15.9) return false;
            next = fmax(next, fabs(poly * x));
        }
        top = next * 1.001;
        if (top > 1.99) return false;
    }
    return true;
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
        if (MODE == GRAM || MODE == POLY) return (i64)symmetric_tiles(J.sp, S::BM, S::BN);
        return (i64)((rows + S::BM - 1) / S::BM) * ((cols + S::BN - 1) / S::BN);
    });
    return js.first[js.n];
}
template <int MODE, class T>
static void product(Jobs& js, const Hyper& h, int cur, hipStream_t st) {
    // the larger tile reads half as much per product; it needs enough tiles to fill the chip
    if constexpr (MODE == GRAM || MODE == POLY) {
        const int n = product_blocks<MODE, OTile128s>(js);
        if (n >= 160) {
            k_ortho_product<MODE, OTile128s, T><<<dim3((u32)n), dim3(OTile128s::THREADS), Staged<OTile128s>::LDS, st>>>(js, h, cur);
            return;
        }
    } else {
        const int n = product_blocks<MODE, OTile128>(js);
        if (n >= 160) {
            k_ortho_product<MODE, OTile128, T><<<dim3((u32)n), dim3(OTile128::THREADS), Staged<OTile128>::LDS, st>>>(js, h, cur);
            return;
        }
    }
    const int n = product_blocks<MODE, OTile64>(js);
    k_ortho_product<MODE, OTile64, T><<<dim3((u32)n), dim3(OTile64::THREADS), Staged<OTile64>::LDS, st>>>(js, h, cur);
}

static int run_narrow(Jobs& js, const Hyper& h, int steps, int dtype, hipStream_t st) {
    each_first(js, [](const Job& J) { return J.n_part; });
    AZ_DISPATCH_DTYPE(dtype, k_ortho_norm<T><<<dim3(js.first[js.n]), dim3(256), 0, st>>>(js, h));
    each_first(js, [](const Job& J) { return J.groups; });
    const dim3 grid(js.first[js.n]), block(NTHREADS);
    AZ_DISPATCH_DTYPE(dtype, k_narrow_init<T><<<grid, block, NBUF, st>>>(js, h));
    for (int it = 0; it + 1 < steps; it++) k_narrow_step<float, false><<<grid, block, 2 * NBUF, st>>>(js, h, it & 1);
    AZ_DISPATCH_DTYPE(dtype, k_narrow_step<T, true><<<grid, block, 2 * NBUF, st>>>(js, h, (steps - 1) & 1));
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
    int cur = 0;
    for (int it = 0; it < steps; it++) {
        product<GRAM, float>(js, h, cur, st);
        product<POLY, float>(js, h, cur, st);
        if (it + 1 < steps) {
            product<STEP, float>(js, h, cur, st);
        } else {
            AZ_DISPATCH_DTYPE(dtype, product<LAST, T>(js, h, cur, st));
        }
        cur ^= 1;
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

static int ortho_check(int dtype, int steps, const double* coeffs, double eps, const void* ws, size_t ws_bytes, size_t need) {
    if (!dtype_ok(dtype)) return refuse("az_orthogonalize: unknown dtype");
    if (steps < 1 || steps > 16) return refuse("az_orthogonalize: steps is 1..16");
    if (!(eps > 0) || !isfinite(eps)) return refuse("az_orthogonalize: eps must be positive and finite");
    if (!coeffs_ok(steps, coeffs)) return refuse("az_orthogonalize: these coefficients leave the range of the products");
    if (ws_bytes < need || (need && (!ws || ((uintptr_t)ws & 255))))
        return refuse("az_orthogonalize: workspace too small or not aligned to 256 bytes");
    return AZ_OK;
}

int az_orthogonalize_dev(int device, int dtype, int64_t batch, int64_t rows, int64_t cols, const void* g_dev, void* out_dev,
                         int steps, const double* coeffs, double eps, void* ws_dev, size_t ws_bytes, void* stream) {
    if (batch < 0 || !dims_ok(rows, cols)) return refuse("az_orthogonalize: bad shape (rows and cols are 1..32768)");
    int rc = ortho_check(dtype, steps, coeffs, eps, ws_dev, ws_bytes, az_orthogonalize_ws(batch, rows, cols));
    if (rc != AZ_OK) return rc;
    if (batch > 0 && (!g_dev || !out_dev)) return refuse("az_orthogonalize: null pointer");
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

int az_muon_step_dev(int device, int dtype, const az_muon_item* items, int64_t n, double lr, double momentum, int nesterov,
                     double weight_decay, int steps, const double* coeffs, double eps, void* ws_dev, size_t ws_bytes,
                     void* stream) {
    if (n < 0 || n > 65536 || (n > 0 && !items)) return refuse("az_muon_step: bad item list");
    if (!dtype_ok(dtype)) return refuse("az_muon_step: unknown dtype");
    for (int64_t i = 0; i < n; i++) {
        if (!dims_ok(items[i].rows, items[i].cols)) return refuse("az_muon_step: bad shape (rows and cols are 1..32768)");
        if (!items[i].w_dev || !items[i].g_dev || !items[i].m_dev) return refuse("az_muon_step: null pointer");
    }
    // what is written (w, m) overlaps nothing else
    auto overlap = [](const void* p, size_t np, const void* q, size_t nq) {
        return (uintptr_t)p < (uintptr_t)q + nq && (uintptr_t)q < (uintptr_t)p + np;
    };
    for (int64_t i = 0; i < n; i++) {
        const size_t ni = (size_t)items[i].rows * items[i].cols, es = dtype_size(dtype);
        for (int64_t k = 0; k < n; k++) {
            const size_t nk = (size_t)items[k].rows * items[k].cols;
            if ((k < i && (overlap(items[i].w_dev, ni * es, items[k].w_dev, nk * es) ||
                           overlap(items[i].m_dev, ni * 4, items[k].m_dev, nk * 4))) ||
                overlap(items[i].w_dev, ni * es, items[k].m_dev, nk * 4) ||
                overlap(items[i].g_dev, ni * es, items[k].w_dev, nk * es) ||
                overlap(items[i].g_dev, ni * es, items[k].m_dev, nk * 4))
                return refuse("az_muon_step: weights and momenta must not overlap each other or a gradient");
        }
    }
    if (!isfinite(lr) || !isfinite(weight_decay) || !(momentum >= 0 && momentum < 1))
        return refuse("az_muon_step: bad lr, weight_decay or momentum (0 <= momentum < 1)");
    int rc = ortho_check(dtype, steps, coeffs, eps, ws_dev, ws_bytes, az_muon_step_ws(items, n));
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
