// az_int8.hip -- evaluation of layers in 8-bit integers: rows quantised with a scale each, products with a scale for each
// row (token) and each output channel.
//
//   q[r][c] = rint(x[r][c] / s[r]),  s[r] = max|x[r]| * (1/127)     y[m][n] = act(s[m] ws[n] sum_k q[m][k] w[n][k] + b[n] + res)
//
// The sums are int32 and exact (|q w| <= 2^14, k <= 131071), so no order of summation changes a result.
#include <math.h>

#include <type_traits>

#include "az_tile.hpp"

namespace az {

constexpr i64 I8_MAX_K = 131071;

// ---------------------------------------------------------------------------------------------------- rows to 8 bits
// x / s rounded to the nearest integer, ties to even, by the exact quotient.  t = rint(x * (1/s)) is off by one at most, and
// only next to a half; e = x - t s is exact (one fma) wherever |e| is near s / 2: both are then multiples of half an ulp
// of s below 2^24 of them, but for x just below s / 2, which rounds to the tie and from there to the even t = 0, as it should.
__device__ inline int quant1(float x, float s, float rs) {
    float t = rintf(x * rs);
    const float e = fmaf(-t, s, x), half = 0.5f * s;
    const bool odd = ((int)t & 1) != 0;
    if (e > half || (e == half && odd)) t += 1.0f;
    else if (e < -half || (e == -half && odd)) t -= 1.0f;
    return (int)fminf(fmaxf(t, -127.0f), 127.0f);
}
// scales below 2^-100 (1/s or s/2 would leave the normal range): the same by a float64 quotient, whose rounding cannot
// cross a half either (53 bits against operands of 24)
__device__ inline int quant1_tiny(float x, float s) {
    return (int)fmin(fmax(rint((double)x / (double)s), -127.0), 127.0);
}
// the scale of a row from the bits of its largest magnitude: times the float32 next to 1/127, NaN if the row is not finite
__device__ inline float row_scale(u32 mx) {
    return mx >= 0x7f800000u ? __builtin_nanf("") : __builtin_bit_cast(float, mx) * (1.0f / 127.0f);
}
constexpr float QUANT_TINY = 7.8886090522101181e-31f;   // 2^-100

// 16 bytes of a row: EPP values
template <class T>
struct Piece {
    static constexpr int EPP = 16 / sizeof(T);
    u32x4 raw;
    __device__ float get(int e) const {
        T v[EPP];
        __builtin_memcpy(v, &raw, 16);
        return to_f32(v[e]);
    }
    // largest magnitude as float32 bits, compared as integers, which keeps a NaN on top (fmaxf would drop it)
    __device__ u32 most() const {
        if constexpr (sizeof(T) == 4) {
            const u32x4 b = raw & 0x7fffffffu;
            const u32 x = b[0] > b[1] ? b[0] : b[1], y = b[2] > b[3] ? b[2] : b[3];
            return x > y ? x : y;
        } else {   // 16-bit magnitudes order alike: two a lane register, widened at the end
            typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
            typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            const u16x8 b = __builtin_bit_cast(u16x8, raw & 0x7fff7fffu);
            const u16x4 c = __builtin_elementwise_max(b.lo, b.hi);
            const u16x2 d = __builtin_elementwise_max(c.lo, c.hi);
            const unsigned short m = d[0] > d[1] ? d[0] : d[1];
            return __builtin_bit_cast(u32, to_f32(__builtin_bit_cast(T, m))) & 0x7fffffffu;
        }
    }
    __device__ void load(const T* p, int n) {   // n values of it, zeros behind
        if (n >= EPP) {
            __builtin_memcpy(&raw, p, 16);
        } else {
            T v[EPP];
#pragma unroll
            for (int e = 0; e < EPP; e++) v[e] = e < n ? p[e] : (T)0.0f;
            __builtin_memcpy(&raw, v, 16);
        }
    }
    static __device__ void pack(const u32 (&g)[EPP], u32 (&out)[EPP / 4]) {
#pragma unroll
        for (int e = 0; e < EPP / 4; e++)   // v_perm_b32: bytes 0..3 are the second operand's, 4..7 the first's
            out[e] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(g[4 * e + 3], g[4 * e + 2], 0x0c0c0400),
                                           __builtin_amdgcn_perm(g[4 * e + 1], g[4 * e], 0x0c0c0400), 0x05040100);
    }
    // the EPP integers as bytes: x * (1/s) + 1.5 2^23 holds rint(x / s) in its low byte, but next to a half, where 1/s may have
    // taken it over: |x (1/s) - t| exceeds 1/2 - 2^-17 there (the fma rounds once, to the integer; 1/s is off by 2^-24 of itself,
    // x (1/s) by 127 * 2^-24 = 7.57e-6, the difference below by 2^-26 more: 7.59e-6 < 2^-17).  False: the exact way it has to go.
    __device__ bool quantize(float rs, u32 (&out)[EPP / 4]) const {
        constexpr float MAGIC = 12582912.0f;
        u32 g[EPP];
        float far = 0;
#pragma unroll
        for (int e = 0; e < EPP; e++) {
            const float x = get(e), m = fmaf(x, rs, MAGIC);
            far = fmaxf(far, fabsf(fmaf(x, rs, MAGIC - m)));
            g[e] = __builtin_bit_cast(u32, m);
        }
        pack(g, out);
        return far <= 0.5f - 0x1p-17f;
    }
    __device__ void quantize_exact(float s, float rs, u32 (&out)[EPP / 4]) const {
        u32 g[EPP];
#pragma unroll
        for (int e = 0; e < EPP; e++) g[e] = (u32)(s >= QUANT_TINY ? quant1(get(e), s, rs) : quant1_tiny(get(e), s));
        pack(g, out);
    }
};

struct Rows {
    i64 rows, cols, ld_x, n_src, ld_q;
    const void* x;
    const i32* index;
    i8* q;
    float* scale;
    u32 taps, per_tap, pieces, magic;   // pieces of a row: taps * per_tap; p / per_tap = (p * magic) >> 32, magic 0: divide
    bool fill;                           // zeros behind the row up to ld_q
    float inv_tap;                       // 1 / per_tap
    u32 x_bytes, row_bytes;              // FAST: bytes of x, and from row to row
};
// where piece p of row r comes from (null: zeros), how many values it has, and its place in the row of q
template <class T>
__device__ inline const T* piece_source(const Rows& R, i64 r, u32 p, int& n, u32& to) {
    constexpr int EPP = Piece<T>::EPP;
    const u32 tap = R.taps == 1 ? 0 : R.magic ? __umulhi(p, R.magic) : p / R.per_tap, in = p - tap * R.per_tap;
    const u32 c = in * EPP, cols = (u32)R.cols;
    n = cols - c < EPP ? (int)(cols - c) : EPP;
    to = tap * cols + c;
    const i64 src = R.index ? (i64)R.index[r * R.taps + tap] : r;
    return src >= 0 && src < R.n_src ? (const T*)R.x + src * R.ld_x + c : nullptr;
}
template <class T>
__device__ inline void piece_store(i8* d, const u32 (&v)[Piece<T>::EPP / 4], int n) {
    constexpr int EPP = Piece<T>::EPP;
    if (n >= EPP) {
        __builtin_memcpy(d, v, EPP);
    } else {
        i8 b[EPP];
        __builtin_memcpy(b, v, EPP);
#pragma unroll
        for (int e = 0; e < EPP; e++)
            if (e < n) d[e] = b[e];
    }
}

template <int CTRL>
__device__ inline u32 dpp_max(u32 v) {
    const u32 o = (u32)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return o > v ? o : v;
}
// over groups of LANES (4, 16, 64) neighbouring lanes, the same in each of them
template <int LANES>
__device__ inline u32 lanes_max(u32 v) {
    v = dpp_max<0xB1>(v);   // quad_perm [1,0,3,2]
    v = dpp_max<0x4E>(v);   // quad_perm [2,3,0,1]
    if (LANES >= 16) {
        v = dpp_max<0x141>(v);   // row_half_mirror: the other quad of 8 (quads agree within)
        v = dpp_max<0x140>(v);   // row_mirror: the other 8 of 16
    }
    if (LANES >= 64) {
        const u32 a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
        const u32 c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
        const u32 x = a > b ? a : b, y = c > d ? c : d;
        v = x > y ? x : y;
    }
    return v;
}

// LANES lanes to a row, NP pieces of 16 bytes to a lane: the row is read once and stays in registers between its largest
// magnitude and its integers.  FAST: the columns are whole pieces, rows are 16-byte aligned, offsets fit 31 bits and the factors
// of a row's offset 24 (full-rate multiplications); rows that are not there are read behind the end of the buffer, as zeros.
// 86016 rows of 9 x 128 fp16 (22 MB read, 99 MB written): 37 us, 3.3 TB/s of the 5.1 that a copy reaches; what bounds it is the VALU
// (94 instructions for 8 values: the quotient, how near a half it is, the packing, the largest: 18.2 M a wave, of 4 cycles each, on 1024
// SIMDs are the kernel's 69 k cycles).  The same in bf16 43 us (conversions), in float32 85 (288 pieces, a row to 256 lanes: see
// rows_dispatch).  4099 x 1001 float32: 6.1 us, 3.4 TB/s.
// One row of 4096 bf16: 3.6 us, all of it latency: the load, the reduction over 4 waves, the launch.
template <class T, int LANES, int NP, bool FAST>
__global__ __launch_bounds__(256) void k_i8_quantize(Rows R) {
    constexpr int PER_BLOCK = 256 / LANES, EPP = Piece<T>::EPP;
    __shared__ u32 part[4];
    const int l = threadIdx.x % LANES;
    // the arguments in one go: asked for where they are used, they take three trips (one row of 4096: 2.7 us, 3.5)
    asm volatile("" ::"s"(R.rows), "s"(R.n_src), "s"(R.ld_q), "s"(R.x), "s"(R.index), "s"(R.q), "s"(R.scale), "s"(R.taps), "s"(R.pieces),
                 "s"(R.x_bytes), "s"(R.row_bytes), "s"(R.inv_tap), "s"((int)R.fill), "s"(R.cols), "s"(R.per_tap));
    for (i64 r0 = (i64)blockIdx.x * PER_BLOCK; r0 < R.rows; r0 += (i64)gridDim.x * PER_BLOCK) {
        const i64 r = r0 + threadIdx.x / LANES;
        const bool live = r < R.rows;
        Piece<T> v[NP];
        int n[NP];
        u32 to[NP], mx = 0;
        if constexpr (FAST) {
            const __amdgpu_buffer_rsrc_t rsrc =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(R.x), 0, (int)R.x_bytes, 0x00020000);
            u32 off[NP], src[NP];
            if (__builtin_expect(R.index != nullptr, 0)) {   // all at once, of lanes without a piece too: they read the row's last one, or the last row's
                const i32* at = R.index + (live ? r : R.rows - 1) * R.taps;
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    // p < 2^11 and, with more than one tap, per_tap <= 2^10: (p + 1/2) / per_tap is further from an integer than its error
                    const u32 p = l + i * LANES, tap = (u32)(((float)p + 0.5f) * R.inv_tap);
                    src[i] = (u32)at[tap < R.taps ? tap : R.taps - 1];
                    off[i] = (p - __umul24(tap, R.per_tap)) * 16;
                }
                loads_first();
            } else {
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    src[i] = (u32)r;
                    off[i] = (l + i * LANES) * 16;
                }
            }
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const bool in = live && l + i * LANES < R.pieces && src[i] < (u32)R.n_src;
                off[i] = in ? __umul24(src[i], R.row_bytes) + off[i] : 0x7ffffff0u;
            }
#pragma unroll
            for (int i = 0; i < NP; i++)
                v[i].raw = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)off[i], 0, 0));
        } else {
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const u32 p = l + i * LANES;
                n[i] = 0;
                v[i].raw = u32x4{0, 0, 0, 0};
                if (live && p < R.pieces) {
                    const T* src = piece_source<T>(R, r, p, n[i], to[i]);
                    if (src) v[i].load(src, n[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const u32 m = v[i].most();
            mx = m > mx ? m : mx;
        }
        mx = lanes_max<(LANES < 64 ? LANES : 64)>(mx);
        if (LANES == 256) {
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; i++) mx = part[i] > mx ? part[i] : mx;
            __syncthreads();
        }
        if (!live) continue;
        const float s = row_scale(mx), rs = 1.0f / s;
        if (l == 0) R.scale[r] = s;
        i8* q = R.q + r * R.ld_q;
        if (R.fill)
            for (i64 c = R.taps * R.cols + l; c < R.ld_q; c += LANES) q[c] = 0;
        u32 again = 0;   // pieces to do over the exact way
        const u32 keep = s >= QUANT_TINY ? ~0u : 0u;   // else s is 0, NaN or tiny
#pragma unroll
        for (int i = 0; i < NP; i++) {
            if (l + i * LANES >= R.pieces) continue;
            u32 out[EPP / 4];
            again |= v[i].quantize(rs, out) ? 0u : 1u << i;
#pragma unroll
            for (int e = 0; e < EPP / 4; e++) out[e] &= keep;
            piece_store<T>(q + (FAST ? (l + i * LANES) * EPP : to[i]), out, FAST ? EPP : n[i]);
        }
        if (!keep) {
            again = 0;
            for (int i = 0; i < NP && s > 0; i++) again |= l + i * LANES < R.pieces ? 1u << i : 0u;
        }
        while (again) {   // one copy of the code: about one piece in 2000 comes here
            const int i = __builtin_ctz(again);
            again &= again - 1;
            Piece<T> w = v[0];
            int k = FAST ? EPP : n[0];
            u32 at = FAST ? (l + i * LANES) * EPP : to[0];
#pragma unroll
            for (int j = 1; j < NP; j++)
                if (i == j) {
                    w = v[j];
                    if (!FAST) k = n[j], at = to[j];
                }
            u32 out[EPP / 4];
            w.quantize_exact(s, rs, out);
            piece_store<T>(q + at, out, k);
        }
    }
}
// rows of more than 256 * 8 pieces: a workgroup a row, read twice (the second time from L2, as a row is 32 KB and more)
template <class T>
__global__ __launch_bounds__(256) void k_i8_quantize_long(Rows R) {
    __shared__ u32 part[4];
    for (i64 r = blockIdx.x; r < R.rows; r += gridDim.x) {
        u32 mx = 0;
        for (u32 p = threadIdx.x; p < R.pieces; p += 256) {
            int n;
            u32 to;
            Piece<T> v;
            const T* src = piece_source<T>(R, r, p, n, to);
            if (!src) continue;
            v.load(src, n);
            const u32 m = v.most();
            mx = m > mx ? m : mx;
        }
        mx = lanes_max<64>(mx);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
        __syncthreads();
        for (int i = 0; i < 4; i++) mx = part[i] > mx ? part[i] : mx;
        __syncthreads();
        const float s = row_scale(mx), rs = 1.0f / s;
        if (threadIdx.x == 0) R.scale[r] = s;
        if (R.fill)
            for (i64 c = R.taps * R.cols + threadIdx.x; c < R.ld_q; c += 256) R.q[r * R.ld_q + c] = 0;
        for (u32 p = threadIdx.x; p < R.pieces; p += 256) {
            int n;
            u32 to;
            Piece<T> v;
            v.raw = u32x4{0, 0, 0, 0};
            const T* src = piece_source<T>(R, r, p, n, to);
            if (src) v.load(src, n);
            u32 out[Piece<T>::EPP / 4] = {};
            if (s > 0 && !(s >= QUANT_TINY && v.quantize(rs, out))) v.quantize_exact(s, rs, out);
            piece_store<T>(R.q + r * R.ld_q + to, out, n);
        }
    }
}

// ---------------------------------------------------------------------------------------------------- products
struct Mm {
    i64 m, n, k;
    const i8 *q, *w;
    i64 ld_q, ld_w;
    const float *qs, *ws, *bias;
    const void* res;
    i64 ld_res;
    void* y;
    i64 ld_y;
    int act;
    bool pair_store;   // every even column of y starts at a multiple of two elements
};

template <class T>
__device__ inline float activate(float v, int act) {
    if (act == AZ_ACT_RELU) return v > 0 || v != v ? v : 0.0f;
    if (act == AZ_ACT_SILU) {
        // For 16-bit results exp2 and rcp of the hardware (2^-22 each, and |v| 2^-24 from the exponent's rounding: far below the
        // 2^-12 of the result's own rounding wherever it is not vanishing): 6 instructions for the 35 of expf and the division,
        // which cost a 128 x 128 tile 4 us.
        if (sizeof(T) == 2) {
            const float e = __builtin_amdgcn_exp2f(v * -1.44269504088896340736f);
            return e == __builtin_inff() ? v * 0.0f : v * __builtin_amdgcn_rcpf(1.0f + e);
        }
        return v / (1.0f + expf(-v));
    }
    return v;
}

// 16 bytes of a row from byte k on, zeros behind its end; rows need not be aligned
__device__ inline u32x4 load_piece(const i8* row, i64 k, i64 K) {
    u32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else if (k < K) {
        u8 b[16];
        for (int i = 0; i < 16; i++) b[i] = k + i < K ? (u8)row[k + i] : (u8)0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

template <class T>
__device__ inline void put(const Mm& p, i64 m, i64 n, int sum, float scale) {
    float v = (float)sum * scale * p.ws[n] + (p.bias ? p.bias[n] : 0.0f);
    if (p.res) v += to_f32(((const T*)p.res)[m * p.ld_res + n]);
    ((T*)p.y)[m * p.ld_y + n] = from_f32<T>(activate<T>(v, p.act));
}

// Rows of both operands at multiples of 16 bytes, k a multiple of 16.  blockIdx.y: which of the `splits` parts of k (whole
// steps each); with more than one the int32 sums go to part[split][m][n] and k_i8_join adds them.
// 8192^3, 256 x 256 tiles: 504 us, 2.2 POP/s of the 2.44 that the library's product reaches; of 804 k cycles the matrix pipe is busy for
// 65 %, LDS for 25 %; a CU's two waves a SIMD spend 30 % at loads and barriers.  86016 x 128 x 1152, 128 x 128 tiles: 27.5 us, 4.4 TB/s of rows
// read and results written, SiLU on the way.  777 x 1003 x 1031, 64 x 64 tiles, 208 workgroups: 7.5 us, one after the other:
// launch, first tiles, 17 steps, residual, stores.
// RES: with a residual, whose values take registers (128 x 128 tile: 96, and 70 without, with which three workgroups a CU fit and not
// two: 86016 x 128 x 1152 29.2 us with one form for both, 27.5 with two; 8192^3 541 and 504).
template <class T, class S, bool RES>
__global__ __launch_bounds__(S::THREADS) void k_i8_mm_tile(Mm p, u32 tiles_m, u32 tiles_n, u32 steps_per_split, int* part) {
    extern __shared__ __attribute__((aligned(128))) u8 lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    u32 tm, tn;
    tile_place(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const i64 m0 = (i64)tm * S::BM, n0 = (i64)tn * S::BN;
    auto span = [](i64 rows, i64 most, i64 ld, i64 k) {   // bytes from the first row on that belong to the operand
        const i64 r = rows < most ? rows : most;
        return (u32)((r - 1) * ld + k);
    };
    const TileSrc<false> a(p.q + m0 * p.ld_q, TILE_KB, (u32)p.ld_q, span(p.m - m0, S::BM, p.ld_q, p.k), lane);
    const TileSrc<S::PAIRS> b(p.w + n0 * p.ld_w, TILE_KB, (u32)p.ld_w, span(p.n - n0, S::BN, p.ld_w, p.k), lane);
    const u32 first = blockIdx.y * steps_per_split;
    u32 kend = (first + steps_per_split) * TILE_KB;
    kend = kend < (u32)p.k ? kend : (u32)p.k;
    // scales of the tile's rows and columns: asked for before the product, which they arrive under, and handed out through LDS
    static_assert(S::THREADS >= S::BM && S::THREADS >= S::BN, "a value a thread");
    const int t = threadIdx.x;
    const float scale_m = p.qs[m0 + t < p.m ? m0 + t : p.m - 1];
    const i64 nt = n0 + t < p.n ? n0 + t : p.n - 1;
    const float scale_n = p.ws[nt], bias_n = p.bias ? p.bias[nt] : 0.0f;
    i32x16 acc[S::FM][S::FN] = {};
    tile_product<KindI8, S>(KindI8(), a, b, first, kend, lds, wave, lane, acc);
    const int wm = wave / S::WN * (S::FM * 32), wn = wave % S::WN * (S::FN * 32);
    const int rows = (int)(p.m - m0 < S::BM ? p.m - m0 : S::BM);
    constexpr int W = S::PAIRS ? 2 : 1;   // neighbouring columns a lane holds
    if (part) {
        part += (i64)blockIdx.y * p.m * p.n;
#pragma unroll
        for (int j = 0; j < S::FN; j += W) {
            const i64 n = n0 + wn + 32 * j + W * (lane & 31);
            if (n >= p.n) continue;
#pragma unroll
            for (int i = 0; i < S::FM; i++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int row = wm + 32 * i + acc_row(r, lane);
                    if (row >= rows) continue;
                    part[(m0 + row) * p.n + n] = acc[i][j][r];
                    if (W == 2 && n + 1 < p.n) part[(m0 + row) * p.n + n + 1] = acc[i][j + W - 1][r];
                }
        }
        return;
    }
    float *sm = (float*)lds, *sn = sm + S::BM, *bn = sn + S::BN;   // its tiles have been read
    if (t < S::BM) sm[t] = scale_m;
    if (t < S::BN) {
        sn[t] = scale_n;
        bn[t] = bias_n;
    }
    __syncthreads();
    auto finish = [&](auto act) {   // a copy for each activation: no branch between the values
#pragma unroll
        for (int j = 0; j < S::FN; j += W) {
            const int c = wn + 32 * j + W * (lane & 31);
            const i64 n = n0 + c;
            const float s0 = sn[c], b0 = bn[c], s1 = sn[c + W - 1], b1 = bn[c + W - 1];
            const bool two = W == 2 && n + 1 < p.n;
            if (n >= p.n) continue;
#pragma unroll
            for (int i = 0; i < S::FM; i++) {
                float res[16][W];
                if constexpr (RES) {   // a block's residuals on their way at once
                    T raw[16][W];
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const i64 m = m0 + wm + 32 * i + acc_row(r, lane);
                        const T* s = (const T*)p.res + (m < p.m ? m : p.m - 1) * p.ld_res + n;
                        raw[r][0] = s[0];
                        if (W == 2) raw[r][W - 1] = s[two ? 1 : 0];
                    }
                    loads_first();
#pragma unroll
                    for (int r = 0; r < 16; r++)
#pragma unroll
                        for (int k = 0; k < W; k++) res[r][k] = to_f32(raw[r][k]);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; r++)
#pragma unroll
                        for (int k = 0; k < W; k++) res[r][k] = -0.0f;   // adds nothing, not even a sign
                }
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int row = wm + 32 * i + acc_row(4 * g, lane);
                    const f32x4 s4 = *(const f32x4*)(sm + row);
                    T* y = (T*)p.y + (m0 + row) * p.ld_y + n;
#pragma unroll
                    for (int e = 0; e < 4; e++, y += p.ld_y) {
                        if (row + e >= rows) break;
                        const int q0 = acc[i][j][4 * g + e], q1 = acc[i][j + W - 1][4 * g + e];
                        float v0 = (float)q0 * s4[e] * s0 + b0 + res[4 * g + e][0], v1 = (float)q1 * s4[e] * s1 + b1 + res[4 * g + e][W - 1];
                        v0 = activate<T>(v0, act);
                        if (two && p.pair_store) {
                            struct __attribute__((aligned(2 * sizeof(T)))) Two { T a, b; };
                            *(Two*)y = Two{from_f32<T>(v0), from_f32<T>(activate<T>(v1, act))};
                        } else {
                            y[0] = from_f32<T>(v0);
                            if (two) y[1] = from_f32<T>(activate<T>(v1, act));
                        }
                    }
                }
            }
        }
    };
    if (p.act == AZ_ACT_SILU) finish(std::integral_constant<int, AZ_ACT_SILU>());
    else if (p.act == AZ_ACT_RELU) finish(std::integral_constant<int, AZ_ACT_RELU>());
    else finish(std::integral_constant<int, AZ_ACT_NONE>());
}
// the parts' sums, and the product's epilogue: 128 x 128 x 4096 in 4 parts, with the tiles, 7.9 us
template <class T>
__global__ __launch_bounds__(256) void k_i8_join(Mm p, u32 splits, const int* __restrict__ part) {
    const i64 total = p.m * p.n;
    for (i64 e = (i64)blockIdx.x * 256 + threadIdx.x; e < total; e += (i64)gridDim.x * 256) {
        int sum = 0;
        for (u32 s = 0; s < splits; s++) sum += part[s * total + e];
        put<T>(p, e / p.n, e % p.n, sum, p.qs[e / p.n]);
    }
}

// Few rows (m <= 16 FM): a workgroup's 8 waves share 16 channels and split k between them, 64 bytes of a row a step, and add
// their int32 sums in LDS.  What bounds it is reading w once: each wave asks for its share of 16 rows, 64 contiguous bytes of
// a row per 4 lanes, with nothing between the loads.  Any alignment.  1 x 4096 x 4096: 5.0 us, 3.4 TB/s of w; 42 x 128 x 1152: 4.6 us
// on 8 workgroups, latency.
constexpr int FEW_WAVES = 8;
template <class T, int FM>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_i8_mm_few(Mm p) {
    __shared__ int sums[FEW_WAVES][FM * 16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, quarter = lane >> 4;
    const i64 n0 = (i64)blockIdx.x * 16, n = n0 + row < p.n ? n0 + row : p.n - 1;   // rows behind the last: the last again
    const i8* w = p.w + n * p.ld_w;
    const i8* q[FM];
#pragma unroll
    for (int f = 0; f < FM; f++) q[f] = p.q + (16 * f + row < p.m ? 16 * f + row : p.m - 1) * p.ld_q;
    i32x4 acc[FM] = {};
    const i64 whole = p.k & ~(i64)63;
    // a step at a time: more waves a CU hide the trips better than several steps' loads at once (us, one | 4 to 8: 42 x 128 x 1152 4.5 |
    // 5.8, 1 x 8192 x 8192 12.5 | 13.1, 64 x 1024 x 1024 5.0 | 7.1)
    for (i64 k = wave * 64; k < whole; k += FEW_WAVES * 64) {
        i32x4 b, a[FM];
        __builtin_memcpy(&b, w + k + quarter * 16, 16);
#pragma unroll
        for (int f = 0; f < FM; f++) __builtin_memcpy(&a[f], q[f] + k + quarter * 16, 16);
#pragma unroll
        for (int f = 0; f < FM; f++) acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[f], b, acc[f], 0, 0, 0);
    }
    if (whole < p.k && wave == (int)(whole / 64 % FEW_WAVES)) {
        const i32x4 b = __builtin_bit_cast(i32x4, load_piece(w, whole + quarter * 16, p.k));
#pragma unroll
        for (int f = 0; f < FM; f++) {
            const i32x4 a = __builtin_bit_cast(i32x4, load_piece(q[f], whole + quarter * 16, p.k));
            acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc[f], 0, 0, 0);
        }
    }
    // 16x16 result: lane holds column (channel) lane & 15 and rows 4 (lane >> 4) + r
#pragma unroll
    for (int f = 0; f < FM; f++)
#pragma unroll
        for (int r = 0; r < 4; r++) sums[wave][16 * f + 4 * quarter + r][row] = acc[f][r];
    __syncthreads();
    for (int e = threadIdx.x; e < FM * 256; e += 64 * FEW_WAVES) {
        const int m = e >> 4, c = e & 15;
        if (m >= p.m || n0 + c >= p.n) continue;
        int sum = 0;
#pragma unroll
        for (int i = 0; i < FEW_WAVES; i++) sum += sums[i][m][c];
        put<T>(p, m, n0 + c, sum, p.qs[m]);
    }
}

// A linear layer on one or two rows of up to 16384: k_i8_mm_few with the rows quantised by every workgroup for itself (they are small
// beside its 16 rows of w, which it asks for first), instead of a launch that the other waits for (us, one launch | two:
// 1 x 4096 x 4096 6.9 | 8.8, 2 x 4096 x 4096 7.8 | 8.9, 1 x 4096 x 16384 19.1 | 21.3, 1 x 128 x 1152 4.8 | 6.7; four rows 10.9 | 9.7).
constexpr int LIN_ROWS = 2, LIN_AHEAD = 8, LIN_LDS = 16 * 1024;
template <class T>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_i8_linear_few(Mm p, const T* __restrict__ x, i64 ld_x) {
    extern __shared__ __attribute__((aligned(16))) u8 lds[];   // m rows of kp integers
    __shared__ u32 part[LIN_ROWS][FEW_WAVES];
    __shared__ int sums[FEW_WAVES][LIN_ROWS][17];
    constexpr int EPP = Piece<T>::EPP, THREADS = 64 * FEW_WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 15, quarter = lane >> 4, m = (int)p.m;
    const i64 n0 = (i64)blockIdx.x * 16, n = n0 + row < p.n ? n0 + row : p.n - 1;
    const i8* w = p.w + n * p.ld_w;
    const i64 whole = p.k & ~(i64)63;
    const int k = (int)p.k, kp = (k + 63) & ~63, pieces = (k + EPP - 1) / EPP;
    i32x4 b[LIN_AHEAD];
#pragma unroll
    for (int i = 0; i < LIN_AHEAD; i++) {   // steps that are not there: the row's beginning again (k >= 64 or nothing is loaded)
        const i64 at = (wave + i * FEW_WAVES) * 64;
        b[i] = i32x4{0, 0, 0, 0};
        if (whole) __builtin_memcpy(&b[i], w + (at < whole ? at : 0) + quarter * 16, 16);
    }
    u32 mx[LIN_ROWS];
#pragma unroll
    for (int r = 0; r < LIN_ROWS; r++) {
        mx[r] = 0;
        if (r < m)
            for (int i = tid; i < pieces; i += THREADS) {
                Piece<T> v;
                v.load(x + r * ld_x + (i64)i * EPP, k - i * EPP < EPP ? k - i * EPP : EPP);
                const u32 t = v.most();
                mx[r] = t > mx[r] ? t : mx[r];
            }
        mx[r] = lanes_max<64>(mx[r]);
        if (lane == 0) part[r][wave] = mx[r];
    }
    __syncthreads();
    float s[LIN_ROWS];
#pragma unroll
    for (int r = 0; r < LIN_ROWS; r++) {
#pragma unroll
        for (int i = 0; i < FEW_WAVES; i++) mx[r] = part[r][i] > mx[r] ? part[r][i] : mx[r];
        s[r] = row_scale(mx[r]);
        if (r >= m) continue;
        const float rs = 1.0f / s[r];
        for (int i = tid; i < kp / EPP; i += THREADS) {   // zeros behind the row
            u32 out[EPP / 4] = {};
            if (i < pieces && s[r] > 0) {
                Piece<T> v;
                v.load(x + r * ld_x + (i64)i * EPP, k - i * EPP < EPP ? k - i * EPP : EPP);
                if (!(s[r] >= QUANT_TINY && v.quantize(rs, out))) v.quantize_exact(s[r], rs, out);
            }
            __builtin_memcpy(lds + r * kp + i * EPP, out, EPP);
        }
    }
    __syncthreads();
    const u8* q = lds + (row < m ? row : m - 1) * kp + quarter * 16;
    i32x4 acc = {};
#pragma unroll
    for (int i = 0; i < LIN_AHEAD; i++) {
        const i64 at = (wave + i * FEW_WAVES) * 64;
        if (at < whole) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(q + at), b[i], acc, 0, 0, 0);
    }
    for (i64 at = (wave + LIN_AHEAD * FEW_WAVES) * 64; at < whole; at += FEW_WAVES * 64) {
        i32x4 v;
        __builtin_memcpy(&v, w + at + quarter * 16, 16);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(q + at), v, acc, 0, 0, 0);
    }
    if (whole < p.k && wave == (int)(whole / 64 % FEW_WAVES))
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*(const i32x4*)(q + whole),
                                                    __builtin_bit_cast(i32x4, load_piece(w, whole + quarter * 16, p.k)), acc, 0, 0, 0);
    if (quarter == 0)   // rows 4 quarter + r
#pragma unroll
        for (int r = 0; r < LIN_ROWS; r++) sums[wave][r][row] = acc[r];
    __syncthreads();
    if (tid < LIN_ROWS * 16) {
        const int r = tid >> 4, c = tid & 15;
        if (r >= m || n0 + c >= p.n) return;
        int sum = 0;
#pragma unroll
        for (int i = 0; i < FEW_WAVES; i++) sum += sums[i][r][c];
        put<T>(p, r, n0 + c, sum, r ? s[1] : s[0]);
    }
}

// Rows of k bytes at any address -> rows of kp (a multiple of 16) with zeros behind k.  16 output bytes a thread; blockIdx.y: which
// operand.  (777 + 1003) x 1031: 4.4 us, a launch and one trip to memory.
struct Align {
    const i8* src[2];
    i64 ld[2], rows[2];
    i8* dst[2];
};
__global__ __launch_bounds__(256) void k_i8_align(Align a, i64 k, i64 kp) {
    const i8* src = blockIdx.y ? a.src[1] : a.src[0];
    i8* dst = blockIdx.y ? a.dst[1] : a.dst[0];
    const i64 ld = blockIdx.y ? a.ld[1] : a.ld[0], rows = blockIdx.y ? a.rows[1] : a.rows[0];
    const i64 pieces = kp / 16, total = rows * pieces;
    for (i64 e = (i64)blockIdx.x * 256 + threadIdx.x; e < total; e += (i64)gridDim.x * 256) {
        const i64 r = e / pieces, c = (e - r * pieces) * 16;
        *(u32x4*)(dst + r * kp + c) = load_piece(src + r * ld, c, k);
    }
}

static bool pairs_ok(const void* y, i64 ld_y, int dtype) { return ld_y % 2 == 0 && (uintptr_t)y % (2 * dtype_size(dtype)) == 0; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
static i64 up(i64 n, i64 to) { return (n + to - 1) / to * to; }

// When k_i8_mm_few takes a product of up to 64 rows.  It reads q from L2 once for every 16 channels, the tiles once for every 64, and
// splits k over 8 waves only, the tiles over 16 workgroups; but it is one launch and takes rows at any address, which the tiles
// need copied first (us, few | tiles: 1 x 4096 x 4096 5.3 | 7.7, 1 x 8192 x 8192 12.4 | 14.7, 8 x 8192 x 8192 14.4 | 15.3, 16 x 4096 x 4096
// 6.3 | 8.5, 16 x 4096 x 8192 9.8 | 11.0, 16 x 8192 x 8192 17.2 | 15.5, 16 x 128 x 16384 15.9 | 10.2, 32 x 4096 x 4096 8.3 | 9.1,
// 32 x 1024 x 4096 7.7 | 8.1, 24 x 512 x 8192 11.4 | 9.0, 32 x 8192 x 8192 24.9 | 16.2, 42 x 128 x 1152 4.5 | 5.2, 48 x 4096 x 1024 4.7 | 5.1,
// 48 x 1024 x 4096 9.6 | 8.3, 64 x 2048 x 2048 7.2 | 7.1, 64 x 4096 x 4096 12.3 | 10.2).
static bool few_rows(i64 m, i64 n, i64 k, bool aligned) {
    if (m > 64) return false;
    if (!aligned) return true;
    if (m <= 16) return k <= 8192 && (m <= 8 || n * k <= 32 << 20);
    return m <= 32 ? k <= 4096 && n * k <= 16 << 20 : k <= 2048 && n * k <= 4 << 20;
}
constexpr i64 TILE_MAX_LD = 1 << 22;  // row distance up to which a tile's addresses fit 32 bits

using Tile256 = TileShape<256, 256, 2, 4, 4, 1>;   // 128 KB; 128 x 64 a wave: 6 operand reads for 8 MFMAs
using Tile128 = TileShape<128, 128, 4, 2, 3, 1>;   // 48 KB: three workgroups a CU (two with a residual), whose stores run under each other's loads
using Tile64 = TileShape<64, 64, 2, 2, 3, 2>;      // few tiles: what counts is the way from step to step, so a barrier every two

// How a product is computed; a function of the sizes and alignments alone, so that the workspace can be asked for first.
struct MmPlan {
    int tile;            // 0: few rows; 64, 128, 256: tile edge
    bool align_q, align_w;
    u32 splits, steps_per_split;
    i64 kp;              // row length of aligned copies
    size_t q_bytes, w_bytes, part_bytes;
    size_t total() const { return q_bytes + w_bytes + part_bytes; }
};
// q_padded: q is the workspace of a linear call, aligned and with zeros behind its rows.
static MmPlan mm_plan(i64 m, i64 n, i64 k, const void* q, i64 ld_q, bool q_padded, const void* w, i64 ld_w) {
    MmPlan P = {};
    P.splits = 1;
    P.kp = up(k, 16);
    if (few_rows(m, n, k, ((uintptr_t)w & 15) == 0 && (ld_w & 15) == 0)) return P;
    // The loads into LDS move 16 aligned bytes; rows whose length is no multiple of 16 need zeros behind them in one operand: q's.
    // (Of w the 16 aligned bytes that hold a row's last ones are read whole: never past what was allocated with them.)
    P.align_q = !q_padded && (((uintptr_t)q & 15) || (ld_q & 15) || (k & 15) || ld_q > TILE_MAX_LD);
    P.align_w = ((uintptr_t)w & 15) || (ld_w & 15) || ld_w > TILE_MAX_LD;
    P.q_bytes = P.align_q ? up256((size_t)m * P.kp) : 0;
    P.w_bytes = P.align_w ? up256((size_t)n * P.kp) : 0;
    auto tiles = [&](i64 e) { return ((m + e - 1) / e) * ((n + e - 1) / e); };
    // A larger tile reads less per product, but must not be mostly padding and must fill the chip: at least 200 of them (us; with
    // 400 or 100 instead: 2048^3 15.3 | 19.3 with 400, 3000 x 3000 x 512 15.8 | 20.9 with 100).
    auto pays = [&](i64 e) { return tiles(e) >= 200 && tiles(e) * e * e <= tiles(e / 2) * (e / 2) * (e / 2) * 9 / 8; };
    P.tile = pays(256) ? 256 : pays(128) ? 128 : 64;
    // k split over workgroups where the tiles are too few for the CUs, from 64 steps on, in parts of at least 16 (us, split | not:
    // 65 x 64 x 8192 8.9 | 15.6, 128 x 128 x 4096 7.9 | 9.6, 70 x 1000 x 4096 8.4 | 9.7, 65 x 64 x 3200 8.1 | 8.0, 256 x 256 x 2048 7.6 | 6.6)
    const u32 steps = (u32)((k + TILE_KB - 1) / TILE_KB);
    u32 splits = 1;
    if (P.tile == 64 && steps >= 64)
        while (splits < 16 && tiles(64) * splits * 2 <= 256 && steps / (splits * 2) >= 16) splits *= 2;
    P.steps_per_split = (steps + splits - 1) / splits;
    P.splits = (steps + P.steps_per_split - 1) / P.steps_per_split;
    P.part_bytes = P.splits > 1 ? up256((size_t)P.splits * m * n * 4) : 0;
    return P;
}

template <class T, class S>
static int launch_tile(const Mm& p, const MmPlan& P, int* part, hipStream_t st) {
    const i64 tm = (p.m + S::BM - 1) / S::BM, tn = (p.n + S::BN - 1) / S::BN;
    if (tm * tn > 0x7fffffff) return refuse("az_i8_matmul: more than 2^31 tiles");
    const dim3 grid((u32)(tm * tn), P.splits), block(S::THREADS);
    if (p.res && !part) k_i8_mm_tile<T, S, true><<<grid, block, S::LDS, st>>>(p, (u32)tm, (u32)tn, P.steps_per_split, part);
    else k_i8_mm_tile<T, S, false><<<grid, block, S::LDS, st>>>(p, (u32)tm, (u32)tn, P.steps_per_split, part);
    if (part) {
        const i64 blocks = (p.m * p.n + 255) / 256;
        k_i8_join<T><<<dim3((u32)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st>>>(p, P.splits, part);
    }
    return launch_status("az_i8_matmul");
}

template <class T>
static int mm_launch(Mm p, const MmPlan& P, char* ws, hipStream_t st) {
    if (P.tile == 0) {
        const i64 blocks = (p.n + 15) / 16;
        if (blocks > 0x7fffffff) return refuse("az_i8_matmul: more than 2^31 tiles");
        const dim3 grid((u32)blocks), block(64 * FEW_WAVES);
        if (p.m <= 16) k_i8_mm_few<T, 1><<<grid, block, 0, st>>>(p);
        else if (p.m <= 32) k_i8_mm_few<T, 2><<<grid, block, 0, st>>>(p);
        else if (p.m <= 48) k_i8_mm_few<T, 3><<<grid, block, 0, st>>>(p);
        else k_i8_mm_few<T, 4><<<grid, block, 0, st>>>(p);
        return launch_status("az_i8_matmul");
    }
    if (P.align_q || P.align_w) {
        Align a = {};
        int n = 0;
        i64 most = 0;
        auto add = [&](const i8*& src, i64& ld, i64 rows, char* dst) {
            a.src[n] = src;
            a.ld[n] = ld;
            a.rows[n] = rows;
            a.dst[n] = (i8*)dst;
            src = (const i8*)dst;
            ld = P.kp;
            most = rows > most ? rows : most;
            n++;
        };
        if (P.align_q) add(p.q, p.ld_q, p.m, ws);
        if (P.align_w) add(p.w, p.ld_w, p.n, ws + P.q_bytes);
        const i64 blocks = (most * (P.kp / 16) + 255) / 256;
        k_i8_align<<<dim3((u32)(blocks < 8192 ? blocks : 8192), n), dim3(256), 0, st>>>(a, p.k, P.kp);
    }
    p.k = P.kp;   // from here on with the zeros (of one operand at least) behind the end
    int* part = P.splits > 1 ? (int*)(ws + P.q_bytes + P.w_bytes) : nullptr;
    if (P.tile == 256) return launch_tile<T, Tile256>(p, P, part, st);
    if (P.tile == 128) return launch_tile<T, Tile128>(p, P, part, st);
    return launch_tile<T, Tile64>(p, P, part, st);
}

static int i8_matmul(const Mm& p, bool q_padded, int dtype, void* ws, hipStream_t st) {
    const MmPlan P = mm_plan(p.m, p.n, p.k, p.q, p.ld_q, q_padded, p.w, p.ld_w);
    AZ_DISPATCH_DTYPE(dtype, return mm_launch<T>(p, P, (char*)ws, st));
    return AZ_OK;
}

template <class T, int LANES, int NP, bool FAST>
static void rows_go(const Rows& R, hipStream_t st) {
    const i64 b = (R.rows + 256 / LANES - 1) / (256 / LANES);
    k_i8_quantize<T, LANES, NP, FAST><<<dim3((u32)(b < 1 << 20 ? b : 1 << 20)), dim3(256), 0, st>>>(R);
}
// Few lanes to a row waste the fewest on its end and on its reduction; with few rows it takes more lanes to fill the chip (us, 16 lanes
// | 64: 300 fp16 values, 16384 rows 8.1 | 10.0, 8192 rows 7.3 | 6.7; 1152 values, 65536 rows 41.3 | 42.8, 16384 rows 17.3 | 15.1).  Longer
// rows than the forms' 144 and 256 pieces go to 256 lanes, whose reduction takes two barriers (86016 rows of 1152 float32, 288 pieces:
// 85 us for a floor of 29; no form between has been tried).
template <class T, bool FAST>
static void rows_dispatch(const Rows& R, hipStream_t st) {
    const u32 P = R.pieces;
    if (P <= 4) rows_go<T, 4, 1, FAST>(R, st);
    else if (P <= 16) rows_go<T, 16, 1, FAST>(R, st);
    else if (P <= 64 && R.rows >= 16384) rows_go<T, 16, 4, FAST>(R, st);
    else if (P > 64 && P <= 144 && R.rows >= 32768) rows_go<T, 16, 9, FAST>(R, st);
    else if (P <= 64) rows_go<T, 64, 1, FAST>(R, st);
    else if (P <= 256) rows_go<T, 64, 4, FAST>(R, st);
    else if (P <= 512) rows_go<T, 256, 2, FAST>(R, st);
    else if (P <= 2048) rows_go<T, 256, 8, FAST>(R, st);
    else k_i8_quantize_long<T><<<dim3((u32)(R.rows < 1 << 20 ? R.rows : 1 << 20)), dim3(256), 0, st>>>(R);
}
template <class T>
static int rows_launch(Rows R, hipStream_t st) {
    const i64 per = (R.cols + Piece<T>::EPP - 1) / Piece<T>::EPP;
    if (per * R.taps > 0x7fffffff) return refuse("az_i8_quantize: rows too long");
    R.per_tap = (u32)per;
    R.pieces = (u32)(per * R.taps);
    R.magic = per > 1 && (u64)R.pieces * (u64)per < (u64)1 << 32 ? (u32)(((u64)1 << 32) / (u64)per + 1) : 0;
    R.inv_tap = 1.0f / (float)per;
    const bool small = R.ld_x < 1 << 22 && R.n_src < 1 << 24 && R.n_src > 0;
    const i64 row = small ? R.ld_x * (i64)sizeof(T) : 0;
    const bool fast = small && R.cols % Piece<T>::EPP == 0 && ((uintptr_t)R.x & 15) == 0 && row % 16 == 0 && R.n_src * row < 0x7ffffff0;
    R.row_bytes = (u32)row;
    R.x_bytes = fast ? (u32)((R.n_src - 1) * row + R.cols * (i64)sizeof(T)) : 0;
    if (fast) rows_dispatch<T, true>(R, st);
    else rows_dispatch<T, false>(R, st);
    return launch_status("az_i8_quantize");
}
static int i8_quantize(int dtype, i64 rows, i64 cols, const void* x, i64 ld_x, i64 n_src, const i32* index, int taps, i8* q,
                       i64 ld_q, bool fill, float* scale, hipStream_t st) {
    Rows R = {};
    R.rows = rows;
    R.cols = cols;
    R.ld_x = ld_x;
    R.n_src = n_src;
    R.ld_q = ld_q;
    R.x = x;
    R.index = index;
    R.q = q;
    R.scale = scale;
    R.taps = (u32)taps;
    R.fill = fill;
    AZ_DISPATCH_DTYPE(dtype, return rows_launch<T>(R, st));
    return AZ_OK;
}

static i64 linear_pitch(i64 k) { return (k + 15) & ~(i64)15; }

}  // namespace az

using namespace az;

extern "C" {

int az_i8_quantize_dev(int device, int dtype, int64_t rows, int64_t cols, const void* x_dev, int64_t ld_x, int64_t n_src,
                       const int32_t* index_dev, int32_t taps, int8_t* q_dev, int64_t ld_q, float* scale_dev,
                       void* stream) {
    if (!dtype_ok(dtype)) return refuse("az_i8_quantize: unknown dtype");
    if (rows < 0 || cols < 1 || n_src < 0 || ld_x < cols) return refuse("az_i8_quantize: bad shape or row distance");
    if (!index_dev && (taps != 1 || n_src != rows)) return refuse("az_i8_quantize: without an index taps is 1 and n_src is rows");
    if (taps < 1 || cols > 0x7fffffff / taps || ld_x > (i64)1 << 40 || ld_q < taps * cols || ld_q > (i64)1 << 40)
        return refuse("az_i8_quantize: bad taps or ld_q");
    if (rows == 0) {
        DeviceScope dev(device);
        return dev.rc;
    }
    if ((!x_dev && n_src > 0) || !q_dev || !scale_dev) return refuse("az_i8_quantize: null pointer");
    const i64 es = (i64)dtype_size(dtype);
    const Span x = {x_dev, n_src, cols * es, ld_x * es}, q = {q_dev, rows, (i64)taps * cols, ld_q}, s = {scale_dev, rows, 4, 4};
    const Span at = {index_dev, rows, taps * (i64)4, taps * (i64)4};
    if (overlap(q, x) || overlap(q, s) || overlap(x, s) || overlap(q, at) || overlap(s, at))
        return refuse("az_i8_quantize: q and scale must not overlap an input or each other");
    DeviceScope dev(device);
    if (dev.rc != AZ_OK) return dev.rc;
    return i8_quantize(dtype, rows, cols, x_dev, ld_x, n_src, index_dev, taps, q_dev, ld_q, false, scale_dev, (hipStream_t)stream);
}

static int mm_check(int64_t m, int64_t n, int64_t k, int64_t ld_x, int64_t ld_w, const void* res, int64_t ld_res, int act,
                    int dtype, int64_t ld_y) {
    if (!dtype_ok(dtype)) return refuse("az_i8_matmul: unknown dtype");
    if (m < 0 || n < 0 || k < 1 || k > I8_MAX_K || m > 0x7fffffff || n > 0x7fffffff)
        return refuse("az_i8_matmul: bad shape (k is 1..131071)");
    const i64 most = (i64)1 << 40;
    if (ld_x < k || ld_w < k || ld_y < n || (res && ld_res < n) || ld_x > most || ld_w > most || ld_y > most || (res && ld_res > most))
        return refuse("az_i8_matmul: bad row distance");
    if (act < AZ_ACT_NONE || act > AZ_ACT_SILU) return refuse("az_i8_matmul: unknown activation");
    return AZ_OK;
}

// y may be the residual itself (each element is read by the thread that writes it, before that); nothing else may be written
static int y_check(const void* y, i64 m, i64 n, i64 ld_y, int dtype, const Span& x, const float* x_scale, const i8* w, i64 k, i64 ld_w,
                   const float* w_scale, const float* bias, const void* res, i64 ld_res) {
    const i64 es = (i64)dtype_size(dtype);
    const Span out = {y, m, n * es, ld_y * es};
    const Span in[] = {x, {x_scale, 1, m * 4, m * 4}, {w, n, k, ld_w}, {w_scale, 1, n * 4, n * 4}, {bias, 1, n * 4, n * 4}};
    for (const Span& s : in)
        if (overlap(out, s)) return refuse("az_i8_matmul: the output must not overlap an input");
    const bool itself = res == y && (ld_res == ld_y || m == 1);
    if (!itself && overlap(out, Span{res, m, n * es, ld_res * es}))
        return refuse("az_i8_matmul: the output must be the residual or not overlap it");
    return AZ_OK;
}

size_t az_i8_matmul_ws(int64_t m, int64_t n, int64_t k, const int8_t* q_dev, int64_t ld_q, const int8_t* w_dev, int64_t ld_w) {
    if (m < 1 || n < 1 || k < 1 || k > I8_MAX_K || m > 0x7fffffff || n > 0x7fffffff) return 0;
    return mm_plan(m, n, k, q_dev, ld_q, false, w_dev, ld_w).total();
}

int az_i8_matmul_dev(int device, int64_t m, int64_t n, int64_t k, const int8_t* q_dev, int64_t ld_q,
                     const float* q_scale_dev, const int8_t* w_dev, int64_t ld_w, const float* w_scale_dev,
                     const float* bias_dev, const void* residual_dev, int64_t ld_res, int act, int dtype, void* y_dev,
                     int64_t ld_y, void* ws_dev, size_t ws_bytes, void* stream) {
    const int rc = mm_check(m, n, k, ld_q, ld_w, residual_dev, ld_res, act, dtype, ld_y);
    if (rc != AZ_OK) return rc;
    const size_t need = az_i8_matmul_ws(m, n, k, q_dev, ld_q, w_dev, ld_w);
    if (ws_bytes < need || (need && (!ws_dev || ((uintptr_t)ws_dev & 255))))
        return refuse("az_i8_matmul: workspace too small or not aligned to 256 bytes");
    if (m > 0 && n > 0 && (!q_dev || !q_scale_dev || !w_dev || !w_scale_dev || !y_dev))
        return refuse("az_i8_matmul: null pointer");
    const int ok = y_check(y_dev, m, n, ld_y, dtype, Span{q_dev, m, k, ld_q}, q_scale_dev, w_dev, k, ld_w, w_scale_dev, bias_dev,
                           residual_dev, ld_res);
    if (ok != AZ_OK) return ok;
    DeviceScope dev(device);
    if (dev.rc != AZ_OK || m == 0 || n == 0) return dev.rc;
    const Mm p = {m, n, k, q_dev, w_dev, ld_q, ld_w, q_scale_dev, w_scale_dev, bias_dev, residual_dev, ld_res, y_dev, ld_y, act, pairs_ok(y_dev, ld_y, dtype)};
    return i8_matmul(p, false, dtype, ws_dev, (hipStream_t)stream);
}

static bool linear_fused(i64 m, i64 k) { return m <= LIN_ROWS && m * up(k, 64) <= LIN_LDS; }

size_t az_i8_linear_ws(int64_t m, int64_t n, int64_t k, const int8_t* w_dev, int64_t ld_w) {
    if (m < 1 || n < 1 || k < 1 || k > I8_MAX_K || m > 0x7fffffff || n > 0x7fffffff || linear_fused(m, k)) return 0;
    return up256((size_t)m * linear_pitch(k)) + up256((size_t)m * 4) +
           mm_plan(m, n, k, nullptr, linear_pitch(k), true, w_dev, ld_w).total();
}

int az_i8_linear_dev(int device, int64_t m, int64_t n, int64_t k, const void* x_dev, int64_t ld_x, const int8_t* w_dev,
                     int64_t ld_w, const float* w_scale_dev, const float* bias_dev, const void* residual_dev,
                     int64_t ld_res, int act, int dtype, void* y_dev, int64_t ld_y, void* ws_dev, size_t ws_bytes,
                     void* stream) {
    int rc = mm_check(m, n, k, ld_x, ld_w, residual_dev, ld_res, act, dtype, ld_y);
    if (rc != AZ_OK) return rc;
    const size_t need = az_i8_linear_ws(m, n, k, w_dev, ld_w);
    if (ws_bytes < need || (need && (!ws_dev || ((uintptr_t)ws_dev & 255))))
        return refuse("az_i8_linear: workspace too small or not aligned to 256 bytes");
    if (m > 0 && n > 0 && (!x_dev || !w_dev || !w_scale_dev || !y_dev)) return refuse("az_i8_linear: null pointer");
    const i64 es = (i64)dtype_size(dtype);
    rc = y_check(y_dev, m, n, ld_y, dtype, Span{x_dev, m, k * es, ld_x * es}, nullptr, w_dev, k, ld_w, w_scale_dev, bias_dev, residual_dev,
                 ld_res);
    if (rc != AZ_OK) return rc;
    DeviceScope dev(device);
    if (dev.rc != AZ_OK || m == 0 || n == 0) return dev.rc;
    hipStream_t st = (hipStream_t)stream;
    if (linear_fused(m, k)) {
        const Mm p = {m, n, k, nullptr, w_dev, 0, ld_w, nullptr, w_scale_dev, bias_dev, residual_dev, ld_res, y_dev, ld_y, act, false};
        const i64 blocks = (n + 15) / 16;
        if (blocks > 0x7fffffff) return refuse("az_i8_linear: more than 2^31 tiles");
        AZ_DISPATCH_DTYPE(dtype, k_i8_linear_few<T><<<dim3((u32)blocks), dim3(64 * FEW_WAVES), (size_t)(m * up(k, 64)), st>>>(
                                     p, (const T*)x_dev, ld_x));
        return launch_status("az_i8_linear");
    }
    i8* q = (i8*)ws_dev;
    float* qs = (float*)((char*)ws_dev + up256((size_t)m * linear_pitch(k)));
    char* rest = (char*)qs + up256((size_t)m * 4);
    rc = i8_quantize(dtype, m, k, x_dev, ld_x, m, nullptr, 1, q, linear_pitch(k), true, qs, st);
    if (rc != AZ_OK) return rc;
    const Mm p = {m, n, k, q, w_dev, linear_pitch(k), ld_w, qs, w_scale_dev, bias_dev, residual_dev, ld_res, y_dev, ld_y, act, pairs_ok(y_dev, ld_y, dtype)};
    return i8_matmul(p, true, dtype, rest, st);
}

}  // extern "C"
