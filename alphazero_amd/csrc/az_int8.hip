// az_int8.hip -- evaluation of layers in 8-bit integers: rows quantised with a scale each, products with a scale for each
// row (token) and each output channel.
//
//   q[r][c] = rint(x[r][c] / s[r]),  s[r] = max|x[r]| * (1/127)     y[m][n] = act(s[m] ws[n] sum_k q[m][k] w[n][k] + b[n] + res)
//
// The sums are int32 and exact (|q w| <= 2^14, k <= 131071), so no order of summation changes a result.
#include <math.h>

#include "az_ops.hpp"

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

template <class T>
__global__ __launch_bounds__(256) void k_i8_quantize(i64 rows, i64 cols, const T* __restrict__ x, i64 ld_x, i64 n_src,
                                                     const i32* __restrict__ index, int taps, i8* __restrict__ q, i64 ld_q,
                                                     float* __restrict__ scale) {
    __shared__ u32 part[4];
    for (i64 r = blockIdx.x; r < rows; r += gridDim.x) {
        // largest magnitude as bits: an unsigned maximum of |x| keeps a NaN on top (fmaxf would drop it)
        u32 mx = 0;
        for (int t = 0; t < taps; t++) {
            const i64 src = index ? (i64)index[r * taps + t] : r;
            if (src < 0 || src >= n_src) continue;
            for (i64 c = threadIdx.x; c < cols; c += 256) {
                const u32 b = __builtin_bit_cast(u32, to_f32(x[src * ld_x + c])) & 0x7fffffffu;
                mx = b > mx ? b : mx;
            }
        }
        for (int o = 32; o; o >>= 1) {
            const u32 b = (u32)__shfl_xor((int)mx, o);
            mx = b > mx ? b : mx;
        }
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
        __syncthreads();
        for (int i = 0; i < 4; i++) mx = part[i] > mx ? part[i] : mx;
        __syncthreads();
        const float s = row_scale(mx);
        if (threadIdx.x == 0) scale[r] = s;
        const float rs = 1.0f / s;
        for (int t = 0; t < taps; t++) {
            const i64 src = index ? (i64)index[r * taps + t] : r;
            const bool real = src >= 0 && src < n_src && s > 0;
            for (i64 c = threadIdx.x; c < cols; c += 256) {
                int v = 0;
                if (real) {
                    const float f = to_f32(x[src * ld_x + c]);
                    v = s >= QUANT_TINY ? quant1(f, s, rs) : quant1_tiny(f, s);
                }
                q[r * ld_q + t * cols + c] = (i8)v;
            }
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
};

__device__ inline float activate(float v, int act) {
    if (act == AZ_ACT_RELU) return v > 0 || v != v ? v : 0.0f;
    if (act == AZ_ACT_SILU) return v / (1.0f + expf(-v));
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

// 64 x 64 outputs per workgroup, 4 waves of 32 x 32, any alignment
template <class T>
__global__ __launch_bounds__(256) void k_i8_mm_any(Mm p) {
    __shared__ __attribute__((aligned(16))) u8 ta[64 * TILE_KB], tb[64 * TILE_KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const i64 tiles_n = (p.n + 63) / 64;
    const i64 m0 = (i64)blockIdx.x / tiles_n * 64, n0 = (i64)blockIdx.x % tiles_n * 64;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    i32x16 acc = {};
    for (i64 k0 = 0; k0 < p.k; k0 += TILE_KB) {
        for (int i = 0; i < 2; i++) {
            const int row = (tid >> 3) + 32 * i, piece = tid & 7;
            const u32x4 zero = {0, 0, 0, 0};
            const u32x4 a = m0 + row < p.m ? load_piece(p.q + (m0 + row) * p.ld_q, k0 + piece * 16, p.k) : zero;
            const u32x4 b = n0 + row < p.n ? load_piece(p.w + (n0 + row) * p.ld_w, k0 + piece * 16, p.k) : zero;
            *(u32x4*)(ta + tile_off(row, piece)) = a;
            *(u32x4*)(tb + tile_off(row, piece)) = b;
        }
        __syncthreads();
        for (int ks = 0; ks < 4; ks++) {
            const int piece = 2 * ks + (lane >> 5);
            const i32x4 a = *(const i32x4*)(ta + tile_off(wm + (lane & 31), piece));
            const i32x4 b = *(const i32x4*)(tb + tile_off(wn + (lane & 31), piece));
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, acc, 0, 0, 0);
        }
        __syncthreads();
    }
    const i64 n = n0 + wn + (lane & 31);
    if (n >= p.n) return;
    const float sw = p.ws[n], bias = p.bias ? p.bias[n] : 0.0f;
    for (int r = 0; r < 16; r++) {
        const i64 m = m0 + wm + acc_row(r, lane);
        if (m >= p.m) continue;
        float v = (float)acc[r] * p.qs[m] * sw + bias;
        if (p.res) v += to_f32(((const T*)p.res)[m * p.ld_res + n]);
        ((T*)p.y)[m * p.ld_y + n] = from_f32<T>(activate(v, p.act));
    }
}

static int i8_matmul(const Mm& p, int dtype, void* ws, size_t ws_bytes, hipStream_t st) {
    const i64 tiles = ((p.m + 63) / 64) * ((p.n + 63) / 64);
    if (tiles > 0x7fffffff) return refuse("az_i8_matmul: more than 2^31 tiles");
    AZ_DISPATCH_DTYPE(dtype, k_i8_mm_any<T><<<dim3((u32)tiles), dim3(256), 0, st>>>(p));
    return launch_status("az_i8_matmul");
}

static int i8_quantize(int dtype, i64 rows, i64 cols, const void* x, i64 ld_x, i64 n_src, const i32* index, int taps, i8* q,
                       i64 ld_q, float* scale, hipStream_t st) {
    const u32 grid = (u32)(rows < 65536 ? rows : 65536);
    AZ_DISPATCH_DTYPE(dtype, k_i8_quantize<T><<<dim3(grid), dim3(256), 0, st>>>(rows, cols, (const T*)x, ld_x, n_src, index,
                                                                             taps, q, ld_q, scale));
    return launch_status("az_i8_quantize");
}

static i64 linear_pitch(i64 k) { return (k + 15) & ~(i64)15; }
static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace az

using namespace az;

extern "C" {

int az_i8_quantize_dev(int device, int dtype, int64_t rows, int64_t cols, const void* x_dev, int64_t ld_x, int64_t n_src,
                       const int32_t* index_dev, int32_t taps, int8_t* q_dev, int64_t ld_q, float* scale_dev,
                       void* stream) {
    if (!dtype_ok(dtype)) return refuse("az_i8_quantize: unknown dtype");
    if (rows < 0 || cols < 1 || n_src < 0 || ld_x < cols) return refuse("az_i8_quantize: bad shape or row distance");
    if (!index_dev && (taps != 1 || n_src != rows)) return refuse("az_i8_quantize: without an index taps is 1 and n_src is rows");
    if (taps < 1 || cols > 0x7fffffff / taps || ld_q < taps * cols) return refuse("az_i8_quantize: bad taps or ld_q");
    if (rows == 0) {
        DeviceScope dev(device);
        return dev.rc;
    }
    if ((!x_dev && n_src > 0) || !q_dev || !scale_dev) return refuse("az_i8_quantize: null pointer");
    DeviceScope dev(device);
    if (dev.rc != AZ_OK) return dev.rc;
    return i8_quantize(dtype, rows, cols, x_dev, ld_x, n_src, index_dev, taps, q_dev, ld_q, scale_dev, (hipStream_t)stream);
}

static int mm_check(int64_t m, int64_t n, int64_t k, int64_t ld_x, int64_t ld_w, const void* res, int64_t ld_res, int act,
                    int dtype, int64_t ld_y) {
    if (!dtype_ok(dtype)) return refuse("az_i8_matmul: unknown dtype");
    if (m < 0 || n < 0 || k < 1 || k > I8_MAX_K || m > (i64)1 << 40 || n > (i64)1 << 40)
        return refuse("az_i8_matmul: bad shape (k is 1..131071)");
    if (ld_x < k || ld_w < k || ld_y < n || (res && ld_res < n)) return refuse("az_i8_matmul: bad row distance");
    if (act < AZ_ACT_NONE || act > AZ_ACT_SILU) return refuse("az_i8_matmul: unknown activation");
    return AZ_OK;
}

size_t az_i8_matmul_ws(int64_t m, int64_t n, int64_t k) { return 0; }

int az_i8_matmul_dev(int device, int64_t m, int64_t n, int64_t k, const int8_t* q_dev, int64_t ld_q,
                     const float* q_scale_dev, const int8_t* w_dev, int64_t ld_w, const float* w_scale_dev,
                     const float* bias_dev, const void* residual_dev, int64_t ld_res, int act, int dtype, void* y_dev,
                     int64_t ld_y, void* ws_dev, size_t ws_bytes, void* stream) {
    const int rc = mm_check(m, n, k, ld_q, ld_w, residual_dev, ld_res, act, dtype, ld_y);
    if (rc != AZ_OK) return rc;
    if (ws_bytes < az_i8_matmul_ws(m, n, k)) return refuse("az_i8_matmul: workspace too small");
    if (m > 0 && n > 0 && (!q_dev || !q_scale_dev || !w_dev || !w_scale_dev || !y_dev))
        return refuse("az_i8_matmul: null pointer");
    DeviceScope dev(device);
    if (dev.rc != AZ_OK || m == 0 || n == 0) return dev.rc;
    const Mm p = {m, n, k, q_dev, w_dev, ld_q, ld_w, q_scale_dev, w_scale_dev, bias_dev, residual_dev, ld_res, y_dev, ld_y, act};
    return i8_matmul(p, dtype, ws_dev, ws_bytes, (hipStream_t)stream);
}

size_t az_i8_linear_ws(int64_t m, int64_t n, int64_t k) {
    if (m < 1 || n < 1 || k < 1 || k > I8_MAX_K) return 0;
    return up256((size_t)m * linear_pitch(k)) + up256((size_t)m * 4) + az_i8_matmul_ws(m, n, k);
}

int az_i8_linear_dev(int device, int64_t m, int64_t n, int64_t k, const void* x_dev, int64_t ld_x, const int8_t* w_dev,
                     int64_t ld_w, const float* w_scale_dev, const float* bias_dev, const void* residual_dev,
                     int64_t ld_res, int act, int dtype, void* y_dev, int64_t ld_y, void* ws_dev, size_t ws_bytes,
                     void* stream) {
    int rc = mm_check(m, n, k, ld_x, ld_w, residual_dev, ld_res, act, dtype, ld_y);
    if (rc != AZ_OK) return rc;
    const size_t need = az_i8_linear_ws(m, n, k);
    if (ws_bytes < need || (need && (!ws_dev || ((uintptr_t)ws_dev & 255))))
        return refuse("az_i8_linear: workspace too small or not aligned to 256 bytes");
    if (m > 0 && n > 0 && (!x_dev || !w_dev || !w_scale_dev || !y_dev)) return refuse("az_i8_linear: null pointer");
    DeviceScope dev(device);
    if (dev.rc != AZ_OK || m == 0 || n == 0) return dev.rc;
    hipStream_t st = (hipStream_t)stream;
    i8* q = (i8*)ws_dev;
    float* qs = (float*)((char*)ws_dev + up256((size_t)m * linear_pitch(k)));
    char* rest = (char*)qs + up256((size_t)m * 4);
    rc = i8_quantize(dtype, m, k, x_dev, ld_x, m, nullptr, 1, q, linear_pitch(k), qs, st);
    if (rc != AZ_OK) return rc;
    const Mm p = {m, n, k, q, w_dev, linear_pitch(k), ld_w, qs, w_scale_dev, bias_dev, residual_dev, ld_res, y_dev, ld_y, act};
    return i8_matmul(p, dtype, rest, ws_bytes - (rest - (char*)ws_dev), st);
}

}  // extern "C"
