// az_ops.hpp -- what the operators on caller-owned device tensors share (az_int8.hip, az_ortho.hip): element types, the
// device of a call, and the byte geometry of their matrix tiles.
#pragma once
#include "az_internal.hpp"

namespace az {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// rounds to nearest, ties to even, as every conversion to 16 bits here
__device__ inline float to_f32(float v) { return v; }
__device__ inline float to_f32(f16 v) { return (float)v; }
__device__ inline float to_f32(bf16 v) { return (float)v; }
template <class T>
__device__ inline T from_f32(float v) {
    return (T)v;
}

// Loads above stay above (left alone, the compiler moves each one to its use to save registers, and every one waits for memory).
__device__ inline void loads_first() { __builtin_amdgcn_sched_barrier(0); }

inline size_t dtype_size(int dtype) { return dtype == AZ_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == AZ_F32 || dtype == AZ_F16 || dtype == AZ_BF16; }

#define AZ_DISPATCH_DTYPE(dtype, ...)                         \
    switch (dtype) {                                          \
        case AZ_F32: { using T = float; __VA_ARGS__; } break; \
        case AZ_F16: { using T = f16; __VA_ARGS__; } break;   \
        default: { using T = bf16; __VA_ARGS__; } break;      \
    }

// Makes `device` current for one call and puts the caller's device back at its end (a caller's other work, torch's
// first of all, goes by the current device).
struct DeviceScope {
    int before = -1, rc = AZ_OK;
    explicit DeviceScope(int device) {
        static const int n = [] {   // the number of devices does not change while the process lives
            int k = 0;
            return hipGetDeviceCount(&k) == hipSuccess ? k : 0;
        }();
        if (n <= 0) {
            (void)hipGetLastError();
            set_error("no usable HIP device: libazamd has no CPU path");
            rc = AZ_ERR_NO_DEVICE;
            return;
        }
        if (device < 0 || device >= n) {
            set_error("device ordinal out of range");
            rc = AZ_ERR_ARG;
            return;
        }
        int cur = -1;
        if (hipGetDevice(&cur) == hipSuccess && cur == device) return;
        if (hipSetDevice(device) != hipSuccess) {
            (void)hipGetLastError();
            set_error("hipSetDevice failed");
            rc = AZ_ERR_HIP;
            return;
        }
        before = cur;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

inline int launch_status(const char* fn) {
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) return AZ_OK;
    set_error(std::string(fn) + ": " + hipGetErrorString(e));
    return AZ_ERR_HIP;
}
inline int refuse(const char* what) {
    set_error(what);
    return AZ_ERR_ARG;
}
inline bool overlap(const void* p, size_t np, const void* q, size_t nq) {   // sizes in bytes
    return (uintptr_t)p < (uintptr_t)q + nq && (uintptr_t)q < (uintptr_t)p + np;
}
// a matrix in memory: rows of `width` bytes, `ld` bytes apart
struct Span {
    const void* p;
    i64 rows, width, ld;
    size_t bytes() const {   // capped far above any memory
        const i64 cap = (i64)1 << 56;
        i64 n;
        if (__builtin_mul_overflow(rows - 1, ld, &n) || __builtin_add_overflow(n, width, &n) || n > cap) n = cap;
        return (size_t)n;
    }
};
// whether two share a byte; columns of one buffer beside each other do not
inline bool overlap(Span a, Span b) {
    if (!a.p || !b.p || a.rows < 1 || b.rows < 1) return false;
    if (a.rows == 1) a.ld = b.ld;
    if (b.rows == 1) b.ld = a.ld;
    if (!overlap(a.p, a.bytes(), b.p, b.bytes())) return false;
    if (a.ld != b.ld || a.width > a.ld || b.width > b.ld) return true;
    const i64 off = (i64)((uintptr_t)b.p - (uintptr_t)a.p) % a.ld, d = off < 0 ? off + a.ld : off;   // b's first column in a's rows
    return d < a.width || d + b.width > a.ld;
}

}  // namespace az
