// c6_ops.h -- what the operators on logits and gradients (policy_ops.hip, grad_clip.hip) share: the three element types, wave and
// workgroup reductions, and the host side's device guard.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/connect6_amd.h"

int c6_set_error(int code, const char *msg);      // engine.cpp: the message c6_last_error() returns

// Every operator computes in f32 and rounds once, to nearest even, on the way out; infinities and NaN pass through.
template <typename T>
__device__ __forceinline__ float c6_get(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T c6_put(float v) { return (T)v; }

template <typename V, typename F>
__device__ __forceinline__ V c6_wave_all(V v, F f) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v = f(v, __shfl_xor(v, off, 64));
    return v;
}

// selects `device` for the life of the object and then puts the caller's choice back
struct C6DeviceScope {
    int prev = 0;
    bool moved = false, ok = true;
    explicit C6DeviceScope(int device) {
        ok = hipGetDevice(&prev) == hipSuccess;
        if (ok && prev != device) {
            ok = hipSetDevice(device) == hipSuccess;
            moved = ok;
        }
    }
    ~C6DeviceScope() {
        if (moved) (void)hipSetDevice(prev);
    }
};

static inline size_t c6_type_bytes(int type) { return type == C6_TYPE_F32 ? 4 : 2; }
static inline bool c6_type_ok(int type) { return type == C6_TYPE_F32 || type == C6_TYPE_F16 || type == C6_TYPE_BF16; }
static inline bool c6_aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// the visible devices, counted once; `what`'s caller reports the message
static inline int c6_check_device(int device) {
    static const int count = c6_device_count();
    if (count < 1) return c6_set_error(C6_ERR_NO_GPU, "no HIP device visible; this library has no CPU fallback");
    if (device < 0 || device >= count) return c6_set_error(C6_ERR_BAD_ARG, "no such device");
    return C6_OK;
}

// f<T>() for the element type named at run time
#define C6_BY_TYPE(type, T, ...)                                        \
    do {                                                                \
        if ((type) == C6_TYPE_F32) { using T = float; __VA_ARGS__; }    \
        else if ((type) == C6_TYPE_F16) { using T = _Float16; __VA_ARGS__; } \
        else { using T = __bf16; __VA_ARGS__; }                         \
    } while (0)
