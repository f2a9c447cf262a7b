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

// 16 bytes at a time: N elements at an address aligned to ONE element (the memory pipeline takes such addresses; a wave's 1024 bytes then touch nine
// lines of 128 bytes instead of eight), in registers as they lie in memory
typedef uint32_t c6_u32x4 __attribute__((ext_vector_type(4)));
template <typename T>
struct C6Vec {
    static constexpr int N = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { c6_u32x4 u; };
    static __device__ __forceinline__ c6_u32x4 load(const T *p) { return reinterpret_cast<const Raw *>(p)->u; }
    static __device__ __forceinline__ void store(T *p, c6_u32x4 u) { reinterpret_cast<Raw *>(p)->u = u; }
    // ... written past the caches: nobody reads it soon, and what they hold is still wanted
    static __device__ __forceinline__ void store_past(T *p, c6_u32x4 u) {
        typedef uint32_t loose __attribute__((ext_vector_type(4), aligned(2)));
        __builtin_nontemporal_store((loose)u, reinterpret_cast<loose *>(p));
    }
    static __device__ __forceinline__ void get(c6_u32x4 u, float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = u[i];      // (a bit cast of the vector's element itself takes element 0)
            if constexpr (sizeof(T) == 4) {
                f[i] = __builtin_bit_cast(float, w);
            } else if constexpr (__is_same(T, __bf16)) {
                f[2 * i] = __builtin_bit_cast(float, w << 16);
                f[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
            } else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = __builtin_bit_cast(h2, w);
                f[2 * i] = (float)h[0];
                f[2 * i + 1] = (float)h[1];
            }
        }
    }
    static __device__ __forceinline__ c6_u32x4 put(const float (&f)[N]) {
        c6_u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) {
                u[i] = __builtin_bit_cast(uint32_t, f[i]);
            } else {
                typedef T t2 __attribute__((ext_vector_type(2)));
                typedef float f2 __attribute__((ext_vector_type(2)));
                u[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{f[2 * i], f[2 * i + 1]}), t2));
            }
        }
        return u;
    }
    // elements whose bit of `ok` is clear become -infinity, in place: all ones or zeros for each bit (a signed bit field), then a bitwise select
    static __device__ __forceinline__ uint32_t ones(uint32_t ok, int i) { return (uint32_t)((int32_t)(ok << (31 - i)) >> 31); }
    static __device__ __forceinline__ void keep(c6_u32x4 &u, uint32_t ok) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t m, fill;
            if constexpr (sizeof(T) == 4) {
                m = ones(ok, i);
                fill = 0xff800000u;
            } else {
                m = (ones(ok, 2 * i) & 0xffffu) | (ones(ok, 2 * i + 1) & 0xffff0000u);
                fill = __is_same(T, __bf16) ? 0xff80ff80u : 0xfc00fc00u;
            }
            u[i] = (u[i] & m) | (fill & ~m);
        }
    }
    // the first n of N elements (the end of a row); the rest reads as `fill`
    static __device__ __forceinline__ void get_some(const T *p, int n, float fill, float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = i < n ? c6_get(p[i]) : fill;
    }
    static __device__ __forceinline__ void put_some(T *p, int n, const float (&f)[N]) {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) p[i] = c6_put<T>(f[i]);
    }
};

// f over each row of 16 lanes, by DPP: xor 1, xor 2, mirror 8, mirror 16
template <typename F>
__device__ __forceinline__ float c6_row_all(float v, F f) {
#define C6_DPP(ctrl) v = f(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true)))
    C6_DPP(0xb1);
    C6_DPP(0x4e);
    C6_DPP(0x141);
    C6_DPP(0x140);
#undef C6_DPP
    return v;
}
// ... and over all 64, the four rows through scalar registers: the same in every lane
template <typename F>
__device__ __forceinline__ float c6_wave_all(float v, F f) {
    const int bits = __builtin_bit_cast(int, c6_row_all(v, f));
    const auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(bits, lane)); };
    return f(f(row(0), row(16)), f(row(32), row(48)));
}
__device__ __forceinline__ float c6_wave_sum(float v) { return c6_wave_all(v, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ double c6_wave_sum(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
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

// Launches and says whether that worked, by the launch's own answer: hipGetLastError() would give an older error of the thread's for this call's.
template <typename T>
struct C6As { typedef T type; };
template <typename... P>
static inline bool c6_launch(void (*kernel)(P...), unsigned grid, unsigned block, hipStream_t s, typename C6As<P>::type... args) {
    void *at[] = {const_cast<void *>(static_cast<const void *>(&args))...};
    const bool ok = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(grid), dim3(block), at, 0, s) == hipSuccess;
    if (!ok) (void)hipGetLastError();      // (reported by the caller: not left behind for somebody else's)
    return ok;
}

static inline size_t c6_type_bytes(int type) { return type == C6_TYPE_F32 ? 4 : 2; }
static inline bool c6_type_ok(int type) { return type == C6_TYPE_F32 || type == C6_TYPE_F16 || type == C6_TYPE_BF16; }
static inline bool c6_aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// the visible devices, counted once
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
