// devutil.h - device helpers of the kernel files beside kernels.hip (kv8.hip,
// token.hip): cross-lane moves without the LDS crossbar, reductions, vector
// types. kernels.hip has the same moves in its own text: measurements on file
// are tied to that text's hash.
#ifndef SURGE_DEVUTIL_H
#define SURGE_DEVUTIL_H

#include <hip/hip_runtime.h>
#include <hip/hip_ext.h>
#include <stdint.h>

#define TPB 256

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef int32_t v4i __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Partner lanes: quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror (i <-> 7-i
// in each 8 lanes), row_ror:8, and the gfx950 swaps across rows and half-waves.
template <int CTRL>
__device__ __forceinline__ uint32_t dppu(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t swap16(uint32_t v) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? p[0] : p[1];
}
__device__ __forceinline__ uint32_t swap32(uint32_t v) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? p[0] : p[1];
}
__device__ __forceinline__ float swap16f(float v) { return __uint_as_float(swap16(__float_as_uint(v))); }
__device__ __forceinline__ float swap32f(float v) { return __uint_as_float(swap32(__float_as_uint(v))); }
// Maximum of unsigned numbers over the wave; every lane gets it. On the bits
// of |x| this is the largest magnitude, with inf above every number and NaN
// above inf.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = max(v, dppu<0xB1>(v));
    v = max(v, dppu<0x4E>(v));
    v = max(v, dppu<0x141>(v));
    v = max(v, dppu<0x128>(v));
    v = max(v, swap16(v));
    return max(v, swap32(v));
}

__device__ __forceinline__ float wave_fmax(float v) {
    v = fmaxf(v, __uint_as_float(dppu<0xB1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dppu<0x4E>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dppu<0x141>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(dppu<0x128>(__float_as_uint(v))));
    v = fmaxf(v, swap16f(v));
    return fmaxf(v, swap32f(v));
}
__device__ __forceinline__ float wave_fsum(float v) {
    v += __uint_as_float(dppu<0xB1>(__float_as_uint(v)));
    v += __uint_as_float(dppu<0x4E>(__float_as_uint(v)));
    v += __uint_as_float(dppu<0x141>(__float_as_uint(v)));
    v += __uint_as_float(dppu<0x128>(__float_as_uint(v)));
    v += swap16f(v);
    return v + swap32f(v);
}

// Four consecutive floats: one 16-byte access where al (the address is
// 16-byte aligned, uniform over the launch), else four.
__device__ __forceinline__ f32x4 ld4(const float *p, bool al) {
    if (al) return *(const f32x4 *)p;
    return (f32x4){p[0], p[1], p[2], p[3]};
}
__device__ __forceinline__ void st4(float *p, f32x4 v, bool al) {
    if (al) { *(f32x4 *)p = v; return; }
    p[0] = v[0]; p[1] = v[1]; p[2] = v[2]; p[3] = v[3];
}

// A launch, and with `done` the event of its own completion: waiting for that
// takes 8.8 us from an empty kernel's launch on, where waiting for the stream,
// which queues a packet behind the kernel, takes 10.9.
template <typename K, typename... A>
static inline void launch(K kernel, dim3 grid, uint32_t threads, hipStream_t s, hipEvent_t done, A... args) {
    if (done) hipExtLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, (hipEvent_t) nullptr, done, 0, args...);
    else hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, args...);
}

#endif
