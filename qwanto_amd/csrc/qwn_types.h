// Element types of the serving operators' activations: vectors of 16 bytes
// loaded and stored as fp32 registers.  gfx950 takes 16-byte global accesses
// at any element's alignment, so rows of an odd stride move as wide as
// aligned ones.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

namespace qwn {

typedef _Float16 f16;
struct bf16 {
    uint16_t bits;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(f16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float to_float(bf16 v) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(v.bits) << 16);
}
// Rounded to the nearest, halves to even.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ f16 from_float<f16>(float v) { return static_cast<f16>(v); }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) {
    return bf16{__builtin_bit_cast(uint16_t, static_cast<__bf16>(v))};
}

// N elements of T at any address T may have.
template <typename T, int N>
struct __attribute__((packed, aligned(alignof(T)))) Vec {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T *p) {
    return *reinterpret_cast<const Vec<T, N> *>(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T *p, const Vec<T, N> &x) {
    *reinterpret_cast<Vec<T, N> *>(p) = x;
}

}  // namespace qwn
