// mp_elem.h -- element types of the operators around the expert products
// (mp_scored.hip, mp_norm.hip, mp_sample.hip): f32, bf16 and fp16 in memory, f32
// in registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mp {

// numbered as MOE_DTYPE_*
constexpr int T_F32 = 0, T_BF16 = 1, T_F16 = 2;

template <int T> struct Elem;
template <> struct Elem<T_F32> {
    typedef float raw;
    static __device__ inline float load(raw v) { return v; }
    static __device__ inline raw store(float v) { return v; }
};
template <> struct Elem<T_BF16> {
    typedef uint16_t raw;
    static __device__ inline float load(raw v) { return __uint_as_float((uint32_t)v << 16); }
    // to the nearest, ties to even; a NaN stays one
    static __device__ inline raw store(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <> struct Elem<T_F16> {
    typedef uint16_t raw;
    static __device__ inline float load(raw v) { return (float)__builtin_bit_cast(_Float16, v); }
    static __device__ inline raw store(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

}  // namespace mp
