// Element types of the entry points that take more than float32 (MVS_DTYPE_*): widened to float, rounded to nearest even once.
#pragma once
#include "mvs_common.h"

namespace mvs {

struct bf16_t { unsigned short bits; };
struct f16_t { _Float16 v; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16_t x) { return __uint_as_float((unsigned)x.bits << 16); }
__device__ __forceinline__ float to_float(f16_t x) { return (float)x.v; }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16_t from_float<bf16_t>(float x) {
    const __bf16 b = (__bf16)x;      // (v_cvt_pk_bf16_f32: nearest even, NaN stays one)
    return bf16_t{__builtin_bit_cast(unsigned short, b)};
}
template <>
__device__ __forceinline__ f16_t from_float<f16_t>(float x) { return f16_t{(_Float16)x}; }

// two values as one 32-bit word of two 16-bit elements (one instruction), and back
__device__ __forceinline__ unsigned pack2(float a, float b, bf16_t) {
    typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
    const pair_t p = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, p);
}
__device__ __forceinline__ unsigned pack2(float a, float b, f16_t) {
    typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
    const pair_t p = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(unsigned, p);
}
__device__ __forceinline__ float low_of(unsigned p, bf16_t) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_of(unsigned p, bf16_t) { return __uint_as_float(p & 0xffff0000u); }
__device__ __forceinline__ float low_of(unsigned p, f16_t) { return (float)__builtin_bit_cast(_Float16, (unsigned short)p); }
__device__ __forceinline__ float high_of(unsigned p, f16_t) { return (float)__builtin_bit_cast(_Float16, (unsigned short)(p >> 16)); }

// largest finite value of a type
template <typename T> struct DtypeMax;
template <> struct DtypeMax<float> { static constexpr float value = 3.4028234663852886e38f; };
template <> struct DtypeMax<bf16_t> { static constexpr float value = 3.3895313892515355e38f; };
template <> struct DtypeMax<f16_t> { static constexpr float value = 65504.0f; };

// VEC elements moved as one access
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

// A Pack written as one access.  (Assigned as a struct beside a branch that writes its elements one by one, the compiler shares the
// elements' stores between the two: three narrow stores in place of a wide one.)
template <typename T, int VEC>
__device__ __forceinline__ void put(void *to, const Pack<T, VEC> &p) {
    if constexpr (sizeof(p) % 8 == 0) {
        typedef unsigned words_t __attribute__((ext_vector_type(sizeof(p) / 4)));
        *static_cast<words_t *>(to) = __builtin_bit_cast(words_t, p);
    } else {
        *static_cast<Pack<T, VEC> *>(to) = p;
    }
}

// A launch counts the threads of a dimension in 32 bits: more than kGridRow workgroups (of at most 1024) are rows of that many, and
// those behind the last one find nothing to do.
constexpr int64_t kGridRow = (int64_t)1 << 21;
inline dim3 grid_of(int64_t groups) {
    return groups <= kGridRow ? dim3((unsigned)groups) : dim3((unsigned)kGridRow, (unsigned)((groups + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ int64_t group_of() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

inline size_t dtype_size(int dtype) { return dtype == MVS_DTYPE_F32 ? 4 : (dtype == MVS_DTYPE_BF16 || dtype == MVS_DTYPE_F16) ? 2 : 0; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace mvs

// f(T()) for the element type that `dtype` names; `dtype` has been checked
#define MVS_DTYPE_DISPATCH(dtype, T, ...)                                   \
    do {                                                                    \
        if ((dtype) == MVS_DTYPE_F32) { using T = float; __VA_ARGS__; }     \
        else if ((dtype) == MVS_DTYPE_BF16) { using T = mvs::bf16_t; __VA_ARGS__; } \
        else { using T = mvs::f16_t; __VA_ARGS__; }                         \
    } while (0)
