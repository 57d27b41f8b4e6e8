// What the kernels of the cross entropy against a table share (linear_ce.hip has the scheme, linear_ce_narrow.hip the one for
// narrow rows).
#pragma once
#include "dtype.h"

namespace mvs {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRowBytes = 128;                  // bytes of k per stage and row

__device__ __forceinline__ void mma16(f32x4_t &c, u32x4_t a, u32x4_t b, float) {
    const f32x4_t fa = __builtin_bit_cast(f32x4_t, a), fb = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j], fb[j], c, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4_t &c, u32x4_t a, u32x4_t b, bf16_t) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ void mma16(f32x4_t &c, u32x4_t a, u32x4_t b, f16_t) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// dl is carried times this
template <typename T> struct GradUnit { static constexpr float value = 1.0f; };
template <> struct GradUnit<f16_t> { static constexpr float value = 16384.0f; };

// One operand of a product: rows of `ld` bytes, the last of them `rows - 1` (a tile's rows beyond it read that one again)
struct Operand {
    const char *p;
    int64_t ld, rows;
};

__device__ __forceinline__ bool ce_kept(int64_t target, int64_t ignore) { return target != ignore; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// ---- narrow rows: linear_ce_narrow.hip
constexpr int kNarrowRows = 128;      // rows that a workgroup of the narrow kernels owns
struct NarrowArgs {
    // `fixed`: the rows a workgroup owns, `moving`: the rows it walks; both of `Cp` elements, `moving_t`: the latter transposed
    Operand fixed, moving, moving_t;
    int64_t per_part;                  // rows of `moving` per blockIdx.y, a multiple of 64
    float scale2;
    const int64_t *target;             // of the rows of x
    int64_t ignore;
    // forward
    float2 *part;                      // [part][n]
    float *own;
    // backward
    const float *lse2, *ratio;
    float *sums;                       // [part][fixed.rows][ld_sums]
    int64_t ld_sums;
    int C;
};
// whether a row of C elements is narrow: at most 256 bytes once padded to whole 128-byte steps
inline bool ce_narrow(int Cp, int es) { return Cp * es <= 256; }
int ce_narrow_stats(int dtype, int row_bytes, const NarrowArgs &a, int parts, hipStream_t st);
int ce_narrow_grad(int dtype, int row_bytes, bool of_table, const NarrowArgs &a, int parts, hipStream_t st);

}  // namespace mvs
