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

// By one workgroup: a row's factor g_n (0 for an ignored one), and its ratio to the largest magnitude; factors[2 n] = that magnitude.
// `tops`: a word of LDS per wave.
__device__ __forceinline__ void ce_factors(const float *__restrict__ grad_loss, const float *__restrict__ kept, const int64_t *__restrict__ target, int64_t n,
                                           int64_t ignore, int reduction, float *__restrict__ factors, float *tops) {
    float common = reduction == 0 ? 0.0f : grad_loss[0];
    if (reduction == 1) common = common / *kept;
    auto factor = [&](int64_t i) { return !ce_kept(target[i], ignore) ? 0.0f : reduction == 0 ? grad_loss[i] : common; };
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) top = fmaxf(top, __builtin_fabsf(factor(i)));
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 64; ++w) top = fmaxf(top, tops[w]);
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const float g = factor(i);
        factors[i] = g;
        factors[n + i] = g == 0.0f ? 0.0f : g / top;
    }
    if (threadIdx.x == 0) factors[2 * n] = top;
}

// out[row][c] = f * factor * the parts' sums, in order; f = g[row] (dx: 0 for an ignored row, whose sums may be anything) or g[0] (dW)
template <typename T, bool PER_ROW>
__device__ __forceinline__ void ce_finish(const float *__restrict__ sums, int parts, int64_t rows, int C, int64_t ld, const float *__restrict__ g, float factor,
                                          T *__restrict__ out, int64_t block) {
    const int64_t quads = ld >> 2, i = block * 256 + threadIdx.x, row = i / quads, c = (i - row * quads) * 4;
    if (row >= rows) return;
    const f32x4_t *from = reinterpret_cast<const f32x4_t *>(sums) + i;
    const int64_t step = rows * quads;
    f32x4_t s = from[0];
    int p = 1;
    for (; p + 8 <= parts; p += 8) {
        f32x4_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = from[(p + j) * step];
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j];
    }
    for (; p < parts; ++p) s += from[p * step];
    const float f = PER_ROW ? g[row] : g[0];
    Pack<T, 4> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o.v[r] = from_float<T>(PER_ROW && f == 0.0f ? 0.0f : s[r] * f * factor);
    T *to = out + row * C + c;
    if ((C & 3) == 0) *reinterpret_cast<Pack<T, 4> *>(to) = o;
    else
        for (int r = 0; r < 4; ++r) if (c + r < C) to[r] = o.v[r];
}

// ---- narrow rows: linear_ce_narrow.hip
constexpr int kNarrowRows = 128;      // rows that a workgroup of the narrow kernels owns
// 16-bit planes per element: float32 is carried as three bfloat16 pieces
inline int ce_planes(int dtype) { return dtype == MVS_DTYPE_F32 ? 3 : 1; }
// whether rows of C elements are narrow
inline bool ce_narrow(int C, int dtype) { return C <= (dtype == MVS_DTYPE_F32 ? 64 : 128); }

struct NarrowOperand {
    const void *source;               // [count][C] as the caller has it
    char *rows;                       // [count][planes][Cp] 16-bit pieces (one plane and C == Cp: `source`)
    char *trans;                      // [C][planes][Mp], Mp = count rounded up to 64, in the order the lanes hold (NULL: not needed)
    int64_t count;
    bool write_rows;
};
struct NarrowArgs {
    NarrowOperand x, w;
    int C, Cp, planes;
    int64_t per_x, per_w;             // table rows per part (the rows of x are fixed), rows of x per part (the table's are)
    int parts_x, parts_w;
    float scale2;                     // scale * log2 e
    const int64_t *target;
    int64_t ignore;
    // forward
    float2 *part;                     // [part][n]
    float *own;
    // backward
    const float *lse2;
    const float *grad_loss, *kept;
    int reduction;
    float *factors;                   // [n] g, [n] g / max|g|, [1] max|g|
    float *sums_x, *sums_w;           // [part][rows][ld_sums]; NULL: that gradient is not wanted
    int64_t ld_sums;
    float factor;                     // scale over the unit that dl is carried in
    void *grad_x, *grad_w;
};
int ce_narrow_forward(int dtype, const NarrowArgs &a, hipStream_t st);       // up to the parts' statistics
int ce_narrow_backward(int dtype, const NarrowArgs &a, hipStream_t st);

}  // namespace mvs
