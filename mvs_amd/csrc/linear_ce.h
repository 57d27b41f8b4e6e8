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
template <typename T> struct GradUnit { static constexpr float value = 1.0f, log2 = 0.0f; };
template <> struct GradUnit<f16_t> { static constexpr float value = 16384.0f, log2 = 14.0f; };

// One operand of a product: rows of `ld` bytes, the last of them `rows - 1` (a tile's rows beyond it read that one again)
struct Operand {
    const char *p;
    int64_t ld, rows;
    int64_t plane;      // (float32 in pieces) bytes from a piece's plane to the next one's
};

__device__ __forceinline__ bool ce_kept(int64_t target, int64_t ignore) { return target != ignore; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// The rows that are kept, moved together (more than kTogether of them: fewer fill one tile anyway): kept row i is row map[i] of the
// caller's, row r of the caller's is kept row place[r], -1 for an ignored one.  Everything between works on the kept rows: tiles and
// steps beyond *count are not begun, and what an ignored row holds is never read.  map == NULL: all rows as they are, in which case
// the kernels look at the targets.
constexpr int kTogether = 128;
struct CeRows {
    const int *map, *place, *count;
    const int64_t *target;            // of the kept rows
    int64_t n;                        // rows of the caller's
    int64_t ignore;
};
__device__ __forceinline__ int64_t ce_count(const CeRows &r) { return r.count ? *r.count : r.n; }
__device__ __forceinline__ int64_t ce_original(const CeRows &r, int64_t i) { return r.map ? r.map[i] : i; }

// g of the rows `first`, `first` + `step`, ... and their ratios to one number, which is the last: factors[i], factors[n + i],
// factors[2 n].  One factor for all rows is that number (0 if no row is kept, whatever comes from above: Inf times dW's empty sums
// would be NaN), the ratios are 1; else it is the largest magnitude, which one workgroup looks for first.  `tops`: a word of LDS per
// wave.
__device__ __forceinline__ void ce_factors(const CeRows &rows, const float *__restrict__ grad_loss, const float *__restrict__ kept, int reduction,
                                           float *__restrict__ factors, int64_t first, int64_t step, float *tops) {
    const int64_t count = ce_count(rows);
    float top = 0.0f;
    if (reduction != 0) {
        const float common = !(*kept > 0.0f) ? 0.0f : reduction == 2 ? grad_loss[0] : grad_loss[0] / *kept;
        for (int64_t i = first; i < count; i += step) {
            const bool here = ce_kept(rows.target[i], rows.ignore) && common != 0.0f;
            factors[i] = here ? common : 0.0f;
            factors[rows.n + i] = here ? common / common : 0.0f;      // (1; NaN where it is not a number to divide by)
        }
        top = common;
    } else {
        auto factor = [&](int64_t i) { return ce_kept(rows.target[i], rows.ignore) ? grad_loss[ce_original(rows, i)] : 0.0f; };
        for (int64_t i = first; i < count; i += step) top = fmaxf(top, __builtin_fabsf(factor(i)));
#pragma unroll
        for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
        for (int w = 0; w < (int)blockDim.x / 64; ++w) top = fmaxf(top, tops[w]);
        for (int64_t i = first; i < count; i += step) {
            const float g = factor(i);
            factors[i] = g;
            factors[rows.n + i] = g == 0.0f ? 0.0f : g / top;
        }
    }
    if (first == 0) factors[2 * rows.n] = top;
}

// out[row][c] = f * factor * the parts' sums, in order.  PER_ROW (dx): f = g[i] of kept row i = place[row]; rows that are ignored
// or have f = 0 are zeros, whatever their sums are.  Else (dW): f = g[0].
template <typename T, bool PER_ROW>
__device__ __forceinline__ void ce_finish(const float *__restrict__ sums, int64_t parts, int64_t rows, int64_t sum_rows, const int *__restrict__ place, int C, int64_t ld,
                                          const float *__restrict__ g, float factor, T *__restrict__ out, int64_t block) {
    const int64_t quads = ld >> 2, i = block * 256 + threadIdx.x, row = i / quads, quad = i - row * quads, c = quad * 4;
    if (row >= rows) return;
    const int64_t at = PER_ROW && place ? place[row] : row, step = sum_rows * quads;
    const float f = !PER_ROW ? g[0] : at >= 0 ? g[at] : 0.0f;
    f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!PER_ROW || f != 0.0f) {
        const f32x4_t *from = reinterpret_cast<const f32x4_t *>(sums) + at * quads + quad;
        s = from[0];
        int64_t p = 1;
        for (; p + 8 <= parts; p += 8) {
            f32x4_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = from[(p + j) * step];
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; p < parts; ++p) s += from[p * step];
    }
    Pack<T, 4> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o.v[r] = from_float<T>(PER_ROW && f == 0.0f ? 0.0f : s[r] * f * factor);
    T *to = out + row * C + c;
    if ((C & 3) == 0) put(to, o);
    else
        for (int r = 0; r < 4; ++r) if (c + r < C) to[r] = o.v[r];
}

// a value's pieces: 8 bits each, the first one cut instead of rounded where rounding would overflow
template <typename E, int PL, typename T>
__device__ __forceinline__ void pieces_of(T value, E (&p)[PL]) {
    if constexpr (PL == 1) {
        p[0] = value;
    } else {
        float v = value;
        p[0] = from_float<E>(v);
        if (__builtin_fabsf(v) > DtypeMax<E>::value && __builtin_fabsf(v) <= DtypeMax<float>::value) p[0].bits = (unsigned short)(__float_as_uint(v) >> 16);
#pragma unroll
        for (int q = 1; q < PL; ++q) {
            v -= to_float(p[q - 1]);
            p[q] = from_float<E>(v);
        }
    }
}

// ---- narrow rows: linear_ce_narrow.hip
constexpr int kNarrowRows = 128;      // rows that a workgroup of the narrow kernels owns
// 16-bit planes per element: float32 is carried as three bfloat16 pieces
inline int ce_planes(int dtype) { return dtype == MVS_DTYPE_F32 ? 3 : 1; }
// whether rows of C elements are narrow
inline bool ce_narrow(int C, int dtype) { return C <= (dtype == MVS_DTYPE_F32 ? 64 : 128); }

// How the work is cut: a workgroup owns kNarrowRows fixed rows and a part of the moving ones, in stages of 64.  `slots` is a number of
// workgroups that fills whole rounds of the chip (256 CUs x 3); every workgroup gets the same number of stages, four at least, so
// that they need at most `slots` (and one more per block of fixed rows).  Little work is one round: a workgroup's start and the sums
// it leaves then count for more than what the shares' rounding leaves idle.  Worked out alike on the host, which does not know how
// many rows are kept, and on the device.
struct NarrowSplit {
    int64_t blocks_x, blocks_w;       // blocks of fixed rows of x (the table moves), of the table (x moves); 0: not wanted
    int64_t parts_x, parts_w;
    int64_t per_x, per_w;             // moving rows per part
};
constexpr int64_t kNarrowRound = 768, kNarrowStatsSlots = 2 * kNarrowRound, kNarrowGradSlots = 4 * kNarrowRound;
__host__ __device__ inline NarrowSplit narrow_split(int64_t count, int64_t V, int64_t slots, bool of_x, bool of_table) {
    NarrowSplit s = {};
    const int64_t stages_v = (V + 63) / 64, stages_n = (count + 63) / 64;
    s.blocks_x = of_x ? (count + kNarrowRows - 1) / kNarrowRows : 0;
    s.blocks_w = of_table ? (V + kNarrowRows - 1) / kNarrowRows : 0;
    const int64_t stages = s.blocks_x * stages_v + s.blocks_w * stages_n;
    if (stages <= 16 * kNarrowRound) slots = kNarrowRound;
    const int64_t share = (stages + slots - 1) / slots, least = share > 4 ? share : 4;
    const int64_t x = stages_v / least > 1 ? (stages_v + stages_v / least - 1) / (stages_v / least) : stages_v;      // stages per part
    const int64_t w = stages_n / least > 1 ? (stages_n + stages_n / least - 1) / (stages_n / least) : stages_n;
    s.per_x = x * 64;
    s.per_w = w * 64;
    s.parts_x = (stages_v + x - 1) / x;
    s.parts_w = w > 0 ? (stages_n + w - 1) / w : 1;
    return s;
}
// workgroups, or parts times blocks, that any number of kept rows up to n can come to
inline int64_t narrow_most(int64_t blocks, int64_t moving, int64_t slots) {
    const int64_t stages = (moving + 63) / 64, whole = blocks * (stages / 4 > 1 ? stages / 4 : 1);
    return whole < slots + blocks ? whole : slots + blocks;
}

struct NarrowOperand {
    const void *source;               // [count][C] as the caller has it
    char *rows;                       // [count][planes][Cp] 16-bit pieces (one plane and C == Cp: `source`)
    char *trans;                      // [C][planes][pitch], pitch = count rounded up to 64, in the order the lanes hold (NULL: not needed)
    int64_t count;                    // (x: of the caller's; the kernels take the kept ones')
    int64_t pitch;
    bool write_rows;
};
struct NarrowArgs {
    NarrowOperand x, w;
    int C, Cp, planes;
    float scale2;                     // scale * log2 e
    CeRows kept_rows;
    // forward
    float2 *part;                     // [part][kept row]
    float *own;
    // backward
    const float *lse2;
    const float *grad_loss, *kept;
    int reduction;
    float *factors;                   // ce_factors
    float *sums_x, *sums_w;           // [part][kept row / table row][ld_sums]; NULL: that gradient is not wanted
    int64_t ld_sums;
    float factor;                     // scale over the unit that dl is carried in
    void *grad_x, *grad_w;
};
int ce_narrow_forward(int dtype, const NarrowArgs &a, hipStream_t st);       // up to the parts' statistics
int ce_narrow_backward(int dtype, const NarrowArgs &a, hipStream_t st);

}  // namespace mvs
