// Cross entropy against a table for NARROW rows (at most 256 bytes: float32 C <= 64, 16 bits C <= 128), the shape of feature
// matching: points of one view against all cells of another.
//
// With so few operations per logit the piecewise scheme of linear_ce.hip is bound by writing and reading dl (20480 x 20480 x 32
// float32: 6.7 GB, against 0.27 TFLOP in all).  Here dl never leaves the registers: a workgroup owns 128 rows, keeps them as matrix
// fragments and walks the other operand 64 rows at a time through LDS (DMA, two stages).  Per 32 rows of it
//     S[m][n] = <moving m, fixed n>      lane: n = lane & 15, m = 4 (lane >> 4) + r, two 16-row tiles
//     dl      = (exp2(S scale2 - lse2) - [target]) ratio
//     sums[c][n] += sum_m moving_t[c][m] dl[m][n]
// and the second product takes dl from the accumulators as they lie: the order of k inside a matrix instruction is free if both
// operands agree, and 4 g + r (float32: four instructions of k = 4, the r-th takes register r) or {4 g + 0..3, 16 + 4 g + 0..3}
// (16 bits: one of k = 32) is the order the lanes hold.  The transposed copy is written in that order (ce_transpose_kernel).
// dx: fixed = x, moving = the table.  dW: fixed = the table, moving = x, whose rows' statistics then run along m.
// The forward pass is the first product alone with a running maximum and sum per lane.
// Operations: 10 N V C forward and backward (the logits three times) instead of 8, all on chip.
#include "linear_ce.h"

namespace mvs {

constexpr int kMoving = 64;      // rows of the moving operand per stage

// RB: bytes of a row, 128 or 256
template <typename T, int RB>
struct Narrow {
    static constexpr int KSTEPS = RB / 64;                       // 64-byte fragments along k
    static constexpr int CT = RB / (int)sizeof(T) / 16;          // 16-column tiles of the result
    static constexpr int ROWS_B = kMoving * RB;                  // moving tile
    static constexpr int TRANS_B = CT * 16 * kMoving * (int)sizeof(T);      // its transpose: the same bytes
    static_assert(ROWS_B == TRANS_B, "");
};

// Copies `rows` rows of 128 bytes (byte `at` of each operand row on) to LDS, chunks exchanged by the row's low three bits; 4 waves.
template <int ROWS>
__device__ __forceinline__ void narrow_copy(const Operand &o, int64_t row0, int64_t at, unsigned lds_to) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r8 = lane >> 3, chunk = (lane & 7) ^ r8;
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i) {
        const int c = wave + i * 4;
        const int64_t row = row0 + c * 8 + r8;
        glds16(o.p + (row < o.rows ? row : o.rows - 1) * o.ld + at + chunk * 16, lds_to + (unsigned)(c * 1024));
    }
}

// the 16-byte fragment of tile row `row` (16-row tile base + lane & 15) at 64-byte step `k`
__device__ __forceinline__ u32x4_t narrow_frag(const char *tile, int row, int k, int rows_per_half) {
    const int fk = (threadIdx.x & 63) >> 4, chunk = (k & 1) * 4 + fk;
    return *reinterpret_cast<const u32x4_t *>(tile + (k >> 1) * rows_per_half * 128 + row * 128 + ((chunk ^ (row & 7)) * 16));
}

template <typename T, int RB>
__global__ __launch_bounds__(256, 2) void narrow_stats_kernel(NarrowArgs a) {
    using X = Narrow<T, RB>;
    __shared__ __align__(1024) char lds[2][X::ROWS_B];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15;
    const int64_t n0 = (int64_t)blockIdx.x * kNarrowRows + wave * 32;
    const int64_t m_begin = (int64_t)blockIdx.y * a.per_part, m_end = min(a.moving.rows, m_begin + a.per_part);
    const unsigned base = (unsigned)(uintptr_t)&lds[0][0];
    auto copy = [&](int64_t m0, int stage) {
#pragma unroll
        for (int h = 0; h < RB / 128; ++h) narrow_copy<kMoving>(a.moving, m0, h * 128, base + (unsigned)(stage * X::ROWS_B + h * kMoving * 128));
    };
    copy(m_begin, 0);
    u32x4_t fixed[2][X::KSTEPS];
    int64_t target[2];
    float top[2], sum[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + j * 16 + ln, row = n < a.fixed.rows ? n : a.fixed.rows - 1;
#pragma unroll
        for (int k = 0; k < X::KSTEPS; ++k) fixed[j][k] = *reinterpret_cast<const u32x4_t *>(a.fixed.p + row * a.fixed.ld + k * 64 + (lane >> 4) * 16);
        target[j] = n < a.fixed.rows ? a.target[n] : -1;
        top[j] = -INFINITY;
        sum[j] = 0.0f;
    }
    int stage = 0;
    for (int64_t m0 = m_begin; m0 < m_end; m0 += kMoving, stage ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (m0 + kMoving < m_end) copy(m0 + kMoving, stage ^ 1);
        const char *tile = lds[stage];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t mh = m0 + half * 32;
            if (mh >= m_end) break;
            f32x4_t s[2][2] = {};
#pragma unroll
            for (int k = 0; k < X::KSTEPS; ++k) {
                u32x4_t f[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) f[i] = narrow_frag(tile, half * 32 + i * 16 + ln, k, kMoving);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) mma16(s[i][j], f[i], fixed[j][k], T());
            }
            const int64_t m_lane = mh + (lane >> 4) * 4;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float l[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) l[e] = s[e >> 2][j][e & 3] * a.scale2;
                if (mh + 32 > m_end) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) if (m_lane + (e >> 2) * 16 + (e & 3) >= m_end) l[e] = -INFINITY;
                }
                const int64_t d = target[j] - mh;
                if (__ballot(d >= 0 && d < 32)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (m_lane + (e >> 2) * 16 + (e & 3) == target[j] && target[j] < m_end) a.own[n0 + j * 16 + ln] = l[e];
                }
                float t = top[j];
#pragma unroll
                for (int e = 0; e < 8; ++e) t = fmaxf(t, l[e]);
                const float low = t == -INFINITY ? 0.0f : t;      // (-Inf alone sums to 0; Inf - Inf and NaN make the sum NaN)
                float add = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) add += __builtin_amdgcn_exp2f(l[e] - low);
                sum[j] = sum[j] * __builtin_amdgcn_exp2f(top[j] - low) + add;
                top[j] = t;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float t = fmaxf(top[j], __shfl_xor(top[j], 16));
        t = fmaxf(t, __shfl_xor(t, 32));
        float r = sum[j] * __builtin_amdgcn_exp2f(top[j] - (t == -INFINITY ? 0.0f : t));
        r += __shfl_xor(r, 16);
        r += __shfl_xor(r, 32);
        const int64_t n = n0 + j * 16 + ln;
        if (lane < 16 && n < a.fixed.rows) a.part[(int64_t)blockIdx.y * a.fixed.rows + n] = make_float2(t, r);
    }
}

// out[c][n] += sum_m trans[c][m] s[m][n] over the 32 rows m of one half of a stage
template <typename T, int CT>
__device__ __forceinline__ void narrow_second(const char *trans, int half, const f32x4_t (&s)[2][2], f32x4_t (&out)[CT][2]) {
    const int ln = threadIdx.x & 15;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)      // (64 bytes of the row: 16 m; half = the 128-byte half)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                const u32x4_t f = narrow_frag(trans, c * 16 + ln, half * 2 + i, CT * 16);
#pragma unroll
                for (int j = 0; j < 2; ++j) mma16(out[c][j], f, __builtin_bit_cast(u32x4_t, s[i][j]), T());
            }
    } else {
        u32x4_t d[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const Pack<T, 2> p{{from_float<T>(s[w >> 1][j][(w & 1) * 2]), from_float<T>(s[w >> 1][j][(w & 1) * 2 + 1])}};
                d[j][w] = __builtin_bit_cast(unsigned, p);
            }
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const u32x4_t f = narrow_frag(trans, c * 16 + ln, half, CT * 16);
#pragma unroll
            for (int j = 0; j < 2; ++j) mma16(out[c][j], f, d[j], T());
        }
    }
}

// OF_TABLE: fixed = table rows, moving = rows of x (statistics along m); else fixed = rows of x, moving = table rows
template <typename T, int RB, bool OF_TABLE>
__global__ __launch_bounds__(256, 2) void narrow_grad_kernel(NarrowArgs a) {
    using X = Narrow<T, RB>;
    constexpr float unit = GradUnit<T>::value;
    __shared__ __align__(1024) char lds[2][X::ROWS_B + X::TRANS_B];
    __shared__ float row_lse[OF_TABLE ? 2 : 1][kMoving], row_ratio[OF_TABLE ? 2 : 1][kMoving];
    __shared__ int row_target[OF_TABLE ? 2 : 1][kMoving];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, group = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * kNarrowRows + wave * 32;
    const int64_t m_begin = (int64_t)blockIdx.y * a.per_part, m_end = min(a.moving.rows, m_begin + a.per_part);
    const unsigned base = (unsigned)(uintptr_t)&lds[0][0];
    // the transposed tile is CT * 16 rows of kMoving elements: one 128-byte half (16 bits) or two (float32)
    constexpr int HALVES_T = kMoving * (int)sizeof(T) / 128;
    auto copy = [&](int64_t m0, int stage) {
        const unsigned to = base + (unsigned)(stage * (X::ROWS_B + X::TRANS_B));
#pragma unroll
        for (int h = 0; h < RB / 128; ++h) narrow_copy<kMoving>(a.moving, m0, h * 128, to + (unsigned)(h * kMoving * 128));
#pragma unroll
        for (int h = 0; h < HALVES_T; ++h)
            narrow_copy<X::CT * 16>(a.moving_t, 0, m0 * (int64_t)sizeof(T) + h * 128, to + (unsigned)(X::ROWS_B + h * X::CT * 16 * 128));
    };
    // statistics of the moving rows of a stage (OF_TABLE): thread t < kMoving's row; loaded ahead, stored with the stage
    auto stats = [&](int64_t m0, float &lse, float &ratio, int &target) {
        const int64_t m = m0 + threadIdx.x;
        const bool kept = threadIdx.x < kMoving && m < m_end && ce_kept(a.target[m], a.ignore);
        lse = kept ? a.lse2[m] : 0.0f;
        ratio = kept ? a.ratio[m] * unit : 0.0f;
        target = kept && a.target[m] >= 0 && a.target[m] < a.fixed.rows ? (int)a.target[m] : -1;
    };
    copy(m_begin, 0);
    float lse_next, ratio_next;
    int target_next;
    if (OF_TABLE) stats(m_begin, lse_next, ratio_next, target_next);
    u32x4_t fixed[2][X::KSTEPS];
    int64_t target[2];
    float lse[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + j * 16 + ln, row = n < a.fixed.rows ? n : a.fixed.rows - 1;
        const bool kept = OF_TABLE || (n < a.fixed.rows && ce_kept(a.target[row], a.ignore));
#pragma unroll
        for (int k = 0; k < X::KSTEPS; ++k) {
            fixed[j][k] = *reinterpret_cast<const u32x4_t *>(a.fixed.p + row * a.fixed.ld + k * 64 + group * 16);
            if (!kept) fixed[j][k] = u32x4_t{0, 0, 0, 0};      // (whatever an ignored row holds; its exponentials are of -Inf)
        }
        target[j] = OF_TABLE ? n : kept ? a.target[row] : -1;
        lse[j] = OF_TABLE ? 0.0f : kept ? a.lse2[row] : INFINITY;
    }
    f32x4_t out[X::CT][2] = {};
    int stage = 0;
    for (int64_t m0 = m_begin; m0 < m_end; m0 += kMoving, stage ^= 1) {
        if (OF_TABLE && threadIdx.x < kMoving) {      // (last read two stages ago, a barrier in between)
            row_lse[stage & (OF_TABLE ? 1 : 0)][threadIdx.x] = lse_next;
            row_ratio[stage & (OF_TABLE ? 1 : 0)][threadIdx.x] = ratio_next;
            row_target[stage & (OF_TABLE ? 1 : 0)][threadIdx.x] = target_next;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (m0 + kMoving < m_end) {
            copy(m0 + kMoving, stage ^ 1);
            if (OF_TABLE) stats(m0 + kMoving, lse_next, ratio_next, target_next);
        }
        const char *tile = lds[stage], *trans = tile + X::ROWS_B;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t mh = m0 + half * 32;
            if (mh >= m_end) break;
            f32x4_t s[2][2] = {};
#pragma unroll
            for (int k = 0; k < X::KSTEPS; ++k) {
                u32x4_t f[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) f[i] = narrow_frag(tile, half * 32 + i * 16 + ln, k, kMoving);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) mma16(s[i][j], f[i], fixed[j][k], T());
            }
            if (OF_TABLE) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int at = half * 32 + i * 16 + group * 4;
                    const f32x4_t l4 = *reinterpret_cast<const f32x4_t *>(&row_lse[stage][at]), r4 = *reinterpret_cast<const f32x4_t *>(&row_ratio[stage][at]);
                    const u32x4_t t4 = *reinterpret_cast<const u32x4_t *>(&row_target[stage][at]);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float d = __builtin_amdgcn_exp2f(s[i][j][r] * a.scale2 - l4[r]);
                            if ((int)t4[r] == (int)(n0 + j * 16 + ln)) d -= 1.0f;
                            s[i][j][r] = r4[r] == 0.0f ? 0.0f : d * r4[r];      // (an ignored row's S may be anything)
                        }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[i][j][r] = __builtin_amdgcn_exp2f(s[i][j][r] * a.scale2 - lse[j]);
                    const int64_t d = target[j] - mh;
                    if (__ballot(d >= 0 && d < 32)) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) if (d == i * 16 + group * 4 + r) s[i][j][r] -= 1.0f;
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[i][j][r] *= unit;
                }
                if (mh + 32 > m_end) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (mh + i * 16 + group * 4 + r >= m_end) s[i][0][r] = s[i][1][r] = 0.0f;
                }
            }
            narrow_second<T, X::CT>(trans, half, s, out);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + j * 16 + ln;
        if (n >= a.fixed.rows) continue;
#pragma unroll
        for (int c = 0; c < X::CT; ++c) {
            const int64_t col = c * 16 + group * 4;
            if (col < a.C) *reinterpret_cast<f32x4_t *>(a.sums + ((int64_t)blockIdx.y * a.fixed.rows + n) * a.ld_sums + col) = out[c][j];
        }
    }
}

template <typename T, int RB>
static void narrow_launch_stats(const NarrowArgs &a, int parts, hipStream_t st) {
    hipLaunchKernelGGL((narrow_stats_kernel<T, RB>), dim3((unsigned)ceil_div(a.fixed.rows, kNarrowRows), (unsigned)parts), dim3(256), 0, st, a);
}
template <typename T, int RB>
static void narrow_launch_grad(bool of_table, const NarrowArgs &a, int parts, hipStream_t st) {
    const dim3 grid((unsigned)ceil_div(a.fixed.rows, kNarrowRows), (unsigned)parts);
    if (of_table) hipLaunchKernelGGL((narrow_grad_kernel<T, RB, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((narrow_grad_kernel<T, RB, false>), grid, dim3(256), 0, st, a);
}

int ce_narrow_stats(int dtype, int row_bytes, const NarrowArgs &a, int parts, hipStream_t st) {
    MVS_DTYPE_DISPATCH(dtype, T, {
        if (row_bytes == 128) narrow_launch_stats<T, 128>(a, parts, st);
        else narrow_launch_stats<T, 256>(a, parts, st);
    });
    return check_launch("mvs_linear_ce_fwd");
}
int ce_narrow_grad(int dtype, int row_bytes, bool of_table, const NarrowArgs &a, int parts, hipStream_t st) {
    MVS_DTYPE_DISPATCH(dtype, T, {
        if (row_bytes == 128) narrow_launch_grad<T, 128>(of_table, a, parts, st);
        else narrow_launch_grad<T, 256>(of_table, a, parts, st);
    });
    return check_launch("mvs_linear_ce_bwd");
}

}  // namespace mvs
