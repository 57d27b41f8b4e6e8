// Cross entropy against a table for NARROW rows (float32 C <= 64, 16 bits C <= 128), the shape of feature matching: points of one
// view against all cells of another.
//
// With so few operations per logit the piecewise scheme of linear_ce.hip is bound by writing and reading dl (20480 x 20480 x 32
// float32: 6.7 GB, against 0.27 TFLOP in all).  Here dl never leaves the registers: a workgroup owns 128 rows, keeps them as matrix
// fragments and walks the other operand through LDS (DMA, two stages).  Per 32 rows of it
//     S[m][n] = <moving m, fixed n>      lane: n = lane & 15, m = 4 (lane >> 4) + r, two 16-row tiles
//     dl      = (exp2(S scale2 - lse2) - [target]) ratio
//     sums[c][n] += sum_m trans[c][m] dl[m][n]
// and the second product takes dl from the accumulators as they lie: the order of k inside a matrix instruction is free if both
// operands agree, and {4 g + 0..3, 16 + 4 g + 0..3} is what lane group g holds of 32 rows.  The transposed copy is written in that
// order.  dx: fixed = x, moving = the table.  dW: fixed = the table, moving = x, whose rows' statistics then run along m.  The forward
// pass is the first product alone with a running maximum and sum per lane.
//
// float32 runs on the bfloat16 pipe: a value is three bfloat16 pieces of 8 bits each (24 in all: nothing is dropped), a product six
// of the nine piece products -- the others are below 2^-24 of it -- summed in float32.  16 times the float32 pipe's rate over six
// products.  dl is split the same way in the registers.  For 16-bit operands dl is two pieces of their type, 16 bits at the least: a
// row's dl sum to 0, so where the table's rows have much in common the gradient is what is left of sums far larger than itself, and
// half a unit of 8 or 11 bits in each dl shows there (4096 x 17296 x 8 bfloat16: dx 1.75 times as far from the exact one as with
// float32 dl).
//
// Operations: 10 N V C forward and backward (the logits three times) instead of 8, all on chip.  A 32 x 32 block of logits costs a
// wave 24 + 24 matrix instructions of 16 cycles (float32, C = 32, a gradient) and about as many cycles of exponentials and splitting.
// Neither pipe is full: of 14336 x 20480 x 32 float32 the gradients take 387 us, the matrix cores busy 52 % of it and the vector unit
// 64 %, the statistics 119 us at 37 and 64 %.  A wave goes through product, exponentials, splitting and second product in order, and
// the 2.3 to 2.6 waves a SIMD holds (LDS of two stages, registers of the fragments) do not hide each other's: 37 to 47 % of their
// cycles wait to issue.  919 x 20480 x 32: gradients 35 us, statistics 14 us, the copies in pieces 7 us a pass.  16 bits have one
// plane, and two pieces of dl: 20480 x 20480 x 32 bfloat16 gradients 286 us (205 with one piece), statistics 119 us -- the float32 ones'
// time, it is the exponentials'; C = 128 617 (454) and 150 us.
#include "linear_ce.h"

namespace mvs {

// E: what the planes hold.  PL planes, KS 64-byte (32-element) steps of k per plane.
template <typename E_, int PL_, int KS_>
struct Narrow {
    using E = E_;
    static constexpr int PL = PL_, KS = KS_;
    static constexpr int DL = PL == 3 ? 3 : 2;                   // pieces of dl
    static constexpr int CT = KS * 2;                            // 16-column tiles of the result
    static constexpr int MR = PL * KS >= 6 ? 32 : 64;            // rows of the moving operand per stage (two workgroups' stages fit a CU)
    static constexpr int RG = MR / 16, HALVES = MR / 32;
    static constexpr int ROWS_COPIES = PL * KS * RG, TRANS_COPIES = PL * HALVES * CT;      // of 1024 bytes: 16 rows of 64
    static constexpr int ROWS_B = ROWS_COPIES * 1024, TRANS_B = TRANS_COPIES * 1024;
};

__device__ __forceinline__ void mma_e(f32x4_t &c, u32x4_t a, u32x4_t b, bf16_t) { mma16(c, a, b, bf16_t()); }
__device__ __forceinline__ void mma_e(f32x4_t &c, u32x4_t a, u32x4_t b, f16_t) { mma16(c, a, b, f16_t()); }

// c += a b over planes, the smallest products first
template <typename E, int PL>
__device__ __forceinline__ void mma_planes(f32x4_t &c, const u32x4_t (&a)[PL], const u32x4_t (&b)[PL]) {
    if constexpr (PL == 3) {
        mma_e(c, a[2], b[0], E());
        mma_e(c, a[1], b[1], E());
        mma_e(c, a[0], b[2], E());
        mma_e(c, a[1], b[0], E());
        mma_e(c, a[0], b[1], E());
    }
    mma_e(c, a[0], b[0], E());
}

// c += a b for the pieces that dl is carried in: float32's three as above, 16-bit operands' two against their one plane
template <typename E, int PL, int DL>
__device__ __forceinline__ void mma_dl(f32x4_t &c, const u32x4_t (&a)[PL], const u32x4_t (&d)[DL]) {
    if constexpr (PL == 3) {
        mma_planes<E, PL>(c, a, d);
    } else {
        mma_e(c, a[0], d[1], E());
        mma_e(c, a[0], d[0], E());
    }
}

// LDS holds sub-tiles of rows of 64 bytes, two rows to a 128-byte line, the eight 16-byte chunks of a line exchanged by the line's
// low three bits: 16 rows' fragments (one chunk each) then spread over all banks.  A wave's copy is 16 rows.
__device__ __forceinline__ void narrow_copy16(const char *rows, int64_t ld, int64_t row0, int64_t last, int64_t at, unsigned lds_to) {
    const int lane = threadIdx.x & 63, line = lane >> 3, in = (lane & 7) ^ line;
    int64_t row = row0 + line * 2 + (in >> 2);
    row = row < last ? row : last;
    glds16(rows + row * ld + at + (in & 3) * 16, lds_to);
}
__device__ __forceinline__ int narrow_lane() {      // a lane's byte within a 16-row block of a sub-tile
    const int ln = threadIdx.x & 15, fk = (threadIdx.x & 63) >> 4;
    return (ln >> 1) * 128 + ((((ln & 1) * 4 + fk) ^ (ln >> 1)) * 16);
}
__device__ __forceinline__ u32x4_t narrow_frag(const char *sub, int block, int lane_at) {
    return *reinterpret_cast<const u32x4_t *>(sub + block * 1024 + lane_at);
}

template <typename X>
__device__ __forceinline__ void narrow_copy_rows(const NarrowOperand &o, int Cp, int64_t m0, unsigned to) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < (X::ROWS_COPIES + 3) / 4; ++i) {
        const int c = wave + i * 4;
        if (X::ROWS_COPIES % 4 != 0 && c >= X::ROWS_COPIES) break;
        const int sub = c / X::RG, rg = c % X::RG, plane = sub / X::KS, k = sub % X::KS;
        narrow_copy16(o.rows, (int64_t)X::PL * Cp * 2, m0 + rg * 16, o.count - 1, plane * Cp * 2 + k * 64, to + (unsigned)(c * 1024));
    }
}
template <typename X>
__device__ __forceinline__ void narrow_copy_trans(const NarrowOperand &o, int C, int64_t m0, unsigned to) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t mp = o.pitch;
#pragma unroll
    for (int i = 0; i < (X::TRANS_COPIES + 3) / 4; ++i) {
        const int c = wave + i * 4;
        if (X::TRANS_COPIES % 4 != 0 && c >= X::TRANS_COPIES) break;
        const int sub = c / X::CT, rg = c % X::CT, plane = sub / X::HALVES, half = sub % X::HALVES;
        narrow_copy16(o.trans, X::PL * mp * 2, rg * 16, C - 1, plane * mp * 2 + m0 * 2 + half * 64, to + (unsigned)(c * 1024));
    }
}

// the fixed rows n0 .. n0 + 31 of a wave as fragments; `keep`: lanes whose row counts (others hold zeros)
template <typename X>
__device__ __forceinline__ void narrow_fixed(const NarrowOperand &o, int Cp, int64_t row, bool keep, u32x4_t (&f)[X::KS][X::PL]) {
    const char *p = o.rows + (row < o.count ? row : o.count - 1) * ((int64_t)X::PL * Cp * 2) + ((threadIdx.x & 63) >> 4) * 16;
#pragma unroll
    for (int k = 0; k < X::KS; ++k)
#pragma unroll
        for (int q = 0; q < X::PL; ++q) {
            f[k][q] = *reinterpret_cast<const u32x4_t *>(p + q * Cp * 2 + k * 64);
            if (!keep) f[k][q] = u32x4_t{0, 0, 0, 0};
        }
}

// S of 32 moving rows (16-row blocks `block`, block + 1 of the stage) against the wave's 32 fixed rows
template <typename X>
__device__ __forceinline__ void narrow_first(const char *stage, int block, int lane_at, const u32x4_t (&fixed)[2][X::KS][X::PL], f32x4_t (&s)[2][2]) {
#pragma unroll
    for (int k = 0; k < X::KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4_t a[X::PL];
#pragma unroll
            for (int q = 0; q < X::PL; ++q) a[q] = narrow_frag(stage + (q * X::KS + k) * X::RG * 1024, block + i, lane_at);
#pragma unroll
            for (int j = 0; j < 2; ++j) mma_planes<typename X::E, X::PL>(s[i][j], a, fixed[j][k]);
        }
}

// eight values of a lane, as they lie, as a fragment of each of their pieces
template <typename E, int DL>
__device__ __forceinline__ void narrow_pieces(const f32x4_t &lo, const f32x4_t &hi, u32x4_t (&d)[DL]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        float v0 = w < 2 ? lo[w * 2] : hi[w * 2 - 4], v1 = w < 2 ? lo[w * 2 + 1] : hi[w * 2 - 3];
#pragma unroll
        for (int q = 0; q < DL; ++q) {
            d[q][w] = pack2(v0, v1, E());
            if (q + 1 < DL) {
                v0 -= low_of(d[q][w], E());
                v1 -= high_of(d[q][w], E());
            }
        }
    }
}

template <typename X>
__global__ __launch_bounds__(256) void narrow_stats_kernel(NarrowArgs a) {
    __shared__ __align__(1024) char lds[2][X::ROWS_B];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, lane_at = narrow_lane();
    NarrowOperand x = a.x;
    x.count = ce_count(a.kept_rows);
    const NarrowSplit split = narrow_split(x.count, a.w.count, kNarrowStatsSlots, true, false);
    if (blockIdx.x >= split.blocks_x * split.parts_x) return;
    const int64_t block = blockIdx.x % split.blocks_x, part = blockIdx.x / split.blocks_x;
    const int64_t n0 = block * kNarrowRows + wave * 32, m_begin = part * split.per_x;
    const int rows = (int)min(split.per_x, a.w.count - m_begin);
    const int64_t *targets = a.kept_rows.target;
    const unsigned base_lds = (unsigned)(uintptr_t)&lds[0][0];
    narrow_copy_rows<X>(a.w, a.Cp, m_begin, base_lds);
    // a negative scale is taken as its magnitude and negated rows: the largest logit is then that of the largest product
    const float scale2 = __builtin_fabsf(a.scale2);
    u32x4_t fixed[2][X::KS][X::PL];
    int target[2];
    float base[2], sum[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + j * 16 + ln;
        narrow_fixed<X>(x, a.Cp, n, true, fixed[j]);
        if (a.scale2 < 0.0f)
#pragma unroll
            for (int k = 0; k < X::KS; ++k)
#pragma unroll
                for (int q = 0; q < X::PL; ++q) fixed[j][k][q] ^= 0x80008000u;
        const int64_t t = (n < x.count ? targets[n] : -1) - m_begin;
        target[j] = t >= 0 && t < rows ? (int)t : -1;
        base[j] = -INFINITY;
        sum[j] = 0.0f;
    }
    int stage = 0;
    for (int m = 0; m < rows; m += X::MR, stage ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (m + X::MR < rows) narrow_copy_rows<X>(a.w, a.Cp, m_begin + m + X::MR, base_lds + (unsigned)((stage ^ 1) * X::ROWS_B));
#pragma unroll
        for (int half = 0; half < X::HALVES; ++half) {
            const int mh = m + half * 32;
            if (mh >= rows) break;
            f32x4_t s[2][2] = {};
            narrow_first<X>(lds[stage], half * 2, lane_at, fixed, s);
            const int m_lane = mh + (lane >> 4) * 4;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (__ballot((unsigned)(target[j] - mh) < 32u)) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (m_lane + (e >> 2) * 16 + (e & 3) == target[j]) a.own[n0 + j * 16 + ln] = s[e >> 2][j][e & 3] * scale2;
                }
                // (rows behind the table's last one repeat it: they do not raise the maximum)
                float top = s[0][j][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e >> 2][j][e & 3]);
                // (a lane whose logits are all -Inf sums to 0; Inf - Inf and NaN make the sum NaN)
                const float next = fmaxf(base[j], top == -INFINITY ? -INFINITY : top * scale2), low = next == -INFINITY ? 0.0f : next;
                float add = 0.0f;
                if (mh + 32 <= rows) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) add += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][j][e & 3], scale2, -low));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (m_lane + (e >> 2) * 16 + (e & 3) < rows) add += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][j][e & 3], scale2, -low));
                }
                sum[j] = __builtin_fmaf(sum[j], __builtin_amdgcn_exp2f(base[j] - low), add);
                base[j] = next;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float t = fmaxf(base[j], __shfl_xor(base[j], 16));
        t = fmaxf(t, __shfl_xor(t, 32));
        float r = sum[j] * __builtin_amdgcn_exp2f(base[j] - (t == -INFINITY ? 0.0f : t));
        r += __shfl_xor(r, 16);
        r += __shfl_xor(r, 32);
        const int64_t n = n0 + j * 16 + ln;
        if (lane < 16 && n < x.count) a.part[part * x.count + n] = make_float2(t, r);
    }
}

// statistics of a stage's moving rows (of_table), in LDS
struct NarrowRows {
    float lse[2][64], ratio[2][64];      // (lse: less the logarithm of the unit that dl is carried in)
    int target[2][64];
};

// OF_TABLE: fixed = table rows, moving = rows of x (statistics along m); else fixed = rows of x, moving = table rows
template <typename X, bool OF_TABLE>
__device__ __forceinline__ void narrow_grad(const NarrowArgs &a, const NarrowOperand &fix, const NarrowOperand &mov, int64_t block, int64_t part, int64_t per, float unit, float log_unit,
                                            char *lds, NarrowRows &row_stats) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, group = lane >> 4, lane_at = narrow_lane();
    const int64_t n0 = block * kNarrowRows + wave * 32, m_begin = part * per;
    const int rows = (int)min(per, mov.count - m_begin);      // (0: no row is kept; dW's sums are then zeros)
    const int64_t *targets = a.kept_rows.target, ignore = a.kept_rows.ignore;
    const unsigned base_lds = (unsigned)(uintptr_t)lds;
    auto copy = [&](int m, int stage) {
        const unsigned to = base_lds + (unsigned)(stage * (X::ROWS_B + X::TRANS_B));
        narrow_copy_rows<X>(mov, a.Cp, m_begin + m, to);
        narrow_copy_trans<X>(mov, a.C, m_begin + m, to + (unsigned)X::ROWS_B);
    };
    const float *ratios = a.factors + a.kept_rows.n;
    float lse_next = 0.0f, ratio_next = 0.0f;
    int target_next = -1;
    auto stats = [&](int m) {      // thread t < MR's row of the stage, loaded a stage ahead
        const int64_t row = m_begin + m + threadIdx.x;
        const bool kept = threadIdx.x < X::MR && m + (int)threadIdx.x < rows && ce_kept(targets[row], ignore);
        lse_next = kept ? a.lse2[row] - log_unit : 0.0f;
        ratio_next = kept ? ratios[row] : 0.0f;
        target_next = kept ? (int)(targets[row] >= 0 && targets[row] < fix.count ? targets[row] : -1) : -1;
    };
    if (rows > 0) copy(0, 0);
    if (OF_TABLE) stats(0);
    u32x4_t fixed[2][X::KS][X::PL];
    int target[2];
    float lse[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + j * 16 + ln, t = !OF_TABLE && n < fix.count ? targets[n] : 0;
        const bool kept = OF_TABLE || (n < fix.count && ce_kept(t, ignore));
        // (whatever an ignored row holds, its S are 0 and its exponentials those of -Inf)
        narrow_fixed<X>(fix, a.Cp, n, kept, fixed[j]);
        lse[j] = OF_TABLE ? 0.0f : kept ? a.lse2[n] - log_unit : INFINITY;
        target[j] = OF_TABLE ? (int)n : kept && t >= m_begin && t - m_begin < rows ? (int)(t - m_begin) : -1;
    }
    f32x4_t out[X::CT][2] = {};
    int stage = 0;
    for (int m = 0; m < rows; m += X::MR, stage ^= 1) {
        if (OF_TABLE && threadIdx.x < X::MR) {      // (last read two stages ago, a barrier in between)
            row_stats.lse[stage][threadIdx.x] = lse_next;
            row_stats.ratio[stage][threadIdx.x] = ratio_next;
            row_stats.target[stage][threadIdx.x] = target_next;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (m + X::MR < rows) {
            copy(m + X::MR, stage ^ 1);
            if (OF_TABLE) stats(m + X::MR);
        }
        const char *tile = lds + stage * (X::ROWS_B + X::TRANS_B), *trans = tile + X::ROWS_B;
#pragma unroll
        for (int half = 0; half < X::HALVES; ++half) {
            const int mh = m + half * 32;
            if (mh >= rows) break;
            f32x4_t s[2][2] = {};
            narrow_first<X>(tile, half * 2, lane_at, fixed, s);
            if (OF_TABLE) {
                // what the 32 rows need beyond the exponential: nothing (factor 1 each, no target among this wave's columns), or all of it
                const int mine = half * 32 + (lane & 31);
                const float my_ratio = row_stats.ratio[stage][mine];
                const bool plain = !__ballot(my_ratio != 1.0f || (unsigned)(row_stats.target[stage][mine] - (int)n0) < 32u);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int at = half * 32 + i * 16 + group * 4;
                    const f32x4_t l4 = *reinterpret_cast<const f32x4_t *>(&row_stats.lse[stage][at]);
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[i][j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j][r], a.scale2, -l4[r]));
                }
                if (!plain)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = half * 32 + i * 16 + group * 4;
                        const f32x4_t r4 = *reinterpret_cast<const f32x4_t *>(&row_stats.ratio[stage][at]);
                        const u32x4_t t4 = *reinterpret_cast<const u32x4_t *>(&row_stats.target[stage][at]);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                float d = s[i][j][r];
                                if ((int)t4[r] == target[j]) d -= unit;
                                s[i][j][r] = r4[r] == 0.0f ? 0.0f : d * r4[r];      // (an ignored row's S may be anything)
                            }
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[i][j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][j][r], a.scale2, -lse[j]));
                    const int d = target[j] - mh;
                    if (__ballot((unsigned)d < 32u)) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) if (d == i * 16 + group * 4 + r) s[i][j][r] -= unit;
                    }
                }
                if (mh + 32 > rows) {
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (mh + i * 16 + group * 4 + r >= rows) s[i][0][r] = s[i][1][r] = 0.0f;
                }
            }
            u32x4_t d[2][X::DL];
#pragma unroll
            for (int j = 0; j < 2; ++j) narrow_pieces<typename X::E, X::DL>(s[0][j], s[1][j], d[j]);
#pragma unroll
            for (int c = 0; c < X::CT; ++c) {
                u32x4_t f[X::PL];
#pragma unroll
                for (int q = 0; q < X::PL; ++q) f[q] = narrow_frag(trans + (q * X::HALVES + half) * X::CT * 1024, c, lane_at);
#pragma unroll
                for (int j = 0; j < 2; ++j) mma_dl<typename X::E, X::PL, X::DL>(out[c][j], f, d[j]);
            }
        }
    }
    float *sums = OF_TABLE ? a.sums_w : a.sums_x;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int64_t n = n0 + j * 16 + ln;
        if (n >= fix.count) continue;
#pragma unroll
        for (int c = 0; c < X::CT; ++c) {
            const int col = c * 16 + group * 4;
            if (col < a.C) *reinterpret_cast<f32x4_t *>(sums + (part * fix.count + n) * a.ld_sums + col) = out[c][j];
        }
    }
}

// One launch for both gradients: the workgroups of dx, then those of dW.
template <typename X>
__global__ __launch_bounds__(256, 2) void narrow_grad_kernel(NarrowArgs a, float unit, float log_unit) {
    __shared__ __align__(1024) char lds[2 * (X::ROWS_B + X::TRANS_B)];
    __shared__ NarrowRows row_stats;
    NarrowOperand x = a.x;
    x.count = ce_count(a.kept_rows);
    const NarrowSplit split = narrow_split(x.count, a.w.count, kNarrowGradSlots, a.sums_x != nullptr, a.sums_w != nullptr);
    const int64_t id = blockIdx.x, groups_x = split.blocks_x * split.parts_x, of_table = id - groups_x;
    if (of_table < 0)
        narrow_grad<X, false>(a, x, a.w, id % split.blocks_x, id / split.blocks_x, split.per_x, unit, log_unit, lds, row_stats);
    else if (of_table < split.blocks_w * split.parts_w)
        narrow_grad<X, true>(a, a.w, x, of_table % split.blocks_w, of_table / split.blocks_w, split.per_w, unit, log_unit, lds, row_stats);
}

// Writes what the other kernels read of x (blockIdx.y = 0) and of the table (1): the rows in pieces and their transpose, 64 rows per
// workgroup.  Backward: blockIdx.y = 2 works out the rows' factors (one workgroup).
template <typename T, typename E, int PL>
__global__ __launch_bounds__(256) void narrow_prepare_kernel(NarrowArgs a) {
    __shared__ T tile[64][128 + 2];
    __shared__ float tops[4];
    const int tid = threadIdx.x;
    if (blockIdx.y == 2) {
        if (a.reduction != 0) ce_factors(a.kept_rows, a.grad_loss, a.kept, a.reduction, a.factors, (int64_t)blockIdx.x * 256 + tid, (int64_t)gridDim.x * 256, tops);
        else if (blockIdx.x == 0) ce_factors(a.kept_rows, a.grad_loss, a.kept, a.reduction, a.factors, tid, 256, tops);
        return;
    }
    const NarrowOperand &o = blockIdx.y ? a.w : a.x;
    const int64_t r0 = (int64_t)blockIdx.x * 64, mp = o.pitch, count = blockIdx.y ? o.count : ce_count(a.kept_rows);
    if (r0 >= count || (!o.write_rows && !o.trans)) return;
    const T *source = static_cast<const T *>(o.source);
    const int here = (int)min((int64_t)64, count - r0);
    const int lane = tid & 31, row = tid >> 5;      // 32 columns x 8 rows at a time
    for (int c = lane; c < a.C; c += 32) {
        T v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int r = row + u * 8;
            if (r < here) v[u] = source[(blockIdx.y ? r0 + r : ce_original(a.kept_rows, r0 + r)) * a.C + c];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) tile[row + u * 8][c] = row + u * 8 < here ? v[u] : from_float<T>(0.0f);
    }
    __syncthreads();
    if (o.write_rows) {
        E *rows = reinterpret_cast<E *>(o.rows);
        for (int c = lane; c < a.Cp; c += 32)
            for (int r = row; r < here; r += 8) {
                E p[PL];
                pieces_of<E, PL>(c < a.C ? tile[r][c] : from_float<T>(0.0f), p);
#pragma unroll
                for (int q = 0; q < PL; ++q) rows[((r0 + r) * PL + q) * a.Cp + c] = p[q];
            }
    }
    if (o.trans) {
        E *trans = reinterpret_cast<E *>(o.trans);
        const int place = tid & 63, r = (place & 32) + ((place >> 3) & 3) * 4 + (place & 3) + ((place & 4) << 2);
        // (ignored rows of x as zeros, whatever they hold)
        const bool keep = r < here && (blockIdx.y || ce_kept(a.kept_rows.target[r0 + r], a.kept_rows.ignore));
        for (int c = tid >> 6; c < a.C; c += 4) {
            E p[PL];
            pieces_of<E, PL>(keep ? tile[r][c] : from_float<T>(0.0f), p);
#pragma unroll
            for (int q = 0; q < PL; ++q) trans[((int64_t)c * PL + q) * mp + r0 + place] = p[q];
        }
    }
}

// both gradients from the parts' sums: workgroups of dx, then of dW
template <typename T>
__global__ __launch_bounds__(256) void narrow_finish_kernel(NarrowArgs a, int64_t groups_x) {
    const int64_t id = group_of(), count = ce_count(a.kept_rows);
    const NarrowSplit split = narrow_split(count, a.w.count, kNarrowGradSlots, a.sums_x != nullptr, a.sums_w != nullptr);
    if (id < groups_x)
        ce_finish<T, true>(a.sums_x, split.parts_x, a.x.count, count, a.kept_rows.place, a.C, a.ld_sums, a.factors, a.factor, static_cast<T *>(a.grad_x), id);
    else
        ce_finish<T, false>(a.sums_w, split.parts_w, a.w.count, a.w.count, (const int *)nullptr, a.C, a.ld_sums, a.factors + 2 * a.x.count, a.factor,
                            static_cast<T *>(a.grad_w), id - groups_x);
}

template <typename T, typename E, int PL>
static void narrow_prepare(const NarrowArgs &a, bool backward, hipStream_t st) {
    const int64_t most = a.x.count > a.w.count ? a.x.count : a.w.count;
    hipLaunchKernelGGL((narrow_prepare_kernel<T, E, PL>), dim3((unsigned)ceil_div(most, 64), backward ? 3 : 2), dim3(256), 0, st, a);
}

template <typename X>
static void narrow_stats(const NarrowArgs &a, hipStream_t st) {
    const int64_t groups = narrow_most(ceil_div(a.x.count, kNarrowRows), a.w.count, kNarrowStatsSlots);
    hipLaunchKernelGGL((narrow_stats_kernel<X>), dim3((unsigned)groups), dim3(256), 0, st, a);
}
template <typename X, typename T>
static void narrow_grads(const NarrowArgs &a, hipStream_t st) {
    const int64_t bx = a.sums_x ? ceil_div(a.x.count, kNarrowRows) : 0, bw = a.sums_w ? ceil_div(a.w.count, kNarrowRows) : 0;
    const int64_t groups = narrow_most(bx, a.w.count, kNarrowGradSlots) + narrow_most(bw, a.x.count, kNarrowGradSlots);
    hipLaunchKernelGGL((narrow_grad_kernel<X>), dim3((unsigned)groups), dim3(256), 0, st, a, GradUnit<T>::value, GradUnit<T>::log2);
}

// f(X()) for the planes and the 32-element steps of a row
template <typename E, int PL, typename F>
static void narrow_steps(int ks, F f) {
    if (ks == 1) f(Narrow<E, PL, 1>());
    else if (ks == 2) f(Narrow<E, PL, 2>());
    else if constexpr (PL == 1) {
        if (ks == 3) f(Narrow<E, PL, 3>());
        else f(Narrow<E, PL, 4>());
    }
}

int ce_narrow_forward(int dtype, const NarrowArgs &a, hipStream_t st) {
    const int ks = a.Cp / 32;
    auto stats = [&](auto x) { narrow_stats<decltype(x)>(a, st); };
    const bool prepare = a.x.write_rows || a.w.write_rows;
    if (dtype == MVS_DTYPE_F32) {
        narrow_prepare<float, bf16_t, 3>(a, false, st);
        narrow_steps<bf16_t, 3>(ks, stats);
    } else if (dtype == MVS_DTYPE_BF16) {
        if (prepare) narrow_prepare<bf16_t, bf16_t, 1>(a, false, st);
        narrow_steps<bf16_t, 1>(ks, stats);
    } else {
        if (prepare) narrow_prepare<f16_t, f16_t, 1>(a, false, st);
        narrow_steps<f16_t, 1>(ks, stats);
    }
    return check_launch("mvs_linear_ce_fwd");
}

int ce_narrow_backward(int dtype, const NarrowArgs &a, hipStream_t st) {
    const int ks = a.Cp / 32;
    const int64_t quads = a.ld_sums / 4, fx = a.sums_x ? ceil_div(a.x.count * quads, 256) : 0, fw = a.sums_w ? ceil_div(a.w.count * quads, 256) : 0;
    const dim3 finish = grid_of(fx + fw);
    if (dtype == MVS_DTYPE_F32) {
        narrow_prepare<float, bf16_t, 3>(a, true, st);
        narrow_steps<bf16_t, 3>(ks, [&](auto x) { narrow_grads<decltype(x), float>(a, st); });
        hipLaunchKernelGGL((narrow_finish_kernel<float>), finish, dim3(256), 0, st, a, fx);
    } else if (dtype == MVS_DTYPE_BF16) {
        narrow_prepare<bf16_t, bf16_t, 1>(a, true, st);
        narrow_steps<bf16_t, 1>(ks, [&](auto x) { narrow_grads<decltype(x), bf16_t>(a, st); });
        hipLaunchKernelGGL((narrow_finish_kernel<bf16_t>), finish, dim3(256), 0, st, a, fx);
    } else {
        narrow_prepare<f16_t, f16_t, 1>(a, true, st);
        narrow_steps<f16_t, 1>(ks, [&](auto x) { narrow_grads<decltype(x), f16_t>(a, st); });
        hipLaunchKernelGGL((narrow_finish_kernel<f16_t>), finish, dim3(256), 0, st, a, fx);
    }
    return check_launch("mvs_linear_ce_bwd");
}

}  // namespace mvs
