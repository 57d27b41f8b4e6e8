// Softmax cross entropy of rows against a large table, without the logits:  l = scale x W^T,  loss_n = lse(l_n) - l_n[t_n].
//
//   forward    a tile of logits lives in the matrix cores' accumulators and leaves as one (max, sum of exponentials) per row and
//              tile; a second launch joins a row's tiles.  2 N V C operations, (N + V) C elements read.
//   backward   dl = (p - 1[t]) g needs the logits again: a piece of the table at a time, one launch forms the tile's logits once more
//              and writes dl, rounded to the operands' type; two products follow, dx += dl W and dW = dl^T x.  6 N V C operations: 8
//              in all, of which 6 are the definition's and 2 buy the N V logits not being kept.
//              A piece is 2^26 / N rows of the table: 16-bit dl is then 128 MB, which stays in the last-level cache, float32 256 MB,
//              with a dl^T of that size beside it where the products need one.  float32 in pieces takes 2^27 / N rows, 805 MB in
//              three planes: its products want a full chip more than the cache.  256 rows at the least, so that beyond 2^18 rows of x
//              dl grows with N.
//
// All four products are one kernel shape, C[m][n] = sum_k A[m][k] B[n][k].  A workgroup owns a BM x BN tile and walks k in 128-byte
// steps: both operands go from memory to LDS by DMA, two stages, the 16-byte chunks of a row exchanged by a few bits of its number so
// that what a wave reads spreads over the banks.  An operand whose rows run along k lies there as BM rows of 128 bytes, a lane's 16
// bytes are one 16x16x32 fragment (16 bits) or four 16x16x4 ones (float32: lane group g holds k = 4 g + j for the j-th, on both
// sides).  Of 16 bits, an operand whose rows run along the tile -- W in dx, x and dl in dW -- lies there as 64 rows of k and is read
// by columns (ds_read_b64_tr_b16), so nothing is transposed in memory: against a pass that transposed W and x and a dl^T beside dl,
// the backward pass of 583 x 49999 x 768 float16 takes 229 instead of 297 us, of 8192 x 64000 x 2048 bfloat16 5.30 instead of 5.64 ms.
// float32, rows with factors of their own (reduction 'none') and rows that fill no more than one tile have those transposes.
// More than 256 float32 rows are carried as three bfloat16 pieces each (pieces_t): the same tiles, over six times the steps of k, at
// 205 to 217 TFLOP/s of float32 products where the float32 matrix instructions reach 85 to 135.
// m runs over table rows or channels, n over the rows of x or of W: a lane of the accumulator then holds four consecutive m of one
// n, so a row's softmax statistics reduce within the lane first, and results leave as vectors.
//
// Bound by the matrix cores: 256 x 256 tiles reach 1340 TFLOP/s in the statistics of 8192 x 64000 x 2048 bfloat16 and 1250 in its
// products (a library product of those operands 1400), half of what the cores could issue at 2.4 GHz.
//
// Numbers: sums, statistics and exponentials in float32, exponents in base 2 (one rounding of scale * log2 e per logit, the same
// one in both passes, so a row's p sum to one).  16-bit dl: float16 carries it times 2^14 (|p - 1| <= 1: no overflow, and p down to
// 4e-9 keeps a normal number's precision), the row's gradient factor is applied after the product in float32 (dx) or, relative to
// the largest one, before the rounding (dW) -- 1 / N of a mean never reaches a 16-bit number.
// The tiles round dl to the operands' type: of two pieces the two products would take their 6.5 ms twice, of 13 in all (8192 x 128000 x
// 2048 bfloat16), where the gradients are 0.0020 of their norm from the exact ones and rounding the results alone makes it 0.0017.
// Few rows keep it in float32, narrow ones in two pieces: there it is little beside what is read.
#include <type_traits>

#include "linear_ce.h"

namespace mvs {

// An element of a float32 operand that is carried as three bfloat16 pieces, a plane each: the products are six of the nine piece
// products (the others are below 2^-24 of it), one after the other along k, the smallest first.
struct pieces_t { unsigned short bits; };
template <typename T> constexpr bool kPieces = std::is_same_v<T, pieces_t>;
template <typename T> struct Given { using type = T; };      // what the caller has
template <> struct Given<pieces_t> { using type = float; };
__device__ __forceinline__ void mma16(f32x4_t &c, u32x4_t a, u32x4_t b, pieces_t) { mma16(c, a, b, bf16_t()); }
constexpr int kPairs = 6;
constexpr unsigned kPieceOfA = 0x001012, kPieceOfB = 0x010210;      // of pair 0, 1, .. from the lowest four bits on

// AHEAD: a wave reads its fragments half a step ahead.  One workgroup of 8 waves per CU needs it; two of 4 waves hide each other's
// reads and are slower with it (8192 x 128000 x 2048 bfloat16 forward: 256 x 256 tiles 3.63 -> 3.52 ms, 128 x 128 4.26 -> 4.70 ms).
// LATE: the copies of a later stage are issued behind the products that follow the barrier, not before them.
template <int BM_, int BN_, int WM_, int WN_, bool AHEAD_, bool LATE_ = false>
struct Tile {
    static constexpr bool AHEAD = AHEAD_, LATE = LATE_;
    static constexpr int BM = BM_, BN = BN_, WAVES_M = WM_, WAVES_N = WN_, WAVES = WM_ * WN_, THREADS = 64 * WAVES;
    static constexpr int TM = BM / WAVES_M / 16, TN = BN / WAVES_N / 16;
    static constexpr int STAGE = (BM + BN) * kRowBytes;
    static constexpr int COPIES = (BM + BN) / 8;                 // wave-wide copies of 8 rows
    static constexpr int PER_WAVE = (COPIES + WAVES - 1) / WAVES;
};

// A lane's 16 bytes at base + offset -> LDS byte address `to` + 16 * lane (the copy of glds16 with a wave's base in scalar registers,
// which the vector unit may have written just before: five instructions' wait).
__device__ __forceinline__ void copy16(const char *base, unsigned offset, unsigned to) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 2\n\t"
                 "global_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(offset), "s"(base), "s"(to)
                 : "memory");
}

// Four rows of 16 elements, 16 bits each: lane 4 r + q of a group of 16 points at elements 4 q .. 4 q + 3 of row r, lane i gets the
// column i.
__device__ __forceinline__ uint2 read_columns(const char *at) {
    typedef short four_t __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) four_t *)(uintptr_t)(unsigned)(uintptr_t)at));
}

// One operand in LDS: `SIDE` tile rows of 128 bytes of k -- or, ALONG (16 bits), 64 rows of k of SIDE elements, as a matrix has them whose
// rows run along the tile: its fragments are read as columns.  The 16-byte chunks of a row are exchanged by a few bits of its number,
// so that what a wave reads at once lies in different banks.
template <int SIDE, bool ALONG>
struct Stage {
    static constexpr bool COLUMNS = ALONG;
    static constexpr int ROW = ALONG ? 2 * SIDE : kRowBytes, CHUNKS = ROW / 16, ROWS = 64 / CHUNKS;      // (ROWS: of one copy of 1 KiB)
    static __device__ __forceinline__ int exchange(int row) { return ALONG ? ((row & 3) | (row >> 1 & 4)) * 2 : row & 7; }
    static __device__ __forceinline__ int row_of(int copy, int lane) { return copy * ROWS + lane / CHUNKS; }
    // byte offset, from the tile's corner, of what lane `lane` of copy `copy` moves; beyond the matrix' last tile row or column: that again
    static __device__ __forceinline__ unsigned offset(const Operand &o, int64_t tile0, int copy, int lane) {
        const int row = row_of(copy, lane), chunk = (lane % CHUNKS) ^ exchange(row);
        if (ALONG) return (unsigned)row * (unsigned)o.ld + (unsigned)min((int64_t)chunk * 16, o.ld - 16 - tile0 * 2);
        return (unsigned)min((int64_t)row, o.rows - 1 - tile0) * (unsigned)o.ld + chunk * 16;
    }
};

// acc[tm][tn] += the tile (m0, n0) of A B^T over the 128-byte steps first .. first + steps - 1 of k (16 bits: 64 elements).  A_ALONG,
// B_ALONG: that operand is given with k along its rows, [k][m] or [k][n].  The steps are walked backward: the one that may end behind
// the last row of k is then the first, and the only copy that has to look.
template <typename T, typename X, bool A_ALONG = false, bool B_ALONG = false>
__device__ __forceinline__ void tile_product(const Operand &a, const Operand &b, int64_t m0, int64_t n0, int first, int steps, char *lds,
                                             f32x4_t (&acc)[X::TM][X::TN]) {
    static_assert((!A_ALONG && !B_ALONG) || sizeof(T) == 2, "columns are read of 16-bit elements");
    using SA = Stage<X::BM, A_ALONG>;
    using SB = Stage<X::BN, B_ALONG>;
    if (steps <= 0) return;
    const int total = kPieces<T> ? kPairs * steps : steps;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / X::WAVES_N, wn = wave % X::WAVES_N;
    const unsigned lds_base = (unsigned)(uintptr_t)lds;
    // copy c moves 1 KiB of the stage, A's and then B's
    constexpr int COPIES_A = X::BM / 8, PER_A = COPIES_A / X::WAVES;
    static_assert(COPIES_A % X::WAVES == 0 && X::COPIES % X::WAVES == 0, "whole copies per wave, of one operand each");
    const int64_t last = first + steps - 1;
    const char *base_a = a.p + (A_ALONG ? last * 64 * a.ld + m0 * 2 : m0 * a.ld + last * kRowBytes);
    const char *base_b = b.p + (B_ALONG ? last * 64 * b.ld + n0 * 2 : n0 * b.ld + last * kRowBytes);
    unsigned offset[X::PER_WAVE];
#pragma unroll
    for (int i = 0; i < X::PER_WAVE; ++i) {
        const int c = wave + i * X::WAVES;
        offset[i] = i < PER_A ? SA::offset(a, m0, c, lane) : SB::offset(b, n0, c - COPIES_A, lane);
    }
    auto issue = [&](int stage, int i, unsigned from) {
        copy16(i < PER_A ? base_a : base_b, from, lds_base + (unsigned)(stage * X::STAGE + (wave + i * X::WAVES) * 1024));
    };
    const char *const start_a = base_a, *const start_b = base_b;
    int pair = 0, left = steps;
    if constexpr (kPieces<T>) {
        base_a += (kPieceOfA & 15) * a.plane;
        base_b += (kPieceOfB & 15) * b.plane;
    }
    auto retreat = [&](bool really) {
        if constexpr (kPieces<T>) {
            const bool over = really && left == 1;
            left = over ? steps : left - (really ? 1 : 0);
            pair += over ? 1 : 0;
            const char *next_a = start_a + (kPieceOfA >> 4 * pair & 15) * a.plane, *next_b = start_b + (kPieceOfB >> 4 * pair & 15) * b.plane;
            base_a = over ? next_a : base_a - (really ? (A_ALONG ? 64 * a.ld : kRowBytes) : 0);
            base_b = over ? next_b : base_b - (really ? (B_ALONG ? 64 * b.ld : kRowBytes) : 0);
        } else {
            base_a -= really ? (A_ALONG ? 64 * a.ld : kRowBytes) : 0;
            base_b -= really ? (B_ALONG ? 64 * b.ld : kRowBytes) : 0;
        }
    };
    auto copy = [&](int stage, bool more = true) {
#pragma unroll
        for (int i = 0; i < X::PER_WAVE; ++i) issue(stage, i, offset[i]);
        retreat(more);
    };
    auto copy_first = [&] {
#pragma unroll
        for (int i = 0; i < X::PER_WAVE; ++i) {
            const int c = wave + i * X::WAVES;
            const bool of_a = i < PER_A;
            unsigned from = offset[i];
            if (!kPieces<T> && (of_a ? A_ALONG : B_ALONG)) {      // (planes end in whole steps, rows of zeros)
                const Operand &o = of_a ? a : b;
                const int64_t behind = last * 64 + (of_a ? SA::row_of(c, lane) : SB::row_of(c - COPIES_A, lane)) - (o.rows - 1);
                if (behind > 0) from -= (unsigned)behind * (unsigned)o.ld;
            }
            issue(0, i, from);
        }
        retreat(total > 1);
    };
    const int frow = lane & 15, fk = lane >> 4;
    // a fragment: 16 tile rows x 64 bytes of k (half a step); a lane's 16 bytes are 8 k of one tile row, or four of each of its two reads
    const int col_row = 8 * fk + (frow >> 2), col_swz = Stage<X::BM, true>::exchange(col_row);
    auto fragment = [&](auto side, const char *at, int tile_row, int half) {
        using S = decltype(side);
        if constexpr (!S::COLUMNS) {
            return *reinterpret_cast<const u32x4_t *>(at + (tile_row + frow) * S::ROW + (((4 * half + fk) ^ (frow & 7)) * 16));
        } else {
            const char *from = at + (half * 32 + col_row) * S::ROW + (((tile_row / 8) ^ col_swz) * 16) + (frow & 3) * 8;
            const uint2 low = read_columns(from), high = read_columns(from + 4 * S::ROW);
            return u32x4_t{low.x, low.y, high.x, high.y};
        }
    };
    auto read = [&](int stage, int half, u32x4_t (&fa)[X::TM], u32x4_t (&fb)[X::TN]) {
        const char *at = lds + stage * X::STAGE;
#pragma unroll
        for (int i = 0; i < X::TM; ++i) fa[i] = fragment(SA(), at, wm * (X::BM / X::WAVES_M) + i * 16, half);
#pragma unroll
        for (int j = 0; j < X::TN; ++j) fb[j] = fragment(SB(), at + X::BM * kRowBytes, wn * (X::BN / X::WAVES_N) + j * 16, half);
    };
    auto multiply = [&](const u32x4_t (&fa)[X::TM], const u32x4_t (&fb)[X::TN], int first, int last) {
#pragma unroll
        for (int i = 0; i < X::TM; ++i)
            if (i >= first && i < last)
#pragma unroll
                for (int j = 0; j < X::TN; ++j) mma16(acc[i][j], fa[i], fb[j], T());
    };
    copy_first();
    if constexpr (X::AHEAD) {
        // The fragments of a half step are read while the matrix cores work on the half before it, across the stages' border too:
        //     read second half of s | first half's products, half of them | stage s + 1 has landed, s is read out | copy s + 2 into
        //     its place | the other half of them | read first half of s + 1 | second half's products
        // The waves of a SIMD meet at the barrier with products left, so that its matrix cores go on.  No branch in the loop: around
        // the reads it would have the compiler wait for them at once.  So the last two steps' copies read the last step's bytes
        // again, into a stage that is not read any more, and the last step's products stand behind the loop.
        constexpr int HALF = X::TM / 2;
        auto pace = [] {      // a fragment's read behind each of the first products (masks: matrix instructions, LDS reads)
#pragma unroll
            for (int i = 0; i < X::TM; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, A_ALONG ? 2 : 1, 0);
            }
#pragma unroll
            for (int j = 0; j < X::TN; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, B_ALONG ? 2 : 1, 0);
            }
        };
        u32x4_t a0[X::TM], b0[X::TN], a1[X::TM], b1[X::TN];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (total > 1) copy(1, total > 2);
        read(0, 0, a0, b0);
        int stage = 0;
        for (int s = 0; s + 1 < total; ++s, stage ^= 1) {
            read(stage, 1, a1, b1);
            multiply(a0, b0, 0, HALF);
            pace();
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();      // (waits for this wave's reads too: the stage may be overwritten)
            const bool more = s + 3 < total;
            if constexpr (X::LATE) {
                multiply(a0, b0, HALF, X::TM);
                __builtin_amdgcn_sched_barrier(0);
                copy(stage, more);
                __builtin_amdgcn_sched_barrier(0);
            } else {
                copy(stage, more);
                multiply(a0, b0, HALF, X::TM);
            }
            read(stage ^ 1, 0, a0, b0);
            multiply(a1, b1, 0, X::TM);
            pace();
            if constexpr (X::LATE) __builtin_amdgcn_sched_barrier(0);
        }
        read(stage, 1, a1, b1);
        multiply(a0, b0, 0, X::TM);
        multiply(a1, b1, 0, X::TM);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the copies of the last steps, before LDS is used for something else
    } else {
        for (int s = 0; s < total; ++s) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();                         // stage s has landed for everybody, and nobody reads the other one any more
            if (s + 1 < total) copy((s + 1) & 1);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                u32x4_t fa[X::TM], fb[X::TN];
                read(s & 1, half, fa, fb);
                multiply(fa, fb, 0, X::TM);
            }
        }
    }
}

// Which tile, and which of the parts that k is cut into, a workgroup owns.  The list is part by part, within it 8 m-tiles wide columns
// of the grid; the XCDs take consecutive runs of it (each has its own L2), so that the tiles an XCD works on share rows of both
// operands.  False for a workgroup that none is left for (fewer tiles than the host could tell).
__device__ __forceinline__ bool tile_of(int64_t id, int64_t tiles_m, int64_t tiles_n, int64_t parts, int64_t &tm, int64_t &tn, int64_t &part) {
    const int64_t tiles = tiles_m * tiles_n, total = tiles * parts;
    if (id >= total) return false;
    const int64_t per = total >> 3, extra = total & 7, xcd = id & 7;
    int64_t at = xcd * per + (xcd < extra ? xcd : extra) + (id >> 3);
    part = at / tiles;
    at -= part * tiles;
    const int64_t band = at / (8 * tiles_n), wide = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8, in = at - band * 8 * tiles_n;
    // (one number for the workgroup, in scalar registers, where the copies' bases come from it)
    tm = __builtin_amdgcn_readfirstlane((int)(band * 8 + in % wide));
    tn = __builtin_amdgcn_readfirstlane((int)(in / wide));
    part = __builtin_amdgcn_readfirstlane((int)part);
    return true;
}
__device__ __forceinline__ bool tile_of(int64_t id, int64_t tiles_m, int64_t tiles_n, int64_t &tm, int64_t &tn) {
    int64_t part;
    return tile_of(id, tiles_m, tiles_n, 1, tm, tn, part);
}

// How many parts dx's product cuts k into, of `steps` in the first piece of the table: as many workgroups as one round of the chip takes
// (two of the small tiles per CU), at least 8 steps each.  Worked out alike on the device, which knows how many rows are kept.
constexpr int64_t kRound = 512;
__host__ __device__ inline int64_t ce_parts(int64_t count, int C, int64_t steps, bool big) {
    const int64_t tiles = ((C + 127) / 128) * ((count + 127) / 128);
    int64_t parts = big || tiles == 0 ? 1 : kRound / tiles;
    if (parts > steps / 8) parts = steps / 8;
    if (parts < 1) parts = 1;
    return (steps + (steps + parts - 1) / parts - 1) / ((steps + parts - 1) / parts);      // (as many as get work)
}

struct CeArgs {
    Operand w, x;                       // table piece and rows, padded along k
    int steps;                          // 128-byte steps of k
    int64_t v_total, v0, v_count;       // table; this piece
    int64_t tiles_m, tiles_n;           // (of all rows; the kernels take the kept ones')
    float scale2;                       // scale * log2 e
    CeRows rows;
    // forward
    float2 *part;                       // [tile_m][n]: max, sum
    float *own;                         // [n]: the target's logit (base 2)
    // backward
    const float *lse2, *ratio;
    void *dl, *dlt;                     // [n][ld_dl], [v][ld_dlt]; either may be NULL
    int64_t ld_dl, ld_dlt;
    int64_t dl_plane;                   // (pieces) bytes from a plane of dl to the next
    int dl_step;                        // dl has rows of zeros behind the last kept one, up to a multiple of this
};

// How far row t of the table lies beyond a lane's first, v_lane, where it is within the wave's rows (16 i + r: the lane's own are
// r = 0 .. 3), -1 elsewhere.  Few tiles hold a given row's target: the epilogues ask the whole wave once and compare element by
// element only there.
template <typename X>
__device__ __forceinline__ int target_ahead(int64_t t, int64_t v_lane) {
    const int64_t d = t - v_lane;
    return d >= 0 && d < X::TM * 16 && (d & 15) < 4 ? (int)d : -1;
}

template <typename T, typename X>
__global__ __launch_bounds__(X::THREADS) void ce_stats_kernel(CeArgs a) {
    extern __shared__ __align__(1024) char lds[];
    const int64_t rows = ce_count(a.rows);
    int64_t tm, tn;
    if (!tile_of(group_of(), a.tiles_m, (rows + X::BN - 1) / X::BN, tm, tn)) return;
    Operand x = a.x;
    x.rows = rows;
    const int64_t m0 = tm * X::BM, n0 = tn * X::BN;
    f32x4_t acc[X::TM][X::TN] = {};
    tile_product<T, X>(a.w, x, m0, n0, 0, a.steps, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / X::WAVES_N, wn = wave % X::WAVES_N;
    const int64_t v_lane = m0 + wm * (X::BM / X::WAVES_M) + (lane >> 4) * 4;
    // rows of the table from a lane's first to the table's end: all of a tile's but where the table ends in it
    const int there = (int)min(a.v_total - v_lane, (int64_t)X::BM);
    const bool ends = m0 + X::BM > a.v_total;
    float2 stat[X::TN];
#pragma unroll
    for (int j = 0; j < X::TN; ++j) {
        const int64_t n = n0 + wn * (X::BN / X::WAVES_N) + j * 16 + (lane & 15);
        const int64_t t = n < rows ? a.rows.target[n] : -1;
        const int ahead = target_ahead<X>(t, v_lane);
        if (__any(ahead >= 0 && t < a.v_total)) {
#pragma unroll
            for (int i = 0; i < X::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (ahead == i * 16 + r && t < a.v_total) a.own[n] = acc[i][j][r] * a.scale2;
        }
        // (a lane's rows behind the table's end, and tiles of -Inf alone, sum to 0; Inf - Inf and NaN make the sum NaN)
        float top = -INFINITY, sum = 0.0f;
        auto statistics = [&](auto whole) {
            constexpr bool WHOLE = decltype(whole)::value;
            float high = -INFINITY, low = INFINITY;      // (the scale may be negative)
#pragma unroll
            for (int i = 0; i < X::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (WHOLE || i * 16 + r < there) {
                        high = fmaxf(high, acc[i][j][r]);
                        low = fminf(low, acc[i][j][r]);
                    }
            if (WHOLE || there > 0) top = fmaxf(high * a.scale2, low * a.scale2);
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < X::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], a.scale2, -base));
                    sum += WHOLE || i * 16 + r < there ? e : 0.0f;
                }
        };
        if (ends) statistics(std::false_type());
        else statistics(std::true_type());
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        stat[j] = make_float2(top, sum);
    }
    // the waves of one n range, through LDS
    float2 *s = reinterpret_cast<float2 *>(lds);
    __syncthreads();
    if (lane < 16)
#pragma unroll
        for (int j = 0; j < X::TN; ++j) s[wm * X::BN + wn * (X::BN / X::WAVES_N) + j * 16 + lane] = stat[j];
    __syncthreads();
    for (int c = threadIdx.x; c < X::BN; c += X::THREADS) {
        if (n0 + c >= rows) continue;
        float2 r = s[c];
#pragma unroll
        for (int w = 1; w < X::WAVES_M; ++w) {
            const float2 o = s[w * X::BN + c];
            const float top = fmaxf(r.x, o.x), base = top == -INFINITY ? 0.0f : top;
            r = make_float2(top, r.y * __builtin_amdgcn_exp2f(r.x - base) + o.y * __builtin_amdgcn_exp2f(o.x - base));
        }
        a.part[tm * a.rows.n + n0 + c] = r;
    }
}

// Joins a row's tiles (`tiles` == 0: the narrow kernels' parts): 16 rows x 16 tiles at a time per workgroup.
__global__ __launch_bounds__(256) void ce_join_kernel(const float2 *__restrict__ part, int64_t tiles, int64_t v_total, CeRows rows,
                                                      const float *__restrict__ own, float *__restrict__ lse2, float *__restrict__ loss) {
    const int64_t n = ce_count(rows), ld = tiles ? rows.n : n;
    if (!tiles) tiles = narrow_split(n, v_total, kNarrowStatsSlots, true, false).parts_x;
    __shared__ float2 s[256];
    const int64_t row = group_of() * 16 + (threadIdx.x & 15);
    float2 r = make_float2(-INFINITY, 0.0f);
    auto join = [](float2 p, float2 q) {
        const float top = fmaxf(p.x, q.x), base = top == -INFINITY ? 0.0f : top;
        return make_float2(top, p.y * __builtin_amdgcn_exp2f(p.x - base) + q.y * __builtin_amdgcn_exp2f(q.x - base));
    };
    if (row < n)
        for (int64_t t = threadIdx.x >> 4; t < tiles; t += 64) {      // (four loads under way)
            float2 p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u] = t + 16 * u < tiles ? part[(t + 16 * u) * ld + row] : make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int u = 0; u < 4; ++u) r = join(r, p[u]);
        }
    s[threadIdx.x] = r;
    __syncthreads();
    if (threadIdx.x < 16 && row < n) {
        for (int t = 1; t < 16; ++t) r = join(r, s[t * 16 + threadIdx.x]);
        const int64_t t = rows.target[row];
        const bool kept = ce_kept(t, rows.ignore), named = t >= 0 && t < v_total;
        const float l = r.x + __builtin_amdgcn_logf(r.y);      // (base 2)
        lse2[row] = kept && !named ? __uint_as_float(0x7fc00000u) : l;
        loss[ce_original(rows, row)] = !kept ? 0.0f : !named ? __uint_as_float(0x7fc00000u) : (l - own[row]) * kLn2;
    }
}

// sum of the rows' losses and how many were kept, in a fixed order, by one workgroup
__global__ __launch_bounds__(1024) void ce_total_kernel(const float *__restrict__ rows, const int64_t *__restrict__ target, int64_t n, int64_t ignore,
                                                        int reduction, float *__restrict__ loss, float *__restrict__ kept) {
    __shared__ double sums[16], counts[16];
    double sum = 0.0, count = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        sum += (double)rows[i];
        count += ce_kept(target[i], ignore) ? 1.0 : 0.0;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) { sum += __shfl_xor(sum, o); count += __shfl_xor(count, o); }
    if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = sum; counts[threadIdx.x >> 6] = count; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) { sum += sums[w]; count += counts[w]; }
        *kept = (float)count;
        if (reduction == 1) *loss = (float)(sum / count);
        if (reduction == 2) *loss = (float)sum;
    }
}

// ---- backward
__global__ __launch_bounds__(1024) void ce_factors_kernel(CeRows rows, const float *grad_loss, const float *kept, int reduction, float *factors) {
    __shared__ float tops[16];
    ce_factors(rows, grad_loss, kept, reduction, factors, (int64_t)blockIdx.x * 1024 + threadIdx.x, (int64_t)gridDim.x * 1024, tops);
}

// FLOATS: dl is left as float32 (few rows)
template <typename T, typename X, bool FLOATS = false>
__global__ __launch_bounds__(X::THREADS) void ce_grad_kernel(CeArgs a) {
    extern __shared__ __align__(1024) char lds[];
    const int64_t rows = ce_count(a.rows);
    int64_t tm, tn;
    if (!tile_of(blockIdx.x, a.tiles_m, (rows + X::BN - 1) / X::BN, tm, tn)) return;
    Operand x = a.x;
    x.rows = rows;
    const int64_t m0 = tm * X::BM, n0 = tn * X::BN;      // (m0 within the piece)
    f32x4_t acc[X::TM][X::TN] = {};
    tile_product<T, X>(a.w, x, m0, n0, 0, a.steps, lds, acc);
    constexpr float unit = GradUnit<T>::value;
    constexpr int PITCH = X::BN * (int)sizeof(T) + 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / X::WAVES_N, wn = wave % X::WAVES_N;
    const int m_lane = wm * (X::BM / X::WAVES_M) + (lane >> 4) * 4;
    const bool ends = m0 + X::BM > a.v_count;      // the piece ends in this tile
    const int64_t dl_rows = (rows + a.dl_step - 1) / a.dl_step * a.dl_step;
    __syncthreads();      // the stages have been read: LDS holds the transpose from here on
#pragma unroll
    for (int j = 0; j < X::TN; ++j) {
        const int nl = wn * (X::BN / X::WAVES_N) + j * 16 + (lane & 15);
        const int64_t n = n0 + nl;
        const int64_t t = n < rows ? a.rows.target[n] : 0;
        const bool kept = n < rows && ce_kept(t, a.rows.ignore);
        const float lse2 = kept ? a.lse2[n] - GradUnit<T>::log2 : 0.0f, ratio = kept ? a.ratio[n] : 0.0f;
#pragma unroll
        for (int i = 0; i < X::TM; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][r], a.scale2, -lse2));      // unit * p
        const int ahead = target_ahead<X>(t, a.v0 + m0 + m_lane);
        if (__any(ahead >= 0)) {
#pragma unroll
            for (int i = 0; i < X::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (ahead == i * 16 + r) acc[i][j][r] -= unit;
        }
        if (ends) {
#pragma unroll
            for (int i = 0; i < X::TM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (m0 + m_lane + i * 16 + r >= a.v_count) acc[i][j][r] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < X::TM; ++i) {
            const int64_t m = m0 + m_lane + i * 16;
            if constexpr (kPieces<T>) {
                Pack<bf16_t, 4> out[3];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bf16_t p[3];
                    pieces_of<bf16_t, 3>(kept ? acc[i][j][r] : 0.0f, p);
#pragma unroll
                    for (int q = 0; q < 3; ++q) out[q].v[r] = p[q];
                }
                if (n < dl_rows && m < a.ld_dl)
#pragma unroll
                    for (int q = 0; q < 3; ++q) put(static_cast<char *>(a.dl) + q * a.dl_plane + (n * a.ld_dl + m) * 2, out[q]);
            } else if constexpr (FLOATS) {
                const f32x4_t out = kept ? acc[i][j] : f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                if (n < dl_rows && m < a.ld_dl) *reinterpret_cast<f32x4_t *>(static_cast<float *>(a.dl) + n * a.ld_dl + m) = out;
            } else {
                Pack<T, 4> out;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float d = kept ? acc[i][j][r] : 0.0f;
                    out.v[r] = from_float<T>(d);
                    if (a.dlt) *reinterpret_cast<T *>(lds + (m_lane + i * 16 + r) * PITCH + nl * (int)sizeof(T)) = from_float<T>(kept ? d * ratio : 0.0f);
                }
                if (a.dl && n < dl_rows && m < a.ld_dl) *reinterpret_cast<Pack<T, 4> *>(static_cast<T *>(a.dl) + n * a.ld_dl + m) = out;
            }
        }
    }
    if (kPieces<T> || FLOATS || !a.dlt) return;
    __syncthreads();
    constexpr int PER16 = 16 / (int)sizeof(T), CHUNKS = X::BN / PER16;
    for (int c = threadIdx.x; c < X::BM * CHUNKS; c += X::THREADS) {
        const int ml = c / CHUNKS, nc = c % CHUNKS * PER16;
        if (m0 + ml < a.v_count && n0 + nc < a.ld_dlt)
            *reinterpret_cast<u32x4_t *>(static_cast<T *>(a.dlt) + (m0 + ml) * a.ld_dlt + n0 + nc) =
                *reinterpret_cast<const u32x4_t *>(lds + ml * PITCH + nc * (int)sizeof(T));
    }
}

// out[n][m] (+)= factor * sum_k A[m][k] B[n][k]
struct CeProduct {
    Operand a, b;
    int steps, first_steps; // of k, of the first piece's k
    int64_t m, n, tiles_m, tiles_n;
    float *sums;            // float32 sums [part][n][ld_sums] (added to if `add`), or NULL: `out` is written, k is not cut
    int64_t ld_sums;
    int add;
    void *out;              // [n][m] of T
    const float *top;       // `out` = sum * *top * factor
    float factor;
    const int *count;       // kept rows: n (sums) or the extent of k (out) is at most that; NULL: as given
};

template <typename T, typename X, bool A_ALONG, bool B_ALONG>
__global__ __launch_bounds__(X::THREADS) void ce_product_kernel(CeProduct a) {
    extern __shared__ __align__(1024) char lds[];
    if (a.count) {
        if (a.sums) {
            a.n = a.b.rows = *a.count;
            a.tiles_n = (a.n + X::BN - 1) / X::BN;
        } else {
            if (A_ALONG && !kPieces<T>) a.a.rows = *a.count;      // (dl, and x in pieces, have rows of zeros behind the last kept one)
            a.steps = (int)((*a.count * (int64_t)sizeof(T) + kRowBytes - 1) / kRowBytes);
        }
    }
    const int64_t parts = a.sums ? ce_parts(a.n, (int)a.m, a.first_steps, X::BM == 256) : 1;
    int64_t tm, tn, part;
    if (!tile_of(blockIdx.x, a.tiles_m, a.tiles_n, parts, tm, tn, part)) return;
    const int64_t m0 = tm * X::BM, n0 = tn * X::BN;
    const int each = (int)((a.steps + parts - 1) / parts), first = (int)part * each, steps = min(each, a.steps - first);
    f32x4_t acc[X::TM][X::TN] = {};
    tile_product<T, X, A_ALONG, B_ALONG>(a.a, a.b, m0, n0, first, steps, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / X::WAVES_N, wn = wave % X::WAVES_N;
    const float f = a.sums ? 1.0f : *a.top * a.factor;
#pragma unroll
    for (int j = 0; j < X::TN; ++j) {
        const int64_t n = n0 + wn * (X::BN / X::WAVES_N) + j * 16 + (lane & 15);
        if (n >= a.n) continue;
#pragma unroll
        for (int i = 0; i < X::TM; ++i) {
            const int64_t m = m0 + wm * (X::BM / X::WAVES_M) + i * 16 + (lane >> 4) * 4;
            if (m >= a.m) continue;
            if (a.sums) {      // (rows of ld_sums floats, a multiple of 4: the padding behind m may be written)
                f32x4_t *to = reinterpret_cast<f32x4_t *>(a.sums + (part * a.n + n) * a.ld_sums + m);
                *to = a.add ? *to + acc[i][j] : acc[i][j];
            } else {
                using O = typename Given<T>::type;
                O *to = static_cast<O *>(a.out) + n * a.m + m;
                Pack<O, 4> o;
#pragma unroll
                for (int r = 0; r < 4; ++r) o.v[r] = from_float<O>(acc[i][j][r] * f);
                if ((a.m & 3) == 0) put(to, o);
                else
                    for (int r = 0; r < 4; ++r) if (m + r < a.m) to[r] = o.v[r];
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void ce_finish_kernel(const float *sums, int64_t first_steps, bool big, CeRows rows, int C, int64_t ld, const float *g, float factor, T *out) {
    const int64_t count = ce_count(rows);
    ce_finish<T, true>(sums, ce_parts(count, C, first_steps, big), rows.n, count, rows.place, C, ld, g, factor, out, group_of());
}

// Moves the kept rows together (CeRows): a workgroup counts the kept rows before its `chunk`, its 16 waves those of their sixteenth,
// then number them (20480 rows: 6 us by 5 workgroups; one that walked them all took 12).
// `loss` (forward): the ignored rows' losses, 0.
__global__ __launch_bounds__(1024) void ce_together_kernel(const int64_t *__restrict__ target, int64_t n, int64_t ignore, int64_t chunk, int *__restrict__ map,
                                                           int *__restrict__ place, int64_t *__restrict__ kept_target, int *__restrict__ count, float *__restrict__ loss) {
    __shared__ int counts[16], before[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t first = blockIdx.x * chunk, per = chunk / 16, begin = min(n, first + wave * per), end = min(n, begin + per);
    int earlier = 0, mine = 0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < first; i += 1024) earlier += ce_kept(target[i], ignore) ? 1 : 0;
#pragma unroll 4
    for (int64_t i = begin + lane; i < end; i += 64) mine += ce_kept(target[i], ignore) ? 1 : 0;
#pragma unroll
    for (int o = 32; o; o >>= 1) { mine += __shfl_xor(mine, o); earlier += __shfl_xor(earlier, o); }
    if (lane == 0) { counts[wave] = mine; before[wave] = earlier; }
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < 16; ++w) { at += before[w] + (w < wave ? counts[w] : 0); all += before[w] + counts[w]; }
    if (threadIdx.x == 0 && first + chunk >= n) *count = all;
    for (int64_t i0 = begin; i0 < end; i0 += 256) {
        int64_t t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) t[u] = i0 + u * 64 + lane < end ? target[i0 + u * 64 + lane] : ignore;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = i0 + u * 64 + lane;
            const bool kept = ce_kept(t[u], ignore);
            const unsigned long long all_kept = __ballot(kept);
            if (kept) {
                const int to = at + __popcll(all_kept & ((1ull << lane) - 1));
                map[to] = (int)i;
                place[i] = to;
                kept_target[to] = t[u];
            } else if (i < end) {
                place[i] = -1;
                if (loss) loss[i] = 0.0f;
            }
            at += __popcll(all_kept);
        }
    }
}

// out[i][0 .. Cp) = in[map[i]][0 .. C), zeros, for the kept rows (all `n` where there is no map); VEC elements per access
template <typename T, int VEC>
__global__ __launch_bounds__(256) void ce_rows_kernel(const T *__restrict__ in, CeRows rows, int C, T *__restrict__ out, int Cp) {
    const int vecs = Cp / VEC;
    const int64_t i = group_of() * 256 + threadIdx.x, row = i / vecs;
    if (row >= ce_count(rows)) return;
    const int c = (int)(i - row * vecs) * VEC;
    Pack<T, VEC> v;
    if (c < C) v = *reinterpret_cast<const Pack<T, VEC> *>(in + ce_original(rows, row) * C + c);
    else
#pragma unroll
        for (int j = 0; j < VEC; ++j) v.v[j] = from_float<T>(0.0f);
    reinterpret_cast<Pack<T, VEC> *>(out)[i] = v;
}

// float32 rows (the kept ones) as three planes of bfloat16 pieces, padded with zeros to rows of Cp and to whole steps of rows
__global__ __launch_bounds__(256) void ce_pieces_kernel(const float *__restrict__ in, CeRows rows, int C, char *__restrict__ out, int Cp, int64_t plane) {
    const int vecs = Cp / 8;
    const int64_t i = group_of() * 256 + threadIdx.x, row = i / vecs, count = ce_count(rows);
    if (row >= ((count + 63) & ~(int64_t)63)) return;
    const int c = (int)(i - row * vecs) * 8;
    const float *from = in + (row < count ? ce_original(rows, row) : 0) * C + c;
    float v[8];
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
        if ((C & 3) == 0 && row < count && c + h < C) {
            const f32x4_t four = *reinterpret_cast<const f32x4_t *>(from + h);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[h + j] = four[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[h + j] = row < count && c + h + j < C ? from[h + j] : 0.0f;
        }
    }
    Pack<bf16_t, 8> o[3];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bf16_t p[3];
        pieces_of<bf16_t, 3>(v[j], p);
#pragma unroll
        for (int q = 0; q < 3; ++q) o[q].v[j] = p[q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) put(out + q * plane + i * 16, o[q]);
}

// ---- few rows (ce_few_rows): both gradients in one pass over the table
// With so few rows a product tile is mostly empty: bound by reading W and writing dW, once each.
// A thread owns VEC columns, keeps x (times the row's ratio) and dx of NR rows there in registers and walks 64 table rows:
//     dx[n] += dl[n][v] W[v],  dW[v] = sum_n dl[n][v] ratio_n x[n]
// Two rows against 32000 x 1024 bfloat16: 25 us for 131 MB; the tiles that form the logits before it read the table at 4.1 TB/s.
constexpr int kFewTable = 64;
// How many rows are few.  16 bits, 32000 x 1024: two rows 55 us against the tiles' 66, four 57, eight 68 (sixteen 145); 100000 x 2048 four
// 388 against 368.  float32, whose tiles need W^T: sixteen 172 against 242.
static int ce_few_rows(int es) { return es == 2 ? 4 : 16; }
struct CeFew {
    const void *w, *x;
    const float *dl;                    // (float32 whatever the operands are: it is little beside the table)
    int64_t count, ld_dl;               // table rows of the piece; elements per row of dl
    int n, C, Cp, threads;              // threads per table row, a power of two
    const float *ratio, *top;
    float factor;
    // (the logits formed here) what dl is made of
    const float *lse2;
    const int64_t *target;
    int64_t ignore, v0;                 // v0: the piece's first table row
    float scale2;
    float2 *part;                       // (statistics) [part]
    float *own;
    void *grad_w;                       // [count][C] or NULL
    float *sums;                        // [part][n][c4] or NULL
    int64_t c4;
    int add;
};

// A single row against BATCH table rows per `threads` threads (their columns of them in p): <w, x> for all of them.  `shares`: of one
// batch; two in turn, the barrier of the batch in between keeps them apart.
template <typename T, int VEC, int BATCH>
__device__ __forceinline__ void few_logits(const Pack<T, VEC> (&p)[BATCH], const float (&x)[VEC], int threads, float (&shares)[4][BATCH], float (&l)[BATCH]) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        l[u] = 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) l[u] = __builtin_fmaf(to_float(p[u].v[j]), x[j], l[u]);
    }
    for (int o = 1; o < threads && o < 64; o <<= 1)
#pragma unroll
        for (int u = 0; u < BATCH; ++u) l[u] += __shfl_xor(l[u], o);
    if (threads <= 64) return;
    const int wave = tid >> 6, waves = threads / 64, first = wave / waves * waves;      // (a row's threads are several waves)
    if ((tid & 63) == 0)
#pragma unroll
        for (int u = 0; u < BATCH; ++u) shares[wave][u] = l[u];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
        l[u] = shares[first][u];
        for (int q = 1; q < waves; ++q) l[u] += shares[first + q][u];
    }
}

// The statistics of a single float32 row whose columns a workgroup holds whole (32000 x 1024: forward 41 us, with tiles of which one
// row in 128 is real 79; 16-bit tiles are bound by reading the table, and faster: 23 us against 33).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void ce_one_stats_kernel(CeFew a) {
    constexpr int BATCH = 8;
    __shared__ float shares[2][4][BATCH], all[kFewTable];
    const int tid = threadIdx.x, col = (tid & (a.threads - 1)) * VEC, sub = tid / a.threads, subs = 256 / a.threads;
    const int64_t v0 = (int64_t)blockIdx.x * kFewTable;
    const int rows = (int)min((int64_t)kFewTable, a.count - v0);
    const bool here = col < a.Cp;
    Pack<T, VEC> px;
    float x[VEC];
    if (here) px = *reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.x) + col);
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = here ? to_float(px.v[j]) : 0.0f;
    const Pack<T, VEC> *w = reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.w) + v0 * a.Cp + col);
    const int stride = a.Cp / VEC;
    for (int b = 0; b * BATCH * subs < rows; ++b) {
        const int v = b * BATCH * subs + sub;
        Pack<T, VEC> p[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            if (here && v + u * subs < rows) p[u] = w[(int64_t)(v + u * subs) * stride];
            else
#pragma unroll
                for (int j = 0; j < VEC; ++j) p[u].v[j] = from_float<T>(0.0f);
        }
        float l[BATCH];
        few_logits<T, VEC, BATCH>(p, x, a.threads, shares[b & 1], l);
        if ((tid & (a.threads - 1)) == 0)
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (v + u * subs < rows) all[v + u * subs] = l[u] * a.scale2;
    }
    __syncthreads();
    if (tid >= 64) return;
    const int64_t t = a.target[0];
    const float l = tid < rows ? all[tid] : -INFINITY;
    if (tid < rows && t == v0 + tid) *a.own = l;
    float top = l;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    float sum = __builtin_amdgcn_exp2f(l - (top == -INFINITY ? 0.0f : top));
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o);
    if (tid == 0) a.part[blockIdx.x] = make_float2(top, sum);
}

// LOGITS: a single row whose columns a workgroup holds whole forms its logits here too, from the values that it has in registers for the
// products -- one read of the table instead of two, and no launch for dl.  (32000 x 1024: bfloat16 48 -> 40 us, float32 122 -> 64; two
// to four rows 54 -> 63 us, their sums across the lanes cost more than a tile's matrix instructions.)
template <typename T, int NR, int VEC, bool LOGITS>
__global__ __launch_bounds__(256) void ce_few_kernel(CeFew a) {
    static_assert(!LOGITS || NR == 1, "a single row");
    constexpr int BATCH = LOGITS ? 8 : 4;      // table rows of a thread under way
    __shared__ float d[LOGITS ? 1 : kFewTable][NR];
    __shared__ float shares[LOGITS ? 2 : 1][4][BATCH];
    __shared__ float joined[256][VEC];
    const int tid = threadIdx.x, col = (blockIdx.y * a.threads + (tid & (a.threads - 1))) * VEC, sub = tid / a.threads, subs = 256 / a.threads;
    const int64_t v0 = (int64_t)blockIdx.x * kFewTable;
    const int rows = (int)min((int64_t)kFewTable, a.count - v0);
    const bool here = col < a.Cp;
    float lse2 = 0.0f, ratio_w = 0.0f;
    int target = -1;
    bool kept = false;
    if constexpr (LOGITS) {
        const int64_t t = a.target[0];
        kept = ce_kept(t, a.ignore);
        if (kept) {
            lse2 = a.lse2[0];
            ratio_w = a.ratio[0];
            target = t - a.v0 >= v0 && t - a.v0 < v0 + rows ? (int)(t - a.v0 - v0) : -1;
        }
    } else for (int i = tid; i < kFewTable * NR; i += 256) {
        const int v = i / NR, r = i % NR;
        d[v][r] = v < rows && r < a.n ? a.dl[r * a.ld_dl + v0 + v] : 0.0f;
    }
    float x[NR][VEC], dx[NR][VEC];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        Pack<T, VEC> p;
        const float ratio = r >= a.n ? 0.0f : !LOGITS ? a.ratio[r] : kept ? 1.0f : 0.0f;      // (LOGITS: x itself)
        if (here && ratio != 0.0f) p = *reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.x) + (int64_t)r * a.Cp + col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            x[r][j] = here && ratio != 0.0f ? to_float(p.v[j]) * ratio : 0.0f;      // (an ignored row's values are not looked at)
            dx[r][j] = 0.0f;
        }
    }
    __syncthreads();
    const float f = a.grad_w ? *a.top * a.factor : 0.0f;
    const Pack<T, VEC> *w = reinterpret_cast<const Pack<T, VEC> *>(static_cast<const T *>(a.w) + v0 * a.Cp + col);
    const int stride = a.Cp / VEC;
    for (int b = 0; b * BATCH * subs < rows; ++b) {
        const int v = b * BATCH * subs + sub;
        Pack<T, VEC> p[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int row = v + u * subs;
            if (here && row < rows && (LOGITS || a.sums)) p[u] = w[(int64_t)row * stride];
            else
#pragma unroll
                for (int j = 0; j < VEC; ++j) p[u].v[j] = from_float<T>(0.0f);
        }
        float g[BATCH][NR];
        if constexpr (LOGITS) {
            float l[BATCH];
            few_logits<T, VEC, BATCH>(p, x[0], a.threads, shares[b & 1], l);
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                // (an ignored row has no gradient, whatever the table holds: a logit of 0 times Inf is NaN)
                const float e = kept ? __builtin_amdgcn_exp2f(__builtin_fmaf(l[u], a.scale2, -lse2)) : 0.0f;
                g[u][0] = v + u * subs == target ? e - 1.0f : e;
            }
        } else {
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
#pragma unroll
                for (int r = 0; r < NR; ++r) g[u][r] = v + u * subs < rows ? d[v + u * subs][r] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            const int row = v + u * subs;
            if (!here || row >= rows) break;
            float out[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) out[j] = 0.0f;
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float gw = LOGITS ? g[u][r] * ratio_w : g[u][r];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (a.sums) dx[r][j] = __builtin_fmaf(g[u][r], to_float(p[u].v[j]), dx[r][j]);
                    out[j] = __builtin_fmaf(gw, x[r][j], out[j]);
                }
            }
            if (a.grad_w && col < a.C) {      // (the padding's columns are nobody's)
                T *to = static_cast<T *>(a.grad_w) + (v0 + row) * a.C + col;
                Pack<T, VEC> o;
#pragma unroll
                for (int j = 0; j < VEC; ++j) o.v[j] = from_float<T>(out[j] * f);
                if (a.C % VEC == 0) put(to, o);
                else
                    for (int j = 0; j < VEC; ++j) if (col + j < a.C) to[j] = o.v[j];
            }
        }
    }
    if (!a.sums) return;
    for (int r = 0; r < a.n; ++r) {      // the threads of a column, in order
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NR; ++q)
            if (q == r)
#pragma unroll
                for (int j = 0; j < VEC; ++j) joined[tid][j] = dx[q][j];
        __syncthreads();
        if (sub == 0 && col < a.c4) {
            float s[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[j] = 0.0f;
            for (int q = 0; q < subs; ++q)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s[j] += joined[q * a.threads + tid][j];
            float *to = a.sums + ((int64_t)blockIdx.x * a.n + r) * a.c4 + col;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (col + j < a.c4) to[j] = a.add ? to[j] + s[j] : s[j];
        }
    }
}

// dx from many parts of few rows: 16 quads of columns x 16 shares of the parts per workgroup, the shares joined in order
template <typename T>
__global__ __launch_bounds__(256) void ce_few_finish_kernel(const float *__restrict__ sums, int parts, int n, int C, int64_t c4, const float *__restrict__ g,
                                                            float factor, T *__restrict__ out) {
    __shared__ f32x4_t shares[16][16];
    const int64_t quads = c4 / 4, i = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15), row = i / quads, step = n * quads;
    const int share = threadIdx.x >> 4;
    const f32x4_t *from = reinterpret_cast<const f32x4_t *>(sums) + i;
    f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row < n)
        for (int p = share; p < parts; p += 128) {
            f32x4_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (p + j * 16 < parts) v[j] = from[(p + j * 16) * step];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (p + j * 16 < parts) s += v[j];
        }
    shares[share][threadIdx.x & 15] = s;
    __syncthreads();
    if (share != 0 || row >= n) return;
    for (int q = 1; q < 16; ++q) s += shares[q][threadIdx.x];
    const float f = g[row];
    const int64_t c = (i - row * quads) * 4;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (c + r < C) out[row * C + c + r] = from_float<T>(f == 0.0f ? 0.0f : s[r] * f * factor);
}

// out[c][r] = in[r][c] for c < C and r < rows, zero for the other r < ld_out and for ignored rows.  64 x 64 tiles through LDS, moved
// VEC elements at a time on both sides (VEC > 1: ld_in, and C or its padding, reach whole vectors).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void ce_transpose_kernel(const T *__restrict__ in, CeRows rows, bool look, int C, int64_t ld_in, T *__restrict__ out,
                                                           int64_t ld_out) {
    constexpr int PITCH = 64 + 4 / (int)sizeof(T), PER = 64 / VEC;
    __shared__ T tile[64][PITCH];
    const int64_t r0 = (int64_t)blockIdx.x * 64, R = ce_count(rows);
    if (r0 >= R + 63) return;      // (nobody reads that far)
    const int c0 = blockIdx.y * 64;
    for (int i = threadIdx.x; i < 64 * PER; i += 256) {
        const int r = i / PER, c = i % PER * VEC;
        const int64_t row = r0 + r;
        Pack<T, VEC> v;
        if (row < R && c0 + c < ld_in && (!look || ce_kept(rows.target[row], rows.ignore))) v = *reinterpret_cast<const Pack<T, VEC> *>(in + row * ld_in + c0 + c);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) v.v[j] = from_float<T>(0.0f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) tile[r][c + j] = v.v[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * PER; i += 256) {
        const int c = i / PER, r = i % PER * VEC;
        if (c0 + c >= C || r0 + r >= ld_out) continue;
        Pack<T, VEC> v;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v.v[j] = tile[r + j][c];
        *reinterpret_cast<Pack<T, VEC> *>(out + (int64_t)(c0 + c) * ld_out + r0 + r) = v;
    }
}

// ---- host side
struct CePlan {
    int es;                          // element size
    bool pieces;                     // wide float32 rows in pieces (then 2)
    bool narrow;                     // linear_ce_narrow.hip
    int Cp;                          // C padded to whole 128-byte steps (narrow: to 32 elements)
    bool pad;                        // the operands are copied to rows of Cp (narrow: and into pieces)
    int64_t c4;                      // C rounded up to 4
    bool few;                        // wide rows, few of them
    bool one;                        // a single one, no longer than a workgroup of its kernels holds
    bool together;                   // the kept rows are moved together
    bool copy_x;                     // (wide) x is copied: padded, or moved together
    size_t xp, wp;                   // byte offsets: those copies
    size_t map, place, targets, count;
    size_t part, own, rows;          // forward
    int64_t tiles;                   // (wide) statistics per row
    // backward
    int64_t piece, np;               // table rows per piece; n padded to 128 bytes of dl^T
    int parts;                       // (few rows) sums of dx
    int64_t first_steps;             // (wide) of k in dx's product, the first piece
    bool big;                        // dx's tiles are 256 x 256
    size_t factors, dl, dlt, wt, xt, sums, sums_w;
    size_t total;
};

// 128 x 128: 64 KiB of stages, two workgroups per CU.  256 x 256: 128 KiB, one workgroup of 8 waves (16 bits only: the float32
// transpose of such a tile does not fit LDS) -- half the LDS and L2 traffic per operation.
using Tile128 = Tile<128, 128, 2, 2, false>;
using Tile256 = Tile<256, 256, 2, 4, true>;
// The statistics read the whole table once, from memory, and take the copies late better (8192 x 64000 x 2048: 1.58 ms against 1.70);
// the backward pass' products read a piece that the caches hold, and take them early (dx's 1.80 ms against 1.96).
using Tile256Late = Tile<256, 256, 2, 4, true, true>;

// Whether the [m][n] tiles of a 16-bit product are 256 x 256.  Both sizes' time goes as the area they cover in whole rounds of the
// chip (256 CUs; two of the small workgroups per CU), and the larger one is 4 / 3 as fast per area: statistics of 8192 x 64000 x 2048
// 1.60 ms against 2.13, of 5120 x 8192 x 2048 (a round of them is not full) 0.162 against 0.187; but the softmax gradient of
// 777 x 49999 x 768, 24 % of whose 256-row tiles is empty, 0.128 against 0.113.
static bool ce_big(int64_t m, int64_t n, int es) {
    if (es != 2) return false;
    const int64_t big = ceil_div(ceil_div(m, 256) * ceil_div(n, 256), 256) * 256, small = ceil_div(ceil_div(m, 128) * ceil_div(n, 128), 512) * 512;
    return big * 3 < small;
}

// Whether wide float32 rows go through the 16-bit matrix cores in pieces: six products at eight times the rate or more, for the
// conversion of the table.  Forward / backward of 300 x 20000 x 256 51 / 127 us against 48 / 157, of 2000 x 32000 x 1024 0.64 / 2.27 ms
// against 0.99 / 2.93, of 4096 x 65536 x 256 0.65 / 3.38 against 1.12 / 3.49.
static bool ce_in_pieces(int64_t n, int C, int dtype) { return dtype == MVS_DTYPE_F32 && !ce_narrow(C, dtype) && n > 256; }

static CePlan ce_plan(int64_t n, int64_t V, int C, int dtype, bool pieces, bool backward, bool need_x, bool need_w) {
    CePlan p = {};
    p.pieces = pieces;
    p.es = pieces ? 2 : (int)dtype_size(dtype);
    p.narrow = ce_narrow(C, dtype);
    p.few = !p.narrow && n <= ce_few_rows(p.es);
    p.c4 = round_up(C, 4);
    const int step = kRowBytes / p.es, planes = ce_planes(dtype);
    p.Cp = (int)round_up(C, p.narrow ? 32 : step);
    p.one = p.few && n == 1 && p.Cp <= 256 * 16 / p.es;
    p.pad = p.Cp != C || (p.narrow && planes > 1) || pieces;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    p.together = n > kTogether;
    p.copy_x = p.pad || p.together;
    if (p.together) {
        p.map = take((size_t)n * 4);
        p.place = take((size_t)n * 4);
        p.targets = take((size_t)n * 8);
        p.count = take(4);
    }
    const size_t row = (size_t)p.Cp * (p.narrow ? 2 * planes : p.es);
    if (p.copy_x) p.xp = take(pieces ? (size_t)round_up(n, 64) * row * 3 : (size_t)n * row);
    if (p.pad) p.wp = take(pieces ? (size_t)round_up(V, 64) * row * 3 : (size_t)V * row);
    const int64_t blocks_x = ceil_div(n, kNarrowRows), blocks_w = ceil_div(V, kNarrowRows);
    if (!backward) {
        p.tiles = p.narrow ? 0 : ceil_div(V, p.one && p.es == 4 ? kFewTable : ce_big(V, n, p.es) ? 256 : 128);
        p.part = take((p.narrow ? (size_t)narrow_most(blocks_x, V, kNarrowStatsSlots) * kNarrowRows : (size_t)p.tiles * n) * sizeof(float2));
        p.own = take((size_t)n * 4);
        p.rows = take((size_t)n * 4);
    } else if (p.narrow) {
        p.factors = take((size_t)(2 * n + 1) * 4);
        if (need_x) {
            p.wt = take((size_t)C * planes * round_up(V, 64) * 2);
            p.sums = take((size_t)narrow_most(blocks_x, V, kNarrowGradSlots) * kNarrowRows * p.c4 * 4);
        }
        if (need_w) {
            p.xt = take((size_t)C * planes * round_up(n, 64) * 2);
            p.sums_w = take((size_t)narrow_most(blocks_w, n, kNarrowGradSlots) * kNarrowRows * p.c4 * 4);
        }
    } else {
        // the piece: dl of at most 2^26 values, whole tiles (float32 in pieces 2^27: the products then fill the chip, 8000 x 60000 x 768
        // 15.2 / 14.0 / 13.4 ms by 2^25 / 2^26 / 2^27)
        p.piece = ((int64_t)1 << (pieces ? 27 : 26)) / (n > 0 ? n : 1) / 256 * 256;
        if (p.piece < 256) p.piece = 256;
        if (p.piece > round_up(V, 256)) p.piece = round_up(V, 256);
        p.np = round_up(n, step);
        p.factors = take((size_t)(2 * n + 1) * 4);
        if (p.few) {
            p.dl = take((size_t)n * p.piece * 4);
            p.parts = (int)ceil_div(V < p.piece ? V : p.piece, kFewTable);
            if (need_x) p.sums = take((size_t)p.parts * n * p.c4 * 4);
        } else {
            if (need_x || p.es == 2) p.dl = take((size_t)p.np * p.piece * p.es * (pieces ? 3 : 1));
            if (need_x && p.es == 4) p.wt = take((size_t)C * p.piece * p.es);
        }
        if (need_x && !p.few) {
            p.first_steps = round_up(V < p.piece ? V : p.piece, step) / step;
            p.big = ce_big(C, n, p.es);
            // rows of all parts' sums, however many rows are kept: whole tiles of a round, or one part of n
            const int64_t most = kRound / ceil_div(C, 128) * 128, even = ceil_div(p.first_steps, 8) * n;
            const int64_t rows = p.big ? n : most < even ? most : even;
            p.sums = take((size_t)(rows > n ? rows : n) * p.c4 * 4);
        }
        if (need_w && !p.few && !pieces) {
            p.dlt = take((size_t)p.piece * p.np * p.es);
            p.xt = take((size_t)C * p.np * p.es);
        }
    }
    p.total = at;
    return p;
}

static CeRows ce_rows(const CePlan &p, const int64_t *target, int64_t n, int64_t ignore, float *loss, char *ws, hipStream_t st) {
    CeRows r = {};
    r.target = target; r.n = n; r.ignore = ignore;
    if (!p.together) return r;
    int *map = reinterpret_cast<int *>(ws + p.map), *place = reinterpret_cast<int *>(ws + p.place), *count = reinterpret_cast<int *>(ws + p.count);
    int64_t *targets = reinterpret_cast<int64_t *>(ws + p.targets);
    const int64_t chunk = round_up(ceil_div(n, 256), 4096);
    hipLaunchKernelGGL(ce_together_kernel, dim3((unsigned)ceil_div(n, chunk)), dim3(1024), 0, st, target, n, ignore, chunk, map, place, targets, count, loss);
    r.map = map; r.place = place; r.count = count; r.target = targets;
    return r;
}

// the arguments of the narrow kernels that both passes share
static NarrowArgs ce_narrow_args(const CePlan &p, int dtype, const void *x, const void *w, const CeRows &rows, int64_t V, int C, float scale, char *ws) {
    NarrowArgs a = {};
    a.x = NarrowOperand{x, p.copy_x ? ws + p.xp : const_cast<char *>(static_cast<const char *>(x)), nullptr, rows.n, round_up(rows.n, 64), p.copy_x};
    a.w = NarrowOperand{w, p.pad ? ws + p.wp : const_cast<char *>(static_cast<const char *>(w)), nullptr, V, round_up(V, 64), p.pad};
    a.C = C; a.Cp = p.Cp; a.planes = ce_planes(dtype);
    a.scale2 = scale * kLog2e; a.kept_rows = rows; a.ld_sums = p.c4;
    return a;
}

static int ce_check(const char *who, const void *x, const void *w, int dtype, const int64_t *target, int64_t n, int64_t V, int C, int reduction,
                    const void *workspace, size_t workspace_bytes, size_t need) {
    if (n < 0 || V < 1 || C < 1 || dtype_size(dtype) == 0 || !w || (n > 0 && (!x || !target)) || reduction < 0 || reduction > 2 || !workspace) {
        set_error("%s: invalid argument (n=%lld, V=%lld, C=%d, dtype=%d, reduction=%d)", who, (long long)n, (long long)V, C, dtype, reduction);
        return MVS_EINVAL;
    }
    if (!aligned16(x) || !aligned16(w) || !aligned16(workspace)) {
        set_error("%s: x, weight and the workspace are to be aligned to 16 bytes", who);
        return MVS_EINVAL;
    }
    if (n > ((int64_t)1 << 29) || V > ((int64_t)1 << 29) || C > (1 << 20) || ceil_div(n, 64) * ceil_div(V, 64) > 0x7fffffff) {
        set_error("%s: n=%lld, V=%lld (at most 2^29 each, n V / 4096 below 2^31), C=%d (at most 2^20)", who, (long long)n, (long long)V, C);
        return MVS_EUNSUPPORTED;
    }
    if (n > ((int64_t)1 << 23) && !ce_narrow(C, dtype)) {      // (a tile's rows of dl^T are addressed in 32 bits)
        set_error("%s: n=%lld rows of C=%d, at most 2^23 of that length at a time", who, (long long)n, C);
        return MVS_EUNSUPPORTED;
    }
    if (workspace_bytes < need) {
        set_error("%s: workspace too small (%zu of %zu bytes)", who, workspace_bytes, need);
        return MVS_EWORKSPACE;
    }
    return MVS_OK;
}

// the operands as the tiles read them: x copied (the kept rows, padded) and the table padded where the plan says so
template <typename T>
static void ce_operands(const CePlan &p, const void *x, const void *w, const CeRows &rows, int64_t V, int C, char *ws, hipStream_t st, CeArgs &a) {
    a.steps = p.Cp * p.es / kRowBytes;
    a.v_total = V;
    a.rows = rows;
    if constexpr (kPieces<T>) {
        auto planes = [&](const void *in, const CeRows &r, char *out) {
            const int64_t padded = round_up(r.n, 64), plane = padded * p.Cp * 2;
            hipLaunchKernelGGL(ce_pieces_kernel, grid_of(ceil_div(padded * (p.Cp / 8), 256)), dim3(256), 0, st, static_cast<const float *>(in), r, C, out, p.Cp, plane);
            return Operand{out, (int64_t)p.Cp * 2, r.n, plane};
        };
        CeRows table = {};
        table.n = V;
        a.x = planes(x, rows, ws + p.xp);
        a.w = planes(w, table, ws + p.wp);
        return;
    } else {
    auto copy = [&](const void *in, const CeRows &r, char *out) {
        constexpr int VEC = 16 / sizeof(T);
        if (C % VEC == 0)
            hipLaunchKernelGGL((ce_rows_kernel<T, VEC>), grid_of(ceil_div(r.n * (p.Cp / VEC), 256)), dim3(256), 0, st, static_cast<const T *>(in), r, C,
                               reinterpret_cast<T *>(out), p.Cp);
        else
            hipLaunchKernelGGL((ce_rows_kernel<T, 1>), grid_of(ceil_div(r.n * p.Cp, 256)), dim3(256), 0, st, static_cast<const T *>(in), r, C,
                               reinterpret_cast<T *>(out), p.Cp);
    };
    a.w = Operand{static_cast<const char *>(w), (int64_t)p.Cp * p.es, V};
    a.x = Operand{static_cast<const char *>(x), (int64_t)p.Cp * p.es, rows.n};
    if (p.copy_x) {
        copy(x, rows, ws + p.xp);
        a.x.p = ws + p.xp;
    }
    if (p.pad) {
        CeRows table = {};
        table.n = V;
        copy(w, table, ws + p.wp);
        a.w.p = ws + p.wp;
    }
    }
}

template <typename T>
static void ce_transpose(const char *in, const CeRows &rows, bool look, int C, int64_t ld_in, char *out, int64_t ld_out, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(T);      // (ld_in and ld_out are whole 128-byte steps)
    hipLaunchKernelGGL((ce_transpose_kernel<T, VEC>), dim3((unsigned)ceil_div(ld_out, 64), (unsigned)ceil_div(C, 64)), dim3(256), 0, st,
                       reinterpret_cast<const T *>(in), rows, look, C, ld_in, reinterpret_cast<T *>(out), ld_out);
}

// a kernel on the tiles of its [m][n]: f(X()) sets the grid and launches
template <typename T, typename F>
static void ce_tiles(int64_t m, int64_t n, F f) {
    if constexpr (sizeof(T) == 2) {
        if (ce_big(m, n, 2)) { f(Tile256()); return; }
    }
    f(Tile128());
}

// two stages of LDS, or what the epilogue lays there if that is more (an error stands for check_launch)
template <typename X, typename F, typename A>
static void ce_launch(F kernel, const A &a, dim3 grid, size_t epilogue, hipStream_t st) {
    const size_t stages = 2 * (size_t)X::STAGE;
    const unsigned bytes = (unsigned)(epilogue > stages ? epilogue : stages);
    // (more than 64 KiB of dynamic LDS has to be asked for)
    if (bytes > 65536 && hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) return;
    hipLaunchKernelGGL(kernel, grid, dim3(X::THREADS), bytes, st, a);
}

template <typename T>
static void ce_few(CeFew d, hipStream_t st) {
    auto launch = [&](auto kernel, int vec) {
        d.threads = 1;
        while (d.threads < 256 && d.threads * vec < d.Cp) d.threads *= 2;
        hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(d.count, kFewTable), (unsigned)ceil_div(d.Cp, d.threads * vec)), dim3(256), 0, st, d);
    };
    // 16-byte accesses while x and dx of NR rows at that many columns fit the registers, 8-byte ones for more
    constexpr int VEC = 16 / sizeof(T);
    if constexpr (sizeof(T) == 4) {
        if (d.part) launch(ce_one_stats_kernel<T, VEC>, VEC);
        else if (d.n > 8) launch(ce_few_kernel<T, 16, VEC / 2, false>, VEC / 2);
        else if (d.n > 4) launch(ce_few_kernel<T, 8, VEC, false>, VEC);
        if (d.part || d.n > 4) return;
    }
    if (d.target) launch(ce_few_kernel<T, 1, VEC, true>, VEC);
    else if (d.n == 1) launch(ce_few_kernel<T, 1, VEC, false>, VEC);
    else launch(ce_few_kernel<T, 4, VEC, false>, VEC);
}

template <typename T>
static int ce_wide_stats(const CePlan &p, const void *x, const void *w, const CeRows &rows, int64_t V, int C, float scale, char *ws, hipStream_t st) {
    CeArgs a = {};
    ce_operands<T>(p, x, w, rows, V, C, ws, st, a);
    a.v_count = V;
    a.scale2 = scale * kLog2e;
    a.part = reinterpret_cast<float2 *>(ws + p.part);
    a.own = reinterpret_cast<float *>(ws + p.own);
    if constexpr (std::is_same_v<T, float>) if (p.one) {
        CeFew d = {};
        d.w = a.w.p; d.x = a.x.p; d.count = V; d.n = 1; d.C = C; d.Cp = p.Cp;
        d.target = rows.target; d.scale2 = a.scale2; d.part = a.part; d.own = a.own;
        ce_few<T>(d, st);
        return check_launch("mvs_linear_ce_fwd");
    }
    ce_tiles<T>(V, rows.n, [&](auto x) {
        using X = std::conditional_t<std::is_same_v<decltype(x), Tile256>, Tile256Late, decltype(x)>;
        a.tiles_m = ceil_div(V, X::BM); a.tiles_n = ceil_div(rows.n, X::BN);
        ce_launch<X>(ce_stats_kernel<T, X>, a, grid_of(a.tiles_m * a.tiles_n), (size_t)X::WAVES_M * X::BN * sizeof(float2), st);
    });
    return check_launch("mvs_linear_ce_fwd");
}

static int ce_forward(int dtype, const void *x, const void *w, const int64_t *target, int64_t n, int64_t V, int C, float scale, int64_t ignore,
                      int reduction, float *loss, float *lse, float *kept, char *ws, hipStream_t st) {
    const CePlan p = ce_plan(n, V, C, dtype, ce_in_pieces(n, C, dtype), false, false, false);
    float *losses = reduction == 0 ? loss : reinterpret_cast<float *>(ws + p.rows);
    if (n > 0) {
        float2 *part = reinterpret_cast<float2 *>(ws + p.part);
        float *own = reinterpret_cast<float *>(ws + p.own);
        const CeRows rows = ce_rows(p, target, n, ignore, losses, ws, st);
        int rc = MVS_OK;
        if (p.narrow) {
            NarrowArgs a = ce_narrow_args(p, dtype, x, w, rows, V, C, scale, ws);
            a.part = part; a.own = own;
            rc = ce_narrow_forward(dtype, a, st);
        } else if (p.pieces) {
            rc = ce_wide_stats<pieces_t>(p, x, w, rows, V, C, scale, ws, st);
        } else {
            MVS_DTYPE_DISPATCH(dtype, T, rc = (ce_wide_stats<T>(p, x, w, rows, V, C, scale, ws, st)));
        }
        if (rc != MVS_OK) return rc;
        hipLaunchKernelGGL(ce_join_kernel, grid_of(ceil_div(n, 16)), dim3(256), 0, st, part, p.tiles, V, rows, own, lse, losses);
    }
    hipLaunchKernelGGL(ce_total_kernel, dim3(1), dim3(1024), 0, st, losses, target, n, ignore, reduction, loss, kept);
    return check_launch("mvs_linear_ce_fwd");
}

template <typename T>
static int ce_wide_backward(const CePlan &p, const void *x, const void *w, const CeRows &rows, const float *lse, const float *kept, const float *grad_loss,
                            int64_t V, int C, float scale, int reduction, void *grad_x, void *grad_w, char *ws, hipStream_t st) {
    using O = typename Given<T>::type;
    const int step = kRowBytes / p.es;
    const int64_t n = rows.n;
    float *factors = reinterpret_cast<float *>(ws + p.factors);
    hipLaunchKernelGGL(ce_factors_kernel, dim3(reduction == 0 ? 1 : (unsigned)ceil_div(n, 1024)), dim3(1024), 0, st, rows, grad_loss, kept, reduction, factors);
    CeArgs a = {};
    ce_operands<T>(p, x, w, rows, V, C, ws, st, a);
    const float factor = scale / GradUnit<T>::value;
    const char *w_rows = a.w.p;
    a.scale2 = scale * kLog2e;
    a.lse2 = lse; a.ratio = factors + n;
    // dW's product takes dl and x as they are, k along their rows, where it can: 16 bits, no row in between that is ignored, one factor
    // for all rows (else dl^T carries the rows' ratios).
    const bool along = sizeof(T) == 2 && p.together && reduction != 0;
    a.dl = grad_x || p.few || (along && grad_w) ? ws + p.dl : nullptr;
    a.dlt = grad_w && !p.few && !along ? ws + p.dlt : nullptr;
    a.ld_dlt = p.np;
    a.dl_plane = p.np * p.piece * 2;
    a.dl_step = along ? step : 1;      // (dW's product reads whole steps of rows; along: dl has p.np of them)
    // x^T once; ignored rows as zeros, whatever they hold
    if constexpr (!kPieces<T>) if (a.dlt) ce_transpose<T>(a.x.p, rows, !p.together, C, p.Cp, ws + p.xt, p.np, st);
    auto product = [&](CeProduct &d, auto a_along, auto b_along) {
        ce_tiles<T>(d.m, d.n, [&](auto x) {
            using X = decltype(x);
            d.tiles_m = ceil_div(d.m, X::BM); d.tiles_n = ceil_div(d.n, X::BN);
            const int64_t tiles = d.tiles_m * d.tiles_n, groups = d.sums && X::BM == 128 && tiles < kRound ? kRound : tiles;
            ce_launch<X>(ce_product_kernel<T, X, decltype(a_along)::value, decltype(b_along)::value>, d, dim3((unsigned)groups), 0, st);
        });
    };
    const bool logits = p.one;
    const float few_factor = logits ? scale : factor;      // (its dl is float32 throughout, not carried in a unit)
    for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
        const int64_t count = V - v0 < p.piece ? V - v0 : p.piece, k = round_up(count, step);
        a.w.p = w_rows + v0 * p.Cp * p.es;
        a.w.rows = count;
        a.v0 = v0; a.v_count = count; a.ld_dl = k;
        auto gradient = [&](auto x, auto kernel) {
            using X = decltype(x);
            a.tiles_m = ceil_div(count, X::BM); a.tiles_n = ceil_div(n, X::BN);
            ce_launch<X>(kernel, a, dim3((unsigned)(a.tiles_m * a.tiles_n)), (size_t)X::BM * (X::BN * sizeof(T) + 16), st);
        };
        if constexpr (!kPieces<T>) if (p.few && !logits) gradient(Tile128(), ce_grad_kernel<T, Tile128, true>);
        if (!p.few) ce_tiles<T>(count, n, [&](auto x) { gradient(x, ce_grad_kernel<T, decltype(x)>); });
        if constexpr (!kPieces<T>) if (p.few) {
            CeFew d = {};
            d.w = a.w.p; d.x = a.x.p; d.dl = static_cast<const float *>(a.dl); d.count = count; d.ld_dl = k;
            d.n = (int)n; d.C = C; d.Cp = p.Cp;
            d.ratio = factors + n; d.top = factors + 2 * n; d.factor = few_factor;
            if (logits) { d.lse2 = lse; d.target = rows.target; d.ignore = rows.ignore; d.v0 = v0; d.scale2 = a.scale2; }
            d.grad_w = grad_w ? static_cast<T *>(grad_w) + v0 * C : nullptr;
            d.sums = grad_x ? reinterpret_cast<float *>(ws + p.sums) : nullptr;
            d.c4 = p.c4; d.add = v0 > 0;
            ce_few<T>(d, st);
            continue;
        }
        if (grad_x) {
            CeProduct d = {};
            if constexpr (sizeof(T) == 2) {
                d.a = a.w;
            } else {
                CeRows table = {};
                table.n = count;
                ce_transpose<T>(a.w.p, table, false, C, p.Cp, ws + p.wt, k, st);
                d.a = Operand{ws + p.wt, k * p.es, C};
            }
            d.b = Operand{ws + p.dl, k * p.es, n, a.dl_plane};
            d.steps = (int)(k / step);
            d.first_steps = (int)p.first_steps;
            d.m = C; d.n = n;
            d.sums = reinterpret_cast<float *>(ws + p.sums); d.ld_sums = p.c4; d.count = rows.count;
            d.add = v0 > 0;
            // (a smaller last piece may have fewer parts of k: the sums of the others stay as they are)
            product(d, std::bool_constant<sizeof(T) == 2>(), std::false_type());
        }
        if (grad_w) {
            CeProduct d = {};
            d.steps = (int)(p.np / step);
            d.m = C; d.n = count;
            d.out = static_cast<O *>(grad_w) + v0 * C;
            d.top = factors + 2 * n; d.factor = factor; d.count = rows.count;
            if constexpr (sizeof(T) == 2) {
                if (along) {
                    d.a = a.x;
                    d.b = Operand{ws + p.dl, k * p.es, p.np, a.dl_plane};
                    product(d, std::true_type(), std::true_type());
                    continue;
                }
            }
            if constexpr (!kPieces<T>) {
                d.a = Operand{ws + p.xt, p.np * p.es, C};
                d.b = Operand{ws + p.dlt, p.np * p.es, count};
                product(d, std::false_type(), std::false_type());
            }
        }
    }
    if (grad_x && p.few)
        hipLaunchKernelGGL((ce_few_finish_kernel<O>), dim3((unsigned)ceil_div(n * (p.c4 / 4), 16)), dim3(256), 0, st, reinterpret_cast<const float *>(ws + p.sums),
                           p.parts, (int)n, C, p.c4, factors, few_factor, static_cast<O *>(grad_x));
    else if (grad_x)
        hipLaunchKernelGGL((ce_finish_kernel<O>), grid_of(ceil_div(n * (p.c4 / 4), 256)), dim3(256), 0, st, reinterpret_cast<const float *>(ws + p.sums),
                           p.first_steps, p.big, rows, C, p.c4, factors, factor, static_cast<O *>(grad_x));
    return check_launch("mvs_linear_ce_bwd");
}

// a gradient of no rows
__global__ __launch_bounds__(256) void ce_zero_kernel(unsigned short *__restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

}  // namespace mvs

using namespace mvs;

extern "C" size_t mvs_linear_ce_workspace_bytes(int64_t n, int64_t V, int C, int dtype, int backward, int need_x, int need_w) {
    if (n < 0 || V < 1 || C < 1 || dtype_size(dtype) == 0) return 0;
    const size_t plain = ce_plan(n, V, C, dtype, false, backward != 0, need_x != 0, need_w != 0).total;
    const size_t pieces = ce_in_pieces(n, C, dtype) ? ce_plan(n, V, C, dtype, true, backward != 0, need_x != 0, need_w != 0).total : 0;
    return (plain > pieces ? plain : pieces) + 256;
}

extern "C" int mvs_linear_ce_fwd(const void *x, const void *weight, int dtype, const int64_t *target, int64_t n, int64_t V, int C, float scale,
                                 int64_t ignore_index, int reduction, float *loss, float *lse, float *kept, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    const int rc = ce_check("mvs_linear_ce_fwd", x, weight, dtype, target, n, V, C, reduction, workspace, workspace_bytes,
                            mvs_linear_ce_workspace_bytes(n, V, C, dtype, 0, 0, 0));
    if (rc != MVS_OK) return rc;
    if (!kept || (!loss && (reduction != 0 || n > 0)) || (!lse && n > 0)) {
        set_error("mvs_linear_ce_fwd: loss, lse and kept are needed");
        return MVS_EINVAL;
    }
    return ce_forward(dtype, x, weight, target, n, V, C, scale, ignore_index, reduction, loss, lse, kept, static_cast<char *>(workspace), as_stream(stream));
}

extern "C" int mvs_linear_ce_bwd(const void *x, const void *weight, int dtype, const int64_t *target, const float *lse, const float *kept,
                                 const float *grad_loss, int64_t n, int64_t V, int C, float scale, int64_t ignore_index, int reduction,
                                 void *grad_x, void *grad_weight, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = ce_check("mvs_linear_ce_bwd", x, weight, dtype, target, n, V, C, reduction, workspace, workspace_bytes,
                            mvs_linear_ce_workspace_bytes(n, V, C, dtype, 1, grad_x != nullptr, grad_weight != nullptr));
    if (rc != MVS_OK) return rc;
    if (!aligned16(grad_x) || !aligned16(grad_weight)) {
        set_error("mvs_linear_ce_bwd: the gradients are to be aligned to 16 bytes");
        return MVS_EINVAL;
    }
    if (n == 0) {
        if (grad_weight)
            hipLaunchKernelGGL(ce_zero_kernel, dim3(1024), dim3(256), 0, as_stream(stream), static_cast<unsigned short *>(grad_weight),
                               V * C * (int64_t)(dtype_size(dtype) / 2));
        return check_launch("mvs_linear_ce_bwd");
    }
    if (!lse || !kept || !grad_loss || (!grad_x && !grad_weight)) {
        set_error("mvs_linear_ce_bwd: lse, kept, grad_loss and a gradient to compute are needed");
        return MVS_EINVAL;
    }
    // (rows with factors of their own need dl^T, which the pieces' products do without)
    const CePlan p = ce_plan(n, V, C, dtype, reduction != 0 && ce_in_pieces(n, C, dtype), true, grad_x != nullptr, grad_weight != nullptr);
    char *ws = static_cast<char *>(workspace);
    const CeRows rows = ce_rows(p, target, n, ignore_index, nullptr, ws, as_stream(stream));
    if (p.narrow) {
        NarrowArgs a = ce_narrow_args(p, dtype, x, weight, rows, V, C, scale, ws);
        a.lse2 = lse; a.grad_loss = grad_loss; a.kept = kept; a.reduction = reduction;
        a.factors = reinterpret_cast<float *>(ws + p.factors);
        if (grad_x) { a.w.trans = ws + p.wt; a.sums_x = reinterpret_cast<float *>(ws + p.sums); }
        if (grad_weight) { a.x.trans = ws + p.xt; a.sums_w = reinterpret_cast<float *>(ws + p.sums_w); }
        a.grad_x = grad_x; a.grad_w = grad_weight;
        a.factor = scale / (dtype == MVS_DTYPE_F16 ? GradUnit<f16_t>::value : 1.0f);
        return ce_narrow_backward(dtype, a, as_stream(stream));
    }
    if (p.pieces)
        return ce_wide_backward<pieces_t>(p, x, weight, rows, lse, kept, grad_loss, V, C, scale, reduction, grad_x, grad_weight, ws, as_stream(stream));
    MVS_DTYPE_DISPATCH(dtype, T, {
        return (ce_wide_backward<T>(p, x, weight, rows, lse, kept, grad_loss, V, C, scale, reduction, grad_x, grad_weight, ws, as_stream(stream)));
    });
}
