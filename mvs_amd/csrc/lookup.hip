// Rows of a table by index, scaled, and the table's gradient by sorted indices.
//
//   out[i] = s T[index i]            grad T[v] = s sum over {i : index i = v}, in the order of i, of g[i]
//
// Forward: bound by the rows it reads and writes; 16 bytes per lane, a power-of-two number of lanes per row.
//
// Backward: every row of the dense gradient is written once, most of them as zeros, and every row of g is read once.  Who adds to a
// row is known only after the indices are sorted.  The sort is stable, so a row's terms come in the order of i and equal calls
// give equal bits; floating-point atomics on the rows would need neither sort nor order, but sum in another order every time.
//   sort   up to kRankMax indices: a term's place is the number of smaller keys, plus that of equal keys in front of it -- one
//          launch, n^2 / 2^14 cycles on the chip; more: least-significant-digit radix sort of (key, i), digits of up to 10 bits,
//          three launches each (count per tile, one workgroup's scan, place).
//   rows   the sorted terms are cut into pieces of kPiece; a piece's lanes walk it with the loads of 8 terms in flight and write
//          the sum of each run of equal keys that lies within the piece.  A run that leaves the piece (a frequent index) leaves
//          float32 partial sums, at most two per piece.  The same launch writes the zero rows (found by binary search, 64 table
//          rows per wave's worth of lanes).
//   join   the pieces of a long run, in order, four spans of them at a time.
#include <utility>

#include "dtype.h"

namespace mvs {

constexpr int kRankMax = 8192;
constexpr int kPiece = 16;         // sorted terms per piece
constexpr int kTile = 4096;        // keys per workgroup of a radix pass
constexpr int kMaxDigit = 10;

struct LookupPlan {
    int64_t n, rows;
    int key_bits, passes, digit_bits;
    int64_t tiles, pieces;
    size_t keys0, vals0, keys1, vals1, hist, part, total;      // byte offsets into the workspace
};

static LookupPlan lookup_plan(int64_t rows, int C, int64_t n) {
    LookupPlan p = {};
    p.n = n; p.rows = rows;
    while (p.key_bits < 32 && ((int64_t)1 << p.key_bits) <= rows) ++p.key_bits;      // keys 0 .. rows (rows: names no row)
    p.passes = n <= kRankMax ? 0 : (p.key_bits + kMaxDigit - 1) / kMaxDigit;
    p.digit_bits = p.passes ? (p.key_bits + p.passes - 1) / p.passes : 0;
    p.tiles = (n + kTile - 1) / kTile;
    p.pieces = (n + kPiece - 1) / kPiece;
    auto align = [](size_t b) { return (b + 255) & ~(size_t)255; };
    size_t at = 0;
    p.keys0 = at; at += align((size_t)n * 4);
    p.vals0 = at; at += align((size_t)n * 4);
    if (p.passes) {
        p.keys1 = at; at += align((size_t)n * 4);
        p.vals1 = at; at += align((size_t)n * 4);
        p.hist = at; at += align((size_t)p.tiles * ((size_t)1 << p.digit_bits) * 4);
    }
    p.part = at; at += align((size_t)p.pieces * 2 * C * 4);
    p.total = at;
    return p;
}

__device__ __forceinline__ unsigned lookup_key(int64_t index, int64_t rows) { return (index >= 0 && index < rows) ? (unsigned)index : (unsigned)rows; }

template <typename T, int VEC>
__global__ __launch_bounds__(256) void lookup_fwd_kernel(const T *__restrict__ table, int64_t rows, int C, const int64_t *__restrict__ index,
                                                         int64_t n, float scale, T *__restrict__ out, int lanes) {
    const int lane = threadIdx.x & (lanes - 1), vecs = C / VEC;
    const int64_t i = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (i >= n) return;
    const int64_t row = index[i];
    const bool named = row >= 0 && row < rows;
    const Pack<T, VEC> *from = reinterpret_cast<const Pack<T, VEC> *>(table + (named ? row : 0) * C);
    Pack<T, VEC> *to = reinterpret_cast<Pack<T, VEC> *>(out + i * C);
    for (int c = lane; c < vecs; c += lanes) {
        Pack<T, VEC> v;
        if (named) v = from[c];
#pragma unroll
        for (int j = 0; j < VEC; ++j) v.v[j] = from_float<T>(named ? to_float(v.v[j]) * scale : 0.0f);
        to[c] = v;
    }
}

// ---- sort
// 64 terms per workgroup, four waves each against a quarter of the keys; the keys pass through LDS 1024 at a time.
__global__ __launch_bounds__(256) void lookup_rank_kernel(const int64_t *__restrict__ index, int n, int64_t rows, unsigned *__restrict__ keys,
                                                          unsigned *__restrict__ vals) {
    __shared__ unsigned tile[1024];
    __shared__ int ranks[256];
    const int tid = threadIdx.x, i = blockIdx.x * 64 + (tid & 63), quarter = tid >> 6;
    const unsigned mine = i < n ? lookup_key(index[i], rows) : 0u;
    int rank = 0;
    for (int base = 0; base < n; base += 1024) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = base + u * 256 + tid;
            tile[u * 256 + tid] = j < n ? lookup_key(index[j], rows) : 0xffffffffu;
        }
        __syncthreads();
        const uint4 *t4 = reinterpret_cast<const uint4 *>(tile + quarter * 256);
        const int j0 = base + quarter * 256;
#pragma unroll 8
        for (int j = 0; j < 64; ++j) {
            const uint4 k = t4[j];      // (one address for the wave)
            const int jj = j0 + j * 4;
            rank += (k.x < mine || (k.x == mine && jj < i)) + (k.y < mine || (k.y == mine && jj + 1 < i)) +
                    (k.z < mine || (k.z == mine && jj + 2 < i)) + (k.w < mine || (k.w == mine && jj + 3 < i));
        }
    }
    ranks[tid] = rank;
    __syncthreads();
    if (quarter == 0 && i < n) {
        const int r = ranks[tid] + ranks[tid + 64] + ranks[tid + 128] + ranks[tid + 192];
        keys[r] = mine;
        vals[r] = (unsigned)i;
    }
}

// counts per (digit, tile), digit-major: their exclusive scan is where a tile's keys of a digit go
template <bool FIRST>
__global__ __launch_bounds__(256) void lookup_count_kernel(const int64_t *__restrict__ index, const unsigned *__restrict__ keys, int64_t n,
                                                           int64_t rows, int shift, int bits, int64_t tiles, unsigned *__restrict__ hist) {
    __shared__ unsigned count[1 << kMaxDigit];
    const int digits = 1 << bits;
    for (int d = threadIdx.x; d < digits; d += 256) count[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kTile;
#pragma unroll 4
    for (int u = 0; u < kTile / 256; ++u) {
        const int64_t i = base + u * 256 + threadIdx.x;
        if (i < n) {
            const unsigned key = FIRST ? lookup_key(index[i], rows) : keys[i];
            atomicAdd(&count[key >> shift & (digits - 1)], 1u);      // (whole numbers: their order does not matter)
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 256) hist[(int64_t)d * tiles + blockIdx.x] = count[d];
}

// exclusive scan of `m` counts in place, by one workgroup
__global__ __launch_bounds__(1024) void lookup_scan_kernel(unsigned *__restrict__ hist, int64_t m) {
    __shared__ unsigned sums[16];
    unsigned carry = 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t base = 0; base < m; base += 8192) {
        const int64_t at = base + (int64_t)threadIdx.x * 8;
        unsigned v[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) { v[j] = at + j < m ? hist[at + j] : 0u; }
#pragma unroll
        for (int j = 0; j < 8; ++j) { const unsigned t = v[j]; v[j] = sum; sum += t; }
        unsigned incl = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned t = (unsigned)__shfl_up((int)incl, o);
            if (lane >= o) incl += t;
        }
        if (lane == 63) sums[wave] = incl;
        __syncthreads();
        unsigned before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) { if (w < wave) before += sums[w]; all += sums[w]; }
        before += incl - sum;
#pragma unroll
        for (int j = 0; j < 8; ++j) if (at + j < m) hist[at + j] = before + v[j];
        carry += all;
        __syncthreads();
    }
}

__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Places a tile's keys: 4 waves, each 1024 consecutive keys in 16 rounds of 64.  A key's place is the tile's start of its digit,
// plus the earlier waves' count of it, plus the wave's own earlier ones, plus the lanes in front of it that hold the same digit.
template <bool FIRST>
__global__ __launch_bounds__(256) void lookup_place_kernel(const int64_t *__restrict__ index, const unsigned *__restrict__ keys_in,
                                                           const unsigned *__restrict__ vals_in, int64_t n, int64_t rows, int shift, int bits,
                                                           int64_t tiles, const unsigned *__restrict__ hist, unsigned *__restrict__ keys_out,
                                                           unsigned *__restrict__ vals_out) {
    __shared__ unsigned count[4][1 << kMaxDigit];
    const int digits = 1 << bits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int d = tid; d < digits; d += 256) {
#pragma unroll
        for (int w = 0; w < 4; ++w) count[w][d] = 0;
    }
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kTile + wave * 1024;
    unsigned key[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) {
        const int64_t i = base + u * 64 + lane;
        key[u] = 0;
        if (i < n) {
            key[u] = FIRST ? lookup_key(index[i], rows) : keys_in[i];
            atomicAdd(&count[wave][key[u] >> shift & (digits - 1)], 1u);
        }
    }
    __syncthreads();
    for (int d = tid; d < digits; d += 256) {
        unsigned at = hist[(int64_t)d * tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < 4; ++w) { const unsigned c = count[w][d]; count[w][d] = at; at += c; }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 16; ++u) {
        const int64_t i = base + u * 64 + lane;
        const bool here = i < n;
        const unsigned digit = key[u] >> shift & (digits - 1);
        unsigned long long same = __ballot(here);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot(here && (digit >> b & 1));
            same &= (digit >> b & 1) ? set : ~set;
        }
        // (only this wave touches count[wave]: LDS serves a wave's accesses in program order, which the fences keep -- every lane
        // reads its digit's start before the first of them moves it on, and the next round reads what that one stored)
        unsigned start = 0;
        if (here) start = count[wave][digit];
        const unsigned ahead = __popcll(same & ((1ull << lane) - 1));
        wave_order();
        if (here && ahead == 0) count[wave][digit] = start + __popcll(same);
        wave_order();
        if (here) {
            const unsigned to = start + ahead;
            keys_out[to] = key[u];
            vals_out[to] = FIRST ? (unsigned)i : vals_in[i];
        }
    }
}

// ---- rows
// first position in keys[0, n) that is not below `key`
__device__ __forceinline__ int64_t lookup_lower(const unsigned *__restrict__ keys, int64_t n, unsigned key) {
    int64_t lo = 0, len = n;
    while (len > 0) {
        const int64_t half = len >> 1;
        if (keys[lo + half] < key) { lo += half + 1; len -= half + 1; } else { len = half; }
    }
    return lo;
}

struct LookupRows {
    const void *grad;
    const unsigned *keys, *vals;
    void *out;
    float *part;           // [pieces][2][C]: the run that comes from the piece before, the run that goes on into the next
    int64_t n, rows, pieces, sum_groups;
    int C, lanes;
    float scale;
};

// Workgroups 0 .. sum_groups - 1 sum pieces (256 / lanes pieces each), the rest write zero rows (64 table rows each).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void lookup_rows_kernel(LookupRows a) {
    const int tid = threadIdx.x, lane = tid & (a.lanes - 1), vecs = a.C / VEC;
    T *out = static_cast<T *>(a.out);
    if (blockIdx.x >= a.sum_groups) {
        __shared__ unsigned long long empty_rows;
        const int64_t v0 = (blockIdx.x - a.sum_groups) * 64;
        if (tid < 64) {
            const int64_t v = v0 + tid;
            bool empty = v < a.rows;
            if (empty) {
                const int64_t at = lookup_lower(a.keys, a.n, (unsigned)v);
                empty = at >= a.n || a.keys[at] != (unsigned)v;
            }
            const unsigned long long m = __ballot(empty);
            if (tid == 0) empty_rows = m;
        }
        __syncthreads();
        const unsigned long long m = empty_rows;
        Pack<T, VEC> zero;
#pragma unroll
        for (int j = 0; j < VEC; ++j) zero.v[j] = from_float<T>(0.0f);
        for (int r = tid / a.lanes; r < 64; r += 256 / a.lanes) {
            if (!(m >> r & 1)) continue;
            Pack<T, VEC> *to = reinterpret_cast<Pack<T, VEC> *>(out + (v0 + r) * a.C);
            for (int c = lane; c < vecs; c += a.lanes) to[c] = zero;
        }
        return;
    }
    const int64_t piece = (int64_t)blockIdx.x * (256 / a.lanes) + tid / a.lanes;
    if (piece >= a.pieces) return;
    const int64_t p0 = piece * kPiece;
    const int count = (int)(a.n - p0 < kPiece ? a.n - p0 : kPiece);
    const unsigned none = (unsigned)a.rows;
    const unsigned before = p0 > 0 ? a.keys[p0 - 1] : 0xffffffffu, behind = p0 + count < a.n ? a.keys[p0 + count] : 0xffffffffu;
    const T *grad = static_cast<const T *>(a.grad);
    unsigned key[kPiece], val[kPiece];
#pragma unroll
    for (int t = 0; t < kPiece; ++t) {
        key[t] = t < count ? a.keys[p0 + t] : 0xffffffffu;
        val[t] = t < count ? a.vals[p0 + t] : 0u;
    }
    for (int c = lane; c < vecs; c += a.lanes) {
        float sum[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
        bool from_before = key[0] == before;
#pragma unroll
        for (int half = 0; half < kPiece; half += 8) {
            Pack<T, VEC> g[8];
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (half + t < count && key[half + t] != none)
                    g[t] = reinterpret_cast<const Pack<T, VEC> *>(grad + (int64_t)val[half + t] * a.C)[c];
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int k = half + t;
                if (k >= count || key[k] == none) continue;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] += to_float(g[t].v[j]);
                const bool last = k == count - 1;
                const unsigned next = last ? behind : key[k + 1 < kPiece ? k + 1 : k];
                if (!last && next == key[k]) continue;
                const bool goes_on = last && behind == key[k];
                if (from_before || goes_on) {
                    // (a run that fills the piece and leaves it on both sides counts as coming from before)
                    float *to = a.part + (piece * 2 + (from_before ? 0 : 1)) * a.C + c * VEC;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) to[j] = sum[j];
                } else {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = from_float<T>(sum[j] * a.scale);
                    reinterpret_cast<Pack<T, VEC> *>(out + (int64_t)key[k] * a.C)[c] = o;
                }
                from_before = false;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
            }
        }
    }
}

// A run that begins in piece p and goes on: its partials are p's second one and the first ones of the pieces behind it that begin
// with its key.  256 threads = 4 spans x 64 columns; 16 pieces are looked at per workgroup.
template <typename T>
__global__ __launch_bounds__(256) void lookup_join_kernel(LookupRows a) {
    __shared__ float spans[4][64];
    const int col = blockIdx.y * 64 + (threadIdx.x & 63), span = threadIdx.x >> 6;
    for (int64_t piece = (int64_t)blockIdx.x * 16; piece < min(a.pieces - 1, (int64_t)blockIdx.x * 16 + 16); ++piece) {
        const int64_t p0 = piece * kPiece, end = p0 + kPiece;      // (not the last piece: it is full)
        const unsigned key = a.keys[end - 1];
        if (key == (unsigned)a.rows || a.keys[end] != key) continue;
        if (a.keys[p0] == key && p0 > 0 && a.keys[p0 - 1] == key) continue;      // (begins further ahead)
        const int64_t stop = lookup_lower(a.keys + end, a.n - end, key + 1) + end;      // first term behind the run
        const int64_t more = (stop - end + kPiece - 1) / kPiece, each = (more + 3) / 4;
        float sum = 0.0f;
        if (col < a.C) {
            if (span == 0) sum = a.part[(piece * 2 + 1) * a.C + col];
            const int64_t from = piece + 1 + span * each, to = min(piece + 1 + more, from + each);
            int64_t q = from;
            for (; q + 8 <= to; q += 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = a.part[(q + j) * 2 * a.C + col];
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += v[j];
            }
            for (; q < to; ++q) sum += a.part[q * 2 * a.C + col];
        }
        __syncthreads();
        spans[span][threadIdx.x & 63] = sum;
        __syncthreads();
        if (span == 0 && col < a.C) {
            const int t = threadIdx.x;
            static_cast<T *>(a.out)[(int64_t)key * a.C + col] = from_float<T>((((spans[0][t] + spans[1][t]) + spans[2][t]) + spans[3][t]) * a.scale);
        }
    }
}

static int lookup_check(const char *who, const void *table, const void *wide, int dtype, const int64_t *index, int64_t rows, int C, int64_t n) {
    if (n < 0 || rows < 1 || C < 1 || dtype_size(dtype) == 0 || !table || (n > 0 && (!wide || !index))) {
        set_error("%s: invalid argument (rows=%lld, C=%d, n=%lld, dtype=%d)", who, (long long)rows, C, (long long)n, dtype);
        return MVS_EINVAL;
    }
    if (rows > 0x7ffffffe || n > 0x7ffffffe) {
        set_error("%s: rows=%lld, n=%lld (at most 2^31 - 2 each)", who, (long long)rows, (long long)n);
        return MVS_EUNSUPPORTED;
    }
    return MVS_OK;
}
// lanes per row: the power of two that covers `vecs` accesses, at most 256
static int lookup_lanes(int vecs) {
    int l = 1;
    while (l < vecs && l < 256) l <<= 1;
    return l;
}
// 16-byte accesses where every row begins on 16 bytes
static bool lookup_wide(const void *a, const void *b, int dtype, int C) { return aligned16(a) && aligned16(b) && (size_t)C * dtype_size(dtype) % 16 == 0; }

template <typename T, int VEC>
static void lookup_launch_fwd(const void *table, int64_t rows, int C, const int64_t *index, int64_t n, float scale, void *out, hipStream_t st) {
    const int lanes = lookup_lanes(C / VEC);
    hipLaunchKernelGGL((lookup_fwd_kernel<T, VEC>), dim3((unsigned)((n * lanes + 255) / 256)), dim3(256), 0, st, static_cast<const T *>(table), rows, C, index,
                       n, scale, static_cast<T *>(out), lanes);
}

template <typename T, int VEC>
static void lookup_launch_rows(LookupRows a, hipStream_t st) {
    a.lanes = lookup_lanes(a.C / VEC);
    a.sum_groups = (a.pieces * a.lanes + 255) / 256;
    const int64_t zero_groups = (a.rows + 63) / 64;
    hipLaunchKernelGGL((lookup_rows_kernel<T, VEC>), dim3((unsigned)(a.sum_groups + zero_groups)), dim3(256), 0, st, a);
    if (a.pieces > 1)
        hipLaunchKernelGGL((lookup_join_kernel<T>), dim3((unsigned)((a.pieces + 15) / 16), (unsigned)((a.C + 63) / 64)), dim3(256), 0, st, a);
}

}  // namespace mvs

using namespace mvs;

extern "C" int mvs_lookup_rows_fwd(const void *table, int dtype, int64_t rows, int C, const int64_t *index, int64_t n, float scale, void *out,
                                   void *stream) {
    const int rc = lookup_check("mvs_lookup_rows_fwd", table, out, dtype, index, rows, C, n);
    if (rc != MVS_OK || n == 0) return rc;
    hipStream_t st = as_stream(stream);
    const bool wide = lookup_wide(table, out, dtype, C);
    MVS_DTYPE_DISPATCH(dtype, T, {
        if (wide) lookup_launch_fwd<T, 16 / sizeof(T)>(table, rows, C, index, n, scale, out, st);
        else lookup_launch_fwd<T, 1>(table, rows, C, index, n, scale, out, st);
    });
    return check_launch("mvs_lookup_rows_fwd");
}

extern "C" size_t mvs_lookup_rows_workspace_bytes(int64_t rows, int C, int64_t n) {
    if (rows < 1 || C < 1 || n < 0 || rows > 0x7ffffffe || n > 0x7ffffffe) return 0;
    return lookup_plan(rows, C, n).total + 256;
}

extern "C" int mvs_lookup_rows_bwd(const void *grad_out, int dtype, const int64_t *index, int64_t n, int64_t rows, int C, float scale,
                                   void *grad_table, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = lookup_check("mvs_lookup_rows_bwd", grad_table, grad_out, dtype, index, rows, C, n);
    if (rc != MVS_OK) return rc;
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < mvs_lookup_rows_workspace_bytes(rows, C, n)) {
        set_error("mvs_lookup_rows_bwd: workspace too small or not aligned to 16 bytes (%zu of %zu bytes)", workspace_bytes,
                  mvs_lookup_rows_workspace_bytes(rows, C, n));
        return MVS_EWORKSPACE;
    }
    hipStream_t st = as_stream(stream);
    const LookupPlan p = lookup_plan(rows, C, n);
    char *ws = static_cast<char *>(workspace);
    unsigned *keys = reinterpret_cast<unsigned *>(ws + p.keys0), *vals = reinterpret_cast<unsigned *>(ws + p.vals0);
    if (n > 0 && p.passes == 0) {
        hipLaunchKernelGGL(lookup_rank_kernel, dim3((unsigned)((n + 63) / 64)), dim3(256), 0, st, index, (int)n, rows, keys, vals);
    } else if (n > 0) {
        unsigned *keys_to = reinterpret_cast<unsigned *>(ws + p.keys1), *vals_to = reinterpret_cast<unsigned *>(ws + p.vals1);
        unsigned *hist = reinterpret_cast<unsigned *>(ws + p.hist);
        for (int pass = 0; pass < p.passes; ++pass) {
            const int shift = pass * p.digit_bits, bits = min(p.digit_bits, p.key_bits - shift);
            const dim3 grid((unsigned)p.tiles), block(256);
            const int64_t m = p.tiles << bits;
            if (pass == 0) {
                hipLaunchKernelGGL((lookup_count_kernel<true>), grid, block, 0, st, index, keys, n, rows, shift, bits, p.tiles, hist);
                hipLaunchKernelGGL(lookup_scan_kernel, dim3(1), dim3(1024), 0, st, hist, m);
                hipLaunchKernelGGL((lookup_place_kernel<true>), grid, block, 0, st, index, keys, vals, n, rows, shift, bits, p.tiles, hist, keys_to, vals_to);
            } else {
                hipLaunchKernelGGL((lookup_count_kernel<false>), grid, block, 0, st, index, keys, n, rows, shift, bits, p.tiles, hist);
                hipLaunchKernelGGL(lookup_scan_kernel, dim3(1), dim3(1024), 0, st, hist, m);
                hipLaunchKernelGGL((lookup_place_kernel<false>), grid, block, 0, st, index, keys, vals, n, rows, shift, bits, p.tiles, hist, keys_to, vals_to);
            }
            std::swap(keys, keys_to);
            std::swap(vals, vals_to);
        }
    }
    LookupRows a = {};
    a.grad = grad_out; a.keys = keys; a.vals = vals; a.out = grad_table; a.part = reinterpret_cast<float *>(ws + p.part);
    a.n = n; a.rows = rows; a.pieces = p.pieces; a.C = C; a.scale = scale;
    const bool wide = lookup_wide(grad_out, grad_table, dtype, C);
    MVS_DTYPE_DISPATCH(dtype, T, {
        if (wide) lookup_launch_rows<T, 16 / sizeof(T)>(a, st);
        else lookup_launch_rows<T, 1>(a, st);
    });
    return check_launch("mvs_lookup_rows_bwd");
}
