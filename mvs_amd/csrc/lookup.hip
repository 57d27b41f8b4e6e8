// Rows of a table by index, scaled, and the table's gradient by sorted indices.
//
//   out[i] = s T[index i]            grad T[v] = s sum over {i : index i = v}, in the order of i, of g[i]
//
// Forward: bound by the rows it reads and writes; 16 bytes per lane, a power-of-two number of lanes per row (65536 of 128000 rows of
// 4 KiB, a few of them most of the batch: 91 us; 1021 rows of 128 bytes: 2.4 us).
//
// Backward: every row of the dense gradient is written once, most of them as zeros, and every row of g is read once.  Who adds to a
// row is known only after the indices are sorted.  The sort is stable, so a row's terms come in the order of i and equal calls
// give equal bits; floating-point atomics on the rows would need neither sort nor order, but sum in another order every time.
//   sort   up to kRankMax indices: the place of term i is the number of (key, i) below its own -- one launch, n^2 comparisons of two
//          instructions; more: least-significant-digit radix sort, digits of up to 10 bits, three launches each (count per tile, one
//          workgroup's scan, place).
//   rows   the sorted terms are cut into pieces of 16 to 128; a piece's lanes walk it with the loads of 8 terms in flight and write
//          the sum of each run of equal keys that lies within the piece.  A run that leaves the piece (a frequent index) leaves
//          float32 partial sums, at most two per piece.  The same launch writes the zero rows (found by binary search, 64 table
//          rows per wave's worth of lanes).
//   join   the partial sums of the runs that leave their piece, in order: short runs a wave each, long ones four spans of pieces at
//          a time.  A run's end is found 64 pieces per look.
// Bound by memory for large ones: 65536 rows of 4 KiB into 128000, a few of them most of the batch (268 MB read, 524 MB written): sort
// 32 us, rows 170 us (4.7 TB/s), join 21 us; by latency for small ones: 1021 rows of 128 bytes into 20480 sort 5.8, rows 7, join
// 3.4 us.  The rank sort takes 5.8 us for 1021 and 16.9 us for 8191 indices, where the radix sort's six launches take 32.
#include <utility>

#include "dtype.h"

namespace mvs {

constexpr int kRankMax = 8192;
constexpr int kJoin = 16;          // pieces that a workgroup of the join looks at
constexpr int kMaxDigit = 10;

struct LookupPlan {
    int64_t n, rows;
    int key_bits, passes, digit_bits;
    int tile;                     // keys per workgroup of a radix pass: small while that fills the chip, large before the scan of the counts is long
    int terms;                    // sorted terms per piece
    int64_t tiles, pieces;
    size_t keys0, vals0, keys1, vals1, hist, part, total;      // byte offsets into the workspace
};

static LookupPlan lookup_plan(int64_t rows, int C, int64_t n) {
    LookupPlan p = {};
    p.n = n; p.rows = rows;
    while (p.key_bits < 32 && ((int64_t)1 << p.key_bits) <= rows) ++p.key_bits;      // keys 0 .. rows (rows: names no row)
    p.passes = n <= kRankMax ? 0 : (p.key_bits + kMaxDigit - 1) / kMaxDigit;
    p.digit_bits = p.passes ? (p.key_bits + p.passes - 1) / p.passes : 0;
    p.tile = n <= 131072 ? 1024 : 4096;
    p.tiles = (n + p.tile - 1) / p.tile;
    // Short pieces fill the chip, long ones leave fewer partial sums: 65536 x 2048 bfloat16 into 128000 rows 227 / 217 / 245 us by pieces
    // of 16 / 32 / 64 where the indices are spread evenly, 290 / 242 / 254 where a few are frequent; 10^6 x 64 float32 171 / 146 / 135
    // and 440 / 276 / 205.
    p.terms = n <= 1 << 14 ? 16 : n <= 1 << 18 ? 32 : n <= 1 << 22 ? 64 : 128;
    p.pieces = (n + p.terms - 1) / p.terms;
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
    const int64_t i = group_of() * (256 / lanes) + threadIdx.x / lanes;
    if (i >= n) return;
    const int64_t row = index[i];
    const bool named = row >= 0 && row < rows;
    const Pack<T, VEC> *from = reinterpret_cast<const Pack<T, VEC> *>(table + (named ? row : 0) * C);
    Pack<T, VEC> *to = reinterpret_cast<Pack<T, VEC> *>(out + i * C);
    for (int c0 = lane; c0 < vecs; c0 += 4 * lanes) {
        Pack<T, VEC> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (named && c0 + u * lanes < vecs) v[u] = from[c0 + u * lanes];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (c0 + u * lanes >= vecs) break;
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[u].v[j] = from_float<T>(named ? to_float(v[u].v[j]) * scale : 0.0f);
            to[c0 + u * lanes] = v[u];
        }
    }
}

// ---- sort
// 64 terms per workgroup, each of 16 waves against a sixteenth of the keys; the keys pass through LDS 2048 at a time.
__global__ __launch_bounds__(1024) void lookup_rank_kernel(const int64_t *__restrict__ index, int n, int64_t rows, unsigned *__restrict__ keys,
                                                           unsigned *__restrict__ vals) {
    __shared__ unsigned long long tile[2048];
    __shared__ int ranks[1024];
    const int tid = threadIdx.x, i = blockIdx.x * 64 + (tid & 63), wave = tid >> 6;
    auto key_of = [&](int j) { return j < n ? (unsigned long long)lookup_key(index[j], rows) << 32 | (unsigned)j : ~0ull; };
    const unsigned long long mine = key_of(i);
    int rank = 0;
    for (int base = 0; base < n; base += 2048) {
        __syncthreads();
        tile[tid] = key_of(base + tid);
        tile[tid + 1024] = key_of(base + tid + 1024);
        __syncthreads();
        const ulonglong2 *t2 = reinterpret_cast<const ulonglong2 *>(tile + wave * 128);
#pragma unroll 16
        for (int j = 0; j < 64; ++j) {
            const ulonglong2 k = t2[j];      // (one address for the wave)
            rank += (k.x < mine) + (k.y < mine);
        }
    }
    ranks[tid] = rank;
    __syncthreads();
    if (wave == 0 && i < n) {
        int r = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) r += ranks[w * 64 + tid];
        keys[r] = (unsigned)(mine >> 32);
        vals[r] = (unsigned)i;
    }
}

// counts per (digit, tile), digit-major: their exclusive scan is where a tile's keys of a digit go
template <bool FIRST>
__global__ __launch_bounds__(256) void lookup_count_kernel(const int64_t *__restrict__ index, const unsigned *__restrict__ keys, int64_t n,
                                                           int64_t rows, int shift, int bits, int64_t tiles, int tile, unsigned *__restrict__ hist) {
    __shared__ unsigned count[1 << kMaxDigit];
    const int digits = 1 << bits;
    for (int d = threadIdx.x; d < digits; d += 256) count[d] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * tile;
#pragma unroll 4
    for (int u = 0; u < tile / 256; ++u) {
        const int64_t i = base + u * 256 + threadIdx.x;
        if (i < n) {
            const unsigned key = FIRST ? lookup_key(index[i], rows) : keys[i];
            atomicAdd(&count[key >> shift & (digits - 1)], 1u);      // (whole numbers: their order does not matter)
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 256) hist[(int64_t)d * tiles + blockIdx.x] = count[d];
}

// exclusive scan of `m` counts in place, by one workgroup: a wave takes 1024 consecutive ones, 256 at a time.  (The last access of
// four may reach behind m, not behind the 256 bytes its region is rounded up to.)
__global__ __launch_bounds__(1024) void lookup_scan_kernel(unsigned *__restrict__ hist, int64_t m) {
    __shared__ unsigned sums[16];
    unsigned carry = 0;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t base = 0; base < m; base += 16384) {
        uint4 v[4];
        unsigned before[4], all = 0;      // of the wave's range: what lies before this lane's four, and its sum
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t at = base + wave * 1024 + r * 256 + lane * 4;
            v[r] = at < m ? *reinterpret_cast<const uint4 *>(hist + at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const unsigned sum = v[r].x + v[r].y + v[r].z + v[r].w;
            unsigned incl = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const unsigned t = (unsigned)__shfl_up((int)incl, o);
                if (lane >= o) incl += t;
            }
            before[r] = all + incl - sum;
            all += (unsigned)__shfl((int)incl, 63);
        }
        if (lane == 0) sums[wave] = all;
        __syncthreads();
        unsigned ahead = carry, total = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) { if (w < wave) ahead += sums[w]; total += sums[w]; }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t at = base + wave * 1024 + r * 256 + lane * 4;
            const unsigned x = ahead + before[r], y = x + v[r].x, z = y + v[r].y, w = z + v[r].z;
            if (at < m) *reinterpret_cast<uint4 *>(hist + at) = make_uint4(x, y, z, w);
        }
        carry += total;
        __syncthreads();
    }
}

__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Places a tile's keys: 4 waves, each a quarter of them in ROUNDS rounds of 64.  A key's place is the tile's start of its digit,
// plus the earlier waves' count of it, plus the wave's own earlier ones, plus the lanes in front of it that hold the same digit.
template <bool FIRST, int ROUNDS>
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
    const int64_t base = ((int64_t)blockIdx.x * 4 + wave) * (ROUNDS * 64);
    unsigned key[ROUNDS];
#pragma unroll
    for (int u = 0; u < ROUNDS; ++u) {
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
    for (int u = 0; u < ROUNDS; ++u) {
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
    int C, lanes, terms;
    float scale;
};

// Workgroups 0 .. sum_groups - 1 sum pieces (256 / lanes pieces each), the rest write zero rows (64 table rows each).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void lookup_rows_kernel(LookupRows a) {
    const int tid = threadIdx.x, lane = tid & (a.lanes - 1), vecs = a.C / VEC;
    T *out = static_cast<T *>(a.out);
    const int64_t group = group_of();
    if (group >= a.sum_groups) {
        __shared__ unsigned long long empty_rows;
        const int64_t v0 = (group - a.sum_groups) * 64;
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
    const int64_t piece = group * (256 / a.lanes) + tid / a.lanes;
    if (piece >= a.pieces) return;
    const int64_t p0 = piece * a.terms;
    const int count = (int)(a.n - p0 < a.terms ? a.n - p0 : a.terms);
    const unsigned none = (unsigned)a.rows;
    const unsigned before = p0 > 0 ? a.keys[p0 - 1] : 0xffffffffu;
    const T *grad = static_cast<const T *>(a.grad);
    // eight terms and the key behind them, read while the eight before them are summed
    struct Terms { unsigned key[9], val[8]; };
    auto terms_at = [&](int from) {
        Terms t;
#pragma unroll
        for (int k = 0; k < 9; ++k) t.key[k] = from + k <= count && p0 + from + k < a.n ? a.keys[p0 + from + k] : 0xffffffffu;
#pragma unroll
        for (int k = 0; k < 8; ++k) t.val[k] = from + k < count ? a.vals[p0 + from + k] : 0u;
        return t;
    };
    const Terms head = terms_at(0);
    for (int c = lane; c < vecs; c += a.lanes) {
        float sum[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
        bool from_before = head.key[0] == before;
        Terms now = head;
        for (int from = 0; from < count; from += 8) {
            Pack<T, VEC> g[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (from + k < count && now.key[k] != none)
                    g[k] = reinterpret_cast<const Pack<T, VEC> *>(grad + (int64_t)now.val[k] * a.C)[c];
            const Terms then = terms_at(from + 8);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const unsigned key = now.key[k];
                if (from + k >= count || key == none) continue;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] += to_float(g[k].v[j]);
                const bool last = from + k == count - 1;
                if (!last && now.key[k + 1] == key) continue;
                const bool goes_on = last && now.key[k + 1] == key;
                if (from_before || goes_on) {
                    // (a run that fills the piece and leaves it on both sides counts as coming from before)
                    float *to = a.part + (piece * 2 + (from_before ? 0 : 1)) * a.C + c * VEC;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) to[j] = sum[j];
                } else {
                    Pack<T, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) o.v[j] = from_float<T>(sum[j] * a.scale);
                    put(reinterpret_cast<Pack<T, VEC> *>(out + (int64_t)key * a.C) + c, o);
                }
                from_before = false;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
            }
            now = then;
        }
    }
}

// The partial sums of a run that begins in piece p and goes on: p's second one, and the first ones of the pieces behind it that begin
// with its key.  A workgroup looks at kJoin pieces and owns 64 * VEC columns.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void lookup_join_kernel(LookupRows a) {
    __shared__ Pack<float, VEC> spans[4][64];
    constexpr int LONG = 16;      // pieces from which the four waves share a run
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = (blockIdx.y * 64 + lane) * VEC;
    const int64_t p0 = (int64_t)blockIdx.x * kJoin, mine = p0 + lane;
    bool owner = lane < kJoin && mine < a.pieces - 1, longer = false;      // (the last piece goes on nowhere; the others are full)
    unsigned my_key = 0;
    if (owner) {
        const int64_t first = mine * a.terms, end = first + a.terms, probe = end + (LONG - 1) * a.terms;
        my_key = a.keys[end - 1];
        const unsigned next = a.keys[end], head = a.keys[first], before = first > 0 ? a.keys[first - 1] : ~0u, far = probe < a.n ? a.keys[probe] : ~0u;
        owner = my_key != (unsigned)a.rows && next == my_key && !(head == my_key && before == my_key);
        longer = owner && far == my_key;
    }
    const unsigned long long owners = __ballot(owner && !longer);      // (the same in all four waves)
    unsigned long long long_ones = __ballot(longer);
    auto length = [&](int64_t piece, unsigned key) {          // pieces behind `piece` that begin with its last key
        int64_t more = 0;
        while (true) {
            const int64_t q = piece + 1 + more + lane;
            const unsigned long long same = __ballot(q < a.pieces && a.keys[q * a.terms] == key);
            if (same != ~0ull) return more + __builtin_ctzll(~same);
            more += 64;
        }
    };
    auto add = [&](float (&sum)[VEC], int64_t from, int64_t to) {      // first partials of pieces [from, to)
        for (int64_t q = from; q < to; q += 8) {
            Pack<float, VEC> v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (q + j < to) v[j] = *reinterpret_cast<const Pack<float, VEC> *>(a.part + (q + j) * 2 * a.C + col);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (q + j < to)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) sum[e] += v[j].v[e];
        }
    };
    auto write = [&](const float (&sum)[VEC], unsigned key) {
        Pack<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.v[e] = from_float<T>(sum[e] * a.scale);
        *reinterpret_cast<Pack<T, VEC> *>(static_cast<T *>(a.out) + (int64_t)key * a.C + col) = o;
    };
    auto begin = [&](float (&sum)[VEC], int64_t piece) {
        const Pack<float, VEC> v = *reinterpret_cast<const Pack<float, VEC> *>(a.part + (piece * 2 + 1) * a.C + col);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] = v.v[e];
    };
    // short runs: every fourth one a wave's
    int turn = 0;
    for (unsigned long long left = owners; left; left &= left - 1, ++turn) {
        if ((turn & 3) != wave) continue;
        const int at = __builtin_ctzll(left);
        const int64_t piece = p0 + at;
        const unsigned key = (unsigned)__shfl((int)my_key, at);
        const int64_t more = length(piece, key);
        if (col < a.C) {
            float sum[VEC];
            begin(sum, piece);
            add(sum, piece + 1, piece + 1 + more);
            write(sum, key);
        }
    }
    for (; long_ones; long_ones &= long_ones - 1) {
        const int at = __builtin_ctzll(long_ones);
        const int64_t piece = p0 + at;
        const unsigned key = (unsigned)__shfl((int)my_key, at);
        const int64_t more = length(piece, key), each = (more + 3) / 4;
        float sum[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] = 0.0f;
        if (col < a.C) {
            if (wave == 0) begin(sum, piece);
            const int64_t from = piece + 1 + wave * each;
            add(sum, from, min(piece + 1 + more, from + each));
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) spans[wave][lane].v[e] = sum[e];
        __syncthreads();
        if (wave == 0 && col < a.C) {
#pragma unroll
            for (int w = 1; w < 4; ++w)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[e] += spans[w][lane].v[e];
            write(sum, key);
        }
    }
}

static int lookup_check(const char *who, const void *table, const void *wide, int dtype, const int64_t *index, int64_t rows, int C, int64_t n) {
    if (n < 0 || rows < 1 || C < 1 || dtype_size(dtype) == 0 || !table || (n > 0 && (!wide || !index))) {
        set_error("%s: invalid argument (rows=%lld, C=%d, n=%lld, dtype=%d)", who, (long long)rows, C, (long long)n, dtype);
        return MVS_EINVAL;
    }
    if (rows > 0x7ffffffe || n > 0x7ffffffe || C > (1 << 20)) {
        set_error("%s: rows=%lld, n=%lld (at most 2^31 - 2 each), C=%d (at most 2^20)", who, (long long)rows, (long long)n, C);
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
    const int lanes = min(64, lookup_lanes(C / VEC));      // (four accesses of a long row in flight per lane)
    hipLaunchKernelGGL((lookup_fwd_kernel<T, VEC>), grid_of((n * lanes + 255) / 256), dim3(256), 0, st, static_cast<const T *>(table), rows, C, index,
                       n, scale, static_cast<T *>(out), lanes);
}

template <typename T, int VEC>
static void lookup_launch_rows(LookupRows a, hipStream_t st) {
    a.lanes = lookup_lanes(a.C / VEC);
    a.sum_groups = (a.pieces * a.lanes + 255) / 256;
    const int64_t zero_groups = (a.rows + 63) / 64;
    hipLaunchKernelGGL((lookup_rows_kernel<T, VEC>), grid_of(a.sum_groups + zero_groups), dim3(256), 0, st, a);
    if (a.pieces > 1) {
        constexpr int JOIN = VEC == 1 ? 1 : 4;      // (rows of whole 16 bytes are whole float4 of sums)
        hipLaunchKernelGGL((lookup_join_kernel<T, JOIN>), dim3((unsigned)((a.pieces + kJoin - 1) / kJoin), (unsigned)((a.C + 64 * JOIN - 1) / (64 * JOIN))), dim3(256), 0, st, a);
    }
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
    if (rows < 1 || C < 1 || n < 0 || rows > 0x7ffffffe || n > 0x7ffffffe || C > (1 << 20)) return 0;
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
        hipLaunchKernelGGL(lookup_rank_kernel, dim3((unsigned)((n + 63) / 64)), dim3(1024), 0, st, index, (int)n, rows, keys, vals);
    } else if (n > 0) {
        unsigned *keys_to = reinterpret_cast<unsigned *>(ws + p.keys1), *vals_to = reinterpret_cast<unsigned *>(ws + p.vals1);
        unsigned *hist = reinterpret_cast<unsigned *>(ws + p.hist);
        auto count = [&](auto kernel, int shift, int bits) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)p.tiles), dim3(256), 0, st, index, keys, n, rows, shift, bits, p.tiles, p.tile, hist);
            hipLaunchKernelGGL(lookup_scan_kernel, dim3(1), dim3(1024), 0, st, hist, p.tiles << bits);
        };
        auto place = [&](auto kernel, int shift, int bits) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)p.tiles), dim3(256), 0, st, index, keys, vals, n, rows, shift, bits, p.tiles, hist, keys_to, vals_to);
        };
        for (int pass = 0; pass < p.passes; ++pass) {
            const int shift = pass * p.digit_bits, bits = min(p.digit_bits, p.key_bits - shift);
            const bool small = p.tile == 1024;
            if (pass == 0) {
                count(lookup_count_kernel<true>, shift, bits);
                if (small) place(lookup_place_kernel<true, 4>, shift, bits);
                else place(lookup_place_kernel<true, 16>, shift, bits);
            } else {
                count(lookup_count_kernel<false>, shift, bits);
                if (small) place(lookup_place_kernel<false, 4>, shift, bits);
                else place(lookup_place_kernel<false, 16>, shift, bits);
            }
            std::swap(keys, keys_to);
            std::swap(vals, vals_to);
        }
    }
    LookupRows a = {};
    a.grad = grad_out; a.keys = keys; a.vals = vals; a.out = grad_table; a.part = reinterpret_cast<float *>(ws + p.part);
    a.n = n; a.rows = rows; a.pieces = p.pieces; a.terms = p.terms; a.C = C; a.scale = scale;
    const bool wide = lookup_wide(grad_out, grad_table, dtype, C);
    MVS_DTYPE_DISPATCH(dtype, T, {
        if (wide) lookup_launch_rows<T, 16 / sizeof(T)>(a, st);
        else lookup_launch_rows<T, 1>(a, st);
    });
    return check_launch("mvs_lookup_rows_bwd");
}
