// An activation held in 8 bits for the backward pass: to codes and scales, and back (act8.h has the form).
//
// Both directions are bound by the memory they move, n (e + 1 + 1/32) bytes for elements of e bytes.  A lane moves 16 bytes of
// the wide side per access, so a block of 32 is 8 lanes (float32) or 4 (16 bits) and its maximum a few lane exchanges; kUnroll
// accesses of a lane are issued together.  16.9 million bfloat16 values: to codes 12.4 us, back 9.4 us (4.1 and 5.5 TB/s; a copy of
// memory of that size moves 5.1); 655360 float32 values, a feature map: 3.6 and 3.2 us, which is what an empty launch takes.
#include "act8.h"
#include "dtype.h"

namespace mvs {

constexpr int kUnroll = 4;

// Any alignment, and the ragged block behind the whole ones: 8 blocks from `block0` on, 32 lanes each, one value a lane.
template <typename T>
__device__ __forceinline__ void act8_quantize_lanes(const T *__restrict__ x, int64_t n, int64_t block0, signed char *__restrict__ codes,
                                                    unsigned char *__restrict__ scales) {
    const int64_t b = block0 + threadIdx.x / 32, i = b * kAct8Block + threadIdx.x % 32;
    const float f = i < n ? to_float(x[i]) : 0.0f;
    unsigned amax = __float_as_uint(f) & 0x7fffffffu;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) amax = umax_xor(amax, o);
    const unsigned byte = act8_scale_byte(amax);
    if (i >= n) return;
    codes[i] = byte == kAct8Nan ? (signed char)0 : (signed char)act8_code(f, act8_inverse(byte));
    if (threadIdx.x % 32 == 0) scales[b] = (unsigned char)byte;
}

// One 16-byte vector of the tensor per lane and step over the `whole` blocks that are moved so (0: off alignment); the workgroups behind
// theirs take the other blocks value by value.
template <typename T>
__global__ __launch_bounds__(256) void act8_quantize_kernel(const T *__restrict__ x, int64_t n, int64_t whole, int64_t groups, signed char *__restrict__ codes,
                                                            unsigned char *__restrict__ scales) {
    const int64_t group = group_of();
    if (group >= groups) {
        act8_quantize_lanes(x, n, whole + (group - groups) * 8, codes, scales);
        return;
    }
    constexpr int VEC = 16 / sizeof(T), LANES = kAct8Block / VEC;
    const int64_t n_vec = whole * LANES;
    const int64_t first = group * 256 * kUnroll + threadIdx.x;
    Pack<T, VEC> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = first + u * 256;
        if (i < n_vec) v[u] = reinterpret_cast<const Pack<T, VEC> *>(x)[i];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = first + u * 256;
        if (i >= n_vec) continue;                      // (whole blocks of lanes leave together: n_vec is a multiple of LANES)
        float f[VEC];
        unsigned amax = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            f[j] = to_float(v[u].v[j]);
            amax = max(amax, __float_as_uint(f[j]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) amax = umax_xor(amax, o);
        const unsigned byte = act8_scale_byte(amax);
        const float inv = byte == kAct8Nan ? 0.0f : act8_inverse(byte);
        Pack<unsigned, VEC / 4> q;
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
            q.v[j / 4] = byte == kAct8Nan ? 0u
                                          : act8_pack4(act8_code(f[j], inv), act8_code(f[j + 1], inv), act8_code(f[j + 2], inv), act8_code(f[j + 3], inv));
        reinterpret_cast<Pack<unsigned, VEC / 4> *>(codes)[i] = q;
        if (i % LANES == 0) scales[i / LANES] = (unsigned char)byte;
    }
}

template <typename T>
__device__ __forceinline__ T act8_back(float v) {
    constexpr float most = DtypeMax<T>::value;
    return from_float<T>(v > most ? most : v < -most ? -most : v);      // (a NaN passes both comparisons)
}

template <typename T>
__global__ __launch_bounds__(256) void act8_dequantize_kernel(const signed char *__restrict__ codes, const unsigned char *__restrict__ scales,
                                                              int64_t n, int64_t whole, int64_t groups, T *__restrict__ out) {
    const int64_t group = group_of();
    if (group >= groups) {
        const int64_t i = whole * kAct8Block + (group - groups) * 256 + threadIdx.x;
        if (i < n) out[i] = act8_back<T>((float)codes[i] * act8_step(scales[i / kAct8Block]));
        return;
    }
    constexpr int VEC = 16 / sizeof(T), LANES = kAct8Block / VEC;
    const int64_t n_vec = whole * LANES;
    const int64_t first = group * 256 * kUnroll + threadIdx.x;
    Pack<unsigned, VEC / 4> q[kUnroll];
    unsigned byte[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = first + u * 256;
        if (i < n_vec) {
            q[u] = reinterpret_cast<const Pack<unsigned, VEC / 4> *>(codes)[i];
            byte[u] = scales[i / LANES];
        }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = first + u * 256;
        if (i >= n_vec) continue;
        const float step = act8_step(byte[u]);
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.v[j] = act8_back<T>(act8_value(q[u].v[j / 4], j % 4, step));
        reinterpret_cast<Pack<T, VEC> *>(out)[i] = o;
    }
}

static int act8_check(const char *who, const void *wide, int dtype, int64_t n, const void *codes, const void *scales) {
    if (n < 0 || (n > 0 && (!wide || !codes || !scales)) || dtype_size(dtype) == 0) {
        set_error("%s: invalid argument (n=%lld, dtype=%d)", who, (long long)n, dtype);
        return MVS_EINVAL;
    }
    if ((reinterpret_cast<uintptr_t>(wide) & (dtype_size(dtype) - 1)) != 0) {
        set_error("%s: the tensor is not aligned to its element size", who);
        return MVS_EINVAL;
    }
    if (n > (int64_t)1 << 38) {
        set_error("%s: n=%lld is beyond 2^38", who, (long long)n);
        return MVS_EUNSUPPORTED;
    }
    return MVS_OK;
}
// both kernels' wide path: 16-byte accesses of the tensor, 4- or 8-byte accesses of the codes
static bool act8_wide(const void *wide, const void *codes) { return aligned16(wide) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0; }

}  // namespace mvs

using namespace mvs;

extern "C" int mvs_act8_quantize(const void *x, int dtype, int64_t n, signed char *codes, unsigned char *scales, void *stream) {
    const int rc = act8_check("mvs_act8_quantize", x, dtype, n, codes, scales);
    if (rc != MVS_OK || n == 0) return rc;
    hipStream_t st = as_stream(stream);
    const int64_t whole = act8_wide(x, codes) ? n / kAct8Block : 0, blocks = (n + kAct8Block - 1) / kAct8Block;
    MVS_DTYPE_DISPATCH(dtype, T, {
        const int64_t groups = (whole * (kAct8Block * (int)sizeof(T) / 16) + 256 * kUnroll - 1) / (256 * kUnroll), rest = (blocks - whole + 7) / 8;
        hipLaunchKernelGGL((act8_quantize_kernel<T>), grid_of(groups + rest), dim3(256), 0, st, static_cast<const T *>(x), n, whole, groups, codes, scales);
    });
    return check_launch("mvs_act8_quantize");
}

extern "C" int mvs_act8_dequantize(const signed char *codes, const unsigned char *scales, int64_t n, int dtype, void *out, void *stream) {
    const int rc = act8_check("mvs_act8_dequantize", out, dtype, n, codes, scales);
    if (rc != MVS_OK || n == 0) return rc;
    hipStream_t st = as_stream(stream);
    const int64_t whole = act8_wide(out, codes) ? n / kAct8Block : 0;
    MVS_DTYPE_DISPATCH(dtype, T, {
        const int64_t groups = (whole * (kAct8Block * (int)sizeof(T) / 16) + 256 * kUnroll - 1) / (256 * kUnroll), rest = (n - whole * kAct8Block + 255) / 256;
        hipLaunchKernelGGL((act8_dequantize_kernel<T>), grid_of(groups + rest), dim3(256), 0, st, codes, scales, n, whole, groups, static_cast<T *>(out));
    });
    return check_launch("mvs_act8_dequantize");
}
