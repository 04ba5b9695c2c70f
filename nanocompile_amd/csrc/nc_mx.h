// The microscaled (MX) formats as the kernels hold them (the Open Compute Project's published
// "Microscaling Formats" specification, v1.0): blocks of 32 values of a row share one scale, a power of two
// kept as its exponent plus 127 in a byte (255 is NaN), times 4-bit (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
// sign) or 8-bit (e4m3: up to 448) floating point elements.
//
// In memory a row is padded with zeros to a multiple of 128 values, the k of one matrix instruction, so the
// products have no tail in k: codes are ceil(K / 128) * 64 or * 128 bytes a row (two 4-bit elements a byte, the
// lower index in the low bits), scales ceil(K / 128) * 4 bytes a row.
//
// The quantizer is exact but for the elements' own rounding: the scale puts the block's largest value into the
// elements' top binade, exponent floor(log2(max |x|)) - 2 (e2m1) or - 8 (e4m3), at least -127; a value times the
// inverse power of two has no rounding, and goes to the nearest element, ties to even, values past the largest
// element to that. A block that holds a NaN or an infinity has scale NaN and zero elements: every value it
// stands for, and every output of a product that reads it, is NaN.
#pragma once

#include "nc_common.h"

namespace nc {

constexpr int kMxBlock = 32, kMxPad = 128, kMxNan = 255;

inline __host__ __device__ int64_t mx_padded(int64_t k) { return (k + kMxPad - 1) / kMxPad * kMxPad; }

// 16 bytes of floats at any address of a float (a row of an odd width starts at one): global memory takes wide
// loads and stores on 4-byte boundaries.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// 4 values from p of which the first `valid` (<= 0: none) are a row's: zeros for the others, which are not read.
__device__ __forceinline__ f32x4 load4(const float *p, int valid) {
    if (valid >= 4) return *reinterpret_cast<const f32x4_any *>(p);
    f32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < valid ? p[j] : 0.0f;
    return v;
}

// KEPT: through the caches as any store, otherwise past them (the last values of a row that are not four excepted).
template <bool KEPT = true>
__device__ __forceinline__ void store4(float *p, f32x4 v, int valid) {
    if (valid >= 4) {
        if constexpr (KEPT) *reinterpret_cast<f32x4_any *>(p) = v;
        else __builtin_nontemporal_store(v, reinterpret_cast<f32x4_any *>(p));
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < valid) p[j] = v[j];
    }
}

// |v| as bits: ordered as the values, an infinity and then the NaNs above them.
__device__ __forceinline__ int32_t magnitude_bits(f32x4 v) {
    int32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_int(v[j]) & 0x7fffffff);
    return m;
}

// A block's scale from its largest magnitude's bits: its exponent field less 2 or 8, at least 0 (an exponent field
// of 0, zero and the subnormals, has floor(log2) < -126 and so the least scale too).
template <int BITS>
__device__ __forceinline__ int mx_scale(int32_t magnitude) {
    return magnitude >= 0x7f800000 ? kMxNan : max((magnitude >> 23) - (BITS == 4 ? 2 : 8), 0);
}

// 4 consecutive values of a block of the given scale to elements, in the low 16 bits or all 32.
// The conversions round to nearest even and keep 4-bit values past 6 at 6 (checked against every rounding
// border); past 464 the 8-bit one would give NaN, hence the clamp. The inverse of a scale 0 .. 252 is the
// normal float of exponent 254 - scale.
template <int BITS>
__device__ __forceinline__ uint32_t mx_encode(f32x4 v, int scale) {
    const float inverse = __uint_as_float((uint32_t)(254 - scale) << 23);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = scale == kMxNan ? 0.0f : __fmul_rn(v[j], inverse);
    if constexpr (BITS == 4) {
        const uint32_t low = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], 1.0f, 0);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(low, v[2], v[3], 1.0f, 1);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __builtin_amdgcn_fmed3f(v[j], -448.0f, 448.0f);
        const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], low, true);
    }
}

// The values 4 elements and their scale stand for: element times power of two, exact unless it overflows or is
// below float32's least subnormal.
template <int BITS>
__device__ __forceinline__ f32x4 mx_decode(uint32_t codes, int scale) {
    // 2^(scale - 127) as a float: subnormal for scale 0, NaN for 255
    const float power = __uint_as_float(scale == 0        ? 0x00400000u
                                        : scale == kMxNan ? 0x7fc00000u
                                                          : (uint32_t)scale << 23);
    f32x4 v;
    auto put = [&](int j, auto pair) { v[j] = __fmul_rn(pair[0], power), v[j + 1] = __fmul_rn(pair[1], power); };
    if constexpr (BITS == 4) {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1));
    } else {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, 1.0f, false));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, 1.0f, true));
    }
    return v;
}

// Workgroups of a launch over two dimensions of the grid, so that none of them has 2^32 threads or more.
constexpr int64_t kGridRow = 1 << 16;
inline dim3 grid_of(int64_t workgroups) {
    return dim3((unsigned)(workgroups < kGridRow ? workgroups : kGridRow),
                (unsigned)((workgroups + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ int64_t workgroup_id() { return (int64_t)blockIdx.y * kGridRow + blockIdx.x; }

inline bool aligned(const void *p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace nc
