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

// 16 and 8 bytes of floats at any address of a float (a row of an odd width starts at one): global memory
// takes wide loads and stores on 4-byte boundaries.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 8 values from p of which the first `valid` (<= 0: none) are a row's: zeros for the others, which are not read.
__device__ __forceinline__ void load8(float (&v)[8], const float *p, int valid) {
    if (valid >= 8) {
        const f32x4 a = *reinterpret_cast<const f32x4_any *>(p), b = *reinterpret_cast<const f32x4_any *>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < valid ? p[j] : 0.0f;
    }
}

__device__ __forceinline__ void store8(float *p, const float (&v)[8], int valid) {
    if (valid >= 8) {
        *reinterpret_cast<f32x4_any *>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_any *>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) p[j] = v[j];
    }
}

// |v| as bits: ordered as the values, an infinity and then the NaNs above them.
__device__ __forceinline__ int32_t magnitude_bits(const float (&v)[8]) {
    int32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_int(v[j]) & 0x7fffffff);
    return m;
}

// A block's scale from its largest magnitude's bits: its exponent field less 2 or 8, at least 0 (an exponent field
// of 0, zero and the subnormals, has floor(log2) < -126 and so the least scale too).
template <int BITS>
__device__ __forceinline__ int mx_scale(int32_t magnitude) {
    return magnitude >= 0x7f800000 ? kMxNan : max((magnitude >> 23) - (BITS == 4 ? 2 : 8), 0);
}

// 8 consecutive values of a block of the given scale to elements: 4 bytes, or 8 (the second word 0 in 4 bits).
// The conversions round to nearest even and keep 4-bit values past 6 at 6 (checked against every rounding
// border); past 464 the 8-bit one would give NaN, hence the clamp. The inverse of a scale 0 .. 252 is the
// normal float of exponent 254 - scale.
template <int BITS>
__device__ __forceinline__ u32x2 mx_encode(const float (&v)[8], int scale) {
    const float inverse = __uint_as_float((uint32_t)(254 - scale) << 23);
    float t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = scale == kMxNan ? 0.0f : __fmul_rn(v[j], inverse);
    u32x2 out = {0u, 0u};
    if constexpr (BITS == 4) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[0], t[1], 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[2], t[3], 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[4], t[5], 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, t[6], t[7], 1.0f, 3);
        out[0] = w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = __builtin_amdgcn_fmed3f(t[j], -448.0f, 448.0f);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * h], t[4 * h + 1], 0, false);
            out[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(t[4 * h + 2], t[4 * h + 3], w, true);
        }
    }
    return out;
}

// The values 8 elements and their scale stand for: element times power of two, exact unless it overflows or is
// below float32's least subnormal.
template <int BITS>
__device__ __forceinline__ void mx_decode(float (&v)[8], u32x2 codes, int scale) {
    // 2^(scale - 127) as a float: subnormal for scale 0, NaN for 255
    const float power = __uint_as_float(scale == 0 ? 0x00400000u : scale == kMxNan ? 0x7fc00000u : (uint32_t)scale << 23);
    auto put = [&](int j, auto pair) { v[j] = pair[0], v[j + 1] = pair[1]; };
    if constexpr (BITS == 4) {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 0));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 1));
        put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 2));
        put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], 1.0f, 3));
    } else {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[0], 1.0f, false));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[0], 1.0f, true));
        put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[1], 1.0f, false));
        put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[1], 1.0f, true));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], power);
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
