// The microscaled formats' row kernels (nc_mx.h has the formats): the quantizer, its inverse, and the residual's
// addition with rms_norm and a quantized output.
//
// Everything here reads and writes each value once and is bound by memory. Where float32 is written a lane takes 4
// consecutive values, so that a wave's store is 1 KB in a row, and the store goes past the caches: whole lines leave
// quicker so, also for a kernel that reads them next (8192 x 8192 from 4 bits: 42 us, 65 through the caches; with a
// pass over the values behind it 102 and 118. Of 8 values a lane, half lines: 103 and 60). The quantizer, which
// writes less than it reads, takes 8 a lane (4096 x 4096 to 4 bits 12.0 us, 14.1 with 4).
#include "nc_mx.h"

namespace {

using nc::f32x4;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;

// A block's largest magnitude from its LANES lanes'.
template <int LANES>
__device__ __forceinline__ int32_t block_magnitude(int32_t magnitude) {
    return nc::butterfly<LANES>(magnitude, [](int32_t a, int32_t b) { return max(a, b); });
}

// A thread a chunk of the padded rows, in order. The row and column of a workgroup's first chunk come from one
// division on the scalar unit; its threads add theirs to the column in 32 bits.
struct Chunk {
    int64_t row;
    uint32_t at;         // in the row
};

__device__ __forceinline__ Chunk chunk_of(int64_t first, uint32_t per_row) {
    const int64_t row = first / per_row;
    const uint32_t at = (uint32_t)(first - row * per_row) + threadIdx.x;
    return {row + at / per_row, at % per_row};
}

constexpr int kQuantized = 8, kDequantized = 4;        // values a chunk

template <int BITS>
__global__ __launch_bounds__(kThreads) void quantize_mx(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                        const float *__restrict__ x, int64_t M, int K,
                                                        uint32_t per_row) {
    const Chunk c = chunk_of(nc::workgroup_id() * kThreads, per_row);
    if (c.row >= M) return;                            // whole groups of four: a row has a multiple of 16 chunks
    const float *p = x + (size_t)c.row * K + (size_t)c.at * 8;
    const int valid = K - (int)c.at * 8;
    const f32x4 low = nc::load4(p, valid), high = nc::load4(p + 4, valid - 4);
    const int scale = nc::mx_scale<BITS>(block_magnitude<4>(max(nc::magnitude_bits(low), nc::magnitude_bits(high))));
    const u32x2 held = {nc::mx_encode<BITS>(low, scale), nc::mx_encode<BITS>(high, scale)};
    const size_t chunk = (size_t)c.row * per_row + c.at;
    if constexpr (BITS == 4) reinterpret_cast<uint32_t *>(codes)[chunk] = held[0] | held[1] << 16;
    else reinterpret_cast<u32x2 *>(codes)[chunk] = held;
    if (c.at % 4 == 0) scales[chunk / 4] = (uint8_t)scale;
}

template <int BITS>
__global__ __launch_bounds__(kThreads) void dequantize_mx(float *__restrict__ x, const uint8_t *__restrict__ codes,
                                                          const uint8_t *__restrict__ scales, int64_t M, int K,
                                                          uint32_t per_row) {
    const Chunk c = chunk_of(nc::workgroup_id() * kThreads, per_row);
    if (c.row >= M) return;
    const size_t chunk = (size_t)c.row * per_row + c.at;
    uint32_t held;
    if constexpr (BITS == 4) held = reinterpret_cast<const uint16_t *>(codes)[chunk];
    else held = reinterpret_cast<const uint32_t *>(codes)[chunk];
    nc::store4<false>(x + (size_t)c.row * K + (size_t)c.at * 4, nc::mx_decode<BITS>(held, scales[chunk / 8]),
                      K - (int)c.at * 4);
}

// f64 sum over a wavefront: the xor butterfly on both halves of each value.
__device__ __forceinline__ double wave_sum_f64(double v) {
    auto step = [](double v, auto off) {
        constexpr int OFF = decltype(off)::value;
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
        if constexpr (OFF >= 16) {
            const auto a = OFF == 32 ? __builtin_amdgcn_permlane32_swap(lo, lo, false, false)
                                     : __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
            const auto b = OFF == 32 ? __builtin_amdgcn_permlane32_swap(hi, hi, false, false)
                                     : __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
            return __builtin_bit_cast(double, (uint64_t)a[0] | (uint64_t)b[0] << 32) +
                   __builtin_bit_cast(double, (uint64_t)a[1] | (uint64_t)b[1] << 32);
        } else {
            const uint32_t a = (uint32_t)nc::xor_partner<OFF>((int32_t)lo);
            const uint32_t b = (uint32_t)nc::xor_partner<OFF>((int32_t)hi);
            return v + __builtin_bit_cast(double, (uint64_t)a | (uint64_t)b << 32);
        }
    };
    v = step(v, std::integral_constant<int, 32>{});
    v = step(v, std::integral_constant<int, 16>{});
    v = step(v, std::integral_constant<int, 8>{});
    v = step(v, std::integral_constant<int, 4>{});
    v = step(v, std::integral_constant<int, 2>{});
    return step(v, std::integral_constant<int, 1>{});
}

struct NormArgs {
    float *sum, *normed;             // either may be NULL; sum may be x or delta
    uint8_t *q;                      // int8 rows of K, or codes of padded rows
    void *qs;                        // float32 a row, or scales of padded rows
    const float *x, *delta, *gamma;  // delta may be NULL
    int64_t M;
    int K;
    float eps;
};

// t = x + delta; normed = (t * r) * gamma, r = 1 / sqrt(sum(t * t) / K + eps); then int8 with the token's scale
// (FORMAT 0, as nc_rms_norm_quant quantizes) or MX elements of FORMAT bits.
//
// The sum of squares runs in 64 bits (a product of two floats is exact there) and r is rounded to float32 once:
// the value before that rounding is the exact one to about 1e-15, so r, and with it every code, does not depend
// on the order of the sum but for one row in hundreds of millions. The rest are single float32 operations.
// WAVES waves a row, each lane V quads in registers, every load in flight at once; rows of up to 1,024 values take one
// wave and no barrier, four rows a workgroup. The new residual goes past the caches (4096 x 4096 to 8 bits 43.6 us,
// 49.4 through them; 512 x 16384 18.2 and 25.0), the codes, which the next product reads, do not.
template <int V, int WAVES, int FORMAT>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void add_rms_norm_quant(NormArgs a) {
    constexpr int LANES = WAVES * 64;
    const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = WAVES == 1 ? nc::workgroup_id() * 4 + (threadIdx.x >> 6) : nc::workgroup_id();
    if (row >= a.M) return;                            // a whole wave, or a whole workgroup
    const int K = a.K;
    f32x4 t[V], g[V];
    {
        f32x4 d[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = (lane + i * LANES) * 4;
            t[i] = nc::load4(a.x + (size_t)row * K + at, K - at);
            if (a.delta) d[i] = nc::load4(a.delta + (size_t)row * K + at, K - at);
        }
        if (a.delta) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) t[i][j] = __fadd_rn(t[i][j], d[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = (lane + i * LANES) * 4;
        g[i] = nc::load4(a.gamma + at, K - at);
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = (lane + i * LANES) * 4;
        if (a.sum) nc::store4<false>(a.sum + (size_t)row * K + at, t[i], K - at);
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = __builtin_fma((double)t[i][j], (double)t[i][j], ss);
    }
    ss = wave_sum_f64(ss);
    if constexpr (WAVES > 1) {
        __shared__ double part[WAVES];
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) ss += part[w];
    }
    const float r = (float)(1.0 / __builtin_sqrt(ss / (double)K + (double)a.eps));
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = (lane + i * LANES) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) t[i][j] = __fmul_rn(__fmul_rn(t[i][j], r), g[i][j]);
        if (a.normed) nc::store4(a.normed + (size_t)row * K + at, t[i], K - at);
    }
    if constexpr (FORMAT == 0) {
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)                // past K: 0 * r * 0, or NaN with the row's other values
                largest = nc::nan_max(largest, fabsf(t[i][j]));
        largest = nc::wave_max_f32(largest);
        if constexpr (WAVES > 1) {
            __shared__ float most[WAVES];
            if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = largest;
            __syncthreads();
            largest = most[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) largest = nc::nan_max(largest, most[w]);
        }
        const float scale = nc::token_scale(largest);
        if (lane == 0) static_cast<float *>(a.qs)[row] = scale;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = (lane + i * LANES) * 4, valid = K - at;
            int8_t b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = nc::quantize_value(t[i][j], scale);
            uint8_t *out = a.q + (size_t)row * K + at;
            if (valid >= 4) {
                __builtin_memcpy(out, b, 4);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < valid) out[j] = (uint8_t)b[j];
            }
        }
    } else {
        const int quads = (int)(nc::mx_padded(K) / 4);
        uint8_t *codes = a.q + (size_t)row * quads * (FORMAT / 2);
        uint8_t *scales = static_cast<uint8_t *>(a.qs) + (size_t)row * (quads / 8);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = lane + i * LANES;
            if (at >= quads) continue;                 // whole groups of eight
#pragma unroll
            for (int j = 0; j < 4; ++j)                // a NaN row's padding is NaN; the format's is 0
                if (at * 4 + j >= K) t[i][j] = 0.0f;
            const int scale = nc::mx_scale<FORMAT>(block_magnitude<8>(nc::magnitude_bits(t[i])));
            const uint32_t held = nc::mx_encode<FORMAT>(t[i], scale);
            if constexpr (FORMAT == 4) reinterpret_cast<uint16_t *>(codes)[at] = (uint16_t)held;
            else reinterpret_cast<uint32_t *>(codes)[at] = held;
            if (at % 8 == 0) scales[at / 8] = (uint8_t)scale;
        }
    }
}

template <int V, int WAVES>
int32_t launch_norm(const NormArgs &a, int64_t format) {
    const dim3 grid = nc::grid_of(WAVES == 1 ? (a.M + 3) / 4 : a.M), block(WAVES < 4 ? 256 : WAVES * 64);
    if (format == 0)
        hipLaunchKernelGGL((add_rms_norm_quant<V, WAVES, 0>), grid, block, 0, nc::stream(), a);
    else if (format == 8)
        hipLaunchKernelGGL((add_rms_norm_quant<V, WAVES, 8>), grid, block, 0, nc::stream(), a);
    else
        hipLaunchKernelGGL((add_rms_norm_quant<V, WAVES, 4>), grid, block, 0, nc::stream(), a);
    return nc::launched("add_rms_norm_quant");
}

// What the quantizer and its inverse take: shapes whose chunks fit the grid.
bool mx_shape(const int64_t *s) {
    return s[0] >= 0 && s[1] > 0 && s[0] < (1 << 26) && s[1] < (1 << 26) &&
           s[0] * (nc::mx_padded(s[1]) / 4) / kThreads < (int64_t)1 << 31;
}

}  // namespace

// p: [codes u8, scales u8, x f32[M,K]];  s: [M, K, bits]
NC_EXPORT int32_t nc_quantize_mx(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[0] && p[1] && p[2], "nc_quantize_mx: null operand");
    NC_REQUIRE(mx_shape(s), "nc_quantize_mx: bad shape");
    NC_REQUIRE(s[2] == 4 || s[2] == 8, "nc_quantize_mx: elements have 4 or 8 bits");
    NC_REQUIRE(nc::aligned(p[0], 16) && nc::aligned(p[1], 4),
               "nc_quantize_mx: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const int64_t per_row = nc::mx_padded(s[1]) / kQuantized;
    auto *kernel = s[2] == 4 ? &quantize_mx<4> : &quantize_mx<8>;
    hipLaunchKernelGGL(kernel, nc::grid_of((s[0] * per_row + kThreads - 1) / kThreads), dim3(kThreads), 0, nc::stream(),
                       (uint8_t *)p[0], (uint8_t *)p[1], (const float *)p[2], s[0], (int)s[1], (uint32_t)per_row);
    return nc::launched("quantize_mx");
}

// p: [x f32[M,K], codes u8, scales u8];  s: [M, K, bits]
NC_EXPORT int32_t nc_dequantize_mx(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[0] && p[1] && p[2], "nc_dequantize_mx: null operand");
    NC_REQUIRE(mx_shape(s), "nc_dequantize_mx: bad shape");
    NC_REQUIRE(s[2] == 4 || s[2] == 8, "nc_dequantize_mx: elements have 4 or 8 bits");
    NC_REQUIRE(nc::aligned(p[1], 16) && nc::aligned(p[2], 4),
               "nc_dequantize_mx: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const int64_t per_row = nc::mx_padded(s[1]) / kDequantized;
    auto *kernel = s[2] == 4 ? &dequantize_mx<4> : &dequantize_mx<8>;
    hipLaunchKernelGGL(kernel, nc::grid_of((s[0] * per_row + kThreads - 1) / kThreads), dim3(kThreads), 0, nc::stream(),
                       (float *)p[0], (const uint8_t *)p[1], (const uint8_t *)p[2], s[0], (int)s[1], (uint32_t)per_row);
    return nc::launched("dequantize_mx");
}

// p: [sum f32[M,K] | NULL, normed f32[M,K] | NULL, q, qs, x f32[M,K], delta f32[M,K] | NULL, gamma f32[K]];
// s: [M, K, eps as float32 bits, format]
NC_EXPORT int32_t nc_add_rms_norm_quant(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[2] && p[3] && p[4] && p[6], "nc_add_rms_norm_quant: null operand");
    NC_REQUIRE(s[0] >= 0 && s[1] > 0 && s[0] < (1 << 26) && s[1] <= 32768, "nc_add_rms_norm_quant: bad shape");
    NC_REQUIRE(s[3] == 0 || s[3] == 4 || s[3] == 8, "nc_add_rms_norm_quant: the format is 0 (int8), 4 or 8");
    NC_REQUIRE(s[3] == 0 || (nc::aligned(p[2], 16) && nc::aligned(p[3], 4)),
               "nc_add_rms_norm_quant: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const NormArgs a{(float *)p[0], (float *)p[1], (uint8_t *)p[2], p[3], (const float *)p[4], (const float *)p[5],
                     (const float *)p[6], s[0], (int)s[1], nc::bits_to_float(s[2])};
    if (a.K <= 512) return launch_norm<2, 1>(a, s[3]);
    if (a.K <= 1024) return launch_norm<4, 1>(a, s[3]);
    if (a.K <= 2048) return launch_norm<2, 4>(a, s[3]);
    if (a.K <= 4096) return launch_norm<4, 4>(a, s[3]);
    if (a.K <= 8192) return launch_norm<8, 4>(a, s[3]);
    if (a.K <= 16384) return launch_norm<4, 16>(a, s[3]);
    return launch_norm<8, 16>(a, s[3]);
}
