// The microscaled formats' row kernels (nc_mx.h has the formats): the quantizer, its inverse, and the residual's
// addition with rms_norm and a quantized output.
//
// Everything here reads and writes each value once and is bound by memory. A lane takes 8 consecutive values:
// 32 bytes of float32 and 4 or 8 bytes of codes, so that a block of 32 is a group of four lanes, whose largest
// magnitude two DPP exchanges give.
#include "nc_mx.h"

namespace {

using nc::u32x2;

constexpr int kThreads = 256;

__device__ __forceinline__ int32_t block_magnitude(const float (&v)[8]) {
    return nc::butterfly<4>(nc::magnitude_bits(v), [](int32_t a, int32_t b) { return max(a, b); });
}

template <int BITS>
__device__ __forceinline__ void store_codes(uint8_t *row, int64_t chunk, u32x2 codes) {
    if constexpr (BITS == 4) reinterpret_cast<uint32_t *>(row)[chunk] = codes[0];
    else reinterpret_cast<u32x2 *>(row)[chunk] = codes;
}

// A thread a chunk of 8 values of the padded rows, in order. The row and column of a workgroup's first chunk
// come from one division on the scalar unit; its threads add theirs to the column in 32 bits.
struct Chunk {
    int64_t row;
    uint32_t at;         // in the row
};

__device__ __forceinline__ Chunk chunk_of(int64_t first, uint32_t per_row) {
    const int64_t row = first / per_row;
    const uint32_t at = (uint32_t)(first - row * per_row) + threadIdx.x;
    return {row + at / per_row, at % per_row};
}

template <int BITS>
__global__ __launch_bounds__(kThreads) void quantize_mx(uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                        const float *__restrict__ x, int64_t M, int K,
                                                        uint32_t per_row) {
    const Chunk c = chunk_of(nc::workgroup_id() * kThreads, per_row);
    if (c.row >= M) return;                            // whole groups of four: a row has a multiple of 16 chunks
    float v[8];
    nc::load8(v, x + (size_t)c.row * K + (size_t)c.at * 8, K - (int)c.at * 8);
    const int scale = nc::mx_scale<BITS>(block_magnitude(v));
    store_codes<BITS>(codes + (size_t)c.row * per_row * BITS, c.at, nc::mx_encode<BITS>(v, scale));
    if (c.at % 4 == 0) scales[((size_t)c.row * per_row + c.at) / 4] = (uint8_t)scale;
}

template <int BITS>
__global__ __launch_bounds__(kThreads) void dequantize_mx(float *__restrict__ x, const uint8_t *__restrict__ codes,
                                                          const uint8_t *__restrict__ scales, int64_t M, int K,
                                                          uint32_t per_row) {
    const Chunk c = chunk_of(nc::workgroup_id() * kThreads, per_row);
    if (c.row >= M) return;
    const uint8_t *row = codes + (size_t)c.row * per_row * BITS;
    u32x2 held = {0u, 0u};
    if constexpr (BITS == 4) held[0] = reinterpret_cast<const uint32_t *>(row)[c.at];
    else held = reinterpret_cast<const u32x2 *>(row)[c.at];
    float v[8];
    nc::mx_decode<BITS>(v, held, scales[((size_t)c.row * per_row + c.at) / 4]);
    nc::store8(x + (size_t)c.row * K + (size_t)c.at * 8, v, K - (int)c.at * 8);
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
            const uint32_t a = (uint32_t)nc::xor_partner<OFF>((int32_t)lo), b = (uint32_t)nc::xor_partner<OFF>((int32_t)hi);
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
// WAVES waves a row, each lane V chunks of 8 values in registers, every load in flight at once; rows of up to
// 1,024 values take one wave and no barrier, four rows a workgroup.
template <int V, int WAVES, int FORMAT>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void add_rms_norm_quant(NormArgs a) {
    constexpr int LANES = WAVES * 64;
    const int lane = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = WAVES == 1 ? nc::workgroup_id() * 4 + (threadIdx.x >> 6) : nc::workgroup_id();
    if (row >= a.M) return;                            // a whole wave, or a whole workgroup
    const int K = a.K;
    float t[V][8];
    {
        float d[V][8];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = (lane + i * LANES) * 8;
            nc::load8(t[i], a.x + (size_t)row * K + at, K - at);
            if (a.delta) nc::load8(d[i], a.delta + (size_t)row * K + at, K - at);
        }
        if (a.delta) {
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) t[i][j] = __fadd_rn(t[i][j], d[i][j]);
        }
    }
    float g[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = (lane + i * LANES) * 8;
        nc::load8(g[i], a.gamma + at, K - at);
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = (lane + i * LANES) * 8;
        if (a.sum) nc::store8(a.sum + (size_t)row * K + at, t[i], K - at);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fma((double)t[i][j], (double)t[i][j], ss);
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
        const int at = (lane + i * LANES) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) t[i][j] = __fmul_rn(__fmul_rn(t[i][j], r), g[i][j]);
        if (a.normed) nc::store8(a.normed + (size_t)row * K + at, t[i], K - at);
    }
    if constexpr (FORMAT == 0) {
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j)                // past K: 0 * r * 0, or NaN with the row's other values
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
            const int at = (lane + i * LANES) * 8, valid = K - at;
            int8_t b[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = nc::quantize_value(t[i][j], scale);
            uint8_t *out = a.q + (size_t)row * K + at;
            if (valid >= 8) {
                __builtin_memcpy(out, b, 8);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < valid) out[j] = (uint8_t)b[j];
            }
        }
    } else {
        const int chunks = (int)(nc::mx_padded(K) / 8);
        uint8_t *codes = a.q + (size_t)row * chunks * FORMAT;
        uint8_t *scales = static_cast<uint8_t *>(a.qs) + (size_t)row * (chunks / 4);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = lane + i * LANES;
            if (at >= chunks) continue;                // whole groups of four
#pragma unroll
            for (int j = 0; j < 8; ++j)                // a NaN row's padding is NaN; the format's is 0
                if (at * 8 + j >= K) t[i][j] = 0.0f;
            const int scale = nc::mx_scale<FORMAT>(block_magnitude(t[i]));
            store_codes<FORMAT>(codes, at, nc::mx_encode<FORMAT>(t[i], scale));
            if (at % 4 == 0) scales[at / 4] = (uint8_t)scale;
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
           s[0] * (nc::mx_padded(s[1]) / 8) / kThreads < (int64_t)1 << 31;
}

}  // namespace

// p: [codes u8, scales u8, x f32[M,K]];  s: [M, K, bits]
NC_EXPORT int32_t nc_quantize_mx(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[0] && p[1] && p[2], "nc_quantize_mx: null operand");
    NC_REQUIRE(mx_shape(s), "nc_quantize_mx: bad shape");
    NC_REQUIRE(s[2] == 4 || s[2] == 8, "nc_quantize_mx: elements have 4 or 8 bits");
    NC_REQUIRE(nc::aligned(p[0], 16) && nc::aligned(p[1], 4), "nc_quantize_mx: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const int64_t per_row = nc::mx_padded(s[1]) / 8;
    const dim3 grid = nc::grid_of((s[0] * per_row + kThreads - 1) / kThreads);
    auto *kernel = s[2] == 4 ? &quantize_mx<4> : &quantize_mx<8>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, nc::stream(), (uint8_t *)p[0], (uint8_t *)p[1],
                       (const float *)p[2], s[0], (int)s[1], (uint32_t)per_row);
    return nc::launched("quantize_mx");
}

// p: [x f32[M,K], codes u8, scales u8];  s: [M, K, bits]
NC_EXPORT int32_t nc_dequantize_mx(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[0] && p[1] && p[2], "nc_dequantize_mx: null operand");
    NC_REQUIRE(mx_shape(s), "nc_dequantize_mx: bad shape");
    NC_REQUIRE(s[2] == 4 || s[2] == 8, "nc_dequantize_mx: elements have 4 or 8 bits");
    NC_REQUIRE(nc::aligned(p[1], 16) && nc::aligned(p[2], 4), "nc_dequantize_mx: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const int64_t per_row = nc::mx_padded(s[1]) / 8;
    const dim3 grid = nc::grid_of((s[0] * per_row + kThreads - 1) / kThreads);
    auto *kernel = s[2] == 4 ? &dequantize_mx<4> : &dequantize_mx<8>;
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, nc::stream(), (float *)p[0], (const uint8_t *)p[1],
                       (const uint8_t *)p[2], s[0], (int)s[1], (uint32_t)per_row);
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
    if (a.K <= 512) return launch_norm<1, 1>(a, s[3]);
    if (a.K <= 1024) return launch_norm<2, 1>(a, s[3]);
    if (a.K <= 2048) return launch_norm<1, 4>(a, s[3]);
    if (a.K <= 4096) return launch_norm<2, 4>(a, s[3]);
    if (a.K <= 8192) return launch_norm<4, 4>(a, s[3]);
    if (a.K <= 16384) return launch_norm<2, 16>(a, s[3]);
    return launch_norm<4, 16>(a, s[3]);
}
