// Projections of microscaled activations by microscaled 4-bit weights (nc_mx.h has the formats):
//
//   y[m, n] = sum over blocks b of 2^(xs[m, b] + ws[n, b] - 254) * sum over k in b of xq[m, k] * q[n, k]
//
// then + bias[n], then residual[m, n] + y; or for a pair of weights silu(gate) * up. Sums in float32.
//
// Activations of 4 bits: one scaled matrix instruction (v_mfma_scale_f32_16x16x128_f8f6f4) takes 16 weight rows and
// 16 rows of x over four blocks, a step of 128 values of k, lane l = 16 g + r the row r of each, block g, and that
// block's scale (measured: off by at most 6.9e-8 of the sum of the products' magnitudes).
// Activations of 8 bits: the same instruction takes them too, but adds the products of 8-bit elements in groups
// of eight that keep 13 bits below the group's largest product (measured: 2^8 + 2^-6 is 2^8, off by up to 2e-4 of the
// magnitudes), which is no 32-bit sum. So both operands are converted to bfloat16, which holds an element
// times its block's power of two exactly (values under 2^-126, whose blocks are subnormal floats, to 2^-133), and a
// step takes four v_mfma_f32_16x16x32_bf16 (off by 2.2e-7 of the magnitudes a step): a quarter of the 4-bit
// rate, 2.5 PFLOP/s. Instruction t takes the values 8 t .. 8 t + 7 of every lane's block: any order of k
// will do that is the same for both operands, and this one leaves a lane with one block, as above.
//
// Either way an instruction returns acc[n = 4 g + r][m = l % 16] with the weights as the first operand: four
// consecutive outputs of a row of y.
#include "nc_epilogue.h"
#include "nc_mx.h"

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
using nc::f32x4;

struct MxArgs {
    float *y;                        // may be the residual
    const uint8_t *xq, *xs;          // [M, steps * 16 * bits], [M, steps * 4]
    const uint8_t *q[2], *ws[2];     // [N, steps * 64], [N, steps * 4]; the second of a pair
    const float *bias, *residual;    // either may be NULL
    int64_t M, N;
    int steps;                       // of 128 values of k
};

// The scale's power of two, 255 as NaN: the conversions and matrix instructions read the exponent only.
__device__ __forceinline__ float power(int scale) { return __int_as_float(scale << 23); }

// A lane's block of 32 values of a step, ready to multiply: 4-bit codes and their scale, or bfloat16 values.
template <int BITS>
struct Block;
template <>
struct Block<4> {
    i32x4 codes;
    int scale;
};
template <>
struct Block<8> {
    bf16x8 part[4];
};

// From 4-bit codes.
template <int BITS>
__device__ __forceinline__ Block<BITS> block_of(i32x4 codes, int scale) {
    if constexpr (BITS == 4) {
        return {codes, scale};
    } else {
        Block<8> b;
        const float p = power(scale);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            bf16x2 v[4];
            v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[t], p, 0);
            v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[t], p, 1);
            v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[t], p, 2);
            v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[t], p, 3);
            b.part[t] = __builtin_bit_cast(bf16x8, v);
        }
        return b;
    }
}

// From 8-bit codes, the block's first 16 and its last.
__device__ __forceinline__ Block<8> block_of(i32x4 lo, i32x4 hi, int scale) {
    Block<8> b;
    const float p = power(scale);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int w0 = t < 2 ? lo[2 * t] : hi[2 * t - 4], w1 = t < 2 ? lo[2 * t + 1] : hi[2 * t - 3];
        bf16x2 v[4];
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, p, false);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, p, true);
        v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, p, false);
        v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, p, true);
        b.part[t] = __builtin_bit_cast(bf16x8, v);
    }
    return b;
}

// c + the products of a step. The compiler does not know that a scaled matrix instruction needs every lane, and may
// move one whose result is used under a lane's condition under that condition: `pin` keeps results outside.
__device__ __forceinline__ f32x4 mx_step(const Block<4> &w, const Block<4> &x, f32x4 c) {
    const i32x8 w8 = __builtin_shufflevector(w.codes, w.codes, 0, 1, 2, 3, -1, -1, -1, -1);
    const i32x8 x8 = __builtin_shufflevector(x.codes, x.codes, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, c, 4, 4, 0, w.scale, 0, x.scale);
}
__device__ __forceinline__ f32x4 mx_step(const Block<8> &w, const Block<8> &x, f32x4 c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.part[t], x.part[t], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ void pin(f32x4 &v) { asm volatile("" : "+v"(v)); }

// A lane's block of x at `p` in memory.
template <int BITS>
__device__ __forceinline__ Block<BITS> load_x(const uint8_t *p, int scale) {
    const i32x4 *q = reinterpret_cast<const i32x4 *>(p);
    if constexpr (BITS == 4) return block_of<4>(q[0], scale);
    else return block_of(q[0], q[1], scale);
}

// Outputs n .. n + 3 of row m from their sums (and for the pair those of the second weight).
template <int NB>
__device__ __forceinline__ void finish(const MxArgs &a, int64_t m, int64_t n, f32x4 g, f32x4 u) {
    if (m >= a.M) return;
    const size_t at = (size_t)m * a.N + n;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (n + r >= a.N) return;
        float v = g[r];
        if constexpr (NB == 2) {
            v = nc::silu_mul(v, u[r]);
        } else {
            if (a.bias) v = __fadd_rn(v, a.bias[n + r]);
            if (a.residual) v = __fadd_rn(a.residual[at + r], v);
        }
        a.y[at + r] = v;
    }
}

constexpr int kWaves = 4;

// A workgroup takes 16 rows of x by 16 weight rows (of each weight), its waves a share of k each; the sums are
// added in the order of the waves. Rows past M or N are the last one, their results not stored.
template <int BITS, int NB>
__global__ __launch_bounds__(kWaves * 64) void mx_few_rows(MxArgs a) {
    const int64_t mtiles = (a.M + 15) / 16, tiles = mtiles * ((a.N + 15) / 16);
    const int64_t tile = nc::workgroup_id();
    if (tile >= tiles) return;
    const int64_t m0 = tile % mtiles * 16, n0 = tile / mtiles * 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, g = lane >> 4;
    const int64_t m = min(m0 + row, a.M - 1), n = min(n0 + row, a.N - 1);
    const uint8_t *xq = a.xq + (size_t)m * a.steps * 16 * BITS + g * 4 * BITS, *xs = a.xs + (size_t)m * a.steps * 4 + g;
    const uint8_t *q[NB], *ws[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        q[b] = a.q[b] + (size_t)n * a.steps * 64 + g * 16;
        ws[b] = a.ws[b] + (size_t)n * a.steps * 4 + g;
    }
    f32x4 acc[NB] = {};
    const int share = (a.steps + kWaves - 1) / kWaves, begin = wave * share, end = min(a.steps, begin + share);
    for (int s = begin; s < end; ++s) {
        const Block<BITS> x = load_x<BITS>(xq + (size_t)s * 16 * BITS, xs[s * 4]);
#pragma unroll
        for (int b = 0; b < NB; ++b)
            acc[b] = mx_step(
                block_of<BITS>(*reinterpret_cast<const i32x4 *>(q[b] + (size_t)s * 64), ws[b][s * 4]), x, acc[b]);
    }
    __shared__ f32x4 part[kWaves][NB][64];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        pin(acc[b]);
        part[wave][b][lane] = acc[b];
    }
    __syncthreads();
    if (wave > 0) return;
    f32x4 sum[2] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum[b] += part[w][b][lane];
    finish<NB>(a, m0 + row, n0 + 4 * g, sum[0], sum[1]);
}

template <int NB>
int32_t launch(const MxArgs &a, int64_t bits) {
    const int64_t tiles = (a.M + 15) / 16 * ((a.N + 15) / 16);
    auto *kernel = bits == 4 ? &mx_few_rows<4, NB> : &mx_few_rows<8, NB>;
    hipLaunchKernelGGL(kernel, nc::grid_of(tiles), dim3(kWaves * 64), 0, nc::stream(), a);
    return nc::launched("mx_few_rows");
}

// Shapes whose outputs are fewer than 2^40 (a terabyte of float32 is 2^38).
bool mx_matmul_shape(const int64_t *s) {
    return s[0] >= 0 && s[1] > 0 && s[2] > 0 && s[0] < (1 << 26) && s[1] < (1 << 26) && s[2] < (1 << 26) &&
           s[0] * s[1] < (int64_t)1 << 40;
}

}  // namespace

// p: [y f32[M,N], xq, xs, q, scales, bias f32[N] | NULL, residual f32[M,N] | NULL];  s: [M, N, K, bits of xq]
NC_EXPORT int32_t nc_matmul_mx(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[0] && p[1] && p[2] && p[3] && p[4], "nc_matmul_mx: null operand");
    NC_REQUIRE(mx_matmul_shape(s), "nc_matmul_mx: bad shape");
    NC_REQUIRE(s[3] == 4 || s[3] == 8, "nc_matmul_mx: activations have 4 or 8 bits");
    NC_REQUIRE(nc::aligned(p[1], 16) && nc::aligned(p[2], 4) && nc::aligned(p[3], 16) && nc::aligned(p[4], 4),
               "nc_matmul_mx: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const MxArgs a{(float *)p[0], (const uint8_t *)p[1], (const uint8_t *)p[2],
                   {(const uint8_t *)p[3], nullptr}, {(const uint8_t *)p[4], nullptr},
                   (const float *)p[5], (const float *)p[6], s[0], s[1], (int)(nc::mx_padded(s[2]) / nc::kMxPad)};
    return launch<1>(a, s[3]);
}

// p: [h f32[M,N], xq, xs, qg, sg, qu, su];  s: [M, N, K, bits of xq]
NC_EXPORT int32_t nc_matmul_mx_swiglu(void **p, const int64_t *s) {
    NC_REQUIRE(p && s && p[0] && p[1] && p[2] && p[3] && p[4] && p[5] && p[6], "nc_matmul_mx_swiglu: null operand");
    NC_REQUIRE(mx_matmul_shape(s), "nc_matmul_mx_swiglu: bad shape");
    NC_REQUIRE(s[3] == 4 || s[3] == 8, "nc_matmul_mx_swiglu: activations have 4 or 8 bits");
    NC_REQUIRE(nc::aligned(p[1], 16) && nc::aligned(p[2], 4) && nc::aligned(p[3], 16) && nc::aligned(p[4], 4) &&
                   nc::aligned(p[5], 16) && nc::aligned(p[6], 4),
               "nc_matmul_mx_swiglu: codes need 16-byte, scales 4-byte alignment");
    if (s[0] == 0) return NC_OK;
    const MxArgs a{(float *)p[0], (const uint8_t *)p[1], (const uint8_t *)p[2],
                   {(const uint8_t *)p[3], (const uint8_t *)p[5]}, {(const uint8_t *)p[4], (const uint8_t *)p[6]},
                   nullptr, nullptr, s[0], s[1], (int)(nc::mx_padded(s[2]) / nc::kMxPad)};
    return launch<2>(a, s[3]);
}
