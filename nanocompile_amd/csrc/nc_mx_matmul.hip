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
using nc::f32x4_any;

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

template <int BITS>
__device__ __forceinline__ Block<BITS> x_block(const i32x4 (&codes)[BITS / 4], int scale) {
    if constexpr (BITS == 4) return block_of<4>(codes[0], scale);
    else return block_of(codes[0], codes[1], scale);
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

// Outputs n .. n + 3 of row m from their sums (and for the pair those of the second weight). Four at once where
// the row has them: global memory takes wide loads and stores on any boundary of a float.
template <int NB>
__device__ __forceinline__ void finish(const MxArgs &a, int64_t m, int64_t n, f32x4 v, f32x4 u) {
    if (m >= a.M || n >= a.N) return;
    const size_t at = (size_t)m * a.N + n;
    if constexpr (NB == 2) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = nc::silu_mul(v[r], u[r]);
    }
    if (n + 4 <= a.N) {
        if constexpr (NB == 1) {
            const f32x4 bias = a.bias ? *reinterpret_cast<const f32x4_any *>(a.bias + n) : f32x4{};
            const f32x4 residual = a.residual ? *reinterpret_cast<const f32x4_any *>(a.residual + at) : f32x4{};
            if (a.bias) v += bias;
            if (a.residual) v = residual + v;
        }
        *reinterpret_cast<f32x4_any *>(a.y + at) = v;
        return;
    }
#pragma unroll
    for (int r = 0; r < 3; ++r) {
        if (n + r >= a.N) return;
        float w = v[r];
        if constexpr (NB == 1) {
            if (a.bias) w = __fadd_rn(w, a.bias[n + r]);
            if (a.residual) w = __fadd_rn(a.residual[at + r], w);
        }
        a.y[at + r] = w;
    }
}

// Workgroup id to tile: the 8 XCDs (workgroup i runs on XCD i % 8) take a contiguous range of tiles each, so that
// the tiles of a band of weight rows, which follow one another, share an L2.
__device__ __forceinline__ int64_t tile_of(int64_t id, int64_t total) {
    return id < (total & ~(int64_t)7) ? (id & 7) * (total >> 3) + (id >> 3) : id;
}

// 16 bytes a lane from memory straight to LDS, at `to` + 16 * lane (`to` the same for every lane).
__device__ __forceinline__ void copy_to_lds(const uint8_t *from, uint8_t *to) {
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void *)from,
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// Staging of 16 rows by a step in LDS, ROW bytes a row. A lane's block lies 16 rows from its neighbours' in memory: read
// as it is multiplied, 16 lanes that go through the cache together would touch 16 lines. So lanes copy whole row
// segments, ROW / 16 of them a row, and the 16-byte chunks of row r are permuted by (r / 2) mod that number, which
// keeps the reads of 16 rows at one chunk free of bank conflicts.
template <int ROW>
struct Stage {
    static constexpr int kChunks = ROW / 16, kCopies = ROW / 64;     // copies of 1 KB
    // The row, and byte in it, that a lane copies (the copy's rows before it not counted).
    static __device__ __forceinline__ int row(int lane) { return lane / kChunks; }
    static __device__ __forceinline__ int column(int lane, int copy) {
        return (lane % kChunks ^ swizzle(copy * (16 / kCopies) + row(lane))) * 16;
    }
    static __device__ __forceinline__ int swizzle(int row) { return row / 2 % kChunks; }
    // Where chunk c of row r lies.
    static __device__ __forceinline__ int at(int r, int c) { return r * ROW + (c ^ swizzle(r)) * 16; }
};

// Few outputs: a workgroup takes 16 MF rows of x by 16 NF weight rows (of each weight), its waves a share of k each,
// every wave through LDS of its own, U steps' copies in flight at once; the sums are added in the order of the waves.
// Rows past M or N are the last one, their results not stored.
template <int BITS, int NB, int MF, int NF, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void mx_split(MxArgs a) {
    using W = Stage<64>;
    using X = Stage<16 * BITS>;
    constexpr int kStep = 1024 * (NB * NF + MF * X::kCopies), kParts = WAVES * NB * MF * NF * 1024;
    __shared__ __align__(1024) uint8_t lds[WAVES * U * kStep > kParts ? WAVES * U * kStep : kParts];

    const int64_t mtiles = (a.M + 16 * MF - 1) / (16 * MF), tiles = mtiles * ((a.N + 16 * NF - 1) / (16 * NF));
    if (nc::workgroup_id() >= tiles) return;
    const int64_t tile = tile_of(nc::workgroup_id(), tiles);
    const int64_t m0 = tile % mtiles * (16 * MF), n0 = tile / mtiles * (16 * NF);
    const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), steps = a.steps;
    // The tile's first rows and a step's place in them are the same for every lane (scalar registers); a lane's
    // row and chunk are an offset of 32 bits.
    auto x_row = [&](int r) { return (uint32_t)min((int64_t)r, a.M - 1 - m0) * (uint32_t)steps; };
    auto w_row = [&](int r) { return (uint32_t)min((int64_t)r, a.N - 1 - n0) * (uint32_t)steps; };
    const uint8_t *xq = a.xq + (size_t)m0 * steps * (16 * BITS), *xs = a.xs + (size_t)m0 * steps * 4;
    const uint8_t *q[NB], *ws[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        q[b] = a.q[b] + (size_t)n0 * steps * 64;
        ws[b] = a.ws[b] + (size_t)n0 * steps * 4;
    }
    uint32_t xat[MF][X::kCopies], xsat[MF], wat[NF], wsat[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
        for (int h = 0; h < X::kCopies; ++h)
            xat[i][h] = x_row(16 * i + h * (16 / X::kCopies) + X::row(lane)) * (16 * BITS) + X::column(lane, h);
        xsat[i] = x_row(16 * i + row) * 4;
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) {
        wat[j] = w_row(16 * j + W::row(lane)) * 64 + W::column(lane, 0);
        wsat[j] = w_row(16 * j + row) * 4;
    }
    f32x4 acc[NB][MF][NF] = {};
    uint8_t *mine = lds + wave * U * kStep;
    auto batch = [&](int s, auto count) {
        constexpr int C = decltype(count)::value;
        typedef uint32_t words __attribute__((ext_vector_type(C == 1 ? 2 : C), aligned(4)));
        words xe[MF], we[NB][NF];
        auto load_words = [&](const uint8_t *p) {
            if constexpr (C == 1) return words{*reinterpret_cast<const uint32_t *>(p), 0u};
            else return *reinterpret_cast<const words *>(p);
        };
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NF; ++j) we[b][j] = load_words(ws[b] + (size_t)s * 4 + wsat[j]);
#pragma unroll
        for (int i = 0; i < MF; ++i) xe[i] = load_words(xs + (size_t)s * 4 + xsat[i]);
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < NF; ++j)
                    copy_to_lds(q[b] + (size_t)(s + c) * 64 + wat[j], mine + c * kStep + (b * NF + j) * 1024);
#pragma unroll
            for (int i = 0; i < MF; ++i)
#pragma unroll
                for (int h = 0; h < X::kCopies; ++h)
                    copy_to_lds(xq + (size_t)(s + c) * (16 * BITS) + xat[i][h],
                                mine + c * kStep + (NB * NF + i * X::kCopies + h) * 1024);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint8_t *at = mine + c * kStep;
            Block<BITS> x[MF];
#pragma unroll
            for (int i = 0; i < MF; ++i) {
                i32x4 codes[BITS / 4];
#pragma unroll
                for (int h = 0; h < BITS / 4; ++h)
                    codes[h] = *reinterpret_cast<const i32x4 *>(at + (NB * NF + i * X::kCopies) * 1024 +
                                                                X::at(row, g * (BITS / 4) + h));
                x[i] = x_block<BITS>(codes, xe[i][c] >> (8 * g) & 255);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < NF; ++j) {
                    const Block<BITS> w = block_of<BITS>(
                        *reinterpret_cast<const i32x4 *>(at + (b * NF + j) * 1024 + W::at(row, g)),
                        we[b][j][c] >> (8 * g) & 255);
#pragma unroll
                    for (int i = 0; i < MF; ++i) acc[b][i][j] = mx_step(w, x[i], acc[b][i][j]);
                }
        }
    };
    const int share = (steps + WAVES - 1) / WAVES, end = min(steps, (wave + 1) * share);
    int s = wave * share;
    for (; s + U <= end; s += U) batch(s, std::integral_constant<int, U>{});
    if constexpr (U > 2) {
        if (s + 2 <= end) batch(s, std::integral_constant<int, 2>{}), s += 2;
    }
    if constexpr (U > 1) {
        if (s < end) batch(s, std::integral_constant<int, 1>{});
    }
    __syncthreads();                                   // every wave is done with its stage
    f32x4 *part = reinterpret_cast<f32x4 *>(lds);      // [WAVES][NB][MF * NF][64]
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                pin(acc[b][i][j]);
                part[((wave * NB + b) * MF * NF + i * NF + j) * 64 + lane] = acc[b][i][j];
            }
    __syncthreads();
    for (int f = wave; f < MF * NF; f += WAVES) {
        f32x4 sum[2] = {};
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) sum[b] += part[((w * NB + b) * MF * NF + f) * 64 + lane];
        finish<NB>(a, m0 + f / NF * 16 + row, n0 + f % NF * 16 + 4 * g, sum[0], sum[1]);
    }
}

template <int BITS, int NB, int MF, int NF, int WAVES, int U>
int32_t launch_split(const MxArgs &a) {
    const int64_t tiles = (a.M + 16 * MF - 1) / (16 * MF) * ((a.N + 16 * NF - 1) / (16 * NF));
    hipLaunchKernelGGL((mx_split<BITS, NB, MF, NF, WAVES, U>), nc::grid_of(tiles), dim3(WAVES * 64), 0, nc::stream(), a);
    return nc::launched("mx_split");
}

template <int BITS, int NB>
int32_t launch(const MxArgs &a) {
    if (a.M > 16) return launch_split<BITS, NB, 2, 2, 4, 2>(a);
    return a.steps >= 16 ? launch_split<BITS, NB, 1, 1, 8, 2>(a) : launch_split<BITS, NB, 1, 1, 4, 2>(a);
}

// Shapes whose outputs are fewer than 2^40 (a terabyte of float32 is 2^38) and whose rows a tile addresses in 32 bits.
bool mx_matmul_shape(const int64_t *s) {
    return s[0] >= 0 && s[1] > 0 && s[2] > 0 && s[0] < (1 << 26) && s[1] < (1 << 26) && s[2] <= (1 << 24) &&
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
    return s[3] == 4 ? launch<4, 1>(a) : launch<8, 1>(a);
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
    return s[3] == 4 ? launch<4, 2>(a) : launch<8, 2>(a);
}
