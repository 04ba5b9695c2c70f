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
#include "nc_mx.h"
#include "nc_rules.h"

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
using nc::f32x4;
using nc::f32x4_any;
typedef float f32x16 __attribute__((ext_vector_type(16)));

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

// silu(g) * u = g * sigmoid(g) * u with e = exp(-|g|): sigmoid = (g < 0 ? e : 1) / (1 + e). nc::silu_mul takes the
// exponential in double, to the reference's bits; here float32 is enough, and 5 million outputs took 10 us of it.
// exp2's argument t keeps what its product with log2(e) rounds off, so e is good to two units in the last place,
// the result to five; e under 2^-126 counts as 0.
__device__ __forceinline__ float silu_times(float g, float u) {
    const float a = fminf(fabsf(g), 150.0f);           // (past 104 e is 0; an infinite g has sigmoid 0 or 1)
    const float t = __fmul_rn(a, -1.44269502f);        // log2(e) = 1.44269502 + 1.9259e-8
    const float low = fmaf(a, -1.44269502f, -t) - a * 1.92596299e-8f;
    const float e0 = __builtin_amdgcn_exp2f(t), e = fmaf(e0, low * 0.693147182f, e0);
    const float sigmoid = (g < 0.0f ? e : 1.0f) * __builtin_amdgcn_rcpf(1.0f + e);
    return g * sigmoid * u;
}

// Outputs n .. n + 3 of rows m, m + apart, .. (R of them) from their sums, of a pair's from its products: + bias, the
// residual + that, stored. Four at once where the row has them: global memory takes wide loads and stores on any
// boundary of a float.
template <int NB, int R>
__device__ __forceinline__ void finish(const MxArgs &a, int64_t m, int apart, int64_t n, f32x4 (&v)[R]) {
    if (n >= a.N) return;
    const bool whole = n + 4 <= a.N;
    if constexpr (NB == 1) {
        f32x4 bias = {}, residual[R];
        if (a.bias) {
            if (whole) {
                bias = *reinterpret_cast<const f32x4_any *>(a.bias + n);
            } else {
                for (int c = 0; c < 3; ++c)
                    if (n + c < a.N) bias[c] = a.bias[n + c];
            }
        }
        if (a.residual) {
#pragma unroll
            for (int r = 0; r < R; ++r)                // every load before the first sum
                if (whole && m + r * apart < a.M)
                    residual[r] = *reinterpret_cast<const f32x4_any *>(a.residual + (size_t)(m + r * apart) * a.N + n);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (a.bias) v[r] += bias;
            if (a.residual && whole) v[r] = residual[r] + v[r];
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (m + r * apart >= a.M) return;
        const size_t at = (size_t)(m + r * apart) * a.N + n;
        if (whole) {
            *reinterpret_cast<f32x4_any *>(a.y + at) = v[r];
            continue;
        }
#pragma unroll
        for (int c = 0; c < 3; ++c)
            if (n + c < a.N) a.y[at + c] = NB == 1 && a.residual ? __fadd_rn(a.residual[at + c], v[r][c]) : v[r][c];
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

// Staging of 16 rows by a step in LDS, ROW bytes a row (64 for 4-bit codes, 128 for 8-bit ones). A lane's block lies a
// row from its neighbours' in memory: read as it is multiplied, 16 lanes that go through the cache together would
// touch 16 lines (measured: 8 x 8192 x 8192 13.5 us so, 8.3 through LDS). So lanes copy whole row segments, and the
// 16-byte chunks of row r, a block's or its two halves 4 apart, are permuted by exclusive or with
// (r / DIV) mod the chunks a row. With DIV 2 the reads of 16 rows by 4 blocks meet no bank conflict, with 128-byte
// rows also those of 32 rows by 2; 64-byte rows need DIV 4 there (4.4 cycles a read of 1 KB, 8.1 with others).
template <int ROW, int DIV>
struct Stage {
    static constexpr int kChunks = ROW / 16, kCopies = ROW / 64;     // copies of 1 KB
    static __device__ __forceinline__ int swizzle(int row) { return row / DIV % kChunks; }
    // The row that a lane copies in copy `copy` of consecutive 16 rows' kCopies, and the byte in it.
    static __device__ __forceinline__ int row(int lane, int copy) {
        return copy / kCopies * 16 + copy % kCopies * (16 / kCopies) + lane / kChunks;
    }
    static __device__ __forceinline__ int column(int lane, int copy) {
        const int slot = lane % kChunks ^ swizzle(row(lane, copy));
        return (ROW == 64 ? slot : slot % 4 * 2 + slot / 4) * 16;
    }
    // Where half h (0 in 4 bits) of block b of row r lies, counted from the first of these rows.
    static __device__ __forceinline__ int at(int r, int b, int h) { return r * ROW + ((b + 4 * h) ^ swizzle(r)) * 16; }
};

// Few outputs: a workgroup takes 16 MF rows of x by 16 NF weight rows (of each weight), its waves a share of k each,
// every wave through LDS of its own, U steps' copies in flight at once; the sums are added in the order of the waves.
// Rows past M or N are the last one, their results not stored.
template <int BITS, int NB, int MF, int NF, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void mx_split(MxArgs a) {
    using W = Stage<64, 2>;
    using X = Stage<16 * BITS, 2>;
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
            xat[i][h] = x_row(X::row(lane, i * X::kCopies + h)) * (16 * BITS) + X::column(lane, h);
        xsat[i] = x_row(16 * i + row) * 4;
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) {
        wat[j] = w_row(W::row(lane, j)) * 64 + W::column(lane, j);
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
                                                                X::at(row, g, h));
                x[i] = x_block<BITS>(codes, xe[i][c] >> (8 * g) & 255);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int j = 0; j < NF; ++j) {
                    const Block<BITS> w = block_of<BITS>(
                        *reinterpret_cast<const i32x4 *>(at + (b * NF + j) * 1024 + W::at(row, g, 0)),
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
        f32x4 v[1] = {sum[0]};
        if constexpr (NB == 2) {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[0][c] = silu_times(sum[0][c], sum[1][c]);
        }
        finish<NB, 1>(a, m0 + f / NF * 16 + row, 0, n0 + f % NF * 16 + 4 * g, v);
    }
}

template <int BITS, int NB, int MF, int NF, int WAVES, int U>
int32_t launch_split(const MxArgs &a) {
    const int64_t tiles = (a.M + 16 * MF - 1) / (16 * MF) * ((a.N + 16 * NF - 1) / (16 * NF));
    hipLaunchKernelGGL((mx_split<BITS, NB, MF, NF, WAVES, U>), nc::grid_of(tiles), dim3(WAVES * 64), 0, nc::stream(), a);
    return nc::launched("mx_split");
}

// c + the products of 64 values of k of 32 weight rows by 32 rows of x, lane l the row l % 32 of each and a block; the
// outputs are acc[n = 8 (r / 4) + 4 (l / 32) + r % 4][m = l % 32].
template <int OP>
__device__ __forceinline__ f32x16 mx_half_step(const Block<4> &w, const Block<4> &x, f32x16 c) {
    const i32x8 w8 = __builtin_shufflevector(w.codes, w.codes, 0, 1, 2, 3, -1, -1, -1, -1);
    const i32x8 x8 = __builtin_shufflevector(x.codes, x.codes, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w8, x8, c, 4, 4, OP, w.scale, OP, x.scale);
}
template <int OP>
__device__ __forceinline__ f32x16 mx_half_step(const Block<8> &w, const Block<8> &x, f32x16 c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w.part[t], x.part[t], c, 0, 0, 0);
    return c;
}

// copy_to_lds for copies that stay in flight past LDS reads: before any read of LDS the compiler waits for every copy it
// knows of, as each might write what is read. Which copies a read needs is counted in mx_tile, so these are hidden
// from it. They write no register; `to` goes through m0, which takes a wait state.
__device__ __forceinline__ void copy_to_lds_counted(const uint8_t *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "m0", "memory");
}

// Many outputs: a workgroup of WM x WN waves takes 32 MF WM rows of x by 32 NF WN weight rows (of each weight), staged in
// a ring of four steps in LDS, each wave 32 MF x 32 NF of them from registers, half a step at a time: while one half
// is multiplied the next is read, and the copies of two steps more are in flight. A wave waits until only the copies
// issued after the next step's are left, and at the barrier for the other waves'. The scales come four steps at a
// time, 16 bytes a row. The outputs go through LDS, a wave's 32 rows at a time, so that whole lines are written (a lane's own
// outputs are 16 bytes of a row: 4096 x 8192 x 8192 took 255 us so, 140 of them without the stores). Needs four steps.
template <int BITS, int NB, int WM, int WN, int MF, int NF>
__global__ __launch_bounds__(WM * WN * 64) void mx_tile(MxArgs a) {
    using W = Stage<64, 4>;
    using X = Stage<16 * BITS, BITS == 4 ? 4 : 2>;
    constexpr int WAVES = WM * WN, BM = 32 * MF * WM, BN = 32 * NF * WN, XH = BITS / 4;
    constexpr int XC = BM / 16 * X::kCopies, WC = BN / 16, SC = (BM + NB * BN) / 64;   // copies a stage, a group
    constexpr int BUFFER = (XC + NB * WC) * 1024;
    constexpr int kCopies = (XC + NB * WC) / WAVES, kScaleCopies = (SC + WAVES - 1) / WAVES;      // a wave's
    constexpr int kOutRow = 32 * NF * 4 + 16;                       // bytes of LDS, and of it a wave has 32 rows
    static_assert(XC % WAVES == 0 && WC % WAVES == 0 && BM % 64 == 0 && BN % 64 == 0, "whole copies a wave");
    static_assert(WAVES * 32 * kOutRow <= 4 * BUFFER + 2 * SC * 1024, "the outputs' way through LDS");
    __shared__ __align__(1024) uint8_t lds[4 * BUFFER + 2 * SC * 1024];
    uint8_t *const scales = lds + 4 * BUFFER;

    const int64_t mtiles = (a.M + BM - 1) / BM, tiles = mtiles * ((a.N + BN - 1) / BN);
    if (nc::workgroup_id() >= tiles) return;
    const int64_t tile = tile_of(nc::workgroup_id(), tiles);
    const int64_t m0 = tile % mtiles * BM, n0 = tile / mtiles * BN;
    const int lane = threadIdx.x & 63, row = lane & 31, g = lane >> 5, steps = a.steps;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN * (32 * MF), wn = wave % WN * (32 * NF);      // this wave's first row of each
    auto x_row = [&](int r) { return (uint32_t)min((int64_t)r, a.M - 1 - m0) * (uint32_t)steps; };
    auto w_row = [&](int r) { return (uint32_t)min((int64_t)r, a.N - 1 - n0) * (uint32_t)steps; };
    const uint8_t *xq = a.xq + (size_t)m0 * steps * (16 * BITS), *xs = a.xs + (size_t)m0 * steps * 4;
    const uint8_t *q[NB], *ws[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        q[b] = a.q[b] + (size_t)n0 * steps * 64;
        ws[b] = a.ws[b] + (size_t)n0 * steps * 4;
    }
    // This lane's part of the wave's copies: copies i * WAVES + wave of a stage, and of a group of scales.
    uint32_t xat[XC / WAVES], wat[WC / WAVES];
    const uint8_t *sat[kScaleCopies];
#pragma unroll
    for (int i = 0; i < XC / WAVES; ++i)
        xat[i] = x_row(X::row(lane, i * WAVES + wave)) * (16 * BITS) + X::column(lane, i * WAVES + wave);
#pragma unroll
    for (int i = 0; i < WC / WAVES; ++i)
        wat[i] = w_row(W::row(lane, i * WAVES + wave)) * 64 + W::column(lane, i * WAVES + wave);
#pragma unroll
    for (int i = 0; i < kScaleCopies; ++i) {
        // (where the copies are fewer than the waves, several waves make the last one)
        const int r = min(i * WAVES + wave, SC - 1) * 64 + lane;
        sat[i] = r < BM        ? xs + x_row(r) * 4
                 : r < BM + BN ? ws[0] + w_row(r - BM) * 4
                               : ws[NB - 1] + w_row(r - BM - BN) * 4;
    }
    const uint32_t base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t *)lds;
    // Steps past the last are copied as the last, to keep the count of copies in flight; they are not multiplied.
    auto copy_stage = [&](int s, int buffer) {
        const uint32_t to = base + buffer * BUFFER + wave * 1024;
        if (buffer == 0) {                                          // s % 4 == 0
            const int first = min(s, steps - 4);                    // 16 bytes of every row are inside it
#pragma unroll
            for (int i = 0; i < kScaleCopies; ++i)
                copy_to_lds_counted(sat[i] + first * 4, base + 4 * BUFFER + (s / 4 % 2 * SC + min(i * WAVES + wave, SC - 1)) * 1024);
        }
        s = min(s, steps - 1);
#pragma unroll
        for (int i = 0; i < XC / WAVES; ++i)
            copy_to_lds_counted(xq + (size_t)s * (16 * BITS) + xat[i], to + i * WAVES * 1024);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < WC / WAVES; ++i)
                copy_to_lds_counted(q[b] + (size_t)s * 64 + wat[i], to + (XC + b * WC + i * WAVES) * 1024);
    };
    // Half a step's operands: a lane's block g + 2 half of every row it multiplies.
    struct Half {
        i32x4 x[MF][XH], w[NB][NF];
    };
    // Every row's four scales of a step, this lane's first block's lowest.
    struct Scales {
        uint32_t x[MF], w[NB][NF];
    };
    auto read_half = [&](Half &f, int buffer, int half) {
        const uint8_t *from = lds + buffer * BUFFER;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                f.w[b][j] = *reinterpret_cast<const i32x4 *>(from + (XC + b * WC) * 1024 + 32 * j * 64 +
                                                             W::at(wn + row, g + 2 * half, 0));
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int h = 0; h < XH; ++h)
                f.x[i][h] = *reinterpret_cast<const i32x4 *>(from + 32 * i * (16 * BITS) + X::at(wm + row, g + 2 * half, h));
    };
    auto read_scales = [&](Scales &e, int s) {
        s = min(s, steps - 1);
        const uint8_t *from = scales + s / 4 % 2 * (SC * 1024) + (s - min(s & ~3, steps - 4)) * 4;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                e.w[b][j] = *reinterpret_cast<const uint32_t *>(from + (BM + b * BN + wn + 32 * j + row) * 16);
#pragma unroll
        for (int i = 0; i < MF; ++i) e.x[i] = *reinterpret_cast<const uint32_t *>(from + (wm + 32 * i + row) * 16);
    };
    f32x16 acc[NB][MF][NF] = {};
    auto multiply = [&](const Half &f, const Scales &e, auto half) {
        constexpr int T = decltype(half)::value;
        // a matrix instruction picks the scale's byte itself; a conversion needs it alone
        auto scale = [&](uint32_t e) { return BITS == 4 ? (int)(e >> (8 * g)) : (int)(e >> (8 * g + 16 * T) & 255); };
        Block<BITS> x[MF];
#pragma unroll
        for (int i = 0; i < MF; ++i) x[i] = x_block<BITS>(f.x[i], scale(e.x[i]));
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NF; ++j) {
                const Block<BITS> w = block_of<BITS>(f.w[b][j], scale(e.w[b][j]));
#pragma unroll
                for (int i = 0; i < MF; ++i) acc[b][i][j] = mx_half_step<2 * T>(w, x[i], acc[b][i][j]);
            }
    };
    constexpr std::integral_constant<int, 0> first_half{};
    constexpr std::integral_constant<int, 1> second_half{};
    Half f0, f1;
    Scales e0, e1;
    // Step s, whose first half f0 and scales e hold; leaves the next step's there and in `next`.
    auto step = [&](int s, auto which, Scales &e, Scales &next) {
        constexpr int U = decltype(which)::value;                   // s % 4, the step's buffer
        // the copies that may stay in flight: those of step s + 2
        constexpr int later = kCopies + (U == 2 ? kScaleCopies : 0);
        read_half(f1, U, 1);
        multiply(f0, e, first_half);
        __builtin_amdgcn_sched_barrier(0);                          // (products may not sink past the waits)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(later) : "memory");
        __builtin_amdgcn_s_barrier();                               // every wave's part has landed, and step s is read
        asm volatile("" ::: "memory");
        read_half(f0, (U + 1) % 4, 0);
        read_scales(next, s + 1);
        copy_stage(s + 3, (U + 3) % 4);
        multiply(f1, e, second_half);
        __builtin_amdgcn_sched_barrier(0);
    };
    copy_stage(0, 0);
    copy_stage(1, 1);
    copy_stage(2, 2);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kCopies) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read_half(f0, 0, 0);
    read_scales(e0, 0);
    for (int s = 0; s < steps; s += 4) {
        step(s, std::integral_constant<int, 0>{}, e0, e1);
        if (s + 1 < steps) step(s + 1, std::integral_constant<int, 1>{}, e1, e0);
        if (s + 2 < steps) step(s + 2, std::integral_constant<int, 2>{}, e0, e1);
        if (s + 3 < steps) step(s + 3, std::integral_constant<int, 3>{}, e1, e0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) asm volatile("" : "+v"(acc[b][i][j]));
    __syncthreads();                                   // the last copies have landed and the last reads are done
    uint8_t *const mine = lds + wave * (32 * kOutRow);
    constexpr int kAcross = 8 * NF, kRows = 64 / kAcross;           // lanes a row of 32 NF outputs, rows at a time
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                f32x4 v;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    v[c] = NB == 1 ? acc[0][i][j][4 * r + c]
                                   : silu_times(acc[0][i][j][4 * r + c], acc[NB - 1][i][j][4 * r + c]);
                *reinterpret_cast<f32x4 *>(mine + row * kOutRow + (32 * j + 8 * r + 4 * g) * 4) = v;
            }
        asm volatile("" ::: "memory");                 // (a wave's LDS accesses are in order)
        const int64_t n = n0 + wn + lane % kAcross * 4;
        f32x4 v[32 / kRows];
#pragma unroll
        for (int k = 0; k < 32 / kRows; ++k)
            v[k] = *reinterpret_cast<const f32x4 *>(mine + (k * kRows + lane / kAcross) * kOutRow + lane % kAcross * 16);
        asm volatile("" ::: "memory");
        finish<NB, 32 / kRows>(a, m0 + wm + 32 * i + lane / kAcross, kRows, n, v);
    }
}

template <int BITS, int NB, int WM, int WN, int MF, int NF>
int32_t launch_tile(const MxArgs &a) {
    constexpr int BM = 32 * MF * WM, BN = 32 * NF * WN;
    const int64_t tiles = (a.M + BM - 1) / BM * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL((mx_tile<BITS, NB, WM, WN, MF, NF>), nc::grid_of(tiles), dim3(WM * WN * 64), 0, nc::stream(), a);
    return nc::launched("mx_tile");
}

template <int BITS, int NB>
int32_t launch(const MxArgs &a) {
    const nc::MxTile tile = nc::mx_tile(a.M, a.N, a.steps, BITS, NB);
    switch (tile) {
        case nc::MxTile::kRow: return launch_split<BITS, NB, 1, 1, 4, 2>(a);
        case nc::MxTile::kLongRow: return launch_split<BITS, NB, 1, 1, 8, 2>(a);
        case nc::MxTile::kSplit: return launch_split<BITS, NB, 2, 2, 4, NB == 1 ? 2 : 1>(a);
        case nc::MxTile::kSmall: return launch_tile<BITS, NB, 2, 2, 1, 1>(a);
        default:
            if constexpr (BITS == 4) return launch_tile<BITS, NB, 2, 4, 4, NB == 1 ? 2 : 1>(a);
            else if constexpr (NB == 1) return launch_tile<BITS, NB, 2, 4, 2, 2>(a);
            else return launch_tile<BITS, NB, 2, 2, 2, 1>(a);
    }
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
