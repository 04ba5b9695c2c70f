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
// That of byte `at` / 8 of four: the conversions ignore the bits about it (checked for every scale and element).
__device__ __forceinline__ float power_at(uint32_t scales, int at) {
    return __uint_as_float(__builtin_amdgcn_alignbit(scales, scales, at + 9));
}

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

// Eight values to bfloat16: 4-bit codes in a word, 8-bit ones in two.
__device__ __forceinline__ bf16x8 to_bf16(int codes, float power) {
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 0),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 2),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, 3)};
    return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ bf16x8 to_bf16(int low, int high, float power) {
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, power, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, power, true),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, power, false),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, power, true)};
    return __builtin_bit_cast(bf16x8, v);
}

// From 4-bit codes.
template <int BITS>
__device__ __forceinline__ Block<BITS> block_of(i32x4 codes, int scale) {
    if constexpr (BITS == 4) {
        return {codes, scale};
    } else {
        const float p = power(scale);
        return {{to_bf16(codes[0], p), to_bf16(codes[1], p), to_bf16(codes[2], p), to_bf16(codes[3], p)}};
    }
}

// From 8-bit codes, the block's first 16 and its last.
__device__ __forceinline__ Block<8> block_of(i32x4 low, i32x4 high, int scale) {
    const float p = power(scale);
    return {{to_bf16(low[0], low[1], p), to_bf16(low[2], low[3], p), to_bf16(high[0], high[1], p),
             to_bf16(high[2], high[3], p)}};
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

// silu(g) * u = g / (1 + exp(-g)) * u. nc::silu_mul takes the exponential in double, to the reference's bits; here
// float32 is enough, and 5 million outputs took 10 us of it. exp2's argument t keeps what its product with log2(e)
// rounds off, so the exponential is good to three units in the last place, the result to six; a sigmoid under 2^-126
// counts as 0.
__device__ __forceinline__ float silu_times(float g, float u) {
    const float a = __builtin_amdgcn_fmed3f(g, -150.0f, 150.0f);       // (past 104 either way it is 0 or 1)
    const float t = __fmul_rn(a, -1.44269502f);        // log2(e) = 1.44269502 + 1.9259e-8
    const float low = fmaf(a, -1.92596299e-8f, fmaf(a, -1.44269502f, -t));
    const float e = __fmul_rn(__builtin_amdgcn_exp2f(t), fmaf(low, 0.693147182f, 1.0f));
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
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

// Workgroup id to tile: the 8 XCDs (workgroup i runs on XCD i % 8) take a contiguous range of tiles each, in an order
// whose neighbours share operands in that XCD's L2: 8 tiles down the rows of x, then the next weight rows.
struct Tile {
    int64_t m, n;
};
__device__ __forceinline__ Tile tile_of(uint32_t id, uint32_t mtiles, uint32_t ntiles) {
    const uint32_t total = mtiles * ntiles;
    if (id < (total & ~7u)) id = (id & 7) * (total >> 3) + (id >> 3);
    const uint32_t band = id / (8 * ntiles), down = min(8u, mtiles - band * 8), in = id - band * 8 * ntiles;
    return {band * 8 + in % down, in / down};
}

// 16 bytes a lane from memory straight to LDS, at `to` + 16 * lane (`to` the same for every lane).
__device__ __forceinline__ void copy_to_lds(const uint8_t *from, uint8_t *to) {
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) const void *)from,
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// Staging of 16 rows by a step in LDS, ROW bytes a row (64 for 4-bit codes, 128 for 8-bit ones). A lane's block lies a
// row from its neighbours' in memory: read as it is multiplied, 16 lanes that go through the cache together would
// touch 16 lines (8 x 8192 x 8192 in 8 bits 13.5 us so, 10.0 through LDS). So lanes copy whole row segments, and the
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
    static __device__ __forceinline__ int slot(int lane, int copy) { return lane % kChunks ^ swizzle(row(lane, copy)); }
    static __device__ __forceinline__ int column(int lane, int copy) {
        const int s = slot(lane, copy);
        return (ROW == 64 ? s : s % 4 * 2 + s / 4) * 16;
    }
    // Where half h (0 in 4 bits) of block b of row r lies, counted from the first of these rows.
    static __device__ __forceinline__ int at(int r, int b, int h) { return r * ROW + ((b + 4 * h) ^ swizzle(r)) * 16; }
};

// Few outputs: a workgroup takes 16 MF rows of x by 16 NF weight rows (of each weight), its waves a share of k each,
// every wave through LDS of its own, U steps' copies in flight at once; the sums are added in the order of the waves.
// Rows past M or N are the last one, their results not stored. Bound by memory, and by the copies in flight: 8 x 8192 x
// 8192 in 8 bits 8.4 us (4.3 TB/s) of 16 x 32 outputs by eight waves, 9.6 of 16 x 16 by four; 1 x 4864 x 896 2.9, of
// which an empty launch takes 2.4.
template <int BITS, int NB, int MF, int NF, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void mx_split(MxArgs a) {
    using W = Stage<64, 2>;
    using X = Stage<16 * BITS, 2>;
    constexpr int kStep = 1024 * (NB * NF + MF * X::kCopies), kParts = WAVES * NB * MF * NF * 1024;
    __shared__ __align__(1024) uint8_t lds[WAVES * U * kStep > kParts ? WAVES * U * kStep : kParts];

    constexpr int BM = 16 * MF, BN = 16 * NF;
    const uint32_t mtiles = ((uint32_t)a.M + BM - 1) / BM, ntiles = ((uint32_t)a.N + BN - 1) / BN;
    if (nc::workgroup_id() >= mtiles * ntiles) return;
    const Tile tile = tile_of((uint32_t)nc::workgroup_id(), mtiles, ntiles);
    const int64_t m0 = tile.m * BM, n0 = tile.n * BN;
    const int lane = threadIdx.x & 63, row = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), steps = a.steps;
    // The tile's first rows and a step's place in them are the same for every lane (scalar registers); a lane's
    // row and chunk are an offset of 32 bits.
    const int x_last = (int)min(a.M - 1 - m0, (int64_t)BM - 1), w_last = (int)min(a.N - 1 - n0, (int64_t)BN - 1);
    auto x_row = [&](int r) { return (uint32_t)(min(r, x_last) * steps); };
    auto w_row = [&](int r) { return (uint32_t)(min(r, w_last) * steps); };
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
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the steps before are read
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
    hipLaunchKernelGGL((mx_split<BITS, NB, MF, NF, WAVES, U>), nc::grid_of(tiles), dim3(WAVES * 64), 0, nc::stream(),
                       a);
    return nc::launched("mx_split");
}

// copy_to_lds for copies that stay in flight past LDS reads: before any read of LDS the compiler waits for every copy
// it knows of, as each might write what is read. Which copies a read needs is counted in mx_tile, so these are
// hidden from it. They write no register; `to` goes through m0, which takes a wait state.
__device__ __forceinline__ void copy_to_lds_counted(const uint8_t *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from),
                 "s"(__builtin_amdgcn_readfirstlane(to)) : "m0", "memory");
}
// From `base`, the same for every lane, and a lane's own offset: no vector instructions for an address (1 to 5% of the
// larger tiles' time).
__device__ __forceinline__ void copy_to_lds_counted(const uint8_t *base, uint32_t offset, uint32_t to) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const uint64_t low = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at);
    const uint64_t high = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(low | high << 32),
                 "s"(__builtin_amdgcn_readfirstlane(to)) : "m0", "memory");
}

// Many outputs: a workgroup of WM x WN waves takes 32 MF WM rows of x by 32 NF WN weight rows (of each weight), each
// wave 32 MF x 32 NF of them. Operands are staged in LDS two steps at a time: 4-bit rows are copied 128 bytes at a
// time, as whole lines of the cache come twice as fast as halves (measured: 33 against 16 TB/s). A wave reads half a
// step's operands into registers while it multiplies the half before.
// With two buffers there is one barrier a pair of steps, before its last half: by then the next pair has landed and
// this one is read, so the copies of the pair after next start, with two steps to land. With one the next pair's copies
// start at that barrier and have landed at another, half a step later: other workgroups, of which a CU takes twice as
// many, fill the wait. Where the steps are odd the last is the second of a pair whose first is not multiplied again.
// The scales come four steps at a time, 16 bytes a row, with the pairs 0, 2, 4 ... The outputs go through LDS, a wave's
// 32 rows at a time, so that whole lines are written (a lane's own outputs are 16 bytes of a row: 4096 x 8192 x 8192
// took 255 us so, 140 of them without the stores).
// With WK > 1 the tile is one wave's, and WK waves have the whole of it and a part of k each, with stages of their own
// and so without barriers; their sums are added in the order of the waves. For the shapes whose tiles are few and k
// long: 512 x 896 x 4864 in 4 bits 6.5 us, in 8 bits 9.1; 128 x 4096 x 4096 in 8 bits 8.1 (8.7, 11.1 and 11.1 with
// mx_split). Needs four steps.
template <int BITS, int NB, int WM, int WN, int MF, int NF, int BUFFERS, int WK>
__global__ __launch_bounds__(WM * WN * WK * 64) void mx_tile(MxArgs a) {
    static_assert(WK == 1 || WM * WN == 1, "k is split over waves that have the whole tile each");
    using S = Stage<128, 2>;
    constexpr int WAVES = WM * WN, BM = 32 * MF * WM, BN = 32 * NF * WN, XH = BITS / 4;
    constexpr int XC = BM / 8, WC = BN / 8, SC = (BM + NB * BN + 63) / 64;      // copies of 128-byte rows, of scales
    constexpr int BUFFER = (XH * XC + NB * WC) * 1024;
    constexpr int kScaleCopies = (SC + WAVES - 1) / WAVES, kCopies = (XH * XC + NB * WC) / WAVES;   // a wave's
    // Of a pair's copies into the second buffer, those that start a half later, with the pair before it: half in 8 bits
    // (512 x 896 x 4864 10.6 us with none, 10.0 so; a pair of 1867 x 8192 x 8192 418 and 400), in 4 no quicker.
    constexpr int kLate = BUFFERS == 2 && BITS == 8 ? kCopies / 2 : 0;
    constexpr int kOutRow = 32 * NF * 4 + 16;                       // bytes of LDS, and of it a wave has 32 rows
    static_assert(XC % WAVES == 0 && WC % WAVES == 0, "whole copies a wave");
    constexpr int kStaged = BUFFERS * (BUFFER + SC * 1024), kOut = WAVES * (WK == 1 ? 1 : NB) * 32 * kOutRow;
    constexpr int kShare = kStaged > kOut ? kStaged : kOut;
    __shared__ __align__(1024) uint8_t all_lds[WK * kShare];
    const int member = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave = WK == 1 ? member : 0, part_of_k = WK == 1 ? 0 : member;
    uint8_t *const lds = all_lds + part_of_k * kShare;
    uint8_t *const scales = lds + BUFFERS * BUFFER;

    const uint32_t mtiles = ((uint32_t)a.M + BM - 1) / BM, ntiles = ((uint32_t)a.N + BN - 1) / BN;
    if (nc::workgroup_id() >= mtiles * ntiles) return;
    const Tile tile = tile_of((uint32_t)nc::workgroup_id(), mtiles, ntiles);
    const int64_t m0 = tile.m * BM, n0 = tile.n * BN;
    const int lane = threadIdx.x & 63, row = lane & 31, g = lane >> 5, steps = a.steps;
    const int wm = wave / WN * (32 * MF), wn = wave % WN * (32 * NF);      // this wave's first row of each
    const int x_last = (int)min(a.M - 1 - m0, (int64_t)BM - 1), w_last = (int)min(a.N - 1 - n0, (int64_t)BN - 1);
    auto x_row = [&](int r) { return (uint32_t)(min(r, x_last) * steps); };
    auto w_row = [&](int r) { return (uint32_t)(min(r, w_last) * steps); };
    const uint8_t *xq = a.xq + (size_t)m0 * steps * (16 * BITS), *xs = a.xs + (size_t)m0 * steps * 4;
    const uint8_t *q[NB], *ws[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        q[b] = a.q[b] + (size_t)n0 * steps * 64;
        ws[b] = a.ws[b] + (size_t)n0 * steps * 4;
    }
    // This lane's part of the wave's copies: copies i * WAVES + wave of an operand, and of a group of scales. 8-bit
    // rows are two 128-byte ones, a step each, the halves of a block four chunks apart.
    uint32_t xat[XC / WAVES], wat[WC / WAVES];
    const uint8_t *sat[kScaleCopies];
#pragma unroll
    for (int i = 0; i < XC / WAVES; ++i) {
        const int c = i * WAVES + wave;
        xat[i] = x_row(S::row(lane, c)) * (16 * BITS) + (BITS == 4 ? S::slot(lane, c) * 16 : S::column(lane, c));
    }
#pragma unroll
    for (int i = 0; i < WC / WAVES; ++i)
        wat[i] = w_row(S::row(lane, i * WAVES + wave)) * 64 + S::slot(lane, i * WAVES + wave) * 16;
#pragma unroll
    for (int i = 0; i < kScaleCopies; ++i) {
        // (where the copies are fewer than the waves, several waves make the last one)
        const int r = min(i * WAVES + wave, SC - 1) * 64 + lane;
        sat[i] = r < BM        ? xs + x_row(r) * 4
                 : r < BM + BN ? ws[0] + w_row(r - BM) * 4
                               : ws[NB - 1] + w_row(r - BM - BN) * 4;
    }
    const uint32_t base = (uint32_t)(size_t)(__attribute__((address_space(3))) uint8_t *)lds;
    // This wave's pairs of steps, and whether its last is the odd step alone.
    const int pairs = (steps + 1) / 2, share = (pairs + WK - 1) / WK;
    const int p_begin = part_of_k * share, p_end = min(pairs, p_begin + share), odd = p_end == pairs ? steps & 1 : 0;
    // Waves that share a stage wait for each other; those with a part of k each have none to wait for.
    auto meet = [] {
        if constexpr (WAVES > 1) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // The first of the two steps in pair p's buffer. Pairs past the last are copied as the last and not multiplied.
    auto first_step = [&](int p) { return min(2 * p, steps - 2); };
    // Copy i of pair p into a buffer.
    auto copy_piece = [&](int p, int buffer, int i) {
        const int s = first_step(p);
        const uint32_t to = base + buffer * BUFFER + wave * 1024;
        if (i < XH * (XC / WAVES)) {
            const int t = i / (XC / WAVES), c = i % (XC / WAVES);
            copy_to_lds_counted(xq + (size_t)(s + t) * (16 * BITS), xat[c], to + (t * XC + c * WAVES) * 1024);
        } else {
            const int j = i - XH * (XC / WAVES), b = j / (WC / WAVES), c = j % (WC / WAVES);
            copy_to_lds_counted(q[b] + (size_t)s * 64, wat[c], to + (XH * XC + b * WC + c * WAVES) * 1024);
        }
    };
    // The scales of the four steps that pair p is of: 16 bytes that lie inside every row.
    auto copy_scales = [&](int p) {
        const int first = min(p / 2 * 4, steps - 4);
#pragma unroll
        for (int i = 0; i < kScaleCopies; ++i) {
            const int to = p / 2 % BUFFERS * SC + min(i * WAVES + wave, SC - 1);
            copy_to_lds_counted(sat[i] + first * 4, base + BUFFERS * BUFFER + to * 1024);
        }
    };
    // Half a step's operands: a lane's block g + 2 half of every row it multiplies.
    struct Half {
        i32x4 x[MF][XH], w[NB][NF];
    };
    // Every row's four scales of a step, this lane's first block's lowest.
    struct Scales {
        uint32_t x[MF], w[NB][NF];
    };
    constexpr int kReads = NB * NF + MF * XH, kRows = NB * NF + MF;        // LDS reads of a half, of a step's scales
    // Read p of half `half` of step `step` (0, 1) of a buffer. (The second step's 4-bit blocks are chunks 4 .. 7.)
    auto read_half = [&](Half &f, int buffer, int step, int half, int p) {
        const uint8_t *from = lds + buffer * BUFFER;
        const int block = g + 2 * half;
        if (p < NB * NF) {
            f.w[p / NF][p % NF] = *reinterpret_cast<const i32x4 *>(
                from + (XH * XC + p / NF * WC) * 1024 + 32 * (p % NF) * 128 + (S::at(wn + row, block, 0) ^ 64 * step));
        } else {
            const int i = (p - NB * NF) / XH, h = (p - NB * NF) % XH;
            f.x[i][h] = *reinterpret_cast<const i32x4 *>(
                from + 32 * i * 128 +
                (BITS == 4 ? S::at(wm + row, block, 0) ^ 64 * step : step * XC * 1024 + S::at(wm + row, block, h)));
        }
    };
    auto read_scales = [&](Scales &e, int s, int p) {
        s = min(s, steps - 1);
        const uint8_t *from = scales + (BUFFERS == 2 ? s >> 2 & 1 : 0) * (SC * 1024) + (s - min(s & ~3, steps - 4)) * 4;
        if (p < NB * NF) {
            const int r = BM + p / NF * BN + wn + 32 * (p % NF) + row;
            e.w[p / NF][p % NF] = *reinterpret_cast<const uint32_t *>(from + r * 16);
        } else {
            e.x[p - NB * NF] = *reinterpret_cast<const uint32_t *>(from + (wm + 32 * (p - NB * NF) + row) * 16);
        }
    };
    f32x16 acc[NB][MF][NF] = {};
    // Half a step's products, the outputs acc[n = 8 (r / 4) + 4 (l / 32) + r % 4][m = l % 32]. `other(p)`, p < pieces,
    // is the next half's reads and copies, spread between the products: in one place they would leave the matrix
    // core idle, as all waves come to them at once. 4 bits: 64 values of k in one instruction, which picks a scale's
    // byte itself.
    auto multiply = [&](const Half &f, const Scales &e, auto half, int pieces, auto other) {
        constexpr int OP = 2 * decltype(half)::value, products = NB * NF * MF;
        auto wide = [](i32x4 v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); };
#pragma unroll
        for (int k = 0; k < products; ++k) {
            const int b = k / (NF * MF), j = k / MF % NF, i = k % MF;
            acc[b][i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                wide(f.w[b][j]), wide(f.x[i][0]), acc[b][i][j], 4, 4, OP, e.w[b][j] >> (8 * g), OP, e.x[i] >> (8 * g));
#pragma unroll
            for (int p = k * pieces / products; p < (k + 1) * pieces / products; ++p) other(p);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // 8 bits: four parts of 8 values a lane, each converted while the part before it is multiplied.
    struct Part {
        bf16x8 x[MF], w[NB][NF];
    } part;
    struct Powers {
        float x[MF], w[NB][NF];
    } powers;
    auto take_powers = [&](const Scales &e, int half) {
        const int at = 8 * g + 16 * half;
#pragma unroll
        for (int i = 0; i < MF; ++i) powers.x[i] = power_at(e.x[i], at);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NF; ++j) powers.w[b][j] = power_at(e.w[b][j], at);
    };
    auto convert = [&](Part &to, const Half &f, int t, int p) {
        if (p < NB * NF) {
            to.w[p / NF][p % NF] = to_bf16(f.w[p / NF][p % NF][t], powers.w[p / NF][p % NF]);
        } else {
            const int i = p - NB * NF;
            to.x[i] = to_bf16(f.x[i][t / 2 % XH][t % 2 * 2], f.x[i][t / 2 % XH][t % 2 * 2 + 1], powers.x[i]);
        }
    };
    // Half f, whose first part is in `part`; leaves the first part of half `half` of a step of scales e, f_next, there.
    auto multiply_converted = [&](const Half &f, const Half &f_next, const Scales &e, int half, int pieces,
                                  auto other) {
        constexpr int products = NB * NF * MF;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            Part next;
            if (t == 3) take_powers(e, half);
#pragma unroll
            for (int k = 0; k < products; ++k) {
                const int b = k / (NF * MF), j = k / MF % NF, i = k % MF;
                acc[b][i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(part.w[b][j], part.x[i], acc[b][i][j], 0, 0, 0);
                // the other work in the first three parts: what it reads is converted in the fourth
                if (t < 3) {
                    const int at = t * products + k, of = 3 * products;
#pragma unroll
                    for (int p = at * pieces / of; p < (at + 1) * pieces / of; ++p) other(p);
                }
#pragma unroll
                for (int p = k * kRows / products; p < (k + 1) * kRows / products; ++p)
                    convert(next, t < 3 ? f : f_next, (t + 1) % 4, p);
                __builtin_amdgcn_sched_barrier(0);
            }
            part = next;
        }
    };
    Half f0, f1;
    Scales e0, e1;
    constexpr std::integral_constant<int, 0> first_half{};
    constexpr std::integral_constant<int, 1> second_half{};
    auto product = [&](const Half &f, const Half &f_next, const Scales &e, const Scales &e_next, auto half, int pieces,
                       auto other) {
        if constexpr (BITS == 4) multiply(f, e, half, pieces, other);
        else multiply_converted(f, f_next, e_next, 1 - decltype(half)::value, pieces, other);
    };
    // A pair's first step (f0 and e0 hold its first half and scales), and then its second's first half read.
    auto first = [&](int p, auto which) {
        constexpr int B = decltype(which)::value;
        product(f0, f1, e0, e0, first_half, kReads + kLate, [&](int i) {
            if (i < kReads) read_half(f1, B, 0, 1, i);
            else copy_piece(p + 1, 1 - B, kCopies - kLate + i - kReads);
        });
        product(f1, f0, e0, e1, second_half, kReads + kRows, [&](int i) {
            if (i < kReads) read_half(f0, B, 1, 0, i);
            else read_scales(e1, first_step(p) + 1, i - kReads);
        });
    };
    // The first half of step `begin` of buffer 0, step s.
    auto begin_pair = [&](int begin, int s) {
#pragma unroll
        for (int i = 0; i < kReads; ++i) read_half(f0, 0, begin, 0, i);
#pragma unroll
        for (int i = 0; i < kRows; ++i) read_scales(e0, s, i);
        if constexpr (BITS == 8) {
            take_powers(e0, 0);
#pragma unroll
            for (int i = 0; i < kRows; ++i) convert(part, f0, 0, i);
        }
    };
    // A pair's second step (f0 and e1 hold its first half and scales); the next pair's first half read, of its second
    // step where that is the last, odd one.
    auto second = [&](int p, auto which) {
        constexpr int B = decltype(which)::value;
        product(f0, f1, e1, e1, first_half, kReads, [&](int i) { read_half(f1, B, 1, 1, i); });
        const int begin = p + 2 == p_end ? odd : 0;
        if constexpr (BUFFERS == 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            meet();                                                 // pair p is read by every wave
            if (p % 2 == 1) copy_scales(p + 1);
            product(f1, f1, e1, e1, second_half, kCopies, [&](int i) { copy_piece(p + 1, 0, i); });
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            meet();                                                 // pair p + 1 has landed
            begin_pair(begin, 2 * p + 2);
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            meet();                                                 // pair p + 1 has landed and p is read, for all
            product(f1, f0, e1, e0, second_half, kReads + kRows + kCopies - kLate, [&](int i) {
                if (i < kReads) read_half(f0, 1 - B, begin, 0, i);
                else if (i < kReads + kRows) read_scales(e0, 2 * p + 2, i - kReads);
                else copy_piece(p + 2, B, i - kReads - kRows);
            });
            if (p % 2 == 0) copy_scales(p + 2);
        }
    };
    auto pair = [&](int p, auto which) {
        if (!odd || p + 1 < p_end) first(p, which);
        else e1 = e0;
        second(p, which);
    };
    if (WK == 1 || p_begin < p_end) {
        copy_scales(p_begin);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) copy_piece(p_begin, 0, i);
        if constexpr (BUFFERS == 2) {
            if (p_begin % 2 == 1) copy_scales(p_begin + 1);
#pragma unroll
            for (int i = 0; i < kCopies - kLate; ++i) copy_piece(p_begin + 1, 1, i);
        }
        // (the second pair's scales may be waited for too)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(BUFFERS == 2 ? kCopies - kLate : 0) : "memory");
        meet();
        const int alone = odd && p_begin + 1 == p_end;              // nothing but the odd step
        begin_pair(alone, 2 * p_begin);
        if constexpr (BUFFERS == 2) {
            for (int p = p_begin; p < p_end; p += 2) {
                pair(p, std::integral_constant<int, 0>{});
                if (p + 1 < p_end) pair(p + 1, std::integral_constant<int, 1>{});
            }
        } else {
            for (int p = p_begin; p < p_end - odd; ++p) {
                first(p, std::integral_constant<int, 0>{});
                second(p, std::integral_constant<int, 0>{});
            }
            if (odd) {                                              // f0, e0: the last step's first half and scales
                product(f0, f1, e0, e0, first_half, kReads, [&](int i) { read_half(f1, 0, 1, 1, i); });
                product(f1, f1, e0, e0, second_half, 0, [](int) {});
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j) asm volatile("" : "+v"(acc[b][i][j]));
    __syncthreads();                                   // the last copies have landed and the last reads are done
    constexpr int kAcross = 8 * NF, kDown = 64 / kAcross;           // lanes a row of 32 NF outputs, rows at a time
    if constexpr (WK > 1) {
        // every wave's sums side by side, then a share of the rows each, added in the order of the waves
        constexpr int kAll = 32 / kDown, kMine = (kAll + WK - 1) / WK;
        static_assert(MF == 1 && kAll % kMine == 0, "32 rows of outputs, whole shares of them");
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f32x4 v;
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[c] = acc[b][0][j][4 * r + c];
                    *reinterpret_cast<f32x4 *>(lds + (b * 32 + row) * kOutRow + (32 * j + 8 * r + 4 * g) * 4) = v;
                }
        __syncthreads();
        if (part_of_k * kMine >= kAll) return;
        const int down = part_of_k * (kMine * kDown) + lane / kAcross;
        f32x4 v[kMine];
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            f32x4 sum[NB] = {};
#pragma unroll
            for (int w = 0; w < WK; ++w)
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    sum[b] += *reinterpret_cast<const f32x4 *>(
                        all_lds + w * kShare + (b * 32 + down + k * kDown) * kOutRow + lane % kAcross * 16);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[k][c] = NB == 1 ? sum[0][c] : silu_times(sum[0][c], sum[NB - 1][c]);
        }
        finish<NB, kMine>(a, m0 + down, kDown, n0 + lane % kAcross * 4, v);
        return;
    }
    uint8_t *const mine = lds + wave * (32 * kOutRow);
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
        f32x4 v[32 / kDown];
#pragma unroll
        for (int k = 0; k < 32 / kDown; ++k)
            v[k] =
                *reinterpret_cast<const f32x4 *>(mine + (k * kDown + lane / kAcross) * kOutRow + lane % kAcross * 16);
        asm volatile("" ::: "memory");
        finish<NB, 32 / kDown>(a, m0 + wm + 32 * i + lane / kAcross, kDown, n, v);
    }
}

template <int BITS, int NB, int WM, int WN, int MF, int NF, int BUFFERS, int WK = 1>
int32_t launch_tile(const MxArgs &a) {
    constexpr int BM = 32 * MF * WM, BN = 32 * NF * WN;
    const int64_t tiles = (a.M + BM - 1) / BM * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL((mx_tile<BITS, NB, WM, WN, MF, NF, BUFFERS, WK>), nc::grid_of(tiles), dim3(WM * WN * WK * 64), 0,
                       nc::stream(), a);
    return nc::launched("mx_tile");
}

template <int BITS, int NB>
int32_t launch(const MxArgs &a) {
    switch (nc::mx_tile(a.M, a.N, a.steps, BITS, NB)) {
        case nc::MxTile::kRow: return launch_split<BITS, NB, 1, 1, 4, 2>(a);
        case nc::MxTile::kLongRow: return launch_split<BITS, NB, 1, 1, 8, 2>(a);
        case nc::MxTile::kWideRow:
            if constexpr (BITS == 8 && NB == 1) return launch_split<8, 1, 1, 2, 8, 2>(a);
            [[fallthrough]];                                        // (no other has it)
        case nc::MxTile::kSplit: return launch_split<BITS, NB, 2, 2, 4, NB == 1 ? 2 : 1>(a);
        case nc::MxTile::kJoined:
            return launch_tile<BITS, NB, 1, 1, 1, BITS == 8 && NB == 1 ? 2 : 1, BITS == 4 && NB == 1 ? 1 : 2, 4>(a);
        case nc::MxTile::kDeep: return launch_tile<BITS, NB, 2, 2, 1, 1, 2>(a);
        case nc::MxTile::kMedium:
            if constexpr (BITS == 8) return launch_tile<8, NB, 2, 2, NB, 3 - NB, 1>(a);
            [[fallthrough]];                                        // (4 bits do not have it)
        case nc::MxTile::kMediumDeep:
            if constexpr (NB == 1) return launch_tile<BITS, 1, 2, 2, BITS == 4 ? 2 : 1, 2, 2>(a);
            [[fallthrough]];                                        // (no pair has it)
        case nc::MxTile::kSmall: return launch_tile<BITS, NB, 2, 2, 1, 1, 1>(a);
        case nc::MxTile::kLarge: return launch_tile<BITS, NB, 2, 4, BITS == 4 ? 4 : 2, NB == 1 ? 2 : 1, 2>(a);
    }
    return NC_BAD_ARGS;
}

// Shapes whose outputs are fewer than 2^39 (two terabytes of float32; tiles of 16 x 16 are counted in 32 bits) and
// whose rows a tile addresses in 32 bits.
bool mx_matmul_shape(const int64_t *s) {
    return s[0] >= 0 && s[1] > 0 && s[2] > 0 && s[0] < (1 << 26) && s[1] < (1 << 26) && s[2] <= (1 << 24) &&
           s[0] * s[1] < (int64_t)1 << 39;
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
