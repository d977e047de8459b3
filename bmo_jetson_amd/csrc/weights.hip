// weights.hip -- 8-bit rows times Q4_0 weights on the matrix cores, plain and
// gated.
//
//   y[m][n] = sum over blocks b of d4[n][b] d8[m][b] sum_j (c_j - 8) q_j
//
// A block's sum is an exact integer: v_mfma_i32 over its 32 elements, the 8-bit
// rows as the rows and the weights (16 (code - 8), one shift and mask from their
// nibbles) as the columns of the result.  It starts from the integer whose bits
// are the float 1.5 * 2^23, so that the result's bits, read as a float, are that
// plus the sum, exactly (sums stay below 2^20), and one fma with d4 takes the
// offset out again: -1.5 * 2^23 * d4 is exact for an fp16 d4.  A second one adds
// d8 times that, so an output is off by the roundings of an fp32 sum of its
// blocks' parts only.  (Converting the integer takes as long as seven fmas.)
//
// Few rows are bound by reading the weights once, many by those two fmas: a
// 32 x 32 tile of a block takes 32 of them a lane and 10 other vector
// instructions beside the one matrix instruction, about 4 clocks each with the
// matrix cores in turn.
#include "kernels.hpp"
#include "product_shape.hpp"
#include "rows_device.hpp"

namespace bmo {

namespace {

typedef int wt_int4 __attribute__((ext_vector_type(4)));
typedef uint32_t wt_uint2 __attribute__((ext_vector_type(2)));
typedef uint32_t wt_uint4 __attribute__((ext_vector_type(4)));
typedef int wt_int16 __attribute__((ext_vector_type(16)));
typedef float wt_float16 __attribute__((ext_vector_type(16)));

constexpr int kMagicBits = 0x4B400000;       // 1.5 * 2^23
constexpr float kMagic = 12582912.0f;
constexpr float kCodeStep = 0.0625f;         // codes enter times 16

// A thread a block: 18 bytes of ggml to its unit.
__global__ __launch_bounds__(256) void pack_kernel(PackParams p, FastDiv div_blocks, uint32_t n) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t nb = (uint32_t) p.g.cols / 32;
    const uint32_t r = div_blocks.div(i);
    const int b = (int) (i - r * nb), row = p.row0 + (int) r;
    const uint16_t *src = reinterpret_cast<const uint16_t *>(p.blocks + (int64_t) i * 18);
    uint32_t qs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) qs[j] = src[1 + j];
    uint8_t *unit = p.w + ((int64_t) (row / kUnitRows) * p.g.chunks + b / 4) * kUnitBytes;
    const int t = b % 4, ri = row % kUnitRows;
    // byte k of a block holds elements k (low) and 16 + k (high): octet g of
    // its elements is the low or high nibbles of bytes 8 (g % 2) ..
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int at = 4 * (g & 1), sh = g & 2 ? 4 : 0;
        const uint32_t lo = (((qs[at] | qs[at + 1] << 16) >> sh) & 0x0F0F0F0Fu);
        const uint32_t hi = (((qs[at + 2] | qs[at + 3] << 16) >> sh) & 0x0F0F0F0Fu);
        reinterpret_cast<uint32_t *>(unit)[(g * kUnitRows + ri) * 4 + t] = (lo | hi << 4) ^ 0x88888888u;
    }
    reinterpret_cast<uint16_t *>(unit + kUnitScales)[ri * 4 + t] = src[0];
}

__device__ __forceinline__ float half_lo(uint32_t u) { return f16_bits_to_f32(u & 0xFFFFu); }
__device__ __forceinline__ float half_hi(uint32_t u) { return f16_bits_to_f32(u >> 16); }

// The activation of a gate times what it lets through.  exp is the hardware's
// 2^x, whose argument a product would leave |a| 2^-24 off, times 1 + ln 2 of what
// that product lost: 4 roundings however large |a| is.  (Clamped past exp's range
// on both sides, so that an infinite argument loses nothing.)  The quotient is a
// product with the hardware's reciprocal, of a sixteenth of the divisor so that it
// stays normal up to exp's overflow.  Some twelve instructions; expf and a division
// take thirty.  (1000 x 5632 x 128, where gates cost most: 16.2 us, without what the
// product lost 15.5.)
__device__ __forceinline__ float gate(float g, float u, int activation) {
    // GELU by its tanh form: 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
    const float a =
        __builtin_amdgcn_fmed3f(activation == kSilu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g), -200.0f, 200.0f);
    constexpr float kTurn = 1.44269502162933349609375f, kTurnRest = 1.92596299e-8f;  // log2 e
    const float t = a * -kTurn, lost = __builtin_fmaf(a, -kTurnRest, __builtin_fmaf(a, -kTurn, -t));
    const float e = __builtin_amdgcn_exp2f(t) * __builtin_fmaf(lost, 0.6931471805599453f, 1.0f);
    return g * 0.0625f * __builtin_amdgcn_rcpf(__builtin_fmaf(e, 0.0625f, 0.0625f)) * u;
}

// A barrier that waits for LDS alone, not for loads under way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The two divisions that place a workgroup.
struct Places {
    FastDiv main, rest;
};
Places make_places(unsigned columns) {
    return {make_fastdiv(columns / 8 ? columns / 8 : 1), make_fastdiv(columns % 8 ? columns % 8 : 1)};
}
__device__ __forceinline__ Place place(const Places &d) {
    return product_place(blockIdx.x, blockIdx.y, gridDim.x, gridDim.y, [&](uint32_t n) { return d.main.div(n); },
                         [&](uint32_t n) { return d.rest.div(n); });
}

// One row: vector units alone, which spend half the instructions on it that the
// matrix cores' sixteen rows take.  A workgroup takes NT tiles of 16 outputs (of
// a gated product two of gates and the two that they let through), its KW waves
// a run of their units each.  Lane (g, i) multiplies block g of a unit's four of
// output i, for which the four octets change places between lanes: eight dot
// products that begin with the float's bits, as the matrix instructions do.  The
// row lies in LDS, its scales in fp32.  Bound by the weights' bytes and the
// launch: 12288 x 4096 in 6.6 us, 4.3 TB/s (a large copy: 5.1), with the matrix
// cores 8.1; gated 2 x 5632 x 4096 7.8 against 9.5.
constexpr int kOneRowChunks = 256;  // of a row in LDS, 144 bytes each

// Dword t of lanes 16 g .. to dword g of lanes 16 t ..: from octet g of four
// blocks to four octets of block g.  (Wait states: the compiler's hazard pass
// does not see inside.)
__device__ __forceinline__ wt_uint4 turn_octets(const wt_uint4 &v) {
    uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
    asm volatile(
        "s_nop 3\n\t"
        "v_permlane32_swap_b32 %0, %2\n\t"
        "v_permlane32_swap_b32 %1, %3\n\t"
        "s_nop 3\n\t"
        "v_permlane16_swap_b32 %0, %1\n\t"
        "v_permlane16_swap_b32 %2, %3\n\t"
        "s_nop 3"
        : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
    return wt_uint4{a, b, c, d};
}

template <int NT, int KW, int PF, bool GATED>
__global__ __launch_bounds__(64 * KW) void one_row_kernel(ProductParams p) {
    static_assert(!GATED || NT == 4, "two tiles of gates and the two that they let through");
    extern __shared__ uint8_t s_row[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int nb = p.g.cols / 32, last = p.g.chunks - 1;
    const int per = (p.g.chunks + KW - 1) / KW, c0 = wave * per, c1 = min(c0 + per, p.g.chunks);
    const uint8_t *w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int tile = GATED ? (int) blockIdx.x * 2 + (n & 1) + (n & 2 ? p.g.tiles / 2 : 0) : (int) blockIdx.x * NT + n;
        w[n] = p.w + (int64_t) min(tile, p.g.tiles - 1) * p.g.chunks * kUnitBytes;
    }
    wt_uint4 q[PF][NT];
    uint32_t d4[PF][NT];
    auto load = [&](int j, int c) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint8_t *u = w[n] + (uint32_t) c * (uint32_t) kUnitBytes;
            q[j][n] = __builtin_nontemporal_load(reinterpret_cast<const wt_uint4 *>(u + lane * 16));
            d4[j][n] = *reinterpret_cast<const uint16_t *>(u + kUnitScales + i16 * 8 + g * 2);
        }
    };
#pragma unroll
    for (int j = 0; j < PF; ++j) load(j, min(c0 + j, last));
    float *s_d8 = reinterpret_cast<float *>(s_row + p.g.chunks * kUnitCols);
    for (int o = threadIdx.x; o < nb * 2; o += 64 * KW)
        reinterpret_cast<wt_uint4 *>(s_row)[o] = reinterpret_cast<const wt_uint4 *>(p.codes)[o];
    // (past the last block weights are zeros, the codes whatever lies there)
    for (int b = threadIdx.x; b < p.g.chunks * 4; b += 64 * KW) s_d8[b] = b < nb ? half_lo(p.scales[b]) : 0.0f;
    lds_barrier();
    float acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = 0.0f;
    for (int c = c0; c < c1; c += PF) {
#pragma unroll
        for (int j = 0; j < PF; ++j) {
            if (c + j >= c1) break;
            const wt_uint4 *x = reinterpret_cast<const wt_uint4 *>(s_row + (c + j) * kUnitCols + g * 32);
            const wt_uint4 xa = x[0], xb = x[1];
            const float d8 = s_d8[4 * (c + j) + g];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const wt_uint4 v = turn_octets(q[j][n]);
                float ds = half_lo(d4[j][n]);
                asm volatile("" : "+v"(ds));  // (in fp32: an fma that widens an operand takes twice the time)
                int z = kMagicBits;
#pragma unroll
                for (int o = 0; o < 4; ++o) {
                    z = __builtin_amdgcn_sdot4((int) (v[o] << 4 & 0xF0F0F0F0u), (int) (o < 2 ? xa : xb)[2 * (o & 1)], z, false);
                    z = __builtin_amdgcn_sdot4((int) (v[o] & 0xF0F0F0F0u), (int) (o < 2 ? xa : xb)[2 * (o & 1) + 1], z, false);
                }
                acc[n] = __builtin_fmaf(d8, __builtin_fmaf(__builtin_bit_cast(float, z), ds, -kMagic * ds), acc[n]);
            }
            if (c + j + PF < c1) load(j, c + j + PF);
        }
    }
    __shared__ float s_acc[KW][NT][16];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        acc[n] += __shfl_xor(acc[n], 16);
        acc[n] += __shfl_xor(acc[n], 32);
        if (g == 0) s_acc[wave][n][i16] = acc[n];
    }
    __syncthreads();
    auto joined = [&](int n, int i) {
        float v = s_acc[0][n][i];
#pragma unroll
        for (int k = 1; k < KW; ++k) v += s_acc[k][n][i];
        return v * kCodeStep;
    };
    const int t = threadIdx.x;
    if constexpr (GATED) {
        if (t >= 32) return;
        const int col = (int) blockIdx.x * 32 + t;
        const float v = gate(joined(t >> 4, t & 15), joined(2 + (t >> 4), t & 15), p.activation);
        if (p.out) store1(p.out, col, v, p.type);
        if (p.out_codes) {
            const Scale8 s = scale_of(half_max(__builtin_fabsf(v)));
            p.out_codes[col] = (int8_t) code1(v, s.inv);
            if (t == 0) p.out_scales[col / 32] = (uint16_t) s.bits;
        }
    } else {
        const int col = (int) blockIdx.x * 16 * NT + t;
        if (t < 16 * NT && col < p.g.rows) store1(p.out, col, joined(t >> 4, t & 15), p.type);
    }
}

template <int NT, int KW, int PF, bool GATED>
hipError_t run_one(const ProductParams &p, hipStream_t stream) {
    ProductParams q = p;
    void *args[] = {&q};
    const int per = GATED ? 2 : NT, tiles = GATED ? p.g.tiles / 2 : p.g.tiles;
    return hipLaunchKernel(reinterpret_cast<const void *>(one_row_kernel<NT, KW, PF, GATED>),
                           dim3((unsigned) ((tiles + per - 1) / per)), dim3(64 * KW), args,
                           (size_t) p.g.chunks * (kUnitCols + 16), stream);
}

constexpr int kRowStride = 144;  // of 128 codes in LDS: 16 rows' octets lie in different banks

// Few rows: a workgroup takes 16 rows and NT tiles of 16 outputs (of a
// gated product two tiles of gates and the two that they let through), its KW
// waves a run of the tiles' units each; their sums are joined in LDS, wave after
// wave.  The 8-bit rows are the rows of the result here: a lane has one output
// of four rows, with the output's scales its own and the rows' read from LDS,
// where the wave puts them.  PF units are under way at once: 2 of the narrowest
// shape, whose waves wait for loads (16 x 4096 x 4096 5.2 against 5.6 us, 64 x 1000 x
// 11264 10.8 against 11.8), 1 of 16 x 64 and of gated products, whose registers a
// second costs waves (16 x 32001 x 4096 16.7 against 18.6, gated 16 x 5632 x 4096 9.7
// against 10.0), and of 16 x 32, whose times in the rule are those of 1 (32 x 4096 x
// 4096 6.7; with 2 6.1).  Bound by a load, its use and the joining in turn: 16 x 4096
// x 4096 takes 5.2 us, where the bytes alone take 1.9 and a launch 1.6.
template <int NT, int KW, int PF, bool GATED>
__global__ __launch_bounds__(64 * KW) void few_rows_kernel(ProductParams p, Places places) {
    static_assert(!GATED || NT == 4, "two tiles of gates and the two that they let through");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const Place at = place(places);
    const int m0 = (int) at.y * 16;
    const int nb = p.g.cols / 32, last = p.g.chunks - 1;
    const int per = (p.g.chunks + KW - 1) / KW, c0 = wave * per, c1 = min(c0 + per, p.g.chunks);
    const uint8_t *w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        int tile = GATED ? (int) at.x * 2 + (n & 1) + (n & 2 ? p.g.tiles / 2 : 0) : (int) at.x * NT + n;
        tile = min(tile, p.g.tiles - 1);
        w[n] = p.w + (int64_t) tile * p.g.chunks * kUnitBytes;
    }
    // The rows' offsets from the workgroup's first fit 32 bits: 15 * 2^24.  (A
    // unit's 128 codes of a row are read by eight lanes, and go through LDS to
    // the lanes that multiply them.)
    const int8_t *codes = p.codes + (int64_t) m0 * p.g.cols;
    const uint16_t *scales = p.scales + (int64_t) m0 * nb;
    uint32_t x_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x_at[i] = (uint32_t) min(8 * i + (lane >> 3), p.n_rows - 1 - m0) * (uint32_t) p.g.cols;
    const uint32_t d_at = (uint32_t) min(i16, p.n_rows - 1 - m0) * (uint32_t) nb;
    wt_uint4 q[PF][NT], x[PF][2];
    wt_uint2 d4[PF][NT];
    uint32_t d8[PF];
    auto load = [&](int j, int c) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint8_t *u = w[n] + (uint32_t) c * (uint32_t) kUnitBytes;
            q[j][n] = __builtin_nontemporal_load(reinterpret_cast<const wt_uint4 *>(u + lane * 16));
            d4[j][n] = *reinterpret_cast<const wt_uint2 *>(u + kUnitScales + i16 * 8);
        }
        // (past the last block weights are zeros)
        const uint32_t e = (uint32_t) min(c * kUnitCols + (lane & 7) * 16, p.g.cols - 16), b = (uint32_t) min(4 * c + g, nb - 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) x[j][i] = *reinterpret_cast<const wt_uint4 *>(codes + (x_at[i] + e));
        d8[j] = scales[d_at + b];
    };
    __shared__ rw_float4 s_acc[KW][NT][64];
    __shared__ float s_d8[KW][4][16];
    __shared__ uint8_t s_x[KW][16][kRowStride];
    rw_float4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] = rw_float4{0, 0, 0, 0};
    const wt_int4 magic = {kMagicBits, kMagicBits, kMagicBits, kMagicBits};
#pragma unroll
    for (int j = 0; j < PF; ++j) load(j, min(c0 + j, last));
    for (int c = c0; c < c1; c += PF) {
#pragma unroll
        for (int j = 0; j < PF; ++j) {
            if (c + j >= c1) break;
            __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses stay in order)
            s_d8[wave][g][i16] = 4 * (c + j) + g < nb ? half_lo(d8[j]) : 0.0f;  // (past the last block nothing)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *reinterpret_cast<wt_uint4 *>(&s_x[wave][8 * i + (lane >> 3)][(lane & 7) * 16]) = x[j][i];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                long wv[NT];
                float ds[NT], off[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t v = q[j][n][t], s = d4[j][n][t >> 1];
                    wv[n] = __builtin_bit_cast(long, wt_uint2{v << 4 & 0xF0F0F0F0u, v & 0xF0F0F0F0u});
                    ds[n] = t & 1 ? half_hi(s) : half_lo(s);
                    asm volatile("" : "+v"(ds[n]));  // (in fp32: an fma that widens an operand takes twice the time)
                    off[n] = -kMagic * ds[n];
                }
                const rw_float4 dr = *reinterpret_cast<const rw_float4 *>(&s_d8[wave][t][4 * g]);
                const long xv = *reinterpret_cast<const long *>(&s_x[wave][i16][t * 32 + g * 8]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const rw_float4 f =
                        __builtin_bit_cast(rw_float4, __builtin_amdgcn_mfma_i32_16x16x32_i8(xv, wv[n], magic, 0, 0, 0));
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[n][r] = __builtin_fmaf(dr[r], __builtin_fmaf(f[r], ds[n], off[n]), acc[n][r]);
                }
            }
            if (c + j + PF < c1) load(j, c + j + PF);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) s_acc[wave][n][lane] = acc[n];
    __syncthreads();
    auto joined = [&](int n) {
        rw_float4 v = s_acc[0][n][lane];
#pragma unroll
        for (int k = 1; k < KW; ++k) v += s_acc[k][n][lane];
        return v * kCodeStep;
    };
    const int64_t row0 = m0 + 4 * g;
    if constexpr (GATED) {
        if (wave != 0) return;
        const int n_out = p.g.rows / 2, n0 = (int) at.x * 32 + i16;
        float h[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const rw_float4 a = joined(n), b = joined(n + 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) h[n][r] = gate(a[r], b[r], p.activation);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t row = row0 + r;
            if (p.out && row < p.n_rows) {
                store1(p.out, row * p.out_stride + n0, h[0][r], p.type);
                store1(p.out, row * p.out_stride + n0 + 16, h[1][r], p.type);
            }
            if (p.out_codes) {
                const Scale8 s =
                    scale_of(row16_max(__builtin_elementwise_maximum(__builtin_fabsf(h[0][r]), __builtin_fabsf(h[1][r]))));
                if (row < p.n_rows) {
                    p.out_codes[row * n_out + n0] = (int8_t) code1(h[0][r], s.inv);
                    p.out_codes[row * n_out + n0 + 16] = (int8_t) code1(h[1][r], s.inv);
                    if (i16 == 0) p.out_scales[row * (n_out / 32) + at.x] = (uint16_t) s.bits;
                }
            }
        }
    } else {
        static_assert(NT <= KW, "a wave joins one tile at most");
        const int n = wave, col = ((int) at.x * NT + n) * 16 + i16;
        if (n >= NT || col >= p.g.rows) return;
        const rw_float4 v = joined(n);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (row0 + r < p.n_rows) store1(p.out, (row0 + r) * p.out_stride + col, v[r], p.type);
    }
}

// The shape's numbers are those of product_shape.hpp.
template <int SHAPE, int PF, bool GATED>
hipError_t run_few(const ProductParams &p, hipStream_t stream) {
    constexpr ProductShape S = GATED ? kGatedShapes[SHAPE] : kProductShapes[SHAPE];
    constexpr int NT = GATED ? 4 : S.outs / 16;
    static_assert(S.rows == 16, "the shape's rows");
    ProductParams q = p;
    const unsigned columns = (unsigned) (((GATED ? p.g.rows / 2 : p.g.rows) + S.outs - 1) / S.outs);
    Places places = make_places(columns);
    void *args[] = {&q, &places};
    return hipLaunchKernel(reinterpret_cast<const void *>(few_rows_kernel<NT, S.waves, PF, GATED>),
                           dim3(columns, (unsigned) ((p.n_rows + S.rows - 1) / S.rows)),
                           dim3(64 * S.waves), args, 0, stream);
}

// Many rows: a workgroup takes MT * 32 rows, a wave NT tiles of 32 outputs (of a
// gated product one of gates and the one that they let through), WN such pieces
// to a workgroup, each shared by KW waves, which take every KW-th unit of it and
// join their sums in LDS.  As with few rows a lane has one output, here of 16
// rows, whose scales are read from LDS.  The rows' codes and scales go there a
// unit ahead: eight lanes read a row's 128 codes, which costs the loads a
// quarter of what reading them as the matrix cores take them does.  D units'
// weights are under way at once.  AHEAD: a tile's matrix instruction stands
// before the fmas of the tile before it, which takes the registers of a second
// unit (64 x 128, D 1 against D 2 without: 1000 x 4096 x 5632 66 against 71 us, 515 x
// 6001 x 4000 48.6 against 51.8; gated 1000 x 5632 x 4096 133 against 139, 2048 rows
// 241 against 244; 64 x 256 plain the other way, 243 against 240 at 2048 x 12288 x
// 4096; narrower ones the same either way).
//
// 2048 x 12288 x 4096 takes 230 to 243 us, 850 to 895 TFLOP/s (64 x 256 outputs a
// workgroup): of 265 in an earlier form of 128 x 128 the vector and matrix
// instructions alone took 205, the accesses to LDS 25 and the loads from memory
// 40 (a copy that skips work); the two waves of a SIMD issue more than half of the
// time.  Three or four waves a SIMD, in 168 or 128 registers, need narrower pieces:
// 287 and 292 in that form.

// Two units' codes of 16 outputs each to a 32-column operand: lanes 16 to 31
// and 48 to 63 of the first change places with lanes 0 to 15 and 32 to 47 of
// the second.  (Wait states: the compiler's hazard pass does not see inside.)
__device__ __forceinline__ void pair_units(wt_uint4 &a, wt_uint4 &b) {
    uint32_t a0 = a[0], a1 = a[1], a2 = a[2], a3 = a[3], b0 = b[0], b1 = b[1], b2 = b[2], b3 = b[3];
    asm volatile(
        "s_nop 3\n\t"
        "v_permlane16_swap_b32 %0, %4\n\t"
        "v_permlane16_swap_b32 %1, %5\n\t"
        "v_permlane16_swap_b32 %2, %6\n\t"
        "v_permlane16_swap_b32 %3, %7\n\t"
        "s_nop 3"
        : "+v"(a0), "+v"(a1), "+v"(a2), "+v"(a3), "+v"(b0), "+v"(b1), "+v"(b2), "+v"(b3));
    a = wt_uint4{a0, a1, a2, a3};
    b = wt_uint4{b0, b1, b2, b3};
}

template <int MT, int NT, int WN, int KW, int D, bool AHEAD, bool GATED>
__global__ __launch_bounds__(64 * WN * KW, 2) void many_rows_kernel(ProductParams p, int n_pieces, Places places) {
    static_assert(!GATED || NT == 2, "a tile of gates and the one that they let through");
    constexpr int WAVES = WN * KW, ROWS = 32 * MT, XL = 4 * MT / WN;  // rows of a workgroup; loads of a lane
    constexpr bool ALONE = WN == 1;  // a wave reads only what it puts into LDS itself
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave % KW, wn = wave / KW;
    const int l32 = lane & 31, h = lane >> 5;
    const Place group = place(places);
    const int piece = (int) group.x * WN + wn;
    const int nb = p.g.cols / 32, last = p.g.chunks - 1;
    // (a tile past the last reads the last and stores nothing)
    const uint32_t tile_bytes = (uint32_t) p.g.chunks * (uint32_t) kUnitBytes;
    const uint8_t *w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int tile = GATED ? piece + n * (p.g.tiles / 4) : NT * piece + n;
        w[n] = p.w + (int64_t) min(2 * tile, p.g.tiles - 2) * tile_bytes;
    }
    const uint32_t scales_at = ((lane >> 4) & 1) * tile_bytes + kUnitScales + (lane & 15) * 8;
    // (the rows' offsets from the workgroup's first fit 32 bits: 63 * 2^24)
    const int first = (int) group.y * ROWS;
    const int8_t *codes = p.codes + (int64_t) first * p.g.cols;
    const uint16_t *scales = p.scales + (int64_t) first * nb;
    const int x_row = wn * (8 * XL) + (lane >> 3), piece16 = lane & 7;
    uint32_t x_at[XL], d_at[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const uint32_t row = (uint32_t) min(x_row + 8 * i, p.n_rows - 1 - first);
        x_at[i] = row * (uint32_t) p.g.cols;
        d_at[i] = row * (uint32_t) nb;
    }
    // A row's sixteens change places by the row, so that eight rows' lie in
    // different banks.  Results 4j + i of a lane are rows 8j + 4h + i: a half's
    // scales lie together.
    __shared__ wt_int4 s_x[KW][ALONE ? 1 : 2][ROWS][8];
    __shared__ float s_d8[KW][ALONE ? 1 : 2][ROWS / 32][4][2][16];
    wt_int4 xr[XL];
    uint32_t dr[XL];
    auto load_x = [&](int c) {  // (past the last block weights are zeros)
        const uint32_t e = (uint32_t) min(c * kUnitCols + piece16 * 16, p.g.cols - 16);
        const uint32_t b = (uint32_t) min(4 * c + (lane & 3), nb - 1);
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            xr[i] = *reinterpret_cast<const wt_int4 *>(codes + (x_at[i] + e));
            dr[i] = scales[d_at[i] + b];
        }
    };
    auto put_x = [&](int buffer, int c) {
        const bool real = 4 * c + (lane & 3) < nb;  // (past the last block nothing)
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int row = x_row + 8 * i;
            s_x[kw][buffer][row][piece16 ^ (x_row & 7)] = xr[i];
            // (lanes 4 apart write the same)
            s_d8[kw][buffer][row >> 5][lane & 3][(row >> 2) & 1][((row >> 3) & 3) * 4 + (row & 3)] =
                real ? half_lo(dr[i]) : 0.0f;
        }
    };
    wt_float16 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.0f;
    wt_int16 magic;
#pragma unroll
    for (int i = 0; i < 16; ++i) magic[i] = kMagicBits;
    asm volatile("" : "+v"(magic));  // (kept, not made again before each use)
    wt_uint4 q[D][NT][2];
    wt_uint2 d4[D][NT];
    auto load_units = [&](int j, int c) {
        const uint32_t at = (uint32_t) c * (uint32_t) kUnitBytes;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                q[j][n][u] = *reinterpret_cast<const wt_uint4 *>(w[n] + (u * tile_bytes + at) + lane * 16);
            d4[j][n] = *reinterpret_cast<const wt_uint2 *>(w[n] + at + scales_at);
        }
    };
    // Step s takes unit s * KW + kw.  Its weights lie in slot s % D, read after
    // step s - D's were used; its rows' codes are read once those of the step
    // before are in LDS.
    const int steps = (last + KW) / KW;
    auto unit_of = [&](int step) { return min(step * KW + kw, last); };
    load_x(unit_of(0));
#pragma unroll
    for (int j = 0; j < D; ++j) load_units(j, unit_of(j));
    for (int step0 = 0; step0 < steps; step0 += D) {
#pragma unroll
        for (int j = 0; j < D; ++j) {
            const int step = step0 + j, at = ALONE ? 0 : step & 1;
            if (step >= steps || (ALONE && step * KW + kw > last)) break;
            if (ALONE) __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses stay in order)
            put_x(at, unit_of(step));
            if (ALONE)
                __builtin_amdgcn_wave_barrier();
            else
                lds_barrier();
            load_x(unit_of(step + 1));
            if (ALONE || KW == 1 || step * KW + kw <= last) {  // (else a unit that another wave has)
#pragma unroll
                for (int n = 0; n < NT; ++n) pair_units(q[j][n][0], q[j][n][1]);
                // What a block of rows needs of LDS is read while the one before
                // it is multiplied.
                constexpr int TILES = 4 * MT * NT;  // of a unit: block e / MT, rows e % MT, outputs n
                wt_int4 xv[2], wv[NT];
                rw_float4 d8[2][4];
                float ds[2][NT], off[2][NT];
                wt_float16 f[2];
                auto read_rows = [&](int e) {
                    const int t = e / MT, m = e % MT;
                    xv[e & 1] = s_x[kw][at][32 * m + l32][(2 * t + h) ^ (l32 & 7)];
                    const rw_float4 *src = reinterpret_cast<const rw_float4 *>(s_d8[kw][at][m][t][h]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) d8[e & 1][i] = src[i];
                };
                auto unpack = [&](int t) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint32_t a = q[j][n][0][t], b = q[j][n][1][t];
                        wv[n] = wt_int4{(int) (a << 4 & 0xF0F0F0F0u), (int) (a & 0xF0F0F0F0u), (int) (b << 4 & 0xF0F0F0F0u),
                                        (int) (b & 0xF0F0F0F0u)};
                        float &d = ds[t & 1][n];
                        d = t & 1 ? half_hi(d4[j][n][t >> 1]) : half_lo(d4[j][n][t >> 1]);
                        asm volatile("" : "+v"(d));  // (in fp32: an fma that widens an operand takes twice the time)
                        off[t & 1][n] = -kMagic * d;
                    }
                };
                auto multiply = [&](int i) {
                    const int e = i / NT;
                    if (i % (NT * MT) == 0) unpack(e / MT);
                    f[i & 1] = __builtin_bit_cast(
                        wt_float16, __builtin_amdgcn_mfma_i32_32x32x32_i8(xv[e & 1], wv[i % NT], magic, 0, 0, 0));
                };
                read_rows(0);
                if (AHEAD) multiply(0);
#pragma unroll
                for (int i = 0; i < TILES; ++i) {
                    const int e = i / NT, t = e / MT, m = e % MT, n = i % NT;
                    if (n == 0 && e + 1 < 4 * MT) read_rows(e + 1);
                    if (!AHEAD)
                        multiply(i);
                    else if (i + 1 < TILES)
                        multiply(i + 1);
                    if (AHEAD) __builtin_amdgcn_sched_barrier(0);  // (else the compiler moves it down to its fmas)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        acc[n][m][r] = __builtin_fmaf(d8[e & 1][r >> 2][r & 3],
                                                      __builtin_fmaf(f[i & 1][r], ds[t & 1][n], off[t & 1][n]), acc[n][m][r]);
                    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
                }
            }
            load_units(j, unit_of(step + D));
        }
    }
    // The waves of a piece add up in the order of their units, each the PART
    // results from kw * PART on, which it stores.
    constexpr int PART = 16 / KW;
    float sum[NT][MT][PART];
    if constexpr (KW > 1) {
        __shared__ float s_acc[WAVES][16 / PART][64][PART];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                __syncthreads();
#pragma unroll
                for (int r = 0; r < 16; ++r) s_acc[wave][r / PART][lane][r % PART] = acc[n][m][r];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < PART; ++i) sum[n][m][i] = s_acc[wave - kw][kw][lane][i];
#pragma unroll
                for (int k = 1; k < KW; ++k)
#pragma unroll
                    for (int i = 0; i < PART; ++i) sum[n][m][i] += s_acc[wave - kw + k][kw][lane][i];
            }
    } else {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[n][m][i] = acc[n][m][i];
    }
    if (piece >= n_pieces) return;
    const int row0 = first + 4 * h;
    // A lane's row of result i, from row0 on.
    auto below = [&](int m, int i) {
        const int r = kw * PART + i;
        return m * 32 + 8 * (r >> 2) + (r & 3);
    };
    if constexpr (GATED) {
        const int n_out = p.g.rows / 2, col = piece * 32 + l32;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < PART; ++i)
                sum[0][m][i] = gate(sum[0][m][i] * kCodeStep, sum[1][m][i] * kCodeStep, p.activation);
        if (p.out) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < PART; ++i)
                    if (row0 + below(m, i) < p.n_rows)
                        store1(p.out, (row0 + (int64_t) below(m, i)) * p.out_stride + col, sum[0][m][i], p.type);
        }
        if (!p.out_codes) return;
        // (no branch between the rows, so that their chains of instructions overlap)
        int8_t *codes_at = p.out_codes + row0 * (int64_t) n_out + col;
        uint16_t *scales8 = p.out_scales + (row0 * (int64_t) (n_out / 32) + piece);
        auto quantize = [&](auto real) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                uint32_t bits[PART];
#pragma unroll
                for (int i = 0; i < PART; ++i) {
                    const Scale8 s = scale_of(half_max(__builtin_fabsf(sum[0][m][i])));
                    const int code = code1(sum[0][m][i], s.inv), dr = below(m, i);
                    bits[i] = s.bits;
                    if (real(dr)) codes_at[(int64_t) dr * n_out] = (int8_t) code;
                }
                // (lane i of a half stores the scale of its row i)
                uint32_t mine = bits[0];
                int dr = below(m, 0);
#pragma unroll
                for (int i = 1; i < PART; ++i) {
                    mine = l32 == i ? bits[i] : mine;
                    dr = l32 == i ? below(m, i) : dr;
                }
                if (l32 < PART && real(dr)) scales8[(int64_t) dr * (n_out / 32)] = (uint16_t) mine;
            }
        };
        if (first + ROWS <= p.n_rows)
            quantize([](int) { return true; });
        else
            quantize([&](int dr) { return row0 + dr < p.n_rows; });
    } else {
        // Results i and i + 1 are two rows of a column.  Neighbouring lanes change
        // halves of their 16-bit pairs, so that each stores two columns of one row.
        auto each = [&](auto store) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int i = 0; i < PART; i += 2)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        store(below(m, i), n * 32, sum[n][m][i] * kCodeStep, sum[n][m][i + 1] * kCodeStep);
        };
        const int col = NT * piece * 32 + l32;
        const bool whole = first + ROWS <= p.n_rows && NT * (piece + 1) * 32 <= p.g.rows;
        const bool pairs = (p.out_stride & 1) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0;
        if (whole && p.type == kTypeF32) {
            float *out = static_cast<float *>(p.out) + row0 * p.out_stride + col;
            each([&](int dr, int dc, float a, float b) {
                float *at = out + dr * p.out_stride + dc;
                at[0] = a;
                at[p.out_stride] = b;
            });
        } else if (whole && pairs) {
            const bool odd = lane & 1;
            uint16_t *out = static_cast<uint16_t *>(p.out) + (row0 + odd) * p.out_stride + (col - odd);
            const uint32_t take = odd ? 0x07060302u : 0x01000504u;  // bytes of (own, other): their high halves or low ones
            auto put = [&](int dr, int dc, uint32_t a, uint32_t b) {
                const uint32_t own = a | b << 16, other = (uint32_t) __builtin_amdgcn_mov_dpp((int) own, 0xB1, 0xF, 0xF, true);
                *reinterpret_cast<uint32_t *>(out + (dr * p.out_stride + dc)) = __builtin_amdgcn_perm(own, other, take);
            };
            if (p.type == kTypeF16)
                each([&](int dr, int dc, float a, float b) { put(dr, dc, f32_to_f16_bits(a), f32_to_f16_bits(b)); });
            else
                each([&](int dr, int dc, float a, float b) { put(dr, dc, bf16_bits(a), bf16_bits(b)); });
        } else {
            each([&](int dr, int dc, float a, float b) {
                if (col + dc >= p.g.rows) return;
                const int64_t at = (row0 + (int64_t) dr) * p.out_stride + col + dc;
                if (row0 + dr < p.n_rows) store1(p.out, at, a, p.type);
                if (row0 + dr + 1 < p.n_rows) store1(p.out, at + p.out_stride, b, p.type);
            });
        }
    }
}

template <int SHAPE, int WN, int D, bool AHEAD, bool GATED>
hipError_t run_many(const ProductParams &p, hipStream_t stream) {
    constexpr ProductShape S = GATED ? kGatedShapes[SHAPE] : kProductShapes[SHAPE];
    constexpr int MT = S.rows / 32, NT = GATED ? 2 : S.outs / (32 * WN), PIECE = GATED ? 32 : 32 * NT;
    static_assert(S.outs == PIECE * WN && S.rows == 32 * MT, "the shape's sizes");
    ProductParams q = p;
    int pieces = ((GATED ? p.g.rows / 2 : p.g.rows) + PIECE - 1) / PIECE;
    const unsigned columns = (unsigned) ((pieces + WN - 1) / WN);
    Places places = make_places(columns);
    void *args[] = {&q, &pieces, &places};
    return hipLaunchKernel(reinterpret_cast<const void *>(many_rows_kernel<MT, NT, WN, S.waves, D, AHEAD, GATED>),
                           dim3(columns, (unsigned) ((p.n_rows + S.rows - 1) / S.rows)),
                           dim3(64 * WN * S.waves), args, 0, stream);
}

}  // namespace

hipError_t launch_product(const ProductParams &p, hipStream_t stream) {
    if (p.n_rows == 1 && p.g.chunks <= kOneRowChunks) {
        if (p.activation) return run_one<4, 8, 1, true>(p, stream);
        // Rows past 4096 columns with no more tiles than CUs: 16 waves to a tile (4096 x
        // 5632 4.8 against 5.2 us, 4096 x 11264 6.8 against 7.8, 2048 x 8192 4.8 against
        // 5.5; else 8: 12288 x 4096 6.7 against 8.2, 5120 x 5120 5.5 against 5.7).
        return p.g.tiles <= 256 && p.g.chunks > 32 ? run_one<1, 16, 2, false>(p, stream) : run_one<1, 8, 2, false>(p, stream);
    }
    if (p.activation) {
        switch (product_shape(true, p.n_rows, p.g.rows / 2, p.g.chunks)) {
        case 0: return run_few<0, 1, true>(p, stream);
        case 1: return run_many<1, 1, 1, false, true>(p, stream);
        case 2: return run_many<2, 1, 1, false, true>(p, stream);
        case 3: return run_many<3, 2, 2, false, true>(p, stream);
        case 4: return run_many<4, 4, 1, false, true>(p, stream);
        case 5: return run_many<5, 2, 1, true, true>(p, stream);
        default: return run_many<6, 4, 1, true, true>(p, stream);
        }
    }
    switch (product_shape(false, p.n_rows, p.g.rows, p.g.chunks)) {
    case 0: return run_few<0, 2, false>(p, stream);
    case 1: return run_few<1, 1, false>(p, stream);
    case 2: return run_few<2, 1, false>(p, stream);
    case 3: return run_many<3, 1, 2, false, false>(p, stream);
    case 4: return run_many<4, 1, 2, false, false>(p, stream);
    case 5: return run_many<5, 1, 1, false, false>(p, stream);
    case 6: return run_many<6, 4, 2, false, false>(p, stream);
    case 7: return run_many<7, 4, 1, false, false>(p, stream);
    case 8: return run_many<8, 2, 1, true, false>(p, stream);
    default: return run_many<9, 4, 2, false, false>(p, stream);
    }
}

hipError_t launch_weights_pack(const PackParams &p, hipStream_t stream) {
    PackParams q = p;
    FastDiv div = make_fastdiv((uint32_t) p.g.cols / 32);
    uint32_t n = (uint32_t) p.n_rows * (uint32_t) (p.g.cols / 32);
    void *args[] = {&q, &div, &n};
    return hipLaunchKernel(reinterpret_cast<const void *>(pack_kernel), dim3((n + 255) / 256), dim3(256), args, 0, stream);
}

}  // namespace bmo
