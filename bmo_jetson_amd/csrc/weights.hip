// weights.hip -- 8-bit rows times Q4_0 weights on the matrix cores, plain and
// gated.
//
//   y[m][n] = sum over blocks b of d4[n][b] d8[m][b] sum_j (c_j - 8) q_j
//
// A block's sum is an exact integer: v_mfma_i32 over its 32 elements, the
// weights (16 (code - 8), one shift and mask from their nibbles) as the rows
// and the 8-bit rows as the columns of the result.  It starts from the integer
// whose bits are the float 1.5 * 2^23, so that the result's bits, read as a
// float, are that plus the sum, exactly (sums stay below 2^20), and one fma
// with d8 takes the offset out again: -1.5 * 2^23 * d8 is exact for an fp16
// d8.  A second one adds d4 times that, so an output is off by the roundings
// of an fp32 sum of its blocks' parts only.
#include "kernels.hpp"
#include "rows_device.hpp"

namespace bmo {

namespace {

typedef int wt_int4 __attribute__((ext_vector_type(4)));
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
    reinterpret_cast<uint16_t *>(unit + kUnitScales)[((ri / 4) * 4 + t) * 4 + ri % 4] = src[0];
}

__device__ __forceinline__ float half_lo(uint32_t u) { return f16_bits_to_f32(u & 0xFFFFu); }
__device__ __forceinline__ float half_hi(uint32_t u) { return f16_bits_to_f32(u >> 16); }

// The activation of a gate times what it lets through.
__device__ __forceinline__ float gate(float g, float u, int activation) {
    // GELU by its tanh form: 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
    const float a = activation == kSilu ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
    return g / (1.0f + expf(-a)) * u;
}

// Outputs n .. n + 3 of row m.
__device__ __forceinline__ void store_quad(const ProductParams &p, int64_t m, int n, int n_out, rw_float4 v) {
    const int64_t at = m * p.out_stride + n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < n_out) store1(p.out, at + j, v[j], p.type);
}

// Few rows: a workgroup takes 16 * MT rows and NT tiles of 16 outputs, its KW
// waves every KW-th unit of the tiles; their sums are joined in LDS, wave after
// wave.
template <int MT, int NT, int KW, bool GATED>
__global__ __launch_bounds__(64 * KW) void few_rows_kernel(ProductParams p) {
    static_assert(!GATED || NT == 4, "two tiles of gates and the two that they let through");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i16 = lane & 15, g = lane >> 4;
    const int m0 = blockIdx.y * 16 * MT;
    const int nb = p.g.cols / 32;
    const uint8_t *w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        int tile = GATED ? (int) blockIdx.x * 2 + (n & 1) + (n & 2 ? p.g.tiles / 2 : 0) : (int) blockIdx.x * NT + n;
        tile = min(tile, p.g.tiles - 1);
        w[n] = p.w + (int64_t) tile * p.g.chunks * kUnitBytes;
    }
    const int8_t *x[MT];
    const uint16_t *d[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = min(m0 + 16 * m + i16, p.n_rows - 1);
        x[m] = p.codes + (int64_t) row * p.g.cols;
        d[m] = p.scales + (int64_t) row * nb;
    }
    rw_float4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = rw_float4{0, 0, 0, 0};
    const wt_int4 magic = {kMagicBits, kMagicBits, kMagicBits, kMagicBits};
    for (int c = wave; c < p.g.chunks; c += KW) {
        uint4 q[NT], s0[NT], s1[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint8_t *u = w[n] + (int64_t) c * kUnitBytes;
            q[n] = *reinterpret_cast<const uint4 *>(u + lane * 16);
            s0[n] = *reinterpret_cast<const uint4 *>(u + kUnitScales + g * 32);
            s1[n] = *reinterpret_cast<const uint4 *>(u + kUnitScales + g * 32 + 16);
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int b = min(4 * c + t, nb - 1);  // (past the last: weights are zeros)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const long xa = *reinterpret_cast<const long *>(x[m] + b * 32 + g * 8);
                const float d8 = f16_bits_to_f32(d[m][b]), off = -kMagic * d8;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t v = (&q[n].x)[t];
                    const uint2 wv = make_uint2(v << 4 & 0xF0F0F0F0u, v & 0xF0F0F0F0u);
                    const wt_int4 z =
                        __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, wv), xa, magic, 0, 0, 0);
                    const rw_float4 f = __builtin_bit_cast(rw_float4, z);
                    const uint32_t sc[2] = {(&(t < 2 ? s0[n] : s1[n]).x)[2 * (t & 1)],
                                            (&(t < 2 ? s0[n] : s1[n]).x)[2 * (t & 1) + 1]};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float part = __builtin_fmaf(f[r], d8, off);
                        acc[m][n][r] = __builtin_fmaf(r & 1 ? half_hi(sc[r >> 1]) : half_lo(sc[r >> 1]), part, acc[m][n][r]);
                    }
                }
            }
        }
    }
    __shared__ rw_float4 s_acc[KW][MT][NT][64];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) s_acc[wave][m][n][lane] = acc[m][n];
    __syncthreads();
    auto joined = [&](int m, int n) {
        rw_float4 v = s_acc[0][m][n][lane];
        for (int k = 1; k < KW; ++k) v += s_acc[k][m][n][lane];
        return v * kCodeStep;
    };
    if constexpr (GATED) {
        const int n_out = p.g.rows / 2;
        for (int m = wave; m < MT; m += KW) {
            const int64_t row = m0 + 16 * m + i16;
            float h[8];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const rw_float4 a = joined(m, n), b = joined(m, n + 2);
#pragma unroll
                for (int r = 0; r < 4; ++r) h[4 * n + r] = gate(a[r], b[r], p.activation);
            }
            const int n0 = (int) blockIdx.x * 32 + 4 * g;
            if (p.out && row < p.n_rows) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    store_quad(p, row, n0 + 16 * n, n_out, rw_float4{h[4 * n], h[4 * n + 1], h[4 * n + 2], h[4 * n + 3]});
            }
            if (p.out_codes) {
                float amax = max_abs8(h);
                amax = __builtin_elementwise_maximum(amax, __shfl_xor(amax, 16));
                amax = __builtin_elementwise_maximum(amax, __shfl_xor(amax, 32));
                const Scale8 s = scale_of(amax);
                if (row < p.n_rows) {
                    uint32_t *dst = reinterpret_cast<uint32_t *>(p.out_codes + row * n_out + n0);
                    dst[0] = codes4(h, s.inv);
                    dst[4] = codes4(h + 4, s.inv);
                    if (g == 0) p.out_scales[row * (n_out / 32) + blockIdx.x] = (uint16_t) s.bits;
                }
            }
        }
    } else {
        for (int i = wave; i < MT * NT; i += KW) {
            const int m = i / NT, n = i % NT;
            const int64_t row = m0 + 16 * m + i16;
            const rw_float4 v = joined(m, n);
            if (row < p.n_rows) store_quad(p, row, ((int) blockIdx.x * NT + n) * 16 + 4 * g, p.g.rows, v);
        }
    }
}

template <int MT, int NT, int KW, bool GATED>
hipError_t run_few(const ProductParams &p, hipStream_t stream) {
    ProductParams q = p;
    void *args[] = {&q};
    const int per = GATED ? 2 : NT, tiles = GATED ? p.g.tiles / 2 : p.g.tiles;
    return hipLaunchKernel(reinterpret_cast<const void *>(few_rows_kernel<MT, NT, KW, GATED>),
                           dim3((unsigned) ((tiles + per - 1) / per), (unsigned) ((p.n_rows + 16 * MT - 1) / (16 * MT))),
                           dim3(64 * KW), args, 0, stream);
}

// Many rows: a wave takes 64 rows and two tiles of 32 outputs (of a gated
// product one of gates and the one that they let through), a workgroup's waves
// WM x WN such pieces, or KW waves share one and take every KW-th unit of it.
constexpr int kManyThreads = 256;

// Two units' codes of 16 rows each to a 32-row operand: lanes 16 to 31 and 48
// to 63 of the first change places with lanes 0 to 15 and 32 to 47 of the
// second.  (Wait states before the first: the compiler's hazard pass does not
// see inside.)
__device__ __forceinline__ void pair_rows(uint4 &a, uint4 &b) {
    asm volatile(
        "s_nop 3\n"
        "v_permlane16_swap_b32 %0, %4\n"
        "v_permlane16_swap_b32 %1, %5\n"
        "v_permlane16_swap_b32 %2, %6\n"
        "v_permlane16_swap_b32 %3, %7\n"
        "s_nop 3"
        : "+v"(a.x), "+v"(a.y), "+v"(a.z), "+v"(a.w), "+v"(b.x), "+v"(b.y), "+v"(b.z), "+v"(b.w));
}

__device__ __forceinline__ uint32_t dword(const uint4 &v, int t) { return t == 0 ? v.x : t == 1 ? v.y : t == 2 ? v.z : v.w; }

template <int KW, bool GATED, bool EVEN>
__global__ __launch_bounds__(kManyThreads, 2) void many_rows_kernel(ProductParams p, int n_pairs) {
    constexpr int WN = KW == 4 ? 1 : 2, WM = 4 / KW / WN, MT = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int kw = wave % KW, wn = wave / KW % WN, wm = wave / KW / WN;
    const int m32 = lane & 31, h = lane >> 5;
    const int m0 = ((int) blockIdx.y * WM + wm) * 32 * MT;
    const int pair = (int) blockIdx.x * WN + wn;
    const int nb = p.g.cols / 32;
    // (tiles of 32 rows; a pair past the last reads the last and stores nothing)
    auto unit = [&](int n, int u) {
        const int tile = GATED ? pair + n * (p.g.tiles / 4) : 2 * pair + n;
        return p.w + (int64_t) min(2 * tile + u, p.g.tiles - 1) * p.g.chunks * kUnitBytes;
    };
    const uint8_t *w[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) w[n][u] = unit(n, u) + lane * 16;
    // A lane carries the scales of four rows in one block: tile lane / 32, unit
    // lane / 16 % 2, rows 4g .., g = lane / 4 % 4, block t = lane % 4.
    const uint8_t *ws = unit(lane >> 5, (lane >> 4) & 1) + kUnitScales + (lane & 15) * 8;
    __shared__ uint4 s_scale[4][2][4][2][2];  // [wave][tile][block][half][32 bytes]
    uint2 *scale_to = reinterpret_cast<uint2 *>(s_scale[wave]) + (lane >> 5) * 32 + (lane & 3) * 8 + ((lane >> 2) & 1) * 4 +
                      ((lane >> 4) & 1) * 2 + ((lane >> 3) & 1);
    const int8_t *x[MT];
    const uint16_t *d[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = min(m0 + 32 * m + m32, p.n_rows - 1);
        x[m] = p.codes + (int64_t) row * p.g.cols + h * 16;
        d[m] = p.scales + (int64_t) row * nb;
    }
    auto load_x = [&](int m, int c, int t) {  // (past the last block: weights are zeros)
        return *reinterpret_cast<const wt_int4 *>(x[m] + min(4 * c + t, nb - 1) * 32);
    };
    auto load_d = [&](int m, int c) {
        if constexpr (EVEN) return *reinterpret_cast<const uint2 *>(d[m] + 4 * c);
        uint32_t v[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = d[m][min(4 * c + t, nb - 1)];
        return make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
    };
    wt_float16 acc[2][MT];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.0f;
    wt_int16 magic;
#pragma unroll
    for (int i = 0; i < 16; ++i) magic[i] = kMagicBits;
    const int last = p.g.chunks - 1;
    int c = min(kw, last);
    uint4 q[2][2], q1[2][2];
    uint2 sc, sc1, dd[MT], dd1[MT];
    wt_int4 xv[4][MT];
    auto load_chunk = [&](int at, uint4 (&qq)[2][2], uint2 &s, uint2 (&e)[MT]) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) qq[n][u] = *reinterpret_cast<const uint4 *>(w[n][u] + (int64_t) at * kUnitBytes);
        s = *reinterpret_cast<const uint2 *>(ws + (int64_t) at * kUnitBytes);
#pragma unroll
        for (int m = 0; m < MT; ++m) e[m] = load_d(m, at);
    };
    load_chunk(c, q, sc, dd);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) xv[t][m] = load_x(m, c, t);
    for (int k = kw; k <= last; k += KW) {
        const int next = min(k + KW, last);
        load_chunk(next, q1, sc1, dd1);
        *scale_to = sc;
#pragma unroll
        for (int n = 0; n < 2; ++n) pair_rows(q[n][0], q[n][1]);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float d8[MT], off[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint32_t v = t < 2 ? dd[m].x : dd[m].y;
                d8[m] = t & 1 ? half_hi(v) : half_lo(v);
                off[m] = -kMagic * d8[m];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint32_t a = dword(q[n][0], t), b = dword(q[n][1], t);
                const wt_int4 av = {(int) (a << 4 & 0xF0F0F0F0u), (int) (a & 0xF0F0F0F0u), (int) (b << 4 & 0xF0F0F0F0u),
                                    (int) (b & 0xF0F0F0F0u)};
                const uint4 s0 = s_scale[wave][n][t][h][0], s1 = s_scale[wave][n][t][h][1];
                const uint32_t sv[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const wt_float16 f = __builtin_bit_cast(
                        wt_float16, __builtin_amdgcn_mfma_i32_32x32x32_i8(av, xv[t][m], magic, 0, 0, 0));
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float part = __builtin_fmaf(f[i], d8[m], off[m]);
                        acc[n][m][i] = __builtin_fmaf(i & 1 ? half_hi(sv[i >> 1]) : half_lo(sv[i >> 1]), part, acc[n][m][i]);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) xv[t][m] = load_x(m, next, t);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) q[n][u] = q1[n][u];
        sc = sc1;
#pragma unroll
        for (int m = 0; m < MT; ++m) dd[m] = dd1[m];
    }
    if constexpr (KW > 1) {
        // the waves of a piece add up in the order of their units
        __shared__ rw_float4 s_acc[4][4][64];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    s_acc[wave][j][lane] = rw_float4{acc[n][m][4 * j], acc[n][m][4 * j + 1], acc[n][m][4 * j + 2],
                                                     acc[n][m][4 * j + 3]};
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    rw_float4 v = s_acc[wave - kw][j][lane];
#pragma unroll
                    for (int k = 1; k < KW; ++k) v += s_acc[wave - kw + k][j][lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[n][m][4 * j + r] = v[r];
                }
            }
    }
    if (pair >= n_pairs) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (KW > 1 && m % KW != kw) continue;  // each stores a part
        const int64_t row = m0 + 32 * m + m32;
        if constexpr (GATED) {
            const int n_out = p.g.rows / 2, n0 = pair * 32 + 4 * h;
            float v[16], amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = gate(acc[0][m][i] * kCodeStep, acc[1][m][i] * kCodeStep, p.activation);
                amax = __builtin_elementwise_maximum(amax, __builtin_fabsf(v[i]));
            }
            if (p.out && row < p.n_rows) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    store_quad(p, row, n0 + 8 * j, n_out, rw_float4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]});
            }
            if (p.out_codes) {
                const Scale8 s = scale_of(__builtin_elementwise_maximum(amax, __shfl_xor(amax, 32)));
                if (row < p.n_rows) {
                    uint32_t *dst = reinterpret_cast<uint32_t *>(p.out_codes + row * n_out + n0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) dst[2 * j] = codes4(v + 4 * j, s.inv);
                    if (h == 0) p.out_scales[row * (n_out / 32) + pair] = (uint16_t) s.bits;
                }
            }
        } else if (row < p.n_rows) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    store_quad(p, row, (2 * pair + n) * 32 + 8 * j + 4 * h, p.g.rows,
                               rw_float4{acc[n][m][4 * j], acc[n][m][4 * j + 1], acc[n][m][4 * j + 2], acc[n][m][4 * j + 3]} *
                                   kCodeStep);
        }
    }
}

template <int KW, bool GATED>
hipError_t run_many(const ProductParams &p, hipStream_t stream) {
    constexpr int WN = KW == 4 ? 1 : 2, WM = 4 / KW / WN;
    ProductParams q = p;
    int pairs = GATED ? p.g.rows / 64 : (p.g.rows + 63) / 64;
    void *args[] = {&q, &pairs};
    const bool even = p.g.cols % 128 == 0 && reinterpret_cast<uintptr_t>(p.scales) % 8 == 0;
    return hipLaunchKernel(even ? reinterpret_cast<const void *>(many_rows_kernel<KW, GATED, true>)
                                : reinterpret_cast<const void *>(many_rows_kernel<KW, GATED, false>),
                           dim3((unsigned) ((pairs + WN - 1) / WN), (unsigned) ((p.n_rows + 64 * WM - 1) / (64 * WM))),
                           dim3(kManyThreads), args, 0, stream);
}

}  // namespace

hipError_t launch_product(const ProductParams &p, hipStream_t stream) {
    if (p.n_rows > 64) {
        if (p.activation) return run_many<1, true>(p, stream);
        return run_many<1, false>(p, stream);
    }
    if (p.activation) return p.n_rows <= 16 ? run_few<1, 4, 8, true>(p, stream) : run_few<2, 4, 4, true>(p, stream);
    return p.n_rows <= 16 ? run_few<1, 1, 8, false>(p, stream) : run_few<4, 2, 4, false>(p, stream);
}

hipError_t launch_weights_pack(const PackParams &p, hipStream_t stream) {
    PackParams q = p;
    FastDiv div = make_fastdiv((uint32_t) p.g.cols / 32);
    uint32_t n = (uint32_t) p.n_rows * (uint32_t) (p.g.cols / 32);
    void *args[] = {&q, &div, &n};
    return hipLaunchKernel(reinterpret_cast<const void *>(pack_kernel), dim3((n + 255) / 256), dim3(256), args, 0, stream);
}

}  // namespace bmo
