// pages_device.hpp -- what the paged cache's attention kernels share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pages.hpp"
#include "q4_0_device.hpp"

namespace bmo {

typedef _Float16 pg_half2 __attribute__((ext_vector_type(2)));
typedef _Float16 pg_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 pg_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pg_float4 __attribute__((ext_vector_type(4)));

constexpr float kPagesLazy = 8.0f;       // lazy rescale threshold, log2 units
constexpr float kPagesFloor = -1.0e30f;  // running-max floor, finite

// Element of its block that slot r of octet c of a dequantized K dword holds
// (byte j of a block: element j low, j + 16 high; the masks pair bytes 0, 2
// and 1, 3).
__host__ __device__ constexpr int octet_elem(int c, int r) {
    return 4 * c + (r & 4 ? 16 : 0) + (r & 1 ? 2 : 0) + ((r >> 1) & 1);
}

// The codes of dword w (bytes 4c..4c+3 of a block) minus 8 as 8 fp16 values,
// exactly, in octet_elem order.  A low nibble n under the fp16 pattern 0x6400
// reads 1024 + n; a high nibble in place (16 n) under 0x5400 reads 64 + n.
__device__ __forceinline__ pg_half8 k_octet(uint32_t w) {
    const pg_half2 lo = {(_Float16) -1032.0f, (_Float16) -1032.0f};
    const pg_half2 hi = {(_Float16) -72.0f, (_Float16) -72.0f};
    const uint32_t y = w >> 8;
    const pg_half2 a = __builtin_bit_cast(pg_half2, (w & 0x000F000Fu) | 0x64006400u) + lo;
    const pg_half2 b = __builtin_bit_cast(pg_half2, (y & 0x000F000Fu) | 0x64006400u) + lo;
    const pg_half2 c = __builtin_bit_cast(pg_half2, (w & 0x00F000F0u) | 0x54005400u) + hi;
    const pg_half2 d = __builtin_bit_cast(pg_half2, (y & 0x00F000F0u) | 0x54005400u) + hi;
    return pg_half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Four 4-bit codes, one a byte, as bf16: the byte n (0..15) read as fp8 e4m3
// is n * 2^-9 (its subnormals run on into the first exponent), which the
// conversion scales back to n exactly.
__device__ __forceinline__ void v_quad(uint32_t nibbles, pg_bf16x2 &a, pg_bf16x2 &b) {
    a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(nibbles, 512.0f, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(nibbles, 512.0f, true);
}
// Eight keys' codes of one V column: nibbles of two tiles' dwords.
__device__ __forceinline__ pg_bf16x8 v_octet(uint32_t x0, uint32_t x1) {
    pg_bf16x2 a, b, c, d;
    v_quad(x0 & 0x0F0F0F0Fu, a, b);
    v_quad(x1 & 0x0F0F0F0Fu, c, d);
    return pg_bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

template <int CTRL>
__device__ __forceinline__ float pg_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// Inclusive prefix sum over the wave's lanes (modulo 2^32).
__device__ __forceinline__ int wave_prefix(int v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (lane >= d) v = (int) ((uint32_t) v + (uint32_t) o);
    }
    return v;
}

// Four elements at p (of type, 4-element aligned) as fp32.
__device__ __forceinline__ pg_float4 load4(const void *p, int64_t i, int type) {
    if (type == kTypeF32) return *reinterpret_cast<const pg_float4 *>(static_cast<const float *>(p) + i);
    const uint2 u = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
    if (type == kTypeF16)
        return pg_float4{f16_bits_to_f32(u.x & 0xFFFFu), f16_bits_to_f32(u.x >> 16), f16_bits_to_f32(u.y & 0xFFFFu),
                         f16_bits_to_f32(u.y >> 16)};
    return pg_float4{__builtin_bit_cast(float, u.x << 16), __builtin_bit_cast(float, u.x & 0xFFFF0000u),
                     __builtin_bit_cast(float, u.y << 16), __builtin_bit_cast(float, u.y & 0xFFFF0000u)};
}
__device__ __forceinline__ float load1(const void *p, int64_t i, int type) {
    if (type == kTypeF32) return static_cast<const float *>(p)[i];
    const uint32_t u = static_cast<const uint16_t *>(p)[i];
    return type == kTypeF16 ? f16_bits_to_f32(u) : __builtin_bit_cast(float, u << 16);
}
// One value of TYPE, rounded to nearest even.
__device__ __forceinline__ void store1(void *p, int64_t i, float x, int type) {
    if (type == kTypeF32) {
        static_cast<float *>(p)[i] = x;
    } else if (type == kTypeF16) {
        static_cast<uint16_t *>(p)[i] = f32_to_f16_bits(x);
    } else {
        const __bf16 h = (__bf16) x;
        static_cast<uint16_t *>(p)[i] = __builtin_bit_cast(uint16_t, h);
    }
}

}  // namespace bmo
