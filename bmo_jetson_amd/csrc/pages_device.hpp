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
typedef float pg_float4 __attribute__((ext_vector_type(4)));

constexpr float kPagesFloor = -1.0e30f;  // running-max floor, finite

// Element of its block that slot r of octet c of a dequantized K dword holds
// (byte j of a block: element j low, j + 16 high; the masks pair bytes 0, 2
// and 1, 3).
__host__ __device__ constexpr int octet_elem(int c, int r) {
    return 4 * c + (r & 4 ? 16 : 0) + (r & 1 ? 2 : 0) + ((r >> 1) & 1);
}

// Patterns under which a 4-bit code reads as fp16: a low nibble n under 0x6400
// is 1024 + n, a nibble in place (16 n) under 0x5400 is 64 + n.  Kept in vector
// registers, so that and-or is one instruction (it takes one scalar operand).
struct Patterns {
    uint32_t lo = 0x64006400u, hi = 0x54005400u;
    __device__ __forceinline__ Patterns() { asm volatile("" : "+v"(lo), "+v"(hi)); }
};
// Codes minus 8, exactly, of the low (high) nibbles of bytes 0 and 2 of x.
__device__ __forceinline__ pg_half2 codes_lo(uint32_t x, const Patterns &c) {
    const pg_half2 off = {(_Float16) -1032.0f, (_Float16) -1032.0f};
    return __builtin_bit_cast(pg_half2, (x & 0x000F000Fu) | c.lo) + off;
}
__device__ __forceinline__ pg_half2 codes_hi(uint32_t x, const Patterns &c) {
    const pg_half2 off = {(_Float16) -72.0f, (_Float16) -72.0f};
    return __builtin_bit_cast(pg_half2, (x & 0x00F000F0u) | c.hi) + off;
}

// The codes of dword w (bytes 4c..4c+3 of a block) minus 8 as 8 fp16 values
// in octet_elem order.
__device__ __forceinline__ pg_half8 k_octet(uint32_t w, const Patterns &p) {
    const uint32_t y = w >> 8;
    const pg_half2 a = codes_lo(w, p), b = codes_lo(y, p), c = codes_hi(w, p), d = codes_hi(y, p);
    return pg_half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// p[i] at a wave-uniform index through the scalar cache, for arrays that no
// kernel writes while the reading one runs (lengths, tables).
__device__ __forceinline__ int uniform_int(const int *p, int i) {
    return ((const __attribute__((address_space(4))) int *) p)[i];
}

// The length of entry b; 0 for one that a plan did not let grow: it asked for
// nothing (n_new) or was refused (status), each array nullable.
__device__ __forceinline__ int granted_len(const int *lens, const int *n_new, const int *status, int b) {
    // (an absent array is read as lens, so that no load waits for another)
    const int len = uniform_int(lens, b);
    const int asked = uniform_int(n_new ? n_new : lens, b), state = uniform_int(status ? status : lens, b);
    return (n_new && asked <= 0) || (status && state != 0) ? 0 : len;
}

// 16 bytes that a launch reads once.
__device__ __forceinline__ uint4 stream16(const uint8_t *p) {
    typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
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
    const bool f16 = type == kTypeF16;  // (both conversions, so that no branch waits for the load)
    pg_float4 v;
    v[0] = f16 ? f16_bits_to_f32(u.x & 0xFFFFu) : __builtin_bit_cast(float, u.x << 16);
    v[1] = f16 ? f16_bits_to_f32(u.x >> 16) : __builtin_bit_cast(float, u.x & 0xFFFF0000u);
    v[2] = f16 ? f16_bits_to_f32(u.y & 0xFFFFu) : __builtin_bit_cast(float, u.y << 16);
    v[3] = f16 ? f16_bits_to_f32(u.y >> 16) : __builtin_bit_cast(float, u.y & 0xFFFF0000u);
    return v;
}
__device__ __forceinline__ float load1(const void *p, int64_t i, int type) {
    if (type == kTypeF32) return static_cast<const float *>(p)[i];
    const uint32_t u = static_cast<const uint16_t *>(p)[i];
    const float h = f16_bits_to_f32(u), b = __builtin_bit_cast(float, u << 16);
    return type == kTypeF16 ? h : b;
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
