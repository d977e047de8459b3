// rows_device.hpp -- what the operators on rows share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pages_device.hpp"
#include "rows.hpp"

namespace bmo {

typedef float rw_float4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t bf16_bits(float x) {
    const __bf16 h = (__bf16) x;
    return __builtin_bit_cast(uint16_t, h);
}

// Eight elements as they lie in memory; the second 16 bytes are fp32's.
struct Raw8 {
    uint4 a, b;
};
__device__ __forceinline__ Raw8 load_raw8(const void *p, int64_t i, int type) {
    const uint8_t *src = static_cast<const uint8_t *>(p) + i * type_bytes(type);
    Raw8 r;
    r.a = *reinterpret_cast<const uint4 *>(src);
    r.b = r.a;
    if (type == kTypeF32) r.b = *reinterpret_cast<const uint4 *>(src + 16);
    return r;
}
__device__ __forceinline__ void widen8(const Raw8 &r, int type, float (&x)[8]) {
    const uint32_t u[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (type == kTypeF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_bit_cast(float, u[j]);
    } else if (type == kTypeF16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = f16_bits_to_f32(j & 1 ? u[j >> 1] >> 16 : u[j >> 1] & 0xFFFFu);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __builtin_bit_cast(float, j & 1 ? u[j >> 1] & 0xFFFF0000u : u[j >> 1] << 16);
    }
}
// Rounds x to the type, as its stored value reads.
__device__ __forceinline__ float round_to(float x, int type) {
    if (type == kTypeF16) return f16_bits_to_f32(f32_to_f16_bits(x));
    if (type == kTypeBF16) return __builtin_bit_cast(float, bf16_bits(x) << 16);
    return x;
}
__device__ __forceinline__ void store8(void *p, int64_t i, const float (&x)[8], int type) {
    if (type == kTypeF32) {
        rw_float4 *dst = reinterpret_cast<rw_float4 *>(static_cast<float *>(p) + i);
        dst[0] = rw_float4{x[0], x[1], x[2], x[3]};
        dst[1] = rw_float4{x[4], x[5], x[6], x[7]};
        return;
    }
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        u[j] = type == kTypeF16 ? f32_to_f16_bits(x[2 * j]) | ((uint32_t) f32_to_f16_bits(x[2 * j + 1]) << 16)
                                : bf16_bits(x[2 * j]) | (bf16_bits(x[2 * j + 1]) << 16);
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = make_uint4(u[0], u[1], u[2], u[3]);
}

// The scale of a block whose largest magnitude is amax: the least fp16 that is
// not below amax / 127, so that no code passes 127.  NaN where that is none (a
// NaN or an infinity in the block, magnitudes past 127 * 65504), with codes 0.
struct Scale8 {
    uint32_t bits;
    float inv;  // 1 / scale, 0 for codes that are 0
};
__device__ __forceinline__ Scale8 scale_of(float amax) {
    // (rounded to fp16 that is the scale or the one before it: of a value that has
    // moved by half a step of fp32 too)
    uint32_t h = f32_to_f16_bits(amax * (1.0f / 127.0f));
    if (f16_bits_to_f32(h) * 127.0f < amax) ++h;  // (18 bits, exact: also where the product was rounded, or is 0)
    if (!(amax <= 127.0f * 65504.0f)) return {0x7E00u, 0.0f};
    const float d = f16_bits_to_f32(h);
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);  // (a scale is normal in fp32)
    return {h, h ? r : 0.0f};
}
// The integer nearest to x * inv (codes of a block whose scale is NaN are 0
// whatever it holds), and four as bytes.
__device__ __forceinline__ int code1(float x, float inv) { return inv != 0.0f ? (int) __builtin_rintf(x * inv) : 0; }
__device__ __forceinline__ uint32_t codes4(const float *x, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= ((uint32_t) code1(x[j], inv) & 0xFFu) << (8 * j);
    return w;
}
__device__ __forceinline__ float max_abs8(const float (&x)[8]) {
    float m = __builtin_fabsf(x[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = __builtin_elementwise_maximum(m, __builtin_fabsf(x[j]));  // NaN if any is
    return m;
}
// The largest of a quad's lanes.
__device__ __forceinline__ float quad_max(float v) {
    v = __builtin_elementwise_maximum(v, pg_dpp<0xB1>(v));
    return __builtin_elementwise_maximum(v, pg_dpp<0x4E>(v));
}

// The largest of a row's 16 lanes.
__device__ __forceinline__ float row16_max(float v) {
    v = quad_max(v);
    v = __builtin_elementwise_maximum(v, pg_dpp<0x124>(v));         // row_ror:4
    return __builtin_elementwise_maximum(v, pg_dpp<0x128>(v));      // row_ror:8
}

// The largest of a half's 32 lanes.  (Rows 0 and 2 of one register change places
// with rows 1 and 3 of the other.  Wait states: the compiler's hazard pass does
// not see inside.)
__device__ __forceinline__ float half_max(float v) {
    float a = row16_max(v), b = a;
    asm volatile("s_nop 3\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 3" : "+v"(a), "+v"(b));
    return __builtin_elementwise_maximum(a, b);
}

}  // namespace bmo
