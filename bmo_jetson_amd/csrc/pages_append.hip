// pages_append.hip -- rows of K and V into the paged cache's slots, and back.
//
// Four lanes move one 32-element block, lane c its bytes 4c .. 4c+3, elements
// 4c .. and 16 + 4c ..: rows are read and written in runs of 32 or 64 bytes,
// and the block's maximum is two steps within a quad.  append quantizes fp32,
// fp16 or bf16 bit-exactly or takes 18 bytes of ggml Q4_0, and spreads the
// bytes over the slot's group (pages_layout.hpp); gather does the reverse.  A
// wave takes 16 / NB consecutive tokens of one kv head, K and V together (two
// loads under way behind that of the slot).  Rows whose slot is out of range
// are skipped (gathered: zeros).
//
// Bound by latency (slot, then row, then the code's own fetch) for a token
// each, by HBM and the quantizer's instructions for prompts: in 32 heads of
// 128, 48 fp32 rows append in 3.1 us and gather in 2.8; six prompts, 5600 bf16
// rows of 8 heads, append in 10 us (30 MB; a copy of them takes 6) and gather
// as fp32 in 10 (52 MB, a copy 11).  One lane a block: 5.0, 4.6, 9.5 and 22.
#include <type_traits>

#include "kernels.hpp"
#include "pages.hpp"
#include "q4_0_device.hpp"

namespace bmo {

namespace {

constexpr int kSlotThreads = 256;
constexpr int kLanes = 4;  // a block

struct SlotsArgs {
    SlotsParams p;
    FastDiv div_kv;
};

typedef float sl_float4 __attribute__((ext_vector_type(4)));

// Four values from src, as fp32.
template <int TYPE>
__device__ __forceinline__ void load_quad(const uint8_t *src, float *x) {
    if constexpr (TYPE == kTypeF32) {
        const sl_float4 v = *reinterpret_cast<const sl_float4 *>(src);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = v[j];
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(src);
        const uint32_t w[2] = {u.x, u.y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t h = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
            x[j] = TYPE == kTypeF16 ? f16_bits_to_f32(h) : __builtin_bit_cast(float, h << 16);
        }
    }
}

__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 r = {(__bf16) a, (__bf16) b};
    return __builtin_bit_cast(uint32_t, r);
}

template <int TYPE>
__device__ __forceinline__ void store_quad(uint8_t *dst, const float *x) {
    if constexpr (TYPE == kTypeF32) {
        *reinterpret_cast<sl_float4 *>(dst) = sl_float4{x[0], x[1], x[2], x[3]};
    } else {
        uint32_t w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            w[j] = TYPE == kTypeF16 ? f32_to_f16_bits(x[2 * j]) | ((uint32_t) f32_to_f16_bits(x[2 * j + 1]) << 16)
                                    : bf16_pair(x[2 * j], x[2 * j + 1]);
        *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    }
}

// The quantizer of a block's four lanes (quantize_block_q4_0_lanes), with the
// short path of the one-lane form: no NaN, no infinity, a scale whose
// reciprocal is finite and one sign at the largest magnitude.  The conditions
// are the quad's, so its lanes go the same way.
__device__ __forceinline__ uint32_t quantize_quad(const float (&x)[8], int c, uint16_t &d16) {
#pragma clang fp contract(off)
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
        hi = __builtin_elementwise_maximum(hi, x[j]);
        lo = __builtin_elementwise_minimum(lo, x[j]);
    }
    auto other = [](float v, auto ctrl) {
        return __builtin_bit_cast(float, dpp_u32<decltype(ctrl)::value>(__builtin_bit_cast(uint32_t, v)));
    };
    using X1 = std::integral_constant<int, 0xB1>;  // lane ^ 1, lane ^ 2
    using X2 = std::integral_constant<int, 0x4E>;
    hi = __builtin_elementwise_maximum(hi, other(hi, X1{}));
    lo = __builtin_elementwise_minimum(lo, other(lo, X1{}));
    hi = __builtin_elementwise_maximum(hi, other(hi, X2{}));
    lo = __builtin_elementwise_minimum(lo, other(lo, X2{}));
    const float amax = __builtin_elementwise_maximum(hi, -lo);  // NaN if any x is
    if (!(amax <= 3.40282347e38f && amax >= 0x1p-124f) || hi == -lo) return quantize_block_q4_0_lanes<kLanes>(x, c, d16);
    const float vmax = hi == amax ? amax : -amax;
    float d = vmax / -8.0f;
    asm volatile("" : "+v"(d));  // materialize d in fp32, as the other forms do
    const float id = 1.0f / d;
    d16 = f32_to_f16_bits(d);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c0 = min((int) (x[j] * id + 8.5f), 15), c1 = min((int) (x[4 + j] * id + 8.5f), 15);
        w |= ((uint32_t) c0 | ((uint32_t) c1 << 4)) << (8 * j);
    }
    return w;
}

// Which part of which block a lane moves.
struct Work {
    int tok, h, blk, c, slot;
    bool live;
};

template <int D>
__device__ __forceinline__ Work work_of(const SlotsArgs &a) {
    constexpr int NB = D / kQK;
    constexpr int TOK = 64 / (NB * kLanes);  // tokens of a wave
    // units: (token tile, kv head), heads fastest, one a wave (below 2^27)
    const uint32_t unit =
        __builtin_amdgcn_readfirstlane(blockIdx.x * (kSlotThreads / 64) + (threadIdx.x >> 6));
    const int lane = threadIdx.x & 63;
    Work w;
    const uint32_t tile = a.div_kv.div(unit);
    w.h = (int) (unit - tile * (uint32_t) a.p.g.n_kv);
    const int64_t tok = (int64_t) tile * TOK + lane / (NB * kLanes);
    w.blk = lane / kLanes % NB;
    w.c = lane % kLanes;
    w.live = tok < a.p.n_tok;
    w.tok = w.live ? (int) tok : 0;
    w.slot = w.live ? a.p.slots[w.tok] : -1;
    return w;
}

// Where a slot's block part and scales are: a dword of K, four bytes of V 16
// bytes apart.
template <int D>
struct Place {
    uint8_t *k, *v;
    uint16_t *kd, *vd;
    __device__ Place(const SlotsParams &p, const Work &w) {
        constexpr int NB = D / kQK, G = 2048 / D;
        const int s = w.slot & (G - 1), t = s >> 4, key = s & 15;
        const int tb = t * NB + w.blk;
        uint8_t *grp = p.base + p.g.group_offset(w.slot, w.h);
        k = grp + (w.c * 16 + key) * 16 + tb * 4;
        v = grp + kVCodeOff + ((key >> 2) * 16 + w.c * 4) * 16 + tb * 4 + (key & 3);
        kd = reinterpret_cast<uint16_t *>(grp + page_scale_offset(tb, key, 0));
        vd = reinterpret_cast<uint16_t *>(grp + page_scale_offset(tb, key, 1));
    }
};

}  // namespace

template <int D, int TYPE>
__global__ __launch_bounds__(kSlotThreads) void pages_append_kernel(SlotsArgs a) {
    constexpr int NB = D / kQK;
    const SlotsParams &p = a.p;
    const Work w = work_of<D>(a);
    // (the lanes of a quad have one token: all of them go on, or none)
    if (!w.live || w.slot < 0 || w.slot >= p.g.n_slots()) return;
    uint16_t d16[2];
    uint32_t qs[2];
    if constexpr (TYPE == kTypeQ4_0) {
        const int64_t at = (((int64_t) w.tok * p.g.n_kv + w.h) * NB + w.blk) * 9;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint16_t *src = static_cast<const uint16_t *>(i == 0 ? p.k : p.v) + at;
            d16[i] = src[0];
            qs[i] = src[1 + 2 * w.c] | ((uint32_t) src[2 + 2 * w.c] << 16);
        }
    } else {
        const int64_t at = (w.tok * p.stride + w.h * D + w.blk * kQK + w.c * 4) * type_bytes(TYPE);
        float x[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint8_t *src = static_cast<const uint8_t *>(i == 0 ? p.k : p.v) + at;
            load_quad<TYPE>(src, x[i]);
            load_quad<TYPE>(src + 16 * type_bytes(TYPE), x[i] + 4);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) qs[i] = quantize_quad(x[i], w.c, d16[i]);
    }
    const Place<D> q(p, w);
    *reinterpret_cast<uint32_t *>(q.k) = qs[0];
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i * 16] = (uint8_t) (qs[1] >> (8 * i));
    if (w.c == 0) {
        *q.kd = d16[0];
        *q.vd = d16[1];
    }
}

template <int D, int TYPE>
__global__ __launch_bounds__(kSlotThreads) void pages_gather_kernel(SlotsArgs a) {
    constexpr int NB = D / kQK;
    const SlotsParams &p = a.p;
    const Work w = work_of<D>(a);
    if (!w.live) return;
    uint32_t qs[2] = {0x88888888u, 0x88888888u};
    uint16_t d16[2] = {0, 0};
    if (w.slot >= 0 && w.slot < p.g.n_slots()) {
        const Place<D> q(p, w);
        d16[0] = *q.kd;
        d16[1] = *q.vd;
        qs[0] = *reinterpret_cast<const uint32_t *>(q.k);
        qs[1] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) qs[1] |= (uint32_t) q.v[i * 16] << (8 * i);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint8_t *rows = static_cast<uint8_t *>(i == 0 ? p.k : p.v);
        if constexpr (TYPE == kTypeQ4_0) {
            uint16_t *dst =
                reinterpret_cast<uint16_t *>(rows) + (((int64_t) w.tok * p.g.n_kv + w.h) * NB + w.blk) * 9;
            if (w.c == 0) dst[0] = d16[i];
            dst[1 + 2 * w.c] = (uint16_t) qs[i];
            dst[2 + 2 * w.c] = (uint16_t) (qs[i] >> 16);
        } else {
            const float d = f16_bits_to_f32(d16[i]);
            float x[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t byte = qs[i] >> (8 * j);
                x[j] = (float) ((int) (byte & 15u) - 8) * d;
                x[4 + j] = (float) ((int) ((byte >> 4) & 15u) - 8) * d;
            }
            uint8_t *dst = rows + (w.tok * p.stride + w.h * D + w.blk * kQK + w.c * 4) * type_bytes(TYPE);
            store_quad<TYPE>(dst, x);
            store_quad<TYPE>(dst + 16 * type_bytes(TYPE), x + 4);
        }
    }
}

// Zeroes whole 16-byte pieces (ggml's zero block in every slot).
__global__ __launch_bounds__(256) void pages_clear_kernel(uint4 *dst, int64_t n) {
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t) gridDim.x * 256)
        dst[i] = make_uint4(0, 0, 0, 0);
}

namespace {

template <int D>
const void *append_of(int type) {
    switch (type) {
    case kTypeF32: return reinterpret_cast<const void *>(pages_append_kernel<D, kTypeF32>);
    case kTypeF16: return reinterpret_cast<const void *>(pages_append_kernel<D, kTypeF16>);
    case kTypeBF16: return reinterpret_cast<const void *>(pages_append_kernel<D, kTypeBF16>);
    default: return reinterpret_cast<const void *>(pages_append_kernel<D, kTypeQ4_0>);
    }
}
template <int D>
const void *gather_of(int type) {
    switch (type) {
    case kTypeF32: return reinterpret_cast<const void *>(pages_gather_kernel<D, kTypeF32>);
    case kTypeF16: return reinterpret_cast<const void *>(pages_gather_kernel<D, kTypeF16>);
    case kTypeBF16: return reinterpret_cast<const void *>(pages_gather_kernel<D, kTypeBF16>);
    default: return reinterpret_cast<const void *>(pages_gather_kernel<D, kTypeQ4_0>);
    }
}

hipError_t launch_slots(const void *kernel, const SlotsParams &p, hipStream_t stream) {
    const int tok = 64 / (p.g.dim / kQK * kLanes);
    const int64_t units = (p.n_tok + (int64_t) tok - 1) / tok * p.g.n_kv;
    SlotsArgs arg{p, make_fastdiv((uint32_t) p.g.n_kv)};
    void *args[] = {&arg};
    return hipLaunchKernel(kernel, dim3((unsigned) ((units + 3) / 4)), dim3(kSlotThreads), args, 0, stream);
}

}  // namespace

hipError_t launch_pages_append(const SlotsParams &p, hipStream_t stream) {
    return launch_slots(p.g.dim == 128 ? append_of<128>(p.type) : append_of<64>(p.type), p, stream);
}
hipError_t launch_pages_gather(const SlotsParams &p, hipStream_t stream) {
    return launch_slots(p.g.dim == 128 ? gather_of<128>(p.type) : gather_of<64>(p.type), p, stream);
}

hipError_t launch_pages_clear(uint8_t *base, int64_t bytes, hipStream_t stream) {
    uint4 *dst = reinterpret_cast<uint4 *>(base);
    int64_t n = bytes / 16;
    void *args[] = {&dst, &n};
    const int64_t wgs = (n + 255) / 256;
    return hipLaunchKernel(reinterpret_cast<const void *>(pages_clear_kernel), dim3((unsigned) (wgs < 8192 ? wgs : 8192)),
                           dim3(256), args, 0, stream);
}

}  // namespace bmo
