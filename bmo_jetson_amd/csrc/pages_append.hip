// pages_append.hip -- rows of K and V into the paged cache's slots, and back.
//
// One thread moves one 32-element block: append reads it (fp32, fp16 or
// bf16, or 18 bytes of ggml Q4_0), quantizes with the bit-exact quantizer and
// spreads its bytes over the slot's group (pages_layout.hpp); gather does the
// reverse.  A workgroup takes TOK consecutive tokens of one kv head, the lanes
// of a wave 64 / NB of them, so that for a prompt, whose slots run on, a
// wave's code dwords fill whole lines.  Rows whose slot is out of range are
// skipped (gathered: zeros), nothing else of them is read.
#include "pages.hpp"
#include "q4_0_device.hpp"

namespace bmo {

namespace {

constexpr int kSlotThreads = 256;

__device__ __forceinline__ float f16_lo(uint32_t v) { return f16_bits_to_f32(v & 0xFFFFu); }
__device__ __forceinline__ float f16_hi(uint32_t v) { return f16_bits_to_f32(v >> 16); }

// 32 elements from src (16-byte aligned) as fp32.
template <int TYPE>
__device__ __forceinline__ void load_block(const void *src, float (&x)[kQK]) {
    if constexpr (TYPE == kTypeF32) {
        load_block_f32(static_cast<const float *>(src), x);
    } else {
        const uint4 *s4 = static_cast<const uint4 *>(src);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint4 u = s4[c];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[8 * c + 2 * j] = TYPE == kTypeF16 ? f16_lo(w[j]) : __builtin_bit_cast(float, w[j] << 16);
                x[8 * c + 2 * j + 1] = TYPE == kTypeF16 ? f16_hi(w[j]) : __builtin_bit_cast(float, w[j] & 0xFFFF0000u);
            }
        }
    }
}

__device__ __forceinline__ uint32_t bf16_rne(float x) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 r = {(__bf16) x, (__bf16) 0.0f};
    return __builtin_bit_cast(uint32_t, r) & 0xFFFFu;
}

template <int TYPE>
__device__ __forceinline__ void store_values(void *dst, const float (&x)[kQK]) {
    if constexpr (TYPE == kTypeF32) {
        float4 *d = static_cast<float4 *>(dst);
#pragma unroll
        for (int c = 0; c < 8; ++c) d[c] = make_float4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
    } else {
        uint4 *d = static_cast<uint4 *>(dst);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = x[8 * c + 2 * j], b = x[8 * c + 2 * j + 1];
                w[j] = TYPE == kTypeF16 ? f32_to_f16_bits(a) | ((uint32_t) f32_to_f16_bits(b) << 16)
                                        : bf16_rne(a) | (bf16_rne(b) << 16);
            }
            d[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// Which block thread x of the grid moves.
struct Work {
    int tok, h, blk, which, slot;
    bool live;
};

template <int D>
__device__ __forceinline__ Work work_of(const SlotsParams &p) {
    constexpr int NB = D / kQK;
    constexpr int TOK = 64 / NB;  // tokens of a wave
    // units: (token tile, kv head, K or V), V fastest, one a wave
    const int64_t unit = (int64_t) blockIdx.x * (kSlotThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    Work w;
    w.which = (int) (unit & 1);
    const int64_t rest = unit >> 1;
    w.h = (int) (rest % p.g.n_kv);
    const int64_t tile = rest / p.g.n_kv;
    const int64_t tok = tile * TOK + lane / NB;
    w.blk = lane % NB;
    w.live = tok < p.n_tok;
    w.tok = w.live ? (int) tok : 0;
    w.slot = w.live ? p.slots[w.tok] : -1;
    return w;
}

// The 16 code bytes and the scale of a slot's block: dwords 4c..4c+3 of K
// stand 64 dwords apart, bytes of V 16 bytes apart.
template <int D>
struct Place {
    uint8_t *codes;
    uint16_t *scale;
    __device__ Place(const SlotsParams &p, const Work &w) {
        constexpr int NB = D / kQK, G = 2048 / D;
        const int s = w.slot & (G - 1), t = s >> 4, key = s & 15;
        const int tb = t * NB + w.blk;
        uint8_t *grp = p.base + p.g.group_offset(w.slot, w.h);
        codes = w.which == 0 ? grp + key * 16 + tb * 4 : grp + kVCodeOff + (key >> 2) * 256 + tb * 4 + (key & 3);
        scale = reinterpret_cast<uint16_t *>(grp + page_scale_offset(tb, key, w.which));
    }
};

}  // namespace

template <int D, int TYPE>
__global__ __launch_bounds__(kSlotThreads) void pages_append_kernel(SlotsParams p) {
    constexpr int NB = D / kQK;
    const Work w = work_of<D>(p);
    if (!w.live || w.slot < 0 || w.slot >= p.g.n_slots()) return;
    uint16_t d16;
    uint32_t qs[4];
    const void *rows = w.which == 0 ? p.k : p.v;
    if constexpr (TYPE == kTypeQ4_0) {
        const uint16_t *src = static_cast<const uint16_t *>(rows) +
                              (((int64_t) w.tok * p.g.n_kv + w.h) * NB + w.blk) * 9;
        d16 = src[0];
#pragma unroll
        for (int c = 0; c < 4; ++c) qs[c] = src[1 + 2 * c] | ((uint32_t) src[2 + 2 * c] << 16);
    } else {
        float x[kQK];
        load_block<TYPE>(static_cast<const uint8_t *>(rows) +
                             (w.tok * p.stride + w.h * D + w.blk * kQK) * type_bytes(TYPE), x);
        quantize_block_q4_0(x, d16, qs);
    }
    const Place<D> q(p, w);
    if (w.which == 0) {
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<uint32_t *>(q.codes + c * 256) = qs[c];
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) q.codes[i * 16] = (uint8_t) (qs[i >> 2] >> (8 * (i & 3)));
    }
    *q.scale = d16;
}

template <int D, int TYPE>
__global__ __launch_bounds__(kSlotThreads) void pages_gather_kernel(SlotsParams p) {
    constexpr int NB = D / kQK;
    const Work w = work_of<D>(p);
    if (!w.live) return;
    uint32_t qs[4] = {0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u};
    uint16_t d16 = 0;
    if (w.slot >= 0 && w.slot < p.g.n_slots()) {
        const Place<D> q(p, w);
        d16 = *q.scale;
        if (w.which == 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c) qs[c] = *reinterpret_cast<const uint32_t *>(q.codes + c * 256);
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t x = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) x |= (uint32_t) q.codes[(4 * c + j) * 16] << (8 * j);
                qs[c] = x;
            }
        }
    }
    void *rows = w.which == 0 ? p.k : p.v;
    if constexpr (TYPE == kTypeQ4_0) {
        uint16_t *dst = static_cast<uint16_t *>(rows) + (((int64_t) w.tok * p.g.n_kv + w.h) * NB + w.blk) * 9;
        dst[0] = d16;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            dst[1 + 2 * c] = (uint16_t) qs[c];
            dst[2 + 2 * c] = (uint16_t) (qs[c] >> 16);
        }
    } else {
        const float d = f16_bits_to_f32(d16);
        float x[kQK];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint32_t byte = qs[j >> 2] >> (8 * (j & 3));
            x[j] = (float) ((int) (byte & 15u) - 8) * d;
            x[j + 16] = (float) ((int) ((byte >> 4) & 15u) - 8) * d;
        }
        store_values<TYPE>(static_cast<uint8_t *>(rows) + (w.tok * p.stride + w.h * D + w.blk * kQK) * type_bytes(TYPE),
                           x);
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
    const int tok = 64 / (p.g.dim / kQK);
    const int64_t units = (p.n_tok + (int64_t) tok - 1) / tok * p.g.n_kv * 2;
    SlotsParams arg = p;
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
