// rows_rope.hip -- rotary positions of query and key rows.
//
// Pair i of a head's first `rot` elements, (2i, 2i + 1) or (i, i + rot / 2),
// turns by position * rates[i] and is scaled by the magnitude; the elements
// behind are copied.  A workgroup takes a part of the items of some tokens:
// pieces of 16 bytes (two, half a turned part apart, where pairs lie so), of 4,
// or single pairs, as the sizes and alignment allow.  A thread's items are
// read first; while they are under way the workgroup makes its tokens' cosines
// and sines, in double, rounded once to fp32.  Each product and sum is rounded
// as the ring's fused rotation does.
#include "angles.hpp"
#include "kernels.hpp"
#include "rows_device.hpp"

namespace bmo {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTable = 1024;  // pairs of a workgroup's tokens

struct RopeArgs {
    RopeParams p;
    int toks;    // tokens of a set
    int splits;  // workgroups of a set
    int items;   // of a head
    int turned;  // those that turn, first
    FastDiv div_items, div_heads, div_splits, div_half;
};

// W elements of 16 bytes (4 of fp32, 8 of 16 bits) or 4 (2 of 16 bits).
template <int W>
__device__ __forceinline__ uint4 load_piece(const uint8_t *p) {
    if constexpr (W == 2) return make_uint4(*reinterpret_cast<const uint32_t *>(p), 0, 0, 0);
    return *reinterpret_cast<const uint4 *>(p);
}
template <int W>
__device__ __forceinline__ void store_piece(uint8_t *p, const uint4 &u) {
    if constexpr (W == 2)
        *reinterpret_cast<uint32_t *>(p) = u.x;
    else
        *reinterpret_cast<uint4 *>(p) = u;
}
template <int W>
__device__ __forceinline__ void widen_piece(const uint4 &u, int type, float (&x)[W]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < W; ++j) {
        if constexpr (W == 4) {
            x[j] = __builtin_bit_cast(float, w[j]);
        } else {
            const uint32_t h = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
            x[j] = type == kTypeF16 ? f16_bits_to_f32(h) : __builtin_bit_cast(float, h << 16);
        }
    }
}
template <int W>
__device__ __forceinline__ uint4 narrow_piece(const float (&x)[W], int type) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < (W == 2 ? 1 : 4); ++j) {
        if constexpr (W == 4)
            w[j] = __builtin_bit_cast(uint32_t, x[j]);
        else
            w[j] = type == kTypeF16 ? f32_to_f16_bits(x[2 * j]) | ((uint32_t) f32_to_f16_bits(x[2 * j + 1]) << 16)
                                    : bf16_bits(x[2 * j]) | (bf16_bits(x[2 * j + 1]) << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Where an item lies, and what was read of it.
struct RopeItem {
    bool live, turns;
    int item;  // of its head
    int tok;   // of the set
    const uint8_t *x;
    uint8_t *out;  // the head's element 0
    uint4 a, b;
};

// W: elements of a piece (4 of fp32, 8 or 2 of 16 bits); 1: single pairs.
template <int W, bool INTER, int ITEMS>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
    __shared__ float2 s_tab[kRopeTable];
    const int half = a.p.rot / 2, type = a.p.type, size = type_bytes(type);
    const uint32_t set = a.div_splits.div(blockIdx.x), split = blockIdx.x - set * (uint32_t) a.splits;
    const int64_t tok0 = (int64_t) set * a.toks;
    const int n = (int) min((int64_t) a.toks, a.p.n_tok - tok0);
    const int heads = a.p.part[0].heads + a.p.part[1].heads;
    const uint32_t total = (uint32_t) n * (uint32_t) heads * (uint32_t) a.items;
    RopeItem it[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        RopeItem &k = it[u];
        const uint32_t i = (split * ITEMS + u) * kRopeThreads + threadIdx.x;
        k.live = i < total;
        const uint32_t at = k.live ? i : 0;
        const uint32_t hd = a.div_items.div(at), t = a.div_heads.div(hd);  // (token, head)
        int h = (int) (hd - t * (uint32_t) heads);
        const bool key = h >= a.p.part[0].heads;
        if (key) h -= a.p.part[0].heads;
        k.item = (int) (at - hd * (uint32_t) a.items);
        k.turns = k.item < a.turned;
        k.tok = (int) t;
        // (selected field by field: an indexed argument would live in scratch)
        const RopePart &q = a.p.part[0], &kv = a.p.part[1];
        const int64_t tok = tok0 + t, in_head = (int64_t) h * a.p.dim;
        k.x = static_cast<const uint8_t *>(key ? kv.x : q.x) + (tok * (key ? kv.stride : q.stride) + in_head) * size;
        k.out = static_cast<uint8_t *>(key ? kv.out : q.out) + (tok * (key ? kv.out_stride : q.out_stride) + in_head) * size;
        if constexpr (W > 1) {
            // (behind the turned ones an item is one piece)
            const int e = INTER || k.turns ? k.item * W : a.p.rot + (k.item - a.turned) * W;
            k.a = load_piece<W>(k.x + e * size);
            if (!INTER) k.b = load_piece<W>(k.x + (k.turns ? e + half : e) * size);
        } else {
            const int e = !k.turns ? a.p.rot + k.item - a.turned : INTER ? 2 * k.item : k.item;
            k.a.x = __builtin_bit_cast(uint32_t, load1(k.x, e, type));
            k.b.x = __builtin_bit_cast(uint32_t, load1(k.x, !k.turns ? e : INTER ? e + 1 : e + half, type));
        }
    }
    for (int i = threadIdx.x; i < n * half; i += kRopeThreads) {
        const int t = (int) a.div_half.div((uint32_t) i);
        double sn, cs;
        sincos_reduced((double) a.p.positions[tok0 + t] * a.p.rates[i - t * half], sn, cs);
        s_tab[i] = make_float2((float) (cs * a.p.magnitude), (float) (sn * a.p.magnitude));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
        const RopeItem &k = it[u];
        if (!k.live) continue;
        const float2 *tab = s_tab + k.tok * half;
        if constexpr (W > 1) {
            if (!k.turns) {
                const int e = INTER ? k.item * W : a.p.rot + (k.item - a.turned) * W;
                store_piece<W>(k.out + e * size, k.a);
                continue;
            }
            float x[W], y[W];
            widen_piece<W>(k.a, type, x);
            if constexpr (INTER) {
#pragma unroll
                for (int j = 0; j < W; j += 2) rope_pair(x[j], x[j + 1], tab[(k.item * W + j) / 2]);
            } else {
                widen_piece<W>(k.b, type, y);
#pragma unroll
                for (int j = 0; j < W; ++j) rope_pair(x[j], y[j], tab[k.item * W + j]);
                store_piece<W>(k.out + (k.item * W + half) * size, narrow_piece<W>(y, type));
            }
            store_piece<W>(k.out + k.item * W * size, narrow_piece<W>(x, type));
        } else if (k.turns) {
            const int e0 = INTER ? 2 * k.item : k.item, e1 = INTER ? e0 + 1 : k.item + half;
            float x = __builtin_bit_cast(float, k.a.x), y = __builtin_bit_cast(float, k.b.x);
            rope_pair(x, y, tab[k.item]);
            store1(k.out, e0, x, type);
            store1(k.out, e1, y, type);
        } else {
            store1(k.out, a.p.rot + k.item - a.turned, __builtin_bit_cast(float, k.a.x), type);
        }
    }
}

// Whether a part's rows can be read in pieces of so many bytes.
bool pieces_fit(const RopePart &q, int type, int bytes) {
    const int64_t size = type_bytes(type);
    auto fits = [&](const void *p, int64_t stride) {
        return reinterpret_cast<uintptr_t>(p) % (uintptr_t) bytes == 0 && stride * size % bytes == 0;
    };
    return q.heads == 0 || (fits(q.x, q.stride) && fits(q.out, q.out_stride));
}
bool pieces_fit(const RopeParams &p, int w) {
    const int bytes = w * type_bytes(p.type);
    return p.dim % w == 0 && p.rot % w == 0 && (p.interleaved || p.rot / 2 % w == 0) && pieces_fit(p.part[0], p.type, bytes) &&
           pieces_fit(p.part[1], p.type, bytes);
}

template <int W, int ITEMS>
const void *rope_function(bool inter) {
    return inter ? reinterpret_cast<const void *>(rope_kernel<W, true, ITEMS>)
                 : reinterpret_cast<const void *>(rope_kernel<W, false, ITEMS>);
}

}  // namespace

hipError_t launch_rope(const RopeParams &p, hipStream_t stream) {
    const int wide = 16 / type_bytes(p.type);
    const int w = pieces_fit(p, wide) ? wide : wide == 8 && pieces_fit(p, 2) ? 2 : 1;
    const bool in_place = p.part[0].x == p.part[0].out && (p.part[1].heads == 0 || p.part[1].x == p.part[1].out);
    RopeArgs a{};
    a.p = p;
    a.turned = w == 1 ? p.rot / 2 : p.interleaved ? p.rot / w : p.rot / 2 / w;
    a.items = a.turned + (in_place ? 0 : (p.dim - p.rot) / w);
    const int heads = p.part[0].heads + p.part[1].heads;
    const int64_t per_tok = (int64_t) a.items * heads;
    // Four items a thread of launches that fill the CUs, two of smaller ones
    // (5600 tokens x 40 heads of 128, neighbours, bf16: 23.5 against 28.8 us; 48 x
    // 64 heads, fp32: 3.0 against 2.6).
    const int items = per_tok * p.n_tok >= (int64_t) 4 * 2048 * kRopeThreads && !(w > 2 && !p.interleaved) ? 4 : 2;
    // Tokens to fill a workgroup's items once, as far as the table holds them;
    // workgroups to share the items of a token that has more.
    const int64_t group = kRopeThreads * items;
    int64_t toks = group / per_tok;
    toks = toks < 1 ? 1 : toks > kRopeTable / (p.rot / 2) ? kRopeTable / (p.rot / 2) : toks;
    a.toks = (int) toks;
    a.splits = (int) ((toks * per_tok + group - 1) / group);
    a.div_items = make_fastdiv((uint32_t) a.items);
    a.div_heads = make_fastdiv((uint32_t) heads);
    a.div_splits = make_fastdiv((uint32_t) a.splits);
    a.div_half = make_fastdiv((uint32_t) p.rot / 2);
    void *args[] = {&a};
    const bool inter = p.interleaved != 0;
    const void *f = nullptr;
    if (items == 4)
        f = w == 1   ? rope_function<1, 4>(inter)
            : w == 2 ? rope_function<2, 4>(inter)
            : w == 4 ? reinterpret_cast<const void *>(rope_kernel<4, true, 4>)
                     : reinterpret_cast<const void *>(rope_kernel<8, true, 4>);
    else
        f = w == 1   ? rope_function<1, 2>(inter)
            : w == 2 ? rope_function<2, 2>(inter)
            : w == 4 ? rope_function<4, 2>(inter)
                     : rope_function<8, 2>(inter);
    const int64_t groups = (p.n_tok + toks - 1) / toks * a.splits;
    return hipLaunchKernel(f, dim3((unsigned) groups), dim3(kRopeThreads), args, 0, stream);
}

}  // namespace bmo
