// rows_rope.hip -- rotary positions of query and key rows.
//
// Pair i of a head's first `rot` elements, (2i, 2i + 1) or (i, i + rot / 2),
// turns by position * rates[i] and is scaled by the magnitude; the elements
// behind are copied.  A workgroup takes a part of the items of some tokens:
// pieces of 16, 8 or 4 bytes (two, half a turned part apart, where pairs lie
// so), or single pairs, and pieces of the copied elements, as the sizes and
// alignment allow.  A thread's items are read first; while they are under way
// the workgroup makes its tokens' cosines and sines, in double, rounded once to
// fp32 (of angles that are products in double: far positions turn by the rounding
// of these too).  Each product and sum is rounded as the ring's fused rotation does.
//
// Bound by its bytes, and in small calls by one load and one sine in turn: 5600
// tokens x 40 heads of 128, bf16, in 24.6 us, 4.7 TB/s (a large copy: 5.1); 48 x
// 64 heads, fp32, in 2.6.  Smaller pieces take more threads to a byte: 4000 x 32
// heads of 80, 20 of them turned by halves, fp16, in 21.5 us (1.9 TB/s), 30 when
// the copied elements went in pieces of 4 bytes like the turned ones.
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
    int tail;    // bytes of the others (0: an element each)
    FastDiv div_items, div_heads, div_splits, div_half;
};

// A piece of 16, 8 or 4 bytes, aligned to them.
__device__ __forceinline__ uint4 load_piece(const uint8_t *p, int bytes) {
    if (bytes == 16) return *reinterpret_cast<const uint4 *>(p);
    if (bytes == 8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        return make_uint4(u.x, u.y, 0, 0);
    }
    return make_uint4(*reinterpret_cast<const uint32_t *>(p), 0, 0, 0);
}
__device__ __forceinline__ void store_piece(uint8_t *p, const uint4 &u, int bytes) {
    if (bytes == 16)
        *reinterpret_cast<uint4 *>(p) = u;
    else if (bytes == 8)
        *reinterpret_cast<uint2 *>(p) = make_uint2(u.x, u.y);
    else
        *reinterpret_cast<uint32_t *>(p) = u.x;
}
// W elements of `SIZE` bytes.
template <int W, int SIZE>
__device__ __forceinline__ void widen_piece(const uint4 &u, int type, float (&x)[W]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < W; ++j) {
        if constexpr (SIZE == 4) {
            x[j] = __builtin_bit_cast(float, w[j]);
        } else {
            const uint32_t h = j & 1 ? w[j >> 1] >> 16 : w[j >> 1] & 0xFFFFu;
            x[j] = type == kTypeF16 ? f16_bits_to_f32(h) : __builtin_bit_cast(float, h << 16);
        }
    }
}
template <int W, int SIZE>
__device__ __forceinline__ uint4 narrow_piece(const float (&x)[W], int type) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < W * SIZE / 4; ++j) {
        if constexpr (SIZE == 4)
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

// W: elements of a turned piece, SIZE: bytes of each; W 1: single pairs.
template <int W, int SIZE, bool INTER, int ITEMS>
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
        const int rest = k.item - a.turned;
        if constexpr (W * SIZE == 16) {
            // (the others are of 16 bytes too, and read as these: no branch around the loads)
            const int e = INTER || k.turns ? k.item * W : a.p.rot + rest * W;
            k.a = load_piece(k.x + e * SIZE, 16);
            if (!INTER) k.b = load_piece(k.x + (k.turns ? e + half : e) * SIZE, 16);
        } else if (!k.turns && a.tail) {
            k.a = load_piece(k.x + a.p.rot * size + rest * a.tail, a.tail);
        } else if (W == 1 || !k.turns) {
            const int e = !k.turns ? a.p.rot + rest : INTER ? 2 * k.item : k.item;
            k.a.x = __builtin_bit_cast(uint32_t, load1(k.x, e, type));
            k.b.x = __builtin_bit_cast(uint32_t, load1(k.x, !k.turns ? e : INTER ? e + 1 : e + half, type));
        } else {
            k.a = load_piece(k.x + k.item * W * SIZE, W * SIZE);
            if (!INTER) k.b = load_piece(k.x + (k.item * W + half) * SIZE, W * SIZE);
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
        const int rest = k.item - a.turned;
        if (!k.turns) {
            if (W * SIZE == 16)
                store_piece(k.out + (a.p.rot + rest * W) * SIZE, k.a, 16);
            else if (a.tail)
                store_piece(k.out + a.p.rot * size + rest * a.tail, k.a, a.tail);
            else
                store1(k.out, a.p.rot + rest, __builtin_bit_cast(float, k.a.x), type);
        } else if constexpr (W > 1) {
            float x[W], y[W];
            widen_piece<W, SIZE>(k.a, type, x);
            if constexpr (INTER) {
#pragma unroll
                for (int j = 0; j < W; j += 2) rope_pair(x[j], x[j + 1], tab[(k.item * W + j) / 2]);
            } else {
                widen_piece<W, SIZE>(k.b, type, y);
#pragma unroll
                for (int j = 0; j < W; ++j) rope_pair(x[j], y[j], tab[k.item * W + j]);
                store_piece(k.out + (k.item * W + half) * SIZE, narrow_piece<W, SIZE>(y, type), W * SIZE);
            }
            store_piece(k.out + k.item * W * SIZE, narrow_piece<W, SIZE>(x, type), W * SIZE);
        } else {
            const int e0 = INTER ? 2 * k.item : k.item, e1 = INTER ? e0 + 1 : k.item + half;
            float x = __builtin_bit_cast(float, k.a.x), y = __builtin_bit_cast(float, k.b.x);
            rope_pair(x, y, tab[k.item]);
            store1(k.out, e0, x, type);
            store1(k.out, e1, y, type);
        }
    }
}

// The largest pieces (16, 8 or 4 bytes; 0: not even those) that so many bytes,
// the rows and their strides consist of.
int piece_bytes(const RopeParams &p, int64_t bytes) {
    const int64_t size = type_bytes(p.type);
    uint64_t all = (uint64_t) bytes | (uint64_t) (p.dim * size) | 16;
    for (const RopePart &q : p.part)
        if (q.heads)
            all |= reinterpret_cast<uintptr_t>(q.x) | reinterpret_cast<uintptr_t>(q.out) | (uint64_t) (q.stride * size) |
                   (uint64_t) (q.out_stride * size);
    const int n = (int) (all & (0 - all));  // its lowest bit
    return n >= 4 ? n : 0;
}

template <int W, int SIZE>
const void *rope_function(bool inter, int items) {
    if (items == 4) {
        if (inter) return reinterpret_cast<const void *>(rope_kernel<W, SIZE, true, 4>);
        if constexpr (W * SIZE < 16) return reinterpret_cast<const void *>(rope_kernel<W, SIZE, false, 4>);
    }
    return inter ? reinterpret_cast<const void *>(rope_kernel<W, SIZE, true, 2>)
                 : reinterpret_cast<const void *>(rope_kernel<W, SIZE, false, 2>);
}

}  // namespace

hipError_t launch_rope(const RopeParams &p, hipStream_t stream) {
    const int size = type_bytes(p.type);
    // (one of two elements at least, for neighbours turn together)
    const int bytes = piece_bytes(p, (int64_t) (p.interleaved ? p.rot : p.rot / 2) * size);
    const int w = bytes >= 2 * size ? bytes / size : 1;
    const bool in_place = p.part[0].x == p.part[0].out && (p.part[1].heads == 0 || p.part[1].x == p.part[1].out);
    RopeArgs a{};
    a.p = p;
    a.turned = p.interleaved ? p.rot / (w == 1 ? 2 : w) : p.rot / 2 / w;
    a.tail = piece_bytes(p, (int64_t) p.rot * size);
    const int rest = in_place ? 0 : (p.dim - p.rot) * size;
    a.items = a.turned + rest / (a.tail ? a.tail : size);
    const int heads = p.part[0].heads + p.part[1].heads;
    const int64_t per_tok = (int64_t) a.items * heads;
    // Four items a thread of launches that fill the CUs, two of smaller ones
    // (5600 tokens x 40 heads of 128, neighbours, bf16: 23.5 against 28.8 us; 48 x
    // 64 heads, fp32: 3.0 against 2.6).
    const int items = per_tok * p.n_tok >= (int64_t) 4 * 2048 * kRopeThreads && !(bytes == 16 && !p.interleaved) ? 4 : 2;
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
    const void *f = w == 1     ? rope_function<1, 0>(inter, items)
                    : w == 8   ? rope_function<8, 2>(inter, items)
                    : size == 4 ? (w == 4 ? rope_function<4, 4>(inter, items) : rope_function<2, 4>(inter, items))
                                : (w == 4 ? rope_function<4, 2>(inter, items) : rope_function<2, 2>(inter, items));
    const int64_t groups = (p.n_tok + toks - 1) / toks * a.splits;
    return hipLaunchKernel(f, dim3((unsigned) groups), dim3(kRopeThreads), args, 0, stream);
}

}  // namespace bmo
