// rows_rope.hip -- rotary positions of query and key rows.
//
// Pair i of a head's first `rot` elements, (2i, 2i + 1) or (i, i + rot / 2),
// turns by position * rates[i] and is scaled by the magnitude; the elements
// behind are copied.  A workgroup takes some tokens: it makes their cosines and
// sines once, in double, rounded once to fp32, and turns every head's pairs
// with them, each product and sum rounded as the ring's fused rotation does.
#include "angles.hpp"
#include "kernels.hpp"
#include "rows_device.hpp"

namespace bmo {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTable = 1024;  // pairs of a workgroup's tokens

struct RopeArgs {
    RopeParams p;
    int toks;         // tokens of a workgroup
    int splits;       // workgroups of a set of tokens
    int items;        // of a head
    int turned;       // those that turn, first
    FastDiv div_items, div_heads;
};

// W: elements of a piece; a piece turns W pairs of halves that lie rot / 2
// apart, or W / 2 pairs of neighbours; W == 1: single pairs of either layout.
template <int W, bool INTER>
__device__ __forceinline__ void turn_item(const RopeArgs &a, const void *x, int64_t at, void *out, int64_t to, int item,
                                          const float2 *tab) {
    const int type = a.p.type, half = a.p.rot / 2;
    if (item >= a.turned) {  // behind the turned elements
        if (x == out) return;
        const int e = a.p.rot + (item - a.turned) * W;
#pragma unroll
        for (int j = 0; j < W; ++j) store1(out, to + e + j, load1(x, at + e + j, type), type);
        return;
    }
    if constexpr (W == 1) {
        const int e0 = INTER ? 2 * item : item, e1 = INTER ? e0 + 1 : item + half;
        float u = load1(x, at + e0, type), v = load1(x, at + e1, type);
        rope_pair(u, v, tab[item]);
        store1(out, to + e0, u, type);
        store1(out, to + e1, v, type);
    }
}

template <int W, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
    __shared__ float2 s_tab[kRopeTable];
    const int half = a.p.rot / 2;
    const int64_t tok0 = (int64_t) (blockIdx.x / (uint32_t) a.splits) * a.toks;
    const int split = (int) (blockIdx.x % (uint32_t) a.splits);
    const int n = (int) min((int64_t) a.toks, a.p.n_tok - tok0);
    for (int i = threadIdx.x; i < n * half; i += kRopeThreads) {
        const int t = i / half;
        double sn, cs;
        sincos_reduced((double) a.p.positions[tok0 + t] * a.p.rates[i - t * half], sn, cs);
        s_tab[i] = make_float2((float) (cs * a.p.magnitude), (float) (sn * a.p.magnitude));
    }
    __syncthreads();
    const int heads = a.p.part[0].heads + a.p.part[1].heads;
    const uint32_t total = (uint32_t) (n * heads * a.items);
    for (uint32_t i = split * kRopeThreads + threadIdx.x; i < total; i += kRopeThreads * a.splits) {
        const uint32_t hd = a.div_items.div(i), item = i - hd * a.items;  // (token, head)
        const uint32_t t = a.div_heads.div(hd);
        int h = (int) (hd - t * heads);
        const int which = h >= a.p.part[0].heads;
        if (which) h -= a.p.part[0].heads;
        // (selected field by field: an indexed argument would live in scratch)
        const RopePart &q = a.p.part[0], &k = a.p.part[1];
        const int64_t tok = tok0 + t, in_head = (int64_t) h * a.p.dim;
        turn_item<W, INTER>(a, which ? k.x : q.x, tok * (which ? k.stride : q.stride) + in_head, which ? k.out : q.out,
                            tok * (which ? k.out_stride : q.out_stride) + in_head, (int) item, s_tab + t * half);
    }
}

}  // namespace

hipError_t launch_rope(const RopeParams &p, hipStream_t stream) {
    RopeArgs a{};
    a.p = p;
    a.toks = 1;
    a.turned = p.rot / 2;
    a.items = a.turned + p.dim - p.rot;
    a.splits = 1;
    a.div_items = make_fastdiv(a.items);
    a.div_heads = make_fastdiv(p.part[0].heads + p.part[1].heads);
    void *args[] = {&a};
    const void *f = p.interleaved ? reinterpret_cast<const void *>(rope_kernel<1, true>)
                                  : reinterpret_cast<const void *>(rope_kernel<1, false>);
    return hipLaunchKernel(f, dim3((unsigned) p.n_tok), dim3(kRopeThreads), args, 0, stream);
}

}  // namespace bmo
