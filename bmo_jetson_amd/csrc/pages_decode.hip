// pages_decode.hip -- attention of one row per entry over its pages.
//
// o = sum_j p_j v_j, p = softmax(scale q . k_j) over the entry's last
// min(len, window) positions.  HBM bounds it: 2 * 18 bytes per 32 elements of
// a position's K and V against 4 operations per element and query head.
//
// One wave step takes 32 positions of one kv head: 16 bytes of K codes and of
// V codes a lane and tile of 16 (pages_layout.hpp), straight from HBM to the
// operands of v_mfma_f32_16x16x32.  The 16 columns of the products hold
//   (head r, block b): heads of the kv head's group, up to 16 / NB of them,
//                      each column with the query of its own block only; or
//   head r:            up to 16 heads, when the group has more than 16 / NB.
// In the first form a lane has one block's products, so the block scales cost
// one multiply a score and one a weight instead of NB each.
//
// K side: q (times scale * log2 e) enters as two fp16 parts hi + lo of
// q * 2^e, e chosen per row, exact to 2^-22 of the row's largest element; the
// codes minus 8 are exact in fp16, products are summed in fp32 per block and
// multiplied by the block's scale in fp32.  V side: p * d (weight times V
// scale) enters as two bf16 parts, exact to 2^-17 of itself whatever its
// range, against the plain codes 0..15, exact in bf16; 8 times the parts' sum,
// from the same matrix instruction with a constant operand, is taken off every
// eight steps, so that this debt does not grow.  An fp32 call is therefore as
// close as fp32 sums (about 1e-6); 16-bit calls use the same kernel, whose
// time the bytes decide.
//
// Softmax is online with a running maximum per column, raised only when a
// score passes it by 8 (log2 units), so that the exchange between the four
// lanes of a column and the rescaling are rare.  Masked positions get weight
// 0 by select, whatever their slots hold.
//
// Work: an item is a run of steps of one (entry, kv head, head set), walked
// by the NW waves of a workgroup in turn and joined in LDS.  When the entries
// are few or long, an entry's steps are cut in ceil(n / c) even runs, with c
// from all entries' steps and the workgroups wanted (every workgroup sums the
// lengths itself), their results kept as (max, sum, row) in the workspace and
// joined by a second kernel in the order of the runs.
#include "pages_device.hpp"

namespace bmo {

namespace {

constexpr int kStep = 32;        // positions a wave step
constexpr int kDecodeWaves = 4;  // waves a workgroup
constexpr int kSettle = 8;       // steps between taking off 8 * sum p d
// Workgroups a split launch is cut for, and the fewest steps a run has.
constexpr int kWantWorkgroups = 512;
constexpr int kMinRun = 8;

struct DecodeArgs {
    PagesDecodeParams p;
    int group;    // query heads a kv head
    int n_hs;     // head sets a kv head
    int units;    // n_kv * n_hs
    int split;    // 0: every entry is one run
    int append;
};

// Steps of an entry: its visible positions are [lo, len).
struct Span {
    int len, lo, step0, n;
};
__device__ __forceinline__ Span span_of(const DecodeArgs &a, int len) {
    Span s;
    const int64_t room = (int64_t) a.p.max_pages << a.p.g.page_shift;
    s.len = (int) min((int64_t) max(len, 0), room);
    s.lo = a.p.window > 0 && s.len > a.p.window ? s.len - a.p.window : 0;
    s.step0 = s.lo / kStep;
    s.n = (int) (((int64_t) s.len + kStep - 1) / kStep) - s.step0;
    return s;
}
__device__ __forceinline__ int runs_of(int n, int c) { return n <= c ? 1 : (n + c - 1) / c; }


// The longest run of steps, from the steps of all entries.
__device__ __forceinline__ int run_length(const DecodeArgs &a, int lane) {
    int64_t total = 0;
    for (int b0 = 0; b0 < a.p.n_batch; b0 += 64) {
        const int b = b0 + lane;
        const int n = b < a.p.n_batch ? span_of(a, a.p.lens[b]).n : 0;
        // (64 entries of at most 2^25 steps)
        total += (uint32_t) __shfl(wave_prefix(n, lane), 63);
    }
    const int64_t c = (total * a.units + kWantWorkgroups - 1) / kWantWorkgroups;
    return (int) min(max(c, (int64_t) kMinRun), (int64_t) INT32_MAX);
}

// Item `item` of a split launch: its entry, run, and the index of its entry's
// first partial result.  False past the last item.
struct Item {
    int b, run, runs, unit, part0;
};
__device__ __forceinline__ bool find_item(const DecodeArgs &a, int item, int c, int lane, Item &it) {
    const int row = item / a.units;  // (entry, run)
    it.unit = item - row * a.units;
    int rows = 0, parts = 0;
    for (int b0 = 0; b0 < a.p.n_batch; b0 += 64) {
        const int b = b0 + lane;
        const int runs = b < a.p.n_batch ? runs_of(span_of(a, a.p.lens[b]).n, c) : 0;
        const int upto = wave_prefix(runs, lane) + rows;
        const int parts_upto = wave_prefix(runs > 1 ? runs : 0, lane) + parts;
        const uint64_t past = __ballot(upto > row);
        if (past) {
            const int l = __ffsll((unsigned long long) past) - 1;
            it.b = b0 + l;
            it.runs = __shfl(runs, l);
            it.run = row - (__shfl(upto, l) - it.runs);
            it.part0 = __shfl(parts_upto, l) - (it.runs > 1 ? it.runs : 0);
            return true;
        }
        rows = __shfl(upto, 63);
        parts = __shfl(parts_upto, 63);
    }
    return false;
}

// Floats of a partial result of HC heads.
template <int D>
__host__ __device__ constexpr int part_floats(int hc) { return hc * (D + 2); }

}  // namespace

// SPREAD: the columns are (head, block); otherwise heads.
template <int D, bool SPREAD>
__global__ __launch_bounds__(64 * kDecodeWaves) void pages_decode_kernel(DecodeArgs a) {
    constexpr int NW = kDecodeWaves;
    constexpr int NB = D / kQK;
    constexpr int TG = kStep * D / 2048;    // groups a step
    constexpr int T = 2 / TG;               // tiles of 16 a group
    constexpr int CB = SPREAD ? NB : 1;     // columns a head
    constexpr int HC = 16 / CB;             // heads a head set
    constexpr int PB = NB / CB;             // blocks a column
    const PagesDecodeParams &p = a.p;
    const PagesGeom &g = p.g;

    __shared__ float s_out[NW][HC][D];
    __shared__ float s_m[NW][HC], s_l[NW][HC];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int col = lane & 15, oct = lane >> 4;
    const int r = col / CB, cb = col % CB;

    Item it{};
    if (a.split) {
        const int c = run_length(a, lane);
        if (!find_item(a, (int) blockIdx.x, c, lane, it)) return;
    } else {
        it.b = (int) blockIdx.x / a.units;
        it.unit = (int) blockIdx.x - it.b * a.units;
        it.runs = 1;
    }
    const int b = __builtin_amdgcn_readfirstlane(it.b);
    const int kvh = it.unit / a.n_hs, hs = it.unit - kvh * a.n_hs;
    const int heads = min(HC, a.group - hs * HC);  // heads of this set
    const int head0 = kvh * a.group + hs * HC;
    const Span sp = span_of(a, p.lens[b]);
    const int s_begin = sp.step0 + (int) ((int64_t) sp.n * it.run / it.runs);
    const int s_end = sp.step0 + (int) ((int64_t) sp.n * (it.run + 1) / it.runs);
    const int *table = p.table + (int64_t) b * p.max_pages;

    // The new token's row goes to its slot before the wave that will read it
    // starts on its steps (of several head sets each writes the same bytes).
    if (a.append && sp.len > 0 && s_end == sp.step0 + sp.n && wave == (s_end - 1 - s_begin) % NW) {
        constexpr int BL = 32 / NB, NE = NB, HE = NE / 2, LPD = 4 / HE;
        const int nb = lane / BL, gi = lane % BL;
        const int64_t src = (int64_t) b * p.kv_stride + kvh * D + (nb % NB) * kQK + gi * HE;
        const void *row = nb < NB ? p.k_new : p.v_new;
        float x[NE];
#pragma unroll
        for (int t = 0; t < HE; ++t) {
            x[t] = load1(row, src + t, p.type);
            x[HE + t] = load1(row, src + 16 + t, p.type);
        }
        uint16_t d16;
        const uint32_t dw = quantize_block_q4_0_lanes<BL>(x, gi, d16);
        const int pos = sp.len - 1;
        const int id = table[pos >> g.page_shift];
        if ((unsigned) id < (unsigned) g.n_pages) {
            const int slot = (id << g.page_shift) | (pos & (g.page - 1));
            uint8_t *grp = p.base + g.group_offset(slot, kvh);
            const int s = slot & (2048 / D - 1), key = s & 15, tb = (s >> 4) * NB + nb % NB;
            const int c = gi / LPD;  // code dword of the block
            if (nb < NB) {
                if (gi % LPD == 0) *reinterpret_cast<uint32_t *>(grp + (c * 16 + key) * 16 + tb * 4) = dw;
            } else {
                // bytes gi * HE .. of the block, each to its own dword
#pragma unroll
                for (int t = 0; t < HE; ++t) {
                    const int i = gi * HE + t;
                    grp[kVCodeOff + ((key >> 2) * 16 + i) * 16 + tb * 4 + (key & 3)] = (uint8_t) (dw >> (8 * (i & 3)));
                }
            }
            if (gi == 0)
                reinterpret_cast<uint16_t *>(grp + (nb < NB ? kPageScaleK : kPageScaleV))[tb * 16 + key] = d16;
        }
        __threadfence_block();
    }

    // The query: hi and lo halves of the column's row, of every block (zero
    // outside the column's own when columns are blocks).
    pg_half8 qh[NB], ql[NB];
    float sq;
    {
        const int64_t src = (int64_t) b * p.q_stride + (int64_t) (head0 + (r < heads ? r : 0)) * D;
        float amax = 0.0f, bad = 0.0f;
        float x[PB][8];
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            const int blk = SPREAD ? cb : i;
            const pg_float4 lo = load4(p.q, src + blk * kQK + 4 * oct, p.type);
            const pg_float4 hi = load4(p.q, src + blk * kQK + 4 * oct + 16, p.type);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = octet_elem(0, j);  // 0..3, 16..19
                x[i][j] = (e < 16 ? lo[e & 3] : hi[e & 3]) * p.qscale;
                if (r >= heads) x[i][j] = 0.0f;
                amax = fmaxf(amax, __builtin_fabsf(x[i][j]));
                bad += x[i][j] * 0.0f;  // NaN if it is not finite
            }
        }
        if constexpr (CB >= 2) {
            amax = fmaxf(amax, pg_dpp<0xB1>(amax));
            bad += pg_dpp<0xB1>(bad);
        }
        if constexpr (CB >= 4) {
            amax = fmaxf(amax, pg_dpp<0x4E>(amax));
            bad += pg_dpp<0x4E>(bad);
        }
        amax = fmaxf(amax, __shfl_xor(amax, 16));
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        bad += __shfl_xor(bad, 16);
        bad += __shfl_xor(bad, 32);
        const int ex = __builtin_amdgcn_frexp_expf(amax);
        sq = bad == 0.0f ? __builtin_amdgcn_ldexpf(1.0f, ex - 15) : __builtin_nanf("");
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
            const bool mine = !SPREAD || blk == cb;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float y = __builtin_amdgcn_ldexpf(x[SPREAD ? 0 : blk][j], 15 - ex);
                const _Float16 h = (_Float16) y;
                qh[blk][j] = mine ? h : (_Float16) 0.0f;
                ql[blk][j] = mine ? (_Float16) (y - (float) h) : (_Float16) 0.0f;
            }
        }
    }

    struct Tile {
        uint4 k[TG], v[TG];
        uint2 ks[2][PB], vs[2][PB];
        bool ok[TG];
    };
    // Page ids, 64 at a time in the lanes.
    int ids = 0, ids0 = -1;
    auto page_of = [&](int col_) {
        if ((col_ & ~63) != ids0) {
            ids0 = col_ & ~63;
            ids = ids0 + lane < p.max_pages ? table[ids0 + lane] : -1;
        }
        return __builtin_amdgcn_readlane(ids, col_ & 63);
    };
    const int last_group = max((sp.len - 1) / (2048 / D), 0);
    auto load = [&](int step, Tile &t) {
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            const int grp = min(step * TG + i, last_group);
            const int id = page_of(grp >> g.group_shift);
            t.ok[i] = (unsigned) id < (unsigned) g.n_pages;
            const uint8_t *at = p.base + (int64_t) (t.ok[i] ? id : 0) * g.page_bytes +
                                (((int64_t) kvh << g.group_shift) + (grp & ((1 << g.group_shift) - 1))) * kGroupBytes;
            t.k[i] = *reinterpret_cast<const uint4 *>(at + lane * 16);
            t.v[i] = *reinterpret_cast<const uint4 *>(at + kVCodeOff + lane * 16);
#pragma unroll
            for (int u = 0; u < T; ++u)
#pragma unroll
                for (int j = 0; j < PB; ++j) {
                    const int tb = u * NB + (SPREAD ? cb : j);
                    t.ks[i * T + u][j] = *reinterpret_cast<const uint2 *>(at + kPageScaleK + tb * 32 + oct * 8);
                    t.vs[i * T + u][j] = *reinterpret_cast<const uint2 *>(at + kPageScaleV + tb * 32 + oct * 8);
                }
        }
    };

    float m = kPagesFloor, mt = kPagesFloor, l = 0.0f;
    pg_float4 acc[NB][2], owed[PB];
    const pg_float4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i][0] = acc[i][1] = zero;
#pragma unroll
    for (int i = 0; i < PB; ++i) owed[i] = zero;
    pg_bf16x8 eight;
#pragma unroll
    for (int j = 0; j < 8; ++j) eight[j] = (__bf16) 8.0f;

    auto settle = [&]() {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            acc[i][0] -= owed[SPREAD ? 0 : i];
            acc[i][1] -= owed[SPREAD ? 0 : i];
        }
#pragma unroll
        for (int i = 0; i < PB; ++i) owed[i] = zero;
    };

    auto word = [](const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
    auto scale_of = [](const uint2 &v, int i) {
        const uint32_t w = i < 2 ? v.x : v.y;
        const pg_half2 h = __builtin_bit_cast(pg_half2, w);
        return (float) (i & 1 ? h.y : h.x);
    };

    auto compute = [&](int step, const Tile &t) {
        float s[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            pg_float4 d = zero;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                const pg_half8 kc = k_octet(word(t.k[u / T], (u % T) * NB + blk));
                if constexpr (!SPREAD) d = zero;
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, qh[blk], d, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc, ql[blk], d, 0, 0, 0);
                if constexpr (!SPREAD) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[i] = __builtin_fmaf(d[i], scale_of(t.ks[u][blk], i), part[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = part[i];
                if constexpr (SPREAD) {
                    x = d[i] * scale_of(t.ks[u][0], i);
                    x += pg_dpp<0xB1>(x);
                    if constexpr (NB == 4) x += pg_dpp<0x4E>(x);
                }
                const int pos = step * kStep + u * 16 + 4 * oct + i;
                const bool ok = pos >= sp.lo && pos < sp.len && t.ok[u / T];
                s[4 * u + i] = ok ? x * sq : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        if (__any(mx > mt)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            mt = m_new + kPagesLazy;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                acc[i][0] *= alpha;
                acc[i][1] *= alpha;
            }
#pragma unroll
            for (int i = 0; i < PB; ++i) owed[i] *= alpha;
        }
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __builtin_amdgcn_exp2f(s[i] - m);
            l += w[i];
        }
#pragma unroll
        for (int j = 0; j < PB; ++j) {
            pg_bf16x8 ph, pl;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = scale_of(t.vs[i >> 2][j], i & 3);
                const float x = s[i] == -INFINITY ? 0.0f : w[i] * d;
                const __bf16 h = (__bf16) x;
                ph[i] = h;
                pl[i] = (__bf16) (x - (float) h);
            }
            owed[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight, ph, owed[j], 0, 0, 0);
            owed[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight, pl, owed[j], 0, 0, 0);
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                if (!SPREAD && blk != j) continue;
                const uint32_t x0 = word(t.v[0], blk);
                const uint32_t x1 = word(t.v[1 / T], (1 % T) * NB + blk);
                const pg_bf16x8 vl = v_octet(x0, x1), vh = v_octet(x0 >> 4, x1 >> 4);
                acc[blk][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vl, ph, acc[blk][0], 0, 0, 0);
                acc[blk][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vl, pl, acc[blk][0], 0, 0, 0);
                acc[blk][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vh, ph, acc[blk][1], 0, 0, 0);
                acc[blk][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vh, pl, acc[blk][1], 0, 0, 0);
            }
        }
    };

    // Steps s_begin + wave, + NW, ...; the next step's loads are in flight
    // while one is computed.
    int step = s_begin + wave;
    if (step < s_end) {
        Tile t0, t1;
        load(step, t0);
        int settle_in = kSettle;
        for (;;) {
            load(min(step + NW, s_end - 1), t1);
            compute(step, t0);
            if ((step += NW) >= s_end) break;
            load(min(step + NW, s_end - 1), t0);
            compute(step, t1);
            if ((step += NW) >= s_end) break;
            if ((settle_in -= 2) <= 0) {
                settle();
                settle_in = kSettle;
            }
        }
    }
    settle();
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // The column's 2 * 4 outputs of its own block (of every block): element
    // 32 blk + 16 half + 4 oct + i.
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
        if (!SPREAD || blk == cb) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                *reinterpret_cast<pg_float4 *>(&s_out[wave][r][blk * kQK + half * 16 + 4 * oct]) = acc[blk][half];
        }
    }
    if (oct == 0 && cb == 0) {
        s_m[wave][r] = m;
        s_l[wave][r] = l;
    }
    __syncthreads();
    const int part = it.part0 + it.run;
    for (int i = threadIdx.x; i < heads * D; i += 64 * NW) {
        const int rr = i / D, e = i % D;
        float M = s_m[0][rr];
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, s_m[w][rr]);
        float L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][rr] - M);
            L = __builtin_fmaf(f, s_l[w][rr], L);
            o = __builtin_fmaf(f, s_out[w][rr][e], o);
        }
        if (it.runs == 1) {
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
            store1(p.out, ((int64_t) b * p.n_heads + head0 + rr) * D + e, o * inv, p.type);
        } else {
            float *dst = p.work + ((int64_t) part * a.units + it.unit) * part_floats<D>(HC);
            dst[rr * D + e] = o;
            if (e == 0) {
                dst[HC * D + rr] = M;
                dst[HC * D + HC + rr] = L;
            }
        }
    }
}

// Joins the runs of the entries that were cut, in order: a workgroup of D
// threads takes one (entry, query head).
template <int D, bool SPREAD>
__global__ __launch_bounds__(D) void pages_join_kernel(DecodeArgs a) {
    constexpr int HC = SPREAD ? 16 / (D / kQK) : 16;
    const PagesDecodeParams &p = a.p;
    const int lane = threadIdx.x & 63;
    const int b = (int) blockIdx.x / p.n_heads, h = (int) blockIdx.x - b * p.n_heads;
    const int c = run_length(a, lane);
    const int runs = runs_of(span_of(a, p.lens[b]).n, c);
    if (runs == 1) return;
    int part0 = 0;
    for (int b0 = 0; b0 < b; b0 += 64) {
        const int i = b0 + lane;
        const int n = i < b ? runs_of(span_of(a, p.lens[i]).n, c) : 0;
        part0 += __shfl(wave_prefix(n > 1 ? n : 0, lane), 63);
    }
    const int kvh = h / a.group, in_group = h - kvh * a.group;
    const int hs = in_group / HC, rr = in_group - hs * HC;
    const int64_t stride = (int64_t) a.units * part_floats<D>(HC);
    const float *src = p.work + ((int64_t) part0 * a.units + kvh * a.n_hs + hs) * part_floats<D>(HC);
    float M = kPagesFloor;
    for (int i = 0; i < runs; ++i) M = fmaxf(M, src[i * stride + HC * D + rr]);
    float L = 0.0f, o = 0.0f;
    for (int i = 0; i < runs; ++i) {
        const float *q = src + i * stride;
        const float f = __builtin_amdgcn_exp2f(q[HC * D + rr] - M);
        L = __builtin_fmaf(f, q[HC * D + HC + rr], L);
        o = __builtin_fmaf(f, q[rr * D + threadIdx.x], o);
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    store1(p.out, ((int64_t) b * p.n_heads + h) * D + threadIdx.x, o * inv, p.type);
}

namespace {

// Heads of a head set: columns are (head, block) while a group fits that way.
bool spread(const PagesGeom &g, int group) { return group <= 16 / (g.dim / kQK); }
int set_heads(const PagesGeom &g, int group) { return spread(g, group) ? 16 / (g.dim / kQK) : 16; }

template <int D, bool SPREAD>
hipError_t launch_of(const DecodeArgs &arg, int64_t items, hipStream_t stream) {
    DecodeArgs a = arg;
    void *args[] = {&a};
    hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(pages_decode_kernel<D, SPREAD>),
                                   dim3((unsigned) items), dim3(64 * kDecodeWaves), args, 0, stream);
    if (e == hipSuccess && a.split)
        e = hipLaunchKernel(reinterpret_cast<const void *>(pages_join_kernel<D, SPREAD>),
                            dim3((unsigned) (a.p.n_batch * a.p.n_heads)), dim3(D), args, 0, stream);
    return e;
}

}  // namespace

// Entries that are cut have n > c steps in ceil(n / c) < 2 n / c runs, and
// c >= units * sum n / kWantWorkgroups, so a launch has fewer than
// 2 * kWantWorkgroups partial results.
int64_t pages_work_bytes(const PagesGeom &g, int n_heads) {
    const int hc = set_heads(g, n_heads / g.n_kv);
    return (int64_t) 2 * kWantWorkgroups * hc * (g.dim + 2) * 4;
}

hipError_t launch_pages_decode(const PagesDecodeParams &p, hipStream_t stream) {
    DecodeArgs a{};
    a.p = p;
    a.group = p.n_heads / p.g.n_kv;
    const int hc = set_heads(p.g, a.group);
    a.n_hs = (a.group + hc - 1) / hc;
    a.units = p.g.n_kv * a.n_hs;
    a.append = p.k_new != nullptr;
    int64_t longest = (int64_t) p.max_pages << p.g.page_shift;
    if (p.max_len > 0 && p.max_len < longest) longest = p.max_len;
    if (p.window > 0 && p.window + kStep < longest) longest = p.window + kStep;
    const int64_t steps = (longest + kStep - 1) / kStep;
    a.split = steps > kMinRun && p.work && p.work_bytes >= pages_work_bytes(p.g, p.n_heads);
    const int64_t items = (int64_t) p.n_batch * a.units + (a.split ? 2 * kWantWorkgroups : 0);
    if (p.g.dim == 128)
        return spread(p.g, a.group) ? launch_of<128, true>(a, items, stream) : launch_of<128, false>(a, items, stream);
    return spread(p.g, a.group) ? launch_of<64, true>(a, items, stream) : launch_of<64, false>(a, items, stream);
}

}  // namespace bmo
