// pages_decode.hip -- attention of one or few rows per entry over its pages.
//
// o = sum_j p_j v_j, p = softmax(scale q . k_j) over the entry's last
// min(len, window) positions.  HBM bounds it: 2 * 18 bytes per 32 elements of
// a position's K and V against 4 operations per element and query head.
//
// One wave step takes 32 positions of one kv head: 16 bytes of K codes and of
// V codes a lane and tile of 16 (pages_layout.hpp), straight from HBM to the
// operands of the matrix instructions.  The 16 columns of the products hold
//   (head r, block b): heads of the kv head's group, up to 16 / NB of them,
//                      each column with the query of its own block only; or
//   head r:            up to 16 heads, when the group has more than 16 / NB
//                      (short calls of dim 128 take it in sets of 4 instead).
// Ragged rows (attend's calls with few of them) are taken as heads are: a
// column is a (token, head of the group) with limits of its own.
// In the first form a lane has one block's products, so the block scales cost
// one multiply a score and one a weight instead of NB each.
//
// K side: q as two fp16 parts times a power of two of its row (16-bit rows: one
// part, exactly), the codes minus 8 exact in fp16, so a query is within 2^-22 of
// each of its elements, however far apart these are, and a block's product meets
// its scale in fp32.  (Whole numbers of 23 bits of the row's largest element, 15
// for 16-bit rows, in base-256 digits on v_mfma_i32_16x16x64_i8 take 3 VALU
// instructions a dword of codes, not 9: 6% less time in fp32, 2 to 4% in 16
// bits.  But a channel 300 times the rest left the others so few bits that
// outputs were 7e-5 off in fp32 and 8e-3 in fp16.)
//
// V side: weight times V scale enters as two fp16 parts (16-bit rows: one)
// against the codes minus 8, exact in fp16, sums in fp32.  Softmax is online.
// What the weights are taken down by in a block follows the largest product of
// weight and scale there, not the largest score: it is put at 2^2 and none
// passes 2^15, so the parts are exact to 2^-22 of a product, or to 2^-27 of the
// largest, whatever scales and weights unimportant positions have.  (Taken from
// the largest score and the largest scale, a position of no weight with a scale
// 2^20 times the others' left these 2e-3 off.)  So an fp32 call is as close as
// fp32 sums; the 16-bit parts stay below the outputs' own rounding.  The four
// lanes of a column look at the products, and rescale, only when a scale passes
// four times the largest so far or a score the room that this leaves: once or
// twice a run, unless positions of little weight have scales 2^8 times the
// important ones'.  Masked positions get weight 0 by select, whatever their
// slots hold.
//
// Work: an item is a run of steps of one (entry, kv head, head set), walked
// by the NW waves of a workgroup in turn and joined in LDS.  The host knows
// how long an entry can be, not how long each is: where that is long for the
// units there are, an entry of n steps has ceil(n / c) even runs, up to a
// number of them for which the grid has workgroups (those of shorter entries
// end at once); results of entries that have several are kept in the workspace,
// with their sums and what both were taken down by, and joined by a second
// kernel in the order of the runs.
//
// Measured, graph replays, every page from HBM, 32 query heads of 128: 64
// entries of 3000 positions on 32 kv heads, fp32, 167 us, 5.3 TB/s (VALU 62% of
// the cycles; the loads alone take 136), bf16 143; 12 entries of 32000 on 8,
// bf16, 84 us, 5.3 TB/s (the loads alone 76: HBM in this page order); one entry
// of 700 on 32, fp32, 9.1 us, six steps a wave one after the other.
#include <algorithm>

#include "kernels.hpp"
#include "pages_device.hpp"

namespace bmo {

namespace {

constexpr int kStep = 32;  // positions a wave step
constexpr int kWaves = 4;  // of a workgroup, where it is not one
// How a launch is cut, see launch_units: waves of a launch that fills
// the card once (few units) and the fewest steps of a run for each of them,
// and the same for launches of several rounds.
constexpr int kFillWaves = 1024, kFillSteps = 4;
constexpr int kSplitWaves = 4096, kSplitSteps = 16;
constexpr int kMaxRuns = 128;  // of an entry
// Softmax, in log2 units: how far a score may pass the one that the weights'
// sum is taken from; and weight times V scale, which enters as fp16: where the
// largest is put, what it has to pass to be put there again when a look is
// taken, and what none passes between two looks.  A scale of zero counts as
// 2^kZeroScale, so that weights stay finite.
constexpr float kScoreLimit = 8.0f;
constexpr float kProductTop = 2.0f, kProductRaise = 4.0f, kProductLimit = 15.0f, kZeroScale = -100.0f;
constexpr int kLowUnits = 512, kLowSteps = 64;  // see there

struct DecodeArgs {
    PagesDecodeParams p;
    int group;          // query heads a kv head
    int n_hs;           // head sets a kv head (of several rows: sets of 16 or fewer rows)
    int units;          // n_kv * n_hs
    int max_runs;       // of an entry; 1: nothing is cut
    int run;            // steps up to which an entry is one run
    int append;
    FastDiv div_group;  // several rows
};

// One head set of an entry and kv head: its columns are the kv head's query
// heads from row0 on, or, of several rows, (token, head) pairs, heads fastest.
// Its columns see positions of [lo, len); all of them those of [lo_max, hi_min).
struct Unit {
    int kvh, row0, cols;
    int start, n_tok, entry_len;  // several rows
    int lo, len, lo_max, hi_min;
    int step0, n, runs;  // steps and runs
    bool whole;          // the table reaches the entry's last position
};
// Positions that the token of a multi-row entry sees end before hi_of, and
// begin with lo_of that.
__device__ __forceinline__ int hi_of(const DecodeArgs &a, const Unit &u, int tok) {
    return a.p.causal ? max(u.entry_len - u.n_tok + tok + 1, 0) : u.entry_len;
}
__device__ __forceinline__ int lo_of(const DecodeArgs &a, int hi) {
    return a.p.window > 0 && hi > a.p.window ? hi - a.p.window : 0;
}
template <bool MULTI, int HC>
__device__ __forceinline__ Unit unit_of(const DecodeArgs &a, int b, int unit) {
    Unit u{};
    const int64_t room = (int64_t) a.p.max_pages << a.p.g.page_shift;
    u.kvh = unit / a.n_hs;
    u.row0 = (unit - u.kvh * a.n_hs) * HC;
    const int given = granted_len(a.p.lens, a.p.n_new, a.p.status, b);
    u.entry_len = (int) min((int64_t) max(given, 0), room);
    u.whole = given <= room;
    if constexpr (MULTI) {
        u.start = uniform_int(a.p.q_start, b);
        const int end = uniform_int(a.p.q_start, b + 1);
        u.n_tok = u.start < 0 || end < u.start || end > a.p.n_rows ? 0 : end - u.start;
        u.cols = min(HC, u.n_tok * a.group - u.row0);
        if (u.cols <= 0) return u;
        u.hi_min = hi_of(a, u, (int) a.div_group.div((uint32_t) u.row0));
        u.len = hi_of(a, u, (int) a.div_group.div((uint32_t) (u.row0 + u.cols - 1)));
    } else {
        u.cols = min(HC, a.group - u.row0);
        u.hi_min = u.len = u.entry_len;
    }
    u.lo = lo_of(a, u.hi_min);
    u.lo_max = lo_of(a, u.len);
    u.step0 = u.lo / kStep;
    u.n = (u.len + kStep - 1) / kStep - u.step0;  // (room is at most 2^30)
    u.runs = a.max_runs == 1 ? 1 : min(max((u.n + a.run - 1) / a.run, 1), a.max_runs);
    return u;
}
// Column r of a unit: where its query and its output row are, and what it sees.
struct Column {
    int64_t q, out;
    int lo, hi;
};
template <bool MULTI, int D>
__device__ __forceinline__ Column column_of(const DecodeArgs &a, const Unit &u, int b, int r) {
    int row = b, head = u.kvh * a.group + u.row0 + r;
    Column c{0, 0, u.lo, u.len};
    if constexpr (MULTI) {
        const int tok = (int) a.div_group.div((uint32_t) (u.row0 + r));
        row = u.start + tok;
        head -= tok * a.group;
        c.hi = hi_of(a, u, tok);
        c.lo = lo_of(a, c.hi);
    }
    c.q = (int64_t) row * a.p.q_stride + (int64_t) head * D;
    c.out = ((int64_t) row * a.p.n_heads + head) * D;
    return c;
}

// Floats of a partial result of HC heads: their rows, what each block's weights
// were taken down by, and each head's score that the sum is taken from, and sum.
template <int D>
__host__ __device__ constexpr int part_floats(int hc) { return hc * (D + D / kQK + 2); }

}  // namespace

// SPREAD: the columns are (head, block); otherwise heads.  F32: the rows are
// fp32, and the query and the weights take a part more.  MULTI: an entry has
// several rows (attend's calls with few of them).
template <int D, bool SPREAD, int NW, bool F32, bool MULTI>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(SPREAD || D == 64 ? 3 : 2))) void pages_decode_kernel(DecodeArgs a) {
    constexpr int NB = D / kQK;
    constexpr int TG = kStep * D / 2048;    // groups a step
    constexpr int T = 2 / TG;               // tiles of 16 a group
    constexpr int CB = SPREAD ? NB : 1;     // columns a head
    constexpr int HC = 16 / CB;             // heads a head set
    constexpr int PB = NB / CB;             // blocks a column
    constexpr int QP = F32 ? 2 : 1;         // fp16 parts of the query
    constexpr int WP = F32 ? 2 : 1;         // parts of a weight
    constexpr int BUF = 2;  // steps resident in registers
    const PagesDecodeParams &p = a.p;
    const PagesGeom &g = p.g;

    __shared__ __align__(16) float s_out[NW][HC][D];
    __shared__ float s_mm[NW][HC][NB], s_m[NW][HC], s_l[NW][HC];

    // (16-bit kernels: known not to be fp32)
    const int type = F32 ? (int) kTypeF32 : p.type == kTypeF16 ? (int) kTypeF16 : (int) kTypeBF16;
    const int lane = threadIdx.x & 63;
    const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int col = lane & 15, oct = lane >> 4;
    const int r = col / CB, cb = col % CB;

    // items: run by run, entry by entry, unit by unit
    const int row = (int) blockIdx.x / a.units;
    const int unit = (int) blockIdx.x - row * a.units;
    const int run = row / p.n_batch, b = row - run * p.n_batch;
    const Unit un = unit_of<MULTI, HC>(a, b, unit);
    if (un.cols <= 0 || run >= un.runs) return;
    const int kvh = un.kvh;
    const Column col_r = column_of<MULTI, D>(a, un, b, r < un.cols ? r : 0);
    const int s_begin = un.step0 + (int) ((int64_t) un.n * run / un.runs);
    const int s_end = un.step0 + (int) ((int64_t) un.n * (run + 1) / un.runs);
    const int *table = p.table + (int64_t) b * p.max_pages;

    // The query's elements of the column's blocks (requested ahead of the
    // steps, so that waiting for them does not wait for those).
    pg_float4 qx[PB][2];
    {
#pragma unroll
        for (int i = 0; i < PB; ++i) {
            const int blk = SPREAD ? cb : i;
            qx[i][0] = load4(p.q, col_r.q + blk * kQK + 4 * oct, type);
            qx[i][1] = load4(p.q, col_r.q + blk * kQK + 4 * oct + 16, type);
        }
    }

    // The new token's row goes to its slot before the wave that will read it
    // starts on its steps (of several head sets each writes the same bytes).  A
    // last position past the table is in no page: its row is dropped.
    if (!MULTI && a.append && un.len > 0 && un.whole && s_end == un.step0 + un.n && wave == (s_end - 1 - s_begin) % NW) {
        constexpr int BL = 32 / NB, NE = NB, HE = NE / 2, LPD = 4 / HE;
        const int nb = lane / BL, gi = lane % BL;
        const int64_t src = (int64_t) b * p.kv_stride + kvh * D + (nb % NB) * kQK + gi * HE;
        const void *row = nb < NB ? p.k_new : p.v_new;
        float x[NE];
#pragma unroll
        for (int t = 0; t < HE; ++t) {
            x[t] = load1(row, src + t, type);
            x[HE + t] = load1(row, src + 16 + t, type);
        }
        uint16_t d16;
        const uint32_t dw = quantize_block_q4_0_lanes<BL>(x, gi, d16);
        const int pos = un.len - 1;
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
            if (gi == 0) *reinterpret_cast<uint16_t *>(grp + page_scale_offset(tb, key, nb < NB ? 0 : 1)) = d16;
        }
        __threadfence_block();
    }

    // Page ids come through the scalar cache, a step ahead of the loads that
    // need them; groups past the entry's last are taken as the last (masked).
    struct Ids {
        int id[TG];
    };
    struct Tile {
        uint4 k[TG], v[TG];
        uint4 sc[2][PB];  // K's and V's scales of the lane's four keys of a tile
        int ok;  // bit i: group i's page is there
    };
    const int last_group = max((un.len - 1) / (2048 / D), 0);
    const uint32_t page_groups = (uint32_t) g.n_kv << g.group_shift, head_groups = (uint32_t) kvh << g.group_shift;
    auto ids_of = [&](int step, Ids &t) {
#pragma unroll
        for (int i = 0; i < TG; ++i)
            t.id[i] = uniform_int(table, min(step * TG + i, last_group) >> g.group_shift);
    };
    auto load = [&](int step, const Ids &ids, Tile &t) {
        t.ok = 0;
#pragma unroll
        for (int i = 0; i < TG; ++i) {
            const int grp = min(step * TG + i, last_group);
            const bool ok = (unsigned) ids.id[i] < (unsigned) g.n_pages;
            t.ok |= ok ? 1 << i : 0;
            // (a layer of 2^32 groups would be 10 TB)
            const uint32_t at_group = (uint32_t) (ok ? ids.id[i] : 0) * page_groups + head_groups +
                                      ((uint32_t) grp & ((1u << g.group_shift) - 1));
            const uint8_t *at = p.base + (uint64_t) at_group * (uint32_t) kGroupBytes;
            t.k[i] = stream16(at + lane * 16);
            t.v[i] = stream16(at + kVCodeOff + lane * 16);
#pragma unroll
            for (int u = 0; u < T; ++u)
#pragma unroll
                for (int j = 0; j < PB; ++j)
                    t.sc[i * T + u][j] =
                        stream16(at + page_scale_offset(u * NB + (SPREAD ? cb : j), 4 * oct, 0));
        }
    };
    const int first = s_begin + wave, last = max(s_end - 1, s_begin);
    // (unconditional, so that the counts of loads in flight are known: an
    // entry without positions reads some page and uses nothing of it)
    Tile buf[BUF];
    Ids ids[BUF];
#pragma unroll
    for (int j = 0; j < BUF; ++j) ids_of(min(first + j * NW, last), ids[j]);
#pragma unroll
    for (int j = 0; j < BUF - 1; ++j) load(min(first + j * NW, last), ids[j], buf[j]);
    __builtin_amdgcn_sched_barrier(0);

    // The query as fp16 parts, times a power of two of its row (of every block;
    // zero outside the column's own when columns are blocks); what the products
    // make of it is multiplied by sq.
    pg_half8 qp[QP][NB];
    float sq;
    {
        float amax = 0.0f, bad = 0.0f;
        float x[PB][8];
#pragma unroll
        for (int i = 0; i < PB; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = octet_elem(0, j);  // 0..3, 16..19
                x[i][j] = r >= un.cols ? 0.0f : e < 16 ? qx[i][0][e & 3] : qx[i][1][e & 3];
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
        // (rows below 2^-90 count as zeros: their scores do)
        const int ex = max(__builtin_amdgcn_frexp_expf(amax), -90);
        // (never 0: masked scores are -inf times it)
        sq = bad == 0.0f ? fmaxf(__builtin_amdgcn_ldexpf(p.qscale, ex - 15), 1e-37f) : __builtin_nanf("");
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float y = __builtin_amdgcn_ldexpf(x[SPREAD ? 0 : blk][j], 15 - ex);
                if (SPREAD && blk != cb) y = 0.0f;
#pragma unroll
                for (int i = 0; i < QP; ++i) {
                    const _Float16 h = (_Float16) y;
                    qp[i][blk][j] = h;
                    y -= (float) h;
                }
            }
    }

    // In log2 units, m is the column's largest score (lazily: none has passed it
    // by kScoreLimit) and mm what its weights are taken down by in each block:
    // the largest weight times V scale there, less kProductTop, lazily too.  No
    // raw score has passed mt and no scale dt (fp16 bits, four times the largest
    // so far), which together keep the products below kProductLimit.
    // to_m = 2^(mm - m) of the first block; l is the sum of this lane's weights
    // from m.
    float m = kPagesFloor, mt = -INFINITY, to_m = 1.0f, l = 0.0f;
    float mm[PB];
    uint32_t dt[PB];
    pg_float4 acc[NB][2];
    const pg_float4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i][0] = acc[i][1] = zero;
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        mm[i] = kPagesFloor;
        dt[i] = 0;
    }
    const Patterns pat;
    float minus_one = -1.0f;  // not known to be: a mixed fma takes it
    asm volatile("" : "+v"(minus_one));

    auto word = [](const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; };
    // x times the scale of key i of a tile, x as it is where y is 0 (one mixed
    // fma, which takes the scale as fp16)
    auto times_scale = [&](float x, const uint4 &v, int which, int i, float y) {
        const pg_half2 h = __builtin_bit_cast(pg_half2, word(v, 2 * which + (i >> 1)));
        return __builtin_fmaf(x, (float) (i & 1 ? h.y : h.x), y);
    };

    auto compute = [&](int step, Tile &t) {
        float s[8];  // scores, to be multiplied by sq
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = 0.0f;
        pg_float4 d[2] = {zero, zero};
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
            pg_half8 kc[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) kc[u] = k_octet(word(t.k[u / T], (u % T) * NB + blk), pat);
            if (!SPREAD) d[0] = d[1] = zero;
#pragma unroll
            for (int i = 0; i < QP; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u) d[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kc[u], qp[i][blk], d[u], 0, 0, 0);
            if (!SPREAD)
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] = times_scale(d[i >> 2][i & 3], t.sc[i >> 2][SPREAD ? 0 : blk], 0, i & 3, s[i]);
        }
        if constexpr (SPREAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float x = times_scale(d[i >> 2][i & 3], t.sc[i >> 2][0], 0, i & 3, 0.0f);
                x += pg_dpp<0xB1>(x);
                if constexpr (NB == 4) x += pg_dpp<0x4E>(x);
                s[i] = x;
            }
        }
        if (!(step * kStep >= un.lo_max && step * kStep + kStep <= un.hi_min && t.ok == (1 << TG) - 1)) {
            // some position is not visible: score -inf, V scale 0
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int u = i >> 2;
                const int pos = step * kStep + u * 16 + 4 * oct + (i & 3);
                const bool ok = pos >= col_r.lo && pos < col_r.hi && ((t.ok >> (u / T)) & 1);
                s[i] = ok ? s[i] : -INFINITY;
                const uint32_t keep = ok ? 0xFFFFFFFFu : i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
#pragma unroll
                for (int j = 0; j < PB; ++j) {
                    if ((i & 3) < 2)
                        t.sc[u][j].z &= keep;
                    else
                        t.sc[u][j].w &= keep;
                }
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        bool raise = mx > mt;
        uint32_t dx[PB];  // the largest scale's fp16 bits
#pragma unroll
        for (int j = 0; j < PB; ++j) {
            typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
            auto mag = [](uint32_t x) { return __builtin_bit_cast(ushort2_t, x & 0x7FFF7FFFu); };
            const ushort2_t top = __builtin_elementwise_max(
                __builtin_elementwise_max(mag(t.sc[0][j].z), mag(t.sc[0][j].w)),
                __builtin_elementwise_max(mag(t.sc[1][j].z), mag(t.sc[1][j].w)));
            dx[j] = max((uint32_t) top.x, (uint32_t) top.y);
            raise = raise || dx[j] > dt[j];
        }
        if (__any(raise)) {
            // (what is changed follows from the column's own scores and scales,
            // whichever asked, so that no column's rounding depends on another's)
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            bool own = mx > mt;
            float top[PB];  // the largest weight, from the largest score here, times scale
            const float most = mx * sq;
            {
                float e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sq, -most));
#pragma unroll
                for (int j = 0; j < PB; ++j) {
                    top[j] = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        // (not known to be the words below, whose conversions
                        // would then be made up here for both)
                        uint32_t d = word(t.sc[i >> 2][j], 2 + ((i & 2) >> 1));
                        asm volatile("" : "+v"(d));
                        const pg_half2 d2 = __builtin_bit_cast(pg_half2, d);
                        top[j] = fmaxf(top[j], __builtin_fabsf(e[i] * (float) d2.x));
                        top[j] = fmaxf(top[j], __builtin_fabsf(e[i + 1] * (float) d2.y));
                    }
                    top[j] = fmaxf(top[j], __shfl_xor(top[j], 16));
                    top[j] = fmaxf(top[j], __shfl_xor(top[j], 32));
                    dx[j] = max(dx[j], (uint32_t) __shfl_xor((int) dx[j], 16));
                    dx[j] = max(dx[j], (uint32_t) __shfl_xor((int) dx[j], 32));
                    own = own || dx[j] > dt[j];
                }
            }
            const float m_old = m;
            m = own ? fmaxf(m, most) : m;
            l *= __builtin_amdgcn_exp2f(m_old - m);
            float alpha[PB], room = m + kScoreLimit;
#pragma unroll
            for (int j = 0; j < PB; ++j) {
                // (infinity counts as the largest scale: what it reaches is not
                // finite, and nothing else is shifted for it)
                const float at = most + fmaxf(__builtin_amdgcn_logf(fminf(top[j], 65504.0f)), kZeroScale);
                const float mm_old = mm[j];
                mm[j] = own && at > mm_old + kProductRaise ? at - kProductTop : mm_old;
                alpha[j] = __builtin_amdgcn_exp2f(mm_old - mm[j]);
                if (dx[j] > dt[j]) dt[j] = min(dx[j] + 0x800u, 0x7C00u);  // four times the scale
                room = fminf(room, mm[j] + kProductLimit - __builtin_amdgcn_logf(fminf(f16_bits_to_f32(dt[j]), 65504.0f)));
            }
            if (own) mt = room / sq;
            to_m = __builtin_amdgcn_exp2f(mm[0] - m);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                acc[i][0] *= alpha[SPREAD ? 0 : i];
                acc[i][1] *= alpha[SPREAD ? 0 : i];
            }
        }
        // weights of the first block; the other blocks' come by a factor
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sq, -mm[0]));
            l = __builtin_fmaf(w[i], to_m, l);
        }
#pragma unroll
        for (int j = 0; j < PB; ++j) {
            const float f = j == 0 ? 1.0f : __builtin_amdgcn_exp2f(mm[0] - mm[j]);
            // keys 0, 2, 1, 3 of each tile's quad, as the masks leave the codes
            pg_half8 wp[WP];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const int a0 = (i & 4) + ((i & 2) >> 1), a1 = a0 + 2;
                float x = w[a0], y = w[a1];
                if (j > 0) {
                    x *= f;
                    y *= f;
                }
                x = times_scale(x, t.sc[a0 >> 2][j], 1, a0 & 3, 0.0f);
                y = times_scale(y, t.sc[a1 >> 2][j], 1, a1 & 3, 0.0f);
                const pg_half2 h = {(_Float16) x, (_Float16) y};
                wp[0][i] = h.x;
                wp[0][i + 1] = h.y;
                if constexpr (WP == 2) {
                    wp[1][i] = (_Float16) __builtin_fmaf((float) h.x, minus_one, x);
                    wp[1][i + 1] = (_Float16) __builtin_fmaf((float) h.y, minus_one, y);
                }
            }
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                if (!SPREAD && blk != j) continue;
                const uint32_t x0 = word(t.v[0], blk), y0 = x0 >> 8;
                const uint32_t x1 = word(t.v[1 / T], (1 % T) * NB + blk), y1 = x1 >> 8;
                const pg_half2 a = codes_lo(x0, pat), b2 = codes_lo(y0, pat), c = codes_lo(x1, pat), d2 = codes_lo(y1, pat);
                const pg_half8 vl = {a.x, a.y, b2.x, b2.y, c.x, c.y, d2.x, d2.y};
                const pg_half2 e = codes_hi(x0, pat), f2 = codes_hi(y0, pat), h = codes_hi(x1, pat), i2 = codes_hi(y1, pat);
                const pg_half8 vh = {e.x, e.y, f2.x, f2.y, h.x, h.y, i2.x, i2.y};
#pragma unroll
                for (int k = 0; k < WP; ++k) {
                    acc[blk][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, wp[k], acc[blk][0], 0, 0, 0);
                    acc[blk][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, wp[k], acc[blk][1], 0, 0, 0);
                }
            }
        }
    };

    // Steps first, first + NW, ...: at the top of a pass buf[u] holds the u-th
    // next step, u < BUF - 1, and ids[BUF - 1] the pages of the one after.
    const int n_steps = (s_end - first + NW - 1) / NW;
    int i = 0;
    for (; i + BUF <= n_steps; i += BUF) {
#pragma unroll
        for (int u = 0; u < BUF; ++u) {
            load(min(first + (i + u + BUF - 1) * NW, last), ids[BUF - 1], buf[(u + BUF - 1) % BUF]);
            ids_of(min(first + (i + u + BUF) * NW, last), ids[BUF - 1]);
            compute(first + (i + u) * NW, buf[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < BUF - 1; ++u)
        if (i + u < n_steps) compute(first + (i + u) * NW, buf[u]);
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
    if (oct == 0) {
#pragma unroll
        for (int j = 0; j < PB; ++j) s_mm[wave][r][SPREAD ? cb : j] = mm[j];
        if (cb == 0) {
            s_m[wave][r] = m;
            s_l[wave][r] = l;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < un.cols * D; i += 64 * NW) {
        const int rr = i / D, e = i % D, blk = e / kQK;
        float M = s_m[0][rr], MM = s_mm[0][rr][blk];
#pragma unroll
        for (int w = 1; w < NW; ++w) {
            M = fmaxf(M, s_m[w][rr]);
            MM = fmaxf(MM, s_mm[w][rr][blk]);
        }
        const float base = un.runs == 1 ? M : MM;
        float L = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            L = __builtin_fmaf(__builtin_amdgcn_exp2f(s_m[w][rr] - M), s_l[w][rr], L);
            o = __builtin_fmaf(__builtin_amdgcn_exp2f(s_mm[w][rr][blk] - base), s_out[w][rr][e], o);
        }
        if (un.runs == 1) {
            const Column c = column_of<MULTI, D>(a, un, b, rr);
            // (a row that sees nothing is zeros whatever its query holds)
            store1(p.out, c.out + e, L > 0.0f ? o * (1.0f / L) : c.hi > c.lo ? o * 0.0f : 0.0f, type);
        } else {
            float *dst = p.work + (int64_t) blockIdx.x * part_floats<D>(HC);
            dst[rr * D + e] = o;
            if (e % kQK == 0) dst[HC * D + rr * NB + blk] = MM;
            if (e == 0) {
                dst[HC * (D + NB) + rr] = M;
                dst[HC * (D + NB + 1) + rr] = L;
            }
        }
    }
}

// Joins the runs of the entries that were cut: a workgroup takes one column,
// its waves every fourth run.
template <int D, bool SPREAD, bool MULTI>
__global__ __launch_bounds__(256) void pages_join_kernel(DecodeArgs a) {
    constexpr int HC = SPREAD ? 16 / (D / kQK) : 16;
    constexpr int NB = D / kQK, E = D / 64, NW = 4;
    const PagesDecodeParams &p = a.p;
    __shared__ float s_w[kMaxRuns][NB];
    __shared__ float s_o[NW][D];
    const int row = (int) blockIdx.x / HC, rr = (int) blockIdx.x - row * HC;
    const int b = row / a.units, unit = row - b * a.units;
    const Unit un = unit_of<MULTI, HC>(a, b, unit);
    if (rr >= un.cols || un.runs == 1) return;
    const int runs = un.runs;
    const int64_t stride = (int64_t) p.n_batch * a.units * part_floats<D>(HC);
    const float *src = p.work + ((int64_t) b * a.units + unit) * part_floats<D>(HC);
    const int lane = threadIdx.x & 63, wave = (int) threadIdx.x >> 6;
    // lane e has elements e, e + 64 of the head, of blocks e / 32, + 2
    float o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    // block `wave`: every run's share of the whole, a run a lane
    if (wave < NB) {
        const float *q = src + HC * D + rr * NB + wave, *ml = src + HC * (D + NB) + rr;
        float M = kPagesFloor, L = 0.0f;
        for (int i = lane; i < runs; i += 64) M = fmaxf(M, ml[i * stride]);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
        for (int i = lane; i < runs; i += 64) {
            s_w[i][wave] = __builtin_amdgcn_exp2f(q[i * stride] - M);
            L = __builtin_fmaf(__builtin_amdgcn_exp2f(ml[i * stride] - M), ml[i * stride + HC], L);
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) L += __shfl_xor(L, d);
        const float inv = L > 0.0f ? 1.0f / L : L * 0.0f;  // (NaN stays)
        for (int i = lane; i < runs; i += 64) s_w[i][wave] *= inv;
    }
    __syncthreads();
#pragma unroll 8
    for (int i = wave; i < runs; i += NW)
#pragma unroll
        for (int e = 0; e < E; ++e)
            o[e] = __builtin_fmaf(s_w[i][2 * e + lane / kQK], src[i * stride + rr * D + e * 64 + lane], o[e]);
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[wave][e * 64 + lane] = o[e];
    __syncthreads();
    if (threadIdx.x < D) {
        const int e = threadIdx.x;
        const Column c = column_of<MULTI, D>(a, un, b, rr);
        store1(p.out, c.out + e, c.hi > c.lo ? (s_o[0][e] + s_o[1][e]) + (s_o[2][e] + s_o[3][e]) : 0.0f, p.type);
    }
}

namespace {

// Columns are (head, block) while there are that few heads (or rows and heads).
bool spread(const PagesGeom &g, int heads) { return heads <= 16 / (g.dim / kQK); }
int set_heads(const PagesGeom &g, int heads) { return spread(g, heads) ? 16 / (g.dim / kQK) : 16; }
int64_t part_bytes(const PagesGeom &g, int hc) {
    return (int64_t) (g.dim == 128 ? part_floats<128>(hc) : part_floats<64>(hc)) * 4;
}
// Workgroups of a launch whose long entries are cut (sets of 16 of dim 128
// leave room for half as many at a time).
int64_t split_workgroups(const PagesGeom &g, int hc) {
    return kSplitWaves / kWaves / (hc == 16 && g.dim == 128 ? 2 : 1);
}

template <int D, bool SPREAD, bool MULTI>
const void *kernel_of(int nw, int type) {
#define BMO_DECODE(NW_, F32_) reinterpret_cast<const void *>(pages_decode_kernel<D, SPREAD, NW_, F32_, MULTI>)
    if constexpr (!MULTI)
        if (type == kTypeF32) return nw == 1 ? BMO_DECODE(1, true) : BMO_DECODE(kWaves, true);
    return nw == 1 ? BMO_DECODE(1, false) : BMO_DECODE(kWaves, false);
#undef BMO_DECODE
}

template <int D, bool SPREAD, bool MULTI>
hipError_t launch_of(const DecodeArgs &arg, int nw, hipStream_t stream) {
    constexpr int HC = SPREAD ? 16 / (D / kQK) : 16;
    DecodeArgs a = arg;
    void *args[] = {&a};
    const int64_t units = (int64_t) a.p.n_batch * a.units;
    hipError_t e = hipLaunchKernel(kernel_of<D, SPREAD, MULTI>(nw, a.p.type), dim3((unsigned) (units * a.max_runs)),
                                   dim3(64 * nw), args, 0, stream);
    if (e == hipSuccess && a.max_runs > 1)
        e = hipLaunchKernel(reinterpret_cast<const void *>(pages_join_kernel<D, SPREAD, MULTI>),
                            dim3((unsigned) (units * HC)), dim3(256), args, 0, stream);
    return e;
}

// Shape of a launch, from its units and the steps that its longest entry can
// have.  us a launch in a graph, pages from HBM, dim 128, 32 heads:
//   one wave a unit or four, fp32:  2048 units x 16 steps 38 / 42, 8192 x 7
//     56 / 87, 1024 x 16 19.7 / 19.2; 2048 x 32 63 / 62, x 63 116 / 109, of 3 to
//     63 steps 85 / 65 (a long unit's one wave is the last to end).
//   more than 4 heads (rows) a kv head in sets of 16 or of 4, while these are no
//     more than two workgroups a CU and 64 steps long, dim 128 (whose sets of
//     16 hold two waves a SIMD and multiply every head with every block):  one
//     entry, 8 heads on each of 4 kv heads, fp32, 150 positions 8.3 / 6.1, 600
//     11.8 / 8.5, 1500 17.1 / 13.1, 12 entries of 1500 18.5 / 14.3; rows of one
//     entry of 32 kv heads, 600 positions, bf16, 12 rows 13.1 / 8.9, 64 rows
//     14.8 / 12.4; past the limits 96 sets x 125 steps 20.8 / 23.3, 960 x 19
//     20.4 / 23.1.
//   long entries cut for 256 workgroups (runs of at least 4 steps a wave), for
//     1024 (of 16), or not; the rule takes the more runs of the first two:  fp32,
//     32 units x 94 steps 12.8 / 23 / 23, x 250 15.8 / 24.4 / 52, 8 x 1000
//     16.6 / 23.7 / 192; bf16, 96 units of 62 to 1000 steps 95 / 61 / 169.  Fewer
//     steps a wave lose:  fp32, 256 x 32 in two runs or one 15.7 / 11.0, 512 x 32
//     25.2 / 17.3.  Sets of 16 rows, bf16, cut for 1024 workgroups, for 512, or
//     not:  132 x 204 steps 52 / 46 / 56, 128 x 500 79 / 71 / 125.
//   runs that load the CUs evenly, bf16:  128 units of up to 250 steps in 3 or 2
//     runs 33.5 / 31.7, 24 of up to 1000 in 15 or 10 29.6 / 26.9, 80 of up to 282
//     in 4 or 3 28.8 / 25.6; past two workgroups a CU it hardly matters (96 of 62
//     to 1000 in 10 or 8 61.0 / 60.0, all of 1000 83 / 81).
template <bool MULTI>
hipError_t launch_units(const PagesDecodeParams &p, int heads, hipStream_t stream) {
    DecodeArgs a{};
    a.p = p;
    a.group = p.n_heads / p.g.n_kv;
    a.div_group = make_fastdiv((uint32_t) a.group);
    a.append = p.k_new != nullptr;
    a.max_runs = 1;
    int64_t longest = (int64_t) p.max_pages << p.g.page_shift;
    if (p.max_len > 0 && p.max_len < longest) longest = p.max_len;
    const int64_t seen = (int64_t) p.window + (MULTI ? p.max_rows : 0) + kStep;
    if (p.window > 0 && seen < longest) longest = seen;
    const int64_t steps = (longest + kStep - 1) / kStep;
    const int narrow = 16 / (p.g.dim / kQK);
    const bool low = p.g.dim == 128 && steps <= kLowSteps &&
                     (int64_t) p.n_batch * p.g.n_kv * ((heads + narrow - 1) / narrow) <= kLowUnits;
    const int hc = low ? narrow : set_heads(p.g, heads);
    a.n_hs = (heads + hc - 1) / hc;
    a.units = p.g.n_kv * a.n_hs;
    const int64_t units = (int64_t) p.n_batch * a.units;
    const int nw = units >= 1024 && steps <= 24 ? 1 : kWaves;
    if (nw == kWaves && p.work) {
        const int64_t room = p.work_bytes / part_bytes(p.g, hc) / units;  // runs that it holds
        const int64_t fill = std::min<int64_t>(kFillWaves / kWaves / units, steps / (kFillSteps * kWaves));
        const int64_t split = std::min<int64_t>(split_workgroups(p.g, hc) / units, steps / (kSplitSteps * kWaves));
        const int64_t most = std::min({std::max(fill, split), room, (int64_t) kMaxRuns});
        int64_t runs = std::max<int64_t>(most, 1);
        if (units * runs <= 512)  // as many as load 256 CUs most evenly
            for (int64_t r = runs - 1; r > 0; --r)
                if ((units * r + 255) / 256 * runs < (units * runs + 255) / 256 * r) runs = r;
        if (runs > 1) {
            a.max_runs = (int) runs;
            a.run = (int) ((steps + runs - 1) / runs);
        }
    }
    if (p.g.dim == 128)
        return hc == 16 ? launch_of<128, false, MULTI>(a, nw, stream) : launch_of<128, true, MULTI>(a, nw, stream);
    return hc == 16 ? launch_of<64, false, MULTI>(a, nw, stream) : launch_of<64, true, MULTI>(a, nw, stream);
}

}  // namespace

// Every workgroup that a launch of sets of 16 may have (sets of fewer have
// smaller results).
int64_t pages_work_bytes(const PagesGeom &g) { return split_workgroups(g, 16) * part_bytes(g, 16); }

hipError_t launch_pages_decode(const PagesDecodeParams &p, hipStream_t stream) {
    return launch_units<false>(p, p.n_heads / p.g.n_kv, stream);
}

hipError_t launch_pages_few_rows(const PagesDecodeParams &p, hipStream_t stream) {
    return launch_units<true>(p, p.max_rows * (p.n_heads / p.g.n_kv), stream);
}

}  // namespace bmo
