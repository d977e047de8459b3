// pages_attend.hip -- attention of ragged query rows over their entries' pages:
// prompt chunks (causal) or cross attention to an encoder's states.
//
// o_i = sum_j p_ij v_j, p_i = softmax(scale q_i . k_j) over the positions row i
// sees.  4 rows keys head_dim operations a query head against the pages' bytes
// once per 128 rows: with long chunks the matrix cores and the exponentials
// bound it, not HBM.
//
// A workgroup of four waves takes 128 rows of one (entry, kv head), 32 a wave.
// A row is a (token, query head of the kv head's group), heads fastest, so
// that grouped queries fill a tile from few tokens.  Positions pass in stages
// of 64: the waves load the groups of the next stage while the present one is
// multiplied, then dequantize them into the other of two LDS buffers, K as
// [key][element] and V as [element][key] (pages_layout.hpp gives four keys of
// a V column to a lane, so nothing is transposed); one barrier a stage.
// S^T = K Q^T with v_mfma_f32_32x32x16_f16 leaves 8 + 8 keys of one row in a
// lane, which is the operand of the next product, O^T = V^T P^T, once V's
// keys stand in the same order: the weights never leave the registers.  Both
// products read their LDS operands eight matrix instructions ahead.
// Row padding: K rows 16 bytes and V rows 16 bytes longer than their data, so
// that 16 lanes reading 16 bytes each from consecutive rows meet every LDS
// bank once.
//
// Measured in a graph, 32 query heads on 8 of 128, bf16: eight chunks of 200 to
// 1024 rows over 300 to 4000 positions 325 us, 755 TFLOP/s; of 1024 rows that all
// see 4096 positions 638 us, 862 TFLOP/s (a large library product reaches 1211).
// Bound by the card's power: with such full tiles the clock stands at 2.02 GHz
// (1.5 in that library product), with 53% of a SIMD's cycles VALU (exponentials,
// dequantizing, masks) and 38% matrix instructions, two waves a SIMD (46% and
// 32% in the eight chunks, whose last workgroups leave CUs idle).  So less work
// helps and another order of it does not: dequantizing and the weights between
// the matrix instructions, or without the LDS reads, run as long; without
// dequantizing 20% less.  Eight waves a workgroup (half the dequantizing a row)
// win 4% with full tiles of one length and lose 10% with ragged ones; stages of
// 32 with three waves a SIMD are 16% slower, scores one stage ahead of the
// weights 5%.
//
// Precision: V enters as (code - 8) * d rounded to fp16, the weights as fp16
// (with all its bits down to 2^-21 of the row's largest), sums in fp32; q enters
// scaled by its row's own power of two, exactly.  K does as V for bf16 rows,
// whose own rounding (1.7e-3) hides it.  For fp16 rows (2.1e-4) it would show
// where scores are large (3.2e-4 in all, and more the larger they are), so K's
// codes enter exactly and its scales meet the products of each block in fp32:
// 754 us where 638 are, see above.  V (and K of bf16 rows) must lie in fp16's
// range; a V block whose scale brings it past makes the rows that see it NaN in
// that block and leaves the others.
#include <algorithm>

#include "kernels.hpp"
#include "pages_device.hpp"

namespace bmo {

namespace {

typedef float pg_float16 __attribute__((ext_vector_type(16)));
typedef _Float16 pg_half4 __attribute__((ext_vector_type(4)));

constexpr int kAttendWaves = 4;
constexpr int kWaveRows = 32;
constexpr int kTileRows = kWaveRows * kAttendWaves;
constexpr int kStage = 64;  // positions a stage
// Softmax, in log2 units: the running maximum is raised when a score passes it
// by kLazy, and its weight is 2^kTop, so that none passes 2^15 and fp16 holds
// weights down to 2^-21 of it with all their bits (those of 2^-32 are still
// some).  4 and 11 would hold 2^-25, for 2 to 3% more time in raising it.
constexpr float kLazy = 8.0f, kTop = 7.0f;

struct AttendArgs {
    PagesAttendParams p;
    int group;          // query heads a kv head
    int max_rows;       // of an entry
    FastDiv div_group;
};

// The entry and first row of tile `tile` of `size` rows; false past the last.
struct RowTile {
    int b, row0, rows;  // row0 and rows count (token, head) pairs
};
__device__ __forceinline__ int entry_rows(const AttendArgs &a, int b) {
    const int s = a.p.q_start[b], e = a.p.q_start[b + 1];
    return s < 0 || e < s || e > a.p.n_rows ? 0 : e - s;
}
// Tiles of up to 64 entries come longest entry first, and an entry's from its
// last rows on: the workgroups that run longest start first.
__device__ __forceinline__ bool find_tile(const AttendArgs &a, int tile, int size, int lane, RowTile &t) {
    int before = 0;
    for (int b0 = 0; b0 < a.p.n_batch; b0 += 64) {
        int b = b0 + lane;
        // (an entry with more rows than the call was said to have takes no
        // tile from the others)
        int rows = b < a.p.n_batch ? min(entry_rows(a, b), a.max_rows) * a.group : 0;
        if (a.p.n_batch <= 64) {
            const int key = rows > 0 ? max(a.p.lens[b], 0) : -1;
            int rank = 0;
            for (int j = 0; j < 64; ++j) {
                const int other = __builtin_amdgcn_readlane(key, j);
                rank += other > key || (other == key && j < lane) ? 1 : 0;
            }
            b = __builtin_amdgcn_ds_permute(rank * 4, b);
            rows = __builtin_amdgcn_ds_permute(rank * 4, rows);
        }
        const int tiles = (rows + size - 1) / size;
        const int upto = wave_prefix(tiles, lane) + before;
        const uint64_t past = __ballot(upto > tile);
        if (past) {
            const int l = __ffsll((unsigned long long) past) - 1;
            t.b = __builtin_amdgcn_readlane(b, l);
            t.rows = __builtin_amdgcn_readlane(rows, l);
            t.row0 = (__builtin_amdgcn_readlane(upto, l) - 1 - tile) * size;
            // (always so, unless q_start is no running sum)
            return t.b < a.p.n_batch && (unsigned) t.row0 < (unsigned) t.rows;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// Whether 8 times a scale (fp16 bits) lies in fp16's range.
__device__ __forceinline__ bool in_range(uint32_t h) { return (h & 0x7FFFu) < 0x7000u; }

}  // namespace

// FINE (fp16 rows): K's codes enter as they are and its scales meet the
// products of each block in fp32.
template <int D, bool FINE>
__global__ __launch_bounds__(64 * kAttendWaves) __attribute__((amdgpu_waves_per_eu(2))) void pages_attend_kernel(AttendArgs a) {
    constexpr int NW = kAttendWaves;
    constexpr int NB = D / kQK;
    constexpr int G = 2048 / D;            // keys a group
    constexpr int NG = kStage / G;         // groups a stage
    constexpr int KROW = D + 8;            // halves of a K row
    constexpr int VROW = kStage + 8;       // halves of a V row
    constexpr int KK = D / 16;             // products of 16 elements a key
    constexpr int WPG = NW / NG;           // waves that fill a group
    static_assert(WPG == 1 || WPG == 2, "every wave fills, all groups are filled");
    const PagesAttendParams &p = a.p;
    const PagesGeom &g = p.g;

    __shared__ __align__(16) _Float16 s_k[2][kStage * KROW];
    __shared__ __align__(16) _Float16 s_v[2][D * VROW];
    __shared__ __align__(8) _Float16 s_d[FINE ? 2 : 1][FINE ? NB * kStage : 4];  // K's scales, [block][key]
    __shared__ int s_flag[2][NW];  // nonzero: a bad page, or a V scale out of range

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int n = lane & 31, half = lane >> 5;

    const int tile = (int) blockIdx.x / g.n_kv;
    const int kvh = (int) blockIdx.x - tile * g.n_kv;
    RowTile rt;
    if (!find_tile(a, tile, kTileRows, lane, rt)) return;
    const int b = rt.b;
    const int start = p.q_start[b];
    const int n_tok = entry_rows(a, b);
    const int64_t room = (int64_t) p.max_pages << g.page_shift;
    const int len = (int) min((int64_t) max(granted_len(p.lens, nullptr, p.status, b), 0), room);
    const int *table = p.table + (int64_t) b * p.max_pages;

    // This lane's row, and the positions [lo, hi) it sees.
    const int rr = rt.row0 + wave * kWaveRows + n;
    const bool row_ok = rr < rt.rows;
    const int tok = (int) a.div_group.div((uint32_t) (row_ok ? rr : rt.row0));
    const int head = kvh * a.group + (row_ok ? rr : rt.row0) - tok * a.group;
    auto last_of = [&](int t) { return p.causal ? len - n_tok + t : len - 1; };  // can be negative
    auto low_of = [&](int t) { return p.window > 0 ? max(last_of(t) - p.window + 1, 0) : 0; };
    const int hi = row_ok ? max(last_of(tok) + 1, 0) : 0;
    const int lo = low_of(tok);
    // The workgroup's, and the wave's least and greatest (the same on every lane).
    const int tok_first = (int) a.div_group.div((uint32_t) rt.row0);
    const int tok_last = (int) a.div_group.div((uint32_t) (min(rt.row0 + kTileRows, rt.rows) - 1));
    const int wg_hi = max(last_of(tok_last) + 1, 0);
    const int stage0 = low_of(tok_first) / kStage;
    const int n_stage = (wg_hi + kStage - 1) / kStage;  // past the last
    const int w_row0 = rt.row0 + wave * kWaveRows;
    const bool w_any = w_row0 < rt.rows;
    const bool w_full = w_row0 + kWaveRows <= rt.rows;
    const int w_tok0 = (int) a.div_group.div((uint32_t) min(w_row0, rt.rows - 1));
    const int w_tok1 = (int) a.div_group.div((uint32_t) (min(w_row0 + kWaveRows, rt.rows) - 1));
    const int w_hi_min = max(last_of(w_tok0) + 1, 0), w_hi_max = max(last_of(w_tok1) + 1, 0);
    const int w_lo_min = low_of(w_tok0), w_lo_max = low_of(w_tok1);

    // ---- filling: WPG waves take a group of a stage, alone K and V, two one each ----
    constexpr int TB = 4;  // (tile, block) pairs of a group
    const int my_group = wave / WPG;
    const bool do_k = WPG == 1 || wave % WPG == 0;
    const bool do_v = WPG == 1 || !do_k;
    const int key16 = lane & 15, oct = lane >> 4;
    const Patterns pat;
    uint32_t kw[TB], vw[TB], kd[TB];
    uint2 vd[TB];
    int flag = 0;
    const int last_group = max((len - 1) / G, 0);
    auto id_of = [&](int stage) { return uniform_int(table, min(stage * NG + my_group, last_group) >> g.group_shift); };
    auto fetch = [&](int stage, int id) {
        const int grp = min(stage * NG + my_group, last_group);
        const bool ok = (unsigned) id < (unsigned) g.n_pages;
        const uint8_t *at = p.base + (int64_t) (ok ? id : 0) * g.page_bytes +
                            (((int64_t) kvh << g.group_shift) + (grp & ((1 << g.group_shift) - 1))) * kGroupBytes;
        flag = ok ? 0 : 1;
        auto codes = [&](const uint8_t *c, uint32_t (&w)[TB]) {
            const uint4 x = *reinterpret_cast<const uint4 *>(c + lane * 16);
            w[0] = x.x;
            w[1] = x.y;
            w[2] = x.z;
            w[3] = x.w;
        };
        if (do_k) {
            codes(at, kw);
#pragma unroll
            for (int i = 0; i < TB; ++i)
                kd[i] = *reinterpret_cast<const uint16_t *>(at + page_scale_offset(i, key16, 0));
        }
        if (do_v) {
            codes(at + kVCodeOff, vw);
#pragma unroll
            for (int i = 0; i < TB; ++i)
                vd[i] = *reinterpret_cast<const uint2 *>(at + page_scale_offset(i, 4 * oct, 1));
        }
    };
    auto fill = [&](int buf) {
        if (do_k) {
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                // row of the key, octet `oct` of the block
                const int t = i / NB, blk = i % NB;
                const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t) kd[i]);
                pg_half8 x = k_octet(kw[i], pat);
                const int key = my_group * G + t * 16 + key16;
                if constexpr (FINE) {
                    if (oct == 0) s_d[buf][blk * kStage + key] = d;
                } else {
                    x *= pg_half8{d, d, d, d, d, d, d, d};
                }
                *reinterpret_cast<pg_half8 *>(&s_k[buf][key * KROW + (blk * 4 + oct) * 8]) = x;
            }
        }
        if (do_v) {
            // 16 times a scale out of range is past 2^17, which no sum of the
            // others in range brings back (sums past the range on their own,
            // scales beyond 500, only cost the look below)
            const _Float16 times = (_Float16) 16.0f;
            pg_half2 check = {(_Float16) 0.0f, (_Float16) 0.0f};
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                check = __builtin_elementwise_fma(__builtin_bit_cast(pg_half2, vd[i].x), pg_half2{times, times}, check);
                check = __builtin_elementwise_fma(__builtin_bit_cast(pg_half2, vd[i].y), pg_half2{times, times}, check);
            }
            check *= pg_half2{(_Float16) 0.0f, (_Float16) 0.0f};
            const bool odd = !(check.x == (_Float16) 0.0f && check.y == (_Float16) 0.0f);
            if (__any(odd)) {  // rare: such blocks are taken as zeros here and marked
                flag = 1;
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    uint32_t w[2] = {vd[i].x, vd[i].y};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (!in_range(w[j])) w[j] &= 0xFFFF0000u;
                        if (!in_range(w[j] >> 16)) w[j] &= 0x0000FFFFu;
                    }
                    vd[i] = make_uint2(w[0], w[1]);
                }
            }
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                // rows key16 and key16 + 16 of the block (elements), a quad of keys
                const int t = i / NB, blk = i % NB;
                const uint32_t w = vw[i], y = w >> 8;
                const pg_half2 da = __builtin_bit_cast(pg_half2, (vd[i].x & 0xFFFFu) | (vd[i].y << 16));
                const pg_half2 db = __builtin_bit_cast(pg_half2, (vd[i].x >> 16) | (vd[i].y & 0xFFFF0000u));
                const pg_half2 e0 = codes_lo(w, pat) * da, e1 = codes_lo(y, pat) * db;
                const pg_half2 h0 = codes_hi(w, pat) * da, h1 = codes_hi(y, pat) * db;
                const int quad = (my_group * G + t * 16) / 4 + oct;  // of the stage
                const int place = (quad & ~3) + 2 * (quad & 1) + ((quad >> 1) & 1);
                _Float16 *row = &s_v[buf][(blk * kQK + key16) * VROW + place * 4];
                *reinterpret_cast<pg_half4 *>(row) = pg_half4{e0.x, e0.y, e1.x, e1.y};  // keys 0, 2, 1, 3
                *reinterpret_cast<pg_half4 *>(row + 16 * VROW) = pg_half4{h0.x, h0.y, h1.x, h1.y};
            }
        }
        if (lane == 0) s_flag[buf][wave] = flag;
    };
    const bool any_stage = stage0 < n_stage;
    int id_next = id_of(stage0 + 1);
    if (any_stage) fetch(stage0, id_of(stage0));

    // The row's query as fp16, times its own power of two.
    pg_half8 q[KK];
    float f;  // what the row's scores are multiplied by
    {
        const int64_t src = (int64_t) (start + tok) * p.q_stride + (int64_t) head * D;
        pg_float4 x[KK][2];
        float amax = 0.0f, bad = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int c = 2 * (kk & 1) + half;  // octet of block kk / 2
            x[kk][0] = load4(p.q, src + (kk >> 1) * kQK + 4 * c, p.type);
            x[kk][1] = load4(p.q, src + (kk >> 1) * kQK + 4 * c + 16, p.type);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                amax = fmaxf(amax, __builtin_fabsf(x[kk][j >> 2][j & 3]));
                bad += x[kk][j >> 2][j & 3] * 0.0f;
            }
        }
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        bad += __shfl_xor(bad, 32);
        const int ex = max(__builtin_amdgcn_frexp_expf(amax), -90) - 15;
        // (never 0: masked scores are -inf times it)
        f = bad == 0.0f ? fmaxf(__builtin_amdgcn_ldexpf(p.qscale, ex), 1e-37f) : __builtin_nanf("");
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = octet_elem(0, j);
                q[kk][j] = (_Float16) __builtin_amdgcn_ldexpf(e < 16 ? x[kk][0][e & 3] : x[kk][1][e & 3], -ex);
            }
    }

    // Running maximum (log2 units), the raw score past which it is raised, sum
    // of this lane's weights, and the outputs' transposed sums.
    float m = kPagesFloor, mt = -INFINITY, l = 0.0f;
    int poison = 0;  // blocks whose V is out of range at a position the row sees
    pg_float16 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;

    // The stage in buffer buf, positions base ..
    auto multiply = [&](int buf, int base, bool edge, uint32_t bad_groups) {
        constexpr int NU = kStage / 32;
        pg_float16 s[NU];
        constexpr int N = KK * NU, AHEAD = FINE ? 4 : 8;
        auto kx = [&](int i) {
            return *reinterpret_cast<const pg_half8 *>(&s_k[buf][((i % NU) * 32 + n) * KROW + ((i / NU) * 2 + half) * 8]);
        };
        pg_half8 kring[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) kring[i] = kx(i);
        if constexpr (!FINE) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) s[u][j] = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                s[i % NU] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kring[i % AHEAD], q[i / NU], s[i % NU], 0, 0, 0);
                if (i + AHEAD < N) kring[i % AHEAD] = kx(i + AHEAD);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (i + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        } else {
            // two products of 16 elements a block, then the block's scales
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                pg_float16 t[NU];
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int j = 0; j < 16; ++j) t[u][j] = 0.0f;
#pragma unroll
                for (int k = 0; k < 2 * NU; ++k) {
                    const int i = blk * 2 * NU + k;
                    t[i % NU] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kring[i % AHEAD], q[i / NU], t[i % NU], 0, 0, 0);
                    if (i + AHEAD < N) kring[i % AHEAD] = kx(i + AHEAD);
                }
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        const pg_half4 d = *reinterpret_cast<const pg_half4 *>(
                            &s_d[buf][blk * kStage + u * 32 + 2 * j + 4 * half]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[u][j + e] = blk == 0 ? (float) d[e] * t[u][j + e]
                                                   : __builtin_fmaf((float) d[e], t[u][j + e], s[u][j + e]);
                    }
            }
        }
        // register j of tile u holds key 32 u + 8 (j / 4) + 4 half + j % 4
        if (edge) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const int off = u * 32 + 8 * (j >> 2) + 4 * half + (j & 3);
                    const int pos = base + off;
                    const bool ok = pos >= lo && pos < hi && !((bad_groups >> (off / G)) & 1u);
                    s[u][j] = ok ? s[u][j] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[u][j]);
        if (__any(mx > mt)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = mx > mt ? fmaxf(m, mx * f) : m;
            const float alpha = __builtin_amdgcn_exp2f(m - m_new);
            if (mx > mt) mt = (m_new + kLazy) / f;
            m = m_new;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] *= alpha;
        }
        constexpr int NV = NB * 2 * NU, VAHEAD = NB == 4 ? 8 : 4;
        auto vx = [&](int i) {  // 2 NU runs of 16 keys, NB blocks of elements each
            return *reinterpret_cast<const pg_half8 *>(&s_v[buf][((i % NB) * kQK + n) * VROW + (i / NB) * 16 + half * 8]);
        };
        pg_half8 ring[VAHEAD], w[2 * NU];
#pragma unroll
        for (int i = 0; i < VAHEAD; ++i) ring[i] = vx(i);
        const pg_half2 one = {(_Float16) 1.0f, (_Float16) 1.0f};
        const float up = kTop - m;
#pragma unroll
        for (int r = 0; r < 2 * NU; ++r) {
            // keys 0, 2, 1, 3 of each quad, as V's rows hold them; their sum is
            // taken from the rounded weights, as the products are
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const int u = r / 2, k = 8 * (r & 1) + (j & 4) + ((j >> 1) & 1);
                const pg_half2 h = {(_Float16) __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][k], f, up)),
                                    (_Float16) __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][k + 2], f, up))};
                w[r][j] = h.x;
                w[r][j + 1] = h.y;
                l = __builtin_amdgcn_fdot2(h, one, l, false);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            acc[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[i % VAHEAD], w[i / NB], acc[i % NB], 0, 0, 0);
            if (i + VAHEAD < NV) ring[i % VAHEAD] = vx(i + VAHEAD);
        }
    };

    if (any_stage) {
        fill(0);
        __syncthreads();
        for (int st = stage0; st < n_stage; ++st) {
            const int buf = (st - stage0) & 1;
            const bool more = st + 1 < n_stage;
            if (more) {
                fetch(st + 1, id_next);
                id_next = id_of(st + 2);
            }
            uint32_t flags = 0;
#pragma unroll
            for (int i = 0; i < NW; ++i) flags |= s_flag[buf][i] ? 1u << (i / WPG) : 0u;
            flags = __builtin_amdgcn_readfirstlane(flags);
            uint32_t bad_groups = 0;
            if (flags) {
                // a bad page, or V scales out of range: look at each
                // group of the stage again
                for (int i = 0; i < NG; ++i) {
                    const int grp = st * NG + i;
                    if (!((flags >> i) & 1u) || grp > last_group) continue;
                    const int id = table[grp >> g.group_shift];
                    if ((unsigned) id >= (unsigned) g.n_pages) {
                        bad_groups |= 1u << i;
                        continue;
                    }
                    const uint8_t *at = p.base + (int64_t) id * g.page_bytes +
                                        (((int64_t) kvh << g.group_shift) + (grp & ((1 << g.group_shift) - 1))) * kGroupBytes;
                    for (int k = 0; k < G; ++k) {
                        const int pos = grp * G + k;
                        for (int blk = 0; blk < NB; ++blk)
                            if (!in_range(*reinterpret_cast<const uint16_t *>(
                                    at + page_scale_offset((k >> 4) * NB + blk, k & 15, 1))) &&
                                pos >= lo && pos < hi)
                                poison |= 1 << blk;
                    }
                }
            }
            const int base = st * kStage;
            if (w_any && base < w_hi_max && base + kStage > w_lo_min)
                multiply(buf, base, !w_full || base + kStage > w_hi_min || base < w_lo_max || bad_groups, bad_groups);
            if (more) fill(buf ^ 1);
            __syncthreads();
        }
    }
    l += __shfl_xor(l, 32);
    if (!row_ok) return;
    const float inv = l > 0.0f ? 1.0f / l : hi > lo ? l * 0.0f : 0.0f;  // (NaN stays)
    uint16_t *out = static_cast<uint16_t *>(p.out) + ((int64_t) (start + tok) * p.n_heads + head) * D;
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
        const float scale = (poison >> blk) & 1 ? __builtin_nanf("") : inv;
        if (hi <= lo) acc[blk] = pg_float16{};  // sees nothing: zeros whatever the query holds
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float x = acc[blk][4 * i + 2 * j] * scale, y = acc[blk][4 * i + 2 * j + 1] * scale;
                if (p.type == kTypeF16) {
                    w[j] = f32_to_f16_bits(x) | ((uint32_t) f32_to_f16_bits(y) << 16);
                } else {
                    const pg_bf16x2 h = {(__bf16) x, (__bf16) y};
                    w[j] = __builtin_bit_cast(uint32_t, h);
                }
            }
            *reinterpret_cast<uint2 *>(out + blk * kQK + 8 * i + 4 * half) = make_uint2(w[0], w[1]);
        }
    }
}

// Calls with few rows are taken a column a row (pages_decode.hip), 16 columns a
// workgroup and an entry's positions shared among workgroups.  A tile's
// workgroup goes over its entry alone, 37 ns a position (27 with every wave
// full), 98 ps of the whole chip's time; a set of 16 columns takes 30 to 40 ps.
// So sets win until they fill the chip as tiles do not (1024 of them), and past
// that where a tile is no more than two sets.  us in a graph, bf16, tiles / sets:
//   32 kv heads of 128, one entry of 4000: 1 row 149 / 13, 16 rows 149 / 20,
//     64 rows 110 / 34; 64 entries of 1000: 4 rows 203 / 53, 16 rows 197 / 90,
//     24 rows 199 / 169, 48 rows 204 / 247.
//   8 kv heads of 128, 32 heads, 16 entries of 8000: 4 rows 286 / 50, 16 rows
//     (512 sets) 220 / 123, 24 (768) 230 / 187, 32 (1024) 242 / 255.
//   16 kv heads of 64, 64 entries of 1000: 16 rows 75 / 26, 32 rows 53 / 44.
static bool few_rows(const PagesAttendParams &p, int max_rows) {
    const int64_t rows = (int64_t) max_rows * (p.n_heads / p.g.n_kv);
    const int64_t units = (int64_t) p.n_batch * p.g.n_kv;
    const int64_t sets = (rows + 15) / 16 * units, tiles = (rows + kTileRows - 1) / kTileRows * units;
    return sets < 1024 || sets <= 2 * tiles;
}

hipError_t launch_pages_attend(const PagesAttendParams &p, hipStream_t stream) {
    // (an entry has no more rows than the call, where max_rows is not known)
    const int max_rows = p.max_rows > 0 ? std::min(p.max_rows, p.n_rows) : p.n_rows;
    if (few_rows(p, max_rows)) {
        PagesDecodeParams d{};
        d.base = const_cast<uint8_t *>(p.base);
        d.g = p.g;
        d.n_batch = p.n_batch;
        d.n_heads = p.n_heads;
        d.lens = p.lens;
        d.status = p.status;
        d.table = p.table;
        d.max_pages = p.max_pages;
        d.window = p.window;
        d.type = p.type;
        d.q = p.q;
        d.q_stride = p.q_stride;
        d.out = p.out;
        d.qscale = p.qscale;
        d.max_len = p.max_len;
        d.work = p.work;
        d.work_bytes = p.work_bytes;
        d.q_start = p.q_start;
        d.n_rows = p.n_rows;
        d.causal = p.causal;
        d.max_rows = max_rows;
        return launch_pages_few_rows(d, stream);
    }
    AttendArgs a{};
    a.p = p;
    a.group = p.n_heads / p.g.n_kv;
    a.max_rows = max_rows;
    a.div_group = make_fastdiv((uint32_t) a.group);
    // tiles: no more than the rows' and one more an entry, nor than every
    // entry's at its most rows
    const int64_t tiles = std::min(((int64_t) p.n_rows * a.group) / kTileRows + p.n_batch,
                                   p.n_batch * (((int64_t) max_rows * a.group + kTileRows - 1) / kTileRows));
    void *args[] = {&a};
    const bool fine = p.type == kTypeF16;
    const void *kernel = p.g.dim == 128 ? fine ? reinterpret_cast<const void *>(pages_attend_kernel<128, true>)
                                               : reinterpret_cast<const void *>(pages_attend_kernel<128, false>)
                         : fine         ? reinterpret_cast<const void *>(pages_attend_kernel<64, true>)
                                        : reinterpret_cast<const void *>(pages_attend_kernel<64, false>);
    return hipLaunchKernel(kernel, dim3((unsigned) (tiles * p.g.n_kv)), dim3(64 * kAttendWaves), args, 0, stream);
}

}  // namespace bmo
