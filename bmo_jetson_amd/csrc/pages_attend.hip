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
// of 64: each wave loads its groups of the next stage while the present one is
// multiplied, then dequantizes them into the other of two LDS buffers, K as
// [key][element] and V as [element][key] (pages_layout.hpp gives four keys of
// a V column to a lane, so nothing is transposed); one barrier a stage.
// S^T = K Q^T with v_mfma_f32_32x32x16_f16 leaves 8 + 8 keys of one row in a
// lane, which is the operand of the next product, O^T = V^T P^T, once V's
// keys stand in the same order: the weights never leave the registers.
// Row padding: K rows 16 bytes and V rows 16 bytes longer than their data, so
// that 16 lanes reading 16 bytes each from consecutive rows meet every LDS
// bank once.
//
// Precision: K and V enter as (code - 8) * d rounded to fp16, the weights as
// fp16, sums in fp32; q enters scaled by its row's own power of two, exactly.
// That is below the rounding of the 16-bit outputs (2e-4 against 2e-3 for
// bf16).  K and V must lie in fp16's range; a V block whose scale is not
// finite makes the rows that see it NaN in that block and leaves the others.
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

struct AttendArgs {
    PagesAttendParams p;
    int group;          // query heads a kv head
    FastDiv div_group;
};

// The entry and first row of tile `tile`; false past the last.
struct RowTile {
    int b, row0, rows;  // row0 and rows count (token, head) pairs
};
__device__ __forceinline__ int entry_rows(const AttendArgs &a, int b) {
    const int s = a.p.q_start[b], e = a.p.q_start[b + 1];
    return s < 0 || e < s || e > a.p.n_rows ? 0 : e - s;
}
__device__ __forceinline__ bool find_tile(const AttendArgs &a, int tile, int lane, RowTile &t) {
    int before = 0;
    for (int b0 = 0; b0 < a.p.n_batch; b0 += 64) {
        const int b = b0 + lane;
        const int rows = b < a.p.n_batch ? entry_rows(a, b) * a.group : 0;
        const int tiles = (rows + kTileRows - 1) / kTileRows;
        const int upto = wave_prefix(tiles, lane) + before;
        const uint64_t past = __ballot(upto > tile);
        if (past) {
            const int l = __ffsll((unsigned long long) past) - 1;
            t.b = b0 + l;
            t.rows = __shfl(rows, l);
            t.row0 = (tile - (__shfl(upto, l) - __shfl(tiles, l))) * kTileRows;
            // (always so, unless q_start is no running sum)
            return (unsigned) t.row0 < (unsigned) t.rows;
        }
        before = __shfl(upto, 63);
    }
    return false;
}

__device__ __forceinline__ bool finite16(uint32_t h) { return (h & 0x7C00u) != 0x7C00u; }

}  // namespace

template <int D>
__global__ __launch_bounds__(64 * kAttendWaves, 2) void pages_attend_kernel(AttendArgs a) {
    constexpr int NW = kAttendWaves;
    constexpr int NB = D / kQK;
    constexpr int G = 2048 / D;           // keys a group
    constexpr int NG = kStage / G;        // groups a stage
    constexpr int KROW = D + 8;           // halves of a K row
    constexpr int VROW = kStage + 8;      // halves of a V row
    constexpr int KK = D / 16;            // products of 16 elements a key
    const PagesAttendParams &p = a.p;
    const PagesGeom &g = p.g;

    __shared__ __align__(16) _Float16 s_k[2][kStage * KROW];
    __shared__ __align__(16) _Float16 s_v[2][D * VROW];
    __shared__ int s_flag[2][NG];  // nonzero: a bad page, or a V scale that is not finite

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    const int n = lane & 31, half = lane >> 5;

    const int tile = (int) blockIdx.x / g.n_kv;
    const int kvh = (int) blockIdx.x - tile * g.n_kv;
    RowTile rt;
    if (!find_tile(a, tile, lane, rt)) return;
    const int b = __builtin_amdgcn_readfirstlane(rt.b);
    const int start = p.q_start[b];
    const int n_tok = entry_rows(a, b);
    const int64_t room = (int64_t) p.max_pages << g.page_shift;
    const int len = (int) min((int64_t) max(p.lens[b], 0), room);
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
        const int ex = __builtin_amdgcn_frexp_expf(amax) - 15;
        f = bad == 0.0f ? __builtin_amdgcn_ldexpf(p.qscale, ex) : __builtin_nanf("");
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = octet_elem(0, j);
                q[kk][j] = (_Float16) __builtin_amdgcn_ldexpf(e < 16 ? x[kk][0][e & 3] : x[kk][1][e & 3], -ex);
            }
    }

    // ---- filling: wave w takes group w, w + 4 .. of a stage ----
    constexpr int LG = (NG + NW - 1) / NW;  // groups a wave loads
    struct Load {
        uint4 k, v;
        uint4 ks;       // the key's block scales: [t][b] halves (low half of each dword)
        uint2 vs[4];    // four keys' scales of each (t, b)
        int flag;
    };
    Load ld[LG];
    const Patterns pat;
    const int last_group = max((len - 1) / G, 0);
    const int key16 = lane & 15, oct = lane >> 4;
    auto fetch = [&](int stage) {
#pragma unroll
        for (int i = 0; i < LG; ++i) {
            const int gi = wave + i * NW;
            if (NG % NW != 0 && gi >= NG) break;
            const int grp = min(stage * NG + gi, last_group);
            const int id = table[grp >> g.group_shift];
            const bool ok = (unsigned) id < (unsigned) g.n_pages;
            const uint8_t *at = p.base + (int64_t) (ok ? id : 0) * g.page_bytes +
                                (((int64_t) kvh << g.group_shift) + (grp & ((1 << g.group_shift) - 1))) * kGroupBytes;
            ld[i].flag = ok ? 0 : 1;
            ld[i].k = *reinterpret_cast<const uint4 *>(at + lane * 16);
            ld[i].v = *reinterpret_cast<const uint4 *>(at + kVCodeOff + lane * 16);
            uint32_t ks[4];
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                ks[tb] = *reinterpret_cast<const uint16_t *>(at + page_scale_offset(tb, key16, 0));
                ld[i].vs[tb] = *reinterpret_cast<const uint2 *>(at + page_scale_offset(tb, 4 * oct, 1));
            }
            ld[i].ks = make_uint4(ks[0], ks[1], ks[2], ks[3]);
        }
    };
    auto fill = [&](int buf) {
#pragma unroll
        for (int i = 0; i < LG; ++i) {
            const int gi = wave + i * NW;
            if (NG % NW != 0 && gi >= NG) break;
            const uint32_t kw[4] = {ld[i].k.x, ld[i].k.y, ld[i].k.z, ld[i].k.w};
            const uint32_t vw[4] = {ld[i].v.x, ld[i].v.y, ld[i].v.z, ld[i].v.w};
            const uint32_t kd[4] = {ld[i].ks.x, ld[i].ks.y, ld[i].ks.z, ld[i].ks.w};
            pg_half2 check = {(_Float16) 0.0f, (_Float16) 0.0f};
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                const pg_half2 z = {(_Float16) 0.0f, (_Float16) 0.0f};
                check = __builtin_elementwise_fma(__builtin_bit_cast(pg_half2, ld[i].vs[tb].x), z, check);
                check = __builtin_elementwise_fma(__builtin_bit_cast(pg_half2, ld[i].vs[tb].y), z, check);
            }
            const bool odd = !(check.x == (_Float16) 0.0f && check.y == (_Float16) 0.0f);
            if (__any(odd)) {  // rare: such blocks are taken as zeros here and marked
                ld[i].flag = 1;
#pragma unroll
                for (int tb = 0; tb < 4; ++tb) {
                    uint32_t w[2] = {ld[i].vs[tb].x, ld[i].vs[tb].y};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (!finite16(w[j])) w[j] &= 0xFFFF0000u;
                        if (!finite16(w[j] >> 16)) w[j] &= 0x0000FFFFu;
                    }
                    ld[i].vs[tb] = make_uint2(w[0], w[1]);
                }
            }
#pragma unroll
            for (int tb = 0; tb < 4; ++tb) {
                const int t = tb / NB, blk = tb % NB;
                // K: row of the key, octet `oct` of the block
                const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t) kd[tb]);
                const pg_half8 kx = k_octet(kw[tb], pat) * pg_half8{d, d, d, d, d, d, d, d};
                const int key = gi * G + t * 16 + key16;
                *reinterpret_cast<pg_half8 *>(&s_k[buf][key * KROW + (blk * 4 + oct) * 8]) = kx;
                // V: rows key16 and key16 + 16 of the block (elements), quad of keys
                const uint32_t w = vw[tb], y = w >> 8;
                const pg_half2 da = __builtin_bit_cast(pg_half2, (ld[i].vs[tb].x & 0xFFFFu) | (ld[i].vs[tb].y << 16));
                const pg_half2 db = __builtin_bit_cast(pg_half2, (ld[i].vs[tb].x >> 16) | (ld[i].vs[tb].y & 0xFFFF0000u));
                const pg_half2 e0 = codes_lo(w, pat) * da, e1 = codes_lo(y, pat) * db;
                const pg_half2 h0 = codes_hi(w, pat) * da, h1 = codes_hi(y, pat) * db;
                const int quad = (gi * G + t * 16) / 4 + oct;  // of the stage
                const int place = (quad & ~3) + 2 * (quad & 1) + ((quad >> 1) & 1);
                _Float16 *row = &s_v[buf][(blk * kQK + key16) * VROW + place * 4];
                *reinterpret_cast<pg_half4 *>(row) = pg_half4{e0.x, e0.y, e1.x, e1.y};  // keys 0, 2, 1, 3
                *reinterpret_cast<pg_half4 *>(row + 16 * VROW) = pg_half4{h0.x, h0.y, h1.x, h1.y};
            }
            if (lane == 0) s_flag[buf][gi] = ld[i].flag;
        }
    };

    float m = kPagesFloor, mt = kPagesFloor, l = 0.0f;
    int poison = 0;  // blocks whose V is not finite at a position the row sees
    pg_float16 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;

    // One tile of 32 keys at LDS row `at`, positions base ...  EDGE: some row
    // of the wave does not see some key.
    auto tile_of = [&](int buf, int at, int base, bool edge, uint32_t bad_groups) {
        pg_float16 s;
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const pg_half8 kx = *reinterpret_cast<const pg_half8 *>(&s_k[buf][(at + n) * KROW + (kk * 2 + half) * 8]);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kx, q[kk], s, 0, 0, 0);
        }
        // register j holds key 8 (j / 4) + 4 half + j % 4
        if (edge) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int off = 8 * (j >> 2) + 4 * half + (j & 3);
                const int pos = base + off;
                const bool ok = pos >= lo && pos < hi && !((bad_groups >> ((at + off) / G)) & 1u);
                s[j] = ok ? s[j] * f : -INFINITY;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[j] *= f;
        }
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
        if (__any(mx > mt)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = fmaxf(m, mx);
            const float alpha = __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            mt = m_new + kPagesLazy;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[i][j] *= alpha;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            s[j] = __builtin_amdgcn_exp2f(s[j] - m);
            l += s[j];
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            pg_half8 w;  // keys 0, 2, 1, 3 of each quad, as V's rows hold them
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = 8 * ks + (j & 4) + (j & 1 ? 2 : 0) + ((j >> 1) & 1);
                w[j] = (_Float16) s[k];
            }
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                const pg_half8 vx = *reinterpret_cast<const pg_half8 *>(
                    &s_v[buf][(blk * kQK + n) * VROW + at + (ks * 2 + half) * 8]);
                acc[blk] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vx, w, acc[blk], 0, 0, 0);
            }
        }
    };

    if (stage0 < n_stage) {
        fetch(stage0);
        fill(0);
        __syncthreads();
        for (int st = stage0; st < n_stage; ++st) {
            const int buf = (st - stage0) & 1;
            const bool more = st + 1 < n_stage;
            if (more) fetch(st + 1);
            uint32_t flags = 0;
#pragma unroll
            for (int i = 0; i < NG; ++i) flags |= s_flag[buf][i] ? 1u << i : 0u;
            flags = __builtin_amdgcn_readfirstlane(flags);
            uint32_t bad_groups = 0;
            if (flags) {
                // a bad page, or V scales that are not finite: look at each
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
                            if (!finite16(*reinterpret_cast<const uint16_t *>(
                                    at + page_scale_offset((k >> 4) * NB + blk, k & 15, 1))) &&
                                pos >= lo && pos < hi)
                                poison |= 1 << blk;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kStage / 32; ++u) {
                const int base = st * kStage + u * 32;
                if (!w_any || base >= w_hi_max || base + 32 <= w_lo_min) continue;
                const bool edge = !w_full || base + 32 > w_hi_min || base < w_lo_max || bad_groups;
                tile_of(buf, u * 32, base, edge, bad_groups);
            }
            if (more) fill(buf ^ 1);
            __syncthreads();
        }
    }
    l += __shfl_xor(l, 32);
    if (!row_ok) return;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint16_t *out = static_cast<uint16_t *>(p.out) + ((int64_t) (start + tok) * p.n_heads + head) * D;
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
        const float scale = (poison >> blk) & 1 ? __builtin_nanf("") : inv;
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

hipError_t launch_pages_attend(const PagesAttendParams &p, hipStream_t stream) {
    AttendArgs a{};
    a.p = p;
    a.group = p.n_heads / p.g.n_kv;
    a.div_group = make_fastdiv((uint32_t) a.group);
    // tiles: no more than the rows' and one more an entry, nor than every
    // entry's at its most rows
    int64_t tiles = ((int64_t) p.n_rows * a.group) / kTileRows + p.n_batch;
    if (p.max_rows > 0) {
        const int64_t most = (int64_t) p.n_batch * (((int64_t) p.max_rows * a.group + kTileRows - 1) / kTileRows);
        tiles = tiles < most ? tiles : most;
    }
    void *args[] = {&a};
    const void *kernel = p.g.dim == 128 ? reinterpret_cast<const void *>(pages_attend_kernel<128>)
                                        : reinterpret_cast<const void *>(pages_attend_kernel<64>);
    return hipLaunchKernel(kernel, dim3((unsigned) (tiles * p.g.n_kv)), dim3(64 * kAttendWaves), args, 0, stream);
}

}  // namespace bmo
