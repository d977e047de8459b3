// pages_plan.hip -- block tables and slot maps from the requests' lengths.
//
// Entry b asks for n_new[b] more positions (or, negative, fewer).  With
// P = page size and pages(x) = ceil(x / P), a growing entry needs
// pages(len + n) - pages(len) pages; it is granted if the needs up to and
// including its own do not pass the number of free pages (so whoever comes
// after the first refusal and needs a page is refused too), and its j-th page
// is the j-th from the end of the list.  A shrinking entry's pages go back in
// the reverse order, which makes a growth that is taken back restore the
// list.  Everything follows from prefix sums over the entries, so the result
// does not depend on the order in which workgroups run.
//
// The entries pass in chunks of 1024, one a thread: one block-wide pass of
// three prefix sums (lane shifts, no LDS but for the waves' sums), then the
// workgroup's share of the chunk's new tokens, each finding its entry by binary
// search in LDS.  The token on a page's first position also enters the page in
// the table; where no call asks for the tokens' places, granted pages are
// walked instead, so that what is refused costs nothing.  With many tokens
// several workgroups do the same scans and share the tokens; lengths, list and
// counts are replaced by the workgroup that arrives last, when every other has
// read them.
//
// Latency bounds it, load after load (lengths, list, table) and the code's own
// fetch: 48 entries with a token each 4.8 us, 256 entries with 64 k tokens of
// prompts 7.2 us in a graph (one workgroup per 1024 tokens; per 4096 8.7 us,
// waves of a quarter as many threads 13 us).  Four returned pages a thread at
// a time cost a token's step 0.5 us more than they save.
#include <algorithm>

#include "pages.hpp"

namespace bmo {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// Tokens a workgroup is meant to place.
constexpr int kPlanShare = 1024;

struct Entry {
    int64_t len, want, count, start;
    int64_t have_pages, want_pages;
    int64_t need, upto;    // pages asked for, and the sum through this entry
    int64_t back, before;  // pages given back, and the sum before this entry
    int state;
    bool live;
};

// Sums saturate at 2^32 - 1, which is past every limit that they are held
// against (saturating sums of counts are still associative).
__device__ __forceinline__ uint32_t sat_add(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
template <int CTRL, int ROWS>
__device__ __forceinline__ void sum_step(uint32_t (&v)[3]) {
#pragma unroll
    for (int k = 0; k < 3; ++k)
        v[k] = sat_add(v[k], (uint32_t) __builtin_amdgcn_update_dpp(0, (int) v[k], CTRL, ROWS, 0xF, false));
}

// Inclusive sums over the workgroup's threads of three counts each; total
// receives the whole sums.
__device__ __forceinline__ void block_sums(uint32_t (&v)[3], uint32_t (*s_wave)[kPlanWaves], uint32_t (&total)[3]) {
    static_assert(kPlanWaves <= 16, "the waves' sums fit in a row of 16 lanes");
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int) threadIdx.x >> 6);
    sum_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8: the rows of 16 lanes
    sum_step<0x112, 0xF>(v);
    sum_step<0x114, 0xF>(v);
    sum_step<0x118, 0xF>(v);
    sum_step<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3, then 31 into 2 and 3
    sum_step<0x143, 0xC>(v);
    __syncthreads();  // the last sums have been read
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < 3; ++k) s_wave[k][wave] = v[k];
    __syncthreads();
    // every wave sums up the waves' sums, in a row of its lanes
    uint32_t w[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) w[k] = s_wave[k][lane & (kPlanWaves - 1)];
    sum_step<0x111, 0xF>(w);
    sum_step<0x112, 0xF>(w);
    sum_step<0x114, 0xF>(w);
    sum_step<0x118, 0xF>(w);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        total[k] = (uint32_t) __builtin_amdgcn_readlane((int) w[k], kPlanWaves - 1);
        const uint32_t before = (uint32_t) __builtin_amdgcn_readlane((int) w[k], max(wave - 1, 0));
        v[k] = wave > 0 ? sat_add(v[k], before) : v[k];
    }
}

// What the entries before a chunk sum up to.
struct Carry {
    int64_t tokens = 0, need = 0, given = 0, back = 0;
};

struct Sums {
    uint32_t wave[3][kPlanWaves];
    uint32_t given;
};

__device__ Entry scan_chunk(const PlanParams &p, int b0, int64_t n_free, Carry &c, Sums &s) {
    Entry e{};
    const int b = b0 + (int) threadIdx.x;
    e.live = b < p.n_batch;
    const int64_t asked = e.live ? p.n_new[b] : 0;
    e.len = e.live ? p.lens[b] : 0;
    const int64_t room = (int64_t) p.max_pages << p.page_shift;
    const int page = 1 << p.page_shift;
    e.want = e.len + asked < 0 ? 0 : e.len + asked;
    e.count = asked > 0 ? asked : 0;
    const bool bad = e.len < 0 || e.len > room || e.want > room;  // (room is at most 2^30)
    e.have_pages = (e.len + page - 1) >> p.page_shift;
    e.want_pages = (e.want + page - 1) >> p.page_shift;
    e.need = !bad && asked > 0 ? e.want_pages - e.have_pages : 0;
    e.back = !bad && asked < 0 ? e.have_pages - e.want_pages : 0;
    // One pass of sums: tokens past max_tok refuse every later entry that asks
    // for some, so what these need after all changes no earlier sum.
    uint32_t v[3] = {(uint32_t) e.count, (uint32_t) e.need, (uint32_t) e.back}, total[3];
    if (threadIdx.x == 0) s.given = 0;  // (between barriers of block_sums)
    block_sums(v, s.wave, total);
    const int64_t tokens_upto = c.tokens + v[0];
    e.start = tokens_upto - e.count;
    e.upto = c.need + v[1];
    e.before = c.back + v[2] - e.back;
    const bool full = e.count > 0 && tokens_upto > p.max_tok;
    const bool refused = e.need > 0 && e.upto > n_free;
    e.state = bad || full ? 2 : refused ? 1 : 0;
    // The granted needs sum up to the last granted entry's sum.
    const uint64_t granted = __ballot(e.state == 0 && e.need > 0);
    if (granted) {
        const uint32_t upto = (uint32_t) __builtin_amdgcn_readlane((int) v[1], 63 - __clzll((long long) granted));
        if ((threadIdx.x & 63) == 0) atomicMax(&s.given, upto);
    }
    if (e.state != 0) e.need = 0;
    __syncthreads();
    c.given = s.given > 0 ? c.need + s.given : c.given;
    c.tokens += total[0];
    c.need += total[1];
    c.back += total[2];
    return e;
}

// The last i of [0, n) with v[i] <= x (v ascending, v[0] <= x).
__device__ __forceinline__ int find(const int *v, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int clamp_int(int64_t v) {
    return (int) min(max(v, (int64_t) INT32_MIN + 1), (int64_t) INT32_MAX);
}

}  // namespace

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanParams p) {
    __shared__ Sums s_sums;
    __shared__ int s_start[kPlanThreads];  // tokens, later pages given back, before each entry
    __shared__ int s_len[kPlanThreads];
    __shared__ int s_have[kPlanThreads];
    __shared__ int s_taken[kPlanThreads];  // list place of an entry's first page; -1: nothing is placed
    __shared__ int s_last;
    const int tid = (int) threadIdx.x;
    const int page = 1 << p.page_shift;
    const int64_t n_free = min(max(p.list[0], 0), p.n_pages);
    const int *ids = p.list + kListHead;

    const bool places = p.tok_slot || p.tok_pos || p.tok_entry;
    Carry c;
    Entry e{};
    for (int b0 = 0; b0 < p.n_batch; b0 += kPlanThreads) {
        const Carry before = c;
        e = scan_chunk(p, b0, n_free, c, s_sums);
        const int n = min(kPlanThreads, p.n_batch - b0);
        __syncthreads();  // the last chunk's tokens are placed
        // (pages before the entry's: of granted ones only these are walked)
        s_start[tid] = clamp_int(places ? e.start : e.upto - e.need - before.need);
        s_len[tid] = (int) e.len;
        s_have[tid] = (int) e.have_pages;
        s_taken[tid] = e.state == 0 ? clamp_int(n_free - 1 - (e.upto - e.need)) : INT32_MIN;
        __syncthreads();
        // tokens (or granted pages, by their first positions) of this chunk, every
        // gridDim.x-th run of them this workgroup's
        const int64_t begin = places ? before.tokens : 0;
        const int64_t end = places ? min(c.tokens, (int64_t) p.max_tok) : c.given - before.need;
        for (int64_t t = begin + (int64_t) blockIdx.x * kPlanThreads + tid; t < end;
             t += (int64_t) gridDim.x * kPlanThreads) {
            const int i = find(s_start, n, (int) t);
            const int taken = s_taken[i];
            int pos = -1, slot = -1;
            if (taken != INT32_MIN) {
                pos = (int) t - s_start[i];
                pos = places ? s_len[i] + pos : (s_have[i] + pos) << p.page_shift;
                const int col = pos >> p.page_shift, off = pos & (page - 1);
                int *entry = p.table + (int64_t) (b0 + i) * p.max_pages + col;
                int id;
                if (col < s_have[i]) {
                    id = *entry;
                } else {
                    id = ids[taken - (col - s_have[i])];
                    if (off == 0) *entry = id;
                }
                slot = (unsigned) id < (unsigned) p.n_pages ? id * page + off : -1;
            }
            if (p.tok_slot) p.tok_slot[t] = slot;
            if (p.tok_pos) p.tok_pos[t] = pos;
            if (p.tok_entry) p.tok_entry[t] = b0 + i;
        }
    }

    if (gridDim.x > 1) {
        // What is replaced below has been read before this arrival: every wave
        // waits for its loads.  Nothing that others wrote is read below, so no
        // cache is written back (with __threadfence 64 workgroups take 22 us, not 7).
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) s_last = atomicAdd(p.list + 1, 1) == (int) gridDim.x - 1;
        __syncthreads();
        if (!s_last) return;
    } else {
        __syncthreads();
    }
    // every workgroup has read what is replaced from here on
    const int64_t left = n_free - c.given;
    const int64_t after = left + c.back;
    Carry d;
    for (int b0 = 0; b0 < p.n_batch; b0 += kPlanThreads) {
        if (p.n_batch > kPlanThreads) {
            e = scan_chunk(p, b0, n_free, d, s_sums);
        } else {
            d = c;
        }
        const int n = min(kPlanThreads, p.n_batch - b0);
        __syncthreads();
        s_start[tid] = clamp_int(e.before);
        s_have[tid] = (int) e.want_pages;
        __syncthreads();
        const int64_t first = s_start[0];
        for (int64_t k = first + tid; k < d.back; k += kPlanThreads) {
            const int i = find(s_start, n, (int) k);
            const int64_t at = after - 1 - k;
            const int id = p.table[(int64_t) (b0 + i) * p.max_pages + s_have[i] + ((int) k - s_start[i])];
            if (at >= 0 && at < p.n_pages) p.list[kListHead + at] = id;
        }
        if (e.live) {
            const int b = b0 + tid;
            if (p.tok_start) p.tok_start[b] = clamp_int(e.start);
            if (p.status) p.status[b] = e.state;
            if (e.state == 0) p.lens[b] = (int) e.want;
        }
        __syncthreads();
    }
    if (tid == 0) {
        if (p.tok_start) p.tok_start[p.n_batch] = clamp_int(c.tokens);
        p.list[0] = (int) min(after, (int64_t) p.n_pages);
        p.list[1] = 0;
    }
}

__global__ __launch_bounds__(256) void list_init_kernel(int *list, int n_pages) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n_pages) list[kListHead + i] = n_pages - 1 - i;
    if (i == 0) {
        list[0] = n_pages;
        list[1] = 0;
    }
}

hipError_t launch_plan(const PlanParams &p, hipStream_t stream) {
    PlanParams arg = p;
    void *args[] = {&arg};
    // without arrays max_tok tells nothing: a token each is what such calls ask for
    const int64_t tokens = p.tok_slot || p.tok_pos || p.tok_entry ? p.max_tok : std::min(p.max_tok, p.n_batch);
    const int64_t wgs = std::max<int64_t>((tokens + kPlanShare - 1) / kPlanShare, 1);
    return hipLaunchKernel(reinterpret_cast<const void *>(plan_kernel), dim3((unsigned) (wgs < 128 ? wgs : 128)),
                           dim3(kPlanThreads), args, 0, stream);
}

hipError_t launch_list_init(int *list, int n_pages, hipStream_t stream) {
    void *args[] = {&list, &n_pages};
    return hipLaunchKernel(reinterpret_cast<const void *>(list_init_kernel), dim3((unsigned) ((n_pages + 255) / 256)),
                           dim3(256), args, 0, stream);
}

}  // namespace bmo
