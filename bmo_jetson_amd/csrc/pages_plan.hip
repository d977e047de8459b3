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
// The entries pass in chunks of 1024, one a thread: three block-wide prefix
// sums, then the workgroup's share of the chunk's new tokens, each finding
// its entry by binary search in LDS.  The token on a page's first position
// also enters the page in the table.  With many tokens several workgroups do
// the same scans and share the tokens; lengths, list and counts are replaced
// by the workgroup that arrives last, when every other has read them.
#include "pages.hpp"

namespace bmo {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
// Tokens a workgroup is meant to place.
constexpr int kPlanShare = 4096;

struct Entry {
    int64_t len, want, count, start;
    int64_t have_pages, want_pages;
    int64_t need, upto;    // pages asked for, and the sum through this entry
    int64_t back, before;  // pages given back, and the sum before this entry
    int state;
    bool live;
};

// Inclusive sum over the workgroup's threads; total receives the whole sum.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t *s_wave, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();  // the last sums have been read
    if (lane == 63) s_wave[wave] = v;
    __syncthreads();
    // every wave sums up the waves' sums, lane by lane
    int64_t upto = s_wave[lane & (kPlanWaves - 1)];
#pragma unroll
    for (int d = 1; d < kPlanWaves; d <<= 1) {
        const int64_t o = __shfl_up(upto, d);
        if ((lane & (kPlanWaves - 1)) >= d) upto += o;
    }
    total = __shfl(upto, kPlanWaves - 1);
    return v + (wave > 0 ? __shfl(upto, wave - 1) : 0);
}

// What the entries before a chunk sum up to.
struct Carry {
    int64_t tokens = 0, need = 0, given = 0, back = 0;
};

__device__ Entry scan_chunk(const PlanParams &p, int b0, int64_t n_free, Carry &c, int64_t *s_wave) {
    Entry e{};
    const int b = b0 + (int) threadIdx.x;
    e.live = b < p.n_batch;
    const int64_t asked = e.live ? p.n_new[b] : 0;
    e.len = e.live ? p.lens[b] : 0;
    const int64_t room = (int64_t) p.max_pages << p.page_shift;
    const int page = 1 << p.page_shift;
    e.want = e.len + asked < 0 ? 0 : e.len + asked;
    e.count = asked > 0 ? asked : 0;
    int64_t total;
    const int64_t upto = block_sum(e.count, s_wave, total) + c.tokens;
    e.start = upto - e.count;
    c.tokens += total;
    const bool bad = e.len < 0 || e.len > room || e.want > room || e.want > INT32_MAX ||
                     (e.count > 0 && upto > p.max_tok);
    e.have_pages = (e.len + page - 1) >> p.page_shift;
    e.want_pages = (e.want + page - 1) >> p.page_shift;
    e.need = !bad && asked > 0 ? e.want_pages - e.have_pages : 0;
    e.upto = block_sum(e.need, s_wave, total) + c.need;
    c.need += total;
    const bool refused = e.need > 0 && e.upto > n_free;
    e.state = bad ? 2 : refused ? 1 : 0;
    (void) block_sum(refused ? 0 : e.need, s_wave, total);
    c.given += total;
    e.back = e.state == 0 && asked < 0 ? e.have_pages - e.want_pages : 0;
    e.before = block_sum(e.back, s_wave, total) - e.back + c.back;
    c.back += total;
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
    __shared__ int64_t s_wave[kPlanWaves];
    __shared__ int s_start[kPlanThreads];  // tokens, later pages given back, before each entry
    __shared__ int s_len[kPlanThreads];
    __shared__ int s_have[kPlanThreads];
    __shared__ int s_taken[kPlanThreads];  // list place of an entry's first page; -1: nothing is placed
    __shared__ int s_last;
    const int tid = (int) threadIdx.x;
    const int page = 1 << p.page_shift;
    const int64_t n_free = min(max(p.list[0], 0), p.n_pages);
    const int *ids = p.list + kListHead;

    Carry c;
    Entry e{};
    for (int b0 = 0; b0 < p.n_batch; b0 += kPlanThreads) {
        const Carry before = c;
        e = scan_chunk(p, b0, n_free, c, s_wave);
        const int n = min(kPlanThreads, p.n_batch - b0);
        __syncthreads();  // the last chunk's tokens are placed
        s_start[tid] = clamp_int(e.start);
        s_len[tid] = (int) e.len;
        s_have[tid] = (int) e.have_pages;
        s_taken[tid] = e.state == 0 ? clamp_int(n_free - 1 - (e.upto - e.need)) : INT32_MIN;
        __syncthreads();
        // tokens of this chunk, every gridDim.x-th run of them this workgroup's
        const int64_t end = min(c.tokens, (int64_t) p.max_tok);
        for (int64_t t = before.tokens + (int64_t) blockIdx.x * kPlanThreads + tid; t < end;
             t += (int64_t) gridDim.x * kPlanThreads) {
            const int i = find(s_start, n, (int) t);
            const int taken = s_taken[i];
            int pos = -1, slot = -1;
            if (taken != INT32_MIN) {
                pos = s_len[i] + ((int) t - s_start[i]);
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
        __threadfence();
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
            e = scan_chunk(p, b0, n_free, d, s_wave);
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
    const int wgs = p.max_tok <= kPlanShare ? 1 : (int) ((p.max_tok + (int64_t) kPlanShare - 1) / kPlanShare);
    return hipLaunchKernel(reinterpret_cast<const void *>(plan_kernel), dim3((unsigned) (wgs < 128 ? wgs : 128)),
                           dim3(kPlanThreads), args, 0, stream);
}

hipError_t launch_list_init(int *list, int n_pages, hipStream_t stream) {
    void *args[] = {&list, &n_pages};
    return hipLaunchKernel(reinterpret_cast<const void *>(list_init_kernel), dim3((unsigned) ((n_pages + 255) / 256)),
                           dim3(256), args, 0, stream);
}

}  // namespace bmo
