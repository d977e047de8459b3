// pages.hpp -- parameter blocks and launchers of the paged cache's kernels
// (internal to libbmo_attn.so; the public surface is include/bmo_attn.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pages_layout.hpp"

namespace bmo {

// Element types of rows (the values of BMO_ATTN_F32 ..).
enum PagesType { kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 2, kTypeQ4_0 = 3 };
constexpr int type_bytes(int type) { return type == kTypeF32 ? 4 : 2; }

// The list of free pages: list[0] is how many there are, list[1] counts
// workgroups inside a call and is 0 between calls, ids from list[2] on.
constexpr int kListHead = 2;

struct PlanParams {
    int *list;
    int n_pages;
    int page_shift;
    int n_batch;
    const int *n_new;
    int *lens;
    int *table;
    int max_pages;
    int *tok_start;  // nullable, like the outputs below
    int max_tok;
    int *tok_slot;
    int *tok_pos;
    int *tok_entry;
    int *status;
};
hipError_t launch_plan(const PlanParams &p, hipStream_t stream);
hipError_t launch_list_init(int *list, int n_pages, hipStream_t stream);

// n_tok rows [n_kv][dim] of K and of V, a row's tokens stride elements apart
// (blocks of 18 bytes: dense), to or from slots slots[t] of one layer.
struct SlotsParams {
    uint8_t *base;  // the layer's pages
    PagesGeom g;
    const int *slots;
    int n_tok;
    int type;
    void *k;
    void *v;
    int64_t stride;
};
hipError_t launch_pages_append(const SlotsParams &p, hipStream_t stream);
hipError_t launch_pages_gather(const SlotsParams &p, hipStream_t stream);
hipError_t launch_pages_clear(uint8_t *base, int64_t bytes, hipStream_t stream);

// Attention of one row per entry over its pages.
struct PagesDecodeParams {
    uint8_t *base;  // the layer's pages
    PagesGeom g;
    int n_batch;
    int n_heads;
    const int *lens;
    const int *n_new;  // what a plan was asked for and its status, nullable: entries
    const int *status; // that did not grow have no positions here
    const int *table;
    int max_pages;
    int window;  // 0: none
    int type;    // of q, k_new, v_new and out
    const void *q;
    int64_t q_stride;
    const void *k_new;  // append_decode only
    const void *v_new;
    int64_t kv_stride;
    void *out;
    float qscale;  // softmax scale * log2(e)
    int max_len;   // no entry is longer (0: not known); what is longer is still read
    float *work;   // partial results, nullable
    int64_t work_bytes;
    // several rows an entry (launch_pages_few_rows), see PagesAttendParams
    const int *q_start;
    int n_rows;
    int causal;
    int max_rows;
};
hipError_t launch_pages_decode(const PagesDecodeParams &p, hipStream_t stream);
// Ragged rows, no more than max_rows an entry, in 16 bits, by the same kernel.
hipError_t launch_pages_few_rows(const PagesDecodeParams &p, hipStream_t stream);
// Bytes of partial results that a launch may keep.
int64_t pages_work_bytes(const PagesGeom &g);

// Attention of ragged rows.
struct PagesAttendParams {
    const uint8_t *base;  // the layer's pages
    PagesGeom g;
    int n_batch;
    int n_heads;
    const int *q_start;  // [n_batch + 1]
    const int *lens;
    const int *status;  // a plan's, nullable: entries that it refused have no positions here
    const int *table;
    int max_pages;
    int n_rows;  // rows of q and out
    int causal;
    int window;
    int type;
    const void *q;
    int64_t q_stride;
    void *out;
    float qscale;
    int max_rows;  // no entry has more (0: not known)
    int max_len;
    float *work;
    int64_t work_bytes;
};
hipError_t launch_pages_attend(const PagesAttendParams &p, hipStream_t stream);

}  // namespace bmo
