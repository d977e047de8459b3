// pages_layout.hpp -- where each Q4_0 block of the paged cache lives in HBM.
//
// A page holds page_size consecutive positions of one request in every kv
// head.  The slots of one (layer, page, kv head) are cut into groups of
// G = 2048 / head_dim (16 at head_dim 128, 32 at 64), 2304 bytes each as in
// the ring, but arranged for the matrix cores: one allocation holds the groups
// as [n_layers][n_pages][n_kv_heads][page_size / G], and in a group, with
// NB = head_dim / 32 blocks a key and T = 4 / NB tiles of 16 keys,
//
//   [0, 1024)     K codes: dword ((c * 16 + key) * 4 + t * NB + b) holds bytes
//                 4c .. 4c+3 of ggml's block b of key t * 16 + key;
//   [1024, 2048)  V codes: byte j of dword ((c * 16 + i) * 4 + t * NB + b) is
//                 byte i of block b of key t * 16 + 4 c + j;
//   [2048, 2304)  scales, fp16: 16 bytes at ((t * NB + b) * 4 + c) * 16 are
//                 those of block b of keys t * 16 + 4 c + 0 .. 3, K's four
//                 and then V's four.
//
// So the 16 bytes at lane * 16 of either code region are what lane c * 16 + i
// of v_mfma_f32_16x16x32 takes of the group: K rows with 8 elements of each
// block (byte j of a ggml block holds elements j and j + 16), or V columns i
// and i + 16 of each block at four keys.  V needs no transposition through
// LDS, and a token is still written in whole bytes, so that appends of
// different tokens touch different bytes.  Codes are ggml's (0..15); a zeroed
// group is ggml's zero block.
#pragma once

#include <stdint.h>

#include "ring_layout.hpp"

namespace bmo {

// Byte offset in a group of the scale of block tb = t * NB + b of key `key`
// of its tile, of K (which 0) or V (which 1).
__host__ __device__ constexpr int page_scale_offset(int tb, int key, int which) {
    return kScaleOff + (tb * 4 + (key >> 2)) * 16 + which * 8 + (key & 3) * 2;
}

struct PagesGeom {
    int n_layers;
    int n_pages;
    int page;      // slots a page, a power of two, a multiple of the group
    int n_kv;
    int dim;
    int page_shift;   // log2(page)
    int group_shift;  // log2(groups per page)
    int64_t page_bytes;
    int64_t layer_bytes;

    __host__ __device__ int n_slots() const { return n_pages << page_shift; }
    // Offset, from the layer's start, of the group of slot s in head h.
    __host__ __device__ int64_t group_offset(int slot, int h) const {
        const int in_page = (slot & (page - 1)) >> (page_shift - group_shift);  // a group: page_size / 2^group_shift
        return (int64_t) (slot >> page_shift) * page_bytes + (((int64_t) h << group_shift) + in_page) * kGroupBytes;
    }
};

inline PagesGeom make_pages_geom(int n_layers, int n_pages, int page, int n_kv, int dim) {
    PagesGeom g{};
    g.n_layers = n_layers;
    g.n_pages = n_pages;
    g.page = page;
    g.n_kv = n_kv;
    g.dim = dim;
    while ((1 << g.page_shift) < page) ++g.page_shift;
    const int groups = page / keys_per_group(dim);
    while ((1 << g.group_shift) < groups) ++g.group_shift;
    g.page_bytes = (int64_t) n_kv * groups * kGroupBytes;
    g.layer_bytes = g.page_bytes * n_pages;
    return g;
}

}  // namespace bmo
