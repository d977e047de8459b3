// rows.hpp -- parameter blocks and launchers of the operators on rows between
// two attentions: norm, 8-bit rows, rotary positions, products with Q4_0
// weights (internal to libbmo_attn.so; the public surface is
// include/bmo_attn.h).
//
// 8-bit rows: int8 codes [rows][cols] and fp16 scales [rows][cols / 32].
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pages.hpp"  // the element types

namespace bmo {

// ---- norm (rows_norm.hip) -----------------------------------------------------

constexpr int kNormMaxDim = 32768;

struct NormParams {
    int n_rows;
    int dim;
    int type;
    const void *x;
    int64_t x_stride;
    int res_type;
    void *res;  // nullable: x is added to it
    int64_t res_stride;
    int w_type;
    const void *w;
    float eps;
    int out_type;
    void *out;  // nullable
    int64_t out_stride;
    int8_t *codes;     // nullable, with scales
    uint16_t *scales;  // fp16
};
hipError_t launch_norm(const NormParams &p, hipStream_t stream);

struct QuantizeParams {
    int n_rows;
    int cols;
    int type;
    const void *x;
    int64_t stride;
    int8_t *codes;
    uint16_t *scales;
};
hipError_t launch_quantize_rows(const QuantizeParams &p, hipStream_t stream);

// ---- rotary positions (rows_rope.hip) -------------------------------------------

struct RopePart {  // rows [tokens][heads][dim]
    int heads;
    const void *x;
    int64_t stride;
    void *out;
    int64_t out_stride;
};
struct RopeParams {
    const double *rates;  // device [rot / 2]: radians a position
    float magnitude;
    int dim;
    int rot;
    int interleaved;
    int n_tok;
    const int *positions;
    int type;
    RopePart part[2];  // the second may have no heads
};
hipError_t launch_rope(const RopeParams &p, hipStream_t stream);

// ---- Q4_0 weights (weights.hip) ---------------------------------------------------

// A matrix of rows x cols lies in units of 16 rows x 128 columns, the units of
// 16 rows one after another, zeros past its edges.  A unit is 1152 bytes:
//
//   [0, 1024)     codes: dword ((g * 16 + i) * 4 + t) holds elements 8g .. 8g+7
//                 of block t of row i, each code - 8 as a signed nibble, byte j
//                 element 8g + j (low) and 8g + 4 + j (high)
//   [1024, 1152)  scales, fp16: element i * 4 + t is that of block t of row i
//
// The 16 bytes at lane * 16 are what lane (g, i) of a 16x16x32 integer matrix
// instruction takes of four blocks: the high nibbles of a dword in place and
// the low ones shifted are 16 (code - 8) as bytes.
constexpr int kUnitRows = 16, kUnitCols = 128, kUnitBytes = 1152, kUnitScales = 1024;

struct WeightsGeom {
    int rows, cols;
    int tiles;   // of 16 rows, an even number
    int chunks;  // of 128 columns
};
inline WeightsGeom make_weights_geom(int rows, int cols) {
    return {rows, cols, (rows + 2 * kUnitRows - 1) / (2 * kUnitRows) * 2, (cols + kUnitCols - 1) / kUnitCols};
}
inline int64_t weights_bytes(const WeightsGeom &g) { return (int64_t) g.tiles * g.chunks * kUnitBytes; }

struct PackParams {
    uint8_t *w;
    WeightsGeom g;
    int row0;
    int n_rows;
    const uint8_t *blocks;  // ggml block_q4_0 [n_rows][cols / 32]
};
hipError_t launch_weights_pack(const PackParams &p, hipStream_t stream);

enum Activation { kNoActivation = 0, kSilu = 1, kGelu = 2 };

struct ProductParams {
    const uint8_t *w;
    WeightsGeom g;
    int n_rows;
    const int8_t *codes;
    const uint16_t *scales;
    int activation;  // else: rows of the first half are gates of the second's
    int type;
    void *out;           // nullable where the result goes to 8 bits
    int64_t out_stride;
    int8_t *out_codes;   // nullable (gated only)
    uint16_t *out_scales;
};
hipError_t launch_product(const ProductParams &p, hipStream_t stream);

}  // namespace bmo
