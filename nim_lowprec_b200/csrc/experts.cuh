// experts.cuh -- the layout of experts' weights as the products read them, and the
// products' arguments.
#pragma once
#include "lp_device.cuh"
#include "lp_internal.h"

namespace lp {
namespace experts {

constexpr int kTileM = 128;   // weight rows of a tile (gated: 64 features, gate and up)
constexpr int kChunkK = 128;  // elements of K of a tile: one 128-byte swizzled row of 8-bit containers
constexpr int kSplitN = 64;   // most rows of a tile whose K may be cut
constexpr int64_t kCounterBytes = 4096;  // one 4-byte counter per CTA of a launch
constexpr int kSfBytes = 512; // scale factors of a tile: 128 rows x 4 blocks of 32

struct Layout {
  int64_t mtiles, kchunks, tiles;     // tiles: experts * mtiles * kchunks
  int64_t tile_bytes;                 // codes of a tile: 8192 (e2m1) or 16384 (e4m3)
};
inline Layout layout(int64_t experts, int64_t rows, int64_t cols, int dtype, bool gated) {
  Layout l;
  l.mtiles = gated ? (rows / 2 + 63) / 64 : (rows + kTileM - 1) / kTileM;
  l.kchunks = (cols + kChunkK - 1) / kChunkK;
  l.tiles = experts * l.mtiles * l.kchunks;
  l.tile_bytes = kTileM * kChunkK / (dtype == LP_E2M1 ? 2 : 1);
  return l;
}

// The row of the expert's matrix that row r of tile mt holds, -1 for none.  Gated:
// each 32 rows (a warp's accumulator lanes) are 16 gate rows and the 16 up rows of
// the same features.
__host__ __device__ inline int64_t source_row(int64_t mt, int r, int64_t rows, bool gated) {
  if (!gated) {
    const int64_t m = mt * kTileM + r;
    return m < rows ? m : -1;
  }
  const int64_t inner = rows / 2, f = mt * 64 + 16 * (r >> 5) + (r & 15);
  return f < inner ? (r & 16 ? inner + f : f) : -1;
}

// The workspace: counters (zero between calls), then the router's counts or the partial
// sums of cut tiles, then rows gathered into the experts' order, codes and scales.
inline int64_t fixed_workspace() {
  const int64_t counts = int64_t{kRouteCtas} * kRouteExperts * 4;
  const int64_t partials = device_info().sm_count * 2ll * kSplitN * kTileM * 4;
  return kCounterBytes + (counts > partials ? counts : partials);
}
inline int64_t scale_row(int64_t cols) { return (cols / 32 + 15) / 16 * 16; }
inline int64_t gather_workspace(int64_t rows, int64_t cols) { return rows * (cols + scale_row(cols)); }
inline lp_rows8 gathered_rows(int64_t rows, int64_t cols, uint8_t* at) {
  return {at, at + rows * cols, rows, cols, cols, scale_row(cols), LP_E4M3, 32};
}

struct Args {
  const uint8_t* wscales;     // atoms, in the order of the tiles
  const uint8_t* xscales;     // E8M0 bytes of the 8-bit rows
  int64_t xscale_stride;
  int xscale_words;           // four scales of a row can be read at once
  int sf_rows, sf_block;      // bytes of the rows' scale factors of a chunk, of four chunks' of both sides
  const int32_t* offsets;
  int experts, mtiles, kchunks, k;
  int rows, tokens;           // rows of the result, rows of x
  int gathered;               // the rows come from the kernel before
  int bn;                     // most rows of a tile, a multiple of 16
  int stages;
  int split;                  // tiles per CTA below which they are cut along K (0: never)
  uint32_t a_bytes;           // of a tile's codes
  uint32_t idesc;             // without N and the scale factors' ids
  uint8_t* out;               // rows (bytes between them: out_stride) or codes
  int64_t out_stride;
  uint8_t* out_scales;        // gated
  int64_t out_scale_stride;
  int out_type;
  int features;               // columns of the result
  float* partials;
  uint32_t* counters;
};

}  // namespace experts
}  // namespace lp
