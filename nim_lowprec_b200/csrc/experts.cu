// experts.cu -- products of 8-bit rows with their experts' weights, on the
// block-scaled 5th-generation tensor cores.
//
//   y[r, m] = sum_k W[e(r)][m, k] x[t(r), k]
//   gated:  h[r, f] = silu(g) u, g = y[r, f], u = y[r, inner + f], as MXFP8 rows
//
// e(r) is the expert whose segment [offsets[e], offsets[e+1]) holds row r; t(r) =
// row_token[r], or r.  Weights are MXFP4 (e2m1) or MXFP8 (e4m3), x is MXFP8: one
// E8M0 scale per 32 elements of K on both sides, which tcgen05.mma
// kind::mxf8f6f4.block_scale applies, so products are exact and sums are fp32.
//
// The weights are operand A (128 rows of a tile are the accumulator's lanes) and
// the rows are operand B (its columns): the rows of an expert are few or many and
// ragged, and N may be any multiple of 16, while M is fixed.  One row costs the
// 16 columns that the weights' stream hides; 240 (two accumulators and the scale
// factors fill the 512 columns of tensor memory) run at the tensor cores' rate.
//
// Weights are laid out once (ExpertWeights): tiles of 128 rows x 128 elements, each
// contiguous, e2m1 at 4 bits (TMA spreads them into the 8-bit containers that the
// MMA reads), scale factors as the 512-byte atoms that tcgen05.cp takes.  So a
// stage is one contiguous read of 8 (16) KB and one of 512 bytes, and odd sizes of
// M and K end in tiles of zeros instead of in the kernel.
//
// One persistent CTA per SM, 8 warps:
//   warp 0     producer: per stage the tile's codes and scales, and the rows' codes
//              by tile (rows in order) or by gather of four rows (row_token)
//   warp 1     copies scale factors to tensor memory and issues the MMAs
//   warps 2-3  the rows' scale factors, gathered, into atoms
//   warps 4-7  epilogue, while the next tile's MMAs fill the other accumulator
// Every wait is bounded, and tensor memory is freed on every path.
#include <cuda.h>

#include <algorithm>

#include "experts.cuh"
#include "rows.cuh"
#include "tc_ptx.cuh"

namespace lp {
namespace {

using namespace tc;
using namespace experts;

// ------------------------------------------------------------- layout
struct PackArgs {
  const uint8_t* codes;   // experts x rows x cols
  const uint8_t* scales;  // experts x rows x cols / 32, fp32 or E8M0 bytes
  uint8_t *tiles, *atoms;
  int64_t experts, rows, cols, mtiles, kchunks;
  int fp4, scale_f32, gated, vec;
};

__global__ void __launch_bounds__(256) k_pack_codes(const PackArgs a) {
  const int per = a.fp4 ? 4 : 8;  // 16-byte pieces of a tile's row
  const int64_t n = a.experts * a.mtiles * a.kchunks * kTileM * per;
  const int64_t row_bytes = a.fp4 ? a.cols / 2 : a.cols;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int piece = static_cast<int>(i % per), r = static_cast<int>(i / per % kTileM);
    const int64_t tile = i / (per * kTileM), kc = tile % a.kchunks, mt = tile / a.kchunks % a.mtiles;
    const int64_t e = tile / (a.kchunks * a.mtiles), m = source_row(mt, r, a.rows, a.gated);
    const int64_t at = kc * (per * 16) + piece * 16;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (m >= 0 && at < row_bytes) {
      const uint8_t* p = a.codes + (e * a.rows + m) * row_bytes + at;
      if (a.vec) {
        v = *reinterpret_cast<const uint4*>(p);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < 16; ++b) w[b >> 2] |= static_cast<uint32_t>(p[b]) << (8 * (b & 3));
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    reinterpret_cast<uint4*>(a.tiles)[i] = v;
  }
}

// Byte of scale block j (of 4) of row r in an atom.
__device__ __forceinline__ int sf_off(int r, int j) { return 16 * (r & 31) + 4 * (r >> 5) + j; }

__global__ void __launch_bounds__(256) k_pack_scales(const PackArgs a) {
  const int64_t n = a.experts * a.mtiles * a.kchunks * kTileM, nsf = a.cols / 32;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int r = static_cast<int>(i % kTileM);
    const int64_t tile = i / kTileM, kc = tile % a.kchunks, mt = tile / a.kchunks % a.mtiles;
    const int64_t e = tile / (a.kchunks * a.mtiles), m = source_row(mt, r, a.rows, a.gated);
    uint32_t word = 0;
    for (int j = 0; j < 4; ++j) {
      const int64_t b = 4 * kc + j;
      if (m < 0 || b >= nsf) continue;
      const int64_t at = (e * a.rows + m) * nsf + b;
      // an fp32 scale is a power of two: its exponent field is the E8M0 code
      const uint32_t code = a.scale_f32 ? __float_as_uint(reinterpret_cast<const float*>(a.scales)[at]) >> 23 & 255u
                                        : a.scales[at];
      word |= code << (8 * j);
    }
    *reinterpret_cast<uint32_t*>(a.atoms + tile * kSfBytes + sf_off(r, 0)) = word;
  }
}

// -------------------------------------------------------------- product
constexpr int kThreads = 256;
constexpr int kMaxN = 240;
constexpr uint32_t kTmemCols = 512, kSfCol = 480;  // accumulators at 0 and 240
constexpr int kSfStage = kSfBytes + 1024;          // A's atom, and B's two
constexpr int kGateTokens = 32, kGatePitch = 65;   // the gated epilogue's transposition
constexpr int kGateBytes = kGateTokens * kGatePitch * 4;

__device__ __forceinline__ uint64_t sf_desc(const void* p) {
  uint64_t d = static_cast<uint64_t>((saddr(p) & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 16;  // core matrices of 8 rows x 16 bytes, one wide
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
__device__ __forceinline__ void sf_copy(uint32_t taddr, const void* atom) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sf_desc(atom)) : "memory");
}
__device__ __forceinline__ void mma_mx8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                        uint32_t sfb, bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; "
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p; }" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(sfa), "r"(sfb)
      : "memory");
}
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* tm, int col, const int* row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(saddr(dst)),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(col), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]),
      "r"(saddr(bar))
      : "memory");
}
__device__ __forceinline__ void bulk_in(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   saddr(dst)),
               "l"(src), "r"(bytes), "r"(saddr(bar))
               : "memory");
}

// The segments, as every CTA reads them from the offsets: an expert's first row,
// its rows, and the tiles of the experts before it.  Offsets are clamped to the
// rows there are, so that no value in them leads out of range.
struct Segments {
  int *row0, *rows, *start;  // start: experts + 1
};
__device__ __forceinline__ int tiles_of(int rows, int bn) { return (rows + bn - 1) / bn; }
// Rows of each tile of a segment: as many tiles as needed, alike, a multiple of 16.
__device__ __forceinline__ int rows_per(int rows, int bn) {
  const int nt = max(1, tiles_of(rows, bn));
  return ((rows + nt - 1) / nt + 15) & ~15;
}

__device__ __forceinline__ void read_segments(const Args& a, const Segments& s, int lane) {
  int carry = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, n = 0, tiles = 0;
    if (e < a.experts) {
      lo = min(max(__ldg(a.offsets + e), 0), a.rows);
      n = max(min(__ldg(a.offsets + e + 1), a.rows) - lo, 0);
      if (n > 0) {
        const int per = rows_per(n, a.bn);
        tiles = min((n + per - 1) / per * a.mtiles, 1 << 24);
      }
    }
    int inc = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    inc = min(inc + carry, 1 << 30);  // (more than any segments in order come to)
    if (e < a.experts) {
      s.row0[e] = lo;
      s.rows[e] = n;
      s.start[e + 1] = inc;
    }
    carry = __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) s.start[0] = 0;
}

// A CTA's work, in order.  Every warp walks it by itself.
struct Tile {
  int e, mt, row0, n;  // expert, weight tile, first row, rows
};
struct Walk {
  const Args& a;
  const Segments& s;
  int t, e = 0;
  __device__ Walk(const Args& args, const Segments& seg) : a(args), s(seg), t(blockIdx.x) {}
  __device__ __forceinline__ bool next(Tile& w) {
    if (t >= s.start[a.experts]) return false;
    while (t >= s.start[e + 1]) ++e;
    const int rows = s.rows[e], per = rows_per(rows, a.bn), nt = (rows + per - 1) / per;
    const int at = t - s.start[e], j = at % nt;
    w.e = e;
    w.mt = at / nt;
    w.row0 = s.row0[e] + j * per;
    w.n = min(per, rows - j * per);
    t += gridDim.x;
    return true;
  }
};

// Four chunks' scale words of one row (nsf scales) from block `blk` of four chunks on.
__device__ __forceinline__ uint4 load_scales(const Args& a, const uint8_t* p, int blk, int nsf) {
  uint32_t w[4] = {0, 0, 0, 0};
  if (p == nullptr) return make_uint4(0, 0, 0, 0);
  const int b0 = 16 * blk;
  if (a.xscale_vec == 16 && b0 + 16 <= nsf) return *reinterpret_cast<const uint4*>(p + b0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int b = b0 + 4 * j;
    if (a.xscale_vec >= 4) {
      if (b < nsf) w[j] = *reinterpret_cast<const uint32_t*>(p + b);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b + i < nsf) w[j] |= static_cast<uint32_t>(p[b + i]) << (8 * i);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float silu_mul(float g, float u) {
  // g / (1 + exp(-g)); the quotient's two units in the last place are far below the
  // e4m3 code's rounding
  return fmul(__fdividef(g, fadd(1.0f, __expf(-g))), u);
}

__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
    k_experts(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Args a) {
  constexpr int kMaxStages = 12;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], sfull[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], done;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int s_abort;

  uint8_t* smem = smem_raw + ((1024u - (saddr(smem_raw) & 1023u)) & 1023u);
  const int stage_bytes = kTileM * kChunkK + a.bn * kChunkK;
  uint8_t* sf_mem = smem + a.stages * stage_bytes;
  uint8_t* gate_mem = sf_mem + a.stages * kSfStage;
  int* seg_mem = reinterpret_cast<int*>(gate_mem + (GATED ? kGateBytes : 0));
  const Segments seg{seg_mem, seg_mem + a.experts, seg_mem + 2 * a.experts};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&sfull[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4);
    }
    mbar_init(&done, 1);
    s_abort = 0;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc(&tmem_base, kTmemCols);
  if (warp == 0) read_segments(a, seg, lane);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tbase = tmem_base;
  Walk walk(a, seg);
  Tile w;

  if (warp == 0) {
    // ------------------------------------------------------ producer
    int it = 0, s = 0, phase = 0;
    bool more = walk.next(w);
    int idx[2][4], nidx[2][4];
    auto rows_of = [&](const Tile& t, int (&ix)[2][4]) {
      // rows past the tile's are row `tokens`, which TMA fills with zeros
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = 4 * (lane + 32 * i) + j;
          int row = a.tokens;
          if (c < t.n) {
            const int v = __ldg(a.row_token + t.row0 + c);
            if (static_cast<uint32_t>(v) < static_cast<uint32_t>(a.tokens)) row = v;
          }
          ix[i][j] = row;
        }
      }
    };
    if (more && a.row_token) rows_of(w, nidx);
    while (more) {
      const int n16 = (w.n + 15) & ~15;
      const int64_t tile = (static_cast<int64_t>(w.e) * a.mtiles + w.mt) * a.kchunks;
      const int row0 = w.row0;
      if (a.row_token) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) idx[i][j] = nidx[i][j];
      }
      more = walk.next(w);
      if (more && a.row_token) rows_of(w, nidx);
      for (int kc = 0; kc < a.kchunks; ++kc, ++it) {
        bool ok = true;
        if (it >= a.stages) ok = mbar_wait(&empty[s], phase ^ 1, &s_abort);
        ok = __all_sync(0xffffffffu, ok && !s_abort);
        if (!ok) break;
        uint8_t* st = smem + s * stage_bytes;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[s], a.a_bytes + kSfBytes + n16 * kChunkK);
          tma_load_2d(st, &tmA, 0, static_cast<int>((tile + kc) * kTileM), &full[s]);
          bulk_in(sf_mem + s * kSfStage, a.wscales + (tile + kc) * kSfBytes, kSfBytes, &full[s]);
        }
        __syncwarp();
        uint8_t* b = st + kTileM * kChunkK;
        if (a.row_token) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int g = lane + 32 * i;
            if (4 * g < n16) tma_gather4(b + g * 4 * kChunkK, &tmB, kc * kChunkK, idx[i], &full[s]);
          }
        } else if (16 * lane < n16) {
          tma_load_2d(b + lane * 16 * kChunkK, &tmB, kc * kChunkK, row0 + 16 * lane, &full[s]);
        }
        if (++s == a.stages) s = 0, phase ^= 1;
      }
      if (s_abort) break;
    }
    // copies in flight end before the CTA does
    for (int u = max(0, it - a.stages); u < it; ++u) mbar_wait(&full[u % a.stages], (u / a.stages) & 1);
  } else if (warp == 1) {
    // --------------------------------------------------- MMA issuer
    if (lane == 0) {
      int s = 0, phase = 0, item = 0, it = 0;
      bool ok = true;
      while (ok && walk.next(w)) {
        const int buf = item & 1;
        if (item >= 2) ok = mbar_wait(&acc_empty[buf], ((item >> 1) & 1) ^ 1, &s_abort);
        fence_after();
        const int n16 = (w.n + 15) & ~15;
        const uint32_t idesc = a.idesc | static_cast<uint32_t>(n16 >> 3) << 17;
        const uint32_t acc = tbase + buf * kMaxN;
        for (int kc = 0; ok && kc < a.kchunks; ++kc, ++it) {
          ok = mbar_wait(&full[s], phase, &s_abort) && mbar_wait(&sfull[s], phase, &s_abort) && !s_abort;
          if (!ok) break;
          fence_after();
          const uint8_t* st = smem + s * stage_bytes;
          const uint8_t* sf = sf_mem + s * kSfStage;
          const uint32_t sfa = tbase + kSfCol + (it & 1) * 12, sfb = sfa + 4;
          sf_copy(sfa, sf);
          sf_copy(sfb, sf + kSfBytes);
          if (n16 > 128) sf_copy(sfb + 4, sf + kSfBytes + 512);
          const uint64_t ad = sw128_desc(st), bd = sw128_desc(st + kTileM * kChunkK);
          const int blocks = min(4, (a.k - kc * kChunkK) >> 5);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < blocks)
              mma_mx8(acc, ad + 2 * j, bd + 2 * j, idesc | static_cast<uint32_t>(j) << 4 | static_cast<uint32_t>(j) << 29,
                      sfa | static_cast<uint32_t>(j) << 30, sfb | static_cast<uint32_t>(j) << 30, kc > 0 || j > 0);
          }
          mma_commit(&empty[s]);
          if (++s == a.stages) s = 0, phase ^= 1;
        }
        mma_commit(&acc_full[buf]);
        ++item;
      }
      // every MMA issued must be finished before tensor memory is freed
      mma_commit(&done);
      mbar_wait(&done, 0);
    }
  } else if (warp < 4) {
    // ------------------------------------------- the rows' scale factors
    const int first = (warp - 2) * 32 + lane, nsf = a.k >> 5, blks = (a.kchunks + 3) / 4;
    const uint8_t *row[4], *nrow[4];
    uint4 nxt[4];
    auto rows_of = [&](const Tile& t, const uint8_t* (&p)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = first + 64 * i;
        p[i] = nullptr;
        if (c < t.n) {
          const int v = a.row_token ? __ldg(a.row_token + t.row0 + c) : t.row0 + c;
          if (static_cast<uint32_t>(v) < static_cast<uint32_t>(a.tokens)) p[i] = a.xscales + v * a.xscale_stride;
        }
      }
    };
    int it = 0, s = 0, phase = 0;
    bool more = walk.next(w), ok = true;
    if (more) {
      rows_of(w, nrow);
#pragma unroll
      for (int i = 0; i < 4; ++i) nxt[i] = load_scales(a, nrow[i], 0, nsf);
    }
    while (more && ok) {
      const int n = w.n;
#pragma unroll
      for (int i = 0; i < 4; ++i) row[i] = nrow[i];
      more = walk.next(w);
      if (more) rows_of(w, nrow);
      for (int blk = 0; ok && blk < blks; ++blk) {
        uint32_t cur[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          cur[i][0] = nxt[i].x, cur[i][1] = nxt[i].y, cur[i][2] = nxt[i].z, cur[i][3] = nxt[i].w;
        }
        if (blk + 1 < blks) {
#pragma unroll
          for (int i = 0; i < 4; ++i) nxt[i] = load_scales(a, row[i], blk + 1, nsf);
        } else if (more) {
#pragma unroll
          for (int i = 0; i < 4; ++i) nxt[i] = load_scales(a, nrow[i], 0, nsf);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (4 * blk + j >= a.kchunks) break;
          if (it >= a.stages) ok = mbar_wait(&empty[s], phase ^ 1, &s_abort);
          ok = __all_sync(0xffffffffu, ok && !s_abort);
          if (!ok) break;
          uint8_t* atoms = sf_mem + s * kSfStage + kSfBytes;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = first + 64 * i;
            if (64 * i < n) *reinterpret_cast<uint32_t*>(atoms + 512 * (c >> 7) + sf_off(c & 127, 0)) = cur[i][j];
          }
          // generic writes, read by tcgen05.cp through the asynchronous proxy
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[s]);
          ++it;
          if (++s == a.stages) s = 0, phase ^= 1;
        }
      }
    }
  } else {
    // ------------------------------------------------------ epilogue
    const int q = warp & 3;  // the warp's lanes of tensor memory
    const uint32_t lanes = static_cast<uint32_t>(32 * q) << 16;
    float* gate = reinterpret_cast<float*>(gate_mem);
    int item = 0;
    while (walk.next(w)) {
      const int buf = item & 1;
      bool ok = mbar_wait(&acc_full[buf], (item >> 1) & 1, &s_abort);
      ok = __all_sync(0xffffffffu, ok && !s_abort);
      if (!ok) break;
      fence_after();
      const uint32_t acc = tbase + lanes + buf * kMaxN;
      if constexpr (!GATED) {
        const int m = w.mt * kTileM + 32 * q + lane;
        uint8_t* out = a.out + w.row0 * a.out_stride + static_cast<int64_t>(m) * size_of(a.out_type);
        for (int c0 = 0; c0 < w.n; c0 += 16) {
          uint32_t v[16];
          tmem_ld16(acc + c0, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(v[i]));
          if (m < a.features) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (c0 + i < w.n) store1_of(out + (c0 + i) * a.out_stride, __uint_as_float(v[i]), a.out_type);
          }
        }
      } else {
        for (int c0 = 0; c0 < w.n; c0 += kGateTokens) {
          uint32_t v[32];
          tmem_ld32(acc + c0, v);  // (past the tile's columns: whatever is there, not stored)
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(v[i]));
          const bool up = lane & 16;  // this lane holds an up row; its partner the gate's
          const int f = 16 * q + (lane & 15);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[16 + i], 16);
            const float g = __uint_as_float(up ? other : v[i]), u = __uint_as_float(up ? v[16 + i] : other);
            gate[(i + (up ? 16 : 0)) * kGatePitch + f] = silu_mul(g, u);
          }
          epilogue_sync();
          // 16 features of a token each; two lanes hold a block of 32
          const int t = 8 * q + (lane >> 2), f0 = 16 * (lane & 3), feature = w.mt * 64 + f0;
          float x[16], top = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[i] = gate[t * kGatePitch + f0 + i];
            top = fmaxf(top, fabsf(x[i]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          const uint32_t code = mx8_scale(top);
          const float inv = mx8_inverse(code);
          if (c0 + t < w.n && feature < a.features) {
            const int64_t row = w.row0 + c0 + t;
            *reinterpret_cast<uint4*>(a.out + row * a.out_stride + feature) =
                make_uint4(e4m3x4(x, inv), e4m3x4(x + 4, inv), e4m3x4(x + 8, inv), e4m3x4(x + 12, inv));
            if (!(lane & 1)) a.out_scales[row * a.out_scale_stride + (feature >> 5)] = static_cast<uint8_t>(code);
          }
          epilogue_sync();
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[buf]);
      ++item;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    tmem_dealloc(tbase, kTmemCols);
  }
}

bool encode_tiles(CUtensorMap* tm, const void* base, int64_t tiles, bool fp4) {
  EncodeFn fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kChunkK), static_cast<cuuint64_t>(tiles * kTileM)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(fp4 ? kChunkK / 2 : kChunkK)};
  const cuuint32_t box[2] = {kChunkK, kTileM}, one[2] = {1, 1};
  return fn(tm, fp4 ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
            const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool encode_rows(CUtensorMap* tm, const void* base, int64_t cols, int64_t rows, int64_t stride, int box_rows) {
  EncodeFn fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kChunkK, static_cast<cuuint32_t>(box_rows)}, one[2] = {1, 1};
  return fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GATED>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const Args& a, int smem, cudaStream_t st) {
  const DeviceInfo& di = device_info();
  auto kern = k_experts<GATED>;
  static int set[kMaxDevices];
  const int slot = di.ordinal % kMaxDevices;
  if (set[slot] < smem) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, di.max_smem_optin - 1024);
    if (e != cudaSuccess) return cuda_status(e);
    set[slot] = di.max_smem_optin - 1024;
  }
  kern<<<di.sm_count, kThreads, smem, st>>>(ta, tb, a);
  return cuda_status(cudaGetLastError());
}

}  // namespace

int launch_pack_experts(const void* codes, const void* scales, int scale_type, const lp_expert_weights& w,
                        cudaStream_t st) {
  const Layout l = layout(w.experts, w.rows, w.cols, w.dtype, w.gated);
  const PackArgs a{static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales),
                   static_cast<uint8_t*>(w.tiles), static_cast<uint8_t*>(w.scales),
                   w.experts, w.rows, w.cols, l.mtiles, l.kchunks,
                   w.dtype == LP_E2M1, scale_type == LP_F32, w.gated,
                   (reinterpret_cast<uintptr_t>(codes) & 15) == 0};
  const int grid = device_info().sm_count * 16;
  k_pack_codes<<<grid, 256, 0, st>>>(a);
  k_pack_scales<<<grid, 256, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

int launch_experts(const lp_expert_weights& w, const lp_rows8& x, const int32_t* offsets, const int32_t* row_token,
                   int64_t rows, const lp_matrix* out, const lp_rows8* out8, void* workspace, cudaStream_t st) {
  const Layout l = layout(w.experts, w.rows, w.cols, w.dtype, w.gated);
  Args a{};
  a.wscales = static_cast<const uint8_t*>(w.scales);
  a.xscales = static_cast<const uint8_t*>(x.scales);
  a.xscale_stride = x.scale_stride;
  const uintptr_t al = reinterpret_cast<uintptr_t>(x.scales) | static_cast<uintptr_t>(x.scale_stride);
  // (a word holds four scales of one row where a row has a multiple of four)
  a.xscale_vec = x.cols % kChunkK ? 1 : (al & 15) == 0 ? 16 : (al & 3) == 0 ? 4 : 1;
  a.offsets = offsets;
  a.row_token = row_token;
  a.experts = static_cast<int>(w.experts);
  a.mtiles = static_cast<int>(l.mtiles);
  a.kchunks = static_cast<int>(l.kchunks);
  a.k = static_cast<int>(w.cols);
  a.rows = static_cast<int>(rows);
  a.tokens = static_cast<int>(x.rows);
  a.a_bytes = static_cast<uint32_t>(l.tile_bytes);
  // A e2m1 (5) or e4m3 (0), B e4m3, both K-major, E8M0 scales, M = 128
  a.idesc = (w.dtype == LP_E2M1 ? 5u << 7 : 0u) | 1u << 23 | static_cast<uint32_t>(128 >> 4) << 24;
  if (out) {
    a.out = static_cast<uint8_t*>(out->data);
    a.out_stride = out->stride * size_of(out->dtype);
    a.out_type = out->dtype;
    a.features = static_cast<int>(out->cols);
  } else {
    a.out = static_cast<uint8_t*>(out8->codes);
    a.out_stride = out8->code_stride;
    a.out_scales = static_cast<uint8_t*>(out8->scales);
    a.out_scale_stride = out8->scale_stride;
    a.features = static_cast<int>(out8->cols);
  }
  a.partials = static_cast<float*>(workspace);
  // A token has at most one row per expert, so no segment is longer than x.
  const int64_t most = row_token ? std::min(rows, x.rows) : rows;
  const int64_t mean = (rows + w.experts - 1) / w.experts;
  int bn = kMaxN;
  if (mean <= 16) bn = 32;
  else if (mean <= 48) bn = 64;
  else if (mean <= 112) bn = 128;
  a.bn = static_cast<int>(std::min<int64_t>(bn, (most + 15) / 16 * 16));
  const int fixed = 1024 + (w.gated ? kGateBytes : 0) + static_cast<int>(3 * w.experts + 1) * 4;
  const int stage = (kTileM + a.bn) * kChunkK + kSfStage;
  a.stages = std::min(12, (device_info().max_smem_optin - 1024 - fixed) / stage);
  if (a.stages < 2) return LP_ERR_UNSUPPORTED;
  CUtensorMap ta, tb;
  if (!encode_tiles(&ta, w.tiles, l.tiles, w.dtype == LP_E2M1) ||
      !encode_rows(&tb, x.codes, x.cols, x.rows, x.code_stride, row_token ? 1 : 16))
    return LP_ERR_UNSUPPORTED;
  const int smem = fixed + a.stages * stage;
  return w.gated ? launch<true>(ta, tb, a, smem, st) : launch<false>(ta, tb, a, smem, st);
}

unsigned int take_error_experts() {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(v)) != cudaSuccess) return LP_ERR_CUDA;
  if (v) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_device_error, &z, sizeof(z));
  }
  return v;
}

}  // namespace lp
