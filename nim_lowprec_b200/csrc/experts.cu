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
// One persistent CTA per SM (or pair of CTAs, whose MMAs take 256 weight rows and the
// rows' halves from both), 16 warps:
//   warp 0       the weights' tiles and, a block of four chunks at a time, their scales
//   warp 1       copies scale factors to tensor memory and issues the MMAs (of a pair, in the
//                leading CTA; in the other it passes on that scale factors are there)
//   warp 2       the rows, a box of up to 240 of them
//   warps 8-11   the rows' scale factors, word by word into atoms (cp.async)
//   warps 4-7, 12-15  epilogue, taking turns with the two accumulators
// Rows named by row_token are gathered by a kernel of their own first.
//
// What bounds it (B200).  Few rows: the weights' bytes, 57 tokens over 8 experts of 28672 x
// 4096 in e2m1 105 us (4.7 TB/s, 5.5 between start and join); the smallest calls the chain of
// offsets, first loads and joins (one token over 8 of 64 experts, 23 MB: 12 us, of which 5
// stream).  Many rows: the products, 64 experts x 1024 rows gated 1.9 to 2.0 PFLOP/s back to
// back; a step of two chunks takes about 1000 cycles where its MMAs take 800 to 960.
// Every wait is bounded, and tensor memory is freed on every path.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

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

// --------------------------------------------------------------- gather
// Rows into the experts' order, scales padded with zeros to whole 16 bytes.  (The
// products' own loaders gathering row by row was slower: a gather of four rows costs
// TMA as much as a tile of 128, and copies of 16 bytes by threads made a prompt's
// gated product 690 us where this and tiles take 390.)
struct GatherArgs {
  const uint8_t *codes, *scales;
  uint8_t *to, *to_scales;
  int64_t code_stride, scale_stride, to_scale_stride;
  const int32_t *end, *row_token;  // end: offsets[experts]
  int64_t rows, tokens;
  int cols;
};
__global__ void __launch_bounds__(256) k_gather(const GatherArgs a) {
  // The product after this one begins once every CTA here has passed the wait: whatever came
  // before the gather is there then, and the product waits for the gathered rows alone.
  asm volatile("griddepcontrol.wait; griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, cp = a.cols / 16, nsf = a.cols / 32;
  const int64_t rows = min(a.rows, static_cast<int64_t>(max(__ldg(a.end), 0)));
  // a warp a row, 16 bytes a lane, four at a time
  for (int64_t row = blockIdx.x * 8ll + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
    const int token = __ldg(a.row_token + row);
    const bool in = static_cast<uint32_t>(token) < static_cast<uint32_t>(a.tokens);
    const uint4* from = reinterpret_cast<const uint4*>(a.codes + (in ? token : 0) * a.code_stride);
    const uint8_t* sf = a.scales + (in ? token : 0) * a.scale_stride;
    uint4* to = reinterpret_cast<uint4*>(a.to + row * a.cols);
    for (int p0 = lane; p0 < cp; p0 += 128) {
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = in && p0 + 32 * i < cp ? __ldg(from + p0 + 32 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p0 + 32 * i < cp) to[p0 + 32 * i] = v[i];
    }
    for (int w = lane; w < a.to_scale_stride / 4; w += 32) {
      uint32_t word = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (in && 4 * w + b < nsf) word |= static_cast<uint32_t>(__ldg(sf + 4 * w + b)) << (8 * b);
      reinterpret_cast<uint32_t*>(a.to_scales + row * a.to_scale_stride)[w] = word;
    }
  }
}

// -------------------------------------------------------------- product
constexpr int kThreads = 512;
constexpr int kMaxN = 240;
// Chunks of K to a stage.  A step through the pipeline has fixed costs beside its products
// (a wait, an issue by one lane: about 300 cycles, where a chunk of 16 rows takes 180 and one
// of 240 rows 480), so two chunks share one: 57 tokens over 8 experts 141 -> 107 us.
constexpr int G = 2;
constexpr int kPairRows = 200;   // mean rows per expert above which two CTAs share a tile
constexpr int kSplitTiles = 32;  // tiles per CTA below which they are cut along K
constexpr int kMaxStages = 12;
constexpr int kSfRing = 3;  // blocks of four chunks' scale factors
constexpr uint32_t kTmemCols = 512, kSfCol = 480;  // accumulators at 0 and 240
constexpr int kGateTokens = 32, kGatePitch = 65;   // the gated epilogue's transposition
constexpr int kGateBytes = 2 * kGateTokens * kGatePitch * 4;  // of two groups of warps
constexpr int kBoxes = 5;

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred P; elect.sync _|P, 0xffffffff; selp.u32 %0, 1, 0, P; }" : "=r"(p));
  return p != 0;
}

struct Maps {
  CUtensorMap a;          // weight tiles
  CUtensorMap b[kBoxes];  // rows in order, by boxes of 32, 64, 128, 192 and bn
};

// A block of 32 x 16 bytes at a shared address, as tcgen05.cp reads it.
__device__ __forceinline__ uint64_t sf_desc(uint32_t at) {
  uint64_t d = static_cast<uint64_t>((at & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(128 >> 4) << 16;  // core matrices of 8 rows x 16 bytes, one wide
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}

// The instructions that differ between one CTA and a pair that shares a tile.
template <int CG>
struct Tc;
#define LP_TC(CG)                                                                                              \
  template <>                                                                                                  \
  struct Tc<CG> {                                                                                              \
    static __device__ __forceinline__ void alloc(uint32_t* dst) {                                              \
      asm volatile("tcgen05.alloc.cta_group::" #CG ".sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(saddr(dst)), \
                   "r"(kTmemCols)                                                                              \
                   : "memory");                                                                                \
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::" #CG ".sync.aligned;" ::: "memory");           \
    }                                                                                                          \
    static __device__ __forceinline__ void dealloc(uint32_t t) {                                               \
      asm volatile("tcgen05.dealloc.cta_group::" #CG ".sync.aligned.b32 %0, %1;" ::"r"(t), "r"(kTmemCols)      \
                   : "memory");                                                                                \
    }                                                                                                          \
    static __device__ __forceinline__ void sf_copy(uint32_t t, uint64_t atom) {                                \
      asm volatile("tcgen05.cp.cta_group::" #CG ".32x128b.warpx4 [%0], %1;" ::"r"(t), "l"(atom)                \
                   : "memory");                                                                                \
    }                                                                                                          \
    static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,             \
                                               uint32_t sfa, uint32_t sfb, bool add) {                         \
      asm volatile(                                                                                            \
          "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::" #CG                                  \
          ".kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p; }" ::"r"(d),                           \
          "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(sfa), "r"(sfb)                      \
          : "memory");                                                                                         \
    }                                                                                                          \
  };
LP_TC(1)
LP_TC(2)
#undef LP_TC

// One arrival once every tcgen05 operation issued so far has finished, in each
// CTA of the pair.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
// The same in this CTA alone.
template <int CG>
__device__ __forceinline__ void commit_own(uint64_t* bar) {
  if constexpr (CG == 1) {
    mma_commit(bar);
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(saddr(bar))
                 : "memory");
  }
}
// The leading CTA's barrier of the same name.
template <int CG>
__device__ __forceinline__ uint32_t lead(uint64_t* bar) {
  uint32_t a = saddr(bar);
  if constexpr (CG == 2) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(saddr(bar)));
  return a;
}
template <int CG>
__device__ __forceinline__ void arrive_lead(uint64_t* bar) {
  if constexpr (CG == 1) mbar_arrive(bar);
  else
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lead<2>(bar)) : "memory");
}
// A converged warp waits for a barrier (its shared address), what the other CTA of a
// pair wrote before its arrival included.  Bounded as mbar_wait is.
template <int CG>
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if constexpr (CG == 1)
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSuspendHintNs)
        : "memory");
  else
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSuspendHintNs)
        : "memory");
  return ok != 0;
}
template <int CG>
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile int* abort) {
  const uint64_t t0 = global_ns();
  while (true) {
    if (__all_sync(0xffffffffu, try_wait<CG>(bar, parity))) return true;
    const bool late = global_ns() - t0 > kWaitLimitNs;
    if (__any_sync(0xffffffffu, late)) {
      raise_error(LP_ERR_TIMEOUT);
      *abort = 1;
      return false;
    }
    if (__any_sync(0xffffffffu, *abort != 0)) return false;
  }
}
// Whether a barrier's phase is over, without waiting.  Asked one step ahead, so that the
// answer is there when it is needed: a wait that finds its barrier ready takes about 100
// cycles all the same, half of what a chunk of few rows may take.
template <int CG>
__device__ __forceinline__ bool peek(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if constexpr (CG == 1)
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
  else
    asm volatile(
        "{ .reg .pred p; mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  return ok != 0;
}
template <int CG>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, bool ready = false) {
  if (__all_sync(0xffffffffu, ready)) return true;
  if (__all_sync(0xffffffffu, try_wait<CG>(bar, parity))) return true;
  return wait_longer<CG>(bar, parity, abort);
}
// A tile of rows into this CTA's shared memory, counted at `bar` (a cluster address).
template <int CG>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* tm, int c0, int c1, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tm)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0)
               : "memory");
}
// One arrival of this thread once the copies that it has issued are there.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(saddr(bar)) : "memory");
}

// The segments that have rows, as every CTA reads them from the offsets: the expert, its
// first row, its rows, and the tiles of those before it.  Offsets are clamped to the rows
// there are, so that no value in them leads out of range.
struct Segments {
  int *id, *row0, *rows, *tiles, *start;  // tiles: along the rows; start: one more
  int* count;
};
// Rows of each tile of a segment: as many tiles as needed, alike, a multiple of 16.
__device__ __forceinline__ int rows_per(int rows, int bn) {
  const int nt = (rows + bn - 1) / bn;
  return ((rows + nt - 1) / nt + 15) & ~15;
}

// One warp; the offsets lie in s.start.
__device__ __forceinline__ void read_segments(const Args& a, const Segments& s, int mtiles, int lane) {
  int carry = 0, kept = 0;
  int next = lane < a.experts ? s.start[lane] : 0;
  for (int e0 = 0; e0 < a.experts; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, n = 0, along = 0, tiles = 0;
    if (e < a.experts) {
      lo = min(max(next, 0), a.rows);
      n = max(min(s.start[e + 1], a.rows) - lo, 0);
      if (n > 0) {
        const int per = rows_per(n, a.bn);
        along = (n + per - 1) / per;
        tiles = min(along * mtiles, 1 << 24);
      }
    }
    next = e + 32 < a.experts ? s.start[e + 32] : 0;
    int inc = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    inc = min(inc + carry, 1 << 30);  // (more than any segments in order come to)
    const uint32_t some = __ballot_sync(0xffffffffu, n > 0);
    __syncwarp();  // (what is written below has been read: at most as many as went by)
    if (n > 0) {
      const int at = kept + __popc(some & ((1u << lane) - 1));
      s.id[at] = e;
      s.row0[at] = lo;
      s.rows[at] = n;
      s.tiles[at] = along;
      s.start[at + 1] = inc;
    }
    kept += __popc(some);
    carry = __shfl_sync(0xffffffffu, inc, 31);
    __syncwarp();
  }
  if (lane == 0) {
    s.start[0] = 0;
    *s.count = kept;
  }
}

// A CTA's (or pair's) work, in order.  Every warp walks it by itself.  Where there
// are many tiles, they go round; where there are few, the chunks of all tiles laid
// end to end are cut into equal shares, and a tile that is cut leaves partial sums.
struct Item {
  int e, mt, row0, n;  // expert, weight tile (of the pair), first row, rows
  int k0, k1;          // chunks of K
  int first, parts;    // of a cut tile: the first CTA that has some of it, and how many have
};
struct Walk {
  const Args& a;
  const Segments& s;
  int ctas, step, total, t, e = 0, steps;  // steps: of a tile
  int at = 0, left = 0, share = 0, more = 0;  // steps: into the tile, of this CTA; `more` CTAs have one more than the share
  bool split;
  __device__ Walk(const Args& args, const Segments& seg, int cta, int n)
      : a(args), s(seg), ctas(n), step(n), total(seg.start[*seg.count]), t(cta),
        steps((args.kchunks + G - 1) / G) {
    split = a.split && total < a.split * n && static_cast<int64_t>(total) * steps < (1 << 30);
    if (split) {
      const int units = total * steps;
      ctas = min(n, max(units * G / kLeastChunks, 1));
      share = units / ctas;
      more = units - share * ctas;
      const int first = cta * share + min(cta, more);
      left = cta < ctas ? share + (cta < more ? 1 : 0) : 0;
      t = first / steps;
      at = first - t * steps;
    }
  }
  static constexpr int kLeastChunks = 4;
  __device__ __forceinline__ int cta_of(int unit) const {
    const int big = more * (share + 1);
    return unit < big ? unit / (share + 1) : more + (unit - big) / share;
  }
  __device__ __forceinline__ bool next(Item& w) {
    w.k0 = 0;
    w.k1 = a.kchunks;
    w.parts = 1;
    if (split ? left == 0 : t >= total) return false;
    if (t >= s.start[e + 1]) {  // the last segment that starts at t or before
      int lo = e + 1, hi = *s.count - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t >= s.start[mid]) lo = mid;
        else hi = mid - 1;
      }
      e = lo;
    }
    const int along = s.tiles[e], in = t - s.start[e];
    w.e = s.id[e];
    if (along == 1) {
      w.mt = in;
      w.row0 = s.row0[e];
      w.n = s.rows[e];
    } else {
      const int rows = s.rows[e], per = rows_per(rows, a.bn);
      w.mt = in / along;
      const int j = in - w.mt * along;
      w.row0 = s.row0[e] + j * per;
      w.n = min(per, rows - j * per);
    }
    if (!split) {
      t += step;
      return true;
    }
    const int n = min(steps - at, left);
    if (n < steps) {
      w.k0 = at * G;
      w.k1 = min(a.kchunks, (at + n) * G);
      w.first = cta_of(t * steps);
      w.parts = cta_of(t * steps + steps - 1) - w.first + 1;
    }
    left -= n;
    at = 0;
    ++t;
    return true;
  }
};

__device__ __forceinline__ float silu_mul(float g, float u) {
  // g / (1 + exp(-g)); the quotient's two units in the last place are far below the
  // e4m3 code's rounding
  return fmul(__fdividef(g, fadd(1.0f, __expf(-g))), u);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release; barrier.cluster.wait.acquire;" ::: "memory");
}
// The warps of a group agree: true where all have seen true.
__device__ __forceinline__ bool epilogue_all(bool ok, int group) {
  uint32_t all;
  asm volatile(
      "{ .reg .pred p, q; setp.ne.b32 p, %1, 0; bar.red.and.pred q, %2, 128, p; selp.u32 %0, 1, 0, q; }"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok)), "r"(1 + group)
      : "memory");
  return all != 0;
}
__device__ __forceinline__ void epilogue_sync(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
}
template <class T>
__device__ __forceinline__ T to(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <int CG, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) k_experts(const __grid_constant__ Maps maps, const Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], sffull[kSfRing], sfempty[kSfRing];
  __shared__ uint64_t acc_full[2], acc_empty[2], done;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int s_abort;
  __shared__ int s_last[2];

  uint8_t* smem = smem_raw + ((1024u - (saddr(smem_raw) & 1023u)) & 1023u);
  constexpr int kABytes = G * kTileM * kChunkK;  // (of shared memory: 8 bits an element)
  const int b_bytes = a.bn / CG * kChunkK, stage_bytes = kABytes + G * b_bytes;
  uint8_t* sf_mem = smem + a.stages * stage_bytes;
  uint8_t* gate_mem = sf_mem + kSfRing * a.sf_block;
  int* seg_mem = reinterpret_cast<int*>(gate_mem + (GATED ? kGateBytes : 0));
  const Segments seg{seg_mem + 1,
                     seg_mem + 1 + a.experts,
                     seg_mem + 1 + 2 * a.experts,
                     seg_mem + 1 + 3 * a.experts,
                     seg_mem + 1 + 4 * a.experts,
                     seg_mem};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? blockIdx.x & 1 : 0, cta = blockIdx.x / CG, ctas = gridDim.x / CG;
  const int mtiles = (a.mtiles + CG - 1) / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      // (of a pair, the leading CTA's count for both)
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kSfRing; ++b) {
      mbar_init(&sffull[b], 1 + 128 + (CG == 2 && rank == 0 ? 1 : 0));
      mbar_init(&sfempty[b], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 4 * CG);
    }
    mbar_init(&done, 1);
    s_abort = 0;
    mbar_fence_init();
  }
  if (warp == 1) Tc<CG>::alloc(&tmem_base);
  if (warp == 2 && lane <= kBoxes)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane ? &maps.b[lane - 1] : &maps.a)) : "memory");
  // What the kernels before this one write is not read before here.
  if (!a.gathered) asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int e = threadIdx.x; e <= a.experts; e += kThreads) seg.start[e] = __ldcg(a.offsets + e);
  __syncthreads();
  if (warp == 0) read_segments(a, seg, mtiles, lane);
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  fence_after();
  const uint32_t tbase = tmem_base;
  const uint32_t stage_at = saddr(smem), sf_at = saddr(sf_mem);
  const uint32_t full_at = saddr(full), empty_at = saddr(empty), sffull_at = saddr(sffull), sfempty_at = saddr(sfempty);
  const uint32_t acc_full_at = saddr(acc_full), acc_empty_at = saddr(acc_empty), full_lead = lead<CG>(full);
  Walk walk(a, seg, cta, ctas);
  Item w;

  if (warp == 0) {
    // ------------------------------------------------------ the weights
    // (the whole warp walks and waits, and one lane issues: operands then come from the
    // uniform registers that these instructions take)
    int it = 0, s = 0, phase = 1, sb = 0, sphase = 1;
    bool ok = true, ready = true;
    while (ok && walk.next(w)) {
      const int mt = min(w.mt * CG + rank, a.mtiles - 1);  // (a pair's second tile may not exist)
      const int tile = (w.e * a.mtiles + mt) * a.kchunks;
      for (int kc = w.k0; kc < w.k1; kc += G, ++it) {
        ok = warp_wait<1>(empty_at + 8 * s, phase, &s_abort, ready);  // (the first round passes)
        if (!ok) break;
        const int s1 = s + 1 == a.stages ? 0 : s + 1;
        ready = peek<1>(empty_at + 8 * s1, s1 ? phase : phase ^ 1);
        if (elect_one()) {
          if (rank == 0) expect_tx(full_at + 8 * s, CG * G * a.a_bytes);
          load_tile<CG>(stage_at + s * stage_bytes, &maps.a, 0, (tile + kc) * kTileM, full_lead + 8 * s);
        }
        __syncwarp();
        if (++s == a.stages) s = 0, phase ^= 1;
        if (kc != w.k0 && (kc & 3)) continue;
        // the atoms of the block of four chunks
        ok = warp_wait<1>(sfempty_at + 8 * sb, sphase, &s_abort);
        if (!ok) break;
        if (elect_one()) {
          const int at = kc & ~3, n = min(4, a.kchunks - at) * kSfBytes;
          expect_tx(sffull_at + 8 * sb, n);
          bulk_in(sf_at + sb * a.sf_block, a.wscales + (tile + at) * int64_t{kSfBytes}, n, sffull_at + 8 * sb);
        }
        __syncwarp();
        if (++sb == kSfRing) sb = 0, sphase ^= 1;
      }
    }
    // What is in flight here, copies and signals, ends before the CTA does: the last stages
    // are waited for as if they were to be filled again.
    for (int u = 0; ok && u < min(it, a.stages); ++u) {
      if (--s < 0) s = a.stages - 1, phase ^= 1;
      ok = warp_wait<1>(empty_at + 8 * s, phase ^ 1, &s_abort);
    }
    if (!ok)
      for (const uint64_t t0 = global_ns(); global_ns() - t0 < 1000000;) __nanosleep(1000);
  } else if (warp == 1) {
    // --------------------------------------------------- MMA issuer
    if (rank == 0) {
      int s = 0, phase = 0, item = 0, sb = 0, sphase = 0;
      bool ok = true, ready = false, sf_ready = false;
      const uint32_t a_desc = static_cast<uint32_t>(sw128_desc(smem));  // (the high word is the same everywhere)
      const uint32_t desc_high = static_cast<uint32_t>(sw128_desc(smem) >> 32);
      auto desc = [&](uint32_t low) { return static_cast<uint64_t>(desc_high) << 32 | low; };
      while (ok && walk.next(w)) {
        const int buf = item & 1;
        ok = warp_wait<CG>(acc_empty_at + 8 * buf, ((item >> 1) & 1) ^ 1, &s_abort);
        const int n16 = (w.n + 15) & ~15;
        const uint32_t idesc = a.idesc | static_cast<uint32_t>(n16 >> 3) << 17;
        const uint32_t acc = tbase + buf * kMaxN;
        const bool wide = n16 > 128;
        fence_after();
        bool add = false;
        for (int k4 = w.k0 & ~3; ok && k4 < w.k1; k4 += 4) {
          ok = warp_wait<CG>(sffull_at + 8 * sb, sphase, &s_abort, sf_ready);
          // the rows' factors came by generic writes, and are read by the asynchronous proxy
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          const uint64_t sf = sf_desc(sf_at + sb * a.sf_block), sfr = sf_desc(sf_at + sb * a.sf_block + 4 * kSfBytes);
#pragma unroll
          for (int c = 0; c < 4; c += G) {
            const int kc = k4 + c;
            if (!ok || kc < w.k0 || kc >= w.k1) continue;
            ok = warp_wait<CG>(full_at + 8 * s, phase, &s_abort, ready);
            if (!ok) continue;
            const int s1 = s + 1 == a.stages ? 0 : s + 1, sb1 = sb + 1 == kSfRing ? 0 : sb + 1;
            const bool last = c + G == 4 || kc + G >= w.k1;  // of its block of scale factors
            ready = peek<CG>(full_at + 8 * s1, s1 ? phase : phase ^ 1);
            if (last) sf_ready = peek<CG>(sffull_at + 8 * sb1, sb1 ? sphase : sphase ^ 1);
            const uint32_t low = a_desc + s * (stage_bytes >> 4);
            if (elect_one()) {
#pragma unroll
              for (int g = 0; g < G; ++g) {
                const int blocks = (a.k - (kc + g) * kChunkK) >> 5;  // (none: a last step's second chunk)
                const uint32_t sfa = tbase + kSfCol + ((c + g) & 1) * 12, sfb = sfa + 4;
                const uint32_t al = low + g * (kTileM * kChunkK >> 4), bl = low + (kABytes >> 4) + g * (b_bytes >> 4);
                const uint64_t rows_at = sfr + (c + g) * (a.sf_rows >> 4);
                Tc<CG>::sf_copy(sfa, sf + (c + g) * (kSfBytes >> 4));
                Tc<CG>::sf_copy(sfb, rows_at);
                if (wide) Tc<CG>::sf_copy(sfb + 4, rows_at + (512 >> 4));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  if (j < blocks)
                    Tc<CG>::mma(acc, desc(al + 2 * j), desc(bl + 2 * j),
                                idesc | static_cast<uint32_t>(j) << 4 | static_cast<uint32_t>(j) << 29,
                                sfa | static_cast<uint32_t>(j) << 30, sfb | static_cast<uint32_t>(j) << 30,
                                add || g > 0 || j > 0);
                }
              }
              commit<CG>(empty_at + 8 * s);
              if (last) commit<CG>(sfempty_at + 8 * sb);
            }
            __syncwarp();
            add = true;
            if (++s == a.stages) s = 0, phase ^= 1;
          }
          if (++sb == kSfRing) sb = 0, sphase ^= 1;
        }
        if (elect_one()) commit<CG>(acc_full_at + 8 * buf);
        __syncwarp();
        ++item;
      }
      // every MMA issued must be finished before tensor memory is freed
      if (elect_one()) commit_own<CG>(&done);
      __syncwarp();
      mbar_wait(&done, 0);
    } else {
      // The other CTA of a pair: its scale factors are there, says this warp to the leading
      // one's barriers.
      int sb = 0, sphase = 0;
      bool ok = true;
      while (ok && walk.next(w)) {
        for (int k4 = w.k0 & ~3; k4 < w.k1; k4 += 4) {
          ok = warp_wait<1>(sffull_at + 8 * sb, sphase, &s_abort);
          if (!ok) break;
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (lane == 0) arrive_lead<CG>(&sffull[sb]);
          __syncwarp();
          if (++sb == kSfRing) sb = 0, sphase ^= 1;
        }
      }
    }
  } else if (warp == 2) {
    // --------------------------------------------------- rows in order
    {
      if (a.gathered) asm volatile("griddepcontrol.wait;" ::: "memory");
      int s = 0, phase = 1;
      bool ok = true, ready = true;
      while (ok && walk.next(w)) {
        const int half = ((w.n + 15) & ~15) / CG;  // of this CTA
        const int box = half <= 32 ? 0 : half <= 64 ? 1 : half <= 128 ? 2 : half <= 192 ? 3 : 4;
        const int rows = min(box == 4 ? 256 : box == 3 ? 192 : 32 << box, a.bn / CG);
        const CUtensorMap* tm = &maps.b[box];
        const int row = w.row0 + rank * half;
        for (int kc = w.k0; kc < w.k1; kc += G) {
          ok = warp_wait<1>(empty_at + 8 * s, phase, &s_abort, ready);
          if (!ok) break;
          const int s1 = s + 1 == a.stages ? 0 : s + 1;
          ready = peek<1>(empty_at + 8 * s1, s1 ? phase : phase ^ 1);
          if (elect_one()) {
            if (rank == 0) expect_tx(full_at + 8 * s, CG * G * rows * kChunkK);
#pragma unroll
            for (int g = 0; g < G; ++g)
              load_tile<CG>(stage_at + s * stage_bytes + kABytes + g * b_bytes, tm, (kc + g) * kChunkK, row,
                            full_lead + 8 * s);
          }
          __syncwarp();
          if (++s == a.stages) s = 0, phase ^= 1;
        }
      }
    }
  } else if (warp >= 8 && warp < 12) {
    // ------------------------------------------- the rows' scale factors
    // (copies that arrive at the barrier by themselves: nothing here waits for memory)
    if (a.gathered) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lt = threadIdx.x - 256, nsf = a.k >> 5;
    int sb = 0, sphase = 1;
    bool ok = true;
    while (ok && walk.next(w)) {
      for (int k4 = w.k0 & ~3; k4 < w.k1; k4 += 4) {
        ok = warp_wait<1>(sfempty_at + 8 * sb, sphase, &s_abort);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = lt + 128 * i, row = w.row0 + c;
          if (128 * i >= w.n) continue;
          const uint32_t to = sf_at + sb * a.sf_block + 4 * kSfBytes + 512 * i + sf_off(lt, 0);
          const bool in = c < w.n && row < a.tokens;
          const uint8_t* p = a.xscales + (in ? row : 0) * a.xscale_stride + 4 * k4;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (a.xscale_words) {
              const bool on = in && 4 * (k4 + j) < nsf;
              cp_async4(to + j * a.sf_rows, on ? p + 4 * j : a.xscales, on);
            } else {
              uint32_t word = 0;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (in && 4 * (k4 + j) + e < nsf) word |= static_cast<uint32_t>(__ldg(p + 4 * j + e)) << (8 * e);
              asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + j * a.sf_rows), "r"(word) : "memory");
            }
          }
        }
        if (a.xscale_words) cp_async_arrive(&sffull[sb]);
        else mbar_arrive(&sffull[sb]);
        if (++sb == kSfRing) sb = 0, sphase ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= 4) {
    // ------------------------------------------------------ epilogue
    // Two groups of four warps take turns: each has an accumulator.
    const int q = warp & 3, group = warp >> 3;  // the warp's lanes of tensor memory, and its group
    const uint32_t acc = tbase + (static_cast<uint32_t>(32 * q) << 16) + group * kMaxN;
    float* gate = reinterpret_cast<float*>(gate_mem) + group * (kGateTokens * kGatePitch);
    for (int item = 0; walk.next(w); ++item) {
      if ((item & 1) != group) continue;
      bool ok = mbar_wait(&acc_full[group], (item >> 1) & 1, &s_abort);
      // (warps that gave up and warps that did not must not part at the barriers below)
      if (!epilogue_all(ok && !s_abort, group)) break;
      fence_after();
      const int mt = w.mt * CG + rank;
      bool write = mt < a.mtiles;
      const float* parts = nullptr;
      if (CG == 1 && w.parts > 1) {
        // partial sums: column by column, 128 rows each; the last CTA to arrive adds
        // them in the CTAs' order
        float* mine = a.partials + (2 * cta + (w.k0 == 0)) * int64_t{kSplitN * kTileM} + 32 * q + lane;
        for (int c0 = 0; c0 < w.n; c0 += 16) {
          uint32_t v[16];
          tmem_ld16(acc + c0, v);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(v[i]));
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (c0 + i < w.n) __stcg(mine + (c0 + i) * kTileM, __uint_as_float(v[i]));
        }
        __threadfence();
        epilogue_sync(group);
        if (q == 0 && lane == 0) {
          const int last = atomicAdd(a.counters + w.first, 1u) == static_cast<uint32_t>(w.parts - 1);
          if (last) a.counters[w.first] = 0;
          __threadfence();
          s_last[group] = last;
        }
        epilogue_sync(group);
        write = s_last[group];
        parts = a.partials + 32 * q + lane;
      }
      // NC accumulators of this thread's row from column c0 on, or the sums of their parts,
      // a part's reads all at once.
      auto columns = [&](auto& v, int c0) {
        constexpr int NC = sizeof(v) / 4;
        if (CG == 1 && parts) {
          const float* at = parts + c0 * kTileM + (2 * w.first + 1) * int64_t{kSplitN * kTileM};
          for (int p = 0; p < w.parts; ++p) {  // (the first CTA's second place, the others' first)
            float x[NC];
#pragma unroll
            for (int i = 0; i < NC; ++i) x[i] = c0 + i < w.n ? __ldcg(at + i * kTileM) : 0.0f;
#pragma unroll
            for (int i = 0; i < NC; ++i)
              v[i] = p ? __float_as_uint(fadd(__uint_as_float(v[i]), x[i])) : __float_as_uint(x[i]);
            at += (p ? 2 : 1) * int64_t{kSplitN * kTileM};
          }
        } else {
          if constexpr (NC == 16) tmem_ld16(acc + c0, v);
          else tmem_ld32(acc + c0, v);  // (past the tile's columns: whatever is there, not stored)
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < NC; ++i) asm volatile("" : "+r"(v[i]));
        }
      };
      if (!write) {
      } else if constexpr (!GATED) {
        const int m = mt * kTileM + 32 * q + lane;
        const bool on = m < a.features;
        auto rows_out = [&](auto type) {
          using T = decltype(type);
          uint8_t* out = a.out + w.row0 * a.out_stride + static_cast<int64_t>(m) * sizeof(T);
          for (int c0 = 0; c0 < w.n; c0 += 16) {
            uint32_t v[16];
            columns(v, c0);
            const int n = on ? w.n - c0 : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (i < n) *reinterpret_cast<T*>(out) = to<T>(__uint_as_float(v[i]));
              out += a.out_stride;
            }
          }
        };
        if (a.out_type == LP_F32) rows_out(float{});
        else if (a.out_type == LP_F16) rows_out(__half{});
        else rows_out(__nv_bfloat16{});
      } else {
        for (int c0 = 0; c0 < w.n; c0 += kGateTokens) {
          uint32_t v[32];
          columns(v, c0);
          const bool up = lane & 16;  // this lane holds an up row; its partner the gate's
          const int f = 16 * q + (lane & 15);
          float* to = gate + (up ? 16 * kGatePitch : 0) + f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[16 + i], 16);
            const float g = __uint_as_float(up ? other : v[i]), u = __uint_as_float(up ? v[16 + i] : other);
            to[i * kGatePitch] = silu_mul(g, u);
          }
          epilogue_sync(group);
          // 16 features of a token each; two lanes hold a block of 32
          const int t = 8 * q + (lane >> 2), f0 = 16 * (lane & 3), feature = mt * 64 + f0;
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
          epilogue_sync(group);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) arrive_lead<CG>(&acc_empty[group]);
    }
  }
  fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // nobody's shared memory goes while the pair still reads or signals there
  if (warp == 1) {
    __syncwarp();
    fence_after();
    Tc<CG>::dealloc(tbase);
  }
}

bool encode_tiles(CUtensorMap* tm, const void* base, int64_t tiles, bool fp4) {
  EncodeFn fn = encoder();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(kChunkK), static_cast<cuuint64_t>(tiles * kTileM)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(fp4 ? kChunkK / 2 : kChunkK)};
  const cuuint32_t box[2] = {kChunkK, G * kTileM}, one[2] = {1, 1};
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

template <int CG, bool GATED>
int launch(const Maps& maps, const Args& a, int smem, cudaStream_t st) {
  const DeviceInfo& di = device_info();
  auto kern = k_experts<CG, GATED>;
  static int ctas[kMaxDevices];  // of a full grid, 0 before the first launch
  const int slot = di.ordinal % kMaxDevices;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t c{};
  c.blockDim = dim3(kThreads);
  c.dynamicSmemBytes = smem;
  c.stream = st;
  c.attrs = attr;
  c.numAttrs = CG;
  if (!ctas[slot]) {
    const int most = di.max_smem_optin - 1024;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return cuda_status(e);
    int n = di.sm_count;
    if (CG == 2) {  // as many pairs as fit at a time
      c.gridDim = dim3(di.sm_count / 2 * 2);
      c.dynamicSmemBytes = most;
      e = cudaOccupancyMaxActiveClusters(&n, kern, &c);
      if (e != cudaSuccess) return cuda_status(e);
      if (n < 1) return LP_ERR_UNSUPPORTED;
      n *= 2;
      c.dynamicSmemBytes = smem;
    }
    ctas[slot] = n;
  }
  c.gridDim = dim3(ctas[slot]);
  return cuda_status(cudaLaunchKernelEx(&c, kern, maps, a));
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

int launch_experts(const lp_expert_weights& w, const lp_rows8& given, const int32_t* offsets, const int32_t* row_token,
                   int64_t rows, const lp_matrix* out, const lp_rows8* out8, void* workspace, cudaStream_t st) {
  uint8_t* space = static_cast<uint8_t*>(workspace);
  lp_rows8 x = given;
  if (row_token) {
    x = gathered_rows(rows, given.cols, space + fixed_workspace());
    const GatherArgs g{static_cast<const uint8_t*>(given.codes), static_cast<const uint8_t*>(given.scales),
                       static_cast<uint8_t*>(x.codes), static_cast<uint8_t*>(x.scales), given.code_stride,
                       given.scale_stride, x.scale_stride, offsets + w.experts, row_token, rows, given.rows,
                       static_cast<int>(given.cols)};
    const int grid = static_cast<int>(std::min<int64_t>((rows + 7) / 8, device_info().sm_count * 16ll));
    if (const int e = launch_early(k_gather, grid, 256, st, g)) return e;
  }
  const Layout l = layout(w.experts, w.rows, w.cols, w.dtype, w.gated);
  Args a{};
  a.wscales = static_cast<const uint8_t*>(w.scales);
  a.xscales = static_cast<const uint8_t*>(x.scales);
  a.xscale_stride = x.scale_stride;
  // (a word holds four scales of one row where a row has a multiple of four, or zeros behind them)
  a.xscale_words = (row_token || x.cols % kChunkK == 0) &&
                   ((reinterpret_cast<uintptr_t>(x.scales) | static_cast<uintptr_t>(x.scale_stride)) & 3) == 0;
  a.offsets = offsets;
  a.gathered = row_token != nullptr;
  a.experts = static_cast<int>(w.experts);
  a.mtiles = static_cast<int>(l.mtiles);
  a.kchunks = static_cast<int>(l.kchunks);
  a.k = static_cast<int>(w.cols);
  a.rows = static_cast<int>(rows);
  a.tokens = static_cast<int>(x.rows);
  a.a_bytes = static_cast<uint32_t>(l.tile_bytes);
  // A e2m1 (5) or e4m3 (0), B e4m3, both K-major, E8M0 scales
  a.idesc = (w.dtype == LP_E2M1 ? 5u << 7 : 0u) | 1u << 23;
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
  a.counters = reinterpret_cast<uint32_t*>(space);
  a.partials = reinterpret_cast<float*>(space + kCounterBytes);
  // A token has at most one row per expert, so no segment is longer than x.
  const int64_t most = row_token ? std::min(rows, given.rows) : rows;
  const int64_t mean = (rows + w.experts - 1) / w.experts;
  // Few rows per expert: tiles of at most 128 rows, one CTA each; many: of 240, two CTAs
  // each.  One CTA / two, us: 32 experts of 2880 x 1440 in e2m1 with 25 rows each 25 / 36,
  // 75 rows 34 / 39, 150 rows 48 / 51; one of 4096 x 4096 with 400 rows 15 / 20; 64 gated of
  // 2816 x 2048 with 1024 rows each 450 / 390, 8 of 4096 x 14336 in e4m3 550 / 470.  (Tiles
  // of at most 64 rows cost the same time as ones of 128 and are more.)
  const int cg = mean > kPairRows ? 2 : 1, bn = cg == 2 ? kMaxN : 128;
  a.bn = static_cast<int>(std::min<int64_t>(bn, (most + 15) / 16 * 16));
  a.split = cg == 1 && a.bn <= kSplitN ? kSplitTiles : 0;  // (pairs do not join parts)
  a.sf_rows = a.bn > 128 ? 1024 : 512;
  a.sf_block = 4 * (kSfBytes + a.sf_rows);
  const int fixed = 1024 + kSfRing * a.sf_block + (w.gated ? kGateBytes : 0)+
                    static_cast<int>(5 * w.experts + 2) * 4;
  const int stage = G * (kTileM + a.bn / cg) * kChunkK;
  a.stages = std::min(kMaxStages, (device_info().max_smem_optin - 1024 - fixed) / stage);
  if (a.stages < 2) return LP_ERR_UNSUPPORTED;
  Maps maps;
  if (!encode_tiles(&maps.a, w.tiles, l.tiles, w.dtype == LP_E2M1)) return LP_ERR_UNSUPPORTED;
  const int boxes[kBoxes] = {32, 64, 128, 192, 256};
  for (int b = 0; b < kBoxes; ++b)
    if (!encode_rows(&maps.b[b], x.codes, x.cols, x.rows, x.code_stride, std::min(boxes[b], a.bn / cg)))
      return LP_ERR_UNSUPPORTED;
  const int smem = fixed + a.stages * stage;
  // M = 128 of a CTA, or 256 of a pair
  a.idesc |= static_cast<uint32_t>(cg * 128 >> 4) << 24;
  if (w.gated) return cg == 2 ? launch<2, true>(maps, a, smem, st) : launch<1, true>(maps, a, smem, st);
  return cg == 2 ? launch<2, false>(maps, a, smem, st) : launch<1, false>(maps, a, smem, st);
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
