// attn_rows.cu -- attention of a few query rows over a paged cache: single
// new tokens (decode), and chunks too short for a tile of the chunk kernel.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  j visible
//
// One pass over the keys with a running maximum and sum per row.  What bounds
// it is the cache's bytes, so the design serves the loads:
//   * A CTA takes up to 8 query rows of one key head, so keys and values are read
//     once for a group of up to 8 query heads (twice for 9 to 16, ...).  Two CTAs of
//     four warps share an SM: one joins its rows while the other streams.
//   * Each warp streams for itself: steps of 16 to 32 keys (keys and values,
//     8 KB) go by cp.async into its own ring of 24 KB, two to five steps ahead
//     of their use, across item boundaries.  No barrier stands between a load
//     and its use, and a step's pages may lie anywhere.
//   * The products are m16n8k16 with 16 rows where there are 8 queries; the
//     other 8 rows carry what 16 bits drop: row i the query's high part, row
//     i + 8 the rest (hi + lo is 22 bits of fp16, 16 of bf16), and likewise
//     for the weights p.  Both parts of a row meet in the same thread.  fp32
//     results with bf16 operands take a second product for a third part (24
//     bits).  fp16 parts are scaled: queries by a power of two per row,
//     queries and weights to at most 2^14, second parts by 2^12 more (which
//     the row's other accumulator takes back).  So they neither overflow nor
//     fall under the type's smallest numbers: weights of 2^-29 of the row's
//     largest keep 22 bits.
//   * An int8 cache's scales are per (token, head): a key's multiplies its
//     score, a value's its weight, so the codes go into the products exactly.
//   * A step's products start from zero and are added to the outputs in fp32
//     registers, rounded: left in the product's own sum they are cut off at
//     each one, which takes 1.0e-4 to 1.6e-4 off 131000 keys of one sign
//     (errors now 3e-7, 1e-7 at 16000 keys and below).
//   * The tensor cores serve here to keep the arithmetic (8 rows: 16 fma per
//     cached byte) off the fp32 pipe; at 8 rows a tile of 128 x N tcgen05
//     rows would be 94 % padding, and the bytes bound the time either way.
// Measured: two requests of 131000 keys, 64 heads on 8 key heads of 128, bf16,
// 200 us (5.4 TB/s, 82 % of a copy's rate; what is missing is the spread of the
// SMs' shares of the bandwidth, 157 us on average); 32 requests under a window
// of 4000, heads of 64, 55 us (4.2 TB/s; 16 us of start and join); 53 requests of
// up to 16000 keys over an int8 cache with fp32 queries, 232 us (3.5 TB/s), with
// bf16 ones 217: latency at two warps per scheduler, each of which issues every
// 4 cycles (49 % of the issue slots, 29 % of the tensor pipe, 57 % of DRAM).
#include <type_traits>

#include "attn.cuh"

namespace lp {
namespace {

using namespace attn;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;
constexpr int kUnit = 32;  // keys per unit: a warp's share of a round
// A CTA takes at least this many units: fewer would cost more in the join of
// the partial results than the spread over more SMs gives back.
constexpr int kMinUnits = 4;  // (one request of 1000 keys: 14.9 us with 1 or 4, 17.2 with 12)
// What an item costs beside its keys, in units (about 4 us against 0.25): 32
// requests under a window 75 us with 8, 56 with 16, 56 with 32.
constexpr int kItemUnits = 16;
constexpr int kTop = 14;       // queries and weights are below 2^kTop in 16 bits
// fp16: second parts, at most 2^(kTop - 11), are held times 2^kLow
constexpr int kLow = 12;
constexpr int kBad = 32;  // steps with cleared values that a warp notes one by one

// The types of the two products: queries x keys, weights x values.  An int8
// code is exact in both 16-bit types.  With the keys fp16 carries the queries
// in two parts; with the values bf16 carries weight x scale, whose range over
// a row's keys fp16 does not span.
template <class C>
struct ValueType { using T = C; };
template <>
struct ValueType<CI8> { using T = CBF16; };

template <class C, int D>
struct Shape {
  static constexpr int ES = C::kInt8 ? 1 : 2;
  static constexpr int KS = C::kInt8 || D == 64 ? 32 : 16;  // keys per step
  static constexpr int NG = KS / 8;                          // n8 groups of keys
  static constexpr int STEPS = D / 16;                       // k16 steps of a score
  static constexpr int TILES = D / 8;                        // n8 tiles of an output
  static constexpr int CHUNKS = D * ES / 16;                 // 16-byte pieces of a row
  // bytes of a row in the ring, and lanes that fetch one
  static constexpr int RS = CHUNKS <= 4 ? 64 : CHUNKS <= 8 ? 128 : 256;
  static constexpr int LPR = RS / 16;
  static constexpr int HALF = KS * RS;                       // keys, then values
  static constexpr int SCALES = C::kInt8 ? KS * 8 : 0;       // key scales, value scales
  static constexpr int STAGE = 2 * HALF + SCALES + 16;       // and presence, first key
  static constexpr int STAGES = 24576 / (2 * HALF);
  static constexpr int RING = STAGES * STAGE;
  static constexpr int SMEM = kWarps * RING + kWarps * kWarps * D * 4;
};

// Elements of an int8 key that a lane reads at once.
__device__ constexpr int key_read(int dim) { return dim % 64 == 0 ? 16 : 8; }

// Where piece `c` of row `r` is.  16-bit rows: so that the eight rows of a
// matrix read meet in no bank.  int8 rows of 128 bytes: so that neither reads
// of two rows of four pieces (keys) nor of four rows of two (values) do.
template <class C, int D>
__device__ __forceinline__ int place(int r, int c) {
  using S = Shape<C, D>;
  const int x = !C::kInt8     ? r & 7
                : S::RS == 64 ? r >> 1 & 3
                              : ((r >> 1 & 3) * 2) ^ ((r & 1) * 4);
  return r * S::RS + ((c ^ x) << 4);
}

template <class C>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (C::kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a * b.
template <class C>
__device__ __forceinline__ void mma_new(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (C::kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// o += weights x values of N times 16 keys, third parts (T3) first.  (32 keys at
// once: one addition to o for two.  An int8 step of 32 keys x 128 takes 5 % more
// time than with sums in the product, others nothing that shows.)
template <class V, bool T3, int N, int M>
__device__ __forceinline__ void add_products(float* o, const uint32_t (&pa)[N][4],
                                             const uint32_t (&pc)[M][4], const uint32_t (&b)[N][2]) {
  float d[4];
  if constexpr (T3) {
    mma_new<V>(d, pc[0], b[0][0], b[0][1]);
#pragma unroll
    for (int i = 1; i < N; ++i) mma<V>(d, pc[i], b[i][0], b[i][1]);
    mma<V>(d, pa[0], b[0][0], b[0][1]);
  } else {
    mma_new<V>(d, pa[0], b[0][0], b[0][1]);
  }
#pragma unroll
  for (int i = 1; i < N; ++i) mma<V>(d, pa[i], b[i][0], b[i][1]);
#pragma unroll
  for (int i = 0; i < 4; i += 2) upk(add2(pk(o[i], o[i + 1]), pk(d[i], d[i + 1])), o[i], o[i + 1]);
}
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0)
               : "memory");
}

template <int N>
__device__ __forceinline__ void lds_words(uint32_t* r, const uint8_t* p) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r[0] = v.x, r[1] = v.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// Head dimension of column n of output tile i.  16-bit values are read as
// matrices, in order.  A lane reads int8 values as pieces of 8 codes (the last
// of D = 96: 4), and takes tile i's from its code i.
template <class C, int D>
__device__ __forceinline__ int value_dim(int n, int i) {
  if constexpr (!C::kInt8) return i * 8 + n;
  else return i < 8 ? n * 8 + i : 64 + n * (D / 8 - 8) + (i - 8);
}
// Head dimension of the first of a lane's four elements in k16 step k: of the
// queries, and of the keys that meet them (16-bit keys: the second pair is 8 on).
template <class C, int D>
__device__ __forceinline__ int key_dim(int k, int c4, int i) {
  if constexpr (!C::kInt8) return k * 16 + 2 * c4 + (i & 1) + (i >> 1) * 8;
  else {
    constexpr int E = key_read(D);
    return (k / (E / 4)) * 4 * E + c4 * E + (k % (E / 4)) * 4 + i;
  }
}

using Part = Walk<kUnit, kRows, kItemUnits>;

template <class C, int D, bool T3>
__global__ void __launch_bounds__(kThreads, 2) k_attn_rows(const __grid_constant__ Args a) {
  using S = Shape<C, D>;
  using V = typename ValueType<C>::T;
  constexpr bool kQ3 = T3 && C::kBf16;
  constexpr float kUp = C::kBf16 ? 1.0f : static_cast<float>(1 << kLow);
  constexpr float kDown = 1.0f / kUp;
  constexpr float kUpV = V::kBf16 ? 1.0f : static_cast<float>(1 << kLow);
  constexpr float kDownV = 1.0f / kUpV;
  __shared__ Cursor cur;
  __shared__ int64_t sums[kWarps];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ int s_last;
  extern __shared__ __align__(128) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem + kWarps * S::RING);  // [warp][row of a pass][D]

  find_share<kUnit, kRows, kItemUnits, kThreads>(a, kMinUnits, &cur, sums);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g8 = lane >> 2, c4 = lane & 3;
  uint8_t* ring = smem + warp * S::RING;
  const uint32_t ring_s = saddr(ring);
  constexpr int SPU = kUnit / S::KS;  // steps per unit

  // ---- the loads: this warp's steps of all the CTA's items, in order.  Unit
  // warp, warp + kWarps, ... of each part, SPU steps each.
  Part ld;
  ld.start(cur);
  bool more = ld.open(a);
  int ld_u = warp, ld_s = 0;  // unit of the part, step of the unit
  int entry = -1;             // the table's, for key0 + lane of the next step
  const bool halves = a.page_size % 16 == 0;  // a page holds each 16 keys of a step
  auto settle = [&] {  // to the next step that exists
    while (more && ld_u >= ld.n) {
      ld.close(a);
      more = ld.open(a);
      ld_u = warp;
    }
  };
  auto look = [&] {  // its pages, one step before they are needed
    entry = -1;
    if (!more) return;
    const int j = ld.key(ld_u) + ld_s * S::KS + lane;
    if ((S::KS == 32 || lane < S::KS) && j <= ld.un.hi && (j >= ld.un.lo || j < a.sinks))
      entry = entry_of(a, ld.b, j);
  };
  // Strides in pieces of 16 bytes (scales: elements) fit 32 bits, so a row's
  // address is two 32 x 32 -> 64 bit products.
  const int r0 = lane / S::LPR, c = lane % S::LPR;  // row and piece of this lane's loads
  constexpr int RPI = 32 / S::LPR, N = S::KS / RPI;  // rows per load, loads
  const bool in = S::LPR == S::CHUNKS || c < S::CHUNKS;
  const uint32_t kp16 = static_cast<uint32_t>(a.k.page * S::ES >> 4);
  const uint32_t kt16 = static_cast<uint32_t>(a.k.token * S::ES >> 4);
  const uint32_t vp16 = static_cast<uint32_t>(a.v.page * S::ES >> 4);
  const uint32_t vt16 = static_cast<uint32_t>(a.v.token * S::ES >> 4);
  auto wide = [](uint32_t x, uint32_t y) { return static_cast<uint64_t>(x) * y; };
  auto issue = [&](int stage) {
    if (more) {
      const int key0 = ld.key(ld_u) + ld_s * S::KS, head = ld.head;
      const int pg = valid_page(a, entry);
      const uint32_t there = __ballot_sync(0xffffffffu, pg >= 0);
      const uint32_t dst = ring_s + stage * S::STAGE;
      if (lane == 0)
        *reinterpret_cast<uint2*>(ring + stage * S::STAGE + 2 * S::HALF + S::SCALES) =
            make_uint2(there, static_cast<uint32_t>(key0));
      const uint8_t* kh = a.k.data + head * a.k.head * S::ES + c * 16;
      const uint8_t* vh = a.v.data + head * a.v.head * S::ES + c * 16;
      if (halves) {
        // addresses advance by constants within a page
        const uint64_t dk = static_cast<uint64_t>(kt16) * (RPI * 16);
        const uint64_t dv = static_cast<uint64_t>(vt16) * (RPI * 16);
#pragma unroll
        for (int h = 0; h < S::KS / 16; ++h) {
          const uint32_t bits = there >> (16 * h) & 0xffffu;
          const uint32_t p0 = __shfl_sync(0xffffffffu, pg, 16 * h + max(__ffs(bits) - 1, 0));
          const uint32_t off = page_offset(a, key0 + 16 * h) + r0;
          const uint32_t d0 = dst + 16 * h * S::RS;  // (place() repeats every eight rows)
          if (bits == 0xffffu) {
            const uint8_t* pk = kh + ((wide(p0, kp16) + wide(off, kt16)) << 4);
            const uint8_t* pv = vh + ((wide(p0, vp16) + wide(off, vt16)) << 4);
            if (in) {
#pragma unroll
              for (int i = 0; i < N * 16 / S::KS; ++i) {
                const uint32_t to = place<C, D>(r0 + i * RPI, c);
                cp16(d0 + to, pk + i * dk);
                cp16(d0 + S::HALF + to, pv + i * dv);
              }
            }
          } else {
            const uint32_t pp = bits ? p0 : 0;
            const uint8_t* pk = kh + ((wide(pp, kp16) + wide(off, kt16)) << 4);
            const uint8_t* pv = vh + ((wide(pp, vp16) + wide(off, vt16)) << 4);
#pragma unroll
            for (int i = 0; i < N * 16 / S::KS; ++i) {
              const int r = r0 + i * RPI;
              const bool on = bits >> r & 1u;
              const uint32_t to = place<C, D>(r, c);
              if (in) {
                cp16(d0 + to, on ? pk + i * dk : a.k.data, on);
                cp16(d0 + S::HALF + to, on ? pv + i * dv : a.v.data, on);
              }
            }
          }
        }
      } else {
        const int my_off = pg >= 0 ? page_offset(a, key0 + lane) : 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int r = r0 + i * RPI;
          const int pr = __shfl_sync(0xffffffffu, pg, r);
          const uint32_t off = __shfl_sync(0xffffffffu, my_off, r);
          const bool on = pr >= 0;
          const uint32_t p = on ? pr : 0;
          if (in) {
            cp16(dst + place<C, D>(r, c), kh + ((wide(p, kp16) + wide(off, kt16)) << 4), on);
            cp16(dst + S::HALF + place<C, D>(r, c), vh + ((wide(p, vp16) + wide(off, vt16)) << 4), on);
          }
        }
      }
      if constexpr (C::kInt8) {
        const bool on = pg >= 0;
        const uint32_t p = on ? pg : 0;
        const uint32_t off = on ? page_offset(a, key0 + lane) : 0;
        cp4(dst + 2 * S::HALF + lane * 4,
            a.k.scales + head * a.k.shead + wide(p, static_cast<uint32_t>(a.k.spage)) +
                wide(off, static_cast<uint32_t>(a.k.stoken)), on);
        cp4(dst + 2 * S::HALF + S::KS * 4 + lane * 4,
            a.v.scales + head * a.v.shead + wide(p, static_cast<uint32_t>(a.v.spage)) +
                wide(off, static_cast<uint32_t>(a.v.stoken)), on);
      }
      if (++ld_s == SPU) {
        ld_s = 0;
        ld_u += kWarps;
        settle();
      }
      look();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  settle();
  look();
#pragma unroll 1
  for (int i = 0; i < S::STAGES - 1; ++i) issue(i);
  int stage = 0;

  Part w;
  w.start(cur);
  while (w.open(a)) {
    const int rows = w.rows;
    // ---- this lane's row: query parts, position, window
    const int r = w.block * kRows + g8;
    const bool row_ok = g8 < rows;
    const int pos = row_ok ? w.rq.base + r / a.group : -1;
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    // keys up to p_first that are at or past lo_last are seen by all of the block's rows
    const int p_first = w.rq.base + w.block * kRows / a.group;
    const int lo_last =
        a.window > 0 ? w.rq.base + (w.block * kRows + rows - 1) / a.group - a.window + 1 : 0;

    uint32_t qa[S::STEPS][4];           // hi, lo, hi, lo of 4 elements
    uint32_t qc[kQ3 ? S::STEPS : 1][2];  // third parts
    float cscale;
    {
      const int64_t q0 = row_ok ? (w.rq.start + r / a.group) * a.q_token +
                                      (w.head * a.group + r % a.group) * a.q_head
                                : 0;
      float x[S::STEPS][4];
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < S::STEPS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[k][i] = row_ok ? load_elem(a.q, a.q_type, q0 + key_dim<C, D>(k, c4, i)) : 0.0f;
#pragma unroll
      for (int k = 0; k < S::STEPS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[k][i]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = row_exponent(amax);
      const float f = pow2(kTop - e);
      cscale = a.scale_log2 * pow2(e - kTop);
#pragma unroll
      for (int k = 0; k < S::STEPS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float y0 = x[k][2 * h] * f, y1 = x[k][2 * h + 1] * f;
          const uint32_t hi = pack16<C>(y0, y1);
          const float r0 = (y0 - low16<C>(hi)) * kUp, r1 = (y1 - high16<C>(hi)) * kUp;
          const uint32_t lo = pack16<C>(r0, r1);
          qa[k][2 * h] = hi;
          qa[k][2 * h + 1] = lo;
          if constexpr (kQ3) qc[k][h] = pack16<C>(r0 - low16<C>(lo), r1 - high16<C>(lo));
        }
    }

    float o[S::TILES][4];
#pragma unroll
    for (int i = 0; i < S::TILES; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int nbad = 0, badkey = 0;  // steps with values that were cleared; the lane-th one's first key

    const int steps = warp < w.n ? (w.n - warp + kWarps - 1) / kWarps * SPU : 0;
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 2) : "memory");
      __syncwarp();  // this step has landed for all lanes, and all are done with the one before
      issue(stage == 0 ? S::STAGES - 1 : stage - 1);
      uint8_t* st = ring + stage * S::STAGE;
      const uint32_t st_s = ring_s + stage * S::STAGE;
      if (++stage == S::STAGES) stage = 0;
      const uint2 info = *reinterpret_cast<const uint2*>(st + 2 * S::HALF + S::SCALES);
      const uint32_t there = info.x;
      const int key0 = static_cast<int>(info.y);
      const bool all = there == (S::KS == 32 ? 0xffffffffu : 0xffffu) &&
                       key0 + S::KS - 1 <= p_first && (key0 >= lo_last || key0 + S::KS <= a.sinks);
      if (!all) {  // see clear_bad
        bool bad = false;
        if constexpr (C::kInt8) {
          bad = clear_bad_scale(reinterpret_cast<float*>(st + 2 * S::HALF) + S::KS + lane);
        } else {
#pragma unroll 4
          for (int i = 0; i < N; ++i)
            if (in) bad |= clear_bad<V>(st + S::HALF + place<C, D>(r0 + i * RPI, c));
        }
        if (__any_sync(0xffffffffu, bad)) {
          if (nbad < kBad) badkey = lane == nbad ? key0 : badkey;
          ++nbad;
        }
        __syncwarp();
      }

      // ---- scores
      float sc[S::NG][4];
#pragma unroll
      for (int n = 0; n < S::NG; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
      if constexpr (!C::kInt8) {
#pragma unroll
        for (int k = 0; k < S::STEPS; k += 2)
#pragma unroll
          for (int n = 0; n < S::NG; ++n) {
            uint32_t kb[4];  // eight keys x 32 dimensions
            ldmatrix4(kb, st_s + place<C, D>(n * 8 + (lane & 7), k * 2 + (lane >> 3)));
            mma<C>(sc[n], qa[k], kb[0], kb[1]);
            mma<C>(sc[n], qa[k + 1], kb[2], kb[3]);
            if constexpr (kQ3) {
              const uint32_t q3[4] = {qc[k][0], 0u, qc[k][1], 0u};
              const uint32_t q4[4] = {qc[k + 1][0], 0u, qc[k + 1][1], 0u};
              mma<C>(sc[n], q3, kb[0], kb[1]);
              mma<C>(sc[n], q4, kb[2], kb[3]);
            }
          }
      } else {
        constexpr int E = key_read(D), LW = E / 4;
#pragma unroll
        for (int x = 0; x < D / (4 * E); ++x)
#pragma unroll
          for (int n = 0; n < S::NG; ++n) {
            uint32_t kw[LW];
            const int byte = x * 4 * E + c4 * E;
            lds_words<LW>(kw, st + place<C, D>(n * 8 + g8, byte >> 4) + (byte & 15));
#pragma unroll
            for (int y = 0; y < LW; ++y) {
              const uint32_t u = kw[y] ^ 0x80808080u;
              mma<C>(sc[n], qa[x * LW + y], codes_f16(u, 0x4140u), codes_f16(u, 0x4342u));
            }
          }
      }
      // ---- weights: log2-domain scores, masks, running maximum
      const float* sks = reinterpret_cast<const float*>(st + 2 * S::HALF);
      float t[S::NG][2];
      float mx = -INFINITY, lnew = 0.0f;
#pragma unroll
      for (int n = 0; n < S::NG; ++n) {
        float2 ks = make_float2(1.0f, 1.0f);
        if constexpr (C::kInt8) ks = *reinterpret_cast<const float2*>(sks + n * 8 + 2 * c4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = fmaf(sc[n][i + 2], kDown, sc[n][i]) * cscale;
          if constexpr (C::kInt8) v *= i ? ks.y : ks.x;
          t[n][i] = v;
        }
      }
      if (!all) {
#pragma unroll
        for (int n = 0; n < S::NG; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int x = n * 8 + 2 * c4 + i, j = key0 + x;
            if (!(there >> x & 1u) || j > pos || (j < row_lo && j >= a.sinks)) t[n][i] = -INFINITY;
          }
      }
#pragma unroll
      for (int n = 0; n < S::NG; ++n) mx = fmaxf(mx, fmaxf(t[n][0], t[n][1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m, mx);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      float p[S::NG][2];  // weights times 2^kTop
#pragma unroll
      for (int n = 0; n < S::NG; ++n) {
        float2 vs = make_float2(1.0f, 1.0f);
        if constexpr (C::kInt8) vs = *reinterpret_cast<const float2*>(sks + S::KS + n * 8 + 2 * c4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[n][i] = ex2(t[n][i] - ref) * static_cast<float>(1 << kTop);
          lnew += p[n][i];
          if constexpr (C::kInt8) p[n][i] *= i ? vs.y : vs.x;
        }
      }
      if (__any_sync(0xffffffffu, mn != m)) {
        const float corr = ex2(m - ref);
        l *= corr;
#pragma unroll
        for (int i = 0; i < S::TILES; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] *= corr;
        m = mn;
      }
      l += lnew;
      // ---- outputs: p in two or three parts times the values, 16 or 32 keys at once
      constexpr int KK = S::KS / 16;
      uint32_t pa[KK][4], pc[T3 ? KK : 1][4];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = p[2 * kk + h][0], p1 = p[2 * kk + h][1];
          const uint32_t hi = pack16<V>(p0, p1);
          const float r0 = (p0 - low16<V>(hi)) * kUpV, r1 = (p1 - high16<V>(hi)) * kUpV;
          pa[kk][2 * h] = hi;
          pa[kk][2 * h + 1] = pack16<V>(r0, r1);
          if constexpr (T3) {
            const uint32_t lo = pa[kk][2 * h + 1];
            pc[kk][2 * h] = pack16<V>(r0 - low16<V>(lo), r1 - high16<V>(lo));
            pc[kk][2 * h + 1] = 0u;
          }
        }
      if constexpr (!C::kInt8) {
#pragma unroll
        for (int i = 0; i < S::TILES; i += 2) {
          uint32_t vb[KK][4];  // 16 keys x 16 dimensions, transposed
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
            ldmatrix4_t(vb[kk], st_s + S::HALF + place<C, D>(kk * 16 + (lane & 15), i + (lane >> 4)));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t b[KK][2];
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) b[kk][0] = vb[kk][2 * y], b[kk][1] = vb[kk][2 * y + 1];
            add_products<V, T3>(o[i + y], pa, pc, b);
          }
        }
      } else {
        // W words of codes a row: the first eight tiles' codes, then the others'
        auto tiles = [&](auto words, int first_byte, int tile) {
          constexpr int W = decltype(words)::value;
          uint32_t vw[KK][4][W];
#pragma unroll
          for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int key = kk * 16 + (x >> 1) * 8 + 2 * c4 + (x & 1);
              const int byte = first_byte + g8 * (4 * W);
              lds_words<W>(vw[kk][x], st + S::HALF + place<C, D>(key, byte >> 4) + (byte & 15));
            }
#pragma unroll
          for (int x = 0; x < W; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t sel = e & 1 ? 0x4342u : 0x4140u, pair = e < 2 ? 0x5140u : 0x7362u;
              uint32_t b[KK][2];
#pragma unroll
              for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                  b[kk][y] = codes_bf16(prmt(vw[kk][2 * y][x], vw[kk][2 * y + 1][x], pair), sel);
              add_products<V, T3>(o[tile + 4 * x + e], pa, pc, b);
            }
        };
        tiles(std::integral_constant<int, 2>{}, 0, 0);
        if constexpr (D > 64) tiles(std::integral_constant<int, (D - 64) / 32>{}, 64, 8);
      }
    }

    // ---- values that are not finite, for the rows that see them: cleared ones of the
    // steps noted; and where an output is not finite, all (an infinity that met a
    // weight's parts one by one is a NaN by now), unless the row's sum is none either.
    // A lane looks at one key.
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float f0 = 0.0f, f1 = 0.0f;
#pragma unroll
    for (int i = 0; i < S::TILES; ++i) {
      f0 = fmaf(o[i][0], 0.0f, f0), f1 = fmaf(o[i][1], 0.0f, f1);
      f0 = fmaf(o[i][2], 0.0f, f0), f1 = fmaf(o[i][3], 0.0f, f1);
    }
    const bool all_steps = __any_sync(0xffffffffu, f0 + f1 != 0.0f && finite(l)) || nbad > kBad;
    if (all_steps || nbad) {
#pragma unroll 1
      for (int b = 0; b < D / 32; ++b) {
        uint32_t up = 0, down = 0;  // of the block's columns: a +inf or NaN, a -inf or NaN
#pragma unroll 1
        for (int s = 0; s < (all_steps ? steps : nbad); ++s) {
          const int key0 = all_steps ? w.key(warp + s / SPU * kWarps) + s % SPU * S::KS
                                     : __shfl_sync(0xffffffffu, badkey, s);
          const int j = key0 + lane;
          const int page = lane < S::KS && j < w.rq.limit ? page_of(a, w.b, j) : -1;
          uint32_t see = __ballot_sync(0xffffffffu, page >= 0) & below(pos + 1 - key0) &
                         (~below(row_lo - key0) | below(a.sinks - key0));
          if (!row_ok) see = 0;
          uint32_t x = 0, y = 0;
          if (page >= 0) bad_columns<C>(a, w.head, page, j, 32 * b, x, y);
          uint32_t keys = __ballot_sync(0xffffffffu, (x | y) != 0);
          while (keys) {
            const int k = __ffs(keys) - 1;
            keys &= keys - 1;
            const uint32_t xs = __shfl_sync(0xffffffffu, x, k), ys = __shfl_sync(0xffffffffu, y, k);
            if (see >> k & 1u) up |= xs, down |= ys;
          }
        }
#pragma unroll
        for (int i = 0; i < S::TILES; ++i)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int d = value_dim<C, D>(2 * c4 + y, i) - 32 * b;
            if (d < 0 || d >= 32 || !((up | down) >> d & 1u)) continue;
            o[i][y] = !(up >> d & 1u) ? -INFINITY : down >> d & 1u ? NAN : INFINITY;
            o[i][y + 2] = 0.0f;
          }
      }
    }
    // ---- join the warps that had steps: a row of the block by one warp
    if (warp < w.n && c4 == 0) {
      s_m[warp][g8] = m;
      s_l[warp][g8] = l;
    }
    const int nw = min(kWarps, w.n);
    constexpr int DL = D / 32;
    const Sharers sh = sharers(w.item0, w.un.n, w.per);
    const bool alone = sh.last == sh.first;
    constexpr int kSlot = kRows * (D + 2);

    auto finish = [&](int row, const float* ro, float rm, float rl) {
      const int rr = w.block * kRows + row;
      const int t = rr / a.group, g = rr % a.group;
      const int qh = w.head * a.group + g;
      const int64_t orow = (w.rq.start + t) * a.o_token + qh * a.o_head;
#pragma unroll
      for (int i = 0; i < DL; ++i)
        store_elem(a.out, a.q_type, orow + lane + 32 * i, rl == 0.0f ? 0.0f : __fdiv_rn(ro[i], rl));
      if (a.lse && lane == 0)
        a.lse[static_cast<int64_t>(w.rq.start + t) * a.heads + qh] =
            rl == 0.0f ? -INFINITY : (rm + (log2f(rl) - kTop)) * kLn2;
    };

    for (int row0 = 0; row0 < rows; row0 += kWarps) {
      if (row0) __syncthreads();
      if (warp < w.n && row_ok && g8 >= row0 && g8 < row0 + kWarps) {
        float* so = s_o + (warp * kWarps + g8 - row0) * D;
#pragma unroll
        for (int i = 0; i < S::TILES; ++i) {
          so[value_dim<C, D>(2 * c4, i)] = fmaf(o[i][2], kDownV, o[i][0]);
          so[value_dim<C, D>(2 * c4 + 1, i)] = fmaf(o[i][3], kDownV, o[i][1]);
        }
      }
      __syncthreads();
      const int row = row0 + warp;
      if (row >= rows) continue;
      float ro[DL], rm = -INFINITY, rl = 0.0f;
#pragma unroll
      for (int i = 0; i < DL; ++i) ro[i] = 0.0f;
      for (int x = 0; x < nw; ++x) rm = fmaxf(rm, s_m[x][row]);
      const float ref = rm == -INFINITY ? 0.0f : rm;
      for (int x = 0; x < nw; ++x) {
        const float f = ex2(s_m[x][row] - ref);
        rl = fmaf(s_l[x][row], f, rl);
#pragma unroll
        for (int i = 0; i < DL; ++i)
          ro[i] = fmaf(s_o[(x * kWarps + warp) * D + lane + 32 * i], f, ro[i]);
      }
      if (alone) {
        finish(row, ro, rm, rl);
      } else {
        float* mine = a.partials + static_cast<int64_t>(slot_of(blockIdx.x, w.item0, w.per)) * kSlot;
#pragma unroll
        for (int i = 0; i < DL; ++i) mine[row * D + lane + 32 * i] = ro[i];
        if (lane == 0) {
          mine[kRows * D + row] = rm;
          mine[kRows * D + kRows + row] = rl;
        }
      }
    }
    // ---- an item of several CTAs: the one that arrives last joins the parts
    if (!alone) {
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();  // (for the block's stores: they are before the barrier)
        const uint32_t n = static_cast<uint32_t>(sh.last - sh.first);
        s_last = atomicInc(a.counters + sh.first, n) == n;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        for (int row = warp; row < rows; row += kWarps) {
          // in CTA order, four parts' loads on their way together
          float ro[DL], rm = -INFINITY, rl = 0.0f;
#pragma unroll
          for (int i = 0; i < DL; ++i) ro[i] = 0.0f;
          for (int x0 = sh.first; x0 <= sh.last; x0 += 4) {
            float pm[4], pl[4], po[4][DL];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const bool on = x0 + y <= sh.last;
              const float* part = a.partials + slot_of(min(x0 + y, sh.last), w.item0, w.per) *
                                                   static_cast<int64_t>(kSlot);
              pm[y] = on ? __ldcg(part + kRows * D + row) : -INFINITY;
              pl[y] = on ? __ldcg(part + kRows * D + kRows + row) : 0.0f;
#pragma unroll
              for (int i = 0; i < DL; ++i) po[y][i] = on ? __ldcg(part + row * D + lane + 32 * i) : 0.0f;
            }
            const float mn = fmaxf(fmaxf(rm, fmaxf(pm[0], pm[1])), fmaxf(pm[2], pm[3]));
            const float ref = mn == -INFINITY ? 0.0f : mn;
            const float f = ex2(rm - ref);
            rl *= f;
#pragma unroll
            for (int i = 0; i < DL; ++i) ro[i] *= f;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const float g = ex2(pm[y] - ref);
              rl = fmaf(pl[y], g, rl);
#pragma unroll
              for (int i = 0; i < DL; ++i) ro[i] = fmaf(po[y][i], g, ro[i]);
            }
            rm = mn;
          }
          finish(row, ro, rm, rl);
        }
      }
    }
    __syncthreads();  // s_o, s_m, s_l, s_last are free for the next item
    w.close(a);
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <class C, int D, bool T3>
int launch(const Args& a, cudaStream_t st) {
  using S = Shape<C, D>;
  const DeviceInfo& di = device_info();
  static int attr_set[kMaxDevices];
  const int slot = di.ordinal % kMaxDevices;
  if (!attr_set[slot]) {
    const cudaError_t e = cudaFuncSetAttribute(
        k_attn_rows<C, D, T3>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return cuda_status(e);
    attr_set[slot] = 1;
  }
  k_attn_rows<C, D, T3><<<2 * di.sm_count, kThreads, S::SMEM, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <class C, bool T3>
int launch_dim(const Args& a, int dim, cudaStream_t st) {
  switch (dim) {
    case 64: return launch<C, 64, T3>(a, st);
    case 96: return launch<C, 96, T3>(a, st);
    case 128: return launch<C, 128, T3>(a, st);
    default: return LP_ERR_UNSUPPORTED;
  }
}

}  // namespace

int launch_attn_rows(const attn::Args& a, int cache_type, int dim, cudaStream_t st) {
  if (cache_type == LP_F16) return launch_dim<CF16, false>(a, dim, st);
  // fp32 results take three parts of bf16, fp16 and bf16 ones two
  const bool full = a.q_type == LP_F32;
  if (cache_type == LP_I8)
    return full ? launch_dim<CI8, true>(a, dim, st) : launch_dim<CI8, false>(a, dim, st);
  return full ? launch_dim<CBF16, true>(a, dim, st) : launch_dim<CBF16, false>(a, dim, st);
}

}  // namespace lp
