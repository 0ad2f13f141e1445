// attn.cuh -- what the paged-attention kernels share: their arguments, the
// split of the work over the grid, the visible keys of a row, and the care for
// what masked keys hold.
//
// Work split.  The query rows of request b and key head h are the pairs (new
// token t, query head g of the group), r = t * G + g, in blocks of RB rows.
// A block sees a contiguous run of keys (with a window: the sinks' run and the
// window's run), cut into units of KU keys.  All units of all (b, h, block)
// items are laid end to end, behind each item XU more for what an item costs
// beside its keys (its queries, the join of its parts, its outputs), and every
// CTA takes one contiguous, equal share, so ragged lengths, few long requests
// and many short ones all fill the grid.
// An item cut by a CTA boundary leaves partial results (running maximum, sum
// and unnormalised output, fp32) in the workspace; the CTA that arrives last
// adds them in CTA order, so results do not depend on the timing.
#pragma once
#include <cuda_bf16.h>

#include "lp_device.cuh"
#include "lp_internal.h"

namespace lp {
namespace attn {

struct Pool {  // one of the cache's two tensors; strides in elements
  const uint8_t* data;
  const float* scales;
  int64_t page, token, head;     // strides of data
  int64_t spage, stoken, shead;  // strides of scales
};

struct Args {
  const void* q;
  void* out;
  float* lse;  // [tokens, heads] or null
  int q_type;  // LP_F32 / LP_F16 / LP_BF16, out's too
  int q_vec;   // rows of q and out start on 16-byte boundaries
  int64_t q_token, q_head, o_token, o_head;
  Pool k, v;
  const int32_t* table;
  const int32_t* qstart;
  const int32_t* seqlens;
  int64_t table_stride;
  int table_width, pages, page_size;
  int page_shift;  // log2 of page_size, -1 where it is no power of two
  int requests, tokens, heads, kv_heads, group;
  int window, sinks;  // window 0: none
  float scale_log2;   // softmax scale * log2(e)
  uint32_t* counters;
  float* partials;
};

// ------------------------------------------------------- requests, rows

struct Request {
  int start, n;  // first row of q, new tokens
  int base;      // position of the first new token (may be negative)
  int limit;     // keys the table can hold, at most the request's length
};

__device__ __forceinline__ Request request(const Args& a, int b) {
  Request r;
  r.start = min(max(__ldg(a.qstart + b), 0), a.tokens);
  r.n = min(max(__ldg(a.qstart + b + 1), r.start), a.tokens) - r.start;
  // (below 2^31 by more than a tile, so that key numbers do not wrap)
  const int seq = min(max(__ldg(a.seqlens + b), 0), 0x7fffff00);
  r.base = seq - r.n;
  r.limit = static_cast<int>(
      min(static_cast<int64_t>(seq), static_cast<int64_t>(a.table_width) * a.page_size));
  return r;
}

// Units that rows [row0, row0 + RB) of a request see: the first `sink` units
// of the cache, then the units from `first` on.
struct Units {
  int sink, first, n;
  int lo, hi;  // the window's run of keys, [lo, hi]
};

template <int KU, int RB>
__device__ __forceinline__ Units units(const Args& a, const Request& r, int block) {
  Units u;
  const int rows = r.n * a.group;
  const int p0 = r.base + block * RB / a.group;
  const int p1 = r.base + (min(block * RB + RB, rows) - 1) / a.group;
  u.hi = min(p1, r.limit - 1);
  u.lo = a.window > 0 ? max(p0 - a.window + 1, 0) : 0;
  const int sinks = a.window > 0 ? min(a.sinks, u.hi + 1) : 0;
  u.sink = sinks > 0 ? (sinks + KU - 1) / KU : 0;
  u.first = max(u.lo / KU, u.sink);
  u.n = u.hi < 0 ? 0 : u.sink + max(u.hi / KU - u.first + 1, 0);
  // a block that sees nothing still writes its zeros: one unit, all masked
  if (u.n <= 0) {
    u.n = 1;
    u.sink = 0;
    u.first = 0;
  }
  return u;
}

template <int KU, int RB, int XU>
__device__ __forceinline__ int64_t request_units(const Args& a, int b) {
  const Request r = request(a, b);
  const int blocks = (r.n * a.group + RB - 1) / RB;
  int64_t s = 0;
  for (int i = 0; i < blocks; ++i) s += units<KU, RB>(a, r, i).n + XU;
  return s;
}

// ------------------------------------------------------- the CTA's share

struct Cursor {
  int64_t begin, end;  // the CTA's units
  int64_t per_cta;     // units per CTA (the last ones may have fewer)
  int64_t item0;       // number of the current item's first unit
  int b, head, block;  // the current item
  int pad;
};

// (64-bit divisions are slow, and the numbers nearly always fit 32 bits)
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if ((a | b) >> 32) return a / b;
  return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
}

// Total units and the item that holds unit `begin` of this CTA.  Each thread
// sums a run of requests, the sums are scanned in shared memory, and the
// thread whose run holds `begin` walks it.  All threads of the block call it.
template <int KU, int RB, int XU, int THREADS>
__device__ void find_share(const Args& a, int64_t min_units, Cursor* cur, int64_t* sums) {
  const int t = threadIdx.x;
  const int run = (a.requests + THREADS - 1) / THREADS;
  const int b0 = min(t * run, a.requests), b1 = min(b0 + run, a.requests);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += request_units<KU, RB, XU>(a, b);
  mine *= a.kv_heads;
  // inclusive scan: within the warp, then over the warps' totals
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if ((t & 31) >= o) inc += y;
  }
  if ((t & 31) == 31) sums[t >> 5] = inc;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < (t >> 5)) before += sums[w];
    total += sums[w];
  }
  const int64_t excl = before + inc - mine;
  const int64_t per = max(divide(total + gridDim.x - 1, gridDim.x), min_units);
  const int64_t begin = min(static_cast<int64_t>(blockIdx.x) * per, total);
  if (t == 0) {
    cur->begin = begin;
    cur->end = min(begin + per, total);
    cur->per_cta = per;
  }
  if (begin >= excl && begin < excl + mine) {
    int64_t at = excl;
    int b = b0;
    int64_t w = request_units<KU, RB, XU>(a, b);
    while (begin >= at + w * a.kv_heads) {
      at += w * a.kv_heads;
      w = request_units<KU, RB, XU>(a, ++b);
    }
    const int head = static_cast<int>(divide(begin - at, w));
    at += head * w;
    const Request r = request(a, b);
    int block = 0;
    int n = units<KU, RB>(a, r, 0).n + XU;
    while (begin >= at + n) {
      at += n;
      n = units<KU, RB>(a, r, ++block).n + XU;
    }
    cur->b = b;
    cur->head = head;
    cur->block = block;
    cur->item0 = at;
  }
  __syncthreads();
}

// The item after (b, head, block); every thread computes the same.
template <int RB>
__device__ __forceinline__ void next_item(const Args& a, int& b, int& head, int& block) {
  Request r = request(a, b);
  if (++block < (r.n * a.group + RB - 1) / RB) return;
  block = 0;
  if (++head < a.kv_heads) return;
  head = 0;
  do {
    if (++b >= a.requests) return;
    r = request(a, b);
  } while (r.n == 0);
}

// A role's walk through the CTA's items, in order.  open() finds the next part
// of an item that has units of its own; close() steps behind it.
template <int KU, int RB, int XU>
struct Walk {
  int64_t at, end, item0, per;
  int b, head, block;
  Request rq;
  Units un;
  int u0, n, rows;  // the part: first unit of the item's, units; rows of the item

  __device__ __forceinline__ void start(const Cursor& c) {
    at = c.begin, end = c.end, item0 = c.item0, per = c.per_cta;
    b = c.b, head = c.head, block = c.block;
  }
  __device__ __forceinline__ bool open(const Args& a) {
    while (at < end) {
      rq = request(a, b);
      un = units<KU, RB>(a, rq, block);
      u0 = static_cast<int>(at - item0);
      n = static_cast<int>(min(static_cast<int64_t>(un.n), end - item0)) - u0;
      rows = min(RB, rq.n * a.group - block * RB);
      if (n > 0) return true;
      skip(a);  // the share begins behind the item's units
    }
    return false;
  }
  __device__ __forceinline__ void close(const Args& a) {
    if (u0 + n == un.n) skip(a);
    else at += n;
  }
  __device__ __forceinline__ void skip(const Args& a) {
    item0 += un.n + XU;
    at = item0;
    next_item<RB>(a, b, head, block);
  }
  // first key of the part's i-th unit
  __device__ __forceinline__ int key(int i) const {
    const int u = u0 + i;
    return (u < un.sink ? u : un.first + u - un.sink) * KU;
  }
};

// CTAs that share an item of units [u0, u0 + n): first..last, and the slot of
// a CTA's partial (0: its share begins inside the item or at its first unit).
struct Sharers {
  int first, last;
};
__device__ __forceinline__ Sharers sharers(int64_t u0, int64_t n, int64_t per) {
  return {static_cast<int>(divide(u0, per)), static_cast<int>(divide(u0 + n - 1, per))};
}
__device__ __forceinline__ int slot_of(int cta, int64_t u0, int64_t per) {
  return 2 * cta + (u0 > static_cast<int64_t>(cta) * per ? 1 : 0);
}

// ------------------------------------------------------- element access

__device__ __forceinline__ float load_elem(const void* p, int type, int64_t i) {
  if (type == LP_F32) return static_cast<const float*>(p)[i];
  if (type == LP_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// One rounding, to the output's type.
__device__ __forceinline__ void store_elem(void* p, int type, int64_t i, float v) {
  if (type == LP_F32) static_cast<float*>(p)[i] = v;
  else if (type == LP_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234e38f; }

// A key's page of its request and its place in the page.  Page sizes are
// nearly always powers of two, and a division is a long chain of instructions.
__device__ __forceinline__ int page_index(const Args& a, int j) {
  return a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
}
__device__ __forceinline__ int page_offset(const Args& a, int j) {
  return a.page_shift >= 0 ? j & (a.page_size - 1) : j % a.page_size;
}

// The table's entry for key j of request b, for use later: valid_page() looks
// at it first, so the load is not waited for where it is made.
__device__ __forceinline__ int entry_of(const Args& a, int b, int j) {
  return __ldg(a.table + b * a.table_stride + page_index(a, j));
}
__device__ __forceinline__ int valid_page(const Args& a, int entry) {
  return static_cast<unsigned>(entry) < static_cast<unsigned>(a.pages) ? entry : -1;
}

// Page of key j of request b, or -1 where the table has none.
__device__ __forceinline__ int page_of(const Args& a, int b, int j) {
  return valid_page(a, entry_of(a, b, j));
}

// ------------------------------------------------------- cache formats

struct CF16 {
  static constexpr bool kInt8 = false, kBf16 = false;
  __device__ static float to_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
};
struct CBF16 {
  static constexpr bool kInt8 = false, kBf16 = true;
  __device__ static float to_float(uint16_t v) {
    return __uint_as_float(static_cast<uint32_t>(v) << 16);
  }
};
struct CI8 {  // codes are widened to fp16, which holds them exactly
  static constexpr bool kInt8 = true, kBf16 = false;
};

// Masked keys.  A masked key's weight is 0, but 0 times an infinity or a NaN in
// its value is a NaN, which no row that does not see the key may get.  So where
// a tile of keys is not seen whole by all rows of an item (its last keys, a
// window's edge, holes in the table), values that are not finite are replaced by
// zeros in shared memory and the tile's first key is noted; afterwards those
// values are added to the outputs of the rows that do see them, which makes them
// what the sum over the row's own keys is.  Tiles that all rows see need none of
// this, and neither do finite values.  But where a weight has several parts, an
// infinity meets them one by one, and a part of 0 makes a NaN of it; so an output
// that is not finite, in a row whose sum of weights is, is found again from all the
// keys that the row sees.

// 16 bytes of values; returns whether one was replaced.
template <class C>
__device__ __forceinline__ bool clear_bad(uint8_t* p) {
  constexpr uint32_t kExp = C::kBf16 ? 0x7f80u : 0x7c00u, kOne = C::kBf16 ? 0x0080u : 0x0400u;
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
  // an exponent of all ones plus one carries into the sign's place
  uint32_t carry = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) carry |= (w[i] & (kExp | kExp << 16)) + (kOne | kOne << 16);
  if (!(carry & 0x80008000u)) return false;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (w[i] & kExp) == kExp, hi = (w[i] >> 16 & kExp) == kExp;
    w[i] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
    bad = bad || lo || hi;
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  return bad;
}
__device__ __forceinline__ bool clear_bad_scale(float* p) {
  const bool bad = !finite(*p);
  if (bad) *p = 0.0f;
  return bad;
}

// Bits of keys key0 .. key0 + 31 that are below x.
__device__ __forceinline__ uint32_t below(int x) {
  return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u;
}

// Value d of key j of request b and key head h, if it is not finite, else 0.
template <class C>
__device__ __forceinline__ float bad_value(const Args& a, int b, int h, int page, int j, int d) {
  const int off = page_offset(a, j);
  const int64_t row = page * a.v.page + off * a.v.token + h * a.v.head + d;
  float v;
  if constexpr (C::kInt8)
    v = static_cast<float>(reinterpret_cast<const int8_t*>(a.v.data)[row]) *
        a.v.scales[page * a.v.spage + off * a.v.stoken + h * a.v.shead];
  else
    v = C::to_float(reinterpret_cast<const uint16_t*>(a.v.data)[row]);
  return finite(v) ? 0.0f : v;
}
// Of values d .. d + 31 of key j: those that are +inf or NaN, and -inf or NaN, a
// bit each.
template <class C>
__device__ __forceinline__ void bad_columns(const Args& a, int h, int page, int j, int d,
                                            uint32_t& up, uint32_t& down) {
  const int off = page_offset(a, j);
  const int64_t row = page * a.v.page + off * a.v.token + h * a.v.head + d;
  up = down = 0;
  if constexpr (C::kInt8) {
    const float s = a.v.scales[page * a.v.spage + off * a.v.stoken + h * a.v.shead];
    if (finite(s)) return;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(a.v.data + row);  // (rows are aligned)
    uint32_t above = 0, below = 0;  // codes over and under 0
#pragma unroll 1
    for (int e = 0; e < 32; e += 4) {
      const uint32_t w = __ldg(p++);
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int code = static_cast<int8_t>(w >> (8 * y) & 255u);
        above |= (code > 0 ? 1u : 0u) << (e + y);
        below |= (code < 0 ? 1u : 0u) << (e + y);
      }
    }
    // a code of 0 gives NaN, and so does a scale
    up = s > 0.0f ? ~below : s < 0.0f ? ~above : 0xffffffffu;
    down = s > 0.0f ? ~above : s < 0.0f ? ~below : 0xffffffffu;
  } else {
    constexpr uint32_t kInf = C::kBf16 ? 0x7f80u : 0x7c00u;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(a.v.data + 2 * row);  // (rows are aligned)
#pragma unroll 1
    for (int e = 0; e < 32; e += 2) {
      const uint32_t w = __ldg(p++);
      const uint32_t x = w & 0xffffu, y = w >> 16;
      up |= ((x & 0x7fffu) > kInf || x == kInf ? 1u << e : 0u) |
            ((y & 0x7fffu) > kInf || y == kInf ? 2u << e : 0u);
      down |= (x >= (kInf | 0x8000u) || (x < 0x8000u && x > kInf) ? 1u << e : 0u) |
              (y >= (kInf | 0x8000u) || (y < 0x8000u && y > kInf) ? 2u << e : 0u);
    }
  }
}
// Whether a row at position pos sees key j (the page aside).
__device__ __forceinline__ bool sees(const Args& a, const Request& r, int pos, int j) {
  return j <= pos && j < r.limit && (a.window == 0 || j > pos - a.window || j < a.sinks);
}

// (a, b) rounded to the 16-bit type of the tensor-core operands, a in the low half
template <class C>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  uint32_t r;
  if constexpr (C::kBf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <class C>
__device__ __forceinline__ float low16(uint32_t w) {
  if constexpr (C::kBf16) return __uint_as_float(w << 16);
  else return h2f(w & 0xffffu);
}
template <class C>
__device__ __forceinline__ float high16(uint32_t w) {
  if constexpr (C::kBf16) return __uint_as_float(w & 0xffff0000u);
  else return h2f(w >> 16);
}

// Bytes u0..u3 of w, each code + 128, to two packed pairs of fp16 codes:
// 0x64 before a byte is the fp16 number 1024 + byte, and 1152 less is the code.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t sel) {
  const uint32_t x = prmt(w, 0x64646464u, sel);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
  return r;
}

// Two signed bytes of w to packed bf16: 0x43 before a byte's low seven bits is
// 128 + those, before its top bit 128 or 256; the difference is the code.
__device__ __forceinline__ uint32_t codes_bf16(uint32_t w, uint32_t sel) {
  const uint32_t x = prmt(w, 0x43434343u, sel);
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x & 0x437f437fu), "r"(x & 0x43804380u));
  return r;
}

// The power of two that brings |x| <= amax below 1 (1 where amax is 0 or not
// finite), as an exponent e: 2^-e * amax < 1 (< 4 next to the type's end).
__device__ __forceinline__ int row_exponent(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 126;
  return amax == 0.0f || !finite(amax) ? 0 : min(max(e, -100), 126);
}
__device__ __forceinline__ float pow2(int e) {  // -126 <= e <= 127
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

}  // namespace attn
}  // namespace lp
