// attn_chunk.cu -- attention of a chunk of new tokens over a paged cache, on
// the 5th-generation tensor cores.
//
//   S = Q K^T, P = exp2(c S - m), O += P V, l += sum P      (one pass over the keys)
//
// CTA = TILES row tiles of 128 query rows (token, head of the group) of one
// key head, key tiles of 128 keys; 16 warps, of which
//   warps 0-3, 4-7  softmax, one thread per row (tensor memory lane).  Two row
//                   tiles: one warpgroup each.  One row tile: both share it,
//                   64 keys each, and swap the row maxima in shared memory.
//   warps 8-11      load keys and values into a ring of swizzled 128-key
//                   tiles, 16 bytes a lane: pages may have any size and any
//                   16-byte strides, and keys that no row of the tile sees
//                   (past the end, before the window, on missing pages) are
//                   zeros, whatever the cache holds there.  fp16 and bf16
//                   pages go by cp.async into the ring; int8 codes by cp.async
//                   into a small ring of their own, from where the thread that
//                   fetched them widens them (exactly) to the operand type.
//   warp 12         issues the products: tcgen05.mma kind::f16,
//                   M = 128, S and O in tensor memory, P from tensor memory
//                   (it takes the columns of the S it came from).
// While one tile's softmax runs, the tensor cores work on the other tile, or,
// with one row tile, on the next key tile's S (two S buffers).
//
// 16-bit queries: two row tiles, P in one part of the operand type.  fp32
// results need more bits than one 16-bit operand has, so queries and weights
// are split into two fp16 or three bf16 parts whose products add up in the
// same fp32 accumulator; that is bound by the products, so one row tile and
// the wider ring serve it.  Which types take which parts: launch_attn_chunk.
//
// Sums in tensor memory are cut off, not rounded, at every product of 16 keys,
// which over a few thousand keys would show in an fp32 result.  So there (one
// row tile) small parts come first, and a key tile's product is added to the
// outputs in the softmax's registers (measured against 64 bits on five prompts
// of up to 4700 keys: 5e-6 without, under 1e-6 with).  With two row tiles and
// tables of more than 16384 keys (bf16 weights: 131072), a sum leaves tensor memory
// for the workspace every so many tiles: values of one sign came out 5.9e-4 low
// over 131000 keys and 1.8e-3 over 400000 in fp16, now within its rounding.  (In
// one kernel for all lengths that took 4 to 7 % more time of short items, for the
// registers; long ones pay 2 to 3 %.)
//
// What bounds it: 16-bit queries the softmax and the products in turn.  4096
// tokens over 16384 cached, 32 heads on 8 key heads of 128, bf16: 1.18 to 1.2 ms by
// itself (1030 to 1050 TFLOP/s, 63 to 64 % of a cuBLAS bf16 product's rate), 1.28 to
// 1.34 ms back to back under the power limit; the special-function unit alone needs 0.5 ms, the
// products 0.76.  Tried and slower there: a third of the exponentials by a
// polynomial on the fp32 pipes (+3 %), the weights' first half handed over early
// (+0.4 %), the row's maximum chunk by chunk in one pass (+9 %).  fp32 over an
// int8 cache: 5 products where 16 bits take 2, and shared memory, which they and
// the loaders share (350 KB per key tile, 2750 cycles of about 6700): five prompts
// of up to 700 tokens over up to 4700 keys 0.32 ms.  Registers: the softmax role and
// the one that issues the products spill (in kernels of one role each, bf16 128
// dimensions, 120 and 304 bytes of stores; fp32 over int8 1508 and 276; the loaders
// none), and what the compiler keeps in the key loop changes with code far from it.
//
// The running maximum moves only when a row's grows by more than 2^8 (the
// weights stay below 2^8 times 1, or 2^15 with fp16's extra 2^7): the sums are
// the same and O is rescaled a few times per row rather than per key tile (a
// published refinement of the running-maximum softmax).
#include <type_traits>

#include "attn.cuh"
#include "tc_ptx.cuh"

namespace lp {
namespace {

using namespace attn;
using namespace tc;

constexpr int kKeys = 128;             // keys per tile, = one unit
constexpr int kSoftThreads = 256;
constexpr int kLoadThreads = 128;
constexpr int kThreads = kSoftThreads + kLoadThreads + 128;  // (whole warpgroups: setmaxnreg)
constexpr int kBlock = 128 * 128;      // bytes of 128 rows x 64 16-bit elements
constexpr int kBad = 16;               // tiles with cleared values that are noted one by one
constexpr int kPlaces = 16;            // items whose notes are held
constexpr float kLazy = 8.0f;          // log2 of the growth that moves the maximum
constexpr int kMinUnits = 2;  // (100 tokens over 4000 keys: 46 us with 1 or 2, 48 with 6, 54 with 12)
// What an item costs beside its keys, in key tiles (queries, start, outputs: 7 to
// 13 us against 1.2 to 2.5 us per tile).  Five fp32 prompts over an int8 cache,
// some of them short: 406 us with 2, 317 with 4, 311 with 7.
constexpr int kItemUnits = 6;

// C: the cache's format; Q: type of the operands of Q K^T, P: of P V;
// NQ, NP: parts of queries and weights; LONG (two row tiles): items may have more
// than HOLD key tiles.
template <class C_, class Q_, class P_, int NQ_, int NP_, int TILES_, int D_, bool LONG_>
struct Cfg {
  using C = C_;
  using Q = Q_;
  using P = P_;
  static constexpr int NQ = NQ_, NP = NP_, TILES = TILES_, D = D_;
  static constexpr bool LONG = LONG_;
  static constexpr int BLOCKS = (D + 63) / 64;
  static constexpr int TILE = BLOCKS * kBlock;  // bytes of a Q part, K or V tile
  static constexpr int STAGES = C::kInt8 ? (D == 64 ? 4 : 3) : D == 64 ? 8 : NQ == 3 ? 3 : 4;
  // int8: tiles of codes on their way, 16 bytes a lane
  static constexpr int RAW = C::kInt8 ? 3 : 0;
  static constexpr int LPR = C::kInt8 && D == 64 ? 4 : 8;  // loading lanes that share a row
  static constexpr int RAW_TILE = kKeys * LPR * 16;
  // key tiles whose presence and scales are held: the loaders write a tile's
  // before its softmax reads them, and, with this many, after the softmax of
  // the tile that had the place is done (int8 loads run a tile further ahead)
  static constexpr int META = C::kInt8 ? 6 : STAGES <= 4 ? 4 : 8;
  static constexpr int ROWS = 128 * TILES;
  static constexpr int SMEM = 1024 + TILES * NQ * TILE + STAGES * TILE + RAW * RAW_TILE;
  // Registers per thread of the roles' warpgroups; 128 each at launch.  One row
  // tile's softmax holds 64 scores and up to 64 outputs, two tiles' 128 scores.
  static constexpr int SOFT_REGS = TILES == 2 ? 200 : 208;
  static constexpr int LOAD_REGS = 64;
  static constexpr int MMA_REGS = TILES == 2 ? 48 : 32;
  static_assert(2 * SOFT_REGS + LOAD_REGS + MMA_REGS == 4 * 128, "");
  // fp16 weights are held times 2^7, bf16 has the range without
  static constexpr float kUp = P::kBf16 ? 1.0f : 128.0f;
  static constexpr float kUpLog = P::kBf16 ? 0.0f : 7.0f;
  // Two row tiles: key tiles whose sum stays in tensor memory.  8 products a tile,
  // each cut off, take 0.6e-6 of the sum a tile: up to 0.7e-4 of an fp16 result and
  // 0.6e-3 of a bf16 one, a sixth of what its rounding is.
  static constexpr int HOLD = P::kBf16 ? 1024 : 128;
  // Cleared values of few tiles are looked for by each row for itself, not by lanes
  // for all of a warp's rows.  That is slower, but finite caches pay neither, and
  // which of the two loops is there decides what the compiler keeps in registers in
  // the key loop: 1536 tokens over 6000, 32/8 heads of 96, bf16 201 us (by lanes 230),
  // fp16 207 (226); five fp32 prompts over int8 324 (366); but bf16 over int8, heads of
  // 96, 387 (361), and bf16 heads of 128, 60 short requests, 110 (106).
  static constexpr bool BY_ROW = TILES == 1 || (D == 96 && !C::kInt8);
};

template <class F>
using WalkOf = Walk<kKeys, F::ROWS, kItemUnits>;

struct Shared {
  Cursor cur;
  int64_t sums[kThreads / 32];
  uint64_t full[8], empty[8];
  uint64_t qfull[2], sfull[2], pfull[2], pvdone[2], done;
  uint32_t tmem;
  volatile int abort;
  int last;
  uint32_t there[8][4];           // keys of a tile that are loaded
  float xmax[2][2][128], xsum[2][128];
  int nbad[kPlaces], badkey[kPlaces][kBad];     // per item: tiles with cleared values, their first keys
  int64_t koff[3][128], voff[3][128];  // rows of a tile in the cache, -1: zeros
};
template <int N>
struct __align__(16) Scales {
  float k[N][128], v[N][128];
};

__device__ __forceinline__ void named_bar(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0)
               : "memory");
}
// Whether the phase is over, without the suspension of try_wait.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(saddr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint64_t pku(uint32_t a, uint32_t b) {
  return pk(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ void upku(uint64_t r, uint32_t& a, uint32_t& b) {
  float x, y;
  upk(r, x, y);
  a = __float_as_uint(x), b = __float_as_uint(y);
}
__device__ __forceinline__ void tie(uint32_t* r, int n) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i < n) asm volatile("" : "+r"(r[i]));
}
// Where a role is in the ring of key and value tiles.
template <int STAGES>
struct Ring {
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == STAGES) stage = 0, phase ^= 1;
  }
};

// ------------------------------------------------------------- loaders

template <class F>
__device__ __forceinline__ void load_role(const Args& a, WalkOf<F> w, Shared& sh,
                                          Scales<F::META>* scales, uint8_t* ring, uint8_t* raw) {
  using C = typename F::C;
  constexpr int ES = C::kInt8 ? 1 : 2;
  constexpr int CH = C::kInt8 ? 16 : 8;       // elements per load
  constexpr int CPR = F::D / CH;              // loads per row (int8: 4, 6, 8; 16-bit: 8, 12, 16)
  constexpr int LPR = F::LPR;                 // lanes that share a row
  constexpr int RPP = kLoadThreads / LPR;     // rows per pass
  constexpr int RPT = kKeys / RPP;            // rows per thread
  const int t = threadIdx.x - kSoftThreads;
  const int sub = t % LPR, row0 = t / LPR;
  Ring<F::STAGES> at;   // the next tile to put
  bool lap = false;     // the ring has been filled once
  uint32_t tile = 0;    // key tiles so far, over all items: meta slot

  uint32_t item = 0;    // items so far, whose notes are in place item % kPlaces
  // Tile i is seen whole by all rows of the item: keys up to the first row's
  // position, from the last row's window on.
  auto whole = [&](int i, uint32_t slot) {
    const int key0 = w.key(i);
    const int p_first = w.rq.base + w.block * F::ROWS / a.group;
    const int lo_last = a.window > 0 ? w.rq.base + (w.block * F::ROWS + w.rows - 1) / a.group - a.window + 1 : 0;
    const uint32_t* th = sh.there[slot % F::META];
    return key0 + kKeys - 1 <= p_first && (key0 >= lo_last || key0 + kKeys <= a.sinks) &&
           (th[0] & th[1] & th[2] & th[3]) == 0xffffffffu;
  };
  auto note = [&](bool bad, int place, int key0) {
    if (__any_sync(0xffffffffu, bad) && (t & 31) == 0) {
      const int n = atomicAdd(&sh.nbad[place], 1);
      if (n < kBad) sh.badkey[place][n] = key0;
    }
  };
  // The table's entry for key t of the item's tile i: looked up a tile ahead.
  int next_entry = -1;
  auto look = [&](int i) {
    const int j = w.key(i) + t;
    next_entry = -1;
    if (j <= w.un.hi && (j >= w.un.lo || j < a.sinks)) next_entry = entry_of(a, w.b, j);
  };
  // where tile i's rows are; its scales and presence for the softmax
  auto locate = [&](int i, uint32_t slot) {
    const int page = valid_page(a, next_entry);
    if (i + 1 < w.n) look(i + 1);
    const bool on = page >= 0;
    const int off = on ? page_offset(a, w.key(i) + t) : 0;
    const int m = slot % 3;
    sh.koff[m][t] = on ? page * a.k.page + off * a.k.token + w.head * a.k.head : -1;
    sh.voff[m][t] = on ? page * a.v.page + off * a.v.token + w.head * a.v.head : -1;
    const int mm = slot % F::META;
    const uint32_t bits = __ballot_sync(0xffffffffu, on);
    if ((t & 31) == 0) sh.there[mm][t >> 5] = bits;
    if constexpr (C::kInt8) {
      const int64_t p = on ? page : 0;
      cp4(saddr(&scales->k[mm][t]),
          a.k.scales + p * a.k.spage + off * a.k.stoken + w.head * a.k.shead, on);
      cp4(saddr(&scales->v[mm][t]),
          a.v.scales + p * a.v.spage + off * a.v.stoken + w.head * a.v.shead, on);
    }
    named_bar(3, kLoadThreads);
  };

  if constexpr (!C::kInt8) {
    Ring<F::STAGES> told;   // the next tile to signal
    int untold = 0;
    // of the tiles not yet signalled, oldest first: values to look through?
    uint32_t look_through = 0;
    int key_q[3] = {0, 0, 0}, item_q[3] = {0, 0, 0};
    auto tell = [&] {  // (the oldest one's copies have landed)
      if (look_through & 1u) {
        uint8_t* p = ring + told.stage * F::TILE;
        bool bad = false;
#pragma unroll 4
        for (int i = 0; i < RPT; ++i) {
          const int r = row0 + i * RPP;
#pragma unroll
          for (int x = 0; x < (CPR + LPR - 1) / LPR; ++x)
            if (x * LPR + sub < CPR) bad |= clear_bad<typename F::P>(p + x * kBlock + r * 128 + ((sub ^ (r & 7)) << 4));
        }
        __syncwarp();
        note(bad, item_q[0], key_q[0]);
      }
      look_through >>= 1;
      key_q[0] = key_q[1], key_q[1] = key_q[2];
      item_q[0] = item_q[1], item_q[1] = item_q[2];
      fence_async();
      mbar_arrive(&sh.full[told.stage]);
      told.next();
      --untold;
    };
    auto put = [&](const Pool& pool, const int64_t* offs, int value_tile) {
      if (lap && !mbar_test(&sh.empty[at.stage], at.phase ^ 1)) {
        // no room yet: what is on its way must not wait for it
        cp_wait<0>();
        while (untold) tell();
        mbar_wait(&sh.empty[at.stage], at.phase ^ 1, &sh.abort);
      }
      const uint32_t dst = saddr(ring + at.stage * F::TILE);
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const int r = row0 + i * RPP;
        const int64_t off = offs[r];
        const uint8_t* src = pool.data + (off < 0 ? 0 : off * ES);
#pragma unroll
        for (int c = 0; c < (CPR + LPR - 1) / LPR; ++c)
          if (c * LPR + sub < CPR)
            cp16(dst + c * kBlock + r * 128 + ((sub ^ (r & 7)) << 4), src + (c * LPR + sub) * 16,
                 off >= 0);
      }
      cp_commit();
      at.next();
      lap = lap || at.stage == 0;
      if (value_tile >= 0 && !whole(value_tile, tile + value_tile)) {
        look_through |= 1u << untold;
        const int key0 = w.key(value_tile), place = item % kPlaces;
        if (untold == 0) key_q[0] = key0, item_q[0] = place;
        else if (untold == 1) key_q[1] = key0, item_q[1] = place;
        else key_q[2] = key0, item_q[2] = place;
      }
      if (++untold > 2) {  // three tiles in flight
        cp_wait<2>();
        tell();
      }
    };
    while (w.open(a)) {
      look(0);
      if (F::TILES == 2) {
        for (int i = 0; i < w.n; ++i) {
          locate(i, tile + i);
          put(a.k, sh.koff[(tile + i) % 3], -1);
          put(a.v, sh.voff[(tile + i) % 3], i);
        }
      } else {
        locate(0, tile);
        put(a.k, sh.koff[tile % 3], -1);
        for (int i = 0; i < w.n; ++i) {
          if (i + 1 < w.n) {
            locate(i + 1, tile + i + 1);
            put(a.k, sh.koff[(tile + i + 1) % 3], -1);
          }
          put(a.v, sh.voff[(tile + i) % 3], i);
        }
      }
      tile += w.n;
      ++item;
      w.close(a);
    }
    cp_wait<0>();
    while (untold) tell();
  } else {
    // The item's tiles in the order of their use, RAW of them on their way.  A
    // thread widens the pieces that it fetched itself, so only its own copies
    // have to have landed.
    uint8_t* mine = raw + t * 16;
    auto kind = [&](int q, int& i) {  // of the q-th tile: key tile i's values?
      if (F::TILES == 2) {
        i = q >> 1;
        return (q & 1) != 0;
      }
      const bool v = q == 2 * w.n - 1 || (q > 0 && (q & 1) == 0);
      i = q == 2 * w.n - 1 ? w.n - 1 : v ? (q >> 1) - 1 : (q + 1) >> 1;
      return v;
    };
    auto issue = [&](int q, int slot) {
      if (q < 2 * w.n) {
        int i;
        const bool v = kind(q, i);
        if (!v) locate(i, tile + i);
        const int m = (tile + i) % 3;
        const Pool& pool = v ? a.v : a.k;
        const int64_t* offs = v ? sh.voff[m] : sh.koff[m];
        const uint32_t dst = saddr(mine + slot * F::RAW_TILE);
#pragma unroll
        for (int x = 0; x < RPT; ++x) {
          const int64_t off = offs[row0 + x * RPP];
          if (sub < CPR) cp16(dst + x * (kLoadThreads * 16), pool.data + (off < 0 ? 0 : off) + sub * 16, off >= 0);
        }
      }
      cp_commit();
    };
    auto widen = [&](auto type, int slot) {
      using T = decltype(type);
      uint8_t* dst = ring + at.stage * F::TILE + (sub >> 2) * kBlock;
      if (sub < CPR) {
#pragma unroll
        for (int x = 0; x < RPT; ++x) {
          const int r = row0 + x * RPP;
          const uint4 u = *reinterpret_cast<const uint4*>(mine + slot * F::RAW_TILE +
                                                          x * (kLoadThreads * 16));
          const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
          uint32_t o[8];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            if constexpr (T::kBf16) {
              o[2 * y] = codes_bf16(w4[y], 0x4140u);
              o[2 * y + 1] = codes_bf16(w4[y], 0x4342u);
            } else {
              o[2 * y] = codes_f16(w4[y] ^ 0x80808080u, 0x4140u);
              o[2 * y + 1] = codes_f16(w4[y] ^ 0x80808080u, 0x4342u);
            }
          }
          uint8_t* p = dst + r * 128;
          // lanes of the two column blocks write their halves in opposite order:
          // eight lanes then meet in no bank
          const bool odd = sub >> 2 & 1;
          const int c = ((sub & 3) * 2 + odd) ^ (r & 7);
          const uint4 h0 = make_uint4(o[0], o[1], o[2], o[3]), h1 = make_uint4(o[4], o[5], o[6], o[7]);
          *reinterpret_cast<uint4*>(p + (c << 4)) = odd ? h1 : h0;
          *reinterpret_cast<uint4*>(p + ((c ^ 1) << 4)) = odd ? h0 : h1;
        }
      }
    };
    while (w.open(a)) {
      look(0);
      for (int q = 0; q < F::RAW; ++q) issue(q, q);
      int slot = 0;
      for (int q = 0; q < 2 * w.n; ++q) {
        cp_wait<F::RAW - 1>();
        if (lap) mbar_wait(&sh.empty[at.stage], at.phase ^ 1, &sh.abort);
        int i;
        if (kind(q, i)) {
          widen(typename F::P{}, slot);
        } else {
          widen(typename F::Q{}, slot);
          // (the value scales came with the keys; the softmax has not seen them)
          if (!whole(i, tile + i))
            note(clear_bad_scale(&scales->v[(tile + i) % F::META][t]), item % kPlaces, w.key(i));
        }
        fence_async();
        mbar_arrive(&sh.full[at.stage]);
        at.next();
        lap = lap || at.stage == 0;
        issue(q + F::RAW, slot);
        slot = slot + 1 == F::RAW ? 0 : slot + 1;
      }
      tile += w.n;
      ++item;
      w.close(a);
    }
    cp_wait<0>();
  }
}

// ------------------------------------------------------------ products

// Tensor memory columns: S (and P) of tile or buffer x, O of tile x, third
// parts of the weights of buffer x.
__device__ __forceinline__ uint32_t s_col(int x) { return 128u * x; }
__device__ __forceinline__ uint32_t o_col(int x) { return 256u + 128u * x; }
__device__ __forceinline__ uint32_t p3_col(int x) { return 384u + 64u * x; }

// One lane of a converged warp, the same one every time.  The warp stays
// together around it, so descriptors and addresses live in uniform registers:
// a lone thread's products each waited about 120 cycles for theirs to be moved
// there, twice what the product takes.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred P; elect.sync _|P, 0xffffffff; selp.u32 %0, 1, 0, P; }" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

template <class F>
__device__ __forceinline__ void mma_role(const Args& a, WalkOf<F> w, Shared& sh, const uint8_t* qs,
                                         const uint8_t* ring) {
  constexpr uint32_t id_qk = idesc_f16(F::Q::kBf16, false, 128, kKeys);
  constexpr uint32_t id_pv = idesc_f16(F::P::kBf16, true, 128, F::D);
  const uint32_t tm = static_cast<uint32_t>(uniform(static_cast<int>(sh.tmem)));
  const uint64_t q_desc = sw128_desc(qs), k_desc = sw128_desc(ring);
  const uint64_t v_desc = sw128_mn_desc(ring, kBlock);
  Ring<F::STAGES> at;
  uint32_t nq[2] = {0, 0};  // items so far, per tile
  uint32_t np[2] = {0, 0};  // weights taken so far, per tile or buffer
  uint32_t nb = 0;          // one row tile: key tiles so far

  auto wait_tile = [&] {
    mbar_wait(&sh.full[at.stage], at.phase, &sh.abort);
    __syncwarp();
    fence_after();
  };
  // a descriptor's address field counts 16 bytes: an offset is an add
  auto qk = [&](int tile, int x, uint32_t stage, bool last) {
    if (elect_one()) {
      const uint64_t kd = k_desc + stage * (F::TILE >> 4);
#pragma unroll
      for (int p = F::NQ - 1; p >= 0; --p) {  // small parts first
        const uint64_t qd = q_desc + (tile * F::NQ + p) * (F::TILE >> 4);
#pragma unroll
        for (int s = 0; s < F::D / 16; ++s) {
          const int o = ((s / 4) * kBlock + (s % 4) * 32) >> 4;
          mma_f16(tm + s_col(x), qd + o, kd + o, id_qk, p + 1 < F::NQ || s > 0);
        }
      }
      mma_commit(&sh.sfull[x]);
      if (last) mma_commit(&sh.empty[stage]);
    }
    __syncwarp();
  };
  auto pv = [&](int tile, int x, uint32_t stage, bool first, bool last) {
    mbar_wait(&sh.pfull[x], np[x]++ & 1, &sh.abort);
    __syncwarp();
    fence_after();
    if (elect_one()) {
      const uint64_t vd = v_desc + stage * (F::TILE >> 4);
#pragma unroll
      for (int p = F::NP - 1; p >= 0; --p)
#pragma unroll
        for (int s = 0; s < kKeys / 16; ++s) {
          const uint32_t col = p < 2 ? s_col(x) + 32 * (s / 2) + 8 * (s % 2) + 16 * p
                                     : p3_col(x) + 8 * s;
          mma_f16_ta(tm + o_col(tile), tm + col, vd + s * (2048 >> 4), id_pv,
                     !first || p + 1 < F::NP || s > 0);
        }
      mma_commit(&sh.pvdone[x]);
      if (last) mma_commit(&sh.empty[stage]);
    }
    __syncwarp();
  };

  while (uniform(w.open(a))) {
    const int n = uniform(w.n);
    const int nt = F::TILES == 2 && uniform(w.rows) > 128 ? 2 : 1;
    for (int t = 0; t < nt; ++t) mbar_wait(&sh.qfull[t], nq[t]++ & 1, &sh.abort);
    __syncwarp();
    if constexpr (F::TILES == 2) {
      wait_tile();
      qk(0, 0, at.stage, nt == 1);
      if (nt == 2) qk(1, 1, at.stage, true);
      at.next();
      for (int i = 0; i < n; ++i) {
        wait_tile();
        const uint32_t vs = at.stage;
        at.next();
        const bool more = i + 1 < n;
        const bool first = F::LONG ? i % F::HOLD == 0 : i == 0;
        pv(0, 0, vs, first, nt == 1);
        if (more) {
          wait_tile();
          qk(0, 0, at.stage, nt == 1);
        }
        if (nt == 2) {
          pv(1, 1, vs, first, true);
          if (more) qk(1, 1, at.stage, true);
        }
        if (more) at.next();
      }
    } else {
      wait_tile();
      qk(0, nb & 1, at.stage, true);
      at.next();
      for (int i = 0; i < n; ++i, ++nb) {
        if (i + 1 < n) {
          wait_tile();
          qk(0, nb + 1 & 1, at.stage, true);
          at.next();
        }
        wait_tile();
        pv(0, nb & 1, at.stage, true, true);  // (the softmax adds the tiles up)
        at.next();
      }
    }
    w.close(a);
  }
  if (elect_one()) mma_commit(&sh.done);  // nothing of ours runs when tensor memory is freed
  mbar_wait(&sh.done, 0, &sh.abort);
}

// ------------------------------------------------------------- softmax

// Query row (request, row r of the item) into its parts in shared memory;
// returns the factor from a score to the exponent of 2.
template <class F>
__device__ __forceinline__ float load_query(const Args& a, const WalkOf<F>& w, int r, bool ok, int row,
                                            int c0, int c1, uint8_t* q) {
  const int rr = w.block * F::ROWS + r;
  const int64_t q0 = ok ? static_cast<int64_t>(w.rq.start + rr / a.group) * a.q_token +
                              (w.head * a.group + rr % a.group) * a.q_head
                        : 0;
  auto eight = [&](int c, float* x) {  // elements 8c .. 8c + 7
    if (!ok) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    } else if (a.q_vec && a.q_type == LP_F32) {
      const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + q0) + 2 * c;
      const float4 u = __ldg(p), v = __ldg(p + 1);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else if (a.q_vec) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + q0) + c);
      const uint32_t h[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = a.q_type == LP_F16 ? low16<CF16>(h[i]) : low16<CBF16>(h[i]);
        x[2 * i + 1] = a.q_type == LP_F16 ? high16<CF16>(h[i]) : high16<CBF16>(h[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = load_elem(a.q, a.q_type, q0 + 8 * c + i);
    }
  };
  // Loads of 64 elements are in flight together: a row is far from the next
  // one, so each costs a trip to L2.
  constexpr int B = 8;
  // fp16 operands from other types: a power of two per row (see attn_rows.cu)
  float f = 1.0f, back = 1.0f;
  if (!F::Q::kBf16 && a.q_type != LP_F16) {
    float amax = 0.0f;
    for (int c = 0; c < F::D / 8; c += B) {
      float x[B][8];
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (c + b < F::D / 8) eight(c + b, x[b]);
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + b < F::D / 8) amax = fmaxf(amax, fabsf(x[b][i]));
    }
    const int e = row_exponent(amax);
    f = pow2(14 - e);
    back = pow2(e - 14);
  }
  // a negative scale goes into the queries, so that larger scores have larger weights
  if (a.scale_log2 < 0.0f) f = -f;
  for (int c = c0; c < c1; c += B) {
    float xs[B][8];
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (c + b < c1) eight(c + b, xs[b]);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (c + b >= c1) break;
      float* x = xs[b];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= f;
      uint8_t* dst = q + ((c + b) / 8) * kBlock + row * 128 + ((((c + b) & 7) ^ (row & 7)) << 4);
#pragma unroll
      for (int p = 0; p < F::NQ; ++p) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i] = pack16<typename F::Q>(x[2 * i], x[2 * i + 1]);
          x[2 * i] -= low16<typename F::Q>(o[i]);
          x[2 * i + 1] -= high16<typename F::Q>(o[i]);
        }
        *reinterpret_cast<uint4*>(dst + p * F::TILE) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
  // (never 0: a masked score of -inf stays one)
  return fmaxf(fabsf(a.scale_log2) * back, 1e-36f);
}

template <class F>
__device__ __forceinline__ void soft_role(const Args& a, WalkOf<F> w, Shared& sh,
                                          const Scales<F::META>* scales, uint8_t* qs) {
  using C = typename F::C;
  using P = typename F::P;
  constexpr int D = F::D;
  constexpr bool kTwo = F::TILES == 2;
  constexpr int COLS = kTwo ? 128 : 64;  // keys of a tile that this thread takes
  const int wg = threadIdx.x >> 7, row = threadIdx.x & 127;
  const int warp = threadIdx.x >> 5;
  const int tile = kTwo ? wg : 0;
  const int col0 = kTwo ? 0 : wg * 64;
  const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
  const uint32_t tm = sh.tmem + lanes;
  // output columns of this thread (D = 96 halves into 64 and 32)
  const int d0 = kTwo ? 0 : wg * (D == 64 ? 32 : 64);
  const int d1 = kTwo ? D : (wg ? D : D == 64 ? 32 : 64);
  constexpr int OB = (kTwo ? D : D == 64 ? 32 : 64) / 32;  // blocks of 32 of them
  uint32_t tiles = 0;  // key tiles so far, over all items: meta slot, S buffer
  uint32_t ns = 0, npv = 0, item = 0;

  while (w.open(a)) {
    const bool live = !kTwo || tile == 0 || w.rows > 128;  // warpgroup uniform
    const int r = tile * 128 + row;
    const bool ok = r < w.rows;
    float c = 0.0f;
    if (live) {
      constexpr int half = (D / 8 + 1) / 2;
      c = load_query<F>(a, w, r, ok, row, kTwo || wg == 0 ? 0 : half,
                        kTwo || wg == 1 ? D / 8 : half, qs + tile * F::NQ * F::TILE);
      fence_async();
      mbar_arrive(&sh.qfull[tile]);
    }

    const int rr = w.block * F::ROWS + r;
    const int pos = ok ? w.rq.base + rr / a.group : -1;
    const int lo = a.window > 0 ? pos - a.window + 1 : 0;
    // the warp's rows: all of them see keys from lo_w up to pos_w
    const int r0 = tile * 128 + (warp & 3) * 32;
    const int pos_w = w.rq.base + (w.block * F::ROWS + r0) / a.group;
    const int last_w = w.rq.base + (w.block * F::ROWS + min(r0 + 31, w.rows - 1)) / a.group;
    const int lo_w = a.window > 0 ? last_w - a.window + 1 : 0;
    const float grow = kLazy / c;
    // a warp without rows only keeps the barriers' count (its lanes' weights, and
    // so their outputs, are whatever tensor memory holds)
    const bool warp_ok = r0 < w.rows;

    float m = -INFINITY, l = 0.0f;  // reference (in scores) and sum
    float o[kTwo ? 1 : OB * 32];    // one row tile: the outputs
#pragma unroll
    for (int e = 0; e < (kTwo ? 1 : OB * 32); ++e) o[e] = 0.0f;
    // adds the last product to the outputs; both become times f
    auto gather = [&](float f) {
      if constexpr (!kTwo) {
#pragma unroll
        for (int b = 0; b < OB; ++b) {
          if (d0 + 32 * b >= d1) break;
          uint32_t u[32];
          tmem_ld32(tm + o_col(0) + d0 + 32 * b, u);
          tmem_wait_ld();
          tie(u, 32);
#pragma unroll
          for (int e = 0; e < 32; ++e)
            o[32 * b + e] = (o[32 * b + e] + __uint_as_float(u[e])) * f;
        }
      }
    };
    // The product with the weights of key tile `slot`.  A barrier must not be
    // waited for two phases early: with one row tile the weights run two
    // products ahead, so each S buffer has its own barrier.
    auto wait_pv = [&](uint32_t slot) {
      if (kTwo) mbar_wait(&sh.pvdone[tile], (npv - 1) & 1, &sh.abort);
      else mbar_wait(&sh.pvdone[slot & 1], slot >> 1 & 1, &sh.abort);
      fence_after();
    };
    // LONG: after each HOLD tiles their sum goes to the place of the item's
    // partial (which takes it at the end), with the reference that it is in units of.
    constexpr int64_t kSlot = static_cast<int64_t>(F::ROWS) * (D + 2);
    auto place = [&] { return a.partials + slot_of(blockIdx.x, w.item0, w.per) * kSlot + r; };
    // the factor that takes the held sums to the reference of now
    auto since_held = [&](const float* held) {
      const float mh = held[D * F::ROWS];
      return mh == -INFINITY ? 0.0f : ex2((mh - m) * c);
    };
    if (live) {
      for (int i = 0; i < w.n; ++i) {
        const int key0 = w.key(i) + col0;
        const uint32_t slot = tiles + i;
        const int x = kTwo ? tile : slot & 1;
        const int mm = slot % F::META;
        const uint32_t sc = tm + s_col(x) + col0;
        if (kTwo) mbar_wait(&sh.sfull[x], ns++ & 1, &sh.abort);
        else mbar_wait(&sh.sfull[x], slot >> 1 & 1, &sh.abort);
        fence_after();
        if (!warp_ok) {
          if (!kTwo) named_bar(2, kSoftThreads);
          fence_before();
          mbar_arrive(&sh.pfull[x]);
          ++npv;
          continue;
        }
        uint32_t see[COLS / 32];
        bool full = key0 + COLS - 1 <= pos_w && (key0 >= lo_w || key0 + COLS <= a.sinks);
#pragma unroll
        for (int h = 0; h < COLS / 32; ++h) {
          see[h] = sh.there[mm][col0 / 32 + h];
          full = full && see[h] == 0xffffffffu;
        }
        if (!full) {
#pragma unroll
          for (int h = 0; h < COLS / 32; ++h) {
            const int k = key0 + 32 * h;
            see[h] &= below(pos + 1 - k) & (~below(lo - k) | below(a.sinks - k));
          }
        }
        const float* sk = C::kInt8 ? &scales->k[mm][col0] : nullptr;
        const float* sv = C::kInt8 ? &scales->v[mm][col0] : nullptr;

        // ---- this thread's scores, with int8 keys' scales and the mask
        uint32_t v[COLS];
#pragma unroll
        for (int h = 0; h < COLS / 32; ++h) tmem_ld32(sc + 32 * h, v + 32 * h);
        tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < COLS / 32; ++h) tie(v + 32 * h, 32);
        if constexpr (C::kInt8) {
#pragma unroll
          for (int e = 0; e < COLS; e += 4) {
            const ulonglong2 k4 = *reinterpret_cast<const ulonglong2*>(sk + e);
            upku(mul2(pku(v[e], v[e + 1]), k4.x), v[e], v[e + 1]);
            upku(mul2(pku(v[e + 2], v[e + 3]), k4.y), v[e + 2], v[e + 3]);
          }
        }
        if (!full) {
#pragma unroll
          for (int e = 0; e < COLS; ++e) v[e] = see[e / 32] >> (e % 32) & 1u ? v[e] : 0xff800000u;
        }
        // ---- the row's maximum
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < COLS; e += 2)
          top[e / 2 % 4] = fmaxf(top[e / 2 % 4], fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
        float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if constexpr (!kTwo) {
          sh.xmax[x][wg][row] = mx;  // (the buffer's last readers are two barriers back)
          named_bar(2, kSoftThreads);
          mx = fmaxf(mx, sh.xmax[x][1 - wg][row]);
        }
        // ---- a new reference, and what there is in its units
        const bool move = mx > m + grow || (m == -INFINITY && mx != -INFINITY);
        const bool moves = i > 0 && __any_sync(0xffffffffu, move);
        float corr = 1.0f;
        if (i == 0) {
          m = mx;
        } else if (moves) {
          corr = !move ? 1.0f : m == -INFINITY ? 0.0f : ex2((m - mx) * c);
          if constexpr (kTwo) {
            wait_pv(slot - 1);
            for (int d = d0; d < d1; d += 16) {
              uint32_t u[16];  // (beside the scores in registers)
              tmem_ld16(tm + o_col(tile) + d, u);
              tmem_wait_ld();
              tie(u, 16);
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * corr);
              tmem_st16(tm + o_col(tile) + d, u);
            }
          }
          l *= corr;
          if (move) m = mx;
        }
        const float mc = m == -INFINITY ? 0.0f : m * c;
        // ---- weights, times kUp
        const float up = F::NP == 1 ? F::kUpLog : 0.0f;
        const uint64_t c2 = pk(c, c), mc2 = pk(up - mc, up - mc);
        uint64_t la = 0, lb = 0;
        constexpr int PW = kTwo ? 16 : 8;  // pairs per store (registers)
#pragma unroll
        for (int h = 0; h < COLS / (2 * PW); ++h) {
          uint32_t p[F::NP][PW];
#pragma unroll
          for (int e = 0; e < PW; ++e) {
            float y0, y1;
            uint64_t y = fma2(pku(v[2 * (PW * h + e)], v[2 * (PW * h + e) + 1]), c2, mc2);
            upk(y, y0, y1);
            y = pk(ex2(y0), ex2(y1));
            // more than one part: 2^7 as a product, which rounds nothing
            if constexpr (F::NP > 1 && F::kUp != 1.0f) y = mul2(y, pk(F::kUp, F::kUp));
            uint64_t& sum = e & 1 ? lb : la;
            sum = add2(sum, y);
            if constexpr (C::kInt8)
              y = mul2(y, *reinterpret_cast<const uint64_t*>(sv + 2 * (PW * h + e)));
#pragma unroll
            for (int q = 0; q < F::NP; ++q) {
              upk(y, y0, y1);
              if (q + 1 == F::NP) {
                p[q][e] = pack16<P>(y0, y1);
              } else if constexpr (P::kBf16) {
                // a part is the upper half of what is left, which the difference keeps exactly
                const uint32_t h0 = __float_as_uint(y0), h1 = __float_as_uint(y1);
                p[q][e] = prmt(h0, h1, 0x7632u);
                y = fma2(pku(h0 & 0xffff0000u, h1 & 0xffff0000u), pk(-1.0f, -1.0f), y);
              } else {
                p[q][e] = pack16<P>(y0, y1);
                y = fma2(pk(low16<P>(p[q][e]), high16<P>(p[q][e])), pk(-1.0f, -1.0f), y);
              }
            }
          }
#pragma unroll
          for (int q = 0; q < F::NP; ++q) {
            // the part's columns begin those of the 32 scores they come from
            const int at = 2 * PW * h;  // first score
            const uint32_t to = q < 2 ? sc + at / 32 * 32 + at % 32 / 2 + 16 * q
                                      : tm + p3_col(x) + (col0 + at) / 2;
            if constexpr (kTwo) tmem_st16(to, p[q]);
            else tmem_st8(to, p[q]);
          }
        }
        {
          float y[4];
          upk(la, y[0], y[1]);
          upk(lb, y[2], y[3]);
          l += (y[0] + y[1]) + (y[2] + y[3]);
        }
        // one row tile: the last product's sum is taken before the next one's starts
        if (!kTwo && i > 0) {
          wait_pv(slot - 1);
          if (moves) gather(corr);
          else gather(1.0f);
        }
        tmem_wait_st();
        fence_before();
        mbar_arrive(&sh.pfull[x]);
        ++npv;
        if (F::LONG && (i + 1) % F::HOLD == 0 && i + 1 < w.n) {
          wait_pv(slot);
          float* held = place();
          const float f = i + 1 > F::HOLD ? since_held(held) : 0.0f;
#pragma unroll 1
          for (int d = 0; d < D; d += 16) {
            uint32_t u[16];
            tmem_ld16(tm + o_col(tile) + d, u);
            tmem_wait_ld();
            tie(u, 16);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float* h = held + (d + e) * F::ROWS;
              *h = i + 1 > F::HOLD ? fmaf(*h, f, __uint_as_float(u[e])) : __uint_as_float(u[e]);
            }
          }
          held[D * F::ROWS] = m;
        }
      }
      wait_pv(tiles + w.n - 1);
      if (warp_ok) gather(1.0f);
    }
    tiles += w.n;
    if constexpr (!kTwo) {  // both halves' sums
      sh.xsum[wg][row] = l;
      named_bar(2, kSoftThreads);
      l += sh.xsum[1 - wg][row];
      named_bar(2, kSoftThreads);
    }
    const float f_held = F::LONG && live && warp_ok && w.n > F::HOLD ? since_held(place()) : 0.0f;
    // from here on the reference in units of log2 (sums carry kUp, like O)
    m = m == -INFINITY ? -INFINITY : m * c;

    // What clear_bad took from keys that the row sees: per block of 32 columns, those
    // with a +inf or NaN and those with a -inf or NaN.  A lane looks at one key for all
    // the warp's rows, so 32 keys cost a few trips to L2.  (Each row for itself took
    // 1.6 us a key and block: at 300000 keys in an item, all of them to be looked at,
    // longer than the other roles wait.  BY_ROW keeps that form for few tiles.)
    uint32_t up[OB] = {}, down[OB] = {};
    const int nbad = live && warp_ok ? sh.nbad[item % kPlaces] : 0;
    // All tiles are looked through where too many are noted and, with several parts of
    // the weights, where an output is not finite though the row's sum is: an infinity
    // that met the parts one by one is a NaN by now.
    bool all_tiles = nbad > kBad;
    if constexpr (F::NP > 1) {
      float f0 = 0.0f, f1 = 0.0f;
#pragma unroll
      for (int e = 0; e < OB * 32; e += 2) f0 = fmaf(o[e], 0.0f, f0), f1 = fmaf(o[e + 1], 0.0f, f1);
      all_tiles = __any_sync(0xffffffffu, warp_ok && f0 + f1 != 0.0f && finite(l)) || all_tiles;
    }
#pragma unroll 1
    for (int i = 0; i < 4 * (all_tiles ? w.n : F::BY_ROW ? 0 : nbad); ++i) {
      const int key0 = (all_tiles ? w.key(i / 4) : sh.badkey[item % kPlaces][i / 4]) + 32 * (i % 4);
      const int j = key0 + (threadIdx.x & 31);
      const int page = j < w.rq.limit ? page_of(a, w.b, j) : -1;
      uint32_t see = __ballot_sync(0xffffffffu, page >= 0) & below(pos + 1 - key0) &
                     (~below(lo - key0) | below(a.sinks - key0));
      if (!ok) see = 0;
#pragma unroll
      for (int b = 0; b < OB; ++b) {
        if (d0 + 32 * b >= d1) break;
        uint32_t u = 0, d = 0;
        if (page >= 0) bad_columns<C>(a, w.head, page, j, d0 + 32 * b, u, d);
        uint32_t keys = __ballot_sync(0xffffffffu, (u | d) != 0);
        while (keys) {
          const int s = __ffs(keys) - 1;
          keys &= keys - 1;
          const uint32_t us = __shfl_sync(0xffffffffu, u, s), ds = __shfl_sync(0xffffffffu, d, s);
          if (see >> s & 1u) up[b] |= us, down[b] |= ds;
        }
      }
    }
    // 32 columns of this CTA's outputs
    auto column_block = [&](int b, float* v) {
      if constexpr (kTwo) {
        uint32_t u[32];
        tmem_ld32(tm + o_col(tile) + 32 * b, u);
        tmem_wait_ld();
        tie(u, 32);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(u[e]);
        if (F::LONG && w.n > F::HOLD) {
          const float* held = place() + 32 * b * F::ROWS;
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = fmaf(held[e * F::ROWS], f_held, v[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = o[32 * b + e];
      }
      if (up[b] | down[b]) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const bool u = up[b] >> e & 1u, d = down[b] >> e & 1u;
          if (u || d) v[e] = u && d ? NAN : u ? INFINITY : -INFINITY;
        }
      }
      if constexpr (F::BY_ROW) {
#pragma unroll 1
        for (int i = 0; i < (all_tiles ? 0 : nbad); ++i) {
          const int key0 = sh.badkey[item % kPlaces][i];
#pragma unroll 1
          for (int j = key0; j < key0 + kKeys; ++j) {
            const int page = ok && sees(a, w.rq, pos, j) ? page_of(a, w.b, j) : -1;
            if (page < 0) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] += bad_value<C>(a, w.b, w.head, page, j, d0 + 32 * b + e);
          }
        }
      }
    };
    // ---- an item of several CTAs: leave the partial, the last one joins
    bool final = true;
    const Sharers ss = sharers(w.item0, w.un.n, w.per);
    if (ss.last > ss.first) {
      float* mine = a.partials + slot_of(blockIdx.x, w.item0, w.per) * kSlot;
      if (live && warp_ok) {
#pragma unroll
        for (int b = 0; b < OB; ++b) {
          const int d = d0 + 32 * b;
          if (d >= d1) break;
          float v[32];
          column_block(b, v);
#pragma unroll
          for (int e = 0; e < 32; ++e) mine[(d + e) * F::ROWS + r] = v[e];
        }
        if (d0 == 0) {
          mine[D * F::ROWS + r] = m;
          mine[(D + 1) * F::ROWS + r] = l;
        }
      }
      named_bar(2, kSoftThreads);
      if (threadIdx.x == 0) {
        __threadfence();  // (for the block's stores: they are before the barrier)
        const uint32_t n = static_cast<uint32_t>(ss.last - ss.first);
        sh.last = atomicInc(a.counters + ss.first, n) == n;
        __threadfence();
      }
      named_bar(2, kSoftThreads);
      final = sh.last != 0;
    }
    if (final) {
      const bool joined = ss.last > ss.first;
      float inv = 0.0f, ref = 0.0f;
      // parts' loads go out four at a time: a trip to L2 each would cost more than
      // the keys of a part
      constexpr int kTogether = 4;
      auto part_of = [&](int k) {
        return a.partials + slot_of(min(k, ss.last), w.item0, w.per) * kSlot;
      };
      if (joined && live && warp_ok) {
        m = -INFINITY, l = 0.0f;
        for (int k = ss.first; k <= ss.last; k += kTogether) {
          float pm[kTogether], pl[kTogether], mn = m;
#pragma unroll
          for (int y = 0; y < kTogether; ++y) {
            const float* part = part_of(k + y);
            pm[y] = __ldcg(part + D * F::ROWS + r);
            pl[y] = __ldcg(part + (D + 1) * F::ROWS + r);
          }
#pragma unroll
          for (int y = 0; y < kTogether; ++y) {
            if (k + y > ss.last) pm[y] = -INFINITY, pl[y] = 0.0f;
            mn = fmaxf(mn, pm[y]);
          }
          ref = mn == -INFINITY ? 0.0f : mn;
          l *= ex2(m - ref);
#pragma unroll
          for (int y = 0; y < kTogether; ++y) l = fmaf(pl[y], ex2(pm[y] - ref), l);
          m = mn;
        }
      }
      const int t = rr / a.group, g = rr % a.group;
      const int qh = w.head * a.group + g;
      const int64_t orow = static_cast<int64_t>(w.rq.start + t) * a.o_token + qh * a.o_head;
      // 32 columns of the joined parts
      auto joined_block = [&](int d, float* v) {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.0f;
        for (int k = ss.first; k <= ss.last; k += kTogether) {
          float f[kTogether], u[kTogether][32];
#pragma unroll
          for (int y = 0; y < kTogether; ++y) {
            const float* part = part_of(k + y);
            f[y] = __ldcg(part + D * F::ROWS + r);
#pragma unroll
            for (int e = 0; e < 32; ++e) u[y][e] = __ldcg(part + (d + e) * F::ROWS + r);
          }
#pragma unroll
          for (int y = 0; y < kTogether; ++y) {
            if (k + y > ss.last) break;
            const float g = ex2(f[y] - ref);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = fmaf(u[y][e], g, v[e]);
          }
        }
      };
      if (live && warp_ok) {
        inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
        for (int b = 0; b < OB; ++b) {
          const int d = d0 + 32 * b;
          if (d >= d1) break;
          float v[32];
          if (joined) joined_block(d, v);
          else column_block(b, v);
          if (ok) {
            if (a.q_vec && a.q_type == LP_F32) {
              float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.out) + orow + d);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                p[e] = make_float4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv,
                                   v[4 * e + 3] * inv);
            } else if (a.q_vec) {
              uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + orow + d);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t h[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                  const float y0 = v[8 * e + 2 * z] * inv, y1 = v[8 * e + 2 * z + 1] * inv;
                  h[z] = a.q_type == LP_F16 ? pack16<CF16>(y0, y1) : pack16<CBF16>(y0, y1);
                }
                p[e] = make_uint4(h[0], h[1], h[2], h[3]);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) store_elem(a.out, a.q_type, orow + d + e, v[e] * inv);
            }
          }
        }
        if (ok && d0 == 0 && a.lse)
          a.lse[static_cast<int64_t>(w.rq.start + t) * a.heads + qh] =
              l == 0.0f ? -INFINITY : (m + (log2f(l) - F::kUpLog)) * kLn2;
      }
    }
    // The warpgroups meet every half round of places.  (With two row tiles nothing
    // else holds the first one while the second one is in a tile's outputs: items
    // of one tile need only the first.)  So they are fewer than kPlaces / 2 items
    // apart, and the place half the round ahead, whose last item is kPlaces / 2
    // back, is behind both; the loaders, whose ring reaches five items, are not
    // there yet, and the places that they write belonged to items further back.
    if (kTwo && item % (kPlaces / 2) == kPlaces / 2 - 1) named_bar(2, kSoftThreads);
    if (threadIdx.x == 0) sh.nbad[(item + kPlaces / 2) % kPlaces] = 0;
    ++item;
    fence_before();
    w.close(a);
  }
}

template <class F>
__global__ void __launch_bounds__(kThreads, 1) k_attn_chunk(const __grid_constant__ Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ Shared sh;
  __shared__ __align__(16) std::conditional_t<F::C::kInt8, Scales<F::META>, int> scale_mem;
  Scales<F::META>* scales = reinterpret_cast<Scales<F::META>*>(&scale_mem);
  uint8_t* qs = smem_raw + ((1024u - (saddr(smem_raw) & 1023u)) & 1023u);
  uint8_t* ring = qs + F::TILES * F::NQ * F::TILE;
  const int warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (int s = 0; s < F::STAGES; ++s) {
      mbar_init(&sh.full[s], kLoadThreads);
      mbar_init(&sh.empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&sh.qfull[x], F::TILES == 2 ? 128 : kSoftThreads);
      mbar_init(&sh.sfull[x], 1);
      mbar_init(&sh.pfull[x], F::TILES == 2 ? 128 : kSoftThreads);
      mbar_init(&sh.pvdone[x], 1);
    }
    mbar_init(&sh.done, 1);
    sh.abort = 0;
    for (int x = 0; x < kPlaces; ++x) sh.nbad[x] = 0;
    mbar_fence_init();
  }
  if (warp == 12) tmem_alloc(&sh.tmem, 512);
  find_share<kKeys, F::ROWS, kItemUnits, kThreads>(a, kMinUnits, &sh.cur, sh.sums);
  fence_before();
  __syncthreads();
  fence_after();
  WalkOf<F> w;
  w.start(sh.cur);
  // a wait that runs out sets sh.abort; the roles then run to their ends
  // without waiting, so no barrier is left short and tensor memory is freed
  if (w.at < w.end) {
    if (warp < 8) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::SOFT_REGS));
      soft_role<F>(a, w, sh, scales, qs);
    } else if (warp < 12) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::LOAD_REGS));
      load_role<F>(a, w, sh, scales, ring, ring + F::STAGES * F::TILE);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::MMA_REGS));
      if (warp == 12) mma_role<F>(a, w, sh, qs, ring);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 12) {
    fence_after();
    tmem_dealloc(sh.tmem, 512);
  }
}

template <class F>
int launch(const Args& a, cudaStream_t st) {
  const DeviceInfo& di = device_info();
  static int attr_set[kMaxDevices];
  const int slot = di.ordinal % kMaxDevices;
  if (!attr_set[slot]) {
    const cudaError_t e = cudaFuncSetAttribute(
        k_attn_chunk<F>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
    if (e != cudaSuccess) return cuda_status(e);
    attr_set[slot] = 1;
  }
  k_attn_chunk<F><<<di.sm_count, kThreads, F::SMEM, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <class C, class Q, class P, int NQ, int NP, int TILES, bool LONG>
int launch_dim(const Args& a, int dim, cudaStream_t st) {
  switch (dim) {
    case 64: return launch<Cfg<C, Q, P, NQ, NP, TILES, 64, LONG>>(a, st);
    case 96: return launch<Cfg<C, Q, P, NQ, NP, TILES, 96, LONG>>(a, st);
    case 128: return launch<Cfg<C, Q, P, NQ, NP, TILES, 128, LONG>>(a, st);
    default: return LP_ERR_UNSUPPORTED;
  }
}

// One row tile.
template <class C, class Q, class P, int NQ, int NP>
int launch_one(const Args& a, int dim, cudaStream_t st) {
  return launch_dim<C, Q, P, NQ, NP, 1, false>(a, dim, st);
}
// Two, by whether the tables have room for items of more than HOLD key tiles.
template <class C, class Q, class P>
int launch_two(const Args& a, int dim, cudaStream_t st) {
  constexpr int64_t keys = int64_t{Cfg<C, Q, P, 1, 1, 2, 64, true>::HOLD} * kKeys;
  return int64_t{a.table_width} * a.page_size > keys
             ? launch_dim<C, Q, P, 1, 1, 2, true>(a, dim, st)
             : launch_dim<C, Q, P, 1, 1, 2, false>(a, dim, st);
}

}  // namespace

// Parts by what the result's type needs (its rounding is the largest error
// that is allowed to show): fp32 about 22 bits of queries and weights, fp16
// 11, bf16 8.  An int8 cache's weights carry the value scales, whose range
// over a row's keys fp16 does not span: bf16.
int launch_attn_chunk(const attn::Args& a, int cache_type, int dim, cudaStream_t st) {
  const bool f32 = a.q_type == LP_F32, f16 = a.q_type == LP_F16;
  if (cache_type == LP_F16)  // a bf16 query is exact in scaled fp16
    return f32 ? launch_one<CF16, CF16, CF16, 2, 2>(a, dim, st)
               : launch_two<CF16, CF16, CF16>(a, dim, st);
  if (cache_type == LP_BF16)
    return f32   ? launch_one<CBF16, CBF16, CBF16, 3, 3>(a, dim, st)
           : f16 ? launch_one<CBF16, CBF16, CBF16, 2, 2>(a, dim, st)
                 : launch_two<CBF16, CBF16, CBF16>(a, dim, st);
  return f32   ? launch_one<CI8, CF16, CBF16, 2, 3>(a, dim, st)
         : f16 ? launch_one<CI8, CF16, CBF16, 1, 2>(a, dim, st)
               : launch_two<CI8, CBF16, CBF16>(a, dim, st);
}

unsigned int take_error_attn_chunk() {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(v)) != cudaSuccess) return LP_ERR_CUDA;
  if (v) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_device_error, &z, sizeof(z));
  }
  return v;
}

}  // namespace lp
