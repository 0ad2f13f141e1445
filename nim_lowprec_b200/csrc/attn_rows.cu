// attn_rows.cu -- attention of a few query rows over a paged cache: single
// new tokens (decode), and every case that the chunk kernel does not take.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  j visible
//
// One pass over the keys with a running maximum and sum per row.  What bounds
// it is the cache's bytes, so the whole design serves the loads:
//   * A CTA takes up to 8 query rows of one key head (all query heads of the
//     group), so keys and values are read once for the group.
//   * Each of its 8 warps takes steps of 16 keys (32 of an int8 cache) and
//     holds keys and values in registers only: a lane's 16-byte loads are
//     already the B fragments of m16n8k16 products, for keys with the head
//     dimension permuted (the queries are permuted alike), for values after
//     byte permutes that pair two keys.  No shared memory, no barrier and no
//     shuffle stands between a load and its use; the next step's keys are in
//     flight while this step's products run.
//   * The products use 16 rows where there are 8 queries; the other 8 rows
//     carry what 16 bits drop: row i the query's high part, row i + 8 the
//     rest (hi + lo is 22 bits of fp16, 16 of bf16), and likewise for the
//     weights p.  Both parts of a row meet in the same thread.  fp32 results
//     with bf16 operands take a second product for a third part (24 bits).
//     fp16 parts are scaled: queries by a power of two per row, queries and
//     weights to at most 2^14, second parts by 2^12 more (which the row's
//     other accumulator takes back).  So they neither overflow nor fall under
//     the type's smallest numbers: weights of 2^-29 of the row's largest keep
//     22 bits.
//   * An int8 cache's scales are per (token, head): a key's multiplies its
//     score, a value's its weight, so the codes go into the products exactly.
//   * The tensor cores serve here to keep the arithmetic (8 rows: 16 fma per
//     cached byte) off the fp32 pipe; at 8 rows a tile of 128 x N tcgen05
//     rows would be 94 % padding, and the bytes bound the time either way.
#include "attn.cuh"

namespace lp {
namespace {

using namespace attn;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;
constexpr int kUnit = 32;  // keys per unit: a warp's share of a round
// A CTA takes at least this many units: fewer would cost more in the join of
// the partial results than the spread over more SMs gives back.
constexpr int kMinUnits = 4;
constexpr int kTop = 14;  // queries and weights are below 2^kTop in 16 bits
// fp16: second parts, at most 2^(kTop - 11), are held times 2^kLow
constexpr int kLow = 12;

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
  static constexpr int KS = C::kInt8 ? 32 : 16;           // keys per step
  static constexpr int NG = KS / 8;                       // n8 groups of keys
  static constexpr int E = C::kInt8 && D % 64 == 0 ? 16 : 8;  // elements per key load and lane
  static constexpr int LW = E * (C::kInt8 ? 1 : 2) / 4;   // words per key load
  static constexpr int KL = D / (4 * E);                  // key loads
  static constexpr int KW = KL * LW;                      // words per key and lane
  static constexpr int KV = KS / 4;                       // values per lane and step
  static constexpr int VE = D / 8;                        // elements per value and lane
  static constexpr int VW = VE * (C::kInt8 ? 1 : 2) / 4;
  static constexpr int STEPS = D / 16;                    // k16 steps of a score
  // first piece of a value row: VP elements per lane, then the rest
  static constexpr int VP = C::kInt8 ? (D == 128 ? 16 : 8) : 8;
};

template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t* r, const uint8_t* p) {
  if constexpr (WORDS == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    r[0] = v.x, r[1] = v.y;
  } else {
    r[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

template <class C>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (C::kBf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Head dimension that element e (0 <= e < D/8) of lane group n's value words is.
template <class C, int D>
__device__ __forceinline__ int value_dim(int n, int e) {
  using S = Shape<C, D>;
  if (S::VE <= S::VP) return n * S::VE + e;
  if (e < S::VP) return n * S::VP + e;
  if (!C::kInt8 && D == 128) return 64 + n * 8 + (e - 8);
  return 8 * S::VP + n * (S::VE - S::VP) + (e - S::VP);
}

// A step's keys (scales and presence with them), as this lane holds them.
template <class C, int D>
struct Keys {
  uint32_t w[Shape<C, D>::NG][Shape<C, D>::KW];
  float ks, vs;   // int8: scales of key (key0 + lane)
  int key0;
  int page;       // the step's page, or -2: looked up key by key
  uint32_t there; // bit i: key0 + i is loaded
};

template <class C, int D, bool T3>
__global__ void __launch_bounds__(kThreads, 1) k_attn_rows(const __grid_constant__ Args a) {
  using S = Shape<C, D>;
  constexpr int ES = C::kInt8 ? 1 : 2;
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
  extern __shared__ __align__(16) float s_o[];  // [warp][row][D]

  find_share<kUnit, kRows, kThreads>(a, kMinUnits, &cur, sums);
  if (cur.begin >= cur.end) return;
  const int64_t end = cur.end, per = cur.per_cta;
  int64_t at = cur.begin, item0 = cur.item0;
  int b = cur.b, head = cur.head, block = cur.block;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g8 = lane >> 2, c4 = lane & 3;
  const bool whole_pages = a.page_size % S::KS == 0;

  while (at < end) {
    const Request rq = request(a, b);
    const Units un = units<kUnit, kRows>(a, rq, block);
    const int u_begin = static_cast<int>(at - item0);
    const int u_end = static_cast<int>(min(static_cast<int64_t>(un.n), end - item0));
    const int rows = min(kRows, rq.n * a.group - block * kRows);

    // ---- this lane's row: query parts, position, window
    const int r = block * kRows + g8;
    const bool row_ok = g8 < rows;
    const int pos = row_ok ? rq.base + r / a.group : -1;
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    // the block's rows: keys up to p_first that are at or past lo_last are seen by all of them
    const int p_first = rq.base + block * kRows / a.group;
    const int lo_last =
        a.window > 0 ? rq.base + (block * kRows + rows - 1) / a.group - a.window + 1 : 0;

    uint32_t qa[S::STEPS][4];                 // hi, lo, hi, lo of 4 elements
    uint32_t qc[kQ3 ? S::STEPS : 1][2];        // third parts
    float cscale;
    {
      const int64_t q0 = row_ok ? (rq.start + r / a.group) * a.q_token +
                                      (head * a.group + r % a.group) * a.q_head
                                : 0;
      float x[S::STEPS][4];
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < S::STEPS; ++k) {
        const int d = (k / (S::E / 4)) * 4 * S::E + c4 * S::E + (k % (S::E / 4)) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[k][i] = row_ok ? load_elem(a.q, a.q_type, q0 + d + i) : 0.0f;
          amax = fmaxf(amax, fabsf(x[k][i]));
        }
      }
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

    float o[S::VE][4];
#pragma unroll
    for (int i = 0; i < S::VE; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // ---- steps: units u_begin + warp, + 8, ..., each of 32 / KS steps
    constexpr int SPU = kUnit / S::KS;
    const int steps = u_begin + warp < u_end ? ((u_end - u_begin - warp + kWarps - 1) / kWarps) * SPU : 0;
    auto key_of = [&](int s) {
      const int u = u_begin + warp + (s / SPU) * kWarps;
      return (u < un.sink ? u : un.first + u - un.sink) * kUnit + (s % SPU) * S::KS;
    };
    // whether some row of the block sees key j (the page aside)
    auto wanted = [&](int j) {
      return j <= un.hi && (j >= un.lo || j < a.sinks);
    };
    auto load_keys = [&](Keys<C, D>& K, int s) {
      K.key0 = key_of(s);
      int mypage = -1;  // of key0 + lane
      const int jl = K.key0 + lane;
      const bool mine = (S::KS == 32 || lane < S::KS) && wanted(jl);
      if (whole_pages) {
        int p = -1;
        if (K.key0 < rq.limit) p = page_of(a, b, K.key0);
        K.page = p;
        mypage = p;
      } else {
        K.page = -2;
        if (mine) mypage = page_of(a, b, jl);
      }
      K.there = __ballot_sync(0xffffffffu, mine && mypage >= 0);
      const int off0 = K.key0 % a.page_size;
#pragma unroll
      for (int n = 0; n < S::NG; ++n) {
        const int i = n * 8 + g8;
        int page = K.page, off = off0 + i;
        if (!whole_pages) {
          page = __shfl_sync(0xffffffffu, mypage, i);
          off = (K.key0 + i) % a.page_size;
        }
        if (K.there >> i & 1u) {
          const uint8_t* p = a.k.data + (page * a.k.page + off * a.k.token + head * a.k.head) * ES +
                             c4 * S::E * ES;
#pragma unroll
          for (int x = 0; x < S::KL; ++x) load_words<S::LW>(K.w[n] + x * S::LW, p + x * 4 * S::E * ES);
        } else {
#pragma unroll
          for (int x = 0; x < S::KW; ++x) K.w[n][x] = 0u;
        }
      }
      if constexpr (C::kInt8) {
        K.ks = 0.0f, K.vs = 0.0f;
        if (K.there >> lane & 1u) {
          const int off = whole_pages ? off0 + lane : jl % a.page_size;
          K.ks = __ldg(a.k.scales + mypage * a.k.spage + off * a.k.stoken + head * a.k.shead);
          K.vs = __ldg(a.v.scales + mypage * a.v.spage + off * a.v.stoken + head * a.v.shead);
        }
      }
      if (!whole_pages) K.page = mypage;  // per lane from here on
    };

    Keys<C, D> K;
    if (steps > 0) load_keys(K, 0);
    for (int s = 0; s < steps; ++s) {
      const int key0 = K.key0;
      const uint32_t there = K.there;
      // ---- this step's values go out
      uint32_t vw[S::KV][S::VW];
      const int off0 = key0 % a.page_size;
#pragma unroll
      for (int x = 0; x < S::KV; ++x) {
        const int i = (x >> 2) * 16 + ((x >> 1) & 1) * 8 + 2 * c4 + (x & 1);
        int page = K.page, off = off0 + i;
        if (!whole_pages) {
          page = __shfl_sync(0xffffffffu, K.page, i);
          off = (key0 + i) % a.page_size;
        }
        if (there >> i & 1u) {
          const uint8_t* p = a.v.data + (page * a.v.page + off * a.v.token + head * a.v.head) * ES;
          if constexpr (!C::kInt8 && D == 128) {
            load_words<4>(vw[x], p + g8 * 16);
            load_words<4>(vw[x] + 4, p + 128 + g8 * 16);
          } else if constexpr (S::VE > S::VP) {  // D = 96
            load_words<S::VP * ES / 4>(vw[x], p + g8 * S::VP * ES);
            load_words<(S::VE - S::VP) * ES / 4>(vw[x] + S::VP * ES / 4,
                                                 p + 8 * S::VP * ES + g8 * (S::VE - S::VP) * ES);
          } else {
            load_words<S::VW>(vw[x], p + g8 * S::VE * ES);
          }
        } else {
#pragma unroll
          for (int y = 0; y < S::VW; ++y) vw[x][y] = 0u;
        }
      }
      // ---- scores
      float sc[S::NG][4];
#pragma unroll
      for (int n = 0; n < S::NG; ++n) {
        sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < S::STEPS; ++k) {
          uint32_t b0, b1;
          if constexpr (C::kInt8) {
            const uint32_t w = K.w[n][k] ^ 0x80808080u;
            b0 = codes_f16(w, 0x4140u);
            b1 = codes_f16(w, 0x4342u);
          } else {
            b0 = K.w[n][2 * k];
            b1 = K.w[n][2 * k + 1];
          }
          mma<C>(sc[n], qa[k], b0, b1);
          if constexpr (kQ3) {
            const uint32_t q3[4] = {qc[k][0], 0u, qc[k][1], 0u};
            mma<C>(sc[n], q3, b0, b1);
          }
        }
      }
      const float ks = K.ks, vs = K.vs;
      // ---- the next step's keys go out
      if (s + 1 < steps) load_keys(K, s + 1);

      // ---- weights: log2-domain scores, masks, running maximum
      const bool all = there == (S::KS == 32 ? 0xffffffffu : 0xffffu) &&
                       key0 + S::KS - 1 <= p_first && (key0 >= lo_last || key0 + S::KS <= a.sinks);
      float t[S::NG][2];
      float mx = -INFINITY, lnew = 0.0f;
#pragma unroll
      for (int n = 0; n < S::NG; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = fmaf(sc[n][i + 2], kDown, sc[n][i]) * cscale;
          if constexpr (C::kInt8) v *= __shfl_sync(0xffffffffu, ks, n * 8 + 2 * c4 + i);
          if (!all) {
            const int x = n * 8 + 2 * c4 + i, j = key0 + x;
            if (!(there >> x & 1u) || j > pos || (j < row_lo && j >= a.sinks)) v = -INFINITY;
          }
          t[n][i] = v;
          mx = fmaxf(mx, v);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m, mx);
      const float ref = mn == -INFINITY ? 0.0f : mn;
      float w[S::NG][2];  // weights times 2^kTop
#pragma unroll
      for (int n = 0; n < S::NG; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[n][i] = ex2(t[n][i] - ref) * static_cast<float>(1 << kTop);
          lnew += w[n][i];
          if constexpr (C::kInt8) {
            const float v = __shfl_sync(0xffffffffu, vs, n * 8 + 2 * c4 + i);
            w[n][i] = w[n][i] == 0.0f ? 0.0f : w[n][i] * v;
          }
        }
      if (__any_sync(0xffffffffu, mn != m)) {
        const float corr = ex2(m - ref);
        l *= corr;
#pragma unroll
        for (int i = 0; i < S::VE; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] *= corr;
        m = mn;
      }
      l += lnew;
      // ---- outputs: p in two or three parts times the values
#pragma unroll
      for (int kk = 0; kk < S::KS / 16; ++kk) {
        uint32_t pa[4], pc[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = w[2 * kk + h][0], p1 = w[2 * kk + h][1];
          const uint32_t hi = pack16<V>(p0, p1);
          const float r0 = (p0 - low16<V>(hi)) * kUpV, r1 = (p1 - high16<V>(hi)) * kUpV;
          pa[2 * h] = hi;
          pa[2 * h + 1] = pack16<V>(r0, r1);
          if constexpr (T3)
            pc[2 * h] = pack16<V>(r0 - low16<V>(pa[2 * h + 1]), r1 - high16<V>(pa[2 * h + 1]));
        }
        const uint32_t* v0 = vw[4 * kk];
        const uint32_t* v1 = vw[4 * kk + 1];
        const uint32_t* v2 = vw[4 * kk + 2];
        const uint32_t* v3 = vw[4 * kk + 3];
        if constexpr (C::kInt8) {
#pragma unroll
          for (int x = 0; x < S::VW; ++x) {
            const uint32_t x0 = prmt(v0[x], v1[x], 0x5140u), x1 = prmt(v0[x], v1[x], 0x7362u);
            const uint32_t y0 = prmt(v2[x], v3[x], 0x5140u), y1 = prmt(v2[x], v3[x], 0x7362u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t sel = e & 1 ? 0x4342u : 0x4140u;
              const uint32_t b0 = codes_bf16(e < 2 ? x0 : x1, sel);
              const uint32_t b1 = codes_bf16(e < 2 ? y0 : y1, sel);
              mma<V>(o[4 * x + e], pa, b0, b1);
              if constexpr (T3) mma<V>(o[4 * x + e], pc, b0, b1);
            }
          }
        } else {
#pragma unroll
          for (int x = 0; x < S::VW; ++x) {
            const uint32_t b0 = prmt(v0[x], v1[x], 0x5410u), b1 = prmt(v2[x], v3[x], 0x5410u);
            const uint32_t d0 = prmt(v0[x], v1[x], 0x7632u), d1 = prmt(v2[x], v3[x], 0x7632u);
            mma<V>(o[2 * x], pa, b0, b1);
            mma<V>(o[2 * x + 1], pa, d0, d1);
            if constexpr (T3) {
              mma<V>(o[2 * x], pc, b0, b1);
              mma<V>(o[2 * x + 1], pc, d0, d1);
            }
          }
        }
      }
    }

    // ---- join the warps: row w of the block by warp w
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* so = s_o + (warp * kRows + g8) * D;
#pragma unroll
    for (int i = 0; i < S::VE; ++i) {
      so[value_dim<C, D>(2 * c4, i)] = fmaf(o[i][2], kDownV, o[i][0]);
      so[value_dim<C, D>(2 * c4 + 1, i)] = fmaf(o[i][3], kDownV, o[i][1]);
    }
    if (c4 == 0) {
      s_m[warp][g8] = m;
      s_l[warp][g8] = l;
    }
    __syncthreads();
    constexpr int DL = D / 32;
    float ro[DL], rm = -INFINITY, rl = 0.0f;
#pragma unroll
    for (int i = 0; i < DL; ++i) ro[i] = 0.0f;
    for (int w = 0; w < kWarps; ++w) rm = fmaxf(rm, s_m[w][warp]);
    for (int w = 0; w < kWarps; ++w) {
      const float mw = s_m[w][warp];
      if (mw == -INFINITY && s_l[w][warp] == 0.0f) continue;  // a warp that saw nothing
      const float f = ex2(mw - (rm == -INFINITY ? 0.0f : rm));
      rl = fmaf(s_l[w][warp], f, rl);
#pragma unroll
      for (int i = 0; i < DL; ++i)
        ro[i] = fmaf(s_o[(w * kRows + warp) * D + lane + 32 * i], f, ro[i]);
    }

    // ---- an item of several CTAs: leave the partial, the last one joins
    bool final = true;
    const Sharers sh = sharers(item0, un.n, per);
    if (sh.last > sh.first) {
      constexpr int kSlot = kRows * (D + 2);
      float* mine = a.partials + static_cast<int64_t>(slot_of(blockIdx.x, item0, per)) * kSlot;
#pragma unroll
      for (int i = 0; i < DL; ++i) mine[warp * D + lane + 32 * i] = ro[i];
      if (lane == 0) {
        mine[kRows * D + warp] = rm;
        mine[kRows * D + kRows + warp] = rl;
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        const uint32_t n = static_cast<uint32_t>(sh.last - sh.first);
        s_last = atomicInc(a.counters + sh.first, n) == n;
        __threadfence();
      }
      __syncthreads();
      final = s_last != 0;
      if (final) {
        rm = -INFINITY, rl = 0.0f;
#pragma unroll
        for (int i = 0; i < DL; ++i) ro[i] = 0.0f;
        for (int c = sh.first; c <= sh.last; ++c) {
          const float* other = a.partials + static_cast<int64_t>(slot_of(c, item0, per)) * kSlot;
          rm = fmaxf(rm, __ldcg(other + kRows * D + warp));
        }
        const float ref = rm == -INFINITY ? 0.0f : rm;
        for (int c = sh.first; c <= sh.last; ++c) {
          const float* other = a.partials + static_cast<int64_t>(slot_of(c, item0, per)) * kSlot;
          const float f = ex2(__ldcg(other + kRows * D + warp) - ref);
          rl = fmaf(__ldcg(other + kRows * D + kRows + warp), f, rl);
#pragma unroll
          for (int i = 0; i < DL; ++i)
            ro[i] = fmaf(__ldcg(other + warp * D + lane + 32 * i), f, ro[i]);
        }
      }
    }
    if (final && warp < rows) {
      const int rr = block * kRows + warp;
      const int t = rr / a.group, g = rr % a.group;
      bool good = finite(rl);
#pragma unroll
      for (int i = 0; i < DL; ++i) good = good && finite(ro[i]);
      if (__all_sync(0xffffffffu, good)) {
        const int qh = head * a.group + g;
        const int64_t orow = (rq.start + t) * a.o_token + qh * a.o_head;
#pragma unroll
        for (int i = 0; i < DL; ++i)
          store_elem(a.out, a.q_type, orow + lane + 32 * i, rl == 0.0f ? 0.0f : __fdiv_rn(ro[i], rl));
        if (a.lse && lane == 0)
          a.lse[static_cast<int64_t>(rq.start + t) * a.heads + qh] =
              rl == 0.0f ? -INFINITY : (rm + (log2f(rl) - kTop)) * kLn2;
      } else {
        exact_row<C, D>(a, b, head, t, g);
      }
    }
    __syncthreads();  // s_o, s_m, s_l are free for the next item
    at = item0 + u_end;
    if (u_end == un.n) {
      item0 += un.n;
      next_item<kRows>(a, b, head, block);
    }
  }
}

template <class C, int D, bool T3>
int launch(const Args& a, cudaStream_t st) {
  const DeviceInfo& di = device_info();
  constexpr int smem = kWarps * kRows * D * 4;
  k_attn_rows<C, D, T3><<<di.sm_count, kThreads, smem, st>>>(a);
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
