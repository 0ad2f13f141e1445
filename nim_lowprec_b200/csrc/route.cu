// route.cu -- routeExperts: each token's k experts, their weights, and the rows
// (one per token and choice) sorted by expert.
//
//   chosen = the k largest logits (ties: the lower expert), w_j = exp(l_j - l_max) / s,
//   s = the sum over the chosen, or over all experts;
//   row order: by expert, then by token;  offsets[e] = rows of experts before e
//
// Latency bounds it.  A warp holds a token's logits and takes the largest k times
// (two reductions a time).  Few tokens: one CTA does all (13 tokens, 64 experts: 4.6 us).
// More: one launch chooses and counts per CTA and expert, one turns the counts of all CTAs
// into offsets (each CTA for itself) and places its rows in order, so that no atomics
// decide an order.  8192 tokens over 128 experts 17 us: about 9 choosing, two launches'
// starts, one trip to L2 for the counts, the placing.

#include <algorithm>

#include "lp_device.cuh"
#include "lp_internal.h"
#include "rows.cuh"

namespace lp {
namespace {

constexpr int kMaxPer = kRouteExperts / 32;  // logits a lane holds
constexpr int kThreads = 512;
constexpr int kOneCta = 64;                  // tokens that one CTA takes

struct RouteArgs {
  const uint8_t* logits;
  int64_t stride;  // bytes
  int type;
  float* weights;
  int32_t *experts, *offsets, *row_token, *places;
  int32_t* counts;  // [experts][kRouteCtas]
  int64_t tokens, per;  // of a CTA
  int n, k, renorm;
};

// A key that orders as the logits do; 0 for -inf and NaN, which are never chosen.
__device__ __forceinline__ uint32_t key_of(float l) {
  if (!(l > -__int_as_float(0x7f800000))) return 0u;
  const uint32_t u = __float_as_uint(l + 0.0f);  // (-0 orders as 0)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ float logit(const RouteArgs& a, int64_t t, int e) {
  const uint8_t* p = a.logits + t * a.stride + int64_t{e} * size_of(a.type);
  if (a.type == LP_F32) return *reinterpret_cast<const float*>(p);
  const uint32_t h = *reinterpret_cast<const unsigned short*>(p);
  return a.type == LP_F16 ? h2f(h) : __uint_as_float(h << 16);
}

// One warp: the choices of token t; lane j holds the j-th expert (-1: none).
template <int PER>
__device__ __forceinline__ int choose(const RouteArgs& a, int64_t t, int lane) {
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = 32 * i + lane < a.n ? key_of(logit(a, t, 32 * i + lane)) : 0u;
  uint32_t mine = 0, top = 0;
  int id = -1;
  float all = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    if (j == 0) {
      top = best;
      if (!a.renorm && best) {
        const float m = value_of(best);
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (key[i]) all = fadd(all, key[i] == best ? 1.0f : expf(fadd(value_of(key[i]), -m)));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all = fadd(all, __shfl_xor_sync(0xffffffffu, all, o));
      }
    }
    if (best == 0u) break;
    uint32_t at = 0xffffffffu;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == best) at = 32 * i + lane;
    at = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == 32u * i + lane) key[i] = 0u;
    if (lane == j) mine = best, id = static_cast<int>(at);
  }
  float p = 0.0f;
  if (id >= 0) p = mine == top ? 1.0f : expf(fadd(value_of(mine), -value_of(top)));
  if (a.renorm) {
    all = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all = fadd(all, __shfl_xor_sync(0xffffffffu, all, o));
  }
  if (lane < a.k) {
    a.weights[t * a.k + lane] = id >= 0 ? __fdiv_rn(p, all) : 0.0f;
    a.experts[t * a.k + lane] = id;
  }
  return id;
}

// Rows of each expert before this CTA's (base) and the offsets, from the counts: a warp
// reads an expert's counts of all CTAs at once, then a scan over the experts.
__device__ __forceinline__ void scan_counts(const RouteArgs& a, int ctas, int32_t* base, int32_t* sums) {
  __shared__ int32_t wsum[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  static_assert(kRouteCtas == 128, "");
  for (int e0 = warp; e0 < a.n; e0 += 4 * (kThreads / 32)) {
    int4 c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = e0 + i * (kThreads / 32);
      c[i] = e < a.n && 4 * lane < ctas ? __ldcg(reinterpret_cast<const int4*>(a.counts + int64_t{e} * kRouteCtas) + lane)
                                        : make_int4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = e0 + i * (kThreads / 32), v[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
      int before = 0, total = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (4 * lane + j < static_cast<int>(blockIdx.x)) before += v[j];
        if (4 * lane + j < ctas) total += v[j];
      }
      before = __reduce_add_sync(0xffffffffu, before);
      total = __reduce_add_sync(0xffffffffu, total);
      if (lane == 0 && e < a.n) {
        base[e] = before;
        sums[e] = total;
      }
    }
  }
  __syncthreads();
  int carry = 0;
  for (int e0 = 0; e0 < a.n; e0 += kThreads) {
    const int e = e0 + threadIdx.x, total = e < a.n ? sums[e] : 0;
    int inc = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int ahead = carry;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) ahead += wsum[w];
      carry += wsum[w];
    }
    if (e < a.n) {
      base[e] += ahead + inc - total;
      if (blockIdx.x == 0) a.offsets[e + 1] = ahead + inc;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[0] = 0;
}

// The rows of tokens [t0, t1) in order, a pair a thread: its place is the expert's base,
// plus the pairs of that expert in warps before, plus those in lanes before.
__device__ __forceinline__ void place(const RouteArgs& a, int64_t t0, int64_t t1, int32_t* base, int32_t* sums,
                                      uint16_t* ahead) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t end = t1 * a.k;
  for (int64_t p0 = t0 * a.k; p0 < end; p0 += kThreads) {
    for (int i = threadIdx.x; i < (kThreads / 32) * a.n; i += kThreads) ahead[i] = 0;
    const int64_t p = p0 + threadIdx.x;
    const int id = p < end ? a.experts[p] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const int rank = __popc(same & ((1u << lane) - 1));
    __syncthreads();
    if (id >= 0 && rank == 0) ahead[warp * a.n + id] = static_cast<uint16_t>(__popc(same));
    __syncthreads();
    for (int e = threadIdx.x; e < a.n; e += kThreads) {
      int run = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        const int c = ahead[w * a.n + e];
        ahead[w * a.n + e] = static_cast<uint16_t>(run);
        run += c;
      }
      sums[e] = run;
    }
    __syncthreads();
    if (p < end) {
      const int at = id >= 0 ? base[id] + ahead[warp * a.n + id] + rank : -1;
      a.places[p] = at;
      if (id >= 0) a.row_token[at] = static_cast<int32_t>(p / a.k);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.n; e += kThreads) base[e] += sums[e];
  }
}

template <int PER, bool ONE>
__global__ void __launch_bounds__(kThreads) k_route_choose(const RouteArgs a) {
  __shared__ int32_t hist[kRouteExperts];
  __shared__ int32_t sums[ONE ? kRouteExperts : 1];
  __shared__ uint16_t ahead[ONE ? kThreads / 32 * kRouteExperts : 1];
  for (int e = threadIdx.x; e < a.n; e += kThreads) hist[e] = 0;
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.tokens);
  const int lane = threadIdx.x & 31;
  for (int64_t t = t0 + (threadIdx.x >> 5); t < t1; t += kThreads / 32) {
    const int id = choose<PER>(a, t, lane);
    if (id >= 0) atomicAdd(&hist[id], 1);  // (a count: its order does not matter)
  }
  // (the launch that places the rows, which waits before it reads anything)
  if constexpr (!ONE) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();
  for (int e = threadIdx.x; e < a.n; e += kThreads) a.counts[int64_t{e} * kRouteCtas + blockIdx.x] = hist[e];
  if constexpr (ONE) {
    __syncthreads();
    scan_counts(a, 1, hist, sums);
    place(a, t0, t1, hist, sums, ahead);
  }
}

__global__ void __launch_bounds__(kThreads) k_route_place(const RouteArgs a) {
  __shared__ int32_t base[kRouteExperts], sums[kRouteExperts];
  __shared__ uint16_t ahead[kThreads / 32 * kRouteExperts];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  scan_counts(a, gridDim.x, base, sums);
  const int64_t t0 = blockIdx.x * a.per, t1 = min(t0 + a.per, a.tokens);
  place(a, t0, t1, base, sums, ahead);
}

template <int PER>
int launch_route_per(const RouteArgs& a, int ctas, cudaStream_t st) {
  if (ctas <= 1) return launch_early(k_route_choose<PER, true>, 1, kThreads, st, a);
  if (const int e = launch_early(k_route_choose<PER, false>, ctas, kThreads, st, a)) return e;
  return launch_early(k_route_place, ctas, kThreads, st, a);
}

}  // namespace

int launch_route(const lp_matrix& logits, float* weights, int32_t* experts, int32_t* offsets, int32_t* row_token,
                 int32_t* places, int64_t k, int renorm, int32_t* counts, cudaStream_t st) {
  RouteArgs a{static_cast<const uint8_t*>(logits.data), logits.stride * size_of(logits.dtype), logits.dtype,
              weights, experts, offsets, row_token, places, counts, logits.rows, 0,
              static_cast<int>(logits.cols), static_cast<int>(k), renorm};
  int ctas = 1;
  if (a.tokens > kOneCta) {
    // a multiple of the CTA's 16 warps each, on as many CTAs as the counts have room for
    a.per = (a.tokens + kRouteCtas - 1) / kRouteCtas;
    a.per = (a.per + 15) / 16 * 16;
    ctas = static_cast<int>((a.tokens + a.per - 1) / a.per);
  } else {
    a.per = a.tokens;
  }
  if (a.n <= 32) return launch_route_per<1>(a, ctas, st);
  if (a.n <= 64) return launch_route_per<2>(a, ctas, st);
  if (a.n <= 128) return launch_route_per<4>(a, ctas, st);
  if (a.n <= 256) return launch_route_per<8>(a, ctas, st);
  return launch_route_per<kMaxPer>(a, ctas, st);
}

}  // namespace lp
