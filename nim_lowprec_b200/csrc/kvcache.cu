// kvcache.cu -- the paged key/value cache: page tables and slot maps from
// request lengths (assignPages), rows written to slots (storeKV) and read
// back (loadKV).
#include <algorithm>

#include "lp_device.cuh"
#include "lp_internal.h"
#include "rows.cuh"

namespace lp {
namespace {

// --------------------------------------------------------- assignPages
//
//   need_b  = pages of [ctx_b, ctx_b + new_b) that ctx_b does not have yet
//   first_b = sum_{a < b} need_a,  qstart_b = sum_{a < b} new_a
//
// A few KB of lengths in, up to MBs of tables and maps out: latency bound, so
// one launch with no pass between CTAs.  Every CTA scans all the lengths by
// itself (1500 requests: two per thread) and keeps the sums at each thread's
// run of requests in shared memory; then requests go to warps for the table's
// new entries, and tokens to threads, which find their request by a binary
// search of those sums.  A token on a new page takes its page from the free
// list itself, so nothing waits for the table's writes.  7 requests 4.4 us, 1500
// requests with 190000 new tokens 10.6 us (a launch with one trip to L2 is 2.5).
constexpr int kAssignThreads = 512;

struct AssignArgs {
  const int32_t *ctx, *add;
  int requests, page_size;
  const int32_t* free_pages;
  int64_t free_len;
  const int32_t* free_head;
  int32_t* table;
  int64_t table_stride;
  int table_width;
  int32_t *qstart, *seqlens;
  int64_t* slots;
  int32_t* positions;
  int64_t tokens;
  int32_t* free_head_out;
};

struct Need {
  int ctx, add, first, count;  // first new table entry, number of them
};

__device__ __forceinline__ Need need_of(const AssignArgs& a, int b) {
  Need n;
  n.ctx = max(__ldg(a.ctx + b), 0);
  n.add = max(__ldg(a.add + b), 0);
  const int64_t ps = a.page_size;
  const int64_t w = a.table_width;
  const int64_t p0 = min((n.ctx + ps - 1) / ps, w);
  const int64_t p1 = min((static_cast<int64_t>(n.ctx) + n.add + ps - 1) / ps, w);
  n.first = static_cast<int>(p0);
  n.count = static_cast<int>(p1 - p0);
  return n;
}

__global__ void __launch_bounds__(kAssignThreads) k_assign_pages(const AssignArgs a) {
  __shared__ int64_t s_tok[kAssignThreads + 1], s_page[kAssignThreads + 1];
  __shared__ int64_t w_tok[kAssignThreads / 32], w_page[kAssignThreads / 32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int run = (a.requests + kAssignThreads - 1) / kAssignThreads;
  const int64_t head = max(__ldg(a.free_head), 0);

  int64_t tok = 0, page = 0;
  for (int b = min(t * run, a.requests), e = min(b + run, a.requests); b < e; ++b) {
    const Need n = need_of(a, b);
    tok += n.add;
    page += n.count;
  }
  int64_t itok = tok, ipage = page;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, itok, o);
    const int64_t z = __shfl_up_sync(0xffffffffu, ipage, o);
    if (lane >= o) itok += y, ipage += z;
  }
  if (lane == 31) w_tok[warp] = itok, w_page[warp] = ipage;
  __syncthreads();
  for (int w = 0; w < warp; ++w) itok += w_tok[w], ipage += w_page[w];
  if (t == 0) s_tok[0] = 0, s_page[0] = 0;
  s_tok[t + 1] = itok;
  s_page[t + 1] = ipage;
  __syncthreads();
  const int64_t total = s_tok[kAssignThreads];

  // sums at request b: those of its thread's run, plus the requests before b in it
  auto sums_at = [&](int b, int64_t& st, int64_t& sp) {
    const int r = b / run;
    st = s_tok[r];
    sp = s_page[r];
    for (int x = r * run; x < b; ++x) {
      const Need n = need_of(a, x);
      st += n.add;
      sp += n.count;
    }
  };
  auto page_at = [&](int64_t i) {  // entry i of the free list
    return i < a.free_len ? __ldg(a.free_pages + i) : -1;
  };

  // ---- table entries, starts and lengths: one request per warp
  const int warps = gridDim.x * (kAssignThreads / 32);
  for (int b = blockIdx.x * (kAssignThreads / 32) + warp; b < a.requests; b += warps) {
    int64_t st, sp;
    sums_at(b, st, sp);
    const Need n = need_of(a, b);
    for (int i = lane; i < n.count; i += 32)
      a.table[b * a.table_stride + n.first + i] = page_at(head + sp + i);
    if (lane == 0) {
      a.qstart[b] = static_cast<int32_t>(min(st, static_cast<int64_t>(INT32_MAX)));
      a.seqlens[b] = static_cast<int32_t>(
          min(static_cast<int64_t>(n.ctx) + n.add, static_cast<int64_t>(INT32_MAX)));
    }
  }
  if (blockIdx.x == 0 && t == 0) {
    a.qstart[a.requests] = static_cast<int32_t>(min(total, static_cast<int64_t>(INT32_MAX)));
    a.free_head_out[0] = static_cast<int32_t>(
        min(head + s_page[kAssignThreads], a.free_len));
  }

  // ---- slots and positions: one token per thread
  const int64_t threads = static_cast<int64_t>(gridDim.x) * kAssignThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kAssignThreads + t; i < a.tokens;
       i += threads) {
    int64_t slot = -1;
    int pos = -1;
    if (i < total) {
      int lo = 0, hi = kAssignThreads;  // s_tok[lo] <= i < s_tok[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_tok[mid] <= i) lo = mid;
        else hi = mid;
      }
      int b = lo * run;
      int64_t st = s_tok[lo], sp = s_page[lo];
      Need n = need_of(a, b);
      while (i >= st + n.add) {
        st += n.add;
        sp += n.count;
        n = need_of(a, ++b);
      }
      const int64_t p = n.ctx + (i - st);
      pos = static_cast<int>(min(p, static_cast<int64_t>(INT32_MAX)));
      const int64_t at = p / a.page_size;
      if (at < a.table_width) {
        const int pg = at < n.first ? a.table[b * a.table_stride + at]
                                    : page_at(head + sp + (at - n.first));
        if (pg >= 0) slot = static_cast<int64_t>(pg) * a.page_size + p % a.page_size;
      }
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = pos;
  }
}

// --------------------------------------------------- storeKV and loadKV
//
// One group of lanes per (token, head), 8 elements per lane (16 into an int8
// cache, whose arithmetic would otherwise bound it; 4 into fp32), the key's and the value's
// row together.  Each is read and written once, which bounds 16-bit caches (8191 x
// 8 fp32 rows of 128: store 15.6 us, 6.4 TB/s, load 17.0).  int8 (4096 x 32 bf16
// rows, store 31 us where the bytes take 15; load to fp32 35 of 26): 19 instructions
// a value, 63 % of the issue slots with 39 % of the warps (registers), and 64 % of
// them with loads that wait for slot, page and scale in turn.
// int8 rows take calibrateSymmetric's scale over the row (the largest
// magnitude / 127, 1 for a zero row; quant.nim:95-110) and quantizeBatch's
// code (divide, round half away from zero; quant.nim:48-60), by the same
// IEEE operations, so the cache's bytes equal the two calls'.
constexpr int kRowThreads = 256;

// Numbers of tokens, heads and pages, and the strides (checked at the call),
// fit 32 bits, so an offset is a sum of 32 x 32 -> 64 bit products.
__device__ __forceinline__ int64_t wide(uint32_t a, uint32_t b) {
  return static_cast<int64_t>(static_cast<uint64_t>(a) * b);
}
struct RowPtr {
  const uint8_t* p;
  uint32_t token, head;  // in elements
  __device__ __forceinline__ int64_t at(uint32_t t, uint32_t h) const {
    return wide(t, token) + wide(h, head);
  }
};
struct PoolPtr {
  uint8_t* p;
  float* scales;
  uint32_t page, token, head;     // in pieces of 16 bytes
  uint32_t spage, stoken, shead;  // in elements
  template <int T>
  __device__ __forceinline__ uint8_t* at(uint32_t pg, uint32_t off, uint32_t h) const {
    return p + ((wide(pg, page) + wide(off, token) + wide(h, head)) << 4);
  }
  __device__ __forceinline__ float* scale(uint32_t pg, uint32_t off, uint32_t h) const {
    return scales + wide(pg, spage) + wide(off, stoken) + wide(h, shead);
  }
};
struct RowsArgs {
  RowPtr k, v;      // storeKV reads, loadKV writes
  PoolPtr kc, vc;
  const int64_t* slots;
  int64_t items;    // tokens * heads
  int heads, dim, page_size, page_shift;
  int64_t slots_end;  // pages * page_size
};

__device__ __forceinline__ void load16_i8(float* x, const uint8_t* p) {
  const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    x[i] = static_cast<float>(static_cast<int8_t>((w[i >> 2] >> (8 * (i & 3))) & 255u));
}

// N elements of a cache row, N * size bytes aligned to themselves, 16 at most.
template <int T, int N>
__device__ __forceinline__ void load_cache(float* x, const uint8_t* p) {
  if constexpr (T == LP_I8 && N == 16) {
    load16_i8(x, p);
  } else if constexpr (T != LP_I8 && N == 8) {
    load8<T, true>(x, p);
  } else {
    constexpr int B = N * (T == LP_I8 ? 1 : 2);
    static_assert(B == 4 || B == 8, "");
    uint32_t w[2];
    if constexpr (B == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = u.x, w[1] = u.y;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (T == LP_I8)
        x[i] = static_cast<float>(static_cast<int8_t>((w[i >> 2] >> (8 * (i & 3))) & 255u));
      else if constexpr (T == LP_F16)
        x[i] = h2f(w[i >> 1] >> (16 * (i & 1)) & 0xffffu);
      else
        x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
  }
}

// A lane's N elements of a row, of which L lanes hold one.
template <int L, int N>
__device__ __forceinline__ void store_i8(uint8_t* p, float* scale, const float* x, bool active,
                                         bool write_scale) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float s = m == 0.0f ? 1.0f : __fdiv_rn(m, 127.0f);
  uint32_t w[N / 4];
  codes<N>(w, x, s);
  if (active) {
    if constexpr (N == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
  if (write_scale) *scale = s;
}

// X: type of the rows, T: type of the cache, L: lanes per row of N elements each
template <int X, int T, int L, int N, bool VEC, bool STORE>
__global__ void __launch_bounds__(kRowThreads) k_rows(const RowsArgs a) {
  const int sub = threadIdx.x & (L - 1);
  const bool lane_in = sub * N < a.dim;
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (kRowThreads / L);
  const int64_t g0 = (static_cast<int64_t>(blockIdx.x) * kRowThreads + threadIdx.x) / L;
  // whole warps run the same number of rounds: the row's maximum meets by shuffles
  const int64_t w0 = g0 - ((threadIdx.x & 31) / L);
  for (int64_t r = 0; w0 + r < a.items; r += groups) {
    const int64_t i = g0 + r;
    const bool in = i < a.items;
    // (64-bit divisions only where 32 bits do not hold the number)
    const uint32_t t = !in ? 0
                       : a.items >> 32 ? static_cast<uint32_t>(i / a.heads)
                                       : static_cast<uint32_t>(i) / static_cast<uint32_t>(a.heads);
    const uint32_t h = in ? static_cast<uint32_t>(i - static_cast<int64_t>(t) * a.heads) : 0;
    const int64_t slot = in ? __ldg(a.slots + t) : -1;
    const int64_t kr = a.k.at(t, h) + sub * N, vr = a.v.at(t, h) + sub * N;
    float x[N] = {}, y[N] = {};
    if constexpr (STORE) {  // the rows do not wait for the slots
      if (in && lane_in) {
#pragma unroll
        for (int b = 0; b < N; b += 8) {
          load8<X, VEC>(x + b, a.k.p + (kr + b) * size_of(X));
          load8<X, VEC>(y + b, a.v.p + (vr + b) * size_of(X));
        }
      }
    }
    const bool there = slot >= 0 && slot < a.slots_end;
    const bool on = in && lane_in && there;
    const int64_t sl = there ? slot : 0;
    const uint32_t page = static_cast<uint32_t>(a.page_shift >= 0 ? sl >> a.page_shift : sl / a.page_size);
    const uint32_t off = static_cast<uint32_t>(sl - static_cast<int64_t>(page) * a.page_size);
    uint8_t* kp = a.kc.template at<T>(page, off, h) + sub * (N * size_of(T));
    uint8_t* vp = a.vc.template at<T>(page, off, h) + sub * (N * size_of(T));
    if constexpr (STORE) {
      if constexpr (T == LP_I8) {
        store_i8<L, N>(kp, a.kc.scale(page, off, h), x, on, on && sub == 0);
        store_i8<L, N>(vp, a.vc.scale(page, off, h), y, on, on && sub == 0);
      } else if (on) {
        store8<T, true>(kp, x);
        store8<T, true>(vp, y);
      }
    } else {
      if (on) {
        load_cache<T, N>(x, kp);
        load_cache<T, N>(y, vp);
        if constexpr (T == LP_I8) {
          const float sk = __ldg(a.kc.scale(page, off, h)), sv = __ldg(a.vc.scale(page, off, h));
#pragma unroll
          for (int j = 0; j < N; ++j) x[j] = fmul(x[j], sk), y[j] = fmul(y[j], sv);
        }
      }
      if (in && lane_in) {  // no row at this slot: zeros
        uint8_t* ko = const_cast<uint8_t*>(a.k.p) + kr * size_of(X);
        uint8_t* vo = const_cast<uint8_t*>(a.v.p) + vr * size_of(X);
        if constexpr (N == 4) {  // (fp32 rows)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            if constexpr (VEC) break;
            reinterpret_cast<float*>(ko)[b] = x[b];
            reinterpret_cast<float*>(vo)[b] = y[b];
          }
          if constexpr (VEC) {
            *reinterpret_cast<float4*>(ko) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(vo) = make_float4(y[0], y[1], y[2], y[3]);
          }
        } else {
#pragma unroll
          for (int b = 0; b < N; b += 8) {
            store8<X, VEC>(ko + b * size_of(X), x + b);
            store8<X, VEC>(vo + b * size_of(X), y + b);
          }
        }
      }
    }
  }
}

template <int X, int T, int L, int N, bool STORE>
int launch_rows_l(const RowsArgs& a, bool vec, cudaStream_t st) {
  const int64_t blocks = (a.items + kRowThreads / L - 1) / (kRowThreads / L);
  const int grid = static_cast<int>(std::min<int64_t>(blocks, device_info().sm_count * 32ll));
  if (vec) k_rows<X, T, L, N, true, STORE><<<grid, kRowThreads, 0, st>>>(a);
  else k_rows<X, T, L, N, false, STORE><<<grid, kRowThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

template <int X, int T, bool STORE>
int launch_rows_t(const RowsArgs& a, bool vec, cudaStream_t st) {
  // fp32 rows out: 4 elements, so that a warp writes whole lines
  constexpr int N = STORE ? (T == LP_I8 ? 16 : 8) : X == LP_F32 ? 4 : 8;
  if constexpr (N == 16) {
    // Few rows: 8 elements a lane, whose chain is shorter (61 x 8 rows of 128:
    // 3.4 us against 4.6; 4096 x 32: 41 against 31).
    if (a.items * a.dim <= int64_t{device_info().sm_count} * kRowThreads * 8) {
      if (a.dim <= 64) return launch_rows_l<X, T, 8, 8, STORE>(a, vec, st);
      if (a.dim <= 128) return launch_rows_l<X, T, 16, 8, STORE>(a, vec, st);
      return launch_rows_l<X, T, 32, 8, STORE>(a, vec, st);
    }
  }
  if (a.dim <= 64) return launch_rows_l<X, T, 64 / N, N, STORE>(a, vec, st);
  if (a.dim <= 128) return launch_rows_l<X, T, 128 / N, N, STORE>(a, vec, st);
  constexpr int W = N == 4 ? 8 : N;  // (a row's lanes are in one warp)
  return launch_rows_l<X, T, 256 / W, W, STORE>(a, vec, st);
}

template <int X, bool STORE>
int launch_rows_x(const RowsArgs& a, int cache_type, bool vec, cudaStream_t st) {
  if (cache_type == LP_F16) return launch_rows_t<X, LP_F16, STORE>(a, vec, st);
  if (cache_type == LP_BF16) return launch_rows_t<X, LP_BF16, STORE>(a, vec, st);
  return launch_rows_t<X, LP_I8, STORE>(a, vec, st);
}

template <bool STORE>
int launch_rows(const RowsArgs& a, int type, int cache_type, bool vec, cudaStream_t st) {
  if (type == LP_F32) return launch_rows_x<LP_F32, STORE>(a, cache_type, vec, st);
  if (type == LP_F16) return launch_rows_x<LP_F16, STORE>(a, cache_type, vec, st);
  return launch_rows_x<LP_BF16, STORE>(a, cache_type, vec, st);
}

RowsArgs rows_args(const lp_kv_cache& c, const lp_rows& k, const lp_rows& v, const int64_t* slots) {
  RowsArgs a;
  auto row = [](const lp_rows& r) {
    return RowPtr{static_cast<const uint8_t*>(r.data), static_cast<uint32_t>(r.token_stride),
                  static_cast<uint32_t>(r.head_stride)};
  };
  auto pool = [&](void* p, float* scales, const int64_t* s, const int64_t* ss) {
    const int64_t es = c.dtype == LP_I8 ? 1 : 2;
    PoolPtr o{static_cast<uint8_t*>(p), scales, 0, 0, 0, 0, 0, 0};
    o.page = static_cast<uint32_t>(s[0] * es / 16);
    o.token = static_cast<uint32_t>(s[1] * es / 16);
    o.head = static_cast<uint32_t>(s[2] * es / 16);
    o.spage = static_cast<uint32_t>(ss[0]);
    o.stoken = static_cast<uint32_t>(ss[1]);
    o.shead = static_cast<uint32_t>(ss[2]);
    return o;
  };
  a.k = row(k);
  a.v = row(v);
  a.kc = pool(c.k, c.k_scales, c.k_strides, c.k_scale_strides);
  a.vc = pool(c.v, c.v_scales, c.v_strides, c.v_scale_strides);
  a.slots = slots;
  a.items = k.tokens * c.kv_heads;
  a.heads = static_cast<int>(c.kv_heads);
  a.dim = c.head_dim;
  a.page_size = static_cast<int>(c.page_size);
  a.page_shift = -1;  // log2 of the page size, where it is a power of two
  for (int i = 0; i < 31; ++i)
    if (c.page_size == int64_t{1} << i) a.page_shift = i;
  a.slots_end = c.pages * c.page_size;
  return a;
}

}  // namespace

int launch_store_kv(const lp_kv_cache& c, const lp_rows& k, const lp_rows& v, const int64_t* slots,
                    bool vec, cudaStream_t st) {
  return launch_rows<true>(rows_args(c, k, v, slots), k.dtype, c.dtype, vec, st);
}

int launch_load_kv(const lp_kv_cache& c, const int64_t* slots, const lp_rows& k, const lp_rows& v,
                   bool vec, cudaStream_t st) {
  return launch_rows<false>(rows_args(c, k, v, slots), k.dtype, c.dtype, vec, st);
}

int launch_assign_pages(const int32_t* ctx, const int32_t* add, int64_t requests,
                        int64_t page_size, const int32_t* free_pages, int64_t free_len,
                        const int32_t* free_head, int32_t* table, int64_t table_stride,
                        int64_t table_width, int32_t* qstart, int32_t* seqlens, int64_t* slots,
                        int64_t tokens, int32_t* positions, int32_t* free_head_out,
                        cudaStream_t st) {
  AssignArgs a{ctx,       add,     static_cast<int>(requests), static_cast<int>(page_size),
               free_pages, free_len, free_head,                table,
               table_stride, static_cast<int>(table_width),    qstart,
               seqlens,   slots,   positions,                  tokens,
               free_head_out};
  const int64_t want = std::max((tokens + kAssignThreads - 1) / kAssignThreads,
                                (requests + kAssignThreads / 32 - 1) / (kAssignThreads / 32));
  const int grid = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(want, device_info().sm_count * 3ll)));
  k_assign_pages<<<grid, kAssignThreads, 0, st>>>(a);
  return cuda_status(cudaGetLastError());
}

}  // namespace lp
