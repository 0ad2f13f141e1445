// rows8.cu -- 8-bit rows: their codec (quantizeRows, dequantizeRows), the
// root-mean-square norm that makes them from a residual stream (addRmsNorm), and
// the sum of a token's experts' rows (combineExperts).
//
// Rows are MXFP8 (e4m3 codes, one E8M0 byte per 32 elements) or int8 (one fp32
// scale per group).  All four stream: bytes bound them for many rows and the
// launch with its chain of loads for few.
#include <algorithm>

#include "lp_device.cuh"
#include "lp_internal.h"
#include "rows.cuh"

namespace lp {
namespace {

// Launched early (launch_early), a kernel waits for the one before it.  It does not let the
// next one begin early: what it writes may be the next GEMV's weights, which that reads
// before its own wait.
__device__ __forceinline__ void begin() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct Mat {  // rows of a matrix; p may be null
  uint8_t* p;
  int64_t stride;  // bytes
  int type;
};
struct Rows8 {
  uint8_t* codes;
  uint8_t* scales;
  int64_t code_stride, scale_stride;  // bytes
  int int8;                           // else MXFP8
  int lanes;                          // of 8 elements, in a group
  int group_shift;                    // log2 of the group
};

// A lane's 8 elements of a row as codes, its group's scale by the group's first
// lane.  The `lanes` lanes of a group are in one warp; `on`: store.
template <bool VEC>
__device__ __forceinline__ void put_rows8(const Rows8& q, int64_t row, int unit, const float* x, bool on) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(x[i]));
  for (int o = 1; o < q.lanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  uint32_t w[2];
  uint8_t* sp = q.scales + row * q.scale_stride;
  const bool first = on && (unit & (q.lanes - 1)) == 0;
  if (q.int8) {
    const float s = m == 0.0f ? 1.0f : __fdiv_rn(m, 127.0f);
    codes<8>(w, x, s);
    if (first) reinterpret_cast<float*>(sp)[(unit * 8) >> q.group_shift] = s;
  } else {
    const uint32_t c = mx8_scale(m);
    const float inv = mx8_inverse(c);
    w[0] = e4m3x4(x, inv);
    w[1] = e4m3x4(x + 4, inv);
    if (first) sp[unit >> 2] = static_cast<uint8_t>(c);
  }
  if (!on) return;
  uint8_t* p = q.codes + row * q.code_stride + unit * 8;
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
  }
}

// ---------------------------------------------------------- addRmsNorm
//
//   r = x + residual, n = r / sqrt(mean r^2 + eps) * weight;  total = r, y = n,
//   codes = n in 8 bits
//
// One pass: a row's elements stay in its CTA's registers (C pieces of 8 a thread)
// between the sum of squares and the scaling.  r is rounded to the stream's type
// before it is squared, so that the norm is that of what the stream carries on.
struct NormArgs {
  Mat x, res, total, y;
  const uint8_t* weight;
  Rows8 q;
  int64_t rows;
  int cols, wtype;
  float eps;
};

template <int C>
__global__ void __launch_bounds__(1024) k_norm(const NormArgs a) {
  begin();
  __shared__ float part[2][32];
  const int units = (a.cols + 7) / 8, warps = blockDim.x >> 5;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    float v[C][8];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int u = c * blockDim.x + threadIdx.x, n = a.cols - 8 * u;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = 0.0f;
      if (u >= units) continue;
      load8_of<false>(v[c], a.x.p + row * a.x.stride + int64_t{8} * u * size_of(a.x.type), a.x.type, n);
      if (a.res.p) {
        float r[8];
        load8_of<false>(r, a.res.p + row * a.res.stride + int64_t{8} * u * size_of(a.res.type), a.res.type, n);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = rounded(fadd(v[c][i], r[i]), a.res.type);
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __fmaf_rn(v[c][i], v[c][i], sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum = fadd(sum, __shfl_xor_sync(0xffffffffu, sum, o));
    if ((threadIdx.x & 31) == 0) part[flip][threadIdx.x >> 5] = sum;
    __syncthreads();  // (two sets of parts: the next row's writes meet no reads)
    float t = (threadIdx.x & 31) < warps ? part[flip][threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = fadd(t, __shfl_xor_sync(0xffffffffu, t, o));
    const float rs = __fdiv_rn(1.0f, __fsqrt_rn(fadd(__fdiv_rn(t, static_cast<float>(a.cols)), a.eps)));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int u = c * blockDim.x + threadIdx.x, n = a.cols - 8 * u;
      const bool on = u < units;
      float w[8] = {}, z[8];
      if (on) {
        if (a.total.p)
          store8_of<false>(a.total.p + row * a.total.stride + int64_t{8} * u * size_of(a.total.type), v[c],
                         a.total.type, n);
        load8_of<false>(w, a.weight + int64_t{8} * u * size_of(a.wtype), a.wtype, n);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = fmul(fmul(v[c][i], rs), w[i]);
      if (on && a.y.p)
        store8_of<false>(a.y.p + row * a.y.stride + int64_t{8} * u * size_of(a.y.type), z, a.y.type, n);
      if (a.q.codes) put_rows8<false>(a.q, row, u, z, on);
    }
  }
}

// The same for aligned rows whose x has type X and whose stream has type R: every load is
// issued before the first is used (8192 rows of 4096 in bf16, 303 MB: 53 us; with a use behind each load, as above, 66).
template <int X, int R, int C>
__global__ void __launch_bounds__(1024) k_norm_vec(const NormArgs a) {
  begin();
  __shared__ float part[2][32];
  const int units = a.cols / 8, warps = blockDim.x >> 5;
  const bool add = a.res.p != nullptr;
  int flip = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, flip ^= 1) {
    Raw8<X> x[C];
    Raw8<R> r[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int u = c * blockDim.x + threadIdx.x;
      x[c].zero();
      r[c].zero();
      if (u >= units) continue;
      x[c].load(a.x.p + row * a.x.stride + int64_t{8} * u * size_of(X));
      if (add) r[c].load(a.res.p + row * a.res.stride + int64_t{8} * u * size_of(R));
    }
    float v[C][8];
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float y[8];
      x[c].get(v[c]);
      if (add) {
        r[c].get(y);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] = rounded(fadd(v[c][i], y[i]), R);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __fmaf_rn(v[c][i], v[c][i], sum);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int u = c * blockDim.x + threadIdx.x;
      if (a.total.p && u < units) store8<R, true>(a.total.p + row * a.total.stride + int64_t{8} * u * size_of(R), v[c]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum = fadd(sum, __shfl_xor_sync(0xffffffffu, sum, o));
    if ((threadIdx.x & 31) == 0) part[flip][threadIdx.x >> 5] = sum;
    __syncthreads();
    float t = (threadIdx.x & 31) < warps ? part[flip][threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = fadd(t, __shfl_xor_sync(0xffffffffu, t, o));
    const float rs = __fdiv_rn(1.0f, __fsqrt_rn(fadd(__fdiv_rn(t, static_cast<float>(a.cols)), a.eps)));
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int u = c * blockDim.x + threadIdx.x;
      const bool on = u < units;
      float w[8] = {}, z[8];
      if (on) load8_of<true>(w, a.weight + int64_t{8} * u * size_of(a.wtype), a.wtype, 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = fmul(fmul(v[c][i], rs), w[i]);
      if (on && a.y.p) {
        uint8_t* yp = a.y.p + row * a.y.stride + int64_t{8} * u * size_of(a.y.type);
        if (a.y.type == X) store8<X, true>(yp, z);
        else store8_of<true>(yp, z, a.y.type, 8);
      }
      if (a.q.codes) put_rows8<true>(a.q, row, u, z, on);
    }
  }
}

// -------------------------------------------- quantizeRows, dequantizeRows
struct CodecArgs {
  Mat x;
  Rows8 q;
  int64_t rows;
  int cols;
};
constexpr int kCodecThreads = 256;

template <bool VEC>
__global__ void __launch_bounds__(kCodecThreads) k_quantize_rows(const CodecArgs a) {
  begin();
  const int per = a.cols / 8;
  const int64_t n = a.rows * per, step = static_cast<int64_t>(gridDim.x) * kCodecThreads;
  // whole warps run the same number of rounds: a group's maximum meets by shuffles
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * kCodecThreads + (threadIdx.x & ~31u); i0 < n; i0 += step) {
    const int64_t i = i0 + (threadIdx.x & 31);
    const bool on = i < n;
    const int64_t row = on ? (n >> 32 ? i / per : static_cast<uint32_t>(i) / static_cast<uint32_t>(per)) : 0;
    const int u = on ? static_cast<int>(i - row * per) : 0;
    float x[8] = {};
    if (on) load8_of<VEC>(x, a.x.p + row * a.x.stride + int64_t{8} * u * size_of(a.x.type), a.x.type, 8);
    put_rows8<VEC>(a.q, row, u, x, on);
  }
}

// Aligned MXFP8 rows: as many codes a thread as make 16 bytes of values, so that a warp
// writes whole lines, four pieces in flight (16 codes a thread, each with two stores 32
// bytes apart from its neighbour's, ran 23 us where this takes 20: 8192 rows of 4096 to bf16, 101 MB).
template <int X>
__global__ void __launch_bounds__(kCodecThreads) k_dequantize_mx8(const CodecArgs a) {
  constexpr int kTake = 4, kCodes = 16 / size_of(X);
  begin();
  const uint32_t per = static_cast<uint32_t>(a.cols / kCodes);
  const int64_t n = a.rows * per, step = static_cast<int64_t>(gridDim.x) * kCodecThreads;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * kCodecThreads + threadIdx.x; i0 < n; i0 += kTake * step) {
    uint32_t c[kTake][kCodes / 4], sc[kTake];
    uint8_t* to[kTake];
#pragma unroll
    for (int h = 0; h < kTake; ++h) {
      const int64_t i = i0 + h * step;
      to[h] = nullptr;
      if (i >= n) continue;
      const int64_t row = n >> 32 ? i / per : static_cast<uint32_t>(i) / per;
      const int u = static_cast<int>(i - row * per);
      const uint8_t* p = a.q.codes + row * a.q.code_stride + int64_t{kCodes} * u;
      if constexpr (kCodes == 8) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        c[h][0] = t.x, c[h][1] = t.y;
      } else {
        c[h][0] = *reinterpret_cast<const uint32_t*>(p);
      }
      sc[h] = a.q.scales[row * a.q.scale_stride + u / (32 / kCodes)];
      to[h] = a.x.p + row * a.x.stride + int64_t{16} * u;
    }
#pragma unroll
    for (int h = 0; h < kTake; ++h) {
      if (!to[h]) continue;
      const float s = e8m0_value(sc[h]);
      float x[kCodes];
#pragma unroll
      for (int j = 0; j < kCodes / 2; ++j) {
        const float2 v = e4m3x2_values(c[h][j >> 1] >> (16 * (j & 1)) & 0xffffu);
        x[2 * j] = fmul(v.x, s);
        x[2 * j + 1] = fmul(v.y, s);
      }
      if constexpr (X == LP_F32) *reinterpret_cast<float4*>(to[h]) = make_float4(x[0], x[1], x[2], x[3]);
      else store8<X, true>(to[h], x);
    }
  }
}

template <bool VEC>
__global__ void __launch_bounds__(kCodecThreads) k_dequantize_rows(const CodecArgs a) {
  begin();
  const int per = a.cols / 8;
  const int64_t n = a.rows * per, step = static_cast<int64_t>(gridDim.x) * kCodecThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCodecThreads + threadIdx.x; i < n; i += step) {
    const int64_t row = n >> 32 ? i / per : static_cast<uint32_t>(i) / static_cast<uint32_t>(per);
    const int u = static_cast<int>(i - row * per);
    const uint8_t* p = a.q.codes + row * a.q.code_stride + int64_t{8} * u;
    const uint8_t* sp = a.q.scales + row * a.q.scale_stride;
    uint32_t w[2] = {0, 0};
    if constexpr (VEC) {
      const uint2 t = *reinterpret_cast<const uint2*>(p);
      w[0] = t.x, w[1] = t.y;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j >> 2] |= static_cast<uint32_t>(p[j]) << (8 * (j & 3));
    }
    float x[8];
    if (a.q.int8) {
      const float s = reinterpret_cast<const float*>(sp)[(u * 8) >> a.q.group_shift];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = fmul(static_cast<float>(static_cast<int8_t>(w[j >> 2] >> (8 * (j & 3)))), s);
    } else {
      const float s = e8m0_value(sp[u >> 2]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = e4m3x2_values(w[j >> 1] >> (16 * (j & 1)) & 0xffffu);
        x[2 * j] = fmul(v.x, s);
        x[2 * j + 1] = fmul(v.y, s);
      }
    }
    store8_of<VEC>(a.x.p + row * a.x.stride + int64_t{8} * u * size_of(a.x.type), x, a.x.type, 8);
  }
}

// ------------------------------------------------------- combineExperts
//
//   out[t] = residual[t] + sum_j weights[t, j] * rows[places[t, j]]
//
// in the order of j, in fp32.  A thread holds 8 elements of a token and reads
// four of its experts' rows at a time.
struct CombineArgs {
  Mat rows, res, out;
  const float* weights;
  const int32_t* places;
  int64_t tokens, nrows;
  int k, cols;
};

__global__ void __launch_bounds__(kCodecThreads) k_combine(const CombineArgs a) {
  begin();
  const int per = (a.cols + 7) / 8;
  const int64_t n = a.tokens * per, step = static_cast<int64_t>(gridDim.x) * kCodecThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCodecThreads + threadIdx.x; i < n; i += step) {
    const int64_t t = n >> 32 ? i / per : static_cast<uint32_t>(i) / static_cast<uint32_t>(per);
    const int u = static_cast<int>(i - t * per), left = a.cols - 8 * u;
    const uint8_t* col = a.rows.p + int64_t{8} * u * size_of(a.rows.type);
    float sum[8] = {};
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      float w[4], x[4][8];
      int64_t place[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = j0 + j < a.k;
        place[j] = in ? a.places[t * a.k + j0 + j] : -1;
        w[j] = in ? a.weights[t * a.k + j0 + j] : 0.0f;
        if (place[j] >= a.nrows) place[j] = -1;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (place[j] >= 0) load8_of<false>(x[j], col + place[j] * a.rows.stride, a.rows.type, left);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (place[j] < 0) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = __fmaf_rn(w[j], x[j][e], sum[e]);
      }
    }
    if (a.res.p) {
      float r[8];
      load8_of<false>(r, a.res.p + t * a.res.stride + int64_t{8} * u * size_of(a.res.type), a.res.type, left);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = fadd(r[e], sum[e]);
    }
    store8_of<false>(a.out.p + t * a.out.stride + int64_t{8} * u * size_of(a.out.type), sum, a.out.type, left);
  }
}

// The same for aligned rows of type Y: a warp's lanes hold a token's neighbouring pieces,
// and all of four rows' loads are issued before the first is used.
template <int Y>
__global__ void __launch_bounds__(kCodecThreads) k_combine_vec(const CombineArgs a) {
  begin();
  const uint32_t per = static_cast<uint32_t>(a.cols / 8);
  const int64_t n = a.tokens * per, step = static_cast<int64_t>(gridDim.x) * kCodecThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kCodecThreads + threadIdx.x; i < n; i += step) {
    const int64_t t = n >> 32 ? i / per : static_cast<uint32_t>(i) / per;
    const int u = static_cast<int>(i - t * per);
    const uint8_t* col = a.rows.p + int64_t{8} * u * size_of(Y);
    float sum[8] = {};
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      Raw8<Y> x[4];
      float w[4];
      bool on[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = j0 + j < a.k;
        const int64_t place = in ? __ldg(a.places + t * a.k + j0 + j) : -1;
        w[j] = in ? __ldg(a.weights + t * a.k + j0 + j) : 0.0f;
        on[j] = place >= 0 && place < a.nrows;
        x[j].zero();
        if (on[j]) x[j].load(col + place * a.rows.stride);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v[8];
        x[j].get(v);
        if (!on[j]) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] = __fmaf_rn(w[j], v[e], sum[e]);
      }
    }
    if (a.res.p) {
      float r[8];
      load8_of<true>(r, a.res.p + t * a.res.stride + int64_t{8} * u * size_of(a.res.type), a.res.type, 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = fadd(r[e], sum[e]);
    }
    store8_of<true>(a.out.p + t * a.out.stride + int64_t{8} * u * size_of(a.out.type), sum, a.out.type, 8);
  }
}

Mat mat(const lp_matrix* m) {
  if (!m) return {nullptr, 0, LP_F32};
  return {static_cast<uint8_t*>(m->data), m->stride * size_of(m->dtype), m->dtype};
}
Rows8 rows8(const lp_rows8* r) {
  if (!r) return {};
  const int shift = 31 - __builtin_clz(static_cast<unsigned>(r->group));
  return {static_cast<uint8_t*>(r->codes), static_cast<uint8_t*>(r->scales), r->code_stride,
          r->scale_stride * (r->dtype == LP_I8 ? 4 : 1), r->dtype == LP_I8, r->group / 8, shift};
}
int codec_grid(int64_t threads) {
  return static_cast<int>(std::min<int64_t>((threads + kCodecThreads - 1) / kCodecThreads,
                                            device_info().sm_count * 32ll));
}

}  // namespace

int launch_norm(const lp_matrix& x, const lp_matrix* residual, const void* weight, int weight_type, float eps,
                const lp_matrix* total, const lp_matrix* y, const lp_rows8* q, bool vec, cudaStream_t st) {
  NormArgs a{mat(&x), mat(residual), mat(total), mat(y), static_cast<const uint8_t*>(weight), rows8(q),
             x.rows, static_cast<int>(x.cols), weight_type, eps};
  const int units = (a.cols + 7) / 8;
  const int sms = device_info().sm_count;
  // Few rows: as many threads as there are pieces, whose chains are shortest; many: two
  // pieces a thread, or four of long rows (8192 rows in bf16, two / four pieces: of 2048 29.3 /
  // 31.2 us, of 4096 57.4 / 53.0).
  int c = 1;
  while ((units + c - 1) / c > 1024) c *= 2;
  if (c == 1 && units > 64 && x.rows > sms) c = units < 512 ? 2 : 4;
  const int threads = ((units + c - 1) / c + 31) / 32 * 32;
  const int grid = static_cast<int>(std::min<int64_t>(x.rows, sms * 16ll));
  const int stream = residual ? residual->dtype : x.dtype;
#define LP_NORM_T(C, X, R) \
  if (x.dtype == X && stream == R) return launch_early(k_norm_vec<X, R, C>, grid, threads, st, a);
#define LP_NORM(C)                                                    \
  if (c == C) {                                                       \
    if (!vec) return launch_early(k_norm<C>, grid, threads, st, a); \
    LP_NORM_T(C, LP_F32, LP_F32)                                      \
    LP_NORM_T(C, LP_F16, LP_F16)                                      \
    LP_NORM_T(C, LP_F16, LP_F32)                                      \
    LP_NORM_T(C, LP_BF16, LP_BF16)                                    \
    LP_NORM_T(C, LP_BF16, LP_F32)                                     \
  }
  LP_NORM(1) LP_NORM(2) LP_NORM(4)
#undef LP_NORM_T
#undef LP_NORM
  return LP_ERR_UNSUPPORTED;
}

int launch_quantize_rows(const lp_matrix& x, const lp_rows8& q, bool vec, cudaStream_t st) {
  const CodecArgs a{mat(&x), rows8(&q), x.rows, static_cast<int>(x.cols)};
  const int grid = codec_grid(x.rows * (x.cols / 8));
  if (vec) return launch_early(k_quantize_rows<true>, grid, kCodecThreads, st, a);
  return launch_early(k_quantize_rows<false>, grid, kCodecThreads, st, a);
}

int launch_dequantize_rows(const lp_rows8& q, const lp_matrix& x, bool vec, cudaStream_t st) {
  const CodecArgs a{mat(&x), rows8(&q), x.rows, static_cast<int>(x.cols)};
  const int grid = codec_grid(x.rows * (x.cols / 8));
  if (vec && q.dtype == LP_E4M3) {
    if (x.dtype == LP_F32)
      return launch_early(k_dequantize_mx8<LP_F32>, codec_grid(x.rows * (x.cols / 4)), kCodecThreads, st, a);
    if (x.dtype == LP_F16) return launch_early(k_dequantize_mx8<LP_F16>, grid, kCodecThreads, st, a);
    return launch_early(k_dequantize_mx8<LP_BF16>, grid, kCodecThreads, st, a);
  }
  if (vec) return launch_early(k_dequantize_rows<true>, grid, kCodecThreads, st, a);
  return launch_early(k_dequantize_rows<false>, grid, kCodecThreads, st, a);
}

int launch_combine(const lp_matrix& rows, const float* weights, const int32_t* places, int64_t k,
                   const lp_matrix* residual, const lp_matrix& out, bool vec, cudaStream_t st) {
  const CombineArgs a{mat(&rows), mat(residual), mat(&out), weights, places, out.rows, rows.rows,
                      static_cast<int>(k), static_cast<int>(out.cols)};
  const int grid = codec_grid(out.rows * ((out.cols + 7) / 8));
  if (vec) {
    if (rows.dtype == LP_F32) return launch_early(k_combine_vec<LP_F32>, grid, kCodecThreads, st, a);
    if (rows.dtype == LP_F16) return launch_early(k_combine_vec<LP_F16>, grid, kCodecThreads, st, a);
    return launch_early(k_combine_vec<LP_BF16>, grid, kCodecThreads, st, a);
  }
  return launch_early(k_combine, grid, kCodecThreads, st, a);
}

}  // namespace lp
