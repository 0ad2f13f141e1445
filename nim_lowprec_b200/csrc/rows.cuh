// rows.cuh -- elements of fp32, fp16 and bf16 rows, eight at a time, and their
// int8 codes.
#pragma once
#include <cuda_bf16.h>

#include "lp_device.cuh"

namespace lp {
namespace {

__device__ __forceinline__ uint32_t pack_h(float a, float b) {
  return static_cast<uint32_t>(__half_as_ushort(__float2half_rn(a))) |
         static_cast<uint32_t>(__half_as_ushort(__float2half_rn(b))) << 16;
}
__device__ __forceinline__ uint32_t pack_b(float a, float b) {
  return static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(a))) |
         static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(b))) << 16;
}

// Eight elements of type T at p.  VEC: p is on a boundary of its 16-byte (or,
// int8, 8-byte) pieces; else element by element.
template <int T, bool VEC>
__device__ __forceinline__ void load8(float* x, const uint8_t* p) {
  if constexpr (T == LP_F32) {
    if constexpr (VEC) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p));
      const float4 w = __ldg(reinterpret_cast<const float4*>(p) + 1);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __ldg(reinterpret_cast<const float*>(p) + i);
    }
  } else {
    uint32_t w[4];
    if constexpr (VEC) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __ldg(h + 2 * i) | static_cast<uint32_t>(__ldg(h + 2 * i + 1)) << 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (T == LP_F16) {
        x[2 * i] = h2f(w[i] & 0xffffu);
        x[2 * i + 1] = h2f(w[i] >> 16);
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}

template <int T, bool VEC>
__device__ __forceinline__ void store8(uint8_t* p, const float* x) {
  if constexpr (T == LP_F32) {
    if constexpr (VEC) {
      reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<float*>(p)[i] = x[i];
    }
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = T == LP_F16 ? pack_h(x[2 * i], x[2 * i + 1]) : pack_b(x[2 * i], x[2 * i + 1]);
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        reinterpret_cast<unsigned short*>(p)[i] =
            static_cast<unsigned short>(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

__host__ __device__ constexpr int size_of(int t) { return t == LP_F32 ? 4 : t == LP_I8 ? 1 : 2; }

// int8 codes of x / s, rounded half away from zero, four to a word.  The quotient
// is exact where it decides something: x * (1 / s) is off by at most 2^-22 of 127,
// so a result further than 2^-14 from the middle between two whole numbers rounds
// as the quotient does; others (and what is not finite) are divided.  (Sixteen divisions a thread took three times the bytes' time.)
template <int N>
__device__ __forceinline__ void codes(uint32_t* w, const float* x, float s) {
  constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are the whole number
  const float inv = __fdiv_rn(1.0f, s);
  bool sure = true;
  uint32_t q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = fmul(x[i], inv);
    const float z = fadd(y, kMagic);
    q[i] = __float_as_uint(z);
    sure = sure && fabsf(fadd(y, -fadd(z, -kMagic))) < 0.5f - 6.1e-5f;  // (not for a NaN)
  }
  if (!sure) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      q[i] = static_cast<uint32_t>(
          static_cast<int>(fminf(fmaxf(roundf(__fdiv_rn(x[i], s)), -128.0f), 127.0f)));
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = prmt(prmt(q[4 * i], q[4 * i + 1], 0x0040u), prmt(q[4 * i + 2], q[4 * i + 3], 0x0040u), 0x5410u);
}

// Eight elements of a type known at run time, the first `n` of them where they
// are read or written one by one (VEC: all, on a 16-byte boundary).  Plain loads:
// the memory may be what the same kernel writes.
template <bool VEC>
__device__ __forceinline__ void load8_of(float* x, const uint8_t* p, int type, int n) {
  if (type == LP_F32) {
    if constexpr (VEC) {
      const float4 u = reinterpret_cast<const float4*>(p)[0], w = reinterpret_cast<const float4*>(p)[1];
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < n ? reinterpret_cast<const float*>(p)[i] : 0.0f;
    }
    return;
  }
  uint32_t w[4];
  if constexpr (VEC) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
    const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (2 * i < n ? h[2 * i] : 0u) | static_cast<uint32_t>(2 * i + 1 < n ? h[2 * i + 1] : 0u) << 16;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (type == LP_F16) {
      x[2 * i] = h2f(w[i] & 0xffffu);
      x[2 * i + 1] = h2f(w[i] >> 16);
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}
// Eight elements of type T as they lie in memory, 16-byte aligned: loads that are issued
// together, before the first is converted.  Plain loads, as above.
template <int T>
struct Raw8 {
  uint4 a, b;
  __device__ __forceinline__ void load(const uint8_t* p) {
    a = *reinterpret_cast<const uint4*>(p);
    if constexpr (T == LP_F32) b = reinterpret_cast<const uint4*>(p)[1];
  }
  __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float* x) const {
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (T == LP_F32) x[i] = __uint_as_float(w[i]);
      else if constexpr (T == LP_F16) x[i] = h2f(w[i >> 1] >> (16 * (i & 1)) & 0xffffu);
      else x[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    }
  }
};
__device__ __forceinline__ void store1_of(uint8_t* p, float x, int type) {
  if (type == LP_F32) *reinterpret_cast<float*>(p) = x;
  else if (type == LP_F16) *reinterpret_cast<__half*>(p) = __float2half_rn(x);
  else *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x);
}
template <bool VEC>
__device__ __forceinline__ void store8_of(uint8_t* p, const float* x, int type, int n) {
  if constexpr (VEC) {
    if (type == LP_F32) store8<LP_F32, true>(p, x);
    else if (type == LP_F16) store8<LP_F16, true>(p, x);
    else store8<LP_BF16, true>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) store1_of(p + i * size_of(type), x[i], type);
  }
}
// x as its type holds it.
__device__ __forceinline__ float rounded(float x, int type) {
  if (type == LP_F16) return __half2float(__float2half_rn(x));
  if (type == LP_BF16) return __bfloat162float(__float2bfloat16_rn(x));
  return x;
}

// ---------------------------------------------------- MXFP8 (OCP MX, e4m3)
// The E8M0 code of a block's scale, 2^(floor(log2 amax) - 8), calibrateMX's rule
// (quant.nim:125-137; 1 for a block of zeros) as a difference of exponent fields;
// an infinity's field is 255, so its code saturates to a value that is infinite.
__device__ __forceinline__ uint32_t mx8_scale(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 8;
  return amax == 0.0f ? 127u : static_cast<uint32_t>(e > 0 ? e : 0);
}
// 2^-(code - 127) of such a code (at most 247), exact.
__device__ __forceinline__ float mx8_inverse(uint32_t code) {
  return __uint_as_float((254u - code) << 23);
}
__device__ __forceinline__ float e8m0_value(uint32_t code) {
  return code == 255u ? __uint_as_float(0x7fffffffu)
                      : code ? __uint_as_float(code << 23) : __uint_as_float(0x00400000u);
}
// Four e4m3 codes of x * inv, rounded to nearest even, at most 448 in magnitude.
__device__ __forceinline__ uint32_t e4m3x4(const float* x, float inv) {
  uint32_t d;
  asm("{ .reg .b16 a, b; cvt.rn.satfinite.e4m3x2.f32 a, %2, %1; cvt.rn.satfinite.e4m3x2.f32 b, %4, %3; "
      "mov.b32 %0, {a, b}; }"
      : "=r"(d)
      : "f"(fmul(x[0], inv)), "f"(fmul(x[1], inv)), "f"(fmul(x[2], inv)), "f"(fmul(x[3], inv)));
  return d;
}
// The values of two e4m3 codes.
__device__ __forceinline__ float2 e4m3x2_values(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(two)));
  return make_float2(h2f(h & 0xffffu), h2f(h >> 16));
}

}  // namespace
}  // namespace lp
