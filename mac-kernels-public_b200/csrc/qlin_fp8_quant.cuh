// Bringing rows of f32, f16 or bf16 to e4m3: loads and conversions shared by the row quantizer and the small-M
// product, which quantizes its few rows itself.
#pragma once
#include <cuda_fp8.h>

#include "../../include/qlin.h"
#include "qlin_ptx.cuh"

namespace qlin {

constexpr float kE4m3Max = 448.f;
constexpr uint32_t kAmaxFloorBits = (127 - 100) << 23;  // 2^-100

// 8 consecutive values as stored: 16 bytes of a 2-byte type, 32 of fp32.
template <int DT>
struct Raw8 {
  uint4 v[DT == QLIN_F32 ? 2 : 1];
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* x, long long i) {
  Raw8<DT> r;
  constexpr int kBytes = DT == QLIN_F32 ? 4 : 2;
  const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(x) + i * kBytes);
  r.v[0] = p[0];
  if constexpr (DT == QLIN_F32) r.v[1] = p[1];
  return r;
}

// The same from any address of the type's alignment: the aligned 16-byte words around the values (load), shifted
// when they have arrived (values).  `lim` is the number of values from x on that are the caller's; where the words
// would reach past them, the values are read one by one.
template <int DT>
struct Around8 {
  static constexpr int kBytes = DT == QLIN_F32 ? 4 : 2;
  static constexpr int kWords = DT == QLIN_F32 ? 12 : 8;  // 32-bit words read
  static constexpr int kOut = DT == QLIN_F32 ? 8 : 4;
  uint4 v[kWords / 4];
  uint32_t off;  // of the values, in bytes from v; 16: the values lie in v as they are

  __device__ __forceinline__ void load(const void* x, long long i, long long lim) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(x), at = begin + i * kBytes, from = at & ~uintptr_t(15);
    const bool inside = from >= begin && from + kWords * 4 <= begin + lim * kBytes;
    off = inside ? (uint32_t)(at & 15) : 16;
#pragma unroll
    for (int j = 0; j < kWords / 4; ++j) v[j] = inside ? reinterpret_cast<const uint4*>(from)[j] : uint4{};
    if (!inside) {
      uint32_t o[kWords] = {};
      for (int j = 0; j < 8; ++j) {
        if constexpr (DT == QLIN_F32) {
          const uint32_t b = reinterpret_cast<const uint32_t*>(x)[i + j];
#pragma unroll
          for (int q = 0; q < 8; ++q) o[q] = q == j ? b : o[q];
        } else {
          const uint32_t b = (uint32_t) reinterpret_cast<const uint16_t*>(x)[i + j] << (16 * (j & 1));
#pragma unroll
          for (int q = 0; q < 4; ++q) o[q] |= q == j / 2 ? b : 0;
        }
      }
#pragma unroll
      for (int j = 0; j < kWords / 4; ++j) v[j] = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
    }
  }
  __device__ __forceinline__ Raw8<DT> values() const {
    uint32_t w[kWords + 1];
#pragma unroll
    for (int j = 0; j < kWords / 4; ++j) {
      w[4 * j] = v[j].x;
      w[4 * j + 1] = v[j].y;
      w[4 * j + 2] = v[j].z;
      w[4 * j + 3] = v[j].w;
    }
    w[kWords] = 0;
#pragma unroll
    for (int j = 0; j + 2 <= kWords; ++j) w[j] = (off & 8) ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j + 1 <= kWords; ++j) w[j] = (off & 4) ? w[j + 1] : w[j];
    uint32_t o[kOut];
#pragma unroll
    for (int j = 0; j < kOut; ++j) o[j] = kBytes == 2 ? __funnelshift_r(w[j], w[j + 1], (off & 2) * 8) : w[j];
    Raw8<DT> r;
    r.v[0] = make_uint4(o[0], o[1], o[2], o[3]);
    if constexpr (DT == QLIN_F32) r.v[1] = make_uint4(o[4], o[5], o[6], o[7]);
    return r;
  }
};

template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8_any(const void* x, long long i, long long lim) {
  Around8<DT> a;
  a.load(x, i, lim);
  return a.values();
}

template <int DT>
__device__ __forceinline__ void raw8_to_float(const Raw8<DT>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == QLIN_F32) {
      f[j] = __uint_as_float(w[j]);
    } else if constexpr (DT == QLIN_F16) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    } else {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
  }
  if constexpr (DT == QLIN_F32) {
    f[4] = __uint_as_float(r.v[1].x);
    f[5] = __uint_as_float(r.v[1].y);
    f[6] = __uint_as_float(r.v[1].z);
    f[7] = __uint_as_float(r.v[1].w);
  }
}

// The same with the values from the n-th on set to zero.
template <int DT>
__device__ __forceinline__ Raw8<DT> raw8_first(Raw8<DT> r, int n) {
  uint32_t w[DT == QLIN_F32 ? 8 : 4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  if constexpr (DT == QLIN_F32) {
    w[4] = r.v[1].x;
    w[5] = r.v[1].y;
    w[6] = r.v[1].z;
    w[7] = r.v[1].w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = j < n ? w[j] : 0;
    r.v[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = 2 * j + 1 < n ? w[j] : 2 * j < n ? w[j] & 0xffffu : 0;
  }
  r.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
  return r;
}

// n of 8 consecutive values, one by one, and zeros.
template <int DT>
__device__ __forceinline__ Raw8<DT> gather_raw8(const void* x, long long i, int n) {
  uint32_t w[DT == QLIN_F32 ? 8 : 4] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= n) continue;
    if constexpr (DT == QLIN_F32) w[j] = reinterpret_cast<const uint32_t*>(x)[i + j];
    else w[j / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(x)[i + j] << (16 * (j & 1));
  }
  Raw8<DT> r;
  r.v[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if constexpr (DT == QLIN_F32) r.v[1] = make_uint4(w[4], w[5], w[6], w[7]);
  return r;
}

// Bit pattern, as fp32, of the largest magnitude among the 8.  Patterns of one type order like the
// magnitudes, with the infinity and the NaNs on top, so 2-byte types are compared two at a time.
template <int DT>
__device__ __forceinline__ uint32_t raw8_amax_bits(const Raw8<DT>& r) {
  const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
  if constexpr (DT == QLIN_F32) {
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) a = max(a, w[j] & 0x7fffffffu);
    const uint32_t x[4] = {r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) a = max(a, x[j] & 0x7fffffffu);
    return a;
  } else {
    uint32_t a = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int j = 1; j < 4; ++j) a = __vmaxu2(a, w[j] & 0x7fff7fffu);
    const uint32_t top = max(a >> 16, a & 0xffffu);
    if constexpr (DT == QLIN_BF16) return top << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top)));
  }
}

// 4 values times r in e4m3, the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d, float r) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * r, b * r), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * r, d * r), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

}  // namespace qlin
