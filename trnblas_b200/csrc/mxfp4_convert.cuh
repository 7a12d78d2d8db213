// Conversion of eight neighbouring values to MXFP4, shared by the quantiser and
// the product that quantises its rows itself.
#pragma once

#include "common.cuh"

namespace tb {

// Eight neighbouring values of a row as they are stored.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* src, int valid, bool vec) {
  Raw8<T> r;
  constexpr int V = static_cast<int>(sizeof(T)) / 2;
  if (vec && valid >= 8) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    return r;
  }
  uint32_t w[4 * V] = {};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) w[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid)
        w[i / 2] |= static_cast<uint32_t>(__ldg(reinterpret_cast<const unsigned short*>(src) + i)) << (16 * (i & 1));
  }
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  return r;
}

// 8 E2M1 codes of 8 floats, the first in the lowest bits: nearest, ties to
// even, saturating at 6.
__device__ __forceinline__ uint32_t e2m1x8(const float (&u)[8]) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(u[0]), "f"(u[1]), "f"(u[2]), "f"(u[3]), "f"(u[4]), "f"(u[5]), "f"(u[6]), "f"(u[7]));
  return w;
}

// Four lanes hold a block of 32 (8 values each). The block's unit is 2^(s - 127)
// with s = max(E, 2) - 2, E the biased fp32 exponent of the block's largest
// magnitude: the largest power of two not above it, divided by 4 (E2M1's
// largest power of two). Scaling by it is exact; the conversion rounds to the
// nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to even, and saturates (a block's
// largest magnitude is below 8 units). A block that holds an infinity or a NaN
// gets the NaN scale 255. The maximum is taken on the magnitudes' bits, which
// order as the values do (16-bit types: two at a time).
template <typename T>
__device__ __forceinline__ uint32_t quantize8(const Raw8<T>& r, uint32_t& s) {
  float x[8];
  uint32_t E;
  if constexpr (sizeof(T) == 4) {
    const uint32_t w[8] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w, r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m = max(m, w[i] & 0x7FFFFFFFu);
      x[i] = __uint_as_float(w[i]);
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    E = m >> 23;
  } else {
    const uint32_t w[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
    uint32_t m = __vimax3_u16x2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu, w[2] & 0x7FFF7FFFu);
    uint32_t o = __shfl_xor_sync(0xffffffffu, m = __vimax3_u16x2(m, w[3] & 0x7FFF7FFFu, 0u), 1);
    m = __vimax3_u16x2(m, o, 0u);
    o = __shfl_xor_sync(0xffffffffu, m, 2);
    m = __vimax3_u16x2(m, o, 0u);
    m = max(m & 0xFFFFu, m >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      E = m >> 7;
    else
      E = __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m)))) >> 23;
  }
  s = max(E, 2u) - 2u;
  const float inv = __uint_as_float((254u - s) << 23);  // 2^(127 - s), normal
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] *= inv;
  uint32_t w = e2m1x8(x);
  if (E == 255) {
    s = 255;
    w = 0;
  }
  return w;
}

}  // namespace tb
