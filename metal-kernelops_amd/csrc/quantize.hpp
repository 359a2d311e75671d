// Symmetric 8-bit quantisation of a row: q = rint(v * (127 / amax)), scale = amax / 127.
#pragma once

#include "common.hpp"

namespace mko {

// |v| as the integer that orders like it.  Its maximum keeps what fmaxf drops: a NaN sorts above
// an infinity and an infinity above every number.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Maximum over the wave, wave-uniform.  The four DPP steps of row16_sum.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xb1, 0xf, 0xf, false)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4e, 0xf, 0xf, false)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xf, 0xf, false)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x140, 0xf, 0xf, false)));
  const uint32_t a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
  const uint32_t c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
  return max(max(a, b), max(c, d));
}

struct RowScale {
  float scale, inv;
};

// From the row's largest |v| (as abs_bits).  Both quotients are IEEE divisions.  A row below
// 2^-100 has the scale 0 (its 127 / amax leaves the range); one that holds an infinity or a NaN
// keeps that in its scale, so that every output of the row is not finite.
__device__ __forceinline__ RowScale row_scale(uint32_t amax) {
  const float a = __uint_as_float(amax);
  RowScale r;
  const bool tiny = a < 0x1p-100f;
  r.scale = tiny ? 0.0f : a / 127.0f;
  r.inv = tiny || amax >= 0x7f800000u ? 0.0f : 127.0f / a;
  return r;
}

// rint(v * inv), to nearest even, as an integer in [-127, 127].  A NaN, in whose row the scale is not
// finite, gives -127: the maximum drops it.
__device__ __forceinline__ int quantise(float v, float inv) {
  const float q = rintf(fp32_value(v * inv));
  return static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// NE bytes from column i of a row of n columns padded to `pitch`, the padding zero.  Rows start at
// any byte.
template <int NE>
__device__ __forceinline__ void store_bytes(int8_t* row, int64_t i, int64_t n, int64_t pitch, const int (&b)[NE]) {
  if (i >= n) return;
  uint32_t w[NE / 4];
#pragma unroll
  for (int k = 0; k < NE / 4; ++k) {
    w[k] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[k] |= (i + 4 * k + e < n ? static_cast<uint32_t>(b[4 * k + e]) & 0xffu : 0u) << (8 * e);
  }
  struct __attribute__((packed)) Any {
    uint32_t w[NE / 4];
  };
  if (i + NE <= pitch) {
    Any o;
#pragma unroll
    for (int k = 0; k < NE / 4; ++k) o.w[k] = w[k];
    *reinterpret_cast<Any*>(row + i) = o;
  } else {
#pragma unroll
    for (int e = 0; e < NE; ++e)
      if (i + e < pitch) row[i + e] = static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)));
  }
}

}  // namespace mko
