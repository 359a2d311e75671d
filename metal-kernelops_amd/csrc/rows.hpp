// Vectors of consecutive elements of a row at any alignment, column sums in a fixed order, and what
// the entry points of the row operators share.
#pragma once

#include "common.hpp"

namespace mko {

__host__ __device__ __forceinline__ int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool half_or_float(int32_t dtype) { return dtype == MKO_F32 || dtype == MKO_F16 || dtype == MKO_BF16; }

// Elements of a 16-byte vector of T.
template <typename T>
constexpr int kVecOf = 16 / static_cast<int>(sizeof(T));

// NE elements of T as loaded.  The words go to and from any address: global accesses of this part
// take every alignment, at full rate where they are aligned.
template <typename T, int NE>
struct Words {
  uint32_t w[kWordsOf<T, NE>];
};
template <typename T, int NE>
struct __attribute__((packed)) AnyWords {
  Words<T, NE> v;
};

// Elements i .. i + NE - 1 of a row of n; those past the end read as zero and nothing past it is read.
template <typename T, int NE>
__device__ __forceinline__ Words<T, NE> load_part(const T* row, int64_t i, int64_t n) {
  if (i + NE <= n) return reinterpret_cast<const AnyWords<T, NE>*>(row + i)->v;
  Words<T, NE> r{};
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    if (i + e >= n) continue;
    if constexpr (sizeof(T) == 4)
      r.w[e] = __builtin_bit_cast(uint32_t, row[i + e]);
    else
      r.w[e / 2] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, row[i + e])) << (16 * (e % 2));
  }
  return r;
}

template <typename T, int NE>
__device__ __forceinline__ void store_part(T* row, int64_t i, int64_t n, const float (&f)[NE]) {
  if (i + NE <= n) {
    AnyWords<T, NE> o;
    pack_words<T, NE>(f, o.v.w);
    *reinterpret_cast<AnyWords<T, NE>*>(row + i) = o;
    return;
  }
#pragma unroll
  for (int e = 0; e < NE; ++e)
    if (i + e < n) row[i + e] = from_f32<T>(f[e]);
}

// NE values of a parameter of a runtime dtype as float32.
template <int NE>
__device__ __forceinline__ void load_param_part(const void* p, int dtype, int64_t i, int64_t n, float (&f)[NE]) {
  if (dtype == MKO_F32)
    unpack_words<float, NE>(load_part<float, NE>(static_cast<const float*>(p), i, n).w, f);
  else if (dtype == MKO_BF16)
    unpack_words<bf16, NE>(load_part<bf16, NE>(static_cast<const bf16*>(p), i, n).w, f);
  else
    unpack_words<_Float16, NE>(load_part<_Float16, NE>(static_cast<const _Float16*>(p), i, n).w, f);
}

// Sum of each of 32 columns of a (rows, columns) array by a workgroup of 1024 threads: thread (r, c)
// adds rows r, r + 32, ..., then the 32 sums of a column are added in order.  The result is in the
// threads below 32; the order depends on the sizes alone.
constexpr int kColumnThreads = 1024;
__device__ __forceinline__ float column_sum(const float* a, int64_t rows, int64_t columns, int64_t column) {
  __shared__ float sums[32][33];
  const int r = threadIdx.x >> 5, c = threadIdx.x & 31;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (column < columns) {
    int64_t i = r;
    for (; i + 96 < rows; i += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] += a[(i + 32 * k) * columns + column];
    }
    for (int k = 0; i < rows; i += 32, ++k) s[k & 3] += a[i * columns + column];
  }
  sums[r][c] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  float t = 0.0f;
  if (r == 0)
    for (int k = 0; k < 32; ++k) t += sums[k][c];
  return t;
}

}  // namespace mko
