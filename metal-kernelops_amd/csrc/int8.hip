// 8-bit integers for gfx950: quantisation of rows, and the matrix product
//   out[m][n] = q_scale[m] w_scale[n] sum_k q[m][k] w[n][k] + bias[n]
// with the sum in int32, exact for fewer than 2^17 terms of at most 2^14.
#include "common.hpp"
#include "io.hpp"
#include "quantize.hpp"

namespace mko {
namespace int8 {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxInner = 131071;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_rows(mko_quantize_params p) {
  __shared__ uint32_t top[kThreads / kWave];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  uint32_t am = 0;
  for (int64_t i = threadIdx.x; i < p.features; i += kThreads) am = max(am, abs_bits(to_f32(x[i])));
  am = wave_max(am);
  if ((threadIdx.x & (kWave - 1)) == 0) top[threadIdx.x / kWave] = am;
  __syncthreads();
  for (int w = 0; w < kThreads / kWave; ++w) am = max(am, top[w]);
  const RowScale q = row_scale(am);
  if (threadIdx.x == 0) p.scale[row] = q.scale;
  for (int64_t i = threadIdx.x; i < p.q_stride; i += kThreads)
    p.q[row * p.q_stride + i] = i < p.features ? static_cast<int8_t>(quantise(to_f32(x[i]), q.inv)) : 0;
}

__global__ void __launch_bounds__(kThreads) product(mko_int8_linear_params p) {
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (n >= p.outer) return;
  const int8_t* w = p.w + n * p.w_stride;
  for (int64_t m = blockIdx.y; m < p.rows; m += gridDim.y) {
    const int8_t* q = p.q + m * p.q_stride;
    int acc = 0;
    for (int64_t k = 0; k < p.inner; ++k) acc += static_cast<int>(q[k]) * w[k];
    float v = static_cast<float>(acc) * p.q_scale[m] * p.w_scale[n];
    if (p.bias) v += p.bias[n];
    store_one(p.out, p.dtype, m * p.outer + n, v);
  }
}

bool half_or_float(int32_t dtype) { return dtype == MKO_F32 || dtype == MKO_F16 || dtype == MKO_BF16; }

int check(const mko_int8_linear_params* p) {
  if (!p || p->rows < 0 || p->inner < 0 || p->outer < 0) {
    mko_set_error("int8_linear: params is NULL or a size is negative");
    return MKO_EINVAL;
  }
  if (!half_or_float(p->dtype)) {
    mko_set_error("int8_linear: dtype must be float32, float16 or bfloat16");
    return MKO_EINVAL;
  }
  if (p->inner > kMaxInner || p->rows > 0x7fffffff || p->outer > 0x7fffffff) {
    mko_set_error("int8_linear: inner is at most %lld, rows and outer at most 2^31 - 1",
                  static_cast<long long>(kMaxInner));
    return MKO_EUNSUPPORTED;
  }
  return MKO_OK;
}

}  // namespace
}  // namespace int8
}  // namespace mko

using namespace mko;

extern "C" size_t mko_sizeof_quantize_params(void) { return sizeof(mko_quantize_params); }
extern "C" size_t mko_sizeof_int8_linear_params(void) { return sizeof(mko_int8_linear_params); }

extern "C" int mko_quantize_int8(const mko_quantize_params* p, void* stream) {
  if (!p || p->rows < 0 || p->features < 0 || p->q_stride < p->features) {
    mko_set_error("quantize_int8: params is NULL, a size is negative or q_stride is smaller than features");
    return MKO_EINVAL;
  }
  if (!int8::half_or_float(p->dtype)) {
    mko_set_error("quantize_int8: dtype must be float32, float16 or bfloat16");
    return MKO_EINVAL;
  }
  if (p->rows > 0x7fffff) {
    mko_set_error("quantize_int8: rows is at most 2^23 - 1");
    return MKO_EUNSUPPORTED;
  }
  if (p->rows == 0) return MKO_OK;
  if (!p->scale || (p->features && (!p->x || !p->q))) {
    mko_set_error("quantize_int8: x, q and scale are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(p->rows);
  if (p->dtype == MKO_F32)
    MKO_TIMED("quantize_int8", s, int8::quantize_rows<float><<<grid, int8::kThreads, 0, s>>>(*p));
  else if (p->dtype == MKO_BF16)
    MKO_TIMED("quantize_int8", s, int8::quantize_rows<bf16><<<grid, int8::kThreads, 0, s>>>(*p));
  else
    MKO_TIMED("quantize_int8", s, int8::quantize_rows<_Float16><<<grid, int8::kThreads, 0, s>>>(*p));
  return mko_check_launch("quantize_int8");
}

extern "C" size_t mko_int8_linear_workspace_size(const mko_int8_linear_params* p) {
  (void)p;
  return 0;
}

extern "C" int mko_int8_linear(const mko_int8_linear_params* p, void* stream) {
  const int st = int8::check(p);
  if (st != MKO_OK) return st;
  if (p->rows == 0 || p->outer == 0) return MKO_OK;
  if ((p->inner && (!p->q || !p->w)) || !p->q_scale || !p->w_scale || !p->out) {
    mko_set_error("int8_linear: q, q_scale, w, w_scale and out are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(int8::cdiv(p->outer, int8::kThreads)),
                  static_cast<unsigned>(p->rows < 16384 ? p->rows : 16384));
  MKO_TIMED("int8_linear", s, int8::product<<<grid, int8::kThreads, 0, s>>>(*p));
  return mko_check_launch("int8_linear");
}
