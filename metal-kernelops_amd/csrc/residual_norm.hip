// RMS norm of the residual stream for gfx950: stream = x + residual, out = stream r weight, with
// r = 1 / sqrt(mean(stream^2) + eps); or the same in 8 bits with a scale per row.
// Backward, with gw = dout weight and xh = stream r:
//   ds = r (gw - xh mean(gw xh)) + dstream,  dweight = sum over rows of dout xh
#include "common.hpp"
#include "io.hpp"
#include "quantize.hpp"

namespace mko {
namespace resnorm {
namespace {

constexpr int kThreads = 256;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 1 / sqrt(ss * inv_n + eps), rounded once.  In 64 bits, because the backward takes the
// difference of two terms that each hold r twice: a narrow row amplifies every rounding of r.
// v_rsq_f64 and one Newton step.
__device__ __forceinline__ float inverse_norm(float ss, double inv_n, float eps) {
  const double a = static_cast<double>(ss) * inv_n + static_cast<double>(eps);
  const double y = __builtin_amdgcn_rsq(a);
  const double e = 0.5 - 0.5 * a * y * y;
  return static_cast<float>(e == e ? y + y * e : y);  // a is 0 or infinite: y is exact
}

// The stream's value at (row, i): x + residual rounded to the stream's type.
template <typename T, typename S>
__device__ __forceinline__ float stream_at(const mko_resnorm_params& p, int64_t row, int64_t i) {
  const float x = to_f32(static_cast<const T*>(p.x)[row * p.x_stride + i]);
  if (!p.residual) return x;
  return to_f32(from_f32<S>(x + to_f32(static_cast<const S*>(p.residual)[row * p.residual_stride + i])));
}

template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) forward(mko_resnorm_params p) {
  __shared__ float slots[kThreads / kWave];
  __shared__ uint32_t top[kThreads / kWave];
  const int64_t row = blockIdx.x;
  float ss = 0.0f;
  uint32_t am = 0;
  for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
    const float s = stream_at<T, S>(p, row, i);
    if (p.residual) static_cast<S*>(p.stream)[row * p.features + i] = from_f32<S>(s);
    ss += s * s;
    am = max(am, abs_bits(s * load_one(p.weight, p.wdtype, i)));
  }
  ss = wave_sum(ss);
  am = wave_max(am);
  if ((threadIdx.x & (kWave - 1)) == 0) {
    slots[threadIdx.x / kWave] = ss;
    top[threadIdx.x / kWave] = am;
  }
  __syncthreads();
  ss = 0.0f;
  for (int w = 0; w < kThreads / kWave; ++w) {
    ss += slots[w];
    am = max(am, top[w]);
  }
  const float r = inverse_norm(ss, 1.0 / static_cast<double>(p.features), p.eps);
  if (threadIdx.x == 0 && p.rstd) p.rstd[row] = r;
  const RowScale q = row_scale(abs_bits(__uint_as_float(am) * r));
  if (p.q && threadIdx.x == 0) p.q_scale[row] = q.scale;
  for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
    const float v = stream_at<T, S>(p, row, i) * r * load_one(p.weight, p.wdtype, i);
    if (p.q)
      p.q[row * p.q_stride + i] = static_cast<int8_t>(quantise(v, q.inv));
    else
      static_cast<T*>(p.out)[row * p.features + i] = from_f32<T>(v);
  }
  if (p.q)
    for (int64_t i = p.features + threadIdx.x; i < p.q_stride; i += kThreads) p.q[row * p.q_stride + i] = 0;
}

template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) backward(mko_resnorm_params p) {
  __shared__ float slots[kThreads / kWave];
  const int64_t row = blockIdx.x;
  const float r = p.rstd[row];
  float c = 0.0f;
  for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
    const float xh = to_f32(static_cast<const S*>(p.stream)[row * p.features + i]) * r;
    c += xh * to_f32(static_cast<const T*>(p.dout)[row * p.features + i]) * load_one(p.weight, p.wdtype, i);
  }
  c = wave_sum(c);
  if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = c;
  __syncthreads();
  c = 0.0f;
  for (int w = 0; w < kThreads / kWave; ++w) c += slots[w];
  c /= static_cast<float>(p.features);
  for (int64_t i = threadIdx.x; i < p.features; i += kThreads) {
    const int64_t j = row * p.features + i;
    const float xh = to_f32(static_cast<const S*>(p.stream)[j]) * r;
    float ds = r * (to_f32(static_cast<const T*>(p.dout)[j]) * load_one(p.weight, p.wdtype, i) - xh * c);
    if (p.dstream) ds += to_f32(static_cast<const S*>(p.dstream)[j]);
    static_cast<T*>(p.dx)[j] = from_f32<T>(ds);
    if (p.dresidual) static_cast<S*>(p.dresidual)[j] = from_f32<S>(ds);
  }
}

template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) weight_grad(mko_resnorm_params p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.features) return;
  double sum = 0.0;
  for (int64_t row = 0; row < p.rows; ++row) {
    const int64_t j = row * p.features + i;
    sum += to_f32(static_cast<const T*>(p.dout)[j]) * (to_f32(static_cast<const S*>(p.stream)[j]) * p.rstd[row]);
  }
  p.dweight[i] = static_cast<float>(sum);
}

bool half_or_float(int32_t dtype) { return dtype == MKO_F32 || dtype == MKO_F16 || dtype == MKO_BF16; }

int check(const mko_resnorm_params* p, const char* what) {
  if (!p || p->rows < 0 || p->features < 0) {
    mko_set_error("%s: params is NULL or a size is negative", what);
    return MKO_EINVAL;
  }
  if (!half_or_float(p->dtype) || !half_or_float(p->stream_dtype) || !half_or_float(p->wdtype)) {
    mko_set_error("%s: dtype, stream_dtype and wdtype must be float32, float16 or bfloat16", what);
    return MKO_EINVAL;
  }
  if (p->stream_dtype != p->dtype && p->stream_dtype != MKO_F32) {
    mko_set_error("%s: the stream is of x's dtype or float32", what);
    return MKO_EINVAL;
  }
  if (p->rows > 0x7fffff) {
    mko_set_error("%s: rows is at most 2^23 - 1", what);
    return MKO_EUNSUPPORTED;
  }
  return MKO_OK;
}

template <typename T, typename S>
void launch_fwd(const mko_resnorm_params& p, hipStream_t s) {
  MKO_TIMED("resnorm_fwd", s, forward<T, S><<<static_cast<unsigned>(p.rows), kThreads, 0, s>>>(p));
}

template <typename T, typename S>
void launch_bwd(const mko_resnorm_params& p, hipStream_t s) {
  MKO_TIMED("resnorm_bwd", s, backward<T, S><<<static_cast<unsigned>(p.rows), kThreads, 0, s>>>(p));
  if (p.dweight)
    MKO_TIMED("resnorm_bwd_weight", s,
              weight_grad<T, S><<<static_cast<unsigned>(cdiv(p.features, kThreads)), kThreads, 0, s>>>(p));
}

}  // namespace
}  // namespace resnorm
}  // namespace mko

using namespace mko;

extern "C" size_t mko_sizeof_resnorm_params(void) { return sizeof(mko_resnorm_params); }

extern "C" int mko_resnorm_fwd(const mko_resnorm_params* p, void* stream) {
  const int st = resnorm::check(p, "resnorm_fwd");
  if (st != MKO_OK) return st;
  if (p->rows == 0 || p->features == 0) return MKO_OK;
  if (!p->x || !p->weight || (!p->out && !p->q) || (p->q && !p->q_scale) || (p->residual && !p->stream)) {
    mko_set_error("resnorm_fwd: x, weight, out (or q and q_scale), and stream with a residual are required");
    return MKO_EINVAL;
  }
  if (!p->residual && p->stream_dtype != p->dtype) {
    mko_set_error("resnorm_fwd: without a residual the stream is x, of its dtype");
    return MKO_EINVAL;
  }
  if (p->q && p->q_stride < p->features) {
    mko_set_error("resnorm_fwd: q_stride is smaller than features");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = p->stream_dtype == MKO_F32;
  if (p->dtype == MKO_F32)
    resnorm::launch_fwd<float, float>(*p, s);
  else if (p->dtype == MKO_BF16)
    wide ? resnorm::launch_fwd<bf16, float>(*p, s) : resnorm::launch_fwd<bf16, bf16>(*p, s);
  else
    wide ? resnorm::launch_fwd<_Float16, float>(*p, s) : resnorm::launch_fwd<_Float16, _Float16>(*p, s);
  return mko_check_launch("resnorm_fwd");
}

extern "C" size_t mko_resnorm_bwd_workspace_size(const mko_resnorm_params* p) {
  (void)p;
  return 0;
}

extern "C" int mko_resnorm_bwd(const mko_resnorm_params* p, void* stream) {
  const int st = resnorm::check(p, "resnorm_bwd");
  if (st != MKO_OK) return st;
  if (p->rows == 0 || p->features == 0) return MKO_OK;  // the caller zero-fills dweight
  if (!p->stream || !p->weight || !p->rstd || !p->dout || !p->dx) {
    mko_set_error("resnorm_bwd: stream, weight, rstd, dout and dx are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = p->stream_dtype == MKO_F32;
  if (p->dtype == MKO_F32)
    resnorm::launch_bwd<float, float>(*p, s);
  else if (p->dtype == MKO_BF16)
    wide ? resnorm::launch_bwd<bf16, float>(*p, s) : resnorm::launch_bwd<bf16, bf16>(*p, s);
  else
    wide ? resnorm::launch_bwd<_Float16, float>(*p, s) : resnorm::launch_bwd<_Float16, _Float16>(*p, s);
  return mko_check_launch("resnorm_bwd");
}
