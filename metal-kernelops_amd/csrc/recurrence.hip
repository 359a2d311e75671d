// Gated linear recurrence for gfx950.
//
// Per channel, with rate = scale softplus(decay):
//   v = rate s(rg),  a = e^-v,  m = sqrt(1 - e^-2v),  h[t] = a h[t-1] + m s(ig) x
// Backward, with g[t] = dy[t] + a[t+1] g[t+1]:
//   dx = g m s(ig),  dig = g m x s(ig) (1 - s(ig)),  drg = dv v (1 - s(rg)),
//   dv = g (s(ig) x a^2 / m - a h[t-1]),  ddecay = scale s(decay) sum(dv s(rg))
#include "common.hpp"

namespace mko {
namespace recur {
namespace {

constexpr int kChunk = MKO_RECUR_CHUNK;
constexpr int kThreads = 256;

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// 1 - e^-2v from v and a = e^-v: below v = 1/8 a six-term series (truncation (2v)^6 / 5040, 5e-8
// relative), where 1 - a^2 would cancel.
__device__ __forceinline__ float one_minus_square(float v, float a) {
  const float w = 2.0f * v;
  const float s = w * (1.0f - w * (1.0f / 2) *
                  (1.0f - w * (1.0f / 3) * (1.0f - w * (1.0f / 4) * (1.0f - w * (1.0f / 5) * (1.0f - w * (1.0f / 6))))));
  return v < 0.125f ? s : 1.0f - a * a;
}

struct Step {
  float si, sr, v, a, m, rm;  // rm = 1 / m, kept finite where v is 0
};

__device__ __forceinline__ Step gates(float ig, float rg, float rate, bool reset) {
  Step s;
  s.si = sigmoid(ig);
  s.sr = sigmoid(rg);
  s.v = rate * s.sr;
  s.a = fast_exp(-s.v);
  const float om = one_minus_square(s.v, s.a);
  s.rm = __builtin_amdgcn_rsqf(fmaxf(om, 1e-37f));
  s.m = om * s.rm;
  if (reset) {  // nothing of the decay gate is used, a NaN in it included
    s.a = s.v = s.sr = 0.0f;
    s.m = 1.0f;
  }
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) forward(mko_recur_params p, int64_t chunks) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t b = blockIdx.y;
  if (d >= p.channels) return;
  const float rate = p.scale * softplus(p.decay[d]);
  float h = p.initial ? p.initial[b * p.channels + d] : 0.0f;
  for (int64_t t = 0; t < p.length; ++t) {
    const float x = to_f32(static_cast<const T*>(p.x)[b * p.x_stride_b + t * p.x_stride_t + d]);
    const float ig = to_f32(static_cast<const T*>(p.input_gate)[b * p.ig_stride_b + t * p.ig_stride_t + d]);
    const float rg = to_f32(static_cast<const T*>(p.decay_gate)[b * p.rg_stride_b + t * p.rg_stride_t + d]);
    const bool reset = p.reset && p.reset[b * p.length + t];
    const Step s = gates(ig, rg, rate, reset);
    h = (reset ? 0.0f : s.a * h) + s.m * s.si * x;  // a dropped state is not read, be it NaN
    static_cast<T*>(p.y)[(b * p.length + t) * p.channels + d] = from_f32<T>(h);
    if ((t + 1) % kChunk == 0 || t + 1 == p.length) p.states[(b * chunks + t / kChunk) * p.channels + d] = h;
  }
  if (p.final_state) p.final_state[b * p.channels + d] = h;
}

// hs: (batch, length, channels), the state before each step; part: (batch, channels).
template <typename T>
__global__ void __launch_bounds__(kThreads) backward(mko_recur_params p, float* hs, float* part) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t b = blockIdx.y;
  if (d >= p.channels) return;
  const float rate = p.scale * softplus(p.decay[d]);
  auto load = [&](int64_t t, float& x) {
    x = to_f32(static_cast<const T*>(p.x)[b * p.x_stride_b + t * p.x_stride_t + d]);
    const float ig = to_f32(static_cast<const T*>(p.input_gate)[b * p.ig_stride_b + t * p.ig_stride_t + d]);
    const float rg = to_f32(static_cast<const T*>(p.decay_gate)[b * p.rg_stride_b + t * p.rg_stride_t + d]);
    return gates(ig, rg, rate, p.reset && p.reset[b * p.length + t]);
  };
  float h = p.initial ? p.initial[b * p.channels + d] : 0.0f, x;
  for (int64_t t = 0; t < p.length; ++t) {
    hs[(b * p.length + t) * p.channels + d] = h;
    const Step s = load(t, x);
    h = (p.reset && p.reset[b * p.length + t] ? 0.0f : s.a * h) + s.m * s.si * x;
  }
  float g = p.dfinal ? p.dfinal[b * p.channels + d] : 0.0f, sum = 0.0f;
  for (int64_t t = p.length - 1; t >= 0; --t) {
    const int64_t i = (b * p.length + t) * p.channels + d;
    const Step s = load(t, x);
    g += to_f32(static_cast<const T*>(p.dy)[i]);
    const bool reset = p.reset && p.reset[b * p.length + t];
    const float dv = reset ? 0.0f : g * (s.si * x * s.a * s.a * s.rm - s.a * hs[i]);
    static_cast<T*>(p.dx)[i] = from_f32<T>(g * s.m * s.si);
    static_cast<T*>(p.dinput_gate)[i] = from_f32<T>(g * s.m * x * s.si * (1.0f - s.si));
    static_cast<T*>(p.ddecay_gate)[i] = from_f32<T>(dv * s.v * (1.0f - s.sr));
    sum += dv * s.sr;
    g = reset ? 0.0f : g * s.a;
  }
  if (p.dinitial) p.dinitial[b * p.channels + d] = g;
  part[b * p.channels + d] = sum;
}

__global__ void __launch_bounds__(kThreads) finish(mko_recur_params p, const float* part) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (d >= p.channels) return;
  float sum = 0.0f;
  for (int64_t b = 0; b < p.batch; ++b) sum += part[b * p.channels + d];
  p.ddecay[d] = sum * p.scale * softplus_grad(p.decay[d]);
}

template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) update(mko_recur_update_params p) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t b = blockIdx.y;
  if (d >= p.channels) return;
  const float rate = p.scale * softplus(p.decay[d]);
  const float x = to_f32(static_cast<const T*>(p.x)[b * p.x_stride + d]);
  const float ig = to_f32(static_cast<const T*>(p.input_gate)[b * p.ig_stride + d]);
  const float rg = to_f32(static_cast<const T*>(p.decay_gate)[b * p.rg_stride + d]);
  const Step s = gates(ig, rg, rate, false);
  const float h = s.a * to_f32(static_cast<const S*>(p.state)[b * p.channels + d]) + s.m * s.si * x;
  static_cast<S*>(p.new_state)[b * p.channels + d] = from_f32<S>(h);
  static_cast<T*>(p.y)[b * p.channels + d] = from_f32<T>(h);
}

bool half_or_float(int32_t dtype) { return dtype == MKO_F32 || dtype == MKO_F16 || dtype == MKO_BF16; }

int check(const mko_recur_params* p, const char* what) {
  if (!p) {
    mko_set_error("%s: params is NULL", what);
    return MKO_EINVAL;
  }
  if (p->batch < 0 || p->length < 0 || p->channels < 0) {
    mko_set_error("%s: negative size", what);
    return MKO_EINVAL;
  }
  if (!half_or_float(p->dtype)) {
    mko_set_error("%s: dtype must be float32, float16 or bfloat16", what);
    return MKO_EINVAL;
  }
  if (p->batch > 65535) {
    mko_set_error("%s: batch is at most 65535", what);
    return MKO_EUNSUPPORTED;
  }
  return MKO_OK;
}

bool empty(const mko_recur_params* p) { return p->batch == 0 || p->length == 0 || p->channels == 0; }

size_t hs_bytes(const mko_recur_params* p) {
  return static_cast<size_t>(p->batch * p->length * p->channels) * sizeof(float);
}

}  // namespace
}  // namespace recur
}  // namespace mko

using namespace mko;

extern "C" size_t mko_sizeof_recur_params(void) { return sizeof(mko_recur_params); }
extern "C" size_t mko_sizeof_recur_update_params(void) { return sizeof(mko_recur_update_params); }

extern "C" size_t mko_recur_states_size(const mko_recur_params* p) {
  if (recur::check(p, "recur_states_size") != MKO_OK || recur::empty(p)) return 0;
  return static_cast<size_t>(p->batch * recur::cdiv(p->length, recur::kChunk) * p->channels) * sizeof(float);
}

extern "C" size_t mko_recur_fwd_workspace_size(const mko_recur_params* p) {
  (void)p;
  return 0;
}

extern "C" int mko_recur_fwd(const mko_recur_params* p, void* stream) {
  int st = recur::check(p, "recur_fwd");
  if (st != MKO_OK) return st;
  if (recur::empty(p)) return MKO_OK;
  if (!p->x || !p->input_gate || !p->decay_gate || !p->decay || !p->y || !p->states) {
    mko_set_error("recur_fwd: x, both gates, decay, y and states are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t chunks = recur::cdiv(p->length, recur::kChunk);
  const dim3 grid(static_cast<unsigned>(recur::cdiv(p->channels, recur::kThreads)), static_cast<unsigned>(p->batch));
  if (p->dtype == MKO_F32)
    MKO_TIMED("recur_fwd", s, recur::forward<float><<<grid, recur::kThreads, 0, s>>>(*p, chunks));
  else if (p->dtype == MKO_BF16)
    MKO_TIMED("recur_fwd", s, recur::forward<bf16><<<grid, recur::kThreads, 0, s>>>(*p, chunks));
  else
    MKO_TIMED("recur_fwd", s, recur::forward<_Float16><<<grid, recur::kThreads, 0, s>>>(*p, chunks));
  return mko_check_launch("recur_fwd");
}

extern "C" size_t mko_recur_bwd_workspace_size(const mko_recur_params* p) {
  if (recur::check(p, "recur_bwd") != MKO_OK || recur::empty(p)) return 0;
  return recur::hs_bytes(p) + static_cast<size_t>(p->batch * p->channels) * sizeof(float);
}

extern "C" int mko_recur_bwd(const mko_recur_params* p, void* stream) {
  int st = recur::check(p, "recur_bwd");
  if (st != MKO_OK) return st;
  if (recur::empty(p)) return MKO_OK;
  if (!p->x || !p->input_gate || !p->decay_gate || !p->decay || !p->states || !p->dy || !p->dx || !p->dinput_gate ||
      !p->ddecay_gate) {
    mko_set_error("recur_bwd: x, both gates, decay, states, dy and their gradients are required");
    return MKO_EINVAL;
  }
  const size_t need = mko_recur_bwd_workspace_size(p);
  if (!p->workspace || p->workspace_bytes < need) {
    mko_set_error("recur_bwd: workspace of %zu bytes needed, %zu given", need, p->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  float* hs = static_cast<float*>(p->workspace);
  float* part = hs + p->batch * p->length * p->channels;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(recur::cdiv(p->channels, recur::kThreads)), static_cast<unsigned>(p->batch));
  if (p->dtype == MKO_F32)
    MKO_TIMED("recur_bwd", s, recur::backward<float><<<grid, recur::kThreads, 0, s>>>(*p, hs, part));
  else if (p->dtype == MKO_BF16)
    MKO_TIMED("recur_bwd", s, recur::backward<bf16><<<grid, recur::kThreads, 0, s>>>(*p, hs, part));
  else
    MKO_TIMED("recur_bwd", s, recur::backward<_Float16><<<grid, recur::kThreads, 0, s>>>(*p, hs, part));
  if (p->ddecay)
    MKO_TIMED("recur_bwd_finish", s, recur::finish<<<grid.x, recur::kThreads, 0, s>>>(*p, part));
  return mko_check_launch("recur_bwd");
}

namespace mko {
namespace recur {
namespace {
template <typename T>
void launch_update(const mko_recur_update_params& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(cdiv(p.channels, kThreads)), static_cast<unsigned>(p.batch));
  if (p.state_dtype == MKO_F32)
    MKO_TIMED("recur_update", s, update<T, float><<<grid, kThreads, 0, s>>>(p));
  else if (p.state_dtype == MKO_BF16)
    MKO_TIMED("recur_update", s, update<T, bf16><<<grid, kThreads, 0, s>>>(p));
  else
    MKO_TIMED("recur_update", s, update<T, _Float16><<<grid, kThreads, 0, s>>>(p));
}
}  // namespace
}  // namespace recur
}  // namespace mko

extern "C" int mko_recur_update(const mko_recur_update_params* p, void* stream) {
  if (!p || p->batch < 0 || p->channels < 0) {
    mko_set_error("recur_update: params is NULL or a size is negative");
    return MKO_EINVAL;
  }
  if (!recur::half_or_float(p->dtype) || !recur::half_or_float(p->state_dtype)) {
    mko_set_error("recur_update: dtype and state_dtype must be float32, float16 or bfloat16");
    return MKO_EINVAL;
  }
  if (p->batch > 65535) {
    mko_set_error("recur_update: batch is at most 65535");
    return MKO_EUNSUPPORTED;
  }
  if (p->batch == 0 || p->channels == 0) return MKO_OK;
  if (!p->x || !p->input_gate || !p->decay_gate || !p->decay || !p->state || !p->new_state || !p->y) {
    mko_set_error("recur_update: x, both gates, decay, state, new_state and y are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == MKO_F32)
    recur::launch_update<float>(*p, s);
  else if (p->dtype == MKO_BF16)
    recur::launch_update<bf16>(*p, s);
  else
    recur::launch_update<_Float16>(*p, s);
  return mko_check_launch("recur_update");
}
