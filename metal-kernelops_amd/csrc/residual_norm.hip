// RMS norm of the residual stream for gfx950: stream = x + residual, out = stream r weight, with
// r = 1 / sqrt(mean(stream^2) + eps); or the same in 8 bits with a scale per row.
// Backward, with gw = dout weight and xh = stream r:
//   ds = r (gw - xh mean(gw xh)) + dstream,  dweight = sum over rows of dout xh
//
// A team of whole waves owns a row and holds it in registers from the load to the store, NV vectors
// of 16 bytes of x a thread, so that every operand crosses memory once.  The 8-bit output needs the
// row's largest |stream weight| beside its sum of squares; both come from one pass.  The backward's
// teams walk rows and keep dweight of their columns in registers; a workgroup adds its teams' in
// order and writes one row of partial sums.  Bound by memory: 8192 x 2560 bf16 forward 30 us (5.6 TB/s),
// backward 49 us (3.5 TB/s: a row's loads are issued after the row before it is stored) and 4 us for the
// 512 partial rows; in 8 bits 1999 x 2560 in 12 us.
#include "common.hpp"
#include "io.hpp"
#include "quantize.hpp"
#include "rows.hpp"

namespace mko {
namespace resnorm {
namespace {

constexpr int kThreads = 256;       // workgroup of teams of up to four waves, forward
constexpr int kMostWaves = 16;      // waves of a team
constexpr int kMostVectors = 8;     // vectors a thread holds, forward
constexpr int kBwdThreads = 512;
constexpr int kBwdMostVectors = 3;  // with five arrays a vector, more would leave one wave a SIMD
constexpr int kBwdBlocks = 512;     // two workgroups a CU; more only add partial sums

struct Geo {
  int team;         // threads of a team
  int64_t blocks;   // backward: workgroups
  int64_t rows_of;  // backward: rows a team walks
};

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

// ------------------------------------------------------------------ forward

template <typename T, typename S, int NV, bool Q>
__global__ void __launch_bounds__(kMostWaves * kWave) forward(mko_resnorm_params p, Geo g) {
  constexpr int VEC = kVecOf<T>;
  __shared__ float slots[kMostWaves];
  __shared__ uint32_t tops[kMostWaves];
  const int team = uniform(static_cast<int>(threadIdx.x) / g.team);
  const int lt = threadIdx.x - team * g.team;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / g.team) + team;
  const bool live = row < p.rows;
  const int64_t n = live ? p.features : 0;
  const T* x = static_cast<const T*>(p.x) + (live ? row * p.x_stride : 0);
  const S* res = static_cast<const S*>(p.residual) + (live ? row * p.residual_stride : 0);

  Words<T, VEC> xr[NV];
  Words<S, VEC> rr[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t i = static_cast<int64_t>(lt + k * g.team) * VEC;
    xr[k] = load_part<T, VEC>(x, i, n);
    if (p.residual) rr[k] = load_part<S, VEC>(res, i, n);
  }
  float w[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k)
    load_param_part<VEC>(p.weight, p.wdtype, static_cast<int64_t>(lt + k * g.team) * VEC, p.features, w[k]);

  float v[NV][VEC], ss = 0.0f;
  uint32_t am = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    unpack_words<T, VEC>(xr[k].w, v[k]);
    if (p.residual) {
      float r[VEC];
      unpack_words<S, VEC>(rr[k].w, r);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k][e] = to_f32(from_f32<S>(v[k][e] + r[e]));
      store_part<S, VEC>(static_cast<S*>(p.stream) + row * p.features, static_cast<int64_t>(lt + k * g.team) * VEC, n,
                         v[k]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ss += v[k][e] * v[k][e];
      if (Q) am = max(am, abs_bits(v[k][e] * w[k][e]));
    }
  }
  ss = wave_sum(ss);
  if (Q) am = wave_max(am);
  if (g.team > kWave) {
    const int wave = threadIdx.x >> 6, waves = g.team >> 6;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      slots[wave] = ss;
      if (Q) tops[wave] = am;
    }
    __syncthreads();
    ss = 0.0f;
    for (int i = 0; i < waves; ++i) {
      ss += slots[team * waves + i];
      if (Q) am = max(am, tops[team * waves + i]);
    }
  }
  if (!live) return;
  const float r = inverse_norm(ss, 1.0 / static_cast<double>(p.features), p.eps);
  if (lt == 0 && p.rstd) p.rstd[row] = r;
  if constexpr (Q) {
    const RowScale q = row_scale(abs_bits(__uint_as_float(am) * r));
    if (lt == 0) p.q_scale[row] = q.scale;
    int8_t* out = p.q + row * p.q_stride;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * g.team) * VEC;
      int b[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) b[e] = quantise(v[k][e] * r * w[k][e], q.inv);
      store_bytes<VEC>(out, i, n, p.q_stride, b);
    }
    // whole vectors past the end, where the rows are padded by more than one
    for (int64_t i = cdiv(n, VEC) * VEC + lt; i < p.q_stride; i += g.team) out[i] = 0;
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = v[k][e] * r * w[k][e];
      store_part<T, VEC>(static_cast<T*>(p.out) + row * p.features, static_cast<int64_t>(lt + k * g.team) * VEC, n, o);
    }
  }
}

// Rows wider than a team's registers: a workgroup walks the row twice.
template <typename T, typename S>
__global__ void __launch_bounds__(1024) forward_wide(mko_resnorm_params p) {
  __shared__ float slots[16];
  __shared__ uint32_t tops[16];
  const int64_t row = blockIdx.x;
  float ss = 0.0f;
  uint32_t am = 0;
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float s = stream_at<T, S>(p, row, i);
    if (p.residual) static_cast<S*>(p.stream)[row * p.features + i] = from_f32<S>(s);
    ss += s * s;
    am = max(am, abs_bits(s * load_one(p.weight, p.wdtype, i)));
  }
  ss = wave_sum(ss);
  am = wave_max(am);
  if ((threadIdx.x & (kWave - 1)) == 0) {
    slots[threadIdx.x / kWave] = ss;
    tops[threadIdx.x / kWave] = am;
  }
  __syncthreads();
  ss = 0.0f;
  for (int w = 0; w < 16; ++w) {
    ss += slots[w];
    am = max(am, tops[w]);
  }
  const float r = inverse_norm(ss, 1.0 / static_cast<double>(p.features), p.eps);
  if (threadIdx.x == 0 && p.rstd) p.rstd[row] = r;
  const RowScale q = row_scale(abs_bits(__uint_as_float(am) * r));
  if (p.q && threadIdx.x == 0) p.q_scale[row] = q.scale;
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float v = stream_at<T, S>(p, row, i) * r * load_one(p.weight, p.wdtype, i);
    if (p.q)
      p.q[row * p.q_stride + i] = static_cast<int8_t>(quantise(v, q.inv));
    else
      static_cast<T*>(p.out)[row * p.features + i] = from_f32<T>(v);
  }
  if (p.q)
    for (int64_t i = p.features + threadIdx.x; i < p.q_stride; i += 1024) p.q[row * p.q_stride + i] = 0;
}

// ------------------------------------------------------------------ backward

template <typename T, typename S, int NV>
__global__ void __launch_bounds__(kBwdThreads) backward(mko_resnorm_params p, Geo g, float* part) {
  constexpr int VEC = kVecOf<T>;
  __shared__ float slots[2][kBwdThreads / kWave];
  extern __shared__ float columns[];  // a team's dweight
  const int teams = blockDim.x / g.team;
  const int team = uniform(static_cast<int>(threadIdx.x) / g.team);
  const int lt = threadIdx.x - team * g.team;
  const float inv_n = 1.0f / static_cast<float>(p.features);

  float w[NV][VEC], dw[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_param_part<VEC>(p.weight, p.wdtype, static_cast<int64_t>(lt + k * g.team) * VEC, p.features, w[k]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[k][e] = 0.0f;
  }
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * teams + team) * g.rows_of;
  for (int64_t it = 0; it < g.rows_of; ++it) {  // every team makes every turn: they meet in it
    const int64_t row = first + it;
    const bool live = row < p.rows;
    const int64_t n = live ? p.features : 0;
    const int64_t base = live ? row * p.features : 0;
    Words<T, VEC> gr[NV];
    Words<S, VEC> sr[NV], hr[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * g.team) * VEC;
      gr[k] = load_part<T, VEC>(static_cast<const T*>(p.dout) + base, i, n);
      sr[k] = load_part<S, VEC>(static_cast<const S*>(p.stream) + base, i, n);
    }
    if (p.dstream) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        hr[k] = load_part<S, VEC>(static_cast<const S*>(p.dstream) + base, static_cast<int64_t>(lt + k * g.team) * VEC, n);
    }
    const float r = live ? p.rstd[row] : 0.0f;
    float c = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float dy[VEC], s[VEC];
      unpack_words<T, VEC>(gr[k].w, dy);
      unpack_words<S, VEC>(sr[k].w, s);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float t = dy[e] * (s[e] * r);
        c += t * w[k][e];
        dw[k][e] += t;
      }
    }
    c = wave_sum(c);
    if (g.team > kWave) {
      const int wave = threadIdx.x >> 6, waves = g.team >> 6;
      float* meet = slots[it & 1];  // written again two turns on, past the turn between's barrier
      if ((threadIdx.x & (kWave - 1)) == 0) meet[wave] = c;
      __syncthreads();
      c = 0.0f;
      for (int i = 0; i < waves; ++i) c += meet[team * waves + i];
    }
    c *= inv_n;
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * g.team) * VEC;
      float dy[VEC], s[VEC], o[VEC];
      unpack_words<T, VEC>(gr[k].w, dy);
      unpack_words<S, VEC>(sr[k].w, s);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = r * (dy[e] * w[k][e] - (s[e] * r) * c);
      if (p.dstream) {
        float h[VEC];
        unpack_words<S, VEC>(hr[k].w, h);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] += h[e];
      }
      store_part<T, VEC>(static_cast<T*>(p.dx) + base, i, n, o);
      if (p.dresidual) store_part<S, VEC>(static_cast<S*>(p.dresidual) + base, i, n, o);
    }
  }
  if (!part) return;
  // the teams' sums in their order
  for (int t = 0; t < teams; ++t) {
    if (teams > 1) __syncthreads();
    if (team != t) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * g.team) * VEC;
      if (t + 1 < teams) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (i + e < p.features) columns[i + e] = (t ? columns[i + e] : 0.0f) + dw[k][e];
      } else {
        float s[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = (t && i + e < p.features ? columns[i + e] : 0.0f) + dw[k][e];
        store_part<float, VEC>(part + blockIdx.x * p.features, i, p.features, s);
      }
    }
  }
}

__global__ void __launch_bounds__(kColumnThreads) finish(const float* part, int64_t blocks, int64_t features,
                                                         float* dweight) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const float s = column_sum(part, blocks, features, i);
  if (threadIdx.x < 32 && i < features) dweight[i] = s;
}

// Rows wider than a team's registers.
template <typename T, typename S>
__global__ void __launch_bounds__(1024) backward_wide(mko_resnorm_params p) {
  __shared__ float slots[16];
  const int64_t row = blockIdx.x;
  const float r = p.rstd[row];
  float c = 0.0f;
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float xh = to_f32(static_cast<const S*>(p.stream)[row * p.features + i]) * r;
    c += xh * to_f32(static_cast<const T*>(p.dout)[row * p.features + i]) * load_one(p.weight, p.wdtype, i);
  }
  c = wave_sum(c);
  if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = c;
  __syncthreads();
  c = 0.0f;
  for (int w = 0; w < 16; ++w) c += slots[w];
  c /= static_cast<float>(p.features);
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const int64_t j = row * p.features + i;
    const float xh = to_f32(static_cast<const S*>(p.stream)[j]) * r;
    float ds = r * (to_f32(static_cast<const T*>(p.dout)[j]) * load_one(p.weight, p.wdtype, i) - xh * c);
    if (p.dstream) ds += to_f32(static_cast<const S*>(p.dstream)[j]);
    static_cast<T*>(p.dx)[j] = from_f32<T>(ds);
    if (p.dresidual) static_cast<S*>(p.dresidual)[j] = from_f32<S>(ds);
  }
}

// Rows [128 y, 128 y + 128) of dweight's sum, for rows wider than a team's registers.
constexpr int kWideRows = 128;
template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) weight_wide(mko_resnorm_params p, float* part) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.features) return;
  float sum = 0.0f;
  const int64_t last = min(p.rows, (static_cast<int64_t>(blockIdx.y) + 1) * kWideRows);
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * kWideRows; row < last; ++row) {
    const int64_t j = row * p.features + i;
    sum += to_f32(static_cast<const T*>(p.dout)[j]) * (to_f32(static_cast<const S*>(p.stream)[j]) * p.rstd[row]);
  }
  part[blockIdx.y * p.features + i] = sum;
}

// ------------------------------------------------------------------ the choice

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
  if (p->rows >= 1 << 22) {
    mko_set_error("%s: rows is below 2^22", what);
    return MKO_EUNSUPPORTED;
  }
  return MKO_OK;
}

int64_t vector_waves(const mko_resnorm_params* p) {  // waves that hold a row at one vector a thread
  return cdiv(p->features, (p->dtype == MKO_F32 ? 4 : 8) * kWave);
}

// Vectors a thread holds, of the counts that are built; 0 if the row is too wide for `most`.
int depth(int64_t waves, int team_waves, int most) {
  const int64_t nv = cdiv(waves, team_waves);
  if (nv > most) return 0;
  return nv <= 5 ? static_cast<int>(nv) : 8;
}

template <typename T, typename S, int NV>
void launch_fwd_n(const mko_resnorm_params& p, const Geo& g, hipStream_t s) {
  const int threads = g.team > kThreads ? g.team : kThreads / g.team * g.team;
  const unsigned grid = static_cast<unsigned>(cdiv(p.rows, threads / g.team));
  if (p.q)
    MKO_TIMED("resnorm_int8", s, forward<T, S, NV, true><<<grid, threads, 0, s>>>(p, g));
  else
    MKO_TIMED("resnorm_fwd", s, forward<T, S, NV, false><<<grid, threads, 0, s>>>(p, g));
}

// Few rows: a vector a thread, for the shortest way from load to store.  Many rows: fewer waves to a
// row, down to one, where nothing has to meet; as long as 2048 waves, two a SIMD, have work.
template <typename T, typename S>
void launch_fwd(const mko_resnorm_params& p, hipStream_t s) {
  const int64_t waves = vector_waves(&p);
  int team = 1;
  while (team < kMostWaves && team < waves && (depth(waves, team, kMostVectors) == 0 || p.rows * team < 2048)) ++team;
  const int nv = depth(waves, team, kMostVectors);
  Geo g{team * kWave, 0, 0};
  switch (nv) {
    case 1: return launch_fwd_n<T, S, 1>(p, g, s);
    case 2: return launch_fwd_n<T, S, 2>(p, g, s);
    case 3: return launch_fwd_n<T, S, 3>(p, g, s);
    case 4: return launch_fwd_n<T, S, 4>(p, g, s);
    case 5: return launch_fwd_n<T, S, 5>(p, g, s);
    case 8: return launch_fwd_n<T, S, 8>(p, g, s);
    default: break;
  }
  MKO_TIMED("resnorm_fwd_wide", s, forward_wide<T, S><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p));
}

struct BwdPlan {
  int nv;  // 0: the row is too wide for registers
  Geo g;
  int teams;
  size_t lds;
};

BwdPlan bwd_plan(const mko_resnorm_params* p) {
  BwdPlan b{};
  const int64_t waves = vector_waves(p);
  constexpr int kWaves = kBwdThreads / kWave;
  int team = 1;
  while (team < kWaves && depth(waves, team, kBwdMostVectors) == 0) ++team;
  b.nv = depth(waves, team, kBwdMostVectors);
  if (b.nv == 0) {
    b.g.blocks = cdiv(p->rows, kWideRows);
    return b;
  }
  b.g.team = team * kWave;
  b.teams = kWaves / team;
  b.lds = b.teams > 1 ? static_cast<size_t>(p->features) * sizeof(float) : 0;
  b.g.rows_of = cdiv(cdiv(p->rows, b.teams), kBwdBlocks);
  b.g.blocks = cdiv(p->rows, b.teams * b.g.rows_of);
  return b;
}

template <typename T, typename S>
void launch_bwd(const mko_resnorm_params& p, const BwdPlan& b, hipStream_t s) {
  float* part = p.dweight ? static_cast<float*>(p.workspace) : nullptr;
  const unsigned grid = static_cast<unsigned>(b.g.blocks), threads = static_cast<unsigned>(b.teams * b.g.team);
  switch (b.nv) {
    case 1: MKO_TIMED("resnorm_bwd", s, backward<T, S, 1><<<grid, threads, b.lds, s>>>(p, b.g, part)); break;
    case 2: MKO_TIMED("resnorm_bwd", s, backward<T, S, 2><<<grid, threads, b.lds, s>>>(p, b.g, part)); break;
    case 3: MKO_TIMED("resnorm_bwd", s, backward<T, S, 3><<<grid, threads, b.lds, s>>>(p, b.g, part)); break;
    default:
      MKO_TIMED("resnorm_bwd_wide", s, backward_wide<T, S><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p));
      if (part) {
        const dim3 wide(static_cast<unsigned>(cdiv(p.features, kThreads)), grid);
        MKO_TIMED("resnorm_bwd_weight_wide", s, weight_wide<T, S><<<wide, kThreads, 0, s>>>(p, part));
      }
  }
  if (part)
    MKO_TIMED("resnorm_bwd_finish", s,
              finish<<<static_cast<unsigned>(cdiv(p.features, 32)), kColumnThreads, 0, s>>>(part, b.g.blocks, p.features,
                                                                                            p.dweight));
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
  if (resnorm::check(p, "resnorm_bwd") != MKO_OK || p->rows == 0 || p->features == 0 || !p->dweight) return 0;
  return static_cast<size_t>(resnorm::bwd_plan(p).g.blocks * p->features) * sizeof(float);
}

extern "C" int mko_resnorm_bwd(const mko_resnorm_params* p, void* stream) {
  const int st = resnorm::check(p, "resnorm_bwd");
  if (st != MKO_OK) return st;
  if (p->rows == 0 || p->features == 0) return MKO_OK;  // the caller zero-fills dweight
  if (!p->stream || !p->weight || !p->rstd || !p->dout || !p->dx) {
    mko_set_error("resnorm_bwd: stream, weight, rstd, dout and dx are required");
    return MKO_EINVAL;
  }
  const size_t need = mko_resnorm_bwd_workspace_size(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) {
    mko_set_error("resnorm_bwd: workspace of %zu bytes needed, %zu given", need, p->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const resnorm::BwdPlan b = resnorm::bwd_plan(p);
  const bool wide = p->stream_dtype == MKO_F32;
  if (p->dtype == MKO_F32)
    resnorm::launch_bwd<float, float>(*p, b, s);
  else if (p->dtype == MKO_BF16)
    wide ? resnorm::launch_bwd<bf16, float>(*p, b, s) : resnorm::launch_bwd<bf16, bf16>(*p, b, s);
  else
    wide ? resnorm::launch_bwd<_Float16, float>(*p, b, s) : resnorm::launch_bwd<_Float16, _Float16>(*p, b, s);
  return mko_check_launch("resnorm_bwd");
}
