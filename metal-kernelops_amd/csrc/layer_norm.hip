// Layer norm of the residual stream for gfx950: stream = x + residual, out = xh weight + bias with
// xh = (stream - mu) r, mu the row's mean and r = 1 / sqrt(mean((stream - mu)^2) + eps).
// Backward, with gw = dout weight:
//   ds = r (gw - mean(gw) - xh mean(gw xh)) + dstream
//   dweight = sum over rows of dout xh,  dbias = sum over rows of dout
//
// A team of lanes owns a row and holds it in registers from the load to the store, NV vectors of 16
// bytes of x a lane: a quarter or half of a wave for narrow rows, else whole waves.  The variance is
// that of the differences from the mean, in a second pass over the registers.  The backward's teams
// walk rows, with the next row's loads in flight, and keep dweight and dbias of their columns in
// registers; a workgroup adds its teams' in order and writes one row of partial sums.
#include <algorithm>

#include "common.hpp"
#include "io.hpp"
#include "rows.hpp"

namespace mko {
namespace layernorm {
namespace {

constexpr int kThreads = 256;       // workgroup of teams of up to four waves, forward
constexpr int kMostWaves = 16;      // waves of a team
constexpr int kMostVectors = 8;     // vectors a lane holds, forward
constexpr int kBwdThreads = 512;    // workgroup of teams of up to eight waves, backward
constexpr int kBwdMostVectors = 3;  // three arrays a vector, twice
constexpr int kBwdBlocks = 512;     // two workgroups a CU; more only add partial sums

struct Geo {
  int team;         // lanes of a team: 16, 32 or whole waves
  int64_t blocks;   // backward: workgroups
  int64_t rows_of;  // backward: rows a team walks
};

// Sum over the SUB lanes of a team inside a wave, in each of them.
template <int SUB>
__device__ __forceinline__ float team_sum(float v) {
  if constexpr (SUB == kWave) return wave_sum(v);
  v = row16_sum(v);
  if constexpr (SUB == 32) v += __shfl_xor(v, 16);
  return v;
}

// The same over teams of several waves, through `slots` of a float a wave; every wave of the workgroup
// comes here, and `slots` is free again after the next barrier but one.
template <int SUB>
__device__ __forceinline__ float team_sum(float v, float* slots, int team, int team_threads) {
  v = team_sum<SUB>(v);
  if (SUB < kWave || team_threads <= kWave) return v;
  const int wave = threadIdx.x >> 6, waves = team_threads >> 6;
  if ((threadIdx.x & (kWave - 1)) == 0) slots[wave] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < waves; ++i) v += slots[team * waves + i];
  return v;
}

// ------------------------------------------------------------------ forward

template <typename T, typename S, int SUB, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) forward(mko_layernorm_params p, Geo g) {
  constexpr int VEC = kVecOf<T>;
  __shared__ float slots[2][kMostWaves];
  const int threads = SUB < kWave ? SUB : g.team;
  const int team = SUB < kWave ? static_cast<int>(threadIdx.x) / SUB : uniform(static_cast<int>(threadIdx.x) / g.team);
  const int lt = threadIdx.x - team * threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / threads) + team;
  const bool live = row < p.rows;
  const int64_t n = live ? p.features : 0;
  const T* x = static_cast<const T*>(p.x) + (live ? row * p.x_stride : 0);
  const S* res = static_cast<const S*>(p.residual) + (live ? row * p.residual_stride : 0);

  Words<T, VEC> xr[NV];
  Words<S, VEC> rr[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t i = static_cast<int64_t>(lt + k * threads) * VEC;
    xr[k] = load_part<T, VEC>(x, i, n);
    if (p.residual) rr[k] = load_part<S, VEC>(res, i, n);
  }
  float w[NV][VEC];  // on its way while the sums meet
#pragma unroll
  for (int k = 0; k < NV; ++k)
    load_param_part<VEC>(p.weight, p.wdtype, static_cast<int64_t>(lt + k * threads) * VEC, p.features, w[k]);
  float v[NV][VEC], sum = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    unpack_words<T, VEC>(xr[k].w, v[k]);
    if (p.residual) {
      float r[VEC];
      unpack_words<S, VEC>(rr[k].w, r);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k][e] = to_f32(from_f32<S>(v[k][e] + r[e]));
      store_part<S, VEC>(static_cast<S*>(p.stream) + row * p.features, static_cast<int64_t>(lt + k * threads) * VEC, n, v[k]);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += v[k][e];
  }
  const double inv_n = 1.0 / static_cast<double>(p.features);
  const float mu = static_cast<float>(team_sum<SUB>(sum, slots[0], team, threads) * inv_n);
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t i = static_cast<int64_t>(lt + k * threads) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[k][e] -= mu;
      ss += i + e < n ? v[k][e] * v[k][e] : 0.0f;
    }
  }
  ss = team_sum<SUB>(ss, slots[1], team, threads);
  if (!live) return;
  const float r = inverse_norm(ss, inv_n, p.eps);
  if (lt == 0 && p.stats) {
    p.stats[2 * row] = mu;
    p.stats[2 * row + 1] = r;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int64_t i = static_cast<int64_t>(lt + k * threads) * VEC;
    float b[VEC], o[VEC];
    if (p.bias) load_param_part<VEC>(p.bias, p.bdtype, i, p.features, b);
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = v[k][e] * r * w[k][e] + (p.bias ? b[e] : 0.0f);
    store_part<T, VEC>(static_cast<T*>(p.out) + row * p.features, i, n, o);
  }
}

// The stream's value at (row, i): x + residual rounded to the stream's type.
template <typename T, typename S>
__device__ __forceinline__ float stream_at(const mko_layernorm_params& p, int64_t row, int64_t i) {
  const float x = to_f32(static_cast<const T*>(p.x)[row * p.x_stride + i]);
  if (!p.residual) return x;
  return to_f32(from_f32<S>(x + to_f32(static_cast<const S*>(p.residual)[row * p.residual_stride + i])));
}

__device__ __forceinline__ float block_sum(float v, float* slots) {  // of 1024 threads
  v = wave_sum(v);
  if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < 16; ++w) v += slots[w];
  return v;
}

// Rows wider than a team's registers: a workgroup walks the row three times.
template <typename T, typename S>
__global__ void __launch_bounds__(1024) forward_wide(mko_layernorm_params p) {
  __shared__ float slots[2][16];
  const int64_t row = blockIdx.x;
  const double inv_n = 1.0 / static_cast<double>(p.features);
  float sum = 0.0f, ss = 0.0f;
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float s = stream_at<T, S>(p, row, i);
    if (p.residual) static_cast<S*>(p.stream)[row * p.features + i] = from_f32<S>(s);
    sum += s;
  }
  const float mu = static_cast<float>(block_sum(sum, slots[0]) * inv_n);
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float d = stream_at<T, S>(p, row, i) - mu;
    ss += d * d;
  }
  const float r = inverse_norm(block_sum(ss, slots[1]), inv_n, p.eps);
  if (threadIdx.x == 0 && p.stats) {
    p.stats[2 * row] = mu;
    p.stats[2 * row + 1] = r;
  }
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float v = (stream_at<T, S>(p, row, i) - mu) * r * load_one(p.weight, p.wdtype, i);
    static_cast<T*>(p.out)[row * p.features + i] = from_f32<T>(v + (p.bias ? load_one(p.bias, p.bdtype, i) : 0.0f));
  }
}

// ------------------------------------------------------------------ backward

// A row's vectors on their way, and its statistics.
template <typename T, typename S, int NV>
struct Row {
  Words<T, kVecOf<T>> g[NV];
  Words<S, kVecOf<T>> s[NV], h[NV];
  float mu, r;
};

template <typename T, typename S, int SUB, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) backward(mko_layernorm_params p, Geo g, float* part) {
  constexpr int VEC = kVecOf<T>;
  __shared__ float slots[2][2][THREADS / kWave];
  extern __shared__ float columns[];  // a team's dweight and dbias
  const int threads = SUB < kWave ? SUB : g.team;
  const int teams = blockDim.x / threads;
  const int team = SUB < kWave ? static_cast<int>(threadIdx.x) / SUB : uniform(static_cast<int>(threadIdx.x) / g.team);
  const int lt = threadIdx.x - team * threads;
  const float inv_n = 1.0f / static_cast<float>(p.features);

  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_param_part<VEC>(p.weight, p.wdtype, static_cast<int64_t>(lt + k * threads) * VEC, p.features, w[k]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.0f;
  }
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * teams + team) * g.rows_of;
  auto load = [&](Row<T, S, NV>& a, int64_t it) {
    const int64_t row = first + it;
    const bool live = it < g.rows_of && row < p.rows;
    const int64_t n = live ? p.features : 0, base = live ? row * p.features : 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * threads) * VEC;
      a.g[k] = load_part<T, VEC>(static_cast<const T*>(p.dout) + base, i, n);
      a.s[k] = load_part<S, VEC>(static_cast<const S*>(p.stream) + base, i, n);
      if (p.dstream) a.h[k] = load_part<S, VEC>(static_cast<const S*>(p.dstream) + base, i, n);
    }
    a.mu = live ? p.stats[2 * row] : 0.0f;
    a.r = live ? p.stats[2 * row + 1] : 0.0f;
  };
  Row<T, S, NV> next;
  load(next, 0);
  for (int64_t it = 0; it < g.rows_of; ++it) {  // every team makes every turn: they meet in it
    const Row<T, S, NV> a = next;
    load(next, it + 1);
    const int64_t row = first + it;
    const bool live = row < p.rows;
    const int64_t n = live ? p.features : 0, base = live ? row * p.features : 0;
    float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float dy[VEC], s[VEC];
      unpack_words<T, VEC>(a.g[k].w, dy);
      unpack_words<S, VEC>(a.s[k].w, s);
      const int count = static_cast<int>(p.features) - (lt + k * threads) * VEC;  // features from this vector on
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = (s[e] - a.mu) * a.r, gw = dy[e] * w[k][e];
        c1 += gw;
        c2 += e < count ? gw * xh : 0.0f;  // beyond the row gw is zero, but -mu r may be infinite
        dw[k][e] += dy[e] * xh;
        db[k][e] += dy[e];
      }
    }
    if (SUB < kWave || threads <= kWave) {
      c1 = team_sum<SUB>(c1);
      c2 = team_sum<SUB>(c2);
    } else {
      c1 = team_sum<SUB>(c1);
      c2 = team_sum<SUB>(c2);
      const int wave = threadIdx.x >> 6, waves = threads >> 6;
      auto& meet = slots[it & 1];  // written again two turns on, past the turn between's barrier
      if ((threadIdx.x & (kWave - 1)) == 0) {
        meet[0][wave] = c1;
        meet[1][wave] = c2;
      }
      __syncthreads();
      c1 = c2 = 0.0f;
      for (int i = 0; i < waves; ++i) {
        c1 += meet[0][team * waves + i];
        c2 += meet[1][team * waves + i];
      }
    }
    c1 *= inv_n;
    c2 *= inv_n;
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * threads) * VEC;
      float dy[VEC], s[VEC], o[VEC];
      unpack_words<T, VEC>(a.g[k].w, dy);
      unpack_words<S, VEC>(a.s[k].w, s);
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = a.r * (dy[e] * w[k][e] - c1 - (s[e] - a.mu) * a.r * c2);
      if (p.dstream) {
        float h[VEC];
        unpack_words<S, VEC>(a.h[k].w, h);
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] += h[e];
      }
      store_part<T, VEC>(static_cast<T*>(p.dx) + base, i, n, o);
      if (p.dresidual) store_part<S, VEC>(static_cast<S*>(p.dresidual) + base, i, n, o);
    }
  }
  if (!part) return;
  if constexpr (SUB < kWave) {  // the teams of a wave first
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if constexpr (SUB == 16) {
          dw[k][e] += __shfl_xor(dw[k][e], 16);
          db[k][e] += __shfl_xor(db[k][e], 16);
        }
        dw[k][e] += __shfl_xor(dw[k][e], 32);
        db[k][e] += __shfl_xor(db[k][e], 32);
      }
    }
  }
  // then the waves', or the wider teams', in their order
  const int groups = SUB < kWave ? blockDim.x / kWave : teams;
  const int group = SUB < kWave ? threadIdx.x / kWave : team;
  const bool mine = SUB == kWave || static_cast<int>(threadIdx.x & (kWave - 1)) < SUB;
  for (int t = 0; t < groups; ++t) {
    if (groups > 1) __syncthreads();
    if (group != t || !mine) continue;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int64_t i = static_cast<int64_t>(lt + k * threads) * VEC;
      if (i >= p.features) continue;
      float s[2][VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const bool in = t && i + e < p.features;
        s[0][e] = (in ? columns[i + e] : 0.0f) + dw[k][e];
        s[1][e] = (in ? columns[p.features + i + e] : 0.0f) + db[k][e];
      }
      if (t + 1 < groups) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (i + e < p.features) {
            columns[i + e] = s[0][e];
            columns[p.features + i + e] = s[1][e];
          }
      } else {
        float* to = part + blockIdx.x * 2 * p.features;
        store_part<float, VEC>(to, i, p.features, s[0]);
        store_part<float, VEC>(to + p.features, i, p.features, s[1]);
      }
    }
  }
}

// Sums of the workgroups' rows of 2 * features partial sums, on a grid of two axes: 2^32 threads, the most that one
// has, are 2^26 features.
constexpr int64_t kFinishColumns = 1 << 16;  // workgroups of 32 sums in a row of the grid
__global__ void __launch_bounds__(kColumnThreads) finish(const float* part, int64_t blocks, int64_t features, float* dweight,
                                                         float* dbias) {
  const int64_t i = (blockIdx.y * kFinishColumns + blockIdx.x) * 32 + (threadIdx.x & 31);
  const float s = column_sum(part, blocks, 2 * features, i);
  if (threadIdx.x >= 32 || i >= 2 * features) return;
  if (i < features) {
    if (dweight) dweight[i] = s;
  } else if (dbias) {
    dbias[i - features] = s;
  }
}

// Rows wider than a team's registers.
template <typename T, typename S>
__global__ void __launch_bounds__(1024) backward_wide(mko_layernorm_params p) {
  __shared__ float slots[2][16];
  const int64_t row = blockIdx.x;
  const float mu = p.stats[2 * row], r = p.stats[2 * row + 1];
  float c1 = 0.0f, c2 = 0.0f;
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const float xh = (to_f32(static_cast<const S*>(p.stream)[row * p.features + i]) - mu) * r;
    const float gw = to_f32(static_cast<const T*>(p.dout)[row * p.features + i]) * load_one(p.weight, p.wdtype, i);
    c1 += gw;
    c2 += gw * xh;
  }
  c1 = block_sum(c1, slots[0]) / static_cast<float>(p.features);
  c2 = block_sum(c2, slots[1]) / static_cast<float>(p.features);
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) {
    const int64_t j = row * p.features + i;
    const float xh = (to_f32(static_cast<const S*>(p.stream)[j]) - mu) * r;
    float ds = r * (to_f32(static_cast<const T*>(p.dout)[j]) * load_one(p.weight, p.wdtype, i) - c1 - xh * c2);
    if (p.dstream) ds += to_f32(static_cast<const S*>(p.dstream)[j]);
    static_cast<T*>(p.dx)[j] = from_f32<T>(ds);
    if (p.dresidual) static_cast<S*>(p.dresidual)[j] = from_f32<S>(ds);
  }
}

// Rows [128 y, 128 y + 128) of the sums of dweight and dbias, for rows wider than a team's registers.
constexpr int kWideRows = 128;
template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) params_wide(mko_layernorm_params p, float* part) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.features) return;
  float dw = 0.0f, db = 0.0f;
  const int64_t last = min(p.rows, (static_cast<int64_t>(blockIdx.y) + 1) * kWideRows);
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * kWideRows; row < last; ++row) {
    const int64_t j = row * p.features + i;
    const float dy = to_f32(static_cast<const T*>(p.dout)[j]);
    dw += dy * ((to_f32(static_cast<const S*>(p.stream)[j]) - p.stats[2 * row]) * p.stats[2 * row + 1]);
    db += dy;
  }
  part[blockIdx.y * 2 * p.features + i] = dw;
  part[(blockIdx.y * 2 + 1) * p.features + i] = db;
}

// ------------------------------------------------------------------ the choice

int check(const mko_layernorm_params* p, const char* what) {
  if (!p || p->rows < 0 || p->features < 0) {
    mko_set_error("%s: params is NULL or a size is negative", what);
    return MKO_EINVAL;
  }
  if (!half_or_float(p->dtype) || !half_or_float(p->stream_dtype) || !half_or_float(p->wdtype) || !half_or_float(p->bdtype)) {
    mko_set_error("%s: dtype, stream_dtype, wdtype and bdtype must be float32, float16 or bfloat16", what);
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
  if (p->features >= 1 << 30) {
    mko_set_error("%s: features is below 2^30", what);
    return MKO_EUNSUPPORTED;
  }
  return MKO_OK;
}

int64_t vectors_of(const mko_layernorm_params* p) { return cdiv(p->features, p->dtype == MKO_F32 ? 4 : 8); }

// Vectors a lane holds, of the counts that are built; 0 if the row is too wide for `most`.
int depth(int64_t waves, int team_waves, int most) {
  const int64_t nv = cdiv(waves, team_waves);
  if (nv > most) return 0;
  return nv <= 5 ? static_cast<int>(nv) : 8;
}

template <typename T, typename S, int SUB, int NV>
void launch_fwd_n(const mko_layernorm_params& p, const Geo& g, hipStream_t s) {
  const int threads = g.team > kThreads ? g.team : kThreads / g.team * g.team;
  const unsigned grid = static_cast<unsigned>(cdiv(p.rows, threads / g.team));
  // Up to four waves may take more registers than sixteen, where four vectors a lane spill 14 to 17 registers, five 78 to 112
  // and eight 146 to 331.  Rows of more than 8192 features take those when a few hundred of them come: 400 x 10240 bf16
  // 15 us, 300 x 16384 23, and 25 beside a float32 stream.
  if (threads <= kThreads)
    MKO_TIMED("layernorm_fwd", s, forward<T, S, SUB, NV, kThreads><<<grid, threads, 0, s>>>(p, g));
  else
    MKO_TIMED("layernorm_fwd", s, forward<T, S, SUB, NV, kMostWaves * kWave><<<grid, threads, 0, s>>>(p, g));
}

// Rows of up to 16 or 32 vectors: four or two to a wave.  Wider ones: for few rows a vector a lane, for
// the shortest way from load to store (7 x 4096: 4.0 us, 10.1 with one wave a row); for many fewer waves
// to a row, down to one, where nothing has to meet, as long as 2048 waves, two a SIMD, have work (8192 x 2560
// bf16: 37 us, 4.5 TB/s, with five vectors a lane, 37 with two or three, 42 with one).
template <typename T, typename S>
void launch_fwd(const mko_layernorm_params& p, hipStream_t s) {
  const int64_t vectors = vectors_of(&p), waves = cdiv(vectors, kWave);
  if (vectors <= 16) return launch_fwd_n<T, S, 16, 1>(p, Geo{16, 0, 0}, s);
  if (vectors <= 32) return launch_fwd_n<T, S, 32, 1>(p, Geo{32, 0, 0}, s);
  int team = 1;
  while (team < kMostWaves && team < waves && (depth(waves, team, kMostVectors) == 0 || p.rows * team < 2048)) ++team;
  const Geo g{team * kWave, 0, 0};
  switch (depth(waves, team, kMostVectors)) {
    case 1: return launch_fwd_n<T, S, 64, 1>(p, g, s);
    case 2: return launch_fwd_n<T, S, 64, 2>(p, g, s);
    case 3: return launch_fwd_n<T, S, 64, 3>(p, g, s);
    case 4: return launch_fwd_n<T, S, 64, 4>(p, g, s);
    case 5: return launch_fwd_n<T, S, 64, 5>(p, g, s);
    case 8: return launch_fwd_n<T, S, 64, 8>(p, g, s);
    default: break;
  }
  MKO_TIMED("layernorm_fwd_wide", s, forward_wide<T, S><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p));
}

struct BwdPlan {
  int nv;  // vectors a lane holds; 0: the row is too wide for registers
  Geo g;
  int teams;
  size_t lds;
};

// One vector a lane as far as a team of sixteen waves goes: it leaves registers for more waves, which hide the
// loads better than more vectors do (8192 x 2560 bf16 42 us, 63 with two a lane and 68 with three; 1003 x 5120 beside
// a float32 stream 26, 28 and 56).  Wider rows take three in teams of up to eight, and
// spill 28 registers, beside a float32 stream 63 (float16) or 127: 8192 x 10240 bf16 187 us, 1003 x 12288 beside a float32
// stream 83.
BwdPlan bwd_plan(const mko_layernorm_params* p) {
  BwdPlan b{};
  const int64_t vectors = vectors_of(p), waves = cdiv(vectors, kWave);
  constexpr int kWaves = kBwdThreads / kWave;
  int team = static_cast<int>(std::min<int64_t>(waves, kMostWaves));
  b.nv = 1;
  if (waves > kMostWaves) {
    b.nv = kBwdMostVectors;
    team = static_cast<int>(cdiv(waves, kBwdMostVectors));
  }
  if (team > (b.nv == 1 ? kMostWaves : kWaves)) {
    b.nv = 0;
    b.g.blocks = cdiv(p->rows, kWideRows);
    return b;
  }
  b.g.team = vectors <= 16 ? 16 : vectors <= 32 ? 32 : team * kWave;
  b.teams = team > kWaves ? 1 : kWaves / team * (team * kWave / b.g.team);
  b.lds = b.teams > 1 ? static_cast<size_t>(p->features) * 2 * sizeof(float) : 0;
  b.g.rows_of = cdiv(cdiv(p->rows, b.teams), kBwdBlocks);
  b.g.blocks = cdiv(p->rows, b.teams * b.g.rows_of);
  return b;
}

template <typename T, typename S>
void launch_bwd(const mko_layernorm_params& p, const BwdPlan& b, hipStream_t s) {
  float* part = p.dweight || p.dbias ? static_cast<float*>(p.workspace) : nullptr;
  const unsigned grid = static_cast<unsigned>(b.g.blocks), threads = static_cast<unsigned>(b.teams * b.g.team);
  if (b.nv == 0) {
    MKO_TIMED("layernorm_bwd_wide", s, backward_wide<T, S><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p));
    if (part) {
      const dim3 wide(static_cast<unsigned>(cdiv(p.features, kThreads)), grid);
      MKO_TIMED("layernorm_bwd_params_wide", s, params_wide<T, S><<<wide, kThreads, 0, s>>>(p, part));
    }
  } else if (b.g.team == 16) {
    MKO_TIMED("layernorm_bwd", s, backward<T, S, 16, 1, kBwdThreads><<<grid, threads, b.lds, s>>>(p, b.g, part));
  } else if (b.g.team == 32) {
    MKO_TIMED("layernorm_bwd", s, backward<T, S, 32, 1, kBwdThreads><<<grid, threads, b.lds, s>>>(p, b.g, part));
  } else if (b.nv == 1 && threads <= kBwdThreads) {
    MKO_TIMED("layernorm_bwd", s, backward<T, S, 64, 1, kBwdThreads><<<grid, threads, b.lds, s>>>(p, b.g, part));
  } else if (b.nv == 1) {
    MKO_TIMED("layernorm_bwd", s, backward<T, S, 64, 1, kMostWaves * kWave><<<grid, threads, b.lds, s>>>(p, b.g, part));
  } else {
    MKO_TIMED("layernorm_bwd", s, backward<T, S, 64, kBwdMostVectors, kBwdThreads><<<grid, threads, b.lds, s>>>(p, b.g, part));
  }
  if (part) {
    const int64_t groups = cdiv(2 * p.features, 32);
    const dim3 columns(static_cast<unsigned>(std::min(groups, kFinishColumns)), static_cast<unsigned>(cdiv(groups, kFinishColumns)));
    MKO_TIMED("layernorm_bwd_finish", s, finish<<<columns, kColumnThreads, 0, s>>>(part, b.g.blocks, p.features, p.dweight, p.dbias));
  }
}

}  // namespace
}  // namespace layernorm
}  // namespace mko

using namespace mko;

extern "C" size_t mko_sizeof_layernorm_params(void) { return sizeof(mko_layernorm_params); }

extern "C" int mko_layernorm_fwd(const mko_layernorm_params* p, void* stream) {
  const int st = layernorm::check(p, "layernorm_fwd");
  if (st != MKO_OK) return st;
  if (p->rows == 0 || p->features == 0) return MKO_OK;
  if (!p->x || !p->weight || !p->out || (p->residual && !p->stream)) {
    mko_set_error("layernorm_fwd: x, weight, out, and stream with a residual are required");
    return MKO_EINVAL;
  }
  if (!p->residual && p->stream_dtype != p->dtype) {
    mko_set_error("layernorm_fwd: without a residual the stream is x, of its dtype");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool wide = p->stream_dtype == MKO_F32;
  if (p->dtype == MKO_F32)
    layernorm::launch_fwd<float, float>(*p, s);
  else if (p->dtype == MKO_BF16)
    wide ? layernorm::launch_fwd<bf16, float>(*p, s) : layernorm::launch_fwd<bf16, bf16>(*p, s);
  else
    wide ? layernorm::launch_fwd<_Float16, float>(*p, s) : layernorm::launch_fwd<_Float16, _Float16>(*p, s);
  return mko_check_launch("layernorm_fwd");
}

extern "C" size_t mko_layernorm_bwd_workspace_size(const mko_layernorm_params* p) {
  if (layernorm::check(p, "layernorm_bwd") != MKO_OK || p->rows == 0 || p->features == 0 || (!p->dweight && !p->dbias))
    return 0;
  return static_cast<size_t>(layernorm::bwd_plan(p).g.blocks * p->features) * 2 * sizeof(float);
}

extern "C" int mko_layernorm_bwd(const mko_layernorm_params* p, void* stream) {
  const int st = layernorm::check(p, "layernorm_bwd");
  if (st != MKO_OK) return st;
  if (p->rows == 0 || p->features == 0) return MKO_OK;  // the caller zero-fills dweight and dbias
  if (!p->stream || !p->weight || !p->stats || !p->dout || !p->dx) {
    mko_set_error("layernorm_bwd: stream, weight, stats, dout and dx are required");
    return MKO_EINVAL;
  }
  const size_t need = mko_layernorm_bwd_workspace_size(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) {
    mko_set_error("layernorm_bwd: workspace of %zu bytes needed, %zu given", need, p->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const layernorm::BwdPlan b = layernorm::bwd_plan(p);
  const bool wide = p->stream_dtype == MKO_F32;
  if (p->dtype == MKO_F32)
    layernorm::launch_bwd<float, float>(*p, b, s);
  else if (p->dtype == MKO_BF16)
    wide ? layernorm::launch_bwd<bf16, float>(*p, b, s) : layernorm::launch_bwd<bf16, bf16>(*p, b, s);
  else
    wide ? layernorm::launch_bwd<_Float16, float>(*p, b, s) : layernorm::launch_bwd<_Float16, _Float16>(*p, b, s);
  return mko_check_launch("layernorm_bwd");
}
