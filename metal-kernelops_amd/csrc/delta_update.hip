// One step of the gated delta rule (delta.hpp): per value row of the state,
//   e = v - a (S k),  S' = a S + beta e k,  y = scale (a (S q) + beta e (k . q)),  a = exp(log decay)
// Both dot products come from one pass over the row, which stays in registers between its load and
// its store, so the state crosses memory once each way; its bytes bound the kernel.  A row belongs to
// LANES lanes, a 16-byte vector each, and a wave walks NR groups of 64 / LANES rows, all loaded
// before the first is used.
#include "io.hpp"
#include "rows.hpp"

namespace mko {
namespace delta_update {
namespace {

// Sum over groups of LANES lanes, in every lane of the group.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (LANES >= 16) {
    v = row16_sum(v);
    if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
    if constexpr (LANES >= 64) v += __shfl_xor(v, 32);
  } else {
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xb1, 0xf, 0xf, false));
    v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4e, 0xf, 0xf, false));
    if constexpr (LANES >= 8) v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xf, 0xf, false));
  }
  return v;
}

template <typename S, int LANES, int NR, bool VEC>
__global__ void __launch_bounds__(256) step(mko_delta_update_params p, int64_t waves, int per_head) {
  constexpr int NE = kVecOf<S>, ROWS = kWave / LANES;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + uniform(threadIdx.x >> 6);
  if (wave >= waves) return;
  const int64_t bh = wave / per_head, b = bh / p.heads, h = bh % p.heads, kh = h / (p.heads / p.key_heads);
  const int lane = threadIdx.x & (kWave - 1), sub = lane % LANES, first = (wave % per_head) * (ROWS * NR) + lane / LANES;
  const int i0 = sub * NE, value = static_cast<int>(p.value);
  const S* s = static_cast<const S*>(p.state) + bh * p.value * p.key;
  S* to = static_cast<S*>(p.new_state) + bh * p.value * p.key;
  Words<S, NE> w[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int row = first + n * ROWS;
    const bool in = row < value;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[n].w[j] = 0u;
      if (in && i0 < p.key) load_words_nt(s + static_cast<int64_t>(row) * p.key + i0, w[n].w);
    } else {
      w[n] = load_part<S, NE>(s + static_cast<int64_t>(in ? row : 0) * p.key, i0, in ? p.key : 0);
    }
  }
  float k[NE], q[NE];
  const int64_t ko = b * p.k_stride_b + kh * p.k_stride_h, qo = b * p.q_stride_b + kh * p.q_stride_h;
  load_param_part<NE>(p.k, p.dtype, ko + i0, ko + p.key, k);
  load_param_part<NE>(p.q, p.dtype, qo + i0, qo + p.key, q);
  const float a = expf(load_one(p.log_decay, p.decay_dtype, bh)), beta = load_one(p.beta, p.beta_dtype, bh);
  float v[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int row = first + n * ROWS;
    v[n] = row < value ? load_one(p.v, p.dtype, b * p.v_stride_b + h * p.v_stride_h + row) : 0.0f;
  }
  float kq = 0.0f;
#pragma unroll
  for (int j = 0; j < NE; ++j) kq += k[j] * q[j];
  kq = group_sum<LANES>(kq);
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int row = first + n * ROWS;
    float f[NE], sk = 0.0f, sq = 0.0f;
    unpack_words<S, NE>(w[n].w, f);
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      sk += f[j] * k[j];
      sq += f[j] * q[j];
    }
    sk = group_sum<LANES>(sk);
    sq = group_sum<LANES>(sq);
    const float u = beta * (v[n] - a * sk);
#pragma unroll
    for (int j = 0; j < NE; ++j) f[j] = a * f[j] + u * k[j];
    if (row >= value) continue;
    if constexpr (VEC) {
      uint32_t o[4];
      pack_words<S, NE>(f, o);
      if (i0 < p.key) store_words_nt(to + static_cast<int64_t>(row) * p.key + i0, o);
    } else {
      store_part<S, NE>(to + static_cast<int64_t>(row) * p.key, i0, p.key, f);
    }
    if (sub == 0) store_one(p.y, p.dtype, bh * p.value + row, p.scale * (a * sq + u * kq));
  }
}

template <typename S, int LANES, int NR>
void launch_n(const mko_delta_update_params& p, hipStream_t s) {
  const int per_head = static_cast<int>(cdiv(p.value, kWave / LANES * NR));
  const int64_t waves = p.batch * p.heads * per_head;
  const unsigned grid = static_cast<unsigned>(cdiv(waves, 4));
  const bool vec = p.key % kVecOf<S> == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(p.new_state) % 16 == 0;
  if (vec)
    MKO_TIMED("delta_update", s, step<S, LANES, NR, true><<<grid, 256, 0, s>>>(p, waves, per_head));
  else
    MKO_TIMED("delta_update", s, step<S, LANES, NR, false><<<grid, 256, 0, s>>>(p, waves, per_head));
}

// Eight groups of rows a wave where that leaves 4096 waves, four a SIMD, or more: 256 sequences of 32 heads of
// 128 x 128 take 193 us (5.6 TB/s), with two groups 203.  One sequence of 16 heads takes 4.8 us with two, 7.5 with eight.
template <typename S, int LANES>
void launch(const mko_delta_update_params& p, hipStream_t s) {
  if (p.batch * p.heads * p.value * LANES / kWave >= 8 * 4096)
    launch_n<S, LANES, 8>(p, s);
  else
    launch_n<S, LANES, 2>(p, s);
}

template <typename S>
void launch(const mko_delta_update_params& p, hipStream_t s) {
  const int64_t vectors = cdiv(p.key, kVecOf<S>);
  if (vectors <= 4) return launch<S, 4>(p, s);
  if (vectors <= 8) return launch<S, 8>(p, s);
  if (vectors <= 16) return launch<S, 16>(p, s);
  if (vectors <= 32) return launch<S, 32>(p, s);
  launch<S, 64>(p, s);
}

}  // namespace
}  // namespace delta_update
}  // namespace mko

using namespace mko;

extern "C" size_t mko_sizeof_delta_update_params(void) { return sizeof(mko_delta_update_params); }

extern "C" int mko_delta_update(const mko_delta_update_params* p, void* stream) {
  if (!p || p->batch < 0 || p->key_heads < 0 || p->heads < 0 || p->key < 0 || p->value < 0) {
    mko_set_error("delta_update: params is NULL or a size is negative");
    return MKO_EINVAL;
  }
  for (int32_t d : {p->dtype, p->decay_dtype, p->beta_dtype, p->state_dtype})
    if (!half_or_float(d)) {
      mko_set_error("delta_update: dtypes must be float32, float16 or bfloat16");
      return MKO_EINVAL;
    }
  if (p->key_heads < 1 || p->heads % p->key_heads || p->key < 1) {
    mko_set_error("delta_update: a key axis, and key_heads that divides heads, are required");
    return MKO_EINVAL;
  }
  if (p->key > MKO_DELTA_MAX_KEY) {
    mko_set_error("delta_update: the key axis has at most %d elements", MKO_DELTA_MAX_KEY);
    return MKO_EUNSUPPORTED;
  }
  const int64_t most = int64_t(1) << 24;
  if (p->batch >= most || p->heads >= most || p->batch * p->heads >= most || p->value >= most ||
      p->batch * p->heads * cdiv(p->value, 8) >= most) {
    mko_set_error("delta_update: batch * heads * (groups of 8 values) must be below 2^24");
    return MKO_EUNSUPPORTED;
  }
  if (p->batch == 0 || p->heads == 0 || p->value == 0) return MKO_OK;
  if (!p->q || !p->k || !p->v || !p->log_decay || !p->beta || !p->state || !p->new_state || !p->y) {
    mko_set_error("delta_update: q, k, v, log_decay, beta, state, new_state and y are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->state_dtype == MKO_F32)
    delta_update::launch<float>(*p, s);
  else if (p->state_dtype == MKO_BF16)
    delta_update::launch<bf16>(*p, s);
  else
    delta_update::launch<_Float16>(*p, s);
  return mko_check_launch("delta_update");
}
