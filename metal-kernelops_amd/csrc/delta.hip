// Gated delta rule, forward (delta.hpp has the formulas).
//
//   prep  per (batch, head, chunk): the decays' sums, T by blocked substitution in float32, and the
//         operands T and P (and their transposes, for the backward)
//   scan  per (batch, head, 16 W value columns), sequential over the chunks: S stays in float32
//         accumulators, and E and Y of the chunk come out of it on the way
#include "delta.hpp"

namespace mko {
namespace delta {
namespace {

__device__ uint4 zero_unit;  // where rows and columns outside come from

constexpr int kPitch = 68;  // of prep's float32 square

// 16 x 16 blocks of the float32 square in LDS as operands: four products over 16 indices, index
// 4 (l / 16) + r in the r-th.
struct Block {
  float v[4];
};
__device__ __forceinline__ Block block_rows(const float* a, int r0, int c0) {
  const float4 v = *reinterpret_cast<const float4*>(a + (r0 + lane_col()) * kPitch + c0 + 4 * lane_quad());
  return Block{{v.x, v.y, v.z, v.w}};
}
__device__ __forceinline__ Block block_columns(const float* a, int r0, int c0) {
  Block b;
#pragma unroll
  for (int r = 0; r < 4; ++r) b.v[r] = a[(r0 + 4 * lane_quad() + r) * kPitch + c0 + lane_col()];
  return b;
}
__device__ __forceinline__ void block_mma(f32x4& acc, const Block& a, const Block& b) {
#pragma unroll
  for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[r], b.v[r], acc, 0, 0, 0);
}
__device__ __forceinline__ Block block_of(const f32x4& acc) { return Block{{acc[0], acc[1], acc[2], acc[3]}}; }
__device__ __forceinline__ void block_store(float* a, int r0, int c0, const f32x4& acc) {
#pragma unroll
  for (int r = 0; r < 4; ++r) a[(r0 + 4 * lane_quad() + r) * kPitch + c0 + lane_col()] = -acc[r];
}

// T = (I + A)^-1 over A's strict lower triangle (64 x 64 in LDS), in place; blocks above the diagonal
// are neither read nor written.  Substitution inside the 16 x 16 diagonal blocks, then
// T21 = -T22 A21 T11 for blocks of 16 and of 32.  A Neumann product would take fewer steps, but
// cancels: with equal keys its terms grow as binomial coefficients.
__device__ __forceinline__ void invert(float* a) {
  const int wave = uniform(threadIdx.x >> 6);
  if (wave == 0) {
    const int b = 16 * lane_quad(), c = lane_col();
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = c == i ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        if (j >= i) continue;
        const float4 v = *reinterpret_cast<const float4*>(a + (b + i) * kPitch + b + j);
        s -= v.x * t[j];
        if (j + 1 < i) s -= v.y * t[j + 1];
        if (j + 2 < i) s -= v.z * t[j + 2];
        if (j + 3 < i) s -= v.w * t[j + 3];
      }
      t[i] = s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) a[(b + i) * kPitch + b + c] = t[i];
  }
  __syncthreads();
  if (wave < 2) {
    const int o = 32 * wave;
    f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
    block_mma(x, block_rows(a, o + 16, o), block_columns(a, o, o));
    block_mma(y, block_rows(a, o + 16, o + 16), block_of(x));
    block_store(a, o + 16, o, y);
  }
  __syncthreads();
  f32x4 x[2];
  const int j = 16 * wave;
  if (wave < 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[i] = f32x4{0, 0, 0, 0};
      if (wave == 0) block_mma(x[i], block_rows(a, 32 + 16 * i, 0), block_columns(a, 0, j));
      block_mma(x[i], block_rows(a, 32 + 16 * i, 16), block_columns(a, 16, j));
    }
  }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 y = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k <= i; ++k) block_mma(y, block_rows(a, 32 + 16 * i, 32 + 16 * k), block_of(x[k]));
      block_store(a, 32 + 16 * i, j, y);
    }
  }
  __syncthreads();
}

// Half h of the operand at `p`.
template <typename TM>
__device__ __forceinline__ void store_half(TM* p, int h, const float (&f)[4]) {
  uint32_t w[kWordsOf<TM, 4>];
  pack_words<TM, 4>(f, w);
  store_words(p + 8 * lane_id() + 4 * h, w);
}

// Wave w owns the row tile w of A and P.
template <typename TM, int KB, bool TRAIN>
__global__ void __launch_bounds__(256) prep(Geo g, Ptrs p) {
  __shared__ Tokens tok;
  __shared__ __align__(16) float a[kC * kPitch];
  const WgId id = wg_id(static_cast<int>(g.heads), static_cast<int>(g.chunks));
  const int64_t h = id.x, c = id.y, b = id.z;
  const int64_t at = (b * g.heads + h) * g.chunks + c, t0 = c * kC;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kC), g.length - t0));
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const TM* q = static_cast<const TM*>(p.q) + b * g.q_b + t0 * g.q_t + h / g.rep * g.q_h;
  const TM* k = static_cast<const TM*>(p.k) + b * g.k_b + t0 * g.k_t + h / g.rep * g.k_h;
  const int key = static_cast<int>(g.key);
  TM* lp = static_cast<TM*>(p.lower) + (2 * at + 1) * kSquare;              // P; T is ahead of it
  TM* up = TRAIN ? static_cast<TM*>(p.upper) + (2 * at + 1) * kSquare : lp;  // and their transposes

  if (wave == 0) {
    const int64_t i = (b * g.length + t0 + lane) * g.heads + h;
    float d = lane < rows ? load_one(p.decay, g.decay_dtype, i) : 0.0f;
    // a decay that clears the state, as -infinity does, with sums that stay finite; NaN stays NaN
    d = d < -1e4f ? -1e4f : d;
    double s = static_cast<double>(d) * 1.4426950408889634;
    for (int o = 1; o < kC; o *= 2) {
      const double u = __shfl_up(s, o);
      if (lane >= o) s += u;
    }
    const double last = __shfl(s, kC - 1);
    tok.c[lane] = s;
    tok.in[lane] = fast_exp2(static_cast<float>(s));
    tok.out[lane] = fast_exp2(static_cast<float>(last - s));
    tok.beta[lane] = lane < rows ? load_one(p.beta, g.beta_dtype, i) : 0.0f;
  }
  __syncthreads();
  {
    uint32_t* to = reinterpret_cast<uint32_t*>(p.tokens + at);
    const uint32_t* from = reinterpret_cast<const uint32_t*>(&tok);
    for (int i = threadIdx.x; i < static_cast<int>(sizeof(Tokens) / 4); i += 256) to[i] = from[i];
  }
  Frag<TM> kf[KB], qf[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    kf[kb] = frag_memory(k, g.k_t, 16 * wave, 32 * kb, rows, key);
    qf[kb] = frag_memory(q, g.q_t, 16 * wave, 32 * kb, rows, key);
  }
  const int tr = 16 * wave + 4 * lane_quad(), tc = 16 * wave + lane_col();  // this tile's tokens as rows and columns
  for (int j = 0; j <= wave; ++j) {
    f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0}, kq = {0, 0, 0, 0};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Frag<TM> o = j == wave ? kf[kb] : frag_memory(k, g.k_t, 16 * j, 32 * kb, rows, key);
      mma(kk, kf[kb], o);             // [t][s]
      mma(kq, o, qf[kb]);             // [s][t]
      if (TRAIN) mma(qk, qf[kb], o);  // [t][s]
    }
    const int sc = 16 * j + lane_col(), sr = 16 * j + 4 * lane_quad();  // the other tile's
    float pt[4], pp[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = tr + r, s = sr + r;
      const float m = t >= sc ? fast_exp2(static_cast<float>(tok.c[t] - tok.c[sc])) * tok.beta[sc] : 0.0f;
      a[t * kPitch + sc] = t > sc ? kk[r] * m : 0.0f;
      if (TRAIN) pt[r] = t >= sc ? g.scale * qk[r] * m : 0.0f;
      pp[r] = tc >= s ? g.scale * kq[r] * fast_exp2(static_cast<float>(tok.c[tc] - tok.c[s])) * tok.beta[s] : 0.0f;
    }
    store_half<TM>(lp + lower_at(wave, j / 2), j % 2, pp);
    if (TRAIN) store_half<TM>(up + upper_at(j, wave / 2), wave % 2, pt);
  }
  if (wave % 2 == 0) {  // the tile right of the diagonal completes a block
    const float none[4] = {0, 0, 0, 0};
    store_half<TM>(lp + lower_at(wave, wave / 2), 1, none);
    if (TRAIN) store_half<TM>(up + upper_at(wave + 1, wave / 2), 0, none);
  }
  __syncthreads();
  invert(a);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j / 2 <= wave / 2) {  // T's rows of tile `wave`, columns of tile j
      const float4 v = *reinterpret_cast<const float4*>(a + tc * kPitch + 16 * j + 4 * lane_quad());
      const bool in = j <= wave;
      const float f[4] = {in ? v.x : 0.0f, in ? v.y : 0.0f, in ? v.z : 0.0f, in ? v.w : 0.0f};
      store_half<TM>(lp - kSquare + lower_at(wave, j / 2), j % 2, f);
    }
    if (TRAIN && j / 2 >= wave / 2) {  // its columns of tile `wave`, rows of tile j
      float f[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) f[r] = j >= wave ? a[(16 * j + 4 * lane_quad() + r) * kPitch + tc] : 0.0f;
      store_half<TM>(up - kSquare + upper_at(wave, j / 2), j % 2, f);
    }
  }
}

// W waves of 16 value columns each.
template <typename TM, int KB, int W, bool TRAIN, bool FAST>
__global__ void __launch_bounds__(64 * W) scan(Geo g, Ptrs p, int parts) {
  constexpr int KP = 32 * KB, BV = 16 * W;
  typedef Feed<TM, KP, BV, W, FAST> Feeder;
  typedef Tile<TM, KP> KTile;
  __shared__ __align__(16) typename Feeder::Buf bufs[Feeder::kBufs];
  const WgId id = wg_id(parts, static_cast<int>(g.heads));
  const int64_t h = id.y, b = id.z, bh = b * g.heads + h;
  const int wave = uniform(threadIdx.x >> 6), col = lane_col(), quad = lane_quad();
  const int v0 = id.x * BV, vc = v0 + 16 * wave + col;  // the lane's column of S and E
  const int key = static_cast<int>(g.key), value = static_cast<int>(g.value);
  const TM* zeros = reinterpret_cast<const TM*>(&zero_unit);
  const Feeder feed{static_cast<const TM*>(p.k) + b * g.k_b + h / g.rep * g.k_h,
                    static_cast<const TM*>(p.q) + b * g.q_b + h / g.rep * g.q_h,
                    static_cast<const TM*>(p.v) + b * g.v_b + h * g.v_h + v0, g.k_t, g.q_t, g.v_t, g.length,
                    p.tokens + bh * g.chunks, static_cast<const TM*>(p.lower) + bh * g.chunks * 2 * kSquare, key, value - v0};

  f32x4 s[2 * KB];  // S transposed: [key][value]
#pragma unroll
  for (int i = 0; i < 2 * KB; ++i) s[i] = f32x4{0, 0, 0, 0};
  if (p.initial && vc < value) load_state<FAST>(s, p.initial, g.state_dtype, (bh * value + vc) * key, key);
  if (FAST && g.chunks > 0) feed.fetch(bufs, 0, wave, zeros);
  for (int64_t c = 0; c < g.chunks; ++c) {
    const int64_t at = bh * g.chunks + c, t0 = c * kC;
    Frag<TM> held[Feeder::kSquares ? 1 : 12];
    if constexpr (!Feeder::kSquares) {
#pragma unroll
      for (int i = 0; i < 12; ++i) held[i] = frag_at(feed.squares + (12 * c + i) * kFrag);
    }
    const typename Feeder::Buf& bf = feed.turn(bufs, c, c + 1, c + 1 < g.chunks, wave, zeros);
    auto square = [&](int which, int i, int j) {  // T, P
      if constexpr (Feeder::kSquares)
        return frag_at(bf.squares + which * kSquare + lower_at(i, j));
      else
        return held[6 * which + lower_at(i, j) / kFrag];
    };

    Frag<TM> so[KB];  // S as an operand over the keys
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) so[kb] = frag_of<TM>(s[2 * kb], s[2 * kb + 1]);
    if (TRAIN && vc < value)
      store_operands<TM, FAST>(static_cast<TM*>(p.states) + (at * value + vc) * key, key, so);
    // V - exp(c) K S0^T
    f32x4 e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 z = {0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) mma(z, KTile::rows(bf.k, 16 * i, 32 * kb), so[kb]);
      const f32x4 vv = Tile<TM, BV>::values(bf.v, 16 * i, 16 * wave);
      const float4 d = *reinterpret_cast<const float4*>(bf.in + 16 * i + 4 * quad);
      e[i] = f32x4{vv[0] - d.x * z[0], vv[1] - d.y * z[1], vv[2] - d.z * z[2], vv[3] - d.w * z[3]};
    }
    const Frag<TM> zo[2] = {frag_of<TM>(e[0], e[1]), frag_of<TM>(e[2], e[3])};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = f32x4{0, 0, 0, 0};
      f32x4 et = {0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j <= i / 2; ++j) {
        const Frag<TM> t = square(0, i, j);
        mma(e[i], t, zo[j]);
        if (TRAIN) mma(et, zo[j], t);  // [value][t], whose lanes hold four values of a token
      }
      if (TRAIN)
        store_four<TM, FAST>(static_cast<TM*>(p.e) + (at * kC + 16 * i + col) * value, v0 + 16 * wave + 4 * quad, value, et);
    }
    const Frag<TM> eo[2] = {frag_of<TM>(e[0], e[1]), frag_of<TM>(e[2], e[3])};
    // Y transposed, so that a lane holds four values of a token
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 y = {0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) mma(y, so[kb], KTile::rows(bf.q, 16 * i, 32 * kb));
      const float d = g.scale * bf.in[16 * i + col];
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] *= d;
#pragma unroll
      for (int j = 0; j <= i / 2; ++j) mma(y, eo[j], square(1, i, j));
      const int64_t t = t0 + 16 * i + col;
      if (t < g.length)
        store_four<TM, FAST>(static_cast<TM*>(p.y) + ((b * g.length + t) * g.heads + h) * value, v0 + 16 * wave + 4 * quad,
                             value, y);
    }
    // S' = exp(c_63) S0 + E^T (beta exp(c_63 - c) K)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 d = *reinterpret_cast<const float4*>(bf.out + 16 * i + 4 * quad);
      const float4 bt = *reinterpret_cast<const float4*>(bf.beta + 16 * i + 4 * quad);
      e[i] = f32x4{e[i][0] * (d.x * bt.x), e[i][1] * (d.y * bt.y), e[i][2] * (d.z * bt.z), e[i][3] * (d.w * bt.w)};
    }
    const Frag<TM> wo[2] = {frag_of<TM>(e[0], e[1]), frag_of<TM>(e[2], e[3])};
    const float last = bf.in[kC - 1];
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[i][r] *= last;
#pragma unroll
      for (int j = 0; j < 2; ++j) mma(s[i], KTile::keys_over_tokens(bf.k, 32 * j, i), wo[j]);
    }
  }
  if (p.final_state && vc < value) store_state<FAST>(p.final_state, g.state_dtype, (bh * value + vc) * key, key, s);
}

// ------------------------------------------------------------------ the choice

template <typename TM, int KB, bool TRAIN>
void launch(const Geo& g, const Ptrs& p, hipStream_t s) {
  constexpr int W = 2;
  const unsigned cells = static_cast<unsigned>(g.batch * g.heads * g.chunks);
  const int parts = static_cast<int>(cdiv(g.value, 16 * W));
  if (cells) MKO_TIMED("delta_prep", s, prep<TM, KB, TRAIN><<<cells, 256, 0, s>>>(g, p));
  const unsigned grid = static_cast<unsigned>(g.batch * g.heads * parts);
  if constexpr (sizeof(TM) == 2) {
    if (fast_rows(g, p)) {
      MKO_TIMED("delta_scan", s, scan<TM, KB, W, TRAIN, true><<<grid, 64 * W, 0, s>>>(g, p, parts));
      return;
    }
  }
  MKO_TIMED("delta_scan", s, scan<TM, KB, W, TRAIN, false><<<grid, 64 * W, 0, s>>>(g, p, parts));
}

template <typename TM, bool TRAIN>
void launch(const Geo& g, const Ptrs& p, hipStream_t s) {
  if (g.key <= 32) return launch<TM, 1, TRAIN>(g, p, s);
  if (g.key <= 64) return launch<TM, 2, TRAIN>(g, p, s);
  if (g.key <= 128) return launch<TM, 4, TRAIN>(g, p, s);
  return launch<TM, 8, TRAIN>(g, p, s);
}

template <typename TM>
void launch(const Geo& g, const Ptrs& p, bool train, hipStream_t s) {
  train ? launch<TM, true>(g, p, s) : launch<TM, false>(g, p, s);
}

}  // namespace

// ------------------------------------------------------------------ sizes

int make_geo(const mko_delta_params* prm, const char* what, Geo* g) {
  if (!prm || prm->batch < 0 || prm->length < 0 || prm->key_heads < 0 || prm->heads < 0 || prm->key < 0 || prm->value < 0) {
    mko_set_error("%s: params is NULL or a size is negative", what);
    return MKO_EINVAL;
  }
  for (int32_t d : {prm->dtype, prm->decay_dtype, prm->beta_dtype, prm->state_dtype})
    if (!half_or_float(d)) {
      mko_set_error("%s: dtypes must be float32, float16 or bfloat16", what);
      return MKO_EINVAL;
    }
  if (prm->key_heads < 1 || prm->heads % prm->key_heads || prm->key < 1) {
    mko_set_error("%s: a key axis, and key_heads that divides heads, are required", what);
    return MKO_EINVAL;
  }
  if (prm->key > MKO_DELTA_MAX_KEY) {
    mko_set_error("%s: the key axis has at most %d elements", what, MKO_DELTA_MAX_KEY);
    return MKO_EUNSUPPORTED;
  }
  // workgroups of 256 threads, counted in 32 bits; each factor is bounded before the product
  const int64_t most = int64_t(1) << 24, chunks = cdiv(prm->length, kC), parts = cdiv(prm->value, 16);
  if (prm->length >= int64_t(1) << 30 || prm->value >= int64_t(1) << 20 || prm->batch >= most || prm->heads >= most ||
      prm->batch * prm->heads >= most || prm->batch * prm->heads * (chunks > parts ? chunks : parts) >= most) {
    mko_set_error("%s: batch * heads * (chunks of %d tokens, or tiles of 16 values) must be below 2^24", what, kC);
    return MKO_EUNSUPPORTED;
  }
  *g = Geo{prm->batch, prm->length, prm->key_heads, prm->heads, prm->key, prm->value,
           prm->q_stride_b, prm->q_stride_t, prm->q_stride_h, prm->k_stride_b, prm->k_stride_t, prm->k_stride_h,
           prm->v_stride_b, prm->v_stride_t, prm->v_stride_h, chunks, static_cast<int>(prm->heads / prm->key_heads),
           prm->scale, prm->dtype, prm->decay_dtype, prm->beta_dtype, prm->state_dtype};
  return MKO_OK;
}

Ptrs base_ptrs(const mko_delta_params* prm) {
  Ptrs p{};
  p.q = prm->q;
  p.k = prm->k;
  p.v = prm->v;
  p.decay = prm->log_decay;
  p.beta = prm->beta;
  p.initial = prm->initial;
  p.dy = prm->dy;
  p.dfinal = prm->dfinal;
  p.y = prm->y;
  p.final_state = prm->final_state;
  p.dq = prm->dq;
  p.dk = prm->dk;
  p.dv = prm->dv;
  p.ddecay = prm->dlog_decay;
  p.dbeta = prm->dbeta;
  p.dinitial = prm->dinitial;
  return p;
}

bool fast_rows(const Geo& g, const Ptrs& p) {
  bool fast = g.key % 8 == 0 && g.value % 8 == 0;
  for (int64_t n : {g.q_b, g.q_t, g.q_h, g.k_b, g.k_t, g.k_h, g.v_b, g.v_t, g.v_h}) fast = fast && n % 8 == 0;
  for (int64_t n : {g.q_t, g.k_t, g.v_t, g.heads * g.value}) fast = fast && n >= 0 && n < int64_t(1) << 24;  // 32-bit offsets of 16 rows
  for (const void* a : {p.q, p.k, p.v, p.dy, static_cast<const void*>(p.dv)}) fast = fast && reinterpret_cast<uintptr_t>(a) % 16 == 0;
  return fast;
}

Layout saved_layout(const Geo& g) {
  Layout l{};
  const size_t cells = static_cast<size_t>(g.batch * g.heads * g.chunks), el = element_size(g.dtype);
  size_t o = 0;
  l.tokens = o; o = align256(o + cells * sizeof(Tokens));
  l.upper = o; o = align256(o + cells * 2 * kSquare * el);
  l.states = o; o = align256(o + cells * g.value * g.key * el);
  l.e = o; o = align256(o + cells * kC * g.value * el);
  l.total = o;
  return l;
}

Layout forward_layout(const Geo& g, bool train) {
  Layout l{};
  const size_t cells = static_cast<size_t>(g.batch * g.heads * g.chunks), el = element_size(g.dtype);
  size_t o = 0;
  l.lower = o; o = align256(o + cells * 2 * kSquare * el);
  l.tokens = o;
  if (!train) o = align256(o + cells * sizeof(Tokens));
  l.total = o;
  return l;
}

}  // namespace delta
}  // namespace mko

using namespace mko;
using namespace mko::delta;

extern "C" size_t mko_sizeof_delta_params(void) { return sizeof(mko_delta_params); }

extern "C" size_t mko_delta_saved_size(const mko_delta_params* prm) {
  Geo g;
  return make_geo(prm, "delta", &g) == MKO_OK ? saved_layout(g).total : 0;
}

extern "C" size_t mko_delta_fwd_workspace_size(const mko_delta_params* prm) {
  Geo g;
  return make_geo(prm, "delta_fwd", &g) == MKO_OK ? forward_layout(g, prm->saved != nullptr).total : 0;
}

extern "C" int mko_delta_fwd(const mko_delta_params* prm, void* stream) {
  Geo g;
  const int st = make_geo(prm, "delta_fwd", &g);
  if (st != MKO_OK) return st;
  if (g.batch == 0 || g.heads == 0 || g.value == 0) return MKO_OK;
  const bool train = prm->saved != nullptr;
  if (g.length > 0 && (!prm->q || !prm->k || !prm->v || !prm->log_decay || !prm->beta || !prm->y)) {
    mko_set_error("delta_fwd: q, k, v, log_decay, beta and y are required");
    return MKO_EINVAL;
  }
  const Layout w = forward_layout(g, train);
  if (w.total && (!prm->workspace || prm->workspace_bytes < w.total)) {
    mko_set_error("delta_fwd: workspace of %zu bytes needed, %zu given", w.total, prm->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  if (reinterpret_cast<uintptr_t>(prm->workspace) % 16 || reinterpret_cast<uintptr_t>(prm->saved) % 16) {
    mko_set_error("delta_fwd: workspace and saved start at multiples of 16 bytes");
    return MKO_EINVAL;
  }
  Ptrs p = base_ptrs(prm);
  char* ws = static_cast<char*>(prm->workspace);
  p.lower = ws + w.lower;
  if (train) {
    const Layout l = saved_layout(g);
    char* sv = static_cast<char*>(prm->saved);
    p.tokens = reinterpret_cast<Tokens*>(sv + l.tokens);
    p.upper = sv + l.upper;
    p.states = sv + l.states;
    p.e = sv + l.e;
  } else {
    p.tokens = reinterpret_cast<Tokens*>(ws + w.tokens);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (g.length == 0 && !p.final_state) return MKO_OK;
  if (g.dtype == MKO_F32)
    launch<float>(g, p, train, s);
  else if (g.dtype == MKO_BF16)
    launch<bf16>(g, p, train, s);
  else
    launch<_Float16>(g, p, train, s);
  return mko_check_launch("delta_fwd");
}
