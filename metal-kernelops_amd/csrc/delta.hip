// Gated delta rule, forward (delta.hpp has the formulas).
//
//   prep  per (batch, head, chunk): the decays' sums, T by blocked substitution in float32, and the
//         operands T and P (and their transposes, for the backward)
//   scan  per (batch, head, 16 W value columns), sequential over the chunks.  W waves carry S in float32
//         accumulators and do only what the next chunk waits for, E and S's update; W
//         others follow a chunk behind with Y, and four fetch the chunk ahead and store what the backward reads.
//
// Four sequences of 4096 tokens with 16 heads of 128 x 128 in bf16: prep 65 us, scan 170.  Prep moves 56 KB a chunk and
// head, 3.4 TB/s, behind the latency of its substitution.  A turn of the scan takes 2.6 us: its chain of products
// about 1.0 (2400 cycles), fetching 48 KB and storing 16 KB for the backward on every CU at once the rest; without
// gradients a turn takes 1.6.  With the chain's waves fetching and storing for themselves the scan took 254 us, with
// the fetches in waves of their own and two buffers 232, with three 163, and 170 with the backward's states stored by them.
//
// Few long sequences leave most of the chip idle, so their chunks are cut into segments that are walked side
// by side.  A segment makes d S0 + S0 N + B of the state S0 before it, d its decay:
//   ends  per (batch, head, segment but the last, 64 columns): the chunks' walk without outputs, from zero (B) and
//         from the unit matrix (d I + N)
//   join  per (batch, head, 16 value columns): S0 of each segment, in their order.  What a state only keeps, d S0,
//         is a float32 product, as in the uncut walk
// and the scan starts each segment from its own S0.  One sequence of 32768 tokens with 16 such heads: 98 + 154 + 8 + 200
// us in four segments; uncut, prep and scan take 100 + 649.
#include <algorithm>

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

// Wave w owns the row tile w of A and P.  Six waves a SIMD, for whose registers and LDS K and A share a place, hide more of
// the substitution than four did, for three or four registers that spill: 72 -> 67 us (the sizes above), 111 -> 101
// without the transposes.
template <typename TM, int KB, bool TRAIN>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(KB * sizeof(TM) <= 8 ? 6 : 1))) prep(Geo g, Ptrs p, bool fast) {
  typedef Tile<TM, 32 * KB> KTile;
  __shared__ Tokens tok;
  __shared__ __align__(16) union {  // K until its products are there, then A and T: room for more workgroups
    TM kt[KTile::kElements];
    float a[kC * kPitch];
  } lds;
  TM* kt = lds.kt;
  float* a = lds.a;
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

  if (fast)
    KTile::template issue<4>(kt, k, g.k_t, rows, key, wave, reinterpret_cast<const TM*>(&zero_unit));
  else
    KTile::template copy<256>(kt, k, g.k_t, rows, key);
  Frag<TM> qf[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) qf[kb] = frag_memory(q, g.q_t, 16 * wave, 32 * kb, rows, key);
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
    const float out = fast_exp2(static_cast<float>(last - s));
    const float beta = lane < rows ? load_one(p.beta, g.beta_dtype, i) : 0.0f;
    tok.out[lane] = out;
    tok.beta[lane] = beta;
    tok.write[lane] = out * beta;
  }
  direct_wait();
  {
    uint32_t* to = reinterpret_cast<uint32_t*>(p.tokens + at);
    const uint32_t* from = reinterpret_cast<const uint32_t*>(&tok);
    for (int i = threadIdx.x; i < static_cast<int>(sizeof(Tokens) / 4); i += 256) to[i] = from[i];
  }
  Frag<TM> kf[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) kf[kb] = KTile::rows(kt, 16 * wave, 32 * kb);
  const int tr = 16 * wave + 4 * lane_quad(), tc = 16 * wave + lane_col();  // this tile's tokens as rows and columns
  float av[4][4];  // A's rows of tile `wave`
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > wave) continue;
    f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0}, kq = {0, 0, 0, 0};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Frag<TM> o = KTile::rows(kt, 16 * j, 32 * kb);
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
      av[j][r] = t > sc ? kk[r] * m : 0.0f;
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
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > wave) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) a[(tr + r) * kPitch + 16 * j + lane_col()] = av[j][r];
  }
  __syncthreads();
  invert(a);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = j <= wave;
    const float4 v = *reinterpret_cast<const float4*>(a + tc * kPitch + 16 * j + 4 * lane_quad());
    const float f[4] = {in ? v.x : 0.0f, in ? v.y : 0.0f, in ? v.z : 0.0f, in ? v.w : 0.0f};
    if (j / 2 <= wave / 2) store_half<TM>(lp - kSquare + lower_at(wave, j / 2), j % 2, f);  // T's rows of tile `wave`
    if (TRAIN && j / 2 >= wave / 2) {  // its columns of tile `wave`, rows of tile j
      float f[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) f[r] = j >= wave ? a[(16 * j + 4 * lane_quad() + r) * kPitch + tc] : 0.0f;
      store_half<TM>(up - kSquare + upper_at(wave, j / 2), j % 2, f);
    }
  }
}

// LDS of `scan`.  FAST: rows of whole units at multiples of 16 bytes, which take direct loads.  T, Q and P are
// there where they have room beside K, V and what is handed over; else T and P stay in registers.
template <typename TM, int KB, int W, bool FAST>
struct ScanLds : Chunks<TM, KB, 16 * W, FAST ? (KB * sizeof(TM) <= 8 && sizeof(TM) == 2 ? 3 : 2) : 1,
                        FAST && KB * sizeof(TM) <= 8 ? (sizeof(TM) == 2 ? 2 : 1) : 0,
                        FAST && KB * sizeof(TM) <= 8 && sizeof(TM) == 2> {
  // Two where there is room; one is read and written in one turn, on two sides of a barrier.
  static constexpr int kHands =
      FAST && sizeof(Chunks<TM, KB, 16 * W, ScanLds::kBufs, ScanLds::kSquares, ScanLds::kQ>) + 2 * W * sizeof(Hand<TM, KB>) <= 160 * 1024
          ? 2 : 1;
  Hand<TM, KB> hand[kHands][W];  // S and E of a chunk
};

// S of 16 value columns, carried through the chunks by one wave.
template <typename TM, int KB>
struct Carrier {
  f32x4 s[2 * KB], e[4];  // S and E transposed: [key][value] and [token][value]
  Frag<TM> so[KB];        // S as an operand over the keys

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) s[i] = f32x4{0, 0, 0, 0};
  }
  // E = T (V - exp(c) K S0^T); `t` gives T's operands.
  template <typename Lds, typename Square>
  __device__ __forceinline__ void errors(const typename Lds::Buf& bf, int v0, bool no_values, Square t) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) so[kb] = frag_of<TM>(s[2 * kb], s[2 * kb + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 z = {0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) mma(z, Lds::KTile::rows(bf.k, 16 * i, 32 * kb), so[kb]);
      const f32x4 vv = no_values ? f32x4{0, 0, 0, 0} : Lds::VTile::values(bf.v, 16 * i, v0);
      const float4 d = *reinterpret_cast<const float4*>(bf.in + 16 * i + 4 * lane_quad());
      e[i] = f32x4{vv[0] - d.x * z[0], vv[1] - d.y * z[1], vv[2] - d.z * z[2], vv[3] - d.w * z[3]};
    }
    const Frag<TM> zo[2] = {frag_of<TM>(e[0], e[1]), frag_of<TM>(e[2], e[3])};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j <= i / 2; ++j) mma(e[i], t(i, j), zo[j]);
    }
  }
  // S' = exp(c_63) S0 + E^T (beta exp(c_63 - c) K)
  template <typename Lds>
  __device__ __forceinline__ void advance(const typename Lds::Buf& bf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 d = *reinterpret_cast<const float4*>(bf.write + 16 * i + 4 * lane_quad());
      e[i] = f32x4{e[i][0] * d.x, e[i][1] * d.y, e[i][2] * d.z, e[i][3] * d.w};
    }
    const Frag<TM> wo[2] = {frag_of<TM>(e[0], e[1]), frag_of<TM>(e[2], e[3])};
    const float last = bf.in[kC - 1];
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[i][r] *= last;
#pragma unroll
      for (int j = 0; j < 2; ++j) mma(s[i], Lds::KTile::keys_over_tokens(bf.k, 32 * j, i), wo[j]);
    }
  }
};

template <typename TM>
__device__ __forceinline__ Source<TM> source(const Geo& g, const Ptrs& p, int64_t b, int64_t h, int v0) {
  const int64_t bh = b * g.heads + h;
  return Source<TM>{static_cast<const TM*>(p.k) + b * g.k_b + h / g.rep * g.k_h,
                    static_cast<const TM*>(p.q) + b * g.q_b + h / g.rep * g.q_h,
                    static_cast<const TM*>(p.v) + b * g.v_b + h * g.v_h + v0, g.k_t, g.q_t, g.v_t, g.length,
                    p.tokens + bh * g.chunks, static_cast<const TM*>(p.lower) + bh * g.chunks * 2 * kSquare,
                    static_cast<int>(g.key), static_cast<int>(g.value) - v0};
}

// LDS of `ends`.
template <typename TM, int KB, int W>
using EndsLds = Chunks<TM, KB, 16 * W, sizeof(Chunks<TM, KB, 16 * W, 3, 1, false>) <= 160 * 1024 ? 3 : 2, 1, false>;
constexpr int kEndsTiles = 4;

template <typename TM, int KB>
__global__ void __launch_bounds__(64 * (kEndsTiles + kFetchers)) ends(Geo g, Ptrs p, int value_parts, int parts) {
  constexpr int W = kEndsTiles, BV = 16 * W;
  typedef EndsLds<TM, KB, W> Lds;
  __shared__ __align__(16) Lds lds;
  const WgId id = wg_id(parts, static_cast<int>(g.heads));
  const int64_t h = id.y, b = id.z / (g.segments - 1), seg = id.z % (g.segments - 1), bh = b * g.heads + h;
  const bool unit = id.x >= value_parts;  // from the unit matrix, whose rows stand for values
  if (unit && seg == 0) return;           // the state before it is known
  const int wave = uniform(threadIdx.x >> 6), col = lane_col(), quad = lane_quad();
  const int v0 = (unit ? id.x - value_parts : id.x) * BV, vc = v0 + 16 * wave + col;
  const int key = static_cast<int>(g.key), value = static_cast<int>(g.value);
  const Source<TM> src = source<TM>(g, p, b, h, unit ? 0 : v0);
  const int64_t first = seg * g.span, at = bh * (g.segments - 1) + seg;

  if (key < 32 * KB) lds.clear(64 * (W + kFetchers));
  if (wave >= W) {
    Fetcher<TM, KB, BV, Lds>(src, reinterpret_cast<const TM*>(&zero_unit), wave - W).template walk<false, 0>(
        lds, first, 1, g.span, [](int64_t) {}, [](int64_t) {});
    return;
  }
  Carrier<TM, KB> carrier;
  carrier.clear();
  if (unit) {
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) carrier.s[i][r] = 16 * (i & ~1) + 4 * (i & 1) + 8 * quad + r == vc ? 1.0f : 0.0f;
    }
  } else if (seg == 0 && p.initial && vc < value) {
    load_state<true>(carrier.s, p.initial, g.state_dtype, (bh * value + vc) * key, key);
  }
  float left = 1.0f;  // of the state, rounded as the walk rounds it
  for (int64_t n = 0; n < g.span; ++n) {
    __syncthreads();
    typename Lds::Buf& bf = lds.buf(n);
    carrier.template errors<Lds>(bf, 16 * wave, unit, [&](int i, int j) { return frag_at(bf.squares + lower_at(i, j)); });
    left *= bf.in[kC - 1];
    carrier.template advance<Lds>(bf);
  }
  if (!unit) {
    if (vc < value) store_row<float, true>(p.ends + (at * value + vc) * key, key, carrier.s);
    return;
  }
  if (vc == 0 && quad == 0) p.kept[at] = left;
  if (vc < key) {  // transposed, as `join` reads it
    float* to = p.maps + at * key * key + vc;
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int k = 16 * (i & ~1) + 4 * (i & 1) + 8 * quad + r;
        if (k < key) to[k * key] = carrier.s[i][r] - (k == vc ? left : 0.0f);
      }
    }
  }
}

// f as TM, and what that leaves of it as TM.
template <typename TM, int N>
__device__ __forceinline__ void split(const float (&f)[N], uint32_t (&hi)[kWordsOf<TM, N>], uint32_t (&lo)[kWordsOf<TM, N>]) {
  float h[N], l[N];
  pack_words<TM, N>(f, hi);
  unpack_words<TM, N>(hi, h);
#pragma unroll
  for (int i = 0; i < N; ++i) l[i] = f[i] - h[i];
  pack_words<TM, N>(l, lo);
}

// The state behind each segment from the one before it, in place of its B: wave i has 16 values of the key tile i and
// takes S0 as an operand from the others.  In 16 bits N and S0 are two operands each, whose products leave
// 2^-16 (bfloat16) of N S0: one rounding of a state for a whole segment would stay where N takes all of it away.
template <typename TM, int KB>
__global__ void __launch_bounds__(128 * KB) join(Geo g, Ptrs p, int tiles) {
  constexpr bool kSplit = sizeof(TM) == 2;
  __shared__ __align__(16) TM lds[2][kSplit ? 2 : 1][KB * kFrag];  // one is read while the next is written
  const int64_t bh = blockIdx.x / tiles;
  const int wave = uniform(threadIdx.x >> 6), col = lane_col(), quad = lane_quad(), key = static_cast<int>(g.key);
  const int64_t vc = blockIdx.x % tiles * 16 + col;
  const bool live = vc < g.value;
  const int k0 = 32 * (wave / 2) + 8 * quad + 4 * (wave % 2);           // the lane's keys of S
  const int kr = 32 * (wave / 2) + 8 * (col / 4) + 4 * (wave % 2) + col % 4;  // and its row of N
  float* row = p.ends + (bh * (g.segments - 1) * g.value + (live ? vc : 0)) * key;
  float s[4];
  unpack_words<float, 4>(load_part<float, 4>(row, k0, key).w, s);
  for (int64_t seg = 1; seg < g.segments - 1; ++seg) {
    row += g.value * key;
    const int64_t at = bh * (g.segments - 1) + seg;
    const float* map = p.maps + at * key * key + (kr < key ? kr * key : 0);
    Words<float, 8> n[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) n[kb] = load_part<float, 8>(map, 32 * kb + 8 * quad, kr < key ? key : 0);
    float b[4];
    unpack_words<float, 4>(load_part<float, 4>(row, k0, key).w, b);
    const float left = p.kept[at];
    TM(&so)[kSplit ? 2 : 1][KB * kFrag] = lds[seg & 1];
    const int to = wave / 2 * kFrag + 8 * lane_id() + 4 * (wave % 2);
    if constexpr (kSplit) {
      uint32_t hi[kWordsOf<TM, 4>], lo[kWordsOf<TM, 4>];
      split<TM, 4>(s, hi, lo);
      store_words(so[0] + to, hi);
      store_words(so[1] + to, lo);
    } else {
      uint32_t w[kWordsOf<TM, 4>];
      pack_words<TM, 4>(s, w);
      store_words(so[0] + to, w);
    }
    __syncthreads();
    f32x4 acc = {b[0] + left * s[0], b[1] + left * s[1], b[2] + left * s[2], b[3] + left * s[3]};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Frag<TM> x = frag_at(so[0] + kb * kFrag);
      if constexpr (kSplit) {
        Frag<TM> hi, lo;
        float f[8];
        unpack_words<float, 8>(n[kb].w, f);
        split<TM, 8>(f, hi.w, lo.w);
        mma(acc, lo, x);
        mma(acc, hi, frag_at(so[1] + kb * kFrag));
        mma(acc, hi, x);
      } else {
        mma(acc, __builtin_bit_cast(Frag<TM>, n[kb]), x);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = acc[r];
    if (live) store_part<float, 4>(row, k0, key, s);
  }
}

// W waves carry 16 value columns each through the chunks, W follow, and four fetch.  Turn n: the first do chunk n,
// the second finish chunk n - 1 and the last bring chunk n + 1, or n + 2 where three have room.
template <typename TM, int KB, int W, bool TRAIN, bool FAST>
__global__ void __launch_bounds__(128 * W + 64 * (FAST ? kFetchers : 0)) scan(Geo g, Ptrs p, int parts) {
  constexpr int KP = 32 * KB, BV = 16 * W, kThreads = 128 * W + 64 * (FAST ? kFetchers : 0);
  typedef ScanLds<TM, KB, W, FAST> Lds;
  typedef typename Lds::KTile KTile;
  constexpr bool kMid = FAST && Lds::kHands == 1;
  __shared__ __align__(16) Lds lds;
  const WgId id = wg_id(parts, static_cast<int>(g.heads));
  const int64_t h = id.y, b = id.z / g.segments, seg = id.z % g.segments, bh = b * g.heads + h;
  const int64_t first = seg * g.span, chunks = min(g.span, g.chunks - first);  // of this segment
  const int wave = uniform(threadIdx.x >> 6), col = lane_col(), quad = lane_quad();
  const int mine = wave % W;  // of the value tiles
  const int v0 = id.x * BV, vt = v0 + 16 * mine, vc = vt + col;  // the lane's column of S and E
  const int key = static_cast<int>(g.key), value = static_cast<int>(g.value);
  const Source<TM> src = source<TM>(g, p, b, h, v0);

  if (FAST && key < KP) lds.clear(kThreads);
  if constexpr (FAST) {
    if (wave >= 2 * W) {
      Storer<TM, KB> storer(wave - 2 * W);
      Fetcher<TM, KB, BV, Lds>(src, reinterpret_cast<const TM*>(&zero_unit), wave - 2 * W).template walk<kMid, 1>(
          lds, first, 1, chunks,
          [&](int64_t n) {
            if (TRAIN && n > 0) storer.take(lds.hand[(n - 1) & (Lds::kHands - 1)][storer.tile]);
          },
          [&](int64_t n) {
            if (!TRAIN || n == 0) return;
            const int64_t at = bh * g.chunks + first + n - 1;
            const int t = v0 + 16 * storer.tile;
            if (storer.rows)
              store_rows<TM, true>(static_cast<TM*>(p.e) + at * kC * value, static_cast<uint32_t>(value), t, value, kC, storer.f, storer.one);
            else if (t + col < value)
              store_operands<TM, true, KB>(static_cast<TM*>(p.states) + (at * value + t + col) * key, key, storer.f);
          });
      return;
    }
  }
  if (wave < W) {
    Carrier<TM, KB> carrier;
    carrier.clear();
    if (seg > 0) {
      if (vc < value)
        load_row<float, FAST>(carrier.s, p.ends + ((bh * (g.segments - 1) + seg - 1) * value + vc) * key, key);
    } else if (p.initial && vc < value) {
      load_state<FAST>(carrier.s, p.initial, g.state_dtype, (bh * value + vc) * key, key);
    }
    Frag<TM> held[Lds::kSquares ? 1 : 6];
    auto hold = [&](int64_t c) {
      if constexpr (!Lds::kSquares) {
#pragma unroll
        for (int i = 0; i < 6; ++i) held[i] = frag_at(src.squares + c * 2 * kSquare + i * kFrag);
      }
    };
    if (chunks > 0) hold(first);
    for (int64_t n = 0; n < chunks; ++n) {
      __syncthreads();
      typename Lds::Buf& bf = lds.buf(n);
      if constexpr (!FAST) {
        copy_chunk<kThreads, TM, Lds>(bf, src, first + n);
        __syncthreads();
      }
      carrier.template errors<Lds>(bf, 16 * mine, false, [&](int i, int j) {
        if constexpr (Lds::kSquares > 0)
          return frag_at(bf.squares + lower_at(i, j));
        else
          return held[lower_at(i, j) / kFrag];
      });
      if (n + 1 < chunks) hold(first + n + 1);
      if constexpr (kMid) __syncthreads();  // what was handed over last has been read
      const Frag<TM> eo[2] = {frag_of<TM>(carrier.e[0], carrier.e[1]), frag_of<TM>(carrier.e[2], carrier.e[3])};
      hand_over(lds.hand[n & (Lds::kHands - 1)][mine], carrier.so, eo);
      carrier.template advance<Lds>(bf);
    }
    __syncthreads();  // the last turn of those that follow
    if constexpr (kMid) __syncthreads();
    if (p.final_state && first + chunks == g.chunks && vc < value) store_state<FAST>(p.final_state, g.state_dtype, (bh * value + vc) * key, key, carrier.s);
    return;
  }

  // Q and P of chunk n are loaded in turn n, from LDS where they are there, and used in the next; wider keys
  // would need more registers than there are, and are loaded where they are used.
  constexpr bool kAhead = KB * sizeof(TM) <= 8;
  Frag<TM> qf[4][kAhead ? KB : 1], pf[6], one[2];
  float in[4];
  unit_halves<TM>(one);
  for (int64_t n = 0; n <= chunks; ++n) {
    __syncthreads();
    Frag<TM> so[KB], eo[2];
    if (n > 0) {
      const Hand<TM, KB>& hand = lds.hand[(n - 1) & (Lds::kHands - 1)][mine];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) so[kb] = frag_at(hand.s + kb * kFrag);
      eo[0] = frag_at(hand.e);
      eo[1] = frag_at(hand.e + kFrag);
    }
    if constexpr (!FAST) {
      if (n < chunks) copy_chunk<kThreads, TM, Lds>(lds.buf(n), src, first + n);
    }
    if (FAST ? kMid : n < chunks) __syncthreads();
    // of tokens and keys that are not there, others' values: those tokens are not stored, and S has zeros at
    // those keys
    auto load_q = [&](int64_t c, int i, int kb) {
      if constexpr (FAST) {
        const char* from = reinterpret_cast<const char*>(src.q + c * kC * g.q_t);
        const uint32_t row = min(16 * i + col, src.rows(c) - 1) * static_cast<uint32_t>(g.q_t);
        const uint32_t at = (row + (32 * kb + 8 * quad < key ? 32 * kb + 8 * quad : 0)) * static_cast<uint32_t>(sizeof(TM));
        Frag<TM> f;
#pragma unroll
        for (int j = 0; j < kWordsOf<TM, 8> / 4; ++j) {
          const uint4 x = *reinterpret_cast<const uint4*>(from + at + 16 * j);
          f.w[4 * j] = x.x;
          f.w[4 * j + 1] = x.y;
          f.w[4 * j + 2] = x.z;
          f.w[4 * j + 3] = x.w;
        }
        return f;
      } else {
        return frag_memory(src.q + c * kC * g.q_t, g.q_t, 16 * i, 32 * kb, src.rows(c), key);
      }
    };
    if (n > 0) {
      const int64_t c = first + n - 1, at = bh * g.chunks + c;
      TM* yp = static_cast<TM*>(p.y) + ((b * g.length + c * kC) * g.heads + h) * value;
      const auto y_row = [&] {  // of FAST, 32 bits
        if constexpr (FAST) return static_cast<uint32_t>(g.heads * value);
        else return g.heads * value;
      }();
      // Y transposed, so that a lane holds four values of a token
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f32x4 y = {0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if constexpr (kAhead)
            mma(y, so[kb], qf[i][kb]);
          else
            mma(y, so[kb], load_q(c, i, kb));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] *= in[i];
#pragma unroll
        for (int j = 0; j <= i / 2; ++j) mma(y, eo[j], pf[lower_at(i, j) / kFrag]);
        if (16 * i + col < src.rows(c))
          store_four<TM, FAST>(yp + (16 * i + col) * y_row, vt + 4 * quad, value, y);
      }
      if constexpr (TRAIN && !FAST) {
        store_rows<TM, false>(static_cast<TM*>(p.e) + at * kC * value, static_cast<int64_t>(value), vt, value, kC, eo, one);
        if (vc < value) store_operands<TM, false, KB>(static_cast<TM*>(p.states) + (at * value + vc) * key, key, so);
      }
    }
    if (n < chunks) {
      typename Lds::Buf& bf = lds.buf(n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        in[i] = g.scale * bf.in[16 * i + col];
        if constexpr (kAhead) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            if constexpr (Lds::kQ)
              qf[i][kb] = KTile::rows(bf.q, 16 * i, 32 * kb);
            else
              qf[i][kb] = load_q(first + n, i, kb);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        if constexpr (Lds::kQ)
          pf[i] = frag_at(bf.squares + kSquare + i * kFrag);
        else
          pf[i] = frag_at(src.squares + (2 * (first + n) + 1) * kSquare + i * kFrag);
      }
    }
  }
}

// ------------------------------------------------------------------ the choice

template <typename TM, int KB, bool TRAIN>
void launch(Geo g, const Ptrs& p, hipStream_t s) {
  constexpr int W = 2;
  const unsigned cells = static_cast<unsigned>(g.batch * g.heads * g.chunks);
  const int parts = static_cast<int>(cdiv(g.value, 16 * W));
  const bool fast = fast_rows(g, p);
  if (cells) MKO_TIMED("delta_prep", s, prep<TM, KB, TRAIN><<<cells, 256, 0, s>>>(g, p, fast));
  const unsigned grid = static_cast<unsigned>(g.batch * g.heads * parts);
  if constexpr (KB * sizeof(TM) <= 16) {
    if (fast) {
      if (g.segments > 1) {
        const int values = static_cast<int>(cdiv(g.value, 16 * kEndsTiles)), all = values + static_cast<int>(cdiv(g.key, 16 * kEndsTiles));
        const int tiles = static_cast<int>(cdiv(g.value, 16));
        const unsigned cells = static_cast<unsigned>(g.batch * g.heads * (g.segments - 1) * all);
        MKO_TIMED("delta_ends", s, ends<TM, KB><<<cells, 64 * (kEndsTiles + kFetchers), 0, s>>>(g, p, values, all));
        if (g.segments > 2)
          MKO_TIMED("delta_join_states", s, join<TM, KB><<<static_cast<unsigned>(g.batch * g.heads * tiles), 128 * KB, 0, s>>>(g, p, tiles));
      }
      const unsigned grid = static_cast<unsigned>(g.batch * g.heads * parts * g.segments);
      MKO_TIMED("delta_scan", s, scan<TM, KB, W, TRAIN, true><<<grid, 128 * W + 64 * kFetchers, 0, s>>>(g, p, parts));
      return;
    }
  }
  g.segments = 1;
  g.span = g.chunks;
  MKO_TIMED("delta_scan", s, scan<TM, KB, W, TRAIN, false><<<grid, 128 * W, 0, s>>>(g, p, parts));
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

// Segments that a sequence is cut into: where its workgroups leave more than two thirds of the 256 CUs without
// work, as many as give each CU one, of 8 chunks or more, and no more than the square root of the chunks, since
// `join` walks them one by one.  The chunks are walked twice, in two turns a chunk of a segment for one of the uncut walk,
// with two launches more.  Where a turn is long that pays from three segments on (kernels but prep, uncut and cut, in
// us: 24 chunks in three, keys of 256 in bfloat16 76 and 65, of 64 in float32 81 and 69; 64 chunks of 84 workgroups 316
// and 176, 205 and 160), for float32 keys of up to 32 from four (40 chunks in five 96 and 57, 64 in three 150 and 181).  Where
// it is short, from 32 turns fewer on (keys of 128 in bfloat16: 50 chunks in six, 32 fewer, 50.3 and 49.3; 64
// in four, 32 fewer, 67 and 63; 64 in three, 20 fewer, 66 and 72; 24 in three 29 and 38; keys of 64: 36 and 35, 54 and 49,
// 47 and 55, 21 and 30).
int64_t segments_of(const mko_delta_params* prm, int64_t chunks) {
  const int64_t groups = prm->batch * prm->heads * cdiv(prm->value, 32);
  if (prm->key % 8 || prm->value % 8 || groups < 1 || 3 * groups > 256) return 1;
  int64_t n = std::min<int64_t>(256 / groups, chunks / 8);
  while (n > 1 && n * n > chunks) --n;
  if (n < (prm->dtype == MKO_F32 && prm->key <= 32 ? 4 : 3)) return 1;
  const int64_t span = cdiv(chunks, n);
  if (prm->dtype != MKO_F32 && prm->key <= 128 && chunks - 2 * span < 32) return 1;
  return cdiv(chunks, span);
}

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
  if (prm->value >= int64_t(1) << 20) {
    mko_set_error("%s: the value axis is below 2^20", what);
    return MKO_EUNSUPPORTED;
  }
  // a launch counts its threads in 32 bits, and `scan` and `grads` have 512 in a workgroup; each factor is bounded before
  // the product
  const int64_t most = int64_t(1) << 23, chunks = cdiv(prm->length, kC), parts = cdiv(prm->value, 16);
  if (prm->length >= int64_t(1) << 30 || prm->batch >= most || prm->heads >= most ||
      prm->batch * prm->heads >= most || prm->batch * prm->heads * (chunks > parts ? chunks : parts) >= most) {
    mko_set_error("%s: batch * heads * (chunks of %d tokens, or tiles of 16 values) must be below 2^23 (of 512 threads; 2^24 of 256 fill a "
                  "launch)", what, kC);
    return MKO_EUNSUPPORTED;
  }
  *g = Geo{prm->batch, prm->length, prm->key_heads, prm->heads, prm->key, prm->value,
           prm->q_stride_b, prm->q_stride_t, prm->q_stride_h, prm->k_stride_b, prm->k_stride_t, prm->k_stride_h,
           prm->v_stride_b, prm->v_stride_t, prm->v_stride_h, chunks, segments_of(prm, chunks), 0,
           static_cast<int>(prm->heads / prm->key_heads),
           prm->scale, prm->dtype, prm->decay_dtype, prm->beta_dtype, prm->state_dtype};
  g->span = cdiv(chunks, g->segments);
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
  for (int64_t n : {g.q_t, g.k_t, g.v_t, g.heads * g.value}) fast = fast && n >= 0 && n < int64_t(1) << 23;  // 32-bit offsets of 64 rows
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
  const size_t ends = static_cast<size_t>(g.batch * g.heads * (g.segments - 1));
  l.ends = o; o = align256(o + ends * g.value * g.key * sizeof(float));
  l.maps = o; o = align256(o + ends * g.key * g.key * sizeof(float));
  l.kept = o; o = align256(o + ends * sizeof(float));
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
  p.ends = reinterpret_cast<float*>(ws + w.ends);
  p.maps = reinterpret_cast<float*>(ws + w.maps);
  p.kept = reinterpret_cast<float*>(ws + w.kept);
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
