// Gated delta rule, backward.  With G the gradient of a chunk's S' and dY that of its outputs:
//   dE = P^T dY + beta exp(c_63 - c) K G^T,  X = T^T dE,  dV = X
//   gradient of S0 = exp(c_63) G + scale (exp(c) dY)^T Q - (exp(c) X)^T K
//   dP = scale dY E^T exp(c_t - c_s) (s <= t),  dA = -X E^T exp(c_t - c_s) (s < t)
//   dq = beta dP K + scale exp(c) dY S0
//   dk = beta dA K - exp(c) X S0 + (beta dP)^T Q + (beta dA)^T K + beta exp(c_63 - c) E G
//   F = dP (q . k) + dA (k . k):  dbeta_s = sum_t F[t][s] + exp(c_63 - c_s) k_s . (E G)_s
// Every factor that holds exp(c_t) is linear in q_t or in k_t as a reader, every one that holds
// exp(-c_s) in k_s as a writer, so
//   dc_t = sum_s beta_s F[t][s] + q_t . (scale exp(c) dY S0)_t - k_t . (exp(c) X S0)_t - beta_t dbeta_t
//   dc_63 += exp(c_63) <G, S0> + sum_s beta_s exp(c_63 - c_s) k_s . (E G)_s
// and the log decay's gradient is dc summed from the chunk's end.  The terms that cancel in that
// sum are read from one float32 F.
//
//   back   per (batch, head, 16 W value columns), sequential from the last chunk: G stays in float32
//          accumulators; writes dV and each chunk's G
//   grads  per (batch, head, chunk): everything else.  Where value heads share a key head, a workgroup takes them
//          one after the other, with dq and dk summed in registers in their order
//   join   that sum where there are few such workgroups, or no room for it in LDS
//
// Four sequences of 4096 tokens with 16 heads of 128 x 128 in bf16: back 143 us, grads 201.  A turn of `back` is 2.2 us of
// 60 products that follow from one another, with their reads of LDS.  `grads` moves 176 KB a chunk and head, 3.7 TB/s;
// two workgroups a CU overlap one's loads and the other's products.
#include "delta.hpp"

namespace mko {
namespace delta {
namespace {

__device__ uint4 zero_unit;  // where rows and columns outside come from

// LDS of `back`; wider keys leave no room for the squares, which then stay in registers.
template <typename TM, int KB, int W, bool FAST>
struct BackLds : Chunks<TM, KB, 16 * W, FAST ? (KB * sizeof(TM) <= 8 && sizeof(TM) == 2 ? 3 : 2) : 1,
                        FAST && KB * sizeof(TM) <= 8 ? 2 : 0, true> {
  // G and X go to the waves that store them where these have room.
  static constexpr bool kHand = FAST && KB * sizeof(TM) <= 8;
  Hand<TM, kHand ? KB : 1> hand[kHand ? W : 1];
};

// W waves carry 16 value columns of G each through the chunks, and four fetch the chunk ahead and store G and dV of
// the chunk before.  In float32 keys of more than 64 spill 20 registers and of more than 128, where nothing is
// fetched ahead, 170: 763 us for two sequences of 1024 tokens with 8 heads of 256 x 128.
template <typename TM, int KB, int W, bool FAST>
__global__ void __launch_bounds__(64 * W + 64 * (FAST ? kFetchers : 0)) back(Geo g, Ptrs p, int parts) {
  constexpr int KP = 32 * KB, BV = 16 * W, kThreads = 64 * W + 64 * (FAST ? kFetchers : 0);
  typedef BackLds<TM, KB, W, FAST> Lds;
  typedef Tile<TM, KP> KTile;
  constexpr bool kHand = Lds::kHand;
  __shared__ __align__(16) Lds lds;
  const WgId id = wg_id(parts, static_cast<int>(g.heads));
  const int64_t h = id.y, b = id.z, bh = b * g.heads + h;
  const int wave = uniform(threadIdx.x >> 6), col = lane_col(), quad = lane_quad();
  const int v0 = id.x * BV, vc = v0 + 16 * wave + col;
  const int key = static_cast<int>(g.key), value = static_cast<int>(g.value);
  const int64_t yrow = g.heads * g.value;  // dy and dv are dense
  TM* dv = static_cast<TM*>(p.dv) + b * g.length * yrow + h * value;
  const Source<TM> src{static_cast<const TM*>(p.k) + b * g.k_b + h / g.rep * g.k_h,
                       static_cast<const TM*>(p.q) + b * g.q_b + h / g.rep * g.q_h,
                       static_cast<const TM*>(p.dy) + b * g.length * yrow + h * value + v0, g.k_t, g.q_t, yrow, g.length,
                       p.tokens + bh * g.chunks, static_cast<const TM*>(p.upper) + bh * g.chunks * 2 * kSquare, key, value - v0};

  if (FAST && key < KP) lds.clear(kThreads);
  if constexpr (FAST) {
    if (wave >= W) {
      const Fetcher<TM, KB, BV, Lds> fetcher(src, reinterpret_cast<const TM*>(&zero_unit), wave - W);
      if constexpr (kHand) {
        Storer<TM, KB> storer(wave - W);
        fetcher.template walk<true, 1>(
            lds, g.chunks - 1, -1, g.chunks,
            [&](int64_t n) {
              if (n > 0) storer.take(lds.hand[storer.tile]);
            },
            [&](int64_t n) {
              if (n == 0) return;
              const int64_t c = g.chunks - n;
              const int t = v0 + 16 * storer.tile;
              if (storer.rows)
                store_rows<TM, true>(dv + c * kC * yrow, static_cast<uint32_t>(yrow), t, value, src.rows(c), storer.f, storer.one);
              else if (t + col < value)
                store_operands<TM, true, KB>(static_cast<TM*>(p.grads) + ((bh * g.chunks + c) * value + t + col) * key, key, storer.f);
            });
      } else {
        fetcher.template walk<false, 0>(lds, g.chunks - 1, -1, g.chunks, [](int64_t) {}, [](int64_t) {});
      }
      return;
    }
  }
  f32x4 s[2 * KB];  // G transposed: [key][value]
#pragma unroll
  for (int i = 0; i < 2 * KB; ++i) s[i] = f32x4{0, 0, 0, 0};
  if (p.dfinal && vc < value) load_state<FAST>(s, p.dfinal, g.state_dtype, (bh * value + vc) * key, key);
  for (int64_t c = g.chunks - 1; c >= 0; --c) {
    const int64_t at = bh * g.chunks + c, t0 = c * kC;
    Frag<TM> held[Lds::kSquares ? 1 : 12];
    if constexpr (!Lds::kSquares) {
#pragma unroll
      for (int i = 0; i < 12; ++i) held[i] = frag_at(src.squares + (12 * c + i) * kFrag);
    }
    __syncthreads();
    typename Lds::Buf& bf = lds.buf(g.chunks - 1 - c);
    if constexpr (!FAST) {
      copy_chunk<kThreads, TM, Lds>(bf, src, c);
      __syncthreads();
    }
    auto square = [&](int which, int i, int j) {  // the transposes of T and P
      if constexpr (Lds::kSquares > 0)
        return frag_at(bf.squares + which * kSquare + upper_at(i, j));
      else
        return held[6 * which + upper_at(i, j) / kFrag];
    };

    Frag<TM> so[KB];  // G as an operand over the keys
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) so[kb] = frag_of<TM>(s[2 * kb], s[2 * kb + 1]);
    if (!kHand && vc < value)
      store_operands<TM, FAST, KB>(static_cast<TM*>(p.grads) + (at * value + vc) * key, key, so);
    Frag<TM> yo[2];  // dY as an operand over the tokens
#pragma unroll
    for (int j = 0; j < 2; ++j) yo[j] = Tile<TM, BV>::over_tokens(bf.v, 32 * j, 16 * wave);
    f32x4 e[4];  // dE
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) mma(e[i], KTile::rows(bf.k, 16 * i, 32 * kb), so[kb]);
      const float4 d = *reinterpret_cast<const float4*>(bf.write + 16 * i + 4 * quad);
      e[i] = f32x4{e[i][0] * d.x, e[i][1] * d.y, e[i][2] * d.z, e[i][3] * d.w};
#pragma unroll
      for (int j = i / 2; j < 2; ++j) mma(e[i], square(1, i, j), yo[j]);
    }
    const Frag<TM> eo[2] = {frag_of<TM>(e[0], e[1]), frag_of<TM>(e[2], e[3])};
    f32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = f32x4{0, 0, 0, 0};
      f32x4 xt = {0, 0, 0, 0};  // [value][t], whose lanes hold four values of a token
#pragma unroll
      for (int j = i / 2; j < 2; ++j) {
        const Frag<TM> t = square(0, i, j);
        mma(x[i], t, eo[j]);
        if (!kHand) mma(xt, eo[j], t);
      }
      const int64_t t = t0 + 16 * i + col;
      if (!kHand && t < g.length) store_four<TM, FAST>(dv + t * yrow, v0 + 16 * wave + 4 * quad, value, xt);
    }
    if constexpr (kHand) {
      __syncthreads();  // what was handed over last has been read
      const Frag<TM> dx[2] = {frag_of<TM>(x[0], x[1]), frag_of<TM>(x[2], x[3])};
      hand_over(lds.hand[wave], so, dx);
    }
    // G of the chunk before
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 d = *reinterpret_cast<const float4*>(bf.in + 16 * i + 4 * quad);
      x[i] = f32x4{-x[i][0] * d.x, -x[i][1] * d.y, -x[i][2] * d.z, -x[i][3] * d.w};
    }
    const Frag<TM> xo[2] = {frag_of<TM>(x[0], x[1]), frag_of<TM>(x[2], x[3])};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float f[8];
      unpack_words<TM, 8>(yo[j].w, f);
#pragma unroll
      for (int e2 = 0; e2 < 8; ++e2) f[e2] *= g.scale * bf.in[32 * j + 16 * (e2 / 4) + 4 * quad + e2 % 4];
      pack_words<TM, 8>(f, yo[j].w);
    }
    const float last = bf.in[kC - 1];
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) s[i][r] *= last;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mma(s[i], KTile::keys_over_tokens(bf.q, 32 * j, i), yo[j]);
        mma(s[i], KTile::keys_over_tokens(bf.k, 32 * j, i), xo[j]);
      }
    }
  }
  if constexpr (kHand) {  // the last turn of those that store
    __syncthreads();
    __syncthreads();
  }
  if (p.dinitial && vc < value) store_state<FAST>(p.dinitial, g.state_dtype, (bh * value + vc) * key, key, s);
}

// Sum over the four quads of a wave (lanes l % 16 alike).
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Eight waves: wave w owns the tokens 16 (w % 4) .. of them, as readers (t) and as writers (s), and one
// half of the keys, w / 4.  Of the 64 x 64 products dY E^T and X E^T the waves of the first half make
// the columns of their t, those of the second the columns of their s, and hand them over through LDS.
template <typename TM, int KB>
struct GradsTiles {
  // values at a time; and whether K and Q are in LDS together
  static constexpr int kValues = sizeof(TM) == 2 && KB <= 4 ? 64 : 32;
  static constexpr bool kBoth = sizeof(TM) == 2 || KB <= 4;
  typedef Tile<TM, 32 * KB> KTile;
  typedef Tile<TM, 32 * KB, kValues> STile;
  typedef Tile<TM, kValues> VTile;
  struct Values {
    TM s0[STile::kElements], gr[STile::kElements], dy[VTile::kElements], x[VTile::kElements], e[VTile::kElements];
  };
  struct Keys {
    TM k[KTile::kElements], q[kBoth ? KTile::kElements : 8];
    TM squares[4][4][2][kFrag];  // dP and dA as operands: [reader, writer] x [dP, dA], token tile, block of 32
  };
  struct Sums {
    Tokens tok;
    float dc[kC], dots[4][3][16], rows[4][16], cols[4][16], gs[8], wrote[4];
  };
  static_assert(sizeof(Sums) % 16 == 0, "the tiles behind it start at multiples of 16 bytes");
};
// GROUP: of a key head, whose K and Q stay while the first values of the next value head fly; otherwise the two
// take turns in one place.
template <typename TM, int KB, bool GROUP>
struct GradsLds : GradsTiles<TM, KB>::Sums {
  union {
    typename GradsTiles<TM, KB>::Values values;
    typename GradsTiles<TM, KB>::Keys keys;
  };
};
template <typename TM, int KB>
struct GradsLds<TM, KB, true> : GradsTiles<TM, KB>::Sums {
  typename GradsTiles<TM, KB>::Values values;
  typename GradsTiles<TM, KB>::Keys keys;
};
// Whether the value heads of a key head may be summed in registers: where K, Q, the squares and the values have
// room in LDS side by side.
template <typename TM, int KB>
constexpr bool kGroups = sizeof(TM) == 2 || KB <= 2;

// Two workgroups a CU, or one of a GROUP or of wide keys, set the registers.  For two in 16 bits with keys of more than 64
// 7 or 8 spill, 28 to 30 with rows that are copied; of a GROUP with keys of more than 128 29 to 51.
template <typename TM, int KB, bool FAST, bool GROUP>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(sizeof(TM) == 2 && KB <= 4 && !GROUP ? 4 : 2)))
grads(Geo g, Ptrs p) {
  constexpr int KT = KB;  // key tiles of a wave
  typedef GradsTiles<TM, KB> Tiles;
  typedef typename Tiles::KTile KTile;
  typedef typename Tiles::STile STile;
  typedef typename Tiles::VTile VTile;
  constexpr int NV = Tiles::kValues;
  constexpr bool kBoth = Tiles::kBoth;
  __shared__ __align__(16) GradsLds<TM, KB, GROUP> lds;
  typename Tiles::Values& lv = lds.values;
  typename Tiles::Keys& lk = lds.keys;
  const WgId id = wg_id(static_cast<int>(GROUP ? g.key_heads : g.heads), static_cast<int>(g.chunks));
  const int64_t h0 = GROUP ? id.x * g.rep : id.x, c = id.y, b = id.z, t0 = c * kC;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kC), g.length - t0));
  const int wave = uniform(threadIdx.x >> 6), tile = wave & 3, half = wave >> 2, col = lane_col(), quad = lane_quad();
  const int key = static_cast<int>(g.key), value = static_cast<int>(g.value);
  const TM* q = static_cast<const TM*>(p.q) + b * g.q_b + t0 * g.q_t + h0 / g.rep * g.q_h;
  const TM* k = static_cast<const TM*>(p.k) + b * g.k_b + t0 * g.k_t + h0 / g.rep * g.k_h;
  const int64_t yrow = g.heads * g.value;
  const TM* zeros = reinterpret_cast<const TM*>(&zero_unit);
  const Tokens& tok = lds.tok;
  auto load_values = [&](int64_t h, int v0) {
    const int64_t at = (b * g.heads + h) * g.chunks + c, y0 = (b * g.length + t0) * yrow + h * value + v0;
    const int64_t s0 = (at * value + v0) * key;
    const int n = value - v0;
    STile::template load<8, FAST>(lv.s0, static_cast<const TM*>(p.states) + s0, key, n, key, wave, zeros);
    STile::template load<8, FAST>(lv.gr, static_cast<const TM*>(p.grads) + s0, key, n, key, wave, zeros);
    VTile::template load<8, FAST>(lv.dy, static_cast<const TM*>(p.dy) + y0, yrow, rows, n, wave, zeros);
    VTile::template load<8, FAST>(lv.x, static_cast<const TM*>(p.dv) + y0, yrow, rows, n, wave, zeros);
    VTile::template load<8, FAST>(lv.e, static_cast<const TM*>(p.e) + at * kC * value + v0, value, kC, n, wave, zeros);
  };
  auto load_keys = [&] {
    KTile::template load<8, FAST>(lk.k, k, g.k_t, rows, key, wave, zeros);
    if constexpr (kBoth) KTile::template load<8, FAST>(lk.q, q, g.q_t, rows, key, wave, zeros);
  };
  const int tc = 16 * tile + col;  // the lane's token
  const bool live = tc < rows;
  f32x4 sq[GROUP ? KT : 1], sk[GROUP ? KT : 1];  // dq and dk of the key head
  if constexpr (GROUP) {
#pragma unroll
    for (int i = 0; i < KT; ++i) sq[i] = sk[i] = f32x4{0, 0, 0, 0};
    load_keys();
  }
  load_values(h0, 0);
  for (int64_t h = h0; h < h0 + (GROUP ? g.rep : 1); ++h) {
  {
    const uint32_t* from = reinterpret_cast<const uint32_t*>(p.tokens + (b * g.heads + h) * g.chunks + c);
    uint32_t* to = reinterpret_cast<uint32_t*>(&lds.tok);
    for (int i = threadIdx.x; i < static_cast<int>(sizeof(Tokens) / 4); i += 512) to[i] = from[i];
  }

  // ---- over the values: the products with the states, and dY E^T and X E^T
  f32x4 aq[KT], ak[KT], aw[KT];  // [key][token]: dY S0, X S0, E G
#pragma unroll
  for (int i = 0; i < KT; ++i) aq[i] = ak[i] = aw[i] = f32x4{0, 0, 0, 0};
  // first half: [s][t] for its t and the tiles s <= t; second: [t][s] for its s and the tiles t >= s
  f32x4 dp[4], da[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dp[i] = da[i] = f32x4{0, 0, 0, 0};
  // tiles above the diagonal; the two waves of a SIMD, `tile` of each half, have five of eight together
  auto outside = [&](int i) { return half ? i < tile : i > tile; };
  float gs = 0.0f;  // <G, S0>
  for (int v0 = 0; v0 < value; v0 += NV) {
    if (v0) {
      __syncthreads();
      load_values(h, v0);
    }
    direct_wait();
#pragma unroll 1
    for (int o = 8 * threadIdx.x; o < STile::kElements; o += 8 * 512) {
      uint32_t w[kWordsOf<TM, 8>];
      float fa[8], fb[8];
      load_words(lv.s0 + o, w);
      unpack_words<TM, 8>(w, fa);
      load_words(lv.gr + o, w);
      unpack_words<TM, 8>(w, fb);
#pragma unroll
      for (int j = 0; j < 8; ++j) gs += fa[j] * fb[j];
    }
#pragma unroll 1
    for (int vb = 0; vb < NV / 32; ++vb) {
      const int v = 32 * vb, lane = lane_again();
      if (v0 + v >= value) break;
      const Frag<TM> my = VTile::rows(lv.dy, 16 * tile, v, lane), mx = VTile::rows(lv.x, 16 * tile, v, lane),
                     me = VTile::rows(lv.e, 16 * tile, v, lane);
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const Frag<TM> fs = STile::keys_over_values(lv.s0, v, half * KT + i, lane);
        mma(aq[i], fs, my);
        mma(ak[i], fs, mx);
        mma(aw[i], STile::keys_over_values(lv.gr, v, half * KT + i, lane), me);
      }
      const Frag<TM> b1 = half ? me : my, b2 = half ? me : mx;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (outside(i)) continue;
        mma(dp[i], VTile::rows(half ? lv.dy : lv.e, 16 * i, v, lane), b1);
        mma(da[i], VTile::rows(half ? lv.x : lv.e, 16 * i, v, lane), b2);
      }
    }
  }
  __syncthreads();
  gs = wave_sum(gs);
  if (lane_id() == 0) lds.gs[wave] = gs;
  if constexpr (GROUP) {
    if (h + 1 < h0 + g.rep) load_values(h + 1, 0);  // K and Q came with the first head's
  } else {
    load_keys();
    direct_wait();
  }

  // ---- the states' parts of dq and dk, [key][token] in place
  const float in = tok.in[tc], out = tok.out[tc], beta = tok.beta[tc];
  float dot[3] = {0.0f, 0.0f, 0.0f};  // q . state part of dq, k . that of dk, k . E G
#pragma unroll
  for (int i = 0; i < KT; ++i) {
    const int n = half * KT + i, k0 = 32 * (n / 2) + 8 * quad + 4 * (n % 2);
    float kv[4], qv[4];
    uint32_t w[kWordsOf<TM, 4>];
    load_words(lk.k + KTile::at(tc, k0), w);
    unpack_words<TM, 4>(w, kv);
    if constexpr (kBoth) {
      load_words(lk.q + KTile::at(tc, k0), w);
      unpack_words<TM, 4>(w, qv);
    } else {
      unpack_words<TM, 4>(load_part<TM, 4>(q + (live ? tc * g.q_t : 0), k0, live ? key : 0).w, qv);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      aq[i][r] *= g.scale * in;
      ak[i][r] *= -in;
      dot[0] += qv[r] * aq[i][r];
      dot[1] += kv[r] * ak[i][r];
      dot[2] += kv[r] * aw[i][r];
      ak[i][r] += beta * out * aw[i][r];
    }
  }
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    dot[d] = quad_sum(dot[d]);
    if (quad == 0 && half == 1) lds.dots[tile][d][col] = dot[d];
  }
  __builtin_amdgcn_sched_barrier(0);

  // ---- dP and dA with their decays, rounded as operands, and F's sums
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // first half: [s of tile i][its t]; second: [t of tile i][its s]
    if (outside(i)) {
      const uint32_t none[kWordsOf<TM, 4>] = {};
      store_words(lk.squares[2 * half][tile][i / 2] + 8 * lane_id() + 4 * (i % 2), none);
      store_words(lk.squares[2 * half + 1][tile][i / 2] + 8 * lane_id() + 4 * (i % 2), none);
      continue;
    }
    f32x4 qk = {0, 0, 0, 0}, kk = {0, 0, 0, 0};
    const int lane = lane_again();  // its own rows are read again for every tile: kept, they would spill
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const Frag<TM> other = KTile::rows(lk.k, 16 * i, 32 * kb, lane), mine = KTile::rows(lk.k, 16 * tile, 32 * kb, lane);
      mma(kk, other, mine);
      if constexpr (kBoth) {
        mma(qk, KTile::rows(half ? lk.q : lk.k, 16 * i, 32 * kb, lane),
            KTile::rows(half ? lk.k : lk.q, 16 * tile, 32 * kb, lane));
      } else {
        const Frag<TM> f = frag_memory(q, g.q_t, 16 * (half ? i : tile), 32 * kb, rows, key);
        mma(qk, half ? f : other, half ? mine : f);
      }
    }
    float vp[4], va[4];
    const double ct = tok.c[tc];
    const float bt = tok.beta[tc];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int o = 16 * i + 4 * quad + r;
      const int ahead = half ? o - tc : tc - o;  // t - s
      const float d = static_cast<float>(tok.c[o] - ct), bs = half ? bt : tok.beta[o];
      const float m = ahead >= 0 ? fast_exp2(half ? d : -d) : 0.0f;
      vp[r] = ahead >= 0 ? g.scale * dp[i][r] * m : 0.0f;
      va[r] = ahead > 0 ? -da[i][r] * m : 0.0f;
      const float f = vp[r] * qk[r] + va[r] * kk[r];
      sum += f * (half ? 1.0f : bs);
      vp[r] *= bs;
      va[r] *= bs;
    }
    uint32_t w[kWordsOf<TM, 4>];
    pack_words<TM, 4>(vp, w);
    store_words(lk.squares[2 * half][tile][i / 2] + 8 * lane + 4 * (i % 2), w);
    pack_words<TM, 4>(va, w);
    store_words(lk.squares[2 * half + 1][tile][i / 2] + 8 * lane + 4 * (i % 2), w);
    asm volatile("" : "+v"(sum));  // a tile at a time, for the registers
    __builtin_amdgcn_sched_barrier(0);
  }
  sum = quad_sum(sum);
  if (quad == 0) (half == 0 ? lds.rows : lds.cols)[tile][col] = sum;

  // ---- and the chunk's
  __syncthreads();
  const int last = lane_again();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const Frag<TM> pr = frag_at(lk.squares[0][tile][j]), ar = frag_at(lk.squares[1][tile][j]),
                   pw = frag_at(lk.squares[2][tile][j]), aw2 = frag_at(lk.squares[3][tile][j]);
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const Frag<TM> ok = KTile::keys_over_tokens(lk.k, 32 * j, half * KT + i, last);
      mma(aq[i], ok, pr);
      mma(ak[i], ok, ar);
      mma(ak[i], ok, aw2);
      if constexpr (kBoth) mma(ak[i], KTile::keys_over_tokens(lk.q, 32 * j, half * KT + i, last), pw);
    }
  }
  if constexpr (!kBoth) {
    __syncthreads();
    KTile::template load<8, FAST>(lk.k, q, g.q_t, rows, key, wave, zeros);
    direct_wait();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const Frag<TM> pw = frag_at(lk.squares[2][tile][j]);
#pragma unroll
      for (int i = 0; i < KT; ++i) mma(ak[i], KTile::keys_over_tokens(lk.k, 32 * j, half * KT + i, last), pw);
    }
  }
  if constexpr (GROUP) {
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      sq[i] += aq[i];
      sk[i] += ak[i];
    }
  } else if (live) {
    const int64_t row = ((b * g.length + t0 + tc) * g.heads + h) * key;
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const int n = half * KT + i, k0 = 32 * (n / 2) + 8 * quad + 4 * (n % 2);
      if (p.pq) {
        store_four<float, FAST>(p.pq + row, k0, key, aq[i]);
        store_four<float, FAST>(p.pk + row, k0, key, ak[i]);
      } else {
        store_four<TM, FAST>(static_cast<TM*>(p.dq) + row, k0, key, aq[i]);
        store_four<TM, FAST>(static_cast<TM*>(p.dk) + row, k0, key, ak[i]);
      }
    }
  }
  // ---- the tokens' own gradients
  if (half == 0) {
    const float dotw = (dot[2] + lds.dots[tile][2][col]) * out, dbeta = lds.cols[tile][col] + dotw;
    if (quad == 0) {
      lds.dc[tc] = lds.rows[tile][col] + (dot[0] + lds.dots[tile][0][col]) + (dot[1] + lds.dots[tile][1][col]) - beta * dbeta;
      if (live) store_one(p.dbeta, g.beta_dtype, (b * g.length + t0 + tc) * g.heads + h, dbeta);
    }
    const float wr = row16_sum(beta * dotw);
    if (lane_id() == 0) lds.wrote[tile] = wr;
  }
  __syncthreads();
  if (wave == 0) {
    const int lane = lane_id();
    float d = lds.dc[lane];
    if (lane == kC - 1) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m += lds.gs[i];
      d += tok.in[kC - 1] * m + ((lds.wrote[0] + lds.wrote[1]) + (lds.wrote[2] + lds.wrote[3]));
    }
    for (int o = 1; o < kC; o *= 2) {
      const float u = __shfl_down(d, o);
      if (lane + o < kC) d += u;
    }
    // d is exp(log decay) <G, S>: of a decay that clears the state, and of one that meets none, only the roundings of
    // what cancels are left
    const bool none = !p.initial && t0 + lane == 0;
    if (none || fast_exp2(static_cast<float>(tok.c[lane] - (lane ? tok.c[lane - 1] : 0.0))) == 0.0f) d = 0.0f;
    if (lane < rows) store_one(p.ddecay, g.decay_dtype, (b * g.length + t0 + lane) * g.heads + h, d);
  }
  if constexpr (GROUP) __syncthreads();  // before the next head's tokens
  }
  if constexpr (GROUP) {
    if (live) {
      const int64_t row = ((b * g.length + t0 + tc) * g.key_heads + id.x) * key;
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        const int n = half * KT + i, k0 = 32 * (n / 2) + 8 * quad + 4 * (n % 2);
        store_four<TM, FAST>(static_cast<TM*>(p.dq) + row, k0, key, sq[i]);
        store_four<TM, FAST>(static_cast<TM*>(p.dk) + row, k0, key, sk[i]);
      }
    }
  }
}

// dq and dk of a key head: the sum over its value heads, four elements a thread.
template <typename TM>
__global__ void __launch_bounds__(256) join(Geo g, Ptrs p, int64_t groups, int per) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= groups) return;
  const int64_t row = i / per, key = g.key;  // a row: (batch, token, key head)
  const int at = static_cast<int>(i % per) * 4;
  const float* from = blockIdx.y ? p.pk : p.pq;
  TM* to = static_cast<TM*>(blockIdx.y ? p.dk : p.dq);
  float s[4] = {0, 0, 0, 0};
  for (int r = 0; r < g.rep; ++r) {
    float f[4];
    unpack_words<float, 4>(load_part<float, 4>(from + (row * g.rep + r) * key, at, key).w, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += f[j];
  }
  store_part<TM, 4>(to + row * key, at, key, s);
}

// Whether they are: with a workgroup or more for each of the 256 CUs.  In us, summed in registers and with partial
// sums in memory: 256 workgroups of two heads in bfloat16 28 and 36 (keys of 128) and 22 and 26 (of 64), in float32
// 49 and 59, of four heads 46 and 60, 35 and 41, 88 and 103; 2048 186 and 217, 137 and 131, 373 and 418, and 318 and
// 423, 240 and 238, 699 and 804.  128 leave CUs idle: 25 and 26, 20 and 21, 46 and 35, and 41 and 35, 33 and 26, 83 and 58.
bool grouped(const Geo& g) {
  return g.rep > 1 && (g.dtype != MKO_F32 || g.key <= 64) && g.batch * g.key_heads * g.chunks >= 256;
}

struct Space {
  size_t grads, pq, pk, total;
};
Space backward_layout(const Geo& g) {
  Space l{};
  const size_t cells = static_cast<size_t>(g.batch * g.heads * g.chunks), el = element_size(g.dtype);
  const size_t part = g.rep > 1 && !grouped(g) ? static_cast<size_t>(g.batch * g.length * g.heads * g.key) * 4 : 0;
  size_t o = 0;
  l.grads = o; o = align256(o + cells * g.value * g.key * el);
  l.pq = o; o = align256(o + part);
  l.pk = o; o = align256(o + part);
  l.total = o;
  return l;
}

template <typename TM, int KB>
void launch(const Geo& g, const Ptrs& p, hipStream_t s) {
  constexpr int W = 2;
  const unsigned cells = static_cast<unsigned>(g.batch * g.heads * g.chunks);
  const int parts = static_cast<int>(cdiv(g.value, 16 * W));
  const unsigned grid = static_cast<unsigned>(g.batch * g.heads * parts);
  const unsigned groups = static_cast<unsigned>(g.batch * g.key_heads * g.chunks);
  bool fast = false;
  if constexpr (KB * sizeof(TM) <= 16) {
    fast = fast_rows(g, p);
    if (fast) {
      MKO_TIMED("delta_back", s, back<TM, KB, W, true><<<grid, 64 * (W + kFetchers), 0, s>>>(g, p, parts));
      if constexpr (kGroups<TM, KB>) {
        if (grouped(g)) MKO_TIMED("delta_grads", s, grads<TM, KB, true, true><<<groups, 512, 0, s>>>(g, p));
      }
      if (!grouped(g)) MKO_TIMED("delta_grads", s, grads<TM, KB, true, false><<<cells, 512, 0, s>>>(g, p));
    }
  }
  if (!fast) {
    MKO_TIMED("delta_back", s, back<TM, KB, W, false><<<grid, 64 * W, 0, s>>>(g, p, parts));
    if constexpr (kGroups<TM, KB>) {
      if (grouped(g)) MKO_TIMED("delta_grads", s, grads<TM, KB, false, true><<<groups, 512, 0, s>>>(g, p));
    }
    if (!grouped(g)) MKO_TIMED("delta_grads", s, grads<TM, KB, false, false><<<cells, 512, 0, s>>>(g, p));
  }
  if (p.pq) {
    const int per = static_cast<int>(cdiv(g.key, 4));
    const int64_t fours = g.batch * g.length * g.key_heads * per;
    MKO_TIMED("delta_join", s, join<TM><<<dim3(static_cast<unsigned>(cdiv(fours, 256)), 2), 256, 0, s>>>(g, p, fours, per));
  }
}

template <typename TM>
void launch(const Geo& g, const Ptrs& p, hipStream_t s) {
  if (g.key <= 32) return launch<TM, 1>(g, p, s);
  if (g.key <= 64) return launch<TM, 2>(g, p, s);
  if (g.key <= 128) return launch<TM, 4>(g, p, s);
  return launch<TM, 8>(g, p, s);
}

}  // namespace
}  // namespace delta
}  // namespace mko

using namespace mko;
using namespace mko::delta;

extern "C" size_t mko_delta_bwd_workspace_size(const mko_delta_params* prm) {
  Geo g;
  return make_geo(prm, "delta_bwd", &g) == MKO_OK ? backward_layout(g).total : 0;
}

extern "C" int mko_delta_bwd(const mko_delta_params* prm, void* stream) {
  Geo g;
  const int st = make_geo(prm, "delta_bwd", &g);
  if (st != MKO_OK) return st;
  if (g.batch == 0 || g.heads == 0 || g.value == 0 || g.length == 0) return MKO_OK;  // the caller fills the gradients
  if (!prm->q || !prm->k || !prm->v || !prm->log_decay || !prm->beta || !prm->saved || !prm->dy || !prm->dq || !prm->dk ||
      !prm->dv || !prm->dlog_decay || !prm->dbeta) {
    mko_set_error("delta_bwd: q, k, v, log_decay, beta, saved, dy and the five gradients are required");
    return MKO_EINVAL;
  }
  const Space w = backward_layout(g);
  if (!prm->workspace || prm->workspace_bytes < w.total) {
    mko_set_error("delta_bwd: workspace of %zu bytes needed, %zu given", w.total, prm->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  if (reinterpret_cast<uintptr_t>(prm->workspace) % 16 || reinterpret_cast<uintptr_t>(prm->saved) % 16) {
    mko_set_error("delta_bwd: workspace and saved start at multiples of 16 bytes");
    return MKO_EINVAL;
  }
  Ptrs p = base_ptrs(prm);
  const Layout l = saved_layout(g);
  char *sv = static_cast<char*>(prm->saved), *ws = static_cast<char*>(prm->workspace);
  p.tokens = reinterpret_cast<Tokens*>(sv + l.tokens);
  p.upper = sv + l.upper;
  p.states = sv + l.states;
  p.e = sv + l.e;
  p.grads = ws + w.grads;
  if (g.rep > 1 && !grouped(g)) {
    p.pq = reinterpret_cast<float*>(ws + w.pq);
    p.pk = reinterpret_cast<float*>(ws + w.pk);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (g.dtype == MKO_F32)
    launch<float>(g, p, s);
  else if (g.dtype == MKO_BF16)
    launch<bf16>(g, p, s);
  else
    launch<_Float16>(g, p, s);
  return mko_check_launch("delta_bwd");
}
