// 8-bit integers for gfx950: quantisation of rows, and the matrix product
//   out[m][n] = q_scale[m] w_scale[n] sum_k q[m][k] w[n][k] + bias[n]
// with the sum in int32, exact for fewer than 2^17 terms of at most 2^14.  Small outputs are
// bound by the weights' bytes (`few`), larger ones by the matrix cores' feed and the power limit
// (`tile`): 8192 x 2560 x 5120 in 121 us (1.78 POP/s), 8192 x 8192 x 4096 in 255 to 265 (2.1), of 2.9 to
// 3.4 POP/s that products of random bytes reach from registers alone.  quantize_rows moves 8192 x 5120 bf16 in 24 us,
// 5.2 TB/s.
#include <type_traits>

#include "common.hpp"
#include "io.hpp"
#include "quantize.hpp"
#include "rows.hpp"

namespace mko {
namespace int8 {
namespace {

constexpr int64_t kMaxInner = 131071;
constexpr int64_t kMaxSide = 1 << 26;

// A team of waves holds a row in registers between its largest value and its bytes, NV vectors of 16
// bytes of x a thread.
template <typename T, int NV>
__global__ void __launch_bounds__(1024) quantize_rows(mko_quantize_params p, int team_threads) {
  constexpr int VEC = kVecOf<T>;
  __shared__ uint32_t tops[16];
  const int team = uniform(static_cast<int>(threadIdx.x) / team_threads);
  const int lt = threadIdx.x - team * team_threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / team_threads) + team;
  const bool live = row < p.rows;
  const int64_t n = live ? p.features : 0;
  const T* x = static_cast<const T*>(p.x) + (live ? row * p.x_stride : 0);
  Words<T, VEC> raw[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) raw[k] = load_part<T, VEC>(x, static_cast<int64_t>(lt + k * team_threads) * VEC, n);
  uint32_t am = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float v[VEC];
    unpack_words<T, VEC>(raw[k].w, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) am = max(am, abs_bits(v[e]));
  }
  am = wave_max(am);
  if (team_threads > kWave) {
    const int wave = threadIdx.x >> 6, waves = team_threads >> 6;
    if ((threadIdx.x & (kWave - 1)) == 0) tops[wave] = am;
    __syncthreads();
    for (int i = 0; i < waves; ++i) am = max(am, tops[team * waves + i]);
  }
  if (!live) return;
  const RowScale q = row_scale(am);
  if (lt == 0) p.scale[row] = q.scale;
  int8_t* out = p.q + row * p.q_stride;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float v[VEC];
    int b[VEC];
    unpack_words<T, VEC>(raw[k].w, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) b[e] = quantise(v[e], q.inv);
    store_bytes<VEC>(out, static_cast<int64_t>(lt + k * team_threads) * VEC, n, p.q_stride, b);
  }
  for (int64_t i = cdiv(n, VEC) * VEC + lt; i < p.q_stride; i += team_threads) out[i] = 0;
}

// Rows wider than a team's registers are read twice.
template <typename T>
__global__ void __launch_bounds__(1024) quantize_wide(mko_quantize_params p) {
  __shared__ uint32_t tops[16];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  uint32_t am = 0;
  for (int64_t i = threadIdx.x; i < p.features; i += 1024) am = max(am, abs_bits(to_f32(x[i])));
  am = wave_max(am);
  if ((threadIdx.x & (kWave - 1)) == 0) tops[threadIdx.x / kWave] = am;
  __syncthreads();
  for (int w = 0; w < 16; ++w) am = max(am, tops[w]);
  const RowScale q = row_scale(am);
  if (threadIdx.x == 0) p.scale[row] = q.scale;
  for (int64_t i = threadIdx.x; i < p.q_stride; i += 1024)
    p.q[row * p.q_stride + i] = i < p.features ? static_cast<int8_t>(quantise(to_f32(x[i]), q.inv)) : 0;
}

template <typename T, int NV>
void launch_quantize_n(const mko_quantize_params& p, int team, hipStream_t s) {
  const int threads = team > 4 ? team * kWave : 4 / team * team * kWave;
  const unsigned grid = static_cast<unsigned>(cdiv(p.rows, threads / (team * kWave)));
  MKO_TIMED("quantize_int8", s, quantize_rows<T, NV><<<grid, threads, 0, s>>>(p, team * kWave));
}

// Teams as for the norm (residual_norm.hip): a vector a thread for few rows, a wave a row for many.
template <typename T>
void launch_quantize(const mko_quantize_params& p, hipStream_t s) {
  const int64_t waves = cdiv(p.features, kVecOf<T> * kWave);
  int team = 1;
  while (team < 16 && team < waves && (cdiv(waves, team) > 8 || p.rows * team < 2048)) ++team;
  const int64_t nv = cdiv(waves, team);
  if (nv <= 1) return launch_quantize_n<T, 1>(p, team, s);
  if (nv <= 2) return launch_quantize_n<T, 2>(p, team, s);
  if (nv <= 3) return launch_quantize_n<T, 3>(p, team, s);
  if (nv <= 5) return launch_quantize_n<T, 5>(p, team, s);
  if (nv <= 8) return launch_quantize_n<T, 8>(p, team, s);
  MKO_TIMED("quantize_int8_wide", s, quantize_wide<T><<<static_cast<unsigned>(p.rows), 1024, 0, s>>>(p));
}

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

// 16 bytes at any address: one load or store of four words (the part takes every alignment).
struct __attribute__((packed)) Bytes16 {
  v4i v;
};

// 16 bytes of a row of `inner` bytes from byte k, zero from the row's end on; nothing past the
// end is read.
__device__ __forceinline__ v4i load_chunk(const int8_t* row, int k, int inner) {
  if (k + 16 <= inner) return reinterpret_cast<const Bytes16*>(row + k)->v;
  v4i r = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < inner) r[i / 4] |= static_cast<int>(static_cast<uint8_t>(row[k + i])) << (8 * (i % 4));
  return r;
}

// ---------------------------------------------------------------- output

// Four consecutive outputs of one token from channel n on: the sums scaled, the bias added.
__device__ __forceinline__ void put4(const mko_int8_linear_params& p, int64_t m, int64_t n, const int (&acc)[4],
                                     float qs) {
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool in = n + i < p.outer;
    v[i] = static_cast<float>(acc[i]) * qs * (in ? p.w_scale[n + i] : 0.0f);
    if (p.bias && in) v[i] += p.bias[n + i];
  }
  const int64_t at = m * p.outer + n;
  if (n + 4 <= p.outer) {
    struct __attribute__((packed)) Two {
      uint32_t w[2];
    };
    struct __attribute__((packed)) Four {
      float w[4];
    };
    if (p.dtype == MKO_F32)
      *reinterpret_cast<Four*>(static_cast<float*>(p.out) + at) = Four{{v[0], v[1], v[2], v[3]}};
    else if (p.dtype == MKO_BF16)
      *reinterpret_cast<Two*>(static_cast<bf16*>(p.out) + at) = Two{{pack2<bf16>(v[0], v[1]), pack2<bf16>(v[2], v[3])}};
    else
      *reinterpret_cast<Two*>(static_cast<_Float16*>(p.out) + at) =
          Two{{pack2<_Float16>(v[0], v[1]), pack2<_Float16>(v[2], v[3])}};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.outer) store_one(p.out, p.dtype, at + i, v[i]);
  }
}

// `cols` of eight consecutive outputs from element `at` on.  ALIGNED: 16-byte stores, with the
// nontemporal hint, which leaves the operands in the L2s (8192 x 2560 x 5120: 128 -> 121 us).
template <bool ALIGNED>
__device__ __forceinline__ void put8(const mko_int8_linear_params& p, int64_t at, int cols, const float (&v)[8]) {
  struct __attribute__((packed)) Words4 {
    mko_u32x4 w;
  };
  if (cols == 8) {
    uint32_t w[8];
    if (p.dtype == MKO_F32) {
      pack_words<float, 8>(v, w);
      if (ALIGNED) {
        store_words_nt(static_cast<float*>(p.out) + at, w);
      } else {
        Words4* o = reinterpret_cast<Words4*>(static_cast<float*>(p.out) + at);
        o[0].w = mko_u32x4{w[0], w[1], w[2], w[3]};
        o[1].w = mko_u32x4{w[4], w[5], w[6], w[7]};
      }
    } else {
      if (p.dtype == MKO_BF16)
        pack_words<bf16, 8>(v, w);
      else
        pack_words<_Float16, 8>(v, w);
      const uint32_t half[4] = {w[0], w[1], w[2], w[3]};
      if (ALIGNED)
        store_words_nt(static_cast<uint16_t*>(p.out) + at, half);
      else
        reinterpret_cast<Words4*>(static_cast<uint16_t*>(p.out) + at)->w = mko_u32x4{w[0], w[1], w[2], w[3]};
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < cols) store_one(p.out, p.dtype, at + e, v[e]);
  }
}

// ---------------------------------------------------------------- few tokens

// A workgroup of W waves computes 16 channels of MT * 16 tokens (grid: channels, tokens); the waves
// take the inner axis in turns of 256 bytes, load both operands straight into the matrix cores'
// registers, and their sums are added in LDS.  Each block of tokens reads the weights once, which is
// what bounds it: one token into 10240 x 2560 takes 8.0 us (3.3 TB/s), 48 tokens into 2560 x 2560 7.6.
template <int MT, int W>
__global__ void __launch_bounds__(W * 64) few(mko_int8_linear_params p) {
  __shared__ __attribute__((aligned(16))) int sums[W][MT][256];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int inner = static_cast<int>(p.inner);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, m0 = static_cast<int64_t>(blockIdx.y) * (MT * 16);
  const int64_t nrow = min(n0 + (lane & 15), p.outer - 1);
  const int8_t* wrow = p.w + nrow * p.w_stride;
  const int8_t* qrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    qrow[t] = p.q + min(m0 + t * 16 + (lane & 15), p.rows - 1) * p.q_stride;
  v4i acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = v4i{0, 0, 0, 0};
  const int part = (lane >> 4) * 16;
  int k0 = wave * 256;
  for (; k0 + 256 <= inner; k0 += W * 256) {
    v4i a[4], b[MT][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      a[s] = reinterpret_cast<const Bytes16*>(wrow + k0 + s * 64 + part)->v;
#pragma unroll
      for (int t = 0; t < MT; ++t) b[t][s] = reinterpret_cast<const Bytes16*>(qrow[t] + k0 + s * 64 + part)->v;
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], b[t][s], acc[t], 0, 0, 0);
  }
  if (k0 < inner) {
    for (int k = k0; k < inner; k += 64) {
      const v4i a = load_chunk(wrow, k + part, inner);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const v4i b = load_chunk(qrow[t], k + part, inner);
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc[t], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
    *reinterpret_cast<v4i*>(&sums[wave][t][(lane & 15) * 16 + (lane >> 4) * 4]) = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 64; i += W * 64) {
    const int t = i >> 6, e = (i & 63) * 4;
    const int64_t m = m0 + t * 16 + (e >> 4), n = n0 + (e & 15);
    if (m >= p.rows || n >= p.outer) continue;
    int s[4] = {0, 0, 0, 0};
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += sums[w][t][e + j];
    put4(p, m, n, s, p.q_scale[m]);
  }
}

// ---------------------------------------------------------------- tiles

__device__ v4i zero_chunk;  // what a lane past the inner axis' end loads instead

template <int VM>
__device__ __forceinline__ void wait_and_meet() {
  // The waves' own loads but the last VM have landed, their LDS reads are done, and all have come here.
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
}

// A tile of BN channels by BM tokens, by WN x WM waves.  A stage holds BK bytes of each of the
// tile's rows in LDS.  Rows start 256 / BK to a sweep of the banks, and 16-byte chunk c of row r
// lies at position c ^ (r / (256 / BK)) of its row, which gives the 16 rows that a quarter wave
// reads at one c 16 different groups of banks.
template <int BN, int BM, int WN, int WM, int BK, int STAGES, bool SPLIT, bool DIRECT>
__global__ void __launch_bounds__(WN * WM * 64) tile(mko_int8_linear_params p, int tiles_n, int tiles_m) {
  constexpr int kWaves = WN * WM;
  constexpr int kTn = BN / WN / 32, kTm = BM / WM / 32;
  constexpr int kChunks = BK / 16, kRows = 64 / kChunks, kSweep = 256 / BK;
  constexpr int kLn = BN / kRows / kWaves, kLm = BM / kRows / kWaves;  // loads of kRows rows a wave makes for a stage
  constexpr int kLoads = kLn + kLm;
  constexpr int kSteps = BK / 32;
  constexpr int kStage = (BN + BM) * BK;
  static_assert(kLn * kRows * kWaves == BN && kLm * kRows * kWaves == BM, "whole loads");
  constexpr int kSums = kWaves * 32 * kTn * 32 * 4;  // the output's way through LDS
  __shared__ __attribute__((aligned(256))) char lds[STAGES * kStage > kSums ? STAGES * kStage : kSums];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wn = wave / WM, wm = wave % WM;
  const int whole = static_cast<int>(p.inner);
  const int inner = DIRECT ? whole & ~15 : whole;  // direct loads take whole chunks; the rest comes first

  // bands of 8 token tiles, token tile fastest: an XCD's workgroups share both operands in its L2
  const WgId id = wg_id(tiles_n * tiles_m, 1);
  const int band = id.x / (8 * tiles_n), in_band = id.x - band * 8 * tiles_n;
  const int band_m = min(8, tiles_m - band * 8);
  const int tn = in_band / band_m, tm = band * 8 + in_band % band_m;
  const int64_t n0 = static_cast<int64_t>(tn) * BN, m0 = static_cast<int64_t>(tm) * BM;

  const int8_t* wbase = p.w + n0 * p.w_stride;
  const int8_t* qbase = p.q + m0 * p.q_stride;
  // load j covers kRows rows of the weights (j < kLn) or the tokens; rows past the end repeat the last
  auto tile_row = [&](int j) { return ((j < kLn ? j : j - kLn) * kWaves + wave) * kRows + lane / kChunks; };
  auto source_row = [&](int j) {
    const int64_t rows = j < kLn ? p.outer - n0 : p.rows - m0;
    return static_cast<int>(min(static_cast<int64_t>(tile_row(j)), min(static_cast<int64_t>(j < kLn ? BN : BM), rows) - 1));
  };
  auto source_k = [&](int j) { return ((lane % kChunks) ^ ((tile_row(j) / kSweep) % kChunks)) * 16; };
  uint32_t off[DIRECT ? kLoads : 1];
  if constexpr (DIRECT) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      off[j] = static_cast<uint32_t>(source_row(j)) * static_cast<uint32_t>(j < kLn ? p.w_stride : p.q_stride) +
               static_cast<uint32_t>(source_k(j));
  }
  const int nk = (inner + BK - 1) / BK;

  auto slot = [&](int st, int j) {  // where a wave's load j lands in a stage
    return lds + st * kStage + (j < kLn ? 0 : BN * BK) + ((j < kLn ? j : j - kLn) * kWaves + wave) * kRows * BK;
  };
  const int8_t* zeros = reinterpret_cast<const int8_t*>(&zero_chunk);
  asm("" : "+s"(zeros));  // its address is formed here, not in the loop
  auto load_to = [&](int st, int j, const int8_t* src) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                     (__attribute__((address_space(3))) uint32_t*)slot(st, j), 16, 0, 0);
  };
  // Part `part` of the loads of stage kt; past the end those of a stage that is there, so that every
  // step makes as many and the waits' counts hold.
  auto issue = [&](int st, int kt, auto part) {
    constexpr int kFrom = decltype(part)::value * kLoads / 3, kTo = (decltype(part)::value + 1) * kLoads / 3;
    if ((kt + 1) * BK <= inner || (kt >= nk && inner >= BK)) {
      const int k0 = kt < nk ? kt * BK : 0;
      const int8_t* wb = wbase + k0;
      const int8_t* qb = qbase + k0;
#pragma unroll
      for (int j = kFrom; j < kTo; ++j) load_to(st, j, (j < kLn ? wb : qb) + off[DIRECT ? j : 0]);
    } else {
      const int k0 = (nk - 1) * BK;
#pragma unroll
      for (int j = kFrom; j < kTo; ++j)
        load_to(st, j, k0 + source_k(j) < inner ? (j < kLn ? wbase : qbase) + k0 + off[DIRECT ? j : 0] : zeros);
    }
  };
  constexpr std::integral_constant<int, 0> part0;
  constexpr std::integral_constant<int, 1> part1;
  constexpr std::integral_constant<int, 2> part2;
  v4i held[DIRECT ? 1 : kLoads];
  auto fetch = [&](int kt) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int64_t r = source_row(j);
      held[DIRECT ? 0 : j] =
          load_chunk(j < kLn ? wbase + r * p.w_stride : qbase + r * p.q_stride, kt * BK + source_k(j), inner);
    }
  };
  auto put_held = [&](int st) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) *reinterpret_cast<v4i*>(slot(st, j) + lane * 16) = held[DIRECT ? 0 : j];
  };

  v16i acc[kTn][kTm];
#pragma unroll
  for (int i = 0; i < kTn; ++i)
#pragma unroll
    for (int j = 0; j < kTm; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  // operands of one step of 32 bytes: row lane % 32 of each 32-row block, chunk 2 s + lane / 32
  const int lr = lane & 31;
  uint32_t at[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) at[s] = lr * BK + (((s * 2 + (lane >> 5)) ^ ((lr / kSweep) % kChunks)) << 4);
  v4i a[2][kTn], b[2][kTm];
  auto read = [&](int st, int s, int to) {
    const char* wl = lds + st * kStage + wn * kTn * 32 * BK + at[s];
    const char* ql = lds + st * kStage + BN * BK + wm * kTm * 32 * BK + at[s];
#pragma unroll
    for (int i = 0; i < kTn; ++i) a[to][i] = *reinterpret_cast<const v4i*>(wl + i * 32 * BK);
#pragma unroll
    for (int j = 0; j < kTm; ++j) b[to][j] = *reinterpret_cast<const v4i*>(ql + j * 32 * BK);
  };
  auto multiply = [&](int from) {
#pragma unroll
    for (int i = 0; i < kTn; ++i)
#pragma unroll
      for (int j = 0; j < kTm; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[from][i], b[from][j], acc[i][j], 0, 0, 0);
  };
  static_assert(kSteps % 2 == 0, "the operand registers alternate");

  // Operands are read one step ahead of their products, across the stages too: the last step's
  // are in registers when the waves meet, after which the stage just read is free and takes the
  // loads of the stage STAGES further on.  With SPLIT those are issued in three parts, a part to a
  // step: a wave that issues all at once waits for the address unit, 27 cycles a load, and multiplies
  // nothing.  Where several workgroups share a CU another one multiplies then, and the earlier
  // loads are worth more: 128 x 128 tiles of 8192 x 8192 x 4096 take 347 us, split 389.
  if constexpr (DIRECT) {
    if (inner < whole) {  // first the step of the bytes that fill no chunk, in the lanes of its first half
#pragma unroll
      for (int i = 0; i < kTn; ++i) {
        const int64_t n = min(n0 + (wn * kTn + i) * 32 + lr, p.outer - 1);
        a[0][i] = load_chunk(p.w + n * p.w_stride, lane < 32 ? inner : whole, whole);
      }
#pragma unroll
      for (int j = 0; j < kTm; ++j) {
        const int64_t m = min(m0 + (wm * kTm + j) * 32 + lr, p.rows - 1);
        b[0][j] = load_chunk(p.q + m * p.q_stride, lane < 32 ? inner : whole, whole);
      }
      multiply(0);
    }
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
      issue(st, st, part0);
      if (SPLIT && st + 1 == STAGES) break;
      issue(st, st, part1);
      issue(st, st, part2);
    }
    wait_and_meet<(STAGES - 2) * kLoads + (SPLIT ? kLoads / 3 : kLoads)>();
    read(0, 0, 0);
    for (int kt = 0; kt < nk; kt += STAGES) {
#pragma unroll
      for (int st = 0; st < STAGES; ++st) {
        if (st > 0 && kt + st >= nk) break;
#pragma unroll
        for (int s = 0; s + 1 < kSteps; ++s) {
          if (SPLIT && s == 0) issue((st + STAGES - 1) % STAGES, kt + st + STAGES - 1, part1);
          if (SPLIT && s == (kSteps > 2 ? 1 : 0)) issue((st + STAGES - 1) % STAGES, kt + st + STAGES - 1, part2);
          read(st, s + 1, (s + 1) & 1);
          multiply(s & 1);
        }
        wait_and_meet<(STAGES - 2) * kLoads>();
        issue(st, kt + st + STAGES, part0);
        if (!SPLIT) {
          issue(st, kt + st + STAGES, part1);
          issue(st, kt + st + STAGES, part2);
        }
        read((st + 1) % STAGES, 0, 0);
        multiply((kSteps - 1) & 1);
      }
    }
    // what was issued past the end must land before this workgroup's LDS is another's
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    fetch(0);
    put_held(0);
    for (int kt = 0; kt < nk; ++kt) {
      __syncthreads();
      if (kt + 1 < nk) fetch(kt + 1);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        read(kt & 1, s, 0);
        multiply(0);
      }
      if (kt + 1 < nk) put_held((kt + 1) & 1);
    }
  }

  // The sums go through LDS, 32 tokens of the wave's channels at a time, so that a lane has 8
  // consecutive channels of a token and the stores of a row are contiguous; the channels' scales
  // are then the same for all of a lane's tokens.  Chunk c of 4 sums lies at c ^ (token / kPer).
  constexpr int kWide = kTn * 32, kRowChunks = kTn * 8, kPer = kRowChunks >= 16 ? 1 : 16 / kRowChunks;
  constexpr int kSpread = kRowChunks < 16 ? kRowChunks : 16;
  wait_and_meet<0>();
  char* mine = lds + wave * 32 * kWide * 4;
  constexpr int kPerRow = kWide / 8;  // lanes to a token
  const bool aligned = (static_cast<uint64_t>(p.outer) % 8 | reinterpret_cast<uintptr_t>(p.out) % 16) == 0;
  const int nl = (lane % kPerRow) * 8;
  const int64_t n = n0 + wn * kWide + nl;
  const int cols = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(8), p.outer - n)));
  float ws[8], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    ws[e] = e < cols ? p.w_scale[n + e] : 0.0f;
    bias[e] = p.bias && e < cols ? p.bias[n + e] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < kTm; ++j) {
    const int shift = (lr / kPer) % kSpread;
#pragma unroll
    for (int i = 0; i < kTn; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = i * 8 + 2 * g + (lane >> 5);
        *reinterpret_cast<v4i*>(mine + lr * kWide * 4 + ((c ^ shift) << 4)) =
            v4i{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
      }
    wave_lds_sync();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 64 / kPerRow) {
      const int row = r0 + lane / kPerRow;
      const int turn = (row / kPer) % kSpread;
      const int64_t m = m0 + (wm * kTm + j) * 32 + row;
      const v4i lo = *reinterpret_cast<const v4i*>(mine + row * kWide * 4 + (((nl / 4) ^ turn) << 4));
      const v4i hi = *reinterpret_cast<const v4i*>(mine + row * kWide * 4 + (((nl / 4 + 1) ^ turn) << 4));
      if (m >= p.rows || cols == 0) continue;
      const float qs = p.q_scale[m];
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(e < 4 ? lo[e] : hi[e - 4]) * qs * ws[e] + bias[e];
      if (aligned)
        put8<true>(p, m * p.outer + n, cols, v);
      else
        put8<false>(p, m * p.outer + n, cols, v);
    }
    wave_lds_sync();
  }
}

// ---------------------------------------------------------------- the choice

template <int MT>
void launch_few(const mko_int8_linear_params& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(cdiv(p.outer, 16)), static_cast<unsigned>(cdiv(p.rows, MT * 16)));
  const int64_t turns = cdiv(p.inner, 256);
  if (turns <= 4 || grid.x >= 2048)
    MKO_TIMED("int8_linear_few", s, few<MT, 4><<<grid, 4 * 64, 0, s>>>(p));
  else
    MKO_TIMED("int8_linear_few", s, few<MT, 8><<<grid, 8 * 64, 0, s>>>(p));
}

template <int BN, int BM, int WN, int WM, int BK, int STAGES, bool SPLIT>
void launch_tile(const mko_int8_linear_params& p, bool direct, hipStream_t s) {
  const int tn = static_cast<int>(cdiv(p.outer, BN)), tm = static_cast<int>(cdiv(p.rows, BM));
  const unsigned grid = static_cast<unsigned>(tn) * static_cast<unsigned>(tm);
  if (direct)
    MKO_TIMED("int8_linear_tile", s,
              tile<BN, BM, WN, WM, BK, STAGES, SPLIT, true><<<grid, WN * WM * 64, 0, s>>>(p, tn, tm));
  else
    MKO_TIMED("int8_linear_tile", s, tile<BN, BM, WN, WM, BK, 2, false, false><<<grid, WN * WM * 64, 0, s>>>(p, tn, tm));
}

// Loads straight into LDS take aligned 16-byte chunks and 32-bit offsets within a tile.  Rows that
// rmsnorm_residual_int8 and quantize_int8 wrote start at such addresses whatever their length.
bool direct_loads(const mko_int8_linear_params& p) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.w) |
                         static_cast<uintptr_t>(p.q_stride) | static_cast<uintptr_t>(p.w_stride);
  return p.inner >= 16 && bits % 16 == 0 && p.q_stride >= 0 && p.w_stride >= 0 && p.q_stride < (1 << 23) && p.w_stride < (1 << 23);
}

// The tile whose rate times the share of the last round of CUs that it fills is the largest.  The
// rates are POP/s of full rounds at inner lengths of 2560 to 5120; a lone 128 x 128 workgroup has a
// CU's four SIMDs one wave each and half the rate of two.  us, of 256 x 256, 256 x 128, 128 x 128 and
// 64 x 64 tiles:
//   8192 x 8192 x 4096: 265, 292, 331, -;   8192 x 2560 x 5120: 140, 121, 125, -;
//   1999 x 10240 x 2560: 77, 67, 68, -;     1000 x 2560 x 2560: -, 25, 20, 16.
void launch(const mko_int8_linear_params& p, hipStream_t s) {
  // `few` reads the tokens again for every 16 channels, so it is for small outputs, and without direct
  // loads for somewhat larger ones.  us, few against 64 x 64 tiles: 17 x 2560 x 2560 5.5 and 8.6, 32 x 2560 x
  // 2560 6.1 and 8.5, 48 x 2560 x 2560 7.6 and 8.6; 17 x 10240 x 2560 10.4 and 9.4, 48 x 5120 x 2560 12.3 and
  // 9.0.  Unaligned, of 256 x 1000, 256 x 1536 and 512 x 1000 outputs (1.95, 3 and 3.9 times 2^17):
  //   inner 1000:  7.5 and 11.2,   8.5 and 10.7,   9.7 and 11.3;   inner 777:   9.4 and 11.0,  11.7 and 10.6,  14.3 and 11.1;
  //   inner 2568:  9.7 and 16.1,  12.5 and 15.7,  20.4 and 16.2;   inner 5000: 18.6 and 24.1,  20.0 and 23.7,  33.6 and 24.1.
  const bool direct = direct_loads(p);
  const int64_t outputs = p.rows * p.outer;
  if (p.rows <= 16) return launch_few<1>(p, s);
  if (p.rows <= 32 && outputs <= 1 << 17) return launch_few<2>(p, s);
  if (p.rows <= 64 && outputs <= 1 << 17) return launch_few<4>(p, s);
  if (p.inner > 0 && !direct && outputs <= 3 << 17) return launch_few<2>(p, s);
  constexpr int64_t kCus = 256;
  auto score = [&](int64_t bn, int64_t bm, double rate) {
    const int64_t tiles = cdiv(p.outer, bn) * cdiv(p.rows, bm);
    return rate * static_cast<double>(tiles) / static_cast<double>(cdiv(tiles, kCus) * kCus);
  };
  const bool pairs = cdiv(p.outer, 128) * cdiv(p.rows, 128) > kCus;
  const double large = score(256, 256, 2.1), wide = score(256, 128, 1.95), middle = score(128, 128, pairs ? 1.58 : 0.85);
  const double small = score(64, 64, 1.0);
  if (large >= wide && large >= middle && large >= small) return launch_tile<256, 256, 4, 2, 128, 2, true>(p, direct, s);
  if (wide >= middle && wide >= small) return launch_tile<256, 128, 4, 2, 128, 3, true>(p, direct, s);
  if (middle >= small) return launch_tile<128, 128, 2, 2, 128, 2, false>(p, direct, s);
  launch_tile<64, 64, 2, 2, 128, 3, true>(p, direct, s);
}

int check(const mko_int8_linear_params* p) {
  if (!p || p->rows < 0 || p->inner < 0 || p->outer < 0) {
    mko_set_error("int8_linear: params is NULL or a size is negative");
    return MKO_EINVAL;
  }
  if (!half_or_float(p->dtype)) {
    mko_set_error("int8_linear: dtype must be float32, float16 or bfloat16");
    return MKO_EINVAL;
  }
  // 64 x 64 tiles of 256 threads stay within 2^32 threads
  if (p->inner > kMaxInner || p->rows > kMaxSide || p->outer > kMaxSide ||
      cdiv(p->rows, 64) * cdiv(p->outer, 64) >= (1 << 24)) {
    mko_set_error("int8_linear: inner is at most %lld, rows and outer at most %lld, and the output below 2^36 values",
                  static_cast<long long>(kMaxInner), static_cast<long long>(kMaxSide));
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
  if (!half_or_float(p->dtype)) {
    mko_set_error("quantize_int8: dtype must be float32, float16 or bfloat16");
    return MKO_EINVAL;
  }
  if (p->rows >= 1 << 22) {
    mko_set_error("quantize_int8: rows is below 2^22");
    return MKO_EUNSUPPORTED;
  }
  if (p->rows == 0) return MKO_OK;
  if (!p->scale || (p->features && !p->x) || (p->q_stride && !p->q)) {
    mko_set_error("quantize_int8: x, q (of a padding alone too) and scale are required");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == MKO_F32)
    int8::launch_quantize<float>(*p, s);
  else if (p->dtype == MKO_BF16)
    int8::launch_quantize<bf16>(*p, s);
  else
    int8::launch_quantize<_Float16>(*p, s);
  return mko_check_launch("quantize_int8");
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
  int8::launch(*p, s);
  return mko_check_launch("int8_linear");
}
