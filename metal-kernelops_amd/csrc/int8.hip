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
constexpr int64_t kMaxSide = 1 << 26;

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

// ---------------------------------------------------------------- few tokens

// A workgroup of W waves computes 16 channels of MT * 16 tokens; the waves take the inner axis in
// turns of 256 bytes, load both operands straight into the matrix cores' registers, and their
// sums are added in LDS.  The weights are read once, which is the time that this takes.
template <int MT, int W>
__global__ void __launch_bounds__(W * 64) few(mko_int8_linear_params p) {
  __shared__ __attribute__((aligned(16))) int sums[W][MT][256];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int inner = static_cast<int>(p.inner);
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t nrow = min(n0 + (lane & 15), p.outer - 1);
  const int8_t* wrow = p.w + nrow * p.w_stride;
  const int8_t* qrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    qrow[t] = p.q + min(static_cast<int64_t>(t * 16 + (lane & 15)), p.rows - 1) * p.q_stride;
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
    const int64_t m = t * 16 + (e >> 4), n = n0 + (e & 15);
    if (m >= p.rows || n >= p.outer) continue;
    int s[4] = {0, 0, 0, 0};
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += sums[w][t][e + j];
    put4(p, m, n, s, p.q_scale[m]);
  }
}

// ---------------------------------------------------------------- tiles

constexpr int kBk = 128;  // bytes of the inner axis in a stage

__device__ v4i zero_chunk;  // what a lane past the inner axis' end loads instead

template <int VM>
__device__ __forceinline__ void wait_and_meet() {
  // The waves' own loads but the last VM have landed, their LDS reads are done, and all have come here.
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
}

// A tile of BN channels by BM tokens, by WN x WM waves.  Each stage holds BK bytes of the tile's
// rows in LDS, 16-byte chunk c of row r at position c ^ (r / 2 mod 8) of its row, which spreads
// the operand reads of neighbouring rows over the banks.
template <int BN, int BM, int WN, int WM, int STAGES, bool DIRECT>
__global__ void __launch_bounds__(WN * WM * 64) tile(mko_int8_linear_params p, int tiles_n, int tiles_m) {
  constexpr int kWaves = WN * WM;
  constexpr int kTn = BN / WN / 32, kTm = BM / WM / 32;
  constexpr int kLn = BN / 8 / kWaves, kLm = BM / 8 / kWaves;  // loads of 8 rows a wave makes for a stage
  constexpr int kStage = (BN + BM) * kBk;
  __shared__ __attribute__((aligned(128))) char lds[STAGES * kStage];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wn = wave / WM, wm = wave % WM;
  const int inner = static_cast<int>(p.inner);

  // bands of 8 token tiles, token tile fastest: an XCD's workgroups share both operands in its L2
  const WgId id = wg_id(tiles_n * tiles_m, 1);
  const int band = id.x / (8 * tiles_n), in_band = id.x - band * 8 * tiles_n;
  const int band_m = min(8, tiles_m - band * 8);
  const int tn = in_band / band_m, tm = band * 8 + in_band % band_m;
  const int64_t n0 = static_cast<int64_t>(tn) * BN, m0 = static_cast<int64_t>(tm) * BM;

  const int8_t* wbase = p.w + n0 * p.w_stride;
  const int8_t* qbase = p.q + m0 * p.q_stride;
  uint32_t off[kLn + kLm];
  int chunk_k[kLn + kLm];
#pragma unroll
  for (int j = 0; j < kLn + kLm; ++j) {
    const bool wside = j < kLn;
    const int row = ((wside ? j : j - kLn) * kWaves + wave) * 8 + (lane >> 3);
    const int last = static_cast<int>(min(static_cast<int64_t>((wside ? BN : BM) - 1),
                                          (wside ? p.outer - n0 : p.rows - m0) - 1));
    chunk_k[j] = ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    off[j] = static_cast<uint32_t>(min(row, last)) * static_cast<uint32_t>(wside ? p.w_stride : p.q_stride) +
             static_cast<uint32_t>(chunk_k[j]);
  }
  const int nk = (inner + kBk - 1) / kBk;

  auto slot = [&](int st, int j) {  // where a wave's load j lands: 8 rows of a stage
    return lds + st * kStage + (j < kLn ? 0 : BN * kBk) + ((j < kLn ? j : j - kLn) * kWaves + wave) * 8 * kBk;
  };
  auto issue = [&](int st, int kt) {
    const int k0 = kt * kBk;
    const int8_t* wb = wbase + k0;
    const int8_t* qb = qbase + k0;
    if (k0 + kBk <= inner) {
#pragma unroll
      for (int j = 0; j < kLn + kLm; ++j)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) uint32_t*)((j < kLn ? wb : qb) + off[j]),
            (__attribute__((address_space(3))) uint32_t*)slot(st, j), 16, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < kLn + kLm; ++j) {
        const int8_t* src = k0 + chunk_k[j] < inner ? (j < kLn ? wb : qb) + off[j]
                                                    : reinterpret_cast<const int8_t*>(&zero_chunk);
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)src,
                                         (__attribute__((address_space(3))) uint32_t*)slot(st, j), 16, 0, 0);
      }
    }
  };
  v4i held[DIRECT ? 1 : kLn + kLm];
  auto fetch = [&](int kt) {
#pragma unroll
    for (int j = 0; j < kLn + kLm; ++j) {
      const bool wside = j < kLn;
      const int row = ((wside ? j : j - kLn) * kWaves + wave) * 8 + (lane >> 3);
      const int64_t last = min(static_cast<int64_t>((wside ? BN : BM) - 1), (wside ? p.outer - n0 : p.rows - m0) - 1);
      const int64_t r = min(static_cast<int64_t>(row), last);
      held[DIRECT ? 0 : j] =
          load_chunk(wside ? wbase + r * p.w_stride : qbase + r * p.q_stride, kt * kBk + chunk_k[j], inner);
    }
  };
  auto put_held = [&](int st) {
#pragma unroll
    for (int j = 0; j < kLn + kLm; ++j) *reinterpret_cast<v4i*>(slot(st, j) + lane * 16) = held[DIRECT ? 0 : j];
  };

  v16i acc[kTn][kTm];
#pragma unroll
  for (int i = 0; i < kTn; ++i)
#pragma unroll
    for (int j = 0; j < kTm; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  const int lr = lane & 31;
  uint32_t at[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) at[s] = lr * kBk + (((s * 2 + (lane >> 5)) ^ ((lr >> 1) & 7)) << 4);

  auto compute = [&](int st) {
    const char* wl = lds + st * kStage + wn * kTn * 32 * kBk;
    const char* ql = lds + st * kStage + BN * kBk + wm * kTm * 32 * kBk;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v4i a[kTn], b[kTm];
#pragma unroll
      for (int i = 0; i < kTn; ++i) a[i] = *reinterpret_cast<const v4i*>(wl + i * 32 * kBk + at[s]);
#pragma unroll
      for (int j = 0; j < kTm; ++j) b[j] = *reinterpret_cast<const v4i*>(ql + j * 32 * kBk + at[s]);
#pragma unroll
      for (int i = 0; i < kTn; ++i)
#pragma unroll
        for (int j = 0; j < kTm; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }
  };

  if constexpr (DIRECT) {
    // STAGES - 1 stages are on their way while one is multiplied.  Every step issues the same
    // number of loads, past the end into the stage that is free by then, so the wait's count holds.
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) issue(st, min(st, nk - 1));  // nk > 0: direct_loads()
    for (int kt = 0; kt < nk; ++kt) {
      wait_and_meet<(STAGES - 2) * (kLn + kLm)>();
      issue((kt + STAGES - 1) % STAGES, min(kt + STAGES - 1, nk - 1));
      compute(kt % STAGES);
    }
    // what was issued past the end must land before this workgroup's LDS is another's
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    fetch(0);
    put_held(0);
    for (int kt = 0; kt < nk; ++kt) {
      __syncthreads();
      if (kt + 1 < nk) fetch(kt + 1);
      compute(kt & 1);
      if (kt + 1 < nk) put_held((kt + 1) & 1);
    }
  }

#pragma unroll
  for (int j = 0; j < kTm; ++j) {
    const int64_t m = m0 + (wm * kTm + j) * 32 + lr;
    if (m >= p.rows) continue;
    const float qs = p.q_scale[m];
#pragma unroll
    for (int i = 0; i < kTn; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t n = n0 + (wn * kTn + i) * 32 + 8 * g + 4 * (lane >> 5);
        const int s[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        if (n < p.outer) put4(p, m, n, s, qs);
      }
  }
}

// ---------------------------------------------------------------- the choice

template <int MT>
void launch_few(const mko_int8_linear_params& p, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(cdiv(p.outer, 16));
  const int64_t turns = cdiv(p.inner, 256);
  if (turns <= 4 || grid >= 2048)
    MKO_TIMED("int8_linear_few", s, few<MT, 4><<<grid, 4 * 64, 0, s>>>(p));
  else
    MKO_TIMED("int8_linear_few", s, few<MT, 8><<<grid, 8 * 64, 0, s>>>(p));
}

template <int BN, int BM, int WN, int WM, int STAGES>
void launch_tile(const mko_int8_linear_params& p, bool direct, hipStream_t s) {
  const int64_t tn = cdiv(p.outer, BN), tm = cdiv(p.rows, BM);
  const unsigned grid = static_cast<unsigned>(tn * tm);
  if (direct)
    MKO_TIMED("int8_linear_tile", s,
              tile<BN, BM, WN, WM, STAGES, true><<<grid, WN * WM * 64, 0, s>>>(
                  p, static_cast<int>(tn), static_cast<int>(tm)));
  else
    MKO_TIMED("int8_linear_tile", s,
              tile<BN, BM, WN, WM, 2, false><<<grid, WN * WM * 64, 0, s>>>(p, static_cast<int>(tn),
                                                                              static_cast<int>(tm)));
}

// Loads straight into LDS take aligned 16-byte chunks and 32-bit offsets within a tile.
bool direct_loads(const mko_int8_linear_params& p) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.w) |
                         static_cast<uintptr_t>(p.q_stride) | static_cast<uintptr_t>(p.w_stride) |
                         static_cast<uintptr_t>(p.inner);
  return p.inner > 0 && bits % 16 == 0 && p.q_stride >= 0 && p.w_stride >= 0 && p.q_stride < (1 << 23) && p.w_stride < (1 << 23);
}

void launch(const mko_int8_linear_params& p, hipStream_t s) {
  if (p.rows <= 16) return launch_few<1>(p, s);
  if (p.rows <= 32) return launch_few<2>(p, s);
  if (p.rows <= 64) return launch_few<4>(p, s);
  const bool direct = direct_loads(p);
  if (cdiv(p.rows, 256) * cdiv(p.outer, 256) >= 200) return launch_tile<256, 256, 2, 4, 2>(p, direct, s);
  if (cdiv(p.rows, 128) * cdiv(p.outer, 128) >= 200) return launch_tile<128, 128, 2, 2, 2>(p, direct, s);
  launch_tile<64, 64, 2, 2, 3>(p, direct, s);
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
  int8::launch(*p, s);
  return mko_check_launch("int8_linear");
}
