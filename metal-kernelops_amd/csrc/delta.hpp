// Gated delta rule for gfx950: what its kernels share.
//
// Per (batch, value head), with state S (value x key) and c the running sum of the log decay:
//   e_t = v_t - exp(g_t) S_{t-1} k_t,  S_t = exp(g_t) S_{t-1} + beta_t e_t k_t^T,  y_t = scale S_t q_t
// In a chunk of 64 tokens with entering state S0 the e of all tokens solve one triangular system:
//   A[t][s] = exp(c_t - c_s) (k_t . k_s) beta_s for s < t,  T = (I + A)^-1
//   E = T (V - exp(c) K S0^T),  P[t][s] = scale exp(c_t - c_s) (q_t . k_s) beta_s for s <= t
//   Y = scale exp(c) Q S0^T + P E,  S' = exp(c_63) S0 + E^T (beta exp(c_63 - c) K)
//
// Everything runs on 16x16 tiles of the matrix cores, whose accumulator layout (lane l holds column
// l % 16, rows 4 (l / 16) + r) is also an operand layout for the next product that contracts over
// those rows: two row tiles make the eight elements a lane of an operand over 32 rows.  So a chain of
// products stays in registers, and only the other operand has to be read in that order.  Which key
// stands in which row of a state's tile is free: row 4 a + r of tile (j, h) is key 32 j + 8 a + 4 h + r,
// which makes the operand's eight elements consecutive in memory.  Tokens stand in their own order.
#pragma once

#include "io.hpp"
#include "rows.hpp"

namespace mko {
namespace delta {

constexpr int kC = 64;             // tokens of a chunk
constexpr int kFrag = 512;         // elements of a 16 x 32 operand
constexpr int kSquare = 6 * kFrag; // elements of a triangular 64 x 64 operand without its empty blocks

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Sizes and strides, in elements.
struct Geo {
  int64_t batch, length, key_heads, heads, key, value;
  int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;
  int64_t chunks;    // of a sequence
  int64_t segments;  // that the forward walks side by side
  int64_t span;      // chunks of a segment, the last one's at most
  int rep;         // value heads of a key head
  float scale;
  int dtype, decay_dtype, beta_dtype, state_dtype;
};

// Per chunk and head, in float32 after 64 doubles: exp(c), beta exp(c_63 - c), exp(c_63 - c) and beta of
// its tokens.
struct Tokens {
  double c[kC];  // c log2(e)
  float in[kC], write[kC], out[kC], beta[kC];
};

struct Ptrs {
  const void *q, *k, *v, *decay, *beta, *initial, *dy, *dfinal;
  void *y, *final_state, *dq, *dk, *dv, *ddecay, *dbeta, *dinitial;
  Tokens* tokens;        // (batch, heads, chunks)
  void *lower, *upper;   // T and P as operands, and their transposes, (batch, heads, chunks, 2, kSquare)
  void *states, *grads;  // S0 and the gradient of S' of each chunk, (batch, heads, chunks, value, key)
  void* e;               // E, (batch, heads, chunks, kC, value)
  float *pq, *pk;        // dq and dk of each value head, where key heads are shared
  float* ends;           // states behind the segments but the last, (batch, heads, segments - 1, value, key)
  // What a segment makes of the state before it, but for its decay: (batch, heads, segments - 1, key, key), and the
  // decay, (batch, heads, segments - 1)
  float *maps, *kept;
};

// A lane's share of a 16 x 32 operand: row (or column) l % 16.  Over tokens element 4 h + r is index
// 16 h + 4 (l / 16) + r of the contraction, over keys and values element e is index 8 (l / 16) + e.
template <typename TM>
struct Frag {
  uint32_t w[kWordsOf<TM, 8>];
};

// acc += a b over the 32 indices.
template <typename TM>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<TM>& a, const Frag<TM>& b) {
  if constexpr (sizeof(TM) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w[e]), __uint_as_float(b.w[e]), acc, 0, 0, 0);
  } else if constexpr (__is_same(TM, bf16)) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
  }
}

// Two accumulators (rows 0..15 and 16..31) as an operand, rounded to TM.
template <typename TM>
__device__ __forceinline__ Frag<TM> frag_of(const f32x4& lo, const f32x4& hi) {
  const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  Frag<TM> r;
  pack_words<TM, 8>(f, r.w);
  return r;
}

__device__ __forceinline__ int lane_id() { return threadIdx.x & (kWave - 1); }
// The lane's number as a value of its own: addresses formed from it are not kept in registers from
// one part of a kernel to the next.
__device__ __forceinline__ int lane_again() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l & (kWave - 1);
}
__device__ __forceinline__ int lane_col() { return threadIdx.x & 15; }         // l % 16
__device__ __forceinline__ int lane_quad() { return (threadIdx.x >> 4) & 3; }  // l / 16

// Operand rows r0 .. r0 + 15, contraction indices k0 .. k0 + 31 in memory's order (both operands
// read this way); rows from `rows` and columns from `cols` on are zero and not read.
template <typename TM>
__device__ __forceinline__ Frag<TM> frag_memory(const TM* base, int64_t stride, int r0, int k0, int rows, int cols) {
  const int row = r0 + lane_col(), col = k0 + 8 * lane_quad();
  const Words<TM, 8> w = load_part<TM, 8>(base + (row < rows ? row * stride : 0), col, row < rows ? cols : 0);
  return __builtin_bit_cast(Frag<TM>, w);
}

// 16 bytes a lane from memory to LDS, to `to` + 16 lane bytes (`to` the same in the wave), in flight until
// the wave waits for its vector memory operations.  In assembly because the compiler would wait for all
// of them ahead of the next LDS read, whatever it reads; it counts fewer operations than there are,
// so its own waits only last longer.  One idle state from the write of m0 to its use by the load; nothing else in
// these kernels uses m0, which cannot be named as overwritten.
__device__ __forceinline__ void direct_load(const void* from, void* to) {
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to));  // a flat address ends in that of LDS
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(uniform(at)), "v"(from));
}

// A pointer that is the same in the wave, in scalar registers.
using mko::uniform;
__device__ __forceinline__ const char* uniform(const void* p) {
  const uint64_t a = reinterpret_cast<uintptr_t>(p);
  const uint64_t lo = static_cast<uint32_t>(uniform(static_cast<int>(a))), hi = static_cast<uint32_t>(uniform(static_cast<int>(a >> 32)));
  return reinterpret_cast<const char*>(hi << 32 | lo);
}

// The same from `base` (the same in the wave) + `off` bytes.
__device__ __forceinline__ void direct_load(const void* base, uint32_t off, const void* to) {
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uniform(at)), "v"(off),
               "s"(uniform(base)));
}

// Every direct load of the workgroup has landed.
__device__ __forceinline__ void direct_wait() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// ---- tiles in LDS

// A ROWS x COLS tile in units of 16 bytes.  Unit u of row r is at place u ^ turn(r) of its row: the 16
// rows that an operand read touches at one unit, and the four rows of four units that a transposing
// read touches, then lie in different banks.
template <typename TM, int COLS, int ROWS = kC>
struct Tile {
  static constexpr int kUnit = 16 / static_cast<int>(sizeof(TM));  // elements
  static constexpr int kUnits = COLS / kUnit;                      // of a row
  static constexpr int kElements = ROWS * COLS;

  static __device__ __forceinline__ int turn(int row) {
    if constexpr (kUnits >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    if constexpr (kUnits == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
    return (row >> 2) & (kUnits - 1);
  }
  static __device__ __forceinline__ int at(int row, int col) {
    return (row * kUnits + ((col / kUnit) ^ turn(row))) * kUnit + col % kUnit;
  }

  // Operand rows r0 .. r0 + 15, contraction over the columns k0 .. k0 + 31 in memory's order.
  static __device__ __forceinline__ Frag<TM> rows(const TM* tile, int r0, int k0, int lane = lane_id()) {
    const int row = r0 + lane % 16, col = k0 + 8 * (lane / 16);
    Frag<TM> f;
    if constexpr (sizeof(TM) == 2) {
      load_words(tile + at(row, col), f.w);
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(tile + at(row, col));
      const uint4 b = *reinterpret_cast<const uint4*>(tile + at(row, col + 4));
      f.w[0] = a.x; f.w[1] = a.y; f.w[2] = a.z; f.w[3] = a.w;
      f.w[4] = b.x; f.w[5] = b.y; f.w[6] = b.z; f.w[7] = b.w;
    }
    return f;
  }

  // Rows r .. r + 3 of column c0 + step (m / 4) + m % 4 with m = l % 16, as words; r is the quad's own.
  // In 16 bits the hardware transposes: of sixteen lanes, lane 4 i + j hands in row r + i, columns
  // c0 + step j ..
  static __device__ __forceinline__ void column(const TM* tile, int r, int c0, int step, uint32_t (&w)[kWordsOf<TM, 4>],
                                                int lane) {
    const int m = lane % 16;
    if constexpr (sizeof(TM) == 2) {
      typedef __attribute__((address_space(3))) s16x4* lds_at;
      const TM* p = tile + at(r + (m >> 2), c0 + step * (m & 3));
      const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_at)p));
      w[0] = v.x;
      w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, tile[at(r + i, c0 + step * (m >> 2) + (m & 3))]);
    }
  }
  static __device__ __forceinline__ Frag<TM> columns(const TM* tile, int lo, int hi, int c0, int step, int lane) {
    constexpr int W = kWordsOf<TM, 4>;
    uint32_t a[W], b[W];
    column(tile, lo, c0, step, a, lane);
    column(tile, hi, c0, step, b, lane);
    Frag<TM> f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      f.w[i] = a[i];
      f.w[W + i] = b[i];
    }
    return f;
  }
  // Operand over the tokens r0 .. r0 + 31 (the tile's rows), its rows the columns c0 .. c0 + 15.
  static __device__ __forceinline__ Frag<TM> over_tokens(const TM* tile, int r0, int c0, int lane = lane_id()) {
    const int r = r0 + 4 * (lane / 16);
    return columns(tile, r, r + 16, c0, 4, lane);
  }
  // The same with a key tile's columns: i = 2 j + h.
  static __device__ __forceinline__ Frag<TM> keys_over_tokens(const TM* tile, int r0, int i, int lane = lane_id()) {
    const int r = r0 + 4 * (lane / 16);
    return columns(tile, r, r + 16, 16 * (i & ~1) + 4 * (i & 1), 8, lane);
  }
  // And over the values r0 .. r0 + 31, where the tile's rows are values.
  static __device__ __forceinline__ Frag<TM> keys_over_values(const TM* tile, int r0, int i, int lane = lane_id()) {
    const int r = r0 + 8 * (lane / 16);
    return columns(tile, r, r + 4, 16 * (i & ~1) + 4 * (i & 1), 8, lane);
  }
  // The tile's values in the accumulator layout: rows r0 .., columns c0 ...
  static __device__ __forceinline__ f32x4 values(const TM* tile, int r0, int c0) {
    uint32_t w[kWordsOf<TM, 4>];
    float f[4];
    column(tile, r0 + 4 * lane_quad(), c0, 4, w, lane_id());
    unpack_words<TM, 4>(w, f);
    return f32x4{f[0], f[1], f[2], f[3]};
  }

  // The tile from memory, complete after a wait for the wave's loads and a barrier.
  template <int WAVES, bool FAST>
  static __device__ __forceinline__ void load(TM* tile, const TM* base, int64_t stride, int rows, int cols, int wave,
                                              const TM* zeros) {
    if constexpr (FAST)
      issue<WAVES>(tile, base, stride, rows, cols, wave, zeros);
    else
      copy<64 * WAVES>(tile, base, stride, rows, cols);
  }

  // From memory through registers; rows from `rows` and columns from `cols` on become zero.
  template <int THREADS>
  static __device__ __forceinline__ void copy(TM* tile, const TM* base, int64_t stride, int rows, int cols) {
    for (int i = static_cast<int>(threadIdx.x); i < ROWS * kUnits; i += THREADS) {
      const int row = i / kUnits, col = i % kUnits * kUnit;
      const Words<TM, kUnit> w = load_part<TM, kUnit>(base + (row < rows ? row * stride : 0), col, row < rows ? cols : 0);
      store_words(tile + at(row, col), w.w);
    }
  }

  // The same without registers: wave `wave` of WAVES issues its share of the loads.  Rows are whole
  // units at multiples of 16 bytes; units outside come from `zeros`.
  template <int WAVES>
  static __device__ __forceinline__ void issue(TM* tile, const TM* base, int64_t stride, int rows, int cols, int wave,
                                               const TM* zeros) {
    constexpr int kLoads = ROWS * kUnits / kWave;
    static_assert(kLoads % WAVES == 0 || kLoads < WAVES, "an equal share of the loads");
    if (kLoads < WAVES && wave >= kLoads) return;
#pragma unroll
    for (int j = 0; j < (kLoads + WAVES - 1) / WAVES; ++j) {
      const int load = j * WAVES + wave, i = load * kWave + lane_id(), row = i / kUnits;
      const int col = ((i % kUnits) ^ turn(row)) * kUnit;
      direct_load(row < rows && col < cols ? base + row * stride + col : zeros, tile + load * kWave * kUnit);
    }
  }
};

// A wave's share of the loads of whole-row tiles, with what is the same for every tile worked out once: a
// lane's offsets repeat every 16 rows, and what differs between loads beyond that is the same in the wave.
// Columns from `cols` on are left as they are.
template <typename TM, int COLS, int WAVES>
struct Lines {
  typedef Tile<TM, COLS> T;
  static constexpr int kRows = kWave / T::kUnits;                       // of a load
  static constexpr int kLoads = kC * T::kUnits / kWave;                 // of a tile
  static constexpr int kMine = (kLoads + WAVES - 1) / WAVES;            // of a wave, one for the first kLoads waves
  static constexpr int kTurns = 16 / kRows / WAVES > 1 ? 16 / kRows / WAVES : 1;  // loads of a wave until offsets repeat
  uint32_t off[kTurns];
  bool in[kTurns];
  int64_t bytes;  // from a load of the wave to the next

  __device__ __forceinline__ Lines(int64_t stride, int cols, int wave) {
    static_assert(kLoads % WAVES == 0 || kLoads < WAVES, "an equal share of the loads");
    const int row = lane_id() / T::kUnits, unit = lane_id() % T::kUnits;
#pragma unroll
    for (int j = 0; j < kTurns; ++j) {
      const int load = j * WAVES + wave, col = (unit ^ T::turn(load * kRows + row)) * T::kUnit;
      off[j] = static_cast<uint32_t>((row * stride + col) * static_cast<int>(sizeof(TM)));
      in[j] = col < cols && load < kLoads;
    }
    bytes = WAVES * kRows * stride * static_cast<int64_t>(sizeof(TM));
  }
  // All 64 rows at `base`, of the same stride.
  __device__ __forceinline__ void issue(TM* tile, const TM* base, int wave) const {
    const char* at = reinterpret_cast<const char*>(base) + wave * (bytes / WAVES);
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      if (in[j % kTurns]) direct_load(at, off[j % kTurns], tile + (j * WAVES + wave) * kWave * T::kUnit);
      at += bytes;
    }
  }
};

// Place of the operand of row tile i and contraction block j in a square: of the lower triangle
// (j <= i / 2) or of its transpose (j >= i / 2).
__host__ __device__ constexpr int lower_at(int i, int j) { return (i < 2 ? i : 2 * i - 2 + j) * kFrag; }
__host__ __device__ constexpr int upper_at(int i, int j) { return (i < 2 ? 2 * i + j : i + 2) * kFrag; }

// Such an operand: eight elements a lane.
template <typename TM>
__device__ __forceinline__ Frag<TM> frag_at(const TM* p) {
  Frag<TM> f;
  load_words(p + 8 * lane_id(), f.w);
  return f;
}

// What a workgroup holds in LDS of the chunks it walks: K, a slice of V or dY, exp(c) and beta exp(c_63 - c);
// SQUARES: one or two triangular squares, Q.  More than one buffer: the loads of the chunks ahead fly while
// one is worked on.  One: it is filled between two barriers.
template <typename TM, int KB, int BV, int BUFS, int SQUARES, bool Q>
struct Chunks {
  static constexpr int kBufs = BUFS, kSquares = SQUARES;
  static constexpr bool kQ = Q;
  typedef Tile<TM, 32 * KB> KTile;
  typedef Tile<TM, BV> VTile;
  struct Buf {
    TM k[KTile::kElements], v[VTile::kElements];
    float in[kC], write[kC];
    TM squares[SQUARES > 0 ? SQUARES * kSquare : 8], q[Q ? KTile::kElements : 8];
  };
  static_assert(sizeof(Buf) % 16 == 0, "every tile starts at a multiple of 16 bytes");
  Buf bufs[BUFS];
  // That of the n-th chunk of the walk.
  __device__ __forceinline__ Buf& buf(int64_t n) { return bufs[BUFS == 1 ? 0 : static_cast<uint32_t>(n) % BUFS]; }

  // Keys that no load fills become zero.
  __device__ __forceinline__ void clear(int threads) {
    constexpr int kUnits = KTile::kElements / KTile::kUnit;
    for (int i = static_cast<int>(threadIdx.x); i < BUFS * kUnits; i += threads) {
      const uint32_t none[4] = {0, 0, 0, 0};
      const int at = i % kUnits * KTile::kUnit;
      store_words(bufs[i / kUnits].k + at, none);
      if constexpr (Q) store_words(bufs[i / kUnits].q + at, none);
    }
    __syncthreads();
  }
};

// Where a head's chunks are.
template <typename TM>
struct Source {
  const TM *k, *q, *v;
  int64_t k_t, q_t, v_t, length;
  const Tokens* tokens;
  const TM* squares;  // two of a chunk
  int key, value;     // columns of K and Q, and of this slice
  __device__ __forceinline__ int rows(int64_t c) const {
    return static_cast<int>(min(static_cast<int64_t>(kC), length - c * kC));
  }
};

// Waves that do nothing but fetch: a wave issues a direct load in about 75 cycles, so one alone brings 13.6
// bytes a cycle to LDS, two 25.7 and four, one on each SIMD, 44; eight no more (64 KB of rows of 256 bytes in L2,
// 256 workgroups).
constexpr int kFetchers = 4;

template <typename TM, int KB, int BV, typename Lds>
struct Fetcher {
  static constexpr int F = kFetchers;
  typedef Tile<TM, 32 * KB> KTile;
  typedef Tile<TM, BV> VTile;
  typedef Lines<TM, 32 * KB, F> KLines;
  typedef Lines<TM, BV, F> VLines;
  static constexpr int kPer = 16 / static_cast<int>(sizeof(TM)) * kWave;  // elements of a load
  static constexpr int kSquareLoads = Lds::kSquares * kSquare / kPer / F;
  static_assert(Lds::kSquares * kSquare % (kPer * F) == 0 || Lds::kSquares == 1, "an equal share of the squares");
  // direct loads of a chunk, of each wave at least
  static constexpr int kLoads =
      (Lds::kQ ? 2 : 1) * KLines::kMine + (VLines::kLoads >= F ? VLines::kMine : 0) + kSquareLoads;
  static constexpr int kFly = Lds::kBufs - 2;  // chunks on their way beside the next
  static_assert(kFly * kLoads < 64, "the count of loads on their way has six bits");

  const Source<TM>& src;
  const TM* zeros;
  int part;
  KLines k_lines, q_lines;
  VLines v_lines;
  __device__ __forceinline__ Fetcher(const Source<TM>& s, const TM* z, int p)
      : src(s), zeros(z), part(p), k_lines(s.k_t, s.key, p), q_lines(s.q_t, s.key, p), v_lines(s.v_t, s.value, p) {}

  __device__ __forceinline__ void keys(typename Lds::Buf& b, int64_t c) const {
    if (src.rows(c) == kC)
      k_lines.issue(b.k, src.k + c * kC * src.k_t, part);
    else
      KTile::template issue<F>(b.k, src.k + c * kC * src.k_t, src.k_t, src.rows(c), src.key, part, zeros);
  }
  __device__ __forceinline__ void rest(typename Lds::Buf& b, int64_t c) const {
    if (part == 0 && lane_id() < 2 * kC / 4) direct_load(src.tokens[c].in + 4 * lane_id(), b.in);
    if (src.rows(c) == kC) {
      v_lines.issue(b.v, src.v + c * kC * src.v_t, part);
      if constexpr (Lds::kQ) q_lines.issue(b.q, src.q + c * kC * src.q_t, part);
    } else {
      VTile::template issue<F>(b.v, src.v + c * kC * src.v_t, src.v_t, src.rows(c), src.value, part, zeros);
      if constexpr (Lds::kQ)
        KTile::template issue<F>(b.q, src.q + c * kC * src.q_t, src.q_t, src.rows(c), src.key, part, zeros);
    }
#pragma unroll
    for (int i = 0; i < (Lds::kSquares * kSquare + kPer * F - 1) / (kPer * F); ++i) {  // the second behind the first
      const int f = (i * F + part) * kPer;
      if (f < Lds::kSquares * kSquare) direct_load(src.squares + c * 2 * kSquare + f, 16u * lane_id(), b.squares + f);
    }
  }
  // The chunks first, first + step, ..., n of them; a barrier each, MORE of them at the end, and MID: another
  // within each turn.  `take(i)` and `put(i)` are what else the wave does in turn i, ahead of and after that; vector
  // memory operations of theirs only make the waits here longer.
  template <bool MID, int MORE, typename Take, typename Put>
  __device__ __forceinline__ void walk(Lds& lds, int64_t first, int64_t step, int64_t n, Take take, Put put) const {
    for (int64_t i = 0; i <= kFly && i < n; ++i) {
      keys(lds.buf(i), first + i * step);
      rest(lds.buf(i), first + i * step);
    }
    for (int64_t i = 0; i < n + MORE; ++i) {
      // Of this wave's vector memory operations, which end in their order, only the chunks' behind i are
      // still on their way, and at the end none; then everyone's.
      if (i + kFly < n)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kFly * kLoads) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      take(i);
      const int64_t j = i + kFly + 1, c = first + j * step;
      if (j < n) keys(lds.buf(j), c);
      if constexpr (MID) __syncthreads();
      if (j < n) rest(lds.buf(j), c);
      put(i);
    }
  }
};

// A state over the keys and a chunk's rows over the tokens as operands, from the wave that carries to those that
// store them.
template <typename TM, int KB>
struct Hand {
  TM s[KB * kFrag], e[2 * kFrag];
};
template <typename TM>
__device__ __forceinline__ void put_frag(TM* p, const Frag<TM>& f) {
  store_words(p + 8 * lane_id(), f.w);
}
template <typename TM, int KB>
__device__ __forceinline__ void hand_over(Hand<TM, KB>& hand, const Frag<TM> (&s)[KB], const Frag<TM> (&e)[2]) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) put_frag(hand.s + kb * kFrag, s[kb]);
  put_frag(hand.e, e[0]);
  put_frag(hand.e + kFrag, e[1]);
}

// A chunk through registers, by all THREADS.
template <int THREADS, typename TM, typename Lds>
__device__ __forceinline__ void copy_chunk(typename Lds::Buf& b, const Source<TM>& src, int64_t c) {
  Lds::KTile::template copy<THREADS>(b.k, src.k + c * kC * src.k_t, src.k_t, src.rows(c), src.key);
  if constexpr (Lds::kQ) Lds::KTile::template copy<THREADS>(b.q, src.q + c * kC * src.q_t, src.q_t, src.rows(c), src.key);
  Lds::VTile::template copy<THREADS>(b.v, src.v + c * kC * src.v_t, src.v_t, src.rows(c), src.value);
  for (int i = static_cast<int>(threadIdx.x); i < 2 * kC; i += THREADS) b.in[i] = src.tokens[c].in[i];
}

// N values at element i of a row of n, those below n; WHOLE: n is a multiple of N.
template <typename T, bool WHOLE, int N>
__device__ __forceinline__ void store_run(T* row, int i, int n, const float (&f)[N]) {
  if constexpr (WHOLE) {
    AnyWords<T, N> o;
    pack_words<T, N>(f, o.v.w);
    if (i < n) *reinterpret_cast<AnyWords<T, N>*>(row + i) = o;
  } else {
    store_part<T, N>(row, i, n, f);
  }
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store_four(T* row, int i, int n, const f32x4& v) {
  const float f[4] = {v[0], v[1], v[2], v[3]};
  store_run<T, WHOLE>(row, i, n, f);
}

// Two key tiles of a lane's state row: keys 32 j + 8 (l / 16) ..
template <typename T, bool WHOLE, int N>
__device__ __forceinline__ void load_row(f32x4 (&s)[N], const T* row, int n) {
  Words<T, 8> w[N / 2];
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const int at = 32 * j + 8 * lane_quad();
    if constexpr (WHOLE)
      w[j] = reinterpret_cast<const AnyWords<T, 8>*>(row + (at < n ? at : 0))->v;
    else
      w[j] = load_part<T, 8>(row, at, n);
  }
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    float f[8];
    unpack_words<T, 8>(w[j].w, f);
    const bool in = 32 * j + 8 * lane_quad() < n;
    s[2 * j] = in ? f32x4{f[0], f[1], f[2], f[3]} : f32x4{0, 0, 0, 0};
    s[2 * j + 1] = in ? f32x4{f[4], f[5], f[6], f[7]} : f32x4{0, 0, 0, 0};
  }
}
template <bool WHOLE, int N>
__device__ __forceinline__ void load_state(f32x4 (&s)[N], const void* p, int dtype, int64_t row, int n) {
  if (dtype == MKO_F32)
    load_row<float, WHOLE>(s, static_cast<const float*>(p) + row, n);
  else if (dtype == MKO_BF16)
    load_row<bf16, WHOLE>(s, static_cast<const bf16*>(p) + row, n);
  else
    load_row<_Float16, WHOLE>(s, static_cast<const _Float16*>(p) + row, n);
}
template <typename T, bool WHOLE, int N>
__device__ __forceinline__ void store_row(T* row, int n, const f32x4 (&s)[N]) {
#pragma unroll
  for (int j = 0; j < N / 2; ++j) {
    const f32x4 &a = s[2 * j], &b = s[2 * j + 1];
    const float f[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    store_run<T, WHOLE>(row, 32 * j + 8 * lane_quad(), n, f);
  }
}
template <bool WHOLE, int N>
__device__ __forceinline__ void store_state(void* p, int dtype, int64_t row, int n, const f32x4 (&s)[N]) {
  if (dtype == MKO_F32)
    store_row<float, WHOLE>(static_cast<float*>(p) + row, n, s);
  else if (dtype == MKO_BF16)
    store_row<bf16, WHOLE>(static_cast<bf16*>(p) + row, n, s);
  else
    store_row<_Float16, WHOLE>(static_cast<_Float16*>(p) + row, n, s);
}

// The same of a state as operands, in TM.
template <typename TM, bool WHOLE, int KB>
__device__ __forceinline__ void store_operands(TM* row, int n, const Frag<TM>* s) {
#pragma unroll
  for (int j = 0; j < KB; ++j) {
    const int at = 32 * j + 8 * lane_quad();
    if constexpr (WHOLE) {
      if (at < n) *reinterpret_cast<AnyWords<TM, 8>*>(row + at) = __builtin_bit_cast(AnyWords<TM, 8>, s[j]);
    } else {
      float f[8];
      unpack_words<TM, 8>(s[j].w, f);
      store_part<TM, 8>(row, at, n, f);
    }
  }
}

// Halves of the unit matrix as operands, which transpose rows over tokens exactly.
template <typename TM>
__device__ __forceinline__ void unit_halves(Frag<TM> (&one)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f32x4 x[2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[0][r] = i == 0 && 4 * lane_quad() + r == lane_col() ? 1.0f : 0.0f;
      x[1][r] = i == 1 && 4 * lane_quad() + r == lane_col() ? 1.0f : 0.0f;
    }
    one[i] = frag_of<TM>(x[0], x[1]);
  }
}
// Rows over tokens to memory: token t's at to + t stride, its values from v on, of the first `rows` tokens.
template <typename TM, bool WHOLE, typename Stride>
__device__ __forceinline__ void store_rows(TM* to, Stride stride, int v, int value, int rows, const Frag<TM>* e,
                                           const Frag<TM> (&one)[2]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x4 et = {0, 0, 0, 0};  // [value][token], whose lanes hold four values of a token
    mma(et, e[i / 2], one[i % 2]);
    if (16 * i + lane_col() < rows) store_four<TM, WHOLE>(to + (16 * i + lane_col()) * stride, v + 4 * lane_quad(), value, et);
  }
}

// What the waves that fetch do beside: two tiles of 16 values, for each of them one wave stores the states and another
// the rows that were handed over in the turn before.
template <typename TM, int KB>
struct Storer {
  Frag<TM> f[KB > 2 ? KB : 2], one[2];
  int tile;
  bool rows;
  __device__ __forceinline__ explicit Storer(int part) : tile(part & 1), rows(part >> 1) { unit_halves<TM>(one); }
  __device__ __forceinline__ void take(const Hand<TM, KB>& hand) {
#pragma unroll
    for (int i = 0; i < (KB > 2 ? KB : 2); ++i) {
      if (rows ? i < 2 : i < KB) f[i] = frag_at((rows ? hand.e : hand.s) + i * kFrag);
    }
  }
};

// Bytes of the arrays that the forward leaves for the backward, and of the workspaces.
struct Layout {
  size_t tokens, lower, upper, states, e, ends, maps, kept, total;
};
Layout saved_layout(const Geo& g);                // tokens, upper, states, e
Layout forward_layout(const Geo& g, bool train);  // lower, ends, maps and kept, and tokens unless they are saved

int make_geo(const mko_delta_params* prm, const char* what, Geo* g);
Ptrs base_ptrs(const mko_delta_params* prm);
// Whether q, k, v and dy can be loaded to LDS directly: rows of whole 16-byte units at multiples of 16 bytes.
bool fast_rows(const Geo& g, const Ptrs& p);

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }
inline size_t element_size(int dtype) { return dtype == MKO_F32 ? 4 : 2; }

}  // namespace delta
}  // namespace mko
