// Gated linear recurrence for gfx950.
//
// Per channel, with rate = scale softplus(decay):
//   v = rate s(rg),  a = e^-v,  m = sqrt(1 - e^-2v),  h[t] = a h[t-1] + m s(ig) x
// Backward, with g[t] = dy[t] + a[t+1] g[t+1]:
//   dx = g m s(ig),  dig = g m x s(ig) (1 - s(ig)),  drg = dv v (1 - s(rg)),
//   dv = g (s(ig) x a^2 / m - a h[t-1]),  ddecay = scale s(decay) sum(dv s(rg))
//
// One pass over the data in each direction, the sequence split into chunks of 64 steps that are joined
// as they are computed (see "the chunks' order"), so that a value is read once, stays in registers, and
// a few long sequences still fill the chip.  Of 4 x 4096 x 2560 bf16 the forward takes 79 us (4.3 TB/s) and
// the backward 129 (4.6 TB/s): the exponentials, reciprocals and roots, six of 28 vector instructions a
// value, take about 54 and 94 us of issue beside the bytes' 54 and 94 at the copy rate.  Chunks of 128
// steps took 126 us forward and 184 backward where 64 took 102 and 175; of 32 steps, 142 and 167.
#include <type_traits>

#include "common.hpp"
#include "rows.hpp"

namespace mko {
namespace recur {
namespace {

constexpr int kChunk = MKO_RECUR_CHUNK;
constexpr int kThreads = 256;
constexpr int kV = 2;  // channels a lane of the scans takes
constexpr int64_t kMostBatch = 65535, kMostSide = int64_t{1} << 31;
constexpr int64_t kMostWorkgroups = int64_t{1} << 22;  // of 512 threads: 2^31 threads in a launch

// A channel's rate in units of the binary exponential: v log2(e) = rate s(rg).
__device__ __forceinline__ float binary_rate(float scale, float decay) { return scale * kLog2e * softplus(decay); }

// 1 - 2^-2u from u and a = 2^-u.  Below u = 1/4 / ln 2, where 1 - a^2 would cancel, u times a fourth
// degree polynomial fitted to (1 - 2^-2u) / u there at Chebyshev points (8.4e-8 relative).
__device__ __forceinline__ float one_minus_square(float u, float a) {
  const float s =
      u * (1.3862942457f + u * (-0.9608914256f + u * (0.4437149763f + u * (-0.1514232010f + u * 0.0346555375f))));
  return u < 0.25f / kLn2 ? s : 1.0f - a * a;
}

struct Step {
  float si, sr, a, m;
};

// `rate` from binary_rate().
__device__ __forceinline__ Step gates(float ig, float rg, float rate, bool reset) {
  Step s;
  s.si = sigmoid(ig);
  s.sr = sigmoid(rg);
  const float u = rate * s.sr;
  s.a = fast_exp2(-u);
  s.m = __builtin_amdgcn_sqrtf(one_minus_square(u, s.a));
  if (reset) {  // nothing of the decay gate is used, a NaN in it included
    s.a = s.sr = 0.0f;
    s.m = 1.0f;
  }
  return s;
}

// ---------------------------------------------------------------- a channel strip's chunk
//
// A workgroup takes kChunk steps of a strip of 64 V channels: lane l the channels l V .. l V + V - 1,
// wave w the steps w T .. w T + T - 1.  A run of steps maps the state before it to the state after
// it by h -> P h + H, and runs compose; with resets, a run that drops the state has P = -0, which
// no product of decays gives and which stays -0 when decays multiply it.

constexpr uint32_t kDropped = 0x80000000u;

template <bool RESET>
__device__ __forceinline__ bool drops(float P) {
  return RESET && __float_as_uint(P) == kDropped;
}

// P h + H; a dropped h is not read, be it NaN.
template <bool RESET>
__device__ __forceinline__ float apply(float P, float H, float h) {
  const float r = P * h + H;
  return drops<RESET>(P) ? H : r;
}

// The decays' product over a run and the run beside it.
template <bool RESET>
__device__ __forceinline__ float both(float P, float Q) {
  const float r = P * Q;
  return drops<RESET>(P) || drops<RESET>(Q) ? __uint_as_float(kDropped) : r;
}

template <typename T, int V>
struct Raw {
  static_assert(V == 2, "a word of 16-bit values");
  uint32_t w[sizeof(T) == 4 ? V : 1];
};

// Where a lane's channels are.  What is the same for a wave (the strip's first channel, a row's
// address) stays apart from the lane's 32-bit offset, so that an access needs one register for its
// address instead of two.
template <bool FULL>
struct Place {
  int64_t first;   // of the strip
  uint32_t off;    // of the lane's first channel in the strip
  uint32_t count;  // channels of the strip; FULL: 64 V in every one
  __device__ __forceinline__ uint32_t at(int e) const { return FULL ? off + e : min(off + e, count - 1); }  // to read
  __device__ __forceinline__ bool has(int e) const { return FULL || off + e < count; }
};

template <int V, bool FULL>
__device__ __forceinline__ Place<FULL> place(int64_t strip, int64_t channels, int lane) {
  const int64_t first = strip * 64 * V;
  const uint32_t count = static_cast<uint32_t>(min(static_cast<int64_t>(64 * V), channels - first));
  return Place<FULL>{first, static_cast<uint32_t>(lane * V), count};
}

template <typename T>
__device__ __forceinline__ uint32_t bits_at(const T* row, uint32_t i) {
  const T v = *at_bytes(row, i * static_cast<uint32_t>(sizeof(T)));
  if constexpr (sizeof(T) == 4)
    return __builtin_bit_cast(uint32_t, v);
  else
    return __builtin_bit_cast(uint16_t, v);
}

// A row's values of a lane; `row` is the same for the wave.
template <typename T, int V, bool FULL>
__device__ __forceinline__ Raw<T, V> load(const T* row, const Place<FULL>& c) {
  struct __attribute__((packed)) Any {
    Raw<T, V> r;
  };
  const T* p = row + c.first;
  Raw<T, V> r;
  if constexpr (FULL) {
    r = reinterpret_cast<const Any*>(at_bytes(p, c.off * static_cast<uint32_t>(sizeof(T))))->r;
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) r.w[e] = bits_at(p, c.at(e));
  } else {
    r.w[0] = bits_at(p, c.at(0)) | bits_at(p, c.at(1)) << 16;
  }
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V>& r, float (&f)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = __uint_as_float(r.w[e]);
  } else {
    unpack2<T>(r.w[0], f[0], f[1]);
  }
}

template <typename T, int V, bool FULL>
__device__ __forceinline__ void store(T* row, const Place<FULL>& c, const float (&f)[V]) {
  if constexpr (FULL) {
    Raw<T, V> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < V; ++e) r.w[e] = __float_as_uint(f[e]);
    } else {
      r.w[0] = pack2<T>(f[0], f[V - 1]);
    }
    // whole rows of the strip that no later workgroup reads: forward 86 -> 80 us, backward 140 -> 132
    // (4 x 4096 x 2560 bf16)
    store_words_nt(at_bytes(row + c.first, c.off * static_cast<uint32_t>(sizeof(T))), r.w);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c.has(e)) *at_bytes(row + c.first, (c.off + e) * static_cast<uint32_t>(sizeof(T))) = from_f32<T>(f[e]);
  }
}

// The NT rows of a wave's run, from row t0 of a sequence on; past its end (unless WHOLE) the last again.
template <typename T, int NT, int V, bool WHOLE, bool FULL>
__device__ __forceinline__ void load_run(const void* p, int64_t sequence, int64_t stride, int64_t t0, int64_t length,
                                         const Place<FULL>& c, Raw<T, V> (&r)[NT]) {
  const T* row = static_cast<const T*>(p) + sequence + (WHOLE ? t0 : min(t0, length - 1)) * stride;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    r[t] = load<T, V>(row, c);
    if (WHOLE || t0 + t + 1 < length) row += stride;
  }
}

// Bit t set if step t of the wave's run is a reset.
template <bool RESET, int T>
__device__ __forceinline__ uint32_t reset_bits(const mko_recur_params& p, int64_t b, int64_t t0, int lane) {
  if (!RESET) return 0;
  const int64_t t = t0 + lane;
  const bool set = lane < T && t < p.length && p.reset[b * p.length + t];
  return static_cast<uint32_t>(__ballot(set));
}

// ---------------------------------------------------------------- the chunks' order
//
// The chunks of a strip are joined in one pass over the data.  A workgroup publishes its chunk's map
// as soon as it has it, looks for the nearest chunk before it whose end state is published, carries
// that state through the maps between, and publishes its own end state.  Whichever end it finds, the
// same products and sums are formed in the same order, so the bits do not depend on the timing.
// Each published word says by itself whether it is there (cells start as all ones, which no value
// is stored as), so relaxed atomics of the whole device are enough.  A workgroup takes its chunk from
// a counter, chunk by chunk of all chains: whatever it waits for belongs to a workgroup that runs
// already and that waits in turn only for earlier ones, so every wait ends.

constexpr uint32_t kAbsent = 0xffffffffu;
constexpr int kWindow = 4;            // chunks looked at in one round trip
constexpr int kMostRounds = 1 << 22;  // seconds; a wait cut short shows as NaN

// v with a NaN in the one form that is not kAbsent.
__device__ __forceinline__ uint32_t publishable(float v) {
  return v == v ? __float_as_uint(v) : 0x7fc00000u;
}

struct Chain {
  uint64_t* maps;   // (batch, chunks, channels): P in the high word, H in the low
  uint32_t* ends;   // (batch, chunks, channels): the value that leaves the chunk
  uint32_t* tickets;  // up to kCounters counters, kCounterGap words apart
};
constexpr int kCounters = kXcds, kCounterGap = 32;

__device__ __forceinline__ void publish_map(uint64_t* cell, float P, float H) {
  __hip_atomic_store(cell, static_cast<uint64_t>(publishable(P)) << 32 | __float_as_uint(H), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish_end(uint32_t* cell, float h) {
  __hip_atomic_store(cell, publishable(h), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The value that enters a chunk, for a whole wave; the lane's channel is `off` channels into the
// strip, whose first is `first`.  `before` chunks of the chain lie before it, the nearest in row
// `cell` of the cells, the others `step` rows apart; `start` enters the first of them.
template <bool RESET>
__device__ __forceinline__ float enter(const Chain& ch, int64_t channels, int64_t first, uint32_t off, int64_t cell,
                                       int step, int before, float start) {
  if (before == 0) return start;
  for (int round = 0; round < kMostRounds; ++round) {
    uint32_t end[kWindow];
    uint64_t map[kWindow];
#pragma unroll
    for (int k = 0; k < kWindow; ++k) {
      const int64_t row = (cell + (k < before ? k : 0) * step) * channels + first;
      end[k] = __hip_atomic_load(at_bytes(ch.ends + row, off * 4), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      map[k] = __hip_atomic_load(at_bytes(ch.maps + row, off * 8), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // the nearest end that is there, with every map nearer than it
    int found = -1;
    bool maps = true;
    float h = 0.0f;
#pragma unroll
    for (int k = 0; k < kWindow; ++k) {
      if (found < 0 && maps && k < before) {
        if (__all(end[k] != kAbsent)) {
          found = k;
          h = __uint_as_float(end[k]);
        }
        maps = __all(static_cast<uint32_t>(map[k] >> 32) != kAbsent);
      }
    }
    if (found >= 0) {
#pragma unroll
      for (int k = kWindow - 2; k >= 0; --k)
        if (k < found)
          h = apply<RESET>(__uint_as_float(static_cast<uint32_t>(map[k] >> 32)),
                           __uint_as_float(static_cast<uint32_t>(map[k])), h);
      return h;
    }
    __builtin_amdgcn_s_sleep(1);
  }
  return __uint_as_float(0x7fc00000u);
}

// A chunk's part in the chain, for a wave whose lanes have channel i of the strip each: joins its
// waves' maps, in the order of the chain, finds what enters the chunk and leaves it in `entered`.
// Returns what leaves the chunk.
template <int NW, int V, bool RESET, bool BACK>
__device__ __forceinline__ float join(const Chain& ch, const float (&P)[NW][64 * V], const float (&R)[NW][64 * V],
                                      float* entered, int64_t channels, int64_t first, uint32_t count, int i,
                                      int64_t cell, int before, int after, float start) {
  constexpr int kFirst = BACK ? NW - 1 : 0, kStep = BACK ? -1 : 1;
  float Pc = P[kFirst][i], Rc = R[kFirst][i];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    const float Pw = P[kFirst + w * kStep][i];
    Rc = apply<RESET>(Pw, R[kFirst + w * kStep][i], Rc);
    Pc = both<RESET>(Pc, Pw);
  }
  const uint32_t off = static_cast<uint32_t>(i);
  if (before > 0 && after > 0 && off < count)
    publish_map(at_bytes(ch.maps + cell * channels + first, off * 8), Pc, Rc);
  const float in = enter<RESET>(ch, channels, first, min(off, count - 1), cell - kStep, -kStep, before, start);
  entered[i] = in;
  return apply<RESET>(Pc, Rc, in);
}

// Marks two runs of cells absent and starts the counters.
__global__ void __launch_bounds__(kThreads) clear(uint4* a, int64_t na, uint4* b, int64_t nb, uint32_t* tickets) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const uint4 none = make_uint4(kAbsent, kAbsent, kAbsent, kAbsent);
  if (i < na) a[i] = none;
  if (i < nb) b[i] = none;
  if (i < kCounters) tickets[i * kCounterGap] = 0;
}

struct Geo {
  int chunks, strips, chains;  // chains = batch * strips
  int counters;
};

// This workgroup's chunk, counted from the end that is first, and its chain, the same for the wave;
// false if there is none for it.  With several counters the chains are dealt to them: workgroup w
// draws from counter w mod `counters`, one for each XCD, so that a chain stays with an XCD.
__device__ __forceinline__ bool take(const Geo& g, uint32_t* tickets, uint32_t* slot, int& chunk, int& chain) {
  const int counter = static_cast<int>(blockIdx.x) % g.counters;
  const int mine = (g.chains + g.counters - 1 - counter) / g.counters;  // chains of this counter
  int turn = static_cast<int>(blockIdx.x) / g.counters;
  if (turn >= mine * g.chunks) return false;
  if (g.chunks > 1) {
    if (threadIdx.x == 0) *slot = atomicAdd(tickets + counter * kCounterGap, 1u);
    __syncthreads();
    turn = uniform(static_cast<int>(*slot));
  }
  chunk = turn / mine;
  chain = (turn - chunk * mine) * g.counters + counter;
  return true;
}

// ---------------------------------------------------------------- forward

template <typename T, int NW, int NT, int V, bool RESET, bool FULL>
__global__ void __launch_bounds__(NW * 64) forward(mko_recur_params p, Geo g, Chain ch) {
  static_assert(NW * NT == kChunk, "a workgroup takes a chunk");
  __shared__ float runs[2][NW][64 * V], entered[64 * V];
  __shared__ uint32_t slot;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int chunk, chain;
  if (!take(g, ch.tickets, &slot, chunk, chain)) return;
  const int64_t b = chain / g.strips, strip = chain % g.strips;
  const Place<FULL> c = place<V, FULL>(strip, p.channels, lane);
  const int64_t t0 = static_cast<int64_t>(chunk) * kChunk + wave * NT;
  const int steps = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(NT), p.length - t0)));

  // the run from a zero state: h = H[t], and P[t] of the state before it
  float H[NT][V], P[NT][V];
  auto form = [&](auto whole) {  // whole: no step of the run is past the end
    constexpr bool WHOLE = decltype(whole)::value;
    Raw<T, V> xr[NT], ir[NT], rr[NT];
    load_run<T, NT, V, WHOLE>(p.x, b * p.x_stride_b, p.x_stride_t, t0, p.length, c, xr);
    load_run<T, NT, V, WHOLE>(p.input_gate, b * p.ig_stride_b, p.ig_stride_t, t0, p.length, c, ir);
    load_run<T, NT, V, WHOLE>(p.decay_gate, b * p.rg_stride_b, p.rg_stride_t, t0, p.length, c, rr);
    const uint32_t cuts = reset_bits<RESET, NT>(p, b, t0, lane);
    float rate[V];
#pragma unroll
    for (int e = 0; e < V; ++e) rate[e] = binary_rate(p.scale, p.decay[c.first + c.at(e)]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[V], ig[V], rg[V];
      unpack<T, V>(xr[t], x);
      unpack<T, V>(ir[t], ig);
      unpack<T, V>(rr[t], rg);
      const bool cut = RESET && (cuts >> t & 1);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const Step s = gates(ig[e], rg[e], rate[e], cut);
        const float u = s.m * s.si * x[e];
        const float before = t ? P[t ? t - 1 : 0][e] : 1.0f;
        const float h = t ? H[t ? t - 1 : 0][e] : 0.0f;
        H[t][e] = (t == 0 || cut ? 0.0f : s.a * h) + u;
        P[t][e] = cut ? __uint_as_float(kDropped) : s.a * before;
        if (!WHOLE && t >= steps) {  // past the end the state stays
          H[t][e] = h;
          P[t][e] = before;
        }
      }
    }
  };
  if (steps == NT)
    form(std::true_type{});
  else
    form(std::false_type{});
#pragma unroll
  for (int e = 0; e < V; ++e) {
    runs[0][wave][lane * V + e] = P[NT - 1][e];
    runs[1][wave][lane * V + e] = H[NT - 1][e];
  }
  __syncthreads();

  if (wave < V) {
    const int i = wave * 64 + lane;
    const int64_t cell = b * g.chunks + chunk;
    const uint32_t off = static_cast<uint32_t>(i);
    const float start = p.initial ? p.initial[b * p.channels + c.first + min(off, c.count - 1)] : 0.0f;
    const float h = join<NW, V, RESET, false>(ch, runs[0], runs[1], entered, p.channels, c.first, c.count, i, cell, chunk,
                                              g.chunks - 1 - chunk, start);
    if (off < c.count) {
      publish_end(at_bytes(ch.ends + cell * p.channels + c.first, off * 4), h);
      if (p.final_state && chunk + 1 == g.chunks) p.final_state[b * p.channels + c.first + i] = h;
    }
  }
  __syncthreads();

  float in[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    in[e] = entered[lane * V + e];
    for (int w = 0; w < wave; ++w) in[e] = apply<RESET>(runs[0][w][lane * V + e], runs[1][w][lane * V + e], in[e]);
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    if (t >= steps) break;
    float y[V];
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = apply<RESET>(P[t][e], H[t][e], in[e]);
    store<T, V>(static_cast<T*>(p.y) + (b * p.length + t0 + t) * p.channels, c, y);
  }
}

// ---------------------------------------------------------------- backward
//
// The states are formed again from the one that enters the chunk, which the forward saved.  What
// flows from a step to the one before it, a[t] g[t], has the forward's maps in the other direction,
// and its chunks are joined from the last to the first.

template <typename T, int NW, int NT, int V, bool RESET, bool FULL>
__global__ void __launch_bounds__(NW * 64, 4) backward(mko_recur_params p, Geo g, Chain ch, float* part) {
  static_assert(NW * NT == kChunk, "a workgroup takes a chunk");
  __shared__ float runs[3][NW][64 * V], entered[64 * V];
  __shared__ uint32_t slot;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int behind, chain;
  if (!take(g, ch.tickets, &slot, behind, chain)) return;
  const int chunk = g.chunks - 1 - behind;
  const int64_t b = chain / g.strips, strip = chain % g.strips;
  const Place<FULL> c = place<V, FULL>(strip, p.channels, lane);
  const int64_t t0 = static_cast<int64_t>(chunk) * kChunk + wave * NT;
  const int steps = static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(NT), p.length - t0)));

  Raw<T, V> xr[NT], gr[NT];
  float rate[V], first[V];
  float si[NT][V], sr[NT][V], a[NT][V], m[NT][V];
  float P[V], H[V], G[V];
  auto form = [&](auto whole) {  // whole: no step of the run is past the end
    constexpr bool WHOLE = decltype(whole)::value;
    Raw<T, V> ir[NT], rr[NT];
    load_run<T, NT, V, WHOLE>(p.decay_gate, b * p.rg_stride_b, p.rg_stride_t, t0, p.length, c, rr);
    load_run<T, NT, V, WHOLE>(p.input_gate, b * p.ig_stride_b, p.ig_stride_t, t0, p.length, c, ir);
    load_run<T, NT, V, WHOLE>(p.x, b * p.x_stride_b, p.x_stride_t, t0, p.length, c, xr);
    load_run<T, NT, V, WHOLE>(p.dy, b * p.length * p.channels, p.channels, t0, p.length, c, gr);
    const uint32_t cuts = reset_bits<RESET, NT>(p, b, t0, lane);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      rate[e] = binary_rate(p.scale, p.decay[c.first + c.at(e)]);
      first[e] = chunk ? p.states[(b * g.chunks + chunk - 1) * p.channels + c.first + c.at(e)]
                       : (p.initial ? p.initial[b * p.channels + c.first + c.at(e)] : 0.0f);
      P[e] = 1.0f;
      H[e] = G[e] = 0.0f;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float x[V], ig[V], rg[V];
      unpack<T, V>(xr[t], x);
      unpack<T, V>(ir[t], ig);
      unpack<T, V>(rr[t], rg);
      const bool cut = RESET && (cuts >> t & 1);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const Step s = gates(ig[e], rg[e], rate[e], cut);
        si[t][e] = s.si;
        sr[t][e] = s.sr;
        a[t][e] = cut ? __uint_as_float(kDropped) : s.a;
        m[t][e] = s.m;
        if (WHOLE || t < steps) {
          H[e] = (cut ? 0.0f : s.a * H[e]) + s.m * s.si * x[e];
          P[e] = cut ? __uint_as_float(kDropped) : s.a * P[e];
        }
      }
    }
#pragma unroll
    for (int t = NT - 1; t >= 0; --t) {
      if (!WHOLE && t >= steps) continue;
      float dy[V];
      unpack<T, V>(gr[t], dy);
#pragma unroll
      for (int e = 0; e < V; ++e) G[e] = apply<RESET>(a[t][e], 0.0f, G[e] + dy[e]);
    }
  };
  if (steps == NT)
    form(std::true_type{});
  else
    form(std::false_type{});
#pragma unroll
  for (int e = 0; e < V; ++e) {
    runs[0][wave][lane * V + e] = P[e];
    runs[1][wave][lane * V + e] = H[e];
    runs[2][wave][lane * V + e] = G[e];
  }
  __syncthreads();

  if (wave < V) {
    const int i = wave * 64 + lane;
    const int64_t cell = b * g.chunks + chunk;
    const uint32_t off = static_cast<uint32_t>(i);
    const float start = p.dfinal ? p.dfinal[b * p.channels + c.first + min(off, c.count - 1)] : 0.0f;
    const float out = join<NW, V, RESET, true>(ch, runs[0], runs[2], entered, p.channels, c.first, c.count, i, cell,
                                               behind, chunk, start);
    if (off < c.count) {
      if (chunk > 0)
        publish_end(at_bytes(ch.ends + cell * p.channels + c.first, off * 4), out);
      else if (p.dinitial)
        p.dinitial[b * p.channels + c.first + i] = out;
    }
  }
  __syncthreads();

  // From here on these are new to the compiler: carried along, the terms it formed of them above
  // would take more registers than it takes to form them again.
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (uint32_t& w : xr[t].w) w = opaque(w);
#pragma unroll
    for (uint32_t& w : gr[t].w) w = opaque(w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      m[t][e] = fp32_value(m[t][e]);
      si[t][e] = fp32_value(si[t][e]);
      sr[t][e] = fp32_value(sr[t][e]);
    }
  }
  float h[NT][V], flow[V], sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float f = first[e];
    for (int w = 0; w < wave; ++w) f = apply<RESET>(runs[0][w][lane * V + e], runs[1][w][lane * V + e], f);
    h[0][e] = f;
    flow[e] = entered[lane * V + e];
    for (int w = NW - 1; w > wave; --w)
      flow[e] = apply<RESET>(runs[0][w][lane * V + e], runs[2][w][lane * V + e], flow[e]);
    sum[e] = 0.0f;
  }
#pragma unroll
  for (int t = 0; t + 1 < NT; ++t) {
    float x[V];
    unpack<T, V>(xr[t], x);
#pragma unroll
    for (int e = 0; e < V; ++e) h[t + 1][e] = apply<RESET>(a[t][e], m[t][e] * si[t][e] * x[e], h[t][e]);
  }
  auto spread = [&](auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int64_t last = (b * p.length + t0 + (WHOLE ? NT : steps) - 1) * p.channels;
    T* to_x = static_cast<T*>(p.dx) + last;
    T* to_ig = static_cast<T*>(p.dinput_gate) + last;
    T* to_rg = static_cast<T*>(p.ddecay_gate) + last;
#pragma unroll
    for (int t = NT - 1; t >= 0; --t) {
      if (!WHOLE && t >= steps) continue;
      float x[V], dy[V], dx[V], dig[V], drg[V];
      unpack<T, V>(xr[t], x);
      unpack<T, V>(gr[t], dy);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float gt = dy[e] + flow[e];
        const float gm = gt * m[t][e];
        const float u = si[t][e] * x[e];
        const float rm = fast_rcp(fmaxf(m[t][e], 1e-19f));  // finite where v is 0
        const float back = a[t][e] * gt;
        float dv = back * (u * a[t][e] * rm - h[t][e]);
        if (drops<RESET>(a[t][e])) dv = 0.0f;
        const float gu = gm * u, term = dv * sr[t][e];
        dx[e] = gm * si[t][e];
        dig[e] = gu - gu * si[t][e];
        drg[e] = rate[e] * (term - term * sr[t][e]);
        sum[e] += term;
        flow[e] = drops<RESET>(a[t][e]) ? 0.0f : back;
      }
      store<T, V>(to_x, c, dx);
      store<T, V>(to_ig, c, dig);
      store<T, V>(to_rg, c, drg);
      to_x -= p.channels;
      to_ig -= p.channels;
      to_rg -= p.channels;
    }
  };
#pragma unroll
  for (int e = 0; e < V; ++e) rate[e] *= kLn2;  // back from the binary exponential's units
  if (steps == NT)
    spread(std::true_type{});
  else
    spread(std::false_type{});
  if (!p.ddecay) return;
  __syncthreads();  // runs is read no more
#pragma unroll
  for (int e = 0; e < V; ++e) runs[0][wave][lane * V + e] = sum[e];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s = 0.0f;
      for (int w = 0; w < NW; ++w) s += runs[0][w][lane * V + e];
      if (c.has(e)) part[(b * g.chunks + chunk) * p.channels + c.first + c.off + e] = s;
    }
  }
}

// ddecay from the chunks' sums (rows of `part`).
__global__ void __launch_bounds__(kColumnThreads) finish(mko_recur_params p, const float* part, int64_t rows) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const float s = column_sum(part, rows, p.channels, d);
  if (threadIdx.x < 32 && d < p.channels) p.ddecay[d] = s * p.scale * softplus_grad(p.decay[d]);
}

template <typename T, typename S>
__global__ void __launch_bounds__(kThreads) update(mko_recur_update_params p) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t b = blockIdx.y;
  if (d >= p.channels) return;
  const float rate = binary_rate(p.scale, p.decay[d]);
  const float x = to_f32(static_cast<const T*>(p.x)[b * p.x_stride + d]);
  const float ig = to_f32(static_cast<const T*>(p.input_gate)[b * p.ig_stride + d]);
  const float rg = to_f32(static_cast<const T*>(p.decay_gate)[b * p.rg_stride + d]);
  const Step s = gates(ig, rg, rate, false);
  const float h = s.a * to_f32(static_cast<const S*>(p.state)[b * p.channels + d]) + s.m * s.si * x;
  static_cast<S*>(p.new_state)[b * p.channels + d] = from_f32<S>(h);
  static_cast<T*>(p.y)[b * p.channels + d] = from_f32<T>(h);
}

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
  const bool sides = p->batch <= kMostBatch && p->channels <= kMostSide && p->length <= kMostSide;
  const int64_t chains = sides ? cdiv(p->batch * cdiv(p->channels, 64 * kV), kCounters) * kCounters : 0;
  // chains * chunks may pass 64 bits
  if (!sides || (p->length > 0 && chains > kMostWorkgroups / cdiv(p->length, kChunk))) {
    mko_set_error("%s: batch is at most 65535, and batch * channels / 128, up to the next multiple of 8, times "
                  "length / 64 at most 2^22", what);
    return MKO_EUNSUPPORTED;
  }
  return MKO_OK;
}

bool empty(const mko_recur_params* p) { return p->batch == 0 || p->length == 0 || p->channels == 0; }

Geo geo(const mko_recur_params* p) {
  Geo g;  // check() keeps the products below 2^23
  g.chunks = static_cast<int>(cdiv(p->length, kChunk));
  g.strips = static_cast<int>(cdiv(p->channels, 64 * kV));
  g.chains = static_cast<int>(p->batch) * g.strips;
  // Eight counters where they share the chains within an eighth: 36 chains of 16 chunks 26 -> 21 us.
  // 20 chains of 512 chunks, three on some XCDs and two on others, 173 us with one counter and 206
  // with eight.
  g.counters = cdiv(g.chains, kCounters) * kCounters * 8 <= 9 * g.chains ? kCounters : 1;
  return g;
}

int64_t cells(const mko_recur_params* p) { return p->batch * cdiv(p->length, kChunk) * p->channels; }
constexpr int64_t kTicketBytes = kCounters * kCounterGap * 4;
int64_t aligned(int64_t n) { return cdiv(n, 16) * 16; }

int64_t maps_bytes(const mko_recur_params* p) { return aligned(cells(p) * 8); }
int64_t ends_bytes(const mko_recur_params* p) { return aligned(cells(p) * 4); }

// Clears what the chunks publish.  A chain of one chunk publishes nothing.
void clear_cells(const mko_recur_params* p, const Chain& ch, hipStream_t s) {
  const int64_t maps = maps_bytes(p) / 16, ends = ends_bytes(p) / 16;
  MKO_TIMED("recur_clear", s,
            clear<<<static_cast<unsigned>(cdiv(maps, kThreads)), kThreads, 0, s>>>(
                reinterpret_cast<uint4*>(ch.maps), maps, reinterpret_cast<uint4*>(ch.ends), ends, ch.tickets));
}

// The chain's cells are cleared 16 bytes at a time, and a map is one 64-bit atomic word.
bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

unsigned workgroups(const Geo& g) {
  return static_cast<unsigned>(cdiv(g.chains, g.counters) * g.counters * g.chunks);
}

constexpr int kFwdSteps = 8, kBwdSteps = 8;  // steps of a wave

template <typename T, bool RESET, bool FULL>
void launch_fwd(const mko_recur_params& p, const Geo& g, const Chain& ch, hipStream_t s) {
  const unsigned grid = workgroups(g);
  constexpr int kNw = kChunk / kFwdSteps;
  MKO_TIMED("recur_fwd", s, forward<T, kNw, kFwdSteps, kV, RESET, FULL><<<grid, kNw * 64, 0, s>>>(p, g, ch));
}

template <typename T, bool RESET, bool FULL>
void launch_bwd(const mko_recur_params& p, const Geo& g, const Chain& ch, float* part, hipStream_t s) {
  const unsigned grid = workgroups(g);
  constexpr int kNw = kChunk / kBwdSteps;
  MKO_TIMED("recur_bwd", s, backward<T, kNw, kBwdSteps, kV, RESET, FULL><<<grid, kNw * 64, 0, s>>>(p, g, ch, part));
}

// The kernels of a dtype, with or without resets, for whole strips (with outputs at addresses that
// their vector stores take) or others.
template <typename T>
void launch(const mko_recur_params& p, const Geo& g, const Chain& ch, float* part, bool back, hipStream_t s) {
  const uintptr_t outputs = back ? reinterpret_cast<uintptr_t>(p.dx) | reinterpret_cast<uintptr_t>(p.dinput_gate) |
                                       reinterpret_cast<uintptr_t>(p.ddecay_gate)
                                 : reinterpret_cast<uintptr_t>(p.y);
  const bool full = p.channels % (64 * kV) == 0 && outputs % (kV * sizeof(T)) == 0;
  if (back) {
    if (p.reset)
      full ? launch_bwd<T, true, true>(p, g, ch, part, s) : launch_bwd<T, true, false>(p, g, ch, part, s);
    else
      full ? launch_bwd<T, false, true>(p, g, ch, part, s) : launch_bwd<T, false, false>(p, g, ch, part, s);
  } else {
    if (p.reset)
      full ? launch_fwd<T, true, true>(p, g, ch, s) : launch_fwd<T, true, false>(p, g, ch, s);
    else
      full ? launch_fwd<T, false, true>(p, g, ch, s) : launch_fwd<T, false, false>(p, g, ch, s);
  }
}

}  // namespace
}  // namespace recur
}  // namespace mko

using namespace mko;

extern "C" size_t mko_sizeof_recur_params(void) { return sizeof(mko_recur_params); }
extern "C" size_t mko_sizeof_recur_update_params(void) { return sizeof(mko_recur_update_params); }

extern "C" size_t mko_recur_states_size(const mko_recur_params* p) {
  if (recur::check(p, "recur_states_size") != MKO_OK || recur::empty(p)) return 0;
  return static_cast<size_t>(recur::ends_bytes(p));
}

extern "C" size_t mko_recur_fwd_workspace_size(const mko_recur_params* p) {
  if (recur::check(p, "recur_fwd") != MKO_OK || recur::empty(p) || p->length <= recur::kChunk) return 0;
  return static_cast<size_t>(recur::maps_bytes(p) + recur::kTicketBytes);
}

extern "C" int mko_recur_fwd(const mko_recur_params* p, void* stream) {
  int st = recur::check(p, "recur_fwd");
  if (st != MKO_OK) return st;
  if (recur::empty(p)) return MKO_OK;
  if (!p->x || !p->input_gate || !p->decay_gate || !p->decay || !p->y || !p->states) {
    mko_set_error("recur_fwd: x, both gates, decay, y and states are required");
    return MKO_EINVAL;
  }
  const size_t need = mko_recur_fwd_workspace_size(p);
  if (need && (!p->workspace || p->workspace_bytes < need)) {
    mko_set_error("recur_fwd: workspace of %zu bytes needed, %zu given", need, p->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  if (need && (recur::misaligned(p->workspace) || recur::misaligned(p->states))) {
    mko_set_error("recur_fwd: workspace and states start at multiples of 16 bytes");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const recur::Geo g = recur::geo(p);
  recur::Chain ch{};
  ch.ends = reinterpret_cast<uint32_t*>(p->states);
  if (g.chunks > 1) {
    ch.maps = static_cast<uint64_t*>(p->workspace);
    ch.tickets = reinterpret_cast<uint32_t*>(static_cast<char*>(p->workspace) + recur::maps_bytes(p));
    recur::clear_cells(p, ch, s);
  }
  if (p->dtype == MKO_F32)
    recur::launch<float>(*p, g, ch, nullptr, false, s);
  else if (p->dtype == MKO_BF16)
    recur::launch<bf16>(*p, g, ch, nullptr, false, s);
  else
    recur::launch<_Float16>(*p, g, ch, nullptr, false, s);
  return mko_check_launch("recur_fwd");
}

extern "C" size_t mko_recur_bwd_workspace_size(const mko_recur_params* p) {
  if (recur::check(p, "recur_bwd") != MKO_OK || recur::empty(p)) return 0;
  const int64_t part = p->ddecay ? recur::ends_bytes(p) : 0;
  const int64_t chain = p->length > recur::kChunk ? recur::maps_bytes(p) + recur::ends_bytes(p) + recur::kTicketBytes : 0;
  return static_cast<size_t>(part + chain);
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
  if (need && (!p->workspace || p->workspace_bytes < need)) {
    mko_set_error("recur_bwd: workspace of %zu bytes needed, %zu given", need, p->workspace_bytes);
    return MKO_EWORKSPACE;
  }
  if (need && recur::misaligned(p->workspace)) {
    mko_set_error("recur_bwd: workspace starts at a multiple of 16 bytes");
    return MKO_EINVAL;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const recur::Geo g = recur::geo(p);
  char* ws = static_cast<char*>(p->workspace);
  float* part = reinterpret_cast<float*>(ws);
  if (p->ddecay) ws += recur::ends_bytes(p);
  recur::Chain ch{};
  if (g.chunks > 1) {
    ch.maps = reinterpret_cast<uint64_t*>(ws);
    ch.ends = reinterpret_cast<uint32_t*>(ws + recur::maps_bytes(p));
    ch.tickets = reinterpret_cast<uint32_t*>(ws + recur::maps_bytes(p) + recur::ends_bytes(p));
    recur::clear_cells(p, ch, s);
  }
  if (p->dtype == MKO_F32)
    recur::launch<float>(*p, g, ch, part, true, s);
  else if (p->dtype == MKO_BF16)
    recur::launch<bf16>(*p, g, ch, part, true, s);
  else
    recur::launch<_Float16>(*p, g, ch, part, true, s);
  if (p->ddecay)
    MKO_TIMED("recur_bwd_finish", s,
              recur::finish<<<static_cast<unsigned>(cdiv(p->channels, 32)), kColumnThreads, 0, s>>>(
                  *p, part, p->batch * g.chunks));
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
  if (!half_or_float(p->dtype) || !half_or_float(p->state_dtype)) {
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
