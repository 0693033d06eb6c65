// causal_conv.cu — the short causal convolution of a state space block: every
// channel of a (channels, tokens) matrix filtered along its tokens with W taps,
//     pre[d, t] = bias[d] + sum_k w[d, k] x[d, t - W + k]   (k = 1..W),
//     y = silu(pre) or pre,
// where x before a sequence's first token is its state (or zero).
//
// Bound by memory: 2 reads or writes of the matrix forward, 3 backward, about
// 4W operations per element.  So a thread owns V neighbouring channels, keeps
// their last W - 1 inputs in registers and walks TT tokens, with the next
// tokens' loads in flight while it computes.  The W - 1 tokens before a tile are
// read again (they hit L2), which is all that is read twice.
//
// bf16, 4 taps, silu, measured on B200: 16384 tokens of 4096 channels forward 55
// us (4.9 TB/s, 0.75 of a copy; 59 us with the state pool of 7 ragged prompts),
// 8192 x 4096 forward 29 us (4.6 TB/s), backward 57 us (3.5 TB/s: 128
// registers leave four warps to a scheduler, whose dependent products and waits
// on shared memory leave half of the issue slots empty) and 4.2 us for conv_fold;
// in Float32 50 and 93 us (conv_bwd with 4 taps spills 116 bytes there); one token
// of 192 entries of 4099 channels (f32, 3 taps) 5.9 us.
#include <type_traits>

#include "tokens.cuh"

namespace {

using namespace mk::tok;

constexpr int kLanes = 32;  // channel vectors of a block
constexpr int kRows = 4;    // token tiles of a block

template <typename T>
struct Conv {
  Seqs q;
  int64_t D;
  const T *x, *dy, *dlast, *init;
  T *y, *dx, *dinit, *last;
  int64_t ldx, ldy, lddy, lddx;
  const float *w, *bias;
  float* parts;              // backward: [part][W + 1][D]
  const int32_t* slots;
  int64_t nslots;
  int64_t tiles;
  int tt;                    // tokens per tile
  int silu;
  unsigned* err;
};

// A thread's channels: four neighbours as one vector, or, where rows are not
// aligned for that, two that are 32 apart (a warp then reads 32 neighbours at a
// time).  8192 x 4095 bf16 forward and backward with one channel per thread
// instead of two: 58 + 140 us, with two 46 + 81 (Float32 73 + 142, 58 + 97).
template <int V> constexpr int kStep = V == 2 ? kLanes : 1;
template <int V>
__device__ __forceinline__ int64_t first_channel() {
  if constexpr (V == 2) return (int64_t)blockIdx.y * kLanes * V + threadIdx.x;
  else return ((int64_t)blockIdx.y * kLanes + threadIdx.x) * V;
}
// Of them, at p; `left` channels are there from the first on.
template <typename T, int V>
__device__ __forceinline__ void load_channels(float (&f)[V], const T* p, int64_t left) {
  if constexpr (V == 2) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i * kStep<V> < left ? to_f(p[i * kStep<V>]) : 0.0f;
  } else {
    load<T, V>(f, p);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_channels(T* p, const Vec<T, V>& r, int64_t left) {
  if constexpr (V == 2) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * kStep<V> < left) p[i * kStep<V>] = r.v[i];
  } else {
    *reinterpret_cast<Vec<T, V>*>(p) = r;
  }
}

// Column `at` of [state | x] of the sequence that begins at lo: the input, or
// for at < lo the state's row, or zero without a state.
template <typename T, int V, int W>
__device__ __forceinline__ void load_seen(float (&f)[V], const Conv<T>& p, int64_t d, int64_t at, int64_t lo,
                                          int64_t row) {
  if (at >= lo) {
    load_channels<T, V>(f, p.x + at * p.ldx + d, p.D - d);
  } else if (p.init && row >= 0) {
    load_channels<T, V>(f, p.init + (row * (W - 1) + (at - lo + W - 1)) * p.D + d, p.D - d);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = 0.0f;
  }
}

// The state after sequence s: the last W - 1 columns of [state | x].  Rows are
// written in ascending order and read at or above the row written, so `last`
// may be `init` itself.
template <typename T, int V, int W>
__device__ __forceinline__ void write_last(const Conv<T>& p, int64_t d, int64_t s) {
  const int64_t row = slot_of(p.slots, p.nslots, s, p.err);
  if (row < 0) return;
  const Span sp = seq_span(p.q, s);
  for (int j = 0; j < W - 1; ++j) {
    float f[V];
    load_seen<T, V, W>(f, p, d, sp.hi - (W - 1) + j, sp.lo, row);
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_f<T>(f[i]);
    store_channels<T, V>(p.last + (row * (W - 1) + j) * p.D + d, r, p.D - d);
  }
}

template <typename T, int V, int W>
__global__ void __launch_bounds__(kLanes* kRows) conv_last(Conv<T> p) {
  const int64_t d = first_channel<V>();
  const int64_t s = (int64_t)blockIdx.x * kRows + threadIdx.y;
  if (d < p.D && s < p.q.nseq) write_last<T, V, W>(p, d, s);
}

// One block of a launch looks the offsets and slots over.
template <typename T>
__device__ __forceinline__ void check_inputs(const Conv<T>& p, int64_t block, int64_t blocks, int tid, int nt) {
  for (int64_t s = block; s < p.q.nseq; s += blocks) {
    if (tid == 0 && p.q.seqs && seq_span(p.q, s).bad) atomicOr(p.err, mk::ERRBIT_SEQS);
    check_distinct(p.slots, s, tid, nt, p.err);
  }
}

// A thread's V channels of a value, in pairs.
template <int V> constexpr int kPairs = V / 2;

template <int V, typename T>
__device__ __forceinline__ void to_pairs(F2 (&f)[kPairs<V>], const T (&v)[V]) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) f[i] = pack(to_f(v[2 * i]), to_f(v[2 * i + 1]));
}
template <int V, typename T>
__device__ __forceinline__ void put_pairs(T* p, const F2 (&f)[kPairs<V>], int64_t left) {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V / 2; ++i) from_f2(&r.v[2 * i], f[i]);
  store_channels<T, V>(p, r, left);
}
template <bool EXACT>
__device__ __forceinline__ F2 sigmoid_pair(F2 x) {
  float a, b;
  unpack(x, a, b);
  return pack(sigmoid<EXACT>(a), sigmoid<EXACT>(b));
}
// w and bias of a thread's channels
template <typename T, int V, int W>
__device__ __forceinline__ void load_taps(F2 (&w)[W][kPairs<V>], F2 (&bias)[kPairs<V>], const Conv<T>& p, int64_t d) {
  float r[V];
  bool live[V];
#pragma unroll
  for (int i = 0; i < V; ++i) live[i] = d + i * kStep<V> < p.D;
#pragma unroll
  for (int k = 0; k < W; ++k) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = live[i] ? p.w[k * p.D + d + i * kStep<V>] : 0.0f;
    to_pairs<V>(w[k], r);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = p.bias && live[i] ? p.bias[d + i * kStep<V>] : 0.0f;
  to_pairs<V>(bias, r);
}
template <typename T, int V, int W>
__device__ __forceinline__ void load_seen_pairs(F2 (&f)[kPairs<V>], const Conv<T>& p, int64_t d, int64_t at, int64_t lo,
                                                int64_t row) {
  float r[V];
  load_seen<T, V, W>(r, p, d, at, lo, row);
  to_pairs<V>(f, r);
}

// A thread's tokens of one matrix, kBatch at a time: kBatches - 1 batches are in
// flight while one is computed.  Vectors go through a ring in shared memory,
// single elements (which may be too small to copy) through registers.
constexpr int kBatch = 4;

template <typename T, int V, int kBatches>
struct Tokens {
  static constexpr bool kRing = V > 2;
  static constexpr int kFlight = kRing ? kBatches - 1 : 1;  // batches asked for ahead
  static constexpr int kSlots = kRing ? kBatch * kBatches * kLanes * kRows : 1;
  Vec<T, V> now[kBatch], next[kRing ? 1 : kBatch];

  // Asks for the batch at t (tokens below `end`) as batch number n; x: at the first of `left` channels.
  __device__ __forceinline__ void ask(Vec<T, V>* ring, const T* x, int64_t ld, int64_t t, int64_t end, int n,
                                      int64_t left) {
    const int tid = threadIdx.y * kLanes + threadIdx.x;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if constexpr (kRing)
        copy_if<sizeof(Vec<T, V>)>(ring + ((n % kBatches) * kBatch + j) * kLanes * kRows + tid, x + (t + j) * ld,
                                   t + j < end);
      else
#pragma unroll
        for (int i = 0; i < V; ++i)
          load_if(reinterpret_cast<Vec<T, 1>&>(next[j].v[i]),
                  reinterpret_cast<const Vec<T, 1>*>(x + (t + j) * ld + i * kStep<V>),
                  t + j < end && i * kStep<V> < left);
    }
  }
  // Batch n, which has arrived, into `now`.
  __device__ __forceinline__ void take(const Vec<T, V>* ring, int n) {
    const int tid = threadIdx.y * kLanes + threadIdx.x;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if constexpr (kRing) now[j] = ring[((n % kBatches) * kBatch + j) * kLanes * kRows + tid];
      else now[j] = next[j];
    }
  }
};

template <typename T, int V, int W>
__global__ void __launch_bounds__(kLanes* kRows) conv_fwd(Conv<T> p) {
  constexpr bool kExact = sizeof(T) == 4;
  using X = Tokens<T, V, 4>;
  __shared__ Vec<T, V> ring[X::kSlots];
  constexpr int kFlight = X::kFlight;
  const int64_t d = first_channel<V>();
  const int64_t tile = (int64_t)blockIdx.x * kRows + threadIdx.y;
  if (blockIdx.y == 0) check_inputs(p, blockIdx.x, gridDim.x, threadIdx.y * kLanes + threadIdx.x, kLanes * kRows);
  if (tile >= p.tiles) return;
  const int64_t t0 = tile * p.tt, t1 = min(p.q.T, t0 + p.tt);
  const int64_t s0 = seq_at(p.q, t0);
  if (d >= p.D) return;
  constexpr int Q = kPairs<V>;
  F2 w[W][Q], bias[Q];
  load_taps<T, V, W>(w, bias, p, d);
  int64_t t = t0;
  for (int64_t s = s0; s < p.q.nseq && t < t1; ++s) {
    const Span sp = seq_span(p.q, s);
    if (sp.hi <= t) continue;
    const int64_t a = max(t, sp.lo), b = min(t1, sp.hi);
    if (sp.lo >= t1) break;
    if (a >= b) continue;  // an empty one behind columns of none
    X x;
#pragma unroll
    for (int n = 0; n < kFlight; ++n) x.ask(ring, p.x + d, p.ldx, a + n * kBatch, b, n, p.D - d), copy_commit();
    const int64_t row = p.init ? slot_of(p.slots, p.nslots, s, p.err) : -1;
    F2 seen[W - 1 + kBatch][Q];  // the last W - 1 inputs, then a batch
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load_seen_pairs<T, V, W>(seen[k], p, d, a - (W - 1) + k, sp.lo, row);
    int n = 0;
    for (t = a; t < b; t += kBatch, ++n) {
      if (X::kRing) {
        x.ask(ring, p.x + d, p.ldx, t + kFlight * kBatch, b, n + kFlight, p.D - d);
        copy_commit();
        copy_wait<kFlight>();
        x.take(ring, n);
      } else {
        x.take(ring, n);
        x.ask(ring, p.x + d, p.ldx, t + kBatch, b, n + 1, p.D - d);
      }
      T* y = p.y + t * p.ldy + d;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        to_pairs<V>(seen[W - 1 + j], x.now[j].v);
        F2 out[Q];
#pragma unroll
        for (int i = 0; i < Q; ++i) {
          F2 acc = bias[i];
#pragma unroll
          for (int k = 0; k < W; ++k) acc = fma2(w[k][i], seen[j + k][i], acc);
          out[i] = p.silu ? mul2(acc, sigmoid_pair<kExact>(acc)) : acc;
        }
        if (t + j < b) put_pairs<V>(y, out, p.D - d);
        y += p.ldy;
      }
#pragma unroll
      for (int k = 0; k < W - 1; ++k)
#pragma unroll
        for (int i = 0; i < Q; ++i) seen[k][i] = seen[kBatch + k][i];
    }
    copy_wait<0>();
    t = b;
  }
  if (p.last) {  // states of the sequences that begin in this tile (the last tile: or behind it)
    int64_t s = s0;
    while (s > 0 && seq_offset(p.q, s - 1) >= t0) --s;
    for (; s < p.q.nseq; ++s) {
      const int64_t at = seq_offset(p.q, s);
      if (at < t0) continue;
      if (at >= t1 && tile != p.tiles - 1) break;
      write_last<T, V, W>(p, d, s);
    }
  }
}

// Backward.  With dp = dy * act'(pre): dx[t] = sum_k w[k] dp[t + W - k], so a
// tile recomputes pre for its own tokens and the W - 1 behind them, keeps the
// last W of dp in registers and writes dx W - 1 tokens late.  dw and dbias are
// summed over the tile in registers, over the block's tiles in shared memory,
// and over blocks by a second launch in a fixed order (no atomics).
template <typename T, int V, int W>
__global__ void __launch_bounds__(kLanes* kRows, 4) conv_bwd(Conv<T> p) {
  using X = Tokens<T, V, sizeof(T) == 4 ? 2 : 4>;  // two rings of Float32: as many as 48 KB hold
  __shared__ Vec<T, V> ring_x[X::kSlots], ring_dy[X::kSlots];
  __shared__ float sm[kRows][(W + 1) * V][kLanes];
  constexpr int kFlight = X::kFlight;
  const int64_t d = first_channel<V>();
  const int64_t tile = (int64_t)blockIdx.x * kRows + threadIdx.y;
  if (blockIdx.y == 0) check_inputs(p, blockIdx.x, gridDim.x, threadIdx.y * kLanes + threadIdx.x, kLanes * kRows);
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int Q = kPairs<V>;
  F2 dw[W][Q], db[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    db[i] = pack(0.0f);
#pragma unroll
    for (int k = 0; k < W; ++k) dw[k][i] = pack(0.0f);
  }
  const int64_t t0 = tile * p.tt, t1 = min(p.q.T, t0 + p.tt);
  const int64_t s0 = tile < p.tiles ? seq_at(p.q, t0) : 0;
  if (d < p.D && tile < p.tiles) {
    F2 w[W][Q], bias[Q];
    load_taps<T, V, W>(w, bias, p, d);
    int64_t t = t0;
    for (int64_t s = s0; s < p.q.nseq && t < t1; ++s) {
      const Span sp = seq_span(p.q, s);
      if (sp.hi <= t) continue;
      const int64_t a = max(t, sp.lo), b = min(t1, sp.hi);
      if (sp.lo >= t1) break;
      if (a >= b) continue;  // an empty one behind columns of none
      const int64_t stop = b + W - 1, end = min(stop, sp.hi);
      X x, up;
#pragma unroll
      for (int n = 0; n < kFlight; ++n) {
        x.ask(ring_x, p.x + d, p.ldx, a + n * kBatch, end, n, p.D - d);
        up.ask(ring_dy, p.dy + d, p.lddy, a + n * kBatch, end, n, p.D - d);
        copy_commit();
      }
      // the last W - 1 inputs and the last W - 1 of dp, each with a batch behind them
      F2 seen[W - 1 + kBatch][Q], win[W - 1 + kBatch][Q];
#pragma unroll
      for (int k = 0; k < W - 1; ++k) {
        load_seen_pairs<T, V, W>(seen[k], p, d, a - (W - 1) + k, sp.lo, s);
#pragma unroll
        for (int i = 0; i < Q; ++i) win[k][i] = pack(0.0f);
      }
      int n = 0;
      for (int64_t c = a; c < stop; c += kBatch, ++n) {
        if (X::kRing) {
          x.ask(ring_x, p.x + d, p.ldx, c + kFlight * kBatch, end, n + kFlight, p.D - d);
          up.ask(ring_dy, p.dy + d, p.lddy, c + kFlight * kBatch, end, n + kFlight, p.D - d);
          copy_commit();
          copy_wait<kFlight>();
          x.take(ring_x, n), up.take(ring_dy, n);
        } else {
          x.take(ring_x, n), up.take(ring_dy, n);
          x.ask(ring_x, p.x + d, p.ldx, c + kBatch, end, n + 1, p.D - d);
          up.ask(ring_dy, p.dy + d, p.lddy, c + kBatch, end, n + 1, p.D - d);
        }
        // FULL: every token of the batch is the tile's, and so is every output
        auto batch = [&](auto full) {
          constexpr bool FULL = decltype(full)::value;
          T* dx = p.dx + (c - (W - 1)) * p.lddx + d;
#pragma unroll
          for (int j = 0; j < kBatch; ++j, dx += p.lddx) {
            const int64_t at = c + j;
            const bool inside = FULL || at < sp.hi, counts = FULL || at < b;
            F2 dp[Q], out[Q];
            to_pairs<V>(seen[W - 1 + j], x.now[j].v);
            to_pairs<V>(dp, up.now[j].v);
#pragma unroll
            for (int i = 0; i < Q; ++i) {
              if (p.silu) {
                F2 pre = bias[i];
#pragma unroll
                for (int k = 0; k < W; ++k) pre = fma2(w[k][i], seen[j + k][i], pre);
                const F2 sg = sigmoid_pair<kExact>(pre);
                // silu' = s + pre s (1 - s)
                dp[i] = mul2(dp[i], fma2(mul2(pre, sg), fma2(sg, pack(-1.0f), pack(1.0f)), sg));
              }
              if (!inside) dp[i] = pack(0.0f);
              if (counts) {
#pragma unroll
                for (int k = 0; k < W; ++k) dw[k][i] = fma2(dp[i], seen[j + k][i], dw[k][i]);
                db[i] = add2(db[i], dp[i]);
              }
              win[W - 1 + j][i] = dp[i];
              out[i] = mul2(w[0][i], win[W - 1 + j][i]);
#pragma unroll
              for (int k = 0; k < W - 1; ++k) out[i] = fma2(w[W - 1 - k][i], win[j + k][i], out[i]);
            }
            if constexpr (FULL) {
              put_pairs<V>(dx, out, p.D - d);
            } else {
              const int64_t o = at - (W - 1);
              if (at < stop && (o >= a || (a == sp.lo && o >= sp.lo - (W - 1)))) {
                if (p.dlast && o >= sp.hi - (W - 1)) {
                  float r[V];
                  F2 more[Q];
                  load_channels<T, V>(r, p.dlast + (s * (W - 1) + (o - sp.hi + W - 1)) * p.D + d, p.D - d);
                  to_pairs<V>(more, r);
#pragma unroll
                  for (int i = 0; i < Q; ++i) out[i] = add2(out[i], more[i]);
                }
                if (o >= a) put_pairs<V>(dx, out, p.D - d);
                else if (p.dinit) put_pairs<V>(p.dinit + (s * (W - 1) + (o - sp.lo + W - 1)) * p.D + d, out, p.D - d);
              }
            }
          }
        };
        if (c > a && c + kBatch <= b) batch(std::true_type{});
        else batch(std::false_type{});
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
          for (int i = 0; i < Q; ++i) seen[k][i] = seen[kBatch + k][i], win[k][i] = win[kBatch + k][i];
      }
      copy_wait<0>();
      t = b;
    }
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
#pragma unroll
    for (int k = 0; k <= W; ++k) {
      float e, o;
      unpack(k < W ? dw[k < W ? k : 0][i] : db[i], e, o);
      sm[threadIdx.y][k * V + 2 * i][threadIdx.x] = e;
      sm[threadIdx.y][k * V + 2 * i + 1][threadIdx.x] = o;
    }
  }
  __syncthreads();
  if (d >= p.D) return;
  float* part = p.parts + (int64_t)blockIdx.x * (W + 1) * p.D;
  for (int j = threadIdx.y; j < (W + 1) * V; j += kRows) {
    float v = 0.0f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) v += sm[r][j][threadIdx.x];
    if (d + j % V * kStep<V> < p.D) part[(int64_t)(j / V) * p.D + d + j % V * kStep<V>] = v;
  }
}

// dinit of empty sequences: the state passes through, so its gradient does.
template <typename T, int W>
__global__ void __launch_bounds__(128) conv_bwd_empty(Conv<T> p) {
  const Span sp = seq_span(p.q, blockIdx.x);
  if (sp.hi > sp.lo) return;
  const int64_t n = (int64_t)(W - 1) * p.D, at = (int64_t)blockIdx.x * n;
  for (int64_t i = threadIdx.x; i < n; i += 128) p.dinit[at + i] = p.dlast ? p.dlast[at + i] : from_f<T>(0.0f);
}

// dw (W * D values), then dbias: sums over the blocks of the launch before.
__global__ void __launch_bounds__(256) conv_fold(float* dw, float* dbias, const float* parts, int64_t nparts,
                                                 int64_t nw, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float v = 0.0f;
#pragma unroll 8
  for (int64_t k = 0; k < nparts; ++k) v += parts[k * n + i];
  if (i < nw) dw[i] = v;
  else if (dbias) dbias[i - nw] = v;
}

// One token per entry: y from [state | x], and the state moved on by it.
template <typename T>
struct ConvStep {
  int64_t D, B, ldx, ldy, nslots;
  const T *x, *state;
  T *y, *next;
  const float *w, *bias;
  const int32_t* slots;
  int silu;
  int64_t dblocks;
  unsigned* err;
};

template <typename T, int V, int W>
__global__ void __launch_bounds__(128) conv_step(ConvStep<T> p) {
  const int64_t e = blockIdx.x / p.dblocks, block = blockIdx.x % p.dblocks;
  if (block == 0) check_distinct(p.slots, e, threadIdx.x, 128, p.err);
  const int64_t d = (block * 128 + threadIdx.x) * V;
  const int64_t row = slot_of(p.slots, p.nslots, e, p.err);
  if (d >= p.D || row < 0) return;
  float seen[W][V], out[V];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) load<T, V>(seen[k], p.state + (row * (W - 1) + k) * p.D + d);
  load<T, V>(seen[W - 1], p.x + e * p.ldx + d);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float acc = p.bias ? p.bias[d + i] : 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) acc = fmaf(p.w[k * p.D + d + i], seen[k][i], acc);
    out[i] = p.silu ? acc * sigmoid<sizeof(T) == 4>(acc) : acc;
  }
#pragma unroll
  for (int k = 0; k < W - 1; ++k) store<T, V>(p.next + (row * (W - 1) + k) * p.D + d, seen[k + 1]);
  store<T, V>(p.y + e * p.ldy + d, out);
}

// ---- host side ----------------------------------------------------------------

int check(const mk_conv_args* a, const char* who) {
  if (!a) return bad(who, "null arguments");
  if (a->type < MK_T_F32 || a->type > MK_T_BF16) return bad(who, "unknown element type");
  if (a->width < 2 || a->width > 4) return bad(who, "2 to 4 taps, got " + std::to_string(a->width));
  if (a->D < 1 || a->T < 0 || a->nseq < 0 || a->len < 0) return bad(who, "negative size or no channels");
  if (a->D > (1ll << 20) || a->T > INT32_MAX || a->nseq > (1ll << 24))
    return bad(who, "more than 2^20 channels, 2^24 sequences or 2^31 - 1 tokens");
  MK_TRY(check_slots(who, a->slots, a->nslots, a->nseq));
  MK_TRY(check_floats(who, "w", a->w, true, false));
  return check_floats(who, "bias", a->bias, false, false);
}

int check_seqs(const mk_conv_args* a, const char* who) {
  if (a->seqs) return MK_OK;
  return (a->nseq && a->len > a->T) || a->nseq * a->len != a->T ? bad(who, "nseq * len is not T") : MK_OK;
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && na && nb && x < y + nb && y < x + na;
}

// Tokens per tile: long tiles read fewer tokens twice, but the launch wants
// four blocks per SM; short inputs take shorter tiles down to 8 tokens.  8192 x
// 4096 forward and backward with tiles of 8, 16, 32, 64, 128 tokens: 175, 126, 102,
// 92, 97 us; 512 x 2048 with 8, 16, 32, 64: 14.7, 15.7, 21, 30 us.
int tokens_per_tile(const mk::Device* dev, int64_t T, int64_t dblocks, int most) {
  int tt = most;
  while (tt > 8 && mk::cdiv(T, (int64_t)tt * kRows) * dblocks < 4ll * dev->sms) tt /= 2;
  return tt;
}

template <typename T>
Conv<T> params(const mk_conv_args* a, mk::Device* dev) {
  Conv<T> p{};
  p.q = Seqs{a->seqs, a->nseq, a->len, a->T};
  p.D = a->D;
  p.x = static_cast<const T*>(a->x);
  p.y = static_cast<T*>(a->y);
  p.dy = static_cast<const T*>(a->dy);
  p.dx = static_cast<T*>(a->dx);
  p.init = static_cast<const T*>(a->init);
  p.last = static_cast<T*>(a->last);
  p.dinit = static_cast<T*>(a->dinit);
  p.dlast = static_cast<const T*>(a->dlast);
  p.ldx = a->ldx, p.ldy = a->ldy, p.lddy = a->lddy, p.lddx = a->lddx;
  p.w = a->w, p.bias = a->bias;
  p.slots = a->slots, p.nslots = a->nslots;
  p.silu = a->silu;
  p.err = dev->err_word;
  return p;
}

template <typename T, int V, int W>
int run_fwd(const mk_conv_args* a, mk::Device* dev, cudaStream_t s) {
  Conv<T> p = params<T>(a, dev);
  const int64_t dblocks = mk::cdiv(a->D, kLanes * V);
  p.tt = tokens_per_tile(dev, a->T, dblocks, 64);
  p.tiles = a->T ? mk::cdiv(a->T, p.tt) : 1;
  // A tile may still read the state that another tile's sequence is about to
  // replace: pools that share memory are written by a launch of their own.
  const size_t pool = (size_t)(a->slots ? a->nslots : a->nseq) * (W - 1) * a->D * sizeof(T);
  const bool apart = a->last && overlap(a->init, pool, a->last, pool);
  if (apart) p.last = nullptr;
  const dim3 block(kLanes, kRows);
  conv_fwd<T, V, W><<<dim3((unsigned)mk::cdiv(p.tiles, kRows), (unsigned)dblocks), block, 0, s>>>(p);
  if (apart) {
    p.last = static_cast<T*>(a->last);
    conv_last<T, V, W><<<dim3((unsigned)mk::cdiv(a->nseq, kRows), (unsigned)dblocks), block, 0, s>>>(p);
  }
  return mk::check_launch("mk_causal_conv: launch");
}

// Blocks along the tokens of the backward launch (the parts that conv_fold sums).
struct BwdPlan {
  int V, tt;
  int64_t dblocks, tiles, parts;
};

BwdPlan plan_bwd(const mk_conv_args* a, const mk::Device* dev) {
  const size_t es = type_bytes(a->type);
  BwdPlan b;
  const int V = 4;
  const bool vec = a->D % V == 0 && vec_ok(a->x, a->ldx, es, V) && vec_ok(a->dy, a->lddy, es, V) &&
                   vec_ok(a->dx, a->lddx, es, V) && vec_ok(a->init, 0, es, V) && vec_ok(a->dinit, 0, es, V) &&
                   vec_ok(a->dlast, 0, es, V);
  b.V = vec ? V : 2;
  b.dblocks = mk::cdiv(a->D, (int64_t)kLanes * b.V);
  b.tt = tokens_per_tile(dev, a->T, b.dblocks, 64);
  b.tiles = mk::cdiv(a->T, b.tt);
  b.parts = mk::cdiv(b.tiles, kRows);
  return b;
}

template <typename T, int V, int W>
int run_bwd(const mk_conv_args* a, mk::Device* dev, cudaStream_t s, const BwdPlan& b) {
  Conv<T> p = params<T>(a, dev);
  p.slots = nullptr;
  p.tt = b.tt;
  p.tiles = b.tiles;
  p.parts = static_cast<float*>(a->workspace);
  if (b.parts)
    conv_bwd<T, V, W><<<dim3((unsigned)b.parts, (unsigned)b.dblocks), dim3(kLanes, kRows), 0, s>>>(p);
  const int64_t n = (int64_t)(W + 1) * a->D;
  conv_fold<<<(unsigned)mk::cdiv(n, 256), 256, 0, s>>>(a->dw, a->dbias, p.parts, b.parts, (int64_t)W * a->D, n);
  if (a->dinit && a->nseq) conv_bwd_empty<T, W><<<(unsigned)a->nseq, 128, 0, s>>>(p);
  return mk::check_launch("mk_causal_conv_grad: launch");
}

template <typename T, int V, int W>
int run_step(const mk_conv_step_args* a, mk::Device* dev, cudaStream_t s) {
  ConvStep<T> p{};
  p.D = a->D, p.B = a->B, p.ldx = a->ldx, p.ldy = a->ldy, p.nslots = a->nslots;
  p.x = static_cast<const T*>(a->x);
  p.state = static_cast<const T*>(a->state);
  p.y = static_cast<T*>(a->y);
  p.next = static_cast<T*>(a->next);
  p.w = a->w, p.bias = a->bias, p.slots = a->slots, p.silu = a->silu;
  p.dblocks = mk::cdiv(a->D, 128 * V);
  p.err = dev->err_word;
  conv_step<T, V, W><<<(unsigned)(a->B * p.dblocks), 128, 0, s>>>(p);
  return mk::check_launch("mk_causal_conv_step: launch");
}

template <typename T, int V, typename F>
int by_width(int width, F&& f) {
  switch (width) {
    case 2: return f.template operator()<T, V, 2>();
    case 3: return f.template operator()<T, V, 3>();
    default: return f.template operator()<T, V, 4>();
  }
}

// A thread takes four channels, or `few` where alignment does not allow it.  (Eight of a 16-bit type would be one
// 16-byte access, but their taps and history leave fewer threads and fewer bytes in flight.)
template <int FEW, typename F>
int dispatch(int type, int width, bool vec, F&& f) {
  if (type == MK_T_F32) return vec ? by_width<float, 4>(width, f) : by_width<float, FEW>(width, f);
  if (type == MK_T_F16) return vec ? by_width<__half, 4>(width, f) : by_width<__half, FEW>(width, f);
  return vec ? by_width<__nv_bfloat16, 4>(width, f) : by_width<__nv_bfloat16, FEW>(width, f);
}

struct FwdOp {
  const mk_conv_args* a;
  mk::Device* dev;
  cudaStream_t s;
  template <typename T, int V, int W> int operator()() const { return run_fwd<T, V, W>(a, dev, s); }
};
struct BwdOp {
  const mk_conv_args* a;
  mk::Device* dev;
  cudaStream_t s;
  BwdPlan b;
  template <typename T, int V, int W> int operator()() const {
    return run_bwd<T, V, W>(a, dev, s, b);
  }
};
struct StepOp {
  const mk_conv_step_args* a;
  mk::Device* dev;
  cudaStream_t s;
  template <typename T, int V, int W> int operator()() const { return run_step<T, V, W>(a, dev, s); }
};

int forward(const mk_conv_args* a, void* stream) {
  const char* who = "mk_causal_conv";
  MK_TRY(check(a, who));
  MK_TRY(check_seqs(a, who));
  const size_t es = type_bytes(a->type);
  MK_TRY(check_matrix(who, "x", a->x, a->D, a->ldx, a->T, es));
  MK_TRY(check_matrix(who, "y", a->y, a->D, a->ldy, a->T, es));
  MK_TRY(check_matrix(who, "init", a->init, a->D, a->D, a->init ? 1 : 0, es));
  MK_TRY(check_matrix(who, "last", a->last, a->D, a->D, a->last ? 1 : 0, es));
  if (a->y == a->x && a->T) return bad(who, "y must not be x (later tokens read it)");
  if (a->nseq == 0) return MK_OK;
  MK_ENTRY_DEVICE(dev);
  const int V = 4;
  const bool vec = a->D % V == 0 && vec_ok(a->x, a->ldx, es, V) && vec_ok(a->y, a->ldy, es, V) &&
                   vec_ok(a->init, 0, es, V) && vec_ok(a->last, 0, es, V);
  return dispatch<2>(a->type, a->width, vec, FwdOp{a, dev, mk::as_stream(stream)});
}

int grad_workspace(const mk_conv_args* a, size_t* bytes) {
  const char* who = "mk_causal_conv_grad_workspace";
  MK_TRY(check(a, who));
  if (!bytes) return bad(who, "null result");
  MK_ENTRY_DEVICE(dev);
  *bytes = (size_t)plan_bwd(a, dev).parts * (a->width + 1) * a->D * sizeof(float);
  return MK_OK;
}

int gradient(const mk_conv_args* a, void* stream) {
  const char* who = "mk_causal_conv_grad";
  MK_TRY(check(a, who));
  MK_TRY(check_seqs(a, who));
  const size_t es = type_bytes(a->type);
  MK_TRY(check_matrix(who, "x", a->x, a->D, a->ldx, a->T, es));
  MK_TRY(check_matrix(who, "dy", a->dy, a->D, a->lddy, a->T, es));
  MK_TRY(check_matrix(who, "dx", a->dx, a->D, a->lddx, a->T, es));
  MK_TRY(check_matrix(who, "init", a->init, a->D, a->D, a->init ? 1 : 0, es));
  MK_TRY(check_matrix(who, "dinit", a->dinit, a->D, a->D, a->dinit ? 1 : 0, es));
  MK_TRY(check_matrix(who, "dlast", a->dlast, a->D, a->D, a->dlast ? 1 : 0, es));
  MK_TRY(check_floats(who, "dw", a->dw, true, false));
  MK_TRY(check_floats(who, "dbias", a->dbias, false, false));
  if (a->slots) return bad(who, "states are per sequence, slots are for serving");
  if (a->T && (a->dx == a->x || a->dx == a->dy)) return bad(who, "dx must not be x or dy (later tokens read them)");
  MK_ENTRY_DEVICE(dev);
  BwdPlan b = plan_bwd(a, dev);
  if (a->nseq == 0) b.parts = b.tiles = 0;
  const size_t need = (size_t)b.parts * (a->width + 1) * a->D * sizeof(float);
  if (need && (!a->workspace || a->workspace_bytes < need || !elem_aligned(a->workspace, 16)))
    return bad(who, "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");
  return dispatch<2>(a->type, a->width, b.V > 2, BwdOp{a, dev, mk::as_stream(stream), b});
}

int step(const mk_conv_step_args* a, void* stream) {
  const char* who = "mk_causal_conv_step";
  if (!a) return bad(who, "null arguments");
  mk_conv_args c{};
  c.type = a->type, c.width = a->width, c.D = a->D, c.T = a->B, c.w = a->w, c.bias = a->bias;
  c.slots = a->slots, c.nslots = a->nslots;
  MK_TRY(check(&c, who));
  MK_TRY(check_slots(who, a->slots, a->nslots, a->B));
  const size_t es = type_bytes(a->type);
  MK_TRY(check_matrix(who, "x", a->x, a->D, a->ldx, a->B, es));
  MK_TRY(check_matrix(who, "y", a->y, a->D, a->ldy, a->B, es));
  MK_TRY(check_matrix(who, "state", a->state, a->D, a->D, a->B, es));
  MK_TRY(check_matrix(who, "next", a->next, a->D, a->D, a->B, es));
  if (a->B == 0) return MK_OK;
  if (a->B * mk::cdiv(a->D, 128) > INT32_MAX) return bad(who, "batch too large for these channels");
  MK_ENTRY_DEVICE(dev);
  const int V = 4;
  const bool vec = a->D % V == 0 && vec_ok(a->x, a->ldx, es, V) && vec_ok(a->y, a->ldy, es, V) &&
                   vec_ok(a->state, 0, es, V) && vec_ok(a->next, 0, es, V);
  return dispatch<1>(a->type, a->width, vec, StepOp{a, dev, mk::as_stream(stream)});
}

}  // namespace

extern "C" int mk_causal_conv(const mk_conv_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return forward(a, stream); });
}

extern "C" int mk_causal_conv_grad_workspace(const mk_conv_args* a, size_t* bytes) {
  mk::clear_error();
  return guarded([&] { return grad_workspace(a, bytes); });
}

extern "C" int mk_causal_conv_grad(const mk_conv_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return gradient(a, stream); });
}

extern "C" int mk_causal_conv_step(const mk_conv_step_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return step(a, stream); });
}
