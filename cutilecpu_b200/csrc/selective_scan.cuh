// selective_scan.cuh — the selective state space scan: per channel d and state
// n, along the tokens of a sequence,
//     h[n] = exp(dt A[n]) h[n] + dt u B[n, t],   y = sum_n C[n, t] h[n] + D u,
// with dt = softplus(delta + bias) and the gate y *= silu(z).
//
// Bound by the exponentials, T * D * N of them at 16 per SM and clock (the
// special function unit), and by issue slots; the bytes are four matrices of
// T * D.  So the recurrence runs in registers, token by token:
//   * lane p * CW + c of a warp (CW = 32 / P) holds states p * NS ... (NS * P
//     >= N) of CH channels, c and c + CW.  Products are taken two states at a
//     time (f32x2), which halves their issue slots; with CH = 2 the values of B
//     and C that a lane reads serve two channels, which matters because shared
//     memory gives an SM only 32 values per clock;
//   * a block takes kTS tokens of its channels at a time.  What a (token,
//     channel) needs once is computed in front of and behind the recurrence by
//     one thread each, over 16-byte vectors: dt and dt u go through shared
//     memory to the P lanes of their channel, the sums over states come back
//     the same way and are gated and stored;
//   * B and C, the same for all channels of a group, are staged in Float32;
//   * the next tile's global loads are in flight while a tile is scanned.
// With few rows (one long sequence, few channels) sequences are cut into
// pieces: a first launch computes each piece's state from zero and its sum of
// dt (the decay over a piece is exp(A sum dt)), a second one chains them to
// the piece's starting state and runs the piece.
#pragma once

#include "tokens.cuh"

namespace mk {
namespace scan {

using namespace mk::tok;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTS = MK_SCAN_PIECE;  // tokens per tile, and between saved states
constexpr int kFwdGroup = 8;        // tokens per unrolled group
// Backward: as few as a sum over the lanes of a channel can be scattered over.
template <int P, int CH> constexpr int kBwdGroup = P / CH > 4 ? 8 : 4;

template <typename T>
struct Scan {
  Seqs q;
  int64_t D, N, G, Dg;  // Dg: channels per group
  int64_t tpg, tiles;   // channel tiles per group, and of all groups
  int64_t items;        // sequences, or pieces of them
  int64_t piece;        // tokens per piece, 0: whole sequences
  const T *u, *delta, *z, *B, *C, *dy;
  T *y, *du, *ddelta, *dz;
  int64_t ldu, lddelta, ldz, ldb, ldc, ldy, lddy, lddu, ldddelta, lddz;
  const float *A, *Dskip, *bias, *init, *dlast;
  float *last, *saved, *dinit;
  float *wstate, *wsum;  // pieces: state and sum of dt, [items][D][N], [items][D]
  float* parts;          // backward: dB, dC of a channel tile, [2][tpg][T][G * N]
  float *partA, *partD;  // backward: [grid items][D][N], [grid items][2][D]
  int64_t grid_items;
  const int32_t* slots;
  int64_t nslots;
  int softplus;
  bool vec_bc;  // B and C may be fetched several values at a time
  unsigned* err;
};

// Where a thread stands in the recurrence: its channels and its states.  With
// CH = 2 lanes with odd p hold their two channels the other way round, so that
// a sum over the lanes of a channel starts with each lane keeping its first.
template <int NS, int P, int CH>
struct Place {
  static constexpr int CW = 32 / P;            // lanes that share their states
  static constexpr int CB = kWarps * CW * CH;  // channels of a block
  static constexpr int NP = NS * P;
  static constexpr int R = P / CH;             // lanes a sum is still spread over after the first step
  int p, c, ch[CH];                            // ch: channels within the block
  int64_t tile, g, tg, base, d[CH];            // base: the block's first channel
  int left;                                    // channels of the block that exist
  bool live[CH];
};

template <int NS, int P, int CH, typename T>
__device__ __forceinline__ Place<NS, P, CH> place(const Scan<T>& q, int64_t tile) {
  Place<NS, P, CH> w;
  const int lane = threadIdx.x & 31;
  w.p = lane / w.CW;
  w.c = lane % w.CW;
  w.tile = tile;
  w.g = tile / q.tpg;
  w.tg = tile % q.tpg;
  w.base = w.g * q.Dg + w.tg * w.CB;
  const int64_t left = q.Dg - w.tg * w.CB;
  w.left = left < w.CB ? (int)left : w.CB;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    w.ch[i] = (threadIdx.x >> 5) * w.CW * CH + (i ^ (w.p & (CH - 1))) * w.CW + w.c;
    w.live[i] = w.ch[i] < w.left;
    w.d[i] = w.base + (w.live[i] ? w.ch[i] : 0);
  }
  return w;
}

// The sums over the P lanes of each channel of v[i][k] (channel register i,
// token k), scattered: a lane ends with channel w.ch[0], tokens e * R + r.
template <int K, int P, int CH>
__device__ __forceinline__ void reduce_states(float (&v)[CH][K], int p, float (&out)[K * CH / P]) {
  constexpr int CW = 32 / P;
  if constexpr (CH == 2) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[0][k] += __shfl_xor_sync(0xffffffffu, v[1][k], CW);
  }
  reduce_scatter<K, P / CH, CW * CH>(v[0], p / CH, out);
}

// Looks sequence i over: its offsets and its slot.  There are at least as many
// items as sequences, so that item i does this for sequence i, whichever
// sequence it is a piece of: where offsets descend, some have no item at all.
template <typename T>
__device__ __forceinline__ void check_sequence(const Scan<T>& p, int64_t i) {
  if (i >= p.q.nseq) return;
  if (threadIdx.x == 0 && seq_span(p.q, i).bad) atomicOr(p.err, mk::ERRBIT_SEQS);
  check_distinct(p.slots, i, threadIdx.x, kThreads, p.err);
}

struct Item {
  int64_t s, c, first;  // sequence, piece of it, number of its first piece
  int64_t lo, hi;       // the sequence's columns
  int64_t t0, t1;       // the piece's
  bool none;            // no such piece
};

template <typename T>
__device__ __forceinline__ Item item_at(const Scan<T>& p, int64_t i) {
  Item it;
  it.s = p.piece ? seq_of_piece(p.q, i, p.piece) : i;
  it.first = p.piece ? first_piece(p.q, it.s, p.piece) : i;
  it.c = i - it.first;
  const Span sp = seq_span(p.q, it.s);
  it.lo = sp.lo;
  it.hi = sp.hi;
  it.t0 = sp.lo + it.c * p.piece;
  it.t1 = p.piece ? min(sp.hi, it.t0 + p.piece) : sp.hi;
  it.none = it.c < 0 || (it.c > 0 && it.t0 >= sp.hi);  // below 0: columns in front of the first sequence
  return it;
}

// A lane's NS states of a row of N floats, register i holding state n0 + (i ^ m).
template <int NS>
__device__ __forceinline__ void load_states(F2 (&h)[NS / 2], const float* at, int64_t n0, int64_t N, int m = 0) {
  float f[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) f[i] = n0 + (i ^ m) < N ? at[n0 + (i ^ m)] : 0.0f;
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) h[i] = pack(f[2 * i], f[2 * i + 1]);
}

template <int NS>
__device__ __forceinline__ void store_states(float* at, const F2 (&h)[NS / 2], int64_t n0, int64_t N, int m = 0) {
#pragma unroll
  for (int i = 0; i < NS / 2; ++i) {
    float a, b;
    unpack(h[i], a, b);
    if (n0 + ((2 * i) ^ m) < N) at[n0 + ((2 * i) ^ m)] = a;
    if (n0 + ((2 * i + 1) ^ m) < N) at[n0 + ((2 * i + 1) ^ m)] = b;
  }
}

// The same in natural order over 16-byte vectors, where N allows.
template <int NS>
__device__ __forceinline__ void store_states_vec(float* at, const F2 (&h)[NS / 2], int64_t n0, int64_t N) {
  if constexpr (NS >= 4) {
    if (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < NS / 2; i += 2)
        if (n0 + 2 * i < N) *reinterpret_cast<ulonglong2*>(at + n0 + 2 * i) = make_ulonglong2(h[i].v, h[i + 1].v);
      return;
    }
  }
  store_states<NS>(at, h, n0, N);
}

// A lane's NS values of a row in shared memory.
template <int NS>
__device__ __forceinline__ void row_of(F2 (&f)[NS / 2], const float* row) {
  if constexpr (NS == 2) {
    f[0].v = *reinterpret_cast<const unsigned long long*>(row);
  } else {
#pragma unroll
    for (int i = 0; i < NS / 2; i += 2) {
      const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(row + 2 * i);
      f[i].v = v.x, f[i + 1].v = v.y;
    }
  }
}

// B and C in M orders (order m holds state i ^ m in place i of each run of M):
// a token's orders stand PAD floats further apart than they are long, which
// keeps both the lanes that read (a different order each) and the threads that
// write (a different run each) in different banks.
template <int NS, int P>
struct Orders {
  static constexpr int NP = NS * P, M = NS < 4 ? NS : 4;
  static constexpr int kStride = NP + (NS < 4 ? 2 : 4);  // floats from an order to the next
  static constexpr int kRow = M * kStride;               // and from a token to the next
};
// A tile of B or C: RB neighbouring values of a token per thread, fetched as
// they are, later put into shared memory as Float32.  `vec`: one access.
template <int NP, typename T>
struct Fetched {
  static constexpr int RB = kTS * NP / kThreads;
  Vec<T, RB> r;
  static __device__ __forceinline__ int row() { return threadIdx.x * RB / NP; }
  static __device__ __forceinline__ int col() { return threadIdx.x * RB % NP; }
  __device__ __forceinline__ void fetch(const T* m, int64_t ld, int64_t from, int64_t N, int64_t t, int64_t t1,
                                        bool vec) {
    const int k = row(), n = col();
    const T* at = m + (t + k) * ld + from + n;
#pragma unroll
    for (int i = 0; i < RB; ++i) r.v[i] = from_f<T>(0.0f);
    const int64_t left = t + k < t1 ? N - n : 0;  // values of the token that exist
    if (vec) {
      constexpr int C = sizeof(T) * RB <= 16 ? RB : 16 / (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < RB; i += C)
        load_if(reinterpret_cast<Vec<T, C>&>(r.v[i]), reinterpret_cast<const Vec<T, C>*>(at + i), i < left);
    } else {
#pragma unroll
      for (int i = 0; i < RB; ++i)
        load_if(reinterpret_cast<Vec<T, 1>&>(r.v[i]), reinterpret_cast<const Vec<T, 1>*>(at + i), i < left);
    }
  }
  __device__ __forceinline__ void put(float* sm) const {
#pragma unroll
    for (int i = 0; i < RB; ++i) sm[threadIdx.x * RB + i] = to_f(r.v[i]);
  }
  template <int NS, int P>
  __device__ __forceinline__ void put_orders(float* sm) const {
    using O = Orders<NS, P>;
    constexpr int M = O::M;
    static_assert(RB % M == 0, "a thread's values are whole runs");
    float* at = sm + row() * O::kRow + col();
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int i = 0; i < RB; i += M) {
        Vec<float, M> v;
#pragma unroll
        for (int x = 0; x < M; ++x) v.v[x] = to_f(r.v[i + (x ^ m)]);
        *reinterpret_cast<Vec<float, M>*>(at + m * O::kStride + i) = v;
      }
  }
};

// The (token, channel) values that threads exchange through shared memory sit
// at k * CB + ch with pairs of neighbours permuted by token and channel, so
// that the threads in front (V channels each, in pairs of 16 bytes) and the
// lanes of the recurrence (8 bytes each) both hit different banks.
template <int CB>
__device__ __forceinline__ int cell2(int k, int ch) {
  return k * CB + (ch ^ ((((ch >> 4) + k * (CB / 16)) & 3) << 1));
}
// The vectors of V channels of a tile, spread over the block's threads.
template <int CB, int V>
struct Spread {
  static constexpr int kPerRow = CB / V;
  static constexpr int kCount = kTS * kPerRow;
  static constexpr int NV = (kCount + kThreads - 1) / kThreads;
  static constexpr int kRows = kThreads / kPerRow;  // rows from a thread's vector to its next
  static __device__ __forceinline__ bool has(int i) {
    return kCount % kThreads == 0 || i * kThreads + (int)threadIdx.x < kCount;
  }
  static __device__ __forceinline__ int row(int i) { return (i * kThreads + threadIdx.x) / kPerRow; }
  static __device__ __forceinline__ int col() { return threadIdx.x % kPerRow * V; }  // the same for every i
};

// A thread's vectors of a tile from its first one's address on, of the rows below
// `rows`.  The address advances by rows: multiplied out for every element it cost
// 4 x 2048 x 4095 (bf16) forward 345 us instead of 301, backward 1267 instead of 1107.
template <typename S, typename T, int V, int NV>
__device__ __forceinline__ void fetch_rows(Vec<T, V> (&r)[NV], const T* at, int64_t ld, int rows) {
#pragma unroll
  for (int i = 0; i < NV; ++i, at += S::kRows * ld)
    load_if(r[i], reinterpret_cast<const Vec<T, V>*>(at), S::has(i) && S::row(i) < rows);
}

template <int E, typename T>
__device__ __forceinline__ F2 pair_of(const T* p) {
  return pack(to_f(p[0]), E == 2 ? to_f(p[E - 1]) : 0.0f);
}

template <int E, typename T>
__device__ __forceinline__ void out_pair(T* p, F2 x) {
  if constexpr (E == 2) {
    from_f2(p, x);
  } else {
    float a, b;
    unpack(x, a, b);
    p[0] = from_f<T>(a);
  }
}

// Two values of a channel and of its neighbour (E == 2) in their cells; zeros where not `in`.
struct Cell {
  F2 a, b;
};
template <int E>
__device__ __forceinline__ void put_cell(float2* cell, F2 a, F2 b, bool in, bool there) {
  float a0, a1, b0, b1;
  unpack(a, a0, a1), unpack(b, b0, b1);
  if (!in) a0 = a1 = b0 = b1 = 0.0f;
  if (!there) return;
  if constexpr (E == 2) *reinterpret_cast<float4*>(cell) = make_float4(a0, b0, a1, b1);
  else *cell = make_float2(a0, b0);
}
template <int E>
__device__ __forceinline__ Cell get_cell(const float2* cell) {
  if constexpr (E == 2) {
    const float4 v = *reinterpret_cast<const float4*>(cell);
    return {pack(v.x, v.z), pack(v.y, v.w)};
  } else {
    return {pack(cell->x, 0.0f), pack(cell->y, 0.0f)};
  }
}
// softplus of a thread's values; single elements are taken two at a time.
template <bool EXACT, int E, int NV, int Q>
__device__ __forceinline__ void softplus_all(F2 (&x)[NV][Q]) {
  if constexpr (E == 2 || NV % 2) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < Q; ++e) x[i][e] = softplus2<EXACT>(x[i][e]);
  } else {
    static_assert(Q == 1, "one element");
#pragma unroll
    for (int i = 0; i < NV; i += 2) {
      float a, b, none;
      unpack(x[i][0], a, none), unpack(x[i + 1][0], b, none);
      unpack(softplus2<EXACT>(pack(a, b)), a, b);
      x[i][0] = pack(a, 0.0f), x[i + 1][0] = pack(b, 0.0f);
    }
  }
}
template <bool EXACT, int E>
__device__ __forceinline__ F2 sigmoid_pair(F2 x) {
  float a, b;
  unpack(x, a, b);
  return pack(sigmoid<EXACT>(a), E == 2 ? sigmoid<EXACT>(b) : 0.0f);
}

// The parameters of channel ch of a block (and of the next, E == 2); zero without any.
template <int E>
__device__ __forceinline__ F2 channel_pair(const float* p, int64_t base, int ch, int left) {
  const float a = p && ch < left ? p[base + ch] : 0.0f;
  return pack(a, E == 2 && p && ch + 1 < left ? p[base + ch + 1] : 0.0f);
}

template <typename T, int V, int NV>
struct RawFwd {
  Vec<T, V> u[NV], delta[NV], z[NV];
};

template <typename T, int V, int NV>
struct RawBwd {
  Vec<T, V> u[NV], delta[NV], dy[NV], z[NV];
};

// FULL: the scan itself.  Otherwise a piece's state from zero and its sum of dt.
// 4 x 2048 tokens of 4096 channels and 16 states (bf16, gate, saved states): 264
// us, 2.05e12 states per second, 44% of what the exponentials alone allow; the
// special function units are 59% busy (with softplus and gate), the shared memory
// pipes 56%, the issue slots 54%, at 3.5 warps per scheduler, which waits between
// dependent steps keep from overlapping further.
template <typename T, int NS, int P, int CH, bool VEC, bool FULL>
__global__ void __launch_bounds__(kThreads, NS <= 4 ? 4 : 3) scan_fwd(Scan<T> p) {
  using W = Place<NS, P, CH>;
  constexpr int NP = W::NP, CB = W::CB, R = W::R, H = NS / 2, K = kFwdGroup;
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  using S = Spread<CB, V>;
  __shared__ __align__(16) float2 cells[kTS * CB];  // dt, dt u; then y, -
  __shared__ __align__(16) float sB[kTS][NP];
  __shared__ __align__(16) float sC[FULL ? kTS : 1][NP];
  const int64_t tile = blockIdx.x % p.tiles, item = blockIdx.x / p.tiles;
  const W w = place<NS, P, CH>(p, tile);
  if (FULL && tile == 0) check_sequence(p, item);
  const Item it = item_at(p, item);
  if (it.none) return;
  const int64_t n0 = w.p * NS;
  const int64_t row = p.init || p.last ? slot_of(p.slots, p.nslots, it.s, p.err) : -1;

  RawFwd<T, V, S::NV> cur, nxt;
  auto load_raw = [&](RawFwd<T, V, S::NV>& r, int64_t tt) {
    const int64_t t = tt + S::row(0), d = w.base + S::col();
    const int rows = S::col() < w.left ? (int)min(it.t1 - tt, (int64_t)kTS) : 0;
    fetch_rows<S>(r.u, p.u + t * p.ldu + d, p.ldu, rows);
    fetch_rows<S>(r.delta, p.delta + t * p.lddelta + d, p.lddelta, rows);
    fetch_rows<S>(r.z, p.z + t * p.ldz + d, p.ldz, FULL && p.z ? rows : 0);
  };
  Fetched<NP, T> fB, fC;
  auto fetch = [&](int64_t tt) {
    fB.fetch(p.B, p.ldb, w.g * p.N, p.N, tt, it.t1, p.vec_bc);
    if (FULL) fC.fetch(p.C, p.ldc, w.g * p.N, p.N, tt, it.t1, p.vec_bc);
  };
  load_raw(cur, it.t0);
  fetch(it.t0);

  F2 A2[CH][H], h[CH][H];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    load_states<NS>(A2[i], p.A + w.d[i] * p.N, n0, p.N);
#pragma unroll
    for (int j = 0; j < H; ++j) A2[i][j] = rate2(A2[i][j]), h[i][j] = pack(0.0f, 0.0f);
    // Pieces: entry 0 of a sequence's workspace is its initial state (read from
    // there by every piece, because `last` may replace it), entry c + 1 the
    // state that piece c leaves when it starts from zero.
    if (!FULL || !p.piece) {
      if (it.c == 0 && p.init && row >= 0) load_states<NS>(h[i], p.init + (row * p.D + w.d[i]) * p.N, n0, p.N);
      if (!FULL) {
        if (it.c == 0 && w.live[i]) store_states_vec<NS>(p.wstate + (item * p.D + w.d[i]) * p.N, h[i], n0, p.N);
#pragma unroll
        for (int j = 0; j < H; ++j) h[i][j] = pack(0.0f, 0.0f);
      }
    } else {
      const float* ws = p.wstate + (it.first * p.D + w.d[i]) * p.N;
      const float* wd = p.wsum + it.first * p.D + w.d[i];
      load_states<NS>(h[i], ws, n0, p.N);
#pragma unroll 4  // loads of several pieces in flight
      for (int64_t k = 0; k < it.c; ++k) {
        F2 add[H];
        load_states<NS>(add, ws + (k + 1) * p.D * p.N, n0, p.N);
        const F2 sum = pack(wd[k * p.D], wd[k * p.D]);
#pragma unroll
        for (int j = 0; j < H; ++j) h[i][j] = fma2(decay2(sum, A2[i][j]), h[i][j], add[j]);
      }
    }
  }
  if (!FULL && it.t1 >= it.hi) return;
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int E = V > 1 ? 2 : 1, Q = V / E;  // values taken at once, and how often
  F2 bias[(V + 1) / 2], skip[(V + 1) / 2];
#pragma unroll
  for (int i = 0; i < V; i += E) {
    bias[i / 2] = channel_pair<E>(p.bias, w.base, S::col() + i, w.left);
    skip[i / 2] = channel_pair<E>(FULL ? p.Dskip : nullptr, w.base, S::col() + i, w.left);
  }
  // where a token's values for this lane's channels sit, relative to the token: the order repeats every KV tokens
  constexpr int KV = CB >= 64 ? 1 : 64 / CB;
  int at[CH][KV];
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int k = 0; k < KV; ++k) at[i][k] = cell2<CB>(k, w.ch[i]) - k * CB;
  float sum_dt[CH] = {};

  for (int64_t tt = it.t0; tt < it.t1; tt += kTS) {
    {
      // one step for all values at a time: a branch per value would keep them from overlapping
      const int rows = S::col() < w.left ? (int)min(it.t1 - tt, (int64_t)kTS) : 0;
      F2 dt[S::NV][Q];
#pragma unroll
      for (int i = 0; i < S::NV; ++i)
#pragma unroll
        for (int e = 0; e < Q; ++e) dt[i][e] = add2(pair_of<E>(cur.delta[i].v + e * E), bias[e]);
      if (p.softplus) softplus_all<kExact, E>(dt);
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        const bool in = S::row(i) < rows;  // no token: the state stays
#pragma unroll
        for (int e = 0; e < Q; ++e)
          put_cell<E>(cells + cell2<CB>(S::row(i), S::col() + e * E), dt[i][e],
                      mul2(dt[i][e], pair_of<E>(cur.u[i].v + e * E)), in, S::has(i));
      }
    }
    fB.put(&sB[0][0]);
    if (FULL) fC.put(&sC[0][0]);
    __syncthreads();
    if (tt + kTS < it.t1) {
      load_raw(nxt, tt + kTS);
      fetch(tt + kTS);
    }
    if (FULL && p.saved) {
      float* sv = p.saved + (first_piece(p.q, it.s, kTS) + (tt - it.lo) / kTS) * p.D * p.N;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (w.live[i]) store_states_vec<NS>(sv + w.d[i] * p.N, h[i], n0, p.N);
    }
    const int groups = it.t1 - tt < kTS ? (int)((it.t1 - tt + K - 1) / K) : kTS / K;
    for (int q = 0; q < groups; ++q) {
      float2* cell = cells + q * K * CB;
      float yk[CH][K];
      // the decays of the whole group first: nothing in them waits for the state
      F2 a[K][CH][H];
      float dtu[K][CH];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const float2 v = cell[k * CB + at[i][k % KV]];
          dtu[k][i] = v.y;
          if (!FULL) sum_dt[i] += v.x;
#pragma unroll
          for (int j = 0; j < H; ++j) a[k][i][j] = fma2(pack(v.x), A2[i][j], pack(kDecayBias));
        }
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int j = 0; j < H; ++j) a[k][i][j] = ex2_2(a[k][i][j]);
      F2 b[2][H], c[2][H];  // this token's and the next's
      row_of<NS>(b[0], &sB[q * K][n0]);
      if (FULL) row_of<NS>(c[0], &sC[q * K][n0]);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (k + 1 < K) {
          row_of<NS>(b[(k + 1) & 1], &sB[q * K + k + 1][n0]);
          if (FULL) row_of<NS>(c[(k + 1) & 1], &sC[q * K + k + 1][n0]);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          F2 acc;
#pragma unroll
          for (int j = 0; j < H; ++j) {
            h[i][j] = fma2(a[k][i][j], h[i][j], mul2(pack(dtu[k][i], dtu[k][i]), b[k & 1][j]));
            if (FULL) acc = j ? fma2(c[k & 1][j], h[i][j], acc) : mul2(c[k & 1][j], h[i][j]);
          }
          if (FULL) yk[i][k] = sum2(acc);
        }
      }
      if constexpr (FULL) {
        float y[K / R];
        reduce_states<K, P, CH>(yk, w.p, y);
        __syncwarp();  // every lane has read the group's values
#pragma unroll
        for (int e = 0; e < K / R; ++e) {
          const int k = e * R + w.p / CH;
          cell[cell2<CB>(k, w.ch[0])].x = y[e];
        }
      }
    }
    __syncthreads();
    if constexpr (FULL) {
      T* to = p.y + (tt + S::row(0)) * p.ldy + w.base + S::col();
      const int rows = S::col() < w.left ? (int)min(it.t1 - tt, (int64_t)kTS) : 0;
#pragma unroll
      for (int i = 0; i < S::NV; ++i, to += S::kRows * p.ldy) {
        if (!S::has(i) || S::row(i) >= rows) continue;
        F2 y[Q];
#pragma unroll
        for (int e = 0; e < Q; ++e)
          y[e] = fma2(skip[e], pair_of<E>(cur.u[i].v + e * E),
                      get_cell<E>(cells + cell2<CB>(S::row(i), S::col() + e * E)).a);
        if (p.z) {
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            const F2 z = pair_of<E>(cur.z[i].v + e * E);
            y[e] = mul2(mul2(y[e], z), sigmoid_pair<kExact, E>(z));
          }
        }
        Vec<T, V> out;
#pragma unroll
        for (int e = 0; e < Q; ++e) out_pair<E>(out.v + e * E, y[e]);
        *reinterpret_cast<Vec<T, V>*>(to) = out;
      }
    }
    cur = nxt;
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (!w.live[i]) continue;
    if constexpr (FULL) {
      if (p.last && row >= 0 && it.t1 >= it.hi)
        store_states_vec<NS>(p.last + (row * p.D + w.d[i]) * p.N, h[i], n0, p.N);
    } else {
      store_states_vec<NS>(p.wstate + ((item + 1) * p.D + w.d[i]) * p.N, h[i], n0, p.N);
      if (w.p == 0) p.wsum[item * p.D + w.d[i]] = sum_dt[i];
    }
  }
}

// Backward over pieces, first launch (4 x 2048 x 4096: 141 us, two thirds of what
// its exponentials allow): what a piece hands to the token before
// it (e = a g of its first token) when nothing comes from behind, and its sum
// of dt.  The first piece of a sequence hands on nothing.
template <typename T, int NS, int P, int CH, bool VEC>
__global__ void __launch_bounds__(kThreads) scan_rev(Scan<T> p) {
  using W = Place<NS, P, CH>;
  constexpr int NP = W::NP, CB = W::CB, H = NS / 2, K = kFwdGroup;
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  using S = Spread<CB, V>;
  __shared__ __align__(16) float2 cells[kTS * CB];  // dt, dyp
  __shared__ __align__(16) float sC[kTS][NP];
  const int64_t tile = blockIdx.x % p.tiles, item = blockIdx.x / p.tiles;
  const W w = place<NS, P, CH>(p, tile);
  const Item it = item_at(p, item);
  if (it.none || it.c == 0) return;
  const int64_t n0 = w.p * NS;
  RawFwd<T, V, S::NV> cur, nxt;  // u: dy
  auto load_raw = [&](RawFwd<T, V, S::NV>& r, int64_t tt) {
    const int64_t t = tt + S::row(0), d = w.base + S::col();
    const int rows = S::col() < w.left ? (int)min(it.t1 - tt, (int64_t)kTS) : 0;
    fetch_rows<S>(r.u, p.dy + t * p.lddy + d, p.lddy, rows);
    fetch_rows<S>(r.delta, p.delta + t * p.lddelta + d, p.lddelta, rows);
    fetch_rows<S>(r.z, p.z + t * p.ldz + d, p.ldz, p.z ? rows : 0);
  };
  Fetched<NP, T> fC;
  const int64_t tiles = (it.t1 - it.t0 + kTS - 1) / kTS;
  int64_t tt = it.t0 + (tiles - 1) * kTS;
  load_raw(cur, tt);
  fC.fetch(p.C, p.ldc, w.g * p.N, p.N, tt, it.t1, p.vec_bc);
  F2 A2[CH][H], e_[CH][H];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    load_states<NS>(A2[i], p.A + w.d[i] * p.N, n0, p.N);
#pragma unroll
    for (int j = 0; j < H; ++j) A2[i][j] = rate2(A2[i][j]), e_[i][j] = pack(0.0f, 0.0f);
  }
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int E = V > 1 ? 2 : 1, Q = V / E;
  F2 bias[(V + 1) / 2];
#pragma unroll
  for (int i = 0; i < V; i += E) bias[i / 2] = channel_pair<E>(p.bias, w.base, S::col() + i, w.left);
  constexpr int KV = CB >= 64 ? 1 : 64 / CB;
  int at[CH][KV];
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int k = 0; k < KV; ++k) at[i][k] = cell2<CB>(k, w.ch[i]) - k * CB;
  float sum_dt[CH] = {};
  for (; tt >= it.t0; tt -= kTS) {
    {
      const int rows = S::col() < w.left ? (int)min(it.t1 - tt, (int64_t)kTS) : 0;
      F2 dt[S::NV][Q], dyp[S::NV][Q];
#pragma unroll
      for (int i = 0; i < S::NV; ++i)
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          dt[i][e] = add2(pair_of<E>(cur.delta[i].v + e * E), bias[e]);
          dyp[i][e] = pair_of<E>(cur.u[i].v + e * E);
        }
      if (p.softplus) softplus_all<kExact, E>(dt);
      if (p.z) {
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            const F2 z = pair_of<E>(cur.z[i].v + e * E);
            dyp[i][e] = mul2(mul2(dyp[i][e], z), sigmoid_pair<kExact, E>(z));
          }
      }
#pragma unroll
      for (int i = 0; i < S::NV; ++i) {
        const bool in = S::row(i) < rows;
#pragma unroll
        for (int e = 0; e < Q; ++e)
          put_cell<E>(cells + cell2<CB>(S::row(i), S::col() + e * E), dt[i][e], dyp[i][e], in, S::has(i));
      }
    }
    fC.put(&sC[0][0]);
    __syncthreads();
    if (tt > it.t0) {
      load_raw(nxt, tt - kTS);
      fC.fetch(p.C, p.ldc, w.g * p.N, p.N, tt - kTS, it.t1, p.vec_bc);
    }
    const int groups = it.t1 - tt < kTS ? (int)((it.t1 - tt + K - 1) / K) : kTS / K;
    for (int q = groups - 1; q >= 0; --q) {
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
        F2 c[H];
        row_of<NS>(c, &sC[q * K + k][n0]);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const float2 v = cells[(q * K + k) * CB + at[i][k % KV]];
          const F2 dt = pack(v.x, v.x), dyp = pack(v.y, v.y);
#pragma unroll
          for (int j = 0; j < H; ++j) e_[i][j] = mul2(decay2(dt, A2[i][j]), fma2(c[j], dyp, e_[i][j]));
          sum_dt[i] += v.x;
        }
      }
    }
    __syncthreads();
    cur = nxt;
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (!w.live[i]) continue;
    store_states_vec<NS>(p.wstate + (item * p.D + w.d[i]) * p.N, e_[i], n0, p.N);
    if (w.p == 0) p.wsum[item * p.D + w.d[i]] = sum_dt[i];
  }
}

// Backward.  With g[t] = C[t] dyp[t] + e[t+1], e[t] = a[t] g[t] (e behind the
// last token: dlast) and q = a[t] h[t-1]:
//   dB += g dt u, dC += dyp h (summed over the channels of the group),
//   dA += g q dt, ddt = sum_n g (q A + B u), du = dt sum_n g B + D dyp.
// A block takes kTS tokens at a time from the end.  Their states are rebuilt
// from the saved state in front of them: one pass keeps the state at every
// fourth token, then each group of 4 tokens, last first, is run again with its
// a and h in registers and walked backwards.
//
// dB and dC are reduced over a warp's channels by shuffles, over the block's
// warps in shared memory, and over blocks by scan_fold in a fixed order.  Half
// of a reduce-scatter by shuffles is choosing what to keep and what to send;
// here lane c holds its states in the order i ^ (c % M) (B and C are staged in
// M such orders), so what it keeps is always its first registers.
//
// 4 x 2048 tokens of 4096 channels, 16 states (bf16): 837 us in pieces, 916 us
// whole; its two exponentials per state and token take 230 us.  What bounds it is
// latency: 255 registers leave two blocks to an SM, two warps to a scheduler,
// whose dependent steps (decay, state, gradient) and shuffles leave half of the
// issue slots empty.  One channel per lane and four blocks per SM measured 1017
// us, 2 states on each of 8 lanes 1056.
template <int NS, int P, int CH, int V>
struct BwdSmem {
  static constexpr int NP = NS * P, CB = kWarps * (32 / P) * CH, M = NS < 4 ? NS : 4;
  float2 X[kTS * CB];  // dt, dt u; then dt, sum g B
  float2 Y[kTS * CB];  // dyp, -; then sum g q A2, y
  alignas(16) float B[kTS * Orders<NS, P>::kRow], C[kTS * Orders<NS, P>::kRow];
  unsigned long long sub[kTS / kBwdGroup<P, CH> - 1][CH][NS / 2][kThreads];
  float red[2][kWarps][kBwdGroup<P, CH>][2][NP];
  float par[2][CB];            // bias and D of the block's channels
  float acc[2][CB][kWarps];    // sums for D and bias, at the end
};

// dB and dC of one token over the warp's channels: vB and vC, NS registers
// each, go to one place per (state, kind) of `red`.
template <int NS, int P>
__device__ __forceinline__ void reduce_channels(F2 (&vB)[NS / 2], F2 (&vC)[NS / 2], int p, int c, float* red) {
  constexpr int CW = 32 / P, NP = NS * P;
  constexpr unsigned kAll = 0xffffffffu;
  float b[NS], d[NS];
#pragma unroll
  for (int j = 0; j < NS / 2; ++j) unpack(vB[j], b[2 * j], b[2 * j + 1]), unpack(vC[j], d[2 * j], d[2 * j + 1]);
  constexpr int M = NS < 4 ? NS : 4;
  // register i of lane c holds state i ^ (c % M): its neighbour at distance x holds the same state in i ^ x
  if constexpr (M == 4) {
#pragma unroll
    for (int j = 0; j < NS; j += 4) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        b[j + i] += __shfl_xor_sync(kAll, b[j + i + 2], 2);
        d[j + i] += __shfl_xor_sync(kAll, d[j + i + 2], 2);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NS; j += M) {
    b[j] += __shfl_xor_sync(kAll, b[j + 1], 1);
    d[j] += __shfl_xor_sync(kAll, d[j + 1], 1);
  }
  // the lanes of one state that are left keep dB or dC
  if constexpr (CW > M) {
    const bool up = (c & M) != 0;
#pragma unroll
    for (int j = 0; j < NS; j += M) {
      const float keep = up ? d[j] : b[j], send = up ? b[j] : d[j];
      b[j] = keep + __shfl_xor_sync(kAll, send, M);
#pragma unroll
      for (int x = 2 * M; x < CW; x *= 2) b[j] += __shfl_xor_sync(kAll, b[j], x);
      if (c < 2 * M) red[(up ? NP : 0) + p * NS + j + (c & (M - 1))] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NS; j += M) {
      red[p * NS + j + (c & (M - 1))] = b[j];
      red[NP + p * NS + j + (c & (M - 1))] = d[j];
    }
  }
}

template <typename T, int NS, int P, int CH, bool VEC>
__global__ void __launch_bounds__(kThreads, CH == 1 && NS <= 4 ? 4 : NS == 2 ? 3 : 2) scan_bwd(Scan<T> p) {
  using W = Place<NS, P, CH>;
  constexpr int NP = W::NP, CB = W::CB, R = W::R, H = NS / 2, K = kBwdGroup<P, CH>;
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  using S = Spread<CB, V>;
  constexpr int M = NS < 4 ? NS : 4;
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int E = V > 1 ? 2 : 1, Q = V / E;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  BwdSmem<NS, P, CH, V>& sm = *reinterpret_cast<BwdSmem<NS, P, CH, V>*>(smem_raw);
  const int64_t tile = blockIdx.x % p.tiles, item0 = blockIdx.x / p.tiles;
  const int warp = threadIdx.x >> 5;
  const W w = place<NS, P, CH>(p, tile);
  const int64_t n0 = w.p * NS;
  const int m = w.c & (M - 1);
  F2 A2[CH][H], dA[CH][H];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    load_states<NS>(A2[i], p.A + w.d[i] * p.N, n0, p.N, m);
#pragma unroll
    for (int j = 0; j < H; ++j) A2[i][j] = rate2(A2[i][j]), dA[i][j] = pack(0.0f, 0.0f);
  }
  // A thread's share of the sums for D and bias: 2 V values of its vectors, summed over the RD lanes of the warp that
  // have the same channels, of which it keeps every RD-th.
  constexpr int RD = S::kPerRow < 32 ? 32 / S::kPerRow : 1, ND = 2 * V / RD;
  float sums[ND] = {};
  // where a token's values for this lane's channels sit, relative to the token: the order repeats every KV tokens
  constexpr int KV = CB >= 64 ? 1 : 64 / CB;
  int at[CH][KV];
#pragma unroll
  for (int i = 0; i < CH; ++i)
#pragma unroll
    for (int k = 0; k < KV; ++k) at[i][k] = cell2<CB>(k, w.ch[i]) - k * CB;
  constexpr int kRow = Orders<NS, P>::kRow;
  const float* lB = sm.B + m * Orders<NS, P>::kStride + n0;
  const float* lC = sm.C + m * Orders<NS, P>::kStride + n0;
  for (int i = threadIdx.x; i < CB; i += kThreads) {
    sm.par[0][i] = p.bias && i < w.left ? p.bias[w.base + i] : 0.0f;
    sm.par[1][i] = p.Dskip && i < w.left ? p.Dskip[w.base + i] : 0.0f;
  }
  auto par_pair = [&](int which, int ch) {
    if constexpr (E == 2) return F2{*reinterpret_cast<const unsigned long long*>(&sm.par[which][ch])};
    else return pack(sm.par[which][ch], 0.0f);
  };
  __syncthreads();
  // a thread's sums of dB and dC over the warps: which, token of the group and state, and where they go
  constexpr int kSums = 2 * K * NP / kThreads > 0 ? 2 * K * NP / kThreads : 1;
  int rb = 0;
  const int64_t GN = p.G * p.N;
  float* part_at[kSums];
#pragma unroll
  for (int x = 0; x < kSums; ++x) {
    const int i = x * kThreads + threadIdx.x, k = i / (2 * NP), which = i / NP % 2, n = i % NP;
    part_at[x] = p.parts + ((which * p.tpg + w.tg) * p.q.T + k) * GN + w.g * p.N + n;
  }
  auto load_raw = [&](RawBwd<T, V, S::NV>& r, int64_t tc, int64_t te) {
    const int64_t t = tc + S::row(0), d = w.base + S::col();
    const int rows = S::col() < w.left ? (int)(te - tc) : 0;
    fetch_rows<S>(r.u, p.u + t * p.ldu + d, p.ldu, rows);
    fetch_rows<S>(r.delta, p.delta + t * p.lddelta + d, p.lddelta, rows);
    fetch_rows<S>(r.dy, p.dy + t * p.lddy + d, p.lddy, rows);
    fetch_rows<S>(r.z, p.z + t * p.ldz + d, p.ldz, p.z ? rows : 0);
  };

  for (int64_t item = item0; item < p.items; item += p.grid_items) {
    if (tile == 0) check_sequence(p, item);
    const Item it = item_at(p, item);
    if (it.none) continue;
    F2 e_[CH][H];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
      for (int j = 0; j < H; ++j) e_[i][j] = pack(0.0f, 0.0f);
      if (p.dlast) load_states<NS>(e_[i], p.dlast + (it.s * p.D + w.d[i]) * p.N, n0, p.N, m);
      if (p.piece) {
#pragma unroll 4
        for (int64_t k = (it.hi - it.lo + p.piece - 1) / p.piece - 1; k > it.c; --k) {
          F2 add[H];
          load_states<NS>(add, p.wstate + ((it.first + k) * p.D + w.d[i]) * p.N, n0, p.N, m);
          const float s1 = p.wsum[(it.first + k) * p.D + w.d[i]];
          const F2 sum = pack(s1, s1);
#pragma unroll
          for (int j = 0; j < H; ++j) e_[i][j] = fma2(decay2(sum, A2[i][j]), e_[i][j], add[j]);
        }
      }
    }
    const int64_t piece0 = first_piece(p.q, it.s, kTS);
    const int64_t last_tile = (it.t1 - it.t0 + kTS - 1) / kTS - 1;
    RawBwd<T, V, S::NV> raw, next;
    Fetched<NP, T> fB, fC;
    F2 h[CH][H];
    // what a tile reads: asked for behind the recurrence of the tile before, whose registers are free then (vectors;
    // single elements take a register each, so they are asked for when they are due)
    auto ask = [&](int64_t ch) {
      const int64_t tc = it.t0 + ch * kTS, te = min(it.t1, tc + kTS);
      load_raw(next, tc, te);
      fB.fetch(p.B, p.ldb, w.g * p.N, p.N, tc, te, p.vec_bc);
      fC.fetch(p.C, p.ldc, w.g * p.N, p.N, tc, te, p.vec_bc);
      const float* sv = p.saved + (piece0 + (tc - it.lo) / kTS) * p.D * p.N;
#pragma unroll
      for (int i = 0; i < CH; ++i) load_states<NS>(h[i], sv + w.d[i] * p.N, n0, p.N, m);
    };
    if (VEC && last_tile >= 0) ask(last_tile);
    for (int64_t ch = last_tile; ch >= 0; --ch) {
      const int64_t tc = it.t0 + ch * kTS, te = min(it.t1, tc + kTS);
      const int nsub = (int)((te - tc + K - 1) / K);
      const int rows = S::col() < w.left ? (int)(te - tc) : 0;  // of this thread's vectors
      F2 dAc[CH][H];  // the tile's sum, so that long sums stay exact
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) dAc[i][j] = pack(0.0f, 0.0f);
      if (!VEC) ask(ch);
      raw = next;
      if (ch > 0) {
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
          if (!S::has(i) || S::col() >= w.left) continue;
          const int64_t t = tc - kTS + S::row(i), d = w.base + S::col();
          prefetch_l2(p.u + t * p.ldu + d);
          prefetch_l2(p.delta + t * p.lddelta + d);
          prefetch_l2(p.dy + t * p.lddy + d);
          if (p.z) prefetch_l2(p.z + t * p.ldz + d);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i)
          prefetch_l2(p.saved + ((piece0 + (tc - it.lo) / kTS - 1) * p.D + w.d[i]) * p.N + (n0 < p.N ? n0 : 0));
      }
      {
        // one step for all values at a time: a branch per value would keep them from overlapping
        F2 dt[S::NV][Q], dyp[S::NV][Q];
#pragma unroll
        for (int i = 0; i < S::NV; ++i)
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            dt[i][e] = add2(pair_of<E>(raw.delta[i].v + e * E), par_pair(0, S::col() + e * E));
            dyp[i][e] = pair_of<E>(raw.dy[i].v + e * E);
          }
        if (p.softplus) softplus_all<kExact, E>(dt);
        if (p.z) {
#pragma unroll
          for (int i = 0; i < S::NV; ++i)
#pragma unroll
            for (int e = 0; e < Q; ++e) {
              const F2 z = pair_of<E>(raw.z[i].v + e * E);
              dyp[i][e] = mul2(mul2(dyp[i][e], z), sigmoid_pair<kExact, E>(z));
            }
        }
#pragma unroll
        for (int i = 0; i < S::NV; ++i) {
          const bool in = S::row(i) < rows;
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            const int c = cell2<CB>(S::row(i), S::col() + e * E);
            put_cell<E>(sm.X + c, dt[i][e], mul2(dt[i][e], pair_of<E>(raw.u[i].v + e * E)), in, S::has(i));
            put_cell<E>(sm.Y + c, dyp[i][e], pack(0.0f), in, S::has(i));
          }
        }
      }
      fB.template put_orders<NS, P>(sm.B);
      fC.template put_orders<NS, P>(sm.C);
      __syncthreads();
      for (int q = 0; q < nsub - 1; ++q) {
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
          for (int j = 0; j < H; ++j) sm.sub[q][i][j][threadIdx.x] = h[i][j].v;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          F2 b[H];
          row_of<NS>(b, lB + (q * K + k) * kRow);
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const float2 v = sm.X[(q * K + k) * CB + at[i][k % KV]];
            const F2 dt = pack(v.x, v.x), dtu = pack(v.y, v.y);
#pragma unroll
            for (int j = 0; j < H; ++j) h[i][j] = fma2(decay2(dt, A2[i][j]), h[i][j], mul2(dtu, b[j]));
          }
        }
      }
      for (int q = nsub - 1; q >= 0; --q) {
        if (q != nsub - 1) {
#pragma unroll
          for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j) h[i][j].v = sm.sub[q][i][j][threadIdx.x];
        }
        float2 *X = sm.X + q * K * CB, *Y = sm.Y + q * K * CB;
        F2 a[K][CH][H], hh[K][CH][H];
        float yk[CH][K], sG[CH][K], sT[CH][K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          F2 b[H], c[H];
          row_of<NS>(b, lB + (q * K + k) * kRow);
          row_of<NS>(c, lC + (q * K + k) * kRow);
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const float2 v = X[k * CB + at[i][k % KV]];
            const F2 dt = pack(v.x, v.x), dtu = pack(v.y, v.y);
            F2 acc;
#pragma unroll
            for (int j = 0; j < H; ++j) {
              a[k][i][j] = decay2(dt, A2[i][j]);
              hh[k][i][j] = fma2(a[k][i][j], k ? hh[k ? k - 1 : 0][i][j] : h[i][j], mul2(dtu, b[j]));
              acc = j ? fma2(c[j], hh[k][i][j], acc) : mul2(c[j], hh[k][i][j]);
            }
            yk[i][k] = sum2(acc);
          }
        }
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
          F2 b[H], c[H], vB[H], vC[H];
          row_of<NS>(b, lB + (q * K + k) * kRow);
          row_of<NS>(c, lC + (q * K + k) * kRow);
#pragma unroll
          for (int i = 0; i < CH; ++i) {
            const float2 v = X[k * CB + at[i][k % KV]];
            const F2 dt = pack(v.x), dtu = pack(v.y), dyp = pack(Y[k * CB + at[i][k % KV]].x);
            F2 accG, accT;
#pragma unroll
            for (int j = 0; j < H; ++j) {
              const F2 g = fma2(c[j], dyp, e_[i][j]);
              const F2 gq = mul2(g, mul2(a[k][i][j], k ? hh[k ? k - 1 : 0][i][j] : h[i][j]));
              vC[j] = i ? fma2(dyp, hh[k][i][j], vC[j]) : mul2(dyp, hh[k][i][j]);
              vB[j] = i ? fma2(dtu, g, vB[j]) : mul2(dtu, g);
              dAc[i][j] = fma2(gq, dt, dAc[i][j]);
              accT = j ? fma2(gq, A2[i][j], accT) : mul2(gq, A2[i][j]);
              accG = j ? fma2(g, b[j], accG) : mul2(g, b[j]);
              e_[i][j] = mul2(a[k][i][j], g);
            }
            sT[i][k] = sum2(accT);
            sG[i][k] = sum2(accG);
          }
          reduce_channels<NS, P>(vB, vC, w.p, w.c, &sm.red[rb][warp][k][0][0]);
        }
        constexpr int KR = K / R;
        float y[KR], rG[KR], rT[KR];
        reduce_states<K, P, CH>(yk, w.p, y);
        reduce_states<K, P, CH>(sG, w.p, rG);
        reduce_states<K, P, CH>(sT, w.p, rT);
        __syncwarp();
#pragma unroll
        for (int e = 0; e < KR; ++e) {
          const int c = cell2<CB>(e * R + w.p / CH, w.ch[0]);
          X[c].y = rG[e];
          Y[c] = make_float2(rT[e], y[e]);
        }
        if (q == 0) load_raw(raw, tc, te);  // again, for what is left to do
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kSums; ++x) {
          const int i = x * kThreads + threadIdx.x, k = i / (2 * NP), which = i / NP % 2, n = i % NP;
          if (i >= 2 * K * NP) continue;
          float v = 0.0f;
#pragma unroll
          for (int y = 0; y < kWarps; ++y) v += sm.red[rb][y][k][which][n];
          const int64_t t = tc + q * K;
          if (t + k < te && n < p.N) part_at[x][t * GN] = v;
        }
        rb ^= 1;
      }
#pragma unroll
      for (int i = 0; i < CH; ++i)
#pragma unroll
        for (int j = 0; j < H; ++j) dA[i][j] = add2(dA[i][j], dAc[i][j]);
      if (VEC && ch > 0) ask(ch - 1);
      float add[2 * V] = {};
      const int64_t t = tc + S::row(0), d = w.base + S::col();
      T *to_u = p.du + t * p.lddu + d, *to_d = p.ddelta + t * p.ldddelta + d, *to_z = p.dz + t * p.lddz + d;
#pragma unroll
      for (int i = 0; i < S::NV;
           ++i, to_u += S::kRows * p.lddu, to_d += S::kRows * p.ldddelta, to_z += S::kRows * p.lddz) {
        if (!S::has(i) || S::row(i) >= rows) continue;
        Vec<T, V> du, dd, dz;
        F2 dyp[Q];
        Cell x[Q], y[Q];
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          const int c = cell2<CB>(S::row(i), S::col() + e * E);
          x[e] = get_cell<E>(sm.X + c), y[e] = get_cell<E>(sm.Y + c);  // dt, sum g B; sum g q A2, y
          dyp[e] = pair_of<E>(raw.dy[i].v + e * E);
        }
        if (p.z) {
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            const F2 z = pair_of<E>(raw.z[i].v + e * E), sz = sigmoid_pair<kExact, E>(z), gz = mul2(z, sz);
            const F2 all = fma2(par_pair(1, S::col() + e * E), pair_of<E>(raw.u[i].v + e * E), y[e].b);
            // silu' = s + z s (1 - s)
            out_pair<E>(dz.v + e * E, mul2(mul2(dyp[e], all), fma2(gz, fma2(sz, pack(-1.0f), pack(1.0f)), sz)));
            dyp[e] = mul2(dyp[e], gz);
          }
        }
        F2 dd2[Q];
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          out_pair<E>(du.v + e * E, fma2(x[e].a, x[e].b, mul2(par_pair(1, S::col() + e * E), dyp[e])));
          dd2[e] = fma2(pair_of<E>(raw.u[i].v + e * E), x[e].b, mul2(y[e].a, pack(kLn2)));
        }
        if (p.softplus) {
#pragma unroll
          for (int e = 0; e < Q; ++e) {
            F2 g;
            softplus2<kExact, true>(add2(pair_of<E>(raw.delta[i].v + e * E), par_pair(0, S::col() + e * E)), &g);
            dd2[e] = mul2(dd2[e], g);
          }
        }
#pragma unroll
        for (int e = 0; e < Q; ++e) {
          out_pair<E>(dd.v + e * E, dd2[e]);
          float a0, a1, b0, b1;
          unpack(mul2(dyp[e], pair_of<E>(raw.u[i].v + e * E)), a0, a1);
          unpack(dd2[e], b0, b1);
          add[e * E] += a0, add[V + e * E] += b0;
          if constexpr (E == 2) add[e * E + 1] += a1, add[V + e * E + 1] += b1;
        }
        *reinterpret_cast<Vec<T, V>*>(to_u) = du;
        *reinterpret_cast<Vec<T, V>*>(to_d) = dd;
        if (p.z) *reinterpret_cast<Vec<T, V>*>(to_z) = dz;
      }
      float more[ND];
      reduce_scatter<2 * V, RD, S::kPerRow>(add, (threadIdx.x & 31) / S::kPerRow, more);
#pragma unroll
      for (int i = 0; i < ND; ++i) sums[i] += more[i];
    }
    if (p.dinit && it.c == 0) {
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (w.live[i]) store_states<NS>(p.dinit + (it.s * p.D + w.d[i]) * p.N, e_[i], n0, p.N, m);
    }
  }
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (w.live[i]) store_states<NS>(p.partA + (item0 * p.D + w.d[i]) * p.N, dA[i], n0, p.N, m);
  for (int i = threadIdx.x; i < 2 * CB * kWarps; i += kThreads) (&sm.acc[0][0][0])[i] = 0.0f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ND; ++i) {
    const int v = i * RD + (threadIdx.x & 31) / S::kPerRow;
    sm.acc[v / V][S::col() + v % V][warp] = sums[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * w.left; i += kThreads) {  // D, then bias, over the warps
    const int which = i >= w.left, ch = i - which * w.left;
    float v = 0.0f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) v += sm.acc[which][ch][x];
    p.partD[(item0 * 2 + which) * p.D + w.base + ch] = v;
  }
}

// The sums over blocks: dB and dC over channel tiles (rounded once), dA, dD
// and dbias over the blocks of a channel.  64 tiles of 8192 tokens and 16 states:
// 21 us, 3.2 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) scan_fold(Scan<T> p, T* dB, T* dC, int64_t lddb, int64_t lddc, float* dA,
                                                 float* dD, float* dbias) {
  const int64_t GN = p.G * p.N, cells = p.q.T * GN, nA = p.D * p.N;
  const int64_t total = 2 * cells + nA + 2 * p.D;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    float v = 0.0f;
    if (i < 2 * cells) {
      const int which = i >= cells;
      const int64_t at = i - which * cells, t = at / GN;
      if (t < seq_offset(p.q, 0) || t >= seq_offset(p.q, p.q.nseq)) continue;
#pragma unroll 8
      for (int64_t k = 0; k < p.tpg; ++k) v += p.parts[(which * p.tpg + k) * cells + at];
      if (which) dC[t * lddc + at % GN] = from_f<T>(v);
      else dB[t * lddb + at % GN] = from_f<T>(v);
    } else if (i < 2 * cells + nA) {
      const int64_t at = i - 2 * cells;
#pragma unroll 8
      for (int64_t k = 0; k < p.grid_items; ++k) v += p.partA[k * nA + at];
      dA[at] = v;
    } else {
      const int64_t at = i - 2 * cells - nA;
      for (int64_t k = 0; k < p.grid_items; ++k) v += p.partD[k * 2 * p.D + at];
      if (at < p.D) {
        if (dD) dD[at] = v;
      } else if (dbias) {
        dbias[at - p.D] = v;
      }
    }
  }
}

// ---- host side ----------------------------------------------------------------

// Lanes per channel and states per lane: 2, 4 or 8 states on 4 lanes, beyond 32 states 8 on 8.
inline int lanes_of(int64_t N) { return N <= 32 ? 4 : 8; }
inline int states_of(int64_t N) { return N <= 8 ? 2 : N <= 16 ? 4 : 8; }
// Whether the gradient's registers hold two channels per lane: not with 8 states,
// nor with Float32 and 2 states (the code for it spilled 576 bytes).
constexpr bool two_channels(int states, size_t type_size) { return states == 4 || (states == 2 && type_size == 2); }

// Whether the token matrices can be taken in vectors of 16 bytes.
inline bool all_vec(const mk_scan_args* a, bool grad) {
  const size_t es = type_bytes(a->type);
  const int V = (int)(16 / es);
  bool ok = a->D / a->G % V == 0 && vec_ok(a->u, a->ldu, es, V) && vec_ok(a->delta, a->lddelta, es, V) &&
            vec_ok(a->z, a->ldz, es, V);
  if (!grad) return ok && vec_ok(a->y, a->ldy, es, V);
  return ok && vec_ok(a->dy, a->lddy, es, V) && vec_ok(a->du, a->lddu, es, V) &&
         vec_ok(a->ddelta, a->ldddelta, es, V) && vec_ok(a->dz, a->lddz, es, V);
}

// The same for B and C, of which a thread fetches kTS * NP / kThreads values of one token.
inline bool bc_vec(const mk_scan_args* a) {
  const size_t es = type_bytes(a->type);
  const int RB = kTS * states_of(a->N) * lanes_of(a->N) / kThreads;
  return a->N % RB == 0 && vec_ok(a->B, a->ldb, es, RB) && vec_ok(a->C, a->ldc, es, RB);
}

struct Plan {
  int ch;
  int64_t tpg, tiles, items, piece, grid_items;
  int64_t rev_tpg, rev_tiles;  // channel tiles of scan_rev, which takes one channel per lane
  size_t piece_bytes, part_bytes, bytes;
};

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T>
Scan<T> params(const mk_scan_args* a, const mk::Device* dev, const Plan& b) {
  Scan<T> p{};
  p.q = Seqs{a->seqs, a->nseq, a->len, a->T};
  p.D = a->D, p.N = a->N, p.G = a->G, p.Dg = a->D / a->G;
  p.tpg = b.tpg, p.tiles = b.tiles, p.items = b.items, p.piece = b.piece, p.grid_items = b.grid_items;
  p.u = static_cast<const T*>(a->u), p.ldu = a->ldu;
  p.delta = static_cast<const T*>(a->delta), p.lddelta = a->lddelta;
  p.z = static_cast<const T*>(a->z), p.ldz = a->ldz;
  p.B = static_cast<const T*>(a->B), p.ldb = a->ldb;
  p.C = static_cast<const T*>(a->C), p.ldc = a->ldc;
  p.y = static_cast<T*>(a->y), p.ldy = a->ldy;
  p.dy = static_cast<const T*>(a->dy), p.lddy = a->lddy;
  p.du = static_cast<T*>(a->du), p.lddu = a->lddu;
  p.ddelta = static_cast<T*>(a->ddelta), p.ldddelta = a->ldddelta;
  p.dz = static_cast<T*>(a->dz), p.lddz = a->lddz;
  p.A = a->A, p.Dskip = a->Dskip, p.bias = a->bias, p.init = a->init, p.dlast = a->dlast;
  p.last = a->last, p.saved = a->saved, p.dinit = a->dinit;
  p.slots = a->slots, p.nslots = a->nslots, p.softplus = a->softplus;
  p.vec_bc = bc_vec(a);
  p.err = dev->err_word;
  char* ws = static_cast<char*>(a->workspace);
  if (b.piece) {
    p.wstate = reinterpret_cast<float*>(ws);
    p.wsum = reinterpret_cast<float*>(ws + align256((size_t)b.items * a->D * a->N * 4));
  }
  ws += b.piece_bytes;
  p.parts = reinterpret_cast<float*>(ws);
  ws += align256((size_t)2 * b.tpg * a->T * a->G * a->N * 4);
  p.partA = reinterpret_cast<float*>(ws);
  p.partD = reinterpret_cast<float*>(ws + align256((size_t)b.grid_items * a->D * a->N * 4));
  return p;
}

template <typename T, int NS, int P, bool VEC>
int run_fwd(const mk_scan_args* a, const mk::Device* dev, const Plan& b, cudaStream_t s) {
  const Scan<T> p = params<T>(a, dev, b);
  const unsigned grid = (unsigned)(b.tiles * b.items);
  if (b.piece) scan_fwd<T, NS, P, 1, VEC, false><<<grid, kThreads, 0, s>>>(p);
  scan_fwd<T, NS, P, 1, VEC, true><<<grid, kThreads, 0, s>>>(p);
  return mk::check_launch("mk_selective_scan: launch");
}

template <typename T, int NS, int P, int CH, bool VEC>
int run_bwd(const mk_scan_args* a, const mk::Device* dev, const Plan& b, cudaStream_t s) {
  const Scan<T> p = params<T>(a, dev, b);
  constexpr size_t smem = sizeof(BwdSmem<NS, P, CH, VEC ? 16 / (int)sizeof(T) : 1>);
  MK_TRY(mk::allow_dynamic_smem(reinterpret_cast<const void*>(&scan_bwd<T, NS, P, CH, VEC>), smem));
  if (b.piece) {
    Scan<T> q = p;
    q.tpg = b.rev_tpg, q.tiles = b.rev_tiles;
    scan_rev<T, NS, P, 1, VEC><<<(unsigned)(q.tiles * b.items), kThreads, 0, s>>>(q);
  }
  if (b.grid_items) scan_bwd<T, NS, P, CH, VEC><<<(unsigned)(b.tiles * b.grid_items), kThreads, smem, s>>>(p);
  const int64_t total = 2 * a->T * a->G * a->N + a->D * (a->N + 2);
  int64_t blocks = mk::cdiv(total, 256);
  if (blocks > (int64_t)dev->sms * 16) blocks = (int64_t)dev->sms * 16;
  scan_fold<T><<<(unsigned)blocks, 256, 0, s>>>(p, static_cast<T*>(a->dB), static_cast<T*>(a->dC), a->lddb, a->lddc,
                                                a->dA, a->dDskip, a->dbias);
  return mk::check_launch("mk_selective_scan_grad: launch");
}

template <typename T, int NS, int P>
int run_vec(const mk_scan_args* a, const mk::Device* dev, const Plan& b, bool grad, cudaStream_t s) {
  const bool vec = all_vec(a, grad);
  if (!grad) return vec ? run_fwd<T, NS, P, true>(a, dev, b, s) : run_fwd<T, NS, P, false>(a, dev, b, s);
  if constexpr (two_channels(NS, sizeof(T))) {
    if (b.ch == 2) return run_bwd<T, NS, P, 2, true>(a, dev, b, s);
  }
  return vec ? run_bwd<T, NS, P, 1, true>(a, dev, b, s) : run_bwd<T, NS, P, 1, false>(a, dev, b, s);
}

template <typename T>
int run_type(const mk_scan_args* a, const mk::Device* dev, const Plan& b, bool grad, cudaStream_t s) {
  if (a->N <= 8) return run_vec<T, 2, 4>(a, dev, b, grad, s);
  if (a->N <= 16) return run_vec<T, 4, 4>(a, dev, b, grad, s);
  if (a->N <= 32) return run_vec<T, 8, 4>(a, dev, b, grad, s);
  return run_vec<T, 8, 8>(a, dev, b, grad, s);
}

// One source file per element type compiles its kernels.
extern template int run_type<float>(const mk_scan_args*, const mk::Device*, const Plan&, bool, cudaStream_t);
extern template int run_type<__half>(const mk_scan_args*, const mk::Device*, const Plan&, bool, cudaStream_t);
extern template int run_type<__nv_bfloat16>(const mk_scan_args*, const mk::Device*, const Plan&, bool, cudaStream_t);

}  // namespace scan
}  // namespace mk
