// selective_scan.cu — the selective state space scan: per channel d and state
// n, along the tokens of a sequence,
//     h[n] = exp(dt A[n]) h[n] + dt u B[n, t],   y = sum_n C[n, t] h[n] + D u,
// with dt = softplus(delta + bias) and the gate y *= silu(z).
//
// Bound by the exponentials: T * D * N of them at 16 per SM and clock (the
// special function unit), and about as many issue slots; the bytes are 4
// matrices of T * D.  So the recurrence runs in registers, token by token:
//   * a warp holds CW = 32 / P channels, P lanes per channel, NS states per
//     lane (NS * P >= N): lane p * CW + c holds states p * NS ... of channel c;
//   * what a (token, channel) needs once (softplus, gate, skip) is computed by
//     one of its P lanes: tokens go in groups of 8, lane p takes tokens p,
//     p + P, ...; dt and dt u reach the other lanes by shuffles, the sums over
//     states come back by a reduce-scatter;
//   * B and C are the same for all channels of a group: a block stages TS
//     tokens of them in shared memory (Float32), double-buffered, and loads the
//     next group's u, delta, z into registers before it computes the present.
// With few rows (one long sequence, few channels) sequences are cut into
// pieces: a first launch computes each piece's state from zero and its sum of
// dt (the decay over a piece is exp(A sum dt)), a second one chains them to
// the piece's starting state and runs the piece.
#include "tokens.cuh"

namespace {

using namespace mk::tok;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kGroup = 8;             // tokens per group
constexpr int kTile = 32;             // tokens of B and C staged at once (forward)
constexpr int kPiece = MK_SCAN_PIECE; // tokens between saved states

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
  unsigned* err;
};

// Where a thread stands: its channel, its states, its piece of a sequence.
template <int NS, int P>
struct Place {
  static constexpr int CW = 32 / P;
  static constexpr int CB = kWarps * CW;  // channels of a block
  static constexpr int NP = NS * P;
  static constexpr int E = kGroup / P;    // tokens of a group that a lane takes
  int warp, p, c;
  int64_t tile, g, tg, d;
  bool live;
};

template <int NS, int P, typename T>
__device__ __forceinline__ Place<NS, P> place(const Scan<T>& q, int64_t tile) {
  Place<NS, P> w;
  const int lane = threadIdx.x & 31;
  w.warp = threadIdx.x >> 5;
  w.p = lane / w.CW;
  w.c = lane % w.CW;
  w.tile = tile;
  w.g = tile / q.tpg;
  w.tg = tile % q.tpg;
  const int64_t at = w.tg * w.CB + w.warp * w.CW + w.c;
  w.live = at < q.Dg;
  w.d = w.g * q.Dg + (w.live ? at : 0);
  return w;
}

struct Item {
  int64_t s, c, first;  // sequence, piece of it, number of its first piece
  int64_t lo, hi;       // the sequence's columns
  int64_t t0, t1;       // the piece's
  bool bad, none;       // none: no such piece
};

template <typename T>
__device__ __forceinline__ Item item_at(const Scan<T>& p, int64_t i) {
  Item it;
  it.s = p.piece ? seq_of_piece(p.q, i, p.piece) : i;
  it.first = p.piece ? first_piece(p.q, it.s, p.piece) : i;
  it.c = i - it.first;
  const Span sp = seq_span(p.q, it.s);
  it.bad = sp.bad;
  it.lo = sp.lo;
  it.hi = sp.hi;
  it.t0 = sp.lo + it.c * p.piece;
  it.t1 = p.piece ? min(sp.hi, it.t0 + p.piece) : sp.hi;
  it.none = it.c > 0 && it.t0 >= sp.hi;
  return it;
}

template <int NS>
__device__ __forceinline__ void load_states(float (&h)[NS], const float* at, int64_t n0, int64_t N) {
  if (N % 4 == 0) {
#pragma unroll
    for (int j = 0; j < NS; j += 4) {
      const float4 v = n0 + j < N ? *reinterpret_cast<const float4*>(at + n0 + j) : make_float4(0, 0, 0, 0);
      h[j] = v.x, h[j + 1] = v.y, h[j + 2] = v.z, h[j + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < NS; ++j) h[j] = n0 + j < N ? at[n0 + j] : 0.0f;
  }
}

template <int NS>
__device__ __forceinline__ void store_states(float* at, const float (&h)[NS], int64_t n0, int64_t N) {
  if (N % 4 == 0) {
#pragma unroll
    for (int j = 0; j < NS; j += 4)
      if (n0 + j < N) *reinterpret_cast<float4*>(at + n0 + j) = make_float4(h[j], h[j + 1], h[j + 2], h[j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (n0 + j < N) at[n0 + j] = h[j];
  }
}

template <int NS>
__device__ __forceinline__ void row_of(float (&f)[NS], const float* row) {
#pragma unroll
  for (int j = 0; j < NS; j += 4) {
    const float4 v = *reinterpret_cast<const float4*>(row + j);
    f[j] = v.x, f[j + 1] = v.y, f[j + 2] = v.z, f[j + 3] = v.w;
  }
}

// A tile of `TS` tokens of B or C: fetched to registers, put into shared memory.
template <int TS, int NP, typename T>
__device__ __forceinline__ void fetch(float (&r)[TS * NP / kThreads], const T* m, int64_t ld, int64_t col, int64_t N,
                                      int64_t t, int64_t t1) {
#pragma unroll
  for (int j = 0; j < TS * NP / kThreads; ++j) {
    const int i = j * kThreads + threadIdx.x, k = i / NP, n = i % NP;
    r[j] = t + k < t1 && n < N ? to_f(m[(t + k) * ld + col + n]) : 0.0f;
  }
}

template <int TS, int NP>
__device__ __forceinline__ void put(float* sm, const float (&r)[TS * NP / kThreads]) {
#pragma unroll
  for (int j = 0; j < TS * NP / kThreads; ++j) sm[j * kThreads + threadIdx.x] = r[j];
}

template <typename T, int E>
struct Raw {
  T u[E], delta[E], z[E], dy[E];
};

// FULL: the scan itself.  Otherwise a piece's state from zero and its sum of dt.
template <typename T, int NS, int P, bool FULL>
__global__ void __launch_bounds__(kThreads) scan_fwd(Scan<T> p) {
  using W = Place<NS, P>;
  constexpr int NP = W::NP, CW = W::CW, E = W::E;
  __shared__ __align__(16) float sB[2][kTile][NP];
  __shared__ __align__(16) float sC[FULL ? 2 : 1][FULL ? kTile : 1][NP];
  const int64_t tile = blockIdx.x % p.tiles, item = blockIdx.x / p.tiles;
  const W w = place<NS, P>(p, tile);
  const Item it = item_at(p, item);
  if (it.none) return;
  const int64_t n0 = w.p * NS;
  if (FULL && tile == 0 && it.c == 0) {
    if (threadIdx.x == 0 && it.bad) atomicOr(p.err, mk::ERRBIT_SEQS);
    check_distinct(p.slots, it.s, threadIdx.x, kThreads, p.err);
  }
  const int64_t row = p.init || p.last ? slot_of(p.slots, p.nslots, it.s, p.err) : -1;

  float A2[NS], h[NS];
  load_states<NS>(A2, p.A + w.d * p.N, n0, p.N);
#pragma unroll
  for (int j = 0; j < NS; ++j) A2[j] *= kLog2e, h[j] = 0.0f;
  // Pieces: entry 0 of a sequence's workspace is its initial state (read from
  // there by every piece, because `last` may replace it), entry c + 1 the
  // state that piece c leaves when it starts from zero.
  const int64_t entry = (item * p.D + w.d) * p.N;
  if (!FULL || !p.piece) {
    if (it.c == 0 && p.init && row >= 0) {
      load_states<NS>(h, p.init + (row * p.D + w.d) * p.N, n0, p.N);
      if (!FULL && w.live) store_states<NS>(p.wstate + entry, h, n0, p.N);
#pragma unroll
      for (int j = 0; j < NS; ++j) h[j] = FULL ? h[j] : 0.0f;
    } else if (!FULL && it.c == 0 && w.live) {
      store_states<NS>(p.wstate + entry, h, n0, p.N);
    }
    if (!FULL && it.t1 >= it.hi) return;
  } else {
    const float* ws = p.wstate + (it.first * p.D + w.d) * p.N;
    const float* wd = p.wsum + it.first * p.D + w.d;
    load_states<NS>(h, ws, n0, p.N);
    for (int64_t k = 0; k < it.c; ++k) {
      float add[NS];
      load_states<NS>(add, ws + (k + 1) * p.D * p.N, n0, p.N);
      const float sum = wd[k * p.D];
#pragma unroll
      for (int j = 0; j < NS; ++j) h[j] = fmaf(ex2(A2[j] * sum), h[j], add[j]);
    }
  }
  const float bias = p.bias ? p.bias[w.d] : 0.0f, skip = FULL && p.Dskip ? p.Dskip[w.d] : 0.0f;
  float sum_dt = 0.0f;

  Raw<T, E> cur, nxt;
  auto load_raw = [&](Raw<T, E>& r, int64_t t) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int64_t at = t + e * P + w.p;
      if (at < it.t1) {
        r.u[e] = p.u[at * p.ldu + w.d];
        r.delta[e] = p.delta[at * p.lddelta + w.d];
        if (FULL && p.z) r.z[e] = p.z[at * p.ldz + w.d];
      }
    }
  };
  float rB[kTile * NP / kThreads], rC[kTile * NP / kThreads];
  fetch<kTile, NP>(rB, p.B, p.ldb, w.g * p.N, p.N, it.t0, it.t1);
  put<kTile, NP>(&sB[0][0][0], rB);
  if constexpr (FULL) {
    fetch<kTile, NP>(rC, p.C, p.ldc, w.g * p.N, p.N, it.t0, it.t1);
    put<kTile, NP>(&sC[0][0][0], rC);
  }
  load_raw(cur, it.t0);
  int buf = 0;
  for (int64_t tt = it.t0; tt < it.t1; tt += kTile, buf ^= 1) {
    __syncthreads();
    const bool more = tt + kTile < it.t1;
    if (more) {
      fetch<kTile, NP>(rB, p.B, p.ldb, w.g * p.N, p.N, tt + kTile, it.t1);
      if constexpr (FULL) fetch<kTile, NP>(rC, p.C, p.ldc, w.g * p.N, p.N, tt + kTile, it.t1);
    }
    if (FULL && p.saved && (tt - it.lo) % kPiece == 0 && w.live)
      store_states<NS>(p.saved + ((first_piece(p.q, it.s, kPiece) + (tt - it.lo) / kPiece) * p.D + w.d) * p.N, h, n0,
                       p.N);
    for (int q = 0; q < kTile / kGroup; ++q) {
      const int64_t t = tt + q * kGroup;
      if (t >= it.t1) break;
      load_raw(nxt, t + kGroup);
      float dt[E], dtu[E], u[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        dt[e] = dtu[e] = u[e] = 0.0f;
        if (t + e * P + w.p < it.t1) {
          u[e] = to_f(cur.u[e]);
          const float x = to_f(cur.delta[e]) + bias;
          dt[e] = p.softplus ? softplus(x) : x;
          dtu[e] = dt[e] * u[e];
        }
        if (!FULL) sum_dt += dt[e];
      }
      float yk[kGroup];
#pragma unroll
      for (int k = 0; k < kGroup; ++k) {
        const int src = (k % P) * CW + w.c;
        const float a_dt = P > 1 ? __shfl_sync(0xffffffffu, dt[k / P], src) : dt[k / P];
        const float a_dtu = P > 1 ? __shfl_sync(0xffffffffu, dtu[k / P], src) : dtu[k / P];
        float b[NS];
        row_of<NS>(b, &sB[buf][q * kGroup + k][n0]);
#pragma unroll
        for (int j = 0; j < NS; ++j) h[j] = fmaf(ex2(a_dt * A2[j]), h[j], a_dtu * b[j]);
        if constexpr (FULL) {
          row_of<NS>(b, &sC[buf][q * kGroup + k][n0]);
          float acc = 0.0f;
#pragma unroll
          for (int j = 0; j < NS; ++j) acc = fmaf(b[j], h[j], acc);
          yk[k] = acc;
        }
      }
      if constexpr (FULL) {
        float y[E];
        reduce_scatter8<P, CW>(yk, w.p, y);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t at = t + e * P + w.p;
          if (at < it.t1 && w.live) {
            float v = fmaf(skip, u[e], y[e]);
            if (p.z) {
              const float z = to_f(cur.z[e]);
              v *= z * sigmoid(z);
            }
            p.y[at * p.ldy + w.d] = from_f<T>(v);
          }
        }
      }
      cur = nxt;
    }
    if (more) {
      put<kTile, NP>(&sB[buf ^ 1][0][0], rB);
      if constexpr (FULL) put<kTile, NP>(&sC[buf ^ 1][0][0], rC);
    }
  }
  if constexpr (FULL) {
    if (p.last && row >= 0 && w.live && it.t1 >= it.hi)
      store_states<NS>(p.last + (row * p.D + w.d) * p.N, h, n0, p.N);
  } else {
#pragma unroll
    for (int bit = CW; bit < 32; bit *= 2) sum_dt += __shfl_xor_sync(0xffffffffu, sum_dt, bit);
    if (w.live) {
      store_states<NS>(p.wstate + entry + p.D * p.N, h, n0, p.N);
      if (w.p == 0) p.wsum[item * p.D + w.d] = sum_dt;
    }
  }
}

// Backward over pieces, first launch: what a piece hands to the token before
// it (e = a g of its first token) when nothing comes from behind, and its sum
// of dt.  The first piece of a sequence hands on nothing.
template <typename T, int NS, int P>
__global__ void __launch_bounds__(kThreads) scan_rev(Scan<T> p) {
  using W = Place<NS, P>;
  constexpr int NP = W::NP, CW = W::CW, E = W::E;
  __shared__ __align__(16) float sC[kTile][NP];
  const int64_t tile = blockIdx.x % p.tiles, item = blockIdx.x / p.tiles;
  const W w = place<NS, P>(p, tile);
  const Item it = item_at(p, item);
  if (it.none || it.c == 0) return;
  const int64_t n0 = w.p * NS;
  float A2[NS], e_[NS];
  load_states<NS>(A2, p.A + w.d * p.N, n0, p.N);
#pragma unroll
  for (int j = 0; j < NS; ++j) A2[j] *= kLog2e, e_[j] = 0.0f;
  const float bias = p.bias ? p.bias[w.d] : 0.0f;
  float sum_dt = 0.0f;
  const int64_t ntile = (it.t1 - it.t0 + kTile - 1) / kTile;
  for (int64_t k = ntile - 1; k >= 0; --k) {
    const int64_t tt = it.t0 + k * kTile;
    float rC[kTile * NP / kThreads];
    fetch<kTile, NP>(rC, p.C, p.ldc, w.g * p.N, p.N, tt, it.t1);
    __syncthreads();
    put<kTile, NP>(&sC[0][0], rC);
    __syncthreads();
    for (int q = kTile / kGroup - 1; q >= 0; --q) {
      const int64_t t = tt + q * kGroup;
      if (t >= it.t1) continue;
      float dt[E], dyp[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int64_t at = t + e * P + w.p;
        dt[e] = dyp[e] = 0.0f;
        if (at < it.t1) {
          const float x = to_f(p.delta[at * p.lddelta + w.d]) + bias;
          dt[e] = p.softplus ? softplus(x) : x;
          dyp[e] = to_f(p.dy[at * p.lddy + w.d]);
          if (p.z) {
            const float z = to_f(p.z[at * p.ldz + w.d]);
            dyp[e] *= z * sigmoid(z);
          }
        }
        sum_dt += dt[e];
      }
#pragma unroll
      for (int i = kGroup - 1; i >= 0; --i) {
        const int src = (i % P) * CW + w.c;
        const float a_dt = P > 1 ? __shfl_sync(0xffffffffu, dt[i / P], src) : dt[i / P];
        const float a_dy = P > 1 ? __shfl_sync(0xffffffffu, dyp[i / P], src) : dyp[i / P];
        float c[NS];
        row_of<NS>(c, &sC[q * kGroup + i][n0]);
#pragma unroll
        for (int j = 0; j < NS; ++j) e_[j] = ex2(a_dt * A2[j]) * fmaf(c[j], a_dy, e_[j]);
      }
    }
  }
#pragma unroll
  for (int bit = CW; bit < 32; bit *= 2) sum_dt += __shfl_xor_sync(0xffffffffu, sum_dt, bit);
  if (w.live) {
    store_states<NS>(p.wstate + (item * p.D + w.d) * p.N, e_, n0, p.N);
    if (w.p == 0) p.wsum[item * p.D + w.d] = sum_dt;
  }
}

// Backward.  With g[t] = C[t] dyp[t] + e[t+1], e[t] = a[t] g[t] (e behind the
// last token: dlast) and q = a[t] h[t-1]:
//   dB += g dt u, dC += dyp h (summed over the channels of the group),
//   dA += g q dt, ddt = sum_n g (q A + B u), du = dt sum_n g B + D dyp.
// A block takes kPiece tokens at a time from the end.  Their states are
// rebuilt from the saved state in front of them: one pass keeps the state at
// every eighth token in shared memory, then each group of 8 tokens, last
// first, is run again with its a and h in registers and walked backwards.  dB
// and dC are reduced over a warp's channels by shuffles, over the block's
// warps in shared memory, and over blocks by scan_fold in a fixed order.
template <int NS, int P>
struct BwdSmem {
  static constexpr int NP = NS * P;
  float B[kPiece][NP], C[kPiece][NP];
  float4 sub[kPiece / kGroup][NS / 4][kThreads];
  float red[2][2][kWarps][kGroup][NP];
};

template <typename T, int NS, int P>
__global__ void __launch_bounds__(kThreads) scan_bwd(Scan<T> p) {
  using W = Place<NS, P>;
  constexpr int NP = W::NP, CW = W::CW, E = W::E;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  BwdSmem<NS, P>& sm = *reinterpret_cast<BwdSmem<NS, P>*>(smem_raw);
  const int64_t tile = blockIdx.x % p.tiles, item0 = blockIdx.x / p.tiles;
  const W w = place<NS, P>(p, tile);
  const int64_t n0 = w.p * NS;
  float A[NS], dA[NS];
  load_states<NS>(A, p.A + w.d * p.N, n0, p.N);
#pragma unroll
  for (int j = 0; j < NS; ++j) dA[j] = 0.0f;
  const float bias = p.bias ? p.bias[w.d] : 0.0f, skip = p.Dskip ? p.Dskip[w.d] : 0.0f;
  float dskip = 0.0f, dbias = 0.0f;
  int rb = 0;
  const int64_t GN = p.G * p.N;

  for (int64_t item = item0; item < p.items; item += p.grid_items) {
    const Item it = item_at(p, item);
    if (it.none) continue;
    if (tile == 0 && it.c == 0 && threadIdx.x == 0 && it.bad) atomicOr(p.err, mk::ERRBIT_SEQS);
    float e_[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) e_[j] = 0.0f;
    if (p.dlast) load_states<NS>(e_, p.dlast + (it.s * p.D + w.d) * p.N, n0, p.N);
    if (p.piece) {
      for (int64_t k = (it.hi - it.lo + p.piece - 1) / p.piece - 1; k > it.c; --k) {
        float add[NS];
        load_states<NS>(add, p.wstate + ((it.first + k) * p.D + w.d) * p.N, n0, p.N);
        const float sum = p.wsum[(it.first + k) * p.D + w.d];
#pragma unroll
        for (int j = 0; j < NS; ++j) e_[j] = fmaf(ex2(A[j] * kLog2e * sum), e_[j], add[j]);
      }
    }
    const int64_t chunks = (it.t1 - it.t0 + kPiece - 1) / kPiece;
    for (int64_t ch = chunks - 1; ch >= 0; --ch) {
      const int64_t tc = it.t0 + ch * kPiece, te = min(it.t1, tc + kPiece);
      const int nsub = (int)((te - tc + kGroup - 1) / kGroup);
      __syncthreads();  // the tile's readers are done
      {
        float r[kPiece * NP / kThreads];
        fetch<kPiece, NP>(r, p.B, p.ldb, w.g * p.N, p.N, tc, te);
        put<kPiece, NP>(&sm.B[0][0], r);
        fetch<kPiece, NP>(r, p.C, p.ldc, w.g * p.N, p.N, tc, te);
        put<kPiece, NP>(&sm.C[0][0], r);
      }
      float h[NS];
      load_states<NS>(h, p.saved + ((first_piece(p.q, it.s, kPiece) + (tc - it.lo) / kPiece) * p.D + w.d) * p.N, n0,
                      p.N);
      __syncthreads();
      for (int q = 0; q < nsub - 1; ++q) {
#pragma unroll
        for (int j = 0; j < NS; j += 4)
          sm.sub[q][j / 4][threadIdx.x] = make_float4(h[j], h[j + 1], h[j + 2], h[j + 3]);
        const int64_t t = tc + q * kGroup;  // a group before the last is full
        float dt[E], dtu[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t at = t + e * P + w.p;
          const float x = to_f(p.delta[at * p.lddelta + w.d]) + bias;
          dt[e] = p.softplus ? softplus(x) : x;
          dtu[e] = dt[e] * to_f(p.u[at * p.ldu + w.d]);
        }
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
          const int src = (k % P) * CW + w.c;
          const float a_dt = P > 1 ? __shfl_sync(0xffffffffu, dt[k / P], src) : dt[k / P];
          const float a_dtu = P > 1 ? __shfl_sync(0xffffffffu, dtu[k / P], src) : dtu[k / P];
          float b[NS];
          row_of<NS>(b, &sm.B[q * kGroup + k][n0]);
#pragma unroll
          for (int j = 0; j < NS; ++j) h[j] = fmaf(ex2(a_dt * (A[j] * kLog2e)), h[j], a_dtu * b[j]);
        }
      }
      for (int q = nsub - 1; q >= 0; --q) {
        if (q != nsub - 1) {
#pragma unroll
          for (int j = 0; j < NS; j += 4) {
            const float4 v = sm.sub[q][j / 4][threadIdx.x];
            h[j] = v.x, h[j + 1] = v.y, h[j + 2] = v.z, h[j + 3] = v.w;
          }
        }
        const int64_t t = tc + q * kGroup;
        float dt[E], u[E], dyp[E], dy[E], z[E], sig[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t at = t + e * P + w.p;
          dt[e] = u[e] = dyp[e] = dy[e] = z[e] = sig[e] = 0.0f;
          if (at < te && w.live) {
            u[e] = to_f(p.u[at * p.ldu + w.d]);
            const float x = to_f(p.delta[at * p.lddelta + w.d]) + bias;
            dt[e] = p.softplus ? softplus(x) : x;
            sig[e] = p.softplus ? sigmoid(x) : 1.0f;
            dy[e] = dyp[e] = to_f(p.dy[at * p.lddy + w.d]);
            if (p.z) {
              z[e] = to_f(p.z[at * p.ldz + w.d]);
              dyp[e] *= z[e] * sigmoid(z[e]);
            }
          }
        }
        float a[kGroup][NS], hh[kGroup][NS], yk[kGroup], sG[kGroup], sT[kGroup];
#pragma unroll
        for (int k = 0; k < kGroup; ++k) {
          const int src = (k % P) * CW + w.c;
          const float a_dt = P > 1 ? __shfl_sync(0xffffffffu, dt[k / P], src) : dt[k / P];
          const float a_u = P > 1 ? __shfl_sync(0xffffffffu, u[k / P], src) : u[k / P];
          float b[NS], c[NS];
          row_of<NS>(b, &sm.B[q * kGroup + k][n0]);
          row_of<NS>(c, &sm.C[q * kGroup + k][n0]);
          yk[k] = 0.0f;
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            a[k][j] = ex2(a_dt * (A[j] * kLog2e));
            hh[k][j] = fmaf(a[k][j], k ? hh[k ? k - 1 : 0][j] : h[j], a_dt * a_u * b[j]);
            yk[k] = fmaf(c[j], hh[k][j], yk[k]);
          }
        }
        float vB[NS][kGroup], vC[NS][kGroup];
#pragma unroll
        for (int k = kGroup - 1; k >= 0; --k) {
          const int src = (k % P) * CW + w.c;
          const float a_dt = P > 1 ? __shfl_sync(0xffffffffu, dt[k / P], src) : dt[k / P];
          const float a_u = P > 1 ? __shfl_sync(0xffffffffu, u[k / P], src) : u[k / P];
          const float a_dy = P > 1 ? __shfl_sync(0xffffffffu, dyp[k / P], src) : dyp[k / P];
          float b[NS], c[NS];
          row_of<NS>(b, &sm.B[q * kGroup + k][n0]);
          row_of<NS>(c, &sm.C[q * kGroup + k][n0]);
          sG[k] = sT[k] = 0.0f;
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            const float g = fmaf(c[j], a_dy, e_[j]);
            const float gq = g * (a[k][j] * (k ? hh[k ? k - 1 : 0][j] : h[j]));
            vC[j][k] = a_dy * hh[k][j];
            vB[j][k] = g * (a_dt * a_u);
            dA[j] = fmaf(gq, a_dt, dA[j]);
            sT[k] = fmaf(gq, A[j], sT[k]);
            sG[k] = fmaf(g, b[j], sG[k]);
            e_[j] = a[k][j] * g;
          }
        }
        // dB and dC of the group: over the warp's channels, then the warps
        constexpr int EC = CW < 8 ? 8 / CW : 1;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          float oB[EC], oC[EC];
          reduce_scatter8<CW, 1>(vB[j], w.c, oB);
          reduce_scatter8<CW, 1>(vC[j], w.c, oC);
          if (w.c < 8) {
#pragma unroll
            for (int e = 0; e < EC; ++e) {
              sm.red[rb][0][w.warp][e * CW + w.c][n0 + j] = oB[e];
              sm.red[rb][1][w.warp][e * CW + w.c][n0 + j] = oC[e];
            }
          }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * kGroup * NP; i += kThreads) {
          const int which = i / (kGroup * NP), k = i / NP % kGroup, n = i % NP;
          float v = 0.0f;
#pragma unroll
          for (int x = 0; x < kWarps; ++x) v += sm.red[rb][which][x][k][n];
          if (t + k < te && n < p.N)
            p.parts[((which * p.tpg + w.tg) * p.q.T + t + k) * GN + w.g * p.N + n] = v;
        }
        rb ^= 1;
        float y[E], rG[E], rT[E];
        reduce_scatter8<P, CW>(yk, w.p, y);
        reduce_scatter8<P, CW>(sG, w.p, rG);
        reduce_scatter8<P, CW>(sT, w.p, rT);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t at = t + e * P + w.p;
          if (at < te && w.live) {
            if (p.z) {
              const float sz = sigmoid(z[e]);
              const float yv = fmaf(skip, u[e], y[e]);
              p.dz[at * p.lddz + w.d] = from_f<T>(dy[e] * yv * (sz * fmaf(z[e], 1.0f - sz, 1.0f)));
            }
            p.du[at * p.lddu + w.d] = from_f<T>(fmaf(dt[e], rG[e], skip * dyp[e]));
            const float dr = fmaf(u[e], rG[e], rT[e]) * sig[e];
            p.ddelta[at * p.ldddelta + w.d] = from_f<T>(dr);
            dbias += dr;
            dskip = fmaf(dyp[e], u[e], dskip);
          }
        }
      }
    }
    if (p.dinit && it.c == 0 && w.live) store_states<NS>(p.dinit + (it.s * p.D + w.d) * p.N, e_, n0, p.N);
  }
#pragma unroll
  for (int bit = CW; bit < 32; bit *= 2) {
    dskip += __shfl_xor_sync(0xffffffffu, dskip, bit);
    dbias += __shfl_xor_sync(0xffffffffu, dbias, bit);
  }
  if (w.live) {
    store_states<NS>(p.partA + (item0 * p.D + w.d) * p.N, dA, n0, p.N);
    if (w.p == 0) {
      p.partD[(item0 * 2) * p.D + w.d] = dskip;
      p.partD[(item0 * 2 + 1) * p.D + w.d] = dbias;
    }
  }
}

// The sums over blocks: dB and dC over channel tiles (rounded once), dA, dD
// and dbias over the blocks of a channel.
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

// One token per batch entry.  Bound by the state: read and written once, 16
// bytes per lane, P lanes per channel in memory order.
template <typename T>
struct Step {
  int64_t D, N, G, Dg, B, nslots, dblocks;
  const T *u, *delta, *z, *Bm, *Cm;
  int64_t ldu, lddelta, ldz, ldb, ldc, ldy;
  const float *A, *Dskip, *bias, *state;
  float* next;
  T* y;
  const int32_t* slots;
  int softplus;
  unsigned* err;
};

template <typename T, int P>
__global__ void __launch_bounds__(128) scan_step(Step<T> p) {
  const int64_t e = blockIdx.x / p.dblocks, block = blockIdx.x % p.dblocks;
  if (block == 0) check_distinct(p.slots, e, threadIdx.x, 128, p.err);
  const int64_t row = slot_of(p.slots, p.nslots, e, p.err);
  if (row < 0) return;
  const int64_t dc = block * (128 / P) + threadIdx.x / P, n0 = threadIdx.x % P * 4;
  const bool live = dc < p.D;
  const int64_t d = live ? dc : 0, g = d / p.Dg, at = (row * p.D + d) * p.N;
  float h[4], A[4], b[4], c[4];
  load_states<4>(h, p.state + at, n0, p.N);
  load_states<4>(A, p.A + d * p.N, n0, p.N);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[j] = n0 + j < p.N ? to_f(p.Bm[e * p.ldb + g * p.N + n0 + j]) : 0.0f;
    c[j] = n0 + j < p.N ? to_f(p.Cm[e * p.ldc + g * p.N + n0 + j]) : 0.0f;
  }
  const float u = to_f(p.u[e * p.ldu + d]);
  const float x = to_f(p.delta[e * p.lddelta + d]) + (p.bias ? p.bias[d] : 0.0f);
  const float dt = p.softplus ? softplus(x) : x;
  float y = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = fmaf(ex2(dt * (A[j] * kLog2e)), h[j], dt * u * b[j]);
    y = fmaf(c[j], h[j], y);
  }
#pragma unroll
  for (int bit = 1; bit < P; bit *= 2) y += __shfl_xor_sync(0xffffffffu, y, bit);
  if (!live) return;
  store_states<4>(p.next + at, h, n0, p.N);
  if (n0 == 0) {
    y = fmaf(p.Dskip ? p.Dskip[d] : 0.0f, u, y);
    if (p.z) {
      const float z = to_f(p.z[e * p.ldz + d]);
      y *= z * sigmoid(z);
    }
    p.y[e * p.ldy + d] = from_f<T>(y);
  }
}

// ---- host side ----------------------------------------------------------------

int check_sizes(const char* who, int type, int64_t D, int64_t N, int64_t G, int64_t T, int64_t nseq) {
  if (type < MK_T_F32 || type > MK_T_BF16) return bad(who, "unknown element type");
  if (D < 1 || T < 0 || nseq < 0) return bad(who, "negative size or no channels");
  if (N < 1 || N > 64) return bad(who, "1 to 64 states, got " + std::to_string(N));
  if (G < 1 || D % G) return bad(who, "the groups do not divide the channels");
  if (D > (1ll << 20) || T > INT32_MAX || nseq > (1ll << 24))
    return bad(who, "more than 2^20 channels, 2^24 sequences or 2^31 - 1 tokens");
  return MK_OK;
}

int check_scan(const char* who, const mk_scan_args* a, bool grad) {
  if (!a) return bad(who, "null arguments");
  MK_TRY(check_sizes(who, a->type, a->D, a->N, a->G, a->T, a->nseq));
  if (a->len < 0 || (!a->seqs && a->nseq * a->len != a->T)) return bad(who, "nseq * len is not T");
  const size_t es = type_bytes(a->type);
  const bool vec = a->N % 4 == 0;
  MK_TRY(check_matrix(who, "u", a->u, a->D, a->ldu, a->T, es));
  MK_TRY(check_matrix(who, "delta", a->delta, a->D, a->lddelta, a->T, es));
  if (a->z) MK_TRY(check_matrix(who, "z", a->z, a->D, a->ldz, a->T, es));
  MK_TRY(check_matrix(who, "B", a->B, a->G * a->N, a->ldb, a->T, es));
  MK_TRY(check_matrix(who, "C", a->C, a->G * a->N, a->ldc, a->T, es));
  MK_TRY(check_floats(who, "A", a->A, true, vec));
  MK_TRY(check_floats(who, "Dskip", a->Dskip, false, false));
  MK_TRY(check_floats(who, "bias", a->bias, false, false));
  MK_TRY(check_floats(who, "init", a->init, false, vec));
  MK_TRY(check_floats(who, "saved", a->saved, grad && a->T > 0, vec));
  if (a->slots && a->nslots < 0) return bad(who, "negative number of slots");
  if (!grad) {
    MK_TRY(check_matrix(who, "y", a->y, a->D, a->ldy, a->T, es));
    return check_floats(who, "last", a->last, false, vec);
  }
  if (a->slots) return bad(who, "states are per sequence, slots are for serving");
  MK_TRY(check_matrix(who, "dy", a->dy, a->D, a->lddy, a->T, es));
  MK_TRY(check_matrix(who, "du", a->du, a->D, a->lddu, a->T, es));
  MK_TRY(check_matrix(who, "ddelta", a->ddelta, a->D, a->ldddelta, a->T, es));
  if (!a->z != !a->dz && a->T) return bad(who, "dz is needed exactly when z is given");
  if (a->z) MK_TRY(check_matrix(who, "dz", a->dz, a->D, a->lddz, a->T, es));
  MK_TRY(check_matrix(who, "dB", a->dB, a->G * a->N, a->lddb, a->T, es));
  MK_TRY(check_matrix(who, "dC", a->dC, a->G * a->N, a->lddc, a->T, es));
  MK_TRY(check_floats(who, "dA", a->dA, true, vec));
  if (!a->Dskip != !a->dDskip || !a->bias != !a->dbias)
    return bad(who, "dDskip and dbias are needed exactly when Dskip and bias are given");
  MK_TRY(check_floats(who, "dDskip", a->dDskip, false, false));
  MK_TRY(check_floats(who, "dbias", a->dbias, false, false));
  MK_TRY(check_floats(who, "dlast", a->dlast, false, vec));
  return check_floats(who, "dinit", a->dinit, false, vec);
}

// Lanes per channel: 4 states per lane up to N = 16, 8 beyond.
int lanes_of(int64_t N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 32 ? 4 : 8; }

struct Plan {
  int64_t tpg, tiles, items, piece, grid_items;
  size_t piece_bytes, part_bytes, bytes;
};

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Whole sequences while their warps give every scheduler about two; with fewer
// rows sequences are cut into pieces, as many as would fill the GPU that far.
// Cutting costs a second pass of exponentials, so it has to win more than 2x.
Plan plan(const mk_scan_args* a, const mk::Device* dev, bool grad) {
  Plan b{};
  const int64_t CB = kWarps * (32 / lanes_of(a->N)), Dg = a->D / a->G;
  b.tpg = mk::cdiv(Dg, CB);
  b.tiles = a->G * b.tpg;
  b.items = a->nseq;
  const int64_t want = (int64_t)dev->sms * 4, have = b.tiles * a->nseq;
  if (have > 0 && have * 3 <= want && a->T >= a->nseq * 4 * kPiece) {
    const int64_t pieces = want / b.tiles;  // over all sequences
    int64_t piece = mk::cdiv(mk::cdiv(a->T, pieces), kPiece) * kPiece;
    b.piece = piece < 2 * kPiece ? 2 * kPiece : piece;
    b.items = a->T / b.piece + a->nseq;
    b.piece_bytes = align256((size_t)b.items * a->D * a->N * 4) + align256((size_t)b.items * a->D * 4);
  }
  if (grad) {
    const int64_t blocks = (int64_t)dev->sms * 16;  // four times what is resident at once
    b.grid_items = mk::cdiv(blocks, b.tiles);
    if (b.grid_items > b.items) b.grid_items = b.items;
    b.part_bytes = align256((size_t)2 * b.tpg * a->T * a->G * a->N * 4) +
                   align256((size_t)b.grid_items * a->D * a->N * 4) + align256((size_t)b.grid_items * 2 * a->D * 4);
  }
  b.bytes = b.piece_bytes + b.part_bytes;
  return b;
}

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

template <typename T, int NS, int P>
int run_fwd(const mk_scan_args* a, const mk::Device* dev, const Plan& b, cudaStream_t s) {
  const Scan<T> p = params<T>(a, dev, b);
  const unsigned grid = (unsigned)(b.tiles * b.items);
  if (b.piece) scan_fwd<T, NS, P, false><<<grid, kThreads, 0, s>>>(p);
  scan_fwd<T, NS, P, true><<<grid, kThreads, 0, s>>>(p);
  return mk::check_launch("mk_selective_scan: launch");
}

template <typename T, int NS, int P>
int run_bwd(const mk_scan_args* a, const mk::Device* dev, const Plan& b, cudaStream_t s) {
  const Scan<T> p = params<T>(a, dev, b);
  constexpr size_t smem = sizeof(BwdSmem<NS, P>);
  MK_TRY(mk::allow_dynamic_smem(reinterpret_cast<const void*>(&scan_bwd<T, NS, P>), smem));
  if (b.piece) scan_rev<T, NS, P><<<(unsigned)(b.tiles * b.items), kThreads, 0, s>>>(p);
  if (b.grid_items) scan_bwd<T, NS, P><<<(unsigned)(b.tiles * b.grid_items), kThreads, smem, s>>>(p);
  const int64_t total = 2 * a->T * a->G * a->N + a->D * (a->N + 2);
  int64_t blocks = mk::cdiv(total, 256);
  if (blocks > (int64_t)dev->sms * 16) blocks = (int64_t)dev->sms * 16;
  scan_fold<T><<<(unsigned)blocks, 256, 0, s>>>(p, static_cast<T*>(a->dB), static_cast<T*>(a->dC), a->lddb, a->lddc,
                                                a->dA, a->dDskip, a->dbias);
  return mk::check_launch("mk_selective_scan_grad: launch");
}

template <typename T>
int run_type(const mk_scan_args* a, const mk::Device* dev, const Plan& b, bool grad, cudaStream_t s) {
  const int64_t N = a->N;
  if (N <= 4) return grad ? run_bwd<T, 4, 1>(a, dev, b, s) : run_fwd<T, 4, 1>(a, dev, b, s);
  if (N <= 8) return grad ? run_bwd<T, 4, 2>(a, dev, b, s) : run_fwd<T, 4, 2>(a, dev, b, s);
  if (N <= 16) return grad ? run_bwd<T, 4, 4>(a, dev, b, s) : run_fwd<T, 4, 4>(a, dev, b, s);
  if (N <= 32) return grad ? run_bwd<T, 8, 4>(a, dev, b, s) : run_fwd<T, 8, 4>(a, dev, b, s);
  return grad ? run_bwd<T, 8, 8>(a, dev, b, s) : run_fwd<T, 8, 8>(a, dev, b, s);
}

int run_scan(const char* who, const mk_scan_args* a, bool grad, void* stream) {
  MK_TRY(check_scan(who, a, grad));
  if (a->nseq == 0 && !grad) return MK_OK;
  MK_ENTRY_DEVICE(dev);
  const Plan b = plan(a, dev, grad);
  if (b.tiles * b.items > INT32_MAX) return bad(who, "too many sequences for these channels");
  if (b.bytes && (!a->workspace || a->workspace_bytes < b.bytes || !elem_aligned(a->workspace, 16)))
    return bad(who, "a 16-byte aligned workspace of " + std::to_string(b.bytes) + " bytes is needed");
  cudaStream_t s = mk::as_stream(stream);
  if (a->type == MK_T_F32) return run_type<float>(a, dev, b, grad, s);
  if (a->type == MK_T_F16) return run_type<__half>(a, dev, b, grad, s);
  return run_type<__nv_bfloat16>(a, dev, b, grad, s);
}

int workspace(const char* who, const mk_scan_args* a, bool grad, size_t* bytes) {
  if (!a || !bytes) return bad(who, "null arguments");
  MK_TRY(check_sizes(who, a->type, a->D, a->N, a->G, a->T, a->nseq));
  MK_ENTRY_DEVICE(dev);
  *bytes = plan(a, dev, grad).bytes;
  return MK_OK;
}

template <typename T>
int run_step(const mk_scan_step_args* a, const mk::Device* dev, cudaStream_t s) {
  Step<T> p{};
  const int P = a->N <= 4 ? 1 : a->N <= 8 ? 2 : a->N <= 16 ? 4 : a->N <= 32 ? 8 : 16;
  p.D = a->D, p.N = a->N, p.G = a->G, p.Dg = a->D / a->G, p.B = a->B, p.nslots = a->nslots;
  p.dblocks = mk::cdiv(a->D, 128 / P);
  p.u = static_cast<const T*>(a->u), p.ldu = a->ldu;
  p.delta = static_cast<const T*>(a->delta), p.lddelta = a->lddelta;
  p.z = static_cast<const T*>(a->z), p.ldz = a->ldz;
  p.Bm = static_cast<const T*>(a->Bmat), p.ldb = a->ldb;
  p.Cm = static_cast<const T*>(a->Cmat), p.ldc = a->ldc;
  p.y = static_cast<T*>(a->y), p.ldy = a->ldy;
  p.A = a->A, p.Dskip = a->Dskip, p.bias = a->bias, p.state = a->state, p.next = a->next;
  p.slots = a->slots, p.softplus = a->softplus, p.err = dev->err_word;
  const unsigned grid = (unsigned)(a->B * p.dblocks);
  switch (P) {
    case 1: scan_step<T, 1><<<grid, 128, 0, s>>>(p); break;
    case 2: scan_step<T, 2><<<grid, 128, 0, s>>>(p); break;
    case 4: scan_step<T, 4><<<grid, 128, 0, s>>>(p); break;
    case 8: scan_step<T, 8><<<grid, 128, 0, s>>>(p); break;
    default: scan_step<T, 16><<<grid, 128, 0, s>>>(p); break;
  }
  return mk::check_launch("mk_selective_scan_step: launch");
}

int step(const mk_scan_step_args* a, void* stream) {
  const char* who = "mk_selective_scan_step";
  if (!a) return bad(who, "null arguments");
  MK_TRY(check_sizes(who, a->type, a->D, a->N, a->G, a->B, 0));
  const size_t es = type_bytes(a->type);
  const bool vec = a->N % 4 == 0, some = a->B > 0;
  MK_TRY(check_matrix(who, "u", a->u, a->D, a->ldu, a->B, es));
  MK_TRY(check_matrix(who, "delta", a->delta, a->D, a->lddelta, a->B, es));
  if (a->z) MK_TRY(check_matrix(who, "z", a->z, a->D, a->ldz, a->B, es));
  MK_TRY(check_matrix(who, "B", a->Bmat, a->G * a->N, a->ldb, a->B, es));
  MK_TRY(check_matrix(who, "C", a->Cmat, a->G * a->N, a->ldc, a->B, es));
  MK_TRY(check_matrix(who, "y", a->y, a->D, a->ldy, a->B, es));
  MK_TRY(check_floats(who, "A", a->A, true, vec));
  MK_TRY(check_floats(who, "Dskip", a->Dskip, false, false));
  MK_TRY(check_floats(who, "bias", a->bias, false, false));
  MK_TRY(check_floats(who, "state", a->state, some, vec));
  MK_TRY(check_floats(who, "next", a->next, some, vec));
  if (a->slots && a->nslots < 0) return bad(who, "negative number of slots");
  if (!some) return MK_OK;
  if (a->B * mk::cdiv(a->D, 8) > INT32_MAX) return bad(who, "batch too large for these channels");
  MK_ENTRY_DEVICE(dev);
  cudaStream_t s = mk::as_stream(stream);
  if (a->type == MK_T_F32) return run_step<float>(a, dev, s);
  if (a->type == MK_T_F16) return run_step<__half>(a, dev, s);
  return run_step<__nv_bfloat16>(a, dev, s);
}

}  // namespace

extern "C" int mk_selective_scan_workspace(const mk_scan_args* a, size_t* bytes) {
  mk::clear_error();
  return guarded([&] { return workspace("mk_selective_scan_workspace", a, false, bytes); });
}

extern "C" int mk_selective_scan(const mk_scan_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return run_scan("mk_selective_scan", a, false, stream); });
}

extern "C" int mk_selective_scan_grad_workspace(const mk_scan_args* a, size_t* bytes) {
  mk::clear_error();
  return guarded([&] { return workspace("mk_selective_scan_grad_workspace", a, true, bytes); });
}

extern "C" int mk_selective_scan_grad(const mk_scan_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return run_scan("mk_selective_scan_grad", a, true, stream); });
}

extern "C" int mk_selective_scan_step(const mk_scan_step_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return step(a, stream); });
}
