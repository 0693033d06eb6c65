// block_norm.cu — the norms around a block, fused with the block's gate and
// its scaled residual: per token column of D channels
//     n = h / rms(h) * hw,  m = n * act(gate),  rout = r + scale * m,
//     y = rout / rms(rout) * w,   rms(x) = sqrt(mean(x^2) + eps).
//
// Bound by memory: every matrix is read or written once; a column stays in
// registers between its reductions, as it is in memory.  A column of up to 32 *
// V * ITEMS channels is one warp's (shuffles only), wider ones a block's.
// Products are taken in pairs (f32x2): at 8 or 16 values per thread the issue
// slots are as scarce as the bandwidth.  Backward recomputes the forward values
// from r, h and gate, which costs no more reads than saving rout and its rms
// would.
#include "tokens.cuh"

namespace {

using namespace mk::tok;

template <typename T, typename R>
struct Norm {
  int D;  // at most 16384
  int64_t T_;
  float eps, inv_d;
  int act;
  const R *r, *drout;
  R *rout, *dr;
  const T *h, *gate, *dy;
  T *y, *dh, *dgate;
  const float *hw, *scale, *w;
  int64_t ldr, ldh, ldgate, ldrout, ldy, lddy, lddrout, lddr, lddh, lddgate;
  float* parts;  // backward: [part][3][D] of w, hw, scale
};

// Sums of two values over the blockDim.x threads of a column.  A column is one
// warp's, or the whole block's: then every thread adds up the warps' sums, and
// as buffers take turns one barrier is enough.
template <int N>  // buffers: sums between two barriers that reuse one
struct alignas(16) Sums {
  float2 part[N][32];  // zeros where there is no warp
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < N * 32; i += blockDim.x * blockDim.y)
      part[i / 32][i % 32] = make_float2(0.0f, 0.0f);
    __syncthreads();
  }
};
template <int N>
__device__ __forceinline__ float2 column_sum(float2 v, Sums<N>& sm, int& turn) {
  // each half of the warp adds up one of the two
  const bool up = (threadIdx.x & 16) != 0;
  float one = up ? v.y : v.x;
  one += __shfl_xor_sync(0xffffffffu, up ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
  if (blockDim.x == 32) {
    const float other = __shfl_xor_sync(0xffffffffu, one, 16);
    return up ? make_float2(other, one) : make_float2(one, other);
  }
  if ((threadIdx.x & 15) == 0) (&sm.part[turn][threadIdx.x >> 5].x)[up] = one;
  __syncthreads();
  const ulonglong2* part = reinterpret_cast<const ulonglong2*>(sm.part[turn]);
  F2 a = pack(0.0f), b = pack(0.0f);
  for (int i = 0; i < (int)(blockDim.x + 63) / 64; ++i) {  // two warps at a time
    const ulonglong2 q = part[i];
    a = add2(a, F2{q.x}), b = add2(b, F2{q.y});
  }
  a = add2(a, b);
  unpack(a, v.x, v.y);
  if (++turn == N) turn = 0;
  return v;
}

// The gate's sigmoid s, and act(g) = s g (silu) or s.
template <bool EXACT>
__device__ __forceinline__ F2 sigmoid2(F2 g) {
  float a, b;
  unpack(g, a, b);
  return pack(sigmoid<EXACT>(a), sigmoid<EXACT>(b));
}
// act' = act (1 - s), and s more for silu
__device__ __forceinline__ F2 act_grad(F2 a, F2 s, bool silu) {
  const F2 left = fma2(s, pack(-1.0f), pack(1.0f));
  return silu ? fma2(a, left, s) : mul2(a, left);
}

// A vector of V elements by loads of 16 bytes.
template <typename X, int V>
__device__ __forceinline__ void load_vec(Vec<X, V>& r, const X* p, bool on) {
  constexpr int C = sizeof(X) * V <= 16 ? V : 16 / (int)sizeof(X);
#pragma unroll
  for (int i = 0; i < V; i += C)
    load_if(reinterpret_cast<Vec<X, C>&>(r.v[i]), reinterpret_cast<const Vec<X, C>*>(p + i), on);
}

// What a thread reads of one column, as it is in memory.  GRAD: dy and drout too.
template <typename T, typename R, int V, int ITEMS, bool GRAD>
struct Column {
  Vec<R, V> r[ITEMS], dro[GRAD ? ITEMS : 1];
  Vec<T, V> h[ITEMS], g[ITEMS], dy[GRAD ? ITEMS : 1];

  // Column t; zeros for what is not there.
  __device__ __forceinline__ void fetch(const Norm<T, R>& p, int64_t t) {
    const R* pr = p.r + t * p.ldr;
    const T *ph = p.h + t * p.ldh, *pg = p.gate + t * p.ldgate;
    const T* pdy = GRAD ? p.dy + t * p.lddy : nullptr;
    const R* pdro = GRAD ? p.drout + t * p.lddrout : nullptr;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        r[k].v[i] = from_f<R>(0.0f), h[k].v[i] = g[k].v[i] = from_f<T>(0.0f);
        if constexpr (GRAD) dro[k].v[i] = from_f<R>(0.0f), dy[k].v[i] = from_f<T>(0.0f);
      }
    }
    // one matrix after the other: whether it is there is asked once, not per vector
    auto all = [&](auto& to, const auto* from, bool there) {
      if (!there) return;
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const int d = (k * (int)blockDim.x + (int)threadIdx.x) * V;
        load_vec(to[k], from + d, d < p.D);
      }
    };
    if (t >= p.T_) return;
    all(h, ph, p.h), all(r, pr, true), all(g, pg, p.gate);
    if constexpr (GRAD) all(dy, pdy, p.dy), all(dro, pdro, p.drout);
  }
  __device__ __forceinline__ float sum_hh() const;
};

// Values 2 j and 2 j + 1 of a thread's vectors, and back.
template <typename X, int V, int ITEMS>
__device__ __forceinline__ F2 pair_at(const Vec<X, V> (&r)[ITEMS], int j) {
  return pack(to_f(r[2 * j / V].v[2 * j % V]), to_f(r[(2 * j + 1) / V].v[(2 * j + 1) % V]));
}
template <typename X, int V, int ITEMS>
__device__ __forceinline__ void put_pair(Vec<X, V> (&r)[ITEMS], int j, F2 x) {
  if constexpr (V > 1) {
    from_f2(&r[2 * j / V].v[2 * j % V], x);
  } else {
    float a, b;
    unpack(x, a, b);
    r[2 * j].v[0] = from_f<X>(a), r[2 * j + 1].v[0] = from_f<X>(b);
  }
}
template <typename X, int V, int ITEMS>
__device__ __forceinline__ void store_column(X* column, int D, const Vec<X, V> (&r)[ITEMS]) {
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int d = (k * (int)blockDim.x + (int)threadIdx.x) * V;
    if (d < D) *reinterpret_cast<Vec<X, V>*>(column + d) = r[k];
  }
}

template <typename T, typename R, int V, int ITEMS, bool GRAD>
__device__ __forceinline__ float Column<T, R, V, ITEMS, GRAD>::sum_hh() const {
  F2 s = pack(0.0f);
#pragma unroll
  for (int j = 0; j < V * ITEMS / 2; ++j) {
    const F2 x = pair_at(h, j);
    s = fma2(x, x, s);
  }
  return sum2(s);
}

// A thread's values of a parameter, ones without it.
template <int V, int ITEMS>
__device__ __forceinline__ void param(F2 (&f)[V * ITEMS / 2], const float* p, int D) {
  Vec<float, V> r[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int d = (k * (int)blockDim.x + (int)threadIdx.x) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) r[k].v[i] = 1.0f;
    load_vec<float, V>(r[k], p + d, p && d < D);
  }
#pragma unroll
  for (int j = 0; j < V * ITEMS / 2; ++j) f[j] = pair_at(r, j);
}

template <typename T, typename R, int V, int ITEMS, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) norm_fwd(Norm<T, R> p) {
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int H = V * ITEMS / 2;
  __shared__ Sums<2> sm;
  int turn = 0;
  const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  Column<T, R, V, ITEMS, false> cur;
  cur.fetch(p, t);
  sm.clear();
  if (t >= p.T_) return;
  float i1 = 1.0f;
  if (p.h && p.hw) i1 = rsqrtf(fmaf(column_sum(make_float2(cur.sum_hh(), 0.0f), sm, turn).x, p.inv_d, p.eps));
  const bool silu = p.act == MK_ACT_SILU;
  F2 x[H], sum = pack(0.0f);
  const F2 i1_2 = pack(i1);
  F2 par[H];
  param<V, ITEMS>(par, p.hw, p.D);
#pragma unroll
  for (int j = 0; j < H; ++j) x[j] = mul2(mul2(pair_at(cur.h, j), i1_2), par[j]);  // zeros without h
  if (p.gate) {
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const F2 g = pair_at(cur.g, j);
      x[j] = mul2(x[j], sigmoid2<kExact>(g));
      if (silu) x[j] = mul2(x[j], g);
    }
  }
  param<V, ITEMS>(par, p.scale, p.D);
#pragma unroll
  for (int j = 0; j < H; ++j) {
    x[j] = fma2(par[j], x[j], pair_at(cur.r, j));
    sum = fma2(x[j], x[j], sum);  // channels beyond D are zeros
  }
  if (p.rout) {
    Vec<R, V> out[ITEMS];
#pragma unroll
    for (int j = 0; j < H; ++j) put_pair(out, j, x[j]);
    store_column(p.rout + t * p.ldrout, p.D, out);
  }
  if (p.y) {
    param<V, ITEMS>(par, p.w, p.D);
    const float2 s = column_sum(make_float2(sum2(sum), 0.0f), sm, turn);
    const F2 i2 = pack(rsqrtf(fmaf(s.x, p.inv_d, p.eps)));
    Vec<T, V> out[ITEMS];
#pragma unroll
    for (int j = 0; j < H; ++j) put_pair(out, j, mul2(par[j], mul2(x[j], i2)));
    store_column(p.y + t * p.ldy, p.D, out);
  }
}

// Backward.  With x = rout i2 and dx = dy w:
//   dro = drout + i2 (dx - x mean(dx x)),  dr = dro,
//   dm = dro scale, dn = dm act, dgate = dm n act', dv = dn hw,
//   dh = i1 (dv - v mean(dv v)), v = h i1;
// dw += dy x, dhw += dn v, dscale += dro m.  A block walks columns and keeps its
// sums for w, hw and scale in shared memory, every thread its own channels'
// (in registers they would leave one block to an SM, and two overlap each
// other's waits); they go to one part per column walker, added up by norm_fold
// in a fixed order.  1027 columns of 1999 channels (f16, single elements): 26 us
// and 4 us for norm_fold; bound by the waits
// on its loads and the three reductions of a column (issue slots 48% used).
template <typename T, typename R, int V, int ITEMS, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) norm_bwd(Norm<T, R> p) {
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int H = V * ITEMS / 2;
  extern __shared__ float2 acc_smem[];  // [column walker][3][pair of values][thread]
  __shared__ Sums<3> sm;
  int turn = 0;
  sm.clear();
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  const int64_t walker = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  float2* acc = acc_smem + threadIdx.y * 3 * H * blockDim.x + threadIdx.x;
  for (int i = 0; i < 3 * H; ++i) acc[i * blockDim.x] = make_float2(0.0f, 0.0f);
  auto add = [&](int which, int j, F2 a, F2 b) {  // a b more
    unsigned long long* at = reinterpret_cast<unsigned long long*>(acc + (which * H + j) * blockDim.x);
    *at = fma2(a, b, F2{*at}).v;
  };
  const bool silu = p.gate && p.act == MK_ACT_SILU;
  for (int64_t t = walker; t < p.T_; t += stride) {
    Column<T, R, V, ITEMS, true> cur;
    cur.fetch(p, t);
    float i1 = 1.0f;
    if (p.h && p.hw) i1 = rsqrtf(fmaf(column_sum(make_float2(cur.sum_hh(), 0.0f), sm, turn).x, p.inv_d, p.eps));
    const F2 i1_2 = pack(i1);
    F2 x[H], sig[H];  // sig: of the gate, ones without
    F2 sxx = pack(0.0f), sdx = pack(0.0f);
    F2 hw[H], sc[H], w[H];
    param<V, ITEMS>(hw, p.hw, p.D), param<V, ITEMS>(sc, p.scale, p.D), param<V, ITEMS>(w, p.w, p.D);
#pragma unroll
    for (int j = 0; j < H; ++j) {  // without h its values are zeros, without dy those
      sig[j] = p.gate ? sigmoid2<kExact>(pair_at(cur.g, j)) : pack(1.0f);
      F2 m = mul2(mul2(mul2(pair_at(cur.h, j), i1_2), hw[j]), sig[j]);
      if (silu) m = mul2(m, pair_at(cur.g, j));
      x[j] = fma2(sc[j], m, pair_at(cur.r, j));
      sxx = fma2(x[j], x[j], sxx);
      sdx = fma2(mul2(pair_at(cur.dy, j), w[j]), x[j], sdx);
    }
    float i2 = 0.0f, mean = 0.0f;
    if (p.dy) {
      const float2 s = column_sum(make_float2(sum2(sxx), sum2(sdx)), sm, turn);
      i2 = rsqrtf(fmaf(s.x, p.inv_d, p.eps));
      mean = s.y * i2 * p.inv_d;
    }
    // Without a norm of rout its infinite values must not meet the zeros that stand for dy.  (Zeroed by a branch
    // instead: 8192 x 4095 bf16 383 -> 437 us.)
    const unsigned long long keep = p.dy ? ~0ull : 0ull;
    const F2 i2_2 = pack(i2), off = pack(-mean * i2);
    F2 sdv = pack(0.0f);
    param<V, ITEMS>(hw, p.hw, p.D), param<V, ITEMS>(sc, p.scale, p.D), param<V, ITEMS>(w, p.w, p.D);
    {
      Vec<R, V> out[ITEMS];
      Vec<T, V> dg[ITEMS];
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const F2 xh = mul2(F2{x[j].v & keep}, i2_2), dy = pair_at(cur.dy, j);
        add(0, j, dy, xh);
        const F2 dro = fma2(xh, off, fma2(mul2(dy, w[j]), i2_2, pair_at(cur.dro, j)));
        put_pair(out, j, dro);
        const F2 v = mul2(pair_at(cur.h, j), i1_2), n = mul2(v, hw[j]), dm = mul2(dro, sc[j]);
        const F2 a = silu ? mul2(sig[j], pair_at(cur.g, j)) : sig[j];
        add(2, j, dro, mul2(n, a));
        const F2 dn = mul2(dm, a);
        if (p.gate) put_pair(dg, j, mul2(mul2(dm, n), act_grad(a, sig[j], silu)));
        add(1, j, dn, v);
        x[j] = mul2(dn, hw[j]);  // from here: the gradient of v
        sdv = fma2(x[j], v, sdv);
      }
      store_column(p.dr + t * p.lddr, p.D, out);
      if (p.gate) store_column(p.dgate + t * p.lddgate, p.D, dg);
    }
    if (p.h) {
      float back = 0.0f;
      if (p.hw) back = column_sum(make_float2(sum2(sdv), 0.0f), sm, turn).x * p.inv_d * i1;
      const F2 minus = pack(-back);
      const unsigned long long keep_h = p.hw ? ~0ull : 0ull;  // likewise those of h without its norm
      Vec<T, V> out[ITEMS];
#pragma unroll
      for (int j = 0; j < H; ++j) put_pair(out, j, mul2(i1_2, fma2(F2{pair_at(cur.h, j).v & keep_h}, minus, x[j])));
      store_column(p.dh + t * p.lddh, p.D, out);
    }
  }
  float* part = p.parts + walker * 3 * p.D;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    Vec<float, V> out[ITEMS];
#pragma unroll
    for (int j = 0; j < H; ++j) put_pair(out, j, F2{*reinterpret_cast<unsigned long long*>(acc + (i * H + j) * blockDim.x)});
    store_column(part + i * p.D, p.D, out);
  }
}

// The same for 16-bit columns of up to 4096 channels whose rows are 16-byte
// vectors, one per thread: a block's registers leave one to an SM, so what
// hides its waits is not another block but the columns ahead.  S - 1 columns
// are on their way into shared memory while one is computed (every thread
// copies and reads back its own pieces, no barrier), the parameters lie there
// in the threads' order, and mean(h^2) of the next column is reduced together
// with the present one's last sum: two reductions per column instead of three.
// 8192 columns of 4096 channels (bf16, r in Float32): 214 us, 3.5 TB/s, against
// 270 us by norm_bwd (2048 channels 95 against 125 us, 1024 46 against 60, 512 30
// against 28).  What is left are waits, on shared memory, shuffles and the two
// reductions of a column, at four warps per scheduler (issue slots 39% used).
template <typename T, typename R, int S>
__global__ void __launch_bounds__(512, 1) norm_bwd_ahead(Norm<T, R> p) {
  constexpr int V = 8, H = V / 2, kR = V * sizeof(R) / 16, kPieces = 2 * kR + 3;  // h, gate, dy, r, drout
  extern __shared__ uint4 ahead_smem[];  // [S][piece][thread], then [parameter][2][thread]
  __shared__ Sums<3> sm;
  int turn = 0;
  const int nt = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
  const int d = threadIdx.x * V;
  const bool mine = d < p.D;
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  const int64_t walker = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  uint4* stages = ahead_smem + tid;
  uint4* par = ahead_smem + S * kPieces * nt + tid;
  const float* given[3] = {p.hw, p.scale, p.w};
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    Vec<float, V> r;
#pragma unroll
    for (int k = 0; k < V; ++k) r.v[k] = 1.0f;
    load_vec<float, V>(r, given[i] + d, given[i] && mine);
    memcpy(par + 2 * i * nt, &r.v[0], 16), memcpy(par + (2 * i + 1) * nt, &r.v[4], 16);
  }
  sm.clear();
  // pairs 2 q and 2 q + 1 of parameter i
  auto param = [&](F2 (&f)[2], int i, int q) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(par + (2 * i + q) * nt);
    f[0].v = v.x, f[1].v = v.y;
  };
  auto copy = [&](int64_t t, int stage) {
    uint4* to = stages + stage * kPieces * nt;
    const bool on = mine && t < p.T_;
    copy_or_zero(to, on && p.h ? (const void*)(p.h + t * p.ldh + d) : p.r, on && p.h);
    copy_or_zero(to + nt, on && p.gate ? (const void*)(p.gate + t * p.ldgate + d) : p.r, on && p.gate);
    copy_or_zero(to + 2 * nt, on && p.dy ? (const void*)(p.dy + t * p.lddy + d) : p.r, on && p.dy);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int at = d + i * (V / kR);
      copy_or_zero(to + (3 + i) * nt, on ? (const void*)(p.r + t * p.ldr + at) : p.r, on);
      copy_or_zero(to + (3 + kR + i) * nt, on && p.drout ? (const void*)(p.drout + t * p.lddrout + at) : p.r,
                   on && p.drout);
    }
    copy_commit();
  };
  auto take16 = [&](Vec<T, V> (&r)[1], int stage, int piece) {
    const uint4 v = read_shared(stages + (stage * kPieces + piece) * nt);
    memcpy(&r[0], &v, 16);
  };
  auto take_r = [&](Vec<R, V> (&r)[1], int stage, int piece) {
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const uint4 v = read_shared(stages + (stage * kPieces + piece + i) * nt);
      memcpy(reinterpret_cast<char*>(&r[0]) + 16 * i, &v, 16);
    }
  };
  auto sum_hh = [&](int stage) {
    Vec<T, V> h[1];
    take16(h, stage, 0);
    F2 s = pack(0.0f);
#pragma unroll
    for (int j = 0; j < H; ++j) s = fma2(pair_at(h, j), pair_at(h, j), s);
    return sum2(s);
  };
  F2 aw[H], ah[H], as[H];
#pragma unroll
  for (int j = 0; j < H; ++j) aw[j] = ah[j] = as[j] = pack(0.0f);
  const bool silu = p.gate && p.act == MK_ACT_SILU, norm_h = p.h && p.hw;
  int64_t t = walker;
  if (t < p.T_) {
#pragma unroll
    for (int i = 0; i < S - 1; ++i) copy(t + i * stride, i);
    copy_wait<S - 2>();
    int n = 0;
    float i1 = 1.0f;
    if (norm_h) i1 = rsqrtf(fmaf(column_sum(make_float2(sum_hh(0), 0.0f), sm, turn).x, p.inv_d, p.eps));
    for (;;) {
      const F2 i1_2 = pack(i1);
      F2 x[H], sig[H], sxx = pack(0.0f), sdx = pack(0.0f);
      // what is read is read again in each part: registers are scarcer than shared memory
      Vec<T, V> h[1], g[1], dy[1];
      Vec<R, V> r[1];
      take16(h, n, 0), take16(g, n, 1), take16(dy, n, 2), take_r(r, n, 3);
#pragma unroll
      for (int q = 0; q < 2; ++q) {  // without h its values are zeros, without dy those
        F2 hw[2], sc[2], w[2];
        param(hw, 0, q), param(sc, 1, q), param(w, 2, q);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = 2 * q + i;
          const F2 gj = pair_at(g, j);
          sig[j] = p.gate ? sigmoid2<false>(gj) : pack(1.0f);
          F2 m = mul2(mul2(pair_at(h, j), i1_2), mul2(hw[i], sig[j]));
          if (silu) m = mul2(m, gj);
          x[j] = fma2(sc[i], m, pair_at(r, j));
          sxx = fma2(x[j], x[j], sxx);
          sdx = fma2(mul2(pair_at(dy, j), w[i]), x[j], sdx);
        }
      }
      float i2 = 0.0f, mean = 0.0f;
      if (p.dy) {
        const float2 s = column_sum(make_float2(sum2(sxx), sum2(sdx)), sm, turn);
        i2 = rsqrtf(fmaf(s.x, p.inv_d, p.eps));
        mean = s.y * i2 * p.inv_d;
      } else {  // no norm of rout: infinite values of it must not meet the zeros of dy
#pragma unroll
        for (int j = 0; j < H; ++j) x[j] = pack(0.0f);
      }
      const F2 i2_2 = pack(i2), off = pack(-mean * i2);
      F2 sdv = pack(0.0f);
      Vec<T, V> dg[1];
      take16(h, n, 0), take16(g, n, 1), take16(dy, n, 2);
      take_r(r, n, 3 + kR);  // drout, and from there dr
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        F2 hw[2], sc[2], w[2];
        param(hw, 0, q), param(sc, 1, q), param(w, 2, q);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = 2 * q + i;
          const F2 xh = mul2(x[j], i2_2), dyj = pair_at(dy, j), v = mul2(pair_at(h, j), i1_2), n_ = mul2(v, hw[i]);
          aw[j] = fma2(dyj, xh, aw[j]);
          const F2 dro = fma2(xh, off, fma2(mul2(dyj, w[i]), i2_2, pair_at(r, j))), dm = mul2(dro, sc[i]);
          put_pair(r, j, dro);
          const F2 a = silu ? mul2(sig[j], pair_at(g, j)) : sig[j];
          as[j] = fma2(dro, mul2(n_, a), as[j]);
          if (p.gate) put_pair(dg, j, mul2(mul2(dm, n_), act_grad(a, sig[j], silu)));
          const F2 dn = mul2(dm, a);
          ah[j] = fma2(dn, v, ah[j]);
          x[j] = mul2(dn, hw[i]);  // from here: the gradient of v
          sdv = fma2(x[j], v, sdv);
        }
      }
      if (mine) {
        *reinterpret_cast<Vec<R, V>*>(p.dr + t * p.lddr + d) = r[0];
        if (p.gate) *reinterpret_cast<Vec<T, V>*>(p.dgate + t * p.lddgate + d) = dg[0];
      }
      const int64_t next = t + stride;
      copy(next + (S - 2) * stride, n == 0 ? S - 1 : n - 1);
      copy_wait<S - 2>();
      const int n_next = n + 1 == S ? 0 : n + 1;
      float back = 0.0f, i1_next = 1.0f;
      if (norm_h) {
        const float2 s = column_sum(make_float2(sum2(sdv), sum_hh(n_next)), sm, turn);
        back = s.x * p.inv_d * i1;
        i1_next = rsqrtf(fmaf(s.y, p.inv_d, p.eps));
      }
      if (p.h) {
        if (norm_h) {  // without, infinite values of h stay out of it
          const F2 minus = pack(-back);
          take16(h, n, 0);
#pragma unroll
          for (int j = 0; j < H; ++j) x[j] = mul2(i1_2, fma2(pair_at(h, j), minus, x[j]));
        }
#pragma unroll
        for (int j = 0; j < H; ++j) put_pair(dg, j, x[j]);
        if (mine) *reinterpret_cast<Vec<T, V>*>(p.dh + t * p.lddh + d) = dg[0];
      }
      t = next;
      if (t >= p.T_) break;
      i1 = i1_next, n = n_next;
    }
    copy_wait<0>();
  }
  float* part = p.parts + walker * 3 * p.D + d;
  if (!mine) return;
  Vec<float, V> out[1];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
#pragma unroll
    for (int j = 0; j < H; ++j) put_pair(out, j, i == 0 ? aw[j] : i == 1 ? ah[j] : as[j]);
    *reinterpret_cast<Vec<float, V>*>(part + i * p.D) = out[0];
  }
}

// dw, dhw, dscale: the sums over the column walkers, 32 values and 16 ranges of
// walkers per block.
constexpr int kFoldRows = 16;
__global__ void __launch_bounds__(32 * kFoldRows) norm_fold(const float* parts, int64_t nparts, int64_t D, float* dw,
                                                            float* dhw, float* dscale) {
  __shared__ float sm[kFoldRows][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x, n = 3 * D;
  float v = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int64_t k = threadIdx.y; k < nparts; k += kFoldRows) v += parts[k * n + i];
  }
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || i >= n) return;
  v = 0.0f;
#pragma unroll
  for (int k = 0; k < kFoldRows; ++k) v += sm[k][threadIdx.x];
  float* out = i < D ? dw : i < 2 * D ? dhw : dscale;
  if (out) out[i % D] = v;
}

// ---- host side ----------------------------------------------------------------

constexpr int64_t kMostChannels = 16384;  // 16 values for each of 1024 threads

int check(const char* who, const mk_norm_args* a, bool grad) {
  if (!a) return bad(who, "null arguments");
  if (a->type < MK_T_F32 || a->type > MK_T_BF16) return bad(who, "unknown element type");
  if (a->rtype != MK_T_F32 && a->rtype != a->type) return bad(who, "r is Float32 or of the type of the others");
  if (a->act != MK_ACT_SILU && a->act != MK_ACT_SIGMOID) return bad(who, "unknown gate activation");
  if (a->D < 1 || a->T < 0) return bad(who, "negative size or no channels");
  if (a->D > kMostChannels) return bad(who, "at most 16384 channels, got " + std::to_string(a->D));
  if (a->T > INT32_MAX) return bad(who, "more than 2^31 - 1 tokens");
  if (!(a->eps >= 0.0f)) return bad(who, "eps must not be negative");
  if (!a->h && (a->gate || a->hw || a->scale) && a->T) return bad(who, "gate, hw and scale belong to h");
  const size_t es = type_bytes(a->type), rs = type_bytes(a->rtype);
  MK_TRY(check_matrix(who, "r", a->r, a->D, a->ldr, a->T, rs));
  if (a->h) MK_TRY(check_matrix(who, "h", a->h, a->D, a->ldh, a->T, es));
  if (a->gate) MK_TRY(check_matrix(who, "gate", a->gate, a->D, a->ldgate, a->T, es));
  MK_TRY(check_floats(who, "hw", a->hw, false, false));
  MK_TRY(check_floats(who, "scale", a->scale, false, false));
  MK_TRY(check_floats(who, "w", a->w, false, false));
  if (!grad) {
    if (a->T && !a->y != !a->w) return bad(who, "y and w are given together");
    if (a->y) MK_TRY(check_matrix(who, "y", a->y, a->D, a->ldy, a->T, es));
    if (a->rout) MK_TRY(check_matrix(who, "rout", a->rout, a->D, a->ldrout, a->T, rs));
    if (a->T && !a->y && !a->rout) return bad(who, "neither y nor rout is given");
    return MK_OK;
  }
  if (a->T && !a->dy && !a->drout) return bad(who, "neither dy nor drout is given");
  if (a->T && !a->dy != !a->w) return bad(who, "dy and w are given together");
  if (!a->w != !a->dw || !a->hw != !a->dhw || !a->scale != !a->dscale)
    return bad(who, "dw, dhw and dscale are needed exactly when w, hw and scale are given");
  if (a->T && (!a->h != !a->dh || !a->gate != !a->dgate))
    return bad(who, "dh and dgate are needed exactly when h and gate are given");
  if (a->dy) MK_TRY(check_matrix(who, "dy", a->dy, a->D, a->lddy, a->T, es));
  if (a->drout) MK_TRY(check_matrix(who, "drout", a->drout, a->D, a->lddrout, a->T, rs));
  MK_TRY(check_matrix(who, "dr", a->dr, a->D, a->lddr, a->T, rs));
  if (a->h) MK_TRY(check_matrix(who, "dh", a->dh, a->D, a->lddh, a->T, es));
  if (a->gate) MK_TRY(check_matrix(who, "dgate", a->dgate, a->D, a->lddgate, a->T, es));
  MK_TRY(check_floats(who, "dw", a->dw, false, false));
  MK_TRY(check_floats(who, "dhw", a->dhw, false, false));
  return check_floats(who, "dscale", a->dscale, false, false);
}

// Whether every matrix and vector can be taken V elements at a time.
bool all_vec(const mk_norm_args* a, int V, bool grad) {
  const size_t es = type_bytes(a->type), rs = type_bytes(a->rtype);
  bool ok = a->D % V == 0 && vec_ok(a->r, a->ldr, rs, V) && vec_ok(a->h, a->ldh, es, V) &&
            vec_ok(a->gate, a->ldgate, es, V) && vec_ok(a->hw, 0, 4, V) && vec_ok(a->scale, 0, 4, V) &&
            vec_ok(a->w, 0, 4, V);
  if (!grad) return ok && vec_ok(a->y, a->ldy, es, V) && vec_ok(a->rout, a->ldrout, rs, V);
  return ok && vec_ok(a->dy, a->lddy, es, V) && vec_ok(a->drout, a->lddrout, rs, V) &&
         vec_ok(a->dr, a->lddr, rs, V) && vec_ok(a->dh, a->lddh, es, V) && vec_ok(a->dgate, a->lddgate, es, V);
}

// Threads of a column and columns of a block.
dim3 block_of(int64_t D, int V, int items) {
  const int64_t threads = mk::cdiv(mk::cdiv(D, V * items), 32) * 32;
  return dim3((unsigned)threads, threads == 32 ? 4 : 1);
}

template <typename T, typename R>
Norm<T, R> params(const mk_norm_args* a) {
  Norm<T, R> p{};
  p.D = (int)a->D, p.T_ = a->T, p.eps = a->eps, p.inv_d = 1.0f / (float)a->D, p.act = a->act;
  p.r = static_cast<const R*>(a->r), p.ldr = a->ldr;
  p.h = static_cast<const T*>(a->h), p.ldh = a->ldh;
  p.gate = static_cast<const T*>(a->gate), p.ldgate = a->ldgate;
  p.rout = static_cast<R*>(a->rout), p.ldrout = a->ldrout;
  p.y = static_cast<T*>(a->y), p.ldy = a->ldy;
  p.hw = a->hw, p.scale = a->scale, p.w = a->w;
  p.dy = static_cast<const T*>(a->dy), p.lddy = a->lddy;
  p.drout = static_cast<const R*>(a->drout), p.lddrout = a->lddrout;
  p.dr = static_cast<R*>(a->dr), p.lddr = a->lddr;
  p.dh = static_cast<T*>(a->dh), p.lddh = a->lddh;
  p.dgate = static_cast<T*>(a->dgate), p.lddgate = a->lddgate;
  p.parts = static_cast<float*>(a->workspace);
  return p;
}

template <typename T, typename R, int V, int ITEMS, int THREADS, int BLOCKS>
int launch_fwd(const mk_norm_args* a, cudaStream_t s) {
  const dim3 block = block_of(a->D, V, ITEMS);
  norm_fwd<T, R, V, ITEMS, THREADS, BLOCKS><<<(unsigned)mk::cdiv(a->T, block.y), block, 0, s>>>(params<T, R>(a));
  return mk::check_launch("mk_block_norm: launch");
}

// 16 values per thread; columns of up to 4096 channels take 256 threads at
// most, so that the registers hold four of them on an SM: 8192 x 4096 (bf16, r in
// Float32) 83 us, 5.7 TB/s, against 116 us with 8 values of 512 threads (2048
// channels 44 against 49, 1024 and 512 the same).  Single elements take more
// registers: 8 values per thread (8192 x 4095 Float32 195 -> 166 us, 1023 bf16 40 ->
// 38), but for the widest of 16 bits (4095 bf16 162 -> 151 us with 16).
template <typename T, typename R>
int run_fwd(const mk_norm_args* a, cudaStream_t s) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  if (all_vec(a, V, false))
    return a->D <= 4096 ? launch_fwd<T, R, V, 16 / V, 256, 4>(a, s) : launch_fwd<T, R, V, 16 / V, 1024, 1>(a, s);
  if (a->D > 4096) return launch_fwd<T, R, 1, 16, 1024, 1>(a, s);
  if constexpr (sizeof(T) == 2) {
    if (a->D > 2048) return launch_fwd<T, R, 1, 16, 256, 3>(a, s);
  }
  return launch_fwd<T, R, 1, 8, 512, 2>(a, s);
}

// Values per thread: 8, and 16 of columns beyond 4096 channels; up to 8192 of
// them that is 512 threads of 128 registers each (4096 x 8192 bf16 630 -> 305 us
// against code for 1024, 5120 channels 458 -> 219).  They spill all the same, 220
// to 630 bytes; beyond 8192 channels, with 64 registers, 1060 to 1860.
struct BwdPlan {
  int V, items;
  dim3 block;
  int64_t grid, parts;
};

BwdPlan plan_bwd(const mk_norm_args* a, const mk::Device* dev) {
  BwdPlan b;
  const bool half = type_bytes(a->type) == 2;
  b.V = all_vec(a, half ? 8 : 4, true) ? (half ? 8 : 4) : 1;
  b.items = (a->D > 4096 ? 16 : 8) / b.V;
  b.block = block_of(a->D, b.V, b.items);
  const int64_t columns = mk::cdiv(a->T, b.block.y);
  const int64_t threads = (int64_t)b.block.x * b.block.y;
  const int64_t most = (int64_t)dev->sms * (threads < 512 ? 512 / threads : 1);  // resident at once
  b.grid = columns < most ? columns : most;
  b.parts = b.grid * b.block.y;
  return b;
}

template <typename T, typename R, int V, int ITEMS, int THREADS, int BLOCKS>
int launch_bwd(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  const Norm<T, R> p = params<T, R>(a);
  const auto kernel = norm_bwd<T, R, V, ITEMS, THREADS, BLOCKS>;
  const size_t smem = (size_t)3 * V * ITEMS * sizeof(float) * b.block.x * b.block.y;
  MK_TRY(mk::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem));
  if (b.grid) kernel<<<(unsigned)b.grid, b.block, smem, s>>>(p);
  norm_fold<<<(unsigned)mk::cdiv(3 * a->D, 32), dim3(32, kFoldRows), 0, s>>>(p.parts, b.parts, a->D, a->dw, a->dhw, a->dscale);
  return mk::check_launch("mk_block_norm_grad: launch");
}

template <typename T, typename R>
int launch_bwd_ahead(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  constexpr int S = 3;
  const Norm<T, R> p = params<T, R>(a);
  const auto kernel = norm_bwd_ahead<T, R, S>;
  const size_t smem = (size_t)(S * (2 * 8 * sizeof(R) / 16 + 3) + 6) * 16 * b.block.x * b.block.y;
  MK_TRY(mk::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem));
  if (b.grid) kernel<<<(unsigned)b.grid, b.block, smem, s>>>(p);
  norm_fold<<<(unsigned)mk::cdiv(3 * a->D, 32), dim3(32, kFoldRows), 0, s>>>(p.parts, b.parts, a->D, a->dw, a->dhw, a->dscale);
  return mk::check_launch("mk_block_norm_grad: launch");
}

template <typename T, typename R>
int run_bwd(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  if constexpr (V == 8) {
    if (b.V == 8 && a->D <= 4096) return launch_bwd_ahead<T, R>(a, b, s);
  }
  if (a->D > 4096 && a->D <= 8192)
    return b.V == V ? launch_bwd<T, R, V, 16 / V, 512, 1>(a, b, s) : launch_bwd<T, R, 1, 16, 512, 1>(a, b, s);
  if (a->D > 4096)
    return b.V == V ? launch_bwd<T, R, V, 16 / V, 1024, 1>(a, b, s) : launch_bwd<T, R, 1, 16, 1024, 1>(a, b, s);
  if constexpr (V == 4) {
    if (b.V == 4) return launch_bwd<T, R, 4, 2, 512, 1>(a, b, s);
  }
  return launch_bwd<T, R, 1, 8, 512, 1>(a, b, s);
}

int forward(const mk_norm_args* a, void* stream) {
  MK_TRY(check("mk_block_norm", a, false));
  if (a->T == 0) return MK_OK;
  MK_ENTRY_DEVICE(dev);
  (void)dev;
  cudaStream_t s = mk::as_stream(stream);
  if (a->type == MK_T_F32) return run_fwd<float, float>(a, s);
  if (a->type == MK_T_F16)
    return a->rtype == MK_T_F32 ? run_fwd<__half, float>(a, s) : run_fwd<__half, __half>(a, s);
  return a->rtype == MK_T_F32 ? run_fwd<__nv_bfloat16, float>(a, s)
                              : run_fwd<__nv_bfloat16, __nv_bfloat16>(a, s);
}

int workspace(const mk_norm_args* a, size_t* bytes) {
  const char* who = "mk_block_norm_grad_workspace";
  if (!a || !bytes) return bad(who, "null arguments");
  if (a->D < 1 || a->D > kMostChannels || a->T < 0) return bad(who, "size out of range");
  MK_ENTRY_DEVICE(dev);
  *bytes = (size_t)plan_bwd(a, dev).parts * 3 * a->D * sizeof(float);
  return MK_OK;
}

int gradient(const mk_norm_args* a, void* stream) {
  const char* who = "mk_block_norm_grad";
  MK_TRY(check(who, a, true));
  MK_ENTRY_DEVICE(dev);
  const BwdPlan b = plan_bwd(a, dev);
  const size_t need = (size_t)b.parts * 3 * a->D * sizeof(float);
  if (need && (!a->workspace || a->workspace_bytes < need || !elem_aligned(a->workspace, 16)))
    return bad(who, "a 16-byte aligned workspace of " + std::to_string(need) + " bytes is needed");
  cudaStream_t s = mk::as_stream(stream);
  if (a->type == MK_T_F32) return run_bwd<float, float>(a, b, s);
  if (a->type == MK_T_F16)
    return a->rtype == MK_T_F32 ? run_bwd<__half, float>(a, b, s) : run_bwd<__half, __half>(a, b, s);
  return a->rtype == MK_T_F32 ? run_bwd<__nv_bfloat16, float>(a, b, s)
                              : run_bwd<__nv_bfloat16, __nv_bfloat16>(a, b, s);
}

}  // namespace

extern "C" int mk_block_norm(const mk_norm_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return forward(a, stream); });
}

extern "C" int mk_block_norm_grad_workspace(const mk_norm_args* a, size_t* bytes) {
  mk::clear_error();
  return guarded([&] { return workspace(a, bytes); });
}

extern "C" int mk_block_norm_grad(const mk_norm_args* a, void* stream) {
  mk::clear_error();
  return guarded([&] { return gradient(a, stream); });
}
