// block_norm.cu — the norms around a block, fused with the block's gate and
// its scaled residual: per token column of D channels
//     n = h / rms(h) * hw,  m = n * act(gate),  rout = r + scale * m,
//     y = rout / rms(rout) * w,   rms(x) = sqrt(mean(x^2) + eps).
//
// Bound by memory: every matrix is read or written once; a column stays in
// registers between its reductions (V * ITEMS values per thread).  A column
// of up to 32 * V * ITEMS channels is one warp's (shuffles only), wider ones a
// block's.  Blocks walk columns: the next ones are on their way into shared
// memory while one is computed, and mean(h^2), which is needed first, is
// reduced together with the column before's last sum, so that a column costs
// one reduction forward and two backward.  Backward recomputes the forward
// values from r, h and gate, which costs no more reads than saving rout and
// its rms would.
#include "tokens.cuh"

namespace {

using namespace mk::tok;

template <typename T, typename R>
struct Norm {
  int64_t D, T_;
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
// as two buffers alternate one barrier is enough.
struct alignas(16) Sums {
  float2 part[2][32];  // zeros where there is no warp
  __device__ __forceinline__ void clear() {
    const int i = threadIdx.y * blockDim.x + threadIdx.x;
    if (i < 64) part[i / 32][i % 32] = make_float2(0.0f, 0.0f);
    if (blockDim.x * blockDim.y < 64 && i < 32) part[1][i] = make_float2(0.0f, 0.0f);
    __syncthreads();
  }
};
__device__ __forceinline__ float2 column_sum(float2 v, Sums& sm, int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (blockDim.x == 32) return v;
  if ((threadIdx.x & 31) == 0) sm.part[turn][threadIdx.x >> 5] = v;
  __syncthreads();
  const ulonglong2* part = reinterpret_cast<const ulonglong2*>(sm.part[turn]);
  F2 a = pack(0.0f), b = pack(0.0f);
  for (int i = 0; i < (int)(blockDim.x + 63) / 64; ++i) {  // two warps at a time
    const ulonglong2 q = part[i];
    a = add2(a, F2{q.x}), b = add2(b, F2{q.y});
  }
  a = add2(a, b);
  unpack(a, v.x, v.y);
  turn ^= 1;
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
  static constexpr int kPR = V * sizeof(R) / 16, kPT = V * sizeof(T) / 16;  // 16-byte pieces of a vector
  static constexpr int kPieces = ITEMS * (GRAD ? 2 * kPR + 3 * kPT : kPR + 2 * kPT);

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        r[k].v[i] = from_f<R>(0.0f), h[k].v[i] = g[k].v[i] = from_f<T>(0.0f);
        if (GRAD) dro[k].v[i] = from_f<R>(0.0f), dy[k].v[i] = from_f<T>(0.0f);
      }
  }
  // F(vector in registers, its place in memory, whether it is there) for h of column t, and for the rest of it
  template <typename F>
  __device__ __forceinline__ void each_h(Vec<T, V> (&h)[ITEMS], const Norm<T, R>& p, int64_t t, F&& f) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      f(h[k], p.h + t * p.ldh + d, d < p.D && t < p.T_ && p.h);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_other(const Norm<T, R>& p, int64_t t, F&& f) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      const bool on = d < p.D && t < p.T_;
      f(r[k], p.r + t * p.ldr + d, on);
      f(g[k], p.gate + t * p.ldgate + d, on && p.gate);
      if constexpr (GRAD) {
        f(dy[k], p.dy + t * p.lddy + d, on && p.dy);
        f(dro[k], p.drout + t * p.lddrout + d, on && p.drout);
      }
    }
  }
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
__device__ __forceinline__ void store_column(X* column, int64_t D, const Vec<X, V> (&r)[ITEMS]) {
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
    if (d < D) *reinterpret_cast<Vec<X, V>*>(column + d) = r[k];
  }
}

// The columns that a thread walks, one after another.  S > 1: S - 1 of them are
// on their way into shared memory while one is computed; every thread copies
// and reads back its own 16-byte pieces, so no barrier is needed.  S == 1:
// straight from memory.
template <typename T, typename R, int V, int ITEMS, bool GRAD, int S>
struct Walk {
  using C = Column<T, R, V, ITEMS, GRAD>;
  C now;
  Vec<T, V> h_next[ITEMS];
  uint4* stages;
  int tid, nt, n = 0;  // n: the stage of the next column
  int64_t stride;

  __device__ __forceinline__ uint4* piece(int stage, int i) { return stages + (stage * C::kPieces + i) * nt + tid; }
  __device__ __forceinline__ void copy(const Norm<T, R>& p, int64_t t, int stage) {
    int i = 0;
    auto f = [&](auto& r, auto* at, bool on) {
#pragma unroll
      for (int x = 0; x < (int)(sizeof(r) / 16); ++x)
        copy_or_zero(piece(stage, i++), on ? (const void*)(reinterpret_cast<const uint4*>(at) + x) : p.r, on);
    };
    now.each_h(now.h, p, t, f);
    now.each_other(p, t, f);
    copy_commit();
  }
  __device__ __forceinline__ Walk(const Norm<T, R>& p, int64_t t, int64_t stride_, uint4* smem) : stride(stride_) {
    stages = smem;
    tid = threadIdx.y * blockDim.x + threadIdx.x;
    nt = blockDim.x * blockDim.y;
    now.clear();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) h_next[k] = now.h[k];
    if constexpr (S > 1) {
#pragma unroll
      for (int i = 0; i < S - 1; ++i) copy(p, t + i * stride, i);
    }
  }
  // h of column t, the next one, into h_next.
  __device__ __forceinline__ void take_h(const Norm<T, R>& p, int64_t t) {
    if constexpr (S > 1) {
      copy(p, t + (S - 1) * stride, n == 0 ? S - 1 : n - 1);
      copy_wait<S - 1>();
      int i = 0;
      now.each_h(h_next, p, t, [&](auto& r, auto*, bool) {
#pragma unroll
        for (int x = 0; x < (int)(sizeof(r) / 16); ++x) {
          const uint4 v = *piece(n, i++);
          memcpy(reinterpret_cast<char*>(&r) + 16 * x, &v, 16);
        }
      });
    } else {
      now.each_h(h_next, p, t, [](auto& r, auto* at, bool on) { load_vec(r, at, on); });
    }
  }
  // The rest of it, and its h to where it belongs: column t is now the present one.
  __device__ __forceinline__ void take_rest(const Norm<T, R>& p, int64_t t) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) now.h[k] = h_next[k];
    if constexpr (S > 1) {
      int i = ITEMS * C::kPT;
      now.each_other(p, t, [&](auto& r, auto*, bool) {
#pragma unroll
        for (int x = 0; x < (int)(sizeof(r) / 16); ++x) {
          const uint4 v = *piece(n, i++);
          memcpy(reinterpret_cast<char*>(&r) + 16 * x, &v, 16);
        }
      });
      n = n + 1 == S ? 0 : n + 1;
    } else {
      now.each_other(p, t, [](auto& r, auto* at, bool on) { load_vec(r, at, on); });
    }
  }
  __device__ __forceinline__ float sum_h_next() const {
    F2 s = pack(0.0f);
#pragma unroll
    for (int j = 0; j < V * ITEMS / 2; ++j) {
      const F2 h = pair_at(h_next, j);
      s = fma2(h, h, s);
    }
    return sum2(s);
  }
  __device__ __forceinline__ void end() {
    if constexpr (S > 1) copy_wait<0>();
  }
};

// Values 2 j and 2 j + 1 of a thread's channels of a parameter, ones without it.
template <int V>
__device__ __forceinline__ F2 param_at(const float* p, int64_t D, int j) {
  const int64_t d0 = ((int64_t)(2 * j / V) * blockDim.x + threadIdx.x) * V + 2 * j % V;
  if constexpr (V > 1) {
    const F2 one = pack(1.0f);
    return p && d0 < D ? F2{*reinterpret_cast<const unsigned long long*>(p + d0)} : one;
  } else {
    const int64_t d1 = d0 + blockDim.x;
    return pack(p && d0 < D ? p[d0] : 1.0f, p && d1 < D ? p[d1] : 1.0f);
  }
}

// All of a thread's values of a parameter.
template <int V, int ITEMS>
__device__ __forceinline__ void param(F2 (&f)[V * ITEMS / 2], const float* p, int64_t D) {
#pragma unroll
  for (int j = 0; j < V * ITEMS / 2; ++j) f[j] = param_at<V>(p, D, j);
}

template <typename T, typename R, int V, int ITEMS, int S>
__global__ void __launch_bounds__(V * ITEMS <= 8 ? 512 : 1024, 1) norm_fwd(Norm<T, R> p) {
  constexpr bool kExact = sizeof(T) == 4;
  constexpr bool kHold = V * ITEMS <= 8;  // parameters in registers
  extern __shared__ uint4 norm_smem[];
  __shared__ Sums sm;
  int turn = 0;
  sm.clear();
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= p.T_) return;
  Walk<T, R, V, ITEMS, false, S> walk(p, t, stride, norm_smem);
  constexpr int H = V * ITEMS / 2;
  F2 hw[H], sc[H], w[H];
  if constexpr (kHold) param<V, ITEMS>(hw, p.hw, p.D), param<V, ITEMS>(sc, p.scale, p.D), param<V, ITEMS>(w, p.w, p.D);
  const bool norm_h = p.h && p.hw;
  walk.take_h(p, t);
  float i1 = 1.0f;
  if (norm_h) i1 = rsqrtf(fmaf(column_sum(make_float2(walk.sum_h_next(), 0.0f), sm, turn).x, p.inv_d, p.eps));
  walk.take_rest(p, t);
  const auto& cur = walk.now;
  for (;;) {
    const bool silu = p.act == MK_ACT_SILU;
    if constexpr (!kHold) param<V, ITEMS>(hw, p.hw, p.D), param<V, ITEMS>(sc, p.scale, p.D);
    F2 x[H], sum = pack(0.0f);
    const F2 i1_2 = pack(i1);
#pragma unroll
    for (int j = 0; j < H; ++j) x[j] = mul2(mul2(pair_at(cur.h, j), i1_2), hw[j]);  // zeros without h
    if (p.gate) {
#pragma unroll
      for (int j = 0; j < H; ++j) {
        const F2 g = pair_at(cur.g, j);
        x[j] = mul2(x[j], sigmoid2<kExact>(g));
        if (silu) x[j] = mul2(x[j], g);
      }
    }
#pragma unroll
    for (int j = 0; j < H; ++j) {
      x[j] = fma2(sc[j], x[j], pair_at(cur.r, j));
      sum = fma2(x[j], x[j], sum);  // channels beyond D are zeros
    }
    if (p.rout) {
      Vec<R, V> out[ITEMS];
#pragma unroll
      for (int j = 0; j < H; ++j) put_pair(out, j, x[j]);
      store_column(p.rout + t * p.ldrout, p.D, out);
    }
    float2 s = make_float2(sum2(sum), 0.0f);
    const int64_t next = t + stride;
    walk.take_h(p, next);
    if (norm_h) s.y = walk.sum_h_next();
    if (p.y || norm_h) s = column_sum(s, sm, turn);
    if (p.y) {
      const F2 i2 = pack(rsqrtf(fmaf(s.x, p.inv_d, p.eps)));
      if constexpr (!kHold) param<V, ITEMS>(w, p.w, p.D);
      Vec<T, V> out[ITEMS];
#pragma unroll
      for (int j = 0; j < H; ++j) put_pair(out, j, mul2(w[j], mul2(x[j], i2)));
      store_column(p.y + t * p.ldy, p.D, out);
    }
    t = next;
    if (t >= p.T_) break;
    if (norm_h) i1 = rsqrtf(fmaf(s.y, p.inv_d, p.eps));
    walk.take_rest(p, t);
  }
  walk.end();
}

// Backward.  With x = rout i2 and dx = dy w:
//   dro = drout + i2 (dx - x mean(dx x)),  dr = dro,
//   dm = dro scale, dn = dm act, dgate = dm n act', dv = dn hw,
//   dh = i1 (dv - v mean(dv v)), v = h i1;
// dw += dy x, dhw += dn v, dscale += dro m.  A block walks columns, keeps its
// sums for w, hw and scale in registers (one part per column walker, added up
// by norm_fold in a fixed order), and keeps the inputs as they are in memory
// between its three reductions.
template <typename T, typename R, int V, int ITEMS, int S>
__global__ void __launch_bounds__(V * ITEMS <= 8 ? 512 : 1024, 1) norm_bwd(Norm<T, R> p) {
  constexpr bool kExact = sizeof(T) == 4;
  extern __shared__ uint4 norm_smem[];
  __shared__ Sums sm;
  int turn = 0;
  sm.clear();
  const int64_t stride = (int64_t)gridDim.x * blockDim.y;
  const int64_t walker = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  constexpr int H = V * ITEMS / 2;
  F2 aw[H], ah[H], as[H];
#pragma unroll
  for (int j = 0; j < H; ++j) aw[j] = ah[j] = as[j] = pack(0.0f);
  // the parameters in shared memory behind the stages, ones for those that are not there
  const float *p_hw = p.hw, *p_scale = p.scale, *p_w = p.w;
  if constexpr (S > 1) {
    float* sp = reinterpret_cast<float*>(norm_smem + S * Column<T, R, V, ITEMS, true>::kPieces * blockDim.x * blockDim.y);
    for (int64_t i = threadIdx.y * blockDim.x + threadIdx.x; i < p.D; i += blockDim.x * blockDim.y) {
      sp[i] = p.hw ? p.hw[i] : 1.0f;
      sp[p.D + i] = p.scale ? p.scale[i] : 1.0f;
      sp[2 * p.D + i] = p.w ? p.w[i] : 1.0f;
    }
    __syncthreads();
    p_hw = sp, p_scale = sp + p.D, p_w = sp + 2 * p.D;
  }
  int64_t t = walker;
  if (t < p.T_) {
    Walk<T, R, V, ITEMS, true, S> walk(p, t, stride, norm_smem);
    const bool norm_h = p.h && p.hw;
    walk.take_h(p, t);
    float i1 = 1.0f;
    if (norm_h) i1 = rsqrtf(fmaf(column_sum(make_float2(walk.sum_h_next(), 0.0f), sm, turn).x, p.inv_d, p.eps));
    walk.take_rest(p, t);
    const auto& cur = walk.now;
    for (;;) {
      F2 x[H], sig[H];  // sig: of the gate, ones without
      const bool silu = p.gate && p.act == MK_ACT_SILU;
      F2 sxx = pack(0.0f), sdx = pack(0.0f);
      const F2 i1_2 = pack(i1);
#pragma unroll
      for (int j = 0; j < H; ++j) sig[j] = p.gate ? sigmoid2<kExact>(pair_at(cur.g, j)) : pack(1.0f);
#pragma unroll
      for (int j = 0; j < H; ++j) {  // without h its values are zeros, without dy those
        F2 m = mul2(mul2(mul2(pair_at(cur.h, j), i1_2), param_at<V>(p_hw, p.D, j)), sig[j]);
        if (silu) m = mul2(m, pair_at(cur.g, j));
        x[j] = fma2(param_at<V>(p_scale, p.D, j), m, pair_at(cur.r, j));
        sxx = fma2(x[j], x[j], sxx);
        sdx = fma2(mul2(pair_at(cur.dy, j), param_at<V>(p_w, p.D, j)), x[j], sdx);
      }
      float i2 = 0.0f, mean = 0.0f;
      if (p.dy) {
        const float2 s = column_sum(make_float2(sum2(sxx), sum2(sdx)), sm, turn);
        i2 = rsqrtf(fmaf(s.x, p.inv_d, p.eps));
        mean = s.y * i2 * p.inv_d;
      }
      const F2 i2_2 = pack(i2), off = pack(-mean * i2);
      F2 dv[H], sdv = pack(0.0f);
      {
        Vec<R, V> out[ITEMS];
        Vec<T, V> dg[ITEMS];
#pragma unroll
        for (int j = 0; j < H; ++j) {
          const F2 xh = mul2(x[j], i2_2), dy = pair_at(cur.dy, j);
          aw[j] = fma2(dy, xh, aw[j]);
          const F2 dro = fma2(xh, off, fma2(mul2(dy, param_at<V>(p_w, p.D, j)), i2_2, pair_at(cur.dro, j)));
          put_pair(out, j, dro);
          const F2 hw = param_at<V>(p_hw, p.D, j);
          const F2 v = mul2(pair_at(cur.h, j), i1_2), n = mul2(v, hw), dm = mul2(dro, param_at<V>(p_scale, p.D, j));
          const F2 a = silu ? mul2(sig[j], pair_at(cur.g, j)) : sig[j];
          as[j] = fma2(dro, mul2(n, a), as[j]);
          const F2 dn = mul2(dm, a);
          if (p.gate) put_pair(dg, j, mul2(mul2(dm, n), act_grad(a, sig[j], silu)));
          ah[j] = fma2(dn, v, ah[j]);
          dv[j] = mul2(dn, hw);
          sdv = fma2(dv[j], v, sdv);
        }
        store_column(p.dr + t * p.lddr, p.D, out);
        if (p.gate) store_column(p.dgate + t * p.lddgate, p.D, dg);
      }
      const int64_t next = t + stride;
      walk.take_h(p, next);
      float back = 0.0f, i1_next = 1.0f;
      if (norm_h) {
        const float2 s = column_sum(make_float2(sum2(sdv), walk.sum_h_next()), sm, turn);
        back = s.x * p.inv_d * i1;
        i1_next = rsqrtf(fmaf(s.y, p.inv_d, p.eps));
      }
      if (p.h) {
        const F2 minus = pack(-back);
        Vec<T, V> out[ITEMS];
#pragma unroll
        for (int j = 0; j < H; ++j) put_pair(out, j, mul2(i1_2, fma2(pair_at(cur.h, j), minus, dv[j])));
        store_column(p.dh + t * p.lddh, p.D, out);
      }
      t = next;
      if (t >= p.T_) break;
      i1 = i1_next;
      walk.take_rest(p, t);
    }
    walk.end();
  }
  float* part = p.parts + walker * 3 * p.D;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    Vec<float, V> out[ITEMS];
#pragma unroll
    for (int j = 0; j < H; ++j) put_pair(out, j, i == 0 ? aw[j] : i == 1 ? ah[j] : as[j]);
    store_column(part + i * p.D, p.D, out);
  }
}

// dw, dhw, dscale: the sums over the column walkers, 32 values and 8 ranges of
// walkers per block.
__global__ void __launch_bounds__(256) norm_fold(const float* parts, int64_t nparts, int64_t D, float* dw, float* dhw,
                                                 float* dscale) {
  __shared__ float sm[8][32];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x, n = 3 * D;
  float v = 0.0f;
  if (i < n) {
#pragma unroll 4
    for (int64_t k = threadIdx.y; k < nparts; k += 8) v += parts[k * n + i];
  }
  sm[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || i >= n) return;
  v = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += sm[k][threadIdx.x];
  float* out = i < D ? dw : i < 2 * D ? dhw : dscale;
  if (out) out[i % D] = v;
}

// ---- host side ----------------------------------------------------------------

constexpr int64_t kMostChannels = 16384;

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
  p.D = a->D, p.T_ = a->T, p.eps = a->eps, p.inv_d = 1.0f / (float)a->D, p.act = a->act;
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

// S stages of the column walk in shared memory, and `more` bytes behind them.
template <int S, typename K, typename... A>
int launch(K kernel, int64_t grid, dim3 block, int pieces, size_t more, cudaStream_t s, const char* who, A... args) {
  const size_t smem = S > 1 ? (size_t)S * pieces * 16 * block.x * block.y + more : 0;
  if (smem) MK_TRY(mk::allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem));
  kernel<<<(unsigned)grid, block, smem, s>>>(args...);
  return mk::check_launch(who);
}

template <typename T, typename R, int V, int ITEMS, int S>
int launch_fwd(const mk_norm_args* a, const mk::Device* dev, cudaStream_t s) {
  const dim3 block = block_of(a->D, V, ITEMS);
  int64_t grid = mk::cdiv(a->T, block.y);
  const int64_t most = (int64_t)dev->sms * (block.x * block.y < 512 ? 512 / (block.x * block.y) : 1);  // resident at once
  if (grid > most) grid = most;
  return launch<S>(norm_fwd<T, R, V, ITEMS, S>, grid, block, Column<T, R, V, ITEMS, false>::kPieces, 0, s,
                   "mk_block_norm: launch", params<T, R>(a));
}

// Vectors per thread: as few as keep a column within the block's threads.  Up
// to 4096 channels the stages fit an SM's shared memory.
template <typename T, typename R>
int run_fwd(const mk_norm_args* a, const mk::Device* dev, cudaStream_t s) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  if (all_vec(a, V, false)) {
    if (a->D <= 4096) return launch_fwd<T, R, V, 8 / V, sizeof(T) == 2 ? 3 : 2>(a, dev, s);
    return launch_fwd<T, R, V, 16 / V, 1>(a, dev, s);
  }
  return a->D <= 2048 ? launch_fwd<T, R, 1, 4, 1>(a, dev, s) : launch_fwd<T, R, 1, 16, 1>(a, dev, s);
}

// ITEMS vectors of V channels per thread.
struct BwdPlan {
  int V, items;
  dim3 block;
  int64_t grid, parts;
};

BwdPlan plan_bwd(const mk_norm_args* a, const mk::Device* dev) {
  BwdPlan b;
  const int wide = type_bytes(a->type) == 2 ? 8 : 4;
  b.V = all_vec(a, wide, true) ? wide : 1;
  const int64_t n = mk::cdiv(a->D, b.V);
  if (b.V == 8) b.items = n <= 512 ? 1 : 2;
  else if (b.V == 4) b.items = n <= 1024 ? 2 : 4;
  else b.items = n <= 2048 ? 4 : 16;
  b.block = block_of(a->D, b.V, b.items);
  const int64_t columns = mk::cdiv(a->T, b.block.y);
  const int64_t threads = (int64_t)b.block.x * b.block.y;
  const int64_t most = (int64_t)dev->sms * (threads < 512 ? 512 / threads : 1);
  b.grid = columns < most ? columns : most;
  b.parts = b.grid * b.block.y;
  return b;
}

template <typename T, typename R, int V, int ITEMS, int S>
int launch_bwd(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  const Norm<T, R> p = params<T, R>(a);
  if (b.grid)
    MK_TRY(launch<S>(norm_bwd<T, R, V, ITEMS, S>, b.grid, b.block, Column<T, R, V, ITEMS, true>::kPieces,
                     3 * a->D * sizeof(float), s,
                     "mk_block_norm_grad: launch", p));
  norm_fold<<<(unsigned)mk::cdiv(3 * a->D, 32), dim3(32, 8), 0, s>>>(p.parts, b.parts, a->D, a->dw, a->dhw, a->dscale);
  return mk::check_launch("mk_block_norm_grad: launch");
}

template <typename T, typename R>
int run_bwd(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (b.V == 8) return b.items == 1 ? launch_bwd<T, R, 8, 1, 3>(a, b, s) : launch_bwd<T, R, 8, 2, 1>(a, b, s);
  } else {
    if (b.V == 4) return b.items == 2 ? launch_bwd<T, R, 4, 2, 2>(a, b, s) : launch_bwd<T, R, 4, 4, 1>(a, b, s);
  }
  return b.items == 4 ? launch_bwd<T, R, 1, 4, 1>(a, b, s) : launch_bwd<T, R, 1, 16, 1>(a, b, s);
}

int forward(const mk_norm_args* a, void* stream) {
  MK_TRY(check("mk_block_norm", a, false));
  if (a->T == 0) return MK_OK;
  MK_ENTRY_DEVICE(dev);
  cudaStream_t s = mk::as_stream(stream);
  if (a->type == MK_T_F32) return run_fwd<float, float>(a, dev, s);
  if (a->type == MK_T_F16)
    return a->rtype == MK_T_F32 ? run_fwd<__half, float>(a, dev, s) : run_fwd<__half, __half>(a, dev, s);
  return a->rtype == MK_T_F32 ? run_fwd<__nv_bfloat16, float>(a, dev, s)
                              : run_fwd<__nv_bfloat16, __nv_bfloat16>(a, dev, s);
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
  if (need && (!a->workspace || a->workspace_bytes < need || !elem_aligned(a->workspace, 4)))
    return bad(who, "a workspace of " + std::to_string(need) + " bytes is needed");
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
