// block_norm.cu — the norms around a block, fused with the block's gate and
// its scaled residual: per token column of D channels
//     n = h / rms(h) * hw,  m = n * act(gate),  rout = r + scale * m,
//     y = rout / rms(rout) * w,   rms(x) = sqrt(mean(x^2) + eps).
//
// Bound by memory: every matrix is read or written once; a column stays in
// registers between its reductions (V * ITEMS values per thread).  A column
// of up to 32 * V * ITEMS channels is one warp's (shuffles only), wider ones a
// block's.  Backward recomputes the forward values from r, h and gate, which
// costs no more reads than saving rout and its rms would.
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

// Sums of N values over the blockDim.x threads of a column.  A column is one
// warp's, or the whole block's.
template <int N>
__device__ __forceinline__ void column_sum(float (&v)[N], float* sm) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (blockDim.x == 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __syncthreads();  // the last sums are read
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) sm[warp * N + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = lane < warps ? sm[lane * N + i] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  }
}

// act(g), and its derivative
__device__ __forceinline__ float act_of(float g, int act) {
  const float s = sigmoid(g);
  return act == MK_ACT_SILU ? g * s : s;
}
__device__ __forceinline__ void act_grad(float g, int act, float& a, float& da) {
  const float s = sigmoid(g);
  a = act == MK_ACT_SILU ? g * s : s;
  da = act == MK_ACT_SILU ? s * fmaf(g, 1.0f - s, 1.0f) : s * (1.0f - s);
}

template <int V>
__device__ __forceinline__ void fill(float (&f)[V], float x) {
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = x;
}

template <typename T, typename R, int V, int ITEMS>
__global__ void __launch_bounds__(1024, 1) norm_fwd(Norm<T, R> p) {
  __shared__ float sm[32];
  const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (t >= p.T_) return;
  float x[ITEMS][V], h[ITEMS][V], g[ITEMS][V];
  float s[1] = {0.0f};
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
    fill(x[k], 0.0f), fill(h[k], 0.0f), fill(g[k], 0.0f);
    if (d < p.D) {
      load<R, V>(x[k], p.r + t * p.ldr + d);
      if (p.h) load<T, V>(h[k], p.h + t * p.ldh + d);
      if (p.gate) load<T, V>(g[k], p.gate + t * p.ldgate + d);
    }
  }
  if (p.h) {
    float i1 = 1.0f;
    if (p.hw) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s[0] = fmaf(h[k][i], h[k][i], s[0]);
      column_sum<1>(s, sm);
      i1 = rsqrtf(fmaf(s[0], p.inv_d, p.eps));
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      if (d < p.D) {
        float hw[V], sc[V];
        fill(hw, 1.0f), fill(sc, 1.0f);
        if (p.hw) load<float, V>(hw, p.hw + d);
        if (p.scale) load<float, V>(sc, p.scale + d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float m = h[k][i] * i1 * hw[i];
          if (p.gate) m *= act_of(g[k][i], p.act);
          x[k][i] = fmaf(sc[i], m, x[k][i]);
        }
      }
    }
  }
  if (p.rout) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      if (d < p.D) store<R, V>(p.rout + t * p.ldrout + d, x[k]);
    }
  }
  if (!p.y) return;
  s[0] = 0.0f;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) s[0] = fmaf(x[k][i], x[k][i], s[0]);
  column_sum<1>(s, sm);
  const float i2 = rsqrtf(fmaf(s[0], p.inv_d, p.eps));
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
    if (d < p.D) {
      float w[V];
      load<float, V>(w, p.w + d);
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] *= x[k][i] * i2;
      store<T, V>(p.y + t * p.ldy + d, w);
    }
  }
}

// Backward.  With x = rout i2 and dx = dy w:
//   dro = drout + i2 (dx - x mean(dx x)),  dr = dro,
//   dm = dro scale, dn = dm act, dgate = dm n act', dv = dn hw,
//   dh = i1 (dv - v mean(dv v)), v = h i1;
// dw += dy x, dhw += dn v, dscale += dro m.  A block walks columns gridDim.x *
// blockDim.y apart and keeps its sums for w, hw and scale in registers; they
// go to one part per column walker, added up by norm_fold in a fixed order.
template <typename T, typename R, int V, int ITEMS>
__global__ void __launch_bounds__(V * ITEMS <= 8 ? 512 : 1024, 1) norm_bwd(Norm<T, R> p) {
  __shared__ float sm[64];
  const int64_t walker = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  float aw[ITEMS][V], ah[ITEMS][V], as[ITEMS][V];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) fill(aw[k], 0.0f), fill(ah[k], 0.0f), fill(as[k], 0.0f);
  for (int64_t t = walker; t < p.T_; t += (int64_t)gridDim.x * blockDim.y) {
    float x[ITEMS][V], h[ITEMS][V], g[ITEMS][V], dy[ITEMS][V], dro[ITEMS][V];
    float s1[1] = {0.0f}, s2[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      fill(x[k], 0.0f), fill(h[k], 0.0f), fill(g[k], 0.0f), fill(dy[k], 0.0f), fill(dro[k], 0.0f);
      if (d < p.D) {
        load<R, V>(x[k], p.r + t * p.ldr + d);
        if (p.h) load<T, V>(h[k], p.h + t * p.ldh + d);
        if (p.gate) load<T, V>(g[k], p.gate + t * p.ldgate + d);
        if (p.dy) load<T, V>(dy[k], p.dy + t * p.lddy + d);
        if (p.drout) load<R, V>(dro[k], p.drout + t * p.lddrout + d);
      }
    }
    float i1 = 1.0f;
    if (p.h && p.hw) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) s1[0] = fmaf(h[k][i], h[k][i], s1[0]);
      column_sum<1>(s1, sm);
      i1 = rsqrtf(fmaf(s1[0], p.inv_d, p.eps));
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      if (d < p.D) {
        float hw[V], sc[V], w[V];
        fill(hw, 1.0f), fill(sc, 1.0f), fill(w, 1.0f);
        if (p.hw) load<float, V>(hw, p.hw + d);
        if (p.scale) load<float, V>(sc, p.scale + d);
        if (p.dy) load<float, V>(w, p.w + d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float m = h[k][i] * i1 * hw[i];
          if (p.gate) m *= act_of(g[k][i], p.act);
          if (p.h) x[k][i] = fmaf(sc[i], m, x[k][i]);
          s2[0] = fmaf(x[k][i], x[k][i], s2[0]);
          s2[1] = fmaf(dy[k][i] * w[i], x[k][i], s2[1]);
        }
      }
    }
    float i2 = 0.0f, mean = 0.0f;
    if (p.dy) {
      column_sum<2>(s2, sm);
      i2 = rsqrtf(fmaf(s2[0], p.inv_d, p.eps));
      mean = s2[1] * i2 * p.inv_d;
    }
    s1[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
      if (d < p.D) {
        float hw[V], sc[V], w[V];
        fill(hw, 1.0f), fill(sc, 1.0f), fill(w, 1.0f);
        if (p.hw) load<float, V>(hw, p.hw + d);
        if (p.scale) load<float, V>(sc, p.scale + d);
        if (p.dy) load<float, V>(w, p.w + d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float xh = x[k][i] * i2;
          if (p.dy) {
            aw[k][i] = fmaf(dy[k][i], xh, aw[k][i]);
            dro[k][i] += i2 * (dy[k][i] * w[i] - xh * mean);
          }
          const float v = h[k][i] * i1, n = v * hw[i], dm = dro[k][i] * sc[i];
          float a = 1.0f, da = 0.0f;
          if (p.gate) act_grad(g[k][i], p.act, a, da);
          as[k][i] = fmaf(dro[k][i], n * a, as[k][i]);
          g[k][i] = dm * n * da;
          const float dn = dm * a;
          ah[k][i] = fmaf(dn, v, ah[k][i]);
          dy[k][i] = dn * hw[i];  // from here: the gradient of v
          s1[0] = fmaf(dy[k][i], v, s1[0]);
        }
        store<R, V>(p.dr + t * p.lddr + d, dro[k]);
        if (p.gate) store<T, V>(p.dgate + t * p.lddgate + d, g[k]);
      }
    }
    if (p.h) {
      float back = 0.0f;
      if (p.hw) {
        column_sum<1>(s1, sm);
        back = s1[0] * p.inv_d * i1;
      }
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
        if (d < p.D) {
#pragma unroll
          for (int i = 0; i < V; ++i) h[k][i] = i1 * fmaf(-h[k][i], back, dy[k][i]);
          store<T, V>(p.dh + t * p.lddh + d, h[k]);
        }
      }
    }
  }
  float* part = p.parts + walker * 3 * p.D;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t d = ((int64_t)k * blockDim.x + threadIdx.x) * V;
    if (d < p.D) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        part[d + i] = aw[k][i];
        part[p.D + d + i] = ah[k][i];
        part[2 * p.D + d + i] = as[k][i];
      }
    }
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

template <typename T, typename R, int V, int ITEMS>
int launch_fwd(const mk_norm_args* a, cudaStream_t s) {
  const dim3 block = block_of(a->D, V, ITEMS);
  norm_fwd<T, R, V, ITEMS><<<(unsigned)mk::cdiv(a->T, block.y), block, 0, s>>>(params<T, R>(a));
  return mk::check_launch("mk_block_norm: launch");
}

// Vectors per thread: as few as keep a column within the block's threads.
template <typename T, typename R>
int run_fwd(const mk_norm_args* a, cudaStream_t s) {
  constexpr int V = sizeof(T) == 2 ? 8 : 4;
  if (all_vec(a, V, false)) {
    const int64_t n = mk::cdiv(a->D, V);
    return n <= 256 ? launch_fwd<T, R, V, 1>(a, s) : launch_fwd<T, R, V, 16 / V>(a, s);
  }
  return a->D <= 4096 ? launch_fwd<T, R, 1, 4>(a, s) : launch_fwd<T, R, 1, 16>(a, s);
}

struct BwdPlan {
  int V, items;
  dim3 block;
  int64_t grid, parts;
};

BwdPlan plan_bwd(const mk_norm_args* a, const mk::Device* dev) {
  BwdPlan b;
  b.V = all_vec(a, 4, true) ? 4 : 1;
  const int64_t n = mk::cdiv(a->D, b.V);
  if (b.V == 4) b.items = n <= 1024 ? 2 : 4;
  else b.items = n <= 2048 ? 4 : 16;
  b.block = block_of(a->D, b.V, b.items);
  const int64_t columns = mk::cdiv(a->T, b.block.y);
  const int64_t threads = (int64_t)b.block.x * b.block.y;
  const int64_t most = (int64_t)dev->sms * (threads <= 512 ? 1024 / threads : 1);
  b.grid = columns < most ? columns : most;
  b.parts = b.grid * b.block.y;
  return b;
}

template <typename T, typename R, int V, int ITEMS>
int launch_bwd(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  const Norm<T, R> p = params<T, R>(a);
  if (b.grid) norm_bwd<T, R, V, ITEMS><<<(unsigned)b.grid, b.block, 0, s>>>(p);
  norm_fold<<<(unsigned)mk::cdiv(3 * a->D, 32), dim3(32, 8), 0, s>>>(p.parts, b.parts, a->D, a->dw, a->dhw, a->dscale);
  return mk::check_launch("mk_block_norm_grad: launch");
}

template <typename T, typename R>
int run_bwd(const mk_norm_args* a, const BwdPlan& b, cudaStream_t s) {
  if (b.V == 4) return b.items == 2 ? launch_bwd<T, R, 4, 2>(a, b, s) : launch_bwd<T, R, 4, 4>(a, b, s);
  return b.items == 4 ? launch_bwd<T, R, 1, 4>(a, b, s) : launch_bwd<T, R, 1, 16>(a, b, s);
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
  return a->rtype == MK_T_F32 ? run_fwd<__nv_bfloat16, float>(a, s) : run_fwd<__nv_bfloat16, __nv_bfloat16>(a, s);
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
