// tokens.cuh — shared by the kernels over token columns (causal_conv.cu,
// selective_scan.cu, block_norm.cu): element types, the packed sequences of a
// (channels, tokens) matrix, and the scalar functions of their formulas.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "mk_common.cuh"

namespace mk {
namespace tok {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// V neighbouring elements as one access, or as several of 16 bytes.
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vec { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void load(float (&f)[V], const T* p) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f(v.v[i]);
}

// r = *p where `on`, else r stays.  A predicated load that stays where it is
// written: as an ordinary conditional load the compiler may move it down to its
// use, behind the work that it is to overlap with, or join it with the value
// for !on by a move that waits for it on the spot.
template <typename X>
__device__ __forceinline__ void load_if(X& r, const X* p, bool on) {
  const unsigned q = on;
  if constexpr (sizeof(X) == 16) {
    uint4 v;
    memcpy(&v, &r, 16);
    asm volatile("{ .reg .pred q; setp.ne.u32 q, %5, 0; @q ld.global.v4.u32 {%0, %1, %2, %3}, [%4]; }"
                 : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
                 : "l"(p), "r"(q));
    memcpy(&r, &v, 16);
  } else if constexpr (sizeof(X) == 8) {
    uint2 v;
    memcpy(&v, &r, 8);
    asm volatile("{ .reg .pred q; setp.ne.u32 q, %3, 0; @q ld.global.v2.u32 {%0, %1}, [%2]; }"
                 : "+r"(v.x), "+r"(v.y)
                 : "l"(p), "r"(q));
    memcpy(&r, &v, 8);
  } else if constexpr (sizeof(X) == 4) {
    unsigned v;
    memcpy(&v, &r, 4);
    asm volatile("{ .reg .pred q; setp.ne.u32 q, %2, 0; @q ld.global.u32 %0, [%1]; }" : "+r"(v) : "l"(p), "r"(q));
    memcpy(&r, &v, 4);
  } else {
    static_assert(sizeof(X) == 2, "no such vector");
    unsigned short v;
    memcpy(&v, &r, 2);
    asm volatile("{ .reg .pred q; setp.ne.u32 q, %2, 0; @q ld.global.u16 %0, [%1]; }" : "+h"(v) : "l"(p), "r"(q));
    memcpy(&r, &v, 2);
  }
}

// Asynchronous copies into shared memory (4, 8 or 16 bytes): loads that cost no
// registers while they are in flight.  The users below copy and read back per
// thread, so they wait for their own groups of copies and need no barrier.
template <int BYTES>
__device__ __forceinline__ void copy_if(void* smem, const void* p, bool on) {
  const unsigned to = (unsigned)__cvta_generic_to_shared(smem), q = on;
  if constexpr (BYTES == 16) {
    asm volatile("{ .reg .pred q; setp.ne.u32 q, %2, 0; @q cp.async.cg.shared.global [%0], [%1], 16; }" ::"r"(to),
                 "l"(p), "r"(q)
                 : "memory");
  } else {
    asm volatile("{ .reg .pred q; setp.ne.u32 q, %2, 0; @q cp.async.ca.shared.global [%0], [%1], %3; }" ::"r"(to),
                 "l"(p), "r"(q), "n"(BYTES)
                 : "memory");
  }
}
// 16 bytes of shared memory, read where it is written (not kept in registers from an earlier read).
__device__ __forceinline__ uint4 read_shared(const uint4* p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"((unsigned)__cvta_generic_to_shared(p)));
  return v;
}
// 16 bytes, or zeros where not `on` (p is an address that may be read all the same).
__device__ __forceinline__ void copy_or_zero(void* smem, const void* p, bool on) {
  const unsigned to = (unsigned)__cvta_generic_to_shared(smem), bytes = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v.v[i] = from_f<T>(f[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = v;
}

// Packed sequences.  With `seqs` sequence s has the columns
// [seqs[s] - 1, seqs[s + 1] - 1) (1-based offsets, as Julia ranges start);
// without it every sequence has `len` columns.  Offsets live on the device,
// so they are read defensively: a sequence that does not lie inside the T
// columns, or ends before it begins, counts as empty and sets `bad`.
struct Seqs {
  const int32_t* seqs;
  int64_t nseq, len, T;
};

struct Span {
  int64_t lo, hi;
  bool bad;
};

__device__ __forceinline__ int64_t seq_offset(const Seqs& q, int64_t s) {
  if (!q.seqs) return s * q.len;
  int64_t o = (int64_t)q.seqs[s] - 1;
  return o < 0 ? 0 : (o > q.T ? q.T : o);
}

__device__ __forceinline__ Span seq_span(const Seqs& q, int64_t s) {
  if (!q.seqs) return {s * q.len, (s + 1) * q.len, false};
  const int64_t lo = (int64_t)q.seqs[s] - 1, hi = (int64_t)q.seqs[s + 1] - 1;
  const bool bad = lo < 0 || hi > q.T || hi < lo;
  const int64_t at = lo < 0 ? 0 : (lo > q.T ? q.T : lo);
  return {at, bad ? at : hi, bad};
}

// The last sequence that begins at or before column t (the first, if none
// does), found by a whole warp: 32 offsets are looked at in one round.
__device__ __forceinline__ int64_t seq_at(const Seqs& q, int64_t t) {
  if (!q.seqs) {
    const int64_t s = q.len ? t / q.len : q.nseq - 1;
    return s < q.nseq ? s : q.nseq - 1;
  }
  int64_t lo = 0, count = q.nseq;
  while (count > 1) {
    const int64_t step = (count + 31) / 32, at = (threadIdx.x & 31) * step;
    const unsigned hit = __ballot_sync(0xffffffffu, at < count && seq_offset(q, lo + at) <= t);
    const int c = __popc(hit);
    const int64_t skip = c ? (c - 1) * step : 0;
    lo += skip;
    count = count - skip < step ? count - skip : step;
  }
  return lo;
}

// A sequence cut into pieces of `piece` columns (the last one shorter): piece
// c of sequence s has the number lo(s) / piece + s + c.  The numbers of
// sequence s + 1 begin behind those of s, because floor(a + b) >= floor(a) +
// floor(b); all lie below T / piece + nseq, so no prefix sum over the
// sequences is needed to place per-piece state.
__device__ __forceinline__ int64_t first_piece(const Seqs& q, int64_t s, int64_t piece) {
  return seq_offset(q, s) / piece + s;
}

// The sequence that piece number `i` falls to (the last s with first_piece <= i;
// the first sequence, if none, when columns in front of it belong to no sequence).
__device__ __forceinline__ int64_t seq_of_piece(const Seqs& q, int64_t i, int64_t piece) {
  int64_t lo = 0, hi = q.nseq - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (first_piece(q, mid, piece) <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Row of the state pool that entry i uses: slots[i] - 1, or i without slots.
// -1: none (slots[i] <= 0); a slot above nslots counts as none and is flagged.
__device__ __forceinline__ int64_t slot_of(const int32_t* slots, int64_t nslots, int64_t i, unsigned* err) {
  if (!slots) return i;
  const int64_t k = (int64_t)slots[i] - 1;
  if (k >= nslots) {
    atomicOr(err, ERRBIT_SLOT);
    return -1;
  }
  return k < 0 ? -1 : k;
}

// Two entries of one call on one slot would race on its state: entry i is
// compared with those before it by the `nt` threads of a block (the caller
// picks one block per entry), and a repeat is flagged.
__device__ __forceinline__ void check_distinct(const int32_t* slots, int64_t i, int tid, int nt, unsigned* err) {
  if (!slots || slots[i] <= 0) return;
  const int32_t mine = slots[i];
  bool twice = false;
  for (int64_t j = tid; j < i; j += nt) twice |= slots[j] == mine;
  if (twice) atomicOr(err, ERRBIT_SLOT);
}

// Each entry is compared with all before it, which bounds their number.
constexpr int64_t kMostSlotted = 1 << 20;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLow = 1.92596299e-8f;  // log2(e) - kLog2e
constexpr float kLn2 = 0.69314718055994530942f;

// 2^x by the special function unit (relative error about 2^-22).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two Float32 values in a register pair, and the packed operations on them:
// one issue slot for two results.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 pack(float a) { return pack(a, a); }
__device__ __forceinline__ void unpack(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 ex2_2(F2 x) {
  float a, b;
  unpack(x, a, b);
  return pack(ex2(a), ex2(b));
}
__device__ __forceinline__ float sum2(F2 x) {
  float a, b;
  unpack(x, a, b);
  return a + b;
}

// exp(dt A) with A2 = A log2(e).  ex2.approx errs low by 2e-8 on average for
// exponents down to -0.25 (measured against 64 bits), and a slow decay adds
// that up over its memory of hundreds of tokens: the exponent gets it back, in
// the same instruction.  A step of dt = 0 still gives exactly 1.
constexpr float kDecayBias = 3.0e-8f;
// A log2(e) of a pair; an infinite rate as the largest finite one, whose product
// with a step of 0 is 0 (a state beyond its sequence's end stays).
__device__ __forceinline__ float rate(float A) {
  const float x = A * kLog2e;
  return x < -FLT_MAX ? -FLT_MAX : x;
}
__device__ __forceinline__ F2 rate2(F2 A) {
  float a, b;
  unpack(A, a, b);
  return pack(rate(a), rate(b));
}
__device__ __forceinline__ float decay(float dt, float A2) { return ex2(fmaf(dt, A2, kDecayBias)); }
__device__ __forceinline__ F2 decay2(F2 dt, F2 A2) { return ex2_2(fma2(dt, A2, pack(kDecayBias))); }

// A pair as two neighbouring elements.
__device__ __forceinline__ void from_f2(float* p, F2 x) { unpack(x, p[0], p[1]); }
__device__ __forceinline__ void from_f2(__half* p, F2 x) {
  float a, b;
  unpack(x, a, b);
  const __half2 h = __floats2half2_rn(a, b);
  p[0] = h.x, p[1] = h.y;
}
__device__ __forceinline__ void from_f2(__nv_bfloat16* p, F2 x) {
  float a, b;
  unpack(x, a, b);
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  p[0] = h.x, p[1] = h.y;
}

// e^x for the elementwise functions.  The rounding of x log2(e) costs |x| 2^-24
// of the result, which is below what 16-bit inputs bring; Float32 inputs get
// the product's rounding error back (EXACT) where e^x is finite: multiplied into
// an infinite one (from 2^128 on) the correction would make it NaN.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) {
  const float t = x * kLog2e;
  const float e = ex2(t);
  if constexpr (!EXACT) return e;
  const float r = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -t));
  return fabsf(t) < 128.0f ? fmaf(e, r * kLn2, e) : e;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool EXACT = true>
__device__ __forceinline__ float sigmoid(float x) { return rcp(1.0f + exp_of<EXACT>(-x)); }

// log(1 + e^x) = max(x, 0) + log1p(e), e = e^-|x| in (0, 1].  log1p(e) = e P(e)
// with P of degree 8 fitted to log1p(e) / e on [0, 1] for the least relative
// error (Remez exchange in 64 bits; 3e-8), so small steps (large negative x)
// keep full precision, which log(1 + e) in 32 bits loses.  With GRAD also the
// derivative 1 / (1 + e^-x), from the same e.
__device__ __forceinline__ constexpr float log1p_term(int i) {
  constexpr float c[9] = {9.999999404e-01f, -4.999949336e-01f, 3.331909776e-01f, -2.484298199e-01f,
                          1.910600662e-01f, -1.366324574e-01f, 7.822595537e-02f, -2.950523980e-02f,
                          5.232694093e-03f};
  return c[i];
}
template <bool EXACT = true>
__device__ __forceinline__ float softplus(float x) {
  const float e = exp_of<EXACT>(-fabsf(x));
  float p = log1p_term(8);
#pragma unroll
  for (int i = 7; i >= 0; --i) p = fmaf(p, e, log1p_term(i));
  return fmaf(p, e, fmaxf(x, 0.0f)) + (x != x ? x : 0.0f);
}
template <bool EXACT, bool GRAD = false>
__device__ __forceinline__ F2 softplus2(F2 x, F2* grad = nullptr) {
  float a, b;
  unpack(x, a, b);
  const float ea = exp_of<EXACT>(-fabsf(a)), eb = exp_of<EXACT>(-fabsf(b));
  const F2 e = pack(ea, eb);
  F2 p = pack(log1p_term(8));
#pragma unroll
  for (int i = 7; i >= 0; --i) p = fma2(p, e, pack(log1p_term(i)));
  if constexpr (GRAD) {
    const float ra = rcp(1.0f + ea), rb = rcp(1.0f + eb);
    *grad = pack(a < 0.0f ? ea * ra : ra, b < 0.0f ? eb * rb : rb);
  }
  return fma2(p, e, pack(fmaxf(a, 0.0f), fmaxf(b, 0.0f)));
}

// The sums of v[0 .. K) over the R <= K lanes that differ in r (lane distance
// STRIDE), scattered: lane r ends with the sums of values e * R + r (out[e]).
// Each stage sends half of what is left, so 8 sums over 8 lanes take 7
// shuffles instead of 24.  The order of the additions is fixed.
template <int K, int R, int STRIDE>
__device__ __forceinline__ void reduce_scatter(float (&v)[K], int r, float (&out)[K / R]) {
  constexpr int E = K / R;
#pragma unroll
  for (int bit = R / 2; bit >= 1; bit /= 2) {
    const bool up = (r & bit) != 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int q = 0; q < bit; ++q) {
        const float lo = v[e * R + q], hi = v[e * R + bit + q];
        const float keep = up ? hi : lo, send = up ? lo : hi;
        v[e * R + q] = keep + __shfl_xor_sync(0xffffffffu, send, bit * STRIDE);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = v[e * R];
}

// Runs a C entry point's body: no C++ exception leaves it.
template <typename F>
inline int guarded(F&& f) {
  try {
    return f();
  } catch (...) {
    return MK_ERR_INVALID;
  }
}

inline size_t type_bytes(int type) { return type == MK_T_F32 ? 4 : 2; }

// Host-side checks shared by the entry points.
inline bool elem_aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Whether a matrix at p with this leading dimension can be read V elements of es bytes at a time.
inline bool vec_ok(const void* p, int64_t ld, size_t es, int V) {
  const int64_t n = (int64_t)es * V < 16 ? (int64_t)es * V : 16;
  return reinterpret_cast<uintptr_t>(p) % n == 0 && (ld * (int64_t)es) % n == 0;
}

inline int bad(const char* who, const std::string& what) {
  return fail(MK_ERR_INVALID, std::string(who) + ": " + what);
}

// A matrix of `cols` columns of `rows` elements: there where it has elements, aligned, ld >= rows.
inline int check_matrix(const char* who, const char* name, const void* p, int64_t rows, int64_t ld, int64_t cols,
                        size_t es) {
  if (cols == 0) return MK_OK;
  if (!p) return bad(who, std::string(name) + " is null");
  if (ld < rows) return bad(who, std::string(name) + " has a leading dimension below its rows");
  if (!elem_aligned(p, es)) return bad(who, std::string(name) + " is not element-aligned");
  return MK_OK;
}

inline int check_slots(const char* who, const int32_t* slots, int64_t nslots, int64_t entries) {
  if (!slots) return MK_OK;
  if (nslots < 0) return bad(who, "negative number of slots");
  return entries > kMostSlotted ? bad(who, "more than 2^20 entries with slots") : MK_OK;
}

// Float32 parameters and states; `vec`: read as 16-byte vectors.
inline int check_floats(const char* who, const char* name, const void* p, bool required, bool vec) {
  if (!p) return required ? bad(who, std::string(name) + " is null") : MK_OK;
  if (!elem_aligned(p, vec ? 16 : 4))
    return bad(who, std::string(name) + (vec ? " is not 16-byte aligned" : " is not 4-byte aligned"));
  return MK_OK;
}

}  // namespace tok
}  // namespace mk

#define MK_TRY(x)                 \
  do {                            \
    const int rc_ = (x);          \
    if (rc_ != MK_OK) return rc_; \
  } while (0)
