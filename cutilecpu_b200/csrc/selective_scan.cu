// selective_scan.cu — entry points of the selective scan (kernels:
// selective_scan.cuh) and its form for single tokens.
#include "selective_scan.cuh"

namespace {

using namespace mk::tok;
using namespace mk::scan;

// One token per batch entry.  Bound by the state: read and written once, 16
// bytes per lane and channel, P lanes per channel in memory order.  A thread
// takes IT channels, so that as many states are in flight and one read of B
// and C serves them all; with IT == P each of the P lanes also computes what
// one of those channels needs once (softplus, gate), and passes it round.  192
// entries of 4096 channels with 16 states: 24.2 us, 4.2 TB/s, with states that are
// not in L2 (as between two tokens of a model), 21.0 us where the call before has
// left part of them there.  Each block waits in turn for its slot, its inputs
// and its states (3.1 of an issue's 9 cycles are waits on global loads, 71% of the
// issue slots are used), and 3 us go into the start and the end of the launch.
template <typename T>
struct Step {
  int64_t D, N, G, Dg, B, nslots, tiles, tpg;  // channel tiles, and of one group
  const T *u, *delta, *z, *Bm, *Cm;
  int64_t ldu, lddelta, ldz, ldb, ldc, ldy;
  const float *A, *Dskip, *bias, *state;
  float* next;
  T* y;
  const int32_t* slots;
  int softplus;
  unsigned* err;
};

__device__ __forceinline__ void load4(float (&h)[4], const float* at, int n0, int N) {
  if (N % 4 == 0) {
    const float4 v = n0 < N ? *reinterpret_cast<const float4*>(at + n0) : make_float4(0, 0, 0, 0);
    h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = n0 + j < N ? at[n0 + j] : 0.0f;
  }
}

__device__ __forceinline__ void store4(float* at, const float (&h)[4], int n0, int N) {
  if (N % 4 == 0) {
    if (n0 < N) *reinterpret_cast<float4*>(at + n0) = make_float4(h[0], h[1], h[2], h[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n0 + j < N) at[n0 + j] = h[j];
  }
}

template <typename T, int P, int IT>
__global__ void __launch_bounds__(128) scan_step(Step<T> p) {
  static_assert(IT == 1 || IT == P, "a channel per lane, or one for all");
  constexpr bool kExact = sizeof(T) == 4;
  constexpr int kChannels = 128 / P;  // a block's channels at a time
  const int64_t e = blockIdx.x / p.tiles;
  const int tile = blockIdx.x % p.tiles, g = tile / p.tpg, lane = threadIdx.x % P;
  const int first = tile % p.tpg * (kChannels * IT) + threadIdx.x / P, base = g * (int)p.Dg;
  const int N = (int)p.N, n0 = lane * 4;  // D * N stays below 2^26
  if (tile == 0) check_distinct(p.slots, e, threadIdx.x, 128, p.err);
  const int64_t row = slot_of(p.slots, p.nslots, e, p.err);
  if (row < 0) return;
  const float* state = p.state + row * p.D * N;
  float* next = p.next + row * p.D * N;
  float h[IT][4], A[IT][4], b[4], c[4];
  int d[IT];
  bool live[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    live[i] = first + i * kChannels < p.Dg;
    d[i] = base + (live[i] ? first + i * kChannels : 0);
    load4(h[i], state + d[i] * N, n0, N);
  }
  // this lane's own channel: what it needs once
  int own = d[0];
  bool own_live = live[0];
#pragma unroll
  for (int i = 1; i < IT; ++i) own = lane == i ? d[i] : own, own_live = lane == i ? live[i] : own_live;
  const float u = to_f(p.u[e * p.ldu + own]);
  float dt = to_f(p.delta[e * p.lddelta + own]) + (p.bias ? p.bias[own] : 0.0f);
  const float z = p.z ? to_f(p.z[e * p.ldz + own]) : 0.0f, skip = p.Dskip ? p.Dskip[own] : 0.0f;
#pragma unroll
  for (int i = 0; i < IT; ++i) load4(A[i], p.A + d[i] * N, n0, N);
  const T *Bm = p.Bm + e * p.ldb + g * N, *Cm = p.Cm + e * p.ldc + g * N;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[j] = n0 + j < N ? to_f(Bm[n0 + j]) : 0.0f;
    c[j] = n0 + j < N ? to_f(Cm[n0 + j]) : 0.0f;
  }
  if (p.softplus) dt = softplus<kExact>(dt);
  const float dtu = dt * u;
  float y[IT], sum[1];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const float dt_i = IT > 1 ? __shfl_sync(0xffffffffu, dt, i, P) : dt;
    const float dtu_i = IT > 1 ? __shfl_sync(0xffffffffu, dtu, i, P) : dtu;
    y[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[i][j] = fmaf(decay(dt_i, rate(A[i][j])), h[i][j], dtu_i * b[j]);
      y[i] = fmaf(c[j], h[i][j], y[i]);
    }
    if (live[i]) store4(next + d[i] * N, h[i], n0, N);
  }
  if constexpr (IT > 1) {
    reduce_scatter<IT, P, 1>(y, lane, sum);
  } else {
    sum[0] = y[0];
#pragma unroll
    for (int bit = 1; bit < P; bit *= 2) sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], bit);
  }
  if (!own_live || (IT == 1 && lane != 0)) return;
  float out = fmaf(skip, u, sum[0]);
  if (p.z) out *= z * sigmoid<kExact>(z);
  p.y[e * p.ldy + own] = from_f<T>(out);
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
  if (a->len < 0 || (!a->seqs && ((a->nseq && a->len > a->T) || a->nseq * a->len != a->T)))
    return bad(who, "nseq * len is not T");
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
  MK_TRY(check_slots(who, a->slots, a->nslots, a->nseq));
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

// Whole sequences or pieces, and the channels per lane (times: B200, bf16, 16
// states; `fill`: blocks of whole sequences over the four that an SM holds).
//
// Forward, cutting costs a second pass of exponentials: it pays below a third
// of a fill (1 x 16384 tokens of 640 channels 829 -> 134 us, 3 x 5461 of 2048 at
// 0.32 396 -> 379 us; 6 x 2730 of 1536 at 0.49 would be 204 -> 300 us).
// Backward the extra pass is a seventh of the work, and more and shorter blocks
// even out the end: up to 3/4 of a fill for equal lengths (4 x 2048 of 2048
// channels 670 -> 499 us, of 4096 at 0.86 916 -> 978 us).  With offsets the
// lengths are the device's, and one that is long takes the whole sequences'
// time: up to 3/2 (96, 1000, 3000 and 4096 tokens of 4096 channels 1659 -> 974 us,
// 4 x 2048 of 6144 at 1.3 1548 -> 1365 us, against the 62 us lost at 0.86).
// Eight blocks per SM, two rounds, measured best among 4 to 16.
//
// Channels per lane, forward: one (two: 262 -> 270 us).  Backward: two halve what
// is read from shared memory and reduced over channels, but also the warps: 1017
// -> 916 us for 4 x 2048 tokens of 4096 channels, 827 -> 922 us of 2560.  So two
// from 1.5 of their blocks per SM on, and in pieces where the blocks that an SM
// holds (two) get 512 tokens each (4 x 2048 of 2048 457 -> 417 us; 1 x 8192 of
// 1024, 443 tokens, 235 -> 254 us).  Single elements take registers that two
// channels need (4 x 2048 x 4095 1273 -> 1302 us), and so does Float32 beside 2
// states per lane (8 states, 4 x 2048 tokens of 4096 channels whole 825 -> 1060 us,
// 16 x 1024 1439 -> 1729; in bf16 two win there, 771 -> 750 us, and in Float32
// with 16 states, 1189 -> 1073): one.
Plan plan(const mk_scan_args* a, const mk::Device* dev, bool grad) {
  Plan b{};
  const int64_t Dg = a->D / a->G, sms = dev->sms, CB = kWarps * (32 / lanes_of(a->N));
  b.rev_tpg = mk::cdiv(Dg, CB);
  b.rev_tiles = a->G * b.rev_tpg;
  const int64_t have = b.rev_tiles * a->nseq, twice = a->G * mk::cdiv(Dg, 2 * CB);
  const bool cut = have > 0 && a->T >= a->nseq * 4 * kTS &&
                   (grad ? have <= sms * (a->seqs ? 6 : 3) : have * 3 <= 4 * sms);
  b.ch = 1;
  if (grad && two_channels(states_of(a->N), type_bytes(a->type)) && all_vec(a, true)) {
    const bool enough = cut ? twice * a->T >= 2 * sms * 512 : 2 * twice * a->nseq >= 3 * sms;
    if (enough) b.ch = 2;
  }
  b.tpg = mk::cdiv(Dg, CB * b.ch);
  b.tiles = a->G * b.tpg;
  b.items = a->nseq;
  if (cut) {
    const int64_t pieces = mk::cdiv(8 * sms, b.tiles);  // over all sequences
    const int64_t piece = mk::cdiv(mk::cdiv(a->T, pieces), kTS) * kTS;
    b.piece = piece < 2 * kTS ? 2 * kTS : piece;
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

int run_scan(const char* who, const mk_scan_args* a, bool grad, void* stream) {
  MK_TRY(check_scan(who, a, grad));
  if (a->nseq == 0 && !grad) return MK_OK;
  MK_ENTRY_DEVICE(dev);
  const Plan b = plan(a, dev, grad);
  if (b.rev_tiles * b.items > INT32_MAX) return bad(who, "too many sequences for these channels");
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

template <typename T, int P>
int launch_step(Step<T> p, const mk::Device* dev, cudaStream_t s) {
  // P channels per thread (up to 8): at 192 entries of 4096 channels and 16 states, states not in L2, 47.6 -> 25.1 us,
  // at 16 entries 6.9 -> 5.3; one where fewer than two blocks per SM would be left (8 entries: 4.5 -> 4.4 us, 1 entry 3.9 -> 3.7)
  constexpr int IT = P <= 8 ? P : 1;
  const int64_t few = p.G * mk::cdiv(p.Dg, IT * (128 / P));
  const bool wide = few * p.B >= 2 * (int64_t)dev->sms;
  p.tpg = wide ? few / p.G : mk::cdiv(p.Dg, 128 / P);
  p.tiles = p.G * p.tpg;
  const unsigned grid = (unsigned)(p.B * p.tiles);
  if (wide) scan_step<T, P, IT><<<grid, 128, 0, s>>>(p);
  else scan_step<T, P, 1><<<grid, 128, 0, s>>>(p);
  return mk::check_launch("mk_selective_scan_step: launch");
}

template <typename T>
int run_step(const mk_scan_step_args* a, const mk::Device* dev, cudaStream_t s) {
  Step<T> p{};
  p.D = a->D, p.N = a->N, p.G = a->G, p.Dg = a->D / a->G, p.B = a->B, p.nslots = a->nslots;
  p.u = static_cast<const T*>(a->u), p.ldu = a->ldu;
  p.delta = static_cast<const T*>(a->delta), p.lddelta = a->lddelta;
  p.z = static_cast<const T*>(a->z), p.ldz = a->ldz;
  p.Bm = static_cast<const T*>(a->Bmat), p.ldb = a->ldb;
  p.Cm = static_cast<const T*>(a->Cmat), p.ldc = a->ldc;
  p.y = static_cast<T*>(a->y), p.ldy = a->ldy;
  p.A = a->A, p.Dskip = a->Dskip, p.bias = a->bias, p.state = a->state, p.next = a->next;
  p.slots = a->slots, p.softplus = a->softplus, p.err = dev->err_word;
  if (a->N <= 4) return launch_step<T, 1>(p, dev, s);
  if (a->N <= 8) return launch_step<T, 2>(p, dev, s);
  if (a->N <= 16) return launch_step<T, 4>(p, dev, s);
  return a->N <= 32 ? launch_step<T, 8>(p, dev, s) : launch_step<T, 16>(p, dev, s);
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
  MK_TRY(check_slots(who, a->slots, a->nslots, a->B));
  if (!some) return MK_OK;
  if (a->B * (mk::cdiv(a->D, 8) + a->G) > INT32_MAX) return bad(who, "batch too large for these channels");
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
