// The end of a transformer block with norms on both sides of it, in one pass:
//
//   p = x * rx * w_post            rx = 1 / sqrt(mean(x^2) + eps)    post-norm of the block's output
//   s = a * residual + gate * p    the next residual stream (a: the residual scale)
//   h = s * rs * w_pre             rs = 1 / sqrt(mean(s^2) + eps)    pre-norm of the next block
//
// Backward, from dh and ds (m = mean over the row):
//
//   u = dh w_pre;  S = ds + rs u - s rs^3 m(u s);   dresidual = a S
//   v = S gate w_post;  dx = rx v - x rx^3 m(v x)
//   dw_pre = sum dh s rs;  with A = sum over the rows of one gate row of S x rx:
//   dgate = w_post A,  dw_post = sum over the gate rows of gate A
//
// so the gate's and the post-norm's weight gradients come from one sum.  s is
// formed again in float32 from x and the residual (as many bytes as reading a
// stored s, and exact); rx and rs are kept from the forward (8 bytes a row).
// All arithmetic is float32, each result rounded once.  HBM bounds it: the
// forward reads two rows and writes two, the backward reads four and writes
// two.
#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace ats {
namespace {

constexpr int kMaxThreads = 1024;

enum Gate { GATE_NONE = 0, GATE_SPAN = 1, GATE_ROW = 2 };  // a gate row per span of rows, or per row

struct NormArgs {
  const void *x, *res, *dh, *ds;  // inputs [rows, H] (dh, ds: backward, may be null)
  void *h, *s, *dx, *dres;        // outputs
  const void *w_post, *w_pre, *gate;
  int w_bf16, gate_bf16;
  void* dgate;        // GATE_ROW: [rows, H] in the gate's type
  float *rx, *rs;     // [rows]
  float *part_a, *part_b;
  int64_t rows, span;  // rows that share a gate row
  int H;
  float scale, eps;
  int units_per_span;  // backward: blocks' row ranges per span
  int64_t units;
};

__device__ __forceinline__ float load_as(const void* p, int64_t i, int is_bf16) {
  return is_bf16 ? __bfloat162float(static_cast<const bf16*>(p)[i]) : static_cast<const float*>(p)[i];
}

__device__ __forceinline__ float gate_at(const NormArgs& p, int gate, int64_t row, int c) {
  if (gate == GATE_NONE) return 1.0f;
  return load_as(p.gate, (gate == GATE_ROW ? row : row / p.span) * p.H + c, p.gate_bf16);
}

// Sum over the block; `red` holds a slot per warp and is safe to reuse after the next call on the other buffer.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
  return t;
}

// ------------------------------------------------------------ rows in registers
// One block walks a run of consecutive rows; a thread owns NV vectors of VB bytes of every row, so its sums over rows
// stay in its registers, and its columns of the weights (and of the gate, per span) in its own places of shared
// memory.  Each thread copies its own pieces of the rows ahead into its own slots of shared memory (cp.async), STAGES
// rows deep: no thread reads another's, so the only barriers are the two row sums.  Two blocks share an SM where their
// registers allow it, so that one's barrier waits pass under the other's arithmetic.  16384 x 4096 bf16 with a gate per
// channel: forward 91 us, backward 146 us with its sums (90% and 84% of the measured copy bandwidth); with the weights
// in registers, one block to an SM and a plain reading of the formulas 100 and 179 us.
//
// Per column, with xr = x rx, t = s rs, and gw = gate w_post:
//   s = a res + gw xr;  u = dh w_pre;  S = ds + rs u - t rs m(u t);  dx = rx (gw S - xr m(gw S xr))
template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

// Copy BYTES, or zeros where `there` is false, without a branch (one for every vector would serialise a row).
template <int BYTES>
__device__ __forceinline__ void copy_ahead(void* dst, const void* src, bool there) {
  if constexpr (BYTES == 2) {  // single bf16: cp.async moves 4, 8 or 16 bytes
    const uint16_t v = *static_cast<const uint16_t*>(src);
    *static_cast<uint16_t*>(dst) = there ? v : (uint16_t)0;
  } else if constexpr (BYTES == 32) {
    copy_ahead<16>(dst, src, there);
    copy_ahead<16>(static_cast<char*>(dst) + 16, static_cast<const char*>(src) + 16, there);
  } else {
    const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst)), n = there ? BYTES : 0;
    if constexpr (BYTES == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(BYTES), "r"(n) : "memory");
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int kRowThreads = 512;  // most threads of a row block

// One thread's part of the rows.
template <typename T, int VB, int NV, int GATE, int TENSORS>
struct Mine {
  static constexpr int VEC = VB / (int)sizeof(T), EPT = NV * VEC;
  static_assert(EPT % 4 == 0, "whole float4s of columns");
  // cp.async moves 4 bytes at least.  Single bf16 are loaded into registers instead, a row ahead, as far as there are
  // registers for them (4096 x 4095: forward 49 us, backward 103 us; stored into the ring, which waits for every load,
  // 62 and 132 us; 2048 x 6001, 64 values of a backward: 150 us in registers, 134 in the ring).
  static constexpr bool HELD = VB == 2 && NV * TENSORS <= 32;
  static constexpr int N_TENSORS = TENSORS;
  static constexpr int ROW = NV * VB;  // bytes of a row of T
  // a gate row streams beside the others, in room for float32, where a thread has few enough columns
  static constexpr bool STREAM_GATE = GATE == 2 && EPT <= 8;
  static constexpr int BLOCKS = ROW <= (VB == 2 ? 8 : 16) && GATE != 2 ? 2 : 1;  // on an SM
  static constexpr int COLS = GATE == 2 && !STREAM_GATE ? 3 : 2;  // sets of columns kept
  using R = typename Raw<VB>::type;
  int nthr, tid, nvec;
  char* ring;
  float4* cols;
  int stage_bytes;
  mutable uint16_t held[HELD ? TENSORS : 1][HELD ? NV : 1];
  __device__ __forceinline__ Mine(int H, char* smem, int stages)
      : nthr((int)blockDim.x), tid((int)threadIdx.x), nvec(H / VEC), ring(smem) {
    stage_bytes = nthr * ((HELD ? 0 : TENSORS * ROW) + (STREAM_GATE ? EPT * 4 : 0));
    cols = reinterpret_cast<float4*>(smem + stages * stage_bytes) + tid;
  }
  static __host__ constexpr int smem(int threads, int stages) {
    return threads * (stages * ((HELD ? 0 : TENSORS * ROW) + (STREAM_GATE ? EPT * 4 : 0)) + COLS * EPT * 4);
  }
  __device__ __forceinline__ bool has(int j) const { return tid + j * nthr < nvec; }
  __device__ __forceinline__ int col(int j) const { return (tid + j * nthr) * VEC; }
  // a column that exists, for addresses
  __device__ __forceinline__ int safe(int j) const { return has(j) ? col(j) : 0; }
  __device__ __forceinline__ char* slot(int st, int t, int j) const {
    return ring + st * stage_bytes + ((t * NV + j) * nthr + tid) * VB;
  }
  __device__ __forceinline__ void ahead(int st, int t, const void* base, int64_t at) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const T* src = static_cast<const T*>(base) + at + safe(j);
      if constexpr (HELD) held[t][j] = *reinterpret_cast<const uint16_t*>(src);
      else copy_ahead<VB>(slot(st, t, j), src, has(j));
    }
  }
  __device__ __forceinline__ void take(int st, int t, float (&v)[EPT]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      R raw;
      if constexpr (HELD) raw = has(j) ? held[t][j] : (uint16_t)0;
      else raw = *reinterpret_cast<const R*>(slot(st, t, j));
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j * VEC + i] = Cvt<T>::to_f(e[i]);
    }
  }
  // the streamed gate: behind the `tensors` row tensors of a stage
  __device__ __forceinline__ char* gate_slot(int st, int j) const {
    return ring + st * stage_bytes + (HELD ? 0 : TENSORS * ROW) * nthr + (j * nthr + tid) * VEC * 4;
  }
  __device__ __forceinline__ void gate_ahead(int st, const void* base, int64_t at, int is_bf16) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (is_bf16) copy_ahead<VEC * 2>(gate_slot(st, j), static_cast<const bf16*>(base) + at + safe(j), has(j));
      else copy_ahead<VEC * 4>(gate_slot(st, j), static_cast<const float*>(base) + at + safe(j), has(j));
    }
  }
  __device__ __forceinline__ void gate_take(int st, int is_bf16, float (&v)[EPT]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float t[VEC];
      if (is_bf16) load_vec<bf16>(reinterpret_cast<const bf16*>(gate_slot(st, j)), t);
      else load_vec<float>(reinterpret_cast<const float*>(gate_slot(st, j)), t);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j * VEC + i] = t[i];
    }
  }
  // EPT values of a row of `p` (bf16 or float32, 16-byte aligned) from element `at`; 0 where the row has no column
  __device__ __forceinline__ void fetch(const void* p, int64_t at, int is_bf16, float (&v)[EPT]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float t[VEC];
      if (is_bf16) load_vec<bf16>(static_cast<const bf16*>(p) + at + safe(j), t);
      else load_vec<float>(static_cast<const float*>(p) + at + safe(j), t);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[j * VEC + i] = has(j) ? t[i] : 0.f;
    }
  }
  __device__ __forceinline__ void put(void* base, int64_t at, const float (&v)[EPT]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      R raw;
      round_n<T, VEC>(v + j * VEC, reinterpret_cast<T*>(&raw));
      if (has(j)) *reinterpret_cast<R*>(static_cast<T*>(base) + at + col(j)) = raw;
    }
  }
  // the same into a bf16 or float32 row that is 16-byte aligned
  __device__ __forceinline__ void put_as(void* base, int64_t at, int is_bf16, const float (&v)[EPT]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (has(j)) {
        if (is_bf16) store_vec<bf16>(static_cast<bf16*>(base) + at + col(j), v + j * VEC);
        else store_vec<float>(static_cast<float*>(base) + at + col(j), v + j * VEC);
      }
  }
  template <typename U>
  __device__ __forceinline__ static void load_vec(const U* p, float (&t)[VEC]) {
    constexpr int BYTES = VEC * (int)sizeof(U), PIECE = BYTES > 16 ? 16 : BYTES, N = PIECE / (int)sizeof(U);
#pragma unroll
    for (int q = 0; q < BYTES / PIECE; ++q) {
      const typename Raw<PIECE>::type raw = reinterpret_cast<const typename Raw<PIECE>::type*>(p)[q];
      const U* e = reinterpret_cast<const U*>(&raw);
#pragma unroll
      for (int i = 0; i < N; ++i) t[q * N + i] = Cvt<U>::to_f(e[i]);
    }
  }
  template <typename U>
  __device__ __forceinline__ static void store_vec(U* p, const float* v) {
    constexpr int BYTES = VEC * (int)sizeof(U), PIECE = BYTES > 16 ? 16 : BYTES, N = PIECE / (int)sizeof(U);
#pragma unroll
    for (int q = 0; q < BYTES / PIECE; ++q) {
      typename Raw<PIECE>::type raw;
      round_n<U, N>(v + q * N, reinterpret_cast<U*>(&raw));
      reinterpret_cast<typename Raw<PIECE>::type*>(p)[q] = raw;
    }
  }
  // set k of this thread's columns, four at a time
  __device__ __forceinline__ void keep(int k, const float (&v)[EPT]) const {
#pragma unroll
    for (int q = 0; q < EPT / 4; ++q)
      cols[(k * (EPT / 4) + q) * nthr] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  }
  __device__ __forceinline__ void kept(int k, float (&v)[EPT]) const {
#pragma unroll
    for (int q = 0; q < EPT / 4; ++q) {
      const float4 t = cols[(k * (EPT / 4) + q) * nthr];
      v[4 * q] = t.x, v[4 * q + 1] = t.y, v[4 * q + 2] = t.z, v[4 * q + 3] = t.w;
    }
  }
};

// Rows in flight: 64 KB of them for 512 threads where two such blocks share an SM, 128 KB for one alone, at most 4.
template <typename M>
__host__ __device__ constexpr int stages_of() {
  if (M::HELD) return 1;
  const int n = (M::BLOCKS == 2 ? 64 : 128) * 1024 / kRowThreads / (M::N_TENSORS * M::ROW + (M::STREAM_GATE ? M::EPT * 4 : 0));
  return n >= 4 ? 4 : n >= 2 ? 2 : 1;
}

enum { COL_GATE_POST = 0, COL_PRE = 1, COL_GATE = 2 };

// Sum over the block by up to 16 warps.
__device__ __forceinline__ float row_sum(float v, float4* red) {
  v = warp_sum(v);
  if (blockDim.x == 32) return v;
  if ((threadIdx.x & 31) == 0) reinterpret_cast<float*>(red)[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kRowThreads / 128; ++i) {
    const float4 q = red[i];  // warps that are not there hold 0
    t += (q.x + q.y) + (q.z + q.w);
  }
  return t;
}

// gate (where there is one per span) times w_post into set COL_GATE_POST.
template <typename M>
__device__ __forceinline__ void keep_gate_post(const M& me, const NormArgs& p, bool gated, int64_t gate_row) {
  float w[M::EPT];
  me.fetch(p.w_post, 0, p.w_bf16, w);
  if (gated) {
    float g[M::EPT];
    me.fetch(p.gate, gate_row * p.H, p.gate_bf16, g);
#pragma unroll
    for (int i = 0; i < M::EPT; ++i) w[i] *= g[i];
  }
  me.keep(COL_GATE_POST, w);
}

template <typename T, int VB, int NV, int GATE>
__global__ void __launch_bounds__(kRowThreads, Mine<T, VB, NV, GATE, 2>::BLOCKS)
    sandwich_fwd_kernel(const __grid_constant__ NormArgs p) {
  using M = Mine<T, VB, NV, GATE, 2>;
  constexpr int EPT = M::EPT, ST = stages_of<M>();
  extern __shared__ __align__(16) char smem[];
  __shared__ float4 red[2][kRowThreads / 128];
  const M me(p.H, smem, ST);
  const int64_t r0 = p.rows * blockIdx.x / gridDim.x, r1 = p.rows * (blockIdx.x + 1) / gridDim.x;
  auto ahead = [&](int64_t row, int st) {
    if (row < r1) {
      me.ahead(st, 0, p.x, row * p.H);
      me.ahead(st, 1, p.res, row * p.H);
      if constexpr (M::STREAM_GATE) me.gate_ahead(st, p.gate, row * p.H, p.gate_bf16);
    }
    copies_commit();
  };
  for (int i = 0; i < ST; ++i) ahead(r0 + i, i);
  if (threadIdx.x < 2 * kRowThreads / 128) (&red[0][0])[threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  {
    float w[EPT];
    me.fetch(p.w_pre, 0, p.w_bf16, w);
    me.keep(COL_PRE, w);
  }
  keep_gate_post(me, p, GATE == GATE_SPAN, GATE == GATE_SPAN ? r0 / p.span : 0);
  int64_t gate_end = GATE == GATE_SPAN ? (r0 / p.span + 1) * p.span : 0;  // first row that needs another gate row
  __syncthreads();
  const float inv_h = 1.0f / (float)p.H;
  int st = 0;
  for (int64_t row = r0; row < r1; ++row) {
    if (GATE == GATE_SPAN && row == gate_end) {
      keep_gate_post(me, p, true, row / p.span);
      gate_end += p.span;
    }
    float g[GATE == GATE_ROW ? EPT : 1];
    if constexpr (GATE == GATE_ROW && !M::STREAM_GATE) me.fetch(p.gate, row * p.H, p.gate_bf16, g);
    copies_wait<ST - 1>();
    float x[EPT], s[EPT];
    me.take(st, 0, x);
    me.take(st, 1, s);
    if constexpr (M::STREAM_GATE) me.gate_take(st, p.gate_bf16, g);
    ahead(row + ST, st);
    if (++st == ST) st = 0;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) ss = fmaf(x[i], x[i], ss);
    const float rx = 1.0f / sqrtf(row_sum(ss, red[0]) * inv_h + p.eps);
    ss = 0.f;
    {
      float w[EPT];
      me.kept(COL_GATE_POST, w);
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const float gw = GATE == GATE_ROW ? g[GATE == GATE_ROW ? i : 0] * w[i] : w[i];
        s[i] = fmaf(gw, x[i] * rx, p.scale * s[i]);
        ss = fmaf(s[i], s[i], ss);
      }
    }
    me.put(p.s, row * p.H, s);
    const float rs = 1.0f / sqrtf(row_sum(ss, red[1]) * inv_h + p.eps);
    float w[EPT];
    me.kept(COL_PRE, w);
#pragma unroll
    for (int i = 0; i < EPT; ++i) s[i] = s[i] * rs * w[i];
    me.put(p.h, row * p.H, s);
    if (threadIdx.x == 0 && p.rx != nullptr) {
      p.rx[row] = rx;
      p.rs[row] = rs;
    }
  }
}

template <typename T, int VB, int NV, int GATE>
__global__ void __launch_bounds__(kRowThreads, Mine<T, VB, NV, GATE, 4>::BLOCKS)
    sandwich_bwd_kernel(const __grid_constant__ NormArgs p) {
  using M = Mine<T, VB, NV, GATE, 4>;
  constexpr int EPT = M::EPT, ST = stages_of<M>();
  extern __shared__ __align__(16) char smem[];
  __shared__ float4 red[2][kRowThreads / 128];
  const M me(p.H, smem, ST);
  tc::launch_dependents();  // the sums' kernel may be brought up; it waits for this one
  // consecutive units (row ranges inside one span): their rows are consecutive too
  const int64_t u0 = p.units * blockIdx.x / gridDim.x, u1 = p.units * (blockIdx.x + 1) / gridDim.x;
  auto first_row = [&](int64_t u) {
    const int64_t i = u / p.units_per_span, k = u - i * p.units_per_span;
    return i * p.span + p.span * k / p.units_per_span;
  };
  const int64_t r0 = first_row(u0), r1 = first_row(u1);
  const bool has_dh = p.dh != nullptr, has_ds = p.ds != nullptr;
  auto ahead = [&](int64_t row, int st) {
    if (row < r1) {
      me.ahead(st, 0, p.x, row * p.H);
      me.ahead(st, 1, p.res, row * p.H);
      if (has_dh) me.ahead(st, 2, p.dh, row * p.H);
      if (has_ds) me.ahead(st, 3, p.ds, row * p.H);
      if constexpr (M::STREAM_GATE) me.gate_ahead(st, p.gate, row * p.H, p.gate_bf16);
    }
    copies_commit();
  };
  for (int i = 0; i < ST; ++i) ahead(r0 + i, i);
  if (threadIdx.x < 2 * kRowThreads / 128) (&red[0][0])[threadIdx.x] = make_float4(0.f, 0.f, 0.f, 0.f);
  {
    float w[EPT];
    me.fetch(p.w_pre, 0, p.w_bf16, w);
    me.keep(COL_PRE, w);
  }
  float A[EPT], Bp[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) A[i] = Bp[i] = 0.f;
  int64_t u = u0, unit_end = first_row(u0 + 1);
  keep_gate_post(me, p, GATE == GATE_SPAN, u / p.units_per_span);
  __syncthreads();
  const float inv_h = 1.0f / (float)p.H;
  float rx = p.rx[r0], rs = p.rs[r0];
  int st = 0;
  for (int64_t row = r0; row < r1; ++row) {
    const int64_t at = row * p.H;
    const int64_t next = row + 1 < r1 ? row + 1 : row;
    const float rx_next = p.rx[next], rs_next = p.rs[next];
    if constexpr (GATE == GATE_ROW && !M::STREAM_GATE) {
      float g[EPT];
      me.fetch(p.gate, at, p.gate_bf16, g);
      me.keep(COL_GATE, g);
    }
    copies_wait<ST - 1>();
    // gate w_post of this row: kept, or formed from the streamed gate
    auto gate_post = [&](float (&w)[EPT]) {
      me.kept(COL_GATE_POST, w);
      if constexpr (GATE == GATE_ROW) {
        float g[EPT];
        if constexpr (M::STREAM_GATE) me.gate_take(st, p.gate_bf16, g);
        else me.kept(COL_GATE, g);
#pragma unroll
        for (int i = 0; i < EPT; ++i) w[i] *= g[i];
      }
    };
    float xr[EPT], S[EPT];
    me.take(st, 0, xr);
    me.take(st, 1, S);
    {
      float w[EPT];
      gate_post(w);
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        xr[i] *= rx;
        S[i] = fmaf(w[i], xr[i], p.scale * S[i]) * rs;  // t
      }
    }
    float c = 0.f;
    if (has_dh) {
      float dh[EPT], w[EPT];
      me.take(st, 2, dh);
      me.kept(COL_PRE, w);
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        Bp[i] = fmaf(dh[i], S[i], Bp[i]);
        dh[i] *= w[i];  // u
        c = fmaf(dh[i], S[i], c);
      }
      const float k = row_sum(c, red[0]) * inv_h * rs;
#pragma unroll
      for (int i = 0; i < EPT; ++i) S[i] = fmaf(rs, dh[i], -S[i] * k);
    } else {
#pragma unroll
      for (int i = 0; i < EPT; ++i) S[i] = 0.f;
      __syncthreads();  // the second sums of two rows use the same place
    }
    if (has_ds) {
      float ds[EPT];
      me.take(st, 3, ds);
#pragma unroll
      for (int i = 0; i < EPT; ++i) S[i] += ds[i];
    }
    float v[EPT];  // gate w_post, then gate w_post S
    gate_post(v);
    c = 0.f;
    if constexpr (GATE == GATE_ROW) {
      float w[EPT], out[EPT];
      me.kept(COL_GATE_POST, w);
#pragma unroll
      for (int i = 0; i < EPT; ++i) out[i] = w[i] * (S[i] * xr[i]);
      me.put_as(p.dgate, at, p.gate_bf16, out);
      if constexpr (M::STREAM_GATE) me.gate_take(st, p.gate_bf16, w);
      else me.kept(COL_GATE, w);
#pragma unroll
      for (int i = 0; i < EPT; ++i) A[i] = fmaf(w[i], S[i] * xr[i], A[i]);
    }
    ahead(row + ST, st);
    if (++st == ST) st = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      if (GATE != GATE_ROW) A[i] = fmaf(S[i], xr[i], A[i]);
      v[i] *= S[i];
      c = fmaf(v[i], xr[i], c);
      S[i] *= p.scale;
    }
    me.put(p.dres, at, S);
    const float k = row_sum(c, red[1]) * inv_h;
#pragma unroll
    for (int i = 0; i < EPT; ++i) v[i] = rx * fmaf(-xr[i], k, v[i]);
    me.put(p.dx, at, v);
    rx = rx_next, rs = rs_next;
    if (row + 1 == unit_end) {
      me.put_as(p.part_a, u * p.H, 0, A);
      if (++u < u1) {
        unit_end = first_row(u + 1);
        if (GATE == GATE_SPAN) keep_gate_post(me, p, true, u / p.units_per_span);
#pragma unroll
        for (int i = 0; i < EPT; ++i) A[i] = 0.f;
      }
    }
  }
  me.put_as(p.part_b, (int64_t)blockIdx.x * p.H, 0, Bp);
}

// ------------------------------------------------- rows too long for that

template <typename T>
__global__ void __launch_bounds__(kMaxThreads) sandwich_fwd_long_kernel(NormArgs p, int gate) {
  __shared__ float red[2][32];
  const T* xp = static_cast<const T*>(p.x);
  const T* rp = static_cast<const T*>(p.res);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int64_t base = row * p.H;
    float ss = 0.f;
    for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
      const float v = Cvt<T>::to_f(xp[base + c]);
      ss = fmaf(v, v, ss);
    }
    const float rx = 1.0f / sqrtf(block_sum(ss, red[0]) / (float)p.H + p.eps);
    ss = 0.f;
    for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
      const float pn = Cvt<T>::to_f(xp[base + c]) * rx * load_as(p.w_post, c, p.w_bf16);
      const float s = fmaf(p.scale, Cvt<T>::to_f(rp[base + c]), gate_at(p, gate, row, c) * pn);
      ss = fmaf(s, s, ss);
    }
    const float rs = 1.0f / sqrtf(block_sum(ss, red[1]) / (float)p.H + p.eps);
    for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
      const float pn = Cvt<T>::to_f(xp[base + c]) * rx * load_as(p.w_post, c, p.w_bf16);
      const float s = fmaf(p.scale, Cvt<T>::to_f(rp[base + c]), gate_at(p, gate, row, c) * pn);
      static_cast<T*>(p.s)[base + c] = Cvt<T>::from_f(s);
      static_cast<T*>(p.h)[base + c] = Cvt<T>::from_f(s * rs * load_as(p.w_pre, c, p.w_bf16));
    }
    if (threadIdx.x == 0 && p.rx != nullptr) {
      p.rx[row] = rx;
      p.rs[row] = rs;
    }
  }
}

// Each block takes whole units (row ranges inside one span) and keeps its sums in its rows of the partial arrays.
template <typename T>
__global__ void __launch_bounds__(kMaxThreads) sandwich_bwd_long_kernel(NormArgs p, int gate) {
  __shared__ float red[2][32];
  const T* xp = static_cast<const T*>(p.x);
  const T* rp = static_cast<const T*>(p.res);
  const T* hp = static_cast<const T*>(p.dh);
  const T* sp = static_cast<const T*>(p.ds);
  const float inv_h = 1.0f / (float)p.H;
  float* pb = p.part_b + (int64_t)blockIdx.x * p.H;
  for (int c = threadIdx.x; c < p.H; c += blockDim.x) pb[c] = 0.f;
  for (int64_t u = blockIdx.x; u < p.units; u += gridDim.x) {
    float* pa = p.part_a + u * p.H;
    for (int c = threadIdx.x; c < p.H; c += blockDim.x) pa[c] = 0.f;
    const int64_t sp_i = u / p.units_per_span, k = u - sp_i * p.units_per_span;
    const int64_t r0 = sp_i * p.span + p.span * k / p.units_per_span;
    const int64_t r1 = sp_i * p.span + p.span * (k + 1) / p.units_per_span;
    for (int64_t row = r0; row < r1; ++row) {
      const int64_t base = row * p.H;
      const float rx = p.rx[row], rs = p.rs[row];
      float c1 = 0.f;
      for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
        const float pn = Cvt<T>::to_f(xp[base + c]) * rx * load_as(p.w_post, c, p.w_bf16);
        const float s = fmaf(p.scale, Cvt<T>::to_f(rp[base + c]), gate_at(p, gate, row, c) * pn);
        const float dh = hp != nullptr ? Cvt<T>::to_f(hp[base + c]) : 0.f;
        c1 = fmaf(dh * load_as(p.w_pre, c, p.w_bf16), s, c1);
        pb[c] += dh * s * rs;
      }
      c1 = block_sum(c1, red[0]) * inv_h * rs * rs * rs;
      float c2 = 0.f;
      auto grad_s = [&](int c, float xv, float g, float wp) {
        const float s = fmaf(p.scale, Cvt<T>::to_f(rp[base + c]), g * (xv * rx * wp));
        const float dh = hp != nullptr ? Cvt<T>::to_f(hp[base + c]) : 0.f;
        const float ds = sp != nullptr ? Cvt<T>::to_f(sp[base + c]) : 0.f;
        return ds + rs * (dh * load_as(p.w_pre, c, p.w_bf16)) - s * c1;
      };
      for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
        const float xv = Cvt<T>::to_f(xp[base + c]), g = gate_at(p, gate, row, c);
        const float wp = load_as(p.w_post, c, p.w_bf16);
        const float S = grad_s(c, xv, g, wp);
        c2 = fmaf(S * g * wp, xv, c2);
        const float A = S * xv * rx;
        pa[c] += gate == GATE_ROW ? g * A : A;
        if (gate == GATE_ROW) {
          if (p.gate_bf16) static_cast<bf16*>(p.dgate)[base + c] = __float2bfloat16_rn(wp * A);
          else static_cast<float*>(p.dgate)[base + c] = wp * A;
        }
      }
      c2 = block_sum(c2, red[1]) * inv_h * rx * rx * rx;
      for (int c = threadIdx.x; c < p.H; c += blockDim.x) {
        const float xv = Cvt<T>::to_f(xp[base + c]), g = gate_at(p, gate, row, c);
        const float wp = load_as(p.w_post, c, p.w_bf16);
        const float S = grad_s(c, xv, g, wp);
        static_cast<T*>(p.dres)[base + c] = Cvt<T>::from_f(p.scale * S);
        static_cast<T*>(p.dx)[base + c] = Cvt<T>::from_f(rx * (S * g * wp) - xv * c2);
      }
    }
  }
}

__device__ __forceinline__ void store_as(void* p, int64_t i, int is_bf16, float v) {
  if (is_bf16) static_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// Sums of the partial rows, 16 columns and 64 lanes of rows to a block, in a fixed order.  The lanes are dealt to the
// spans (64 / spans each, or a span at a time each where there are more): dgate = w_post A of the span, and the
// spans' gate A add up to dw_post.
constexpr int kSumCols = 16, kSumLanes = 64;

// n values of a column in four running sums
__device__ __forceinline__ float lane_sum(const float (*v)[kSumCols + 1], int first, int n, int cl) {
  float u[4] = {0.f, 0.f, 0.f, 0.f};
  int q = 0;
  for (; q + 4 <= n; q += 4)
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] += v[first + q + i][cl];
  for (; q < n; ++q) u[0] += v[first + q][cl];
  return (u[0] + u[1]) + (u[2] + u[3]);
}

__global__ void __launch_bounds__(kSumCols* kSumLanes) sandwich_sums_kernel(NormArgs p, int gate, int64_t spans,
                                                                           int64_t blocks, void* dw_post,
                                                                           void* dw_pre) {
  __shared__ float red[3][kSumLanes][kSumCols + 1];
  const int cl = threadIdx.x % kSumCols, rl = threadIdx.x / kSumCols;
  const int col = blockIdx.x * kSumCols + cl;
  const bool in = col < p.H;
  const int64_t ups = p.units_per_span;
  int groups = 1;  // spans at a time
  while (groups < spans && groups < kSumLanes) groups <<= 1;
  const int per = kSumLanes / groups;
  const float wp = in ? load_as(p.w_post, col, p.w_bf16) : 0.f;
  tc::wait_prerequisites();
  float post = 0.f, a = 0.f, pre = 0.f;
  for (int64_t i = rl / per; i < spans; i += groups) {  // once where a span has several lanes
    a = 0.f;
    if (in) {
#pragma unroll 4
      for (int64_t k = rl % per; k < ups; k += per) a += p.part_a[(i * ups + k) * p.H + col];
      if (gate == GATE_SPAN) {
        post = fmaf(a, load_as(p.gate, i * p.H + col, p.gate_bf16), post);
        if (per == 1) store_as(p.dgate, i * p.H + col, p.gate_bf16, wp * a);
      } else {
        post += a;
      }
    }
  }
  if (in) {
#pragma unroll 4
    for (int64_t q = rl; q < blocks; q += kSumLanes) pre += p.part_b[q * p.H + col];
  }
  red[0][rl][cl] = post;
  red[1][rl][cl] = pre;
  red[2][rl][cl] = a;
  __syncthreads();
  if (!in) return;
  if (rl == 0) store_as(dw_post, col, p.w_bf16, lane_sum(red[0], 0, kSumLanes, cl));
  if (rl == 2) store_as(dw_pre, col, p.w_bf16, lane_sum(red[1], 0, kSumLanes, cl));  // another warp
  if (gate == GATE_SPAN && per > 1 && rl % per == per - 1 && rl / per < spans)
    store_as(p.dgate, rl / per * (int64_t)p.H + col, p.gate_bf16, wp * lane_sum(red[2], rl / per * per, per, cl));
}

struct BwdPlan {
  int64_t spans, units, blocks;
  int units_per_span;
};

// Blocks of a backward on an SM, at most: those of fewer columns are smaller, and their partial rows cost less.
int64_t most_per_sm(int64_t H) { return H >= 4096 ? 2 : H <= 256 ? 32 : 8192 / H; }

// Row ranges (units) of the backward, none across a span, for `per_sm` blocks on each SM, but 4 rows to a block before
// a second one on an SM: a partial row is as many bytes as a row or more (1674 x 3000 bf16: 25.2 us, with 8 rows 29.9 us;
// 2232 x 371: 12.4 and 14.5 us; 3087 x 64: 10.3 us, with 2 rows 12.0 us).
BwdPlan bwd_plan(int64_t rows, int64_t span, int64_t per_sm) {
  BwdPlan b;
  const int64_t sms = num_sms();
  int64_t want = rows / 4 < sms ? sms : rows / 4;
  if (want > sms * per_sm) want = sms * per_sm;
  b.spans = rows / span;
  int64_t per = b.spans >= want ? 1 : want / b.spans;
  if (per > span) per = span;
  b.units_per_span = (int)per;
  b.units = b.spans * per;
  b.blocks = b.units < want ? b.units : want;
  return b;
}

int check(const void* x, const void* res, int64_t rows, int64_t H, ats_dtype dt, const void* w_post, const void* w_pre,
          ats_dtype wdt, const void* gate, ats_dtype gdt, int64_t span, const char* what) {
  if (dt != ATS_BF16 && dt != ATS_F32) return fail(ATS_EBADARG, "%s: dtype", what);
  if (wdt != ATS_BF16 && wdt != ATS_F32) return fail(ATS_EBADARG, "%s: weight dtype", what);
  if (gate != nullptr && gdt != ATS_BF16 && gdt != ATS_F32) return fail(ATS_EBADARG, "%s: gate dtype", what);
  if (rows < 0 || H <= 0 || H >= (1 << 30))
    return fail(ATS_EBADARG, "%s: rows=%lld hidden=%lld", what, (long long)rows, (long long)H);
  if (gate != nullptr && rows > 0 && (span < 1 || rows % span != 0))
    return fail(ATS_EBADARG, "%s: %lld rows per gate row do not divide %lld rows", what, (long long)span,
                (long long)rows);
  if (rows > 0 && (x == nullptr || res == nullptr)) return fail(ATS_EBADARG, "%s: null input", what);
  if (w_post == nullptr || w_pre == nullptr) return fail(ATS_EBADARG, "%s: null weight", what);
  return ATS_OK;
}

int gate_kind(const void* gate, int64_t span) { return gate == nullptr ? GATE_NONE : span == 1 ? GATE_ROW : GATE_SPAN; }

int threads_for(int64_t H) {
  int t = 128;
  while (t < 512 && t * 8 < H) t <<= 1;
  return t;
}

// Calls go(integral constants VB, NV) with the widest vectors that the width and every pointer allow, and as few of
// them per thread as give at most kRowThreads threads; false where a row has too many for 16 elements a thread.
template <typename T, typename F>
bool pick_vectors(int64_t H, uintptr_t addr, F go) {
  const int64_t es = sizeof(T);
  if (addr % (uintptr_t)es != 0) return false;
  int vb = 16;
  while (vb > (int)es && (H * es % vb != 0 || addr % (uintptr_t)vb != 0)) vb >>= 1;
  const int64_t per = (H * es / vb + kRowThreads - 1) / kRowThreads;  // vectors a thread needs
#define ATS_PICK(VB_, NV_)                                                                   \
  if (vb == VB_ && per <= NV_) {                                                              \
    go(std::integral_constant<int, VB_>{}, std::integral_constant<int, NV_>{});               \
    return true;                                                                             \
  }
  if constexpr (sizeof(T) == 2) {
    ATS_PICK(16, 1) ATS_PICK(16, 2) ATS_PICK(8, 1) ATS_PICK(8, 2) ATS_PICK(8, 4) ATS_PICK(4, 2) ATS_PICK(4, 8)
    ATS_PICK(2, 4) ATS_PICK(2, 8) ATS_PICK(2, 16)
  } else {
    ATS_PICK(16, 1) ATS_PICK(16, 2) ATS_PICK(16, 4) ATS_PICK(8, 2) ATS_PICK(8, 8) ATS_PICK(4, 4) ATS_PICK(4, 16)
  }
#undef ATS_PICK
  return false;
}

// Threads of a row: whole warps with nv vectors each.
int row_threads(int H, int vec, int nv) { return ((H / vec + nv - 1) / nv + 31) / 32 * 32; }

uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Low bits of the rows' addresses.  The weights, the gate and its gradient are read and written in pieces of up to 16
// bytes whatever the rows' vectors are: 1 (no vectors at all) where one of them is not aligned to that.
uintptr_t row_bits(const NormArgs& p) {
  const uintptr_t other = bits(p.w_post) | bits(p.w_pre) | bits(p.gate) | bits(p.dgate);
  return bits(p.x) | bits(p.res) | (other % 16 != 0 ? 1 : 0);
}

// Blocks of `threads` threads and `smem` bytes that an SM holds, 1 to 32: `regs` registers a thread.
int64_t resident(int regs, int threads, int smem) {
  const int64_t by_regs = 65536 / ((int64_t)(regs + 7) / 8 * 8 * threads), by_smem = 227 * 1024 / (smem + 1536);
  const int64_t n = by_regs < by_smem ? by_regs : by_smem;
  return n < 1 ? 1 : n > 32 ? 32 : n;
}

template <auto KERNEL>
int regs_of() {
  static const int regs = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, KERNEL) == cudaSuccess ? a.numRegs : 128;
  }();
  return regs;
}

// go(GATE constant) for the gate of this call.
template <typename F>
int by_gate(int gate, F go) {
  if (gate == GATE_NONE) return go(std::integral_constant<int, GATE_NONE>{});
  if (gate == GATE_SPAN) return go(std::integral_constant<int, GATE_SPAN>{});
  return go(std::integral_constant<int, GATE_ROW>{});
}

template <typename T>
int fwd_t(const NormArgs& p, int gate, cudaStream_t st) {
  int rc = ATS_OK;
  const bool ok = pick_vectors<T>(p.H, row_bits(p) | bits(p.s) | bits(p.h), [&](auto vb, auto nv) {
    rc = by_gate(gate, [&](auto g) {
      using M = Mine<T, vb.value, nv.value, g.value, 2>;
      constexpr auto kernel = sandwich_fwd_kernel<T, vb.value, nv.value, g.value>;
      const int t = row_threads(p.H, M::VEC, nv.value), smem = M::smem(t, stages_of<M>());
      ATS_TRY(allow_smem<kernel>("sandwich_norm_fwd"));
      const int64_t cap = num_sms() * resident(regs_of<kernel>(), t, smem);
      kernel<<<(unsigned)(p.rows < cap ? p.rows : cap), t, smem, st>>>(p);
      return check_launch("sandwich_norm_fwd");
    });
  });
  if (ok) return rc;
  const int64_t cap = (int64_t)num_sms() * 16;
  sandwich_fwd_long_kernel<T><<<(unsigned)(p.rows < cap ? p.rows : cap), threads_for(p.H), 0, st>>>(p, gate);
  return check_launch("sandwich_norm_fwd");
}

template <typename T>
int bwd_t(NormArgs p, int gate, float* workspace, void* dw_post, void* dw_pre, cudaStream_t st) {
  BwdPlan b;
  auto plan = [&](int64_t per_sm) {
    const int64_t most = most_per_sm(p.H);
    b = bwd_plan(p.rows, p.span, per_sm < most ? per_sm : most);
    p.units_per_span = b.units_per_span, p.units = b.units;
    p.part_a = workspace;
    p.part_b = workspace + b.units * p.H;
  };
  int rc = ATS_OK;
  const uintptr_t addr = row_bits(p) | bits(p.dh) | bits(p.ds) | bits(p.dx) | bits(p.dres);
  const bool ok = pick_vectors<T>(p.H, addr, [&](auto vb, auto nv) {
    rc = by_gate(gate, [&](auto g) {
      using M = Mine<T, vb.value, nv.value, g.value, 4>;
      constexpr auto kernel = sandwich_bwd_kernel<T, vb.value, nv.value, g.value>;
      const int t = row_threads(p.H, M::VEC, nv.value), smem = M::smem(t, stages_of<M>());
      ATS_TRY(allow_smem<kernel>("sandwich_norm_bwd"));
      plan(resident(regs_of<kernel>(), t, smem));
      kernel<<<(unsigned)b.blocks, t, smem, st>>>(p);
      return check_launch("sandwich_norm_bwd");
    });
  });
  if (!ok) {
    plan(2);
    sandwich_bwd_long_kernel<T><<<(unsigned)b.blocks, threads_for(p.H), 0, st>>>(p, gate);
    rc = check_launch("sandwich_norm_bwd");
  }
  ATS_TRY(rc);
  cudaLaunchAttribute attr[1];  // brought up while the rows are still worked on
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.H + kSumCols - 1) / kSumCols));
  cfg.blockDim = dim3(kSumCols * kSumLanes);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, sandwich_sums_kernel, p, gate, b.spans, b.blocks, dw_post, dw_pre);
  if (e != cudaSuccess) return fail(ATS_ECUDA, "sandwich_sums: %s", cudaGetErrorString(e));
  return check_launch("sandwich_sums");
}

}  // namespace
}  // namespace ats

using namespace ats;

extern "C" {

int ats_sandwich_norm_fwd(const void* x, const void* residual, ats_dtype dtype, const void* w_post, const void* w_pre,
                          ats_dtype w_dtype, const void* gate, ats_dtype gate_dtype, int64_t rows_per_gate,
                          float residual_scale, float eps, void* sum, void* h, float* rstd_x, float* rstd_sum,
                          int64_t rows, int64_t hidden, void* stream) {
  ATS_TRY(check(x, residual, rows, hidden, dtype, w_post, w_pre, w_dtype, gate, gate_dtype, rows_per_gate,
                "sandwich_norm_fwd"));
  if (rows == 0) return ATS_OK;
  if (sum == nullptr || h == nullptr || (rstd_x == nullptr) != (rstd_sum == nullptr))
    return fail(ATS_EBADARG, "sandwich_norm_fwd: null output");
  NormArgs p{};
  p.x = x, p.res = residual, p.s = sum, p.h = h, p.w_post = w_post, p.w_pre = w_pre, p.gate = gate;
  p.w_bf16 = w_dtype == ATS_BF16, p.gate_bf16 = gate_dtype == ATS_BF16;
  p.rx = rstd_x, p.rs = rstd_sum;
  p.rows = rows, p.span = rows_per_gate, p.H = (int)hidden, p.scale = residual_scale, p.eps = eps;
  const int g = gate_kind(gate, rows_per_gate);
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == ATS_BF16 ? fwd_t<bf16>(p, g, st) : fwd_t<float>(p, g, st);
}

size_t ats_sandwich_norm_bwd_workspace_bytes(int64_t rows, int64_t hidden, int64_t rows_per_gate) {
  if (rows <= 0 || hidden <= 0 || rows_per_gate < 0 || (rows_per_gate > 0 && rows % rows_per_gate != 0)) return 0;
  const int64_t blocks = num_sms() * most_per_sm(hidden), spans = rows_per_gate > 1 ? rows / rows_per_gate : 1;
  return (size_t)((spans > blocks ? spans : blocks) + blocks) * (size_t)hidden * sizeof(float);
}

int ats_sandwich_norm_bwd(const void* dh, const void* dsum, const void* x, const void* residual, ats_dtype dtype,
                          const void* w_post, const void* w_pre, ats_dtype w_dtype, const void* gate,
                          ats_dtype gate_dtype, int64_t rows_per_gate, float residual_scale, const float* rstd_x,
                          const float* rstd_sum, void* dx, void* dresidual, void* dw_post, void* dw_pre, void* dgate,
                          void* workspace, size_t workspace_bytes, int64_t rows, int64_t hidden, void* stream) {
  ATS_TRY(check(x, residual, rows, hidden, dtype, w_post, w_pre, w_dtype, gate, gate_dtype, rows_per_gate,
                "sandwich_norm_bwd"));
  if (rows == 0) return fail(ATS_EBADARG, "sandwich_norm_bwd: no rows");
  if (rstd_x == nullptr || rstd_sum == nullptr || dx == nullptr || dresidual == nullptr || dw_post == nullptr ||
      dw_pre == nullptr || (gate != nullptr && dgate == nullptr))
    return fail(ATS_EBADARG, "sandwich_norm_bwd: null pointer");
  const int g = gate_kind(gate, rows_per_gate);
  if (workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < ats_sandwich_norm_bwd_workspace_bytes(rows, hidden, gate != nullptr ? rows_per_gate : 0))
    return fail(ATS_EBADARG, "sandwich_norm_bwd: workspace too small");
  NormArgs p{};
  p.x = x, p.res = residual, p.dh = dh, p.ds = dsum, p.dx = dx, p.dres = dresidual;
  p.w_post = w_post, p.w_pre = w_pre, p.gate = gate, p.dgate = dgate;
  p.w_bf16 = w_dtype == ATS_BF16, p.gate_bf16 = gate_dtype == ATS_BF16;
  p.rx = const_cast<float*>(rstd_x), p.rs = const_cast<float*>(rstd_sum);
  p.rows = rows, p.span = g == GATE_SPAN ? rows_per_gate : rows;
  p.H = (int)hidden, p.scale = residual_scale;
  cudaStream_t st = (cudaStream_t)stream;
  float* ws = static_cast<float*>(workspace);
  return dtype == ATS_BF16 ? bwd_t<bf16>(p, g, ws, dw_post, dw_pre, st) : bwd_t<float>(p, g, ws, dw_post, dw_pre, st);
}

}  // extern "C"
