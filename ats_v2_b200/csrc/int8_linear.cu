// Projection with 8-bit integer weights and activations:
//
//   y[m][n] = (sum_k q[m][k] w[n][k]) * (sx[m] * sw[n]) + bias[n]
//
// w are int8 weights with a float32 scale per output channel; q are the
// activations quantised here, a scale per token:
//
//   amax = max(max_k |x[m][k]|, 2^-100);  q = rint(x * (127 / amax));  sx = amax / 127
//
// in float32 (a row with an infinity or NaN gets a NaN scale, so its outputs
// are NaN).  The sum is exact in int32: K <= 131072 keeps 127 * 128 * K below
// 2^31.  The scales and the bias are applied in float32, rounded once.
#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace ats {
namespace {

constexpr int kMaxK = 131072;
constexpr int64_t kMaxRows = 1 << 30;  // tokens and channels
constexpr long long kWaitBudget = 4000000000LL;  // SM cycles, about 2 s
// Budget of the main-loop waits and the first wait that gave up on this device (0: none), as for the other
// tensor-core GEMMs; the waits that drain copies and MMAs always keep kWaitBudget.
__device__ long long g_int8_wait_budget = kWaitBudget;
__device__ int g_int8_status;

__device__ __forceinline__ void give_up(volatile int* abort, int code) {
  *abort = 1;
  atomicCAS(&g_int8_status, 0, code);
}

// ------------------------------------------------------------- quantisation
// |v| as an unsigned integer orders like |v|, and puts NaN above infinity above every number.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// scale and 127 / amax of a row from the largest |x|'s bits
__device__ __forceinline__ float row_scale(uint32_t bits, float& inv) {
  if (bits >= 0x7f800000u) {
    inv = 0.f;
    return __uint_as_float(0x7fc00000u);
  }
  const float amax = fmaxf(__uint_as_float(bits), 7.888609052210118e-31f);  // 2^-100
  inv = 127.0f / amax;
  return amax / 127.0f;
}

// rint(v * inv) as a byte, for |v * inv| below 2^22: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and
// leaves it in the low bits.  |v| <= amax keeps |v * inv| within 127 (1 + 2^-22), which rounds to at most 127.
__device__ __forceinline__ uint32_t quant(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f));
}

// 16 consecutive values of a 16-byte aligned row from element k, as they are stored; those at or past K are zero.
template <typename T>
__device__ __forceinline__ void load16(const T* row, int k, int K, uint4 (&v)[sizeof(T)]) {
  if (k + 16 <= K) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) v[i] = reinterpret_cast<const uint4*>(row + k)[i];
  } else {
    T e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = k + i < K ? row[k + i] : Cvt<T>::from_f(0.f);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T); ++i) v[i] = reinterpret_cast<const uint4*>(e)[i];
  }
}

// The same of a row aligned to P only, of which K is whole pieces: G threads load their G * 16 values from `base` on side
// by side and pass them through `stage`, where thread t finds its 16.  8192 x 2047 bf16, the same rows again from L2:
// 12.2 us, 2046: 8.8 us; 16 loads by each thread for itself took 20.4 us.  (From HBM 18 to 23 and 11 us.)
template <typename T, int G, typename P>
__device__ __forceinline__ void stage16(const T* row, int base, int t, int K, char* stage, uint4 (&v)[sizeof(T)]) {
  constexpr int E = (int)(sizeof(P) / sizeof(T)), N = 16 / E;
  const int first = base / E + t, last = K / E - 1;
  P p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = reinterpret_cast<const P*>(row)[min(first + i * G, last)];
  auto sync = [] {
    if constexpr (G == 32) __syncwarp();
    else __syncthreads();
  };
  sync();  // the last step's values have been taken
#pragma unroll
  for (int i = 0; i < N; ++i) reinterpret_cast<P*>(stage)[t + i * G] = first + i * G <= last ? p[i] : P(0);
  sync();
#pragma unroll
  for (int i = 0; i < (int)sizeof(T); ++i) v[i] = reinterpret_cast<const uint4*>(stage)[t * (int)sizeof(T) + i];
}

// The largest |value|'s bits of 16; bf16 two at a time, as the high halves of float32.
template <typename T>
__device__ __forceinline__ uint32_t max16(const uint4 (&v)[sizeof(T)], uint32_t m) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(v);
  if constexpr (sizeof(T) == 2) {
    uint32_t two = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) two = __vmaxu2(two, w[i] & 0x7fff7fffu);
    return max(m, max(two << 16, two & 0xffff0000u));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  }
}

// Four bytes; zeros for a row without a finite scale (inv is 0).
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __byte_perm(quant(a, inv), quant(b, inv), 0x0040);
  const uint32_t hi = __byte_perm(quant(c, inv), quant(d, inv), 0x0040);
  return inv != 0.f ? __byte_perm(lo, hi, 0x5410) : 0u;
}

template <typename T>
__device__ __forceinline__ uint4 quant16(const uint4 (&v)[sizeof(T)], float inv) {
  const T* e = reinterpret_cast<const T*>(v);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = pack4(Cvt<T>::to_f(e[4 * i]), Cvt<T>::to_f(e[4 * i + 1]), Cvt<T>::to_f(e[4 * i + 2]),
                 Cvt<T>::to_f(e[4 * i + 3]), inv);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 4 values from element k, zero at or past K; vec: the row is aligned to 4 elements.
template <typename T>
__device__ __forceinline__ void load4(const T* row, int k, int K, int vec, float (&v)[4]) {
  if (vec && k + 4 <= K) {
    if constexpr (sizeof(T) == 2) {
      const uint2 raw = *reinterpret_cast<const uint2*>(row + k);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = Cvt<T>::to_f(e[i]);
    } else {
      load_n<T, 4>(row + k, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < K ? Cvt<T>::to_f(row[k + i]) : 0.f;
  }
}

// G threads to a row (a warp, or all of a block), each with 16 consecutive values per step and the first kKeep steps
// held in registers; a longer row is read again.  q rows are written in 16-byte pieces where they are aligned for it
// (Q16), zeros up to the next multiple of 16 at most ldq.  x rows are aligned to P.
constexpr int kKeep = 4;

template <typename T, int G, typename P, bool Q16>
__global__ void __launch_bounds__(G < 128 ? 128 : G) int8_quantize_kernel(const T* __restrict__ x, int64_t ldx,
                                                                         int8_t* __restrict__ q, int64_t ldq,
                                                                         float* __restrict__ scale, int64_t rows,
                                                                         int K) {
  constexpr int THREADS = G < 128 ? 128 : G;
  // In this order: a dependent kernel reads its weights before its own wait, and what wrote them has ended by now.
  tc::wait_prerequisites();
  tc::launch_dependents();
  constexpr bool VEC = sizeof(P) == 16;
  __shared__ uint32_t red[THREADS / 32];
  __shared__ __align__(16) char stage[VEC ? 16 : THREADS * 16 * sizeof(T)];
  const int64_t row = (int64_t)blockIdx.x * (THREADS / G) + threadIdx.x / G;
  const int t = threadIdx.x % G;
  if (G == 32 && row >= rows) return;
  const T* xr = x + row * ldx;
  auto fetch = [&](int base, uint4 (&v)[sizeof(T)]) {  // by all of the row's threads
    if constexpr (!VEC) stage16<T, G, P>(xr, base, t, K, stage + threadIdx.x / G * (G * 16 * sizeof(T)), v);
    else if (base + t * 16 < K) load16<T>(xr, base + t * 16, K, v);
  };
  uint4 raw[kKeep][sizeof(T)];  // 16 values of T
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    if (j * G * 16 < K) fetch(j * G * 16, raw[j]);
  }
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if ((j * G + t) * 16 < K) m = max16<T>(raw[j], m);
  for (int base = kKeep * G * 16; base < K; base += G * 16) {
    uint4 u[sizeof(T)];
    fetch(base, u);
    if (base + t * 16 < K) m = max16<T>(u, m);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G / 32; ++i) m = max(m, red[i]);
  }
  float inv;
  const float s = row_scale(m, inv);
  if (t == 0) scale[row] = s;
  int8_t* qr = q + row * ldq;
  auto put = [&](int k, const uint4 (&u)[sizeof(T)]) {
    const uint4 w = quant16<T>(u, inv);
    if (Q16) {
      *reinterpret_cast<uint4*>(qr + k) = w;
    } else {
      const int8_t* e = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (k + i < ldq) qr[k + i] = e[i];
    }
  };
#pragma unroll
  for (int j = 0; j < kKeep; ++j) {
    const int k = (j * G + t) * 16;
    if (k < K) put(k, raw[j]);
  }
  for (int base = kKeep * G * 16; base < K; base += G * 16) {
    uint4 u[sizeof(T)];
    fetch(base, u);
    if (base + t * 16 < K) put(base + t * 16, u);
  }
  for (int64_t k = (K + 15) / 16 * 16 + t; k < ldq; k += G) qr[k] = 0;
}

// Launch whose prologue may start before the stream's previous kernel has ended (every kernel here waits for it with
// wait_prerequisites), in clusters of CTAs.
template <auto KERNEL, typename... A>
int launch_after(dim3 grid, int threads, int smem, dim3 cluster, cudaStream_t st, const char* what, A... args) {
  ATS_TRY(allow_smem<KERNEL>(what, true));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster.x;
  attr[1].val.clusterDim.y = cluster.y;
  attr[1].val.clusterDim.z = cluster.z;
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster.x * cluster.y * cluster.z > 1 ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, KERNEL, args...);
  if (e != cudaSuccess) return fail(ATS_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

template <typename T, int G>
int quantize_g(const T* x, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int K, cudaStream_t st) {
  const bool q16 = aligned16(q) && ldq % 16 == 0;
  constexpr int THREADS = G < 128 ? 128 : G;
  const int64_t per = THREADS / G;
  const unsigned grid = (unsigned)((rows + per - 1) / per);
  auto with = [&](auto piece, auto by_16) {
    return launch_after<int8_quantize_kernel<T, G, decltype(piece), by_16.value>>(
        dim3(grid), THREADS, 0, dim3(1), st, "int8_quantize", x, ldx, q, ldq, scale, rows, K);
  };
  auto go = [&](auto piece) { return q16 ? with(piece, std::true_type{}) : with(piece, std::false_type{}); };
  if (aligned16(x) && ldx % Chunk<T>::N == 0) return go(uint4{});
  if constexpr (sizeof(T) == 2) {
    if (reinterpret_cast<uintptr_t>(x) % 4 != 0 || ldx % 2 != 0 || K % 2 != 0) return go(uint16_t{});
  }
  return go(uint32_t{});
}

// As many threads as hold the row in their registers: 32, 128 or 512 (8192x2048 bf16, the same rows again from L2: 6.7
// us with a warp a row; 256 threads, half of them idle there, took 18.4.  From HBM a warp a row takes 10 to 12).
template <typename T>
int quantize_t(const void* x, int64_t ldx, void* q, int64_t ldq, float* scale, int64_t rows, int64_t K,
               cudaStream_t st) {
  auto* xp = static_cast<const T*>(x);
  auto* qp = static_cast<int8_t*>(q);
  if (K <= 32 * 16 * kKeep) return quantize_g<T, 32>(xp, ldx, qp, ldq, scale, rows, (int)K, st);
  if (K <= 128 * 16 * kKeep) return quantize_g<T, 128>(xp, ldx, qp, ldq, scale, rows, (int)K, st);
  return quantize_g<T, 512>(xp, ldx, qp, ldq, scale, rows, (int)K, st);
}

// ------------------------------------------------------------------ epilogue
struct Out {
  void* y;
  const float* sx;
  const float* sw;
  const void* bias;
  int bias_bf16;
  int M, N;
};

// The scaled sum, and the bias added: rounded apart in every kernel here (never fused), so that a token's result does
// not depend on how many come with it.
__device__ __forceinline__ float scaled(int sum, float sx, float sw) { return __fmul_rn((float)sum, __fmul_rn(sx, sw)); }

__device__ __forceinline__ float bias_at(const Out& o, int n) {
  if (o.bias == nullptr) return 0.f;
  return o.bias_bf16 ? __bfloat162float(static_cast<const bf16*>(o.bias)[n]) : static_cast<const float*>(o.bias)[n];
}

// --------------------------------------------------------------- one token
// One launch: every block quantises the token into its shared memory (it comes from L2), with the first weights of
// its warps already in flight, then a warp takes an output channel at a time: 16 weights per lane and step against
// the token's integers.  The weights are read once; latency bounds it at this size (4096 x 4096: 7.1 us with the weights
// from HBM, 2.4 TB/s; 5.2 from L2, where the tensor-core kernel below takes 6.6 with its quantisation).
constexpr int kDotThreads = 256, kDotStep = 8;
constexpr int kDotLongest = 16384;  // a warp walks its channels 4 KB at a time: longer rows are split over SMs instead

template <typename T>
__global__ void __launch_bounds__(kDotThreads, 4) int8_dot_kernel(const T* __restrict__ x,
                                                                 const int8_t* __restrict__ w, int64_t ldw, Out o,
                                                                 int K, int vec) {
  extern __shared__ __align__(16) int8_t qs[];  // [Kp]
  __shared__ uint32_t red[kDotThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int full = K / 16, Kp = (K + 15) / 16 * 16;
  const int64_t stride = (int64_t)gridDim.x * (kDotThreads / 32);
  int64_t n = (int64_t)blockIdx.x * (kDotThreads / 32) + warp;
  uint4 wv[kDotStep];
  tc::wait_prerequisites();
  auto load = [&](int64_t row, int c0) {
    const int8_t* p = w + row * ldw;
#pragma unroll
    for (int j = 0; j < kDotStep; ++j) {
      const int c = c0 + j * 32 + lane;
      if (c < full) wv[j] = __ldcs(reinterpret_cast<const uint4*>(p + (int64_t)c * 16));
    }
  };
  if (n < o.N) load(n, 0);

  uint32_t m = 0;
#pragma unroll 4
  for (int k = threadIdx.x * 4; k < K; k += kDotThreads * 4) {
    float v[4];
    load4<T>(x, k, K, vec, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, abs_bits(v[i]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kDotThreads / 32; ++i) m = max(m, red[i]);
  float inv;
  const float sx = row_scale(m, inv);
#pragma unroll 4
  for (int k = threadIdx.x * 4; k < Kp; k += kDotThreads * 4) {
    float v[4];
    load4<T>(x, k, K, vec, v);
    *reinterpret_cast<uint32_t*>(qs + k) = pack4(v[0], v[1], v[2], v[3], inv);
  }
  __syncthreads();

  for (; n < o.N; n += stride) {
    int acc = 0;
    for (int c0 = 0; c0 < full; c0 += kDotStep * 32) {
#pragma unroll
      for (int j = 0; j < kDotStep; ++j) {
        const int c = c0 + j * 32 + lane;
        if (c < full) {
          const uint4 qv = *reinterpret_cast<const uint4*>(qs + c * 16);
          acc = __dp4a((int)wv[j].x, (int)qv.x, acc);
          acc = __dp4a((int)wv[j].y, (int)qv.y, acc);
          acc = __dp4a((int)wv[j].z, (int)qv.z, acc);
          acc = __dp4a((int)wv[j].w, (int)qv.w, acc);
        }
      }
      // the next weights of this channel, or the first of the warp's next one
      if (c0 + kDotStep * 32 < full) load(n, c0 + kDotStep * 32);
      else if (n + stride < o.N) load(n + stride, 0);
    }
    const int k = full * 16 + lane;
    if (lane < 16 && k < K) acc += (int)w[n * ldw + k] * (int)qs[k];
    acc = warp_sum_i(acc);
    if (lane == 0) {
      float v = scaled(acc, sx, o.sw[n]);
      if (o.bias != nullptr) v = __fadd_rn(v, bias_at(o, (int)n));
      static_cast<T*>(o.y)[n] = Cvt<T>::from_f(v);
    }
  }
}

// ------------------------------------------------- tensor cores, many tokens
// tcgen05.mma kind::i8, K in blocks of 128 bytes, 256 tokens x 256 channels on a cluster of two CTAs (cta_group::2):
// persistent, each CTA with a TMA producer warp and eight epilogue warps (two per TMEM lane quadrant, half of the
// columns each) that scale and round into a swizzled box of shared memory, 32 rows of 128 bytes, which a TMA store
// empties beside the next box's arithmetic (8192 x 8192 x 512 bf16: 54 us, where filling the result with a constant
// takes 35; with the box read back and stored by the warp 58, before the last waits took a lane to each barrier).  CTA
// 0's MMA warp issues for both, into two accumulators.  Each CTA loads its 128 tokens and half of the channels, 32 KB
// a block where a single CTA of 128 x 256 loads 48: single CTAs were held by what L2 delivers to the SMs, about 15
// TB/s (8192^3: 440 us against 386 in pairs, both with an earlier quantisation; 355 to 375 us now).  All loads of a
// block count on CTA 0's full barrier; its commits reach the empty and accumulator barriers of both; both epilogues
// release the accumulator on CTA 0.  From one commit of the MMA warp to the next it is 509 to 544 SM cycles, about the
// 512 that a block's MMAs take (the commits themselves jitter), so the clock under the power limit bounds it.
constexpr int BM = 128, BKB = 128;
constexpr int kEpiWarps = 8, kTileThreads = 64 + 32 * kEpiWarps;
constexpr int kBox = 32 * 128;  // an epilogue warp's staging: 32 rows of 128 bytes
constexpr int kBandM = 16;                        // M tiles per band of the tile order

constexpr int TM = 2 * BM, BN = 256, B_ROWS = BN / 2;  // a pair's tile, and the channels one CTA loads
constexpr int kTileStage = (BM + B_ROWS) * BKB, kTileStages = 192 * 1024 / kTileStage;

struct TileArgs {
  Out o;
  int kb;       // K blocks
  int mt, nt;   // tiles
  int vec_out;   // rows of y are 16-byte multiples
  int even_out;  // 4-byte multiples
};

// Tile t: bands of kBandM M tiles, M fastest inside a band, so that the CTAs that run together share weights and
// the band's tokens in L2.
__device__ __forceinline__ void tile_of(const TileArgs& p, int t, int& m, int& n) {
  const int band = t / (kBandM * p.nt), m0 = band * kBandM;
  const int gm = p.mt - m0 < kBandM ? p.mt - m0 : kBandM;
  const int r = t - band * kBandM * p.nt;
  n = r / gm;
  m = m0 + (r - n * gm);
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads, 1) int8_tile_kernel(const __grid_constant__ CUtensorMap tmA,
                                                                   const __grid_constant__ CUtensorMap tmB,
                                                                   const __grid_constant__ CUtensorMap tmY,
                                                                   TileArgs p) {
  constexpr int STAGE = kTileStage, NST = kTileStages;
  constexpr uint32_t IDESC = tc::idesc_i8(TM, BN);
  constexpr int BOX_COLS = 128 / (int)sizeof(T);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* staging = ring + NST * STAGE;
  __shared__ __align__(8) uint64_t full_bar[NST], empty_bar[NST], tfull_bar[2], tempty_bar[2], done_bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ int peer_issued_s;  // CTA 0: blocks that CTA 1 loaded
  __shared__ int used_s, tiles_s;  // blocks multiplied and accumulators handed over, by CTA 0 for both
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long budget = g_int8_wait_budget;
  const int total = p.mt * p.nt;
  const uint32_t cta = tc::cluster_ctarank();
  const int t_first = (int)blockIdx.x / 2, t_step = (int)gridDim.x / 2;
  auto stop = [&](int code) {  // a role that gives up stops the others, in both CTAs of a pair
    give_up(&abort_flag, code);
    tc::st_cluster_u32(tc::cluster_addr(tc::smem_u32((const void*)&abort_flag), cta ^ 1u), 1u);
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      tc::mbar_init(&full_bar[s], 1);
      tc::mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(&tfull_bar[a], 1);
      tc::mbar_init(&tempty_bar[a], 2 * kEpiWarps);
    }
    tc::mbar_init(&done_bar, 1);
    tc::fence_barrier_init();
    tc::fence_proxy_async_smem();
    abort_flag = 0;
  }
  if (warp == 1) {
    tc::tmem_alloc_pair(&tmem_base_s, 2 * BN);
    tc::tmem_relinquish_pair();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::cluster_sync();  // both CTAs' barriers exist before either signals the other's
  tc::tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  // By a whole warp, a lane to each of `depth` barriers that n arrivals went round: waits for the last phase of every
  // one; true where all have landed.  One barrier after the other took 1.5 us of every call (2000^3: 17.4 us, so 16.0).
  auto landed = [&](uint64_t* bar, int depth, int n) {
    bool ok = true;
    if (lane < depth && lane < n) {
      const int last = lane + (n - 1 - lane) / depth * depth;
      ok = tc::mbar_wait(&bar[lane], (uint32_t)((last / depth) & 1), nullptr, kWaitBudget);
    }
    return __all_sync(0xffffffffu, ok) != 0;
  };
  int issued_blocks = 0;
  tc::wait_prerequisites();  // the quantised tokens and their scales

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t full0 = tc::cluster_addr(tc::smem_u32(&full_bar[0]), 0u);
    for (int t = t_first; t < total; t += t_step) {
      int m, n;
      tile_of(p, t, m, n);
      const int row = m * TM + (int)cta * BM, col = n * BN + (int)cta * B_ROWS;
      bool ok = true;
      for (int kb = 0; kb < p.kb; ++kb) {
        ok = tc::mbar_wait_warp(&empty_bar[stage], phase ^ 1u, &abort_flag, budget);
        if (!ok) break;
        if (tc::elect_one()) {
          uint8_t* sa = ring + stage * STAGE;
          if (cta == 0) tc::mbar_arrive_expect_tx(&full_bar[stage], 2 * STAGE);
          tc::tma_load_2d_pair(sa, &tmA, kb * BKB, row, full0 + (uint32_t)stage * 8u);
          tc::tma_load_2d_pair(sa + BM * BKB, &tmB, kb * BKB, col, full0 + (uint32_t)stage * 8u);
        }
        ++issued_blocks;
        if (++stage == NST) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) {
        stop(31);
        break;
      }
    }
    if (cta != 0 && lane == 0)  // CTA 0 drains the loads of both after the first cluster barrier
      tc::st_cluster_u32(tc::cluster_addr(tc::smem_u32(&peer_issued_s), 0u), (uint32_t)issued_blocks);
  } else if (warp == 1) {
    if (cta == 0) {
      const uint64_t desc = tc::smem_desc(tc::smem_u32(ring), 16u, 1024u, tc::kLayoutSW128);
      auto commit = [&](uint64_t* bar) {  // to the same barrier of both CTAs
        tc::mma_commit_pair(tc::cluster_addr(tc::smem_u32(bar), 0u));
        tc::mma_commit_pair(tc::cluster_addr(tc::smem_u32(bar), 1u));
      };
      int stage = 0, i = 0, used = 0, tiles = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = t_first; t < total && ok; t += t_step, ++i) {
        const int acc = i & 1;
        ok = tc::mbar_wait_warp(&tempty_bar[acc], ((uint32_t)(i >> 1) & 1u) ^ 1u, &abort_flag, budget);
        if (!ok) {
          stop(32);
          break;
        }
        tc::tc_fence_after();
        for (int kb = 0; kb < p.kb; ++kb) {
          ok = tc::mbar_wait_warp(&full_bar[stage], phase, &abort_flag, budget);
          if (!ok) {
            stop(33);
            break;
          }
          tc::tc_fence_after();
          // the start address of a descriptor is in units of 16 bytes; the ring ends below 2^18
          const uint64_t da = desc + (uint64_t)(stage * (STAGE / 16)), db = da + BM * BKB / 16;
          if (tc::elect_one()) {
#pragma unroll
            for (int k = 0; k < BKB / 32; ++k)
              tc::mma_i8_pair(tmem_base + (uint32_t)(acc * BN), da + k * 2, db + k * 2, IDESC,
                              (kb > 0 || k > 0) ? 1u : 0u);
            commit(&empty_bar[stage]);
            if (kb == p.kb - 1) commit(&tfull_bar[acc]);
          }
          ++used;
          if (kb == p.kb - 1) ++tiles;
          if (++stage == NST) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (used > 0) {  // all MMAs complete before TMEM is freed
        if (tc::elect_one()) tc::mma_commit_pair(tc::cluster_addr(tc::smem_u32(&done_bar), 0u));
        if (!tc::mbar_wait_warp(&done_bar, 0u, nullptr, kWaitBudget)) atomicCAS(&g_int8_status, 0, 36);
      }
      if (lane < 2) {
        tc::st_cluster_u32(tc::cluster_addr(tc::smem_u32(&used_s), (uint32_t)lane), (uint32_t)used);
        tc::st_cluster_u32(tc::cluster_addr(tc::smem_u32(&tiles_s), (uint32_t)lane), (uint32_t)tiles);
      }
    }
  } else {
    const int quad = warp & 3, chalf = (warp - 2) >> 2;
    uint8_t* box = staging + (warp - 2) * kBox;
    int i = 0;
    // the whole warp goes on or leaves: the flag may be set while its lanes read it
    for (int t = t_first; t < total && !__any_sync(0xffffffffu, abort_flag); t += t_step, ++i) {
      int m, n;
      tile_of(p, t, m, n);
      const int acc = i & 1;
      const int row0 = m * TM + (int)cta * BM + quad * 32, row = row0 + lane;
      const float sx = row < p.o.M ? p.o.sx[row] : 0.f;
      float sw[BN / 64], bw[BN / 64];  // of column lane + 32 j of the warp's half, in flight during the wait
#pragma unroll
      for (int j = 0; j < BN / 64; ++j) {
        const int col = n * BN + chalf * (BN / 2) + j * 32 + lane;
        sw[j] = col < p.o.N ? p.o.sw[col] : 0.f;
        bw[j] = col < p.o.N ? bias_at(p.o, col) : 0.f;
      }
      if (!tc::mbar_wait_warp(&tfull_bar[acc], (uint32_t)(i >> 1) & 1u, &abort_flag, budget)) {
        stop(34);
        break;
      }
      tc::tc_fence_after();
      const uint32_t t_row = tmem_base + (uint32_t)(acc * BN + chalf * (BN / 2)) + ((uint32_t)(quad * 32) << 16);
#pragma unroll
      for (int c = 0; c < BN / 2; c += BOX_COLS) {
        const int col0 = n * BN + chalf * (BN / 2) + c;
        uint32_t r[BOX_COLS];
#pragma unroll
        for (int h = 0; h < BOX_COLS; h += 16) tc::tmem_ld16_async(t_row + c + h, r + h);
        tc::tmem_ld_wait(r);
        if (c + BOX_COLS == BN / 2) {  // the accumulator is read: the next tile's products may start
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (cta != 0) tc::mbar_arrive_cluster(tc::cluster_addr(tc::smem_u32(&tempty_bar[acc]), 0u));
            else tc::mbar_arrive(&tempty_bar[acc]);
          }
        }
        float v[BOX_COLS];
#pragma unroll
        for (int e = 0; e < BOX_COLS; ++e)
          v[e] = scaled((int)r[e], sx, __shfl_sync(0xffffffffu, sw[(c + e) / 32], (c + e) % 32));
        if (p.o.bias != nullptr)  // one branch: one for each element would serialise them
#pragma unroll
          for (int e = 0; e < BOX_COLS; ++e)
            v[e] = __fadd_rn(v[e], __shfl_sync(0xffffffffu, bw[(c + e) / 32], (c + e) % 32));
        if (lane == 0) tc::bulk_wait_read<0>();  // the box's last store has read it
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {  // row `lane`, 16-byte piece q at its swizzled place (conflict-free)
          float u[Chunk<T>::N];
#pragma unroll
          for (int j = 0; j < Chunk<T>::N; ++j) u[j] = v[q * Chunk<T>::N + j];
          uint4 w;
          pack_chunk<T>(u, w);
          *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = w;
        }
        if (p.vec_out) {
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < p.o.M && col0 < p.o.N) {
            tc::tma_store_2d(&tmY, box, col0, row0);  // what lies past the last row or column is left out
            tc::bulk_commit();
          }
        } else {  // rows of y that are not 16-byte multiples: piece by piece, along the rows (8192 x 8190: 79 us)
          __syncwarp();
          auto store = [&](auto piece) {
            using P = decltype(piece);
#pragma unroll 8
            for (int rr = 0; rr < 32; ++rr)
#pragma unroll
              for (int byte = lane * (int)sizeof(P); byte < 128; byte += 32 * (int)sizeof(P)) {
                const int col = col0 + byte / (int)sizeof(T);
                const P w = *reinterpret_cast<const P*>(box + rr * 128 + (((byte >> 4) ^ (rr & 7)) << 4) + (byte & 15));
                if (row0 + rr < p.o.M && col < p.o.N)
                  *reinterpret_cast<P*>(static_cast<T*>(p.o.y) + (int64_t)(row0 + rr) * p.o.N + col) = w;
              }
          };
          if (sizeof(T) == 4 || p.even_out) store(uint32_t{});
          else store(uint16_t{});
        }
        __syncwarp();  // the accumulator is read, and the flag voted on, by whole warps
      }
    }
    if (lane == 0) tc::bulk_wait<0>();  // every store is complete before the CTA exits
  }
  tc::tc_fence_before();
  __syncthreads();
  // CTA 0's MMAs read CTA 1's ring and write its TMEM, its commits signal the barriers of both, and CTA 1's loads and
  // epilogue signal CTA 0's.  After the first barrier each knows how many blocks were loaded and multiplied, and waits
  // for the commits' last arrivals at its own barriers: at most one is due at each, since a stage or an accumulator is
  // used again only after both CTAs have seen the last one.  Where only one of them loaded a block (the other gave up)
  // CTA 0 settles that block's count -- the half that never came counted as done, the half on its way expected -- and
  // waits for every phase.  So no load and no arrival is in flight when the second barrier lets both exit.
  tc::cluster_sync();
  if (warp == 0) {
    int bad = landed(empty_bar, NST, used_s) && landed(tfull_bar, 2, tiles_s) ? 0 : 38;
    if (cta == 0) {
      const int own = issued_blocks, peer = peer_issued_s;
      const int lo = own < peer ? own : peer, hi = own < peer ? peer : own;
      if (hi - lo > NST) {  // cannot happen: a stage is loaded again only after both halves of its last load
        bad = 37;
      } else {
        if (lane == 0)
          for (int k = lo; k < hi; ++k) {
            if (k < own) tc::mbar_complete_tx(&full_bar[k % NST], STAGE);
            else tc::mbar_arrive_expect_tx(&full_bar[k % NST], STAGE);
          }
        __syncwarp();
        if (!landed(full_bar, NST, hi)) bad = 35;
      }
    }
    if (bad != 0 && lane == 0) atomicCAS(&g_int8_status, 0, bad);
  }
  __syncwarp();
  tc::cluster_sync_relaxed();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc_pair(tmem_base, 2 * BN);
  }
}

// -------------------------------------------------- tensor cores, few tokens
// The weights take the MMA's 128 rows and TN tokens its columns, and a cluster of `split` CTAs (1, 2, 3, 4, 6 or 8)
// shares K: each sums its part of K in TMEM, puts its int32 tile into its shared memory, and every CTA adds the parts of
// its share of the tokens through distributed shared memory.  So a decoding batch reads the weights with every SM, and
// no workspace or atomics are needed.  The weights' loads start before the quantisation has ended.  48 tokens through
// 11008 x 4096, in 3 parts: 13.7 us with the quantisation and the weights from HBM, 3.4 TB/s; sums over distributed
// shared memory cost about as much as their bytes at 3.3 TB/s, which is why few columns may be split further than many.
constexpr int kPartThreads = 64 + 32 * kEpiWarps, kMaxSplit = 8;

// Two CTAs share an SM, with half of its shared memory each.
__host__ __device__ constexpr int part_stage_bytes(int tn) { return (BM + tn) * BKB; }
__host__ __device__ constexpr int part_stages(int tn) { return 104 * 1024 / part_stage_bytes(tn); }

struct PartOut {
  const int* tile;                     // [TN][128] sums of this CTA's part of K
  const float *sx_s, *sw_s, *bw_s;
  int n0, m0, first, share, vec_out;  // tokens [first, first + share) of the tile are this CTA's
};

// Add the S parts of this CTA's tokens and write them: a warp takes tokens, a lane four channels, with 8 reads in
// flight, 9 where S is 3 and 6 where it is 6 (a read of another CTA's shared memory takes hundreds of cycles).  Each
// thread arrives at the cluster's closing barrier between its last read of another CTA's tile and the stores that use
// it: the reads are done with before any CTA may leave, and the barrier does not wait for these stores.  It does wait
// for the stores of a round before, which a third token at a time saves the parts in threes of up to 30 tokens each.
template <typename T, int S>
__device__ __forceinline__ void reduce_parts(const Out& o, const PartOut& p) {
  constexpr int U = S == 3 ? 3 : kMaxSplit / S, W = kPartThreads / 32;
  const int warp = threadIdx.x >> 5, r4 = (threadIdx.x & 31) * 4, n = p.n0 + r4;
  const float4 sw = *reinterpret_cast<const float4*>(p.sw_s + r4), bw = *reinterpret_cast<const float4*>(p.bw_s + r4);
  const bool whole = p.vec_out && n + 4 <= o.N;
  uint32_t base[S];
#pragma unroll
  for (int z = 0; z < S; ++z) {
    const uint32_t mine = tc::smem_u32(p.tile + p.first * BM + r4);
    base[z] = S == 1 ? mine : tc::cluster_addr(mine, (uint32_t)z);
  }
  const int left = o.M - p.m0 - p.first;
  const int share = p.share < left ? p.share : left;
  if (S > 1 && warp >= share) tc::cluster_arrive();  // nothing to read
  for (int i0 = warp; i0 < share; i0 += U * W) {
    int4 b[U][S];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * W;
      const bool there = i < share && n < o.N;  // what is read is stored
#pragma unroll
      for (int z = 0; z < S; ++z) {
        if constexpr (S > 1) b[u][z] = tc::ld_cluster_v4(base[z] + (uint32_t)i * BM * 4u, there);
        else b[u][z] = there ? *reinterpret_cast<const int4*>(p.tile + (p.first + i) * BM + r4) : make_int4(0, 0, 0, 0);
      }
    }
    if (S > 1 && i0 + U * W >= share) tc::cluster_arrive();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * W;
      int4 a = b[u][0];
#pragma unroll
      for (int z = 1; z < S; ++z) a.x += b[u][z].x, a.y += b[u][z].y, a.z += b[u][z].z, a.w += b[u][z].w;
      const float sx = i < share ? p.sx_s[p.first + i] : 0.f;
      float v[4] = {scaled(a.x, sx, sw.x), scaled(a.y, sx, sw.y), scaled(a.z, sx, sw.z), scaled(a.w, sx, sw.w)};
      if (o.bias != nullptr) {
        v[0] = __fadd_rn(v[0], bw.x), v[1] = __fadd_rn(v[1], bw.y);
        v[2] = __fadd_rn(v[2], bw.z), v[3] = __fadd_rn(v[3], bw.w);
      }
      T* y = static_cast<T*>(o.y) + (int64_t)(p.m0 + p.first + i) * o.N + n;
      if (whole && i < share) {
        T e[4] = {Cvt<T>::from_f(v[0]), Cvt<T>::from_f(v[1]), Cvt<T>::from_f(v[2]), Cvt<T>::from_f(v[3])};
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(e);
        else *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(e);
      } else if (i < share) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < o.N) y[j] = Cvt<T>::from_f(v[j]);
      }
    }
  }
}

template <typename T, int TN>
__global__ void __launch_bounds__(kPartThreads, 2) int8_part_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                   const __grid_constant__ CUtensorMap tmX, Out o,
                                                                   int kb_all, int vec_out) {
  constexpr int STAGE = part_stage_bytes(TN), NST = part_stages(TN);
  constexpr int TCOLS = TN < 32 ? 32 : TN;
  constexpr uint32_t IDESC = tc::idesc_i8(BM, TN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full_bar[NST], empty_bar[NST], tfull_bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int abort_flag;
  __shared__ float sx_s[TN];
  __shared__ __align__(16) float sw_s[BM], bw_s[BM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long budget = g_int8_wait_budget;
  const int split = (int)gridDim.z, part = (int)blockIdx.z;  // the cluster is all of z
  const int kb0 = (int)((int64_t)kb_all * part / split), kb1 = (int)((int64_t)kb_all * (part + 1) / split);
  const int n0 = blockIdx.x * BM, m0 = blockIdx.y * TN;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      tc::mbar_init(&full_bar[s], 1);
      tc::mbar_init(&empty_bar[s], 1);
    }
    tc::mbar_init(&tfull_bar, 1);
    tc::fence_barrier_init();
    tc::fence_proxy_async_smem();
    abort_flag = 0;
  }
  if (warp == 1) {
    tc::tmem_alloc(&tmem_base_s, TCOLS);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;

  const int nkb = kb1 - kb0;
  if (warp == 0) {
    const int ahead = nkb < NST ? nkb : NST;
    if (tc::elect_one())
      for (int s = 0; s < ahead; ++s) {
        tc::mbar_arrive_expect_tx(&full_bar[s], STAGE);
        tc::tma_load_2d(ring + s * STAGE, &tmW, (kb0 + s) * BKB, n0, &full_bar[s]);
      }
    __syncwarp();
    tc::wait_prerequisites();
    if (tc::elect_one())
      for (int s = 0; s < ahead; ++s)
        tc::tma_load_2d(ring + s * STAGE + BM * BKB, &tmX, (kb0 + s) * BKB, m0, &full_bar[s]);
    __syncwarp();
    int issued = ahead, stage = 0;
    uint32_t phase = 0;
    for (int i = ahead; i < nkb; ++i) {
      if (!tc::mbar_wait_warp(&empty_bar[stage], phase, &abort_flag, budget)) {
        give_up(&abort_flag, 41);
        break;
      }
      if (tc::elect_one()) {
        tc::mbar_arrive_expect_tx(&full_bar[stage], STAGE);
        tc::tma_load_2d(ring + stage * STAGE, &tmW, (kb0 + i) * BKB, n0, &full_bar[stage]);
        tc::tma_load_2d(ring + stage * STAGE + BM * BKB, &tmX, (kb0 + i) * BKB, m0, &full_bar[stage]);
      }
      ++issued;
      if (++stage == NST) {
        stage = 0;
        phase ^= 1u;
      }
    }
    for (int s = 0; s < NST && s < issued; ++s) {  // every load issued lands before the CTA may exit
      const int last = s + (issued - 1 - s) / NST * NST;
      if (!tc::mbar_wait(&full_bar[s], (uint32_t)((last / NST) & 1), nullptr, kWaitBudget))
        atomicCAS(&g_int8_status, 0, 45);
    }
  } else if (warp == 1) {
    const uint64_t desc = tc::smem_desc(tc::smem_u32(ring), 16u, 1024u, tc::kLayoutSW128);
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!tc::mbar_wait_warp(&full_bar[stage], phase, &abort_flag, budget)) {
        give_up(&abort_flag, 43);
        break;
      }
      tc::tc_fence_after();
      const uint64_t da = desc + (uint64_t)(stage * (STAGE / 16)), db = da + BM * BKB / 16;
      if (tc::elect_one()) {
#pragma unroll
        for (int k = 0; k < BKB / 32; ++k)
          tc::mma_i8(tmem_base, da + k * 2, db + k * 2, IDESC, (i > 0 || k > 0) ? 1u : 0u);
        tc::mma_commit(&empty_bar[stage]);
      }
      if (++stage == NST) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // also after a wait that gave up: the MMAs issued complete before TMEM is freed
    if (tc::elect_one()) tc::mma_commit(&tfull_bar);
  }
  __syncwarp();
  if (warp >= 2 && warp < 6) {
    const int r = threadIdx.x - 64, n = n0 + r;
    sw_s[r] = n < o.N ? o.sw[n] : 0.f;
    bw_s[r] = n < o.N ? bias_at(o, n) : 0.f;
    tc::wait_prerequisites();  // the tokens' scales
    if (r < TN) sx_s[r] = m0 + r < o.M ? o.sx[m0 + r] : 0.f;
  }
  if (!tc::mbar_wait_warp(&tfull_bar, 0u, nullptr, kWaitBudget)) atomicCAS(&g_int8_status, 0, 44);
  tc::tc_fence_after();
  int* tile = reinterpret_cast<int*>(ring);  // [TN][128]: the ring is no longer read or written
  if (warp >= 2) {
#pragma unroll 2
    for (int c = (warp - 2) / 4 * 16; c < TN; c += 32) {  // two warps per TMEM lane quadrant
      uint32_t r[16];
      tc::tmem_ld16(tmem_base + (uint32_t)c + ((uint32_t)((warp & 3) * 32) << 16), r);
#pragma unroll
      for (int j = 0; j < 16; ++j) tile[(c + j) * BM + (warp & 3) * 32 + lane] = (int)r[j];
    }
  }
  __syncwarp();
  if (split > 1) tc::cluster_sync();
  else __syncthreads();
  const int each = (TN + split - 1) / split, first = part * each;
  const PartOut po{tile, sx_s, sw_s, bw_s, n0, m0, first, TN - first < each ? TN - first : each, vec_out};
  switch (split) {
    case 1: reduce_parts<T, 1>(o, po); break;
    case 2: reduce_parts<T, 2>(o, po); break;
    case 3: reduce_parts<T, 3>(o, po); break;
    case 4: reduce_parts<T, 4>(o, po); break;
    case 6: reduce_parts<T, 6>(o, po); break;
    default: reduce_parts<T, 8>(o, po);
  }
  __syncwarp();
  if (split > 1) tc::cluster_wait();  // no CTA leaves while another reads its tile
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tmem_base, TCOLS);
}

// ---------------------------------------------------------------------- host
int64_t padded_k(int64_t K) { return (K + 15) / 16 * 16; }

size_t q_bytes(int64_t M, int64_t K) { return align_up((size_t)(M * padded_k(K)), 256); }

PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

// Rows [rows, cols] of `es`-byte elements: boxes of 128 bytes x `box_rows`, 128-byte swizzle; what is loaded from past an
// end is 0, what is stored there is left out.
int row_map(CUtensorMap* m, CUtensorMapDataType type, int es, const void* base, int64_t cols, int64_t rows, int64_t ld,
            int box_rows) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  });
  if (g_encode == nullptr) return fail(ATS_ECUDA, "int8_linear: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * es)};
  cuuint32_t box[2] = {(cuuint32_t)(BKB / es), (cuuint32_t)box_rows};
  cuuint32_t step[2] = {1, 1};
  CUresult r = g_encode(m, type, 2, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ATS_ECUDA, "int8_linear: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return ATS_OK;
}

int operand_map(CUtensorMap* m, const int8_t* base, int64_t K, int64_t rows, int64_t ld, int box_rows) {
  return row_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, base, K, rows, ld, box_rows);
}

template <typename T>
int dot(const void* x, const int8_t* w, int64_t ldw, const Out& o, int K, cudaStream_t st) {
  const int warps = kDotThreads / 32;
  // a limit on the GEMMs' SMs leaves one block to each
  const int64_t want = (o.N + warps - 1) / warps, cap = gemm_ctas() < num_sms() ? gemm_ctas() : (int64_t)num_sms() * 4;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  return launch_after<int8_dot_kernel<T>>(dim3(grid), kDotThreads, (int)padded_k(K), dim3(1), st, "int8_dot",
                      static_cast<const T*>(x), w, ldw, o, K, aligned16(x) ? 1 : 0);
}

// Pairs of CTAs that are resident at once on the current device.
template <auto KERNEL>
int pairs_that_fit(int smem, int* out) {
  static thread_local int fit[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return fail(ATS_ECUDA, "int8_tile: no current device");
  if (fit[dev] == 0) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(num_sms() / 2 * 2));
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    ATS_TRY(allow_smem<KERNEL>("int8_tile", true));
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg);
    if (e != cudaSuccess || n < 1) return fail(ATS_ECUDA, "int8_tile: no pair fits (%s)", cudaGetErrorString(e));
    fit[dev] = n;
  }
  *out = fit[dev];
  return ATS_OK;
}

template <typename T>
int tiles(const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, const Out& o, int K, cudaStream_t st) {
  CUtensorMap ma, mb, my;
  ATS_TRY(operand_map(&ma, q, K, o.M, ldq, BM));
  ATS_TRY(operand_map(&mb, w, K, o.N, ldw, B_ROWS));
  const int vec = (int64_t)o.N * (int64_t)sizeof(T) % 16 == 0 && aligned16(o.y);
  if (vec) {
    constexpr auto type = sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    ATS_TRY(row_map(&my, type, (int)sizeof(T), o.y, o.N, o.M, o.N, 32));
  } else {
    my = ma;  // not used
  }
  const TileArgs p{o, (K + BKB - 1) / BKB, (o.M + TM - 1) / TM, (o.N + BN - 1) / BN, vec,
                   o.N % 2 == 0 && reinterpret_cast<uintptr_t>(o.y) % 4 == 0};
  const int64_t total = (int64_t)p.mt * p.nt;
  if (total > 0x7fffffff - 4096) return fail(ATS_EUNSUPPORTED, "int8_linear: too many tiles");
  const int smem = 1024 + kTileStages * kTileStage + kEpiWarps * kBox;
  int pairs = 0;
  ATS_TRY(pairs_that_fit<int8_tile_kernel<T>>(smem, &pairs));
  if (pairs > gemm_ctas() / 2) pairs = gemm_ctas() / 2;
  if (pairs > total) pairs = (int)total;
  if (pairs < 1) pairs = 1;
  return launch_after<int8_tile_kernel<T>>(dim3(2 * (unsigned)pairs), kTileThreads, smem, dim3(2), st, "int8_tile", ma, mb,
                                           my, p);
}

template <typename T, int TN>
int parts(const int8_t* q, int64_t ldq, const int8_t* w, int64_t ldw, const Out& o, int K, int split, cudaStream_t st) {
  CUtensorMap mw, mx;
  ATS_TRY(operand_map(&mw, w, K, o.N, ldw, BM));
  ATS_TRY(operand_map(&mx, q, K, o.M, ldq, TN));
  const dim3 grid((unsigned)((o.N + BM - 1) / BM), (unsigned)((o.M + TN - 1) / TN), (unsigned)split);
  const int smem = 1024 + part_stages(TN) * part_stage_bytes(TN);
  return launch_after<int8_part_kernel<T, TN>>(grid, kPartThreads, smem, dim3(1, 1, (unsigned)split), st, "int8_part", mw, mx, o,
                      (K + BKB - 1) / BKB, o.N % 4 == 0 && aligned16(o.y) ? 1 : 0);
}

template <typename T>
int linear(const void* x, int64_t ldx, const int8_t* w, int64_t ldw, Out o, int64_t K, int8_t* q, float* sx,
           cudaStream_t st) {
  if (o.M == 1 && K <= kDotLongest) return dot<T>(x, w, ldw, o, (int)K, st);
  const int64_t ldq = padded_k(K);
  ATS_TRY(quantize_t<T>(x, ldx, q, ldq, sx, o.M, K, st));
  o.sx = sx;
  // Few tiles of 128 channels: as many token columns as hold the tokens, at most 64, or 128 where 64 would make more
  // than two CTAs per SM.
  // Under a limit on the GEMMs' SMs the parts get one CTA to an SM, and what does not fit takes the persistent pairs.
  const int sms = gemm_ctas();
  const int64_t nt = (o.N + BM - 1) / BM, two = sms < num_sms() ? sms : 2 * (int64_t)sms;
  const int kb = (int)((K + BKB - 1) / BKB);
  const int tn = o.M <= 16 ? 16 : o.M <= 32 ? 32 : nt * ((o.M + 63) / 64) <= two ? 64 : 128;
  const int64_t mt = (o.M + tn - 1) / tn, ctas = nt * mt;
  // One round of pair tiles beats two CTAs to an SM where it keeps three quarters of the pairs busy (from L2,
  // 2000^3: 16.8 us against 20.4; 3000 x 1000 x 1000, 48 tiles: 13.7 against 14.3; 1024 x 2048 x 4096, 32 tiles: 19.0
  // against 15.6; the pair tiles' last waits have since become shorter, 2000^3 16.0).
  const int64_t pair_tiles = ((o.M + TM - 1) / TM) * ((o.N + BN - 1) / (int64_t)BN);
  const bool one_round = ctas > sms && tn == 128 && 8 * pair_tiles >= 3 * (int64_t)sms;
  if (ctas > two || mt > 65535 || one_round) return tiles<T>(q, ldq, w, ldw, o, (int)K, st);
  // K is split so that the fullest SM, of one or two CTAs, has the least to do, where each part has 2 blocks of K, or 8
  // where SMs have two parts, and at most 256 columns are summed; for the same load into more parts where each still
  // has 16 blocks.  In us, one sweep of the same tokens: 48 tokens 4096x11008 25.7 whole, 16.6 in 2, 12.6 in 4, 16.2
  // in 8; 48 tokens 11008x4096 14.3 in 2, 12.9 in 3; 200 tokens 2048x8192 14.5 in 2, 13.2 in 4; 500 tokens 2048x2048 8.6
  // whole, 9.3 in 2.  (Those chosen, each call with tokens and weights of its own from HBM: 14.1 to 14.7, 13.7, 13.5 and
  // 9.3 to 9.6.)  Clusters of 3
  // or 6 leave places free that others fill: 288 CTAs in clusters of 3 did not fit on 148 SMs at once (100 tokens
  // 6144x4096: 16.7 in 3, 12.3 in 2), so they get nine tenths of the places.
  int split = 1;
  double load = (double)((ctas + sms - 1) / sms);  // in whole tiles
  for (int n : {2, 3, 4, 6, 8}) {
    const int64_t all = n * ctas;
    if (n * tn > 256 || all > ((n & (n - 1)) == 0 ? two : two * 9 / 10) || kb < n * (all <= sms ? 2 : 8)) continue;
    const double l = (double)((all + sms - 1) / sms) / n;
    if (l < load || (l == load && kb >= 16 * n)) load = l, split = n;
  }
  switch (tn) {
    case 16: return parts<T, 16>(q, ldq, w, ldw, o, (int)K, split, st);
    case 32: return parts<T, 32>(q, ldq, w, ldw, o, (int)K, split, st);
    case 64: return parts<T, 64>(q, ldq, w, ldw, o, (int)K, split, st);
    default: return parts<T, 128>(q, ldq, w, ldw, o, (int)K, split, st);
  }
}

}  // namespace

int int8_set_wait_budget(long long cycles) {
  const long long v = cycles > 0 ? cycles : kWaitBudget;
  cudaError_t e = cudaMemcpyToSymbol(g_int8_wait_budget, &v, sizeof(v));
  if (e != cudaSuccess) return fail(ATS_ECUDA, "set_wait_budget (int8): %s", cudaGetErrorString(e));
  return ATS_OK;
}

int int8_take_status(int* code) {
  const int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(code, g_int8_status, sizeof(int));
  if (e == cudaSuccess && *code != 0) e = cudaMemcpyToSymbol(g_int8_status, &zero, sizeof(int));
  if (e != cudaSuccess) return fail(ATS_ECUDA, "device_status (int8): %s", cudaGetErrorString(e));
  return ATS_OK;
}

}  // namespace ats

using namespace ats;

extern "C" {

int ats_int8_quantize(const void* x, int64_t x_row_stride, ats_dtype dtype, void* q, int64_t q_row_stride,
                      float* scale, int64_t rows, int64_t K, void* stream) {
  if (dtype != ATS_F32 && dtype != ATS_BF16) return fail(ATS_EBADARG, "int8_quantize: dtype");
  if (rows < 0 || rows > kMaxRows || K < 1 || K > kMaxK || q_row_stride < K || x_row_stride < 0)
    return fail(ATS_EBADARG, "int8_quantize: rows=%lld K=%lld (at most %d) row stride %lld", (long long)rows,
                (long long)K, kMaxK, (long long)q_row_stride);
  if (rows == 0) return ATS_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return fail(ATS_EBADARG, "int8_quantize: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == ATS_BF16 ? quantize_t<bf16>(x, x_row_stride, q, q_row_stride, scale, rows, K, st)
                           : quantize_t<float>(x, x_row_stride, q, q_row_stride, scale, rows, K, st);
}

size_t ats_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 1 || K < 1 || (M == 1 && K <= kDotLongest)) return 0;  // one token is quantised where it is used
  return q_bytes(M, K) + align_up((size_t)M * sizeof(float), 256);
}

int ats_int8_linear(const void* x, int64_t x_row_stride, ats_dtype dtype, const void* w, int64_t w_row_stride,
                    const float* w_scale, const void* bias, ats_dtype bias_dtype, void* y, int64_t M, int64_t N,
                    int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != ATS_F32 && dtype != ATS_BF16) return fail(ATS_EBADARG, "int8_linear: dtype");
  if (bias != nullptr && bias_dtype != ATS_F32 && bias_dtype != ATS_BF16)
    return fail(ATS_EBADARG, "int8_linear: bias dtype");
  if (M < 0 || M > kMaxRows || N < 1 || N > kMaxRows || K < 1 || K > kMaxK || x_row_stride < 0)
    return fail(ATS_EBADARG, "int8_linear: M=%lld N=%lld K=%lld (K at most %d)", (long long)M, (long long)N,
                (long long)K, kMaxK);
  if (w_row_stride < K || w_row_stride % 16 != 0 || !aligned16(w))
    return fail(ATS_EBADARG, "int8_linear: weight rows must start every multiple of 16 bytes (row stride %lld)",
                (long long)w_row_stride);
  if (M == 0) return ATS_OK;
  if (x == nullptr || w == nullptr || w_scale == nullptr || y == nullptr)
    return fail(ATS_EBADARG, "int8_linear: null pointer");
  const size_t need = ats_int8_linear_workspace_bytes(M, N, K);
  if (need > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < need))
    return fail(ATS_EBADARG, "int8_linear: workspace too small");
  int8_t* q = static_cast<int8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(q + q_bytes(M, K));
  const int8_t* wp = static_cast<const int8_t*>(w);
  const Out o{y, nullptr, w_scale, bias, bias_dtype == ATS_BF16, (int)M, (int)N};
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == ATS_BF16 ? linear<bf16>(x, x_row_stride, wp, w_row_stride, o, K, q, sx, st)
                           : linear<float>(x, x_row_stride, wp, w_row_stride, o, K, q, sx, st);
}

}  // extern "C"
