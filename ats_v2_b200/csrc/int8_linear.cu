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
#include "common.cuh"

namespace ats {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kMaxK = 131072;

// |v| as an unsigned integer orders like |v|, and puts NaN above infinity above every number.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t warp_max_u(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }

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

__device__ __forceinline__ int quant(float v, float inv) {
  const float r = rintf(v * inv);
  return r == r ? (int)fminf(fmaxf(r, -127.f), 127.f) : 0;
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) int8_quantize_kernel(const T* __restrict__ x, int64_t ldx,
                                                                     int8_t* __restrict__ q, int64_t ldq,
                                                                     float* __restrict__ scale, int64_t rows, int K) {
  __shared__ uint32_t red[kQuantThreads / 32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  uint32_t m = 0;
  for (int k = threadIdx.x; k < K; k += kQuantThreads) {
    const uint32_t b = abs_bits(Cvt<T>::to_f(xr[k]));
    m = b > m ? b : m;
  }
  m = warp_max_u(m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int i = 0; i < kQuantThreads / 32; ++i) m = red[i] > m ? red[i] : m;
  float inv;
  const float s = row_scale(m, inv);
  if (threadIdx.x == 0) scale[row] = s;
  for (int k = threadIdx.x; k < K; k += kQuantThreads) q[row * ldq + k] = (int8_t)quant(Cvt<T>::to_f(xr[k]), inv);
  for (int64_t k = K + threadIdx.x; k < ldq; k += kQuantThreads) q[row * ldq + k] = 0;
}

// A warp per output channel and kTok tokens.
constexpr int kTok = 4, kDotWarps = 8;

template <typename T>
__global__ void __launch_bounds__(32 * kDotWarps) int8_dot_kernel(const int8_t* __restrict__ q, int64_t ldq,
                                                                 const float* __restrict__ sx,
                                                                 const int8_t* __restrict__ w, int64_t ldw,
                                                                 const float* __restrict__ sw, const void* bias,
                                                                 int bias_bf16, T* __restrict__ y, int64_t M,
                                                                 int64_t N, int K) {
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * kDotWarps + (threadIdx.x >> 5);
  if (n >= N) return;
  for (int64_t m0 = (int64_t)blockIdx.y * kTok; m0 < M; m0 += (int64_t)gridDim.y * kTok) {
    const int nt = M - m0 < kTok ? (int)(M - m0) : kTok;
    int acc[kTok] = {};
    const int full = K / 16;
    for (int c = lane; c < full; c += 32) {
      const uint4 wv = *reinterpret_cast<const uint4*>(w + n * ldw + (int64_t)c * 16);
#pragma unroll
      for (int t = 0; t < kTok; ++t)
        if (t < nt) {
          const uint4 qv = *reinterpret_cast<const uint4*>(q + (m0 + t) * ldq + (int64_t)c * 16);
          acc[t] = __dp4a((int)wv.x, (int)qv.x, acc[t]);
          acc[t] = __dp4a((int)wv.y, (int)qv.y, acc[t]);
          acc[t] = __dp4a((int)wv.z, (int)qv.z, acc[t]);
          acc[t] = __dp4a((int)wv.w, (int)qv.w, acc[t]);
        }
    }
    const int k = full * 16 + lane;
    if (lane < 16 && k < K)
#pragma unroll
      for (int t = 0; t < kTok; ++t)
        if (t < nt) acc[t] += (int)w[n * ldw + k] * (int)q[(m0 + t) * ldq + k];
#pragma unroll
    for (int t = 0; t < kTok; ++t) {
      const int a = warp_sum_i(acc[t]);
      if (lane == 0 && t < nt) {
        float v = (float)a * (sx[m0 + t] * sw[n]);
        if (bias != nullptr)
          v += bias_bf16 ? __bfloat162float(static_cast<const bf16*>(bias)[n]) : static_cast<const float*>(bias)[n];
        y[(m0 + t) * N + n] = Cvt<T>::from_f(v);
      }
    }
  }
}

template <typename T>
int quantize_t(const void* x, int64_t ldx, void* q, int64_t ldq, float* scale, int64_t rows, int64_t K,
               cudaStream_t st) {
  int8_quantize_kernel<T><<<(unsigned)rows, kQuantThreads, 0, st>>>(static_cast<const T*>(x), ldx,
                                                                   static_cast<int8_t*>(q), ldq, scale, rows, (int)K);
  return check_launch("int8_quantize");
}

int64_t padded_k(int64_t K) { return (K + 15) / 16 * 16; }

size_t q_bytes(int64_t M, int64_t K) { return align_up((size_t)(M * padded_k(K)), 256); }

}  // namespace
}  // namespace ats

using namespace ats;

extern "C" {

int ats_int8_quantize(const void* x, int64_t x_row_stride, ats_dtype dtype, void* q, int64_t q_row_stride,
                      float* scale, int64_t rows, int64_t K, void* stream) {
  if (dtype != ATS_F32 && dtype != ATS_BF16) return fail(ATS_EBADARG, "int8_quantize: dtype");
  if (rows < 0 || rows > 0x7fffffff || K < 1 || K > kMaxK || q_row_stride < K || x_row_stride < 0)
    return fail(ATS_EBADARG, "int8_quantize: rows=%lld K=%lld (at most %d) row stride %lld", (long long)rows,
                (long long)K, kMaxK, (long long)q_row_stride);
  if (rows == 0) return ATS_OK;
  if (x == nullptr || q == nullptr || scale == nullptr) return fail(ATS_EBADARG, "int8_quantize: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == ATS_BF16 ? quantize_t<bf16>(x, x_row_stride, q, q_row_stride, scale, rows, K, st)
                           : quantize_t<float>(x, x_row_stride, q, q_row_stride, scale, rows, K, st);
}

size_t ats_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 1 || K < 1) return 0;
  return q_bytes(M, K) + align_up((size_t)M * sizeof(float), 256);
}

int ats_int8_linear(const void* x, int64_t x_row_stride, ats_dtype dtype, const void* w, int64_t w_row_stride,
                    const float* w_scale, const void* bias, ats_dtype bias_dtype, void* y, int64_t M, int64_t N,
                    int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (dtype != ATS_F32 && dtype != ATS_BF16) return fail(ATS_EBADARG, "int8_linear: dtype");
  if (bias != nullptr && bias_dtype != ATS_F32 && bias_dtype != ATS_BF16)
    return fail(ATS_EBADARG, "int8_linear: bias dtype");
  if (M < 0 || M > 0x7fffffff || N < 1 || N > 0x7fffffff || K < 1 || K > kMaxK || x_row_stride < 0)
    return fail(ATS_EBADARG, "int8_linear: M=%lld N=%lld K=%lld (K at most %d)", (long long)M, (long long)N,
                (long long)K, kMaxK);
  if (w_row_stride < K || w_row_stride % 16 != 0 || !aligned16(w))
    return fail(ATS_EBADARG, "int8_linear: weight rows must start every multiple of 16 bytes (row stride %lld)",
                (long long)w_row_stride);
  if (M == 0) return ATS_OK;
  if (x == nullptr || w == nullptr || w_scale == nullptr || y == nullptr)
    return fail(ATS_EBADARG, "int8_linear: null pointer");
  if (workspace == nullptr || !aligned16(workspace) || workspace_bytes < ats_int8_linear_workspace_bytes(M, N, K))
    return fail(ATS_EBADARG, "int8_linear: workspace too small");
  int8_t* q = static_cast<int8_t*>(workspace);
  float* sx = reinterpret_cast<float*>(q + q_bytes(M, K));
  const int64_t ldq = padded_k(K);
  cudaStream_t st = (cudaStream_t)stream;
  ATS_TRY(ats_int8_quantize(x, x_row_stride, dtype, q, ldq, sx, M, K, stream));
  const int64_t mt = (M + kTok - 1) / kTok;
  const dim3 grid((unsigned)((N + kDotWarps - 1) / kDotWarps), (unsigned)(mt < 65535 ? mt : 65535));
  const int8_t* wp = static_cast<const int8_t*>(w);
  if (dtype == ATS_BF16)
    int8_dot_kernel<bf16><<<grid, 32 * kDotWarps, 0, st>>>(q, ldq, sx, wp, w_row_stride, w_scale, bias,
                                                         bias_dtype == ATS_BF16, static_cast<bf16*>(y), M, N, (int)K);
  else
    int8_dot_kernel<float><<<grid, 32 * kDotWarps, 0, st>>>(q, ldq, sx, wp, w_row_stride, w_scale, bias,
                                                          bias_dtype == ATS_BF16, static_cast<float*>(y), M, N, (int)K);
  return check_launch("int8_dot");
}

}  // extern "C"
