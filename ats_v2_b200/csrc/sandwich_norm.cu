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
#include "common.cuh"

namespace ats {
namespace {

constexpr int kMaxThreads = 1024;
constexpr int kReduceCols = 32, kReduceLanes = 32;

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

template <typename T>
__global__ void __launch_bounds__(kMaxThreads) sandwich_fwd_kernel(NormArgs p, int gate) {
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
__global__ void __launch_bounds__(kMaxThreads) sandwich_bwd_kernel(NormArgs p, int gate) {
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

// Column sums of n rows of `part` for 32 columns, by 32 lanes of rows and then the lanes in order; valid in lane 0.
__device__ __forceinline__ float column_sum(const float* part, int64_t n, int H, int col, int rl,
                                            float (*red)[kReduceCols + 1]) {
  const int cl = threadIdx.x % kReduceCols;
  float t = 0.f;
  if (col < H)
    for (int64_t q = rl; q < n; q += kReduceLanes) t += part[q * H + col];
  __syncthreads();
  red[rl][cl] = t;
  __syncthreads();
  float u = 0.f;
  if (rl == 0)
    for (int q = 0; q < kReduceLanes; ++q) u += red[q][cl];
  return u;
}

__device__ __forceinline__ void store_as(void* p, int64_t i, int is_bf16, float v) {
  if (is_bf16) static_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// One span: dgate = w_post A, and gate A into row `span` of part_a's first rows' place for the sum over spans.
__global__ void __launch_bounds__(kReduceCols* kReduceLanes) sandwich_gate_kernel(NormArgs p, float* gate_a) {
  __shared__ float red[kReduceLanes][kReduceCols + 1];
  const int cl = threadIdx.x % kReduceCols, rl = threadIdx.x / kReduceCols;
  const int col = blockIdx.x * kReduceCols + cl;
  const int64_t spans = p.rows / p.span;
  for (int64_t i = blockIdx.y; i < spans; i += gridDim.y) {
    const float A = column_sum(p.part_a + i * p.units_per_span * p.H, p.units_per_span, p.H, col, rl, red);
    if (rl == 0 && col < p.H) {
      store_as(p.dgate, i * p.H + col, p.gate_bf16, load_as(p.w_post, col, p.w_bf16) * A);
      gate_a[i * p.H + col] = load_as(p.gate, i * p.H + col, p.gate_bf16) * A;
    }
  }
}

__global__ void __launch_bounds__(kReduceCols* kReduceLanes) sandwich_dw_kernel(NormArgs p, const float* a, int64_t na,
                                                                               int64_t nb, void* dw_post,
                                                                               void* dw_pre) {
  __shared__ float red[kReduceLanes][kReduceCols + 1];
  const int cl = threadIdx.x % kReduceCols, rl = threadIdx.x / kReduceCols;
  const int col = blockIdx.x * kReduceCols + cl;
  const float A = column_sum(a, na, p.H, col, rl, red);
  const float Bp = column_sum(p.part_b, nb, p.H, col, rl, red);
  if (rl == 0 && col < p.H) {
    store_as(dw_post, col, p.w_bf16, A);
    store_as(dw_pre, col, p.w_bf16, Bp);
  }
}

struct BwdPlan {
  int64_t spans, units, blocks;
  int units_per_span;
};

// Row ranges of the backward: about two blocks per SM, none across a span.
BwdPlan bwd_plan(int64_t rows, int64_t span, int gate) {
  BwdPlan b;
  if (gate != GATE_SPAN) span = rows;
  b.spans = rows / span;
  const int64_t want = (int64_t)num_sms() * 2;
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
  const int64_t cap = (int64_t)num_sms() * 16;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == ATS_BF16) sandwich_fwd_kernel<bf16><<<grid, threads_for(hidden), 0, st>>>(p, g);
  else sandwich_fwd_kernel<float><<<grid, threads_for(hidden), 0, st>>>(p, g);
  return check_launch("sandwich_norm_fwd");
}

size_t ats_sandwich_norm_bwd_workspace_bytes(int64_t rows, int64_t hidden, int64_t rows_per_gate) {
  if (rows <= 0 || hidden <= 0 || rows_per_gate < 0 || (rows_per_gate > 0 && rows % rows_per_gate != 0)) return 0;
  const BwdPlan b = bwd_plan(rows, rows_per_gate > 1 ? rows_per_gate : rows, rows_per_gate > 1 ? GATE_SPAN : GATE_NONE);
  return (size_t)(b.units + b.blocks + (rows_per_gate > 1 ? b.spans : 0)) * (size_t)hidden * sizeof(float);
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
  if (workspace == nullptr ||
      workspace_bytes < ats_sandwich_norm_bwd_workspace_bytes(rows, hidden, gate != nullptr ? rows_per_gate : 0))
    return fail(ATS_EBADARG, "sandwich_norm_bwd: workspace too small");
  const BwdPlan b = bwd_plan(rows, rows_per_gate, g);
  NormArgs p{};
  p.x = x, p.res = residual, p.dh = dh, p.ds = dsum, p.dx = dx, p.dres = dresidual;
  p.w_post = w_post, p.w_pre = w_pre, p.gate = gate, p.dgate = dgate;
  p.w_bf16 = w_dtype == ATS_BF16, p.gate_bf16 = gate_dtype == ATS_BF16;
  p.rx = const_cast<float*>(rstd_x), p.rs = const_cast<float*>(rstd_sum);
  p.rows = rows, p.span = g == GATE_SPAN ? rows_per_gate : rows;
  p.H = (int)hidden, p.scale = residual_scale;
  p.units_per_span = b.units_per_span, p.units = b.units;
  p.part_a = static_cast<float*>(workspace);
  p.part_b = p.part_a + b.units * hidden;
  float* gate_a = p.part_b + b.blocks * hidden;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == ATS_BF16) sandwich_bwd_kernel<bf16><<<(unsigned)b.blocks, threads_for(hidden), 0, st>>>(p, g);
  else sandwich_bwd_kernel<float><<<(unsigned)b.blocks, threads_for(hidden), 0, st>>>(p, g);
  ATS_TRY(check_launch("sandwich_norm_bwd"));
  const unsigned cols = (unsigned)((hidden + kReduceCols - 1) / kReduceCols);
  const float* a = p.part_a;
  int64_t na = b.units;
  if (g == GATE_SPAN) {
    sandwich_gate_kernel<<<dim3(cols, (unsigned)(b.spans < 1024 ? b.spans : 1024)), kReduceCols * kReduceLanes, 0, st>>>(
        p, gate_a);
    ATS_TRY(check_launch("sandwich_gate"));
    a = gate_a, na = b.spans;
  }
  sandwich_dw_kernel<<<cols, kReduceCols * kReduceLanes, 0, st>>>(p, a, na, b.blocks, dw_post, dw_pre);
  return check_launch("sandwich_dw");
}

}  // extern "C"
