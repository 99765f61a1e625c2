// Rotary embedding with several position axes (time, height, width of images
// and video) for q and k in one launch, forward and adjoint.
//
// Pair j of a head joins columns j and j + pairs; its angle at a token is
//   pos[axis(j)][token] * inv_freq[j]
// and (a, b) -> (a cos - b sin, b cos + a sin); columns past 2*pairs are copied.
// The adjoint negates the sine.  The arithmetic is float32, rounded once.
//
// The angle is formed in turns, pos * inv_freq / 2pi, in two doubles and
// reduced to about [-1/2, 1/2] there, so a far position loses nothing; the sine
// and cosine of the remainder are float32 (sincospif).  A block owns a few tokens
// and all (or a share) of their heads: it computes the tokens' cosines and
// sines once into shared memory, so that work is spread over the heads, and
// then streams the heads through registers.  Every element is read once and
// written once; HBM bounds it.
#include "common.cuh"

namespace ats {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;          // rows in flight per thread
constexpr int kItemsPerThread = 8;  // vectors a thread handles in a full block
constexpr double kInv2PiHi = 0.15915494309189535, kInv2PiLo = -9.839338337591243e-18;  // 1 / (2 pi) in two parts
constexpr int kTableMax = 2048;     // cosine/sine entries of a block (16 KB)

struct AxesTensor {
  const void* in;
  void* out;
  int heads;
  int64_t is_b, is_h, is_s, os_b, os_h, os_s;  // strides in elements
};

struct AxesArgs {
  AxesTensor q, k;
  const void* pos;
  int pos_type;
  int64_t ps_a, ps_b, ps_s;
  const float* inv_freq;
  int64_t n_tokens, S;
  int D, pairs;
  int tokens_per_block, heads_per_block;
  float sign;  // of the sine: +1 forward, -1 adjoint
  uint8_t axis[ATS_ROPE_MAX_PAIRS];
};

// V consecutive elements of T moved as one access.
template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };

__device__ __forceinline__ double load_pos(const AxesArgs& p, int64_t i) {
  if (p.pos_type == ATS_POS_I64) return (double)static_cast<const int64_t*>(p.pos)[i];
  if (p.pos_type == ATS_POS_I32) return (double)static_cast<const int32_t*>(p.pos)[i];
  return (double)static_cast<const float*>(p.pos)[i];
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const __grid_constant__ AxesArgs p) {
  using R = typename Raw<V * (int)sizeof(T)>::type;
  extern __shared__ float table[];  // cosines [tokens][pairs], then sines
  const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
  const int ntok = (int)(p.n_tokens - tok0 < p.tokens_per_block ? p.n_tokens - tok0 : p.tokens_per_block);
  const int heads_all = p.q.heads + p.k.heads;
  const int h0 = blockIdx.y * p.heads_per_block;
  const int nh = heads_all - h0 < p.heads_per_block ? heads_all - h0 : p.heads_per_block;
  float* cosv = table;
  float* sinv = table + p.tokens_per_block * p.pairs;
  const unsigned rows = (unsigned)ntok * nh;  // (token, head) rows of this block

  // address of row r (token-major): the row's first element in the input and the output
  auto locate = [&](unsigned r, const T*& src, T*& dst, int& t) {
    t = (int)(r / (unsigned)nh);
    const int h = h0 + (int)(r - (unsigned)t * nh);
    const int64_t tok = tok0 + t;
    const int64_t b = tok / p.S, s = tok - b * p.S;
    const bool isq = h < p.q.heads;
    const AxesTensor& x = isq ? p.q : p.k;
    const int hh = isq ? h : h - p.q.heads;
    src = static_cast<const T*>(x.in) + b * x.is_b + hh * x.is_h + s * x.is_s;
    dst = static_cast<T*>(x.out) + b * x.os_b + hh * x.os_h + s * x.os_s;
  };

  // a thread keeps one vector position of the pairs and walks the rows
  const int vecs = p.pairs / V;
  const int rows_per_step = kThreads / vecs;
  const int my_row = threadIdx.x / vecs;
  const int col = (threadIdx.x - my_row * vecs) * V;
  const bool active = my_row < rows_per_step;
  R ra[kUnroll], rb[kUnroll];
  auto load = [&](unsigned base) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned r = base + u * rows_per_step;
      if (active && r < rows) {
        const T* src;
        T* dst;
        int t;
        locate(r, src, dst, t);
        ra[u] = *reinterpret_cast<const R*>(src + col);
        rb[u] = *reinterpret_cast<const R*>(src + col + p.pairs);
      }
    }
  };
  load(my_row);  // in flight while the table is computed

  for (int i = threadIdx.x; i < ntok * p.pairs; i += kThreads) {
    const int t = i / p.pairs, j = i - t * p.pairs;
    const int64_t tok = tok0 + t;
    const int64_t b = tok / p.S, s = tok - b * p.S;
    const double pos = load_pos(p, p.axis[j] * p.ps_a + b * p.ps_b + s * p.ps_s);
    const double f = (double)p.inv_freq[j];
    // f / 2pi as a sum of two doubles, so that the fraction of a turn is right for every position below 2^53
    const double c = f * kInv2PiHi, c_low = fma(f, kInv2PiHi, -c) + f * kInv2PiLo;
    const double t_high = pos * c;
    const float rest = (float)((t_high - rint(t_high)) + (fma(pos, c, -t_high) + pos * c_low));
    float sn, cs;
    sincospif(2.0f * rest, &sn, &cs);
    cosv[i] = cs;
    sinv[i] = sn * p.sign;
  }
  __syncthreads();

  for (unsigned base = my_row; base < rows; base += kUnroll * rows_per_step) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const unsigned r = base + u * rows_per_step;
      if (active && r < rows) {
        const T* src;
        T* dst;
        int t;
        locate(r, src, dst, t);
        const float* cs = cosv + t * p.pairs + col;
        const float* sn = sinv + t * p.pairs + col;
        const T* a = reinterpret_cast<const T*>(&ra[u]);
        const T* b = reinterpret_cast<const T*>(&rb[u]);
        R oa, ob;
        T* pa = reinterpret_cast<T*>(&oa);
        T* pb = reinterpret_cast<T*>(&ob);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = Cvt<T>::to_f(a[i]), y = Cvt<T>::to_f(b[i]);
          pa[i] = Cvt<T>::from_f(x * cs[i] - y * sn[i]);
          pb[i] = Cvt<T>::from_f(y * cs[i] + x * sn[i]);
        }
        *reinterpret_cast<R*>(dst + col) = oa;
        *reinterpret_cast<R*>(dst + col + p.pairs) = ob;
      }
    }
    load(base + kUnroll * rows_per_step);
  }

  // columns that are not rotated
  const int rest = (p.D - 2 * p.pairs) / V;
  for (int64_t i = threadIdx.x; i < (int64_t)rows * rest; i += kThreads) {
    const unsigned r = (unsigned)(i / rest);
    const int c = 2 * p.pairs + (int)(i - (int64_t)r * rest) * V;
    const T* src;
    T* dst;
    int t;
    locate(r, src, dst, t);
    *reinterpret_cast<R*>(dst + c) = *reinterpret_cast<const R*>(src + c);
  }
}

// Elements one access may move: the largest power of two (at most 16 bytes) that divides the pairs, the copied
// columns and every stride, and to which every pointer is aligned.
int vector_width(const AxesArgs& p, int elem) {
  int64_t bits = p.pairs | (p.D - 2 * p.pairs);
  uintptr_t addr = 0;
  for (const AxesTensor* t : {&p.q, &p.k}) {
    if (t->heads == 0) continue;
    bits |= t->is_b | t->is_h | t->is_s | t->os_b | t->os_h | t->os_s;
    addr |= reinterpret_cast<uintptr_t>(t->in) | reinterpret_cast<uintptr_t>(t->out);
  }
  int v = 16 / elem;
  while (v > 1 && (bits % v != 0 || addr % (uintptr_t)(v * elem) != 0)) v >>= 1;
  return v;
}

template <typename T, int V>
int launch_v(AxesArgs& p, cudaStream_t st) {
  const int heads = p.q.heads + p.k.heads;
  // Tokens per block: about kItemsPerThread vectors a thread, within the table.  The heads are split over
  // blocks only where the tokens alone leave SMs idle.
  const int64_t per_token = (int64_t)heads * (p.pairs / V);
  int64_t tpb = ((int64_t)kThreads * kItemsPerThread + per_token - 1) / per_token;
  if (tpb > kTableMax / p.pairs) tpb = kTableMax / p.pairs;
  const int64_t spread = (p.n_tokens + num_sms() - 1) / num_sms();
  if (tpb > spread) tpb = spread;
  if (tpb < 1) tpb = 1;
  const int64_t blocks = (p.n_tokens + tpb - 1) / tpb;
  if (blocks > 0x7fffffff) return fail(ATS_EUNSUPPORTED, "rope_axes: too many tokens");
  int64_t parts = (num_sms() + blocks - 1) / blocks;
  if (parts > heads) parts = heads;
  p.tokens_per_block = (int)tpb;
  p.heads_per_block = (int)((heads + parts - 1) / parts);
  const unsigned gy = (unsigned)((heads + p.heads_per_block - 1) / p.heads_per_block);
  if (gy > 65535) return fail(ATS_EUNSUPPORTED, "rope_axes: too many heads");
  const size_t smem = (size_t)tpb * p.pairs * 2 * sizeof(float);
  rope_axes_kernel<T, V><<<dim3((unsigned)blocks, gy), kThreads, smem, st>>>(p);
  return check_launch("rope_axes_apply");
}

}  // namespace
}  // namespace ats

using namespace ats;

extern "C" int ats_rope_axes_apply(const void* q_in, void* q_out, int64_t Hq, const int64_t q_in_strides[3],
                                   const int64_t q_out_strides[3], const void* k_in, void* k_out, int64_t Hk,
                                   const int64_t k_in_strides[3], const int64_t k_out_strides[3],
                                   const void* positions, int pos_type, const int64_t pos_strides[3], int axes,
                                   const float* inv_freq, const uint8_t* axis_of_pair, int pairs, int64_t B,
                                   int64_t S, int64_t D, ats_dtype x_dtype, int backward, void* stream) {
  if (B < 0 || S < 0 || D <= 0 || D > (1 << 20) || pairs <= 0 || pairs > ATS_ROPE_MAX_PAIRS || 2 * (int64_t)pairs > D ||
      Hq < 0 || Hq > (1 << 20))
    return fail(ATS_EBADARG, "rope_axes: bad shape B=%lld S=%lld D=%lld pairs=%d Hq=%lld", (long long)B, (long long)S,
                (long long)D, pairs, (long long)Hq);
  if (x_dtype != ATS_F32 && x_dtype != ATS_BF16) return fail(ATS_EBADARG, "rope_axes: unsupported dtype");
  if (pos_type != ATS_POS_I32 && pos_type != ATS_POS_I64 && pos_type != ATS_POS_F32)
    return fail(ATS_EBADARG, "rope_axes: unsupported position type %d", pos_type);
  if (axes < 1 || axes > 256 || axis_of_pair == nullptr) return fail(ATS_EBADARG, "rope_axes: axes");
  for (int j = 0; j < pairs; ++j)
    if (axis_of_pair[j] >= axes) return fail(ATS_EBADARG, "rope_axes: pair %d names axis %d of %d", j, axis_of_pair[j], axes);
  if (q_in_strides == nullptr || q_out_strides == nullptr || pos_strides == nullptr)
    return fail(ATS_EBADARG, "rope_axes: null strides");
  const bool has_k = k_in != nullptr;
  if (has_k && (k_out == nullptr || Hk < 0 || Hk > (1 << 20) || k_in_strides == nullptr || k_out_strides == nullptr))
    return fail(ATS_EBADARG, "rope_axes: incomplete k arguments");
  if (B == 0 || S == 0 || Hq + (has_k ? Hk : 0) == 0) return ATS_OK;
  if ((Hq > 0 && (q_in == nullptr || q_out == nullptr)) || positions == nullptr || inv_freq == nullptr)
    return fail(ATS_EBADARG, "rope_axes: null pointer");
  AxesArgs p{};
  p.q = AxesTensor{q_in, q_out, (int)Hq, q_in_strides[0], q_in_strides[1], q_in_strides[2],
                   q_out_strides[0], q_out_strides[1], q_out_strides[2]};
  if (has_k)
    p.k = AxesTensor{k_in, k_out, (int)Hk, k_in_strides[0], k_in_strides[1], k_in_strides[2],
                     k_out_strides[0], k_out_strides[1], k_out_strides[2]};
  p.pos = positions;
  p.pos_type = pos_type;
  p.ps_a = pos_strides[0], p.ps_b = pos_strides[1], p.ps_s = pos_strides[2];
  p.inv_freq = inv_freq;
  p.n_tokens = B * S;
  p.S = S;
  p.D = (int)D;
  p.pairs = pairs;
  p.sign = backward != 0 ? -1.0f : 1.0f;
  for (int j = 0; j < pairs; ++j) p.axis[j] = axis_of_pair[j];
  cudaStream_t st = (cudaStream_t)stream;
  if (x_dtype == ATS_BF16) {
    switch (vector_width(p, 2)) {
      case 8: return launch_v<bf16, 8>(p, st);
      case 4: return launch_v<bf16, 4>(p, st);
      case 2: return launch_v<bf16, 2>(p, st);
      default: return launch_v<bf16, 1>(p, st);
    }
  }
  switch (vector_width(p, 4)) {
    case 4: return launch_v<float, 4>(p, st);
    case 2: return launch_v<float, 2>(p, st);
    default: return launch_v<float, 1>(p, st);
  }
}
