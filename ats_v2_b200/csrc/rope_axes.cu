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
// sines once into shared memory, so that work is spread over the heads; each
// thread reads those of its vector there and streams heads past them.  Every element is read once and
// written once; HBM bounds it: q [4,32,4096,128] and k [4,8,4096,128] bf16 take
// 53 us a direction, 97% of the measured copy bandwidth (94 us with one thread
// per vector and head, which spent its time on indices).
#include "common.cuh"

namespace ats {
namespace {

constexpr int kThreads = 256;
// Heads in flight per thread: 3 where a head is 16 bytes in each half, so that 64 registers hold them (2: 55 us for the
// q and k above, 4: 56 us), else 4 (8 heads of 93 pairs in each of 21,244 tokens: 84 us; 2: 95 us, 3: 90 us).
template <typename T, int V> struct Unroll { static constexpr int value = V * (int)sizeof(T) == 16 ? 3 : 4; };
// Heads a thread handles: 16 of narrow vectors, to make up for the cost of a table (24 heads of 40 columns, 5514 tokens:
// 20 us, with 8: 26 us), 8 of 16 bytes (the q and k above: 53 us, with 16: 55 us).
template <typename T, int V> struct MostHeads { static constexpr int value = V * (int)sizeof(T) == 16 ? 8 : 16; };
constexpr double kInv2PiHi = 0.15915494309189535, kInv2PiLo = -9.839338337591243e-18;  // 1 / (2 pi) in two parts
constexpr int kTableMax = 2048;  // cosine/sine entries of a block (16 KB)
constexpr int kPosMax = 1024;    // positions of a block (8 KB)

struct AxesTensor {
  const void* in;
  void* out;
  int heads;
  int64_t is_b, is_h, is_s, os_b, os_h, os_s;  // strides in elements
  int64_t i_step, o_step;  // from a thread's head to its next one
};

struct AxesArgs {
  AxesTensor q, k;
  const void* pos;
  int pos_type;
  int64_t ps_a, ps_b, ps_s;
  const float* inv_freq;
  int64_t n_tokens, S;
  int D, pairs, axes;
  int rest_vec;  // elements per access of the copied columns
  int width;     // threads to a head
  int tokens_per_block, group, heads_each;  // `group` threads share a token's heads, heads_each to each
  unsigned by_width, by_group, by_pairs;  // for quotient()
  float sign;  // of the sine: +1 forward, -1 adjoint
  uint8_t axis[ATS_ROPE_MAX_PAIRS];
};

// Batch and sequence index of a token.
__device__ __forceinline__ void split(const AxesArgs& p, int64_t tok, int64_t& b, int64_t& s) {
  if (p.n_tokens <= 0x7fffffff) b = (unsigned)tok / (unsigned)p.S;  // S <= n_tokens
  else b = tok / p.S;
  s = tok - b * p.S;
}

// i / d for i <= 2048 and d <= 256, where m = 2^20 / d + 1: m d exceeds 2^20 by at most d, and i d < 2^20.
__device__ __forceinline__ int quotient(int i, unsigned m) { return (int)((unsigned)i * m >> 20); }

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

// A thread owns one vector position of the pairs of one token and heads_each heads, `group` apart; consecutive threads
// take consecutive vectors of a head's row.
template <typename T, int V, bool REST>  // REST: there are columns to copy
__global__ void __launch_bounds__(kThreads, 4) rope_axes_kernel(const __grid_constant__ AxesArgs p) {
  constexpr int kUnroll = Unroll<T, V>::value;
  using R = typename Raw<V * (int)sizeof(T)>::type;
  // frequencies [pairs], positions [axes][tokens], cosines [tokens][pairs], sines, axes [pairs]
  extern __shared__ __align__(16) double2 freq_s[];
  double* pos_s = reinterpret_cast<double*>(freq_s + p.pairs);
  const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
  const int ntok = (int)(p.n_tokens - tok0 < p.tokens_per_block ? p.n_tokens - tok0 : p.tokens_per_block);
  const int heads = p.q.heads + p.k.heads;
  float* cosv = reinterpret_cast<float*>(pos_s + (p.axes * p.tokens_per_block + 1) / 2 * 2);
  float* sinv = cosv + p.tokens_per_block * p.pairs;
  int* axis_s = reinterpret_cast<int*>(sinv + p.tokens_per_block * p.pairs);  // [pairs] first position of the pair's axis

  const int vecs = p.pairs / V, width = REST ? p.width : vecs;
  const int rest = quotient(threadIdx.x, p.by_width), vec = (int)threadIdx.x - rest * width;
  const int col = !REST || vec < vecs ? vec * V : 0;
  const int t = quotient(rest, p.by_group);
  const int h0 = (int)blockIdx.y * p.group * p.heads_each + (rest - t * p.group);
  const bool active = t < ntok;
  // where the heads of this thread's token begin: q's, then k's
  int64_t b, s;
  split(p, tok0 + (active ? t : 0), b, s);
  const T* qi = static_cast<const T*>(p.q.in) + b * p.q.is_b + s * p.q.is_s;
  const T* ki = static_cast<const T*>(p.k.in) + b * p.k.is_b + s * p.k.is_s - p.q.heads * p.k.is_h;
  T* qo = static_cast<T*>(p.q.out) + b * p.q.os_b + s * p.q.os_s;
  T* ko = static_cast<T*>(p.k.out) + b * p.k.os_b + s * p.k.os_s - p.q.heads * p.k.os_h;
  auto source = [&](int h) { return h < p.q.heads ? qi + h * p.q.is_h : ki + h * p.k.is_h; };
  auto target = [&](int h) { return h < p.q.heads ? qo + h * p.q.os_h : ko + h * p.k.os_h; };
  const int h_end = !active ? 0 : h0 + p.group * p.heads_each < heads ? h0 + p.group * p.heads_each : heads;
  // the heads one after the other by steps, from q over to k once: an address costs a few additions, where a product
  // for each head took most of the time of narrow vectors
  const int k0 = h0 < p.q.heads ? h0 + (p.q.heads - h0 + p.group - 1) / p.group * p.group : h0;  // first of k
  const T* src = source(h0) + col;
  T* dst = target(h0) + col;
  const T* src_k = ki + k0 * p.k.is_h + col;
  T* dst_k = ko + k0 * p.k.os_h + col;
  const int h_turn = !REST || vec < vecs ? h_end : 0;  // threads past the pairs' only copy
  R ra[kUnroll], rb[kUnroll];
  auto load = [&](int first) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = first + u * p.group;
      if (h < h_turn) {
        ra[u] = *reinterpret_cast<const R*>(src);
        rb[u] = *reinterpret_cast<const R*>(src + p.pairs);
      }
      src = h + p.group == k0 ? src_k : src + (h < p.q.heads ? p.q.i_step : p.k.i_step);
    }
  };
  load(h0);  // in flight while the table is computed

  // positions and frequencies first, so that the table waits for memory once and not for every entry
  for (int i = threadIdx.x; i < p.axes * ntok; i += kThreads) {
    const int a = i / ntok;
    int64_t tb, ts;
    split(p, tok0 + (i - a * ntok), tb, ts);
    pos_s[i] = load_pos(p, a * p.ps_a + tb * p.ps_b + ts * p.ps_s);
  }
  for (int j = threadIdx.x; j < p.pairs; j += kThreads) {
    // frequency / 2pi as a sum of two doubles, so that the fraction of a turn is right for every position below 2^53
    const double f = (double)p.inv_freq[j], c = f * kInv2PiHi;
    freq_s[j] = make_double2(c, fma(f, kInv2PiHi, -c) + f * kInv2PiLo);
    axis_s[j] = p.axis[j] * ntok;  // neighbouring pairs read different words of the parameters: slow, so once a pair
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ntok * p.pairs; i += kThreads) {
    const int ti = quotient(i, p.by_pairs), j = i - ti * p.pairs;
    const double pos = pos_s[axis_s[j] + ti];
    const double2 c = freq_s[j];
    const double high = pos * c.x;
    const float left = (float)((high - rint(high)) + (fma(pos, c.x, -high) + pos * c.y));
    float sine, cosine;
    sincospif(2.0f * left, &sine, &cosine);
    // vectors of 8 are kept as two planes of four, so that neighbouring threads' reads do not share banks
    const int at = V == 8 ? ti * p.pairs + (j >> 2 & 1) * (p.pairs / 2) + (j >> 3) * 4 + (j & 3) : i;
    cosv[at] = cosine;
    sinv[at] = sine * p.sign;
  }
  __syncthreads();

  // this vector's cosines and sines: read where they are used, four at a time, which leaves registers for a fourth
  // block on the SM
  constexpr int W = V < 4 ? V : 4;
  const float* cs = cosv + t * p.pairs + (V == 8 ? col / 2 : col);
  const float* sn = sinv + t * p.pairs + (V == 8 ? col / 2 : col);
  const int far = V == 8 ? p.pairs / 2 : 4;  // from the first four to the next
  for (int first = h0; first < h_turn; first += kUnroll * p.group) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = first + u * p.group;
      if (h < h_turn) {
        const T* xa = reinterpret_cast<const T*>(&ra[u]);
        const T* xb = reinterpret_cast<const T*>(&rb[u]);
        R oa, ob;
        float fa[V], fb[V];
#pragma unroll
        for (int w = 0; w < V; w += W) {
          float c[W], d[W];
          if constexpr (W == 4) {
            *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cs + w / 4 * far);
            *reinterpret_cast<float4*>(d) = *reinterpret_cast<const float4*>(sn + w / 4 * far);
          } else {
#pragma unroll
            for (int i = 0; i < W; ++i) c[i] = cs[w + i], d[i] = sn[w + i];
          }
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const float x = Cvt<T>::to_f(xa[w + i]), y = Cvt<T>::to_f(xb[w + i]);
            fa[w + i] = x * c[i] - y * d[i];
            fb[w + i] = y * c[i] + x * d[i];
          }
        }
        round_n<T, V>(fa, reinterpret_cast<T*>(&oa));
        round_n<T, V>(fb, reinterpret_cast<T*>(&ob));
        *reinterpret_cast<R*>(dst) = oa;
        *reinterpret_cast<R*>(dst + p.pairs) = ob;
      }
      dst = h + p.group == k0 ? dst_k : dst + (h < p.q.heads ? p.q.o_step : p.k.o_step);
    }
    if (first + kUnroll * p.group < h_turn) load(first + kUnroll * p.group);
  }

  // Columns that are not rotated, `rest_vec` elements at a time.  Where a head has a piece for each of its threads they
  // walk the heads as above (40 heads of 96 columns, 10 turned, of 7074 tokens: 33 us, dealt out 60), else
  // all of the token's pieces are dealt out to its threads (8 heads of 190 columns, 186 turned: 83 us, walked 97).
  if (REST && active) {
    const int extra = (p.D - 2 * p.pairs) / p.rest_vec;
    auto walk = [&](auto raw) {
      using C = decltype(raw);
      constexpr int U = 4;  // heads in flight
      src = source(h0) + 2 * p.pairs, src_k += 2 * p.pairs - col;
      dst = target(h0) + 2 * p.pairs, dst_k += 2 * p.pairs - col;
      for (int first = h0; first < h_end; first += U * p.group) {
        const C* from[U];
        C* to[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = first + u * p.group;
          from[u] = reinterpret_cast<const C*>(src);
          to[u] = reinterpret_cast<C*>(dst);
          src = h + p.group == k0 ? src_k : src + (h < p.q.heads ? p.q.i_step : p.k.i_step);
          dst = h + p.group == k0 ? dst_k : dst + (h < p.q.heads ? p.q.o_step : p.k.o_step);
        }
        for (int c = vec; c < extra; c += width) {
          C v[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (first + u * p.group < h_end) v[u] = from[u][c];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (first + u * p.group < h_end) to[u][c] = v[u];
        }
      }
    };
    auto deal = [&](auto raw) {
      using C = decltype(raw);
      const int hb = (int)blockIdx.y * p.group * p.heads_each;
      const int nh = heads - hb < p.group * p.heads_each ? heads - hb : p.group * p.heads_each;
      const int team = p.group * width;  // pieces: at most 256 of a head, of 4096 heads
      for (int i = (int)threadIdx.x - t * team; i < nh * extra; i += team) {
        const int r = (int)((unsigned)i / (unsigned)extra), c = i - r * extra;
        reinterpret_cast<C*>(target(hb + r) + 2 * p.pairs)[c] =
            reinterpret_cast<const C*>(source(hb + r) + 2 * p.pairs)[c];
      }
    };
    auto copy = [&](auto raw) {
      if (extra >= width) walk(raw);
      else deal(raw);
    };
    const int bytes = p.rest_vec * (int)sizeof(T);
    if (bytes == 16) copy(uint4{});
    else if (bytes == 8) copy(uint2{});
    else if (bytes == 4) copy(uint32_t{});
    else copy(uint16_t{});
  }
}

// Elements one access may move: the largest power of two (at most 16 bytes) that divides `cols` and every stride, and
// to which every pointer is aligned.
int vector_width(const AxesArgs& p, int64_t cols, int elem) {
  int64_t bits = cols;
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
  const int heads = p.q.heads + p.k.heads, vecs = p.pairs / V;
  // Threads to a head: one for each vector of pairs, but 8 where that is fewer and four times as many pieces are only
  // copied, so that neighbours copy neighbours (10 heads of 128 columns, 12 turned, of 51456 tokens: 92 us, with three
  // threads to a head 210; 40 heads of 96 columns, 10 turned, of 7074 tokens: 33 us, with five 39, with 32 61).
  const int extra = (p.D - 2 * p.pairs) / p.rest_vec;
  p.width = extra >= 4 * vecs ? (extra < 8 ? extra : 8) : vecs;
  if (p.width < vecs) p.width = vecs;
  const int most = kThreads / p.width;  // heads at a time
  // Heads to a thread: as many as leave three blocks to each SM, at most kMostHeads (the cosines and sines are then
  // computed once for many; a call of few tokens has one head to a thread and waits on latency alone).  From that
  // down to half of it, the number that leaves the fewest threads of a block idle.
  const double work = (double)p.n_tokens * p.width * heads / ((double)kThreads * 3 * num_sms());
  constexpr int kMostHeads = MostHeads<T, V>::value;
  int n = work < 1 ? 1 : work > kMostHeads ? kMostHeads : (int)work;
  if (n > heads) n = heads;
  int group = most < heads ? most : heads, each = n;  // where a block has no room for all the heads of a token
  double best = 0;
  for (int m = n; m >= 1 && 2 * m >= n; --m) {
    const int g = (heads + m - 1) / m;
    if (g > most) break;
    const double full = (double)(kThreads / (p.width * g)) * p.width * heads / ((double)kThreads * m);
    if (full > best) best = full, group = g, each = m;
  }
  int tpb = kThreads / (p.width * group);
  if (tpb > kTableMax / p.pairs) tpb = kTableMax / p.pairs;
  if (tpb > kPosMax / p.axes) tpb = kPosMax / p.axes;
  if (tpb > p.n_tokens) tpb = (int)p.n_tokens;
  const int64_t parts = (heads + (int64_t)group * each - 1) / ((int64_t)group * each);
  const int64_t blocks = (p.n_tokens + tpb - 1) / tpb;
  if (blocks > 0x7fffffff || parts > 65535) return fail(ATS_EUNSUPPORTED, "rope_axes: too many tokens or heads");
  p.tokens_per_block = tpb, p.group = group, p.heads_each = each;
  for (AxesTensor* t : {&p.q, &p.k}) t->i_step = group * t->is_h, t->o_step = group * t->os_h;
  auto inverse = [](int d) { return (1u << 20) / (unsigned)d + 1; };
  p.by_width = inverse(p.width), p.by_group = inverse(group), p.by_pairs = inverse(p.pairs);
  const size_t smem = (size_t)p.pairs * sizeof(double2) + (size_t)(tpb * p.axes + 1) / 2 * 16 +
                      (size_t)(2 * tpb + 1) * p.pairs * sizeof(float);
  const dim3 grid((unsigned)blocks, (unsigned)parts);
  if (p.D > 2 * p.pairs) rope_axes_kernel<T, V, true><<<grid, kThreads, smem, st>>>(p);
  else rope_axes_kernel<T, V, false><<<grid, kThreads, smem, st>>>(p);
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
  p.axes = axes;
  p.sign = backward != 0 ? -1.0f : 1.0f;
  for (int j = 0; j < pairs; ++j) p.axis[j] = axis_of_pair[j];
  cudaStream_t st = (cudaStream_t)stream;
  p.rest_vec = vector_width(p, 2 * (int64_t)pairs | (D - 2 * (int64_t)pairs), x_dtype == ATS_BF16 ? 2 : 4);
  if (x_dtype == ATS_BF16) {
    switch (vector_width(p, pairs, 2)) {
      case 8: return launch_v<bf16, 8>(p, st);
      case 4: return launch_v<bf16, 4>(p, st);
      case 2: return launch_v<bf16, 2>(p, st);
      default: return launch_v<bf16, 1>(p, st);
    }
  }
  switch (vector_width(p, pairs, 4)) {
    case 4: return launch_v<float, 4>(p, st);
    case 2: return launch_v<float, 2>(p, st);
    default: return launch_v<float, 1>(p, st);
  }
}
