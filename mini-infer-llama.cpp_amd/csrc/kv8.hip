// kv8.hip -- rows on their way into and out of a KV cache: the 8-bit form
// (quantised as it is written, read back), the rows of a tree that a step
// keeps, and the norms of queries and keys per head with the rotation and the
// append in one pass.
//
// The 8-bit form. A group of values shares the scale d, the smallest f16
// number with 127 d >= max |x|; a value is the whole number q nearest to x / d
// (ties to even), so |q| <= 127 and |x - q d| <= d / 2. A K row has a group
// per 32 dims: channels of K differ by large factors (a projection's bias),
// and one of them costs only its own group precision. A V row is one group,
// whose scale the attention folds into the row's probability. Values (int8)
// and scales (f16) lie in planes of their own, [head_dim, n_head_kv, n_ctx]
// and [groups, n_head_kv, n_ctx], so both keep their natural alignment. A
// group that holds an infinity or a NaN, or whose d passes the f16 range
// (max |x| > 8319008), reads back as NaN.
//
// Every kernel here reads each input once and writes each output once; the
// arithmetic is far below what the memory takes.
#include <cmath>

#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

constexpr int kGroup = 32;  // dims per K scale

__device__ inline float f16_bits(unsigned b) { return (float)__builtin_bit_cast(_Float16, (unsigned short)b); }

// |x| as bits, ordered like the value with NaN above infinity, so that a
// maximum over a group keeps them.
__device__ inline unsigned abs_bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

// The f16 bits of the smallest d with 127 d >= amax. The rounded quotient is
// at most one step off either way; 127 times an f16 number is exact in float.
__device__ inline unsigned scale_bits(float amax) {
  unsigned b = __builtin_bit_cast(unsigned short, (_Float16)(amax * (1.f / 127.f)));
  if (127.f * f16_bits(b) < amax) ++b;
  else if (b > 0 && 127.f * f16_bits(b - 1) >= amax) --b;
  return b;
}

// The whole number nearest to x / d, ties to even; inv = 1 / d rounded (0 for
// d = 0 and where d is not a number). The product can round across a border
// between two whole numbers, so the remainder x - k d decides, which one
// fused multiply-add gives exactly.
__device__ inline int quantize(float x, float d, float inv) {
  float k = rintf(x * inv);
  const float r = fmaf(-k, d, x), two = 2.f * fabsf(r);
  const bool odd = ((int)k & 1) != 0;
  if (two > d || (two == d && odd)) k += copysignf(1.f, r);
  return k == k ? (int)k : 0;
}

__device__ inline float inverse(float d) { return d > 0.f && d < INFINITY ? 1.f / d : 0.f; }

// Maximum over the aligned group of N lanes (a power of two) this lane is in.
template <int N>
__device__ inline unsigned group_max(unsigned x) {
#pragma unroll
  for (int off = N / 2; off >= 1; off >>= 1) x = max(x, (unsigned)__shfl_xor((int)x, off, kWave));
  return x;
}
template <int N>
__device__ inline float group_sum(float x) {
#pragma unroll
  for (int off = N / 2; off >= 1; off >>= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

__device__ inline float ldf(const char* p, int64_t off) { return gload<float>(p + off); }

// Row (which, pos, head) of a cache and its scales.
__device__ inline char* row_of(const CacheView& c, int which, int64_t pos, int h) {
  return c.t[which] + pos * c.s2 + (int64_t)h * c.s1;
}
__device__ inline char* scale_of(const CacheView& c, int which, int64_t pos, int h) {
  const int n = which == 0 ? c.head_dim / kGroup : 1;
  return c.scale[which] + (pos * c.n_head_kv + h) * 2 * n;
}

// One row with a wave: lane holds dims lane + 64 i. Stores it as the cache's
// type has it.
template <int E>
__device__ inline void store_row(const CacheView& c, int which, int64_t pos, int h, int lane, const float (&x)[E]) {
  char* const row = row_of(c, which, pos, h);
  if (c.elt == 1) {
    unsigned a[E];
#pragma unroll
    for (int i = 0; i < E; ++i) a[i] = group_max<32>(abs_bits(x[i]));
    if (which == 1) {
      unsigned all = 0;
#pragma unroll
      for (int i = 0; i < E; ++i) all = max(all, a[i]);
      all = max(all, (unsigned)__shfl_xor((int)all, 32, kWave));
#pragma unroll
      for (int i = 0; i < E; ++i) a[i] = all;
    }
    char* const sc = scale_of(c, which, pos, h);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const unsigned b = scale_bits(__builtin_bit_cast(float, a[i]));
      const float d = f16_bits(b);
      if (lane + 64 * i < c.head_dim) {
        gstore<int8_t>(row + lane + 64 * i, (int8_t)quantize(x[i], d, inverse(d)));
        if (which == 0 ? lane % kGroup == 0 : lane + 64 * i == 0)
          gstore<unsigned short>(sc + 2 * ((lane + 64 * i) / kGroup), (unsigned short)b);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (c.elt == 2) gstore<_Float16>(row + 2 * (lane + 64 * i), (_Float16)x[i]);
    else gstore<float>(row + 4 * (lane + 64 * i), x[i]);
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Quantising rows as they are written, reading them back, keeping some
// ---------------------------------------------------------------------------
struct QuantizeArgs {
  CacheView c;
  const char* src;
  int64_t nb[3];
  int64_t rows;  // n_tokens * n_head_kv
  int32_t which, pos0;
};

template <int E>
__global__ __launch_bounds__(256) void kv_quantize_kernel(const QuantizeArgs p) {
  const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kWave;
  if (r >= p.rows) return;
  const int lane = threadIdx.x % kWave;
  const int h = (int)(r % p.c.n_head_kv);
  const int64_t t = r / p.c.n_head_kv;
  float x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = ldf(p.src, t * p.nb[2] + h * p.nb[1] + (lane + 64 * i) * p.nb[0]);
  store_row<E>(p.c, p.which, p.pos0 + t, h, lane, x);
}

hipError_t launch_kv_quantize(const CacheView& c, int which, const char* src, const int64_t src_nb[3], int pos0,
                              int n_tokens, hipStream_t stream) {
  QuantizeArgs p{c, src, {src_nb[0], src_nb[1], src_nb[2]}, (int64_t)n_tokens * c.n_head_kv, which, pos0};
  if (p.rows == 0) return hipSuccess;
  const dim3 grid((unsigned)((p.rows + 3) / 4));
  if (c.head_dim == 64) hipLaunchKernelGGL(kv_quantize_kernel<1>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(kv_quantize_kernel<2>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

struct ReadArgs {
  CacheView c;
  char* dst;
  int64_t nb[3];
  int64_t rows;
  int32_t which, pos0;
};

template <typename DT>
__global__ __launch_bounds__(256) void kv_read_kernel(const ReadArgs p) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = idx / p.c.head_dim;
  const int d = (int)(idx % p.c.head_dim);
  if (r >= p.rows) return;
  const int h = (int)(r % p.c.n_head_kv);
  const int64_t t = r / p.c.n_head_kv;
  const char* const row = row_of(p.c, p.which, p.pos0 + t, h);
  float x;
  if (p.c.elt == 1) {
    const char* const sc = scale_of(p.c, p.which, p.pos0 + t, h);
    x = (float)gload<int8_t>(row + d) * (float)gload<_Float16>(sc + (p.which == 0 ? 2 * (d / kGroup) : 0));
  } else {
    x = p.c.elt == 2 ? (float)gload<_Float16>(row + 2 * d) : gload<float>(row + 4 * d);
  }
  gstore<DT>(p.dst + t * p.nb[2] + h * p.nb[1] + d * p.nb[0], (DT)x);
}

hipError_t launch_kv_read(const CacheView& c, int which, int pos0, int n_tokens, char* dst, bool dst_f16,
                          const int64_t dst_nb[3], hipStream_t stream) {
  ReadArgs p{c, dst, {dst_nb[0], dst_nb[1], dst_nb[2]}, (int64_t)n_tokens * c.n_head_kv, which, pos0};
  if (p.rows == 0) return hipSuccess;
  const dim3 grid((unsigned)((p.rows * c.head_dim + 255) / 256));
  if (dst_f16) hipLaunchKernelGGL(kv_read_kernel<_Float16>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(kv_read_kernel<float>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Two bytes of one position's plane per thread, the kept rows in order: row
// n_past + i is written after it has been read (as some idx[j] <= i, j <= i),
// by the same thread, so the move may overlap itself.
__global__ __launch_bounds__(256) void kv_keep_kernel(const KvKeep p) {
  const int plane = blockIdx.y % p.n_planes, layer = blockIdx.y / p.n_planes;
  const int at = 2 * (blockIdx.x * 256 + threadIdx.x);
  const int64_t row = p.bytes[plane];
  if (at >= row) return;
  char* const base = p.plane[plane] + layer * p.layer[plane] + (int64_t)p.n_past * row + at;
  for (int i = 0; i < p.n; ++i)
    if (p.idx[i] != i) gstore<unsigned short>(base + i * row, gload<unsigned short>(base + p.idx[i] * row));
}

hipError_t launch_kv_keep(const KvKeep& p, hipStream_t stream) {
  int most = 0;
  for (int i = 0; i < p.n_planes; ++i) most = p.bytes[i] > most ? p.bytes[i] : most;
  hipLaunchKernelGGL(kv_keep_kernel, dim3((unsigned)((most / 2 + 255) / 256), (unsigned)(p.n_planes * p.n_layer)),
                     dim3(256), 0, stream, p);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Norms of Q and K per head, rotation, append
// ---------------------------------------------------------------------------
// Per row x of Q or K: y = x / sqrt(mean(x^2) + eps) * w (sums in float), then
// the rotation of rope.hip (angle = position * freq, one float product; cosine
// and sine in double, rounded): pair (i, i + n_dims / 2) of the first n_dims.
//
// A wave per row, any strides and n_dims: the row passes through LDS so that a
// lane finds its dims' partners.
template <int E>
__global__ __launch_bounds__(256) void norm_rope_row_kernel(const NormRope p) {
  __shared__ float rows[4][64 * E];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int hkv = p.cache.n_head_kv, per_tok = p.n_head + 2 * hkv;
  const int64_t r = (int64_t)blockIdx.x * 4 + wave;
  if (r >= (int64_t)p.n_tokens * per_tok) return;
  const int t = (int)(r / per_tok);
  int h = (int)(r - (int64_t)t * per_tok);
  const int kind = h < p.n_head ? 0 : h < p.n_head + hkv ? 1 : 2;  // Q, K, V
  h -= kind == 0 ? 0 : kind == 1 ? p.n_head : p.n_head + hkv;
  const char* const src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
  const int64_t* const nb = kind == 0 ? p.q_nb : kind == 1 ? p.k_nb : p.v_nb;
  const int64_t so = t * nb[2] + h * nb[1];
  float x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = ldf(src, so + (lane + 64 * i) * nb[0]);
  if (kind < 2) {
    const float* const w = kind == 0 ? p.q_norm : p.k_norm;
    if (w) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) ss += x[i] * x[i];
      ss = group_sum<64>(ss);
      const float inv = 1.f / sqrtf(ss / (64 * E) + p.eps);
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = x[i] * inv * gload<float>(w + lane + 64 * i);
    }
    float* const row = rows[wave];
#pragma unroll
    for (int i = 0; i < E; ++i) row[lane + 64 * i] = x[i];
    wave_lds_fence();
    const int half = p.n_dims / 2;
    const int pos = p.pos ? gload<int>(p.pos + t) : p.n_past + t;
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma clang fp contract(off)
      const int d = lane + 64 * i;
      if (d >= p.n_dims) continue;
      const int j = d < half ? d : d - half;
      double s, c;
      sincos((double)((float)pos * p.freq[j]), &s, &c);
      const float a = row[j], b = row[j + half];
      x[i] = d < half ? a * (float)c - b * (float)s : a * (float)s + b * (float)c;
    }
  }
  if (kind == 0) {
    char* const o = p.q_out + t * p.qo_nb[2] + h * p.qo_nb[1];
#pragma unroll
    for (int i = 0; i < E; ++i) gstore<float>(o + (lane + 64 * i) * p.qo_nb[0], x[i]);
  } else {
    store_row<E>(p.cache, kind - 1, (int64_t)p.n_past + t, h, lane, x);
  }
}

hipError_t launch_norm_rope(const NormRope& p, hipStream_t stream) {
  const int64_t rows = (int64_t)p.n_tokens * (p.n_head + 2 * p.cache.n_head_kv);
  if (rows == 0) return hipSuccess;
  const dim3 grid((unsigned)((rows + 3) / 4));
  if (p.cache.head_dim == 64) hipLaunchKernelGGL(norm_rope_row_kernel<1>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(norm_rope_row_kernel<2>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mi
