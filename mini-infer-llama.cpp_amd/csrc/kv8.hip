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
// arithmetic is far below what the memory takes. 16384 positions of 4 heads of
// 128, us a kernel: K quantised 10.4 (42 MB, 4.1 TB/s), V 9.3, read back as F16
// 6.0 (26 MB, 4.2 TB/s); norms, RoPE and append of 4096 tokens, 28/4 heads of 128,
// F16 cache 23.4, 8-bit 23.8 (143 MB, of which the launch before has left a part in
// the memory-side cache; among other passes 32.1, 4.4 TB/s); a few rows 2 to 4, a
// launch's own time.
#include <cmath>
#include <type_traits>

#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

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
__device__ inline double group_sum(double x) {
#pragma unroll
  for (int off = N / 2; off >= 1; off >>= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

// Over aligned groups of N = 4, 8 or 16 lanes (DPP moves within rows of 16).
template <int N, typename T, typename F>
__device__ inline T fold_lanes(T x, F f) {
  auto move = [](T v, auto ctrl) {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x = f(x, move(x, std::integral_constant<int, 0xB1>{}));  // quad_perm [1,0,3,2]
  x = f(x, move(x, std::integral_constant<int, 0x4E>{}));  // quad_perm [2,3,0,1]
  if constexpr (N >= 8) x = f(x, move(x, std::integral_constant<int, 0x141>{}));   // row_half_mirror
  if constexpr (N >= 16) x = f(x, move(x, std::integral_constant<int, 0x140>{}));  // row_mirror
  return x;
}
template <int N>
__device__ inline unsigned max_of_lanes(unsigned x) {
  return fold_lanes<N>(x, [](unsigned a, unsigned b) { return max(a, b); });
}
template <int N>
__device__ inline float sum_of_lanes(float x) {
  return fold_lanes<N>(x, [](float a, float b) { return a + b; });
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

// Rows of contiguous, 16-byte aligned values: a lane takes eight dims (a K
// group is four lanes, a row D / 8), reads 32 bytes and writes 8. 4096 positions
// of 4 heads of 128: 4.6 us a call, 7.1 with a wave per row.
template <int D, int WHICH>
__global__ __launch_bounds__(256) void kv_quantize_rows_kernel(const QuantizeArgs p) {
  constexpr int LANES = D / 8;
  const unsigned r = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int d = 8 * (threadIdx.x % LANES);
  if (r >= (unsigned)p.rows) return;
  const unsigned t = r / (unsigned)p.c.n_head_kv, h = r - t * (unsigned)p.c.n_head_kv;
  const char* const src = p.src + t * p.nb[2] + h * p.nb[1] + 4 * d;
  const f32x4 a = gload<f32x4>(src), b = gload<f32x4>(src + 16);
  float x[8];
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = i < 4 ? a[i] : b[i - 4];
    most = max(most, abs_bits(x[i]));
  }
  most = max_of_lanes<WHICH == 0 ? 4 : LANES>(most);
  const unsigned sb = scale_bits(__builtin_bit_cast(float, most));
  const float sc = f16_bits(sb), inv = inverse(sc);
  u32x2 q = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i / 4] |= ((unsigned)quantize(x[i], sc, inv) & 0xffu) << (8 * (i % 4));
  const int64_t pos = (int64_t)p.pos0 + t;
  gstore(row_of(p.c, WHICH, pos, h) + d, q);
  if (d % (WHICH == 0 ? kGroup : D) == 0)
    gstore<unsigned short>(scale_of(p.c, WHICH, pos, h) + 2 * (d / kGroup), (unsigned short)sb);
}

// Whether rows (byte strides nb) can be read or written 16 bytes at a time,
// `elt` bytes an element.
static bool rows_aligned(const char* p, const int64_t nb[3], int elt) {
  return nb[0] == elt && nb[1] % 16 == 0 && nb[2] % 16 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}

hipError_t launch_kv_quantize(const CacheView& c, int which, const char* src, const int64_t src_nb[3], int pos0,
                              int n_tokens, hipStream_t stream) {
  QuantizeArgs p{c, src, {src_nb[0], src_nb[1], src_nb[2]}, (int64_t)n_tokens * c.n_head_kv, which, pos0};
  if (p.rows == 0) return hipSuccess;
  if (rows_aligned(src, src_nb, 4) && p.rows < INT32_MAX) {
    const dim3 grid((unsigned)((p.rows * (c.head_dim / 8) + 255) / 256));
    if (c.head_dim == 64) {
      if (which == 0) hipLaunchKernelGGL((kv_quantize_rows_kernel<64, 0>), grid, dim3(256), 0, stream, p);
      else hipLaunchKernelGGL((kv_quantize_rows_kernel<64, 1>), grid, dim3(256), 0, stream, p);
    } else {
      if (which == 0) hipLaunchKernelGGL((kv_quantize_rows_kernel<128, 0>), grid, dim3(256), 0, stream, p);
      else hipLaunchKernelGGL((kv_quantize_rows_kernel<128, 1>), grid, dim3(256), 0, stream, p);
    }
    return hipGetLastError();
  }
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

// Into contiguous, 16-byte aligned rows: a lane takes eight dims. 4096 positions
// of 4 heads of 128, 8-bit: 4.5 us a call, 8.1 with a lane per value.
template <int D, int ELT, typename DT>
__global__ __launch_bounds__(256) void kv_read_rows_kernel(const ReadArgs p) {
  constexpr int LANES = D / 8;
  const unsigned r = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int d = 8 * (threadIdx.x % LANES);
  if (r >= (unsigned)p.rows) return;
  const unsigned t = r / (unsigned)p.c.n_head_kv, h = r - t * (unsigned)p.c.n_head_kv;
  const int64_t pos = (int64_t)p.pos0 + t;
  const char* const row = row_of(p.c, p.which, pos, h) + d * ELT;
  float x[8];
  if constexpr (ELT == 1) {
    const float sc = (float)gload<_Float16>(scale_of(p.c, p.which, pos, h) + (p.which == 0 ? 2 * (d / kGroup) : 0));
    const u32x2 q = gload<u32x2>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(q[i / 4] >> (8 * (i % 4)) & 0xffu) * sc;
  } else if constexpr (ELT == 2) {
    const f16x8 q = gload<f16x8>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)q[i];
  } else {
    const f32x4 a = gload<f32x4>(row), b = gload<f32x4>(row + 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < 4 ? a[i] : b[i - 4];
  }
  char* const dst = p.dst + t * p.nb[2] + h * p.nb[1] + d * (int)sizeof(DT);
  if constexpr (sizeof(DT) == 2) {
    f16x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (_Float16)x[i];
    gstore(dst, y);
  } else {
    gstore(dst, f32x4{x[0], x[1], x[2], x[3]});
    gstore(dst + 16, f32x4{x[4], x[5], x[6], x[7]});
  }
}

template <int D, typename DT>
static void launch_kv_read_rows(const ReadArgs& p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.rows * (D / 8) + 255) / 256));
  if (p.c.elt == 1) hipLaunchKernelGGL((kv_read_rows_kernel<D, 1, DT>), grid, dim3(256), 0, stream, p);
  else if (p.c.elt == 2) hipLaunchKernelGGL((kv_read_rows_kernel<D, 2, DT>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((kv_read_rows_kernel<D, 4, DT>), grid, dim3(256), 0, stream, p);
}

hipError_t launch_kv_read(const CacheView& c, int which, int pos0, int n_tokens, char* dst, bool dst_f16,
                          const int64_t dst_nb[3], hipStream_t stream) {
  ReadArgs p{c, dst, {dst_nb[0], dst_nb[1], dst_nb[2]}, (int64_t)n_tokens * c.n_head_kv, which, pos0};
  if (p.rows == 0) return hipSuccess;
  if (rows_aligned(dst, dst_nb, dst_f16 ? 2 : 4) && p.rows < INT32_MAX) {
    if (c.head_dim == 64) {
      if (dst_f16) launch_kv_read_rows<64, _Float16>(p, stream);
      else launch_kv_read_rows<64, float>(p, stream);
    } else {
      if (dst_f16) launch_kv_read_rows<128, _Float16>(p, stream);
      else launch_kv_read_rows<128, float>(p, stream);
    }
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((p.rows * c.head_dim + 255) / 256));
  if (dst_f16) hipLaunchKernelGGL(kv_read_kernel<_Float16>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(kv_read_kernel<float>, grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Bound: one read's latency per eight rows (6 of 25 rows, 14/2 heads of 64: 3.4 us).
// Two bytes of one position's plane per thread, the kept rows in order: row
// n_past + i is written after it has been read (as some idx[j] <= i, j <= i),
// by the same thread, so the move may overlap itself. kInFlight rows are read
// before they are written: the rows of a batch lie at or behind where it writes
// (idx[j] >= j), and so do those of the batches after it.
__global__ __launch_bounds__(256) void kv_keep_kernel(const KvKeep p) {
  constexpr int kInFlight = 8;
  const int plane = blockIdx.y % p.n_planes, layer = blockIdx.y / p.n_planes;
  const int at = 2 * (blockIdx.x * 256 + threadIdx.x);
  const int64_t row = p.bytes[plane];
  if (at >= row) return;
  char* const base = p.plane[plane] + layer * p.layer[plane] + (int64_t)p.n_past * row + at;
  for (int i = 0; i < p.n; i += kInFlight) {
    unsigned short x[kInFlight];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j)
      if (i + j < p.n) x[j] = gload<unsigned short>(base + p.idx[i + j] * row);
#pragma unroll
    for (int j = 0; j < kInFlight; ++j)
      if (i + j < p.n) gstore<unsigned short>(base + (i + j) * row, x[j]);
  }
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
// Per row x of Q or K: y = x / sqrt(mean(x^2) + eps) * w (the sum in float, in
// double for a row whose squares leave float's range), then
// the rotation of rope.hip (angle = position * freq, one float product; cosine
// and sine in double, rounded): pair (i, i + n_dims / 2) of the first n_dims.
//
// A wave per row, any strides and n_dims, each lane with angles of its own in double
// precision (4096 tokens of 28/4 heads of 128 with 96 dims rotated: 72.4 us, 8-bit
// cache 80.9, where the form below, whose angles are once per token, takes 23 to 25
// for all dims): the row passes through LDS so that a
// lane finds its dims' partners. K on its way to an 8-bit cache stays in double
// precision until it is quantised, as in the form for aligned rows below.
template <int E, bool Q8>
__global__ __launch_bounds__(256) void norm_rope_row_kernel(const NormRope p) {
  __shared__ float rows[4][64 * E];
  __shared__ double rows_d[Q8 ? 4 : 1][64 * E];
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
    const bool exact = Q8 && kind == 1;
    const float* const w = kind == 0 ? p.q_norm : p.k_norm;
    double y[E];  // the row where it is not rounded on the way
    if (exact) {
#pragma unroll
      for (int i = 0; i < E; ++i) y[i] = x[i];
    }
    if (w) {
      double ss = 0.0;  // (in double in any case: this is not the fast form)
#pragma unroll
      for (int i = 0; i < E; ++i) ss += (double)x[i] * x[i];
      const double inv = 1.0 / sqrt(group_sum<64>(ss) / (64 * E) + (double)p.eps);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float wi = gload<float>(w + lane + 64 * i);
        if (exact) y[i] = y[i] * inv * wi;
        else x[i] = (float)(x[i] * inv) * wi;
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (exact) rows_d[Q8 ? wave : 0][lane + 64 * i] = y[i];
      else rows[wave][lane + 64 * i] = x[i];
    }
    wave_lds_fence();
    const int half = p.n_dims / 2;
    const int pos = p.pos ? gload<int>(p.pos + t) : p.n_past + t;
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma clang fp contract(off)
      const int d = lane + 64 * i;
      if (exact) x[i] = (float)y[i];
      if (d >= p.n_dims) continue;
      const int j = d < half ? d : d - half;
      double s, c;
      sincos((double)((float)pos * p.freq[j]), &s, &c);
      if (exact) {
        const double a = rows_d[Q8 ? wave : 0][j], b = rows_d[Q8 ? wave : 0][j + half];
        x[i] = (float)(d < half ? a * c - b * s : a * s + b * c);
      } else {
        const float a = rows[wave][j], b = rows[wave][j + half];
        x[i] = d < half ? a * (float)c - b * (float)s : a * (float)s + b * (float)c;
      }
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

// All dims rotated, rows contiguous and 16-byte aligned: D / 8 lanes a row, each
// with dims 4 j .. 4 j + 3 and their partners D / 2 further on. A workgroup
// takes `tokens` tokens (gridDim.y pieces of their rows): the angles' cosines
// and sines once per token in LDS (double precision, about as much work as the
// rest of a token's rows together), then the rows from registers to the cache.
// K on its way to an 8-bit cache stays in double precision until it is
// quantised, since a value next to a border between two steps should not cross
// it by a rounding.
constexpr int kRopeTokens = 4;

template <int D>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRope p, int tokens) {
  constexpr int LANES = D / 8, HALF = D / 2;
  __shared__ float2 cs[kRopeTokens][HALF];
  __shared__ double cs_d[kRopeTokens][HALF][2];  // 8-bit caches
  const int hkv = p.cache.n_head_kv, per_tok = p.n_head + 2 * hkv;
  const int t0 = blockIdx.x * tokens, nt = min(tokens, p.n_tokens - t0);
  const bool q8 = p.cache.elt == 1;
  for (int i = threadIdx.x; i < nt * HALF; i += 256) {
    const int t = i / HALF, j = i % HALF;
    const int pos = p.pos ? gload<int>(p.pos + t0 + t) : p.n_past + t0 + t;
    double sn, c;
    sincos((double)((float)pos * p.freq[j]), &sn, &c);
    cs[t][j] = float2{(float)c, (float)sn};
    if (q8) {
      cs_d[t][j][0] = c;
      cs_d[t][j][1] = sn;
    }
  }
  __syncthreads();
  const int j4 = 4 * (threadIdx.x % LANES);
  const int step = 256 / LANES * gridDim.y;
  for (int row = blockIdx.y * (256 / LANES) + threadIdx.x / LANES; row < nt * per_tok; row += step) {
    const int t = row / per_tok;
    int h = row - t * per_tok;
    const int kind = h < p.n_head ? 0 : h < p.n_head + hkv ? 1 : 2;  // Q, K, V
    h -= kind == 0 ? 0 : kind == 1 ? p.n_head : p.n_head + hkv;
    const char* const src = (kind == 0 ? p.q : kind == 1 ? p.k : p.v) +
                            (t0 + t) * (kind == 0 ? p.q_nb[2] : kind == 1 ? p.k_nb[2] : p.v_nb[2]) +
                            h * (kind == 0 ? p.q_nb[1] : kind == 1 ? p.k_nb[1] : p.v_nb[1]) + 4 * j4;
    f32x4 a = gload<f32x4>(src), b = gload<f32x4>(src + 4 * HALF);
    if (kind < 2) {
      const float* const w = kind == 0 ? p.q_norm : p.k_norm;
      f32x4 wa = {1.f, 1.f, 1.f, 1.f}, wb = wa;
      if (w) {
        wa = gload<f32x4>(w + j4);
        wb = gload<f32x4>(w + HALF + j4);
      }
      const bool exact = q8 && kind == 1;
      bool wide = exact;
      float inv_f = 1.f;
      double inv = 1.0;
      if (w && !exact) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
        const float mean = sum_of_lanes<LANES>(ss) / D + p.eps;
        wide = !(mean > 1e-30f && mean < INFINITY);
        inv_f = 1.f / sqrtf(mean);
      }
      if (w && wide) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += (double)a[i] * a[i] + (double)b[i] * b[i];
        inv = 1.0 / sqrt(group_sum<LANES>(ss) / D + (double)p.eps);
      }
      if (exact) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double x = a[i] * inv * wa[i], y = b[i] * inv * wb[i];
          const double c = cs_d[t][j4 + i][0], sn = cs_d[t][j4 + i][1];
          a[i] = (float)(x * c - y * sn);
          b[i] = (float)(x * sn + y * c);
        }
      } else {
#pragma clang fp contract(off)
        if (w) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i] = (wide ? (float)(a[i] * inv) : a[i] * inv_f) * wa[i];
            b[i] = (wide ? (float)(b[i] * inv) : b[i] * inv_f) * wb[i];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 r = cs[t][j4 + i];
          const float x = a[i], y = b[i];
          a[i] = x * r.x - y * r.y;
          b[i] = x * r.y + y * r.x;
        }
      }
    }
    if (kind == 0) {
      char* const o = p.q_out + (t0 + t) * p.qo_nb[2] + h * p.qo_nb[1] + 4 * j4;
      gstore(o, a);
      gstore(o + 4 * HALF, b);
      continue;
    }
    const int64_t pos = (int64_t)p.n_past + t0 + t;
    char* const o = row_of(p.cache, kind - 1, pos, h);
    if (q8) {
      unsigned ma = 0, mb = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ma = max(ma, abs_bits(a[i]));
        mb = max(mb, abs_bits(b[i]));
      }
      if (kind == 1) {
        ma = max_of_lanes<8>(ma);
        mb = max_of_lanes<8>(mb);
      } else {
        ma = mb = max_of_lanes<LANES>(max(ma, mb));
      }
      const unsigned ba = scale_bits(__builtin_bit_cast(float, ma)), bb = scale_bits(__builtin_bit_cast(float, mb));
      const float da = f16_bits(ba), db = f16_bits(bb), ia = inverse(da), ib = inverse(db);
      unsigned qa = 0, qb = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        qa |= ((unsigned)quantize(a[i], da, ia) & 0xffu) << (8 * i);
        qb |= ((unsigned)quantize(b[i], db, ib) & 0xffu) << (8 * i);
      }
      gstore(o + j4, qa);
      gstore(o + HALF + j4, qb);
      char* const sc = scale_of(p.cache, kind - 1, pos, h);
      if (kind == 1 && j4 % kGroup == 0) {
        gstore<unsigned short>(sc + 2 * (j4 / kGroup), (unsigned short)ba);
        gstore<unsigned short>(sc + 2 * ((HALF + j4) / kGroup), (unsigned short)bb);
      }
      if (kind == 2 && j4 == 0) gstore<unsigned short>(sc, (unsigned short)ba);
    } else if (p.cache.elt == 2) {
      gstore(o + 2 * j4, f16x4{(_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3]});
      gstore(o + 2 * (HALF + j4), f16x4{(_Float16)b[0], (_Float16)b[1], (_Float16)b[2], (_Float16)b[3]});
    } else {
      gstore(o + 4 * j4, a);
      gstore(o + 4 * (HALF + j4), b);
    }
  }
}

hipError_t launch_norm_rope(const NormRope& p, hipStream_t stream) {
  const auto at16 = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; };
  if (p.n_dims == p.cache.head_dim && (!p.q || (rows_aligned(p.q, p.q_nb, 4) && rows_aligned(p.q_out, p.qo_nb, 4))) &&
      rows_aligned(p.k, p.k_nb, 4) && rows_aligned(p.v, p.v_nb, 4) && at16(p.q_norm) && at16(p.k_norm)) {
    if (p.n_tokens == 0) return hipSuccess;
    // Up to two workgroups of kRopeTokens tokens per CU: a workgroup per 256 lanes'
    // worth of one token's rows instead, more angles for more workgroups. 28/4 heads
    // of 128, F16 cache (us): 64 tokens 3.5 (by fours 8.9), 1024 8.8 (11.7), 2048
    // 15.6 (15.2), 4096 26.7 (23.8).
    const int per_tok = p.n_head + 2 * p.cache.n_head_kv, rows = 256 / (p.cache.head_dim / 8);
    const bool few = p.n_tokens < 2 * 256 * kRopeTokens;
    const dim3 grid((unsigned)(few ? p.n_tokens : (p.n_tokens + kRopeTokens - 1) / kRopeTokens),
                    (unsigned)(few ? (per_tok + rows - 1) / rows : 1));
    if (p.cache.head_dim == 64) hipLaunchKernelGGL(norm_rope_kernel<64>, grid, dim3(256), 0, stream, p, few ? 1 : kRopeTokens);
    else hipLaunchKernelGGL(norm_rope_kernel<128>, grid, dim3(256), 0, stream, p, few ? 1 : kRopeTokens);
    return hipGetLastError();
  }
  const int64_t rows = (int64_t)p.n_tokens * (p.n_head + 2 * p.cache.n_head_kv);
  if (rows == 0) return hipSuccess;
  const dim3 grid((unsigned)((rows + 3) / 4));
  const bool q8 = p.cache.elt == 1;
  if (p.cache.head_dim == 64) {
    if (q8) hipLaunchKernelGGL((norm_rope_row_kernel<1, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((norm_rope_row_kernel<1, false>), grid, dim3(256), 0, stream, p);
  } else {
    if (q8) hipLaunchKernelGGL((norm_rope_row_kernel<2, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((norm_rope_row_kernel<2, false>), grid, dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace mi
