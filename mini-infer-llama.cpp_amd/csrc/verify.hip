// verify.hip -- verification of drafted tokens against the target's
// probabilities, from given random numbers.
//
// p_v = softmax(logits_v / T). The tests (u Z < p or u q < p) and the draw are those
// of the header, all in double: which token comes out depends on which side of a
// border between two tokens a number falls, and with 2^-24 in each of 150000
// probabilities about one draw in a hundred would fall differently. Equal logits
// have equal weights exactly (each is 2^0).
//
// verify_rows_kernel: a workgroup has a chunk of one row in registers and leaves its
// largest logit m and sum 2^((x - m) log2(e) / T), so every logit is read once.
// verify_walk_kernel: a workgroup per sequence joins the chunks of its rows, finds
// each drafted token's probability, walks from node to node, and draws: the
// chunks' sums say which chunk the token is in, whose weights are then formed once
// more. Where a draft's token was turned down, what is left is a difference of
// probabilities that has to be summed over the row first: verify_rest_kernel does
// that with several workgroups a sequence, the last of which draws.
//
// Bound: for many rows the vector unit, 27 instructions a logit, 20 of them double
// (384 rows of 151936: 54 us, 33 to read them), for few the launches' chains of loads
// (up to six rows 13 us).
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any 4 bytes
__device__ inline f32x4 load4(const char* p) { return *(const __attribute__((address_space(1))) f32x4_any*)p; }

constexpr int kRowThreads = 256, kWalkThreads = 512, kWalkWaves = kWalkThreads / kWave;

// Four values from element i on of a row of n, `pad` behind its end.
__device__ inline f32x4 load_row(const char* row, int i, int n, float pad) {
  if (i + 4 <= n) return load4(row + 4 * (int64_t)i);
  f32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = i + j < n ? gload<float>(row + 4 * (int64_t)(i + j)) : pad;
  return v;
}

// 2^t for t <= 0 (down to -infinity): the whole part is the low word of t + 1.5 2^52,
// the fraction f in [-1/2, 1/2] by 1 + f g(f), g of
// degree 9 through (2^f - 1) / f at the ten Chebyshev points: at most 6e-16 off, and 1
// for 0. (The power series needs two terms more.)
__device__ inline double exp2_d(double t) {
  t = fmax(t, -2000.0);
  const double m = t + 0x1.8p+52, f = t - (m - 0x1.8p+52);
  double s = 0x1.e5e9f548e5726p-28;
  s = fma(s, f, 0x1.b6571de2f2351p-24);
  s = fma(s, f, 0x1.62bfe46117445p-20);
  s = fma(s, f, 0x1.ffcb76789860fp-17);
  s = fma(s, f, 0x1.4309130378460p-13);
  s = fma(s, f, 0x1.5d87fe908f88ap-10);
  s = fma(s, f, 0x1.3b2ab6fba385fp-7);
  s = fma(s, f, 0x1.c6b08d7044119p-5);
  s = fma(s, f, 0x1.ebfbdff82c590p-3);
  s = fma(s, f, 0x1.62e42fefa39f7p-1);
  s = fma(s, f, 1.0);
  return __builtin_amdgcn_ldexp(s, (int)__builtin_bit_cast(uint64_t, m));
}
constexpr double kLog2e = 0x1.71547652b82fep+0;

// What a row's logits are multiplied by, 0 for the greedy choice.
__device__ inline double row_scale(const Verify& p, int seq) {
  const float t = p.temperature ? p.temperature[seq] : 1.f;
  return t > 0.f ? fmax(kLog2e / (double)t, 1e-300) : 0.0;  // (infinity: all weights 1)
}
__device__ inline double weight(float x, float top, double scale) { return exp2_d(((double)x - (double)top) * scale); }

__device__ inline double wave_scan(double x, int lane) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const double y = __shfl_up(x, off, kWave);
    x += lane >= off ? y : 0.0;
  }
  return x;
}
__device__ inline int wave_min(int x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = min(x, __shfl_xor(x, off, kWave));
  return x;
}
__device__ inline int wave_max_int(int x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = max(x, __shfl_xor(x, off, kWave));
  return x;
}
// NaN if one is.
__device__ inline float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

}  // namespace

template <int CHUNK>
__global__ __launch_bounds__(kRowThreads) void verify_rows_kernel(const Verify p) {
  constexpr int PER = CHUNK / (4 * kRowThreads), WAVES = kRowThreads / kWave;
  __shared__ float tops[WAVES];
  __shared__ double sums[WAVES];
  __shared__ int bests[WAVES];
  const int row = p.row0 + blockIdx.y, base = blockIdx.x * CHUNK, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int n = min(CHUNK, p.n_vocab - base);
  const char* const in = p.logits + row * p.nb + 4 * (int64_t)base;
  f32x4 x[PER];
  if (n == CHUNK) {  // (all on their way at once)
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = load4(in + 16 * (tid + kRowThreads * k));
  } else {
#pragma unroll
    for (int k = 0; k < PER; ++k) x[k] = load_row(in, 4 * (tid + kRowThreads * k), n, -INFINITY);
  }
  int seq = 0;  // the last sequence that begins at or before the row
  if (p.temperature) {
    for (int i = 0; i < p.n_seq; i += kWave)
      seq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(i + lane < p.n_seq && p.off[i + lane] <= row));
    seq = max(seq - 1, 0);
  }
  const double scale = row_scale(p, seq);
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < PER; ++k)
    top = max_nan(max_nan(max_nan(top, x[k][0]), x[k][1]), max_nan(x[k][2], x[k][3]));
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = max_nan(top, __shfl_xor(top, off, kWave));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = max_nan(top, tops[w]);
  VerifyPart r{0.0, top, 0};
  if (top > -INFINITY && top < INFINITY) {
    if (scale > 0.0) {
      double sum = 0.0;
#pragma unroll
      for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += weight(x[k][j], top, scale);
      sum = wave_sum_f64(sum);
      if (lane == 0) sums[wave] = sum;
    } else {
      int best = INT32_MAX;
#pragma unroll
      for (int k = 0; k < PER; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) best = x[k][j] == top ? min(best, base + 4 * (tid + kRowThreads * k) + j) : best;
      best = wave_min(best);
      if (lane == 0) bests[wave] = best;
    }
    __syncthreads();
    if (scale > 0.0) {
      for (int w = 0; w < WAVES; ++w) r.sum += sums[w];
    } else {
      r.best = INT32_MAX;
      for (int w = 0; w < WAVES; ++w) r.best = min(r.best, bests[w]);
    }
  }
  if (tid == 0) p.parts[(int64_t)row * gridDim.x + blockIdx.x] = r;
}

namespace {

// A row's chunks together: the largest logit, the sum of the weights, the lowest
// token of the largest (greedy rows). By a whole wave.
struct RowSums {
  float top;  // not finite: the row has no distribution
  double sum;
  int best;
};
__device__ inline RowSums join_row(const Verify& p, int row, double scale, int lane) {
  const VerifyPart* const part = p.parts + (int64_t)row * p.n_chunks;
  RowSums r{-INFINITY, 0.0, INT32_MAX};
  for (int i = lane; i < p.n_chunks; i += kWave) {
    const VerifyPart c = part[i];
    const float top = max_nan(r.top, c.top);
    if (scale > 0.0) {
      if (top > -INFINITY) r.sum = r.sum * weight(r.top, top, scale) + c.sum * weight(c.top, top, scale);
    } else {
      r.best = c.top > r.top ? c.best : c.top == r.top ? min(r.best, c.best) : r.best;
    }
    r.top = top;
  }
  float top = r.top;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = max_nan(top, __shfl_xor(top, off, kWave));
  if (!(top > -INFINITY && top < INFINITY)) return RowSums{top, 0.0, 0};
  if (scale > 0.0) r.sum = wave_sum_f64(r.top > -INFINITY ? r.sum * weight(r.top, top, scale) : 0.0);
  else r.best = wave_min(r.top == top ? r.best : INT32_MAX);
  r.top = top;
  return r;
}

// The walk's shared memory: arrays of as many nodes as a sequence can have.
struct Walk {
  double* prob;  // of each node's token in its parent's row
  double* bar;   // u, or u draft
  double* sum;   // rows
  float* top;
  int* best;
  int *token, *up, *down;
  double* part;  // of the waves
  int* last;
  struct Found {
    int cur, n_down, len, chunk, joins, unused;
    double before, target;
  }* f;
  static constexpr int kNodeBytes = 3 * 8 + 5 * 4, kFixed = kWalkWaves * (8 + 2 * 4) + (int)sizeof(Found);
  __device__ inline Walk(char* lds, int nodes) {
    f = reinterpret_cast<Found*>(lds);
    part = reinterpret_cast<double*>(f + 1);
    prob = part + kWalkWaves;
    bar = prob + nodes;
    sum = bar + nodes;
    top = reinterpret_cast<float*>(sum + nodes);
    best = reinterpret_cast<int*>(top + nodes);
    token = best + nodes;
    up = token + nodes;
    down = up + nodes;
    last = down + nodes;
  }
};

// The sum over the workgroup, the same on every thread.
__device__ inline double block_total(Walk& s, double x) {
  x = wave_sum_f64(x);
  __syncthreads();  // (s.part has been read)
  if (threadIdx.x % kWave == 0) s.part[threadIdx.x / kWave] = x;
  __syncthreads();
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < kWalkWaves; ++w) all += s.part[w];
  return all;
}
// The same, and `below`: over the threads below.
__device__ inline double block_sum(Walk& s, double x, double& below) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const double incl = wave_scan(x, lane);
  __syncthreads();  // (s.part has been read)
  if (lane == kWave - 1) s.part[wave] = incl;
  __syncthreads();
  double all = 0.0, before = 0.0;
#pragma unroll
  for (int w = 0; w < kWalkWaves; ++w) {
    before += w < wave ? s.part[w] : 0.0;
    all += s.part[w];
  }
  below = before + (incl - x);
  return all;
}

// What a sequence's last token is drawn from: p of the row, or with LESS max(p - draft,
// 0), in chunks of CHUNK tokens, PER in a row for each thread.
template <int CHUNK, bool LESS>
struct Remainder {
  static constexpr int PER = CHUNK / kWalkThreads;
  const char *x, *q;  // the row's logits, the draft's probabilities
  float top;
  double scale, inv;  // inv: 1 / the sum of the weights
  int n_vocab;
  const int *token, *down;  // n_out tokens of the vocabulary that are left out: token[down[e]]
  int n_out;

  struct Tokens {
    f32x4 x[PER / 4], q[PER / 4];
  };
  __device__ __forceinline__ void load(int k, Tokens& v) const {
    const int base = k * CHUNK, m = min(CHUNK, n_vocab - base), i0 = (int)threadIdx.x * PER;
    const char* const xk = x + 4 * (int64_t)base;
    const char* const qk = LESS ? q + 4 * (int64_t)base : nullptr;
    if (m == CHUNK) {  // (all on their way at once)
#pragma unroll
      for (int j = 0; j < PER / 4; ++j) {
        v.x[j] = load4(xk + 4 * (i0 + 4 * j));
        if (LESS) v.q[j] = load4(qk + 4 * (i0 + 4 * j));
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER / 4; ++j) {
        v.x[j] = load_row(xk, i0 + 4 * j, m, -INFINITY);
        if (LESS) v.q[j] = load_row(qk, i0 + 4 * j, m, 0.f);
      }
    }
  }
  // The thread's tokens of chunk k: what is left of each, and their sum.
  __device__ __forceinline__ double rest(int k, const Tokens& v, double (&w)[PER]) const {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      w[j] = weight(v.x[j / 4][j % 4], top, scale);
      if (LESS) w[j] = fmax(w[j] * inv - (double)v.q[j / 4][j % 4], 0.0);
    }
    for (int e = 0; e < n_out; ++e) {
      const unsigned t = (unsigned)(token[down[e]] - k * CHUNK - (int)threadIdx.x * PER);
#pragma unroll
      for (int j = 0; j < PER; ++j) w[j] = t == (unsigned)j ? 0.0 : w[j];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += w[j];
    return sum;
  }

  // The token drawn by u, given each chunk's sum: the first with a weight up to which
  // the sum is above u times the whole; -1 if nothing is left. Called by all threads,
  // valid on thread 0.
  template <typename ChunkSum>
  __device__ int draw(Walk& s, double u, int n_chunks, ChunkSum chunk_sum) const {
    const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
    if (wave == 0) {
      double total = 0.0, first[2] = {0.0, 0.0};  // (the first 128 chunks' are kept)
      for (int k = 0; k < n_chunks; k += kWave) {
        const double c = k + lane < n_chunks ? chunk_sum(k + lane) : 0.0;
        if (k < kWave) first[0] = c;
        else if (k < 2 * kWave) first[1] = c;
        total += wave_sum_f64(c);
      }
      const double target = u * total;
      double before = 0.0, start = 0.0;
      int chunk = -1;
      for (int k = 0; k < n_chunks; k += kWave) {
        const double c = k < kWave ? first[0] : k < 2 * kWave ? first[1] : k + lane < n_chunks ? chunk_sum(k + lane) : 0.0;
        const double incl = before + wave_scan(c, lane);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(c > 0.0 && incl > target);
        const uint64_t any = __builtin_amdgcn_ballot_w64(c > 0.0);
        if (hit || any) {  // (the last with a weight, if rounding passes them all)
          const int at = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
          chunk = k + at;
          start = __shfl(incl - c, at, kWave);
        }
        if (hit) break;
        before = __shfl(incl, kWave - 1, kWave);
      }
      if (lane == 0) {
        s.f->chunk = chunk;
        s.f->before = start;
        s.f->target = target;
      }
    }
    __syncthreads();
    const int chunk = s.f->chunk;
    if (chunk < 0) return -1;
    Tokens v;
    double w[PER], below;
    load(chunk, v);
    const double target = s.f->target;
    block_sum(s, rest(chunk, v, w), below);
    double cum = s.f->before + below;
    int first = INT32_MAX, last = -1;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      cum += w[j];
      const int t = chunk * CHUNK + tid * PER + j;
      if (w[j] > 0.0) {
        last = t;
        if (cum > target) first = min(first, t);
      }
    }
    first = wave_min(first);
    last = wave_max_int(last);
    if (lane == 0) {
      s.last[wave] = last;
      s.last[kWalkWaves + wave] = first;
    }
    __syncthreads();
    for (int o = 0; o < kWalkWaves; ++o) {
      last = max(last, s.last[o]);
      first = min(first, s.last[kWalkWaves + o]);
    }
    return first != INT32_MAX ? first : last;
  }
};

}  // namespace

// A workgroup per sequence.
template <int CHUNK, bool DRAFT>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(const Verify p) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  Walk s(lds_raw, p.max_nodes);
  const int seq = p.seq0 + blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int r0 = min(max(p.off[seq], 0), p.n_rows), n = min(min(max(p.off[seq + 1], r0), p.n_rows) - r0, p.max_nodes);
  int* const path = reinterpret_cast<int*>(p.path + seq * p.path_nb);
  int* const out = reinterpret_cast<int*>(p.tokens + seq * p.tokens_nb);
  if (DRAFT && tid == 0) p.left[blockIdx.x].down = -1;  // (nothing for verify_rest_kernel)
  if (n <= 0) {
    for (int i = tid; i < p.max_path; i += kWalkThreads) path[i] = out[i] = -1;
    if (tid == 0) p.n_path[seq] = 0;
    return;
  }
  const double scale = row_scale(p, seq);
  // Each node's token, its logit in the parent's row, and its test.
  float mine = 0.f;  // thread c's node c, of the first kWalkThreads
  auto node = [&](int c) __attribute__((always_inline)) -> float {
    const int t = p.token[r0 + c], v = p.parent ? p.parent[r0 + c] : c - 1;
    const float u = fminf(fmaxf(p.u[r0 + c], 0.f), 0x1.fffffep-1f);
    const bool there = c > 0 && v >= 0 && v < c && (unsigned)t < (unsigned)p.n_vocab;
    s.token[c] = t;
    s.up[c] = c > 0 && v >= 0 && v < c ? v : -1;
    s.bar[c] = DRAFT && there ? (double)u * (double)gload<float>(p.draft + (r0 + c) * p.draft_nb + 4 * (int64_t)t) : (double)u;
    return there ? gload<float>(p.logits + (r0 + v) * p.nb + 4 * (int64_t)t) : -INFINITY;
  };
  if (tid < n) mine = node(tid);
  for (int r = wave; r < n; r += kWalkWaves) {
    const RowSums row = join_row(p, r0 + r, scale, lane);
    if (lane == 0) {
      s.top[r] = row.top;
      s.sum[r] = row.sum;
      s.best[r] = row.best;
    }
  }
  __syncthreads();
  for (int c = tid; c < n; c += kWalkThreads) {
    const float x = c < kWalkThreads ? mine : node(c);
    const int v = s.up[c];
    double pc = 0.0;
    if (v >= 0 && x > -INFINITY && s.top[v] < INFINITY)
      pc = scale > 0.0 ? weight(x, s.top[v], scale) / s.sum[v] : s.token[c] == s.best[v] ? 1.0 : 0.0;
    s.prob[c] = pc;
  }
  __syncthreads();
  if (tid == 0) {
    int cur = 0, len = 1, n_down = 0;
    double left = 1.0;
    path[0] = 0;
    for (int c = 1; c < n && len < p.max_path; ++c) {
      if (s.up[c] != cur) continue;
      bool again = false;
      for (int e = 0; e < n_down; ++e) again = again || s.token[s.down[e]] == s.token[c];
      const double pc = again ? 0.0 : s.prob[c];
      if ((DRAFT ? s.bar[c] : s.bar[c] * left) < pc) {
        out[len - 1] = s.token[c];
        path[len++] = c;
        cur = c;
        n_down = 0;
        left = 1.0;
      } else {
        left -= pc;
        // (a token outside the vocabulary takes nothing off the row, and has no chunk of it)
        if (DRAFT || (unsigned)s.token[c] < (unsigned)p.n_vocab) s.down[n_down++] = c;
      }
    }
    s.f->cur = cur;
    s.f->len = len;
    s.f->n_down = len < p.max_path ? n_down : 0;
    p.n_path[seq] = len;
  }
  __syncthreads();
  const int cur = s.f->cur, n_down = s.f->n_down, len = s.f->len;
  for (int i = len + tid; i < p.max_path; i += kWalkThreads) path[i] = out[i] = -1;
  const bool less = DRAFT && n_down > 0;  // the draft's probabilities come off
  const float top = s.top[cur];
  const char* const x = p.logits + (r0 + cur) * p.nb;
  if (!(top > -INFINITY && top < INFINITY)) {  // no distribution, no token
    if (tid == 0) out[len - 1] = -1;
    return;
  }
  if (scale == 0.0) {
    // (the best token is never turned down, unless a draft had nothing else)
    if (tid == 0) {
      const int t = s.best[cur];
      const float q = less ? gload<float>(p.draft + (r0 + s.down[0]) * p.draft_nb + 4 * (int64_t)t) : 0.f;
      out[len - 1] = q < 1.f ? t : -1;
    }
    return;
  }
  if (less) {  // the rest of the row is another kernel's
    if (tid == 0) p.left[blockIdx.x] = VerifyLeft{scale, 1.0 / s.sum[cur], s.bar[0], top, r0 + cur, r0 + s.down[0], len - 1};
    return;
  }
  const Remainder<CHUNK, false> row{x, nullptr, top, scale, 0.0, p.n_vocab, s.token, s.down, DRAFT ? 0 : n_down};
  // Chunks that tokens turned down have left are summed anew (into s.prob, by the token).
  for (int e = 0; e < row.n_out; ++e) {
    const int chunk = s.token[s.down[e]] / CHUNK;
    typename Remainder<CHUNK, false>::Tokens v;
    double w[Remainder<CHUNK, false>::PER];
    row.load(chunk, v);
    const double all = block_total(s, row.rest(chunk, v, w));
    if (tid == 0) s.prob[e] = all;
  }
  __syncthreads();
  const int t = row.draw(s, s.bar[0], p.n_chunks, [&](int k) __attribute__((always_inline)) -> double {
    const VerifyPart c = p.parts[(int64_t)(r0 + cur) * p.n_chunks + k];
    double sum = c.top > -INFINITY ? c.sum * weight(c.top, top, scale) : 0.0;
    for (int e = 0; e < row.n_out; ++e) sum = s.token[s.down[e]] / CHUNK == k ? s.prob[e] : sum;
    return sum;
  });
  if (tid == 0) out[len - 1] = t;
}

// Sequences whose draft's token was turned down: the workgroups of grid row y sum what
// is left of the row of sequence seq0 + y, the last to arrive draws.
template <int CHUNK>
__global__ __launch_bounds__(kWalkThreads) void verify_rest_kernel(const Verify p) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  typedef Remainder<CHUNK, true> R;
  Walk s(lds_raw, 0);
  const VerifyLeft left = p.left[blockIdx.y];
  if (left.down < 0) return;
  const R row{p.logits + left.row * p.nb, p.draft + left.down * p.draft_nb, left.top, left.scale, left.inv, p.n_vocab,
              nullptr, nullptr, 0};
  double* const sums = p.sums + (int64_t)blockIdx.y * p.n_chunks;
  const int tid = threadIdx.x;
  typename R::Tokens v;
  double w[R::PER];
  row.load(blockIdx.x, v);
  for (int k = blockIdx.x; k < p.n_chunks; k += gridDim.x) {
    if (k != (int)blockIdx.x) row.load(k, v);
    const double all = block_total(s, row.rest(k, v, w));
    if (tid == 0)
      __hip_atomic_store(reinterpret_cast<uint64_t*>(sums + k), __builtin_bit_cast(uint64_t, all), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
  }
  if (tid == 0) {
    wait_vmem<0>();
    unsigned* const counter = p.arrived + kArrivalWords * blockIdx.y;
    const unsigned done = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (done == gridDim.x - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s.f->joins = done == gridDim.x - 1;
  }
  __syncthreads();
  if (!s.f->joins) return;
  const int t = row.draw(s, left.u, p.n_chunks, [&](int k) __attribute__((always_inline)) -> double {
    return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(sums + k), __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT));
  });
  if (tid == 0) reinterpret_cast<int*>(p.tokens + (p.seq0 + (int)blockIdx.y) * p.tokens_nb)[left.at] = t;
}

// Chunks of 2048 tokens while a launch has few workgroups.
static int chunk_of(int64_t n_rows, int n_vocab, int n_cu) {
  return n_rows * ((n_vocab + 4095) / 4096) <= 2 * n_cu ? 2048 : 4096;
}

size_t verify_scratch(int n_rows, int n_seq, int n_vocab, int n_cu) {
  const int chunk = chunk_of(n_rows, n_vocab, n_cu);
  const size_t chunks = ((size_t)n_vocab + chunk - 1) / chunk;
  return chunks * (size_t)n_rows * sizeof(VerifyPart) + (size_t)std::min(n_seq, kArrivals) * (sizeof(VerifyLeft) + chunks * sizeof(double));
}

template <int CHUNK>
static hipError_t launch_verify_t(Verify p, int n_cu, hipStream_t stream) {
  constexpr int kRows = 65535;  // of a grid
  p.n_chunks = (p.n_vocab + CHUNK - 1) / CHUNK;
  p.left = reinterpret_cast<VerifyLeft*>(p.parts + (int64_t)p.n_rows * p.n_chunks);
  p.sums = reinterpret_cast<double*>(p.left + std::min(p.n_seq, kArrivals));
  p.max_nodes = std::min(p.n_rows, kVerifyMaxNodes);
  const int lds = Walk::kFixed + Walk::kNodeBytes * p.max_nodes;
  hipError_t e = hipSuccess;
  for (p.row0 = 0; p.row0 < p.n_rows && e == hipSuccess; p.row0 += kRows) {
    hipLaunchKernelGGL(verify_rows_kernel<CHUNK>, dim3((unsigned)p.n_chunks, (unsigned)std::min(kRows, p.n_rows - p.row0)),
                       dim3(kRowThreads), 0, stream, p);
    e = hipGetLastError();
  }
  // As many sequences a launch as there are arrival counters.
  for (p.seq0 = 0; p.seq0 < p.n_seq && e == hipSuccess; p.seq0 += kArrivals) {
    const int n = std::min(kArrivals, p.n_seq - p.seq0);
    if (!p.draft) {
      hipLaunchKernelGGL((verify_walk_kernel<CHUNK, false>), dim3((unsigned)n), dim3(kWalkThreads), lds, stream, p);
    } else {
      hipLaunchKernelGGL((verify_walk_kernel<CHUNK, true>), dim3((unsigned)n), dim3(kWalkThreads), lds, stream, p);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
      // (up to 16 workgroups per CU: 4 of them, with the next chunk on its way, 64 rows 7 us slower)
      const unsigned wgs = (unsigned)std::min(p.n_chunks, std::max(1, 16 * n_cu / n));
      hipLaunchKernelGGL(verify_rest_kernel<CHUNK>, dim3(wgs, (unsigned)n), dim3(kWalkThreads), Walk::kFixed, stream, p);
    }
    e = hipGetLastError();
  }
  return e;
}

hipError_t launch_verify(const Verify& p, int n_cu, hipStream_t stream) {
  return chunk_of(p.n_rows, p.n_vocab, n_cu) == 2048 ? launch_verify_t<2048>(p, n_cu, stream) : launch_verify_t<4096>(p, n_cu, stream);
}

}  // namespace mi
