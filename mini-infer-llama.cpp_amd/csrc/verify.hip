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
// probabilities that has to be summed over the row first: then the sequence has a
// workgroup per chunk, all of which walk, each sums its chunk, and the last one to
// get there draws.
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

// 2^t for t <= 0 (down to -infinity): the power series of e^(f ln 2) for the fraction
// f in [-1/2, 1/2], whose twelfth term is below 2^-47 and thirteenth below 2^-52.
__device__ inline double exp2_d(double t) {
  t = fmax(t, -2000.0);
  const double n = __builtin_rint(t), f = (t - n) * 0x1.62e42fefa39efp-1;  // ln 2
  double s = 1.0 / 479001600.0;
  s = fma(s, f, 1.0 / 39916800.0);
  s = fma(s, f, 1.0 / 3628800.0);
  s = fma(s, f, 1.0 / 362880.0);
  s = fma(s, f, 1.0 / 40320.0);
  s = fma(s, f, 1.0 / 5040.0);
  s = fma(s, f, 1.0 / 720.0);
  s = fma(s, f, 1.0 / 120.0);
  s = fma(s, f, 1.0 / 24.0);
  s = fma(s, f, 1.0 / 6.0);
  s = fma(s, f, 0.5);
  s = fma(s, f, 1.0);
  s = fma(s, f, 1.0);
  return __builtin_amdgcn_ldexp(s, (int)n);
}
constexpr double kLog2e = 0x1.71547652b82fep+0;

// What a row's logits are multiplied by, 0 for the greedy choice.
__device__ inline double row_scale(const Verify& p, int seq) {
  const float t = p.temperature ? p.temperature[seq] : 1.f;
  return t > 0.f ? kLog2e / (double)t : 0.0;
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
#pragma unroll
  for (int k = 0; k < PER; ++k) x[k] = load_row(in, 4 * (tid + kRowThreads * k), n, -INFINITY);
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

// The walk's shared memory.
struct Walk {
  double prob[kVerifyMaxNodes];  // of each node's token in its parent's row
  double bar[kVerifyMaxNodes];   // u, or u draft
  double sum[kVerifyMaxNodes];   // rows
  float top[kVerifyMaxNodes];
  int best[kVerifyMaxNodes];
  int token[kVerifyMaxNodes], up[kVerifyMaxNodes], down[kVerifyMaxNodes];
  double part[kWalkWaves];
  int last[kWalkWaves];
  int cur, n_down, len, chunk, joins;
  double before, target;
};

// The sum over the workgroup, the same on every thread; `below`: over the threads below.
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

}  // namespace

// CHUNK tokens a chunk, eight or four in a row per thread.
template <int CHUNK, bool DRAFT>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(const Verify p) {
  constexpr int PER = CHUNK / kWalkThreads;
  __shared__ Walk s;
  const int seq = p.seq0 + blockIdx.y, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const bool writes = blockIdx.x == 0;
  const int r0 = min(max(p.off[seq], 0), p.n_rows), n = min(min(max(p.off[seq + 1], r0), p.n_rows) - r0, kVerifyMaxNodes);
  int* const path = reinterpret_cast<int*>(p.path + seq * p.path_nb);
  int* const out = reinterpret_cast<int*>(p.tokens + seq * p.tokens_nb);
  if (n <= 0) {
    if (!writes) return;
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
    if (writes) path[0] = 0;
    for (int c = 1; c < n && len < p.max_path; ++c) {
      if (s.up[c] != cur) continue;
      bool again = false;
      for (int e = 0; e < n_down; ++e) again = again || s.token[s.down[e]] == s.token[c];
      const double pc = again ? 0.0 : s.prob[c];
      if ((DRAFT ? s.bar[c] : s.bar[c] * left) < pc) {
        if (writes) {
          out[len - 1] = s.token[c];
          path[len] = c;
        }
        ++len;
        cur = c;
        n_down = 0;
        left = 1.0;
      } else {
        left -= pc;
        s.down[n_down++] = c;
      }
    }
    s.cur = cur;
    s.len = len;
    s.n_down = len < p.max_path ? n_down : 0;
    if (writes) p.n_path[seq] = len;
  }
  __syncthreads();
  const int cur = s.cur, n_down = s.n_down, len = s.len;
  const bool less = DRAFT && n_down > 0;  // the draft's probabilities come off
  if (!less && !writes) return;
  if (writes) {
    for (int i = len + tid; i < p.max_path; i += kWalkThreads) path[i] = out[i] = -1;
  }
  const float top = s.top[cur];
  const char* const x = p.logits + (r0 + cur) * p.nb;
  const char* const q = less ? p.draft + (r0 + s.down[0]) * p.draft_nb : nullptr;
  if (!(top > -INFINITY && top < INFINITY)) {  // no distribution, no token
    if (writes && tid == 0) out[len - 1] = -1;
    return;
  }
  if (scale == 0.0) {
    // (the best token is never turned down, unless a draft had nothing else)
    if (writes && tid == 0) {
      const int t = s.best[cur];
      out[len - 1] = less && !(gload<float>(q + 4 * (int64_t)t) < 1.f) ? -1 : t;
    }
    return;
  }
  // What is left of chunk k: the thread's PER tokens in w, their sum.
  const double inv = 1.0 / s.sum[cur];
  auto rest = [&](int k, double (&w)[PER]) __attribute__((always_inline)) -> double {
    const int base = k * CHUNK, m = min(CHUNK, p.n_vocab - base), i0 = tid * PER;
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; j += 4) {
      const f32x4 v = load_row(x + 4 * (int64_t)base, i0 + j, m, -INFINITY);
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
      if (less) d = load_row(q + 4 * (int64_t)base, i0 + j, m, 0.f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[j + e] = weight(v[e], top, scale);
        if (less) w[j + e] = fmax(w[j + e] * inv - (double)d[e], 0.0);
      }
    }
    if (!DRAFT) {
      for (int e = 0; e < n_down; ++e) {
        const unsigned t = (unsigned)(s.token[s.down[e]] - base - i0);
#pragma unroll
        for (int j = 0; j < PER; ++j) w[j] = t == (unsigned)j ? 0.0 : w[j];
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += w[j];
    return sum;
  };
  double w[PER], below;
  double* const sums = p.sums + (int64_t)blockIdx.y * p.n_chunks;  // of the sequence's chunks, where `less`
  if (less) {
    for (int k = blockIdx.x; k < p.n_chunks; k += gridDim.x) {
      const double all = block_sum(s, rest(k, w), below);
      if (tid == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t*>(sums + k), __builtin_bit_cast(uint64_t, all), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid == 0) {
      wait_vmem<0>();
      unsigned* const counter = p.arrived + kArrivalWords * blockIdx.y;
      const unsigned done = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (done == gridDim.x - 1) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s.joins = done == gridDim.x - 1;
    }
    __syncthreads();
    if (!s.joins) return;
  }
  // Chunks that tokens turned down have left are summed anew (into s.prob, by the token).
  const int n_out = DRAFT ? 0 : n_down;
  for (int e = 0; e < n_out; ++e) {
    const int t = s.token[s.down[e]];
    const double all = (unsigned)t < (unsigned)p.n_vocab ? block_sum(s, rest(t / CHUNK, w), below) : 0.0;
    if (tid == 0) s.prob[e] = all;
  }
  __syncthreads();
  auto chunk_sum = [&](int k) __attribute__((always_inline)) -> double {
    if (k >= p.n_chunks) return 0.0;
    if (less)
      return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(sums + k), __ATOMIC_RELAXED,
                                                          __HIP_MEMORY_SCOPE_AGENT));
    const VerifyPart c = p.parts[(int64_t)(r0 + cur) * p.n_chunks + k];
    double sum = c.top > -INFINITY ? c.sum * weight(c.top, top, scale) : 0.0;
    for (int e = 0; e < n_out; ++e) sum = s.token[s.down[e]] / CHUNK == k ? s.prob[e] : sum;
    return sum;
  };
  // The chunk that holds the token.
  if (wave == 0) {
    double total = 0.0;
    for (int k = 0; k < p.n_chunks; k += kWave) total += wave_sum_f64(chunk_sum(k + lane));
    const double target = s.bar[0] * total;
    double before = 0.0, start = 0.0;
    int chunk = -1;
    for (int k = 0; k < p.n_chunks; k += kWave) {
      const double c = chunk_sum(k + lane);
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
      s.chunk = chunk;
      s.before = start;
      s.target = target;
    }
  }
  __syncthreads();
  const int chunk = s.chunk;
  if (chunk < 0) {  // nothing is left
    if (tid == 0) out[len - 1] = -1;
    return;
  }
  // The token: the first with a weight whose sum is above the target, or the last.
  const double mine_sum = rest(chunk, w), target = s.target;
  block_sum(s, mine_sum, below);
  double cum = s.before + below;
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
  __syncthreads();
  if (lane == 0) {
    s.last[wave] = last;
    s.down[wave] = first;
  }
  __syncthreads();
  if (tid == 0) {
    for (int o = 1; o < kWalkWaves; ++o) {
      first = min(first, s.down[o]);
      last = max(last, s.last[o]);
    }
    out[len - 1] = first != INT32_MAX ? first : last;
  }
}

// Chunks of 2048 tokens while a launch has few workgroups.
static int chunk_of(int64_t n_rows, int n_vocab, int n_cu) {
  return n_rows * ((n_vocab + 4095) / 4096) <= 2 * n_cu ? 2048 : 4096;
}

size_t verify_scratch(int n_rows, int n_seq, int n_vocab, int n_cu) {
  const int chunk = chunk_of(n_rows, n_vocab, n_cu);
  const size_t chunks = ((size_t)n_vocab + chunk - 1) / chunk;
  return chunks * ((size_t)n_rows * sizeof(VerifyPart) + (size_t)std::min(n_seq, kArrivals) * sizeof(double));
}

template <int CHUNK>
static hipError_t launch_verify_t(Verify p, int n_cu, hipStream_t stream) {
  constexpr int kRows = 65535;  // of a grid
  p.n_chunks = (p.n_vocab + CHUNK - 1) / CHUNK;
  p.sums = reinterpret_cast<double*>(p.parts + (int64_t)p.n_rows * p.n_chunks);
  hipError_t e = hipSuccess;
  for (p.row0 = 0; p.row0 < p.n_rows && e == hipSuccess; p.row0 += kRows) {
    hipLaunchKernelGGL(verify_rows_kernel<CHUNK>, dim3((unsigned)p.n_chunks, (unsigned)std::min(kRows, p.n_rows - p.row0)),
                       dim3(kRowThreads), 0, stream, p);
    e = hipGetLastError();
  }
  // As many sequences a launch as there are arrival counters.
  for (p.seq0 = 0; p.seq0 < p.n_seq && e == hipSuccess; p.seq0 += kArrivals) {
    const int n = std::min(kArrivals, p.n_seq - p.seq0);
    const unsigned wgs = p.draft ? (unsigned)std::min(p.n_chunks, std::max(1, 2 * n_cu / n)) : 1u;
    if (p.draft) hipLaunchKernelGGL((verify_walk_kernel<CHUNK, true>), dim3(wgs, (unsigned)n), dim3(kWalkThreads), 0, stream, p);
    else hipLaunchKernelGGL((verify_walk_kernel<CHUNK, false>), dim3(wgs, (unsigned)n), dim3(kWalkThreads), 0, stream, p);
    e = hipGetLastError();
  }
  return e;
}

hipError_t launch_verify(const Verify& p, int n_cu, hipStream_t stream) {
  return chunk_of(p.n_rows, p.n_vocab, n_cu) == 2048 ? launch_verify_t<2048>(p, n_cu, stream) : launch_verify_t<4096>(p, n_cu, stream);
}

}  // namespace mi
