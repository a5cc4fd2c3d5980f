// verify.hip -- verification of drafted tokens against the target's
// probabilities, from given random numbers.
//
// p_v = softmax(logits_v / T), all in double: which token comes out depends on
// which side of a border between two tokens a number falls, and with 2^-24 in
// each of 150000 probabilities about one draw in a hundred would fall
// differently. The tests (u Z < p or u q < p) and the draw are those of the
// header; equal logits have equal weights exactly (each is exp(0)).
#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

// Larger for the larger value, and for the lower token among equal values; -0 is 0.
__device__ inline uint64_t key_of(float v, int t) {
  const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);
  const unsigned o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (unsigned)~t;
}
__device__ inline float key_value(uint64_t k) {
  const unsigned o = (unsigned)(k >> 32);
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ inline uint64_t shfl_xor64(uint64_t x, int off) {
  return (uint64_t)(unsigned)__shfl_xor((int)(x >> 32), off, kWave) << 32 | (unsigned)__shfl_xor((int)x, off, kWave);
}
__device__ inline double wave_scan(double x, int lane) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const double y = __shfl_up(x, off, kWave);
    x += lane >= off ? y : 0.0;
  }
  return x;
}

// The weight of a token relative to the row's largest logit m.
__device__ inline double weight(float x, int t, const VerifyRow& r, double inv_t) {
  if (inv_t == 0.0) return t == r.best ? 1.0 : 0.0;
  return x == -INFINITY ? 0.0 : exp(((double)x - (double)r.top) * inv_t);
}

// 1 / temperature, 0 for the greedy choice.
__device__ inline double inverse_temperature(const Verify& p, int seq) {
  const float t = p.temperature ? p.temperature[seq] : 1.f;
  return t > 0.f ? 1.0 / (double)t : 0.0;
}

constexpr int kRowThreads = 256, kWalkThreads = 1024;

}  // namespace

__global__ __launch_bounds__(kRowThreads) void verify_rows_kernel(const Verify p) {
  __shared__ uint64_t best[kRowThreads / kWave];
  __shared__ int bad[kRowThreads / kWave];
  __shared__ double part[kRowThreads / kWave];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int seq = 0;  // the last sequence that begins at or before the row
  for (int hi = p.n_seq - 1; seq < hi;) {
    const int mid = (seq + hi + 1) / 2;
    if (p.off[mid] <= row) seq = mid;
    else hi = mid - 1;
  }
  const double inv_t = inverse_temperature(p, seq);
  const char* const x = p.logits + row * p.nb;
  uint64_t top = 0;
  bool not_ok = false;
  for (int t = tid; t < p.n_vocab; t += kRowThreads) {
    const float v = gload<float>(x + 4 * (int64_t)t);
    not_ok |= !(v < INFINITY);
    const uint64_t k = key_of(v, t);
    top = k > top ? k : top;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint64_t y = shfl_xor64(top, off);
    top = y > top ? y : top;
  }
  if (lane == 0) best[wave] = top;
  if (lane == 0) bad[wave] = 0;
  if (__builtin_amdgcn_ballot_w64(not_ok) != 0ull && lane == 0) bad[wave] = 1;
  __syncthreads();
  int any = 0;
  for (int w = 0; w < kRowThreads / kWave; ++w) {
    top = best[w] > top ? best[w] : top;
    any |= bad[w];
  }
  VerifyRow r;
  r.best = (int)~(unsigned)top;
  r.top = any ? NAN : key_value(top);
  double sum = 0.0;
  for (int t = tid; t < p.n_vocab; t += kRowThreads) sum += weight(gload<float>(x + 4 * (int64_t)t), t, r, inv_t);
  sum = wave_sum_f64(sum);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    r.sum = 0.0;
    for (int w = 0; w < kRowThreads / kWave; ++w) r.sum += part[w];
    p.rows[row] = r;
  }
}

__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(const Verify p) {
  constexpr int kWaves = kWalkThreads / kWave;
  __shared__ double prob[kVerifyMaxNodes];  // of each node's token in its parent's row
  __shared__ double bar[kVerifyMaxNodes];   // u, or u draft
  __shared__ int token[kVerifyMaxNodes], up[kVerifyMaxNodes], down[kVerifyMaxNodes];
  __shared__ double part[kWaves];
  __shared__ int last[kWaves], s_cur, s_down, s_len;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int r0 = min(max(p.off[seq], 0), p.n_rows), n = min(min(max(p.off[seq + 1], r0), p.n_rows) - r0, kVerifyMaxNodes);
  int* const path = reinterpret_cast<int*>(p.path + seq * p.path_nb);
  int* const out = reinterpret_cast<int*>(p.tokens + seq * p.tokens_nb);
  for (int i = tid; i < p.max_path; i += kWalkThreads) path[i] = out[i] = -1;
  if (n <= 0) {
    if (tid == 0) p.n_path[seq] = 0;
    return;
  }
  const double inv_t = inverse_temperature(p, seq);
  for (int c = tid; c < n; c += kWalkThreads) {
    const int t = p.token[r0 + c], v = p.parent ? p.parent[r0 + c] : c - 1;
    double pc = 0.0;
    if (c > 0 && v >= 0 && v < c && (unsigned)t < (unsigned)p.n_vocab) {
      const VerifyRow r = p.rows[r0 + v];
      if (r.top > -INFINITY)
        pc = weight(gload<float>(p.logits + (r0 + v) * p.nb + 4 * (int64_t)t), t, r, inv_t) / r.sum;
    }
    const double u = (double)fminf(fmaxf(p.u[r0 + c], 0.f), 0x1.fffffep-1f);
    prob[c] = pc;
    bar[c] = p.draft && c > 0 && (unsigned)t < (unsigned)p.n_vocab
                 ? u * (double)gload<float>(p.draft + (r0 + c) * p.draft_nb + 4 * (int64_t)t) : u;
    token[c] = t;
    up[c] = v;
  }
  __syncthreads();
  if (tid == 0) {
    int cur = 0, len = 1, n_down = 0;
    double left = 1.0;
    path[0] = 0;
    for (int c = 1; c < n && len < p.max_path; ++c) {
      if (up[c] != cur) continue;
      bool again = false;
      for (int e = 0; e < n_down; ++e) again = again || token[down[e]] == token[c];
      const double pc = again ? 0.0 : prob[c];
      if ((p.draft ? bar[c] : bar[c] * left) < pc) {
        out[len - 1] = token[c];
        path[len++] = c;
        cur = c;
        n_down = 0;
        left = 1.0;
      } else {
        left -= pc;
        down[n_down++] = c;
      }
    }
    s_cur = cur;
    s_len = len;
    s_down = len < p.max_path ? n_down : 0;
    p.n_path[seq] = len;
  }
  __syncthreads();
  const int cur = s_cur, n_down = s_down;
  const VerifyRow r = p.rows[r0 + cur];
  if (!(r.top > -INFINITY)) return;  // (the token stays -1)
  const char* const x = p.logits + (r0 + cur) * p.nb;
  const char* const q = p.draft && n_down > 0 ? p.draft + (r0 + down[0]) * p.draft_nb : nullptr;
  auto rest = [&](int t) -> double {
    const double w = weight(gload<float>(x + 4 * (int64_t)t), t, r, inv_t);
    if (q) return fmax(w / r.sum - (double)gload<float>(q + 4 * (int64_t)t), 0.0);
    if (!p.draft)
      for (int e = 0; e < n_down; ++e)
        if (token[down[e]] == t) return 0.0;
    return w;
  };
  // A wave's part of the tokens is in one piece.
  const int per = (p.n_vocab + kWaves - 1) / kWaves, t0 = wave * per, t1 = min(t0 + per, p.n_vocab);
  double sum = 0.0;
  int most = -1;  // the last token with a weight
  for (int t = t0 + lane; t < t1; t += kWave) {
    const double w = rest(t);
    sum += w;
    if (w > 0.0) most = t;
  }
  sum = wave_sum_f64(sum);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) most = max(most, __shfl_xor(most, off, kWave));
  if (lane == 0) {
    part[wave] = sum;
    last[wave] = most;
  }
  __syncthreads();
  double total = 0.0, before = 0.0;
  for (int w = 0; w < kWaves; ++w) total += part[w];
  const double target = bar[0] * total;
  int mine = -1;  // the wave that holds the token, or -1: rounding passed the last one
  for (int w = 0; w < kWaves; ++w) {
    if (before + part[w] > target) {
      mine = w;
      break;
    }
    before += part[w];
  }
  if (mine < 0) {
    for (int w = 0; w < kWaves; ++w) mine = last[w] >= 0 ? w : mine;
    if (tid == 0 && mine >= 0) out[s_len - 1] = last[mine];
    return;
  }
  if (wave != mine) return;
  for (int t = t0; t < t1; t += kWave) {
    const double w = t + lane < t1 ? rest(t + lane) : 0.0;
    const double cum = before + wave_scan(w, lane);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(w > 0.0 && cum > target);
    if (hit) {
      if (lane == 0) out[s_len - 1] = t + __builtin_ctzll(hit);
      return;
    }
    before = __shfl(cum, kWave - 1, kWave);
  }
  if (lane == 0) out[s_len - 1] = last[mine];
}

hipError_t launch_verify(const Verify& p, hipStream_t stream) {
  if (p.n_rows > 0) hipLaunchKernelGGL(verify_rows_kernel, dim3((unsigned)p.n_rows), dim3(kRowThreads), 0, stream, p);
  hipLaunchKernelGGL(verify_walk_kernel, dim3((unsigned)p.n_seq), dim3(kWalkThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mi
