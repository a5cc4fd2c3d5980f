// logits.hip -- penalties for repeated tokens, biases and a grammar's mask on
// rows of logits, and the greedy id of each row.
//
// Per row, token t with count c(t) in the row's history:
//   c > 0: y = x > 0 ? x / repeat : x * repeat, then y -= c * frequency + presence
//   y += the sum of t's biases (in the list's order)
//   y = -inf where the mask's bit is clear
// every product, sum and quotient rounded on its own, and id = the lowest t of
// the largest y that is neither -inf nor NaN, -1 if there is none.
//
// A workgroup owns a chunk of one row. It counts the history's tokens that lie
// in its chunk in LDS (whole numbers, so the atomics' order does not show),
// adds up the biases, passes over its logits once and leaves the chunk's best
// as one 64-bit key (value order, then lower token); a second kernel takes
// the row's best. Each logit is read and written once; a row's history is
// read by every chunk of the row, from the caches.
#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kChunk = 4096;
constexpr int kThreads = 256;

// Larger for the larger value, and for the lower token among equal values; 0
// for what is never chosen.
__device__ inline uint64_t key_of(float v, int t) {
  if (!(v > -INFINITY)) return 0ull;
  const unsigned u = __builtin_bit_cast(unsigned, v + 0.f);  // -0 is 0
  const unsigned o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)o << 32 | (unsigned)~t;
}

__device__ inline uint64_t wave_max_u64(uint64_t x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint64_t y = (uint64_t)(unsigned)__shfl_xor((int)(x >> 32), off, kWave) << 32 |
                       (unsigned)__shfl_xor((int)x, off, kWave);
    x = y > x ? y : x;
  }
  return x;
}

}  // namespace

__global__ __launch_bounds__(kThreads) void logits_kernel(const LogitsAdjust p) {
  __shared__ unsigned count[kChunk];
  __shared__ float bias[kChunk];
  __shared__ uint64_t best[kThreads / kWave];
  const int row = blockIdx.y, base = blockIdx.x * kChunk;
  const int n = min(kChunk, p.n_vocab - base);
  const int tid = threadIdx.x, lane = tid % kWave;
  const int h0 = p.hist && p.penalties ? p.hist_off[row] : 0, h1 = p.hist && p.penalties ? p.hist_off[row + 1] : 0;
  const int b0 = p.bias_id ? p.bias_off[row] : 0, b1 = p.bias_id ? p.bias_off[row + 1] : 0;
  const bool counts = h1 > h0, biases = b1 > b0;
  if (counts || biases) {
    for (int i = tid; i < kChunk; i += kThreads) {
      count[i] = 0u;
      bias[i] = 0.f;
    }
    __syncthreads();
    for (int i = h0 + tid; i < h1; i += kThreads) {
      const unsigned at = (unsigned)p.hist[i] - (unsigned)base;
      if (at < (unsigned)n) atomicAdd(&count[at], 1u);
    }
    // One wave adds the biases, lane by lane, so that a token that is listed
    // twice gets the same sum every time.
    if (tid < kWave) {
      for (int i = b0; i < b1; i += kWave) {
        const unsigned at = i + lane < b1 ? (unsigned)p.bias_id[i + lane] - (unsigned)base : ~0u;
        const float v = i + lane < b1 ? p.bias[i + lane] : 0.f;
        uint64_t todo = __builtin_amdgcn_ballot_w64(at < (unsigned)n);
        while (todo) {
          const int who = __builtin_ctzll(todo);
          todo &= todo - 1;
          if (lane == who) bias[at] += v;
          wave_lds_fence();
        }
      }
    }
    __syncthreads();
  }
  const float repeat = p.penalties ? p.penalties[3 * row] : 1.f;
  const float frequency = p.penalties ? p.penalties[3 * row + 1] : 0.f;
  const float presence = p.penalties ? p.penalties[3 * row + 2] : 0.f;
  const char* const in = p.in + row * p.in_nb + 4 * (int64_t)base;
  char* const out = p.out + row * p.out_nb + 4 * (int64_t)base;
  const char* const mask = p.mask ? p.mask + row * p.mask_nb + base / 8 : nullptr;
  const bool vec = ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  uint64_t top = 0ull;
  for (int i = 4 * tid; i < n; i += 4 * kThreads) {
#pragma clang fp contract(off)
    float x[4];
    const int m = min(4, n - i);
    if (vec && m == 4) {
      const f32x4 v = gload<f32x4>(in + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = j < m ? gload<float>(in + 4 * (i + j)) : -INFINITY;
    }
    const unsigned allow = mask ? gload<unsigned>(mask + (i / 32) * 4) >> (i % 32) : ~0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= m) continue;
      if (counts) {
        const unsigned c = count[i + j];
        if (c > 0u) {
          const float y = x[j] > 0.f ? x[j] / repeat : x[j] * repeat;
          x[j] = y - ((float)c * frequency + presence);
        }
      }
      if (biases) x[j] += bias[i + j];
      if (!(allow >> j & 1u)) x[j] = -INFINITY;
      const uint64_t k = key_of(x[j], base + i + j);
      top = k > top ? k : top;
    }
    if (vec && m == 4) {
      gstore(out + 4 * i, f32x4{x[0], x[1], x[2], x[3]});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < m) gstore<float>(out + 4 * (i + j), x[j]);
    }
  }
  if (!p.ids) return;
  top = wave_max_u64(top);
  if (lane == 0) best[tid / kWave] = top;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) top = best[w] > top ? best[w] : top;
    p.part[(int64_t)row * gridDim.x + blockIdx.x] = top;
  }
}

// One wave per row: the best of the row's chunks.
__global__ __launch_bounds__(kWave) void logits_best_kernel(const uint64_t* part, int n_chunks, int32_t* ids) {
  uint64_t top = 0ull;
  for (int i = threadIdx.x; i < n_chunks; i += kWave) {
    const uint64_t k = part[(int64_t)blockIdx.x * n_chunks + i];
    top = k > top ? k : top;
  }
  top = wave_max_u64(top);
  if (threadIdx.x == 0) ids[blockIdx.x] = top ? (int32_t)~(unsigned)top : -1;
}

int logits_chunks(int n_vocab) { return (n_vocab + kChunk - 1) / kChunk; }

hipError_t launch_logits_adjust(const LogitsAdjust& p, hipStream_t stream) {
  const int chunks = logits_chunks(p.n_vocab);
  hipLaunchKernelGGL(logits_kernel, dim3(chunks, p.n_rows), dim3(kThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.ids) return e;
  hipLaunchKernelGGL(logits_best_kernel, dim3(p.n_rows), dim3(kWave), 0, stream, p.part, chunks, p.ids);
  return hipGetLastError();
}

}  // namespace mi
