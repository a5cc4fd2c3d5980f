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
// A workgroup owns a chunk of one row. Its logits are on their way while it
// counts the history's tokens that lie in the chunk in LDS (whole numbers, so the
// atomics' order does not show) and one wave adds up the biases; then each logit
// is finished, stored, and the chunk's best kept as one 64-bit key (value order,
// then lower token); the row's last workgroup takes the best of those. Each logit
// is read and written once; a row's history is read by every chunk of the row, from
// the caches. Bound: memory for many rows, the chain of dependent loads (offsets,
// history, LDS) for few; there the chunks are smaller, so that more workgroups
// share a row.
#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Chunks of 2048 logits; of 4096 and 512 threads where rows have histories, which
// every chunk reads (64 rows of 151936 with histories, biases and a mask 24.9 us,
// by 2048 26.5; 48 rows without lists 12.7, by 2048 11.3); of 1024 while a launch
// has at most four of them per CU (in a graph, one row of 32000 5.5 us, by 2048
// 6.4, 16 rows 6.1 and 6.9; of 151936 7.1 and 8.6 either way, where more workgroups
// take longer to be counted).
constexpr int64_t kFewPerCu = 4;

// A row may start at any multiple of 4 bytes (an odd vocabulary); loads and stores
// of four take that as they are.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
__device__ inline f32x4 load4(const char* p) { return *(const __attribute__((address_space(1))) f32x4_any*)p; }
// (The logits are not read again here: nontemporal, so that a launch does not end
// by writing its XCDs' L2s back. 48 rows of 151936: 11.7 us instead of 14.9.)
__device__ inline void store4(char* p, f32x4 v) {
  __builtin_nontemporal_store((f32x4_any)v, (__attribute__((address_space(1))) f32x4_any*)p);
}

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

template <int CHUNK, int THREADS>
__global__ __launch_bounds__(THREADS) void logits_kernel(const LogitsAdjust p) {
  constexpr int PER = CHUNK / (4 * THREADS);  // groups of four logits per thread
  constexpr int kInFlight = 8;                 // history ids per thread
  __shared__ __attribute__((aligned(16))) unsigned count[CHUNK];
  __shared__ __attribute__((aligned(16))) float bias[CHUNK];
  __shared__ uint64_t best[THREADS / kWave];
  const int row = blockIdx.y, base = blockIdx.x * CHUNK;
  const int n = min(CHUNK, p.n_vocab - base);
  const int tid = threadIdx.x, lane = tid % kWave;
  const int h0 = p.hist ? p.hist_off[row] : 0, h1 = p.hist ? p.hist_off[row + 1] : 0;
  const int b0 = p.bias_id ? p.bias_off[row] : 0, b1 = p.bias_id ? p.bias_off[row + 1] : 0;
  const bool counts = h1 > h0, biases = b1 > b0;
  const char* const in = p.in + row * p.in_nb + 4 * (int64_t)base;
  char* const out = p.out + row * p.out_nb + 4 * (int64_t)base;
  const char* const mask = p.mask ? p.mask + row * p.mask_nb + base / 8 : nullptr;

  // The lists' first loads, then the logits': loads come back in order, and the
  // lists are worked on while the logits are on their way.
  unsigned at[kInFlight], bat = ~0u;
  float bval = 0.f;
  auto read_hist = [&](int i) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kInFlight; ++u)
      at[u] = i + u * THREADS < h1 ? (unsigned)p.hist[i + u * THREADS] - (unsigned)base : ~0u;
  };
  auto read_bias = [&](int i) __attribute__((always_inline)) {
    bat = i < b1 ? (unsigned)p.bias_id[i] - (unsigned)base : ~0u;
    bval = i < b1 ? p.bias[i] : 0.f;
  };
  if (counts) read_hist(h0 + tid);
  if (biases && tid < kWave) read_bias(b0 + lane);

  // Group k of thread tid: logits 4 (tid + THREADS k) .. of the chunk.
  float x[PER][4];
  unsigned allow[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = 4 * (tid + THREADS * k);
    allow[k] = ~0u;
    if (i + 4 <= n) {
      const f32x4 v = load4(in + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[k][j] = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[k][j] = i + j < n ? gload<float>(in + 4 * (i + j)) : -INFINITY;
    }
    if (mask && i < n) allow[k] = gload<unsigned>(mask + (i / 32) * 4) >> (i % 32);
  }
  if (counts || biases) {
    for (int i = 4 * tid; i < CHUNK; i += 4 * THREADS) {
      *reinterpret_cast<f32x4*>(count + i) = f32x4{0.f, 0.f, 0.f, 0.f};
      *reinterpret_cast<f32x4*>(bias + i) = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
    for (int i = h0 + tid; i < h1;) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
        if (at[u] < (unsigned)n) atomicAdd(&count[at[u]], 1u);
      i += kInFlight * THREADS;
      if (i < h1) read_hist(i);
    }
    // One wave adds the biases, lane by lane, so that a token that is listed
    // twice gets the same sum every time.
    if (tid < kWave) {
      for (int i = b0; i < b1;) {
        uint64_t todo = __builtin_amdgcn_ballot_w64(bat < (unsigned)n);
        while (todo) {
          const int who = __builtin_ctzll(todo);
          todo &= todo - 1;
          if (lane == who) bias[bat] += bval;
          wave_lds_fence();
        }
        i += kWave;
        if (i < b1) read_bias(i + lane);
      }
    }
    __syncthreads();
  }
  const float repeat = counts ? p.penalties[3 * row] : 1.f;
  const float frequency = counts ? p.penalties[3 * row + 1] : 0.f;
  const float presence = counts ? p.penalties[3 * row + 2] : 0.f;
  uint64_t top = 0ull;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
#pragma clang fp contract(off)
    const int i = 4 * (tid + THREADS * k);
    if (i >= n) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float y = x[k][j];
      if (counts) {
        const unsigned c = count[i + j];
        if (c > 0u) y = (y > 0.f ? y / repeat : y * repeat) - ((float)c * frequency + presence);
      }
      if (biases) y += bias[i + j];
      if (!(allow[k] >> j & 1u)) y = -INFINITY;
      x[k][j] = y;
      if (i + j < n) {
        const uint64_t key = key_of(y, base + i + j);
        top = key > top ? key : top;
      }
    }
    if (i + 4 <= n) {
      store4(out + 4 * i, f32x4{x[k][0], x[k][1], x[k][2], x[k][3]});
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) gstore<float>(out + 4 * (i + j), x[k][j]);
    }
  }
  if (!p.ids) return;
  top = wave_max_u64(top);
  if (lane == 0) best[tid / kWave] = top;
  __syncthreads();
  // The last workgroup of the row to get here takes the best of its chunks, whose
  // keys are in memory before they are counted: agent-scope stores go through the
  // L2, and the wave waits for its own. (With a second launch for this, us a call:
  // one row of 151936 10.1 instead of 7.9, 48 rows 11.7 instead of 11.1; in a graph
  // 6.2 instead of 7.1, one row of 32000 5.6 instead of 5.5.)
  if (tid >= kWave) return;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) top = best[w] > top ? best[w] : top;
  uint64_t* const part = p.part + (int64_t)row * gridDim.x;
  unsigned before = 0;
  if (lane == 0) {
    __hip_atomic_store(part + blockIdx.x, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wait_vmem<0>();
    before = __hip_atomic_fetch_add(p.arrived + kArrivalWords * row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (__builtin_amdgcn_readfirstlane((int)before) != (int)gridDim.x - 1) return;
  top = 0ull;
  for (int i = lane; i < (int)gridDim.x; i += kWave) {
    const uint64_t k = __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    top = k > top ? k : top;
  }
  top = wave_max_u64(top);
  if (lane == 0) {
    p.ids[row] = top ? (int32_t)~(unsigned)top : -1;
    __hip_atomic_store(p.arrived + kArrivalWords * row, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

int logits_chunks(int n_vocab) { return (n_vocab + 1023) / 1024; }

template <int CHUNK, int THREADS>
static hipError_t launch_logits(const LogitsAdjust& p, hipStream_t stream) {
  const dim3 grid((unsigned)((p.n_vocab + CHUNK - 1) / CHUNK), (unsigned)p.n_rows);
  hipLaunchKernelGGL((logits_kernel<CHUNK, THREADS>), grid, dim3(THREADS), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_logits_adjust(const LogitsAdjust& p, int n_cu, hipStream_t stream) {
  if ((int64_t)logits_chunks(p.n_vocab) * p.n_rows <= kFewPerCu * n_cu) return launch_logits<1024, 256>(p, stream);
  return p.hist ? launch_logits<4096, 512>(p, stream) : launch_logits<2048, 256>(p, stream);
}

}  // namespace mi
