// paged.hip -- a step's block tables, and the row and position of each token,
// from the requests' lengths.
//
// Sequence i needs need = ceil((cached + new) / page) pages and holds held: it
// takes max(0, need - held) from the ring's head, behind what the sequences
// before it take, or gives max(0, held - need) to its tail. Three running sums
// over the sequences (tokens, pages taken, pages given) say where each one's
// tokens and pages lie. A sequence whose sum of taken pages passes what is free
// is refused, and so are all behind it that take any: the sum only grows, so
// those that are granted lie where their sums say.
//
// The ring is read at [head, head + taken) and written at [tail, tail + given),
// modulo its length: free pages and held pages together are at most its length,
// so the two do not meet.
//
// One workgroup sums over the sequences, then a thread per token looks up its
// sequence. Bound: the latency of that chain.
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

constexpr int kPlanThreads = 1024;

__device__ inline int64_t shfl_up64(int64_t x, int off) {
  return (int64_t)((uint64_t)(unsigned)__shfl_up((int)(x >> 32), off, kWave) << 32 |
                   (unsigned)__shfl_up((int)x, off, kWave));
}
__device__ inline int64_t wave_scan(int64_t x, int lane) {
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int64_t y = shfl_up64(x, off);
    x += lane >= off ? y : 0;
  }
  return x;
}

// The running sum up to and with this thread over the workgroup's threads, and
// the sum over all of them.
__device__ inline int64_t block_scan(int64_t x, int64_t* part, int64_t& all) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  x = wave_scan(x, lane);
  __syncthreads();  // (what was in part has been read)
  if (lane == kWave - 1) part[wave] = x;
  __syncthreads();
  int64_t before = 0;
  all = 0;
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    before += w < wave ? part[w] : 0;
    all += part[w];
  }
  return x + before;
}

}  // namespace

__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(const PageTables p) {
  __shared__ int64_t part[kPlanThreads / kWave];
  __shared__ int refused_all;
  const int tid = threadIdx.x;
  int head = p.ring_at[0] % p.n_pages;
  head += head < 0 ? p.n_pages : 0;
  const int64_t n_free = max((int64_t)0, min((int64_t)p.ring_at[1] - p.ring_at[0], (int64_t)p.n_pages));
  if (tid == 0) refused_all = 0;
  __syncthreads();
  int64_t tokens0 = 0, take0 = 0, give0 = 0, granted = 0;
  for (int base = 0; base < p.n_seq; base += kPlanThreads) {
    const int i = base + tid;
    const bool there = i < p.n_seq;
    const int64_t cached = there ? max(p.n_cached[i], 0) : 0, fresh = there ? max(p.n_new[i], 0) : 0;
    const int held = there ? min(max(p.held[i], 0), p.max_pages) : 0;
    const int64_t need = (cached + fresh + (1 << p.page_shift) - 1) >> p.page_shift;
    int64_t all;
    const int64_t end = tokens0 + block_scan(fresh, part, all);
    tokens0 += all;
    const bool fits = need <= p.max_pages && end <= p.max_tokens;
    int64_t take = fits ? max((int64_t)0, need - held) : 0;
    const int64_t take_end = take0 + block_scan(take, part, all);
    take0 += all;
    const bool refused = !fits || (take > 0 && take_end > n_free);
    if (refused) take = 0;
    const int64_t give = refused ? 0 : max((int64_t)0, held - need);
    const int64_t give_end = give0 + block_scan(give, part, all);
    give0 += all;
    block_scan(take, part, all);
    granted += all;
    if (there) {
      p.q_off[i + 1] = (int)min(end, (int64_t)p.max_tokens);
      p.n_kv[i] = refused ? 0 : (int)min(cached + fresh, (int64_t)INT32_MAX);
      p.held_out[i] = (int)(held + take - give);
      int* const row = reinterpret_cast<int*>(p.table + i * p.table_nb);
      for (int k = 0; k < take; ++k) row[held + k] = p.ring[(head + take_end - take + k) % p.n_pages];
      for (int k = 0; k < give; ++k) p.ring[(head + n_free + give_end - give + k) % p.n_pages] = row[need + k];
      if (refused) atomicAdd(&refused_all, 1);
    }
  }
  __syncthreads();
  if (tid == 0) {
    p.q_off[0] = 0;
    const int64_t h = head + granted, t = head + n_free + give0, laps = h / p.n_pages * p.n_pages;
    p.ring_at_out[0] = (int)(h - laps);
    p.ring_at_out[1] = (int)(t - laps);
    if (p.n_refused) p.n_refused[0] = refused_all;
  }
}

__global__ __launch_bounds__(256) void page_slots_kernel(const PageTables p) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= p.max_tokens) return;
  int slot = -1, pos = 0, seq = -1;
  if (t < p.q_off[p.n_seq]) {
    int lo = 0, hi = p.n_seq - 1;  // the last sequence that begins at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (p.q_off[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    seq = lo;
    pos = max(p.n_cached[seq], 0) + t - p.q_off[seq];
    if (p.n_kv[seq] > 0) {
      const int page = reinterpret_cast<const int*>(p.table + seq * p.table_nb)[pos >> p.page_shift];
      if ((unsigned)page < (unsigned)p.n_pages) slot = (page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    }
  }
  p.slots[t] = slot;
  if (p.pos) p.pos[t] = pos;
  if (p.seq) p.seq[t] = seq;
}

hipError_t launch_page_tables(const PageTables& p, hipStream_t stream) {
  hipLaunchKernelGGL(page_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.max_tokens == 0) return e;
  hipLaunchKernelGGL(page_slots_kernel, dim3((unsigned)((p.max_tokens + 255) / 256)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mi
