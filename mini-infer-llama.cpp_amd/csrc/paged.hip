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
// so the two do not meet. A token's page is read from the table if its sequence
// held it, else from the ring, never from an entry that this call writes.
//
// So workgroups need nothing of each other: each forms the sums of 1024 sequences
// at a time by itself, into LDS, and takes its share of their pages and tokens, a
// thread for each, whose sequence it finds there. (Lengths that are also written
// cannot be read by several workgroups: held or ring_at in place, one does it all, 1024
// requests with 38000 tokens in 40 us instead of 7.)
// Bound: the chain of two loads (lengths, then pages) and the launch (8 requests 6.4 us,
// 1024 requests with 37000 tokens 8.6, an empty launch 3.6).
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

constexpr int kSeqs = 1024, kWaves = kSeqs / kWave;  // sequences at a time, a thread each

__device__ inline unsigned add_sat(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }

// x plus those of the lanes below, up to 2^32 - 1.
__device__ inline unsigned wave_scan_sat(unsigned x) {
#define MI_SCAN_STEP(ctrl, rows) x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false))
  MI_SCAN_STEP(0x111, 0xf);  // row_shr:1
  MI_SCAN_STEP(0x112, 0xf);
  MI_SCAN_STEP(0x114, 0xf);
  MI_SCAN_STEP(0x118, 0xf);
  MI_SCAN_STEP(0x142, 0xa);  // row_bcast:15 to rows 1 and 3
  MI_SCAN_STEP(0x143, 0xc);  // row_bcast:31 to rows 2 and 3
#undef MI_SCAN_STEP
  return x;
}

struct Shared {
  unsigned q_end[kSeqs], take_end[kSeqs], give_end[kSeqs];  // running sums with this sequence
  int cached[kSeqs], fresh[kSeqs], held[kSeqs], need[kSeqs];
  bool refused[kSeqs];
  unsigned part[3][kWaves];
  unsigned n_refused, granted;
};

// The first of n running sums that is above x (n - 1 if none is).
__device__ inline int find(const unsigned* end, int n, unsigned x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (end[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

}  // namespace

__global__ __launch_bounds__(kSeqs) void page_tables_kernel(const PageTables p) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const unsigned n_pages = (unsigned)p.n_pages;
  // Of the pages and the tokens, in 64 bits: the running sums may be any 32 bits, and a
  // start that wrapped would fall on what belongs to the sequences before.
  const uint64_t at = blockIdx.x * kSeqs + tid, step = gridDim.x * kSeqs;
  const bool writes = blockIdx.x == 0;
  const int head0 = p.ring_at[0], tail0 = p.ring_at[1];
  unsigned tokens = 0, taken = 0, given = 0, granted = 0;  // before the sequences at hand
  unsigned head = 0, n_free = 0;
  if (tid == 0) s.n_refused = s.granted = 0;
  for (int first = 0; first < p.n_seq; first += kSeqs) {
    const int i = first + tid, n = min(kSeqs, p.n_seq - first);
    const bool there = tid < n;
    const int cached = there ? max(p.n_cached[i], 0) : 0, fresh = there ? max(p.n_new[i], 0) : 0;
    const int held = there ? min(max(p.held[i], 0), p.max_pages) : 0;
    if (first == 0) {
      const int h = head0 % p.n_pages;
      head = (unsigned)(h < 0 ? h + p.n_pages : h);
      n_free = (unsigned)max((int64_t)0, min((int64_t)tail0 - head0, (int64_t)p.n_pages));
    }
    const unsigned need = (unsigned)(((uint64_t)cached + (uint64_t)fresh + (1u << p.page_shift) - 1u) >> p.page_shift);
    bool fits = need <= (unsigned)p.max_pages;
    unsigned take = fits && need > (unsigned)held ? need - held : 0u, give = need < (unsigned)held ? held - need : 0u;
    unsigned end[3];
    auto sums = [&]() __attribute__((always_inline)) {
      const unsigned x[3] = {wave_scan_sat((unsigned)fresh), wave_scan_sat(take), wave_scan_sat(give)};
      __syncthreads();  // (the part sums, and the sequences before, have been read)
      if (lane == kWave - 1) {
        for (int k = 0; k < 3; ++k) s.part[k][wave] = x[k];
      }
      __syncthreads();
      // lane w of each wave has wave w's part
      for (int k = 0; k < 3; ++k) {
        const unsigned below = wave_scan_sat(lane < kWaves ? s.part[k][lane] : 0u);
        const unsigned upto = (unsigned)__shfl((int)below, max(wave - 1, 0), kWave);
        end[k] = add_sat(x[k], wave == 0 ? 0u : upto);
      }
    };
    sums();
    const unsigned most = (unsigned)p.max_tokens;
    // Tokens that do not fit refuse their sequences, which then take and give nothing.
    if (__syncthreads_or(add_sat(tokens, end[0]) > most)) {
      if (add_sat(tokens, end[0]) > most) {
        fits = false;
        take = give = 0u;
      }
      sums();
    }
    end[0] = add_sat(tokens, end[0]);
    end[1] = add_sat(taken, end[1]);
    end[2] = add_sat(given, end[2]);
    const bool refused = !fits || (take > 0u && end[1] > n_free);
    s.q_end[tid] = end[0];
    s.take_end[tid] = end[1];
    s.give_end[tid] = end[2];
    s.cached[tid] = cached;
    s.fresh[tid] = fresh;
    s.held[tid] = held;
    s.need[tid] = (int)need;
    s.refused[tid] = refused;
    const uint64_t no = __builtin_amdgcn_ballot_w64(there && refused);
    if (lane == 0 && no) atomicAdd(&s.n_refused, (unsigned)__builtin_popcountll(no));
    // (granted sums only grow: the last one is the largest)
    const uint64_t yes = __builtin_amdgcn_ballot_w64(there && !refused && take > 0u);
    if (yes && lane == 63 - __builtin_clzll(yes)) atomicMax(&s.granted, end[1]);
    if (writes && there) {
      p.q_off[i + 1] = (int)min(end[0], most);
      p.n_kv[i] = refused ? 0 : (int)min((unsigned)cached + (unsigned)fresh, (unsigned)INT32_MAX);
      p.held_out[i] = refused ? held : (int)need;
    }
    __syncthreads();
    granted = s.granted;
    // Pages taken by these sequences: page k of the ring's.
    for (uint64_t k64 = taken + at; k64 < granted; k64 += step) {
      const unsigned k = (unsigned)k64;
      const int q = find(s.take_end, n, k);
      int* const row = reinterpret_cast<int*>(p.table + (int64_t)(first + q) * p.table_nb);
      row[s.need[q] - (int)(s.take_end[q] - k)] = p.ring[(head + k) % n_pages];
    }
    // Pages given back.
    const unsigned given_end = s.give_end[kSeqs - 1];
    for (uint64_t k64 = given + at; k64 < given_end; k64 += step) {
      const unsigned k = (unsigned)k64;
      const int q = find(s.give_end, n, k);
      const int* const row = reinterpret_cast<const int*>(p.table + (int64_t)(first + q) * p.table_nb);
      p.ring[(head + n_free + k) % n_pages] = row[s.held[q] - (int)(s.give_end[q] - k)];
    }
    // Tokens.
    const unsigned q_end = min(s.q_end[kSeqs - 1], most);
    for (uint64_t t64 = tokens + at; t64 < q_end; t64 += step) {
      const unsigned t = (unsigned)t64;
      const int q = find(s.q_end, n, t);
      const int pos = (int)((unsigned)s.cached[q] + (t - (s.q_end[q] - (unsigned)s.fresh[q])));
      int slot = -1;
      if (!s.refused[q]) {
        const int k = pos >> p.page_shift, held_q = s.held[q];
        const unsigned from = s.take_end[q] - (unsigned)max(s.need[q] - held_q, 0);  // its first page in the ring
        const int page = k < held_q ? reinterpret_cast<const int*>(p.table + (int64_t)(first + q) * p.table_nb)[k]
                                    : p.ring[(head + from + (unsigned)(k - held_q)) % n_pages];
        if ((unsigned)page < n_pages) slot = (page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
      }
      p.slots[t] = slot;
      if (p.pos) p.pos[t] = pos;
      if (p.seq) p.seq[t] = first + q;
    }
    tokens = s.q_end[kSeqs - 1];
    taken = s.take_end[kSeqs - 1];
    given = given_end;
  }
  if (p.n_seq == 0) {
    const int h = head0 % p.n_pages;
    head = (unsigned)(h < 0 ? h + p.n_pages : h);
    n_free = (unsigned)max((int64_t)0, min((int64_t)tail0 - head0, (int64_t)p.n_pages));
  }
  // The batch's padding.
  for (uint64_t t = min(tokens, (unsigned)p.max_tokens) + at; t < (unsigned)p.max_tokens; t += step) {
    p.slots[t] = -1;
    if (p.pos) p.pos[t] = 0;
    if (p.seq) p.seq[t] = -1;
  }
  if (writes && tid == 0) {
    p.q_off[0] = 0;
    const unsigned h = head + granted, t = head + n_free + given, laps = h / n_pages * n_pages;
    p.ring_at_out[0] = (int)(h - laps);
    p.ring_at_out[1] = (int)(t - laps);
    if (p.n_refused) p.n_refused[0] = (int)s.n_refused;
  }
}

hipError_t launch_page_tables(const PageTables& p, int n_cu, hipStream_t stream) {
  // Two tokens a thread; one workgroup where what it reads is written.
  const bool in_place = p.held == p.held_out || p.ring_at == p.ring_at_out;
  const int n_wg = in_place ? 1 : std::max(1, std::min(n_cu, p.max_tokens / (2 * kSeqs)));
  hipLaunchKernelGGL(page_tables_kernel, dim3((unsigned)n_wg), dim3(kSeqs), 0, stream, p);
  return hipGetLastError();
}

}  // namespace mi
