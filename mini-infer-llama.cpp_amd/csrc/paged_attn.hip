// paged_attn.hip -- attention of each sequence's new tokens over its pages.
//
// out_j = sum_t p_t v_t / sum_t p_t over the positions t up to the query's own,
// p_t = 2^(s_t - m), s_t = scale log2(e) q_j.k_t, m the maximum so far, position t
// in row table[t / page] page + t % page. A wave takes one query row: a lane's
// key is its own for the scores, its dims are its own for the sums.
#include "attn_common.h"
#include "kernels.h"

namespace mi {

namespace {

// Element d of a row (K: a scale per 32 dims, V: one).
template <typename KT, bool K>
__device__ inline float element(const CacheView& c, int64_t row, int h, int d) {
  const char* const at = c.t[K ? 0 : 1] + row * c.s2 + h * c.s1;
  if constexpr (sizeof(KT) == 1) {
    const int n = K ? c.head_dim / 32 : 1;
    const char* const sc = c.scale[K ? 0 : 1] + ((row * c.n_head_kv + h) * n + (K ? d / 32 : 0)) * 2;
    return (float)gload<int8_t>(at + d) * (float)gload<_Float16>(sc);
  } else {
    return (float)gload<KT>(at + d * (int)sizeof(KT));
  }
}

}  // namespace

template <int D, typename KT>
__global__ __launch_bounds__(kWave) void paged_attn_kernel(const PagedAttn p) {
  __shared__ float qs[D];
  __shared__ float ps[kWave];
  __shared__ int64_t rows[kWave];
  const int lane = threadIdx.x, row = blockIdx.x, h = blockIdx.y, g = h / p.n_rep;
  int seq = 0;  // the last sequence that begins at or before the row
  for (int hi = p.n_seq - 1; seq < hi;) {
    const int mid = (seq + hi + 1) / 2;
    if (p.q_off[mid] <= row) seq = mid;
    else hi = mid - 1;
  }
  const int q0 = min(max(p.q_off[seq], 0), p.n_tokens), q1 = min(max(p.q_off[seq + 1], q0), p.n_tokens);
  if (row < q0 || row >= q1 || row - q0 >= p.max_new) return;
  const int n_kv = min(max(p.n_kv[seq], 0), p.max_kv);
  const int lim = n_kv - (q1 - q0) + (row - q0) + 1;  // positions seen
  const char* const q = p.q + row * p.q_s2 + h * p.q_s1;
  for (int d = lane; d < D; d += kWave) qs[d] = gload<float>(q + 4 * d) * p.scale_log2e;
  __syncthreads();
  const int* const table = reinterpret_cast<const int*>(p.table + seq * p.table_nb);
  float m = -INFINITY, l = 0.f, o[D / kWave];
  for (float& x : o) x = 0.f;
  for (int t0 = 0; t0 < lim; t0 += kWave) {
    const int t = t0 + lane;
    float s = -INFINITY;
    rows[lane] = -1;
    if (t < lim) {
      const int page = table[t >> p.page_shift];
      if ((unsigned)page < (unsigned)p.n_pages) {
        const int64_t r = ((int64_t)page << p.page_shift) + (t & ((1 << p.page_shift) - 1));
        rows[lane] = r;
        s = 0.f;
        for (int d = 0; d < D; ++d) s = fmaf(element<KT, true>(p.cache, r, g, d), qs[d], s);
      } else {
        s = NAN;
      }
    }
    float top = s;
    bool bad = __builtin_amdgcn_ballot_w64(s != s) != 0ull;
    top = wave_max(top);
    const float now = fmaxf(m, top);
    const float at = now == -INFINITY ? 0.f : now;
    const float alpha = fast_exp2(m - at), e = fast_exp2(s - at);
    m = now;
    l = bad ? NAN : l * alpha + wave_sum(e);
    ps[lane] = e;
    __syncthreads();
    for (float& x : o) x *= alpha;
    for (int j = 0; j < kWave && t0 + j < lim; ++j)
      if (rows[j] >= 0)
        for (int i = 0; i < D / kWave; ++i) o[i] = fmaf(ps[j], element<KT, false>(p.cache, rows[j], g, lane + kWave * i), o[i]);
    __syncthreads();
  }
  const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
  char* const out = p.out + row * p.o_s2 + h * p.o_s1;
  for (int i = 0; i < D / kWave; ++i) gstore<float>(out + 4 * (lane + kWave * i), o[i] * inv);
}

template <int D>
static void launch_d(const PagedAttn& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.n_tokens, (unsigned)(p.n_rep * p.cache.n_head_kv));
  if (p.cache.elt == 1) hipLaunchKernelGGL((paged_attn_kernel<D, int8_t>), grid, dim3(kWave), 0, stream, p);
  else if (p.cache.elt == 2) hipLaunchKernelGGL((paged_attn_kernel<D, _Float16>), grid, dim3(kWave), 0, stream, p);
  else hipLaunchKernelGGL((paged_attn_kernel<D, float>), grid, dim3(kWave), 0, stream, p);
}

hipError_t launch_paged_attn(const PagedAttn& p, hipStream_t stream) {
  if (p.cache.head_dim == 64) launch_d<64>(p, stream);
  else launch_d<128>(p, stream);
  return hipGetLastError();
}

}  // namespace mi
