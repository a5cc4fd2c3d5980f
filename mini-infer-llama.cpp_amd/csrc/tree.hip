// tree.hip -- attention of several query tokens per sequence over a KV cache
// whose last n_tokens rows are those tokens' own (a tree of drafted tokens
// with a visibility mask, a causal chunk, or one token), F32, F16 or 8-bit
// cache, several sequences in one launch.
//
// Mathematics. Query j of a sequence sees key t when t < n_past, or when bit
// t - n_past of its mask row is set (no mask: t - n_past <= j). Its output is
// sum_t p_t v_t / sum_t p_t with p_t = 2^(s_t - m), s_t = scale log2(e) q.k_t
// and m near the maximum over the keys seen so far, so the keys pass once;
// when m moves, what has been summed is rescaled by 2^(m_old - m_new). A row
// that sees no key has m = -inf and an output of zeros.
//
// Decomposition. The n_tokens * n_rep query rows that read one KV head are
// cut into row tiles (row r is token r / n_rep, head r % n_rep of the group),
// the keys into splits of whole 32-key tiles. A workgroup owns (item, KV head,
// row tile, split). With one split its result is the output, otherwise it is a
// record in the workspace that tree_combine_kernel joins: a second launch, 4 to 6
// us of a split call. (Joined by a group's last workgroup instead, whose records
// come from other XCDs, one token over 4000 keys of 64 took 20.5 us, not 11.3. A join
// by all workgroups of the launch, as in decode.hip, has not been tried here.)
//
// This kernel: one tile of 16 or 32 rows, for calls that need no more. Its waves
// take the split's key tiles in turn, K and V straight to registers, and meet in
// LDS at the end. (More rows: tree_wide.hip.)
//
// Per key tile of 32 (lane = (c = lane % 16, q = lane / 16)), 16x16 MFMAs:
//   S^T = K . Q^T: A is K (key c), B the queries (row c); a lane ends up with
//   keys 4 q + j and 16 + 4 q + j (j < 4) of row c, so the softmax runs within
//   lanes but for an exchange between the four lanes of a row, and P is already
//   the B operand of O^T += V^T . P^T. V's A operand is loaded as rows: a lane
//   takes the NE = D / 16 consecutive dims NE c .. of its eight keys, so row c of
//   output block db is dim NE c + db.
// (The wide kernel does the same with 32x32 MFMAs: lane = (c = lane % 32, kh =
// lane / 32), a lane has the 16 keys 8 (i / 4) + 4 kh + i % 4 of row c.)
//
// Products. F32 cache: v_mfma_f32_16x16x4f32. F16 and 8-bit caches: the cache
// operand is exact in f16, the queries and the probabilities are f16 pairs
// hi = RNE(x), lo = RNE(x - hi), two v_mfma_f32_16x16x32_f16 a step. So that
// lo stays normal, each query row is scaled by the power of two that puts its
// largest element in [2^13, 2^14) (undone in the exponent's multiply-add), and
// the probabilities are 2^(s - ref) for a reference that keeps the largest
// between 2^6 and 2^14 (move_ref; the division by their sum undoes it; with an
// F32 cache 2^-14 times that, since its values may be of any size): 2^-22
// relative to the row's largest element.
//   8-bit K: a row's scales (one per 32 dims) multiply the S^T of their own
//   32 dims. 8-bit V: the row's one scale multiplies the probability; ref keeps
//   the largest such product in that range.
//
// Bound: F16, memory, each byte of the cache once: 24 sequences of one token over
// 2788 to 4096 keys (28/4 heads of 128, 170 MB) at 5.1 TB/s, 32.5 us with the join.
// 8-bit caches are half the bytes and no faster: the same call 36.3 us, since four
// values take about five instructions to widen, for 7 rows of 16 that are there; with
// 14/2 heads of 64 14.4 us, F16 14.1: a row of 64 bytes is half a line, the other KV
// head's half is fetched by another XCD (40 MB for the cache's 22). Over few keys the
// start, a tile's chain of loads, products and exponentials and the join's launch (one
// token over 4000: 10.6 us). Rows beyond the group's are work for nothing: with 32x32
// MFMAs, whose tile is 32 rows, the F16 call of 128 dims took 57 us, and twice the
// registers let one workgroup less onto a CU.
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"
#include "tree_rows.h"

namespace mi {

namespace {

constexpr int kTreeRows = 32;  // rows of this kernel's records

// One (KV head, split) of an item, for tree_rows.
template <int D, typename KT>
struct TreeWork {
  static constexpr int ELT = (int)sizeof(KT);
  const TreeParams& p;
  const TreeItem& it;
  int g, n_past, n_kv, rows, n_rep, tile0, tile1, k_s2, v_s2;
  float scale_log2e;
  const char* kbase;
  const char* vbase;
  float* rec;

  __device__ __forceinline__ int thread() const { return (int)threadIdx.x; }
  __device__ __forceinline__ void at_tile(int) {}
  __device__ __forceinline__ unsigned none() const { return 0u; }
  // The descriptors start at the tile's first row (64-bit), so a cache of any
  // length is addressed, and end after its last valid row.
  __device__ __forceinline__ TileRows rows_at(const char* base, int s2, int key0) const {
    const int n = min(n_kv - key0, kTreeTile);
    const rsrc_t r = make_rsrc(base + (int64_t)key0 * s2, (unsigned)((n - 1) * s2 + D * ELT));
    return TileRows{{r, r}, {0u, (unsigned)(16 * s2)}};
  }
  __device__ __forceinline__ TileRows k_rows(int key0) const { return rows_at(kbase, k_s2, key0); }
  __device__ __forceinline__ TileRows v_rows(int key0) const { return rows_at(vbase, v_s2, key0); }
  template <int NB>
  __device__ __forceinline__ void scales(int key0, int c32, int half, unsigned& ksc, unsigned& vsc) const {
    const int n = min(n_kv - key0, kTreeTile);
    const int64_t at = (int64_t)key0 * p.n_head_kv + g;
    const rsrc_t rk = make_rsrc(it.k_scale + at * (2 * NB), (unsigned)((n - 1) * p.n_head_kv * 2 * NB + 2 * NB));
    ksc = NB == 4 ? buf_b32(rk, (unsigned)(c32 * p.n_head_kv * 8 + 4 * half)) : buf_b16(rk, (unsigned)(c32 * p.n_head_kv * 4 + 2 * half));
    const rsrc_t rv = make_rsrc(it.v_scale + at * 2, (unsigned)((n - 1) * p.n_head_kv * 2 + 2));
    vsc = buf_b16(rv, (unsigned)(c32 * p.n_head_kv * 2));
  }
  __device__ __forceinline__ unsigned visible(int token, int key0) const { return visible_bits(it, token, key0); }
  __device__ __forceinline__ const char* q_row(int token, int h) const {
    return reinterpret_cast<const char*>(it.q) + (int64_t)token * p.q_s2 + (int64_t)(g * p.n_rep + h) * p.q_s1;
  }
  __device__ __forceinline__ char* out_row(int token, int h) const {
    return reinterpret_cast<char*>(it.out) + (int64_t)token * p.o_s2 + (int64_t)(g * p.n_rep + h) * p.o_s1;
  }
  __device__ __forceinline__ bool is_part() const { return it.n_split > 1; }
  __device__ __forceinline__ void put_sums(int r, float ref, float l) const {
    rec[kTreeRows * D + r] = ref;
    rec[kTreeRows * D + kTreeRows + r] = l;
  }
  __device__ __forceinline__ void put_part(int r, int d, f32x4 x) const { put_record(rec + tree_record_at(D, r, d), x); }
};

}  // namespace

template <int D, typename KT, int RT>
__global__ __launch_bounds__(kTreeWaves* kWave, (TreeCfg<D, KT, RT>::WAVES_PER_SIMD)) void tree_kernel(const TreeParams p) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  // Workgroup -> (KV head, split) unit; units go to the 8 XCDs in turn. (One row
  // tile: calls of more rows take the wide kernel.)
  const TreeItem& it = p.item[blockIdx.y];
  const int n_split = it.n_split;
  const int unit = (blockIdx.x / 8) * 8 + (int)((blockIdx.x - it.xcd0) % 8);
  if (unit >= p.n_head_kv * n_split) return;
  const int g = unit / n_split, sp = unit % n_split;
  const int n_past = it.n_past, n_kv = n_past + it.n_tokens;
  const int tile0 = sp * it.tiles_per_split;
  const int tile1 = min(tile0 + it.tiles_per_split, (n_kv + kTreeTile - 1) / kTreeTile);
  TreeWork<D, KT> w{p, it, g, n_past, n_kv, it.n_tokens * p.n_rep, p.n_rep, tile0, tile1, (int)p.k_s2, (int)p.v_s2, p.scale_log2e,
                    it.k + (int64_t)g * p.k_s1, it.v + (int64_t)g * p.v_s1,
                    p.rec + ((int64_t)it.rec0 + (int64_t)g * n_split + sp) * (kTreeRows * (D + 2))};
  tree_rows<D, KT, RT>(w, (lds_t*)lds_raw);
}

// Joins the splits' records: out = sum_s 2^(ref_s - M) O_s / sum_s 2^(ref_s - M)
// l_s. A wave takes 1 KB of the records, eight dims of 32 rows (lane: row lane %
// 32, dims 4 (lane / 32) ..), `slices` waves every slices-th record each with a
// running maximum, kInFlight of them on their way at once; the slices meet in
// LDS in order. The records were just written and come from the caches, so the
// time is their latency: few records in turn per wave is what counts.
constexpr int kJoinInFlight = 8, kJoinSlices = 16;

template <int D>
__global__ __launch_bounds__(kJoinSlices* kWave) void tree_combine_kernel(const TreeParams p, int tile_rows, int slices) {
  constexpr int kInFlight = kJoinInFlight;
  __shared__ f32x4 part[kJoinSlices][kWave];
  __shared__ f32x2 ml[kJoinSlices][kWave];
  const TreeItem& it = p.item[blockIdx.y];
  const int rows = it.n_tokens * p.n_rep, n_split = it.n_split;
  if (n_split <= 1) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int slice = wave % slices;
  const int groups = (rows + 31) / 32;  // of 32 rows, per KV head
  const int unit = blockIdx.x * ((int)blockDim.x / kWave / slices) + wave / slices;
  const int chunk = unit % (D / 8), grp = unit / (D / 8) % groups, g = unit / (D / 8) / groups;
  const bool valid = g < p.n_head_kv;
  const int64_t rec_floats = (int64_t)tile_rows * (D + 2);
  const int rt = grp * 32 / tile_rows, rr = grp * 32 % tile_rows;
  const float* const rec =
      p.rec + ((int64_t)it.rec0 + (int64_t)((valid ? g : 0) * it.n_rt + rt) * n_split) * rec_floats;
  const int o_at = rr * D + chunk * 256 + lane * 4, m_at = tile_rows * D + rr + lane % 32, l_at = m_at + tile_rows;
  float mx = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = slice; s0 < n_split; s0 += kInFlight * slices) {
    float ms[kInFlight], ls[kInFlight];
    f32x4 os[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int s = s0 + u * slices;
      const float* const q = rec + (s < n_split ? s : s0) * rec_floats;
      ms[u] = gload<float>(q + m_at);
      ls[u] = gload<float>(q + l_at);
      os[u] = gload<f32x4>(q + o_at);
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      if (s0 + u * slices >= n_split) continue;
      const float mn = fmaxf(mx, ms[u]);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float a = fast_exp2(mx - mu), b = fast_exp2(ms[u] - mu);
      // (a split without a key for the row may have left its sums unwritten)
      acc = acc * a + (ms[u] == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : os[u] * b);
      l = l * a + ls[u] * b;
      mx = mn;
    }
  }
  if (slices > 1) {
    part[wave][lane] = acc;
    ml[wave][lane] = f32x2{mx, l};
    __syncthreads();
    if (slice != 0) return;
    float top = mx;
    for (int s = 1; s < slices; ++s) top = fmaxf(top, ml[wave + s][lane][0]);
    const float mu = top == -INFINITY ? 0.f : top;
    const float a = fast_exp2(mx - mu);
    acc *= a;
    l *= a;
    for (int s = 1; s < slices; ++s) {
      const float b = fast_exp2(ml[wave + s][lane][0] - mu);
      acc += part[wave + s][lane] * b;
      l += ml[wave + s][lane][1] * b;
    }
    mx = top;
  }
  const int r = grp * 32 + lane % 32;
  if (!valid || r >= rows) return;
  // (no key at all: zeros; every score NaN: the sum is)
  const float inv = mx == -INFINITY && l == 0.f ? 0.f : 1.f / l;
  const int t = r / p.n_rep, h = g * p.n_rep + r % p.n_rep;
  gstore(reinterpret_cast<char*>(it.out) + (int64_t)t * p.o_s2 + (int64_t)h * p.o_s1 + 32 * chunk + 16 * (lane / 32),
         acc * inv);
}

// The kernel that streams keys to registers for up to 32 rows, else the wide
// kernel (tree_wide.hip), whose waves without rows only fetch. Eight times 28 rows
// over 4000 8-bit keys of 128 (us): 20.9, wide 32.6; F16 keys of 64 12.2, 13.6.
int tree_tile_rows(int rows) { return rows <= 32 ? 32 : 128; }

size_t tree_record_floats(int head_dim, int tile_rows) { return (size_t)tile_rows * (head_dim + 2); }

template <int D, typename KT, int RT>
static hipError_t launch_narrow_t(const TreeParams& p, dim3 grid, hipStream_t stream) {
  typedef TreeCfg<D, KT, RT> C;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&tree_kernel<D, KT, RT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((tree_kernel<D, KT, RT>), grid, dim3(kTreeWaves * kWave), C::LDS, stream, p);
  return hipGetLastError();
}

// 16 rows where they are enough: half the products and vector instructions. 24
// times 14 rows over 3000 8-bit keys of 64 (us): 14.6, with two tiles 19.2.
template <int D>
static hipError_t launch_narrow(const TreeParams& p, dim3 grid, int elt, bool two, hipStream_t stream) {
  if (elt == 1) return two ? launch_narrow_t<D, int8_t, 2>(p, grid, stream) : launch_narrow_t<D, int8_t, 1>(p, grid, stream);
  if (elt == 2) return two ? launch_narrow_t<D, _Float16, 2>(p, grid, stream) : launch_narrow_t<D, _Float16, 1>(p, grid, stream);
  return two ? launch_narrow_t<D, float, 2>(p, grid, stream) : launch_narrow_t<D, float, 1>(p, grid, stream);
}

hipError_t launch_tree(const TreeParams& p, int n_items, int head_dim, int elt, int tile_rows, hipStream_t stream) {
  unsigned gx = 0;
  int64_t units = 0;  // waves' worth of records to join, of the largest item
  int splits = 1, most = 0;
  for (int i = 0; i < n_items; ++i) {
    const TreeItem& it = p.item[i];
    most = std::max(most, it.n_tokens * p.n_rep);
    gx = std::max(gx, (((unsigned)p.n_head_kv * it.n_split << p.row_shift) + 7) / 8 * 8 * (unsigned)it.unit_rt);
    if (it.n_split > 1)
      units = std::max(units, ((int64_t)it.n_tokens * p.n_rep + 31) / 32 * p.n_head_kv * (head_dim / 8));
    splits = std::max(splits, it.n_split);
  }
  const dim3 grid(gx, n_items);
  const hipError_t e = tile_rows == 128  ? launch_tree_wide(p, grid, head_dim, elt, stream)
                       : head_dim == 64 ? launch_narrow<64>(p, grid, elt, most > 16, stream)
                                        : launch_narrow<128>(p, grid, elt, most > 16, stream);
  if (e != hipSuccess || units == 0) return e;
  // slices: one batch of records in flight each, as far as a workgroup goes
  int slices = 1;
  while (slices < kJoinSlices && slices * kJoinInFlight < splits) slices *= 2;
  const int waves = std::max(4, slices);
  const dim3 cgrid((unsigned)((units * slices + waves - 1) / waves), n_items);
  if (head_dim == 64) hipLaunchKernelGGL(tree_combine_kernel<64>, cgrid, dim3(waves * kWave), 0, stream, p, tile_rows, slices);
  else hipLaunchKernelGGL(tree_combine_kernel<128>, cgrid, dim3(waves * kWave), 0, stream, p, tile_rows, slices);
  return hipGetLastError();
}

}  // namespace mi
