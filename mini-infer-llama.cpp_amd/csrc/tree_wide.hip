// tree_wide.hip -- tree attention (tree.hip has the mathematics, the layout of
// the products and of the records) for more than 32 query rows per KV head.
//
// With many rows the products bound the work, so a key tile is fetched and
// turned into f16 once per workgroup and every wave reads it from LDS: wave w
// owns rows 32 w .. 32 w + 31 of the row tile (waves without rows only help to
// fetch), its queries stay in registers, and no wave waits for another's part
// at the end. A tile is TK keys (4096 values of K and of V), two tiles in LDS:
// while the waves compute on one, the next is on its way to registers; it is
// converted and stored after the products, then one barrier.
//
// F32 caches: a row of K or V becomes f16 pairs of its values times 2^-e, the
// power of two that brings its largest into [2^14, 2^15), so a value is at most
// 2^-22 of itself or 2^-39 of the row's largest off (V: or 2^-124), and a product
// of pairs is hi.lo + lo.hi + hi.hi (three v_mfma_f32_32x32x16_f16, 5 times the
// rate of v_mfma_f32_32x32x2f32): 22 bits an operand where up to 32 rows, which
// those do not bound, take all 24. K's exponent is added to its scores, V's belongs to
// the probability like the scale of an 8-bit row.
//
// LDS rows are a key's D f16 values in 16-byte slots, permuted by row so that
// the reads spread over the banks: K as A operand wants one slot of 32
// consecutive rows (slot ^ swz(row)), V is read transposed (16 lanes take four
// rows' 16 dims and each ends up with one dim of the four keys), which wants
// the 64 bytes of four consecutive rows apart (slot ^ 4 (row % 4)). The keys of
// a lane's V operand are those of its S^T registers, so P needs no exchange.
// Operands are read one group of products ahead of their use.
//
// Bound: the matrix and the vector pipe, one after the other. Per 32 keys and 32
// rows of 128 over an 8-bit cache a wave has 32 matrix instructions (1024 cycles) and
// 266 others (1064, and 16 exponentials at a quarter of the rate); two waves share a
// SIMD, whose matrix pipe is busy 43% of the time and whose vector pipe 52%: the two
// waves hardly ever use them at once. Four 64-token trees over 12304 to 16384 8-bit
// keys (28/4 heads of 128): 146 us, 717 TFLOP/s of f16 products, of the 1106 that a large
// product reaches. Fetching two tiles ahead, and the softmax of one tile beside the
// products of the next, took as long: the registers they need spill or the LDS
// latency shows. Few keys: the start (about 6 us) and the join.
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"
#include "tree_wide_rows.h"

namespace mi {

namespace {

// One unit's row tile of an item, for tree_wide_rows.
template <int D, typename KT>
struct WideWork {
  static constexpr int ELT = (int)sizeof(KT), TK = WideCfg<D, KT>::TK, NDB = D / 32, ROWS = WideCfg<D, KT>::ROWS;
  static constexpr bool kJoins = false;
  const TreeParams& p;
  const TreeItem& it;
  int g, n_past, n_kv, row0, rows, n_rep, key_begin, key_end;
  float scale_log2e;
  const char* kbase;
  const char* vbase;
  float* rec;

  __device__ __forceinline__ int thread() const { return (int)threadIdx.x; }
  __device__ __forceinline__ void at_tile(int) {}
  __device__ __forceinline__ unsigned none() const { return 0u; }
  // The descriptor starts at the tile's first row and ends after its last valid one.
  struct Rows {
    rsrc_t r;
    unsigned s2;
    __device__ __forceinline__ Rows(const WideWork& w, int which, int key0) {
      const int stride = which == 0 ? (int)w.p.k_s2 : (int)w.p.v_s2, n = min(w.n_kv - key0, TK);
      s2 = (unsigned)stride;
      // (unsigned: 63 rows of up to 2^26 bytes pass 2^31)
      r = make_rsrc((which == 0 ? w.kbase : w.vbase) + (int64_t)key0 * stride, (unsigned)(n - 1) * s2 + D * ELT);
    }
    __device__ __forceinline__ rsrc_t rows(int) const { return r; }
    __device__ __forceinline__ unsigned row_at(unsigned row, int) const { return row * s2; }
  };
  struct Scale {
    int stride;
    const char* src;
    __device__ __forceinline__ Scale(const WideWork& w, bool k, int group) {
      stride = w.p.n_head_kv * 2 * (k ? NDB : 1);
      src = ELT == 1 ? (k ? w.it.k_scale + 2 * (w.g * NDB + group) : w.it.v_scale + 2 * w.g) : nullptr;
    }
    __device__ __forceinline__ const char* at(const WideWork& w, int key0, int key) const {
      return src + (int64_t)min(key0 + key, w.n_kv - 1) * stride;
    }
  };
  __device__ __forceinline__ const char* v_row(int key) const { return vbase + (int64_t)key * (int)p.v_s2; }
  __device__ __forceinline__ const char* v_scale(int key) const {
    return it.v_scale + ((int64_t)key * p.n_head_kv + g) * 2;
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
    rec[ROWS * D + r] = ref;
    rec[ROWS * D + ROWS + r] = l;
  }
  __device__ __forceinline__ void put_part(int r, int d, f32x4 x) const { put_record(rec + tree_record_at(D, r, d), x); }
};

}  // namespace

template <int D, typename KT>
__global__ __launch_bounds__(kTreeWaves* kWave, (WideCfg<D, KT>::WAVES_PER_SIMD)) void tree_wide_kernel(const TreeParams p) {
  typedef WideCfg<D, KT> C;
  constexpr int ROWS = C::ROWS, TK = C::TK, THREADS = kTreeWaves * kWave;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int tid = threadIdx.x;

  // Workgroup -> unit and row tile, as in tree_kernel: a unit is (KV head, split,
  // every 2^row_shift-th row tile), its row tiles with the most keys come first.
  const TreeItem& it = p.item[blockIdx.y];
  const int n_rt = it.n_rt, n_split = it.n_split;
  const int y = blockIdx.x / 8, yu = y / it.unit_rt;
  const int unit = yu * 8 + (int)((blockIdx.x - it.xcd0) % 8);
  const int gs = unit >> p.row_shift;
  const int rt = n_rt - 1 - ((y - yu * it.unit_rt) << p.row_shift) - (unit - (gs << p.row_shift));
  if (gs >= p.n_head_kv * n_split || rt < 0) return;
  const int g = gs / n_split, sp = gs - g * n_split;
  const int n_past = it.n_past, n_kv = n_past + it.n_tokens;
  const int rows = it.n_tokens * p.n_rep;
  const int row0 = rt * ROWS;
  const int last_token = min(row0 + ROWS - 1, rows - 1) / p.n_rep;
  const int lim = it.mask ? n_kv : min(n_kv, n_past + last_token + 1);
  // Each row tile cuts the keys that it sees into n_split parts (whole tiles), so
  // that the units, and with them the XCDs, have the same work (2048 8-bit keys
  // and as many tokens, 14/2 heads of 64: 87 -> 65 us; all row tiles of a unit on
  // one XCD, that is with row_shift 0: 65 instead of 49).
  const int tiles = (lim + TK - 1) / TK;
  const int per_split = it.mask ? it.tiles_per_split * kTreeTile : (tiles + n_split - 1) / n_split * TK;
  const int key_begin = min(sp * per_split, lim);
  const int key_end = min(lim, key_begin + per_split);
  if (key_begin >= key_end && n_split > 1) {  // no key for these rows: nothing to join
    float* const rec = p.rec + ((int64_t)it.rec0 + (int64_t)(g * n_rt + rt) * n_split + sp) * (ROWS * (D + 2));
    for (int i = tid; i < 2 * ROWS; i += THREADS) rec[ROWS * D + i] = i < ROWS ? -INFINITY : 0.f;
    return;
  }
  WideWork<D, KT> w{p, it, g, n_past, n_kv, row0, rows, p.n_rep, key_begin, key_end, p.scale_log2e,
                    it.k + (int64_t)g * p.k_s1, it.v + (int64_t)g * p.v_s1,
                    p.rec + ((int64_t)it.rec0 + (int64_t)(g * n_rt + rt) * n_split + sp) * (ROWS * (D + 2))};
  tree_wide_rows<D, KT>(w, (lds_t*)lds_raw);
}

template <int D, typename KT>
static hipError_t launch_wide_t(const TreeParams& p, dim3 grid, hipStream_t stream) {
  typedef WideCfg<D, KT> C;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&tree_wide_kernel<D, KT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((tree_wide_kernel<D, KT>), grid, dim3(kTreeWaves * kWave), C::LDS, stream, p);
  return hipGetLastError();
}

hipError_t launch_tree_wide(const TreeParams& p, dim3 grid, int head_dim, int elt, hipStream_t stream) {
  if (head_dim == 64)
    return elt == 1   ? launch_wide_t<64, int8_t>(p, grid, stream)
           : elt == 2 ? launch_wide_t<64, _Float16>(p, grid, stream)
                      : launch_wide_t<64, float>(p, grid, stream);
  return elt == 1   ? launch_wide_t<128, int8_t>(p, grid, stream)
         : elt == 2 ? launch_wide_t<128, _Float16>(p, grid, stream)
                    : launch_wide_t<128, float>(p, grid, stream);
}

}  // namespace mi
