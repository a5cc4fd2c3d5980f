// tree_wide.hip -- tree attention (tree.hip has the mathematics, the layout of
// the products and of the records) for many query rows per KV head, F16 and
// 8-bit caches.
//
// With many rows the products bound the work, not the memory, so here a key
// tile is fetched and converted to f16 once per workgroup and every wave reads
// it from LDS: wave w owns rows 32 w .. 32 w + 31 of the workgroup's row tile,
// its queries stay in registers, and no wave waits for another's part at the
// end. A tile is TK keys (4096 values of K and of V), two tiles in LDS: while
// the waves compute on one, the next is on its way to registers; it is
// converted and stored after the products, then one barrier.
//
// LDS rows are a key's D f16 values in 16-byte slots, permuted by row so that
// the reads spread over the banks: K as A operand wants one slot of 32
// consecutive rows (slot ^ swz(row)), V is read transposed (16 lanes take four
// rows' 16 dims and each ends up with one dim of the four keys), which wants
// the 64 bytes of four consecutive rows apart (slot ^ 4 (row % 4)). The keys of
// a lane's V operand are those of its S^T registers, so P needs no exchange.
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"
#include "tree_common.h"

namespace mi {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Lane i of 16 names row i / 4 and four of its f16 values; it receives value i
// of the 16 (i % 4 of chunk i / 4) of all four rows. (A plain function: in a
// kernel template the host pass rejects the builtin.)
__device__ inline u32x2 lds_transposed(const lds_t* p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}

}  // namespace

template <int D, typename KT>
struct WideCfg {
  static constexpr int ELT = (int)sizeof(KT);
  static constexpr bool Q8 = ELT == 1;
  static constexpr int NDB = D / 32;
  static constexpr int ROWS = 32 * kTreeWaves;
  static constexpr int TK = 4096 / D;            // keys per tile
  static constexpr int SUB = TK / 32;            // 32-key blocks of a tile
  static constexpr int NSLOT = D / 8;            // 16-byte slots per LDS row
  static constexpr int PER = 4096 / 8 / (kTreeWaves * kWave);  // slots a thread fetches of K, and of V
  static constexpr int TILE = 8192;              // bytes of a K or V tile
  static constexpr int L_K = 0, L_V = 2 * TILE;  // two buffers each
  static constexpr int L_SC = 4 * TILE;          // per buffer: K scales [NDB][TK], V scales [TK], f16, the V scales' exponent
  static constexpr int SC = (NDB + 1) * TK * 2 + 16;
  static constexpr int L_NF = L_SC + (Q8 ? 2 * SC : 0);  // per buffer: the last tile with values that are not finite
  static constexpr int LDS = L_NF + 16;
};

template <int D, typename KT>
__global__ __launch_bounds__(kTreeWaves* kWave, 2) void tree_wide_kernel(const TreeParams p) {
  typedef WideCfg<D, KT> C;
  constexpr int NDB = C::NDB, ROWS = C::ROWS, ELT = C::ELT, TK = C::TK, SUB = C::SUB, NSLOT = C::NSLOT, PER = C::PER;
  constexpr bool Q8 = C::Q8;
  constexpr int THREADS = kTreeWaves * kWave;
  __shared__ __attribute__((aligned(16))) char lds_raw[C::LDS];
  lds_t* const lds = (lds_t*)lds_raw;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int c = lane & 31, kh = lane >> 5;

  // workgroup -> unit and row tile, as in tree_kernel
  const TreeItem& it = p.item[blockIdx.y];
  const int n_rt = it.n_rt, n_split = it.n_split;
  const int y = blockIdx.x / 8;
  const int rt = n_rt - 1 - y % n_rt;
  const int unit = (y / n_rt) * 8 + (int)((blockIdx.x - it.xcd0) % 8);
  if (unit >= p.n_head_kv * n_split) return;
  const int g = unit / n_split, sp = unit % n_split;
  const int n_kv = it.n_past + it.n_tokens;
  const int rows = it.n_tokens * p.n_rep;
  const int row0 = rt * ROWS;
  const int last_token = min(row0 + ROWS - 1, rows - 1) / p.n_rep;
  const int lim = it.mask ? n_kv : min(n_kv, it.n_past + last_token + 1);
  const int key_begin = sp * it.tiles_per_split * kTreeTile;
  const int key_end = min(lim, key_begin + it.tiles_per_split * kTreeTile);

  // ---- fetching a tile --------------------------------------------------------
  // Thread t takes slots t and t + 256 of the tile's rows (a row's slots are in
  // consecutive threads). The descriptors start at the tile's first row and end
  // after its last valid one: rows past n_kv read zeros.
  const char* const kbase = it.k + (int64_t)g * p.k_s1;
  const char* const vbase = it.v + (int64_t)g * p.v_s1;
  const int ks2 = (int)p.k_s2, vs2 = (int)p.v_s2;
  constexpr int WORDS = 8 * ELT / 4;  // of 8 values
  unsigned kw[PER][WORDS], vw[PER][WORDS], scw = 0;
  unsigned ko[PER], vo[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = (tid + THREADS * i) / NSLOT, s = (tid + THREADS * i) % NSLOT;
    ko[i] = (unsigned)(r * ks2 + 8 * ELT * s);
    vo[i] = (unsigned)(r * vs2 + 8 * ELT * s);
  }
  // 8-bit: thread t's scale of a tile: the K scales (key t / NDB, group t % NDB),
  // then the V scales. Every thread loads one (those behind the last scale that
  // of key 0, not stored) from a row that is there.
  const bool sc_k = tid < TK * NDB, sc_v = !sc_k && tid < TK * (NDB + 1);
  const int sc_key = sc_k ? tid / NDB : sc_v ? tid - TK * NDB : 0;
  const int sc_stride = p.n_head_kv * 2 * (sc_k ? NDB : 1);
  const char* const sc_src = Q8 ? (sc_k ? it.k_scale + 2 * (g * NDB + tid % NDB) : it.v_scale + 2 * g) : nullptr;
  auto fetch = [&](int key0) __attribute__((always_inline)) {
    const int n = min(n_kv - key0, TK);
    const rsrc_t rk = make_rsrc(kbase + (int64_t)key0 * ks2, (unsigned)((n - 1) * ks2 + D * ELT));
    const rsrc_t rv = make_rsrc(vbase + (int64_t)key0 * vs2, (unsigned)((n - 1) * vs2 + D * ELT));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if constexpr (Q8) {
        const u32x2 a = buf_b64(rk, ko[i]), b = buf_b64(rv, vo[i]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          kw[i][j] = a[j];
          vw[i][j] = b[j];
        }
      } else {
        const u32x4 a = buf_b128(rk, ko[i]), b = buf_b128(rv, vo[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kw[i][j] = a[j];
          vw[i][j] = b[j];
        }
      }
    }
    if constexpr (Q8) {
      scw = gload<unsigned short>(sc_src + (int64_t)(key0 + min(sc_key, n - 1)) * sc_stride);
    }
  };
  // Eight values as f16: an 8-bit value v as v 2^-10 (see bytes_f16).
  auto widen = [](const unsigned (&w)[WORDS]) __attribute__((always_inline)) {
    if constexpr (Q8) {
      const unsigned a = w[0] ^ 0x80808080u, b = w[1] ^ 0x80808080u;
      const f16x2 x0 = bytes_f16<0, 1>(a, a), x1 = bytes_f16<2, 3>(a, a), x2 = bytes_f16<0, 1>(b, b),
                  x3 = bytes_f16<2, 3>(b, b);
      return u32x4{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1), __builtin_bit_cast(unsigned, x2),
                   __builtin_bit_cast(unsigned, x3)};
    } else {
      return u32x4{w[0], w[1], w[2], w[3]};
    }
  };
  constexpr int VSWZ = NSLOT >= 16 ? 3 : 1;  // rows of 128 bytes: two of them span the banks
  auto put = [&](int buf, int key0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = (tid + THREADS * i) / NSLOT, s = (tid + THREADS * i) % NSLOT;
      lds_store<u32x4>(lds + C::L_K + buf * C::TILE + r * (2 * D) + 16 * (s ^ swz<NSLOT>(r)), widen(kw[i]));
      u32x4 v = widen(vw[i]);
      if constexpr (!Q8) {
        // A masked key's probability of 0 times such a value would not be 0:
        // in a tile that some rows do not see they become zeros, and the tile
        // is marked for the rows that do.
        if (key0 + TK > it.n_past) {
          unsigned any = 0u;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const unsigned b = not_finite2(v[j]);
            any |= b;
            v[j] &= (b & 1u ? 0u : 0xffffu) | (b & 2u ? 0u : 0xffff0000u);
          }
          if (any) lds_store<int>(lds + C::L_NF + 4 * buf, key0);
        }
      }
      lds_store<u32x4>(lds + C::L_V + buf * C::TILE + r * (2 * D) + 16 * (s ^ 4 * (r & VSWZ)), v);
    }
    if constexpr (Q8) {
      lds_t* const sc = lds + C::L_SC + buf * C::SC;
      if (sc_k) lds_store<unsigned short>(sc + ((tid % NDB) * TK + sc_key) * 2, (unsigned short)scw);
      if (sc_v) {  // TK threads of one wave
        lds_store<unsigned short>(sc + tid * 2, (unsigned short)scw);
        const float v = (float)__builtin_bit_cast(_Float16, (unsigned short)scw);
        float top = row_max16(v < INFINITY ? v : 0.f);
#pragma unroll
        for (int off = 16; off < TK; off *= 2) top = fmaxf(top, __shfl_xor(top, off, kWave));
        if (tid == TK * NDB) lds_store<float>(sc + (NDB + 1) * TK * 2, (float)scale_exponent(top));
      }
    }
  };
  if (tid < 2) lds_store<int>(lds + C::L_NF + 4 * tid, -1);
  if (key_begin < key_end) fetch(key_begin);

  // ---- queries: row c of the wave's 32, dims 16 s + 8 kh + j of step s -----------
  const int r = row0 + 32 * wave + c;
  const bool valid = r < rows;
  const int token = valid ? r / p.n_rep : 0;
  const int h = g * p.n_rep + (valid ? r - token * p.n_rep : 0);
  f16x8 qh[D / 16], ql[D / 16];
  float unscale = 1.f;
  {
    const char* const qp = reinterpret_cast<const char*>(it.q) + (int64_t)token * p.q_s2 + (int64_t)h * p.q_s1;
    float x[D / 2], amax = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 v = gload<f32x4>(qp + 4 * (16 * s + 8 * kh + 4 * e));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[8 * s + 4 * e + j] = valid ? v[j] * p.scale_log2e : 0.f;
          amax = fmaxf(amax, fabsf(x[8 * s + 4 * e + j]));
        }
      }
    amax = max32(amax);
    float f = 1.f;
    if (amax > 0.f && amax < INFINITY) {
      const int e = min(13 - ilogbf(amax), 100);
      f = ldexpf(1.f, e);
      unscale = ldexpf(1.f, -e);
    }
    if constexpr (Q8) unscale *= kByteUnscale;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        f16x2 hi, lo;
        split2(x[8 * s + j] * f, x[8 * s + j + 1] * f, hi, lo);
        qh[s][j] = hi[0];
        qh[s][j + 1] = hi[1];
        ql[s][j] = lo[0];
        ql[s][j + 1] = lo[1];
      }
  }
  floatx16 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = (floatx16)(0.f);
  float ref = -INFINITY, l = 0.f;

  // lane parts of the LDS addresses
  const lds_t* const krow = lds + C::L_K + c * (2 * D);
  const int kx = swz<NSLOT>(c);  // (rows 32 apart have the same)
  const int vi = lane & 15;
  const lds_t* const vrow = lds + C::L_V + (4 * kh + (vi >> 2)) * (2 * D) + 8 * (vi & 1);
  const int vs = 2 * ((lane >> 4) & 1) + ((vi & 3) >> 1), vx = 4 * ((vi >> 2) & VSWZ);

  if (key_begin < key_end) put(0, key_begin);
  __syncthreads();
  int buf = 0;
  for (int key0 = key_begin; key0 < key_end; key0 += TK, buf ^= 1) {
    const int next = key0 + TK;
    if (next < key_end) fetch(next);

    // ---- S^T = K . Q^T ----------------------------------------------------------
    floatx16 s[SUB];
    const lds_t* const sc_base = lds + C::L_SC + buf * C::SC;
    const lds_t* const sc = sc_base + 8 * kh;  // the lane's keys 8 q + 4 kh ..
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      s[u] = (floatx16)(0.f);
      floatx16 part;
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const f16x8 k8 = lds_load<f16x8>(krow + buf * C::TILE + u * 32 * (2 * D) + 16 * ((2 * st + kh) ^ kx));
        if constexpr (Q8) {
          if (st % 2 == 0) part = (floatx16)(0.f);
          part = mfma_f16(k8, ql[st], part);
          part = mfma_f16(k8, qh[st], part);
          if (st % 2 == 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f16x4 x = lds_load<f16x4>(sc + ((st / 2) * TK + 32 * u + 8 * q) * 2);
#pragma unroll
              for (int j = 0; j < 4; ++j) s[u][4 * q + j] = fmaf(part[4 * q + j], (float)x[j], s[u][4 * q + j]);
            }
          }
        } else {
          s[u] = mfma_f16(k8, ql[st], s[u]);
          s[u] = mfma_f16(k8, qh[st], s[u]);
        }
      }
    }

    // ---- mask -------------------------------------------------------------------
    const bool masked = next > it.n_past;
    unsigned vis[SUB];
    if (masked) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        vis[u] = visible_bits(it, token, key0 + 32 * u);
        const unsigned mine = vis[u] >> (4 * kh);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[u][e] = mine >> (8 * (e >> 2) + (e & 3)) & 1u ? s[u][e] : -INFINITY;
      }
    }

    // ---- softmax, relative to ref ---------------------------------------------------
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUB; ++u) top = max16(s[u], top);
    top = max32(top) * unscale;
    if constexpr (Q8) top += lds_load<float>(sc_base + (NDB + 1) * TK * 2);
    const float alpha = move_ref(ref, top);
    const float at = ref == -INFINITY ? 0.f : ref;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[u][e] = fast_exp2(fmaf(s[u][e], unscale, -at));
        sum[e & 3] += s[u][e];
      }
    l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if constexpr (Q8) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f16x4 x = lds_load<f16x4>(sc + (NDB * TK + 32 * u + 8 * q) * 2);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][4 * q + j] = fmaf(s[u][4 * q + j], (float)x[j], 0.f);
        }
      if (masked) {  // (a scale may not be finite: 0 times it is not 0)
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          const unsigned mine = vis[u] >> (4 * kh);
#pragma unroll
          for (int e = 0; e < 16; ++e) s[u][e] = mine >> (8 * (e >> 2) + (e & 3)) & 1u ? s[u][e] : 0.f;
        }
      }
    }
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0ull) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= alpha;
    }

    // ---- O^T += V^T . P^T -------------------------------------------------------------
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        f16x8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          f16x2 hi, lo;
          split2(s[u][8 * w + j], s[u][8 * w + j + 1], hi, lo);
          ph[j] = hi[0];
          ph[j + 1] = hi[1];
          pl[j] = lo[0];
          pl[j + 1] = lo[1];
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const lds_t* const at = vrow + buf * C::TILE + (32 * u + 16 * w) * (2 * D) + 16 * ((4 * db + vs) ^ vx);
          const u32x2 a = lds_transposed(at), b = lds_transposed(at + 8 * (2 * D));
          const f16x8 v8 = __builtin_bit_cast(f16x8, u32x4{a[0], a[1], b[0], b[1]});
          o[db] = mfma_f16(v8, pl, o[db]);
          o[db] = mfma_f16(v8, ph, o[db]);
        }
      }

    if constexpr (!Q8) {
      // rows that see a value which is not finite get NaN in its dim
      if (masked && lds_load<int>(lds + C::L_NF + 4 * buf) == key0) {
        const int n = min(n_kv - key0, TK);
        for (int t = 0; t < n; ++t) {
          unsigned word = vis[0];
          if constexpr (SUB > 1) word = t < 32 ? vis[0] : vis[1];
          const bool sees = word >> (t & 31) & 1u;
          const char* const vr = vbase + (int64_t)(key0 + t) * vs2;
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const unsigned x = gload<unsigned short>(vr + 2 * (32 * db + 8 * (e >> 2) + 4 * kh + (e & 3)));
              if (sees && not_finite2(x) != 0u) o[db][e] = NAN;
            }
        }
      }
    }
    if (next < key_end) put(buf ^ 1, next);
    __syncthreads();
  }

  // ---- the wave's rows ------------------------------------------------------------
  const float lt = sum32(l);
  constexpr float unit_o = Q8 ? kByteUnscale : 1.f;  // of the values' 2^-10
  if (n_split > 1) {
    float* const rec = p.rec + ((int64_t)it.rec0 + (int64_t)(g * n_rt + rt) * n_split + sp) * (ROWS * (D + 2));
    const int rr = 32 * wave + c;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        gstore(rec + rr * D + 32 * db + 8 * q + 4 * kh,
               f32x4{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]} * unit_o);
    if (kh == 0) {
      rec[ROWS * D + rr] = ref;
      rec[ROWS * D + ROWS + rr] = lt;
    }
    return;
  }
  if (!valid) return;
  const float inv = ref == -INFINITY ? 0.f : unit_o / lt;
  char* const out = reinterpret_cast<char*>(it.out) + (int64_t)token * p.o_s2 + (int64_t)h * p.o_s1;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      gstore(out + 4 * (32 * db + 8 * q + 4 * kh),
             f32x4{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]} * inv);
}

template <int D, typename KT>
static hipError_t launch_wide_t(const TreeParams& p, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL((tree_wide_kernel<D, KT>), grid, dim3(kTreeWaves * kWave), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_tree_wide(const TreeParams& p, dim3 grid, int head_dim, int elt, hipStream_t stream) {
  if (head_dim == 64) return elt == 1 ? launch_wide_t<64, int8_t>(p, grid, stream) : launch_wide_t<64, _Float16>(p, grid, stream);
  return elt == 1 ? launch_wide_t<128, int8_t>(p, grid, stream) : launch_wide_t<128, _Float16>(p, grid, stream);
}

}  // namespace mi
