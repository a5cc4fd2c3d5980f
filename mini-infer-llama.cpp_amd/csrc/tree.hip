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
// record in the workspace that tree_combine_kernel joins (a second launch, so
// that neither needs a counter and both may be captured into a graph).
//
// This kernel: row tiles of 32, for calls that need no more. Its waves take the
// split's key tiles in turn, K and V straight to registers, and meet in LDS at
// the end. (More rows: tree_wide.hip.)
//
// Per key tile (lane = (c = lane % 32, kh = lane / 32)), 32x32 MFMAs:
//   S^T = K . Q^T: A is K (key c), B the queries (row c); a lane ends up with
//   the 16 keys 8 (i / 4) + 4 kh + i % 4 of row c, so the softmax runs within
//   lanes but for one exchange between lane and lane ^ 32, and P is already
//   the B operand of O^T += V^T . P^T. V's A operand is loaded as rows: lane
//   (c, kh) takes the NDB = D / 32 consecutive dims NDB c .. of its 16 keys,
//   so row c of output block db is dim NDB c + db.
//
// Products. F32 cache: v_mfma_f32_32x32x2f32. F16 and 8-bit caches: the cache
// operand is exact in f16, the queries and the probabilities are f16 pairs
// hi = RNE(x), lo = RNE(x - hi), two v_mfma_f32_32x32x16_f16 a step. So that
// lo stays normal, each query row is scaled by the power of two that puts its
// largest element in [2^13, 2^14) (undone in the exponent's multiply-add), and
// the probabilities are 2^(s - ref) for a reference that keeps the largest
// between 2^6 and 2^14 (move_ref; the division by their sum undoes it): 2^-22
// relative to the row's largest element.
//   8-bit K: a row's scales (one per 32 dims) multiply the S^T of their own
//   32 dims. 8-bit V: the row's one scale multiplies the probability; ref keeps
//   the largest such product in that range.
#include <algorithm>

#include "attn_common.h"
#include "kernels.h"
#include "tree_common.h"

namespace mi {

// KT: float, _Float16 or int8_t.
template <int D, typename KT>
struct TreeCfg {
  static constexpr int ELT = (int)sizeof(KT);
  static constexpr bool Q8 = ELT == 1, F32 = ELT == 4;
  static constexpr int NDB = D / 32;             // output blocks of 32 dims; scales per 8-bit K row
  static constexpr int ROWS = 32;
  static constexpr int KW = D * ELT / 8;         // 32-bit words of K per lane and tile
  static constexpr int VW = NDB * ELT >= 4 ? NDB * ELT / 4 : 1;  // words of V per lane and key
  static constexpr int XS = 36;                  // exchange row stride (floats)
  static constexpr int L_X = 0;                  // waves' outputs of one 32-dim block
  static constexpr int L_ML = kTreeWaves * ROWS * XS * 4;  // reference, sum per wave and row
  static constexpr int LDS = L_ML + kTreeWaves * ROWS * 2 * 4;
  // While the keys stream, a wave keeps the tile's scales in its own part of
  // the exchange area: NDB blocks of 32 K scales, 32 V scales, 32 exponents.
  static constexpr int SC = (NDB + 2) * 32 * 4;
  static_assert(SC <= ROWS * XS * 4, "scales fit a wave's exchange area");
  // head_dim 128 takes more registers than two workgroups per CU leave.
  static constexpr int WAVES_PER_SIMD = D == 64 ? 2 : 1;
};

template <int D, typename KT>
__global__ __launch_bounds__(kTreeWaves* kWave, (TreeCfg<D, KT>::WAVES_PER_SIMD)) void tree_kernel(const TreeParams p) {
  typedef TreeCfg<D, KT> C;
  constexpr int NDB = C::NDB, ROWS = C::ROWS, ELT = C::ELT, KW = C::KW, VW = C::VW;
  constexpr bool Q8 = C::Q8, F32 = C::F32;
  __shared__ __attribute__((aligned(16))) char lds_raw[C::LDS];
  lds_t* const lds = (lds_t*)lds_raw;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 31, kh = lane >> 5;

  // Workgroup -> (KV head, split) unit and row tile. The row tiles of a unit
  // read the same keys, so they are numbered 8 apart: workgroups go to the 8
  // XCDs in turn, and theirs then share an L2. Later row tiles of a causal
  // chunk see more keys, so they come first.
  const TreeItem& it = p.item[blockIdx.y];
  const int n_rt = it.n_rt, n_split = it.n_split;
  const int y = blockIdx.x / 8;
  const int rt = n_rt - 1 - y % n_rt;
  const int unit = (y / n_rt) * 8 + (int)((blockIdx.x - it.xcd0) % 8);
  if (unit >= p.n_head_kv * n_split) return;
  const int g = unit / n_split, sp = unit % n_split;
  const int n_past = it.n_past, n_kv = n_past + it.n_tokens;
  const int rows = it.n_tokens * p.n_rep;
  const int row0 = rt * ROWS;
  // keys that some row of the tile may see
  const int last_token = min(row0 + ROWS - 1, rows - 1) / p.n_rep;
  const int lim = it.mask ? n_kv : min(n_kv, n_past + last_token + 1);
  const int tile0 = sp * it.tiles_per_split;
  const int tile1 = min(tile0 + it.tiles_per_split, (lim + kTreeTile - 1) / kTreeTile);

  // ---- loads of a key tile --------------------------------------------------
  // The descriptors start at the tile's first row (64-bit), so a cache of any
  // length is addressed, and end after its last valid row: rows past n_kv
  // read zeros.
  const char* const kbase = it.k + (int64_t)g * p.k_s1;
  const char* const vbase = it.v + (int64_t)g * p.v_s1;
  const int ks2 = (int)p.k_s2, vs2 = (int)p.v_s2;
  unsigned kw[KW], vw[16 * VW], ksc = 0, vsc = 0;
  const unsigned ko = (unsigned)(c * ks2 + 16 * kh);
  const unsigned vo = (unsigned)(4 * kh * vs2 + c * NDB * ELT);
  lds_t* const sc_lds = lds + wave * ROWS * C::XS * 4;
  auto load_k = [&](int tile) __attribute__((always_inline)) {
    const int key0 = tile * kTreeTile;
    const int n = min(n_kv - key0, kTreeTile);
    const rsrc_t r = make_rsrc(kbase + (int64_t)key0 * ks2, (unsigned)((n - 1) * ks2 + D * ELT));
#pragma unroll
    for (int s = 0; s < KW / 4; ++s) {
      const u32x4 x = buf_b128(r, ko + 32 * s);
#pragma unroll
      for (int j = 0; j < 4; ++j) kw[4 * s + j] = x[j];
    }
    if constexpr (Q8) {
      // the scales of key c: lane half kh takes half of the K row's
      const int64_t at = (int64_t)key0 * p.n_head_kv + g;
      const rsrc_t rk = make_rsrc(it.k_scale + at * (2 * NDB), (unsigned)((n - 1) * p.n_head_kv * 2 * NDB + 2 * NDB));
      ksc = NDB == 4 ? buf_b32(rk, (unsigned)(c * p.n_head_kv * 8 + 4 * kh)) : buf_b16(rk, (unsigned)(c * p.n_head_kv * 4 + 2 * kh));
      const rsrc_t rv = make_rsrc(it.v_scale + at * 2, (unsigned)((n - 1) * p.n_head_kv * 2 + 2));
      vsc = buf_b16(rv, (unsigned)(c * p.n_head_kv * 2));
    }
  };
  auto load_v = [&](int tile) __attribute__((always_inline)) {
    const int key0 = tile * kTreeTile;
    const int n = min(n_kv - key0, kTreeTile);
    const rsrc_t r = make_rsrc(vbase + (int64_t)key0 * vs2, (unsigned)((n - 1) * vs2 + D * ELT));
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      const unsigned at = vo + (unsigned)((8 * (t >> 2) + (t & 3)) * vs2);
      if constexpr (NDB * ELT == 16) {
        const u32x4 x = buf_b128(r, at);
#pragma unroll
        for (int j = 0; j < 4; ++j) vw[4 * t + j] = x[j];
      } else if constexpr (NDB * ELT == 8) {
        const u32x2 x = buf_b64(r, at);
        vw[2 * t] = x[0];
        vw[2 * t + 1] = x[1];
      } else if constexpr (NDB * ELT == 4) {
        vw[t] = buf_b32(r, at);
      } else {
        vw[t] = buf_b16(r, at);
      }
    }
  };
  if (tile0 >= tile1 && n_split > 1) {  // no key for these rows: nothing to join
    float* const rec = p.rec + ((int64_t)it.rec0 + (int64_t)(g * n_rt + rt) * n_split + sp) * (ROWS * (D + 2));
    if (threadIdx.x < 2 * ROWS) rec[ROWS * D + threadIdx.x] = threadIdx.x < ROWS ? -INFINITY : 0.f;
    return;
  }
  int tile = tile0 + wave;
  if (tile < tile1) {
    load_k(tile);
    load_v(tile);
  }

  // ---- queries ------------------------------------------------------------
  // Dims of B's step s, lane half kh, element j (A's are loaded the same way):
  // F32 8 (s / 4) + 4 kh + s % 4; F16 16 s + 8 kh + j; 8-bit
  // 32 (s / 2) + 16 kh + 8 (s % 2) + j. Each is 16 consecutive bytes of K.
  float qf[F32 ? D / 2 : 1];
  f16x8 qh[F32 ? 1 : D / 16], ql[F32 ? 1 : D / 16];
  float unscale = 1.f;
  const bool valid = row0 + c < rows;
  const int token = valid ? (row0 + c) / p.n_rep : 0;
  {
    const int h = g * p.n_rep + (valid ? row0 + c - token * p.n_rep : 0);
    const char* const qp = reinterpret_cast<const char*>(it.q) + (int64_t)token * p.q_s2 + (int64_t)h * p.q_s1;
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < D / 2; s += 4) {
        const f32x4 x = gload<f32x4>(qp + 4 * (2 * s + 4 * kh));
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[s + j] = valid ? x[j] * p.scale_log2e : 0.f;
      }
    } else {
      float x[D / 2];
      float amax = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        const int dim = Q8 ? 32 * (s / 2) + 16 * kh + 8 * (s % 2) : 16 * s + 8 * kh;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 v = gload<f32x4>(qp + 4 * (dim + 4 * e));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[8 * s + 4 * e + j] = valid ? v[j] * p.scale_log2e : 0.f;
            amax = fmaxf(amax, fabsf(x[8 * s + 4 * e + j]));
          }
        }
      }
      amax = max32(amax);
      int qexp = 0;
      if (amax > 0.f && amax < INFINITY) qexp = max(ilogbf(amax) - 13, -100);
      unscale = ldexpf(Q8 ? kByteUnscale : 1.f, qexp);
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          f16x2 hi, lo;
          split2(ldexpf(x[8 * s + j], -qexp), ldexpf(x[8 * s + j + 1], -qexp), hi, lo);
          qh[s][j] = hi[0];
          qh[s][j + 1] = hi[1];
          ql[s][j] = lo[0];
          ql[s][j + 1] = lo[1];
        }
    }
  }

  // ---- state --------------------------------------------------------------
  floatx16 o[NDB];
  float ref = -INFINITY, l = 0.f;
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = (floatx16)(0.f);

  for (; tile < tile1; tile += kTreeWaves) {
    const int key0 = tile * kTreeTile;
    const int next = tile + kTreeWaves;
    // ---- S^T = K . Q^T ------------------------------------------------------
    floatx16 s = (floatx16)(0.f);
    f32x4 vfac[4], vexp[4];  // 8-bit: V scales of the lane's keys and their exponents
    if constexpr (F32) {
#pragma unroll
      for (int st = 0; st < D / 2; ++st) s = mfma_f32(__builtin_bit_cast(float, kw[st]), qf[st], s);
    } else if constexpr (!Q8) {
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const f16x8 k8 = __builtin_bit_cast(f16x8, u32x4{kw[4 * st], kw[4 * st + 1], kw[4 * st + 2], kw[4 * st + 3]});
        s = mfma_f16(k8, ql[st], s);
        s = mfma_f16(k8, qh[st], s);
      }
    } else {
      // the scales, to where each lane can read those of its own 16 keys
      auto h2f = [](unsigned x) { return (float)__builtin_bit_cast(_Float16, (unsigned short)x); };
      if constexpr (NDB == 4) {
        lds_store<float>(sc_lds + (64 * kh + c) * 4, h2f(ksc & 0xffffu));
        lds_store<float>(sc_lds + (64 * kh + 32 + c) * 4, h2f(ksc >> 16));
      } else {
        lds_store<float>(sc_lds + (32 * kh + c) * 4, h2f(ksc));
      }
      const float v = h2f(vsc);
      if (kh == 0) {
        lds_store<float>(sc_lds + (32 * NDB + c) * 4, v);
        lds_store<float>(sc_lds + (32 * NDB + 32 + c) * 4, (float)scale_exponent(v < INFINITY ? v : 0.f));
      }
      wave_lds_fence();
#pragma unroll
      for (int b = 0; b < NDB; ++b) {
        floatx16 part = (floatx16)(0.f);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const unsigned w0 = kw[4 * b + 2 * e] ^ 0x80808080u, w1 = kw[4 * b + 2 * e + 1] ^ 0x80808080u;
          const f16x2 x0 = bytes_f16<0, 1>(w0, w0), x1 = bytes_f16<2, 3>(w0, w0);
          const f16x2 x2 = bytes_f16<0, 1>(w1, w1), x3 = bytes_f16<2, 3>(w1, w1);
          const f16x8 k8 = {x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
          part = mfma_f16(k8, ql[2 * b + e], part);
          part = mfma_f16(k8, qh[2 * b + e], part);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 sc = lds_load<f32x4>(sc_lds + (32 * b + 8 * q + 4 * kh) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[4 * q + j] = fmaf(part[4 * q + j], sc[j], s[4 * q + j]);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        vfac[q] = lds_load<f32x4>(sc_lds + (32 * NDB + 8 * q + 4 * kh) * 4);
        vexp[q] = lds_load<f32x4>(sc_lds + (32 * NDB + 32 + 8 * q + 4 * kh) * 4);
      }
      wave_lds_fence();  // the scales are read before the next tile's are written
    }
    if (next < tile1) load_k(next);

    // ---- mask -----------------------------------------------------------------
    unsigned vis = ~0u;
    const bool masked = key0 + kTreeTile > n_past;  // a tile of drafted keys
    if (masked) {
      vis = visible_bits(it, token, key0);
      const unsigned mine = vis >> (4 * kh);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = mine >> (8 * (e >> 2) + (e & 3)) & 1u ? s[e] : -INFINITY;
    }

    // ---- softmax, relative to ref -----------------------------------------------
    float top;
    if constexpr (Q8) {  // of the probability times the V row's scale
      floatx16 x;
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = fmaf(s[e], unscale, vexp[e >> 2][e & 3]);
      top = max32(max16(x, -INFINITY));
    } else {
      top = max32(max16(s, -INFINITY)) * unscale;
    }
    const float alpha = move_ref(ref, top);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0ull) {
      l *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= alpha;
    }
    const float at = ref == -INFINITY ? 0.f : ref;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = fast_exp2(fmaf(s[e], unscale, -at));
      sum[e & 3] += s[e];
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    if constexpr (Q8) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] *= vfac[e >> 2][e & 3];
      if (masked) {  // (a scale may not be finite: 0 times it is not 0)
        const unsigned mine = vis >> (4 * kh);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = mine >> (8 * (e >> 2) + (e & 3)) & 1u ? s[e] : 0.f;
      }
    }

    // ---- values that are not finite, in a tile that some rows do not see --------
    // Their products with a masked key's probability of 0 would not be 0: they
    // are taken as zeros, and the rows that do see them get NaN there.
    unsigned nf[NDB];  // bit t: the lane's key t, dim NDB c + db
    bool any_nf = false;
    if constexpr (!Q8) {
      if (masked) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) nf[db] = 0u;
#pragma unroll
        for (int t = 0; t < 16; ++t) {
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            if constexpr (F32) {
              if (not_finite(__builtin_bit_cast(float, vw[VW * t + w]))) {
                nf[w] |= 1u << t;
                vw[VW * t + w] = 0u;
              }
            } else {
              const unsigned b = not_finite2(vw[VW * t + w]);
              nf[2 * w] |= (b & 1u) << t;
              nf[2 * w + 1] |= (b >> 1) << t;
              vw[VW * t + w] &= (b & 1u ? 0u : 0xffffu) | (b & 2u ? 0u : 0xffff0000u);
            }
          }
        }
        unsigned all = 0u;
#pragma unroll
        for (int db = 0; db < NDB; ++db) all |= nf[db];
        any_nf = __builtin_amdgcn_ballot_w64(all != 0u) != 0ull;
      }
    }

    // ---- O^T += V^T . P^T -----------------------------------------------------
    if constexpr (F32) {
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] = mfma_f32(__builtin_bit_cast(float, vw[VW * t + db]), s[t], o[db]);
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f16x8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          f16x2 hi, lo;
          split2(s[8 * u + j], s[8 * u + j + 1], hi, lo);
          ph[j] = hi[0];
          ph[j + 1] = hi[1];
          pl[j] = lo[0];
          pl[j + 1] = lo[1];
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          f16x8 v8;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const int t = 8 * u + j;
            f16x2 x;
            if constexpr (Q8) {
              const unsigned w0 = vw[t] ^ 0x80808080u, w1 = vw[t + 1] ^ 0x80808080u;
              x = db == 0 ? bytes_f16<0, 4>(w1, w0) : db == 1 ? bytes_f16<1, 5>(w1, w0)
                : db == 2 ? bytes_f16<2, 6>(w1, w0) : bytes_f16<3, 7>(w1, w0);
            } else {
              const unsigned w0 = vw[VW * t + db / 2], w1 = vw[VW * (t + 1) + db / 2];
              x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(w1, w0, db & 1 ? 0x07060302u : 0x05040100u));
            }
            v8[j] = x[0];
            v8[j + 1] = x[1];
          }
          o[db] = mfma_f16(v8, pl, o[db]);
          o[db] = mfma_f16(v8, ph, o[db]);
        }
      }
    }
    if constexpr (!Q8) {
      if (masked && any_nf) {
        for (int src = 0; src < kWave; ++src) {  // the lane that holds the values
          const int sc = src & 31, sh = src >> 5;
          unsigned bits[NDB], some = 0u;
#pragma unroll
          for (int db = 0; db < NDB; ++db) {
            bits[db] = (unsigned)__builtin_amdgcn_readlane((int)nf[db], src);
            some |= bits[db];
          }
          if (some == 0u) continue;
          const unsigned x = vis >> (4 * sh);  // the row's sight of that lane's keys, bit t
          const unsigned seen = (x & 0xfu) | (x >> 4 & 0xf0u) | (x >> 8 & 0xf00u) | (x >> 12 & 0xf000u);
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if ((bits[db] & seen) != 0u && 8 * (e >> 2) + 4 * kh + (e & 3) == sc) o[db][e] = NAN;
        }
      }
    }
    if (next < tile1) load_v(next);
  }

  // ---- the waves' parts ---------------------------------------------------------
  wave_lds_fence();
  const float ls = sum32(l);
  if (kh == 0) {
    lds_store<float>(lds + C::L_ML + ((wave * ROWS + c) * 2) * 4, ref);
    lds_store<float>(lds + C::L_ML + ((wave * ROWS + c) * 2 + 1) * 4, ls);
  }
  __syncthreads();
  float mt = -INFINITY, lt = 0.f;
  {
    constexpr float unit_o = Q8 ? kByteUnscale : 1.f;  // of the values' 2^-10
    f32x2 ml[kTreeWaves];
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) {
      ml[w] = lds_load<f32x2>(lds + C::L_ML + ((w * ROWS + c) * 2) * 4);
      mt = fmaxf(mt, ml[w][0]);
    }
    const float mu = mt == -INFINITY ? 0.f : mt;
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) lt += ml[w][1] * fast_exp2(ml[w][0] - mu);
    const float wt = fast_exp2(ref - mu) * unit_o;
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] *= wt;
  }
  // One 32-dim block at a time through LDS; a thread sums the waves' parts of
  // its (row, column) pairs.
  constexpr int PER = ROWS * 32 / (kTreeWaves * kWave);
  float acc[PER][NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    if (db > 0) __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
      lds_store<f32x4>(lds + ((wave * ROWS + c) * C::XS + 8 * q + 4 * kh) * 4,
                       f32x4{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]});
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int idx = e * kTreeWaves * kWave + threadIdx.x;
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kTreeWaves; ++w) x += lds_load<float>(lds + ((w * ROWS + idx / 32) * C::XS + idx % 32) * 4);
      acc[e][db] = x;
    }
  }
  if (n_split > 1) {
    float* const rec = p.rec + ((int64_t)it.rec0 + (int64_t)(g * n_rt + rt) * n_split + sp) * (ROWS * (D + 2));
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int idx = e * kTreeWaves * kWave + threadIdx.x;
      if (row0 + idx / 32 >= rows) continue;
      float* const w = rec + tree_record_at(D, idx / 32, (NDB * (idx % 32)) & ~3);
      if constexpr (NDB == 4) gstore(w, f32x4{acc[e][0], acc[e][1], acc[e][2], acc[e][3]});
      else gstore(w + 2 * (idx % 2), f32x2{acc[e][0], acc[e][1]});
    }
    if (wave == 0 && kh == 0) {
      rec[ROWS * D + c] = mt;
      rec[ROWS * D + ROWS + c] = lt;
    }
    return;
  }
  // the rows' sums to where the storing threads read them
  if (wave == 0 && kh == 0) lds_store<float>(lds + C::L_ML + c * 4, mt == -INFINITY ? 0.f : 1.f / lt);
  __syncthreads();
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int idx = e * kTreeWaves * kWave + threadIdx.x;
    const int r = row0 + idx / 32;
    if (r >= rows) continue;
    const float inv = lds_load<float>(lds + C::L_ML + (idx / 32) * 4);
    const int t = r / p.n_rep, h = g * p.n_rep + r % p.n_rep;
    char* const w = reinterpret_cast<char*>(it.out) + (int64_t)t * p.o_s2 + (int64_t)h * p.o_s1 + 4 * NDB * (idx % 32);
    if constexpr (NDB == 4) gstore(w, f32x4{acc[e][0] * inv, acc[e][1] * inv, acc[e][2] * inv, acc[e][3] * inv});
    else gstore(w, f32x2{acc[e][0] * inv, acc[e][1] * inv});
  }
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
// kernel (tree_wide.hip), whose waves without rows only fetch.
int tree_tile_rows(int rows) { return rows <= 32 ? 32 : 128; }

size_t tree_record_floats(int head_dim, int tile_rows) { return (size_t)tile_rows * (head_dim + 2); }

template <int D>
static hipError_t launch_narrow(const TreeParams& p, dim3 grid, int elt, hipStream_t stream) {
  if (elt == 1) hipLaunchKernelGGL((tree_kernel<D, int8_t>), grid, dim3(kTreeWaves * kWave), 0, stream, p);
  else if (elt == 2) hipLaunchKernelGGL((tree_kernel<D, _Float16>), grid, dim3(kTreeWaves * kWave), 0, stream, p);
  else hipLaunchKernelGGL((tree_kernel<D, float>), grid, dim3(kTreeWaves * kWave), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_tree(const TreeParams& p, int n_items, int head_dim, int elt, int tile_rows, hipStream_t stream) {
  unsigned gx = 0;
  int64_t units = 0;  // waves' worth of records to join, of the largest item
  int splits = 1;
  for (int i = 0; i < n_items; ++i) {
    const TreeItem& it = p.item[i];
    gx = std::max(gx, ((unsigned)p.n_head_kv * it.n_split + 7) / 8 * 8 * (unsigned)it.n_rt);
    if (it.n_split > 1)
      units = std::max(units, ((int64_t)it.n_tokens * p.n_rep + 31) / 32 * p.n_head_kv * (head_dim / 8));
    splits = std::max(splits, it.n_split);
  }
  const dim3 grid(gx, n_items);
  const hipError_t e = tile_rows == 128  ? launch_tree_wide(p, grid, head_dim, elt, stream)
                       : head_dim == 64 ? launch_narrow<64>(p, grid, elt, stream)
                                        : launch_narrow<128>(p, grid, elt, stream);
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
