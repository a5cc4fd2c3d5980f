// tree_rows.h -- up to 32 query rows of one KV head over a range of key tiles (tree.hip has the
// mathematics and the layout of the products). A workgroup's waves take the
// tiles in turn, K and V straight to registers, and meet in LDS at the end.
//
// What the rows and keys are is W's matter (TreeWork of tree.hip: a run of cache
// rows; paged_attn.hip: pages):
//   thread(): threadIdx.x;
//   n_past, rows, n_rep, scale_log2e, k_s2, v_s2 (bytes between rows), tile0, tile1
//   at_tile(tile): the tile whose rows are loaded next;
//   k_rows(key0), v_rows(key0): descriptors of its two times 16 rows, which read
//     zeros past the last valid one;
//   scales<NB>(..): 8-bit caches: the scales of the lane's key;
//   none(): of the tile at hand, which 16 rows have no page (their keys are NaN);
//   visible(token, key0): which of 32 keys a query sees;
//   q_row, out_row(token, head of the group);
//   is_part(): the result is one part of the rows' keys: put_sums, put_part take it.
#pragma once

#include "tree_common.h"

namespace mi {

namespace {

__device__ inline f32x4 mfma16_f16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma16_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Over the four lanes that share lane % 16. v_permlane16_swap exchanges the odd
// rows of 16 lanes of one operand with the even rows of the other, so two copies
// of x become x of the even and of the odd row of the pair. (s_nop: as in swap32.)
__device__ inline void swap16(float x, float& a, float& b) {
  float y = x;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  a = x;
  b = y;
}
__device__ inline float max_quarters(float x) {
  float a, b;
  swap16(x, a, b);
  return max32(fmaxf(a, b));
}
__device__ inline float sum_quarters(float x) {
  float a, b;
  swap16(x, a, b);
  return sum32(a + b);
}

// Bits 4 q .. 4 q + 3 and 16 + 4 q .. of a tile's 32 keys: the eight of a lane.
__device__ inline unsigned slots_of(unsigned keys, int q) {
  return (keys >> (4 * q) & 0xfu) | (keys >> (16 + 4 * q) & 0xfu) << 4;
}

// The two times 16 rows of a key tile: descriptors, and what is added to a lane's offset.
struct TileRows {
  rsrc_t rows[2];
  unsigned at[2];
};

}  // namespace

// KT: float, _Float16 or int8_t; RT: 16-row tiles of queries.
template <int D, typename KT, int RT>
struct TreeCfg {
  static constexpr int ELT = (int)sizeof(KT);
  static constexpr bool Q8 = ELT == 1, F32 = ELT == 4;
  static constexpr int NB = D / 32;              // 32-dim blocks (of K; scales per 8-bit K row)
  static constexpr int NE = D / 16;              // V dims per lane and key; output blocks of 16 dims
  static constexpr int ROWS = 16 * RT;
  static constexpr int KB = F32 ? 2 * NB : NB;   // K loads per 16 keys
  static constexpr int KW = F32 || ELT == 2 ? 4 : 2;  // words of one
  static constexpr int VW = NE * ELT / 4;        // words of V per lane and key
  static constexpr int XS = D + 4;               // exchange row stride (floats)
  static constexpr int L_ML = kTreeWaves * ROWS * XS * 4;  // reference, sum per wave and row
  static constexpr int LDS = L_ML + kTreeWaves * ROWS * 2 * 4;
  // While the keys stream, a wave keeps the tile's scales in its own part of
  // the exchange area: NB blocks of 32 K scales, 32 V scales, 32 exponents.
  static constexpr int SC = (NB + 2) * 32 * 4;
  static_assert(SC <= ROWS * XS * 4, "scales fit a wave's exchange area");
  // head_dim 128, two tiles: more registers than two workgroups on a CU leave.
  static constexpr int WAVES_PER_SIMD = D == 128 && RT == 2 ? 1 : 2;
};

template <int D, typename KT, int RT, typename W>
__device__ __forceinline__ void tree_rows(W& w, lds_t* const lds) {
  typedef TreeCfg<D, KT, RT> C;
  constexpr int NB = C::NB, NE = C::NE, ROWS = C::ROWS, ELT = C::ELT, KB = C::KB, KW = C::KW, VW = C::VW;
  constexpr bool Q8 = C::Q8, F32 = C::F32;
  const int tid = w.thread(), lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int c = lane & 15, q4 = lane >> 4;

  // ---- loads of a key tile --------------------------------------------------
  const int ks2 = w.k_s2, vs2 = w.v_s2;
  unsigned kw[2][KB][KW], vw[8][VW], ksc = 0, vsc = 0;
  const unsigned ko = (unsigned)(c * ks2 + 4 * KW * q4);
  const unsigned vo = (unsigned)(4 * q4 * vs2 + c * NE * ELT);
  lds_t* const sc_lds = lds + wave * ROWS * C::XS * 4;
  const int c32 = lane & 31, half = lane >> 5;
  auto load_k = [&](int tile) __attribute__((always_inline)) {
    const int key0 = tile * kTreeTile;
    const TileRows r = w.k_rows(key0);
#pragma unroll
    for (int hk = 0; hk < 2; ++hk)
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const unsigned at = ko + r.at[hk] + 16 * KW * b;
        if constexpr (KW == 4) {
          const u32x4 x = buf_b128(r.rows[hk], at);
#pragma unroll
          for (int j = 0; j < 4; ++j) kw[hk][b][j] = x[j];
        } else {
          const u32x2 x = buf_b64(r.rows[hk], at);
          kw[hk][b][0] = x[0];
          kw[hk][b][1] = x[1];
        }
      }
    // the scales of key lane % 32: each half of the wave takes half of the K row's
    if constexpr (Q8) w.template scales<NB>(key0, c32, half, ksc, vsc);
  };
  auto load_v = [&](int tile) __attribute__((always_inline)) {
    const int key0 = tile * kTreeTile;
    const TileRows r = w.v_rows(key0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // keys 16 (j / 4) + 4 q4 + j % 4
      const unsigned at = vo + r.at[j / 4] + (unsigned)(j % 4 * vs2);
      if constexpr (VW >= 4) {
#pragma unroll
        for (int e = 0; e < VW; e += 4) {
          const u32x4 x = buf_b128(r.rows[j / 4], at + 4 * e);
#pragma unroll
          for (int i = 0; i < 4; ++i) vw[j][e + i] = x[i];
        }
      } else if constexpr (VW == 2) {
        const u32x2 x = buf_b64(r.rows[j / 4], at);
        vw[j][0] = x[0];
        vw[j][1] = x[1];
      } else {
        vw[j][0] = buf_b32(r.rows[j / 4], at);
      }
    }
  };
  int tile = w.tile0 + wave;
  const int tile1 = w.tile1;
  if (tile < tile1) {
    w.at_tile(tile);
    load_k(tile);
    load_v(tile);
  }

  // ---- queries: row c of tile i; dims as K's ------------------------------------
  float qf[F32 ? RT : 1][F32 ? D / 4 : 1];
  f16x8 qh[F32 ? 1 : RT][F32 ? 1 : NB], ql[F32 ? 1 : RT][F32 ? 1 : NB];
  float unscale[RT];
  int token[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = 16 * i + c;
    const bool valid = r < w.rows;
    token[i] = valid ? r / w.n_rep : 0;
    unscale[i] = 1.f;
    const char* const qp = w.q_row(token[i], valid ? r - token[i] * w.n_rep : 0);
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < D / 4; s += 4) {  // dims 4 s + 4 q4 + j
        const f32x4 x = gload<f32x4>(qp + 4 * (4 * s + 4 * q4));
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[i][s + j] = valid ? x[j] * w.scale_log2e : 0.f;
      }
    } else {
      float x[D / 4], amax = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const f32x4 v = gload<f32x4>(qp + 4 * (32 * b + 8 * q4 + 4 * e));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[8 * b + 4 * e + j] = valid ? v[j] * w.scale_log2e : 0.f;
            amax = fmaxf(amax, fabsf(x[8 * b + 4 * e + j]));
          }
        }
      amax = max_quarters(amax);
      int qexp = 0;
      if (amax > 0.f && amax < INFINITY) qexp = max(ilogbf(amax) - 13, -100);
      unscale[i] = ldexpf(Q8 ? kByteUnscale : 1.f, qexp);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          f16x2 hi, lo;
          split2(ldexpf(x[8 * b + j], -qexp), ldexpf(x[8 * b + j + 1], -qexp), hi, lo);
          qh[i][b][j] = hi[0];
          qh[i][b][j + 1] = hi[1];
          ql[i][b][j] = lo[0];
          ql[i][b][j + 1] = lo[1];
        }
    }
  }

  // ---- state --------------------------------------------------------------
  f32x4 o[RT][NE];
  float ref[RT], l[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    ref[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int db = 0; db < NE; ++db) o[i][db] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  for (; tile < tile1; tile += kTreeWaves) {
    const int key0 = tile * kTreeTile;
    const int next = tile + kTreeWaves;
    const unsigned none = w.none();  // bit hk: keys 16 hk .. have no page
    // ---- S^T = K . Q^T: s[i][4 hk + j] is key 16 hk + 4 q4 + j of row c ----------
    float s[RT][8];
    f32x4 vfac[2], vexp[2];  // 8-bit: V scales of the lane's keys and their exponents
    if constexpr (Q8) {
      // the scales, to where each lane can read those of its own keys
      auto h2f = [](unsigned x) { return (float)__builtin_bit_cast(_Float16, (unsigned short)x); };
      if constexpr (NB == 4) {
        lds_store<float>(sc_lds + (64 * half + c32) * 4, h2f(ksc & 0xffffu));
        lds_store<float>(sc_lds + (64 * half + 32 + c32) * 4, h2f(ksc >> 16));
      } else {
        lds_store<float>(sc_lds + (32 * half + c32) * 4, h2f(ksc));
      }
      const float v = h2f(vsc);
      if (half == 0) {
        lds_store<float>(sc_lds + (32 * NB + c32) * 4, v);
        lds_store<float>(sc_lds + (32 * NB + 32 + c32) * 4, (float)scale_exponent(v < INFINITY ? v : 0.f));
      }
      wave_lds_fence();
    }
#pragma unroll
    for (int hk = 0; hk < 2; ++hk) {
      f32x4 acc[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (F32) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < RT; ++i)
              acc[i] = mfma16_f32(__builtin_bit_cast(float, kw[hk][b][j]), qf[i][4 * b + j], acc[i]);
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          f16x8 k8;
          if constexpr (Q8) {
            const unsigned w0 = kw[hk][b][0] ^ 0x80808080u, w1 = kw[hk][b][1] ^ 0x80808080u;
            const f16x2 x0 = bytes_f16<0, 1>(w0, w0), x1 = bytes_f16<2, 3>(w0, w0);
            const f16x2 x2 = bytes_f16<0, 1>(w1, w1), x3 = bytes_f16<2, 3>(w1, w1);
            k8 = f16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
          } else {
            k8 = __builtin_bit_cast(f16x8, u32x4{kw[hk][b][0], kw[hk][b][1], kw[hk][b][2], kw[hk][b][3]});
          }
          if constexpr (Q8) {
            const f32x4 sc = lds_load<f32x4>(sc_lds + (32 * b + 16 * hk + 4 * q4) * 4);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              f32x4 part = mfma16_f16(k8, ql[i][b], f32x4{0.f, 0.f, 0.f, 0.f});
              part = mfma16_f16(k8, qh[i][b], part);
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(part[j], sc[j], acc[i][j]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              acc[i] = mfma16_f16(k8, ql[i][b], acc[i]);
              acc[i] = mfma16_f16(k8, qh[i][b], acc[i]);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][4 * hk + j] = acc[i][j];
    }
    if constexpr (Q8) {
#pragma unroll
      for (int hk = 0; hk < 2; ++hk) {
        vfac[hk] = lds_load<f32x4>(sc_lds + (32 * NB + 16 * hk + 4 * q4) * 4);
        vexp[hk] = lds_load<f32x4>(sc_lds + (32 * NB + 32 + 16 * hk + 4 * q4) * 4);
      }
      wave_lds_fence();  // the scales are read before the next tile's are written
    }
    if (next < tile1) {
      w.at_tile(next);
      load_k(next);
    }

    // ---- mask -----------------------------------------------------------------
    // bit 4 hk + j of vis: the row sees the lane's key 16 hk + 4 q4 + j
    unsigned row_vis[RT], vis[RT];
    const bool masked = key0 + kTreeTile > w.n_past || none != 0u;  // a tile of drafted keys
    if (masked) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        row_vis[i] = w.visible(token[i], key0);
        vis[i] = slots_of(row_vis[i], q4);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[i][e] = vis[i] >> e & 1u ? (none >> (e / 4) & 1u ? NAN : s[i][e]) : -INFINITY;
      }
    }

    // ---- softmax, relative to ref -----------------------------------------------
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        // (8-bit: of the probability times the V row's scale)
        const float a = Q8 ? fmaf(s[i][e], unscale[i], vexp[e / 4][e % 4]) : s[i][e];
        const float b = Q8 ? fmaf(s[i][e + 1], unscale[i], vexp[e / 4][e % 4 + 1]) : s[i][e + 1];
        top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, a), b);
      }
      const float alpha = move_ref(ref[i], max_quarters(top) * (Q8 ? 1.f : unscale[i]));
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0ull) {
        l[i] *= alpha;
#pragma unroll
        for (int db = 0; db < NE; ++db) o[i][db] *= alpha;
      }
      // (F32: probabilities up to 1, so that no product with a value leaves float's range)
      const float at = ref[i] == -INFINITY ? 0.f : ref[i] + (F32 ? kRefMost : 0.f);
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[i][e] = fast_exp2(fmaf(s[i][e], unscale[i], -at));
        sum[e & 1] += s[i][e];
        if constexpr (Q8) s[i][e] *= vfac[e / 4][e % 4];
      }
      l[i] += sum[0] + sum[1];
      if constexpr (Q8) {
        if (masked) {  // (a scale may not be finite: 0 times it is not 0)
#pragma unroll
          for (int e = 0; e < 8; ++e) s[i][e] = vis[i] >> e & 1u ? s[i][e] : 0.f;
        }
      }
    }

    // ---- values that are not finite, in a tile that some rows do not see --------
    // Their products with a masked key's probability of 0 would not be 0: they
    // are taken as zeros, and the rows that do see them get NaN there.
    unsigned nf[NE];  // bit j: the lane's key j, dim NE c + db
    bool any_nf = false;
    if constexpr (!Q8) {
      if (masked) {
#pragma unroll
        for (int db = 0; db < NE; ++db) nf[db] = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
          for (int e = 0; e < VW; ++e) {
            if constexpr (F32) {
              if (not_finite(__builtin_bit_cast(float, vw[j][e]))) {
                nf[e] |= 1u << j;
                vw[j][e] = 0u;
              }
            } else {
              const unsigned b = not_finite2(vw[j][e]);
              nf[2 * e] |= (b & 1u) << j;
              nf[2 * e + 1] |= (b >> 1) << j;
              vw[j][e] &= (b & 1u ? 0u : 0xffffu) | (b & 2u ? 0u : 0xffff0000u);
            }
          }
        }
        unsigned all = 0u;
#pragma unroll
        for (int db = 0; db < NE; ++db) all |= nf[db];
        any_nf = __builtin_amdgcn_ballot_w64(all != 0u) != 0ull;
      }
    }

    // ---- O^T += V^T . P^T: o[i][db][j] is dim NE (4 q4 + j) + db of row c ----------
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int db = 0; db < NE; ++db)
#pragma unroll
          for (int i = 0; i < RT; ++i) o[i][db] = mfma16_f32(__builtin_bit_cast(float, vw[j][db]), s[i][j], o[i][db]);
    } else {
      f16x8 ph[RT], pl[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          f16x2 hi, lo;
          split2(s[i][j], s[i][j + 1], hi, lo);
          ph[i][j] = hi[0];
          ph[i][j + 1] = hi[1];
          pl[i][j] = lo[0];
          pl[i][j + 1] = lo[1];
        }
      if constexpr (Q8) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < VW; ++e) vw[j][e] ^= 0x80808080u;
      }
#pragma unroll
      for (int db = 0; db < NE; ++db) {
        f16x8 v8;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          f16x2 x;
          if constexpr (Q8) {
            const unsigned w0 = vw[j][db / 4], w1 = vw[j + 1][db / 4];
            x = db % 4 == 0 ? bytes_f16<0, 4>(w1, w0) : db % 4 == 1 ? bytes_f16<1, 5>(w1, w0)
              : db % 4 == 2 ? bytes_f16<2, 6>(w1, w0) : bytes_f16<3, 7>(w1, w0);
          } else {
            x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(vw[j + 1][db / 2], vw[j][db / 2],
                                                                db & 1 ? 0x07060302u : 0x05040100u));
          }
          v8[j] = x[0];
          v8[j + 1] = x[1];
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          o[i][db] = mfma16_f16(v8, pl[i], o[i][db]);
          o[i][db] = mfma16_f16(v8, ph[i], o[i][db]);
        }
      }
    }
    if constexpr (!Q8) {
      if (masked && any_nf) {
        for (int src = 0; src < kWave; ++src) {  // the lane that holds the values
          const int sc = src & 15, sq = src >> 4;
          unsigned bits[NE], some = 0u;
#pragma unroll
          for (int db = 0; db < NE; ++db) {
            bits[db] = (unsigned)__builtin_amdgcn_readlane((int)nf[db], src);
            some |= bits[db];
          }
          if (some == 0u) continue;
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            const unsigned seen = slots_of(row_vis[i], sq);
#pragma unroll
            for (int db = 0; db < NE; ++db)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if ((bits[db] & seen) != 0u && 4 * q4 + j == sc) o[i][db][j] = NAN;
          }
        }
      }
    }
    if (next < tile1) load_v(next);
  }

  // ---- the waves' parts, through LDS -----------------------------------------------
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const float lt = sum_quarters(l[i]);
    if (q4 == 0) lds_store<f32x2>(lds + C::L_ML + ((wave * ROWS + 16 * i + c) * 2) * 4, f32x2{ref[i], lt});
  }
  __syncthreads();
  constexpr float unit_o = Q8 ? kByteUnscale : 1.f;  // of the values' 2^-10
  float mt[RT], lt[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    f32x2 ml[kTreeWaves];
    mt[i] = -INFINITY;
    lt[i] = 0.f;
#pragma unroll
    for (int o = 0; o < kTreeWaves; ++o) {
      ml[o] = lds_load<f32x2>(lds + C::L_ML + ((o * ROWS + 16 * i + c) * 2) * 4);
      mt[i] = fmaxf(mt[i], ml[o][0]);
    }
    const float mu = mt[i] == -INFINITY ? 0.f : mt[i];
#pragma unroll
    for (int o = 0; o < kTreeWaves; ++o) lt[i] += ml[o][1] * fast_exp2(ml[o][0] - mu);
    const float wt = fast_exp2(ref[i] - mu) * unit_o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int db = 0; db < NE; db += 4)
        lds_store<f32x4>(lds + ((wave * ROWS + 16 * i + c) * C::XS + NE * (4 * q4 + j) + db) * 4,
                         f32x4{o[i][db][j], o[i][db + 1][j], o[i][db + 2][j], o[i][db + 3][j]} * wt);
  }
  __syncthreads();
  if (w.is_part()) {
    if (wave == 0 && q4 == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i) w.put_sums(16 * i + c, mt[i], lt[i]);
    }
  } else {
    // the rows' factors to where the storing threads read them (where the waves'
    // references lay: every wave has read them)
    if (wave == 0 && q4 == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i)
        lds_store<float>(lds + C::L_ML + (16 * i + c) * 4, mt[i] == -INFINITY && lt[i] == 0.f ? 0.f : 1.f / lt[i]);
    }
    __syncthreads();
  }
  // thread: four dims of a row
#pragma unroll
  for (int e = 0; e < ROWS * D / 4; e += kTreeWaves * kWave) {
    const int idx = e + tid, r = idx / (D / 4), d = 4 * (idx % (D / 4));
    if (r >= w.rows) continue;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < kTreeWaves; ++o) x += lds_load<f32x4>(lds + ((o * ROWS + r) * C::XS + d) * 4);
    if (w.is_part()) {
      w.put_part(r, d, x);
    } else {
      const int t = r / w.n_rep;
      gstore(w.out_row(t, r - t * w.n_rep) + 4 * d, x * lds_load<float>(lds + C::L_ML + r * 4));
    }
  }
}

}  // namespace mi
