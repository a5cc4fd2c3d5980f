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
#include "tree_common.h"

namespace mi {

namespace {

constexpr int kTreeRows = 32;  // rows of this kernel's records

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

template <int D, typename KT, int RT>
__global__ __launch_bounds__(kTreeWaves* kWave, (TreeCfg<D, KT, RT>::WAVES_PER_SIMD)) void tree_kernel(const TreeParams p) {
  typedef TreeCfg<D, KT, RT> C;
  constexpr int NB = C::NB, NE = C::NE, ROWS = C::ROWS, ELT = C::ELT, KB = C::KB, KW = C::KW, VW = C::VW;
  constexpr bool Q8 = C::Q8, F32 = C::F32;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  lds_t* const lds = (lds_t*)lds_raw;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, q4 = lane >> 4;

  // Workgroup -> (KV head, split) unit; units go to the 8 XCDs in turn. (One row
  // tile: calls of more rows take the wide kernel.)
  const TreeItem& it = p.item[blockIdx.y];
  const int n_split = it.n_split;
  const int unit = (blockIdx.x / 8) * 8 + (int)((blockIdx.x - it.xcd0) % 8);
  if (unit >= p.n_head_kv * n_split) return;
  const int g = unit / n_split, sp = unit % n_split;
  const int n_past = it.n_past, n_kv = n_past + it.n_tokens;
  const int rows = it.n_tokens * p.n_rep;
  const int tile0 = sp * it.tiles_per_split;
  const int tile1 = min(tile0 + it.tiles_per_split, (n_kv + kTreeTile - 1) / kTreeTile);

  // ---- loads of a key tile --------------------------------------------------
  // The descriptors start at the tile's first row (64-bit), so a cache of any
  // length is addressed, and end after its last valid row: rows past n_kv
  // read zeros.
  const char* const kbase = it.k + (int64_t)g * p.k_s1;
  const char* const vbase = it.v + (int64_t)g * p.v_s1;
  const int ks2 = (int)p.k_s2, vs2 = (int)p.v_s2;
  unsigned kw[2][KB][KW], vw[8][VW], ksc = 0, vsc = 0;
  const unsigned ko = (unsigned)(c * ks2 + 4 * KW * q4);
  const unsigned vo = (unsigned)(4 * q4 * vs2 + c * NE * ELT);
  lds_t* const sc_lds = lds + wave * ROWS * C::XS * 4;
  const int c32 = lane & 31, half = lane >> 5;
  auto load_k = [&](int tile) __attribute__((always_inline)) {
    const int key0 = tile * kTreeTile;
    const int n = min(n_kv - key0, kTreeTile);
    const rsrc_t r = make_rsrc(kbase + (int64_t)key0 * ks2, (unsigned)((n - 1) * ks2 + D * ELT));
#pragma unroll
    for (int hk = 0; hk < 2; ++hk)
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const unsigned at = ko + (unsigned)(16 * hk * ks2) + 16 * KW * b;
        if constexpr (KW == 4) {
          const u32x4 x = buf_b128(r, at);
#pragma unroll
          for (int j = 0; j < 4; ++j) kw[hk][b][j] = x[j];
        } else {
          const u32x2 x = buf_b64(r, at);
          kw[hk][b][0] = x[0];
          kw[hk][b][1] = x[1];
        }
      }
    if constexpr (Q8) {
      // the scales of key lane % 32: each half of the wave takes half of the K row's
      const int64_t at = (int64_t)key0 * p.n_head_kv + g;
      const rsrc_t rk = make_rsrc(it.k_scale + at * (2 * NB), (unsigned)((n - 1) * p.n_head_kv * 2 * NB + 2 * NB));
      ksc = NB == 4 ? buf_b32(rk, (unsigned)(c32 * p.n_head_kv * 8 + 4 * half)) : buf_b16(rk, (unsigned)(c32 * p.n_head_kv * 4 + 2 * half));
      const rsrc_t rv = make_rsrc(it.v_scale + at * 2, (unsigned)((n - 1) * p.n_head_kv * 2 + 2));
      vsc = buf_b16(rv, (unsigned)(c32 * p.n_head_kv * 2));
    }
  };
  auto load_v = [&](int tile) __attribute__((always_inline)) {
    const int key0 = tile * kTreeTile;
    const int n = min(n_kv - key0, kTreeTile);
    const rsrc_t r = make_rsrc(vbase + (int64_t)key0 * vs2, (unsigned)((n - 1) * vs2 + D * ELT));
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // keys 16 (j / 4) + 4 q4 + j % 4
      const unsigned at = vo + (unsigned)((16 * (j / 4) + j % 4) * vs2);
      if constexpr (VW >= 4) {
#pragma unroll
        for (int w = 0; w < VW; w += 4) {
          const u32x4 x = buf_b128(r, at + 4 * w);
#pragma unroll
          for (int i = 0; i < 4; ++i) vw[j][w + i] = x[i];
        }
      } else if constexpr (VW == 2) {
        const u32x2 x = buf_b64(r, at);
        vw[j][0] = x[0];
        vw[j][1] = x[1];
      } else {
        vw[j][0] = buf_b32(r, at);
      }
    }
  };
  int tile = tile0 + wave;
  if (tile < tile1) {
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
    const bool valid = r < rows;
    token[i] = valid ? r / p.n_rep : 0;
    unscale[i] = 1.f;
    const int h = g * p.n_rep + (valid ? r - token[i] * p.n_rep : 0);
    const char* const qp = reinterpret_cast<const char*>(it.q) + (int64_t)token[i] * p.q_s2 + (int64_t)h * p.q_s1;
    if constexpr (F32) {
#pragma unroll
      for (int s = 0; s < D / 4; s += 4) {  // dims 4 s + 4 q4 + j
        const f32x4 x = gload<f32x4>(qp + 4 * (4 * s + 4 * q4));
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[i][s + j] = valid ? x[j] * p.scale_log2e : 0.f;
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
            x[8 * b + 4 * e + j] = valid ? v[j] * p.scale_log2e : 0.f;
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
    if (next < tile1) load_k(next);

    // ---- mask -----------------------------------------------------------------
    // bit 4 hk + j of vis: the row sees the lane's key 16 hk + 4 q4 + j
    unsigned row_vis[RT], vis[RT];
    const bool masked = key0 + kTreeTile > n_past;  // a tile of drafted keys
    if (masked) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        row_vis[i] = visible_bits(it, token[i], key0);
        vis[i] = slots_of(row_vis[i], q4);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[i][e] = vis[i] >> e & 1u ? s[i][e] : -INFINITY;
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
          for (int w = 0; w < VW; ++w) {
            if constexpr (F32) {
              if (not_finite(__builtin_bit_cast(float, vw[j][w]))) {
                nf[w] |= 1u << j;
                vw[j][w] = 0u;
              }
            } else {
              const unsigned b = not_finite2(vw[j][w]);
              nf[2 * w] |= (b & 1u) << j;
              nf[2 * w + 1] |= (b >> 1) << j;
              vw[j][w] &= (b & 1u ? 0u : 0xffffu) | (b & 2u ? 0u : 0xffff0000u);
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
          for (int w = 0; w < VW; ++w) vw[j][w] ^= 0x80808080u;
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
    for (int w = 0; w < kTreeWaves; ++w) {
      ml[w] = lds_load<f32x2>(lds + C::L_ML + ((w * ROWS + 16 * i + c) * 2) * 4);
      mt[i] = fmaxf(mt[i], ml[w][0]);
    }
    const float mu = mt[i] == -INFINITY ? 0.f : mt[i];
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) lt[i] += ml[w][1] * fast_exp2(ml[w][0] - mu);
    const float wt = fast_exp2(ref[i] - mu) * unit_o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int db = 0; db < NE; db += 4)
        lds_store<f32x4>(lds + ((wave * ROWS + 16 * i + c) * C::XS + NE * (4 * q4 + j) + db) * 4,
                         f32x4{o[i][db][j], o[i][db + 1][j], o[i][db + 2][j], o[i][db + 3][j]} * wt);
  }
  __syncthreads();
  float* const rec = p.rec + ((int64_t)it.rec0 + (int64_t)g * n_split + sp) * (kTreeRows * (D + 2));
  if (n_split > 1) {
    if (wave == 0 && q4 == 0) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        rec[kTreeRows * D + 16 * i + c] = mt[i];
        rec[kTreeRows * D + kTreeRows + 16 * i + c] = lt[i];
      }
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
    const int idx = e + threadIdx.x, r = idx / (D / 4), d = 4 * (idx % (D / 4));
    if (r >= rows) continue;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) x += lds_load<f32x4>(lds + ((w * ROWS + r) * C::XS + d) * 4);
    if (n_split > 1) {
      put_record(rec + tree_record_at(D, r, d), x);
    } else {
      const int t = r / p.n_rep, h = g * p.n_rep + r - t * p.n_rep;
      gstore(reinterpret_cast<char*>(it.out) + (int64_t)t * p.o_s2 + (int64_t)h * p.o_s1 + 4 * d,
             x * lds_load<float>(lds + C::L_ML + r * 4));
    }
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
