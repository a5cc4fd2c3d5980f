// tree_wide_rows.h -- a tile of up to 128 query rows of one KV head over a range of keys
// (tree_wide.hip has how, tree.hip the mathematics).
//
// What the rows and keys are is W's matter (WideWork of tree_wide.hip: a run of
// cache rows; paged_attn.hip: pages):
//   thread(): threadIdx.x;
//   n_past, n_kv, row0, rows, n_rep, scale_log2e, key_begin, key_end (whole tiles
//     but for the last);
//   at_tile(key0): the tile that is fetched next; none(): of the tile fetched
//     last, which 16 rows have no page (their keys are NaN);
//   Rows(w, which, key0): descriptors of its K (which 0) or V rows by runs of 16,
//     which read zeros past the last valid one, and a row's offset;
//   Scale(w, of K, group).at(w, key0, key): 8-bit caches: a key's scale;
//   v_row, v_scale(key); visible(token, key0): which of 32 keys a query sees;
//   q_row, out_row(token, head of the group);
//   is_part(): the result is one part of the rows' keys: put_sums, put_part take it,
//     or (kJoins) join, which every wave calls.
#pragma once

#include "tree_common.h"

namespace mi {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Lane i of 16 names four f16 values of row i / 4, the (i % 4)th four of 16; it
// receives value i of the 16 of all four rows. (A plain function: in a kernel
// template the host pass rejects the builtin.)
__device__ inline u32x2 lds_transposed(const lds_t* p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
}

// The exponents of F32 rows: 2^-e times the row's largest lies in [2^14, 2^15)
// (below it for a row without a normal number, whose values 2^-e times are exact).
__device__ inline int row_exponent(float most) { return (int)(__builtin_bit_cast(unsigned, most) >> 23) - 127 - 14; }
// V's: the probabilities of a row are relative to what includes e (move_ref), and
// their sum has to stay in float's range, so there e counts as -90 at least. Rows
// below that still take a smaller e, as the products p 2^e have 2^9 to spare before
// their pairs are less exact than 2^-22; values below 2^-102 are then at most
// 2^-124 off, as a probability times one is.
constexpr int kLeastVExponent = -99, kLeastRefExponent = -90;

// Maximum over aligned groups of N = 8 or 16 lanes.
template <int N>
__device__ inline float max_lanes(float x) {
  x = fmaxf(x, dpp_mov<0xB1>(x));   // quad_perm [1,0,3,2]
  x = fmaxf(x, dpp_mov<0x4E>(x));   // quad_perm [2,3,0,1]
  x = fmaxf(x, dpp_mov<0x141>(x));  // row_half_mirror
  if constexpr (N == 16) x = fmaxf(x, dpp_mov<0x140>(x));  // row_mirror
  return x;
}

}  // namespace

template <int D, typename KT>
struct WideCfg {
  static constexpr int ELT = (int)sizeof(KT);
  static constexpr bool Q8 = ELT == 1, F32 = ELT == 4;
  static constexpr int NDB = D / 32;
  static constexpr int ROWS = 32 * kTreeWaves;
  static constexpr int TK = 4096 / D;            // keys per tile
  static constexpr int SUB = TK / 32;            // 32-key blocks of a tile
  static constexpr int NSLOT = D / 8;            // 16-byte slots per LDS row
  static constexpr int PER = 4096 / 8 / (kTreeWaves * kWave);  // slots a thread fetches of K, and of V
  static constexpr int PL = F32 ? 2 : 1;         // f16 planes of a tile
  static constexpr int PLANE = 8192;             // bytes of one
  static constexpr int TILE = PL * PLANE;
  static constexpr int L_K = 0, L_V = 2 * TILE;  // two buffers each
  // What goes with a tile's rows, per buffer: K's scales (8-bit: f16
  // [NDB][TK]; F32: exponents, int [TK]), V's factors (float [TK]) and their
  // exponents (f16 [TK]).
  static constexpr int L_SC = 4 * TILE;
  static constexpr int SC_K = 0, SC_V = Q8 ? NDB * TK * 2 : TK * 4, SC_E = SC_V + TK * 4, SC = SC_E + TK * 2;
  // Per buffer and wave: the last tile in which the wave fetched values that are not
  // finite. Each wave sets up and writes its own words, in order; the others read
  // them behind the barrier that ends the fetch.
  static constexpr int L_NF = L_SC + (ELT == 2 ? 0 : 2 * SC);
  static constexpr int NF = 4 * kTreeWaves;  // bytes of a buffer's
  static constexpr int LDS = L_NF + 2 * NF;
  static_assert(L_NF % 16 == 0, "a buffer's words are read at once");
  // F32 tiles at head_dim 128 take more registers than two workgroups per CU
  // leave each other.
  static constexpr int WAVES_PER_SIMD = D == 128 && F32 ? 1 : 2;
};

template <int D, typename KT, typename W>
__device__ __forceinline__ void tree_wide_rows(W& w, lds_t* const lds) {
  typedef WideCfg<D, KT> C;
  constexpr int NDB = C::NDB, ELT = C::ELT, TK = C::TK, SUB = C::SUB, NSLOT = C::NSLOT, PER = C::PER;
  constexpr int PL = C::PL, PLANE = C::PLANE;
  constexpr bool Q8 = C::Q8, F32 = C::F32;
  constexpr int THREADS = kTreeWaves * kWave;
  const int tid = w.thread(), lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int c = lane & 31, kh = lane >> 5;

  // ---- fetching a tile --------------------------------------------------------
  // Thread t takes slots t and t + 256 of the tile's rows (a row's slots are in
  // consecutive threads); rows past the last valid one read zeros.
  const int key_begin = w.key_begin, key_end = w.key_end;
  const bool active = w.row0 + 32 * wave < w.rows;  // the wave has rows
  constexpr int WORDS = 8 * ELT / 4;  // of 8 values
  unsigned kw[PER][WORDS], vw[PER][WORDS], scw = 0;
  // 8-bit: thread t's scale of a tile: the K scales (key t / NDB, group t % NDB),
  // then the V scales. Every thread loads one (those behind the last scale that
  // of key 0, not stored) from a row that is there.
  const bool sc_k = tid < TK * NDB, sc_v = !sc_k && tid < TK * (NDB + 1);
  const int sc_key = sc_k ? tid / NDB : sc_v ? tid - TK * NDB : 0;
  const typename W::Scale sc_src(w, sc_k, tid % NDB);
  auto fetch_rows = [&](int which, int key0, unsigned (&words)[PER][WORDS]) __attribute__((always_inline)) {
    const typename W::Rows src(w, which, key0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const unsigned t = (unsigned)(tid + THREADS * i);
      // (a wave's rows lie in one run of 16)
      const int run = (wave * (kWave / NSLOT) + THREADS / NSLOT * i) / 16;
      const rsrc_t r = src.rows(run);
      const unsigned at = src.row_at(t / NSLOT, run) + 8 * ELT * (t % NSLOT);
      if constexpr (Q8) {
        const u32x2 a = buf_b64(r, at);
        words[i][0] = a[0];
        words[i][1] = a[1];
      } else {
#pragma unroll
        for (int q = 0; q < WORDS / 4; ++q) {
          const u32x4 a = buf_b128(r, at + 16 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) words[i][4 * q + j] = a[j];
        }
      }
    }
  };
  auto fetch = [&](int key0) __attribute__((always_inline)) {
    w.at_tile(key0);
    fetch_rows(0, key0, kw);
    fetch_rows(1, key0, vw);
    if constexpr (Q8) scw = gload<unsigned short>(sc_src.at(w, key0, sc_key));
  };
  // Eight values as f16 in PL planes: an 8-bit value v as v 2^-10 (bytes_f16), a
  // float times 2^-e as a pair.
  auto widen = [](const unsigned (&w)[WORDS], int e, u32x4 (&out)[PL]) __attribute__((always_inline)) {
    if constexpr (Q8) {
      const unsigned a = w[0] ^ 0x80808080u, b = w[1] ^ 0x80808080u;
      const f16x2 x0 = bytes_f16<0, 1>(a, a), x1 = bytes_f16<2, 3>(a, a), x2 = bytes_f16<0, 1>(b, b),
                  x3 = bytes_f16<2, 3>(b, b);
      out[0] = u32x4{__builtin_bit_cast(unsigned, x0), __builtin_bit_cast(unsigned, x1), __builtin_bit_cast(unsigned, x2),
                     __builtin_bit_cast(unsigned, x3)};
    } else if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f16x2 hi, lo;
        split2(ldexpf(__builtin_bit_cast(float, w[2 * j]), -e), ldexpf(__builtin_bit_cast(float, w[2 * j + 1]), -e), hi, lo);
        out[0][j] = __builtin_bit_cast(unsigned, hi);
        out[1][j] = __builtin_bit_cast(unsigned, lo);
      }
    } else {
      out[0] = u32x4{w[0], w[1], w[2], w[3]};
    }
  };
  // The largest finite magnitude of a float row: over the NSLOT threads that
  // hold it.
  auto row_most = [](const unsigned (&w)[WORDS]) __attribute__((always_inline)) {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < WORDS; j += 2)
      most = __builtin_elementwise_maximum(__builtin_elementwise_maximum(most, fabsf(__builtin_bit_cast(float, w[j]))),
                                           fabsf(__builtin_bit_cast(float, w[j + 1])));
    if (__builtin_amdgcn_ballot_w64(!(most < INFINITY)) != 0ull) {
      most = 0.f;
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        const float x = fabsf(__builtin_bit_cast(float, w[j]));
        most = fmaxf(most, x < INFINITY ? x : 0.f);
      }
    }
    return max_lanes<NSLOT>(most);
  };
  constexpr int VSWZ = NSLOT >= 16 ? 3 : 1;  // rows of 128 bytes: two of them span the banks
  lds_t* const nf = lds + C::L_NF + 4 * wave;  // the wave's word of buffer 0
  // In a tile that some rows do not see, V values (8-bit: scales) that are not
  // finite become zeros, since a masked key's probability of 0 times them would
  // not be 0, and the tile is marked for the rows that do see them.
  auto put = [&](int buf, int key0) __attribute__((always_inline)) {
    const bool masked = key0 + TK > w.n_past;
    lds_t* const sc = lds + C::L_SC + buf * C::SC;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = (tid + THREADS * i) / NSLOT, s = (tid + THREADS * i) % NSLOT;
      u32x4 x[PL];
      int e = 0;
      if constexpr (F32) {
        e = row_exponent(row_most(kw[i]));
        lds_store<int>(sc + C::SC_K + 4 * r, e);  // (by all of the row's threads)
      }
      widen(kw[i], e, x);
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
        lds_store<u32x4>(lds + C::L_K + buf * C::TILE + pl * PLANE + r * (2 * D) + 16 * (s ^ swz<NSLOT>(r)), x[pl]);
      if constexpr (F32) {
        e = max(row_exponent(row_most(vw[i])), kLeastVExponent);
        lds_store<float>(sc + C::SC_V + 4 * r, ldexpf(1.f, e));
        lds_store<_Float16>(sc + C::SC_E + 2 * r, (_Float16)max(e, kLeastRefExponent));
      }
      if constexpr (!Q8) {
        if (masked) {
          unsigned any = 0u;
#pragma unroll
          for (int j = 0; j < WORDS; ++j) {
            if constexpr (F32) {
              const bool b = not_finite(__builtin_bit_cast(float, vw[i][j]));
              any |= b;
              vw[i][j] = b ? 0u : vw[i][j];
            } else {
              const unsigned b = not_finite2(vw[i][j]);
              any |= b;
              vw[i][j] &= (b & 1u ? 0u : 0xffffu) | (b & 2u ? 0u : 0xffff0000u);
            }
          }
          if (any) lds_store<int>(nf + C::NF * buf, key0);
        }
      }
      widen(vw[i], e, x);
#pragma unroll
      for (int pl = 0; pl < PL; ++pl)
        lds_store<u32x4>(lds + C::L_V + buf * C::TILE + pl * PLANE + r * (2 * D) + 16 * (s ^ 4 * (r & VSWZ)), x[pl]);
    }
    if constexpr (Q8) {
      if (sc_k) lds_store<unsigned short>(sc + C::SC_K + ((tid % NDB) * TK + sc_key) * 2, (unsigned short)scw);
      if (sc_v) {
        float v = (float)__builtin_bit_cast(_Float16, (unsigned short)scw);
        const bool finite = v < INFINITY;  // (scales are not negative)
        if (masked && !finite) {
          lds_store<int>(nf + C::NF * buf, key0);
          v = 0.f;
        }
        lds_store<float>(sc + C::SC_V + 4 * sc_key, v);
        lds_store<_Float16>(sc + C::SC_E + 2 * sc_key, (_Float16)scale_exponent(finite ? v : 0.f));
      }
    }
  };
  if (lane < 2) lds_store<int>(nf + C::NF * lane, -1);
  if (key_begin < key_end) fetch(key_begin);

  // ---- queries: row c of the wave's 32, dims 16 s + 8 kh + j of step s -----------
  const int r = w.row0 + 32 * wave + c;
  const bool valid = r < w.rows;
  const int token = valid ? r / w.n_rep : 0;
  const int h = valid ? r - token * w.n_rep : 0;
  f16x8 qh[D / 16], ql[D / 16];
  int qexp = 0;  // the scores' exponent: undoes what the queries are scaled by
  {
    const char* const qp = w.q_row(token, h);
    float x[D / 2], amax = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 v = gload<f32x4>(qp + 4 * (16 * s + 8 * kh + 4 * e));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[8 * s + 4 * e + j] = valid ? v[j] * w.scale_log2e : 0.f;
          amax = fmaxf(amax, fabsf(x[8 * s + 4 * e + j]));
        }
      }
    if (key_begin < key_end) put(0, key_begin);  // (under the queries' loads)
    amax = max32(amax);
    if (amax > 0.f && amax < INFINITY) qexp = F32 ? ilogbf(amax) - 13 : max(ilogbf(amax) - 13, -100);
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
  // (F32: the exponents are applied to the scores, where either alone could
  // leave float's range)
  const float unscale = F32 ? 1.f : ldexpf(Q8 ? kByteUnscale : 1.f, qexp);
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

  // none: bit i: keys 16 i .. of the tile have no page
  auto compute = [&](int buf, int key0, unsigned none) __attribute__((always_inline)) {
    const bool masked = key0 + TK > w.n_past || none != 0u;
    const lds_t* const sc = lds + C::L_SC + buf * C::SC;  // the lane's keys: 8 q + 4 kh + j of each 32
    // ---- S^T = K . Q^T: groups of KG steps, 8-bit: the 32 dims of one scale --------
    constexpr int KG = 2, NG = D / 16 / KG;
    floatx16 s[SUB];
    f16x8 kf[2][KG][PL];
    auto read_k = [&](int i) __attribute__((always_inline)) {
      const int u = i / NG, g0 = i % NG;
#pragma unroll
      for (int e = 0; e < KG; ++e)
#pragma unroll
        for (int pl = 0; pl < PL; ++pl)
          kf[i & 1][e][pl] = lds_load<f16x8>(krow + buf * C::TILE + pl * PLANE + u * 32 * (2 * D) +
                                             16 * ((2 * (KG * g0 + e) + kh) ^ kx));
    };
    f16x4 ksc[2][4];
    auto read_ksc = [&](int i) __attribute__((always_inline)) {
      if constexpr (Q8) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          ksc[i & 1][q] = lds_load<f16x4>(sc + C::SC_K + ((i % NG) * TK + 32 * (i / NG) + 8 * q + 4 * kh) * 2);
      }
    };
    read_k(0);
    read_ksc(0);
    floatx16 part[2];
#pragma unroll
    for (int i = 0; i < SUB * NG; ++i) {
      if (i + 1 < SUB * NG) {
        read_k(i + 1);
        read_ksc(i + 1);
      }
      __builtin_amdgcn_sched_barrier(0);
      const int u = i / NG, g0 = i % NG;
      floatx16 acc = Q8 || g0 == 0 ? (floatx16)(0.f) : s[u];
#pragma unroll
      for (int e = 0; e < KG; ++e) {
        const int st = KG * g0 + e;
        if constexpr (F32) acc = mfma_f16(kf[i & 1][e][1], qh[st], acc);
        acc = mfma_f16(kf[i & 1][e][0], ql[st], acc);
        acc = mfma_f16(kf[i & 1][e][0], qh[st], acc);
      }
      if constexpr (Q8) {
        // The scale products wait for the group's own matrix products. (Two parts in
        // turn, of which one is in use: with one the compiler assigns registers
        // otherwise, 1024 tokens after 1337, 14/2 heads of 64: 34.6 us instead of 33.9.)
        part[i & 1] = acc;
        auto scale = [&](int k) __attribute__((always_inline)) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              s[k / NG][4 * q + j] = fmaf(part[k & 1][4 * q + j], (float)ksc[k & 1][q][j], k % NG == 0 ? 0.f : s[k / NG][4 * q + j]);
        };
        scale(i);
      } else {
        s[u] = acc;
      }
    }
    // ---- V's operands of 16 keys, one group ahead --------------------------------
    f16x8 vf[2][NDB][PL];
    auto read_v = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int pl = 0; pl < PL; ++pl) {
          const lds_t* const at = vrow + buf * C::TILE + pl * PLANE + 16 * i * (2 * D) + 16 * ((4 * db + vs) ^ vx);
          const u32x2 a = lds_transposed(at), b = lds_transposed(at + 8 * (2 * D));
          vf[i & 1][db][pl] = __builtin_bit_cast(f16x8, u32x4{a[0], a[1], b[0], b[1]});
        }
    };
    read_v(0);
    if constexpr (F32) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const i32x4 e = lds_load<i32x4>(sc + C::SC_K + (32 * u + 8 * q + 4 * kh) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][4 * q + j] = ldexpf(s[u][4 * q + j], e[j] + qexp);
        }
    }
    // ---- mask -------------------------------------------------------------------
    unsigned vis[SUB];
    if (masked) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        vis[u] = w.visible(token, key0 + 32 * u);
        const unsigned mine = vis[u] >> (4 * kh);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[u][e] = mine >> (8 * (e >> 2) + (e & 3)) & 1u ? (none >> (2 * u + (e >> 3)) & 1u ? NAN : s[u][e]) : -INFINITY;
      }
    }
    // ---- softmax, relative to ref -----------------------------------------------
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      if constexpr (ELT == 2) {
        top = max16(s[u], top);
      } else {  // of the probability times the V row's factor
        floatx16 x;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f16x4 e = lds_load<f16x4>(sc + C::SC_E + (32 * u + 8 * q + 4 * kh) * 2);
#pragma unroll
          for (int j = 0; j < 4; ++j) x[4 * q + j] = fmaf(s[u][4 * q + j], unscale, (float)e[j]);
        }
        top = max16(x, top);
      }
    }
    top = max32(top) * (ELT == 2 ? unscale : 1.f);
    const float alpha = move_ref(ref, top);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0ull) {
      l *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= alpha;
    }
    const float at = ref == -INFINITY ? 0.f : ref;
    // ---- probabilities and O^T += V^T . P^T, 16 keys at a time ---------------------
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * SUB; ++i) {
      const int u = i / 2, half = i % 2;
      if (i + 1 < 2 * SUB) read_v(i + 1);
      float pv[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        f32x4 f = {1.f, 1.f, 1.f, 1.f};
        if constexpr (ELT != 2) f = lds_load<f32x4>(sc + C::SC_V + (16 * i + 8 * q + 4 * kh) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = s[u][8 * half + 4 * q + j];
          const float e = fast_exp2(F32 ? x - at : fmaf(x, unscale, -at));
          sum[j] += e;
          pv[4 * q + j] = ELT == 2 ? e : e * f[j];
        }
      }
      f16x8 ph, pl;
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        f16x2 hi, lo;
        split2(pv[j], pv[j + 1], hi, lo);
        ph[j] = hi[0];
        ph[j + 1] = hi[1];
        pl[j] = lo[0];
        pl[j + 1] = lo[1];
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        if constexpr (F32) o[db] = mfma_f16(vf[i & 1][db][1], ph, o[db]);
        o[db] = mfma_f16(vf[i & 1][db][0], pl, o[db]);
        o[db] = mfma_f16(vf[i & 1][db][0], ph, o[db]);
      }
    }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    // rows that see a value which is not finite get NaN in its dim (8-bit: in all)
    static_assert(kTreeWaves == 4, "a word for each wave");
    bool marked = false;
    if (masked) {
      const i32x4 m = lds_load<i32x4>(lds + C::L_NF + C::NF * buf);
      marked = m[0] == key0 || m[1] == key0 || m[2] == key0 || m[3] == key0;
    }
    if (marked) {
      const int n = min(w.n_kv - key0, TK);
      for (int t = 0; t < n; ++t) {
        unsigned word = vis[0];
        if constexpr (SUB > 1) word = t < 32 ? vis[0] : vis[1];
        const bool sees = word >> (t & 31) & 1u;
        if constexpr (Q8) {
          const unsigned x = gload<unsigned short>(w.v_scale(key0 + t));
          if (sees && not_finite2(x) != 0u) l = NAN;
        } else {
          const char* const vr = w.v_row(key0 + t);
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const char* const a = vr + ELT * (32 * db + 8 * (e >> 2) + 4 * kh + (e & 3));
              const bool bad = F32 ? not_finite(gload<float>(a)) : not_finite2(gload<unsigned short>(a)) != 0u;
              if (sees && bad) o[db][e] = NAN;
            }
        }
      }
    }
  };

  __syncthreads();
  int buf = 0;
  for (int key0 = key_begin; key0 < key_end; key0 += TK, buf ^= 1) {
    const int next = key0 + TK;
    const unsigned none = w.none();
    if (next < key_end) fetch(next);
    if (active) compute(buf, key0, none);
    if (next < key_end) put(buf ^ 1, next);
    __syncthreads();
  }

  // ---- the wave's rows ------------------------------------------------------------
  const float lt = sum32(l);
  constexpr float unit_o = Q8 ? kByteUnscale : 1.f;  // of the values' 2^-10
  if constexpr (W::kJoins) {
    if (w.is_part()) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= unit_o;
      w.join(o, ref, lt, active);
      return;
    }
  }
  if (!active) return;
  if (w.is_part()) {
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        w.put_part(32 * wave + c, 32 * db + 8 * q + 4 * kh,
                   f32x4{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]} * unit_o);
    if (kh == 0) w.put_sums(32 * wave + c, ref, lt);
    return;
  }
  if (!valid) return;
  const float inv = ref == -INFINITY ? 0.f : unit_o / lt;
  char* const out = w.out_row(token, h);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      gstore(out + 4 * (32 * db + 8 * q + 4 * kh),
             f32x4{o[db][4 * q], o[db][4 * q + 1], o[db][4 * q + 2], o[db][4 * q + 3]} * inv);
}

}  // namespace mi
