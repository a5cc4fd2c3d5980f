// paged_attn.hip -- attention of each sequence's new tokens over its pages: one, a
// few or thousands per sequence, in one call, with all lengths read on the device.
//
// The mathematics and the products are tree.hip's: query j of a sequence sees the
// positions up to its own, its output is sum_t p_t v_t / sum_t p_t with a running
// reference. Sequences of few query rows per KV head go through tree_rows.h, others
// in row tiles of 128 through tree_wide_rows.h.
//
// Work. The host does not know the lengths, so every workgroup finds its share
// itself: the key tiles of all units (sequence, KV head, row tile) of a kind form one line,
// of which workgroup w takes tiles w * per .. (w + 1) * per - 1 whatever they belong
// to: whole units, the end of one, the start of another. So workgroups have the
// same work however ragged the lengths are. A causal unit has the tiles that its
// rows see; to find the unit at a place of the line without adding up row tiles,
// row tile r of n lies beside row tile n - 1 - r: together they have the same number
// of tiles, but for a few that are empty. Each wave reads the lengths of 64
// sequences at a time and adds up their tiles by itself, a round of loads and six
// additions for each 64, in up to three passes (the later ones have the first 64
// sequences' lengths in LDS), then goes on from the first ones to its share.
//
// Parts. A unit that lies in several workgroups' shares leaves a record from each
// (its first part in slot 2 w + 1 of the workgroup w where it begins, the others in
// slot 2 w), and the last of them to arrive joins the records in their order, so
// the bits do not depend on who that is. Records pass between XCDs: they are
// written and read with agent-scope accesses, which go past the L2s.
//
// Pages. 16 keys lie in one page at least, so a tile of 32 has two page numbers,
// the same for the whole wave: the rows' descriptors are in scalar registers as
// for one run of rows. A lane holds the page number of 16 keys, a wave those of
// 1024, the next 1024 on their way.
//
// Bound: single tokens by the cache's bytes (64 over 8192 keys, 28/4 heads of 128, 8-bit:
// 467 MB in 107 us, 6.9 TB/s for a read of nothing else takes 68, and widening the
// bytes the rest), long chunks by the matrix pipe (2048 tokens after 6000, F16: 424 us,
// two products at a large matrix product's rate 363). Between them what a share costs
// besides its tiles is what counts: about 6 us from the launch to the first tile
// (lengths, pages, rows: three loads one after the other), and 8 to 10 for records to
// go through memory and be joined, which short chunks pay twice (1000 tokens from
// nothing, 28/4 heads of 128, F16: 52 us in a row of calls, 13 of them products).
#include <algorithm>
#include <type_traits>

#include "attn_common.h"
#include "kernels.h"
#include "tree_rows.h"
#include "tree_wide_rows.h"

namespace mi {

namespace {

constexpr int kRun = 16;  // keys that share a page at least

// threadIdx.x as a value of its own: what is formed from it is formed where it is
// used, and not kept in registers across the units of a workgroup (which spill
// for it: 1000 tokens after 1337 among 31 single tokens over 2667 to 4000 keys, 28/4
// heads of 128, F16 189 us, so 122). Of the 18 kernels one still spills a register,
// the mixed one of 8-bit caches and heads of 128.
__device__ __forceinline__ int thread_here() {
  int t = (int)threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// x plus those of the lanes below.
__device__ inline unsigned wave_scan(unsigned x) {
  auto add = [&](auto ctrl, auto rows) {
    x += (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});  // row_shr:1
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15 to rows 1 and 3
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31 to rows 2 and 3
  return x;
}

// A sequence's queries and keys, clamped to what is there.
struct SeqLens {
  int q0;      // its first row of q
  int n_new;   // its queries (up to max_new)
  int n_past;  // the first query's position (negative: the first queries see nothing)
  int n_seen;  // positions that its last query sees
};
__device__ inline SeqLens seq_lens(const PagedAttn& p, int i) {
  SeqLens s{0, 0, 0, 0};
  if (i < p.n_seq) {
    // (the end at the start at least: the difference of any two numbers may leave 32 bits)
    const int a = min(max(gload<int>(p.q_off + i), 0), p.n_tokens), b = min(max(gload<int>(p.q_off + i + 1), a), p.n_tokens);
    const int n_kv = min(max(gload<int>(p.n_kv + i), 0), p.max_kv);
    s.q0 = a;
    s.n_new = min(b - a, p.max_new);
    s.n_past = n_kv - (b - a);
    s.n_seen = max(s.n_past + s.n_new, 0);
  }
  return s;
}

__device__ inline unsigned padded(unsigned x, unsigned pad) { return pad > 1u ? (x + pad - 1u) / pad * pad : x; }

// Units of a sequence on the line, for row tiles of ROWS rows and key tiles of TK.
template <int ROWS, int TK>
struct Units {
  int n_rt, n_past, n_new, n_seen, n_rep;
  unsigned pair;  // tiles of a pair of row tiles, a few empty ones among them

  __device__ inline Units(const SeqLens& s, int rep) : n_past(s.n_past), n_new(s.n_new), n_seen(s.n_seen), n_rep(rep) {
    n_rt = (s.n_new * rep + ROWS - 1) / ROWS;
    // The two row tiles see at most 2 n_past + ((n_rt + 1) ROWS - 2) / n_rep + 2 keys.
    // (and twice what the last one sees: where queries are more than positions, those that
    // see nothing would fill the line, beyond what it is counted in)
    const unsigned keys = 2u * (unsigned)max(s.n_past, 0) + ((unsigned)(n_rt + 1) * ROWS - 2u) / (unsigned)rep + 2u;
    pair = min((keys + 2 * TK - 2) / TK, 2u * (((unsigned)max(s.n_seen, 1) + TK - 1) / TK));
  }
  // Key tiles of row tile rt, one at least (rows without a key are written too).
  __device__ inline int tiles(int rt) const {
    const int last = min(((rt + 1) * ROWS - 1) / n_rep, n_new - 1);
    return (max(min(n_past + last + 1, n_seen), 1) + TK - 1) / TK;
  }
  __device__ inline int count() const { return n_rt; }  // of a head
  // Places of a head's units on the line: whole units, or their tiles; pairs and the
  // middle row tile in multiples of `pad`, so that no share of that size holds two.
  __device__ inline unsigned per_head(bool whole, unsigned pad) const {
    if (whole) return (unsigned)n_rt;
    return (unsigned)(n_rt / 2) * padded(pair, pad) + (n_rt & 1 ? padded((unsigned)tiles(n_rt / 2), pad) : 0u);
  }
  // The row tile and key tile at a place; false behind the last one, then with what
  // is left of the empty places.
  __device__ inline bool find(unsigned off, bool whole, unsigned pad, int& rt, int& n_tiles, int& tile, unsigned& left) const {
    tile = 0;
    if (whole) {
      rt = n_rt - 1 - (int)off;
      n_tiles = tiles(rt);
      return true;
    }
    const unsigned pairs = (unsigned)(n_rt / 2), span = padded(pair, pad), j = min(off / span, pairs);
    off -= j * span;
    rt = n_rt - 1 - (int)j;  // (the middle one, where it is alone, is both)
    n_tiles = tiles(rt);
    left = (j < pairs ? span : padded((unsigned)n_tiles, pad)) - off;
    if (j < pairs && off >= (unsigned)n_tiles) {
      off -= (unsigned)n_tiles;
      rt = (int)j;
      n_tiles = tiles(rt);
    }
    tile = (int)off;
    return off < (unsigned)n_tiles;
  }
};

// The same where all rows are one tile.
template <int TK>
struct OneUnit {
  int n_tiles_;
  __device__ inline OneUnit(const SeqLens& s, int) : n_tiles_((max(s.n_seen, 1) + TK - 1) / TK) {}
  __device__ inline int count() const { return 1; }
  __device__ inline unsigned per_head(bool whole, unsigned pad) const { return whole ? 1u : padded((unsigned)n_tiles_, pad); }
  __device__ inline bool find(unsigned off, bool whole, unsigned pad, int& rt, int& n_tiles, int& tile, unsigned& left) const {
    rt = 0;
    n_tiles = n_tiles_;
    tile = whole ? 0 : (int)off;
    left = per_head(whole, pad) - off;
    return tile < n_tiles_;
  }
};

// The pages of a sequence, as a wave reads them: RUNS runs of 16 keys per tile.
template <int RUNS>
struct Pages {
  const int* table;
  int shift, n_pages, last;  // the last run that is there
  int win, here, next;       // page numbers of runs 64 win + lane, and of the 64 behind
  int slot[RUNS];            // cache row of each run of the tile at hand
  unsigned none = 0u;        // runs without a page

  __device__ __forceinline__ Pages(const PagedAttn& p, int seq, int n_seen)
      : table(reinterpret_cast<const int*>(p.table + (int64_t)seq * p.table_nb)), shift(p.page_shift), n_pages(p.n_pages),
        last(max(n_seen - 1, 0) / kRun) {}
  __device__ __forceinline__ int read(int w) const {
    return gload<int>(table + (min(64 * w + thread_here() % kWave, last) * kRun >> shift));
  }
  __device__ __forceinline__ void start(int run) {
    win = run / 64;
    here = read(win);
    next = read(win + 1);
  }
  // Runs run .. run + RUNS - 1 (a multiple of RUNS; tiles are taken in order, 64
  // runs further at most).
  __device__ __forceinline__ void at(int run) {
    if (run / 64 != win) {
      win = run / 64;
      here = next;
      next = read(win + 1);
    }
    none = 0u;
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int page = __builtin_amdgcn_readlane(here, (run + i) & 63);
      const bool ok = (unsigned)page < (unsigned)n_pages;
      none |= ok ? 0u : 1u << i;
      slot[i] = ((ok ? page : 0) << shift) + ((run + i) * kRun & ((1 << shift) - 1));
    }
  }
  __device__ __forceinline__ int slot_of(int i) const {
    const int a = slot[0], b = slot[1], c = slot[RUNS - 2], d = slot[RUNS - 1];  // (values: not a choice of addresses)
    return i < RUNS - 2 ? (i == 0 ? a : b) : (i == RUNS - 2 ? c : d);
  }
  // Any key's row, -1 if it has none.
  __device__ __forceinline__ int row(int key) const {
    const int page = gload<int>(table + (min(key / kRun, last) * kRun >> shift));
    return (unsigned)page < (unsigned)n_pages ? (page << shift) + (key & ((1 << shift) - 1)) : -1;
  }
};

// A record: 16-byte pieces of four dims of a row, then each row's reference and sum.
// Pieces that a wave holds lie together: few rows' row by row, many rows' those of
// 32 rows side by side. Written by one XCD, read by another, so with the cache bit
// that goes past the L2s (8 bytes at a time, as atomics do, and with rows apart, a
// prompt's chunk of 1000 tokens after 1337 took 137 us, not 101).
constexpr int kSc1 = 16;
template <int D, int ROWS>
struct Record {
  static constexpr int FLOATS = ROWS * (D + 2), BYTES = FLOATS * 4;
  static __device__ __forceinline__ unsigned piece_at(int r, int d) {
    if constexpr (ROWS > 32) return (unsigned)((r / 32) * (128 * D) + (d / 4) * 512 + (r % 32) * 16);
    else return (unsigned)(r * D + d) * 4;
  }
  static __device__ __forceinline__ unsigned sums_at(int r) { return (unsigned)(ROWS * D + 2 * r) * 4; }
};
__device__ inline void shared_store4(rsrc_t r, unsigned at, f32x4 x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, at, 0, kSc1);
}
__device__ inline void shared_store2(rsrc_t r, unsigned at, f32x2 x) {
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, x), r, at, 0, kSc1);
}
__device__ inline f32x4 shared_load4(rsrc_t r, unsigned at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kSc1));
}
__device__ inline f32x2 shared_load2(rsrc_t r, unsigned at) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, kSc1));
}

// One unit's rows and the part of its key tiles that this workgroup has.
template <int D, typename KT, int ROWS>
struct UnitRows {
  static constexpr int kRows = ROWS;
  const PagedAttn& p;
  int g, q0, n_past, n_kv, rows, n_rep, row0;  // rows: of the sequence; row0: of the row tile
  float scale_log2e;
  int parts, mine;     // how many workgroups share the rows' keys, which of them this is
  float* rec;          // the record of this part
  unsigned* arrived;   // how many have left theirs
  lds_t* word;         // for the workgroup to agree on who joins

  // The records of all parts: part k's at part_at(k).
  __device__ __forceinline__ const float* first_record() const {
    return rec - (int64_t)max(2 * mine - 1, 0) * Record<D, ROWS>::FLOATS;
  }
  static __device__ __forceinline__ unsigned part_at(int k) { return (unsigned)max(2 * k - 1, 0) * Record<D, ROWS>::BYTES; }
  // Counts this part; true for the last one. Every wave's records are in memory
  // before that.
  __device__ __forceinline__ bool arrive() const {
    wait_vmem<0>();
    __syncthreads();
    if (threadIdx.x == 0) {
      const int done = (int)__hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (done == parts - 1) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      lds_store<int>(word, done == parts - 1);
    }
    __syncthreads();
    return lds_load<int>(word) != 0;
  }
  __device__ __forceinline__ int thread() const { return thread_here(); }
  __device__ __forceinline__ unsigned visible(int token, int key0) const {
    const int n = n_past + token - key0 + 1;
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
  }
  __device__ __forceinline__ const char* q_row(int token, int h) const {
    return p.q + (int64_t)(q0 + token) * p.q_s2 + (int64_t)(g * n_rep + h) * p.q_s1;
  }
  __device__ __forceinline__ char* out_row(int token, int h) const {
    return p.out + (int64_t)(q0 + token) * p.o_s2 + (int64_t)(g * n_rep + h) * p.o_s1;
  }
  __device__ __forceinline__ bool is_part() const { return parts > 1; }
  __device__ __forceinline__ rsrc_t record() const { return make_rsrc(rec, Record<D, ROWS>::BYTES); }
  __device__ __forceinline__ void put_sums(int r, float ref, float l) const {
    shared_store2(record(), Record<D, ROWS>::sums_at(r), f32x2{ref, l});
  }
  __device__ __forceinline__ void put_part(int r, int d, f32x4 x) const {
    shared_store4(record(), Record<D, ROWS>::piece_at(r, d), x);
  }
};

// tree_rows over pages.
template <int D, typename KT, int ROWS>
struct FewRows : UnitRows<D, KT, ROWS> {
  static constexpr int ELT = (int)sizeof(KT);
  int tile0, tile1, k_s2, v_s2;
  const char* kbase;
  const char* vbase;
  Pages<2> pages;

  __device__ __forceinline__ FewRows(const UnitRows<D, KT, ROWS>& u, int seq, int t0, int t1)
      : UnitRows<D, KT, ROWS>(u), tile0(t0), tile1(t1), k_s2((int)u.p.cache.s2), v_s2((int)u.p.cache.s2),
        kbase(u.p.cache.t[0] + u.g * u.p.cache.s1), vbase(u.p.cache.t[1] + u.g * u.p.cache.s1), pages(u.p, seq, u.n_kv) {
    pages.start(2 * tile0);
  }
  __device__ __forceinline__ void at_tile(int tile) { pages.at(2 * tile); }
  __device__ __forceinline__ unsigned none() const { return pages.none; }
  __device__ __forceinline__ TileRows rows_at(const char* base, int key0) const {
    TileRows t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = pages.none >> i & 1u ? 0 : min(this->n_kv - key0 - kRun * i, kRun);
      t.rows[i] = make_rsrc(base + (int64_t)pages.slot[i] * k_s2, n > 0 ? (unsigned)((n - 1) * k_s2 + D * ELT) : 0u);
      t.at[i] = 0u;
    }
    return t;
  }
  __device__ __forceinline__ TileRows k_rows(int key0) const { return rows_at(kbase, key0); }
  __device__ __forceinline__ TileRows v_rows(int key0) const { return rows_at(vbase, key0); }
  // (every row of a page is there, so the lanes past the last key read what their
  // queries do not see)
  template <int NB>
  __device__ __forceinline__ void scales(int, int c32, int half, unsigned& ksc, unsigned& vsc) const {
    const CacheView& c = this->p.cache;
    const int64_t at = (int64_t)(pages.slot_of(c32 / kRun) + c32 % kRun) * c.n_head_kv + this->g;
    if constexpr (NB == 4) ksc = gload<unsigned>(c.scale[0] + at * 8 + 4 * half);
    else ksc = gload<unsigned short>(c.scale[0] + at * 4 + 2 * half);
    vsc = gload<unsigned short>(c.scale[1] + at * 2);
  }
};

// tree_wide_rows over pages.
template <int D, typename KT>
struct ManyRows : UnitRows<D, KT, WideCfg<D, KT>::ROWS> {
  typedef UnitRows<D, KT, WideCfg<D, KT>::ROWS> Base;
  static constexpr int ELT = (int)sizeof(KT), TK = WideCfg<D, KT>::TK, NDB = D / 32, RUNS = TK / kRun;
  int key_begin, key_end;
  const char* kbase;
  const char* vbase;
  Pages<RUNS> pages;

  __device__ __forceinline__ ManyRows(const Base& u, int seq, int k0, int k1)
      : Base(u), key_begin(k0), key_end(k1), kbase(u.p.cache.t[0] + u.g * u.p.cache.s1),
        vbase(u.p.cache.t[1] + u.g * u.p.cache.s1), pages(u.p, seq, u.n_kv) {
    pages.start(key_begin / kRun);
  }
  __device__ __forceinline__ void at_tile(int key0) { pages.at(key0 / kRun); }
  // The last part to arrive adds up all of them in their order: a wave its 32 rows,
  // lanes as the products left them, kInFlight parts on their way at once.
  static constexpr bool kJoins = true;
  __device__ __forceinline__ void join(const floatx16 (&own)[NDB], float ref, float l, bool active) const {
    const int tid = thread_here(), lane = tid % kWave, kh = lane / 32;
    const int r = 32 * uniform(tid / kWave) + lane % 32;
    if (active && this->row0 + r < this->rows) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          this->put_part(r, 32 * db + 8 * q + 4 * kh, f32x4{own[db][4 * q], own[db][4 * q + 1], own[db][4 * q + 2], own[db][4 * q + 3]});
      if (kh == 0) this->put_sums(r, ref, l);
    }
    if (!this->arrive()) return;
    // (up to 64 rows: two waves for each 32, a half of the dims each)
    const int wave = uniform(tid / kWave), blocks = uniform((min(this->rows - this->row0, Base::kRows) + 31) / 32);
    if (blocks <= 2) add_up<NDB / 2, D == 64 ? 8 : 4>(wave & 1, wave / 2 * (NDB / 2), lane);
    else add_up<NDB, D == 64 ? 4 : 2>(wave, 0, lane);
  }
  // Rows 32 `block` .., dims 32 db0 .. 32 (db0 + DBS) - 1.
  template <int DBS, int kInFlight>
  __device__ __forceinline__ void add_up(int block, int db0, int lane) const {
    typedef Record<D, Base::kRows> R;
    const int r = 32 * block + lane % 32, kh = lane / 32, row = this->row0 + r, n = this->parts;
    if (row >= this->rows) return;
    const rsrc_t recs = make_rsrc(this->first_record(), (unsigned)(2 * n - 1) * R::BYTES);
    f32x4 acc[DBS][4];
#pragma unroll
    for (int db = 0; db < DBS; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[db][q] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;
    for (int k0 = 0; k0 < n; k0 += kInFlight) {
      f32x4 x[kInFlight][DBS][4];
      f32x2 ml[kInFlight];
#pragma unroll
      for (int e = 0; e < kInFlight; ++e) {
        const unsigned at = Base::part_at(min(k0 + e, n - 1));
        ml[e] = shared_load2(recs, at + R::sums_at(r));
#pragma unroll
        for (int db = 0; db < DBS; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q) x[e][db][q] = shared_load4(recs, at + R::piece_at(r, 32 * (db0 + db) + 8 * q + 4 * kh));
      }
#pragma unroll
      for (int e = 0; e < kInFlight; ++e) {
        if (k0 + e >= n) continue;
        const float now = fmaxf(top, ml[e][0]), mu = now == -INFINITY ? 0.f : now;
        const float a = fast_exp2(top - mu), b = fast_exp2(ml[e][0] - mu);
        top = now;
        sum = sum * a + ml[e][1] * b;
#pragma unroll
        for (int db = 0; db < DBS; ++db)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[db][q] = acc[db][q] * a + x[e][db][q] * b;
      }
    }
    const int token = row / this->n_rep;
    const float inv = top == -INFINITY && sum == 0.f ? 0.f : 1.f / sum;
    char* const out = this->out_row(token, row - token * this->n_rep);
#pragma unroll
    for (int db = 0; db < DBS; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) gstore(out + 4 * (32 * (db0 + db) + 8 * q + 4 * kh), acc[db][q] * inv);
  }
  __device__ __forceinline__ unsigned none() const { return pages.none; }
  struct Rows {
    const ManyRows& w;
    const char* base;
    int s2, key0;
    __device__ __forceinline__ Rows(const ManyRows& u, int which, int key)
        : w(u), base(which == 0 ? u.kbase : u.vbase), s2((int)u.p.cache.s2), key0(key) {}
    __device__ __forceinline__ rsrc_t rows(int run) const {
      const int slot = w.pages.slot_of(run);
      const int n = w.pages.none >> run & 1u ? 0 : min(w.n_kv - key0 - kRun * run, kRun);
      return make_rsrc(base + (int64_t)slot * s2, n > 0 ? (unsigned)((n - 1) * s2 + D * ELT) : 0u);
    }
    __device__ __forceinline__ unsigned row_at(unsigned row, int run) const { return (row - kRun * run) * (unsigned)s2; }
  };
  struct Scale {
    int n;  // scales of a row
    const char* src;
    __device__ __forceinline__ Scale(const ManyRows& w, bool k, int group) {
      n = k ? NDB : 1;
      src = ELT == 1 ? w.p.cache.scale[k ? 0 : 1] + 2 * (w.g * n + (k ? group : 0)) : nullptr;
    }
    // (every row of a page is there)
    __device__ __forceinline__ const char* at(const ManyRows& w, int, int key) const {
      const int slot = w.pages.slot_of(key / kRun);
      return src + (int64_t)(slot + key % kRun) * (w.p.cache.n_head_kv * 2 * n);
    }
  };
  // (of a key without a page: of row 0, whose value does not matter beside the NaN)
  __device__ __forceinline__ const char* v_row(int key) const {
    return vbase + (int64_t)max(pages.row(key), 0) * (int)this->p.cache.s2;
  }
  __device__ __forceinline__ const char* v_scale(int key) const {
    return this->p.cache.scale[1] + ((int64_t)max(pages.row(key), 0) * this->p.cache.n_head_kv + this->g) * 2;
  }
};

// The records of a unit's parts into its rows: out = sum_k 2^(ref_k - M) O_k / sum_k 2^(ref_k - M) l_k. A thread
// takes four dims of a row; where there are few rows, groups of threads take every
// `groups`-th part and meet in LDS in order. What it takes is the records' latency,
// so as few rounds of loads as the registers allow.
template <int D, int ROWS, typename U>
__device__ __forceinline__ void join_parts(const U& u, int n_rows, lds_t* lds) {
  constexpr int kInFlight = 16, THREADS = kTreeWaves * kWave;
  typedef Record<D, ROWS> R;
  const int tid = thread_here(), units = n_rows * (D / 4);
  const int n = u.parts;
  const rsrc_t recs = make_rsrc(u.first_record(), (unsigned)(2 * n - 1) * R::BYTES);
  // A thread's part in LDS: four dims, and behind those of all threads its reference and sum.
  constexpr int kDims = 16, kPair = 8, kSums = THREADS * kDims;
  static_assert(kDims % alignof(f32x4) == 0 && kPair % alignof(f32x2) == 0 && kSums % alignof(f32x2) == 0,
                "every thread's part has its type's alignment");
  static_assert(kSums + THREADS * kPair <= TreeCfg<D, float, 1>::LDS, "they fit the kernel's LDS");
  int groups = 1;
  while (units * groups * 2 <= THREADS) groups *= 2;
  const int span = THREADS / groups, grp = tid / span;
  auto finish = [&](int i, f32x4 acc, float m, float l) __attribute__((always_inline)) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4)), token = (u.row0 + r) / u.n_rep;
    const float inv = m == -INFINITY && l == 0.f ? 0.f : 1.f / l;
    gstore(u.out_row(token, u.row0 + r - token * u.n_rep) + 4 * d, acc * inv);
  };
  for (int i = tid % span; i < units; i += span) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = grp; k0 < n; k0 += kInFlight * groups) {
      f32x2 ml[kInFlight];
      f32x4 o[kInFlight];
#pragma unroll
      for (int e = 0; e < kInFlight; ++e) {
        const unsigned at = U::part_at(min(k0 + e * groups, n - 1));
        ml[e] = shared_load2(recs, at + R::sums_at(r));
        o[e] = shared_load4(recs, at + R::piece_at(r, d));
      }
#pragma unroll
      for (int e = 0; e < kInFlight; ++e) {
        if (k0 + e * groups >= n) continue;
        const float mn = fmaxf(m, ml[e][0]), mu = mn == -INFINITY ? 0.f : mn;
        const float x = fast_exp2(m - mu), y = fast_exp2(ml[e][0] - mu);
        acc = acc * x + o[e] * y;
        l = l * x + ml[e][1] * y;
        m = mn;
      }
    }
    if (groups > 1) {  // (every thread has at most one unit)
      lds_store<f32x4>(lds + tid * kDims, acc);
      lds_store<f32x2>(lds + kSums + tid * kPair, f32x2{m, l});
    } else {
      finish(i, acc, m, l);
    }
  }
  if (groups == 1) return;
  __syncthreads();
  if (tid >= units) return;
  float m = -INFINITY, l = 0.f;
  for (int o = 0; o < groups; ++o) m = fmaxf(m, lds_load<float>(lds + kSums + (tid + o * span) * kPair));
  const float mu = m == -INFINITY ? 0.f : m;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int o = 0; o < groups; ++o) {
    const f32x2 ml = lds_load<f32x2>(lds + kSums + (tid + o * span) * kPair);
    const float y = fast_exp2(ml[0] - mu);
    acc += lds_load<f32x4>(lds + (tid + o * span) * kDims) * y;
    l += ml[1] * y;
  }
  finish(tid, acc, m, l);
}

}  // namespace

// A line of units: sequences of more than few_rows query rows per KV head in row
// tiles of 128 (WIDE), or those of up to that many (at most 16 RT) in one.
template <int D, typename KT, int RT, bool WIDE>
struct LineCfg {
  static constexpr int ROWS = WIDE ? WideCfg<D, KT>::ROWS : 16 * RT, TK = WIDE ? WideCfg<D, KT>::TK : kTreeTile;
  static constexpr int LDS = WIDE ? WideCfg<D, KT>::LDS : TreeCfg<D, KT, RT>::LDS;
  static constexpr int WAVES_PER_SIMD = WIDE ? WideCfg<D, KT>::WAVES_PER_SIMD : TreeCfg<D, KT, RT>::WAVES_PER_SIMD;
};

// LDS behind the kernels': each wave's sequences at hand, and a word for who joins.
constexpr int kState = kTreeWaves * 5 * 4 * kWave + 16;

// This workgroup's share of a line.
template <int D, typename KT, int RT, bool WIDE>
__device__ __forceinline__ void run_line(const PagedAttn& p, const PagedLine& line, lds_t* const lds, lds_t* const state) {
  typedef LineCfg<D, KT, RT, WIDE> C;
  typedef typename std::conditional<WIDE, Units<C::ROWS, C::TK>, OneUnit<C::TK>>::type U;
  constexpr int ROWS = C::ROWS, TK = C::TK;
  bool whole = line.rec == nullptr;  // no unit in parts, as there are no records
  unsigned pad = 1u;
  unsigned n_units = 0u;  // of the lane's sequences and a head
  bool pairs = false;     // of row tiles
  auto units_of = [&](const SeqLens& s) __attribute__((always_inline)) -> unsigned {
    const int rows = s.n_new * p.n_rep;
    if (rows == 0 || WIDE != (rows > p.few_rows)) return 0u;
    const U u(s, p.n_rep);
    n_units += (unsigned)u.count();
    pairs = pairs || u.count() > 1;
    return u.per_head(whole, pad) * (unsigned)p.cache.n_head_kv;
  };

  // ---- the line: lane i has sequence `first` + i ------------------------------------
  // Lengths and running sums are kept in LDS, by each wave its own: while a unit is
  // worked on, the registers are its own.
  lds_t* const kept_at = state + uniform(thread_here() / kWave) * (5 * 4 * kWave);
  int first = 0;
  unsigned before = 0u;  // units of the sequences before
  auto keep = [&](int lane, const SeqLens& s, unsigned end) __attribute__((always_inline)) {
    const int x[5] = {s.q0, s.n_new, s.n_past, s.n_seen, (int)end};
#pragma unroll
    for (int j = 0; j < 5; ++j) lds_store<int>(kept_at + 4 * (kWave * j + lane), x[j]);
  };
  unsigned total = 0u;
  int longest = 0;  // keys, about
  auto add_up = [&](bool again) __attribute__((always_inline)) {
    total = 0u;
    for (int i = (p.n_seq - 1) / kWave * kWave; i >= 0; i -= kWave) {  // (the first 64 last: they stay)
      const int lane = thread_here() % kWave;
      SeqLens s;
      if (again && i == 0) {
        auto x = [&](int j) __attribute__((always_inline)) { return lds_load<int>(kept_at + 4 * (kWave * j + lane)); };
        s = SeqLens{x(0), x(1), x(2), x(3)};
      } else {
        s = seq_lens(p, i + lane);
      }
      const unsigned units = units_of(s), end = wave_scan(units);
      total += (unsigned)__builtin_amdgcn_readlane((int)end, 63);
      longest = max(longest, units > 0u ? s.n_seen : 0);
      if (i == 0) keep(lane, s, end);
    }
  };
  // Shares: the same for every workgroup, few rows in whole rounds of the waves.
  const unsigned n_wg = gridDim.x;
  unsigned per = 1u;
  auto rounds = [&](unsigned x) __attribute__((always_inline)) -> unsigned {
    return WIDE ? x : (x + kTreeWaves - 1) / kTreeWaves * kTreeWaves;
  };
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {  // (one copy of the code, which a short call waits for)
    wave_lds_fence();
    add_up(pass > 0);
    if (pass == 0) {
      per = max((total + n_wg - 1) / n_wg, 1u);
      if (whole || total == 0u) break;
      per = rounds(per);
      // A unit's parts are joined some at a time, so a long one takes per + (tiles /
      // per) `join` tiles' time, the least for per = sqrt(tiles join).
      const float tiles = wave_max_dpp((float)longest) * (1.f / TK);
      const unsigned want = rounds((unsigned)uniform((int)fminf(fmaxf((float)line.least, sqrtf(tiles * line.join)), ceilf(tiles))));
      const unsigned units = (unsigned)__builtin_amdgcn_readlane((int)wave_scan(n_units), 63) * (unsigned)p.cache.n_head_kv;
      // Parts cost `fixed` tiles' time too: units up to that long stay whole while each
      // has a workgroup of its own.
      if (units <= n_wg && tiles <= 2.f * sqrtf(tiles * line.join) + line.fixed) {
        whole = true;
        per = 1u;
        continue;
      }
      // Where shares of `want` are fewer than the workgroups, or a few tiles more a share
      // make them so, none has two units.
      if (want > per) {
        per = pad = want;
      } else {
        if (units > n_wg / 2 || __builtin_amdgcn_ballot_w64(pairs) != 0ull) break;
        pad = max(rounds((total - 1) / (n_wg - units / 2) + 1), per);
        if (pad - per > (unsigned)line.spare) {
          pad = 1u;
          break;
        }
      }
    } else if (pass == 1) {
      if (whole) break;
      if ((total + pad - 1) / pad <= n_wg) {
        per = pad;
        break;
      }
      pad = 1u;
    }
  }
  // (all of these are the wave's, which the compiler has to know: descriptors that it
  // takes for a lane's own are loaded through in loops)
  per = (unsigned)uniform((int)per);
  pad = (unsigned)uniform((int)pad);
  total = (unsigned)uniform((int)total);
  // An XCD's workgroups (every eighth) have one piece of the line, all XCDs as many.
  const unsigned busy = (total + per - 1) / per, each = (busy + 7) / 8;
  // (the two lines of a launch from its two ends, so that short ones have workgroups of
  // their own: 300 tokens among 8 chats over 1000, 28/4 heads of 128, F16, timed alone
  // 33 us, from the same end 43)
  const unsigned block = WIDE ? n_wg - 1 - blockIdx.x : blockIdx.x;
  if (block / 8 >= each) return;
  const unsigned wg = block % 8 * each + block / 8;
  unsigned x = min(wg * per, total);
  const unsigned x_end = min(x + per, total);

  while (x < x_end) {
    wave_lds_fence();
    const int lane = thread_here() % kWave;
    unsigned end = (unsigned)lds_load<int>(kept_at + 4 * (kWave * 4 + lane));
    for (;;) {
      const unsigned all = (unsigned)__builtin_amdgcn_readlane((int)end, 63);
      if (x < before + all) break;
      before += all;
      first += kWave;
      const SeqLens s = seq_lens(p, first + lane);
      end = wave_scan(units_of(s));
      keep(lane, s, end);
      wave_lds_fence();
    }
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end > x - before));
    auto kept = [&](int j) __attribute__((always_inline)) { return uniform(lds_load<int>(kept_at + 4 * (kWave * j + at))); };
    const SeqLens s{kept(0), kept(1), kept(2), kept(3)};
    const U u(s, p.n_rep);
    const unsigned per_head = u.per_head(whole, pad), seq_end = (unsigned)__builtin_amdgcn_readlane((int)end, at);
    const unsigned y = x - before - (seq_end - per_head * (unsigned)p.cache.n_head_kv);
    const int g = uniform((int)(y / per_head));
    int rt, tiles, tile;
    unsigned left = 0u;
    if (!u.find(y - (unsigned)g * per_head, whole, pad, rt, tiles, tile, left)) {
      x += left;
      continue;
    }
    rt = uniform(rt);
    tiles = uniform(tiles);
    tile = uniform(tile);
    const int n = whole ? tiles : (int)min((unsigned)(tiles - tile), x_end - x);
    const bool part = n < tiles;
    // its first tile's place: who begins it, and how many share it
    const unsigned x0 = x - (unsigned)tile, owner = part && tile > 0 ? x0 / per : wg;
    const int parts = part ? (int)((x0 + (unsigned)tiles - 1) / per - owner) + 1 : 1, mine = (int)(wg - owner);
    float* const rec = part ? line.rec + (int64_t)(2 * wg + (mine == 0 ? 1 : 0)) * Record<D, ROWS>::FLOATS : nullptr;
    const UnitRows<D, KT, ROWS> rows{p, g, s.q0, s.n_past, s.n_seen, s.n_new * p.n_rep, p.n_rep, rt * ROWS, p.scale_log2e,
                                     parts, mine, rec, line.arrived + kArrivalWords * owner, state + kState - 16};
    if constexpr (WIDE) {
      const int lim = min(s.n_seen, max(s.n_past + min(((rt + 1) * ROWS - 1) / p.n_rep, s.n_new - 1) + 1, 0));
      ManyRows<D, KT> w(rows, first + at, tile * TK, min((tile + n) * TK, lim));
      tree_wide_rows<D, KT>(w, lds);
    } else {
      FewRows<D, KT, ROWS> w(rows, first + at, tile, min(tile + n, (s.n_seen + TK - 1) / TK));
      tree_rows<D, KT, RT>(w, lds);
      if (part && rows.arrive()) join_parts<D, ROWS>(rows, rows.rows, lds);
    }
    x += whole ? 1u : (unsigned)n;
    __syncthreads();  // the LDS is free for the next unit
  }
}

// Few rows in every sequence.
template <int D, typename KT, int RT>
__global__ __launch_bounds__(kTreeWaves* kWave, (TreeCfg<D, KT, RT>::WAVES_PER_SIMD)) void paged_few_kernel(const PagedAttn p) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  lds_t* const lds = (lds_t*)lds_raw;
  run_line<D, KT, RT, false>(p, p.few, lds, lds + TreeCfg<D, KT, RT>::LDS);
}

// Sequences of any number of rows: up to 16 on one line, more on another. A
// workgroup has a share of both; the second half of the workgroups begins with the one,
// the first with the other, so that a CU that holds one of each has keys to
// stream, which memory bounds, beside products (1000 tokens after 1337 among 31
// single tokens over 2667 to 4000 keys, 28/4 heads of 128, F16: 117 us, the halves the
// other way round 124 to 127, in two launches 144).
template <int D, typename KT>
struct MixedCfg {
  typedef LineCfg<D, KT, 1, false> Few;
  typedef LineCfg<D, KT, 1, true> Many;
  static constexpr int LDS = Few::LDS > Many::LDS ? Few::LDS : Many::LDS;
};
template <int D, typename KT>
__global__ __launch_bounds__(kTreeWaves* kWave, (WideCfg<D, KT>::WAVES_PER_SIMD)) void paged_mixed_kernel(const PagedAttn p) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  lds_t* const lds = (lds_t*)lds_raw;
  lds_t* const state = lds + MixedCfg<D, KT>::LDS;
  const bool few_first = 2 * blockIdx.x >= gridDim.x;
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
    if ((turn == 0) == few_first) run_line<D, KT, 1, false>(p, p.few, lds, state);
    else run_line<D, KT, 1, true>(p, p.many, lds, state);
  }
}

template <typename K>
static hipError_t launch_kernel(K kernel, const PagedAttn& p, int n_wg, int lds, hipStream_t stream) {
  hipLaunchKernelGGL(kernel, dim3((unsigned)n_wg), dim3(kTreeWaves * kWave), lds, stream, p);
  return hipGetLastError();
}
template <int D, typename KT, int RT>
static hipError_t launch_few(const PagedAttn& p, int n_wg, hipStream_t stream) {
  constexpr int lds = TreeCfg<D, KT, RT>::LDS + kState;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_few_kernel<D, KT, RT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  return attr != hipSuccess ? attr : launch_kernel(paged_few_kernel<D, KT, RT>, p, n_wg, lds, stream);
}
template <int D, typename KT>
static hipError_t launch_mixed(const PagedAttn& p, int n_wg, hipStream_t stream) {
  constexpr int lds = MixedCfg<D, KT>::LDS + kState;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_mixed_kernel<D, KT>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  return attr != hipSuccess ? attr : launch_kernel(paged_mixed_kernel<D, KT>, p, n_wg, lds, stream);
}

// Workgroups: what the CUs hold at once, as far as there are arrival counters (one
// for each and line) and records (two), a multiple of the XCDs.
static int workgroups(int64_t n, int64_t counters, size_t part_bytes, size_t record_bytes) {
  return (int)(std::min({n, counters, (int64_t)(part_bytes / (2 * record_bytes))}) / 8 * 8);
}

template <int D, typename KT>
static hipError_t launch_paged(PagedAttn p, float* parts, size_t part_bytes, unsigned* arrived, int n_cu, hipStream_t stream) {
  // Most query rows per KV head that a sequence can have decide what is launched.
  const int64_t most = (int64_t)std::min(p.max_new, p.n_tokens) * p.n_rep;
  const bool mixed = most > 32, two = !mixed && most > 16;
  p.few_rows = two ? 32 : 16;
  p.few.least = 8;
  p.many.least = D == 64 ? 2 : 4;
  // In tiles (one of 32 keys in few rows is a wave's, F32's take longer): 500 keys of one
  // token, 14/2 heads of 64, F16 whole 8.2 us, in parts 9.6; 100 tokens from nothing,
  // 28/4 heads of 128, F16 21 and 31, timed alone.
  p.few.fixed = (D == 64 ? 12.f : 8.f) - (sizeof(KT) == 4 ? 4.f : 0.f);
  p.many.fixed = D == 64 && sizeof(KT) == 4 ? 1.f : 2.f;
  p.few.spare = mixed ? 0 : 4;
  p.many.spare = 1;
  p.few.join = D == 64 ? 0.35f : 0.5f;
  p.many.join = D == 64 ? 0.4f : sizeof(KT) == 4 ? 0.7f : 1.2f;
  p.few.arrived = arrived;
  p.many.arrived = arrived + kArrivalWords * (kArrivals / 2);
  p.few.rec = p.many.rec = nullptr;
  const size_t few_bytes = (two ? 32 : 16) * (D + 2) * sizeof(float), many_bytes = 128 * (D + 2) * sizeof(float);
  const int per_cu = mixed ? WideCfg<D, KT>::WAVES_PER_SIMD : two ? (D == 64 ? 2 : 1) : (D == 64 ? 3 : 2);
  int n_wg = workgroups((int64_t)n_cu * per_cu, mixed ? kArrivals / 2 : kArrivals, parts ? part_bytes : 0,
                        few_bytes + (mixed ? many_bytes : 0));
  if (n_wg > 0) {
    p.many.rec = parts;
    p.few.rec = mixed ? parts + (size_t)2 * n_wg * many_bytes / sizeof(float) : parts;
  } else {  // no room for records: no unit in parts
    n_wg = n_cu * per_cu / 8 * 8;
  }
  if (mixed) return launch_mixed<D, KT>(p, n_wg, stream);
  return two ? launch_few<D, KT, 2>(p, n_wg, stream) : launch_few<D, KT, 1>(p, n_wg, stream);
}

hipError_t launch_paged_attn(const PagedAttn& p, float* parts, size_t part_bytes, unsigned* arrived, int n_cu, hipStream_t stream) {
  if (p.cache.head_dim == 64)
    return p.cache.elt == 1   ? launch_paged<64, int8_t>(p, parts, part_bytes, arrived, n_cu, stream)
           : p.cache.elt == 2 ? launch_paged<64, _Float16>(p, parts, part_bytes, arrived, n_cu, stream)
                              : launch_paged<64, float>(p, parts, part_bytes, arrived, n_cu, stream);
  return p.cache.elt == 1   ? launch_paged<128, int8_t>(p, parts, part_bytes, arrived, n_cu, stream)
         : p.cache.elt == 2 ? launch_paged<128, _Float16>(p, parts, part_bytes, arrived, n_cu, stream)
                            : launch_paged<128, float>(p, parts, part_bytes, arrived, n_cu, stream);
}

}  // namespace mi
