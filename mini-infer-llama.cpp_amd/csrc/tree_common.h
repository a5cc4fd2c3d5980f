// tree_common.h -- what the tree-attention kernels (tree.hip, tree_wide.hip) and those over
// pages (paged_attn.hip) share.
#pragma once

#include "attn_common.h"

namespace mi {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

namespace {

constexpr int kTreeWaves = 4;  // per workgroup

// lane ^ 32's x and x itself, in some order. As asm: the compiler's builtin
// drops one of the two results when they are used as floats. s_nop: the two
// wait states that a VALU write of an operand needs before the swap reads it.
__device__ inline void swap32(float x, float& a, float& b) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  a = x;
  b = y;
}
__device__ inline float max32(float x) {
  float a, b;
  swap32(x, a, b);
  return fmaxf(a, b);
}
__device__ inline float sum32(float x) {
  float a, b;
  swap32(x, a, b);
  return a + b;
}

__device__ inline u32x4 buf_b128(rsrc_t r, unsigned vo) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, vo, 0, 0));
}
__device__ inline u32x2 buf_b64(rsrc_t r, unsigned vo) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, vo, 0, 0));
}
__device__ inline unsigned buf_b32(rsrc_t r, unsigned vo) {
  return __builtin_amdgcn_raw_buffer_load_b32(r, vo, 0, 0);
}
__device__ inline unsigned buf_b16(rsrc_t r, unsigned vo) {
  return __builtin_amdgcn_raw_buffer_load_b16(r, vo, 0, 0);
}
__device__ inline floatx16 mfma_f16(f16x8 a, f16x8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx16 mfma_f32(float a, float b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// Bytes i and j of (hi : lo) -- 0..3 in lo, 4..7 in hi -- as two f16 numbers
// (b - 128) 2^-10, for bytes that hold an int8 value plus 128: as f16 bits the
// zero-extended byte is b 2^-24, and one packed multiply-add is exact.
template <int I, int J>
__device__ inline f16x2 bytes_f16(unsigned hi, unsigned lo) {
  const unsigned x = __builtin_amdgcn_perm(hi, lo, 0x0c000c00u | (unsigned)J << 16 | (unsigned)I);
  const _Float16 up = (_Float16)16384.f, off = (_Float16)-0.125f;
  return __builtin_bit_cast(f16x2, x) * f16x2{up, up} + f16x2{off, off};
}
constexpr float kByteUnscale = 1024.f;  // what the 2^-10 above takes away

// hi = RNE(x), lo = RNE(x - hi) of two values (x - hi is exact in float). The
// differences as asm: mixed-precision multiply-adds, which read hi as f16; the
// compiler widens it first, an instruction more for each.
__device__ inline void split2(float x0, float x1, f16x2& hi, f16x2& lo) {
  hi = __builtin_convertvector((f32x2{x0, x1}), f16x2);
  const unsigned h = __builtin_bit_cast(unsigned, hi);
  float d0, d1;
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d0) : "v"(h), "v"(x0));
  asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d1) : "v"(h), "v"(x1));
  lo = __builtin_convertvector((f32x2{d0, d1}), f16x2);
}

// The largest of 16 and `x`; NaN if one is (the row's output is then NaN, what
// it is compared with does not matter). The maximum that passes NaN on has a
// three-operand instruction; fmaxf would take one more for each operand.
__device__ inline float max16(const floatx16& s, float x) {
#pragma unroll
  for (int e = 0; e < 16; e += 2) x = __builtin_elementwise_maximum(__builtin_elementwise_maximum(x, s[e]), s[e + 1]);
  return x;
}

// A softmax row's running reference: probabilities are 2^(s - ref). It moves
// only when one would pass 2^14 (f16's range holds it, and the products with
// what it scales), and then to 2^6 for the largest seen: rows move after their
// first tile hardly ever, so that what has been summed is hardly ever rescaled.
// `top`: the tile's largest score (plus the V scales' exponent). Returns the
// factor of what has been summed. (No contraction: `top` may be a product that
// is -inf, and fused with ref = -inf it would be compared before it is rounded.)
constexpr float kRefMost = 14.f, kRefNew = 6.f;
__device__ inline float move_ref(float& ref, float top) {
#pragma clang fp contract(off)
  if (!(top - ref > kRefMost)) return 1.f;
  const float now = top - kRefNew, alpha = fast_exp2(ref - now);
  ref = now;
  return alpha;
}

// A record (a row tile's part from one split): its sums, then every row's
// reference, then every row's sum of probabilities. The four dims d, d + 1, ..
// (d a multiple of 4) of row r: 32 rows' pieces of 16 bytes lie together, those
// of d and d + 4 in 1 KB, as the lanes of a wave hold them.
__device__ inline int tree_record_at(int head_dim, int r, int d) {
  return (r / 32) * 32 * head_dim + (d / 8) * 256 + ((d / 4) % 2) * 128 + (r % 32) * 4;
}

// A record's values are for other XCDs, after the kernel: nontemporal, so that
// less is left in the L2 to be written back at its end (a 25-token tree over
// 4107 F16 keys, 8 MB of records: 16.2 -> 15.0 us, the join 0.6 us more).
__device__ inline void put_record(float* at, f32x4 x) { __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(at)); }

// The e for which scales up to `top` are below 2^e (at least that of the
// smallest scale there is).
__device__ inline int scale_exponent(float top) { return top > 0.f ? ilogbf(top) + 1 : -24; }

// Which keys key0 .. key0 + 31 the query `token` sees, as bits: those of the
// item's first n_past all, the rest by the mask or (none) up to its own.
__device__ inline unsigned visible_bits(const TreeItem& it, int token, int key0) {
  const int b0 = key0 - it.n_past;  // the first key as a bit of the mask row
  const int left = it.n_past + it.n_tokens - key0;
  if (left <= 0) return 0u;
  if (!it.mask) {
    const int n = token - b0 + 1;
    return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
  }
  const char* const row = it.mask + (int64_t)token * it.mask_nb;
  unsigned v;
  if (b0 >= 0) {
    const int w = b0 >> 6, sh = b0 & 63;
    uint64_t x = gload<uint64_t>(row + 8 * (int64_t)w) >> sh;
    if (sh > 32 && w + 1 < (it.n_tokens + 63) / 64) x |= gload<uint64_t>(row + 8 * (int64_t)(w + 1)) << (64 - sh);
    v = (unsigned)x;
  } else if (b0 > -32) {
    v = (unsigned)gload<uint64_t>(row) << -b0 | ((1u << -b0) - 1u);
  } else {
    v = ~0u;
  }
  return left >= 32 ? v : v & ((1u << left) - 1u);
}

__device__ inline bool not_finite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u; }
// of two f16: bit 0 for the low one, bit 1 for the high one
__device__ inline unsigned not_finite2(unsigned x) {
  return ((x & 0x7c00u) == 0x7c00u ? 1u : 0u) | ((x & 0x7c000000u) == 0x7c000000u ? 2u : 0u);
}

}  // namespace

}  // namespace mi
