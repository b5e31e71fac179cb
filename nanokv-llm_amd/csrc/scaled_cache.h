// The block-scaled K/V cache: 8-bit codes with one scale for every 32 tokens and head. Its form and
// the conversions, shared by the kernels that write it, read it back and attend over it.
//
// A page's rows stand in tiles of 32 tokens. A tile of a head holds E4M3 codes of x * 2^-e and its e,
// stored as the byte e + 127. With a power of two both x * 2^-e and code * 2^e are exact (a code has
// four significant bits: code * 2^e is exact in bf16), so what a call leaves in a cache does not depend on
// how its work was split, and E4M3, being a floating format, loses at most one bit of its 18 binades
// against a scale that fits exactly. It does depend on the calls: where a later one raises a tile's scale the
// rows held are rounded again, in the subnormal range, each time by at most half of its step and by less
// than one step of the last scale in all.
//   e: the smallest in [-100, 119] with max |x| <= 448 * 2^e (448: E4M3's largest; the finite x's)
// Below -100 nothing is left to hold (values up to 2^-110 become zero) and every scaled value stays
// a normal number; above 119 a code could reach 2^128. Byte 0: nothing written yet.
//
// A tile of a layer's K (or V) is 32 * (Hk * D + 16) bytes: each head's codes (32 * D bytes), then Hk
// scale bytes; the rest is unused. It is the same span that 32 rows of Hk * D + 16 bytes take, so a
// cache is [pages, block, Hk * D + 16] and a copy of a page brings its scales with it. Codes stand in
// the order in which a wave's lanes feed the matrix instructions (lane = row + 16 g), so that every
// load of a wave is 1 KiB of consecutive bytes and nothing is transposed on the way:
//   K: [t: 2][i: D/64][lane][b: 16]       token 8 (row / 4) + 4 t + row % 4, dim 64 i + 16 g + b
//   V: [j: D/32][lane][u: 2][tt: 8]       token 8 g + tt, dim 32 j + 16 u + row
// S^T = K q^T leaves lane (column, g) the scores of tokens 8 g + 4 t + 0..3: with both t the eight
// tokens whose codes the lane's V operand holds.
#pragma once

#include "nkv_common.h"

namespace nkv {

constexpr int kTileRows = 32;
constexpr int kRowPad = 16;  // bytes of a row beside its codes (NKV_SCALED_ROW_PAD)
constexpr int kMinScale = 127 - 100, kMaxScale = 127 + 119;  // bytes
constexpr bool scaled_dim_ok(int64_t D) { return D == 64 || D == 128; }

// Offset of the eight codes of dims 8 hx .. 8 hx + 7 of a token in a head's K tile.
template <int D>
__device__ __forceinline__ int k_piece(int token, int hx) {
  const int t = (token >> 2) & 1, row = 4 * (token >> 3) + (token & 3);
  return ((t * (D / 64) + (hx >> 3)) * 64 + row + 16 * ((hx >> 1) & 3)) * 16 + 8 * (hx & 1);
}
// Offset of the eight codes of tokens 8 g .. 8 g + 7 of a dim in a head's V tile.
__device__ __forceinline__ int v_piece(int g, int dim) {
  return ((dim >> 5) * 64 + (dim & 15) + 16 * g) * 16 + 8 * ((dim >> 4) & 1);
}

// The scale byte for values up to a (finite, >= 0): 448 is 1.75 * 2^8.
__device__ __forceinline__ int scale_byte(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
  return min(max(e, kMinScale), kMaxScale);
}
__device__ __forceinline__ int stored_scale(int byte) {
  return min(max(byte, kMinScale), kMaxScale);
}
__device__ __forceinline__ float scale_of(int byte) { return __int_as_float(byte << 23); }
__device__ __forceinline__ float inverse_scale(int byte) {
  return __int_as_float((254 - byte) << 23);
}

// The word that holds a head's scale byte (its offset: scale_at & ~3): loaded whole and taken apart
// where it is used, since the compiler widens a loaded byte at once, and waits for it.
__device__ __forceinline__ int byte_of(uint32_t word, int scale_at) {
  return (int)(word >> (8 * (scale_at & 3)) & 0xffu);
}

// Eight codes times a scale -> eight bf16 (exact).
__device__ __forceinline__ u32x4_t codes_to_bf16(uint32_t lo, uint32_t hi, float scale) {
  return u32x4_t{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
}

// What every operator over such caches checks (0: fine).
int scaled_check(const char* what, const void* k_cache, const void* v_cache, int64_t n_kv_heads,
                 int64_t head_dim);
int scaled_check_tables(const char* what, const int32_t* block_tables, int64_t bt_row_stride,
                        int64_t max_blocks, int64_t block_size, int64_t n_blocks);
// ... and attention's: the query heads and the scale.
int scaled_check_heads(const char* what, int64_t n_q_heads, int64_t n_kv_heads, int64_t most,
                       double scale);

}  // namespace nkv
