// The 4-bit K/V cache: format and layout (rldx_kv4_* in rldx_amd.h).
//
// Format (OCP MX, MXFP4): e2m1 elements (sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6) in blocks
// of 32 along head_dim with one e8m0 scale each: byte e stands for 2^(e - 127), 255 for NaN.
// code * 2^k is exact in bf16, and gfx950 converts two codes with their scale to packed bf16 in
// one instruction (v_cvt_scalef32_pk_bf16_fp4), so the attention multiplies exact values.
//
// Layout: a page of page_tokens slots (a power of two, 32 or more) of one KV head is page_tokens / 32
// tiles of 32 slots, each 32 D + 2 D bytes (D = head_dim, 64 or 128; w = D / 16):
//   [0, 16 D)     K codes  byte slot D/2 + d/2, the even d in its low half: a row per slot.  Lane
//                 l of a v_mfma_f32_16x16x32_bf16 A operand takes key l % 16 and the D/4 dimensions
//                 from (D/4)(l / 16): one load, and all of them under one or half of one scale.
//   [16 D, 32 D)  V codes  unit ((slot/4 % 4) 16 + d/w) 8 + slot/16 4 + slot%4 of w/2 bytes, holding
//                 d % w = 0 .. w-1: lane l's 8 units are the 8 slots of its V^T operand
//                 (4 (l/16) .. +3 and 16 + 4 (l/16) .. +3, the order in which S^T leaves the
//                 probabilities in its registers) at the dimensions w (l % 16) .. + w - 1.  A
//                 unit belongs to one slot, so slots are written without reading their neighbours.
//   [32 D, 33 D)  K scales byte slot D/32 + d/32
//   [33 D, 34 D)  V scales byte (d/32 4 + slot/4 % 4) 8 + slot/16 4 + slot%4
#pragma once

#include "rldx_amd.h"
#include "rldx_common.h"

namespace rldx {
namespace kv4 {

constexpr int kTile = 32;  // slots per tile
RLDX_HD constexpr int tile_bytes(int d) { return 34 * d; }
constexpr uint32_t kScaleNan = 255;

// Place of slot s in the order of a tile's V part: its unit within a lane's 8, and the lane group.
RLDX_HD constexpr int v_unit(int s) { return (s >> 4) * 4 + (s & 3); }
RLDX_HD constexpr int v_group(int s) { return (s >> 2) & 3; }

// Scale exponent of a block from the bits of its largest magnitude (fp32): the power of two under
// which amax lies in [4, 7) or [3.5, 4): amax / 2^e rounds to at most 6, so no element is
// further off than half of e2m1's last step.  (floor(log2 amax) - 2 alone leaves [7, 8), cut off at 6.)
// Bounds: 0.5 2^-125 is the smallest normal value, 6 2^125 the largest that is finite.
RLDX_HD int block_exponent(uint32_t amax_bits) {
  const int p = static_cast<int>(amax_bits >> 23) - 127;
  const int e = p - 2 + ((amax_bits & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return e < -125 ? -125 : e > 125 ? 125 : e;
}

// Code of x 2^-e: the nearest of the grid, ties to the even code, cut off at 6.
RLDX_HD uint32_t element_code(float x, int e) {
  uint32_t u;
  __builtin_memcpy(&u, &x, 4);
  const float y = __builtin_ldexpf(__builtin_fabsf(x), -e);  // exact: x is a bf16 and y < 8 (or underflows to 0)
  const uint32_t c = (y > 0.25f) + (y >= 0.75f) + (y > 1.25f) + (y >= 1.75f) + (y > 2.5f) + (y >= 3.5f) + (y > 5.f);
  return c | ((u >> 28) & 8u);
}

}  // namespace kv4

// Whether the sizes, strides and alignments of a cache are those that the kernels take (kv4_cache.hip).
bool kv4_cache_ok(const rldx_kv4_cache_t* c);

}  // namespace rldx
