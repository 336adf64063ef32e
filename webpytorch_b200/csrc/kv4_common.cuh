// The paged 4-bit key/value cache: layout, and the decoding of its codes.
//
// cache: uint8 [num_pages][NKV][page / 16][block]. A block holds 16 consecutive positions of one
// key/value head in one contiguous record (2304 bytes at HD = 128, G = 64), so a position range of
// a head is read with one bulk copy a block whatever the page size:
//     K codes [16][HD / 2] | K (s, m) [16][HD / G] half2 | V codes [16][HD / 2] | V (s, m) [16][HD / G]
// Codes are packed LSB-first along the head dimension, as AutoGPTQ packs along K. For each group of
// G elements of one position, m = half(min), s = half((max - min) / 15), n = rint((x - m) / s) in
// [0, 15], and a code stands for half(s n + m): one rounding, so the fp16 value that feeds the
// tensor cores IS the value and every kernel agrees on it. A group whose s or m is not a finite half
// (an input that is inf, nan or beyond 65504) has s = m = nan and stands for nan.
#pragma once

#include "ql_common.cuh"

namespace ql {
namespace kv4 {

constexpr int kBlock = 16;   // positions of a block

__host__ __device__ constexpr int code_bytes(int HD) { return kBlock * HD / 2; }
__host__ __device__ constexpr int scale_bytes(int HD, int G) { return kBlock * (HD / G) * 4; }
__host__ __device__ constexpr int block_bytes(int HD, int G) { return 2 * (code_bytes(HD) + scale_bytes(HD, G)); }

// The sizes every entry point of the cache accepts.
inline bool sizes_ok(int NKV, int HD, int page, int group) {
  return NKV > 0 && (HD == 64 || HD == 128 || HD == 256) && page >= kBlock && page <= 4096 &&
         (page & (page - 1)) == 0 && (group == 32 || group == 64 || group == 128) && group <= HD;
}

__device__ __forceinline__ __half2 h2_const(uint32_t u) { return u32_as_h2(u); }

// The 8 codes of a word as four half2 of exact integers: out[j] = (nibble j, nibble j + 4).
// 0x6400 | n is 1024 + n; nibbles at bits 4..7 give 1024 + 16 n, brought back by one fma.
__device__ __forceinline__ void codes_h2(uint32_t w, __half2 (&out)[4]) {
  const __half2 k1024 = h2_const(0xE400E400u);    // -1024
  const __half2 k16 = h2_const(0x2C002C00u);      // 1 / 16
  const __half2 k64 = h2_const(0xD400D400u);      // -64
  const uint32_t u = w >> 8;
  out[0] = __hadd2(u32_as_h2(lop3_andor(w, 0x000F000Fu, kMagicF16x2)), k1024);
  out[1] = __hfma2(u32_as_h2(lop3_andor(w, 0x00F000F0u, kMagicF16x2)), k16, k64);
  out[2] = __hadd2(u32_as_h2(lop3_andor(u, 0x000F000Fu, kMagicF16x2)), k1024);
  out[3] = __hfma2(u32_as_h2(lop3_andor(u, 0x00F000F0u, kMagicF16x2)), k16, k64);
}

// Whether some value of a group with (s, m) may not be finite: a group that stands for nan, or a last code past
// fp16's range.
__device__ __forceinline__ bool may_not_be_finite(__half2 sm) {
  const __half top = __hfma(__habs(__low2half(sm)), __ushort_as_half((unsigned short)0x4B80), __habs(__high2half(sm)));   // 15 |s| + |m|
  return (__half_as_ushort(top) & 0x7fffu) >= 0x7c00u;
}

// A pair of values, those that are not finite as zero.
__device__ __forceinline__ __half2 finite_or_zero(__half2 v) {
  uint32_t u = h2_as_u32(v);
  if ((u & 0x7c00u) == 0x7c00u) u &= 0xffff0000u;
  if ((u & 0x7c000000u) == 0x7c000000u) u &= 0x0000ffffu;
  return u32_as_h2(u);
}

}  // namespace kv4
}  // namespace ql
