// Microscaled rows: numbers in blocks of 32 along a row, each an element of 4 bits (e2m1: magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) or 8 (e4m3: up to
// 448) times its block's scale, a power of two 2^e held as the byte e + 127 (255: every value of the block is NaN).
//
// A block's scale is the smallest power of two under which its largest magnitude lies at most half a step beyond the largest element (7 for e2m1, 464
// for e4m3), so that no element is further from its number than half a step of the elements there; never below 2^-127. Elements are rounded to the
// nearest, ties to the even one. A block with an infinity or a NaN has the scale 255, as has one whose scale would lie beyond 2^127 (the norm's rows alone can have numbers that large).
//
// They lie in the order in which the matrix cores take them, so that a wavefront's operand is one run of memory. Tiles of 16 rows by 128 numbers follow one another
// along the row; a tile is units of 16 bytes, [group][row of 16]: of e2m1 4 groups of 32 numbers (two to a byte, the first in the low half), of e4m3 8 groups of 16.
// Behind all tiles come the scales, 64 bytes a tile: [row of 16][block of 4]. Rows are filled up to a multiple of 128 with zeros; what the rows behind the last one of
// the last tile hold is of no account (an output depends on one row of each operand alone).
#pragma once

#include "common.h"

namespace alofa {

enum MxKind : int { kE4M3 = 0, kE2M1 = 4 };      // (as the matrix instructions number them)

__host__ __device__ constexpr int64_t mx_tiles(int64_t n, int64_t to) { return (n + to - 1) / to; }
__host__ __device__ constexpr int mx_units(int kind) { return kind == kE2M1 ? 64 : 128; }      // 16-byte units of a tile
// where the scales begin, in bytes
__host__ __device__ constexpr int64_t mx_scales_at(int64_t rows, int64_t k, int kind) { return mx_tiles(rows, 16) * mx_tiles(k, 128) * mx_units(kind) * 16; }

__host__ constexpr int64_t mx_bytes(int64_t rows, int64_t k, int kind) { return mx_scales_at(rows, k, kind) + mx_tiles(rows, 16) * mx_tiles(k, 128) * 64; }

// Where an operand lies: so many rows of so many bytes, ld bytes apart; microscaled rows are one run. Blocks write while others still read, so what is written may not meet what is read.
struct MxPlace {
  uintptr_t at;
  int64_t ld, rows, bytes;
  static MxPlace run(const void* p, int64_t bytes) { return {reinterpret_cast<uintptr_t>(p), bytes, 1, bytes}; }
  static MxPlace held(const void* p, int64_t rows, int64_t k, int kind) { return run(p, mx_bytes(rows, k, kind)); }
  static MxPlace numbers(const void* p, int64_t ld, int64_t rows, int64_t k, int size) { return {reinterpret_cast<uintptr_t>(p), ld * size, rows, k * size}; }
  uintptr_t end() const { return at + (rows - 1) * ld + bytes; }
  // (columns side by side in the same rows do not meet; rows of different lengths that lie between each other are taken to)
  bool meets(const MxPlace& o) const {
    if (at == 0 || o.at == 0 || at >= o.end() || o.at >= end()) return false;
    const int64_t step = rows > 1 ? ld : o.ld;
    if ((rows > 1 && o.rows > 1 && ld != o.ld) || step < bytes || step < o.bytes) return true;
    const int64_t apart = o.at >= at ? static_cast<int64_t>((o.at - at) % step) : (step - static_cast<int64_t>((at - o.at) % step)) % step;
    return apart < bytes || apart + o.bytes > step;
  }
};

// The scale byte of a block whose largest magnitude has these bits (infinities and NaN included: their bits are the largest)
template <int kKind>
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t top) {
  const int e = static_cast<int>(top >> 23);
  constexpr uint32_t beyond = kKind == kE2M1 ? 0x600000u : 0x680000u;      // behind the point: 1.75 (of 4), 1.8125 (of 256)
  const int code = e - (kKind == kE2M1 ? 2 : 8) + static_cast<int>((top & 0x7fffffu) > beyond);
  return e == 255 ? 255u : static_cast<uint32_t>(max(code, 0));
}
// the scale as the conversion instructions take it: a float, of which they read the exponent (2^-127 is its smallest)
__device__ __forceinline__ float mx_scale_float(uint32_t code) { return __uint_as_float(code == 0 ? 0x400000u : code << 23); }

// Eight numbers under one scale, as elements: 4 bytes of e2m1 in out[0], 8 of e4m3
template <int kKind>
__device__ __forceinline__ void mx_pack8(const float (&v)[8], uint32_t code, uint32_t (&out)[2]) {
  if (code == 255) {      // (every value of the block is NaN, whatever its elements)
    out[0] = out[1] = 0;
    return;
  }
  const float s = mx_scale_float(code);
  if constexpr (kKind == kE2M1) {
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    out[0] = q, out[1] = 0;
  } else {
    typedef short pair_t __attribute__((ext_vector_type(2)));
    pair_t a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], s, true);
    out[0] = __builtin_bit_cast(uint32_t, a), out[1] = __builtin_bit_cast(uint32_t, b);
  }
}

__device__ __forceinline__ uint32_t mx_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// the largest over four neighbouring lanes, for each of them
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xB1, 0xf, 0xf, false)));      // lane ^ 1
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xf, 0xf, false)));   // lane ^ 2
}

// Where in memory eight elements of row r begin, the numbers 8 c .. 8 c + 7 (k_tiles: tiles along a row); and their block's scale
template <int kKind>
__device__ __forceinline__ int64_t mx_place8(int64_t r, int c, int k_tiles) {
  const int64_t tile = (r / 16) * k_tiles + c / 16;
  const int in = c % 16, row = static_cast<int>(r % 16);
  if constexpr (kKind == kE2M1) return (tile * 64 + (in / 4) * 16 + row) * 16 + (in % 4) * 4;
  return (tile * 128 + (in / 2) * 16 + row) * 16 + (in % 2) * 8;
}
__device__ __forceinline__ int64_t mx_scale_place(int64_t r, int block, int k_tiles) { return (((r / 16) * k_tiles + block / 4) * 16 + r % 16) * 4 + block % 4; }

}  // namespace alofa
