// Microscaled rows (microscaled.h): made from numbers, read back, laid out from a checkpoint's codes, and made by the norm between two sub-layers.
#include "microscaled.h"

namespace alofa {

// Eight numbers of a row from column c0 on, zeros behind the last column. kVec: rows and row starts are 16-byte aligned and k is a multiple of 8.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* __restrict__ row, int c0, int k, float (&v)[8]) {
  if constexpr (kVec && sizeof(T) == 4) {
    const float4 a = c0 < k ? *reinterpret_cast<const float4*>(row + c0) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float4 b = c0 < k ? *reinterpret_cast<const float4*>(row + c0 + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else if constexpr (kVec) {
    const uint4 a = c0 < k ? *reinterpret_cast<const uint4*>(row + c0) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[2 * e] = __uint_as_float(w[e] << 16), v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c0 + e < k ? load_f32(row + c0 + e) : 0.f;
  }
}

// The largest magnitude of a block, of which a lane has eight numbers and its neighbours the three other eights
__device__ __forceinline__ uint32_t block_top(const float (&v)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, mx_magnitude(v[e]));
  return quad_max(top);
}
// Those eight numbers times 2^kUp to memory, under the scale that its largest magnitude asks for: beyond the scales' range NaN
template <int kKind, int kUp = 0>
__device__ __forceinline__ void put8(uint8_t* __restrict__ out, int64_t scales_at, int64_t r, int c, int k_tiles, const float (&v)[8], uint32_t top) {
  uint32_t code = mx_scale_of<kKind>(top);
  uint32_t q[2];
  mx_pack8<kKind>(v, code, q);
  if constexpr (kUp != 0) code = min(code + kUp, 255u);
  uint8_t* at = out + mx_place8<kKind>(r, c, k_tiles);
  if constexpr (kKind == kE2M1) *reinterpret_cast<uint32_t*>(at) = q[0];
  else *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
  if (c % 4 == 0) out[scales_at + mx_scale_place(r, c / 4, k_tiles)] = static_cast<uint8_t>(code);
}

// ---- numbers to microscaled rows and back --------------------------------------
// A block takes 16 rows by 512 columns, four tiles: a wave has four of the rows, a lane eight numbers of each. The tiles are put together in LDS and leave as whole runs (row by row, 16 bytes of each 256 would be
// written at a time). Memory bounds both ways: 18,944 x 3,584 of bfloat16 to and from e2m1 35.2 us, 4.9 TB/s (a copy of 1 GiB: 5.2, of 4: 4.8); rows that 16-byte loads cannot read, or write, go number by number, 86 and 104 us, 2.0 and 1.7 TB/s
// (no model here has such widths). Elements are
// rounded by the conversion instructions, once, from the number itself (a power of two as the scale loses nothing).
constexpr int kStrip = 4;      // tiles along a row that a block takes

template <typename T, int kKind, bool kVec>
__global__ void __launch_bounds__(256) mx_quantize_kernel(uint8_t* __restrict__ out, int64_t scales_at, const T* __restrict__ x, int64_t ldx, int rows, int k, int k_tiles, int strips) {
  constexpr int kTile = mx_units(kKind) * 16;
  __shared__ __attribute__((aligned(16))) uint8_t tiles[kStrip * (kTile + 64)];      // ... and their scales behind them, as in memory
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, row_tile = blockIdx.x / strips, strip = blockIdx.x % strips, c = strip * kStrip * 16 + lane;
  float v[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = static_cast<int64_t>(row_tile) * 16 + 4 * wave + i;
    if (r < rows) load8<T, kVec>(x + r * ldx, 8 * c, k, v[i]);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) put8<kKind>(tiles, kStrip * kTile, 4 * wave + i, lane, kStrip, v[i], block_top(v[i]));
  __syncthreads();
  const int64_t first = static_cast<int64_t>(row_tile) * k_tiles + strip * kStrip;
  const int there = min(kStrip, k_tiles - strip * kStrip);
  for (int i = threadIdx.x; i < there * (kTile / 16); i += 256) reinterpret_cast<uint4*>(out + first * kTile)[i] = reinterpret_cast<const uint4*>(tiles)[i];
  if (static_cast<int>(threadIdx.x) < there * 4) reinterpret_cast<uint4*>(out + scales_at + first * 64)[threadIdx.x] = reinterpret_cast<const uint4*>(tiles + kStrip * kTile)[threadIdx.x];
}

__device__ __forceinline__ float mx_scaled(float element, uint32_t code) { return code == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(element, static_cast<int>(code) - 127); }

template <typename T, int kKind, bool kVec>
__global__ void __launch_bounds__(256) mx_values_kernel(T* __restrict__ out, int64_t ldo, const uint8_t* __restrict__ q, int64_t scales_at, int rows, int k, int k_tiles, int strips) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  constexpr int kTile = mx_units(kKind) * 16;
  __shared__ __attribute__((aligned(16))) uint8_t tiles[kStrip * kTile];
  __shared__ __attribute__((aligned(16))) uint8_t scales[kStrip * 64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, row_tile = blockIdx.x / strips, strip = blockIdx.x % strips, c = strip * kStrip * 16 + lane;
  const int64_t first = static_cast<int64_t>(row_tile) * k_tiles + strip * kStrip;
  const int there = min(kStrip, k_tiles - strip * kStrip);
  for (int i = threadIdx.x; i < there * (kTile / 16); i += 256) reinterpret_cast<uint4*>(tiles)[i] = reinterpret_cast<const uint4*>(q + first * kTile)[i];
  if (static_cast<int>(threadIdx.x) < there * 4) reinterpret_cast<uint4*>(scales)[threadIdx.x] = reinterpret_cast<const uint4*>(q + scales_at + first * 64)[threadIdx.x];
  __syncthreads();
  if (8 * c >= k) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = static_cast<int64_t>(row_tile) * 16 + 4 * wave + i;
    if (r >= rows) return;
    const uint32_t code = scales[mx_scale_place(4 * wave + i, lane / 4, kStrip)];
    const uint8_t* at = tiles + mx_place8<kKind>(4 * wave + i, lane, kStrip);
    float v[8];
    if constexpr (kKind == kE2M1) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
      const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1);
      const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3);
      v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(at);
      const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
      const f32x2_t d = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true);
      v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = mx_scaled(v[e], code);
    T* to = out + r * ldo + 8 * c;
    if constexpr (kVec && sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else if constexpr (kVec) {
      *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * c + e < k) store_f32(to + e, v[e]);
    }
  }
}

// ---- a checkpoint's codes, row by row, into the order above --------------------
// A thread lays out eight elements of a row, byte by byte (checkpoints' rows begin anywhere; it runs once, where weights are laid out). What the codes hold behind the last number of a row is not looked at.
template <int kKind>
__global__ void __launch_bounds__(256) mx_from_codes_kernel(uint8_t* __restrict__ out, int64_t scales_at, const uint8_t* __restrict__ codes, int64_t ld_codes,
                                                            const uint8_t* __restrict__ scales, int64_t ld_scales, int rows, int k, int k_tiles) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int per_row = 16 * k_tiles;
  const int64_t r = i / per_row;
  const int c = static_cast<int>(i % per_row);
  if (r >= rows) return;
  const uint8_t* row = codes + r * ld_codes;
  uint32_t q[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int at = 8 * c + e;
    if (at >= k) continue;
    if constexpr (kKind == kE2M1) q[0] |= ((row[at / 2] >> (at % 2 * 4)) & 15u) << (4 * e);
    else q[e / 4] |= static_cast<uint32_t>(row[at]) << (e % 4 * 8);
  }
  uint8_t* to = out + mx_place8<kKind>(r, c, k_tiles);
  if constexpr (kKind == kE2M1) *reinterpret_cast<uint32_t*>(to) = q[0];
  else *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
  if (c % 4 == 0) out[scales_at + mx_scale_place(r, c / 4, k_tiles)] = 8 * c < k ? scales[r * ld_scales + c / 4] : 0;
}

// ---- the norm between two sub-layers -------------------------------------------
// y rounded to 24 bits so that a later rounding to fewer (22 at most) is the rounding of y itself: towards zero, and the last bit set where anything was lost. What lies beyond the largest float comes out as that one.
__device__ __forceinline__ float round_to_odd(double y) {
  const float f = static_cast<float>(y);
  const double d = static_cast<double>(f);
  uint32_t u = __float_as_uint(f);
  if (d != y) u = (u - (fabs(d) > fabs(y) ? 1u : 0u)) | 1u;
  return y != y ? f : __uint_as_float(u);
}

// sum += add[1] + add[2] + .. in this order, three shares' loads on their way together
template <bool kVec>
__device__ __forceinline__ void add_shares(const float* __restrict__ row, int64_t share_stride, int shares, int c0, int k, float (&sum)[8]) {
  for (int s = 1; s < shares; s += 3) {
    float part[3][8];
#pragma unroll
    for (int u = 0; u < 3; ++u) load8<float, kVec>(row + min(s + u, shares - 1) * share_stride, c0, k, part[u]);
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (s + u < shares) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += part[u][e];
      }
  }
}

// total = x + (add[0] + add[1] + ..) in float, y = total / sqrt(mean(total^2) + eps) * w in double, y to microscaled rows. A block takes a row. The squares' sum and
// y are in double so that no element depends on the order of a sum: a value next to the middle of two elements would become one or the other.
// Memory bounds many rows: 2,048 x 3,584 with one share 26.8 us (3.6 TB/s; without shares 16.2, 2.3), 2,048 x 5,120 with two 45.0 (4.0); few are bound by one row's steps one after the other, 4.4 us at 1 x 896 and 5.6 at 64 x 5,120 with four
// shares. Rows that 16-byte loads cannot read go number by number: 2,000 x 5,001 with one share 83. A block of four rows would write 64 bytes at a time for 16: 26.1 us at 2,048 rows, but 11.6 for 8.0 at 512.
// kStay: a row of at most 8 kThreads numbers (8,192) stays in registers between the sum and the scaling, eight a thread; else any row, read twice. (256 threads with two and three eights took 6.5 us for 5.4 at
// 64 x 5,120 and 27.2 for 26.8 at 2,048 x 3,584: a row's steps are shorter.)
template <int kKind, int kThreads, bool kStay, bool kVec>
__global__ void __launch_bounds__(kThreads) rmsnorm_mx_kernel(uint8_t* __restrict__ out, int64_t scales_at, const float* x, int64_t ldx, const float* __restrict__ add, int shares,
                                                         int64_t share_stride, int64_t ld_add, float* total, int64_t ld_total, const float* __restrict__ w, float eps, int k, int k_tiles) {
  __shared__ double scratch[kThreads / kWave];
  const int64_t r = blockIdx.x;
  const int per_row = 16 * k_tiles;
  auto take = [&](int c, float (&v)[8]) {
    load8<float, kVec>(x + r * ldx, 8 * c, k, v);
    if (shares == 0) return;
    float sum[8];
    load8<float, kVec>(add + r * ld_add, 8 * c, k, sum);
    add_shares<kVec>(add + r * ld_add, share_stride, shares, 8 * c, k, sum);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += sum[e];
  };
  auto keep = [&](int c, const float (&v)[8]) {
    if (total == nullptr || 8 * c >= k) return;
    float* to = total + r * ld_total + 8 * c;
    if constexpr (kVec) {
      *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(to + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * c + e < k) to[e] = v[e];
    }
  };
  auto leave = [&](int c, const float (&v)[8], const float (&weight)[8], double scale) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = round_to_odd(static_cast<double>(v[e]) * scale * static_cast<double>(weight[e]));
    const uint32_t top = block_top(y);
    if (top != 0x7f7fffffu) {
      put8<kKind>(out, scales_at, r, c, k_tiles, y, top);
      return;
    }
    // a y beyond the largest float (the scales go on to 464 times 2^127): the block again, divided by 2^16 (what that takes from small numbers is far below the block's elements)
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = round_to_odd(static_cast<double>(v[e]) * (scale * 0x1p-16) * static_cast<double>(weight[e]));
    put8<kKind, 16>(out, scales_at, r, c, k_tiles, y, block_top(y));
  };
  double ss = 0;
  if constexpr (kStay) {
    const int c = threadIdx.x;
    float v[8], weight[8];
    load8<float, kVec>(w, 8 * c, k, weight);
    take(c, v);      // (nothing but zeros behind the row's end)
    keep(c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += static_cast<double>(v[e]) * static_cast<double>(v[e]);
    ss = block_sum<double, kThreads>(ss, scratch);
    const double scale = 1.0 / sqrt(ss / static_cast<double>(k) + static_cast<double>(eps));
    if (c < per_row) leave(c, v, weight, scale);
  } else {
    for (int c = threadIdx.x; c < per_row; c += kThreads) {
      float v[8];
      take(c, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += static_cast<double>(v[e]) * static_cast<double>(v[e]);
    }
    ss = block_sum<double, kThreads>(ss, scratch);
    const double scale = 1.0 / sqrt(ss / static_cast<double>(k) + static_cast<double>(eps));
    for (int c = threadIdx.x; c < per_row; c += kThreads) {
      float v[8];
      take(c, v);      // (`total` may be x itself: a thread reads its numbers again before it writes them)
      keep(c, v);
      float weight[8];
      load8<float, kVec>(w, 8 * c, k, weight);
      leave(c, v, weight, scale);
    }
  }
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static bool sizes_fit(const char* what, int kind, int64_t rows, int64_t k) {
  if (kind != kE2M1 && kind != kE4M3) set_error("%s: no such kind of element: %d", what, kind);
  else if (rows < 1 || k < 1 || rows > INT32_MAX - 16 || k > (1 << 24)) set_error("%s: rows=%lld k=%lld", what, static_cast<long long>(rows), static_cast<long long>(k));
  else if (mx_tiles(rows * 16 * mx_tiles(k, 128), 256) >= 1 << 24) set_error("%s: more blocks than a launch takes: rows=%lld k=%lld", what, static_cast<long long>(rows), static_cast<long long>(k));
  else return true;
  return false;
}

}  // namespace alofa

using namespace alofa;

extern "C" int alofa_mx_quantize(void* out, int kind, const void* x, int dtype, int64_t ldx, int64_t rows, int64_t k, hipStream_t stream) {
  if (!sizes_fit("mx_quantize", kind, rows, k)) return 1;
  ALOFA_REQUIRE(out && x && aligned16(out) && (dtype == kF32 || dtype == kBF16) && ldx >= 0, "mx_quantize: operands do not fit: dtype=%d ldx=%lld", dtype, static_cast<long long>(ldx));
  ALOFA_REQUIRE(!MxPlace::held(out, rows, k, kind).meets(MxPlace::numbers(x, ldx, rows, k, dtype == kF32 ? 4 : 2)), "mx_quantize: what is written overlaps what is read");
  const int k_tiles = static_cast<int>(mx_tiles(k, 128));
  const int64_t at = mx_scales_at(rows, k, kind);
  const int strips = (k_tiles + kStrip - 1) / kStrip;
  const unsigned blocks = static_cast<unsigned>(mx_tiles(rows, 16) * strips);
  const bool vec = aligned16(x) && k % 8 == 0 && ldx % (dtype == kF32 ? 4 : 8) == 0;
  const int r = static_cast<int>(rows), n = static_cast<int>(k);
#define GO(T, KIND, VEC) mx_quantize_kernel<T, KIND, VEC><<<blocks, 256, 0, stream>>>(static_cast<uint8_t*>(out), at, static_cast<const T*>(x), ldx, r, n, k_tiles, strips)
#define GO_VEC(T, KIND) do { if (vec) GO(T, KIND, true); else GO(T, KIND, false); } while (0)
  if (dtype == kF32) { if (kind == kE2M1) GO_VEC(float, kE2M1); else GO_VEC(float, kE4M3); }
  else { if (kind == kE2M1) GO_VEC(bf16_t, kE2M1); else GO_VEC(bf16_t, kE4M3); }
#undef GO_VEC
#undef GO
  return check_launch("mx_quantize");
}

extern "C" int alofa_mx_values(void* out, int dtype, int64_t ldo, const void* q, int kind, int64_t rows, int64_t k, hipStream_t stream) {
  if (!sizes_fit("mx_values", kind, rows, k)) return 1;
  ALOFA_REQUIRE(out && q && aligned16(q) && (dtype == kF32 || dtype == kBF16) && ldo >= 0, "mx_values: operands do not fit: dtype=%d ldo=%lld", dtype, static_cast<long long>(ldo));
  ALOFA_REQUIRE(!MxPlace::held(q, rows, k, kind).meets(MxPlace::numbers(out, ldo, rows, k, dtype == kF32 ? 4 : 2)), "mx_values: what is written overlaps what is read");
  const int k_tiles = static_cast<int>(mx_tiles(k, 128)), strips = (k_tiles + kStrip - 1) / kStrip;
  const int64_t at = mx_scales_at(rows, k, kind);
  const unsigned blocks = static_cast<unsigned>(mx_tiles(rows, 16) * strips);
  const bool vec = aligned16(out) && k % 8 == 0 && ldo % (dtype == kF32 ? 4 : 8) == 0;
  const int r = static_cast<int>(rows), n = static_cast<int>(k);
#define GO(T, KIND, VEC) mx_values_kernel<T, KIND, VEC><<<blocks, 256, 0, stream>>>(static_cast<T*>(out), ldo, static_cast<const uint8_t*>(q), at, r, n, k_tiles, strips)
#define GO_VEC(T, KIND) do { if (vec) GO(T, KIND, true); else GO(T, KIND, false); } while (0)
  if (dtype == kF32) { if (kind == kE2M1) GO_VEC(float, kE2M1); else GO_VEC(float, kE4M3); }
  else { if (kind == kE2M1) GO_VEC(bf16_t, kE2M1); else GO_VEC(bf16_t, kE4M3); }
#undef GO_VEC
#undef GO
  return check_launch("mx_values");
}

extern "C" int alofa_mx_from_codes(void* out, int kind, const void* codes, int64_t ld_codes, const void* scales, int64_t ld_scales, int64_t rows, int64_t k, hipStream_t stream) {
  if (!sizes_fit("mx_from_codes", kind, rows, k)) return 1;
  ALOFA_REQUIRE(out && codes && scales && aligned16(out) && ld_codes >= 0 && ld_scales >= 0, "mx_from_codes: operands do not fit");
  const MxPlace held = MxPlace::held(out, rows, k, kind);
  ALOFA_REQUIRE(!held.meets(MxPlace::numbers(codes, ld_codes, rows, kind == kE2M1 ? mx_tiles(k, 2) : k, 1)) && !held.meets(MxPlace::numbers(scales, ld_scales, rows, mx_tiles(k, 32), 1)),
                "mx_from_codes: what is written overlaps what is read");
  const int k_tiles = static_cast<int>(mx_tiles(k, 128));
  const int64_t at = mx_scales_at(rows, k, kind);
  const unsigned blocks = static_cast<unsigned>(mx_tiles(rows * 16 * k_tiles, 256));
#define GO(KIND) mx_from_codes_kernel<KIND><<<blocks, 256, 0, stream>>>(static_cast<uint8_t*>(out), at, static_cast<const uint8_t*>(codes), ld_codes, static_cast<const uint8_t*>(scales), \
                                                                        ld_scales, static_cast<int>(rows), static_cast<int>(k), k_tiles)
  if (kind == kE2M1) GO(kE2M1); else GO(kE4M3);
#undef GO
  return check_launch("mx_from_codes");
}

extern "C" int alofa_rmsnorm_mx(void* out, int kind, const float* x, int64_t ldx, const float* add, int shares, int64_t share_stride, int64_t ld_add, float* total, int64_t ld_total,
                                const float* w, float eps, int64_t rows, int64_t k, hipStream_t stream) {
  if (!sizes_fit("rmsnorm_mx", kind, rows, k)) return 1;
  ALOFA_REQUIRE(out && x && w && aligned16(out) && shares >= 0 && (shares == 0 || add) && (shares == 0 || total) && ldx >= 0 && ld_add >= 0 && share_stride >= 0 && ld_total >= 0 && eps > 0.f,
                "rmsnorm_mx: operands do not fit: shares=%d eps=%g", shares, static_cast<double>(eps));
  {
    const MxPlace held = MxPlace::held(out, rows, k, kind), from = MxPlace::numbers(x, ldx, rows, k, 4), sum = MxPlace::numbers(total, ld_total, rows, k, 4), weights = MxPlace::run(w, 4 * k);
    bool meet = held.meets(from) || held.meets(sum) || held.meets(weights) || sum.meets(weights) || ((total != x || (rows > 1 && ld_total != ldx)) && sum.meets(from));
    for (int s = 0; s < shares; ++s) {
      const MxPlace share = MxPlace::numbers(add + s * share_stride, ld_add, rows, k, 4);
      meet = meet || held.meets(share) || sum.meets(share);
    }
    ALOFA_REQUIRE(!meet, "rmsnorm_mx: what is written overlaps what is read (the sum may take the place of x itself)");
  }
  const int k_tiles = static_cast<int>(mx_tiles(k, 128)), n = static_cast<int>(k), units = 16 * k_tiles;
  const int threads = units <= 256 ? 256 : units <= 512 ? 512 : units <= 768 ? 768 : units <= 1024 ? 1024 : 256;
  ALOFA_REQUIRE(rows * threads < INT64_C(1) << 32, "rmsnorm_mx: more rows than a launch takes: %lld of %lld numbers", static_cast<long long>(rows), static_cast<long long>(k));
  const int64_t at = mx_scales_at(rows, k, kind);
  const bool vec = k % 8 == 0 && aligned16(x) && ldx % 4 == 0 && aligned16(w) && (shares == 0 || (aligned16(add) && ld_add % 4 == 0 && share_stride % 4 == 0)) && (!total || (aligned16(total) && ld_total % 4 == 0));
#define GO(KIND, THREADS, STAY, VEC) rmsnorm_mx_kernel<KIND, THREADS, STAY, VEC><<<static_cast<unsigned>(rows), THREADS, 0, stream>>>(static_cast<uint8_t*>(out), at, x, ldx, add, shares, share_stride, ld_add, total, ld_total, w, eps, n, k_tiles)
#define GO_VEC(KIND, THREADS, STAY) do { if (vec) GO(KIND, THREADS, STAY, true); else GO(KIND, THREADS, STAY, false); } while (0)
#define GO_WIDTH(KIND) do { if (units > 1024) GO_VEC(KIND, 256, false); else if (threads == 256) GO_VEC(KIND, 256, true); else if (threads == 512) GO_VEC(KIND, 512, true); else if (threads == 768) GO_VEC(KIND, 768, true); else GO_VEC(KIND, 1024, true); } while (0)
  if (kind == kE2M1) GO_WIDTH(kE2M1); else GO_WIDTH(kE4M3);
#undef GO_WIDTH
#undef GO_VEC
#undef GO
  return check_launch("rmsnorm_mx");
}
