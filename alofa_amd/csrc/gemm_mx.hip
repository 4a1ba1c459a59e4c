// Products of microscaled rows with microscaled matrices (microscaled.h): out[m, n] = sum_k a[m, k] w[n, k], the matrix in e2m1, the rows in e4m3 or e2m1.
// The matrix cores take elements and scales as they lie in memory and add in float.
//
// Operands of v_mfma_scale_f32_16x16x128_f8f6f4, lane l: e2m1: row l % 16, the 32 numbers from 32 (l / 16) on, in four registers; e4m3: row l % 16, the sixteen from 16 (l / 16) on in
// the first four registers and the sixteen from 64 + 16 (l / 16) on in the other four; a scale: row l % 16, the numbers of block l / 16. The matrix is the first operand: acc[e]
// holds its row 4 (l / 16) + e against the activations' row l % 16, four outputs that lie side by side.
#include "gemm_mx.h"

namespace alofa {

template <int kKind>
struct MxFragment {
  uint4 half[kKind == kE2M1 ? 1 : 2];
  uint32_t scale;      // of the row's four blocks
  __device__ __forceinline__ void load(const MxMatrix& m, int row_tile, int k_tile, int k_tiles, int lane) {
    const int64_t tile = static_cast<int64_t>(row_tile) * k_tiles + k_tile;
    const uint4* at = reinterpret_cast<const uint4*>(m.units) + tile * mx_units(kKind) + lane;
    half[0] = at[0];
    if constexpr (kKind == kE4M3) half[1] = at[64];
    scale = reinterpret_cast<const uint32_t*>(m.scales)[tile * 16 + lane % 16];
  }
};

// What goes through the instruction: e2m1 once, e4m3 in two parts
template <int kKind>
struct MxOperand {
  i32x8 part[kKind == kE2M1 ? 1 : 2];
  int scale;      // (its low byte)
  __device__ __forceinline__ MxOperand(const MxFragment<kKind>& f, int shift) {
    const uint32_t a[4] = {f.half[0].x, f.half[0].y, f.half[0].z, f.half[0].w};
    if constexpr (kKind == kE2M1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[0][i] = static_cast<int>(a[i]), part[0][4 + i] = 0;
    } else {
      const uint32_t b[4] = {f.half[1].x, f.half[1].y, f.half[1].z, f.half[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t large, small;
        mx_apart(i < 4 ? a[i] : b[i - 4], large, small);
        part[0][i] = static_cast<int>(small), part[1][i] = static_cast<int>(large);
      }
    }
    scale = static_cast<int>(f.scale >> shift);
  }
};

template <int kAct>
__device__ __forceinline__ f32x4 mx_multiply(const MxOperand<kE2M1>& w, const MxOperand<kAct>& a, f32x4 acc) {
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.part[0], a.part[0], acc, kE2M1, kAct, 0, w.scale, 0, a.scale);
  if constexpr (kAct == kE4M3) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.part[0], a.part[1], acc, kE2M1, kAct, 0, w.scale, 0, a.scale);
  return acc;
}

// ---- few rows: the matrix is streamed once -------------------------------------
// A block computes NT tiles of 16 outputs for MT tiles of 16 rows. Its waves share out K tile by tile, every wave with U tiles of 128 on their way; the waves' sums meet in
// LDS and are added in the waves' order.
template <int kAct, int NT, int MT, int kWaves, int U>
__device__ __forceinline__ void mx_stream(const MxMatrix& a, const MxMatrix (&w)[NT], const int (&w_tile)[NT], int first_m_tile, int k_begin, int k_end, int k_tiles, f32x4 (&acc)[NT][MT]) {
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, shift = 8 * (lane / 16);
  int a_tile[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) a_tile[j] = min(first_m_tile + j, a.tiles - 1);      // (results of rows behind the last are not stored)
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kt = k_begin + wave; kt < k_end; kt += kWaves * U) {
    MxFragment<kE2M1> fw[U][NT];
    MxFragment<kAct> fa[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(kt + u * kWaves, k_end - 1);
#pragma unroll
      for (int i = 0; i < NT; ++i) fw[u][i].load(w[i], w_tile[i], at, k_tiles, lane);
#pragma unroll
      for (int j = 0; j < MT; ++j) fa[u][j].load(a, a_tile[j], at, k_tiles, lane);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kt + u * kWaves >= k_end) break;      // (uniform over the wave)
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        const MxOperand<kAct> a_op(fa[u][j], shift);
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[i][j] = mx_multiply<kAct>(MxOperand<kE2M1>(fw[u][i], shift), a_op, acc[i][j]);
      }
    }
  }
}

template <typename TO, int kAct, int MT, int kWaves, int U>
__global__ void __launch_bounds__(kWaves * kWave) mx_stream_kernel(TO* __restrict__ out, int64_t ldo, int64_t share_stride, MxMatrix a, MxMatrix w, const float* __restrict__ bias, int M, int N,
                                                                   int k_tiles, int epilogue, int vec) {
  __shared__ f32x4 sums[MT][kWaves][kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int shares = gridDim.z, share = blockIdx.z;
  const int k_begin = static_cast<int>(static_cast<int64_t>(k_tiles) * share / shares), k_end = static_cast<int>(static_cast<int64_t>(k_tiles) * (share + 1) / shares);
  const MxMatrix ws[1] = {w};
  const int tiles[1] = {static_cast<int>(blockIdx.x)};
  f32x4 acc[1][MT];
  mx_stream<kAct, 1, MT, kWaves, U>(a, ws, tiles, blockIdx.y * MT, k_begin, k_end, k_tiles, acc);
#pragma unroll
  for (int j = 0; j < MT; ++j) sums[j][wave][lane] = acc[0][j];
  __syncthreads();
  if (wave >= MT) return;
  f32x4 v = sums[wave][0][lane];
#pragma unroll
  for (int s = 1; s < kWaves; ++s) v += sums[wave][s][lane];
  mx_store4(out + share * share_stride, ldo, bias, (blockIdx.y * MT + wave) * 16 + lane % 16, blockIdx.x * 16 + lane / 16 * 4, M, N, v, epilogue, vec != 0);
}

// Gate and up of the same 32 outputs, act(gate) * up, one block of a microscaled row of the output.
template <int kAct, int kOut, int MT, int kWaves, int U>
__global__ void __launch_bounds__(kWaves * kWave) mx_stream_gated_kernel(uint8_t* __restrict__ out, int64_t out_scales_at, int out_tiles, MxMatrix a, MxMatrix gate, MxMatrix up, int M, int N,
                                                                         int k_tiles, int gelu) {
  __shared__ f32x4 sums[4][kWaves][kWave];
  __shared__ float acts[16][36];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const MxMatrix ws[4] = {gate, gate, up, up};
  const int t0 = min(2 * static_cast<int>(blockIdx.x), gate.tiles - 1), t1 = min(2 * static_cast<int>(blockIdx.x) + 1, gate.tiles - 1);
  const int tiles[4] = {t0, t1, t0, t1};
  f32x4 acc[4][MT];
  mx_stream<kAct, 4, MT, kWaves, U>(a, ws, tiles, blockIdx.y * MT, 0, k_tiles, k_tiles, acc);
  for (int j = 0; j < MT; ++j) {
    __syncthreads();
#pragma unroll
    for (int jj = 0; jj < MT; ++jj)
      if (jj == j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i][wave][lane] = acc[i][jj];
      }
    __syncthreads();
    if (wave < 2) {
      f32x4 g = sums[wave][0][lane], u = sums[wave + 2][0][lane];
#pragma unroll
      for (int s = 1; s < kWaves; ++s) g += sums[wave][s][lane], u += sums[wave + 2][s][lane];
      const int n = wave * 16 + lane / 16 * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) acts[lane % 16][n + e] = static_cast<int>(blockIdx.x) * 32 + n + e < N ? gate_of(g[e], gelu != 0) * u[e] : 0.f;
    }
    __syncthreads();
    const int row = lane / 4, m = (blockIdx.y * MT + j) * 16 + row;
    if (wave == 0 && m < M) {
      float v[8];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acts[row][lane % 4 * 8 + e], top = max(top, mx_magnitude(v[e]));
      const uint32_t code = mx_scale_of<kOut>(quad_max(top));
      uint32_t q[2];
      mx_pack8<kOut>(v, code, q);
      const int c = static_cast<int>(blockIdx.x) * 4 + lane % 4;
      uint8_t* to = out + mx_place8<kOut>(m, c, out_tiles);
      if constexpr (kOut == kE2M1) *reinterpret_cast<uint32_t*>(to) = q[0];
      else *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
      if (lane % 4 == 0) out[out_scales_at + mx_scale_place(m, blockIdx.x, out_tiles)] = static_cast<uint8_t>(code);
    }
  }
}

static MxMatrix matrix_of(const void* p, int64_t rows, int64_t k, int kind) {
  const uint8_t* at = static_cast<const uint8_t*>(p);
  return {at, at + mx_scales_at(rows, k, kind), static_cast<int>(mx_tiles(rows, 16))};
}

static bool product_fits(const char* what, const void* a, int a_kind, const void* w, int64_t M, int64_t N, int64_t K) {
  const bool ok = a && w && reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && (a_kind == kE2M1 || a_kind == kE4M3) && M >= 1 && N >= 1 && K >= 1 &&
                  M <= (1 << 20) && N <= (1 << 24) && K <= (1 << 24);
  if (!ok) set_error("%s: operands do not fit: M=%lld N=%lld K=%lld kind=%d", what, static_cast<long long>(M), static_cast<long long>(N), static_cast<long long>(K), a_kind);
  return ok;
}

// Tiles, and what a block of them takes: us a slab of 128 where a compute unit has one block, where it has several (each), and besides the slabs. Measured at 64 to 1,024 blocks of 16 and 48 slabs.
struct MxCost {
  int form, rows, columns;
  float alone, each, besides;
};
constexpr MxCost kMxRows8[] = {{kMx256x256, 256, 256, 2.58f, 2.58f, 11.f}, {kMx256x192, 256, 192, 2.05f, 2.05f, 9.f},  {kMx256x160, 256, 160, 1.85f, 1.78f, 8.f}, {kMx256x128, 256, 128, 1.48f, 1.44f, 7.5f},
                               {kMx128x128, 128, 128, 0.86f, 0.71f, 5.8f}, {kMx128x64, 128, 64, 0.60f, 0.44f, 5.f}, {kMx64x64, 64, 64, 0.57f, 0.31f, 5.f}};
constexpr MxCost kMxRows4[] = {{kMx256x256, 256, 256, 0.99f, 0.99f, 9.5f}, {kMx256x192, 256, 192, 0.82f, 0.83f, 8.5f}, {kMx256x160, 256, 160, 0.72f, 0.74f, 8.f}, {kMx256x128, 256, 128, 0.58f, 0.53f, 7.f},
                               {kMx128x128, 128, 128, 0.40f, 0.30f, 6.f}, {kMx128x64, 128, 64, 0.27f, 0.17f, 5.f}, {kMx64x64, 64, 64, 0.21f, 0.10f, 5.f}};

// Which form a product of M rows with N rows of a matrix (gate and up together) takes: the matrix streamed for up to 64 rows, the tiles that the figures above foretell to be done first for more
static int form_of(int64_t M, int64_t N, int k_tiles, int kind, bool gated, int shares) {
  if (M <= 64) return kMxStream;
  int best = kMx64x64;
  float least = 0.f;
  for (const MxCost& c : kind == kE2M1 ? kMxRows4 : kMxRows8) {
    if (gated && c.form == kMx256x160) continue;
    const int64_t blocks = mx_tiles(M, c.rows) * mx_tiles(N, c.columns) * shares, units = compute_units(), each = mx_tiles(blocks, units);
    const float us = c.besides + 3.f * static_cast<float>(each - 1) + static_cast<float>(mx_tiles(k_tiles, shares)) * fmaxf(c.alone, static_cast<float>(each) * c.each);
    if (least == 0.f || us < least) best = c.form, least = us;
  }
  return best;
}

}  // namespace alofa

using namespace alofa;

// out (dtype) = a w^T (+ bias), or += with the residual epilogue (float). shares > 1: `out` is [shares, M, N] floats, share_stride apart, each the sum over a part of K.
extern "C" int alofa_gemm_mx(void* out, int dtype, int64_t ldo, int shares, int64_t share_stride, const void* a, int a_kind, const void* w, const float* bias, int64_t M, int64_t N, int64_t K,
                             int epilogue, int form, hipStream_t stream) {
  if (!product_fits("gemm_mx", a, a_kind, w, M, N, K)) return 1;
  ALOFA_REQUIRE(out && (dtype == kF32 || dtype == kBF16) && ldo >= 0 && (epilogue == kMxStore || (epilogue == kMxResidual && dtype == kF32 && !bias)), "gemm_mx: output does not fit: dtype=%d epilogue=%d", dtype, epilogue);
  ALOFA_REQUIRE(shares >= 1 && shares <= mx_tiles(K, 128) && (shares == 1 || (dtype == kF32 && epilogue == kMxStore && !bias)), "gemm_mx: shares=%d K=%lld", shares, static_cast<long long>(K));
  const int k_tiles = static_cast<int>(mx_tiles(K, 128));
  const MxMatrix ma = matrix_of(a, M, K, a_kind), mw = matrix_of(w, N, K, kE2M1);
  const int vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo % (dtype == kF32 ? 4 : 8) == 0 && (shares == 1 || share_stride % 4 == 0);
  ALOFA_REQUIRE(form >= -1 && form < kMxForms, "gemm_mx: form=%d", form);
  if (form < 0) form = form_of(M, N, k_tiles, a_kind, false, shares);
  if (form != kMxStream) return launch_mx_tiles(form, out, dtype, ldo, shares, share_stride, ma, a_kind, mw, bias, static_cast<int>(M), static_cast<int>(N), k_tiles, epilogue, vec, stream);
  const int mt = ma.tiles >= 4 ? 4 : ma.tiles >= 2 ? 2 : 1;
  const dim3 grid(mw.tiles, (ma.tiles + mt - 1) / mt, shares);
#define GO(T, ACT, MT) mx_stream_kernel<T, ACT, MT, 8, 4><<<grid, 512, 0, stream>>>(static_cast<T*>(out), ldo, share_stride, ma, mw, bias, static_cast<int>(M), static_cast<int>(N), k_tiles, epilogue, vec)
#define GO_MT(T, ACT) do { if (mt == 1) GO(T, ACT, 1); else if (mt == 2) GO(T, ACT, 2); else GO(T, ACT, 4); } while (0)
  if (dtype == kF32) { if (a_kind == kE2M1) GO_MT(float, kE2M1); else GO_MT(float, kE4M3); }
  else { if (a_kind == kE2M1) GO_MT(bf16_t, kE2M1); else GO_MT(bf16_t, kE4M3); }
#undef GO_MT
#undef GO
  return check_launch("gemm_mx");
}

// out (microscaled rows [M, N]) = act(a gate^T) * (a up^T)
extern "C" int alofa_gemm_swiglu_mx(void* out, int out_kind, const void* a, int a_kind, const void* gate, const void* up, int64_t M, int64_t N, int64_t K, int gelu, int form, hipStream_t stream) {
  if (!product_fits("gemm_swiglu_mx", a, a_kind, gate, M, N, K) || !product_fits("gemm_swiglu_mx", a, a_kind, up, M, N, K)) return 1;
  ALOFA_REQUIRE(out && reinterpret_cast<uintptr_t>(out) % 16 == 0 && (out_kind == kE2M1 || out_kind == kE4M3), "gemm_swiglu_mx: output does not fit: kind=%d", out_kind);
  const int k_tiles = static_cast<int>(mx_tiles(K, 128)), out_tiles = static_cast<int>(mx_tiles(N, 128));
  const MxMatrix ma = matrix_of(a, M, K, a_kind), mg = matrix_of(gate, N, K, kE2M1), mu = matrix_of(up, N, K, kE2M1);
  const int64_t at = mx_scales_at(M, N, out_kind);
  ALOFA_REQUIRE(form >= -1 && form < kMxForms, "gemm_swiglu_mx: form=%d", form);
  if (form < 0) form = form_of(M, 256 * static_cast<int64_t>(out_tiles), k_tiles, a_kind, true, 1);
  if (form != kMxStream) return launch_mx_tiles_gated(form, static_cast<uint8_t*>(out), out_kind, at, out_tiles, ma, a_kind, mg, mu, static_cast<int>(M), static_cast<int>(N), k_tiles, gelu != 0, stream);
  const int mt = ma.tiles >= 2 ? 2 : 1;
  const dim3 grid(4 * out_tiles, (ma.tiles + mt - 1) / mt);
#define GO(ACT, OUT, MT) mx_stream_gated_kernel<ACT, OUT, MT, 8, 2><<<grid, 512, 0, stream>>>(static_cast<uint8_t*>(out), at, out_tiles, ma, mg, mu, static_cast<int>(M), static_cast<int>(N), k_tiles, gelu)
#define GO_MT(ACT, OUT) do { if (mt == 1) GO(ACT, OUT, 1); else GO(ACT, OUT, 2); } while (0)
  if (a_kind == kE2M1) { if (out_kind == kE2M1) GO_MT(kE2M1, kE2M1); else GO_MT(kE2M1, kE4M3); }
  else { if (out_kind == kE2M1) GO_MT(kE4M3, kE2M1); else GO_MT(kE4M3, kE4M3); }
#undef GO_MT
#undef GO
  return check_launch("gemm_swiglu_mx");
}
