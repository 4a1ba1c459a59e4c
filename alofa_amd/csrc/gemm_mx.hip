// Products of microscaled rows with microscaled matrices (microscaled.h): out[m, n] = sum_k a[m, k] w[n, k], the matrix in e2m1, the rows in e4m3 or e2m1.
// The matrix cores take elements and scales as they lie in memory and add in float.
//
// Operands of v_mfma_scale_f32_16x16x128_f8f6f4, lane l: e2m1: row l % 16, the 32 numbers from 32 (l / 16) on, in four registers; e4m3: row l % 16, the sixteen from 16 (l / 16) on in
// the first four registers and the sixteen from 64 + 16 (l / 16) on in the other four; a scale: row l % 16, the numbers of block l / 16. The matrix is the first operand: acc[e]
// holds its row 4 (l / 16) + e against the activations' row l % 16, four outputs that lie side by side.
#include "gemm_mx.h"

#include <initializer_list>

namespace alofa {

template <int kKind>
struct MxFragment {
  uint4 half[kKind == kE2M1 ? 1 : 2];
  uint32_t scale;      // of the row's four blocks
  // tile: which of the matrix's; at: the lane's unit of it (its row and group)
  __device__ __forceinline__ void load(const MxMatrix& m, int64_t tile, int at) {
    const uint4* from = reinterpret_cast<const uint4*>(m.units) + tile * mx_units(kKind) + at;
    half[0] = from[0];
    if constexpr (kKind == kE4M3) half[1] = from[64];
    scale = reinterpret_cast<const uint32_t*>(m.scales)[tile * 16 + at % 16];
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

// ---- few rows: the matrix is streamed once -------------------------------------
// A block computes NT tiles of 16 outputs for MT tiles of 16 rows. Its waves share out K tile by tile, every wave with the next tile of the matrix on its way under the products of one; the waves' sums meet in LDS and are
// added in the waves' order. Nothing is waited for together but at the end. Lanes whose row lies behind the last one read the last one again: memory is asked for rows that there are only.
// Up to 16 rows memory bounds it: gate and up of 18,944 x 3,584 take 16.9 us (4.3 TB/s; 27,648 x 5,120 30.8, 4.9), 3,584 x 18,944 8.5 (4.3), 7,168 x 5,120 6.1. What keeps it busy is waves side by side, not tiles ahead: with
// two and three tiles a set, whose registers leave room for fewer, 5,120 x 5,120 against 8 rows took 7.1 and 9.1 us (6.0), gate and up with eight waves a block 22.3.
// With more rows it is what the caches give, 13 TB/s over all compute units (333 rows against 18,944 x 3,584 by 4 x 4 tiles: 622 MB in 48 to 52 us); so rows and matrix are taken by equal numbers of tiles where blocks are many. Where
// they are few, 2 x 4 tiles and eight waves keep more compute units busy: 64 rows against 4,608 x 3,584 take 7.6 us (4 x 4: 10.1; 1 x 4: 11.0), against 18,944 x 3,584 20.8 (17.2).
template <int kAct, int NT, int MT, int kWaves>
__device__ __forceinline__ void mx_stream(const MxMatrix& a, const MxMatrix (&w)[NT], const int (&w_tile)[NT], int M, int first_m_tile, int k_begin, int k_end, int k_tiles, f32x4 (&acc)[NT][MT]) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave, shift = 8 * (lane / 16);
  int64_t a_tile[MT];
  int a_at[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int t = min(first_m_tile + j, a.tiles - 1);
    a_tile[j] = static_cast<int64_t>(t) * k_tiles;
    a_at[j] = lane / 16 * 16 + min(lane % 16, M - 1 - 16 * t);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Two sets of the matrix's fragments, one of the rows': a tile of rows is asked for anew as soon as its registers are free, i.e. taken into the instruction's operands.
  typedef MxFragment<kE2M1> Matrix[NT];
  Matrix w0, w1;
  MxFragment<kAct> rows[MT];
  auto load = [&](Matrix& f, int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NT; ++i) f[i].load(w[i], static_cast<int64_t>(w_tile[i]) * k_tiles + kt, lane);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](const Matrix& f, auto more, int next) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const MxOperand<kAct> a_op(rows[j], shift);
      if constexpr (decltype(more)::value) {
        rows[j].load(a, a_tile[j] + next, a_at[j]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int part = 0; part < (kAct == kE2M1 ? 1 : 2); ++part)      // (an instruction whose sums are those of the one before it waits for them)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const MxOperand<kE2M1> w_op(f[i], shift);
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w_op.part[0], a_op.part[part], acc[i][j], kE2M1, kAct, 0, w_op.scale, 0, a_op.scale);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const int first = k_begin + wave, last = k_end - 1 - (k_end - 1 - first) % kWaves;      // this wave's tiles: first, first + kWaves, .., last
  if (first >= k_end) return;      // (uniform over the wave)
#pragma unroll
  for (int j = 0; j < MT; ++j) rows[j].load(a, a_tile[j] + first, a_at[j]);
  load(w0, first);
  int kt = first;
  for (; kt < last; kt += 2 * kWaves) {      // (behind an even number of tiles the last one is asked for again: a branch around the loads would have the compiler wait for all that are on their way)
    const int after = min(kt + 2 * kWaves, last);
    load(w1, kt + kWaves);
    multiply(w0, std::true_type{}, kt + kWaves);
    load(w0, after);
    multiply(w1, std::true_type{}, after);
  }
  if (kt == last) multiply(w0, std::false_type{}, 0);
}

template <typename TO, int kAct, int NT, int MT, int kWaves>
__global__ void __launch_bounds__(kWaves * kWave, MT == 4 ? 2 : 3) mx_stream_kernel(TO* __restrict__ out, int64_t ldo, int64_t share_stride, MxMatrix a, MxMatrix w, const float* __restrict__ bias, int M, int N,
                                                                   int k_tiles, int epilogue, int vec) {
  __shared__ f32x4 sums[NT * MT][kWaves][kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int shares = gridDim.z, share = blockIdx.z;
  const int k_begin = static_cast<int>(static_cast<int64_t>(k_tiles) * share / shares), k_end = static_cast<int>(static_cast<int64_t>(k_tiles) * (share + 1) / shares);
  MxMatrix ws[NT];
  int tiles[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) ws[i] = w, tiles[i] = min(static_cast<int>(blockIdx.x) * NT + i, w.tiles - 1);
  f32x4 acc[NT][MT];
  mx_stream<kAct, NT, MT, kWaves>(a, ws, tiles, M, blockIdx.y * MT, k_begin, k_end, k_tiles, acc);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[i * MT + j][wave][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < NT * MT; f += kWaves) {
    f32x4 v = sums[f][0][lane];
#pragma unroll
    for (int s = 1; s < kWaves; ++s) v += sums[f][s][lane];
    mx_store4(out + share * share_stride, ldo, bias, (blockIdx.y * MT + f % MT) * 16 + lane % 16, (blockIdx.x * NT + f / MT) * 16 + lane / 16 * 4, M, N, v, epilogue, vec != 0);
  }
}

// Gate and up of the same 32 outputs, act(gate) * up, one block of a microscaled row of the output. 18,944 x 3,584: 16.3 us up to 8 rows (4.4 TB/s of matrices), 16.9 at 16, 19.9 at 32, where memory waits for the products;
// four tiles of rows would take 245 registers and 28.0 us at 64, as tiles of 64 x 64 do. The gate is the general form with expf and a division here; the tiles' epilogue, which has more of it to do, takes __expf and `over`, so that a
// row's outputs by the one and by the other differ by more than the order of a sum (2^-15 of a number at most where gates are below 2^7, before it becomes an element).
template <int kAct, int kOut, int MT, int kWaves>
__global__ void __launch_bounds__(kWaves * kWave, MT == 2 ? 2 : 4) mx_stream_gated_kernel(uint8_t* __restrict__ out, int64_t out_scales_at, int out_tiles, MxMatrix a, MxMatrix gate, MxMatrix up, int M, int N,
                                                                         int k_tiles, int gelu) {
  __shared__ f32x4 sums[4][kWaves][kWave];
  __shared__ float acts[16][36];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const MxMatrix ws[4] = {gate, gate, up, up};
  const int t0 = min(2 * static_cast<int>(blockIdx.x), gate.tiles - 1), t1 = min(2 * static_cast<int>(blockIdx.x) + 1, gate.tiles - 1);
  const int tiles[4] = {t0, t1, t0, t1};
  f32x4 acc[4][MT];
  mx_stream<kAct, 4, MT, kWaves>(a, ws, tiles, M, blockIdx.y * MT, 0, k_tiles, k_tiles, acc);
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

constexpr int64_t kMxMostRows = 65535 * 64;      // (what the streaming kernel's grid has room for)

static bool product_fits(const char* what, const void* a, int a_kind, const void* w, int64_t M, int64_t N, int64_t K) {
  const bool ok = a && w && reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(w) % 16 == 0 && (a_kind == kE2M1 || a_kind == kE4M3) && M >= 1 && N >= 1 && K >= 1 &&
                  M <= kMxMostRows && N <= (1 << 24) && K <= (1 << 24);
  if (!ok) set_error("%s: operands do not fit: M=%lld N=%lld K=%lld kind=%d", what, static_cast<long long>(M), static_cast<long long>(N), static_cast<long long>(K), a_kind);
  return ok;
}

// The shares of a sum added up in their order, on to the epilogue. A thread takes four outputs of a row. A launch's own time bounds it where shares pay: 64 x 3,584 of four shares 4.6 us, 32 x 3,584 of two 3.6.
template <typename TO>
__global__ void __launch_bounds__(256) mx_sum_kernel(TO* __restrict__ out, int64_t ldo, const float* __restrict__ parts, int shares, const float* __restrict__ bias, int M, int N, int epilogue, int vec) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int quads = (N + 3) / 4;
  const int m = static_cast<int>(i / quads), n = static_cast<int>(i % quads) * 4;
  if (m >= M) return;
  const int64_t share = static_cast<int64_t>(M) * N;
  const float* at = parts + static_cast<int64_t>(m) * N + n;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < shares; ++s, at += share) {
    if (N % 4 == 0) {
      const float4 x = *reinterpret_cast<const float4*>(at);
      v += f32x4{x.x, x.y, x.z, x.w};
    } else {
      for (int e = 0; e < 4; ++e)
        if (n + e < N) v[e] += at[e];
    }
  }
  mx_store4(out, ldo, bias, m, n, M, N, v, epilogue, vec != 0);
}

// What a product takes in each form, in us, and how it is chosen: besides + more (each - 1) + turns max(alone, each * of_each), where a compute unit has `each` blocks and a block takes `step` slabs of 128 along K in a
// turn. Fitted to 2,412 timings of 360 products (1 to 2,048 rows, the streaming kernel's up to 512, matrices of 1,152 x 896 to 18,944 x 3,584 and 3,584 x 18,944; 3 % off in the mean with e4m3, 6 % with e2m1).
// Of 500 other products and gated products (1 to 2,048 rows, any widths of 300 to 27,648) the form it takes is 0.8 % slower than the quickest in the mean with e4m3 (1.24 times at worst), 2.7 % with e2m1 (1.45). Read along a column: tiles of 256 x 256 pay where all
// compute units have some, small ones and the streaming kernel where blocks are few: 333 rows against 4,608 x 3,584 take 16.7 us by 64 x 64 streamed, 18.3 and 18.8 by tiles of 64 x 64 and 64 x 128, 25.5 by 128 x 128 and 40.8 by
// 256 x 128; 700 rows against 18,944 x 3,584 95.8, 90.7, 89.8, 79.9 and 85.7. A sum that is shared out over K takes a launch more, which adds the shares up, unless a norm does.
struct MxCost {
  int form, rows, columns, step;
  float alone, of_each, besides, more;
};
constexpr MxCost kMxTiles8[] = {{kMx256x256, 256, 256, 1, 2.31f, 2.31f, 7.9f, 9.7f},  {kMx256x192, 256, 192, 1, 1.87f, 1.87f, 6.6f, 5.8f}, {kMx256x160, 256, 160, 1, 1.63f, 1.63f, 6.5f, 7.8f},
                                {kMx256x128, 256, 128, 1, 1.35f, 1.35f, 5.5f, 4.3f},  {kMx128x128, 128, 128, 1, 0.76f, 0.65f, 5.3f, 1.6f}, {kMx128x64, 128, 64, 1, 0.52f, 0.43f, 4.2f, 0.8f},
                                {kMx64x128, 64, 128, 1, 0.48f, 0.42f, 4.4f, 0.9f},    {kMx64x64, 64, 64, 1, 0.35f, 0.22f, 4.2f, 0.5f}};
constexpr MxCost kMxTiles4[] = {{kMx256x256, 256, 256, 1, 0.82f, 0.82f, 7.8f, 10.2f}, {kMx256x192, 256, 192, 1, 0.73f, 0.74f, 6.1f, 5.5f}, {kMx256x160, 256, 160, 1, 0.61f, 0.61f, 6.5f, 9.3f},
                                {kMx256x128, 256, 128, 1, 0.55f, 0.51f, 5.2f, 1.5f},  {kMx128x128, 128, 128, 1, 0.34f, 0.31f, 5.3f, 1.2f}, {kMx128x64, 128, 64, 1, 0.25f, 0.21f, 4.1f, 0.5f},
                                {kMx64x128, 64, 128, 1, 0.25f, 0.22f, 4.3f, 0.8f},    {kMx64x64, 64, 64, 1, 0.19f, 0.12f, 4.2f, 0.3f}};
// The streaming kernel: for one, two and four tiles of rows, and for one and two with a gate (columns of gate and up together); four by four
constexpr MxCost kMxStream8[] = {{kMxStream, 16, 16, 8, 0.4f, 0.4f, 4.3f, 0.f}, {kMxStream, 32, 32, 8, 0.75f, 0.75f, 4.3f, 0.f}, {kMxStream, 64, 32, 8, 1.09f, 1.09f, 4.3f, 1.5f},
                                 {kMxStream, 16, 64, 4, 0.6f, 0.6f, 4.3f, 0.f}, {kMxStream, 32, 64, 4, 0.59f, 0.59f, 4.3f, 0.4f}};
constexpr MxCost kMxStream4[] = {{kMxStream, 16, 16, 8, 0.25f, 0.25f, 4.3f, 0.f}, {kMxStream, 32, 32, 8, 0.45f, 0.45f, 4.3f, 0.f}, {kMxStream, 64, 32, 8, 0.47f, 0.47f, 4.3f, 0.5f},
                                 {kMxStream, 16, 64, 4, 0.55f, 0.55f, 4.3f, 0.f}, {kMxStream, 32, 64, 4, 0.55f, 0.55f, 4.3f, 0.f}};
constexpr MxCost kMxWide8 = {kMxStream64x64, 64, 64, 4, 0.87f, 0.77f, 4.3f, 1.1f}, kMxWide4 = {kMxStream64x64, 64, 64, 4, 0.45f, 0.36f, 4.3f, 1.5f};
constexpr int kMxStreamRows = 2048;      // most rows that the streaming kernel is weighed for. 382 products of 513 to 2,048 rows for which the rule takes it, beside every other form: with e4m3 0.4 % slower than the quickest in the mean (1.11 times at worst; without it 15 to 45 %), with e2m1 6 %, where rows are long (20,000 numbers) 1.3 to 1.55 times

struct MxPlan {
  int form, shares;
  float us;
};

// tiles of rows that a block of the streaming kernel takes
static int stream_tiles(int64_t M, bool gated) { return M > 32 && !gated ? 4 : M > 16 ? 2 : 1; }

// The quickest form for so many shares
static MxPlan plan_for(int64_t M, int64_t N, int k_tiles, int kind, bool gated, int shares) {
  MxPlan best = {kMx64x64, shares, 0.f};
  const int64_t units = compute_units(), slabs = mx_tiles(k_tiles, shares);
  auto consider = [&](const MxCost& c) {
    const int64_t blocks = mx_tiles(M, c.rows) * mx_tiles(N, c.columns) * shares;
    const float each = static_cast<float>(mx_tiles(blocks, units)), us = c.besides + c.more * (each - 1.f) + static_cast<float>(mx_tiles(slabs, c.step)) * fmaxf(c.alone, each * c.of_each);
    if (best.us == 0.f || us < best.us) best = {c.form, shares, us};
  };
  const bool few = kind == kE2M1;
  if (M <= kMxStreamRows) {
    const int mt = stream_tiles(M, gated), which = (gated ? 3 : 0) + mt / 2;
    consider(few ? kMxStream4[which] : kMxStream8[which]);
    if (mt == 4) consider(few ? kMxWide4 : kMxWide8);
  }
  if (M > 16)
    for (const MxCost& c : few ? kMxTiles4 : kMxTiles8)
      if (!gated || c.form != kMx256x160) consider(c);
  return best;
}

// ... and for any number of them
static MxPlan plan_of(int64_t M, int64_t N, int k_tiles, int kind, bool norm_adds) {
  MxPlan best = plan_for(M, N, k_tiles, kind, false, 1);
  for (int shares : {2, 3, 4, 6, 8}) {
    if (shares * 4 > k_tiles) break;
    MxPlan p = plan_for(M, N, k_tiles, kind, false, shares);
    p.us += static_cast<float>(shares) * static_cast<float>(M) * static_cast<float>(N) * 2e-6f + (norm_adds ? 0.5f : 3.5f);
    if (p.us < best.us) best = p;
  }
  return best;
}

static int product_shares(void* out, int dtype, int64_t ldo, int shares, int64_t share_stride, const void* a, int a_kind, const void* w, const float* bias, int64_t M, int64_t N, int64_t K, int epilogue, int form,
                          int vec, hipStream_t stream) {
  const int k_tiles = static_cast<int>(mx_tiles(K, 128));
  const MxMatrix ma = matrix_of(a, M, K, a_kind), mw = matrix_of(w, N, K, kE2M1);
  if (form != kMxStream && form != kMxStream64x64) return launch_mx_tiles(form, out, dtype, ldo, shares, share_stride, ma, a_kind, mw, bias, static_cast<int>(M), static_cast<int>(N), k_tiles, epilogue, vec, stream);
  const int mt = form == kMxStream64x64 ? 4 : stream_tiles(M, false), nt = form == kMxStream64x64 ? 4 : mt > 1 ? 2 : 1;
  ALOFA_REQUIRE(shares <= 65535, "gemm_mx: more shares than the streaming kernel's grid has room for: %d", shares);
  const dim3 grid((mw.tiles + nt - 1) / nt, (ma.tiles + mt - 1) / mt, shares);
#define GO(T, ACT, NT, MT, WAVES) mx_stream_kernel<T, ACT, NT, MT, WAVES><<<grid, WAVES * 64, 0, stream>>>(static_cast<T*>(out), ldo, share_stride, ma, mw, bias, static_cast<int>(M), static_cast<int>(N), k_tiles, epilogue, vec)
#define GO_FORM(T, ACT) do { if (nt == 4) GO(T, ACT, 4, 4, 4); else if (mt == 4) GO(T, ACT, 2, 4, 8); else if (mt == 2) GO(T, ACT, 2, 2, 8); else GO(T, ACT, 1, 1, 8); } while (0)
  if (dtype == kF32) { if (a_kind == kE2M1) GO_FORM(float, kE2M1); else GO_FORM(float, kE4M3); }
  else { if (a_kind == kE2M1) GO_FORM(bf16_t, kE2M1); else GO_FORM(bf16_t, kE4M3); }
#undef GO_FORM
#undef GO
  return check_launch("gemm_mx");
}

}  // namespace alofa

using namespace alofa;

// Into how many shares of K the product of M rows of a kind with an [N, K] matrix is cut: by alofa_gemm_mx, whose `parts` then has room for [shares, M, N] floats; or where a norm adds them up
extern "C" int alofa_gemm_mx_shares(int64_t M, int64_t N, int64_t K, int kind, int norm_adds) {
  return M < 1 || N < 1 || K < 1 || K > (1 << 24) ? 1 : plan_of(M, N, static_cast<int>(mx_tiles(K, 128)), kind, norm_adds != 0).shares;
}

// out (dtype) = a w^T (+ bias), or += with the residual epilogue (float). shares > 1: the sums over as many parts of K are left in `parts` [shares, M, N]; with `out` they are added up from there.
extern "C" int alofa_gemm_mx(void* out, int dtype, int64_t ldo, int shares, float* parts, const void* a, int a_kind, const void* w, const float* bias, int64_t M, int64_t N, int64_t K,
                             int epilogue, int form, hipStream_t stream) {
  if (!product_fits("gemm_mx", a, a_kind, w, M, N, K)) return 1;
  ALOFA_REQUIRE((out || parts) && (dtype == kF32 || dtype == kBF16) && ldo >= 0 && (epilogue == kMxStore || (epilogue == kMxResidual && dtype == kF32 && !bias)), "gemm_mx: output does not fit: dtype=%d epilogue=%d", dtype, epilogue);
  const int k_tiles = static_cast<int>(mx_tiles(K, 128));
  ALOFA_REQUIRE(shares >= 1 && shares <= k_tiles && (out == nullptr || (shares > 1) == (parts != nullptr)) && reinterpret_cast<uintptr_t>(parts) % 16 == 0, "gemm_mx: shares=%d K=%lld", shares, static_cast<long long>(K));
  ALOFA_REQUIRE(form >= -1 && form < kMxForms, "gemm_mx: form=%d", form);
  {
    const MxPlace read[] = {MxPlace::held(a, M, K, a_kind), MxPlace::held(w, N, K, kE2M1), MxPlace::run(bias, 4 * N)}, to = MxPlace::numbers(out, ldo, M, N, dtype == kF32 ? 4 : 2), sums = MxPlace::run(parts, shares * M * N * 4);
    bool meet = to.meets(sums);
    for (const MxPlace& r : read) meet = meet || to.meets(r) || sums.meets(r);
    ALOFA_REQUIRE(!meet, "gemm_mx: what is written overlaps what is read");
  }
  if (form < 0) form = plan_for(M, N, k_tiles, a_kind, false, shares).form;
  auto aligned = [](const void* p, int64_t ld, int code) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % (code == kF32 ? 4 : 8) == 0; };
  const int out_vec = out && aligned(out, ldo, dtype);
  if (parts) {
    const int rc = product_shares(parts, kF32, N, shares, M * N, a, a_kind, w, nullptr, M, N, K, kMxStore, form, N % 4 == 0, stream);
    if (rc || !out) return rc;
    const int64_t blocks = mx_tiles(M * mx_tiles(N, 4), 256);
    ALOFA_REQUIRE(blocks < 1 << 24, "gemm_mx: more outputs than a launch takes: M=%lld N=%lld", static_cast<long long>(M), static_cast<long long>(N));
    if (dtype == kF32) mx_sum_kernel<float><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<float*>(out), ldo, parts, shares, bias, static_cast<int>(M), static_cast<int>(N), epilogue, out_vec);
    else mx_sum_kernel<bf16_t><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<bf16_t*>(out), ldo, parts, shares, bias, static_cast<int>(M), static_cast<int>(N), epilogue, out_vec);
    return check_launch("gemm_mx");
  }
  return product_shares(out, dtype, ldo, 1, 0, a, a_kind, w, bias, M, N, K, epilogue, form, out_vec, stream);
}

// out (microscaled rows [M, N]) = act(a gate^T) * (a up^T)
extern "C" int alofa_gemm_swiglu_mx(void* out, int out_kind, const void* a, int a_kind, const void* gate, const void* up, int64_t M, int64_t N, int64_t K, int gelu, int form, hipStream_t stream) {
  if (!product_fits("gemm_swiglu_mx", a, a_kind, gate, M, N, K) || !product_fits("gemm_swiglu_mx", a, a_kind, up, M, N, K)) return 1;
  ALOFA_REQUIRE(out && reinterpret_cast<uintptr_t>(out) % 16 == 0 && (out_kind == kE2M1 || out_kind == kE4M3), "gemm_swiglu_mx: output does not fit: kind=%d", out_kind);
  const MxPlace held = MxPlace::held(out, M, N, out_kind);
  ALOFA_REQUIRE(!held.meets(MxPlace::held(a, M, K, a_kind)) && !held.meets(MxPlace::held(gate, N, K, kE2M1)) && !held.meets(MxPlace::held(up, N, K, kE2M1)), "gemm_swiglu_mx: what is written overlaps what is read");
  const int k_tiles = static_cast<int>(mx_tiles(K, 128)), out_tiles = static_cast<int>(mx_tiles(N, 128));
  const MxMatrix ma = matrix_of(a, M, K, a_kind), mg = matrix_of(gate, N, K, kE2M1), mu = matrix_of(up, N, K, kE2M1);
  const int64_t at = mx_scales_at(M, N, out_kind);
  ALOFA_REQUIRE(form >= -1 && form < kMxForms, "gemm_swiglu_mx: form=%d", form);
  if (form < 0) form = plan_for(M, 256 * static_cast<int64_t>(out_tiles), k_tiles, a_kind, true, 1).form;
  if (form != kMxStream) return launch_mx_tiles_gated(form, static_cast<uint8_t*>(out), out_kind, at, out_tiles, ma, a_kind, mg, mu, static_cast<int>(M), static_cast<int>(N), k_tiles, gelu != 0, stream);
  const int mt = stream_tiles(M, true);
  ALOFA_REQUIRE(mx_tiles(ma.tiles, mt) <= 65535, "gemm_swiglu_mx: more rows than the streaming kernel's grid has room for: %lld", static_cast<long long>(M));
  const dim3 grid(4 * out_tiles, (ma.tiles + mt - 1) / mt);
#define GO(ACT, OUT, MT) mx_stream_gated_kernel<ACT, OUT, MT, 4><<<grid, 256, 0, stream>>>(static_cast<uint8_t*>(out), at, out_tiles, ma, mg, mu, static_cast<int>(M), static_cast<int>(N), k_tiles, gelu)
#define GO_MT(ACT, OUT) do { if (mt == 1) GO(ACT, OUT, 1); else GO(ACT, OUT, 2); } while (0)
  if (a_kind == kE2M1) { if (out_kind == kE2M1) GO_MT(kE2M1, kE2M1); else GO_MT(kE2M1, kE4M3); }
  else { if (out_kind == kE2M1) GO_MT(kE4M3, kE2M1); else GO_MT(kE4M3, kE4M3); }
#undef GO_MT
#undef GO
  return check_launch("gemm_swiglu_mx");
}
