// Products of microscaled rows with microscaled matrices by tiles, for many rows.
//
// A block computes 32 NF WN outputs for 32 MF WM rows, a wave NF x MF tiles of 32 x 32 of them (v_mfma_scale_f32_32x32x64_f8f6f4; the matrix is the first operand, so that a lane holds four
// outputs of one row side by side). Slabs of 128 along K come from memory straight into a ring of S slabs in LDS (global_load_lds); elements and scales lie in memory as the
// fragments are read, so a slab is whole runs of 1 KB, one per wave and instruction, and 16 lanes' fragments are 256 bytes in a row: nothing is permuted and no banks meet.
//
// A block of four waves and fewer outputs than a compute unit can work on at once has two teams (KS = 2): each multiplies one half of every slab, 64 along K, and the second's sums go to the first at the end. A wave's own
// products and arithmetic do not overlap (a turn of 357 cycles of products and one of 121 of arithmetic took 469 together), another wave's do: tiles of 64 x 64 took 13.1 us where one team took 18.9 (64 rows against
// 4,608 x 3,584), of 128 x 128 25.4 for 27.8 (and 42.5 for 44.0, 333 rows against 18,944 x 3,584).
// Many rows are bound by the products' rate, at which the card's power allows 4.1 to 4.3 PFLOP/s of e4m3 instructions, i.e. 2.1 of products in two passes, and 5.3 to 6.2 of e2m1: 2,048 x 8,192 x 8,192 runs at 1.7 and 3.9.
//
// Operands of the instruction, lane l: row l % 32; e2m1: the 32 numbers from 32 (l / 32) on; e4m3: the sixteen from 16 (l / 32) on and the sixteen from 32 + 16 (l / 32) on; the scale of block
// l / 32. acc[e] holds the matrix's row 8 (e / 4) + 4 (l / 32) + e % 4 against the activations' row l % 32.
#include "gemm_mx.h"
#include "gemm_tiles.h"

namespace alofa {

template <int kAct, int NF_, int MF_, int WN_, int WM_, int S_, int KS_ = 1>
struct MxTile {
  static constexpr int NF = NF_, MF = MF_, WN = WN_, WM = WM_, S = S_, KS = KS_, kTeam = WN * WM, kWaves = kTeam * KS;
  static constexpr int BN = 32 * NF * WN, BM = 32 * MF * WM;
  static constexpr int kRowsPieces = BM / 16 * (kAct == kE2M1 ? 1 : 2), kPieces = BN / 16 + kRowsPieces;      // of 1 KB
  static_assert((BN + BM) / 64 <= kWaves, "a wave brings the scales of four tiles at most");
  static constexpr int kLoads = (kPieces + kWaves - 1) / kWaves + 1;    // a wave's, per slab (a wave with a piece less brings its first one again)
  static constexpr int kScales = kPieces * 1024, kSlab = kScales + kWaves * 256;
  static_assert(S >= 2 && S * kSlab <= 160 * 1024 && (S - 2) * kLoads < 64, "the ring fits LDS, what is on its way is counted");
  static_assert(KS == 1 || (KS == 2 && kTeam * NF * MF * 4096 <= S * kSlab), "a slab has two halves of 64; their sums meet in the ring");
};

// A wave's loads of a slab have come, and its reads from LDS; those of `behind` slabs behind it, kMost at most, stay on their way.
template <int kMost, int kLoads>
__device__ __forceinline__ void wait_for(int behind) {
  if (behind >= kMost) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(kMost * kLoads) : "memory");
  else if constexpr (kMost > 0) wait_for<kMost - 1, kLoads>(behind);
}

// What a wave multiplies: acc[i][j] of the matrix's i-th 32 rows and the activations' j-th. `gated`: the first half of a wave's 32-row groups is the gate's, the second the same outputs' of up.
template <int kAct, typename T, bool kGated>
__device__ __forceinline__ void mx_tile_product(char* ring, const MxMatrix a, const MxMatrix w, const MxMatrix w2, int m_tile, int n_tile, int k_begin, int k_end, int k_tiles, f32x16 (&acc)[T::NF][T::MF]) {
  constexpr int NF = T::NF, MF = T::MF, S = T::S, kLoads = T::kLoads, kMatrixPieces = T::BN / 16, kHalf = kMatrixPieces / 2;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int wn = wave % T::WN, wm = wave % T::kTeam / T::WN, team = wave / T::kTeam;

  // what this wave brings: pieces wave, wave + kWaves, ..; a piece is a run of 1 KB (tiles behind the last of a matrix come from the last; their results are not stored)
  const uint8_t *const units = w.units, *const up_units = w2.units, *const scales_of = w.scales, *const up_scales = w2.scales;
  const uint8_t* from[kLoads - 1];
  int step[kLoads - 1], piece[kLoads - 1];
#pragma unroll
  for (int i = 0; i < kLoads - 1; ++i) {
    const int p = piece[i] = wave + i * T::kWaves < T::kPieces ? wave + i * T::kWaves : wave;
    if (p < kMatrixPieces) {
      const bool second = kGated && p >= kHalf;
      const int t = min(n_tile + (second ? p - kHalf : p), w.tiles - 1);
      from[i] = (second ? up_units : units) + (static_cast<int64_t>(t) * k_tiles + k_begin) * 1024;
      step[i] = 1024;
    } else {
      const int q = p - kMatrixPieces, t = min(m_tile + (kAct == kE2M1 ? q : q / 2), a.tiles - 1);
      from[i] = a.units + (static_cast<int64_t>(t) * k_tiles + k_begin) * (mx_units(kAct) * 16) + (kAct == kE2M1 ? 0 : q % 2 * 1024);
      step[i] = mx_units(kAct) * 16;
    }
  }
  // ... and the scales of four tiles, the matrix's first
  const uint8_t* scales_from;
  {
    const int p = min(4 * wave + lane / 16, kMatrixPieces + T::BM / 16 - 1);
    const uint8_t* base;
    int t;
    if (p < kMatrixPieces) {
      const bool second = kGated && p >= kHalf;
      t = min(n_tile + (second ? p - kHalf : p), w.tiles - 1);
      base = second ? up_scales : scales_of;
    } else {
      t = min(m_tile + p - kMatrixPieces, a.tiles - 1);
      base = a.scales;
    }
    scales_from = base + (static_cast<int64_t>(t) * k_tiles + k_begin) * 64 + lane % 16 * 4;
  }
  // (Written out as instructions: the compiler, which cannot tell the ring's slabs apart, would wait for every load on its way before any read from LDS. M0 holds the LDS address of the
  // wave's first lane.)
  const unsigned ring_at = static_cast<unsigned>(reinterpret_cast<uintptr_t>(ring));
  const unsigned lane_at = lane * 16;
  auto bring = [&](unsigned slab_at) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLoads - 1; ++i) {
      const uint64_t run = reinterpret_cast<uint64_t>(from[i]);      // (the wave's own: said to the compiler, which keeps it in vector registers otherwise)
      const uint64_t base = (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(run >> 32)))) << 32) |
                            static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(run)));
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :: "s"(__builtin_amdgcn_readfirstlane(ring_at + slab_at + piece[i] * 1024)), "v"(lane_at), "s"(base), "r"(ring) : "memory", "m0");
      from[i] += step[i];
    }
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(ring_at + slab_at + T::kScales + wave * 256)), "v"(scales_from), "r"(ring) : "memory", "m0");
    scales_from += 64;
  };

#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int j = 0; j < MF; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // where this lane's fragments lie within a slab
  const int half = lane / 32, shift = 8 * half + 16 * team, in_tile = lane % 16 * 16;
  int w_tile[NF], a_tile[MF];
#pragma unroll
  for (int i = 0; i < NF; ++i) w_tile[i] = kGated ? (i < NF / 2 ? (wn * (NF / 2) + i) * 2 : kHalf + (wn * (NF / 2) + i - NF / 2) * 2) : (wn * NF + i) * 2;
#pragma unroll
  for (int j = 0; j < MF; ++j) a_tile[j] = (wm * MF + j) * 2;
  const int odd = lane % 32 / 16;

  auto multiply = [&](const char* slab) __attribute__((always_inline)) {
    const uint32_t* scales = reinterpret_cast<const uint32_t*>(slab + T::kScales) + lane % 32;
    int ws[NF], as[MF];
#pragma unroll
    for (int i = 0; i < NF; ++i) ws[i] = static_cast<int>(scales[w_tile[i] * 16] >> shift);
#pragma unroll
    for (int j = 0; j < MF; ++j) as[j] = static_cast<int>(scales[(kMatrixPieces + a_tile[j]) * 16] >> shift);
    auto step64 = [&](auto number) __attribute__((always_inline)) {
      constexpr int s = decltype(number)::value;
      i32x8 wf[NF], af[MF][kAct == kE2M1 ? 1 : 2];
#pragma unroll
      for (int i = 0; i < NF; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(slab + (w_tile[i] + odd) * 1024 + (2 * (s + team) + half) * 256 + in_tile);
        wf[i] = {static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < MF; ++j) {
        const char* rows = slab + kMatrixPieces * 1024;
        if constexpr (kAct == kE2M1) {
          const uint4 v = *reinterpret_cast<const uint4*>(rows + (a_tile[j] + odd) * 1024 + (2 * (s + team) + half) * 256 + in_tile);
          af[j][0] = {static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0};
        } else {
          const char* at = rows + (a_tile[j] + odd) * 2048 + (4 * (s + team) + half) * 256 + in_tile;
          const uint4 lo = *reinterpret_cast<const uint4*>(at), hi = *reinterpret_cast<const uint4*>(at + 512);
          const uint32_t x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t large, small;
            mx_apart(x[e], large, small);
            af[j][0][e] = static_cast<int>(small), af[j][1][e] = static_cast<int>(large);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < MF; ++j)
#pragma unroll
        for (int part = 0; part < (kAct == kE2M1 ? 1 : 2); ++part)
#pragma unroll
          for (int i = 0; i < NF; ++i) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[i], af[j][part], acc[i][j], kE2M1, kAct, 2 * s, ws[i], 2 * s, as[j]);
    };
    step64(std::integral_constant<int, 0>{});
    if constexpr (T::KS == 1) step64(std::integral_constant<int, 1>{});
  };

  // Slab k + S - 1 is set out once every wave has read slab k - 1, whose place it takes, i.e. behind the barrier of step k. A wave waits for its own loads of slab k (those of the S - 2 behind it
  // stay on their way) before the barrier; behind the barrier all of the slab is there.
  unsigned next_at = 0, at = 0;
  const auto advance = [](unsigned x) { return x == (S - 1) * T::kSlab ? 0u : x + T::kSlab; };
#pragma unroll
  for (int p = 0; p < S - 1; ++p)
    if (k_begin + p < k_end) {
      bring(next_at);
      next_at = advance(next_at);
    }
  for (int k = k_begin; k < k_end; ++k) {
    const int behind = k_end - 1 - k;
    wait_for<S - 2, kLoads>(behind);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (behind >= S - 1) {
      bring(next_at);
      next_at = advance(next_at);
    }
    multiply(ring + at);
    at = advance(at);
  }
  if constexpr (T::KS == 2) {      // the second team's sums, to the first
    __syncthreads();
    float4* sums = reinterpret_cast<float4*>(ring) + wave % T::kTeam * (NF * MF * 256) + lane;
    if (team == 1) {
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) sums[((i * MF + j) * 4 + q) * 64] = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
    }
    __syncthreads();
    if (team == 0) {
#pragma unroll
      for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MF; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 v = sums[((i * MF + j) * 4 + q) * 64];
            acc[i][j][4 * q] += v.x, acc[i][j][4 * q + 1] += v.y, acc[i][j][4 * q + 2] += v.z, acc[i][j][4 * q + 3] += v.w;
          }
    }
  }
}

// A wave's tiles on their way out, by way of LDS (`room`: the wave's own): a lane holds four outputs of one row, and rows leave in runs of up to 256 bytes. G: 32-row groups of the matrix at a time.
template <typename TO>
constexpr int kGroups = sizeof(TO) == 4 ? 2 : 4;
template <typename TO>
constexpr int kRoom = 32 * (kGroups<TO> * 32 * static_cast<int>(sizeof(TO)) + 16);

template <typename TO, int G>
__device__ __forceinline__ void mx_tile_rows(const f32x16* const (&acc)[G], char* room, TO* __restrict__ out, int64_t ldo, const float* __restrict__ bias, int m0, int n0, int M, int N, int epilogue, bool vec, int lane) {
  constexpr int kRow = G * 32 * static_cast<int>(sizeof(TO)) + 16, kEach = 16 / static_cast<int>(sizeof(TO)), kLanes = G * 32 / kEach;      // bytes of a row; numbers of a lane; lanes of a row
  constexpr int kAtOnce = 64 / kLanes, kTimes = 32 / kAtOnce;
  if (n0 >= N || m0 >= M) return;      // (uniform over the wave)
  wave_lds_sync();      // (what was there before has been read)
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      char* at = room + (lane % 32) * kRow + (32 * i + 8 * q + 4 * (lane / 32)) * static_cast<int>(sizeof(TO));
      const float v[4] = {(*acc[i])[4 * q], (*acc[i])[4 * q + 1], (*acc[i])[4 * q + 2], (*acc[i])[4 * q + 3]};
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      if (bias != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = bias[min(n0 + 32 * i + 8 * q + 4 * (lane / 32) + e, N - 1)];
      }
      if constexpr (sizeof(TO) == 4) *reinterpret_cast<float4*>(at) = make_float4(v[0] + b[0], v[1] + b[1], v[2] + b[2], v[3] + b[3]);
      else *reinterpret_cast<uint2*>(at) = make_uint2(pack_bf16x2(v[0] + b[0], v[1] + b[1]), pack_bf16x2(v[2] + b[2], v[3] + b[3]));
    }
  wave_lds_sync();
  const int r0 = lane / kLanes, n = n0 + lane % kLanes * kEach;
  const char* from = room + r0 * kRow + lane % kLanes * 16;
  TO* to = out + static_cast<int64_t>(m0 + r0) * ldo + n;
  if (n >= N) return;
  const int last = M - m0 - r0;      // rows of this lane's steps of kAtOnce
  if (vec && n + kEach <= N) {
    if constexpr (sizeof(TO) == 4) {
      if (epilogue == kMxResidual) {
        float4 old[kTimes];
#pragma unroll
        for (int t = 0; t < kTimes; ++t)
          if (t * kAtOnce < last) old[t] = *reinterpret_cast<const float4*>(to + static_cast<int64_t>(t * kAtOnce) * ldo);
#pragma unroll
        for (int t = 0; t < kTimes; ++t) {
          if (t * kAtOnce >= last) break;
          const float4 v = *reinterpret_cast<const float4*>(from + t * kAtOnce * kRow);
          *reinterpret_cast<float4*>(to + static_cast<int64_t>(t * kAtOnce) * ldo) = make_float4(old[t].x + v.x, old[t].y + v.y, old[t].z + v.z, old[t].w + v.w);
        }
        return;
      }
    }
#pragma unroll
    for (int t = 0; t < kTimes; ++t)
      if (t * kAtOnce < last) *reinterpret_cast<uint4*>(to + static_cast<int64_t>(t * kAtOnce) * ldo) = *reinterpret_cast<const uint4*>(from + t * kAtOnce * kRow);
    return;
  }
  for (int t = 0; t * kAtOnce < last && t < kTimes; ++t) {
    const TO* v = reinterpret_cast<const TO*>(from + t * kAtOnce * kRow);
    TO* row = to + static_cast<int64_t>(t * kAtOnce) * ldo;
    for (int e = 0; e < kEach && n + e < N; ++e) {
      if (sizeof(TO) == 4 && epilogue == kMxResidual) store_f32(row + e, load_f32(row + e) + load_f32(v + e));
      else row[e] = v[e];
    }
  }
}

template <typename TO, int kAct, typename T>
__global__ void __launch_bounds__(T::kWaves * 64) mx_tile_kernel(TO* __restrict__ out, int64_t ldo, int64_t share_stride, MxMatrix a, MxMatrix w, const float* __restrict__ bias, int M, int N, int k_tiles, int tiles_m,
                                                                 int tiles_n, int shares, int epilogue, int vec) {
  __shared__ __attribute__((aligned(1024))) char ring[T::S * T::kSlab];
  const TilePlace place = place_tile(blockIdx.x, tiles_m, tiles_n, shares, true);
  const int k_begin = static_cast<int>(static_cast<int64_t>(k_tiles) * place.share / shares), k_end = static_cast<int>(static_cast<int64_t>(k_tiles) * (place.share + 1) / shares);
  f32x16 acc[T::NF][T::MF];
  mx_tile_product<kAct, T, false>(ring, a, w, w, place.bm * (T::BM / 16), place.bn * (T::BN / 16), k_begin, k_end, k_tiles, acc);
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, wn = wave % T::WN, wm = wave / T::WN;
  out += place.share * share_stride;
  __syncthreads();      // (the ring is free: nothing is on its way, and every wave has read the last slab)
  if (wave >= T::kTeam) return;
  static_assert(T::kTeam * kRoom<TO> <= sizeof(ring), "the rows' way out fits the ring");
  char* room = ring + wave * kRoom<TO>;
#pragma unroll
  for (int j = 0; j < T::MF; ++j) {
    const int m0 = place.bm * T::BM + (wm * T::MF + j) * 32, n0 = place.bn * T::BN + wn * T::NF * 32;
    constexpr int G = kGroups<TO>;
#pragma unroll
    for (int i = 0; i + G <= T::NF; i += G) {
      const f32x16* group[G];
#pragma unroll
      for (int g = 0; g < G; ++g) group[g] = &acc[i + g][j];
      mx_tile_rows<TO, G>(group, room, out, ldo, bias, m0, n0 + 32 * i, M, N, epilogue, vec != 0, lane);
    }
    if constexpr (T::NF % G >= 2) {
      const f32x16* group[2] = {&acc[T::NF / G * G][j], &acc[T::NF / G * G + 1][j]};
      mx_tile_rows<TO, 2>(group, room, out, ldo, bias, m0, n0 + 32 * (T::NF / G * G), M, N, epilogue, vec != 0, lane);
    }
    if constexpr (T::NF % 2 == 1) {
      const f32x16* group[1] = {&acc[T::NF - 1][j]};
      mx_tile_rows<TO, 1>(group, room, out, ldo, bias, m0, n0 + 32 * (T::NF - 1), M, N, epilogue, vec != 0, lane);
    }
  }
}

// Gate and up, act(gate) * up, to microscaled rows: a lane has half the numbers of a block of 32, the lane 32 further on the other half.
template <int kAct, int kOut, typename T, bool kGelu>
__global__ void __launch_bounds__(T::kWaves * 64) mx_tile_gated_kernel(uint8_t* __restrict__ out, int64_t out_scales_at, int out_tiles, MxMatrix a, MxMatrix gate, MxMatrix up, int M, int N, int k_tiles, int tiles_m,
                                                                       int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char ring[T::S * T::kSlab];
  const TilePlace place = place_tile(blockIdx.x, tiles_m, tiles_n, 1, true);
  f32x16 acc[T::NF][T::MF];
  mx_tile_product<kAct, T, true>(ring, a, gate, up, place.bm * (T::BM / 16), place.bn * (T::BN / 32), 0, k_tiles, k_tiles, acc);
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, wn = wave % T::WN, wm = wave / T::WN, half = lane / 32;
  if (wave >= T::kTeam) return;
#pragma unroll
  for (int j = 0; j < T::MF; ++j)
#pragma unroll
    for (int i = 0; i < T::NF / 2; ++i) {
      const int m = place.bm * T::BM + (wm * T::MF + j) * 32 + lane % 32, block = place.bn * (T::BN / 64) + wn * (T::NF / 2) + i;
      if (block >= 4 * out_tiles) continue;      // (uniform over the wave: columns of the last tile behind what the rows are filled up to)
      float v[16];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int n = 32 * block + 8 * (e / 4) + 4 * half + e % 4;
        v[e] = n < N ? gate_of<kGelu>(acc[i][j][e]) * acc[i + T::NF / 2][j][e] : 0.f;
        top = max(top, mx_magnitude(v[e]));
      }
      const auto other = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      const uint32_t code = mx_scale_of<kOut>(max(static_cast<uint32_t>(other[0]), static_cast<uint32_t>(other[1])));
      const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}, hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
      uint32_t x[2], y[2];
      mx_pack8<kOut>(lo, code, x);
      mx_pack8<kOut>(hi, code, y);
      // the lanes exchange what they hold so that each has a run: the lower ones the block's first half, the upper ones its second
      const int64_t tile = static_cast<int64_t>(m / 16) * out_tiles + block / 4;
      if constexpr (kOut == kE4M3) {
        const auto p = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false), q = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
        if (m < M) *reinterpret_cast<uint4*>(out + ((tile * 8 + 2 * (block % 4) + half) * 16 + m % 16) * 16) = make_uint4(p[0], p[1], q[0], q[1]);
      } else {
        const auto p = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
        const uint32_t mine = p[0], its = p[1];      // (four elements of either half, for two runs of eight)
        if (m < M) *reinterpret_cast<uint2*>(out + ((tile * 4 + block % 4) * 16 + m % 16) * 16 + 8 * half) = make_uint2((mine & 0xffffu) | (its << 16), (mine >> 16) | (its & 0xffff0000u));
      }
      if (m < M && half == 0) out[out_scales_at + mx_scale_place(m, block, out_tiles)] = static_cast<uint8_t>(code);
    }
}

namespace {

template <typename TO, int kAct, typename T>
int go(void* out, int64_t ldo, int shares, int64_t share_stride, const MxMatrix& a, const MxMatrix& w, const float* bias, int M, int N, int k_tiles, int epilogue, bool vec, hipStream_t stream) {
  const int tiles_m = (M + T::BM - 1) / T::BM, tiles_n = (N + T::BN - 1) / T::BN;
  const int64_t blocks = static_cast<int64_t>(tiles_m) * tiles_n * shares;
  ALOFA_REQUIRE(blocks * T::kWaves * 64 < INT64_C(1) << 32, "gemm_mx: more tiles than a launch takes: M=%d N=%d shares=%d", M, N, shares);
  mx_tile_kernel<TO, kAct, T><<<static_cast<unsigned>(blocks), T::kWaves * 64, 0, stream>>>(static_cast<TO*>(out), ldo, share_stride, a, w, bias, M, N, k_tiles, tiles_m, tiles_n, shares, epilogue, vec);
  return check_launch("gemm_mx");
}

template <int kAct, int kOut, typename T>
int go_gated(uint8_t* out, int64_t at, int out_tiles, const MxMatrix& a, const MxMatrix& gate, const MxMatrix& up, int M, int N, int k_tiles, bool gelu, hipStream_t stream) {
  const int tiles_m = (M + T::BM - 1) / T::BM, tiles_n = (out_tiles * 128 + T::BN / 2 - 1) / (T::BN / 2);
  const int64_t all = static_cast<int64_t>(tiles_m) * tiles_n;
  ALOFA_REQUIRE(all * T::kWaves * 64 < INT64_C(1) << 32, "gemm_swiglu_mx: more tiles than a launch takes: M=%d N=%d", M, N);
  const unsigned blocks = static_cast<unsigned>(all);
  if (gelu) mx_tile_gated_kernel<kAct, kOut, T, true><<<blocks, T::kWaves * 64, 0, stream>>>(out, at, out_tiles, a, gate, up, M, N, k_tiles, tiles_m, tiles_n);
  else mx_tile_gated_kernel<kAct, kOut, T, false><<<blocks, T::kWaves * 64, 0, stream>>>(out, at, out_tiles, a, gate, up, M, N, k_tiles, tiles_m, tiles_n);
  return check_launch("gemm_swiglu_mx");
}

// Rows by columns of the matrix. A wave of e4m3 has one group of 32 rows, which it takes apart, and as many of the matrix as the tile is wide.
template <int kAct> using T256x256 = MxTile<kAct, kAct == kE2M1 ? 4 : 8, kAct == kE2M1 ? 2 : 1, kAct == kE2M1 ? 2 : 1, kAct == kE2M1 ? 4 : 8, kAct == kE2M1 ? 4 : 3>;
template <int kAct> using T256x192 = MxTile<kAct, 6, 1, 1, 8, 3>;
template <int kAct> using T256x160 = MxTile<kAct, 5, 1, 1, 8, 3>;
template <int kAct> using T256x128 = MxTile<kAct, 4, 1, 1, 8, 3>;
template <int kAct> using T128x128 = MxTile<kAct, 4, 1, 1, 4, kAct == kE2M1 ? 4 : 3, 2>;
template <int kAct> using T128x64 = MxTile<kAct, 2, 1, 1, 4, 3, 2>;
template <int kAct> using T64x128 = MxTile<kAct, 2, 1, 2, 2, 4, 2>;
template <int kAct> using T64x64 = MxTile<kAct, 2, 1, 1, 2, 4, 2>;

}  // namespace

template <int kAct, typename TO>
static int by_form(int form, void* out, int64_t ldo, int shares, int64_t share_stride, const MxMatrix& a, const MxMatrix& w, const float* bias, int M, int N, int k_tiles, int epilogue, bool vec, hipStream_t stream) {
#define GO(T) return go<TO, kAct, T<kAct>>(out, ldo, shares, share_stride, a, w, bias, M, N, k_tiles, epilogue, vec, stream)
  switch (form) {
    case kMx256x256: GO(T256x256);
    case kMx256x192: GO(T256x192);
    case kMx256x160: GO(T256x160);
    case kMx256x128: GO(T256x128);
    case kMx128x128: GO(T128x128);
    case kMx128x64: GO(T128x64);
    case kMx64x128: GO(T64x128);
    default: GO(T64x64);
  }
#undef GO
}

int launch_mx_tiles(int form, void* out, int dtype, int64_t ldo, int shares, int64_t share_stride, const MxMatrix& a, int a_kind, const MxMatrix& w, const float* bias, int M, int N, int k_tiles, int epilogue,
                    bool vec, hipStream_t stream) {
#define GO(ACT, TO) by_form<ACT, TO>(form, out, ldo, shares, share_stride, a, w, bias, M, N, k_tiles, epilogue, vec, stream)
  if (a_kind == kE2M1) return dtype == kF32 ? GO(kE2M1, float) : GO(kE2M1, bf16_t);
  return dtype == kF32 ? GO(kE4M3, float) : GO(kE4M3, bf16_t);
#undef GO
}

template <int kAct, int kOut>
static int by_form_gated(int form, uint8_t* out, int64_t at, int out_tiles, const MxMatrix& a, const MxMatrix& gate, const MxMatrix& up, int M, int N, int k_tiles, bool gelu, hipStream_t stream) {
#define GO(T) return go_gated<kAct, kOut, T<kAct>>(out, at, out_tiles, a, gate, up, M, N, k_tiles, gelu, stream)
  switch (form) {
    case kMx256x256: GO(T256x256);
    case kMx256x192: GO(T256x192);
    case kMx256x128: GO(T256x128);
    case kMx128x128: GO(T128x128);
    case kMx128x64: GO(T128x64);
    case kMx64x128: GO(T64x128);
    case kMx64x64: GO(T64x64);
    default: set_error("gemm_swiglu_mx: gate and up do not share tiles of this form: %d", form); return 1;
  }
#undef GO
}

int launch_mx_tiles_gated(int form, uint8_t* out, int out_kind, int64_t out_scales_at, int out_tiles, const MxMatrix& a, int a_kind, const MxMatrix& gate, const MxMatrix& up, int M, int N, int k_tiles, bool gelu,
                          hipStream_t stream) {
#define GO(ACT, OUT) by_form_gated<ACT, OUT>(form, out, out_scales_at, out_tiles, a, gate, up, M, N, k_tiles, gelu, stream)
  if (a_kind == kE2M1) return out_kind == kE2M1 ? GO(kE2M1, kE2M1) : GO(kE2M1, kE4M3);
  return out_kind == kE2M1 ? GO(kE4M3, kE2M1) : GO(kE4M3, kE4M3);
#undef GO
}

}  // namespace alofa
