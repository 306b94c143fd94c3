// table_loss_few.h -- softmax cross entropy (table_loss.hip) of a few rows against the table: ONE pass over the table forward, one
// backward, which writes dW as it goes.
//
// With 16 rows or less every product is bound by the table's bytes, so what counts is that each is read once, as it lies in memory
// (any alignment, f32 included), with enough of them in flight.  A workgroup takes 16 items at a time; its four waves share the COLUMNS:
// each brings its slice of the items into its own part of the LDS (no barrier), contracts it with its slice of the rows, and the
// four partial logits meet in LDS (one barrier a stage).  Backward each wave then knows g and makes its columns of both gradients:
//   dX (rows x columns, in registers over the whole walk)  A = items transposed (4 of a column a lane), B = g (row, 4 items)
//   dW (16 items x columns, stored at once)                A = rows transposed (kept),                  B = g turned over in LDS (item, 4 rows)
// f32 goes as three bf16 planes, split on the way into the LDS: the matrix pipe has time.
// Up to 128 columns a wave takes whole items instead, each its own stretch of the table, and nothing meets before the end.
// Rows of any alignment go in and out in 16-byte pieces: element by element the stores of 8 rows' dW (538 194 items of 337, f16) took
// 532 us, so 274.
// Measured: backward of 8 rows, 500 000 items of 384 (bf16, 384 MB read and written) 235 us = 3.3 TB/s, through G 389; of 9 rows, 496 726
// of 64 27 and 63; of 8 f32 rows, 300 000 of 384 351 and 1 167.  Forward (few_pays in table_loss.hip: where the table would need an image)
// of 2 rows, 688 025 of 678 at an odd stride 266, backward 641, through images and G 2 744 in all.
#pragma once

#include "table_loss_rows.h"

namespace asx {

typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
template <int FMT>
__device__ __forceinline__ f32x4 few_mfma16(u32x2 a, u32x2 b, f32x4 c) {  // 16 x 16 x 16
  if constexpr (FMT == AS_BF16) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v, a), __builtin_bit_cast(short4v, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4, a), __builtin_bit_cast(half4, b), c, 0, 0, 0);
}
struct LossFewArgs {
  const char *rows, *table;
  size_t rows_ld, table_ld;       // bytes
  uint32_t n, v, d;
  float scale;
  const float *bias;
  float2 *part;                   // forward: [walker][n]
  uint32_t slices, row_blocks;    // forward: workgroups a block of rows
  // backward
  const float *lse, *every, *entry, *rest;
  const int *target;
  const float *coef;
  float *sums;                    // [workgroup][n][sums_pitch]
  uint32_t sums_pitch;
  void *out;                      // dW
  size_t out_stride;
  float *grad_bias;
  int want_x;
};

// KC steps of 32 columns a wave (d <= 128 KC); RT tiles of 16 rows
template <int DT, int KC, bool BIAS>
struct FewSlice {
  static constexpr int FMT = format_of(DT), P = planes_of(DT);
  static constexpr uint32_t CW = 32 * KC, kRow = CW * 2 + 16, kPlane = 16 * kRow, kWave = P * kPlane;  // (16 bytes between rows: eight rows of a read in different banks)
  LrPiece<DT, true> piece[KC];
  f32x4 bias;  // of this lane's four items
  __device__ __forceinline__ void load(const LossFewArgs &a, uint32_t column0, uint32_t stage) {
    const uint32_t lane = threadIdx.x & 63;
    bias = f32x4{0.f, 0.f, 0.f, 0.f};
    if (BIAS && a.bias) {
      const uint32_t item = stage * 16 + (lane >> 4) * 4;
      if (stage * 16 + 16 <= a.v) {
        __builtin_memcpy(&bias, a.bias + item, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = a.bias[nt_min(item + e, a.v - 1)];
      }
    }
#pragma unroll
    for (int t = 0; t < KC; ++t) {
      const uint32_t idx = t * 64 + lane, row = idx / (4 * KC), slot = idx % (4 * KC);
      piece[t].load(a.table + (size_t)nt_min(stage * 16 + row, a.v - 1) * a.table_ld, column0 + slot * 8, a.d, 0);
    }
  }
  __device__ __forceinline__ void store(char *dst) const {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int t = 0; t < KC; ++t) {
      const uint32_t idx = t * 64 + lane, row = idx / (4 * KC), slot = idx % (4 * KC);
      u32x4 o[P];
      piece[t].template planes<FMT, P>(o);
#pragma unroll
      for (int p = 0; p < P; ++p) *(u32x4 *)(dst + p * kPlane + row * kRow + slot * 16) = o[p];
    }
  }
  // 16 items x 16 RT rows, this wave's columns
  template <int RT>
  __device__ __forceinline__ static void logits(const char *src, const u32x4 (&R)[P][RT][KC], f32x4 (&z)[RT]) {
    const uint32_t lane = threadIdx.x & 63, q = lane >> 4, at = (lane & 15) * kRow + q * 16;
#pragma unroll
    for (int j = 0; j < RT; ++j) z[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < KC; ++t)
#pragma unroll
      for (int p = P - 1; p >= 0; --p) {
        const u32x4 A = lr_row(src, p * kPlane + at + t * 64);
#pragma unroll
        for (int o = P - 1 - p; o >= 0; --o)
#pragma unroll
          for (int j = 0; j < RT; ++j) z[j] = nt_mfma<FMT>(A, R[o][j][t], z[j]);
      }
  }
};
template <int DT, int KC, int RT>
__device__ __forceinline__ void few_rows(const LossFewArgs &a, uint32_t n, uint32_t column0, u32x4 (&R)[FewSlice<DT, KC, false>::P][RT][KC]) {
  constexpr int P = FewSlice<DT, KC, false>::P, FMT = FewSlice<DT, KC, false>::FMT;
  const uint32_t lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
#pragma unroll
  for (int j = 0; j < RT; ++j)
#pragma unroll
    for (int t = 0; t < KC; ++t) {
      LrPiece<DT, true> piece;
      piece.load(a.rows + (size_t)nt_min(j * 16 + col, n - 1) * a.rows_ld, column0 + t * 32 + q * 8, a.d, 0);
      u32x4 o[P];
      piece.template planes<FMT, P>(o);
#pragma unroll
      for (int p = 0; p < P; ++p) R[p][j][t] = o[p];
    }
}

// WK waves share the columns: 4, or 1
template <int DT, int KC, int RT, bool GENERAL, int WK, int WAVES>
__global__ __launch_bounds__(256, WAVES) void loss_few_sums_kernel(LossFewArgs a) {
  typedef FewSlice<DT, KC, GENERAL> Slice;
  constexpr int P = Slice::P, TS = WK == 1 ? RT : 1;  // TS: row tiles whose statistics a wave keeps (WK 4: wave w those of tile w)
  __shared__ __attribute__((aligned(16))) char smem[4 * Slice::kWave];
  __shared__ f32x4 meet[WK == 4 ? 2 : 1][4][RT][64];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
  // a die (8 blocks apart) takes the blocks of rows of a stretch of the table one after another: its L2 has the items then
  const uint32_t turn = blockIdx.x >> 3, block = turn % a.row_blocks, slice_at = turn / a.row_blocks * 8 + (blockIdx.x & 7);
  if (slice_at >= a.slices) return;
  a.rows += (size_t)block * 16 * RT * a.rows_ld;
  const uint32_t row0 = block * 16 * RT, n = a.n - row0;
  const uint32_t column0 = (WK == 4 ? wave : 0) * Slice::CW, stages = (a.v + 15) / 16;
  const uint32_t walker = WK == 4 ? slice_at : slice_at * 4 + wave, walkers = a.slices * (4 / WK);
  const uint32_t s_lo = (uint32_t)((uint64_t)stages * walker / walkers), s_hi = (uint32_t)((uint64_t)stages * (walker + 1) / walkers);
  char *mine = smem + wave * Slice::kWave;
  Slice even, odd;  // two stages under way
  if (s_lo < s_hi) even.load(a, column0, s_lo);
  if (s_lo + 1 < s_hi) odd.load(a, column0, s_lo + 1);
  u32x4 R[P][RT][KC];
  few_rows<DT, KC, RT>(a, n, column0, R);
  const float unit = GENERAL ? kLog2e : a.scale * kLog2e, slack = fminf(20.f / unit, 1e30f);
  float ref[TS], base[TS], sum[TS];
#pragma unroll
  for (int t = 0; t < TS; ++t) ref[t] = -INFINITY, base[t] = 0.f, sum[t] = 0.f;
  auto step = [&](uint32_t s, Slice &slice) {
    slice.store(mine);
    const f32x4 bias = slice.bias;
    if (s + 2 < s_hi) slice.load(a, column0, s + 2);
    wave_lds_order();
    f32x4 z[RT];
    Slice::template logits<RT>(mine, R, z);
    if constexpr (WK == 4) {
#pragma unroll
      for (int j = 0; j < RT; ++j) meet[s & 1][wave][j][lane] = z[j];
      __syncthreads();
      if (wave >= RT) return;
    }
#pragma unroll
    for (int t = 0; t < TS; ++t) {
      f32x4 l = z[t];
      if constexpr (WK == 4) l = meet[s & 1][0][wave][lane] + meet[s & 1][1][wave][lane] + meet[s & 1][2][wave][lane] + meet[s & 1][3][wave][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t item = s * 16 + q * 4 + e;
        if (GENERAL) l[e] = fmaf(l[e], a.scale, bias[e]);
        if (item >= a.v) l[e] = -INFINITY;
      }
      const float top = fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3]));
      if (__any(top > ref[t] + slack)) {
        if (top > ref[t]) {
          const float to = GENERAL ? top : base_of(top, unit);
          sum[t] *= GENERAL ? __builtin_amdgcn_exp2f((ref[t] - top) * unit) : rebased(ref[t], base[t], to);
          ref[t] = top, base[t] = to;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[t] += __builtin_amdgcn_exp2f(GENERAL ? (l[e] - base[t]) * unit : fmaf(l[e], unit, base[t]));
    }
  };
  for (uint32_t s = s_lo; s < s_hi; s += 2) {
    step(s, even);
    if (s + 1 < s_hi) step(s + 1, odd);
  }
  if (WK == 4 && wave >= RT) return;
#pragma unroll
  for (int t = 0; t < TS; ++t) {
    float m = ref[t];
    if (!GENERAL && m != -INFINITY) {
      m *= a.scale;
      sum[t] = sum_against(ref[t], unit, base[t], a.scale, m, sum[t]);
    }
#pragma unroll
    for (int x = 16; x < 64; x <<= 1) {
      const float mo = __shfl_xor(m, x), so = __shfl_xor(sum[t], x);
      const float mm = fmaxf(m, mo), b = mm == -INFINITY ? 0.f : mm;
      sum[t] = sum[t] * __builtin_amdgcn_exp2f((m - b) * kLog2e) + so * __builtin_amdgcn_exp2f((mo - b) * kLog2e);
      m = mm;
    }
    const uint32_t row = (WK == 4 ? wave : t) * 16 + col;
    if (q == 0 && row < n) a.part[(size_t)walker * a.n + row0 + row] = float2{m, sum[t]};
  }
}

template <int DT, int KC, bool BIAS, int WK, int WAVES>
__global__ __launch_bounds__(256, WAVES) void loss_few_grad_kernel(LossFewArgs a) {
  typedef FewSlice<DT, KC, BIAS> Slice;
  constexpr int P = Slice::P, FMT = Slice::FMT;
  __shared__ __attribute__((aligned(16))) char smem[4 * Slice::kWave];
  __shared__ f32x4 meet[WK == 4 ? 2 : 1][4][64];
  __shared__ __attribute__((aligned(16))) char turn[4][P][512];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
  const uint32_t column0 = (WK == 4 ? wave : 0) * Slice::CW, stages = (a.v + 15) / 16;
  const uint32_t walker = WK == 4 ? blockIdx.x : blockIdx.x * 4 + wave, walkers = gridDim.x * (4 / WK);
  const uint32_t s_lo = (uint32_t)((uint64_t)stages * walker / walkers), s_hi = (uint32_t)((uint64_t)stages * (walker + 1) / walkers);
  char *mine = smem + wave * Slice::kWave;
  constexpr int AHEAD = KC * P <= 4 ? 2 : 1;  // stages under way
  Slice ring[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (s_lo + i < s_hi) ring[i].load(a, column0, s_lo + i);
  u32x4 R[P][1][KC];
  few_rows<DT, KC, 1>(a, a.n, column0, R);
  // the rows transposed: columns 32 j + 8 (col / 4) + 4 h + col % 4 of rows 4 q .. 4 q + 3 (rows that are not there: zeros)
  u32x2 XT[P][2 * KC];
#pragma unroll
  for (int t = 0; t < 2 * KC; ++t) {
    const uint32_t c = column0 + (t >> 1) * 32 + (col >> 2) * 8 + (t & 1) * 4 + (col & 3);
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = q * 4 + e < a.n && c < a.d ? load_as_f32<DT>(a.rows + (size_t)(q * 4 + e) * a.rows_ld, c) : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[P];
      pack_planes<FMT, P>(x[2 * h], x[2 * h + 1], w);
#pragma unroll
      for (int p = 0; p < P; ++p) XT[p][t][h] = w[p];
    }
  }
  // this lane's row (arrays are filled to 64)
  const float lse = a.lse[col], every = a.every[col], entry = a.entry[col], f = a.scale * a.coef[1];
  const uint32_t target = (uint32_t)a.target[col];
  f32x4 dx[2 * KC];
#pragma unroll
  for (int t = 0; t < 2 * KC; ++t) dx[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t trow = q * 4 + ((lane >> 2) & 3);
  auto step = [&](uint32_t s, Slice &slice) {
    slice.store(mine);
    const f32x4 bias = slice.bias;
    if (s + AHEAD < s_hi) slice.load(a, column0, s + AHEAD);
    wave_lds_order();
    f32x4 z[1];
    Slice::template logits<1>(mine, R, z);
    f32x4 g = z[0];
    if constexpr (WK == 4) {
      meet[s & 1][wave][lane] = g;
      __syncthreads();
      g = meet[s & 1][0][lane] + meet[s & 1][1][lane] + meet[s & 1][2][lane] + meet[s & 1][3][lane];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t item = s * 16 + q * 4 + e;
      const float l = BIAS ? fmaf(g[e], a.scale, bias[e]) - lse : fmaf(g[e], a.scale, -lse);
      g[e] = item < a.v ? every * probability(l * kLog2e) : 0.f;
      if (target == item) g[e] = entry;
    }
    if constexpr (BIAS) {
      if ((WK == 1 || wave == 0) && a.grad_bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float b = add16(g[e]);
          if (col == 0 && s * 16 + q * 4 + e < a.v) a.grad_bias[s * 16 + q * 4 + e] = b * a.coef[1];
        }
      }
    }
    u32x2 G[P];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[P];
      pack_planes<FMT, P>(g[2 * h], g[2 * h + 1], w);
#pragma unroll
      for (int p = 0; p < P; ++p) G[p][h] = w[p];
    }
    if (a.want_x) {
#pragma unroll
      for (int t = 0; t < 2 * KC; ++t)
#pragma unroll
        for (int p = P - 1; p >= 0; --p) {
          const u32x2 Y = lr_column4(mine, p * Slice::kPlane + trow * Slice::kRow + (t >> 1) * 64 + (lane & 3) * 16 + (t & 1) * 8);
#pragma unroll
          for (int o = P - 1 - p; o >= 0; --o) dx[t] = few_mfma16<FMT>(Y, G[o], dx[t]);
        }
    }
    if (a.out) {
      u32x2 T[P];
#pragma unroll
      for (int p = 0; p < P; ++p) *(u32x2 *)(turn[wave][p] + col * 32 + q * 8) = G[p];
      wave_lds_order();
#pragma unroll
      for (int p = 0; p < P; ++p) T[p] = lr_column4(turn[wave][p], trow * 32 + (lane & 3) * 8);
      const uint32_t item = s * 16 + col;
      const uint32_t met = P == 1 ? (uint32_t)__ballot(lane < 16 && target - s * 16 < 16u) : 0u;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        f32x4 w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = P - 1; p >= 0; --p)
#pragma unroll
            for (int o = P - 1 - p; o >= 0; --o) w[h] = few_mfma16<FMT>(XT[p][2 * j + h], T[o], w[h]);
        }
        const uint32_t c = column0 + j * 32 + q * 8;
        if (met) {  // what 16 bits left of the entries at the targets
          for (uint32_t m = met; m; m &= m - 1) {
            const uint32_t t = __builtin_ctz(m);
            if ((uint32_t)a.target[t] != item) continue;
            const float rest = a.rest[t];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < a.d) w[e >> 2][e & 3] += rest * load_as_f32<DT>(a.rows + (size_t)t * a.rows_ld, c + e);
          }
        }
        w[0] *= f, w[1] *= f;
        if (item >= a.v || c >= a.d) continue;
        if (c + 8 <= a.d) {
          store8<DT>(a.out, (size_t)item * a.out_stride + c, w[0], w[1]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < a.d) store_from_f32<DT>(a.out, (size_t)item * a.out_stride + c + e, w[e >> 2][e & 3]);
        }
      }
    }
  };
  for (uint32_t s = s_lo; s < s_hi; s += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s + i < s_hi) step(s + i, ring[i]);
  }
  if (!a.want_x) return;
  if constexpr (WK == 1) {  // the four waves' dX, in their order
    __syncthreads();
    f32x4 *other = (f32x4 *)smem;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      if (wave == w) {
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t) other[t * 64 + lane] = dx[t];
      }
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int t = 0; t < 2 * KC; ++t) dx[t] += other[t * 64 + lane];
      }
      __syncthreads();
    }
    if (wave) return;
  }
  if (col < a.n) {
#pragma unroll
    for (int j = 0; j < KC; ++j) {
      const uint32_t c = column0 + j * 32 + q * 8;
      if (c >= a.d) continue;
      f32x4 *o = (f32x4 *)(a.sums + ((size_t)blockIdx.x * a.n + col) * a.sums_pitch + c);
      o[0] = dx[2 * j], o[1] = dx[2 * j + 1];
    }
  }
}

}  // namespace asx
