// table_loss.hip -- softmax cross entropy of rows against a table of items, without keeping the logits, and its gradient.
//
//   l_tv = scale <x_t, w_v> + bias_v      lse_t = log sum_v exp(l_tv)      loss_t = lse_t - l_{t, y_t}
//   with gl = dL/dloss (0 where the row is ignored), ge = dL/dlse:   g_tv = (gl_t + ge_t) exp(l_tv - lse_t) - gl_t [v = y_t]
//   dX = scale G W      dW = scale G^T X      dbias_v = sum_t g_tv
//
// Forward: one product (nt_product.h, the table on the m side, so that a lane holds many items of ONE row) whose ending keeps a
// running maximum and sum of exponentials per lane and row; what leaves the chip is one (maximum, sum) per row and stretch of the
// table.  A second kernel joins them and takes the target's logit from a product of its own in f64.
// Backward, three forms.  Rows of up to 256 values (f32: 128): the gradient G of the logits stays in registers (table_loss_rows.h).  Up
// to 16 rows: one pass over the table that writes dW as it goes (table_loss_few.h).  Else in pieces of the table: per piece the logits
// are made again, G leaves in 16 bits, once, and two more products, which read their operands transposed, give the piece's rows of dW
// and its part of dX (f32, added up over the pieces in a buffer, rounded once at the end).
// Nothing is added with atomics: results do not change from run to run.
// What bounds it: 2 n v d flops forward, 8 more backward, of which 2 are the logits again (through G: 6, written and read once: 2 bytes a
// logit each).  8 192 rows x 131 072 items of 1 024 (bf16), forward and backward: 8.04 ms = 1 094 TFLOP/s, one library product of this
// size runs at 1 076; 4 096 x 100 000 of 768 with a bias: 2.67 ms; 1 024 x 1 000 000 of 128: 1.27 ms, 2.01 through G; 777 x 31 013 of 200
// (f16): 0.14, 0.18 through G; f32, 512 x 100 000 of 128: 0.47, 0.55 through G.
// Types.  bf16 and f16 go to the matrix pipe as they are.  f32 values go as a sum of three bf16 (table_loss_rows.h): 24 bits, of values
// below 2^-108 what a step of 2^-133 leaves, and no scale that one large value would set for everyone.  Six products a pair of values: 2.5
// PFLOP/s / 6 against the 0.157 of the f32 instruction.  (Two f16 under a power of two a matrix need three: the same step 0.31.  But a value
// keeps 22 bits only down to 2^-17 of the matrix' largest, 14 at 2^-24: a row of garbage in the padding left the others none.)
// Rounding.  16-bit matrices: G is rounded to their type, in units of the largest coefficient (coef_scale_kernel): half a step per entry, as
// the gradients that leave are rounded themselves (f32: three planes, as the values).  The entries at the targets, nearly the coefficient itself and
// the same in all rows of an item, come from a product of their own in f64, and what 16 bits leave of them is added in f32: with half a
// step there, dX of well-trained rows was off by twice the rounding of the result.  Everything else -- logits, maxima, sums, dX over pieces,
// dbias -- is f32 or wider.
#include "table_loss_few.h"

using namespace asx;

namespace {

constexpr int kChips = 256;  // compute units: how many workgroups of the large tile run at once

struct LossArgs {
  // operands of the product: A the table side (m), B the rows (n)
  const char *table, *rows;
  size_t table_ld, rows_ld;       // bytes
  size_t table_plane, rows_plane; // bytes from plane to plane
  uint32_t n, v;                  // rows of B and of A
  uint32_t steps, all;            // steps of 64 along k, and with every pair of planes
  uint32_t per;                   // tiles of A a workgroup walks
  uint32_t v_tiles, n_tiles, chunks;
  float scale;
  const float *bias;
};

// ---- forward --------------------------------------------------------------------------------------------------------------------------
// GENERAL: with a bias, or a scale that is not positive (the maximum is then taken of the scaled logits); else of the raw products.
template <int FMT, class TILE_, bool GENERAL>
__global__ __launch_bounds__(TILE_::NT) void loss_sums_kernel(LossArgs a, float2 *part) {
  using TILE = TILE_;
  __shared__ __attribute__((aligned(1024))) char smem[2 * TILE::kStage];
  TILE T;
  T.init(smem);
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  uint32_t nt, chunk;
  grid_order(work, a.n_tiles, a.chunks, &nt, &chunk);
  const uint32_t n0 = nt * TILE::BN, vt_end = nt_min((chunk + 1) * a.per, a.v_tiles);
  uint32_t vt = chunk * a.per;
  const float unit = GENERAL ? kLog2e : a.scale * kLog2e;  // exponentials of (x - maximum) * unit to the base 2
  const uint32_t wm = T.wave / TILE::WN, wn = T.wave % TILE::WN, q = T.lane >> 4, col = T.lane & 15;
  NtOperand B{a.rows + (size_t)n0 * a.rows_ld, a.rows_ld, nt_min(TILE::BN, a.n - n0) - 1, 0, a.rows_plane};
  auto side = [&](uint32_t tile) {
    const uint32_t r0 = tile * TILE::BM;
    return NtOperand{a.table + (size_t)r0 * a.table_ld, a.table_ld, nt_min(TILE::BM, a.v - r0) - 1, 0, a.table_plane};
  };
  const uint32_t all = a.all;
  float top[TILE::TN], sum[TILE::TN], shift[TILE::TN];
#pragma unroll
  for (int j = 0; j < TILE::TN; ++j) top[j] = -INFINITY, sum[j] = shift[j] = 0.f;
  f32x4 acc[TILE::TM][TILE::TN];
  NtOperand A = side(vt);
  T.fetch(0, A, B, 0, a.steps);
  int buf = 0;
  for (; vt < vt_end; ++vt) {
    T.zero(acc);
    const uint32_t last = A.last;
    for (uint32_t s = 0; s < all; ++s) {
      TILE::turn();
      if (s + 1 < all) {
        T.fetch(buf ^ 1, A, B, s + 1, a.steps);
      } else if (vt + 1 < vt_end) {
        A = side(vt + 1);
        T.fetch(buf ^ 1, A, B, 0, a.steps);
      }
      T.contract(buf, acc);
      buf ^= 1;
    }
    // this tile's logits: a lane holds 4 TM items of each of its TN rows
    const uint32_t row0 = wm * (TILE::TM * 16) + q * 8;
    if constexpr (GENERAL) {
#pragma unroll
      for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t r = row0 + (i >> 1) * 32 + (i & 1) * 4 + e;
          const float b = a.bias && r <= last ? a.bias[(size_t)vt * TILE::BM + r] : 0.f;
#pragma unroll
          for (int j = 0; j < TILE::TN; ++j) acc[i][j][e] = r > last ? -INFINITY : fmaf(acc[i][j][e], a.scale, b);
        }
    } else if (last + 1 < TILE::BM) {
#pragma unroll
      for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t r = row0 + (i >> 1) * 32 + (i & 1) * 4 + e;
          if (r > last)
#pragma unroll
            for (int j = 0; j < TILE::TN; ++j) acc[i][j][e] = -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < TILE::TN; ++j) {
      float m = top[j];
#pragma unroll
      for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) m = fmaxf(m, acc[i][j][e]);
      // (with a bias the difference first: a bias of the type's lowest value times log2 e would be infinite)
      const float base = m == -INFINITY ? 0.f : m, to = GENERAL ? 0.f : base_of(base, unit);
      auto power = [&](float x) { return __builtin_amdgcn_exp2f(GENERAL ? (x - base) * unit : fmaf(x, unit, to)); };
      float s0 = sum[j] * (GENERAL ? power(top[j]) : rebased(top[j], shift[j], to)), s1 = 0.f;
      shift[j] = to;
#pragma unroll
      for (int i = 0; i < TILE::TM; ++i) {
        s0 += power(acc[i][j][0]);
        s1 += power(acc[i][j][1]);
        s0 += power(acc[i][j][2]);
        s1 += power(acc[i][j][3]);
      }
      top[j] = m;
      sum[j] = s0 + s1;
    }
  }
  // the four lane groups of a row
#pragma unroll
  for (int j = 0; j < TILE::TN; ++j) {
    float m = top[j], s = sum[j];
    if (!GENERAL && m != -INFINITY) {
      m *= a.scale;
      s = sum_against(top[j], unit, shift[j], a.scale, m, s);
    }
#pragma unroll
    for (int x = 16; x < 64; x <<= 1) {
      const float mo = __shfl_xor(m, x), so = __shfl_xor(s, x);
      const float mm = fmaxf(m, mo), base = mm == -INFINITY ? 0.f : mm;
      s = s * __builtin_amdgcn_exp2f((m - base) * kLog2e) + so * __builtin_amdgcn_exp2f((mo - base) * kLog2e);
      m = mm;
    }
    const uint32_t t = n0 + wn * (TILE::TN * 16) + (j >> 1) * 32 + (col >> 2) * 8 + (j & 1) * 4 + (col & 3);
    if (q == 0 && t < a.n) part[(size_t)(chunk * TILE::WM + wm) * a.n + t] = float2{m, s};
  }
}

// Workgroups of the kernels that take four rows of the batch each: a launch holds less than 2^32 threads, 2^26 rows of a wave.
unsigned row_groups(uint64_t rows) { return (unsigned)std::min<uint64_t>((rows + 3) / 4, 1u << 20); }

// A wave a row: the stretches' (maximum, sum) joined, the target's logit from the inputs themselves.  f64 behind the sums: the loss is a
// difference of two near numbers where the model is right.
template <int DT>
__global__ __launch_bounds__(256) void loss_join_kernel(const float2 *part, uint32_t parts, const void *x, size_t x_stride, const void *table,
                                                        size_t table_stride, const float *bias, const int64_t *targets, uint32_t n, uint32_t v,
                                                        uint32_t d, float scale, int64_t ignore, float *losses, float *lse_out) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t t = blockIdx.x * 4 + (threadIdx.x >> 6); t < n; t += gridDim.x * 4) {
    float top = -INFINITY;
    double s = 0.0;
    for (uint32_t p0 = 0; p0 < parts; p0 += 1024) {
      float2 o[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint32_t p = p0 + k * 64 + lane;
        o[k] = p < parts ? part[(size_t)p * n + t] : float2{-INFINITY, 0.f};
      }
      float m = top;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = fmaxf(m, o[k].x);
      const float base = m == -INFINITY ? 0.f : m;
      float here = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) here += o[k].y * __builtin_amdgcn_exp2f((o[k].x - base) * kLog2e);
      s = s * (double)__builtin_amdgcn_exp2f((top - base) * kLog2e) + (double)here;
      top = m;
    }
    const float m = top;
    for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
    const float base = top == -INFINITY ? 0.f : top;
    s *= (double)__builtin_amdgcn_exp2f((m - base) * kLog2e);
    for (int k = 1; k < 64; k <<= 1) s += __shfl_xor(s, k);
    const int64_t y = targets[t];
    const bool ignored = y == ignore, inside = y >= 0 && y < (int64_t)v;
    double dot = 0.0;
    if (!ignored && inside) {
      const size_t xr = (size_t)t * x_stride, wr = (size_t)y * table_stride;
      for (uint32_t k = lane; k < d; k += 64) dot += (double)load_as_f32<DT>(x, xr + k) * (double)load_as_f32<DT>(table, wr + k);
      for (int k = 1; k < 64; k <<= 1) dot += __shfl_xor(dot, k);
    }
    if (lane == 0) {
      // (no item left by the bias: the maximum and every term are -inf, s = 0; without a bias these are products that overflowed)
      const double lse = s == 0.0 ? (bias ? -INFINITY : NAN) : (double)base + log(s);
      const double logit = (double)scale * dot + (inside && bias ? (double)bias[y] : 0.0);
      lse_out[t] = (float)lse;
      losses[t] = ignored || (s == 0.0 && bias) ? 0.f : !inside ? NAN : (float)(lse - logit);
    }
  }
}

// ---- what the products are made of ----------------------------------------------------------------------------------------------------
// A matrix and its image: rows with their length filled to whole steps by zeros, f32 as three planes.
struct ImageJob {
  const char *src;
  size_t stride;           // bytes
  uint32_t n, d, pitch;
  unsigned short *out;
};
struct ImageJobs {
  ImageJob job[2];
};
// A matrix in pieces of eight columns, `across` a row, dealt to all threads of the grid, four at a time under way.  f(piece, row, column)
template <int DT, int THREADS, class F>
__device__ __forceinline__ void each_piece(const ImageJob &j, uint32_t across, F &&f) {
  const uint32_t threads = gridDim.x * THREADS, first = blockIdx.x * THREADS + threadIdx.x;
  const uint32_t row_step = threads / across, column_step = threads % across;
  uint32_t row = first / across, column = first % across;
  while (row < j.n) {
    LrPiece<DT, true> piece[4];
    uint32_t r[4], c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = row, c[i] = column * 8;
      if (row < j.n) piece[i].load(j.src + (size_t)row * j.stride, c[i], j.d, 0);
      row += row_step, column += column_step;
      if (column >= across) column -= across, ++row;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] < j.n) f(piece[i], r[i], c[i]);
  }
}
template <int DT>
__global__ __launch_bounds__(256) void image_kernel(ImageJobs jobs) {
  constexpr int P = planes_of(DT);
  const ImageJob &j = jobs.job[blockIdx.y];
  each_piece<DT, 256>(j, j.pitch / 8, [&](const LrPiece<DT, true> &piece, uint32_t row, uint32_t column) {
    unsigned short *o = j.out + (size_t)row * j.pitch * P + column;
    u32x4 w[P];
    piece.template planes<format_of(DT), P>(w);
#pragma unroll
    for (int p = 0; p < P; ++p) *(u32x4 *)(o + p * j.pitch) = w[p];
  });
}
// ---- gradient of the logits ---------------------------------------------------------------------------------------------------------------
struct GradArgs {
  LossArgs l;
  uint32_t v_begin;                // first item of the piece (the operand A starts there)
  const float *lse, *every, *entry;  // by row, filled to whole tiles (loss_rows_kernel)
  const int *target;
  const float *coef;               // {factor, 1 / factor} of G
  unsigned short *G;               // (rows filled to whole tiles) x (planes * g_pitch)
  uint32_t g_pitch;
  float *bias_part;                // (n_tiles WN) x g_pitch sums over the tile's rows, or null
};

template <int FMT, class TILE_, int P, bool BIAS>
__global__ __launch_bounds__(TILE_::NT) void loss_grad_kernel(GradArgs g) {
  using TILE = TILE_;
  __shared__ __attribute__((aligned(1024))) char smem[2 * TILE::kStage];
  const LossArgs &a = g.l;
  TILE T;
  T.init(smem);
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  uint32_t nt, chunk;
  grid_order(work, a.n_tiles, a.chunks, &nt, &chunk);
  const uint32_t n0 = nt * TILE::BN, vt_end = nt_min((chunk + 1) * a.per, a.v_tiles);
  uint32_t vt = chunk * a.per;
  const uint32_t wm = T.wave / TILE::WN, wn = T.wave % TILE::WN, q = T.lane >> 4, col = T.lane & 15;
  NtOperand B{a.rows + (size_t)n0 * a.rows_ld, a.rows_ld, nt_min(TILE::BN, a.n - n0) - 1, 0, a.rows_plane};
  auto side = [&](uint32_t tile) {
    const uint32_t r0 = tile * TILE::BM;
    return NtOperand{a.table + (size_t)r0 * a.table_ld, a.table_ld, nt_min(TILE::BM, a.v - r0) - 1, 0, a.table_plane};
  };
  // this lane's rows
  uint32_t row[TILE::TN];
  float lse[TILE::TN], every[TILE::TN], entry[TILE::TN];
  int32_t hit[TILE::TN];  // the target within the piece, or far off
#pragma unroll
  for (int j = 0; j < TILE::TN; ++j) {
    const uint32_t t = n0 + wn * (TILE::TN * 16) + (j >> 1) * 32 + (col >> 2) * 8 + (j & 1) * 4 + (col & 3);
    row[j] = t;
    lse[j] = g.lse[t];
    every[j] = g.every[t];
    entry[j] = g.entry[t];
    const uint32_t at = (uint32_t)g.target[t] - g.v_begin;
    hit[j] = at < a.v ? (int32_t)at : -1;
  }
  const uint32_t all = a.all;
  f32x4 acc[TILE::TM][TILE::TN];
  NtOperand A = side(vt);
  T.fetch(0, A, B, 0, a.steps);
  int buf = 0;
  for (; vt < vt_end; ++vt) {
    T.zero(acc);
    const uint32_t last = A.last;
    for (uint32_t s = 0; s < all; ++s) {
      TILE::turn();
      if (s + 1 < all) {
        T.fetch(buf ^ 1, A, B, s + 1, a.steps);
      } else if (vt + 1 < vt_end) {
        A = side(vt + 1);
        T.fetch(buf ^ 1, A, B, 0, a.steps);
      }
      T.contract(buf, acc);
      buf ^= 1;
    }
    const uint32_t row0 = wm * (TILE::TM * 16) + q * 8;   // within the tile
    const uint32_t at0 = vt * TILE::BM;                   // of the tile within the piece
#pragma unroll
    for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t r = row0 + (i >> 1) * 32 + (i & 1) * 4 + e;
        float b = 0.f;
        if constexpr (BIAS) b = r > last ? -INFINITY : a.bias[at0 + r];
#pragma unroll
        for (int j = 0; j < TILE::TN; ++j) {
          const float z = BIAS ? fmaf(acc[i][j][e], a.scale, b) - lse[j] : fmaf(acc[i][j][e], a.scale, -lse[j]);
          acc[i][j][e] = every[j] * probability(z * kLog2e);
        }
      }
    if (last + 1 < TILE::BM) {
#pragma unroll
      for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row0 + (i >> 1) * 32 + (i & 1) * 4 + e > last)
#pragma unroll
            for (int j = 0; j < TILE::TN; ++j) acc[i][j][e] = 0.f;
    }
    // the targets: few of the tiles hold one of the wave's rows' (hit < 0 is far above any place of the tile)
    const uint32_t wave0 = at0 + wm * (TILE::TM * 16);
    bool any = false;
#pragma unroll
    for (int j = 0; j < TILE::TN; ++j) any |= (uint32_t)hit[j] - wave0 < (uint32_t)(TILE::TM * 16) && hit[j] >= 0;
    if (__any(any)) {
#pragma unroll
      for (int j = 0; j < TILE::TN; ++j)
#pragma unroll
        for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (hit[j] == (int32_t)(at0 + row0 + (i >> 1) * 32 + (i & 1) * 4 + e)) acc[i][j][e] = entry[j];
    }
    if constexpr (BIAS) {
      if (g.bias_part) {
        float *bp = g.bias_part + (size_t)(nt * TILE::WN + wn) * g.g_pitch + at0;
#pragma unroll
        for (int i = 0; i < TILE::TM; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < TILE::TN; ++j) s += row[j] < a.n ? acc[i][j][e] : 0.f;
            s = add16(s);
            if (col == 0) bp[row0 + (i >> 1) * 32 + (i & 1) * 4 + e] = s;
          }
      }
    }
    // eight consecutive items a lane (rows behind the last: zeros, the product over the batch reads them)
    const size_t gp = (size_t)g.g_pitch * P;
#pragma unroll
    for (int j = 0; j < TILE::TN; ++j) {
      unsigned short *o = g.G + (size_t)row[j] * gp + at0 + row0;
#pragma unroll
      for (int i = 0; i < TILE::TM; i += 2) {
        u32x4 w[P];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t pair[P];
          pack_planes<FMT, P>(acc[i + (h >> 1)][j][2 * (h & 1)], acc[i + (h >> 1)][j][2 * (h & 1) + 1], pair);
#pragma unroll
          for (int p = 0; p < P; ++p) w[p][h] = pair[p];
        }
#pragma unroll
        for (int p = 0; p < P; ++p) *(u32x4 *)(o + (size_t)p * g.g_pitch + i * 16) = w[p];
      }
    }
  }
}

// The rows of the batch that meet each 64 items of the table, in order, a workgroup each, its waves an eighth of the batch each (64 kept:
// the entries of further rows stay rounded, as all other entries of G are).
constexpr uint32_t kMet = 64;
__global__ __launch_bounds__(512) void met_kernel(const int *target, uint32_t n, u32x2 *list, uint32_t *count) {
  __shared__ u32x2 part[8][kMet];
  __shared__ uint32_t part_len[8];
  const uint32_t group = blockIdx.x, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t each = (n + 511) / 512 * 64, lo = w * each, hi = nt_min(lo + each, n);
  uint32_t len = 0;
  for (uint32_t t0 = lo; t0 < hi && len < kMet; t0 += 512) {
    uint32_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = t0 + k * 64 + lane < hi ? (uint32_t)target[t0 + k * 64 + lane] - group * 64 : ~0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint64_t met = __ballot(v[k] < 64);
      const uint32_t place = len + (uint32_t)__popcll(met & ((1ull << lane) - 1));
      if (v[k] < 64 && place < kMet) part[w][place] = u32x2{t0 + k * 64 + lane, v[k]};
      len += (uint32_t)__popcll(met);
    }
  }
  if (lane == 0) part_len[w] = nt_min(len, kMet);
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t o = 0; o < 8; ++o) {
    if (o < w) before += part_len[o];
    all += part_len[o];
  }
  if (lane < part_len[w] && before + lane < kMet) list[(size_t)group * kMet + before + lane] = part[w][lane];
  if (threadIdx.x == 0) count[group] = nt_min(all, kMet);
}

// ---- the two gradients: plain products ------------------------------------------------------------------------------------------------------
// A (m: columns of x or of the table) is read transposed, a row per k; B (n: g) transposed for dW, along k for dX.
struct ProductArgs {
  const char *A, *B;
  size_t a_ld, b_ld;
  size_t a_plane, b_plane;          // bytes
  uint32_t a_cols, b_cols;          // 16-byte pieces of a row that may be read (transposed)
  uint32_t k_a, k_b;                // rows that may be read (transposed)
  uint32_t m, n, m_tiles, n_tiles;
  uint32_t steps, pairs, splits;    // steps of 64 of the whole contraction, a split takes an even share of them; pairs of planes
  float scale;
  const float *coef;                // 1 / factor of G at [1]
  void *out;                        // n x m rows of `out_stride` elements
  size_t out_stride;
  float *sums;                      // instead: f32 [split][n][sums_pitch], added to unless `first`
  uint32_t sums_pitch;
  int first;
  // dW of one plane: by 64 items the rows of the batch that meet them, what 16 bits left of those rows' entries (null: none)
  const u32x2 *met;
  const uint32_t *met_count;
  const float *rest;
};
template <int FMT, class TILE>
__device__ __forceinline__ void add_rest(const ProductArgs &p, const TILE &T, uint32_t m0, uint32_t n0, f32x4 (&acc)[TILE::TM][TILE::TN]) {
  static_assert(TILE::TN == 4, "a wave's columns are one list's items");
  const uint32_t wm = T.wave / TILE::WN, wn = T.wave % TILE::WN, q = T.lane >> 4, col = T.lane & 15;
  if (n0 + wn * 64 >= p.n) return;
  const uint32_t group = (n0 >> 6) + wn, len = p.met_count[group];
  if (!len) return;
  const u32x2 mine = p.met[(size_t)group * kMet + (T.lane < len ? T.lane : 0)];
  const float mine_rest = p.rest[mine[0]];
  // Each column of lanes takes the rows that meet its own four items, all columns at once (one row after the other, 300 rows at 300 items
  // took eight times the product).
  uint64_t met = 0;
  for (uint32_t k = 0; k < len; ++k) {
    const uint32_t in = __builtin_amdgcn_readlane(mine[1], k);
    if (((((in >> 3) & 3) << 2) | (in & 3)) == col) met |= 1ull << k;
  }
  while (__any(met != 0)) {
    const int k = met ? __builtin_ctzll(met) : 0;
    const uint32_t row = __shfl(mine[0], k), in = __shfl(mine[1], k), jj = ((in >> 5) << 1) | ((in >> 2) & 1);
    const float r = __shfl(mine_rest, k);
    if (met) {
#pragma unroll
      for (int i = 0; i < TILE::TM; i += 2) {
        const uint32_t m = m0 + wm * (TILE::TM * 16) + i * 16 + q * 8;
        if (m >= p.m) continue;
        const u32x4 w = *(const u32x4 *)(p.A + (size_t)row * p.a_ld + m * 2);  // (zeros behind the row's values)
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned short u = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
          y[e] = FMT == AS_BF16 ? bf16_to_f32(u) : (float)__builtin_bit_cast(_Float16, u);
        }
#pragma unroll
        for (uint32_t j = 0; j < TILE::TN; ++j)
          if (j == jj) {
            acc[i][j] += f32x4{y[0], y[1], y[2], y[3]} * r;
            acc[i + 1][j] += f32x4{y[4], y[5], y[6], y[7]} * r;
          }
        if (i & 2) __builtin_amdgcn_sched_barrier(0);  // (two pieces at a time: more would spill)
      }
    }
    met &= met - 1;
  }
}
template <int FMT, class TILE_, int OUT, bool BT>  // OUT: element type of `out`, or 0 (AS_F64) = into `sums`; BT: dW, else dX
__global__ __launch_bounds__(TILE_::NT) void product_kernel(ProductArgs p) {
  using TILE = TILE_;
  __shared__ __attribute__((aligned(1024))) char smem[2 * TILE::kStage];
  TILE T;
  T.init(smem);
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  const uint32_t split = work / (p.m_tiles * p.n_tiles);
  uint32_t mt, nt;
  grid_order(work - split * p.m_tiles * p.n_tiles, p.n_tiles, p.m_tiles, &nt, &mt);
  const uint32_t m0 = mt * TILE::BM, n0 = nt * TILE::BN;
  const uint32_t k0 = (uint32_t)((uint64_t)p.steps * split / p.splits), k1 = (uint32_t)((uint64_t)p.steps * (split + 1) / p.splits);
  const uint32_t steps = k1 - k0, all = p.pairs * steps;
  const NtOperand A{p.A + (size_t)k0 * 64 * p.a_ld + m0 * 2, p.a_ld, p.a_cols - 1 - m0 / 8, p.k_a - 1 - k0 * 64, p.a_plane};
  const NtOperand B = BT ? NtOperand{p.B + (size_t)k0 * 64 * p.b_ld + n0 * 2, p.b_ld, p.b_cols - 1 - n0 / 8, p.k_b - 1 - k0 * 64, p.b_plane}
                         : NtOperand{p.B + (size_t)n0 * p.b_ld + (size_t)k0 * 128, p.b_ld, nt_min(TILE::BN, p.n - n0) - 1, 0, p.b_plane};
  f32x4 acc[TILE::TM][TILE::TN];
  T.zero(acc);
  if (all) T.fetch(0, A, B, 0, steps);
  int buf = 0;
  for (uint32_t s = 0; s < all; ++s) {
    TILE::turn();
    if (s + 1 < all) T.fetch(buf ^ 1, A, B, s + 1, steps);
    T.contract(buf, acc);
    buf ^= 1;
  }
  if constexpr (BT && OUT != AS_F32)
    if (p.met && split == 0) add_rest<FMT>(p, T, m0, n0, acc);
  const uint32_t wm = T.wave / TILE::WN, wn = T.wave % TILE::WN, q = T.lane >> 4, col = T.lane & 15;
  const float f = OUT == 0 ? 1.f : p.scale * p.coef[1];
#pragma unroll
  for (int j = 0; j < TILE::TN; ++j) {
    const uint32_t n = n0 + wn * (TILE::TN * 16) + (j >> 1) * 32 + (col >> 2) * 8 + (j & 1) * 4 + (col & 3);
    if (n >= p.n) continue;
#pragma unroll
    for (int i = 0; i < TILE::TM; i += 2) {
      const uint32_t m = m0 + wm * (TILE::TM * 16) + i * 16 + q * 8;
      if (m >= p.m) continue;
      const f32x4 u = acc[i][j] * f, v = acc[i + 1][j] * f;
      if constexpr (OUT == 0) {
        float *o = p.sums + ((size_t)split * p.n + n) * p.sums_pitch + m;
        f32x4 *o4 = (f32x4 *)o;  // (the pitch is a multiple of 8)
        if (p.first) o4[0] = u, o4[1] = v;
        else o4[0] += u, o4[1] += v;
      } else if (m + 8 <= p.m) {
        store8<OUT>(p.out, (size_t)n * p.out_stride + m, u, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (m + e < p.m) store_from_f32<OUT>(p.out, (size_t)n * p.out_stride + m + e, e < 4 ? u[e & 3] : v[e & 3]);
      }
    }
  }
}

// dX (or dW) from its parts, in a fixed order.  A lane four columns; WAYS lanes a share of the parts each (64: quarters of 16 waves, 4:
// waves): a few rows have a thousand parts, one thread's chain of them would be the whole time; many rows have lanes enough.
template <int DT, int WAYS>
__global__ __launch_bounds__(WAYS == 64 ? 1024 : 256) void grad_rows_join_kernel(const float *sums, uint32_t splits, uint32_t pitch, uint32_t n, uint32_t d, float scale,
                                                                                 const float *coef, const int *target, const float *rest,
                                                                                 const void *table, size_t table_stride, void *out, size_t out_stride) {
  constexpr uint32_t WAVES = WAYS == 64 ? 16 : 4, LANES = WAYS == 64 ? 16 : 64, EACH = WAYS == 1 ? 1024 : LANES * 4;  // EACH: columns a workgroup
  __shared__ f32x4 s[WAVES][LANES];
  const uint32_t lane = threadIdx.x & (LANES - 1), w = threadIdx.x >> 6, sub = WAYS == 1 ? 0 : threadIdx.x / LANES;
  const uint32_t lo = splits * sub / WAYS, hi = splits * (sub + 1) / WAYS;
  const float f = scale * coef[1];
  const uint64_t total = (uint64_t)n * pitch;
  for (uint64_t i0 = (uint64_t)blockIdx.x * EACH; i0 < total; i0 += (uint64_t)gridDim.x * EACH) {
    const uint64_t i = i0 + (WAYS == 1 ? w * 256 : 0) + lane * 4, t = i / pitch, k = i - t * pitch;
    const bool mine = sub == 0 && i < total;
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, more = {0.f, 0.f, 0.f, 0.f};
    if (mine && rest) {  // of the entry at the row's target, times that item
      const int y = target[t];
      const float z = rest[t];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (y >= 0 && k + e < d) more[e] = z * load_as_f32<DT>(table, (size_t)y * table_stride + k + e);
    }
    if (i < total) {
      uint32_t p = lo;
      for (; p + 8 <= hi; p += 8) {
        f32x4 part[8];
#pragma unroll
        for (int o = 0; o < 8; ++o) part[o] = *(const f32x4 *)(sums + (p + o) * total + i);
#pragma unroll
        for (int o = 0; o < 8; ++o) x += part[o];
      }
      for (; p < hi; ++p) x += *(const f32x4 *)(sums + p * total + i);
    }
    if constexpr (WAYS == 64) {
#pragma unroll
      for (int o = 16; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], o);
    }
    if constexpr (WAYS > 1) {
      if ((threadIdx.x & 63) < LANES) s[w][lane] = x;
      __syncthreads();
      if (sub == 0)
        for (uint32_t o = 1; o < WAVES; ++o) x += s[o][lane];
      __syncthreads();
    }
    if (mine) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < d) store_from_f32<DT>(out, t * out_stride + k + e, (x[e] + more[e]) * f);
    }
  }
}
__global__ __launch_bounds__(256) void bias_join_kernel(const float *part, uint32_t parts, uint32_t pitch, uint32_t v, const float *coef, float *out) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= v) return;
  float s = 0.f;
#pragma unroll 16
  for (uint32_t p = 0; p < parts; ++p) s += part[(size_t)p * pitch + i];
  out[i] = s * coef[1];
}
template <int DT>
__global__ __launch_bounds__(256) void zero_rows_kernel(void *out, size_t stride, uint64_t n, uint32_t d) {
  const uint64_t total = n * d;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256)
    store_from_f32<DT>(out, (i / d) * stride + i % d, 0.f);
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------------
template <int FMT, bool AT = false, bool BT = false>
using Slim = NtTile<FMT, 4, 4, 4, 1, AT, BT>;   // 256 x 64
template <int FMT, bool AT = false, bool BT = false>
using Square = NtTile<FMT, 4, 4, 2, 2, AT, BT>; // 128 x 128
template <int FMT, bool AT = false, bool BT = false>
using Large = NtTile<FMT, 8, 4, 2, 4, AT, BT>;  // 256 x 256
enum { kSlim = 0, kSquare = 1, kLarge = 2 };
struct TileShape {
  uint32_t bm, bn, wm, wn;
};
constexpr TileShape kShape[3] = {{256, 64, 4, 1}, {128, 128, 2, 2}, {256, 256, 2, 4}};

uint32_t up(uint64_t a, uint32_t b) { return (uint32_t)((a + b - 1) / b * b); }

// How a matrix reaches the products: as it is, or as an image (whole steps of 64, 16-byte rows; f32 always: its planes).
struct Source {
  const void *p;
  size_t stride;
  uint32_t rows, d;
  int dt;
  uint32_t whole;  // columns of an image
  bool direct() const { return dt != AS_F32 && d == whole && stride % 8 == 0 && ((uintptr_t)p & 15) == 0; }
  uint32_t pitch() const { return whole; }
  uint32_t planes() const { return planes_of(dt); }
  uint64_t image_elems(bool raw) const { return direct() || raw ? 0 : (uint64_t)rows * pitch() * planes(); }
};

// Which tile.  Rounds of workgroups times what one takes: the large one has the chip's 256 units to itself, two square ones share a
// unit, each a quarter of the work at 0.8 of the rate (8192 x 16384 x 1024: 259 and 330 us).
bool large_pays(uint32_t m, uint32_t n) {
  const uint64_t large = (uint64_t)cdiv(m, 256) * cdiv(n, 256), square = (uint64_t)cdiv(m, 128) * cdiv(n, 128);
  return 1.6 * (double)((large + kChips - 1) / kChips) <= (double)((square + 2 * kChips - 1) / (2 * kChips));
}
int product_tile(uint32_t m, uint32_t n) { return n <= 64 ? kSlim : n <= 128 || m <= 128 || !large_pays(m, n) ? kSquare : kLarge; }

struct Plan {
  uint32_t n, v, d, planes, steps, pitch, parts;
  int dt;
  int rows_tiles;  // forward for short rows: tiles of 16 rows a wave, 0: the tiled form
  int tile;
  uint32_t n_tiles, v_tiles, per, chunks;
  // backward
  uint32_t piece, pieces, splits;
  int tile_w, tile_x;
  int fused;                 // steps of 32 columns of the form for short rows (table_loss_rows.h), 0: through G in memory
  int few;                   // steps of 32 columns a wave of the form for few rows (table_loss_few.h), 0: not taken
  uint32_t few_groups;       // its workgroups
  bool raw;                  // ... reads the matrices as they are where they cannot be operands at once (else images are made)
  uint32_t x_blocks, w_blocks, w_splits, n_pad;
  bool want_x, want_w, want_b;
};
Plan make_plan(uint32_t n, uint32_t v, uint32_t d, int dt) {
  Plan p{};
  p.n = n, p.v = v, p.d = d, p.dt = dt;
  p.planes = planes_of(dt);
  p.steps = cdiv(d, 64);
  p.pitch = p.steps * 64;
  p.tile = product_tile(v, n);
  p.n_tiles = cdiv(n, kShape[p.tile].bn);
  p.v_tiles = cdiv(v, kShape[p.tile].bm);
  return p;
}
// workgroups of a tile that the chip runs at once
uint32_t slots_of(int tile) { return tile == kLarge ? kChips : 2 * kChips; }
// tiles a workgroup walks: so many that whole rounds of workgroups fill the chip (1 024 workgroups of six tiles on 256 units: the fifth
// round is nearly empty, 18 % of the time)
void plan_walk(Plan &p) {
  const uint32_t slots = slots_of(p.tile);
  uint64_t best = ~0ull;
  for (uint32_t r = 1; r <= 8; ++r) {
    const uint32_t chunks = std::max(1u, std::min((uint32_t)((uint64_t)slots * r / p.n_tiles), p.v_tiles)), per = cdiv(p.v_tiles, chunks);
    const uint64_t blocks = (uint64_t)p.n_tiles * cdiv(p.v_tiles, per);
    // rounds of tiles, and a twentieth of a tile for each workgroup's start
    const uint64_t cost = (blocks + slots - 1) / slots * (20ull * per + 1);
    if (cost < best) {
      best = cost;
      p.per = per;
    }
  }
  p.chunks = cdiv(p.v_tiles, p.per);
}
// parts of a contraction whose output has so many tiles
uint32_t plan_splits(uint64_t tiles, uint32_t slots, uint32_t most) {
  uint32_t best = 1;
  double cost = 1e30;
  for (uint32_t s = 1; s <= std::min(most, 64u); ++s) {
    const double c = (double)((tiles * s + slots - 1) / slots) / s * (1 + 0.01 * s);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best;
}

// the form for short rows: its steps of 32 columns, and tiles of 16 rows a wave holds (what 256 registers take)
int fused_steps(uint32_t d, uint32_t planes) { return d <= 64 ? 2 : d <= 128 ? 4 : d <= 256 && planes == 1 ? 8 : 0; }
// ... and waves a SIMD.  1 024 rows x 1 M items, bf16, us (dW / dX): 64 values 2 tiles x 4 waves 270 / -, 3 x 3 257 / -, 4 x 2 283 / 264;
// 128 values 2 x 3 515 / 439, 3 x 2 490 / 480, 4 x 2 728 / 632 (spills); 256 values 1 x 2 1 273 / 1 262, 2 x 2 1 437 / 1 410 (spills).
// f32 (stages of three planes: one workgroup a unit at 128 values), 512 rows x 100 000 items: 64 values 2 x 3 79 / 62, 4 x 2 81 / 81; 128 values
// 1 x 1 244 / 191, 2 x 1 218 / 147, 4 x 1 181 / 138
constexpr int fused_rows(int steps, int planes, bool items) { return planes > 1 ? steps : steps == 8 ? 1 : steps == 2 || items ? 3 : 2; }
constexpr int fused_waves(int steps, int planes, bool items) { return planes > 1 ? (steps == 2 ? 3 : 1) : steps == 8 ? 2 : steps == 2 || !items ? 3 : 2; }
// The form for few rows: its steps of 32 columns a wave, as many columns as four waves hold; up to 128 columns (four steps) a wave takes
// whole items.  Waves a SIMD: what its registers leave.
int few_steps(uint32_t d) {
  if (d > 1024) return 0;
  if (d <= 128) return d <= 32 ? 1 : d <= 64 ? 2 : 4;
  const int kc = (int)cdiv(d, 128);
  return kc <= 4 ? kc : kc <= 6 ? 6 : 8;
}
int few_share(uint32_t d) { return d <= 128 ? 1 : 4; }
enum { kFewOne, kFewTwo, kFewFour, kFewGrad };  // forward with one, two or four tiles of 16 rows, backward
constexpr int few_waves(int steps, bool f32, int what) {
  return f32 ? (steps <= (what == kFewOne ? 4 : 2) ? 2 : 1) : what == kFewOne ? (steps <= 4 ? 4 : steps <= 6 ? 3 : 2) : what == kFewTwo ? (steps <= 2 ? 4 : steps <= 4 ? 3 : 2) : what == kFewFour ? (steps <= 1 ? 4 : steps <= 6 ? 2 : 1) : steps <= 2 ? 4 : 2;
}
uint32_t few_groups(int steps, uint32_t d, bool f32, int what, uint32_t v) {
  return std::max(1u, std::min((uint32_t)few_waves(steps, f32, what) * kChips, cdiv(v, 16 * (4 / few_share(d)))));
}
// An image is read and written once more than the matrix itself; reading the matrix as it is costs each workgroup that walks it the
// splitting or shifting of its pieces.  A step of 512 f32 rows of 128, 100 000 items: images 490 us, as they are 515; 777 rows of 200
// (f16, odd stride), 31 013 items: 171 and 198; one or two blocks of rows: the images would be a third of the time.
bool raw_pays(const Plan &p) { return p.n <= 128; }
void plan_backward(Plan &p, bool x, bool w, bool b) {
  p.want_x = x, p.want_w = w, p.want_b = b;
  p.few = p.n <= 16 ? few_steps(p.d) : 0;
  if (p.few) {
    p.few_groups = p.splits = few_groups(p.few, p.d, p.planes > 1, kFewGrad, p.v);
    p.n_pad = 64;
    p.w_splits = 1;
    return;
  }
  p.fused = fused_steps(p.d, p.planes);
  if (p.fused) {
    const uint32_t stages = cdiv(p.v, 64), groups = fused_waves(p.fused, p.planes, false) * kChips;
    p.pitch = p.fused * 32;
    p.raw = raw_pays(p);
    p.x_blocks = cdiv(p.n, 64 * fused_rows(p.fused, p.planes, false));
    p.w_blocks = cdiv(p.v, 64 * fused_rows(p.fused, p.planes, true));
    p.n_pad = up(p.n, 64);
    // the items in parts, so that the workgroups are there that a compute unit holds; the batch too, where the table is short
    p.splits = std::max(1u, std::min(groups / std::min(p.x_blocks, groups), stages));
    p.w_splits = std::max(1u, std::min(groups / std::min(p.w_blocks, groups), cdiv(p.n, 256)));
    return;
  }
  const uint32_t bm = kShape[p.tile].bm, bn = kShape[p.tile].bn;
  p.n_pad = up(p.n, std::max(bn, 64u));
  // G of a piece: some 256 MB, what the last cache before memory holds, and whole rounds of the large tile for the piece's dW
  const uint64_t per_item = (uint64_t)p.n_pad * 2 * p.planes;
  const uint32_t round = std::max(1u, (uint32_t)kChips / cdiv(p.d, 256)) * 256;
  uint64_t piece = std::max<uint64_t>((320ull << 20) / per_item / round, 1) * round;
  if (piece * per_item > (512ull << 20)) piece = std::max<uint64_t>((256ull << 20) / per_item / 256 * 256, 256);
  piece = std::min<uint64_t>(piece, up(p.v, bm));
  p.piece = (uint32_t)up(piece, bm);
  p.pieces = cdiv(p.v, p.piece);
  p.piece = up(cdiv(p.v, p.pieces), bm);  // even pieces
  p.pieces = cdiv(p.v, p.piece);
  p.v_tiles = cdiv(p.piece, bm);
  plan_walk(p);
  p.tile_w = product_tile(p.d, std::min(p.piece, p.v));
  p.tile_x = p.n <= 64 ? kSlim : p.d <= 128 || p.n <= 128 ? kSquare : kLarge;
  const uint64_t tiles = (uint64_t)cdiv(p.d, kShape[p.tile_x].bm) * cdiv(p.n, kShape[p.tile_x].bn);
  // the contraction over the piece is split where the output alone does not fill the chip
  p.splits = plan_splits(tiles, slots_of(p.tile_x), cdiv(p.piece, 256));
  // so is the batch where the table is short (6 000 rows, 150 items of 800)
  const uint64_t w_tiles = (uint64_t)cdiv(p.d, kShape[p.tile_w].bm) * cdiv(p.v, kShape[p.tile_w].bn);
  p.w_splits = p.pieces == 1 && w_tiles * 2 <= slots_of(p.tile_w) ? plan_splits(w_tiles, slots_of(p.tile_w), cdiv(p.n, 512)) : 1;
}

// waves a SIMD of the forward (1 024 rows x 1 M items of 128: four tiles of rows x 2 waves 293 us, x 3 282, two x 4 316)
constexpr int sums_waves(int steps, int planes, int tiles) { return planes > 1 ? (steps == 2 ? 2 : 1) : steps == 8 || tiles < 4 ? 2 : steps == 4 ? 3 : 4; }
// Forward, up to 64 rows: a table that is an operand as it lies streams through the other forms at 5 to 6 TB/s (4 to 64 rows, 512 187 items
// of 640 (f16): 124 us, in the form for few rows 190 to 281; small tables are quicker without the tiles: 20 rows, 10 000 of 768 16 and
// 19 us).  What would need an image does not: 56 bf16 rows, 500 000 of 700 at an odd stride, 297 and 432 us; 16 rows of 200 47 and 75
// (60 rows 84 and 81); 24 f32 rows, 500 000 of 128 98 and 135
// (of 64: 51 and 48).  16-bit rows of up to 128 are shifted as quickly by
// the short rows' form (16 rows of 100, 50 us, here 57).
bool few_pays(const Plan &p, bool table_direct) {
  if (p.n > 64) return false;
  if (p.planes > 1) return p.n <= 32 || p.d > 128;  // (718 298 items of 384: 24 rows 500 us, 48 535, by images 1 020; only long rows of small tables lose: 48 x 100 000 of 768 402 and 311)
  if (table_direct) return !p.fused && (uint64_t)p.v * p.d < (16ull << 20);
  return p.d > 128 && (p.n <= 32 || p.d > 256);
}
void plan_forward(Plan &p, bool table_direct) {
  p.fused = fused_steps(p.d, p.planes);
  p.few = few_pays(p, table_direct) ? few_steps(p.d) : 0;
  if (p.few) {
    p.fused = 0;
    p.few_groups = few_groups(p.few, p.d, p.planes > 1, p.n <= 16 || p.planes > 1 ? kFewOne : p.n <= 32 ? kFewTwo : kFewFour, p.v);
    p.parts = p.few_groups * (4 / few_share(p.d));
    return;
  }
  if (p.fused) {
    p.pitch = p.fused * 32;
    p.rows_tiles = p.n <= 64 ? 1 : p.n <= 128 ? 2 : 4;
    p.raw = raw_pays(p);
    p.x_blocks = cdiv(p.n, 64 * p.rows_tiles);
    // few rows: the pass over the table is all there is, four workgroups a compute unit keep it in flight
    const uint32_t groups = (p.rows_tiles == 1 ? 4 : sums_waves(p.fused, p.planes, p.rows_tiles)) * kChips;
    p.splits = std::max(1u, std::min(groups / std::min(p.x_blocks, groups), cdiv(p.v, 64)));
    p.parts = p.splits;
    return;
  }
  plan_walk(p);
  p.parts = p.chunks * kShape[p.tile].wm;
}

struct ForwardScratch {
  float2 *part;
  unsigned short *x_image, *t_image;
};
uint64_t forward_layout(const Plan &p, const Source &x, const Source &t, char *base, ForwardScratch &s) {
  Layout l{base};
  s.part = l.take<float2>((uint64_t)p.parts * p.n);
  s.x_image = l.take<unsigned short>(x.image_elems(p.few || (p.fused && p.raw)));
  s.t_image = l.take<unsigned short>(t.image_elems(p.few || (p.fused && p.raw)));
  return l.at;
}
struct BackwardScratch {
  float *coef;
  unsigned short *x_image, *t_image, *G;
  u32x2 *met;
  uint32_t *met_count;
  float *sums, *w_sums, *bias_part;
  float *lse, *every, *entry, *rest;
  int *target;
};
uint64_t backward_layout(const Plan &p, const Source &x, const Source &t, char *base, BackwardScratch &s) {
  Layout l{base};
  const uint64_t pl = p.planes;
  s.coef = l.take<float>(2);
  s.x_image = l.take<unsigned short>(x.image_elems(p.few || (p.fused && p.raw)));
  s.t_image = l.take<unsigned short>(t.image_elems(p.few || (p.fused && p.raw)));
  s.lse = l.take<float>(p.n_pad);
  s.every = l.take<float>(p.n_pad);
  s.entry = l.take<float>(p.n_pad);
  s.rest = l.take<float>(p.n_pad);
  s.target = l.take<int>(p.n_pad);
  if (p.fused || p.few) {
    s.sums = l.take<float>(p.want_x ? (uint64_t)p.splits * p.n * up(p.d, 8) : 0);
    s.w_sums = l.take<float>(p.w_splits > 1 ? (uint64_t)p.w_splits * p.v * up(p.d, 8) : 0);
    s.bias_part = l.take<float>(p.w_splits > 1 ? (uint64_t)p.w_splits * p.v : 0);
    return l.at;
  }
  s.G = l.take<unsigned short>((uint64_t)p.n_pad * p.piece * pl);
  const uint64_t groups = p.want_w && p.planes == 1 ? (p.v + 63) / 64 : 0;
  s.met = l.take<u32x2>(groups * kMet);
  s.met_count = l.take<uint32_t>(groups);
  s.sums = l.take<float>(p.want_x ? (uint64_t)p.splits * p.n * up(p.d, 8) : 0);
  s.w_sums = l.take<float>(p.want_w && p.w_splits > 1 ? (uint64_t)p.w_splits * p.v * up(p.d, 8) : 0);
  s.bias_part = l.take<float>(p.want_b ? (uint64_t)p.n_tiles * kShape[p.tile].wn * p.piece : 0);
  return l.at;
}

template <class F>
void by_tile(int tile, F &&f) {
  if (tile == kSlim) f(std::integral_constant<int, kSlim>{});
  else if (tile == kSquare) f(std::integral_constant<int, kSquare>{});
  else f(std::integral_constant<int, kLarge>{});
}
template <int FMT, int K, bool AT = false, bool BT = false>
using TileOf = std::conditional_t<K == kSlim, Slim<FMT, AT, BT>, std::conditional_t<K == kSquare, Square<FMT, AT, BT>, Large<FMT, AT, BT>>>;
template <class F>
void by_type(int dt, F &&f) {
  if (dt == AS_F32) f(std::integral_constant<int, AS_F32>{});
  else if (dt == AS_BF16) f(std::integral_constant<int, AS_BF16>{});
  else f(std::integral_constant<int, AS_F16>{});
}
unsigned spread(uint64_t items, uint64_t per_block) { return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>((items + per_block - 1) / per_block, 16384)); }

// The two matrices as the products read them: each as it is, or its image.
struct Operands {
  const char *x, *t;
  size_t x_ld, t_ld;
};
// (raw: the kernels take the matrices as they are)
int make_operands(as_ctx *ctx, const Source &x, const Source &t, bool raw, unsigned short *x_image, unsigned short *t_image, Operands *out) {
  ImageJobs jobs{};
  uint32_t count = 0;
  uint64_t most = 1;
  auto add = [&](const Source &s, unsigned short *image, const char **p, size_t *ld) {
    const size_t es = dtype_size(s.dt);
    if (s.direct() || raw) {
      *p = (const char *)s.p;
      *ld = s.stride * es;
    } else {
      *p = (const char *)image;
      *ld = (size_t)s.pitch() * s.planes() * 2;
    }
    if (s.direct() || raw) return;
    jobs.job[count++] = ImageJob{(const char *)s.p, s.stride * es, s.rows, s.d, s.pitch(), image};
    most = std::max<uint64_t>(most, (uint64_t)s.rows * s.pitch() / 4096);
  };
  add(x, x_image, &out->x, &out->x_ld);
  add(t, t_image, &out->t, &out->t_ld);
  if (!count) return AS_OK;
  by_type(x.dt, [&](auto dt) {
    hipLaunchKernelGGL((image_kernel<decltype(dt)::value>), dim3((unsigned)std::min<uint64_t>(most, 2048), count), dim3(256), 0, ctx->stream, jobs);
  });
  AS_HIP(ctx, hipGetLastError());
  return AS_OK;
}
template <class F>
void by_steps(int dt, bool raw, int steps, F &&f) {  // f(type, raw, steps)
  constexpr std::integral_constant<int, AS_F32> f32{};
  constexpr std::integral_constant<int, AS_BF16> bf{};
  constexpr std::integral_constant<int, AS_F16> hf{};
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  auto by = [&](auto type, auto rw) {
    if (steps == 2) f(type, rw, std::integral_constant<int, 2>{});
    else if (steps == 4) f(type, rw, std::integral_constant<int, 4>{});
    else if constexpr (decltype(type)::value != AS_F32) f(type, rw, std::integral_constant<int, 8>{});
  };
  if (dt == AS_F32) raw ? by(f32, yes) : by(f32, no);
  else if (dt == AS_BF16) raw ? by(bf, yes) : by(bf, no);
  else raw ? by(hf, yes) : by(hf, no);
}
template <bool ITEMS>
void launch_rows_grad(as_ctx *ctx, int dt, bool raw, int steps, bool bias, const LossRowsArgs &a) {
  by_steps(dt, raw, steps, [&](auto type, auto rw, auto kd) {
    constexpr int DT = decltype(type)::value, KD = decltype(kd)::value, P = planes_of(DT), RT = fused_rows(KD, P, ITEMS), W = fused_waves(KD, P, ITEMS);
    constexpr bool RAW = decltype(rw)::value;
    if (bias) hipLaunchKernelGGL((loss_rows_grad_kernel<DT, RAW, RT, KD, ITEMS, true, W>), dim3(a.r_blocks * a.splits), dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((loss_rows_grad_kernel<DT, RAW, RT, KD, ITEMS, false, W>), dim3(a.r_blocks * a.splits), dim3(256), 0, ctx->stream, a);
  });
}
template <class F>
void by_few_steps(int dt, int steps, uint32_t d, F &&f) {  // f(type, steps, waves that share the columns)
  by_type(dt, [&](auto type) {
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 4> four{};
    if (few_share(d) == 1) {
      if (steps == 1) f(type, one, one);
      else if (steps == 2) f(type, std::integral_constant<int, 2>{}, one);
      else f(type, four, one);
    } else {
      if (steps == 2) f(type, std::integral_constant<int, 2>{}, four);
      else if (steps == 3) f(type, std::integral_constant<int, 3>{}, four);
      else if (steps == 4) f(type, four, four);
      else if (steps == 6) f(type, std::integral_constant<int, 6>{}, four);
      else f(type, std::integral_constant<int, 8>{}, four);
    }
  });
}
void launch_few_sums(as_ctx *ctx, const Plan &p, bool general, LossFewArgs a) {
  by_few_steps(p.dt, p.few, p.d, [&](auto type, auto kc, auto share) {
    constexpr int DT = decltype(type)::value, KC = decltype(kc)::value, WK = decltype(share)::value;
    constexpr bool F32 = DT == AS_F32;
    a.slices = p.few_groups;
    if constexpr (F32) {  // (16 rows at a time, their planes leave no room for more)
      a.row_blocks = cdiv(p.n, 16);
      const dim3 grid(up(p.few_groups, 8) * a.row_blocks);
      if (general) hipLaunchKernelGGL((loss_few_sums_kernel<DT, KC, 1, true, WK, few_waves(KC, F32, kFewOne)>), grid, dim3(256), 0, ctx->stream, a);
      else hipLaunchKernelGGL((loss_few_sums_kernel<DT, KC, 1, false, WK, few_waves(KC, F32, kFewOne)>), grid, dim3(256), 0, ctx->stream, a);
    } else if constexpr (WK == 4) {  // (few_pays: 16-bit rows of up to 128 columns, and 33 to 64 of up to 256, go another way)
      auto go = [&](auto tiles, auto gen) {
        constexpr int RT = decltype(tiles)::value;
        hipLaunchKernelGGL((loss_few_sums_kernel<DT, KC, RT, decltype(gen)::value, WK, few_waves(KC, F32, RT == 1 ? kFewOne : RT == 2 ? kFewTwo : kFewFour)>),
                           dim3(up(p.few_groups, 8)), dim3(256), 0, ctx->stream, a);
      };
      auto by_rows = [&](auto gen) {
        if (p.n <= 16) go(std::integral_constant<int, 1>{}, gen);
        else if (p.n <= 32) go(std::integral_constant<int, 2>{}, gen);
        else if constexpr (KC > 2) go(std::integral_constant<int, 4>{}, gen);
      };
      a.row_blocks = 1;
      if (general) by_rows(std::true_type{});
      else by_rows(std::false_type{});
    }
  });
}
void launch_few_grad(as_ctx *ctx, const Plan &p, const LossFewArgs &a) {
  by_few_steps(p.dt, p.few, p.d, [&](auto type, auto kc, auto share) {
    constexpr int DT = decltype(type)::value, KC = decltype(kc)::value, WK = decltype(share)::value, W = few_waves(KC, DT == AS_F32, kFewGrad);
    if (a.bias) hipLaunchKernelGGL((loss_few_grad_kernel<DT, KC, true, WK, W>), dim3(p.few_groups), dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((loss_few_grad_kernel<DT, KC, false, WK, W>), dim3(p.few_groups), dim3(256), 0, ctx->stream, a);
  });
}
template <int RT>
void launch_rows_sums(as_ctx *ctx, int dt, bool raw, int steps, bool general, const LossSumsArgs &a) {
  by_steps(dt, raw, steps, [&](auto type, auto rw, auto kd) {
    constexpr int DT = decltype(type)::value, KD = decltype(kd)::value, W = sums_waves(KD, planes_of(DT), RT);
    constexpr bool RAW = decltype(rw)::value;
    if (general) hipLaunchKernelGGL((loss_rows_sums_kernel<DT, RAW, RT, KD, true, W>), dim3(a.r_blocks * a.splits), dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL((loss_rows_sums_kernel<DT, RAW, RT, KD, false, W>), dim3(a.r_blocks * a.splits), dim3(256), 0, ctx->stream, a);
  });
}
void launch_product(as_ctx *ctx, int fmt, int tile, bool w, int out_type, const ProductArgs &p) {
  by_tile(tile, [&](auto k) {
    constexpr int K = decltype(k)::value;
    const dim3 grid(p.m_tiles * p.n_tiles * p.splits);
    auto go = [&](auto f, auto o, auto bt) {
      constexpr int FMT = decltype(f)::value, OUT = decltype(o)::value;
      constexpr bool BT = decltype(bt)::value;
      typedef TileOf<FMT, K, true, BT> TILE;
      hipLaunchKernelGGL((product_kernel<FMT, TILE, OUT, BT>), grid, dim3(TILE::NT), 0, ctx->stream, p);
    };
    constexpr std::integral_constant<int, AS_BF16> bf{};
    constexpr std::integral_constant<int, AS_F16> hf{};
    constexpr std::integral_constant<int, AS_F32> f32{};
    constexpr std::integral_constant<int, 0> acc{};
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    if (fmt == AS_BF16) !w ? go(bf, acc, no) : out_type == 0 ? go(bf, acc, yes) : out_type == AS_F32 ? go(bf, f32, yes) : go(bf, bf, yes);
    else !w ? go(hf, acc, no) : out_type == 0 ? go(hf, acc, yes) : go(hf, hf, yes);
  });
}

struct LossCall {
  uint64_t n, v, d, x_stride, table_stride;
  int dt;
  float scale;
};
int check_loss(as_ctx *ctx, const LossCall &c) {
  if (!ctx) return AS_ERR_ARG;
  if (hipSetDevice(ctx->device) != hipSuccess) return fail(ctx, AS_ERR_HIP, "hipSetDevice failed");
  ctx_enter(ctx);
  if (!dtype_is_training(c.dt)) return fail(ctx, AS_ERR_ARG, "dtype must be AS_F32, AS_BF16 or AS_F16");
  if (c.v == 0 || c.d == 0) return fail(ctx, AS_ERR_SHAPE, "the table needs at least one row and one column");
  if (c.n >= (1ull << 31) || c.v >= (1ull << 31) || c.d > 65536) return fail(ctx, AS_ERR_UNSUPPORTED, "at most 2^31 - 1 rows and items and 65536 columns");
  if (c.x_stride < c.d || c.table_stride < c.d) return fail(ctx, AS_ERR_ARG, "a row stride below the number of columns");
  if (!std::isfinite(c.scale)) return fail(ctx, AS_ERR_ARG, "scale must be finite");
  return AS_OK;
}
// targets in host memory are looked over here; on the device a target outside the table makes its loss NaN (and its row counts as ignored
// in the gradients)
int check_targets(as_ctx *ctx, const int64_t *targets, uint64_t n, uint64_t v, int64_t ignore) {
  if (n == 0 || pointer_home(ctx, targets) != 0) return AS_OK;
  for (uint64_t t = 0; t < n; ++t)
    if (targets[t] != ignore && (targets[t] < 0 || targets[t] >= (int64_t)v))
      return fail(ctx, AS_ERR_ARG, "target " + std::to_string(targets[t]) + " of row " + std::to_string(t) + " is outside the table");
  return AS_OK;
}
uint64_t span(uint64_t rows, uint64_t stride, uint64_t d, int dt) { return rows ? ((rows - 1) * stride + d) * dtype_size(dt) : 0; }

int forward_call(as_ctx *ctx, const LossCall &c, const void *x, const void *table, const float *bias, const int64_t *targets, int64_t ignore, float *losses,
                 float *lse, void *workspace, uint64_t workspace_bytes) {
  AS_TRY(check_loss(ctx, c));
  if (c.n == 0) return AS_OK;
  if (!x || !table || !targets || !losses || !lse) return fail(ctx, AS_ERR_ARG, "null argument");
  AS_TRY(check_targets(ctx, targets, c.n, c.v, ignore));
  BytesIn X, W, Bi, Y;
  BytesOut L, S;
  AS_TRY(X.bind(ctx, x, span(c.n, c.x_stride, c.d, c.dt)));
  AS_TRY(W.bind(ctx, table, span(c.v, c.table_stride, c.d, c.dt)));
  AS_TRY(Bi.bind(ctx, bias, bias ? c.v * 4 : 0));
  AS_TRY(Y.bind(ctx, targets, c.n * 8));
  AS_TRY(L.bind(ctx, losses, c.n * 4));
  AS_TRY(S.bind(ctx, lse, c.n * 4));
  Plan p = make_plan((uint32_t)c.n, (uint32_t)c.v, (uint32_t)c.d, c.dt);
  const int columns = fused_steps(p.d, p.planes) * 32;
  plan_forward(p, Source{W.p, (size_t)c.table_stride, p.v, p.d, c.dt, columns ? columns : p.pitch}.direct());
  const Source xs{X.p, (size_t)c.x_stride, p.n, p.d, c.dt, p.pitch}, ts{W.p, (size_t)c.table_stride, p.v, p.d, c.dt, p.pitch};
  ForwardScratch s{};
  Scratch scratch;
  AS_TRY(scratch.open(ctx, workspace, workspace_bytes, forward_layout(p, xs, ts, nullptr, s)));
  forward_layout(p, xs, ts, scratch.base, s);
  ProfScope prof(ctx, "cross_entropy");
  LossArgs a{};
  Operands o{};
  if (!p.few) AS_TRY(make_operands(ctx, xs, ts, p.fused && p.raw, s.x_image, s.t_image, &o));
  a.rows = o.x, a.rows_ld = o.x_ld, a.table = o.t, a.table_ld = o.t_ld;
  a.table_plane = a.rows_plane = (size_t)p.pitch * 2;
  a.n = p.n, a.v = p.v, a.steps = p.steps, a.all = p.steps * pairs_of(p.planes), a.per = p.per, a.v_tiles = p.v_tiles, a.n_tiles = p.n_tiles, a.chunks = p.chunks;
  a.scale = c.scale, a.bias = (const float *)Bi.p;
  const bool general = bias || !(c.scale > 0.f);
  if (p.few) {
    LossFewArgs r{};
    r.rows = (const char *)X.p, r.rows_ld = c.x_stride * dtype_size(c.dt), r.table = (const char *)W.p, r.table_ld = c.table_stride * dtype_size(c.dt);
    r.n = p.n, r.v = p.v, r.d = p.d, r.scale = c.scale, r.bias = a.bias, r.part = s.part;
    launch_few_sums(ctx, p, general, r);
  } else if (p.fused) {
    LossSumsArgs r{};
    r.r = a.rows, r.r_ld = a.rows_ld, r.nr = p.n, r.k = a.table, r.k_ld = a.table_ld, r.nk = p.v, r.d = p.d;
    r.r_blocks = p.x_blocks, r.splits = p.splits, r.scale = c.scale, r.bias = a.bias, r.part = s.part;
    const bool raw = p.raw && !(xs.direct() && ts.direct());
    if (p.rows_tiles == 1) launch_rows_sums<1>(ctx, c.dt, raw, p.fused, general, r);
    else if (p.rows_tiles == 2) launch_rows_sums<2>(ctx, c.dt, raw, p.fused, general, r);
    else launch_rows_sums<4>(ctx, c.dt, raw, p.fused, general, r);
  } else {
    by_tile(p.tile, [&](auto k) {
      constexpr int K = decltype(k)::value;
      auto go = [&](auto f, auto gen) {
        constexpr int FMT = decltype(f)::value;
        hipLaunchKernelGGL((loss_sums_kernel<FMT, TileOf<FMT, K>, decltype(gen)::value>), dim3(p.n_tiles * p.chunks), dim3(TileOf<FMT, K>::NT), 0, ctx->stream, a,
                           s.part);
      };
      constexpr std::integral_constant<int, AS_BF16> bf{};
      constexpr std::integral_constant<int, AS_F16> hf{};
      if (format_of(c.dt) == AS_BF16) general ? go(bf, std::true_type{}) : go(bf, std::false_type{});
      else general ? go(hf, std::true_type{}) : go(hf, std::false_type{});
    });
  }
  AS_HIP(ctx, hipGetLastError());
  by_type(c.dt, [&](auto dt) {
    hipLaunchKernelGGL((loss_join_kernel<decltype(dt)::value>), dim3(row_groups(c.n)), dim3(256), 0, ctx->stream, (const float2 *)s.part,
                       p.parts, X.p, (size_t)c.x_stride, W.p, (size_t)c.table_stride, (const float *)Bi.p, (const int64_t *)Y.p, p.n, p.v, p.d,
                       c.scale, ignore, (float *)L.p, (float *)S.p);
  });
  AS_HIP(ctx, hipGetLastError());
  AS_TRY(L.finish(ctx));
  AS_TRY(S.finish(ctx));
  return finish_call(ctx);
}

int backward_call(as_ctx *ctx, const LossCall &c, const void *x, const void *table, const float *bias, const int64_t *targets, int64_t ignore, const float *lse,
                  const float *gl, const float *ge, void *gx, uint64_t gx_stride, void *gw, uint64_t gw_stride, float *gb, void *workspace,
                  uint64_t workspace_bytes) {
  AS_TRY(check_loss(ctx, c));
  if (gb && !bias) return fail(ctx, AS_ERR_ARG, "a gradient of the bias without a bias");
  if ((gx && gx_stride < c.d) || (gw && gw_stride < c.d)) return fail(ctx, AS_ERR_ARG, "a row stride below the number of columns");
  if (!gx && !gw && !gb) return AS_OK;
  if ((gx && (gx == x || gx == table || gx == gw)) || (gw && (gw == x || gw == table)))
    return fail(ctx, AS_ERR_ARG, "gradients must not share memory with the inputs or each other");
  if (c.n && (!x || !table || !targets || !lse || !gl)) return fail(ctx, AS_ERR_ARG, "null argument");
  AS_TRY(check_targets(ctx, targets, c.n, c.v, ignore));
  BytesIn X, W, Bi, Y, Ls, Gl, Ge;
  BytesOut Ox, Ow, Ob;
  AS_TRY(X.bind(ctx, x, span(c.n, c.x_stride, c.d, c.dt)));
  AS_TRY(W.bind(ctx, table, span(c.n ? c.v : 0, c.table_stride, c.d, c.dt)));
  AS_TRY(Bi.bind(ctx, bias, bias ? c.v * 4 : 0));
  AS_TRY(Y.bind(ctx, targets, c.n * 8));
  AS_TRY(Ls.bind(ctx, lse, c.n * 4));
  AS_TRY(Gl.bind(ctx, gl, c.n * 4));
  AS_TRY(Ge.bind(ctx, ge, ge ? c.n * 4 : 0));
  if (gx && c.n && pointer_home(ctx, gx) == 0 && gx_stride != c.d) return fail(ctx, AS_ERR_ARG, "gradients in host memory must be dense");
  if (gw && pointer_home(ctx, gw) == 0 && gw_stride != c.d) return fail(ctx, AS_ERR_ARG, "gradients in host memory must be dense");
  AS_TRY(Ox.bind(ctx, gx, span(c.n, gx_stride, c.d, c.dt)));
  AS_TRY(Ow.bind(ctx, gw, span(c.v, gw_stride, c.d, c.dt)));
  AS_TRY(Ob.bind(ctx, gb, c.v * 4));
  ProfScope prof(ctx, "cross_entropy_backward");
  if (c.n == 0) {  // a sum over no rows
    if (gw)
      by_type(c.dt, [&](auto dt) {
        hipLaunchKernelGGL((zero_rows_kernel<decltype(dt)::value>), dim3(spread(c.v * c.d, 1024)), dim3(256), 0, ctx->stream, Ow.p, (size_t)gw_stride, c.v, (uint32_t)c.d);
      });
    if (gb) hipLaunchKernelGGL((zero_rows_kernel<AS_F32>), dim3(spread(c.v, 1024)), dim3(256), 0, ctx->stream, Ob.p, (size_t)1, c.v, 1u);
    AS_HIP(ctx, hipGetLastError());
    AS_TRY(Ow.finish(ctx));
    AS_TRY(Ob.finish(ctx));
    return finish_call(ctx);
  }
  Plan p = make_plan((uint32_t)c.n, (uint32_t)c.v, (uint32_t)c.d, c.dt);
  plan_backward(p, gx != nullptr, gw != nullptr, gb != nullptr);
  const Source xs{X.p, (size_t)c.x_stride, p.n, p.d, c.dt, p.pitch}, ts{W.p, (size_t)c.table_stride, p.v, p.d, c.dt, p.pitch};
  BackwardScratch s{};
  Scratch scratch;
  AS_TRY(scratch.open(ctx, workspace, workspace_bytes, backward_layout(p, xs, ts, nullptr, s)));
  backward_layout(p, xs, ts, scratch.base, s);
  GradArgs g{};
  LossArgs &a = g.l;
  Operands o{};
  if (!p.few) AS_TRY(make_operands(ctx, xs, ts, p.fused && p.raw, s.x_image, s.t_image, &o));
  const char *table16 = o.t;
  a.rows = o.x, a.rows_ld = o.x_ld, a.table_ld = o.t_ld;
  AS_HIP(ctx, hipGetLastError());
  const float *coef = s.coef;
  const float *rest = p.planes == 1 ? s.rest : nullptr;
  const LossRowInputs by_row{X.p, W.p, (size_t)c.x_stride, (size_t)c.table_stride, p.d, p.n, p.n_pad, p.v, (const float *)Bi.p, (const float *)Ls.p,
                             (const float *)Gl.p, (const float *)Ge.p, (const int64_t *)Y.p, ignore, c.scale, c.dt == AS_F16 ? 14 : 0, s.coef, s.lse, s.every,
                             s.entry, s.rest, s.target};
  if (p.n > kFewRows)
    hipLaunchKernelGGL(coef_scale_kernel, dim3(1), dim3(1024), 0, ctx->stream, by_row.gl, by_row.ge, by_row.targets, ignore, p.n, by_row.power, s.coef);
  by_type(c.dt, [&](auto dt) {
    constexpr int DT = decltype(dt)::value, FMT = format_of(DT);
    if (p.n > kFewRows) hipLaunchKernelGGL((loss_rows_kernel<DT, FMT, false>), dim3(row_groups(p.n_pad)), dim3(256), 0, ctx->stream, by_row);
    else hipLaunchKernelGGL((loss_rows_kernel<DT, FMT, true>), dim3(row_groups(p.n_pad)), dim3(256), 0, ctx->stream, by_row);
  });
  AS_HIP(ctx, hipGetLastError());
  // dX from its parts, or dW where the batch was split
  auto join = [&](const float *sums, uint32_t splits, uint32_t n, bool with_rest, void *out, uint64_t stride) {
    by_type(c.dt, [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
      const uint32_t pitch = up(p.d, 8);
      const uint64_t total = (uint64_t)n * pitch;
      const float *r = with_rest ? rest : nullptr;
      auto go = [&](auto ways) {
        constexpr int WAYS = decltype(ways)::value;
        hipLaunchKernelGGL((grad_rows_join_kernel<DT, WAYS>), dim3(spread(total, WAYS == 64 ? 64 : WAYS == 4 ? 256 : 1024)), dim3(WAYS == 64 ? 1024 : 256), 0, ctx->stream,
                           sums, splits, pitch, n, p.d, c.scale, coef, (const int *)s.target, r, W.p, (size_t)c.table_stride, out, (size_t)stride);
      };
      // 16 waves a compute unit, or as many ways as parts: 777 x 200 from 64 parts 7 us in 4 ways, 25 in 64; 9 x 64 from 1 024 parts 5.6 us
      // in 64, 12 in 16
      const uint64_t waves = cdiv(total, 256);
      if (splits <= 4 || waves >= 16 * kChips) go(std::integral_constant<int, 1>{});
      else if (splits <= 16 || waves >= kChips) go(std::integral_constant<int, 4>{});
      else go(std::integral_constant<int, 64>{});
    });
  };
  if (p.few) {
    LossFewArgs r{};
    r.rows = (const char *)X.p, r.rows_ld = c.x_stride * dtype_size(c.dt), r.table = (const char *)W.p, r.table_ld = c.table_stride * dtype_size(c.dt);
    r.n = p.n, r.v = p.v, r.d = p.d, r.scale = c.scale, r.bias = (const float *)Bi.p;
    r.lse = s.lse, r.every = s.every, r.entry = s.entry, r.rest = s.rest, r.target = s.target, r.coef = coef;
    r.sums = s.sums, r.sums_pitch = up(p.d, 8), r.want_x = p.want_x;
    r.out = Ow.p, r.out_stride = gw_stride;
    r.grad_bias = (float *)Ob.p;
    launch_few_grad(ctx, p, r);
    AS_HIP(ctx, hipGetLastError());
  } else if (p.fused) {
    const bool raw = p.raw && !(xs.direct() && ts.direct());
    LossRowsArgs r{};
    r.d = p.d, r.scale = c.scale, r.bias = (const float *)Bi.p, r.coef = coef;
    r.lse = s.lse, r.every = s.every, r.entry = s.entry, r.rest = s.rest, r.target = s.target;
    r.sums_pitch = up(p.d, 8);
    if (p.want_w || p.want_b) {
      r.r = o.t, r.r_ld = o.t_ld, r.nr = p.v;
      r.k = o.x, r.k_ld = o.x_ld, r.nk = p.n;
      r.r_blocks = p.w_blocks, r.splits = p.w_splits;
      if (p.w_splits > 1) r.sums = s.w_sums;
      r.out = Ow.p, r.out_stride = gw_stride;
      r.grad_bias = !p.want_b ? nullptr : p.w_splits > 1 ? s.bias_part : (float *)Ob.p;
      launch_rows_grad<true>(ctx, c.dt, raw, p.fused, bias != nullptr, r);
      if (p.w_splits > 1) {
        if (p.want_w) join(s.w_sums, p.w_splits, p.v, false, Ow.p, gw_stride);
        if (p.want_b)
          hipLaunchKernelGGL(bias_join_kernel, dim3(cdiv(p.v, 256)), dim3(256), 0, ctx->stream, (const float *)s.bias_part, p.w_splits, p.v, p.v, coef, (float *)Ob.p);
      }
    }
    if (p.want_x) {
      r.r = o.x, r.r_ld = o.x_ld, r.nr = p.n;
      r.k = o.t, r.k_ld = o.t_ld, r.nk = p.v;
      r.r_blocks = p.x_blocks, r.splits = p.splits;
      r.sums = s.sums;
      launch_rows_grad<false>(ctx, c.dt, raw, p.fused, bias != nullptr, r);
    }
    AS_HIP(ctx, hipGetLastError());
  }
  a.table_plane = a.rows_plane = (size_t)p.pitch * 2;
  a.n = p.n, a.steps = p.steps, a.all = p.steps * pairs_of(p.planes), a.n_tiles = p.n_tiles, a.per = p.per;
  a.scale = c.scale;
  g.lse = s.lse, g.every = s.every, g.entry = s.entry, g.target = s.target, g.coef = coef;
  g.G = s.G, g.g_pitch = p.piece;
  g.bias_part = p.want_b ? s.bias_part : nullptr;
  const int fmt = format_of(c.dt);
  if (!p.fused && !p.few && rest && p.want_w) {
    const uint32_t groups = cdiv(p.v, 64);
    hipLaunchKernelGGL(met_kernel, dim3(groups), dim3(512), 0, ctx->stream, (const int *)s.target, p.n, s.met, s.met_count);
  }
  for (uint32_t v0 = 0; !p.fused && !p.few && v0 < p.v; v0 += p.piece) {
    const uint32_t items = std::min(p.piece, p.v - v0);
    a.table = table16 + (size_t)v0 * a.table_ld;
    a.v = items, a.v_tiles = cdiv(items, kShape[p.tile].bm), a.chunks = cdiv(a.v_tiles, p.per);
    a.bias = bias ? (const float *)Bi.p + v0 : nullptr;
    g.v_begin = v0;
    by_tile(p.tile, [&](auto k) {
      constexpr int K = decltype(k)::value;
      auto go = [&](auto f, auto planes, auto with_bias) {
        constexpr int FMT = decltype(f)::value;
        hipLaunchKernelGGL((loss_grad_kernel<FMT, TileOf<FMT, K>, decltype(planes)::value, decltype(with_bias)::value>), dim3(a.n_tiles * a.chunks),
                           dim3(TileOf<FMT, K>::NT), 0, ctx->stream, g);
      };
      constexpr std::integral_constant<int, AS_BF16> bf{};
      constexpr std::integral_constant<int, AS_F16> hf{};
      constexpr std::true_type yes{};
      constexpr std::false_type no{};
      constexpr std::integral_constant<int, 1> one{};
      constexpr std::integral_constant<int, kF32Planes> three{};
      if (c.dt == AS_BF16) bias ? go(bf, one, yes) : go(bf, one, no);
      else if (c.dt == AS_F16) bias ? go(hf, one, yes) : go(hf, one, no);
      else bias ? go(bf, three, yes) : go(bf, three, no);
    });
    if (p.want_b)
      hipLaunchKernelGGL(bias_join_kernel, dim3(cdiv(items, 256)), dim3(256), 0, ctx->stream, (const float *)s.bias_part, p.n_tiles * kShape[p.tile].wn, p.piece, items,
                         coef, (float *)Ob.p + v0);
    ProductArgs w{};
    w.B = (const char *)s.G, w.b_ld = (size_t)p.piece * p.planes * 2, w.b_plane = (size_t)p.piece * 2, w.b_cols = p.piece / 8, w.k_b = p.n_pad;
    w.m = p.d, w.a_plane = (size_t)p.pitch * 2, w.a_cols = p.pitch / 8, w.pairs = pairs_of(p.planes);
    w.scale = c.scale, w.coef = coef;
    if (p.want_w) {
      w.A = a.rows, w.a_ld = a.rows_ld, w.k_a = p.n;
      w.n = items, w.m_tiles = cdiv(p.d, kShape[p.tile_w].bm), w.n_tiles = cdiv(items, kShape[p.tile_w].bn);
      w.steps = cdiv(p.n, 64), w.splits = p.w_splits;
      w.sums = s.w_sums, w.sums_pitch = up(p.d, 8), w.first = 1;
      w.out = (char *)Ow.p + (size_t)v0 * gw_stride * dtype_size(c.dt), w.out_stride = gw_stride;
      if (rest) w.met = s.met + (size_t)(v0 / 64) * kMet, w.met_count = s.met_count + v0 / 64, w.rest = rest;
      launch_product(ctx, fmt, p.tile_w, true, p.w_splits > 1 ? 0 : c.dt, w);
      if (p.w_splits > 1) join(s.w_sums, p.w_splits, p.v, false, Ow.p, gw_stride);
    }
    if (p.want_x) {
      w.met = nullptr;
      w.A = a.table, w.a_ld = a.table_ld, w.k_a = items;
      w.n = p.n, w.m_tiles = cdiv(p.d, kShape[p.tile_x].bm), w.n_tiles = cdiv(p.n, kShape[p.tile_x].bn);
      w.steps = cdiv(items, 64), w.splits = p.splits;
      w.sums = s.sums, w.sums_pitch = up(p.d, 8), w.first = v0 == 0;
      launch_product(ctx, fmt, p.tile_x, false, 0, w);
    }
    AS_HIP(ctx, hipGetLastError());
  }
  if (p.want_x) {
    join(s.sums, p.splits, p.n, true, Ox.p, gx_stride);
    AS_HIP(ctx, hipGetLastError());
  }
  AS_TRY(Ox.finish(ctx));
  AS_TRY(Ow.finish(ctx));
  AS_TRY(Ob.finish(ctx));
  return finish_call(ctx);
}

}  // namespace

extern "C" {

uint64_t as_cross_entropy_workspace(uint64_t n, uint64_t n_items, uint64_t dim, int dtype, int backward) {
  if (n == 0 || n_items == 0 || dim == 0 || n >= (1ull << 31) || n_items >= (1ull << 31) || dim > 65536 || !dtype_is_training(dtype)) return 0;
  Plan p = make_plan((uint32_t)n, (uint32_t)n_items, (uint32_t)dim, dtype);
  // (a stride of dim + 1: room for the images whether or not the matrices can be taken as they are)
  auto source = [&](uint64_t rows) { return Source{nullptr, (size_t)dim + 1, (uint32_t)rows, p.d, dtype, p.pitch}; };
  if (backward) {
    plan_backward(p, true, true, true);
    BackwardScratch s{};
    return backward_layout(p, source(n), source(n_items), nullptr, s);
  }
  // whichever form the alignment leads to
  uint64_t most = 0;
  for (bool direct : {false, true}) {
    p = make_plan((uint32_t)n, (uint32_t)n_items, (uint32_t)dim, dtype);
    plan_forward(p, direct);
    ForwardScratch s{};
    most = std::max(most, forward_layout(p, source(n), source(n_items), nullptr, s));
  }
  return most;
}

int as_cross_entropy(as_ctx *ctx, const void *x, uint64_t n, uint64_t x_stride, const void *table, uint64_t n_items, uint64_t table_stride, uint64_t dim,
                     int dtype, const float *bias, const int64_t *targets, int64_t ignore_index, double scale, float *losses, float *lse, void *workspace,
                     uint64_t workspace_bytes) {
  DeviceScope keep;
  return guarded(ctx, [&] {
    return forward_call(ctx, LossCall{n, n_items, dim, x_stride, table_stride, dtype, (float)scale}, x, table, bias, targets, ignore_index, losses, lse, workspace,
                        workspace_bytes);
  });
}

int as_cross_entropy_backward(as_ctx *ctx, const void *x, uint64_t n, uint64_t x_stride, const void *table, uint64_t n_items, uint64_t table_stride,
                              uint64_t dim, int dtype, const float *bias, const int64_t *targets, int64_t ignore_index, double scale, const float *lse,
                              const float *grad_losses, const float *grad_lse, void *grad_x, uint64_t grad_x_stride, void *grad_table,
                              uint64_t grad_table_stride, float *grad_bias, void *workspace, uint64_t workspace_bytes) {
  DeviceScope keep;
  return guarded(ctx, [&] {
    return backward_call(ctx, LossCall{n, n_items, dim, x_stride, table_stride, dtype, (float)scale}, x, table, bias, targets, ignore_index, lse, grad_losses, grad_lse,
                         grad_x, grad_x_stride, grad_table, grad_table_stride, grad_bias, workspace, workspace_bytes);
  });
}

}  // extern "C"
