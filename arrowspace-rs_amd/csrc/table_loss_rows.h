// table_loss_rows.h -- the gradients of the softmax cross entropy (table_loss.hip) for short rows: the gradient of the logits never
// leaves the registers.
//
// out_r = sum_k g(r, k) y_k with the logits l(r, k) = <r, y_k>: the rows r are the batch and the k the items for dX, the other way
// round for dW, so ONE kernel does both.  A wave keeps 16 RT rows r as operands and their whole output (RT x d accumulators) in
// registers and walks the k side in stages of 64 rows, which two products use:
//   logits     A = 16 rows k of the stage, B = the rows r: a lane ends up with 8 consecutive k of ONE row r (nt_product.h's interleaving)
//   gradient   of those 8 logits in f32, rounded to 16 bits: exactly the operand (row r, 8 consecutive k a lane group) of
//   output     A = the SAME stage read transposed (ds_read_b64_tr_b16: 4 rows k of a column a lane), B = the gradients.
// Against the form over G in memory this saves writing and reading 2 x 2 bytes a logit twice, for 2 d flops more a logit: a million
// items of 128 values and 1 024 rows (bf16), backward 2.8 ms through G, 1.0 ms here.  d is bounded by the registers (d <= 256, f32 128).
#pragma once

#include "nt_product.h"

namespace asx {

constexpr float kLog2e = 1.44269504088896340736f;
// the power of two a matrix with this largest magnitude is multiplied by (0 or not a number: 1)
__device__ __forceinline__ float plane_scale(unsigned int top_bits) {
  const int e = (int)(top_bits >> 23);
  if (e == 0 || e >= 255) return 1.f;
  const int s = min(max(14 - (e - 127), -100), 100);
  return __uint_as_float((unsigned int)(127 + s) << 23);
}
// Workgroups are dealt to the 8 dies in turn; consecutive pieces of work should share a die's cache, so die d takes the d-th eighth.
__device__ __forceinline__ uint32_t die_order(uint32_t b, uint32_t total) {
  const uint32_t die = b & 7, at = b >> 3, each = total >> 3, rest = total & 7;
  return die * each + nt_min(die, rest) + at;
}

// quad-wide exchange: the value of lane ^ 1 / lane ^ 2
__device__ __forceinline__ uint32_t quad_xor1(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true); }
__device__ __forceinline__ uint32_t quad_xor2(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true); }
__device__ __forceinline__ float add16(float v) {  // sum over the 16 lanes of a row of lanes, in a fixed order
  v += __uint_as_float(quad_xor1(__float_as_uint(v)));
  v += __uint_as_float(quad_xor2(__float_as_uint(v)));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));
  return v;
}

template <int FMT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  if constexpr (FMT == AS_BF16) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const bf2 p = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, p);
  } else {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    const half2v p = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(uint32_t, p);
  }
}
__device__ __forceinline__ float low_part(float x) {  // what f16 leaves of x (nothing of an infinity)
  const float hi = (float)(_Float16)x;
  return __builtin_isfinite(hi) ? x - hi : 0.f;
}


struct LossRowsArgs {
  const char *r, *k;              // the two sides' rows in 16 bits, whole 64 KD / 2 columns (zeros behind d)
  size_t r_ld, k_ld;              // bytes
  size_t r_plane, k_plane;        // bytes to the low plane (f32)
  uint32_t nr, nk, d;
  uint32_t r_blocks, splits;      // blocks of rows r; parts of the k side (sums: one buffer each)
  float scale;
  const unsigned int *r_top, *k_top;  // f32: bits of the largest magnitude of the two matrices
  // by row of the batch, filled to whole 64s (probability 0, no target)
  const float *lse, *every, *one;
  const int *target;
  const float *bias;              // by item, or null
  const float *coef;              // {factor, 1 / factor} of g, or null
  float *sums;                    // r = batch: f32 [split][nr][sums_pitch]
  uint32_t sums_pitch;
  void *out;                      // r = items: rows of out_stride elements
  size_t out_stride;
  int aligned;
  float *grad_bias;               // r = items: sum over k of g, or null
};

// lanes' coefficients of the gradient by row of the batch
__global__ __launch_bounds__(256) void loss_rows_kernel(const float *lse, const float *gl, const float *ge, const int64_t *targets, int64_t ignore, uint32_t n,
                                                        uint32_t padded, uint32_t v, const float *coef, float *o_lse, float *o_every, float *o_one, int *o_target) {
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  if (t >= padded) return;
  float s = INFINITY, every = 0.f, one = 0.f;
  int at = -1;
  if (t < n && lse[t] != -INFINITY) {  // (-inf: the bias left no item, no gradient)
    const float f = coef ? coef[0] : 1.f;
    const int64_t y = targets[t];
    if (y != ignore && y >= 0 && y < (int64_t)v) {
      at = (int)y;
      one = gl[t] * f;
    }
    s = lse[t];
    every = one + (ge ? ge[t] * f : 0.f);
  }
  o_lse[t] = s, o_every[t] = every, o_one[t] = one, o_target[t] = at;
}

template <int OFF>
__device__ __forceinline__ void lr_read4(u32x4 (&x)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%8\n\tds_read_b128 %1, %5 offset:%8\n\tds_read_b128 %2, %6 offset:%8\n\tds_read_b128 %3, %7 offset:%8\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(OFF)
      : "memory");
}
template <int OFF>
__device__ __forceinline__ void lr_read2(u32x4 &x, u32x4 &y, uint32_t a0, uint32_t a1) {
  asm volatile("ds_read_b128 %0, %2 offset:%4\n\tds_read_b128 %1, %3 offset:%4\n\ts_waitcnt lgkmcnt(0)"
               : "=&v"(x), "=&v"(y)
               : "v"(a0), "v"(a1), "n"(OFF)
               : "memory");
}
// two tiles (columns 4 h .. of each eight) of 4 + 4 rows, transposed: HALF bytes from rows 0 .. 3 to rows 4 .. 7
template <int HALF>
__device__ __forceinline__ void lr_transposed2(u32x4 &x, u32x4 &y, uint32_t a) {
  u32x2 x0, x1, y0, y1;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%5\n\tds_read_b64_tr_b16 %2, %4 offset:8\n\tds_read_b64_tr_b16 %3, %4 offset:%6\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x0), "=&v"(x1), "=&v"(y0), "=&v"(y1)
      : "v"(a), "n"(HALF), "n"(HALF + 8)
      : "memory");
  x = u32x4{x0[0], x0[1], x1[0], x1[1]};
  y = u32x4{y0[0], y0[1], y1[0], y1[1]};
}

// ---- forward for short rows -----------------------------------------------------------------------------------------------------------------
// The same walk with only the statistics behind it: rows in registers, items in stages of 64, a running maximum and sum of exponentials
// per lane and row.  For 128 values the matrix pipe needs 16 cycles for 64 logits and the exponentials' path (maximum, multiply-add,
// exp, add) some 26, so what is saved counts: the maximum that the exponentials are taken against moves only when it is exceeded
// by 2^20, once per walk in practice, and the rescaling with it.
struct LossSumsArgs {
  const char *r, *k;
  size_t r_ld, k_ld, r_plane, k_plane;
  uint32_t nr, nk, r_blocks, splits;
  float scale;
  const unsigned int *r_top, *k_top;
  const float *bias;
  float2 *part;  // [split][nr] (maximum, sum of exponentials against it)
};
template <int FMT, int P, int RT, int KD, bool GENERAL>
__global__ __launch_bounds__(256, 2) void loss_rows_sums_kernel(LossSumsArgs a) {
  constexpr uint32_t kRow = KD * 64, kPlane = 64 * kRow, kExtra = GENERAL ? 256 : 0, kStage = P * kPlane + kExtra;
  __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
  const uint32_t lds = (uint32_t)(size_t)(nt_lds *)smem;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  const uint32_t rb = work % a.r_blocks, split = work / a.r_blocks;
  const uint32_t r0 = (rb * 4 + wave) * (16 * RT);
  const uint32_t stages = (a.nk + 63) / 64;
  const uint32_t s_lo = (uint32_t)((uint64_t)stages * split / a.splits), s_hi = (uint32_t)((uint64_t)stages * (split + 1) / a.splits);
  const float nat = a.scale * (P == 2 ? 1.f / plane_scale(*a.r_top) / plane_scale(*a.k_top) : 1.f);
  const float unit = GENERAL ? kLog2e : nat * kLog2e, slack = fminf(20.f / unit, 1e30f);
  auto swz = [](uint32_t row) { const uint32_t key = (row & 3) | ((row >> 1) & 4); return KD >= 4 ? key << 1 : key; };
  auto fetch = [&](int buf, uint32_t s) {
    char *dst = smem + buf * kStage;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int t = 0; t < KD; ++t) {
        const uint32_t idx = t * 256 + threadIdx.x, row = idx / (KD * 4), slot = idx % (KD * 4);
        const uint32_t k = nt_min(s * 64 + row, a.nk - 1);
        __builtin_amdgcn_global_load_lds((nt_gbl *)(a.k + (size_t)k * a.k_ld + p * a.k_plane + ((slot ^ swz(row)) << 4)),
                                         (nt_lds *)(dst + p * kPlane + (t * 256 + wave * 64) * 16), 16, 0, 0);
      }
    if constexpr (GENERAL) {
      if (wave == 0 && a.bias)
        __builtin_amdgcn_global_load_lds((nt_gbl *)(a.bias + nt_min(s * 64 + lane, a.nk - 1)), (nt_lds *)(dst + P * kPlane), 4, 0, 0);
    }
  };
  if (s_lo < s_hi) fetch(0, s_lo);
  u32x4 R[P][RT][KD];
  float ref[RT], base[RT], sum[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const uint32_t row = nt_min(r0 + j * 16 + col, a.nr - 1);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int s = 0; s < KD; ++s) R[p][j][s] = *(const u32x4 *)(a.r + (size_t)row * a.r_ld + p * a.r_plane + s * 64 + q * 16);
    ref[j] = -INFINITY;
    base[j] = sum[j] = 0.f;
  }
  const uint32_t frow = ((col >> 2) << 3) + (col & 3), fa = frow * kRow + ((q ^ swz(frow)) << 4);
  const bool here = r0 < a.nr;  // (a wave without rows only brings its part of the stages)
  int buf = 0;
  for (uint32_t s = s_lo; s < s_hi; ++s, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < s_hi) fetch(buf ^ 1, s + 1);
    if (!here) continue;
#pragma unroll 1
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t k0 = s * 64 + h * 32;
      f32x4 z[2][RT];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < RT; ++j) z[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const uint32_t at = lds + buf * kStage + h * 32 * kRow + fa;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int s4 = 0; s4 < KD; s4 += 4) {
            u32x4 A[4];
            const uint32_t ap = at + p * kPlane;
            if constexpr (KD == 2) i == 0 ? lr_read2<0>(A[0], A[1], ap, ap ^ 64) : lr_read2<4 * kRow>(A[0], A[1], ap, ap ^ 64);
            else i == 0 ? lr_read4<0>(A, ap ^ (s4 << 6), ap ^ ((s4 + 1) << 6), ap ^ ((s4 + 2) << 6), ap ^ ((s4 + 3) << 6))
                        : lr_read4<4 * kRow>(A, ap ^ (s4 << 6), ap ^ ((s4 + 1) << 6), ap ^ ((s4 + 2) << 6), ap ^ ((s4 + 3) << 6));
#pragma unroll
            for (int t = 0; t < (KD < 4 ? KD : 4); ++t)
#pragma unroll
              for (int j = 0; j < RT; ++j) {
                z[i][j] = nt_mfma<FMT>(A[t], R[0][j][s4 + t], z[i][j]);
                if (P == 2 && p == 0) z[i][j] = nt_mfma<FMT>(A[t], R[P - 1][j][s4 + t], z[i][j]);
              }
          }
        if constexpr (GENERAL) {
          f32x4 kb = {0.f, 0.f, 0.f, 0.f};
          if (a.bias)
            asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(kb) : "v"(lds + buf * kStage + P * kPlane + h * 128 + q * 32 + i * 16) : "memory");
#pragma unroll
          for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[i][j][e] = fmaf(z[i][j][e], nat, kb[e]);
        }
        if (k0 + 32 > a.nk) {  // items behind the last
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + q * 8 + i * 4 + e >= a.nk)
#pragma unroll
              for (int j = 0; j < RT; ++j) z[i][j][e] = -INFINITY;
        }
      }
      float top[RT];
      bool over = false;
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        top[j] = fmaxf(fmaxf(fmaxf(z[0][j][0], z[0][j][1]), fmaxf(z[0][j][2], z[0][j][3])), fmaxf(fmaxf(z[1][j][0], z[1][j][1]), fmaxf(z[1][j][2], z[1][j][3])));
        over |= top[j] > ref[j] + slack;
      }
      if (__any(over)) {
#pragma unroll
        for (int j = 0; j < RT; ++j)
          if (top[j] > ref[j]) {
            const float was = ref[j];
            ref[j] = top[j];
            sum[j] *= __builtin_amdgcn_exp2f((was - top[j]) * unit);  // (nothing yet: -inf, 0)
            base[j] = GENERAL ? top[j] : -top[j] * unit;
          }
      }
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        auto power = [&](float x) { return __builtin_amdgcn_exp2f(GENERAL ? (x - base[j]) * unit : fmaf(x, unit, base[j])); };
        float s0 = power(z[0][j][0]) + power(z[0][j][1]), s1 = power(z[0][j][2]) + power(z[0][j][3]);
        s0 += power(z[1][j][0]) + power(z[1][j][1]);
        s1 += power(z[1][j][2]) + power(z[1][j][3]);
        sum[j] += s0 + s1;
      }
    }
  }
  if (!here) return;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    float m = GENERAL ? ref[j] : ref[j] == -INFINITY ? -INFINITY : ref[j] * nat, s = sum[j];
#pragma unroll
    for (int x = 16; x < 64; x <<= 1) {
      const float mo = __shfl_xor(m, x), so = __shfl_xor(s, x);
      const float mm = fmaxf(m, mo), b = mm == -INFINITY ? 0.f : mm;
      s = s * __builtin_amdgcn_exp2f((m - b) * kLog2e) + so * __builtin_amdgcn_exp2f((mo - b) * kLog2e);
      m = mm;
    }
    const uint32_t row = r0 + j * 16 + col;
    if (q == 0 && row < a.nr) a.part[(size_t)split * a.nr + row] = float2{m, s};
  }
}

// FMT the operands' type; P planes; RT tiles of 16 rows r a wave; KD steps of 32 columns; ITEMS: the rows r are items (dW), else the
// batch (dX); OUT: type of dW
template <int FMT, int P, int RT, int KD, bool ITEMS, bool BIAS, int OUT>
__global__ __launch_bounds__(256, 2) void loss_rows_grad_kernel(LossRowsArgs a) {
  constexpr uint32_t kRow = KD * 64, kPlane = 64 * kRow, kExtra = 1024, kStage = P * kPlane + kExtra;
  constexpr bool FAST = !BIAS && P == 1;  // 16-bit gradients: the exponent in one multiply-add (its constants are rounded: 2e-6 of the probability)
  __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
  const uint32_t lds = (uint32_t)(size_t)(nt_lds *)smem;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  const uint32_t rb = work % a.r_blocks, split = work / a.r_blocks;
  const uint32_t r0 = (rb * 4 + wave) * (16 * RT);
  const uint32_t stages = (a.nk + 63) / 64;
  const uint32_t s_lo = (uint32_t)((uint64_t)stages * split / a.splits), s_hi = (uint32_t)((uint64_t)stages * (split + 1) / a.splits);
  const float nat = a.scale * (P == 2 ? 1.f / plane_scale(*a.r_top) / plane_scale(*a.k_top) : 1.f);
  const float c = FAST ? nat * kLog2e : nat;
  auto swz = [](uint32_t row) { const uint32_t key = (row & 3) | ((row >> 1) & 4); return KD >= 4 ? key << 1 : key; };
  auto fetch = [&](int buf, uint32_t s) {
    char *dst = smem + buf * kStage;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int t = 0; t < KD; ++t) {
        const uint32_t idx = t * 256 + threadIdx.x, row = idx / (KD * 4), slot = idx % (KD * 4);
        const uint32_t k = nt_min(s * 64 + row, a.nk - 1);
        __builtin_amdgcn_global_load_lds((nt_gbl *)(a.k + (size_t)k * a.k_ld + p * a.k_plane + ((slot ^ swz(row)) << 4)),
                                         (nt_lds *)(dst + p * kPlane + (t * 256 + wave * 64) * 16), 16, 0, 0);
      }
    if constexpr (ITEMS) {  // by row of the batch: the waves bring one array each
      const char *src = wave == 0 ? (const char *)a.lse : wave == 1 ? (const char *)a.every : wave == 2 ? (const char *)a.one : (const char *)a.target;
      __builtin_amdgcn_global_load_lds((nt_gbl *)(src + ((size_t)s * 64 + lane) * 4), (nt_lds *)(dst + P * kPlane + wave * 256), 4, 0, 0);
    } else if constexpr (BIAS) {
      if (wave == 0)
        __builtin_amdgcn_global_load_lds((nt_gbl *)(a.bias + nt_min(s * 64 + lane, a.nk - 1)), (nt_lds *)(dst + P * kPlane), 4, 0, 0);
    }
  };
  if (s_lo < s_hi) fetch(0, s_lo);
  // this wave's rows
  u32x4 R[P][RT][KD];
  float lse[RT], every[RT], one[RT], rbias[RT], bsum[RT];
  int hit[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const uint32_t row = nt_min(r0 + j * 16 + col, a.nr - 1);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int s = 0; s < KD; ++s) R[p][j][s] = *(const u32x4 *)(a.r + (size_t)row * a.r_ld + p * a.r_plane + s * 64 + q * 16);
    lse[j] = every[j] = one[j] = rbias[j] = bsum[j] = 0.f;
    hit[j] = -1;
    if constexpr (ITEMS) {
      if (BIAS) rbias[j] = a.bias[row];
    } else {
      lse[j] = FAST ? a.lse[row] * kLog2e : a.lse[row];
      every[j] = a.every[row];
      one[j] = a.one[row];
      hit[j] = a.target[row];
    }
  }
  f32x4 out[2 * KD][RT];
#pragma unroll
  for (int t = 0; t < 2 * KD; ++t)
#pragma unroll
    for (int j = 0; j < RT; ++j) out[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // addresses within a stage: fragment rows of the logits (k = 8 (row / 4) + 4 i + row % 4), rows of the transposed reads (8 q + ...)
  const uint32_t frow = ((col >> 2) << 3) + (col & 3), trow = (q << 3) + ((lane >> 2) & 3);
  const uint32_t fa = frow * kRow + ((q ^ swz(frow)) << 4), ta = trow * kRow + (((lane & 3) ^ swz(trow)) << 4);
  int buf = 0;
  for (uint32_t s = s_lo; s < s_hi; ++s, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < s_hi) fetch(buf ^ 1, s + 1);
    const uint32_t base = lds + buf * kStage;
#pragma unroll 1
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t k0 = s * 64 + h * 32, extra = base + P * kPlane + h * 128;
      uint32_t G[P][RT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 z[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) z[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const uint32_t at = base + h * 32 * kRow + fa;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int s4 = 0; s4 < KD; s4 += 4) {
            u32x4 A[4];
            const uint32_t ap = at + p * kPlane;
            if constexpr (KD == 2) i == 0 ? lr_read2<0>(A[0], A[1], ap, ap ^ 64) : lr_read2<4 * kRow>(A[0], A[1], ap, ap ^ 64);
            else i == 0 ? lr_read4<0>(A, ap ^ (s4 << 6), ap ^ ((s4 + 1) << 6), ap ^ ((s4 + 2) << 6), ap ^ ((s4 + 3) << 6))
                        : lr_read4<4 * kRow>(A, ap ^ (s4 << 6), ap ^ ((s4 + 1) << 6), ap ^ ((s4 + 2) << 6), ap ^ ((s4 + 3) << 6));
#pragma unroll
            for (int t = 0; t < (KD < 4 ? KD : 4); ++t)
#pragma unroll
              for (int j = 0; j < RT; ++j) {
                z[j] = nt_mfma<FMT>(A[t], R[0][j][s4 + t], z[j]);
                if (P == 2 && p == 0) z[j] = nt_mfma<FMT>(A[t], R[P - 1][j][s4 + t], z[j]);
              }
          }
        // the gradients of four logits a row
        u32x4 kl, ke;
        f32x4 kb = {0.f, 0.f, 0.f, 0.f};
        if constexpr (ITEMS) {
          lr_read2<0>(kl, ke, extra + q * 32 + i * 16, extra + 256 + q * 32 + i * 16);
        } else if constexpr (BIAS) {
          asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(kb) : "v"(extra + q * 32 + i * 16) : "memory");
        }
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          f32x4 g;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float l = ITEMS ? __uint_as_float(kl[e]) : lse[j], w = ITEMS ? __uint_as_float(ke[e]) : every[j];
            float x;
            if constexpr (FAST) x = fmaf(z[j][e], c, ITEMS ? -l * kLog2e : -l);
            else if constexpr (BIAS) x = (fmaf(z[j][e], c, ITEMS ? rbias[j] : kb[e]) - l) * kLog2e;
            else x = fmaf(z[j][e], c, -l) * kLog2e;
            g[e] = w * __builtin_amdgcn_exp2f(x);
          }
          z[j] = g;
        }
        if (!ITEMS && k0 + 32 > a.nk) {  // items behind the last
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + q * 8 + i * 4 + e >= a.nk)
#pragma unroll
              for (int j = 0; j < RT; ++j) z[j][e] = 0.f;
        }
        // targets: rare
        if constexpr (ITEMS) {
          int tg;
          asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(tg) : "v"(extra + 768 + (lane & 31) * 4) : "memory");
          if (__any((uint32_t)tg - r0 < 16u * RT)) {
            u32x4 kt, ko;
            lr_read2<0>(kt, ko, extra + 768 + q * 32 + i * 16, extra + 512 + q * 32 + i * 16);
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (kt[e] == r0 + j * 16 + col) z[j][e] -= __uint_as_float(ko[e]);
          }
        } else {
          bool any = false;
#pragma unroll
          for (int j = 0; j < RT; ++j) any |= (uint32_t)hit[j] - k0 < 32u;
          if (__any(any)) {
#pragma unroll
            for (int j = 0; j < RT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if ((uint32_t)hit[j] == k0 + q * 8 + i * 4 + e) z[j][e] -= one[j];
          }
        }
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          if constexpr (ITEMS && BIAS) bsum[j] += (z[j][0] + z[j][1]) + (z[j][2] + z[j][3]);
          G[0][j][2 * i] = pack2<FMT>(z[j][0], z[j][1]);
          G[0][j][2 * i + 1] = pack2<FMT>(z[j][2], z[j][3]);
          if constexpr (P == 2) {
            G[1][j][2 * i] = pack2<FMT>(low_part(z[j][0]), low_part(z[j][1]));
            G[1][j][2 * i + 1] = pack2<FMT>(low_part(z[j][2]), low_part(z[j][3]));
          }
        }
      }
      const uint32_t at = base + h * 32 * kRow + ta;
#pragma unroll
      for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          u32x4 y0, y1;
          lr_transposed2<4 * kRow>(y0, y1, (at + p * kPlane) ^ (t << 6));
#pragma unroll
          for (int j = 0; j < RT; ++j) {
            const u32x4 g0 = u32x4{G[0][j][0], G[0][j][1], G[0][j][2], G[0][j][3]};
            out[2 * t][j] = nt_mfma<FMT>(y0, g0, out[2 * t][j]);
            out[2 * t + 1][j] = nt_mfma<FMT>(y1, g0, out[2 * t + 1][j]);
            if (P == 2 && p == 0) {
              const u32x4 g1 = u32x4{G[P - 1][j][0], G[P - 1][j][1], G[P - 1][j][2], G[P - 1][j][3]};
              out[2 * t][j] = nt_mfma<FMT>(y0, g1, out[2 * t][j]);
              out[2 * t + 1][j] = nt_mfma<FMT>(y1, g1, out[2 * t + 1][j]);
            }
          }
        }
    }
  }
  const float f = ITEMS ? a.scale * (a.coef ? a.coef[1] : 1.f) * (P == 2 ? 1.f / plane_scale(*a.k_top) : 1.f) : 1.f;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const uint32_t row = r0 + j * 16 + col;
    if constexpr (ITEMS && BIAS) {
      float b = bsum[j];
      b += __shfl_xor(b, 16);
      b += __shfl_xor(b, 32);
      if (a.grad_bias && q == 0 && row < a.nr) a.grad_bias[row] = b * (a.coef ? a.coef[1] : 1.f);
    }
    if (row >= a.nr) continue;
#pragma unroll
    for (int t = 0; t < KD; ++t) {
      const uint32_t m = t * 32 + q * 8;
      if (m >= a.d) continue;
      const f32x4 u = out[2 * t][j] * f, v = out[2 * t + 1][j] * f;
      if constexpr (!ITEMS) {
        f32x4 *o = (f32x4 *)(a.sums + ((size_t)split * a.nr + row) * a.sums_pitch + m);
        o[0] = u, o[1] = v;
      } else if (a.out == nullptr) {
        continue;  // (the bias' gradient alone)
      } else if (a.aligned && m + 8 <= a.d) {
        if constexpr (OUT == AS_F32) {
          f32x4 *o = (f32x4 *)((float *)a.out + (size_t)row * a.out_stride + m);
          o[0] = u, o[1] = v;
        } else {
          *(u32x4 *)((unsigned short *)a.out + (size_t)row * a.out_stride + m) =
              u32x4{pack2<OUT>(u[0], u[1]), pack2<OUT>(u[2], u[3]), pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3])};
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (m + e < a.d) store_from_f32<OUT>(a.out, (size_t)row * a.out_stride + m + e, e < 4 ? u[e & 3] : v[e & 3]);
      }
    }
  }
}

}  // namespace asx
