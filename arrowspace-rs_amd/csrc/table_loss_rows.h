// table_loss_rows.h -- the gradients of the softmax cross entropy (table_loss.hip) for short rows: the gradient of the logits never
// leaves the registers.
//
// out_r = sum_k g(r, k) y_k with the logits l(r, k) = <r, y_k>: the rows r are the batch and the k the items for dX, the other way
// round for dW, so ONE kernel does both.  A wave keeps 16 RT rows r as operands and their whole output (RT x d accumulators) in
// registers and walks the k side in stages of 64 rows, which two products use:
//   logits     A = 16 rows k of the stage, B = the rows r: a lane ends up with 8 consecutive k of ONE row r (nt_product.h's interleaving)
//   gradient   of those 8 logits in f32, rounded to 16 bits: exactly the operand (row r, 8 consecutive k a lane group) of
//   output     A = the SAME stage read transposed (ds_read_b64_tr_b16: 4 rows k of a column a lane), B = the gradients.
// Against the form over G in memory this saves writing and reading 2 bytes a logit, for 2 d flops more a logit: forward and backward of a
// million items of 128 values and 1 024 rows (bf16) 2.01 ms through G, 1.27 ms so (sums 282 us, dX 440, dW 490); the gradients of 512 f32 rows,
// 100 000 items of 128: 453 and 374 us.  What bounds it there: the matrix pipe and the exponentials' and packing's vector work of two waves a SIMD
// take turns (0.27 TFLOP of logits at 282 us: 950 TFLOP/s).  d is bounded by the registers (d <= 256, f32 128).
#pragma once

#include "nt_product.h"

namespace asx {

constexpr float kLog2e = 1.44269504088896340736f;
// Workgroups are dealt to the 8 dies in turn; consecutive pieces of work should share a die's cache, so die d takes the d-th eighth.
__device__ __forceinline__ uint32_t die_order(uint32_t b, uint32_t total) {
  const uint32_t die = b & 7, at = b >> 3, each = total >> 3, rest = total & 7;
  return die * each + nt_min(die, rest) + at;
}

// A grid of rows x cols pieces of work, walked in groups of four columns: the 32 workgroups a die runs at once are 8 x 4 pieces and
// read 12 sides, not 33 (8192^3 in bf16: 1 049 TFLOP/s in rows of one column, 1 280 so).
__device__ __forceinline__ void grid_order(uint32_t work, uint32_t rows, uint32_t cols, uint32_t *row, uint32_t *col) {
  const uint32_t group = work / (4 * rows), at = work - group * 4 * rows, width = nt_min(4, cols - group * 4);
  *row = at / width;
  *col = group * 4 + at % width;
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
__device__ __forceinline__ float rounded16(float x) {
  if constexpr (FMT == AS_BF16) return (float)(__bf16)x;
  else return (float)(_Float16)x;
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
// What the matrix pipe is fed, by the type of the matrices: their own 16-bit type, or f32 as the sum of three bf16 (24 bits, the exponents
// of f32: no scale that an outlier would set for everyone).  Of the nine products of two such sums the six of 2^-18 and more are made: planes
// (p, o) with p + o <= 2; what is left out is 2^-26 of a product.
constexpr int kF32Planes = 3;
constexpr int format_of(int dt) { return dt == AS_F16 ? AS_F16 : AS_BF16; }
constexpr int planes_of(int dt) { return dt == AS_F32 ? kF32Planes : 1; }
constexpr uint32_t pairs_of(uint32_t planes) { return planes == 1 ? 1 : 6; }
// P planes of a value.  Three: the first is the nearest finite bf16 (values next to the largest would round to infinity), so an infinity
// or NaN goes on into the second, where the third stops it.
template <int P>
__device__ __forceinline__ void split_planes(float x, float (&o)[P]) {
  o[0] = x;
  if constexpr (P == 3) {
    constexpr float largest = 0x1.fep127f;
    o[0] = __builtin_amdgcn_fmed3f(x, -largest, largest);
    const float r = x - (float)(__bf16)o[0];
    o[1] = r;
    o[2] = __builtin_isfinite(r) ? r - (float)(__bf16)r : 0.f;
  }
}
template <int FMT, int P>
__device__ __forceinline__ void pack_planes(float x, float y, uint32_t (&o)[P]) {
  float a[P], b[P];
  split_planes<P>(x, a);
  split_planes<P>(y, b);
#pragma unroll
  for (int p = 0; p < P; ++p) o[p] = pack2<FMT>(a[p], b[p]);
}

// eight consecutive values of a row, of any alignment
template <int DT>
__device__ __forceinline__ void store8(void *out, size_t at, f32x4 u, f32x4 v) {
  if constexpr (DT == AS_F32) {
    __builtin_memcpy((float *)out + at, &u, 16);
    __builtin_memcpy((float *)out + at + 4, &v, 16);
  } else {
    const u32x4 x = {pack2<DT>(u[0], u[1]), pack2<DT>(u[2], u[3]), pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    __builtin_memcpy((unsigned short *)out + at, &x, 16);
  }
}

// e^(logit - lse) from the exponent to the base 2: at most 1 -- of logits in the millions the lse and the logits of another kernel's order
// of sums are whole units apart.  (The bound is a modifier of the instruction.)
__device__ __forceinline__ float probability(float x) { return __builtin_amdgcn_fmed3f(__builtin_amdgcn_exp2f(x), 0.f, 1.f); }

struct LossRowsArgs {
  const char *r, *k;              // the two sides' rows as they are
  size_t r_ld, k_ld;              // bytes
  uint32_t nr, nk, d;
  uint32_t r_blocks, splits;      // blocks of rows r; parts of the k side (sums: one buffer each)
  float scale;
  // by row of the batch, filled to whole 64s (probability 0, no target)
  const float *lse, *every, *entry, *rest;
  const int *target;
  const float *bias;              // by item, or null
  const float *coef;              // {factor, 1 / factor} of g
  float *sums;                    // f32 [split][nr][sums_pitch] (r = items: where the batch is split), or null
  uint32_t sums_pitch;
  void *out;                      // r = items, not split: rows of out_stride elements, or null
  size_t out_stride;
  float *grad_bias;               // r = items: sum over k of g (split: [split][nr], in units of coef), or null
};

// The unit the gradient of the logits is rounded in: the largest |grad_losses|, so that the entry of a target, -grad_losses (1 - p), is
// a whole number of steps where all rows weigh the same (the mean of the losses: without this every such entry is off by the SAME
// part of 2^-9 in bf16, which no sum averages out).  f16: 2^14 of these units, entries down to 2^-28 of one keep all 11 bits.
// Where grad_lse outweighs grad_losses the largest of their sum.  Threads of a workgroup together; 16 bytes a row.
template <int THREADS>
__device__ __forceinline__ void unit_of_rows(const float *gl, const float *ge, const int64_t *targets, int64_t ignore, uint32_t n, int power, float *factor, float *unit) {
  __shared__ float s[2][THREADS / 64];
  float one = 0.f, both = 0.f;
  for (uint32_t t0 = threadIdx.x; t0 < n; t0 += 4 * THREADS) {
    float l[4], e[4];
    int64_t y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t t = t0 + k * THREADS, at = t < n ? t : threadIdx.x;
      y[k] = targets[at], l[k] = gl[at], e[k] = ge ? ge[at] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = y[k] == ignore ? 0.f : l[k], b = fabsf(x + e[k]), o = fabsf(x);
      if (o < INFINITY) one = fmaxf(one, o);
      if (b < INFINITY) both = fmaxf(both, b);
    }
  }
  for (int k = 1; k < 64; k <<= 1) {
    one = fmaxf(one, __shfl_xor(one, k));
    both = fmaxf(both, __shfl_xor(both, k));
  }
  if ((threadIdx.x & 63) == 0) s[0][threadIdx.x >> 6] = one, s[1][threadIdx.x >> 6] = both;
  __syncthreads();
  for (int w = 0; w < THREADS / 64; ++w) one = fmaxf(one, s[0][w]), both = fmaxf(both, s[1][w]);
  float m = both <= 2.f * one ? one : both;
  m = m > 0.f ? fmaxf(m, 0x1p-100f) : 1.f;  // (its inverse is finite behind the power too; f16 has its bits left for 2^-100 and less)
  *unit = m * __uint_as_float((unsigned int)(127 - power) << 23);
  *factor = 1.f / *unit;
}
__global__ __launch_bounds__(1024) void coef_scale_kernel(const float *gl, const float *ge, const int64_t *targets, int64_t ignore, uint32_t n, int power, float *out) {
  float factor, unit;
  unit_of_rows<1024>(gl, ge, targets, ignore, n, power, &factor, &unit);
  if (threadIdx.x == 0) out[0] = factor, out[1] = unit;
}

// By row of the batch, a wave each: the coefficient of its probabilities, and its entry at its target.  That entry is most of a row's
// gradient and often all of its item's, so it comes from a product in f64, the kernels put it in place of their own, and what 16 bits
// leave of it (`rest`, as much as the rounding of the result) is added in f32: to dX where its parts are joined, to dW behind the
// product.  coef: {factor, 1 / factor} of g, made here where FEW (up to kFewRows rows, every workgroup for itself).
constexpr uint32_t kFewRows = 1024;
struct LossRowInputs {
  const void *x, *table;
  size_t x_stride, table_stride;
  uint32_t d, n, padded, v;
  const float *bias, *lse, *gl, *ge;
  const int64_t *targets;
  int64_t ignore;
  float scale;
  int power;
  float *coef;
  float *o_lse, *o_every, *o_entry, *o_rest;
  int *o_target;
};
template <int DT, int FMT, bool FEW>
__global__ __launch_bounds__(256) void loss_rows_kernel(LossRowInputs a) {
  const uint32_t lane = threadIdx.x & 63;
  float f, unit;
  if constexpr (FEW) {
    unit_of_rows<256>(a.gl, a.ge, a.targets, a.ignore, a.n, a.power, &f, &unit);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.coef[0] = f, a.coef[1] = unit;
  } else {
    f = a.coef[0];
  }
  for (uint32_t t = blockIdx.x * 4 + (threadIdx.x >> 6); t < a.padded; t += gridDim.x * 4) {
    float s = INFINITY, every = 0.f, entry = 0.f;   // (behind the last row: probability 0)
    int at = -1;
    if (t < a.n && a.lse[t] != -INFINITY) {  // (-inf: the bias left no item, no gradient)
      const int64_t y = a.targets[t];
      float one = 0.f;
      s = a.lse[t];
      if (y != a.ignore && y >= 0 && y < (int64_t)a.v) {
        at = (int)y;
        one = a.gl[t] * f;
      }
      every = one + (a.ge ? a.ge[t] * f : 0.f);
      if (every == 0.f) s = INFINITY;                          // (nothing but the entry: probability 0, whatever a padded row holds)
      else if (!(s < INFINITY)) every = __builtin_nanf("");    // (no normaliser, no gradient: probability() gives no NaN)
      if (at >= 0) {
        double dot = 0.0;
#pragma unroll 4
        for (uint32_t k = lane; k < a.d; k += 64)
          dot += (double)load_as_f32<DT>(a.x, (size_t)t * a.x_stride + k) * (double)load_as_f32<DT>(a.table, (size_t)y * a.table_stride + k);
        for (int k = 1; k < 64; k <<= 1) dot += __shfl_xor(dot, k);
        const double z = (double)a.scale * dot + (a.bias ? (double)a.bias[y] : 0.0) - (double)a.lse[t];
        entry = (float)((double)every * (z > 0.0 ? 1.0 : exp(z)) - (double)one);
      }
    }
    if (lane == 0) {
      a.o_lse[t] = s, a.o_every[t] = every, a.o_entry[t] = entry, a.o_target[t] = at;
      a.o_rest[t] = DT == AS_F32 || !__builtin_isfinite(entry) ? 0.f : entry - rounded16<FMT>(entry);
    }
  }
}

// Stages go through registers into LDS and not by direct loads: behind a direct load in flight hipcc waits for it in front of every
// LDS read, and reads written by hand, each batch with its own wait, left the two waves of a SIMD waiting half their time (565 us for
// the dX of 1 024 rows against a million items of 128; 440 so).
typedef short short4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 lr_row(const char *smem, uint32_t at) { return *(const u32x4 *)(smem + at); }
// four rows of this lane's column, transposed
__device__ __forceinline__ u32x2 lr_column4(const char *smem, uint32_t at) {
  typedef __attribute__((address_space(3))) short4v lds_short4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(smem + at)));
}
// LDS written and read by one wave only: the hardware keeps its operations in order, the compiler is told to
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}
// rows 0 .. 3 and 4 .. 7 (`half` bytes on) of this lane's column, transposed
__device__ __forceinline__ u32x4 lr_column(const char *smem, uint32_t at, uint32_t half) {
  typedef __attribute__((address_space(3))) short4v lds_short4;
  const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(smem + at)));
  const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(smem + at + half)));
  return u32x4{x[0], x[1], y[0], y[1]};
}
// Eight consecutive values of a row, as the matrix holds them (columns behind the row's d: zeros) and as 16-bit operands.  RAW: rows of
// any alignment and length; else whole 16-byte pieces, f32 as images of its planes (`plane` bytes apart).
template <int DT, bool RAW>
struct LrPiece {
  u32x4 w[DT != AS_F32 ? 1 : RAW ? 2 : kF32Planes];
  __device__ __forceinline__ void load(const char *row, uint32_t column, uint32_t d, uint32_t plane) {
    if constexpr (!RAW) {
#pragma unroll
      for (int p = 0; p < planes_of(DT); ++p) w[p] = *(const u32x4 *)(row + p * plane + column * 2);
    } else {
      Piece8<DT> raw;
      raw.load(row, column, d);
      w[0] = raw.w[0];
      if constexpr (DT == AS_F32) w[1] = raw.w[1];
    }
  }
  template <int FMT, int P>
  __device__ __forceinline__ void planes(u32x4 (&o)[P]) const {
    if constexpr (P == 1) {
      o[0] = w[0];
    } else if constexpr (!RAW) {
#pragma unroll
      for (int p = 0; p < P; ++p) o[p] = w[p];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t pair[P];
        pack_planes<FMT, P>(__uint_as_float(w[e >> 1][2 * (e & 1)]), __uint_as_float(w[e >> 1][2 * (e & 1) + 1]), pair);
#pragma unroll
        for (int p = 0; p < P; ++p) o[p][e] = pair[p];
      }
    }
  }
};
// A stage of 64 rows of the k side, P planes of 64 KD bytes a row: 16-byte piece c of row r at place c ^ swizzle(r), so that a fragment
// read (8 rows) and a transposed read (4 rows) spread over the banks
template <int FMT, int P, int KD, int DT, bool RAW>
struct LrStage {
  static constexpr uint32_t kRow = KD * 64, kPlane = 64 * kRow;
  LrPiece<DT, RAW> piece[KD];
  __device__ __forceinline__ static uint32_t swizzle(uint32_t row) {
    const uint32_t key = (row & 3) | ((row >> 1) & 4);
    return KD >= 4 ? key << 1 : key;
  }
  __device__ __forceinline__ void load(const char *k, size_t ld, uint32_t d, uint32_t nk, uint32_t s) {
#pragma unroll
    for (int t = 0; t < KD; ++t) {
      const uint32_t idx = t * 256 + threadIdx.x, row = idx / (KD * 4), slot = idx % (KD * 4);
      piece[t].load(k + (size_t)nt_min(s * 64 + row, nk - 1) * ld, (slot ^ swizzle(row)) * 8, d, kRow);
    }
  }
  __device__ __forceinline__ void store(char *dst) const {
#pragma unroll
    for (int t = 0; t < KD; ++t) {
      u32x4 o[P];
      piece[t].template planes<FMT, P>(o);
#pragma unroll
      for (int p = 0; p < P; ++p) *(u32x4 *)(dst + p * kPlane + (t * 256 + threadIdx.x) * 16) = o[p];
    }
  }
};
// a wave's 16 RT rows as operands, from row r0 (rows behind the last: the last)
template <int FMT, int P, int RT, int KD, int DT, bool RAW>
__device__ __forceinline__ void lr_rows(u32x4 (&R)[P][RT][KD], const char *rows, size_t ld, uint32_t r0, uint32_t nr, uint32_t d) {
  const uint32_t lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const char *row = rows + (size_t)nt_min(r0 + j * 16 + col, nr - 1) * ld;
#pragma unroll
    for (int s = 0; s < KD; ++s) {
      LrPiece<DT, RAW> piece;
      piece.load(row, s * 32 + q * 8, d, KD * 64);
      u32x4 o[P];
      piece.template planes<FMT, P>(o);
#pragma unroll
      for (int p = 0; p < P; ++p) R[p][j][s] = o[p];
    }
  }
}

// ---- forward for short rows -----------------------------------------------------------------------------------------------------------------
// The same walk with only the statistics behind it: rows in registers, items in stages of 64, a running maximum and sum of exponentials
// per lane and row.  For 128 values the matrix pipe needs 16 cycles for 64 logits and the exponentials' path (maximum, multiply-add,
// exp, add) some 26, so what is saved counts: the maximum that the exponentials are taken against moves only when it is exceeded
// by 2^20, once per walk in practice, and the rescaling with it.
struct LossSumsArgs {
  const char *r, *k;              // the batch and the table as they are
  size_t r_ld, k_ld;              // bytes
  uint32_t nr, nk, d, r_blocks, splits;
  float scale;
  const float *bias;
  float2 *part;  // [split][nr] (maximum, sum of exponentials against it)
};
// Without a bias the exponent of a product x is fma(x, unit, base) with base = -(the largest) unit, rounded down: no term overflows, all of
// them carry 2^off, where off = fma(largest, unit, base) <= 0 is that rounding.  Logits behind 2^29 lie further apart than exp2 has range for
// there, so that the largest is all of the sum.
__device__ __forceinline__ float base_of(float largest, float unit) {
  const float base = -largest * unit;
  return fmaf(largest, unit, base) > 0.f ? base - fabsf(base) * 0x1p-23f : base;
}
// ... the sum against m = largest scale (rounded as well: what that leaves belongs to the sum, while it has range for it)
__device__ __forceinline__ float sum_against(float largest, float unit, float base, float scale, float m, float sum) {
  const float off = fmaf(largest, unit, base), rest = fmaf(largest, scale, -m) * kLog2e;
  return off < -64.f ? 1.f : sum * __builtin_amdgcn_exp2f((fabsf(rest) > 32.f ? 0.f : rest) - off);
}
// ... and what it is multiplied by when the base moves (nothing yet: 0)
__device__ __forceinline__ float rebased(float before, float base, float now) { return before == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(now - base); }
template <int DT, bool RAW, int RT, int KD, bool GENERAL, int WAVES>
__global__ __launch_bounds__(256, WAVES) void loss_rows_sums_kernel(LossSumsArgs a) {
  constexpr int FMT = format_of(DT), P = planes_of(DT);
  typedef LrStage<FMT, P, KD, DT, RAW> Stage;
  constexpr uint32_t kRow = Stage::kRow, kPlane = Stage::kPlane, kExtra = GENERAL ? 256 : 0, kStage = P * kPlane + kExtra;
  __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  const uint32_t rb = work % a.r_blocks, split = work / a.r_blocks;
  const uint32_t r0 = (rb * 4 + wave) * (16 * RT);
  const uint32_t stages = (a.nk + 63) / 64;
  const uint32_t s_lo = (uint32_t)((uint64_t)stages * split / a.splits), s_hi = (uint32_t)((uint64_t)stages * (split + 1) / a.splits);
  const float unit = GENERAL ? kLog2e : a.scale * kLog2e, slack = fminf(20.f / unit, 1e30f);
  Stage stage;
  float extra = 0.f;
  auto load = [&](uint32_t s) {
    stage.load(a.k, a.k_ld, a.d, a.nk, s);
    if (GENERAL && a.bias && threadIdx.x < 64) extra = a.bias[nt_min(s * 64 + threadIdx.x, a.nk - 1)];
  };
  auto store = [&](int buf) {
    stage.store(smem + buf * kStage);
    if (GENERAL && threadIdx.x < 64) *(float *)(smem + buf * kStage + P * kPlane + threadIdx.x * 4) = extra;
  };
  if (s_lo < s_hi) load(s_lo);
  u32x4 R[P][RT][KD];
  lr_rows<FMT, P, RT, KD, DT, RAW>(R, a.r, a.r_ld, r0, a.nr, a.d);
  float ref[RT], base[RT], sum[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    ref[j] = -INFINITY;
    base[j] = sum[j] = 0.f;
  }
  const uint32_t frow = ((col >> 2) << 3) + (col & 3), fa = frow * kRow + ((q ^ Stage::swizzle(frow)) << 4);
  const bool here = r0 < a.nr;  // (a wave without rows only brings its part of the stages)
  if (s_lo < s_hi) store(0);
  int buf = 0;
  for (uint32_t s = s_lo; s < s_hi; ++s, buf ^= 1) {
    __syncthreads();
    if (s + 1 < s_hi) load(s + 1);
    const char *here_in = smem + buf * kStage;
#pragma unroll 1
    for (uint32_t h = 0; h < 2 && here; ++h) {
      const uint32_t k0 = s * 64 + h * 32;
      f32x4 z[2][RT];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < RT; ++j) z[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const uint32_t at = h * 32 * kRow + fa + i * 4 * kRow;
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int t = 0; t < KD; ++t) {
            const u32x4 A = lr_row(here_in, p * kPlane + (at ^ (t << 6)));
#pragma unroll
            for (int o = P - 1 - p; o >= 0; --o)
#pragma unroll
              for (int j = 0; j < RT; ++j) z[i][j] = nt_mfma<FMT>(A, R[o][j][t], z[i][j]);
          }
        if constexpr (GENERAL) {
          const f32x4 kb = *(const f32x4 *)(here_in + P * kPlane + h * 128 + q * 32 + i * 16);
#pragma unroll
          for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[i][j][e] = fmaf(z[i][j][e], a.scale, kb[e]);
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
            const float to = GENERAL ? top[j] : base_of(top[j], unit);
            sum[j] *= GENERAL ? __builtin_amdgcn_exp2f((ref[j] - top[j]) * unit) : rebased(ref[j], base[j], to);  // (nothing yet: 0)
            ref[j] = top[j], base[j] = to;
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
    if (s + 1 < s_hi) store(buf ^ 1);
  }
  if (!here) return;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    float m = ref[j], s = sum[j];
    if (!GENERAL && m != -INFINITY) {
      m *= a.scale;
      s = sum_against(ref[j], unit, base[j], a.scale, m, s);
    }
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

// DT, RAW: the matrices (LrPiece); RT tiles of 16 rows r a wave; KD steps of 32 columns; ITEMS: the rows r are items (dW), else the
// batch (dX)
template <int DT, bool RAW, int RT, int KD, bool ITEMS, bool BIAS, int WAVES>
__global__ __launch_bounds__(256, WAVES) void loss_rows_grad_kernel(LossRowsArgs a) {
  constexpr int FMT = format_of(DT), P = planes_of(DT), OUT = DT;
  typedef LrStage<FMT, P, KD, DT, RAW> Stage;
  constexpr uint32_t kRow = Stage::kRow, kPlane = Stage::kPlane, kExtra = 1024, kStage = P * kPlane + kExtra;
  constexpr bool FAST = !BIAS && P == 1;  // 16-bit gradients: the exponent in one multiply-add (its constants are rounded: 2e-6 of the probability)
  __shared__ __attribute__((aligned(1024))) char smem[2 * kStage];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, q = lane >> 4, col = lane & 15;
  const uint32_t work = die_order(blockIdx.x, gridDim.x);
  const uint32_t rb = work % a.r_blocks, split = work / a.r_blocks;
  const uint32_t r0 = (rb * 4 + wave) * (16 * RT);
  const uint32_t stages = (a.nk + 63) / 64;
  const uint32_t s_lo = (uint32_t)((uint64_t)stages * split / a.splits), s_hi = (uint32_t)((uint64_t)stages * (split + 1) / a.splits);
  const float c = FAST ? a.scale * kLog2e : a.scale;
  constexpr uint32_t kList = 64;  // (the entries of further rows stay rounded, as all others are)
  __shared__ u32x2 list[ITEMS && P == 1 ? 4 : 1][kList];
  uint32_t list_len = 0;
  Stage stage;
  float extra = 0.f;
  // by row of the batch: the waves bring one array each; else the items' bias
  const float *by_k = ITEMS ? (wave == 0 ? a.lse : wave == 1 ? a.every : wave == 2 ? a.entry : (const float *)a.target) : a.bias;
  auto load = [&](uint32_t s) {
    stage.load(a.k, a.k_ld, a.d, a.nk, s);
    if (ITEMS) extra = by_k[s * 64 + lane];
    else if (BIAS && wave == 0) extra = by_k[nt_min(s * 64 + lane, a.nk - 1)];
  };
  auto store = [&](int buf) {
    stage.store(smem + buf * kStage);
    if (ITEMS || (BIAS && wave == 0)) *(float *)(smem + buf * kStage + P * kPlane + threadIdx.x * 4) = extra;
  };
  if (s_lo < s_hi) load(s_lo);
  // this wave's rows
  u32x4 R[P][RT][KD];
  lr_rows<FMT, P, RT, KD, DT, RAW>(R, a.r, a.r_ld, r0, a.nr, a.d);
  float lse[RT], every[RT], entry[RT], rbias[RT], bsum[RT];
  int hit[RT];
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const uint32_t row = nt_min(r0 + j * 16 + col, a.nr - 1);
    lse[j] = every[j] = entry[j] = rbias[j] = bsum[j] = 0.f;
    hit[j] = -1;
    if constexpr (ITEMS) {
      if (BIAS) rbias[j] = a.bias[row];
    } else {
      lse[j] = FAST ? a.lse[row] * kLog2e : a.lse[row];
      every[j] = a.every[row];
      entry[j] = a.entry[row];
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
  const uint32_t fa = frow * kRow + ((q ^ Stage::swizzle(frow)) << 4), ta = trow * kRow + (((lane & 3) ^ Stage::swizzle(trow)) << 4);
  if (s_lo < s_hi) store(0);
  int buf = 0;
  for (uint32_t s = s_lo; s < s_hi; ++s, buf ^= 1) {
    __syncthreads();
    if (s + 1 < s_hi) load(s + 1);
    const char *here_in = smem + buf * kStage;
#pragma unroll 1
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t k0 = s * 64 + h * 32, by = P * kPlane + h * 128;
      uint32_t G[P][RT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f32x4 z[RT];
#pragma unroll
        for (int j = 0; j < RT; ++j) z[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        // (the matrix work of one wave goes in front of the others' exponentials: 4 %)
        __builtin_amdgcn_s_setprio(1);
        const uint32_t at = h * 32 * kRow + fa + i * 4 * kRow;
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int t = 0; t < KD; ++t) {
            const u32x4 A = lr_row(here_in, p * kPlane + (at ^ (t << 6)));
#pragma unroll
            for (int o = P - 1 - p; o >= 0; --o)
#pragma unroll
              for (int j = 0; j < RT; ++j) z[j] = nt_mfma<FMT>(A, R[o][j][t], z[j]);
          }
        __builtin_amdgcn_s_setprio(0);
        // the gradients of four logits a row
        u32x4 kl = {}, ke = {};
        f32x4 kb = {0.f, 0.f, 0.f, 0.f};
        if constexpr (ITEMS) {
          kl = lr_row(here_in, by + q * 32 + i * 16);
          ke = lr_row(here_in, by + 256 + q * 32 + i * 16);
        } else if constexpr (BIAS) {
          kb = *(const f32x4 *)(here_in + by + q * 32 + i * 16);
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
            g[e] = w * probability(x);
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
        // targets: few of the steps hold one
        bool any = false;
        const uint32_t tg = ITEMS ? *(const uint32_t *)(here_in + by + 768 + (lane & 31) * 4) - r0 : 0u;
        if constexpr (ITEMS) {
          any = tg < 16u * RT;
        } else {
#pragma unroll
          for (int j = 0; j < RT; ++j) any |= (uint32_t)hit[j] - k0 < 32u;
        }
        if (__any(any)) {
          u32x4 kt = {}, kg = {};
          if constexpr (ITEMS) {
            kt = lr_row(here_in, by + 768 + q * 32 + i * 16);
            kg = lr_row(here_in, by + 512 + q * 32 + i * 16);
            if (P == 1 && i == 0) {  // the rows that meet this wave's items, in order, for the end
              const uint32_t met = (uint32_t)__ballot(any && lane < 32);
              const uint32_t place = list_len + __popc(met & ((1u << (lane & 31)) - 1));
              if (any && lane < 32 && place < kList) list[wave][place] = u32x2{k0 + lane, tg};
              list_len += __popc(met);
            }
          }
#pragma unroll
          for (int j = 0; j < RT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (ITEMS ? kt[e] == r0 + j * 16 + col : (uint32_t)hit[j] == k0 + q * 8 + i * 4 + e) z[j][e] = ITEMS ? __uint_as_float(kg[e]) : entry[j];
        }
#pragma unroll
        for (int j = 0; j < RT; ++j) {
          if constexpr (ITEMS && BIAS) bsum[j] += (z[j][0] + z[j][1]) + (z[j][2] + z[j][3]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t pair[P];
            pack_planes<FMT, P>(z[j][2 * h], z[j][2 * h + 1], pair);
#pragma unroll
            for (int p = 0; p < P; ++p) G[p][j][2 * i + h] = pair[p];
          }
        }
      }
      __builtin_amdgcn_s_setprio(1);
      const uint32_t at = h * 32 * kRow + ta;
#pragma unroll
      for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int p = P - 1; p >= 0; --p) {
          // columns 4 h .. 4 h + 3 of each eight: two tiles
          const u32x4 y0 = lr_column(here_in, p * kPlane + (at ^ (t << 6)), 4 * kRow), y1 = lr_column(here_in, p * kPlane + (at ^ (t << 6)) + 8, 4 * kRow);
#pragma unroll
          for (int o = P - 1 - p; o >= 0; --o)
#pragma unroll
            for (int j = 0; j < RT; ++j) {
              const u32x4 g = u32x4{G[o][j][0], G[o][j][1], G[o][j][2], G[o][j][3]};
              out[2 * t][j] = nt_mfma<FMT>(y0, g, out[2 * t][j]);
              out[2 * t + 1][j] = nt_mfma<FMT>(y1, g, out[2 * t + 1][j]);
            }
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (s + 1 < s_hi) store(buf ^ 1);
  }
  if constexpr (ITEMS && P == 1) {  // what 16 bits left of the entries at the targets
    list_len = nt_min(list_len, kList);
    // each column of lanes its own items' rows, all columns at once
    uint64_t mine = 0;
    for (uint32_t n = 0; n < list_len; ++n)
      if ((list[wave][n][1] & 15) == col) mine |= 1ull << n;
    while (mine) {
      const int n = __builtin_ctzll(mine);
      mine &= mine - 1;
      const uint32_t t = list[wave][n][0], at = list[wave][n][1];
      const float rest = a.rest[t];
#pragma unroll
      for (int s = 0; s < KD; ++s) {
        LrPiece<DT, RAW> piece;
        piece.load(a.k + (size_t)t * a.k_ld, s * 32 + q * 8, a.d, kRow);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned short u = (unsigned short)(piece.w[0][e >> 1] >> (16 * (e & 1)));
          y[e] = FMT == AS_BF16 ? bf16_to_f32(u) : (float)__builtin_bit_cast(_Float16, u);
        }
#pragma unroll
        for (uint32_t j = 0; j < RT; ++j)
          if (j == at >> 4) {
            out[2 * s][j] += f32x4{y[0], y[1], y[2], y[3]} * rest;
            out[2 * s + 1][j] += f32x4{y[4], y[5], y[6], y[7]} * rest;
          }
        if (s & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  const float f = ITEMS && !a.sums ? a.scale * a.coef[1] : 1.f;
#pragma unroll
  for (int j = 0; j < RT; ++j) {
    const uint32_t row = r0 + j * 16 + col;
    if constexpr (ITEMS && BIAS) {
      float b = bsum[j];
      b += __shfl_xor(b, 16);
      b += __shfl_xor(b, 32);
      if (a.grad_bias && q == 0 && row < a.nr) a.grad_bias[(size_t)split * a.nr + row] = a.splits > 1 ? b : b * a.coef[1];
    }
    if (row >= a.nr) continue;
#pragma unroll
    for (int t = 0; t < KD; ++t) {
      const uint32_t m = t * 32 + q * 8;
      if (m >= a.d) continue;
      const f32x4 u = out[2 * t][j] * f, v = out[2 * t + 1][j] * f;
      if (!ITEMS || a.sums) {
        f32x4 *o = (f32x4 *)(a.sums + ((size_t)split * a.nr + row) * a.sums_pitch + m);
        o[0] = u, o[1] = v;
      } else if (a.out == nullptr) {
        continue;  // (the bias' gradient alone)
      } else if (m + 8 <= a.d) {
        store8<OUT>(a.out, (size_t)row * a.out_stride + m, u, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (m + e < a.d) store_from_f32<OUT>(a.out, (size_t)row * a.out_stride + m + e, e < 4 ? u[e & 3] : v[e & 3]);
      }
    }
  }
}

}  // namespace asx
