// table4.hip -- a table of rows held in 4 bits with group scales, and its products with a few rows (the scores of single queries).
//
//   W_vk = s_{v, k / g} (q_vk - z_{v, k / g}),  q in 0 .. 15, z = 8 where the table has none        y_mv = sum_k x_mk W_vk
//
// What bounds it: d v / 2 bytes of codes (and 2 d v / g of 16-bit scales) for 2 m d v flops -- memory, up to some 64 rows.  So the
// codes are streamed once, unpacked in registers and fed to the matrix pipe whatever m is: 16 items x 16 rows x 32 k an instruction,
// rows that are not there cost nothing that is scarce.
// Unpacking.  A 32-bit word holds 8 codes, interleaved so that code k sits in the low and code k + 1 in the high half of a mask:
// (w & 0x000f000f) | 0x6400 is the f16 pair 1024 + q, (w & 0x00f000f0) | 0x6400 the pair 1024 + 16 q; one packed add or multiply-add
// takes 1024 + z off (exact: small integers), a shift by 8 brings the other four.  9 instructions for 8 values.
// Types.  Codes less zero points are integers, exact in f16; rows of f16 go as they are, bf16 after a power of two a row that brings its
// largest finite value to 2^14 .. 2^15 (8 bits fit, down to 2^-28 of that), f32 after the same as a sum of two f16 (22 bits).  Products
// of a group are summed in f32 by the matrix pipe, groups in f32 after their scale.
// Layout (made once, by the handle): tiles of 16 items x 128 k, 1 KB: lane l of a wave holds item l & 15 and, of each 32 k, the 8
// from 8 (l >> 4): its operand of four instructions in one 16-byte load.  Scales of a tile: item by item its 4 / 2 / 1 groups.
#include "table_common.h"

using namespace asx;

struct as_table4 {
  int device = 0;
  uint64_t v = 0, d = 0;
  uint32_t group = 0;
  int scale_dt = AS_F32;
  bool zeros = false;
  uint32_t v_tiles = 0, k_tiles = 0;
  unsigned int *codes = nullptr;   // v_tiles x k_tiles x 64 x 4
  void *scales = nullptr;          // v_tiles x k_tiles x 16 x (128 / group)
  unsigned char *z = nullptr;      // the same shape, or null
};

namespace {

constexpr uint32_t kTileItems = 16, kTileK = 128;

__device__ __forceinline__ float scale_to_f32(const void *p, int dt, size_t i) {
  return dt == AS_F32 ? ((const float *)p)[i] : dt == AS_BF16 ? bf16_to_f32(((const unsigned short *)p)[i]) : (float)((const _Float16 *)p)[i];
}

// place of code k (0 .. 7) in its word
__device__ __forceinline__ uint32_t code_shift(uint32_t k) { return ((k & 1) * 4 + (k >> 1)) * 4; }

// ---- making the handle ----------------------------------------------------------------------------------------------------------------
// A thread a word of the image.  Plain codes: row v is ceil(d / 2) bytes, column 2 j in the low half of byte j.
__global__ __launch_bounds__(256) void import_codes_kernel(const unsigned char *codes, uint64_t v, uint32_t d, uint32_t k_tiles, uint64_t words, unsigned int *out) {
  const uint64_t row_bytes = (d + 1) / 2;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (uint64_t)gridDim.x * 256) {
    const uint32_t j = i & 3, lane = (i >> 2) & 63;
    const uint64_t tile = i >> 8;
    const uint64_t item = tile / k_tiles * kTileItems + (lane & 15);
    const uint32_t k0 = (uint32_t)(tile % k_tiles) * kTileK + j * 32 + (lane >> 4) * 8;
    unsigned int w = 0;
    if (item < v)
      for (uint32_t k = 0; k < 8 && k0 + k < d; ++k) {
        const unsigned int b = codes[item * row_bytes + ((k0 + k) >> 1)];
        w |= (((k0 + k) & 1 ? b >> 4 : b) & 15u) << code_shift(k);
      }
    out[i] = w;
  }
}
__global__ __launch_bounds__(256) void export_codes_kernel(const unsigned int *image, uint64_t v, uint32_t d, uint32_t k_tiles, unsigned char *codes) {
  const uint64_t row_bytes = (d + 1) / 2, total = v * row_bytes;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint64_t item = i / row_bytes;
    unsigned int b = 0;
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t k = (uint32_t)(i % row_bytes) * 2 + h;
      if (k >= d) break;
      const uint32_t kk = k % kTileK, lane = (uint32_t)(item & 15) + 16 * ((kk & 31) >> 3);
      const unsigned int w = image[((item / kTileItems * k_tiles + k / kTileK) * 64 + lane) * 4 + (kk >> 5)];
      b |= ((w >> code_shift(kk & 7)) & 15u) << (4 * h);
    }
    codes[i] = (unsigned char)b;
  }
}
// scales (and zero points) between the plain form, v x groups, and the tiles; TO: into the tiles.  bad: a zero point above 15
template <class S, bool TO>
__global__ __launch_bounds__(256) void scales_kernel(S *plain, unsigned char *plain_z, uint64_t v, uint32_t groups, uint32_t per, uint32_t k_tiles, uint64_t slots,
                                                     S *tiles, unsigned char *tiles_z, unsigned int *bad) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < slots; i += (uint64_t)gridDim.x * 256) {
    const uint32_t g = i % per;
    const uint64_t r = i / per, item = r / 16 / k_tiles * kTileItems + (r & 15);
    const uint32_t group = (uint32_t)(r / 16 % k_tiles) * per + g;
    const bool there = item < v && group < groups;
    if (TO) {
      tiles[i] = there ? plain[item * groups + group] : S(0);
      if (tiles_z) {
        const unsigned char z = there ? plain_z[item * groups + group] : 8;
        if (z > 15) atomicOr(bad, 1u);
        tiles_z[i] = z & 15;
      }
    } else if (there) {
      plain[item * groups + group] = tiles[i];
      if (plain_z) plain_z[item * groups + group] = tiles_z ? tiles_z[i] : 8;
    }
  }
}
// Rows to codes: the scale of a group is its largest magnitude over 7, rounded to the scales' type first, so that the codes fit the
// scale that is kept; codes are rounded to even.  A wave a group of an item.  bad: 1 a value, 2 a scale that is not finite
template <int DT>
__global__ __launch_bounds__(256) void quantise_kernel(const void *rows, size_t stride, uint64_t v, uint32_t d, uint32_t group, uint32_t groups, int scale_dt,
                                                       unsigned char *codes, void *scales, unsigned int *bad) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t row_bytes = (d + 1) / 2, total = v * groups;
  for (uint64_t u = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < total; u += (uint64_t)gridDim.x * 4) {
    const uint64_t item = u / groups;
    const uint32_t g = (uint32_t)(u % groups), k = g * group + lane * 2;  // (a group has at most 128 columns: a byte a lane)
    const bool mine = lane * 2 < group;
    const float x = mine && k < d ? load_as_f32<DT>(rows, item * stride + k) : 0.f, y = mine && k + 1 < d ? load_as_f32<DT>(rows, item * stride + k + 1) : 0.f;
    float m = fmaxf(fabsf(x), fabsf(y));
    if (!(fabsf(x) < INFINITY) || !(fabsf(y) < INFINITY)) atomicOr(bad, 1u);
    for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
    float s = m / 7.f;
    if (scale_dt == AS_BF16) s = (float)(__bf16)s;
    else if (scale_dt == AS_F16) s = (float)(_Float16)s;
    if (!(s < INFINITY)) {
      if (lane == 0) atomicOr(bad, 2u);
      s = 0.f;
    }
    auto code = [&](float a) { return s > 0.f ? (unsigned int)(int)(fminf(fmaxf(rintf(a / s), -8.f), 7.f) + 8.f) : 8u; };
    if (mine && k < d) codes[item * row_bytes + k / 2] = (unsigned char)(code(x) | (k + 1 < d ? code(y) << 4 : 0u));
    if (lane == 0) {
      const size_t at = item * groups + g;
      if (scale_dt == AS_F32) ((float *)scales)[at] = s;
      else if (scale_dt == AS_BF16) ((__bf16 *)scales)[at] = (__bf16)s;
      else ((_Float16 *)scales)[at] = (_Float16)s;
    }
  }
}
__global__ void clear_word_kernel(unsigned int *w) { *w = 0u; }

// ---- the product --------------------------------------------------------------------------------------------------------------------------
struct ScoresArgs {
  const u32x4 *codes;
  const void *scales;
  const unsigned char *z;
  uint32_t v, d, v_tiles, k_tiles, units, split;  // units of kVT tiles; waves of a workgroup that share a unit's k
  const void *x;
  size_t x_stride;
  uint32_t m;
  void *out;
  size_t out_stride;
  // rows that do not fit the LDS: their operand image and factors, made by rows_image_kernel
  const u32x4 *image;
  const float *undo;
};

// the power of two that brings a largest magnitude to 2^14 .. 2^15 (1 for zero)
__device__ __forceinline__ float row_scale(unsigned int top) {
  const int e = (int)(top >> 23);
  if (e == 0 || e >= 255) return 1.f;
  return __uint_as_float((unsigned int)(127 + min(max(14 - (e - 127), -100), 100)) << 23);
}
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
  const half2v p = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ float f16_rest(float a) {
  const float hi = (float)(_Float16)a;
  return __builtin_isfinite(hi) ? a - hi : 0.f;
}

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
// 8 codes less their zero points; minus = {-(1024 + z), -(64 + z)} as pairs
__device__ __forceinline__ half8 unpack8(uint32_t w, h2 minus_1024, h2 minus_64) {
  const uint32_t w8 = w >> 8;
  const h2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  const h2 a = __builtin_bit_cast(h2, (w & 0x000f000fu) | 0x64006400u) + minus_1024;
  const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00f000f0u) | 0x64006400u), sixteenth, minus_64);
  const h2 c = __builtin_bit_cast(h2, (w8 & 0x000f000fu) | 0x64006400u) + minus_1024;
  const h2 e = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w8 & 0x00f000f0u) | 0x64006400u), sixteenth, minus_64);
  return half8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

constexpr int kVT = 2;          // tiles of 16 items a wave takes at once: an operand of the rows, read from LDS, serves both
constexpr int kWaves = 8;
constexpr uint32_t kLdsRows = 64;

// rows in LDS: row r at r * pitch, pitch = k_tiles * 128 + 8 halves (16 B: the rows of an operand read start in different banks)
__device__ __forceinline__ uint32_t lds_pitch(uint32_t k_tiles) { return k_tiles * kTileK + 8; }

// DT: the rows' type; SDT: the scales'; PG: groups of a tile (128 / group); MB: blocks of 16 rows; FEW: at most 4 rows, row t at place
// 4 t of the instruction, so that a lane has one result to scale and not four; STAGED: rows in LDS, else from the image
template <int DT, int SDT, int PG, bool ZERO, int MB, bool FEW, bool STAGED>
__global__ __launch_bounds__(64 * kWaves) void scores_kernel(ScoresArgs a) {
  constexpr int PLANES = DT == AS_F32 ? 2 : 1, NI = FEW ? 1 : 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
  _Float16 *rows = (_Float16 *)smem;                               // [PLANES][m][pitch]
  const uint32_t pitch = lds_pitch(a.k_tiles);
  float *undo = (float *)(smem + (STAGED ? (size_t)PLANES * a.m * pitch * 2 : 0));   // [64]
  unsigned int *tops = (unsigned int *)(undo + kLdsRows);                          // [64]
  float *part = (float *)(tops + kLdsRows);                                         // [kWaves][kVT][MB][NI][64] where k is shared
  if constexpr (STAGED) {
    // the rows: 512 / m threads each
    uint32_t share = 64 * kWaves;
    while (share > 1 && share * a.m > 64 * kWaves) share >>= 1;
    const uint32_t row = threadIdx.x / share, at = threadIdx.x % share;
    const uint32_t k_all = a.k_tiles * kTileK;
    if (DT != AS_F16) {
      if (threadIdx.x < kLdsRows) tops[threadIdx.x] = 0u;
      __syncthreads();
      float m = 0.f;
      if (row < a.m)
        for (uint32_t k = at; k < a.d; k += share) {
          const float y = fabsf(load_as_f32<DT>(a.x, (size_t)row * a.x_stride + k));
          if (y < INFINITY) m = fmaxf(m, y);
        }
      for (uint32_t s = 1; s < 64 && s < share; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
      if (row < a.m && (at & 63) == 0) atomicMax(&tops[row], __float_as_uint(m));
      __syncthreads();
    }
    if (row < a.m) {
      const float f = DT == AS_F16 ? 1.f : row_scale(tops[row]);
      if (at == 0) undo[row] = 1.f / f;
      for (uint32_t k = at * 2; k < k_all; k += share * 2) {
        const float x = k < a.d ? load_as_f32<DT>(a.x, (size_t)row * a.x_stride + k) * f : 0.f;
        const float y = k + 1 < a.d ? load_as_f32<DT>(a.x, (size_t)row * a.x_stride + k + 1) * f : 0.f;
        *(uint32_t *)(rows + (size_t)row * pitch + k) = f16_pair(x, y);
        if (PLANES == 2) *(uint32_t *)(rows + (size_t)(a.m + row) * pitch + k) = f16_pair(f16_rest(x), f16_rest(y));
      }
    }
    __syncthreads();
  }
  // this lane's rows of the operand
  uint32_t src[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const uint32_t r = FEW ? col >> 2 : b * 16 + col;
    src[b] = (r < a.m ? r : a.m - 1) * pitch + q * 8;
  }
  const uint32_t sub = wave % a.split, groups_here = kWaves / a.split;
  const uint32_t k_lo = (uint32_t)((uint64_t)a.k_tiles * sub / a.split), k_hi = (uint32_t)((uint64_t)a.k_tiles * (sub + 1) / a.split);
  const uint32_t rounds = (a.units + gridDim.x * groups_here - 1) / (gridDim.x * groups_here);
  for (uint32_t round = 0; round < rounds; ++round) {
    const uint32_t unit = (round * gridDim.x + blockIdx.x) * groups_here + wave / a.split;
    const bool live = unit < a.units;
    f32x4 acc[kVT][MB];
#pragma unroll
    for (int t = 0; t < kVT; ++t)
#pragma unroll
      for (int b = 0; b < MB; ++b) acc[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (live) {
      uint32_t tile[kVT];
#pragma unroll
      for (int t = 0; t < kVT; ++t) tile[t] = unit * kVT + t < a.v_tiles ? unit * kVT + t : a.v_tiles - 1;
      for (uint32_t kt = k_lo; kt < k_hi; ++kt) {
        u32x4 w[kVT];
        float s[kVT][PG];
        h2 m1[kVT][PG], m6[kVT][PG];
#pragma unroll
        for (int t = 0; t < kVT; ++t) {
          const size_t at = (size_t)tile[t] * a.k_tiles + kt;
          w[t] = __builtin_nontemporal_load(a.codes + at * 64 + lane);
          const size_t sat = (at * 16 + col) * PG;
#pragma unroll
          for (int g = 0; g < PG; ++g) {
            s[t][g] = load_as_f32<SDT>(a.scales, sat + g);
            uint32_t z = 0x00080008u;
            if constexpr (ZERO) z = a.z[sat + g] * 0x00010001u;
            m1[t][g] = __builtin_bit_cast(h2, z | 0xE400E400u);
            m6[t][g] = __builtin_bit_cast(h2, (z << 4) | 0xD400D400u);
          }
        }
#pragma unroll
        for (int g = 0; g < PG; ++g) {
          f32x4 d[kVT][MB];
#pragma unroll
          for (int t = 0; t < kVT; ++t)
#pragma unroll
            for (int b = 0; b < MB; ++b) d[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = g * (4 / PG); j < (g + 1) * (4 / PG); ++j) {
            half8 u[kVT];
#pragma unroll
            for (int t = 0; t < kVT; ++t) u[t] = unpack8(w[t][j], m1[t][g], m6[t][g]);
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
              for (int p = PLANES - 1; p >= 0; --p) {
                half8 x;
                if constexpr (STAGED) x = *(const half8 *)(rows + (size_t)p * a.m * pitch + src[b] + kt * kTileK + j * 32);
                else x = __builtin_bit_cast(half8, a.image[(((size_t)b * PLANES + p) * a.k_tiles * 4 + kt * 4 + j) * 64 + lane]);
#pragma unroll
                for (int t = 0; t < kVT; ++t) d[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, u[t], d[t][b], 0, 0, 0);
              }
          }
#pragma unroll
          for (int t = 0; t < kVT; ++t)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
              for (int e = 0; e < NI; ++e) acc[t][b][e] = fmaf(d[t][b][e], s[t][g], acc[t][b][e]);
        }
      }
    }
    if (a.split > 1) {  // the waves of a unit add up in the first one's order
      __syncthreads();
      if (sub) {
#pragma unroll
        for (int t = 0; t < kVT; ++t)
#pragma unroll
          for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int e = 0; e < NI; ++e) part[((((size_t)wave * kVT + t) * MB + b) * NI + e) * 64 + lane] = acc[t][b][e];
      }
      __syncthreads();
      if (!sub)
        for (uint32_t o = 1; o < a.split; ++o)
#pragma unroll
          for (int t = 0; t < kVT; ++t)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
              for (int e = 0; e < NI; ++e) acc[t][b][e] += part[((((size_t)(wave + o) * kVT + t) * MB + b) * NI + e) * 64 + lane];
    }
    if (live && !sub) {
#pragma unroll
      for (int t = 0; t < kVT; ++t) {
        const uint32_t item = (unit * kVT + t) * kTileItems + col;
        if (unit * kVT + t >= a.v_tiles || item >= a.v) continue;
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int e = 0; e < NI; ++e) {
            const uint32_t r = FEW ? q : b * 16 + q * 4 + e;
            if (r < a.m) store_from_f32<DT>(a.out, (size_t)r * a.out_stride + item, acc[t][b][e] * (STAGED ? undo[r] : a.undo[r]));
          }
      }
    }
  }
}

// Rows that do not fit the LDS: the same f16 planes as operands, [block][plane][step of 32][lane][8], and what undoes each row's factor.
// A workgroup a row of a block of 16 (rows that are not there: zeros).
template <int DT>
__global__ __launch_bounds__(256) void rows_image_kernel(const void *x, size_t stride, uint32_t m, uint32_t d, uint32_t k_tiles, unsigned int *image, float *undo) {
  constexpr int PLANES = DT == AS_F32 ? 2 : 1;
  __shared__ unsigned int top;
  const uint32_t row = blockIdx.x, b = row >> 4, r = row & 15, words = k_tiles * kTileK / 2;
  if (threadIdx.x == 0) top = 0u;
  __syncthreads();
  if (DT != AS_F16 && row < m) {
    float t = 0.f;
    for (uint32_t k = threadIdx.x; k < d; k += 256) {
      const float y = fabsf(load_as_f32<DT>(x, (size_t)row * stride + k));
      if (y < INFINITY) t = fmaxf(t, y);
    }
    for (int s = 1; s < 64; s <<= 1) t = fmaxf(t, __shfl_xor(t, s));
    if ((threadIdx.x & 63) == 0) atomicMax(&top, __float_as_uint(t));
  }
  __syncthreads();
  const float f = DT == AS_F16 ? 1.f : row_scale(top);
  if (threadIdx.x == 0) undo[row] = 1.f / f;
  for (uint32_t w = threadIdx.x; w < words; w += 256) {
    const uint32_t k = w * 2;
    const float u = row < m && k < d ? load_as_f32<DT>(x, (size_t)row * stride + k) * f : 0.f;
    const float v = row < m && k + 1 < d ? load_as_f32<DT>(x, (size_t)row * stride + k + 1) * f : 0.f;
    const uint32_t step = k >> 5, q = (k & 31) >> 3, in = (k & 7) >> 1;
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
      image[((((size_t)b * PLANES + p) * k_tiles * 4 + step) * 64 + q * 16 + r) * 4 + in] = p ? f16_pair(f16_rest(u), f16_rest(v)) : f16_pair(u, v);
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------------
constexpr size_t kLdsBytes = 160u << 10;
constexpr uint32_t kPass = 64;  // rows of one pass over the codes

struct Form {
  uint32_t m, mb;
  bool few, staged;
  size_t rows_bytes;
};
Form form_of(uint32_t m, uint32_t k_tiles, int dt) {
  Form f;
  f.m = m;
  f.mb = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  f.few = m <= 4;
  f.rows_bytes = (size_t)(dt == AS_F32 ? 2 : 1) * m * (k_tiles * kTileK + 8) * 2;
  f.staged = f.rows_bytes <= (96u << 10);
  return f;
}
uint64_t image_words(const as_table4 *t, uint32_t m, int dt) { return (uint64_t)cdiv(m, 16) * (dt == AS_F32 ? 2 : 1) * t->k_tiles * 4 * 64 * 4; }
struct ScoresScratch {
  unsigned int *image;
  float *undo;
};
uint64_t scores_layout(const as_table4 *t, uint32_t m, int dt, char *base, ScoresScratch &s) {
  Layout l{base};
  const uint32_t pass = std::min(m, kPass);
  const Form f = form_of(pass, t->k_tiles, dt);
  s = ScoresScratch{};
  if (f.staged) return 0;
  s.image = l.take<unsigned int>(image_words(t, f.mb * 16, dt));
  s.undo = l.take<float>(kPass);
  return l.at;
}

int check_shape(as_ctx *ctx, uint64_t v, uint64_t d, uint64_t group, int scale_dt) {
  if (!ctx) return AS_ERR_ARG;
  if (hipSetDevice(ctx->device) != hipSuccess) return fail(ctx, AS_ERR_HIP, "hipSetDevice failed");
  if (v == 0 || d == 0) return fail(ctx, AS_ERR_SHAPE, "the table needs at least one row and one column");
  if (v >= (1ull << 31) || d > (1u << 20)) return fail(ctx, AS_ERR_UNSUPPORTED, "at most 2^31 - 1 items and 2^20 columns");
  if (group != 32 && group != 64 && group != 128) return fail(ctx, AS_ERR_UNSUPPORTED, "groups of 32, 64 or 128 columns");
  if (!dtype_is_training(scale_dt)) return fail(ctx, AS_ERR_ARG, "scales must be AS_F32, AS_BF16 or AS_F16");
  if (stream_is_capturing(ctx->stream)) return fail(ctx, AS_ERR_UNSUPPORTED, "a table cannot be made on a stream that is being captured");
  return AS_OK;
}
void release(as_table4 *t) {
  if (!t) return;
  if (t->codes) (void)handle_free(t->codes);
  if (t->scales) (void)handle_free(t->scales);
  if (t->z) (void)handle_free(t->z);
  delete t;
}
struct Owner {
  as_table4 *t;
  ~Owner() { release(t); }
  as_table4 *give() {
    as_table4 *r = t;
    t = nullptr;
    return r;
  }
};
template <class S>
void move_scales(as_ctx *ctx, const as_table4 *t, bool to, void *plain, unsigned char *plain_z, unsigned int *bad) {
  const uint32_t per = kTileK / t->group;
  const uint64_t slots = (uint64_t)t->v_tiles * t->k_tiles * 16 * per;
  const dim3 grid((unsigned)std::min<uint64_t>((slots + 255) / 256, 16384));
  const uint32_t groups = cdiv(t->d, t->group);
  if (to)
    hipLaunchKernelGGL((scales_kernel<S, true>), grid, dim3(256), 0, ctx->stream, (S *)plain, plain_z, t->v, groups, per, t->k_tiles, slots, (S *)t->scales, t->z, bad);
  else
    hipLaunchKernelGGL((scales_kernel<S, false>), grid, dim3(256), 0, ctx->stream, (S *)plain, plain_z, t->v, groups, per, t->k_tiles, slots, (S *)t->scales, t->z, bad);
}
// the handle's memory, and its image from plain codes, scales and zero points in HBM
int make_table(as_ctx *ctx, uint64_t v, uint64_t d, uint64_t group, int scale_dt, const unsigned char *codes, const void *scales, const unsigned char *zeros,
               unsigned int *bad, as_table4 *t) {
  t->device = ctx->device;
  t->v = v, t->d = d, t->group = (uint32_t)group, t->scale_dt = scale_dt, t->zeros = zeros != nullptr;
  t->v_tiles = cdiv(v, kTileItems), t->k_tiles = cdiv(d, kTileK);
  const uint64_t tiles = (uint64_t)t->v_tiles * t->k_tiles, slots = tiles * 16 * (kTileK / group);
  AS_HIP(ctx, handle_malloc((void **)&t->codes, tiles * 1024));
  AS_HIP(ctx, handle_malloc(&t->scales, slots * dtype_size(scale_dt)));
  if (zeros) AS_HIP(ctx, handle_malloc((void **)&t->z, slots));
  const uint64_t words = tiles * 256;
  hipLaunchKernelGGL(import_codes_kernel, dim3((unsigned)std::min<uint64_t>((words + 255) / 256, 65536)), dim3(256), 0, ctx->stream, codes, v, (uint32_t)d, t->k_tiles,
                     words, t->codes);
  if (scale_dt == AS_F32) move_scales<float>(ctx, t, true, (void *)scales, (unsigned char *)zeros, bad);
  else move_scales<unsigned short>(ctx, t, true, (void *)scales, (unsigned char *)zeros, bad);
  AS_HIP(ctx, hipGetLastError());
  return AS_OK;
}
int read_word(as_ctx *ctx, const unsigned int *dev, unsigned int *host) {
  AS_HIP(ctx, copy_d2h(ctx, host, dev, sizeof(unsigned int)));
  return AS_OK;
}

template <int DT, int SDT, int PG, bool ZERO>
const void *scores_function(const Form &f) {
#define AS_SCORES(MB, FEW) (f.staged ? (const void *)scores_kernel<DT, SDT, PG, ZERO, MB, FEW, true> : (const void *)scores_kernel<DT, SDT, PG, ZERO, MB, FEW, false>)
  return f.few ? AS_SCORES(1, true) : f.mb == 1 ? AS_SCORES(1, false) : f.mb == 2 ? AS_SCORES(2, false) : AS_SCORES(4, false);
#undef AS_SCORES
}
template <int DT, int SDT>
const void *scores_function(const as_table4 *t, const Form &f) {
  if (t->group == 32) return t->zeros ? scores_function<DT, SDT, 4, true>(f) : scores_function<DT, SDT, 4, false>(f);
  if (t->group == 64) return t->zeros ? scores_function<DT, SDT, 2, true>(f) : scores_function<DT, SDT, 2, false>(f);
  return t->zeros ? scores_function<DT, SDT, 1, true>(f) : scores_function<DT, SDT, 1, false>(f);
}
template <int DT>
const void *scores_function(const as_table4 *t, const Form &f) {
  return t->scale_dt == AS_F32 ? scores_function<DT, AS_F32>(t, f) : t->scale_dt == AS_BF16 ? scores_function<DT, AS_BF16>(t, f) : scores_function<DT, AS_F16>(t, f);
}

int scores_pass(as_ctx *ctx, const as_table4 *t, const char *x, uint32_t m, size_t x_stride, int dt, char *out, size_t out_stride, const ScoresScratch &s) {
  const Form f = form_of(m, t->k_tiles, dt);
  ScoresArgs a{};
  a.codes = (const u32x4 *)t->codes, a.scales = t->scales, a.z = t->z;
  a.v = (uint32_t)t->v, a.d = (uint32_t)t->d, a.v_tiles = t->v_tiles, a.k_tiles = t->k_tiles, a.units = cdiv(t->v_tiles, kVT);
  a.x = x, a.x_stride = x_stride, a.m = m, a.out = out, a.out_stride = out_stride;
  if (!f.staged) {
    a.image = (const u32x4 *)s.image, a.undo = s.undo;
    const dim3 grid(f.mb * 16);
    if (dt == AS_F32) hipLaunchKernelGGL((rows_image_kernel<AS_F32>), grid, dim3(256), 0, ctx->stream, x, x_stride, m, a.d, a.k_tiles, s.image, s.undo);
    else if (dt == AS_BF16) hipLaunchKernelGGL((rows_image_kernel<AS_BF16>), grid, dim3(256), 0, ctx->stream, x, x_stride, m, a.d, a.k_tiles, s.image, s.undo);
    else hipLaunchKernelGGL((rows_image_kernel<AS_F16>), grid, dim3(256), 0, ctx->stream, x, x_stride, m, a.d, a.k_tiles, s.image, s.undo);
    AS_HIP(ctx, hipGetLastError());
  }
  // waves that share a unit's k: until there are 8 waves a compute unit or each has one tile
  a.split = 1;
  while (a.split < (uint32_t)kWaves && a.split * 2 <= t->k_tiles && (uint64_t)a.units * a.split < 256 * 8) a.split *= 2;
  const size_t lds = (f.staged ? f.rows_bytes : 0) + 2 * kLdsRows * 4 + (a.split > 1 ? (size_t)kWaves * kVT * f.mb * (f.few ? 1 : 4) * 64 * 4 : 0);
  if (lds > kLdsBytes) return fail(ctx, AS_ERR_UNSUPPORTED, "rows too long for the kernel's LDS");
  const uint32_t here = kWaves / a.split, wanted = cdiv(a.units, here);
  // workgroups that stay: the staging of the rows is paid once each
  const uint32_t per_cu = (uint32_t)std::max<size_t>(1, std::min<size_t>(4, kLdsBytes / lds));
  const uint32_t blocks = std::min(wanted, 256 * per_cu);
  const void *fn = dt == AS_F32 ? scores_function<AS_F32>(t, f) : dt == AS_BF16 ? scores_function<AS_BF16>(t, f) : scores_function<AS_F16>(t, f);
  if (lds > (64u << 10)) AS_HIP(ctx, hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  void *args[] = {&a};
  AS_HIP(ctx, hipLaunchKernel(fn, dim3(blocks), dim3(64 * kWaves), args, lds, ctx->stream));
  return AS_OK;
}

}  // namespace

extern "C" {

int as_table4_import(as_ctx *ctx, const uint8_t *codes, const void *scales, const uint8_t *zeros, uint64_t n_items, uint64_t dim, uint64_t group, int scale_dtype,
                     as_table4 **out) {
  DeviceScope keep;
  return guarded(ctx, [&]() -> int {
    if (out) *out = nullptr;
    AS_TRY(check_shape(ctx, n_items, dim, group, scale_dtype));
    if (!out || !codes || !scales) return fail(ctx, AS_ERR_ARG, "null argument");
    const uint64_t groups = cdiv(dim, group);
    BytesIn C, S, Z;
    AS_TRY(C.bind(ctx, codes, n_items * ((dim + 1) / 2)));
    AS_TRY(S.bind(ctx, scales, n_items * groups * dtype_size(scale_dtype)));
    AS_TRY(Z.bind(ctx, zeros, zeros ? n_items * groups : 0));
    DevBuf<unsigned int> bad;
    AS_TRY(bad.alloc(ctx, 1));
    hipLaunchKernelGGL(clear_word_kernel, dim3(1), dim3(1), 0, ctx->stream, bad.p);
    Owner t{new as_table4()};
    AS_TRY(make_table(ctx, n_items, dim, group, scale_dtype, (const unsigned char *)C.p, S.p, (const unsigned char *)Z.p, bad.p, t.t));
    unsigned int b = 0;
    AS_TRY(read_word(ctx, bad.p, &b));
    if (b) return fail(ctx, AS_ERR_ARG, "zero points must be 0 .. 15");
    *out = t.give();
    return AS_OK;
  });
}

int as_table4_pack(as_ctx *ctx, const void *rows, uint64_t n_items, uint64_t row_stride, uint64_t dim, int dtype, uint64_t group, int scale_dtype, as_table4 **out) {
  DeviceScope keep;
  return guarded(ctx, [&]() -> int {
    if (out) *out = nullptr;
    AS_TRY(check_shape(ctx, n_items, dim, group, scale_dtype));
    if (!out || !rows) return fail(ctx, AS_ERR_ARG, "null argument");
    if (dtype != AS_F64 && !dtype_is_training(dtype)) return fail(ctx, AS_ERR_ARG, "unknown dtype");
    if (row_stride < dim) return fail(ctx, AS_ERR_ARG, "a row stride below the number of columns");
    BytesIn R;
    AS_TRY(R.bind(ctx, rows, ((n_items - 1) * row_stride + dim) * dtype_size(dtype)));
    const uint32_t groups = cdiv(dim, group);
    DevBuf<unsigned char> codes;
    DevBuf<char> scales;
    DevBuf<unsigned int> bad;
    AS_TRY(codes.alloc(ctx, n_items * ((dim + 1) / 2)));
    AS_TRY(scales.alloc(ctx, n_items * groups * dtype_size(scale_dtype)));
    AS_TRY(bad.alloc(ctx, 1));
    hipLaunchKernelGGL(clear_word_kernel, dim3(1), dim3(1), 0, ctx->stream, bad.p);
    const dim3 grid((unsigned)std::min<uint64_t>((n_items * groups + 3) / 4, 65536));
    auto go = [&](auto dt) {
      hipLaunchKernelGGL((quantise_kernel<decltype(dt)::value>), grid, dim3(256), 0, ctx->stream, R.p, (size_t)row_stride, n_items, (uint32_t)dim, (uint32_t)group, groups,
                         scale_dtype, codes.p, (void *)scales.p, bad.p);
    };
    if (dtype == AS_F64) go(std::integral_constant<int, AS_F64>{});
    else if (dtype == AS_F32) go(std::integral_constant<int, AS_F32>{});
    else if (dtype == AS_BF16) go(std::integral_constant<int, AS_BF16>{});
    else go(std::integral_constant<int, AS_F16>{});
    AS_HIP(ctx, hipGetLastError());
    Owner t{new as_table4()};
    AS_TRY(make_table(ctx, n_items, dim, group, scale_dtype, codes.p, scales.p, nullptr, bad.p, t.t));
    unsigned int b = 0;
    AS_TRY(read_word(ctx, bad.p, &b));
    if (b & 1) return fail(ctx, AS_ERR_NONFINITE, "rows hold a value that is not finite in 32 bits");
    if (b & 2) return fail(ctx, AS_ERR_UNSUPPORTED, "a group's scale does not fit the type of the scales");
    *out = t.give();
    return AS_OK;
  });
}

int as_table4_export(as_ctx *ctx, const as_table4 *t, uint8_t *codes, void *scales, uint8_t *zeros) {
  DeviceScope keep;
  return guarded(ctx, [&]() -> int {
    if (!ctx) return AS_ERR_ARG;
    if (!t || !codes || !scales) return fail(ctx, AS_ERR_ARG, "null argument");
    if (t->device != ctx->device) return fail(ctx, AS_ERR_ARG, "a table of another device than the context's");
    if (hipSetDevice(ctx->device) != hipSuccess) return fail(ctx, AS_ERR_HIP, "hipSetDevice failed");
    const uint64_t groups = cdiv(t->d, t->group), row_bytes = (t->d + 1) / 2;
    BytesOut C, S, Z;
    AS_TRY(C.bind(ctx, codes, t->v * row_bytes));
    AS_TRY(S.bind(ctx, scales, t->v * groups * dtype_size(t->scale_dt)));
    AS_TRY(Z.bind(ctx, zeros, zeros ? t->v * groups : 0));
    hipLaunchKernelGGL(export_codes_kernel, dim3((unsigned)std::min<uint64_t>((t->v * row_bytes + 255) / 256, 65536)), dim3(256), 0, ctx->stream, t->codes, t->v,
                       (uint32_t)t->d, t->k_tiles, (unsigned char *)C.p);
    if (t->scale_dt == AS_F32) move_scales<float>(ctx, t, false, S.p, (unsigned char *)Z.p, nullptr);
    else move_scales<unsigned short>(ctx, t, false, S.p, (unsigned char *)Z.p, nullptr);
    AS_HIP(ctx, hipGetLastError());
    AS_TRY(C.finish(ctx));
    AS_TRY(S.finish(ctx));
    AS_TRY(Z.finish(ctx));
    return finish_call(ctx);
  });
}

void as_table4_destroy(as_table4 *t) {
  if (!t) return;
  DeviceScope keep;
  (void)hipSetDevice(t->device);
  release(t);
}
uint64_t as_table4_items(const as_table4 *t) { return t ? t->v : 0; }
uint64_t as_table4_dim(const as_table4 *t) { return t ? t->d : 0; }
uint64_t as_table4_group(const as_table4 *t) { return t ? t->group : 0; }
int as_table4_scale_dtype(const as_table4 *t) { return t ? t->scale_dt : -1; }

uint64_t as_table4_workspace(const as_table4 *t, uint64_t m, int dtype) {
  if (!t || m == 0 || !dtype_is_training(dtype)) return 0;
  ScoresScratch s;
  return scores_layout(t, (uint32_t)std::min<uint64_t>(m, kPass), dtype, nullptr, s);
}

int as_table4_scores(as_ctx *ctx, const as_table4 *t, const void *x, uint64_t m, uint64_t x_stride, int dtype, void *out, uint64_t out_stride, void *workspace,
                     uint64_t workspace_bytes) {
  DeviceScope keep;
  return guarded(ctx, [&]() -> int {
    if (!ctx) return AS_ERR_ARG;
    if (!t) return fail(ctx, AS_ERR_ARG, "null argument");
    if (t->device != ctx->device) return fail(ctx, AS_ERR_ARG, "a table of another device than the context's");
    if (hipSetDevice(ctx->device) != hipSuccess) return fail(ctx, AS_ERR_HIP, "hipSetDevice failed");
    if (!dtype_is_training(dtype)) return fail(ctx, AS_ERR_ARG, "dtype must be AS_F32, AS_BF16 or AS_F16");
    if (m == 0) return AS_OK;
    if (!x || !out) return fail(ctx, AS_ERR_ARG, "null argument");
    if (x_stride < t->d || out_stride < t->v) return fail(ctx, AS_ERR_ARG, "a row stride below the number of columns");
    const uint64_t es = dtype_size(dtype);
    BytesIn X;
    BytesOut O;
    AS_TRY(X.bind(ctx, x, ((m - 1) * x_stride + t->d) * es));
    if (pointer_home(ctx, out) == 0 && out_stride != t->v) return fail(ctx, AS_ERR_ARG, "scores in host memory must be dense");
    AS_TRY(O.bind(ctx, out, ((m - 1) * out_stride + t->v) * es));
    ScoresScratch s;
    Scratch scratch;
    const uint32_t first = (uint32_t)std::min<uint64_t>(m, kPass);
    AS_TRY(scratch.open(ctx, workspace, workspace_bytes, scores_layout(t, first, dtype, nullptr, s)));
    scores_layout(t, first, dtype, scratch.base, s);
    ProfScope prof(ctx, "table4_scores");
    for (uint64_t r = 0; r < m; r += kPass)
      AS_TRY(scores_pass(ctx, t, (const char *)X.p + r * x_stride * es, (uint32_t)std::min<uint64_t>(m - r, kPass), x_stride, dtype, (char *)O.p + r * out_stride * es,
                         out_stride, s));
    AS_TRY(O.finish(ctx));
    return finish_call(ctx);
  });
}

}  // extern "C"
