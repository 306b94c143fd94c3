// table4.hip -- a table of rows held in 4 bits with group scales, and its products with a few rows (the scores of single queries).
//
//   W_vk = s_{v, k / g} (q_vk - z_{v, k / g}),  q in 0 .. 15, z = 8 where the table has none        y_mv = sum_k x_mk W_vk
//
// What bounds it: d v / 2 bytes of codes (and 2 d v / g of 16-bit scales) for 2 m d v flops -- memory, up to 16 rows; with 64 the
// unpacking and the operands' way out of LDS take as long.  So the codes are streamed once, unpacked in registers and fed to the matrix
// pipe whatever m is: 16 items x 16 rows x 32 k an instruction, rows that are not there cost nothing that is scarce.
// Measured: 8 bf16 rows, 1 000 000 items of 768 in groups of 128 (412 MB): 84 us, 4.9 TB/s; one f32 row, 1 000 000 of 128 in groups of 32
// (76 MB, in the last cache): 17 us; 16 f16 rows, 11 000 of 4 000: 12 us; 64 bf16 rows, 362 031 of 1 280: 139 us.
// Unpacking.  A 32-bit word holds 8 codes, interleaved so that code k sits in the low and code k + 1 in the high half of a mask:
// (w & 0x000f000f) | 0x6400 is the f16 pair 1024 + q, (w & 0x00f000f0) | 0x6400 the pair 1024 + 16 q; one packed add or multiply-add
// takes 1024 + z off (exact: small integers), a shift by 8 brings the other four.  9 instructions for 8 values.  (5 without the
// subtraction, codes as f16 subnormals and 8 sum(x) taken off before the first product, gave sums 2^-17 off: the matrix pipe aligns
// products by exponents as they are encoded.)
// Types.  Codes less zero points are integers, exact in f16; rows of f16 go as they are, bf16 after a power of two a row that brings its
// largest finite value to 2^14 .. 2^15 (8 bits fit, down to 2^-28 of that), f32 after the same as a sum of two f16 (22 bits).  Products
// of a group are summed in f32 by the matrix pipe, groups in f32 after their scale.
// Layout (made once, by the handle): tiles of 16 items x 128 k, 1 KB: lane l of a wave holds item l & 15 and, of each 32 k, the 8
// from 8 (l >> 4): its operand of four instructions in one 16-byte load.  Scales of a tile: item by item its 4 / 2 / 1 groups.
#include "table4_address.h"
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
// Eight codes of a plain row, code k at bits 4 k, to their places in a word of the image.
__device__ __forceinline__ uint32_t place_codes(uint32_t w) {
  auto pack = [](uint32_t x) {  // the low halves of four bytes, side by side
    x = (x | x >> 4) & 0x00ff00ffu;
    return (x | x >> 8) & 0xffffu;
  };
  return pack(w & 0x0f0f0f0fu) | pack(w >> 4 & 0x0f0f0f0fu) << 16;
}
// A thread four words of the image.  Plain codes: row v is ceil(d / 2) bytes, column 2 j in the low half of byte j.
__global__ __launch_bounds__(256) void import_codes_kernel(const unsigned char *codes, uint64_t v, uint32_t d, uint32_t k_tiles, uint64_t lanes, u32x4 *out) {
  const uint64_t row_bytes = (d + 1) / 2;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < lanes; i += (uint64_t)gridDim.x * 256) {
    const uint32_t lane = i & 63;
    const uint64_t tile = i >> 6, item = tile / k_tiles * kTileItems + (lane & 15);
    const uint32_t first = (uint32_t)(tile % k_tiles) * kTileK + (lane >> 4) * 8;
    u32x4 o = {0u, 0u, 0u, 0u};
    if (item < v)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k0 = first + j * 32;
        const unsigned char *p = codes + item * row_bytes + (k0 >> 1);
        uint32_t w = 0;
        if (k0 + 8 <= d) {
          __builtin_memcpy(&w, p, 4);
        } else {
          for (uint32_t k = 0; k < 8 && k0 + k < d; ++k) w |= (p[k >> 1] >> (4 * (k & 1)) & 15u) << (4 * k);
        }
        o[j] = place_codes(w);
      }
    out[i] = o;
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
  uint32_t v, d, v_tiles, k_tiles, units;
  int dt, scale_bf16;
  const char *x;
  size_t x_stride;
  uint32_t m;
  void *out;
  size_t out_stride;
  uint32_t split;        // rows in LDS: waves of a workgroup that share a unit's k
  // rows that are read as operands from memory: f16 rows themselves, or their image, made by rows_image_kernel
  const char *operand;
  size_t lane_row, plane;  // bytes between rows, planes
  uint32_t lane_q, per_step, per_tile, k_bytes;  // ... 8 k, 32 k, 128 k; what is there of a row
  const float *undo;     // what undoes each row's factor, null: 1
  uint32_t supers;       // parts of k that different workgroups take, and where their sums meet: [super][m][v]
  float *part;
};

// the power of two that brings a largest finite magnitude to 2^14 .. 2^15 (those below 2^-112: as far as 2^126 goes, 2^0 and more)
__device__ __forceinline__ float row_scale(unsigned int top) { return __uint_as_float((unsigned int)(127 + min(141 - (int)(top >> 23), 126)) << 23); }
__device__ __forceinline__ uint32_t f16_pair(float a, float b) {
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
  const half2v p = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ float f16_rest(float a) {
  const float hi = (float)(_Float16)a;
  return __builtin_isfinite(hi) ? a - hi : 0.f;
}
// Eight values of a row (PLANES 1: 16 bits a value, bf16 or f16 by `dt`; 2: f32)
template <int PLANES>
struct RowPiece {
  Piece8<PLANES == 2 ? AS_F32 : AS_F16> raw;
  __device__ __forceinline__ float value(int dt, int e) const {
    if constexpr (PLANES == 2) return __uint_as_float(raw.w[e >> 2][e & 3]);
    const unsigned short h = (unsigned short)(raw.w[0][e >> 1] >> (16 * (e & 1)));
    return dt == AS_BF16 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
  }
  __device__ __forceinline__ float top(int dt) const {  // its largest finite magnitude
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = fabsf(value(dt, e));
      t = y < INFINITY ? fmaxf(t, y) : t;
    }
    return t;
  }
  __device__ __forceinline__ void planes(int dt, float f, u32x4 (&o)[PLANES]) const {
    if (PLANES == 1 && dt == AS_F16) {
      o[0] = raw.w[0];
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = value(dt, 2 * i) * f, v = value(dt, 2 * i + 1) * f;
      o[0][i] = f16_pair(u, v);
      if constexpr (PLANES == 2) o[PLANES - 1][i] = f16_pair(f16_rest(u), f16_rest(v));
    }
  }
};

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
// The constants of the unpacking in registers: as literals they keep the compiler from taking mask and exponent in one instruction.
struct Unpack {
  uint32_t low = 0x000f000fu, high = 0x00f000f0u, exponent = 0x64006400u;
  __device__ __forceinline__ Unpack() { asm("" : "+v"(low), "+v"(high), "+s"(exponent)); }
  // 8 codes less their zero points; minus = {-(1024 + z), -(64 + z)} as pairs
  __device__ __forceinline__ half8 operator()(uint32_t w, h2 minus_1024, h2 minus_64) const {
    const uint32_t w8 = w >> 8;
    const h2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const h2 a = __builtin_bit_cast(h2, (w & low) | exponent) + minus_1024;
    const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & high) | exponent), sixteenth, minus_64);
    const h2 c = __builtin_bit_cast(h2, (w8 & low) | exponent) + minus_1024;
    const h2 e = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w8 & high) | exponent), sixteenth, minus_64);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
  }
};

constexpr int kVT = 2;          // tiles of 16 items a wave takes at once (a unit): an operand of the rows, read from LDS, serves both
constexpr uint32_t kWaves = 8;
constexpr uint32_t kLdsRows = 64;
__device__ __forceinline__ uint32_t at_most(uint32_t a, uint32_t b) { return a < b ? a : b; }

// One step of a wave: kVT tiles of 16 items x 128 k as they lie in memory.  WIDE: scales of 32 bits; PG: groups of a tile
template <bool WIDE, int PG, bool ZERO>
struct Tiles {
  static constexpr int SW = WIDE ? PG : PG == 4 ? 2 : 1;  // words of an item's scales
  u32x4 w[kVT];
  uint32_t s[kVT][SW], z[kVT];
  __device__ __forceinline__ void load(const ScoresArgs &a, uint32_t unit, uint32_t kt) {
    const uint32_t lane = threadIdx.x & 63, col = lane & 15;
#pragma unroll
    for (int t = 0; t < kVT; ++t) {
      const size_t at = (size_t)at_most(unit * kVT + t, a.v_tiles - 1) * a.k_tiles + kt;
      w[t] = a.codes[at * 64 + lane];
      const char *sp = (const char *)a.scales + at * (16 * PG * (WIDE ? 4 : 2));
      if constexpr (WIDE || PG > 1) {
#pragma unroll
        for (int i = 0; i < SW; ++i) s[t][i] = ((const uint32_t *)sp)[col * SW + i];
      } else {
        s[t][0] = ((const unsigned short *)sp)[col];
      }
      if constexpr (ZERO) {
        const unsigned char *zp = a.z + at * (16 * PG);
        if constexpr (PG == 4) z[t] = ((const uint32_t *)zp)[col];
        else if constexpr (PG == 2) z[t] = ((const unsigned short *)zp)[col];
        else z[t] = zp[col];
      }
    }
  }
  __device__ __forceinline__ float scale(int bf16, int t, int g) const {
    if constexpr (WIDE) return __uint_as_float(s[t][g]);
    const uint32_t h = PG == 1 ? s[t][0] : s[t][g >> 1] >> (16 * (g & 1));
    return bf16 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (unsigned short)h);
  }
  // acc += its products with the rows; rows(p, b, j): plane p of block b's operand for the 32 k from 32 j
  template <int PLANES, int MB, int NI, class Rows>
  __device__ __forceinline__ void multiply(const Unpack &unpack, int bf16, Rows &&rows, float (&acc)[kVT][MB][NI]) const {
#pragma unroll
    for (int g = 0; g < PG; ++g) {
      f32x4 d[kVT][MB];
      h2 m1[kVT], m6[kVT];
#pragma unroll
      for (int t = 0; t < kVT; ++t) {
        const uint32_t zero = ZERO ? ((z[t] >> (8 * g)) & 255u) * 0x00010001u : 0x00080008u;
        m1[t] = __builtin_bit_cast(h2, zero | 0xE400E400u);
        m6[t] = __builtin_bit_cast(h2, (zero << 4) | 0xD400D400u);
#pragma unroll
        for (int b = 0; b < MB; ++b) d[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int j = g * (4 / PG); j < (g + 1) * (4 / PG); ++j) {
        half8 u[kVT];
#pragma unroll
        for (int t = 0; t < kVT; ++t) u[t] = unpack(w[t][j], m1[t], m6[t]);
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int p = PLANES - 1; p >= 0; --p) {
            const half8 x = __builtin_bit_cast(half8, rows(p, b, j));
#pragma unroll
            for (int t = 0; t < kVT; ++t) d[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, u[t], d[t][b], 0, 0, 0);
          }
      }
#pragma unroll
      for (int t = 0; t < kVT; ++t) {
        const float s = scale(bf16, t, g);
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int e = 0; e < NI; ++e) acc[t][b][e] = fmaf(d[t][b][e], s, acc[t][b][e]);
      }
    }
  }
};
template <int PLANES>
__device__ __forceinline__ void put_score(const ScoresArgs &a, uint32_t r, uint32_t item, float y) {
  if (PLANES == 2) store_from_f32<AS_F32>(a.out, (size_t)r * a.out_stride + item, y);
  else if (a.dt == AS_BF16) store_from_f32<AS_BF16>(a.out, (size_t)r * a.out_stride + item, y);
  else store_from_f32<AS_F16>(a.out, (size_t)r * a.out_stride + item, y);
}

// Workgroups of a compute unit, the grid's size, and steps a wave's loads are ahead.  More workgroups stage the rows more often; fewer, or
// a shorter lead, leave too little under way.  One query, 419 724 items of 768 / 1 000 000 of 128, eight of 1 000 000 of 768 (us): 2
// workgroups 2 steps ahead 34 / 18.6 / 89, 1 step 34 / 18.7 / 92; 3 workgroups 35 / 22.6 / 96; 1 workgroup 32 / 20.5 / 93; 4, none ahead
// 41 / 22.5 / 91.
constexpr int resident_groups(int mb, int groups_of_tile) { return mb == 4 || (mb == 2 && groups_of_tile == 4) ? 1 : 2; }

// rows in LDS: row r at r * pitch, pitch = k_tiles * 128 + 8 halves (16 B: the rows of an operand read start in different banks)
__host__ __device__ __forceinline__ uint32_t lds_pitch(uint32_t k_tiles) { return k_tiles * kTileK + 8; }

// Where a wave's operand of the rows comes from.  Rows in LDS serve workgroups that walk many units; a workgroup of one unit would wait for
// memory twice, first for all rows and then for its tiles: it takes both from memory at once.
enum { kInLds, kInMemory };
template <int PLANES, int FROM>
struct RowOperands {};
template <int PLANES>
struct RowOperands<PLANES, kInMemory> {
  u32x4 x[PLANES][4];
  __device__ __forceinline__ void load(const ScoresArgs &a, size_t row_at, uint32_t q, uint32_t kt) {
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t k = kt * a.per_tile + j * a.per_step;
        const u32x4 y = *(const u32x4 *)(a.operand + p * a.plane + row_piece_at(row_at, q * a.lane_q, q * 16, k, a.k_bytes));
        x[p][j] = row_piece_there(q * 16, k, a.k_bytes) ? y : u32x4{0u, 0u, 0u, 0u};
      }
  }
};

// PLANES: 2 for f32 rows; MB: blocks of 16 rows; FEW: at most 4 rows, row t at places 4 t .. 4 t + 3 of the instruction, so that a
// lane has one result to scale and not four
template <int PLANES, bool WIDE, int PG, bool ZERO, int MB, bool FEW, int FROM>
__global__ __launch_bounds__(64 * kWaves, 2 * resident_groups(MB, PG)) void scores_kernel(ScoresArgs a) {
  constexpr int NI = FEW ? 1 : 4, NT = 64 * kWaves, AHEAD = MB == 1 && FROM == kInLds ? 2 : 1;
  struct Step {
    Tiles<WIDE, PG, ZERO> tiles;
    RowOperands<PLANES, FROM> rows;
  };
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
  _Float16 *rows = (_Float16 *)smem;                               // [PLANES][m][pitch]
  const uint32_t pitch = lds_pitch(a.k_tiles);
  float *undo = (float *)(smem + (FROM == kInLds ? (size_t)PLANES * a.m * pitch * 2 : 0));   // [64]
  unsigned int *tops = (unsigned int *)(undo + kLdsRows);          // [64]
  float *part = (float *)(tops + kLdsRows);                        // [kWaves][kVT][MB][NI][64] where k is shared
  const uint32_t sub = wave % a.split, teams = kWaves / a.split, stride = gridDim.x * teams;
  const uint32_t k_lo = (uint32_t)((uint64_t)a.k_tiles * sub / a.split), k_hi = (uint32_t)((uint64_t)a.k_tiles * (sub + 1) / a.split);
  const uint32_t first = blockIdx.x * teams + wave / a.split;
  const uint32_t rounds = (a.units + stride - 1) / stride;
  const size_t row_at = at_most(FEW ? col >> 2 : col, a.m - 1) * a.lane_row;
  Step ring[AHEAD + 1];
  uint32_t ahead_unit = first, ahead_kt = k_lo;  // what is asked for next (behind the last unit: that one again)
  auto ask = [&](Step &s) {
    s.tiles.load(a, at_most(ahead_unit, a.units - 1), ahead_kt);
    if constexpr (FROM == kInMemory) s.rows.load(a, row_at, q, ahead_kt);
    if (++ahead_kt == k_hi) ahead_kt = k_lo, ahead_unit += stride;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) ask(ring[i]);
  if constexpr (FROM == kInMemory) {
    if (threadIdx.x < kLdsRows) undo[threadIdx.x] = a.undo && threadIdx.x < a.m ? a.undo[threadIdx.x] : 1.f;
    __syncthreads();
  } else {
    // the rows: NT / m threads each
    uint32_t share = NT;
    while (share > 1 && share * a.m > NT) share >>= 1;
    const uint32_t row = threadIdx.x / share, at = threadIdx.x % share, pieces = a.k_tiles * (kTileK / 8);
    const char *src = a.x + (size_t)at_most(row, a.m - 1) * a.x_stride * (PLANES == 2 ? 4 : 2);
    const bool as_is = PLANES == 1 && a.dt == AS_F16;
    constexpr int B = PLANES == 2 ? 4 : 8;  // pieces under way
    if (!as_is) {
      if (threadIdx.x < kLdsRows) tops[threadIdx.x] = 0u;
      __syncthreads();
      float m = 0.f;
      for (uint32_t p0 = at; p0 < pieces; p0 += B * share) {
        RowPiece<PLANES> piece[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (p0 + i * share < pieces) piece[i].raw.load(src, (p0 + i * share) * 8, a.d);
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (p0 + i * share < pieces) m = fmaxf(m, piece[i].top(a.dt));
      }
      for (uint32_t s = 1; s < 64 && s < share; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
      if (row < a.m && (at & 63) == 0) atomicMax(&tops[row], __float_as_uint(m));
      __syncthreads();
    }
    if (row < a.m) {
      const float f = as_is ? 1.f : row_scale(tops[row]);
      if (at == 0) undo[row] = 1.f / f;
      for (uint32_t p0 = at; p0 < pieces; p0 += B * share) {
        RowPiece<PLANES> piece[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (p0 + i * share < pieces) piece[i].raw.load(src, (p0 + i * share) * 8, a.d);
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const uint32_t p = p0 + i * share;
          if (p >= pieces) break;
          u32x4 o[PLANES];
          piece[i].planes(a.dt, f, o);
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) *(u32x4 *)(rows + (size_t)(pl * a.m + row) * pitch + p * 8) = o[pl];
        }
      }
    }
    __syncthreads();
  }
  // this lane's rows of the operand
  uint32_t src[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) src[b] = at_most(FEW ? col >> 2 : b * 16 + col, a.m - 1) * pitch + q * 8;
  const uint32_t plane = a.m * pitch;
  const Unpack unpack;
  float acc[kVT][MB][NI];
#pragma unroll
  for (int t = 0; t < kVT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int e = 0; e < NI; ++e) acc[t][b][e] = 0.f;
  uint32_t unit = first, kt = k_lo, round = 0;
  auto step = [&](const Step &now, Step &next) {
    const bool last = kt + 1 == k_hi;
    ask(next);
    now.tiles.template multiply<PLANES, MB, NI>(unpack, a.scale_bf16, [&](int p, int b, int j) {
      if constexpr (FROM == kInMemory) return now.rows.x[p][j];
      else return *(const u32x4 *)(rows + p * plane + src[b] + kt * kTileK + j * 32);
    }, acc);
    ++kt;
    if (!last) return;
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
#pragma unroll
    for (int t = 0; t < kVT; ++t) {
      const uint32_t tile = unit * kVT + t, item = tile * kTileItems + col;
      const bool there = !sub && unit < a.units && tile < a.v_tiles && item < a.v;
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int e = 0; e < NI; ++e) {
          const uint32_t r = FEW ? q : b * 16 + q * 4 + e;
          if (there && r < a.m) put_score<PLANES>(a, r, item, acc[t][b][e] * undo[r]);
          acc[t][b][e] = 0.f;
        }
    }
    unit += stride, kt = k_lo, ++round;
  };
  while (round < rounds) {
#pragma unroll
    for (int i = 0; i <= AHEAD; ++i)
      if (round < rounds) step(ring[i], ring[(i + AHEAD) % (AHEAD + 1)]);
  }
}

// More than 16 rows that do not fit the LDS: a workgroup's 8 units walk k together, 128 at a time, the rows' operands for them in LDS twice; where there
// are few items, workgroups take parts of k (super) and scores_join_kernel adds them up.
template <int PLANES, bool WIDE, int PG, bool ZERO, int MB>
__global__ __launch_bounds__(64 * kWaves) void scores_long_kernel(ScoresArgs a) {
  constexpr uint32_t NT = 64 * kWaves, kPieces = MB * PLANES * 256, kEach = (kPieces + NT - 1) / NT;
  typedef Tiles<WIDE, PG, ZERO> Step;
  __shared__ u32x4 buffer[2][kPieces];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
  const uint32_t super = blockIdx.x % a.supers, unit = blockIdx.x / a.supers * kWaves + wave, from = at_most(unit, a.units - 1);
  const uint32_t k_lo = (uint32_t)((uint64_t)a.k_tiles * super / a.supers), k_hi = (uint32_t)((uint64_t)a.k_tiles * (super + 1) / a.supers);
  u32x4 chunk[kEach];
  auto fetch = [&](uint32_t kt) {
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t at = i * NT + threadIdx.x;
      if (kPieces % NT == 0 || at < kPieces) chunk[i] = ((const u32x4 *)a.operand)[((size_t)(at >> 8) * a.k_tiles + kt) * 256 + (at & 255)];
    }
  };
  Step even, odd;
  fetch(k_lo);
  even.load(a, from, k_lo);
  const Unpack unpack;
  float acc[kVT][MB][4];
#pragma unroll
  for (int t = 0; t < kVT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][b][e] = 0.f;
  auto step = [&](uint32_t kt, u32x4 *rows, const Step &now, Step &next) {
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      const uint32_t at = i * NT + threadIdx.x;
      if (kPieces % NT == 0 || at < kPieces) rows[at] = chunk[i];
    }
    if (kt + 1 < k_hi) {
      fetch(kt + 1);
      next.load(a, from, kt + 1);
    }
    __syncthreads();
    now.template multiply<PLANES, MB, 4>(unpack, a.scale_bf16, [&](int p, int b, int j) { return rows[(b * PLANES + p) * 256 + j * 64 + lane]; }, acc);
  };
  for (uint32_t kt = k_lo; kt < k_hi; kt += 2) {
    step(kt, buffer[0], even, odd);
    if (kt + 1 < k_hi) step(kt + 1, buffer[1], odd, even);
  }
  if (unit >= a.units) return;
#pragma unroll
  for (int t = 0; t < kVT; ++t) {
    const uint32_t tile = unit * kVT + t, item = tile * kTileItems + col;
    if (tile >= a.v_tiles || item >= a.v) continue;
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t r = b * 16 + q * 4 + e;
        if (r >= a.m) continue;
        const float y = acc[t][b][e] * a.undo[r];
        if (a.supers > 1) a.part[((size_t)super * a.m + r) * a.v + item] = y;
        else put_score<PLANES>(a, r, item, y);
      }
  }
}
template <int DT>
__global__ __launch_bounds__(256) void scores_join_kernel(const float *part, uint32_t supers, uint32_t m, uint32_t v, void *out, size_t out_stride) {
  const size_t total = (size_t)m * v;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    float y = 0.f;
    for (uint32_t s = 0; s < supers; ++s) y += part[s * total + i];
    store_from_f32<DT>(out, i / v * out_stride + i % v, y);
  }
}
// The f16 planes of rows as operands, [block][plane][step of 32][lane][8], and what undoes each row's factor.
// A workgroup a row of a block of 16 (rows that are not there: zeros).
template <int PLANES>
__global__ __launch_bounds__(512) void rows_image_kernel(const char *x, size_t stride, int dt, uint32_t m, uint32_t d, uint32_t k_tiles, u32x4 *image, float *undo) {
  __shared__ unsigned int top;
  const uint32_t row = blockIdx.x, b = row >> 4, r = row & 15, pieces = k_tiles * (kTileK / 8);
  const char *src = x + (size_t)at_most(row, m - 1) * stride * (PLANES == 2 ? 4 : 2);
  const bool as_is = PLANES == 1 && dt == AS_F16;
  if (threadIdx.x == 0) top = 0u;
  __syncthreads();
  if (!as_is) {
    float t = 0.f;
    for (uint32_t p = threadIdx.x; p < pieces; p += 512) {
      RowPiece<PLANES> piece;
      piece.raw.load(src, p * 8, d);
      t = fmaxf(t, piece.top(dt));
    }
    for (int s = 1; s < 64; s <<= 1) t = fmaxf(t, __shfl_xor(t, s));
    if ((threadIdx.x & 63) == 0) atomicMax(&top, __float_as_uint(t));
  }
  __syncthreads();
  const float f = as_is ? 1.f : row_scale(top);
  if (threadIdx.x == 0) undo[row] = 1.f / f;
  for (uint32_t p = threadIdx.x; p < pieces; p += 512) {
    RowPiece<PLANES> piece;
    piece.raw.load(src, row < m ? p * 8 : d, d);
    u32x4 o[PLANES];
    piece.planes(dt, f, o);
#pragma unroll
    for (int pl = 0; pl < PLANES; ++pl) image[(((size_t)b * PLANES + pl) * k_tiles * 4 + (p >> 2)) * 64 + (p & 3) * 16 + r] = o[pl];
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------------
constexpr size_t kLdsBytes = 160u << 10;
constexpr uint32_t kPass = 64;  // rows of one pass over the codes
constexpr uint32_t kChips = 256;

struct Form {
  int mb;
  bool few, in_lds, as_is;   // rows in LDS; else: rows are read where they lie
  uint32_t split, blocks, supers;
  size_t lds;
};
// aligned: rows start at multiples of 16 bytes
Form form_of(const as_table4 *t, uint32_t m, int dt, bool aligned) {
  Form f{};
  const uint32_t units = cdiv(t->v_tiles, kVT);
  f.mb = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  const size_t rows = (size_t)(dt == AS_F32 ? 2 : 1) * m * lds_pitch(t->k_tiles) * 2 + 2 * kLdsRows * 4;
  f.few = m <= 4;
  // waves that share a unit's k: until there are 8 waves a compute unit or each has one tile
  f.split = 1;
  while (f.split < kWaves && f.split * 2 <= t->k_tiles && (uint64_t)units * f.split < kChips * kWaves) f.split *= 2;
  const size_t meet = f.split > 1 ? (size_t)kWaves * kVT * f.mb * (f.few ? 1 : 4) * 64 * 4 : 0;
  f.lds = rows + meet;
  f.in_lds = f.lds <= kLdsBytes;
  f.supers = 1;
  const uint32_t wanted = cdiv(units, kWaves / f.split);
  // A workgroup whose waves have one unit each takes f16 rows of whole 16-byte pieces from memory as they lie (16 rows, 11 000 items of
  // 4 000: 12 us, from LDS 16); so it does, from an image, rows of 16 bits that leave room for one workgroup a compute unit (16 bf16 rows,
  // 54 422 items of 3 712: 30 us, from LDS 43; f32 rows, twice the operands: 80 us for 154 422 of 1 900, from LDS 50).
  f.as_is = f.mb == 1 && !f.few && aligned && dt == AS_F16 && t->d % 8 == 0 && wanted <= 2 * kChips;
  if (f.as_is || (f.mb == 1 && !f.few && dt != AS_F32 && f.lds > kLdsBytes / 2)) f.in_lds = false;
  if (f.in_lds) {
    // workgroups that stay: the rows are read once each
    const uint32_t per_cu = (uint32_t)std::min<size_t>(resident_groups(f.mb, kTileK / t->group), kLdsBytes / f.lds);
    f.blocks = std::min(wanted, kChips * per_cu);
  } else if (f.mb == 1) {
    f.lds = 2 * kLdsRows * 4 + (f.split > 1 ? (size_t)kWaves * kVT * 4 * 64 * 4 : 0);
    f.blocks = std::min(wanted, kChips * 2);
    f.few = false;
  } else {
    f.lds = 0;
    const uint32_t groups = cdiv(units, kWaves);
    if (groups < kChips) f.supers = std::max(1u, std::min(t->k_tiles / 2, kChips / groups));
    f.blocks = groups * f.supers;
  }
  return f;
}
struct ScoresScratch {
  u32x4 *image;
  float *undo, *part;
};
uint64_t scores_layout(const as_table4 *t, uint32_t m, int dt, char *base, ScoresScratch &s) {
  Layout l{base};
  const uint32_t pass = std::min(m, kPass);
  const Form f = form_of(t, pass, dt, false);
  s = ScoresScratch{};
  if (f.in_lds) return 0;  // (so are the fewer rows of a last pass)
  s.image = l.take<u32x4>((uint64_t)f.mb * (dt == AS_F32 ? 2 : 1) * t->k_tiles * 256);
  s.undo = l.take<float>(kPass);
  s.part = l.take<float>(f.supers > 1 ? (uint64_t)f.supers * pass * t->v : 0);
  return l.at;
}
int check_shape(as_ctx *ctx, uint64_t v, uint64_t d, uint64_t group, int scale_dt) {
  if (!ctx) return AS_ERR_ARG;
  if (hipSetDevice(ctx->device) != hipSuccess) return fail(ctx, AS_ERR_HIP, "hipSetDevice failed");
  ctx_enter(ctx);
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
  hipLaunchKernelGGL(import_codes_kernel, dim3((unsigned)std::min<uint64_t>((tiles * 64 + 255) / 256, 65536)), dim3(256), 0, ctx->stream, codes, v, (uint32_t)d,
                     t->k_tiles, tiles * 64, (u32x4 *)t->codes);
  if (scale_dt == AS_F32) move_scales<float>(ctx, t, true, (void *)scales, (unsigned char *)zeros, bad);
  else move_scales<unsigned short>(ctx, t, true, (void *)scales, (unsigned char *)zeros, bad);
  AS_HIP(ctx, hipGetLastError());
  return AS_OK;
}
int read_word(as_ctx *ctx, const unsigned int *dev, unsigned int *host) {
  AS_HIP(ctx, copy_d2h(ctx, host, dev, sizeof(unsigned int)));
  return AS_OK;
}

template <int PLANES, bool WIDE, int PG, bool ZERO>
const void *scores_function(const Form &f) {
  if (!f.in_lds)
    return f.mb == 1 ? (const void *)scores_kernel<PLANES, WIDE, PG, ZERO, 1, false, kInMemory> : f.mb == 2 ? (const void *)scores_long_kernel<PLANES, WIDE, PG, ZERO, 2>
                                                                                                           : (const void *)scores_long_kernel<PLANES, WIDE, PG, ZERO, 4>;
  return f.few ? (const void *)scores_kernel<PLANES, WIDE, PG, ZERO, 1, true, kInLds> : f.mb == 1 ? (const void *)scores_kernel<PLANES, WIDE, PG, ZERO, 1, false, kInLds>
         : f.mb == 2 ? (const void *)scores_kernel<PLANES, WIDE, PG, ZERO, 2, false, kInLds> : (const void *)scores_kernel<PLANES, WIDE, PG, ZERO, 4, false, kInLds>;
}
template <int PLANES, bool WIDE>
const void *scores_function(const as_table4 *t, const Form &f) {
  if (t->group == 32) return t->zeros ? scores_function<PLANES, WIDE, 4, true>(f) : scores_function<PLANES, WIDE, 4, false>(f);
  if (t->group == 64) return t->zeros ? scores_function<PLANES, WIDE, 2, true>(f) : scores_function<PLANES, WIDE, 2, false>(f);
  return t->zeros ? scores_function<PLANES, WIDE, 1, true>(f) : scores_function<PLANES, WIDE, 1, false>(f);
}
template <int PLANES>
const void *scores_function(const as_table4 *t, const Form &f) {
  return t->scale_dt == AS_F32 ? scores_function<PLANES, true>(t, f) : scores_function<PLANES, false>(t, f);
}

int scores_pass(as_ctx *ctx, const as_table4 *t, const char *x, uint32_t m, size_t x_stride, int dt, char *out, size_t out_stride, const ScoresScratch &s) {
  const Form f = form_of(t, m, dt, x_stride % 8 == 0 && ((uintptr_t)x & 15) == 0);
  ScoresArgs a{};
  a.codes = (const u32x4 *)t->codes, a.scales = t->scales, a.z = t->z, a.scale_bf16 = t->scale_dt == AS_BF16;
  a.v = (uint32_t)t->v, a.d = (uint32_t)t->d, a.v_tiles = t->v_tiles, a.k_tiles = t->k_tiles, a.units = cdiv(t->v_tiles, kVT);
  a.dt = dt, a.x = x, a.x_stride = x_stride, a.m = m, a.out = out, a.out_stride = out_stride;
  a.split = f.split, a.supers = f.supers, a.part = s.part;
  if (!f.in_lds && f.as_is) {
    a.operand = x, a.lane_row = x_stride * 2, a.lane_q = 16, a.per_step = 64, a.per_tile = 256, a.k_bytes = a.d * 2;
  } else if (!f.in_lds) {
    a.operand = (const char *)s.image, a.lane_row = 16, a.lane_q = 256, a.per_step = 1024, a.per_tile = 4096, a.k_bytes = ~0u, a.plane = (size_t)a.k_tiles * 4096;
    a.undo = s.undo;
    const dim3 grid(f.mb * 16);
    if (dt == AS_F32) hipLaunchKernelGGL((rows_image_kernel<2>), grid, dim3(512), 0, ctx->stream, x, x_stride, dt, m, a.d, a.k_tiles, s.image, s.undo);
    else hipLaunchKernelGGL((rows_image_kernel<1>), grid, dim3(512), 0, ctx->stream, x, x_stride, dt, m, a.d, a.k_tiles, s.image, s.undo);
    AS_HIP(ctx, hipGetLastError());
  }
  const void *fn = dt == AS_F32 ? scores_function<2>(t, f) : scores_function<1>(t, f);
  if (f.lds > (64u << 10)) AS_HIP(ctx, hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)f.lds));
  void *args[] = {&a};
  AS_HIP(ctx, hipLaunchKernel(fn, dim3(f.blocks), dim3(64 * kWaves), args, f.lds, ctx->stream));
  if (f.supers > 1) {
    const dim3 grid((unsigned)std::min<uint64_t>(((uint64_t)m * t->v + 255) / 256, 8192));
    if (dt == AS_F32) hipLaunchKernelGGL((scores_join_kernel<AS_F32>), grid, dim3(256), 0, ctx->stream, s.part, f.supers, m, a.v, (void *)out, out_stride);
    else if (dt == AS_BF16) hipLaunchKernelGGL((scores_join_kernel<AS_BF16>), grid, dim3(256), 0, ctx->stream, s.part, f.supers, m, a.v, (void *)out, out_stride);
    else hipLaunchKernelGGL((scores_join_kernel<AS_F16>), grid, dim3(256), 0, ctx->stream, s.part, f.supers, m, a.v, (void *)out, out_stride);
    AS_HIP(ctx, hipGetLastError());
  }
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
    ctx_enter(ctx);
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
    ctx_enter(ctx);
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
