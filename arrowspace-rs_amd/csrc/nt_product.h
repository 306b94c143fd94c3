// nt_product.h -- the tiled product C[n][m] = sum_k A[m][k] B[n][k], 16-bit elements, f32 sums, on the matrix pipe; each operand's
// matrix lies with its rows along k, or transposed, a row per k.  The softmax cross entropy of table_loss.hip is four such products
// with different endings (logits -> statistics, logits -> gradient of the logits, and the two gradients), so the walk over k is here
// once.
//
// Tile.  A workgroup of WM x WN waves owns (16 TM WM) x (16 TN WN) of the output; a wave holds TM x TN accumulators of the
// 16 x 16 x 32 instruction.  Per 64 k a wave of 8 x 4 reads (8 + 4) x 2 KB of LDS for 64 instructions of 16 cycles: the
// workgroup of eight waves needs 1 536 cycles of LDS (128 B a cycle) for 2 048 cycles of matrix work a SIMD; a square 4 x 4 wave
// needs 512 for 512, which is why the large tile is taken wherever the output has enough of them (product_tile in table_loss.hip).
// Measured: 1 024 x 16 384 x 8 192, 208 us = 1 320 TFLOP/s, as the library's product of this size.  Four buffers of half the
// depth with the waves of a SIMD half a step apart (one reads while the other multiplies): 209 us, not kept.
// Staging.  Both operands come by direct loads into LDS, 16 B a lane, two buffers: while one is contracted the other fills; one
// barrier a step, in front of which a wave waits for its own loads (they had a whole step to land).
// Banks.  Rows along k: a row of a stage is 64 k = 128 B, all rows would start in one bank; the 16-byte piece c of row r lies at place
// c ^ (r & 7), chosen on the global side of the load (a direct load writes LDS linearly), so eight rows of a fragment read spread
// over all banks.  A row per k: a stage is 64 rows of the tile's width, read transposed (four rows' values of a column in a lane, two
// reads an operand); piece c of row r lies at c ^ 4 (r & 3), so the four rows of a read do.
// Rows of the output.  Accumulator (i, e) of lane group q holds output row 16 i + 4 q + e of the instruction.  The stage is filled (or
// read) so that tiles 2 j and 2 j + 1 interleave: a lane's 2 x 4 values are EIGHT consecutive rows (columns likewise over pairs of lanes'
// quads), so that every ending stores 16 bytes a lane.
#pragma once

#include "table_common.h"

namespace asx {

typedef __attribute__((address_space(3))) void nt_lds;
typedef const __attribute__((address_space(1))) void nt_gbl;

struct NtOperand {
  const char *p;      // this workgroup's side: its first row (or column, transposed)
  size_t ld;          // bytes from row to row of the matrix
  uint32_t last;      // rows behind this one read it instead (their results are dropped); transposed: 16-byte pieces of a row
  uint32_t last_k;    // transposed: rows behind this one read it instead (the other operand has zeros there)
  size_t plane;       // bytes from plane to plane (f32: three bf16, table_loss_rows.h)
};

template <int FMT>  // AS_BF16 / AS_F16
__device__ __forceinline__ f32x4 nt_mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (FMT == AS_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t nt_min(uint32_t a, uint32_t b) { return a < b ? a : b; }
// row of the output that LDS row R of a side holds
__device__ __forceinline__ uint32_t nt_row(uint32_t R) {
  const uint32_t i = R >> 4, r = R & 15;
  return ((i >> 1) << 5) + ((r >> 2) << 3) + ((i & 1) << 2) + (r & 3);
}

// Four fragments (16 rows apart: 2 048 B) from one address.  Behind a direct load in flight hipcc waits for it in front of every
// LDS read it knows of (it cannot tell the two buffers apart), so the reads are written out, each batch with its own wait.
__device__ __forceinline__ void nt_read8(u32x4 &a0, u32x4 &a1, u32x4 &a2, u32x4 &a3, u32x4 &b0, u32x4 &b1, u32x4 &b2, u32x4 &b3, uint32_t aa, uint32_t ba) {
  asm volatile(
      "ds_read_b128 %4, %9\n\tds_read_b128 %5, %9 offset:2048\n\tds_read_b128 %6, %9 offset:4096\n\tds_read_b128 %7, %9 offset:6144\n\t"
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %8 offset:2048\n\tds_read_b128 %2, %8 offset:4096\n\tds_read_b128 %3, %8 offset:6144\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a0), "=&v"(a1), "=&v"(a2), "=&v"(a3), "=&v"(b0), "=&v"(b1), "=&v"(b2), "=&v"(b3)
      : "v"(aa), "v"(ba)
      : "memory");
}
__device__ __forceinline__ void nt_read4(u32x4 &a0, u32x4 &a1, u32x4 &a2, u32x4 &a3, uint32_t aa) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:2048\n\tds_read_b128 %2, %4 offset:4096\n\tds_read_b128 %3, %4 offset:6144\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a0), "=&v"(a1), "=&v"(a2), "=&v"(a3)
      : "v"(aa)
      : "memory");
}

// the same, one side or both transposed: 8-byte reads of rows 0 .. 3 and 4 .. 7 (AROW x 4 bytes on) of columns 0 .. 3 and 4 .. 7 of
// each eight, from two addresses (32 columns apart)
template <uint32_t FOUR>
__device__ __forceinline__ void nt_read_t(u32x2 (&x)[8], uint32_t a0, uint32_t a1) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\tds_read_b64_tr_b16 %2, %8 offset:8\n\tds_read_b64_tr_b16 %3, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %4, %9\n\tds_read_b64_tr_b16 %5, %9 offset:%10\n\tds_read_b64_tr_b16 %6, %9 offset:8\n\tds_read_b64_tr_b16 %7, %9 offset:%11\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
      : "v"(a0), "v"(a1), "n"(FOUR), "n"(FOUR + 8)
      : "memory");
}
template <uint32_t FOUR>
__device__ __forceinline__ void nt_read_tn(u32x2 (&x)[8], u32x4 (&b)[4], uint32_t a0, uint32_t a1, uint32_t ba) {
  asm volatile(
      "ds_read_b128 %8, %14\n\tds_read_b128 %9, %14 offset:2048\n\tds_read_b128 %10, %14 offset:4096\n\tds_read_b128 %11, %14 offset:6144\n\t"
      "ds_read_b64_tr_b16 %0, %12\n\tds_read_b64_tr_b16 %1, %12 offset:%15\n\tds_read_b64_tr_b16 %2, %12 offset:8\n\tds_read_b64_tr_b16 %3, %12 offset:%16\n\t"
      "ds_read_b64_tr_b16 %4, %13\n\tds_read_b64_tr_b16 %5, %13 offset:%15\n\tds_read_b64_tr_b16 %6, %13 offset:8\n\tds_read_b64_tr_b16 %7, %13 offset:%16\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3])
      : "v"(a0), "v"(a1), "v"(ba), "n"(FOUR), "n"(FOUR + 8)
      : "memory");
}
template <uint32_t FOURA, uint32_t FOURB>
__device__ __forceinline__ void nt_read_tt(u32x2 (&x)[8], u32x2 (&y)[8], uint32_t a0, uint32_t a1, uint32_t b0, uint32_t b1) {
  asm volatile(
      "ds_read_b64_tr_b16 %8, %18\n\tds_read_b64_tr_b16 %9, %18 offset:%22\n\tds_read_b64_tr_b16 %10, %18 offset:8\n\tds_read_b64_tr_b16 %11, %18 offset:%23\n\t"
      "ds_read_b64_tr_b16 %12, %19\n\tds_read_b64_tr_b16 %13, %19 offset:%22\n\tds_read_b64_tr_b16 %14, %19 offset:8\n\tds_read_b64_tr_b16 %15, %19 offset:%23\n\t"
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%20\n\tds_read_b64_tr_b16 %2, %16 offset:8\n\tds_read_b64_tr_b16 %3, %16 offset:%21\n\t"
      "ds_read_b64_tr_b16 %4, %17\n\tds_read_b64_tr_b16 %5, %17 offset:%20\n\tds_read_b64_tr_b16 %6, %17 offset:8\n\tds_read_b64_tr_b16 %7, %17 offset:%21\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3]),
        "=&v"(y[4]), "=&v"(y[5]), "=&v"(y[6]), "=&v"(y[7])
      : "v"(a0), "v"(a1), "v"(b0), "v"(b1), "n"(FOURA), "n"(FOURA + 8), "n"(FOURB), "n"(FOURB + 8)
      : "memory");
}
// four operands from their halves
__device__ __forceinline__ void nt_join(u32x4 (&a)[4], const u32x2 (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = u32x4{x[2 * k][0], x[2 * k][1], x[2 * k + 1][0], x[2 * k + 1][1]};
}

// AT, BT: the operand's matrix has a row per k
template <int FMT, int TM_, int TN_, int WM_, int WN_, bool AT = false, bool BT = false>
struct NtTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr uint32_t BM = 16 * TM * WM, BN = 16 * TN * WN, NT = 64 * WM * WN;
  static constexpr int kStage = (BM + BN) * 128;  // bytes of one buffer
  static constexpr uint32_t PA = BM * 8 / NT, PB = BN * 8 / NT;  // 16-byte pieces a thread brings per step
  static_assert((TM == 4 || TM == 8) && TN == 4, "fragment batches of four");
  static_assert(PA * NT == BM * 8 && PB * NT == BN * 8, "whole passes");

  uint32_t lds;        // address of the two buffers
  uint32_t wave, lane;
  uint32_t fa, fb;     // this lane's fragment addresses within a buffer
  char *smem;

  // places of a transposed stage: W columns a row
  template <uint32_t W>
  __device__ __forceinline__ static uint32_t swizzle(uint32_t row) { return (row & 3) << (W >= 128 ? 2 : 1); }
  template <uint32_t W>
  __device__ __forceinline__ uint32_t column_address(uint32_t column0) const {
    const uint32_t q = lane >> 4, row = q * 8 + ((lane >> 2) & 3);
    return row * (W * 2) + (((column0 >> 3) + (lane & 3)) ^ swizzle<W>(row)) * 16;
  }
  __device__ __forceinline__ void init(char *shared) {
    smem = shared;
    lds = (uint32_t)(size_t)(nt_lds *)shared;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    const uint32_t r = lane & 15, q = lane >> 4;
    const uint32_t piece = ((q ^ (r & 7)) << 4);
    const uint32_t ra = (wave / WN) * (TM * 16), rb = (wave % WN) * (TN * 16);
    fa = AT ? column_address<BM>(ra) : (ra + r) * 128 + piece;
    fb = BM * 128 + (BT ? column_address<BN>(rb) : (rb + r) * 128 + piece);
  }
  // Step s of `steps` a pair of planes; three planes: the pairs (A, B) 00, 01, 10, 11, 02, 20.
  template <bool T, uint32_t W, uint32_t PIECES>
  __device__ __forceinline__ void fetch_side(char *dst, const NtOperand &o, uint32_t k, uint32_t plane) const {
    const char *src = o.p + plane * o.plane + (T ? 0 : (size_t)k * 128);
#pragma unroll
    for (uint32_t p = 0; p < PIECES; ++p) {
      const char *from;
      if constexpr (T) {
        const uint32_t idx = p * NT + threadIdx.x, row = idx / (W / 8), slot = idx % (W / 8);
        from = src + (size_t)nt_min(k * 64 + row, o.last_k) * o.ld + nt_min(slot ^ swizzle<W>(row), o.last) * 16;
      } else {
        const uint32_t R = p * (NT / 8) + (threadIdx.x >> 3);
        from = src + (size_t)nt_min(nt_row(R), o.last) * o.ld + (((threadIdx.x & 7) ^ (R & 7)) << 4);
      }
      __builtin_amdgcn_global_load_lds((nt_gbl *)from, (nt_lds *)(dst + (p * NT + wave * 64) * 16), 16, 0, 0);
    }
  }
  __device__ __forceinline__ void fetch(int buf, const NtOperand &A, const NtOperand &B, uint32_t s, uint32_t steps) const {
    char *dst = smem + buf * kStage;
    const uint32_t pair = s < steps ? 0 : s / steps, k = s - pair * steps;
    fetch_side<AT, BM, PA>(dst, A, k, 0x850u >> (2 * pair) & 3);
    fetch_side<BT, BN, PB>(dst + BM * 128, B, k, 0x244u >> (2 * pair) & 3);
  }
  __device__ __forceinline__ void zero(f32x4 (&acc)[TM][TN]) const {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void contract(int buf, f32x4 (&acc)[TM][TN]) const {
    const uint32_t base = lds + buf * kStage;
    constexpr uint32_t FA = BM * 8, FB = BN * 8;  // transposed: four rows
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 a[4], b[4];
      const uint32_t aa = AT ? base + fa + h * (64 * BM) : (base + fa) ^ (h * 64), ba = BT ? base + fb + h * (64 * BN) : (base + fb) ^ (h * 64);
      if constexpr (AT && BT) {
        u32x2 x[8], y[8];
        nt_read_tt<FA, FB>(x, y, aa, aa ^ 64, ba, ba ^ 64);
        nt_join(a, x);
        nt_join(b, y);
      } else if constexpr (AT) {
        u32x2 x[8];
        nt_read_tn<FA>(x, b, aa, aa ^ 64, ba);
        nt_join(a, x);
      } else {
        nt_read8(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], aa, ba);
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = nt_mfma<FMT>(a[i], b[j], acc[i][j]);
      __builtin_amdgcn_s_setprio(0);
      if constexpr (TM == 8) {
        if constexpr (AT) {
          u32x2 x[8];
          nt_read_t<FA>(x, aa ^ 128, aa ^ 192);
          nt_join(a, x);
        } else {
          nt_read4(a[0], a[1], a[2], a[3], aa + 8192);
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[4 + i][j] = nt_mfma<FMT>(a[i], b[j], acc[4 + i][j]);
        __builtin_amdgcn_s_setprio(0);
      }
    }
  }
  // one step's turn: everyone has its part of the stage in LDS, and has left the other buffer
  __device__ __forceinline__ static void turn() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
};

}  // namespace asx
