// nt_product.h -- the tiled product of two matrices whose rows both run along the contraction: C[n][m] = sum_k A[m][k] B[n][k],
// 16-bit elements, f32 sums, on the matrix pipe.  The softmax cross entropy of table_loss.hip is four such products with
// different endings (logits -> statistics, logits -> gradient of the logits, and the two gradients), so the walk over k is here once.
//
// Tile.  A workgroup of WM x WN waves owns (16 TM WM) x (16 TN WN) of the output; a wave holds TM x TN accumulators of the
// 16 x 16 x 32 instruction.  Per 64 k a wave of 8 x 4 reads (8 + 4) x 2 KB of LDS for 64 instructions of 16 cycles: the
// workgroup of eight waves needs 1 536 cycles of LDS (128 B a cycle) for 2 048 cycles of matrix work a SIMD; a square 4 x 4 wave
// needs 512 for 512, which is why the large tile is taken wherever the output has enough of them (tile_of in table_loss.hip).
// Staging.  Both operands come by direct loads into LDS, 16 B a lane, two buffers: while one is contracted the other fills; one
// barrier a step, in front of which a wave waits for its own loads (they had a whole step to land).
// Banks.  A row of a stage is 64 k = 128 B, all rows would start in one bank; the 16-byte piece c of row r lies at place
// c ^ (r & 7), chosen on the global side of the load (a direct load writes LDS linearly), so eight rows of a fragment read spread
// over all banks.
// Rows of the output.  Accumulator (i, e) of lane group q holds output row 16 i + 4 q + e of the instruction.  The stage is filled
// so that tiles 2 j and 2 j + 1 interleave: a lane's 2 x 4 values are EIGHT consecutive rows (columns likewise over pairs of lanes'
// quads), so that every ending stores 16 bytes a lane.
#pragma once

#include "table_common.h"

namespace asx {

typedef __attribute__((address_space(3))) void nt_lds;
typedef const __attribute__((address_space(1))) void nt_gbl;

struct NtOperand {
  const char *p;      // row 0 of this workgroup's side
  size_t ld;          // bytes from row to row
  uint32_t last;      // rows behind this one read it instead (their results are dropped)
  uint32_t plane;     // 64-wide steps from the high to the low plane (two planes: f32 values as a sum of two f16)
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

template <int FMT, int TM_, int TN_, int WM_, int WN_>
struct NtTile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr uint32_t BM = 16 * TM * WM, BN = 16 * TN * WN, NT = 64 * WM * WN;
  static constexpr int kStage = (BM + BN) * 128;  // bytes of one buffer
  static constexpr uint32_t PA = BM * 8 / NT, PB = BN * 8 / NT;  // 16-byte pieces a thread brings per step
  static_assert((TM == 4 || TM == 8) && TN == 4, "fragment batches of four");
  static_assert(PA * NT == BM * 8 && PB * NT == BN * 8, "whole passes");

  uint32_t lds;        // address of the two buffers
  uint32_t wave, lane;
  uint32_t fa, fb;     // this lane's fragment addresses within a buffer (step half 0; half 1 is ^ 64)
  char *smem;

  __device__ __forceinline__ void init(char *shared) {
    smem = shared;
    lds = (uint32_t)(size_t)(nt_lds *)shared;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63;
    const uint32_t r = lane & 15, q = lane >> 4;
    const uint32_t piece = ((q ^ (r & 7)) << 4);
    fa = ((wave / WN) * (TM * 16) + r) * 128 + piece;
    fb = (BM + (wave % WN) * (TN * 16) + r) * 128 + piece;
  }
  __device__ __forceinline__ void fetch(int buf, const NtOperand &A, const NtOperand &B, uint32_t acol, uint32_t bcol) const {
    char *dst = smem + buf * kStage;
#pragma unroll
    for (uint32_t p = 0; p < PA; ++p) {
      const uint32_t R = p * (NT / 8) + (threadIdx.x >> 3);
      const uint32_t row = nt_min(nt_row(R), A.last);
      __builtin_amdgcn_global_load_lds((nt_gbl *)(A.p + (size_t)acol * 128 + (size_t)row * A.ld + (((threadIdx.x & 7) ^ (R & 7)) << 4)),
                                       (nt_lds *)(dst + (p * NT + wave * 64) * 16), 16, 0, 0);
    }
#pragma unroll
    for (uint32_t p = 0; p < PB; ++p) {
      const uint32_t R = p * (NT / 8) + (threadIdx.x >> 3);
      const uint32_t row = nt_min(nt_row(R), B.last);
      __builtin_amdgcn_global_load_lds((nt_gbl *)(B.p + (size_t)bcol * 128 + (size_t)row * B.ld + (((threadIdx.x & 7) ^ (R & 7)) << 4)),
                                       (nt_lds *)(dst + BM * 128 + (p * NT + wave * 64) * 16), 16, 0, 0);
    }
  }
  __device__ __forceinline__ void zero(f32x4 (&acc)[TM][TN]) const {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void contract(int buf, f32x4 (&acc)[TM][TN]) const {
    const uint32_t base = lds + buf * kStage;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 a[4], b[4];
      nt_read8(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3], (base + fa) ^ (h * 64), (base + fb) ^ (h * 64));
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = nt_mfma<FMT>(a[i], b[j], acc[i][j]);
      __builtin_amdgcn_s_setprio(0);
      if constexpr (TM == 8) {
        nt_read4(a[0], a[1], a[2], a[3], ((base + fa) ^ (h * 64)) + 8192);
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

// the columns (64-wide steps) of step s of `steps`: with two planes high x high, high x low, low x high -- the product of the two low
// planes is 2^-24 of the whole and left out
__device__ __forceinline__ uint32_t nt_col_a(uint32_t s, uint32_t steps, uint32_t plane) { return s < steps ? s : s < 2 * steps ? s - steps : s - 2 * steps + plane; }
__device__ __forceinline__ uint32_t nt_col_b(uint32_t s, uint32_t steps, uint32_t plane) { return s < steps ? s : s < 2 * steps ? s - steps + plane : s - 2 * steps; }

}  // namespace asx
