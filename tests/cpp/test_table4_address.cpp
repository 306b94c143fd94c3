// Every address that the scores of a table in 4 bits form for f16 rows read as they lie, against the rows' own bytes.
#include <cstdio>
#include <initializer_list>

#include "../../arrowspace-rs_amd/csrc/table4_address.h"

int main() {
  long wrong = 0, checked = 0;
  for (uint32_t d = 8; d <= 520; d += 8)
    for (uint32_t pad : {0u, 8u, 24u})
      for (uint32_t m = 1; m <= 16; ++m) {
        const size_t stride = (d + pad) * 2, end = (m - 1) * stride + d * 2;
        const uint32_t k_tiles = (d + 127) / 128;
        for (uint32_t lane = 0; lane < 64; ++lane) {
          const uint32_t col = lane & 15, q = lane >> 4, row = col < m ? col : m - 1;
          for (uint32_t kt = 0; kt < k_tiles; ++kt)
            for (uint32_t j = 0; j < 4; ++j) {
              const uint32_t k = kt * 256 + j * 64;
              const size_t at = asx::row_piece_at(row * stride, q * 16, q * 16, k, d * 2);
              const bool there = asx::row_piece_there(q * 16, k, d * 2);
              ++checked;
              if (at + 16 > end || at < row * stride || at + 16 > row * stride + d * 2) ++wrong;
              if (there != (kt * 128 + j * 32 + q * 8 < d) || (there && at != row * stride + (kt * 128 + j * 32 + q * 8) * 2)) ++wrong;
            }
        }
      }
  std::printf("%ld addresses, %ld wrong\n", checked, wrong);
  return wrong != 0;
}
