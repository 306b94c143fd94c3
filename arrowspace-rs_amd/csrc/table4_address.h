// table4_address.h -- where the scores of a table in 4 bits (table4.hip) read rows in memory.  Plain C++ (constexpr: host and device), so
// that the bounds are tested without a GPU.
#pragma once

#include <cstddef>
#include <cstdint>

namespace asx {

// Bytes from the first row to the 16-byte piece that lane group q of a wave reads of a row: `row_at` to the row's start, `group_at` from
// there to the group's piece of the first step, `k` on to its step; `in_row` is what lies in front of the group's piece in a plain row and
// `k_bytes` what is there of a row.  A piece that is not there is read where the row starts, and dropped.
constexpr bool row_piece_there(uint32_t in_row, uint32_t k, uint32_t k_bytes) { return in_row + k < k_bytes; }
constexpr size_t row_piece_at(size_t row_at, uint32_t group_at, uint32_t in_row, uint32_t k, uint32_t k_bytes) {
  return row_at + (row_piece_there(in_row, k, k_bytes) ? group_at + k : 0u);
}

}  // namespace asx
