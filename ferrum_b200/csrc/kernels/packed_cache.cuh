// The layout of a cache held in 4 bits, shared by the kernels that write and read it.
//
// A page of a KV head is page_size / 16 blocks of 16 positions.  A block is one run of bytes: the codes of the 16 keys (D / 2 bytes a
// position), the codes of the 16 values, a (step, middle) pair of the cache's 16-bit type per 64 elements of every key, the same of
// every value: 18 * D bytes, a multiple of 128, so that one bulk copy brings all that 16 positions of a head consist of.  Nibble i of a row
// (low half of a byte first) is element i; it stands for middle + step * (code - 8): 4.5 bits an element.
#pragma once
#include "common.cuh"

constexpr int PACKED_POS = 16;      // positions of a block
constexpr int PACKED_GROUP = 64;    // elements that share a step and a middle

template <int D>
struct PackedBlock {
  static constexpr int ROW = D / 2;                        // bytes of a position's codes
  static constexpr int GROUPS = D / PACKED_GROUP;
  static constexpr int V_CODES = PACKED_POS * ROW;         // byte offsets in a block
  static constexpr int K_PAIRS = 2 * V_CODES;
  static constexpr int V_PAIRS = K_PAIRS + PACKED_POS * GROUPS * 4;
  static constexpr int BYTES = V_PAIRS + PACKED_POS * GROUPS * 4;
};
static_assert(PackedBlock<64>::BYTES == 18 * 64 && PackedBlock<128>::BYTES == 18 * 128, "packed block size");

// Requests with at most this many packed rows (tokens x query heads of a KV head) in a step are decoded ones: they are read straight
// from the packed pages.
constexpr int PACKED_FEW_ROWS = 16;

inline bool packed_page_ok(int page_size) { return page_size > 0 && page_size % PACKED_POS == 0; }
