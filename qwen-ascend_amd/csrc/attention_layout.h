// How the keys and values of a tile are held: heads in blocks of 32 elements, rows in LDS, the
// 16-byte pieces that lanes load. Plain C++ but for its qualifiers.
#pragma once
#ifdef __HIP__
#include "qmoe_common.h"
#else
#define QMOE_HOST_DEV inline
#endif

// Heads of up to 32 * NK elements. In LDS rows are DP elements apart; the 16-byte pieces of a row are XOR'd with
// its number, so that what one instruction reads of many rows spreads over the banks: rows of K one piece
// each, rows of V 64 bytes each.
template <int NK>
struct Layout {
  static constexpr int DC = 32 * NK, D_LEAST = NK == 2 ? 8 : NK == 3 ? 72 : NK == 4 ? 104 : NK == 6 ? 136 : 200;
  static constexpr int DP = NK <= 2 ? 64 : NK <= 4 ? 128 : 256, STRIDE = 2 * DP;
  static constexpr int PIECES = DP / 8, RPI = 64 / PIECES;  // rows of a wave's load instruction
  static constexpr int TILE = 64 * STRIDE, LDS = 4 * TILE;
  QMOE_HOST_DEV static constexpr bool always(int ks) { return 16 * ks + 15 < D_LEAST; }  // within every such head
  QMOE_HOST_DEV static constexpr int k_swizzle(int row) { return DP == 64 ? (row >> 1) & 7 : DP == 128 ? row & 15 : row & 7; }
  QMOE_HOST_DEV static constexpr int v_swizzle(int row) { return DP == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3); }
  // The piece of a head of D elements (FULL: of DC) that a lane loads to its place in LDS, in row `row` of the tile.
  // Rows in LDS are wider than heads of other sizes than 64, 128 and 256: the lanes behind a head's pieces load its
  // last one again, as what follows it may lie behind the cache.
  template <bool FULL, bool KEYS>
  QMOE_HOST_DEV static constexpr int piece_of(int lane, int row, int D) {
    const int piece = (lane % PIECES) ^ (KEYS ? k_swizzle(row) : v_swizzle(row)), last = (FULL ? DC : D) / 8 - 1;
    return (FULL && DC == DP) || piece < last ? piece : last;
  }
};

// NK of heads of D elements.
QMOE_HOST_DEV constexpr int blocks_of(int D) { return D <= 64 ? 2 : D <= 96 ? 3 : D <= 128 ? 4 : D <= 192 ? 6 : 8; }
