// Instances of the experts' products, one translation unit for each kind of operand (grouped_inst_*.hip).
#pragma once
#include "grouped_kernel.hpp"
#include "grouped_stream.hpp"

namespace cumpsgemm_amd {

struct GroupedTable {
  // [A K-contiguous][through registers, direct][tile]; B K-contiguous
  GroupedKernel columns[2][2][kGroupedClasses];
  GroupedKernel over_k[2][kGroupedClasses]; // ragged K, both row-contiguous
  GroupedKernel stream[2];                  // few tokens; [A K-contiguous]
};

template <Elem E, bool A_KC, bool B_KC, int BM, int BN, int WM, int WN, int ROW_BYTES, int NSTAGE, bool DIRECT, bool RAGGED_K,
          bool CAREFUL = false>
constexpr GroupedKernel grouped_of() {
  return grouped_entry<GroupedCfg<E, A_KC, B_KC, BM, BN, WM, WN, ROW_BYTES, NSTAGE, DIRECT, RAGGED_K, 2, CAREFUL>>();
}

template <Elem E> constexpr GroupedTable grouped_table_f32() {
  GroupedTable t{};
  t.columns[0][0][TILE_128] = grouped_of<E, false, true, 128, 128, 64, 32, 64, 2, false, false>();
  t.columns[1][0][TILE_128] = grouped_of<E, true, true, 128, 128, 64, 32, 64, 2, false, false>();
  t.columns[0][1][TILE_256] = grouped_of<E, false, true, 256, 128, 64, 64, 64, 2, true, false>();
  t.columns[0][1][TILE_128] = grouped_of<E, false, true, 128, 128, 64, 32, 64, 2, true, false>();
  t.columns[0][1][TILE_NARROW] = grouped_of<E, false, true, 128, 32, 32, 32, 64, 2, true, false>();
  t.columns[1][1][TILE_256] = grouped_of<E, true, true, 256, 128, 64, 64, 64, 2, true, false>();
  t.columns[1][1][TILE_128] = grouped_of<E, true, true, 128, 128, 64, 32, 64, 2, true, false>();
  t.columns[1][1][TILE_NARROW] = grouped_of<E, true, true, 128, 32, 32, 32, 64, 2, true, false>();
  t.over_k[0][TILE_128] = grouped_of<E, false, false, 128, 128, 64, 32, 64, 2, false, true>();
  t.over_k[1][TILE_256] = grouped_of<E, false, false, 256, 128, 64, 64, 64, 2, true, true>();
  t.over_k[1][TILE_128] = grouped_of<E, false, false, 128, 128, 64, 32, 64, 2, true, true>();
  t.stream[0] = stream_entry<E, false>();
  t.stream[1] = stream_entry<E, true>();
  return t;
}

template <Elem E> constexpr GroupedTable grouped_table_16() {
  GroupedTable t{};
  t.columns[0][0][TILE_128] = grouped_of<E, false, true, 128, 128, 64, 64, 128, 2, false, false>();
  t.columns[1][0][TILE_128] = grouped_of<E, true, true, 128, 128, 64, 64, 128, 2, false, false>();
  t.columns[0][1][TILE_256] = grouped_of<E, false, true, 256, 256, 128, 64, 128, 2, true, false>();
  t.columns[0][1][TILE_128] = grouped_of<E, false, true, 128, 128, 64, 64, 128, 2, true, false>();
  t.columns[0][1][TILE_NARROW] = grouped_of<E, false, true, 128, 32, 32, 32, 128, 4, true, false>();
  t.columns[1][1][TILE_256] = grouped_of<E, true, true, 256, 256, 128, 64, 128, 2, true, false>();
  t.columns[1][1][TILE_128] = grouped_of<E, true, true, 128, 128, 64, 64, 128, 2, true, false>();
  t.columns[1][1][TILE_NARROW] = grouped_of<E, true, true, 128, 32, 32, 32, 128, 4, true, false>();
  t.over_k[0][TILE_128] = grouped_of<E, false, false, 128, 128, 64, 64, 128, 2, false, true>();
  t.over_k[0][SHORT_LINES] = grouped_of<E, false, false, 128, 128, 64, 64, 128, 2, false, true, true>();
  t.over_k[1][TILE_256] = grouped_of<E, false, false, 256, 256, 128, 64, 128, 2, true, true>();
  t.over_k[1][TILE_128] = grouped_of<E, false, false, 128, 128, 64, 64, 128, 2, true, true>();
  t.stream[0] = stream_entry<E, false>();
  t.stream[1] = stream_entry<E, true>();
  return t;
}

template <Elem E> constexpr GroupedTable grouped_table_i8() {
  GroupedTable t{};
  t.columns[1][0][TILE_128] = grouped_of<E, true, true, 128, 128, 64, 64, 128, 2, false, false>();
  t.columns[1][1][TILE_256] = grouped_of<E, true, true, 256, 256, 128, 64, 128, 2, true, false>();
  t.columns[1][1][TILE_128] = grouped_of<E, true, true, 128, 128, 64, 64, 128, 2, true, false>();
  t.columns[1][1][TILE_NARROW] = grouped_of<E, true, true, 128, 32, 32, 32, 128, 4, true, false>();
  t.stream[1] = stream_entry<E, true>();
  return t;
}

#define CUMPSGEMM_GROUPED_F32(sym, E) GroupedTable sym = grouped_table_f32<E>();
#define CUMPSGEMM_GROUPED_16(sym, E) GroupedTable sym = grouped_table_16<E>();
#define CUMPSGEMM_GROUPED_I8(sym, E) GroupedTable sym = grouped_table_i8<E>();

} // namespace cumpsgemm_amd
