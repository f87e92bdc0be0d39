// Products of experts' layers: what the kernels take, and who launches them.
//
//   ragged columns (gemm_grouped, gemm_i8): C[:, j] = alpha op(A_g) B[:, j] + beta C[:, j]   for j in group g
//   ragged K (gemm_grouped_k):              C_g     = alpha A[:, g] B[:, g]^T + beta C_g
//
// Column-major throughout.  Where a group begins and ends is read from device memory by the kernels themselves
// (offsets[g], offsets[g + 1], brought into [0, count] and into order there, so that no value of them leads out of
// the operands): a call waits for nothing and can be captured into a graph.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cumpsgemm_amd {

// What a kernel multiplies: FP32 in one of the four splits (gemm_kernel.hpp), FP16, BF16 or 8-bit integers.
enum class Elem : int { F32_FP16TCEC = 0, F32_FP16TC = 1, F32_BF16X3 = 2, F32_BF16X2 = 3, F16 = 4, BF16 = 5, I8 = 6 };
constexpr int kNumElems = 7;

enum GroupedOut : uint32_t { OUT_F32 = 0, OUT_F16 = 1, OUT_BF16 = 2 };

struct GroupedArgs {
  uint32_t m, n, k;         // n (ragged K: k) counts the tokens of all groups
  uint32_t groups;
  const int *offsets;       // [groups + 1] in device memory; null: one group of everything
  const char *a, *b;
  char *c;
  uint64_t lda, ldb, ldc;   // in elements
  uint64_t stride_a;        // between the groups' A (ragged K: unused)
  uint64_t stride_c;        // between the groups' C (ragged K only)
  float alpha, beta;
  uint32_t out;             // GroupedOut
  uint32_t vec_c;           // four results of a column can be stored at once
  const float *scale_a;     // 8-bit integers: [groups][m] and [n]
  const float *scale_b;
  // ragged K: each group's K in this many parts of whole steps, whose sums go to `partial` as whole tiles, [group]
  // [tile column][tile row][part][column of the tile][row of the tile], and are added in that order by a second launch
  uint32_t splits;          // 1: none
  float *partial;
};

struct GroupedKernel {
  void (*launch)(const GroupedArgs &, uint32_t workgroups, hipStream_t);
  int bm, bn;
};

// Kernels of ragged columns: three tiles of the tiled kernel, from the largest, and the kernel of few tokens to a group
// (grouped_stream.hpp).  Ragged K: the first two, and one for matrices of fewer than eight 16-bit rows or columns.
enum KernelClass : int { TILE_256 = 0, TILE_128 = 1, TILE_NARROW = 2, SHORT_LINES = 2, kGroupedClasses = 3, STREAM = 3 };

// Ragged K: how the lists of tiles, one for each group and part of its K, are dealt to the eight XCDs.  Each list is cut
// into 2^log2_shares shares of at most `most` tiles; one after the other goes to the XCDs in turns of eight.
struct DealOverK {
  uint32_t log2_shares, most;
};
__host__ __device__ inline DealOverK deal_over_k(uint32_t tiles, uint64_t lists, uint32_t groups) {
  // Groups differ in length, and four shares or more to an XCD even that out; a share is as large as that allows, since
  // its tiles read the same operands.
  const uint32_t all = groups == 1 ? 8 : 32;
  uint32_t log2_shares = 0;
  while (log2_shares < 3 && (lists << log2_shares) < all) log2_shares++;
  return {log2_shares, (tiles + (1u << log2_shares) - 1) >> log2_shares};
}
inline uint64_t workgroups_over_k(uint32_t tiles, uint64_t lists, uint32_t groups) {
  const DealOverK d = deal_over_k(tiles, lists, groups);
  return ((lists << d.log2_shares) + 7) / 8 * 8 * d.most;
}

// Adds the parts (bm x bn: the tile that they were computed with).
void launch_grouped_join(const GroupedArgs &args, int bm, int bn, hipStream_t stream);

} // namespace cumpsgemm_amd
