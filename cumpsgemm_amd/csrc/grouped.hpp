// Products of experts' layers: what the kernels take, and who launches them.
//
//   ragged columns (gemm_grouped, gemm_i8): C[:, j] = alpha op(A_g) B[:, j] + beta C[:, j]   for j in group g
//   ragged K (gemm_grouped_k):              C_g     = alpha A[:, g] B[:, g]^T + beta C_g
// and of gated feed-forward blocks, whose columns are ragged too, or all of one group:
//   projections (gemm_gated):               C[:, j] = act(G[:, j]) * U[:, j],  G = op(gate_g) B, U = op(up_g) B
//   their gradient (gemm_gated_backward):   dG = D * U * act'(G), dU = D * act(G),  D = op(A_g) B
//
// Column-major throughout.  Where a group begins and ends is read from device memory by the kernels themselves
// (offsets[g], offsets[g + 1], brought into [0, count] and into order there, so that no value of them leads out of
// the operands): a call waits for nothing and can be captured into a graph.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cumpsgemm_amd {

// What a kernel multiplies: FP32 in one of the four splits (gemm_kernel.hpp), FP16, BF16, 8-bit integers, or 8-bit floating
// point (f8_kernel.hpp), A in E4M3 and B in E4M3 or E5M2.
enum class Elem : int { F32_FP16TCEC = 0, F32_FP16TC = 1, F32_BF16X3 = 2, F32_BF16X2 = 3, F16 = 4, BF16 = 5, I8 = 6, E4M3 = 7, E5M2 = 8 };
constexpr int kNumElems = 9;

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
  // gated blocks.  Projections: `a` is the gate's matrix, `up` the other one, laid out like it; z[0], z[1]: where G and U go
  // (null: nowhere).  Gradient: z is read, d[0] and d[1] get dG and dU, c act(G) * U (null: nowhere).
  const char *up;
  char *z[2];
  char *d[2];
  uint64_t ldz, ldd;
  uint32_t act;             // cuMpSGEMM_activation_t
  // 8-bit floating point: one scale for 128 x 128 of A, as it is stored, and for 128 values of a column of B
  const float *scale_up;
  uint64_t stride_scale;    // between the groups' scales of A
  // ragged K: each group's K in this many parts of whole steps, whose sums go to `partial` as whole tiles, [group]
  // [tile column][tile row][part][column of the tile][row of the tile], and are added in that order by a second launch
  uint32_t splits;          // 1: none
  float *partial;
};

struct GroupedKernel {
  void (*launch)(const GroupedArgs &, uint32_t workgroups, hipStream_t);
  int bm, bn;
  int threads; // of a workgroup
};

// What becomes of the sums: C as they are, a gated block's result, or its gradient.  (STORE_EXACT, GATED_EXACT: the kernels of STORE
// and GATED for 8-bit floating point whose products are exact and summed in FP32, f8_kernel.hpp.)
enum class Epilogue : int { STORE = 0, GATED = 1, GATED_BACKWARD = 2, GATED_EXACT = 3, STORE_EXACT = 4 };

// Kernels of ragged columns: three tiles of the tiled kernel, from the largest, and the kernel of few tokens to a group
// (grouped_stream.hpp).  Gated blocks and 8-bit floating point: a tile of 64 tokens as well, three stages deep.  Ragged K: the first
// two, and one for matrices of fewer than eight 16-bit rows or columns.
enum KernelClass : int { TILE_256 = 0, TILE_128 = 1, TILE_NARROW = 2, SHORT_LINES = 2, STREAM = 3, TILE_64 = 4, kGroupedClasses = 5 };

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
