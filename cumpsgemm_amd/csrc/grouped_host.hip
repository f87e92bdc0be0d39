// Experts' products: arguments, the choice of a kernel, launch.  See grouped.hpp.
#include "grouped_table.hpp"
#include "handle.hpp"
#include <algorithm>
#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_amd {

extern GroupedTable g_grouped_f32_fp16tcec, g_grouped_f32_fp16tc, g_grouped_f32_bf16x3, g_grouped_f32_bf16x2,
    g_grouped_f16, g_grouped_bf16, g_grouped_i8;

// direct: the operands can take the shorter way into LDS (grouped_kernel.hpp); the kernel of few tokens takes any
const GroupedKernel *lookup_grouped(Elem e, bool a_kc, bool ragged_k, bool direct, int cls) {
  static const GroupedTable *const tables[kNumElems] = {&g_grouped_f32_fp16tcec, &g_grouped_f32_fp16tc, &g_grouped_f32_bf16x3,
                                                        &g_grouped_f32_bf16x2, &g_grouped_f16, &g_grouped_bf16, &g_grouped_i8};
  const GroupedTable &t = *tables[(int)e];
  const GroupedKernel *k = ragged_k ? (cls == STREAM ? nullptr : &t.over_k[direct][cls])
                           : cls == STREAM ? &t.stream[a_kc] : &t.columns[a_kc][direct][cls];
  return k != nullptr && k->launch != nullptr ? k : nullptr;
}

// One thread: four rows of one column of a tile, the parts in their order.
__global__ __launch_bounds__(256) void grouped_join_kernel(const GroupedArgs args, const uint32_t bm, const uint32_t bn) {
  const uint32_t tiles_m = (args.m + bm - 1) / bm, tiles_n = (args.n + bn - 1) / bn, fours = bm * bn / 4;
  const uint32_t at = blockIdx.x % (fours / 256) * 256 + threadIdx.x; // of the tile's fours
  const uint64_t tile = blockIdx.x / (fours / 256);
  const uint32_t row = tile % tiles_m * bm + at % (bm / 4) * 4, col = tile / tiles_m % tiles_n * bn + at / (bm / 4);
  if (row >= args.m || col >= args.n) return;
  const float *p = args.partial + tile * args.splits * (bm * bn) + (uint64_t)at * 4;
  f4v_t x = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t s = 0; s < args.splits; s++) {
    const f4v_t y = *reinterpret_cast<const f4v_t *>(p + (uint64_t)s * (bm * bn));
#pragma unroll
    for (int v = 0; v < 4; v++) x[v] += y[v];
  }
#pragma unroll
  for (int v = 0; v < 4; v++) x[v] *= args.alpha;
  const uint64_t c = (tile / (tiles_m * tiles_n)) * args.stride_c + (uint64_t)col * args.ldc + row;
  const bool vec = args.vec_c != 0;
  if (args.out == OUT_F32) store_four<OUT_F32>(args.c + c * 4, x, args.beta, row, args.m, vec);
  else if (args.out == OUT_F16) store_four<OUT_F16>(args.c + c * 2, x, args.beta, row, args.m, vec);
  else store_four<OUT_BF16>(args.c + c * 2, x, args.beta, row, args.m, vec);
}

void launch_grouped_join(const GroupedArgs &args, int bm, int bn, hipStream_t stream) {
  const uint64_t tiles = (uint64_t)((args.m + bm - 1) / bm) * ((args.n + bn - 1) / bn) * args.groups;
  hipLaunchKernelGGL(grouped_join_kernel, dim3((uint32_t)(tiles * (bm * bn / 4 / 256))), dim3(256), 0, stream, args, (uint32_t)bm,
                     (uint32_t)bn);
}

namespace {

constexpr uint64_t kMost = 0x7fffffffull;
constexpr uint64_t kMostWorkgroups = 0xffffffffull / 512; // (a launch has fewer than 2^32 threads)

bool elem_of(hipDataType type, cuMpSGEMM_compute_mode_t mode, Elem &e) {
  if (type == HIP_R_16F) e = Elem::F16;
  else if (type == HIP_R_16BF) e = Elem::BF16;
  else if (type != HIP_R_32F) return false;
  else if (mode == CUMPSGEMM_FP16TCEC) e = Elem::F32_FP16TCEC;
  else if (mode == CUMPSGEMM_FP16TC) e = Elem::F32_FP16TC;
  else if (mode == CUMPSGEMM_TF32TCEC) e = Elem::F32_BF16X3;
  else if (mode == CUMPSGEMM_TF32TC) e = Elem::F32_BF16X2;
  else return false;
  return true;
}
bool out_of(hipDataType type, uint32_t &out) {
  if (type == HIP_R_32F) out = OUT_F32;
  else if (type == HIP_R_16F) out = OUT_F16;
  else if (type == HIP_R_16BF) out = OUT_BF16;
  else return false;
  return true;
}
uint32_t bytes_of(Elem e) { return (int)e <= 3 ? 4 : e == Elem::I8 ? 1 : 2; }

// Whether an operand can go straight from memory to LDS: its contiguous extent is whole 16-byte chunks, they are
// aligned, and the offsets of a tile and step fit 32 bits (`lines`: rows or K-lines that a step spans).
// FP32: the offsets alone.
bool chunks_ok(const void *p, uint64_t extent, uint64_t ld, uint64_t stride, uint32_t bytes, uint64_t lines) {
  if (bytes == 4) return lines * ld * bytes < 0x7fffffffull;
  return (uintptr_t)p % 16 == 0 && extent * bytes % 16 == 0 && ld * bytes % 16 == 0 && stride * bytes % 16 == 0 &&
         lines * ld * bytes < 0x7fffffffull;
}

bool four_at_once(const void *c, uint64_t m, uint64_t ldc, uint64_t stride, uint32_t out) {
  const uint32_t bytes = out == OUT_F32 ? 4 : 2;
  return (uintptr_t)c % (4 * bytes) == 0 && m % 4 == 0 && ldc % 4 == 0 && stride % 4 == 0;
}

hipblasStatus_t launched() {
  return hipGetLastError() == hipSuccess ? HIPBLAS_STATUS_SUCCESS : HIPBLAS_STATUS_EXECUTION_FAILED;
}

// What a kernel takes, in us: fixed + steps * part * max(alone, each * (workgroups / CUs + 0.2 of a round beyond the first)).
// alone: a step where a CU has one workgroup; each: of a workgroup's step where they queue; part: of a step for tiles with
// `filled` of their columns, least + (1 - least) * filled.  Fitted to 956 calls (m x k of 512^2 to 4096 x 2048, 1 - 64 groups
// of 1 - 8192 tokens, uneven by e^(0.4 N(0,1))) with every kernel in turn: op T, aligned operands, in BF16, 8 bits, FP16TCEC and
// TF32TCEC.  By tokens to a group alone (192, 48, 8) the choice lost 25, 28, 21 and 28 % against the best kernel there.  What it
// loses now, as a geometric mean over 235 calls of those sizes, %:
//                     BF16   8 bits   FP16TCEC   TF32TCEC   FP16TC   TF32TC
//   op T               3.2     2.9       2.8        2.7       4.4      2.6
//   op N               3.1                4.1        3.1       3.9      4.5
//   op T, unaligned   14.7     6.3
//   op N, unaligned    1.5
// Not fitted to, and it shows: op T unaligned with 1 - 8 tokens to a group, where the kernel of few tokens takes two to four
// times as long as the 128 x 128 tiles, at the aligned figures; and op N with 16 - 64 tokens in few groups, where it takes a
// third to two thirds of the others' time, but is counted too high (run_columns).
struct Cost {
  float fixed, alone, each;
  int slots, step; // workgroups to a CU; K-values of a step (the kernel of few tokens: of its eight waves)
  float least;
};
const Cost &cost_of(Elem e, int cls) {
  static const Cost sixteen[4] = {{4.4f, 1.38f, 2.33f, 1, 64, 0.46f}, {4.0f, 0.58f, 0.75f, 2, 64, 0.67f},
                                  {4.4f, 0.24f, 0.39f, 2, 64, 1.00f}, {3.4f, 0.90f, 0.96f, 2, 512, 0.41f}};
  static const Cost eight[4] = {{6.5f, 1.87f, 3.02f, 1, 128, 0.27f}, {5.4f, 0.72f, 0.94f, 2, 128, 0.41f},
                                {4.7f, 0.24f, 0.42f, 2, 128, 0.87f}, {3.1f, 1.14f, 1.01f, 2, 1024, 0.46f}};
  static const Cost fp32[4] = {{8.1f, 1.03f, 1.71f, 1, 32, 0.61f}, {5.9f, 0.62f, 0.91f, 1, 32, 0.62f},
                               {6.1f, 0.45f, 0.49f, 3, 32, 1.00f}, {4.0f, 0.90f, 0.99f, 2, 256, 0.42f}};
  static const Cost fp32x3[4] = {{11.1f, 1.93f, 2.64f, 1, 32, 0.42f}, {7.2f, 1.06f, 1.40f, 1, 32, 0.57f},
                                 {5.8f, 0.78f, 0.61f, 2, 32, 0.88f}, {4.1f, 0.89f, 0.98f, 2, 256, 0.43f}};
  return (e == Elem::I8 ? eight : e == Elem::F32_BF16X3 ? fp32x3 : (int)e <= 3 ? fp32 : sixteen)[cls];
}
double cost_us(const Cost &c, double workgroups, double steps, double cus, double filled = 1.0) {
  return c.fixed + steps * (c.least + (1.0 - c.least) * filled) * std::max<double>(c.alone, c.each * (workgroups / cus + (workgroups > cus * c.slots ? 0.2 * c.slots : 0.0)));
}
// For products over K (342 calls, 1 - 64 groups of 16 - 16384 tokens, results of 256^2 - 4096 x 2048, K in 1 - 16 parts, both
// tiles; BF16, FP16TCEC and TF32TCEC, aligned), whose groups often have a few steps only: every round of tiles also costs
// `round`, their first loads and the write-out; a group's K can be longer than the average one's, which counts where a CU
// has one workgroup; and parts are written and read once more, at 5.3 TB/s.  Loses 1.4 % (BF16), 2.0 % (FP16TCEC) and 0.4 % (TF32TCEC); without `round`
// 3.6, 2.4 and 0.8 %.
struct CostOverK {
  float fixed, alone, each, round;
  int slots, step;
};
double cost_over_k_us(Elem e, int cls, double tiles, double tile_bytes, double k, bool groups, uint32_t splits, double cus) {
  static const CostOverK sixteen[2] = {{12.3f, 1.29f, 1.57f, 15.8f, 1, 64}, {6.0f, 0.70f, 0.47f, 3.8f, 2, 64}};
  static const CostOverK fp32[2] = {{10.8f, 1.18f, 1.43f, 10.9f, 1, 32}, {6.7f, 0.76f, 0.83f, 5.3f, 1, 32}};
  static const CostOverK fp32x3[2] = {{13.9f, 1.94f, 2.29f, 14.9f, 1, 32}, {6.5f, 1.13f, 1.25f, 5.1f, 1, 32}};
  const CostOverK &c = (e == Elem::F32_BF16X3 ? fp32x3 : (int)e <= 3 ? fp32 : sixteen)[cls];
  const double steps = k / c.step + 0.5, workgroups = tiles * splits, rounds = workgroups / cus;
  if (splits > 1 && steps < 2.0 * splits) return 1e30; // (two steps to a part, at least)
  return c.fixed + c.round * std::max(0.0, rounds - 1.0) +
         steps / splits * std::max<double>(c.alone * (groups ? 1.6 : 1.0), c.each * (rounds + (rounds > c.slots ? 0.1 * c.slots : 0.0))) +
         (splits == 1 ? 0.0 : 3.0 + tiles * tile_bytes * (splits + 1) / 5.3e6);
}
// CUMPSGEMM_FORCE_TILE_CLASS goes before the rule where there is such a kernel.
bool forced(Elem e, bool a_kc, bool ragged_k, bool direct, int &cls) {
  const int want = tuning().force_cls;
  if (want < 0 || want > STREAM || (ragged_k && want == SHORT_LINES) || lookup_grouped(e, a_kc, ragged_k, direct, want) == nullptr) return false;
  cls = want;
  return true;
}

// Ragged columns: no more tiles than this, where every group has a column of them that is not full.
uint64_t most_tiles(const GroupedArgs &args, const GroupedKernel &k) {
  const uint64_t columns = args.offsets == nullptr ? (args.n + k.bn - 1) / k.bn
                                                   : (uint64_t)args.n / k.bn + std::min(args.n, args.groups);
  return columns * ((args.m + k.bm - 1) / k.bm);
}

// Ragged columns: B and C have args.n columns in args.groups groups.
hipblasStatus_t run_columns(cuMpSGEMM_handle *h, Elem e, bool a_kc, GroupedArgs &args, const char *label) {
  const uint32_t bytes = bytes_of(e);
  const bool direct = chunks_ok(args.a, a_kc ? args.k : args.m, args.lda, args.stride_a, bytes, a_kc ? 256 : 64) &&
                      chunks_ok(args.b, args.k, args.ldb, 0, bytes, 256);
  int cls = TILE_128;
  if (bytes == 2 && !direct && !a_kc && args.m < 8) {
    cls = STREAM; // (a line is shorter than the chunks that the tiled kernels read)
  } else if (!forced(e, a_kc, false, direct, cls)) {
    double best = 0.0;
    for (int c = TILE_256; c <= STREAM; c++) {
      const GroupedKernel *const kern = lookup_grouped(e, a_kc, false, direct, c);
      if (kern == nullptr || most_tiles(args, *kern) > kMostWorkgroups) continue;
      // columns of tiles, the groups' sizes being unknown here: half of each group's last one, or one for each group
      const double some = std::min(args.n, args.groups), each = (double)args.n / args.groups;
      const double columns = args.groups == 1 ? (args.n + kern->bn - 1) / kern->bn
                             : each < kern->bn / 2 ? some : (double)args.n / kern->bn + 0.5 * some;
      const Cost &cost = cost_of(e, c);
      // (the kernel of few tokens: in workgroups of 16 rows, as fitted with op T; where rows are contiguous it has 64 in one,
      // and this is too high)
      const double rows = c == STREAM ? (args.m + 15) / 16 : (args.m + kern->bm - 1) / kern->bm;
      const double us = cost_us(cost, columns * rows, (args.k + cost.step - 1) / cost.step, h->num_cus,
                                std::min(1.0, each / kern->bn));
      if (best == 0.0 || us < best) best = us, cls = c;
    }
  }
  const GroupedKernel *k = lookup_grouped(e, a_kc, false, direct, cls);
  if (k == nullptr) return HIPBLAS_STATUS_INTERNAL_ERROR;
  const uint64_t workgroups = most_tiles(args, *k);
  if (workgroups > kMostWorkgroups) return HIPBLAS_STATUS_INVALID_VALUE;
  ProfileScope prof(h, label);
  k->launch(args, (uint32_t)workgroups, h->stream);
  return launched();
}
} // namespace
} // namespace cumpsgemm_amd

using namespace cumpsgemm_amd;
extern "C" {

hipblasStatus_t cuMpSGEMM_gemm_grouped(cuMpSGEMM_handle_t h, hipblasOperation_t op_A, uint64_t m, uint64_t n, uint64_t k,
                                       const float *alpha, const void *a, uint64_t lda, uint64_t stridea, const void *b,
                                       uint64_t ldb, const float *beta, void *c, uint64_t ldc, const int *offsets,
                                       uint64_t group_count, cuMpSGEMM_compute_mode_t mode, hipDataType type_ab,
                                       hipDataType type_c) {
  if (h == nullptr || alpha == nullptr || beta == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (op_A != HIPBLAS_OP_N && op_A != HIPBLAS_OP_T && op_A != HIPBLAS_OP_C) return HIPBLAS_STATUS_INVALID_VALUE;
  if (m > kMost || n > kMost || k > kMost || group_count > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
  Elem e;
  uint32_t out;
  if (!elem_of(type_ab, mode, e) || !out_of(type_c, out) || (type_c != type_ab && type_c != HIP_R_32F))
    return HIPBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || group_count == 0) return HIPBLAS_STATUS_SUCCESS;
  const bool a_kc = op_A != HIPBLAS_OP_N;
  if (ldc < m || c == nullptr || offsets == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (k != 0 && (lda < (a_kc ? k : m) || ldb < k || a == nullptr || b == nullptr)) return HIPBLAS_STATUS_INVALID_VALUE;
  GroupedArgs args{};
  args.m = (uint32_t)m;
  args.n = (uint32_t)n;
  args.k = (uint32_t)k;
  args.groups = (uint32_t)group_count;
  args.offsets = offsets;
  args.a = (const char *)a;
  args.b = (const char *)b;
  args.c = (char *)c;
  args.lda = lda;
  args.ldb = ldb;
  args.ldc = ldc;
  args.stride_a = stridea;
  args.alpha = *alpha;
  args.beta = *beta;
  args.out = out;
  args.vec_c = four_at_once(c, m, ldc, 0, out);
  return run_columns(h, e, a_kc, args, "gemm_grouped");
}

hipblasStatus_t cuMpSGEMM_gemm_grouped_k(cuMpSGEMM_handle_t h, uint64_t m, uint64_t n, uint64_t k, const float *alpha,
                                         const void *a, uint64_t lda, const void *b, uint64_t ldb, const float *beta, void *c,
                                         uint64_t ldc, uint64_t stridec, const int *offsets, uint64_t group_count,
                                         cuMpSGEMM_compute_mode_t mode, hipDataType type_ab, hipDataType type_c) {
  if (h == nullptr || alpha == nullptr || beta == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (m > kMost || n > kMost || k > kMost || group_count > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
  Elem e;
  uint32_t out;
  if (!elem_of(type_ab, mode, e) || !out_of(type_c, out) || (type_c != type_ab && type_c != HIP_R_32F))
    return HIPBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || group_count == 0) return HIPBLAS_STATUS_SUCCESS;
  if (ldc < m || c == nullptr || offsets == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (group_count > 1 && stridec < ldc * (n - 1) + m) return HIPBLAS_STATUS_INVALID_VALUE; // (groups' results overlap)
  if (k != 0 && (lda < m || ldb < n || a == nullptr || b == nullptr)) return HIPBLAS_STATUS_INVALID_VALUE;
  GroupedArgs args{};
  args.m = (uint32_t)m;
  args.n = (uint32_t)n;
  args.k = (uint32_t)k;
  args.groups = (uint32_t)group_count;
  args.offsets = offsets;
  args.a = (const char *)a;
  args.b = (const char *)b;
  args.c = (char *)c;
  args.lda = lda;
  args.ldb = ldb;
  args.ldc = ldc;
  args.stride_c = stridec;
  args.alpha = *alpha;
  args.beta = *beta;
  args.out = out;
  args.vec_c = four_at_once(c, m, ldc, stridec, out);
  const uint32_t bytes = bytes_of(e);
  const bool direct = chunks_ok(a, m, lda, 0, bytes, 64) && chunks_ok(b, n, ldb, 0, bytes, 64);
  // The tile, and in how many parts K is taken: at least two steps to a part.
  int cls = TILE_128;
  args.splits = 1;
  const bool short_lines = bytes == 2 && !direct && (m < 8 || n < 8);
  if (short_lines) cls = SHORT_LINES;
  const bool fixed_cls = short_lines || forced(e, false, true, direct, cls);
  double best = 0.0;
  for (int c = fixed_cls ? cls : (int)TILE_256; c <= (fixed_cls ? cls : (int)TILE_128); c++) {
    const GroupedKernel *const kern = lookup_grouped(e, false, true, direct, c);
    if (kern == nullptr) continue;
    const double tiles = (double)((m + kern->bm - 1) / kern->bm) * ((n + kern->bn - 1) / kern->bn) * group_count;
    for (uint32_t s = 1; s <= 16; s *= 2) {
      if (s > 1 && tiles * s > 8.0 * h->num_cus) break;
      const double us = cost_over_k_us(e, c == SHORT_LINES ? (int)TILE_128 : c, tiles, kern->bm * kern->bn * 4.0,
                                       (double)k / group_count, group_count > 1, s, h->num_cus);
      if (best == 0.0 || us < best) best = us, cls = c, args.splits = s;
    }
  }
  if (tuning().force_split > 0) args.splits = (uint32_t)std::min(tuning().force_split, 64);
  const GroupedKernel *const kern = lookup_grouped(e, false, true, direct, cls);
  if (kern == nullptr) return HIPBLAS_STATUS_INTERNAL_ERROR;
  const uint64_t per = ((m + kern->bm - 1) / kern->bm) * ((n + kern->bn - 1) / kern->bn);
  if (per > kMostWorkgroups || per * group_count > kMostWorkgroups) return HIPBLAS_STATUS_INVALID_VALUE;
  // (the launch that joins the parts has up to 64 workgroups to a tile)
  if (per * group_count > kMostWorkgroups / 64) args.splits = 1;
  if (args.splits > 1) {
    bool failed = false;
    args.partial = (float *)ensure_pack_workspace(h, per * group_count * args.splits * kern->bm * kern->bn * 4, &failed);
    if (failed) return HIPBLAS_STATUS_EXECUTION_FAILED;
    if (args.partial == nullptr) args.splits = 1; // (no memory, or a graph is being captured)
  }
  const uint64_t workgroups = workgroups_over_k((uint32_t)per, group_count * args.splits, args.groups);
  if (workgroups > kMostWorkgroups) return HIPBLAS_STATUS_INVALID_VALUE;
  ProfileScope prof(h, "gemm_grouped_k");
  kern->launch(args, (uint32_t)workgroups, h->stream);
  if (args.splits > 1) launch_grouped_join(args, kern->bm, kern->bn, h->stream);
  return launched();
}

hipblasStatus_t cuMpSGEMM_gemm_i8(cuMpSGEMM_handle_t h, uint64_t m, uint64_t n, uint64_t k, const int8_t *a, uint64_t lda,
                                  uint64_t stridea, const float *scale_a, const int8_t *b, uint64_t ldb, const float *scale_b,
                                  void *c, uint64_t ldc, hipDataType type_c, const int *offsets, uint64_t group_count) {
  if (h == nullptr || m > kMost || n > kMost || group_count > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
  // (128 * 128 * 131072 is 2^31: a longer sum might not fit 32 bits)
  if (k > 131071) return HIPBLAS_STATUS_INVALID_VALUE;
  uint32_t out;
  if (!out_of(type_c, out)) return HIPBLAS_STATUS_INVALID_VALUE;
  if (m == 0 || n == 0 || group_count == 0) return HIPBLAS_STATUS_SUCCESS;
  if (ldc < m || c == nullptr || scale_a == nullptr || scale_b == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (offsets == nullptr && group_count != 1) return HIPBLAS_STATUS_INVALID_VALUE;
  if (k != 0 && (lda < k || ldb < k || a == nullptr || b == nullptr)) return HIPBLAS_STATUS_INVALID_VALUE;
  GroupedArgs args{};
  args.m = (uint32_t)m;
  args.n = (uint32_t)n;
  args.k = (uint32_t)k;
  args.groups = (uint32_t)group_count;
  args.offsets = offsets;
  args.a = (const char *)a;
  args.b = (const char *)b;
  args.c = (char *)c;
  args.lda = lda;
  args.ldb = ldb;
  args.ldc = ldc;
  args.stride_a = stridea;
  args.alpha = 1.0f;
  args.out = out;
  args.vec_c = four_at_once(c, m, ldc, 0, out);
  args.scale_a = scale_a;
  args.scale_b = scale_b;
  return run_columns(h, Elem::I8, true, args, "gemm_i8");
}
}
