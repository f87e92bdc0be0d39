// Experts' products: arguments, the choice of a kernel, launch.  See grouped.hpp.
#include "grouped_table.hpp"
#include "handle.hpp"
#include <algorithm>
#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_amd {

extern GroupedTable g_grouped_f32_fp16tcec, g_grouped_f32_fp16tc, g_grouped_f32_bf16x3, g_grouped_f32_bf16x2,
    g_grouped_f16, g_grouped_bf16, g_grouped_i8;
extern GroupedTable g_gated_f32_fp16tcec, g_gated_f32_fp16tc, g_gated_f32_bf16x3, g_gated_f32_bf16x2, g_gated_f16, g_gated_bf16;
extern GroupedTable g_gated_backward_f32_fp16tcec, g_gated_backward_f32_fp16tc, g_gated_backward_f32_bf16x3,
    g_gated_backward_f32_bf16x2, g_gated_backward_f16, g_gated_backward_bf16;
extern GroupedTable g_f8_e4m3, g_f8_e5m2, g_f8_exact_e4m3, g_f8_exact_e5m2, g_gated_f8_e4m3, g_gated_f8_e5m2, g_gated_f8_exact_e4m3,
    g_gated_f8_exact_e5m2;

// direct: the operands can take the shorter way into LDS (grouped_kernel.hpp); the kernel of few tokens takes any
const GroupedKernel *lookup_grouped(Elem e, bool a_kc, bool ragged_k, bool direct, int cls, Epilogue epi = Epilogue::STORE) {
  static const GroupedTable *const tables[5][kNumElems] = {
      {&g_grouped_f32_fp16tcec, &g_grouped_f32_fp16tc, &g_grouped_f32_bf16x3, &g_grouped_f32_bf16x2, &g_grouped_f16,
       &g_grouped_bf16, &g_grouped_i8, &g_f8_e4m3, &g_f8_e5m2},
      {&g_gated_f32_fp16tcec, &g_gated_f32_fp16tc, &g_gated_f32_bf16x3, &g_gated_f32_bf16x2, &g_gated_f16, &g_gated_bf16,
       nullptr, &g_gated_f8_e4m3, &g_gated_f8_e5m2},
      {&g_gated_backward_f32_fp16tcec, &g_gated_backward_f32_fp16tc, &g_gated_backward_f32_bf16x3, &g_gated_backward_f32_bf16x2,
       &g_gated_backward_f16, &g_gated_backward_bf16},
      {nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, &g_gated_f8_exact_e4m3, &g_gated_f8_exact_e5m2},
      {nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, &g_f8_exact_e4m3, &g_f8_exact_e5m2}};
  if (tables[(int)epi][(int)e] == nullptr) return nullptr;
  const GroupedTable &t = *tables[(int)epi][(int)e];
  const GroupedKernel *k = ragged_k ? (cls > SHORT_LINES ? nullptr : &t.over_k[direct][cls])
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
uint32_t bytes_of(Elem e) { return (int)e <= 3 ? 4 : (int)e >= (int)Elem::I8 ? 1 : 2; }

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
  float tail; // a tile's first loads and write-out, in steps (0: in the others)
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
// Gated blocks, their gradients and 8-bit floating point (exact sums, and the FAST ones), in the same terms, with what their larger epilogues cost, and apart for
// operands that go straight to LDS and for others (_any): fitted to 200 calls of each kind (and 100 of any alignment; sizes as
// above, m to 4096, k to 4096 in FP8 and 2048 else, 1 - 16384 tokens) with every kernel in turn.  On 100 other calls each the choice
// loses 3.4 % (gated, 16 bits), 3.5 (gradient), 4.1 and 3.3 (gated FP32: FP16TCEC, TF32TCEC), 1.9 and 1.9 (gradients), 1.3 (FP8) and 3.3
// (gated FP8), of any alignment 1.5, 3.0, 1.4 (FP8) and 2.4 (gated FP8), with FAST sums 5.9, 4.1, 4.6 and 2.2, against the best kernel for
// each; by the figures of the plain products 24 % for gated blocks of any alignment, 5 - 10 % for the others.
const Cost &gated_cost_of(Elem e, int cls, Epilogue epi, bool direct) {
  static const Cost gated16[5] = {{2.4f, 1.45f, 2.05f, 1, 64, 0.38f, 5.5f}, {5.7f, 0.52f, 0.71f, 2, 64, 0.51f, 2.1f},
                                  {6.3f, 0.14f, 0.29f, 2, 64, 0.95f, 2.8f}, {5.7f, 1.18f, 0.82f, 2, 512, 0.82f, 0.4f},
                                  {6.0f, 0.25f, 0.41f, 2, 64, 0.79f, 2.4f}};
  static const Cost backward16[5] = {{0.6f, 1.60f, 1.96f, 1, 64, 0.25f, 19.8f}, {6.1f, 0.66f, 0.67f, 2, 64, 0.26f, 12.0f},
                                     {7.6f, 0.17f, 0.27f, 2, 64, 0.72f, 5.9f}, {7.6f, 0.90f, 0.33f, 2, 512, 0.61f, 0.8f},
                                     {7.3f, 0.33f, 0.41f, 2, 64, 0.45f, 7.3f}};
  static const Cost gated16_any[5] = {{}, {6.2f, 0.86f, 1.02f, 2, 64, 0.47f, 2.2f}, {5.4f, 0.47f, 0.55f, 2, 64, 0.93f, 2.2f},
                                      {3.5f, 6.33f, 2.82f, 2, 512, 0.83f, 0.2f}, {}};
  static const Cost backward16_any[5] = {{}, {5.8f, 1.03f, 1.03f, 2, 64, 0.27f, 11.2f}, {6.7f, 0.40f, 0.47f, 2, 64, 0.72f, 4.4f},
                                         {7.3f, 1.62f, 1.37f, 2, 512, 0.74f, 0.1f}, {}};
  static const Cost gated32[5] = {{1.3f, 1.18f, 1.61f, 1, 32, 0.55f, 6.7f}, {3.3f, 0.63f, 0.84f, 1, 32, 0.65f, 6.5f},
                                  {5.4f, 0.43f, 0.46f, 2, 32, 0.95f, 1.4f}, {6.3f, 0.96f, 1.17f, 2, 256, 0.74f, 0.2f},
                                  {5.8f, 0.43f, 0.57f, 2, 32, 0.84f, 2.2f}};
  static const Cost gated32x3[5] = {{2.1f, 2.23f, 2.63f, 1, 32, 0.44f, 3.3f}, {3.9f, 1.12f, 1.46f, 1, 32, 0.63f, 2.7f},
                                    {5.3f, 0.67f, 0.62f, 2, 32, 0.90f, 0.8f}, {6.2f, 0.92f, 1.13f, 2, 256, 0.77f, 0.5f},
                                    {6.1f, 0.76f, 0.83f, 2, 32, 0.70f, 0.9f}};
  static const Cost backward32[5] = {{0.4f, 1.52f, 1.98f, 1, 32, 0.49f, 9.7f}, {0.8f, 0.84f, 1.03f, 1, 32, 0.60f, 11.5f},
                                     {5.5f, 0.66f, 0.62f, 2, 32, 0.78f, 2.1f}, {7.7f, 0.58f, 0.46f, 2, 256, 0.71f, 0.4f},
                                     {3.7f, 0.73f, 0.68f, 2, 32, 0.67f, 7.1f}};
  static const Cost backward32x3[5] = {{0.5f, 2.37f, 2.92f, 1, 32, 0.42f, 7.5f}, {1.0f, 1.27f, 1.47f, 1, 32, 0.58f, 8.2f},
                                       {4.2f, 0.90f, 0.67f, 2, 32, 0.77f, 4.1f}, {6.1f, 1.05f, 0.48f, 2, 256, 0.83f, 0.9f},
                                       {5.0f, 0.97f, 0.87f, 2, 32, 0.65f, 5.0f}};
  static const Cost f8[5] = {{1.5f, 1.51f, 1.90f, 1, 128, 0.39f, 6.9f}, {4.8f, 0.74f, 0.74f, 2, 128, 0.45f, 2.6f},
                             {4.3f, 0.51f, 0.44f, 2, 128, 0.74f, 2.8f}, {5.1f, 1.80f, 0.59f, 2, 1024, 0.74f, 0.4f},
                             {5.0f, 0.46f, 0.46f, 2, 128, 0.62f, 2.9f}};
  static const Cost f8_any[5] = {{}, {3.0f, 1.92f, 1.31f, 2, 128, 0.50f, 3.3f}, {3.2f, 1.32f, 0.88f, 2, 128, 0.82f, 1.8f},
                                 {2.6f, 7.52f, 2.24f, 2, 1024, 0.78f, 0.1f}, {}};
  static const Cost f8_exact[5] = {{}, {4.6f, 1.17f, 1.11f, 2, 128, 0.44f, 1.5f}, {4.6f, 0.46f, 0.45f, 2, 128, 0.76f, 2.4f},
                                   {4.9f, 0.86f, 0.61f, 2, 1024, 0.56f, 2.1f}, {4.2f, 0.74f, 0.69f, 2, 128, 0.70f, 1.7f}};
  static const Cost f8_exact_any[5] = {{}, {4.5f, 2.68f, 1.65f, 2, 128, 0.44f, 1.2f}, {3.3f, 0.99f, 0.65f, 2, 128, 0.86f, 2.5f},
                                       {4.7f, 2.85f, 2.54f, 2, 1024, 0.66f, 0.1f}, {4.1f, 1.29f, 0.92f, 2, 128, 0.64f, 1.9f}};
  static const Cost gated_f8[5] = {{3.7f, 1.41f, 1.81f, 1, 128, 0.34f, 6.2f}, {6.6f, 0.54f, 0.72f, 2, 128, 0.43f, 2.0f},
                                   {5.9f, 0.32f, 0.39f, 2, 128, 0.80f, 2.9f}, {6.3f, 1.11f, 0.99f, 2, 1024, 0.75f, 0.9f},
                                   {6.3f, 0.32f, 0.42f, 2, 128, 0.69f, 2.7f}};
  static const Cost gated_f8_exact[5] = {{}, {6.8f, 0.95f, 1.03f, 2, 128, 0.32f, 1.4f}, {6.1f, 0.36f, 0.41f, 2, 128, 0.69f, 2.6f},
                                         {6.9f, 1.14f, 1.10f, 2, 1024, 0.53f, 0.7f}, {6.2f, 0.57f, 0.62f, 2, 128, 0.57f, 1.8f}};
  static const Cost gated_f8_exact_any[5] = {{}, {4.6f, 2.24f, 1.53f, 2, 128, 0.47f, 2.1f}, {5.2f, 0.99f, 0.75f, 2, 128, 0.76f, 1.9f},
                                             {2.7f, 4.36f, 2.55f, 2, 1024, 0.95f, 0.6f}, {5.2f, 1.31f, 0.98f, 2, 128, 0.61f, 2.0f}};
  static const Cost gated_f8_any[5] = {{}, {5.1f, 1.95f, 1.37f, 2, 128, 0.50f, 1.9f}, {4.5f, 1.12f, 0.75f, 2, 128, 0.87f, 2.1f},
                                       {5.5f, 3.26f, 2.28f, 2, 1024, 0.69f, 0.9f}, {}};
  if (e == Elem::E4M3 || e == Elem::E5M2) {
    if (epi == Epilogue::STORE) return (direct ? f8 : f8_any)[cls];
    if (epi == Epilogue::STORE_EXACT) return (direct ? f8_exact : f8_exact_any)[cls];
    if (epi == Epilogue::GATED) return (direct ? gated_f8 : gated_f8_any)[cls];
    return (direct ? gated_f8_exact : gated_f8_exact_any)[cls];
  }
  const bool forward = epi == Epilogue::GATED;
  if (e == Elem::F32_BF16X3) return (forward ? gated32x3 : backward32x3)[cls];
  if ((int)e <= 3) return (forward ? gated32 : backward32)[cls];
  return (forward ? direct ? gated16 : gated16_any : direct ? backward16 : backward16_any)[cls];
}
double cost_us(const Cost &c, double workgroups, double steps, double cus, double filled = 1.0) {
  return c.fixed + (steps + c.tail) * (c.least + (1.0 - c.least) * filled) * std::max<double>(c.alone, c.each * (workgroups / cus + (workgroups > cus * c.slots ? 0.2 * c.slots : 0.0)));
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
bool forced(Elem e, bool a_kc, bool ragged_k, bool direct, int &cls, Epilogue epi = Epilogue::STORE) {
  const int want = tuning().force_cls;
  if (want < 0 || want >= kGroupedClasses || (ragged_k && want >= SHORT_LINES) || lookup_grouped(e, a_kc, ragged_k, direct, want, epi) == nullptr) return false;
  cls = want;
  return true;
}

// Ragged columns: no more tiles than this, where every group has a column of them that is not full.
uint64_t most_tiles(const GroupedArgs &args, const GroupedKernel &k) {
  const uint64_t columns = args.offsets == nullptr ? (args.n + k.bn - 1) / k.bn
                                                   : (uint64_t)args.n / k.bn + std::min(args.n, args.groups);
  return columns * ((args.m + k.bm - 1) / k.bm);
}

uint64_t most_workgroups(const GroupedKernel &k) { return 0xffffffffull / k.threads; } // (a launch has fewer than 2^32 threads)

// Ragged columns: B and C have args.n columns in args.groups groups.
hipblasStatus_t run_columns(cuMpSGEMM_handle *h, Elem e, bool a_kc, GroupedArgs &args, const char *label,
                            Epilogue epi = Epilogue::STORE) {
  const uint32_t bytes = bytes_of(e);
  const bool direct = chunks_ok(args.a, a_kc ? args.k : args.m, args.lda, args.stride_a, bytes, a_kc ? 256 : bytes == 1 ? 128 : 64) &&
                      chunks_ok(args.b, args.k, args.ldb, 0, bytes, 256) &&
                      ((epi != Epilogue::GATED && epi != Epilogue::GATED_EXACT) || chunks_ok(args.up, 16, args.lda, args.stride_a, bytes, 0));
  int cls = -1; // (none: more tiles than a launch has, of all of them)
  if (bytes == 2 && !direct && !a_kc && args.m < 8) {
    cls = STREAM; // (a line is shorter than the chunks that the tiled kernels read)
  } else if (!forced(e, a_kc, false, direct, cls, epi)) {
    double best = 0.0;
    for (int c = TILE_256; c < kGroupedClasses; c++) {
      const GroupedKernel *const kern = lookup_grouped(e, a_kc, false, direct, c, epi);
      if (kern == nullptr || most_tiles(args, *kern) > most_workgroups(*kern)) continue;
      // columns of tiles, the groups' sizes being unknown here: half of each group's last one, or one for each group
      const double some = std::min(args.n, args.groups), each = (double)args.n / args.groups;
      const double columns = args.groups == 1 ? (args.n + kern->bn - 1) / kern->bn
                             : each < kern->bn / 2 ? some : (double)args.n / kern->bn + 0.5 * some;
      const bool plain = epi == Epilogue::STORE && e != Elem::E4M3 && e != Elem::E5M2;
      const Cost &cost = plain ? cost_of(e, c) : gated_cost_of(e, c, epi, direct);
      // (the kernel of few tokens: in workgroups of 16 rows, as fitted with op T; where rows are contiguous it has 64 in one,
      // and this is too high)
      const double rows = c == STREAM ? (args.m + 15) / 16 : (args.m + kern->bm - 1) / kern->bm;
      const double us = cost_us(cost, columns * rows, (args.k + cost.step - 1) / cost.step, h->num_cus,
                                std::min(1.0, each / kern->bn));
      if (best == 0.0 || us < best) best = us, cls = c;
    }
  }
  if (cls < 0) return HIPBLAS_STATUS_INVALID_VALUE;
  const GroupedKernel *k = lookup_grouped(e, a_kc, false, direct, cls, epi);
  if (k == nullptr) return HIPBLAS_STATUS_INTERNAL_ERROR;
  const uint64_t workgroups = most_tiles(args, *k);
  if (workgroups > most_workgroups(*k)) return HIPBLAS_STATUS_INVALID_VALUE;
  ProfileScope prof(h, label);
  k->launch(args, (uint32_t)workgroups, h->stream);
  return launched();
}

// What products of 8-bit floating point and gated blocks of it are given alike.  nothing: there is nothing to compute.
hipblasStatus_t f8_arguments(cuMpSGEMM_handle *h, uint64_t m, uint64_t n, uint64_t k, bool a_kc, const void *a, uint64_t lda,
                             uint64_t stridea, hipDataType type_a, const float *scale_a, uint64_t stridescale, const void *b,
                             uint64_t ldb, hipDataType type_b, const float *scale_b, void *c, uint64_t ldc, hipDataType type_c,
                             const int *offsets, uint64_t group_count, Elem &e, bool &nothing, GroupedArgs &args) {
  nothing = false;
  if (h == nullptr || m > kMost || n > kMost || k > kMost || group_count > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
  if (type_a != HIP_R_8F_E4M3 || (type_b != HIP_R_8F_E4M3 && type_b != HIP_R_8F_E5M2)) return HIPBLAS_STATUS_INVALID_VALUE;
  if (!out_of(type_c, args.out) || (offsets == nullptr && group_count > 1)) return HIPBLAS_STATUS_INVALID_VALUE;
  nothing = m == 0 || n == 0 || group_count == 0;
  if (nothing) return HIPBLAS_STATUS_SUCCESS;
  if (ldc < m || c == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (k != 0 && (lda < (a_kc ? k : m) || ldb < k || a == nullptr || b == nullptr || scale_a == nullptr || scale_b == nullptr))
    return HIPBLAS_STATUS_INVALID_VALUE;
  e = type_b == HIP_R_8F_E4M3 ? Elem::E4M3 : Elem::E5M2;
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
  args.scale_a = scale_a;
  args.scale_b = scale_b;
  args.stride_scale = stridescale;
  return HIPBLAS_STATUS_SUCCESS;
}

// What gated blocks and their gradients are given alike.  nothing: there is nothing to compute.
hipblasStatus_t gated_arguments(cuMpSGEMM_handle *h, hipblasOperation_t op_A, cuMpSGEMM_activation_t activation, uint64_t m,
                                uint64_t n, uint64_t k, const void *a, uint64_t lda, uint64_t stridea, const void *b, uint64_t ldb,
                                const int *offsets, uint64_t group_count, cuMpSGEMM_compute_mode_t mode, hipDataType type, Elem &e,
                                bool &nothing, GroupedArgs &args) {
  nothing = false;
  if (h == nullptr || (op_A != HIPBLAS_OP_N && op_A != HIPBLAS_OP_T && op_A != HIPBLAS_OP_C)) return HIPBLAS_STATUS_INVALID_VALUE;
  if ((int)activation < CUMPSGEMM_SILU || (int)activation > CUMPSGEMM_RELU) return HIPBLAS_STATUS_INVALID_VALUE;
  if (m > kMost || n > kMost || k > kMost || group_count > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
  if (!elem_of(type, mode, e) || !out_of(type, args.out)) return HIPBLAS_STATUS_INVALID_VALUE;
  if (offsets == nullptr && group_count > 1) return HIPBLAS_STATUS_INVALID_VALUE;
  nothing = m == 0 || n == 0 || group_count == 0;
  if (nothing) return HIPBLAS_STATUS_SUCCESS;
  if (k != 0 && (lda < (op_A != HIPBLAS_OP_N ? k : m) || ldb < k || a == nullptr || b == nullptr)) return HIPBLAS_STATUS_INVALID_VALUE;
  args.m = (uint32_t)m;
  args.n = (uint32_t)n;
  args.k = (uint32_t)k;
  args.groups = (uint32_t)group_count;
  args.offsets = offsets;
  args.a = (const char *)a;
  args.b = (const char *)b;
  args.lda = lda;
  args.ldb = ldb;
  args.stride_a = stridea;
  args.act = (uint32_t)activation;
  return HIPBLAS_STATUS_SUCCESS;
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

hipblasStatus_t cuMpSGEMM_gemm_gated(cuMpSGEMM_handle_t h, hipblasOperation_t op_A, cuMpSGEMM_activation_t activation, uint64_t m,
                                     uint64_t n, uint64_t k, const void *gate, const void *up, uint64_t lda, uint64_t stridea,
                                     const void *b, uint64_t ldb, void *c, uint64_t ldc, void *z_gate, void *z_up, uint64_t ldz,
                                     const int *offsets, uint64_t group_count, cuMpSGEMM_compute_mode_t mode, hipDataType type) {
  GroupedArgs args{};
  Elem e;
  bool nothing;
  const hipblasStatus_t st = gated_arguments(h, op_A, activation, m, n, k, gate, lda, stridea, b, ldb, offsets, group_count, mode, type, e, nothing, args);
  if (st != HIPBLAS_STATUS_SUCCESS || nothing) return st;
  if (ldc < m || c == nullptr || (k != 0 && up == nullptr)) return HIPBLAS_STATUS_INVALID_VALUE;
  if ((z_gate == nullptr) != (z_up == nullptr) || (z_gate != nullptr && ldz < m)) return HIPBLAS_STATUS_INVALID_VALUE;
  args.up = (const char *)up;
  args.c = (char *)c;
  args.ldc = ldc;
  args.z[0] = (char *)z_gate;
  args.z[1] = (char *)z_up;
  args.ldz = ldz;
  return run_columns(h, e, op_A != HIPBLAS_OP_N, args, "gemm_gated", Epilogue::GATED);
}

hipblasStatus_t cuMpSGEMM_gemm_gated_backward(cuMpSGEMM_handle_t h, hipblasOperation_t op_A, cuMpSGEMM_activation_t activation,
                                              uint64_t m, uint64_t n, uint64_t k, const void *a, uint64_t lda, uint64_t stridea,
                                              const void *b, uint64_t ldb, const void *z_gate, const void *z_up, uint64_t ldz,
                                              void *d_gate, void *d_up, uint64_t ldd, void *c, uint64_t ldc, const int *offsets,
                                              uint64_t group_count, cuMpSGEMM_compute_mode_t mode, hipDataType type) {
  GroupedArgs args{};
  Elem e;
  bool nothing;
  const hipblasStatus_t st = gated_arguments(h, op_A, activation, m, n, k, a, lda, stridea, b, ldb, offsets, group_count, mode, type, e, nothing, args);
  if (st != HIPBLAS_STATUS_SUCCESS || nothing) return st;
  if (z_gate == nullptr || z_up == nullptr || ldz < m || d_gate == nullptr || d_up == nullptr || ldd < m || (c != nullptr && ldc < m))
    return HIPBLAS_STATUS_INVALID_VALUE;
  // (in place: with another leading dimension a column's gradients would be written over another's values)
  if ((d_gate == z_gate || d_up == z_up || d_gate == z_up || d_up == z_gate) && (ldd != ldz || d_gate == z_up || d_up == z_gate))
    return HIPBLAS_STATUS_INVALID_VALUE;
  args.z[0] = (char *)z_gate;
  args.z[1] = (char *)z_up;
  args.ldz = ldz;
  args.d[0] = (char *)d_gate;
  args.d[1] = (char *)d_up;
  args.ldd = ldd;
  args.c = (char *)c;
  args.ldc = ldc;
  return run_columns(h, e, op_A != HIPBLAS_OP_N, args, "gemm_gated_backward", Epilogue::GATED_BACKWARD);
}

hipblasStatus_t cuMpSGEMM_gemm_f8(cuMpSGEMM_handle_t h, hipblasOperation_t op_A, uint64_t m, uint64_t n, uint64_t k, const void *a,
                                  uint64_t lda, uint64_t stridea, hipDataType type_a, const float *scale_a, uint64_t stridescale,
                                  const void *b, uint64_t ldb, hipDataType type_b, const float *scale_b, void *c, uint64_t ldc,
                                  hipDataType type_c, const int *offsets, uint64_t group_count) {
  if (op_A != HIPBLAS_OP_N && op_A != HIPBLAS_OP_T && op_A != HIPBLAS_OP_C) return HIPBLAS_STATUS_INVALID_VALUE;
  const bool a_kc = op_A != HIPBLAS_OP_N;
  GroupedArgs args{};
  Elem e;
  bool nothing;
  const hipblasStatus_t st = f8_arguments(h, m, n, k, a_kc, a, lda, stridea, type_a, scale_a, stridescale, b, ldb, type_b, scale_b, c,
                                          ldc, type_c, offsets, group_count, e, nothing, args);
  if (st != HIPBLAS_STATUS_SUCCESS || nothing) return st;
  return run_columns(h, e, a_kc, args, "gemm_f8", h->f8_sums == CUMPSGEMM_F8_SUMS_FAST ? Epilogue::STORE : Epilogue::STORE_EXACT);
}

hipblasStatus_t cuMpSGEMM_gemm_gated_f8(cuMpSGEMM_handle_t h, cuMpSGEMM_activation_t activation, uint64_t m, uint64_t n, uint64_t k,
                                        const void *gate, const void *up, uint64_t lda, uint64_t stridea, hipDataType type_a,
                                        const float *scale_gate, const float *scale_up, uint64_t stridescale, const void *b,
                                        uint64_t ldb, hipDataType type_b, const float *scale_b, void *c, uint64_t ldc,
                                        hipDataType type_c, const int *offsets, uint64_t group_count) {
  if ((int)activation < CUMPSGEMM_SILU || (int)activation > CUMPSGEMM_RELU) return HIPBLAS_STATUS_INVALID_VALUE;
  GroupedArgs args{};
  Elem e;
  bool nothing;
  const hipblasStatus_t st = f8_arguments(h, m, n, k, true, gate, lda, stridea, type_a, scale_gate, stridescale, b, ldb, type_b, scale_b,
                                          c, ldc, type_c, offsets, group_count, e, nothing, args);
  if (st != HIPBLAS_STATUS_SUCCESS || nothing) return st;
  if (k != 0 && (up == nullptr || scale_up == nullptr)) return HIPBLAS_STATUS_INVALID_VALUE;
  args.up = (const char *)up;
  args.scale_up = scale_up;
  args.act = (uint32_t)activation;
  // (f8_kernel.hpp says why results wider than BF16 come from exact sums in any case)
  return run_columns(h, e, true, args, "gemm_gated_f8",
                     h->f8_sums == CUMPSGEMM_F8_SUMS_FAST && args.out == OUT_BF16 ? Epilogue::GATED : Epilogue::GATED_EXACT);
}

hipblasStatus_t cuMpSGEMM_set_f8_sums(cuMpSGEMM_handle_t h, cuMpSGEMM_f8_sums_t sums) {
  if (h == nullptr || (sums != CUMPSGEMM_F8_SUMS_FP32 && sums != CUMPSGEMM_F8_SUMS_FAST)) return HIPBLAS_STATUS_INVALID_VALUE;
  h->f8_sums = sums;
  return HIPBLAS_STATUS_SUCCESS;
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
