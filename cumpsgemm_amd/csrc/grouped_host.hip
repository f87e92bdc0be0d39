// Experts' products: arguments, the choice of a kernel, launch.  See grouped.hpp.
#include "grouped_table.hpp"
#include "handle.hpp"
#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_amd {

extern GroupedTable g_grouped_f32_fp16tcec, g_grouped_f32_fp16tc, g_grouped_f32_bf16x3, g_grouped_f32_bf16x2,
    g_grouped_f16, g_grouped_bf16, g_grouped_i8;

// direct: the operands can take the shorter way into LDS (grouped_kernel.hpp); the kernel of few tokens takes any
const GroupedKernel *lookup_grouped(Elem e, bool a_kc, bool ragged_k, bool direct, int cls) {
  static const GroupedTable *const tables[kNumElems] = {&g_grouped_f32_fp16tcec, &g_grouped_f32_fp16tc, &g_grouped_f32_bf16x3,
                                                        &g_grouped_f32_bf16x2, &g_grouped_f16, &g_grouped_bf16, &g_grouped_i8};
  const GroupedTable &t = *tables[(int)e];
  const GroupedKernel *k = ragged_k ? (cls >= STREAM_16 ? nullptr : &t.over_k[direct][cls])
                           : cls >= STREAM_16 ? &t.stream[a_kc][cls - STREAM_16] : &t.columns[a_kc][direct][cls];
  return k != nullptr && k->launch != nullptr ? k : nullptr;
}

namespace {

constexpr uint64_t kMost = 0x7fffffffull;

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

// CUMPSGEMM_FORCE_TILE_CLASS (0 - 4) goes before the rules; where there is no such kernel, the 128 x 128 one serves.
const GroupedKernel *choose(Elem e, bool a_kc, bool ragged_k, bool direct, int cls) {
  const int forced = tuning().force_cls;
  const GroupedKernel *k = lookup_grouped(e, a_kc, ragged_k, direct, forced >= 0 && forced < kKernelClasses ? forced : cls);
  return k != nullptr ? k : lookup_grouped(e, a_kc, ragged_k, direct, TILE_128);
}

// Ragged columns: B and C have args.n columns in args.groups groups.
hipblasStatus_t run_columns(cuMpSGEMM_handle *h, Elem e, bool a_kc, GroupedArgs &args, const char *label) {
  const uint32_t bytes = bytes_of(e);
  const bool direct = chunks_ok(args.a, a_kc ? args.k : args.m, args.lda, args.stride_a, bytes, a_kc ? 256 : 64) &&
                      chunks_ok(args.b, args.k, args.ldb, 0, bytes, 256);
  const uint64_t each = args.n / args.groups; // tokens of a group, on average
  int cls = each >= 192 ? TILE_256 : each >= 48 ? TILE_128 : each > 8 ? TILE_NARROW : STREAM_16;
  const GroupedKernel *k = choose(e, a_kc, false, direct, cls);
  if (k == nullptr) return HIPBLAS_STATUS_INTERNAL_ERROR;
  // no more tiles of columns than this: every group has one that is not full
  const uint64_t columns = args.offsets == nullptr ? (args.n + k->bn - 1) / k->bn
                                                   : (uint64_t)args.n / k->bn + std::min(args.n, args.groups);
  const uint64_t workgroups = columns * ((args.m + k->bm - 1) / k->bm);
  if (workgroups > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
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
  const uint64_t tiles = ((m + 255) / 256) * ((n + 255) / 256) * group_count;
  const int cls = direct && tiles >= h->num_cus ? TILE_256 : TILE_128;
  const GroupedKernel *kern = choose(e, false, true, direct, cls);
  if (kern == nullptr) return HIPBLAS_STATUS_INTERNAL_ERROR;
  const uint64_t per = ((m + kern->bm - 1) / kern->bm) * ((n + kern->bn - 1) / kern->bn);
  if (per > kMost || per * group_count > kMost) return HIPBLAS_STATUS_INVALID_VALUE;
  ProfileScope prof(h, "gemm_grouped_k");
  kern->launch(args, (uint32_t)(per * group_count), h->stream);
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
