// Columns to 8-bit integers with a scale each (activations on their way into a product of 8-bit integers).
//
//   scale[j] = max_i |x[i, j]| / 127,   q[i, j] = rint(127 x[i, j] / max_i |x[i, j]|)
//
// HBM-bound: each value read once, a byte written.  One workgroup a column; a thread keeps what it read in registers
// until the column's maximum is known, so only columns of more than 8192 values are read twice.  The maximum is taken
// over the bits of |x| as integers, where an infinity is larger than every finite value and a NaN larger than both.
#include "handle.hpp"
#include "grouped.hpp"
#include <algorithm>
#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_amd {
namespace {

constexpr int kThreads = 256, kVec = 8, kHeld = 4;

struct QuantizeArgs {
  const void *x;
  int8_t *q;
  float *scale;
  uint64_t ldx, ldq;
  uint32_t k, n;
};
constexpr uint32_t kMostWorkgroups = 1u << 20; // (a launch has fewer than 2^32 threads; more columns in turns)

template <class T, bool ALIGNED>
__device__ inline void load_eight(const T *p, int have, float (&v)[kVec]) {
  if (ALIGNED) { // (k is a multiple of 8 then: all or nothing)
    typedef T t8_t __attribute__((ext_vector_type(8)));
    if (have > 0) {
      const t8_t x = *reinterpret_cast<const t8_t *>(p);
#pragma unroll
      for (int i = 0; i < kVec; i++) v[i] = (float)x[i];
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kVec; i++) v[i] = i < have ? (float)p[i] : 0.0f;
}

template <class T, bool ALIGNED> __global__ __launch_bounds__(kThreads) void quantize_kernel(const QuantizeArgs args) {
  for (uint32_t column = blockIdx.x; column < args.n; column += gridDim.x) {
    const T *x = reinterpret_cast<const T *>(args.x) + (uint64_t)column * args.ldx;
    int8_t *q = args.q + (uint64_t)column * args.ldq;
    const uint32_t k = args.k, stride = kThreads * kVec, first = threadIdx.x * kVec;
    float held[kHeld][kVec];
    uint32_t most = 0;
    auto widen = [&](const float (&v)[kVec]) {
#pragma unroll
      for (int i = 0; i < kVec; i++) {
        const uint32_t bits = __float_as_uint(v[i]) & 0x7fffffffu;
        most = most > bits ? most : bits;
      }
    };
#pragma unroll
    for (int h = 0; h < kHeld; h++) {
      const int64_t at = (int64_t)first + (int64_t)h * stride;
      load_eight<T, ALIGNED>(x + at, (int)((int64_t)k - at < kVec ? (int64_t)k - at : kVec), held[h]);
    }
#pragma unroll
    for (int h = 0; h < kHeld; h++) widen(held[h]);
    for (int64_t at = (int64_t)first + (int64_t)kHeld * stride; at < (int64_t)k; at += stride) {
      float v[kVec];
      load_eight<T, ALIGNED>(x + at, (int)((int64_t)k - at < kVec ? (int64_t)k - at : kVec), v);
      widen(v);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const uint32_t o = __shfl_xor(most, d, 64);
      most = most > o ? most : o;
    }
    __shared__ uint32_t waves[kThreads / 64];
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) most = most > waves[w] ? most : waves[w];

    // A column that holds an infinity or a NaN has no scale: NaN, and with it everything computed from the column.
    const bool finite = most < 0x7f800000u;
    const float scale = finite ? __uint_as_float(most) / 127.0f : __uint_as_float(0x7fc00000u);
    if (threadIdx.x == 0) args.scale[column] = scale;
    // q = rint(x * num / den).  127 / max: for 16-bit x the product is exact and so is a quotient half way between two
    // integers, which then goes to the even one as the formula says (divided by the rounded scale, one such value in a
    // few tens of columns went to the other side).  Near the largest numbers both are taken 2^-10 times, which is exact;
    // a subnormal scale is itself so coarse that the values are divided by it.
    const float peak = __uint_as_float(most);
    const bool huge = most >= 0x7b000000u, coarse = most < 0x04000000u; // 2^119; 2^-119
    const float num = coarse ? 1.0f : huge ? 127.0f / 1024.0f : 127.0f;
    const float den = coarse ? scale : huge ? peak / 1024.0f : peak;
    const bool some = finite && scale != 0.0f; // (a maximum of a few of the smallest numbers has a scale of zero)
    auto emit = [&](int64_t at, const float (&v)[kVec]) {
      const int have = (int)((int64_t)k - at < kVec ? (int64_t)k - at : kVec);
      int8_t out[kVec];
#pragma unroll
      for (int i = 0; i < kVec; i++) {
        const float r = some ? rintf(v[i] * num / den) : 0.0f;
        out[i] = (int8_t)(int)fminf(fmaxf(r, -127.0f), 127.0f); // (beyond 127 with a subnormal scale only)
      }
      if (ALIGNED) {
        if (have > 0) {
          typedef int8_t b8v_t __attribute__((ext_vector_type(8)));
          b8v_t o;
#pragma unroll
          for (int i = 0; i < kVec; i++) o[i] = out[i];
          *reinterpret_cast<b8v_t *>(q + at) = o;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kVec; i++)
          if (i < have) q[at + i] = out[i];
      }
    };
#pragma unroll
    for (int h = 0; h < kHeld; h++) {
      const int64_t at = (int64_t)first + (int64_t)h * stride;
      if (at < (int64_t)k) emit(at, held[h]);
    }
    for (int64_t at = (int64_t)first + (int64_t)kHeld * stride; at < (int64_t)k; at += stride) {
      float v[kVec];
      load_eight<T, ALIGNED>(x + at, (int)((int64_t)k - at < kVec ? (int64_t)k - at : kVec), v);
      emit(at, v);
    }
    __syncthreads(); // (the waves' maxima are read before the next column's are written)
  }
}

template <class T> void launch_quantize(const QuantizeArgs &args, uint32_t columns, hipStream_t stream) {
  const bool aligned = args.k % 8 == 0 && args.ldx * sizeof(T) % 16 == 0 && args.ldq % 8 == 0 &&
                       (uintptr_t)args.x % 16 == 0 && (uintptr_t)args.q % 8 == 0;
  if (aligned) hipLaunchKernelGGL((quantize_kernel<T, true>), dim3(std::min(columns, kMostWorkgroups)), dim3(kThreads), 0, stream, args);
  else hipLaunchKernelGGL((quantize_kernel<T, false>), dim3(std::min(columns, kMostWorkgroups)), dim3(kThreads), 0, stream, args);
}
} // namespace
} // namespace cumpsgemm_amd

using namespace cumpsgemm_amd;
extern "C" hipblasStatus_t cuMpSGEMM_quantize_i8(cuMpSGEMM_handle_t h, uint64_t k, uint64_t n, const void *x, uint64_t ldx,
                                                 hipDataType type_x, int8_t *q, uint64_t ldq, float *scale) {
  if (h == nullptr || k > 0x7fffffffull || n > 0x7fffffffull) return HIPBLAS_STATUS_INVALID_VALUE;
  if (type_x != HIP_R_32F && type_x != HIP_R_16F && type_x != HIP_R_16BF) return HIPBLAS_STATUS_INVALID_VALUE;
  if (n == 0) return HIPBLAS_STATUS_SUCCESS;
  if (ldx < k || ldq < k || scale == nullptr || (k != 0 && (x == nullptr || q == nullptr))) return HIPBLAS_STATUS_INVALID_VALUE;
  const QuantizeArgs args{x, q, scale, ldx, ldq, (uint32_t)k, (uint32_t)n};
  ProfileScope prof(h, "quantize_i8");
  if (type_x == HIP_R_32F) launch_quantize<float>(args, (uint32_t)n, h->stream);
  else if (type_x == HIP_R_16F) launch_quantize<_Float16>(args, (uint32_t)n, h->stream);
  else launch_quantize<__bf16>(args, (uint32_t)n, h->stream);
  return hipGetLastError() == hipSuccess ? HIPBLAS_STATUS_SUCCESS : HIPBLAS_STATUS_EXECUTION_FAILED;
}
