// Columns to 8-bit integers with a scale each (activations on their way into a product of 8-bit integers).
//
//   scale[j] = max_i |x[i, j]| / 127,   q[i, j] = rint(127 x[i, j] / max_i |x[i, j]|)
//
// HBM-bound: each value read once, a byte written (8192 columns of 4096 in BF16: 23.1 us, 4.4 TB/s; in FP32 25.7, 6.5 with what
// the last-level cache holds).  One workgroup a column; a thread keeps what it read in registers until the column's maximum
// is known, so only columns of more than 8192 values are read twice.  The maximum is taken over the bits of |x| as
// integers, where an infinity is larger than every finite value and a NaN larger than both.
#include "handle.hpp"
#include "grouped.hpp"
#include <algorithm>
#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_amd {
namespace {

constexpr int kVec = 8;

struct QuantizeArgs {
  const void *x;
  int8_t *q;
  float *scale;
  uint64_t ldx, ldq;
  uint32_t k, n;
};

// eight values as they lie in memory
template <class T> struct Eight {
  T v[kVec] __attribute__((aligned(16)));
  __device__ inline float operator[](int i) const { return (float)v[i]; }
};
// ALIGNED: k is a multiple of 8, a chunk exists or does not.  One that does not is read from the column's start instead,
// without a branch, so that no wait for the ones before it has to count on less.
template <class T, bool ALIGNED> __device__ inline Eight<T> load_eight(const T *column, int64_t at, int64_t k) {
  Eight<T> x;
  if constexpr (ALIGNED) {
    x = *reinterpret_cast<const Eight<T> *>(column + (at < k ? at : 0));
  } else {
#pragma unroll
    for (int i = 0; i < kVec; i++) x.v[i] = at + i < k ? column[at + i] : (T)0.0f;
  }
  return x;
}

// HELD: of the chunks of eight that a thread has of a column, how many stay in registers.
template <class T, bool ALIGNED, int HELD, int kThreads> __global__ __launch_bounds__(kThreads) void quantize_kernel(const QuantizeArgs args) {
  const uint32_t k = args.k, stride = kThreads * kVec, first = threadIdx.x * kVec;
  Eight<T> held[HELD];
  auto fetch = [&](uint32_t column, Eight<T> (&to)[HELD]) {
    const T *x = reinterpret_cast<const T *>(args.x) + (uint64_t)column * args.ldx;
#pragma unroll
    for (int h = 0; h < HELD; h++) to[h] = load_eight<T, ALIGNED>(x, (int64_t)first + (int64_t)h * stride, k);
  };
  for (uint32_t column = blockIdx.x; column < args.n; column += gridDim.x) {
    const T *x = reinterpret_cast<const T *>(args.x) + (uint64_t)column * args.ldx;
    int8_t *q = args.q + (uint64_t)column * args.ldq;
    if (k > 0) fetch(column, held);
    uint32_t most = 0;
    auto widen = [&](const Eight<T> &v) {
#pragma unroll
      for (int i = 0; i < kVec; i++) {
        const uint32_t bits = __float_as_uint(v[i]) & 0x7fffffffu;
        most = most > bits ? most : bits;
      }
    };
    if (k > 0) {
#pragma unroll
      for (int h = 0; h < HELD; h++) widen(held[h]);
    }
    for (int64_t at = (int64_t)first + (int64_t)HELD * stride; at < (int64_t)k; at += stride)
      widen(load_eight<T, ALIGNED>(x, at, k));
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
    // A division for each value would be two thirds of this kernel's instructions (31 for a value: 27 us for 8192 columns of
    // 4096 in BF16, whose bytes take 19; so: 23).  Instead it is multiplied by 127 / max, whose two roundings and the two of
    // the quotient that it stands for are less than 2^-15 apart (127 * 4 * 2^-24): that far from a half, both go to the same
    // integer.  (1.5 * 2^23 added leaves the integer in the last bits of the sum.)  Near a half, where FP16 and BF16 values
    // often are, the remainder decides, which is exact for them: at most 15 bits of 127 x, 18 of the integer times max.
    const bool quick = some && !coarse && !huge;
    const float times = num / den, magic = 12582912.0f, near_half = 0.5f - 0x1p-14f;
    auto emit = [&](int64_t at, const Eight<T> &v) {
      const int have = (int)((int64_t)k - at < kVec ? (int64_t)k - at : kVec);
      int8_t out[kVec];
      float off = 0.0f;
#pragma unroll
      for (int i = 0; i < kVec; i++) {
        const float sum = v[i] * times + magic;
        off = fmaxf(off, fabsf(v[i] * times - (sum - magic)));
        out[i] = (int8_t)__float_as_uint(sum);
      }
      if (sizeof(T) == 2 && quick) {
        if (off > near_half) {
#pragma unroll
          for (int i = 0; i < kVec; i++) {
            const float sum = v[i] * times + magic, rest = fmaf(magic - sum, peak, v[i] * 127.0f), much = fabsf(rest);
            const int bits = (int)__float_as_uint(sum);
            const bool other = much > peak * 0.5f || (much == peak * 0.5f && (bits & 1) != 0);
            out[i] = (int8_t)(bits + (other ? (rest > 0.0f ? 1 : -1) : 0));
          }
        }
      } else if (!quick || off > near_half) {
#pragma unroll
        for (int i = 0; i < kVec; i++) {
          const float r = some ? rintf(v[i] * num / den) : 0.0f;
          out[i] = (int8_t)(int)fminf(fmaxf(r, -127.0f), 127.0f); // (beyond 127 with a subnormal scale only)
        }
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
    for (int h = 0; h < HELD; h++) {
      const int64_t at = (int64_t)first + (int64_t)h * stride;
      if (at < (int64_t)k) emit(at, held[h]);
    }
    for (int64_t at = (int64_t)first + (int64_t)HELD * stride; at < (int64_t)k; at += stride)
      emit(at, load_eight<T, ALIGNED>(x, at, k));
    __syncthreads(); // (the waves' maxima are read before the next column's are written)
  }
}

constexpr uint32_t kMostWorkgroups = 1u << 20; // (a launch has fewer than 2^32 threads; more columns in turns)
template <class T, bool ALIGNED, int HELD, int THREADS> void launch_quantize(const QuantizeArgs &args, hipStream_t stream) {
  hipLaunchKernelGGL((quantize_kernel<T, ALIGNED, HELD, THREADS>), dim3(std::min(args.n, kMostWorkgroups)), dim3(THREADS), 0, stream, args);
}
template <class T, bool ALIGNED> void launch_quantize(const QuantizeArgs &args, int cus, hipStream_t stream) {
  // No more waves to a column than it fills, where there are workgroups for all CUs: what a column costs beside its values,
  // the maximum over its threads and two divisions, each wave pays (BF16, us, four waves / as many as here: 16384 columns
  // of 2048 34.2 / 22.2, 8192 of 4096 26.4 / 23.1, 4096 of 515 16.2 / 7.5).  With
  // fewer columns the waves are needed for the loads: 256 of 1536 3.5 / 4.9, of 1024 4.1 / 4.0.
  const bool many = args.n >= (uint32_t)cus * 8;
  if (args.k <= 64 * kVec * 2 || (many && args.k <= 64 * kVec * 4)) launch_quantize<T, ALIGNED, 4, 64>(args, stream);
  else if (many && args.k <= 128 * kVec * 4) launch_quantize<T, ALIGNED, 4, 128>(args, stream);
  else launch_quantize<T, ALIGNED, 4, 256>(args, stream);
}
template <class T> void launch_quantize(const QuantizeArgs &args, int cus, hipStream_t stream) {
  const bool aligned = args.k % 8 == 0 && args.ldx * sizeof(T) % 16 == 0 && args.ldq % 8 == 0 &&
                       (uintptr_t)args.x % 16 == 0 && (uintptr_t)args.q % 8 == 0;
  if (aligned) launch_quantize<T, true>(args, cus, stream);
  else launch_quantize<T, false>(args, cus, stream);
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
  if (type_x == HIP_R_32F) launch_quantize<float>(args, h->num_cus, h->stream);
  else if (type_x == HIP_R_16F) launch_quantize<_Float16>(args, h->num_cus, h->stream);
  else launch_quantize<__bf16>(args, h->num_cus, h->stream);
  return hipGetLastError() == hipSuccess ? HIPBLAS_STATUS_SUCCESS : HIPBLAS_STATUS_EXECUTION_FAILED;
}
