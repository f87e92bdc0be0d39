// Columns to 8-bit floating point with a scale for each block of 128 (activations on their way into a product of FP8, and its
// matrices).
//
//   scale = max |x| / M,   q = M x / max |x| rounded to nearest even,   M = 448 (E4M3) or 57344 (E5M2)
//
// HBM-bound: each value read once, a byte written; 8192 tokens of 4096 values in BF16 21 - 24 us, 4.2 - 4.8 TB/s (a copy of 1 GiB:
// 5.2), in FP32 31 us, 5.4 TB/s; one token of 4096 2.8 us, the launch.  Tokens: sixteen lanes have a block, eight values each, and find its
// maximum among themselves.  Matrices: a workgroup has 128 x 128, kept in registers until the maximum is known.  The maximum is
// taken over the bits of |x| as integers, where an infinity is larger than every finite value and a NaN larger than both.
#include "handle.hpp"
#include <algorithm>
#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_amd {
namespace {

constexpr int kVec = 8, kBlock = 128, kLanes = kBlock / kVec, kThreads = 256;

struct QuantizeF8Args {
  const void *x;
  uint8_t *q;
  float *scale;
  uint64_t ldx, ldq, stride_x, stride_q;
  uint32_t k, n, kb, nb; // kb x nb blocks for a matrix
  uint64_t units;        // blocks of all matrices
};

template <class T> struct Eight {
  typedef T chunk __attribute__((ext_vector_type(kVec), aligned(16)));
  typedef T anywhere __attribute__((ext_vector_type(kVec), aligned(sizeof(T))));
  T v __attribute__((ext_vector_type(kVec)));
};
// the values of a chunk that exist, zeros for the others.  ALIGNED: k is a multiple of 8, a chunk exists or does not.  (Otherwise
// all chunks but a column's last are one access too, at any address; value by value 5274 tokens of 1585 values in FP16 15.6 us, so
// 10.4.)
template <class T, bool ALIGNED> __device__ inline Eight<T> load_eight(const T *column, uint32_t at, uint32_t k) {
  Eight<T> x;
  if constexpr (ALIGNED) {
    // (one behind the end reads the first; with a branch here, chunks went through memory that every thread has of its own: 8192
    // tokens of 4096 values in BF16 24.4 us, so 21.5)
    x.v = *reinterpret_cast<const typename Eight<T>::chunk *>(column + (at < k ? at : 0));
#pragma unroll
    for (int i = 0; i < kVec; i++) x.v[i] = at < k ? x.v[i] : (T)0.0f;
  } else {
    if (at + kVec <= k) {
      x.v = *reinterpret_cast<const typename Eight<T>::anywhere *>(column + at);
    } else {
#pragma unroll
      for (int i = 0; i < kVec; i++) x.v[i] = at + i < k ? column[at + i] : (T)0.0f;
    }
  }
  return x;
}
template <class T> __device__ inline uint32_t most_of(const Eight<T> &x, uint32_t most) {
#pragma unroll
  for (int i = 0; i < kVec; i++) {
    const uint32_t bits = __float_as_uint((float)x.v[i]) & 0x7fffffffu;
    most = most > bits ? most : bits;
  }
  return most;
}

// How a block's values become FP8.  q = M x / max: M x is exact for 16-bit x, and the quotient comes from two steps of a
// division whose remainder is exact, so that a quotient half way between two values of FP8, where 16-bit x often leads, is
// found as such.  (Multiplied by M / max, rounded, a few values in a hundred thousand go to the other side; and a division for
// each value would be most of the kernel.)  Both numbers are taken times a power of two, which is exact, so that neither
// overflows and neither is subnormal.
template <bool E5M2> struct BlockScale {
  static constexpr float M = E5M2 ? 57344.0f : 448.0f;
  float scale, times, peak, inverse;
  __device__ inline BlockScale(uint32_t most) {
    const bool finite = most < 0x7f800000u;
    const uint32_t e = most >> 23 > 20 ? (most >> 23 < 254 ? most >> 23 : 254) : 20;
    const float up = __uint_as_float((256 - e) << 23), down = __uint_as_float((e - 2) << 23); // 2^(129 - e) at most 2^109, and its inverse
    const float big = __uint_as_float(most) * up; // 4 .. 8, or less if the maximum is below 2^-107
    // big / M: a multiplication and the remainder, as above
    const float s = big * (1.0f / M);
    scale = finite ? fmaf(fmaf(-s, M, big), 1.0f / M, s) * down : __uint_as_float(0x7fc00000u);
    const bool some = finite && scale != 0.0f;
    times = some ? up * M : 0.0f;
    peak = some ? big : 1.0f;
    inverse = __builtin_amdgcn_rcpf(peak);
  }
  __device__ inline float operator()(float x) const {
    const float y = x * times, q = y * inverse;
    return fmaf(fmaf(-q, peak, y), inverse, q);
  }
};
template <bool E5M2, class T, bool ALIGNED>
__device__ inline void store_eight(uint8_t *q, uint32_t at, uint32_t k, const Eight<T> &x, const BlockScale<E5M2> &s, bool finite) {
  uint32_t out[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = finite ? s((float)x.v[4 * i + j]) : 0.0f;
    int y = 0;
    if constexpr (E5M2) {
      y = __builtin_amdgcn_cvt_pk_bf8_f32(v[0], v[1], y, false);
      y = __builtin_amdgcn_cvt_pk_bf8_f32(v[2], v[3], y, true);
    } else {
      y = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], y, false);
      y = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], y, true);
    }
    out[i] = (uint32_t)y;
  }
  if constexpr (ALIGNED) {
    if (at < k) *reinterpret_cast<uint2 *>(q + at) = make_uint2(out[0], out[1]);
  } else if (at + kVec <= k) {
    typedef uint32_t anywhere __attribute__((ext_vector_type(2), aligned(1)));
    *reinterpret_cast<anywhere *>(q + at) = anywhere{out[0], out[1]};
  } else {
#pragma unroll
    for (int i = 0; i < kVec; i++)
      if (at + i < k) q[at + i] = (uint8_t)(out[i / 4] >> (i % 4 * 8));
  }
}

// Tokens.  BIG: more units than 32 bits count.  AT_ONCE: the blocks of sixteen lanes, read together.
template <class T, bool E5M2, bool ALIGNED, bool BIG, int AT_ONCE>
__global__ __launch_bounds__(kThreads) void quantize_f8_kernel(const QuantizeF8Args args) {
  const uint32_t lane = threadIdx.x % kLanes;
  constexpr int GROUPS = kThreads / kLanes;
  const uint64_t step = (uint64_t)gridDim.x * (GROUPS * AT_ONCE);
  // where a unit lies: its matrix and column, its first value
  auto place = [&](uint64_t unit, uint64_t &matrix, uint64_t &column, uint32_t &at) {
    uint32_t b;
    if constexpr (BIG) {
      column = unit / args.kb;
      b = (uint32_t)(unit - column * args.kb);
    } else {
      const uint32_t c = (uint32_t)unit / args.kb;
      column = c;
      b = (uint32_t)unit - c * args.kb;
    }
    matrix = 0;
    if (args.units != (uint64_t)args.kb * args.n) { // (several matrices)
      matrix = column / args.n;
      column -= matrix * args.n;
    }
    at = b * kBlock + lane * kVec;
  };
  for (uint64_t first = (uint64_t)blockIdx.x * (GROUPS * AT_ONCE) + threadIdx.x / kLanes; first < args.units; first += step) {
    Eight<T> x[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) { // (one beyond the last: that again, not stored)
      uint64_t matrix, column;
      uint32_t at;
      const uint64_t unit = first + i * GROUPS;
      place(unit < args.units ? unit : args.units - 1, matrix, column, at);
      x[i] = load_eight<T, ALIGNED>(reinterpret_cast<const T *>(args.x) + matrix * args.stride_x + column * args.ldx, at, args.k);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; i++) {
      uint32_t most = most_of(x[i], 0);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) {
        const uint32_t o = __shfl_xor(most, d, kLanes);
        most = most > o ? most : o;
      }
      const uint64_t unit = first + i * GROUPS;
      if (unit >= args.units) continue; // (the sixteen lanes together)
      uint64_t matrix, column;
      uint32_t at;
      place(unit, matrix, column, at);
      const BlockScale<E5M2> s(most);
      if (lane == 0) args.scale[unit] = s.scale;
      store_eight<E5M2, T, ALIGNED>(args.q + matrix * args.stride_q + column * args.ldq, at, args.k, x[i], s, most < 0x7f800000u);
    }
  }
}

// Matrices.
template <class T, bool E5M2, bool ALIGNED> __global__ __launch_bounds__(kThreads) void quantize_f8_matrix_kernel(const QuantizeF8Args args) {
  constexpr int ROUNDS = kBlock / (kThreads / kLanes); // columns of a thread
  __shared__ uint32_t waves[kThreads / 64];
  for (uint64_t unit = blockIdx.x; unit < args.units; unit += gridDim.x) {
    const uint64_t per = (uint64_t)args.kb * args.nb, matrix = unit / per, in = unit - matrix * per;
    const uint32_t first = (uint32_t)(in / args.kb) * kBlock, at = (uint32_t)(in % args.kb) * kBlock + threadIdx.x % kLanes * kVec;
    const T *x = reinterpret_cast<const T *>(args.x) + matrix * args.stride_x;
    Eight<T> held[ROUNDS];
    uint32_t most = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
      const uint32_t column = first + r * (kThreads / kLanes) + threadIdx.x / kLanes;
      held[r] = load_eight<T, ALIGNED>(x + (column < args.n ? column : 0) * args.ldx, column < args.n ? at : args.k, args.k);
    }
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) most = most_of(held[r], most);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const uint32_t o = __shfl_xor(most, d, 64);
      most = most > o ? most : o;
    }
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) most = most > waves[w] ? most : waves[w];
    const BlockScale<E5M2> s(most);
    if (threadIdx.x == 0) args.scale[unit] = s.scale;
#pragma unroll
    for (int r = 0; r < ROUNDS; r++) {
      const uint32_t column = first + r * (kThreads / kLanes) + threadIdx.x / kLanes;
      if (column < args.n) store_eight<E5M2, T, ALIGNED>(args.q + matrix * args.stride_q + column * args.ldq, at, args.k, held[r], s, most < 0x7f800000u);
    }
    __syncthreads(); // (the waves' maxima are read before the next block's are written)
  }
}

constexpr uint64_t kMostWorkgroups = 1u << 20; // (a launch has fewer than 2^32 threads; more blocks in turns)

template <class T, bool E5M2, bool ALIGNED> void launch_quantize_f8(const QuantizeF8Args &args, bool matrices, int cus, hipStream_t stream) {
  if (matrices) {
    hipLaunchKernelGGL((quantize_f8_matrix_kernel<T, E5M2, ALIGNED>), dim3((uint32_t)std::min(args.units, kMostWorkgroups)), dim3(kThreads), 0,
                       stream, args);
    return;
  }
  // Two blocks at once keep enough loads under way where there are several workgroups of them for every CU.  (TB/s with one, two, four
  // and eight, inputs that are in no cache, BF16: 16384 tokens of 4096 values 4.3, 4.7, 4.7, 4.5; 4096 of 2048 3.25, 3.28, 3.06, 2.72.)
  constexpr uint64_t GROUPS = kThreads / kLanes;
  auto launch = [&](auto kernel, uint64_t each) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)std::min((args.units + GROUPS * each - 1) / (GROUPS * each), kMostWorkgroups)), dim3(kThreads), 0,
                       stream, args);
  };
  if (args.units >> 32) launch(quantize_f8_kernel<T, E5M2, ALIGNED, true, 2>, 2);
  else if (args.units >= 4 * GROUPS * 2 * (uint64_t)cus) launch(quantize_f8_kernel<T, E5M2, ALIGNED, false, 2>, 2);
  else launch(quantize_f8_kernel<T, E5M2, ALIGNED, false, 1>, 1);
}
template <class T> void launch_quantize_f8(const QuantizeF8Args &args, bool matrices, bool e5m2, int cus, hipStream_t stream) {
  const bool aligned = args.k % kVec == 0 && args.ldx * sizeof(T) % 16 == 0 && args.stride_x * sizeof(T) % 16 == 0 && args.ldq % kVec == 0 &&
                       args.stride_q % kVec == 0 && (uintptr_t)args.x % 16 == 0 && (uintptr_t)args.q % kVec == 0;
  if (e5m2) {
    if (aligned) launch_quantize_f8<T, true, true>(args, matrices, cus, stream);
    else launch_quantize_f8<T, true, false>(args, matrices, cus, stream);
  } else {
    if (aligned) launch_quantize_f8<T, false, true>(args, matrices, cus, stream);
    else launch_quantize_f8<T, false, false>(args, matrices, cus, stream);
  }
}
} // namespace
} // namespace cumpsgemm_amd

using namespace cumpsgemm_amd;
extern "C" hipblasStatus_t cuMpSGEMM_quantize_f8(cuMpSGEMM_handle_t h, uint64_t k, uint64_t n, const void *x, uint64_t ldx, uint64_t stridex,
                                                 hipDataType type_x, uint64_t block_n, void *q, uint64_t ldq, uint64_t strideq,
                                                 hipDataType type_q, float *scale, uint64_t batch_count) {
  if (h == nullptr || k > 0x7fffffffull || n > 0x7fffffffull || batch_count > 0x7fffffffull) return HIPBLAS_STATUS_INVALID_VALUE;
  if (type_x != HIP_R_32F && type_x != HIP_R_16F && type_x != HIP_R_16BF) return HIPBLAS_STATUS_INVALID_VALUE;
  if ((type_q != HIP_R_8F_E4M3 && type_q != HIP_R_8F_E5M2) || (block_n != 1 && block_n != kBlock)) return HIPBLAS_STATUS_INVALID_VALUE;
  if (n == 0 || k == 0 || batch_count == 0) return HIPBLAS_STATUS_SUCCESS;
  if (ldx < k || ldq < k || scale == nullptr || x == nullptr || q == nullptr) return HIPBLAS_STATUS_INVALID_VALUE;
  if (batch_count > 1 && strideq < ldq * (n - 1) + k) return HIPBLAS_STATUS_INVALID_VALUE; // (matrices of q overlap)
  QuantizeF8Args args{x, (uint8_t *)q, scale, ldx, ldq, stridex, strideq, (uint32_t)k, (uint32_t)n, 0, 0, 0};
  args.kb = (uint32_t)((k + kBlock - 1) / kBlock);
  args.nb = (uint32_t)((n + block_n - 1) / block_n);
  if ((uint64_t)args.kb * args.nb > ~0ull / batch_count) return HIPBLAS_STATUS_INVALID_VALUE;
  args.units = (uint64_t)args.kb * args.nb * batch_count;
  ProfileScope prof(h, "quantize_f8");
  const bool matrices = block_n != 1, e5m2 = type_q == HIP_R_8F_E5M2;
  if (type_x == HIP_R_32F) launch_quantize_f8<float>(args, matrices, e5m2, h->num_cus, h->stream);
  else if (type_x == HIP_R_16F) launch_quantize_f8<_Float16>(args, matrices, e5m2, h->num_cus, h->stream);
  else launch_quantize_f8<__bf16>(args, matrices, e5m2, h->num_cus, h->stream);
  return hipGetLastError() == hipSuccess ? HIPBLAS_STATUS_SUCCESS : HIPBLAS_STATUS_EXECUTION_FAILED;
}
