// Experts' products for few tokens to a group (serving): the matrices are read once, straight into MFMA fragments.
//
// Bound by reading the weights: one token to each of 40 of 64 experts (and 24 more) of 2048 x 1024 in BF16 33.0 us, 5.1 TB/s, with
// 24 sets of matrices in turn; 30.0 with the same set again and again, part of which the last-level cache holds.  (All 64
// experts 48.4 us, 5.5 TB/s, where the 128 x 32 tiles, whose step is longer, read 6.0.)  At one or two tokens of 1024 x 1024
// by the launch and the way of a load, 5.5 us.  A workgroup of eight waves has 16 rows of one group's matrix (64 where the
// rows, not K, are contiguous) and up to 16 of its tokens.  The waves share out K, 128 bytes of every row at a time, so
// that the workgroup reads 1 KiB of each row side by side; each wave keeps several such loads under way, without LDS and
// without a barrier, and the eight partial sums are added through LDS in a fixed order at the end.
// Splitting K over waves rather than giving each wave rows of its own keeps a CU's share of a small matrix small: 1024
// rows are 64 workgroups, and a wave of the 128 KiB that 16 rows of 2048 FP32 values are reads 16.
#pragma once
#include "grouped_kernel.hpp"

namespace cumpsgemm_amd {

constexpr int kStreamWaves = 8, kStreamTokens = 16;

template <Elem E, bool A_KC> struct StreamCfg {
  using T = elem_traits<E>;
  // 16 rows of the matrix each, for a workgroup (row-contiguous: four rows a lane).  K-contiguous with four, us, with one
  // -> four: BF16 2048 x 1024, 2 tokens to 2 of 8 groups 4.8 -> 7.0, 64 to 27 of 64 27.4 -> 22.1, where the 128 x 32 tiles take
  // 21.0 (the same 113 MB of matrices again and again: they stay in the last-level cache).
  static constexpr int BLOCKS = A_KC ? 1 : 4, ROWS = BLOCKS * 16;
  // K-values of a wave's step: 128 bytes of a row, one or two MFMAs deep (row-contiguous: one, 32 lines)
  static constexpr int SLICES = A_KC && !T::F32 ? 2 : 1;
  static constexpr int KS = SLICES * 4 * T::CHUNK;
  static constexpr int UNROLL = A_KC ? 4 : 2; // steps under way
};

// eight or sixteen K-values of a 16-byte chunk (FP32: 32 bytes), as they lie in memory
template <Elem E> struct stream_raw {
  typename std::conditional<elem_traits<E>::F32, f8_t, u4_t>::type v;
};
template <Elem E> __device__ inline void stream_terms(const stream_raw<E> &raw, u4_t (&out)[elem_traits<E>::NP]) {
  if constexpr (elem_traits<E>::F32) splitter<elem_traits<E>::P>::run(raw.v, out);
  else out[0] = raw.v;
}
// a whole chunk, at an address that is aligned to its elements
template <Elem E> __device__ inline stream_raw<E> stream_load(const char *p) {
  using T = elem_traits<E>;
  stream_raw<E> r;
  if constexpr (T::F32) {
    typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
    const f4u_t x = reinterpret_cast<const f4u_t *>(p)[0], y = reinterpret_cast<const f4u_t *>(p)[1];
    r.v = f8_t{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  } else {
    typedef uint32_t u4u2_t __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t u4u1_t __attribute__((ext_vector_type(4), aligned(1)));
    typedef typename std::conditional<T::I8, u4u1_t, u4u2_t>::type u4u_t;
    const u4u_t x = *reinterpret_cast<const u4u_t *>(p);
    r.v = u4_t{x.x, x.y, x.z, x.w};
  }
  return r;
}
// the first `have` values of a chunk, zeros for the others
template <Elem E> __device__ inline stream_raw<E> stream_load_part(const char *p, int have) {
  using T = elem_traits<E>;
  stream_raw<E> r;
  if constexpr (T::F32) {
#pragma unroll
    for (int j = 0; j < 8; j++) r.v[j] = j < have ? reinterpret_cast<const float *>(p)[j] : 0.0f;
  } else {
    typedef typename std::conditional<T::I8, uint8_t, uint16_t>::type V;
    constexpr int BITS = T::BYTES * 8, PER = 32 / BITS;
    u4_t x = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < T::CHUNK; j++)
      if (j < have) x[j / PER] |= (uint32_t)reinterpret_cast<const V *>(p)[j] << (j % PER * BITS);
    r.v = x;
  }
  return r;
}

// Four neighbouring rows of one K-line (row-contiguous matrices): FP32 values, or two words of 16-bit ones.
template <Elem E> struct stream_line {
  typename std::conditional<elem_traits<E>::F32, f4v_t, uint2>::type v;
};
template <Elem E> __device__ inline stream_line<E> stream_load_line(const char *p) {
  stream_line<E> r;
  if constexpr (elem_traits<E>::F32) {
    typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
    const f4u_t x = *reinterpret_cast<const f4u_t *>(p);
    r.v = f4v_t{x.x, x.y, x.z, x.w};
  } else {
    typedef uint32_t u2u_t __attribute__((ext_vector_type(2), aligned(2)));
    const u2u_t x = *reinterpret_cast<const u2u_t *>(p);
    r.v = make_uint2(x.x, x.y);
  }
  return r;
}
// the first `have` rows, zeros for the others
template <Elem E> __device__ inline stream_line<E> stream_load_line_part(const char *p, int have) {
  stream_line<E> r;
  if constexpr (elem_traits<E>::F32) {
#pragma unroll
    for (int i = 0; i < 4; i++) r.v[i] = i < have ? reinterpret_cast<const float *>(p)[i] : 0.0f;
  } else {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = i < have ? reinterpret_cast<const uint16_t *>(p)[i] : 0u;
    r.v = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  }
  return r;
}

template <Elem E, bool A_KC>
__global__ __launch_bounds__(kStreamWaves * 64) void grouped_stream_kernel(const GroupedArgs args) {
  using T = elem_traits<E>;
  using C = StreamCfg<E, A_KC>;
  constexpr int BLOCKS = C::BLOCKS;
  __shared__ __attribute__((aligned(16))) float sums[kStreamWaves][kStreamTokens][C::ROWS + 4];
  const int tid = threadIdx.x, lane = tid & 63, frow = lane & 15, fg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t tiles_m = (args.m + C::ROWS - 1) / C::ROWS;
  TilePlace t;
  if (!place_tile(args, blockIdx.x, tiles_m, kStreamTokens, t)) return;
  const uint32_t m0 = t.tm * C::ROWS, n0 = t.lo + t.tn * kStreamTokens;
  const uint32_t tokens = t.hi - n0 < kStreamTokens ? t.hi - n0 : kStreamTokens;
  const uint32_t k = args.k;
  const char *a = uniform_address(args.a + (uint64_t)t.group * args.stride_a * T::BYTES);
  const char *b = uniform_address(args.b);
  // a token beyond the last reads the last again; its results are not stored
  const uint64_t b_row = (uint64_t)(n0 + ((uint32_t)frow < tokens ? frow : tokens - 1)) * args.ldb;

  typename T::acc_t acc[T::NACC][C::BLOCKS];
#pragma unroll
  for (int s = 0; s < T::NACC; s++)
#pragma unroll
    for (int i = 0; i < C::BLOCKS; i++)
#pragma unroll
      for (int v = 0; v < 4; v++) acc[s][i][v] = 0;
  auto multiply = [&](const u4_t (&fa)[T::NP], const u4_t (&fb)[T::NP], const int i) {
#pragma unroll
    for (int q = 0; q < T::NPROD; q++) {
      const int pa = T::F32 ? prec_traits<T::P>::PA[q] : 0, pb = T::F32 ? prec_traits<T::P>::PB[q] : 0;
      const int ac = T::F32 ? prec_traits<T::P>::ACC[q] : 0;
      acc[ac][i] = grouped_mfma<E>(fa[pa], fb[pb], acc[ac][i]);
    }
  };

  const int whole = (int)(k / C::KS), left = (int)(k % C::KS);
  if constexpr (A_KC) {
    // lane: row (token) l % 16, chunk l / 16 of the slice's four
    const char *pa[BLOCKS];
#pragma unroll
    for (int i = 0; i < BLOCKS; i++) {
      const uint32_t row = m0 + i * 16 + frow < args.m ? m0 + i * 16 + frow : args.m - 1;
      pa[i] = a + ((uint64_t)row * args.lda + fg * T::CHUNK) * T::BYTES;
    }
    const char *pb = b + (b_row + fg * T::CHUNK) * T::BYTES;
    struct Step {
      stream_raw<E> a[BLOCKS][C::SLICES], b[C::SLICES];
    };
    auto load = [&](Step &x, int s) {
#pragma unroll
      for (int h = 0; h < C::SLICES; h++) {
        const uint64_t at = ((uint64_t)s * C::KS + h * 4 * T::CHUNK) * T::BYTES;
        x.b[h] = stream_load<E>(pb + at);
#pragma unroll
        for (int i = 0; i < BLOCKS; i++) x.a[i][h] = stream_load<E>(pa[i] + at);
      }
    };
    auto take = [&](const Step &x) {
#pragma unroll
      for (int h = 0; h < C::SLICES; h++) {
        u4_t fb[T::NP];
        stream_terms<E>(x.b[h], fb);
#pragma unroll
        for (int i = 0; i < BLOCKS; i++) {
          u4_t fa[T::NP];
          stream_terms<E>(x.a[i][h], fa);
          multiply(fa, fb, i);
        }
      }
    };
    constexpr int U = C::UNROLL;
    int s = wave;
    for (; s + (U - 1) * kStreamWaves < whole; s += U * kStreamWaves) {
      Step x[U];
#pragma unroll
      for (int u = 0; u < U; u++) load(x[u], s + u * kStreamWaves);
#pragma unroll
      for (int u = 0; u < U; u++) take(x[u]);
    }
    for (; s < whole; s += kStreamWaves) {
      Step x;
      load(x, s);
      take(x);
    }
    if (left != 0 && s == whole) { // the last, partial step belongs to the wave whose turn it is
      Step x;
#pragma unroll
      for (int h = 0; h < C::SLICES; h++) {
        const int have = left - (h * 4 + fg) * T::CHUNK;
        const uint64_t at = ((uint64_t)whole * C::KS + h * 4 * T::CHUNK) * T::BYTES;
        x.b[h] = stream_load_part<E>(pb + at, have);
#pragma unroll
        for (int i = 0; i < BLOCKS; i++) x.a[i][h] = stream_load_part<E>(pa[i] + at, have);
      }
      take(x);
    }
  } else {
    // lane: rows 4 (l % 16) .. + 3, one of each MFMA's row block, and K-lines 8 (l / 16) .. + 7
    const uint32_t row = m0 + 4 * frow;
    const int rows = row < args.m ? (int)(args.m - row < 4 ? args.m - row : 4) : 0;
    const char *pa = a + ((uint64_t)(fg * 8) * args.lda + (rows > 0 ? row : 0)) * T::BYTES;
    const char *pb = b + (b_row + fg * 8) * T::BYTES;
    const uint64_t line = args.lda * T::BYTES;
    const bool inside = m0 + C::ROWS <= args.m; // (uniform)
    auto take = [&](const stream_line<E> (&ra)[8], const stream_raw<E> &rb) {
      u4_t fb[T::NP];
      stream_terms<E>(rb, fb);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        stream_raw<E> x;
        if constexpr (T::F32) {
#pragma unroll
          for (int j = 0; j < 8; j++) x.v[j] = ra[j].v[i];
        } else {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const uint32_t lo = i < 2 ? ra[2 * q].v.x : ra[2 * q].v.y, hi = i < 2 ? ra[2 * q + 1].v.x : ra[2 * q + 1].v.y;
            x.v[q] = __builtin_amdgcn_perm(hi, lo, i % 2 == 0 ? 0x05040100 : 0x07060302);
          }
        }
        u4_t fa[T::NP];
        stream_terms<E>(x, fa);
        multiply(fa, fb, i);
      }
    };
    auto load = [&](int s, stream_line<E> (&ra)[8], stream_raw<E> &rb) {
      const char *p = pa + (uint64_t)s * C::KS * line;
      if (inside) {
#pragma unroll
        for (int j = 0; j < 8; j++) ra[j] = stream_load_line<E>(p + (uint64_t)j * line);
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) ra[j] = stream_load_line_part<E>(p + (uint64_t)j * line, rows);
      }
      rb = stream_load<E>(pb + (uint64_t)s * C::KS * T::BYTES);
    };
    constexpr int U = C::UNROLL;
    int s = wave;
    for (; s + (U - 1) * kStreamWaves < whole; s += U * kStreamWaves) {
      stream_line<E> ra[U][8];
      stream_raw<E> rb[U];
#pragma unroll
      for (int u = 0; u < U; u++) load(s + u * kStreamWaves, ra[u], rb[u]);
#pragma unroll
      for (int u = 0; u < U; u++) take(ra[u], rb[u]);
    }
    for (; s < whole; s += kStreamWaves) {
      stream_line<E> ra[8];
      stream_raw<E> rb;
      load(s, ra, rb);
      take(ra, rb);
    }
    if (left != 0 && s == whole) {
      stream_line<E> ra[8];
      const char *p = pa + (uint64_t)whole * C::KS * line;
      const int have = left - fg * 8;
#pragma unroll
      for (int j = 0; j < 8; j++) ra[j] = stream_load_line_part<E>(p + (uint64_t)j * line, j < have ? rows : 0);
      take(ra, stream_load_part<E>(pb + (uint64_t)whole * C::KS * T::BYTES, have));
    }
  }

  // ---- sums of the waves, in their order ----
  // Register v of lane l: MFMA row 4 (l / 16) + v, token l % 16.  Row-contiguous: row r of block i is row 4 r + i.
#pragma unroll
  for (int i = 0; i < C::BLOCKS; i++)
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const int r = 4 * fg + v;
      float x;
      if constexpr (T::I8) {
        x = __int_as_float(acc[0][i][v]);
      } else {
        x = acc[0][i][v];
        if constexpr (T::NACC == 2) x += acc[1][i][v] * prec_traits<T::P>::CORR_SCALE;
      }
      sums[wave][frow][A_KC ? i * 16 + r : 4 * r + i] = x;
    }
  __syncthreads();
  for (int e = tid; e < C::ROWS * kStreamTokens; e += kStreamWaves * 64) {
    const uint32_t r = e % C::ROWS, j = e / C::ROWS, row = m0 + r, col = n0 + j;
    if (j >= tokens || row >= args.m) continue;
    float x;
    if constexpr (T::I8) {
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kStreamWaves; w++) sum += __float_as_int(sums[w][j][r]);
      x = (float)sum * args.scale_a[(uint64_t)t.group * args.m + row] * args.scale_b[col];
    } else {
      x = 0.0f;
#pragma unroll
      for (int w = 0; w < kStreamWaves; w++) x += sums[w][j][r];
      x *= args.alpha;
    }
    const uint64_t at = (uint64_t)col * args.ldc + row;
    auto put = [&](auto *c) {
      typedef typename std::remove_pointer<decltype(c)>::type O;
      c[at] = (O)(args.beta != 0.0f ? x + args.beta * (float)c[at] : x);
    };
    if (T::F32 || args.out == OUT_F32) put(reinterpret_cast<float *>(args.c));
    else if (E == Elem::F16 || (T::I8 && args.out == OUT_F16)) put(reinterpret_cast<_Float16 *>(args.c));
    else put(reinterpret_cast<__bf16 *>(args.c));
  }
}

template <Elem E, bool A_KC> void launch_grouped_stream(const GroupedArgs &args, uint32_t workgroups, hipStream_t stream) {
  hipLaunchKernelGGL((grouped_stream_kernel<E, A_KC>), dim3(workgroups), dim3(kStreamWaves * 64), 0, stream, args);
}
template <Elem E, bool A_KC> constexpr GroupedKernel stream_entry() {
  return {&launch_grouped_stream<E, A_KC>, StreamCfg<E, A_KC>::ROWS, kStreamTokens};
}

} // namespace cumpsgemm_amd
