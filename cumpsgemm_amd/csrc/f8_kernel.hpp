// Products of 8-bit floating point with a scale for each block of 128 (gfx950, wave64).
//
//   C[i, j] = sum_b scale_a[i / 128, b] scale_b[b, j] sum_{l in block b of 128} A[l, i] B[l, j]
//
// The tiles, their loads and the write-out are those of grouped_kernel.hpp; a step is one block of K, 128 bytes of a row: four
// v_mfma_f32_16x16x32_bf16 deep, of fragments that are converted to BF16, or (FAST, below) one v_mfma_f32_16x16x128_f8f6f4.  Their
// sums start from zero, and a lane's four are multiplied with the block's scales and added in FP32 by vector instructions, beside
// the MFMAs that follow.  (They cannot go on with the sums of the block before: those have other scales.)
//
// What the FP8 MFMAs keep, measured with single products: products of eight K-values (two registers of a lane) are cut to
// multiples of 2^-13 of the largest one's power of two, then the sixteen such sums of a block are added in FP32, cut to 2^-23.
// Products of random values come out 2e-5 of their norm from exact, a hundredth of what a result in BF16 is rounded by, a
// tenth of FP16's.  (v_mfma_f32_16x16x32_fp8_fp8, at half the rate, gives the same bits.)
// EXACT kernels take BF16 MFMAs instead, to which FP8 converts without rounding: products are exact, sums FP32, at half the
// rate and with a conversion of every fragment.  They serve every call, unless the handle was told FAST sums: then the FP8 MFMAs
// are taken where they are faster, but for few tokens, which wait for memory anyway, and for gated blocks whose result is wider
// than BF16.  Such a result is FP8 again in the layer behind, where a value that was near half way between two of E4M3's comes
// out a whole step away, and 2e-5 more before makes 4e-4 to 1e-3 of that layer's result (FP16's own rounding: 2e-4; in BF16 the
// block is 2.1e-3 from FP64 with FAST sums, 1.7e-3 with exact ones).
//
// LDS images: rows of 128 bytes as for 8-bit integers.  Operands whose rows, not K, are contiguous (A of op N): 128 lines of
// BM bytes, read by ds_read_b64_tr_b8, which takes eight lines of sixteen rows and hands each lane one row's eight K-values.
// The 16-byte pieces of a line are exchanged so that the eight lines that each of two quarters of a wave reads at a time cover
// all banks.  Behind the operands come the step's scales: one for each token, and those of the rows.
//
// What it spends its time on (us).  8192 tokens, 4096 x 4096, exact sums, 128 x 128 tiles: 245 - 275, up to 1120 TFLOP/s (the
// library's product of that size in BF16: 198): 192 vector instructions, two thirds of them conversions, beside the 64 MFMAs of a
// wave's step, and the clock.  FAST, 256 x 256 tiles: 123 - 136, up to 2230 TFLOP/s (this card's best FP8 product of that size, with
// one scale for each matrix, takes 99 to 112).  An FP8 MFMA with its four multiply-adds takes 37 clocks, the MFMA alone 32; of a wave's
// time MFMAs are 56 % and waits 33; no LDS read meets another's bank; on zeros, which leave the clock higher, a fifth less.  128 x 256
// and 256 x 128 tiles in three buffers were slower, two 128 x 128 workgroups on a CU too where 256 x 256 tiles fill the chip.  64
// tokens to 40 of 64 experts, a gated block of 2 x 1024 x 2048: reading the matrices, 35 (4.8 TB/s) in tiles of 32 tokens (FAST: of
// 64, 36), 39 by the kernel of few tokens.  One token of 4096 x 4096: 6, the launch and a memory's round trip for every four of a
// wave's steps.  1531 tokens to 7 of 8 experts, 2048 x 1536, the matrices read along their rows: 22, FAST 17, a tile's twelve steps
// with no other workgroup beside it.
#pragma once
#include "grouped_table.hpp"

namespace cumpsgemm_amd {

typedef int i8v_t __attribute__((ext_vector_type(8)));

// B in E; A is E4M3
template <Elem E> __device__ inline f4v_t f8_mfma(const i8v_t a, const i8v_t b) {
  // (format 0: E4M3, 1: E5M2; scales of zero: none)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f4v_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, E == Elem::E5M2 ? 1 : 0, 0, 0, 0, 0);
}

// eight values as BF16
template <bool E5M2> __device__ inline u4_t f8_widen(const int lo, const int hi) {
  typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
  u4_t x;
  if constexpr (E5M2) {
    x.x = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, 1.0f, false));
    x.y = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, 1.0f, true));
    x.z = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, 1.0f, false));
    x.w = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, 1.0f, true));
  } else {
    x.x = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    x.y = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    x.z = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    x.w = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  }
  return x;
}
// a fragment of 32 K-values, as the kernels multiply it: FP8 for one MFMA, or BF16 for four
struct F8Wide {
  u4_t v[4];
};
template <bool EXACT, bool E5M2> __device__ inline typename std::conditional<EXACT, F8Wide, i8v_t>::type f8_fragment(const i8v_t x) {
  if constexpr (EXACT) {
    F8Wide y;
#pragma unroll
    for (int c = 0; c < 4; c++) y.v[c] = f8_widen<E5M2>(x[2 * c], x[2 * c + 1]);
    return y;
  } else {
    return x;
  }
}
// (E: B's type, as above)
template <Elem E> __device__ inline f4v_t f8_block(const i8v_t &a, const i8v_t &b) { return f8_mfma<E>(a, b); }
template <Elem E> __device__ inline f4v_t f8_block(const F8Wide &a, const F8Wide &b) {
  f4v_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int c = 0; c < 4; c++) x = mfma_block<true>(a.v[c], b.v[c], x);
  return x;
}

// Where a step's scales lie: those of A belong to 128 x 128 of the matrix as it is stored, blocks along its contiguous side
// first.
struct F8Scales {
  uint32_t kb, mb; // blocks of K and of rows
  __device__ inline F8Scales(const GroupedArgs &args) : kb((args.k + 127) / 128), mb((args.m + 127) / 128) {}
  template <bool A_KC> __device__ inline const float *of_rows(const float *scale, const GroupedArgs &args, uint32_t group, uint32_t block) const {
    const uint32_t at = block < mb ? block : mb - 1;
    return scale + group * args.stride_scale + (A_KC ? (uint64_t)at * kb : (uint64_t)at);
  }
  // from one block of K to the next, in bytes
  template <bool A_KC> __device__ inline uint64_t step_of_rows() const { return A_KC ? 4 : (uint64_t)mb * 4; }
};

template <Elem E, bool A_KC, int BM, int BN, int WM, int WN, int NSTAGE, bool DIRECT, Epilogue EPI, bool EXACT_>
struct F8Cfg : GroupedCfg<E, A_KC, true, BM, BN, WM, WN, 128, NSTAGE, DIRECT, false, 2, false, EPI> {
  using Base = GroupedCfg<E, A_KC, true, BM, BN, WM, WN, 128, NSTAGE, DIRECT, false, 2, false, EPI>;
  static_assert(Base::BK == 128, "a step is a block");
  // Scales: tokens by the first waves, 64 each, the rows' by the others (all the same ones): a load a wave, so that all waves
  // have equally many
  static constexpr int TOKEN_WAVES = BN >= 64 ? BN / 64 : 1;
  static_assert(TOKEN_WAVES < Base::WAVES_M * Base::WAVES_N, "a wave for the rows' scales");
  static constexpr int SCALES_A = TOKEN_WAVES * 256; // bytes
  static constexpr int STAGE = Base::STAGE + SCALES_A + 256;
  static constexpr int LDS_BYTES = NSTAGE * STAGE > Base::OUT_BYTES ? NSTAGE * STAGE : Base::OUT_BYTES;
  static_assert(LDS_BYTES <= 160 * 1024, "LDS");
  static constexpr int SIDES = Base::GATED ? 2 : 1;
  static constexpr bool EXACT = EXACT_;
};

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// a scale for each lane, memory -> LDS (as grouped_loader::direct)
__device__ inline void f8_direct_scales(const char *p, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(p) : "memory", "m0");
}
#pragma clang diagnostic pop

// One tile, TN column blocks of 16 for each wave (see multiply_tile).
template <class Cfg, int TN>
__device__ inline void multiply_f8_tile(const GroupedArgs &args, const TileWork &w, char *lds) {
  using T = typename Cfg::T;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, TM = Cfg::TM, NT = Cfg::NT, SIDES = Cfg::SIDES;
  constexpr int SCALES = Cfg::A_STAGE + Cfg::B_STAGE; // where a stage's scales begin
  const int tid = threadIdx.x, lane = tid & 63, frow = lane & 15, fg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;
  using LA = grouped_loader<Cfg::E, Cfg::A_KC, BM, 128, NT, Cfg::GATED>;
  using LB = grouped_loader<Cfg::E, true, BN, 128, NT>;
  constexpr int UB = (TN * 16 * Cfg::WAVES_N * 8 + NT - 1) / NT; // rounds of loads that B's columns need
  const char *a = w.a, *b = w.b;
  if constexpr (Cfg::GATED) a = uniform_address(w.a + (uint64_t)LA::side(wave) * (uint64_t)(w.up - w.a)); // (no choice of two: it would put w into memory)
  const uint64_t a_step = Cfg::A_KC ? 128 : 128 * args.lda, b_step = 128;

  // ---- scales ----
  const F8Scales sc(args);
  const char *scale; // this lane's for block 0
  uint64_t scale_step = 4;
  if (wave < Cfg::TOKEN_WAVES) {
    const int t = wave * 64 + lane;
    scale = reinterpret_cast<const char *>(args.scale_b + (uint64_t)(w.n0 + (t < w.rows_b ? t : w.rows_b - 1)) * sc.kb);
  } else {
    scale = reinterpret_cast<const char *>(
        sc.of_rows<Cfg::A_KC>(Cfg::GATED && lane >= 32 ? args.scale_up : args.scale_a, args, w.group, w.m0 / 128 + (lane & 31)));
    scale_step = sc.step_of_rows<Cfg::A_KC>();
  }
  const uint32_t scale_to = SCALES + (wave < Cfg::TOKEN_WAVES ? wave * 256 : Cfg::SCALES_A); // in a stage
  const int block = wm * Cfg::WAVE_ROWS_OUT / 128; // which of the tile's blocks of rows this wave's are in

  f4v_t acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++) acc[j][i] = f4v_t{0.0f, 0.0f, 0.0f, 0.0f};

  // ---- fragments ----
  // Lane l supplies row l % 16 and chunks l / 16 and 4 + l / 16 of its 128 bytes, the same K-values of both operands.
  auto frag = [&](const char *op, const int row0, auto kc_tag) -> i8v_t {
    if constexpr (decltype(kc_tag)::value) {
      const u4_t x = *reinterpret_cast<const u4_t *>(op + chunk_offset<128>(row0 + frow, fg));
      const u4_t y = *reinterpret_cast<const u4_t *>(op + chunk_offset<128>(row0 + frow, fg + 4));
      return i8v_t{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
    } else {
      typedef int i2_t __attribute__((ext_vector_type(2)));
      typedef __attribute__((address_space(3))) i2_t *tr_t;
      i8v_t out;
#pragma unroll
      for (int q = 0; q < 4; q++) {
        // lane l % 16 names line (l % 16) / 2 of eight and half of a piece
        const int k = (q >> 1) * 64 + fg * 16 + (q & 1) * 8 + (frow >> 1);
        const i2_t x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (tr_t)(op + k * BM + (((row0 >> 4) ^ byte_line_swizzle<BM>(k)) << 4) + (frow & 1) * 8));
        out[2 * q] = x[0];
        out[2 * q + 1] = x[1];
      }
      return out;
    }
  };
  // row blocks of A on their way ahead of the one that is multiplied (two, in tiles of 256 rows: level)
  constexpr int AHEAD = 1, A_RING = 2 * AHEAD;
  static_assert(TM % A_RING == 0, "a step begins where the ring does");
  i8v_t fa[A_RING];
  typename std::conditional<Cfg::EXACT, F8Wide, i8v_t>::type fb[TN];
  float now[SIDES][TN], old[SIDES][TN], next_scales[SIDES][TN]; // of this step, the one before, the one behind
  auto read_a = [&](const char *stage, const int g) {
    fa[g % A_RING] = frag(stage, wm * Cfg::WM + g % TM * 16, std::integral_constant<bool, Cfg::A_KC>{});
  };
  auto read_b = [&](const char *stage, const int j) {
    fb[j] = f8_fragment<Cfg::EXACT, Cfg::E == Elem::E5M2>(frag(stage + Cfg::A_STAGE, (j * Cfg::WAVES_N + wn) * 16, std::true_type{}));
  };
  auto read_scales = [&](const char *stage) {
    const float *s = reinterpret_cast<const float *>(stage + SCALES);
    float of_rows[SIDES];
#pragma unroll
    for (int side = 0; side < SIDES; side++) of_rows[side] = s[Cfg::SCALES_A / 4 + side * 32 + block];
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const float x = s[(j * Cfg::WAVES_N + wn) * 16 + frow];
#pragma unroll
      for (int side = 0; side < SIDES; side++) next_scales[side][j] = x * of_rows[side];
    }
  };
  auto begin = [&](const char *stage) {
#pragma unroll
    for (int g = 0; g < AHEAD; g++) read_a(stage, g);
#pragma unroll
    for (int j = 0; j < TN; j++) read_b(stage, j);
    read_scales(stage);
  };
  // The MFMAs' results are taken DELAY MFMAs later, in the next step if need be.
  constexpr int MFMAS = TM * TN, DELAY = MFMAS > 3 ? 3 : MFMAS - 1, RING = DELAY + 1;
  static_assert(MFMAS % RING == 0 && TM % 2 == 0, "a step ends where the rings begin");
  f4v_t sums[RING];
#pragma unroll
  for (int q = 0; q < RING; q++) sums[q] = f4v_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int side = 0; side < SIDES; side++)
#pragma unroll
    for (int j = 0; j < TN; j++) now[side][j] = old[side][j] = next_scales[side][j] = 0.0f;
  auto take = [&](const int q, const float (&s)[SIDES][TN]) { // (q: of a step)
    const int i = q / TN, j = q % TN;
#pragma unroll
    for (int v = 0; v < 4; v++) acc[j][i][v] = fmaf(sums[q % RING][v], s[SIDES > 1 ? i & 1 : 0][j], acc[j][i][v]);
  };
  // (else the compiler moves all of a step's additions behind its MFMAs, whose results then have no registers)
  auto hold = [&](const int q) { asm volatile("" : "+v"(acc[q % TN][q / TN])); };
  auto enter = [&]() { // a step begins
#pragma unroll
    for (int side = 0; side < SIDES; side++)
#pragma unroll
      for (int j = 0; j < TN; j++) {
        old[side][j] = now[side][j];
        now[side][j] = next_scales[side][j];
      }
  };
  // Row blocks `from` .. `to` - 1 of a step; `beside(g)`: what else is done beside block g.  next: the next step's stage, if its
  // first fragments are to be read beside the last block (it is complete by then).
  auto multiply = [&](const char *stage, auto next, auto from, auto to, auto beside) {
    constexpr bool HAS_NEXT = !std::is_same<decltype(next), std::nullptr_t>::value;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = from.value; g < to.value; g++) {
      if (g + AHEAD < TM) read_a(stage, g + AHEAD);
      else if constexpr (HAS_NEXT) read_a(next, g + AHEAD - TM);
      beside(g);
      const auto a_now = f8_fragment<Cfg::EXACT, false>(fa[g % A_RING]);
#pragma unroll
      for (int j = 0; j < TN; j++) {
        const int q = g * TN + j;
        sums[q % RING] = f8_block<Cfg::E>(a_now, fb[j]);
        if (q >= DELAY) take(q - DELAY, now);
        else take(q - DELAY + MFMAS, old);
        hold(q >= DELAY ? q - DELAY : q - DELAY + MFMAS);
        if constexpr (HAS_NEXT) {
          // (the columns' next fragments take the place of the ones just used: there are no registers for both)
          __builtin_amdgcn_sched_barrier(0);
          if (g + 1 == TM) read_b(next, j);
        }
      }
      if constexpr (HAS_NEXT) {
        if (g + 1 == TM) read_scales(next);
      }
      if constexpr (!HAS_NEXT) {
#pragma unroll
        for (int j = 0; j < TN; j++) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); // MFMA
          __builtin_amdgcn_sched_group_barrier(0x002, 5, 0); // vector
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0); // LDS reads
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto nothing = [](int) {};
  constexpr std::integral_constant<int, 0> first;
  constexpr std::integral_constant<int, TM - AHEAD> last;
  constexpr std::integral_constant<int, TM> end;

  // ---- K loop ----
  const int whole = (int)(w.klen / 128), left = (int)w.klen - whole * 128;
  const int partial = left != 0, steps = whole + partial;
  if constexpr (Cfg::DIRECT) {
    // as multiply_tile's: a K that ends inside a step has that step first; one barrier a step, in front of its last row block
    auto block_of = [&](int s) -> uint64_t { return s < partial ? whole : s - partial; };
    uint32_t offb[UB];
    typedef typename std::conditional<Cfg::GATED && LA::LINES, uint64_t, uint32_t>::type offa_t;
    offa_t offa[LA::U];
#pragma unroll
    for (int u = 0; u < LA::U; u++) offa[u] = (offa_t)LA::offset(tid + u * NT, args.lda, w.rows_a);
#pragma unroll
    for (int u = 0; u < UB; u++) offb[u] = (uint32_t)LB::offset(tid + u * NT, args.ldb, w.rows_b);
    constexpr int LOADS = LA::U + UB + 1;
    const uint32_t lds0 = lds_address(lds);
    auto issue = [&](int l, const char *pa, const char *pb, const char *ps, uint32_t stage) {
      if (l < LA::U) LA::direct(l, pa, offa[l], stage, wave);
      else if (l < LA::U + UB) LB::direct(l - LA::U, pb, offb[l - LA::U], stage + Cfg::A_STAGE, wave);
      else f8_direct_scales(ps, stage + scale_to);
    };
    // (what the compiler has loaded is waited for here: a wait of its own inside the loop would be one for all loads)
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    for (int s = 0; s < Cfg::NSTAGE && s < steps; s++) {
      const uint32_t stage = lds0 + s * Cfg::STAGE;
      const char *pa = a + block_of(s) * a_step, *pb = b + block_of(s) * b_step, *ps = scale + block_of(s) * scale_step;
      if (s < partial) {
#pragma unroll
        for (int u = 0; u < LA::U; u++) LA::direct_tail(u, pa, offa[u], stage, tid, wave, left);
#pragma unroll
        for (int u = 0; u < UB; u++) LB::direct_tail(u, pb, offb[u], stage + Cfg::A_STAGE, tid, wave, left);
        issue(LOADS - 1, pa, pb, ps, stage);
      } else {
#pragma unroll
        for (int l = 0; l < LOADS; l++) issue(l, pa, pb, ps, stage);
      }
    }
    if (steps > 0) {
      if (steps >= Cfg::NSTAGE) __builtin_amdgcn_s_waitcnt(waitcnt_vm(LOADS * (Cfg::NSTAGE - 1)));
      else __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      block_sync_lds();
      begin(lds);
    }
    constexpr int SPREAD = TM / 2 > AHEAD ? TM / 2 : AHEAD; // a step's loads are spread over half of one
    int at = 0, before = 0; // buffers of steps s and s - 1
    const char *qa = uniform_address(a + block_of(Cfg::NSTAGE) * a_step), *qb = uniform_address(b + block_of(Cfg::NSTAGE) * b_step);
    const char *qs = scale + block_of(Cfg::NSTAGE) * scale_step; // of step s + NSTAGE
    for (int s = 0; s < steps; s++) {
      const int next = at + 1 == Cfg::NSTAGE ? 0 : at + 1;
      const char *here = lds + at * Cfg::STAGE;
      const bool rest = s > 0 && s - 1 + Cfg::NSTAGE < steps; // of what was begun beside the last row block of the step before
      const char *pa = qa - a_step, *pb = qb - b_step, *ps = qs - scale_step;
      const uint32_t old_stage = lds0 + before * Cfg::STAGE;
      enter();
      multiply(here, nullptr, first, last, [&](int g) {
        if (rest) {
#pragma unroll
          for (int l = 0; l < LOADS; l++)
            if (l * SPREAD / LOADS == g + AHEAD) issue(l, pa, pb, ps, old_stage);
        }
      });
      if (s + Cfg::NSTAGE <= steps) __builtin_amdgcn_s_waitcnt(waitcnt_vm(LOADS * (Cfg::NSTAGE - 2)));
      else __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      block_sync_lds();
      const uint32_t stage = lds0 + at * Cfg::STAGE;
      const bool more = s + Cfg::NSTAGE < steps;
      // (behind the last step, unused values are read)
      multiply(here, (const char *)lds + next * Cfg::STAGE, last, end, [&](int g) {
        if (more) {
#pragma unroll
          for (int l = 0; l < LOADS; l++)
            if (l * SPREAD / LOADS == g - last.value) issue(l, qa, qb, qs, stage);
        }
      });
      qa += a_step;
      qb += b_step;
      qs += scale_step;
      before = at;
      at = next;
    }
  } else {
    // any alignment: through registers, the next step's values on their way beside this one's MFMAs
    static_assert(Cfg::NSTAGE == 2, "two buffers");
    typename LA::Regs ra;
    typename LB::Regs rb;
    float rs = 0.0f;
    uint64_t apart = 0;
    if constexpr (Cfg::GATED && LA::LINES) apart = (uint64_t)(w.up - w.a);
    // PLAIN: whole steps without the checks that the last one needs.  (128 x 128 tiles with exact sums have no registers for the
    // offsets.  4225 tokens of 8 experts, 1024 x 1016: 21.0 us, so 16.4.)
    constexpr bool PLAIN = !Cfg::EXACT || BN < 128;
    uint64_t offa[LA::U], offb[UB];
    if constexpr (PLAIN) {
#pragma unroll
      for (int u = 0; u < LA::U; u++) offa[u] = LA::offset(tid + u * NT, args.lda, w.rows_a, apart);
#pragma unroll
      for (int u = 0; u < UB; u++) offb[u] = LB::offset(tid + u * NT, args.ldb, w.rows_b);
    }
    const bool short_lines = !Cfg::A_KC && (args.m < (uint32_t)T::CHUNK || args.lda < (uint64_t)T::CHUNK);
    auto ask = [&](int s) {
      const int have = (int)w.klen - s * 128;
      const char *pa = a + (uint64_t)s * a_step, *pb = b + (uint64_t)s * b_step;
      // (not the matrix's last lines, whose chunks must not be read beyond its end)
      if (PLAIN && have >= (Cfg::A_KC ? 128 : 129) && !short_lines) {
#pragma unroll
        for (int u = 0; u < LA::U; u++) LA::template fetch<false, false>(ra, u, pa, args.lda, offa[u], w.rows_a, 0, tid);
#pragma unroll
        for (int u = 0; u < UB; u++) LB::template fetch<false, false>(rb, u, pb, args.ldb, offb[u], w.rows_b, 0, tid);
      } else {
#pragma unroll
        for (int u = 0; u < LA::U; u++)
          LA::fetch_tail(ra, u, pa, args.lda, w.rows_a, have, Cfg::A_KC ? w.safe_a : w.safe_a - s * 128, tid, apart);
#pragma unroll
        for (int u = 0; u < UB; u++) LB::fetch_tail(rb, u, pb, args.ldb, w.rows_b, have, w.safe_b, tid);
      }
      rs = *reinterpret_cast<const float *>(scale + (uint64_t)s * scale_step);
    };
    auto put = [&](char *stage) {
#pragma unroll
      for (int u = 0; u < LA::U; u++) LA::put(ra, u, stage, tid);
#pragma unroll
      for (int u = 0; u < UB; u++) LB::put(rb, u, stage + Cfg::A_STAGE, tid);
      reinterpret_cast<float *>(stage + scale_to)[lane] = rs;
    };
    if (steps > 0) {
      ask(0);
      put(lds);
      block_sync_lds();
    }
    for (int s = 0; s < steps; s++) {
      const char *here = lds + (s & 1) * Cfg::STAGE;
      if (s + 1 < steps) ask(s + 1);
      begin(here);
      enter();
      multiply(here, nullptr, first, end, nothing);
      if (s + 1 < steps) put(lds + ((s + 1) & 1) * Cfg::STAGE);
      block_sync_lds();
    }
  }
#pragma unroll
  for (int q = MFMAS - DELAY; q < MFMAS; q++) take(q, now);

  write_tile<Cfg, TN>(
      args, w, lds, [&](const int j, const int i, const int v) { return acc[j][i][v]; },
      [&]() {
#pragma unroll
        for (int j = 0; j + 1 < TN; j++)
#pragma unroll
          for (int i = 0; i < TM; i++) acc[j][i] = acc[j + 1][i];
      });
}

template <class Cfg>
__global__ __launch_bounds__(Cfg::NT) __attribute__((amdgpu_waves_per_eu(Cfg::OCC, Cfg::OCC)))
void f8_kernel(const GroupedArgs args) {
  constexpr int BN = Cfg::BN, TN = Cfg::TN;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const uint32_t tiles_m = (args.m + Cfg::ROWS_OUT - 1) / Cfg::ROWS_OUT;
  TilePlace t;
  if (!place_tile(args, blockIdx.x, tiles_m, BN, t)) return;
  TileWork w;
  w.c = args.c;
  w.n0 = t.lo + t.tn * BN;
  w.n_end = t.hi;
  w.klen = args.k;
  w.group = t.group;
  w.m0 = t.tm * Cfg::ROWS_OUT;
  w.rows_a = (int)(args.m - w.m0 < (uint32_t)Cfg::ROWS_OUT ? args.m - w.m0 : Cfg::ROWS_OUT);
  w.rows_b = (int)(w.n_end - w.n0 < (uint32_t)BN ? w.n_end - w.n0 : BN);
  w.a = uniform_address(args.a + (uint64_t)t.group * args.stride_a + (Cfg::A_KC ? (uint64_t)w.m0 * args.lda : (uint64_t)w.m0));
  if constexpr (Cfg::GATED) w.up = uniform_address(w.a + (args.up - args.a));
  w.b = uniform_address(args.b + (uint64_t)w.n0 * args.ldb);
  // rows (lines) whose 16-byte chunks may be read whole, since another follows that is as long
  const bool chunk_a = (Cfg::A_KC ? args.k : args.m) >= 16 && args.lda >= 16;
  w.safe_a = !chunk_a ? 0 : Cfg::A_KC ? (int64_t)args.m - w.m0 - 1 : (int64_t)args.k - 1;
  w.safe_b = args.k >= 16 && args.ldb >= 16 ? (int64_t)args.n - w.n0 - 1 : 0;
  static_assert(TN == 2 || TN == 4, "column blocks of a wave");
  const int blocks = (w.rows_b + 16 * Cfg::WAVES_N - 1) / (16 * Cfg::WAVES_N);
  if (blocks >= TN) multiply_f8_tile<Cfg, TN>(args, w, lds);
  else if (blocks == 1) multiply_f8_tile<Cfg, 1>(args, w, lds);
  else if constexpr (TN == 4) {
    if (blocks == 2) multiply_f8_tile<Cfg, 2>(args, w, lds);
    else multiply_f8_tile<Cfg, 3>(args, w, lds);
  }
}

template <class Cfg> void launch_f8(const GroupedArgs &args, uint32_t workgroups, hipStream_t stream) {
  static device_flags_t done = {};
  allow_dynamic_lds(reinterpret_cast<const void *>(&f8_kernel<Cfg>), Cfg::LDS_BYTES, done);
  hipLaunchKernelGGL(f8_kernel<Cfg>, dim3(workgroups), dim3(Cfg::NT), Cfg::LDS_BYTES, stream, args);
}
template <Elem E, bool A_KC, int BM, int BN, int WM, int WN, int NSTAGE, bool DIRECT, Epilogue EPI, bool EXACT>
constexpr GroupedKernel f8_entry() {
  using Cfg = F8Cfg<E, A_KC, BM, BN, WM, WN, NSTAGE, DIRECT, EPI, EXACT>;
  return {&launch_f8<Cfg>, Cfg::ROWS_OUT, Cfg::BN, Cfg::NT};
}

// ---- few tokens: the matrices are read once, straight into MFMA fragments (grouped_stream.hpp) ----
// Sixteen rows (of both matrices, for a gated block) and up to sixteen tokens for a workgroup of eight waves, which take the
// blocks of K in turn.  K-contiguous matrices only.
template <Elem E, Epilogue EPI>
__global__ __launch_bounds__(kStreamWaves * 64) void f8_stream_kernel(const GroupedArgs args) {
  constexpr int SIDES = EPI == Epilogue::GATED ? 2 : 1, ROWS = 16;
  __shared__ __attribute__((aligned(16))) float sums[SIDES][kStreamWaves][kStreamTokens][ROWS + 4];
  const int tid = threadIdx.x, lane = tid & 63, frow = lane & 15, fg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  TilePlace t;
  if (!place_tile(args, blockIdx.x, (args.m + ROWS - 1) / ROWS, kStreamTokens, t)) return;
  const uint32_t m0 = t.tm * ROWS, n0 = t.lo + t.tn * kStreamTokens;
  const uint32_t tokens = t.hi - n0 < kStreamTokens ? t.hi - n0 : kStreamTokens;
  const uint32_t row = m0 + frow < args.m ? m0 + frow : args.m - 1;
  const uint32_t token = n0 + ((uint32_t)frow < tokens ? frow : tokens - 1); // (beyond the last: that again, not stored)
  const F8Scales sc(args);
  const char *pa[SIDES];
  const float *row_scale[SIDES];
#pragma unroll
  for (int side = 0; side < SIDES; side++) {
    pa[side] = (side ? args.up : args.a) + (uint64_t)t.group * args.stride_a + (uint64_t)row * args.lda + fg * 16;
    row_scale[side] = sc.of_rows<true>(side ? args.scale_up : args.scale_a, args, t.group, m0 / 128);
  }
  const char *pb = args.b + (uint64_t)token * args.ldb + fg * 16;
  const float *token_scale = args.scale_b + (uint64_t)token * sc.kb;
  f4v_t acc[SIDES];
#pragma unroll
  for (int side = 0; side < SIDES; side++) acc[side] = f4v_t{0.0f, 0.0f, 0.0f, 0.0f};
  struct Step {
    stream_raw<E> a[SIDES][2], b[2];
    float rows[SIDES], tokens;
  };
  auto load = [&](Step &x, int s) {
    const uint64_t at = (uint64_t)s * 128;
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int side = 0; side < SIDES; side++) x.a[side][h] = stream_load<E>(pa[side] + at + h * 64);
      x.b[h] = stream_load<E>(pb + at + h * 64);
    }
#pragma unroll
    for (int side = 0; side < SIDES; side++) x.rows[side] = row_scale[side][s];
    x.tokens = token_scale[s];
  };
  auto both = [](const stream_raw<E> &x, const stream_raw<E> &y) {
    return i8v_t{(int)x.v.x, (int)x.v.y, (int)x.v.z, (int)x.v.w, (int)y.v.x, (int)y.v.y, (int)y.v.z, (int)y.v.w};
  };
  auto take = [&](const Step &x) { // (exact: bound by memory)
    const F8Wide fb = f8_fragment<true, E == Elem::E5M2>(both(x.b[0], x.b[1]));
#pragma unroll
    for (int side = 0; side < SIDES; side++) {
      const f4v_t y = f8_block<E>(f8_fragment<true, false>(both(x.a[side][0], x.a[side][1])), fb);
      const float s = x.tokens * x.rows[side];
#pragma unroll
      for (int v = 0; v < 4; v++) acc[side][v] = fmaf(y[v], s, acc[side][v]);
    }
  };
  const int whole = (int)(args.k / 128), left = (int)(args.k % 128);
  int s = wave;
  auto several = [&](auto count) {
    constexpr int U = decltype(count)::value;
    for (; s + (U - 1) * kStreamWaves < whole; s += U * kStreamWaves) {
      Step x[U];
#pragma unroll
      for (int u = 0; u < U; u++) load(x[u], s + u * kStreamWaves);
#pragma unroll
      for (int u = 0; u < U; u++) take(x[u]);
    }
  };
  several(std::integral_constant<int, 4>{});
  several(std::integral_constant<int, 2>{});
  several(std::integral_constant<int, 1>{});
  if (left != 0 && s == whole) { // the last, partial block belongs to the wave whose turn it is
    Step x;
    const uint64_t at = (uint64_t)whole * 128;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int have = left - (h * 4 + fg) * 16;
#pragma unroll
      for (int side = 0; side < SIDES; side++) x.a[side][h] = stream_load_part<E>(pa[side] + at + h * 64, have);
      x.b[h] = stream_load_part<E>(pb + at + h * 64, have);
    }
#pragma unroll
    for (int side = 0; side < SIDES; side++) x.rows[side] = row_scale[side][whole];
    x.tokens = token_scale[whole];
    take(x);
  }

  // ---- sums of the waves, in their order ----
#pragma unroll
  for (int side = 0; side < SIDES; side++)
#pragma unroll
    for (int v = 0; v < 4; v++) sums[side][wave][frow][4 * fg + v] = acc[side][v];
  __syncthreads();
  const uint32_t r = tid % ROWS, j = tid / ROWS;
  if (j >= tokens || m0 + r >= args.m) return;
  float x[SIDES];
#pragma unroll
  for (int side = 0; side < SIDES; side++) {
    x[side] = 0.0f;
#pragma unroll
    for (int w = 0; w < kStreamWaves; w++) x[side] += sums[side][w][j][r];
  }
  float y = x[0];
  if constexpr (EPI == Epilogue::GATED) {
    with_activation(args.act, [&](auto act) {
      float slope;
      const float a = args.out == OUT_F32 ? activation<act.value, true, false>(x[0], slope) : activation<act.value, false, false>(x[0], slope);
      y = a * x[SIDES - 1];
    });
  }
  const uint64_t at = (uint64_t)(n0 + j) * args.ldc + m0 + r;
  if (args.out == OUT_F32) reinterpret_cast<float *>(args.c)[at] = y;
  else if (args.out == OUT_F16) reinterpret_cast<_Float16 *>(args.c)[at] = (_Float16)y;
  else reinterpret_cast<__bf16 *>(args.c)[at] = (__bf16)y;
}
template <Elem E, Epilogue EPI> void launch_f8_stream(const GroupedArgs &args, uint32_t workgroups, hipStream_t stream) {
  hipLaunchKernelGGL((f8_stream_kernel<E, EPI>), dim3(workgroups), dim3(kStreamWaves * 64), 0, stream, args);
}

// ---- tables ----
// Tiles of 32 tokens wait for memory, and are exact.  Exact sums have no 256 x 256 tile (its fragments in BF16 leave too few
// registers, and with fewer results under way it was 2 - 9 % faster at best: 8192 tokens, 4096 x 4096 240 us for 262), and for lines
// of any alignment no 128 x 128 one, which spills, but one of 64 tokens, which rows of any alignment have as well (1531 tokens, 2047 x
// 1535 25.6 us for 32.5; 8192, 4095 x 4095 446 for 333).
template <Elem E, Epilogue EPI, bool A_KC, bool EXACT> constexpr void f8_entries(GroupedTable &t) {
  if constexpr (A_KC || !EXACT) t.columns[A_KC][0][TILE_128] = f8_entry<E, A_KC, 128, 128, 64, 64, 2, false, EPI, EXACT>();
  if constexpr (EXACT) t.columns[A_KC][0][TILE_64] = f8_entry<E, A_KC, 128, 64, 64, 32, 2, false, EPI, true>();
  t.columns[A_KC][0][TILE_NARROW] = f8_entry<E, A_KC, 128, 32, 32, 32, 2, false, EPI, true>();
  if constexpr (!EXACT) t.columns[A_KC][1][TILE_256] = f8_entry<E, A_KC, 256, 256, 128, 64, 2, true, EPI, false>();
  t.columns[A_KC][1][TILE_128] = f8_entry<E, A_KC, 128, 128, 64, 64, 2, true, EPI, EXACT>();
  t.columns[A_KC][1][TILE_NARROW] = f8_entry<E, A_KC, 128, 32, 32, 32, 3, true, EPI, true>();
  t.columns[A_KC][1][TILE_64] = f8_entry<E, A_KC, 128, 64, 64, 32, 3, true, EPI, EXACT>();
  if constexpr (A_KC) t.stream[A_KC] = {&launch_f8_stream<E, EPI>, 16, kStreamTokens, kStreamWaves * 64};
}
template <Elem E, bool EXACT> constexpr GroupedTable f8_table() {
  GroupedTable t{};
  f8_entries<E, Epilogue::STORE, false, EXACT>(t);
  f8_entries<E, Epilogue::STORE, true, EXACT>(t);
  return t;
}
template <Elem E, bool EXACT> constexpr GroupedTable gated_f8_table() {
  GroupedTable t{};
  f8_entries<E, Epilogue::GATED, true, EXACT>(t);
  return t;
}

#define CUMPSGEMM_F8(kind, E)                                        \
  GroupedTable g_f8_##kind = f8_table<E, false>();                   \
  GroupedTable g_f8_exact_##kind = f8_table<E, true>();              \
  GroupedTable g_gated_f8_##kind = gated_f8_table<E, false>();       \
  GroupedTable g_gated_f8_exact_##kind = gated_f8_table<E, true>();

} // namespace cumpsgemm_amd
