// Tiled kernels of the experts' products (gfx950, wave64).
//
// One workgroup computes a BM x BN tile of one group's result.  A K-step of both operands lies in LDS, in NSTAGE
// buffers; fragments are read from there and multiplied with 16-row MFMAs, whose rows are rows of C (m) and whose
// columns are tokens (n), so that a lane holds four results next to each other in memory.
//
// LDS images of an operand's K-step (ROWS rows of C or tokens):
//   K-contiguous: ROWS rows of ROW_BYTES bytes (128 or 64) of 16-bit or 8-bit values; 64 bytes (32 values) in each
//     plane of a split FP32 operand.  The 16-byte chunks of a row are exchanged (chunk ^ f(row)) so that the sixteen
//     rows that one part of a ds_read_b128 touches fall on sixteen different bank groups.
//   row-contiguous (16-bit operands whose rows, not K, are contiguous: op N weights, and both operands of the
//     weights' gradient): BK lines of ROWS values, as they come from memory.  ds_read_b64_tr_b16 reads four lines of
//     sixteen rows and hands each lane one row's four K-values, so nothing is transposed by vector instructions.
//     The 32-byte pieces of a line are exchanged by two line bits and one of the eight-line bits: the sixteen lines of
//     one read cover all banks twice, the least that 512 bytes can.
// FP32 operands are split while they are staged, whatever their layout: a thread reads eight K-values of one row and
// writes one chunk to each plane.
//
// What it spends its time on, as far as measurements tell (us).  BF16, 16384 tokens of 8 experts, 4096 x 2048: 272 with uneven
// experts, 230 with even ones, which are whole rounds of tiles, 190 on zeros, which leave the clock higher (random values:
// 1.98 GHz, 44 % of it MFMAs); rows padded by 64 or 192 values are level.  8 bits, 8192 x 4096: 23.4 a thousand K-values
// (2870 TOP/s) and 27 beside that, a tile's first loads, its write-out and the launch: at K = 4096 123, 2230 TOP/s.  FP16TCEC,
// 4096 tokens of 8, 2048 x 1024: 78 with uneven experts in 128 x 128 tiles, 60 with even ones (256 x 128 tiles: 54, zeros 44);
// 28 % MFMAs, and beside them as many clocks of LDS reads, which the schedule does not hide whole.
#pragma once
#include "gemm_kernel.hpp"
#include "grouped.hpp"
#include "gemm_table.hpp"

namespace cumpsgemm_amd {

typedef int i4_t __attribute__((ext_vector_type(4)));

template <Elem E> struct elem_traits {
  static constexpr bool F32 = (int)E <= 3;
  static constexpr bool I8 = E == Elem::I8;
  static constexpr Prec P = F32 ? (Prec)(int)E : Prec::FP16TC;
  static constexpr bool IS_BF16 = F32 ? prec_traits<P>::IS_BF16 : E == Elem::BF16;
  static constexpr int BYTES = F32 ? 4 : I8 ? 1 : 2; // of an element in memory
  static constexpr int NP = F32 ? prec_traits<P>::NP : 1;
  static constexpr int NPROD = F32 ? prec_traits<P>::NPROD : 1;
  static constexpr int NACC = F32 ? prec_traits<P>::NACC : 1;
  static constexpr int CHUNK = I8 ? 16 : 8;         // K-values of a 16-byte chunk in LDS
  typedef typename std::conditional<I8, i4_t, f4v_t>::type acc_t;
};

// 16 zero bytes: where a lane reads that has nothing to read (a K-value past the end)
static __device__ const u4_t g_grouped_zeros = {0, 0, 0, 0};

// offset of a 16-byte chunk in a K-contiguous image
template <int ROW_BYTES> __device__ inline int row_swizzle(int row) {
  return ROW_BYTES == 64 ? lds_swizzle(row) : (row >> 1) & 7;
}
template <int ROW_BYTES> __device__ inline int chunk_offset(int row, int chunk) {
  return row * ROW_BYTES + ((chunk ^ row_swizzle<ROW_BYTES>(row)) << 4);
}
// what M0 holds for a load to LDS (wave-uniform)
__device__ inline uint32_t lds_address(const char *p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p);
}
// an address that is the same for all lanes, whatever the compiler can see of that
// (and one of global memory: a pointer made of a number would be read with flat loads, which wait for LDS as well)
__device__ inline const char *uniform_address(const char *p) {
  const uint64_t x = (uint64_t)p;
  const uint32_t high = __builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)), low = __builtin_amdgcn_readfirstlane((uint32_t)x);
  typedef const char __attribute__((address_space(1))) *gptr_t;
  return (const char *)(gptr_t)((uint64_t)high << 32 | low); // (low is unsigned here: the builtin's own int would carry its sign up)
}
// which 32-byte piece of line k holds piece p of a row-contiguous image
__device__ inline int line_swizzle(int k) { return (k & 3) | (((k >> 3) & 1) << 2); }

// A tile's place: its group, and where that begins and ends.
struct TilePlace {
  uint32_t group, tm, tn;
  uint32_t lo, hi; // tokens of the group
};

// One group's tokens, brought into [0, count] and into order.
__device__ inline void group_span(const int *offsets, uint32_t g, uint32_t count, uint32_t &lo, uint32_t &hi) {
  const int a = offsets[g], b = offsets[g + 1], c = (int)count;
  const int l = a < 0 ? 0 : a > c ? c : a;
  lo = (uint32_t)l;
  hi = (uint32_t)(b < l ? l : b > c ? c : b);
}

__device__ inline uint32_t wave_inclusive_sum(uint32_t x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

// Workgroups that the dispatcher places on one XCD (id mod 8) take one contiguous range of the list of tiles, so that
// they share that XCD's L2.
__device__ inline uint32_t xcd_range(uint32_t bid, uint32_t total) {
  if (total < 32) return bid;
  const uint32_t q = total / 8, r = total % 8, xcd = bid % 8, loc = bid / 8;
  return xcd * q + (xcd < r ? xcd : r) + loc;
}
// Column groups of up to 8 tile rows within one group's tiles: compact patches.
__device__ inline void raster(uint32_t in, uint32_t tiles_m, uint32_t tiles_n, uint32_t &tm, uint32_t &tn) {
  const uint32_t per = 8 * tiles_n, first = in / per * 8, rows = tiles_m - first < 8 ? tiles_m - first : 8;
  const uint32_t rest = in % per;
  tm = first + rest % rows;
  tn = rest / rows;
}

// Ragged columns: the tile of workgroup `bid` in the list of all groups' tiles: whole columns of tiles first, then the
// groups' last columns, which have fewer than bn tokens and take less time, so that what keeps some CUs longest is short.
// (Every wave works it out for itself, 64 groups at a time, one a lane.)  False: there are fewer tiles.
__device__ inline bool place_tile(const GroupedArgs &args, uint32_t bid, uint32_t tiles_m, uint32_t bn, TilePlace &t) {
  const int lane = threadIdx.x & 63;
  auto span_of = [&](uint32_t g, uint32_t &lo, uint32_t &hi) {
    lo = hi = 0;
    if (g >= args.groups) return;
    if (args.offsets != nullptr) group_span(args.offsets, g, args.n, lo, hi);
    else hi = args.n;
  };
  // a lane's group: its span, how many whole columns, how many of the 64 groups up to it have in all
  uint32_t lo, hi, full, sum;
  auto look = [&](uint32_t g0) {
    span_of(g0 + lane, lo, hi);
    full = (hi - lo) / bn;
    // (few tokens to a group: no group has a whole column, and nothing is to be added)
    sum = __ballot(full != 0) != 0 ? wave_inclusive_sum(full, lane) : 0;
  };
  uint32_t whole = 0, last = 0; // columns of tiles, of all groups
  for (uint32_t g0 = 0; g0 < args.groups; g0 += 64) {
    look(g0);
    whole += __builtin_amdgcn_readlane(sum, 63);
    last += __builtin_popcountll(__ballot((hi - lo) % bn != 0));
  }
  const bool in_whole = bid < whole * tiles_m;
  if (!in_whole && bid - whole * tiles_m >= last * tiles_m) return false;
  const uint32_t id = in_whole ? xcd_range(bid, whole * tiles_m) : xcd_range(bid - whole * tiles_m, last * tiles_m);
  const uint32_t column = id / tiles_m;
  uint32_t before = 0;
  for (uint32_t g0 = 0; g0 < args.groups; g0 += 64) {
    if (args.groups > 64) look(g0); // (or they are still there)
    const uint64_t rest = __ballot((hi - lo) % bn != 0);
    // columns up to this group's last: whole ones, or last ones
    const uint32_t upto = before + (in_whole ? sum : (uint32_t)__builtin_popcountll(rest & (~0ull >> (63 - lane))));
    const uint64_t beyond = __ballot(column < upto);
    if (beyond != 0) {
      const int at = __builtin_ctzll(beyond);
      t.group = g0 + at;
      t.lo = __builtin_amdgcn_readlane(lo, at);
      t.hi = __builtin_amdgcn_readlane(hi, at);
      if (in_whole) {
        const uint32_t tiles_n = __builtin_amdgcn_readlane(full, at);
        raster(id - (__builtin_amdgcn_readlane(upto, at) - tiles_n) * tiles_m, tiles_m, tiles_n, t.tm, t.tn);
      } else {
        t.tm = id % tiles_m;
        t.tn = __builtin_amdgcn_readlane(full, at);
      }
      // (offsets out of order can make these sums overflow: no tile outside its group)
      return t.tm < tiles_m && (uint64_t)t.tn * bn < t.hi - t.lo;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// Over K: the tile of workgroup `bid` and its part of K.  False: there is none.  The groups' results are equally many
// tiles, but take as long as the groups are.  Each XCD (id mod 8) gets shares of several groups' tiles (deal_over_k), and
// the longest groups come first, so that short ones are left for the CUs that are done early: 8 uneven experts, 16384
// tokens, 4096 x 2048 in BF16: 307 us; the groups' tiles in contiguous ranges, as for ragged columns, 416 us (even ones:
// 266 and 293 us).
__device__ inline bool place_over_k(const GroupedArgs &args, uint32_t bid, uint32_t tiles_m, uint32_t tiles_n, TilePlace &t,
                                    uint32_t &split) {
  const uint32_t lists = args.groups * args.splits, per = tiles_m * tiles_n;
  const DealOverK d = deal_over_k(per, lists, args.groups);
  const uint32_t turn = bid / 8 / d.most, in = bid / 8 - turn * d.most, xcd = bid % 8;
  // (every other turn goes the other way round)
  const uint32_t share = turn * 8 + (turn % 2 ? 7 - xcd : xcd);
  const uint32_t list = share >> d.log2_shares, part = share & ((1u << d.log2_shares) - 1);
  if (list >= lists) return false;
  const uint32_t tile = ((part * per) >> d.log2_shares) + in;
  if (tile >= ((part + 1) * per) >> d.log2_shares) return false;
  raster(tile, tiles_m, tiles_n, t.tm, t.tn);
  t.group = args.splits == 1 ? list : list / args.splits;
  split = args.splits == 1 ? 0 : list % args.splits;
  // In place of a group's number its rank, by length in quarters of the mean.  (Not if all tiles are begun at once.  More
  // groups: their lengths even out; short ones: looking takes as long as they do.)
  if (args.groups > 1 && args.groups <= 64 && args.k / 128 >= args.groups && (uint64_t)per * lists > 256) {
    const uint32_t lane = threadIdx.x & 63, quarter = args.k / args.groups / 4;
    uint32_t lo = 0, hi = 0;
    if (lane < args.groups) group_span(args.offsets, lane, args.k, lo, hi);
    uint64_t longer = 0, as_long;
    for (uint32_t least = 8 * quarter;; least -= quarter) {
      if (least < quarter) least = 0;
      as_long = __ballot(lane < args.groups && hi - lo >= least);
      if (least == 0 || (uint32_t)__builtin_popcountll(as_long) > t.group) break;
      longer = as_long;
    }
    const uint32_t rank = t.group - (uint32_t)__builtin_popcountll(longer);
    as_long &= ~longer;
    const uint32_t before = __builtin_amdgcn_mbcnt_hi((uint32_t)(as_long >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)as_long, 0));
    t.group = __builtin_ctzll(__ballot((as_long >> lane & 1) != 0 && before == rank));
  }
  return true;
}

// DIRECT: 16-bit and 8-bit operands go straight from memory to LDS, 16 aligned bytes a lane; FP32 operands, which are
// split in registers, are read with 32-bit offsets from uniform bases.  Otherwise: any alignment, any size; but lines of
// 16-bit values that are shorter than a chunk are for the CAREFUL kernels.
template <Elem E_, bool A_KC_, bool B_KC_, int BM_, int BN_, int WM_, int WN_, int ROW_BYTES_, int NSTAGE_, bool DIRECT_,
          bool RAGGED_K_, int OCC_, bool CAREFUL_>
struct GroupedCfg {
  using T = elem_traits<E_>;
  static constexpr Elem E = E_;
  static constexpr bool A_KC = A_KC_, B_KC = B_KC_, DIRECT = DIRECT_, RAGGED_K = RAGGED_K_, CAREFUL = CAREFUL_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NSTAGE = NSTAGE_, OCC = OCC_;
  static constexpr int WAVES_M = BM / WM, WAVES_N = BN / WN, NT = WAVES_M * WAVES_N * 64;
  static constexpr int TM = WM / 16, TN = WN / 16;
  static constexpr int ROW_BYTES = ROW_BYTES_;
  static constexpr int BK = ROW_BYTES / 16 * T::CHUNK; // K-values of a step
  static constexpr int SLICES = ROW_BYTES / 64;        // MFMAs deep
  static_assert(ROW_BYTES == 64 || (ROW_BYTES == 128 && !T::F32), "rows in LDS");
  static constexpr int A_PLANE = BM * ROW_BYTES, B_PLANE = BN * ROW_BYTES;
  static constexpr int A_STAGE = A_PLANE * T::NP, B_STAGE = B_PLANE * T::NP, STAGE = A_STAGE + B_STAGE;
  // (the results pass through LDS: sixteen columns of each wave at a time, four floats further
  // apart than they are long, so that sixteen columns' pieces fall on different banks)
  static constexpr int PITCH = WM + 4, OUT_BYTES = WAVES_M * WAVES_N * 16 * PITCH * 4;
  static constexpr int LDS_BYTES = NSTAGE * STAGE > OUT_BYTES ? NSTAGE * STAGE : OUT_BYTES;
  static_assert(!T::I8 || (A_KC && B_KC), "8-bit integers: K-contiguous operands");
  static_assert(A_KC || T::F32 || BM >= 128, "a line's pieces are exchanged among eight");
  static_assert(B_KC || T::F32 || BN >= 128, "a line's pieces are exchanged among eight");
  static_assert(LDS_BYTES <= 160 * 1024, "LDS");
  // (the waits of the direct form count a step's loads, the same number for every wave)
  static_assert(!DIRECT || T::F32 || (BM * ROW_BYTES / 16 % NT == 0 && BN * ROW_BYTES / 16 % NT == 0), "whole rounds of loads");
};

// (M0 is among the registers that the loads below say they change; nothing of the compiler's lives in it longer than
// from one instruction to the next, which is what it warns of)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Staging of one operand's K-step by NT threads.  A unit is one 16-byte chunk of LDS (FP32: one in each plane).
template <Elem E, bool KC, int ROWS, int ROW_BYTES, int NT> struct grouped_loader {
  using T = elem_traits<E>;
  // row-contiguous images exist for 16-bit values only; FP32 ends in K-contiguous planes either way
  static constexpr bool LINES = !KC && !T::F32;
  static constexpr int UNITS = ROWS * ROW_BYTES / 16;
  static constexpr int U = (UNITS + NT - 1) / NT;
  static constexpr bool PARTIAL = UNITS < NT;
  static_assert(UNITS % NT == 0 || (PARTIAL && UNITS % 64 == 0), "whole waves");
  static constexpr int LINE_CHUNKS = ROWS / 8;            // 16-byte chunks of a line
  static constexpr int ROW_CHUNKS = ROW_BYTES / 16;

  __device__ static inline bool active(int tid) { return !PARTIAL || tid < UNITS; }

  // Position `id` of the image (in 16-byte chunks, as memory -> LDS loads fill it): row (LINES: first of 8 rows) and
  // first K-value (LINES: the line) of what lies there.
  __device__ static inline void at(int id, int &row, int &k) {
    if constexpr (LINES) {
      k = id / LINE_CHUNKS;
      const int c = id % LINE_CHUNKS;
      row = ((((c >> 1) ^ line_swizzle(k)) << 1) | (c & 1)) * 8;
    } else if constexpr (T::F32) {
      // (not an image position: FP32 chunks are written one by one, in whatever order reads memory best)
      if constexpr (KC) {
        row = id / ROW_CHUNKS;
        k = id % ROW_CHUNKS * T::CHUNK;
      } else {
        row = id % ROWS;
        k = id / ROWS * T::CHUNK;
      }
    } else {
      row = id / ROW_CHUNKS;
      k = ((id % ROW_CHUNKS) ^ row_swizzle<ROW_BYTES>(row)) * T::CHUNK;
    }
  }

  // FP32: the K-value of the step that stands at place j of the chunk of place k on.  Any order will do that both operands
  // have; with this one, four lanes' loads are 64 bytes side by side.  (As they come, every other 16: 128 x 128 tiles in one
  // term, 4096 x 2048 x 1024 in 8 groups 43.6 us, so 39.2; in two or three terms 0 - 4 %.)
  __device__ static constexpr int value_of(int k, int j) { return k / 2 + (j & 3) + (j >> 2) * 16; }

  // Byte offset from the tile's origin (row 0, K-value 0 of the step) of the unit that fills position id.
  // `rows`: those that exist; one (LINES: eight) beyond them reads the last again (its products are not stored).
  __device__ static inline uint64_t offset(int id, uint64_t ld, int rows) {
    int row, k;
    at(id, row, k);
    const int last = LINES ? (rows - 1) & ~7 : rows - 1;
    row = row < last ? row : last;
    if constexpr (T::F32) k = value_of(k, 0);
    return (KC ? (uint64_t)row * ld + k : (uint64_t)k * ld + row) * T::BYTES;
  }

  // memory -> LDS, 16 bytes a lane: load number u of a whole step, from the uniform base + off.
  // (Assembly: of such a load the compiler knows no more than that it writes LDS, and makes every read of LDS beside
  // one wait for all reads before it, and a transposing read for the loads themselves: 8 experts, 16384 x 4096 x 2048
  // over K in BF16, 898 us that way.  The kernel waits for them itself, before the barrier in front of their first
  // read; they write no register.  M0 must be written one instruction ahead, and an address that a vector instruction put
  // into scalar registers five, which the compiler does not see to here.)
  __device__ static inline void direct(int u, const char *base, uint32_t off, uint32_t lds_op, int wave) {
    const uint32_t to = lds_op + (uint32_t)((wave * 64 + u * NT) * 16);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
  }
  // ... of a step that has only `left` K-values: zeros from there on
  __device__ static inline void direct_tail(int u, const char *base, uint32_t off, uint32_t lds_op, int tid, int wave, int left) {
    int row, k;
    at(tid + u * NT, row, k);
    const char *p = k < left ? base + off : reinterpret_cast<const char *>(&g_grouped_zeros);
    const uint32_t to = lds_op + (uint32_t)((wave * 64 + u * NT) * 16);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(p) : "memory", "m0");
  }

  struct Regs {
    typename std::conditional<T::F32, f8_t, u4_t>::type v[U];
  };

  // memory -> registers, unit u of a whole step.  off: the unit's offset() from the uniform base, in 32 bits if FAST.
  // A chunk of a line (LINES) may stick out beyond the rows, into the next line: not for the matrix's last line, unless
  // CAREFUL (rows, safe: see fetch_tail).
  template <bool FAST, bool CAREFUL, class OFF>
  __device__ static inline void fetch(Regs &r, int u, const char *base, uint64_t ld, OFF off, int rows, int64_t safe, int tid) {
    if (!active(tid)) return;
    if constexpr (T::F32 && KC) {
      typedef float f4u_t __attribute__((ext_vector_type(4), aligned(4)));
      const f4u_t *p = reinterpret_cast<const f4u_t *>(base + off);
      const f4u_t x = p[0], y = p[4];
      r.v[u] = f8_t{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    } else if constexpr (T::F32 && FAST) {
      // the descriptor holds the uniform base, the scalar offset picks the K-line: no vector arithmetic
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, 0xffffffff, 0x00020000);
      const uint32_t line = __builtin_amdgcn_readfirstlane((uint32_t)ld * 4u);
#pragma unroll
      for (int j = 0; j < 8; j++)
        r.v[u][j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, value_of(0, j) * line, 0));
    } else if constexpr (T::F32) {
      const float *p = reinterpret_cast<const float *>(base + off);
#pragma unroll
      for (int j = 0; j < 8; j++) r.v[u][j] = p[(uint64_t)value_of(0, j) * ld];
    } else {
      // (rows of 16-bit values may begin anywhere: the type promises no more and leaves the instruction to the compiler)
      typedef uint32_t u4u2_t __attribute__((ext_vector_type(4), aligned(2)));
      typedef uint32_t u4u1_t __attribute__((ext_vector_type(4), aligned(1)));
      typedef typename std::conditional<T::I8, u4u1_t, u4u2_t>::type u4u_t;
      if (!LINES || !CAREFUL) {
        const u4u_t x = *reinterpret_cast<const u4u_t *>(base + off);
        r.v[u] = u4_t{x.x, x.y, x.z, x.w};
      } else {
        fetch_tail(r, u, base, ld, rows, 1 << 30, safe, tid);
      }
    }
  }

  // ... any step: `left` K-values (one at least) from its first to the end.  Zeros come in the place of K-values beyond
  // it, the last row again in that of rows.  A 16-byte chunk that sticks out beyond the last row (LINES) or K-value is
  // read whole all the same, where what follows it is the next line or row of the matrix: for the first `safe` lines
  // (rows, K-contiguous) counted from the base.  The others are read value by value.
  __device__ static inline void fetch_tail(Regs &r, int u, const char *base, uint64_t ld, int rows, int left, int64_t safe, int tid) {
    if (!active(tid)) return;
    int row, k;
    at(tid + u * NT, row, k);
    if constexpr (T::F32) {
      row = row < rows ? row : rows - 1;
      const uint64_t step = KC ? 1 : ld;
      const float *p = reinterpret_cast<const float *>(base) + (KC ? (uint64_t)row * ld : (uint64_t)row);
      // (without branches: a value past the end is read from the step's first K-value and replaced)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int at = value_of(k, j);
        const bool in = at < left;
        const float x = p[in ? (uint64_t)at * step : 0];
        r.v[u][j] = in ? x : 0.0f;
      }
    } else {
      typedef typename std::conditional<T::I8, uint8_t, uint16_t>::type V;
      typedef uint32_t u4u2_t __attribute__((ext_vector_type(4), aligned(2)));
      typedef uint32_t u4u1_t __attribute__((ext_vector_type(4), aligned(1)));
      typedef typename std::conditional<T::I8, u4u1_t, u4u2_t>::type u4u_t;
      constexpr int BITS = T::BYTES * 8, PER = 32 / BITS;
      const int last = LINES ? (rows - 1) & ~7 : rows - 1;
      row = row < last ? row : last;
      const int begins = k < left ? k : 0;               // (a chunk with nothing in it reads the step's first)
      const int keep = LINES ? (k < left ? 8 : 0) : left - k; // values of the chunk that count
      const int have = LINES ? rows - row : left - begins;    // ... that exist
      const V *p = reinterpret_cast<const V *>(base) + (KC ? (uint64_t)row * ld + begins : (uint64_t)begins * ld + row);
      u4_t x = {0, 0, 0, 0};
      if (have >= T::CHUNK || (LINES ? begins : row) < safe) {
        const u4u_t y = *reinterpret_cast<const u4u_t *>(p);
        x = u4_t{y.x, y.y, y.z, y.w};
      } else {
        for (int j = 0; j < T::CHUNK; j++)
          if (j < have) x[j / PER] |= (uint32_t)p[j] << (j % PER * BITS);
      }
#pragma unroll
      for (int d = 0; d < 4; d++) {
        const int n = keep - d * PER; // values of this word that count
        x[d] = n >= PER ? x[d] : n > 0 ? x[d] & ((1u << (n * BITS & 31)) - 1) : 0;
      }
      r.v[u] = x;
    }
  }

  // registers -> LDS
  __device__ static inline void put(const Regs &r, int u, char *lds_op, int tid) {
    if (!active(tid)) return;
    const int id = tid + u * NT;
    if constexpr (T::F32) {
      int row, k;
      at(id, row, k);
      u4_t out[T::NP];
#pragma unroll
      for (int q = 0; q < 4; q++) {
        uint32_t terms[T::NP];
        split_pair<T::P, false>(r.v[u][2 * q], r.v[u][2 * q + 1], 1.0f, 2048.0f, terms);
#pragma unroll
        for (int p = 0; p < T::NP; p++) out[p][q] = terms[p];
      }
#pragma unroll
      for (int p = 0; p < T::NP; p++)
        *reinterpret_cast<u4_t *>(lds_op + p * ROWS * ROW_BYTES + chunk_offset<ROW_BYTES>(row, k / T::CHUNK)) = out[p];
    } else {
      *reinterpret_cast<u4_t *>(lds_op + id * 16) = r.v[u];
    }
  }
};

#pragma clang diagnostic pop

template <Elem E>
__device__ inline typename elem_traits<E>::acc_t grouped_mfma(const u4_t a, const u4_t b, const typename elem_traits<E>::acc_t c) {
  if constexpr (E == Elem::I8)
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4_t, a), __builtin_bit_cast(i4_t, b), c, 0, 0, 0);
  else
    return mfma_block<elem_traits<E>::IS_BF16>(a, b, c);
}

// Results of a column, one or four of them, in the type that C has.
template <uint32_t OUT> struct out_type;
template <> struct out_type<OUT_F32> { typedef float type; };
template <> struct out_type<OUT_F16> { typedef _Float16 type; };
template <> struct out_type<OUT_BF16> { typedef __bf16 type; };

// x[0 .. 3]: rows row .. row + 3 of one column; `c`: where row `row` lies.  Not stored: rows from m on.
template <uint32_t OUT>
__device__ inline void store_four(char *c, const f4v_t x, float beta, uint32_t row, uint32_t m, bool vec) {
  typedef typename out_type<OUT>::type O;
  typedef O o4_t __attribute__((ext_vector_type(4)));
  O *p = reinterpret_cast<O *>(c);
  if (vec) { // (m is a multiple of 4)
    if (row >= m) return;
    f4v_t y = x;
    if (beta != 0.0f) {
      const o4_t old = *reinterpret_cast<const o4_t *>(p);
#pragma unroll
      for (int v = 0; v < 4; v++) y[v] += beta * (float)old[v];
    }
    *reinterpret_cast<o4_t *>(p) = __builtin_convertvector(y, o4_t);
  } else {
#pragma unroll
    for (int v = 0; v < 4; v++)
      if (row + v < m) p[v] = (O)(beta != 0.0f ? x[v] + beta * (float)p[v] : x[v]);
  }
}

// A tile's place in memory: what its loops need to know.
struct TileWork {
  const char *a, *b;       // row m0, token n0 (ragged K: column n0), K-value 0
  char *c;                 // of its group
  float *partial;          // where a part's sums go (ragged K in parts)
  uint32_t group, m0, n0, n_end, klen;
  int rows_a, rows_b;      // rows and columns that exist
  // lines (rows, K-contiguous operand) from a and b to the matrix's last but one; 0 where one is shorter than a chunk
  int64_t safe_a, safe_b;
};

// One tile, TN column blocks of 16 for each wave: all that a wave has room for, or (a group's last tile) as many as the
// tile's columns need.  The waves take column blocks in turn, so that a part of a tile is a part of every wave's work.
template <class Cfg, int TN>
__device__ inline void multiply_tile(const GroupedArgs &args, const TileWork &w, char *lds) {
  using T = typename Cfg::T;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, TM = Cfg::TM, NT = Cfg::NT, BK = Cfg::BK, RB = Cfg::ROW_BYTES, SLICES = Cfg::SLICES;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % Cfg::WAVES_M, wn = wave / Cfg::WAVES_M;
  using LA = grouped_loader<Cfg::E, Cfg::A_KC, BM, RB, NT>;
  using LB = grouped_loader<Cfg::E, Cfg::B_KC, BN, RB, NT>;
  // rounds of loads that B's columns need
  constexpr int UB = LB::LINES ? LB::U : (TN * 16 * Cfg::WAVES_N * RB / 16 + NT - 1) / NT;
  const char *a = w.a, *b = w.b;
  const uint64_t a_step = (Cfg::A_KC ? (uint64_t)BK : (uint64_t)BK * args.lda) * T::BYTES;
  const uint64_t b_step = (Cfg::B_KC ? (uint64_t)BK : (uint64_t)BK * args.ldb) * T::BYTES;

  typename T::acc_t acc[T::NACC][TN][TM];
#pragma unroll
  for (int s = 0; s < T::NACC; s++)
#pragma unroll
    for (int j = 0; j < TN; j++)
#pragma unroll
      for (int i = 0; i < TM; i++)
#pragma unroll
        for (int v = 0; v < 4; v++) acc[s][j][i][v] = 0;

  // ---- fragments ----
  // Lane l of a 16-row MFMA supplies row l % 16 and the 16 bytes number l / 16 of the slice's 64.
  const int frow = lane & 15, fg = lane >> 4;
  auto frag = [&](const char *op, const int row0, const int p, const int slice, auto kc_tag, auto rows_tag) -> u4_t {
    constexpr bool KC = decltype(kc_tag)::value;
    constexpr int ROWS = decltype(rows_tag)::value;
    if constexpr (KC || T::F32) {
      return *reinterpret_cast<const u4_t *>(op + p * ROWS * RB + chunk_offset<RB>(row0 + frow, slice * 4 + fg));
    } else {
      typedef short s4_t __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4_t *tr_t;
      typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
      // lane l % 16 of a quarter names line (l % 16) / 4 and a quarter of the 32-byte piece; the quarter's K-values are
      // 8 fg .. 8 fg + 3, then + 4 (line_swizzle is the same for both)
      const int k = slice * 32 + fg * 8 + (frow >> 2);
      const int off = k * (ROWS * 2) + (((row0 >> 4) ^ line_swizzle(k)) << 5) + (frow & 3) * 8;
      const u2_t x = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)(op + off)));
      const u2_t y = __builtin_bit_cast(u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_t)(op + off + 4 * ROWS * 2)));
      return u4_t{x[0], x[1], y[0], y[1]};
    }
  };
  // A step's MFMAs go row block after row block of every slice.  The fragments of the row blocks to come and of the
  // next slice's columns are on their way meanwhile: AHEAD_A row blocks (FP32, whose blocks are three or six times as
  // many MFMAs: one) in a ring of four, columns in two sets.
  constexpr int BLOCKS = SLICES * TM, AHEAD_A = T::F32 ? 1 : 2, RING = T::F32 ? 2 : 4;
  static_assert(BLOCKS % RING == 0, "a step begins where the ring does");
  constexpr int SCHED_VALU = 3; // vector instructions beside an MFMA of FP32 operands (two waves of a SIMD take turns)
  // IN_PLACE: no registers are left for a second set of columns
  constexpr bool IN_PLACE = T::F32 && T::NACC * Cfg::TM * Cfg::TN * 4 >= 128;
  u4_t fa[RING][T::NP], fb[2][T::NP][TN];
  auto read_a = [&](const char *stage, const int g) {
#pragma unroll
    for (int p = 0; p < T::NP; p++)
      fa[g % RING][p] = frag(stage, wm * Cfg::WM + (g % TM) * 16, p, g / TM, std::integral_constant<bool, Cfg::A_KC>{},
                             std::integral_constant<int, BM>{});
  };
  auto frag_b = [&](const char *stage, const int p, const int j, const int s) {
    return frag(stage + Cfg::A_STAGE, (j * Cfg::WAVES_N + wn) * 16, p, s, std::integral_constant<bool, Cfg::B_KC>{},
                std::integral_constant<int, BN>{});
  };
  auto read_b = [&](const char *stage, const int s, const int set) { // (set: of fragments)
#pragma unroll
    for (int p = 0; p < T::NP; p++)
#pragma unroll
      for (int j = 0; j < TN; j++) fb[set][p][j] = frag_b(stage, p, j, s);
  };
  // the fragments that a step's first MFMAs need
  auto begin = [&](const char *stage) {
    read_a(stage, 0);
    read_b(stage, 0, 0);
    if (AHEAD_A > 1) read_a(stage, 1);
  };
  // Row blocks `from` .. `to` - 1 of a step; `beside(g)`: what else is done beside block g.  next: the next step's
  // buffer, if its first fragments are to be read beside the last blocks (it is complete by then).
  // par: which set the step's first columns are in.
  auto multiply = [&](const char *stage, auto next, auto from, auto to, const int par, auto beside) {
    constexpr bool HAS_NEXT = !std::is_same<decltype(next), std::nullptr_t>::value;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = from.value; g < to.value; g++) {
      const int s = g / TM, i = g % TM;
      if (g + AHEAD_A < BLOCKS) read_a(stage, g + AHEAD_A);
      else if constexpr (HAS_NEXT) read_a(next, g + AHEAD_A - BLOCKS);
      if (i == (TM > 4 ? TM - 3 : TM > 1 ? TM - 2 : 0) && s + 1 < SLICES) read_b(stage, s + 1, (s + 1 + par) % 2);
      if constexpr (HAS_NEXT) {
        if (!IN_PLACE && g == BLOCKS - AHEAD_A) read_b(next, 0, (SLICES + par) % 2);
      }
      beside(g);
#pragma unroll
      for (int q = 0; q < T::NPROD; q++) {
        const int pa = T::F32 ? prec_traits<T::P>::PA[q] : 0, pb = T::F32 ? prec_traits<T::P>::PB[q] : 0;
        const int ac = T::F32 ? prec_traits<T::P>::ACC[q] : 0;
#pragma unroll
        for (int j = 0; j < TN; j++)
          acc[ac][j][i] = grouped_mfma<Cfg::E>(fa[g % RING][pa], fb[(s + par) % 2][pb][j], acc[ac][j][i]);
        if constexpr (HAS_NEXT && IN_PLACE) {
          // a term's columns are read again behind the last product that has the old ones
          __builtin_amdgcn_sched_barrier(0);
          bool later = false;
#pragma unroll
          for (int q2 = q + 1; q2 < T::NPROD; q2++) later |= prec_traits<T::P>::PB[q2] == pb;
          if (!later) {
#pragma unroll
            for (int j = 0; j < TN; j++) fb[par][pb][j] = frag_b(next, pb, j, 0);
          }
        }
      }
      if constexpr (T::F32) {
        // the splitting between the MFMAs, not in front of them: both waves of a SIMD pass the barrier together
#pragma unroll
        for (int x = 0; x < T::NPROD * TN; x++) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0); // MFMA
          __builtin_amdgcn_sched_group_barrier(0x002, SCHED_VALU, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0); // LDS reads
          __builtin_amdgcn_sched_group_barrier(0x200, 1, 0); // LDS writes
          __builtin_amdgcn_sched_group_barrier(0x020, 1, 0); // loads
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto nothing = [](int) {};
  constexpr std::integral_constant<int, 0> first;
  constexpr std::integral_constant<int, BLOCKS> end;

  // ---- K loop ----
  // A K that ends inside a step has that step multiplied first, so that the loop has whole steps only: step s begins
  // at K-value (s - partial) BK, the partial one behind them all.
  // (Lines of any alignment: the last step counts as partial even if it is whole, since a chunk of the matrix's last line
  // must not be read beyond its end.)
  constexpr bool LAST_ASIDE = !T::F32 && !Cfg::DIRECT && (!Cfg::A_KC || !Cfg::B_KC);
  const int whole = LAST_ASIDE ? (int)((w.klen > 0 ? w.klen - 1 : 0) / BK) : (int)(w.klen / BK), left = (int)w.klen - whole * BK;
  const int partial = left != 0, steps = whole + partial;
  auto a_at = [&](int s) { return a + (uint64_t)(s < partial ? whole : s - partial) * a_step; };
  auto b_at = [&](int s) { return b + (uint64_t)(s < partial ? whole : s - partial) * b_step; };
  typedef typename std::conditional<Cfg::DIRECT, uint32_t, uint64_t>::type off_t;
  off_t offa[LA::U], offb[UB];
#pragma unroll
  for (int u = 0; u < LA::U; u++) offa[u] = (off_t)LA::offset(tid + u * NT, args.lda, w.rows_a);
#pragma unroll
  for (int u = 0; u < UB; u++) offb[u] = (off_t)LB::offset(tid + u * NT, args.ldb, w.rows_b);
  constexpr int LOADS = LA::U + UB;
  if constexpr (Cfg::DIRECT && !T::F32) {
    // One barrier a step, in front of its last AHEAD_A row blocks, whose fragments every wave has in registers by then.
    // Behind it the step's buffer is free, and the loads of step s + NSTAGE begin to go there; and the next step's buffer
    // is complete, so that its first fragments are read beside the last MFMAs of this one.
    static_assert(SLICES == 2, "the two sets of column fragments");
    constexpr std::integral_constant<int, BLOCKS - AHEAD_A> last;
    const uint32_t lds0 = lds_address(lds);
    auto issue = [&](int l, const char *pa, const char *pb, uint32_t stage) {
      if (l < LA::U) LA::direct(l, pa, offa[l], stage, wave);
      else LB::direct(l - LA::U, pb, offb[l - LA::U], stage + Cfg::A_STAGE, wave);
    };
    // (what the compiler has loaded is waited for here: a wait of its own inside the loop would be one for all loads)
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    for (int s = 0; s < Cfg::NSTAGE && s < steps; s++) {
      const uint32_t stage = lds0 + s * Cfg::STAGE;
      const char *pa = a_at(s), *pb = b_at(s);
      if (s < partial) {
#pragma unroll
        for (int u = 0; u < LA::U; u++) LA::direct_tail(u, pa, offa[u], stage, tid, wave, left);
#pragma unroll
        for (int u = 0; u < UB; u++) LB::direct_tail(u, pb, offb[u], stage + Cfg::A_STAGE, tid, wave, left);
      } else {
#pragma unroll
        for (int l = 0; l < LOADS; l++) issue(l, pa, pb, stage);
      }
    }
    if (steps > 0) {
      if (steps >= Cfg::NSTAGE) __builtin_amdgcn_s_waitcnt(waitcnt_vm(LOADS * (Cfg::NSTAGE - 1)));
      else __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      block_sync_lds();
      begin(lds);
    }
    // A CU takes 16 clocks for each of these loads, as long as an MFMA, and a wave that asks for more waits with its
    // MFMAs: they are spread over half a step, and land in the other half.
    constexpr int SPREAD = BLOCKS / 2 > AHEAD_A ? BLOCKS / 2 : AHEAD_A;
    int at = 0, before = 0; // buffers of steps s and s - 1
    const char *qa = uniform_address(a_at(Cfg::NSTAGE)), *qb = uniform_address(b_at(Cfg::NSTAGE)); // of step s + NSTAGE
    for (int s = 0; s < steps; s++) {
      const int next = at + 1 == Cfg::NSTAGE ? 0 : at + 1;
      const char *here = lds + at * Cfg::STAGE;
      // the rest of what was begun beside the last row blocks of the step before
      const bool rest = s > 0 && s - 1 + Cfg::NSTAGE < steps;
      const char *pa = qa - a_step, *pb = qb - b_step;
      const uint32_t old_stage = lds0 + before * Cfg::STAGE;
      multiply(here, nullptr, first, last, 0, [&](int g) {
        if (rest) {
#pragma unroll
          for (int l = 0; l < LOADS; l++)
            if (l * SPREAD / LOADS == g + AHEAD_A) issue(l, pa, pb, old_stage);
        }
      });
      // everything but the loads of the steps behind the next one has landed (at the end none are left out of the wait)
      if (s + Cfg::NSTAGE <= steps) __builtin_amdgcn_s_waitcnt(waitcnt_vm(LOADS * (Cfg::NSTAGE - 2)));
      else __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
      block_sync_lds();
      const uint32_t stage = lds0 + at * Cfg::STAGE;
      const bool more = s + Cfg::NSTAGE < steps;
      // (behind the last step, unused values are read)
      multiply(here, (const char *)lds + next * Cfg::STAGE, last, end, 0, [&](int g) {
        if (more) {
#pragma unroll
          for (int l = 0; l < LOADS; l++)
            if (l * SPREAD / LOADS == g - last.value) issue(l, qa, qb, stage);
        }
      });
      qa += a_step;
      qb += b_step;
      before = at;
      at = next;
    }
  } else {
    // through registers: step s + 1 is written to LDS and step s + 1 + SETS asked for beside the MFMAs of step s
    static_assert(Cfg::NSTAGE == 2 || (Cfg::DIRECT && !T::F32), "two buffers");
    // which of a step's units (A's, then B's) come beside row block g
    auto share = [](int g, int blocks, auto f) {
#pragma unroll
      for (int l = 0; l < LOADS; l++)
        if (l * blocks / LOADS == g) f(l);
    };
    // SETS of registers: a load's way is longer than a step
    constexpr int SETS = IN_PLACE ? 1 : 2;
    // EARLY: the barrier comes before a step's last row block, beside which the next step's first fragments are read, as
    // above.  The buffer that is written meanwhile was last read before the barrier of the step before.  (FP16TCEC, 4096 x
    // 2048 x 1024 in 8 groups, 128 x 128 tiles: 66.0 us with all fragments read behind the barrier, so 61.8; 256 x 128: 58.2,
    // so 55.9.)
    constexpr bool EARLY = T::F32;
    constexpr std::integral_constant<int, BLOCKS - AHEAD_A> last;
    typename LA::Regs ra[SETS];
    typename LB::Regs rb[SETS];
    auto put = [&](int l, const int set, char *stage) {
      if (l < LA::U) LA::put(ra[set], l, stage, tid);
      else LB::put(rb[set], l - LA::U, stage + Cfg::A_STAGE, tid);
    };
    auto fetch = [&](int l, const int set, const char *pa, const char *pb, int64_t k0) { // (k0: the step's first K-value)
      constexpr bool FAST = Cfg::DIRECT, CAREFUL = Cfg::CAREFUL;
      if (l < LA::U)
        LA::template fetch<FAST, CAREFUL>(ra[set], l, pa, args.lda, offa[l], w.rows_a, Cfg::A_KC ? w.safe_a : w.safe_a - k0, tid);
      else
        LB::template fetch<FAST, CAREFUL>(rb[set], l - LA::U, pb, args.ldb, offb[l - LA::U], w.rows_b, Cfg::B_KC ? w.safe_b : w.safe_b - k0, tid);
    };
    auto ask = [&](int s, const int set) {
      const char *pa = a_at(s), *pb = b_at(s);
#pragma unroll
      for (int l = 0; l < LOADS; l++) fetch(l, set, pa, pb, (int64_t)(s - partial) * BK);
    };
    if (steps > 0) {
      if (partial) {
        const char *pa = a_at(0), *pb = b_at(0);
#pragma unroll
        for (int u = 0; u < LA::U; u++)
          LA::fetch_tail(ra[0], u, pa, args.lda, w.rows_a, left, Cfg::A_KC ? w.safe_a : w.safe_a - whole * BK, tid);
#pragma unroll
        for (int u = 0; u < UB; u++)
          LB::fetch_tail(rb[0], u, pb, args.ldb, w.rows_b, left, Cfg::B_KC ? w.safe_b : w.safe_b - whole * BK, tid);
      } else {
        ask(0, 0);
      }
      if (SETS > 1 && steps > 1) ask(1, SETS - 1);
#pragma unroll
      for (int l = 0; l < LOADS; l++) put(l, 0, lds);
      if (steps > SETS) ask(SETS, 0);
      block_sync_lds();
      if (EARLY) begin(lds);
    }
    // step s: s + 1 goes to LDS from its set (the steps' take turns), and s + 1 + SETS is asked for (the last ones again,
    // unused)
    auto run = [&](int s, const int set, const int par) {
      const int far = s + 1 + SETS < steps ? s + 1 + SETS : steps - 1;
      const char *pa = a_at(far), *pb = b_at(far);
      const char *here = lds + (s & 1) * Cfg::STAGE;
      char *stage = lds + ((s + 1) & 1) * Cfg::STAGE;
      auto beside = [&](int g) {
        share(g, EARLY ? last.value : BLOCKS, [&](int l) {
          put(l, set, stage);
          fetch(l, set, pa, pb, (int64_t)(far - partial) * BK);
        });
      };
      if constexpr (EARLY) {
        multiply(here, nullptr, first, last, par, beside);
        block_sync_lds();
        multiply(here, (const char *)stage, last, end, par, nothing);
      } else {
        begin(here);
        multiply(here, nullptr, first, end, 0, beside);
        block_sync_lds();
      }
    };
    int s = 0;
    for (; s + SETS < steps; s += SETS) {
      run(s, SETS - 1, 0);
      if constexpr (SETS > 1) run(s + 1, 0, 1);
    }
    auto finish = [&](const int par) {
      const char *here = lds + ((steps - 1) & 1) * Cfg::STAGE;
      if (!EARLY) begin(here);
      multiply(here, nullptr, first, end, EARLY ? par : 0, nothing);
    };
    if (SETS > 1 && s + 1 < steps) {
      run(s, SETS - 1, 0);
      finish(SETS - 1);
    } else if (steps > 0) {
      finish(0);
    }
  }

  // ---- results ----
  // Register v of lane l: MFMA row 4 (l / 16) + v (of C), column l % 16 (token).  One column block after the other passes
  // through LDS, each wave's through a part of its own, so that a wave's store covers the columns' whole WM rows.
  block_sync_lds(); // (every wave has read its last fragments)
  constexpr int PITCH = Cfg::PITCH;
  float *mine = reinterpret_cast<float *>(lds) + wave * (16 * PITCH);
  const uint32_t row0 = w.m0 + wm * Cfg::WM;
#pragma unroll
  for (int j = 0; j < TN; j++) {
#pragma unroll
    for (int i = 0; i < TM; i++) {
      f4v_t x;
#pragma unroll
      for (int v = 0; v < 4; v++) {
        x[v] = (float)acc[0][j][i][v];
        if constexpr (T::NACC == 2) x[v] += acc[1][j][i][v] * prec_traits<T::P>::CORR_SCALE;
      }
      *reinterpret_cast<f4v_t *>(mine + frow * PITCH + i * 16 + fg * 4) = x;
    }
    // (a wave's own writes and reads of LDS are carried out in order)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    constexpr int LANES = Cfg::WM / 4, COLS = 64 / LANES; // lanes of a column, columns of a round
    const uint32_t row = row0 + (lane % LANES) * 4, col0 = w.n0 + (j * Cfg::WAVES_N + wn) * 16;
    f4v_t sa = {args.alpha, args.alpha, args.alpha, args.alpha};
    if constexpr (T::I8) {
#pragma unroll
      for (int v = 0; v < 4; v++)
        sa[v] = args.scale_a[(uint64_t)w.group * args.m + (row + v < args.m ? row + v : args.m - 1)];
    }
#pragma unroll 1
    for (int r = 0; r < 16; r += COLS) {
      const uint32_t col = col0 + r + lane / LANES;
      if (col >= w.n_end) continue;
      f4v_t x = *reinterpret_cast<const f4v_t *>(mine + (r + lane / LANES) * PITCH + (lane % LANES) * 4);
      if constexpr (Cfg::RAGGED_K) {
        if (args.splits > 1) {
          *reinterpret_cast<f4v_t *>(w.partial + (uint64_t)(col - w.n0) * BM + (row - w.m0)) = x;
          continue;
        }
      }
      const float sb = T::I8 ? args.scale_b[col] : 1.0f;
#pragma unroll
      for (int v = 0; v < 4; v++) x[v] = T::I8 ? x[v] * sa[v] * sb : x[v] * sa[v];
      const uint64_t at = (uint64_t)col * args.ldc + row;
      if (T::F32 || args.out == OUT_F32) store_four<OUT_F32>(w.c + at * 4, x, args.beta, row, args.m, args.vec_c != 0);
      else if (Cfg::E == Elem::F16 || (T::I8 && args.out == OUT_F16))
        store_four<OUT_F16>(w.c + at * 2, x, args.beta, row, args.m, args.vec_c != 0);
      else store_four<OUT_BF16>(w.c + at * 2, x, args.beta, row, args.m, args.vec_c != 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  }
}

template <class Cfg>
__global__ __launch_bounds__(Cfg::NT) __attribute__((amdgpu_waves_per_eu(Cfg::OCC, Cfg::OCC)))
void grouped_kernel(const GroupedArgs args) {
  using T = typename Cfg::T;
  constexpr int BM = Cfg::BM, BN = Cfg::BN, TN = Cfg::TN;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const uint32_t tiles_m = (args.m + BM - 1) / BM;
  TilePlace t;
  TileWork w;
  const char *a = args.a, *b = args.b;
  w.c = args.c;
  if constexpr (Cfg::RAGGED_K) {
    const uint32_t tiles_n = (args.n + BN - 1) / BN;
    uint32_t split;
    if (!place_over_k(args, blockIdx.x, tiles_m, tiles_n, t, split)) return;
    group_span(args.offsets, t.group, args.k, t.lo, t.hi);
    t.lo = __builtin_amdgcn_readfirstlane(t.lo);
    t.hi = __builtin_amdgcn_readfirstlane(t.hi);
    if (args.splits > 1) {
      const uint32_t len = t.hi - t.lo, part = ((len + Cfg::BK - 1) / Cfg::BK + args.splits - 1) / args.splits * Cfg::BK;
      const uint32_t from = split * part < len ? split * part : len;
      t.hi = t.lo + (len - from < part ? len : from + part);
      t.lo += from;
      w.partial = args.partial + (((uint64_t)t.group * tiles_n + t.tn) * tiles_m + t.tm) * args.splits * (BM * BN) +
                  (uint64_t)split * (BM * BN);
    }
    w.n0 = t.tn * BN;
    w.n_end = args.n;
    w.klen = t.hi - t.lo;
    a += (uint64_t)t.lo * args.lda * T::BYTES;
    b += (uint64_t)t.lo * args.ldb * T::BYTES;
    w.c += (uint64_t)t.group * args.stride_c * (args.out == OUT_F32 ? 4 : 2);
  } else {
    if (!place_tile(args, blockIdx.x, tiles_m, BN, t)) return;
    w.n0 = t.lo + t.tn * BN;
    w.n_end = t.hi;
    w.klen = args.k;
    a += (uint64_t)t.group * args.stride_a * T::BYTES;
  }
  w.group = t.group;
  w.m0 = t.tm * BM;
  w.rows_a = (int)(args.m - w.m0 < (uint32_t)BM ? args.m - w.m0 : BM);
  w.rows_b = (int)(w.n_end - w.n0 < (uint32_t)BN ? w.n_end - w.n0 : BN);
  w.a = uniform_address(a + (Cfg::A_KC ? (uint64_t)w.m0 * args.lda : (uint64_t)w.m0) * T::BYTES);
  w.b = uniform_address(b + (Cfg::B_KC ? (uint64_t)w.n0 * args.ldb : (uint64_t)w.n0) * T::BYTES);
  // (what a chunk of 8 or 16 values can stick out by is less than a line that long)
  auto safe = [&](bool kc, uint64_t ld, uint64_t extent, int64_t rows, int64_t lines) -> int64_t {
    return extent < (uint64_t)T::CHUNK || ld < (uint64_t)T::CHUNK ? 0 : kc ? rows - 1 : lines - 1;
  };
  const int64_t lines = Cfg::RAGGED_K ? (int64_t)args.k - t.lo : (int64_t)args.k;
  w.safe_a = safe(Cfg::A_KC, args.lda, Cfg::A_KC ? args.k : args.m, (int64_t)args.m - w.m0, lines);
  w.safe_b = safe(Cfg::B_KC, args.ldb, Cfg::B_KC ? args.k : args.n, (int64_t)args.n - w.n0, lines);
  if constexpr (Cfg::RAGGED_K) {
    multiply_tile<Cfg, TN>(args, w, lds);
  } else {
    static_assert(TN == 2 || TN == 4, "column blocks of a wave");
    const int blocks = (w.rows_b + 16 * Cfg::WAVES_N - 1) / (16 * Cfg::WAVES_N);
    if (blocks >= TN) multiply_tile<Cfg, TN>(args, w, lds);
    else if (blocks == 1) multiply_tile<Cfg, 1>(args, w, lds);
    else if constexpr (TN == 4) {
      if (blocks == 2) multiply_tile<Cfg, 2>(args, w, lds);
      else multiply_tile<Cfg, 3>(args, w, lds);
    }
  }
}

template <class Cfg> void launch_grouped(const GroupedArgs &args, uint32_t workgroups, hipStream_t stream) {
  static device_flags_t done = {};
  allow_dynamic_lds(reinterpret_cast<const void *>(&grouped_kernel<Cfg>), Cfg::LDS_BYTES, done);
  hipLaunchKernelGGL(grouped_kernel<Cfg>, dim3(workgroups), dim3(Cfg::NT), Cfg::LDS_BYTES, stream, args);
}
template <class Cfg> constexpr GroupedKernel grouped_entry() { return {&launch_grouped<Cfg>, Cfg::BM, Cfg::BN}; }

} // namespace cumpsgemm_amd
