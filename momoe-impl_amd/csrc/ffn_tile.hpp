// Products of a dense SwiGLU block in tiles of BM x 128: a workgroup a tile, 64 k-values a stage, any contraction of a multiple of 32.
//
// For launches of few tiles, short contractions, few rows; the large ones run in the loop of gemm_span.hpp, whose operands and fragment
// layout these are (the first input of the MFMA is the weight side: a lane holds, for one tile row (lane % 16), four consecutive
// columns).  4 waves, 2 x 2.  STAGES stages in LDS; the fragments of one half of a stage are read while
// the other is multiplied (read and then multiplied, one after the other, a stage took 0.36 to 0.75 us whatever was on the way).  A
// contraction may be cut into `slices`, each a tile of its own that leaves fp32 sums for another kernel.
// Bound by a stage's chain of fragment reads, products, wait and barrier.  Of 64 x 128 a stage takes 0.39 us where one workgroup is on
// a CU, whether 64 CUs have one or all, and 0.64 where two are; of 32 x 128 0.31 and 0.45 (63 to 92 GB/s a CU; slopes of x W1 over
// contractions of 2048 to 8192).  The matrix instructions are 0.11 of the 0.39; of a wavefront's time 30 % is waits for transfers and
// at the barrier, another 30 % for its turn to issue, and LDS banks do not conflict.  1000 tokens through 2176 x 1152: x W1 26 us (0.38
// PFLOP/s; 288 tiles of 34 stages, of which the 32 CUs that have two take 22), h W2 16 (0.31).  24 through 4096 x 11264: x W1 36.5 (176
// workgroups; 43.5 with weights of which the cache holds nothing), h W2 17.6 (5.2 TB/s, 512).
#pragma once
#include "gemm_span.hpp"

namespace momoe {

constexpr int kFfnCols = 128;

// Rows of a matrix at any pitch, k-contiguous, rows past the last one repeat it.  `K`: of 32 k-values the stage's first half is all
// there is, and stands in the second, too.
template <int ROWS>
struct FfnRows : SpanGatheredRows<ROWS> {
  using Base = SpanGatheredRows<ROWS>;
  using L = SpanRowsLayout<ROWS>;
  __device__ __forceinline__ void init(const bf16* mat, int64_t ld, int64_t row0, int rows, int K) {
    Base::base = mat + row0 * ld;
    const int l = fresh_lane();
    const uint32_t piece = L::piece_bytes(l) & (K == 32 ? 0x3Fu : ~0u);
#pragma unroll
    for (int j = 0; j < L::DEP; ++j) Base::off[j] = (uint32_t)min(32 * j + L::first_row(l), rows - 1) * (uint32_t)(2 * ld) + piece;
  }
};
// Rows of a k-blocked matrix [K / 32][ldm][32]
template <int ROWS>
struct FfnBlockedRows : SpanBlockedRows<ROWS> {
  using Base = SpanBlockedRows<ROWS>;
  int64_t far;  // elements to the second half of a stage
  __device__ __forceinline__ void init(const bf16* mat, int64_t ldm, int64_t row0, int rows, int K) {
    Base::init(mat, ldm, row0, rows);
    far = K == 32 ? 0 : ldm * kHalf;
  }
  template <int j>
  __device__ __forceinline__ void deposit(const bf16* src, uint32_t slot) const {
    constexpr int h = j / Base::PER_HALF, q = j % Base::PER_HALF;
    dma16_at<h * (ROWS * kHalf * 2) + q * kSpanWaves * 1024>(h ? src + far : src, Base::off[q], slot);
  }
};

// 32 rows: one deposit of the four waves, two of them a half each
template <>
struct FfnBlockedRows<32> {
  static constexpr int DEP = 1, ELEMS = 32 * kSpan;
  using Full = SpanBlockedRows<64>;
  const bf16* base;
  int64_t kstride;
  uint32_t off;
  __device__ __forceinline__ void init(const bf16* mat, int64_t ldm, int64_t row0, int rows, int K) {
    const int l = fresh_lane(), half = wave_id() >> 1, row = (wave_id() & 1) * 16 + (l >> 2);
    kstride = ldm * kHalf;
    base = mat + row0 * kHalf + (half && K != 32 ? kstride : 0);
    off = (uint32_t)min(row, rows - 1) * (kHalf * 2) + (((l & 3) ^ Full::swz(row)) * 16);
  }
  __device__ __forceinline__ const bf16* source(int k) const { return base + (int64_t)(k / kHalf) * kstride; }
  template <int j>
  __device__ __forceinline__ void deposit(const bf16* src, uint32_t slot) const {
    dma16_at<0>(src, off, slot);
  }
  using Lane = Full::Lane;
  static __device__ __forceinline__ bf16x8 frag(const bf16* slot, const Lane& ln, int i, int h) {
    return *(const bf16x8*)((const char*)slot + ln.o + h * (32 * kHalf * 2) + i * (32 * kHalf));
  }
};

// k-strided columns ([k][n] weights), as SpanCols.  PAIRED: a wave's second half of fragments are the columns 64 further on.
template <bool PAIRED>
struct FfnCols {
  static constexpr int COLS = kFfnCols, DEP = COLS / 32, FN = COLS / 32;
  static constexpr int ELEMS = COLS * kSpan;
  static constexpr int PIECES = COLS / 8, RPD = 64 / PIECES, STEP = RPD * kSpanWaves;
  static_assert(STEP == 16, "one pattern of swizzles in all deposits, two deposits a half stage");
  static __device__ __forceinline__ int swz(int k) { return 2 * (k & 3) + 8 * ((k >> 3) & 1); }
  const bf16* base;
  uint32_t off, pitch, wrap;  // bytes; wrap: of the k-rows that a stage's second half lies behind the first
  template <class ColOff>
  __device__ __forceinline__ void init(const bf16* base_, int ld, int K, ColOff coloff) {
    base = base_;
    pitch = (uint32_t)ld * 2;
    wrap = K == 32 ? 0 : 2 * STEP * pitch;
    const int l = fresh_lane(), krow = wave_id() * RPD + l / PIECES;
    off = (uint32_t)krow * pitch + (uint32_t)coloff(((l % PIECES) ^ swz(krow)) * 8) * 2;
  }
  __device__ __forceinline__ const bf16* source(int k) const { return (const bf16*)((const char*)base + (uint32_t)k * pitch); }
  template <int j>
  __device__ __forceinline__ void deposit(const bf16* src, uint32_t slot) const {
    dma16_at<j * kSpanWaves * 1024>((const char*)src + (uint32_t)(STEP * (j % 2)) * pitch + (j / 2 ? wrap : 0u), off, slot);
  }
  struct Lane {
    int o;  // first fragment, in bytes
    __device__ __forceinline__ explicit Lane(int org) {
      const int l = fresh_lane(), krow = 8 * (l >> 4) + ((l & 15) >> 2), col = org + 4 * (l & 3);
      o = (krow * COLS + (((col >> 3) ^ swz(krow)) << 3) + (col & 7)) * 2;
    }
  };
  static __device__ __forceinline__ bf16x8 frag(const bf16* slot, const Lane& ln, int i, int h) {
    // (pieces 1 to 3 bits up are permuted, so what is added to a column there is an exclusive or)
    const int add = PAIRED ? 32 * (i % (FN / 2)) ^ (i >= FN / 2 ? COLS : 0) : 32 * i;
    const bf16* p = (const bf16*)((const char*)slot + (ln.o ^ add)) + h * (kHalf * COLS);
    const bf16x4 lo = lds_read_tr4(p), hi = lds_read_tr4(p + 4 * COLS);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Columns of a matrix whose rows are the contraction (tokens), for either side: token t of column c at t * pitch + lane_bytes(c) bytes from
// base; tokens past the last one repeat it.  LDS and fragments as FfnCols.
struct FfnTokenCols : FfnCols<false> {
  using L = FfnCols<false>;
  uint32_t last;
  int krow;
  template <class LaneBytes>
  __device__ __forceinline__ void init(const void* base_, uint32_t pitch_bytes, int tokens, LaneBytes lane_bytes) {
    base = (const bf16*)base_;
    pitch = pitch_bytes;
    last = tokens - 1;
    const int l = fresh_lane();
    krow = wave_id() * RPD + l / PIECES;
    off = lane_bytes(((l % PIECES) ^ swz(krow)) * 8);
  }
  struct Source {
    const bf16* base;
    int k;
  };
  __device__ __forceinline__ Source source(int k) const { return {base, k}; }
  template <int j>
  __device__ __forceinline__ void deposit(const Source& src, uint32_t slot) const {
    dma16_at<j * kSpanWaves * 1024>(src.base, off + min((uint32_t)(src.k + STEP * j + krow), last) * pitch, slot);
  }
};

// rows at a fixed pitch (k-contiguous weights): a multiple of 32 of them, the last 32 repeated where the tile sticks out
struct FfnWeightRows : SpanPitchedRows<kFfnCols> {
  using Base = SpanPitchedRows<kFfnCols>;
  __device__ __forceinline__ void init(const bf16* mat, int K, int row0, int nrows) {
    Base::init(mat, K, row0, nrows);
    if (K == 32) {
      const int l = fresh_lane();
      off = (uint32_t)L::first_row(l) * pitch + (L::piece_bytes(l) & 0x3F);
    }
  }
};

// until of the stages on their way, of `loads` transfers each, at most min(MOST, after) are left
template <int LOADS, int MOST>
__device__ __forceinline__ void wait_for_stage(int after) {
  if constexpr (MOST == 0) {
    wait_vmcnt<0>();
  } else {
    if (after >= MOST) wait_vmcnt<LOADS * MOST>();
    else wait_for_stage<LOADS, MOST - 1>(after);
  }
}

// A tile program P: P::Rows, P::Weights, FM; K, slices, rows, row_tiles, col_tiles; setup(row0, rows, tn, A, W), n_org(wn): first column
// of a wave's fragments in the tile; epilogue(row0, rows, tn, slice, wm, wn, acc).  block: of this program's, from a multiple of 8 on.
template <class P, int STAGES>
__device__ __forceinline__ void run_ffn_tile(const P& prog, int block) {
  using Rows = typename P::Rows;
  using Weights = typename P::Weights;
  constexpr int FM = P::FM, FN = 4, BM = 32 * FM;
  constexpr int LOADS = Rows::DEP + Weights::DEP;
  // An XCD has a contiguous eighth of the tiles, row tiles fastest: those that share weights meet in one L2
  const int total = prog.row_tiles * prog.col_tiles * prog.slices, chunk = (total + 7) >> 3;
  int t = (block & 7) * chunk + (block >> 3);
  if ((block >> 3) >= chunk || t >= total) return;
  const int row_tile = t % prog.row_tiles;
  t /= prog.row_tiles;
  const int slice = t % prog.slices, tn = t / prog.slices;
  const int64_t row0 = (int64_t)row_tile * BM;
  const int rows = (int)min((int64_t)BM, prog.rows - row0);
  Rows A;
  Weights W;
  prog.setup(row0, rows, tn, A, W);
  bf16* const lds = dyn_lds();
  constexpr int STAGE = Rows::ELEMS + Weights::ELEMS;  // elements
  const uint32_t addr = lds_address(lds) + wave_id() * 1024;
  const int wn = wave_id() & 1, wm = wave_id() >> 1;
  // this slice's stages; the last of all may be half a one
  const SpanStages all(prog.K);
  const int first = (int)((int64_t)all.count * slice / prog.slices), count = (int)((int64_t)all.count * (slice + 1) / prog.slices) - first;
  const bool tail = all.tail && slice == prog.slices - 1;
  int k = first * kSpan, put = 0, got = 0;
  if (first == all.count - 1) k = max(0, min(k, all.kmax));
  auto request = [&] {
    const auto asrc = A.source(k);
    const auto wsrc = W.source(k);
    const uint32_t to = addr + (uint32_t)put * (STAGE * 2);
    unrolled<0, Rows::DEP>([&](auto D) { A.template deposit<decltype(D)::value>(asrc, to); });
    unrolled<0, Weights::DEP>([&](auto D) { W.template deposit<decltype(D)::value>(wsrc, to + Rows::ELEMS * 2); });
    k = max(0, all.after(k));
    put = put + 1 == STAGES ? 0 : put + 1;
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
    if (s < count) request();
  f32x4 acc[FN][FM] = {};
  const typename Rows::Lane alane(wm * 16 * FM);
  const typename Weights::Lane wlane(prog.n_org(wn));
  bf16x8 wf[2][FN], af[2][FM];
  auto read = [&](auto H) {
    constexpr int h = decltype(H)::value;
    const bf16 *sa = lds + got * STAGE, *sw = sa + Rows::ELEMS;
#pragma unroll
    for (int j = 0; j < FN; ++j) wf[h][j] = Weights::frag(sw, wlane, j, h);
#pragma unroll
    for (int i = 0; i < FM; ++i) af[h][i] = Rows::frag(sa, alane, i, h);
  };
  auto multiply = [&](auto H) {
    constexpr int h = decltype(H)::value;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[j][i] = mfma16(wf[h][j], af[h][i], acc[j][i]);
  };
  wait_for_stage<LOADS, STAGES - 1>(count - 1);
  __builtin_amdgcn_s_barrier();
  order_fence();
  read(IntC<0>{});
  order_fence();
  for (int s = 0; s < count; ++s) {
    // a last stage that is not whole starts at K - 64: its first half has been multiplied (of 32 k-values the first is all)
    const bool part = s + 1 == count && tail;
    read(IntC<1>{});
    order_fence();
    if (!part || prog.K == 32) multiply(IntC<0>{});
    order_fence();
    if (s + 1 < count) {  // the next stage has landed, and every wave is done reading this one, whose place the one after takes
      wait_for_stage<LOADS, STAGES - 2>(count - 2 - s);
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      order_fence();
      got = got + 1 == STAGES ? 0 : got + 1;
      read(IntC<0>{});
      if (s + STAGES < count) request();
    }
    order_fence();
    if (!part || prog.K != 32) multiply(IntC<1>{});
    order_fence();
  }
  prog.epilogue(row0, rows, tn, slice, wm, wn, acc);
}
template <class P, int STAGES>
constexpr size_t kFfnLds = (size_t)STAGES * (P::Rows::ELEMS + P::Weights::ELEMS) * sizeof(bf16);

}  // namespace momoe
