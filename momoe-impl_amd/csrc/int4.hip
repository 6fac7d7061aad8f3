// SwiGLU blocks with weights in 4 bits, forward only: the experts of a mixture, or one dense block.
//
// A weight is (code - zero) * scale: a code of 4 bits, a zero (0 to 15) and a 16-bit scale for each `group` (32, 64, 128) consecutive
// k-values of a column.  A product over a group is
//   sum_k x_k (code_k - zero) scale = scale * (sum_k x_k (128 + code_k) - (128 + zero) * sum_k x_k)
// 128 + code is a bf16 whose low bits are the code: bits 0x4300 | code, one instruction for two of them and no conversion.  The sum
// of x_k is a product with ones by the same matrix instruction, whose rate a call of few rows does not use up, in the same lanes.  All
// of it in fp32: what is subtracted is up to 143 / 8 times as large as what is left, so that four bits of 24 go.  The scale, fp32 again,
// meets the sum: a weight itself is never rounded.
//
// Kept in the order in which a wavefront holds them as the second input of v_mfma_f32_16x16x32_bf16 (column lane % 16, k-values
// 8 * (lane / 16) .. +7):
//   codes   [expert][16 columns][128 k-values]: 1024 bytes = [64 lanes][4 words], word m the k-values 32 m + 8 * (lane / 16) .. +7 of
//           column lane % 16; k-value 2 i in bits 4 i .. +3, 2 i + 1 in bits 16 + 4 i .. +3, so that a shift and a mask give a pair
//   scales  [expert][16 columns][128 k-values][16][128 / group] words: the scale's fp32 bits (of a 16-bit type: the low 13 are zero) and,
//           in the low four, the zero
// Past the last k-value the codes are the zero of their group, or the scales are zero.  The columns of the first product are those of its
// two halves in turn, 16 a and 16 b.
#include <algorithm>

#include "gemm_span.hpp"

namespace momoe {
namespace {

constexpr int kInt4Block = 128;
constexpr int kInt4Frag = 1024;  // bytes of 16 columns x 128 k-values

__host__ __device__ inline int64_t int4_blocks(int64_t n) { return (n + kInt4Block - 1) / kInt4Block; }

struct Int4Args {
  const bf16* rows;  // [M or Msum][ld]
  int64_t ld;
  const uint8_t* w;
  const uint32_t* scale;
  const int32_t *idx, *table;  // of experts; null: a dense block of M rows
  int M;                       // (0: experts)
  int K, KB, pairs;            // contraction, its blocks; pairs of 16-column groups
  const float* s;              // second product of experts
  int64_t sn, sm;
  void* out;                   // h bf16 [.][ldo]; ys fp32 [.][ldo] of experts, y bf16 of a dense block
  int64_t ldo;
  // tall tiles whose contraction is cut: sums by slices, fp32 [slices][all rows][2 H or D], and what there is of rows
  int slices;
  float* part;
  int64_t all_rows;
  // elements from h to what its rounding to bf16 leaves, of tiles of up to 16 rows; 0: not kept
  int64_t rest;
};

// Eight codes of a word as 128 + code, two at a time; k128: 0x43004300 in a vector register (of two constants outside them the and and
// the or are an instruction each)
__device__ __forceinline__ uint32_t two_codes(uint32_t w, int i, uint32_t k128) { return ((w >> (4 * i)) & 0x000F000Fu) | k128; }
__device__ __forceinline__ bf16x8 bf16_of_codes(uint32_t w, uint32_t k128) {
  return __builtin_bit_cast(bf16x8, u32x4{two_codes(w, 0, k128), two_codes(w, 1, k128), two_codes(w, 2, k128), two_codes(w, 3, k128)});
}
__device__ __forceinline__ uint32_t two_of_128() {
  uint32_t v = 0x43004300u;
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ float scale_of_word(uint32_t w) { return __uint_as_float(w & ~15u); }
__device__ __forceinline__ float zero_of_word(uint32_t w) { return __uint_as_float(0x43000000u | (w & 15u) << 16); }  // 128 + zero

// Tiles of experts, by the index build's table, or of a dense block, which has none: all rows are those of one expert
struct Int4Sched {
  TileSchedT<1> experts;
  int row_tiles, total, pos, end, tile_rows, rows;
  // (of a dense block `experts` reads the first two words of the codes, and nothing is made of them)
  __device__ __forceinline__ Int4Sched(const Int4Args& p, int nb, int tile_rows_)
      : experts(p.table ? p.table : (const int32_t*)p.w, nb, tile_rows_), tile_rows(tile_rows_), rows(p.M) {
    // an XCD has a contiguous eighth, row tiles fastest: those that share weights meet in one L2
    row_tiles = (rows + tile_rows - 1) / tile_rows;
    total = row_tiles * nb;
    const int chunk = (total + 7) >> 3, begin = (int)(blockIdx.x & 7) * chunk;
    end = min(begin + chunk, total);
    pos = begin + (int)(blockIdx.x >> 3);
  }
  __device__ __forceinline__ TileCoord next() {
    if (rows == 0) return experts.next();
    TileCoord t = {};
    t.valid = pos < end;
    if (!t.valid) return t;
    t.tn = pos / row_tiles;
    t.row0 = (pos - t.tn * row_tiles) * tile_rows;
    t.rows = min(tile_rows, rows - t.row0);
    pos += gridDim.x >> 3;
    return t;
  }
};

// column `col` of both groups of a pair, of one row: h of a and b, or two columns of the result, of experts times the gate weight
template <bool FIRST>
__device__ __forceinline__ void store_pair(const Int4Args& p, int64_t row, int pair, int col, float v0, float v1, float s) {
  if constexpr (FIRST) {
    const float h = v0 * v1 * sigmoidf_fast(v1);
    bf16* const to = (bf16*)p.out + row * p.ldo + 16 * pair + col;
    const bf16 first = f2bf(h);
    to[0] = first;
    if (p.rest) to[p.rest] = f2bf(rest_of(h, first));
  } else {
    const int64_t to = row * p.ldo + 32 * pair + col;
    if (p.idx) {
      ((float*)p.out)[to] = v0 * s;
      ((float*)p.out)[to + 16] = v1 * s;
    } else {
      ((bf16*)p.out)[to] = f2bf(v0);
      ((bf16*)p.out)[to + 16] = f2bf(v1);
    }
  }
}

// Tiles of up to 32 rows.  A wavefront owns a pair of 16-column groups; KS of them share its contraction, a block of 128 k-values in
// KS each, and their sums meet in LDS.  Codes and scales go straight into registers, AHEAD blocks ahead; the rows come to LDS,
// kFewBytes of them at a time, for all wavefronts.  Bound by the rows' way to LDS where they are many, 50 tokens through 2176 x 1152
// in groups of 32 in 14.6 and 11.1 us, else by the first answer of memory: 8 of 128 experts of 2048 x 768, 7.6 and 6.5 us.
constexpr int kFewThreads = 256, kFewWaves = kFewThreads / 64, kFewBytes = 32 << 10;

// REST: of the second product, with what bf16 left of h (for all of them: 50 tokens, 2176 x 1152, groups of 32, 28 us instead of 25).
template <bool FIRST, bool REST, int KS, int SG>
__global__ __launch_bounds__(kFewThreads, 2) void int4_few_rows_kernel(Int4Args p) {
  constexpr int FR = 2, ROWS = 16 * FR, PW = kFewWaves / KS;
  constexpr int AHEAD = SG == 4 ? 2 : 4;  // (four of the smallest groups' scales were spilled)
  __shared__ __attribute__((aligned(16))) uint8_t lds[kFewBytes];  // rows [block][row][256], then the sums of KS wavefronts
  static_assert(kFewWaves * 64 * 2 * FR * 16 <= kFewBytes, "sums of all wavefronts");
  typedef uint32_t Words __attribute__((ext_vector_type(SG)));
  const int tid = threadIdx.x, l = tid & 63, wave = wave_id(), kw = wave % KS, cw = wave / KS;
  Int4Sched sched(p, (p.pairs + PW - 1) / PW, ROWS);
  const uint32_t k128 = two_of_128();
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
  for (TileCoord tc = sched.next(); tc.valid; tc = sched.next()) {
    const int pair = min(tc.tn * PW + cw, p.pairs - 1);
    const bool real = tc.tn * PW + cw < p.pairs;
    // of up to 16 rows of h a second fragment holds what the first one's rounding left
    const bool twice = REST && tc.rows <= 16;
    const int nf = twice ? 2 : (tc.rows + 15) >> 4, held = twice ? 2 * tc.rows : tc.rows;
    int at_row[FR];
#pragma unroll
    for (int i = 0; i < FR; ++i) at_row[i] = min((twice ? 0 : 16 * i) + (l & 15), tc.rows - 1) + (twice ? i * tc.rows : 0);
    const int64_t group = ((int64_t)tc.expert * p.pairs + pair) * 2 * p.KB;
    const uint8_t* const w0 = p.w + group * kInt4Frag + l * 16;
    const uint32_t* const s0 = p.scale + (group * 16 + (l & 15)) * SG;
    f32x4 acc[2][FR] = {};
    const int chunk = kFewBytes / (held * kInt4Block * 2);  // blocks of the tile's rows that LDS holds, four at least
    for (int k0 = 0; k0 < p.KB; k0 += chunk) {
      const int blocks = min(chunk, p.KB - k0), steps = (blocks - kw + KS - 1) / KS;  // (none for a wavefront past the last)
      u32x4 wq[AHEAD][2];
      Words sq[AHEAD][2];
      const auto load = [&](int q, int step) {
        const int64_t at = k0 + step * KS + kw;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          wq[q][j] = *(const u32x4*)(w0 + (j * (int64_t)p.KB + at) * kInt4Frag);
          sq[q][j] = *(const Words*)(s0 + (j * (int64_t)p.KB + at) * (16 * SG));
        }
      };
      unrolled<0, AHEAD>([&](auto QC) {
        if (decltype(QC)::value < steps) load(decltype(QC)::value, decltype(QC)::value);
      });
      __syncthreads();  // (the last rows, or sums, are done with)
      // 16 pieces of 8 values a row and block, piece c of row r at c ^ (r % 16): the 16 rows of a fragment read meet different
      // banks.  Rows that the tile does not have are read as its last one, and nobody stores what becomes of them.
      const int all = blocks * held * 16;
      for (int q0 = tid; q0 < all; q0 += 2 * kFewThreads) {
        bf16x8 v[2];
        int to[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int q = min(q0 + a * kFewThreads, all - 1), piece = q & 15, kb = (q >> 4) / held, r = (q >> 4) - kb * held;
          const bool rest = REST && r >= tc.rows;
          const int c = (k0 + kb) * kInt4Block + piece * 8, row = tc.row0 + (rest ? r - tc.rows : r);
          v[a] = *(const bf16x8*)(p.rows + (rest ? p.rest : 0) + (int64_t)(FIRST && p.idx ? p.idx[row] : row) * p.ld + min(c, p.K - 8));
          if (c >= p.K) v[a] = bf16x8{};
          to[a] = (kb * held + r) * 256 + ((piece ^ (r & 15)) << 4);
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) *(bf16x8*)(lds + to[a]) = v[a];
      }
      __syncthreads();
      const auto multiply = [&](int q, int step) {
        const int kb = step * KS + kw;
        bf16x8 wf[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int m = 0; m < 4; ++m) wf[j][m] = bf16_of_codes(wq[q][j][m], k128);
        unrolled<0, FR>([&](auto IC) {
          constexpr int i = decltype(IC)::value;
          if (i >= nf) return;  // (the same for all lanes)
          const int row = at_row[i];
          const uint8_t* const from = lds + (kb * held + row) * 256;
          bf16x8 rf[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) rf[m] = *(const bf16x8*)(from + (((4 * m + (l >> 4)) ^ (row & 15)) << 4));
#pragma unroll
          for (int g = 0; g < SG; ++g) {
            f32x4 t[2] = {}, sum = {};
#pragma unroll
            for (int m = g * (4 / SG); m < (g + 1) * (4 / SG); ++m) {
              sum = mfma16(rf[m], ones, sum);
#pragma unroll
              for (int j = 0; j < 2; ++j) t[j] = mfma16(rf[m], wf[j][m], t[j]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const float sc = scale_of_word(sq[q][j][g]), zc = zero_of_word(sq[q][j][g]);
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(sc, fmaf(-zc, sum[r], t[j][r]), acc[j][i][r]);
              asm volatile("" : "+v"(acc[j][i]));  // (the products of all fragments were formed first, and spilled)
            }
          }
        });
      };
      // what is multiplied last has nothing to request: apart, as behind a request that may not be made the compiler waits for all
      int step = 0;
#pragma unroll 1
      for (; step + 2 * AHEAD <= steps; step += AHEAD)
        unrolled<0, AHEAD>([&](auto QC) {
          constexpr int q = decltype(QC)::value;
          multiply(q, step + q);
          load(q, step + q + AHEAD);
        });
      unrolled<0, AHEAD>([&](auto QC) {
        constexpr int q = decltype(QC)::value;
        if (step + q < steps) multiply(q, step + q);
        if (step + q + AHEAD < steps) load(q, step + q + AHEAD);
      });
      unrolled<0, AHEAD>([&](auto QC) {
        constexpr int q = decltype(QC)::value;
        if (step + q + AHEAD < steps) multiply(q, step + q + AHEAD);
      });
    }
    if (twice) {
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[j][0] += acc[j][1];
    }
    if constexpr (KS > 1) {
      __syncthreads();
      f32x4* const sums = (f32x4*)lds + wave * (2 * FR) * 64 + l;
#pragma unroll
      for (int n = 0; n < 2 * FR; ++n) sums[n * 64] = acc[n / FR][n % FR];
      __syncthreads();
      if (kw == 0) {
#pragma unroll
        for (int n = 0; n < 2 * FR; ++n)
#pragma unroll
          for (int k = 1; k < KS; ++k) acc[n / FR][n % FR] += sums[(k * (2 * FR) + n) * 64];
      }
    }
    if (!real || kw != 0) continue;
    // a lane has column lane % 16 of rows 4 * (lane / 16) .. +3 of a fragment
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 16 * i + 4 * (l >> 4) + r;
        if (at >= tc.rows) continue;
        const int64_t row = tc.row0 + at;
        float s = 1.0f;
        if (!FIRST && p.idx) s = p.s[(int64_t)tc.expert * p.sn + (int64_t)p.idx[row] * p.sm];
        store_pair<FIRST>(p, row, pair, l & 15, acc[0][i][r], acc[1][i][r], s);
      }
  }
}

// Tiles of 64 rows x 256 columns, for more rows than that: a wavefront owns 64 columns of them, two pairs of groups.  The rows come to LDS by
// direct transfers, 128 k-values a stage, the codes and scales straight into registers; both are requested a stage ahead, and two
// workgroups share a CU, so that one's products stand beside the other's vector work: for each 64 matrix instructions of a wavefront's
// stage there are 112 instructions that make bf16 of codes and 64 that bring the sums of a group to the others (groups of 32: 256).
// acc += scale * sum_k x_k (128 + code_k) as each group ends; what that is too much by, (128 + zero) scale * sum_k x_k, is a product
// of fp32 itself, contracted over the groups, and taken away four of them at a time by v_mfma_f32_16x16x4_f32.  (All at the end would
// let sums of thousands of 128 x_k meet.)  Each of the first wavefronts sums one fragment of rows, for all of them, in LDS; two sets in
// turn, as a barrier a stage lies between the writing of one and its use.  4096 tokens, 4096 x 11264: 1333 us with sums and differences
// of their own in each wavefront, 1243 this way, 0.91 PFLOP/s.  It is bound by issue, the matrix instructions being busy half of the
// time and the vector ones two thirds.  8 of 128 experts of 2048 x 768, groups of 128, whole calls: 0.35 PFLOP/s at 1000 tokens, 0.46 at
// 2000, 0.53 at 4096, 0.57 at 16384.
// Not faster: 128 rows a tile; wavefronts of 32 columns, eight a workgroup (1672) or four, of 64 rows and three workgroups a CU (1391;
// 1000 tokens to 8 of 128 experts, groups of 64, 224 | 227) or of 96 and two (1439; 232); all fragments without a branch between
// them, which spills (1566).
// Fragments of rows that the tile does not have are left out.  A launch of few tiles has its contraction cut into slices,
// whose sums int4_h_of_slices_kernel or the last kernel adds up.
struct Int4Rows {
  static constexpr int BM = 64, DEP = BM * 256 / (kSpanWaves * 1024), STAGE = BM * 256;  // bytes
  const char *base, *second;  // of the second deposit, which may be what the first one's rounding left
  uint32_t off[DEP];
  __device__ __forceinline__ void init(const Int4Args& p, const TileCoord& tc, bool gather, bool twice) {
    const int l = fresh_lane();
    base = (const char*)p.rows;
    if (!gather) base += (int64_t)tc.row0 * p.ld * 2;
    second = twice ? base + p.rest * 2 : base;
#pragma unroll
    for (int j = 0; j < DEP; ++j) {
      const int r = min(((twice ? 0 : j) * kSpanWaves + wave_id()) * 4 + (l >> 4), tc.rows - 1);
      off[j] = (uint32_t)(gather ? p.idx[tc.row0 + r] : r) * (uint32_t)(2 * p.ld);
    }
  }
  // 16 rows a deposit; piece c of row r at c ^ (r % 16).  Past the row's end its last piece is repeated: codes that are the zero of their
  // group, or a scale of zero, make nothing of it.
  __device__ __forceinline__ void request(int kb, int K, int nf, uint32_t slot) const {
    const int l = fresh_lane(), piece = (l & 15) ^ ((wave_id() * 4 + (l >> 4)) & 15);
    const uint32_t at = (uint32_t)min(kb * kInt4Block + piece * 8, K - 8) * 2;
    unrolled<0, DEP>([&](auto J) {
      constexpr int j = decltype(J)::value;
      if (j < nf) dma16_at<j * kSpanWaves * 1024>(j == 1 ? second : base, off[j] + at, slot);
    });
  }
};

template <bool FIRST, int SG>
__global__ __launch_bounds__(kSpanThreads, 2) void int4_tile_kernel(Int4Args p) {
  using Rows = Int4Rows;
  constexpr int PAIRS = 2 * kSpanWaves, STEPS = 4 / SG;
  typedef uint32_t Words __attribute__((ext_vector_type(SG)));
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * Rows::STAGE];
  __shared__ float sums[2][4][Rows::BM];  // of x_k over each of four groups, of a row
  const int l = lane_id(), wave = wave_id();
  const uint32_t addr = lds_address((bf16*)lds) + wave * 1024;
  Int4Sched sched(p, (p.pairs + PAIRS - 1) / PAIRS * p.slices, Rows::BM);
  const uint32_t k128 = two_of_128();
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
  struct Tile {
    TileCoord tc;
    int slice, kb0, kb1, nf, pair0;
    bool twice;  // of up to 16 rows of h a second fragment holds what the first one's rounding left
    __device__ __forceinline__ void place(const Int4Args& p, const TileCoord& t) {
      tc = t;
      const int tn = t.tn / p.slices;
      slice = t.tn - tn * p.slices;
      kb0 = (int)((int64_t)p.KB * slice / p.slices), kb1 = (int)((int64_t)p.KB * (slice + 1) / p.slices);
      twice = !FIRST && p.rest && t.rows <= 16;
      nf = twice ? 2 : (t.rows + 15) >> 4;
      pair0 = tn * PAIRS + 2 * wave_id();
    }
  };
  Tile cur, next;
  next.place(p, sched.next());
  if (!next.tc.valid) return;
  Rows A;
  const uint8_t* w[4];
  const uint32_t* sc[4];
  u32x4 wq[4];
  Words sq[4];
  const auto load = [&](int kb) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      wq[j] = *(const u32x4*)(w[j] + (int64_t)kb * kInt4Frag + l * 16);
      sq[j] = *(const Words*)(sc[j] + (int64_t)kb * (16 * SG) + (l & 15) * SG);
    }
  };
  // the first stage of the next tile, into the half of LDS that nobody reads
  int q = 0, parity = 0;
  const auto begin = [&] {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t group = (((int64_t)next.tc.expert * p.pairs + min(next.pair0 + j / 2, p.pairs - 1)) * 2 + j % 2) * p.KB;
      w[j] = p.w + group * kInt4Frag;
      sc[j] = p.scale + group * (16 * SG);
    }
    A.request(next.kb0, p.K, next.nf, addr + q * Rows::STAGE);
    load(next.kb0);
  };
  A.init(p, next.tc, FIRST && p.idx, next.twice);
  begin();
  while (true) {
    cur = next;
    next.place(p, sched.next());
    Rows B;  // rows of the next tile: their tokens travel meanwhile
    if (next.tc.valid) B.init(p, next.tc, FIRST && p.idx, next.twice);
    const int nf = cur.nf;
    f32x4 acc[4][4] = {};
    // -(128 + zero) scale of up to four groups, lane l that of group l / 16 and column l % 16, for what these take away of acc
    float away[4] = {};
    int held = 0;
    const auto take_away = [&] {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= nf) break;
        const float sum = l >> 4 < held ? sums[parity][l >> 4][16 * i + (l & 15)] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(sum, away[j], acc[j][i], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) away[j] = 0.0f;
      held = 0;
      parity ^= 1;
    };
    for (int kb = cur.kb0; kb < cur.kb1; ++kb) {
      wait_vmcnt<0>();
      wait_lgkm0();
      __builtin_amdgcn_s_barrier();
      order_fence();
      if (held == 4) take_away();
      if (kb + 1 < cur.kb1) A.request(kb + 1, p.K, nf, addr + (q ^ 1) * Rows::STAGE);
      order_fence();
      u32x4 codes[4];
      Words scales[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) codes[j] = wq[j], scales[j] = sq[j];
      load(min(kb + 1, cur.kb1 - 1));
      order_fence();
      const uint8_t* const rows = lds + q * Rows::STAGE + (l & 15) * 256;
      unrolled<0, SG>([&](auto GC) {
        constexpr int g = decltype(GC)::value;
        bf16x8 wf[4][STEPS];
        float s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[j] = scale_of_word(scales[j][g]);
          if (l >> 4 == held + g) away[j] = -s[j] * zero_of_word(scales[j][g]);
#pragma unroll
          for (int m = 0; m < STEPS; ++m) wf[j][m] = bf16_of_codes(codes[j][g * STEPS + m], k128);
        }
        unrolled<0, 4>([&](auto IC) {
          constexpr int i = decltype(IC)::value;
          if (i >= nf) return;  // (the same for all lanes)
          bf16x8 rf[STEPS];
#pragma unroll
          for (int m = 0; m < STEPS; ++m)
            rf[m] = *(const bf16x8*)(rows + i * (16 * 256) + (((4 * (g * STEPS + m) + (l >> 4)) ^ (l & 15)) << 4));
          f32x4 t[4] = {};
#pragma unroll
          for (int m = 0; m < STEPS; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = mfma16(rf[m], wf[j][m], t[j]);
          if (i == wave) {
            f32x4 sum = {};
#pragma unroll
            for (int m = 0; m < STEPS; ++m) sum = mfma16(ones, rf[m], sum);
            if (l < 16) sums[parity][held + g][16 * i + l] = sum[0];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(s[j], t[j][r], acc[j][i][r]);
            asm volatile("" : "+v"(acc[j][i]));  // (the products of all fragments were formed first, and spilled)
          }
        });
      });
      held += SG;
      order_fence();
      q ^= 1;
    }
    wait_lgkm0();
    __builtin_amdgcn_s_barrier();
    order_fence();
    take_away();
    if (cur.twice) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j][0] += acc[j][1];
    }
    if (next.tc.valid) {
      A = B;
      begin();
    }
    const int col = l & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i >= nf) break;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 16 * i + 4 * (l >> 4) + r;
        if (at >= cur.tc.rows) continue;
        const int64_t row = cur.tc.row0 + at;
        float s = 1.0f;
        if (!FIRST && p.idx) s = p.s[(int64_t)cur.tc.expert * p.sn + (int64_t)p.idx[row] * p.sm];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int pair = cur.pair0 + c;
          if (pair >= p.pairs) continue;
          const float v0 = acc[2 * c][i][r], v1 = acc[2 * c + 1][i][r];
          if (p.slices == 1) {
            store_pair<FIRST>(p, row, pair, col, v0, v1, s);
          } else if (FIRST) {
            float* const to = p.part + (cur.slice * p.all_rows + row) * (2 * p.ldo) + 16 * pair + col;
            to[0] = v0;
            to[p.ldo] = v1;
          } else {
            float* const to = p.part + (cur.slice * p.all_rows + row) * p.ldo + 32 * pair + col;
            to[0] = v0 * s;
            to[16] = v1 * s;
          }
        }
      }
    }
    if (!next.tc.valid) break;
  }
}

// The sum of eight at a time of `slices` values that lie `stride` apart, in their order
__device__ __forceinline__ f32x4 sum_of_slices(const float* p, int slices, int64_t stride) {
  f32x4 sum = {};
  for (int s = 0; s < slices; s += 8) {
    f32x4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = *(const f32x4*)(p + min(s + j, slices - 1) * stride);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s + j < slices) sum += v[j];
  }
  return sum;
}
// h from the slices of a | b, fp32 [slices][rows][2H]
__global__ __launch_bounds__(256) void int4_h_of_slices_kernel(const float* __restrict__ part, bf16* __restrict__ h, int64_t rows, int H,
                                                               int slices, int64_t rest) {
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x, row = q / (H / 4);
  const int col = (int)(q - row * (H / 4)) * 4;
  if (row >= rows) return;
  const float* const from = part + row * 2 * H + col;
  const f32x4 a = sum_of_slices(from, slices, rows * 2 * H), b = sum_of_slices(from + H, slices, rows * 2 * H);
  bf16x4 v, left;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = a[e] * b[e] * sigmoidf_fast(b[e]);
    v[e] = f2bf(x);
    left[e] = f2bf(rest_of(x, v[e]));
  }
  *(bf16x4*)(h + row * H + col) = v;
  if (rest) *(bf16x4*)(h + rest + row * H + col) = left;
}
// y of a dense block from its slices, fp32 [slices][n]
__global__ __launch_bounds__(256) void int4_sum_slices_kernel(const float* __restrict__ part, bf16* __restrict__ y, int64_t n, int slices) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const f32x4 v = sum_of_slices(part + at, slices, n);
  *(bf16x4*)(y + at) = pack_bf16x4(v, 1.0f);
}

// out[m] = the sum of the rows of its experts, slice by slice, fp32, rounded once.  The row numbers and then the rows with unconditional
// loads, as in combine_kernel.
__global__ __launch_bounds__(256) void int4_combine_kernel(const float* __restrict__ rows, int slices, const int32_t* __restrict__ inv,
                                                           bf16* __restrict__ out, int64_t M, int D, int K, int64_t msum) {
  for (int64_t m = blockIdx.x; m < M; m += gridDim.x)
    for (int c = threadIdx.x; c < D / 4; c += blockDim.x) {
      f32x4 sum = {};
      for (int k0 = 0; k0 < K; k0 += 8) {
        int32_t r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = inv[m * K + min(k0 + j, K - 1)];
        for (int s = 0; s < slices; ++s) {
          const float* const from = rows + s * msum * D + c * 4;
          f32x4 v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const bool ok = k0 + j < K && (uint32_t)r[j] < (uint64_t)msum;
            v[j] = *(const f32x4*)(from + (int64_t)(ok ? r[j] : 0) * D);
            if (!ok) v[j] = f32x4{};
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) sum += v[j];
        }
      }
      *(bf16x4*)(out + m * D + c * 4) = pack_bf16x4(sum[0], sum[1], sum[2], sum[3]);
    }
}

// Workgroups of 256 of a launch that has `n` of them to do: a launch has fewer than 2^32 threads, and what is left they do in turn.
unsigned workgroups_for(int64_t n) { return (unsigned)std::min<int64_t>(n, 1 << 23); }

// ---- laying weights out ---------------------------------------------------------------------------------------------------
struct Int4PackArgs {
  const uint8_t* w;  // [N][R / 2][C], C = halves * cols
  const void* scale; // [N][ceil(R / group)][C], bf16 or fp16
  const uint8_t* zero;
  int64_t N;
  int R, cols, halves, group, f16;
  uint32_t *codes, *words;
};
// of group `g` of 16 columns, in the order in which they are kept, column c
__device__ __forceinline__ int column_of(const Int4PackArgs& p, int g, int c) { return g % p.halves * p.cols + g / p.halves * 16 + c; }

__global__ __launch_bounds__(256) void int4_pack_codes_kernel(Int4PackArgs p) {
  const int KB = (int)int4_blocks(p.R), C = p.cols * p.halves, groups = C / 16;
  const int64_t all = p.N * groups * KB * 256;  // [N][groups][KB][64][4]
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < all; q += (int64_t)gridDim.x * 256) {
    const int m = q & 3, l = (int)(q >> 2) & 63;
    const int64_t f = q >> 8;
    const int kb = (int)(f % KB), g = (int)(f / KB % groups);
    const int64_t e = f / KB / groups;
    const int k = kb * kInt4Block + 32 * m + 8 * (l >> 4), col = column_of(p, g, l & 15);
    const int KG = (p.R + p.group - 1) / p.group, kg = k / p.group;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t b = 0;
      if (k + 2 * i < p.R) b = p.w[(e * (p.R / 2) + k / 2 + i) * C + col];
      else if (kg < KG) b = (p.zero ? p.zero[(e * KG + kg) * C + col] & 15u : 8u) * 17u;  // the zero of its group
      word |= (b & 15u) << (4 * i) | (b >> 4) << (16 + 4 * i);
    }
    p.codes[q] = word;
  }
}

__global__ __launch_bounds__(256) void int4_pack_scales_kernel(Int4PackArgs p) {
  const int KB = (int)int4_blocks(p.R), C = p.cols * p.halves, groups = C / 16, SG = kInt4Block / p.group;
  const int KG = (p.R + p.group - 1) / p.group;
  const int64_t all = p.N * groups * KB * 16 * SG;  // [N][groups][KB][16][SG]
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < all; q += (int64_t)gridDim.x * 256) {
    const int sg = (int)(q % SG), c = (int)(q / SG) & 15;
    const int64_t f = q / SG >> 4;
    const int kb = (int)(f % KB), g = (int)(f / KB % groups), kg = kb * SG + sg;
    uint32_t word = 0;
    if (kg < KG) {
      const int64_t at = (f / KB / groups * KG + kg) * C + column_of(p, g, c);
      const float s = p.f16 ? (float)((const _Float16*)p.scale)[at] : (float)((const bf16*)p.scale)[at];
      word = (__float_as_uint(s) & ~15u) | (p.zero ? p.zero[at] & 15u : 8u);
    }
    p.words[q] = word;
  }
}

int check_int4(int64_t M, int64_t D, int64_t H, int64_t N, int64_t Msum, int group) {
  if (M <= 0 || D <= 0 || H <= 0 || N <= 0 || Msum <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || H % 32 != 0 || Msum >= (1ll << 31) - 512 || M >= (1ll << 31) - 512 || D >= (1 << 22) || H >= (1 << 22))
    return MOMOE_ERR_UNSUPPORTED;
  return group == 32 || group == 64 || group == 128 ? MOMOE_OK : MOMOE_ERR_UNSUPPORTED;
}
bool unaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }

template <bool FIRST, bool REST, int SG>
int launch_few(const Int4Args& a, int64_t tiles, hipStream_t st) {
  const int64_t wanted = 3 * persistent_grid();
  const auto enough = [&](int ks) { return a.KB < 2 * ks || tiles * cdiv64(a.pairs, kFewWaves / ks) >= wanted; };
  auto kernel = enough(1)   ? int4_few_rows_kernel<FIRST, REST, 1, SG>
                : enough(2) ? int4_few_rows_kernel<FIRST, REST, 2, SG>
                            : int4_few_rows_kernel<FIRST, REST, 4, SG>;
  kernel<<<(unsigned)wanted, kFewThreads, 0, st>>>(a);
  return launch_status();
}
template <bool FIRST, int SG>
int launch_rows(const Int4Args& a, int64_t tiles, int tile_rows, hipStream_t st) {
  if constexpr (!FIRST)
    if (tile_rows == 32 && a.rest) return launch_few<false, true, SG>(a, tiles, st);
  if (tile_rows == 32) return launch_few<FIRST, false, SG>(a, tiles, st);
  int4_tile_kernel<FIRST, SG><<<(unsigned)(2 * persistent_grid()), kSpanThreads, 0, st>>>(a);
  return launch_status();
}
// `tiles` of `tile_rows` rows (32 or 64)
template <bool FIRST>
int launch(const Int4Args& a, int64_t tiles, int tile_rows, int group, hipStream_t st) {
  return group == 128 ? launch_rows<FIRST, 1>(a, tiles, tile_rows, st)
         : group == 64 ? launch_rows<FIRST, 2>(a, tiles, tile_rows, st) : launch_rows<FIRST, 4>(a, tiles, tile_rows, st);
}
// row tiles that a launch has about: one for each expert that may hold a row; more where the rows fill more than that
int64_t row_tiles_of(int64_t Msum, int64_t N, int tile_rows) { return std::max(std::min(N, Msum), cdiv64(Msum, tile_rows)); }
// Which tiles.  Those of 32 rows bring their rows to LDS for few columns at a time, but cut a contraction among the wavefronts of a
// workgroup: they are the better ones for few rows and small weights, where the taller ones leave sums to another launch.
// Rule: by what all rows together read of codes, or of one block by its size.
// Record, us, 32 rows | 64:
//   8 of 128 experts of 2048 x 768, 1 token 20 | 25, 16 tokens 71 | 63, 131 128 | 85
//   dense, 1024 x 2816, 4 tokens 14 | 19, 16 18 | 19, 32 29 | 23, 200 42 | 41;  512 x 1024, 200 17 | 27;  2048 x 5632, 4 19 | 21, 16 31 | 24
//          4096 x 11264, 1 token 30 | 28;  groups of 32, 2176 x 1152, 50 27 | 37
int tile_rows_of(int64_t Msum, int64_t D, int64_t H, int64_t N) {
  const int64_t codes = 3 * D * H / 2;
  return Msum * codes <= (64 << 20) || (N == 1 && Msum <= 256 && codes <= (4 << 20)) ? 32 : 64;
}
// Rule: slices of a contraction of K in 64-row tiles over `cols` columns (of both halves): as many as give every CU two tiles, of two
// stages at least, up to 64 MiB of sums.
// Record, us, a dense block with both contractions whole | cut:
//   4096 x 11264, 1 token 105 | 30, 64 194 | 62;  2048 x 5632, 300 106 | 66, 1000 137 | 113;  1024 x 2816, 600 62 | 55
int slices_of(int64_t Msum, int64_t N, int64_t cols, int64_t K, int tile_rows) {
  if (tile_rows != 64) return 1;
  const int64_t tiles = row_tiles_of(Msum, N, tile_rows) * cdiv64(cols, 256);
  int64_t n = std::max<int64_t>(1, std::min(2 * persistent_grid() / tiles, int4_blocks(K) / 2));
  n = std::max<int64_t>(1, std::min<int64_t>(n, (64 << 20) / (Msum * cols * 4)));
  return (int)n;
}

// Rule: what bf16 leaves of h is kept, too, of up to 16 rows an expert on average, and meets the weights as rows of their tiles' second
// fragments: of so few results the error depends on the few large values of h (one token against 64 bits 0.0017 to 0.0024 of the norm,
// 0.0017 this way).  It costs the second product of 16 tokens through 8 of 128 experts, 64-row tiles, 25.6 us instead of 21.3, of one
// token 6.5 instead of 5.7.
bool keeps_rest(int64_t Msum, int64_t N) { return Msum <= 16 * N; }

// the first product, of experts or of a dense block, with the sums of its slices in the workspace
int launch_first(Int4Args a, int64_t N, int64_t Msum, int tile_rows, int group, void* workspace, int64_t workspace_bytes, hipStream_t st) {
  a.slices = slices_of(Msum, N, 2 * a.ldo, a.K, tile_rows);
  a.part = (float*)workspace;
  a.all_rows = Msum;
  a.rest = keeps_rest(Msum, N) ? Msum * a.ldo : 0;
  if (a.slices > 1 && (!workspace || workspace_bytes < a.slices * Msum * 2 * a.ldo * 4)) return MOMOE_ERR_BAD_ARG;
  const int status = launch<true>(a, row_tiles_of(Msum, N, tile_rows), tile_rows, group, st);
  if (status != MOMOE_OK || a.slices == 1) return status;
  const int64_t quads = Msum * (a.ldo / 4);
  int4_h_of_slices_kernel<<<(unsigned)cdiv64(quads, 256), 256, 0, st>>>(a.part, (bf16*)a.out, Msum, (int)a.ldo, a.slices, a.rest);
  return launch_status();
}

}  // namespace
}  // namespace momoe

using namespace momoe;

extern "C" int64_t momoe_int4_weight_bytes(int64_t N, int64_t R, int64_t C) {
  if (N <= 0 || R <= 0 || C <= 0 || C % 16 != 0) return -1;
  return N * (C / 16) * int4_blocks(R) * kInt4Frag;
}
extern "C" int64_t momoe_int4_scale_words(int64_t N, int64_t R, int64_t C, int group) {
  if (N <= 0 || R <= 0 || C <= 0 || C % 16 != 0 || (group != 32 && group != 64 && group != 128)) return -1;
  return N * C * int4_blocks(R) * (kInt4Block / group);
}

extern "C" int momoe_int4_pack_weights(const void* codes_NRC, const void* scale, int scale_type, const void* zero, int64_t N, int64_t R,
                                       int64_t C, int halves, int group, void* packed, void* words, void* stream) {
  if (!codes_NRC || !scale || !packed || !words || N <= 0 || R <= 0 || C <= 0 || halves < 1 || halves > 2) return MOMOE_ERR_BAD_ARG;
  if (scale_type != MOMOE_TYPE_BF16 && scale_type != MOMOE_TYPE_F16) return MOMOE_ERR_BAD_ARG;
  if (unaligned16(packed) || unaligned16(words) || ((uintptr_t)scale & 1)) return MOMOE_ERR_BAD_ARG;
  if (R % 32 != 0 || C % (16 * halves) != 0 || R >= (1 << 22) || C >= (1 << 24)) return MOMOE_ERR_UNSUPPORTED;
  const int64_t bytes = momoe_int4_weight_bytes(N, R, C), nwords = momoe_int4_scale_words(N, R, C, group);
  if (nwords < 0) return MOMOE_ERR_UNSUPPORTED;
  const Int4PackArgs a{(const uint8_t*)codes_NRC, scale, (const uint8_t*)zero, N, (int)R, (int)(C / halves), halves, group,
                       scale_type == MOMOE_TYPE_F16, (uint32_t*)packed, (uint32_t*)words};
  int4_pack_codes_kernel<<<workgroups_for(bytes / 1024), 256, 0, (hipStream_t)stream>>>(a);
  int4_pack_scales_kernel<<<workgroups_for(cdiv64(nwords, 256)), 256, 0, (hipStream_t)stream>>>(a);
  return launch_status();
}

extern "C" int momoe_int4_tile_rows(int64_t Msum, int64_t D, int64_t H, int64_t N) {
  return Msum <= 0 || D <= 0 || H <= 0 || N <= 0 ? 0 : tile_rows_of(Msum, D, H, N);
}
extern "C" int64_t momoe_int4_h_rows(int64_t Msum, int64_t N) { return Msum < 0 || N <= 0 ? -1 : keeps_rest(Msum, N) ? 2 * Msum : Msum; }
extern "C" int momoe_int4_slices(int64_t Msum, int64_t N, int64_t cols, int64_t K, int tile_rows) {
  return Msum <= 0 || N <= 0 || cols <= 0 || K <= 0 ? 0 : slices_of(Msum, N, cols, K, tile_rows);
}

extern "C" int momoe_int4_lin1_swiglu_fwd(const void* x_MD, int64_t ldx, const void* Wl1_packed, const void* Wl1_words, int group,
                                          const int32_t* idx_Msum, const int32_t* tile_table, int tile_rows, void* h_MsumH,
                                          void* workspace, int64_t workspace_bytes, int64_t M, int64_t D, int64_t H, int64_t N,
                                          int64_t Msum, void* stream) {
  if (!x_MD || !Wl1_packed || !Wl1_words || !idx_Msum || !tile_table || !h_MsumH || ldx < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_int4(M, D, H, N, Msum, group);
  if (st != MOMOE_OK) return st;
  if (unaligned16(x_MD) || unaligned16(Wl1_packed) || unaligned16(Wl1_words) || unaligned16(h_MsumH) || unaligned16(workspace))
    return MOMOE_ERR_BAD_ARG;
  // (the taller tiles gather their rows at 32-bit offsets)
  if (ldx % 8 != 0 || (tile_rows != 32 && tile_rows != 64) || (tile_rows == 64 && M * ldx * 2 >= (1ll << 32))) return MOMOE_ERR_UNSUPPORTED;
  Int4Args a{(const bf16*)x_MD, ldx, (const uint8_t*)Wl1_packed, (const uint32_t*)Wl1_words, idx_Msum, tile_table, 0, (int)D,
             (int)int4_blocks(D), (int)(H / 16)};
  a.out = h_MsumH;
  a.ldo = H;
  return launch_first(a, N, Msum, tile_rows, group, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int momoe_int4_lin2_scale_fwd(const void* h_MsumH, const void* Wl2_packed, const void* Wl2_words, int group, const float* s_NM,
                                         int64_t s_stride_n, int64_t s_stride_m, const int32_t* idx_Msum, const int32_t* tile_table,
                                         int tile_rows, float* ys_MsumD, int64_t M, int64_t D, int64_t H, int64_t N, int64_t Msum,
                                         void* stream) {
  if (!h_MsumH || !Wl2_packed || !Wl2_words || !s_NM || !idx_Msum || !tile_table || !ys_MsumD) return MOMOE_ERR_BAD_ARG;
  const int st = check_int4(M, D, H, N, Msum, group);
  if (st != MOMOE_OK) return st;
  if (unaligned16(h_MsumH) || unaligned16(Wl2_packed) || unaligned16(Wl2_words) || unaligned16(ys_MsumD)) return MOMOE_ERR_BAD_ARG;
  if (tile_rows != 32 && tile_rows != 64) return MOMOE_ERR_UNSUPPORTED;
  Int4Args a{(const bf16*)h_MsumH, H, (const uint8_t*)Wl2_packed, (const uint32_t*)Wl2_words, idx_Msum, tile_table, 0, (int)H,
             (int)int4_blocks(H), (int)(D / 32)};
  a.s = s_NM;
  a.sn = s_stride_n;
  a.sm = s_stride_m;
  a.out = ys_MsumD;
  a.ldo = D;
  a.slices = slices_of(Msum, N, D, H, tile_rows);
  a.part = ys_MsumD;
  a.all_rows = Msum;
  a.rest = keeps_rest(Msum, N) ? Msum * H : 0;
  return launch<false>(a, row_tiles_of(Msum, N, tile_rows), tile_rows, group, (hipStream_t)stream);
}

extern "C" int momoe_int4_combine(const float* ys_MsumD, int slices, const int32_t* inv_MK, void* out_MD, int64_t M, int64_t D, int64_t K,
                                  int64_t Msum, void* stream) {
  if (!ys_MsumD || !inv_MK || !out_MD || M <= 0 || D <= 0 || K <= 0 || Msum <= 0 || slices <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || M >= (1ll << 31) || Msum >= (1ll << 31)) return MOMOE_ERR_UNSUPPORTED;
  if (unaligned16(ys_MsumD) || unaligned16(out_MD)) return MOMOE_ERR_BAD_ARG;
  int4_combine_kernel<<<workgroups_for(M), 256, 0, (hipStream_t)stream>>>(ys_MsumD, slices, inv_MK, (bf16*)out_MD, M, (int)D, (int)K, Msum);
  return launch_status();
}

extern "C" int64_t momoe_int4_ffn_workspace_bytes(int64_t M, int64_t D, int64_t H) {
  if (M <= 0 || D <= 0 || H <= 0) return -1;
  const int tile_rows = tile_rows_of(M, D, H, 1);
  const int64_t n1 = slices_of(M, 1, 2 * H, D, tile_rows), n2 = slices_of(M, 1, D, H, tile_rows);
  return std::max(n1 > 1 ? n1 * M * 2 * H * 4 : 0, n2 > 1 ? n2 * M * D * 4 : 0);
}

extern "C" int momoe_int4_ffn_fwd(const void* x_MD, int64_t ldx, const void* Wl1_packed, const void* Wl1_words, const void* Wl2_packed,
                                  const void* Wl2_words, int group, void* h_MH, void* y_MD, void* workspace, int64_t workspace_bytes,
                                  int64_t M, int64_t D, int64_t H, void* stream) {
  if (!x_MD || !Wl1_packed || !Wl1_words || !Wl2_packed || !Wl2_words || !h_MH || !y_MD || ldx < D) return MOMOE_ERR_BAD_ARG;
  int st = check_int4(M, D, H, 1, M, group);
  if (st != MOMOE_OK) return st;
  for (const void* q : {x_MD, Wl1_packed, Wl1_words, Wl2_packed, Wl2_words, (const void*)h_MH, (const void*)y_MD, (const void*)workspace})
    if (unaligned16(q)) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0 || ldx >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  const int64_t need = momoe_int4_ffn_workspace_bytes(M, D, H);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MOMOE_ERR_BAD_ARG;
  const int tile_rows = tile_rows_of(M, D, H, 1);
  Int4Args a{(const bf16*)x_MD, ldx, (const uint8_t*)Wl1_packed, (const uint32_t*)Wl1_words, nullptr, nullptr, (int)M, (int)D,
             (int)int4_blocks(D), (int)(H / 16)};
  a.out = h_MH;
  a.ldo = H;
  hipStream_t to = (hipStream_t)stream;
  st = launch_first(a, 1, M, tile_rows, group, workspace, workspace_bytes, to);
  if (st != MOMOE_OK) return st;
  Int4Args b{(const bf16*)h_MH, H, (const uint8_t*)Wl2_packed, (const uint32_t*)Wl2_words, nullptr, nullptr, (int)M, (int)H,
             (int)int4_blocks(H), (int)(D / 32)};
  b.out = y_MD;
  b.ldo = D;
  b.slices = slices_of(M, 1, D, H, tile_rows);
  b.part = (float*)workspace;
  b.all_rows = M;
  b.rest = keeps_rest(M, 1) ? M * H : 0;
  st = launch<false>(b, cdiv64(M, tile_rows), tile_rows, group, to);
  if (st != MOMOE_OK || b.slices == 1) return st;
  int4_sum_slices_kernel<<<(unsigned)cdiv64(M * D, 1024), 256, 0, to>>>(b.part, (bf16*)y_MD, M * D, b.slices);
  return launch_status();
}
