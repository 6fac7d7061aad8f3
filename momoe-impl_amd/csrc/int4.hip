// SwiGLU blocks with weights in 4 bits, forward only: the experts of a mixture, or one dense block.
//
// A weight is (code - zero) * scale: a code of 4 bits, a zero (0 to 15) and a 16-bit scale for each `group` (32, 64, 128) consecutive
// k-values of a column.  A product over a group is
//   sum_k x_k (code_k - zero) scale = scale * (sum_k x_k (128 + code_k) - (128 + zero) * sum_k x_k)
// 128 + code is a bf16 whose low bits are the code: bits 0x4300 | code, one instruction for two of them and no conversion.  The sum of
// x_k is a product with ones by the same matrix instruction, whose rate such a call does not use up; it comes in the same lanes.  All
// of it in fp32: what is subtracted is up to 143 / 8 times as large as what is left, so that four bits of 24 go.  The scale, fp32 again,
// meets the sum: a weight itself is never rounded.
//
// Kept in the order in which a wavefront holds them as the second input of v_mfma_f32_16x16x32_bf16 (column lane % 16, k-values
// 8 * (lane / 16) .. +7):
//   codes   [expert][16 columns][128 k-values]: 1024 bytes = [64 lanes][4 words], word m the k-values 32 m + 8 * (lane / 16) .. +7 of
//           column lane % 16; k-value 2 i in bits 4 i .. +3, 2 i + 1 in bits 16 + 4 i .. +3, so that a shift and a mask give a pair
//   scales  [expert][16 columns][128 k-values][16][128 / group] words: the scale's fp32 bits (of a 16-bit type: the low 13 are zero) and,
//           in the low four, the zero
// zeros past the last k-value.  The columns of the first product are those of its two halves in turn, 16 a and 16 b.
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
};

// eight codes of a word as 128 + code
__device__ __forceinline__ bf16x8 bf16_of_codes(uint32_t w) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
  return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ float scale_of_word(uint32_t w) { return __uint_as_float(w & ~15u); }
__device__ __forceinline__ float zero_of_word(uint32_t w) { return __uint_as_float(0x43000000u | (w & 15u) << 16); }  // 128 + zero

// Tiles of experts, by the index build's table, or of a dense block, which has none: all rows are those of one expert
struct Int4Sched {
  TileSchedT<1> experts;
  int nb, total, pos, tile_rows, rows;
  // (of a dense block `experts` reads the first two words of the codes, and nothing is made of them)
  __device__ __forceinline__ Int4Sched(const Int4Args& p, int nb_, int tile_rows_)
      : experts(p.table ? p.table : (const int32_t*)p.w, nb_, tile_rows_), nb(nb_), pos(blockIdx.x), tile_rows(tile_rows_), rows(p.M) {
    total = (rows + tile_rows - 1) / tile_rows * nb;
  }
  __device__ __forceinline__ TileCoord next() {
    if (rows == 0) return experts.next();
    TileCoord t = {};
    t.valid = pos < total;
    if (!t.valid) return t;
    t.row0 = pos / nb * tile_rows;
    t.tn = pos % nb;
    t.rows = min(tile_rows, rows - t.row0);
    pos += gridDim.x;
    return t;
  }
};

// Tiles of up to 16 FR rows.  A wavefront owns a pair of 16-column groups; KS of them share its contraction, a block of 128 k-values in
// KS each, and their sums meet in LDS.  Codes and scales go straight into registers, AHEAD blocks ahead; the rows come to LDS,
// kFewBytes of them at a time, for all wavefronts.
constexpr int kFewThreads = 256, kFewWaves = kFewThreads / 64, kFewBytes = 64 << 10;

template <bool FIRST, int FR, int KS, int SG>
__global__ __launch_bounds__(kFewThreads, 2) void int4_few_rows_kernel(Int4Args p) {
  constexpr int ROWS = 16 * FR, PW = kFewWaves / KS, CHUNK = kFewBytes / (ROWS * kInt4Block * 2);
  constexpr int AHEAD = FR * SG >= 16 ? 2 : 4;  // (four of the smallest groups' scales and 64 rows' sums were spilled)
  __shared__ __attribute__((aligned(16))) uint8_t lds[kFewBytes];  // rows [block][row][256], then the sums of KS wavefronts
  static_assert(kFewWaves * 64 * 2 * FR * 16 <= kFewBytes, "sums of all wavefronts");
  typedef uint32_t Words __attribute__((ext_vector_type(SG)));
  const int tid = threadIdx.x, l = tid & 63, wave = wave_id(), kw = wave % KS, cw = wave / KS;
  Int4Sched sched(p, (p.pairs + PW - 1) / PW, ROWS);
  const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
  for (TileCoord tc = sched.next(); tc.valid; tc = sched.next()) {
    const int pair = min(tc.tn * PW + cw, p.pairs - 1);
    const bool real = tc.tn * PW + cw < p.pairs;
    const int nf = (tc.rows + 15) >> 4;
    const int64_t group = ((int64_t)tc.expert * p.pairs + pair) * 2 * p.KB;
    const uint8_t* const w0 = p.w + group * kInt4Frag + l * 16;
    const uint32_t* const s0 = p.scale + (group * 16 + (l & 15)) * SG;
    f32x4 acc[2][FR] = {};
    for (int k0 = 0; k0 < p.KB; k0 += CHUNK) {
      const int blocks = min(CHUNK, p.KB - k0), steps = (blocks - kw + KS - 1) / KS;  // (none for a wavefront past the last)
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
      // banks.  (What is left in LDS for rows that the tile does not have goes into rows that nobody stores.)
      const int all = blocks * tc.rows * 16;
      for (int q0 = tid; q0 < all; q0 += 2 * kFewThreads) {
        bf16x8 v[2];
        int to[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const int q = min(q0 + a * kFewThreads, all - 1), piece = q & 15, kb = (q >> 4) / tc.rows, r = (q >> 4) - kb * tc.rows;
          const int c = (k0 + kb) * kInt4Block + piece * 8, row = tc.row0 + r;
          v[a] = *(const bf16x8*)(p.rows + (int64_t)(FIRST && p.idx ? p.idx[row] : row) * p.ld + min(c, p.K - 8));
          if (c >= p.K) v[a] = bf16x8{};
          to[a] = (kb * ROWS + r) * 256 + ((piece ^ (r & 15)) << 4);
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
          for (int m = 0; m < 4; ++m) wf[j][m] = bf16_of_codes(wq[q][j][m]);
        unrolled<0, FR>([&](auto IC) {
          constexpr int i = decltype(IC)::value;
          if (i >= nf) return;  // (the same for all lanes)
          const uint8_t* const from = lds + (kb * ROWS + 16 * i + (l & 15)) * 256;
          bf16x8 rf[4];
#pragma unroll
          for (int m = 0; m < 4; ++m) rf[m] = *(const bf16x8*)(from + (((4 * m + (l >> 4)) ^ (l & 15)) << 4));
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
        if constexpr (FIRST) {
          const float a = acc[0][i][r], b = acc[1][i][r];
          ((bf16*)p.out)[row * p.ldo + 16 * pair + (l & 15)] = f2bf(a * b * sigmoidf_fast(b));
        } else {
          const int64_t to = row * p.ldo + 32 * pair + (l & 15);
          if (p.idx) {
            const float s = p.s[(int64_t)tc.expert * p.sn + (int64_t)p.idx[row] * p.sm];
            ((float*)p.out)[to] = acc[0][i][r] * s;
            ((float*)p.out)[to + 16] = acc[1][i][r] * s;
          } else {
            ((bf16*)p.out)[to] = f2bf(acc[0][i][r]);
            ((bf16*)p.out)[to + 16] = f2bf(acc[1][i][r]);
          }
        }
      }
  }
}

// out[m] = the sum of the rows of its experts, fp32, rounded once.  The row numbers and then the rows with unconditional loads, as in
// combine_kernel.
__global__ __launch_bounds__(256) void int4_combine_kernel(const float* __restrict__ rows, const int32_t* __restrict__ inv,
                                                           bf16* __restrict__ out, int D, int K, int64_t msum) {
  const int64_t m = blockIdx.x;
  for (int c = threadIdx.x; c < D / 4; c += blockDim.x) {
    f32x4 sum = {};
    for (int k0 = 0; k0 < K; k0 += 8) {
      int32_t r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = inv[m * K + min(k0 + j, K - 1)];
      f32x4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool ok = k0 + j < K && (uint32_t)r[j] < (uint64_t)msum;
        v[j] = *(const f32x4*)(rows + (int64_t)(ok ? r[j] : 0) * D + c * 4);
        r[j] = ok ? 1 : 0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += r[j] ? v[j][e] : 0.0f;
    }
    *(bf16x4*)(out + m * D + c * 4) = pack_bf16x4(sum[0], sum[1], sum[2], sum[3]);
  }
}

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
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;  // [N][groups][KB][64][4]
  if (q >= p.N * groups * KB * 256) return;
  const int m = q & 3, l = (int)(q >> 2) & 63;
  const int64_t f = q >> 8;
  const int kb = (int)(f % KB), g = (int)(f / KB % groups);
  const int64_t e = f / KB / groups;
  const int k = kb * kInt4Block + 32 * m + 8 * (l >> 4), col = column_of(p, g, l & 15);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (k + 2 * i >= p.R) break;
    const uint32_t b = p.w[(e * (p.R / 2) + k / 2 + i) * C + col];
    word |= (b & 15u) << (4 * i) | (b >> 4) << (16 + 4 * i);
  }
  p.codes[q] = word;
}

__global__ __launch_bounds__(256) void int4_pack_scales_kernel(Int4PackArgs p) {
  const int KB = (int)int4_blocks(p.R), C = p.cols * p.halves, groups = C / 16, SG = kInt4Block / p.group;
  const int KG = (p.R + p.group - 1) / p.group;
  const int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x;  // [N][groups][KB][16][SG]
  if (q >= p.N * groups * KB * 16 * SG) return;
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

int check_int4(int64_t M, int64_t D, int64_t H, int64_t N, int64_t Msum, int group) {
  if (M <= 0 || D <= 0 || H <= 0 || N <= 0 || Msum <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || H % 32 != 0 || Msum >= (1ll << 31) - 512 || M >= (1ll << 31) - 512 || D >= (1 << 22) || H >= (1 << 22))
    return MOMOE_ERR_UNSUPPORTED;
  return group == 32 || group == 64 || group == 128 ? MOMOE_OK : MOMOE_ERR_UNSUPPORTED;
}
bool unaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }

template <bool FIRST, int FR, int SG>
int launch_few(const Int4Args& a, int64_t tiles, hipStream_t st) {
  const int64_t wanted = 2 * persistent_grid();
  const auto enough = [&](int ks) { return a.KB < 2 * ks || tiles * cdiv64(a.pairs, kFewWaves / ks) >= wanted; };
  auto kernel = enough(1) ? int4_few_rows_kernel<FIRST, FR, 1, SG> : enough(2) ? int4_few_rows_kernel<FIRST, FR, 2, SG>
                                                                              : int4_few_rows_kernel<FIRST, FR, 4, SG>;
  kernel<<<(unsigned)wanted, kFewThreads, 0, st>>>(a);
  return launch_status();
}
// `tiles` of `tile_rows` rows (32 or 64)
template <bool FIRST>
int launch_few(const Int4Args& a, int64_t tiles, int tile_rows, int group, hipStream_t st) {
  if (tile_rows == 32)
    return group == 128 ? launch_few<FIRST, 2, 1>(a, tiles, st) : group == 64 ? launch_few<FIRST, 2, 2>(a, tiles, st) : launch_few<FIRST, 2, 4>(a, tiles, st);
  return group == 128 ? launch_few<FIRST, 4, 1>(a, tiles, st) : group == 64 ? launch_few<FIRST, 4, 2>(a, tiles, st) : launch_few<FIRST, 4, 4>(a, tiles, st);
}
template <bool FIRST>
int launch_experts(const Int4Args& a, int64_t N, int64_t Msum, int tile_rows, int group, hipStream_t st) {
  // a tile for each expert that may hold a row; more where the rows fill more than that
  return launch_few<FIRST>(a, std::max(std::min(N, Msum), Msum / tile_rows), tile_rows, group, st);
}
template <bool FIRST>
int launch_dense(const Int4Args& a, int group, hipStream_t st) {
  const int tile_rows = a.M <= 32 ? 32 : 64;
  return launch_few<FIRST>(a, cdiv64(a.M, tile_rows), tile_rows, group, st);
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
  if (nwords < 0 || bytes / 1024 >= (1ll << 31) || nwords / 256 >= (1ll << 31) - 1) return MOMOE_ERR_UNSUPPORTED;
  const Int4PackArgs a{(const uint8_t*)codes_NRC, scale, (const uint8_t*)zero, N, (int)R, (int)(C / halves), halves, group,
                       scale_type == MOMOE_TYPE_F16, (uint32_t*)packed, (uint32_t*)words};
  int4_pack_codes_kernel<<<(unsigned)(bytes / 1024), 256, 0, (hipStream_t)stream>>>(a);
  int4_pack_scales_kernel<<<(unsigned)cdiv64(nwords, 256), 256, 0, (hipStream_t)stream>>>(a);
  return launch_status();
}

extern "C" int momoe_int4_tile_rows(int64_t Msum, int64_t N) {
  return Msum <= 0 || N <= 0 ? 0 : Msum >= 20 * N ? 64 : 32;
}

extern "C" int momoe_int4_lin1_swiglu_fwd(const void* x_MD, int64_t ldx, const void* Wl1_packed, const void* Wl1_words, int group,
                                          const int32_t* idx_Msum, const int32_t* tile_table, int tile_rows, void* h_MsumH, int64_t M,
                                          int64_t D, int64_t H, int64_t N, int64_t Msum, void* stream) {
  if (!x_MD || !Wl1_packed || !Wl1_words || !idx_Msum || !tile_table || !h_MsumH || ldx < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_int4(M, D, H, N, Msum, group);
  if (st != MOMOE_OK) return st;
  if (unaligned16(x_MD) || unaligned16(Wl1_packed) || unaligned16(Wl1_words) || unaligned16(h_MsumH)) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0 || (tile_rows != 32 && tile_rows != 64)) return MOMOE_ERR_UNSUPPORTED;
  Int4Args a{(const bf16*)x_MD, ldx, (const uint8_t*)Wl1_packed, (const uint32_t*)Wl1_words, idx_Msum, tile_table, 0, (int)D,
             (int)int4_blocks(D), (int)(H / 16)};
  a.out = h_MsumH;
  a.ldo = H;
  return launch_experts<true>(a, N, Msum, tile_rows, group, (hipStream_t)stream);
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
  return launch_experts<false>(a, N, Msum, tile_rows, group, (hipStream_t)stream);
}

extern "C" int momoe_int4_combine(const float* ys_MsumD, const int32_t* inv_MK, void* out_MD, int64_t M, int64_t D, int64_t K, int64_t Msum,
                                  void* stream) {
  if (!ys_MsumD || !inv_MK || !out_MD || M <= 0 || D <= 0 || K <= 0 || Msum <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || M >= (1ll << 31) || Msum >= (1ll << 31)) return MOMOE_ERR_UNSUPPORTED;
  if (unaligned16(ys_MsumD) || unaligned16(out_MD)) return MOMOE_ERR_BAD_ARG;
  int4_combine_kernel<<<(unsigned)M, 256, 0, (hipStream_t)stream>>>(ys_MsumD, inv_MK, (bf16*)out_MD, (int)D, (int)K, Msum);
  return launch_status();
}

extern "C" int momoe_int4_ffn_fwd(const void* x_MD, int64_t ldx, const void* Wl1_packed, const void* Wl1_words, const void* Wl2_packed,
                                  const void* Wl2_words, int group, void* h_MH, void* y_MD, int64_t M, int64_t D, int64_t H, void* stream) {
  if (!x_MD || !Wl1_packed || !Wl1_words || !Wl2_packed || !Wl2_words || !h_MH || !y_MD || ldx < D) return MOMOE_ERR_BAD_ARG;
  int st = check_int4(M, D, H, 1, M, group);
  if (st != MOMOE_OK) return st;
  for (const void* q : {x_MD, Wl1_packed, Wl1_words, Wl2_packed, Wl2_words, (const void*)h_MH, (const void*)y_MD})
    if (unaligned16(q)) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0) return MOMOE_ERR_UNSUPPORTED;
  Int4Args a{(const bf16*)x_MD, ldx, (const uint8_t*)Wl1_packed, (const uint32_t*)Wl1_words, nullptr, nullptr, (int)M, (int)D,
             (int)int4_blocks(D), (int)(H / 16)};
  a.out = h_MH;
  a.ldo = H;
  st = launch_dense<true>(a, group, (hipStream_t)stream);
  if (st != MOMOE_OK) return st;
  Int4Args b{(const bf16*)h_MH, H, (const uint8_t*)Wl2_packed, (const uint32_t*)Wl2_words, nullptr, nullptr, (int)M, (int)H,
             (int)int4_blocks(H), (int)(D / 32)};
  b.out = y_MD;
  b.ldo = D;
  return launch_dense<false>(b, group, (hipStream_t)stream);
}
