// The experts in 8-bit floating point, for serving: h = a * b * sigmoid(b) with a | b = x . Wl1, and (h . Wl2) scaled by the gate
// weight, both products of e4m3 rows and e4m3 weights with a scale for each block of 128 (fp8.hpp):
//   sum over the blocks kb of (scale of the row's block * scale of the weights' block) * (sum of the 128 products),
// the inner sum by one v_mfma_f32_16x16x128_f8f6f4 from a zero accumulator, the outer one in fp32 by one multiply-add for each of its
// results.
//
// The MFMA's first input is the weight-side fragment (16 columns), its second the row-side one (16 rows): a lane holds, for one
// row (lane % 16), columns 4 * (lane / 16) .. +3, so that a row's scale and what is done with its result stay in the lane.
#include "fp8.hpp"
#include "gemm_span.hpp"

namespace momoe {
namespace {

struct Fp8Args {
  const uint8_t* rows;     // e4m3 [M or Msum][KB * 128]
  const uint8_t* codes;    // [M or Msum][KB rounded up to 4]
  const uint8_t* w;        // fragments
  const float* w_scale;
  const int32_t* idx;
  const int32_t* table;
  int KB, pairs;           // blocks of the contraction; pairs of 16-column groups
  // first product
  uint8_t* hq;             // [Msum][HB * 128]
  uint8_t* h_codes;        // [Msum][HB rounded up to 4]
  int HB;
  // second product
  const float* s;
  int64_t sn, sm;
  uint16_t* out;           // [Msum][D / 8] packets
  int D, DB;
};

// LDS of a block's rows: [row][128], the 16-byte piece c of row r at position c ^ ((r / 2) % 8): the 16 rows x 16 bytes that 16 lanes
// of a fragment read cover all banks.
__device__ __forceinline__ int row_piece_at(int r, int c) { return r * kFp8Block + ((c ^ ((r >> 1) & 7)) << 4); }

// row fragment i of a block, lane l
__device__ __forceinline__ i32x8 row_frag(const uint8_t* block, int l, int i) {
  const int r = 16 * i + (l & 15), g = l >> 4;
  const u32x4 lo = *(const u32x4*)(block + row_piece_at(r, g)), hi = *(const u32x4*)(block + row_piece_at(r, 4 + g));
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
template <bool ONCE>
__device__ __forceinline__ i32x8 weight_frag(const uint8_t* at) {
  const uint32_t l = fresh_lane();  // (an offset beside a uniform address; hoisted, the sum takes registers of its own)
  const u32x4 lo = load_maybe_once<ONCE>((const u32x4*)(at + l * 16)), hi = load_maybe_once<ONCE>((const u32x4*)(at + (l * 16 + 1024)));
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// a * b * sigmoid(b)
__device__ __forceinline__ f32x4 swiglu(const f32x4& a, const f32x4& b) {
  f32x4 h;
#pragma unroll
  for (int r = 0; r < 4; ++r) h[r] = a[r] * b[r] * sigmoidf_fast(b[r]);
  return h;
}

// Tiles of up to 32 rows: launches that stream their weights.  A wavefront multiplies a pair of 16-column groups (of the first product
// one of each half), their weights straight into registers, kFewAhead blocks of 128 k-values ahead.  KS wavefronts share a pair's
// contraction, a block in KS each, and their sums meet in LDS: one token has few columns to spread over the CUs.  The tile's rows
// are brought to 8 bits by the workgroup that multiplies them, which has the first weights on their way meanwhile: a few rows read
// again for each block of columns, against a launch before either product.
//
// Products in bf16 (fp8.hpp): the conversions and the slower products hide behind the stream.  Bound by HBM: of 128 experts of
// 2048 x 768, one row each, x . Wl1 64 us, 6.3 TB/s, h . Wl2 30 us, 6.6 TB/s; 19 rows each 72 and 37.  Two workgroups share a CU, so
// that one streams while the other starts or ends a tile: with four blocks ahead, the registers of which leave room for one, it is
// 63 and 37, at 19 rows 78 and 48.  One token, 8 experts: 11 and 6 us, of which the weights alone are 4 and 2: its chain of table, token,
// row, product and sum.  Two rows at a time are as fast as four; each wavefront's blocks in another order, against all of them
// at the same place of a row's stretch, changed nothing.
constexpr int kFewRows = MOMOE_FP8_FEW_ROWS, kFewChunk = 16, kFewAhead = 2, kRowsAtOnce = 2;

struct FewArgs {
  const void* rows;      // [M or Msum][ld]
  int64_t ld;
  const uint8_t* w;
  const float* w_scale;
  const int32_t *idx, *table;
  int K, KB, pairs;      // contraction, its blocks; pairs of 16-column groups
  float* h;              // first product: [Msum][H]
  int H, HB;
  const float* s;        // second product
  int64_t sn, sm;
  uint16_t* out;         // [Msum][D / 8] packets
  int D, DB;
};

template <bool FIRST, bool ONCE, class X, int KS>
__global__ __launch_bounds__(kThreads, 4) void fp8_few_rows_kernel(FewArgs p) {
  constexpr int FR = kFewRows / 16, PW = kWaves / KS;
  __shared__ __attribute__((aligned(16))) uint8_t rows_lds[kFewChunk * kFewRows * kFp8Block];  // then the sums of KS wavefronts
  __shared__ float scale_lds[kFewChunk][kFewRows];
  static_assert(kWaves * 64 * 4 * FR * 2 * 4 <= (int)sizeof(rows_lds), "16 sums a lane");
  const int tid = threadIdx.x, l = tid & 63, wave = wave_id(), kw = wave % KS, cw = wave / KS;
  TileSchedT<1> sched(p.table, (p.pairs + PW - 1) / PW, kFewRows);
  for (TileCoord tc = sched.next(); tc.valid; tc = sched.next()) {
    const int pair = min(tc.tn * PW + cw, p.pairs - 1);
    const bool real = tc.tn * PW + cw < p.pairs, two = tc.rows > 16;
    const uint8_t* const w0 = p.w + ((int64_t)tc.expert * p.pairs + pair) * 2 * p.KB * kFp8Frag;
    const uint8_t* const w1 = w0 + (int64_t)p.KB * kFp8Frag;
    f32x4 acc[2][FR] = {};
    for (int k0 = 0; k0 < p.KB; k0 += kFewChunk) {
      const int blocks = min(kFewChunk, p.KB - k0), steps = (blocks - kw + KS - 1) / KS;  // (none for a wavefront past the last)
      i32x8 wq[kFewAhead][2];
      const auto load = [&](int q, int step) {
        const int64_t at = (int64_t)(k0 + step * KS + kw) * kFp8Frag;
        wq[q][0] = weight_frag<ONCE>(w0 + at);
        wq[q][1] = weight_frag<ONCE>(w1 + at);
      };
      unrolled<0, kFewAhead>([&](auto QC) {
        if (decltype(QC)::value < steps) load(decltype(QC)::value, decltype(QC)::value);
      });
      // the weights' scales, of block k0 + lane in a lane
      float ws[2];
      {
        const int64_t k = (int64_t)tc.expert * p.KB + k0 + min(l, blocks - 1);
        ws[0] = FIRST ? p.w_scale[k * 2 * p.HB + pair / 8] : p.w_scale[k * p.DB + pair / 4];
        ws[1] = FIRST ? p.w_scale[k * 2 * p.HB + p.HB + pair / 8] : ws[0];
      }
      __syncthreads();  // (the last rows, or sums, are done with)
      // sixteen lanes a block of a row.  (What is left in LDS for rows that the tile does not have meets columns that nobody reads.)
      const int all = blocks * tc.rows;
      for (int q0 = tid >> 4; q0 < all; q0 += kRowsAtOnce * (kThreads / 16)) {
        float v[kRowsAtOnce][8];
        const auto place = [&](int a, int& r, int& kb) {
          const int q = min(q0 + a * (kThreads / 16), all - 1);
          kb = q / tc.rows;
          r = q - kb * tc.rows;
          return (k0 + kb) * kFp8Block + (l & 15) * 8;
        };
#pragma unroll
        for (int a = 0; a < kRowsAtOnce; ++a) {
          int r, kb;
          const int c = place(a, r, kb), row = tc.row0 + r;
          load8((const X*)p.rows + (int64_t)(FIRST ? p.idx[row] : row) * p.ld + min(c, p.K - 8), v[a]);
        }
#pragma unroll
        for (int a = 0; a < kRowsAtOnce; ++a) {
          int r, kb;
          const int c = place(a, r, kb);
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[a][e] = c < p.K ? v[a][e] : 0.0f;
            top = max(top, magnitude(v[a][e]));
          }
          const RowScale s(__float_as_uint(over_lanes<16>(__uint_as_float(top), LargerBits{})));
          *(u32x2*)(rows_lds + kb * (kFewRows * kFp8Block) + row_piece_at(r, (l & 15) >> 1) + (l & 1) * 8) =
              u32x2{pack_e4m3(v[a][0], v[a][1], v[a][2], v[a][3], s.scale), pack_e4m3(v[a][4], v[a][5], v[a][6], v[a][7], s.scale)};
          if ((l & 15) == 0) scale_lds[kb][r] = scale_of_code(s.code);
        }
      }
      __syncthreads();
      const auto multiply = [&](int q, int step) {
        const int kb = step * KS + kw;
        const float s0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ws[0]), kb));
        const float s1 = FIRST ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ws[1]), kb)) : s0;
        bf16x8 wf[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int m = 0; m < 4; ++m) wf[j][m] = bf16_of_e4m3(wq[q][j][2 * m], wq[q][j][2 * m + 1], 1.0f);
        unrolled<0, FR>([&](auto IC) {
          constexpr int i = decltype(IC)::value;
          if (i > 0 && !two) return;  // (wave-uniform)
          const i32x8 rq = row_frag(rows_lds + kb * (kFewRows * kFp8Block), l, i);
          const float rs = scale_lds[kb][16 * i + (l & 15)];
          f32x4 t[2] = {};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const bf16x8 rf = bf16_of_e4m3(rq[2 * m], rq[2 * m + 1], rs);
#pragma unroll
            for (int j = 0; j < 2; ++j) t[j] = mfma16(wf[j][m], rf, t[j]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[0][i][r] = fmaf(t[0][r], s0, acc[0][i][r]);
            acc[1][i][r] = fmaf(t[1][r], s1, acc[1][i][r]);
          }
        });
      };
      // what is multiplied last has nothing to request: apart, as behind a request that may not be made the compiler waits for all
      int step = 0;
#pragma unroll 1
      for (; step + 2 * kFewAhead <= steps; step += kFewAhead)
        unrolled<0, kFewAhead>([&](auto QC) {
          constexpr int q = decltype(QC)::value;
          multiply(q, step + q);
          load(q, step + q + kFewAhead);
        });
      unrolled<0, kFewAhead>([&](auto QC) {
        constexpr int q = decltype(QC)::value;
        if (step + q < steps) multiply(q, step + q);
        if (step + q + kFewAhead < steps) load(q, step + q + kFewAhead);
      });
      unrolled<0, kFewAhead>([&](auto QC) {
        constexpr int q = decltype(QC)::value;
        if (step + q + kFewAhead < steps) multiply(q, step + q + kFewAhead);
      });
    }
    if constexpr (KS > 1) {
      __syncthreads();
      f32x4* const sums = (f32x4*)rows_lds + wave * (2 * FR) * 64 + l;
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
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const int r = 16 * i + (l & 15);
      if (r >= tc.rows) continue;
      const int64_t row = tc.row0 + r;
      if (FIRST)
        *(f32x4*)(p.h + row * p.H + 16 * pair + 4 * (l >> 4)) = swiglu(acc[0][i], acc[1][i]);
      else
        *(u32x4*)(p.out + row * p.D + 32 * pair + 8 * (l >> 4)) = Packet::of(acc[0][i], acc[1][i], p.s[tc.expert * p.sn + p.idx[row] * p.sm]).w;
    }
  }
}

// Tiles of up to 256 rows x 256 columns, a persistent workgroup on a CU.  Each of its eight wavefronts owns 32 columns of all rows: it
// reads their weights straight into registers, each byte once per workgroup; the rows come to LDS by direct transfers.  Both are
// requested two stages of 128 k-values ahead, in three slots of LDS and two register sets, and the last two stages of a tile
// request the first two of the next one.
//
// A stage: the fragments of 16 rows travel from LDS one ahead of the products, the fp32 sums follow one behind them.  Its barrier lies
// behind the first rows, not at its end: by then the next stage's rows have landed for every wavefront, and the slot of the
// last one is free.
//
// Bound by the issue of what is not a product, and by the clock.  8192 tokens, 2048 x 768, 8 of 128 experts: x . Wl1 235 to 265 us (1.6 to
// 1.75 PFLOP/s), h . Wl2 165 to 177.  A stage takes 3400 clocks, of which the 64 matrix instructions of a SIMD's two wavefronts
// are some 2050; the fp32 sums are part of the rest (without them 209 and 146 us).  The clock is 1.78 GHz under this data: with zeros the same
// takes 216 and 146.  A tile's end (h, its largest, packing; packets of 15 bits) is 10 to 18 thousand clocks with no product beside
// it: in h . Wl2, whose six stages are 20 thousand, a third to nearly half of the tile.  A library's plain product of 8192^3 reaches 2.98
// PFLOP/s, with neither block scales nor such an end.  Two wavefronts of a SIMD half a stage apart: 274 to 277 and 180.  128 rows x 64
// columns a wavefront, half the reads of LDS: 306 and 256, with spills.
constexpr int kTileRows = 256, kTileBlocks = 64;  // most blocks of a contraction
constexpr int kTileSlot = kTileRows * kFp8Block, kSlots = 3;
constexpr int kTileCodes = kTileRows * kTileBlocks;  // bytes: [four blocks][row][block]
constexpr int kTileLds = kSlots * kTileSlot + 2 * kTileCodes + 2 * kTileRows * 4 + 4 * kTileBlocks * 4 + kTileRows * 4;

// `v` is in its registers here: what it is made of lies before this point, what it goes into behind it.  (Without, the compiler
// forms all products of a stage first and keeps them.)
template <class T>
__device__ __forceinline__ void keep(T& v) {
  asm volatile("" : "+v"(v));
}
// a value that is the same in every lane, as one that the compiler knows to be
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <class T>
__device__ __forceinline__ const T* uniform(const T* p) {
  const uint64_t v = (uint64_t)p;
  return (const T*)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}
// 4 bytes per lane, global -> LDS, as dma16: at a uniform base and an offset, or anywhere
__device__ __forceinline__ void dma4(const void* from, uint32_t lds_wave_base) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(__builtin_amdgcn_readfirstlane(lds_wave_base)) : "memory");
}
__device__ __forceinline__ void dma4(const void* uniform_base, uint32_t byte_offset, uint32_t lds_wave_base) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(byte_offset), "s"(uniform_base),
               "s"(__builtin_amdgcn_readfirstlane(lds_wave_base))
               : "memory");
}
// wavefronts meet: what they have read from or written to LDS is done with, what they have on the way stays there
__device__ __forceinline__ void meet() {
  wait_lgkm0();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// memory that stores at offsets of `bytes` and more do not reach
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)uniform((const char*)p), 0, uniform(bytes), 0x00027000);
}

// The rows of a tile, as a wavefront requests them
template <bool FIRST>
struct TileRows {
  static constexpr int DEP = kTileRows / (8 * kWaves);  // transfers of 8 rows each
  const uint8_t* base;
  uint32_t off[DEP];
  // `idx`: the tokens of the tile's rows (of the first product, whose rows are gathered)
  __device__ __forceinline__ void place(const Fp8Args& p, const TileCoord& tc, const int32_t* idx) {
    const int l = fresh_lane();
    base = FIRST ? p.rows : p.rows + (int64_t)uniform(tc.row0) * p.KB * kFp8Block;
#pragma unroll
    for (int j = 0; j < DEP; ++j) {
      const int r = (j * kWaves + wave_id()) * 8 + (l >> 3);
      const uint32_t src = FIRST ? idx[r] : min(r, tc.rows - 1);
      off[j] = src * (uint32_t)(p.KB * kFp8Block) + (((l & 7) ^ ((r >> 1) & 7)) << 4);
    }
  }
  __device__ __forceinline__ void request(int kb, uint32_t slot) const {
    const bf16* const b = uniform((const bf16*)(base + (int64_t)kb * kFp8Block));
#pragma unroll
    for (int j = 0; j < DEP; ++j) dma16(b, off[j], slot + (j * kWaves + wave_id()) * 1024);
  }
};

template <bool FIRST, bool ONCE>
__global__ __launch_bounds__(kThreads, 2) void fp8_tile_kernel(Fp8Args p) {
  uint8_t* const lds = (uint8_t*)dyn_lds();
  uint8_t* const codes_lds = lds + kSlots * kTileSlot;
  uint32_t* const top_lds = (uint32_t*)(codes_lds + 2 * kTileCodes);  // [2][row]
  float* const gate_lds = (float*)top_lds;                            // of the second product: [2][row]
  float* const scales_lds = (float*)(top_lds + 2 * kTileRows);        // [2][set][block]
  int32_t* const tokens_lds = (int32_t*)(scales_lds + 4 * kTileBlocks);
  const uint32_t addr = lds_address(dyn_lds()), codes_addr = addr + kSlots * kTileSlot, gates_addr = codes_addr + 2 * kTileCodes;
  const uint32_t scales_addr = gates_addr + 2 * kTileRows * 4, tokens_addr = scales_addr + 4 * kTileBlocks * 4;
  const int wave = wave_id(), stages = max(p.KB, 2), code_bytes = fp8_code_bytes(p.KB);
  TileSchedT<1> sched(p.table, (p.pairs + kWaves - 1) / kWaves, kTileRows);
  TileCoord cur = sched.next();
  if (!cur.valid) return;

  const auto pair_of = [&](const TileCoord& tc) { return min(tc.tn * kWaves + wave, p.pairs - 1); };
  const auto weights_of = [&](const TileCoord& tc) { return p.w + ((int64_t)tc.expert * p.pairs + pair_of(tc)) * 2 * p.KB * kFp8Frag; };
  // The scales of a tile's weights, block by block, one set of two a wavefront (and again by others): of the two halves; of the two
  // blocks of columns
  const auto request_weight_scales = [&](const TileCoord& tc, int to) {
    const int set = wave & 1, k = min(fresh_lane(), p.KB - 1);
    const float* const base = p.w_scale + (int64_t)uniform(tc.expert) * p.KB * (FIRST ? 2 * p.HB : p.DB) +
                              (FIRST ? set * p.HB + uniform(tc.tn) : min(2 * uniform(tc.tn) + set, p.DB - 1));
    dma4(uniform(base), k * (FIRST ? 2 * p.HB : p.DB) * 4, scales_addr + (2 * to + set) * (kTileBlocks * 4));
  };
  // the tokens of a tile's rows, the last one's for those that it does not have: 64 of them a wavefront, and again by another one
  const auto request_tokens = [&](const TileCoord& tc) {
    const int q = wave & 3, have = min(q * 64 + fresh_lane(), tc.rows - 1);
    dma4(uniform(p.idx + tc.row0), have * 4, tokens_addr + q * 256);
  };
  // The codes of its rows: four blocks of 64 rows a transfer, as many transfers in every wavefront
  const int dwords = code_bytes / 4;
  const auto request_codes = [&](const TileCoord& tc, int to) {
    const uint8_t* const base = FIRST ? p.codes : p.codes + (int64_t)uniform(tc.row0) * code_bytes;
    const int q = wave & 3, r = q * 64 + fresh_lane();
    const uint32_t src = FIRST ? tokens_lds[r] : min(r, tc.rows - 1);
    for (int n = 0; n < dwords; n += 2) {
      const int d = min(n + wave / 4, dwords - 1);
      dma4(uniform(base + 4 * d), src * (uint32_t)code_bytes, codes_addr + to * kTileCodes + (d * kTileRows + q * 64) * 4);
    }
  };
  // the gate weights of its rows
  const auto request_gates = [&](const TileCoord& tc, int to) {
    const int q = wave & 3;
    dma4(p.s + (tc.expert * p.sn + tokens_lds[q * 64 + fresh_lane()] * p.sm), gates_addr + (to * kTileRows + q * 64) * 4);
  };

  // the first tile's requests
  i32x8 wf[2][2];
  TileRows<FIRST> rows;
  request_tokens(cur);
  wait_vmcnt<0>();
  meet();
  rows.place(p, cur, tokens_lds);
  rows.request(0, addr);
  rows.request(min(1, p.KB - 1), addr + kTileSlot);
  request_codes(cur, 0);
  const uint8_t* w = weights_of(cur);
  const auto weights = [&](i32x8 (&set)[2], int kb) {
    set[0] = weight_frag<ONCE>(w + (int64_t)kb * kFp8Frag);
    set[1] = weight_frag<ONCE>(w + (int64_t)(p.KB + kb) * kFp8Frag);
  };
  weights(wf[0], 0);
  weights(wf[1], min(1, p.KB - 1));
  request_weight_scales(cur, 0);
  if (!FIRST) request_gates(cur, 0);
  wait_vmcnt<0>();
  meet();

  uint32_t slot = 0, slot2 = 2 * kTileSlot;  // of the stage at hand, of the one two further on: byte offsets
  int buffer = 0;                            // of the codes and gate weights
  while (true) {
    TileCoord nxt = sched.next();
    const bool last = !nxt.valid;
    if (last) nxt = cur;  // (requested again for nothing)
    request_tokens(nxt);
    // the largest of each row's values so far, for this tile's epilogue (the other buffer may still be read in the last one's)
    if (FIRST) top_lds[buffer * kTileRows + wave * 32 + (fresh_lane() & 31)] = 0;

    const auto tile = [&](auto NAC) {
      constexpr int NA = decltype(NAC)::value;
      f32x4 acc[2][NA];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < NA; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      const int end = stages - 2;
      // Stage kb with register set B.  (The last two, which request the next tile's first ones, are not code of their own: apart, they
      // cost the register allocation of the whole loop.)
      const auto stage = [&](auto BC, int kb) {
        constexpr int b = decltype(BC)::value;
        if (kb == end) {  // `rows` and `w` are the next tile's from here on
          if (end <= 1) {  // (later stages have met behind a wait of their own: the tokens are there)
            wait_vmcnt<0>();
            meet();
          }
          rows.place(p, nxt, tokens_lds);
          w = weights_of(nxt);
        }
        const int rk = min(kb < end ? kb + 2 : kb - end, p.KB - 1);
        keep(wf[b][0]);
        keep(wf[b][1]);
        const int kc = min(kb, p.KB - 1);
        // (a stage past the last block, where there is but one, counts for nothing)
        const int live = kb < p.KB ? -1 : 0;
        const float* const ws = scales_lds + 2 * buffer * kTileBlocks + kc;
        const float s0 = __int_as_float(uniform(__float_as_int(ws[FIRST ? 0 : (wave >> 2) * kTileBlocks])) & live);
        const float s1 = FIRST ? __int_as_float(uniform(__float_as_int(ws[kTileBlocks])) & live) : s0;
        const int l = fresh_lane();
        const uint8_t* const at = lds + slot;
        const uint8_t* const my_codes = codes_lds + buffer * kTileCodes + (kc >> 2) * (kTileRows * 4) + (kc & 3) + (l & 15) * 4;
        i32x8 rf[2];
        int codes[2];
        f32x4 t[2][2];
        rf[0] = row_frag(at, l, 0);
        codes[0] = my_codes[0];
        order_fence();
        unrolled<0, NA>([&](auto IC) {
          constexpr int i = decltype(IC)::value, c = i & 1;
          keep(rf[c]);
          if constexpr (i + 1 < NA) {
            rf[c ^ 1] = row_frag(at, l, i + 1);
            codes[c ^ 1] = my_codes[64 * (i + 1)];
          }
          t[c][0] = mfma_e4m3<0>(wf[b][0], rf[c], codes[c]);
          t[c][1] = mfma_e4m3<0>(wf[b][1], rf[c], codes[c]);
          order_fence();
          if constexpr (i > 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              acc[0][i - 1][r] = fmaf(t[c ^ 1][0][r], s0, acc[0][i - 1][r]);
              acc[1][i - 1][r] = fmaf(t[c ^ 1][1][r], s1, acc[1][i - 1][r]);
            }
            keep(acc[0][i - 1]);
            keep(acc[1][i - 1]);
          }
          order_fence();
          if constexpr (i == 1) {
            // the rows of the next stage have landed (younger than they: its weights; of a tile's second stage they had
            // before the last epilogue); every wavefront is past the stage before, whose slot the requests go to
            if (kb > 0) wait_vmcnt<4>();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            rows.request(rk, addr + slot2);
            if (kb == end) {
              request_codes(nxt, buffer ^ 1);
              request_weight_scales(nxt, buffer ^ 1);
              if (!FIRST) request_gates(nxt, buffer ^ 1);
            }
            order_fence();
          }
        });
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          acc[0][NA - 1][r] = fmaf(t[(NA - 1) & 1][0][r], s0, acc[0][NA - 1][r]);
          acc[1][NA - 1][r] = fmaf(t[(NA - 1) & 1][1][r], s1, acc[1][NA - 1][r]);
        }
        weights(wf[b], rk);
        slot2 = slot;  // (free behind the next stage's barrier)
        slot = slot == (kSlots - 1) * kTileSlot ? 0 : slot + kTileSlot;
        order_fence();
      };
      int kb = 0;
#pragma unroll 1
      for (; kb + 2 <= stages; kb += 2) {
        stage(IntC<0>{}, kb);
        stage(IntC<1>{}, kb + 1);
      }
      if (kb < stages) stage(IntC<0>{}, kb);
      wait_vmcnt<4>();  // the rows of the next tile's second stage
      order_fence();

      // Stores go at offsets from the tile's first row, and those past its last one are dropped.
      const int l = fresh_lane(), r0 = l & 15, pair = cur.tn * kWaves + wave;
      if constexpr (FIRST) {
        uint32_t* const top = top_lds + buffer * kTileRows + r0;
        if (pair >= p.pairs) {  // columns past the last: zeros, up to a whole block
#pragma unroll
          for (int i = 0; i < NA; ++i) acc[0][i] = acc[1][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          acc[0][i] = swiglu(acc[0][i], acc[1][i]);
          __hip_atomic_fetch_max(top + 16 * i, largest(acc[0][i][0], acc[0][i][1], acc[0][i][2], acc[0][i][3]), __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        meet();
        const int row_bytes = p.HB * kFp8Block, code_row = fp8_code_bytes(p.HB);
        const __amdgpu_buffer_rsrc_t h = buffer_of(p.hq + (int64_t)cur.row0 * row_bytes, cur.rows * row_bytes);
        const __amdgpu_buffer_rsrc_t codes = buffer_of(p.h_codes + (int64_t)cur.row0 * code_row, wave == 0 ? cur.rows * code_row : 0);
        int at = r0 * row_bytes + cur.tn * kFp8Block + wave * 16 + 4 * (l >> 4), code_at = r0 * code_row + cur.tn;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const RowScale s(top[16 * i]);
          __builtin_amdgcn_raw_buffer_store_b32(pack_e4m3(acc[0][i][0], acc[0][i][1], acc[0][i][2], acc[0][i][3], s.scale), h, at, 0, 0);
          __builtin_amdgcn_raw_buffer_store_b8((uint8_t)s.code, codes, code_at, 0, 0);  // (the four lanes of a row the same)
          at += 16 * row_bytes;
          code_at += 16 * code_row;
        }
      } else {
        const __amdgpu_buffer_rsrc_t out = buffer_of(p.out + (int64_t)cur.row0 * p.D, pair < p.pairs ? cur.rows * p.D * 2 : 0);
        int at = r0 * p.D * 2 + pair * 64 + 16 * (l >> 4);
        const float* const gate = gate_lds + buffer * kTileRows + r0;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          __builtin_amdgcn_raw_buffer_store_b128(Packet::of(acc[0][i], acc[1][i], gate[16 * i]).w, out, at, 0, 0);
          at += 16 * p.D * 2;
        }
        meet();  // (of two stages, the next tile's first one requests codes where this tile's have been read)
      }
    };
    const int quads = __builtin_amdgcn_readfirstlane((cur.rows + 63) >> 6);
    if (quads == 4) tile(IntC<16>{});
    else if (quads == 3) tile(IntC<12>{});
    else if (quads == 2) tile(IntC<8>{});
    else tile(IntC<4>{});
    if (last) break;
    if (stages & 1) {  // the register sets have changed places
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const i32x8 other = wf[0][j];
        wf[0][j] = wf[1][j];
        wf[1][j] = other;
      }
    }
    buffer ^= 1;
    cur = nxt;
  }
  wait_vmcnt<0>();  // nothing is on its way to LDS when the workgroup ends
}

// out[m] = the sum of its experts' rows, in fp32, in the order of the experts: packet 4 p + g of a row holds columns 32 p + 4 g .. +3
// and 32 p + 16 + 4 g .. +3.  Bound by HBM, as momoe_combine, whose loads it has: 8192 x 8 rows of 2048 in 47 us, 6.4 TB/s.
template <bool ONCE>
__global__ __launch_bounds__(256) void fp8_combine_kernel(const u32x4* __restrict__ packets, const int32_t* __restrict__ inv,
                                                          bf16* __restrict__ out, int D, int K, int64_t msum) {
  const int64_t m = blockIdx.x;
  for (int c = threadIdx.x; c < D / 8; c += blockDim.x) {
    float sum[8] = {};
    for (int k0 = 0; k0 < K; k0 += 8) {
      int32_t r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = inv[m * K + min(k0 + j, K - 1)];
      Packet v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool ok = k0 + j < K && (uint32_t)r[j] < (uint64_t)msum;
        v[j].w = load_maybe_once<ONCE>(packets + (int64_t)(ok ? r[j] : 0) * (D / 8) + c);
        r[j] = ok ? 1 : 0;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (r[j]) v[j].add_to(sum);
    }
    bf16x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = (bf16)sum[e];
      hi[e] = (bf16)sum[4 + e];
    }
    bf16* const at = out + m * D + 32 * (c >> 2) + 4 * (c & 3);
    *(bf16x4*)at = lo;
    *(bf16x4*)(at + 16) = hi;
  }
}

// Whether both products take tiles of 256 rows: from an average of 20 rows an expert on, and for contractions of up to kTileBlocks
// blocks.  Both products of 128 experts of 2048 x 768 at 8, 16, 25, 32 rows each: 111, 116, 115, 114 us by tiles of 256 rows, and 4 for
// bringing the rows to 8 bits before; 98, 106, 117, 123 by tiles of 32, and twice as much past 32 rows, which some experts hold before
// the average does.  8 experts of 1408 x 2048 at 20, 32 rows each: 31, 32 and 4 more; 33, 40.
bool takes_tiles(int64_t Msum, int64_t N, int64_t D, int64_t H) {
  return Msum >= 20 * N && std::max(D, H) <= kTileBlocks * kFp8Block;
}

int check_fp8(int64_t M, int64_t D, int64_t H, int64_t N, int64_t Msum) {
  if (M <= 0 || D <= 0 || H <= 0 || N <= 0 || Msum <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || H % 32 != 0 || Msum >= (1ll << 31) || M >= (1ll << 31) || D >= (1 << 22) || H >= (1 << 22))
    return MOMOE_ERR_UNSUPPORTED;
  return MOMOE_OK;
}
// Whether the weights, each read by one tile, go past the last-level cache: those that do not fit it.  With the hint | without, us between
// events, calls one behind the other.  128 experts of 2048 x 768, the first product's 384 MiB: 16 tokens 43 | 46, 131 69 | 75, 1000
// 80 | 85.  64 experts of 1024 x 768, which stay in the cache from call to call, 96 and 48 MiB: 16 tokens 19.0 | 18.8 and 13.4 | 12.8, 500 33.2 | 32.2
// and 21.5 | 18.4.  (In between, and where other layers' data pass through the cache before the next call, the hint would win
// below the line, too: the second product's 192 MiB of the 128 experts 26 | 28 at 16 tokens, 37 | 43 at 131, 58 | 59 at 1000.)
template <class A>
bool read_once(const A& a, int64_t Msum, int64_t N, int64_t tile_rows) {
  return Msum <= tile_rows * N && std::min(N, Msum) * a.pairs * 2 * a.KB * kFp8Frag >= kBeyondCache;
}

template <bool FIRST, bool ONCE>
int launch_tiles(const Fp8Args& a, hipStream_t st) {
  static LdsLimit limit;
  if (!allow_lds(fp8_tile_kernel<FIRST, ONCE>, kTileLds, limit)) return MOMOE_ERR_LAUNCH;
  fp8_tile_kernel<FIRST, ONCE><<<persistent_grid(), kThreads, kTileLds, st>>>(a);
  return launch_status();
}
template <bool FIRST>
int launch_tiles(const Fp8Args& a, int64_t M, int64_t D, int64_t H, int64_t N, int64_t Msum, hipStream_t st) {
  // the rows of the first product are gathered at 32-bit offsets
  if (std::max(D, H) > kTileBlocks * kFp8Block || (FIRST && M * a.KB * kFp8Block >= (1ll << 32))) return MOMOE_ERR_UNSUPPORTED;
  return read_once(a, Msum, N, kTileRows) ? launch_tiles<FIRST, true>(a, st) : launch_tiles<FIRST, false>(a, st);
}
// As many wavefronts to a pair's contraction as give every CU two workgroups, with as many tiles as there are at the least.  (Sharing
// it among more costs: each workgroup has fewer columns, and the rows are brought to 8 bits more often.  Many rows come here if the
// contraction is past 8192; with a tile counted for each expert only, 2000 tokens of 8224 x 2112, 3 of 12 experts, took 2600 us instead
// of 1470, 600 of 8224 x 1024, 2 of 8, 433 instead of 220.)
template <bool FIRST, bool ONCE, class X>
int launch_few(const FewArgs& a, int64_t tiles, hipStream_t st) {
  const int64_t wanted = 2 * persistent_grid();
  const auto enough = [&](int ks) { return a.KB < 2 * ks || tiles * cdiv64(a.pairs, kWaves / ks) >= wanted; };
  auto kernel = enough(1) ? fp8_few_rows_kernel<FIRST, ONCE, X, 1> : enough(2) ? fp8_few_rows_kernel<FIRST, ONCE, X, 2>
              : enough(4) ? fp8_few_rows_kernel<FIRST, ONCE, X, 4> : fp8_few_rows_kernel<FIRST, ONCE, X, 8>;
  kernel<<<(unsigned)wanted, kThreads, 0, st>>>(a);
  return launch_status();
}
template <bool FIRST, class X>
int launch_few(const FewArgs& a, int64_t Msum, int64_t N, hipStream_t st) {
  // a tile for each expert that may hold a row (one token's K experts); more where the rows fill more than that
  const int64_t tiles = std::max(std::min(N, Msum), Msum / kFewRows);
  return read_once(a, Msum, N, kFewRows) ? launch_few<FIRST, true, X>(a, tiles, st) : launch_few<FIRST, false, X>(a, tiles, st);
}
bool unaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }

}  // namespace
}  // namespace momoe

using namespace momoe;

extern "C" int momoe_fp8_tile_rows(int64_t Msum, int64_t D, int64_t H, int64_t N) {
  return Msum <= 0 || D <= 0 || H <= 0 || N <= 0 ? 0 : takes_tiles(Msum, N, D, H) ? kTileRows : kFewRows;
}

extern "C" int momoe_fp8_lin1_swiglu_fwd(const void* x_q, const void* x_codes, const void* Wl1_packed, const float* Wl1_scale,
                                         const int32_t* idx_Msum, const int32_t* tile_table, void* h_q, void* h_codes, int64_t M,
                                         int64_t D, int64_t H, int64_t N, int64_t Msum, void* stream) {
  if (!x_q || !x_codes || !Wl1_packed || !Wl1_scale || !idx_Msum || !tile_table || !h_q || !h_codes) return MOMOE_ERR_BAD_ARG;
  const int st = check_fp8(M, D, H, N, Msum);
  if (st != MOMOE_OK) return st;
  if (unaligned16(x_q) || unaligned16(Wl1_packed) || unaligned16(h_q) || (((uintptr_t)x_codes | (uintptr_t)h_codes) & 3)) return MOMOE_ERR_BAD_ARG;
  Fp8Args a{(const uint8_t*)x_q, (const uint8_t*)x_codes, (const uint8_t*)Wl1_packed, Wl1_scale, idx_Msum, tile_table, (int)fp8_blocks(D), (int)(H / 16)};
  a.hq = (uint8_t*)h_q;
  a.h_codes = (uint8_t*)h_codes;
  a.HB = (int)fp8_blocks(H);
  return launch_tiles<true>(a, M, D, H, N, Msum, (hipStream_t)stream);
}

extern "C" int momoe_fp8_lin2_scale_fwd(const void* h_q, const void* h_codes, const void* Wl2_packed, const float* Wl2_scale,
                                        const float* s_NM, int64_t s_stride_n, int64_t s_stride_m, const int32_t* idx_Msum,
                                        const int32_t* tile_table, void* ys_packets, int64_t M, int64_t D, int64_t H, int64_t N,
                                        int64_t Msum, void* stream) {
  if (!h_q || !h_codes || !Wl2_packed || !Wl2_scale || !s_NM || !idx_Msum || !tile_table || !ys_packets) return MOMOE_ERR_BAD_ARG;
  const int st = check_fp8(M, D, H, N, Msum);
  if (st != MOMOE_OK) return st;
  if (unaligned16(h_q) || unaligned16(Wl2_packed) || unaligned16(ys_packets) || ((uintptr_t)h_codes & 3)) return MOMOE_ERR_BAD_ARG;
  Fp8Args a{(const uint8_t*)h_q, (const uint8_t*)h_codes, (const uint8_t*)Wl2_packed, Wl2_scale, idx_Msum, tile_table, (int)fp8_blocks(H), (int)(D / 32)};
  a.s = s_NM;
  a.sn = s_stride_n;
  a.sm = s_stride_m;
  a.out = (uint16_t*)ys_packets;
  a.D = (int)D;
  a.DB = (int)fp8_blocks(D);
  return launch_tiles<false>(a, M, D, H, N, Msum, (hipStream_t)stream);
}

extern "C" int momoe_fp8_few_lin1_swiglu_fwd(const void* x, int type, int64_t ldx, const void* Wl1_packed, const float* Wl1_scale,
                                             const int32_t* idx_Msum, const int32_t* tile_table, float* h_MsumH, int64_t M,
                                             int64_t D, int64_t H, int64_t N, int64_t Msum, void* stream) {
  if (!x || !Wl1_packed || !Wl1_scale || !idx_Msum || !tile_table || !h_MsumH || ldx < D) return MOMOE_ERR_BAD_ARG;
  if (type != MOMOE_TYPE_BF16 && type != MOMOE_TYPE_F32 && type != MOMOE_TYPE_F16) return MOMOE_ERR_BAD_ARG;
  const int st = check_fp8(M, D, H, N, Msum);
  if (st != MOMOE_OK) return st;
  if (unaligned16(x) || unaligned16(Wl1_packed) || unaligned16(h_MsumH)) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0) return MOMOE_ERR_UNSUPPORTED;
  FewArgs a{x, ldx, (const uint8_t*)Wl1_packed, Wl1_scale, idx_Msum, tile_table, (int)D, (int)fp8_blocks(D), (int)(H / 16)};
  a.h = h_MsumH;
  a.H = (int)H;
  a.HB = (int)fp8_blocks(H);
  hipStream_t to = (hipStream_t)stream;
  return type == MOMOE_TYPE_BF16 ? launch_few<true, bf16>(a, Msum, N, to)
         : type == MOMOE_TYPE_F32 ? launch_few<true, float>(a, Msum, N, to) : launch_few<true, _Float16>(a, Msum, N, to);
}

extern "C" int momoe_fp8_few_lin2_scale_fwd(const float* h_MsumH, const void* Wl2_packed, const float* Wl2_scale, const float* s_NM,
                                            int64_t s_stride_n, int64_t s_stride_m, const int32_t* idx_Msum,
                                            const int32_t* tile_table, void* ys_packets, int64_t M, int64_t D, int64_t H,
                                            int64_t N, int64_t Msum, void* stream) {
  if (!h_MsumH || !Wl2_packed || !Wl2_scale || !s_NM || !idx_Msum || !tile_table || !ys_packets) return MOMOE_ERR_BAD_ARG;
  const int st = check_fp8(M, D, H, N, Msum);
  if (st != MOMOE_OK) return st;
  if (unaligned16(h_MsumH) || unaligned16(Wl2_packed) || unaligned16(ys_packets)) return MOMOE_ERR_BAD_ARG;
  FewArgs a{h_MsumH, H, (const uint8_t*)Wl2_packed, Wl2_scale, idx_Msum, tile_table, (int)H, (int)fp8_blocks(H), (int)(D / 32)};
  a.s = s_NM;
  a.sn = s_stride_n;
  a.sm = s_stride_m;
  a.out = (uint16_t*)ys_packets;
  a.D = (int)D;
  a.DB = (int)fp8_blocks(D);
  return launch_few<false, float>(a, Msum, N, (hipStream_t)stream);
}

extern "C" int momoe_fp8_combine(const void* ys_packets, const int32_t* inv_MK, void* out_MD, int64_t M, int64_t D, int64_t K,
                                 int64_t Msum, void* stream) {
  if (!ys_packets || !inv_MK || !out_MD || M <= 0 || D <= 0 || K <= 0 || Msum <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || M >= (1ll << 31) || Msum >= (1ll << 31)) return MOMOE_ERR_UNSUPPORTED;
  if (unaligned16(ys_packets) || unaligned16(out_MD)) return MOMOE_ERR_BAD_ARG;
  auto kernel = Msum * D * 2 >= kBeyondCache ? fp8_combine_kernel<true> : fp8_combine_kernel<false>;
  kernel<<<(unsigned)M, 256, 0, (hipStream_t)stream>>>((const u32x4*)ys_packets, inv_MK, (bf16*)out_MD, (int)D, (int)K, Msum);
  return launch_status();
}
