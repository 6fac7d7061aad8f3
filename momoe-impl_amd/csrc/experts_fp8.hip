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
  int64_t msum;
};

constexpr int kFewRows = 32, kFewChunk = 16;  // rows of a tile, blocks of the contraction whose rows are in LDS

// LDS of a chunk: [block][row][128], the 16-byte piece c of row r at position c ^ ((r / 2) % 8): the 16 rows x 16 bytes that 16 lanes
// read cover all banks.
__device__ __forceinline__ int row_piece_at(int r, int c) { return r * kFp8Block + ((c ^ ((r >> 1) & 7)) << 4); }

template <int ROWS>
__device__ __forceinline__ i32x8 row_frag(const uint8_t* block, int i) {
  const int l = threadIdx.x & 63, r = 16 * i + (l & 15), g = l >> 4;
  const u32x4 lo = *(const u32x4*)(block + row_piece_at(r, g)), hi = *(const u32x4*)(block + row_piece_at(r, 4 + g));
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
__device__ __forceinline__ i32x8 weight_frag(const uint8_t* at) {
  const uint32_t l = fresh_lane();  // (an offset beside a uniform address; hoisted, the sum takes registers of its own)
  const u32x4 lo = *(const u32x4*)(at + l * 16), hi = *(const u32x4*)(at + (l * 16 + 1024));
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// A row's columns 32 * pair + 4 * (lane / 16) .. +3 and those 16 further on, times s
__device__ __forceinline__ void store_packet(const Fp8Args& p, int64_t row, int pair, int l, const f32x4& a, const f32x4& b, float s) {
  const float v[8] = {a[0] * s, a[1] * s, a[2] * s, a[3] * s, b[0] * s, b[1] * s, b[2] * s, b[3] * s};
  *(u32x4*)(p.out + row * p.D + 32 * pair + 8 * (l >> 4)) = Packet::of(v).w;
}

// the largest of the four lanes that hold a row
__device__ __forceinline__ uint32_t top_of_rows(uint32_t v) {
  const auto larger = [](auto pair) { return (uint32_t)max((uint32_t)pair[0], (uint32_t)pair[1]); };
  v = larger(__builtin_amdgcn_permlane16_swap(v, v, false, false));
  return larger(__builtin_amdgcn_permlane32_swap(v, v, false, false));
}

// Tiles of up to 32 rows: a wavefront owns a pair of 16-column groups (of the first product one of each half) and streams
// their weights; the rows of the tile lie in LDS.
template <bool FIRST>
__global__ __launch_bounds__(kThreads) void fp8_few_rows_kernel(Fp8Args p) {
  constexpr int FR = kFewRows / 16;
  __shared__ __attribute__((aligned(16))) uint8_t rows_lds[kFewChunk * kFewRows * kFp8Block];
  __shared__ float scale_lds[kFewChunk][kFewRows];
  __shared__ uint32_t top_lds[kWaves][kFewRows];
  const int tid = threadIdx.x, l = tid & 63, wave = wave_id();
  TileSchedT<1> sched(p.table, (p.pairs + kWaves - 1) / kWaves, kFewRows);
  for (TileCoord tc = sched.next(); tc.valid; tc = sched.next()) {
    const int pair = min(tc.tn * kWaves + wave, p.pairs - 1);
    const bool real = tc.tn * kWaves + wave < p.pairs;
    const uint8_t* const w0 = p.w + ((int64_t)tc.expert * p.pairs + pair) * 2 * p.KB * kFp8Frag;
    const uint8_t* const w1 = w0 + (int64_t)p.KB * kFp8Frag;
    f32x4 acc[2][FR] = {};
    for (int k0 = 0; k0 < p.KB; k0 += kFewChunk) {
      const int blocks = min(kFewChunk, p.KB - k0);
      __syncthreads();
      for (int q = tid; q < blocks * kFewRows * 8; q += kThreads) {
        const int c = q & 7, r = (q >> 3) % kFewRows, kb = q / (8 * kFewRows);
        const int row = tc.row0 + min(r, tc.rows - 1);
        const int64_t src = FIRST ? p.idx[row] : row;
        *(u32x4*)(rows_lds + kb * (kFewRows * kFp8Block) + row_piece_at(r, c)) =
            *(const u32x4*)(p.rows + (src * p.KB + k0 + kb) * kFp8Block + c * 16);
      }
      for (int q = tid; q < blocks * kFewRows; q += kThreads) {
        const int r = q % kFewRows, kb = q / kFewRows, row = tc.row0 + min(r, tc.rows - 1);
        const int64_t src = FIRST ? p.idx[row] : row;
        scale_lds[kb][r] = scale_of_code(p.codes[src * fp8_code_bytes(p.KB) + k0 + kb]);
      }
      __syncthreads();
      for (int kb = 0; kb < blocks; ++kb) {
        const int k = k0 + kb;
        const i32x8 wq[2] = {weight_frag(w0 + (int64_t)k * kFp8Frag), weight_frag(w1 + (int64_t)k * kFp8Frag)};
        bf16x8 wf[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int m = 0; m < 4; ++m) wf[j][m] = bf16_of_e4m3(wq[j][2 * m], wq[j][2 * m + 1], 1.0f);
        float ws[2];
        if (FIRST) {
          const float* at = p.w_scale + ((int64_t)tc.expert * p.KB + k) * 2 * p.HB + pair / 8;
          ws[0] = load_uniform(at);
          ws[1] = load_uniform(at + p.HB);
        } else {
          ws[0] = ws[1] = load_uniform(p.w_scale + ((int64_t)tc.expert * p.KB + k) * p.DB + pair / 4);
        }
#pragma unroll
        for (int i = 0; i < FR; ++i) {
          const i32x8 rq = row_frag<kFewRows>(rows_lds + kb * (kFewRows * kFp8Block), i);
          const float rs = scale_lds[kb][16 * i + (l & 15)];
          f32x4 t[2] = {};
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const bf16x8 rf = bf16_of_e4m3(rq[2 * m], rq[2 * m + 1], rs);
#pragma unroll
            for (int j = 0; j < 2; ++j) t[j] = mfma16(wf[j][m], rf, t[j]);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(t[j][r], ws[j], acc[j][i][r]);
        }
      }
    }
    if (FIRST) {
      // h of 16 columns in each wavefront; the eight of a workgroup hold a block of 128
      f32x4 h[FR];
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        uint32_t top = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          h[i][r] = real ? acc[0][i][r] * acc[1][i][r] * sigmoidf_fast(acc[1][i][r]) : 0.0f;
          top = max(top, magnitude(h[i][r]));
        }
        top = top_of_rows(top);
        if (l < 16) top_lds[wave][16 * i + l] = top;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        const int r = 16 * i + (l & 15);
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = max(top, top_lds[w][r]);
        const RowScale s(top);
        if (r < tc.rows) {
          const int64_t row = tc.row0 + r;
          *(uint32_t*)(p.hq + (row * p.HB + tc.tn) * kFp8Block + wave * 16 + 4 * (l >> 4)) =
              pack_e4m3(h[i][0] * s.inverse, h[i][1] * s.inverse, h[i][2] * s.inverse, h[i][3] * s.inverse);
          if (wave == 0 && l < 16) p.h_codes[row * fp8_code_bytes(p.HB) + tc.tn] = (uint8_t)s.code;
        }
      }
    } else if (real) {
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        const int r = 16 * i + (l & 15);
        if (r >= tc.rows) continue;
        const int64_t row = tc.row0 + r;
        const float s = p.s[tc.expert * p.sn + p.idx[row] * p.sm];
        store_packet(p, row, pair, l, acc[0][i], acc[1][i], s);
      }
    }
  }
}

// Tiles of up to 256 rows x 256 columns, a workgroup on a CU.  Each of its eight wavefronts owns 32 columns of all rows: it reads
// their weights straight into registers, each byte once per workgroup, a stage of 128 k-values ahead and more; the rows of a stage
// come to LDS by direct transfers, a stage ahead, in two slots.
constexpr int kTileRows = 256, kTileChunk = 64;  // blocks of the contraction whose scales are held at a time
constexpr int kTileSlot = kTileRows * kFp8Block;
constexpr int kCodePitch = kTileChunk / 4 + 1;   // dwords; odd: sixteen rows read different banks
constexpr int kTileLds = 2 * kTileSlot + kTileRows * kCodePitch * 4 + kWaves * kTileRows * 4;

// `v` is in its registers here: what it is made of lies before this point, what it goes into behind it.  (Without, the compiler
// forms all products of a stage first and keeps them.)
template <class T>
__device__ __forceinline__ void keep(T& v) {
  asm volatile("" : "+v"(v));
}

template <bool FIRST>
struct TileRows {
  static constexpr int DEP = kTileRows / (8 * kWaves);  // transfers of 8 rows each
  const uint8_t* base;
  uint32_t off[DEP];
  __device__ __forceinline__ void init(const Fp8Args& p, const TileCoord& tc) {
    const int l = threadIdx.x & 63;
    base = FIRST ? p.rows : p.rows + (int64_t)tc.row0 * p.KB * kFp8Block;
#pragma unroll
    for (int j = 0; j < DEP; ++j) {
      const int r = (j * kWaves + wave_id()) * 8 + (l >> 3), have = min(r, tc.rows - 1);
      const uint32_t src = FIRST ? p.idx[tc.row0 + have] : have;
      off[j] = src * (uint32_t)(p.KB * kFp8Block) + (((l & 7) ^ ((r >> 1) & 7)) << 4);
    }
  }
  __device__ __forceinline__ void request(int kb, uint32_t slot) const {
    const bf16* const b = (const bf16*)(base + (int64_t)kb * kFp8Block);
#pragma unroll
    for (int j = 0; j < DEP; ++j) dma16(b, off[j], slot + (j * kWaves + wave_id()) * 1024);
  }
};

template <bool FIRST>
__global__ __launch_bounds__(kThreads, 2) void fp8_tile_kernel(Fp8Args p) {
  uint8_t* const lds = (uint8_t*)dyn_lds();
  uint32_t* const codes_lds = (uint32_t*)(lds + 2 * kTileSlot);
  uint32_t* const top_lds = codes_lds + kTileRows * kCodePitch;  // [wave][row]
  float* const gate_lds = (float*)top_lds;  // of the second product
  const uint32_t addr = lds_address(dyn_lds());
  const int tid = threadIdx.x, l = tid & 63, wave = wave_id();
  const int code_bytes = fp8_code_bytes(p.KB);
  TileSchedT<1> sched(p.table, (p.pairs + kWaves - 1) / kWaves, kTileRows);
  for (TileCoord tc = sched.next(); tc.valid; tc = sched.next()) {
    const int pair = min(tc.tn * kWaves + wave, p.pairs - 1);
    const bool real = tc.tn * kWaves + wave < p.pairs;
    const uint8_t* const w0 = p.w + ((int64_t)tc.expert * p.pairs + pair) * 2 * p.KB * kFp8Frag;
    const uint8_t* const w1 = w0 + (int64_t)p.KB * kFp8Frag;
    TileRows<FIRST> rows;
    rows.init(p, tc);
    static_assert(2 * kTileRows == kThreads, "two threads a row");
    const int my_row = tc.row0 + min(tid >> 1, tc.rows - 1), code_row = FIRST ? p.idx[my_row] : my_row;
    if (!FIRST) {
      __syncthreads();
      gate_lds[tid >> 1] = p.s[tc.expert * p.sn + p.idx[my_row] * p.sm];
    }

    const auto tile = [&](auto NAC) {
      constexpr int NA = decltype(NAC)::value;
      f32x4 acc[2][NA];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < NA; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int k0 = 0; k0 < p.KB; k0 += kTileChunk) {
        const int blocks = min(kTileChunk, p.KB - k0);
        __syncthreads();
        rows.request(k0, addr);
        // the scales of the chunk: the rows' in LDS, a row's by two threads, the weights' of block k0 + lane in a lane
        {
          constexpr int EACH = kTileChunk / 8;
          const uint32_t* const from = (const uint32_t*)(p.codes + (int64_t)code_row * code_bytes + k0);
          const int d0 = (tid & 1) * EACH, have = (blocks + 3) / 4;
          uint32_t v[EACH];
#pragma unroll
          for (int d = 0; d < EACH; ++d) v[d] = from[min(d0 + d, have - 1)];
#pragma unroll
          for (int d = 0; d < EACH; ++d) codes_lds[(tid >> 1) * kCodePitch + d0 + d] = v[d];
        }
        float ws[2];
        {
          const int64_t k = (int64_t)tc.expert * p.KB + k0 + min(l, blocks - 1);
          ws[0] = FIRST ? p.w_scale[k * 2 * p.HB + pair / 8] : p.w_scale[k * p.DB + pair / 4];
          ws[1] = FIRST ? p.w_scale[k * 2 * p.HB + p.HB + pair / 8] : ws[0];
        }
        i32x8 wf[2][2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int64_t at = (int64_t)(k0 + min(b, blocks - 1)) * kFp8Frag;
          wf[b][0] = weight_frag(w0 + at);
          wf[b][1] = weight_frag(w1 + at);
        }
        wait_vmcnt<0>();
        __syncthreads();
        const uint32_t* const my_codes = codes_lds + (l & 15) * kCodePitch;
        const auto stage = [&](auto BYTE, int kb) {
          constexpr int byte = decltype(BYTE)::value, b = byte & 1;
          if (kb > 0) {
            // this stage's weights and rows have landed (what was requested after them: the weights of the next stage), for all
            wait_vmcnt<4>();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
          }
          keep(wf[b][0]);
          keep(wf[b][1]);
          if (kb + 1 < blocks) rows.request(k0 + kb + 1, addr + (b ^ 1) * kTileSlot);
          const float s0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ws[0]), kb));
          const float s1 = FIRST ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ws[1]), kb)) : s0;
          const uint8_t* const slot = lds + b * kTileSlot;
          // row fragment i + 1 is on its way and the results of i - 1 are added while i is multiplied
          i32x8 rf[2];
          int codes[2];  // the four blocks' scales of the rows
          f32x4 t[2][2];
          int quad = kb / 4;
          asm volatile("" : "+s"(quad));  // (read anew in each stage: kept, they were spilled)
          rf[0] = row_frag<kTileRows>(slot, 0);
          codes[0] = my_codes[quad];
          order_fence();
          unrolled<0, NA>([&](auto IC) {
            constexpr int i = decltype(IC)::value, c = i & 1;
            keep(rf[c]);
            if constexpr (i + 1 < NA) {
              rf[c ^ 1] = row_frag<kTileRows>(slot, i + 1);
              codes[c ^ 1] = my_codes[16 * (i + 1) * kCodePitch + quad];
            }
            t[c][0] = mfma_e4m3<byte>(wf[b][0], rf[c], codes[c]);
            t[c][1] = mfma_e4m3<byte>(wf[b][1], rf[c], codes[c]);
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
          });
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[0][NA - 1][r] = fmaf(t[(NA - 1) & 1][0][r], s0, acc[0][NA - 1][r]);
            acc[1][NA - 1][r] = fmaf(t[(NA - 1) & 1][1][r], s1, acc[1][NA - 1][r]);
          }
          const int64_t at = (int64_t)(k0 + min(kb + 2, blocks - 1)) * kFp8Frag;
          wf[b][0] = weight_frag(w0 + at);
          wf[b][1] = weight_frag(w1 + at);
        };
        // whole fours apart from the rest: behind a stage that may not run, the compiler waits for all that is on its way
        int kb = 0;
#pragma unroll 1
        for (; kb + 4 <= blocks; kb += 4) {
          stage(IntC<0>{}, kb);
          stage(IntC<1>{}, kb + 1);
          stage(IntC<2>{}, kb + 2);
          stage(IntC<3>{}, kb + 3);
        }
        if (kb < blocks) {
          stage(IntC<0>{}, kb);
          if (kb + 1 < blocks) stage(IntC<1>{}, kb + 1);
          if (kb + 2 < blocks) stage(IntC<2>{}, kb + 2);
        }
      }
      const int l = fresh_lane();
      if constexpr (FIRST) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          uint32_t top = 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[0][i][r] = real ? acc[0][i][r] * acc[1][i][r] * sigmoidf_fast(acc[1][i][r]) : 0.0f;
            top = max(top, magnitude(acc[0][i][r]));
          }
          top = top_of_rows(top);
          if (l < 16) top_lds[wave * kTileRows + 16 * i + l] = top;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const int r = 16 * i + (l & 15);
          uint32_t top = 0;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) top = max(top, top_lds[w * kTileRows + r]);
          const RowScale s(top);
          if (r < tc.rows) {
            const int64_t row = tc.row0 + r;
            *(uint32_t*)(p.hq + (row * p.HB + tc.tn) * kFp8Block + wave * 16 + 4 * (l >> 4)) =
                pack_e4m3(acc[0][i][0] * s.inverse, acc[0][i][1] * s.inverse, acc[0][i][2] * s.inverse, acc[0][i][3] * s.inverse);
            if (wave == 0 && l < 16) p.h_codes[row * fp8_code_bytes(p.HB) + tc.tn] = (uint8_t)s.code;
          }
        }
      } else if (real) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const int r = 16 * i + (l & 15);
          if (r >= tc.rows) continue;
          const int64_t row = tc.row0 + r;
          const float s = gate_lds[r];
          store_packet(p, row, pair, l, acc[0][i], acc[1][i], s);
        }
      }
    };
    const int quads = __builtin_amdgcn_readfirstlane((tc.rows + 63) >> 6);
    if (quads == 4) tile(IntC<16>{});
    else if (quads == 3) tile(IntC<12>{});
    else if (quads == 2) tile(IntC<8>{});
    else tile(IntC<4>{});
  }
}

// out[m] = the sum of its experts' rows, in fp32, in the order of the experts: packet 4 p + g of a row holds columns 32 p + 4 g .. +3
// and 32 p + 16 + 4 g .. +3.  Bound by HBM, as momoe_combine, whose loads it has.
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

// Whether a launch takes tiles of 256 rows: from an average of 48 rows an expert on (PROVISIONAL)
bool takes_tiles(int64_t Msum, int64_t N) { return Msum >= 48 * N; }

int check_fp8(int64_t M, int64_t D, int64_t H, int64_t N, int64_t Msum) {
  if (M <= 0 || D <= 0 || H <= 0 || N <= 0 || Msum <= 0) return MOMOE_ERR_BAD_ARG;
  if (D % 32 != 0 || H % 32 != 0 || Msum >= (1ll << 31) || M >= (1ll << 31) || D >= (1 << 22) || H >= (1 << 22))
    return MOMOE_ERR_UNSUPPORTED;
  return MOMOE_OK;
}
template <bool FIRST>
int launch_fp8(const Fp8Args& a, int64_t M, int64_t Msum, int64_t N, hipStream_t st) {
  if (!takes_tiles(Msum, N)) {
    fp8_few_rows_kernel<FIRST><<<2 * persistent_grid(), kThreads, 0, st>>>(a);
    return launch_status();
  }
  // the rows of the first product are gathered at 32-bit offsets
  if (FIRST && M * a.KB * kFp8Block >= (1ll << 32)) return MOMOE_ERR_UNSUPPORTED;
  static LdsLimit limit;
  if (!allow_lds(fp8_tile_kernel<FIRST>, kTileLds, limit)) return MOMOE_ERR_LAUNCH;
  fp8_tile_kernel<FIRST><<<persistent_grid(), kThreads, kTileLds, st>>>(a);
  return launch_status();
}
bool unaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }

}  // namespace
}  // namespace momoe

using namespace momoe;

extern "C" int momoe_fp8_tile_rows(int64_t Msum, int64_t N) {
  return Msum <= 0 || N <= 0 ? 0 : takes_tiles(Msum, N) ? kTileRows : kFewRows;
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
  a.msum = Msum;
  return launch_fp8<true>(a, M, Msum, N, (hipStream_t)stream);
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
  a.msum = Msum;
  return launch_fp8<false>(a, M, Msum, N, (hipStream_t)stream);
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
