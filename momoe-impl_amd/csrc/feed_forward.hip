// A dense SwiGLU block, forward and backward: the layers beside the mixture that have no router.
//
//   a | b = x W1,  h = a b sig(b),  y = h W2
//   u = G_y W2^T,  G_a = u b sig(b),  G_b = u a sig(b) (1 + b (1 - sig(b))),
//   G_x = (G_a | G_b) W1^T,  G_W1 = x^T (G_a | G_b),  G_W2 = h^T G_y
//
// Rows are tokens as they come: no routing index, no gather, no gate weights, no sum over experts.  The products' operands are bf16;
// what meets in an epilogue is not rounded before: a | b that are kept for the backward, and u where a | b are made again, go through
// memory in fp32, as whole accumulator fragments ([row / 16][column / 16][64 lanes][4]: 1 KiB a store).  (In bf16 they cost half as much
// traffic and a rounding each, which doubles the error of the weight gradients.)
//   h       [H / 32][ldm][32]    k-blocked, as the second product contracts over it; of up to kTwiceRows rows each of them is two, bf16
//                                of it and of what that leaves, as a tile has room for both: rounded, the h of one token, few of which
//                                are large, can be more of y's error than y's own rounding (0.0023 to 0.0024 of the norm against 64
//                                bits, then 0.0017)
//   gz      [2H / 32][ldm][32]   G_a | G_b, k-blocked, for G_x and the gradient of W1; zeros behind the last row up to a multiple of 32
//   hT      [rows / 32][H][32]   h once more, feature-major in groups of 32 rows, zeros behind the last row: for the gradient of W2
// The weights' gradients are momoe_wgrad of one expert where their launches are large, and tiles of 128 x 128 where they are small.
#include <algorithm>
#include <type_traits>

#include "ffn_tile.hpp"

namespace momoe {
namespace {

constexpr int64_t kTwiceRows = 16;
int64_t rows_of_h(int64_t rows) { return rows <= kTwiceRows ? 2 * rows : rows; }

struct FfnArgs {
  const bf16* x;   // x, or G_y of the products with W2^T
  int64_t ldx;
  const bf16* w;   // W1 [D][2H] or W2 [H][D]
  int64_t rows;    // of this launch
  int64_t ldm;     // rows of the k-blocked matrices
  int D, H;
  bf16* h;         // k-blocked; read by the second product
  float* ab;       // fragments of a | b
  int64_t ab_rows; // rows that have them, a multiple of 32
  float* u;        // fragments of u
  bf16* gz;
  bf16* ht;
  bf16* out;       // y or G_x, row-major, D columns
  float* part;     // its sums by slices of the contraction, [slices][rows][D], where there are several
  int64_t total;   // tokens that a gradient of the weights is contracted over
  int slices = 1;
  bool twice = false;  // h W2 of rows that are two each: sums of both go to `part`
  int32_t* counts; // {0, all tokens}: what momoe_wgrad takes as the rows of its one expert
  unsigned long long* clk = clock_trace_buffer();
};

// fragment (row / 16, column / 16) of a matrix of `cols` columns, this lane's four values
__device__ __forceinline__ int64_t fragment_at(int64_t rf, int cf, int cols, int lane) {
  return ((rf * (cols >> 4) + cf) << 8) + lane * 4;
}

__device__ __forceinline__ float swiglu(float a, float b) { return a * b * sigmoidf_fast(b); }
struct SwigluGrad {
  float a, b, h;
  __device__ __forceinline__ SwigluGrad(float av, float bv, float u) {
    const float sg = sigmoidf_fast(bv), t = bv * sg;  // silu(b)
    h = av * t;
    a = u * t;
    b = (u * av) * silu_slope(bv, sg);
  }
};

// ---- small tiles --------------------------------------------------------------------------------------------------------------
template <int FM_>
struct FfnProg {
  static constexpr int FM = FM_;
  const FfnArgs& p;
  int K, slices, row_tiles, col_tiles;
  int64_t rows;
  __device__ __forceinline__ FfnProg(const FfnArgs& p_, int K_, int col_tiles_, int slices_ = 1)
      : p(p_), K(K_), slices(slices_), row_tiles((int)((p_.rows + 32 * FM - 1) / (32 * FM))), col_tiles(col_tiles_), rows(p_.rows) {}
  // rows as they come out of the accumulators
  __device__ __forceinline__ void store_rows_plain(int64_t row0, int rows_, int slice, int col0, f32x4 (&acc)[4][FM], int wm) const {
    const int l = lane_id();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = col0 + 16 * j + 4 * (l >> 4);
      if (col >= p.D) continue;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = 16 * (wm * FM + i) + (l & 15);
        if (r >= rows_) continue;
        if (slices > 1 || p.twice) *(f32x4*)(p.part + (slice * rows + row0 + r) * p.D + col) = acc[j][i];
        else *(bf16x4*)(p.out + (row0 + r) * p.D + col) = pack_bf16x4(acc[j][i], 1.0f);
      }
    }
  }
  // four columns of G_a, G_b and h of a row; `some`: it is one of the rows, and not of those that pad gz and hT
  __device__ __forceinline__ void store_grads(int64_t row, bool some, int col, const f32x4& a, const f32x4& b, const f32x4& u) const {
    bf16x4 va, vb;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const SwigluGrad g(a[e], b[e], u[e]);
      va[e] = f2bf(some ? g.a : 0.0f);
      vb[e] = f2bf(some ? g.b : 0.0f);
      if (p.ht) p.ht[((row >> 5) * p.H + col + e) * 32 + (row & 31)] = f2bf(some ? g.h : 0.0f);
    }
    *(bf16x4*)(p.gz + ((int64_t)(col >> 5) * p.ldm + row) * 32 + (col & 31)) = va;
    *(bf16x4*)(p.gz + ((int64_t)((p.H + col) >> 5) * p.ldm + row) * 32 + (col & 31)) = vb;
  }
};

// a | b = x W1: 64 columns of each half.  BWD: with u, into the gradients
template <int FM, bool BWD>
struct FfnLin1 : FfnProg<FM> {
  using Base = FfnProg<FM>;
  using Rows = FfnRows<32 * FM>;
  using Weights = FfnCols<true>;
  using Base::p;
  __device__ __forceinline__ explicit FfnLin1(const FfnArgs& p_) : Base(p_, p_.D, (p_.H + 63) / 64) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 32; }
  __device__ __forceinline__ void setup(int64_t row0, int rows, int tn, Rows& A, Weights& W) const {
    const int H = p.H, j0 = tn * 64;
    A.init(p.x, p.ldx, row0, rows, p.D);
    W.init(p.w, 2 * H, p.D, [&](int c) { return (c / 64) * H + min(j0 + c % 64, H - 8); });
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int slice, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    const int l = lane_id(), j0 = tn * 64 + wn * 32;
    if (j0 >= p.H) return;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r0 = 16 * (wm * FM + i), r = r0 + (l & 15);
      if (r0 >= (rows + 31 & ~31)) break;
      const int64_t row = row0 + r;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const f32x4 &a = acc[f][i], &b = acc[2 + f][i];
        const int col = j0 + 16 * f + 4 * (l >> 4);
        if constexpr (BWD) {
          f32x4 u = {};
          if (r0 < rows) u = *(const f32x4*)(p.u + fragment_at((row0 + r0) >> 4, (j0 >> 4) + f, p.H, l));
          Base::store_grads(row, r < rows, col, a, b, u);
        } else {
          if (r < rows) {
            const f32x4 h{swiglu(a[0], b[0]), swiglu(a[1], b[1]), swiglu(a[2], b[2]), swiglu(a[3], b[3])};
            bf16* const to = p.h + ((int64_t)(col >> 5) * p.ldm + row) * 32 + (col & 31);
            const bf16x4 first = pack_bf16x4(h, 1.0f);
            *(bf16x4*)to = first;
            if (p.rows <= kTwiceRows) {
              bf16x4 rest;
#pragma unroll
              for (int e = 0; e < 4; ++e) rest[e] = f2bf(rest_of(h[e], first[e]));
              *(bf16x4*)(to + p.rows * 32) = rest;
            }
          }
          if (row0 + r0 < p.ab_rows) {
            *(f32x4*)(p.ab + fragment_at((row0 + r0) >> 4, (j0 >> 4) + f, 2 * p.H, l)) = a;
            *(f32x4*)(p.ab + fragment_at((row0 + r0) >> 4, ((p.H + j0) >> 4) + f, 2 * p.H, l)) = b;
          }
        }
      }
    }
  }
};

// y = h W2
template <int FM>
struct FfnLin2 : FfnProg<FM> {
  using Base = FfnProg<FM>;
  using Rows = FfnBlockedRows<32 * FM>;
  using Weights = FfnCols<false>;
  using Base::p;
  __device__ __forceinline__ explicit FfnLin2(const FfnArgs& p_) : Base(p_, p_.H, (p_.D + kFfnCols - 1) / kFfnCols, p_.slices) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 64; }
  __device__ __forceinline__ void setup(int64_t row0, int rows, int tn, Rows& A, Weights& W) const {
    const int D = p.D, d0 = tn * kFfnCols;
    A.init(p.h, p.ldm, row0, rows, p.H);
    W.init(p.w, D, p.H, [&](int c) { return min(d0 + c, D - 8); });
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int slice, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    Base::store_rows_plain(row0, rows, slice, tn * kFfnCols + wn * 64, acc, wm);
  }
};

// u = G_y W2^T.  SAVED: with the a | b that were kept, into the gradients
template <int FM, bool SAVED>
struct FfnDh : FfnProg<FM> {
  using Base = FfnProg<FM>;
  using Rows = FfnRows<32 * FM>;
  using Weights = FfnWeightRows;
  using Base::p;
  __device__ __forceinline__ explicit FfnDh(const FfnArgs& p_) : Base(p_, p_.D, (p_.H + kFfnCols - 1) / kFfnCols) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 64; }
  __device__ __forceinline__ void setup(int64_t row0, int rows, int tn, Rows& A, Weights& W) const {
    A.init(p.x, p.ldx, row0, rows, p.D);
    W.init(p.w, p.D, tn * kFfnCols, p.H);
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int slice, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    const int l = lane_id(), j0 = tn * kFfnCols + wn * 64;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int r0 = 16 * (wm * FM + i), r = r0 + (l & 15);
      if (r0 >= (rows + 31 & ~31)) break;
      const int64_t row = row0 + r;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        if (j0 + 16 * f >= p.H) break;
        if constexpr (SAVED) {
          f32x4 a = {}, b = {};
          if (r0 < rows) {
            a = *(const f32x4*)(p.ab + fragment_at((row0 + r0) >> 4, (j0 >> 4) + f, 2 * p.H, l));
            b = *(const f32x4*)(p.ab + fragment_at((row0 + r0) >> 4, ((p.H + j0) >> 4) + f, 2 * p.H, l));
          }
          Base::store_grads(row, r < rows, j0 + 16 * f + 4 * (l >> 4), a, b, acc[f][i]);
        } else if (r0 < rows) {
          *(f32x4*)(p.u + fragment_at((row0 + r0) >> 4, (j0 >> 4) + f, p.H, l)) = acc[f][i];
        }
      }
    }
  }
};

// G_x = (G_a | G_b) W1^T
template <int FM>
struct FfnDx : FfnProg<FM> {
  using Base = FfnProg<FM>;
  using Rows = FfnBlockedRows<32 * FM>;
  using Weights = FfnWeightRows;
  using Base::p;
  __device__ __forceinline__ explicit FfnDx(const FfnArgs& p_) : Base(p_, 2 * p_.H, (p_.D + kFfnCols - 1) / kFfnCols, p_.slices) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 64; }
  __device__ __forceinline__ void setup(int64_t row0, int rows, int tn, Rows& A, Weights& W) const {
    A.init(p.gz, p.ldm, row0, rows, 2 * p.H);
    W.init(p.w, 2 * p.H, tn * kFfnCols, p.D);
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int slice, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    Base::store_rows_plain(row0, rows, slice, tn * kFfnCols + wn * 64, acc, wm);
  }
};

// Gradients of the weights, contracted over the tokens: W2 [H][D] from hT and G_y (the tokens of hT are padded with zeros, those of G_y
// repeat the last), W1 [D][2H] from x and gz (gz is padded).  p.D is the output's columns, p.out the gradient.
template <bool SECOND>
struct FfnWgrad {
  static constexpr int FM = 4;
  const FfnArgs& p;
  int K, slices, row_tiles, col_tiles;
  int64_t rows;
  using Rows = std::conditional_t<SECOND, FfnBlockedRows<128>, FfnTokenCols>;
  using Weights = FfnTokenCols;
  __device__ __forceinline__ explicit FfnWgrad(const FfnArgs& p_)
      : p(p_), K((int)((p_.total + 31) & ~31ll)), slices(p_.slices), row_tiles((int)((p_.rows + 127) / 128)),
        col_tiles((p_.D + kFfnCols - 1) / kFfnCols), rows(p_.rows) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 64; }
  __device__ __forceinline__ void setup(int64_t row0, int rows_, int tn, Rows& A, Weights& W) const {
    const int M = (int)p.total, y0 = tn * kFfnCols;
    if constexpr (SECOND) {
      A.init(p.ht, p.rows, row0, rows_, K);
      W.init(p.x + y0, (uint32_t)p.ldx * 2, M, [&](int c) { return (uint32_t)min(c, p.D - 8 - y0) * 2; });
    } else {
      A.init(p.x + row0, (uint32_t)p.ldx * 2, M, [&](int c) { return (uint32_t)min(c, rows_ - 8) * 2; });
      W.init(p.gz + (int64_t)(y0 >> 5) * p.ldm * 32, 64, K, [&](int c) {
        const int col = min(c, p.D - 8 - y0);
        return (uint32_t)(col >> 5) * (uint32_t)p.ldm * 64 + (col & 31) * 2;
      });
    }
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows_, int tn, int slice, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    const int l = lane_id();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = tn * kFfnCols + wn * 64 + 16 * j + 4 * (l >> 4);
      if (col >= p.D) continue;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = 16 * (wm * FM + i) + (l & 15);
        if (r >= rows_) continue;
        if (slices > 1) *(f32x4*)(p.part + (slice * rows + row0 + r) * p.D + col) = acc[j][i];
        else *(bf16x4*)(p.out + (row0 + r) * p.D + col) = pack_bf16x4(acc[j][i], 1.0f);
      }
    }
  }
};

template <class P, int STAGES>
__global__ __launch_bounds__(kSpanThreads, 2) void ffn_tile_kernel(FfnArgs p) {
  if (p.counts && blockIdx.x == 0 && threadIdx.x < 2) p.counts[threadIdx.x] = threadIdx.x ? (int)p.total : 0;
  run_ffn_tile<P, STAGES>(P(p), blockIdx.x);
}
// Sums of slices, in their order, of the products of a launch; eight are asked for at once (one behind the other: 5.0 us for 16 slices of
// one token)
struct FfnSums {
  const float* part[3];
  bf16* out[3];
  int64_t n[3];
  int slices[3], count = 0;
  void add(const FfnArgs& a) {
    if (a.slices == 1 && !a.twice) return;
    // (the second half of a slice's rows as a slice of its own)
    part[count] = a.part, out[count] = a.out, n[count] = a.rows * a.D / (a.twice ? 2 : 1), slices[count++] = a.slices * (a.twice ? 2 : 1);
  }
};
__global__ __launch_bounds__(256) void ffn_sum_slices_kernel(FfnSums p) {
  const int64_t n = p.n[blockIdx.y], at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const float* const part = p.part[blockIdx.y];
  const int slices = p.slices[blockIdx.y];
  f32x4 sum = {};
  for (int s = 0; s < slices; s += 8) {
    f32x4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = *(const f32x4*)(part + min(s + j, slices - 1) * n + at);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s + j < slices) sum += v[j];
  }
  *(bf16x4*)(p.out[blockIdx.y] + at) = pack_bf16x4(sum, 1.0f);
}
int sum_slices(const FfnSums& sums, hipStream_t st) {
  if (sums.count > 0) {
    const int64_t most = *std::max_element(sums.n, sums.n + sums.count);
    ffn_sum_slices_kernel<<<dim3((unsigned)cdiv64(most, 1024), (unsigned)sums.count), 256, 0, st>>>(sums);
  }
  return launch_status();
}

constexpr int64_t kMostTiles = (1ll << 32) / kSpanThreads - 8;  // a launch has fewer than 2^32 threads
template <class P>
int64_t blocks_of(const FfnArgs& a) {
  return cdiv64(cdiv64(a.rows, 32 * P::FM) * cdiv64(a.D, kFfnCols) * a.slices, 8) * 8;
}
template <class P, int STAGES>
int launch_tiles(const FfnArgs& a, int64_t col_tiles, hipStream_t st) {
  static LdsLimit lds;
  const int64_t tiles = cdiv64(a.rows, 32 * P::FM) * col_tiles * a.slices;
  if (tiles > kMostTiles) return MOMOE_ERR_UNSUPPORTED;
  if (!allow_lds(ffn_tile_kernel<P, STAGES>, kFfnLds<P, STAGES>, lds)) return MOMOE_ERR_LAUNCH;
  ffn_tile_kernel<P, STAGES><<<(unsigned)(cdiv64(tiles, 8) * 8), kSpanThreads, kFfnLds<P, STAGES>, st>>>(a);
  FfnSums sums;
  sums.add(a);
  return sum_slices(sums, st);
}
// The three products that need gz or hT and no more, in one launch, as none of them fills the CUs; x, w1, w2: null, or what is wanted.
// 1000 tokens, 2176 x 1152: 15.5 + 23.6 + 25.3 us apart, 40 so (0.75 PFLOP/s); 128, 96 x 64: 4.5 + 4.9 + 3.5 and 5.
template <class Dx, int STAGES>
__global__ __launch_bounds__(kSpanThreads, 2) void ffn_gradients_kernel(FfnArgs x, FfnArgs w1, FfnArgs w2, int x_blocks, int w1_blocks) {
  const int block = blockIdx.x;
  if (block < x_blocks) run_ffn_tile<Dx, STAGES>(Dx(x), block);
  else if (block < x_blocks + w1_blocks) run_ffn_tile<FfnWgrad<false>, 2>(FfnWgrad<false>(w1), block - x_blocks);
  else run_ffn_tile<FfnWgrad<true>, 2>(FfnWgrad<true>(w2), block - x_blocks - w1_blocks);
}
template <class Dx, int STAGES>
int launch_gradients(const FfnArgs* x, const FfnArgs* w1, const FfnArgs* w2, hipStream_t st) {
  static LdsLimit lds;
  constexpr size_t bytes = std::max(kFfnLds<Dx, STAGES>, std::max(kFfnLds<FfnWgrad<false>, 2>, kFfnLds<FfnWgrad<true>, 2>));
  const int64_t bx = x ? blocks_of<Dx>(*x) : 0, b1 = w1 ? blocks_of<FfnWgrad<false>>(*w1) : 0, b2 = w2 ? blocks_of<FfnWgrad<true>>(*w2) : 0;
  if (bx + b1 + b2 == 0) return MOMOE_OK;
  if (bx + b1 + b2 > kMostTiles) return MOMOE_ERR_UNSUPPORTED;
  if (!allow_lds(ffn_gradients_kernel<Dx, STAGES>, bytes, lds)) return MOMOE_ERR_LAUNCH;
  const FfnArgs none{};
  ffn_gradients_kernel<Dx, STAGES><<<(unsigned)(bx + b1 + b2), kSpanThreads, bytes, st>>>(x ? *x : none, w1 ? *w1 : none, w2 ? *w2 : none, (int)bx, (int)b1);
  FfnSums sums;
  for (const FfnArgs* a : {x, w1, w2})
    if (a) sums.add(*a);
  return sum_slices(sums, st);
}
// Rule: tiles of 32 rows as long as no CU has more than two of them, else of 64.  A contraction is cut, where there is somewhere to
// leave its sums, until every CU has two tiles, into slices of at least 8 stages and not past 10 MB of sums: a stage takes as long
// however few tiles there are (ffn_tile.hpp), so that a launch of few takes as long as their contraction is.
// Record, us.  Contraction whole | cut in 2 | 4 | 8:
//   h W2, 1 token, 2048 x 8192     47 | 26 | 16 | 12        h W2, 300 tokens, 2048 x 5632    40 | 26 | 23 | 24
//         24, 4096 x 11264         64 | 34 | 22 | 21              1000, 1024 x 2816          21 | 17 | 19 | 25
//         128, 4096 x 4096         25 | 18 | 17 | 21              1000, 2176 x 1152          16 | 23 | 27 | 36
// 32 rows | 64, weights from memory (in brackets one matrix again and again, of which the cache holds a part or all):
//   x W1, 16 tokens, 2048 x 5632   20.9 | 21.4 (13.3 | 15.7)      x W1, 64, 2048 x 5632      20.8 | 23.9 (13.7 | 15.9)
//         24, 2048 x 8192          21.1 | 21.8 (14.7 | 16.2)            500, 2048 x 512      15.7 | 18.1 (13.1 | 15.8)
//         24, 4096 x 11264         43.5 | 43.7 (32.6 | 30.7)            1000, 2048 x 512     15.8 | 17.8 (13.5 | 15.9)
//   past two of 32 rows a CU: 1000 tokens, 2176 x 1152 32.6 | 22.8; 2000, 2048 x 2048 70.3 | 49.5.  Between one and two the line is too
//   high for 48 tokens, 4096 x 11264 (352 tiles): 71.1 | 46.0.
// 128 rows a tile, or a deeper ring and one workgroup a CU, were faster nowhere but for 8 % of one launch (1000 tokens, x W1 of
// 1024 x 2816).
struct FfnPlan {
  int fm, slices;
};
FfnPlan plan_of(int64_t rows, int64_t col_tiles, int64_t contraction, int64_t cols) {
  const int64_t room = 2 * persistent_grid();
  FfnPlan plan{cdiv64(rows, 32) * col_tiles <= room ? 1 : 2, 1};
  const int64_t tiles = cdiv64(rows, 32 * plan.fm) * col_tiles;
  if (cols > 0) plan.slices = (int)std::max<int64_t>(1, std::min({room / tiles, cdiv64(contraction, kSpan) / 8, (10 << 20) / (rows * cols * 4), (int64_t)16}));
  return plan;
}
template <template <int> class P>
int launch_by_plan(FfnArgs a, const FfnPlan& plan, int64_t col_tiles, hipStream_t st) {
  a.slices = plan.slices;
  return plan.fm == 1 ? launch_tiles<P<1>, 4>(a, col_tiles, st) : launch_tiles<P<2>, 3>(a, col_tiles, st);
}
template <int FM> using Lin1Fwd = FfnLin1<FM, false>;
template <int FM> using Lin1Bwd = FfnLin1<FM, true>;
template <int FM> using DhPlain = FfnDh<FM, false>;
template <int FM> using DhSaved = FfnDh<FM, true>;

// ---- large launches: the loop of gemm_span.hpp ------------------------------------------------------------------------------------
// Its tiles of a dense block: as SpanSched deals those of one expert that holds all rows, without a table.
struct DenseSpanSched {
  using Tiles = TileSchedT<WideSpan::WROWS, WideSpan::MAX_ROWS, kSpanWaves>;
  static constexpr int kBand = Tiles::kBandTiles;
  struct Raw {
    int q;
    bool any, piece;
  };
  int rows, nb, nt, begin, limit, pos, stride, rest, cut;
  __device__ __forceinline__ DenseSpanSched(int rows_, int nb_) : rows(rows_), nb(nb_), nt((rows_ + WideSpan::MAX_ROWS - 1) / WideSpan::MAX_ROWS) {
    const int total = nt * nb, chunk = (total + 7) >> 3;
    begin = (int)(blockIdx.x & 7) * chunk;
    limit = max(0, min(chunk, total - begin));
    pos = blockIdx.x >> 3;
    stride = gridDim.x >> 3;
    rest = limit % stride;
    cut = 8 * rest <= stride ? 8 : 4 * rest <= stride ? 4 : 2;
    if (2 * rest > stride || rest == 0) cut = 0;
    else limit -= rest;
  }
  __device__ __forceinline__ int order() const { return blockIdx.x >> 3; }
  __device__ __forceinline__ Raw fetch() {
    const bool whole = pos < limit;
    Raw r;
    r.piece = !whole && cut > 0 && order() < rest * cut;
    r.any = whole || r.piece;
    r.q = begin + (whole ? pos : limit + order() / max(cut, 1));
    if (!whole) rest = 0;
    pos += stride;
    return r;
  }
  __device__ __forceinline__ TileCoord resolve(const Raw& r) const {
    TileCoord tc;
    tc.valid = r.any;
    if (!r.any) return tc;
    const int nfe = (rows + 31) >> 5, fbase = nfe / nt, fextra = nfe - fbase * nt;
    const int band = r.q / (kBand * nb), in_band = r.q - band * (kBand * nb), band_rows = min(kBand, nt - band * kBand);
    const int tl = band * kBand + in_band % band_rows;
    tc.tn = in_band / band_rows;
    int f0 = tl * fbase + min(tl, fextra), nf = fbase + (tl < fextra ? 1 : 0);
    if (r.piece) {
      const int part = order() % cut, base = nf / cut, extra = nf - base * cut;
      f0 += part * base + min(part, extra);
      nf = base + (part < extra ? 1 : 0);
    }
    tc.expert = 0;
    tc.row0 = tc.prow0 = 32 * f0;
    tc.rows = min(32 * nf, rows - 32 * f0);
    tc.alone = false;
    tc.valid = tc.rows > 0;
    Tiles::deal(tc);
    return tc;
  }
  __device__ __forceinline__ TileCoord next() { return resolve(fetch()); }
};

struct DenseSpan {
  using G = WideSpan;
  static constexpr bool EXCHANGE = false;
  struct Ids {};
  struct Late {};
  const FfnArgs& p;
  const int K;
  int n_org;
  __device__ __forceinline__ DenseSpan(const FfnArgs& p_, int K_, int width) : p(p_), K(K_), n_org(wave_id() % G::WCOLS * width) {}
  __device__ __forceinline__ void gather(const TileCoord&, Ids&) const {}
  __device__ __forceinline__ void late(const TileCoord&, const Ids&, Late&) const {}
  __device__ __forceinline__ void settle(Ids&) const {}
  __device__ __forceinline__ void settle(Late&) const {}
  __device__ __forceinline__ void finish(const TileCoord&, bf16*) const {}
  template <int NA>
  __device__ __forceinline__ void store_out(const TileCoord& tc, f32x4 (&acc)[G::FN][NA], bf16* staging) const {
    store_rows(acc, staging, p.out, (int64_t)tc.row0 + tc.mbase, tc.rows - tc.mbase, p.D, tc.tn * G::COLS + n_org, fresh_lane(),
               [](int) { return 1.0f; });
  }
};

// gz and hT of the 64 hidden columns from j0 of a wave's rows.  load(i): the values of fragment row i that come from memory are asked for;
// values(i, f, a, b, u): all of fragment (i, f).  Staging areas: 0 G_a, 1 G_b, 2 and 3 h of 32 rows.
template <int NA, class Load, class Values>
__device__ __forceinline__ void store_gradients(const FfnArgs& p, const TileCoord& tc, int j0, bf16* staging, Load load, Values values) {
  constexpr int HF = 4;
  using Stager = SpanStager<16 * HF>;
  static_assert(4 * Stager::ELEMS <= kStagingElems && NA % 2 == 0, "four areas; groups of 32 rows");
  const int H = p.H, l = fresh_lane(), rows = tc.rows - tc.mbase;
  const Stager stager(staging, l);
  const int64_t r0 = (int64_t)tc.row0 + tc.mbase;
  bf16* const gza = p.gz + ((int64_t)(j0 >> 5) * p.ldm + r0) * 32;  // uniform
  const int64_t to_b = (int64_t)(H >> 5) * p.ldm * 32;
  const uint32_t off = (stager.block_row() * 32 + stager.block_col()) * 2;
  bf16x8 v[2][2][Stager::PASSES];
  auto store_gz = [&](int i) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int q = 0; q < Stager::PASSES; ++q)
        store16(gza + half * to_b + ((int64_t)q * p.ldm + 16 * i) * 32, off, j0 + 32 * q < H, v[i & 1][half][q]);
  };
  bf16* const ht = p.ht + ((r0 >> 5) * H + j0) * 32;  // uniform
  const uint32_t hoff = (l & 15) * 64 + (l >> 4) * 16;
  bf16x8 hv[HF];
  auto store_h = [&](int i) {
    if (!p.ht) return;
#pragma unroll
    for (int q = 0; q < HF; ++q) store16(ht + ((int64_t)(i / 2) * H + 16 * q) * 32, hoff, j0 + 16 * q < H, hv[q]);
  };
  load(0);
#pragma unroll
  for (int i = 0; i < NA; ++i) {
    if (i + 1 < NA) load(i + 1);
    const bool some = 16 * i + (l & 15) < rows;
#pragma unroll
    for (int f = 0; f < HF; ++f) {
      f32x4 a, b, u;
      values(i, f, a, b, u);
      float va[4], vb[4], vh[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const SwigluGrad g(a[e], b[e], u[e]);
        va[e] = some ? g.a : 0.0f, vb[e] = some ? g.b : 0.0f, vh[e] = some ? g.h : 0.0f;
      }
      stager.put(0, f, pack_bf16x4(va[0], va[1], va[2], va[3]));
      stager.put(1, f, pack_bf16x4(vb[0], vb[1], vb[2], vb[3]));
      stager.put(2 + (i & 1), f, pack_bf16x4(vh[0], vh[1], vh[2], vh[3]));
    }
    if (i > 0) store_gz(i - 1);
    if (i > 0 && i % 2 == 0) store_h(i - 1);
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int q = 0; q < Stager::PASSES; ++q) v[i & 1][half][q] = stager.get_block(half, q);
    if (i % 2 == 1) {
#pragma unroll
      for (int q = 0; q < HF; ++q) hv[q] = stager.get_rows(2, q);
    }
    order_fence();  // (loads of several rounds ahead were spilled)
  }
  store_gz(NA - 1);
  store_h(NA - 1);
}
// where fragment row i of a wave's lies among the fragments of a matrix of `cols` columns, from column col; past the last row or column
// (of which nothing is used) at one that exists
__device__ __forceinline__ const float* fragment_of(const float* m, const FfnArgs& p, const TileCoord& tc, int i, int cols, int col, bool in) {
  const int64_t rf = min((int64_t)tc.row0 + tc.mbase + 16 * i, p.rows - 1) >> 4;
  return m + ((rf * (cols >> 4) + (in ? col >> 4 : 0)) << 8);
}

template <bool BWD>
struct Lin1DenseSpan : DenseSpan {
  static constexpr int BNH = G::COLS / 2, WIDTH = 8 * G::FN, HF = G::FN / 2;  // hidden columns of a tile, of a wave
  using Rows = FfnRows<256>;
  using Weights = SpanCols<true>;
  __device__ __forceinline__ explicit Lin1DenseSpan(const FfnArgs& p_) : DenseSpan(p_, p_.D, WIDTH) {}
  __device__ __forceinline__ void setup(const TileCoord& t, const Ids&, Rows& A, Weights& W) const {
    const int H = p.H, j0 = t.tn * BNH;
    A.init(p.x, p.ldx, t.row0, t.rows, K);
    W.init(p.w, 2 * H, [&](int c) { return (c / BNH) * H + min(j0 + (c % BNH), H - 8); });
  }
  template <int NA>
  __device__ __forceinline__ void epilogue(const TileCoord& tc, f32x4 (&acc)[G::FN][NA], const Ids&, const Late&, bf16* staging) const {
    const int H = p.H, j0 = tc.tn * BNH + n_org;  // first hidden column of this wave
    if constexpr (BWD) {
      f32x4 uq[2][HF];
      const int l = fresh_lane();
      store_gradients<NA>(
          p, tc, j0, staging,
          [&](int i) {
#pragma unroll
            for (int f = 0; f < HF; ++f) uq[i & 1][f] = *(const f32x4*)(fragment_of(p.u, p, tc, i, H, j0 + 16 * f, j0 + 16 * f < H) + 4 * l);
          },
          [&](int i, int f, f32x4& a, f32x4& b, f32x4& u) { a = acc[f][i], b = acc[HF + f][i], u = uq[i & 1][f]; });
    } else {
      using Stager = SpanStager<WIDTH>;
      const Stager stager(staging, fresh_lane());
      const int rows = tc.rows - tc.mbase;
      const int64_t r0 = (int64_t)tc.row0 + tc.mbase;
      keep_in_place(acc);
      bf16* const first = p.h + ((int64_t)(j0 >> 5) * p.ldm + r0) * 32;  // uniform
      const uint32_t off = (stager.block_row() * 32 + stager.block_col()) * 2;
      bf16x8 v[2][Stager::PASSES];
      auto store = [&](int i) {
#pragma unroll
        for (int q = 0; q < Stager::PASSES; ++q)
          store16(first + ((int64_t)q * p.ldm + 16 * i) * 32, off, 16 * i + stager.block_row() < rows && j0 + 32 * q < H, v[i & 1][q]);
      };
#pragma unroll
      for (int i = 0; i < NA; ++i) {
#pragma unroll
        for (int f = 0; f < HF; ++f) {
          float hv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) hv[e] = swiglu(acc[f][i][e], acc[HF + f][i][e]);
          stager.put(i & 1, f, pack_bf16x4(hv[0], hv[1], hv[2], hv[3]));
        }
        if (i > 0) store(i - 1);
#pragma unroll
        for (int q = 0; q < Stager::PASSES; ++q) v[i & 1][q] = stager.get_block(i & 1, q);
      }
      store(NA - 1);
      if (r0 < p.ab_rows) {
        keep_in_place(acc);
        const int l = fresh_lane();
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          if (r0 + 16 * i >= p.ab_rows) break;
#pragma unroll
          for (int f = 0; f < G::FN; ++f) {
            const int col = j0 + 16 * (f % HF);
            if (col >= H) continue;
            float* const to = p.ab + ((((r0 >> 4) + i) * (2 * H >> 4) + ((f / HF * H + col) >> 4)) << 8);
            *(f32x4*)(to + 4 * l) = acc[f][i];
          }
        }
      }
    }
  }
};

struct Lin2DenseSpan : DenseSpan {
  using Rows = SpanBlockedRows<256>;
  using Weights = SpanCols<>;
  __device__ __forceinline__ explicit Lin2DenseSpan(const FfnArgs& p_) : DenseSpan(p_, p_.H, 16 * G::FN) {}
  __device__ __forceinline__ void setup(const TileCoord& t, const Ids&, Rows& A, Weights& W) const {
    const int D = p.D, d0 = t.tn * G::COLS;
    A.init(p.h, p.ldm, t.row0, t.rows);
    W.init(p.w, D, [&](int c) { return min(d0 + c, D - 8); });
  }
  template <int NA>
  __device__ __forceinline__ void epilogue(const TileCoord& tc, f32x4 (&acc)[G::FN][NA], const Ids&, const Late&, bf16* staging) const {
    store_out(tc, acc, staging);
  }
};

template <bool SAVED>
struct DhDenseSpan : DenseSpan {
  using Rows = FfnRows<256>;
  using Weights = SpanPitchedRows<G::COLS>;
  __device__ __forceinline__ explicit DhDenseSpan(const FfnArgs& p_) : DenseSpan(p_, p_.D, 16 * G::FN) {}
  __device__ __forceinline__ void setup(const TileCoord& t, const Ids&, Rows& A, Weights& W) const {
    A.init(p.x, p.ldx, t.row0, t.rows, K);
    W.init(p.w, p.D, t.tn * G::COLS, p.H);
  }
  template <int NA>
  __device__ __forceinline__ void epilogue(const TileCoord& tc, f32x4 (&acc)[G::FN][NA], const Ids&, const Late&, bf16* staging) const {
    const int H = p.H, j0 = tc.tn * G::COLS + n_org, l = fresh_lane();
    if constexpr (SAVED) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int jh = j0 + 64 * half;
        f32x4 ab[2][4][2];
        store_gradients<NA>(
            p, tc, jh, staging,
            [&](int i) {
#pragma unroll
              for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                  ab[i & 1][f][q] = *(const f32x4*)(fragment_of(p.ab, p, tc, i, 2 * H, q * H + jh + 16 * f, jh + 16 * f < H) + 4 * l);
            },
            [&](int i, int f, f32x4& a, f32x4& b, f32x4& u) { a = ab[i & 1][f][0], b = ab[i & 1][f][1], u = acc[4 * half + f][i]; });
      }
    } else {
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        if (16 * i >= tc.rows - tc.mbase) break;
#pragma unroll
        for (int f = 0; f < G::FN; ++f)
          if (j0 + 16 * f < H)
            *(f32x4*)(const_cast<float*>(fragment_of(p.u, p, tc, i, H, j0 + 16 * f, true)) + 4 * l) = acc[f][i];
      }
    }
  }
};

struct DxDenseSpan : DenseSpan {
  using Rows = SpanBlockedRows<256>;
  using Weights = SpanPitchedRows<G::COLS>;
  __device__ __forceinline__ explicit DxDenseSpan(const FfnArgs& p_) : DenseSpan(p_, 2 * p_.H, 16 * G::FN) {}
  __device__ __forceinline__ void setup(const TileCoord& t, const Ids&, Rows& A, Weights& W) const {
    A.init(p.gz, p.ldm, t.row0, t.rows);
    W.init(p.w, K, t.tn * G::COLS, p.D);
  }
  template <int NA>
  __device__ __forceinline__ void epilogue(const TileCoord& tc, f32x4 (&acc)[G::FN][NA], const Ids&, const Late&, bf16* staging) const {
    store_out(tc, acc, staging);
  }
};

template <class P>
__global__ __launch_bounds__(kSpanThreads, 1) void ffn_span_kernel(FfnArgs p, int nb) {
  const ClockTrace trace(p.clk);
  if (p.counts && blockIdx.x == 0 && threadIdx.x < 2) p.counts[threadIdx.x] = threadIdx.x ? (int)p.total : 0;
  run_span_tiles_of<P>(p, DenseSpanSched((int)p.rows, nb));
  trace.finish();
}

// ---- which of the two -----------------------------------------------------------------------------------------------------------
// Rule: 256 x 256 tiles where the results are three tenths of a round of one a CU at least (and there are two stages of k-values).
// Record, us, small tiles | these, and the number of these:
//   x W1, 700 tokens, 2048 x 2816    25.4 | 27.5   66       h W2, 1000 tokens, 4096 x 2048    34.4 | 48.5   32
//         1250, 2048 x 2048          35.4 | 27.0   80             1250, 1024 x 4096           22.0 | 17.3   80
//         1200, 1024 x 2176          19.9 | 16.9   85             2000, 2048 x 2048           26.3 | 26.5   64
//         2000, 2048 x 2048          44.5 | 31.8   128
//         4000, 2048 x 2048          93.0 | 51.6   256
//         24, 4096 x 11264           36.5 | 58     88, hardly filled
// 8192 tokens through 2048 x 8192 take 414 (1.33 PFLOP/s) and 199 (1.38), 16384 through 4096 x 11264 2329 (1.30) and 1064 (1.42): what a
// large library product of these sizes reaches; bound by the matrix instructions at the clock that the card holds.
inline bool takes_span(int64_t rows, int64_t cols, int64_t contraction) {
  return rows > 2 * kTwiceRows && contraction >= WideSpan::AHEAD * kSpan && 10 * rows * cols >= 3 * persistent_grid() * (int64_t)(WideSpan::MAX_ROWS * WideSpan::COLS);
}
template <class P>
int launch_dense_span(const FfnArgs& a, int64_t cols, hipStream_t st) {
  static LdsLimit lds;
  if (!allow_lds(ffn_span_kernel<P>, kSpanLds, lds)) return MOMOE_ERR_LAUNCH;
  ffn_span_kernel<P><<<persistent_grid(), kSpanThreads, kSpanLds, st>>>(a, (int)cdiv64(cols, WideSpan::COLS));
  return launch_status();
}
// cols, contraction: of the product (of x W1 both halves' columns)
template <class Span, template <int> class P>
int launch(const FfnArgs& a, int64_t cols, int64_t contraction, int64_t col_tiles, hipStream_t st) {
  if (takes_span(a.rows, cols, contraction)) return launch_dense_span<Span>(a, cols, st);
  return launch_by_plan<P>(a, plan_of(a.rows, col_tiles, contraction, a.part ? cols : 0), col_tiles, st);
}
// fp32 partial sums of a product with D columns that is cut along its contraction
int64_t slices_bytes(int64_t rows, int64_t D, int64_t contraction) {
  if (takes_span(rows, D, contraction)) return 0;
  const FfnPlan plan = plan_of(rows, cdiv64(D, kFfnCols), contraction, D);
  return plan.slices > 1 ? plan.slices * rows * D * 4 : 0;
}

// of h W2, whose rows may be two each
int64_t lin2_bytes(int64_t rows, int64_t D, int64_t H) {
  if (rows > kTwiceRows) return slices_bytes(rows, D, H);
  return plan_of(2 * rows, cdiv64(D, kFfnCols), H, D).slices * 2 * rows * D * 4;
}

int check_ffn(int64_t rows, int64_t ldm, int64_t D, int64_t H) {
  if (rows <= 0 || D <= 0 || H <= 0 || ldm < rows) return MOMOE_ERR_BAD_ARG;
  // 32-bit byte offsets into a weight matrix, and from a k-blocked tile's first row
  if (D % 32 != 0 || H % 32 != 0 || ldm >= (1ll << 31) - 512 || D * H * 4 >= (1ll << 32) || D >= (1 << 22) || H >= (1 << 22))
    return MOMOE_ERR_UNSUPPORTED;
  return MOMOE_OK;
}
// Rule: gradients of the weights in tiles of 128 x 128 as long as no CU has more than two of them and none contracts over more than 8192
// tokens; where the tiles are fewer, the tokens are cut, into slices of at least 512, and past 10 MB of sums of at least 2048.
// Record, us, W2 and W1, momoe_wgrad | these:
//   31 tokens, 64 x 96       6.9, 7.1 | 4.1, 4.3            8192, 1024 x 2816     79.7, 164 | 69.2, 118
//   512, 512 x 512           17.8, 18.5 | 8.7, 9.2          65536, 1024 x 2816    476, 751 | 952, 933
//   1000, 1024 x 2816        28.3, 30.8 | 16.6, 23.2        more tiles than two a CU: 300, 2048 x 5632    17.1, 32.6 | 18.1, 31.4
//   4096, 512 x 512          87.5, 95.6 | 15.8, 19.1                                  2048, 2048 x 8192   56.7, 116 | 84.8, 159
int wgrad_slices(int64_t rows, int64_t X, int64_t Y) {
  const int64_t tiles = cdiv64(X, kFfnCols) * cdiv64(Y, kFfnCols), room = 2 * persistent_grid();
  return (int)std::max<int64_t>(1, std::min({room / tiles, cdiv64(rows, kSpan) / 8, std::max((10 << 20) / (X * Y * 4), rows / 2048), (int64_t)16}));
}
bool wgrad_in_small_tiles(int64_t rows, int64_t X, int64_t Y) {
  return cdiv64(X, kFfnCols) * cdiv64(Y, kFfnCols) <= 2 * persistent_grid() && rows <= 8192 * (int64_t)wgrad_slices(rows, X, Y);
}
// An expert of all rows is cut along them, through the workspace, where its tiles leave CUs idle in their last round; tiles that fill 5
// of 6 are done whole, which saves the partial sums' way through memory.  Us, 8192 tokens, D = 2048, H = 8192 (256 and 512 tiles of 256 x
// 256), cut | whole: W2 335 | 256, W1 640 | 470.
int64_t large_wgrad_bytes(int64_t rows, int64_t X, int64_t Y) {
  const int64_t bytes = momoe_wgrad_workspace_bytes(1, X, Y, rows);
  if (bytes <= 0) return bytes;
  const int64_t tiles = cdiv64(X, 256) * cdiv64(Y, 256), grid = persistent_grid(), rounds = cdiv64(tiles, grid);
  return 6 * tiles >= 5 * rounds * grid ? 0 : bytes;
}
// scratch of one gradient
int64_t wgrad_bytes(int64_t rows, int64_t X, int64_t Y) {
  if (!wgrad_in_small_tiles(rows, X, Y)) return std::max<int64_t>(0, large_wgrad_bytes(rows, X, Y));
  const int64_t slices = wgrad_slices(rows, X, Y);
  return slices > 1 ? slices * X * Y * 4 : 0;
}
int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }
struct FfnScratch {
  int64_t x, w1, w2;
  FfnScratch(int64_t rows, int64_t D, int64_t H, bool x_, bool w1_, bool w2_)
      : x(x_ ? aligned(slices_bytes(rows, D, 2 * H)) : 0), w1(w1_ ? aligned(wgrad_bytes(rows, D, 2 * H)) : 0),
        w2(w2_ ? aligned(wgrad_bytes(rows, H, D)) : 0) {}
  int64_t bytes() const { return x + w1 + w2; }
};
bool unaligned16(const void* p) { return ((uintptr_t)p & 15) != 0; }
bool any_unaligned(std::initializer_list<const void*> all) { return std::any_of(all.begin(), all.end(), unaligned16); }

}  // namespace
}  // namespace momoe

using namespace momoe;

extern "C" int64_t momoe_ffn_fragment_floats(int64_t rows, int64_t cols) {
  return rows < 0 || cols <= 0 || cols % 16 != 0 ? -1 : (rows + 15) / 16 * 16 * cols;
}

extern "C" int momoe_ffn_lin1_fwd(const void* x, int64_t ldx, const void* W1_D2H, void* h_blocked, float* ab, int64_t ab_rows, int64_t rows,
                                  int64_t ldm, int64_t D, int64_t H, void* stream) {
  if (!x || !W1_D2H || !h_blocked || (ab_rows > 0 && !ab) || ab_rows < 0 || ab_rows > (rows + 31) / 32 * 32 || ldx < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows_of_h(rows), ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({x, W1_D2H, h_blocked, ab})) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0 || ldx >= (1 << 22) || ab_rows % 32 != 0) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)x, ldx, (const bf16*)W1_D2H, rows, ldm, (int)D, (int)H};
  a.h = (bf16*)h_blocked;
  a.ab = ab;
  a.ab_rows = std::min((rows + 15) / 16 * 16, ab_rows);
  return launch<Lin1DenseSpan<false>, Lin1Fwd>(a, 2 * H, D, cdiv64(H, 64), (hipStream_t)stream);
}

extern "C" int64_t momoe_ffn_workspace_bytes(int64_t rows, int64_t D, int64_t H) {
  return rows <= 0 || D <= 0 || H <= 0 ? -1 : lin2_bytes(rows, D, H);
}
extern "C" int64_t momoe_ffn_h_rows(int64_t rows) { return rows < 0 ? -1 : rows_of_h(rows); }

extern "C" int momoe_ffn_lin2_fwd(const void* h_blocked, const void* W2_HD, void* y, int64_t rows, int64_t ldm, int64_t D, int64_t H,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  if (!h_blocked || !W2_HD || !y || workspace_bytes < 0 || (workspace_bytes > 0 && !workspace)) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows_of_h(rows), ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({h_blocked, W2_HD, y, workspace}) || workspace_bytes < lin2_bytes(rows, D, H)) return MOMOE_ERR_BAD_ARG;
  FfnArgs a{nullptr, 0, (const bf16*)W2_HD, rows_of_h(rows), ldm, (int)D, (int)H};
  a.twice = rows <= kTwiceRows;
  a.part = (float*)workspace;
  a.h = (bf16*)h_blocked;
  a.out = (bf16*)y;
  return launch<Lin2DenseSpan, FfnLin2>(a, D, H, cdiv64(D, kFfnCols), (hipStream_t)stream);
}

extern "C" int momoe_ffn_dgrad_h(const void* Gy, int64_t ldgy, const void* W2_HD, float* u, int64_t rows, int64_t D, int64_t H, void* stream) {
  if (!Gy || !W2_HD || !u || ldgy < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows, rows, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({Gy, W2_HD, u})) return MOMOE_ERR_BAD_ARG;
  if (ldgy % 8 != 0 || ldgy >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)Gy, ldgy, (const bf16*)W2_HD, rows, rows, (int)D, (int)H};
  a.u = u;
  return launch<DhDenseSpan<false>, DhPlain>(a, H, D, cdiv64(H, kFfnCols), (hipStream_t)stream);
}

extern "C" int momoe_ffn_swiglu_bwd(const void* x, int64_t ldx, const void* W1_D2H, const float* u, void* gz_blocked, void* hT, int32_t* counts2,
                                    int64_t tokens, int64_t rows, int64_t ldm, int64_t D, int64_t H, void* stream) {
  if (!x || !W1_D2H || !u || !gz_blocked || ldx < D || tokens < rows) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn((rows + 31) / 32 * 32, ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({x, W1_D2H, u, gz_blocked, hT})) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0 || ldx >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)x, ldx, (const bf16*)W1_D2H, rows, ldm, (int)D, (int)H};
  a.u = const_cast<float*>(u);
  a.gz = (bf16*)gz_blocked;
  a.ht = (bf16*)hT;
  a.counts = counts2;
  a.total = tokens;
  return launch<Lin1DenseSpan<true>, Lin1Bwd>(a, 2 * H, D, cdiv64(H, 64), (hipStream_t)stream);
}

extern "C" int momoe_ffn_dgrad_h_saved(const void* Gy, int64_t ldgy, const void* W2_HD, const float* ab, void* gz_blocked, void* hT,
                                       int32_t* counts2, int64_t tokens, int64_t rows, int64_t ldm, int64_t D, int64_t H, void* stream) {
  if (!Gy || !W2_HD || !ab || !gz_blocked || ldgy < D || tokens < rows) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn((rows + 31) / 32 * 32, ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({Gy, W2_HD, ab, gz_blocked, hT})) return MOMOE_ERR_BAD_ARG;
  if (ldgy % 8 != 0 || ldgy >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)Gy, ldgy, (const bf16*)W2_HD, rows, ldm, (int)D, (int)H};
  a.ab = const_cast<float*>(ab);
  a.gz = (bf16*)gz_blocked;
  a.ht = (bf16*)hT;
  a.counts = counts2;
  a.total = tokens;
  return launch<DhDenseSpan<true>, DhSaved>(a, H, D, cdiv64(H, kFfnCols), (hipStream_t)stream);
}

// (no size that momoe_wgrad refuses has few enough tiles for the small ones)
extern "C" int momoe_ffn_gradients_take(int64_t D, int64_t H, int wants_W1, int wants_W2) {
  constexpr int64_t most = 1 << 20;
  return D > 0 && H > 0 && (!(wants_W1 || wants_W2) || D <= most) && (!wants_W1 || 2 * H <= most) && (!wants_W2 || H <= most);
}

extern "C" int64_t momoe_ffn_gradients_workspace_bytes(int64_t rows, int64_t D, int64_t H, int wants_x, int wants_W1, int wants_W2) {
  return rows <= 0 || D <= 0 || H <= 0 ? -1 : FfnScratch(rows, D, H, wants_x, wants_W1, wants_W2).bytes();
}

extern "C" int momoe_ffn_gradients(const void* x, int64_t ldx, const void* Gy, int64_t ldgy, const void* gz_blocked, const void* hT,
                                   const void* W1_D2H, const int32_t* counts2, void* Gx, void* GW1_D2H, void* GW2_HD, void* workspace,
                                   int64_t workspace_bytes, int64_t rows, int64_t ldm, int64_t D, int64_t H, void* stream) {
  if ((Gx && (!gz_blocked || !W1_D2H)) || (GW1_D2H && (!x || !gz_blocked || !counts2 || ldx < D)) || (GW2_HD && (!hT || !Gy || !counts2 || ldgy < D)))
    return MOMOE_ERR_BAD_ARG;
  if (rows <= 0 || workspace_bytes < 0 || (workspace_bytes > 0 && !workspace)) return MOMOE_ERR_BAD_ARG;
  const int status = check_ffn((rows + 31) / 32 * 32, ldm, D, H);
  if (status != MOMOE_OK) return status;
  if (!momoe_ffn_gradients_take(D, H, GW1_D2H != nullptr, GW2_HD != nullptr)) return MOMOE_ERR_UNSUPPORTED;
  // tokens are addressed at 32-bit offsets
  if ((GW1_D2H && (ldx % 8 != 0 || rows * ldx * 2 >= (1ll << 32) || 8 * ldm * 64 >= (1ll << 32))) ||
      (GW2_HD && (ldgy % 8 != 0 || rows * ldgy * 2 >= (1ll << 32))))
    return MOMOE_ERR_UNSUPPORTED;
  const FfnScratch scratch(rows, D, H, Gx, GW1_D2H, GW2_HD);
  if (any_unaligned({x, Gy, gz_blocked, hT, W1_D2H, Gx, GW1_D2H, GW2_HD, workspace}) || workspace_bytes < scratch.bytes()) return MOMOE_ERR_BAD_ARG;
  const hipStream_t st = (hipStream_t)stream;
  char* const ws = (char*)workspace;
  const auto args = [&](const void* tokens, int64_t ld, const void* w, int64_t out_rows, int64_t out_cols, void* out, char* part) {
    FfnArgs a{(const bf16*)tokens, ld, (const bf16*)w, out_rows, ldm, (int)out_cols, (int)H};
    a.gz = (bf16*)const_cast<void*>(gz_blocked);
    a.ht = (bf16*)const_cast<void*>(hT);
    a.out = (bf16*)out;
    a.part = (float*)part;
    a.total = rows;
    return a;
  };
  FfnArgs ax = args(nullptr, 0, W1_D2H, rows, D, Gx, ws), a1 = args(x, ldx, nullptr, D, 2 * H, GW1_D2H, ws + scratch.x),
          a2 = args(Gy, ldgy, nullptr, H, D, GW2_HD, ws + scratch.x + scratch.w1);
  const FfnPlan plan = plan_of(rows, cdiv64(D, kFfnCols), 2 * H, D);
  ax.slices = plan.slices;
  a1.slices = wgrad_slices(rows, D, 2 * H);
  a2.slices = wgrad_slices(rows, H, D);
  const bool x_span = takes_span(rows, D, 2 * H), small1 = wgrad_in_small_tiles(rows, D, 2 * H), small2 = wgrad_in_small_tiles(rows, H, D);
  if (GW2_HD && !small2) {
    const int s = momoe_wgrad(hT, H, MOMOE_LAYOUT_TRANSPOSED, nullptr, Gy, ldgy, MOMOE_LAYOUT_ROWS, nullptr, counts2, GW2_HD, rows, 1, H, D, rows,
                              scratch.w2 ? a2.part : nullptr, scratch.w2, stream);
    if (s != MOMOE_OK) return s;
  }
  if (GW1_D2H && !small1) {
    const int s = momoe_wgrad(x, ldx, MOMOE_LAYOUT_ROWS, nullptr, gz_blocked, ldm, MOMOE_LAYOUT_KBLOCKED, nullptr, counts2, GW1_D2H, rows, 1, D,
                              2 * H, rows, scratch.w1 ? a1.part : nullptr, scratch.w1, stream);
    if (s != MOMOE_OK) return s;
  }
  if (Gx && x_span) {
    ax.slices = 1;
    const int s = launch_dense_span<DxDenseSpan>(ax, D, st);
    if (s != MOMOE_OK) return s;
  }
  const FfnArgs *px = Gx && !x_span ? &ax : nullptr, *p1 = GW1_D2H && small1 ? &a1 : nullptr, *p2 = GW2_HD && small2 ? &a2 : nullptr;
  return plan.fm == 1 ? launch_gradients<FfnDx<1>, 4>(px, p1, p2, st) : launch_gradients<FfnDx<2>, 3>(px, p1, p2, st);
}
