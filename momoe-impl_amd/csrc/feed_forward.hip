// A dense SwiGLU block, forward and backward: the layers beside the mixture that have no router.
//
//   a | b = x W1,  h = a b sig(b),  y = h W2
//   u = G_y W2^T,  G_a = u b sig(b),  G_b = u a sig(b) (1 + b (1 - sig(b))),  G_x = (G_a | G_b) W1^T,  G_W1 = x^T (G_a | G_b),  G_W2 = h^T G_y
//
// Rows are tokens as they come: no routing index, no gather, no gate weights, no sum over experts.  The products' operands are bf16;
// what meets in an epilogue is not rounded before: a | b that are kept for the backward, and u where a | b are made again, go through
// memory in fp32, as whole accumulator fragments ([row / 16][column / 16][64 lanes][4]: 1 KiB a store).  (In bf16 they cost half as much
// traffic and a rounding each, which doubles the error of the weight gradients.)
//   h       [H / 32][ldm][32]    k-blocked, as the second product contracts over it
//   gz      [2H / 32][ldm][32]   G_a | G_b, k-blocked, for G_x and the gradient of W1
//   hT      [rows / 32][H][32]   h once more, feature-major in groups of 32 rows, zeros behind the last row: for the gradient of W2
// The weights' gradients are momoe_wgrad of one expert.
#include <algorithm>

#include "ffn_tile.hpp"

namespace momoe {
namespace {

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
  int32_t* counts; // {0, ldm}: what momoe_wgrad takes as the rows of its one expert
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
    b = (u * av) * __builtin_fmaf(-t, sg, sg + t);  // d silu / d b = sg (1 + b (1 - sg))
  }
};

// ---- small tiles --------------------------------------------------------------------------------------------------------------
template <int FM_>
struct FfnProg {
  static constexpr int FM = FM_;
  const FfnArgs& p;
  int K, row_tiles, col_tiles;
  int64_t rows;
  __device__ __forceinline__ FfnProg(const FfnArgs& p_, int K_, int col_tiles_)
      : p(p_), K(K_), row_tiles((int)((p_.rows + 32 * FM - 1) / (32 * FM))), col_tiles(col_tiles_), rows(p_.rows) {}
  // rows as they come out of the accumulators
  __device__ __forceinline__ void store_rows_plain(int64_t row0, int rows_, int col0, f32x4 (&acc)[4][FM], int wm) const {
    const int l = lane_id();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = col0 + 16 * j + 4 * (l >> 4);
      if (col >= p.D) continue;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int r = 16 * (wm * FM + i) + (l & 15);
        if (r < rows_) *(bf16x4*)(p.out + (row0 + r) * p.D + col) = pack_bf16x4(acc[j][i], 1.0f);
      }
    }
  }
  // four columns of G_a, G_b and h of a row; `some`: it is one of the rows, and not of those that pad hT
  __device__ __forceinline__ void store_grads(int64_t row, bool some, int col, const f32x4& a, const f32x4& b, const f32x4& u) const {
    bf16x4 va, vb;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const SwigluGrad g(a[e], b[e], u[e]);
      va[e] = f2bf(g.a);
      vb[e] = f2bf(g.b);
      if (p.ht) p.ht[((row >> 5) * p.H + col + e) * 32 + (row & 31)] = some ? f2bf(g.h) : f2bf(0.0f);
    }
    if (!some) return;
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
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int wm, int wn, f32x4 (&acc)[4][FM]) const {
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
          if (p.h && r < rows)
            *(bf16x4*)(p.h + ((int64_t)(col >> 5) * p.ldm + row) * 32 + (col & 31)) =
                pack_bf16x4(f32x4{swiglu(a[0], b[0]), swiglu(a[1], b[1]), swiglu(a[2], b[2]), swiglu(a[3], b[3])}, 1.0f);
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
  __device__ __forceinline__ explicit FfnLin2(const FfnArgs& p_) : Base(p_, p_.H, (p_.D + kFfnCols - 1) / kFfnCols) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 64; }
  __device__ __forceinline__ void setup(int64_t row0, int rows, int tn, Rows& A, Weights& W) const {
    const int D = p.D, d0 = tn * kFfnCols;
    A.init(p.h, p.ldm, row0, rows, p.H);
    W.init(p.w, D, p.H, [&](int c) { return min(d0 + c, D - 8); });
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    Base::store_rows_plain(row0, rows, tn * kFfnCols + wn * 64, acc, wm);
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
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int wm, int wn, f32x4 (&acc)[4][FM]) const {
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
  __device__ __forceinline__ explicit FfnDx(const FfnArgs& p_) : Base(p_, 2 * p_.H, (p_.D + kFfnCols - 1) / kFfnCols) {}
  __device__ __forceinline__ int n_org(int wn) const { return wn * 64; }
  __device__ __forceinline__ void setup(int64_t row0, int rows, int tn, Rows& A, Weights& W) const {
    A.init(p.gz, p.ldm, row0, rows, 2 * p.H);
    W.init(p.w, 2 * p.H, tn * kFfnCols, p.D);
  }
  __device__ __forceinline__ void epilogue(int64_t row0, int rows, int tn, int wm, int wn, f32x4 (&acc)[4][FM]) const {
    Base::store_rows_plain(row0, rows, tn * kFfnCols + wn * 64, acc, wm);
  }
};

template <class P>
__global__ __launch_bounds__(kSpanThreads, P::FM == 2 ? 2 : 1) void ffn_tile_kernel(FfnArgs p) {
  if (p.counts && blockIdx.x == 0 && threadIdx.x < 2) p.counts[threadIdx.x] = threadIdx.x ? (int)p.ldm : 0;
  run_ffn_tile(P(p));
}

template <class P>
int launch_tiles(const FfnArgs& a, int64_t col_tiles, hipStream_t st) {
  static LdsLimit lds;
  const int64_t tiles = cdiv64(a.rows, 32 * P::FM) * col_tiles;
  if (tiles >= (1ll << 31) - 8) return MOMOE_ERR_UNSUPPORTED;
  if (!allow_lds(ffn_tile_kernel<P>, kFfnLds<P>, lds)) return MOMOE_ERR_LAUNCH;
  ffn_tile_kernel<P><<<(unsigned)(cdiv64(tiles, 8) * 8), kSpanThreads, kFfnLds<P>, st>>>(a);
  return launch_status();
}
// 128 rows a tile, or 64 where that leaves CUs without one
template <template <int> class P>
int launch_by_rows(const FfnArgs& a, int64_t col_tiles, hipStream_t st) {
  if (cdiv64(a.rows, 128) * col_tiles < persistent_grid()) return launch_tiles<P<2>>(a, col_tiles, st);
  return launch_tiles<P<4>>(a, col_tiles, st);
}
template <int FM> using Lin1Fwd = FfnLin1<FM, false>;
template <int FM> using Lin1Bwd = FfnLin1<FM, true>;
template <int FM> using DhPlain = FfnDh<FM, false>;
template <int FM> using DhSaved = FfnDh<FM, true>;

int check_ffn(int64_t rows, int64_t ldm, int64_t D, int64_t H) {
  if (rows <= 0 || D <= 0 || H <= 0 || ldm < rows) return MOMOE_ERR_BAD_ARG;
  // 32-bit byte offsets into a weight matrix, and from a k-blocked tile's first row
  if (D % 32 != 0 || H % 32 != 0 || ldm >= (1ll << 31) - 512 || D * H * 4 >= (1ll << 32) || D >= (1 << 22) || H >= (1 << 22))
    return MOMOE_ERR_UNSUPPORTED;
  return MOMOE_OK;
}
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
  const int st = check_ffn(rows, ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({x, W1_D2H, h_blocked, ab})) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0 || ldx >= (1 << 22) || ab_rows % 32 != 0) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)x, ldx, (const bf16*)W1_D2H, rows, ldm, (int)D, (int)H};
  a.h = (bf16*)h_blocked;
  a.ab = ab;
  a.ab_rows = std::min((rows + 15) / 16 * 16, ab_rows);
  return launch_by_rows<Lin1Fwd>(a, cdiv64(H, 64), (hipStream_t)stream);
}

extern "C" int momoe_ffn_lin2_fwd(const void* h_blocked, const void* W2_HD, void* y, int64_t rows, int64_t ldm, int64_t D, int64_t H,
                                  void* stream) {
  if (!h_blocked || !W2_HD || !y) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows, ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({h_blocked, W2_HD, y})) return MOMOE_ERR_BAD_ARG;
  FfnArgs a{nullptr, 0, (const bf16*)W2_HD, rows, ldm, (int)D, (int)H};
  a.h = (bf16*)h_blocked;
  a.out = (bf16*)y;
  return launch_by_rows<FfnLin2>(a, cdiv64(D, kFfnCols), (hipStream_t)stream);
}

extern "C" int momoe_ffn_dgrad_h(const void* Gy, int64_t ldgy, const void* W2_HD, float* u, int64_t rows, int64_t D, int64_t H, void* stream) {
  if (!Gy || !W2_HD || !u || ldgy < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows, rows, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({Gy, W2_HD, u})) return MOMOE_ERR_BAD_ARG;
  if (ldgy % 8 != 0 || ldgy >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)Gy, ldgy, (const bf16*)W2_HD, rows, rows, (int)D, (int)H};
  a.u = u;
  return launch_by_rows<DhPlain>(a, cdiv64(H, kFfnCols), (hipStream_t)stream);
}

extern "C" int momoe_ffn_swiglu_bwd(const void* x, int64_t ldx, const void* W1_D2H, const float* u, void* gz_blocked, void* hT, int32_t* counts2,
                                    int64_t rows, int64_t ldm, int64_t D, int64_t H, void* stream) {
  if (!x || !W1_D2H || !u || !gz_blocked || ldx < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows, ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({x, W1_D2H, u, gz_blocked, hT})) return MOMOE_ERR_BAD_ARG;
  if (ldx % 8 != 0 || ldx >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)x, ldx, (const bf16*)W1_D2H, rows, ldm, (int)D, (int)H};
  a.u = const_cast<float*>(u);
  a.gz = (bf16*)gz_blocked;
  a.ht = (bf16*)hT;
  a.counts = counts2;
  return launch_by_rows<Lin1Bwd>(a, cdiv64(H, 64), (hipStream_t)stream);
}

extern "C" int momoe_ffn_dgrad_h_saved(const void* Gy, int64_t ldgy, const void* W2_HD, const float* ab, void* gz_blocked, void* hT,
                                       int32_t* counts2, int64_t rows, int64_t ldm, int64_t D, int64_t H, void* stream) {
  if (!Gy || !W2_HD || !ab || !gz_blocked || ldgy < D) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows, ldm, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({Gy, W2_HD, ab, gz_blocked, hT})) return MOMOE_ERR_BAD_ARG;
  if (ldgy % 8 != 0 || ldgy >= (1 << 22)) return MOMOE_ERR_UNSUPPORTED;
  FfnArgs a{(const bf16*)Gy, ldgy, (const bf16*)W2_HD, rows, ldm, (int)D, (int)H};
  a.ab = const_cast<float*>(ab);
  a.gz = (bf16*)gz_blocked;
  a.ht = (bf16*)hT;
  a.counts = counts2;
  return launch_by_rows<DhSaved>(a, cdiv64(H, kFfnCols), (hipStream_t)stream);
}

extern "C" int momoe_ffn_dgrad_x(const void* gz_blocked, const void* W1_D2H, void* Gx, int64_t rows, int64_t D, int64_t H,
                                 void* stream) {
  if (!gz_blocked || !W1_D2H || !Gx) return MOMOE_ERR_BAD_ARG;
  const int st = check_ffn(rows, rows, D, H);
  if (st != MOMOE_OK) return st;
  if (any_unaligned({gz_blocked, W1_D2H, Gx})) return MOMOE_ERR_BAD_ARG;
  FfnArgs a{nullptr, 0, (const bf16*)W1_D2H, rows, rows, (int)D, (int)H};
  a.gz = (bf16*)const_cast<void*>(gz_blocked);
  a.out = (bf16*)Gx;
  return launch_by_rows<FfnDx>(a, cdiv64(D, kFfnCols), (hipStream_t)stream);
}
