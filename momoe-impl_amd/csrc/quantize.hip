// To 8-bit floating point: rows of activations, and weights with the order they are kept in (fp8.hpp).
#include "fp8.hpp"

namespace momoe {
namespace {

typedef _Float16 f16;

// Sixteen lanes a block of 128 values, eight in each.  Bound by HBM, the values read once: 8192 x 2048 of bf16 in 12 us, 4.2 TB/s both
// ways.
template <class T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int cols, int KB,
                                                            uint8_t* __restrict__ q, uint8_t* __restrict__ code) {
  const int64_t block = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (block >= rows * KB) return;  // (all sixteen lanes of a block)
  const int64_t row = block / KB;
  const int kb = (int)(block - row * KB), c = kb * kFp8Block + (threadIdx.x & 15) * 8;
  float v[8];
  load8(x + row * ldx + min(c, cols - 8), v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = c < cols ? v[i] : 0.0f;
    top = max(top, magnitude(v[i]));
  }
  const RowScale s(__float_as_uint(over_lanes<16>(__uint_as_float(top), LargerBits{})));
  *(u32x2*)(q + row * (KB * kFp8Block) + c) = u32x2{pack_e4m3(v[0], v[1], v[2], v[3], s.scale), pack_e4m3(v[4], v[5], v[6], v[7], s.scale)};
  if ((threadIdx.x & 15) == 0) code[row * fp8_code_bytes(KB) + kb] = (uint8_t)s.code;
}

struct PackArgs {
  const void* w;  // [N][R][C], C = halves * cols
  int R, cols, halves;
  uint8_t* packed;
  float* scale;  // [N][row blocks][halves][column blocks]; written if the weights come in bf16
};

// One workgroup a block of 128 x 128: read along the columns into LDS, written in fragments.
template <bool QUANTIZE>
__global__ __launch_bounds__(256) void pack_weights_kernel(PackArgs p) {
  __shared__ uint8_t tile[kFp8Block][kFp8Block + 4];
  __shared__ uint32_t top_of[4];
  const int CB = (int)fp8_blocks(p.cols), KB = (int)fp8_blocks(p.R);
  const int cb = blockIdx.x / p.halves, half = blockIdx.x % p.halves, kb = blockIdx.y;
  const int64_t e = blockIdx.z;
  const int C = p.cols * p.halves, c0 = cb * kFp8Block, k0 = kb * kFp8Block;
  const int tid = threadIdx.x, width = min(kFp8Block, p.cols - c0), depth = min(kFp8Block, p.R - k0);
  const int64_t at = (e * p.R + k0) * C + half * p.cols + c0;
  if constexpr (QUANTIZE) {
    // 16 lanes a row of 128, eight rows a thread
    float v[8][8];
    const int c = (tid & 15) * 8;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = (tid >> 4) + 16 * i;
      load8((const bf16*)p.w + at + (int64_t)min(k, depth - 1) * C + min(c, width - 8), v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = k < depth && c < width ? v[i][j] : 0.0f;
        top = max(top, magnitude(v[i][j]));
      }
    }
    top = __float_as_uint(over_lanes<64>(__uint_as_float(top), LargerBits{}));
    if ((tid & 63) == 0) top_of[tid >> 6] = top;
    __syncthreads();
    const RowScale s(max(max(top_of[0], top_of[1]), max(top_of[2], top_of[3])));
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *(uint32_t*)&tile[(tid >> 4) + 16 * i][c + 4 * h] =
            pack_e4m3(v[i][4 * h], v[i][4 * h + 1], v[i][4 * h + 2], v[i][4 * h + 3], s.scale);
    if (tid == 0) p.scale[((e * KB + kb) * p.halves + half) * CB + cb] = scale_of_code(s.code);
  } else {
    const int c = (tid & 31) * 4;  // 32 lanes a row, four columns in each
    for (int k = tid >> 5; k < kFp8Block; k += 8) {
      const uint32_t v = k < depth && c < width ? *(const uint32_t*)((const uint8_t*)p.w + at + (int64_t)k * C + c) : 0;
      *(uint32_t*)&tile[k][c] = v;
    }
  }
  __syncthreads();
  // 16-byte pieces: [16 columns][half of the k-values][lane]
  const int groups = p.cols / 16 * p.halves;
  for (int q = tid; q < width / 16 * 128; q += 256) {
    const int l = q & 63, h = (q >> 6) & 1, g = q >> 7;
    const int col = 16 * g + (l & 15), k = 64 * h + 16 * (l >> 4);
    u32x4 piece;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      piece[w] = tile[k + 4 * w][col] | tile[k + 4 * w + 1][col] << 8 | tile[k + 4 * w + 2][col] << 16 | (uint32_t)tile[k + 4 * w + 3][col] << 24;
    const int64_t group = (int64_t)(cb * 8 + g) * p.halves + half;
    *(u32x4*)(p.packed + ((e * groups + group) * KB + kb) * kFp8Frag + h * 1024 + l * 16) = piece;
  }
}

}  // namespace
}  // namespace momoe

using namespace momoe;

extern "C" int64_t momoe_fp8_row_bytes(int64_t cols) { return cols <= 0 ? -1 : fp8_blocks(cols) * kFp8Block; }

extern "C" int64_t momoe_fp8_code_bytes(int64_t cols) { return cols <= 0 ? -1 : (fp8_blocks(cols) + 3) & ~(int64_t)3; }

extern "C" int momoe_fp8_quantize_rows(const void* x, int type, int64_t ldx, int64_t rows, int64_t cols, void* q, void* code,
                                       void* stream) {
  if (!x || !q || !code || rows <= 0 || cols <= 0 || ldx < cols) return MOMOE_ERR_BAD_ARG;
  if (type != MOMOE_TYPE_BF16 && type != MOMOE_TYPE_F32 && type != MOMOE_TYPE_F16) return MOMOE_ERR_BAD_ARG;
  if (((uintptr_t)x | (uintptr_t)q) & 15 || (uintptr_t)code & 3) return MOMOE_ERR_BAD_ARG;
  const int64_t KB = fp8_blocks(cols), groups = cdiv64(rows * KB, 16);
  if (cols % 8 != 0 || ldx % 8 != 0 || cols >= (1ll << 31) - kFp8Block || rows >= (1ll << 31) || groups >= (1ll << 31))
    return MOMOE_ERR_UNSUPPORTED;
  const auto launch = [&](auto t) {
    using T = decltype(t);
    quantize_rows_kernel<T><<<(unsigned)groups, 256, 0, (hipStream_t)stream>>>((const T*)x, ldx, rows, (int)cols, (int)KB, (uint8_t*)q, (uint8_t*)code);
  };
  if (type == MOMOE_TYPE_BF16) launch(bf16{});
  else if (type == MOMOE_TYPE_F32) launch(float{});
  else launch(f16{});
  return launch_status();
}

extern "C" int64_t momoe_fp8_weight_bytes(int64_t N, int64_t R, int64_t C) {
  if (N <= 0 || R <= 0 || C <= 0 || C % 16 != 0) return -1;
  return N * (C / 16) * fp8_blocks(R) * kFp8Frag;
}

extern "C" int momoe_fp8_pack_weights(const void* W_NRC, int quantized, int64_t N, int64_t R, int64_t C, int halves, void* packed,
                                      float* scale, void* stream) {
  if (!W_NRC || !packed || (!quantized && !scale) || N <= 0 || R <= 0 || C <= 0 || halves < 1 || halves > 2) return MOMOE_ERR_BAD_ARG;
  if (((uintptr_t)W_NRC | (uintptr_t)packed) & 15) return MOMOE_ERR_BAD_ARG;
  if (C % (16 * halves) != 0 || R >= (1 << 22) || C >= (1 << 30) || N > 65535) return MOMOE_ERR_UNSUPPORTED;
  const PackArgs a{W_NRC, (int)R, (int)(C / halves), halves, (uint8_t*)packed, scale};
  const dim3 grid((unsigned)(fp8_blocks(C / halves) * halves), (unsigned)fp8_blocks(R), (unsigned)N);
  (quantized ? pack_weights_kernel<false> : pack_weights_kernel<true>)<<<grid, 256, 0, (hipStream_t)stream>>>(a);
  return launch_status();
}
