// 8-bit floating point (e4m3, the OCP form: largest value 448, no infinities) with a scale for each 128 values.
//
// Rows (activations): each 128 consecutive values of a row have the least power of two as their scale that leaves none above
// 448.  A power of two: dividing by it is exact, so that a value is rounded once, to e4m3, whatever computes it, and of e4m3's 18
// binades at most one is given up; the error (half a step, 2^-4 of the value) is that of any scale.  Stored as
//   q     [rows][KB * 128] bytes, KB = ceil(cols / 128), zeros past the last column
//   code  [rows][KB rounded up to 4] bytes: the scale as the matrix instruction takes it, 2^(code - 127), 255: NaN
// Weights: any fp32 scale for each 128 x 128 block.  Stored in the order in which a wavefront holds them as the first input of
// v_mfma_f32_16x16x128_f8f6f4, which takes one block of k-values in one instruction:
//   [expert][16 columns][128 k-values]: 2048 bytes = [2][64 lanes][16], k-values 64 * half + 16 * (lane / 16) .. +15 of column lane % 16
// zeros past the last row.  A wavefront reads its columns' weights with whole 1 KiB requests, straight into registers, and
// the k-values of 16 columns are consecutive in memory.  (Which k-value stands where in a fragment does not matter as long as both
// operands agree: a product is the sum over all of them.)
// The columns of the first product are those of its two halves in turn, 16 a and 16 b: h = a * b * sigmoid(b) is formed in a lane.
#pragma once
#include "lanes.hpp"

namespace momoe {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = 128;
constexpr int kFp8Frag = 2048;  // bytes of 16 columns (rows) x 128 k-values
constexpr uint32_t kLeastAmax = 0x0D800000u;  // 2^-100: a row of smaller values, of zeros too, is scaled as if this were its largest

__host__ __device__ inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

constexpr int fp8_code_bytes(int blocks) { return (blocks + 3) & ~3; }

// The scale of values of which the largest has magnitude `amax`, and its code; `amax` as bits, so that a NaN is the largest of
// all.  NaN or infinity: the code of NaN, which makes NaN of every result that the values are part of.
struct RowScale {
  uint32_t code;
  float scale;
  __device__ __forceinline__ explicit RowScale(uint32_t amax) {
    // 448 = 1.75 * 2^8: one binade more where the mantissa exceeds 1.75
    const uint32_t field = ((max(amax, kLeastAmax) + 0x1FFFFFu) >> 23) - 8;
    code = amax >= 0x7F800000u ? 255 : field;
    scale = __uint_as_float(field << 23);
  }
};
__device__ __forceinline__ float scale_of_code(uint32_t code) { return __uint_as_float(code == 255 ? 0x7FC00000u : code << 23); }
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
// eight consecutive values on a 16-byte boundary
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  struct alignas(16) Vec { T t[16 / sizeof(T)]; };
#pragma unroll
  for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) {
    const Vec w = ((const Vec*)p)[i];
#pragma unroll
    for (int e = 0; e < (int)(16 / sizeof(T)); ++e) v[i * (16 / sizeof(T)) + e] = (float)w.t[e];
  }
}

// the larger of two magnitudes, for reductions over lanes
struct LargerBits {
  __device__ __forceinline__ float operator()(float a, float b) const {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
  }
};
// the largest magnitude of four values, NaN if there is one, as bits: two instructions
__device__ __forceinline__ uint32_t largest(float a, float b, float c, float d) {
  const float three = __builtin_elementwise_maximum(__builtin_fabsf(a), __builtin_elementwise_maximum(__builtin_fabsf(b), __builtin_fabsf(c)));
  return magnitude(__builtin_elementwise_maximum(three, __builtin_fabsf(d)));
}
// four values divided by `scale`, a power of two, and rounded to e4m3
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d, float scale) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  i16x2 v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(i16x2{0, 0}, a, b, scale, false);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(v, c, d, scale, true);
  return __builtin_bit_cast(uint32_t, v);
}

// first . second * the scales of the rows of `second`, byte BYTE of `codes` in the lanes of that row
//
// The instruction adds the products of eight consecutive k-values with what lies 13 binades and more below the largest of them cut
// off (measured with pairs of powers of two; from one eight to the next nothing is lost but fp32's own rounding): a
// result is off by 2^-15 of the sum of magnitudes on N(0, 1) operands at most, and by 1.2e-5 of itself in the median.
template <int BYTE>
__device__ __forceinline__ f32x4 mfma_e4m3(i32x8 first, i32x8 second, int codes) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(first, second, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 127, BYTE, codes);
}

// The same by v_mfma_f32_16x16x32_bf16, at half the rate and with fp32's rounding alone: eight k-values at a time of operands turned
// to bf16, which holds every value of e4m3, the rows' times their scale (a power of two).
__device__ __forceinline__ bf16x8 bf16_of_e4m3(uint32_t lo, uint32_t hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Rows of the second product between it and their sum over a token's experts: eight values in 16 bytes, each 15 bits of the
// largest one's binade, whose exponent is in the eight bits left, one in the lowest bit of each half word.  Off by 2^-14 of the
// largest of the eight, where bf16 of the same size is off by 2^-9 of each: the sum of eight such rows is rounded once, to bf16,
// and not visibly before.  (fp32 rows would be twice the bytes, which are a sixth of a large call's time as it is.)  Values below
// 2^-112 are zeros; an infinity or a NaN makes NaN of all eight.
struct Packet {
  u32x4 w;
  // of v * s
  static __device__ __forceinline__ Packet of(const f32x4& a, const f32x4& b, float s) {
    const auto larger = [](float x, float y, float z) {  // (NaN if there is one)
      return __builtin_elementwise_maximum(__builtin_fabsf(x), __builtin_elementwise_maximum(__builtin_fabsf(y), __builtin_fabsf(z)));
    };
    const float all = __builtin_elementwise_maximum(larger(b[2], b[3], larger(a[0], a[1], a[2])), larger(a[3], b[0], b[1]));
    // (a value that would round up to 2^14 counts for the next binade; of a NaN with nearly all bits set that would be one past
    // the last, of which eight bits hold nothing)
    const uint32_t binade = min((magnitude(all * s) + 0x200) >> 23, 255u), field = max(binade, 15u);
    // 2^13 / 2^(field - 127) * s; a sum with 1.5 * 2^23 has the rounded product in its lowest bits
    const float unit = binade - 15 >= 255 - 15 ? 0.0f : __uint_as_float((127 + 13 + 127 - field) << 23) * s;
    const auto rounded = [&](float v) { return __float_as_uint(fmaf(v, unit, 12582912.0f)); };
    const uint32_t spread = field | field << 12;  // bit i of the field in bit i, bit i + 4 in bit 16 + i
    Packet p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4& v = i < 2 ? a : b;
      const uint32_t both = __builtin_amdgcn_perm(rounded(v[2 * (i & 1) + 1]), rounded(v[2 * (i & 1)]), 0x05040100);  // the low half words
      p.w[i] = (0x10001u & spread >> i) | (~0x10001u & both << 1);
    }
    return p;
  }
  // sum[i] += value i
  __device__ __forceinline__ void add_to(float (&sum)[8]) const {
    const uint32_t t = (w[0] & 0x10001) | (w[1] & 0x10001) << 1 | (w[2] & 0x10001) << 2 | (w[3] & 0x10001) << 3;
    const uint32_t field = (t & 0xF) | (t >> 12 & 0xF0);
    const float unit = __uint_as_float(field == 255 ? 0x7FC00000u : (field - 13) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[2 * i] = fmaf((float)((int)(w[i] << 16) >> 17), unit, sum[2 * i]);
      sum[2 * i + 1] = fmaf((float)((int)w[i] >> 17), unit, sum[2 * i + 1]);
    }
  }
};

}  // namespace momoe
