// 4-bit microscaled formats: what the quantisation, the product and the norm that writes 4 bits share.
//
//   nvfp4  x ~ code * scale[row, k / 16] * row_scale[row], scale e4m3, row_scale a power of two in fp32
//   mxfp4  x ~ code * scale[row, k / 32], scale = 2^(byte - 127)
// Codes are e2m1 (sign, 0 0.5 1 1.5 2 3 4 6), the even element in the low half of a byte.
//
// Why the row scale is a power of two: every decision is then exact.  A block's scale is e4m3(max / 6 / 2^p) and a
// code is the e2m1 number nearest to x / (scale * 2^p), i.e. quotients of x by a number of at most four bits.  A boundary
// times that number has at most seven bits: an x that is not on it is at least one of its last places away, and the
// quotient more than half a last place of the boundary.  So a quotient rounded once to fp32 decides like the infinitely
// precise one, for fp32 rows as for 16-bit ones.  e4m3 is a floating format: the up to one bit of its
// range that a power of two leaves unused costs no precision.
//
// Block scales lie as the tensor core reads them: tiles of 128 rows x 4 scales = 512 bytes, byte
// (r % 32) * 16 + (r / 32) * 4 + k; a panel of 128 rows is its tiles one after another, padded to whole steps of
// 256 columns (16 nvfp4 or 8 mxfp4 scales).  Padding is zero.
#pragma once

#include "common.cuh"

namespace cdb {

constexpr int FP4_STEP_COLS = 256;  // K columns of one pipeline step of the product: panels are padded to it
constexpr int FP4_MAX_COLS = 16384;

__host__ __device__ constexpr int fp4_block(bool nv) { return nv ? 16 : 32; }
// Tiles (of 512 bytes) in a panel of 128 rows.
__host__ __device__ constexpr int64_t fp4_panel_tiles(int64_t cols, bool nv) {
  return (cols + FP4_STEP_COLS - 1) / FP4_STEP_COLS * (FP4_STEP_COLS / fp4_block(nv) / 4);
}
// Byte offset of the word that holds the scales 4 * word .. 4 * word + 3 of a row.
__host__ __device__ __forceinline__ int64_t fp4_scale_word(int64_t row, int word, int64_t panel_tiles) {
  const int r = (int)(row & 127);
  return ((row >> 7) * panel_tiles + word) * 512 + (r & 31) * 16 + (r >> 5) * 4;
}

#ifdef __CUDACC__
// Four pairs of fp32 -> eight e2m1 codes (round to nearest even, saturating); v[0] in the lowest four bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// Eight e2m1 codes -> four packed f16 pairs (exact).
__device__ __forceinline__ void e2m1x8_to_half2(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)byte));
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ uint32_t float_to_e4m3(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xffu;
}
__device__ __forceinline__ float e8m0_to_float(uint32_t byte) {
  // 255 stands for NaN, 0 for 2^-127 (a subnormal float)
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}
template <bool NV>
__device__ __forceinline__ float fp4_scale_value(uint32_t byte) {
  return NV ? e4m3_to_float(byte) : e8m0_to_float(byte);
}

// row_scale of a row whose largest magnitude is `top`: the smallest power of two >= top / 2688 (2688 = 6 * 448) and
// >= 2^-100.  top = m * 2^e: 2^(e - 11) if m <= 2688 / 2048, else 2^(e - 10).  NaN if the row holds an infinity or NaN.
__device__ __forceinline__ float fp4_row_scale(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x280000u ? 11 : 10);  // 1.3125 = 1 + 0x280000 / 2^23
  return __uint_as_float((uint32_t)(max(e, -100) + 127) << 23);
}

// The scale byte of a block whose largest magnitude is `top`, and how its elements become codes:
// code = e2m1(q), q = x / step.  nvfp4: q from an approximate reciprocal and one correction, q' = q + (x - q step) inverse:
// the residual is exact and the correction good to 2^-40, while the quotient of an fp32 number by one of four bits is no
// nearer than 1/30 of a last place to the middle of two fp32 numbers: q' is the nearest fp32 number; mxfp4: step is a power of two, x * inverse is exact.
struct Fp4Step {
  uint32_t byte;
  float step, inverse;
};
template <bool NV>
__device__ __forceinline__ Fp4Step fp4_block_step(float top, float row_scale) {
  Fp4Step s;
  if constexpr (NV) {
    // top / row_scale / 6: the first division is exact, the second is corrected to the nearest fp32
    const float a = __fmul_rn(top, __uint_as_float(0x7f000000u - __float_as_uint(row_scale)));  // top / 2^p: exact
    constexpr float sixth = 1.0f / 6.0f;
    float t = __fmul_rn(a, sixth);
    t = fmaf(fmaf(-t, 6.0f, a), sixth, t);
    const bool finite = row_scale == row_scale;
    s.byte = finite ? float_to_e4m3(t) : 0u;
    const float v = e4m3_to_float(s.byte);
    s.step = v * row_scale;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.inverse) : "f"(s.step));
    if (s.byte == 0u) s.inverse = 0.f;
  } else {
    const uint32_t e = __float_as_uint(top) >> 23;  // top >= 0
    s.byte = e == 255u ? 255u : e > 2u ? e - 2u : 0u;
    s.step = e8m0_to_float(s.byte);
    s.inverse = e == 255u ? 0.f : __uint_as_float((254u - s.byte) << 23);
  }
  return s;
}
// Eight elements of a block -> their codes.
template <bool NV>
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], const Fp4Step& s) {
  float q[8];
  const uint64_t inverse = f32_pair(s.inverse, s.inverse), minus_step = f32_pair(-s.step, -s.step);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint64_t v = f32_pair(x[j], x[j + 1]);
    uint64_t e = f32_mul2(v, inverse);
    // a block of zeros (inverse 0) has step 0: the correction adds x * 0
    if constexpr (NV) e = f32_fma2(f32_fma2(e, minus_step, v), inverse, e);
    f32_unpair(e, q[j], q[j + 1]);
  }
  return e2m1x8(q);
}
#endif

}  // namespace cdb
