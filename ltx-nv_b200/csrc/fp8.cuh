// Rows in 8-bit floating point with a power-of-two scale per block of 128 columns: the
// element conversions and the scale layout shared by the kernels that write such rows
// (quantiser, norm, GEMM epilogue) and those that read them (GEMM, dequantiser).
//
// Value of column c of row r: e4m3(data[r][c]) * 2^(code - 127), code the byte of block
// c / 128. A power of two makes the scaling exact in both directions, so the only
// rounding of the format is the one to e4m3 (at most half a step, 2^-4 relative), and it
// is what the tensor core multiplies block products by itself (UE8M0).
//
// Scale layout: one 32-bit word holds the codes of four consecutive blocks (512
// columns) of a row, byte j = block 4 kq + j. Words are grouped by 128 rows in the order
// that tensor memory wants them, row i of a group at word (i % 32) * 4 + i / 32, the
// groups of one kq follow each other, and the row count is padded to a multiple of 256:
//   word(r, kq) = scales[kq * rows_padded + (r / 128) * 128 + (r % 32) * 4 + (r % 128) / 32]
// so the 512 bytes of (128 rows, 512 columns) are one contiguous, 16-byte aligned piece.
#pragma once
#include "ltx_kernels.cuh"

namespace ltx {
namespace detail {

constexpr int kFp8Block = 128;      // columns per scale
constexpr int kFp8Quad = 512;       // columns per scale word
constexpr int kFp8RowPad = 256;     // rows_padded granularity

inline int64_t fp8_rows_padded(int64_t rows) { return (rows + kFp8RowPad - 1) / kFp8RowPad * kFp8RowPad; }
inline int64_t fp8_quads(int64_t cols) { return (cols + kFp8Quad - 1) / kFp8Quad; }

LTX_DEVICE int64_t fp8_word(int64_t r, int64_t kq, int64_t rows_padded) {
  return kq * rows_padded + (r & ~int64_t(127)) + (r & 31) * 4 + ((r >> 5) & 3);
}

// Scale code of a block whose largest finite magnitude is amax: code - 127 is the least
// e >= -126 with amax <= 448 * 2^e = 1.75 * 2^(e + 8), read off amax = m * 2^E, 1 <= m < 2:
// e = E - 8, one more where m > 1.75. A block of zeros has scale 1.
LTX_DEVICE int fp8_scale_code(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int code = int(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return u == 0 ? 127 : (code < 1 ? 1 : code);
}
// 2^-(code - 127); codes are 1..247, so the result is a normal number.
LTX_DEVICE float fp8_inv_scale(int code) { return __uint_as_float(uint32_t(254 - code) << 23); }
LTX_DEVICE float fp8_scale(int code) { return __uint_as_float(uint32_t(code) << 23); }

// Four values, already divided by their scale, to e4m3 (round to nearest even), a in the
// low byte. NaN gives the 8-bit NaN; the callers turn infinities into NaN first, since the
// format has no infinity and the conversion would saturate them.
LTX_DEVICE uint32_t fp8_pack4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}\n"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
LTX_DEVICE void fp8_unpack2(uint32_t w, float& lo, float& hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(w)));
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}\n"
      : "=f"(lo), "=f"(hi)
      : "r"(h));
}

// max(|a|, |b|, |c|), NaN if any of them is.
LTX_DEVICE float max3_abs_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Quantise the 16 consecutive columns this lane holds; the 8 lanes of an aligned group
// share a block of 128 columns, the warp a quad of 512. Returns the block's scale code.
// A warp without NaN and infinities (the maximum keeps both) takes neither the second
// maximum, over finite values only, nor the replacement of infinities by NaN.
LTX_DEVICE int fp8_quantize16(float (&v)[16], uint4& out) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) top = max3_abs_nan(top, v[i], v[i + 1]);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max3_abs_nan(top, __shfl_xor_sync(0xffffffffu, top, o), 0.f);
  const float inf = __int_as_float(0x7f800000);
  if (__any_sync(0xffffffffu, !(top < inf))) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (fabsf(v[i]) < inf)
        top = fmaxf(top, fabsf(v[i]));
      else
        v[i] = __int_as_float(0x7fffffff);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const int code = fp8_scale_code(top);
  const float inv = fp8_inv_scale(code);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = fp8_pack4(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
  out = make_uint4(w[0], w[1], w[2], w[3]);
  return code;
}
// The warp's four scale bytes of a quad into its word, one from each group of 8 lanes.
LTX_DEVICE void fp8_store_codes(uint32_t* word, int code) {
  if ((lane_id() & 7) == 0) reinterpret_cast<uint8_t*>(word)[lane_id() >> 3] = uint8_t(code);
}

}  // namespace detail
}  // namespace ltx
