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

// |v| where it is finite, 0 where v is NaN or infinite (those take no part in a scale).
LTX_DEVICE float fp8_abs_finite(float v) {
  const float a = fabsf(v);
  return a < __int_as_float(0x7f800000) ? a : 0.f;
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

// Two values, already divided by their scale, to e4m3 (round to nearest even); lo in the
// low byte. NaN gives the 8-bit NaN; the callers turn infinities into NaN first, since the
// format has no infinity and the conversion would saturate them.
LTX_DEVICE uint32_t fp8_pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
LTX_DEVICE void fp8_unpack2(uint32_t w, float& lo, float& hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(w)));
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}\n"
      : "=f"(lo), "=f"(hi)
      : "r"(h));
}

// v / scale, NaN where v is infinite or NaN (v - v is 0 for finite v, NaN otherwise).
LTX_DEVICE float fp8_scaled(float v, float inv) { return fmaf(v, inv, v - v); }

// Quantise the 16 consecutive columns this lane holds; the 8 lanes of an aligned group
// share a block of 128 columns, the warp a quad of 512. Returns the block's scale code.
LTX_DEVICE int fp8_quantize16(const float (&v)[16], uint4& out) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) a = fmaxf(a, fp8_abs_finite(v[i]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  const int code = fp8_scale_code(a);
  const float inv = fp8_inv_scale(code);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = fp8_pack2(fp8_scaled(v[4 * i], inv), fp8_scaled(v[4 * i + 1], inv)) |
           (fp8_pack2(fp8_scaled(v[4 * i + 2], inv), fp8_scaled(v[4 * i + 3], inv)) << 16);
  out = make_uint4(w[0], w[1], w[2], w[3]);
  return code;
}
// The word of the warp's four blocks, from the codes of lanes 0, 8, 16, 24 (all lanes).
LTX_DEVICE uint32_t fp8_quad_word(int code) {
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= uint32_t(__shfl_sync(0xffffffffu, code, 8 * j)) << (8 * j);
  return w;
}

}  // namespace detail
}  // namespace ltx
