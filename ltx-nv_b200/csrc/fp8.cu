// Rows in 8-bit floating point (fp8.cuh) and the linear layers on them:
//   ltx_quantize_fp8, ltx_dequantize_fp8, ltx_fp8_pack_scales   the format
//   ltx_norm_modulate_fp8   norm + adaLN modulation written as 8-bit rows
//   ltx_linear_fp8          C = epilogue(A W^T), A and W 8-bit rows
//   ltx_quantize_linear_fp8 the same from F32 / BF16 rows
// None has a counterpart in the reference, which runs its linear layers in bf16
// (ltx_nn.py:126-158, 188-192, 244-245).
#include <algorithm>
#include <cmath>

#include "fp8.cuh"

namespace ltx {
namespace detail {

// 16 consecutive values, 32 (bf16) or 64 (fp32) bytes, 32-byte aligned.
template <typename T> LTX_DEVICE void ld16v(const T* p, float (&v)[16]);
template <> LTX_DEVICE void ld16v<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[16]) {
  uint32_t r[8];
  ldg_32b(p, r);
#pragma unroll
  for (int i = 0; i < 8; ++i) unpack_bf16x2(r[i], v[2 * i], v[2 * i + 1]);
}
template <> LTX_DEVICE void ld16v<float>(const float* p, float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t r[8];
    ldg_32b(p + 8 * h, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * h + i] = __uint_as_float(r[i]);
  }
}
template <typename T> LTX_DEVICE void st16v(T* p, const float (&v)[16]);
template <> LTX_DEVICE void st16v<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[16]) {
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  stg_32b(p, r);
}
template <> LTX_DEVICE void st16v<float>(float* p, const float (&v)[16]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[8 * h + i]);
    stg_32b(p + 8 * h, r);
  }
}

// How the rows of an operand may be read: 0 by element, 1 by 16 bytes, 2 by 32 bytes.
template <typename T>
inline int row_vec(const T* p, int64_t ld) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const int64_t b = ld * int64_t(sizeof(T));
  return a % 32 == 0 && b % 32 == 0 ? 2 : a % 16 == 0 && b % 16 == 0 && ld % 8 == 0 ? 1 : 0;
}

// 16 consecutive columns [c, c + 16) of a row, zeros from `cols` on.
template <typename T>
LTX_DEVICE void load16(const T* row, int64_t c, int64_t cols, int vec, float (&v)[16]) {
  if (vec == 2 && c + 16 <= cols) {
    ld16v<T>(row + c, v);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t c8 = c + 8 * h;
    float t[8];
    if (vec && c8 + 8 <= cols) {
      ld8<T>(row + c8, t);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = c8 + i < cols ? ld_elem<T>(row + c8 + i) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * h + i] = t[i];
  }
}

// A warp per (row, 512 columns): 32 bytes (bf16) per lane in, 16 out. HBM-bound: 47.5 us at
// 12288 x 8192 bf16 = 6.4 TB/s, 97 % of the measured copy. Many short warps per SM keep
// more bytes in flight than several rows per warp (two rows 65 us, four 98).
template <typename T>
__global__ void __launch_bounds__(256, 6) quantize_fp8_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                              int64_t cols, int quads, int vec,
                                                              uint8_t* __restrict__ q, int64_t ldq,
                                                              uint32_t* __restrict__ scales, int64_t rows_padded) {
  pdl_wait();
  pdl_trigger();
  const int64_t task = int64_t(blockIdx.x) * 8 + warp_id();
  const int64_t r = task / quads;
  if (r >= rows) return;
  const int kq = int(task - r * quads);
  const int64_t c = int64_t(kq) * kFp8Quad + lane_id() * 16;
  float v[16];
  load16<T>(x + r * ldx, c, cols, vec, v);
  uint4 out;
  const int code = fp8_quantize16(v, out);
  if (c < cols) *reinterpret_cast<uint4*>(q + r * ldq + c) = out;
  fp8_store_codes(scales + fp8_word(r, kq, rows_padded), code);
}

constexpr int kDequantRows = 4;
// A warp takes 512 columns of four rows, all of whose loads are in flight together.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_fp8_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                             const uint32_t* __restrict__ scales, int64_t rows_padded,
                                                             int64_t rows, int64_t cols, int quads, int vec,
                                                             T* __restrict__ x, int64_t ldx) {
  pdl_wait();
  pdl_trigger();
  const int64_t task = int64_t(blockIdx.x) * 8 + warp_id();
  const int64_t r0 = task / quads * kDequantRows;
  const int kq = int(task % quads);
  const int64_t c = int64_t(kq) * kFp8Quad + lane_id() * 16;
  if (r0 >= rows || c >= cols) return;
  uint4 w[kDequantRows];
  uint32_t word[kDequantRows];
#pragma unroll
  for (int i = 0; i < kDequantRows; ++i) {
    const int64_t r = r0 + i < rows ? r0 + i : rows - 1;
    w[i] = *reinterpret_cast<const uint4*>(q + r * ldq + c);  // inside the row: ldq is a multiple of 16
    word[i] = scales[fp8_word(r, kq, rows_padded)];
  }
#pragma unroll
  for (int i = 0; i < kDequantRows; ++i) {
    if (r0 + i >= rows) break;
    const float s = fp8_scale((word[i] >> (8 * (lane_id() >> 3))) & 255);
    const uint32_t b[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
    float v[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      fp8_unpack2(b[j], v[4 * j], v[4 * j + 1]);
      fp8_unpack2(b[j] >> 16, v[4 * j + 2], v[4 * j + 3]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] *= s;
    T* row = x + (r0 + i) * ldx;
    if (vec == 2 && c + 16 <= cols) {
      st16v<T>(row + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (c + j < cols) st_elem<T>(row + c + j, v[j]);
    }
  }
}

// float32 powers of two (rows, blocks) -> the scale words; one thread per word.
__global__ void __launch_bounds__(256) fp8_pack_scales_kernel(const float* __restrict__ s, int64_t ld, int64_t rows,
                                                              int64_t blocks, int quads, uint32_t* __restrict__ out,
                                                              int64_t rows_padded) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= rows * quads) return;
  const int64_t kq = i / rows, r = i - kq * rows;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t b = kq * 4 + j;
    const uint32_t code = b < blocks ? (__float_as_uint(s[r * ld + b]) >> 23) & 255u : 127u;
    w |= code << (8 * j);
  }
  out[fp8_word(r, kq, rows_padded)] = w;
}

// Modulation vector of 8 columns in fp32: table + mod, unrounded (one rounding at the
// end of the operator; ModVec::at8 rounds the sum for the bf16 path).
template <typename T>
LTX_DEVICE void modvec8(const ModVec<T>& m, int64_t b, int64_t t, int64_t c, float (&v)[8]) {
  float a[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  if (m.table) {
    ld8<T>(m.table + m.toff + c, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += a[i];
  }
  if (m.mod) {
    ld8<T>(m.mod + b * m.ldb + t * m.ldt + m.moff + c, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += a[i];
  }
}

// Modulation vectors of this lane's 16 columns as pairs: 1 + scale and shift.
template <typename T>
LTX_DEVICE void norm_vectors(const ModVec<T>& scale, const ModVec<T>& shift, int64_t b, int64_t t, int c, int D,
                             uint64_t (&sc)[8], uint64_t (&sh)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float a[8], e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = e[i] = 0.f;
    if (scale.on && c + 8 * h < D) modvec8<T>(scale, b, t, c + 8 * h, a);
    if (shift.on && c + 8 * h < D) modvec8<T>(shift, b, t, c + 8 * h, e);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[4 * h + i] = f2_pack(1.f + a[2 * i], 1.f + a[2 * i + 1]);
      sh[4 * h + i] = f2_pack(e[2 * i], e[2 * i + 1]);
    }
  }
}

// Sixteen columns as loaded: raw bits, so that a prefetched bf16 row costs 8 registers.
template <typename T>
struct Raw16 {
  static constexpr int N = 4 * int(sizeof(T));
  uint32_t r[N];
  LTX_DEVICE void load(const T* row, int c, int cols, int vec) {
    if (vec == 2 && c + 16 <= cols) {
#pragma unroll
      for (int h = 0; h < N / 8; ++h) {
        uint32_t t[8];
        ldg_32b(reinterpret_cast<const uint8_t*>(row + c) + 32 * h, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[8 * h + i] = t[i];
      }
      return;
    }
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {  // columns are a multiple of 8: 16-byte pieces are whole
      const int at = c + h * (16 / int(sizeof(T)));
      const uint4 u = at < cols ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0, 0, 0, 0);
      r[4 * h] = u.x; r[4 * h + 1] = u.y; r[4 * h + 2] = u.z; r[4 * h + 3] = u.w;
    }
  }
  LTX_DEVICE void get(uint64_t (&v)[8]) const {  // fp32 pairs
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2)
        v[i] = f2_pack(__uint_as_float(r[i] << 16), __uint_as_float(r[i] & 0xffff0000u));
      else
        v[i] = f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    }
  }
};

// y = norm(x) * (1 + scale) + shift in fp32, quantised once. A row takes `wr` warps, 512
// columns each, 16 per lane; a CTA holds groups = 8 / wr rows at a time (wr <= 8) and walks
// `per_cta` rows of one sample, whose vectors stay in registers (HOIST: per-sample vectors
// and rows of at most 8192 columns). The next row is loaded before this one is reduced: one
// __syncthreads per row (two for LayerNorm, whose squares are taken about the mean).
// 12288 x 2048 bf16: 19.9 us = 3.8 TB/s, 58 % of the measured copy, bound by instruction
// issue (65 % active, 330 instructions per 512 columns before the packed arithmetic); rows
// with their vectors reloaded took 49 us, a deeper prefetch changed nothing.
template <typename T, int KIND, bool HOIST, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 3 : 1)
    norm_modulate_fp8_kernel(const T* __restrict__ x, int64_t ldx, int vec, int64_t rows, int64_t rows_per_batch, int D,
                             int wr, int chunks, int per_cta, float eps, ModVec<T> shift, ModVec<T> scale,
                             uint8_t* __restrict__ q, int64_t ldq, uint32_t* __restrict__ scales,
                             int64_t rows_padded) {
  __shared__ float red[4][32];
  const int groups = int(blockDim.x >> 5) / wr, group = warp_id() / wr, w = warp_id() - group * wr;
  const int c = (w * 32 + lane_id()) * 16;
  // rows [r0, r1) of sample b; this group's are r0 + group, step groups
  const int64_t b = blockIdx.x / chunks;
  const int64_t r0 = b * rows_per_batch + int64_t(blockIdx.x - b * chunks) * per_cta;
  const int64_t r1 = min(min(r0 + per_cta, (b + 1) * rows_per_batch), rows);
  pdl_wait();
  pdl_trigger();
  Raw16<T> raw;
  if (r0 + group < r1) raw.load(x + (r0 + group) * ldx, c, D, vec);
  uint64_t sc[8], sh[8];
  if constexpr (HOIST) norm_vectors<T>(scale, shift, b, 0, c, D, sc, sh);
  const bool whole = c + 16 <= D;  // all of this lane's columns exist
  const float inv_d = 1.f / float(D);
  int phase = 0;
  // Sum over the row's warps, in warp order (the same value in all of them).
  auto row_sum = [&](float s) {
    s = warp_sum(s);
    if (wr > 1) {
      if (lane_id() == 0) red[phase][warp_id()] = s;
      __syncthreads();
      s = 0.f;
#pragma unroll 4
      for (int i = 0; i < wr; ++i) s += red[phase][group * wr + i];
      phase = (phase + 1) & 3;  // a buffer is written again three barriers later
    }
    return s;
  };
  for (int64_t base = r0; base < r1; base += groups) {  // the same count for every thread
    const int64_t row = base + group;
    uint64_t v[8];
    raw.get(v);
    if (row + groups < r1) raw.load(x + (row + groups) * ldx, c, D, vec);
    auto total = [](const uint64_t (&t)[4]) {
      float lo, hi;
      f2_unpack(f2_add(f2_add(t[0], t[1]), f2_add(t[2], t[3])), lo, hi);
      return lo + hi;
    };
    // columns past D hold zeros and stay zeros
    auto clear = [&]() {
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + 2 * i >= D) v[i] = 0;
      }
    };
    if constexpr (KIND == LTX_NORM_LAYER) {
      uint64_t t[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
      for (int i = 4; i < 8; ++i) t[i - 4] = f2_add(t[i - 4], v[i]);
      const float mean = row_sum(total(t)) * inv_d;
      const uint64_t m2 = f2_pack(mean, mean);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = f2_sub(v[i], m2);
      clear();
    }
    if constexpr (KIND != LTX_NORM_NONE) {
      uint64_t t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = f2_fma(v[i + 4], v[i + 4], f2_mul(v[i], v[i]));
      // one Newton step on the approximate root: within an ulp
      const float a = fmaf(row_sum(total(t)), inv_d, eps), y = rsqrtf(a);
      const float rstd = a > 0.f && a < __int_as_float(0x7f800000) ? fmaf(0.5f * y, fmaf(-a * y, y, 1.f), y) : y;
      const uint64_t r2 = f2_pack(rstd, rstd);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = f2_mul(v[i], r2);
    }
    if (row >= r1) continue;  // uniform over the row's warps
    if constexpr (!HOIST) norm_vectors<T>(scale, shift, b, row - b * rows_per_batch, c, D, sc, sh);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f2_fma(v[i], sc[i], sh[i]);
    clear();
    float y[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) f2_unpack(v[i], y[2 * i], y[2 * i + 1]);
    uint4 out;
    const int code = fp8_quantize16(y, out);
    if (c < D) *reinterpret_cast<uint4*>(q + row * ldq + c) = out;
    fp8_store_codes(scales + fp8_word(row, w, rows_padded), code);
  }
}

// GELU (tanh form) as v * sigmoid(2 z), z = sqrt(2/pi) (v + 0.044715 v^3): one exponential
// and one division, accurate to a few fp32 units in the last place.
LTX_DEVICE float gelu_sigmoid(float v) {
  const float z2 = 1.5957691216057308f * fmaf(0.044715f * v * v, v, v);
  return __fdividef(v, 1.f + __expf(-z2));
}

// 4 consecutive values, 8 (bf16) or 16 (fp32) bytes, aligned.
template <typename T> LTX_DEVICE void ld4v(const T* p, float (&v)[4]);
template <> LTX_DEVICE void ld4v<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  unpack_bf16x2(u.x, v[0], v[1]);
  unpack_bf16x2(u.y, v[2], v[3]);
}
template <> LTX_DEVICE void ld4v<float>(const float* p, float (&v)[4]) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
template <typename T> LTX_DEVICE void st4v(T* p, const float (&v)[4]);
template <> LTX_DEVICE void st4v<__nv_bfloat16>(__nv_bfloat16* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
template <> LTX_DEVICE void st4v<float>(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
// SiLU's division gives 0 where the divisor passes 2^126 (v below -87; the value is within
// 2^-119 of 0 there).
// Epilogue of W (1, 4 or 16) accumulators, columns [col, col + W) of row `row` (sample sb, token
// st), in fp32 and rounded once on the store: acc + bias, then the activation, residual +
// gate * (acc + bias), or + row_vec on marked rows. W > 1 needs every vector aligned there.
template <typename T, int W, int STRIDE = 1>
LTX_DEVICE void fp8_epilogue(const Epi<T>& e, T* __restrict__ crow, int64_t row, int64_t sb, int64_t st, int col,
                             float (&v)[W], int N = 0) {
  auto load = [&](const T* p, float (&x)[W]) {
    if constexpr (STRIDE > 1) {
#pragma unroll
      for (int i = 0; i < W; ++i) x[i] = col + i * STRIDE < N ? ld_elem<T>(p + i * STRIDE) : 0.f;
    } else if constexpr (W == 16)
      ld16v<T>(p, x);
    else if constexpr (W == 4)
      ld4v<T>(p, x);
    else
      x[0] = ld_elem<T>(p);
  };
  float a[W];
  if (e.bias) {
    load(e.bias + col, a);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += a[i];
  }
  if (e.kind == LTX_EPI_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = gelu_sigmoid(v[i]);
  } else if (e.kind == LTX_EPI_SILU) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = __fdividef(v[i], 1.f + __expf(-v[i]));
  } else if (e.kind == LTX_EPI_GATE_RESIDUAL) {
    float g[W];
#pragma unroll
    for (int i = 0; i < W; ++i) g[i] = e.gate.on ? 0.f : 1.f;
    if (e.gate.table) {
      load(e.gate.table + e.gate.toff + col, a);
#pragma unroll
      for (int i = 0; i < W; ++i) g[i] += a[i];
    }
    if (e.gate.mod) {
      load(e.gate.mod + sb * e.gate.ldb + st * e.gate.ldt + e.gate.moff + col, a);
#pragma unroll
      for (int i = 0; i < W; ++i) g[i] += a[i];
    }
    load(e.residual + row * e.ld_res + col, a);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = fmaf(g[i], v[i], a[i]);
  } else if (e.kind == LTX_EPI_ROW_MASK_ADD && e.row_mask[row] > 0.f) {
    load(e.row_vec + col, a);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += a[i];
  }
  if constexpr (STRIDE > 1) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (col + i * STRIDE < N) st_elem<T>(crow + col + i * STRIDE, v[i]);
  } else if constexpr (W == 16)
    st16v<T>(crow + col, v);
  else if constexpr (W == 4)
    st4v<T>(crow + col, v);
  else
    st_elem<T>(crow + col, v[0]);
}
// 16 columns of which those below N exist; `vec`: 32-byte accesses are allowed.
template <typename T>
LTX_DEVICE void fp8_epilogue_cols(const Epi<T>& e, bool vec, T* __restrict__ crow, int64_t row, int64_t sb, int64_t st,
                                  int col, int N, float (&v)[16]) {
  if (vec && col + 16 <= N) {
    fp8_epilogue<T, 16>(e, crow, row, sb, st, col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (col + i < N) {
        float x[1] = {v[i]};
        fp8_epilogue<T, 1>(e, crow, row, sb, st, col + i, x);
      }
  }
}

// ---------------------------------------------------------------------------------
// C = epilogue(A W^T) on 8-bit rows with the block-scaled tensor-core MMA.
//
// acc[m][n] = sum over blocks b of 2^(ea[m][b] + ew[n][b]) sum_{k in b} a[m][k] w[n][k]: the MMA
// takes e4m3 operands and a power of two per row and 32 values of K, so a block of 128
// columns is one 128-byte slab of both operands and four MMAs (K = 32) that read the same
// scale byte; sums stay in fp32 in tensor memory, no scaling is left for the CUDA cores.
//
// A scale word holds four blocks, so scales move once per four slabs: 512 bytes per 128 rows
// by TMA beside the slab (that order is the format's, fp8.cuh), then one tcgen05.cp per 128
// rows into tensor memory, in order with the MMAs that follow it; two buffers alternate.
// Four more warps that stored the words with tcgen05.st, off the issuing thread, were
// slower: 660 against 565 clocks per slab at 12288 x 2048 x 8192 (the issuer waits for them).
// ---------------------------------------------------------------------------------

// One 128 x 128 tile per CTA, K split over the `split` CTAs of a cluster, whose fp32 partial
// tiles are added through distributed shared memory in rank order: short and wide problems
// spread over the SMs without a workspace or a second launch, and the sum's order does not
// depend on timing. Tiles whose output cannot be stored 32 bytes at a time take the same
// way through shared memory, so that neighbouring threads store neighbouring columns. Two
// CTAs with three stages each share an SM, so that one starts and ends under the other's
// MMAs (12288 x 2048 x 2048: 61.6 us, 124 us with one CTA of six stages).
struct Fp8TileCfg {
  static constexpr int STAGES = 3;
  static constexpr int SLAB = 128 * 128;             // 128 rows x 128 bytes
  static constexpr int SF = 512;                     // scale words of 128 rows, four slabs
  static constexpr int STAGE_BYTES = 2 * SLAB;
  static constexpr int RING = STAGES * STAGE_BYTES;
  static constexpr int TMEM_COLS = 256;              // accumulator [0, 128), scales [128, 144)
  static constexpr int LD_PART = 128 + 4;            // floats per row of a partial tile (no bank conflicts)
  static constexpr int SMEM = RING + STAGES * 2 * SF + 256 + 1024;
  static_assert(128 * LD_PART * 4 <= RING, "the partial tile reuses the operand ring");
};

// The rows rank, rank + SPLIT, .. of the tile whose SPLIT fp32 partials lie in the cluster's
// CTAs are added in rank order into this CTA's own part (at `own`, shared address `base`).
// One warp per row, so that a part's row is one contiguous 512-byte read, and 8 / SPLIT rows at
// a time, so that 8 reads are in flight (with a lane per row the reads of 128 rows and 8
// parts took 20 us).
template <int SPLIT>
LTX_DEVICE void fp8_add_parts(float* own, uint32_t base, int rows, int rank) {
  constexpr int U = 8 / SPLIT;
  const int lane = lane_id();
  uint32_t part[SPLIT];
#pragma unroll
  for (int p = 0; p < SPLIT; ++p) part[p] = mapa_shared(base, uint32_t(p)) + 16u * lane;
  for (int r0 = warp_id() * SPLIT * U + rank; r0 < rows; r0 += 6 * SPLIT * U) {
    float4 x[U][SPLIT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * SPLIT < rows ? r0 + u * SPLIT : r0;
      const uint32_t at = uint32_t(r * Fp8TileCfg::LD_PART) * 4u;
#pragma unroll
      for (int p = 0; p < SPLIT; ++p) x[u][p] = ld_cluster_f4(part[p] + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + u * SPLIT >= rows) break;
#pragma unroll
      for (int p = 1; p < SPLIT; ++p) {
        x[u][0].x += x[u][p].x;
        x[u][0].y += x[u][p].y;
        x[u][0].z += x[u][p].z;
        x[u][0].w += x[u][p].w;
      }
      reinterpret_cast<float4*>(own + (r0 + u * SPLIT) * Fp8TileCfg::LD_PART)[lane] = x[u][0];
    }
  }
}

// Epilogue and store of the rows rank, rank + split, .. of a tile in shared memory, a warp per
// row (the row that fp8_add_parts gave the same lanes of some warp: the caller has
// synchronised). Lanes take four neighbouring columns, or, where those cannot be stored
// together, columns 32 apart. The loop is kept small: with the epilogue inlined per element
// and eight rows at a time its code ran from memory (1001 x 1371 x 1037: 25 us against 11.5).
template <typename T>
LTX_DEVICE void fp8_store_rows(const Epi<T>& epi, bool vec, T* __restrict__ C, int64_t ldc, int m0, int n0, int rows,
                               int cols, int rank, int split, const float* part) {
  const int lane = lane_id(), N = n0 + cols;
  vec = vec && cols % 4 == 0;
#pragma unroll 1
  for (int r = warp_id() * split + rank; r < rows; r += 6 * split) {
    const float* row = part + r * Fp8TileCfg::LD_PART;
    const int64_t m = int64_t(m0) + r;
    const int64_t sb = int64_t(int(m) / int(epi.rows_per_batch)), st = m - sb * epi.rows_per_batch;
    if (vec) {
      if (lane * 4 >= cols) continue;
      const float4 x = reinterpret_cast<const float4*>(row)[lane];
      float v[4] = {x.x, x.y, x.z, x.w};
      fp8_epilogue<T, 4>(epi, C + m * ldc, m, sb, st, n0 + lane * 4, v);
    } else {
      float v[4] = {row[lane], row[lane + 32], row[lane + 64], row[lane + 96]};
      fp8_epilogue<T, 4, 32>(epi, C + m * ldc, m, sb, st, n0 + lane, v, N);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(192, 2)
    gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                         T* __restrict__ C, int64_t ldc, int M, int N, int K, int split, int vec, Epi<T> epi) {
  using Cfg = Fp8TileCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t* sf_smem = smem + Cfg::RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf_smem + Cfg::STAGES * 2 * Cfg::SF);
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* tfull = empty + Cfg::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  // the CTAs of a cluster are neighbours in x: rank = blockIdx.x % split
  const int tile = int(blockIdx.x) / split, rank = int(blockIdx.x) - tile * split;
  const int n_tiles = (N + 127) / 128;
  const int m0 = (tile / n_tiles) * 128, n0 = (tile % n_tiles) * 128;
  const int k_blocks = (K + 127) / 128;
  const int kb0 = int(int64_t(k_blocks) * rank / split), kb1 = int(int64_t(k_blocks) * (rank + 1) / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  const bool staged = split > 1 || !vec;
  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int it = kb - kb0, s = it % Cfg::STAGES;
        if (!mbar_wait(&empty[s], (uint32_t(it / Cfg::STAGES) & 1) ^ 1, abort_flag)) break;
        uint8_t* st = smem + s * Cfg::STAGE_BYTES;
        const bool quad = kb == kb0 || (kb & 3) == 0;  // a new scale word
        mbar_arrive_expect_tx(&full[s], Cfg::STAGE_BYTES + (quad ? 2 * Cfg::SF : 0));
        tma_load_2d(st, &tmA, &full[s], kb * 128, m0);
        tma_load_2d(st + Cfg::SLAB, &tmB, &full[s], kb * 128, n0);
        if (quad) {
          tma_load_2d(sf_smem + s * 2 * Cfg::SF, &tmSA, &full[s], m0, kb >> 2);
          tma_load_2d(sf_smem + s * 2 * Cfg::SF + Cfg::SF, &tmSB, &full[s], n0, kb >> 2);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t lo0 = umma_desc_sw128_lo(smem_u32(smem)), sf0 = umma_desc_rows16_lo(smem_u32(sf_smem));
      int s = 0;
      uint32_t par = 0, accumulate = 0;
      for (int kb = kb0 & ~3; ok && kb < kb1; kb += 4) {  // by scale words
        const uint32_t sfa = tmem + 128u + uint32_t((kb >> 2) & 1) * 8u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kb + j >= kb0 && kb + j < kb1) {
            ok = ok && mbar_wait(&full[s], par, abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (j == 0 || kb + j == kb0) {
              const uint32_t sf = sf0 + uint32_t(s) * (2 * Cfg::SF / 16);
              tmem_cp_scales(sfa, umma_desc_rows16_of(sf));
              tmem_cp_scales(sfa + 4u, umma_desc_rows16_of(sf + Cfg::SF / 16));
            }
            const uint32_t lo = lo0 + uint32_t(s) * (Cfg::STAGE_BYTES / 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              umma_mx8_ss(tmem, umma_desc_sw128_of(lo + 2 * k), umma_desc_sw128_of(lo + Cfg::SLAB / 16 + 2 * k),
                          umma_idesc_mx8(128, 128, j), sfa, sfa + 4u, accumulate);
              accumulate = 1;
            }
            umma_commit(&empty[s]);
            if (++s == Cfg::STAGES) {
              s = 0;
              par ^= 1;
            }
          }
        }
      }
      if (ok) umma_commit(tfull);
    }
  } else {
    const int q = warp & 3;  // TMEM lane quadrant
    const uint32_t tquad = tmem + (uint32_t(q * 32) << 16);
    const int64_t m = int64_t(m0) + q * 32 + lane;
    const bool live = m < M;
    if (mbar_wait(tfull, 0, abort_flag)) {
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem) + (q * 32 + lane) * Cfg::LD_PART;
      const int64_t sb = int64_t(int(m) / int(epi.rows_per_batch)), st = m - sb * epi.rows_per_batch;
#pragma unroll 1
      for (int c0 = 0; c0 < 128 && n0 + c0 < N; c0 += 32) {
        uint32_t rr[32];
        tmem_read32(tquad + uint32_t(c0), rr);
        if (live && staged) {
          // every MMA of this CTA has read its operands: the ring is free
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(part + c0 + j) = make_uint4(rr[j], rr[j + 1], rr[j + 2], rr[j + 3]);
        } else if (live) {
#pragma unroll
          for (int j = 0; j < 32; j += 16) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(rr[j + e]);
            fp8_epilogue_cols<T>(epi, true, C + m * ldc, m, sb, st, n0 + c0 + j, N, v);
          }
        }
        __syncwarp();  // the next read is the whole warp's
      }
    }
  }
  __syncwarp();
  if (staged) {
    if (split > 1)
      cluster_sync_all();
    else
      __syncthreads();
    const int rows = min(128, M - m0), cols = min(128, N - n0);
    float* part = reinterpret_cast<float*>(smem);
    switch (split) {
      case 1: break;
      case 2: fp8_add_parts<2>(part, smem_u32(smem), rows, rank); break;
      case 4: fp8_add_parts<4>(part, smem_u32(smem), rows, rank); break;
      default: fp8_add_parts<8>(part, smem_u32(smem), rows, rank); break;
    }
    if (split > 1) cluster_sync_all();  // sums are in place, and no CTA reads another's part any more
    fp8_store_rows<T>(epi, vec, C, ldc, m0, n0, rows, cols, rank, split, part);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

// Large problems: a CTA pair (cluster of two SMs, cta_group::2 MMAs) per 256 x 256 tile,
// persistent over the tiles, N fastest so that the rows of A stay in L2. Each CTA loads its
// 128 rows of A and 128 of the 256 rows of W (32 KB per slab and SM for 512 clocks of MMA);
// its tensor memory holds its rows' scales and those of all 256 columns.
//
// Two 256-column accumulators and two scale buffers of 12 columns do not fit in 512, so the
// accumulators share 32 columns, [224, 256): the epilogue of a tile reads that slab first
// and lets the next tile's MMAs start behind it (`tover`), long before the whole
// accumulator is drained (`tempty`, which the tile after next waits for). Those arrivals
// cross to the leader without a release: they order tensor-memory reads, which
// tcgen05.wait and the fence have completed, and no other memory; with a cluster-scope
// release each cost 1.2 us behind the tile's stores (725 -> 635 clocks per slab at
// 12288 x 8192 x 2048).
struct Fp8PairCfg {
  static constexpr int STAGES = 6;
  static constexpr int SLAB = 128 * 128;
  static constexpr int SF_A = 512, SF_B = 1024;  // scale words of 128 / 256 rows, four slabs
  static constexpr int SF = SF_A + SF_B;
  static constexpr int RING = STAGES * 2 * SLAB;
  static constexpr int SMEM = RING + STAGES * SF + 256 + 1024;
  static constexpr uint32_t ACC1 = 224;    // accumulator 1 at [224, 480), accumulator 0 at [0, 256)
  static constexpr uint32_t SF_COL = 480;  // two buffers of 4 (A) + 8 (W) columns
};

// Warp 0 TMA, warp 1 MMA issuer (leader), warps 2-9 epilogue.
template <typename T>
__global__ void __launch_bounds__(320, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                         T* __restrict__ C, int64_t ldc, int M, int N, int K, int vec, Epi<T> epi) {
  using Cfg = Fp8PairCfg;
  constexpr int S = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint8_t* sf_smem = smem + Cfg::RING;
  uint64_t* full = reinterpret_cast<uint64_t*>(sf_smem + S * Cfg::SF);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* tover = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tover + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int n_tiles = (N + 255) / 256, num_tiles = ((M + 255) / 256) * n_tiles;
  const int k_blocks = (K + 127) / 128;
  const int tile0 = int(blockIdx.x >> 1), tile_step = int(gridDim.x >> 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 16);  // every epilogue warp of both CTAs
    }
    mbar_init(tover, 8);  // the four warps of both CTAs that read the shared slab
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmSA);
    tma_prefetch_desc(&tmSB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // both CTAs' barriers and tensor memory before any cross-CTA use
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      for (int tile = tile0; ok && tile < num_tiles; tile += tile_step) {
        const int m0 = (tile / n_tiles) * 256 + int(rank) * 128, n0 = (tile % n_tiles) * 256;
        for (int kb = 0; kb < k_blocks; ++kb, ++it) {
          const int s = it % S;
          ok = mbar_wait(&empty[s], (uint32_t(it / S) & 1) ^ 1, abort_flag);
          if (!ok) break;
          uint8_t* sa = smem + s * 2 * Cfg::SLAB;
          const uint32_t fb = mapa_shared(smem_u32(&full[s]), 0);  // both CTAs' bytes complete on the leader's
          const bool quad = (kb & 3) == 0;                             // a new scale word
          if (leader) mbar_arrive_expect_tx(&full[s], 4 * Cfg::SLAB + (quad ? 2 * Cfg::SF : 0));
          tma_load_2d_pair(sa, &tmA, fb, kb * 128, m0);
          tma_load_2d_pair(sa + Cfg::SLAB, &tmB, fb, kb * 128, n0 + int(rank) * 128);
          if (quad) {
            tma_load_2d_pair(sf_smem + s * Cfg::SF, &tmSA, fb, m0, kb >> 2);
            tma_load_2d_pair(sf_smem + s * Cfg::SF + Cfg::SF_A, &tmSB, fb, n0, kb >> 2);
          }
        }
      }
    }
  } else if (warp == 1) {
    // One thread issues every MMA, so its own instructions count: the descriptors' constant
    // halves are built once and stages and parities are kept, not divided out (0.185 ms ->
    // 0.15 ms at 12288 x 8192 x 2048, 986 -> 785 clocks per slab).
    if (lane == 0 && leader) {
      const uint32_t lo0 = umma_desc_sw128_lo(smem_u32(smem)), sf0 = umma_desc_rows16_lo(smem_u32(sf_smem));
      int s = 0, local = 0;
      uint32_t par = 0, sfa = tmem + Cfg::SF_COL;
      bool ok = true;
      for (int tile = tile0; ok && tile < num_tiles; tile += tile_step, ++local) {
        const int acc = local & 1;
        ok = mbar_wait(&tempty[acc], (uint32_t(local >> 1) & 1) ^ 1, abort_flag) &&
             (local == 0 || mbar_wait(tover, uint32_t(local - 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + (acc ? Cfg::ACC1 : 0u);
        uint32_t accumulate = 0;
        for (int kb = 0; kb < k_blocks; kb += 4) {
          const int n = min(4, k_blocks - kb);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < n) {
              ok = ok && mbar_wait(&full[s], par, abort_flag);
              if (!ok) break;
              tc_fence_after();
              if (j == 0) {
                const uint32_t sf = sf0 + uint32_t(s) * (Cfg::SF / 16);
                tmem_cp_scales_pair(sfa, umma_desc_rows16_of(sf));
                tmem_cp_scales_pair(sfa + 4u, umma_desc_rows16_of(sf + Cfg::SF_A / 16));
                tmem_cp_scales_pair(sfa + 8u, umma_desc_rows16_of(sf + Cfg::SF_A / 16 + 32));
              }
              const uint32_t lo = lo0 + uint32_t(s) * (2 * Cfg::SLAB / 16);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                umma_mx8_ss_pair(d, umma_desc_sw128_of(lo + 2 * k), umma_desc_sw128_of(lo + Cfg::SLAB / 16 + 2 * k),
                                 umma_idesc_mx8(256, 256, j), sfa, sfa + 4u, accumulate);
                accumulate = 1;
              }
              umma_commit_pair(&empty[s], 3);
              if (++s == S) {
                s = 0;
                par ^= 1;
              }
            }
          }
          if (!ok) break;
          sfa = 2 * (tmem + Cfg::SF_COL) + 12u - sfa;  // the other buffer
        }
        if (ok) umma_commit_pair(&tfull[acc], 3);
      }
    }
  } else {
    // Epilogue warps 2..9: TMEM lane quadrant warp % 4 (one accumulator row per thread),
    // column half (warp - 2) / 4.
    const int q = warp & 3, half = (warp - 2) >> 2;
    int local = 0;
    for (int tile = tile0; tile < num_tiles; tile += tile_step, ++local) {
      const int acc = local & 1;
      const int m0 = (tile / n_tiles) * 256 + int(rank) * 128, n0 = (tile % n_tiles) * 256;
      const int64_t m = int64_t(m0) + q * 32 + lane;
      const bool live = m < M;
      const int64_t sb = int64_t(int(m) / int(epi.rows_per_batch)), st = m - sb * epi.rows_per_batch;
      if (!mbar_wait(&tfull[acc], uint32_t(local >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      const uint32_t tbase = tmem + (acc ? Cfg::ACC1 : 0u) + (uint32_t(q * 32) << 16);
      // accumulator 0 shares its last slab (half 1), accumulator 1 its first (half 0)
      const bool shares = half == (acc ^ 1);
      T* crow = C + m * ldc;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        const int c0 = half * 128 + (acc ? j : 3 - j) * 32;
        uint32_t rr[32];
        tmem_read32(tbase + uint32_t(c0), rr);
        if (j == 0 && shares) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(tover), 0));
        }
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
          if (live && n0 + c0 + c < N) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(rr[c + e]);
            fp8_epilogue_cols<T>(epi, vec, crow, m, sb, st, n0 + c0 + c, N, v);
          }
        }
        __syncwarp();  // the next read is the whole warp's
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&tempty[acc]), 0));
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();  // no CTA of the pair leaves while the other may still signal its barriers
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Which kernel, and over how many CTAs of a cluster the tile kernel splits K. Microseconds
// measured on the B200 (graph replay, weights not in L2), at M x N x K:
//   tile kernel  4.0 + 0.37 per slab of a CTA, times the CTAs per SM; adding the parts of a
//                split costs 3.4 / 2.4 / 3.8 for 2 / 4 / 8 of them, 0.7 with few rows
//                (126 x 2048 x 2048: 10.0 whole, 10.5 / 7.8 / 9.0 split; 2 x 1024 x 8192: 29.2
//                whole, 16.7 / 10.2 / 7.2 split; 12288 x 2048 x 2048: 61.6)
//   CTA pairs    4.5 + 0.5 per tile and 0.4 per slab of a pair (1024 x 4096 x 4096: 16.9
//                against 29.6; 1024 x 1024 x 1024: 7.8 against 6.5)
// Outputs that cannot be stored 32 bytes at a time take the tile kernel's staging.
struct Fp8Plan {
  bool pair = false;
  int split = 1;
};
static thread_local int g_fp8_force_pair = -1;  // ltx_test_fp8_force_pair

inline Fp8Plan fp8_plan(int64_t M, int64_t N, int64_t K, bool vec, int sms) {
  const double kb = double((K + 127) / 128);
  const double tiles = double((M + 127) / 128) * double((N + 127) / 128);
  constexpr double kAdd[4] = {0.0, 3.4, 2.4, 3.8};
  Fp8Plan p;
  double best = 0;
  for (int i = 0, split = 1; i < 4; ++i, split *= 2) {
    if (split > 1 && (tiles * split > 2 * sms || kb < 2 * split)) break;
    const double us = 4.0 + std::ceil(kb / split) * 0.37 * std::max(1.0, tiles * split / sms) +
                      (i == 0 ? 0.0 : M > 16 ? kAdd[i] : 0.7);
    if (i == 0 || us < best) {
      best = us;
      p.split = split;
    }
  }
  const double pairs = std::ceil(double((M + 255) / 256) * double((N + 255) / 256) / (sms / 2));
  p.pair = vec && 4.5 + pairs * (0.5 + 0.4 * kb) < best;
  if (g_fp8_force_pair >= 0) p.pair = g_fp8_force_pair != 0;
  return p;
}

template <typename T>
void launch_linear_fp8(const void* A, int64_t lda, const void* As, const void* W, int64_t ldw, const void* Ws, T* C,
                       int64_t ldc, int64_t M, int64_t N, int64_t K, const Epi<T>& epi, bool vec, cudaStream_t s) {
  const auto [pair, split] = fp8_plan(M, N, K, vec, num_sms());
  const CUtensorMap ta = make_tmap_u8_2d(A, uint64_t(K), uint64_t(M), uint64_t(lda), 128);
  const CUtensorMap tb = make_tmap_u8_2d(W, uint64_t(K), uint64_t(N), uint64_t(ldw), 128);
  const uint64_t quads = uint64_t(fp8_quads(K));
  const CUtensorMap tsa = make_tmap_u32_2d(As, uint64_t(fp8_rows_padded(M)), quads, 128);
  const CUtensorMap tsb = make_tmap_u32_2d(Ws, uint64_t(fp8_rows_padded(N)), quads, pair ? 256 : 128);
  static std::atomic<uint64_t> smem_done[2] = {};
  if (pair) {
    auto kern = gemm_fp8_pair_kernel<T>;
    ensure_smem_limit(smem_done[1], kern, Fp8PairCfg::SMEM);
    const int64_t tiles = ((M + 255) / 256) * ((N + 255) / 256);
    LTX_UNSUPPORTED(tiles < (int64_t(1) << 31) - 65536, "too many tiles for one launch");
    const int64_t pairs = std::min<int64_t>(num_sms() / 2, tiles);
    launch_pdl(kern, dim3(unsigned(2 * pairs)), dim3(320), Fp8PairCfg::SMEM, s, 2, ta, tb, tsa, tsb, C, ldc, int(M),
               int(N), int(K), int(vec), epi);
    return;
  }
  auto kern = gemm_fp8_tile_kernel<T>;
  ensure_smem_limit(smem_done[0], kern, Fp8TileCfg::SMEM);
  const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
  LTX_UNSUPPORTED(tiles * split < (int64_t(1) << 31), "too many tiles for one launch");
  launch_pdl(kern, dim3(unsigned(tiles * split)), dim3(192), Fp8TileCfg::SMEM, s, unsigned(split), ta, tb, tsa, tsb, C,
             ldc, int(M), int(N), int(K), split, int(vec), epi);
}

// ---------------------------------------------------------------------------------
// One to eight rows (adaLN: one row per sample): the product is reading W once. One launch
// quantises the rows in every CTA (M * K values, from L2) and streams W through registers:
// a CTA takes 16 rows of W at a time, warp w of 8 the blocks w, w + 8, .. of 128 columns, so
// that a group's bytes are in flight at once; each block is four warp-level MMAs (16 rows of
// W by 8 of x, K = 32) from zero, and the sums are multiplied by both scales and added in
// fp32. A dot product does not depend on the order of its terms, so lane l feeds the MMAs
// the 32 contiguous bytes l % 4 of its rows' 128 (the same of W and of x). The eight warps'
// sums are added in order through shared memory. CUDA-core products, two rows of W per
// warp, took 14.3 us at 2 x 12288 x 2048 (unpacking e4m3 bounds them) and the tile kernel 13.
// ---------------------------------------------------------------------------------
LTX_DEVICE void mma_e4m3_16x8x32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kFp8RowsMax = 8;

// 32 bytes of a row of W from column c on, zeros from K on (the row's padding may hold any
// byte, and must not meet the MMA as NaN). wide: 32-byte aligned rows.
LTX_DEVICE void fp8_load_w32(const uint8_t* row, int c, int K, bool wide, uint32_t (&v)[8]) {
  if (wide && c + 32 <= K) {
    ldg_32b(row + c, v);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int at = c + 16 * h;
    const uint4 u = at < K ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0, 0, 0, 0);
    const uint32_t b[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int left = K - at - 4 * i;  // bytes of this word that exist
      v[4 * h + i] = left >= 4 ? b[i] : left <= 0 ? 0u : b[i] & ((1u << (8 * left)) - 1u);
    }
  }
}

template <typename T, typename X>
__global__ void __launch_bounds__(256, 2)
    linear_fp8_rows_kernel(const X* __restrict__ x, int64_t ldx, int vec_x, const uint8_t* __restrict__ W, int64_t ldw,
                           int wide, const uint32_t* __restrict__ Ws, int64_t w_padded, T* __restrict__ C, int64_t ldc,
                           int M, int N, int K, Epi<T> epi) {
  extern __shared__ __align__(16) uint8_t rows_smem[];
  __shared__ float part[2][8][16][kFp8RowsMax];
  const int quads = (K + kFp8Quad - 1) / kFp8Quad, blocks = (K + kFp8Block - 1) / kFp8Block;
  const int ldxq = quads * kFp8Quad + 16;                             // no bank conflicts between rows
  float* sa = reinterpret_cast<float*>(rows_smem + M * ldxq);         // [M][quads * 4]
  const int lane = lane_id(), warp = warp_id(), row = lane >> 2, piece = lane & 3;
  pdl_wait();
  pdl_trigger();

  constexpr int PRE = 2;  // blocks per warp in flight
  uint32_t w[PRE][2][8], sw[PRE][2];
  // blocks warp + 8 i, i in [i0, i0 + PRE), of the 16 rows from n0 on
  auto fetch = [&](int n0, int i0) {
#pragma unroll
    for (int j = 0; j < PRE; ++j) {
      const int kb = warp + 8 * (i0 + j);
      if (kb >= blocks) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t n = min(n0 + row + 8 * h, N - 1);
        fp8_load_w32(W + n * ldw, kb * kFp8Block + piece * 32, K, wide, w[j][h]);
        sw[j][h] = Ws[fp8_word(n, kb >> 2, w_padded)];
      }
    }
  };
  unsigned n0 = blockIdx.x * 16;  // unsigned: the step behind the last rows may pass 2^31
  fetch(n0, 0);
  for (int i = warp; i < M * quads; i += 8) {
    const int m = i / quads, kq = i - m * quads;
    float v[16];
    load16<X>(x + m * ldx, kq * kFp8Quad + lane * 16, K, vec_x, v);
    uint4 q;
    const int code = fp8_quantize16(v, q);
    *reinterpret_cast<uint4*>(rows_smem + m * ldxq + kq * kFp8Quad + lane * 16) = q;
    if ((lane & 7) == 0) sa[i * 4 + (lane >> 3)] = fp8_scale(code);
  }
  __syncthreads();
  const int per_warp = (blocks - warp + 7) / 8;
  for (int buf = 0; n0 < unsigned(N); n0 += gridDim.x * 16, buf ^= 1) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < per_warp; i0 += PRE) {
#pragma unroll
      for (int j = 0; j < PRE; ++j) {
        const int kb = warp + 8 * (i0 + j);
        if (kb >= blocks) break;
        uint32_t b[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (row < M) {
          const uint4* p = reinterpret_cast<const uint4*>(rows_smem + row * ldxq + kb * kFp8Block + piece * 32);
          const uint4 u0 = p[0], u1 = p[1];
          b[0] = u0.x; b[1] = u0.y; b[2] = u0.z; b[3] = u0.w;
          b[4] = u1.x; b[5] = u1.y; b[6] = u1.z; b[7] = u1.w;
        }
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 8; t += 2)
          mma_e4m3_16x8x32(c, w[j][0][t], w[j][1][t], w[j][0][t + 1], w[j][1][t + 1], b[t], b[t + 1]);
        // c: (W row `row`, x rows 2 piece and 2 piece + 1), then the same of W row `row` + 8
        const float a0 = 2 * piece < M ? sa[2 * piece * quads * 4 + kb] : 0.f;
        const float a1 = 2 * piece + 1 < M ? sa[(2 * piece + 1) * quads * 4 + kb] : 0.f;
        const float s0 = fp8_scale((sw[j][0] >> (8 * (kb & 3))) & 255u);
        const float s1 = fp8_scale((sw[j][1] >> (8 * (kb & 3))) & 255u);
        // The scales' product first: it is exact, and infinite or zero only where the result is
        // above 2^110 or below 2^-124 as well. c times one scale (2^118) could leave fp32 before
        // the other brings it back.
        acc[0] = fmaf(c[0], a0 * s0, acc[0]);
        acc[1] = fmaf(c[1], a1 * s0, acc[1]);
        acc[2] = fmaf(c[2], a0 * s1, acc[2]);
        acc[3] = fmaf(c[3], a1 * s1, acc[3]);
      }
      if (i0 + PRE < per_warp) fetch(n0, i0 + PRE);
    }
    const unsigned next = n0 + gridDim.x * 16;
    if (next < unsigned(N)) fetch(next, 0);
    *reinterpret_cast<float2*>(&part[buf][warp][row][2 * piece]) = make_float2(acc[0], acc[1]);
    *reinterpret_cast<float2*>(&part[buf][warp][row + 8][2 * piece]) = make_float2(acc[2], acc[3]);
    __syncthreads();  // the other buffer is rewritten only behind the next one
    for (int i = threadIdx.x; i < 16 * M; i += 256) {
      const int m = i >> 4, r = i & 15;
      if (n0 + r < unsigned(N)) {
        float v[1] = {0.f};
#pragma unroll
        for (int p = 0; p < 8; ++p) v[0] += part[buf][p][r][m];
        const int64_t sb = m / epi.rows_per_batch, st = m - sb * epi.rows_per_batch;
        fp8_epilogue<T, 1>(epi, C + m * ldc, m, sb, st, n0 + r, v);
      }
    }
  }
}

inline int64_t fp8_rows_smem(int64_t M, int64_t K) { return M * (fp8_quads(K) * (512 + 16) + 16); }
// The streaming kernel, as long as two CTAs' quantised rows fit in an SM's shared memory.
inline bool fp8_use_rows(int64_t M, int64_t K) {
  return M <= kFp8RowsMax && fp8_rows_smem(M, K) <= 96 * 1024 && g_fp8_force_pair < 0;
}

template <typename T, typename X>
void launch_fp8_rows(const X* x, int64_t ldx, const void* W, int64_t ldw, const void* Ws, T* C, int64_t ldc, int64_t M,
                     int64_t N, int64_t K, const Epi<T>& epi, cudaStream_t s) {
  const int smem = int(fp8_rows_smem(M, K));
  auto kern = linear_fp8_rows_kernel<T, X>;
  static std::atomic<uint64_t> smem_done{0};
  ensure_smem_limit(smem_done, kern, 96 * 1024);
  const int64_t grid = std::min<int64_t>((N + 15) / 16, int64_t(num_sms()) * 2);
  const int vec = row_vec(x, ldx);
  const int wide = reinterpret_cast<uintptr_t>(W) % 32 == 0 && ldw % 32 == 0;
  launch_pdl(kern, dim3(unsigned(grid)), dim3(256), size_t(smem), s, 1, x, ldx, vec, static_cast<const uint8_t*>(W), ldw,
             wide, static_cast<const uint32_t*>(Ws), fp8_rows_padded(N), C, ldc, int(M), int(N), int(K), epi);
}

}  // namespace detail
}  // namespace ltx

using namespace ltx;
using namespace ltx::detail;

namespace {

// ltx_epilogue as the 8-bit products take it: the same fields as make_epi, but vectors of
// any alignment and stride (a column count that is not a multiple of 8 has them).
// `vec` tells whether every vector may be read 32 bytes at a time.
template <typename T>
Epi<T> make_epi_any(const ltx_epilogue* p, int64_t N, bool& vec) {
  Epi<T> e;
  vec = true;
  if (p == nullptr) return e;
  auto take = [&](const void* ptr) {
    if (reinterpret_cast<uintptr_t>(ptr) % sizeof(T))
      throw ApiError{LTX_ERR_INVALID, "an epilogue vector is not aligned to its type"};
    if (reinterpret_cast<uintptr_t>(ptr) % 32) vec = false;
    return static_cast<const T*>(ptr);
  };
  if (p->kind < LTX_EPI_NONE || p->kind > LTX_EPI_ROW_MASK_ADD)
    throw ApiError{LTX_ERR_INVALID, "unknown epilogue kind"};
  if (p->silu_input) throw ApiError{LTX_ERR_INVALID, "silu_input is not an epilogue of 8-bit rows"};
  e.kind = p->kind;
  e.bias = take(p->bias);
  // rows are below 2^31: a longer sample is all of them (the kernels divide in 32 bits)
  e.rows_per_batch = p->rows_per_batch > 0 ? std::min<int64_t>(p->rows_per_batch, INT32_MAX) : 1;
  if (e.kind == LTX_EPI_GATE_RESIDUAL) {
    if (p->residual == nullptr) throw ApiError{LTX_ERR_INVALID, "GATE_RESIDUAL needs a residual"};
    if (p->ld_residual < N) throw ApiError{LTX_ERR_INVALID, "ld_residual must hold the columns"};
    e.residual = take(p->residual);
    e.ld_res = p->ld_residual;
    if (e.ld_res % 16) vec = false;
    const ltx_modulation& g = p->gate;
    if (g.has_scale && (g.table != nullptr || g.mod != nullptr)) {
      e.gate.table = take(g.table);
      e.gate.mod = take(g.mod);
      e.gate.ldb = g.mod_ld_batch;
      e.gate.ldt = g.mod_ld_tok;
      e.gate.toff = g.scale_table_off;
      e.gate.moff = g.scale_mod_off;
      e.gate.on = 1;
      if ((e.gate.ldb % 16) || (e.gate.ldt % 16) || (e.gate.toff % 16) || (e.gate.moff % 16)) vec = false;
    }
  }
  if (e.kind == LTX_EPI_ROW_MASK_ADD) {
    if (p->row_mask == nullptr || p->row_vec == nullptr)
      throw ApiError{LTX_ERR_INVALID, "ROW_MASK_ADD needs row_mask and row_vec"};
    if (reinterpret_cast<uintptr_t>(p->row_mask) % 4)
      throw ApiError{LTX_ERR_INVALID, "row_mask is not aligned to its type"};
    e.row_mask = p->row_mask;
    e.row_vec = take(p->row_vec);
  }
  return e;
}

// Checks of one operand in the 8-bit row format.
void check_fp8_rows(const void* q, int64_t ldq, const void* scales, int64_t rows, int64_t cols, const char* what) {
  auto need = [&](bool ok, const char* msg) {
    if (!ok) throw ApiError{LTX_ERR_INVALID, std::string(what) + ": " + msg};
  };
  need(q != nullptr && scales != nullptr, "data and scales must be non-NULL");
  need(rows > 0 && cols > 0, "rows and columns must be positive");
  need(rows < (int64_t(1) << 31) - 256 && cols < (int64_t(1) << 31) - 512, "size out of range");
  need(ldq % 16 == 0 && ldq >= cols, "the row stride must be a multiple of 16 bytes and hold the columns");
  need(reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0,
       "data and scales must be 16-byte aligned");
}

unsigned grid_for(int64_t blocks) {
  if (blocks >= (int64_t(1) << 31)) throw ApiError{LTX_ERR_UNSUPPORTED, "too many rows and columns for one launch"};
  return unsigned(blocks);
}

}  // namespace

extern "C" size_t ltx_fp8_scale_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return size_t(fp8_rows_padded(rows)) * size_t(fp8_quads(cols)) * 4;
}

static void launch_quantize(const void* x, int64_t ldx, int64_t rows, int64_t cols, void* q, int64_t ldq, void* scales,
                            int dtype, cudaStream_t s) {
  const int quads = int(fp8_quads(cols));
  const unsigned grid = grid_for((rows * quads + 7) / 8);
  auto run = [&](auto* xp, auto kern) {
    launch_pdl(kern, dim3(grid), dim3(256), 0, s, 1, xp, ldx, rows, cols, quads, row_vec(xp, ldx), static_cast<uint8_t*>(q), ldq,
               static_cast<uint32_t*>(scales), fp8_rows_padded(rows));
  };
  if (dtype == LTX_F32)
    run(static_cast<const float*>(x), quantize_fp8_kernel<float>);
  else
    run(static_cast<const __nv_bfloat16*>(x), quantize_fp8_kernel<__nv_bfloat16>);
}

extern "C" int ltx_quantize_fp8(const void* x, int64_t ldx, int64_t rows, int64_t cols, void* q, int64_t ldq,
                                void* scales, int dtype, void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(x != nullptr, "x must be non-NULL");
  check_fp8_rows(q, ldq, scales, rows, cols, "ltx_quantize_fp8: output");
  LTX_REQUIRE(ldx >= cols, "ldx must hold the columns");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(x) % (dtype == LTX_F32 ? 4 : 2) == 0, "x is not aligned to its type");
  launch_quantize(x, ldx, rows, cols, q, ldq, scales, dtype, static_cast<cudaStream_t>(stream));
  LTX_API_END
}

extern "C" int ltx_dequantize_fp8(const void* q, int64_t ldq, const void* scales, int64_t rows, int64_t cols, void* x,
                                  int64_t ldx, int dtype, void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(x != nullptr, "x must be non-NULL");
  check_fp8_rows(q, ldq, scales, rows, cols, "ltx_dequantize_fp8: input");
  LTX_REQUIRE(ldx >= cols, "ldx must hold the columns");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(x) % (dtype == LTX_F32 ? 4 : 2) == 0, "x is not aligned to its type");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int quads = int(fp8_quads(cols));
  const unsigned grid = grid_for(((rows + kDequantRows - 1) / kDequantRows * quads + 7) / 8);
  auto run = [&](auto* xp, auto kern) {
    launch_pdl(kern, dim3(grid), dim3(256), 0, s, 1, static_cast<const uint8_t*>(q), ldq,
               static_cast<const uint32_t*>(scales), fp8_rows_padded(rows), rows, cols, quads, row_vec(xp, ldx), xp,
               ldx);
  };
  if (dtype == LTX_F32)
    run(static_cast<float*>(x), dequantize_fp8_kernel<float>);
  else
    run(static_cast<__nv_bfloat16*>(x), dequantize_fp8_kernel<__nv_bfloat16>);
  LTX_API_END
}

extern "C" int ltx_fp8_pack_scales(const float* s, int64_t ld, int64_t rows, int64_t cols, void* scales,
                                   void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(s != nullptr && scales != nullptr, "s and scales must be non-NULL");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(s) % 4 == 0, "s is not aligned to its type");
  LTX_REQUIRE(rows > 0 && cols > 0, "rows and columns must be positive");
  LTX_REQUIRE(rows < (int64_t(1) << 31) - 256 && cols < (int64_t(1) << 31) - 512, "size out of range");
  const int64_t blocks = (cols + kFp8Block - 1) / kFp8Block;
  LTX_REQUIRE(ld >= blocks, "ld must hold one scale per 128 columns");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(scales) % 16 == 0, "scales must be 16-byte aligned");
  const int quads = int(fp8_quads(cols));
  launch_pdl(fp8_pack_scales_kernel, dim3(grid_for((rows * quads + 255) / 256)), dim3(256), 0,
             static_cast<cudaStream_t>(stream), 1, s, ld, rows, blocks, quads, static_cast<uint32_t*>(scales),
             fp8_rows_padded(rows));
  LTX_API_END
}

extern "C" int ltx_norm_modulate_fp8(const void* x, int64_t ldx, void* q, int64_t ldq, void* scales, int64_t rows,
                                     int64_t rows_per_batch, int D, int norm_kind, float eps,
                                     const ltx_modulation* mod, int dtype, void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(x != nullptr, "x must be non-NULL");
  LTX_REQUIRE(D > 0 && D % 8 == 0, "D must be a positive multiple of 8");
  check_fp8_rows(q, ldq, scales, rows, D, "ltx_norm_modulate_fp8: output");
  LTX_UNSUPPORTED(D <= 16384, "D must be at most 16384");
  LTX_REQUIRE(ldx % 8 == 0 && ldx >= D, "ldx must be a multiple of 8 and >= D");
  LTX_REQUIRE(rows_per_batch > 0, "rows_per_batch must be positive");
  LTX_REQUIRE(norm_kind == LTX_NORM_RMS || norm_kind == LTX_NORM_LAYER || norm_kind == LTX_NORM_NONE, "bad norm_kind");
  check_vec_ptr(x, "x");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* xp) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(xp)>>;
    const ModVec<T> sh = make_modvec<T>(mod, 0), sc = make_modvec<T>(mod, 1);
    const bool per_tok = (sh.on && sh.mod && sh.ldt != 0) || (sc.on && sc.mod && sc.ldt != 0);
    const int wr = (D + kFp8Quad - 1) / kFp8Quad, groups = std::max(1, 8 / wr);
    const int threads = 32 * wr * groups;  // <= 256 up to 4096 columns
    const bool hoist = !per_tok && threads <= 512;
    // as many CTAs as the SMs hold, each an even share of one sample's rows
    const int64_t rpb = std::min(rows_per_batch, rows), samples = (rows + rows_per_batch - 1) / rows_per_batch;
    const int64_t target = int64_t(num_sms()) * (threads <= 256 ? 3 * 256 / threads : threads <= 512 ? 1 : 2);
    const int64_t per = std::min<int64_t>(rpb, std::max<int64_t>(groups, (rows + target - 1) / target));
    const int64_t chunks = (rpb + per - 1) / per;
    const unsigned grid = grid_for(samples * chunks);
    auto go = [&](auto kern) {
      launch_pdl(kern, dim3(grid), dim3(unsigned(threads)), 0, s, 1, xp, ldx, row_vec(xp, ldx), rows, rows_per_batch, D,
                 wr, int(chunks), int(per), eps, sh, sc, static_cast<uint8_t*>(q), ldq, static_cast<uint32_t*>(scales),
                 fp8_rows_padded(rows));
    };
    auto kind = [&](auto kc) {
      constexpr int KIND = decltype(kc)::value;
      if (hoist && threads <= 256)
        go(norm_modulate_fp8_kernel<T, KIND, true, 256>);
      else if (hoist)
        go(norm_modulate_fp8_kernel<T, KIND, true, 512>);
      else if (threads <= 256)
        go(norm_modulate_fp8_kernel<T, KIND, false, 256>);
      else
        go(norm_modulate_fp8_kernel<T, KIND, false, 1024>);
    };
    switch (norm_kind) {
      case LTX_NORM_RMS: kind(std::integral_constant<int, LTX_NORM_RMS>{}); break;
      case LTX_NORM_LAYER: kind(std::integral_constant<int, LTX_NORM_LAYER>{}); break;
      default: kind(std::integral_constant<int, LTX_NORM_NONE>{}); break;
    }
  };
  if (dtype == LTX_F32)
    run(static_cast<const float*>(x));
  else
    run(static_cast<const __nv_bfloat16*>(x));
  LTX_API_END
}

extern "C" int ltx_linear_fp8(const void* A, int64_t lda, const void* a_scales, const void* W, int64_t ldw,
                              const void* w_scales, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K,
                              const ltx_epilogue* epi, int dtype, void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(C != nullptr, "C must be non-NULL");
  LTX_REQUIRE(M > 0 && N > 0 && K > 0, "M, N, K must be positive");
  check_fp8_rows(A, lda, a_scales, M, K, "ltx_linear_fp8: A");
  check_fp8_rows(W, ldw, w_scales, N, K, "ltx_linear_fp8: W");
  LTX_REQUIRE(ldc >= N, "ldc must hold the columns");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(C) % (dtype == LTX_F32 ? 4 : 2) == 0, "C is not aligned to its type");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto run = [&](auto* cp) {
    using T = std::remove_pointer_t<decltype(cp)>;
    bool vec;
    const Epi<T> e = make_epi_any<T>(epi, N, vec);
    vec = vec && reinterpret_cast<uintptr_t>(C) % 32 == 0 && ldc % 16 == 0;
    launch_linear_fp8<T>(A, lda, a_scales, W, ldw, w_scales, cp, ldc, M, N, K, e, vec, s);
  };
  if (dtype == LTX_F32)
    run(static_cast<float*>(C));
  else
    run(static_cast<__nv_bfloat16*>(C));
  LTX_CUDA(cudaGetLastError());
  LTX_API_END
}

// Workspace of ltx_quantize_linear_fp8: the quantised rows' data, then their scales.
static size_t quantized_data_bytes(int64_t M, int64_t K) { return size_t(M) * size_t((K + 15) / 16 * 16); }
static size_t quantized_bytes(int64_t M, int64_t K) { return quantized_data_bytes(M, K) + ltx_fp8_scale_bytes(M, K); }

extern "C" size_t ltx_quantize_linear_fp8_workspace_bytes(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0 || fp8_use_rows(M, K)) return 0;
  return quantized_bytes(M, K);
}

// Whether any of M rows of `a` (na bytes, lda between rows) shares a byte with one of `b`.
static bool rows_overlap(const void* a, int64_t lda, int64_t na, const void* b, int64_t ldb, int64_t nb, int64_t M) {
  const intptr_t pa = reinterpret_cast<intptr_t>(a), pb = reinterpret_cast<intptr_t>(b);
  for (int64_t i = 0; i < M; ++i)
    for (int64_t j = 0; j < M; ++j)
      if (pa + i * lda < pb + j * ldb + nb && pb + j * ldb < pa + i * lda + na) return true;
  return false;
}

extern "C" int ltx_quantize_linear_fp8(const void* x, int64_t ldx, int x_dtype, const void* W, int64_t ldw,
                                       const void* w_scales, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K,
                                       const ltx_epilogue* epi, void* workspace, size_t workspace_bytes, int dtype,
                                       void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(x_dtype == LTX_F32 || x_dtype == LTX_BF16, "x_dtype must be F32 or BF16");
  LTX_REQUIRE(x != nullptr && C != nullptr, "x and C must be non-NULL");
  LTX_REQUIRE(M > 0 && N > 0 && K > 0, "M, N, K must be positive");
  LTX_REQUIRE(M < (int64_t(1) << 31) - 256, "size out of range");
  check_fp8_rows(W, ldw, w_scales, N, K, "ltx_quantize_linear_fp8: W");
  LTX_REQUIRE(ldx >= K, "ldx must hold the columns");
  LTX_REQUIRE(ldc >= N, "ldc must hold the columns");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(x) % (x_dtype == LTX_F32 ? 4 : 2) == 0, "x is not aligned to its type");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(C) % (dtype == LTX_F32 ? 4 : 2) == 0, "C is not aligned to its type");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // Every CTA of the streaming kernel quantises x for itself, at its own time: the result must
  // not overwrite x before the last of them has.
  const int64_t xs = x_dtype == LTX_F32 ? 4 : 2, cs = dtype == LTX_F32 ? 4 : 2;
  if (!fp8_use_rows(M, K) || rows_overlap(x, ldx * xs, K * xs, C, ldc * cs, N * cs, M)) {
    LTX_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                    workspace_bytes >= quantized_bytes(M, K),
                "the workspace must be 16-byte aligned and hold the 8-bit rows of x: "
                "ltx_quantize_linear_fp8_workspace_bytes(M, K) bytes, and where C overlaps x M * (K rounded up to 16) "
                "+ ltx_fp8_scale_bytes(M, K) for any M");
    const int64_t ldq = (K + 15) / 16 * 16;
    void* scales = static_cast<char*>(workspace) + quantized_data_bytes(M, K);
    bool unused;  // the epilogue is checked before the first launch
    if (dtype == LTX_F32)
      make_epi_any<float>(epi, N, unused);
    else
      make_epi_any<__nv_bfloat16>(epi, N, unused);
    launch_quantize(x, ldx, M, K, workspace, ldq, scales, x_dtype, s);
    return ltx_linear_fp8(workspace, ldq, scales, W, ldw, w_scales, C, ldc, M, N, K, epi, dtype, stream);
  }
  auto run = [&](auto* xp, auto* cp) {
    using T = std::remove_pointer_t<decltype(cp)>;
    bool unused;
    launch_fp8_rows(xp, ldx, W, ldw, w_scales, cp, ldc, M, N, K, make_epi_any<T>(epi, N, unused), s);
  };
  auto run_c = [&](auto* xp) {
    if (dtype == LTX_F32)
      run(xp, static_cast<float*>(C));
    else
      run(xp, static_cast<__nv_bfloat16*>(C));
  };
  if (x_dtype == LTX_F32)
    run_c(static_cast<const float*>(x));
  else
    run_c(static_cast<const __nv_bfloat16*>(x));
  LTX_API_END
}

extern "C" int ltx_test_fp8_force_pair(int pair) {
  LTX_API_BEGIN
  LTX_REQUIRE(pair >= -1 && pair <= 1, "pair must be -1, 0 or 1");
  g_fp8_force_pair = pair;
  LTX_API_END
}
