// Rows in 8-bit floating point (fp8.cuh) and the linear layers on them:
//   ltx_quantize_fp8, ltx_dequantize_fp8, ltx_fp8_pack_scales   the format
//   ltx_norm_modulate_fp8   norm + adaLN modulation written as 8-bit rows
//   ltx_linear_fp8          C = epilogue(A W^T), A and W 8-bit rows
// None has a counterpart in the reference, which runs its linear layers in bf16
// (ltx_nn.py:126-158, 188-192, 244-245).
#include "fp8.cuh"

namespace ltx {
namespace detail {

// 16 consecutive columns [c, c + 16) of a row, zeros from `cols` on. `vec`: the row is
// 16-byte aligned and whole groups of 8 columns may be loaded at once.
template <typename T>
LTX_DEVICE void load16(const T* row, int64_t c, int64_t cols, bool vec, float (&v)[16]) {
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

// One warp per (row, 512 columns): two 16-byte loads and one 16-byte store per lane.
template <typename T>
__global__ void __launch_bounds__(256) quantize_fp8_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
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
  const uint32_t word = fp8_quad_word(code);
  if (c < cols) *reinterpret_cast<uint4*>(q + r * ldq + c) = out;
  if (lane_id() == 0) scales[fp8_word(r, kq, rows_padded)] = word;
}

// One thread per 8 columns.
template <typename T>
__global__ void __launch_bounds__(256) dequantize_fp8_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                             const uint32_t* __restrict__ scales, int64_t rows_padded,
                                                             int64_t rows, int64_t cols, int vec, T* __restrict__ x,
                                                             int64_t ldx) {
  pdl_wait();
  pdl_trigger();
  const int64_t per_row = (cols + 7) / 8;
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= rows * per_row) return;
  const int64_t r = i / per_row, c = (i - r * per_row) * 8;
  const uint32_t word = scales[fp8_word(r, c / kFp8Quad, rows_padded)];
  const float s = fp8_scale((word >> (8 * ((c / kFp8Block) & 3))) & 255);
  const uint2 w = *reinterpret_cast<const uint2*>(q + r * ldq + c);  // ldq % 16 == 0: in the padded row
  float v[8];
  fp8_unpack2(w.x, v[0], v[1]);
  fp8_unpack2(w.x >> 16, v[2], v[3]);
  fp8_unpack2(w.y, v[4], v[5]);
  fp8_unpack2(w.y >> 16, v[6], v[7]);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] *= s;
  if (vec && c + 8 <= cols) {
    st8<T>(x + r * ldx + c, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (c + k < cols) st_elem<T>(x + r * ldx + c + k, v[k]);
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

// y = norm(x) * (1 + scale) + shift in fp32, quantised once. One CTA per row, one warp
// per 512 columns, 16 columns per lane.
template <typename T>
__global__ void __launch_bounds__(1024) norm_modulate_fp8_kernel(const T* __restrict__ x, int64_t ldx,
                                                                 int64_t rows_per_batch, int D, int kind, float eps,
                                                                 ModVec<T> shift, ModVec<T> scale,
                                                                 uint8_t* __restrict__ q, int64_t ldq,
                                                                 uint32_t* __restrict__ scales, int64_t rows_padded) {
  __shared__ float red[32];
  pdl_wait();
  pdl_trigger();
  const int64_t row = blockIdx.x;
  const int64_t b = row / rows_per_batch, t = row - b * rows_per_batch;
  const int c = threadIdx.x * 16;
  float v[16];
  load16<T>(x + row * ldx, c, D, true, v);
  float mean = 0.f, rstd = 1.f;
  if (kind != LTX_NORM_NONE) {
    if (kind == LTX_NORM_LAYER) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += v[i];
      mean = block_sum(s, red) / float(D);
    }
    float s2 = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = c + i < D ? v[i] - mean : 0.f;
      s2 = fmaf(d, d, s2);
    }
    rstd = 1.f / sqrtf(block_sum(s2, red) / float(D) + eps);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float sc[8], sh[8];
    const bool in = c + 8 * h < D;
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] = sh[i] = 0.f;
    if (in && scale.on) modvec8<T>(scale, b, t, c + 8 * h, sc);
    if (in && shift.on) modvec8<T>(shift, b, t, c + 8 * h, sh);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = (v[8 * h + i] - mean) * rstd;
      v[8 * h + i] = in ? fmaf(y, 1.f + sc[i], sh[i]) : 0.f;
    }
  }
  uint4 out;
  const int code = fp8_quantize16(v, out);
  const uint32_t word = fp8_quad_word(code);
  if (c < D) *reinterpret_cast<uint4*>(q + row * ldq + c) = out;
  if (lane_id() == 0) scales[fp8_word(row, warp_id(), rows_padded)] = word;
}

// GELU (tanh form) as v * sigmoid(2 z), z = sqrt(2/pi) (v + 0.044715 v^3): one exponential
// and one division, accurate to a few fp32 units in the last place.
LTX_DEVICE float gelu_sigmoid(float v) {
  const float z2 = 1.5957691216057308f * fmaf(0.044715f * v * v, v, v);
  return __fdividef(v, 1.f + __expf(-z2));
}

// Epilogue of one accumulator in fp32, rounded once on the store:
// v + bias, then the activation, residual + gate * v, or v + row_vec on marked rows.
template <typename T>
LTX_DEVICE float fp8_epilogue1(const Epi<T>& e, int64_t row, int64_t col, float v) {
  if (e.bias) v += ld_elem<T>(e.bias + col);
  switch (e.kind) {
    case LTX_EPI_GELU_TANH:
      return gelu_sigmoid(v);
    case LTX_EPI_SILU:
      return __fdividef(v, 1.f + __expf(-v));
    case LTX_EPI_GATE_RESIDUAL: {
      float g = 1.f;
      if (e.gate.on) {
        const int64_t b = row / e.rows_per_batch, t = row - b * e.rows_per_batch;
        g = 0.f;
        if (e.gate.table) g += ld_elem<T>(e.gate.table + e.gate.toff + col);
        if (e.gate.mod) g += ld_elem<T>(e.gate.mod + b * e.gate.ldb + t * e.gate.ldt + e.gate.moff + col);
      }
      return fmaf(g, v, ld_elem<T>(e.residual + row * e.ld_res + col));
    }
    case LTX_EPI_ROW_MASK_ADD:
      return e.row_mask[row] > 0.f ? v + ld_elem<T>(e.row_vec + col) : v;
    default:
      return v;
  }
}

// Plain form of the product: 64x64 tile, 32 columns of K at a time, values scaled as they
// are staged in shared memory, fp32 sums.
template <typename T>
__global__ void __launch_bounds__(256)
    linear_fp8_simt_kernel(const uint8_t* __restrict__ A, int64_t lda, const uint32_t* __restrict__ As,
                           int64_t a_padded, const uint8_t* __restrict__ W, int64_t ldw,
                           const uint32_t* __restrict__ Ws, int64_t w_padded, T* __restrict__ C, int64_t ldc, int M,
                           int N, int K, Epi<T> epi) {
  __shared__ float sa[32][64 + 4];
  __shared__ float sw[32][64 + 4];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t m0 = int64_t(blockIdx.y) * 64, n0 = int64_t(blockIdx.x) * 64;
  float acc[4][4] = {};
  auto value = [&](const uint8_t* p, int64_t ld, const uint32_t* s, int64_t padded, int64_t r, int k) {
    float lo, hi;
    fp8_unpack2(p[r * ld + k], lo, hi);
    const uint32_t word = s[fp8_word(r, k / kFp8Quad, padded)];
    return lo * fp8_scale((word >> (8 * ((k / kFp8Block) & 3))) & 255);
  };
  for (int k0 = 0; k0 < K; k0 += 32) {
    for (int e = tid; e < 64 * 32; e += 256) {
      const int r = e >> 5, kk = e & 31;
      const bool in = k0 + kk < K;
      sa[kk][r] = in && m0 + r < M ? value(A, lda, As, a_padded, m0 + r, k0 + kk) : 0.f;
      sw[kk][r] = in && n0 + r < N ? value(W, ldw, Ws, w_padded, n0 + r, k0 + kk) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < 32; ++kk) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[kk][ty * 4 + i], sw[kk][tx * 4 + j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n < N) st_elem<T>(C + m * ldc + n, fp8_epilogue1<T>(epi, m, n, acc[i][j]));
    }
  }
}

}  // namespace detail
}  // namespace ltx

using namespace ltx;
using namespace ltx::detail;

namespace {

// ltx_epilogue as the 8-bit products take it: the same fields as make_epi, but vectors of
// any alignment and stride (a column count that is not a multiple of 8 has them).
// `vec` tells whether every vector may be read 16 bytes at a time.
template <typename T>
Epi<T> make_epi_any(const ltx_epilogue* p, int64_t N, bool& vec) {
  Epi<T> e;
  vec = true;
  if (p == nullptr) return e;
  auto take = [&](const void* ptr) {
    if (reinterpret_cast<uintptr_t>(ptr) % sizeof(T))
      throw ApiError{LTX_ERR_INVALID, "an epilogue vector is not aligned to its type"};
    if (reinterpret_cast<uintptr_t>(ptr) % 16) vec = false;
    return static_cast<const T*>(ptr);
  };
  if (p->kind < LTX_EPI_NONE || p->kind > LTX_EPI_ROW_MASK_ADD)
    throw ApiError{LTX_ERR_INVALID, "unknown epilogue kind"};
  if (p->silu_input) throw ApiError{LTX_ERR_INVALID, "silu_input is not an epilogue of 8-bit rows"};
  e.kind = p->kind;
  e.bias = take(p->bias);
  e.rows_per_batch = p->rows_per_batch > 0 ? p->rows_per_batch : 1;
  if (e.kind == LTX_EPI_GATE_RESIDUAL) {
    if (p->residual == nullptr) throw ApiError{LTX_ERR_INVALID, "GATE_RESIDUAL needs a residual"};
    if (p->ld_residual < N) throw ApiError{LTX_ERR_INVALID, "ld_residual must hold the columns"};
    e.residual = take(p->residual);
    e.ld_res = p->ld_residual;
    if (e.ld_res % 8) vec = false;
    const ltx_modulation& g = p->gate;
    if (g.has_scale && (g.table != nullptr || g.mod != nullptr)) {
      e.gate.table = take(g.table);
      e.gate.mod = take(g.mod);
      e.gate.ldb = g.mod_ld_batch;
      e.gate.ldt = g.mod_ld_tok;
      e.gate.toff = g.scale_table_off;
      e.gate.moff = g.scale_mod_off;
      e.gate.on = 1;
      if ((e.gate.ldb % 8) || (e.gate.ldt % 8) || (e.gate.toff % 8) || (e.gate.moff % 8)) vec = false;
    }
  }
  if (e.kind == LTX_EPI_ROW_MASK_ADD) {
    if (p->row_mask == nullptr || p->row_vec == nullptr)
      throw ApiError{LTX_ERR_INVALID, "ROW_MASK_ADD needs row_mask and row_vec"};
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

bool vec_ok(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

unsigned grid_for(int64_t blocks) {
  if (blocks >= (int64_t(1) << 31)) throw ApiError{LTX_ERR_UNSUPPORTED, "too many rows and columns for one launch"};
  return unsigned(blocks);
}

}  // namespace

extern "C" size_t ltx_fp8_scale_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return size_t(fp8_rows_padded(rows)) * size_t(fp8_quads(cols)) * 4;
}

extern "C" int ltx_quantize_fp8(const void* x, int64_t ldx, int64_t rows, int64_t cols, void* q, int64_t ldq,
                                void* scales, int dtype, void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(x != nullptr, "x must be non-NULL");
  check_fp8_rows(q, ldq, scales, rows, cols, "ltx_quantize_fp8: output");
  LTX_REQUIRE(ldx >= cols, "ldx must hold the columns");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(x) % (dtype == LTX_F32 ? 4 : 2) == 0, "x is not aligned to its type");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int quads = int(fp8_quads(cols));
  const unsigned grid = grid_for((rows * quads + 7) / 8);
  const int vec = vec_ok(x, ldx);
  auto run = [&](auto* xp, auto kern) {
    launch_pdl(kern, dim3(grid), dim3(256), 0, s, 1, xp, ldx, rows, cols, quads, vec, static_cast<uint8_t*>(q), ldq,
               static_cast<uint32_t*>(scales), fp8_rows_padded(rows));
  };
  if (dtype == LTX_F32)
    run(static_cast<const float*>(x), quantize_fp8_kernel<float>);
  else
    run(static_cast<const __nv_bfloat16*>(x), quantize_fp8_kernel<__nv_bfloat16>);
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
  const unsigned grid = grid_for((rows * ((cols + 7) / 8) + 255) / 256);
  const int vec = vec_ok(x, ldx);
  auto run = [&](auto* xp, auto kern) {
    launch_pdl(kern, dim3(grid), dim3(256), 0, s, 1, static_cast<const uint8_t*>(q), ldq,
               static_cast<const uint32_t*>(scales), fp8_rows_padded(rows), rows, cols, vec, xp, ldx);
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
    launch_pdl(norm_modulate_fp8_kernel<T>, dim3(unsigned(rows)), dim3(unsigned((D + 511) / 512 * 32)), 0, s, 1, xp,
               ldx, rows_per_batch, D, norm_kind, eps, make_modvec<T>(mod, 0), make_modvec<T>(mod, 1),
               static_cast<uint8_t*>(q), ldq, static_cast<uint32_t*>(scales), fp8_rows_padded(rows));
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
    const dim3 grid{unsigned((N + 63) / 64), unsigned((M + 63) / 64)};
    LTX_UNSUPPORTED(grid.y < 65536, "M too large");
    linear_fp8_simt_kernel<T><<<grid, 256, 0, s>>>(
        static_cast<const uint8_t*>(A), lda, static_cast<const uint32_t*>(a_scales), fp8_rows_padded(M),
        static_cast<const uint8_t*>(W), ldw, static_cast<const uint32_t*>(w_scales), fp8_rows_padded(N), cp, ldc,
        int(M), int(N), int(K), e), note_launch();
  };
  if (dtype == LTX_F32)
    run(static_cast<float*>(C));
  else
    run(static_cast<__nv_bfloat16*>(C));
  LTX_CUDA(cudaGetLastError());
  LTX_API_END
}
