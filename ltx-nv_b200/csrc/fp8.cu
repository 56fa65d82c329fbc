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

// Epilogue of eight accumulators (columns [col, col + 8) of row `row`, sample sb, token st)
// in fp32, rounded once on the store: acc + bias, then the activation, residual + gate *
// (acc + bias), or + row_vec on marked rows. `vec`: 16-byte accesses are allowed.
template <typename T>
LTX_DEVICE void fp8_epilogue8(const Epi<T>& e, bool vec, T* __restrict__ crow, int64_t row, int64_t sb, int64_t st,
                              int col, int N, float (&v)[8]) {
  const bool whole = vec && col + 8 <= N;
  auto load = [&](const T* p, float (&x)[8]) {
    if (whole) {
      ld8<T>(p, x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = col + i < N ? ld_elem<T>(p + i) : 0.f;
    }
  };
  float a[8];
  if (e.bias) {
    load(e.bias + col, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += a[i];
  }
  if (e.kind == LTX_EPI_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu_sigmoid(v[i]);
  } else if (e.kind == LTX_EPI_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fdividef(v[i], 1.f + __expf(-v[i]));
  } else if (e.kind == LTX_EPI_GATE_RESIDUAL) {
    float g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = e.gate.on ? 0.f : 1.f;
    if (e.gate.table) {
      load(e.gate.table + e.gate.toff + col, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] += a[i];
    }
    if (e.gate.mod) {
      load(e.gate.mod + sb * e.gate.ldb + st * e.gate.ldt + e.gate.moff + col, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] += a[i];
    }
    load(e.residual + row * e.ld_res + col, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(g[i], v[i], a[i]);
  } else if (e.kind == LTX_EPI_ROW_MASK_ADD && e.row_mask[row] > 0.f) {
    load(e.row_vec + col, a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += a[i];
  }
  if (whole) {
    st8<T>(crow + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < N) st_elem<T>(crow + col + i, v[i]);
  }
}

// ---------------------------------------------------------------------------------
// C = epilogue(A W^T) on 8-bit rows with the block-scaled tensor-core MMA.
//
// acc[m][n] = sum over blocks b of 2^(ea[m][b] + ew[n][b]) sum_{k in b} a[m][k] w[n][k]: the MMA
// takes e4m3 operands and a power of two per row and 32 values of K, so a block of 128
// columns is one 128-byte slab of both operands and four MMAs (K = 32) that read the same
// scale byte; sums stay in fp32 in tensor memory, no scaling is left for the CUDA cores.
// A scale word holds four blocks, so scales move once per four slabs: 512 bytes per 128
// rows by TMA next to the slab, then one tcgen05.cp into tensor memory, ordered with the
// MMAs that follow it; two scale buffers alternate.
// ---------------------------------------------------------------------------------

// One 128 x 128 tile per CTA, K split over the CTAs of a cluster (SPLIT = cluster size),
// whose fp32 partial tiles are added through distributed shared memory in rank order:
// short and wide problems spread over the SMs without a workspace or a second launch,
// and the sum's order does not depend on timing.
struct Fp8TileCfg {
  static constexpr int STAGES = 6;
  static constexpr int SLAB = 128 * 128;             // 128 rows x 128 bytes
  static constexpr int SF = 512;                     // scale words of 128 rows, one quad
  static constexpr int STAGE_BYTES = 2 * SLAB + 2 * SF;
  static constexpr int TMEM_COLS = 256;              // accumulator [0, 128), scales [128, 144)
  static constexpr int LD_PART = 128 + 4;            // floats per row of a partial tile (no bank conflicts)
  static constexpr int SMEM = STAGES * STAGE_BYTES + 256 + 1024;
  static_assert(128 * LD_PART * 4 <= STAGES * STAGE_BYTES, "the partial tile reuses the operand ring");
};

template <typename T>
__global__ void __launch_bounds__(192, 1)
    gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                         T* __restrict__ C, int64_t ldc, int M, int N, int K, int split, int vec, Epi<T> epi) {
  using Cfg = Fp8TileCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES);
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

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int it = kb - kb0, s = it % Cfg::STAGES;
        if (!mbar_wait(&empty[s], (uint32_t(it / Cfg::STAGES) & 1) ^ 1, abort_flag)) break;
        uint8_t* st = smem + s * Cfg::STAGE_BYTES;
        const bool sf = kb == kb0 || (kb & 3) == 0;  // a new scale word
        mbar_arrive_expect_tx(&full[s], sf ? Cfg::STAGE_BYTES : 2 * Cfg::SLAB);
        tma_load_2d(st, &tmA, &full[s], kb * 128, m0);
        tma_load_2d(st + Cfg::SLAB, &tmB, &full[s], kb * 128, n0);
        if (sf) {
          tma_load_2d(st + 2 * Cfg::SLAB, &tmSA, &full[s], m0, kb >> 2);
          tma_load_2d(st + 2 * Cfg::SLAB + Cfg::SF, &tmSB, &full[s], n0, kb >> 2);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int it = kb - kb0, s = it % Cfg::STAGES;
        if (!mbar_wait(&full[s], uint32_t(it / Cfg::STAGES) & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t a = smem_u32(smem + s * Cfg::STAGE_BYTES), b = a + Cfg::SLAB;
        const uint32_t sfa = tmem + 128u + uint32_t((kb >> 2) & 1) * 8u, sfb = sfa + 4u;
        if (kb == kb0 || (kb & 3) == 0) {
          tmem_cp_scales(sfa, umma_desc_rows16(a + 2 * Cfg::SLAB));
          tmem_cp_scales(sfb, umma_desc_rows16(a + 2 * Cfg::SLAB + Cfg::SF));
        }
        const uint32_t idesc = umma_idesc_mx8(128, 128, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_mx8_ss(tmem, umma_desc_sw128(a + k * 32, 16, 1024), umma_desc_sw128(b + k * 32, 16, 1024), idesc, sfa,
                      sfb, (it > 0 || k > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
      }
      if (ok) umma_commit(tfull);
    }
  } else {
    const int q = warp & 3;  // TMEM lane quadrant
    const int64_t m = int64_t(m0) + q * 32 + lane;
    const bool live = m < M;
    ok = mbar_wait(tfull, 0, abort_flag);
    if (ok) {
      tc_fence_after();
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16);
      float* part = reinterpret_cast<float*>(smem) + (q * 32 + lane) * Cfg::LD_PART;
      const int64_t sb = m / epi.rows_per_batch, st = m - sb * epi.rows_per_batch;
#pragma unroll 1
      for (int c0 = 0; c0 < 128 && n0 + c0 < N; c0 += 32) {
        uint32_t rr[32];
        tmem_ld32(tbase + uint32_t(c0), rr);
        tmem_wait_ld();
        if (!live) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (split > 1) {
            // every MMA of this CTA has read its operands: the ring is free
            *reinterpret_cast<uint4*>(part + c0 + 8 * j) = make_uint4(rr[8 * j], rr[8 * j + 1], rr[8 * j + 2], rr[8 * j + 3]);
            *reinterpret_cast<uint4*>(part + c0 + 8 * j + 4) =
                make_uint4(rr[8 * j + 4], rr[8 * j + 5], rr[8 * j + 6], rr[8 * j + 7]);
          } else if (n0 + c0 + 8 * j < N) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(rr[8 * j + e]);
            fp8_epilogue8<T>(epi, vec, C + m * ldc, m, sb, st, n0 + c0 + 8 * j, N, v);
          }
        }
      }
    }
  }
  __syncwarp();
  if (split > 1) {
    cluster_sync_all();
    // CTA `rank` finishes the tile's column groups of 8 with index % split == rank
    const int rows = min(128, M - m0), groups = (min(128, N - n0) + 7) / 8;
    const int mine = (groups - rank + split - 1) / split;
    const uint32_t base = smem_u32(smem);
    for (int i = threadIdx.x; i < rows * mine; i += blockDim.x) {
      const int r = i / mine, c = ((i - r * mine) * split + rank) * 8;
      float v[8] = {};
      for (int p = 0; p < split; ++p) {
        const uint32_t at = mapa_shared(base, uint32_t(p)) + uint32_t(r * Cfg::LD_PART + c) * 4u;
        const float4 x = ld_cluster_f4(at), y = ld_cluster_f4(at + 16);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
        v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
      }
      const int64_t m = int64_t(m0) + r;
      const int64_t sb = m / epi.rows_per_batch, st = m - sb * epi.rows_per_batch;
      fp8_epilogue8<T>(epi, vec, C + m * ldc, m, sb, st, n0 + c, N, v);
    }
    cluster_sync_all();  // no CTA leaves while another reads its partial tile
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

// CTAs of one cluster over K: as many as keep the grid within the SMs, at least two
// slabs each, 1, 2, 4 or 8.
inline int fp8_split(int64_t tiles, int64_t k_blocks) {
  int split = 1;
  while (split < 8 && tiles * split * 2 <= num_sms() && k_blocks >= 4 * split) split *= 2;
  return split;
}

template <typename T>
void launch_fp8_tile(const void* A, int64_t lda, const void* As, const void* W, int64_t ldw, const void* Ws, T* C,
                     int64_t ldc, int64_t M, int64_t N, int64_t K, const Epi<T>& epi, bool vec, cudaStream_t s) {
  using Cfg = Fp8TileCfg;
  const uint64_t quads = uint64_t(fp8_quads(K));
  const CUtensorMap ta = make_tmap_u8_2d(A, uint64_t(K), uint64_t(M), uint64_t(lda), 128);
  const CUtensorMap tb = make_tmap_u8_2d(W, uint64_t(K), uint64_t(N), uint64_t(ldw), 128);
  const CUtensorMap tsa = make_tmap_u32_2d(As, uint64_t(fp8_rows_padded(M)), quads, 128);
  const CUtensorMap tsb = make_tmap_u32_2d(Ws, uint64_t(fp8_rows_padded(N)), quads, 128);
  auto kern = gemm_fp8_tile_kernel<T>;
  static std::atomic<uint64_t> smem_done{0};
  ensure_smem_limit(smem_done, kern, Cfg::SMEM);
  const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
  const int split = fp8_split(tiles, (K + 127) / 128);
  LTX_UNSUPPORTED(tiles * split < (int64_t(1) << 31), "too many tiles for one launch");
  launch_pdl(kern, dim3(unsigned(tiles * split)), dim3(192), Cfg::SMEM, s, unsigned(split), ta, tb, tsa, tsb, C, ldc,
             int(M), int(N), int(K), split, int(vec), epi);
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
    vec = vec && vec_ok(C, ldc);
    launch_fp8_tile<T>(A, lda, a_scales, W, ldw, w_scales, cp, ldc, M, N, K, e, vec, s);
  };
  if (dtype == LTX_F32)
    run(static_cast<float*>(C));
  else
    run(static_cast<__nv_bfloat16*>(C));
  LTX_CUDA(cudaGetLastError());
  LTX_API_END
}
