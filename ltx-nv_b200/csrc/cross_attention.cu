// Attention with a per-sample key mask: softmax(Q K^T * scale + mask) V per (sample,
// head), Tq queries and Tk keys of another length (a padded text context), with the
// per-(token, head) output gate 2*sigmoid(logit) of attention.cu. Takes the place of
// sdpa's mask argument (ltx_nn.py:22-26) for masks that do not depend on the query.
//
// A key is left out when its boolean mask is 0, or its additive mask is at or below half
// of the type's lowest finite value (the "lowest value" and -inf conventions alike);
// what K and V hold at such a key (NaN and infinities included) does not reach any
// output. A row whose keys are all left out, or whose scores are all -inf, is zero.
#include <algorithm>

#include "ltx_kernels.cuh"

namespace ltx {
namespace detail {

// Half of the lowest finite value of fp32 and of bf16.
constexpr float kMaskLowestF32 = -0x1.fffffep126f, kMaskLowestBf16 = -0x1.fep126f;

struct KeyMask {
  const void* p;
  int64_t ld;  // elements between samples (0: one mask for all)
  int kind;    // LTX_MASK_BOOL, LTX_MASK_F32, LTX_MASK_BF16

  // What is added to the score of key t of sample b; -inf: left out.
  LTX_DEVICE float at(int64_t b, int64_t t) const {
    const int64_t i = b * ld + t;
    if (kind == LTX_MASK_BOOL) return static_cast<const uint8_t*>(p)[i] ? 0.f : -INFINITY;
    if (kind == LTX_MASK_F32) {
      const float v = static_cast<const float*>(p)[i];
      return v <= kMaskLowestF32 ? -INFINITY : v;
    }
    const float v = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return v <= kMaskLowestBf16 ? -INFINITY : v;
  }
};

// One query per thread, key tiles of 32 in shared memory, online softmax in fp32. 2 x 16 heads
// of 64, 256 keys, 1024 queries: 151 us, 14 TFLOP/s; the fp32 pipe is a third busy, since every
// multiply-add takes its own shared-memory operand and every key rescales the D sums.
template <typename T, int D>
__global__ void __launch_bounds__(128) masked_attn_simt_kernel(const T* __restrict__ Q, int64_t ldq,
                                                               const T* __restrict__ K, int64_t ldk,
                                                               const T* __restrict__ V, int64_t ldv,
                                                               T* __restrict__ O, int64_t ldo, int Tq, int Tk,
                                                               float scale, KeyMask mask, const T* __restrict__ gate,
                                                               int64_t ld_gate) {
  constexpr int KT = 32;
  __shared__ float sk[KT][D];
  __shared__ float sv[KT][D];
  __shared__ float sb[KT];
  const int h = blockIdx.y, b = blockIdx.z;
  const int qi = blockIdx.x * 128 + threadIdx.x;
  const bool active = qi < Tq;
  float q[D], acc[D];
  const T* qp = Q + (int64_t(b) * Tq + (active ? qi : 0)) * ldq + int64_t(h) * D;
#pragma unroll
  for (int c = 0; c < D; ++c) {
    q[c] = active ? ld_elem<T>(qp + c) : 0.f;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int k0 = 0; k0 < Tk; k0 += KT) {
    __syncthreads();
    if (threadIdx.x < KT) sb[threadIdx.x] = k0 + int(threadIdx.x) < Tk ? mask.at(b, k0 + threadIdx.x) : -INFINITY;
    for (int i = threadIdx.x; i < KT * D; i += blockDim.x) {
      const int r = i / D, c = i - r * D;
      const bool in = k0 + r < Tk;
      const int64_t row = int64_t(b) * Tk + k0 + r;
      sk[r][c] = in ? ld_elem<T>(K + row * ldk + int64_t(h) * D + c) : 0.f;
      sv[r][c] = in ? ld_elem<T>(V + row * ldv + int64_t(h) * D + c) : 0.f;
    }
    __syncthreads();
    for (int r = 0; r < KT; ++r) {
      const float bias = sb[r];
      if (bias == -INFINITY) continue;
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < D; ++c) s = fmaf(q[c], sk[r][c], s);
      s = fmaf(s, scale, bias);
      const float mn = fmaxf(m, s);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float corr = expf(m - ref);
      const float p = expf(s - ref);
      l = l * corr + p;
#pragma unroll
      for (int c = 0; c < D; ++c) acc[c] = fmaf(acc[c], corr, p * sv[r][c]);
      m = mn;
    }
  }
  if (!active) return;
  const int64_t orow = int64_t(b) * Tq + qi;
  float g = 1.f;
  if (gate != nullptr) g = 2.f / (1.f + expf(-ld_elem<T>(gate + orow * ld_gate + h)));
  const float inv = l == 0.f ? 0.f : g / l;
  T* op = O + orow * ldo + int64_t(h) * D;
#pragma unroll
  for (int c = 0; c < D; ++c) st_elem<T>(op + c, acc[c] * inv);
}

// ---------------------------------------------------------------------------------
// Few queries (serving's single tokens), bound by the bytes of K and V: a unit is (sample,
// head, one query or four), and its kept keys are streamed once, straight from memory to
// registers. A warp takes 32 keys at a time: their masks in one load (the next ones' ahead
// of the arithmetic), then K and V in pieces of 8 columns a lane, D / 8 lanes to a key, BATCH
// keys a lane in flight; a left-out key is not read at all. Scores, statistics and sums are
// fp32; every group of D / 8 lanes keeps its own running maximum, and groups, warps and the
// CTAs of a cluster that share a unit's keys are joined at the end in a fixed order. 2 x 32
// heads of 128, 4096 keys, one query: 134 MB in 27.9 us, 4.8 TB/s.
// ---------------------------------------------------------------------------------
// Queries of a unit: 1, or up to 4 that share the loads and the conversions of a key.
// (2 samples, 32 heads of 128, 4096 keys, one query: 4 warps with 8 keys a lane 28.4 us, 4
// keys 34.9, 8 warps with 4 keys 35.6; four queries: 8 warps with 4 keys 54.5, 4 warps 61.1.)
constexpr int few_warps(int queries) { return queries == 1 ? 4 : 8; }

template <typename T>
LTX_DEVICE float few_exp2(float x) {
  return std::is_same<T, float>::value ? exp2f(x) : ex2_approx(x);
}

LTX_DEVICE uint4 few_load(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
LTX_DEVICE void few_load8(const __nv_bfloat16* p, uint4 (&r)[1]) { r[0] = few_load(p); }
LTX_DEVICE void few_load8(const float* p, uint4 (&r)[2]) {
  r[0] = few_load(p);
  r[1] = few_load(p + 4);
}
LTX_DEVICE void few_values(const uint4 (&r)[1], float (&v)[8]) {
  const uint32_t w[4] = {r[0].x, r[0].y, r[0].z, r[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
LTX_DEVICE void few_values(const uint4 (&r)[2], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(r[i].x);
    v[4 * i + 1] = __uint_as_float(r[i].y);
    v[4 * i + 2] = __uint_as_float(r[i].z);
    v[4 * i + 3] = __uint_as_float(r[i].w);
  }
}

template <typename T, int D, int QN>
__global__ void __launch_bounds__(few_warps(QN) * 32, QN == 1 ? 4 : 2)
    masked_attn_few_kernel(const T* Q, int64_t ldq, const T* K, int64_t ldk, const T* V, int64_t ldv, T* O,
                           int64_t ldo, int Tq, int Tk, int H, int split, float scale_log2, KeyMask mask,
                           const T* gate, int64_t ld_gate) {
  constexpr int LG = D / 8, G = 32 / LG;  // lanes of a key, keys of a warp at a time
  constexpr int REGS = sizeof(T) / 2;     // 16-byte registers of 8 columns
  constexpr int BATCH = (QN == 1 ? 8 : 4) / REGS;
  constexpr int PARTS = QN * D, WARPS = few_warps(QN);
  __shared__ float part_o[WARPS][PARTS], part_ml[WARPS][QN][2];
  __shared__ float cta_o[PARTS], cta_ml[QN][2];
  const int lane = lane_id(), warp = warp_id(), group = lane / LG, col = lane % LG * 8;
  const int unit = int(blockIdx.x) / split, rank = int(blockIdx.x) % split;
  const int h = unit % H, nq = (Tq + QN - 1) / QN, q0 = unit / H % nq * QN;
  const int64_t b = unit / H / nq, qrow = b * Tq + q0;
  const int queries = min(QN, Tq - q0);
  pdl_wait();
  pdl_trigger();

  const T* kp = K + b * Tk * ldk + int64_t(h) * D + col;
  const T* vp = V + b * Tk * ldv + int64_t(h) * D + col;
  const int64_t step = int64_t(split) * WARPS * 32;
  auto bias_at = [&](int64_t t) { return t < Tk ? mask.at(b, t) * 1.4426950408889634f : -INFINITY; };
  int64_t t0 = (int64_t(rank) * WARPS + warp) * 32;
  float next = bias_at(t0 + lane);
  float q[QN][8], acc[QN][8], m[QN], l[QN];
#pragma unroll
  for (int n = 0; n < QN; ++n) {  // queries past the last repeat it, and are not stored
    uint4 r[REGS];
    few_load8(Q + (qrow + min(n, queries - 1)) * ldq + int64_t(h) * D + col, r);
    few_values(r, q[n]);
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[n][e] *= scale_log2;
      acc[n][e] = 0.f;
    }
  }
  for (; t0 < Tk; t0 += step) {
    const float bias = next;
    next = bias_at(t0 + step + lane);
    const uint32_t kept = __ballot_sync(0xffffffffu, bias != -INFINITY);
#pragma unroll
    for (int j = 0; j < 32 / G; j += BATCH) {
      if ((kept >> (j * G) & (BATCH * G == 32 ? 0xffffffffu : (1u << (BATCH * G % 32)) - 1u)) == 0) continue;
      uint4 kr[BATCH][REGS], vr[BATCH][REGS];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = (j + i) * G + group;
#pragma unroll
        for (int w = 0; w < REGS; ++w) kr[i][w] = vr[i][w] = make_uint4(0, 0, 0, 0);
        if (kept >> r & 1u) {
          few_load8(kp + (t0 + r) * ldk, kr[i]);
          few_load8(vp + (t0 + r) * ldv, vr[i]);
        }
      }
      float sc[QN][BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        float kv[8];
        few_values(kr[i], kv);
#pragma unroll
        for (int n = 0; n < QN; ++n) {
          sc[n][i] = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sc[n][i] = fmaf(q[n][e], kv[e], sc[n][i]);
        }
      }
#pragma unroll
      for (int off = LG / 2; off > 0; off /= 2)
#pragma unroll
        for (int n = 0; n < QN; ++n)
#pragma unroll
          for (int i = 0; i < BATCH; ++i) sc[n][i] += __shfl_xor_sync(0xffffffffu, sc[n][i], off);
      float add[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) add[i] = __shfl_sync(0xffffffffu, bias, (j + i) * G + group);
#pragma unroll
      for (int n = 0; n < QN; ++n) {
        float mx = m[n];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          sc[n][i] = add[i] == -INFINITY ? -INFINITY : sc[n][i] + add[i];
          mx = fmaxf(mx, sc[n][i]);
        }
        const float ref = mx == -INFINITY ? 0.f : mx, alpha = few_exp2<T>(m[n] - ref);
        m[n] = mx;
        l[n] *= alpha;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[n][e] *= alpha;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          sc[n][i] = few_exp2<T>(sc[n][i] - ref);
          l[n] += sc[n][i];
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        float vv[8];
        few_values(vr[i], vv);
#pragma unroll
        for (int n = 0; n < QN; ++n)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[n][e] = fmaf(sc[n][i], vv[e], acc[n][e]);
      }
    }
  }

  // join the groups of a warp, ...
#pragma unroll
  for (int n = 0; n < QN; ++n) {
#pragma unroll
    for (int off = LG; off < 32; off *= 2) {
      const float mo = __shfl_xor_sync(0xffffffffu, m[n], off), lo = __shfl_xor_sync(0xffffffffu, l[n], off);
      const float mx = fmaxf(m[n], mo), ref = mx == -INFINITY ? 0.f : mx;
      const float f = few_exp2<T>(m[n] - ref), fo = few_exp2<T>(mo - ref);
      l[n] = l[n] * f + lo * fo;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[n][e] = acc[n][e] * f + __shfl_xor_sync(0xffffffffu, acc[n][e], off) * fo;
      m[n] = mx;
    }
    if (lane < LG) {
#pragma unroll
      for (int e = 0; e < 8; ++e) part_o[warp][n * D + col + e] = acc[n][e];
      if (lane == 0) part_ml[warp][n][0] = m[n], part_ml[warp][n][1] = l[n];
    }
  }
  __syncthreads();
  // ... the warps, ...
  for (int i = threadIdx.x; i < queries * D; i += WARPS * 32) {
    const int n = i / D;
    float o = 0.f, L = 0.f, M = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, part_ml[w][n][0]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = few_exp2<T>(part_ml[w][n][0] - ref);
      L += part_ml[w][n][1] * f;
      o += part_o[w][i] * f;
    }
    if (split == 1) {
      float g = 1.f;
      if (gate != nullptr) g = 2.f / (1.f + expf(-ld_elem<T>(gate + (qrow + n) * ld_gate + h)));
      st_elem<T>(O + (qrow + n) * ldo + int64_t(h) * D + i % D, L == 0.f ? 0.f : o * (g / L));
    } else {
      cta_o[i] = o;
      if (i % D == 0) cta_ml[n][0] = M, cta_ml[n][1] = L;
    }
  }
  if (split == 1) return;
  // ... and the CTAs of a cluster (each takes its share of the columns).
  cluster_sync_all();
  for (int i = rank * WARPS * 32 + threadIdx.x; i < queries * D; i += split * WARPS * 32) {
    const int n = i / D;
    float po[8], pm[8], pl[8], M = -INFINITY, o = 0.f, L = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      pm[r] = -INFINITY, pl[r] = po[r] = 0.f;
      if (r < split) {
        pm[r] = ld_cluster_f1(mapa_shared(smem_u32(&cta_ml[n][0]), r));
        pl[r] = ld_cluster_f1(mapa_shared(smem_u32(&cta_ml[n][1]), r));
        po[r] = ld_cluster_f1(mapa_shared(smem_u32(&cta_o[i]), r));
      }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) M = fmaxf(M, pm[r]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float f = few_exp2<T>(pm[r] - ref);
      o += po[r] * f;
      L += pl[r] * f;
    }
    float g = 1.f;
    if (gate != nullptr) g = 2.f / (1.f + expf(-ld_elem<T>(gate + (qrow + n) * ld_gate + h)));
    st_elem<T>(O + (qrow + n) * ldo + int64_t(h) * D + i % D, L == 0.f ? 0.f : o * (g / L));
  }
  cluster_sync_all();  // no CTA leaves while another reads its sums
}

// bf16: for up to 4 queries a sample, where a unit of the tensor-core kernel would be one row
// of 256 (2 samples, 32 heads of 128, 64 / 1024 / 4096 keys: one query 4.0 / 10.3 / 27.9 us
// against 8.5 / 21.8 / 57.2, four 7.5 / 16.2 / 54.3 against 8.4 / 22.1 / 57.2, eight 7.8 / 28.7
// / 99.2 against 8.5 / 22.1 / 57.5).
// fp32: while the kernel of one query per thread would leave SMs without a block, or at 128
// columns a head, where its accumulators do not stay in registers, with four of them (heads
// of 64: 1 x 8 heads, 200 keys, 480 queries 29 us against 96; 2 x 8, 256, 1024 112 / 118; 2 x
// 16, 256, 1024 218 / 150. Heads of 128: 46 / 333, 181 / 418, 357 / 465; 2 x 32, 128, 6144
// 3238 / 2780).
inline bool use_few(int64_t B, int64_t Tq, int H, int D, bool bf16) {
  if (B * Tq * H >= int64_t(1) << 27) return false;
  return bf16 ? Tq <= 4 : Tq <= 4 || B * H * ((Tq + 127) / 128) < num_sms() * (D == 128 ? 4 : 1);
}

template <typename T, int D>
void launch_masked_few(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* o,
                       int64_t ldo, int B, int64_t Tq, int64_t Tk, int H, float scale, const KeyMask& mask,
                       const void* gate, int64_t ld_gate, cudaStream_t s) {
  const bool one = Tq == 1;
  const int64_t units = int64_t(B) * (one ? 1 : (Tq + 3) / 4) * H;
  const int warps = one ? few_warps(1) : few_warps(4);
  // Up to 32 warps for every SM, while every warp still has a chunk of 32 keys.
  int split = 1;
  while (split < 8 && units * split * warps < 32 * num_sms() && Tk > int64_t(split) * warps * 32) split *= 2;
  launch_pdl(one ? masked_attn_few_kernel<T, D, 1> : masked_attn_few_kernel<T, D, 4>, dim3(unsigned(units * split)),
             dim3(warps * 32), 0, s, unsigned(split), static_cast<const T*>(q), ldq, static_cast<const T*>(k), ldk,
             static_cast<const T*>(v), ldv, static_cast<T*>(o), ldo, int(Tq), int(Tk), H, split,
             scale * 1.4426950408889634f, mask, static_cast<const T*>(gate), ld_gate);
}

// ---------------------------------------------------------------------------------
// bf16: persistent tcgen05 kernel. A unit is (sample, head, 256 queries) = two 128-row Q
// tiles; CTAs walk the units in steps of the grid, and every role runs straight on from
// one unit to the next, so a unit's Q load, first Q K^T and output store overlap its
// neighbours' softmax: with the few key tiles of a text context, the fixed cost of a
// unit would otherwise be as large as its work.
//   warps 0-3, 4-7  softmax of Q tile 0 / 1 (one query row per thread = TMEM lane)
//   warp 8          reads a sample's mask into the list of its key tiles (128 keys each) that
//                   hold any key, loads Q and the listed K / V tiles by TMA, and leaves a
//                   descriptor (MaTile) beside each stage that the other roles follow
//   warps 9, 10     MMA issuers of Q tile 0 / 1 (head_dim 128: warp 9 issues both)
//   warp 11         tiles that need more than plain scores: what each key adds to them (-inf:
//                   left out) in shared memory, and V rows of left-out keys set to zero, so
//                   that no NaN there can reach P V (0 * NaN)
// Tiles without a key are never loaded; plain tiles run the unmasked softmax (packed
// arithmetic, part of the exponentials on the FMA pipe, lazy rescaling: attention.cu).
// TMEM as in attention.cu: head_dim 64 keeps P beside S (S_i is computed two tiles
// ahead), head_dim 128 writes P over S.
// P is rounded to bf16, the type that an MMA with bf16 V takes, as in attention.cu (the row sum
// is not): 2^-8 of each weight at the most, 2.2e-3 rel-L2 of the result against float64, where
// rounding the result alone gives 1.7e-3.
// 2 x 6144 queries, 1024 keys, 32 heads of 64: 181 us with every key kept, 112 with half of them;
// no unit is full (issue slots 44 %, special functions 39 %, tensor pipe 27 %): the two softmax
// warps of a scheduler wait for tensor memory and barriers in turn.
// split > 1 (few units, many key tiles): the CTAs of a cluster take shares of one unit's
// list and merge their fp32 O / l and log-sum-exp through distributed shared memory, in
// rank order.
// ---------------------------------------------------------------------------------
template <int D>
struct MaCfg {
  static constexpr int SUB = D / 64;              // 64-column (128-byte) sub-tiles per row
  static constexpr int TILE = 128 * D * 2;        // one Q, K or V tile
  static constexpr bool SEP_P = D == 64;          // P in its own TMEM columns
  static constexpr int STAGES = SEP_P ? 4 : 2;    // K / V ring
  static constexpr int QBUF = SEP_P ? 2 : 1;      // units whose Q is in shared memory
  static constexpr int ISSUERS = SEP_P ? 2 : 1;
  static constexpr int MAX_TILES = 4096;          // list entries: Tk <= 524288
  static constexpr int RING = TILE * 2 * (QBUF + STAGES);
  static constexpr int BIAS = STAGES * 128 * 4;
  static constexpr int LIST = MAX_TILES * 2;
  static constexpr int SMEM = RING + BIAS + LIST + 768 + 1024;
  static constexpr int LD_PART = D + 4;           // floats per row of a split unit's partial
  static_assert(256 * LD_PART * 4 + 256 * 4 <= RING, "the partial reuses the operand ring");
  static constexpr uint32_t s_col(int i) { return uint32_t(128 * i); }
  static constexpr uint32_t p_col(int i) { return SEP_P ? uint32_t(256 + 64 * i) : uint32_t(128 * i); }
  static constexpr uint32_t o_col(int i) { return SEP_P ? uint32_t(384 + 64 * i) : uint32_t(256 + D * i); }
};

struct MaParams {
  int H, Tq, Tk, nq2;
  int units, split;  // split: CTAs of a cluster that share a unit
  float scale_log2;
  KeyMask mask;
  const __nv_bfloat16* gate;
  int64_t ld_gate;
  __nv_bfloat16* O;
  int64_t ldo;

  LTX_DEVICE int sample(int u) const { return u / (nq2 * H); }
  LTX_DEVICE int head(int u) const { return (u / nq2) % H; }
  LTX_DEVICE int q0(int u) const { return (u % nq2) * 256; }
};

// What a K / V stage holds: a key tile of a unit. FIRST / LAST of the unit's tiles; MARKED:
// its scores need sbias; TWO: Q tile 1 of the unit has rows; END: no more tiles.
struct MaTile {
  int flags, unit, tile, pad;
};
enum : int { MA_FIRST = 1, MA_LAST = 2, MA_MARKED = 4, MA_TWO = 8, MA_END = 16 };

// The same once per unit, for the softmax, whose tile loop then reads no descriptor (a wait
// and a load per tile cost it 15 %): `tiles` of them (0: no more units), and which of the
// first 64 are marked (of a longer unit's later tiles, the stage's descriptor says it).
struct MaUnit {
  int unit, tiles, flags, pad;
  uint32_t marked[2];
  uint32_t pad2[2];
};
// The sum of weights below which a row has none. The key that m_ref was taken from weighs 1 (at
// scores of 1e9, where a product's rounding shows, 2^-60), and m_ref only rises with the next
// such key; a row of -inf scores alone sums the cubic's remainders, 36 * 19 * 2^-149 a tile, over
// at most 4096 tiles.
constexpr float kMaDeadRow = 0x1p-126f;
constexpr int kMaUnits = 4;  // units the producer may be ahead

LTX_DEVICE void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int D>
constexpr int ma_control_bytes() {
  return (2 * MaCfg<D>::QBUF + 4 * MaCfg<D>::STAGES + 8 + 2 * kMaUnits) * 8 + MaCfg<D>::STAGES * int(sizeof(MaTile)) +
         kMaUnits * int(sizeof(MaUnit)) + 8;
}
static_assert(ma_control_bytes<64>() <= 768 && ma_control_bytes<128>() <= 768, "barriers and descriptors");

template <int D>
__global__ void __launch_bounds__(384, 1)
    masked_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, const MaParams P) {
  using Cfg = MaCfg<D>;
  constexpr int S = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = fa_align1024(smem_raw);
  uint8_t* sQ = smem;                               // unit buffer k, Q tile i at (2k + i) * TILE
  uint8_t* sKV = smem + 2 * Cfg::QBUF * Cfg::TILE;  // stage s: K at 2s * TILE, V behind it
  float* sbias = reinterpret_cast<float*>(smem + Cfg::RING);  // [S][128], log2 units
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + Cfg::RING + Cfg::BIAS);  // warp 8's
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::RING + Cfg::BIAS + Cfg::LIST);
  uint64_t* q_full = bars;                   // [QBUF]
  uint64_t* q_empty = q_full + Cfg::QBUF;    // [QBUF]
  uint64_t* k_full = q_empty + Cfg::QBUF;    // [S] descriptor and K
  uint64_t* v_full = k_full + S;             // [S]
  uint64_t* v_fix = v_full + S;              // [S] V and bias ready (warp 11)
  uint64_t* kv_empty = v_fix + S;            // [S] both Q tiles' P V done
  uint64_t* s_full = kv_empty + S;           // [2]
  uint64_t* s_free = s_full + 2;             // [2] SEP_P only
  uint64_t* p_full = s_free + 2;             // [2]
  uint64_t* o_done = p_full + 2;             // [2]
  uint64_t* u_full = o_done + 2;             // [kMaUnits] unit descriptor written
  uint64_t* u_empty = u_full + kMaUnits;     // [kMaUnits] read by the eight softmax warps
  MaTile* desc = reinterpret_cast<MaTile*>(u_empty + kMaUnits);  // [S]
  MaUnit* units = reinterpret_cast<MaUnit*>(desc + S);           // [kMaUnits]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(units + kMaUnits);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    for (int k = 0; k < Cfg::QBUF; ++k) {
      mbar_init(&q_full[k], 1);
      mbar_init(&q_empty[k], Cfg::ISSUERS);
    }
    for (int s = 0; s < S; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_fix[s], 1);
      mbar_init(&kv_empty[s], 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 128);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    for (int k = 0; k < kMaUnits; ++k) {
      mbar_init(&u_full[k], 1);
      mbar_init(&u_empty[k], 8);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  // this CTA's units, and its share of each unit's list
  const int u0 = int(blockIdx.x) / P.split, rank = int(blockIdx.x) - u0 * P.split;
  const int u_step = P.split > 1 ? P.units : int(gridDim.x);
  // softmax state of a split unit, for the merge
  float m_ref = -INFINITY, l_run = 0.f;
  bool have = false;

  if (warp == 8) {
    // ------------------------- lists and TMA producer -------------------------
    const int n_tiles = (P.Tk + 127) / 128;
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    int b = -1, lo = 0, n = 0, g = 0, un = 0;
    uint32_t marked[2] = {0, 0};  // of this CTA's first 64 tiles of the sample
    bool ok = true;
    for (int u = u0; ok && u < P.units; u += u_step) {
      const int nb = P.sample(u), h = P.head(u), q0 = P.q0(u);
      if (nb != b) {
        b = nb;
        int count = 0;
        __syncwarp();
        for (int t0 = 0; t0 < n_tiles; t0 += 32) {
          uint32_t any = 0, plain = 0;  // bit j: tile t0 + j
          const int nt = min(32, n_tiles - t0);
#pragma unroll 4
          for (int j = 0; j < nt; ++j) {
            const int key = (t0 + j) * 128 + lane;
            bool a = false, p = true;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float v = key + 32 * c < P.Tk ? P.mask.at(b, key + 32 * c) : -INFINITY;
              a |= v != -INFINITY;
              p &= v == 0.f;
            }
            if (__any_sync(0xffffffffu, a)) any |= 1u << j;
            if (__all_sync(0xffffffffu, p)) plain |= 1u << j;
          }
          if ((any >> lane) & 1u)
            list[count + __popc(any & ((1u << lane) - 1u))] =
                uint16_t((t0 + lane) | (((plain >> lane) & 1u) ? 0 : 0x8000));
          count += __popc(any);
        }
        __syncwarp();
        lo = int(int64_t(count) * rank / P.split);
        n = int(int64_t(count) * (rank + 1) / P.split) - lo;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          marked[j] = __ballot_sync(0xffffffffu, 32 * j + lane < n && (list[lo + 32 * j + lane] & 0x8000));
      }
      if (n == 0) {
        if (P.split == 1) {  // no key: zero rows
          constexpr int LPR = D / 8;  // lanes per row, 16 bytes each
          for (int r = lane / LPR; r < min(256, P.Tq - q0); r += 32 / LPR)
            *reinterpret_cast<uint4*>(P.O + (int64_t(b) * P.Tq + q0 + r) * P.ldo + int64_t(h) * D + (lane % LPR) * 8) =
                make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      if (lane == 0) {
        const int k = un % Cfg::QBUF, col0 = h * D, two = q0 + 128 < P.Tq ? 1 : 0;
        ok = mbar_wait(&u_empty[un % kMaUnits], (uint32_t(un / kMaUnits) & 1) ^ 1, abort_flag) &&
             mbar_wait(&q_empty[k], (uint32_t(un / Cfg::QBUF) & 1) ^ 1, abort_flag);
        if (ok) {
          units[un % kMaUnits] = MaUnit{u, n, two ? MA_TWO : 0, 0, {marked[0], marked[1]}, {0, 0}};
          mbar_arrive(&u_full[un % kMaUnits]);
          mbar_arrive_expect_tx(&q_full[k], (1 + two) * Cfg::TILE);
          for (int i = 0; i <= two; ++i)
#pragma unroll
            for (int j = 0; j < Cfg::SUB; ++j)
              tma_load_2d(sQ + (2 * k + i) * Cfg::TILE + j * 16384, &tmQ, &q_full[k], col0 + 64 * j,
                          b * P.Tq + q0 + i * 128);
        }
        for (int t = 0; ok && t < n; ++t, ++g) {
          const int s = g % S;
          ok = mbar_wait(&kv_empty[s], (uint32_t(g / S) & 1) ^ 1, abort_flag);
          if (!ok) break;
          const int e = list[lo + t], tile = e & 0x7fff;
          desc[s] = MaTile{(t == 0 ? MA_FIRST : 0) | (t == n - 1 ? MA_LAST : 0) | ((e & 0x8000) ? MA_MARKED : 0) |
                               (two ? MA_TWO : 0), u, tile, 0};
          uint8_t* sk = sKV + 2 * s * Cfg::TILE;
          const int row = b * P.Tk + tile * 128;
          mbar_arrive_expect_tx(&k_full[s], Cfg::TILE);
#pragma unroll
          for (int j = 0; j < Cfg::SUB; ++j) tma_load_2d(sk + j * 16384, &tmK, &k_full[s], col0 + 64 * j, row);
          mbar_arrive_expect_tx(&v_full[s], Cfg::TILE);
#pragma unroll
          for (int j = 0; j < Cfg::SUB; ++j)
            tma_load_2d(sk + Cfg::TILE + j * 16384, &tmV, &v_full[s], col0 + 64 * j, row);
        }
      }
      ok = __shfl_sync(0xffffffffu, int(ok), 0) != 0;
      ++un;
    }
    if (lane == 0 && ok && mbar_wait(&u_empty[un % kMaUnits], (uint32_t(un / kMaUnits) & 1) ^ 1, abort_flag) &&
        mbar_wait(&kv_empty[g % S], (uint32_t(g / S) & 1) ^ 1, abort_flag)) {
      units[un % kMaUnits] = MaUnit{0, 0, 0, 0, {0, 0}, {0, 0}};
      mbar_arrive(&u_full[un % kMaUnits]);
      desc[g % S] = MaTile{MA_END, 0, 0, 0};
      mbar_arrive(&k_full[g % S]);
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------ MMA issuers ------------------------------
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, 0);
    constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 1);
    // Scores of tile g for Q tile i (k: the unit's Q buffer). A unit without a Q tile 1 has
    // no MMAs there; its barriers advance all the same, so every phase is the tile's number.
    auto issue_qk = [&](int i, int g, int k, int flags) {
      if (i == 0 || (flags & MA_TWO)) {
        const uint32_t qa = smem_u32(sQ) + uint32_t((2 * k + i) * Cfg::TILE);
        const uint32_t ka = smem_u32(sKV + 2 * (g % S) * Cfg::TILE);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = uint32_t((kk >> 2) * 16384 + (kk & 3) * 32);
          umma_ss(tmem + Cfg::s_col(i), umma_desc_sw128(qa + off, 16, 1024), umma_desc_sw128(ka + off, 16, 1024),
                  idesc_s, kk > 0 ? 1u : 0u);
        }
      }
      umma_commit(&s_full[i]);
    };
    auto issue_pv = [&](int i, int g, int flags) {
      if (i == 0 || (flags & MA_TWO)) {
        const uint32_t va = smem_u32(sKV + (2 * (g % S) + 1) * Cfg::TILE);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          umma_ts(tmem + Cfg::o_col(i), tmem + Cfg::p_col(i) + uint32_t(kk * 8),
                  umma_desc_sw128(va + uint32_t(kk * 2048), 16384, 1024), idesc_o,
                  (!(flags & MA_FIRST) || kk > 0) ? 1u : 0u);
      }
      umma_commit(&o_done[i]);
      umma_commit(&kv_empty[g % S]);  // count 2: both Q tiles' P V of this stage
    };
    auto wait_k = [&](int g) { return mbar_wait(&k_full[g % S], uint32_t(g / S) & 1, abort_flag); };
    auto wait_q = [&](int un) {
      return mbar_wait(&q_full[un % Cfg::QBUF], uint32_t(un / Cfg::QBUF) & 1, abort_flag);
    };
    if (lane == 0 && warp - 9 < Cfg::ISSUERS) {
      int gq = 0, un = 0;  // next tile whose scores are issued, and its unit
      bool more = true;    // no END seen yet
      if constexpr (Cfg::SEP_P) {
        // Q tile i: P_i V_g, then Q_i K_{g+2}^T (attention.cu).
        const int i = warp - 9;
        auto qk_step = [&]() {
          if (!wait_k(gq)) return false;
          const int flags = desc[gq % S].flags;
          if (flags & MA_END) {
            more = false;
            return true;
          }
          if ((flags & MA_FIRST) && !wait_q(un)) return false;
          if (gq > 0 && !mbar_wait(&s_free[i], uint32_t(gq - 1) & 1, abort_flag)) return false;
          tc_fence_after();
          issue_qk(i, gq, un % Cfg::QBUF, flags);
          if (flags & MA_LAST) umma_commit(&q_empty[un++ % Cfg::QBUF]);
          ++gq;
          return true;
        };
        bool ok = qk_step() && (!more || qk_step());
        for (int g = 0; ok && g < gq; ++g) {
          const int s = g % S, flags = desc[s].flags;
          ok = mbar_wait(&v_fix[s], uint32_t(g / S) & 1, abort_flag) &&
               mbar_wait(&p_full[i], uint32_t(g) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          issue_pv(i, g, flags);
          if (more) ok = qk_step();
        }
      } else {
        // Both Q tiles: P_0 V_g, Q_0 K_{g+1}^T, P_1 V_g, Q_1 K_{g+1}^T (attention.cu).
        bool ok = wait_k(0);
        int flags = ok ? desc[0].flags : MA_END;
        if (ok && !(flags & MA_END)) {
          ok = wait_q(0);
          if (ok) {
            tc_fence_after();
            issue_qk(0, 0, 0, flags);
            issue_qk(1, 0, 0, flags);
            if (flags & MA_LAST) umma_commit(&q_empty[0]), ++un;
          }
        }
        for (int g = 0; ok && !(flags & MA_END); ++g) {
          ok = mbar_wait(&v_fix[g % S], uint32_t(g / S) & 1, abort_flag);
          int next = MA_END;
          for (int i = 0; ok && i < 2; ++i) {
            if (!mbar_wait(&p_full[i], uint32_t(g) & 1, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            issue_pv(i, g, flags);
            if (i == 0) {  // the next tile's K (and Q), awaited behind the first P V
              ok = wait_k(g + 1);
              if (!ok) break;
              next = desc[(g + 1) % S].flags;
              if ((next & MA_FIRST) && !(ok = wait_q(un))) break;
              tc_fence_after();
            }
            if (!(next & MA_END)) {
              issue_qk(i, g + 1, un % Cfg::QBUF, next);
              if (i == 1 && (next & MA_LAST)) umma_commit(&q_empty[un++ % Cfg::QBUF]);
            }
          }
          flags = next;
        }
      }
    }
  } else if (warp == 11) {
    // ------------------------- marked tiles: bias and V -------------------------
    for (int g = 0;; ++g) {
      const int s = g % S;
      const uint32_t par = uint32_t(g / S) & 1;
      if (!mbar_wait(&k_full[s], par, abort_flag)) break;
      const MaTile d = desc[s];
      if (d.flags & MA_END) break;
      float v[4];
      uint32_t keep[4];
      if (d.flags & MA_MARKED) {
        const int b = P.sample(d.unit);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = d.tile * 128 + 32 * c + lane;
          v[c] = key < P.Tk ? P.mask.at(b, key) : -INFINITY;
        }
      }
      if (!mbar_wait(&v_full[s], par, abort_flag)) break;
      if (d.flags & MA_MARKED) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sbias[s * 128 + 32 * c + lane] = v[c] * 1.4426950408889634f;
          keep[c] = __ballot_sync(0xffffffffu, v[c] != -INFINITY);
        }
        uint8_t* sv = sKV + (2 * s + 1) * Cfg::TILE + (lane >> 3) * 128 + (lane & 7) * 16;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int r = 0; r < 32; r += 4) {
            if (!((keep[c] >> (r + (lane >> 3))) & 1u)) {
#pragma unroll
              for (int j = 0; j < Cfg::SUB; ++j)
                *reinterpret_cast<uint4*>(sv + j * 16384 + (32 * c + r) * 128) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(&v_fix[s]);
    }
  } else {
    // --------------------- softmax / correction / epilogue ---------------------
    const int qt = warp >> 2;                // Q tile of this warpgroup
    const int row = (warp & 3) * 32 + lane;  // row within the tile == TMEM lane
    const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + Cfg::s_col(qt) + lane_off;
    const uint32_t p_tmem = tmem + Cfg::p_col(qt) + lane_off;
    const uint32_t o_tmem = tmem + Cfg::o_col(qt) + lane_off;
    // Softmax of tile g (`first` of its unit) from S to P. Plain and marked tiles are separate
    // code: the plain one is that of attention.cu, without the mask's registers.
    auto tile = [&](auto marked_c, int g, bool first) {
      constexpr bool MARKED = decltype(marked_c)::value;
      const int s = g % S;
      if (!mbar_wait(&s_full[qt], uint32_t(g) & 1, abort_flag)) return false;
      tc_fence_after();
      uint32_t su[128];
      tmem_read128(s_tmem, su);
      float sv[128];
#pragma unroll
      for (int e = 0; e < 128; ++e) sv[e] = __uint_as_float(su[e]);
      if constexpr (Cfg::SEP_P) {
        tc_fence_before();
        mbar_arrive(&s_free[qt]);
      }
      if constexpr (MARKED) {
        // scores in log2 units with the mask added; a left-out key's is -inf whatever K held
        if (!mbar_wait(&v_fix[s], uint32_t(g / S) & 1, abort_flag)) return false;
        const float4* bias = reinterpret_cast<const float4*>(sbias + s * 128);
#pragma unroll
        for (int e = 0; e < 128; e += 4) {
          const float4 bb = bias[e >> 2];
          sv[e] = bb.x == -INFINITY ? -INFINITY : fmaf(sv[e], P.scale_log2, bb.x);
          sv[e + 1] = bb.y == -INFINITY ? -INFINITY : fmaf(sv[e + 1], P.scale_log2, bb.y);
          sv[e + 2] = bb.z == -INFINITY ? -INFINITY : fmaf(sv[e + 2], P.scale_log2, bb.z);
          sv[e + 3] = bb.w == -INFINITY ? -INFINITY : fmaf(sv[e + 3], P.scale_log2, bb.w);
        }
      }
      // The maximum keeps a NaN score, and as m_ref carries it into every weight of the row:
      // the cubic below would lose it, and only some keys take the cubic.
      float m8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) m8[e] = sv[e];
#pragma unroll
      for (int e = 8; e < 120; e += 16)
#pragma unroll
        for (int j = 0; j < 8; ++j) m8[j] = fmax3_nan(m8[j], sv[e + j], sv[e + 8 + j]);
#pragma unroll
      for (int j = 0; j < 8; ++j) m8[j] = fmax3_nan(m8[j], sv[120 + j], sv[120 + j]);
      const float mx =
          fmax3_nan(fmax3_nan(m8[0], m8[1], m8[2]), fmax3_nan(m8[3], m8[4], m8[5]), fmax3_nan(m8[6], m8[7], m8[7]));
      const float m_cand = MARKED ? mx : mx * P.scale_log2;
      const bool need = first || !(m_cand <= m_ref + 8.f);
      float alpha = 1.f;
      if (need) {
        const float m_new = fmax3_nan(m_ref, m_cand, m_cand);
        alpha = first || m_new == -INFINITY ? 0.f : ex2_approx(m_ref - m_new);
        m_ref = m_new;
      }
      const float m_sub = m_ref == -INFINITY ? 0.f : m_ref;  // a row of -inf so far: weights 0
      const uint64_t sc2 = f2_pack(P.scale_log2, P.scale_log2);
      const uint64_t nm2 = f2_pack(-m_sub, -m_sub);
      uint64_t rs2[4] = {0, 0, 0, 0};
      uint32_t pk[64];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float x0, x1, p0, p1;
          const uint64_t s2 = f2_pack(sv[c * 32 + e], sv[c * 32 + e + 1]);
          f2_unpack(MARKED ? f2_add(s2, nm2) : f2_fma(s2, sc2, nm2), x0, x1);
          if (!MARKED && ((kFaPolyPairs >> (c * 16 + (e >> 1))) & 1u)) {
            ex2_poly2(x0, x1, p0, p1);
          } else {
            p0 = ex2_approx(x0);
            p1 = ex2_approx(x1);
          }
          rs2[(e >> 1) & 3] = f2_add(rs2[(e >> 1) & 3], f2_pack(p0, p1));
          pk[c * 16 + (e >> 1)] = pack_bf16x2(p0, p1);
        }
        if constexpr (!Cfg::SEP_P) tmem_st16(p_tmem + uint32_t(c * 16), *reinterpret_cast<uint32_t(*)[16]>(&pk[c * 16]));
      }
      if constexpr (Cfg::SEP_P) {
        // P_i V_{g-1} has read P_i, and the issuer has seen p_full of tile g - 1
        if (g > 0) {
          if (!mbar_wait(&o_done[qt], uint32_t(g - 1) & 1, abort_flag)) return false;
          tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          tmem_st16(p_tmem + uint32_t(c * 16), *reinterpret_cast<uint32_t(*)[16]>(&pk[c * 16]));
      }
      float r0, r1;
      f2_unpack(f2_add(f2_add(rs2[0], rs2[1]), f2_add(rs2[2], rs2[3])), r0, r1);
      if (!first && __any_sync(0xffffffffu, need)) {
        if (!Cfg::SEP_P) {
          if (!mbar_wait(&o_done[qt], uint32_t(g - 1) & 1, abort_flag)) return false;
          tc_fence_after();
        }
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t rr[32];
          tmem_read32(o_tmem + uint32_t(c0), rr);
#pragma unroll
          for (int e = 0; e < 32; ++e) rr[e] = __float_as_uint(__uint_as_float(rr[e]) * alpha);
          tmem_st32(o_tmem + uint32_t(c0), rr);
        }
      }
      l_run = l_run * alpha + (r0 + r1);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[qt]);
      return true;
    };
    bool ok = true;
    int g = 0;
    for (int un = 0; ok; ++un) {
      if (!mbar_wait(&u_full[un % kMaUnits], uint32_t(un / kMaUnits) & 1, abort_flag)) break;
      const MaUnit* ud = &units[un % kMaUnits];
      const int unit = ud->unit, two = ud->flags & MA_TWO;
      const int n = int(__reduce_max_sync(0xffffffffu, unsigned(ud->tiles)));  // warp-uniform
      const uint32_t marked0 = ud->marked[0], marked1 = ud->marked[1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&u_empty[un % kMaUnits]);
      if (n == 0) break;
      if (qt == 1 && !two) {
        for (int t = 0; t < n; ++t, ++g) {
          // one p_full phase ahead of the issuer at most, as below
          ok = mbar_wait(&s_full[qt], uint32_t(g) & 1, abort_flag) &&
               (g == 0 || mbar_wait(&o_done[qt], uint32_t(g - 1) & 1, abort_flag));
          if (!ok) break;
          if (Cfg::SEP_P) mbar_arrive(&s_free[qt]);
          mbar_arrive(&p_full[qt]);
        }
        continue;
      }
      m_ref = -INFINITY;
      l_run = 0.f;
      for (int t = 0; t < n; ++t, ++g) {
        bool marked = ((t < 32 ? marked0 : marked1) >> (t & 31)) & 1u;
        if (t >= 64) {
          ok = mbar_wait(&k_full[g % S], uint32_t(g / S) & 1, abort_flag);
          if (!ok) break;
          marked = desc[g % S].flags & MA_MARKED;
        }
        ok = marked ? tile(std::true_type{}, g, t == 0) : tile(std::false_type{}, g, t == 0);
        if (!ok) break;
      }
      // ------------------------- the unit's output rows -------------------------
      if (!ok || !mbar_wait(&o_done[qt], uint32_t(g - 1) & 1, abort_flag)) break;
      tc_fence_after();
      if (P.split > 1) {
        have = true;
        break;  // the only unit
      }
      const int b = P.sample(unit), h = P.head(unit);
      const int qi = P.q0(unit) + qt * 128 + row;
      const bool live = qi < P.Tq;
      const int64_t orow = int64_t(b) * P.Tq + qi;
      const bool dead = l_run < kMaDeadRow;
      const bool any_dead = __any_sync(0xffffffffu, dead);
      float f = dead ? 0.f : 1.f / l_run;
      if (P.gate != nullptr && live) f *= 2.f / (1.f + __expf(-__bfloat162float(P.gate[orow * P.ld_gate + h])));
      __nv_bfloat16* op = P.O + orow * P.ldo + int64_t(h) * D;
#pragma unroll
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t rr[32];
        tmem_read32(o_tmem + uint32_t(c0), rr);
        if (any_dead) {
#pragma unroll
          for (int e = 0; e < 32; ++e) rr[e] = dead ? 0u : rr[e];
        }
        if (live) {
#pragma unroll
          for (int e8 = 0; e8 < 32; e8 += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(rr[e8 + e]) * f;
            st8<__nv_bfloat16>(op + c0 + e8, v);
          }
        }
        __syncwarp();  // the next read is the whole warp's
      }
    }
    if (P.split > 1) {
      // fp32 O / l and the row's log2-sum-exp of this share, in the operand ring (every P V of
      // both Q tiles has completed once all eight warps are here)
      named_bar_sync(1, 256);
      float* part = reinterpret_cast<float*>(smem);
      float* lse = part + 256 * Cfg::LD_PART;
      const int r = qt * 128 + row;
      const bool some = have && !(l_run < kMaDeadRow);
      if (have) {
        const float inv = some ? 1.f / l_run : 0.f;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t rr[32];
          tmem_read32(o_tmem + uint32_t(c0), rr);
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<float4*>(part + r * Cfg::LD_PART + c0 + e) =
                make_float4(__uint_as_float(rr[e]) * inv, __uint_as_float(rr[e + 1]) * inv,
                            __uint_as_float(rr[e + 2]) * inv, __uint_as_float(rr[e + 3]) * inv);
        }
      }
      lse[r] = some ? m_ref + log2f(l_run) : -INFINITY;
    }
  }
  __syncwarp();
  if (P.split > 1) {
    cluster_sync_all();
    const int u = u0, b = P.sample(u), h = P.head(u), q0 = P.q0(u);
    const int rows = min(256, P.Tq - q0);
    constexpr int C8 = D / 8;
    const uint32_t base = smem_u32(smem);
    // the ranks take the row pieces of 8 columns in turn
    for (int i = int(threadIdx.x) * P.split + rank; i < rows * C8; i += 384 * P.split) {
      const int r = i / C8, c = (i - r * C8) * 8;
      const uint32_t at_l = base + uint32_t(256 * Cfg::LD_PART + r) * 4u;
      const uint32_t at_o = base + uint32_t(r * Cfg::LD_PART + c) * 4u;
      float top = -INFINITY, sum = 0.f, v[8] = {};
      float wl[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        wl[p] = p < P.split ? ld_cluster_f1(mapa_shared(at_l, uint32_t(p))) : -INFINITY;
        top = fmaxf(top, wl[p]);
      }
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if (p < P.split && wl[p] != -INFINITY) {
          const float wp = exp2f(wl[p] - top);
          const uint32_t a = mapa_shared(at_o, uint32_t(p));
          const float4 x = ld_cluster_f4(a), y = ld_cluster_f4(a + 16);
          sum += wp;
          v[0] += wp * x.x; v[1] += wp * x.y; v[2] += wp * x.z; v[3] += wp * x.w;
          v[4] += wp * y.x; v[5] += wp * y.y; v[6] += wp * y.z; v[7] += wp * y.w;
        }
      }
      const int64_t orow = int64_t(b) * P.Tq + q0 + r;
      float f = sum == 0.f ? 0.f : 1.f / sum;
      if (P.gate != nullptr) f *= 2.f / (1.f + __expf(-__bfloat162float(P.gate[orow * P.ld_gate + h])));
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
      st8<__nv_bfloat16>(P.O + orow * P.ldo + int64_t(h) * D + c, v);
    }
    cluster_sync_all();  // no CTA leaves while another reads its part
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// CTAs of a cluster per unit: as many as keep the grid within the SMs, at least two key
// tiles each, 1, 2, 4 or 8.
inline int ma_split(int64_t units, int64_t Tk) {
  int split = 1;
  while (split < 8 && units * split * 2 <= num_sms() && Tk >= 128 * 4 * split) split *= 2;
  return split;
}

template <int D>
void launch_masked_tc(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* o,
                      int64_t ldo, int B, int64_t Tq, int64_t Tk, int H, float scale, const KeyMask& mask,
                      const void* gate, int64_t ld_gate, cudaStream_t s) {
  using Cfg = MaCfg<D>;
  LTX_UNSUPPORTED(Tk <= int64_t(Cfg::MAX_TILES) * 128, "at most 524288 keys under a mask");
  const uint64_t cols = uint64_t(H) * D;
  const CUtensorMap tq = make_tmap_bf16_2d(q, cols, uint64_t(B) * Tq, uint64_t(ldq), 64, 128);
  const CUtensorMap tk = make_tmap_bf16_2d(k, cols, uint64_t(B) * Tk, uint64_t(ldk), 64, 128);
  const CUtensorMap tv = make_tmap_bf16_2d(v, cols, uint64_t(B) * Tk, uint64_t(ldv), 64, 128);
  auto kern = masked_attn_tc_kernel<D>;
  static std::atomic<uint64_t> smem_done{0};
  ensure_smem_limit(smem_done, kern, Cfg::SMEM);
  MaParams p{};
  p.H = H;
  p.Tq = int(Tq);
  p.Tk = int(Tk);
  p.nq2 = int((Tq + 255) / 256);
  const int64_t units = int64_t(B) * H * p.nq2;
  LTX_UNSUPPORTED(units < (int64_t(1) << 31) - 65536, "too many queries for one launch");
  p.units = int(units);
  p.split = ma_split(units, Tk);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.mask = mask;
  p.gate = static_cast<const __nv_bfloat16*>(gate);
  p.ld_gate = ld_gate;
  p.O = static_cast<__nv_bfloat16*>(o);
  p.ldo = ldo;
  const int64_t grid = p.split > 1 ? units * p.split : std::min<int64_t>(units, num_sms());
  launch_pdl(kern, dim3(unsigned(grid)), dim3(384), Cfg::SMEM, s, unsigned(p.split), tq, tk, tv, p);
}

}  // namespace detail
}  // namespace ltx

using namespace ltx;
using namespace ltx::detail;

extern "C" int ltx_attention_masked(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                    int64_t ldv, void* o, int64_t ldo, int B, int64_t Tq, int64_t Tk, int heads,
                                    int head_dim, float scale, const void* mask, int64_t ld_mask, int mask_kind,
                                    const void* gate_logits, int64_t ld_gate, int dtype, void* stream) {
  LTX_API_BEGIN
  LTX_REQUIRE(dtype == LTX_F32 || dtype == LTX_BF16, "dtype must be F32 or BF16");
  LTX_REQUIRE(q && k && v && o && mask, "q, k, v, o and mask must be non-NULL");
  LTX_REQUIRE(B > 0 && Tq > 0 && Tk > 0 && heads > 0, "B, Tq, Tk and heads must be positive");
  LTX_REQUIRE(B < 65536 && heads < 65536, "B and heads must be below 65536");
  LTX_REQUIRE(Tq < (int64_t(1) << 31) / B && Tk < (int64_t(1) << 31) / B, "too many rows");
  LTX_UNSUPPORTED(head_dim == 64 || head_dim == 128 || (dtype == LTX_F32 && head_dim == 32),
                  "masked attention supports head_dim 64 and 128 (and 32 in fp32)");
  const int64_t inner = int64_t(heads) * head_dim;
  LTX_REQUIRE(ldq >= inner && ldk >= inner && ldv >= inner && ldo >= inner, "leading dimensions too small");
  LTX_REQUIRE(mask_kind == LTX_MASK_BOOL || mask_kind == LTX_MASK_F32 || mask_kind == LTX_MASK_BF16, "bad mask_kind");
  LTX_REQUIRE(ld_mask == 0 || ld_mask >= Tk, "ld_mask must be 0 or hold the keys");
  LTX_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  if (gate_logits) LTX_REQUIRE(ld_gate >= heads, "ld_gate must be >= heads");
  LTX_REQUIRE(reinterpret_cast<uintptr_t>(gate_logits) % (dtype == LTX_F32 ? 4 : 2) == 0,
              "gate_logits is not aligned to its type");
  LTX_REQUIRE(ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 8 == 0, "leading dims must be multiples of 8");
  check_vec_ptr(q, "q");
  check_vec_ptr(k, "k");
  check_vec_ptr(v, "v");
  check_vec_ptr(o, "o");
  LTX_REQUIRE(mask_kind == LTX_MASK_BOOL || reinterpret_cast<uintptr_t>(mask) % (mask_kind == LTX_MASK_F32 ? 4 : 2) == 0,
              "mask is not aligned to its type");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const KeyMask km{mask, ld_mask, mask_kind};
  const dim3 grid{unsigned((Tq + 127) / 128), unsigned(heads), unsigned(B)};
  auto run = [&](auto* qp, auto dim) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(qp)>>;
    masked_attn_simt_kernel<T, decltype(dim)::value><<<grid, 128, 0, s>>>(
        qp, ldq, static_cast<const T*>(k), ldk, static_cast<const T*>(v), ldv, static_cast<T*>(o), ldo, int(Tq),
        int(Tk), scale, km, static_cast<const T*>(gate_logits), ld_gate), note_launch();
  };
  if (use_few(B, Tq, heads, head_dim, dtype == LTX_BF16)) {
    const auto few = [&](auto elem, auto dim) {
      launch_masked_few<decltype(elem), decltype(dim)::value>(q, ldq, k, ldk, v, ldv, o, ldo, B, Tq, Tk, heads, scale,
                                                              km, gate_logits, ld_gate, s);
    };
    if (dtype == LTX_BF16)
      head_dim == 64 ? few(__nv_bfloat16{}, std::integral_constant<int, 64>{})
                     : few(__nv_bfloat16{}, std::integral_constant<int, 128>{});
    else if (head_dim == 32)
      few(0.f, std::integral_constant<int, 32>{});
    else
      head_dim == 64 ? few(0.f, std::integral_constant<int, 64>{}) : few(0.f, std::integral_constant<int, 128>{});
  } else if (dtype == LTX_F32) {
    auto qp = static_cast<const float*>(q);
    if (head_dim == 32)
      run(qp, std::integral_constant<int, 32>{});
    else if (head_dim == 64)
      run(qp, std::integral_constant<int, 64>{});
    else
      run(qp, std::integral_constant<int, 128>{});
  } else if (head_dim == 64) {
    launch_masked_tc<64>(q, ldq, k, ldk, v, ldv, o, ldo, B, Tq, Tk, heads, scale, km, gate_logits, ld_gate, s);
  } else {
    launch_masked_tc<128>(q, ldq, k, ldk, v, ldv, o, ldo, B, Tq, Tk, heads, scale, km, gate_logits, ld_gate, s);
  }
  LTX_CUDA(cudaGetLastError());
  LTX_API_END
}
