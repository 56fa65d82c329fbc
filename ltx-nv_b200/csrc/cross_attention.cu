// Attention with a per-sample key mask: softmax(Q K^T * scale + mask) V per (sample,
// head), Tq queries and Tk keys of another length (a padded text context), with the
// per-(token, head) output gate 2*sigmoid(logit) of attention.cu. Takes the place of
// sdpa's mask argument (ltx_nn.py:22-26) for masks that do not depend on the query.
//
// A key is left out when its boolean mask is 0, or its additive mask is at or below half
// of the type's lowest finite value (the "lowest value" and -inf conventions alike);
// what K and V hold at such a key (NaN and infinities included) does not reach any
// output. A row whose keys are all left out, or whose scores are all -inf, is zero.
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

// One query per thread, key tiles of 32 in shared memory, online softmax in fp32.
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
  if (dtype == LTX_F32) {
    auto qp = static_cast<const float*>(q);
    if (head_dim == 32)
      run(qp, std::integral_constant<int, 32>{});
    else if (head_dim == 64)
      run(qp, std::integral_constant<int, 64>{});
    else
      run(qp, std::integral_constant<int, 128>{});
  } else {
    auto qp = static_cast<const __nv_bfloat16*>(q);
    if (head_dim == 64)
      run(qp, std::integral_constant<int, 64>{});
    else
      run(qp, std::integral_constant<int, 128>{});
  }
  LTX_CUDA(cudaGetLastError());
  LTX_API_END
}
