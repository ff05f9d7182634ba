// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence b owns logits rows [cu[b], cu[b+1]): one for each of its n drafts and one more.  With p_j = softmax(row j
// / temperature) and q_j the distribution that draft d_j was drawn from (all of it on d_j without draft_probs):
//   draft j is accepted where u_j q_j(d_j) < p_j(d_j);
//   at the first refusal the next token is drawn from (p_j - q_j)+, after n acceptances from p_n,
//   as argmax_v r(v) / noise(v) with noise ~ Exp(1) (ties: the lowest id), so emitted tokens follow p.
// temperature <= 0: p_j is 1 at the row's largest logit (lowest id among equals).
// NaN logits count as -inf; rows without a finite or +inf logit accept nothing and give token -1.
//
// One CTA per sequence; statistics of one row after another until a draft is refused.  All sums in fp32.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.cuh"
#include "status.h"

namespace mb {
namespace {

constexpr int kThreads = 1024;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ float logit_at(const T* row, int v) {
  const float x = to_f(row[v]);
  return x != x ? -INFINITY : x;
}

// exp((x - top) / temperature); a row whose top is +inf spreads its mass over the infinite logits
__device__ __forceinline__ float weight(float x, float top, float heat) {
  return x == top ? 1.f : expf(__fdiv_rn(x - top, heat));
}

// The larger score, the lower id among equals.
__device__ __forceinline__ void better(float& s, int& v, float s2, int v2) {
  if (s2 > s || (s2 == s && v2 < v)) {
    s = s2;
    v = v2;
  }
}

struct Best {
  float s;
  int v;
};
__device__ Best block_best(float s, int v, float* sh_s, int* sh_v) {
  for (int o = 16; o > 0; o >>= 1) better(s, v, __shfl_xor_sync(~0u, s, o), __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    sh_s[threadIdx.x >> 5] = s;
    sh_v[threadIdx.x >> 5] = v;
  }
  __syncthreads();
  s = sh_s[0];
  v = sh_v[0];
  for (int w = 1; w < kThreads / 32; ++w) better(s, v, sh_s[w], sh_v[w]);
  return {s, v};
}

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads)
    verify_kernel(const T* __restrict__ logits, const int* __restrict__ cu, const int64_t* __restrict__ drafts,
                  const float* __restrict__ uniforms, const float* __restrict__ noise,
                  const float* __restrict__ temperature, const Q* __restrict__ draft_probs, int* __restrict__ accepted,
                  int64_t* __restrict__ token, float* __restrict__ probs, int K, int V, int rows, int* status) {
  __shared__ float sh_s[kThreads / 32];
  __shared__ int sh_v[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x, tid = threadIdx.x;
  const float heat = temperature[b];
  const bool greedy = !(heat > 0.f);
  const int r0 = cu[b];
  const int n = cu[b + 1] - r0 - 1;
  if (r0 < 0 || n < 0 || n > K || r0 + n >= rows) {
    if (tid == 0) {
      set_status(status, kErrBounds);
      accepted[b] = 0;
      token[b] = -1;
    }
    for (int j = tid; j <= K; j += kThreads) probs[(size_t)b * (K + 1) + j] = 0.f;
    return;
  }
  int a = 0;
  for (;; ++a) {
    const T* row = logits + (size_t)(r0 + a) * V;
    float s = -INFINITY;
    int at = V;
    for (int v = tid; v < V; v += kThreads) better(s, at, logit_at(row, v), v);
    const Best top = block_best(s, at, sh_s, sh_v);
    const bool empty = top.s == -INFINITY;
    float sum = 0.f;
    if (!greedy && !empty)
      for (int v = tid; v < V; v += kThreads) sum += weight(logit_at(row, v), top.s, heat);
    sum = warp_sum(sum);
    __syncthreads();
    if ((tid & 31) == 0) sh_s[tid >> 5] = sum;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < kThreads / 32; ++w) sum += sh_s[w];
    if (greedy) sum = 1.f;
    const int64_t d = a < n ? drafts[(size_t)b * K + a] : -1;
    const Q* qrow = draft_probs && a < n ? draft_probs + ((size_t)b * K + a) * V : nullptr;
    auto p_of = [&](int v) {
      if (greedy) return v == top.v ? 1.f : 0.f;
      return __fdiv_rn(weight(logit_at(row, v), top.s, heat), sum);
    };
    bool pass = false;
    float pd = 0.f;
    if (!empty && d >= 0 && d < V) {
      pd = p_of((int)d);
      pass = uniforms[(size_t)b * K + a] * (qrow ? to_f(qrow[d]) : 1.f) < pd;
    }
    if (pass) {
      if (tid == 0) probs[(size_t)b * (K + 1) + a] = pd;
      continue;
    }
    // the next token: from the rest of p where a draft was refused, else (or where nothing is left) from p
    Best best = {0.f, V};
    for (int full = a < n ? 0 : 1; full < 2 && best.v == V && !empty; ++full) {
      float bs = 0.f;
      int bv = V;
      for (int v = tid; v < V; v += kThreads) {
        float r = p_of(v);
        if (!full) r -= qrow ? to_f(qrow[v]) : (v == d ? 1.f : 0.f);
        if (r > 0.f) better(bs, bv, __fdiv_rn(r, noise[(size_t)b * V + v]), v);
      }
      best = block_best(bs, bv, sh_s, sh_v);
    }
    const int v = best.v < V ? best.v : -1;
    if (tid == 0) {
      accepted[b] = a;
      token[b] = v;
      probs[(size_t)b * (K + 1) + a] = v >= 0 ? p_of(v) : 0.f;
    }
    for (int j = a + 1 + tid; j <= K; j += kThreads) probs[(size_t)b * (K + 1) + j] = 0.f;
    return;
  }
}

}  // namespace

void verify_sampled(const at::Tensor& logits, const at::Tensor& cu, const at::Tensor& drafts,
                    const at::Tensor& uniforms, const at::Tensor& noise, const at::Tensor& temperature,
                    const c10::optional<at::Tensor>& draft_probs, at::Tensor& accepted, at::Tensor& token,
                    at::Tensor& probs) {
  TORCH_CHECK(logits.dim() == 2 && logits.is_contiguous() && logits.is_cuda() &&
                  (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
              "verify_sampled: logits must be contiguous [rows, vocab], bf16 or fp32, on a CUDA device");
  TORCH_CHECK(drafts.dim() == 2 && drafts.scalar_type() == at::kLong, "verify_sampled: drafts must be int64 [B, K]");
  const int64_t B = drafts.size(0), K = drafts.size(1), V = logits.size(1);
  TORCH_CHECK(V > 0 && V < (int64_t)1 << 30, "verify_sampled: vocabulary size out of range");
  TORCH_CHECK(cu.scalar_type() == at::kInt && cu.numel() == B + 1, "verify_sampled: cu must be int32 [B + 1]");
  TORCH_CHECK(uniforms.scalar_type() == at::kFloat && uniforms.sizes() == drafts.sizes(),
              "verify_sampled: uniforms must be fp32 [B, K]");
  TORCH_CHECK(noise.scalar_type() == at::kFloat && noise.dim() == 2 && noise.size(0) == B && noise.size(1) == V,
              "verify_sampled: noise must be fp32 [B, vocab]");
  TORCH_CHECK(temperature.scalar_type() == at::kFloat && temperature.numel() == B,
              "verify_sampled: temperature must be fp32 [B]");
  TORCH_CHECK(accepted.scalar_type() == at::kInt && accepted.numel() == B && token.scalar_type() == at::kLong &&
                  token.numel() == B && probs.scalar_type() == at::kFloat && probs.numel() == B * (K + 1),
              "verify_sampled: outputs must be int32 [B], int64 [B] and fp32 [B, K + 1]");
  for (const auto& t : {cu, drafts, uniforms, noise, temperature, accepted, token, probs})
    TORCH_CHECK(t.is_contiguous() && t.device() == logits.device(),
                "verify_sampled: every tensor must be contiguous and on the logits' device");
  if (draft_probs)
    TORCH_CHECK(draft_probs->dim() == 3 && draft_probs->size(0) == B && draft_probs->size(1) == K &&
                    draft_probs->size(2) == V && draft_probs->is_contiguous() &&
                    draft_probs->device() == logits.device() &&
                    (draft_probs->scalar_type() == at::kFloat || draft_probs->scalar_type() == at::kBFloat16),
                "verify_sampled: draft_probs must be contiguous [B, K, vocab], bf16 or fp32, on the logits' device");
  if (B == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto* lp, auto* qp) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(lp)>>;
    using Q = std::remove_const_t<std::remove_pointer_t<decltype(qp)>>;
    launch_k(verify_kernel<T, Q>, (int)B, kThreads, 0, st, (const T*)lp, cu.data_ptr<int>(), drafts.data_ptr<int64_t>(),
             uniforms.data_ptr<float>(), noise.data_ptr<float>(), temperature.data_ptr<float>(), (const Q*)qp,
             accepted.data_ptr<int>(), token.data_ptr<int64_t>(), probs.data_ptr<float>(), (int)K, (int)V,
             (int)logits.size(0), status_ptr(logits.device().index()));
  };
  const void* lp = logits.data_ptr();
  const void* qp = draft_probs ? draft_probs->data_ptr() : nullptr;
  const bool qb = draft_probs && draft_probs->scalar_type() == at::kBFloat16;
  auto with_q = [&](auto* l) {
    if (qb) go(l, static_cast<const __nv_bfloat16*>(qp));
    else go(l, static_cast<const float*>(qp));
  };
  if (logits.scalar_type() == at::kBFloat16) with_q(static_cast<const __nv_bfloat16*>(lp));
  else with_q(static_cast<const float*>(lp));
}

}  // namespace mb
