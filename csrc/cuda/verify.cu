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
// Bound by HBM: every logit is read once for its row's largest value and sum of exponentials (a CTA for each part of a
// row, its values in registers between the two), and of each sequence one row more with its noise (and q) for the next
// token.  Two launches:
//   rows:  (largest logit, its lowest id, sum of exp((x - largest) / temperature)) of each part of each row;
//   token: every CTA joins its sequence's parts and decides on the drafts, as all CTAs of the sequence do alike, then
//          takes its part of the row that the next token is drawn from; the last one of the sequence joins the parts.
// A draw compares r / noise of all ids.  Approximate bounds of it (2^-16 either way) leave a handful of candidates in a
// part, and only those are computed with the correctly rounded divisions and the full exponential that the outcome is
// defined by: three divisions for each id would take longer than reading it.  Sums are in fp32.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.cuh"
#include "status.h"

namespace mb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMaxDrafts = 1023;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }

// Part `part` of row[0..V): the values at ids id(k, e) in registers, `outside` where there is no id.  Aligned 16-byte
// loads wherever a whole vector lies in the row; the row may begin anywhere.
template <typename T, int VECS>
struct Part {
  static constexpr int kVec = 16 / sizeof(T), kIds = kThreads * VECS * kVec;
  float x[VECS * kVec];
  int first;  // id of x[0]; the next vector is kThreads * kVec ids on
  __device__ __forceinline__ int id(int i) const { return first + (i / kVec) * (kThreads * kVec) + i % kVec; }
  __device__ __forceinline__ void load(const T* row, int V, int part, float outside) {
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kVec);
    first = part * kIds + threadIdx.x * kVec - skew;
    uint4 raw[VECS];
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      const int v = id(k * kVec);
      if (v >= 0 && v + kVec <= V) raw[k] = __ldg(reinterpret_cast<const uint4*>(row + v));
    }
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      const int v = id(k * kVec);
      const T* y = reinterpret_cast<const T*>(&raw[k]);
      if (v >= 0 && v + kVec <= V) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[k * kVec + e] = to_f(y[e]);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) x[k * kVec + e] = v + e >= 0 && v + e < V ? to_f(row[v + e]) : outside;
      }
    }
  }
};

// p[v0 .. v0 + N) within p[0..V): in 16-byte loads (8 bytes of four bf16) where they are aligned.
template <int N, typename X>
__device__ __forceinline__ void load_some(const X* p, int v0, int V, float (&out)[N]) {
  constexpr int kBytes = N * sizeof(X) < 16 ? 8 : 16, kPer = kBytes / sizeof(X);
  if (v0 >= 0 && v0 + N <= V && reinterpret_cast<uintptr_t>(p + v0) % kBytes == 0) {
#pragma unroll
    for (int i = 0; i < N; i += kPer) {
      uint4 raw;
      if constexpr (kBytes == 16) {
        raw = __ldg(reinterpret_cast<const uint4*>(p + v0 + i));
      } else {
        const uint2 half = __ldg(reinterpret_cast<const uint2*>(p + v0 + i));
        raw = make_uint4(half.x, half.y, 0, 0);
      }
      const X* y = reinterpret_cast<const X*>(&raw);
#pragma unroll
      for (int e = 0; e < kPer; ++e) out[i + e] = to_f(y[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = v0 + e >= 0 && v0 + e < V ? to_f(p[v0 + e]) : 1.f;
  }
}

// Parts of a row of V ids, wherever it begins.
template <typename T, int VECS>
int parts_of(int64_t V) {
  using P = Part<T, VECS>;
  return (int)((V + P::kVec - 1 + P::kIds - 1) / P::kIds);
}

__device__ __forceinline__ float no_nan(float x) { return x != x ? -INFINITY : x; }

// exp((x - top) / temperature); a row whose top is +inf spreads its mass over the infinite logits
__device__ __forceinline__ float weight(float x, float top, float heat) {
  return x == top ? 1.f : expf(__fdiv_rn(x - top, heat));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger score, the lower id among equals.
__device__ __forceinline__ void better(float& s, int& v, float s2, int v2) {
  if (s2 > s || (s2 == s && v2 < v)) {
    s = s2;
    v = v2;
  }
}
__device__ __forceinline__ void warp_better(float& s, int& v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(s, v, __shfl_xor_sync(~0u, s, o), __shfl_xor_sync(~0u, v, o));
}
__device__ __forceinline__ float block_max(float x, float* sh) {
  x = warp_max(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = x;
  __syncthreads();
  x = sh[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) x = fmaxf(x, sh[w]);
  return x;
}

struct RowPart {
  float top;
  int at;  // lowest id with it
  float sum;
  int pad;
};
struct TokenPart {
  float s[2];  // best of the rest of p, best of p
  int v[2];
};

struct VerifyArgs {
  const void* logits;
  const void* draft_probs;
  const int* cu;
  const int64_t* drafts;
  const float *uniforms, *noise, *temperature;
  int* accepted;
  int64_t* token;
  float* probs;
  RowPart* rows;      // [B, K + 1, parts]
  TokenPart* tokens;  // [B, parts]
  int* done;          // [B]
  int B, K, V, num_rows, row_parts, token_parts;
  int* status;
};

// Rows of sequence b: the first one and the number of drafts, -1 where they do not lie in the logits.
__device__ __forceinline__ int2 rows_of(const VerifyArgs& a, int b) {
  const int r0 = a.cu[b], n = a.cu[b + 1] - r0 - 1;
  return make_int2(r0, r0 < 0 || n < 0 || n > a.K || r0 + n >= a.num_rows ? -1 : n);
}

template <typename T, int VECS>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ float sh[kWarps];
  __shared__ int at;
  pdl_wait();
  pdl_trigger();
  const int part = blockIdx.x, j = blockIdx.y, b = blockIdx.z;
  if (part == 0 && j == 0 && threadIdx.x == 0) a.done[b] = 0;
  const int2 r = rows_of(a, b);
  if (j > r.y) return;
  Part<T, VECS> p;
  p.load(static_cast<const T*>(a.logits) + (size_t)(r.x + j) * a.V, a.V, part, -INFINITY);
  const float heat = a.temperature[b];
  if (threadIdx.x == 0) at = INT_MAX;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < VECS * p.kVec; ++i) {
    p.x[i] = no_nan(p.x[i]);
    top = fmaxf(top, p.x[i]);
  }
  const float mine = top;
  top = block_max(top, sh);
  float sum = 0.f;
  if (heat > 0.f) {
    if (top != -INFINITY) {
      const float f = 1.4426950408889634f / heat;
#pragma unroll
      for (int i = 0; i < VECS * p.kVec; ++i) sum += p.x[i] == top ? 1.f : ex2((p.x[i] - top) * f);
    }
  } else if (mine == top && top != -INFINITY) {  // greedy: the lowest id is wanted, no sum
    int v = INT_MAX;
#pragma unroll
    for (int i = 0; i < VECS * p.kVec; ++i)
      if (p.x[i] == top) v = min(v, p.id(i));
    atomicMin(&at, v);
  }
  sum = warp_sum(sum);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < kWarps; ++w) sum += sh[w];
    a.rows[((size_t)b * (a.K + 1) + j) * a.row_parts + part] = {top, at, sum, 0};
  }
}

template <typename T, typename Q, int VECS>
__global__ void __launch_bounds__(kThreads) verify_token_kernel(const __grid_constant__ VerifyArgs a) {
  extern __shared__ float dyn[];  // [K + 1] of each: largest logit, sum, p of the draft; lowest id of the largest
  float *tops = dyn, *sums = tops + a.K + 1, *pds = sums + a.K + 1;
  int* ats = reinterpret_cast<int*>(pds + a.K + 1);
  __shared__ float sh[kWarps];
  __shared__ TokenPart best_of[kWarps];
  __shared__ int first_refused, last;
  const int part = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int2 r = rows_of(a, b);
  const int n = r.y;
  if (n < 0) {
    if (part == 0) {
      if (tid == 0) {
        set_status(a.status, kErrBounds);
        a.accepted[b] = 0;
        a.token[b] = -1;
      }
      for (int j = tid; j <= a.K; j += kThreads) a.probs[(size_t)b * (a.K + 1) + j] = 0.f;
    }
    return;
  }
  const T* logits = static_cast<const T*>(a.logits) + (size_t)r.x * a.V;
  const Q* probs = static_cast<const Q*>(a.draft_probs);
  const float heat = a.temperature[b];
  const bool greedy = !(heat > 0.f);
  // p of id v under row j
  auto p_of = [&](float x, int v, int j) {
    if (greedy) return v == ats[j] ? 1.f : 0.f;
    return __fdiv_rn(weight(no_nan(x), tops[j], heat), sums[j]);
  };
  if (tid == 0) first_refused = n;
  __syncthreads();
  for (int j = warp; j <= n; j += kWarps) {  // a warp joins a row's parts and decides on its draft
    const RowPart* rp = a.rows + ((size_t)b * (a.K + 1) + j) * a.row_parts;
    const int64_t d = j < n ? a.drafts[(size_t)b * a.K + j] : -1;
    const bool inside = d >= 0 && d < a.V;
    const float xd = inside ? to_f(logits[(size_t)j * a.V + d]) : -INFINITY;
    const float u = j < n ? a.uniforms[(size_t)b * a.K + j] : 0.f;
    const float qd = inside && probs ? to_f(probs[((size_t)b * a.K + j) * a.V + d]) : 1.f;
    float top = -INFINITY, sum = 0.f;
    int at = INT_MAX;
    for (int i = lane; i < a.row_parts; i += 32) {
      const RowPart x = rp[i];
      const float to = fmaxf(top, x.top);
      if (to != -INFINITY && !greedy)
        sum = (top == to ? sum : sum * ex2((top - to) * (1.4426950408889634f / heat))) +
              (x.top == to ? x.sum : x.sum * ex2((x.top - to) * (1.4426950408889634f / heat)));
      better(top, at, x.top, x.at);
    }
    float all = top;
    int all_at = at;
    warp_better(all, all_at);
    sum = all == -INFINITY || greedy ? 0.f : warp_sum(top == all ? sum : sum * ex2((top - all) * (1.4426950408889634f / heat)));
    if (lane == 0) {
      tops[j] = all;
      sums[j] = greedy ? 1.f : sum;
      ats[j] = all_at;
      const float pd = inside && all != -INFINITY ? p_of(xd, (int)d, j) : 0.f;
      pds[j] = pd;
      if (j < n && !(inside && all != -INFINITY && u * qd < pd)) atomicMin(&first_refused, j);
    }
  }
  __syncthreads();
  const int k = first_refused;
  const bool refused = k < n, empty = tops[k] == -INFINITY;
  const float top = tops[k], sum = sums[k];
  const T* row = logits + (size_t)k * a.V;
  const float* noise = a.noise + (size_t)b * a.V;
  const int64_t d = refused ? a.drafts[(size_t)b * a.K + k] : -1;
  const Q* q = refused && probs ? probs + ((size_t)b * a.K + k) * a.V : nullptr;
  // the next token: from the rest of p where a draft was refused, else (or where nothing is left) from p
  float s1 = 0.f, s2 = 0.f;
  int v1 = INT_MAX, v2 = INT_MAX;
  auto precise = [&](float x, int v) {
    const float p = p_of(x, v, k), z = noise[v];
    if (p > 0.f) better(s2, v2, __fdiv_rn(p, z), v);
    if (refused) {
      const float rest = p - (q ? to_f(q[v]) : v == d ? 1.f : 0.f);
      if (rest > 0.f) better(s1, v1, __fdiv_rn(rest, z), v);
    }
  };
  if (greedy) {
    if (!empty && part == 0 && tid == 0) precise(top, ats[k]);  // p is elsewhere 0
  } else if (!empty) {
    Part<T, VECS> x;
    constexpr int NV = Part<T, VECS>::kVec, N = VECS * NV;
    static_assert(N <= 32, "a candidate is a bit");
    x.load(row, a.V, part, -INFINITY);
    constexpr float kUp = 1.f + 1.f / 65536, kDown = 1.f - 1.f / 65536;
    const float f = 1.4426950408889634f / heat, g = 1.f / sum;
    float hi1[N], hi2[N], lo1 = 0.f, lo2 = 0.f;  // bounds of the scores of the rest and of p
#pragma unroll
    for (int i = 0; i < N; i += NV) {
      const int v0 = x.id(i);
      float z[NV], qv[NV];
      load_some<NV>(noise, v0, a.V, z);
      if (q) load_some<NV>(q, v0, a.V, qv);
#pragma unroll
      for (int e = 0; e < NV; ++e) {
        const int v = v0 + e;
        const float y = no_nan(x.x[i + e]);
        hi1[i + e] = hi2[i + e] = -1.f;
        if (v >= 0 && v < a.V) {
          const float p = (y == top ? 1.f : ex2((y - top) * f)) * g, w = __fdividef(1.f, z[e]);
          hi2[i + e] = p * w * (kUp * kUp);
          lo2 = fmaxf(lo2, p * w * (kDown * kDown));
          if (refused) {
            const float t = q ? qv[e] : v == d ? 1.f : 0.f;
            hi1[i + e] = fmaxf(p * kUp - t, 0.f) * w * kUp;
            lo1 = fmaxf(lo1, (p * kDown - t) * w * kDown);
          }
        }
      }
    }
    lo2 = block_max(lo2, sh);
    lo1 = refused ? block_max(lo1, sh) : 0.f;
    // bounds this small say nothing (a rest that is all rounding, weights next to underflow): everything is a candidate
    if (!(lo1 > 1e-30f)) lo1 = 0.f;
    if (!(lo2 > 1e-30f)) lo2 = 0.f;
    uint32_t candidates = 0;  // of p too where a draft was refused: whether its rest is empty is known in the end
#pragma unroll
    for (int i = 0; i < N; ++i) candidates |= (uint32_t)(hi2[i] >= lo2 || (refused && hi1[i] >= lo1)) << i;
#pragma unroll 1
    for (; candidates; candidates &= candidates - 1) {
      const int v = x.id(__ffs(candidates) - 1);
      precise(to_f(row[v]), v);
    }
  }
  warp_better(s1, v1);
  warp_better(s2, v2);
  if (lane == 0) best_of[warp] = {{s1, s2}, {v1, v2}};
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) {
      better(s1, v1, best_of[w].s[0], best_of[w].v[0]);
      better(s2, v2, best_of[w].s[1], best_of[w].v[1]);
    }
    a.tokens[(size_t)b * a.token_parts + part] = {{s1, s2}, {v1, v2}};
    __threadfence();
    last = atomicAdd(&a.done[b], 1) == a.token_parts - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (warp == 0) {
    s1 = s2 = 0.f;
    v1 = v2 = INT_MAX;
    for (int i = lane; i < a.token_parts; i += 32) {
      const TokenPart x = a.tokens[(size_t)b * a.token_parts + i];
      better(s1, v1, x.s[0], x.v[0]);
      better(s2, v2, x.s[1], x.v[1]);
    }
    warp_better(s1, v1);
    warp_better(s2, v2);
    const int v = v1 < INT_MAX ? v1 : v2 < INT_MAX ? v2 : -1;
    if (lane == 0) {
      a.accepted[b] = k;
      a.token[b] = v;
      a.probs[(size_t)b * (a.K + 1) + k] = v >= 0 ? p_of(to_f(row[v]), v, k) : 0.f;
    }
  }
  for (int j = tid; j <= a.K; j += kThreads)
    if (j != k) a.probs[(size_t)b * (a.K + 1) + j] = j < k ? pds[j] : 0.f;
}

}  // namespace

// Bytes of workspace: parts of the smallest size, whatever the types.
int64_t verify_sampled_ws(int64_t B, int64_t K, int64_t V) {
  const int64_t parts = std::max(parts_of<float, 2>(V), parts_of<__nv_bfloat16, 1>(V));
  return B * ((K + 1) * parts * (int64_t)sizeof(RowPart) + parts * (int64_t)sizeof(TokenPart) + 16);
}

void verify_sampled(const at::Tensor& logits, const at::Tensor& cu, const at::Tensor& drafts,
                    const at::Tensor& uniforms, const at::Tensor& noise, const at::Tensor& temperature,
                    const c10::optional<at::Tensor>& draft_probs, at::Tensor& accepted, at::Tensor& token,
                    at::Tensor& probs, at::Tensor& workspace) {
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
  TORCH_CHECK(K <= kMaxDrafts && B <= 65535, "verify_sampled: at most ", kMaxDrafts, " drafts and 65535 sequences");
  TORCH_CHECK(workspace.is_contiguous() && workspace.device() == logits.device() &&
                  (int64_t)workspace.nbytes() >= verify_sampled_ws(B, K, V) &&
                  reinterpret_cast<uintptr_t>(workspace.data_ptr()) % 16 == 0,
              "verify_sampled: workspace too small");
  if (B == 0) return;
  c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  static int sms = 0;
  if (!sms) C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, logits.device().index()));
  VerifyArgs a;
  a.logits = logits.data_ptr();
  a.draft_probs = draft_probs ? draft_probs->data_ptr() : nullptr;
  a.cu = cu.data_ptr<int>();
  a.drafts = drafts.data_ptr<int64_t>();
  a.uniforms = uniforms.data_ptr<float>(), a.noise = noise.data_ptr<float>();
  a.temperature = temperature.data_ptr<float>();
  a.accepted = accepted.data_ptr<int>(), a.token = token.data_ptr<int64_t>(), a.probs = probs.data_ptr<float>();
  a.B = (int)B, a.K = (int)K, a.V = (int)V, a.num_rows = (int)logits.size(0);
  a.status = status_ptr(logits.device().index());
  // large parts where they fill the GPU twice, small ones where there are few rows
  auto rows = [&](auto* t, auto vecs) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int VECS = decltype(vecs)::value;
    a.row_parts = parts_of<T, VECS>(V);
    launch_k(verify_rows_kernel<T, VECS>, dim3(a.row_parts, (unsigned)(K + 1), (unsigned)B), kThreads, 0, st, a);
  };
  auto tokens = [&](auto* t, auto* qt, auto vecs) {
    using T = std::remove_pointer_t<decltype(t)>;
    using Q = std::remove_pointer_t<decltype(qt)>;
    constexpr int VECS = decltype(vecs)::value;
    a.token_parts = parts_of<T, VECS>(V);
    launch_k(verify_token_kernel<T, Q, VECS>, dim3(a.token_parts, (unsigned)B), kThreads, (size_t)(16 * (K + 1)), st, a);
  };
  auto go = [&](auto* t, auto* qt, auto small, auto large) {
    using T = std::remove_pointer_t<decltype(t)>;
    // one region for both sizes of parts
    const int64_t most = parts_of<T, decltype(small)::value>(V);
    uint8_t* ws = static_cast<uint8_t*>(workspace.data_ptr());
    a.rows = reinterpret_cast<RowPart*>(ws);
    a.tokens = reinterpret_cast<TokenPart*>(ws + B * (K + 1) * most * (int64_t)sizeof(RowPart));
    a.done = reinterpret_cast<int*>(a.tokens + B * most);
    const int64_t wide = parts_of<T, decltype(large)::value>(V);
    if ((int64_t)a.num_rows * wide >= 2 * sms) rows(t, large);
    else rows(t, small);
    if (B * wide >= 2 * sms) tokens(t, qt, large);
    else tokens(t, qt, small);
  };
  auto with_q = [&](auto* t, auto small, auto large) {
    if (draft_probs && draft_probs->scalar_type() == at::kBFloat16) go(t, (__nv_bfloat16*)nullptr, small, large);
    else go(t, (float*)nullptr, small, large);
  };
  // vectors a thread: 8 or 32 ids of bf16 (2 or 8 KB a part), 8 or 16 of fp32 (8 or 16 KB)
  if (logits.scalar_type() == at::kBFloat16)
    with_q((__nv_bfloat16*)nullptr, std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  else
    with_q((float*)nullptr, std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
}

}  // namespace mb
