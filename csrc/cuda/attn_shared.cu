// Attention of one or a few query tokens a sequence over the paged KV cache, for batches whose sequences come in
// groups that share the pages of a prefix.
//
// q        [T, Hq, D] bf16; sequence b owns rows [cu_q[b], cu_q[b+1]) (one row each without cu_q)
// caches   K [pages, Hkv, 16, D], V [pages, Hkv, D, 16]; block_tables [B, max_blocks] int32
// ctx_lens [B]: tokens of each sequence, the query tokens included: query i of nq sees keys < ctx - nq + i + 1
// group_offs [G+1], shared_lens [G]: the tables of sequences [group_offs[g], group_offs[g+1]) agree in their first
//          shared_lens[g] / 16 entries
//
// One warp per (query token, head): running maximum and sum over the keys of the sequence's own table (base 2), D / 32
// output elements a lane.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.cuh"
#include "status.h"

namespace mb {
namespace {

template <int D>
__global__ void attn_shared_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ kc,
                                   const __nv_bfloat16* __restrict__ vc, const int* __restrict__ tables,
                                   const int* __restrict__ ctx_lens, const int* __restrict__ cu_q,
                                   __nv_bfloat16* __restrict__ out, int T, int B, int Hq, int Hkv, int max_blocks,
                                   int pages, float scale_log2, int* status) {
  constexpr int kPer = D / 32;
  pdl_wait();
  pdl_trigger();
  const int row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (row >= T * Hq) return;
  const int t = row / Hq, h = row % Hq, hk = h / (Hq / Hkv);
  int b = t, nq = 1, i = 0;
  if (cu_q) {
    int lo = 0, hi = B;  // the last sequence that begins at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (mid < B && cu_q[mid] <= t) lo = mid; else hi = mid - 1;
    }
    b = lo;
    i = t - cu_q[b];
    nq = cu_q[b + 1] - cu_q[b];
  }
  const int keys = (i >= 0 && i < nq) ? min(ctx_lens[b], max_blocks * 16) - nq + i + 1 : 0;
  float qf[kPer], acc[kPer], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    qf[e] = __bfloat162float(q[(size_t)row * D + lane * kPer + e]) * scale_log2;
    acc[e] = 0.f;
  }
  for (int j = 0; j < keys; ++j) {
    const int page = tables[(size_t)b * max_blocks + j / 16];
    if (page < 0 || page >= pages) {
      set_status(status, kErrBounds);
      continue;
    }
    const __nv_bfloat16* kp = kc + (((size_t)page * Hkv + hk) * 16 + j % 16) * D + lane * kPer;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) s += qf[e] * __bfloat162float(kp[e]);
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    const float corr = exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * corr + p;
    const __nv_bfloat16* vp = vc + (((size_t)page * Hkv + hk) * D + lane * kPer) * 16 + j % 16;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = acc[e] * corr + p * __bfloat162float(vp[e * 16]);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) out[(size_t)row * D + lane * kPer + e] = __float2bfloat16(acc[e] * inv);
}

}  // namespace

void attn_shared(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                 const at::Tensor& block_tables, const at::Tensor& ctx_lens, const c10::optional<at::Tensor>& cu_q,
                 at::Tensor& out, double scale) {
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 && k_cache.scalar_type() == at::kBFloat16 &&
                  v_cache.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16,
              "attn_shared: q, caches and out must be bf16");
  TORCH_CHECK(q.dim() == 3 && q.is_contiguous() && out.is_contiguous() && out.sizes() == q.sizes(),
              "attn_shared: q and out must be contiguous [T, Hq, D]");
  TORCH_CHECK(k_cache.is_contiguous() && v_cache.is_contiguous() && k_cache.dim() == 4 && v_cache.dim() == 4 &&
                  k_cache.size(2) == 16 && v_cache.size(3) == 16 && v_cache.size(2) == k_cache.size(3) &&
                  k_cache.size(0) == v_cache.size(0) && k_cache.size(1) == v_cache.size(1),
              "attn_shared: caches must be contiguous K [pages, Hkv, 16, D] and V [pages, Hkv, D, 16]");
  const int T = (int)q.size(0), Hq = (int)q.size(1), D = (int)q.size(2), Hkv = (int)k_cache.size(1);
  TORCH_CHECK(k_cache.size(3) == D && Hq % Hkv == 0, "attn_shared: heads do not fit the cache");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.is_contiguous(),
              "attn_shared: block_tables must be contiguous int32 [B, max_blocks]");
  if (T == 0) return;
  c10::cuda::CUDAGuard guard(q.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto kernel) {
    launch_k(kernel, (T * Hq + 7) / 8, 256, 0, st, reinterpret_cast<const __nv_bfloat16*>(q.data_ptr()),
             reinterpret_cast<const __nv_bfloat16*>(k_cache.data_ptr()),
             reinterpret_cast<const __nv_bfloat16*>(v_cache.data_ptr()), block_tables.data_ptr<int>(),
             ctx_lens.data_ptr<int>(), cu_q ? cu_q->data_ptr<int>() : nullptr,
             reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), T, (int)block_tables.size(0), Hq, Hkv,
             (int)block_tables.size(1), (int)k_cache.size(0), (float)(scale * 1.4426950408889634),
             status_ptr(q.device().index()));
  };
  if (D == 64) go(attn_shared_kernel<64>);
  else if (D == 128) go(attn_shared_kernel<128>);
  else if (D == 256) go(attn_shared_kernel<256>);
  else TORCH_CHECK(false, "attn_shared: head_dim must be 64, 128 or 256");
}

}  // namespace mb
