// Pages of the KV cache: batched copies across every layer (the data of a fork) and compaction of the pool.
//
// kv_copy_pages: k[l][dst[i]] = k[l][src[i]] and the same for v, in every layer, one launch for up to 64 layers.
// kv_compact: n live pages (those that a row's table refers to within its length) end up as pages 0 .. n-1.  Live
//   pages below n stay; the i-th live page at or past n moves to the i-th dead page below n.  Sources and targets
//   are disjoint, so the moves may run in any order.
// Both are bound by HBM: each moved byte is read and written once.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.cuh"
#include "status.h"

namespace mb {
namespace {

constexpr int kMaxLayers = 64;
struct PagePtrs {
  uint4* p[2 * kMaxLayers];  // K of each layer, then V of each layer
};

// One CTA copies one page of one tensor.  n (device) bounds the pairs when it is given, `pairs` otherwise.
__global__ void copy_pages_kernel(const __grid_constant__ PagePtrs ptrs, const int* __restrict__ src,
                                  const int* __restrict__ dst, const int* __restrict__ n, int pairs, int vecs,
                                  int num_pages, int* status) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x;
  if (i >= (n ? *n : pairs)) return;
  const int s = src[i], d = dst[i];
  if (s < 0 || d < 0) return;
  if (s >= num_pages || d >= num_pages) {
    set_status(status, kErrBounds);
    return;
  }
  uint4* base = ptrs.p[blockIdx.y];
  const uint4* from = base + (size_t)s * vecs;
  uint4* to = base + (size_t)d * vecs;
  for (int j = threadIdx.x; j < vecs; j += blockDim.x) to[j] = from[j];
}

// marks[page] = 1 for every page that a row refers to within its length
__global__ void mark_pages_kernel(const int* __restrict__ tables, const int* __restrict__ lens, int* marks, int width,
                                  int num_pages, int* status) {
  pdl_wait();
  pdl_trigger();
  const int used = min(width, (max(0, lens[blockIdx.x]) + 15) / 16);
  for (int j = threadIdx.x; j < used; j += blockDim.x) {
    const int p = tables[(size_t)blockIdx.x * width + j];
    if (p < 0 || p >= num_pages) set_status(status, kErrBounds);
    else marks[p] = 1;
  }
}

// One thread: the moves and the new id of every page.
__global__ void plan_moves_kernel(const int* __restrict__ marks, int num_pages, int* remap, int* src, int* dst,
                                  int* moves, int* live) {
  pdl_wait();
  pdl_trigger();
  int n = 0;
  for (int p = 0; p < num_pages; ++p) n += marks[p] != 0;
  int hole = 0, m = 0;
  for (int p = 0; p < num_pages; ++p) {
    int to = marks[p] ? p : -1;
    if (marks[p] && p >= n) {
      while (marks[hole]) ++hole;
      src[m] = p;
      dst[m++] = to = hole++;
    }
    remap[p] = to;
  }
  *moves = m;
  *live = n;
}

__global__ void remap_tables_kernel(const int* __restrict__ tables, const int* __restrict__ lens,
                                    const int* __restrict__ remap, int* out, int width, int num_pages) {
  pdl_wait();
  pdl_trigger();
  const int used = min(width, (max(0, lens[blockIdx.x]) + 15) / 16);
  for (int j = threadIdx.x; j < width; j += blockDim.x) {
    const int p = tables[(size_t)blockIdx.x * width + j];
    out[(size_t)blockIdx.x * width + j] = j < used && p >= 0 && p < num_pages ? remap[p] : 0;
  }
}

// The caches' page count and 16-byte vectors a page.
std::pair<int, int> check_caches(const char* who, const std::vector<at::Tensor>& k, const std::vector<at::Tensor>& v) {
  TORCH_CHECK(!k.empty() && k.size() == v.size(), who, ": one K and one V cache for each layer");
  const int64_t pages = k[0].size(0), elems = pages ? k[0].numel() / pages : 0;
  for (const auto* side : {&k, &v})
    for (const auto& t : *side)
      TORCH_CHECK(t.is_cuda() && t.device() == k[0].device() && t.is_contiguous() && t.dim() == 4 &&
                      t.scalar_type() == k[0].scalar_type() && t.size(0) == pages && t.numel() == pages * elems &&
                      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                  who, ": caches must be contiguous 4-d tensors of one type, device, page count and page size");
  TORCH_CHECK(elems * k[0].element_size() % 16 == 0, who, ": a page must be a multiple of 16 bytes");
  return {(int)pages, (int)(elems * k[0].element_size() / 16)};
}

void launch_copies(const std::vector<at::Tensor>& k, const std::vector<at::Tensor>& v, const int* src, const int* dst,
                   const int* n, int pairs, int num_pages, int vecs, cudaStream_t st) {
  for (size_t l0 = 0; l0 < k.size(); l0 += kMaxLayers) {
    const int L = (int)std::min<size_t>(kMaxLayers, k.size() - l0);
    PagePtrs ptrs;
    for (int l = 0; l < L; ++l) {
      ptrs.p[l] = reinterpret_cast<uint4*>(k[l0 + l].data_ptr());
      ptrs.p[L + l] = reinterpret_cast<uint4*>(v[l0 + l].data_ptr());
    }
    launch_k(copy_pages_kernel, dim3(pairs, 2 * L), 256, 0, st, ptrs, src, dst, n, pairs, vecs, num_pages,
             status_ptr(k[0].device().index()));
  }
}

}  // namespace

void kv_copy_pages(const std::vector<at::Tensor>& k, const std::vector<at::Tensor>& v, const at::Tensor& src,
                   const at::Tensor& dst) {
  const auto [pages, vecs] = check_caches("kv_copy_pages", k, v);
  TORCH_CHECK(src.scalar_type() == at::kInt && dst.scalar_type() == at::kInt && src.dim() == 1 &&
                  src.sizes() == dst.sizes() && src.is_contiguous() && dst.is_contiguous() &&
                  src.device() == k[0].device() && dst.device() == k[0].device(),
              "kv_copy_pages: src and dst must be int32 vectors of one length on the caches' device");
  if (src.numel() == 0) return;
  c10::cuda::CUDAGuard guard(k[0].device());
  launch_copies(k, v, src.data_ptr<int>(), dst.data_ptr<int>(), nullptr, (int)src.numel(), pages, vecs,
                at::cuda::getCurrentCUDAStream());
}

void kv_compact(const std::vector<at::Tensor>& k, const std::vector<at::Tensor>& v, const at::Tensor& tables,
                const at::Tensor& lens, at::Tensor& out_tables, at::Tensor& remap, at::Tensor& live,
                at::Tensor& workspace) {
  const auto [pages, vecs] = check_caches("kv_compact", k, v);
  for (const auto& t : {tables, lens, out_tables, remap, live, workspace})
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == k[0].device(),
                "kv_compact: tables, lens and outputs must be contiguous int32 on the caches' device");
  TORCH_CHECK(tables.dim() == 2 && lens.numel() == tables.size(0) && out_tables.sizes() == tables.sizes() &&
                  remap.numel() == pages && live.numel() == 1 && workspace.numel() >= 3 * (int64_t)pages + 1,
              "kv_compact: lens [R], tables and out [R, max_blocks], remap [pages], live [1], workspace [3 pages + 1]");
  c10::cuda::CUDAGuard guard(k[0].device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int R = (int)tables.size(0), W = (int)tables.size(1);
  int* ws = workspace.data_ptr<int>();
  int *marks = ws, *src = ws + pages, *dst = src + pages, *moves = dst + pages;
  int* status = status_ptr(k[0].device().index());
  C10_CUDA_CHECK(cudaMemsetAsync(marks, 0, sizeof(int) * pages, st));
  if (R > 0 && W > 0)
    launch_k(mark_pages_kernel, R, 128, 0, st, tables.data_ptr<int>(), lens.data_ptr<int>(), marks, W, pages, status);
  launch_k(plan_moves_kernel, 1, 1, 0, st, marks, pages, remap.data_ptr<int>(), src, dst, moves, live.data_ptr<int>());
  if (R > 0 && W > 0)
    launch_k(remap_tables_kernel, R, 128, 0, st, tables.data_ptr<int>(), lens.data_ptr<int>(), remap.data_ptr<int>(),
             out_tables.data_ptr<int>(), W, pages);
  if (pages > 1) launch_copies(k, v, src, dst, moves, pages / 2, pages, vecs, st);
}

}  // namespace mb
