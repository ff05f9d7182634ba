// Pages of the KV cache: batched copies across every layer (the data of a fork) and compaction of the pool.
//
// kv_copy_pages: k[l][dst[i]] = k[l][src[i]] and the same for v, in every layer, one launch for up to 64 layers.
// kv_compact: n live pages (those that a row's table refers to within its length) end up as pages 0 .. n-1.  Live
//   pages below n stay; the i-th live page at or past n moves to the i-th dead page below n.  Sources and targets
//   are disjoint, so the moves may run in any order.
// Both are bound by HBM: each moved byte is read and written once.  A copy is a grid of as many CTAs as fit, each taking
// one page of one tensor after another with up to eight 16-byte loads in flight a thread.  The plan of a compaction is one CTA
// with the live pages as bits in shared memory.  Measured on one B200: 333 of 1500 pages of 36 layers (1.57 GB read and
// written) 257 us, 0.93 of the copy rate, after a plan of 11 us; 192 copies of 24 pages of 48 layers (302 MB written)
// 69 us.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.cuh"
#include "status.h"

namespace mb {
namespace {

constexpr int kMaxLayers = 64;
constexpr int kCopyThreads = 256, kPlanThreads = 1024;
constexpr int kMaxPages = 1 << 20;  // bits of the plan's shared memory: 128 KB
struct PagePtrs {
  uint4* p[2 * kMaxLayers];  // K of each layer, then V of each layer
};

// Rows of page ids: what a compaction writes beside the pages.
struct Tables {
  const int *tables, *lens, *remap;
  int* out;
  int rows, width;
};

__device__ __forceinline__ int used_of(const int* lens, int row, int width) {
  return min(width, (int)((max(0, lens[row]) + 15ll) / 16));
}

// Pairs x tensors, one page copy at a time.  n (device) gives the pairs where there is one, `pairs` otherwise.
__global__ void __launch_bounds__(kCopyThreads)
    copy_pages_kernel(const __grid_constant__ PagePtrs ptrs, const int* __restrict__ src, const int* __restrict__ dst,
                      const int* __restrict__ n, int pairs, int tensors, int vecs, int num_pages,
                      const __grid_constant__ Tables t, int* status) {
  pdl_wait();
  pdl_trigger();
  for (int row = blockIdx.x; row < t.rows; row += gridDim.x) {
    const int used = used_of(t.lens, row, t.width);
    for (int j = threadIdx.x; j < t.width; j += kCopyThreads) {
      const int p = j < used ? t.tables[(size_t)row * t.width + j] : -1;
      t.out[(size_t)row * t.width + j] = p >= 0 && p < num_pages ? t.remap[p] : 0;
    }
  }
  const int64_t items = (int64_t)(n ? *n : pairs) * tensors;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int i = (int)(item / tensors), s = src[i], d = dst[i];
    if (s < 0 || d < 0) continue;
    if (s >= num_pages || d >= num_pages) {
      set_status(status, kErrBounds);
      continue;
    }
    uint4* base = ptrs.p[item % tensors];
    const uint4* from = base + (size_t)s * vecs;
    uint4* to = base + (size_t)d * vecs;
    constexpr int kDeep = 8;
    for (int j = threadIdx.x; j < vecs; j += kDeep * kCopyThreads) {
      uint4 x[kDeep];
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (j + k * kCopyThreads < vecs) x[k] = from[j + k * kCopyThreads];
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (j + k * kCopyThreads < vecs) to[j + k * kCopyThreads] = x[k];
    }
  }
}

// Sum over the threads before this one, and over all of them.
__device__ __forceinline__ int2 block_scan(int x, int* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += y;
  }
  __syncthreads();
  if (lane == 31) sh[warp] = s;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += sh[w];
    all += sh[w];
  }
  return make_int2(before + s - x, all);
}

// One CTA: which pages are live, where each goes, and the moves (the i-th live page at or past n to the i-th hole).
__global__ void __launch_bounds__(kPlanThreads)
    plan_moves_kernel(const int* __restrict__ tables, const int* __restrict__ lens, int rows, int width, int num_pages,
                      int* remap, int* src, int* dst, int* moves, int* live, int* status) {
  extern __shared__ uint32_t bits[];
  __shared__ int sh[kPlanThreads / 32];
  const int tid = threadIdx.x, words = (num_pages + 31) / 32;
  for (int i = tid; i < words; i += kPlanThreads) bits[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  for (int row = tid >> 5; row < rows; row += kPlanThreads / 32) {  // a warp a row
    const int used = used_of(lens, row, width);
    for (int j = tid & 31; j < used; j += 32) {
      const int p = tables[(size_t)row * width + j];
      if (p < 0 || p >= num_pages) set_status(status, kErrBounds);
      else atomicOr(&bits[p >> 5], 1u << (p & 31));
    }
  }
  __syncthreads();
  int count = 0;
  for (int i = tid; i < words; i += kPlanThreads) count += __popc(bits[i]);
  const int n = block_scan(count, sh).y;
  int moved = 0, holes = 0;
  for (int base = 0; base < words; base += kPlanThreads) {  // 32 pages a thread, in order
    const int i = base + tid, p0 = i * 32;
    const uint32_t b = i < words ? bits[i] : 0;
    const uint32_t valid = i >= words ? 0u : num_pages - p0 >= 32 ? ~0u : (1u << (num_pages - p0)) - 1;
    const uint32_t low = i >= words || n <= p0 ? 0u : n - p0 >= 32 ? ~0u : (1u << (n - p0)) - 1;  // ids below n
    uint32_t from = b & ~low, to = ~b & low & valid;
    const int2 f = block_scan(__popc(from), sh), t = block_scan(__popc(to), sh);
    for (int k = moved + f.x; from; from &= from - 1) src[k++] = p0 + __ffs(from) - 1;
    for (int k = holes + t.x; to; to &= to - 1) dst[k++] = p0 + __ffs(to) - 1;
    moved += f.y;
    holes += t.y;
  }
  for (int p = tid; p < num_pages; p += kPlanThreads) remap[p] = (bits[p >> 5] >> (p & 31)) & 1 ? p : -1;
  __syncthreads();
  for (int k = tid; k < moved; k += kPlanThreads) remap[src[k]] = dst[k];
  if (tid == 0) {
    *moves = moved;
    *live = n;
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
                   const int* n, int pairs, int num_pages, int vecs, Tables t, cudaStream_t st) {
  const int dev = k[0].device().index();
  static int sms[64] = {0};
  if (!sms[dev]) C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev));
  for (size_t l0 = 0; l0 < k.size(); l0 += kMaxLayers) {
    const int L = (int)std::min<size_t>(kMaxLayers, k.size() - l0);
    PagePtrs ptrs;
    for (int l = 0; l < L; ++l) {
      ptrs.p[l] = reinterpret_cast<uint4*>(k[l0 + l].data_ptr());
      ptrs.p[L + l] = reinterpret_cast<uint4*>(v[l0 + l].data_ptr());
    }
    const int64_t items = std::max<int64_t>((int64_t)pairs * 2 * L, t.rows);
    launch_k(copy_pages_kernel, (unsigned)std::min<int64_t>(items, 8 * sms[dev]), kCopyThreads, 0, st, ptrs, src, dst, n,
             pairs, 2 * L, vecs, num_pages, t, status_ptr(dev));
    t.rows = 0;  // the tables are written once
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
  launch_copies(k, v, src.data_ptr<int>(), dst.data_ptr<int>(), nullptr, (int)src.numel(), pages, vecs, Tables{},
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
                  remap.numel() == pages && live.numel() == 1 && workspace.numel() >= 2 * (int64_t)pages + 1,
              "kv_compact: lens [R], tables and out [R, max_blocks], remap [pages], live [1], workspace [2 pages + 1]");
  TORCH_CHECK(pages <= kMaxPages, "kv_compact: at most ", kMaxPages, " pages");
  c10::cuda::CUDAGuard guard(k[0].device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int dev = k[0].device().index(), R = (int)tables.size(0), W = (int)tables.size(1);
  int *src = workspace.data_ptr<int>(), *dst = src + pages, *moves = dst + pages;
  const int smem = (pages + 31) / 32 * 4;
  static bool attr[64] = {false};
  if (!attr[dev]) {  // whatever this call takes: the 48 KB that need no asking count the kernel's static bytes too
    C10_CUDA_CHECK(cudaFuncSetAttribute(plan_moves_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPages / 8));
    attr[dev] = true;
  }
  launch_k(plan_moves_kernel, 1, kPlanThreads, smem, st, tables.data_ptr<int>(), lens.data_ptr<int>(), W > 0 ? R : 0, W,
           pages, remap.data_ptr<int>(), src, dst, moves, live.data_ptr<int>(), status_ptr(dev));
  Tables t{tables.data_ptr<int>(), lens.data_ptr<int>(), remap.data_ptr<int>(), out_tables.data_ptr<int>(), W > 0 ? R : 0, W};
  if (pages > 1 || t.rows > 0) launch_copies(k, v, src, dst, moves, pages / 2, pages, vecs, t, st);
}

}  // namespace mb
