// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence b owns logits rows [cu[b], cu[b+1]): one for each of its n drafts and one more.  With p_j = softmax(row j
// / temperature) and q_j the distribution that draft d_j was drawn from (all of it on d_j without draft_probs):
//   draft j is accepted where u_j q_j(d_j) < p_j(d_j);
//   at the first refusal the next token is drawn from (p_j - q_j)+, after n acceptances from p_n,
//   as argmax_v r(v) / noise(v) with noise ~ Exp(1) (ties: the lowest id), so emitted tokens follow p.
// temperature <= 0: p_j is 1 at the row's largest logit (lowest id among equals).  Others count as at least 2^-126 and at
// most the largest finite number, between which 1 / temperature and what it multiplies stay numbers.
// NaN logits count as -inf; rows without a finite or +inf logit accept nothing and give token -1.
//
// Bound by HBM: every logit is read once for its row's largest value and sum of exponentials, and of each sequence one
// row more with its noise (and q) for the next token.  Two launches, each of which cuts its rows into as many parts as
// fill the GPU, a CTA each:
//   rows:  (largest logit, its lowest id, sum of exp((x - largest) / temperature)) of each part of each row, with a running
//          maximum and sum in every thread and one reduction in the end;
//   token: every CTA joins its sequence's parts and decides on the drafts, as all CTAs of the sequence do alike, then
//          takes its part of the row that the next token is drawn from; the last one of the sequence joins the parts.
// A draw compares r / noise of all ids.  Each thread keeps approximate bounds of it (2^-16 either way): its largest
// upper bound with the id, the second largest, and the largest lower bound.  An id below its part's largest lower bound
// is out, so that one or two are left, and only those are computed with the correctly rounded divisions and the full
// exponential that the outcome is defined by: three divisions for each id take longer than reading it.  Sums are in fp32.
//
// Measured on one B200: 64 sequences with 0 to 4 drafts, 151936 ids, bf16: 39 us in a CUDA graph, about half for the 52 MB
// of logits (170 rows) and half for the draws (39 MB of noise).  Neither end is reached: the first launch runs 12
// instructions a logit with 55 to 58% of the issue slots taken at 2.5 TB/s and 41% of the warps resident, the second 46% at
// 1.7 TB/s and 27%, so that the latency of loads that too few warps cover bounds both.  24 sequences with a draft model's
// probabilities in fp32 27 us; one sequence 14 us, a chain of dependent loads.
#include <cfloat>

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

// N neighbouring values, loaded as 16-byte vectors (8 bytes of four bf16).  Loading and looking are apart so that the
// loads of several are under way together.
template <int N, typename X>
struct Vec {
  static constexpr int kWords = N * (int)sizeof(X) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const X* p, bool ok) {
    if constexpr (kWords == 2) {
      if (ok) {
        const uint2 y = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = y.x, w[1] = y.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        if (ok) {
          const uint4 y = __ldg(reinterpret_cast<const uint4*>(p) + i / 4);
          w[i] = y.x, w[i + 1] = y.y, w[i + 2] = y.z, w[i + 3] = y.w;
        }
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(X) == 4) return __uint_as_float(w[e]);
    else return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
  }
  static __device__ __forceinline__ bool aligned(const X* p) {
    return reinterpret_cast<uintptr_t>(p) % (kWords == 2 ? 8 : 16) == 0;
  }
};
// p[v .. v + N) one by one, `outside` where [0, end) does not reach.
template <int N, typename X>
__device__ __forceinline__ void load_each(const X* p, int v, int end, float outside, float (&x)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = v + e >= 0 && v + e < end ? to_f(p[v + e]) : outside;
}

// A thread's ids of part `part` of a row: kIds = 16 bytes' worth from each of at(0), at(1), ... while they are below end.
// The vectors lie on 16-byte boundaries wherever the row begins.
template <typename T>
struct Span {
  static constexpr int kIds = 16 / sizeof(T), kStep = kThreads * kIds;
  int first, end;
  __device__ __forceinline__ Span(const T* row, int V, int part, int steps) {
    const int skew = (int)((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kIds);
    first = part * steps * kStep + threadIdx.x * kIds - skew;
    end = min(V, (part + 1) * steps * kStep - skew);
  }
};

// Steps (of a CTA's 4 KB) a part and parts a row for `rows` rows of V ids: parts that fill `ctas` places once.
template <typename T>
void cut(int64_t V, int64_t rows, int64_t ctas, int& steps, int& parts) {
  const int64_t all = (V + Span<T>::kIds - 1 + Span<T>::kStep - 1) / Span<T>::kStep;  // a row may begin inside a vector
  const int64_t want = std::min(all, std::max<int64_t>(1, ctas / std::max<int64_t>(1, rows)));
  steps = (int)((all + want - 1) / want);
  parts = (int)((all + steps - 1) / steps);
}

__device__ __forceinline__ float no_nan(float x) { return fmaxf(x, -INFINITY); }

// exp((x - top) / temperature); a row whose top is +inf spreads its mass over the infinite logits
__device__ __forceinline__ float weight(float x, float top, float heat) {
  return x == top ? 1.f : expf(__fdiv_rn(x - top, heat));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float ex2_ftz(float x) {  // without results below 2^-126, one instruction
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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
  float s;  // the best score and its id
  int v;
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
  int B, K, V, num_rows, row_steps, row_parts, token_steps, token_parts;
  int* status;
};

__device__ __forceinline__ float heat_of(const VerifyArgs& a, int b) {
  const float t = a.temperature[b];
  return t > 0.f ? fminf(fmaxf(t, FLT_MIN), FLT_MAX) : t;
}

// Rows of sequence b: the first one and the number of drafts, -1 where they do not lie in the logits.
__device__ __forceinline__ int2 rows_of(const VerifyArgs& a, int b) {
  const int r0 = a.cu[b], r1 = a.cu[b + 1];  // compared with the ends before they are subtracted: nothing overflows
  return make_int2(r0, r0 < 0 || r1 <= r0 || r1 > a.num_rows || r1 - r0 - 1 > a.K ? -1 : r1 - r0 - 1);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_rows_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ float sh[kWarps];
  __shared__ int at;
  pdl_wait();
  pdl_trigger();
  const int part = blockIdx.x, j = blockIdx.y, b = blockIdx.z;
  if (part == 0 && j == 0 && threadIdx.x == 0) a.done[b] = 0;
  const float heat = heat_of(a, b);
  const int2 r = rows_of(a, b);
  if (j > r.y) return;
  if (threadIdx.x == 0) at = INT_MAX;
  const T* row = static_cast<const T*>(a.logits) + (size_t)(r.x + j) * a.V;
  const Span<T> ids(row, a.V, part, a.row_steps);
  constexpr int N = Span<T>::kIds, kStep = Span<T>::kStep, kDeep = 4;
  const bool greedy = !(heat > 0.f);
  const float f = greedy ? 0.f : 1.4426950408889634f / heat;
  float top = -INFINITY, sum = 0.f;
  int mine = INT_MAX;
  for (int v0 = ids.first; v0 < ids.end; v0 += kDeep * kStep) {
    Vec<N, T> raw[kDeep];
    bool in[kDeep];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int v = v0 + k * kStep;
      in[k] = v >= 0 && v + N <= ids.end;
      raw[k].load(row + v, in[k]);
    }
    float x[kDeep][N];
#pragma unroll
    for (int k = 0; k < kDeep; ++k) {
      const int v = v0 + k * kStep;
      if (!in[k]) {  // the row's ends
        load_each<N>(row, v, v < ids.end ? ids.end : 0, -INFINITY, x[k]);
#pragma unroll
        for (int e = 0; e < N; ++e) x[k][e] = no_nan(x[k][e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[k][e] = no_nan(raw[k].get(e));
      }
    }
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) m = fmaxf(m, x[k][e]);
    if (m == -INFINITY) continue;
    if (greedy) {
      if (m > top) {
        top = m;
#pragma unroll
        for (int k = kDeep - 1; k >= 0; --k)
#pragma unroll
          for (int e = N - 1; e >= 0; --e)
            if (x[k][e] == m) mine = v0 + k * kStep + e;
      }
      continue;
    }
    if (m > top) {
      sum *= ex2((top - m) * f);
      top = m;
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e)
        s[e & 3] += top == INFINITY ? (x[k][e] == top ? 1.f : 0.f) : ex2_ftz((x[k][e] - top) * f);
    sum += (s[0] + s[1]) + (s[2] + s[3]);
  }
  const float all = block_max(top, sh);
  if (greedy) {
    if (top == all && mine != INT_MAX) atomicMin(&at, mine);
  } else {
    sum = top == all || top == -INFINITY ? sum : sum * ex2((top - all) * f);
  }
  sum = warp_sum(sum);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < kWarps; ++w) sum += sh[w];
    a.rows[((size_t)b * (a.K + 1) + j) * a.row_parts + part] = {all, at, sum, 0};
  }
}

template <typename T, typename Q>
__global__ void __launch_bounds__(kThreads, 3) verify_token_kernel(const __grid_constant__ VerifyArgs a) {
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
  const float heat = heat_of(a, b);
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
  float best = 0.f;
  int at = INT_MAX;
  auto precise = [&](int v, bool rest) {
    float p = p_of(to_f(row[v]), v, k);
    if (rest) p -= q ? to_f(q[v]) : v == d ? 1.f : 0.f;
    if (p > 0.f) better(best, at, __fdiv_rn(p, noise[v]), v);
  };
  if (greedy) {
    if (!empty && part == 0 && tid == 0) precise(ats[k], refused);  // p is elsewhere 0
  } else if (!empty) {
    const Span<T> ids(row, a.V, part, a.token_steps);
    constexpr int N = Span<T>::kIds, kStep = Span<T>::kStep;
    constexpr float kUp = 1.f + 1.f / 65536, kDown = 1.f - 1.f / 65536, kTiny = 1.2e-38f;
    const float f = 1.4426950408889634f / heat;
    const bool z_ok = Vec<N, float>::aligned(noise + ids.first), q_ok = q && Vec<N, Q>::aligned(q + ids.first);
    float up1 = 0.f, up2 = 0.f, low = 0.f;  // the two largest upper bounds, the largest lower one
    int id1 = -1;
    // `take` sees N ids from v on with their logits and noise; where the row does not reach, -inf and 1
    auto each = [&](auto take) {
      constexpr int kDeep = 2;
      for (int v0 = ids.first; v0 < ids.end; v0 += kDeep * kStep) {
        Vec<N, T> raw[kDeep];
        Vec<N, float> zs[kDeep];
        bool in[kDeep];
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
          const int v = v0 + k * kStep;
          in[k] = v >= 0 && v + N <= ids.end;
          raw[k].load(row + v, in[k]);
          zs[k].load(noise + v, in[k] && z_ok);
        }
#pragma unroll
        for (int k = 0; k < kDeep; ++k) {
          const int v = v0 + k * kStep, end = v < ids.end ? ids.end : 0;
          float x[N], z[N];
          if (in[k]) {
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] = raw[k].get(e);
          } else {
            load_each<N>(row, v, end, -INFINITY, x);
          }
          if (in[k] && z_ok) {
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = zs[k].get(e);
          } else {
            load_each<N>(noise, v, end, 1.f, z);
          }
          take(v, end, in[k], x, z);
        }
      }
    };
    if (!q) {
      // p but for its factor: 2^(60 + ...) keeps every p that is not zero in 32 bits above the flush to zero
      const int only = refused && d >= 0 && d < a.V ? (int)d : -1;  // a certain draft's rest: p elsewhere
      each([&](int v, int, bool, float (&x)[N], float (&z)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float p = ex2_ftz(fmaf(no_nan(x[e]) - top, f, 60.f));
          if (top == INFINITY) p = x[e] == top ? 1.f : 0.f;
          const float s = v + e == only ? 0.f : p * __fdividef(1.f, z[e]);
          up2 = fmaxf(up2, fminf(s, up1));
          if (s > up1) id1 = v + e;
          up1 = fmaxf(up1, s);
        }
      });
      const float g = (top == INFINITY ? 1.f : 0x1p-60f) / sum;
      low = up1 * g * (kDown * kDown);
      up1 *= g * (kUp * kUp);
      up2 *= g * (kUp * kUp);
    } else {
      const float g = 1.f / sum;
      each([&](int v, int end, bool in, float (&x)[N], float (&z)[N]) {
        float t[N];
        if (in && q_ok) {
          Vec<N, Q> qs;
          qs.load(q + v, true);
#pragma unroll
          for (int e = 0; e < N; ++e) t[e] = qs.get(e);
        } else {
          load_each<N>(q, v, end, 2.f, t);  // 2: outside, nothing is left
        }
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float y = no_nan(x[e]), w = __fdividef(1.f, z[e]);
          const float p = (y == top ? 1.f : ex2_ftz((y - top) * f)) * g;
          const float s = fmaxf(fmaf(p, kUp, kTiny) - t[e], 0.f) * w * kUp;  // kTiny: a p that was flushed to zero
          low = fmaxf(low, (p * kDown - t[e]) * w * kDown);
          up2 = fmaxf(up2, fminf(s, up1));
          if (s > up1) id1 = v + e;
          up1 = fmaxf(up1, s);
        }
      });
    }
    const float most = block_max(up1, sh);
    low = block_max(low, sh);
    // Bounds near underflow say nothing.  Such a part has no winner where the row's largest logit is in the race, whose
    // score is at least 1 / (V noise); else (it was refused, or q leaves rounding only) every id of it is computed.
    const bool top_runs = !refused || (!q && !(d >= 0 && d < a.V && to_f(row[d]) == top));
    if (most == 0.f || (!(low > 1e-30f) && top_runs)) {
    } else if (!(low > 1e-30f) || up2 >= low) {
      for (int v0 = ids.first; v0 < ids.end; v0 += kStep)
        for (int v = max(v0, 0); v < min(v0 + N, ids.end); ++v) precise(v, refused);
    } else if (up1 >= low) {
      precise(id1, refused);
    }
  }
  warp_better(best, at);
  if (lane == 0) best_of[warp] = {best, at};
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kWarps; ++w) better(best, at, best_of[w].s, best_of[w].v);
    a.tokens[(size_t)b * a.token_parts + part] = {best, at};
    __threadfence();
    last = atomicAdd(&a.done[b], 1) == a.token_parts - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  best = 0.f;
  at = INT_MAX;
  if (tid < 32) {
    for (int i = lane; i < a.token_parts; i += 32) {
      const TokenPart x = a.tokens[(size_t)b * a.token_parts + i];
      better(best, at, x.s, x.v);
    }
    warp_better(best, at);
    if (lane == 0) best_of[0] = {best, at};
  }
  __syncthreads();
  if (best_of[0].v == INT_MAX && refused && !empty) {  // q took all of p: the whole row again, from p
    best = 0.f;
    at = INT_MAX;
    for (int v = tid; v < a.V; v += kThreads) precise(v, false);
    warp_better(best, at);
    __syncthreads();
    if (lane == 0) best_of[warp] = {best, at};
    __syncthreads();
    if (tid == 0)
      for (int w = 1; w < kWarps; ++w) better(best_of[0].s, best_of[0].v, best_of[w].s, best_of[w].v);
    __syncthreads();
  }
  if (warp == 0) {
    const int v = best_of[0].v < INT_MAX ? best_of[0].v : -1;
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

// Bytes of workspace, whatever the types: parts of 4 KB.
int64_t verify_sampled_ws(int64_t B, int64_t K, int64_t V) {
  const int64_t parts = (V + 1024 + 8) / 1024 + 1;
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
  auto go = [&](auto* t, auto* qt) {
    using T = std::remove_pointer_t<decltype(t)>;
    using Q = std::remove_pointer_t<decltype(qt)>;
    // as many CTAs as are resident: four an SM for the rows, three for the token, whose threads hold more
    cut<T>(V, a.num_rows, 4 * sms, a.row_steps, a.row_parts);
    cut<T>(V, B, 3 * sms, a.token_steps, a.token_parts);
    uint8_t* ws = static_cast<uint8_t*>(workspace.data_ptr());
    a.rows = reinterpret_cast<RowPart*>(ws);
    a.tokens = reinterpret_cast<TokenPart*>(a.rows + B * (K + 1) * a.row_parts);
    a.done = reinterpret_cast<int*>(a.tokens + B * a.token_parts);
    launch_k(verify_rows_kernel<T>, dim3(a.row_parts, (unsigned)(K + 1), (unsigned)B), kThreads, 0, st, a);
    launch_k(verify_token_kernel<T, Q>, dim3(a.token_parts, (unsigned)B), kThreads, (size_t)(16 * (K + 1)), st, a);
  };
  auto with_q = [&](auto* t) {
    if (draft_probs && draft_probs->scalar_type() == at::kBFloat16) go(t, (__nv_bfloat16*)nullptr);
    else go(t, (float*)nullptr);
  };
  if (logits.scalar_type() == at::kBFloat16) with_q((__nv_bfloat16*)nullptr);
  else with_q((float*)nullptr);
}

}  // namespace mb
