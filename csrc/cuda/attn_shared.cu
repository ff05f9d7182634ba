// Attention of one or a few query tokens a sequence over the paged KV cache, for batches whose sequences come in
// groups that share the pages of a prefix.
//
// q        [T, Hq, D] bf16; sequence b owns rows [cu_q[b], cu_q[b+1]) (one row each without cu_q)
// caches   K [pages, Hkv, 16, D], V [pages, Hkv, D, 16]; block_tables [B, max_blocks] int32
// ctx_lens [B]: tokens of each sequence, the query tokens included: query i of nq sees keys < ctx - nq + i + 1
// group_offs [G+1], shared_lens [G]: the tables of sequences [group_offs[g], group_offs[g+1]) agree in their first
//          shared_lens[g] / 16 entries
//
// Mathematics: with o = sum_j 2^(s_j - m) v_j and l = sum_j 2^(s_j - m) over a set of keys (s in units of log2 e), two
// sets join as o 2^(m - M) + o' 2^(m' - M), l likewise, M = max(m, m').  So a group's prefix is computed once for all
// of its rows (a row is a query token and a query head of one KV head's group), each sequence's own tokens for its own
// rows, and long key ranges are cut anywhere.
//
// Three launches after the step's plan: own tokens of few rows (lean kernel), the other units (attention kernel), join
// (merge kernel).
//
// Work of the attention kernel: a unit is up to 256 rows that read one key range for one KV head: a group's prefix (256
// rows: two 128-row tiles against the same key tiles) or the own tokens of a sequence with many query rows (128 rows).
// The plan kernel lists the units of a step with their costs and cuts the list into equal shares, one for every SM, at
// key-tile boundaries, so that long and short prefixes fill the GPU alike.  Units that a cut divides, and rows that have
// a prefix and a tail, leave (o, m, l) partials in fp32 which the merge kernel joins; the others are written at once.
//
// The attention kernel is one persistent CTA per SM:
//   TMA warp   : key tiles (K, then V) of 64 tokens, one copy per page, into a ring of slots
//   Q warp     : the rows of the next pieces into two tile buffers (128-byte swizzle; by cp.async where the heads of a
//                group do not divide a tile)
//   2 MMA warps: S = Q.K^T (fp32 in TMEM), O += P.V with P read from TMEM, where it overwrites S as bf16: 32 columns of S
//                hold 32 keys' P
//   2 x 4 warps: softmax of one 128-row tile each, a row a thread; a row's O is rescaled only where its running
//                maximum has grown by more than 2^8 (P stays below 256, so bf16 and fp32 lose nothing)
// The two tiles are independent pipelines that share the tensor cores, and each has two S: while the softmax of one
// runs, the products of the other are done.  A piece of one tile only lets its even and odd key tiles take the two
// pipelines and joins their halves in TMEM.  At D = 256 TMEM holds one pipeline.
//
// Sums, maxima and O are in fp32.  P enters the second product as two bf16 terms (16 bits of it): one term alone makes the
// whole result's error 1.4 times that of its final rounding, two cost 1 to 4% of the time (132 -> 133 us on 32768 shared
// tokens under 128 sequences, 33 -> 35 us on 8192 under 64).
// Token slots past the context may hold anything: their scores are masked by selection and their V columns are zeroed
// in shared memory.  Every wait is bounded.
//
// Measured on one B200 (a layer's three launches in a CUDA graph; the step's plan is another 10 us, 12 with 128 sequences):
// 32 heads on 4 KV heads, 32768 shared tokens under 128 sequences with up to 1024 own: 129 to 137 us from run to run, 540
// TFLOP/s.  A 64-key step of 256 rows takes 2250 clocks more (counters at 8192 and 16384 shared tokens), of which the tensor
// cores are busy 1570 (three products, one of them for the second term of P) and the special-function units 1024; a tile's
// chain of product, softmax (about 1450 in each of two warps an SM quarter) and product fills the rest.  55 steps an SM are
// 63 us at 1965 MHz, 71 at the 1747 that such calls one after another settle at under the power limit; the own tokens take 28
// before them, starts, partial rows and the join what remains.  2048 shared under 64 with up to 512 own: 29 us, of which
// about 12 the own tokens, 11 the prefix (a start of 4500 clocks and 9000 clocks to write 256 partial rows an SM around one
// step) and the rest the join.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "launch.cuh"
#include "status.h"

namespace mb {

PFN_cuTensorMapEncodeTiled_v12000 get_encode();

namespace {

constexpr int kWideRows = 256;    // rows of a prefix unit at D <= 128 (two tiles)
constexpr int kTileRows = 128;
constexpr int kTileKeys = 64;
constexpr int kNoLimit = 1 << 29;
// Own tokens of up to kLeanRows rows a sequence take the lean kernel (D <= 128): 20 rows of drafts 34 us there, 36 us as
// units of the attention kernel.
constexpr int kLeanRows = 64;
constexpr int kLeanWarps = 16;    // lean pieces aimed at, for each SM
constexpr int kLeanPages = 8;     // least pages of a piece (4 instead: -2 us on drafts, +2 us on 8 x 16 samples)

// Costs: a tile of keys against one and against two tiles of rows, and a unit's start and end.  A share costs its partial
// rows, written and read again, so none is cheaper than kCostShare (measured 1 / 8 / 12 / 24 / 40: 16 sequences on 8192
// tokens 27 / 25 / 23 / 25 / 32 us, 64 on 2048 31 / 30 / 33 / 36 / 43 us).
constexpr int kCostNarrow = 2, kCostWide = 3, kCostUnit = 8;
constexpr int kCostShare = 8;

struct Unit {
  int row0;      // first row, in (token, head of the group) order
  int rows;
  int seq;       // whose table is read
  int key0;      // first key (a multiple of 16)
  int key_end;   // past the last key that any row sees
  int lim;       // query token t sees keys < lim + t
  int solo;      // no other unit has keys for these rows
  int tiles;
};

// A lean piece: up to 16 rows of a sequence against some pages of its table.
struct Piece {
  int row0, rows, seq;
  int page0, pages;  // entries of the table
  int ctx, lim;      // query token t sees keys < min(ctx, lim + t)
  int direct;        // these are all the keys of its rows
};

// The plan's parts in one int32 buffer.
struct PlanView {
  int* lean;    // [max_pieces] Piece
  int* seqs;    // [B] (first lean piece, pieces of 16 rows)
  int* hdr;     // [4]: units of a head, cost of a head's units, rows of a head's units, lean pieces of a head
  int* units;   // [max_units] Unit
  int* cost;    // [max_units + 1] exclusive sums
  int* rowcum;  // [max_units] exclusive sums
  int* cuts;    // [shares + 1] (unit, tile)
  int* inside;  // [heads * max_units] (first share that begins inside the unit, how many do)
  int* tok;     // [T] (first prefix unit or -1, group's first token, own tokens, sequence's first token);
                // own tokens: -1 none, the first unit, or -2 - b where they are sequence b's lean pieces
};

struct PlanDims {
  int T, B, G, Gq, Hkv, wide_rows, shares, max_blocks, max_units, max_pieces, lean_rows;
};

__host__ __device__ inline int64_t plan_ints(const PlanDims& d) {
  return 4 + (int64_t)d.max_units * 8 + (d.max_units + 1) + d.max_units + 2 * (d.shares + 1) +
         2 * (int64_t)d.Hkv * d.max_units + 4 * (int64_t)d.T + 8 * (int64_t)d.max_pieces + 2 * (int64_t)d.B + 16;
}

__host__ __device__ inline PlanView plan_view(int* p, const PlanDims& d) {
  PlanView v;
  v.tok = p;  // 16-byte records first
  v.units = v.tok + 4 * (size_t)d.T;
  v.lean = v.units + (size_t)d.max_units * 8;
  v.hdr = v.lean + (size_t)d.max_pieces * 8;
  v.seqs = v.hdr + 4;
  v.cuts = v.seqs + 2 * (size_t)d.B;
  v.inside = v.cuts + 2 * (d.shares + 1);
  v.cost = v.inside + 2 * (size_t)d.Hkv * d.max_units;
  v.rowcum = v.cost + d.max_units + 1;
  return v;
}

// ------------------------------------------------------------------------------------------------ plan
constexpr int kPlanThreads = 1024;

// Exclusive sums of a[0..n) in place, the total in a[n]; every thread of the block calls it.
__device__ void block_scan(int* a, int n, int* sh) {
  int carry = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int x = i < n ? a[i] : 0;
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, s, o);
      if (lane >= o) s += y;
    }
    if (lane == 31) sh[warp] = s;
    __syncthreads();
    if (warp == 0) {
      int w = sh[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, w, o);
        if (lane >= o) w += y;
      }
      sh[lane] = w;
    }
    __syncthreads();
    if (i < n) a[i] = carry + s - x + (warp ? sh[warp - 1] : 0);
    carry += sh[31];
    __syncthreads();
  }
  if (threadIdx.x == 0) a[n] = carry;
  __syncthreads();
}

// *total += x of every thread; each thread of the block calls it.  One shared-memory addition a warp: 64-bit ones are retried
// where threads collide, and 128 sequences made the plan 6 us longer that way.
__device__ __forceinline__ void add_all(unsigned long long* total, unsigned long long x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  if ((threadIdx.x & 31) == 0 && x) atomicAdd(total, x);
}

// The last i of [0, n) with a[i] <= x (a ascending), -1 if there is none.
__device__ __forceinline__ int last_le(const int* a, int n, int x) {
  int lo = -1, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// One CTA, once a step; every layer's launches use its result.
__global__ void __launch_bounds__(kPlanThreads)
    attn_shared_plan_kernel(const int* __restrict__ ctx_lens, const int* __restrict__ group_offs,
                            const int* __restrict__ shared_lens, const int* __restrict__ cu_q, int* plan, PlanDims d,
                            int* status) {
  extern __shared__ int sm[];
  __shared__ int sh[32];
  int* offs = sm;                 // [G + 1]
  int* pre = offs + d.G + 1;      // [G] prefix tokens that are computed once
  int* lead = pre + d.G;          // [G] first sequence with a context
  int* gu = lead + d.G;           // [G + 1] prefix units
  int* su = gu + d.G + 1;         // [B + 1] own units
  int* le = su + d.B + 1;         // [B + 1] lean pieces
  int* cu = le + d.B + 1;         // [B + 1]
  __shared__ unsigned long long lean_pages, total_cost;  // past 32 bits with thousands of long sequences
  const PlanView v = plan_view(plan, d);
  const int tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) lean_pages = total_cost = 0;
  for (int i = tid; i <= d.G; i += kPlanThreads) offs[i] = min(max(group_offs[i], 0), d.B);
  for (int i = tid; i < d.G; i += kPlanThreads) {
    pre[i] = max(shared_lens[i], 0) & ~15;
    lead[i] = INT_MAX;
  }
  for (int i = tid; i <= d.B; i += kPlanThreads) cu[i] = cu_q ? min(max(cu_q[i], 0), d.T) : i;
  __syncthreads();
  // What follows searches both: offsets that descend make a plan of nothing (every row is written as zeros).
  bool bad = false;
  for (int i = tid; i < d.G; i += kPlanThreads) bad |= offs[i + 1] < offs[i];
  for (int i = tid; i < d.B; i += kPlanThreads) bad |= cu[i + 1] < cu[i];
  bad = __syncthreads_or(bad);
  auto group_of = [&](int b) {
    const int g = last_le(offs, d.G + 1, b);
    return g >= 0 && g < d.G ? g : -1;
  };
  auto ctx_of = [&](int b) { return min(max(ctx_lens[b], 0), d.max_blocks * 16); };
  // a prefix ends before the first query token of every sequence of its group: its rows see all of it
  for (int b = tid; b < d.B; b += kPlanThreads) {
    const int g = group_of(b), c = ctx_of(b), nq = cu[b + 1] - cu[b];
    if (g >= 0 && c > 0 && nq > 0) {
      atomicMin(&pre[g], max(0, c - nq) & ~15);
      atomicMin(&lead[g], b);
    }
  }
  __syncthreads();
  for (int g = tid; g < d.G; g += kPlanThreads) {
    const int s0 = offs[g], s1 = offs[g + 1];
    if (s1 - s0 < 2 || lead[g] == INT_MAX) pre[g] = 0;  // nobody to share with: the sequence's own unit takes it all
    const int rows = bad ? 0 : (cu[s1] - cu[s0]) * d.Gq;
    gu[g] = pre[g] > 0 ? (rows + d.wide_rows - 1) / d.wide_rows : 0;
  }
  __syncthreads();
  unsigned long long mine = 0;
  for (int b = tid; b < d.B; b += kPlanThreads) {
    const int g = group_of(b), p = g >= 0 ? pre[g] : 0, c = ctx_of(b), rows = (cu[b + 1] - cu[b]) * d.Gq;
    const bool any = c > p && rows > 0, lean = rows <= d.lean_rows;
    su[b] = any && !lean ? (rows + kTileRows - 1) / kTileRows : 0;
    le[b] = any && lean ? (rows + 15) / 16 : 0;
    if (le[b]) mine += (unsigned long long)le[b] * ((c - p + 15) / 16);
  }
  add_all(&lean_pages, mine);
  __syncthreads();
  // pages of a lean piece: as many pieces as the warps that run them, but no less than kLeanPages
  const int64_t page_work = (int64_t)lean_pages * d.Hkv;
  const int chunk = (int)min((int64_t)1 << 24,  // no table is wider
                             max((int64_t)kLeanPages, (page_work + d.shares * kLeanWarps - 1) / (d.shares * kLeanWarps)));
  for (int b = tid; b < d.B; b += kPlanThreads) {
    const int g = group_of(b), pages = (ctx_of(b) - (g >= 0 ? pre[g] : 0) + 15) / 16;
    const int chunks = le[b] ? (pages + chunk - 1) / chunk : 0;
    v.seqs[2 * b + 1] = chunks;
    le[b] *= chunks;
  }
  __syncthreads();
  block_scan(gu, d.G, sh);
  block_scan(su, d.B, sh);
  block_scan(le, d.B, sh);
  int n_lean = le[d.B];
  const int nG = gu[d.G];
  int n = nG + su[d.B];
  if (bad || n > d.max_units || n_lean > d.max_pieces) {
    if (tid == 0) set_status(status, kErrBounds);
    n = n_lean = 0;
  }
  for (int b = tid; b < d.B; b += kPlanThreads) v.seqs[2 * b] = le[b];
  for (int i = tid; i < n_lean; i += kPlanThreads) {
    const int b = last_le(le, d.B, i), g = group_of(b), p = g >= 0 ? pre[g] : 0, rows = (cu[b + 1] - cu[b]) * d.Gq;
    const int tiles = (rows + 15) / 16, chunks = (le[b + 1] - le[b]) / tiles;
    const int tile = (i - le[b]) / chunks, c = (i - le[b]) % chunks, pages = (ctx_of(b) - p + 15) / 16;
    Piece x;
    x.row0 = cu[b] * d.Gq + tile * 16;
    x.rows = min(16, rows - tile * 16);
    x.seq = b;
    x.page0 = p / 16 + c * chunk;
    x.pages = min(chunk, pages - c * chunk);
    x.ctx = ctx_of(b);
    x.lim = x.ctx - cu[b + 1] + 1;
    x.direct = p == 0 && chunks == 1;
    reinterpret_cast<Piece*>(v.lean)[i] = x;
  }
  mine = 0;
  for (int i = tid; i < n; i += kPlanThreads) {
    Unit u;
    if (i < nG) {
      const int g = last_le(gu, d.G, i), s0 = offs[g], tile = i - gu[g];
      u.row0 = cu[s0] * d.Gq + tile * d.wide_rows;
      u.rows = min(d.wide_rows, (cu[offs[g + 1]] - cu[s0]) * d.Gq - tile * d.wide_rows);
      u.seq = lead[g];
      u.key0 = 0;
      u.key_end = pre[g];
      u.lim = kNoLimit;
      u.solo = 0;
    } else {
      const int b = last_le(su, d.B, i - nG), tile = i - nG - su[b], g = group_of(b), nq = cu[b + 1] - cu[b];
      u.row0 = cu[b] * d.Gq + tile * kTileRows;
      u.rows = min(kTileRows, nq * d.Gq - tile * kTileRows);
      u.seq = b;
      u.key0 = g >= 0 ? pre[g] : 0;
      u.lim = ctx_of(b) - cu[b + 1] + 1;
      u.key_end = min(ctx_of(b), u.lim + (u.row0 + u.rows - 1) / d.Gq);
      u.solo = u.key0 == 0;
    }
    u.tiles = max(0, (u.key_end - u.key0 + kTileKeys - 1) / kTileKeys);
    reinterpret_cast<Unit*>(v.units)[i] = u;
    v.cost[i] = u.tiles * (u.rows > kTileRows ? kCostWide : kCostNarrow) + kCostUnit;
    v.rowcum[i] = u.rows;
    mine += v.cost[i];
  }
  add_all(&total_cost, mine);
  __syncthreads();
  if (total_cost > INT_MAX) {  // the cuts below are searched for in 32-bit sums: a plan of nothing
    if (tid == 0) set_status(status, kErrBounds);
    n = n_lean = 0;
  }
  block_scan(v.cost, n, sh);
  block_scan(v.rowcum, n, sh);  // its total falls into the slack behind the array
  for (int i = tid; i < n * d.Hkv; i += kPlanThreads) {
    v.inside[2 * i] = INT_MAX;
    v.inside[2 * i + 1] = 0;
  }
  __syncthreads();
  const int W0 = v.cost[n];
  const int64_t W = (int64_t)W0 * d.Hkv;
  const int shares = (int)min((int64_t)d.shares, max((int64_t)1, W / kCostShare));
  for (int c = tid; c <= d.shares; c += kPlanThreads) {
    int u = n * d.Hkv, t = 0;
    if (c < shares && W > 0) {
      const int64_t target = W * c / shares;
      const int hk = (int)(target / W0), rem = (int)(target % W0);
      const int u0 = last_le(v.cost, n, rem);
      const Unit& e = reinterpret_cast<const Unit*>(v.units)[u0];
      const int tc = e.rows > kTileRows ? kCostWide : kCostNarrow;
      t = max(0, rem - v.cost[u0] - kCostUnit + tc / 2) / tc;
      u = hk * n + u0;
      if (t >= e.tiles) {
        t = 0;
        ++u;
      }
      if (t > 0) {
        atomicMin(&v.inside[2 * u], c);
        atomicAdd(&v.inside[2 * u + 1], 1);
      }
    }
    v.cuts[2 * c] = u;
    v.cuts[2 * c + 1] = t;
  }
  for (int t = tid; t < d.T; t += kPlanThreads) {
    int4 m = make_int4(-1, 0, -1, 0);
    const int b = last_le(cu, d.B, t);
    if (n + n_lean > 0 && b >= 0 && t < cu[b + 1] && ctx_of(b) > 0) {
      const int g = group_of(b);
      if (g >= 0 && pre[g] > 0) m.x = gu[g], m.y = cu[offs[g]];
      if (su[b + 1] > su[b]) m.z = nG + su[b], m.w = cu[b];
      else if (le[b + 1] > le[b]) m.z = -2 - b, m.w = cu[b];
    }
    reinterpret_cast<int4*>(v.tok)[t] = m;
  }
  if (tid == 0) {
    v.hdr[0] = n;
    v.hdr[1] = W0;
    v.hdr[2] = v.rowcum[n];
    v.hdr[3] = n_lean;
  }
}

// ------------------------------------------------------------------------------------------------ attention
template <int D>
struct Cfg {
  static constexpr int kPipes = D > 128 ? 1 : 2;
  static constexpr int kKeys = kTileKeys;
  static constexpr int kBlocks = kKeys / 16;
  static constexpr int kChunks = D / 64;
  static constexpr int kSlot = kKeys * D * 2;           // K or V of a tile
  static constexpr int kSlots = D > 128 ? 5 : 10;
  static constexpr int kQBytes = kTileRows * D * 2;
  static constexpr int kSoftWarps = kPipes * 4;
  static constexpr int kThreads = (kSoftWarps + kPipes + 2) * 32;
  static constexpr int kBars = 2 * kSlots + 9 * kPipes + 1;
  // room to begin at a multiple of 1024 bytes, query tiles, ring, (m, l) of a tile's rows, barriers, TMEM address
  static constexpr int kSmem = 1024 + kPipes * kQBytes + kSlots * kSlot + kTileRows * 8 + kBars * 8 + 16;
  static_assert(kSmem <= 227 * 1024, "more shared memory than a CTA can have");
  // TMEM: two S (and P over them) of each pipeline, O behind them
  static __device__ __forceinline__ uint32_t s_col(int p, int i) { return p * 128 + i * kKeys; }
  static __device__ __forceinline__ uint32_t o_col(int p) { return 256 + p * D; }
};

__device__ __forceinline__ uint64_t desc_k128(uint32_t addr, uint32_t group_stride) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(group_stride >> 4) << 32;  // between 8-row groups
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}
__device__ __forceinline__ uint64_t desc_k32(uint32_t addr) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(256 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)6 << 61;  // 32-byte swizzle
  return d;
}
// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// mbar_wait with its limit on the SM's clock, which a waiting warp reads for nothing beside %globaltimer.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int* status) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255) == 0 && clock64() - t0 > 4000000000ll) break;  // about 2 s
  }
  set_status(status, kErrMbarTimeout);
  return false;
}
// 32 consecutive TMEM columns of this warp's lanes, a row a lane; the values are there after tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 r;
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return r;
}
// A whole 32-byte sector: lanes write rows of their own, and half sectors would be written twice.
__device__ __forceinline__ void store32(float* p, const float* f) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]),
               "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
               : "memory");
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// This share's pieces: a unit (of a KV head) and a range of its key tiles.  Every role walks the same list.
struct Walk {
  const Unit* units;
  int n, u, t, u_end, t_end;
  Unit e;
  int hk, u0, t0, t1;
  bool wide;  // two tiles against the same keys
  __device__ Walk(const PlanView& v, int share) {
    units = reinterpret_cast<const Unit*>(v.units);
    n = v.hdr[0];
    const int2 a = reinterpret_cast<const int2*>(v.cuts)[share], b = reinterpret_cast<const int2*>(v.cuts)[share + 1];
    u = a.x, t = a.y, u_end = b.x, t_end = b.y;
  }
  // The unit once more, for what is needed after a long stretch that has better use for its registers.
  __device__ Unit again() const {
    Unit x;
    const int4* q = reinterpret_cast<const int4*>(units + u0);
    asm volatile("ld.global.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(x.row0), "=r"(x.rows), "=r"(x.seq), "=r"(x.key0) : "l"(q));
    asm volatile("ld.global.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(x.key_end), "=r"(x.lim), "=r"(x.solo), "=r"(x.tiles) : "l"(q + 1));
    return x;
  }
  __device__ bool next() {
    while (u < u_end || (u == u_end && t < t_end)) {
      hk = u / n;
      u0 = u - hk * n;
      e = units[u0];
      t0 = t;
      t1 = u == u_end ? t_end : e.tiles;
      ++u;
      t = 0;
      if (t1 > t0) {
        wide = e.rows > kTileRows;
        return true;
      }
    }
    return false;
  }
};

struct AttnArgs {
  const __nv_bfloat16* q;
  const int* tables;
  __nv_bfloat16* out;
  float* part_o;   // [partial rows, D]
  float2* part_ml; // [partial rows] (maximum, sum)
  int* plan;
  PlanDims dims;
  int tma_q;       // a 128-row tile is a number of whole tokens
  int Hq, pages, over;  // over: first partial row of pieces that begin inside a unit (256 for each share)
  float scale_log2;
  int* status;
};

template <int D>
__global__ void __launch_bounds__(Cfg<D>::kThreads, 1)
    attn_shared_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ AttnArgs a) {
  using C = Cfg<D>;
  constexpr int NP = C::kPipes, KT = C::kKeys, NS = C::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = sm;                                   // [NP][kQBytes]
  uint8_t* sKV = sQ + NP * C::kQBytes;                // [NS][kSlot]
  float2* stat = reinterpret_cast<float2*>(sKV + NS * C::kSlot);  // [128] second pipeline's (m, l)
  uint64_t* bars = reinterpret_cast<uint64_t*>(stat + kTileRows);
  uint64_t* full = bars;             // [NS]
  uint64_t* empty = full + NS;       // [NS]
  uint64_t* q_full = empty + NS;     // [NP]
  uint64_t* q_empty = q_full + NP;   // [NP]
  uint64_t* s_ready = q_empty + NP;  // [NP][2] scores are in TMEM
  uint64_t* p_ready = s_ready + 2 * NP;  // [NP][2] weights are in TMEM, O may be accumulated
  uint64_t* pv_done = p_ready + 2 * NP;  // [NP] a tile's second product is complete
  uint64_t* o_done = pv_done + NP;   // [NP] a piece's last one is
  uint64_t* o_free = o_done + NP;    // [NP] O has been read
  uint64_t* stat_ready = o_free + NP;
  static_assert(C::kBars == 2 * NS + 9 * NP + 1, "the barriers above");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kBars);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NP);
    }
    for (int i = 0; i < NP; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], NP);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&s_ready[2 * i + k], 1);
        mbar_init(&p_ready[2 * i + k], 4);
      }
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_free[i], 4);
    }
    mbar_init(stat_ready, 4);
    fence_mbar_init();
  }
  if (warp == C::kSoftWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (tid == (C::kSoftWarps + NP) * 32) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The lean kernel before this one lets it begin once it has itself waited for what came before: the plan, q and the
  // caches are there.  What is left to wait for is the lean kernel's own end (below), for the merge kernel's sake.
  if (D > 128) pdl_wait();  // no lean kernel
  pdl_trigger();
  const PlanView pv = plan_view(a.plan, a.dims);
  Walk w(pv, blockIdx.x);

  if (warp >= C::kSoftWarps && warp < C::kSoftWarps + NP) {
    // ---------------------------------------------------------------- MMA
    // A warp for each pipeline.  The whole warp walks and waits, one elected lane issues, and what an instruction takes
    // is made uniform first: a product that one lane of a divergent warp issues costs over 200 clocks, three times its
    // 64 on the tensor cores.
    constexpr uint32_t idesc_s = make_idesc_bf16(128, KT), idesc_o = make_idesc_bf16(128, D);
    const bool el = elect_one_sync();
    const int p = (int)uniform(warp - C::kSoftWarps);
    const uint32_t tm = uniform(tmem);
    struct Pending {  // scores whose second product has not been issued
      uint32_t slot, par;
      int blocks;
      bool any, first, last;
    } pend0 = {}, pend1 = {};
    uint32_t visits = 0, begun = 0, starts = 0;  // first products, second products, pieces
    uint32_t q_par = 0, tile = 0, n = 0, qn = 0;
    bool ok = true;
    auto finish = [&](Pending& x, const int i) {  // O += P.V of scores i
      if (!x.any || !ok) return;
      x.any = false;
      ok = bar_wait(&p_ready[2 * p + i], (begun >> 1) & 1, a.status) && bar_wait(&full[x.slot], x.par, a.status);
      ++begun;
      starts += x.first;
      if (x.first && starts > 1) ok = ok && bar_wait(&o_free[p], starts & 1, a.status);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      tc_fence_after();
      const uint32_t slot = uniform(x.slot);
      const uint64_t vd = desc_k32(smem_u32(sKV) + slot * C::kSlot);
      const uint32_t o = tm + C::o_col(p), w0 = tm + C::s_col(p, i);
      const uint32_t acc = uniform(!x.first);
      const int blocks = (int)uniform(x.blocks);
      if (el) {
        if (blocks == C::kBlocks) {
#pragma unroll
          for (int kb = 0; kb < C::kBlocks; ++kb)
            mma_ts(o, w0 + (kb >> 1) * 32 + (kb & 1) * 8, vd + kb * (D * 32 / 16), idesc_o, kb ? 1 : acc);
#pragma unroll
          for (int kb = 0; kb < C::kBlocks; ++kb)
            mma_ts(o, w0 + (kb >> 1) * 32 + (kb & 1) * 8 + 16, vd + kb * (D * 32 / 16), idesc_o, 1);
        } else {
#pragma unroll 1
          for (int kb = 0; kb < blocks; ++kb) {
            mma_ts(o, w0 + (kb >> 1) * 32 + (kb & 1) * 8, vd + kb * (D * 32 / 16), idesc_o, kb ? 1 : acc);
            mma_ts(o, w0 + (kb >> 1) * 32 + (kb & 1) * 8 + 16, vd + kb * (D * 32 / 16), idesc_o, 1);
          }
        }
        tc_commit(&empty[slot]);
        tc_commit(&pv_done[p]);
        if (x.last) tc_commit(&o_done[p]);
      }
      __syncwarp();
    };
    // S = Q.K^T of a tile into scores i, after the second product of what was there
    auto begin = [&](Pending& x, const int i, uint32_t load, uint32_t buf, int blocks, bool first, bool last) {
      finish(x, i);
      const uint32_t kslot = uniform(load % NS);
      ok = ok && bar_wait(&full[kslot], (load / NS) & 1, a.status);
      if (first) ok = ok && bar_wait(&q_full[buf], (q_par >> buf) & 1, a.status);
      ok = __all_sync(~0u, ok);
      if (!ok) return;
      tc_fence_after();
      const uint64_t qd = desc_k128(smem_u32(sQ) + buf * C::kQBytes, 1024);
      const uint64_t kd = desc_k128(smem_u32(sKV) + kslot * C::kSlot, C::kChunks * 1024);
      if (el) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma_bf16(tm + C::s_col(p, i), qd + ((kk >> 2) * 16384 + (kk & 3) * 32) / 16,
                      kd + ((kk >> 2) * 1024 + (kk & 3) * 32) / 16, idesc_s, kk > 0);
        tc_commit(&s_ready[2 * p + i]);
        tc_commit(&empty[kslot]);
      }
      __syncwarp();
      x.slot = (load + 1) % NS;
      x.par = ((load + 1) / NS) & 1;
      x.blocks = blocks;
      x.any = true;
      x.first = first;
      x.last = last;
      ++visits;
    };
    while (ok && w.next()) {
      const int nt = w.t1 - w.t0, step = w.wide ? 1 : NP, bufs = w.wide ? NP : 1;
      const int j0 = w.wide ? 0 : (int)((p + NP - n % NP) % NP);  // this pipeline's first tile
      const int keys = w.e.key_end - w.e.key0 - w.t0 * KT;
      const uint32_t buf = uniform((qn + (w.wide ? p : 0)) % NP);
      for (int j = 0; j < nt && ok; ++j, ++tile) {
        const uint32_t load = 2 * tile;
        if (j >= j0 && (j - j0) % step == 0) {
          const int blocks = (min(KT, keys - j * KT) + 15) / 16;
          const bool first = j == j0, last = j + step >= nt;
          if (visits & 1) begin(pend1, 1, load, buf, blocks, first, last);
          else begin(pend0, 0, load, buf, blocks, first, last);
        } else {  // the other pipeline's: seen to have arrived, and given up
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const uint32_t slot = (load + kv) % NS;
            ok = ok && bar_wait(&full[slot], ((load + kv) / NS) & 1, a.status);
            if (ok && el) mbar_arrive(&empty[slot]);
          }
          ok = __all_sync(~0u, ok);
        }
      }
      // the rows are free when both pipelines are done with them
      for (int i = 0; i < bufs; ++i) {
        const uint32_t b = (qn + i) % NP;
        ok = __all_sync(~0u, ok && bar_wait(&q_full[b], (q_par >> b) & 1, a.status));
        if (ok && el) tc_commit(&q_empty[b]);
        q_par ^= 1u << b;
      }
      // a piece's last second products wait for no later piece: their results may free what that one waits for
      if (visits & 1) {
        finish(pend1, 1);
        finish(pend0, 0);
      } else {
        finish(pend0, 0);
        finish(pend1, 1);
      }
      qn += bufs;
      n = w.wide ? 0 : n + nt;
    }
  } else if (warp == C::kSoftWarps + NP) {
    // ---------------------------------------------------------------- K and V loads
    const bool el = elect_one_sync();
    uint32_t load = 0;
    bool ok = true;
    while (ok && w.next()) {
      const int* bt = a.tables + (size_t)w.e.seq * a.dims.max_blocks + w.e.key0 / 16;
      const int last = (w.e.key_end - w.e.key0 + 15) / 16;  // pages of the unit
      auto page_of = [&](int t) {
        const int i = t * C::kBlocks + lane;
        return lane < C::kBlocks && i < last ? bt[i] : 0;
      };
      int page = page_of(w.t0);
      for (int t = w.t0; t < w.t1 && ok; ++t) {
        const int blocks = min(C::kBlocks, last - t * C::kBlocks);
        int at = page * a.dims.Hkv + w.hk;
        if (lane < blocks && (page < 0 || page >= a.pages)) {  // no such page: past the end, where copies read zeros
          set_status(a.status, kErrBounds);
          at = a.pages * a.dims.Hkv;
        }
        if (t + 1 < w.t1) page = page_of(t + 1);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++load) {
          const uint32_t slot = load % NS;
          if (lane == 0) {
            ok = bar_wait(&empty[slot], ((load / NS) & 1) ^ 1, a.status);
            if (ok) mbar_arrive_expect_tx(&full[slot], blocks * 16 * D * 2);
          }
          ok = __shfl_sync(~0u, ok, 0);
          if (!ok) break;
          const uint32_t us = uniform(slot);
          uint8_t* dst = sKV + us * C::kSlot;
#pragma unroll
          for (int i = 0; i < C::kBlocks; ++i) {
            const int page_at = __shfl_sync(~0u, at, i);
            if (i < blocks && el) {
              if (kv == 0) tma_load_4d(dst + i * 16 * D * 2, &tmK, &full[us], 0, 0, 0, page_at * 2);
              else tma_load_3d(dst + i * 16 * D * 2, &tmV, &full[us], 0, 0, page_at);
            }
          }
          __syncwarp();
        }
      }
    }
    // no copy may be in flight when the CTA leaves
    if (lane == 0)
      for (uint32_t i = load > NS ? load - NS : 0; i < load; ++i) bar_wait(&full[i % NS], (i / NS) & 1, a.status);
  } else if (warp == C::kSoftWarps + NP + 1) {
    // ---------------------------------------------------------------- Q rows
    const bool el = elect_one_sync();
    uint32_t uses = 0, qn = 0;  // uses: a bit for each buffer
    bool ok = true;
    constexpr int kLanes = D / 8;  // 16-byte pieces of a row
    while (ok && w.next()) {
      for (int i = 0; i < (w.wide ? NP : 1); ++i, ++qn) {
        const int buf = qn % NP;
        if (lane == 0) ok = bar_wait(&q_empty[buf], ((uses >> buf) & 1) ^ 1, a.status);
        ok = __shfl_sync(~0u, ok, 0);
        if (!ok) break;
        uses ^= 1u << buf;
        const int rows = min(kTileRows, w.e.rows - i * kTileRows);
        const int row0 = w.e.row0 + i * kTileRows;
        if (a.tma_q) {  // whole tokens: rows past the unit's are other tokens' and are ignored
          const uint32_t ub = uniform(buf), token = uniform(row0 / a.dims.Gq), head = uniform(w.hk * a.dims.Gq);
          if (el) {
            mbar_arrive_expect_tx(&q_full[ub], C::kQBytes);
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_3d(sQ + ub * C::kQBytes + c * 16384, &tmQ, &q_full[ub], c * 64, head, token);
          }
          __syncwarp();
          continue;
        }
#pragma unroll 4
        for (int x = lane; x < rows * kLanes; x += 32) {
          const int r = x / kLanes, c = x % kLanes, tok = (row0 + r) / a.dims.Gq, g = (row0 + r) % a.dims.Gq;
          uint32_t byte = r * 128 + (c & 7) * 16;
          byte ^= ((byte >> 7) & 7) << 4;
          cp_async16(sQ + buf * C::kQBytes + (c >> 3) * 16384 + byte,
                     a.q + ((size_t)tok * a.Hq + w.hk * a.dims.Gq + g) * D + c * 8);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[buf]);
      }
    }
    if (lane == 0)  // as above: the last copy into each buffer
      for (uint32_t i = qn > NP ? qn - NP : 0; i < qn; ++i)
        bar_wait(&q_full[i % NP], (i / NP) & 1, a.status);
  } else {
    // ---------------------------------------------------------------- softmax, a row a thread
    const int p = warp >> 2, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lanes + C::o_col(p);
    uint32_t n = 0, tile = 0, visits = 0, pieces0 = 0, pieces1 = 0, joins = 0;
    bool ok = true;
    while (ok && w.next()) {
      const int nt = w.t1 - w.t0;
      const bool wide = w.wide;
      const int rows = w.e.rows - (wide ? p * kTileRows : 0);  // rows of this tile (may exceed 128)
      const bool live = (row & ~31) < rows;                     // some row of this warp is one
      const int key0 = w.e.key0 + w.t0 * KT;                    // of the piece
      const int keys = w.e.key_end - key0;                      // that some row sees, from there
      // this row sees the first `seen` of them
      const int seen = min(keys, w.e.lim + (w.e.row0 + (wide ? p * kTileRows : 0) + row) / a.dims.Gq - key0);
      float m = -INFINITY, l = 0.f;
      const int j0 = wide ? 0 : (int)((p + NP - n % NP) % NP);  // this pipeline's first tile
      const bool mine = j0 < nt;
      for (int j = j0; j < nt; j += wide ? 1 : NP) {
        const int at = 2 * p + (visits & 1);
        const uint32_t tS = tmem + lanes + C::s_col(p, visits & 1);
        if (lane == 0) ok = bar_wait(&s_ready[at], (visits >> 1) & 1, a.status);
        ok = __shfl_sync(~0u, ok, 0);
        ++visits;
        if (!ok) break;
        tc_fence_after();
        if (live) {
          uint32_t s[KT];
#pragma unroll
          for (int c = 0; c < KT; c += 32) tmem_ld32(tS + c, s + c);
          tmem_wait_ld();
          if (__any_sync(~0u, seen - j * KT < KT)) {
#pragma unroll
            for (int c = 0; c < KT; ++c)
              if (c >= seen - j * KT) s[c] = 0xff800000u;  // -inf
          }
          float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < KT; c += 2)
            t[(c >> 1) & 3] = fmaxf(t[(c >> 1) & 3], fmaxf(__uint_as_float(s[c]), __uint_as_float(s[c + 1])));
          const float mx = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * a.scale_log2;
          // the reference point moves only when the maximum has grown by more than 2^8
          if (j == j0) {
            m = mx;
          } else if (__any_sync(~0u, row < rows && mx > m + 8.f)) {
            // (O is complete up to the tile before: its second product has been)
            if (lane == 0) ok = bar_wait(&pv_done[p], (visits - 2) & 1, a.status);
            ok = __shfl_sync(~0u, ok, 0);
            if (!ok) break;
            tc_fence_after();
            const bool up = row < rows && mx > m + 8.f;
            const float f = up ? ex2(m - mx) : 1.f;  // rows that stay are multiplied by one: bit for bit as they were
            if (up) m = mx;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(tO + c, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= f;
              tmem_st16(tO + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
          const float2 sc = make_float2(a.scale_log2, a.scale_log2);
          const float2 ref = m == -INFINITY ? make_float2(0.f, 0.f) : make_float2(-m, -m);
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int c = 0; c < KT; c += 32) {  // 32 keys: their P over the first 16 of their columns
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float2 x = fma2(make_float2(__uint_as_float(s[c + e]), __uint_as_float(s[c + e + 1])), sc, ref);
              x = make_float2(ex2(x.x), ex2(x.y));
              sum = add2(sum, x);
              pk[e >> 1] = pack_bf16(x.x, x.y);
              s[c + e] = __float_as_uint(x.x);
              s[c + e + 1] = __float_as_uint(x.y);
            }
            tmem_st16(tS + c, pk);
            // what the rounding left, as a second product's weights, over the other 16
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              pk[e >> 1] = pack_bf16(__uint_as_float(s[c + e]) - __uint_as_float(pk[e >> 1] << 16),
                                     __uint_as_float(s[c + e + 1]) - __uint_as_float(pk[e >> 1] & 0xffff0000u));
            tmem_st16(tS + c + 16, pk);
          }
          l += sum.x + sum.y;
          tmem_wait_st();
        }
        // V of token slots past the context in the last page: zero, whatever lies there
        const int end = keys - j * KT;
        if (end < KT && (end & 15)) {
          const uint32_t vload = 2 * (tile + j) + 1, slot = vload % NS;
          if (lane == 0) ok = bar_wait(&full[slot], (vload / NS) & 1, a.status);
          ok = __shfl_sync(~0u, ok, 0);
          if (!ok) break;
          uint8_t* vb = sKV + slot * C::kSlot + (end >> 4) * D * 32;
          for (int d = row; d < D; d += kTileRows)
            for (int x = end & 15; x < 16; ++x) {
              uint32_t byte = d * 32 + x * 2;
              byte ^= ((byte >> 7) & 1) << 4;
              *reinterpret_cast<uint16_t*>(vb + byte) = 0;
            }
          fence_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[at]);
      }
      if (!ok) break;
      // ---- the piece's result
      const bool both = !wide && NP == 2 && nt >= 2;  // the second pipeline's half joins the first's
      pieces0 += both || wide || NP == 1 || n % 2 == 0;
      pieces1 += both || wide || n % 2 == 1;
      if (both && p == 1) {
        // the last joined halves have been read once their O is free
        if (lane == 0 && pieces1 > 1) ok = bar_wait(&o_free[NP - 1], pieces1 & 1, a.status);
        ok = __shfl_sync(~0u, ok, 0);
        if (!ok) break;
        stat[row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(stat_ready);
      } else if (mine) {
        if (lane == 0) {
          ok = bar_wait(&o_done[p], ((p ? pieces1 : pieces0) - 1) & 1, a.status);
          if (both) {
            ok = ok && bar_wait(&o_done[NP - 1], (pieces1 - 1) & 1, a.status);
            ok = ok && bar_wait(stat_ready, joins & 1, a.status);
          }
        }
        ok = __shfl_sync(~0u, ok, 0);
        if (!ok) break;
        tc_fence_after();
        if (live) {
          float f0 = 1.f, f1 = 0.f;  // weights of this pipeline's O and of the other's
          if (both) {
            const float2 x = stat[row];
            const float to = fmaxf(m, x.x);
            f0 = m == -INFINITY ? 0.f : ex2(m - to);
            f1 = x.x == -INFINITY ? 0.f : ex2(x.x - to);
            l = l * f0 + x.y * f1;
            m = to;
          }
          const int u0 = w.u0, off = wide ? p * kTileRows : 0;
          const Unit e = w.again();
          const bool valid = row < rows, direct = e.solo && nt == e.tiles;
          if (direct) {
            const float inv = l > 0.f ? 1.f / l : 0.f;
            f0 *= inv;
            f1 *= inv;
          }
          const size_t at = (w.t0 == 0 ? (size_t)w.hk * pv.hdr[2] + pv.rowcum[u0]
                                       : (size_t)a.over + (size_t)blockIdx.x * kWideRows) + off + row;
          if (valid && !direct) a.part_ml[at] = make_float2(m, l);
          const int ar = e.row0 + off + row, tok = ar / a.dims.Gq;
          __nv_bfloat16* dst = a.out + ((size_t)tok * a.Hq + w.hk * a.dims.Gq + ar - tok * a.dims.Gq) * D;
          float* part = a.part_o + at * D;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float f[16];
            tmem_ld16(tO + c, f);
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] *= f0;
            if (both) {
              float o1[16];
              tmem_ld16(tmem + lanes + C::o_col(NP - 1) + c, o1);
#pragma unroll
              for (int e = 0; e < 16; ++e) f[e] += o1[e] * f1;
            }
            if (valid && direct) {
#pragma unroll
              for (int e = 0; e < 16; e += 8)
                *reinterpret_cast<uint4*>(dst + c + e) =
                    make_uint4(pack_bf16(f[e], f[e + 1]), pack_bf16(f[e + 2], f[e + 3]),
                               pack_bf16(f[e + 4], f[e + 5]), pack_bf16(f[e + 6], f[e + 7]));
            } else if (valid) {
              store32(part + c, f);
              store32(part + c + 8, f + 8);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&o_free[p]);
          if (both) mbar_arrive(&o_free[NP - 1]);
        }
      }
      if (both) ++joins;
      n = w.wide ? 0 : n + nt;
      tile += nt;
    }
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  if (warp == C::kSoftWarps) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------------ lean
// A sequence's own tokens for its few rows: HBM-bound, so what counts is bytes in flight and little around them.  A warp
// owns a piece (16 rows, some pages) and a ring of pages of its own, each a bulk copy of K and one of V.  The fragments
// of the 16 x 8 x 16 products are read as the pages lie: both dimensions that are summed over are permuted for it.  Lane
// c of a quad takes the head dims 8 (4 i + c) ... + 7 of Q and K in 16-byte loads (the same for both, so S is
// unchanged), and the tokens 4 c ... 4 c + 3 of V's rows in 8-byte loads, which are the tokens whose S it holds.  P
// enters the second product as two bf16 terms.  128 sequences with up to 1024 own tokens (4 KV heads, 134 MB): about 28 us,
// 0.73 of the measured copy rate; with one page in flight a warp 35 us.
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
// An untiled copy of whole 16-byte units into this CTA's shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(~0u, x, 1));
  return fmaxf(x, __shfl_xor_sync(~0u, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(~0u, x, 1);
  return x + __shfl_xor_sync(~0u, x, 2);
}

struct LeanArgs {
  const __nv_bfloat16 *q, *k, *v;
  const int* tables;
  __nv_bfloat16* out;
  float* part_o;
  float2* part_ml;
  int* plan;
  PlanDims dims;
  int Hq, pages, lean0;  // lean0: first partial row (16 for each piece)
  float scale_log2;
  int* status;
};

constexpr int kLeanStages = 3;
template <int D>
constexpr int lean_smem() { return 4 * kLeanStages * D * 64 + 4 * kLeanStages * 8; }

template <int D>
__global__ void __launch_bounds__(128, 2) attn_shared_lean_kernel(const __grid_constant__ LeanArgs a) {
  constexpr int NT = D / 8, KV = D / 32;  // column tiles of O, 16-byte loads of a K row's part
  constexpr int ST = kLeanStages, kPage = D * 32;       // bytes of a page of K or V of a head
  extern __shared__ __align__(128) uint8_t ring[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & 3, r = lane >> 2;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + 4 * ST * 2 * kPage) + warp * ST;
  uint8_t* mine = ring + warp * ST * 2 * kPage;
  const bool el = elect_one_sync();
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  const PlanView v = plan_view(a.plan, a.dims);
  const int Hkv = a.dims.Hkv, Gq = a.dims.Gq, items = v.hdr[3] * Hkv;
  uint32_t asked = 0, taken = 0;  // pages, over all pieces
  bool ok = true;
  for (int item = warp * gridDim.x + blockIdx.x; item < items && ok; item += gridDim.x * 4) {
    const Piece x = reinterpret_cast<const Piece*>(v.lean)[item / Hkv];
    const int hk = item % Hkv;
    const int* bt = a.tables + (size_t)x.seq * a.dims.max_blocks + x.page0;
    int ids = lane < x.pages ? bt[lane] : 0;  // of 32 pages
    auto ask = [&](int i) {  // copies page i of the piece
      if ((i & 31) == 0 && i) ids = i + lane < x.pages ? bt[i + lane] : 0;
      const int id = __shfl_sync(~0u, ids, i & 31);
      const uint32_t slot = asked % ST;
      ++asked;
      const size_t at = ((size_t)(id < 0 || id >= a.pages ? 0 : id) * Hkv + hk) * (16 * D);
      if (el) {
        mbar_arrive_expect_tx(&full[slot], 2 * kPage);
        bulk_load(mine + slot * 2 * kPage, a.k + at, kPage, &full[slot]);
        bulk_load(mine + slot * 2 * kPage + kPage, a.v + at, kPage, &full[slot]);
      }
      __syncwarp();
    };
    uint32_t bad = 0;  // pages of the piece, from the one that is taken next, that there is none of
    auto check = [&](int i) {
      if ((i & 31) == 0) {
        const int id = i + lane < x.pages ? bt[i + lane] : 0;
        bad = __ballot_sync(~0u, id < 0 || id >= a.pages);
        if (bad) set_status(a.status, kErrBounds);
      }
      return (bad >> (i & 31)) & 1;
    };
    for (int i = 0; i < min(ST, x.pages); ++i) ask(i);
    const bool has0 = r < x.rows, has1 = r + 8 < x.rows;
    const int t0 = (x.row0 + r) / Gq, t1 = (x.row0 + r + 8) / Gq;
    const size_t o0 = ((size_t)t0 * a.Hq + hk * Gq + x.row0 + r - t0 * Gq) * D;
    const size_t o1 = ((size_t)t1 * a.Hq + hk * Gq + x.row0 + r + 8 - t1 * Gq) * D;
    uint4 q0[KV], q1[KV];
#pragma unroll
    for (int i = 0; i < KV; ++i) {
      q0[i] = has0 ? load16(a.q + o0 + i * 32 + c * 8) : make_uint4(0, 0, 0, 0);
      q1[i] = has1 ? load16(a.q + o1 + i * 32 + c * 8) : make_uint4(0, 0, 0, 0);
    }
    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    // keys of this lane in a page: 4 c + {0, 1, 2, 3}; row r sees those below lim
    const int base = x.page0 * 16 + 4 * c;
    const int lim0 = min(x.ctx, x.lim + t0), lim1 = min(x.ctx, x.lim + t1);
    const int tk = 4 * (r >> 1) + (r & 1);  // the token of K that this lane reads for the first column tile; + 2: the second
    for (int i = 0; i < x.pages; ++i, ++taken) {
      const bool gone = check(i);
      const uint32_t slot = taken % ST;
      ok = __all_sync(~0u, bar_wait(&full[slot], (taken / ST) & 1, a.status));
      if (!ok) break;
      const uint8_t* kp = mine + slot * 2 * kPage + tk * D * 2 + c * 16;
      const uint8_t* vp = mine + slot * 2 * kPage + kPage + r * 32 + c * 8;
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int t = 0; t < KV; ++t) {
          const uint4 k = *reinterpret_cast<const uint4*>(kp + j * 4 * D + t * 64);
          mma_16816(s[j], q0[t].x, q1[t].x, q0[t].y, q1[t].y, k.x, k.y);
          mma_16816(s[j], q0[t].z, q1[t].z, q0[t].w, q1[t].w, k.z, k.w);
        }
      }
      const int key = base + i * 16;
      const int seen0 = gone ? 0 : lim0 - key, seen1 = gone ? 0 : lim1 - key;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[j][e] = 2 * j + e < seen0 ? s[j][e] * a.scale_log2 : -INFINITY;
          s[j][2 + e] = 2 * j + e < seen1 ? s[j][2 + e] * a.scale_log2 : -INFINITY;
        }
      const float x0 = quad_max(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])));
      const float x1 = quad_max(fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3])));
      // the reference points move only when a maximum has grown by more than 2^8
      const bool up0 = has0 && (m0 == -INFINITY ? x0 > m0 : x0 > m0 + 8.f);
      const bool up1 = has1 && (m1 == -INFINITY ? x1 > m1 : x1 > m1 + 8.f);
      if (__any_sync(~0u, up0 || up1)) {
        const float f0 = up0 ? ex2(m0 - x0) : 1.f, f1 = up1 ? ex2(m1 - x1) : 1.f;
        if (up0) m0 = x0;
        if (up1) m1 = x1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t][0] *= f0, acc[t][1] *= f0, acc[t][2] *= f1, acc[t][3] *= f1;
      }
      const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = ex2(s[j][e] - (e < 2 ? r0 : r1));
        l0 += y[0] + y[1];
        l1 += y[2] + y[3];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          hi[2 * j + e] = pack_bf16(y[2 * e], y[2 * e + 1]);
          lo[2 * j + e] = pack_bf16(y[2 * e] - __uint_as_float(hi[2 * j + e] << 16),
                                    y[2 * e + 1] - __uint_as_float(hi[2 * j + e] & 0xffff0000u));
        }
      }
      // token slots past the context may hold anything
      const int left = gone ? 0 : x.ctx - key;
      const uint32_t k0 = left >= 2 ? ~0u : left == 1 ? 0xffffu : 0u, k1 = left >= 4 ? ~0u : left == 3 ? 0xffffu : 0u;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint2 y = *reinterpret_cast<const uint2*>(vp + t * 256);
        y.x &= k0;
        y.y &= k1;
        mma_16816(acc[t], hi[0], hi[1], hi[2], hi[3], y.x, y.y);
        mma_16816(acc[t], lo[0], lo[1], lo[2], lo[3], y.x, y.y);
      }
      __syncwarp();  // the page has been read
      if (i + ST < x.pages) ask(i + ST);
    }
    if (!ok) break;
    l0 = quad_sum(l0);
    l1 = quad_sum(l1);
    if (x.direct) {
      const float i0 = l0 > 0.f ? 1.f / l0 : 0.f, i1 = l1 > 0.f ? 1.f / l1 : 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (has0) *reinterpret_cast<uint32_t*>(a.out + o0 + t * 8 + 2 * c) = pack_bf16(acc[t][0] * i0, acc[t][1] * i0);
        if (has1) *reinterpret_cast<uint32_t*>(a.out + o1 + t * 8 + 2 * c) = pack_bf16(acc[t][2] * i1, acc[t][3] * i1);
      }
    } else {
      const size_t at = (size_t)a.lean0 + (size_t)item * 16 + r;
      if (c == 0 && has0) a.part_ml[at] = make_float2(m0, l0);
      if (c == 0 && has1) a.part_ml[at + 8] = make_float2(m1, l1);
      float* p = a.part_o + at * D + 2 * c;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (has0) *reinterpret_cast<float2*>(p + t * 8) = make_float2(acc[t][0], acc[t][1]);
        if (has1) *reinterpret_cast<float2*>(p + 8 * D + t * 8) = make_float2(acc[t][2], acc[t][3]);
      }
    }
  }
  // no copy may be in flight when the CTA leaves
  for (; taken < asked; ++taken) bar_wait(&full[taken % ST], (taken / ST) & 1, a.status);
}

// Joins the partials of a row (a warp each) and writes the rows that no unit covers as zeros.
template <int D>
__global__ void __launch_bounds__(256)
    attn_shared_merge_kernel(const float* __restrict__ part_o, const float2* __restrict__ part_ml, int* plan,
                             PlanDims d, __nv_bfloat16* __restrict__ out, int Hq, int over, int lean0) {
  constexpr int kPer = D / 32;
  struct alignas(kPer * 4 < 16 ? kPer * 4 : 16) V {
    float x[kPer];
  };
  pdl_wait();
  pdl_trigger();
  const int row = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (row >= d.T * Hq) return;
  const PlanView v = plan_view(plan, d);
  const int t = row / Hq, h = row % Hq, hk = h / d.Gq, g = h % d.Gq;
  const int4 tk = reinterpret_cast<const int4*>(v.tok)[t];
  const int n = v.hdr[0], rows0 = v.hdr[2];
  // the row's pieces: the one that begins each unit, then those of the shares that begin inside it
  size_t first_at[2] = {0, 0};
  int share0[2] = {0, 0}, count[2] = {0, 0}, within[2] = {0, 0};
  bool lean = false;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int first = side ? tk.z : tk.x;
    if (side && first <= -2) {  // lean pieces of the row's 16-row tile
      const int2 sq = reinterpret_cast<const int2*>(v.seqs)[-2 - first];
      if (tk.x < 0 && sq.y == 1) return;  // one piece had every key: written already
      const int rr = (t - tk.w) * d.Gq + g;
      first_at[1] = (size_t)lean0 + ((size_t)(sq.x + rr / 16 * sq.y) * d.Hkv + hk) * 16 + rr % 16;
      count[1] = sq.y;
      lean = true;
    }
    if (first < 0) continue;
    const int per = side ? kTileRows : d.wide_rows;
    const int rr = (t - (side ? tk.w : tk.y)) * d.Gq + g, u0 = first + rr / per, r = rr % per, u = hk * n + u0;
    if (reinterpret_cast<const Unit*>(v.units)[u0].tiles == 0) continue;  // queries before the context's first token
    const int2 in = reinterpret_cast<const int2*>(v.inside)[u];
    if (side && tk.x < 0 && in.y == 0) return;  // one piece had every key: written already
    first_at[side] = (size_t)hk * rows0 + v.rowcum[u0] + r;
    share0[side] = in.x - 1;
    count[side] = 1 + in.y;
    within[side] = r;
  }
  const int total = count[0] + count[1];
  auto place = [&](int i) {  // partial row of piece i, -1 for a share that was left nothing
    const bool side = i >= count[0];
    if (side) i -= count[0];
    if (side && lean) return (int64_t)(first_at[1] + (size_t)i * d.Hkv * 16);
    if (i == 0) return (int64_t)(side ? first_at[1] : first_at[0]);
    const int c = (side ? share0[1] : share0[0]) + i;
    const int2 x = reinterpret_cast<const int2*>(v.cuts)[c], y = reinterpret_cast<const int2*>(v.cuts)[c + 1];
    return x.x == y.x && x.y == y.y ? (int64_t)-1 : (int64_t)over + (int64_t)c * kWideRows + (side ? within[1] : within[0]);
  };
  float M = -INFINITY, L = 0.f, acc[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.f;
  for (int base = 0; base < total; base += 32) {  // a piece a lane for the weights, all lanes for each piece's row
    const int64_t at = base + lane < total ? place(base + lane) : -1;
    const float2 ml = at >= 0 ? part_ml[at] : make_float2(-INFINITY, 0.f);
    const float to = fmaxf(M, warp_max(ml.x));
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - to), old = M == -INFINITY ? 0.f : ex2(M - to);
    M = to;
    L = L * old + warp_sum(ml.y * f);
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] *= old;
    const int cnt = min(32, total - base);
    constexpr int kDeep = 8;
    for (int i = 0; i < cnt; i += kDeep) {
      V o[kDeep];
      float fi[kDeep];
#pragma unroll
      for (int k = 0; k < kDeep; ++k) {
        fi[k] = __shfl_sync(~0u, f, (i + k) & 31);
        const int64_t ai = __shfl_sync(~0u, at, (i + k) & 31);
        if (i + k >= cnt) fi[k] = 0.f;
        if (fi[k] != 0.f) o[k] = *reinterpret_cast<const V*>(part_o + ai * D + lane * kPer);
      }
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (fi[k] != 0.f) {  // the same for all lanes
#pragma unroll
          for (int e = 0; e < kPer; ++e) acc[e] += o[k].x[e] * fi[k];
        }
    }
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(out + (size_t)row * D + lane * kPer);
#pragma unroll
  for (int e = 0; e < kPer; e += 2) dst[e / 2] = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
}

int sm_count(int device) {
  static int sms[64] = {0};
  if (!sms[device]) C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms[device], cudaDevAttrMultiProcessorCount, device));
  return sms[device];
}

PlanDims plan_dims(int64_t T, int64_t B, int64_t G, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_blocks,
                   int device) {
  PlanDims d;
  d.T = (int)T, d.B = (int)B, d.G = (int)G, d.Gq = (int)(Hq / Hkv), d.Hkv = (int)Hkv;
  d.wide_rows = D > 128 ? kTileRows : kWideRows;
  d.shares = sm_count(device);
  d.max_blocks = (int)max_blocks;
  d.max_units = (int)(T * d.Gq / d.wide_rows + G + T * d.Gq / kTileRows + B + 2);
  d.lean_rows = D > 128 ? 0 : kLeanRows;
  // one for each 16 rows of a sequence, and one more for each whole chunk of pages, of which there are about as many as warps
  d.max_pieces = D > 128 ? 0 : (int)(T * d.Gq / 16 + B + d.shares * kLeanWarps / Hkv + 2);
  return d;
}

// Partial rows: first pieces of units, then pieces that begin inside one, then lean pieces.
int64_t partial_rows(const PlanDims& d, int64_t Hq) {
  return 2 * (int64_t)d.T * Hq + (int64_t)d.shares * kWideRows + 16 * (int64_t)d.max_pieces * d.Hkv;
}

void check_dims(const char* who, int64_t T, int64_t Hq, int64_t Hkv, int64_t D) {
  TORCH_CHECK(D == 64 || D == 128 || D == 256, who, ": head_dim must be 64, 128 or 256");
  TORCH_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && T >= 0 && T * Hq <= (int64_t)1 << 26, who, ": heads or tokens out of range");
}

CUtensorMap map_of(const at::Tensor& t, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                   const cuuint32_t* box, CUtensorMapSwizzle sw) {
  CUtensorMap m;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const CUresult r = get_encode()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, t.data_ptr(), dims, strides,
                                            box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "attn_shared: cuTensorMapEncodeTiled failed (", (int)r, ")");
  return m;
}

}  // namespace

// Elements of the int32 plan buffer and of the fp32 workspace of a step.
std::tuple<int64_t, int64_t> attn_shared_sizes(int64_t T, int64_t B, int64_t G, int64_t Hq, int64_t Hkv, int64_t D,
                                               int64_t max_blocks, int64_t device) {
  check_dims("attn_shared_plan", T, Hq, Hkv, D);
  const PlanDims d = plan_dims(T, B, G, Hq, Hkv, D, max_blocks, (int)device);
  const int64_t rows = partial_rows(d, Hq);
  return {plan_ints(d), rows * (D + 2)};
}

void attn_shared_plan(const at::Tensor& block_tables, const at::Tensor& ctx_lens, const at::Tensor& group_offs,
                      const at::Tensor& shared_lens, const c10::optional<at::Tensor>& cu_q, int64_t T, int64_t Hq,
                      int64_t Hkv, int64_t D, at::Tensor& plan) {
  check_dims("attn_shared_plan", T, Hq, Hkv, D);
  TORCH_CHECK(block_tables.is_cuda() && block_tables.dim() == 2, "attn_shared_plan: block_tables must be [B, max_blocks]");
  const int64_t B = block_tables.size(0), G = shared_lens.numel();
  for (const auto& t : {ctx_lens, group_offs, shared_lens, plan})
    TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == block_tables.device(),
                "attn_shared_plan: lengths, offsets and plan must be contiguous int32 on the tables' device");
  TORCH_CHECK(ctx_lens.numel() == B && group_offs.numel() == G + 1,
              "attn_shared_plan: ctx_lens [B], group_offs [G + 1], shared_lens [G]");
  if (cu_q) {
    TORCH_CHECK(cu_q->scalar_type() == at::kInt && cu_q->is_contiguous() && cu_q->numel() == B + 1 &&
                    cu_q->device() == block_tables.device(),
                "attn_shared_plan: cu_q must be contiguous int32 [B + 1] on the tables' device");
  } else {
    TORCH_CHECK(T == B, "attn_shared_plan: without cu_q every sequence has one query token");
  }
  TORCH_CHECK(B <= 8192 && G <= 8192, "attn_shared_plan: at most 8192 sequences and groups");
  TORCH_CHECK(block_tables.size(1) < (1 << 24), "attn_shared_plan: block_tables too wide");
  c10::cuda::CUDAGuard guard(block_tables.device());
  const int dev = block_tables.device().index();
  const PlanDims d = plan_dims(T, B, G, Hq, Hkv, D, block_tables.size(1), dev);
  TORCH_CHECK(plan.numel() >= plan_ints(d), "attn_shared_plan: plan buffer too small");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(plan.data_ptr()) % 16 == 0, "attn_shared_plan: plan must be 16-byte aligned");
  const int smem = (int)(4 * (4 * G + 3 * B + 8));
  static bool attr[64] = {false};
  if (!attr[dev]) {  // whatever this call takes: the 48 KB that need no asking count the kernel's static bytes too
    C10_CUDA_CHECK(cudaFuncSetAttribute(attn_shared_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024));
    attr[dev] = true;
  }
  launch_k(attn_shared_plan_kernel, 1, kPlanThreads, smem, at::cuda::getCurrentCUDAStream(), ctx_lens.data_ptr<int>(),
           group_offs.data_ptr<int>(), shared_lens.data_ptr<int>(), cu_q ? cu_q->data_ptr<int>() : nullptr,
           plan.data_ptr<int>(), d, status_ptr(dev));
}

template <int D>
static void launch_attn(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, AttnArgs a, cudaStream_t st, int dev) {
  using C = Cfg<D>;
  const cuuint64_t heads = (cuuint64_t)k_cache.size(0) * k_cache.size(1);
  // K as (64 elements, 8 rows, D / 64 chunks, groups of 8 rows): a page's two groups arrive as swizzle atoms
  const cuuint64_t kd[4] = {64, 8, C::kChunks, heads * 2}, ks[3] = {D * 2, 128, D * 16};
  const cuuint32_t kb[4] = {64, 8, C::kChunks, 2};
  const cuuint64_t vd[3] = {16, D, heads}, vs[2] = {32, D * 32};
  const cuuint32_t vb[3] = {16, D, 1};
  const cuuint64_t qd[3] = {D, (cuuint64_t)a.Hq, (cuuint64_t)a.dims.T}, qs[2] = {D * 2, (cuuint64_t)a.Hq * D * 2};
  a.tma_q = kTileRows % a.dims.Gq == 0;
  const cuuint32_t qb[3] = {64, a.tma_q ? (cuuint32_t)a.dims.Gq : 1, a.tma_q ? (cuuint32_t)(kTileRows / a.dims.Gq) : 1};
  const CUtensorMap tq = map_of(q, 3, qd, qs, qb, CU_TENSOR_MAP_SWIZZLE_128B);
  const CUtensorMap tk = map_of(k_cache, 4, kd, ks, kb, CU_TENSOR_MAP_SWIZZLE_128B);
  const CUtensorMap tv = map_of(v_cache, 3, vd, vs, vb, CU_TENSOR_MAP_SWIZZLE_32B);
  static bool attr[64] = {false};
  if (!attr[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(attn_shared_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    attr[dev] = true;
  }
  const int lean0 = a.over + a.dims.shares * kWideRows;
  if constexpr (D <= 128) {
    LeanArgs x;
    x.q = a.q;
    x.k = reinterpret_cast<const __nv_bfloat16*>(k_cache.data_ptr());
    x.v = reinterpret_cast<const __nv_bfloat16*>(v_cache.data_ptr());
    x.tables = a.tables, x.out = a.out, x.part_o = a.part_o, x.part_ml = a.part_ml, x.plan = a.plan, x.dims = a.dims;
    x.Hq = a.Hq, x.pages = a.pages, x.lean0 = lean0, x.scale_log2 = a.scale_log2, x.status = a.status;
    static bool attr[64] = {false};
    if (!attr[dev]) {
      C10_CUDA_CHECK(cudaFuncSetAttribute(attn_shared_lean_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          lean_smem<D>()));
      attr[dev] = true;
    }
    launch_k(attn_shared_lean_kernel<D>, a.dims.shares * 2, 128, lean_smem<D>(), st, x);
  }
  launch_k(attn_shared_kernel<D>, a.dims.shares, C::kThreads, C::kSmem, st, tq, tk, tv, a);
  launch_k(attn_shared_merge_kernel<D>, (a.dims.T * a.Hq + 7) / 8, 256, 0, st, (const float*)a.part_o,
           (const float2*)a.part_ml, a.plan, a.dims, a.out, a.Hq, a.over, lean0);
}

void attn_shared(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                 const at::Tensor& block_tables, int64_t groups, at::Tensor& plan, at::Tensor& workspace,
                 at::Tensor& out, double scale) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && k_cache.scalar_type() == at::kBFloat16 &&
                  v_cache.scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16,
              "attn_shared: q, caches and out must be bf16 on a CUDA device");
  TORCH_CHECK(q.dim() == 3 && q.is_contiguous() && out.is_contiguous() && out.sizes() == q.sizes(),
              "attn_shared: q and out must be contiguous [T, Hq, D]");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  TORCH_CHECK(k_cache.is_contiguous() && v_cache.is_contiguous() && k_cache.dim() == 4 && v_cache.dim() == 4 &&
                  k_cache.size(2) == 16 && k_cache.size(3) == D && v_cache.size(2) == D && v_cache.size(3) == 16 &&
                  k_cache.size(0) == v_cache.size(0) && k_cache.size(1) == v_cache.size(1),
              "attn_shared: caches must be contiguous K [pages, Hkv, 16, D] and V [pages, Hkv, D, 16]");
  const int64_t Hkv = k_cache.size(1), pages = k_cache.size(0);
  check_dims("attn_shared", T, Hq, Hkv, D);
  TORCH_CHECK(pages * Hkv * 2 < ((int64_t)1 << 31) - 4, "attn_shared: cache too large");
  TORCH_CHECK(std::isfinite(scale) && scale > 0, "attn_shared: scale must be finite and positive");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.is_contiguous() &&
                  plan.scalar_type() == at::kInt && workspace.scalar_type() == at::kFloat,
              "attn_shared: block_tables must be contiguous int32 [B, max_blocks]");
  for (const auto& t : {k_cache, v_cache, block_tables, plan, workspace, out})
    TORCH_CHECK(t.device() == q.device(), "attn_shared: every tensor must be on q's device");
  for (const auto& t : {q, k_cache, v_cache, out})
    TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "attn_shared: tensors must be 16-byte aligned");
  if (T == 0) return;
  TORCH_CHECK(pages > 0, "attn_shared: empty cache");
  c10::cuda::CUDAGuard guard(q.device());
  const int dev = q.device().index();
  AttnArgs a;
  a.dims = plan_dims(T, block_tables.size(0), groups, Hq, Hkv, D, block_tables.size(1), dev);
  a.over = (int)(2 * T * Hq);
  const int64_t rows = partial_rows(a.dims, Hq);
  TORCH_CHECK(plan.numel() >= plan_ints(a.dims) && workspace.numel() >= rows * (D + 2) && plan.is_contiguous() &&
                  workspace.is_contiguous(),
              "attn_shared: plan or workspace too small or not contiguous");
  // records of 16 bytes, partial rows stored by 32
  TORCH_CHECK(reinterpret_cast<uintptr_t>(plan.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(workspace.data_ptr()) % 32 == 0,
              "attn_shared: plan must be 16-byte and workspace 32-byte aligned");
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.tables = block_tables.data_ptr<int>();
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.part_o = workspace.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * D);
  a.plan = plan.data_ptr<int>();
  a.Hq = (int)Hq;
  a.pages = (int)pages;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.status = status_ptr(dev);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  if (D == 64) launch_attn<64>(q, k_cache, v_cache, a, st, dev);
  else if (D == 128) launch_attn<128>(q, k_cache, v_cache, a, st, dev);
  else launch_attn<256>(q, k_cache, v_cache, a, st, dev);
}

}  // namespace mb
