// Batch plan: the block table, the slot map and the positions of a ragged batch's new tokens,
// from the segments, the arena, the descriptor table and the new tokens' counts.
//
// Sequence i has blocks j < n with v_j valid tokens; start_j = sum of v before j; context =
// sum of all v; its q new tokens are the last ones.  A block without tokens lists nowhere.  Of the
// others (rank r = how many come before), a window keeps those with start < sinks, which are
// the first P, and those with start + v > context - q - window + 1, which are the ones from
// rank S on; so block r lists at r when r < P and at P + r - max(S, P) when r >= S, and no second
// scan is needed: only the two border ranks.
//
// A cluster of CTAs takes one sequence: every thread loads kItems consecutive blocks (arena, then
// the descriptor: two dependent loads, all items of all threads in flight together), one scan of
// (tokens, non-empty blocks) runs through the CTA and then over the cluster's CTA totals in
// distributed shared memory.  A sequence longer than the cluster's kRound blocks is taken in
// rounds, after a first pass that only adds up its tokens (the window and the new tokens are
// counted from the end).
//
// The bound is latency: launch, the segment, the arena, the descriptor, the scan and the stores follow one another,
// and the bytes (20 read and at most 20 written for a block) take less than a microsecond.  Measured: 8 sequences of
// 100 to 900 tokens, 5.3 us; 64 of 8192 tokens, 5.4 us; 48 of 1000 to 131072 with a window, 9.9 us with clusters of up
// to 8 CTAs a sequence and 43.5 us with one.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "codec.cuh"
#include "common.cuh"
#include "hlkv.h"

namespace hlkv {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kItems = 4;
constexpr uint32_t kRound = kThreads * kItems;  // blocks per CTA and round
constexpr int kMaxCluster = 8;

struct Params {
  HlkvBatchPlan plan;
  const uint4* table;
  const uint32_t* arena;
  const uint2* segs;
  const uint32_t* qlens;  // nullptr: one each
  uint32_t* err;
  uint32_t table_size, arena_size, T, layout_id;
  uint32_t prefix_done;  // d_block_first and d_token_first are filled already
};

// Tokens, non-empty blocks and their cost to the attention, added as one.
struct Sum {
  uint32_t tokens, blocks, cost;
  __device__ __forceinline__ Sum operator+(const Sum& o) const {
    return {tokens + o.tokens, blocks + o.blocks, cost + o.cost};
  }
};

// What a block of v tokens costs the attention, which works on tiles of 16 tokens: in proportion to the
// time measured for caches of one format (2.0, 1.0 and 1.1 us a tile of 8 heads of 128 per SM); used for every shape.
__device__ __forceinline__ uint32_t block_cost(uint32_t info, uint32_t v) {
  const uint32_t f = info & 0xFu;
  return (v + 15) / 16 * (f == dev::kFp16 ? 14u : 7u);
}
__device__ __forceinline__ Sum block_sum(uint32_t info, uint32_t v) {
  return v > 0 ? Sum{v, 1u, block_cost(info, v)} : Sum{0u, 0u, 0u};
}

struct Shared {
  Sum warp[kWarps];
  Sum cta[2][kMaxCluster];  // every CTA's total, written by its owner into each CTA (two rounds' worth)
  uint64_t prefix[2][kWarps];
  uint32_t border[4];  // P and S, and the cost before each
};

// Checks block j of the segment as kernel (1) does, without the pools; its descriptor in *d.
// Returns its valid tokens, 0 for a block that fails.
__device__ __forceinline__ uint32_t load_block(const Params& p, uint2 seg, uint32_t j, uint4* d, uint32_t* bad) {
  const uint64_t pos = uint64_t{seg.x} + j;
  if (pos >= p.arena_size) {
    *bad |= dev::kErrArenaRange;
    return 0;
  }
  const uint32_t id = __ldg(p.arena + pos);
  if (id >= p.table_size) {
    *bad |= dev::kErrBlockIdRange;
    return 0;
  }
  *d = __ldg(p.table + id);
  const uint32_t f = d->y & 0xFu, mode = (d->y >> 4) & 3u, layout = (d->y >> 6) & 0xFu, v = (d->y >> 10) & 0x3FFu;
  uint32_t e = 0;
  if (d->w != id) e = dev::kErrDescMismatch;
  else if (f == dev::kInvalidFormat) e = dev::kErrNotExecutable;
  else if (f > 3) e = dev::kErrBadFormat;
  else if (layout != p.layout_id) e = dev::kErrLayout;
  else if (f != dev::kFp16 && (mode > 2 || (mode != 0 && !dev::block_params_ok(f, mode, d->z)))) e = dev::kErrScaleMode;
  else if (v > p.T) e = dev::kErrValidTokens;
  *bad |= e;
  return e ? 0u : v;
}

// The sums of (length, new tokens) over the sequences before i, and sequence i's own.
__device__ __forceinline__ void sums_before(const Params& p, uint32_t i, Shared& s, uint64_t* blocks, uint64_t* tokens) {
  uint64_t a = 0, b = 0;
  for (uint32_t k = threadIdx.x; k < i; k += kThreads) {
    a += p.segs[k].y;
    b += p.qlens ? __ldg(p.qlens + k) : 1u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, o);
    b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
  }
  if ((threadIdx.x & 31) == 0) {
    s.prefix[0][threadIdx.x >> 5] = a;
    s.prefix[1][threadIdx.x >> 5] = b;
  }
  __syncthreads();
  a = b = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    a += s.prefix[0][w];
    b += s.prefix[1][w];
  }
  *blocks = a;
  *tokens = b;
}

// Exclusive scan of every thread's sum over the cluster's threads in CTA order; *total of all.
// `phase` alternates from call to call: a CTA may still read the other phase's totals.
__device__ __forceinline__ Sum cluster_scan(cg::cluster_group& cluster, Shared& s, Sum v, uint32_t phase, Sum* total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sum x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sum y{__shfl_up_sync(0xFFFFFFFFu, x.tokens, o), __shfl_up_sync(0xFFFFFFFFu, x.blocks, o),
                __shfl_up_sync(0xFFFFFFFFu, x.cost, o)};
    if (lane >= static_cast<uint32_t>(o)) x = x + y;
  }
  __syncthreads();  // the warp totals of the call before have been read
  if (lane == 31) s.warp[warp] = x;
  __syncthreads();
  Sum before{0, 0, 0}, all{0, 0, 0};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < static_cast<int>(warp)) before = before + s.warp[w];
    all = all + s.warp[w];
  }
  const uint32_t n = cluster.num_blocks(), rank = cluster.block_rank();
  if (n > 1) {
    if (threadIdx.x < n) cluster.map_shared_rank(&s, threadIdx.x)->cta[phase & 1][rank] = all;
    cluster.sync();
    all = Sum{0, 0, 0};
    for (uint32_t c = 0; c < n; ++c) {
      if (c < rank) before = before + s.cta[phase & 1][c];
      all = all + s.cta[phase & 1][c];
    }
  }
  *total = all;
  return Sum{before.tokens + x.tokens - v.tokens, before.blocks + x.blocks - v.blocks, before.cost + x.cost - v.cost};
}

__global__ void __launch_bounds__(kThreads) batch_plan_kernel(const Params p) {
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t n_ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t i = blockIdx.x / n_ctas;
  const HlkvBatchPlan& plan = p.plan;
  if (n_ctas > 1) cluster.barrier_arrive();  // waited for before the first write into another CTA's shared memory
  const uint2 seg = p.segs[i];
  const uint32_t q = p.qlens ? __ldg(p.qlens + i) : 1u;
  uint64_t first, tfirst;
  if (p.prefix_done) {
    first = plan.d_block_first[i];
    tfirst = plan.d_token_first[i];
  } else {
    sums_before(p, i, s, &first, &tfirst);
  }
  const bool fits = first + seg.y <= plan.block_cap && tfirst + q <= plan.token_cap && q <= plan.max_query;
  const uint32_t n = fits ? seg.y : 0u;
  uint32_t bad = fits ? 0u : dev::kErrPlanRange;

  const uint32_t round = kRound * n_ctas;
  const uint32_t mine = rank * kRound + threadIdx.x * kItems;  // this thread's first block of a round
  const bool one_round = n <= round;
  uint32_t phase = 0;
  uint4 d[kItems];
  uint32_t v[kItems];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const uint32_t j = base + mine + k;
      d[k] = make_uint4(0u, 0u, 0u, 0u);
      v[k] = 0;
      if (j < n && j >= base) v[k] = load_block(p, seg, j, &d[k], &bad);
    }
  };
  auto own_sum = [&]() {
    Sum x{0, 0, 0};
#pragma unroll
    for (int k = 0; k < kItems; ++k) x = x + block_sum(d[k].y, v[k]);
    return x;
  };

  Sum before{0, 0, 0}, total{0, 0, 0};
  if (threadIdx.x < 4) s.border[threadIdx.x] = 0xFFFFFFFFu;  // written by all after the scan's barrier
  if (one_round) {
    load(0);
    if (n_ctas > 1) cluster.barrier_wait();
    before = cluster_scan(cluster, s, own_sum(), phase++, &total);
  } else {
    Sum x{0, 0, 0};
    for (uint64_t base = 0; base < n; base += round) {
      load(static_cast<uint32_t>(base));
      x = x + own_sum();
    }
    if (n_ctas > 1) cluster.barrier_wait();
    cluster_scan(cluster, s, x, phase++, &total);
  }
  const uint32_t context = total.tokens;

  // The window's borders.
  const uint32_t seen_from = context > q ? context - q : 0u;  // position of the first new token
  const uint32_t low = plan.window != 0 && seen_from + 1u > plan.window ? seen_from + 1u - plan.window : 0u;
  const bool trimmed = low > 0;
  uint32_t n_first = total.blocks, n_skip = 0;  // P and S; without a trim every block is one of the first
  uint32_t cost_first = total.cost, cost_skip = 0;
  Sum carry{0, 0, 0};
  const uint32_t token_base = static_cast<uint32_t>(tfirst);  // used for rows of a sequence that fits only
  const uint32_t missing = q > context ? q - context : 0u;    // new tokens that the sequence does not have
  for (uint64_t base64 = 0; base64 < n; base64 += round) {
    if (!one_round) {
      load(static_cast<uint32_t>(base64));
      Sum t;
      before = cluster_scan(cluster, s, own_sum(), phase++, &t) + carry;
      carry = carry + t;
    }
    if (trimmed) {
      // The least ranks of a non-empty block behind the sinks and of one in the window, to every
      // CTA of the cluster.  Both conditions hold from some rank on, so the minima are the borders.
      uint32_t behind = 0xFFFFFFFFu, within = 0xFFFFFFFFu, cost_behind = 0xFFFFFFFFu, cost_within = 0xFFFFFFFFu;
      Sum x = before;
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        if (v[k] == 0) continue;
        if (x.tokens >= plan.sinks) {
          behind = min(behind, x.blocks);
          cost_behind = min(cost_behind, x.cost);
        }
        if (x.tokens + v[k] > low) {
          within = min(within, x.blocks);
          cost_within = min(cost_within, x.cost);
        }
        x = x + block_sum(d[k].y, v[k]);
      }
      behind = __reduce_min_sync(0xFFFFFFFFu, behind);
      within = __reduce_min_sync(0xFFFFFFFFu, within);
      cost_behind = __reduce_min_sync(0xFFFFFFFFu, cost_behind);
      cost_within = __reduce_min_sync(0xFFFFFFFFu, cost_within);
      if ((threadIdx.x & 31) < n_ctas) {
        Shared* o = cluster.map_shared_rank(&s, threadIdx.x & 31);
        if (behind != 0xFFFFFFFFu) {
          atomicMin(&o->border[0], behind);
          atomicMin(&o->border[2], cost_behind);
        }
        if (within != 0xFFFFFFFFu) {
          atomicMin(&o->border[1], within);
          atomicMin(&o->border[3], cost_within);
        }
      }
      if (n_ctas > 1) cluster.sync();
      else __syncthreads();
      n_first = min(s.border[0], total.blocks);
      n_skip = s.border[1];
      cost_first = min(s.border[2], total.cost);
      cost_skip = s.border[3];
    }
    const uint32_t skip = max(n_skip, n_first), cost_gap = max(cost_skip, cost_first) - cost_first;
    Sum x = before;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      if (v[k] == 0) continue;
      const uint32_t r = x.blocks, start = x.tokens;
      if (r < n_first || r >= n_skip) {
        const uint32_t at = static_cast<uint32_t>(first) + (r < n_first ? r : n_first + r - skip);
        reinterpret_cast<uint4*>(plan.d_blocks)[at] = make_uint4(d[k].x, d[k].y, d[k].z, start);
        const uint32_t cost = x.cost + block_cost(d[k].y, v[k]);
        plan.d_block_cost[at] = r < n_first ? cost : cost - cost_gap;
      }
      const uint32_t end = start + v[k];
      for (uint32_t t = max(start, seen_from); t < end; ++t) {
        const uint32_t row = token_base + missing + (t - seen_from);
        reinterpret_cast<uint2*>(plan.d_targets)[row] = make_uint2(d[k].w, t - start);
        plan.d_positions[row] = static_cast<int32_t>(t);
      }
      x = x + block_sum(d[k].y, v[k]);
    }
  }

  if (bad) atomicOr(p.err, bad);
  // Padding: rows of new tokens that the sequence does not have (or of one that does not fit),
  // and behind the last sequence's, up to the end of the arrays.
  auto pad = [&](uint64_t from, uint64_t to) {
    to = min(to, uint64_t{plan.token_cap});
    for (uint64_t row = from + threadIdx.x; row < to; row += kThreads) {
      reinterpret_cast<uint2*>(plan.d_targets)[row] = make_uint2(0xFFFFFFFFu, 0xFFFFFFFFu);
      plan.d_positions[row] = 0;
    }
  };
  if (rank == 0) {
    if (!fits) pad(tfirst, tfirst + q);
    else if (missing) pad(tfirst, tfirst + missing);
    if (i + 1 == plan.nseq) pad(tfirst + q, plan.token_cap);
    if (threadIdx.x == 0) {
      if (fits && missing) atomicOr(p.err, dev::kErrPlanRange);
      plan.d_block_count[i] = trimmed ? (n_skip == 0xFFFFFFFFu ? n_first : n_first + total.blocks - max(n_skip, n_first))
                                      : total.blocks;
      plan.d_cost[i] = trimmed ? (n_skip == 0xFFFFFFFFu ? cost_first : cost_first + total.cost - max(cost_skip, cost_first))
                               : total.cost;
      plan.d_context[i] = context;
      if (!p.prefix_done) {
        plan.d_block_first[i] = static_cast<uint32_t>(min(first, uint64_t{plan.block_cap}));
        plan.d_token_first[i] = static_cast<uint32_t>(min(tfirst, uint64_t{plan.token_cap}));
      }
      if (i + 1 == plan.nseq) {
        plan.d_token_first[i + 1] = static_cast<uint32_t>(min(tfirst + q, uint64_t{plan.token_cap}));
      }
    }
  }
  // (Every write into another CTA's shared memory lies before a barrier of the cluster: no CTA leaves too early.)
}

// d_block_first and d_token_first of a large batch: one CTA, a chunked scan.  A sum beyond its
// array's end is written as the end, where no sequence with blocks or tokens fits either.
__global__ void __launch_bounds__(1024) batch_plan_prefix(const uint2* __restrict__ segs, const uint32_t* __restrict__ qlens,
                                                          HlkvBatchPlan plan) {
  __shared__ uint64_t s_sum[2][32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t carry_b = 0, carry_t = 0;
  for (uint64_t base = 0; base < plan.nseq; base += 1024) {
    const uint64_t i = base + threadIdx.x;
    const uint64_t vb = i < plan.nseq ? segs[i].y : 0u;
    const uint64_t vt = i < plan.nseq ? (qlens ? qlens[i] : 1u) : 0u;
    uint64_t b = vb, t = vt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t ob = __shfl_up_sync(0xFFFFFFFFu, b, o), ot = __shfl_up_sync(0xFFFFFFFFu, t, o);
      if (lane >= static_cast<uint32_t>(o)) {
        b += ob;
        t += ot;
      }
    }
    if (lane == 31) {
      s_sum[0][warp] = b;
      s_sum[1][warp] = t;
    }
    __syncthreads();
    uint64_t before_b = carry_b, before_t = carry_t;
    for (uint32_t w = 0; w < 32; ++w) {
      if (w < warp) {
        before_b += s_sum[0][w];
        before_t += s_sum[1][w];
      }
      carry_b += s_sum[0][w];
      carry_t += s_sum[1][w];
    }
    if (i < plan.nseq) {
      plan.d_block_first[i] = static_cast<uint32_t>(min(before_b + b - vb, uint64_t{plan.block_cap}));
      plan.d_token_first[i] = static_cast<uint32_t>(min(before_t + t - vt, uint64_t{plan.token_cap}));
    }
    __syncthreads();
  }
}

// Every CTA adds up the lengths of the sequences before its own: 12 bytes a sequence from L2, the
// square of the batch in all.  Past this many sequences one more launch does it once.
constexpr uint32_t kOwnPrefix = 2048;

}  // namespace
}  // namespace hlkv

extern "C" int hlkv_batch_plan(const HlkvBatchPlan* plan, const HlkvLayout* layout, const HlkvExecDescriptor* d_table,
                               uint32_t table_size, const uint32_t* d_arena, uint32_t arena_size,
                               const HlkvSegment* d_segs, const uint32_t* d_query_lens, uint32_t* d_err,
                               hlkv_stream_t stream) {
  using namespace hlkv;
  if (plan == nullptr || !layout_ok(layout) || d_err == nullptr || plan->max_query == 0) return HLKV_INVALID_ARGUMENT;
  if (plan->nseq == 0) return HLKV_OK;
  if (plan->d_block_first == nullptr || plan->d_block_count == nullptr || plan->d_token_first == nullptr ||
      plan->d_context == nullptr || d_segs == nullptr || plan->d_cost == nullptr ||
      (plan->block_cap > 0 && (plan->d_blocks == nullptr || plan->d_block_cost == nullptr)) ||
      (plan->token_cap > 0 && (plan->d_targets == nullptr || plan->d_positions == nullptr)) ||
      (table_size > 0 && d_table == nullptr) || (arena_size > 0 && d_arena == nullptr) ||
      (reinterpret_cast<uintptr_t>(plan->d_blocks) & 15u) != 0 || (reinterpret_cast<uintptr_t>(plan->d_targets) & 7u) != 0 ||
      (reinterpret_cast<uintptr_t>(d_table) & 15u) != 0 || (reinterpret_cast<uintptr_t>(d_segs) & 7u) != 0) {
    return HLKV_INVALID_ARGUMENT;
  }
  // Grids stay below 2^31 CTAs with any cluster size.
  if (plan->nseq > 0x7FFFFFFFu / kMaxCluster) return HLKV_INVALID_ARGUMENT;
  // Positions are 31 bits, and the sum of the costs (at most 14 per 16 tokens or block) 32.
  if (uint64_t{plan->block_cap} * layout->block_tokens > 0x7FFFFFFFull || plan->block_cap > (1u << 27)) {
    return HLKV_INVALID_ARGUMENT;
  }
  Params p{};
  p.plan = *plan;
  p.table = reinterpret_cast<const uint4*>(d_table);
  p.arena = d_arena;
  p.segs = reinterpret_cast<const uint2*>(d_segs);
  p.qlens = d_query_lens;
  p.err = d_err;
  p.table_size = table_size;
  p.arena_size = arena_size;
  p.T = layout->block_tokens;
  p.layout_id = layout->layout_id;
  const cudaStream_t launch_stream = reinterpret_cast<cudaStream_t>(stream);
  if (plan->nseq > kOwnPrefix) {
    p.prefix_done = 1;
    batch_plan_prefix<<<1, 1024, 0, launch_stream>>>(p.segs, p.qlens, *plan);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_status(e);
  }
  // One CTA per kRound blocks of an average sequence, as far as the clusters still fit the GPU.
  const uint64_t average = plan->block_cap / plan->nseq;
  unsigned ctas = 1;
  while (ctas < kMaxCluster && uint64_t{ctas} * kRound < average &&
         uint64_t{plan->nseq} * ctas * 2 <= static_cast<uint64_t>(sm_count()) * 4) {
    ctas *= 2;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(plan->nseq * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = launch_stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, batch_plan_kernel, p));
}
