// What the kernels of the batch attention share: the call's parameters, the checks of a plan's
// blocks, and barrier and copy instructions.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "codec.cuh"
#include "common.cuh"
#include "hlkv.h"

namespace hlkv {
namespace battn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kMaxGroup = 32;
// Sequences whose query rows per KV head (new tokens x group) are at most this many are streamed
// (stream_kernel); the others go to the tile kernel.
constexpr uint32_t kStreamRows = 16;

struct DevPool {
  const uint8_t* base;
  uint64_t slot_bytes;
  uint32_t num_slots;
};

struct Params {
  DevPool pool[4];
  uint64_t code_bytes[4];
  const uint32_t *block_first, *block_count, *token_first, *context, *block_cost, *cost;
  const uint4* blocks;
  const uint16_t* q;
  uint16_t* out;
  uint64_t q_stride, out_stride;
  uint32_t* err;
  uint32_t nseq, T, H, q_heads, group, window, sinks, block_cap, token_cap;
  uint32_t max_rows;  // most query rows per (sequence, KV head): max_query * group
  float qscale;       // softmax_scale * log2(e)
  // stream kernel and merge
  uint32_t head_groups;  // KV heads are taken in groups of at most 8
  uint32_t ctas;
  uint32_t slot_rows;    // rows per head of a partial result
  uint64_t* prefix;      // [nseq + 1] cost of the sequences before
  float* partial;        // [ctas + nseq * head_groups][8][slot_rows][kD + 4]: outputs, max, sum
};

// The new tokens of sequence i: rows [first, first + q) of Q, kept inside the arrays whatever the
// plan holds.
struct Rows {
  uint32_t first, q;
};
__device__ __forceinline__ Rows rows_of(const Params& p, uint32_t i) {
  const uint32_t a = min(p.token_first[i], p.token_cap), b = min(p.token_first[i + 1], p.token_cap);
  return Rows{a, b > a ? b - a : 0u};
}
__device__ __forceinline__ uint32_t count_of(const Params& p, uint32_t i, uint32_t* first) {
  *first = min(p.block_first[i], p.block_cap);
  return min(p.block_count[i], p.block_cap - *first);
}

// The pool checks of a listed block; returns the format (4 = left out) and the slot's address.
__device__ __forceinline__ uint32_t open_block(const Params& p, uint4 b, const uint8_t** payload) {
  const uint32_t f = b.y & 0xFu;
  uint32_t bad = 0;
  if (f > 3 || p.pool[f].base == nullptr) bad = dev::kErrBadFormat;
  else if (b.x >= p.pool[f].num_slots) bad = dev::kErrSlotRange;
  if (bad) {
    atomicOr(p.err, bad);
    return 4;
  }
  *payload = p.pool[f].base + uint64_t{b.x} * p.pool[f].slot_bytes;
  return f;
}

// ---- barriers in shared memory and bulk copies ------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_fence_init() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// Waits for the phase of the given parity to complete; false when it gives up (each try suspends
// for a hardware time limit, so this is far beyond any kernel's time).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t a = smem_addr(bar);
  for (uint32_t i = 0; i < (1u << 24); ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return false;
}
// Global -> shared (by address), `bytes` a multiple of 16, both addresses 16-byte aligned.
__device__ __forceinline__ void bulk_load(uint32_t dst, uint64_t src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// Launches of the kernels (their translation units).
cudaError_t launch_stream(uint32_t head_dim, const Params& p, cudaStream_t s);
size_t stream_workspace(uint32_t nseq, uint32_t H, uint32_t head_dim, uint32_t max_rows, uint32_t ctas);
void stream_layout(Params* p, void* ws);

}  // namespace battn
}  // namespace hlkv
