// What the kernels of the batch attention share: the call's parameters, the checks of a plan's
// blocks, and barrier and copy instructions.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "codec.cuh"
#include "common.cuh"
#include "hlkv.h"

namespace hlkv {
namespace battn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kMaxGroup = 32, kMaxKvHeads = 128;  // (a token's parameters of all heads come in one copy)
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
  uint32_t max_query;
  uint32_t max_rows;  // most query rows per (sequence, KV head): max_query * group
  float qscale;       // softmax_scale * log2(e)
  // stream kernel and merge
  uint32_t head_groups;  // KV heads are taken in groups of at most 8
  uint32_t ctas;
  uint32_t slot_rows;    // rows per head of a partial result
  uint64_t* prefix;      // [nseq + 1] cost of the sequences before
  float* partial;        // [ctas + nseq * head_groups][8][slot_rows][kD + 4]: outputs, max, sum
  // tile kernel and join
  float* tile_partial;  // [ctas][256][kD + 4]
  uint32_t* tile_redo;  // [ctas]
  uint32_t tile_ranks;  // more than 128 sequences: CTAs (of a head) take ranks; 0: one for each tile of the plan
};

// The new tokens of sequence i: rows [first, first + q) of Q, kept inside the arrays whatever the
// plan holds.  A sequence with more than max_query of them, which the plan rejected, has none here: grids and
// workspaces are made for max_query.
struct Rows {
  uint32_t first, q;
};
__device__ __forceinline__ Rows rows_of(const Params& p, uint32_t i) {
  const uint32_t a = min(p.token_first[i], p.token_cap), b = min(p.token_first[i + 1], p.token_cap);
  return Rows{a, b > a && b - a <= p.max_query ? b - a : 0u};
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

// ---- codes as binary16 ------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Two FP8 codes in the low (or high) half of w -> their values as binary16.
template <uint32_t kF>
__device__ __forceinline__ uint32_t fp8_lo(uint32_t w) {
  uint32_t h;
  if constexpr (kF == dev::kE4M3) {
    asm("{.reg .b16 l, u; mov.b32 {l, u}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(h) : "r"(w));
  } else {
    h = __byte_perm(w, 0u, 0x1404);  // an E5M2 code is the upper byte of its binary16 value
  }
  return h;
}
template <uint32_t kF>
__device__ __forceinline__ uint32_t fp8_hi(uint32_t w) {
  uint32_t h;
  if constexpr (kF == dev::kE4M3) {
    asm("{.reg .b16 l, u; mov.b32 {l, u}, %1; cvt.rn.f16x2.e4m3x2 %0, u;}" : "=r"(h) : "r"(w));
  } else {
    h = __byte_perm(w, 0u, 0x3424);
  }
  return h;
}
__device__ __forceinline__ bool has_nonfinite(uint32_t h2) {
  return (h2 & 0x7C00u) == 0x7C00u || (h2 & 0x7C000000u) == 0x7C000000u;
}

// 1024 + c and 1024 + 16 c from masks -> (c - 8) / 8 by (1024 + c) / 8 - 129 and (1024 + 16 c) / 128 - 9: exact.
// One logic operation holds one immediate, the mask; the other constant comes in a register.
__device__ __forceinline__ uint32_t magic1024() {
  uint32_t m;
  asm("mov.b32 %0, 0x64006400;" : "=r"(m));
  return m;
}
__device__ __forceinline__ uint32_t nibble_lo(uint32_t x, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r) : "r"(x), "r"(magic));
  return hfma2(r, 0x30003000u, 0xD808D808u);
}
__device__ __forceinline__ uint32_t nibble_hi(uint32_t x, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(r) : "r"(x), "r"(magic));
  return hfma2(r, 0x20002000u, 0xC880C880u);
}

// 2^x by the hardware's approximation (2^-22 of the result; subnormal results are 0).
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// 2^-k for a whole k >= 0.
__device__ __forceinline__ float halvings(float k) { return k > 126.0f ? 0.0f : __int_as_float((127 - static_cast<int>(k)) << 23); }

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
// Waits for the phase of the given parity to complete; false when it gives up, after tries whose sum is far beyond
// any wait of these kernels (a tile's copy or products: microseconds).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t a = smem_addr(bar);
  for (uint32_t i = 0; i < (1u << 22); ++i) {
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

// ---- one row by one warp --------------------------------------------------------------------------
// kN consecutive elements of a row from element e, and the row's {scale, bias}: the codes' values
// without the parameters.
template <int kN>
__device__ __forceinline__ void load_codes(uint32_t f, const uint8_t* payload, uint64_t elem, float (&x)[kN]) {
  static_assert(kN == 2 || kN == 4);
  if (f == dev::kFp16) {
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(payload + (elem + i) * 2));
      x[i] = v.x;
      x[i + 1] = v.y;
    }
  } else if (f == dev::kInt4) {
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      const uint32_t w = payload[(elem + i) >> 1];
      x[i] = static_cast<float>(w & 15u);
      x[i + 1] = static_cast<float>(w >> 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; i += 2) {
      const uint32_t w = *reinterpret_cast<const uint16_t*>(payload + elem + i);
      const float2 v = f == dev::kE4M3 ? dev::fp8x2_exact<dev::kE4M3>(w) : dev::fp8x2_exact<dev::kE5M2>(w);
      x[i] = v.x;
      x[i + 1] = v.y;
    }
  }
}

__device__ __forceinline__ float2 params_of_row(uint32_t f, uint32_t info, uint32_t sref, const uint8_t* params, uint32_t row) {
  if (f == dev::kFp16) return make_float2(1.0f, 0.0f);
  const uint32_t mode = (info >> 4) & 3u;
  if (mode != 0) return dev::block_params_value(mode, sref);
  if (f == dev::kInt4) return __ldg(reinterpret_cast<const float2*>(params) + row);
  return make_float2(__ldg(reinterpret_cast<const float*>(params) + row), 0.0f);
}

// One row (new token of sequence i at position pos, query head qh) by one warp, token by token: lane l holds
// elements [l kN, (l + 1) kN) of the head.
template <int kD>
__device__ __noinline__ void attend_row(const Params& p, uint32_t i, uint32_t token, int64_t pos, uint32_t qh) {
  constexpr int kN = kD / 32;
  const uint32_t lane = threadIdx.x & 31, h = qh / p.group;
  float q[kN], acc[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    q[i] = __half2float(__ushort_as_half(p.q[token * p.q_stride + uint64_t{qh} * kD + lane * kN + i])) * p.qscale;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  uint32_t first;
  const uint32_t count = count_of(p, i, &first);
  for (uint32_t j = 0; j < count; ++j) {
    const uint4 b = __ldg(p.blocks + first + j);
    const uint32_t vt = min((b.y >> 10) & 0x3FFu, p.T);
    const uint8_t* payload;
    const uint32_t f = open_block(p, b, &payload);
    if (f > 3) continue;
    for (uint32_t k_tok = 0; k_tok < vt; ++k_tok) {
      const int64_t t = int64_t{b.w} + k_tok;
      if (t > pos || (p.window != 0 && pos - t >= p.window && t >= p.sinks)) continue;
      float k[kN], v[kN];
      const uint32_t krow = k_tok * p.H + h, vrow = krow + p.T * p.H;
      load_codes<kN>(f, payload, uint64_t{krow} * kD + lane * kN, k);
      load_codes<kN>(f, payload, uint64_t{vrow} * kD + lane * kN, v);
      const float2 kp = params_of_row(f, b.y, b.z, payload + p.code_bytes[f], krow);
      const float2 vp = params_of_row(f, b.y, b.z, payload + p.code_bytes[f], vrow);
      float x = 0.0f;
#pragma unroll
      for (int e = 0; e < kN; ++e) x = fmaf(q[e], fmaf(k[e], kp.x, kp.y), x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
      const float mn = fmaxf(m, x);
      const float a = mn == -INFINITY ? 1.0f : exp2f(m - mn), w = x == -INFINITY ? 0.0f : exp2f(x - mn);
      l = fmaf(l, a, w);
#pragma unroll
      for (int e = 0; e < kN; ++e) acc[e] = fmaf(acc[e], a, w * fmaf(v[e], vp.x, vp.y));
      m = mn;
    }
  }
#pragma unroll
  for (int e = 0; e < kN; ++e) {
    const float r = m == -INFINITY && l == 0.0f ? 0.0f : acc[e] / l;
    p.out[token * p.out_stride + uint64_t{qh} * kD + lane * kN + e] = __half_as_ushort(__float2half_rn(r));
  }
}

// A kernel's permission for large shared memory, asked for once per device (a microsecond of each call).
struct SharedMemoryOnce {
  std::atomic<uint64_t> done{0};
  cudaError_t allow(const void* kernel, uint32_t bytes) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? uint64_t{1} << device : 0u;
    if ((done.load(std::memory_order_relaxed) & bit) != 0) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
  }
};

// Launches of the kernels (their translation units).
cudaError_t launch_stream(uint32_t head_dim, const Params& p, cudaStream_t s);
size_t stream_workspace(uint32_t nseq, uint32_t H, uint32_t head_dim, uint32_t max_rows, uint32_t ctas);
void stream_layout(Params* p, void* ws);
size_t tile_workspace(uint32_t nseq, uint32_t head_dim, uint32_t max_rows, uint32_t ctas);
uint64_t tiles_of_plan(const Params& p);
uint32_t tile_ranks(const Params& p);
uint64_t tile_ctas(const Params& p);  // the tile kernel's grid: 0 when no sequence can have its rows
cudaError_t launch_tiles(uint32_t head_dim, const Params& p, cudaStream_t s);

}  // namespace battn
}  // namespace hlkv
