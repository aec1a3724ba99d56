// Rotary append: Q and K of new tokens turned by their positions, Q written out in binary16, K and
// V encoded into their blocks' formats, in one pass over the projection's output.
//
// Pair j of a head turns by a = position[axis_j] * inv_freq_j.  For positions below 2^29 the
// binary64 product is exact (29 + 24 bits), and a is reduced by pi/2 in binary64: a position of
// 10^6 costs no digit, where a binary32 angle would be off by 0.06.  cos and sin are
// the Taylor series on [-pi/4, pi/4] up to r^17, rounded once to binary32.  They are computed once
// per token and CTA and shared by all its heads.
//
// A row (one head of one token) is handled by D/16 lanes with two 8-element chunks each, l and
// l + D/16, as kernel (2) lays it out; for a fully rotated head in halves the two chunks are the
// partners of each other.
//
// The bound is memory for prompts: 2 D (2 q_heads + 2 kv_heads) bytes and the codes of a token, once each; for a
// decode step it is the chain target, descriptor, store after the launch.  Measured with 32 query and 8 KV heads of
// 128: 8192 tokens 39 us (4.4 TB/s of Q, K and V alone), 64 tokens 3.8 us.  A row's loads are issued while the row
// before is turned and encoded; quotients are taken by a bracket of two products and divided only where its ends
// round apart.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "codec.cuh"
#include "common.cuh"
#include "hlkv.h"
#include "row_encode.cuh"

namespace hlkv {
namespace {

constexpr int kThreads = 256;
constexpr int kChunks = 2;
constexpr uint32_t kMaxTokens = 8;  // of a CTA

enum : int { kHalves = 0, kHalvesPartial = 1, kAdjacent = 2 };  // how pairs lie in a head

struct DevPool {
  uint8_t* base;
  uint64_t slot_bytes;
  uint32_t num_slots;
};

struct Params {
  DevPool pool[4];
  uint64_t code_bytes[4];
  const uint4* table;
  const uint2* targets;
  const int32_t* positions;
  int64_t pos_token, pos_axis;
  const uint16_t *q, *k, *v;
  uint16_t* q_out;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;
  uint32_t* err;
  uint32_t table_size, T, H, layout_id, q_heads, n, tokens_per_cta;
  FastDiv rows_per_token;  // q_heads + 2 H
  HlkvRotary rope;
};

// sin and cos of an angle in binary64, |x| < 2^48: x - k pi/2 with pi/2 in two parts (the product
// k * hi is exact inside the fused operation), then the series; the quadrant swaps and signs.
__device__ __forceinline__ void sincos64(double x, double* sn, double* cs) {
  const double k = rint(x * 0.63661977236758134308);  // 2 / pi
  double r = fma(-k, 1.57079632679489661923, x);      // pi / 2
  r = fma(-k, 6.123233995736766e-17, r);              // pi / 2 - binary64(pi / 2)
  const double z = r * r;
  double s = 1.0 / 355687428096000.0;  // 1 / 17!
  s = fma(s, -z, 1.0 / 1307674368000.0);
  s = fma(s, -z, 1.0 / 6227020800.0);
  s = fma(s, -z, 1.0 / 39916800.0);
  s = fma(s, -z, 1.0 / 362880.0);
  s = fma(s, -z, 1.0 / 5040.0);
  s = fma(s, -z, 1.0 / 120.0);
  s = fma(s, -z, 1.0 / 6.0);
  s = fma(s * -z, r, r);
  double c = 1.0 / 20922789888000.0;  // 1 / 16!
  c = fma(c, -z, 1.0 / 87178291200.0);
  c = fma(c, -z, 1.0 / 479001600.0);
  c = fma(c, -z, 1.0 / 3628800.0);
  c = fma(c, -z, 1.0 / 40320.0);
  c = fma(c, -z, 1.0 / 720.0);
  c = fma(c, -z, 1.0 / 24.0);
  c = fma(c, -z, 0.5);
  c = fma(c, -z, 1.0);
  const long long n = static_cast<long long>(k);
  const double a = (n & 1) ? c : s, b = (n & 1) ? s : c;
  *sn = (n & 2) ? -a : a;
  *cs = ((n + 1) & 2) ? -b : b;
}

__device__ __forceinline__ void widen(uint4 raw, float* x) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 narrow(const float* x) {
  return make_uint4(dev::pack_f16x2(x[0], x[1]), dev::pack_f16x2(x[2], x[3]), dev::pack_f16x2(x[4], x[5]),
                    dev::pack_f16x2(x[6], x[7]));
}

// (x, y) -> (x c - y s, y c + x s), each operation rounded: a fused form would depend on which
// product it fuses.
__device__ __forceinline__ float turned_x(float x, float y, float2 cs) {
  return __fsub_rn(__fmul_rn(x, cs.x), __fmul_rn(y, cs.y));
}
__device__ __forceinline__ float turned_y(float x, float y, float2 cs) {
  return __fadd_rn(__fmul_rn(y, cs.x), __fmul_rn(x, cs.y));
}

// Scales whose reciprocal, and so the bracket around a quotient, is exact to 2^-24: outside of them (a factor far from
// one) the reciprocal overflows or is subnormal, and every quotient is a division.
__device__ __forceinline__ bool reciprocal_ok(float scale) { return scale >= 0x1p-126f && scale <= 0x1p126f; }

// One row of binary32 values (two chunks of 8 per lane) in format f into row `row` of a slot.  The
// rules are dev::encode_row's (the reference's quantize_reference) but for the scale, which is the
// product amax * (1 / max_finite) or range * (1 / 15) with the reciprocal in binary32 instead of the
// quotient: within 1.5 units in the last place of the exact value where the quotient is within half
// a unit.  That is the operator's definition, not a gain (8192 tokens take 49.7 us with the gather, and 49.8 with the
// quotient): a row's bytes can differ from append_encode's of the same values.  Codes are the IEEE quotients by
// that scale, rounded to nearest even.
template <int kD>
__device__ __forceinline__ uint32_t encode_row_f32(uint32_t f, const float (&x)[16], uint32_t lane, uint32_t mask,
                                                   uint8_t* payload, uint32_t row, uint64_t code_bytes) {
  constexpr int kLanes = kD / 16;
  if (f == dev::kFp16) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      reinterpret_cast<uint4*>(payload + uint64_t{row} * kD * 2)[c * kLanes + lane] = dev::canon_f16x8(narrow(x + 8 * c));
    }
    return 0;
  }
  if (f == dev::kInt4) {
    float mn = x[0], mx = x[0];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      mn = fminf(mn, x[i]);
      mx = fmaxf(mx, x[i]);
      fine = fine && dev::finite_f32(x[i]);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      mn = fminf(mn, __shfl_xor_sync(mask, mn, o, kLanes));
      mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o, kLanes));
    }
    const float range = __fsub_rn(mx, mn);
    if (!__all_sync(mask, fine) || !dev::finite_f32(range)) return dev::kErrNonFinite;
    const float scale = __fmul_rn(range, 1.0f / 15.0f);
    uint32_t word[2] = {0u, 0u};
    if (scale > 0.0f) {
      const float y = __frcp_rn(scale), ylo = __fmul_rn(y, dev::kBracketLo), yhi = __fmul_rn(y, dev::kBracketHi);
      uint32_t diff = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float d = __fsub_rn(x[i], mn);
        const uint32_t qa = dev::rint_u(__fmul_rn(d, ylo)), qb = dev::rint_u(__fmul_rn(d, yhi));
        diff |= qa ^ qb;
        word[i / 8] |= min(qa, 15u) << (4 * (i % 8));
      }
      if (diff != 0 || !reciprocal_ok(scale)) {  // near the middle of two codes: the divisions themselves
        word[0] = word[1] = 0u;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t q = dev::rint_u(__fdiv_rn(__fsub_rn(x[i], mn), scale));
          word[i / 8] |= min(q, 15u) << (4 * (i % 8));
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      reinterpret_cast<uint32_t*>(payload + uint64_t{row} * (kD / 2))[c * kLanes + lane] = word[c];
    }
    if (lane == 0) reinterpret_cast<float2*>(payload + code_bytes)[row] = make_float2(scale, mn);
    return 0;
  }
  // Magnitude bits order as magnitudes; Inf and NaN are the ones from 0x7F800000 up.
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(mask, m, o, kLanes));
  if (m >= 0x7F800000u) return dev::kErrNonFinite;
  float scale = 1.0f;
  if (m > 0) scale = fmaxf(__fmul_rn(__uint_as_float(m), f == dev::kE4M3 ? 1.0f / 448.0f : 1.0f / 57344.0f), 1.17549435e-38f);
  const float y = __frcp_rn(scale), ylo = __fmul_rn(y, dev::kBracketLo), yhi = __fmul_rn(y, dev::kBracketHi);
  uint32_t r[8], diff = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a0 = __fmul_rn(x[2 * i], ylo), a1 = __fmul_rn(x[2 * i + 1], ylo);
    const float b0 = __fmul_rn(x[2 * i], yhi), b1 = __fmul_rn(x[2 * i + 1], yhi);
    r[i] = f == dev::kE4M3 ? dev::cvt_e4m3x2(a0, a1) : dev::cvt_e5m2x2(a0, a1);
    diff |= r[i] ^ (f == dev::kE4M3 ? dev::cvt_e4m3x2(b0, b1) : dev::cvt_e5m2x2(b0, b1));
  }
  if (diff != 0 || !reciprocal_ok(scale)) {  // near the middle of two codes: the divisions themselves
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = __fdiv_rn(x[2 * i], scale), b = __fdiv_rn(x[2 * i + 1], scale);
      r[i] = f == dev::kE4M3 ? dev::cvt_e4m3x2(a, b) : dev::cvt_e5m2x2(a, b);
    }
  }
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    reinterpret_cast<uint2*>(payload + uint64_t{row} * kD)[c * kLanes + lane] =
        make_uint2(r[4 * c] | r[4 * c + 1] << 16, r[4 * c + 2] | r[4 * c + 3] << 16);
  }
  if (lane == 0) reinterpret_cast<float*>(payload + code_bytes)[row] = scale;
  return 0;
}

// Where a token's K and V go: resolved once per token and CTA.
struct Place {
  uint8_t* payload;
  uint32_t f;      // format; kSkip: no store; kPadding: nothing at all
  uint32_t token;  // slot in the block
};
constexpr uint32_t kSkip = 16, kPadding = 17;

template <int kD, int kMode>
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = kD / 16;
  constexpr int kRowsPerIter = kThreads / kLanes;
  // [tokens_per_cta][rotary_dim / 2] cos and sin: two pairs to 16 bytes, those of all chunks side by side, so that the
  // lanes of a row read neighbouring ones.  (In the order of the pairs lanes lie 64 bytes apart: 42 us against 39
  // for 8192 tokens.)
  extern __shared__ __align__(16) float2 s_cs[];
  constexpr uint32_t kPairs = kMode == kAdjacent ? 4 : 8;  // of a chunk
  __shared__ Place s_place[kMaxTokens];
  const uint32_t lane = threadIdx.x % kLanes;
  const uint32_t mask = dev::row_mask<kD, kChunks>();
  const uint32_t pairs = p.rope.rotary_dim / 2, cs_chunks = pairs / kPairs;
  const uint32_t token0 = blockIdx.x * p.tokens_per_cta;
  const uint32_t tokens = min(p.tokens_per_cta, p.n - token0);
  const uint32_t rows = tokens * p.rows_per_token.d;

  // A row's source: its loads do not wait for the angles or the targets.
  auto source = [&](uint32_t g, uint32_t* t, uint32_t* r) {
    *t = p.rows_per_token.div(g);
    *r = g - *t * p.rows_per_token.d;
    const uint32_t token = token0 + *t;
    return *r < p.q_heads         ? p.q + token * p.q_stride + uint64_t{*r} * kD
           : *r < p.q_heads + p.H ? p.k + token * p.k_stride + uint64_t{*r - p.q_heads} * kD
                                  : p.v + token * p.v_stride + uint64_t{*r - p.q_heads - p.H} * kD;
  };
  uint32_t g = threadIdx.x / kLanes, t = 0, r = 0;
  const uint16_t* src = nullptr;
  uint4 next[kChunks];
  if (g < rows) {
    src = source(g, &t, &r);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) next[c] = __ldcs(reinterpret_cast<const uint4*>(src) + c * kLanes + lane);
  }

  // The last threads resolve the targets while the first ones take the angles.
  const uint32_t back = kThreads - 1 - threadIdx.x;
  if (back < tokens) {
    const uint2 target = __ldg(p.targets + token0 + back);
    Place place{nullptr, kSkip, target.y};
    uint32_t bad = 0;
    if (target.x == 0xFFFFFFFFu && target.y == 0xFFFFFFFFu) {
      place.f = kPadding;
    } else if (target.x >= p.table_size) {
      bad = dev::kErrBlockIdRange;
    } else {
      const uint4 d = __ldg(p.table + target.x);
      const uint32_t f = d.y & 0xFu, mode = (d.y >> 4) & 3u, layout = (d.y >> 6) & 0xFu;
      if (d.w != target.x) bad = dev::kErrDescMismatch;
      else if (f == dev::kInvalidFormat) bad = dev::kErrNotExecutable;
      else if (f > 3 || p.pool[f].base == nullptr || p.pool[f].num_slots == 0) bad = dev::kErrBadFormat;
      else if (layout != p.layout_id) bad = dev::kErrLayout;
      else if (f != dev::kFp16 && mode != 0) bad = dev::kErrScaleMode;
      else if (target.y >= p.T) bad = dev::kErrTokenRange;
      else if (d.x >= p.pool[f].num_slots) bad = dev::kErrSlotRange;
      else {
        place.payload = p.pool[f].base + uint64_t{d.x} * p.pool[f].slot_bytes;
        place.f = f;
      }
    }
    if (bad) atomicOr(p.err, bad);
    s_place[back] = place;
  }
  for (uint32_t i = threadIdx.x; i < tokens * pairs; i += kThreads) {
    const uint32_t k = i / pairs, j = i - k * pairs;
    const int32_t pos = __ldg(p.positions + (token0 + k) * p.pos_token + p.rope.pair_axis[j] * p.pos_axis);
    double sn, cs;
    sincos64(static_cast<double>(pos) * static_cast<double>(p.rope.inv_freq[j]), &sn, &cs);
    const double f = p.rope.factor;
    s_cs[k * pairs + (j % kPairs / 2 * cs_chunks + j / kPairs) * 2 + j % 2] = make_float2(static_cast<float>(cs * f), static_cast<float>(sn * f));
  }
  __syncthreads();

  for (; g < rows; g += kRowsPerIter) {
    // Everything below is uniform over the lanes of row g.
    const uint32_t token = token0 + t, row_t = t, row_r = r;
    const uint16_t* const row_src = src;
    uint4 raw[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) raw[c] = next[c];
    if (g + kRowsPerIter < rows) {  // the next row's loads
      src = source(g + kRowsPerIter, &t, &r);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) next[c] = __ldcs(reinterpret_cast<const uint4*>(src) + c * kLanes + lane);
    }
    const uint32_t f = s_place[row_t].f;
    const bool is_q = row_r < p.q_heads, is_v = row_r >= p.q_heads + p.H;
    if (f == kPadding || (f == kSkip && !is_q)) continue;

    float x[16];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) widen(raw[c], x + 8 * c);
    if (!is_v) {
      const float4* cs = reinterpret_cast<const float4*>(s_cs + row_t * pairs);
      // pairs 2 i and 2 i + 1 of a chunk
      auto two = [&](uint32_t of_chunk, uint32_t i) { return cs[i * cs_chunks + of_chunk]; };
      if constexpr (kMode == kHalves) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const float4 w = two(lane, i / 2);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 wk = k ? make_float2(w.z, w.w) : make_float2(w.x, w.y);
            const float a = x[i + k], b = x[8 + i + k];
            x[i + k] = turned_x(a, b, wk);
            x[8 + i + k] = turned_y(a, b, wk);
          }
        }
      } else if constexpr (kMode == kAdjacent) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t chunk = c * kLanes + lane;
          if (chunk * 8 < p.rope.rotary_dim) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 w2 = two(chunk, i / 2);
              const float2 w = i & 1 ? make_float2(w2.z, w2.w) : make_float2(w2.x, w2.y);
              const float a = x[8 * c + 2 * i], b = x[8 * c + 2 * i + 1];
              x[8 * c + 2 * i] = turned_x(a, b, w);
              x[8 * c + 2 * i + 1] = turned_y(a, b, w);
            }
          }
        }
      } else {
        // The partner chunk lies rotary_dim / 2 elements on or back, in another lane or in this
        // one: read it again.
        const uint32_t half = p.rope.rotary_dim / 16;  // chunks per half
        uint4 other[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t chunk = c * kLanes + lane;
          other[c] = raw[c];
          if (chunk < 2 * half) {
            other[c] = __ldcs(reinterpret_cast<const uint4*>(row_src) + (chunk < half ? chunk + half : chunk - half));
          }
        }
        __syncwarp(mask);  // d_q_out may be d_q: every lane has read its partner before one writes
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const uint32_t chunk = c * kLanes + lane;
          if (chunk < 2 * half) {
            float y[8];
            widen(other[c], y);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 w2 = two(chunk < half ? chunk : chunk - half, i / 2);
              const float2 w = i & 1 ? make_float2(w2.z, w2.w) : make_float2(w2.x, w2.y);
              x[8 * c + i] = chunk < half ? turned_x(x[8 * c + i], y[i], w) : turned_y(y[i], x[8 * c + i], w);
            }
          }
        }
      }
    }
    if (is_q) {
      uint4* dst = reinterpret_cast<uint4*>(p.q_out + token * p.q_out_stride + uint64_t{row_r} * kD);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) dst[c * kLanes + lane] = narrow(x + 8 * c);
      continue;
    }
    const uint32_t h = row_r - p.q_heads - (is_v ? p.H : 0u);
    const uint32_t row = ((is_v ? p.T : 0u) + s_place[row_t].token) * p.H + h;
    const uint32_t e = encode_row_f32<kD>(f, x, lane, mask, s_place[row_t].payload, row, p.code_bytes[f]);
    if (e != 0 && lane == 0) atomicOr(p.err, e);
  }
}

template <int kD>
void (*kernel_for(int mode))(const Params) {
  return mode == kHalves ? rotary_append_kernel<kD, kHalves>
         : mode == kAdjacent ? rotary_append_kernel<kD, kAdjacent>
                             : rotary_append_kernel<kD, kHalvesPartial>;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool rotary_ok(const HlkvRotary* r, uint32_t head_dim) {
  if (r == nullptr || r->rotary_dim == 0 || r->rotary_dim % 16 != 0 || r->rotary_dim > head_dim || r->interleaved > 1 ||
      r->axes < 1 || r->axes > 4 || !std::isfinite(r->factor)) {
    return false;
  }
  for (uint32_t j = 0; j < r->rotary_dim / 2; ++j) {
    if (!(std::fabs(r->inv_freq[j]) <= 65536.0f) || r->pair_axis[j] >= r->axes) return false;
  }
  return true;
}

}  // namespace
}  // namespace hlkv

extern "C" int hlkv_rotary_append(const HlkvPools* pools, const HlkvLayout* layout, const HlkvExecDescriptor* d_table,
                                  uint32_t table_size, const HlkvAppendTarget* d_targets, uint32_t n,
                                  const HlkvRotary* rotary, const int32_t* d_positions, int64_t position_token_stride,
                                  int64_t position_axis_stride, const uint16_t* d_q, uint32_t q_heads,
                                  uint64_t q_stride, const uint16_t* d_k, uint64_t k_stride, const uint16_t* d_v,
                                  uint64_t v_stride, uint16_t* d_q_out, uint64_t q_out_stride, uint32_t* d_err,
                                  hlkv_stream_t stream) {
  using namespace hlkv;
  if (pools == nullptr || !layout_ok(layout) || d_err == nullptr || !rotary_ok(rotary, layout->head_dim)) {
    return HLKV_INVALID_ARGUMENT;
  }
  if (n == 0) return HLKV_OK;
  const uint64_t D = layout->head_dim, H = layout->kv_heads;
  if (d_targets == nullptr || d_positions == nullptr || d_k == nullptr || d_v == nullptr ||
      (table_size > 0 && d_table == nullptr) || !aligned16(d_table) || (reinterpret_cast<uintptr_t>(d_targets) & 7u) != 0 || !aligned16(d_k) ||
      !aligned16(d_v) || k_stride % 8 != 0 || v_stride % 8 != 0 || k_stride < H * D || v_stride < H * D) {
    return HLKV_INVALID_ARGUMENT;
  }
  if (q_heads > 0 && (d_q == nullptr || d_q_out == nullptr || !aligned16(d_q) || !aligned16(d_q_out) ||
                      q_stride % 8 != 0 || q_out_stride % 8 != 0 || q_stride < q_heads * D || q_out_stride < q_heads * D ||
                      (d_q == d_q_out && q_stride != q_out_stride))) {
    return HLKV_INVALID_ARGUMENT;
  }
  const uint64_t rows_per_token = uint64_t{q_heads} + 2 * H;
  if (rows_per_token * n >= (uint64_t{1} << 31)) return HLKV_INVALID_ARGUMENT;
  Params p{};
  const uint64_t elems = 2 * layout->block_tokens * H * D;
  for (int f = 0; f < 4; ++f) {
    const HlkvPool& q = pools->pool[f];
    p.code_bytes[f] = layout_code_bytes(f, elems);
    if (q.base == nullptr || q.num_slots == 0) continue;
    if (!aligned16(q.base) || (q.slot_bytes & 15u) != 0 || q.slot_bytes < hlkv_layout_slot_bytes(f, layout)) {
      return HLKV_INVALID_ARGUMENT;
    }
    p.pool[f] = DevPool{static_cast<uint8_t*>(q.base), q.slot_bytes, q.num_slots};
  }
  p.table = reinterpret_cast<const uint4*>(d_table);
  p.targets = reinterpret_cast<const uint2*>(d_targets);
  p.positions = d_positions;
  p.pos_token = position_token_stride;
  p.pos_axis = position_axis_stride;
  p.q = d_q;
  p.k = d_k;
  p.v = d_v;
  p.q_out = d_q_out;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.q_out_stride = q_out_stride;
  p.err = d_err;
  p.table_size = table_size;
  p.T = layout->block_tokens;
  p.H = layout->kv_heads;
  p.layout_id = layout->layout_id;
  p.q_heads = q_heads;
  p.n = n;
  p.rows_per_token = FastDiv(static_cast<uint32_t>(rows_per_token));
  p.rope = *rotary;
  // Tokens of a CTA: rows enough for three rounds of its threads (8192 tokens of 48 rows with the gather: 63, 53, 54 us at
  // 1, 2, 4 tokens a CTA; 1285 of 16 short rows: 11.2, 9.6, 8.8, 9.6 us at 1, 2, 4, 8), as long as every SM has two CTAs
  // (64 tokens: 9.7 us at 1, 10.0 at 2).
  const uint64_t threads = rows_per_token * (D / 16);
  p.tokens_per_cta = 1;
  while (p.tokens_per_cta < kMaxTokens && p.tokens_per_cta * threads < 3 * kThreads &&
         n / (2 * p.tokens_per_cta) >= 2 * static_cast<uint32_t>(sm_count())) {
    p.tokens_per_cta *= 2;
  }
  const int mode = rotary->interleaved ? kAdjacent : rotary->rotary_dim == D ? kHalves : kHalvesPartial;
  const unsigned grid = (n + p.tokens_per_cta - 1) / p.tokens_per_cta;
  const size_t smem = size_t{p.tokens_per_cta} * rotary->rotary_dim / 2 * sizeof(float2);
  void (*kernel)(const Params) = D == 64 ? kernel_for<64>(mode) : D == 128 ? kernel_for<128>(mode) : kernel_for<256>(mode);
  kernel<<<grid, kThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return cuda_status(cudaGetLastError());
}
