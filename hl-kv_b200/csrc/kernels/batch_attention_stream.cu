// Batch attention for few query rows (decode, a few proposed tokens): the cache is streamed once.
//
// The bound is memory: a token of a KV head is 512 (FP16), 264 (FP8) or 144 bytes (INT4) of K and V for
// heads of 128, read once, against 4 * 128 operations for each of at most 16 query rows.
//
// One CTA per SM takes an equal share of the batch's cost (the plan's per-block costs, in proportion
// to the bytes), whatever the sequences' lengths: its range of the line on which all (sequence, head
// group) units lie end to end.  A producer warp copies the blocks' codes and parameters as they are,
// by bulk copies, into a byte ring in shared memory: tiles of 16 tokens of a block, all heads of the
// group (up to 8) at once, so that a copy is one long piece of the slot; a ring of bytes, not of
// fixed stages, keeps as many INT4 bytes in flight as FP16 ones.  Consumer warps take one (tile, head)
// each and turn codes into binary16 matrix fragments in registers:
//   S^T = K Q^T (tokens x rows), a running softmax, O^T += V^T P^T.
// A code's binary16 value is exact (E4M3, E5M2, an INT4 code's integer), so the parameters stay out of
// the matrices: the K row's scale multiplies the score in binary32 and its bias enters as
// bias * sum(q); the V row's scale multiplies the weight, and its bias is summed apart in binary32.
// A weight is rounded once, to binary16 (2^-12 of it), after being scaled by 2^-E: E follows the
// exponents of the tiles' scales, so that weights stay in binary16's normal range whatever the values'
// size, and the accumulators are in units of 2^E.
// The order of contraction is free, so every lane takes contiguous bytes of a row and pairs them
// where they lie: K elements (j, j + 4) of each 8, V tokens (2q, 2q + 1).
#include <cmath>

#include "batch_attention.cuh"

namespace hlkv {
namespace battn {
namespace {

constexpr uint32_t kStages = 16;
constexpr uint32_t kTiles = 8;  // (tile, head) units of a stage: one per warp of a consumer group

struct Tile {
  uint32_t fn;   // format | tokens << 8 | scale mode << 16 | parameters in global memory << 24
  uint32_t pos;  // position of its first token
  uint32_t kc, vc;  // ring offsets of the K and V codes: [tokens][heads][row bytes]
  uint32_t kp, vp;  // ring offsets of the first row's parameters, or the two halves of the K row's address
  float ws, wb;     // block-wide parameters
};
enum : uint32_t { kFirst = 1, kLast = 2, kDone = 4, kDirect = 8 };
struct Stage {
  Tile tile[kTiles];
  uint32_t tiles, flags;
  uint32_t seq, head0, heads, unit_slot;
};

template <int kD, int kNB>
struct Config {
  static constexpr int kWarps = kNB == 1 ? 16 : 8;  // consumers: 56 to 100 registers a lane hold the state of 8 or 16 rows
  static constexpr int kGroups = kWarps / 8;
  static constexpr int kThreads = (kWarps + 1) * 32;
  static constexpr int kRowsPad = kD + 4;  // floats of a row in the merge buffer: outputs, max, sum
  static constexpr uint32_t kMergeBytes = kWarps * 8 * kNB * kRowsPad * 4;
  static constexpr uint32_t kRing = (226u * 1024u - kMergeBytes - static_cast<uint32_t>(sizeof(Stage)) * kStages - 1024u) / 128u * 128u;
  static constexpr uint32_t kSmem = kRing + kMergeBytes + sizeof(Stage) * kStages + 1024;
};

struct Shared {
  uint64_t full[kStages], empty[kStages], merged;
  uint32_t offset[kStages];  // ring offsets of the stages' data
  uint64_t warp_sum[17];
  uint64_t total, base;  // cost of the batch; of the sequences before `seq`
  uint32_t seq;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8x8 matrix of binary16 held two columns to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t m, uint32_t o) { return (a & m) | o; }
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

// Row bytes of a format.
template <int kD, uint32_t kF>
constexpr uint32_t kRow = kF == dev::kFp16 ? kD * 2 : kF == dev::kInt4 ? kD / 2 : kD;

// Four pairs (j, j + 4) of the 8 elements at `w`, as binary16 (INT4: the code times 2^-24, binary16's
// smallest step, so that masking a code is its conversion).
template <uint32_t kF>
__device__ __forceinline__ void k_pairs(const uint32_t* w, uint32_t (&a)[4]) {
  if constexpr (kF == dev::kFp16) {
    a[0] = __byte_perm(w[0], w[2], 0x5410);
    a[1] = __byte_perm(w[0], w[2], 0x7632);
    a[2] = __byte_perm(w[1], w[3], 0x5410);
    a[3] = __byte_perm(w[1], w[3], 0x7632);
  } else if constexpr (kF == dev::kInt4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (w[0] >> (4 * j)) & 0x000F000Fu;
  } else {
    const uint32_t x = __byte_perm(w[0], w[1], 0x5140), y = __byte_perm(w[0], w[1], 0x7362);
    a[0] = fp8_lo<kF>(x);
    a[1] = fp8_hi<kF>(x);
    a[2] = fp8_lo<kF>(y);
    a[3] = fp8_hi<kF>(y);
  }
}

// Words that 8 elements take.
template <uint32_t kF>
constexpr int kWords = kF == dev::kFp16 ? 4 : kF == dev::kInt4 ? 1 : 2;

// Eight elements of two tokens -> for each element the pair (token a, token b): FP16 as they are,
// E4M3 times 2^-8, E5M2 times 2^-15, INT4 (code - 8) / 8.  At these sizes a row's codes reach 0.5 to 1.75
// in every quantized format, and weight times row scale is about weight times row maximum.
template <uint32_t kF>
__device__ __forceinline__ void v_pairs(const uint32_t* a, const uint32_t* b, uint32_t (&v)[8]) {
  if constexpr (kF == dev::kFp16) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = __byte_perm(a[j], b[j], 0x5410);
      v[2 * j + 1] = __byte_perm(a[j], b[j], 0x7632);
    }
  } else if constexpr (kF == dev::kInt4) {
    // 1024 + c and 1024 + 16 c by masks, then (1024 + c) / 8 - 129 and (1024 + 16 c) / 128 - 9: exact.
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t x = __byte_perm(a[0], b[0], j == 0 ? 0x5410 : 0x7632), y = x >> 8;
      v[4 * j] = hfma2(lop_and_or(x, 0x000F000Fu, 0x64006400u), 0x30003000u, 0xD808D808u);
      v[4 * j + 1] = hfma2(lop_and_or(x, 0x00F000F0u, 0x64006400u), 0x20002000u, 0xC880C880u);
      v[4 * j + 2] = hfma2(lop_and_or(y, 0x000F000Fu, 0x64006400u), 0x30003000u, 0xD808D808u);
      v[4 * j + 3] = hfma2(lop_and_or(y, 0x00F000F0u, 0x64006400u), 0x20002000u, 0xC880C880u);
    }
  } else {
    constexpr uint32_t kDown = kF == dev::kE4M3 ? 0x1C001C00u : 0x02000200u;  // 2^-8, 2^-15
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t x = __byte_perm(a[j], b[j], 0x5140), y = __byte_perm(a[j], b[j], 0x7362);
      v[4 * j] = hmul2(fp8_lo<kF>(x), kDown);
      v[4 * j + 1] = hmul2(fp8_hi<kF>(x), kDown);
      v[4 * j + 2] = hmul2(fp8_lo<kF>(y), kDown);
      v[4 * j + 3] = hmul2(fp8_hi<kF>(y), kDown);
    }
  }
}
// The factors that k_pairs and v_pairs leave out.
template <uint32_t kF>
constexpr float kKeyUnit = kF == dev::kInt4 ? 0x1p24f : 1.0f;
template <uint32_t kF>
constexpr float kValueUnit = kF == dev::kFp16 ? 1.0f : kF == dev::kE4M3 ? 0x1p8f : kF == dev::kE5M2 ? 0x1p15f : 8.0f;

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// A warp's state for one (unit, head): lane (g, q) = (lane / 4, lane % 4) holds query columns 2q and
// 2q + 1 of each column block, and head elements [g kD/8, (g + 1) kD/8).
template <int kD, int kNB>
struct State {
  uint32_t q[kNB][kD / 16][2];  // Q^T fragments: column g, pairs (j, j + 4) of elements [quad kD/4, ...)
  float acc[kNB][kD / 16][4];   // [.][mt]: element 2 mt of columns 2q, 2q + 1, then element 2 mt + 1; units of 2^E
  float m[kNB][2], l[kNB][2], bias[kNB][2];  // l and bias: this lane's tokens only
  float qsum[kNB][2];
  int32_t pos[kNB][2];  // positions of the columns' tokens
  int E;
};
constexpr int kNoExponent = -1000;

template <int kD, int kNB>
__device__ __forceinline__ void begin_piece(const Params& p, State<kD, kNB>& s, Rows rows, uint32_t context, uint32_t head,
                                            uint32_t lane) {
  const uint32_t g = lane >> 2, quad = lane & 3;
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) {
    const uint32_t r = nb * 8 + g, tok = r / p.group, in_group = r % p.group;
    const bool live = r < rows.q * p.group;
    const uint4* src = reinterpret_cast<const uint4*>(p.q + (rows.first + (live ? tok : 0u)) * p.q_stride +
                                                      uint64_t{head * p.group + (live ? in_group : 0u)} * kD) +
                       quad * (kD / 32);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kD / 32; ++i) {
      const uint4 w = live ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
      uint32_t a[4];
      k_pairs<dev::kFp16>(x, a);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s.q[nb][2 * i + j / 2][j % 2] = a[j];
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[j]));
        sum += f.x + f.y;
      }
    }
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      s.qsum[nb][c] = __shfl_sync(0xFFFFFFFFu, sum, (quad * 2 + c) * 4) * p.qscale;
      s.pos[nb][c] = static_cast<int32_t>(context - rows.q + (nb * 8 + quad * 2 + c) / p.group);
      s.m[nb][c] = -INFINITY;
      s.l[nb][c] = s.bias[nb][c] = 0.0f;
    }
#pragma unroll
    for (int mt = 0; mt < kD / 16; ++mt) s.acc[nb][mt][0] = s.acc[nb][mt][1] = s.acc[nb][mt][2] = s.acc[nb][mt][3] = 0.0f;
  }
  s.E = kNoExponent;
}

// One tile (up to 16 tokens of one block and head).  `whole`: every row sees all its tokens.
template <int kD, int kNB, uint32_t kF>
__device__ __forceinline__ void tile_step(const Params& p, State<kD, kNB>& s, const uint8_t* kc, const uint8_t* vc,
                                          uint32_t token_bytes, float2 (&kp)[2], float2 (&vp)[2], uint32_t n, uint32_t tile_pos,
                                          bool whole, uint32_t lane) {
  const uint32_t g = lane >> 2, quad = lane & 3;
  constexpr int kW = kWords<kF>;
  // ---- scores
  float sc[kNB][4];
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) sc[nb][0] = sc[nb][1] = sc[nb][2] = sc[nb][3] = 0.0f;
  {
    constexpr int kG8 = kD / 32;                 // groups of 8 elements in a lane's quarter row
    constexpr uint32_t kBytes = kRow<kD, kF> / 4;  // of a quarter row: 8 to 64
    const uint8_t* r0 = kc + g * token_bytes + quad * kBytes;
    const uint8_t* r1 = r0 + 8 * token_bytes;
    constexpr int kPer = kF == dev::kFp16 ? 1 : kF == dev::kInt4 ? kG8 : 2;  // groups per load
#pragma unroll
    for (int i = 0; i < kG8; i += kPer) {
      uint32_t w0[kPer * kW], w1[kPer * kW];
      if constexpr (kPer * kW == 4) {
        *reinterpret_cast<uint4*>(w0) = *reinterpret_cast<const uint4*>(r0 + i * kW * 4);
        *reinterpret_cast<uint4*>(w1) = *reinterpret_cast<const uint4*>(r1 + i * kW * 4);
      } else {
        *reinterpret_cast<uint2*>(w0) = *reinterpret_cast<const uint2*>(r0 + i * kW * 4);
        *reinterpret_cast<uint2*>(w1) = *reinterpret_cast<const uint2*>(r1 + i * kW * 4);
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        uint32_t a[4], b[4];
        k_pairs<kF>(w0 + j * kW, a);
        k_pairs<kF>(w1 + j * kW, b);
#pragma unroll
        for (int nb = 0; nb < kNB; ++nb) {
          mma16816(sc[nb], a[0], b[0], a[1], b[1], s.q[nb][2 * (i + j)][0], s.q[nb][2 * (i + j)][1]);
          mma16816(sc[nb], a[2], b[2], a[3], b[3], s.q[nb][2 * (i + j) + 1][0], s.q[nb][2 * (i + j) + 1][1]);
        }
      }
    }
  }
  // ---- softmax; this lane: tokens g and g + 8 (t), columns 2 quad and 2 quad + 1 (c)
  float pr[kNB][4];
  const bool v0 = g < n, v1 = g + 8 < n;
  const float k0 = kp[0].x * (p.qscale * kKeyUnit<kF>), k1 = kp[1].x * (p.qscale * kKeyUnit<kF>);
  bool grow = false;
  float mx[kNB][2];
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x0 = sc[nb][c] * k0, x1 = sc[nb][2 + c] * k1;
      if constexpr (kF != dev::kFp16) {
        x0 = fmaf(kp[0].y, s.qsum[nb][c], x0);
        x1 = fmaf(kp[1].y, s.qsum[nb][c], x1);
      }
      bool s0 = v0, s1 = v1;
      if (!whole) {
        const int32_t d0 = s.pos[nb][c] - static_cast<int32_t>(tile_pos + g), d1 = d0 - 8;
        s0 = s0 && d0 >= 0 && (p.window == 0 || static_cast<uint32_t>(d0) < p.window || tile_pos + g < p.sinks);
        s1 = s1 && d1 >= 0 && (p.window == 0 || static_cast<uint32_t>(d1) < p.window || tile_pos + g + 8 < p.sinks);
      }
      pr[nb][c] = s0 ? x0 : -INFINITY;
      pr[nb][2 + c] = s1 ? x1 : -INFINITY;
      float v = fmaxf(pr[nb][c], pr[nb][2 + c]);
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
      mx[nb][c] = v;
      grow = grow || v > s.m[nb][c] + 8.0f;
    }
  }
  // The reference maximum moves only when a score passes it by 8: weights reach 2^8 at most.
  if (__any_sync(0xFFFFFFFFu, grow)) {
#pragma unroll
    for (int nb = 0; nb < kNB; ++nb) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float mn = fmaxf(s.m[nb][c], mx[nb][c]);
        const float a = mn == -INFINITY ? 1.0f : exp2f(s.m[nb][c] - mn);
        s.m[nb][c] = mn;
        s.l[nb][c] *= a;
        s.bias[nb][c] *= a;
#pragma unroll
        for (int mt = 0; mt < kD / 16; ++mt) {
          s.acc[nb][mt][c] *= a;
          s.acc[nb][mt][2 + c] *= a;
        }
      }
    }
  }
  // ---- the tile's exponent: of the largest finite value scale among its tokens
  const float u0 = v0 ? vp[0].x * kValueUnit<kF> : 0.0f, u1 = v1 ? vp[1].x * kValueUnit<kF> : 0.0f;
  const uint32_t b0 = __float_as_uint(u0) & 0x7FFFFFFFu, b1 = __float_as_uint(u1) & 0x7FFFFFFFu;
  const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, max(b0 < 0x7F800000u ? b0 : 0u, b1 < 0x7F800000u ? b1 : 0u));
  // (scales beyond 2^60 or below 2^-60 are taken as those)
  const int e = min(max(static_cast<int>(top >> 23) - 127, -60), 60);
  if (e > s.E + 6 || (e < s.E - 6 && top != 0)) {
    if (s.E != kNoExponent) {
      const float f = exp2f(static_cast<float>(s.E - e));
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb) {
#pragma unroll
        for (int mt = 0; mt < kD / 16; ++mt) {
#pragma unroll
          for (int k = 0; k < 4; ++k) s.acc[nb][mt][k] *= f;
        }
      }
    }
    s.E = e;
  }
  const float down = pow2(-s.E), f0 = u0 * down, f1 = u1 * down;
  const float beta0 = kF == dev::kInt4 ? fmaf(8.0f, vp[0].x, vp[0].y) : vp[0].y;
  const float beta1 = kF == dev::kInt4 ? fmaf(8.0f, vp[1].x, vp[1].y) : vp[1].y;
  uint32_t pb[kNB][2];
#pragma unroll
  for (int nb = 0; nb < kNB; ++nb) {
    float w[4];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float ref = s.m[nb][c] == -INFINITY ? 0.0f : s.m[nb][c];
      const float p0 = exp2f(pr[nb][c] - ref), p1 = exp2f(pr[nb][2 + c] - ref);
      pr[nb][c] = p0;
      pr[nb][2 + c] = p1;
      s.l[nb][c] += p0 + p1;
      // a hidden token's weight is 0 whatever its parameters hold
      w[c] = p0 == 0.0f ? 0.0f : p0 * f0;
      w[2 + c] = p1 == 0.0f ? 0.0f : p1 * f1;
      if constexpr (kF != dev::kFp16) {
        s.bias[nb][c] += (p0 == 0.0f ? 0.0f : p0 * beta0) + (p1 == 0.0f ? 0.0f : p1 * beta1);
      }
    }
    pb[nb][0] = transpose8(dev::pack_f16x2(w[0], w[1]));
    pb[nb][1] = transpose8(dev::pack_f16x2(w[2], w[3]));
  }
  // ---- values; this lane: tokens 2 quad, 2 quad + 1, 2 quad + 8, 2 quad + 9
  // In a tile that some row sees in part, a value that is not finite, or a scale far above the others',
  // must not touch the rows that do not see it: such a tile is taken row by row.
  bool apart = false;
  if (!whole && n > 0) {
    const uint32_t low0 = v0 ? b0 : 0xFFFFFFFFu, low1 = v1 ? b1 : 0xFFFFFFFFu;
    const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, min(low0, low1));
    apart = __any_sync(0xFFFFFFFFu, (v0 && b0 >= 0x7F800000u) || (v1 && b1 >= 0x7F800000u)) || top > low + (8u << 23);
  }
#pragma unroll
  for (int i = 0; i < kD / 64; ++i) {
    uint32_t lo[8], hi[8];
    {
      uint32_t w[4][kW];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t tok = 2 * quad + (t & 1) + (t & 2) * 4;
        const uint8_t* r = vc + tok * token_bytes + g * (kRow<kD, kF> / 8) + i * kW * 4;
        if constexpr (kW == 4) *reinterpret_cast<uint4*>(w[t]) = *reinterpret_cast<const uint4*>(r);
        else if constexpr (kW == 2) *reinterpret_cast<uint2*>(w[t]) = *reinterpret_cast<const uint2*>(r);
        else w[t][0] = *reinterpret_cast<const uint32_t*>(r);
        if (tok >= n) {
#pragma unroll
          for (int k = 0; k < kW; ++k) w[t][k] = 0u;
        }
      }
      v_pairs<kF>(w[0], w[1], lo);
      v_pairs<kF>(w[2], w[3], hi);
    }
    if (!whole) {
      bool bad = false;
#pragma unroll
      for (int k = 0; k < 8; ++k) bad = bad || has_nonfinite(lo[k]) || has_nonfinite(hi[k]);
      if (__any_sync(0xFFFFFFFFu, bad) || apart) {
#pragma unroll 1
        for (int col = 0; col < 8 * kNB; ++col) {
          // this row's view of the 16 tokens, and the exponent of the scales that it sees
          const int32_t at = __shfl_sync(0xFFFFFFFFu, kNB == 1 || col < 8 ? ((col & 1) ? s.pos[0][1] : s.pos[0][0])
                                                                         : ((col & 1) ? s.pos[kNB - 1][1] : s.pos[kNB - 1][0]),
                                         (col & 7) >> 1);
          auto sees = [&](uint32_t tok) {
            const int32_t d = at - static_cast<int32_t>(tile_pos + tok);
            return tok < n && d >= 0 && (p.window == 0 || static_cast<uint32_t>(d) < p.window || tile_pos + tok < p.sinks);
          };
          const uint32_t mine = __reduce_max_sync(0xFFFFFFFFu, max(sees(g) && b0 < 0x7F800000u ? b0 : 0u,
                                                                  sees(g + 8) && b1 < 0x7F800000u ? b1 : 0u));
          const int ec = min(max(static_cast<int>(mine >> 23) - 127, -60), 60);
          const float dc = pow2(-ec), up = exp2f(static_cast<float>(ec - s.E));
          const int nb = col >> 3;
          float w[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float p0 = nb == 0 ? pr[0][c] : pr[kNB - 1][c], p1 = nb == 0 ? pr[0][2 + c] : pr[kNB - 1][2 + c];
            w[c] = p0 == 0.0f ? 0.0f : p0 * (u0 * dc);
            w[2 + c] = p1 == 0.0f ? 0.0f : p1 * (u1 * dc);
          }
          const uint32_t x0 = transpose8(dev::pack_f16x2(w[0], w[1])), x1 = transpose8(dev::pack_f16x2(w[2], w[3]));
          const uint32_t keep_lo = (sees(2 * quad) ? 0xFFFFu : 0u) | (sees(2 * quad + 1) ? 0xFFFF0000u : 0u);
          const uint32_t keep_hi = (sees(2 * quad + 8) ? 0xFFFFu : 0u) | (sees(2 * quad + 9) ? 0xFFFF0000u : 0u);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma16816(t, lo[2 * k] & keep_lo, lo[2 * k + 1] & keep_lo, hi[2 * k] & keep_hi, hi[2 * k + 1] & keep_hi, x0, x1);
#pragma unroll
            for (int b = 0; b < kNB; ++b) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (static_cast<int>(b * 8 + quad * 2 + c) == col) {
                  s.acc[b][4 * i + k][c] = fmaf(t[c], up, s.acc[b][4 * i + k][c]);
                  s.acc[b][4 * i + k][2 + c] = fmaf(t[2 + c], up, s.acc[b][4 * i + k][2 + c]);
                }
              }
            }
          }
        }
        continue;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb) {
        mma16816(s.acc[nb][4 * i + k], lo[2 * k], lo[2 * k + 1], hi[2 * k], hi[2 * k + 1], pb[nb][0], pb[nb][1]);
      }
    }
  }
}

// ---- the producer warp -------------------------------------------------------------------------
template <int kD, int kNB>
struct Producer {
  using C = Config<kD, kNB>;
  const Params& p;
  Shared& sh;
  Stage* stages;
  uint8_t* ring;
  uint32_t lane;
  uint32_t st = 0, oldest = 0, head = 0;
  bool ok = true;

  __device__ __forceinline__ bool pop() {
    ok = ok && mbar_wait(&sh.empty[oldest % kStages], (oldest / kStages) & 1);
    ++oldest;
    return ok;
  }

  // Space for `bytes` (a multiple of 16) in the ring, in stage order.
  __device__ __forceinline__ uint32_t reserve(uint32_t bytes) {
    if (st - oldest == kStages) pop();
    uint32_t at = head;
    if (head + bytes > C::kRing) {
      at = 0;
      while (oldest != st && ok) {
        const uint32_t o = sh.offset[oldest % kStages];
        if (!(o >= head || o < bytes)) break;
        pop();
      }
    } else {
      while (oldest != st && ok) {
        const uint32_t o = sh.offset[oldest % kStages];
        if (!(o >= at && o < at + bytes)) break;
        pop();
      }
    }
    if (oldest == st) at = 0;  // empty: start over
    head = at + bytes;
    return at;
  }

  // One stage: lanes < tiles hold a tile each (payload, its descriptor fields and tokens [t0, t0 + n)).
  __device__ __forceinline__ void emit(uint32_t tiles, uint32_t flags, uint32_t seq, uint32_t head0, uint32_t heads, uint32_t slot,
                                       const uint8_t* payload, uint32_t f, uint32_t mode, uint32_t sref, uint32_t t0, uint32_t n,
                                       uint32_t pos) {
    const bool mine = lane < tiles;
    const bool packed = heads == p.H;  // all heads of a token: a tile is one piece of the slot
    const uint32_t rb = f == dev::kFp16 ? kD * 2 : f == dev::kInt4 ? kD / 2 : kD, pb = f == dev::kInt4 ? 8 : 4;
    const bool params = mine && f != dev::kFp16 && mode == 0;
    const uint32_t codes = mine ? n * heads * rb : 0u;
    uint64_t ka = 0, va = 0;  // byte addresses of the first row's parameters
    uint32_t kn = 0, vn = 0;  // bytes copied of them
    if (params) {
      ka = p.code_bytes[f] + uint64_t{t0 * p.H + head0} * pb;
      va = ka + uint64_t{p.T} * p.H * pb;
      if (packed) {
        const uint32_t len = n * p.H * pb;
        kn = static_cast<uint32_t>(((ka + len + 15) & ~uint64_t{15}) - (ka & ~uint64_t{15}));
        vn = static_cast<uint32_t>(((va + len + 15) & ~uint64_t{15}) - (va & ~uint64_t{15}));
      }
    }
    const uint32_t bytes = 2 * codes + kn + vn;
    uint32_t off = bytes;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, off, o);
      if (lane >= static_cast<uint32_t>(o)) off += x;
    }
    const uint32_t total = __shfl_sync(0xFFFFFFFFu, off, 7);  // lanes from `tiles` on add nothing
    off -= bytes;
    const uint32_t at = reserve(total);
    const uint32_t slot_i = st % kStages;
    Stage& m = stages[slot_i];
    off += at;
    if (mine) {
      Tile t;
      t.fn = f | n << 8 | mode << 16 | (params && !packed ? 1u << 24 : 0u);
      t.pos = pos;
      t.kc = off;
      t.vc = off + codes;
      if (packed) {
        t.kp = off + 2 * codes + static_cast<uint32_t>(ka & 15);
        t.vp = off + 2 * codes + kn + static_cast<uint32_t>(va & 15);
      } else {
        const uint64_t a = reinterpret_cast<uint64_t>(payload) + ka;
        t.kp = static_cast<uint32_t>(a);
        t.vp = static_cast<uint32_t>(a >> 32);
      }
      const float2 w = mode != 0 ? dev::block_params_value(mode, sref) : make_float2(1.0f, 0.0f);
      t.ws = w.x;
      t.wb = w.y;
      m.tile[lane] = t;
    }
    if (lane == 0) {
      m.tiles = tiles;
      m.flags = flags;
      m.seq = seq;
      m.head0 = head0;
      m.heads = heads;
      m.unit_slot = slot;
      sh.offset[slot_i] = at;
    }
    __syncwarp();
    ++st;
    if (!ok) return;  // gave up: nothing more is copied, and the consumers give up as well
    uint64_t* bar = &sh.full[slot_i];
    if (lane == 0) mbar_arrive_expect(bar, total);
    __syncwarp();
    if (packed) {
      if (mine) {
        const uint64_t row = uint64_t{t0} * heads * rb;
        bulk_load(ring + off, payload + row, codes, bar);
        bulk_load(ring + off + codes, payload + uint64_t{p.T} * heads * rb + row, codes, bar);
        if (kn) bulk_load(ring + off + 2 * codes, payload + (ka & ~uint64_t{15}), kn, bar);
        if (vn) bulk_load(ring + off + 2 * codes + kn, payload + (va & ~uint64_t{15}), vn, bar);
      }
    } else {
      for (uint32_t t = 0; t < tiles; ++t) {  // a copy per token and kind: its heads lie together
        const uint64_t base = __shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(payload), t);
        const uint32_t nt = __shfl_sync(0xFFFFFFFFu, n, t), tt = __shfl_sync(0xFFFFFFFFu, t0, t);
        const uint32_t r = __shfl_sync(0xFFFFFFFFu, rb, t), o = __shfl_sync(0xFFFFFFFFu, off, t);
        const uint32_t i = lane & 15, kv = lane >> 4;
        if (i < nt) {
          bulk_load(ring + o + (kv * nt + i) * heads * r,
                    reinterpret_cast<const uint8_t*>(base) + (uint64_t{kv * p.T + tt + i} * p.H + head0) * r, heads * r, bar);
        }
      }
    }
  }

  // First k in [0, count) with cost[k] >= target (count if none).
  __device__ __forceinline__ uint32_t find(const uint32_t* cost, uint32_t count, uint32_t target) {
    uint32_t a = 0, b = count;
    while (b - a > 0) {
      const uint32_t step = (b - a + 31) / 32, k = a + lane * step;
      const uint32_t last = min(k + step, b) - 1;  // lanes past the end repeat the last
      const bool hit = k < b ? __ldg(cost + last) >= target : true;
      const uint32_t first = __ffs(__ballot_sync(0xFFFFFFFFu, hit));
      if (first == 0) return b;  // no lane: b - a <= 32 step, all below
      const uint32_t lo = a + (first - 1) * step;
      if (lo >= b) return b;
      b = min(lo + step, b);
      a = lo;
      if (step == 1) return lo;
    }
    return a;
  }

  __device__ __forceinline__ void run() {
    const uint64_t W = sh.total, x0 = blockIdx.x * W / gridDim.x, x1 = (uint64_t{blockIdx.x} + 1) * W / gridDim.x;
    uint64_t base = sh.base;  // of sequence i's units
    for (uint32_t i = sh.seq; i < p.nseq && base < x1 && ok; ++i) {
      const Rows rows = rows_of(p, i);
      uint32_t w = p.cost[i];
      if (rows.q == 0 || uint64_t{rows.q} * p.group > kStreamRows) w = 0;
      if (w == 0) continue;
      uint32_t first;
      const uint32_t count = count_of(p, i, &first);
      uint32_t hg = x0 > base ? static_cast<uint32_t>((x0 - base) / w) : 0u;
      for (; hg < p.head_groups && ok; ++hg) {
        const uint64_t ub = base + uint64_t{hg} * w;
        if (ub >= x1) break;
        const uint32_t lo = x0 > ub ? static_cast<uint32_t>(x0 - ub) : 0u;
        const uint32_t hi = x1 - ub < w ? static_cast<uint32_t>(x1 - ub) : w;
        piece(i, hg, lo, hi, w, first, count);
      }
      base += uint64_t{p.head_groups} * w;
    }
    for (int k = 0; k < C::kGroups && ok; ++k) emit(0, kDone, 0, 0, p.H, 0, nullptr, 0, 0, 0, 0, 0, 0);
  }

  // The blocks of unit (i, hg) whose cost begins in [lo, hi).
  __device__ __forceinline__ void piece(uint32_t i, uint32_t hg, uint32_t lo, uint32_t hi, uint32_t w, uint32_t first,
                                        uint32_t count) {
    const uint32_t head0 = hg * 8, heads = min(8u, p.H - head0), per_stage = kTiles / heads;
    const uint32_t slot = blockIdx.x + i * p.head_groups + hg;
    const uint32_t direct = lo == 0 && hi == w ? kDirect : 0u;
    const uint32_t* cost = p.block_cost + first;
    uint32_t j0 = lo == 0 ? 0u : find(cost, count, lo) + 1;
    // Stages alternate between the consumer groups.  The first stage of each carries kFirst; at the end
    // every group gets a stage without tiles that carries kLast, after as many empty ones as bring the
    // piece to a multiple of kGroups.
    const uint32_t flags = kFirst | direct;
    uint32_t done = 0;
    bool more = true;
    while (more && ok) {
      const uint32_t j = j0 + lane;
      uint4 b = make_uint4(0u, 0u, 0u, 0u);
      const uint8_t* payload = nullptr;
      uint32_t f = 4, v = 0;
      bool inside = false;
      if (j < count) {
        const uint32_t start = j > 0 ? __ldg(cost + j - 1) : 0u;
        inside = start < hi;
        if (inside) {
          b = __ldg(p.blocks + first + j);
          f = open_block(p, b, &payload);
          if (f <= 3) v = min((b.y >> 10) & 0x3FFu, p.T);
        }
      }
      more = __all_sync(0xFFFFFFFFu, inside);  // else the piece ends in this batch
      uint32_t nt = (v + 15) / 16, upto = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= static_cast<uint32_t>(o)) upto += x;
      }
      const uint32_t total = __shfl_sync(0xFFFFFFFFu, upto, 31);
      const uint32_t ps = static_cast<uint32_t>(reinterpret_cast<uint64_t>(payload)),
                     pt = static_cast<uint32_t>(reinterpret_cast<uint64_t>(payload) >> 32);
      for (uint32_t t = 0; t < total && ok; t += per_stage) {
        // lane k of the stage: tile t + k, in the first block whose running count passes it
        const uint32_t k = t + lane;
        const uint32_t tiles = min(per_stage, total - t);
        uint32_t at = 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint32_t x = __shfl_sync(0xFFFFFFFFu, upto, at + o - 1);
          if (x <= k) at += o;
        }
        at = min(at, 31u);
        const uint32_t before = __shfl_sync(0xFFFFFFFFu, upto - nt, at);
        const uint32_t tf = __shfl_sync(0xFFFFFFFFu, f, at), tv = __shfl_sync(0xFFFFFFFFu, v, at);
        const uint32_t ti = __shfl_sync(0xFFFFFFFFu, b.y, at), tr = __shfl_sync(0xFFFFFFFFu, b.z, at);
        const uint32_t tw = __shfl_sync(0xFFFFFFFFu, b.w, at);
        const uint64_t pl = __shfl_sync(0xFFFFFFFFu, ps, at) | uint64_t{__shfl_sync(0xFFFFFFFFu, pt, at)} << 32;
        const uint32_t t0 = lane < tiles ? (k - before) * 16 : 0u;
        const uint32_t n = lane < tiles ? min(16u, tv - t0) : 0u;
        emit(tiles, done < C::kGroups ? flags : direct, i, head0, heads, slot, reinterpret_cast<const uint8_t*>(pl), tf, tf == dev::kFp16 ? 0u : (ti >> 4) & 3u, tr,
             t0, n, tw + t0);
        ++done;
      }
      j0 += 32;
    }
    // Closing stages, one per group, without tiles.
    const uint32_t fill = (C::kGroups - done % C::kGroups) % C::kGroups + C::kGroups;
    for (uint32_t k = 0; k < fill && ok; ++k) {
      const uint32_t fl = (done < C::kGroups ? flags : direct) | (k + C::kGroups >= fill ? kLast : 0u);
      emit(0, fl, i, head0, heads, slot, nullptr, 0, 0, 0, 0, 0, 0);
      ++done;
    }
  }
};

template <int kD, int kNB>
__global__ void __launch_bounds__(Config<kD, kNB>::kThreads, 1) stream_kernel(const __grid_constant__ Params p) {
  using C = Config<kD, kNB>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem + C::kRing);
  Stage* stages = reinterpret_cast<Stage*>(smem + C::kRing + C::kMergeBytes);
  __shared__ Shared sh;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 8);
    }
    mbar_init(&sh.merged, C::kWarps);
    mbar_fence_init();
  }
  // ---- where this CTA's share begins: the costs of the sequences, added up in chunks of consecutive ones
  {
    const uint32_t chunk = (p.nseq + C::kThreads - 1) / C::kThreads;
    const uint32_t a = min(threadIdx.x * chunk, p.nseq), b = min(a + chunk, p.nseq);
    auto cost_of = [&](uint32_t i) -> uint64_t {
      const Rows rows = rows_of(p, i);
      return rows.q == 0 || uint64_t{rows.q} * p.group > kStreamRows ? 0u : p.cost[i];
    };
    uint64_t sum = 0;
    for (uint32_t i = a; i < b; ++i) sum += cost_of(i);
    uint64_t upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += x;
    }
    if (lane == 31) sh.warp_sum[warp] = upto;
    if (threadIdx.x == 0) {
      sh.seq = p.nseq;
      sh.base = 0;
    }
    __syncthreads();
    uint64_t total = 0;
    for (uint32_t w = 0; w <= C::kWarps; ++w) {
      if (w < warp) upto += sh.warp_sum[w];
      total += sh.warp_sum[w];
    }
    const uint64_t W = total * p.head_groups, x0 = blockIdx.x * W / gridDim.x;
    uint64_t at = upto - sum;
    if (blockIdx.x == 0) {  // the merge finds its units by these
      for (uint32_t i = a; i < b; ++i) {
        p.prefix[i] = at;
        at += cost_of(i);
      }
      if (threadIdx.x == 0) p.prefix[p.nseq] = total;
      at = upto - sum;
    }
    if (threadIdx.x == 0) sh.total = W;
    if (sum > 0 && at * p.head_groups <= x0 && x0 < upto * p.head_groups) {
      uint32_t i = a;
      for (uint64_t c; i < b && (at + (c = cost_of(i))) * p.head_groups <= x0; ++i) at += c;
      sh.seq = i;
      sh.base = at * p.head_groups;
    }
    __syncthreads();
  }

  if (warp == C::kWarps) {
    Producer<kD, kNB> producer{p, sh, stages, ring, lane};
    producer.run();
    if (!producer.ok && lane == 0) atomicOr(p.err, dev::kErrInternal);
    return;
  }

  // ---- consumers
  const uint32_t group = warp / 8, w8 = warp % 8;
  State<kD, kNB> s;
  uint32_t heads = 1, tile_i = 0, head_i = 0, head0 = 0, slot = 0;
  int32_t pos0 = 0;
  Rows rows{0, 0};
  uint32_t meets = 0;
  // All consumer warps, with a limit as every wait.
  auto meet = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.merged);
    return mbar_wait(&sh.merged, meets++ & 1);
  };
  for (uint32_t st = group;; st += C::kGroups) {
    const uint32_t si = st % kStages;
    if (!mbar_wait(&sh.full[si], (st / kStages) & 1)) {
      if (lane == 0) atomicOr(p.err, dev::kErrInternal);
      break;
    }
    const Stage& m = stages[si];
    const uint32_t flags = m.flags;
    if (flags & kDone) break;
    if (flags & kFirst) {
      heads = m.heads;
      head0 = m.head0;
      slot = m.unit_slot;
      tile_i = w8 / heads;
      head_i = w8 % heads;
      rows = rows_of(p, m.seq);
      const uint32_t context = p.context[m.seq];
      pos0 = static_cast<int32_t>(context - rows.q);
      begin_piece<kD, kNB>(p, s, rows, context, head0 + head_i, lane);
    }
    if (tile_i < m.tiles) {
      const Tile& t = m.tile[tile_i];
      const uint32_t fn = t.fn, f = fn & 0xFFu, n = (fn >> 8) & 0xFFu, mode = (fn >> 16) & 0xFFu, tile_pos = t.pos;
      const uint32_t rb = f == dev::kFp16 ? kD * 2 : f == dev::kInt4 ? kD / 2 : kD;
      const uint32_t token_bytes = heads * rb;
      const uint8_t* kc = ring + t.kc + head_i * rb;
      const uint8_t* vc = ring + t.vc + head_i * rb;
      float2 kp[2], vp[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t tok = (lane >> 2) + 8 * h;
        kp[h] = vp[h] = make_float2(t.ws, t.wb);
        if (f != dev::kFp16 && mode == 0 && tok < n) {
          if (fn >> 24) {
            const uint8_t* a = reinterpret_cast<const uint8_t*>(uint64_t{t.kp} | uint64_t{t.vp} << 32);
            const uint64_t row = uint64_t{tok} * p.H + head_i, up = uint64_t{p.T} * p.H;
            if (f == dev::kInt4) {
              kp[h] = __ldg(reinterpret_cast<const float2*>(a) + row);
              vp[h] = __ldg(reinterpret_cast<const float2*>(a) + row + up);
            } else {
              kp[h] = make_float2(__ldg(reinterpret_cast<const float*>(a) + row), 0.0f);
              vp[h] = make_float2(__ldg(reinterpret_cast<const float*>(a) + row + up), 0.0f);
            }
          } else {
            const uint32_t row = tok * heads + head_i;
            if (f == dev::kInt4) {
              kp[h] = reinterpret_cast<const float2*>(ring + t.kp)[row];
              vp[h] = reinterpret_cast<const float2*>(ring + t.vp)[row];
            } else {
              kp[h] = make_float2(reinterpret_cast<const float*>(ring + t.kp)[row], 0.0f);
              vp[h] = make_float2(reinterpret_cast<const float*>(ring + t.vp)[row], 0.0f);
            }
          }
        }
      }
      const int32_t tp = static_cast<int32_t>(tile_pos), last = pos0 + static_cast<int32_t>(rows.q) - 1;
      const bool whole = tp + static_cast<int32_t>(n) - 1 <= pos0 &&
                         (p.window == 0 || static_cast<uint32_t>(last - tp) < p.window || tile_pos + n <= p.sinks);
      switch (f) {
        case dev::kFp16: tile_step<kD, kNB, dev::kFp16>(p, s, kc, vc, token_bytes, kp, vp, n, tile_pos, whole, lane); break;
        case dev::kE4M3: tile_step<kD, kNB, dev::kE4M3>(p, s, kc, vc, token_bytes, kp, vp, n, tile_pos, whole, lane); break;
        case dev::kE5M2: tile_step<kD, kNB, dev::kE5M2>(p, s, kc, vc, token_bytes, kp, vp, n, tile_pos, whole, lane); break;
        default: tile_step<kD, kNB, dev::kInt4>(p, s, kc, vc, token_bytes, kp, vp, n, tile_pos, whole, lane); break;
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[si]);

    if (flags & kLast) {
      // ---- merge the warps of each head: outputs, max and sum of every row
      const uint32_t g = lane >> 2, quad = lane & 3;
      const float unit = s.E == kNoExponent ? 0.0f : exp2f(static_cast<float>(s.E));
#pragma unroll
      for (int nb = 0; nb < kNB; ++nb) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float l = s.l[nb][c], b = s.bias[nb][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
            b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
          }
          float* row = merge + (warp * 8 * kNB + nb * 8 + quad * 2 + c) * C::kRowsPad;
#pragma unroll
          for (int mt = 0; mt < kD / 16; ++mt) {
            *reinterpret_cast<float2*>(row + g * (kD / 8) + 2 * mt) =
                make_float2(fmaf(s.acc[nb][mt][c], unit, b), fmaf(s.acc[nb][mt][2 + c], unit, b));
          }
          if (g == 0) *reinterpret_cast<float2*>(row + kD) = make_float2(s.m[nb][c], l);
        }
      }
      if (!meet()) {
        if (lane == 0) atomicOr(p.err, dev::kErrInternal);
        break;
      }
      const uint32_t n_rows = rows.q * p.group, n_tiles = kTiles / heads;
      for (uint32_t i = threadIdx.x; i < heads * n_rows * (kD / 4); i += C::kWarps * 32) {
        const uint32_t e = i % (kD / 4), r = (i / (kD / 4)) % n_rows, h = i / (kD / 4) / n_rows;
        float M = -INFINITY, L = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int gr = 0; gr < C::kGroups; ++gr) {
          for (uint32_t t = 0; t < n_tiles; ++t) {
            M = fmaxf(M, merge[((gr * 8 + t * heads + h) * 8 * kNB + r) * C::kRowsPad + kD]);
          }
        }
        for (int gr = 0; gr < C::kGroups; ++gr) {
          for (uint32_t t = 0; t < n_tiles; ++t) {
            const float* row = merge + ((gr * 8 + t * heads + h) * 8 * kNB + r) * C::kRowsPad;
            const float2 ml = *reinterpret_cast<const float2*>(row + kD);
            const float a = M == -INFINITY ? 1.0f : exp2f(ml.x - M);
            const float4 x = *reinterpret_cast<const float4*>(row + 4 * e);
            L = fmaf(ml.y, a, L);
            o.x = fmaf(x.x, a, o.x);
            o.y = fmaf(x.y, a, o.y);
            o.z = fmaf(x.z, a, o.z);
            o.w = fmaf(x.w, a, o.w);
          }
        }
        if (flags & kDirect) {
          if (L == 0.0f && M == -INFINITY) L = 1.0f;  // sees nothing: zeros
          const uint32_t tok = r / p.group, gi = r % p.group;
          *reinterpret_cast<uint2*>(p.out + (rows.first + tok) * p.out_stride + uint64_t{(head0 + h) * p.group + gi} * kD + 4 * e) =
              make_uint2(dev::pack_f16x2(o.x / L, o.y / L), dev::pack_f16x2(o.z / L, o.w / L));
        } else {
          float* dst = p.partial + ((uint64_t{slot} * 8 + h) * p.slot_rows + r) * C::kRowsPad;
          *reinterpret_cast<float4*>(dst + 4 * e) = o;
          if (e == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(M, L);
        }
      }
      if (!meet()) {  // the buffer is written again
        if (lane == 0) atomicOr(p.err, dev::kErrInternal);
        break;
      }
    }
  }
}

// Joins the partial results of the units that several CTAs took: one CTA of kD / 4 threads x rows per
// (sequence, head).  Also writes the zeros of rows whose sequence lists no block.
template <int kD>
__global__ void __launch_bounds__(128) merge_kernel(const __grid_constant__ Params p) {
  constexpr int kPad = kD + 4, kLanes = kD / 4, kRows = 128 / kLanes;
  const uint32_t i = blockIdx.x / p.H, head = blockIdx.x % p.H, hg = head / 8, h = head % 8;
  const Rows rows = rows_of(p, i);
  const uint32_t n_rows = rows.q * p.group;
  if (n_rows == 0 || uint64_t{rows.q} * p.group > kStreamRows) return;
  const uint32_t e = threadIdx.x % kLanes;
  const uint64_t W = p.prefix[p.nseq] * p.head_groups, w = p.prefix[i + 1] - p.prefix[i];
  uint32_t c0 = 0, c1 = 0;
  if (w > 0) {
    const uint64_t a = p.prefix[i] * p.head_groups + hg * w, b = a + w - 1;
    // CTA c takes [c W / G, (c + 1) W / G): the one that holds x is the largest c with c W / G <= x
    c0 = static_cast<uint32_t>(((a + 1) * p.ctas - 1) / W);
    c1 = static_cast<uint32_t>(((b + 1) * p.ctas - 1) / W);
    if (c0 == c1) return;  // one CTA had it all and wrote the rows
  }
  const uint64_t unit = uint64_t{i} * p.head_groups + hg;
  for (uint32_t r = threadIdx.x / kLanes; r < n_rows; r += kRows) {
    float M = -INFINITY, L = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (w > 0) {
      const float* base = p.partial + ((c0 + unit) * 8 + h) * p.slot_rows * kPad + uint64_t{r} * kPad;
      const uint64_t step = uint64_t{8} * p.slot_rows * kPad;
      // a CTA whose range is empty (more CTAs than cost) took nothing and wrote nothing
      auto empty = [&](uint32_t c) { return p.ctas > W && c * W / p.ctas == (uint64_t{c} + 1) * W / p.ctas; };
#pragma unroll 4
      for (uint32_t c = c0; c <= c1; ++c) {
        if (!empty(c)) M = fmaxf(M, base[(c - c0) * step + kD]);
      }
#pragma unroll 4
      for (uint32_t c = c0; c <= c1; ++c) {
        if (empty(c)) continue;
        const float* s = base + (c - c0) * step;
        const float2 ml = *reinterpret_cast<const float2*>(s + kD);
        const float4 x = *reinterpret_cast<const float4*>(s + 4 * e);
        const float a = M == -INFINITY ? 1.0f : exp2f(ml.x - M);
        L = fmaf(ml.y, a, L);
        o.x = fmaf(x.x, a, o.x);
        o.y = fmaf(x.y, a, o.y);
        o.z = fmaf(x.z, a, o.z);
        o.w = fmaf(x.w, a, o.w);
      }
    }
    if (L == 0.0f && M == -INFINITY) L = 1.0f;
    const uint32_t tok = r / p.group, gi = r % p.group;
    *reinterpret_cast<uint2*>(p.out + (rows.first + tok) * p.out_stride + uint64_t{head * p.group + gi} * kD + 4 * e) =
        make_uint2(dev::pack_f16x2(o.x / L, o.y / L), dev::pack_f16x2(o.z / L, o.w / L));
  }
}

template <int kD, int kNB>
cudaError_t launch(const Params& p, cudaStream_t s) {
  using C = Config<kD, kNB>;
  const cudaError_t e = cudaFuncSetAttribute(stream_kernel<kD, kNB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(C::kSmem));
  if (e != cudaSuccess) return e;
  stream_kernel<kD, kNB><<<p.ctas, C::kThreads, C::kSmem, s>>>(p);
  const cudaError_t e2 = cudaGetLastError();
  if (e2 != cudaSuccess) return e2;
  merge_kernel<kD><<<p.nseq * p.H, 128, 0, s>>>(p);
  return cudaGetLastError();
}

uint64_t prefix_bytes(uint32_t nseq) { return ((uint64_t{nseq} + 1) * 8 + 15) / 16 * 16; }

}  // namespace

size_t stream_workspace(uint32_t nseq, uint32_t H, uint32_t head_dim, uint32_t max_rows, uint32_t ctas) {
  const uint64_t rows = max_rows < kStreamRows ? max_rows : kStreamRows, groups = (H + 7) / 8;
  return static_cast<size_t>(prefix_bytes(nseq) + (ctas + nseq * groups) * 8 * rows * (head_dim + 4) * sizeof(float));
}

void stream_layout(Params* p, void* ws) {
  p->prefix = static_cast<uint64_t*>(ws);
  p->partial = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + prefix_bytes(p->nseq));
  p->slot_rows = p->max_rows < kStreamRows ? p->max_rows : kStreamRows;
  p->head_groups = (p->H + 7) / 8;
}

cudaError_t launch_stream(uint32_t head_dim, const Params& p, cudaStream_t s) {
  if (p.slot_rows <= 8) return head_dim == 64 ? launch<64, 1>(p, s) : launch<128, 1>(p, s);
  return head_dim == 64 ? launch<64, 2>(p, s) : launch<128, 2>(p, s);
}

}  // namespace battn
}  // namespace hlkv
