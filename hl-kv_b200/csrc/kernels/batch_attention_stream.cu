// Batch attention for few query rows (decode, a few proposed tokens): the cache is streamed once.
//
// The bound is memory: a token of a KV head is 512 (FP16), 264 (FP8) or 144 bytes (INT4) of K and V for
// heads of 128, read once, against 4 * 128 operations for each of at most 16 query rows.
//
// One CTA per SM takes an equal share of the batch's cost (the plan's per-block costs, in proportion to the time measured
// for a tile of a cache of one format: 14 for FP16, 7 for FP8 and INT4, taken with 8 heads of 128 and used for all
// shapes), whatever the sequences' lengths: its range of the line on which all (sequence, head
// group) units lie end to end.  Two producer warps (K, V) copy the blocks' codes and parameters as they are,
// by bulk copies, into a byte ring in shared memory: tiles of 16 tokens of a block, all heads of the
// group (up to 8) at once, so that a copy is one long piece of the slot; a ring of bytes, not of
// fixed stages, keeps as many INT4 bytes in flight as FP16 ones.  Consumer warps take one (tile, head)
// each and turn codes into binary16 matrix fragments in registers:
//   S^T = K Q^T (tokens x rows), a running softmax, O^T += V^T P^T.
// A code's binary16 value is exact (E4M3, E5M2, an INT4 code's integer), so the parameters stay out of
// the matrices: the K row's scale multiplies the score in binary32 and its bias enters as
// bias * sum(q); the V row's scale multiplies the weight, and its bias is summed apart in binary32.
// A weight is rounded once, to binary16 (2^-11 of it at most; the matrix unit takes no wider one at this rate), in a unit of its row
// that follows the row's weights: those down to 2^-20 of the largest one stay in binary16's normal range, whatever sizes other
// rows' and tokens' values have.
// The order of contraction is free, so every lane takes contiguous bytes of a row and pairs them
// where they lie: K elements (j, j + 4) of each 8, V tokens (2q, 2q + 1).
//
// Measured (8 KV heads of 128, 32 query heads): 64 sequences of 8192 tokens, most in INT4, one new token each, 213 us:
// 3.9 TB/s, 0.59 of the copy rate; what is left is the consumers' instructions, about as many for an INT4 tile as
// for an FP16 one of 3.5 times the bytes.  32 windows of 4100 tokens with four new tokens each, 131 us, of which the
// copies alone take 49: every tile is converted once for each 8 of the 16 rows.  Four sequences of 300 to 1100
// tokens, 27 us: 3 to launch, 12 until the first tiles lie in shared memory (five dependent trips to memory), 6 of
// arithmetic, 6 to join the partials.
#include <cmath>
#include <cstddef>

#include "batch_attention.cuh"

namespace hlkv {
namespace battn {
namespace {

constexpr uint32_t kStages = 16;
constexpr uint32_t kTiles = 8;  // (tile, head) units of a stage: one per warp of a consumer group, or a pair

// A tile's description (words at fixed offsets: consumers read them by address).
struct alignas(16) Tile {
  uint32_t fn;      // format | tokens << 8 | (1 << 16: every row sees all its tokens)
  uint32_t pos;     // position of its first token
  uint32_t kc, kp;  // shared-memory addresses of the K codes, [tokens][heads][row bytes], and of the first row's parameters
  uint32_t vc, vp;  // the same for V
  uint32_t row_step, token_step;  // bytes from a head's parameters to the next head's, and the next token's (0: block-wide)
  float ws, wb;     // block-wide parameters
  uint32_t unused[2];
};
enum : uint32_t { kFirst = 1, kLast = 2, kDone = 4, kDirect = 8, kFirstStages = 16 };
struct alignas(16) Stage {
  Tile tile[2 * kTiles];
  uint32_t tiles, flags, seq, head0;
  uint32_t heads, unit_slot;
  uint32_t pairs;  // two tiles a warp, of one format, 16 tokens each and seen whole
};

// What the producers prepare for 32 tiles before they hand them out stage by stage.
struct alignas(16) Job {
  uint64_t src, psrc;              // codes and parameters of the tile's half
  uint32_t codes, pn, upto, delta;  // bytes of each, of the jobs up to this one, from the parameters' copy to the first one
  uint32_t fn, pos, row_step, token_step;
  float ws, wb;
  uint32_t unused[2];
};

constexpr int kWarps = 16;                   // consumers, two groups of 8
// And four more, of which two produce and two end at once: with 18 warps a block the same code measured 5 to 10 %
// slower (decode of 64 x 8192 tokens 232 us against 220 us).
constexpr int kThreads = (kWarps + 4) * 32;

// kTwo: 9 to 16 query rows.  Each consumer group then takes all stages for 8 of the rows; with up to 8
// rows the groups take the stages in turn.
template <int kD, bool kTwo>
struct Config {
  static constexpr uint32_t kStep = kTwo ? 1 : 2;      // a group's stages are every kStep-th
  static constexpr uint32_t kReaders = kTwo ? 16 : 8;  // warps that read a stage
  static constexpr int kRowsPad = kD + 4;              // floats of a row in the merge buffer: outputs, max, sum
  static constexpr uint32_t kMergeBytes = 8 * 8 * kRowsPad * 4;  // one consumer group's state
  static constexpr uint32_t kQueryBytes = kWarps * ((kD / 32) * 512 + 64 + 16);  // WarpRows
  static constexpr uint32_t kOther = kMergeBytes + static_cast<uint32_t>(sizeof(Stage)) * kStages + kQueryBytes + 2 * 32 * sizeof(Job);
  static constexpr uint32_t kRing = (226u * 1024u - kOther) / 256u * 128u;  // of each half
  static constexpr uint32_t kSmem = 2 * kRing + kOther;
};

// The piece of a unit that a producer is handing out.
struct Piece {
  uint32_t seq, head0, heads, slot, direct, single, q;
  int32_t pos0;  // of the first new token
  uint32_t fit;  // tiles of any format that the ring holds: a copy's parameters are those of all heads
};

struct Shared {
  Piece pieces[2];
  uint64_t full[2][kStages], empty[2][kStages], merged;  // of a stage's K half and its V half
  uint32_t offset[2][kStages];  // ring offsets of the halves' data
  uint64_t warp_sum[20];
  uint64_t total, base;  // cost of the batch; of the sequences before `seq`
  uint32_t seq;
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8x8 matrix of binary16 held two columns to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
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
    const uint32_t magic = magic1024();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t x = __byte_perm(a[0], b[0], j == 0 ? 0x5410 : 0x7632), y = x >> 8;
      v[4 * j] = nibble_lo(x, magic);
      v[4 * j + 1] = nibble_hi(x, magic);
      v[4 * j + 2] = nibble_lo(y, magic);
      v[4 * j + 3] = nibble_hi(y, magic);
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

// Loads by shared-memory address: 32 bits of address where a generic pointer takes 64.
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void sts64(uint32_t a, uint2 v) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ float2 lds_f2(uint32_t a) {
  const uint2 v = lds64(a);
  return make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
}

// A warp's state for one (unit, head): lane (g, q) = (lane / 4, lane % 4) holds query columns 2q and
// 2q + 1, and head elements [g kD/8, (g + 1) kD/8).
template <int kD>
struct State {
  float acc[kD / 16][4];       // [mt]: element 2 mt of columns 2q, 2q + 1, then element 2 mt + 1; units of 2^m / down
  float m[2], l[2], bias[2];   // l and bias: this lane's tokens only, in units of 2^m
  float down[2];               // a power of two
};
constexpr int kMostDown = 60;  // down is in 2^+-60: sizes of values from 2^-74 to 2^58 are followed

// What a warp keeps in shared memory for a piece: its Q^T fragments, and per column the scaled sum of q
// and the position.
template <int kD>
struct WarpRows {
  uint4 q[kD / 32][32];  // column g, pairs (j, j + 4) of the 8-element groups of a quarter row
  float qsum[8];
  int32_t pos[8];
  uint4 place;  // heads, head, first tile of a stage, tiles per round
};

// The warp's place in a stage.
struct Place {
  uint32_t rows;  // address of its WarpRows
  uint32_t heads, head_i, lane;
};

template <int kD>
__device__ __forceinline__ void begin_piece(const Params& p, State<kD>& s, WarpRows<kD>* wr, Rows rows, uint32_t context,
                                            uint32_t head, uint32_t row0, uint32_t lane) {
  const uint32_t g = lane >> 2, quad = lane & 3;
  const uint32_t r = row0 + g, tok = r / p.group, in_group = r % p.group;
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
    wr->q[i][lane] = make_uint4(a[0], a[1], a[2], a[3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a[j]));
      sum += f.x + f.y;
    }
  }
  sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
  sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
  if (quad == 0) {
    wr->qsum[g] = sum * p.qscale;
    wr->pos[g] = static_cast<int32_t>(context - rows.q + tok);
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    s.m[c] = -INFINITY;
    s.l[c] = s.bias[c] = 0.0f;
    s.down[c] = pow2(kMostDown);
  }
#pragma unroll
  for (int mt = 0; mt < kD / 16; ++mt) s.acc[mt][0] = s.acc[mt][1] = s.acc[mt][2] = s.acc[mt][3] = 0.0f;
  __syncwarp();
}

// {scale, bias} of the rows of tokens g and g + 8; `at` names the parameters' address in the description.
// Rows behind the tile's tokens give what lies there in shared memory: their weights are 0.
template <uint32_t kF>
__device__ __forceinline__ void row_params(uint32_t t, uint32_t word, const Place& at, float2 (&out)[2]) {
  if constexpr (kF == dev::kFp16) {
    out[0] = out[1] = make_float2(1.0f, 0.0f);
  } else {
    const uint2 step = lds64(t + 24);
    const uint32_t a = lds32(t + word) + at.head_i * step.x + (at.lane >> 2) * step.y, b = a + 8 * step.y;
    if constexpr (kF == dev::kInt4) {
      out[0] = lds_f2(a);
      out[1] = lds_f2(b);
    } else {
      out[0] = make_float2(__uint_as_float(lds32(a)), 0.0f);
      out[1] = make_float2(__uint_as_float(lds32(b)), 0.0f);
    }
  }
}

// Scores of tiles t[] in units of log2: lane (g, quad) has tokens g, g + 8 of columns 2 quad, 2 quad + 1.
template <int kD, uint32_t kF, int kNT>
__device__ __forceinline__ void scores(const Params& p, const uint32_t (&t)[kNT], const Place& at, float (&sc)[kNT][4]) {
  const uint32_t g = at.lane >> 2, quad = at.lane & 3;
  constexpr uint32_t kRb = kRow<kD, kF>;
  constexpr int kW = kWords<kF>;
  constexpr int kG8 = kD / 32;           // groups of 8 elements in a lane's quarter row
  constexpr uint32_t kBytes = kRb / 4;  // of a quarter row: 8 to 64
  constexpr int kPer = kF == dev::kFp16 ? 1 : kF == dev::kInt4 ? kG8 : 2;  // groups per load
  const uint32_t row = (at.head_i + g * at.heads) * kRb + quad * kBytes, eight = 8 * at.heads * kRb;
  uint32_t r0[kNT];
#pragma unroll
  for (int k = 0; k < kNT; ++k) {
    r0[k] = lds32(t[k] + 8) + row;
    sc[k][0] = sc[k][1] = sc[k][2] = sc[k][3] = 0.0f;
  }
  const uint32_t qa = at.rows + at.lane * 16;
#pragma unroll
  for (int i = 0; i < kG8; i += kPer) {
    uint32_t w[kNT][2][kPer * kW];
#pragma unroll
    for (int k = 0; k < kNT; ++k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t r = r0[k] + (h ? eight : 0u) + i * kW * 4;
        if constexpr (kPer * kW == 4) *reinterpret_cast<uint4*>(w[k][h]) = lds128(r);
        else *reinterpret_cast<uint2*>(w[k][h]) = lds64(r);
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
#pragma unroll
      for (int k = 0; k < kNT; ++k) {
        uint32_t a[4], b[4];
        k_pairs<kF>(w[k][0] + j * kW, a);
        k_pairs<kF>(w[k][1] + j * kW, b);
        const uint4 q = lds128(qa + (i + j) * 512);
        mma16816(sc[k], a[0], b[0], a[1], b[1], q.x, q.y);
        mma16816(sc[k], a[2], b[2], a[3], b[3], q.z, q.w);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kNT; ++k) {
    float2 kp[2];
    row_params<kF>(t[k], 12, at, kp);
    const float unit = p.qscale * kKeyUnit<kF>, k0 = kp[0].x * unit, k1 = kp[1].x * unit;
    float2 qs = make_float2(0.0f, 0.0f);
    if constexpr (kF == dev::kInt4) qs = lds_f2(at.rows + kG8 * 512 + quad * 2 * 4);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sc[k][c] *= k0;
      sc[k][2 + c] *= k1;
      if constexpr (kF == dev::kInt4) {
        sc[k][c] = fmaf(kp[0].y, c ? qs.y : qs.x, sc[k][c]);
        sc[k][2 + c] = fmaf(kp[1].y, c ? qs.y : qs.x, sc[k][2 + c]);
      }
    }
  }
}

__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 0xFFu) - 127; }

// The reference maximum moves only when a score passes it by 8: exponentials reach 2^8 at most.  It moves by whole numbers,
// so that what is scaled keeps its bits.  `top`: this lane's largest scores.
template <int kD>
__device__ __forceinline__ void follow_maximum(State<kD>& s, float (&top)[2]) {
  if (__any_sync(0xFFFFFFFFu, top[0] > s.m[0] + 8.0f || top[1] > s.m[1] + 8.0f)) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float v = top[c];
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
      const float mn = fmaxf(s.m[c], ceilf(v));
      if (mn == s.m[c]) continue;
      const float up = mn - s.m[c], a = halvings(up);
      s.l[c] *= a;
      s.bias[c] *= a;
      if (s.m[c] != -INFINITY) {  // (before it there is nothing in the outputs)
        // the outputs' unit stays, unless it is too far from the maximum's
        const float d = static_cast<float>(exponent_of(s.down[c])) + up, over = fmaxf(d - kMostDown, 0.0f), f = halvings(over);
        s.down[c] = pow2(static_cast<int>(d - over));
        if (over > 0.0f) {
#pragma unroll
          for (int mt = 0; mt < kD / 16; ++mt) {
            s.acc[mt][c] *= f;
            s.acc[mt][2 + c] *= f;
          }
        }
      }
      s.m[c] = mn;
    }
  }
}

// A row's outputs have a unit of their own, which follows its weights (the exponential times the value row's scale in its unit,
// about the row's largest value): where one passes 2^14 in that unit, the unit grows until it is below 2^7.  So
// the largest weight so far is 2^6 at least, and binary16 holds those down to 2^-20 of it without a loss, whatever sizes
// other rows' and tokens' values have.  w: the weights of tokens g and g + 8 of columns 2 quad, 2 quad + 1.
__device__ __forceinline__ bool too_large(const float (&w)[4]) {
  return fmaxf(fmaxf(fabsf(w[0]), fabsf(w[1])), fmaxf(fabsf(w[2]), fabsf(w[3]))) > 0x1p14f;
}
template <int kD>
__device__ __forceinline__ void follow_weights(State<kD>& s, float (&w)[4]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    // infinities (scales that are not finite) move nothing
    const float a = fabsf(w[c]), b = fabsf(w[2 + c]);
    float v = fmaxf(a < INFINITY ? a : 0.0f, b < INFINITY ? b : 0.0f);
    v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
    v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
    if (!(v > 0x1p14f)) continue;
    const int d = exponent_of(s.down[c]), up = min(exponent_of(v) - 6, d + kMostDown);
    const float f = halvings(static_cast<float>(up));
    s.down[c] = pow2(d - up);
    w[c] *= f;
    w[2 + c] *= f;
#pragma unroll
    for (int mt = 0; mt < kD / 16; ++mt) {
      s.acc[mt][c] *= f;
      s.acc[mt][2 + c] *= f;
    }
  }
}

// Encoders store an FP8 row of zeros with scale 1, a size that its values do not have.  Whether this lane's tokens g (bit 0)
// and g + 8 (bit 1) of tile t are such rows.
template <int kD, uint32_t kF>
__device__ __forceinline__ uint32_t zero_rows(uint32_t t, const Place& at) {
  constexpr uint32_t kRb = kRow<kD, kF>;
  const uint32_t base = lds32(t + 16) + (at.head_i + (at.lane >> 2) * at.heads) * kRb + (at.lane & 3) * (kRb / 4);
  uint32_t zeros = 0;
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    uint32_t any = 0;
#pragma unroll
    for (uint32_t i = 0; i < kRb / 64; ++i) {
      const uint4 w = lds128(base + h * 8 * at.heads * kRb + i * 16);
      any |= w.x | w.y | w.z | w.w;
    }
    any |= __shfl_xor_sync(0xFFFFFFFFu, any, 1);
    any |= __shfl_xor_sync(0xFFFFFFFFu, any, 2);
    if ((any & 0x7F7F7F7Fu) == 0) zeros |= 1u << h;
  }
  return zeros;
}

// Takes the weights of rows of zeros out.
__device__ __forceinline__ void without_zeros(uint32_t zeros, float (&w)[4]) {
  if (zeros & 1u) w[0] = w[1] = 0.0f;
  if (zeros & 2u) w[2] = w[3] = 0.0f;
}

// A lane's chunk of 8 elements (i-th of kD / 64) of tokens 2 quad, + 1, + 8, + 9 of a tile at `base` -> pairs of
// the first two and of the last two.  kShort: tokens from n on are taken as zeros.
template <int kD, uint32_t kF, bool kShort>
struct Chunks {
  static constexpr int kW = kWords<kF>, kOnce = kF == dev::kFp16 ? 1 : kD / 64;  // in one load where it is at most 16 bytes
  uint32_t w[4][kOnce * kW];
  __device__ __forceinline__ void take(uint32_t base, uint32_t token_bytes, int i, uint32_t quad, uint32_t n, uint32_t (&lo)[8],
                                       uint32_t (&hi)[8]) {
    if (i % kOnce == 0) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t tok = (t & 1) + (t & 2) * 4, r = base + tok * token_bytes + i * kW * 4;
        if constexpr (kOnce * kW == 4) *reinterpret_cast<uint4*>(w[t]) = lds128(r);
        else if constexpr (kOnce * kW == 2) *reinterpret_cast<uint2*>(w[t]) = lds64(r);
        else w[t][0] = lds32(r);
        if (kShort && 2 * quad + tok >= n) {
#pragma unroll
          for (int k = 0; k < kOnce * kW; ++k) w[t][k] = 0u;
        }
      }
    }
    v_pairs<kF>(w[0] + i % kOnce * kW, w[1] + i % kOnce * kW, lo);
    v_pairs<kF>(w[2] + i % kOnce * kW, w[3] + i % kOnce * kW, hi);
  }
};

// Scores and exponentials of kNT tiles of one format that every row sees whole; kShort: with n[] tokens.
// The K half of the stage is given back after the scores, if empty_k names it.
template <int kD, uint32_t kF, int kNT, bool kShort>
__device__ __forceinline__ bool step(const Params& p, State<kD>& s, const uint32_t (&t)[kNT], const uint32_t (&n)[kNT],
                                     const Place& at, uint64_t* empty_k, uint64_t* full_v, uint32_t parity) {
  const uint32_t g = at.lane >> 2, quad = at.lane & 3;
  constexpr uint32_t kRb = kRow<kD, kF>;
  float pr[kNT][4];
  scores<kD, kF, kNT>(p, t, at, pr);
  if (kNT == 2 || empty_k != nullptr) {
    __syncwarp();
    if (at.lane == 0) mbar_arrive(empty_k);
  }
  float top[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    top[c] = -INFINITY;
#pragma unroll
    for (int k = 0; k < kNT; ++k) {
      if constexpr (kShort) {
        if (g >= n[k]) pr[k][c] = -INFINITY;
        if (g + 8 >= n[k]) pr[k][2 + c] = -INFINITY;
      }
      top[c] = fmaxf(top[c], fmaxf(pr[k][c], pr[k][2 + c]));
    }
  }
  follow_maximum(s, top);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float ref = s.m[c] == -INFINITY ? 0.0f : s.m[c];  // no score so far that is not minus infinity
#pragma unroll
    for (int k = 0; k < kNT; ++k) {
      pr[k][c] = ex2(pr[k][c] - ref);
      pr[k][2 + c] = ex2(pr[k][2 + c] - ref);
      s.l[c] += pr[k][c] + pr[k][2 + c];
    }
  }
  if (!mbar_wait(full_v, parity)) return false;
#pragma unroll
  for (int k = 0; k < kNT; ++k) {
    if (kShort && n[k] == 0) continue;
    // ---- weights: the exponential times the value row's scale, in the outputs' unit
    float2 vp[2];
    row_params<kF>(t[k], 20, at, vp);
    if constexpr (kShort) {
      if (g >= n[k]) vp[0] = make_float2(0.0f, 0.0f);
      if (g + 8 >= n[k]) vp[1] = make_float2(0.0f, 0.0f);
    }
    const float u0 = vp[0].x * kValueUnit<kF>, u1 = vp[1].x * kValueUnit<kF>;
    float w[4];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      w[c] = pr[k][c] * (u0 * s.down[c]);
      w[2 + c] = pr[k][2 + c] * (u1 * s.down[c]);
    }
    if (__any_sync(0xFFFFFFFFu, too_large(w))) {
      if constexpr (kF == dev::kE4M3 || kF == dev::kE5M2) without_zeros(zero_rows<kD, kF>(t[k], at), w);
      follow_weights(s, w);
    }
    const float beta0 = fmaf(8.0f, vp[0].x, vp[0].y), beta1 = fmaf(8.0f, vp[1].x, vp[1].y);
    const uint32_t pb[2] = {transpose8(dev::pack_f16x2(w[0], w[1])), transpose8(dev::pack_f16x2(w[2], w[3]))};
    if constexpr (kF == dev::kInt4) {
#pragma unroll
      for (int c = 0; c < 2; ++c) s.bias[c] = fmaf(pr[k][2 + c], beta1, fmaf(pr[k][c], beta0, s.bias[c]));
    }
    // ---- O^T += V^T W^T
    const uint32_t token_bytes = at.heads * kRb;
    const uint32_t base = lds32(t[k] + 16) + (at.head_i + 2 * quad * at.heads) * kRb + g * (kRb / 8);
    Chunks<kD, kF, kShort> ch;
#pragma unroll
    for (int i = 0; i < kD / 64; ++i) {
      uint32_t lo[8], hi[8];
      ch.take(base, token_bytes, i, quad, n[k], lo, hi);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mma16816(s.acc[4 * i + j], lo[2 * j], lo[2 * j + 1], hi[2 * j], hi[2 * j + 1], pb[0], pb[1]);
      }
    }
  }
  return true;
}

// ---- tiles that some row sees in part: one at a time, out of line ------------------------------------

// One tile as a warp sees it.
struct View {
  uint32_t t, n, pos;
};
// Whether the query row at position `at` sees a tile's token.
__device__ __forceinline__ bool visible(const Params& p, int32_t at, const View& v, uint32_t tok) {
  const int32_t d = at - static_cast<int32_t>(v.pos + tok);
  return tok < v.n && d >= 0 && (p.window == 0 || static_cast<uint32_t>(d) < p.window || v.pos + tok < p.sinks);
}
// A query column's position.
template <int kD>
__device__ __forceinline__ int32_t position(const Place& at, uint32_t col) {
  return static_cast<int32_t>(lds32(at.rows + (kD / 32) * 512 + 32 + col * 4));
}

// O^T += V^T W^T of such a tile.  Where it holds values that are not finite, it is taken row by row, so that a row is
// not touched by what it does not see.
template <int kD, uint32_t kF>
__device__ __forceinline__ void edge_values(const Params& p, State<kD>& s, const View& v, const Place& at,
                                            const float (&pr)[4]) {
  const uint32_t g = at.lane >> 2, quad = at.lane & 3;
  constexpr uint32_t kRb = kRow<kD, kF>;
  float2 vp[2];
  row_params<kF>(v.t, 20, at, vp);
  const float u0 = vp[0].x * kValueUnit<kF>, u1 = vp[1].x * kValueUnit<kF>;
  const float beta0 = fmaf(8.0f, vp[0].x, vp[0].y), beta1 = fmaf(8.0f, vp[1].x, vp[1].y);  // INT4: what (code - 8) / 8 leaves
  float w[4];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float p0 = pr[c], p1 = pr[2 + c];
    // a hidden token's weight is 0 whatever its parameters hold
    w[c] = p0 == 0.0f ? 0.0f : p0 * (u0 * s.down[c]);
    w[2 + c] = p1 == 0.0f ? 0.0f : p1 * (u1 * s.down[c]);
    if constexpr (kF == dev::kInt4) {
      if (p0 != 0.0f) s.bias[c] = fmaf(p0, beta0, s.bias[c]);
      if (p1 != 0.0f) s.bias[c] = fmaf(p1, beta1, s.bias[c]);
    }
  }
  if (__any_sync(0xFFFFFFFFu, too_large(w))) {
    if constexpr (kF == dev::kE4M3 || kF == dev::kE5M2) without_zeros(zero_rows<kD, kF>(v.t, at), w);
    follow_weights(s, w);
  }
  const uint32_t pb[2] = {transpose8(dev::pack_f16x2(w[0], w[1])), transpose8(dev::pack_f16x2(w[2], w[3]))};
  const uint32_t token_bytes = at.heads * kRb;
  const uint32_t base = lds32(v.t + 16) + (at.head_i + 2 * quad * at.heads) * kRb + g * (kRb / 8);
  Chunks<kD, kF, true> ch;
#pragma unroll
  for (int i = 0; i < kD / 64; ++i) {
    uint32_t lo[8], hi[8];
    ch.take(base, token_bytes, i, quad, v.n, lo, hi);
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) bad = bad || has_nonfinite(lo[k]) || has_nonfinite(hi[k]);
    if (__any_sync(0xFFFFFFFFu, bad)) {
#pragma unroll 1
      for (int col = 0; col < 8; ++col) {
        // this row's view of the 16 tokens
        const int32_t row_at = position<kD>(at, col);
        const uint32_t keep_lo = (visible(p, row_at, v, 2 * quad) ? 0xFFFFu : 0u) | (visible(p, row_at, v, 2 * quad + 1) ? 0xFFFF0000u : 0u);
        const uint32_t keep_hi = (visible(p, row_at, v, 2 * quad + 8) ? 0xFFFFu : 0u) |
                                 (visible(p, row_at, v, 2 * quad + 9) ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float t[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma16816(t, lo[2 * k] & keep_lo, lo[2 * k + 1] & keep_lo, hi[2 * k] & keep_hi, hi[2 * k + 1] & keep_hi, pb[0], pb[1]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (static_cast<int>(quad * 2 + c) == col) {
              s.acc[4 * i + k][c] += t[c];
              s.acc[4 * i + k][2 + c] += t[2 + c];
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mma16816(s.acc[4 * i + k], lo[2 * k], lo[2 * k + 1], hi[2 * k], hi[2 * k + 1], pb[0], pb[1]);
      }
    }
  }
}

template <int kD, uint32_t kF>
__device__ __forceinline__ void edge_step(const Params& p, State<kD>& s, const View& v, const Place& at) {
  const uint32_t g = at.lane >> 2, quad = at.lane & 3;
  const uint32_t t[1] = {v.t};
  float sc[1][4], top[2];
  scores<kD, kF, 1>(p, t, at, sc);
  float(&pr)[4] = sc[0];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int32_t row_at = position<kD>(at, quad * 2 + c);
    if (!visible(p, row_at, v, g)) pr[c] = -INFINITY;
    if (!visible(p, row_at, v, g + 8)) pr[2 + c] = -INFINITY;
    top[c] = fmaxf(pr[c], pr[2 + c]);
  }
  follow_maximum(s, top);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float ref = s.m[c] == -INFINITY ? 0.0f : s.m[c];  // nothing seen yet
    pr[c] = ex2(pr[c] - ref);
    pr[2 + c] = ex2(pr[2 + c] - ref);
    s.l[c] += pr[c] + pr[2 + c];
  }
  edge_values<kD, kF>(p, s, v, at, pr);
}

// Out of line, with the state in memory: these tiles are few, and their code's registers are not the stream's.
template <int kD>
__device__ __noinline__ void edge_tile(const Params& p, State<kD>* state, uint32_t t, const Place at) {
  State<kD> s = *state;
  const uint2 a = lds64(t);
  const View v{t, (a.x >> 8) & 0xFFu, a.y};
  switch (a.x & 0xFFu) {
    case dev::kFp16: edge_step<kD, dev::kFp16>(p, s, v, at); break;
    case dev::kE4M3: edge_step<kD, dev::kE4M3>(p, s, v, at); break;
    case dev::kE5M2: edge_step<kD, dev::kE5M2>(p, s, v, at); break;
    default: edge_step<kD, dev::kInt4>(p, s, v, at); break;
  }
  *state = s;
}

// ---- the producer warps --------------------------------------------------------------------------
// One fills the ring of the K halves, one that of the V halves; both walk the same stages.  The K warp also
// writes the stages' descriptions.
template <int kD, bool kTwo>
struct Producer {
  using C = Config<kD, kTwo>;
  const Params& p;
  Shared& sh;
  uint32_t stages;  // address of the stages' descriptions
  uint32_t jobs;    // of this warp's 32 jobs
  uint32_t ring;    // of this half's ring
  uint32_t half, lane;
  uint32_t st = 0;      // stages emitted
  uint32_t oldest = 0;  // the first stage whose data is still in use
  uint32_t head = 0;
  uint32_t first_st = 0;  // of the piece
  bool finished = false;
  bool ok = true;

  __device__ __forceinline__ void pop() {
    ok = ok && mbar_wait(&sh.empty[half][oldest % kStages], (oldest / kStages) & 1);
    ++oldest;
  }

  // Space for `bytes` (a multiple of 16) in the ring, in order, and the stage's slot.
  __device__ __forceinline__ uint32_t reserve(uint32_t bytes) {
    if (st - oldest == kStages) pop();
    // the description is still read with the V half
    if (half == 0 && st >= kStages) ok = ok && mbar_wait(&sh.empty[1][st % kStages], (st / kStages - 1) & 1);
    uint32_t at = head;
    const bool wrap = head + bytes > C::kRing;
    if (wrap) at = 0;
    while (oldest != st && ok) {
      const uint32_t o = sh.offset[half][oldest % kStages];
      if (wrap ? !(o >= head || o < bytes) : !(o >= at && o < at + bytes)) break;
      pop();
    }
    if (oldest == st) at = 0;  // empty: start over
    head = at + bytes;
    return at;
  }

  // The next stage: `tiles` jobs from job `from` on (none: only its description).
  __device__ __forceinline__ void emit(uint32_t from, uint32_t tiles, bool pairs, uint32_t flags) {
    const uint32_t job = jobs + (from + lane) * static_cast<uint32_t>(sizeof(Job));
    uint4 size = make_uint4(0u, 0u, 0u, 0u);  // codes, pn, upto, delta
    if (lane < tiles) size = lds128(job + 16);
    size.z -= __shfl_sync(0xFFFFFFFFu, size.z - size.x - size.y, 0);  // counted from the stage's first tile
    const uint32_t total = tiles ? __shfl_sync(0xFFFFFFFFu, size.z, tiles - 1) : 0u;
    const uint32_t at = reserve(total);
    if (!ok) return;  // gave up: nothing more is copied, and the consumers give up as well
    const uint32_t slot = st % kStages, m = stages + slot * static_cast<uint32_t>(sizeof(Stage));
    const uint32_t off = ring + at + size.z - size.x - size.y, where = m + lane * static_cast<uint32_t>(sizeof(Tile));
    const bool packed = sh.pieces[half].heads == p.H;  // all heads of a token: a tile's codes are one piece of the slot
    if (lane == 0) {
      sh.offset[half][slot] = at;
      if (half == 0) {
        constexpr uint32_t kHead = offsetof(Stage, tiles), kHead2 = offsetof(Stage, heads);
        const uint32_t fl = sh.pieces[half].direct | flags | (flags & kFirstStages && st - first_st < C::kStep ? kFirst : 0u);
        sts128(m + kHead, make_uint4(tiles, fl, sh.pieces[half].seq, sh.pieces[half].head0));
        sts128(m + kHead2, make_uint4(sh.pieces[half].heads, sh.pieces[half].slot, pairs, 0u));
      }
    }
    if (lane < tiles) {
      const uint32_t po = size.y ? off + size.x + size.w : where + offsetof(Tile, ws);
      if (half == 0) {
        const uint4 d = lds128(job + 32);  // fn, pos, row_step, token_step
        const uint2 w = lds64(job + 48);
        sts128(where, make_uint4(d.x, d.y, off, po));
        sts64(where + 24, make_uint2(d.z, d.w));
        sts64(where + 32, w);
      } else {
        sts64(where + 16, make_uint2(off, po));
      }
    }
    __syncwarp();
    uint64_t* bar = &sh.full[half][slot];
    if (lane == 0) mbar_arrive_expect(bar, total);
    __syncwarp();
    if (lane < tiles) {
      const uint4 a = lds128(job);
      if (packed) bulk_load(off, uint64_t{a.x} | uint64_t{a.y} << 32, size.x, bar);
      if (size.y) bulk_load(off + size.x, uint64_t{a.z} | uint64_t{a.w} << 32, size.y, bar);
    }
    if (!packed) {
      for (uint32_t i = 0; i < tiles; ++i) {  // a copy per token: its heads lie together
        const uint32_t j = jobs + (from + i) * static_cast<uint32_t>(sizeof(Job));
        const uint2 a = lds64(j);
        const uint32_t fn = lds32(j + 32), f = fn & 0xFFu, rb = f == dev::kFp16 ? kD * 2 : f == dev::kInt4 ? kD / 2 : kD;
        const uint32_t to = __shfl_sync(0xFFFFFFFFu, off, i);
        if (lane < ((fn >> 8) & 0xFFu)) {
          bulk_load(to + lane * sh.pieces[half].heads * rb, (uint64_t{a.x} | uint64_t{a.y} << 32) + uint64_t{lane} * p.H * rb,
                    sh.pieces[half].heads * rb, bar);
        }
      }
    }
    ++st;
  }

  // Tiles of lanes < count: tokens [t0, t0 + n) of a block at `payload`.  They go out sorted by format (their order
  // does not matter to the sum), so that two tiles of one format share a softmax step: all but FP16 ones, whose
  // halves would fill too much of the ring, and those that some row sees in part.
  __device__ __forceinline__ void hand_out(uint32_t count, const uint8_t* payload, uint32_t f, uint32_t mode, uint32_t sref, uint32_t t0,
                                           uint32_t n, uint32_t pos) {
    const bool live = lane < count;
    __syncwarp();  // the jobs before have been read
    {
      // Whether every row sees all the tile's tokens.
      const int32_t pos0 = sh.pieces[half].pos0, first = static_cast<int32_t>(pos), end = first + static_cast<int32_t>(n);
      const bool whole =
          end <= pos0 + 1 && (p.window == 0 || static_cast<uint32_t>(pos0 + static_cast<int32_t>(sh.pieces[half].q) - 1 - first) < p.window ||
                              pos + n <= p.sinks);
      const uint32_t key = whole && n == 16 ? f : 4u;
      uint32_t rank = 0;
#pragma unroll
      for (uint32_t k = 0; k <= 4; ++k) {
        const uint32_t of_k = __ballot_sync(0xFFFFFFFFu, live && key == k);
        if (key > k) rank += __popc(of_k);
        else if (key == k) rank += __popc(of_k & ((1u << lane) - 1u));
      }
      const uint32_t heads = sh.pieces[half].heads, head0 = sh.pieces[half].head0;
      const uint32_t rb = f == dev::kFp16 ? kD * 2 : f == dev::kInt4 ? kD / 2 : kD, pb = f == dev::kInt4 ? 8 : 4;
      const uint32_t row0 = half ? p.T + t0 : t0;
      // The parameters of all heads of the tile's tokens, rounded out to 16 bytes (the slot's end is).
      uint64_t pa = 0;
      uint32_t pn = 0;
      if (live && f != dev::kFp16 && mode == 0) {  // (a lane without a tile has no format)
        pa = p.code_bytes[f] + uint64_t{row0} * p.H * pb;
        pn = static_cast<uint32_t>(((pa + n * p.H * pb + 15) & ~uint64_t{15}) - (pa & ~uint64_t{15}));
      }
      const uint64_t src = reinterpret_cast<uint64_t>(payload) + (uint64_t{row0} * p.H + head0) * rb;
      const uint64_t psrc = reinterpret_cast<uint64_t>(payload) + (pa & ~uint64_t{15});
      if (live) {
        const uint32_t job = jobs + rank * static_cast<uint32_t>(sizeof(Job));
        sts128(job, make_uint4(static_cast<uint32_t>(src), static_cast<uint32_t>(src >> 32), static_cast<uint32_t>(psrc),
                               static_cast<uint32_t>(psrc >> 32)));
        sts128(job + 16, make_uint4(n * heads * rb, pn, 0u, static_cast<uint32_t>(pa & 15) + head0 * pb));
        sts128(job + 32, make_uint4(f | n << 8 | (whole ? 1u << 16 : 0u), pos, pn ? pb : 0u, pn ? p.H * pb : 0u));
        const float2 w = mode != 0 ? dev::block_params_value(mode, sref) : make_float2(1.0f, 0.0f);
        sts64(job + 48, make_uint2(__float_as_uint(w.x), __float_as_uint(w.y)));
      }
    }
    __syncwarp();
    const uint32_t mine = jobs + lane * static_cast<uint32_t>(sizeof(Job));
    uint32_t upto = 0, fn = 0;
    if (live) {
      const uint2 size = lds64(mine + 16);
      upto = size.x + size.y;
      fn = lds32(mine + 32);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += y;
    }
    if (live) sts32(mine + 24, upto);
    const uint32_t next = __shfl_down_sync(0xFFFFFFFFu, fn, 1);
    // bit k: jobs k and k + 1 are alike and may share a step
    const uint32_t alike = __ballot_sync(0xFFFFFFFFu, lane + 1 < count && fn == next && fn >> 8 == (1u << 8 | 16u) && (fn & 0xFFu) != dev::kFp16);
    __syncwarp();
    const uint32_t single = sh.pieces[half].single, fit = sh.pieces[half].fit;
    for (uint32_t from = 0, tiles; from < count && ok; from += tiles) {
      const uint32_t links = (1u << (2 * single - 1)) - 1u;
      const bool pairs = 2 * single <= fit && ((alike >> from) & links) == links;
      tiles = pairs ? 2 * single : min(min(single, fit), count - from);
      emit(from, tiles, pairs, kFirstStages);
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
      if (first == 0) return b;  // no lane: b - a == 32 step, all below
      const uint32_t lo = a + (first - 1) * step;
      if (lo >= b) return b;
      b = min(lo + step, b);
      a = lo;
      if (step == 1) return lo;
    }
    return a;
  }

  __device__ __forceinline__ void run() {
    uint64_t base = sh.base;  // of sequence i's units
    for (uint32_t i = sh.seq; i < p.nseq && ok; ++i) {
      const uint64_t W = sh.total, x0 = blockIdx.x * W / gridDim.x, x1 = (uint64_t{blockIdx.x} + 1) * W / gridDim.x;
      if (base >= x1) break;
      const Rows rows = rows_of(p, i);
      uint32_t w = p.cost[i];
      if (rows.q == 0 || uint64_t{rows.q} * p.group > kStreamRows) w = 0;
      if (w == 0) continue;
      uint32_t hg = x0 > base ? static_cast<uint32_t>((x0 - base) / w) : 0u;
      for (; hg < p.head_groups && ok; ++hg) {
        const uint64_t ub = base + uint64_t{hg} * w;
        if (ub >= x1) break;
        const uint32_t lo = x0 > ub ? static_cast<uint32_t>(x0 - ub) : 0u;
        const uint32_t hi = x1 - ub < w ? static_cast<uint32_t>(x1 - ub) : w;
        // Both producers describe the piece, in the same words, each before it goes on to it; a producer
        // that is ahead of the other has the description of its own half.
        const uint32_t heads = min(8u, p.H - hg * 8);
        __syncwarp();
        if (lane == 0) {
          Piece& pc = sh.pieces[half];
          pc.seq = i;
          pc.head0 = hg * 8;
          pc.heads = heads;
          pc.slot = blockIdx.x + i * p.head_groups + hg;
          pc.direct = lo == 0 && hi == w ? kDirect : 0u;
          pc.single = heads > 4 ? 1u : heads > 2 ? 2u : heads > 1 ? 4u : 8u;  // tiles that occupy a group's warps
          const uint32_t codes = 16 * heads * kD, params = 16 * p.H * 4 + 32;
          pc.fit = C::kRing / max(2 * codes, max(codes + params, codes / 2 + 2 * params));
          pc.q = rows.q;
          pc.pos0 = static_cast<int32_t>(p.context[i] - rows.q);
        }
        __syncwarp();
        uint32_t first;
        const uint32_t count = count_of(p, i, &first);
        finished = x1 - ub <= w;  // the share ends in this piece
        piece(first, count, lo, hi);
      }
      base += uint64_t{p.head_groups} * w;
    }
    if (!finished) {  // no piece: a share without work
      if (lane == 0) sh.pieces[half] = Piece{};
      __syncwarp();
      for (uint32_t k = 0; k < C::kStep && ok; ++k) emit(0, 0, false, kDone);
    }
  }

  // The blocks of a unit whose cost begins in [lo, hi).
  __device__ __forceinline__ void piece(uint32_t first, uint32_t count, uint32_t lo, uint32_t hi) {
    const uint32_t* cost = p.block_cost + first;
    uint32_t j0 = lo == 0 ? 0u : find(cost, count, lo) + 1;
    // The first stage of each consumer group carries kFirst; at the end every group gets a stage without tiles
    // that carries kLast, after as many empty ones as bring the piece to a multiple of kStep.
    first_st = st;
    bool more = true;
    while (more && ok) {
      const uint32_t j = j0 + lane;
      uint4 b = make_uint4(0u, 0u, 0u, 0u);
      const uint8_t* payload = nullptr;
      uint32_t f = 4, v = 0;
      bool inside = false;
      if (j < count) {
        const uint32_t start = j > 0 ? __ldg(cost + j - 1) : 0u;
        b = __ldg(p.blocks + first + j);
        inside = start < hi;
        if (inside) {
          f = open_block(p, b, &payload);
          if (f <= 3) v = min((b.y >> 10) & 0x3FFu, p.T);
        }
      }
      more = __all_sync(0xFFFFFFFFu, inside);  // else the piece ends in this batch
      const uint32_t nt = (v + 15) / 16;
      const uint32_t mode = f == dev::kFp16 ? 0u : (b.y >> 4) & 3u;
      if (__all_sync(0xFFFFFFFFu, nt == 1 || (nt == 0 && !inside))) {
        hand_out(__popc(__ballot_sync(0xFFFFFFFFu, nt > 0)), payload, f, mode, b.z, 0u, v, b.w);  // a tile for every block, from lane 0 on
      } else {
        uint32_t upto = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, upto, o);
          if (lane >= static_cast<uint32_t>(o)) upto += x;
        }
        const uint32_t total = __shfl_sync(0xFFFFFFFFu, upto, 31);
        for (uint32_t t = 0; t < total && ok; t += 32) {
          // this lane: tile t + lane, in the first block whose running count passes it
          const uint32_t k = t + lane;
          uint32_t at = 0;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const uint32_t x = __shfl_sync(0xFFFFFFFFu, upto, at + o - 1);
            if (x <= k) at += o;
          }
          at = min(at, 31u);
          const uint32_t before = __shfl_sync(0xFFFFFFFFu, upto - nt, at), tv = __shfl_sync(0xFFFFFFFFu, v, at);
          const uint32_t t0 = k < total ? (k - before) * 16 : 0u;
          hand_out(min(32u, total - t),
                   reinterpret_cast<const uint8_t*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(payload), at)),
                   __shfl_sync(0xFFFFFFFFu, f, at), __shfl_sync(0xFFFFFFFFu, mode, at), __shfl_sync(0xFFFFFFFFu, b.z, at), t0,
                   k < total ? min(16u, tv - t0) : 0u, __shfl_sync(0xFFFFFFFFu, b.w, at) + t0);
        }
      }
      j0 += 32;
    }
    const uint32_t done = st - first_st, fill = (C::kStep - done % C::kStep) % C::kStep + C::kStep;
    for (uint32_t k = 0; k < fill && ok; ++k) emit(0, 0, false, kFirstStages | (k + C::kStep >= fill ? kLast | (finished ? kDone : 0u) : 0u));
  }
};

template <int kD, bool kTwo>
__global__ void __launch_bounds__(kThreads, 1) stream_kernel(const __grid_constant__ Params p) {
  using C = Config<kD, kTwo>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;
  float* merge = reinterpret_cast<float*>(smem + 2 * C::kRing);
  Stage* stages = reinterpret_cast<Stage*>(smem + 2 * C::kRing + C::kMergeBytes);
  __shared__ Shared sh;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  dev::allow_dependents_to_launch();  // the merge, which waits for this kernel's end

  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kStages; ++i) {
      for (int half = 0; half < 2; ++half) {
        mbar_init(&sh.full[half][i], 1);
        mbar_init(&sh.empty[half][i], C::kReaders);
      }
    }
    mbar_init(&sh.merged, kWarps);
    mbar_fence_init();
  }
  // ---- where this CTA's share begins: the costs of the sequences, added up in chunks of consecutive ones
  {
    const uint32_t chunk = (p.nseq + kThreads - 1) / kThreads;
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
    for (uint32_t w = 0; w < kThreads / 32; ++w) {
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

  if (warp >= kWarps) {
    const uint32_t half = warp - kWarps;
    if (half > 1) return;
    const uint32_t base = smem_addr(ring);
    Producer<kD, kTwo> producer{p, sh, smem_addr(stages), base + C::kSmem - (2 - half) * 32 * static_cast<uint32_t>(sizeof(Job)),
                                base + half * C::kRing, half, lane};
    producer.run();
    if (!producer.ok && lane == 0) atomicOr(p.err, dev::kErrInternal);
    return;
  }

  // ---- consumers
  const uint32_t group = warp / 8, w8 = warp % 8;
  const uint32_t wr_at = smem_addr(smem + 2 * C::kRing + C::kMergeBytes + sizeof(Stage) * kStages) + warp * static_cast<uint32_t>(sizeof(WarpRows<kD>));
  const uint32_t stages_at = smem_addr(stages);
  State<kD> s;
  uint32_t meets = 0;
  // All consumer warps, with a limit as every wait.
  auto meet = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.merged);
    return mbar_wait(&sh.merged, meets++ & 1);
  };
  for (uint32_t st = kTwo ? 0u : group;; st += C::kStep) {
    const uint32_t si = st % kStages, parity = (st / kStages) & 1;
    if (!mbar_wait(&sh.full[0][si], parity)) {
      if (lane == 0) atomicOr(p.err, dev::kErrInternal);
      break;
    }
    const uint32_t m = stages_at + si * static_cast<uint32_t>(sizeof(Stage));  // address of its description
    constexpr uint32_t kHead = offsetof(Stage, tiles), kHead2 = offsetof(Stage, heads);
    if ((lds32(m + kHead + 4) & (kDone | kLast)) == kDone) break;  // a share without work
    if (lds32(m + kHead + 4) & kFirst) {
      WarpRows<kD>* wr = reinterpret_cast<WarpRows<kD>*>(smem + 2 * C::kRing + C::kMergeBytes + sizeof(Stage) * kStages) + warp;
      const uint32_t heads = lds32(m + kHead2), seq = lds32(m + kHead + 8), head0 = lds32(m + kHead + 12);
      const uint32_t single = heads > 4 ? 1u : heads > 2 ? 2u : heads > 1 ? 4u : 8u;
      // a group's warps beyond `single` x heads have no tile
      if (lane == 0) wr->place = make_uint4(heads, w8 % heads, w8 / heads < single ? w8 / heads : 1u << 16, single);
      begin_piece<kD>(p, s, wr, rows_of(p, seq), p.context[seq], head0 + w8 % heads, kTwo ? group * 8 : 0u, lane);
    }
    const uint4 place = lds128(wr_at + static_cast<uint32_t>(sizeof(WarpRows<kD>)) - 16);
    const Place at{wr_at, place.x, place.y, lane};
    const uint32_t tile_i = place.z, single = place.w;
    // This warp's tiles of the stage: tile_i, and every `single`-th behind it.
    const uint32_t n_tiles = lds32(m + kHead);
    uint64_t *empty_k = &sh.empty[0][si], *full_v = &sh.full[1][si];
    bool ok = true;
    if (tile_i < n_tiles && lds32(m + kHead2 + 8) != 0) {
      const uint32_t t0 = m + tile_i * static_cast<uint32_t>(sizeof(Tile)), two[2] = {t0, t0 + single * static_cast<uint32_t>(sizeof(Tile))};
      const uint32_t n[2] = {16, 16};
      switch (lds32(t0) & 0xFFu) {
        case dev::kE4M3: ok = step<kD, dev::kE4M3, 2, false>(p, s, two, n, at, empty_k, full_v, parity); break;
        case dev::kE5M2: ok = step<kD, dev::kE5M2, 2, false>(p, s, two, n, at, empty_k, full_v, parity); break;
        default: ok = step<kD, dev::kInt4, 2, false>(p, s, two, n, at, empty_k, full_v, parity); break;
      }
    } else {
      uint64_t* give = nullptr;  // the K half's barrier with the last tile's scores, null once it is given back
#pragma unroll 1
      for (uint32_t i = tile_i; i < n_tiles && ok; i += single) {
        const uint32_t one[1] = {m + i * static_cast<uint32_t>(sizeof(Tile))};
        const uint32_t fn = lds32(one[0]), n[1] = {(fn >> 8) & 0xFFu};
        give = i + single < n_tiles || !(fn >> 16) ? nullptr : empty_k;
        if (fn >> 16) {
          switch (fn & 0xFFFFu) {
            case dev::kFp16 | 16 << 8: ok = step<kD, dev::kFp16, 1, false>(p, s, one, n, at, give, full_v, parity); break;
            case dev::kE4M3 | 16 << 8: ok = step<kD, dev::kE4M3, 1, false>(p, s, one, n, at, give, full_v, parity); break;
            case dev::kInt4 | 16 << 8: ok = step<kD, dev::kInt4, 1, false>(p, s, one, n, at, give, full_v, parity); break;
            default:
              switch (fn & 0xFFu) {
                case dev::kFp16: ok = step<kD, dev::kFp16, 1, true>(p, s, one, n, at, give, full_v, parity); break;
                case dev::kE4M3: ok = step<kD, dev::kE4M3, 1, true>(p, s, one, n, at, give, full_v, parity); break;
                case dev::kE5M2: ok = step<kD, dev::kE5M2, 1, true>(p, s, one, n, at, give, full_v, parity); break;
                default: ok = step<kD, dev::kInt4, 1, true>(p, s, one, n, at, give, full_v, parity); break;
              }
          }
        } else {
          ok = mbar_wait(full_v, parity);
          State<kD> copy = s;
          if (ok) edge_tile<kD>(p, &copy, one[0], at);
          s = copy;
        }
      }
      if (tile_i >= n_tiles) ok = mbar_wait(full_v, parity);
      if (give == nullptr) {
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_k);
      }
    }
    if (!ok) {
      if (lane == 0) atomicOr(p.err, dev::kErrInternal);
      break;
    }
    const uint4 head = lds128(m + kHead);  // tiles, flags, seq, head0
    const uint32_t slot = lds32(m + kHead2 + 4), flags = head.y;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.empty[1][si]);

    if (flags & kLast) {
      // ---- merge the warps of each head: outputs, max and sum of every row.  Groups that took the stages in
      // turn: the second leaves its state in the buffer, the first joins it to its own warp by warp and
      // leaves the sum there.  Groups of different rows use the buffer one after the other.
      const uint32_t g = lane >> 2, quad = lane & 3;
      float* mine = merge + w8 * 8 * C::kRowsPad;
      const Rows rows = rows_of(p, head.z);
      const uint32_t head0 = head.w, heads = at.heads, n_rows = rows.q * p.group;
      bool met = true;
#pragma unroll 1
      for (uint32_t turn = 0; turn < 2; ++turn) {
        if (group == 1 - turn) {
          const bool join = !kTwo && turn == 1;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float l = s.l[c], b = s.bias[c], m_own = s.m[c], fo = 1.0f, ft = 0.0f;
            const float unit = pow2(-exponent_of(s.down[c]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
              l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
              b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
            }
            float* row = mine + (quad * 2 + c) * C::kRowsPad;
            if (join) {
              const float2 ml = *reinterpret_cast<const float2*>(row + kD);
              const float M = fmaxf(m_own, ml.x);
              fo = M == -INFINITY ? 1.0f : exp2f(m_own - M);
              ft = M == -INFINITY ? 1.0f : exp2f(ml.x - M);
              l = fmaf(l, fo, ml.y * ft);
              m_own = M;
            }
#pragma unroll
            for (int mt = 0; mt < kD / 16; ++mt) {
              float2* at2 = reinterpret_cast<float2*>(row + g * (kD / 8) + 2 * mt);
              float2 x = make_float2(fmaf(s.acc[mt][c], unit, b), fmaf(s.acc[mt][2 + c], unit, b));
              if (join) {
                const float2 y = *at2;
                x = make_float2(fmaf(x.x, fo, y.x * ft), fmaf(x.y, fo, y.y * ft));
              }
              *at2 = x;
            }
            __syncwarp();  // every lane has read the other group's max and sum
            if (g == 0) *reinterpret_cast<float2*>(row + kD) = make_float2(m_own, l);
          }
        }
        met = met && meet();
        if (!met) break;
        if (!kTwo && turn == 0) continue;
        const uint32_t row0 = kTwo ? (1 - turn) * 8 : 0u, rows_here = n_rows > row0 ? min(8u, n_rows - row0) : 0u;
        for (uint32_t i = threadIdx.x; i < heads * rows_here * (kD / 4); i += kWarps * 32) {
          const uint32_t e = i % (kD / 4), r = (i / (kD / 4)) % rows_here, h = i / (kD / 4) / rows_here;
          float M = -INFINITY, L = 0.0f;
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (uint32_t t = 0; t < single; ++t) M = fmaxf(M, merge[((t * heads + h) * 8 + r) * C::kRowsPad + kD]);
          for (uint32_t t = 0; t < single; ++t) {
            const float* row = merge + ((t * heads + h) * 8 + r) * C::kRowsPad;
            const float2 ml = *reinterpret_cast<const float2*>(row + kD);
            const float a = M == -INFINITY ? 1.0f : exp2f(ml.x - M);
            const float4 x = *reinterpret_cast<const float4*>(row + 4 * e);
            L = fmaf(ml.y, a, L);
            o.x = fmaf(x.x, a, o.x);
            o.y = fmaf(x.y, a, o.y);
            o.z = fmaf(x.z, a, o.z);
            o.w = fmaf(x.w, a, o.w);
          }
          if (flags & kDirect) {
            if (L == 0.0f && M == -INFINITY) L = 1.0f;  // sees nothing: zeros
            const uint32_t tok = (row0 + r) / p.group, gi = (row0 + r) % p.group;
            *reinterpret_cast<uint2*>(p.out + (rows.first + tok) * p.out_stride + uint64_t{(head0 + h) * p.group + gi} * kD + 4 * e) =
                make_uint2(dev::pack_f16x2(o.x / L, o.y / L), dev::pack_f16x2(o.z / L, o.w / L));
          } else {
            float* dst = p.partial + ((uint64_t{slot} * 8 + h) * p.slot_rows + row0 + r) * C::kRowsPad;
            *reinterpret_cast<float4*>(dst + 4 * e) = o;
            if (e == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(M, L);
          }
        }
        met = met && meet();  // the buffer is written again
        if (!met) break;
      }
      if (!met) {
        if (lane == 0) atomicOr(p.err, dev::kErrInternal);
        break;
      }
      if (flags & kDone) break;
    }
  }
}

// Joins the partial results of the units that several CTAs took: kSplit warps for each (sequence, head, row), taking
// the partials in turn with a running maximum of their own.  Also writes the zeros of rows whose sequence lists
// no block.
constexpr uint32_t kMergeWarps = 8;
template <int kD, uint32_t kSplit>
__global__ void __launch_bounds__(kMergeWarps * 32) merge_kernel(const __grid_constant__ Params p) {
  constexpr int kPad = kD + 4, kPer = kD / 32;  // floats of a row; elements of a lane
  __shared__ float s_o[kSplit > 1 ? kMergeWarps : 1][kD];
  __shared__ float2 s_ml[kMergeWarps];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % kSplit;
  const uint32_t id = blockIdx.x * (kMergeWarps / kSplit) + warp / kSplit;
  const uint32_t r = id % p.slot_rows, unit_head = id / p.slot_rows;
  const uint32_t i = unit_head / p.H, head = unit_head % p.H, hg = head / 8, h = head % 8;
  dev::wait_for_prerequisites();
  // (uniform over the warps of a row; with kSplit > 1 a CTA has one row)
  if (i >= p.nseq) return;
  const Rows rows = rows_of(p, i);
  const uint32_t n_rows = rows.q * p.group;
  if (r >= n_rows || uint64_t{rows.q} * p.group > kStreamRows) return;
  const uint64_t W = p.prefix[p.nseq] * p.head_groups, before = p.prefix[i], w = p.prefix[i + 1] - before;
  uint32_t c0 = 0, c1 = 0;
  if (w > 0) {
    const uint64_t a = before * p.head_groups + hg * w, b = a + w - 1;
    // CTA c takes [c W / G, (c + 1) W / G): the one that holds x is the largest c with c W / G <= x
    c0 = static_cast<uint32_t>(((a + 1) * p.ctas - 1) / W);
    c1 = static_cast<uint32_t>(((b + 1) * p.ctas - 1) / W);
    if (c0 == c1) return;  // one CTA had it all and wrote the rows
  }
  float M = -INFINITY, L = 0.0f, o[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) o[k] = 0.0f;
  if (w > 0) {
    const uint64_t step = uint64_t{8} * p.slot_rows * kPad;
    const float* base = p.partial + (c0 + uint64_t{i} * p.head_groups + hg) * step + (uint64_t{h} * p.slot_rows + r) * kPad;
    // a CTA whose range is empty (more CTAs than cost) took nothing and may have written nothing
    auto empty = [&](uint32_t c) { return p.ctas > W && c * W / p.ctas == (uint64_t{c} + 1) * W / p.ctas; };
#pragma unroll 4
    for (uint32_t c = c0 + part; c <= c1; c += kSplit) {
      if (empty(c)) continue;
      const float* s = base + (c - c0) * step;
      const float2 ml = *reinterpret_cast<const float2*>(s + kD);
      float x[kPer];
      if constexpr (kPer == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(s + 4 * lane);
      else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(s + 2 * lane);
      const float m = fmaxf(M, ml.x);
      const float fo = m == -INFINITY ? 1.0f : exp2f(M - m), ft = m == -INFINITY ? 1.0f : exp2f(ml.x - m);
      M = m;
      L = fmaf(L, fo, ml.y * ft);
#pragma unroll
      for (int k = 0; k < kPer; ++k) o[k] = fmaf(o[k], fo, x[k] * ft);
    }
  }
  const uint32_t tok = r / p.group, gi = r % p.group;
  uint16_t* dst = p.out + (rows.first + tok) * p.out_stride + uint64_t{head * p.group + gi} * kD;
  if constexpr (kSplit == 1) {
    if (L == 0.0f && M == -INFINITY) L = 1.0f;  // sees nothing: zeros
    if constexpr (kPer == 4) {
      *reinterpret_cast<uint2*>(dst + 4 * lane) = make_uint2(dev::pack_f16x2(o[0] / L, o[1] / L), dev::pack_f16x2(o[2] / L, o[3] / L));
    } else {
      *reinterpret_cast<uint32_t*>(dst + 2 * lane) = dev::pack_f16x2(o[0] / L, o[1] / L);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) s_o[warp][lane * kPer + k] = o[k];
    if (lane == 0) s_ml[warp] = make_float2(M, L);
    __syncthreads();
    const uint32_t e = threadIdx.x;
    if (e >= kD) return;
    M = -INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < kSplit; ++k) M = fmaxf(M, s_ml[k].x);
    float sum = 0.0f;
    L = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kSplit; ++k) {
      const float a = M == -INFINITY ? 1.0f : exp2f(s_ml[k].x - M);
      L = fmaf(s_ml[k].y, a, L);
      sum = fmaf(s_o[k][e], a, sum);
    }
    if (L == 0.0f && M == -INFINITY) L = 1.0f;  // sees nothing: zeros
    dst[e] = __half_as_ushort(__float2half_rn(sum / L));
  }
}

template <int kD, bool kTwo>
cudaError_t launch(const Params& p, cudaStream_t s) {
  using C = Config<kD, kTwo>;
  static SharedMemoryOnce once;
  const cudaError_t e = once.allow(reinterpret_cast<const void*>(stream_kernel<kD, kTwo>), C::kSmem);
  if (e != cudaSuccess) return e;
  stream_kernel<kD, kTwo><<<p.ctas, kThreads, C::kSmem, s>>>(p);
  const cudaError_t e2 = cudaGetLastError();
  if (e2 != cudaSuccess) return e2;
  // The merge's CTAs start while the stream's last ones run, and wait for them.
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kMergeWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // A warp a row where a unit has few partials (32 windows of 16 rows, 5 each: 132 us with it, 137 us with a CTA a row),
  // a CTA a row where it has many (4 short sequences, 37 each: 27 us with it, 37 us with a warp a row).  The border lies
  // between these two, by no other case.
  const uint32_t rows = p.nseq * p.H * p.slot_rows;
  if (uint64_t{p.nseq} * p.head_groups * 12 > p.ctas) {
    cfg.gridDim = dim3((rows + kMergeWarps - 1) / kMergeWarps);
    return cudaLaunchKernelEx(&cfg, merge_kernel<kD, 1>, p);
  }
  cfg.gridDim = dim3(rows);
  return cudaLaunchKernelEx(&cfg, merge_kernel<kD, kMergeWarps>, p);
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
  if (p.slot_rows <= 8) return head_dim == 64 ? launch<64, false>(p, s) : launch<128, false>(p, s);
  return head_dim == 64 ? launch<64, true>(p, s) : launch<128, true>(p, s);
}

}  // namespace battn
}  // namespace hlkv
