// Batch attention for many query rows (prompts and chunks of prompts): tiles on the fifth-generation tensor
// cores.
//
// A row is a (new token, query head) pair of one (sequence, KV head); 4 D operations for each token it sees, so
// the bound is the matrix rate, and next to it the exponentials (16 a clock and SM) and the conversion of codes.
// A CTA takes 256 rows as two accumulator tiles of 128 and walks the sequence's visible tokens in tiles of
// 128:
//   S = Q K^T (tcgen05.mma, both operands in shared memory), a running softmax by one thread per row,
//   O += P V (P from tensor memory, V from shared memory).
// Eight warps convert the blocks' codes to binary16 in the 128-byte-swizzled layout, one tile ahead, once for both
// accumulator tiles; the two tiles' softmax warpgroups alternate with the tensor cores: while one exponentiates,
// the other's products run.  Tensor memory: S0, S1, O0, O1; P overwrites S.
// As in the stream kernel a code's binary16 value is exact and its parameters stay outside: the K row's scale and
// bias in the score, the V row's scale in the weight, its bias in a sum of its own, all in binary32.  A weight is
// rounded once, to binary16 (2^-11 of it at most; the matrix unit takes no wider one at this rate), against a reference of its row
// that follows scores and value scales together.
// Codes are laid in the order (0, 4, 1, 5, 2, 6, 3, 7) of each 8, where the formats' words hold them: Q's elements
// lie the same way, and the outputs are put back in order at the end.
//
// Measured (8 KV heads of 128, 32 query heads; six chunks of up to 1645 new tokens over contexts of up to 8024, formats
// mixed): 945 us, 394 TFLOP/s, 0.24 of the matrix rate; the caches of one format alone: FP16 757, E4M3 927, INT4 1008 us.
// The products of the tiles that are walked, 388 GFLOP, would take 234 us at the matrix rate; on copies that left the other
// part out the conversion took 640 us and the softmax 950.  The softmax's two warps per scheduler wait on their own chains (an issue every 2.2 cycles), and the per-token
// parameters are broadcast from shared memory: a float4 load returns 512 bytes to a warp, 2048 cycles of a tile for FP8
// and 4096 for INT4.  Five prompts of heads of 64 with a window of 1024: 155 us; a CTA there walks 6.5 tiles on
// average, of which the last and the sinks' are short.  250 new tokens over 8000, four row tiles a head: 139 us.
// References of one row each, next to a unit that 128 tokens shared, took chunks from 954 to 950 us (FP16 alone 827 to 757,
// E4M3 924 to 927, INT4 994 to 1008), the heads of 64 from 154 to 158 and few rows over 8000 tokens from 73 to 77.
// Tried and slower than 928 us (the same without the split over tokens, whose code costs 2 %): halves of 64 tokens with scores of their own (1020 us), products issued by a softmax warp (1190),
// half the loads in flight (1070), FP8 and INT4 rows in 16-byte pieces a tile ahead (985).
#include <algorithm>
#include <cmath>

#include "batch_attention.cuh"

namespace hlkv {
namespace battn {
namespace {

constexpr int kSoftmaxWarps = 8, kStageWarps = 8;
constexpr int kThreads = (kSoftmaxWarps + kStageWarps + 1) * 32;  // and one that issues the products
constexpr uint32_t kTile = 128;                                  // tokens of a tile
constexpr uint32_t kRowsCta = 256;

template <int kD>
struct Config {
  static constexpr uint32_t kPanels = kD / 64;               // 64 elements of a row make 128 bytes
  static constexpr uint32_t kPanel = kTile * 128;            // bytes
  static constexpr uint32_t kOperand = kPanels * kPanel;     // 128 rows of kD binary16 values
  static constexpr uint32_t kQ = 0, kK = 2 * kOperand, kV = kK + 2 * kOperand, kEnd = kV + 2 * kOperand;
  static constexpr uint32_t kSmem = kEnd + 1024;  // the operands start on 1024 bytes
};

// 256 rows of a sequence.
struct RowTile {
  uint32_t seq, tile;  // tile 0xFFFFFFFF: none
};

struct Shared {
  RowTile mine;
  uint32_t splits, part;  // of the row tile's tokens
  bool split;             // this row tile's
  uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2];  // of the two stages
  uint64_t s_full[2], p_full[2], o_done[2];               // of the two accumulator tiles
  // Of the tokens of the last four tiles: a K half may be written again while the softmax of the tile two before
  // still reads these.
  alignas(16) float ks[4][kTile], kb[4][kTile], vs[4][kTile], vb[4][kTile];  // read four at a time
  alignas(16) float es[4][kTile];  // where the scales of 16 tokens lie far apart: a token's exponent under theirs
  int exponent[4][kStageWarps];
  uint32_t kind[4][kStageWarps];  // of 16 tokens: 1 a scale, 2 a bias, 4 some token does not exist, 8 scales far apart
  uint32_t exists[4][kStageWarps];
  uint32_t tmem, redo;
  uint32_t sums[kThreads / 32];
};

// ---- tcgen05 ---------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  // start address, leading and stride byte offsets in units of 16 bytes, version 1, 128-byte swizzle
  return uint64_t{(addr >> 4) & 0x3FFFu} | uint64_t{lbo >> 4} << 16 | uint64_t{sbo >> 4} << 32 | uint64_t{1} << 46 | uint64_t{2} << 61;
}
// binary16 operands, binary32 accumulator, M = 128.
constexpr uint32_t instruction(uint32_t n, bool b_transposed) {
  return 1u << 4 | (b_transposed ? 1u << 16 : 0u) | n / 8 << 17 | 128u / 16 << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
               "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
               "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
               : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of this warp's 32 rows: one row a lane.
__device__ __forceinline__ void tmem_load32(uint32_t a, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(a));
}
__device__ __forceinline__ void tmem_load16(uint32_t a, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(a));
}
__device__ __forceinline__ void tmem_store16(uint32_t a, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t a, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
      "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Two binary32 operations in one instruction.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Pair pair(uint32_t x, uint32_t y) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ float2 split(Pair a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// Eight elements in one of the formats -> binary16 in the order (0, 4, 1, 5, 2, 6, 3, 7).  FP16 as it is; a K row's
// FP8 codes as they are, a V row's E4M3 times 2^-8 and E5M2 times 2^-15; INT4 (code - 8) / 8.
template <bool kValue>
__device__ __forceinline__ uint4 convert(uint32_t f, uint4 raw) {
  uint32_t a0, a1, a2, a3;
  if (f == dev::kFp16) {
    a0 = __byte_perm(raw.x, raw.z, 0x5410);
    a1 = __byte_perm(raw.x, raw.z, 0x7632);
    a2 = __byte_perm(raw.y, raw.w, 0x5410);
    a3 = __byte_perm(raw.y, raw.w, 0x7632);
  } else if (f == dev::kInt4) {
    const uint32_t magic = magic1024(), y = raw.x >> 8;
    a0 = nibble_lo(raw.x, magic);
    a1 = nibble_hi(raw.x, magic);
    a2 = nibble_lo(y, magic);
    a3 = nibble_hi(y, magic);
  } else {
    const uint32_t x = __byte_perm(raw.x, raw.y, 0x5140), y = __byte_perm(raw.x, raw.y, 0x7362);
    if (f == dev::kE4M3) {
      a0 = fp8_lo<dev::kE4M3>(x);
      a1 = fp8_hi<dev::kE4M3>(x);
      a2 = fp8_lo<dev::kE4M3>(y);
      a3 = fp8_hi<dev::kE4M3>(y);
    } else {
      a0 = fp8_lo<dev::kE5M2>(x);
      a1 = fp8_hi<dev::kE5M2>(x);
      a2 = fp8_lo<dev::kE5M2>(y);
      a3 = fp8_hi<dev::kE5M2>(y);
    }
    if constexpr (kValue) {
      const uint32_t down = f == dev::kE4M3 ? 0x1C001C00u : 0x02000200u;
      a0 = hmul2(a0, down);
      a1 = hmul2(a1, down);
      a2 = hmul2(a2, down);
      a3 = hmul2(a3, down);
    }
  }
  return make_uint4(a0, a1, a2, a3);
}

template <uint32_t kF>
struct Format {
  static constexpr uint32_t value = kF;
};

// Shared-memory address of 16-byte chunk c (of kD / 8) of row r in an operand: panels of 64 elements, the chunk
// index of a row's 128 bytes XORed with the row's place in its 8.
__device__ __forceinline__ uint32_t chunk_at(uint32_t base, uint32_t r, uint32_t c) {
  return base + (c >> 3) * (kTile * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// The tokens that a row tile's rows see, as positions: [0, a) and [b0, b1), walked in tiles of 128 from tile `from` on.
struct Walk {
  uint32_t a, b0, b1, from;
  __device__ __forceinline__ uint32_t first_tiles() const { return (a + kTile - 1) / kTile; }
  __device__ __forceinline__ uint32_t tiles() const { return first_tiles() + (b1 - b0 + kTile - 1) / kTile; }
  __device__ __forceinline__ bool begins(uint32_t j) const { return j == 0 || j + from == first_tiles(); }  // a run of tiles
  __device__ __forceinline__ void tile(uint32_t j, uint32_t* pos, uint32_t* n) const {
    j += from;
    const uint32_t fa = first_tiles();
    if (j < fa) {
      *pos = j * kTile;
      *n = min(kTile, a - *pos);
    } else {
      *pos = b0 + (j - fa) * kTile;
      *n = min(kTile, b1 - *pos);
    }
  }
};

__device__ __forceinline__ Walk walk_of(const Params& p, uint32_t n_blocks, int32_t p_lo, int32_t p_hi) {
  if (p_hi < 0 || n_blocks == 0) return Walk{0, 0, 0, 0};
  const uint32_t end = static_cast<uint32_t>(p_hi) + 1;
  const int64_t low = p.window == 0 ? 0 : int64_t{p_lo} - p.window + 1;
  if (low <= int64_t{p.sinks}) return Walk{0, 0, end, 0};
  return Walk{min(p.sinks, end), static_cast<uint32_t>(low), end, 0};
}

// Positions that the rows [row0, row0 + rows) of a sequence with `base` tokens before its new ones have.
__device__ __forceinline__ int32_t position_of(const Params& p, int32_t base, uint32_t row) {
  return base + static_cast<int32_t>(row / p.group);
}

// Few row tiles over long contexts: each one's tokens are split over as many CTAs as the GPU has left, kSplitTiles tiles
// each at least, and joined by join_kernel.  A batch whose row tiles fill half the GPU is not split.  (One sequence of 250
// new tokens over 8000: 124 us, 340 without; two of 5 to 8 new tokens: 70 us and 283.  The join's launch costs an
// unsplit batch 2 to 4 us.)
constexpr uint32_t kMaxSplits = 16, kSplitTiles = 4;
__device__ __forceinline__ uint32_t splits_of(const Params& p, uint32_t row_tiles) {
  const uint32_t units = row_tiles * p.H;
  return units == 0 ? 1u : max(1u, min(kMaxSplits, p.ctas / units));
}
__device__ __forceinline__ uint32_t parts_of(uint32_t splits, uint32_t n_tiles) {
  return max(1u, min(splits, n_tiles / kSplitTiles));
}

// Most sequences to look through: 30 sequences of up to 300 new tokens over up to 3000 took 419 us so and 447 us with
// the last tiles of all first, 100 of them 1401 and 1417 us, 250 of them 3875 and 3742 us.
constexpr uint32_t kOrdered = 128;

// A tile sees at most `cap` tokens; its level is its last token's tile of 128, or the one of the cap.
__device__ __forceinline__ uint32_t token_cap_of(const Params& p) {
  const uint64_t cap = p.window == 0 ? 0x7FFFFFFFu : uint64_t{p.window} + p.sinks + kRowsCta / p.group + 1;
  return static_cast<uint32_t>(min(cap, uint64_t{0x7FFFFFFFu}));
}
// Row tiles of sequence i at level x and above: from the first one whose last token lies behind (x - 1) 128.
__device__ __forceinline__ uint32_t row_tiles_above(const Params& p, uint32_t i, uint32_t x, uint32_t cap) {
  const Rows rows = rows_of(p, i);
  const uint64_t n_rows = uint64_t{rows.q} * p.group;
  if (n_rows <= kStreamRows) return 0u;
  const uint32_t n = static_cast<uint32_t>((n_rows + kRowsCta - 1) / kRowsCta);
  if (x == 0) return n;
  const uint64_t from = uint64_t{x - 1} * kTile;
  const int64_t tok = static_cast<int64_t>(from) - (int64_t{p.context[i]} - rows.q);  // that token as a new one
  if (from >= cap || tok >= int64_t{rows.q}) return 0u;
  return tok <= 0 ? n : n - static_cast<uint32_t>(uint64_t(tok) * p.group / kRowsCta);
}
// All row tiles of the batch, counted by a warp.
__device__ __forceinline__ uint32_t count_row_tiles(const Params& p) {
  uint32_t c = 0;
  for (uint32_t i = threadIdx.x & 31; i < p.nseq; i += 32) c += row_tiles_above(p, i, 0, 0);
  return __reduce_add_sync(0xFFFFFFFFu, c);
}

// The r-th (sequence, row tile) of the batch when they are ordered by the tiles of tokens that they walk, most first:
// CTAs start in that order, and the last ones to end are short.  Found by a warp: the level of r by bisection over
// counts (a sequence's tiles of a level and above are its last ones), then its place among the level's tiles.
__device__ __forceinline__ RowTile row_tile_of_rank(const Params& p, uint32_t r) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t cap = token_cap_of(p);
  auto above = [&](uint32_t i, uint32_t x) { return row_tiles_above(p, i, x, cap); };
  auto count = [&](uint32_t x) {
    uint32_t c = 0;
    for (uint32_t i = lane; i < p.nseq; i += 32) c += above(i, x);
    return __reduce_add_sync(0xFFFFFFFFu, c);
  };
  uint32_t longest = 0;
  for (uint32_t i = lane; i < p.nseq; i += 32) longest = max(longest, min(p.context[i], cap));
  uint32_t lo = 0, hi = (__reduce_max_sync(0xFFFFFFFFu, longest) + kTile - 1) / kTile + 1;  // count(hi) == 0
  while (hi - lo > 1) {
    const uint32_t x = (lo + hi) / 2;
    if (count(x) > r) lo = x;
    else hi = x;
  }
  uint32_t left = r - count(lo + 1);  // place among the level's tiles
  for (uint32_t base = 0; base < p.nseq; base += 32) {
    const uint32_t i = base + lane;
    const uint32_t more = i < p.nseq ? above(i, lo) : 0u, less = i < p.nseq ? above(i, lo + 1) : 0u;
    uint32_t upto = more - less;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += y;
    }
    const uint32_t here = __ballot_sync(0xFFFFFFFFu, upto > left);
    if (here != 0) {
      const uint32_t owner = __ffs(here) - 1;
      const uint32_t before = __shfl_sync(0xFFFFFFFFu, upto - (more - less), owner), above_it = __shfl_sync(0xFFFFFFFFu, less, owner);
      const uint32_t seq = base + owner;
      const uint32_t n = static_cast<uint32_t>((uint64_t{rows_of(p, seq).q} * p.group + kRowsCta - 1) / kRowsCta);
      return RowTile{seq, n - 1 - above_it - (left - before)};
    }
    left -= __shfl_sync(0xFFFFFFFFu, upto, 31);
  }
  return RowTile{0u, 0xFFFFFFFFu};
}

// Whether an FP8 row holds zeros alone.  Out of line: few rows are looked at.
__device__ __noinline__ bool zero_row(const uint8_t* row, uint32_t bytes) {
  uint32_t any = 0;
  for (uint32_t i = 0; i < bytes; i += 16) {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(row + i));
    any |= w.x | w.y | w.z | w.w;
  }
  return (any & 0x7F7F7F7Fu) == 0;
}

// The r-th (sequence, row tile) of a batch of many sequences, the last tiles of all sequences first: tiles o from a
// sequence's last one on make level o, and the levels before it hold the sum of min(row tiles, o).  Found by the CTA, a
// thread for consecutive sequences.
__device__ __noinline__ RowTile row_tile_of_many(const Params& p, uint32_t r, uint32_t* sums, RowTile* found) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t chunk = (p.nseq + kThreads - 1) / kThreads, a = min(threadIdx.x * chunk, p.nseq), b = min(a + chunk, p.nseq);
  auto before = [&](uint32_t o) {
    uint32_t c = 0;
    for (uint32_t i = a; i < b; ++i) c += min(row_tiles_above(p, i, 0, 0), o);
    c = __reduce_add_sync(0xFFFFFFFFu, c);
    if (lane == 0) sums[warp] = c;
    __syncthreads();
    uint32_t all = 0;
    for (uint32_t w = 0; w < kThreads / 32; ++w) all += sums[w];
    __syncthreads();
    return all;
  };
  uint32_t lo = 0, hi = static_cast<uint32_t>((uint64_t{p.max_rows} + kRowsCta - 1) / kRowsCta), skip = 0;
  if (r >= before(hi)) return RowTile{0u, 0xFFFFFFFFu};
  while (hi - lo > 1) {
    const uint32_t o = (lo + hi) / 2, n = before(o);
    if (n <= r) {
      lo = o;
      skip = n;
    } else {
      hi = o;
    }
  }
  uint32_t mine = 0;
  for (uint32_t i = a; i < b; ++i) mine += row_tiles_above(p, i, 0, 0) > lo;
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= static_cast<uint32_t>(o)) upto += y;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  for (uint32_t w = 0; w < warp; ++w) upto += sums[w];
  uint32_t left = r - skip;  // place in the level
  if (left < upto && left >= upto - mine) {
    left -= upto - mine;
    for (uint32_t i = a; i < b; ++i) {
      const uint32_t n = row_tiles_above(p, i, 0, 0);
      if (n > lo && left-- == 0) *found = RowTile{i, n - 1 - lo};
    }
  }
  __syncthreads();
  return *found;
}

template <int kD>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ Params p) {
  using C = Config<kD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;

  // ---- the CTA's rows: those that see most tokens first; the heads of the same rows side by side, since a token's
  // heads lie together
  dev::allow_dependents_to_launch();  // join_kernel, which waits for this kernel's end
  const uint32_t h = blockIdx.x % p.H;
  RowTile mine;
  uint32_t splits = 1, part = 0;
  if (p.nseq <= kOrdered) {
    if (warp == 0) {
      const uint32_t n = count_row_tiles(p);
      splits = splits_of(p, n);
      uint32_t rank = blockIdx.x / p.H;
      if (n > 0) part = rank / n;
      mine = RowTile{0u, 0xFFFFFFFFu};
      if (n > 0 && part < splits) mine = row_tile_of_rank(p, rank - part * n);
      if (lane == 0) {
        sh.mine = mine;
        sh.splits = splits;
        sh.part = part;
      }
    }
    __syncthreads();
    mine = sh.mine;
    splits = sh.splits;
    part = sh.part;
  } else if (p.tile_ranks != 0) {
    mine = row_tile_of_many(p, blockIdx.x / p.H, sh.sums, &sh.mine);
  } else {  // last tiles of all sequences first
    const uint32_t seq = blockIdx.x / p.H % p.nseq, order = blockIdx.x / p.H / p.nseq;
    const uint64_t n_rows = uint64_t{rows_of(p, seq).q} * p.group, n = (n_rows + kRowsCta - 1) / kRowsCta;
    mine = RowTile{seq, n_rows > kStreamRows && order < n ? static_cast<uint32_t>(n) - 1 - order : 0xFFFFFFFFu};
  }
  if (mine.tile == 0xFFFFFFFFu) return;
  const uint32_t seq = mine.seq;
  const Rows rows = rows_of(p, seq);
  const uint32_t n_rows = rows.q * p.group;
  const uint32_t row0 = mine.tile * kRowsCta, rows_here = min(kRowsCta, n_rows - row0);
  const uint32_t n_acc = rows_here > 128 ? 2 : 1;
  const uint32_t ctx = p.context[seq];
  const int32_t pos_base = static_cast<int32_t>(ctx) - static_cast<int32_t>(rows.q);  // of the first new token
  const int32_t p_lo = pos_base + static_cast<int32_t>(row0 / p.group), p_hi = pos_base + static_cast<int32_t>((row0 + rows_here - 1) / p.group);
  uint32_t first_block;
  const uint32_t n_blocks = count_of(p, seq, &first_block);
  Walk walk = walk_of(p, n_blocks, p_lo, p_hi);
  uint32_t n_tiles = walk.tiles();
  const uint32_t parts = parts_of(splits, n_tiles);
  if (part >= parts) return;
  if (parts > 1) {  // this CTA's share of the tiles
    walk.from = static_cast<uint32_t>(uint64_t{n_tiles} * part / parts);
    n_tiles = static_cast<uint32_t>(uint64_t{n_tiles} * (part + 1) / parts) - walk.from;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.k_full[i], kStageWarps);
      mbar_init(&sh.v_full[i], kStageWarps);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], 4);
      mbar_init(&sh.o_done[i], 1);
    }
    sh.redo = 0;
    sh.split = parts > 1;
    mbar_fence_init();
  }
  if (warp == kSoftmaxWarps + kStageWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // ---- Q into its two operands, rows behind the last one zeros
  for (uint32_t i = threadIdx.x; i < n_acc * 128 * (kD / 8); i += kThreads) {
    const uint32_t c = i % (kD / 8), r = i / (kD / 8), row = row0 + r;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows_here) {
      v = __ldg(reinterpret_cast<const uint4*>(p.q + (rows.first + row / p.group) * p.q_stride + uint64_t{h * p.group + row % p.group} * kD) + c);
    }
    v = convert<false>(dev::kFp16, v);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(base + C::kQ + (r >> 7) * C::kOperand, r & 127, c)), "r"(v.x), "r"(v.y),
                 "r"(v.z), "r"(v.w)
                 : "memory");
  }
  dev::fence_proxy_async_smem();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  bool ok = true;

  if (warp < kSoftmaxWarps) {
    // ================= softmax: one row a thread =================
    const uint32_t acc = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = ((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + acc * 128, t_o = tmem + lanes + 256 + acc * kD;
    const uint32_t row = row0 + acc * 128 + r;
    const bool live = acc * 128 + r < rows_here;
    const uint32_t tok = row / p.group, head = h * p.group + row % p.group;
    const int32_t pos = pos_base + static_cast<int32_t>(tok);
    // the first token of the window
    const int32_t low = p.window == 0 ? -1 : static_cast<int32_t>(max(int64_t{pos} - p.window + 1, int64_t{-1}));
    float qsum = 0.0f;
    if (live) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (rows.first + tok) * p.q_stride + uint64_t{head} * kD);
      for (int i = 0; i < kD / 8; ++i) {
        const uint4 w = __ldg(src + i);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[k]));
          qsum += f.x + f.y;
        }
      }
    }
    qsum *= p.qscale;
    float ref = -INFINITY, l = 0.0f, bias = 0.0f;  // of the row; l, bias and O in units of 2^ref
    if (acc < n_acc) {
      for (uint32_t j = 0; j < n_tiles; ++j) {
        const uint32_t info = j & 3;
        uint32_t tp, n;
        walk.tile(j, &tp, &n);
        ok = __all_sync(0xFFFFFFFFu, ok && mbar_wait(&sh.s_full[acc], j & 1));
        if (!ok) break;
        fence_after();
        __syncwarp();
        // Whether all 128 rows see all 128 tokens.
        const int32_t t0 = static_cast<int32_t>(tp), acc_lo = pos_base + static_cast<int32_t>((row0 + acc * 128) / p.group);
        uint32_t any_kind = 0;
#pragma unroll
        for (int g = 0; g < kStageWarps; ++g) any_kind |= sh.kind[info][g];
        const bool masked = n < kTile || (any_kind & 4u) != 0 || t0 + 127 > acc_lo ||
                            (p.window != 0 && t0 + 128 > static_cast<int32_t>(min(p.sinks, 0x7FFFFF00u)) &&
                             p_hi - t0 >= static_cast<int32_t>(min(p.window, 0x7FFFFFFFu)));
        // ---- scores of 32 tokens from tensor memory, in pairs: S ks (+ kb sum(q)) + add
        const Pair q2 = pair(qsum, qsum), scale2 = pair(p.qscale, p.qscale);
        auto scores = [&](uint32_t c, Pair add0, Pair add1, Pair (&x)[16]) {
          uint32_t raw[32];
          tmem_load32(t_s + c * 32, raw);
          wait_ld();
          const uint32_t kind = sh.kind[info][2 * c] | sh.kind[info][2 * c + 1];
          if (kind & 3u) {
            const float4 *ks = reinterpret_cast<const float4*>(&sh.ks[info][c * 32]), *kb = reinterpret_cast<const float4*>(&sh.kb[info][c * 32]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              Pair a0 = i < 4 ? add0 : add1, a1 = a0;
              if (kind & 2u) {
                const float4 b = kb[i];
                a0 = fma2(pair(b.x, b.y), q2, a0);
                a1 = fma2(pair(b.z, b.w), q2, a1);
              }
              const float4 k = ks[i];
              x[2 * i] = fma2(pair(raw[4 * i], raw[4 * i + 1]), pair(k.x, k.y), a0);
              x[2 * i + 1] = fma2(pair(raw[4 * i + 2], raw[4 * i + 3]), pair(k.z, k.w), a1);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = fma2(pair(raw[2 * i], raw[2 * i + 1]), scale2, i < 8 ? add0 : add1);
          }
          if (masked) {
            // a bit per token: up to the row's own, and from the window's first one on or among the sinks
            const int32_t tc = t0 + static_cast<int32_t>(c) * 32;
            auto below = [](int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; };
            const uint32_t see = below(pos - tc + 1) & (~below(low - tc) | below(static_cast<int32_t>(min(p.sinks, 0x7FFFFFFFu)) - tc)) &
                                 (sh.exists[info][2 * c] | sh.exists[info][2 * c + 1] << 16);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 v = split(x[i]);
              x[i] = pair(see & 1u << (2 * i) ? v.x : -INFINITY, see & 2u << (2 * i) ? v.y : -INFINITY);
            }
          }
        };
        const Pair zero = pair(0.0f, 0.0f);
        auto rescale = [&](float f) {  // O of this tile's row, once the products before have been added to it
          if (j == 0) return true;
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(&sh.o_done[acc], (j - 1) & 1))) return false;
          fence_after();
#pragma unroll 1
          for (uint32_t c = 0; c < kD / 32; ++c) {
            uint32_t o[32];
            tmem_load32(t_o + c * 32, o);
            wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_store32(t_o + c * 32, o);
          }
          wait_st();
          return true;
        };
        // ---- weights, in one pass: 32 tokens at a time, against the row's reference so far.  A token counts by its score
        // and the exponent of its 16 tokens' value scales (its own where these lie far apart), so that a weight, the
        // exponential times the scale, is at most 2^14 where no sum passes the reference by more than kAbove.  Where one
        // does, the reference moves to kBelow under it, by a whole number, and what was made with the old one (O, the
        // sums, this tile's weights so far) is scaled by a power of two.  So the largest weight is in [2^5, 2^14] (2^-1 where
        // it is of a token whose scale is 2^6 below its neighbours'), and binary16 holds those down to 2^-19 (2^-13)
        // of it without a loss, whatever other rows and tokens hold.
        constexpr float kAbove = 14.0f, kBelow = 6.0f;
#pragma unroll 1
        for (uint32_t c = 0; c < (n + 31) / 32; ++c) {  // the products take no further tokens
          const uint32_t kind0 = sh.kind[info][2 * c], kind1 = sh.kind[info][2 * c + 1];
          const int e0 = kind0 & 3u ? sh.exponent[info][2 * c] : 0, e1 = kind1 & 3u ? sh.exponent[info][2 * c + 1] : 0;
          const float from = ref == -INFINITY ? 0.0f : ref;
          const float add0 = static_cast<float>(e0) - from, add1 = static_cast<float>(e1) - from;
          Pair x[16];
          scores(c, pair(add0, add0), pair(add1, add1), x);
          float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 u = split(x[i]), v = split(x[8 + i]);
            top0 = fmaxf(top0, fmaxf(u.x, u.y));
            top1 = fmaxf(top1, fmaxf(v.x, v.y));
          }
          float top = fmaxf(top0, top1);  // above the reference
          const float above = ref == -INFINITY ? -INFINITY : kAbove;
          if (__any_sync(0xFFFFFFFFu, top > above)) {
            if ((kind0 | kind1) & 8u) {  // each token by its own scale
              const float4* es = reinterpret_cast<const float4*>(&sh.es[info][c * 32]);
              top = -INFINITY;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 d = (i < 4 ? kind0 : kind1) & 8u ? es[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float2 u = split(x[2 * i]), v = split(x[2 * i + 1]);
                top = fmaxf(top, fmaxf(fmaxf(u.x + d.x, u.y + d.y), fmaxf(v.x + d.z, v.y + d.w)));
              }
            }
            const bool grow = top > above;
            if (__any_sync(0xFFFFFFFFu, grow)) {
              const float up = grow ? ceilf(top) - kBelow : 0.0f;
              const float a = ref == -INFINITY ? (grow ? 0.0f : 1.0f) : halvings(up);
              ok = rescale(a);
              if (!ok) break;
              if (grow) ref = from + up;
              l *= a;
              bias *= a;
              wait_st();  // this tile's weights so far: a load is ordered behind the stores before it by this alone
#pragma unroll 1
              for (uint32_t k = 0; k < c; ++k) {
                uint32_t w[16];
                tmem_load16(t_s + k * 16, w);
                wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                  w[i] = dev::pack_f16x2(v.x * a, v.y * a);
                }
                tmem_store16(t_s + k * 16, w);
              }
              const Pair down = pair(-up, -up);
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = add2(x[i], down);
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 v = split(x[i]);
            x[i] = pair(ex2(v.x), ex2(v.y));
          }
          const float back0 = pow2(-e0), back1 = pow2(-e1);  // the sums leave the exponents out
          Pair s0 = x[0], s1 = x[8];
#pragma unroll
          for (int i = 1; i < 8; ++i) {
            s0 = add2(s0, x[i]);
            s1 = add2(s1, x[8 + i]);
          }
          const float2 l0 = split(s0), l1 = split(s1);
          l = fmaf(l0.x + l0.y, back0, fmaf(l1.x + l1.y, back1, l));
          if ((kind0 | kind1) & 2u) {
            const float4* vb = reinterpret_cast<const float4*>(&sh.vb[info][c * 32]);
            Pair b0 = zero, b1 = zero;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 u = vb[i], v = vb[4 + i];
              b0 = fma2(x[2 * i + 1], pair(u.z, u.w), fma2(x[2 * i], pair(u.x, u.y), b0));
              b1 = fma2(x[2 * i + 9], pair(v.z, v.w), fma2(x[2 * i + 8], pair(v.x, v.y), b1));
            }
            const float2 y0 = split(b0), y1 = split(b1);
            bias = fmaf(y0.x + y0.y, back0, fmaf(y1.x + y1.y, back1, bias));
          }
          uint32_t w[16];
          if ((kind0 | kind1) & 3u) {
            const float4* vs = reinterpret_cast<const float4*>(&sh.vs[info][c * 32]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 v = vs[i];
              x[2 * i] = mul2(x[2 * i], pair(v.x, v.y));
              x[2 * i + 1] = mul2(x[2 * i + 1], pair(v.z, v.w));
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 v = split(x[i]);
            w[i] = dev::pack_f16x2(v.x, v.y);
          }
          tmem_store16(t_s + c * 16, w);
        }
        if (!ok) break;
        wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[acc]);
      }
      // ---- the rows' results
      if (ok && n_tiles > 0) ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sh.o_done[acc], (n_tiles - 1) & 1));
      if (ok) {
        fence_after();
        const bool none = ref == -INFINITY && l == 0.0f;
#pragma unroll 1
        for (uint32_t c = 0; c < kD / 32; ++c) {
          uint32_t o[32];
          if (n_tiles > 0) {
            tmem_load32(t_o + c * 32, o);
            wait_ld();
          }
          __syncwarp();
          if (sh.split) {
            float* dst = p.tile_partial + (uint64_t{blockIdx.x} * kRowsCta + acc * 128 + r) * (kD + 4);
            if (c == 0) *reinterpret_cast<float2*>(dst + kD) = make_float2(ref, l);
#pragma unroll
            for (int k = 0; k < 8; ++k) {  // in the order of the accumulators: join_kernel puts it right
              float4 y;
              float* x = &y.x;
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = none ? 0.0f : __uint_as_float(o[4 * k + i]) + bias;
              reinterpret_cast<float4*>(dst + c * 32)[k] = y;
            }
            continue;
          }
          uint4* dst = reinterpret_cast<uint4*>(p.out + (rows.first + tok) * p.out_stride + uint64_t{head} * kD + c * 32);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              // elements 2 i and 2 i + 1 of the 8 lie at 0 4 1 5 2 6 3 7
              const int e0 = 8 * k + (i < 2 ? 4 * i : 4 * (i - 2) + 1), e1 = e0 + 2;
              const float a = none ? 0.0f : (__uint_as_float(o[e0]) + bias) / l, b = none ? 0.0f : (__uint_as_float(o[e1]) + bias) / l;
              y[i] = dev::pack_f16x2(a, b);
            }
            if (live) dst[k] = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
      }
      fence_before();
    }
  } else if (warp < kSoftmaxWarps + kStageWarps) {
    // ================= conversion: 16 tokens of a tile per warp =================
    // A pipeline of batches of rows: the loads of a batch are issued before the one before it is converted, and the
    // next tile's blocks are looked up while this one's rows are.
    const uint32_t sw = warp - kSoftmaxWarps;
    const uint4* blocks = p.blocks + first_block;
    constexpr uint32_t kChunks = kD / 8, kRowsIter = 32 / kChunks, kIters = 16 / kRowsIter;  // 16-byte pieces of an operand's row
    constexpr uint32_t kBatch = 4, kBatches = kIters / kBatch;                               // of a half: 2 or 1
    const uint32_t chunk = lane % kChunks, sub = lane / kChunks;

    // A lane's token of a tile (lanes 16 to 31 repeat 0 to 15).
    struct Token {
      uint64_t k;     // address of its K row
      uint32_t f;     // 4: it does not exist
      float2 kp, vp;  // its rows' {scale, bias}
      uint64_t first;  // all 16 in one block: address of the first one's K row,
      uint32_t step;   // and bytes from a token's row to the next one's (0: they are not)
    };
    uint32_t cur = 0, cur_start = 0;  // a block at or before this warp's next first token, and its first position
    uint32_t at_k = 0;                // the block that `entry` is
    uint4 entry = make_uint4(0u, 0u, 0u, 0u);
    auto position = [&](uint32_t j, uint32_t* t) {
      uint32_t tp, n;
      walk.tile(j, &tp, &n);
      const uint32_t i = sw * 16 + (lane & 15);
      *t = tp + i;
      return i < n;
    };
    // First half of the lookup for tile j: the block that holds the token if those since `cur` are full.
    auto look = [&](uint32_t j) {
      uint32_t t;
      const bool in = position(j, &t);
      if (walk.begins(j)) {  // a run begins: the last block that starts at or before the first token
        const uint32_t first = __shfl_sync(0xFFFFFFFFu, t, 0);
        uint32_t a = 0, b = n_blocks;
        while (b - a > 1) {
          const uint32_t step = (b - a + 31) / 32, k = a + lane * step;
          const uint32_t hits = __popc(__ballot_sync(0xFFFFFFFFu, k < b && __ldg(&blocks[k].w) <= first));
          const uint32_t at = a + (hits > 0 ? hits - 1 : 0u) * step;
          b = min(at + step, b);
          a = at;
        }
        cur = a;
        cur_start = __ldg(&blocks[a].w);
      }
      at_k = cur + (t > cur_start ? (t - cur_start) / p.T : 0u);
      if (in && at_k < n_blocks) entry = __ldg(blocks + at_k);
    };
    // Second half: partly filled blocks put the token further on.
    auto find = [&](uint32_t j) {
      uint32_t t;
      Token tok;
      tok.f = 4;
      tok.k = 0;
      tok.kp = tok.vp = make_float2(1.0f, 0.0f);
      if (position(j, &t)) {
        while (at_k < n_blocks && t >= entry.w && t - entry.w >= min((entry.y >> 10) & 0x3FFu, p.T)) {
          if (++at_k < n_blocks) entry = __ldg(blocks + at_k);
        }
        if (at_k < n_blocks && t >= entry.w) {  // else not listed
          const uint8_t* payload = nullptr;
          tok.f = open_block(p, entry, &payload);
          if (tok.f <= 3) {
            const uint32_t row = (t - entry.w) * p.H + h;
            tok.k = reinterpret_cast<uint64_t>(payload) + uint64_t{row} * (tok.f == dev::kFp16 ? kD * 2 : tok.f == dev::kInt4 ? kD / 2 : kD);
            tok.kp = params_of_row(tok.f, entry.y, entry.z, payload + p.code_bytes[tok.f], row);
            tok.vp = params_of_row(tok.f, entry.y, entry.z, payload + p.code_bytes[tok.f], row + p.T * p.H);
            if (tok.f != dev::kFp16 && tok.f != dev::kInt4 && ((entry.y >> 4) & 3u) == 0 && tok.vp.x == 1.0f) {
              // What encoders store for an FP8 row of zeros: a size that its values do not have.
              if (zero_row(payload + (uint64_t{row} + uint64_t{p.T} * p.H) * kD, kD)) tok.vp.x = 0.0f;
            }
          }
        }
      }
      const uint32_t rb = tok.f == dev::kFp16 ? kD * 2 : tok.f == dev::kInt4 ? kD / 2 : kD;
      tok.first = __shfl_sync(0xFFFFFFFFu, tok.k, 0);
      const uint32_t k0 = __shfl_sync(0xFFFFFFFFu, at_k, 0), w0 = __shfl_sync(0xFFFFFFFFu, entry.w, 0);
      tok.step = __all_sync(0xFFFFFFFFu, tok.f <= 3 && at_k == k0) ? p.H * rb : 0u;
      if (k0 < n_blocks) {
        cur = k0;
        cur_start = w0;
      }
      return tok;
    };
    uint4 raw[2][kBatch];
    uint32_t fr[2][kBatch];
    // Batch b of a tile: of its K half, then of its V half.
    auto load = [&](const Token& tok, uint32_t b, uint4 (&r)[kBatch], uint32_t (&fs)[kBatch]) {
      const uint32_t half = b / kBatches, it0 = b % kBatches * kBatch;
      if (tok.step != 0) {  // 16 rows of one block: equally far apart
        const uint64_t a = tok.first + (half ? uint64_t{tok.step} * p.T : 0u) + uint64_t{it0 * kRowsIter + sub} * tok.step;
        const uint32_t step = kRowsIter * tok.step;
        if (tok.f == dev::kFp16) {
#pragma unroll
          for (uint32_t it = 0; it < kBatch; ++it) r[it] = __ldg(reinterpret_cast<const uint4*>(a + it * step) + chunk);
        } else if (tok.f == dev::kInt4) {
#pragma unroll
          for (uint32_t it = 0; it < kBatch; ++it) r[it].x = __ldg(reinterpret_cast<const uint32_t*>(a + it * step) + chunk);
        } else {
#pragma unroll
          for (uint32_t it = 0; it < kBatch; ++it) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(a + it * step) + chunk);
            r[it].x = w.x;
            r[it].y = w.y;
          }
        }
        return;
      }
      const uint64_t row_bytes = tok.f == dev::kFp16 ? kD * 2 : tok.f == dev::kInt4 ? kD / 2 : kD;
      const uint64_t src = tok.k + (half ? row_bytes * p.T * p.H : 0u);
#pragma unroll
      for (uint32_t it = 0; it < kBatch; ++it) {
        const uint32_t from = (it0 + it) * kRowsIter + sub;
        const uint64_t a = __shfl_sync(0xFFFFFFFFu, src, from);
        fs[it] = __shfl_sync(0xFFFFFFFFu, tok.f, from);
        r[it] = make_uint4(0u, 0u, 0u, 0u);
        if (fs[it] == dev::kFp16) r[it] = __ldg(reinterpret_cast<const uint4*>(a) + chunk);
        else if (fs[it] == dev::kInt4) r[it].x = __ldg(reinterpret_cast<const uint32_t*>(a) + chunk);
        else if (fs[it] < 4) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(a) + chunk);
          r[it].x = w.x;
          r[it].y = w.y;
        }
      }
    };
    bool bad = false, part = false;
    auto store = [&](uint32_t j, uint32_t b, bool even, uint32_t f, const uint4 (&r)[kBatch], const uint32_t (&fs)[kBatch]) {
      const uint32_t half = b / kBatches, it0 = b % kBatches * kBatch;
      const uint32_t operand = base + (half ? C::kV : C::kK) + (j & 1) * C::kOperand;
      if (even && !(half && part)) {
        auto all = [&](auto format) {
          constexpr uint32_t kF = decltype(format)::value;
#pragma unroll
          for (uint32_t it = 0; it < kBatch; ++it) {
            const uint4 v = half ? convert<true>(kF, r[it]) : convert<false>(kF, r[it]);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(operand, sw * 16 + (it0 + it) * kRowsIter + sub, chunk)),
                         "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                         : "memory");
          }
        };
        if (f == dev::kFp16) all(Format<dev::kFp16>{});
        else if (f == dev::kE4M3) all(Format<dev::kE4M3>{});
        else if (f == dev::kE5M2) all(Format<dev::kE5M2>{});
        else all(Format<dev::kInt4>{});
        return;
      }
#pragma unroll
      for (uint32_t it = 0; it < kBatch; ++it) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t ft = even ? f : fs[it];
        if (ft < 4) v = half ? convert<true>(ft, r[it]) : convert<false>(ft, r[it]);
        if (half && part) bad = bad || has_nonfinite(v.x) || has_nonfinite(v.y) || has_nonfinite(v.z) || has_nonfinite(v.w);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(chunk_at(operand, sw * 16 + (it0 + it) * kRowsIter + sub, chunk)), "r"(v.x),
                     "r"(v.y), "r"(v.z), "r"(v.w)
                     : "memory");
      }
    };
    Token tok;
    if (n_tiles > 0) {
      look(0);
      tok = find(0);
      load(tok, 0, raw[0], fr[0]);
    }
    for (uint32_t j = 0; j < n_tiles; ++j) {
      Token next = tok;
      // ---- what the softmax needs of the tokens
      uint32_t tp, n;
      walk.tile(j, &tp, &n);
      const uint32_t i = sw * 16 + (lane & 15), f = tok.f;
      const uint32_t kinds = __reduce_or_sync(0xFFFFFFFFu, f > 3 ? 4u : f == dev::kInt4 ? 3u : f == dev::kFp16 ? 0u : 1u);
      const uint32_t exists = __ballot_sync(0xFFFFFFFFu, f <= 3) & 0xFFFFu;
      const bool scaled = (kinds & 3u) != 0;
      const float unit = f == dev::kFp16 ? 1.0f : f == dev::kE4M3 ? 0x1p8f : f == dev::kE5M2 ? 0x1p15f : 8.0f;
      const float u = f > 3 ? 0.0f : tok.vp.x * unit;
      const uint32_t ub = __float_as_uint(u) & 0x7FFFFFFFu;
      // The 16 tokens' exponent is that of their largest scale.  Where others, zeros among them, lie more than 2^6 below
      // it, each token counts in the reference by its own (2^-100 of the largest at least: the exponentials, of up to
      // 2^113 then, and their sums stay in binary32's range).
      const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, ub < 0x7F800000u ? ub : 0u);
      const bool apart = __any_sync(0xFFFFFFFFu, f <= 3 && ub < 0x7F800000u && top > ub + (6u << 23));
      auto exponent_of = [](uint32_t bits) { return min(max(static_cast<int>(bits >> 23) - 127, -60), 60); };
      const int e = exponent_of(top), below = ub < 0x7F800000u ? max(exponent_of(ub) - e, -100) : 0;
      // A tile that some row sees in part: values that are not finite would touch rows that do not see them.  Such a
      // CTA's rows are done over, one by one (four chunks of 1000 tokens, all rows: 260 ms instead of 0.75).
      const int32_t t0 = static_cast<int32_t>(tp);
      part = n < kTile || t0 + 127 > p_lo ||
             (p.window != 0 && t0 + 128 > static_cast<int32_t>(min(p.sinks, 0x7FFFFF00u)) &&
              p_hi - t0 >= static_cast<int32_t>(min(p.window, 0x7FFFFFFFu)));
      bad = bad || (part && f <= 3 && (ub >= 0x7F800000u || !dev::finite_f32(tok.vp.y)));
      const bool more = j + 1 < n_tiles;
      if (more) look(j + 1);
#pragma unroll
      for (uint32_t b = 0; b < 2 * kBatches; ++b) {
        const uint32_t half = b / kBatches;
        // the next batch's loads
        if (b + 1 < 2 * kBatches) {
          load(tok, b + 1, raw[(b + 1) & 1], fr[(b + 1) & 1]);
        } else if (more) {
          next = find(j + 1);
          load(next, 0, raw[(b + 1) & 1], fr[(b + 1) & 1]);
        }
        if (b % kBatches == 0) {
          if (j >= 2) ok = ok && mbar_wait(half ? &sh.v_empty[j & 1] : &sh.k_empty[j & 1], (j / 2 - 1) & 1);
          if (!ok) break;
          if (half == 0 && lane < 16) {
            const uint32_t info = j & 3;
            sh.ks[info][i] = f > 3 ? 0.0f : tok.kp.x * (p.qscale * (f == dev::kInt4 ? 8.0f : 1.0f));
            sh.kb[info][i] = f == dev::kInt4 ? fmaf(8.0f, tok.kp.x, tok.kp.y) : 0.0f;
            sh.vs[info][i] = scaled ? u * pow2(-e) : 1.0f;
            if (apart) sh.es[info][i] = static_cast<float>(below);
            sh.vb[info][i] = f == dev::kInt4 ? fmaf(8.0f, tok.vp.x, tok.vp.y) : 0.0f;
            if (lane == 0) {
              sh.kind[info][sw] = kinds | (apart ? 8u : 0u);
              sh.exists[info][sw] = exists;
              sh.exponent[info][sw] = e;
            }
          }
        }
        store(j, b, tok.step != 0, tok.f, raw[b & 1], fr[b & 1]);
        if (b % kBatches == kBatches - 1) {
          dev::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(half ? &sh.v_full[j & 1] : &sh.k_full[j & 1]);
        }
      }
      tok = next;
      if (!ok) break;
    }
    if (bad) sh.redo = 1;
  } else if (warp == kSoftmaxWarps + kStageWarps) {
    // ================= products: one thread =================
    if (lane == 0 && n_tiles > 0) {
      constexpr uint32_t kIdS = instruction(kTile, false), kIdO = instruction(kD, true);
      auto scores = [&](uint32_t acc, uint32_t j) {
        const uint32_t q = base + C::kQ + acc * C::kOperand, k = base + C::kK + (j & 1) * C::kOperand;
#pragma unroll
        for (uint32_t s = 0; s < kD / 16; ++s) {
          const uint32_t at = (s / 4) * C::kPanel + (s % 4) * 32;
          mma_ss(tmem + acc * 128, desc(q + at, 16, 1024), desc(k + at, 16, 1024), kIdS, s > 0);
        }
        commit(&sh.s_full[acc]);
      };
      ok = mbar_wait(&sh.k_full[0], 0);
      fence_after();
      for (uint32_t acc = 0; acc < n_acc && ok; ++acc) scores(acc, 0);
      if (ok) commit(&sh.k_empty[0]);
      for (uint32_t j = 0; j < n_tiles && ok; ++j) {
        for (uint32_t acc = 0; acc < n_acc && ok; ++acc) {
          ok = mbar_wait(&sh.p_full[acc], j & 1) && (acc > 0 || mbar_wait(&sh.v_full[j & 1], (j >> 1) & 1));
          if (!ok) break;
          fence_after();
          const uint32_t v = base + C::kV + (j & 1) * C::kOperand;
          uint32_t tp, n;
          walk.tile(j, &tp, &n);
          const uint32_t steps = (n + 31) / 32 * 2;
#pragma unroll
          for (uint32_t s = 0; s < kTile / 16; ++s) {
            if (s < steps) mma_ts(tmem + 256 + acc * kD, tmem + acc * 128 + s * 8, desc(v + s * 2048, C::kPanel, 1024), kIdO, j > 0 || s > 0);
          }
          commit(&sh.o_done[acc]);
          if (j + 1 < n_tiles) {
            if (acc == 0) ok = mbar_wait(&sh.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1);
            if (!ok) break;
            fence_after();
            scores(acc, j + 1);
          }
        }
        if (!ok) break;
        commit(&sh.v_empty[j & 1]);
        if (j + 1 < n_tiles) commit(&sh.k_empty[(j + 1) & 1]);
      }
    }
    __syncwarp();
  }
  if (!ok && lane == 0) atomicOr(p.err, dev::kErrInternal);
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kSoftmaxWarps + kStageWarps) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  if (sh.split) {
    if (threadIdx.x == 0) p.tile_redo[blockIdx.x] = sh.redo;
  } else if (sh.redo) {
    for (uint32_t r = warp; r < rows_here; r += kThreads / 32) {
      const uint32_t row = row0 + r, tok = row / p.group;
      attend_row<kD>(p, seq, rows.first + tok, int64_t{pos_base} + tok, h * p.group + row % p.group);
    }
  }
}

// Joins the parts of split row tiles: a CTA for 16 rows of a (row tile, head), a warp for a row at a time.  Rows of which
// some part asks for it are done over, token by token.
constexpr uint32_t kJoinWarps = 8, kJoinRows = 16;
template <int kD>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ Params p) {
  constexpr int kPer = kD / 32;
  __shared__ RowTile s_mine;
  __shared__ uint32_t s_n, s_splits;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr uint32_t kGroups = kRowsCta / kJoinRows;
  const uint32_t unit = blockIdx.x / kGroups, rank = unit / p.H, h = unit % p.H;
  if (warp == 0) {  // of the plan, which is older than the kernel before
    const uint32_t n = count_row_tiles(p), splits = splits_of(p, n);
    RowTile mine{0u, 0xFFFFFFFFu};
    if (splits > 1 && rank < n) mine = row_tile_of_rank(p, rank);
    if (lane == 0) {
      s_mine = mine;
      s_n = n;
      s_splits = splits;
    }
  }
  __syncthreads();
  dev::wait_for_prerequisites();
  const RowTile mine = s_mine;
  if (mine.tile == 0xFFFFFFFFu) return;
  const Rows rows = rows_of(p, mine.seq);
  const uint32_t n_rows = rows.q * p.group, row0 = mine.tile * kRowsCta, rows_here = min(kRowsCta, n_rows - row0);
  const int32_t base = static_cast<int32_t>(p.context[mine.seq]) - static_cast<int32_t>(rows.q);
  uint32_t first_block;
  const uint32_t n_blocks = count_of(p, mine.seq, &first_block);
  const uint32_t parts =
      parts_of(s_splits, walk_of(p, n_blocks, position_of(p, base, row0), position_of(p, base, row0 + rows_here - 1)).tiles());
  if (parts == 1) return;  // written already
  // CTA (part, rank, head) of the tile kernel
  auto slot = [&](uint32_t part) { return (uint64_t{part} * s_n + rank) * p.H + h; };
  uint32_t redo = 0;
  for (uint32_t k = 0; k < parts; ++k) redo |= p.tile_redo[slot(k)];
  for (uint32_t r = blockIdx.x % kGroups * kJoinRows + warp; r < (blockIdx.x % kGroups + 1) * kJoinRows && r < rows_here; r += kJoinWarps) {
    const uint32_t row = row0 + r, tok = row / p.group, head = h * p.group + row % p.group;
    if (redo != 0) {
      attend_row<kD>(p, mine.seq, rows.first + tok, int64_t{base} + tok, head);
      continue;
    }
    float M = -INFINITY, L = 0.0f, o[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = 0.0f;
#pragma unroll 4
    for (uint32_t k = 0; k < parts; ++k) {
      const float* src = p.tile_partial + (slot(k) * kRowsCta + r) * (kD + 4);
      const float2 ml = *reinterpret_cast<const float2*>(src + kD);
      const float m = fmaxf(M, ml.x);
      const float fo = m == -INFINITY ? 1.0f : exp2f(M - m), ft = m == -INFINITY ? 1.0f : exp2f(ml.x - m);
      M = m;
      L = fmaf(L, fo, ml.y * ft);
#pragma unroll
      for (int i = 0; i < kPer; ++i) o[i] = fmaf(o[i], fo, src[i * 32 + lane] * ft);
    }
    if (L == 0.0f && M == -INFINITY) L = 1.0f;  // sees nothing: zeros
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      // place x of a chunk of 8 is element (x / 2) + 4 (x % 2)
      const uint32_t at = i * 32 + lane, x = at & 7, e = (at & ~7u) + (x >> 1) + 4 * (x & 1);
      p.out[(rows.first + tok) * p.out_stride + uint64_t{head} * kD + e] = __half_as_ushort(__float2half_rn(o[i] / L));
    }
  }
}

template <int kD>
cudaError_t launch(const Params& p, cudaStream_t s) {
  static SharedMemoryOnce once;
  const cudaError_t e = once.allow(reinterpret_cast<const void*>(tile_kernel<kD>), Config<kD>::kSmem);
  if (e != cudaSuccess) return e;
  tile_kernel<kD><<<static_cast<unsigned>(tile_ctas(p)), kThreads, Config<kD>::kSmem, s>>>(p);
  const cudaError_t e2 = cudaGetLastError();
  if (e2 != cudaSuccess || p.nseq > kOrdered) return e2;
  // Rows that see so few tokens (at most a tile more for each of the walk's two runs) are not split: no join.
  uint64_t most = uint64_t{p.block_cap} * p.T;
  if (p.window != 0) most = std::min(most, uint64_t{p.window} + p.sinks + kRowsCta / p.group + 1);
  if (most / kTile + 2 < 2 * kSplitTiles) return e2;
  // At most half as many (row tile, head) as the GPU has SMs are split.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.ctas / 2 * (kRowsCta / kJoinRows));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_kernel<kD>, p);
}

}  // namespace

// A tile for each 256 rows that every sequence may have.
uint64_t tiles_of_plan(const Params& p) { return uint64_t{p.nseq} * ((uint64_t{p.max_rows} + kRowsCta - 1) / kRowsCta); }
// CTAs that take ranks need be no more than the batch's tokens can make: whole tiles, and one more for each sequence of
// more than kStreamRows rows.
uint64_t tiles_of_tokens(const Params& p) {
  const uint64_t rows = uint64_t{p.token_cap} * p.group;
  return rows / kRowsCta + std::min<uint64_t>(p.nseq, rows / (kStreamRows + 1));
}

// Past kOrdered sequences a CTA for each tile of the plan needs no look-up, and a plan whose sequences may have many
// more rows than its tokens make is taken by ranks.  (250 sequences of up to 300 new tokens: 4421 us in a plan for 300 new
// tokens each, without ranks; in one for 8192, 5955 us without and 4578 with them.  129 sequences of one new token
// in that plan: 934 and 60 us.)
uint32_t tile_ranks(const Params& p) {
  if (p.nseq <= kOrdered || tiles_of_plan(p) <= 2 * tiles_of_tokens(p)) return 0;
  return static_cast<uint32_t>(std::max<uint64_t>(tiles_of_tokens(p), 1));
}

uint64_t tile_ctas(const Params& p) {
  if (p.nseq > kOrdered) return (p.tile_ranks != 0 ? p.tile_ranks : tiles_of_plan(p)) * p.H;
  const uint64_t tiles = std::min(tiles_of_plan(p), tiles_of_tokens(p));
  return tiles == 0 ? 0u : std::max<uint64_t>(tiles * p.H, p.ctas);  // (parts of few)
}
size_t tile_workspace(uint32_t nseq, uint32_t head_dim, uint32_t max_rows, uint32_t ctas) {
  if (max_rows <= kStreamRows || nseq > kOrdered) return 0;
  return size_t{ctas} * kRowsCta * (head_dim + 4) * sizeof(float) + size_t{ctas} * sizeof(uint32_t);
}

cudaError_t launch_tiles(uint32_t head_dim, const Params& p, cudaStream_t s) {
  return head_dim == 64 ? launch<64>(p, s) : launch<128>(p, s);
}

}  // namespace battn
}  // namespace hlkv
