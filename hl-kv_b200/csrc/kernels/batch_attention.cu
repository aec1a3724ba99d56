// Batch attention: the new tokens of a plan's sequences attend to the sequences' cached tokens,
// read from the quantized blocks.
//
// For query row (token at position p, head qh) over the tokens t that it sees (t <= p, and inside
// the window or one of the sinks):
//   x_t = softmax_scale log2(e) <q, k_t>,  m = max x_t,  out = sum 2^(x_t - m) v_t / sum 2^(x_t - m),
// in one pass with a running maximum.  k_t and v_t are the values of the codes under their
// parameters, in binary32.
#include <cmath>

#include "batch_attention.cuh"

namespace hlkv {
namespace battn {
namespace {

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

__device__ __forceinline__ float2 row_params(uint32_t f, uint32_t info, uint32_t sref, const uint8_t* params, uint32_t row) {
  if (f == dev::kFp16) return make_float2(1.0f, 0.0f);
  const uint32_t mode = (info >> 4) & 3u;
  if (mode != 0) return dev::block_params_value(mode, sref);
  if (f == dev::kInt4) return __ldg(reinterpret_cast<const float2*>(params) + row);
  return make_float2(__ldg(reinterpret_cast<const float*>(params) + row), 0.0f);
}

constexpr int kRowThreads = 128;

// One warp per (new token, query head); lane l holds elements [l kN, (l + 1) kN) of the head.
template <int kD>
__global__ void __launch_bounds__(kRowThreads) batch_attention_rows(const Params p) {
  constexpr int kN = kD / 32;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t id = uint64_t{blockIdx.x} * (kRowThreads / 32) + (threadIdx.x >> 5);
  const uint32_t token = static_cast<uint32_t>(id / p.q_heads), qh = static_cast<uint32_t>(id % p.q_heads), h = qh / p.group;
  if (token >= p.token_first[p.nseq]) return;
  uint32_t lo = 0, hi = p.nseq;  // the sequence with token_first[lo] <= token < token_first[lo + 1]
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (p.token_first[mid] <= token) lo = mid; else hi = mid;
  }
  const uint32_t q_len = p.token_first[lo + 1] - p.token_first[lo], ctx = p.context[lo];
  if (uint64_t{q_len} * p.group <= kStreamRows) return;  // the stream kernel's
  const int64_t pos = int64_t{ctx} - q_len + (token - p.token_first[lo]);

  float q[kN], acc[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    q[i] = __half2float(__ushort_as_half(p.q[token * p.q_stride + uint64_t{qh} * kD + lane * kN + i])) * p.qscale;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  uint32_t first;
  const uint32_t count = count_of(p, lo, &first);
  for (uint32_t j = 0; j < count; ++j) {
    const uint4 b = __ldg(p.blocks + first + j);
    const uint32_t vt = min((b.y >> 10) & 0x3FFu, p.T);
    const uint8_t* payload;
    const uint32_t f = open_block(p, b, &payload);
    if (f > 3) continue;
    for (uint32_t i = 0; i < vt; ++i) {
      const int64_t t = int64_t{b.w} + i;
      if (t > pos || (p.window != 0 && pos - t >= p.window && t >= p.sinks)) continue;
      float k[kN], v[kN];
      const uint32_t krow = i * p.H + h, vrow = krow + p.T * p.H;
      load_codes<kN>(f, payload, uint64_t{krow} * kD + lane * kN, k);
      load_codes<kN>(f, payload, uint64_t{vrow} * kD + lane * kN, v);
      const float2 kp = row_params(f, b.y, b.z, payload + p.code_bytes[f], krow);
      const float2 vp = row_params(f, b.y, b.z, payload + p.code_bytes[f], vrow);
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace battn
}  // namespace hlkv

extern "C" size_t hlkv_batch_attention_workspace_bytes(const HlkvBatchPlan* plan, const HlkvLayout* layout,
                                                       uint32_t q_heads) {
  if (plan == nullptr || layout == nullptr || plan->nseq == 0 || plan->token_cap == 0 || layout->kv_heads == 0 ||
      q_heads < layout->kv_heads || (layout->head_dim != 64 && layout->head_dim != 128)) {
    return 0;
  }
  const uint64_t rows = uint64_t{plan->max_query} * (q_heads / layout->kv_heads);
  return hlkv::battn::stream_workspace(plan->nseq, layout->kv_heads, layout->head_dim,
                                       static_cast<uint32_t>(rows < 0xFFFFFFFFu ? rows : 0xFFFFFFFFu),
                                       static_cast<uint32_t>(hlkv::sm_count()));
}

extern "C" int hlkv_batch_attention(const HlkvPools* pools, const HlkvLayout* layout, const HlkvBatchPlan* plan,
                                    const uint16_t* d_q, uint32_t q_heads, uint64_t q_stride, float softmax_scale,
                                    void* d_workspace, size_t workspace_bytes, uint16_t* d_out, uint64_t out_stride,
                                    uint32_t* d_err, hlkv_stream_t stream) {
  using namespace hlkv;
  using namespace hlkv::battn;
  if (pools == nullptr || plan == nullptr || !layout_ok(layout) || d_err == nullptr) return HLKV_INVALID_ARGUMENT;
  const uint64_t D = layout->head_dim;
  if (D != 64 && D != 128) return HLKV_INVALID_ARGUMENT;
  const uint32_t H = layout->kv_heads;
  if (q_heads == 0 || q_heads % H != 0 || q_heads / H > kMaxGroup) return HLKV_INVALID_ARGUMENT;
  if (!(softmax_scale > 0.0f) || !std::isfinite(softmax_scale)) return HLKV_INVALID_ARGUMENT;
  if (plan->nseq == 0 || plan->token_cap == 0) return HLKV_OK;
  if (plan->d_block_first == nullptr || plan->d_block_count == nullptr || plan->d_token_first == nullptr ||
      plan->d_context == nullptr || plan->d_cost == nullptr ||
      (plan->block_cap > 0 && (plan->d_blocks == nullptr || plan->d_block_cost == nullptr)) || !aligned16(plan->d_blocks) ||
      plan->max_query == 0 || d_q == nullptr || d_out == nullptr || !aligned16(d_q) || !aligned16(d_out) ||
      q_stride % 8 != 0 || out_stride % 8 != 0 || q_stride < q_heads * D || out_stride < q_heads * D) {
    return HLKV_INVALID_ARGUMENT;
  }
  const size_t need = hlkv_batch_attention_workspace_bytes(plan, layout, q_heads);
  if (need > 0) {
    if (d_workspace == nullptr || !aligned16(d_workspace)) return HLKV_INVALID_ARGUMENT;
    if (workspace_bytes < need) return HLKV_BUFFER_TOO_SMALL;
  }
  Params p{};
  const uint64_t elems = uint64_t{2} * layout->block_tokens * H * D;
  for (int f = 0; f < 4; ++f) {
    const HlkvPool& q = pools->pool[f];
    p.code_bytes[f] = layout_code_bytes(f, elems);
    if (q.base == nullptr || q.num_slots == 0) continue;
    if (!aligned16(q.base) || (q.slot_bytes & 15u) != 0 || q.slot_bytes < hlkv_layout_slot_bytes(f, layout)) {
      return HLKV_INVALID_ARGUMENT;
    }
    p.pool[f] = DevPool{static_cast<const uint8_t*>(q.base), q.slot_bytes, q.num_slots};
  }
  const uint64_t rows = uint64_t{plan->token_cap} * q_heads;
  if (rows > 0x7FFFFFFFull || uint64_t{plan->nseq} * H * kStreamRows > 0x7FFFFFFFull) return HLKV_INVALID_ARGUMENT;
  p.block_first = plan->d_block_first;
  p.block_count = plan->d_block_count;
  p.token_first = plan->d_token_first;
  p.context = plan->d_context;
  p.blocks = reinterpret_cast<const uint4*>(plan->d_blocks);
  p.q = d_q;
  p.out = d_out;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.err = d_err;
  p.nseq = plan->nseq;
  p.T = layout->block_tokens;
  p.H = H;
  p.q_heads = q_heads;
  p.group = q_heads / H;
  p.window = plan->window;
  p.sinks = plan->sinks;
  p.block_cap = plan->block_cap;
  p.block_cost = plan->d_block_cost;
  p.cost = plan->d_cost;
  p.token_cap = plan->token_cap;
  const uint64_t max_rows = uint64_t{plan->max_query} * p.group;
  p.max_rows = static_cast<uint32_t>(max_rows < 0xFFFFFFFFu ? max_rows : 0xFFFFFFFFu);
  p.qscale = softmax_scale * kLog2e;
  p.ctas = static_cast<uint32_t>(sm_count());
  stream_layout(&p, d_workspace);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_stream(layout->head_dim, p, s);
  if (e != cudaSuccess || p.max_rows <= kStreamRows) return cuda_status(e);
  const unsigned grid = static_cast<unsigned>((rows + kRowThreads / 32 - 1) / (kRowThreads / 32));
  if (D == 64) batch_attention_rows<64><<<grid, kRowThreads, 0, s>>>(p);
  else batch_attention_rows<128><<<grid, kRowThreads, 0, s>>>(p);
  return cuda_status(cudaGetLastError());
}
