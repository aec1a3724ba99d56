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
  const uint32_t max_rows = static_cast<uint32_t>(rows < 0xFFFFFFFFu ? rows : 0xFFFFFFFFu);
  const uint32_t ctas = static_cast<uint32_t>(hlkv::sm_count());
  return hlkv::battn::stream_workspace(plan->nseq, layout->kv_heads, layout->head_dim, max_rows, ctas) +
         hlkv::battn::tile_workspace(plan->nseq, layout->head_dim, max_rows, ctas);
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
  if (H > kMaxKvHeads || q_heads == 0 || q_heads % H != 0 || q_heads / H > kMaxGroup) return HLKV_INVALID_ARGUMENT;
  if (!(softmax_scale > 0.0f) || softmax_scale > 0x1p60f) return HLKV_INVALID_ARGUMENT;
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
  p.max_query = plan->max_query;
  const uint64_t max_rows = uint64_t{plan->max_query} * p.group;
  p.max_rows = static_cast<uint32_t>(max_rows < 0xFFFFFFFFu ? max_rows : 0xFFFFFFFFu);
  p.qscale = softmax_scale * kLog2e;
  p.ctas = static_cast<uint32_t>(sm_count());
  stream_layout(&p, d_workspace);
  // behind the stream kernel's part, a multiple of 16 bytes
  p.tile_partial = reinterpret_cast<float*>(static_cast<uint8_t*>(d_workspace) +
                                            stream_workspace(p.nseq, H, layout->head_dim, p.max_rows, p.ctas));
  p.tile_redo = reinterpret_cast<uint32_t*>(p.tile_partial + uint64_t{p.ctas} * 256 * (D + 4));
  p.tile_ranks = tile_ranks(p);
  const uint64_t tiles = p.max_rows <= kStreamRows ? 0u : tile_ctas(p);
  if (tiles > 0x7FFFFFFFull || (p.tile_ranks != 0 && tiles_of_plan(p) * H > 0x7FFFFFFFull)) return HLKV_INVALID_ARGUMENT;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_stream(layout->head_dim, p, s);
  if (e != cudaSuccess || tiles == 0) return cuda_status(e);
  return cuda_status(launch_tiles(layout->head_dim, p, s));
}
