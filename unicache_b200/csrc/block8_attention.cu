// Attention over the 8-bit block cache (ucb_block8_attention).
#include "block8.cuh"

namespace ucb {
namespace block8 {
namespace {

struct AttnParams {
  ucb_block8_cache c;
  const void* q;
  int64_t q_ss, q_sl, q_sh;
  int queries, q_heads;
  const int32_t* blocks;
  int selected;
  float scale;
  void* out;
  float* lse;
  unsigned int* err;
};

// One warp per query row, one token at a time.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_rows_kernel(const AttnParams p) {
  constexpr int PER = D / 32;
  const ucb_block8_cache& c = p.c;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)c.num_seqs * p.queries * p.q_heads) return;
  const int qh = (int)(row % p.q_heads);
  const int l = (int)(row / p.q_heads % p.queries);
  const int s = (int)(row / p.q_heads / p.queries);
  const int h = qh / (p.q_heads / c.kv_heads);
  const T* q = static_cast<const T*>(p.q) + s * p.q_ss + l * p.q_sl + qh * p.q_sh;
  float qv[PER], o[PER];
  for (int i = 0; i < PER; ++i) qv[i] = Dtype<T>::to_f(q[lane * PER + i]), o[i] = 0.f;
  const int limit = held_tokens(c, s, p.err) - p.queries + l + 1;  // tokens this row sees
  const int count = p.blocks ? p.selected : (max(limit, 0) + c.block_tokens - 1) / c.block_tokens;
  float m = -INFINITY, sum = 0.f;
  for (int k = 0; k < count; ++k) {
    const int j = p.blocks ? p.blocks[((int64_t)s * c.kv_heads + h) * p.selected + k] : k;
    if (j < 0 || j >= c.max_blocks) continue;
    const int n = min(c.block_tokens, limit - j * c.block_tokens);
    if (n <= 0) continue;
    const int64_t block = pool_block(c, s, j, p.err);
    if (block < 0) continue;
    const int64_t at = (block * c.kv_heads + h) * c.block_tokens * D + lane * PER;
    const float ks = c.key_scale[block * c.kv_heads + h] * p.scale, vs = c.value_scale[block * c.kv_heads + h];
    for (int t = 0; t < n; ++t) {
      float x = 0.f;
      for (int i = 0; i < PER; ++i) x = fmaf(qv[i], (float)c.key_code[at + t * D + i], x);
      for (int k2 = 16; k2 > 0; k2 >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k2);
      x *= ks;
      const float top = fmaxf(m, x), keep = m == -INFINITY ? 0.f : expf(m - top);
      const float w = x == -INFINITY ? 0.f : expf(x - (top == -INFINITY ? 0.f : top));
      sum = sum * keep + w;
      for (int i = 0; i < PER; ++i) o[i] = o[i] * keep + w * vs * (float)c.value_code[at + t * D + i];
      m = top;
    }
  }
  T* out = static_cast<T*>(p.out) + row * D + lane * PER;
  for (int i = 0; i < PER; ++i) out[i] = Dtype<T>::from_f(sum == 0.f ? 0.f : o[i] / sum);
  if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + logf(sum);
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

extern "C" int64_t ucb_block8_attention_workspace_bytes(const ucb_block8_cache* cache, int queries, int q_heads) {
  return b8::check_cache(cache, "ucb_block8_attention_workspace_bytes") || queries < 1 || q_heads < 1 ? -1 : 0;
}

extern "C" int ucb_block8_attention(const ucb_block8_cache* cache, const void* query, int64_t q_ss, int64_t q_sl,
                                    int64_t q_sh, int queries, int q_heads, const int32_t* blocks, int num_selected,
                                    float softmax_scale, void* out, float* lse, void* workspace, void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_attention")) return rc;
  if (!query || !out) return set_error(UCB_ERR_INVALID, "ucb_block8_attention: null pointer");
  if (queries < 1 || queries > 16) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_attention: 1 to 16 query tokens");
  if (q_heads < 1 || q_heads % cache->kv_heads)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: query heads must be divisible by KV heads");
  if (blocks && num_selected < 1)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: a selection needs at least one entry");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_block8_attention: device error word unavailable");
  const b8::AttnParams p{*cache, query, q_ss, q_sl, q_sh, queries, q_heads, blocks, num_selected, softmax_scale, out, lse, err};
  const int64_t rows = (int64_t)cache->num_seqs * queries * q_heads;
  const unsigned grid = (unsigned)((rows + 3) / 4);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == UCB_BF16;
  if (cache->head_dim == 128) {
    if (bf) b8::attention_rows_kernel<__nv_bfloat16, 128><<<grid, 128, 0, s>>>(p);
    else b8::attention_rows_kernel<__half, 128><<<grid, 128, 0, s>>>(p);
  } else {
    if (bf) b8::attention_rows_kernel<__nv_bfloat16, 64><<<grid, 128, 0, s>>>(p);
    else b8::attention_rows_kernel<__half, 64><<<grid, 128, 0, s>>>(p);
  }
  return ucb_host::check_launch("block8 attention_rows_kernel");
}
