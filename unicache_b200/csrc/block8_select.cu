// The blocks of the 8-bit block cache that a query may need most (ucb_block8_select).
#include "block8.cuh"

namespace ucb {
namespace block8 {
namespace {

struct SelectParams {
  ucb_block8_cache c;
  const void* q;
  int64_t q_ss, q_sh;
  int q_heads, count, first, recent;
  int32_t* blocks;
  uint32_t* keys;  // [num_seqs, kv_heads, max_blocks]
  unsigned int* err;
};

constexpr int THREADS = 256;

// Unsigned keys in the order of the scores; NaN above every number, so that a
// poisoned block is read and shows.
constexpr uint32_t KEY_NAN = 0xFFFFFFFEu, KEY_FORCED = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return KEY_NAN;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 and 0 are one value
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) select_kernel(const SelectParams p) {
  const ucb_block8_cache& c = p.c;
  const int s = blockIdx.x, h = blockIdx.y, d = c.head_dim, group = p.q_heads / c.kv_heads;
  const int tokens = held_tokens(c, s, p.err);
  const int n = (tokens + c.block_tokens - 1) / c.block_tokens;
  uint32_t* keys = p.keys + ((int64_t)s * c.kv_heads + h) * c.max_blocks;
  int32_t* out = p.blocks + ((int64_t)s * c.kv_heads + h) * p.count;
  for (int j = threadIdx.x; j < n; j += THREADS) keys[j] = 0;
  __shared__ float top[THREADS / 32];
  __shared__ int codes[128];
  __shared__ unsigned long long best;
  __shared__ float best_scale;
  // scores: the largest over the group's heads, kept as floats until the last head
  float* scores = reinterpret_cast<float*>(keys);
  for (int g = 0; g < group; ++g) {
    const T* q = static_cast<const T*>(p.q) + s * p.q_ss + (h * group + g) * p.q_sh;
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned int m = 0;
      for (int i = 0; i < d; ++i) m = max(m, __float_as_uint(Dtype<T>::to_f(q[i])) & 0x7fffffffu);
      best_scale = scale_of(__uint_as_float(m));
    }
    __syncthreads();
    const float qs = best_scale, inverse = __fdiv_rn(1.f, qs);
    if (threadIdx.x < d) codes[threadIdx.x] = code_of(Dtype<T>::to_f(q[threadIdx.x]), inverse);
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += THREADS) {
      const int64_t block = pool_block(c, s, j, p.err);
      if (block < 0) continue;
      const int64_t at = (block * c.kv_heads + h) * d;
      int sum = 0;
      for (int i = 0; i < d; ++i) sum += max(codes[i] * c.key_low[at + i], codes[i] * c.key_high[at + i]);
      const float x = __fmul_rn((float)sum, qs), old = scores[j];
      scores[j] = g == 0 ? x : (x != x || old != old ? x + old : fmaxf(x, old));
    }
  }
  for (int j = threadIdx.x; j < n; j += THREADS) {
    const int64_t block = pool_block(c, s, j, p.err);
    const float x = block < 0 ? -INFINITY : __fmul_rn(scores[j], c.key_scale[block * c.kv_heads + h]);
    keys[j] = j < p.first || j >= n - p.recent ? KEY_FORCED : key_of(x);
  }
  // the largest key, lowest block first, `count` times; a taken block's key is 0
  (void)top;
  for (int k = 0; k < min(p.count, n); ++k) {
    __syncthreads();
    if (threadIdx.x == 0) best = 0;
    __syncthreads();
    unsigned long long mine = 0;
    for (int j = threadIdx.x; j < n; j += THREADS)
      mine = max(mine, ((unsigned long long)keys[j] << 32) | (0xFFFFFFFFu - (unsigned)j));
    atomicMax(&best, mine);
    __syncthreads();
    if (threadIdx.x == 0) keys[0xFFFFFFFFu - (unsigned)best] = 0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int k = 0;
    for (int j = 0; j < n; ++j)
      if (keys[j] == 0) out[k++] = j;
    for (; k < p.count; ++k) out[k] = -1;
  }
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

extern "C" int64_t ucb_block8_select_workspace_bytes(const ucb_block8_cache* cache) {
  if (b8::check_cache(cache, "ucb_block8_select_workspace_bytes")) return -1;
  return (int64_t)cache->num_seqs * cache->kv_heads * cache->max_blocks * 4;
}

extern "C" int ucb_block8_select(const ucb_block8_cache* cache, const void* query, int64_t q_ss, int64_t q_sh,
                                 int q_heads, int count, int first, int recent, int32_t* blocks, void* workspace,
                                 void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_select")) return rc;
  if (!query || !blocks || !workspace) return set_error(UCB_ERR_INVALID, "ucb_block8_select: null pointer");
  if (q_heads < 1 || q_heads % cache->kv_heads)
    return set_error(UCB_ERR_INVALID, "ucb_block8_select: query heads must be divisible by KV heads");
  if (first < 0 || recent < 0 || count < 1 || (int64_t)first + recent > count)
    return set_error(UCB_ERR_INVALID, "ucb_block8_select: need first + recent <= count and count >= 1");
  if (count > 4096) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_select: at most 4096 blocks");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_block8_select: device error word unavailable");
  const b8::SelectParams p{*cache, query, q_ss, q_sh, q_heads, count, first, recent, blocks,
                           static_cast<uint32_t*>(workspace), err};
  const dim3 grid(cache->num_seqs, cache->kv_heads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->dtype == UCB_BF16)
    b8::select_kernel<__nv_bfloat16><<<grid, b8::THREADS, 0, s>>>(p);
  else
    b8::select_kernel<__half><<<grid, b8::THREADS, 0, s>>>(p);
  return ucb_host::check_launch("block8 select_kernel");
}
