// Writes to and reads from the 8-bit block cache (ucb_block8_write / _read).
#include "block8.cuh"

namespace ucb {
namespace block8 {

int check_cache(const ucb_block8_cache* c, const char* what) {
  using ucb_host::set_error;
  if (!c || !c->key_code || !c->value_code || !c->key_scale || !c->value_scale || !c->key_low || !c->key_high ||
      !c->pending_key || !c->pending_value || !c->block_table || !c->lengths)
    return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (c->num_seqs < 1 || c->max_blocks < 1 || c->kv_heads < 1 || c->num_blocks < 1)
    return set_error(UCB_ERR_INVALID, "%s: bad shape", what);
  if (c->num_seqs > 4096) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most 4096 sequences", what);
  if (c->kv_heads > 65535) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most 65535 KV heads", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
  if (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64 && c->block_tokens != 128)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: block_tokens must be 16, 32, 64 or 128", what);
  if ((int64_t)c->max_blocks * c->block_tokens > 0x7fffffff)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: a sequence holds at most 2^31 - 1 tokens", what);
  if (c->dtype != UCB_BF16 && c->dtype != UCB_F16)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: dtype must be bfloat16 or float16", what);
  const uintptr_t all = reinterpret_cast<uintptr_t>(c->key_code) | reinterpret_cast<uintptr_t>(c->value_code) |
                        reinterpret_cast<uintptr_t>(c->key_low) | reinterpret_cast<uintptr_t>(c->key_high) |
                        reinterpret_cast<uintptr_t>(c->pending_key) | reinterpret_cast<uintptr_t>(c->pending_value);
  if (all & 15) return set_error(UCB_ERR_INVALID, "%s: cache tensors must be 16-byte aligned", what);
  return UCB_OK;
}

namespace {

struct WriteParams {
  ucb_block8_cache c;
  const void *key, *value;
  int64_t k_st, k_sh, v_st, v_sh, rows;
  const int32_t* starts;
  unsigned int* err;
};

constexpr int THREADS = 256;

// Row range [a, e) of sequence s among the call's rows; false when malformed.
__device__ __forceinline__ bool row_range(const int32_t* starts, int s, int64_t rows, int64_t& a, int64_t& e) {
  a = starts ? starts[s] : s;
  e = starts ? starts[s + 1] : s + 1;
  return a >= 0 && a <= e && e <= rows;
}

// The sequence whose rows hold row r (starts ascending).
__device__ __forceinline__ int seq_of_row(const int32_t* starts, int seqs, int64_t r) {
  if (!starts) return (int)r;
  int lo = 0, hi = seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= r) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// One side (keys or values) of one block and head: rows [0, held) come from the
// pending rows, rows [held, m) from the call's.
template <typename T, bool KEY>
__device__ void write_block(const WriteParams& p, int s, int h, int64_t block, int m, int held, int64_t first_row) {
  __shared__ unsigned int amax_bits;
  __shared__ int low[THREADS], high[THREADS];
  const ucb_block8_cache& c = p.c;
  const int d = c.head_dim, bt = c.block_tokens;
  const int ch = threadIdx.x % d, g = threadIdx.x / d, groups = THREADS / d;
  const int64_t st = KEY ? p.k_st : p.v_st;
  const T* src = static_cast<const T*>(KEY ? p.key : p.value) + h * (KEY ? p.k_sh : p.v_sh) + ch;
  T* pend = static_cast<T*>(KEY ? c.pending_key : c.pending_value) + ((int64_t)s * c.kv_heads + h) * bt * d + ch;
  int8_t* codes = (KEY ? c.key_code : c.value_code) + (block * c.kv_heads + h) * bt * d + ch;
  auto row = [&](int r) { return r < held ? pend[(int64_t)r * d] : src[(first_row + r - held) * st]; };
  if (threadIdx.x == 0) amax_bits = 0;
  __syncthreads();
  unsigned int top = 0;
  for (int r = g; r < m; r += groups)  // magnitude bits: their order is the values', with NaN above infinity
    top = max(top, __float_as_uint(Dtype<T>::to_f(row(r))) & 0x7fffffffu);
  atomicMax(&amax_bits, top);
  __syncthreads();
  const float scale = scale_of(__uint_as_float(amax_bits));
  const float inverse = __fdiv_rn(1.f, scale);
  int lo = 127, hi = -127;
  for (int r = g; r < m; r += groups) {
    const T x = row(r);
    const int q = code_of(Dtype<T>::to_f(x), inverse);
    codes[(int64_t)r * d] = (int8_t)q;
    lo = min(lo, q);
    hi = max(hi, q);
    if (m < bt && r >= held) pend[(int64_t)r * d] = x;
  }
  if (threadIdx.x == 0) (KEY ? c.key_scale : c.value_scale)[block * c.kv_heads + h] = scale;
  if (KEY) {
    low[threadIdx.x] = lo;
    high[threadIdx.x] = hi;
    __syncthreads();
    if (g == 0) {
      for (int k = 1; k < groups; ++k) lo = min(lo, low[k * d + ch]), hi = max(hi, high[k * d + ch]);
      c.key_low[(block * c.kv_heads + h) * d + ch] = (int8_t)lo;
      c.key_high[(block * c.kv_heads + h) * d + ch] = (int8_t)hi;
    }
  }
  __syncthreads();
}

// Work items of a head: item s < num_seqs is sequence s's first touched block
// and then its last, incomplete one (one CTA, since the first reads the pending rows that
// the last overwrites); item num_seqs + i is the whole block in between that
// holds row i * block_tokens of the call (every such block holds exactly one
// multiple of block_tokens).
template <typename T>
__global__ void __launch_bounds__(THREADS) write_kernel(const WriteParams p) {
  const ucb_block8_cache& c = p.c;
  const int bt = c.block_tokens, h = blockIdx.y;
  const bool ends = blockIdx.x < c.num_seqs;
  const int64_t probe = ends ? 0 : (int64_t)(blockIdx.x - c.num_seqs) * bt;
  const int s = ends ? blockIdx.x : seq_of_row(p.starts, c.num_seqs, probe);
  int64_t a, e;
  const bool ok = row_range(p.starts, s, p.rows, a, e);
  const int64_t n = e - a, len = c.lengths[s], old = len - n;
  if (!ok || old < 0 || len > (int64_t)c.max_blocks * bt) {
    if (ends && h == 0 && threadIdx.x == 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    return;
  }
  if (n == 0) return;
  const int first = (int)(old / bt), last = (int)((len - 1) / bt);
  auto one = [&](int j) {
    const int64_t block = pool_block(c, s, j, p.err);
    if (block < 0) return;
    const int64_t t0 = (int64_t)j * bt;
    const int m = (int)min((int64_t)bt, len - t0);
    const int held = (int)max((int64_t)0, min((int64_t)m, old - t0));
    const int64_t row = a + t0 + held - old;
    write_block<T, true>(p, s, h, block, m, held, row);
    write_block<T, false>(p, s, h, block, m, held, row);
  };
  if (ends) {
    one(first);
    if (last > first && len % bt) one(last);
  } else {
    if (probe < a || probe >= e) return;
    const int64_t j = (old + probe - a) / bt;
    if (j > first && (j + 1) * bt <= len) one((int)j);
  }
}

struct ReadParams {
  ucb_block8_cache c;
  int64_t rows;
  const int32_t* starts;
  void *key, *value;
  unsigned int* err;
};

// One warp per row: four codes of each side at a time over the row's heads.
template <typename T>
__global__ void __launch_bounds__(THREADS) read_kernel(const ReadParams p) {
  const ucb_block8_cache& c = p.c;
  const int64_t r = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
  if (r >= p.rows) return;
  const int lane = threadIdx.x & 31, d = c.head_dim, bt = c.block_tokens;
  const int s = seq_of_row(p.starts, c.num_seqs, r);
  int64_t a, e;
  const bool ok = row_range(p.starts, s, p.rows, a, e);
  const int64_t len = c.lengths[s], t = len - (e - r);
  if (!ok || r < a || r >= e || len - (e - a) < 0 || len > (int64_t)c.max_blocks * bt) {
    if (lane == 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    return;
  }
  const int64_t block = pool_block(c, s, (int)(t / bt), p.err);
  if (block < 0) return;
  for (int i = lane; i < c.kv_heads * d / 4; i += 32) {
    const int h = i / (d / 4), ch = i % (d / 4) * 4;
    const int64_t at = ((block * c.kv_heads + h) * bt + t % bt) * d + ch;
    const int64_t to = (r * c.kv_heads + h) * d + ch;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const char4 q = *reinterpret_cast<const char4*>((side ? c.value_code : c.key_code) + at);
      const float x = (side ? c.value_scale : c.key_scale)[block * c.kv_heads + h];
      T* out = static_cast<T*>(side ? p.value : p.key) + to;
      out[0] = Dtype<T>::from_f(q.x * x);
      out[1] = Dtype<T>::from_f(q.y * x);
      out[2] = Dtype<T>::from_f(q.z * x);
      out[3] = Dtype<T>::from_f(q.w * x);
    }
  }
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

extern "C" int ucb_block8_write(const ucb_block8_cache* cache, const void* key, int64_t k_st, int64_t k_sh,
                                const void* value, int64_t v_st, int64_t v_sh, int64_t rows, const int32_t* starts,
                                void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_write")) return rc;
  if (rows < 0 || (!starts && rows != cache->num_seqs))
    return set_error(UCB_ERR_INVALID, "ucb_block8_write: one row for each sequence, or starts");
  if (rows == 0) return UCB_OK;
  if (!key || !value) return set_error(UCB_ERR_INVALID, "ucb_block8_write: null pointer");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_block8_write: device error word unavailable");
  const b8::WriteParams p{*cache, key, value, k_st, k_sh, v_st, v_sh, rows, starts, err};
  const int64_t items = cache->num_seqs + (starts ? (rows + cache->block_tokens - 1) / cache->block_tokens : 0);
  if (items > 0x7fffffff) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_write: too many rows");
  const dim3 grid((unsigned)items, cache->kv_heads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->dtype == UCB_BF16)
    b8::write_kernel<__nv_bfloat16><<<grid, b8::THREADS, 0, s>>>(p);
  else
    b8::write_kernel<__half><<<grid, b8::THREADS, 0, s>>>(p);
  return ucb_host::check_launch("block8 write_kernel");
}

extern "C" int ucb_block8_read(const ucb_block8_cache* cache, int64_t rows, const int32_t* starts, void* key,
                               void* value, void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_read")) return rc;
  if (rows < 0 || (!starts && rows != cache->num_seqs))
    return set_error(UCB_ERR_INVALID, "ucb_block8_read: one row for each sequence, or starts");
  if (rows == 0) return UCB_OK;
  if (!key || !value) return set_error(UCB_ERR_INVALID, "ucb_block8_read: null pointer");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_block8_read: device error word unavailable");
  const b8::ReadParams p{*cache, rows, starts, key, value, err};
  const int64_t blocks = (rows + b8::THREADS / 32 - 1) / (b8::THREADS / 32);
  if (blocks > 0x7fffffff) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_read: too many rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cache->dtype == UCB_BF16)
    b8::read_kernel<__nv_bfloat16><<<(unsigned)blocks, b8::THREADS, 0, s>>>(p);
  else
    b8::read_kernel<__half><<<(unsigned)blocks, b8::THREADS, 0, s>>>(p);
  return ucb_host::check_launch("block8 read_kernel");
}
