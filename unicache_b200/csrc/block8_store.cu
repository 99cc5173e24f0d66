// Writes to and reads from the 8-bit block cache (ucb_block8_write / _read):
//   scale = max(amax / 127, 2^-120),  code = clamp(rint(x * (1 / scale)), -127, 127)
// Prompts move 2 bytes in and 1 out a value, and back: 45880
// tokens x 4 heads x 128, keys and values, written in 27.5 us (5.1 TB/s, 75% of the issue slots busy) and
// restored in 27.2 (waiting for table, scale and codes, one after the other).  One token of each of 32 sequences is a chain of round
// trips: 3.8 us.  A CTA holds a whole block of one head in registers, so each row is
// read once; the block's largest magnitude and its channels' bounds are reduced
// through one barrier.
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
  int aligned;  // rows start on 16 bytes
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

// The sequence whose rows hold row r (starts ascending), found by the whole warp: a round trip for every factor of 32
// in the number of sequences.
__device__ __forceinline__ int seq_of_row(const int32_t* starts, int seqs, int64_t r) {
  if (!starts) return (int)r;
  const int lane = threadIdx.x & 31;
  int lo = 0, n = seqs;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const bool before = lane * step < n && starts[lo + lane * step] <= r;
    const int skip = (max(__popc(__ballot_sync(0xffffffffu, before)), 1) - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// Eight adjacent 16-bit elements; rows that do not start on 16 bytes element by element.
__device__ __forceinline__ uint4 load8(const uint16_t* x, bool aligned) {
  if (aligned) return *reinterpret_cast<const uint4*>(x);
  return make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16,
                    x[6] | (uint32_t)x[7] << 16);
}

template <bool BF> __device__ __forceinline__ float low_half(uint32_t w) {
  return BF ? Dtype<__nv_bfloat16>::lo(w) : Dtype<__half>::lo(w);
}
template <bool BF> __device__ __forceinline__ float high_half(uint32_t w) {
  return BF ? Dtype<__nv_bfloat16>::hi(w) : Dtype<__half>::hi(w);
}
template <bool BF> __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  if (BF) {
    const __nv_bfloat162 m = __hmin2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  const __half2 m = __hmin2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <bool BF> __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  if (BF) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
  const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}

// Four codes: rint of the fp32 product by adding 1.5 * 2^23 (two roundings, as code_of has; the products are
// below 128), whose low byte is the code.  `inverse` 0 stands for a scale that is no number: codes 0.
template <bool BF> __device__ __forceinline__ uint32_t codes4(uint32_t w0, uint32_t w1, float inverse) {
  if (inverse == 0.f) return 0;
  const float x[4] = {low_half<BF>(w0), high_half<BF>(w0), low_half<BF>(w1), high_half<BF>(w1)};
  uint32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inverse), 12582912.f));
  return prmt(prmt(v[0], v[1], 0x0040), prmt(v[2], v[3], 0x0040), 0x5410);
}

// 1 / scale, 0 for a scale that is no number.
__device__ __forceinline__ float inverse_of(float scale) { return scale < INFINITY ? __fdiv_rn(1.f, scale) : 0.f; }

// Keys and values of block j of sequence s and one head: rows [0, held) are pending ones, rows [held, m) the call's.
// The new rows decide whether the block's scale grows: where it does not, the codes
// of the held rows stand (they depend on the scale alone, and the scale of a
// larger magnitude is never the smaller), and only the new rows are written.  Where rows
// of the block were withdrawn since (the record counts more than `held`), scale and bounds
// come from the held rows again (one token to each of 32 sequences, the one before it withdrawn: 3.9 us against 3.8).  Nothing is written where the held rows are not there any more, or never were.
// FRESH: a block without held rows.  KEEP: the last block that the call writes, whose rows stay pending.
template <bool BF, int D, int BT, bool FRESH>
__device__ __forceinline__ void write_block(const WriteParams& p, int s, int h, int64_t block, int j, int m, int held,
                                            int64_t first_row, bool keep) {
  if (FRESH) held = 0;
  constexpr int UNITS = D / 8, STRIDE = THREADS / UNITS, PASSES = (BT + STRIDE - 1) / STRIDE, WARPS = THREADS / 32;
  __shared__ uint32_t warp_top[2][WARPS];
  __shared__ __align__(16) uint32_t warp_low[WARPS][D / 2], warp_high[WARPS][D / 2];
  const ucb_block8_cache& c = p.c;
  const int unit = threadIdx.x % UNITS, g = threadIdx.x / UNITS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t at = (block * c.kv_heads + h) * (int64_t)(BT * D) + unit * 8;
  const int64_t scale_at = block * c.kv_heads + h;
  const int64_t pending_at = ((int64_t)s * c.kv_heads + h) * (BT * D) + unit * 8;
  const float old[2] = {held ? c.key_scale[scale_at] : 0.f, held ? c.value_scale[scale_at] : 0.f};
  uint4* record_at = reinterpret_cast<uint4*>(static_cast<uint16_t*>(c.pending_key) +
                                              ((int64_t)s * c.kv_heads + h) * (BT * D) + (BT - 1) * D);
  const uint4 record = held ? *record_at : make_uint4(0, 0, 0, 0);

  // ---- new rows: loads of both sides together.  x holds row g + i * STRIDE of the block.
  uint4 x[2][PASSES];
  uint32_t top[2] = {0, 0}, low[4], high[4];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint16_t* src = static_cast<const uint16_t*>(side ? p.value : p.key) + h * (side ? p.v_sh : p.k_sh) + unit * 8;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = g + i * STRIDE;
      if (row >= held && row < m) x[side][i] = load8(src + (first_row + row - held) * (side ? p.v_st : p.k_st), p.aligned);
    }
  }
  auto load_held = [&](int side) {
    const uint16_t* src = static_cast<const uint16_t*>(side ? c.pending_value : c.pending_key) + pending_at;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = g + i * STRIDE;
      if (row < held) x[side][i] = *reinterpret_cast<const uint4*>(src + row * D);
    }
  };
  bool again = false;  // rows were withdrawn
  if (held && is_record(record)) {
    if (record.y != (uint32_t)j || record.z < (uint32_t)held) {
      if (threadIdx.x == 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
      return;
    }
    again = record.z > (uint32_t)held;
    if (again) load_held(0), load_held(1);
  }
  const int from = again ? 0 : held;
  constexpr uint32_t INF2 = BF ? 0x7f807f80u : 0x7c007c00u;
#pragma unroll
  for (int k = 0; k < 4; ++k) low[k] = INF2, high[k] = INF2 | 0x80008000u;
  auto bounds = [&](uint4 w) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) low[k] = min2<BF>(low[k], v[k]), high[k] = max2<BF>(high[k], v[k]);
  };
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
    if (g + i * STRIDE >= from && g + i * STRIDE < m) {
#pragma unroll
      for (int side = 0; side < 2; ++side) {  // magnitude bits: their order is the values', with NaN above infinity
        const uint4 w = x[side][i];
        top[side] = __vmaxu2(top[side], __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu),
                                                 __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
      }
      bounds(x[0][i]);
    }
  auto share_bounds = [&]() {  // over the warp's rows, then one row of shared memory a warp
#pragma unroll
    for (int o = UNITS; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        low[k] = min2<BF>(low[k], __shfl_xor_sync(0xffffffffu, low[k], o));
        high[k] = max2<BF>(high[k], __shfl_xor_sync(0xffffffffu, high[k], o));
      }
    if (lane < UNITS) {
      *reinterpret_cast<uint4*>(&warp_low[warp][unit * 4]) = make_uint4(low[0], low[1], low[2], low[3]);
      *reinterpret_cast<uint4*>(&warp_high[warp][unit * 4]) = make_uint4(high[0], high[1], high[2], high[3]);
    }
  };
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint32_t t = __reduce_max_sync(0xffffffffu, max(top[side] & 0xffffu, top[side] >> 16));
    if (lane == 0) warp_top[side][warp] = t;
  }
  share_bounds();
  __syncthreads();
  float scale[2], inverse[2];
  bool changed[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) t = max(t, warp_top[side][w]);
    const float mine = scale_of(low_half<BF>(t));
    changed[side] = !held || (again ? !(mine == old[side]) : mine > old[side] || (mine != mine && old[side] == old[side]));
    scale[side] = changed[side] ? mine : old[side];
    inverse[side] = inverse_of(scale[side]);
  }

  // ---- a larger scale: the held rows too
  if (held && !again) {
    if (changed[0]) {
      load_held(0);
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
        if (g + i * STRIDE < held) bounds(x[0][i]);
      __syncthreads();  // the new rows' bounds were read by no one yet, but other warps' are in place
      share_bounds();
      __syncthreads();
    }
    if (changed[1]) load_held(1);
  }
  // ---- codes, and the new rows themselves where more of the block may come, or come again
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = g + i * STRIDE;
      if (row >= m || (row < held && !changed[side])) continue;
      const uint4 w = x[side][i];
      *reinterpret_cast<uint2*>((side ? c.value_code : c.key_code) + at + row * D) =
          make_uint2(codes4<BF>(w.x, w.y, inverse[side]), codes4<BF>(w.z, w.w, inverse[side]));
      if (keep && row >= held && row < BT - 1)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(side ? c.pending_value : c.pending_key) + pending_at + row * D) = w;
    }
  if (threadIdx.x < 2 && changed[threadIdx.x ? 1 : 0])
    (threadIdx.x ? c.value_scale : c.key_scale)[scale_at] = threadIdx.x ? scale[1] : scale[0];
  // ---- bounds of the key codes: rounding keeps order, so they are the codes of the channels' bounds
  for (int pair = threadIdx.x; pair < D / 2; pair += THREADS) {
    uint32_t lo = warp_low[0][pair], hi = warp_high[0][pair];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) lo = min2<BF>(lo, warp_low[w][pair]), hi = max2<BF>(hi, warp_high[w][pair]);
    const uint32_t q = codes4<BF>(lo, hi, inverse[0]);  // low of two channels, high of two channels
    char2 low2 = make_char2((signed char)(q & 255), (signed char)(q >> 8 & 255));
    char2 high2 = make_char2((signed char)(q >> 16 & 255), (signed char)(q >> 24));
    char2* low_to = reinterpret_cast<char2*>(c.key_low + scale_at * D) + pair;
    char2* high_to = reinterpret_cast<char2*>(c.key_high + scale_at * D) + pair;
    if (!changed[0] && !again) {
      const char2 a = *low_to, b = *high_to;
      low2 = make_char2(min(low2.x, a.x), min(low2.y, a.y));
      high2 = make_char2(max(high2.x, b.x), max(high2.y, b.y));
    }
    *low_to = low2;
    *high_to = high2;
  }
  // every thread read the old record before the barrier; the rows of a block that the call leaves behind are not kept
  if (!FRESH && threadIdx.x == 0) *record_at = make_record(j, keep ? m : 0);
}

// Rows of block j from `held` on are skipped: rows in their places from before, withdrawn or an earlier sequence's, are not theirs.
__device__ __forceinline__ void drop_record(uint4* at, int j, int held) {
  const uint4 record = *at;
  if (is_record(record) && record.y == (uint32_t)j && record.z > (uint32_t)held) *at = make_record(j, held);
}

// Work items of a head: item s < num_seqs is sequence s's first touched block
// and then its last one (one CTA, since the first reads the pending rows that
// the last overwrites); item num_seqs + i is the whole block in between that
// holds row i * block_tokens of the call (every such block holds exactly one
// multiple of block_tokens).
// Four CTAs a multiprocessor where a block fits 64 registers a thread: store of the
// prompts above 27.6 us against 30.5 with three.
template <bool BF, int D, int BT>
__global__ void __launch_bounds__(THREADS, D * BT > 8192 ? 2 : 4) write_kernel(const WriteParams p) {
  const ucb_block8_cache& c = p.c;
  const int bt = BT, h = blockIdx.y;
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
  if (!ends) {
    if (probe < a || probe >= e) return;
    const int64_t j = (old + probe - a) / bt;
    if (j <= first || j >= last) return;
    const int64_t block = pool_block(c, s, (int)j, p.err);
    if (block >= 0) write_block<BF, D, BT, true>(p, s, h, block, (int)j, bt, 0, a + j * bt - old, false);
    return;
  }
  // where the last block is nowhere, the first one's rows stay pending: the step may be taken back into it
  const int at_last = first < last ? c.block_table[(int64_t)s * c.max_blocks + last] : 0;
  const bool stays = at_last < 0 || at_last >= c.num_blocks;
  int j = first;
#pragma unroll 1  // one copy of write_block
  while (true) {
    const int64_t block = pool_block(c, s, j, p.err);
    const int64_t t0 = (int64_t)j * bt;
    const int m = (int)min((int64_t)bt, len - t0);
    const int held = (int)max((int64_t)0, min((int64_t)m, old - t0));
    if (block >= 0) {
      write_block<BF, D, BT, false>(p, s, h, block, j, m, held, a + t0 + held - old, stays || j == last);
    } else {
      drop_record(pending_record(c, s, h), j, held);  // every thread the same: as one thread's, prompts in blocks of 16 took 57.4 us in the place of 55.6
    }
    if (j == last) break;
    j = last;
    __syncthreads();  // the pending rows of the first block are read
  }
}

struct ReadParams {
  ucb_block8_cache c;
  int64_t rows;
  const int32_t* starts;
  void *key, *value;
  unsigned int* err;
};

// A warp restores ROWS consecutive rows: lanes find one row's block each, then all
// lanes take units of 8 codes of every row's heads, keys and values.
constexpr int READ_ROWS = 4;

template <bool BF, int D> __global__ void __launch_bounds__(THREADS) read_kernel(const ReadParams p) {
  const ucb_block8_cache& c = p.c;
  const int lane = threadIdx.x & 31, bt = c.block_tokens;
  const int64_t r0 = ((int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5)) * READ_ROWS;
  int block = -1, in_block = 0;
  if (r0 >= p.rows) return;
  const int s0 = seq_of_row(p.starts, c.num_seqs, r0);
  if (lane < READ_ROWS && r0 + lane < p.rows) {
    const int64_t r = r0 + lane;
    int s = p.starts ? s0 : (int)r;
    while (p.starts && s + 1 < c.num_seqs && p.starts[s + 1] <= r) ++s;
    int64_t a, e;
    const bool ok = row_range(p.starts, s, p.rows, a, e);
    const int64_t len = c.lengths[s], t = len - (e - r);
    if (!ok || r < a || r >= e || len - (e - a) < 0 || len > (int64_t)c.max_blocks * bt) {
      atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    } else {
      block = (int)pool_block(c, s, (int)(t / bt), p.err);
      in_block = (int)(t % bt);
    }
  }
  int where[READ_ROWS], row[READ_ROWS];
#pragma unroll
  for (int k = 0; k < READ_ROWS; ++k) {
    where[k] = __shfl_sync(0xffffffffu, block, k);
    row[k] = __shfl_sync(0xffffffffu, in_block, k);
  }
  const int units = c.kv_heads * (D / 8);
  for (int i = lane; i < 2 * units; i += 32) {
    const int side = i >= units, u = side ? i - units : i, h = u / (D / 8), d = u % (D / 8) * 8;
    const int8_t* codes = side ? c.value_code : c.key_code;
    const float* scales = side ? c.value_scale : c.key_scale;
    uint16_t* out = static_cast<uint16_t*>(side ? p.value : p.key);
    uint2 q[READ_ROWS];
    float scale[READ_ROWS];
#pragma unroll
    for (int k = 0; k < READ_ROWS; ++k)
      if (where[k] >= 0) {
        const int64_t at = (int64_t)where[k] * c.kv_heads + h;
        q[k] = *reinterpret_cast<const uint2*>(codes + (at * bt + row[k]) * D + d);
        scale[k] = scales[at];
      }
#pragma unroll
    for (int k = 0; k < READ_ROWS; ++k) {
      if (r0 + k >= p.rows) continue;
      uint32_t y[4] = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};  // NaN where the row is in no block
#pragma unroll
      for (int j = 0; j < 4 && where[k] >= 0; ++j) {
        const uint32_t two = (j < 2 ? q[k].x : q[k].y) >> (j % 2 * 16);
        const float x0 = (float)(int)(signed char)(two & 255) * scale[k], x1 = (float)(int)(signed char)(two >> 8 & 255) * scale[k];
        y[j] = BF ? pack_bf16x2(x0, x1) : pack_f16x2(x0, x1);
      }
      *reinterpret_cast<uint4*>(out + ((r0 + k) * c.kv_heads + h) * D + d) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

template <bool BF, int D> int launch_write(const WriteParams& p, dim3 grid, cudaStream_t s) {
  const char* what = "block8 write_kernel";
  switch (p.c.block_tokens) {
    case 16: return launch(write_kernel<BF, D, 16>, grid, dim3(THREADS), 0, s, p, what);
    case 32: return launch(write_kernel<BF, D, 32>, grid, dim3(THREADS), 0, s, p, what);
    case 64: return launch(write_kernel<BF, D, 64>, grid, dim3(THREADS), 0, s, p, what);
    default: return launch(write_kernel<BF, D, 128>, grid, dim3(THREADS), 0, s, p, what);
  }
}

template <bool BF, int D> int launch_read(const ReadParams& p, unsigned blocks, cudaStream_t s) {
  return launch(read_kernel<BF, D>, dim3(blocks), dim3(THREADS), 0, s, p, "block8 read_kernel");
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
  b8::WriteParams p{*cache, key, value, k_st, k_sh, v_st, v_sh, rows, 0, starts, err};
  p.aligned = ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) == 0 &&
              ((k_st | k_sh | v_st | v_sh) & 7) == 0;
  const int64_t items = cache->num_seqs + (starts ? (rows + cache->block_tokens - 1) / cache->block_tokens : 0);
  if (items > 0x7fffffff) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_write: too many rows");
  const dim3 grid((unsigned)items, cache->kv_heads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == UCB_BF16;
  if (cache->head_dim == 128) return bf ? b8::launch_write<true, 128>(p, grid, s) : b8::launch_write<false, 128>(p, grid, s);
  return bf ? b8::launch_write<true, 64>(p, grid, s) : b8::launch_write<false, 64>(p, grid, s);
}

extern "C" int ucb_block8_read(const ucb_block8_cache* cache, int64_t rows, const int32_t* starts, void* key,
                               void* value, void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_read")) return rc;
  if (rows < 0 || (!starts && rows != cache->num_seqs))
    return set_error(UCB_ERR_INVALID, "ucb_block8_read: one row for each sequence, or starts");
  if (rows == 0) return UCB_OK;
  if (!key || !value) return set_error(UCB_ERR_INVALID, "ucb_block8_read: null pointer");
  if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15)
    return set_error(UCB_ERR_INVALID, "ucb_block8_read: outputs must be 16-byte aligned");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_block8_read: device error word unavailable");
  const b8::ReadParams p{*cache, rows, starts, key, value, err};
  const int64_t each = b8::THREADS / 32 * b8::READ_ROWS, blocks = (rows + each - 1) / each;
  if (blocks > 0x7fffffff) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_read: too many rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == UCB_BF16;
  const unsigned grid = (unsigned)blocks;
  if (cache->head_dim == 128) return bf ? b8::launch_read<true, 128>(p, grid, s) : b8::launch_read<false, 128>(p, grid, s);
  return bf ? b8::launch_read<true, 64>(p, grid, s) : b8::launch_read<false, 64>(p, grid, s);
}
