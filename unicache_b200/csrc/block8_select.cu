// The blocks of the 8-bit block cache that a query may need most (ucb_block8_select).
//
//   I_hj = sum_d max(q_d low_jd, q_d high_jd) = sum_d max(q_d, 0) high_jd + min(q_d, 0) low_jd
//   score_j = key_scale_j * max_h (I_hj * qscale_h)
//
// over whole numbers: the query heads are rounded to 8 bits by the cache's own
// rule, so I is exact in the int32 matrix instructions (16 blocks x 8 heads x
// 32 channels each), and the two fp32 products fix the scores bit for bit.
// The kernel reads 2 D bytes of bounds for each block: memory bound for
// many sequences, a few dependent round trips long for one.
//
// A cluster of CTAs scores one (sequence, KV head), each CTA its share of the
// blocks, into the first CTA's shared memory (into global memory where
// a row of keys does not fit there); that CTA then finds the count-th largest key
// by up to four 8-bit radix passes and writes the kept blocks in ascending order.
// One sequence is a chain of round trips (lengths, table and query together;
// bounds; keys): 469 blocks x 4 heads in 6.5 us.  8 sequences of 2048 blocks
// (17 MB of bounds, 2.6 us) take 10: 3.8 us to the scores, 0.9 for the cluster's
// exchange, 2.7 for the radix passes, 1.2 to write the blocks.
#include <cooperative_groups.h>

#include <algorithm>
#include <utility>

#include "block8.cuh"

namespace cg = cooperative_groups;

namespace ucb {
namespace block8 {
namespace {

struct SelectParams {
  ucb_block8_cache c;
  const void* q;
  int64_t q_ss, q_sh;
  int group, count, first, recent;
  int32_t* blocks;
  uint32_t* spill;  // [num_seqs, kv_heads, max_blocks] when keys do not fit shared memory, else null
  unsigned int* err;
};

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int AHEAD = 2;  // tiles of a warp whose table entries are loaded before the lengths are known
constexpr int MOST_SHARED_KEYS = 49152;  // 192 KB

// Unsigned keys in the order of the scores; NaN above every number, so that a
// poisoned block is read and shows.
constexpr uint32_t KEY_NAN = 0xFFFFFFFEu, KEY_FORCED = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return KEY_NAN;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 and 0 are one value
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// D (16 blocks x 8 heads) += A (16 x 32 bytes) B (32 x 8 bytes), signed.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename T, int D> __global__ void __launch_bounds__(THREADS) select_kernel(const SelectParams p) {
  constexpr int KS = D / 32;  // products of 32 channels on each side
  extern __shared__ __align__(16) uint32_t row_keys[];
  __shared__ __align__(16) int8_t q_code[8][2][D + 16];  // [head][min(q, 0) or max(q, 0)][channel], rows on distinct banks
  __shared__ float q_scale[8];
  __shared__ __align__(16) int histogram[4][256];
  __shared__ int2 warp_counts[WARPS];
  const ucb_block8_cache& c = p.c;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = cluster.num_blocks(), part = cluster.block_rank();
  auto started = cluster.barrier_arrive();  // waited for before the first key goes to another CTA
  const int pair = blockIdx.x / parts, s = pair / c.kv_heads, h = pair % c.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cq = lane & 3;
  int32_t* out = p.blocks + (int64_t)pair * p.count;
  uint32_t* keys = p.spill ? p.spill + (int64_t)pair * c.max_blocks : cluster.map_shared_rank(row_keys, 0);
  const int32_t* table = c.block_table + (int64_t)s * c.max_blocks;

  // ---- what does not depend on the lengths: query heads (warp w rounds head g0 + w), table entries of the
  // warp's first tiles
  constexpr int PER = D / 32;
  auto load_head = [&](int g, float (&x)[PER]) {
    const T* q = static_cast<const T*>(p.q) + s * p.q_ss + (int64_t)(h * p.group + g) * p.q_sh + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = g < p.group ? Dtype<T>::to_f(q[i]) : 0.f;
  };
  float x[PER];
  load_head(warp, x);
  const int tile0 = part * WARPS + warp, tile_step = parts * WARPS;
  int entry[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    const int j = (tile0 + i * tile_step) * 16 + (lane & 15);
    entry[i] = j < c.max_blocks ? table[j] : -1;
  }
  const int tokens = held_tokens(c, s, p.err);
  const int n = (int)(((int64_t)tokens + c.block_tokens - 1) / c.block_tokens);
  const bool all = n <= p.count;  // nothing to choose
  for (int i = threadIdx.x; i < 4 * 256; i += THREADS) histogram[0][i] = 0;

  // bounds and key scales of a tile's blocks: lane i the scale of block i, lane (r, cq) units cq and cq + 4 of blocks
  // r and r + 8
  struct Tile {
    uint4 x[2][D / 64][2];
    float ks;
    int block0, block1;
  };
  auto load_tile = [&](int tile, int block) {
    Tile a;
    if (tile * 16 + (lane & 15) >= n) block = -1;
    else if (block < 0 || block >= c.num_blocks) {
      block = -1;
      atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    }
    a.ks = block >= 0 ? c.key_scale[(int64_t)block * c.kv_heads + h] : 0.f;
    a.block0 = __shfl_sync(0xffffffffu, block, r);
    a.block1 = __shfl_sync(0xffffffffu, block, r + 8);
    const int64_t at0 = ((int64_t)max(a.block0, 0) * c.kv_heads + h) * D + 16 * cq;
    const int64_t at1 = ((int64_t)max(a.block1, 0) * c.kv_heads + h) * D + 16 * cq;
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int half = 0; half < D / 64; ++half) {
        const int8_t* bounds = (side ? c.key_high : c.key_low) + half * 64;
        a.x[side][half][0] = *reinterpret_cast<const uint4*>(bounds + at0);
        a.x[side][half][1] = *reinterpret_cast<const uint4*>(bounds + at1);
      }
    return a;
  };

  const int tiles = (n + 15) / 16;
  Tile next;
  if (!all && tile0 < tiles) next = load_tile(tile0, entry[0]);
  cluster.barrier_wait(std::move(started));
  if (!all) {
    for (int g0 = 0; g0 < p.group; g0 += 8) {
      // ---- query heads in 8 bits
      if (g0) {
        __syncthreads();
        load_head(g0 + warp, x);
        if (tile0 < tiles) next = load_tile(tile0, entry[0]);
      }
      unsigned int top = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
      top = __reduce_max_sync(0xffffffffu, top);
      const float scale = scale_of(__uint_as_float(top)), inverse = __fdiv_rn(1.f, scale);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int code = code_of(x[i], inverse);
        q_code[warp][0][lane * PER + i] = (int8_t)min(code, 0);
        q_code[warp][1][lane * PER + i] = (int8_t)max(code, 0);
      }
      if (lane == 0) q_scale[warp] = scale;
      __syncthreads();
      // operand words in the order of the bounds' 16-byte units
      uint32_t b[2][KS][2];
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int at = (k / 2) * 64 + 16 * cq + (k % 2) * 8;
          b[side][k][0] = *reinterpret_cast<const uint32_t*>(&q_code[r][side][at]);
          b[side][k][1] = *reinterpret_cast<const uint32_t*>(&q_code[r][side][at + 4]);
        }
      const float scale0 = q_scale[2 * cq], scale1 = q_scale[2 * cq + 1];
      const bool real0 = g0 + 2 * cq < p.group, real1 = g0 + 2 * cq + 1 < p.group;

      for (int tile = tile0, i = 0; tile < tiles; tile += tile_step, ++i) {
        const Tile a = next;
        const int after = tile + tile_step;
        if (after < tiles) {
          const int j = after * 16 + (lane & 15);
          int block = -1;
          if (i + 1 < AHEAD) block = entry[1];
          else if (j < n) block = table[j];
          next = load_tile(after, block);
        }
        int sum[4] = {0, 0, 0, 0};
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
          for (int half = 0; half < D / 64; ++half) {
            const uint4 u = a.x[side][half][0], v = a.x[side][half][1];
            mma_s8(sum, u.x, v.x, u.y, v.y, b[side][half * 2][0], b[side][half * 2][1]);
            mma_s8(sum, u.z, v.z, u.w, v.w, b[side][half * 2 + 1][0], b[side][half * 2 + 1][1]);
          }
        // largest over the heads: two columns here, the others in the quad's lanes
        const float ks0 = __shfl_sync(0xffffffffu, a.ks, r), ks1 = __shfl_sync(0xffffffffu, a.ks, r + 8);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float top = -INFINITY;
          if (real0) top = max_nan(top, __fmul_rn((float)sum[2 * k], scale0));
          if (real1) top = max_nan(top, __fmul_rn((float)sum[2 * k + 1], scale1));
          top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int j = tile * 16 + r + 8 * k;
          if (cq == 0 && j < n) {
            // groups of more than 8 heads: the raw maximum goes from pass to pass
            if (g0) top = max_nan(top, __uint_as_float(keys[j]));
            uint32_t key = __float_as_uint(top);
            if (g0 + 8 >= p.group) {
              const bool known = (k ? a.block1 : a.block0) >= 0;
              key = j < p.first || j >= n - p.recent ? KEY_FORCED
                    : known ? key_of(__fmul_rn(top, k ? ks1 : ks0)) : key_of(-INFINITY);
            }
            keys[j] = key;
          }
        }
      }
    }
    cluster.sync();  // every CTA's keys are in place
  }
  if (part) return;

  if (all) {
    for (int k = threadIdx.x; k < p.count; k += THREADS) {
      if (k < n && (table[k] < 0 || table[k] >= c.num_blocks)) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
      out[k] = k < n ? k : -1;
    }
    return;
  }
  uint32_t* own = p.spill ? keys : row_keys;

  // ---- the count-th largest key: its bits from the top, 8 at a time; every warp finds the bin by itself.  Done
  // early when a bin is taken whole.  (Counting a warp's equal digits once, by __match_any_sync, took 5.7 us for 2048 keys
  // where these atomics take 1.)
  uint32_t threshold = 0;  // keys from here on, of the equal ones `need`
  int need = p.count;
#pragma unroll 1  // instructions of a second pass are at hand, a second copy's are not
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    const uint32_t mask = pass == 0 ? 0u : 0xFFFFFFFFu << (shift + 8);
    for (int j = threadIdx.x; j < n; j += THREADS) {
      const uint32_t key = own[j];
      if ((key & mask) == threshold) atomicAdd(&histogram[pass][key >> shift & 255], 1);
    }
    __syncthreads();
    // lane i holds bins 255 - 8 i down to 248 - 8 i
    const int4 hi = *reinterpret_cast<const int4*>(&histogram[pass][252 - 8 * lane]);
    const int4 lo = *reinterpret_cast<const int4*>(&histogram[pass][248 - 8 * lane]);
    const int v[8] = {hi.w, hi.z, hi.y, hi.x, lo.w, lo.z, lo.y, lo.x};
    int sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[i];
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += u;
    }
    before -= sum;
    int bin = -1, left = 0, held = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (bin < 0 && before < need && before + v[i] >= need) bin = 255 - 8 * lane - i, left = need - before, held = v[i];
      before += v[i];
    }
    const int owner = __ffs(__ballot_sync(0xffffffffu, bin >= 0)) - 1;
    bin = __shfl_sync(0xffffffffu, bin, owner);
    need = __shfl_sync(0xffffffffu, left, owner);
    held = __shfl_sync(0xffffffffu, held, owner);
    threshold |= (uint32_t)bin << shift;
    if (held == need) {  // every key from the threshold on
      threshold -= threshold > 0;  // no key is 0
      need = 0;
      break;
    }
  }

  // ---- kept blocks in ascending order: each thread a contiguous slice; of the keys equal to the threshold the
  // first `need`
  const int slice = (n + THREADS - 1) / THREADS;
  const int j0 = min(n, (int)threadIdx.x * slice), j1 = min(n, j0 + slice);
  int above = 0, equal = 0;
  for (int j = j0; j < j1; ++j) {
    const uint32_t key = own[j];
    above += key > threshold;
    equal += key == threshold;
  }
  int above_in = above, equal_in = equal;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, above_in, o), v = __shfl_up_sync(0xffffffffu, equal_in, o);
    if (lane >= o) above_in += u, equal_in += v;
  }
  if (lane == 31) warp_counts[warp] = make_int2(above_in, equal_in);
  __syncthreads();
  int above_before = above_in - above, equal_before = equal_in - equal;
  for (int w = 0; w < warp; ++w) above_before += warp_counts[w].x, equal_before += warp_counts[w].y;
  int at = above_before + min(equal_before, need);
  for (int j = j0; j < j1; ++j) {
    const uint32_t key = own[j];
    if (key > threshold || (key == threshold && equal_before < need)) out[at++] = j;
    equal_before += key == threshold;
  }
}

template <typename T, int D> int launch_select(const SelectParams& p, cudaStream_t stream) {
  static bool ready[64] = {false};  // the attribute is a device's; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (!ready[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(select_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               MOST_SHARED_KEYS * 4);
    if (e != cudaSuccess) return ucb_host::set_error(UCB_ERR_CUDA, "ucb_block8_select: %s", cudaGetErrorString(e));
    ready[dev & 63] = true;
  }
  const int64_t pairs = (int64_t)p.c.num_seqs * p.c.kv_heads;
  // CTAs of a pair: until every warp has a tile, as long as the chip has room for more (two on a multiprocessor)
  const int64_t room = 2 * ucb_host::multiprocessors();
  int parts = 1;
  while (parts < 8 && pairs * parts * 2 <= room && p.c.max_blocks > parts * 16 * WARPS) parts *= 2;
  return block8::launch(select_kernel<T, D>, dim3((unsigned)(pairs * parts)), dim3(THREADS),
                        p.spill ? 16 : (size_t)p.c.max_blocks * 4, stream, p, "block8 select_kernel", parts);
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

extern "C" int64_t ucb_block8_select_workspace_bytes(const ucb_block8_cache* cache) {
  if (b8::check_cache(cache, "ucb_block8_select_workspace_bytes")) return -1;
  if (cache->max_blocks <= b8::MOST_SHARED_KEYS) return 0;
  return (int64_t)cache->num_seqs * cache->kv_heads * cache->max_blocks * 4;
}

extern "C" int ucb_block8_select(const ucb_block8_cache* cache, const void* query, int64_t q_ss, int64_t q_sh,
                                 int q_heads, int count, int first, int recent, int32_t* blocks, void* workspace,
                                 void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_select")) return rc;
  const bool spill = cache->max_blocks > b8::MOST_SHARED_KEYS;
  if (!query || !blocks || (spill && !workspace)) return set_error(UCB_ERR_INVALID, "ucb_block8_select: null pointer");
  if (q_heads < 1 || q_heads % cache->kv_heads)
    return set_error(UCB_ERR_INVALID, "ucb_block8_select: query heads must be divisible by KV heads");
  if (first < 0 || recent < 0 || count < 1 || (int64_t)first + recent > count)
    return set_error(UCB_ERR_INVALID, "ucb_block8_select: need first + recent <= count and count >= 1");
  if (count > 4096) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_select: at most 4096 blocks");
  if ((int64_t)cache->num_seqs * cache->kv_heads > 0x0fffffff)
    return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_select: too many sequences and heads");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_block8_select: device error word unavailable");
  const b8::SelectParams p{*cache, query, q_ss, q_sh, q_heads / cache->kv_heads, count, first, recent, blocks,
                           spill ? static_cast<uint32_t*>(workspace) : nullptr, err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = cache->dtype == UCB_BF16;
  if (cache->head_dim == 128)
    return bf ? b8::launch_select<__nv_bfloat16, 128>(p, s) : b8::launch_select<__half, 128>(p, s);
  return bf ? b8::launch_select<__nv_bfloat16, 64>(p, s) : b8::launch_select<__half, 64>(p, s);
}
