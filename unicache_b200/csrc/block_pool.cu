// Blocks of the 8-bit block cache given to sequences, shared, copied and moved
// (ucb_block_pool_*).  The state is whole numbers on the device: the table, each
// sequence's length and number of blocks, and for each block how many table
// entries name it.  A free block (no entry) is always the lowest one, so every
// result is defined; what has to be found in order is found by one cluster of CTAs
// that ranks the pool's free blocks.
#include <cooperative_groups.h>

#include <algorithm>

#include "block8.cuh"

namespace ucb {
namespace block8 {
namespace {

namespace cg = cooperative_groups;

constexpr int PLAN_THREADS = 1024;
constexpr int MAX_SEQS = 4096;
constexpr int EACH = MAX_SEQS / PLAN_THREADS;  // sequences (pairs) a thread
constexpr int MAX_CLUSTER = 8;
constexpr int LANE_BLOCKS = 32;  // blocks a lane holds at once, a bit each

struct PoolParams {
  ucb_block_pool pool;
  unsigned int* err;
};

// Sum of the threads' values in front of this one, and of all.
template <typename V> __device__ __forceinline__ V scan_block(V mine, V* warp_sum, V& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V v = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
  __syncthreads();  // warp_sum may still be read
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  V w = lane < PLAN_THREADS / 32 ? warp_sum[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += x;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const V before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return v - mine + (warp ? before : 0);
}

// The references from `first` on, `per` of them: bit i set where block first + i is referred to by no entry.  Blocks past the
// pool have no bit.
__device__ __forceinline__ uint32_t free_bits(const int32_t* references, int64_t n, int64_t first, int per) {
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < LANE_BLOCKS / 4; ++k) {
    const int64_t at = first + 4 * k;
    if (4 * k >= per || at >= n) continue;
    int4 v = make_int4(1, 1, 1, 1);
    if (at + 4 <= n) {
      v = *reinterpret_cast<const int4*>(references + at);
    } else {
      v.x = references[at];
      if (at + 1 < n) v.y = references[at + 1];
      if (at + 2 < n) v.z = references[at + 2];
    }
    bits |= ((v.x == 0) | (v.y == 0) << 1 | (v.z == 0) << 2 | (v.w == 0) << 3) << (4 * k);
  }
  return bits;
}

// A cluster's pass over the pool in ascending order: in each round a lane has `per` adjacent blocks.
struct Pass {
  int rank, ctas, per;
  int64_t round_blocks;
  __device__ explicit Pass(int64_t n) {
    cg::cluster_group cluster = cg::this_cluster();
    rank = cluster.block_rank(), ctas = cluster.num_blocks();
    const int64_t threads = (int64_t)ctas * PLAN_THREADS, each = (n + threads - 1) / threads;
    per = (int)min((int64_t)LANE_BLOCKS, (each + 3) / 4 * 4);
    round_blocks = threads * per;
  }
  __device__ int64_t first(int64_t round) const {
    return round * round_blocks + ((int64_t)rank * PLAN_THREADS + threadIdx.x) * per;
  }
  // A barrier of the cluster in two halves, for what lies between not to wait: every CTA runs, and has passed arrive(), behind wait().
  __device__ void arrive() const {
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  }
  __device__ void wait() const {
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
};

struct RankSpace {
  int warp_sum[32];
  int cta_total[2][MAX_CLUSTER];  // every CTA's, by turns: the last round's may still be read
};

// How many of the round's marked blocks are in front of this thread's `mine`, and the round's in all, over the cluster.  It stores into
// the other CTAs' shared memory: behind a barrier of the cluster, since a CTA's memory is there once it runs.
__device__ __forceinline__ int rank_round(RankSpace& space, const Pass& pass, int mine, int turn, int& total) {
  int before = scan_block(mine, space.warp_sum, total);
  if (pass.ctas == 1) return before;
  cg::cluster_group cluster = cg::this_cluster();
  if (threadIdx.x < pass.ctas) *cluster.map_shared_rank(&space.cta_total[turn & 1][pass.rank], threadIdx.x) = total;
  cluster.sync();
  total = 0;
#pragma unroll
  for (int r = 0; r < MAX_CLUSTER; ++r) {
    const int t = r < pass.ctas ? space.cta_total[turn & 1][r] : 0;
    if (r < pass.rank) before += t;
    total += t;
  }
  return before;
}

// ---------------------------------------------------------------- release
struct ReleaseParams {
  PoolParams p;
  const int32_t* sequences;
};

// One CTA a sequence.  Whoever takes the number of its blocks gives them back, so a sequence named twice is released once.
__global__ void __launch_bounds__(256) release_kernel(const ReleaseParams q) {
  const ucb_block_pool& pool = q.p.pool;
  __shared__ int blocks;
  const int s = q.sequences[blockIdx.x];
  if (s < 0 || s >= pool.num_seqs) {
    if (threadIdx.x == 0) atomicOr(q.p.err, DEVERR_BAD_DESCRIPTOR);
    return;
  }
  if (threadIdx.x == 0) {
    blocks = min(atomicExch(&pool.held[s], 0), pool.max_blocks);
    pool.lengths[s] = 0;
  }
  __syncthreads();
  int32_t* row = pool.block_table + (int64_t)s * pool.max_blocks;
  for (int j = threadIdx.x; j < blocks; j += blockDim.x) {
    const int b = row[j];
    row[j] = -1;
    if (b >= 0 && b < pool.num_blocks) {
      atomicSub(&pool.references[b], 1);
    } else {
      atomicOr(q.p.err, DEVERR_BAD_DESCRIPTOR);
    }
  }
}

// ---------------------------------------------------------------- advance
struct AdvanceParams {
  PoolParams p;
  const int32_t* tokens;
  int each;
};

// A sequence that grows from a block's start may hold that block from a longer length, and others may share it: its rows would
// change theirs.  Then the entries from there on are given back, before blocks are taken (only leading blocks are
// shared, so where that one is not, none behind it is).
// Most steps of a decode want no block and end after the lengths: 3.3 us for 32 sequences, 4.0 for 2048, whatever the pool (3.7 and 4.5
// with divisions by the block's tokens); where 8 sequences end and as many prompts of up to 256 blocks come in 8.2 with the
// release.  Whether a block is shared costs the calls that ask 0.5.
__global__ void __launch_bounds__(PLAN_THREADS) advance_kernel(const AdvanceParams q) {
  const ucb_block_pool& pool = q.p.pool;
  __shared__ int base[MAX_SEQS];   // blocks wanted by the sequences in front of each, 2^31 - 1 for more than that
  __shared__ int start[MAX_SEQS];  // where in a sequence's row the block of rank 0 would be
  __shared__ int64_t wide_sum[32];
  __shared__ RankSpace space;
  const int seqs = pool.num_seqs, bt = pool.block_tokens, shift = 31 - __clz(bt);  // a power of two
  const Pass pass(pool.num_blocks);
  int length[EACH], held[EACH], want[EACH];
  int64_t mine = 0, wanted;
  bool bad = false;
  unsigned given_back = 0;  // bit i: the thread's i-th sequence
  auto shared = [&](int s, int j) {
    const int b = pool.block_table[(int64_t)s * pool.max_blocks + j];
    return b >= 0 && b < pool.num_blocks && pool.references[b] > 1;
  };
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = threadIdx.x * EACH + i;
    length[i] = held[i] = want[i] = 0;
    if (s >= seqs) continue;
    const int before = pool.lengths[s];
    const int64_t most = (int64_t)pool.max_blocks << shift;
    int64_t t = (int64_t)before + (q.tokens ? q.tokens[s] : q.each);
    held[i] = pool.held[s];
    bad |= t < 0 || t > most;
    if (t < before) {
      if (t > 0 && (t & (bt - 1)) && t < most && shared(s, (int)(t >> shift))) t = before, bad = true;  // the next write would change it
    } else if (t > before && before >= 0 && (before & (bt - 1)) == 0 && (before >> shift) < min(held[i], pool.max_blocks) &&
               shared(s, before >> shift)) {
      held[i] = before >> shift, given_back |= 1u << i;
    }
    length[i] = (int)max((int64_t)0, min(t, (int64_t)0x7fffffff));
    want[i] = max(0, (int)((min((int64_t)length[i], most) + bt - 1) >> shift) - held[i]);
    mine += want[i];
  }
  pass.arrive();  // lengths, table, references and numbers of blocks are read
  int64_t at = scan_block(mine, wide_sum, wanted);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = threadIdx.x * EACH + i;
    if (s < seqs) {
      base[s] = (int)min(at, (int64_t)0x7fffffff);
      start[s] = held[i] - base[s];
    }
    at += want[i];
  }
  const bool any_given_back = __syncthreads_or(given_back);  // the same in every CTA
  pass.wait();
  if (any_given_back) {
    if (pass.rank == 0) {
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        for (unsigned lanes = __ballot_sync(0xffffffffu, given_back >> i & 1); lanes; lanes &= lanes - 1) {
          const int owner = __ffs(lanes) - 1, s = ((threadIdx.x & ~31) + owner) * EACH + i;
          const int from = __shfl_sync(0xffffffffu, held[i], owner), to = min(pool.held[s], pool.max_blocks);
          int32_t* row = pool.block_table + (int64_t)s * pool.max_blocks;
          for (int j = from + lane; j < to; j += 32) {
            const int b = row[j];
            row[j] = -1;
            if (b >= 0 && b < pool.num_blocks) atomicSub(&pool.references[b], 1); else bad = true;
          }
        }
    }
    if (pass.ctas > 1) cg::this_cluster().sync(); else __syncthreads();
  }
  int64_t found = 0;
  for (int round = 0; found < wanted && round * pass.round_blocks < pool.num_blocks; ++round) {
    const int64_t first = pass.first(round);
    uint32_t bits = free_bits(pool.references, pool.num_blocks, first, pass.per);
    int total;
    int64_t r = found + rank_round(space, pass, __popc(bits), round, total);
    if (bits && r < wanted) {
      int s = 0, n = seqs;  // the last sequence whose blocks begin at r or before: the one that wants this one
      while (n > 1) {
        const int half = n / 2;
        if (base[s + half] <= r) s += half, n -= half; else n = half;
      }
      int32_t* row = pool.block_table + (int64_t)s * pool.max_blocks + start[s];
      for (; bits && r < wanted; bits &= bits - 1, ++r) {
        if (s + 1 < seqs && base[s + 1] <= r) {  // the next one that wants any
          do ++s;
          while (s + 1 < seqs && base[s + 1] <= r);
          row = pool.block_table + (int64_t)s * pool.max_blocks + start[s];
        }
        const int block = (int)(first + __ffs(bits) - 1);
        pool.references[block] = 1;
        row[r] = block;
      }
    }
    found += total;
  }
  if (pass.rank) return;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = threadIdx.x * EACH + i;
    if (s >= seqs) continue;
    pool.lengths[s] = length[i];
    const int64_t given = max((int64_t)0, min((int64_t)want[i], found - base[s]));
    if (given || (given_back >> i & 1)) pool.held[s] = held[i] + (int)given;
    bad |= given < want[i];
  }
  if (bad) atomicOr(q.p.err, DEVERR_BAD_DESCRIPTOR);
}

// ---------------------------------------------------------------- fork
struct ForkParams {
  PoolParams p;
  const int32_t *parents, *children;
  int count;
  int4* jobs;  // of each pair: source and target block of its incomplete block (a JobKind: nothing to copy), parent and above it rows, child
};

enum PairState : int { SKIPPED = -2, WHOLE = -1 };  // otherwise the rank of the block that the pair takes
enum JobKind : int { AT_A_BLOCKS_END = -2, NO_JOB = -1 };

__global__ void __launch_bounds__(PLAN_THREADS) fork_kernel(const ForkParams q) {
  const ucb_block_pool& pool = q.p.pool;
  __shared__ int state[MAX_SEQS];      // first the lowest pair that names a sequence as its child, then each pair's state
  __shared__ int pair_of[MAX_SEQS];    // the pair that takes the block of a rank
  __shared__ RankSpace space;
  const int bt = pool.block_tokens, W = pool.max_blocks;
  const Pass pass(pool.num_blocks);
  launch_dependents();
  for (int i = threadIdx.x; i < MAX_SEQS; i += PLAN_THREADS) state[i] = 0x7fffffff;
  __syncthreads();
  int parent[EACH], child[EACH], mine[EACH];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = threadIdx.x * EACH + e;
    mine[e] = SKIPPED;
    if (i >= q.count) continue;
    parent[e] = q.parents[i], child[e] = q.children[i];
    if (parent[e] < 0 || parent[e] >= pool.num_seqs || child[e] < 0 || child[e] >= pool.num_seqs) {
      bad = true;
    } else if (parent[e] != child[e]) {
      mine[e] = WHOLE;
      atomicMin(&state[child[e]], i);
    }
  }
  __syncthreads();
  int copies = 0, wanted;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = threadIdx.x * EACH + e;
    if (mine[e] == SKIPPED) continue;
    const int length = pool.lengths[parent[e]];
    if (state[child[e]] != i || state[parent[e]] != 0x7fffffff || length < 0 || length > (int64_t)W * bt ||
        (length + bt - 1) / bt > pool.held[parent[e]]) {
      mine[e] = SKIPPED, bad = true;
    } else if (length % bt) {
      mine[e] = copies++;
    }
  }
  const int before = scan_block(copies, space.warp_sum, wanted);  // its barriers: every owner is read
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int i = threadIdx.x * EACH + e;
    if (i >= q.count) continue;
    if (mine[e] >= 0) pair_of[mine[e] += before] = i;
    state[i] = mine[e];
  }
  __syncthreads();
  // the children's blocks are given back, a warp a pair
  const int lane = threadIdx.x & 31, warp = pass.rank * (PLAN_THREADS / 32) + (threadIdx.x >> 5);
  const int warps = pass.ctas * (PLAN_THREADS / 32);
  for (int i = warp; i < q.count; i += warps) {
    if (state[i] == SKIPPED) continue;
    const int c = q.children[i], held = min(pool.held[c], W);
    int32_t* row = pool.block_table + (int64_t)c * W;
    for (int j = lane; j < held; j += 32) {
      const int b = row[j];
      row[j] = -1;
      if (b >= 0 && b < pool.num_blocks) atomicSub(&pool.references[b], 1); else bad = true;
    }
  }
  if (pass.ctas > 1) cg::this_cluster().sync(); else __syncthreads();
  // blocks for the copies
  int64_t found = 0;
  for (int round = 0; found < wanted && round * pass.round_blocks < pool.num_blocks; ++round) {
    const int64_t first = pass.first(round);
    uint32_t bits = free_bits(pool.references, pool.num_blocks, first, pass.per);
    int total;
    int64_t r = found + rank_round(space, pass, __popc(bits), round, total);
    for (; bits && r < wanted; bits &= bits - 1, ++r) {
      const int block = (int)(first + __ffs(bits) - 1);
      pool.references[block] = 1;
      q.jobs[pair_of[r]].y = block;
    }
    found += total;
  }
  if (pass.ctas > 1) cg::this_cluster().sync(); else __syncthreads();
  // the children's rows
  for (int i = warp; i < q.count; i += warps) {
    const int s = state[i], from = q.parents[i], to = q.children[i];
    if (s == SKIPPED) {
      if (lane == 0) q.jobs[i].y = NO_JOB;
      continue;
    }
    const int length = pool.lengths[from], shared = length / bt;
    const bool fits = s == WHOLE || s < found;
    const int32_t* source = pool.block_table + (int64_t)from * W;
    int32_t* row = pool.block_table + (int64_t)to * W;
    for (int j = lane; fits && j < shared; j += 32) {
      const int b = source[j];
      row[j] = b;
      if (b >= 0 && b < pool.num_blocks) atomicAdd(&pool.references[b], 1); else bad = true;
    }
    if (lane == 0) {
      int4 job = make_int4(-1, s == WHOLE ? AT_A_BLOCKS_END : NO_JOB, from | (length % bt) << 24, to);
      if (s >= 0 && fits) {
        const int b = source[shared], block = q.jobs[i].y;
        row[shared] = block;
        if (b >= 0 && b < pool.num_blocks) job.x = b, job.y = block; else bad = true;
      }
      q.jobs[i] = job;
      pool.lengths[to] = fits ? length : 0;
      pool.held[to] = fits ? shared + (s >= 0) : 0;
      bad |= !fits;
    }
  }
  if (bad) atomicOr(q.p.err, DEVERR_BAD_DESCRIPTOR);
}

// A piece of memory to be copied by a group of threads, 16 bytes at a time: loaded first, stored when other loads are on their way.
template <int AHEAD> struct Piece {
  uint4 x[AHEAD];
  __device__ __forceinline__ void load(const void* from, int bytes, int thread, int threads) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (thread + k * threads < bytes / 16) x[k] = static_cast<const uint4*>(from)[thread + k * threads];
  }
  __device__ __forceinline__ void store(void* to, int bytes, int thread, int threads) const {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (thread + k * threads < bytes / 16) static_cast<uint4*>(to)[thread + k * threads] = x[k];
  }
};

struct ForkCopyParams {
  const int4* jobs;
  const ucb_block8_cache* caches;
};

constexpr int FORK_WARPS = 4;

// Pair blockIdx.x, layer blockIdx.y; a warp copies a head's keys or values: the codes of the rows that count, the rows themselves, and
// of the keys the record of whose rows they are and the bounds.  What a warp copies is a few KB and waits for the pair, then for
// the data: 56 pairs x 28 layers x 4 heads x 128 (203 MB, as seven children read the same parent) in 39 us; a CTA for each head took 142.
__global__ void __launch_bounds__(FORK_WARPS * 32) fork_copy_kernel(const ForkCopyParams q) {
  const ucb_block8_cache c = q.caches[blockIdx.y];
  const int lane = threadIdx.x & 31, item = blockIdx.z * FORK_WARPS + (threadIdx.x >> 5), h = item >> 1, value = item & 1;
  if (h >= c.kv_heads) return;
  wait_for_primary();
  const int4 job = q.jobs[blockIdx.x];
  const int rows = job.z >> 24, parent = job.z & 0xffffff, child = job.w;
  if (job.y == AT_A_BLOCKS_END && !value && lane == 0) {
    // The block is shared from now on, so neither may write into its middle, wherever their lengths are taken back to; and what the child's
    // slot holds is another sequence's.  Rows without a record are their owner's affair: where neither was ever written to they stay.
    // (Other pairs of the parent may do the same at once: either record of the parent's begins with RECORD.)
    uint4 *of_child = pending_record(c, child, h), *of_parent = pending_record(c, parent, h);
    const bool written = of_parent->x == RECORD;
    if (written) *of_parent = record_of_nothing();
    if (written || is_record(*of_child)) *of_child = record_of_nothing();
  }
  if (job.y < 0) return;
  const int64_t block = (int64_t)c.block_tokens * c.head_dim;
  const int64_t from = (int64_t)job.x * c.kv_heads + h, to = (int64_t)job.y * c.kv_heads + h;
  int8_t* code = value ? c.value_code : c.key_code;
  const int8_t* code_from = code + from * block;
  int8_t* code_to = code + to * block;
  char* pending = static_cast<char*>(value ? c.pending_value : c.pending_key);
  const char* pending_from = pending + ((int64_t)parent * c.kv_heads + h) * block * 2;
  char* pending_to = pending + ((int64_t)child * c.kv_heads + h) * block * 2;
  // the bounds and the record: of 16 bytes a lane, head_dim / 16 lanes each of the bounds, head_dim / 8 of the record
  const int bound_lanes = value ? 0 : c.head_dim / 16, record_lanes = value ? 0 : c.head_dim / 8;
  const int64_t record = (block - c.head_dim) * 2;
  uint4 low, high, rec;
  if (lane < bound_lanes) {
    low = reinterpret_cast<const uint4*>(c.key_low + from * c.head_dim)[lane];
    high = reinterpret_cast<const uint4*>(c.key_high + from * c.head_dim)[lane];
  }
  if (lane < record_lanes) rec = reinterpret_cast<const uint4*>(pending_from + record)[lane];
  float* scale = value ? c.value_scale : c.key_scale;
  const float scale_from = scale[from];
  constexpr int CODES = 4, ROWS = 8, STEP = CODES * 32 * 16;  // bytes of codes at a time, and twice as many of rows
  const int bytes = rows * c.head_dim;
  for (int at = 0; at < bytes; at += STEP) {
    Piece<CODES> codes;
    Piece<ROWS> held;
    codes.load(code_from + at, bytes - at, lane, 32);
    held.load(pending_from + 2 * at, 2 * (bytes - at), lane, 32);
    codes.store(code_to + at, bytes - at, lane, 32);
    held.store(pending_to + 2 * at, 2 * (bytes - at), lane, 32);
  }
  if (lane < bound_lanes) {
    reinterpret_cast<uint4*>(c.key_low + to * c.head_dim)[lane] = low;
    reinterpret_cast<uint4*>(c.key_high + to * c.head_dim)[lane] = high;
  }
  if (lane < record_lanes) reinterpret_cast<uint4*>(pending_to + record)[lane] = rec;
  if (lane == 0) scale[to] = scale_from;
}

// ---------------------------------------------------------------- compact
struct CompactParams {
  PoolParams p;
  int32_t* live;    // the number of live blocks, for the caller
  int32_t* moves;   // the number of moved ones
  int32_t* holes;   // targets in ascending order
  int32_t* movers;  // sources in ascending order
  int32_t* place;   // of a moved block
  const ucb_block8_cache* caches;
  int layers;
};

__global__ void __launch_bounds__(PLAN_THREADS) compact_kernel(const CompactParams q) {
  const ucb_block_pool& pool = q.p.pool;
  __shared__ RankSpace space;
  const Pass pass(pool.num_blocks);
  launch_dependents();
  pass.arrive();
  int64_t live = pool.num_blocks;
  int turn = 0, total;
  for (int round = 0; round * pass.round_blocks < pool.num_blocks; ++round) {
    const int free = __popc(free_bits(pool.references, pool.num_blocks, pass.first(round), pass.per));
    if (round == 0) pass.wait();
    rank_round(space, pass, free, turn++, total);
    live -= total;
  }
  // the i-th live block behind the live count goes to the i-th hole in front of it: as many are the ones as the others
  int64_t holes = 0, movers = 0;
  for (int round = 0; round * pass.round_blocks < pool.num_blocks; ++round) {
    const int64_t first = pass.first(round), front = max((int64_t)0, min((int64_t)32, live - first));
    const int64_t inside = max((int64_t)0, min((int64_t)pass.per, pool.num_blocks - first));
    const uint32_t before_live = front >= 32 ? 0xffffffffu : (1u << front) - 1, in_pool = inside >= 32 ? 0xffffffffu : (1u << inside) - 1;
    const uint32_t free = free_bits(pool.references, pool.num_blocks, first, pass.per);
    uint32_t hole = free & before_live, mover = ~free & in_pool & ~before_live;
    int64_t r = holes + rank_round(space, pass, __popc(hole), turn++, total);
    holes += total;
    for (; hole; hole &= hole - 1, ++r) q.holes[r] = (int)(first + __ffs(hole) - 1);
    r = movers + rank_round(space, pass, __popc(mover), turn++, total);
    movers += total;
    for (; mover; mover &= mover - 1, ++r) q.movers[r] = (int)(first + __ffs(mover) - 1);
  }
  if (pass.ctas > 1) cg::this_cluster().sync(); else __syncthreads();
  for (int64_t i = (int64_t)pass.rank * PLAN_THREADS + threadIdx.x; i < movers; i += (int64_t)pass.ctas * PLAN_THREADS) {
    const int from = q.movers[i], to = q.holes[i];
    pool.references[to] = pool.references[from];
    pool.references[from] = 0;
    q.place[from] = to;
  }
  if (pass.rank == 0 && threadIdx.x == 0) *q.live = (int)live, *q.moves = (int)movers;
}

constexpr int MOVE_THREADS = 256;

// The moved blocks, and the table's entries.  blockIdx.y is a layer's keys or values, whose addresses a CTA looks up once; it
// goes from move to move, the next one's blocks known before.
__global__ void __launch_bounds__(MOVE_THREADS) compact_copy_kernel(const CompactParams q) {
  const ucb_block_pool& pool = q.p.pool;
  const ucb_block8_cache& c = q.caches[blockIdx.y >> 1];
  const int value = blockIdx.y & 1, heads = c.kv_heads, bound_bytes = heads * c.head_dim;
  const int64_t block = (int64_t)bound_bytes * c.block_tokens;
  int8_t* code = value ? c.value_code : c.key_code;
  int8_t* bound = value ? c.key_high : c.key_low;
  float* scale = value ? c.value_scale : c.key_scale;
  wait_for_primary();
  const int live = *q.live, moves = *q.moves;
  if (moves == 0) return;
  int k = blockIdx.x;
  int64_t from = 0, to = 0;
  if (k < moves) from = q.movers[k], to = q.holes[k];
  while (k < moves) {
    const int8_t* code_from = code + from * block;
    int8_t* code_to = code + to * block;
    const int8_t* bound_from = bound + from * bound_bytes;
    int8_t* bound_to = bound + to * bound_bytes;
    const float* scale_from = scale + from * heads;
    float* scale_to = scale + to * heads;
    k += gridDim.x;
    if (k < moves) from = q.movers[k], to = q.holes[k];
    for (int at = threadIdx.x * 16; at < bound_bytes; at += MOVE_THREADS * 16)
      *reinterpret_cast<uint4*>(bound_to + at) = *reinterpret_cast<const uint4*>(bound_from + at);
    for (int h = threadIdx.x; h < heads; h += MOVE_THREADS) scale_to[h] = scale_from[h];
    constexpr int AHEAD = 8, STEP = AHEAD * MOVE_THREADS * 16;
    for (int64_t at = 0; at < block; at += STEP) {
      Piece<AHEAD> x;
      const int bytes = (int)min((int64_t)STEP, block - at);
      x.load(code_from + at, bytes, threadIdx.x, MOVE_THREADS);
      x.store(code_to + at, bytes, threadIdx.x, MOVE_THREADS);
    }
  }
  const int cta = blockIdx.y * gridDim.x + blockIdx.x, ctas = gridDim.x * gridDim.y;
  for (int s = cta; s < pool.num_seqs; s += ctas) {
    int32_t* row = pool.block_table + (int64_t)s * pool.max_blocks;
    const int held = min(pool.held[s], pool.max_blocks);
    for (int j = threadIdx.x; j < held; j += MOVE_THREADS) {
      const int b = row[j];
      if (b >= live && b < pool.num_blocks) row[j] = q.place[b];
    }
  }
}

// ---------------------------------------------------------------- host side
int check_pool(const ucb_block_pool* p, const char* what) {
  using ucb_host::set_error;
  if (!p || !p->block_table || !p->lengths || !p->held || !p->references)
    return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (p->num_seqs < 1 || p->max_blocks < 1 || p->num_blocks < 1) return set_error(UCB_ERR_INVALID, "%s: bad shape", what);
  if (p->num_seqs > MAX_SEQS) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most %d sequences", what, MAX_SEQS);
  if (p->num_blocks > 0x7fffffff) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 blocks", what);
  if (p->block_tokens != 16 && p->block_tokens != 32 && p->block_tokens != 64 && p->block_tokens != 128)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: block_tokens must be 16, 32, 64 or 128", what);
  if ((int64_t)p->max_blocks * p->block_tokens > 0x7fffffff)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: a sequence holds at most 2^31 - 1 tokens", what);
  if (reinterpret_cast<uintptr_t>(p->references) & 15)
    return set_error(UCB_ERR_INVALID, "%s: references must be 16-byte aligned", what);
  return UCB_OK;
}

// One CTA for pools of up to 16 blocks a thread, for larger ones more: admission of 256 of 2048 sequences to a pool of 110000 blocks
// takes 16.9 us so and 21.0 with 32 a thread; with 4 the cluster's start costs a pool of 8600 blocks 0.8 us.
int plan_cluster(int64_t blocks) {
  int ctas = 1;
  while (ctas < MAX_CLUSTER && (int64_t)ctas * PLAN_THREADS * 16 < blocks) ctas *= 2;
  return ctas;
}

int check_layers(const void* caches, int layers, int kv_heads, const char* what) {
  if (!caches || layers < 1 || kv_heads < 1) return ucb_host::set_error(UCB_ERR_INVALID, "%s: no caches", what);
  if (layers > 32767 || kv_heads > 32767)
    return ucb_host::set_error(UCB_ERR_UNSUPPORTED, "%s: at most 32767 caches of 32767 KV heads", what);
  if (reinterpret_cast<uintptr_t>(caches) & 7) return ucb_host::set_error(UCB_ERR_INVALID, "%s: caches must be 8-byte aligned", what);
  return UCB_OK;
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

extern "C" int ucb_block_pool_release(const ucb_block_pool* pool, const int32_t* sequences, int count, void* stream) {
  const char* what = "ucb_block_pool_release";
  if (int rc = b8::check_pool(pool, what)) return rc;
  if (count < 0) return set_error(UCB_ERR_INVALID, "%s: bad count", what);
  if (count == 0) return UCB_OK;
  if (!sequences) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  const b8::ReleaseParams q{{*pool, err}, sequences};
  return b8::launch(b8::release_kernel, dim3(count), dim3(256), 0, static_cast<cudaStream_t>(stream), q, "block pool release_kernel");
}

extern "C" int ucb_block_pool_advance(const ucb_block_pool* pool, const int32_t* tokens, int each, void* stream) {
  const char* what = "ucb_block_pool_advance";
  if (int rc = b8::check_pool(pool, what)) return rc;
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  const b8::AdvanceParams q{{*pool, err}, tokens, each};
  return b8::launch(b8::advance_kernel, dim3(b8::plan_cluster(pool->num_blocks)), dim3(b8::PLAN_THREADS), 0,
                    static_cast<cudaStream_t>(stream), q, "block pool advance_kernel", b8::plan_cluster(pool->num_blocks));
}

extern "C" int64_t ucb_block_pool_fork_workspace_bytes(int count) { return count < 0 ? -1 : (int64_t)count * 16; }

extern "C" int ucb_block_pool_fork(const ucb_block_pool* pool, const int32_t* parents, const int32_t* children, int count,
                                   const ucb_block8_cache* caches, int layers, int kv_heads, void* workspace, void* stream) {
  const char* what = "ucb_block_pool_fork";
  if (int rc = b8::check_pool(pool, what)) return rc;
  if (count < 0 || count > pool->num_seqs) return set_error(UCB_ERR_INVALID, "%s: at most one pair for each sequence", what);
  if (int rc = b8::check_layers(caches, layers, kv_heads, what)) return rc;
  if (count == 0) return UCB_OK;
  if (!parents || !children || !workspace) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_error(UCB_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const b8::ForkParams q{{*pool, err}, parents, children, count, static_cast<int4*>(workspace)};
  // a warp a pair: many pairs have the widest cluster (56 pairs of 64 blocks 50.4 us against 51.8; 7 pairs 12.0 against 10.2)
  const int ctas = count > b8::PLAN_THREADS / 32 ? b8::MAX_CLUSTER : b8::plan_cluster(pool->num_blocks);
  if (int rc = b8::launch(b8::fork_kernel, dim3(ctas), dim3(b8::PLAN_THREADS), 0, s, q, "block pool fork_kernel", ctas)) return rc;
  const b8::ForkCopyParams c{q.jobs, caches};
  return b8::launch(b8::fork_copy_kernel, dim3(count, layers, (2 * kv_heads + b8::FORK_WARPS - 1) / b8::FORK_WARPS),
                    dim3(b8::FORK_WARPS * 32), 0, s, c, "block pool fork_copy_kernel", 1, true);
}

// The number of moves, then holes and movers (half of the pool at most each), then every block's place.
extern "C" int64_t ucb_block_pool_compact_workspace_bytes(const ucb_block_pool* pool) {
  if (b8::check_pool(pool, "ucb_block_pool_compact_workspace_bytes")) return -1;
  return 4 * (4 + 2 * (pool->num_blocks / 2) + pool->num_blocks);
}

extern "C" int ucb_block_pool_compact(const ucb_block_pool* pool, const ucb_block8_cache* caches, int layers, int kv_heads,
                                      int32_t* live, void* workspace, void* stream) {
  const char* what = "ucb_block_pool_compact";
  if (int rc = b8::check_pool(pool, what)) return rc;
  if (int rc = b8::check_layers(caches, layers, kv_heads, what)) return rc;
  if (!live || !workspace) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(workspace) & 3) return set_error(UCB_ERR_INVALID, "%s: workspace must be 4-byte aligned", what);
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int32_t* w = static_cast<int32_t*>(workspace);
  const int64_t half = pool->num_blocks / 2;
  const b8::CompactParams q{{*pool, err}, live, w, w + 4, w + 4 + half, w + 4 + 2 * half, caches, layers};
  const int ctas = b8::plan_cluster(pool->num_blocks);
  if (int rc = b8::launch(b8::compact_kernel, dim3(ctas), dim3(b8::PLAN_THREADS), 0, s, q, "block pool compact_kernel", ctas)) return rc;
  const int sms = ucb_host::multiprocessors();
  if (sms < 1) return set_error(UCB_ERR_CUDA, "%s: the device's multiprocessors are unknown", what);
  // CTAs of a few moves each, spread over the layers' keys and values: 390 moves in 28 layers (917 MB there and back, with the
  // admission around them) take 153 us with 64 a multiprocessor, of which three are resident; with 8 173, with 200 165
  const int64_t across = std::max<int64_t>(1, std::min<int64_t>(std::max<int64_t>(half, 1), (int64_t)sms * 64 / (2 * layers)));
  return b8::launch(b8::compact_copy_kernel, dim3((unsigned)across, 2 * layers), dim3(b8::MOVE_THREADS), 0, s, q,
                    "block pool compact_copy_kernel", 1, true);
}
