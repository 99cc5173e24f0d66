// Attention over the 8-bit block cache (ucb_block8_attention): one to sixteen
// query tokens a sequence, split over the whole chip.
//
//   s_t = softmax_scale * key_scale[b(t)] * (q . ck_t),   w_t = exp(s_t - max),
//   o   = sum_b value_scale[b] * sum_{t in b} w_t cv_t  /  sum_t w_t
//
// Each KV head's codes are read once for all its query rows (group x queries),
// in tiles of 16 tokens: 2 x 16 x D bytes.  That is 4 * rows FLOP a byte pair, so
// up to a dozen rows the pool's bytes bound it.
//
// Work split: the tiles of all (sequence, KV head, row tile) triples in one
// flat order, every warp of the grid an equal contiguous share (lengths are
// read on the device, so a captured step follows them).  A warp that holds
// a whole triple writes its output; the others' states (reference maximum, sum,
// unnormalised rows) are merged in shared memory within a CTA, and across CTAs by
// a second small kernel.
//
// Loads: each lane copies by cp.async exactly the bytes that its own matrix
// fragments need, into slots that no other lane reads: a deep private queue
// without barriers, and conflict-free.  The order of channels within a
// product of 16 (and of tokens) is free as long as both operands have it, so
// the fragments are 16-byte runs of the pool's rows: key lane (r, c) holds
// channels 16c.. of tokens r and r + 8, value lane (r, c) channels 16r.. of
// tokens 2c, 2c + 1, 2c + 8, 2c + 9.
//
// Arithmetic: codes become fp16 exactly (bytes placed under 1024's exponent, minus
// 1152); a query row is scaled by a power of two to at most 2^14 and held in
// fp16 (bf16 and fp16 rows exactly, but for elements 2^-28 of the row's largest);
// logits, sums and outputs in fp32.  Weights are rounded to fp16 for
// the value product only, at 2^6 to 2^14 times their softmax value relative to the
// running reference, so that weights down to 2^-20 keep 11 bits.
#include <algorithm>

#include "block8.cuh"

namespace ucb {
namespace block8 {
namespace {

struct AttnParams {
  ucb_block8_cache c;
  const void* q;
  int64_t q_ss, q_sl, q_sh;
  int queries, q_heads, group, rows, row_tiles;  // rows = group * queries of a KV head
  const int32_t* blocks;
  int selected;
  int tile_shift;    // log2(tiles of 16 tokens in a block)
  float scale_log2;  // softmax scale * log2(e)
  void* out;
  float* lse;
  float* partials;  // [2 * grid] states of pairs that cross CTAs
  int* links;       // [grid][4]: last CTA of the pair that starts in this CTA and goes on (-1: none), s, h, row tile
  unsigned int* err;
};

constexpr int TILE = 16;
constexpr int MIN_TILES = 2;  // a warp's least share, where there is more than that
constexpr float LIFT = 6.f;   // log2 of a weight at the reference maximum
constexpr float LAZY = 14.f;  // a weight may reach 2^LAZY before the reference moves

template <int D, int NT> struct Shape {
  static constexpr int ROWS = 8 * NT;
  static constexpr int WARPS = NT == 1 ? 12 : 8;
  static constexpr int STAGES = D == 64 ? 6 : NT == 1 ? 3 : 4;
  static constexpr int STAGE_BYTES = 2 * TILE * D;
  static constexpr int ROW_FLOATS = D + 4;  // unnormalised row, reference, sum, padding
  static constexpr int STATE_BYTES = ROWS * ROW_FLOATS * 4;
  static constexpr int RING_BYTES = STAGES * STAGE_BYTES > STATE_BYTES ? STAGES * STAGE_BYTES : STATE_BYTES;
  static constexpr int WARP_BYTES = RING_BYTES + STATE_BYTES;
};

__device__ __forceinline__ void cp_async16_some(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async8_some(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two of the codes in w (offset by 128, selected into the low bytes of 1024-based halves) as fp16.
__device__ __forceinline__ uint32_t halves(uint32_t w, uint32_t select) {
  uint32_t x = prmt(w, 0x64646464u, select), y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64806480u));
  return y;
}

// A (sequence, KV head, row tile) triple and where a share of its tiles begins.
struct Pair {
  int s, h, rt, tiles;
  int64_t base;  // flat index of its first tile
};

// Segment of one warp in shared memory, for the merge of its CTA.
struct Segment {
  int used, ends;  // ends: holds the pair's last tile
  int s, h, rt;
};

template <typename T, int D>
__device__ __forceinline__ void write_row(const AttnParams& p, int s, int h, int row, int d0, const float* o, int n,
                                          float inverse) {
  const int l = row / p.group, head = h * p.group + row % p.group;
  T* out = static_cast<T*>(p.out) + (((int64_t)s * p.queries + l) * p.q_heads + head) * D + d0;
  for (int i = 0; i < n; ++i) out[i] = Dtype<T>::from_f(o[i] * inverse);
}

__device__ __forceinline__ void write_lse(const AttnParams& p, int s, int h, int row, float ref, float sum) {
  const int l = row / p.group, head = h * p.group + row % p.group;
  if (p.lse)
    p.lse[((int64_t)s * p.queries + l) * p.q_heads + head] =
        sum == 0.f ? -INFINITY : (ref == -INFINITY ? sum : (ref + log2f(sum)) * 0.693147180559945309f);
}

// A row's states merged: reference, sum and one channel.  A state without a token has
// reference -inf and sum 0; products, not branches, so that a NaN comes through.
struct Merged {
  float ref, sum, value;
};
template <typename Get> __device__ __forceinline__ Merged merge_states(int n, Get get) {
  Merged m{-INFINITY, 0.f, 0.f};
  for (int i = 0; i < n; ++i) m.ref = fmaxf(m.ref, get(i).ref);
  for (int i = 0; i < n; ++i) {
    const Merged x = get(i);
    const float f = x.ref == -INFINITY ? 0.f : fast_exp2(x.ref - m.ref);
    m.sum = fmaf(f, x.sum, m.sum);
    m.value = fmaf(f, x.value, m.value);
  }
  return m;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::WARPS * 32, 1) attention_kernel(const AttnParams p) {
  using S = Shape<D, NT>;
  constexpr int MT = D / 16;        // value products of 16 channels
  constexpr int KS = D / 16;        // key products of 16 channels
  constexpr int VB = D / 8;         // bytes of a value row that a lane holds
  const ucb_block8_cache& c = p.c;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Segment segments[S::WARPS][2];
  __shared__ int warp_sums[S::WARPS];
  int* prefix = reinterpret_cast<int*>(smem + S::WARPS * S::WARP_BYTES);  // [num_seqs + 1], dense only
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cq = lane & 3;
  const int bt = c.block_tokens, heads_rows = c.kv_heads * p.row_tiles;
  const int tiles_in_block = 1 << p.tile_shift;

  // ---- the flat order: tiles of every sequence (at least one, so that every row is written)
  int64_t total;
  const int listed_tiles = p.selected << p.tile_shift;
  if (p.blocks) {
    total = (int64_t)c.num_seqs * listed_tiles * heads_rows;
  } else {
    int carry = 0;
    if (threadIdx.x == 0) prefix[0] = 0;
    for (int base = 0; base < c.num_seqs; base += S::WARPS * 32) {
      const int i = base + threadIdx.x;
      int v = i < c.num_seqs ? max(1, (held_tokens(c, i, p.err) + TILE - 1) / TILE) : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) warp_sums[warp] = v;
      __syncthreads();
      int before = carry;
      for (int w = 0; w < S::WARPS; ++w) {
        if (w < warp) before += warp_sums[w];
        carry += warp_sums[w];
      }
      if (i < c.num_seqs) prefix[i + 1] = before + v;
      __syncthreads();
    }
    total = (int64_t)carry * heads_rows;
  }
  const int64_t all_workers = (int64_t)gridDim.x * S::WARPS;
  const int64_t workers = max((int64_t)1, min(all_workers, total / MIN_TILES));
  const int64_t worker = (int64_t)blockIdx.x * S::WARPS + warp;
  if (lane == 0) segments[warp][0].used = segments[warp][1].used = 0;
  auto share = [&](int64_t w) { return w >= workers ? total : total * w / workers; };
  auto locate = [&](int64_t t) {
    Pair a;
    if (p.blocks) {
      const int64_t pair = t / listed_tiles;
      a.s = (int)(pair / heads_rows);
      a.tiles = listed_tiles;
      const int u = (int)(pair % heads_rows);
      a.h = u / p.row_tiles;
      a.rt = u % p.row_tiles;
      a.base = pair * listed_tiles;
    } else {
      const int unit = (int)(t / heads_rows);
      int lo = 0, hi = c.num_seqs - 1;  // the last sequence whose first tile is not after t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= unit) lo = mid; else hi = mid - 1;
      }
      a.s = lo;
      a.tiles = prefix[lo + 1] - prefix[lo];
      const int64_t first = (int64_t)prefix[lo] * heads_rows;
      const int u = (int)((t - first) / a.tiles);
      a.h = u / p.row_tiles;
      a.rt = u % p.row_tiles;
      a.base = first + (int64_t)u * a.tiles;
    }
    return a;
  };

  unsigned char* ring = smem + warp * S::WARP_BYTES;
  const uint32_t ring_at = smem_u32(ring);
  int64_t t = share(worker);
  const int64_t t_end = share(worker + 1);
  if (worker < workers) while (t < t_end) {
    const Pair a = locate(t);
    const int begin = (int)(t - a.base), end = (int)min((int64_t)a.tiles, t_end - a.base);
    t = a.base + end;
    const int len = held_tokens(c, a.s, p.err);
    const int32_t* list = p.blocks ? p.blocks + ((int64_t)a.s * c.kv_heads + a.h) * p.selected : nullptr;
    const int32_t* table = c.block_table + (int64_t)a.s * c.max_blocks;
    const int entries = p.blocks ? p.selected : (len + bt - 1) / bt;

    // ---- block descriptors: lane i holds entry window + i, `next` the 32 entries after
    struct Entry {
      int block, token;
      float ks, vs;
    };
    auto fetch = [&](int k) {
      Entry e{-1, 0, 0.f, 0.f};
      if (k < entries) {
        const int j = list ? list[k] : k;
        if (j >= 0 && j < c.max_blocks && (int64_t)j * bt < len) {
          e.token = j * bt;
          const int b = table[j];
          if (b >= 0 && b < c.num_blocks) e.block = b;
          else atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
        }
      }
      return e;
    };
    auto fetch_scales = [&](Entry& e) {
      if (e.block >= 0) {
        const int64_t at = (int64_t)e.block * c.kv_heads + a.h;
        e.ks = c.key_scale[at];
        e.vs = c.value_scale[at];
      }
    };
    int window = begin >> p.tile_shift;
    Entry now = fetch(window + lane), next = fetch(window + 32 + lane);
    fetch_scales(now);
    bool next_scaled = false;

    // ---- query rows as fp16 operands
    uint32_t qb[NT][KS][2];
    float row_scale[NT];  // of row nt * 8 + r
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = a.rt * S::ROWS + nt * 8 + r;
      const bool real = row < p.rows;
      const T* q = static_cast<const T*>(p.q) + a.s * p.q_ss + (real ? row / p.group : 0) * p.q_sl +
                   (a.h * p.group + (real ? row % p.group : 0)) * p.q_sh;
      float x[KS][4];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[i][k] = real ? Dtype<T>::to_f(q[64 * (i / 4) + 16 * cq + 4 * (i % 4) + k]) : 0.f;
          top = fmaxf(top, fabsf(x[i][k]));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // power of two that brings the largest element to [2^13, 2^14); both factors are normal numbers
      const int e = min(126, top > 0.f && top <= 3.4028235e38f ? 140 - (int)(__float_as_uint(top) >> 23) : 0);
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
      row_scale[nt] = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        qb[nt][i][0] = pack_f16x2(x[i][0] * up, x[i][1] * up);
        qb[nt][i][1] = pack_f16x2(x[i][2] * up, x[i][3] * up);
      }
    }
    float col_scale[NT][2];
    int col_limit[NT][2];  // tokens that the columns' rows see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        col_scale[nt][k] = __shfl_sync(0xffffffffu, row_scale[nt], 4 * (2 * cq + k));
        const int row = a.rt * S::ROWS + nt * 8 + 2 * cq + k;
        col_limit[nt][k] = len - p.queries + 1 + (row < p.rows ? row / p.group : 0);
      }
    const int sure = len - p.queries + 1;  // tokens that every row sees

    float o[NT][MT][4], acc[NT][MT][4], ref[NT][2], sum[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      ref[nt][0] = ref[nt][1] = -INFINITY;
      sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[nt][j][k] = acc[nt][j][k] = 0.f;
    }
    float open_scale = 0.f;
    int open_entry = -1, open_token = 0;
    // the open block's products, times its scale, into the output; a row that sees none of the block takes
    // nothing of it, a scale that is not a number included
    auto flush = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float scale[2] = {open_token < col_limit[nt][0] ? open_scale : 0.f,
                                open_token < col_limit[nt][1] ? open_scale : 0.f};
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            o[nt][j][k] = fmaf(acc[nt][j][k], scale[k & 1], o[nt][j][k]);
            acc[nt][j][k] = 0.f;
          }
      }
    };

    auto issue = [&](int i) {
      if (i < end) {
        const int rel = (i >> p.tile_shift) - window;
        const int block = __shfl_sync(0xffffffffu, rel < 32 ? now.block : next.block, rel & 31);
        const int token = __shfl_sync(0xffffffffu, rel < 32 ? now.token : next.token, rel & 31);
        const int row0 = (i & (tiles_in_block - 1)) * TILE, n = len - token - row0;
        if (block >= 0 && n > 0) {
          const int64_t at = (((int64_t)block * c.kv_heads + a.h) * bt + row0) * D;
          const int8_t* k = c.key_code + at + r * D + 16 * cq;
          const int8_t* v = c.value_code + at + 2 * cq * D + VB * r;
          const uint32_t to = ring_at + ((i - begin) % S::STAGES) * S::STAGE_BYTES;
          const int k0 = r < n ? 16 : 0, k1 = r + 8 < n ? 16 : 0;
          cp_async16_some(to + lane * 16, k, k0);
          cp_async16_some(to + 512 + lane * 16, k + 8 * D, k1);
          if (D == 128) {
            cp_async16_some(to + 1024 + lane * 16, k + 64, k0);
            cp_async16_some(to + 1536 + lane * 16, k + 8 * D + 64, k1);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int tok = 2 * cq + (x & 1) + (x & 2) * 4;
              cp_async16_some(to + 2048 + x * 512 + lane * 16, v + ((x & 1) + (x & 2) * 4) * D, tok < n ? 16 : 0);
            }
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int tok = 2 * cq + (x & 1) + (x & 2) * 4;
              cp_async8_some(to + 1024 + x * 256 + lane * 8, v + ((x & 1) + (x & 2) * 4) * D, tok < n ? 8 : 0);
            }
          }
        }
      }
      cp_async_commit();
    };

#pragma unroll
    for (int x = 0; x < S::STAGES - 1; ++x) issue(begin + x);
    for (int i = begin; i < end; ++i) {
      int entry = i >> p.tile_shift;
      if (entry - window >= 32) {
        if (!next_scaled) fetch_scales(next);
        now = next;
        window += 32;
        next = fetch(window + 32 + lane);
        next_scaled = false;
      } else if (!next_scaled && i > begin) {
        fetch_scales(next);
        next_scaled = true;
      }
      cp_async_wait<S::STAGES - 2>();
      issue(i + S::STAGES - 1);  // into the slot of the tile before, whose values were used
      const int rel = entry - window;
      const int block = __shfl_sync(0xffffffffu, now.block, rel);
      const int first_token = __shfl_sync(0xffffffffu, now.token, rel) + (i & (tiles_in_block - 1)) * TILE;
      if (block < 0 || first_token >= len) continue;
      const float ks = __shfl_sync(0xffffffffu, now.ks, rel);
      if (entry != open_entry) {
        if (open_entry >= 0) flush();
        open_entry = entry;
        open_scale = __shfl_sync(0xffffffffu, now.vs, rel);
        open_token = __shfl_sync(0xffffffffu, now.token, rel);
      }
      const unsigned char* slot = ring + ((i - begin) % S::STAGES) * S::STAGE_BYTES;

      // ---- logits of 16 tokens (rows) and 8 query rows (columns)
      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int half = 0; half < KS / 4; ++half) {
        const uint4 ka = *reinterpret_cast<const uint4*>(slot + half * 1024 + lane * 16);
        const uint4 kb = *reinterpret_cast<const uint4*>(slot + half * 1024 + 512 + lane * 16);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t xa = wa[w] ^ 0x80808080u, xb = wb[w] ^ 0x80808080u;
          const uint32_t f[4] = {halves(xa, 0x4140), halves(xb, 0x4140), halves(xa, 0x4342), halves(xb, 0x4342)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], f, qb[nt][half * 4 + w][0], qb[nt][half * 4 + w][1]);
        }
      }

      // ---- weights 2^(s - ref)
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[nt][k] *= col_scale[nt][k & 1] * ks;
      if (first_token + TILE > sure) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (first_token + r + (k & 2) * 4 >= col_limit[nt][k & 1]) s[nt][k] = -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) move |= fmaxf(s[nt][k], s[nt][k + 2]) > ref[nt][k] + LAZY;
      if (__any_sync(0xffffffffu, move)) {
        flush();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float top = fmaxf(s[nt][k], s[nt][k + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float to = fmaxf(ref[nt][k], top - LIFT);
            const float f = ref[nt][k] == -INFINITY ? 0.f : fast_exp2(ref[nt][k] - to);
            // a NaN that the sums already hold stays: 0 * NaN
            sum[nt][k] *= f;
            ref[nt][k] = to;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[nt][j][k] *= f;
              o[nt][j][k + 2] *= f;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float base = ref[nt][k & 1];
          w[k] = fast_exp2(s[nt][k] - (base == -INFINITY ? 0.f : base));
        }
        sum[nt][0] += w[0] + w[2];
        sum[nt][1] += w[1] + w[3];
        pb[nt][0] = movmatrix_trans(pack_f16x2(w[0], w[1]));
        pb[nt][1] = movmatrix_trans(pack_f16x2(w[2], w[3]));
      }

      // ---- output: channels (rows) of 16 tokens times the weights
      uint32_t vw[4][D / 32];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (D == 128) {
          const uint4 v = *reinterpret_cast<const uint4*>(slot + 2048 + x * 512 + lane * 16);
          vw[x][0] = v.x, vw[x][1] = v.y, vw[x][D / 32 - 2] = v.z, vw[x][D / 32 - 1] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(slot + 1024 + x * 256 + lane * 8);
          vw[x][0] = v.x, vw[x][1] = v.y;
        }
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t w0 = vw[0][w] ^ 0x80808080u, w1 = vw[1][w] ^ 0x80808080u;
        const uint32_t w2 = vw[2][w] ^ 0x80808080u, w3 = vw[3][w] ^ 0x80808080u;
#pragma unroll
        for (int y = 0; y < 2; ++y) {  // channel pairs (4w, 4w + 1) and (4w + 2, 4w + 3) of the lane's run
          const uint32_t x01 = prmt(w0, w1, y ? 0x7362 : 0x5140), x23 = prmt(w2, w3, y ? 0x7362 : 0x5140);
          const uint32_t f[4] = {halves(x01, 0x4140), halves(x01, 0x4342), halves(x23, 0x4140), halves(x23, 0x4342)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt][2 * w + y], f, pb[nt][0], pb[nt][1]);
        }
      }
    }
    cp_async_wait<0>();
    if (open_entry >= 0) flush();

    // ---- the segment's result: lane (r, cq) holds channels VB * r .. of rows 2 cq and 2 cq + 1
    const bool whole = begin == 0 && end == a.tiles;
    const int which = begin == 0 ? 1 : 0;
    float* state = reinterpret_cast<float*>(which ? ring : ring + S::RING_BYTES);
    __syncwarp();  // every lane is done with the ring before states overwrite it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = sum[nt][k];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int in_tile = nt * 8 + 2 * cq + k, row = a.rt * S::ROWS + in_tile;
        float run[2 * MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          run[2 * j] = o[nt][j][k];
          run[2 * j + 1] = o[nt][j][k + 2];
        }
        if (whole) {
          if (row < p.rows) {
            write_row<T, D>(p, a.s, a.h, row, VB * r, run, VB, l == 0.f ? 0.f : __fdividef(1.f, l));
            if (r == 0) write_lse(p, a.s, a.h, row, ref[nt][k], l);
          }
        } else {
          float* at = state + in_tile * S::ROW_FLOATS;
#pragma unroll
          for (int i = 0; i < VB; i += 4)
            *reinterpret_cast<float4*>(at + VB * r + i) = make_float4(run[i], run[i + 1], run[i + 2], run[i + 3]);
          if (r == 0) at[D] = ref[nt][k], at[D + 1] = l;
        }
      }
    if (!whole && lane == 0) segments[warp][which] = Segment{1, end == a.tiles, a.s, a.h, a.rt};
  }
  __syncthreads();

  // ---- chains of segments of one pair: complete ones are written, the CTA's first and last may go on
  // in other CTAs.  A warp's slot 0 continues the pair that was open before it, slot 1 opens one.
  auto state_of = [&](int w, int which) {
    return reinterpret_cast<const float*>(smem + w * S::WARP_BYTES + (which ? 0 : S::RING_BYTES));
  };
  if (threadIdx.x == 0) p.links[blockIdx.x * 4] = -1;
  int open_w = 0, open_which = 0, open_n = 0;  // the open chain: first segment and count
  bool from_before = false;
  auto emit = [&](const Segment& seg, bool ended) {
    const int n = open_n, w0 = open_w, which0 = open_which;
    const bool complete = ended && !from_before;
    float* to = p.partials + ((int64_t)blockIdx.x * 2 + (from_before ? 0 : 1)) * (S::ROWS * S::ROW_FLOATS);
    for (int item = threadIdx.x; item < S::ROWS * D; item += S::WARPS * 32) {
      const int in_tile = item / D, d = item % D, row = seg.rt * S::ROWS + in_tile;
      if (row >= p.rows) break;
      const Merged m = merge_states(n, [&](int i) {
        const float* at = state_of(w0 + i, i ? 0 : which0) + in_tile * S::ROW_FLOATS;
        return Merged{at[D], at[D + 1], at[d]};
      });
      if (complete) {
        const float value = m.sum == 0.f ? 0.f : m.value / m.sum;
        write_row<T, D>(p, seg.s, seg.h, row, d, &value, 1, 1.f);
        if (d == 0) write_lse(p, seg.s, seg.h, row, m.ref, m.sum);
      } else {
        to[in_tile * S::ROW_FLOATS + d] = m.value;
        if (d == 0) to[in_tile * S::ROW_FLOATS + D] = m.ref, to[in_tile * S::ROW_FLOATS + D + 1] = m.sum;
      }
    }
  };
  Segment last{};
  for (int w = 0; w < S::WARPS; ++w) {
    const Segment s0 = segments[w][0], s1 = segments[w][1];
    if (s0.used) {
      if (open_n == 0) open_w = w, open_which = 0, from_before = true;
      ++open_n;
      last = s0;
      if (s0.ends) {
        emit(s0, true);
        open_n = 0;
        from_before = false;
      }
    }
    if (s1.used) {
      open_w = w, open_which = 1, open_n = 1, from_before = false;
      last = s1;
    }
  }
  if (open_n) {
    emit(last, false);
    if (!from_before && threadIdx.x == 0) {  // the pair that starts here ends in a later CTA
      const int64_t mine = share(min(workers, ((int64_t)blockIdx.x + 1) * S::WARPS)) - 1;
      const Pair a = locate(mine);
      const int64_t tile = a.base + a.tiles - 1;
      int64_t w = min(workers - 1, ((tile + 1) * workers - 1) / total);
      int* link = p.links + blockIdx.x * 4;
      link[1] = a.s, link[2] = a.h, link[3] = a.rt;
      link[0] = (int)(w / S::WARPS);
    }
  }
}

// Pairs that cross CTAs: block (c, row) merges row `row` of the pair that
// starts in CTA c: its state there and those that the CTAs up to its last one continue it by.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(D) attention_merge_kernel(const AttnParams p) {
  using S = Shape<D, NT>;
  const int* link = p.links + blockIdx.x * 4;
  const int end = link[0];
  if (end < 0) return;
  const int row = link[3] * S::ROWS + blockIdx.y, d = threadIdx.x;
  if (row >= p.rows) return;
  const Merged m = merge_states(end - (int)blockIdx.x + 1, [&](int i) {
    const int64_t slot = (int64_t)(blockIdx.x + i) * 2 + (i == 0);
    const float* at = p.partials + (slot * S::ROWS + blockIdx.y) * S::ROW_FLOATS;
    return Merged{at[D], at[D + 1], at[d]};
  });
  const float value = m.sum == 0.f ? 0.f : m.value / m.sum;
  write_row<T, D>(p, link[1], link[2], row, d, &value, 1, 1.f);
  if (d == 0) write_lse(p, link[1], link[2], row, m.ref, m.sum);
}

int multiprocessors() {
  static int counts[64] = {0};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (counts[dev] == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) counts[dev] = n;
  return counts[dev];
}

template <typename T, int D, int NT> int launch(const AttnParams& p, int sms, cudaStream_t stream) {
  using S = Shape<D, NT>;
  const int smem = S::WARPS * S::WARP_BYTES + (p.blocks ? 0 : (p.c.num_seqs + 1) * 4);
  const cudaError_t e = cudaFuncSetAttribute(attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return ucb_host::set_error(UCB_ERR_CUDA, "ucb_block8_attention: %s", cudaGetErrorString(e));
  const int64_t entries = p.blocks ? p.selected : p.c.max_blocks;
  const int64_t tiles = (entries << p.tile_shift) * p.c.num_seqs * p.c.kv_heads * p.row_tiles;
  const int64_t wanted = (tiles + S::WARPS * MIN_TILES - 1) / (S::WARPS * MIN_TILES);
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(sms, wanted));
  attention_kernel<T, D, NT><<<grid, S::WARPS * 32, smem, stream>>>(p);
  attention_merge_kernel<T, D, NT><<<dim3(grid, S::ROWS), D, 0, stream>>>(p);
  return ucb_host::check_launch("block8 attention_kernel");
}

template <typename T> int launch_shape(const AttnParams& p, int sms, cudaStream_t stream) {
  const bool wide = p.rows > 8;
  if (p.c.head_dim == 128) return wide ? launch<T, 128, 2>(p, sms, stream) : launch<T, 128, 1>(p, sms, stream);
  return wide ? launch<T, 64, 2>(p, sms, stream) : launch<T, 64, 1>(p, sms, stream);
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

// States of two pairs and one link for each CTA, up to 16 rows.
extern "C" int64_t ucb_block8_attention_workspace_bytes(const ucb_block8_cache* cache, int queries, int q_heads) {
  if (b8::check_cache(cache, "ucb_block8_attention_workspace_bytes") || queries < 1 || q_heads < 1) return -1;
  const int64_t sms = b8::multiprocessors();
  const int rows = (int64_t)q_heads / cache->kv_heads * queries > 8 ? 16 : 8;
  return sms > 0 ? sms * (2 * rows * (cache->head_dim + 4) * 4 + 16) : -1;
}

extern "C" int ucb_block8_attention(const ucb_block8_cache* cache, const void* query, int64_t q_ss, int64_t q_sl,
                                    int64_t q_sh, int queries, int q_heads, const int32_t* blocks, int num_selected,
                                    float softmax_scale, void* out, float* lse, void* workspace, void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_attention")) return rc;
  if (!query || !out || !workspace) return set_error(UCB_ERR_INVALID, "ucb_block8_attention: null pointer");
  if (queries < 1 || queries > 16) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_attention: 1 to 16 query tokens");
  if (q_heads < 1 || q_heads % cache->kv_heads)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: query heads must be divisible by KV heads");
  if (blocks && (num_selected < 1 || num_selected > 1 << 20))
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: a selection needs 1 to 2^20 entries");
  if (reinterpret_cast<uintptr_t>(workspace) & 15)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: workspace must be 16-byte aligned");
  unsigned int* err = ucb_host::device_error_word();
  const int sms = b8::multiprocessors();
  if (!err || sms < 1) return set_error(UCB_ERR_CUDA, "ucb_block8_attention: no device");
  b8::AttnParams p{};
  p.c = *cache;
  p.q = query;
  p.q_ss = q_ss, p.q_sl = q_sl, p.q_sh = q_sh;
  p.queries = queries, p.q_heads = q_heads;
  p.group = q_heads / cache->kv_heads;
  p.rows = p.group * queries;
  const int tile_rows = p.rows > 8 ? 16 : 8;
  p.row_tiles = (p.rows + tile_rows - 1) / tile_rows;
  p.blocks = blocks, p.selected = num_selected;
  p.tile_shift = cache->block_tokens == 16 ? 0 : cache->block_tokens == 32 ? 1 : cache->block_tokens == 64 ? 2 : 3;
  p.scale_log2 = softmax_scale * 1.44269504088896341f;
  p.out = out, p.lse = lse;
  p.partials = static_cast<float*>(workspace);
  p.links = reinterpret_cast<int*>(p.partials + (int64_t)sms * 2 * tile_rows * (cache->head_dim + 4));
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == UCB_BF16 ? b8::launch_shape<__nv_bfloat16>(p, sms, s) : b8::launch_shape<__half>(p, sms, s);
}
