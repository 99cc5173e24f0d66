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
// flat order, each triple's preceded by START empty ones for what its start
// costs, every warp of the grid an equal contiguous share (lengths are
// read on the device, so a captured step follows them).  A warp that holds
// a whole triple writes its output; the others' states (unit, reference, sum,
// unnormalised rows) are merged in shared memory within a CTA, and across CTAs by
// a second small kernel.
//
// Loads: every warp copies its own steps by cp.async, whole 128-byte lines an instruction,
// into a private ring of shared memory, without barriers.  The
// order of channels within a product of 16 (and of tokens) is free as long as both
// operands have it, so the fragments are 16-byte units of the pool's rows:
// key lane (r, c) reads units c and c + 4 of tokens r and r + 8, value lane
// (r, c) unit r (8 bytes of it at D = 64) of tokens 2c, 2c + 1, 2c + 8, 2c + 9.
// A unit lies at its place within 128 bytes XOR (t & 6) ^ (t & 1) << 2 of its
// token t, which makes both reads and the copies free of bank conflicts.
//
// Arithmetic: codes become fp16 exactly (bytes placed under 1024's exponent, minus
// 1152); a query row is scaled by a power of two to at most 2^14 and held in
// fp16 (bf16 and fp16 rows exactly, but for elements 2^-28 of the row's largest);
// logits, sums and outputs in fp32.  A weight is rounded to fp16 for the value
// product only, after its block's value scale has been multiplied into it,
// relative to the largest such product so far (at 2^6, up to 2^14 before the
// unit moves): every contribution to the output above 2^-20 of the largest
// keeps 11 bits, whatever the blocks' scales are.  The sum of weights is kept
// in fp32 against the reference alone.  The output's unit is held as its distance
// from the reference (`gap`, a number of the size of the scales' logarithms), never as
// a logit plus a logarithm, which would round the scale to the spacing of fp32 at the logit.
//
// Measured (B200, device): 1.07 GB of codes (32 x 32768 tokens, 4 KV heads of
// 128) in 173-177 us a call over a dozen calls, 6.2 TB/s, 94% of the copy rate; 194 us over 0.15 s and 207 over two
// seconds (79%), where the card is at its power cap and its clock at 1.65 GHz.  135 MB in 33 us, of which the stream
// takes 18; 404 MB at head_dim 64, 48 ragged sequences, in 74 us, of which the stream takes 62; one sequence of 700
// tokens 9.0 us.  16 tokens cost 479 warp instructions at 128 channels and 253 at 64 (two tiles a step), prologue and merges
// included.  Both halves of a weight in fp16 (22 bits) take 183 us instead of 174 for the gigabyte, 34.9 instead
// of 33.3 for 135 MB and 76.5 instead of 74: below the outputs' own rounding, so the weights have one.
#include <algorithm>

#include "block8.cuh"

namespace ucb {
namespace block8 {
namespace {

struct AttnParams {
  ucb_block8_cache c;
  const void* q;
  int64_t q_ss, q_sl, q_sh;
  int queries, q_heads, group, rows, row_tiles, heads_rows;  // rows = group * queries of a KV head
  const int32_t* blocks;
  int selected;
  uint32_t group_magic, heads_rows_magic, row_tiles_magic;  // floor(2^32 / divisor)
  int step_shift;    // log2(steps in a block)
  float scale_log2;  // softmax scale * log2(e)
  void* out;
  float* lse;
  float* partials;  // [2 * grid] states of pairs that cross CTAs
  int* links;       // [grid][4]: last CTA of the pair that starts in this CTA and goes on (-1: none), s, h, row tile
  unsigned int* err;
};

constexpr int TILE = 16;  // tokens of one matrix product
// Steps that the start of a pair costs a warp, in the flat order.  Device time with 0, 2, 4 and 8 of them: 8 sequences of up
// to 5003 tokens x 4 queries 31.4, 20.7, 20.9 and 21.0 us; 48 of 1 to 16384 tokens 83.4, 74.4, 73.8 and 74.4; 16 of 8192
// 35.3, 33.2, 32.9 and 32.9; 32 of 32768 174.7, 172.6, 172.5 and 172.7.
constexpr int START = 4;
constexpr int CTAS_PER_SM = 2;
constexpr float LIFT = 6.f;        // log2 of the largest scaled weight when the output's unit is set
constexpr float LAZY = 14.f;       // a scaled weight may reach 2^LAZY before the unit moves
constexpr float LAZY_SUM = 100.f;  // an unscaled one 2^LAZY_SUM before the reference does

// U tiles of 16 tokens a step.  OWN: a CTA has one pair to itself, all of a multiprocessor's registers and no second
// kernel after it; else two CTAs a multiprocessor.
template <int D, int NT, int U, bool OWN> struct Shape {
  static constexpr int ROWS = 8 * NT;
  static constexpr int WARPS = OWN || NT == 1 ? 8 : D == 64 ? 6 : 4;
  static constexpr int STEP_BYTES = U * 2 * TILE * D;
  static constexpr int STAGES = (OWN ? 131072 : 65536) / (WARPS * STEP_BYTES);
  static constexpr int ROW_FLOATS = D + 4;  // unnormalised row, its gap, its reference, the sum
  static constexpr int STATE_FLOATS = ROWS * ROW_FLOATS;
  static constexpr int RING_BYTES = STAGES * STEP_BYTES;
  static constexpr int SMEM_BYTES = WARPS * (RING_BYTES + STATE_FLOATS * 4);  // without the prefix sums
  static_assert(RING_BYTES >= STATE_FLOATS * 4, "a state fits a ring");
};

__device__ __forceinline__ void cp_async16_some(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// A (sequence, KV head, row tile) triple and where its steps begin in the flat order.
struct Pair {
  int s, h, rt, steps, base;
};

// Segment of one warp, for the merge of its CTA.
struct Segment {
  int used, ends;  // ends: holds the pair's last step
  int s, h, rt;
  int end_cta;  // the CTA that holds the pair's last step
  int apart;    // the state is not in the warp's ring but in its other place
};

// x / divisor, by the divisor's floor(2^32 / divisor): at most one below.
__device__ __forceinline__ int divide(int x, int divisor, uint32_t magic) {
  const int q = (int)__umulhi((uint32_t)x, magic);
  return q + (x - q * divisor >= divisor);
}

template <bool BF> __device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  return BF ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}

__device__ __forceinline__ int64_t out_row(const AttnParams& p, int s, int h, int row) {
  const int l = divide(row, p.group, p.group_magic);
  return ((int64_t)s * p.queries + l) * p.q_heads + h * p.group + row - l * p.group;
}

// A state's sum of weights is in units of 2^ref, its unnormalised values are in units of 2^(ref + gap).  Without a token the
// reference is NO_REF and the sum 0, without a value above zero the gap is NO_GAP: finite, so that differences of them are
// numbers (or -inf) and need no branch, and far below what either can be.
constexpr float NO_REF = -3.402823466e38f, NO_GAP = -1e30f;

__device__ __forceinline__ void write_lse(const AttnParams& p, int64_t row, float ref, float sum) {
  if (p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.693147180559945309f;
}

// 2^gap / sum, the factor of an unnormalised row; 0 where no token was seen.
__device__ __forceinline__ float normaliser(float gap, float sum) {
  return sum == 0.f ? 0.f : fast_exp2(gap) * __fdividef(1.f, sum);
}

// States of one row merged, four channels of it; products, not branches, so that a NaN comes through.
// `get(i)` points to state i's row: D channels, then gap, reference, sum.
struct Merged {
  float4 value;
  float gap, ref, sum;
};
// One more state; m's units are not below its own.
__device__ __forceinline__ void merge_in(Merged& m, float4 value, float4 meta) {
  const float fall = meta.y - m.ref, f = fast_exp2(fall + (meta.x - m.gap));
  m.value.x = fmaf(f, value.x, m.value.x);
  m.value.y = fmaf(f, value.y, m.value.y);
  m.value.z = fmaf(f, value.z, m.value.z);
  m.value.w = fmaf(f, value.w, m.value.w);
  m.sum = fmaf(fast_exp2(fall), meta.z, m.sum);
}
template <int D, typename Get> __device__ __forceinline__ Merged merge_states(int first, int n, int stride, int d, Get get) {
  Merged m{make_float4(0.f, 0.f, 0.f, 0.f), NO_GAP, NO_REF, 0.f};
#pragma unroll 1
  for (int i = first; i < n; i += 4 * stride) {  // four at a time, their loads together
    float4 x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // past the end, the last one again: not counted below
      const float* at = get(min(i + k * stride, n - 1));
      x[k] = *reinterpret_cast<const float4*>(at + D);
      y[k] = *reinterpret_cast<const float4*>(at + d);
    }
    const Merged old = m;
    float ref = fmaxf(fmaxf(x[0].y, x[1].y), fmaxf(x[2].y, x[3].y));
    ref = fmaxf(ref, old.ref);
    float gap = fmaxf(old.gap + (old.ref - ref), NO_GAP);
#pragma unroll
    for (int k = 0; k < 4; ++k) gap = fmaxf(gap, x[k].x + (x[k].y - ref));
    m = Merged{make_float4(0.f, 0.f, 0.f, 0.f), gap, ref, 0.f};
    merge_in(m, old.value, make_float4(old.gap, old.ref, old.sum, 0.f));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k * stride < n) merge_in(m, y[k], x[k]);
  }
  return m;
}

template <bool BF> __device__ __forceinline__ void write_four(const AttnParams& p, int64_t at, const Merged& m) {
  const float f = normaliser(m.gap, m.sum);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
      make_uint2(pack_out<BF>(m.value.x * f, m.value.y * f), pack_out<BF>(m.value.z * f, m.value.w * f));
}

template <bool BF, int D, int NT, int U, bool OWN>
__global__ void __launch_bounds__(Shape<D, NT, U, OWN>::WARPS * 32, OWN ? 1 : 2) attention_kernel(const AttnParams p) {
  using S = Shape<D, NT, U, OWN>;
  constexpr int MT = D / 16;          // value products of 16 channels
  constexpr int KS = D / 16;          // key products of 16 channels
  constexpr int VB = D / 8;           // bytes of a value row that a lane holds
  constexpr int STEP = U * TILE;      // tokens of a step
  const ucb_block8_cache& c = p.c;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Segment segments[S::WARPS][2];
  __shared__ int warp_sums[S::WARPS];
  int* prefix = reinterpret_cast<int*>(smem + S::SMEM_BYTES);  // [num_seqs + 1], dense only
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, cq = lane & 3;
  const int bt = c.block_tokens, heads_rows = p.heads_rows;
  const int step_mask = (1 << p.step_shift) - 1;

  // ---- the flat order: steps of every sequence (at least one, so that every row is written)
  int total;
  const int start = OWN ? 0 : START;
  const int listed_steps = (p.selected << p.step_shift) + start;
  auto steps_of = [&](int s) { return max(1, (held_tokens(c, s, p.err) + STEP - 1) / STEP) + start; };
  const int own_s = divide(blockIdx.x, heads_rows, p.heads_rows_magic);
  if (OWN) {
    total = p.blocks ? listed_steps : steps_of(own_s);
  } else if (p.blocks) {
    total = c.num_seqs * listed_steps * heads_rows;
  } else {
    int carry = 0;
    if (threadIdx.x == 0) prefix[0] = 0;
    for (int base = 0; base < c.num_seqs; base += S::WARPS * 32) {
      const int i = base + threadIdx.x;
      int v = i < c.num_seqs ? steps_of(i) : 0;
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
    total = carry * heads_rows;
  }
  const int worker = OWN ? warp : blockIdx.x * S::WARPS + warp;
  if (lane == 0) segments[warp][0].used = segments[warp][1].used = 0;
  // equal shares, the first `longer` of one step more
  const int workers = max(1, min(OWN ? S::WARPS : (int)gridDim.x * S::WARPS, total));
  const int each = total / workers, longer = total - each * workers;
  auto share = [&](int w) { return w < workers ? w * each + min(w, longer) : total; };
  auto worker_of = [&](int step) {
    const int split = longer * (each + 1);
    return step < split ? step / (each + 1) : longer + (step - split) / each;
  };
  auto locate = [&](int t) {
    Pair a;
    const int unit = divide(t, heads_rows, p.heads_rows_magic);
    int first;
    if (OWN) {
      const int u = blockIdx.x - own_s * heads_rows;
      a.h = divide(u, p.row_tiles, p.row_tiles_magic);
      return Pair{own_s, a.h, u - a.h * p.row_tiles, total, 0};
    }
    if (p.blocks) {
      a.s = unit / listed_steps;
      a.steps = listed_steps;
      first = a.s * listed_steps;
    } else {
      int lo = 0, hi = c.num_seqs - 1;  // the last sequence whose first step is not after t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= unit) lo = mid; else hi = mid - 1;
      }
      a.s = lo;
      first = prefix[lo];
      a.steps = prefix[lo + 1] - first;
    }
    first *= heads_rows;
    const int u = (t - first) / a.steps;
    a.base = first + u * a.steps;
    a.h = divide(u, p.row_tiles, p.row_tiles_magic);
    a.rt = u - a.h * p.row_tiles;
    return a;
  };

  unsigned char* ring = smem + warp * S::RING_BYTES;
  const uint32_t ring_at = smem_u32(ring);
  // places of units in the ring: what this lane copies, its key and its value fragments
  auto place = [&](int token, int unit) {
    const int x = (unit ^ (token & 6) ^ ((token & 1) << 2)) * 16;
    return (D == 128 ? token : token >> 1) * 128 + x;
  };
  const int copy_token = lane / (D / 16), copy_place = place(copy_token, lane % (D / 16));
  const int key_place = place(r, cq);
  const int value_place = D == 128 ? place(2 * cq, r) : place(2 * cq, r >> 1) + (r & 1) * 8;
  const int value_place1 = D == 128 ? place(2 * cq + 1, r) : place(2 * cq + 1, r >> 1) + (r & 1) * 8;
  int t = share(worker);
  const int t_end = share(worker + 1);
  while (t < t_end) {
    const Pair a = locate(t);
    const int begin = max(t - a.base - start, 0), end = min(a.steps, t_end - a.base) - start, steps = a.steps - start;
    t = a.base + end + start;
    if (end <= 0) continue;  // the rest of the pair's start: its tiles are the next warp's
    const int len = held_tokens(c, a.s, p.err);
    const int32_t* list = p.blocks ? p.blocks + ((int64_t)a.s * c.kv_heads + a.h) * p.selected : nullptr;
    const int32_t* table = c.block_table + (int64_t)a.s * c.max_blocks;
    const int entries = p.blocks ? p.selected : (len + bt - 1) / bt;

    // ---- query rows, two elements a register: row nt * 8 + r, channels of the key fragments
    uint2 raw[NT][KS];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = a.rt * S::ROWS + nt * 8 + r;
      const int l = divide(row, p.group, p.group_magic);
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + a.s * p.q_ss + l * p.q_sl +
                          (a.h * p.group + row - l * p.group) * p.q_sh + 16 * cq;
#pragma unroll
      for (int i = 0; i < KS; ++i)
        raw[nt][i] = row < p.rows ? *reinterpret_cast<const uint2*>(q + 64 * (i / 4) + 4 * (i % 4)) : make_uint2(0, 0);
    }

    // ---- block descriptors: lane i holds entry window + i, `next` the 32 entries after
    struct Entry {
      int block, token;  // pool block (-1: skipped) and its first token (-1: no entry)
      float ks, lv;      // key scale, log2 of the value scale
    };
    auto fetch = [&](int k) {  // the table's entry as it is, checked when it is first used
      Entry e{-1, -1, 0.f, 0.f};
      if (k < entries) {
        const int j = list ? list[k] : k;
        if (j >= 0 && j < c.max_blocks && (int64_t)j * bt < len) {
          e.token = j * bt;
          e.block = table[j];
        }
      }
      return e;
    };
    auto check = [&](Entry& e) {  // a block outside the pool is skipped
      if (e.token >= 0 && (e.block < 0 || e.block >= c.num_blocks)) {
        atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
        e.block = -1;
      }
    };
    auto fetch_scales = [&](Entry& e) {
      if (e.block >= 0) {
        const int64_t at = (int64_t)e.block * c.kv_heads + a.h;
        e.ks = c.key_scale[at];
        e.lv = __log2f(c.value_scale[at]);
      }
    };
    int window = begin >> p.step_shift;
    Entry now = fetch(window + lane), next{-1, -1, 0.f, 0.f};
    bool next_scaled = true;
    if (((end - 1) >> p.step_shift) - window >= 32) {
      next = fetch(window + 32 + lane);
      check(next);
      next_scaled = false;
    }
    check(now);

    auto issue = [&](int i) {
      if (i < end) {
        const int rel = (i >> p.step_shift) - window;
        const int block = __shfl_sync(0xffffffffu, rel < 32 ? now.block : next.block, rel & 31);
        const int token = __shfl_sync(0xffffffffu, rel < 32 ? now.token : next.token, rel & 31);
        const int row0 = (i & step_mask) * STEP, n = len - token - row0;
        if (block >= 0 && n > 0) {
          const int64_t at = (((int64_t)block * c.kv_heads + a.h) * bt + row0) * D + lane * 16;
          const int8_t *k = c.key_code + at, *v = c.value_code + at;
          const uint32_t to = ring_at + ((i - begin) % S::STAGES) * S::STEP_BYTES;
#pragma unroll
          for (int x = 0; x < STEP * D / 512; ++x) {  // 512 bytes: the rows of 4 (or 8) tokens
            const int bytes = x * (512 / D) + copy_token < n ? 16 : 0;
            const uint32_t at_ring = to + x * 512 + (D == 128 && (x & 1) ? copy_place ^ 64 : copy_place);
            cp_async16_some(at_ring, k + x * 512, bytes);
            cp_async16_some(at_ring + STEP * D, v + x * 512, bytes);
          }
        }
      }
      cp_async_commit();
    };
    // After step i, whose slot every lane has read: the step STAGES after it goes into that slot, and step i + 1 is waited
    // for.  Where all warps stream, one slot less is in flight: that uses the bandwidth up, and a deeper queue only makes
    // every first access wait (172.5 us against 175.4 for a gigabyte).  A pair on its own waits for round trips.
    auto advance = [&](int i) {
      __syncwarp();
      if (!OWN) cp_async_wait<S::STAGES - 2>();
      issue(i + S::STAGES);
      if (OWN) cp_async_wait<S::STAGES - 1>();
      __syncwarp();  // the other lanes' copies
    };
#pragma unroll 1
    for (int x = 0; x < S::STAGES - 1; ++x) issue(begin + x);
    fetch_scales(now);

    // ---- query rows as fp16 operands, times the power of two that brings their largest element to [2^13, 2^14)
    uint32_t qb[NT][KS][2];
    float row_scale[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t top = 0;  // largest magnitude, as bits of the two halves
#pragma unroll
      for (int i = 0; i < KS; ++i)
        top = __vmaxu2(top, __vmaxu2(raw[nt][i].x & 0x7fff7fffu, raw[nt][i].y & 0x7fff7fffu));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = max(top & 0xffffu, top >> 16);
      const uint32_t exponent = __float_as_uint(BF ? __uint_as_float(top << 16) : __half2float(__ushort_as_half((unsigned short)top))) >> 23;
      // both factors are normal numbers; a row of zeros, infinities or NaN is left as it is
      const int e = exponent == 0 && top == 0 || exponent == 255 ? 0 : min(126, 140 - (int)exponent);
      const float up = __uint_as_float((uint32_t)(127 + e) << 23);
      row_scale[nt] = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint32_t w[2] = {raw[nt][i].x, raw[nt][i].y};
#pragma unroll
        for (int k = 0; k < 2; ++k)
          qb[nt][i][k] = BF ? pack_f16x2(Dtype<__nv_bfloat16>::lo(w[k]) * up, Dtype<__nv_bfloat16>::hi(w[k]) * up)
                            : pack_f16x2(Dtype<__half>::lo(w[k]) * up, Dtype<__half>::hi(w[k]) * up);
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
        col_limit[nt][k] = len - p.queries + 1 + (row < p.rows ? divide(row, p.group, p.group_magic) : 0);
      }
    const int sure = len - p.queries + 1;  // tokens that every row sees

    // Sum of weights in units of 2^ref, unnormalised output in units of 2^(ref + gap).
    float o[NT][MT][4], gap[NT][2], sum[NT][2], ref[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      gap[nt][0] = gap[nt][1] = NO_GAP;
      ref[nt][0] = ref[nt][1] = NO_REF;
      sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[nt][j][k] = 0.f;
    }

#pragma unroll 1
    for (int i = begin - 1; i < end; advance(i++)) {
      if (i < begin) continue;
      const int entry = i >> p.step_shift;
      if (entry - window >= 32) {
        if (!next_scaled) fetch_scales(next);
        now = next;
        window += 32;
        next = fetch(window + 32 + lane);
        check(next);
        next_scaled = false;
      } else if (!next_scaled && i > begin) {
        fetch_scales(next);
        next_scaled = true;
      }
      const int rel = entry - window;
      const int block = __shfl_sync(0xffffffffu, now.block, rel);
      const int first_token = __shfl_sync(0xffffffffu, now.token, rel) + (i & step_mask) * STEP;
      if (block < 0 || first_token >= len) continue;
      const float ks = __shfl_sync(0xffffffffu, now.ks, rel);
      const float lv = __shfl_sync(0xffffffffu, now.lv, rel);
      const unsigned char* slot = ring + ((i - begin) % S::STAGES) * S::STEP_BYTES;

      // ---- logits of 16 tokens (rows) and 8 query rows (columns)
      float s[U][NT][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float part[KS / 4][NT][4];
#pragma unroll
        for (int half = 0; half < KS / 4; ++half) {
          const unsigned char* at = slot + u * TILE * D + (half ? key_place ^ 64 : key_place);
          const uint4 ka = *reinterpret_cast<const uint4*>(at);
          const uint4 kb = *reinterpret_cast<const uint4*>(at + 8 * D);
          const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) part[half][nt][0] = part[half][nt][1] = part[half][nt][2] = part[half][nt][3] = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t xa = wa[w] ^ 0x80808080u, xb = wb[w] ^ 0x80808080u;
            const uint32_t f[4] = {halves(xa, 0x4140), halves(xb, 0x4140), halves(xa, 0x4342), halves(xb, 0x4342)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(part[half][nt], f, qb[nt][half * 4 + w][0], qb[nt][half * 4 + w][1]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            s[u][nt][k] = (KS == 8 ? part[0][nt][k] + part[KS / 4 - 1][nt][k] : part[0][nt][k]) * (col_scale[nt][k & 1] * ks);
      }
      const bool masked = first_token + STEP > sure;
      if (masked) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (first_token + u * TILE + r + (k & 2) * 4 >= col_limit[nt][k & 1]) s[u][nt][k] = -INFINITY;
      }

      // ---- references
      float top[NT][2];
      bool move = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          top[nt][k] = fmaxf(s[0][nt][k], s[0][nt][k + 2]);
          if (U == 2) top[nt][k] = fmaxf(top[nt][k], fmaxf(s[U - 1][nt][k], s[U - 1][nt][k + 2]));
          move |= top[nt][k] - ref[nt][k] > fminf(gap[nt][k] - lv + LAZY, LAZY_SUM);
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float m = top[nt][k];
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            const float to = fmaxf(ref[nt][k], m), fall = ref[nt][k] - to;
            const float gap_to = fmaxf(fmaxf(gap[nt][k] + fall, (m - to) + lv - LIFT), NO_GAP);
            // a NaN that the sums already hold stays: 0 * NaN
            const float f = fast_exp2(fall + (gap[nt][k] - gap_to));
            sum[nt][k] *= fast_exp2(fall);
            gap[nt][k] = gap_to;
            ref[nt][k] = to;
#pragma unroll
            for (int j = 0; j < MT; ++j) {
              o[nt][j][k] *= f;
              o[nt][j][k + 2] *= f;
            }
          }
      }

      // ---- weights, times the value scale for the output
      uint32_t pb[U][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float scale[2];  // the value scale in the output's unit (weights below 2^-126 are 0: no factor above 2^126 is needed)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float lift = lv - gap[nt][k];
          scale[k] = fast_exp2(lift > 126.f ? 126.f : lift);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float e = fast_exp2(s[u][nt][k] - ref[nt][k & 1]);
            sum[nt][k & 1] += e;
            w[k] = masked && s[u][nt][k] == -INFINITY ? 0.f : e * scale[k & 1];  // 0 whatever the block's scale is
          }
          pb[u][nt][0] = movmatrix_trans(pack_f16x2(w[0], w[1]));
          pb[u][nt][1] = movmatrix_trans(pack_f16x2(w[2], w[3]));
        }
      }

      // ---- output: channels (rows) of 16 tokens times the weights
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t vw[4][D / 32];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const unsigned char* at = slot + STEP * D + (u * TILE + (x >> 1) * 8) * D + (x & 1 ? value_place1 : value_place);
          if (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            vw[x][0] = v.x, vw[x][1] = v.y, vw[x][D / 32 - 2] = v.z, vw[x][D / 32 - 1] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
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
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * w + y], f, pb[u][nt][0], pb[u][nt][1]);
          }
        }
      }
    }
    cp_async_wait<0>();

    // ---- the segment's result: lane (r, cq) holds channels VB * r .. of rows 2 cq and 2 cq + 1.  A warp's last
    // segment stays in its ring, an earlier one that a warp before began has a place of its own.
    const bool whole = begin == 0 && end == steps;
    const int which = begin == 0 ? 1 : 0;
    const bool apart = t < t_end;
    float* state = reinterpret_cast<float*>(apart ? smem + S::WARPS * S::RING_BYTES + warp * (S::STATE_FLOATS * 4) : ring);
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
        const float f = whole ? normaliser(gap[nt][k], l) : 1.f;
        float run[VB];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          run[2 * j] = o[nt][j][k] * f;
          run[2 * j + 1] = o[nt][j][k + 2] * f;
        }
        if (whole) {
          if (row < p.rows) {
            const int64_t to = out_row(p, a.s, a.h, row);
            uint4* out = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to * D + VB * r);
#pragma unroll
            for (int i = 0; i < VB / 8; ++i)
              out[i] = make_uint4(pack_out<BF>(run[8 * i], run[8 * i + 1]), pack_out<BF>(run[8 * i + 2], run[8 * i + 3]),
                                  pack_out<BF>(run[8 * i + 4], run[8 * i + 5]), pack_out<BF>(run[8 * i + 6], run[8 * i + 7]));
            if (r == 0) write_lse(p, to, ref[nt][k], l);
          }
        } else {
          float* at = state + in_tile * S::ROW_FLOATS;
#pragma unroll
          for (int i = 0; i < VB; i += 4)
            *reinterpret_cast<float4*>(at + VB * r + i) = make_float4(run[i], run[i + 1], run[i + 2], run[i + 3]);
          if (r == 0) *reinterpret_cast<float4*>(at + D) = make_float4(gap[nt][k], ref[nt][k], l, 0.f);
        }
      }
    if (!whole && lane == 0)
      segments[warp][which] = Segment{1, end == steps, a.s, a.h, a.rt, worker_of(a.base + a.steps - 1) / S::WARPS, apart};
  }
  __syncthreads();

  if (!OWN) launch_dependents();

  // ---- chains of segments of one pair: complete ones are written, the CTA's first and last may go on
  // in other CTAs.  A warp's slot 0 continues the pair that was open before it, slot 1 opens one; a state outside
  // the rings ends its chain, since its warp went on to another pair.
  if (threadIdx.x == 0 && !OWN) p.links[blockIdx.x * 4] = -1;
  const Segment& mine = segments[min(lane, 2 * S::WARPS - 1) >> 1][lane & 1];
  unsigned used = __ballot_sync(0xffffffffu, lane < 2 * S::WARPS && mine.used);
  while (used) {  // a chain: the segments up to the next one that opens a pair
    const int first = __ffs(used) - 1;
    const unsigned opening = used & 0xAAAAAAAAu & ~(1u << first);
    const unsigned chain = opening ? used & ((1u << (__ffs(opening) - 1)) - 1) : used;
    used &= ~chain;
    const int open_w = first >> 1, open_n = __popc(chain), final = 31 - __clz(chain);
    const Segment last = segments[final >> 1][final & 1];
    const bool from_before = !(first & 1), ended = last.ends;
    // the chain ends, here or in a later CTA
    const bool complete = ended && !from_before;
    float* to = p.partials + ((int64_t)blockIdx.x * 2 + (from_before ? 0 : 1)) * S::STATE_FLOATS;
    for (int item = threadIdx.x; item < S::ROWS * D / 4; item += S::WARPS * 32) {
      const int in_tile = item / (D / 4), d = item % (D / 4) * 4, row = last.rt * S::ROWS + in_tile;
      if (row >= p.rows) break;
      // the chain's states lie a ring apart, the last one perhaps in its warp's other place
      const unsigned char* states = smem + open_w * S::RING_BYTES + in_tile * (S::ROW_FLOATS * 4);
      const unsigned char* end_state = last.apart ? smem + S::WARPS * S::RING_BYTES + ((final >> 1) * S::ROWS + in_tile) * (S::ROW_FLOATS * 4)
                                                  : states + (open_n - 1) * S::RING_BYTES;
      auto state = [&](int i) { return reinterpret_cast<const float*>(i < open_n - 1 ? states + i * S::RING_BYTES : end_state); };
      Merged m{make_float4(0.f, 0.f, 0.f, 0.f), NO_GAP, NO_REF, 0.f};
#pragma unroll 2
      for (int i = 0; i < open_n; ++i) {
        const float2 x = *reinterpret_cast<const float2*>(state(i) + D);
        const float top = fmaxf(m.ref, x.y);
        m.gap = fmaxf(m.gap + (m.ref - top), x.x + (x.y - top));
        m.ref = top;
      }
#pragma unroll 2
      for (int i = 0; i < open_n; ++i) merge_in(m, *reinterpret_cast<const float4*>(state(i) + d), *reinterpret_cast<const float4*>(state(i) + D));
      if (complete) {
        const int64_t out = out_row(p, last.s, last.h, row);
        write_four<BF>(p, out * D + d, m);
        if (d == 0) write_lse(p, out, m.ref, m.sum);
      } else {
        float* at = to + in_tile * S::ROW_FLOATS;
        *reinterpret_cast<float4*>(at + d) = m.value;
        if (d == 0) *reinterpret_cast<float4*>(at + D) = make_float4(m.gap, m.ref, m.sum, 0.f);
      }
    }
    if (!ended && !from_before && threadIdx.x == 0)  // the pair that starts here ends in a later CTA
      *reinterpret_cast<int4*>(p.links + blockIdx.x * 4) = make_int4(last.end_cta, last.s, last.h, last.rt);
  }
}

// Pairs that cross CTAs: block (c, row) merges row `row` of the pair that
// starts in CTA c: its state there and those that the CTAs up to its last one
// continue it by, every MERGE_GROUPS-th by one group of D / 4 threads.
constexpr int MERGE_GROUPS = 4;

template <bool BF, int D, int NT, int U>
__global__ void __launch_bounds__(MERGE_GROUPS * D / 4) attention_merge_kernel(const AttnParams p) {
  using S = Shape<D, NT, U, false>;
  __shared__ float groups[MERGE_GROUPS][D + 4];
  wait_for_primary();
  const int4 link = *reinterpret_cast<const int4*>(p.links + blockIdx.x * 4);
  if (link.x < 0) return;
  const int row = link.w * S::ROWS + blockIdx.y, d = threadIdx.x % (D / 4) * 4, g = threadIdx.x / (D / 4);
  if (row >= p.rows) return;
  Merged m = merge_states<D>(g, link.x - (int)blockIdx.x + 1, MERGE_GROUPS, d, [&](int i) {
    const int64_t slot = (int64_t)(blockIdx.x + i) * 2 + (i == 0);
    return p.partials + (slot * S::ROWS + blockIdx.y) * S::ROW_FLOATS;
  });
  *reinterpret_cast<float4*>(groups[g] + d) = m.value;
  if (d == 0) *reinterpret_cast<float4*>(groups[g] + D) = make_float4(m.gap, m.ref, m.sum, 0.f);
  __syncthreads();
  if (g > 0) return;
  m = merge_states<D>(0, MERGE_GROUPS, 1, d, [&](int i) { return static_cast<const float*>(groups[i]); });
  const int64_t out = out_row(p, link.y, link.z, row);
  write_four<BF>(p, out * D + d, m);
  if (d == 0) write_lse(p, out, m.ref, m.sum);
}

constexpr int MOST_SEQS = 4096;

template <bool BF, int D, int NT, int U, bool OWN> int launch_shape(AttnParams& p, int sms, cudaStream_t stream) {
  using S = Shape<D, NT, U, OWN>;
  static bool ready[64] = {false};  // the attribute is a device's; setting it twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  if (!ready[dev & 63]) {
    const cudaError_t e = cudaFuncSetAttribute(attention_kernel<BF, D, NT, U, OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               S::SMEM_BYTES + (OWN ? 0 : (MOST_SEQS + 1) * 4));
    if (e != cudaSuccess) return ucb_host::set_error(UCB_ERR_CUDA, "ucb_block8_attention: %s", cudaGetErrorString(e));
    ready[dev & 63] = true;
  }
  p.step_shift = (p.c.block_tokens == 16 ? 0 : p.c.block_tokens == 32 ? 1 : p.c.block_tokens == 64 ? 2 : 3) - (U - 1);
  const int64_t pairs = (int64_t)p.c.num_seqs * p.heads_rows;
  if constexpr (OWN) {
    return block8::launch(attention_kernel<BF, D, NT, U, true>, dim3((unsigned)pairs), dim3(S::WARPS * 32), S::SMEM_BYTES,
                          stream, p, "block8 attention_kernel");
  } else {
    const int64_t entries = p.blocks ? p.selected : p.c.max_blocks;
    const int64_t steps = ((entries << p.step_shift) + START) * pairs;
    if (steps > 0x3fffffff) return ucb_host::set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_attention: too many tokens in one call");
    const int64_t wanted = (steps + S::WARPS - 1) / S::WARPS;
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(CTAS_PER_SM * sms, wanted));
    p.links = reinterpret_cast<int*>(p.partials + (int64_t)CTAS_PER_SM * sms * 2 * S::STATE_FLOATS);
    const int smem = S::SMEM_BYTES + (p.blocks ? 0 : (p.c.num_seqs + 1) * 4);
    if (int rc = block8::launch(attention_kernel<BF, D, NT, U, false>, dim3(grid), dim3(S::WARPS * 32), smem, stream, p,
                                "block8 attention_kernel"))
      return rc;
    return block8::launch(attention_merge_kernel<BF, D, NT, U>, dim3(grid, S::ROWS), dim3(MERGE_GROUPS * D / 4), 0, stream, p,
                          "block8 attention_merge_kernel", 1, true);
  }
}

// Tokens of capacity up to which a pair is one CTA's, where all are resident: one launch and no merge.  Device time with
// and without, 7 rows of 128 channels: 4 pairs of 64 tokens 4.4 and 6.2 us, 512 7.8 and 8.4, 700 9.1 and 8.5, 1000 10.6 and
// 8.5; 32 pairs of 700 9.2 and 10.2, 1000 10.8 and 10.6; 72 pairs of 1000 10.9 and 12.6; 144 of 1000 x 64 channels 8.6 and
// 11.6.  A call from the host takes 11.2 and 13.4, the second launch.  So a pair has its own CTA where that is the shorter on
// the device, and a little beyond: as far as it loses less there (at most 1.4 us, 32 pairs of 1000 tokens in blocks of 16)
// than it saves the host.  More pairs fill more of the chip, so the limit rises with them.
constexpr int OWN_TOKENS = 768, OWN_TOKENS_A_PAIR = 8, MOST_OWN_TOKENS = 1024;

template <bool BF, int D, int NT> int launch_block(AttnParams& p, int sms, cudaStream_t stream) {
  const int64_t tokens = (int64_t)(p.blocks ? p.selected : p.c.max_blocks) * p.c.block_tokens;
  const int64_t triples = (int64_t)p.c.num_seqs * p.heads_rows;
  const bool own = triples <= sms && tokens <= std::min<int64_t>(MOST_OWN_TOKENS, OWN_TOKENS + OWN_TOKENS_A_PAIR * triples);
  const bool pairs = p.c.block_tokens > TILE;
  if (own) return pairs ? launch_shape<BF, D, NT, 2, true>(p, sms, stream) : launch_shape<BF, D, NT, 1, true>(p, sms, stream);
  // Two tiles a step where the registers hold them: at D = 64 (48 sequences of up to 16384 tokens x 8 heads: 74 us
  // against 91) and for 16 rows (eight of up to 5003 tokens, four queries each: 20.9 against 21.8).
  if constexpr (D == 64 || NT == 2) {
    if (pairs) return launch_shape<BF, D, NT, 2, false>(p, sms, stream);
  }
  return launch_shape<BF, D, NT, 1, false>(p, sms, stream);
}

template <bool BF> int launch_heads(AttnParams& p, int sms, cudaStream_t stream) {
  if (p.c.head_dim == 128) return p.rows > 8 ? launch_block<BF, 128, 2>(p, sms, stream) : launch_block<BF, 128, 1>(p, sms, stream);
  return p.rows > 8 ? launch_block<BF, 64, 2>(p, sms, stream) : launch_block<BF, 64, 1>(p, sms, stream);
}

}  // namespace
}  // namespace block8
}  // namespace ucb

using ucb_host::set_error;
namespace b8 = ucb::block8;

// For each CTA: states of two pairs that cross CTAs, one link.
extern "C" int64_t ucb_block8_attention_workspace_bytes(const ucb_block8_cache* cache, int queries, int q_heads) {
  if (b8::check_cache(cache, "ucb_block8_attention_workspace_bytes") || queries < 1 || q_heads < 1) return -1;
  const int64_t sms = ucb_host::multiprocessors();
  const int64_t rows = (int64_t)q_heads / cache->kv_heads * queries > 8 ? 16 : 8;
  return sms > 0 ? sms * b8::CTAS_PER_SM * (2 * rows * (cache->head_dim + 4) * 4 + 16) : -1;
}

extern "C" int ucb_block8_attention(const ucb_block8_cache* cache, const ucb_block8_attention_args* a, void* stream) {
  if (int rc = b8::check_cache(cache, "ucb_block8_attention")) return rc;
  if (!a || !a->query || !a->out || !a->workspace)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: null pointer");
  if (a->queries < 1 || a->queries > 16)
    return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_attention: 1 to 16 query tokens");
  if (a->q_heads < 1 || a->q_heads % cache->kv_heads)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: query heads must be divisible by KV heads");
  if (a->blocks && (a->num_selected < 1 || a->num_selected > 1 << 20))
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: a selection needs 1 to 2^20 entries");
  if (reinterpret_cast<uintptr_t>(a->query) & 7 || (a->q_stride_seq | a->q_stride_query | a->q_stride_head) & 3)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: query rows must start on 8 bytes");
  if (a->q_heads > 65535) return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_attention: at most 65535 query heads");
  if ((reinterpret_cast<uintptr_t>(a->workspace) | reinterpret_cast<uintptr_t>(a->out)) & 15)
    return set_error(UCB_ERR_INVALID, "ucb_block8_attention: out and workspace must be 16-byte aligned");
  unsigned int* err = ucb_host::device_error_word();
  const int sms = ucb_host::multiprocessors();
  if (!err || sms < 1) return set_error(UCB_ERR_CUDA, "ucb_block8_attention: no device");
  b8::AttnParams p{};
  p.c = *cache;
  p.q = a->query;
  p.q_ss = a->q_stride_seq, p.q_sl = a->q_stride_query, p.q_sh = a->q_stride_head;
  p.queries = a->queries, p.q_heads = a->q_heads;
  p.group = a->q_heads / cache->kv_heads;
  p.rows = p.group * a->queries;
  const int tile_rows = p.rows > 8 ? 16 : 8;
  p.row_tiles = (p.rows + tile_rows - 1) / tile_rows;
  p.heads_rows = cache->kv_heads * p.row_tiles;
  // floor(2^32 / d), 2^32 - 1 for 1 (one below in the product, as divide() takes it)
  auto magic = [](int d) { return (uint32_t)std::min<uint64_t>(0xffffffffu, (1ull << 32) / d); };
  p.group_magic = magic(p.group), p.heads_rows_magic = magic(p.heads_rows), p.row_tiles_magic = magic(p.row_tiles);
  p.blocks = a->blocks, p.selected = a->blocks ? a->num_selected : 0;
  p.scale_log2 = a->softmax_scale * 1.44269504088896341f;
  p.out = a->out, p.lse = a->lse;
  p.partials = static_cast<float*>(a->workspace);
  p.err = err;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cache->dtype == UCB_BF16 ? b8::launch_heads<true>(p, sms, s) : b8::launch_heads<false>(p, sms, s);
}

extern "C" int ucb_block8_sparse_attention(const ucb_block8_cache* cache, const ucb_block8_attention_args* a, int first,
                                           int recent, void* select_workspace, void* stream) {
  if (!a || !a->blocks) return set_error(UCB_ERR_INVALID, "ucb_block8_sparse_attention: null pointer");
  if (a->queries != 1)
    return set_error(UCB_ERR_UNSUPPORTED, "ucb_block8_sparse_attention: one query token chooses blocks");
  if (int rc = ucb_block8_select(cache, a->query, a->q_stride_seq, a->q_stride_head, a->q_heads, a->num_selected, first,
                                 recent, const_cast<int32_t*>(a->blocks), select_workspace, stream))
    return rc;
  return ucb_block8_attention(cache, a, stream);
}
