// Verification of drafted tokens against the target's distribution (ucb_verify_drafts):
//   p_j = softmax(logits_j / T),  draft x_j stays while u_j q_j(x_j) < p_j(x_j);
// at the first one that does not, a, the next token is drawn from max(p_a - q_a, 0), after all of
// them from p_n: the first token whose running sum is above u_n times the sum.
//
// The first kernel reads every row once, many CTAs a row, with a running maximum and
// sum in fp32: the tests compare numbers of relative error 1e-6 with a random one.  The
// draw is another matter: in the long flat tail of a vocabulary a running
// sum off by d names another token with a probability of up to d times the number of
// tokens, which is percents for fp32.  So the one row of each sequence that is drawn from
// is summed in fp64, exponentials included, by a cluster of CTAs.
#include <cooperative_groups.h>

#include <algorithm>

#include "block8.cuh"

namespace ucb {
namespace verify {
namespace {

namespace cg = cooperative_groups;

constexpr int MAX_ROWS = 32;  // of a sequence: its drafts and the one behind them
constexpr int ROW_THREADS = 256, ROW_AHEAD = 4;
constexpr int DRAW_THREADS = 512, DRAW_WARPS = DRAW_THREADS / 32, DRAW_CLUSTER = 8;
constexpr float LOG2E = 1.4426950408889634f;

struct Partial {
  float top, sum;  // of exp((x - top) / T)
  int best;        // the first index of the top, where it is asked for
  int unused;
};

struct VerifyParams {
  ucb_verify_args a;
  Partial* partials;  // [seqs * rows][splits]
  int splits;
  unsigned int* err;
};

// A row of the vocabulary as 16-byte vectors from the aligned address at or before its start: vector k holds the elements
// k * VEC - shift and on; the first and the last one may have places outside.
template <typename T> struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  const T* x;
  int shift, vocab, vectors;
  __device__ Row(const void* base, int64_t at, int vocab_) : x(static_cast<const T*>(base) + at), vocab(vocab_) {
    shift = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    vectors = (int)(((int64_t)vocab + shift + VEC - 1) / VEC);
  }
  __device__ __forceinline__ int first(int k) const { return k * VEC - shift; }
  __device__ __forceinline__ void load(int k, float (&v)[VEC]) const {  // -inf outside
    const int i = first(k);
    if (i >= 0 && i + VEC <= vocab) {
      const uint4 w = *reinterpret_cast<const uint4*>(x + i);
      if constexpr (sizeof(T) == 2) {
        v[0] = Dtype<T>::lo(w.x), v[1] = Dtype<T>::hi(w.x), v[2] = Dtype<T>::lo(w.y), v[3] = Dtype<T>::hi(w.y);
        v[4] = Dtype<T>::lo(w.z), v[5] = Dtype<T>::hi(w.z), v[6] = Dtype<T>::lo(w.w), v[7] = Dtype<T>::hi(w.w);
      } else {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = i + e >= 0 && i + e < vocab ? Dtype<T>::to_f(x[i + e]) : -INFINITY;
    }
  }
};

// N elements of a row of draft probabilities from i on, 0 outside the vocabulary.
template <typename Q, int N> __device__ __forceinline__ void load_probs(const Q* q, int i, int vocab, float (&v)[N]) {
  constexpr int BYTES = N * sizeof(Q), ALIGN = BYTES < 16 ? BYTES : 16;
  if (i >= 0 && i + N <= vocab && reinterpret_cast<uintptr_t>(q + i) % ALIGN == 0) {
    union {
      uint4 w16[(BYTES + 15) / 16];
      uint2 w8;
      Q e[N];
    } u;
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int k = 0; k < BYTES / 16; ++k) u.w16[k] = reinterpret_cast<const uint4*>(q + i)[k];
    } else {
      u.w8 = *reinterpret_cast<const uint2*>(q + i);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = Dtype<Q>::to_f(u.e[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = i + e >= 0 && i + e < vocab ? Dtype<Q>::to_f(q[i + e]) : 0.f;
  }
}

__device__ __forceinline__ float temperature_of(const ucb_verify_args& a, int s) { return a.temperature ? a.temperature[s] : a.temperature_all; }

// What the exponent's differences are multiplied with: greedy sequences have their log-probabilities at temperature 1.
__device__ __forceinline__ float heat_of(float temperature) { return temperature <= 0.f ? 1.f : temperature; }

__device__ __forceinline__ int count_of(const ucb_verify_args& a, int s) {
  return a.counts ? max(0, min(a.counts[s], a.drafts_n)) : a.drafts_n;
}

// (top, sum) of two parts.  A top of -inf has no sum to scale (0, or NaN, which stays).
__device__ __forceinline__ void join(float& top, float& sum, float other_top, float other_sum, float c) {
  const float t = fmaxf(top, other_top);
  if (t == -INFINITY) {
    sum += other_sum;
  } else {
    sum = sum * fast_exp2((top - t) * c) + other_sum * fast_exp2((other_top - t) * c);
  }
  top = t;
}

// The better of two (value, index): the larger, of equals the lower index.
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
  if (v2 > v || (v2 == v && i2 < i)) v = v2, i = i2;
}

// One CTA a part of a row.
template <typename T> __global__ void __launch_bounds__(ROW_THREADS) verify_rows_kernel(const VerifyParams p) {
  constexpr int VEC = Row<T>::VEC, WARPS = ROW_THREADS / 32;
  const ucb_verify_args& a = p.a;
  block8::launch_dependents();
  const int rows = a.drafts_n + 1, split = blockIdx.x % p.splits, r = blockIdx.x / p.splits, s = r / rows, j = r % rows;
  if (j > count_of(a, s)) return;
  const Row<T> row(a.logits, s * a.logits_stride_seq + j * a.logits_stride_row, a.vocab);
  const float temperature = temperature_of(a, s), c = LOG2E / heat_of(temperature);
  const bool greedy = temperature <= 0.f;
  const int each = (row.vectors + p.splits - 1) / p.splits, begin = split * each, end = min(row.vectors, begin + each);
  float top = -INFINITY, sum = 0.f, best_value = -INFINITY;
  int best = 0x7fffffff;
  for (int k = begin + threadIdx.x; k < end; k += ROW_THREADS * ROW_AHEAD) {
    float x[ROW_AHEAD][VEC];
#pragma unroll
    for (int u = 0; u < ROW_AHEAD; ++u) {
      if (k + u * ROW_THREADS < end) {
        row.load(k + u * ROW_THREADS, x[u]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[u][e] = -INFINITY;
      }
    }
    float t = top;
#pragma unroll
    for (int u = 0; u < ROW_AHEAD; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) t = fmaxf(t, x[u][e]);
    if (greedy) {
#pragma unroll
      for (int u = 0; u < ROW_AHEAD; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (x[u][e] > best_value) best_value = x[u][e], best = row.first(k + u * ROW_THREADS) + e;
    }
    if (t > top) sum *= fast_exp2((top - t) * c);
    top = t;
    const float from = t == -INFINITY ? 0.f : t;
#pragma unroll
    for (int u = 0; u < ROW_AHEAD; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += fast_exp2((x[u][e] - from) * c);
  }
  __shared__ Partial part[WARPS];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, top, o), q = __shfl_xor_sync(0xffffffffu, sum, o);
    if (greedy) {
      const float v = __shfl_xor_sync(0xffffffffu, best_value, o);
      const int i = __shfl_xor_sync(0xffffffffu, best, o);
      better(best_value, best, v, i);
    }
    join(top, sum, t, q, c);
  }
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = {top, sum, best, 0};
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < WARPS; ++w) {
    better(best_value, best, part[w].top, part[w].best);
    join(top, sum, part[w].top, part[w].sum, c);
  }
  p.partials[blockIdx.x] = {top, sum, best, 0};
}

enum Weights { ALL, LEFT, OTHERS };  // p; what the draft's distribution leaves of it; p without the draft

// One cluster a sequence: the tests, then the next token.
template <typename T, typename Q> __global__ void __launch_bounds__(DRAW_THREADS) verify_draw_kernel(const VerifyParams p) {
  constexpr int VEC = Row<T>::VEC;
  const ucb_verify_args& a = p.a;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = cluster.block_rank(), ctas = cluster.num_blocks(), s = blockIdx.x / ctas;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = a.drafts_n + 1, count = count_of(a, s);
  __shared__ Partial part[MAX_ROWS];
  __shared__ int accepted_at;
  __shared__ double warp_sum[2][DRAW_WARPS], all_sum[DRAW_WARPS * DRAW_CLUSTER], drawn[3];
  const float temperature = temperature_of(a, s);
  const bool greedy = temperature <= 0.f;
  const float c = LOG2E / heat_of(temperature);
  const double inverse = 1.0 / (double)heat_of(temperature);
  block8::wait_for_primary();
  for (int j = warp; j <= count; j += DRAW_WARPS) {
    float top = -INFINITY, sum = 0.f, best_value = -INFINITY;
    int best = 0x7fffffff;
    for (int i = lane; i < p.splits; i += 32) {
      const Partial x = p.partials[((int64_t)s * rows + j) * p.splits + i];
      better(best_value, best, x.top, x.best);
      join(top, sum, x.top, x.sum, c);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, top, o), q = __shfl_xor_sync(0xffffffffu, sum, o);
      const float v = __shfl_xor_sync(0xffffffffu, best_value, o);
      const int i = __shfl_xor_sync(0xffffffffu, best, o);
      better(best_value, best, v, i);
      join(top, sum, t, q, c);
    }
    if (lane == 0) part[j] = {top, sum, best, 0};
  }
  __syncthreads();
  // ---- the drafts, a lane each
  const T* logits = static_cast<const T*>(a.logits) + s * a.logits_stride_seq;
  const Q* probs = static_cast<const Q*>(a.draft_probs) + s * a.probs_stride_seq;
  auto draft_of = [&](int j) {
    const int64_t at = s * a.drafts_stride_seq + j;
    return a.drafts_64 ? static_cast<const int64_t*>(a.drafts)[at] : (int64_t)static_cast<const int32_t*>(a.drafts)[at];
  };
  auto logprob_of = [&](int j, int64_t x) {
    return ((double)Dtype<T>::to_f(logits[j * a.logits_stride_row + x]) - (double)part[j].top) * inverse - log((double)part[j].sum);
  };
  if (warp == 0) {
    bool stays = false, outside = false;
    int64_t x = -1;
    double logprob = 0.0;
    if (lane < count) {
      x = draft_of(lane);
      outside = x < 0 || x >= a.vocab;
      if (!outside) {
        logprob = logprob_of(lane, x);
        const double q = a.draft_probs ? (double)Dtype<Q>::to_f(probs[lane * a.probs_stride_row + x]) : 1.0;
        stays = greedy ? x == part[lane].best && part[lane].sum < INFINITY : (double)a.uniforms[s * a.uniforms_stride_seq + lane] * q < exp(logprob);
      }
    }
    const unsigned falls = ~__ballot_sync(0xffffffffu, stays);
    const int accepted = min(count, falls ? __ffs(falls) - 1 : 32);
    if (lane == 0) accepted_at = accepted;
    if (rank == 0) {
      if (lane < rows && lane != accepted) {
        a.tokens[s * rows + lane] = lane < accepted ? (int)x : -1;
        a.logprobs[s * rows + lane] = lane < accepted ? (float)logprob : 0.f;
      }
      if (lane == 0) {
        a.accepted[s] = accepted;
        if (a.lengths) a.lengths[s] -= count - accepted;
        if (a.counts && a.counts[s] != count) outside = true;
      }
      if (outside && lane <= accepted) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    }
  }
  __syncthreads();
  const int j = accepted_at;
  const float sum = part[j].sum;
  auto answer = [&](int token) {
    a.tokens[s * rows + j] = token;
    a.logprobs[s * rows + j] = token < 0 ? __int_as_float(0x7fffffff) : (float)logprob_of(j, token);
    if (token < 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
  };
  const bool none = !(sum > 0.f && sum < INFINITY);  // a NaN or an infinity among the logits, or nothing but -inf
  if (none || greedy) {
    if (rank == 0 && threadIdx.x == 0) answer(none ? -1 : part[j].best);
    return;
  }
  // ---- the draw, over the whole row in fp64
  const Row<T> row(logits, j * a.logits_stride_row, a.vocab);
  const Q* left = probs + j * a.probs_stride_row;
  const int64_t draft = j < count ? draft_of(j) : -1;
  const bool named = draft >= 0 && draft < a.vocab;
  Weights kind = !named ? ALL : a.draft_probs ? LEFT : OTHERS;
  const double top = part[j].top;
  double unit = 1.0;  // 1 / the sum of the exponentials, where p itself is needed
  const int parts = ctas * DRAW_WARPS, mine = rank * DRAW_WARPS + warp, each = (row.vectors + parts - 1) / parts;
  const int begin = min(row.vectors, mine * each), end = min(row.vectors, begin + each);
  auto weights = [&](int k, Weights of, double (&w)[VEC]) {
    float x[VEC], q[VEC];
    row.load(k, x);
    if (of == LEFT) load_probs<Q, VEC>(left, row.first(k), a.vocab, q);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[e] = exp(((double)x[e] - top) * inverse);
      if (of == LEFT) {
        const double rest = w[e] * unit - (double)q[e];
        w[e] = rest <= 0.0 ? 0.0 : rest;  // a NaN stays
      } else if (of == OTHERS && row.first(k) + e == draft) {
        w[e] = 0.0;
      }
    }
  };
  int turn = 0;
  // The sum over the row, and of the parts in front of the one that holds `share` of it; the part.
  auto add_up = [&](Weights of, double share, double& before, int& owner) {
    double mine_sum = 0.0;
    for (int k = begin + lane; k < end; k += 32) {
      double w[VEC];
      weights(k, of, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) mine_sum += w[e];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine_sum += __shfl_xor_sync(0xffffffffu, mine_sum, o);
    if (lane == 0) warp_sum[turn][warp] = mine_sum;
    cluster.sync();
    for (int i = threadIdx.x; i < parts; i += DRAW_THREADS)
      all_sum[i] = *cluster.map_shared_rank(&warp_sum[turn][i % DRAW_WARPS], i / DRAW_WARPS);
    turn ^= 1;
    __syncthreads();
    if (warp == 0) {
      constexpr int EACH = DRAW_WARPS * DRAW_CLUSTER / 32;
      double v[EACH], lane_sum = 0.0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = lane * EACH + i < parts ? all_sum[lane * EACH + i] : 0.0, lane_sum += v[i];
      double run = lane_sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += x;
      }
      const double total = __shfl_sync(0xffffffffu, run, 31), target = share * total;
      double at = __shfl_up_sync(0xffffffffu, run, 1);
      if (lane == 0) at = 0.0;
      // the first part that reaches above the target; where rounding leaves none, the last one with a weight
      int found = parts, last = -1;
      double found_at = 0.0, last_at = 0.0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        if (v[i] > 0.0) {
          if (found == parts && at + v[i] > target) found = lane * EACH + i, found_at = at;
          last = lane * EACH + i, last_at = at;
        }
        at += v[i];
      }
      const int first = __reduce_min_sync(0xffffffffu, found), final = __reduce_max_sync(0xffffffffu, last);
      const int which = first < parts ? first : final;
      if (lane == 0) drawn[0] = total, drawn[1] = which;
      __syncwarp();
      if (which >= 0 && lane == which / EACH) drawn[2] = first < parts ? found_at : last_at;
    }
    __syncthreads();
    const double total = drawn[0];
    before = drawn[2], owner = (int)drawn[1];
    return total;
  };
  const double share = (double)a.uniforms[s * a.uniforms_stride_seq + a.drafts_n];
  double before, total;
  int owner;
  if (kind == LEFT) unit = 1.0 / add_up(ALL, share, before, owner);
  total = add_up(kind, share, before, owner);
  if (kind != ALL && total == 0.0) {  // nothing is left: from p itself
    kind = ALL;
    total = add_up(ALL, share, before, owner);
  }
  cluster.sync();  // no CTA ends while others read its sums
  if (!(total > 0.0 && total < INFINITY)) {
    if (rank == 0 && threadIdx.x == 0) answer(-1);
    return;
  }
  if (mine != owner) return;
  const double target = share * total;
  double run = before;
  int last = -1;
  for (int k0 = begin; k0 < end; k0 += 32) {
    const int k = k0 + lane;
    double w[VEC], sum = 0.0;
    if (k < end) {
      weights(k, kind, w);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = 0.0;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += w[e];
    double upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    double at = __shfl_up_sync(0xffffffffu, upto, 1);
    at = run + (lane ? at : 0.0);
    int token = -1, positive = -1;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (w[e] > 0.0) {
        positive = row.first(k) + e;
        if (token < 0 && at + w[e] > target) token = positive;
      }
      at += w[e];
    }
    last = max(last, __reduce_max_sync(0xffffffffu, positive));
    const unsigned found = __ballot_sync(0xffffffffu, token >= 0);
    if (found) {
      last = __shfl_sync(0xffffffffu, token, __ffs(found) - 1);
      break;
    }
    run += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (lane == 0) answer(last);
}

template <typename T, typename Q> int launch_draw(const VerifyParams& p, cudaStream_t s) {
  return block8::launch(verify_draw_kernel<T, Q>, dim3((unsigned)p.a.seqs * DRAW_CLUSTER), dim3(DRAW_THREADS), 0, s, p,
                        "verify_draw_kernel", DRAW_CLUSTER, true);
}

template <typename T> int launch_all(const VerifyParams& p, cudaStream_t s) {
  const unsigned grid = (unsigned)((int64_t)p.a.seqs * (p.a.drafts_n + 1) * p.splits);
  if (int rc = block8::launch(verify_rows_kernel<T>, dim3(grid), dim3(ROW_THREADS), 0, s, p, "verify_rows_kernel")) return rc;
  switch (p.a.draft_probs ? p.a.probs_dtype : UCB_F32) {
    case UCB_BF16: return launch_draw<T, __nv_bfloat16>(p, s);
    case UCB_F16: return launch_draw<T, __half>(p, s);
    default: return launch_draw<T, float>(p, s);
  }
}

// Parts of a row: CTAs for every multiprocessor, none with less than one round of its threads' loads.
int splits_of(int64_t rows, int vocab, int dtype) {
  const int sms = ucb_host::multiprocessors();
  if (sms < 1) return -1;
  const int64_t vectors = (vocab + 7) / (dtype == UCB_F32 ? 4 : 8) + 1;
  const int64_t most = std::max<int64_t>(1, vectors / ROW_THREADS), wanted = (sms * 6 + rows - 1) / rows;
  return (int)std::min<int64_t>(64, std::min(most, wanted));
}

}  // namespace
}  // namespace verify
}  // namespace ucb

using ucb_host::set_error;
namespace uv = ucb::verify;

extern "C" int64_t ucb_verify_drafts_workspace_bytes(int seqs, int drafts, int vocab, int dtype) {
  if (seqs < 1 || drafts < 0 || drafts >= uv::MAX_ROWS || vocab < 1) return -1;
  const int splits = uv::splits_of((int64_t)seqs * (drafts + 1), vocab, dtype);
  return splits < 1 ? -1 : (int64_t)seqs * (drafts + 1) * splits * (int64_t)sizeof(uv::Partial);
}

extern "C" int ucb_verify_drafts(const ucb_verify_args* a, void* stream) {
  const char* what = "ucb_verify_drafts";
  if (!a) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (a->seqs < 0 || a->drafts_n < 0 || a->vocab < 1) return set_error(UCB_ERR_INVALID, "%s: bad shape", what);
  if (a->drafts_n >= uv::MAX_ROWS) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most %d drafts", what, uv::MAX_ROWS - 1);
  if (a->vocab > 0x7fffff00 || (int64_t)a->seqs * (a->drafts_n + 1) > 0x1ffffff)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: too many rows or tokens", what);
  if (!(a->temperature_all >= 0.f && a->temperature_all < 3.0e38f)) return set_error(UCB_ERR_INVALID, "%s: bad temperature", what);
  if (a->seqs == 0) return UCB_OK;
  if (!a->logits || (a->drafts_n && !a->drafts) || !a->uniforms || !a->tokens || !a->accepted || !a->logprobs || !a->workspace)
    return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return set_error(UCB_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  if (a->draft_probs && a->probs_dtype != UCB_BF16 && a->probs_dtype != UCB_F16 && a->probs_dtype != UCB_F32)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: unsupported dtype", what);
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  const int splits = uv::splits_of((int64_t)a->seqs * (a->drafts_n + 1), a->vocab, a->dtype);
  if (splits < 1) return set_error(UCB_ERR_CUDA, "%s: the device's multiprocessors are unknown", what);
  const uv::VerifyParams p{*a, static_cast<uv::Partial*>(a->workspace), splits, err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case UCB_BF16: return uv::launch_all<__nv_bfloat16>(p, s);
    case UCB_F16: return uv::launch_all<__half>(p, s);
    case UCB_F32: return uv::launch_all<float>(p, s);
    default: return set_error(UCB_ERR_UNSUPPORTED, "%s: unsupported dtype", what);
  }
}
