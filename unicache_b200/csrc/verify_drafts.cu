// Verification of drafted tokens against the target's distribution (ucb_verify_drafts):
//   p_j = softmax(logits_j / T),  draft x_j stays while u_j q_j(x_j) < p_j(x_j);
// at the first one that does not, a, the next token is drawn from max(p_a - q_a, 0), after all of
// them from p_n: the first token whose running sum is above u_n times the sum.
//
// The first kernel reads every row once, many CTAs a row, maximum and sum in fp32: the tests compare numbers of
// relative error 1e-6 with a random one.  The draw is another matter: in the long flat tail of a vocabulary a running
// sum off by d names another token with a probability of up to d times the number of
// tokens, which is percents for fp32.  So the one row of each sequence that is drawn from
// is summed in fp64, exponentials included, by the second kernel.
//
// Measured on the device: 32 sequences of 4 drafts, 151936 tokens in bf16 with fp32 draft distributions (68 MB, 10.4 us of memory) take
// 32.8 us: 13 for the rows, 19 for the draw, of which 7 are the sums and 8 the way from test to token.  64 sequences of 7
// drafts in fp32 (331 MB, 50.6 us) take 73, 83 where most of the drafts fall; one sequence of 4 drafts, 32000 tokens 10.4, of which 8 are that way.
#include <algorithm>
#include <type_traits>

#include "block8.cuh"

namespace ucb {
namespace verify {
namespace {

constexpr int MAX_ROWS = 32;  // of a sequence: its drafts and the one behind them
constexpr int ROW_THREADS = 256, ROW_AHEAD = 4, ROW_VECTORS = ROW_THREADS * ROW_AHEAD;  // of a part of a row
constexpr int DRAW_THREADS = 256, DRAW_WARPS = DRAW_THREADS / 32, DRAW_CTAS = 3;
constexpr int MAX_PARTS = 1024;  // of the row that is drawn from, a warp each
constexpr float LOWEST = -3.40282347e38f;
constexpr float LOG2E = 1.4426950408889634f;

struct Partial {
  float top, sum;  // of exp((x - top) / T)
  int best;        // the first index of the top, where it is asked for
  int unused;
};

enum Weights : int { ALL, LEFT, OTHERS, ANSWERED };  // p; what the draft's distribution leaves of it; p without the draft; no draw

// Of some elements: the sum of their e; and for LEFT what remains of them, the e of those of which something does, and how many
// of them are so near to the border that they may be on its other side (TOO_MANY: more than were kept).
struct __align__(16) Sums {
  double all, left, e_left, near;
};
struct __align__(16) NearElement {
  double e;
  float q;
  float unused;
};
constexpr int NEAR_KEPT = 8;  // of a part
constexpr double TOO_MANY = 1e9;

struct VerifyParams {
  ucb_verify_args a;
  Partial* partials;  // [seqs * rows][splits]
  Sums* sums;         // [seqs][ctas * DRAW_WARPS]
  NearElement* near;  // [seqs][ctas * DRAW_WARPS][NEAR_KEPT]
  unsigned int* done;  // [seqs]: CTAs whose sums are there
  int splits, ctas, part_vectors;
  unsigned int* err;
};

// A row of the vocabulary as 16-byte vectors from the aligned address at or before its start: vector k holds the elements
// k * VEC - shift and on.  Vectors [full_begin, full_end) lie inside; one before and one behind them may have some elements.
template <typename T> struct Row {
  static constexpr int VEC = 16 / sizeof(T);
  const T* x;
  int shift, vocab, vectors, full_begin, full_end;
  __device__ Row(const void* base, int64_t at, int vocab_) : x(static_cast<const T*>(base) + at), vocab(vocab_) {
    shift = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    vectors = (int)(((int64_t)vocab + shift + VEC - 1) / VEC);
    full_begin = shift ? 1 : 0;
    full_end = (int)(((int64_t)vocab + shift) / VEC);
  }
  __device__ __forceinline__ int first(int k) const { return k * VEC - shift; }
  static __device__ __forceinline__ void to_float(uint4 w, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 2) {
      v[0] = Dtype<T>::lo(w.x), v[1] = Dtype<T>::hi(w.x), v[2] = Dtype<T>::lo(w.y), v[3] = Dtype<T>::hi(w.y);
      v[4] = Dtype<T>::lo(w.z), v[5] = Dtype<T>::hi(w.z), v[6] = Dtype<T>::lo(w.w), v[7] = Dtype<T>::hi(w.w);
    } else {
      v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
  }
  static __device__ __forceinline__ uint4 nothing() {  // -inf throughout
    const uint32_t w = sizeof(T) == 4 ? 0xff800000u : Dtype<T>::code == UCB_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    return make_uint4(w, w, w, w);
  }
  // The largest of some vectors' elements that are numbers; two 16-bit ones at a time.
  template <int N> static __device__ __forceinline__ float top_of(const uint4 (&w)[N]) {
    if constexpr (sizeof(T) == 2) {
      uint32_t top = nothing().x;
#pragma unroll
      for (int u = 0; u < N; ++u) top = larger(larger(top, larger(w[u].x, w[u].y)), larger(w[u].z, w[u].w));
      return fmaxf(Dtype<T>::lo(top), Dtype<T>::hi(top));
    } else {
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < N; ++u)
        top = fmaxf(fmaxf(fmaxf(top, __uint_as_float(w[u].x)), __uint_as_float(w[u].y)), fmaxf(__uint_as_float(w[u].z), __uint_as_float(w[u].w)));
      return top;
    }
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {  // of two pairs, that of a number and a NaN the number
    if constexpr (Dtype<T>::code == UCB_BF16) {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __half2 m = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&m);
    }
  }
  // Any vector as bits, -inf outside the row.
  __device__ __forceinline__ uint4 load(int k) const {
    if (k >= full_begin && k < full_end) return *reinterpret_cast<const uint4*>(x + first(k));
    union {
      uint4 w;
      T e[VEC];
    } u;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int i = first(k) + e;
      u.e[e] = i >= 0 && i < vocab ? x[i] : Dtype<T>::from_f(-INFINITY);
    }
    return u.w;
  }
};

// N elements of a row of draft probabilities from i on, as they lie in memory; 0 outside the vocabulary.
template <typename Q, int N> struct Probs {
  static constexpr int BYTES = N * sizeof(Q), ALIGN = BYTES < 16 ? BYTES : 16;
  union {
    uint4 w16[(BYTES + 15) / 16];
    uint2 w8;
    Q e[N];
  };
  __device__ __forceinline__ Probs() {}
  __device__ __forceinline__ void load(const Q* q) {  // all of them inside
    if (reinterpret_cast<uintptr_t>(q) % ALIGN == 0) {
      if constexpr (BYTES >= 16) {
#pragma unroll
        for (int k = 0; k < BYTES / 16; ++k) w16[k] = reinterpret_cast<const uint4*>(q)[k];
      } else {
        w8 = *reinterpret_cast<const uint2*>(q);
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) e[k] = q[k];
    }
  }
  __device__ __forceinline__ void load(const Q* q, int i, int vocab) {
    if (i >= 0 && i + N <= vocab) {
      load(q + i);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) e[k] = i + k >= 0 && i + k < vocab ? q[i + k] : Dtype<Q>::from_f(0.f);
    }
  }
  __device__ __forceinline__ float operator[](int k) const { return Dtype<Q>::to_f(e[k]); }
};

__device__ __forceinline__ float temperature_of(const ucb_verify_args& a, int s) { return a.temperature ? a.temperature[s] : a.temperature_all; }

// The temperature that exponents are divided by: 1 for the log-probabilities of greedy sequences, else within 1e-30 to 1e30, where
// neither the division nor a masked element's exponent leaves fp32's range.  NaN stays, and leaves no distribution.
__device__ __forceinline__ float heat_of(float temperature) {
  return temperature <= 0.f ? 1.f : temperature < 1e-30f ? 1e-30f : temperature > 1e30f ? 1e30f : temperature;
}

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

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float2 halves_of(uint64_t a) {
  float2 v;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(a));
  return v;
}

// One CTA a part of a row, all of it loaded at once: its maximum first, then the exponentials against that.  512 rows of 151936 in
// fp32 (311 MB) take 46 us (6.8 TB/s).  160 rows in bf16 (49 MB) take 13: four rounds of CTAs, each of which waits for its count and
// then for its loads; twice the loads a thread 14.3, half of them 14.5, several parts a CTA with the next one in flight 13.8.
template <typename T> __global__ void __launch_bounds__(ROW_THREADS) verify_rows_kernel(const VerifyParams p) {
  constexpr int VEC = Row<T>::VEC, WARPS = ROW_THREADS / 32;
  const ucb_verify_args& a = p.a;
  block8::launch_dependents();
  const int split = blockIdx.x, j = blockIdx.y, s = blockIdx.z;
  if (j > count_of(a, s)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (j == 0 && split == 0 && threadIdx.x == 0) p.done[s] = 0;  // for the next kernel
  const Row<T> row(a.logits, s * a.logits_stride_seq + j * a.logits_stride_row, a.vocab);
  const int begin = split * ROW_VECTORS + threadIdx.x;
  uint4 raw[ROW_AHEAD];
#pragma unroll
  for (int u = 0; u < ROW_AHEAD; ++u) {
    const int k = begin + u * ROW_THREADS;
    raw[u] = k < row.vectors ? row.load(k) : Row<T>::nothing();
  }
  const float temperature = temperature_of(a, s), c = LOG2E / heat_of(temperature);
  float top = Row<T>::top_of(raw);
  __shared__ float warp_top[WARPS], warp_sum[WARPS];
  __shared__ int warp_best[WARPS];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, warp_top[w]);
  const float from = top == -INFINITY ? 0.f : -top;  // where there is nothing above -inf the exponentials are 0, or NaN
  const uint64_t from2 = pair_of(from, from), c2 = pair_of(c, c);
  uint64_t sum2 = 0;
#pragma unroll
  for (int u = 0; u < ROW_AHEAD; ++u) {
    float x[VEC];
    Row<T>::to_float(raw[u], x);
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const uint64_t y = mul_pair(add_pair(pair_of(x[e], x[e + 1]), from2), c2);
      const float2 each = halves_of(y);
      sum2 = add_pair(sum2, pair_of(fast_exp2(each.x), fast_exp2(each.y)));
    }
  }
  const float2 sums = halves_of(sum2);
  float sum = sums.x + sums.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  int best = 0x7fffffff;
  if (temperature <= 0.f) {  // the first of the largest
#pragma unroll
    for (int u = ROW_AHEAD - 1; u >= 0; --u) {
      float x[VEC];
      Row<T>::to_float(raw[u], x);
#pragma unroll
      for (int e = VEC - 1; e >= 0; --e)
        if (x[e] == top) best = row.first(begin + u * ROW_THREADS) + e;
    }
    best = __reduce_min_sync(0xffffffffu, best);
  }
  if (lane == 0) warp_sum[warp] = sum, warp_best[warp] = best;
  __syncthreads();
  if (threadIdx.x) return;
#pragma unroll
  for (int w = 1; w < WARPS; ++w) sum += warp_sum[w], best = min(best, warp_best[w]);
  p.partials[((int64_t)s * gridDim.y + j) * gridDim.x + split] = {top, sum, best, 0};
}

// exp(d * T^-1) of the draw, by a table as in Tang, "Table-Driven Implementation of the Exponential Function in IEEE Floating-Point
// Arithmetic" (ACM TOMS 1989): 2^(k / 16), k the nearest whole number of the exponent in sixteenths, times a
// polynomial in what is left of it (Taylor's to the fifth power, off by 1.4e-13 at most).  What is below e^-350 is taken as something
// between e^-350 and e^-700: with masked elements it is below NOTHING wherever weights are compared.
constexpr double NOTHING = 1e-145;
constexpr double SIXTEENTH = 0.69314718055994530942 / 16.0;
struct Steps {
  double power[6], magic, sixteenth[16];  // 2^(j / 16)
};
// The magic number is 1.5 * 2^52, whose last bit is 1.
__constant__ Steps STEPS = {{1.0, SIXTEENTH, SIXTEENTH * SIXTEENTH / 2.0, SIXTEENTH * SIXTEENTH * SIXTEENTH / 6.0,
                             SIXTEENTH * SIXTEENTH * SIXTEENTH * SIXTEENTH / 24.0,
                             SIXTEENTH * SIXTEENTH * SIXTEENTH * SIXTEENTH * SIXTEENTH / 120.0},
                            6755399441055744.0,
                            {1.00000000000000000000, 1.04427378242741384032, 1.09050773266525765921, 1.13878863475669165370,
                             1.18920711500272106672, 1.24185781207348404859, 1.29683955465100966593, 1.35425554693689272830,
                             1.41421356237309504880, 1.47682614593949931139, 1.54221082540794082361, 1.61049033194925430818,
                             1.68179283050742908606, 1.75625216037329948311, 1.83400808640934246349, 1.91520656139714729387}};
template <typename T> struct Exponential {
  double top, scale;  // 16 log2(e) / T
  float floor;        // no more than 700 T below the top
  bool halved;        // of the elements' halves: next to fp32's lowest number nothing lies between an element and -inf
  const double* table;
  __device__ Exponential(float top_, double heat, const double* table_) : table(table_) {
    halved = sizeof(T) == 4 && top_ < 0.5f * LOWEST;
    if (halved) top_ *= 0.5f, heat *= 0.5;
    top = top_;
    // where T is so small that the next smaller number is below e^-350 already, any T for which it is will do
    heat = fmax(heat, (top - (double)nextafterf(top_, -INFINITY)) / 350.0);
    scale = 16.0 * 1.4426950408889634074 / heat;
    floor = fmaxf(__double2float_rd(top - 350.0 * heat), LOWEST);
  }
  template <int N> __device__ __forceinline__ void prepare(float (&x)[N]) const {
    if (sizeof(T) == 4 && halved)
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] *= 0.5f;
  }
  __device__ __forceinline__ double operator()(float x) const {  // of a prepared element
    const double d = (double)fmaxf(x, floor) - top, t = fma(d, scale, STEPS.magic), f = fma(d, scale, STEPS.magic - t);
    const int k = __double2loint(t);
    double e = fma(f, STEPS.power[5], STEPS.power[4]);
    e = fma(f, e, STEPS.power[3]);
    e = fma(f, e, STEPS.power[2]);
    e = fma(f, e, STEPS.power[1]);
    e = fma(f, e, STEPS.power[0]);
    const double step = table[k & 15];
    return e * __hiloint2double(__double2hiint(step) + ((k & ~15) << 16), __double2loint(step));
  }
};

// Whether something remains: above 0, or no number.  By the bits, no compare on the fp64 pipe.
__device__ __forceinline__ bool remains(double rest) { return ((uint32_t)__double2hiint(rest) ^ 0x80000000u) > 0x7ff00000u; }

// Whether an element's rest is below some 2^-19 of q, by the numbers' upper words.  Infinities and NaN count as near.
__device__ __forceinline__ bool is_near(double rest, double q) { return (__double2hiint(rest) & 0x7fffffff) + (19 << 20) < __double2hiint(q); }

// Adds what remains of an element, predicated: a branch would cost more.
__device__ __forceinline__ void add_remaining(Sums& s, double rest, double e) {
  asm("{\n .reg .pred p;\n setp.gt.u32 p, %2, 0x7ff00000;\n @p add.f64 %0, %0, %3;\n @p add.f64 %1, %1, %4;\n}\n"
      : "+d"(s.left), "+d"(s.e_left)
      : "r"(__double2hiint(rest) ^ 0x80000000), "d"(rest), "d"(e));
}

// The sums of a warp's vectors [begin, end), the lanes side by side, the same in every lane.  What the draft leaves of p,
// max(e / Z - q, 0) with Z the sum of all e, would need a pass for Z first.  This one takes the fp32 sum instead, 1 / `unit`: as long as
// the same elements remain, the sums of what they leave and of their e give those for Z itself.  Elements that are so near to the border
// that they may change sides are kept, for the two sums to be put right; where they are too many (a draft's distribution that is
// the target's but for its rounding), the pass is made again with Z.  One loop of little code: most calls go
// through it once or a few times, and what costs most then is to fetch the instructions.
template <typename T, typename Q> __device__ __forceinline__ Sums sum_vectors(const Row<T>& row, const Q* left, int begin, int end,
                                                                              const Exponential<T>& exponential, Weights kind,
                                                                              double unit, int fallen, NearElement* kept) {
  constexpr int VEC = Row<T>::VEC;
  const int lane = threadIdx.x & 31, first = max(begin, row.full_begin), last = min(end, row.full_end);
  const int but = kind == OTHERS ? fallen : -1;
  Sums s = {0.0, 0.0, 0.0, 0.0};
  int near_mine = 0;
  NearElement near_first, near_second;
  auto keep = [&](double e, double rest, double q) {
    if (!is_near(rest, q)) return;
    (near_mine ? near_second : near_first) = {e, (float)q, 0.f};
    ++near_mine;
  };
  // ---- the full vectors, the next one in flight
  int i = row.first(first + lane), left_over = (last - first - lane + 31) >> 5;
  const uint4* at = reinterpret_cast<const uint4*>(row.x + i);
  uint4 next_x = make_uint4(0, 0, 0, 0);
  Probs<Q, VEC> next_q;
#pragma unroll
  for (int e = 0; e < VEC; ++e) next_q.e[e] = Dtype<Q>::from_f(0.f);
  if (left_over > 0) {
    next_x = *at;
    if (kind == LEFT) next_q.load(left + i);
  }
#pragma unroll 1
  for (; left_over > 0; --left_over) {
    float x[VEC];
    Row<T>::to_float(next_x, x);
    exponential.prepare(x);
    const Probs<Q, VEC> now_q = next_q;
    if ((unsigned)(but - i) < VEC)
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (i + e == but) x[e] = -INFINITY;
    at += 32, i += 32 * VEC;
    if (left_over > 1) {
      next_x = *at;
      if (kind == LEFT) next_q.load(left + i);
    }
    double e[VEC];
#pragma unroll
    for (int u = 0; u < VEC; ++u) e[u] = exponential(x[u]);
    if (kind == LEFT) {
      bool near = false;
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const double q = (double)now_q[u], rest = fma(e[u], unit, -q);
        add_remaining(s, rest, e[u]);
        near |= is_near(rest, q);
      }
      if (near)
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          const double q = (double)now_q[u], rest = fma(e[u], unit, -q);
          keep(e[u], rest, q);
        }
    }
#pragma unroll
    for (int o = 1; o < VEC; o *= 2)
#pragma unroll
      for (int u = 0; u < VEC; u += 2 * o) e[u] += e[u + o];
    s.all += e[0];
  }
  // ---- the row's ends, an element a lane: those in front of the first full vector, then those behind the last one
  if (begin < end && (begin < row.full_begin || end > row.full_end)) {
    const int front = begin < row.full_begin ? min(row.first(row.full_begin), row.vocab) : 0;
    const int behind = end > row.full_end && row.full_end >= row.full_begin ? row.vocab - row.first(row.full_end) : 0;
    const int at_end = lane < front ? lane : row.vocab - behind + lane - front;
    if (lane < front + behind) {
      float x[1] = {at_end == but ? -INFINITY : Dtype<T>::to_f(row.x[at_end])};
      exponential.prepare(x);
      const double e = exponential(x[0]);
      s.all += e;
      if (kind == LEFT) {
        const double q = (double)Dtype<Q>::to_f(left[at_end]), rest = fma(e, unit, -q);
        add_remaining(s, rest, e);
        keep(e, rest, q);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.all += __shfl_xor_sync(0xffffffffu, s.all, o);
    if (kind == LEFT) {
      s.left += __shfl_xor_sync(0xffffffffu, s.left, o);
      s.e_left += __shfl_xor_sync(0xffffffffu, s.e_left, o);
    }
  }
  if (kind == LEFT && __any_sync(0xffffffffu, near_mine)) {
    const unsigned one = __ballot_sync(0xffffffffu, near_mine >= 1), two = __ballot_sync(0xffffffffu, near_mine >= 2);
    const int count = __popc(one) + __popc(two);
    const unsigned before = (1u << lane) - 1;
    s.near = __any_sync(0xffffffffu, near_mine > 2) || count > NEAR_KEPT ? TOO_MANY : count;
    if (kept && s.near < TOO_MANY) {
      if (near_mine >= 1) kept[__popc(one & before)] = near_first;
      if (near_mine >= 2) kept[__popc(one) + __popc(two & before)] = near_second;
    }
  }
  return s;
}

// The weight of summed elements; `correction` is the right unit less the one that they were summed with.
__device__ __forceinline__ double weight_of(const Sums& s, Weights kind, double correction) {
  return kind != LEFT ? s.all : fma(s.e_left, correction, s.left);
}

struct Found {
  double unit, total, before;  // before: the weight in front of the owner's part
  int owner;                   // the part that holds the drawn token; -1: none
  Weights kind;
  bool again;
};

// The whole CTA: from the sums of all parts, the part with the drawn token, or that they have to be made again.  A thread has a few
// adjacent parts.
__device__ __forceinline__ void locate(Sums* sums, const NearElement* kept, int parts, Weights kind, double unit, double share,
                                      bool first_time, Found& found_part) {
  __shared__ Sums warp_sums[DRAW_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = (parts + DRAW_THREADS - 1) / DRAW_THREADS;
  const int begin = min(parts, (int)threadIdx.x * each), end = min(parts, begin + each);
  if (threadIdx.x == 0) found_part.owner = -1, found_part.again = false;
  Sums own, upto, whole, front;
  double right = unit;
#pragma unroll 1
  for (bool settled = !first_time || kind != LEFT;; settled = true) {
    own = {0.0, 0.0, 0.0, 0.0};
    for (int i = begin; i < end; ++i) own.all += sums[i].all, own.left += sums[i].left, own.e_left += sums[i].e_left, own.near += sums[i].near;
    upto = own;  // and the threads in front
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double all = __shfl_up_sync(0xffffffffu, upto.all, o), left = __shfl_up_sync(0xffffffffu, upto.left, o);
      const double e_left = __shfl_up_sync(0xffffffffu, upto.e_left, o), near = __shfl_up_sync(0xffffffffu, upto.near, o);
      if (lane >= o) upto.all += all, upto.left += left, upto.e_left += e_left, upto.near += near;
    }
    if (lane == 31) warp_sums[warp] = upto;
    __syncthreads();
    whole = front = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int i = 0; i < DRAW_WARPS; ++i) {
      if (i == warp) front = whole;
      const Sums x = warp_sums[i];
      whole.all += x.all, whole.left += x.left, whole.e_left += x.e_left, whole.near += x.near;
    }
    if (kind == LEFT) right = 1.0 / whole.all;
    if (settled) break;
    // Elements near the border of the unit that they were summed with may be on its other side for the right one: as long as the two
    // are no further apart than they were looked for, those that were kept are all.
    if (fabs(right - unit) * (1 << 20) > right || whole.near >= TOO_MANY) {
      if (threadIdx.x == 0) found_part.again = true, found_part.unit = right, found_part.kind = kind;
      __syncthreads();
      return;
    }
    if (whole.near == 0.0) break;
    for (int i = begin; i < end; ++i)
      for (int k = 0; k < (int)sums[i].near; ++k) {
        NearElement x;
        *reinterpret_cast<uint4*>(&x) = __ldcg(reinterpret_cast<const uint4*>(kept + i * NEAR_KEPT + k));
        const bool counted = remains(fma(x.e, unit, -(double)x.q));
        const double rest = fma(x.e, right, -(double)x.q);
        if (counted != remains(rest)) sums[i].left += counted ? -rest : rest;
      }
    __syncthreads();
  }
  if (kind == LEFT && whole.left < NOTHING) {
    kind = ALL;  // nothing remains: from p itself, whose sums are here
  } else if (kind == OTHERS && whole.all < NOTHING) {
    kind = ALL;
    if (threadIdx.x == 0) found_part.again = true;
  }
  const double correction = right - unit, total = weight_of(whole, kind, correction), target = share * total;
  front.all += upto.all - own.all, front.left += upto.left - own.left, front.e_left += upto.e_left - own.e_left;
  // The first part that reaches above the target.  The threads' own weights in front may, rounded apart, leave none or two: the lowest
  // part of those, and else the last one with a weight.
  double at = weight_of(front, kind, correction), found_at = at, last_at = at;
  int found = parts, last = -1;
  for (int i = begin; i < end; ++i) {
    const double v = weight_of(sums[i], kind, correction);
    if (v > NOTHING) {
      if (found == parts && at + v > target) found = i, found_at = at;
      last = i, last_at = at;
    }
    at += v;
  }
  __shared__ int firsts[DRAW_WARPS], lasts[DRAW_WARPS];
  const int first = __reduce_min_sync(0xffffffffu, found), final = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) firsts[warp] = first, lasts[warp] = final;
  __syncthreads();
  int which = parts, fallback = -1;
#pragma unroll
  for (int i = 0; i < DRAW_WARPS; ++i) which = min(which, firsts[i]), fallback = max(fallback, lasts[i]);
  const bool reached = which < parts;
  if (!reached) which = fallback;
  if (threadIdx.x == 0) found_part.unit = right, found_part.total = total, found_part.kind = kind;
  if (which >= begin && which < end) found_part.owner = which, found_part.before = reached ? found_at : last_at;
  __syncthreads();
}

__device__ __forceinline__ unsigned int count_release_acquire(unsigned int* n) {
  unsigned int before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(n) : "memory");
  return before;
}

// ln p of a token from its logit.
__device__ __forceinline__ float logprob_of(float logit, const Partial& row, double inverse) {
  return (float)(((double)logit - (double)row.top) * inverse - (double)logf(row.sum));
}

// Some CTAs a sequence, each with some parts of the row that the next token is drawn from, a part a warp.  Which row that is every
// one of them finds by the tests; the first writes down what they say, and whichever is the last to have its sums finds the token.
// 24 rows of 151936 take 19 us.  The sums, 47 instructions an element, issue at 41% of the slots with the 24 warps a multiprocessor
// that 80 registers leave (fp64 pipe 23%; 64 registers spill and take 2 us more, 128 as long); the rest is a chain of
// memory round trips: sums of the rows, tests, counting, all sums, the part, the token.  A cluster of CTAs a sequence in the place of
// the count took 22 us, as some multiprocessors had two sequences' CTAs and others none.
template <typename T, typename Q> __global__ void __launch_bounds__(DRAW_THREADS, DRAW_CTAS) verify_draw_kernel(const VerifyParams p) {
  constexpr int VEC = Row<T>::VEC;
  const ucb_verify_args& a = p.a;
  const int s = blockIdx.y, cta = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = a.drafts_n + 1, count = count_of(a, s);
  __shared__ Partial part[MAX_ROWS];
  __shared__ int accepted_at, fallen_draft;
  __shared__ double sixteenths[16];
  __shared__ bool is_last;
  const float temperature = temperature_of(a, s), heat = heat_of(temperature), c = LOG2E / heat;
  const bool greedy = temperature <= 0.f;
  const double inverse = 1.0 / (double)heat;
  const T* logits = static_cast<const T*>(a.logits) + s * a.logits_stride_seq;
  const Q* probs = static_cast<const Q*>(a.draft_probs) + s * a.probs_stride_seq;
  // what the tests need of the inputs, a lane a draft: before the rows' sums are there
  int64_t draft = -1;
  float draft_logit = 0.f, draft_uniform = 0.f, draft_q = 1.f;
  bool outside = false;
  if (warp == 0 && lane < count) {
    const int64_t at = s * a.drafts_stride_seq + lane;
    draft = a.drafts_64 ? static_cast<const int64_t*>(a.drafts)[at] : (int64_t)static_cast<const int32_t*>(a.drafts)[at];
    draft_uniform = a.uniforms[s * a.uniforms_stride_seq + lane];
    outside = draft < 0 || draft >= a.vocab;
    if (!outside) {
      draft_logit = Dtype<T>::to_f(logits[lane * a.logits_stride_row + draft]);
      if (a.draft_probs) draft_q = Dtype<Q>::to_f(probs[lane * a.probs_stride_row + draft]);
    }
  }
  const double share = fmax((double)a.uniforms[s * a.uniforms_stride_seq + a.drafts_n], 1e-130);  // 0: what is above NOTHING
  if (threadIdx.x < 16) sixteenths[threadIdx.x] = STEPS.sixteenth[threadIdx.x];
  block8::wait_for_primary();
#pragma unroll 1
  for (int j = warp; j <= count; j += DRAW_WARPS) {
    float top = -INFINITY, sum = 0.f, best_value = -INFINITY;
    int best = 0x7fffffff;
#pragma unroll 1
    for (int i = lane; i < p.splits; i += 32) {
      const Partial x = p.partials[((int64_t)s * rows + j) * p.splits + i];
      better(best_value, best, x.top, x.best);
      join(top, sum, x.top, x.sum, c);
    }
    float highest = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, o));
    join(top, sum, highest, 0.f, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    best = __reduce_min_sync(0xffffffffu, best_value == highest ? best : 0x7fffffff);
    if (lane == 0) part[j] = {highest, sum, best, 0};
  }
  __syncthreads();
  // ---- the drafts
  if (warp == 0) {
    bool stays = false;
    if (lane < count && !outside) {
      const Partial& x = part[lane];
      // the sum is off by some 1e-7 in any case, and so may the exponential be
      stays = greedy ? draft == x.best && x.sum > 0.f && x.sum < INFINITY  // a row of nothing but -inf has no best token
                     : (double)draft_uniform * draft_q * (double)x.sum < (double)fast_exp2((draft_logit - x.top) * c);
    }
    const unsigned falls = ~__ballot_sync(0xffffffffu, stays);
    const int accepted = min(count, falls ? __ffs(falls) - 1 : 32);
    if (lane == accepted) fallen_draft = lane < count && !outside ? (int)draft : -1;
    if (lane == 0) accepted_at = accepted;
  }
  __syncthreads();
  const int j = accepted_at, fallen = fallen_draft;
  const Partial here = part[j];
  const bool none = !(here.sum > 0.f && here.sum < INFINITY);  // a NaN or an infinity among the logits, or nothing but -inf
  Weights kind = none || greedy ? ANSWERED : fallen < 0 ? ALL : a.draft_probs ? LEFT : OTHERS;
  auto answer = [&](int token, float logit) {
    a.tokens[s * rows + j] = token;
    a.logprobs[s * rows + j] = token < 0 ? __int_as_float(0x7fffffff) : logprob_of(logit, here, inverse);
    if (token < 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
  };
  if (cta == 0 && warp == 0) {
    if (lane < rows && lane != j) {
      a.tokens[s * rows + lane] = lane < j ? (int)draft : -1;
      a.logprobs[s * rows + lane] = lane < j ? logprob_of(draft_logit, part[lane], inverse) : 0.f;
    }
    if (lane == 0) {
      a.accepted[s] = j;
      if (a.lengths) a.lengths[s] -= count - j;
      if (a.counts && a.counts[s] != count) outside = true;
      if (kind == ANSWERED) answer(none ? -1 : here.best, here.top);
    }
    if (outside && lane <= j) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
  }
  if (kind == ANSWERED) return;

  // ---- the sums of this warp's part
  const Row<T> row(logits, j * a.logits_stride_row, a.vocab);
  const Q* left = probs + j * a.probs_stride_row;
  const Exponential<T> exponential(here.top, heat, sixteenths);
  const int parts = p.ctas * DRAW_WARPS, mine = cta * DRAW_WARPS + warp;
  auto begin_of = [&](int part) { return (int)min((int64_t)row.vectors, (int64_t)part * p.part_vectors); };
  double unit = 1.0 / (double)here.sum;
  __shared__ Sums sums[MAX_PARTS];
  __shared__ Found found_part;
  {
    const Sums w = sum_vectors<T, Q>(row, left, begin_of(mine), begin_of(mine + 1), exponential, kind, unit, fallen,
                                             p.near + ((int64_t)s * parts + mine) * NEAR_KEPT);
    if (lane == 0) p.sums[(int64_t)s * parts + mine] = w;
  }
  __syncthreads();
  // the barrier orders the CTA's sums before the count, which releases them to whoever counts last
  if (threadIdx.x == 0) is_last = count_release_acquire(&p.done[s]) == p.ctas - 1;
  __syncthreads();
  if (!is_last) return;

  // ---- the part that the next token lies in
  for (int i = threadIdx.x; i < 2 * parts; i += DRAW_THREADS)
    reinterpret_cast<uint4*>(sums)[i] = __ldcg(reinterpret_cast<const uint4*>(p.sums + (int64_t)s * parts) + i);
#pragma unroll 1
  for (bool first_time = true;; first_time = false) {
    __syncthreads();
    locate(sums, p.near + (int64_t)s * parts * NEAR_KEPT, parts, kind, unit, share, first_time, found_part);
    kind = found_part.kind, unit = found_part.unit;
    if (!found_part.again) break;
    __syncthreads();
#pragma unroll 1
    for (int i = warp; i < parts; i += DRAW_WARPS) {
      const Sums w = sum_vectors<T, Q>(row, left, begin_of(i), begin_of(i + 1), exponential, kind, unit, fallen, nullptr);
      if (lane == 0) sums[i] = w;
    }
  }
  const double total = found_part.total;
  if (!(total > NOTHING && total < INFINITY)) {
    if (threadIdx.x == 0) answer(-1, 0.f);
    return;
  }
  // ---- the token: a warp for each 32 vectors of the part.  Each time what is looked for is the first that reaches above the
  // target, or where rounding leaves none, the last with a weight.
  __shared__ double warp_weight[DRAW_WARPS];
  __shared__ int firsts[DRAW_WARPS], lasts[DRAW_WARPS], fallback_token;
  __shared__ float fallback_logit;
  const double target = share * total;
  const int begin = begin_of(found_part.owner), end = begin_of(found_part.owner + 1);
  double before = found_part.before;
  bool any = false;  // whether there is a fallback
#pragma unroll 1
  for (int base = begin; base < end; base += DRAW_THREADS) {
    const int k = base + threadIdx.x;
    double w[VEC], all = 0.0;
    float x[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = 0.0, x[i] = 0.f;
    if (k < end) {
      Probs<Q, VEC> q;
      Row<T>::to_float(row.load(k), x);
      if (kind == LEFT) q.load(left, row.first(k), a.vocab);
      float prepared[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) prepared[i] = x[i];
      exponential.prepare(prepared);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        w[i] = exponential(prepared[i]);
        if (kind == LEFT) {
          const double rest = fma(w[i], unit, -(double)q[i]);
          w[i] = remains(rest) ? rest : 0.0;
        } else if (kind == OTHERS && row.first(k) + i == fallen) {
          w[i] = 0.0;
        }
        if (w[i] < NOTHING) w[i] = 0.0;
        all += w[i];
      }
    }
    double upto = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    __syncthreads();  // the last round's weights are read
    if (lane == 31) warp_weight[warp] = upto;
    __syncthreads();
    double at = before;
#pragma unroll
    for (int i = 0; i < DRAW_WARPS; ++i) {
      if (i == warp) at = before;
      before += warp_weight[i];
    }
    double mine_at = __shfl_up_sync(0xffffffffu, upto, 1);
    mine_at = at + (lane ? mine_at : 0.0);
    int token = -1;  // of this lane's
    float logit = 0.f;
    bool reached = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (w[i] > 0.0 && !reached) {
        token = row.first(k) + i, logit = x[i];
        reached = mine_at + w[i] > target;
      }
      mine_at += w[i];
    }
    const unsigned reach = __ballot_sync(0xffffffffu, reached), some = __ballot_sync(0xffffffffu, token >= 0);
    if (lane == 0) firsts[warp] = reach ? warp : DRAW_WARPS, lasts[warp] = some ? warp : -1;
    __syncthreads();
    int first = DRAW_WARPS, latest = -1;
#pragma unroll
    for (int i = 0; i < DRAW_WARPS; ++i) first = min(first, firsts[i]), latest = max(latest, lasts[i]);
    if (first < DRAW_WARPS) {
      if (warp == first && lane == __ffs(reach) - 1) answer(token, logit);
      return;
    }
    if (latest >= 0) {
      any = true;
      if (warp == latest && lane == 31 - __clz(some)) fallback_token = token, fallback_logit = logit;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) answer(any ? fallback_token : -1, any ? fallback_logit : 0.f);
}

template <typename T, typename Q> int launch_draw(const VerifyParams& p, cudaStream_t s) {
  return block8::launch(verify_draw_kernel<T, Q>, dim3(p.ctas, p.a.seqs), dim3(DRAW_THREADS), 0, s, p, "verify_draw_kernel", 1,
                        true);
}

template <typename T> int launch_all(const VerifyParams& p, cudaStream_t s) {
  const dim3 grid(p.splits, p.a.drafts_n + 1, p.a.seqs);
  if (int rc = block8::launch(verify_rows_kernel<T>, grid, dim3(ROW_THREADS), 0, s, p, "verify_rows_kernel")) return rc;
  switch (p.a.draft_probs ? p.a.probs_dtype : UCB_F32) {
    case UCB_BF16: return launch_draw<T, __nv_bfloat16>(p, s);
    case UCB_F16: return launch_draw<T, __half>(p, s);
    default: return launch_draw<T, float>(p, s);
  }
}

// How a call is cut up; false where the device cannot be asked.
struct Layout {
  int64_t splits, ctas, part_vectors, partials_bytes, sums_bytes, near_bytes, bytes;
  bool make(int64_t seqs, int64_t rows, int64_t vocab, int dtype) {
    const int sms = ucb_host::multiprocessors();
    if (sms < 1) return false;
    const int64_t vectors = vocab / (dtype == UCB_F32 ? 4 : 8) + 2;  // with those that rows not starting on 16 bytes add
    splits = (vectors + ROW_VECTORS - 1) / ROW_VECTORS;
    // the row that is drawn from: as many CTAs as are resident together
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(MAX_PARTS / DRAW_WARPS, (int64_t)sms * DRAW_CTAS / seqs));
    part_vectors = (vectors + most * DRAW_THREADS - 1) / (most * DRAW_THREADS) * 32;
    ctas = (vectors + part_vectors * DRAW_WARPS - 1) / (part_vectors * DRAW_WARPS);
    partials_bytes = seqs * rows * splits * (int64_t)sizeof(Partial);
    sums_bytes = seqs * ctas * DRAW_WARPS * (int64_t)sizeof(Sums);
    near_bytes = seqs * ctas * DRAW_WARPS * NEAR_KEPT * (int64_t)sizeof(NearElement);
    bytes = partials_bytes + sums_bytes + near_bytes + seqs * (int64_t)sizeof(unsigned int);
    return true;
  }
};

}  // namespace
}  // namespace verify
}  // namespace ucb

using ucb_host::set_error;
namespace uv = ucb::verify;

extern "C" int64_t ucb_verify_drafts_workspace_bytes(int seqs, int drafts, int vocab, int dtype) {
  if (seqs < 1 || seqs > 65535 || drafts < 0 || drafts >= uv::MAX_ROWS || vocab < 1 || vocab > 1 << 30) return -1;
  uv::Layout layout;
  return layout.make(seqs, drafts + 1, vocab, dtype) ? layout.bytes : -1;
}

extern "C" int ucb_verify_drafts(const ucb_verify_args* a, void* stream) {
  const char* what = "ucb_verify_drafts";
  if (!a) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (a->seqs < 0 || a->drafts_n < 0 || a->vocab < 1) return set_error(UCB_ERR_INVALID, "%s: bad shape", what);
  if (a->drafts_n >= uv::MAX_ROWS) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most %d drafts", what, uv::MAX_ROWS - 1);
  if (a->vocab > 1 << 30 || a->seqs > 65535) return set_error(UCB_ERR_UNSUPPORTED, "%s: too many sequences or tokens", what);
  if (!(a->temperature_all >= 0.f && a->temperature_all < 3.0e38f)) return set_error(UCB_ERR_INVALID, "%s: bad temperature", what);
  if (a->seqs == 0) return UCB_OK;
  if (!a->logits || (a->drafts_n && !a->drafts) || !a->uniforms || !a->tokens || !a->accepted || !a->logprobs || !a->workspace)
    return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return set_error(UCB_ERR_INVALID, "%s: workspace must be 16-byte aligned", what);
  if (a->draft_probs && a->probs_dtype != UCB_BF16 && a->probs_dtype != UCB_F16 && a->probs_dtype != UCB_F32)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: unsupported dtype", what);
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  uv::Layout layout;
  if (!layout.make(a->seqs, a->drafts_n + 1, a->vocab, a->dtype))
    return set_error(UCB_ERR_CUDA, "%s: the device's multiprocessors are unknown", what);
  char* w = static_cast<char*>(a->workspace);
  const uv::VerifyParams p{*a, reinterpret_cast<uv::Partial*>(w), reinterpret_cast<uv::Sums*>(w + layout.partials_bytes),
                           reinterpret_cast<uv::NearElement*>(w + layout.partials_bytes + layout.sums_bytes),
                           reinterpret_cast<unsigned int*>(w + layout.partials_bytes + layout.sums_bytes + layout.near_bytes),
                           (int)layout.splits, (int)layout.ctas, (int)layout.part_vectors, err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case UCB_BF16: return uv::launch_all<__nv_bfloat16>(p, s);
    case UCB_F16: return uv::launch_all<__half>(p, s);
    case UCB_F32: return uv::launch_all<float>(p, s);
    default: return set_error(UCB_ERR_UNSUPPORTED, "%s: unsupported dtype", what);
  }
}
