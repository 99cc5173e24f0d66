// RMS norm of every query and key head and the rotary embedding of its
// position in one pass over the rows (ucb_head_norm_rope):
//   y = x * rsqrt(mean(x^2) + eps) * w,  (a, b) -> (a c - b s, b c + a s)
// in fp32 with one rounding.  Each row is read and written once: 16384 tokens x 32 heads x 128 move 277 MB.
#include <algorithm>

#include "common.cuh"

namespace ucb {
namespace {

struct HeadNormParams {
  const void *q, *k, *qw, *kw;
  void *qo, *ko;
  const float *cos, *sin;
  const void* pos;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;
  int64_t tokens, table_rows;
  int hq, hk, d, rot, interleaved, pos64;
  float eps;
  unsigned int* err;
};

constexpr int MAX_HEAD_DIM = 256;
constexpr int LANES_THREADS = 128;

__device__ __forceinline__ int64_t position_of(const HeadNormParams& p, int64_t t) {
  return p.pos64 ? static_cast<const int64_t*>(p.pos)[t] : (int64_t)static_cast<const int32_t*>(p.pos)[t];
}

// Any head_dim up to 256, any stride and alignment: one warp per row, the
// normalised row in shared memory for the exchange of the rotation pairs, element by element.  16384 tokens x 32 heads
// x 96 in bf16 take 253 us (0.8 TB/s), 32 tokens 3.9: a form for shapes that the lanes below do not take.
template <typename T>
__global__ void __launch_bounds__(256) head_norm_rows_kernel(const HeadNormParams p) {
  __shared__ float rows[8][MAX_HEAD_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.hq + p.hk;
  const int64_t row = (int64_t)blockIdx.x * 8 + warp;
  if (row >= p.tokens * heads) return;
  const int64_t t = row / heads;
  const int head = (int)(row % heads);
  const bool is_q = head < p.hq;
  const T* src = is_q ? static_cast<const T*>(p.q) + t * p.q_st + head * p.q_sh
                      : static_cast<const T*>(p.k) + t * p.k_st + (head - p.hq) * p.k_sh;
  T* dst = is_q ? static_cast<T*>(p.qo) + t * p.qo_st + head * p.qo_sh
                : static_cast<T*>(p.ko) + t * p.ko_st + (head - p.hq) * p.ko_sh;
  const T* w = static_cast<const T*>(is_q ? p.qw : p.kw);
  float* y = rows[warp];
  float ss = 0.f;
  for (int i = lane; i < p.d; i += 32) {
    const float v = Dtype<T>::to_f(src[i]);
    y[i] = v;
    ss = fmaf(v, v, ss);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float r = rsqrtf(ss / (float)p.d + p.eps);
  for (int i = lane; i < p.d; i += 32) y[i] = y[i] * r * (w ? Dtype<T>::to_f(w[i]) : 1.f);
  __syncwarp();
  int64_t pos = 0;
  bool bad = false;
  if (p.rot) {
    pos = position_of(p, t);
    bad = pos < 0 || pos >= p.table_rows;
    if (bad) {
      if (lane == 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
      pos = 0;
    }
  }
  const int half = p.rot / 2;
  for (int i = lane; i < p.d; i += 32) {
    float v = y[i];
    if (i < p.rot) {
      const int pair = p.interleaved ? i >> 1 : i % half;
      const bool second = p.interleaved ? (i & 1) : i >= half;
      const int partner = p.interleaved ? i ^ 1 : (second ? i - half : i + half);
      const float c = p.cos[pos * half + pair], s = p.sin[pos * half + pair];
      v = second ? fmaf(v, c, y[partner] * s) : fmaf(v, c, -y[partner] * s);
    }
    dst[i] = Dtype<T>::from_f(bad ? __int_as_float(0x7fffffff) : v);
  }
}

// Four adjacent elements, as loaded and as fp32.
template <typename T> struct Four {
  uint2 w;
  __device__ __forceinline__ void load(const T* src) { w = *reinterpret_cast<const uint2*>(src); }
  __device__ __forceinline__ void to(float* x) const {
    x[0] = Dtype<T>::lo(w.x), x[1] = Dtype<T>::hi(w.x), x[2] = Dtype<T>::lo(w.y), x[3] = Dtype<T>::hi(w.y);
  }
};
template <> struct Four<float> {
  float4 w;
  __device__ __forceinline__ void load(const float* src) { w = *reinterpret_cast<const float4*>(src); }
  __device__ __forceinline__ void to(float* x) const { x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w; }
};
template <typename T> __device__ __forceinline__ void store4(T* dst, const float* x) {
  if constexpr (sizeof(T) == 2) {
    const bool bf = Dtype<T>::code == UCB_BF16;
    *reinterpret_cast<uint2*>(dst) = make_uint2(bf ? pack_bf16x2(x[0], x[1]) : pack_f16x2(x[0], x[1]),
                                                bf ? pack_bf16x2(x[2], x[3]) : pack_f16x2(x[2], x[3]));
  } else {
    *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// head_dim 64, 128 or 256 with rows that start on four elements: L = head_dim / 8
// lanes a row.  A lane holds two runs of four channels that are each
// other's rotation partners (in the halves' form runs i and i + rotary_dim / 2), so
// that the rotation needs no exchange and the lane four angles, which the HEADS rows
// of one token that it has in flight share.  With STREAM a group of lanes goes from
// token to token, the next one's rows and angles in flight.  Measured for
// 16384 tokens x 32 heads x 128 (277 MB): 53 us (5.2 TB/s) with STREAM, one token
// a group 57; 2 rows a lane 75, 1 row 85, 8 rows 84; blocks of 256 threads 59.  Neither memory nor issue slots (61%) are used
// up there: 16 warps a multiprocessor, all that 128 registers leave, wait for their loads.  In fp32 (537 MB) 93 us, 5.8 TB/s.
template <typename T, int L, int HEADS, bool PAIRS, bool STREAM>
__global__ void __launch_bounds__(LANES_THREADS, 1)
    head_norm_lanes_kernel(const HeadNormParams p, uint32_t q_units, uint32_t units, uint32_t token_step) {
  const uint32_t group = (blockIdx.x * (uint32_t)LANES_THREADS + threadIdx.x) / L;
  const int lane = threadIdx.x % L;
  const uint32_t t0 = group / units, u = group - t0 * units;
  const bool is_q = u < q_units;
  const int half = p.rot / 2;
  const bool turned = lane * (PAIRS ? 8 : 4) < (PAIRS ? p.rot : half);
  const int rest = p.rot + 8 * (lane - half / 4);  // channels that are only normalised
  const int d0 = PAIRS ? 8 * lane : turned ? 4 * lane : rest, d1 = PAIRS || !turned ? d0 + 4 : d0 + half;
  const int head0 = (is_q ? u : u - q_units) * HEADS;
  const int rows = t0 < token_step ? (is_q ? p.hq : p.hk) - head0 : 0;  // of this group; 0 past the last group
  const int64_t sh = is_q ? p.q_sh : p.k_sh, oh = is_q ? p.qo_sh : p.ko_sh;
  const int64_t st = is_q ? p.q_st : p.k_st, ot = is_q ? p.qo_st : p.ko_st;
  const T* src = static_cast<const T*>(is_q ? p.q : p.k) + head0 * sh;
  T* dst = static_cast<T*>(is_q ? p.qo : p.ko) + head0 * oh;
  Four<T> w[2];
  const T* weight = static_cast<const T*>(is_q ? p.qw : p.kw);
  if (weight) w[0].load(weight + d0), w[1].load(weight + d1);

  struct Ahead {
    Four<T> raw[HEADS][2];
    float4 c, s;
    bool bad;
  };
  auto position = [&](uint32_t t) { return p.rot && t < p.tokens ? position_of(p, t) : 0; };
  auto fetch = [&](uint32_t t, int64_t pos) {
    Ahead a;
    a.bad = false;
    if (t >= p.tokens) return a;
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      if (i < rows) {
        a.raw[i][0].load(src + t * st + i * sh + d0);
        a.raw[i][1].load(src + t * st + i * sh + d1);
      }
    a.bad = p.rot && (pos < 0 || pos >= p.table_rows);
    if (turned) {
      const int64_t at = (a.bad ? 0 : pos) * half + 4 * lane;
      a.c = *reinterpret_cast<const float4*>(p.cos + at);
      a.s = *reinterpret_cast<const float4*>(p.sin + at);
    }
    return a;
  };
  uint32_t t = t0;
  Ahead next = fetch(t, position(t));
  int64_t pos = STREAM ? position(t + token_step) : 0;
#pragma unroll 1
  while (t < p.tokens) {
    const Ahead now = next;
    if (STREAM) {
      next = fetch(t + token_step, pos);
      pos = position(t + 2 * token_step);
    }
    if (now.bad && lane == 0 && rows > 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    const float c[4] = {now.c.x, now.c.y, now.c.z, now.c.w}, s[4] = {now.s.x, now.s.y, now.s.z, now.s.w};
    float wf[8];
    if (weight) w[0].to(wf), w[1].to(wf + 4);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      float x[8], ss = 0.f;
      now.raw[i][0].to(x);
      now.raw[i][1].to(x + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, L);
      const float r = now.bad ? __int_as_float(0x7fffffff) : rsqrtf(ss * (1.f / (8 * L)) + p.eps);
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = weight ? x[k] * r * wf[k] : x[k] * r;
      if (turned) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int first = PAIRS ? 2 * k : k, other = PAIRS ? 2 * k + 1 : k + 4;
          const float a = x[first], b = x[other];
          x[first] = fmaf(a, c[k], -b * s[k]);
          x[other] = fmaf(b, c[k], a * s[k]);
        }
      }
      if (i < rows) {
        store4(dst + t * ot + i * oh + d0, x);
        store4(dst + t * ot + i * oh + d1, x + 4);
      }
    }
    if (!STREAM) break;
    t += token_step;
  }
}

// Whether every row of one side starts on four elements.
template <typename T> bool aligned(const void* x, int64_t st, int64_t sh) {
  return reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0 && st % 4 == 0 && sh % 4 == 0;
}

template <typename T, int L, int HEADS, bool STREAM> int launch_lanes(const HeadNormParams& p, cudaStream_t s) {
  const uint32_t q_units = (p.hq + HEADS - 1) / HEADS, units = q_units + (p.hk + HEADS - 1) / HEADS;
  const auto kernel = p.interleaved ? head_norm_lanes_kernel<T, L, HEADS, true, STREAM>
                                    : head_norm_lanes_kernel<T, L, HEADS, false, STREAM>;
  uint32_t step = (uint32_t)p.tokens;  // tokens that are worked on at once
  if (STREAM) {  // as many as are resident, in equal turns
    static int resident[64][2] = {{0}};  // CTAs on a multiprocessor, by device
    int dev = 0;
    cudaGetDevice(&dev);
    int& ctas = resident[dev & 63][p.interleaved != 0];
    if (ctas == 0 && cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, LANES_THREADS, 0) != cudaSuccess)
      return ucb_host::check_launch("head_norm_lanes_kernel");
    const int64_t most = std::max<int64_t>(1, (int64_t)ctas * ucb_host::multiprocessors() * (LANES_THREADS / L) / units);
    const int64_t turns = (p.tokens + most - 1) / most;
    step = (uint32_t)((p.tokens + turns - 1) / turns);
  }
  const unsigned blocks = (unsigned)(((int64_t)step * units * L + LANES_THREADS - 1) / LANES_THREADS);
  kernel<<<blocks, LANES_THREADS, 0, s>>>(p, q_units, units, step);
  return ucb_host::check_launch("head_norm_lanes_kernel");
}

template <typename T, int L> int launch_heads(const HeadNormParams& p, cudaStream_t s) {
  // Four rows a lane once one row a lane would fill the chip's threads (4999 tokens x 18 heads x 64: 5.6 us against
  // 8.0 with one row; below that, one row has the shorter way); from token to token once that makes several turns
  // (where it makes two or three, 6.6 us for the same case).
  const int64_t lanes = p.tokens * (p.hq + p.hk) * L, threads = (int64_t)ucb_host::multiprocessors() * 2048;
  if (lanes >= threads * 8) return launch_lanes<T, L, 4, true>(p, s);
  if (lanes >= threads) return launch_lanes<T, L, 4, false>(p, s);
  return launch_lanes<T, L, 1, false>(p, s);
}

template <typename T> int launch(const HeadNormParams& p, cudaStream_t s) {
  const bool tables = reinterpret_cast<uintptr_t>(p.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sin) % 16 == 0;
  const bool rows = (!p.hq || (aligned<T>(p.q, p.q_st, p.q_sh) && aligned<T>(p.qo, p.qo_st, p.qo_sh))) &&
                    (!p.hk || (aligned<T>(p.k, p.k_st, p.k_sh) && aligned<T>(p.ko, p.ko_st, p.ko_sh))) &&
                    (reinterpret_cast<uintptr_t>(p.qw) | reinterpret_cast<uintptr_t>(p.kw)) % (4 * sizeof(T)) == 0;
  // the lanes' 32-bit indexes hold tokens * heads * 32
  if (rows && tables && p.rot % 8 == 0 && p.tokens <= 0x3ffffff / (p.hq + p.hk)) {
    if (p.d == 128) return launch_heads<T, 16>(p, s);
    if (p.d == 64) return launch_heads<T, 8>(p, s);
    if (p.d == 256) return launch_heads<T, 32>(p, s);
  }
  const int64_t blocks = (p.tokens * (p.hq + p.hk) + 7) / 8;
  if (blocks > 0x7fffffff) return ucb_host::set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: too many rows");
  head_norm_rows_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(p);
  return ucb_host::check_launch("head_norm_rows_kernel");
}

}  // namespace
}  // namespace ucb

using ucb_host::set_error;

extern "C" int ucb_head_norm_rope(const ucb_head_norm_args* a, void* stream) {
  if (!a) return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: null pointer");
  if (a->tokens < 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads + (int64_t)a->k_heads == 0)
    return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: bad shape");
  if (a->q_heads + (int64_t)a->k_heads > 65535)
    return set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: at most 65535 heads");
  if (a->head_dim < 2 || a->head_dim > ucb::MAX_HEAD_DIM)
    return set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: head_dim must be 2..%d", ucb::MAX_HEAD_DIM);
  if (a->rotary_dim < 0 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
    return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: rotary_dim must be even and at most head_dim");
  if (a->tokens == 0) return UCB_OK;
  if ((a->q_heads && (!a->query || !a->q_out)) || (a->k_heads && (!a->key || !a->k_out)) ||
      (a->rotary_dim && (!a->cos || !a->sin || !a->positions)))
    return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: null pointer");
  if (a->rotary_dim && a->table_rows < 1) return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: empty tables");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_head_norm_rope: device error word unavailable");
  const ucb::HeadNormParams p{a->query, a->key, a->q_weight, a->k_weight, a->q_out, a->k_out, a->cos, a->sin, a->positions,
                              a->q_stride_token, a->q_stride_head, a->k_stride_token, a->k_stride_head,
                              a->qo_stride_token, a->qo_stride_head, a->ko_stride_token, a->ko_stride_head,
                              a->tokens, a->table_rows, a->q_heads, a->k_heads, a->head_dim, a->rotary_dim,
                              a->interleaved, a->positions_64, a->eps, err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case UCB_BF16: return ucb::launch<__nv_bfloat16>(p, s);
    case UCB_F16: return ucb::launch<__half>(p, s);
    case UCB_F32: return ucb::launch<float>(p, s);
    default: return set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: unsupported dtype");
  }
}
