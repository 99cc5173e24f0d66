// RMS norm of query and key heads with the rotation of their positions: the kernels, whose entry points are in head_norm.cu (one
// position a token) and head_norm_axes.cu (a position of each axis).
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace ucb {
namespace {

constexpr int MAX_HEAD_DIM = 256;

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
  // with several axes: their number (0: one position a token), the axis of rotation pair i in bits 2 (i % 16) of word i / 16,
  // and the distance of two axes' positions
  int axes;
  uint32_t axis[MAX_HEAD_DIM / 32];
  int64_t axis_stride;
};

constexpr int LANES_THREADS = 128;

__device__ __forceinline__ int axis_of(const HeadNormParams& p, int pair) { return p.axis[pair >> 4] >> (2 * (pair & 15)) & 3; }

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
  if (p.axes) {  // a lane an axis: those that no pair turns by are not looked at
    if (lane < p.axes) pos = position_of(p, t + lane * p.axis_stride);
    unsigned used = 0;
    for (int i = lane; i < p.rot / 2; i += 32) used |= 1u << axis_of(p, i);
    used = __reduce_or_sync(0xffffffffu, used);
    bad = __any_sync(0xffffffffu, lane < p.axes && (used >> lane & 1) && (pos < 0 || pos >= p.table_rows));
  } else if (p.rot) {
    pos = position_of(p, t);
    bad = pos < 0 || pos >= p.table_rows;
  }
  if (bad) {
    if (lane == 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    pos = 0;
  }
  const int half = p.rot / 2;
  for (int i0 = 0; i0 < p.d; i0 += 32) {
    const int i = i0 + lane, pair = i >= p.rot ? 0 : p.interleaved ? i >> 1 : i % half;
    const int64_t at = p.axes ? __shfl_sync(0xffffffffu, pos, axis_of(p, pair)) : pos;
    if (i >= p.d) continue;
    float v = y[i];
    if (i < p.rot) {
      const bool second = p.interleaved ? (i & 1) : i >= half;
      const int partner = p.interleaved ? i ^ 1 : (second ? i - half : i + half);
      const float c = p.cos[at * half + pair], s = p.sin[at * half + pair];
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
// 16384 tokens x 32 heads x 128 (277 MB): 47 us (5.9 TB/s) with STREAM; while positions were waited for where they are loaded 53, one
// token a group 57, 2 rows a lane 75, 1 row 85, 8 rows 84, blocks of 256 threads 59.  Neither memory nor issue slots are used
// up there: 16 warps a multiprocessor, all that 128 registers leave, wait for their loads.
// AXES: each pair's angle is that of its own axis' position.  ONE_AXIS: a lane's four pairs share an axis, as sections
// of whole fours have it, so that only the address of its position differs (47 us too); ANY_AXIS: four positions and eight single
// loads of angles a lane (52; with the registers of three CTAs a multiprocessor 65).
enum Axes { NO_AXES, ONE_AXIS, ANY_AXIS };
template <typename T, int L, int HEADS, bool PAIRS, bool STREAM, Axes AXES>
__global__ void __launch_bounds__(LANES_THREADS, AXES == ANY_AXIS && sizeof(T) == 2 ? 4 : 1)
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
  // A token's positions as they are loaded, two tokens ahead: nothing may be computed from them before they are needed, or the
  // lane waits for them there (32-bit positions that were extended at once cost 16384 tokens x 32 heads x 128 5 us).
  struct Raw {
    uint32_t low;
    int32_t high;  // of 64 bits
  };
  struct Rows {  // with axes those of the lane's pairs; of 64 bits that are no row of the tables -1
    int of[4];
  };
  using Pos = std::conditional_t<AXES == NO_AXES, Raw, std::conditional_t<AXES == ONE_AXIS, int, Rows>>;
  auto raw_of = [&](int64_t i) {
    Raw r{0, 0};
    if (p.pos64) {
      const uint2 v = static_cast<const uint2*>(p.pos)[i];
      r.low = v.x, r.high = (int32_t)v.y;
    } else {
      r.low = static_cast<const uint32_t*>(p.pos)[i];
    }
    return r;
  };
  auto row_of = [&](uint32_t t, int pair) {
    const int64_t i = t + axis_of(p, pair) * p.axis_stride;
    if (!p.pos64) return static_cast<const int32_t*>(p.pos)[i];
    const int64_t pos = static_cast<const int64_t*>(p.pos)[i];
    return pos < 0 || pos >= p.table_rows ? -1 : (int)pos;
  };
  auto position = [&](uint32_t t) {
    if constexpr (AXES == NO_AXES) {
      return p.rot && t < p.tokens ? raw_of(t) : Raw{0, 0};
    } else if constexpr (AXES == ONE_AXIS) {
      return turned && t < p.tokens ? row_of(t, 4 * lane) : 0;
    } else {
      Rows r{{0, 0, 0, 0}};
      if (turned && t < p.tokens)
#pragma unroll
        for (int k = 0; k < 4; ++k) r.of[k] = row_of(t, 4 * lane + k);
      return r;
    }
  };
  auto fetch = [&](uint32_t t, Pos pos) {
    Ahead a;
    a.bad = false;
    if (t >= p.tokens) return a;
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
      if (i < rows) {
        a.raw[i][0].load(src + t * st + i * sh + d0);
        a.raw[i][1].load(src + t * st + i * sh + d1);
      }
    if constexpr (AXES == ANY_AXIS) {
      a.bad = false;
      if (turned) {
        float c[4], s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool inside = pos.of[k] >= 0 && pos.of[k] < p.table_rows;
          const int64_t at = (int64_t)(inside ? pos.of[k] : 0) * half + 4 * lane + k;
          a.bad |= !inside;
          c[k] = p.cos[at], s[k] = p.sin[at];
        }
        a.c = make_float4(c[0], c[1], c[2], c[3]), a.s = make_float4(s[0], s[1], s[2], s[3]);
      }
    } else {
      int64_t row;
      if constexpr (AXES == NO_AXES) row = p.pos64 ? (int64_t)pos.high << 32 | pos.low : (int64_t)(int32_t)pos.low;
      else row = pos;
      a.bad = p.rot && (row < 0 || row >= p.table_rows);
      if (turned) {
        const int64_t at = (a.bad ? 0 : row) * half + 4 * lane;
        a.c = *reinterpret_cast<const float4*>(p.cos + at);
        a.s = *reinterpret_cast<const float4*>(p.sin + at);
      }
    }
    return a;
  };
  uint32_t t = t0;
  Ahead next = fetch(t, position(t));
  Pos pos{};
  if (STREAM) pos = position(t + token_step);
#pragma unroll 1
  while (t < p.tokens) {
    const Ahead now = next;
    if (STREAM) {
      next = fetch(t + token_step, pos);
      pos = position(t + 2 * token_step);
    }
    if (now.bad && (AXES != NO_AXES || lane == 0) && rows > 0) atomicOr(p.err, DEVERR_BAD_DESCRIPTOR);
    const float c[4] = {now.c.x, now.c.y, now.c.z, now.c.w}, s[4] = {now.s.x, now.s.y, now.s.z, now.s.w};
    float wf[8];
    if (weight) w[0].to(wf), w[1].to(wf + 4);
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      // a position of any lane's that is outside the tables reaches the row's other lanes through the sum of squares
      float x[8], ss = AXES != NO_AXES && now.bad ? __int_as_float(0x7fffffff) : 0.f;
      now.raw[i][0].to(x);
      now.raw[i][1].to(x + 4);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(x[k], x[k], ss);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, L);
      const float r = AXES == NO_AXES && now.bad ? __int_as_float(0x7fffffff) : rsqrtf(ss * (1.f / (8 * L)) + p.eps);
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

template <typename T, int L, int HEADS, bool STREAM, Axes AXES> int launch_lanes(const HeadNormParams& p, cudaStream_t s) {
  const uint32_t q_units = (p.hq + HEADS - 1) / HEADS, units = q_units + (p.hk + HEADS - 1) / HEADS;
  const auto kernel = p.interleaved ? head_norm_lanes_kernel<T, L, HEADS, true, STREAM, AXES>
                                    : head_norm_lanes_kernel<T, L, HEADS, false, STREAM, AXES>;
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

template <typename T, int L, Axes AXES> int launch_heads(const HeadNormParams& p, cudaStream_t s) {
  // Four rows a lane once one row a lane would fill the chip's threads (4999 tokens x 18 heads x 64: 5.6 us against
  // 8.0 with one row; below that, one row has the shorter way); from token to token once that makes several turns
  // (where it makes two or three, 6.6 us for the same case).
  const int64_t lanes = p.tokens * (p.hq + p.hk) * L, threads = (int64_t)ucb_host::multiprocessors() * 2048;
  if (lanes >= threads * 8) return launch_lanes<T, L, 4, true, AXES>(p, s);
  if (lanes >= threads) return launch_lanes<T, L, 4, false, AXES>(p, s);
  return launch_lanes<T, L, 1, false, AXES>(p, s);
}

template <typename T, Axes AXES> int launch(const HeadNormParams& p, cudaStream_t s) {
  const bool tables = reinterpret_cast<uintptr_t>(p.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sin) % 16 == 0;
  const bool rows = (!p.hq || (aligned<T>(p.q, p.q_st, p.q_sh) && aligned<T>(p.qo, p.qo_st, p.qo_sh))) &&
                    (!p.hk || (aligned<T>(p.k, p.k_st, p.k_sh) && aligned<T>(p.ko, p.ko_st, p.ko_sh))) &&
                    (reinterpret_cast<uintptr_t>(p.qw) | reinterpret_cast<uintptr_t>(p.kw)) % (4 * sizeof(T)) == 0;
  // the lanes' 32-bit indexes hold tokens * heads * 32, and their rows of several axes the tables'
  if ((AXES == NO_AXES || p.table_rows <= 0x7fffffff) && rows && tables && p.rot % 8 == 0 && p.tokens <= 0x3ffffff / (p.hq + p.hk)) {
    if (p.d == 128) return launch_heads<T, 16, AXES>(p, s);
    if (p.d == 64) return launch_heads<T, 8, AXES>(p, s);
    if (p.d == 256) return launch_heads<T, 32, AXES>(p, s);
  }
  const int64_t blocks = (p.tokens * (p.hq + p.hk) + 7) / 8;
  if (blocks > 0x7fffffff) return ucb_host::set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: too many rows");
  head_norm_rows_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(p);
  return ucb_host::check_launch("head_norm_rows_kernel");
}

// Checks a call and fills its parameters; a->tokens may be 0.
int make_params(const ucb_head_norm_args* a, const char* what, HeadNormParams& p) {
  using ucb_host::set_error;
  if (!a) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (a->tokens < 0 || a->q_heads < 0 || a->k_heads < 0 || a->q_heads + (int64_t)a->k_heads == 0)
    return set_error(UCB_ERR_INVALID, "%s: bad shape", what);
  if (a->q_heads + (int64_t)a->k_heads > 65535) return set_error(UCB_ERR_UNSUPPORTED, "%s: at most 65535 heads", what);
  if (a->head_dim < 2 || a->head_dim > MAX_HEAD_DIM)
    return set_error(UCB_ERR_UNSUPPORTED, "%s: head_dim must be 2..%d", what, MAX_HEAD_DIM);
  if (a->rotary_dim < 0 || a->rotary_dim % 2 || a->rotary_dim > a->head_dim)
    return set_error(UCB_ERR_INVALID, "%s: rotary_dim must be even and at most head_dim", what);
  if (a->tokens == 0) return UCB_OK;
  if ((a->q_heads && (!a->query || !a->q_out)) || (a->k_heads && (!a->key || !a->k_out)) ||
      (a->rotary_dim && (!a->cos || !a->sin || !a->positions)))
    return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (a->rotary_dim && a->table_rows < 1) return set_error(UCB_ERR_INVALID, "%s: empty tables", what);
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "%s: device error word unavailable", what);
  p = HeadNormParams{a->query, a->key, a->q_weight, a->k_weight, a->q_out, a->k_out, a->cos, a->sin, a->positions,
                     a->q_stride_token, a->q_stride_head, a->k_stride_token, a->k_stride_head,
                     a->qo_stride_token, a->qo_stride_head, a->ko_stride_token, a->ko_stride_head,
                     a->tokens, a->table_rows, a->q_heads, a->k_heads, a->head_dim, a->rotary_dim,
                     a->interleaved, a->positions_64, a->eps, err};
  return UCB_OK;
}

template <Axes AXES> int launch_type(const HeadNormParams& p, int dtype, const char* what, cudaStream_t s) {
  switch (dtype) {
    case UCB_BF16: return launch<__nv_bfloat16, AXES>(p, s);
    case UCB_F16: return launch<__half, AXES>(p, s);
    case UCB_F32: return launch<float, AXES>(p, s);
    default: return ucb_host::set_error(UCB_ERR_UNSUPPORTED, "%s: unsupported dtype", what);
  }
}

}  // namespace
}  // namespace ucb
