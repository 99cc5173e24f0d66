// RMS norm of every query and key head and the rotary embedding of its
// position in one pass over the rows (ucb_head_norm_rope).
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

__device__ __forceinline__ int64_t position_of(const HeadNormParams& p, int64_t t) {
  return p.pos64 ? static_cast<const int64_t*>(p.pos)[t] : (int64_t)static_cast<const int32_t*>(p.pos)[t];
}

// Any head_dim up to 256, any stride and alignment: one warp per row, the
// normalised row in shared memory for the exchange of the rotation pairs.
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

template <typename T> int launch(const HeadNormParams& p, cudaStream_t s) {
  const int64_t blocks = (p.tokens * (p.hq + p.hk) + 7) / 8;
  if (blocks > 0x7fffffff) return ucb_host::set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: too many rows");
  head_norm_rows_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(p);
  return ucb_host::check_launch("head_norm_rows_kernel");
}

}  // namespace
}  // namespace ucb

using ucb_host::set_error;

extern "C" int ucb_head_norm_rope(const void* q, int64_t q_st, int64_t q_sh, int hq, const void* k, int64_t k_st,
                                  int64_t k_sh, int hk, const void* qw, const void* kw, const float* cos_t,
                                  const float* sin_t, const void* positions, int positions_64, int64_t table_rows,
                                  int64_t tokens, int head_dim, int rotary_dim, int interleaved, int dtype, float eps,
                                  void* qo, int64_t qo_st, int64_t qo_sh, void* ko, int64_t ko_st, int64_t ko_sh,
                                  void* stream) {
  if (tokens < 0 || hq < 0 || hk < 0 || hq + hk == 0)
    return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: bad shape");
  if (head_dim < 2 || head_dim > ucb::MAX_HEAD_DIM)
    return set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: head_dim must be 2..%d", ucb::MAX_HEAD_DIM);
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: rotary_dim must be even and at most head_dim");
  if (tokens == 0) return UCB_OK;
  if ((hq && (!q || !qo)) || (hk && (!k || !ko)) || (rotary_dim && (!cos_t || !sin_t || !positions)))
    return set_error(UCB_ERR_INVALID, "ucb_head_norm_rope: null pointer");
  unsigned int* err = ucb_host::device_error_word();
  if (!err) return set_error(UCB_ERR_CUDA, "ucb_head_norm_rope: device error word unavailable");
  const ucb::HeadNormParams p{q,     k,     qw,    kw,    qo,    ko,         cos_t, sin_t, positions,  q_st,        q_sh,         k_st, k_sh,
                              qo_st, qo_sh, ko_st, ko_sh, tokens, table_rows, hq,    hk,    head_dim, rotary_dim, interleaved, positions_64, eps,  err};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case UCB_BF16: return ucb::launch<__nv_bfloat16>(p, s);
    case UCB_F16: return ucb::launch<__half>(p, s);
    case UCB_F32: return ucb::launch<float>(p, s);
    default: return set_error(UCB_ERR_UNSUPPORTED, "ucb_head_norm_rope: unsupported dtype");
  }
}
