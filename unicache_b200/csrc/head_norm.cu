// RMS norm of every query and key head and the rotary embedding of its
// position in one pass over the rows (ucb_head_norm_rope):
//   y = x * rsqrt(mean(x^2) + eps) * w,  (a, b) -> (a c - b s, b c + a s)
// in fp32 with one rounding.  Each row is read and written once: 16384 tokens x 32 heads x 128 move 277 MB.
#include "head_norm.cuh"

extern "C" int ucb_head_norm_rope(const ucb_head_norm_args* a, void* stream) {
  const char* what = "ucb_head_norm_rope";
  ucb::HeadNormParams p;
  if (int rc = ucb::make_params(a, what, p)) return rc;
  if (a->tokens == 0) return UCB_OK;
  return ucb::launch_type<ucb::NO_AXES>(p, a->dtype, what, static_cast<cudaStream_t>(stream));
}
