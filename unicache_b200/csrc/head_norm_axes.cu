// The head norm with rotation where a token has a position on each of several axes (time, height and
// width of image and video tokens) and each rotation pair turns by one of them (ucb_head_norm_rope_axes).  The same bytes as with
// one position a token.
#include <iterator>

#include "head_norm.cuh"

using ucb_host::set_error;

extern "C" int ucb_head_norm_rope_axes(const ucb_head_norm_args* a, const ucb_rope_axes* axes, void* stream) {
  const char* what = "ucb_head_norm_rope_axes";
  if (!axes) return set_error(UCB_ERR_INVALID, "%s: null pointer", what);
  if (axes->count < 1 || axes->count > 4) return set_error(UCB_ERR_UNSUPPORTED, "%s: 1 to 4 axes", what);
  if (a && a->rotary_dim == 0) return set_error(UCB_ERR_INVALID, "%s: no rotation to have axes", what);
  bool fours = true;
  for (int i = 0; a && i < std::min(a->rotary_dim, ucb::MAX_HEAD_DIM) / 2; ++i) {
    const int axis = axes->axis[i / 16] >> (2 * (i % 16)) & 3;
    if (axis >= axes->count) return set_error(UCB_ERR_INVALID, "%s: a pair's axis is not among the axes", what);
    fours &= axis == (int)(axes->axis[i / 16] >> (2 * (i % 16 / 4 * 4)) & 3);
  }
  ucb::HeadNormParams p;
  if (int rc = ucb::make_params(a, what, p)) return rc;
  if (a->tokens == 0) return UCB_OK;
  p.axes = axes->count;
  p.axis_stride = axes->position_stride;
  std::copy(std::begin(axes->axis), std::end(axes->axis), std::begin(p.axis));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return fours ? ucb::launch_type<ucb::ONE_AXIS>(p, a->dtype, what, s) : ucb::launch_type<ucb::ANY_AXIS>(p, a->dtype, what, s);
}
