// Shared pieces of the 8-bit block cache kernels (ucb_block8_*).
#pragma once

#include "common.cuh"

namespace ucb {
namespace block8 {

constexpr float LEAST_SCALE = 7.52316384526264e-37f;  // 2^-120: 1 / scale stays finite, blocks of zeros have codes 0

// A block's scale from the largest magnitude of its values.  NaN stays NaN.
__device__ __forceinline__ float scale_of(float amax) {
  const float s = __fdiv_rn(amax, 127.f);
  return s < LEAST_SCALE ? LEAST_SCALE : s;
}

// clamp(rint(x * inverse)): the products that are not numbers (a NaN or infinite
// input, whose scale is NaN or infinite) become 0, as __float2int_rn gives.
__device__ __forceinline__ int code_of(float x, float inverse) {
  const int c = __float2int_rn(__fmul_rn(x, inverse));
  return max(-127, min(127, c));
}

// Pool block of a sequence's j-th block, -1 (and the error bit) when the table
// names none.
__device__ __forceinline__ int64_t pool_block(const ucb_block8_cache& c, int s, int j, unsigned int* err) {
  const int b = c.block_table[(int64_t)s * c.max_blocks + j];
  if (b < 0 || b >= c.num_blocks) {
    atomicOr(err, DEVERR_BAD_DESCRIPTOR);
    return -1;
  }
  return b;
}

// Tokens of a sequence, limited to what its table row can hold.
__device__ __forceinline__ int held_tokens(const ucb_block8_cache& c, int s, unsigned int* err) {
  const int n = c.lengths[s];
  const int64_t most = (int64_t)c.max_blocks * c.block_tokens;
  if (n >= 0 && n <= most) return n;
  atomicOr(err, DEVERR_BAD_DESCRIPTOR);
  return n < 0 ? 0 : (int)most;
}

// Programmatic dependent launch: a kernel launched as `dependent` may become resident once every CTA of the kernel before
// it in its stream has called launch_dependents (or ended).  It calls wait_for_primary before its first access to global
// memory, which returns when that kernel is complete and its writes are visible.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_primary() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename P>
int launch(void (*kernel)(const P), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const P& params,
           const char* what, int cluster = 1, bool dependent = false) {
  cudaLaunchAttribute attribute[2];
  int attributes = 0;
  if (dependent) {
    attribute[attributes].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[attributes++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attribute[attributes].id = cudaLaunchAttributeClusterDimension;
    attribute[attributes].val.clusterDim.x = cluster;
    attribute[attributes].val.clusterDim.y = attribute[attributes].val.clusterDim.z = 1;
    ++attributes;
  }
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = attribute;
  config.numAttrs = attributes;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, params);
  if (e != cudaSuccess) return ucb_host::set_error(UCB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return UCB_OK;
}

// Checks that every entry point makes before it touches the GPU.
int check_cache(const ucb_block8_cache* c, const char* what);

}  // namespace block8
}  // namespace ucb
