#include "block_norm_launch.h"

int fssim_host::block_norm_bf16(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  return block_norm_types<__nv_bfloat16, __nv_bfloat16>(backward, l, p, stream);
}
