#include "block_norm_launch.h"

int fssim_host::block_norm_f32_f16(bool backward, const BlockLaunch& l, const fssim::BlockParams& p, cudaStream_t stream) {
  return block_norm_types<float, __half>(backward, l, p, stream);
}
