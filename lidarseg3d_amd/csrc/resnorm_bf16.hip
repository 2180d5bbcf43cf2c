// resnorm_bf16.hip — the residual-norm kernels (resnorm.h) of one pair of element types: x, y as ls3d_bf16, residual and sum as ls3d_bf16.
#include "resnorm.h"

bool ls3d_rn_launch_bf16(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream) {
  return ls3d_rn_launch_types<ls3d_bf16, ls3d_bf16>(fwd, full, nt, a, lpr, vpt, blocks, stream);
}
