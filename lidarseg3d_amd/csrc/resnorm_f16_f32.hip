// resnorm_f16_f32.hip — the residual-norm kernels (resnorm.h) of one pair of element types: x, y as ls3d_f16, residual and sum as float.
#include "resnorm.h"

bool ls3d_rn_launch_f16_f32(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream) {
  return ls3d_rn_launch_types<ls3d_f16, float>(fwd, full, nt, a, lpr, vpt, blocks, stream);
}
