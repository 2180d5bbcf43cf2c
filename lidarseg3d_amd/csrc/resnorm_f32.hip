// resnorm_f32.hip — the residual-norm kernels (resnorm.h) of one pair of element types: x, y as float, residual and sum as float.
#include "resnorm.h"

bool ls3d_rn_launch_f32(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream) {
  return ls3d_rn_launch_types<float, float>(fwd, full, nt, a, lpr, vpt, blocks, stream);
}
