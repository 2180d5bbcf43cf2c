// dropout.hip — dropout whose mask comes from a counter-based generator (blocks_common.h) and is never stored.
//
//   forward   y = keep ? act(x) / (1 - p) : 0        act: identity or ReLU
//   backward  dx = keep ? dy / (1 - p) : 0           (ReLU: where y != 0, which says both that x was positive and that it was kept: no generator)
//
// A dropped element is zero whatever stands in its place (a select, no product: Inf and NaN behind the mask do not get through).  Bound by memory:
// a pass reads one tensor and writes one.
#include "blocks_common.h"

// one chunk of 8 columns per thread and trip; index type 32 bits where the chunk count allows (the division by the row's chunk count)
template <typename T, typename I, bool RELU>
__global__ __launch_bounds__(256) void k_dropout_fwd(const T *__restrict__ x, size_t x_ld, I total, uint32_t groups, long long c, uint32_t thr, float inv,
                                                     const int64_t *__restrict__ state, uint32_t call, T *__restrict__ y) {
  const ls3d_dropout_key key = ls3d_dropout_key_load(state, call);
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / groups), g = (uint32_t)(t - (I)row * groups);
    const long long col = (long long)g * 8;
    const int m = c - col < 8 ? (int)(c - col) : 8;
    float v[8];
    ls3d_unpack8<T>(ls3d_load8<T>(x + (size_t)row * x_ld, col, c), m, v);
    const uint32_t keep = ls3d_keep8(key, g, row, thr);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ((keep >> j) & 1u) && !(RELU && v[j] <= 0.0f) ? v[j] * inv : 0.0f;
    ls3d_store8<T>(y + (size_t)row * c + col, v, m);
  }
}

template <typename T, typename I, bool RELU>
__global__ __launch_bounds__(256) void k_dropout_bwd(const T *__restrict__ dy, size_t dy_ld, const T *__restrict__ y, I total, uint32_t groups, long long c,
                                                     uint32_t thr, float inv, const int64_t *__restrict__ state, uint32_t call, T *__restrict__ dx) {
  const ls3d_dropout_key key = RELU ? ls3d_dropout_key{} : ls3d_dropout_key_load(state, call);
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / groups), g = (uint32_t)(t - (I)row * groups);
    const long long col = (long long)g * 8;
    const int m = c - col < 8 ? (int)(c - col) : 8;
    float v[8];
    ls3d_unpack8<T>(ls3d_load8<T>(dy + (size_t)row * dy_ld, col, c), m, v);
    if (RELU) {
      float o[8];
      ls3d_unpack8<T>(ls3d_load8<T>(y + (size_t)row * c, col, c), m, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = !(o[j] <= 0.0f) ? v[j] * inv : 0.0f;
    } else {
      const uint32_t keep = ls3d_keep8(key, g, row, thr);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = ((keep >> j) & 1u) ? v[j] * inv : 0.0f;
    }
    ls3d_store8<T>(dx + (size_t)row * c + col, v, m);
  }
}

template <typename T, bool RELU>
static void dropout_launch(bool fwd, const void *a, size_t ld, const void *y_in, long long rows, long long c, uint32_t thr, float inv, const int64_t *state,
                           uint32_t call, void *out, hipStream_t stream) {
  const uint32_t groups = (uint32_t)((c + 7) / 8);
  const long long total = rows * (long long)groups;
  const dim3 grid = ls3d_grid(total);
  if (total < (1ll << 31)) {
    if (fwd) hipLaunchKernelGGL((k_dropout_fwd<T, uint32_t, RELU>), grid, dim3(256), 0, stream, (const T *)a, ld, (uint32_t)total, groups, c, thr, inv, state, call, (T *)out);
    else hipLaunchKernelGGL((k_dropout_bwd<T, uint32_t, RELU>), grid, dim3(256), 0, stream, (const T *)a, ld, (const T *)y_in, (uint32_t)total, groups, c, thr, inv, state, call, (T *)out);
  } else {
    if (fwd) hipLaunchKernelGGL((k_dropout_fwd<T, unsigned long long, RELU>), grid, dim3(256), 0, stream, (const T *)a, ld, (unsigned long long)total, groups, c, thr, inv, state, call, (T *)out);
    else hipLaunchKernelGGL((k_dropout_bwd<T, unsigned long long, RELU>), grid, dim3(256), 0, stream, (const T *)a, ld, (const T *)y_in, (unsigned long long)total, groups, c, thr, inv, state, call, (T *)out);
  }
}

static int dropout_run(bool fwd, const void *a, long long ld, const void *y_in, long long rows, long long c, int dtype, float p, const int64_t *state,
                       uint32_t call, int relu, void *out, hipStream_t stream) {
  uint32_t thr;
  float inv;
  if (rows < 0 || c < 0 || rows > 0x7FFFFFFFll || c > 0x7FFFFFFFll || !ls3d_dtype_ok(dtype) || !ls3d_dropout_threshold(p, &thr, &inv)) return LS3D_ERR_ARG;
  if (rows == 0 || c == 0) return LS3D_OK;
  if (!a || !out || ld < c || !state || ((uintptr_t)state & 7) || (!fwd && relu && !y_in)) return LS3D_ERR_ARG;
  if (((uintptr_t)a | (uintptr_t)out | (uintptr_t)y_in) & (ls3d_dtype_size(dtype) - 1)) return LS3D_ERR_ARG;
#define DROPOUT_GO(T)                                                                                                             \
  do {                                                                                                                            \
    if (relu) dropout_launch<T, true>(fwd, a, (size_t)ld, y_in, rows, c, thr, inv, state, call, out, stream);                     \
    else dropout_launch<T, false>(fwd, a, (size_t)ld, y_in, rows, c, thr, inv, state, call, out, stream);                         \
  } while (0)
  if (dtype == LS3D_DTYPE_F32) DROPOUT_GO(float);
  else if (dtype == LS3D_DTYPE_BF16) DROPOUT_GO(ls3d_bf16);
  else DROPOUT_GO(ls3d_f16);
#undef DROPOUT_GO
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}

extern "C" int ls3d_dropout_forward(const void *x, long long x_ld, long long rows, long long c, int dtype, float p, const int64_t *state, uint32_t call,
                                    int relu, void *y, ls3d_stream_t stream) {
  return dropout_run(true, x, x_ld, nullptr, rows, c, dtype, p, state, call, relu, y, (hipStream_t)stream);
}

extern "C" int ls3d_dropout_backward(const void *dy, long long dy_ld, const void *y, long long rows, long long c, int dtype, float p, const int64_t *state,
                                     uint32_t call, int relu, void *dx, ls3d_stream_t stream) {
  return dropout_run(false, dy, dy_ld, y, rows, c, dtype, p, state, call, relu, dx, (hipStream_t)stream);
}
