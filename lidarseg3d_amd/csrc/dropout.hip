// dropout.hip — dropout whose mask comes from a counter-based generator (blocks_common.h) and is never stored.
//
//   forward   y = keep ? act(x) / (1 - p) : 0        act: identity or ReLU
//   backward  dx = keep ? dy / (1 - p) : 0
//
// A dropped element is zero whatever stands in its place (a select, no product: Inf and NaN behind the mask do not get through).  Bound by memory:
// a pass reads one tensor and writes one.  With the ReLU the backward pass needs to know where x was positive: the forward pass leaves one bit per
// element (kept and positive), a byte per chunk of 8 columns, where reading x or y again would be a third tensor in the backward pass: 360000 x 192 f32
// (276 MB), backward 163 us from y, 113 us from the bits, forward 111 us without them, 117 us with (4.8 TB/s; a large copy: 5.1).
#include "blocks_common.h"

// one chunk of 8 columns per thread and trip; index type 32 bits where the chunk count allows (the division by the row's chunk count)
template <typename T, typename I, bool RELU>
__global__ __launch_bounds__(256) void k_dropout_fwd(const T *__restrict__ x, size_t x_ld, I total, uint32_t groups, long long c, uint32_t thr, float inv,
                                                     const int64_t *__restrict__ state, uint32_t call, T *__restrict__ y, uint8_t *__restrict__ bits) {
  const ls3d_dropout_key key = ls3d_dropout_key_load(state, call);
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / groups), g = (uint32_t)(t - (I)row * groups);
    const long long col = (long long)g * 8;
    const int m = c - col < 8 ? (int)(c - col) : 8;
    float v[8];
    ls3d_unpack8<T>(ls3d_load8<T>(x + (size_t)row * x_ld, col, c), m, v);
    uint32_t keep = ls3d_keep8(key, g, row, thr);
    if (RELU) {
#pragma unroll
      for (int j = 0; j < 8; ++j) keep &= ~(v[j] <= 0.0f ? 1u << j : 0u);  // (NaN passes, as through torch.relu)
      if (bits) bits[t] = (uint8_t)keep;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ((keep >> j) & 1u) ? v[j] * inv : 0.0f;
    ls3d_store8<T>(y + (size_t)row * c + col, v, m);
  }
}

template <typename T, typename I, bool RELU>
__global__ __launch_bounds__(256) void k_dropout_bwd(const T *__restrict__ dy, size_t dy_ld, const uint8_t *__restrict__ bits, I total, uint32_t groups, long long c,
                                                     uint32_t thr, float inv, const int64_t *__restrict__ state, uint32_t call, T *__restrict__ dx) {
  const ls3d_dropout_key key = RELU ? ls3d_dropout_key{} : ls3d_dropout_key_load(state, call);
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / groups), g = (uint32_t)(t - (I)row * groups);
    const long long col = (long long)g * 8;
    const int m = c - col < 8 ? (int)(c - col) : 8;
    const uint32_t keep = RELU ? bits[t] : ls3d_keep8(key, g, row, thr);
    float v[8];
    ls3d_unpack8<T>(ls3d_load8<T>(dy + (size_t)row * dy_ld, col, c), m, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ((keep >> j) & 1u) ? v[j] * inv : 0.0f;
    ls3d_store8<T>(dx + (size_t)row * c + col, v, m);
  }
}

template <typename T, bool RELU>
static void dropout_launch(bool fwd, const void *a, size_t ld, uint8_t *bits, long long rows, long long c, uint32_t thr, float inv, const int64_t *state,
                           uint32_t call, void *out, hipStream_t stream) {
  const uint32_t groups = (uint32_t)((c + 7) / 8);
  const long long total = rows * (long long)groups;
  const dim3 grid = ls3d_grid(total);
#define DROPOUT_GO(I_)                                                                                                                                                    \
  do {                                                                                                                                                                    \
    if (fwd) hipLaunchKernelGGL((k_dropout_fwd<T, I_, RELU>), grid, dim3(256), 0, stream, (const T *)a, ld, (I_)total, groups, c, thr, inv, state, call, (T *)out, bits); \
    else hipLaunchKernelGGL((k_dropout_bwd<T, I_, RELU>), grid, dim3(256), 0, stream, (const T *)a, ld, (const uint8_t *)bits, (I_)total, groups, c, thr, inv, state,    \
                            call, (T *)out);                                                                                                                              \
  } while (0)
  if (total < (1ll << 31)) DROPOUT_GO(uint32_t);
  else DROPOUT_GO(unsigned long long);
#undef DROPOUT_GO
}

static int dropout_run(bool fwd, const void *a, long long ld, uint8_t *bits, long long rows, long long c, int dtype, float p, const int64_t *state, uint32_t call,
                       int relu, void *out, hipStream_t stream) {
  uint32_t thr;
  float inv;
  if (rows < 0 || c < 0 || rows > 0x7FFFFFFFll || c > 0x7FFFFFFFll || !ls3d_dtype_ok(dtype) || !ls3d_dropout_threshold(p, &thr, &inv)) return LS3D_ERR_ARG;
  if (rows == 0 || c == 0) return LS3D_OK;
  if (!a || !out || ld < c || !state || ((uintptr_t)state & 7) || (!fwd && relu && !bits)) return LS3D_ERR_ARG;
  if (((uintptr_t)a | (uintptr_t)out) & (ls3d_dtype_size(dtype) - 1)) return LS3D_ERR_ARG;
#define DROPOUT_TYPE(T)                                                                                                           \
  do {                                                                                                                            \
    if (relu) dropout_launch<T, true>(fwd, a, (size_t)ld, bits, rows, c, thr, inv, state, call, out, stream);                     \
    else dropout_launch<T, false>(fwd, a, (size_t)ld, nullptr, rows, c, thr, inv, state, call, out, stream);                      \
  } while (0)
  if (dtype == LS3D_DTYPE_F32) DROPOUT_TYPE(float);
  else if (dtype == LS3D_DTYPE_BF16) DROPOUT_TYPE(ls3d_bf16);
  else DROPOUT_TYPE(ls3d_f16);
#undef DROPOUT_TYPE
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}

extern "C" int ls3d_dropout_forward(const void *x, long long x_ld, long long rows, long long c, int dtype, float p, const int64_t *state, uint32_t call,
                                    int relu, void *y, uint8_t *bits, ls3d_stream_t stream) {
  return dropout_run(true, x, x_ld, bits, rows, c, dtype, p, state, call, relu, y, (hipStream_t)stream);
}

extern "C" int ls3d_dropout_backward(const void *dy, long long dy_ld, const uint8_t *bits, long long rows, long long c, int dtype, float p, const int64_t *state,
                                     uint32_t call, int relu, void *dx, ls3d_stream_t stream) {
  return dropout_run(false, dy, dy_ld, const_cast<uint8_t *>(bits), rows, c, dtype, p, state, call, relu, dx, (hipStream_t)stream);
}
