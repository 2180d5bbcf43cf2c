// dropout.hip — dropout whose mask comes from a counter-based generator (blocks_common.h) and is never stored.
//
//   forward   y = keep ? act(x) / (1 - p) : 0        act: identity or ReLU
//   backward  dx = keep ? dy / (1 - p) : 0
//
// A dropped element is zero whatever stands in its place (a select, no product: Inf and NaN behind the mask do not get through).  Bound by memory:
// a pass reads one tensor and writes one.  With the ReLU the backward pass needs to know where x was positive: the forward pass leaves one bit per
// element (kept and positive), a byte per chunk of 8 columns, where reading x or y again would be a third tensor in the backward pass: 360000 x 192 f32
// (276 MB), backward 163 us from y, 113 us from the bits.  Forward and backward of that case take 183 us in all, 6.1 TB/s.
#include "blocks_common.h"

// Tensors in and out of more than 256 MB together pass through no cache that would still hold them for the next kernel: non-temporal accesses, 276 + 276 MB f32
// 206 -> 188 us forward and backward, 138 + 138 MB bf16 108 -> 99; below, they cost: 33 + 33 MB bf16 32 -> 35 us.
constexpr long long DROPOUT_NT_BYTES = 256ll << 20;

// One 16-byte piece of a row per thread and trip: W = 8 columns of a 2-byte type, 4 of f32 (a counter's eight draws then serve two threads, which both run the
// generator: its instructions fit under the memory time, while 32 bytes per lane read with two loads 16 bytes apart reach 5.1 TB/s where 16 bytes reach 5.8).
// NT: non-temporal accesses, for tensors that no cache keeps until they are used again (see dropout_launch).  Index type 32 bits where the count allows.
template <typename T> struct dropout_piece { typedef ls3d_u32x4_a2 type; };
template <> struct dropout_piece<float> { typedef ls3d_u32x4_a4 type; };

template <typename T, bool NT>
__device__ __forceinline__ void dropout_load(const T *__restrict__ p, int m, float (&v)[16 / sizeof(T)]) {
  constexpr int W = 16 / sizeof(T);
  T t[W];
  if (m >= W) {
    const ls3d_u32x4 q = NT ? __builtin_nontemporal_load((const typename dropout_piece<T>::type *)p) : *(const typename dropout_piece<T>::type *)p;
    __builtin_memcpy(t, &q, 16);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) t[j] = j < m ? p[j] : (T)0.0f;
  }
#pragma unroll
  for (int j = 0; j < W; ++j) v[j] = (float)t[j];
}

template <typename T, bool NT>
__device__ __forceinline__ void dropout_store(T *__restrict__ p, int m, const float (&v)[16 / sizeof(T)]) {
  constexpr int W = 16 / sizeof(T);
  T t[W];
#pragma unroll
  for (int j = 0; j < W; ++j) t[j] = (T)v[j];
  if (m >= W) {
    ls3d_u32x4 q;
    __builtin_memcpy(&q, t, 16);
    if (NT) __builtin_nontemporal_store(q, (typename dropout_piece<T>::type *)p);
    else *(typename dropout_piece<T>::type *)p = q;
  } else {
#pragma unroll
    for (int j = 0; j < W - 1; ++j)
      if (j < m) p[j] = t[j];
  }
}

// bits: one byte per counter (8 columns); with W = 4 two neighbouring lanes hold its halves (pieces per row are even: both are in the same wave and row)
template <typename T, typename I, bool RELU, bool NT>
__global__ __launch_bounds__(256) void k_dropout_fwd(const T *__restrict__ x, size_t x_ld, I total, uint32_t pieces, long long c, uint32_t thr, float inv,
                                                     const int64_t *__restrict__ state, uint32_t call, T *__restrict__ y, uint8_t *__restrict__ bits) {
  constexpr int W = 16 / sizeof(T);
  const ls3d_dropout_key key = ls3d_dropout_key_load(state, call);
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / pieces), g = (uint32_t)(t - (I)row * pieces);
    const long long col = (long long)g * W;
    const int m = c - col < W ? (int)(c - col) : W;
    float v[W];
    dropout_load<T, NT>(x + (size_t)row * x_ld + col, m, v);
    uint32_t keep = ls3d_keep8(key, W == 8 ? g : g >> 1, row, thr);
    if (W == 4) keep = (g & 1u ? keep >> 4 : keep) & 15u;
    if (RELU) {
#pragma unroll
      for (int j = 0; j < W; ++j) keep &= ~(v[j] <= 0.0f ? 1u << j : 0u);  // (NaN passes, as through torch.relu)
      if (bits) {
        if (W == 8) bits[t] = (uint8_t)keep;
        else {
          const uint32_t other = __shfl_xor(keep, 1);
          if (!(g & 1u)) bits[t >> 1] = (uint8_t)(keep | other << 4);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = ((keep >> j) & 1u) ? v[j] * inv : 0.0f;
    dropout_store<T, NT>(y + (size_t)row * c + col, m, v);
  }
}

template <typename T, typename I, bool RELU, bool NT>
__global__ __launch_bounds__(256) void k_dropout_bwd(const T *__restrict__ dy, size_t dy_ld, const uint8_t *__restrict__ bits, I total, uint32_t pieces, long long c,
                                                     uint32_t thr, float inv, const int64_t *__restrict__ state, uint32_t call, T *__restrict__ dx) {
  constexpr int W = 16 / sizeof(T);
  const ls3d_dropout_key key = RELU ? ls3d_dropout_key{} : ls3d_dropout_key_load(state, call);
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(t / pieces), g = (uint32_t)(t - (I)row * pieces);
    const long long col = (long long)g * W;
    const int m = c - col < W ? (int)(c - col) : W;
    uint32_t keep = RELU ? bits[W == 8 ? t : t >> 1] : ls3d_keep8(key, W == 8 ? g : g >> 1, row, thr);
    if (W == 4) keep = g & 1u ? keep >> 4 : keep;
    float v[W];
    dropout_load<T, NT>(dy + (size_t)row * dy_ld + col, m, v);
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = ((keep >> j) & 1u) ? v[j] * inv : 0.0f;
    dropout_store<T, NT>(dx + (size_t)row * c + col, m, v);
  }
}

template <typename T, bool RELU>
static void dropout_launch(bool fwd, const void *a, size_t ld, uint8_t *bits, long long rows, long long c, uint32_t thr, float inv, const int64_t *state,
                           uint32_t call, void *out, hipStream_t stream) {
  const uint32_t pieces = (uint32_t)((c + 7) / 8) * (sizeof(T) == 4 ? 2 : 1);  // whole counters: an even number of f32 pieces
  const long long total = rows * (long long)pieces;
  const bool nt = total * 32 > DROPOUT_NT_BYTES;
  // two trips a thread on large tensors (276 MB f32, forward and backward: 208 us on 2048 workgroups, 188 on 16384, 183 on 65536 = two trips)
  const dim3 grid = total < (1 << 20) ? ls3d_grid(total) : ls3d_grid(total, 512, 1 << 22);
#define DROPOUT_GO(I_, NT_)                                                                                                                                                    \
  do {                                                                                                                                                                         \
    if (fwd) hipLaunchKernelGGL((k_dropout_fwd<T, I_, RELU, NT_>), grid, dim3(256), 0, stream, (const T *)a, ld, (I_)total, pieces, c, thr, inv, state, call, (T *)out, bits); \
    else hipLaunchKernelGGL((k_dropout_bwd<T, I_, RELU, NT_>), grid, dim3(256), 0, stream, (const T *)a, ld, (const uint8_t *)bits, (I_)total, pieces, c, thr, inv, state,    \
                            call, (T *)out);                                                                                                                                  \
  } while (0)
  if (total >= (1ll << 31)) DROPOUT_GO(unsigned long long, true);
  else if (nt) DROPOUT_GO(uint32_t, true);
  else DROPOUT_GO(uint32_t, false);
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
