// blocks_common.h — what the training-block operators share (resnorm.h, dropout.hip, embedding.hip): element types, rows in chunks of eight columns,
// the counter-based generator.
#pragma once
#include "common.h"

// ---- element types: f32, bf16, f16 in memory, f32 in registers.  A chunk is 8 columns: one 16-byte access of a 2-byte type, two of f32.  The
//      chunks of a row with an odd width start at any multiple of the element size; gfx950 takes global accesses at any alignment.
//
// LS3D_OPAQUE: a value the compiler knows nothing about from here on.  Column counts go through it once per row: comparisons with them would
// otherwise be made before the row loop, 8 lane masks a chunk, and parked in scalar registers there are not enough of.
#ifdef HIPSIM
#define LS3D_OPAQUE(x) ((void)0)
#else
#define LS3D_OPAQUE(x) asm("" : "+v"(x))
#endif

// between an LDS access of some lanes and one of others of the same wave: the compiler keeps their order (the hardware does by itself)
#ifdef HIPSIM
#define LS3D_WAVE_SYNC() ((void)__ballot(1))
#else
#define LS3D_WAVE_SYNC()                               \
  do {                                                 \
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); \
    __builtin_amdgcn_wave_barrier();                   \
  } while (0)
#endif
typedef __bf16 ls3d_bf16;
typedef _Float16 ls3d_f16;
typedef uint32_t ls3d_u32x4 __attribute__((ext_vector_type(4)));
typedef ls3d_u32x4 ls3d_u32x4_a2 __attribute__((aligned(2)));
typedef ls3d_u32x4 ls3d_u32x4_a4 __attribute__((aligned(4)));

template <typename T>
struct ls3d_raw8 { ls3d_u32x4 q[sizeof(T) / 2]; };  // a chunk as it stands in memory

// the chunk at column `col` of a row of c columns, whatever of it lies inside: where fewer than 8 columns are left the LAST 8 of the row are read instead
// (one access at any width and no branch around it; ls3d_unpack8 moves them into place), and a chunk that lies behind the row reads them too.  NT: a
// non-temporal access of a 2-byte type.
template <typename T, bool NT = false>
__device__ __forceinline__ ls3d_raw8<T> ls3d_load8(const T *__restrict__ row, long long col, long long c) {
  ls3d_raw8<T> r;
  if (c >= 8) {
    const T *__restrict__ p = row + (col < c - 8 ? col : c - 8);
    if (sizeof(T) == 2) r.q[0] = NT ? __builtin_nontemporal_load((const ls3d_u32x4_a2 *)p) : *(const ls3d_u32x4_a2 *)p;
    else {
      r.q[0] = *(const ls3d_u32x4_a4 *)p;
      r.q[sizeof(T) / 2 - 1] = *(const ls3d_u32x4_a4 *)((const char *)p + 16);
    }
    return r;
  }
  T t[8];  // rows of fewer than 8 columns: one chunk, element by element, aligned to its end like the rest
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = j >= 8 - (int)c ? row[j - (8 - (int)c)] : (T)0.0f;
  __builtin_memcpy(&r, t, sizeof(t));
  return r;
}

// a chunk with m live columns as f32: m >= 8 all; fewer: the loaded columns are the row's last ones, the live ones move to the front and zeros follow;
// m <= 0: zeros whatever was read
template <typename T>
__device__ __forceinline__ void ls3d_unpack8(const ls3d_raw8<T> &r, int m, float (&v)[8]) {
  T t[8];
  __builtin_memcpy(t, &r, sizeof(t));
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
  if (m < 8) {
    LS3D_OPAQUE(m);  // the comparisons below are made here, not shared with every other chunk of the row
    const int s = m > 0 ? 8 - m : 8;
#pragma unroll
    for (int step = 8; step >= 1; step >>= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (s & step) ? (j + step < 8 ? v[j + step] : 0.0f) : v[j];
  }
}

// rounds to T once (to nearest, ties to even) and stores the live columns
template <typename T, bool NT = false>
__device__ __forceinline__ void ls3d_store8(T *__restrict__ p, const float (&v)[8], int m) {
  T t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (T)v[j];
  if (m >= 8) {
    ls3d_raw8<T> r;
    __builtin_memcpy(&r, t, sizeof(t));
    if (sizeof(T) == 2) {
      if (NT) __builtin_nontemporal_store(r.q[0], (ls3d_u32x4_a2 *)p);
      else *(ls3d_u32x4_a2 *)p = r.q[0];
    } else {
      *(ls3d_u32x4_a4 *)p = r.q[0];
      *(ls3d_u32x4_a4 *)((char *)p + 16) = r.q[sizeof(T) / 2 - 1];
    }
    return;
  }
  if (m > 0) {
    LS3D_OPAQUE(m);
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < m) p[j] = t[j];
  }
}

// half a chunk, 4 columns of f32 in one 16-byte access; the same treatment of the row's end
template <bool NT>
__device__ __forceinline__ ls3d_u32x4 ls3d_load4(const float *__restrict__ row, int col, int c) {
  if (c >= 4) {
    const ls3d_u32x4_a4 *p = (const ls3d_u32x4_a4 *)(row + (col < c - 4 ? col : c - 4));
    return NT ? __builtin_nontemporal_load(p) : *p;
  }
  float t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = j >= 4 - c ? row[j - (4 - c)] : 0.0f;
  ls3d_u32x4 r;
  __builtin_memcpy(&r, t, sizeof(t));
  return r;
}
__device__ __forceinline__ void ls3d_unpack4(const ls3d_u32x4 &r, int m, float *v) {
  float t[4];
  __builtin_memcpy(t, &r, sizeof(t));
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = t[j];
  if (m < 4) {
    LS3D_OPAQUE(m);
    const int s = m > 0 ? 4 - m : 4;
#pragma unroll
    for (int step = 4; step >= 1; step >>= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (s & step) ? (j + step < 4 ? v[j + step] : 0.0f) : v[j];
  }
}
template <bool NT>
__device__ __forceinline__ void ls3d_store4(float *__restrict__ p, const float *v, int m) {
  if (m >= 4) {
    ls3d_u32x4 r;
    __builtin_memcpy(&r, v, 16);
    if (NT) __builtin_nontemporal_store(r, (ls3d_u32x4_a4 *)p);
    else *(ls3d_u32x4_a4 *)p = r;
  } else if (m > 0) {
    LS3D_OPAQUE(m);
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < m) p[j] = v[j];
  }
}

// a chunk of a parameter vector of any of the types; NULL reads as `otherwise`; zeros behind the end
__device__ __forceinline__ void ls3d_param8(const void *__restrict__ p, int dtype, int col, int c, float otherwise, float (&v)[8]) {
  const int m = c - col;
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < m ? otherwise : 0.0f;
  } else if (dtype == LS3D_DTYPE_F32) ls3d_unpack8<float>(ls3d_load8<float>((const float *)p, col, c), m, v);
  else if (dtype == LS3D_DTYPE_BF16) ls3d_unpack8<ls3d_bf16>(ls3d_load8<ls3d_bf16>((const ls3d_bf16 *)p, col, c), m, v);
  else ls3d_unpack8<ls3d_f16>(ls3d_load8<ls3d_f16>((const ls3d_f16 *)p, col, c), m, v);
}
// half a chunk of one
__device__ __forceinline__ void ls3d_param4(const void *__restrict__ p, int dtype, int col, int c, float otherwise, float *v) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = col + j < c ? otherwise : 0.0f;
  } else if (dtype == LS3D_DTYPE_F32) ls3d_unpack4(ls3d_load4<false>((const float *)p, col, c), c - col, v);
  else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = col + j >= c ? 0.0f : dtype == LS3D_DTYPE_BF16 ? (float)((const ls3d_bf16 *)p)[col + j] : (float)((const ls3d_f16 *)p)[col + j];
  }
}
__device__ __forceinline__ void ls3d_param_store(void *__restrict__ p, int dtype, size_t i, float v) {
  if (dtype == LS3D_DTYPE_F32) ((float *)p)[i] = v;
  else if (dtype == LS3D_DTYPE_BF16) ((ls3d_bf16 *)p)[i] = (ls3d_bf16)v;
  else ((ls3d_f16 *)p)[i] = (ls3d_f16)v;
}

// ---- counter-based generator: Philox4x32, 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC11).  Key =
//      (low, high half of the seed), counter = (column / 8, row, call, step): any element's draw comes from its place alone, so the backward pass
//      makes the forward's mask again and nothing is stored.  The four output words are eight 16-bit draws, low half first: one round function for
//      eight elements (with 32-bit draws the multiplications of a bf16 dropout would take longer than its memory traffic).
struct ls3d_dropout_key { uint32_t k0, k1, call, step; };

__device__ __forceinline__ ls3d_dropout_key ls3d_dropout_key_load(const int64_t *__restrict__ state, uint32_t call) {
  const uint64_t seed = (uint64_t)state[0];
  return ls3d_dropout_key{(uint32_t)seed, (uint32_t)(seed >> 32), call, (uint32_t)(uint64_t)state[1]};
}

// bit j: column 8 * group + j of the row is kept (its draw is not below thr, 0 <= thr <= 65536)
__device__ __forceinline__ uint32_t ls3d_keep8(const ls3d_dropout_key &key, uint32_t group, uint32_t row, uint32_t thr) {
  uint32_t c0 = group, c1 = row, c2 = key.call, c3 = key.step, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    keep |= (w[j] & 0xFFFFu) >= thr ? 1u << (2 * j) : 0u;
    keep |= (w[j] >> 16) >= thr ? 2u << (2 * j) : 0u;
  }
  return keep;
}

// p in [0, 1] as the threshold of a 16-bit draw, and the factor that keeps the expectation for THAT probability; false: p is no probability
static inline bool ls3d_dropout_threshold(float p, uint32_t *thr, float *inv) {
  if (!(p >= 0.0f && p <= 1.0f)) return false;
  *thr = (uint32_t)((double)p * 65536.0 + 0.5);
  *inv = *thr < 65536u ? 65536.0f / (float)(65536u - *thr) : 0.0f;
  return true;
}

static inline bool ls3d_dtype_ok(int t) { return t == LS3D_DTYPE_F32 || t == LS3D_DTYPE_BF16 || t == LS3D_DTYPE_F16; }
static inline size_t ls3d_dtype_size(int t) { return t == LS3D_DTYPE_F32 ? 4 : 2; }
