// resnorm.h — a transformer block's residual in one pass, forward and backward; instantiated per pair of element types by resnorm_*.hip.
//
//   t = N_in(x)                           N: layer norm, RMS norm or nothing; statistics and sums in f32
//   d = keep ? t / (1 - p) : 0            counter-based mask (blocks_common.h)
//   s = alpha * residual + gate * d       gate: one value per channel, per element, or none
//   y = N_out(s)                          from s as it stands in registers: y does not see s's rounding to its type
//
// Backward, per row, with S the gradient that reaches s:
//   u = dy * w_out;  S = ds + rstd (u - [mean u] - shat mean(u shat))        ([.]: layer norm only)
//   dresidual = alpha S;  d gate = S d;  dt = keep ? gate S / (1 - p) : 0;  dx = N_in's gradient of dt, the same formula
//   and the column sums  dw_out = sum dy shat, db_out = sum dy, dw_in = sum dt xhat, db_in = sum dt, dgate = sum S d.
// s is computed again from x and the residual rather than kept: the forward's inputs are what autograd holds anyway.
//
// Bound by memory: x, residual (, gate) in and y (, s) out; backward dy (, ds) in addition, dx, dresidual out.  One pass: a row lives in the registers of
// LPR lanes, VPT chunks of 8 columns each (LPR <= 64: 64 / LPR rows side by side in a wave, sums by lane exchange; LPR = 256: a row per
// workgroup, sums through LDS).  Few lanes per row keep the exchanges few: 96 columns are 4 lanes x 3 chunks and two exchange steps a sum.
#pragma once
#include "blocks_common.h"

struct ls3d_rn_args {
  const void *x, *res, *gate;
  size_t x_ld, res_ld, gate_ld;
  int n, c;
  int kind_in, kind_out, gate_kind;
  const void *w_in, *b_in, *w_out, *b_out;
  int w_in_t, b_in_t, w_out_t, b_out_t, gate_t;
  float eps_in, eps_out, alpha, inv;
  float share, whole;  // a row's mean: the sum of share * value divided by whole; share: a power of two, whole: c * share in (0.5, 1]
  uint32_t thr, call;
  const int64_t *state;
  float *stats;  // [n][4]: mean, rstd of N_in, mean, rstd of N_out
  void *y, *s;   // forward's outputs
  const void *dy, *ds;
  size_t dy_ld, ds_ld;
  void *dx, *dres, *dgate;  // dgate: [n, c] of a full gate
  float *partial;           // [blocks][columns' sums][c]
  int nsum;                 // sums a block writes: the slots below that are wanted, packed
  int slot[5];              // dw_out, db_out, dw_in, db_in, dgate (channel): place among the block's sums, -1: not wanted
};

// threads of a workgroup: 256, or the lanes of a row where that is more
template <int LPR>
constexpr int ls3d_rn_threads() { return LPR > 256 ? LPR : 256; }

// Where a lane's 8 columns of chunk i lie in the row.  Two-byte types: 8 in a row, one 16-byte access.  f32 throughout on 16 lanes or more (SPLIT): 4 + 4, in the two
// halves of the LPR * 8 columns that the lanes cover together, so that each of the two accesses of a wave is contiguous over the lanes of a row: what
// non-temporal accesses need (32 bytes a lane as two accesses 16 bytes apart: a plain copy of 276 MB 4.0 TB/s with them, 5.1 without; contiguous: 6.3 and 5.8).
// m: live columns from the lane's first one on.
template <typename TX, typename TR>
constexpr bool ls3d_rn_split(int lpr) { return sizeof(TX) == 4 && sizeof(TR) == 4 && lpr >= 16; }

template <int LPR, bool SPLIT>
struct ls3d_rn_map {
  static __device__ __forceinline__ int first(int lane, int i) { return SPLIT ? i * LPR * 8 + lane * 4 : (lane + i * LPR) * 8; }
  static __device__ __forceinline__ int column(int lane, int i, int j) { return first(lane, i) + (SPLIT && j >= 4 ? LPR * 4 + j - 4 : j); }
  template <typename T, bool NT>
  static __device__ __forceinline__ ls3d_raw8<T> load(const void *__restrict__ base, size_t row, size_t ld, int lane, int i, int c) {
    const T *__restrict__ p = (const T *)base + row * ld;
    if constexpr (SPLIT) {
      ls3d_raw8<T> r;
      r.q[0] = ls3d_load4<NT>((const float *)p, first(lane, i), c);
      r.q[1] = ls3d_load4<NT>((const float *)p, first(lane, i) + LPR * 4, c);
      return r;
    } else return ls3d_load8<T, NT>(p, first(lane, i), c);
  }
  template <typename T>
  static __device__ __forceinline__ void unpack(const ls3d_raw8<T> &r, int m, float (&v)[8]) {
    if constexpr (SPLIT) {
      ls3d_unpack4(r.q[0], m, v);
      ls3d_unpack4(r.q[1], m - LPR * 4, v + 4);
    } else ls3d_unpack8<T>(r, m, v);
  }
  template <typename T, bool NT>
  static __device__ __forceinline__ void store(void *__restrict__ base, size_t row, int lane, int i, int c, const float (&v)[8], int m) {
    T *__restrict__ p = (T *)base + row * c + first(lane, i);
    if constexpr (SPLIT) {
      ls3d_store4<NT>((float *)p, v, m);
      ls3d_store4<NT>((float *)p + LPR * 4, v + 4, m - LPR * 4);
    } else ls3d_store8<T, NT>(p, v, m);
  }
  static __device__ __forceinline__ void param(const void *__restrict__ p, int dtype, int lane, int i, int c, float otherwise, float (&v)[8]) {
    if constexpr (SPLIT) {
      ls3d_param4(p, dtype, first(lane, i), c, otherwise, v);
      ls3d_param4(p, dtype, first(lane, i) + LPR * 4, c, otherwise, v + 4);
    } else ls3d_param8(p, dtype, first(lane, i), c, otherwise, v);
  }
  // zeros behind the row's end, m live columns: what a norm makes of the zeros there, (0 - mean) / std, is infinite for a mean near the largest values and NaN for a
  // row that holds infinities, and even a product with zero would carry that into the row's sums
  static __device__ __forceinline__ void clip(float (&v)[8], int m) {
    if (m >= (SPLIT ? LPR * 4 + 4 : 8)) return;
    LS3D_OPAQUE(m);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (SPLIT && j >= 4 ? LPR * 4 + j - 4 : j) < m ? v[j] : 0.0f;
  }
  static __device__ __forceinline__ uint32_t keep(const ls3d_dropout_key &key, int lane, int i, uint32_t row, uint32_t thr) {
    if constexpr (SPLIT) {  // halves of two counters
      const uint32_t a = (uint32_t)first(lane, i), b = a + LPR * 4;
      const uint32_t x = ls3d_keep8(key, a >> 3, row, thr), y = ls3d_keep8(key, b >> 3, row, thr);
      return ((x >> (a & 4)) & 15u) | ((y >> (b & 4)) & 15u) << 4;
    } else return ls3d_keep8(key, (uint32_t)first(lane, i) >> 3, row, thr);
  }
};

// sums of two values over the LPR lanes of a row; LPR > 64: over the workgroup (`lds`: 2 x 16 x 2 floats, halves used in turn so that one barrier a sum is enough)
template <int LPR>
struct ls3d_row_sums {
  float *lds;
  int turn;
  __device__ __forceinline__ ls3d_row_sums(float *l) : lds(l), turn(0) {}
  __device__ __forceinline__ void operator()(float &a, float &b) {
#pragma unroll
    for (int d = (LPR < 64 ? LPR : 64) / 2; d >= 1; d >>= 1) {
      a += __shfl_xor(a, d);
      b += __shfl_xor(b, d);
    }
    if (LPR > 64) {
      float *half = lds + turn * 32;
      if ((threadIdx.x & 63) == 0) { half[(threadIdx.x >> 6) * 2] = a; half[(threadIdx.x >> 6) * 2 + 1] = b; }
      __syncthreads();
      half += (threadIdx.x / LPR) * (LPR / 64) * 2;  // the waves of this thread's row
      a = half[0];
      b = half[1];
#pragma unroll
      for (int w = 1; w < LPR / 64; ++w) { a += half[2 * w]; b += half[2 * w + 1]; }
      turn ^= 1;
    }
  }
  __device__ __forceinline__ void operator()(float &a) {
    if (LPR > 64) {
      float b = 0.0f;
      (*this)(a, b);
      return;
    }
#pragma unroll
    for (int d = (LPR < 64 ? LPR : 64) / 2; d >= 1; d >>= 1) a += __shfl_xor(a, d);
  }
};

// mean and 1 / sqrt(variance + eps) of a row's values (two passes over registers: no cancellation); RMS: mean 0.  Columns behind the row's end hold zeros;
// m0: live columns from the lane's first chunk on.  The mean is summed in shares, so that a row of the type's lowest values does not overflow, and a share is
// exact: equal values of 2-byte types then have their value as mean and deviation 0 at any c (in shares of 1 / c each is rounded: 60000 at c = 96 is off by 0.01
// alike in every column, which the norm makes +-1 of).  Cost: a division a row.
template <int LPR, int VPT, bool SPLIT>
__device__ __forceinline__ void ls3d_rn_stats(const float (&v)[VPT][8], int kind, int m0, const ls3d_rn_args &A, float inv_c, float eps, ls3d_row_sums<LPR> &sums,
                                              float &mean, float &rstd) {
  mean = 0.0f;
  if (kind == LS3D_NORM_LAYER) {
    float a = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) a = fmaf(v[i][j], A.share, a);
    sums(a);
    mean = a / A.whole;
  }
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int m = m0 - i * LPR * 8;
    if (m >= (SPLIT ? LPR * 4 + 4 : 8)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = v[i][j] - mean;
        q = fmaf(d, d, q);
      }
    } else if (m > 0) {
      int k = m;
      LS3D_OPAQUE(k);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float d = (SPLIT && j >= 4 ? LPR * 4 + j - 4 : j) < k ? v[i][j] - mean : 0.0f;
        q = fmaf(d, d, q);
      }
    }
  }
  sums(q);
  rstd = 1.0f / sqrtf(q * inv_c + eps);
}

// FULL: a norm before or a gate; without them neither their registers nor their sums exist.  NT: non-temporal accesses to the rows (rn_streams in resnorm.hip)
template <typename TX, typename TR, int LPR, int VPT, bool FULL, bool NT>
__global__ __launch_bounds__(ls3d_rn_threads<LPR>()) void k_resnorm_fwd(const ls3d_rn_args A) {
  constexpr bool SPLIT = ls3d_rn_split<TX, TR>(LPR);
  typedef ls3d_rn_map<LPR, SPLIT> M;
  __shared__ float s_sum[64];
  constexpr int ROWS = ls3d_rn_threads<LPR>() / LPR;
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR, c = A.c;
  const float inv_c = 1.0f / (float)c;
  ls3d_dropout_key key = {};
  if (A.thr) key = ls3d_dropout_key_load(A.state, A.call);
  ls3d_row_sums<LPR> sums(s_sum);
  float wo[VPT][8], bo[VPT][8], wi[FULL ? VPT : 1][8], bi[FULL ? VPT : 1][8], g[FULL ? VPT : 1][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    M::param(A.w_out, A.w_out_t, lane, i, c, 1.0f, wo[i]);
    M::param(A.b_out, A.b_out_t, lane, i, c, 0.0f, bo[i]);
    if (FULL) {
      M::param(A.w_in, A.w_in_t, lane, i, c, 1.0f, wi[i]);
      M::param(A.b_in, A.b_in_t, lane, i, c, 0.0f, bi[i]);
      M::param(A.gate_kind == LS3D_GATE_CHANNEL ? A.gate : nullptr, A.gate_t, lane, i, c, 1.0f, g[i]);
    }
  }
  for (long long row0 = (long long)blockIdx.x * ROWS; row0 < A.n; row0 += (long long)gridDim.x * ROWS) {  // the same trips for every lane of a wave / workgroup
    const bool live = row0 + sub < A.n;
    const size_t row = (size_t)(live ? row0 + sub : A.n - 1);
    int m0 = live ? c - M::first(lane, 0) : 0;  // a dead row reads the last one and counts as zeros
    LS3D_OPAQUE(m0);
    ls3d_raw8<TX> rx[VPT], rg[FULL ? VPT : 1];
    ls3d_raw8<TR> rr[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) rx[i] = M::template load<TX, NT>(A.x, row, A.x_ld, lane, i, c);
    if (A.res) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) rr[i] = M::template load<TR, NT>(A.res, row, A.res_ld, lane, i, c);
    }
    if (FULL && A.gate_kind == LS3D_GATE_FULL) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) rg[i] = M::template load<TX, NT>(A.gate, row, A.gate_ld, lane, i, c);
    }
    float v[VPT][8];
#pragma unroll
    for (int i = 0; i < VPT; ++i) M::template unpack<TX>(rx[i], m0 - i * LPR * 8, v[i]);
    float st[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (FULL && A.kind_in) {
      ls3d_rn_stats<LPR, VPT, SPLIT>(v, A.kind_in, m0, A, inv_c, A.eps_in, sums, st[0], st[1]);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf((v[i][j] - st[0]) * st[1], wi[i][j], bi[i][j]);
        M::clip(v[i], m0 - i * LPR * 8);
      }
    }
    if (A.thr) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uint32_t keep = M::keep(key, lane, i, (uint32_t)row, A.thr);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = ((keep >> j) & 1u) ? v[i][j] * A.inv : 0.0f;
      }
    }
    if (FULL && A.gate_kind) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (A.gate_kind == LS3D_GATE_FULL) M::template unpack<TX>(rg[i], m0 - i * LPR * 8, g[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= g[i][j];
      }
    }
    if (A.res) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float r[8];
        M::template unpack<TR>(rr[i], m0 - i * LPR * 8, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = fmaf(A.alpha, r[j], v[i][j]);
      }
    }
    if (A.s) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) M::template store<TR, NT>(A.s, row, lane, i, c, v[i], m0 - i * LPR * 8);
    }
    if (A.kind_out) {
      ls3d_rn_stats<LPR, VPT, SPLIT>(v, A.kind_out, m0, A, inv_c, A.eps_out, sums, st[2], st[3]);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = fmaf((v[i][j] - st[2]) * st[3], wo[i][j], bo[i][j]);
        M::template store<TX, NT>(A.y, row, lane, i, c, o, m0 - i * LPR * 8);
      }
    }
    if (A.stats && live && lane == 0) *(float4 *)(A.stats + row * 4) = make_float4(st[0], st[1], st[2], st[3]);
  }
}

template <typename TX, typename TR, int LPR, int VPT, bool FULL, bool NT>
__global__ __launch_bounds__(ls3d_rn_threads<LPR>(), LPR > 512 ? 4 : 2) void k_resnorm_bwd(const ls3d_rn_args A) {
  constexpr int THREADS = ls3d_rn_threads<LPR>(), ROWS = THREADS / LPR, WIDTH = LPR * VPT * 8, NV = FULL ? VPT : 1, NSUM = FULL ? 5 : 2;
  constexpr bool SPLIT = ls3d_rn_split<TX, TR>(LPR);
  typedef ls3d_rn_map<LPR, SPLIT> M;
  __shared__ float s_sum[64];
  constexpr int PARTS = LPR <= 64 ? 4 : ROWS;  // row groups that meet in LDS: the waves (their own groups by lane exchange), or the rows of a workgroup
  __shared__ float s_col[PARTS > 1 ? PARTS * WIDTH : 1];
  const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR, c = A.c;
  const float inv_c = 1.0f / (float)c;
  ls3d_dropout_key key = {};
  if (A.thr) key = ls3d_dropout_key_load(A.state, A.call);
  ls3d_row_sums<LPR> sums(s_sum);
  float acc[NSUM][VPT][8], wo[VPT][8], wi[NV][8], bi[NV][8], g[NV][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
#pragma unroll
    for (int k = 0; k < NSUM; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[k][i][j] = 0.0f;
    M::param(A.w_out, A.w_out_t, lane, i, c, 1.0f, wo[i]);
    if (FULL) {
      M::param(A.w_in, A.w_in_t, lane, i, c, 1.0f, wi[i]);
      M::param(A.b_in, A.b_in_t, lane, i, c, 0.0f, bi[i]);
      M::param(A.gate_kind == LS3D_GATE_CHANNEL ? A.gate : nullptr, A.gate_t, lane, i, c, 1.0f, g[i]);
    }
  }
  for (long long row0 = (long long)blockIdx.x * ROWS; row0 < A.n; row0 += (long long)gridDim.x * ROWS) {
    const bool live = row0 + sub < A.n;
    const size_t row = (size_t)(live ? row0 + sub : A.n - 1);
    int m0 = live ? c - M::first(lane, 0) : 0;
    LS3D_OPAQUE(m0);
    ls3d_raw8<TX> rx[VPT], ry[VPT], rg[NV];
    ls3d_raw8<TR> rr[VPT], rs[VPT];
    // every load of the row before the first use of one
#pragma unroll
    for (int i = 0; i < VPT; ++i) rx[i] = M::template load<TX, NT>(A.x, row, A.x_ld, lane, i, c);
    if (A.res) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) rr[i] = M::template load<TR, NT>(A.res, row, A.res_ld, lane, i, c);
    }
    if (A.dy) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) ry[i] = M::template load<TX, NT>(A.dy, row, A.dy_ld, lane, i, c);
    }
    if (A.ds) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) rs[i] = M::template load<TR, NT>(A.ds, row, A.ds_ld, lane, i, c);
    }
    if (FULL && A.gate_kind == LS3D_GATE_FULL) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) rg[i] = M::template load<TX, NT>(A.gate, row, A.gate_ld, lane, i, c);
    }
    const float4 st = *(const float4 *)(A.stats + row * 4);
    float xh[NV][8], sh[VPT][8], S[VPT][8];
    uint32_t keep[VPT];
    // s again, as the forward pass computed it
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      M::template unpack<TX>(rx[i], m0 - i * LPR * 8, sh[i]);
      if (FULL) {
#pragma unroll
        for (int j = 0; j < 8; ++j) xh[i][j] = A.kind_in ? (sh[i][j] - st.x) * st.y : sh[i][j];
        M::clip(xh[i], m0 - i * LPR * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[i][j] = A.kind_in ? fmaf(xh[i][j], wi[i][j], bi[i][j]) : xh[i][j];
      }
      keep[i] = 0xFFu;
      if (A.thr) {
        keep[i] = M::keep(key, lane, i, (uint32_t)row, A.thr);
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[i][j] = ((keep[i] >> j) & 1u) ? sh[i][j] * A.inv : 0.0f;
      }
      if (FULL) {
        if (A.gate_kind == LS3D_GATE_FULL) M::template unpack<TX>(rg[i], m0 - i * LPR * 8, g[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[i][j] *= g[i][j];
      }
      if (A.res) {
        float r[8];
        M::template unpack<TR>(rr[i], m0 - i * LPR * 8, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[i][j] = fmaf(A.alpha, r[j], sh[i][j]);
      }
    }
    // the gradient of s
    if (A.dy) {
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        M::template unpack<TX>(ry[i], m0 - i * LPR * 8, S[i]);  // zeros behind the row's end keep what stands there out of every sum
#pragma unroll
        for (int j = 0; j < 8; ++j) sh[i][j] = (sh[i][j] - st.z) * st.w;
        M::clip(sh[i], m0 - i * LPR * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc[0][i][j] = fmaf(S[i][j], sh[i][j], acc[0][i][j]);
          acc[1][i][j] += S[i][j];
          S[i][j] *= wo[i][j];
          s1 += S[i][j];
          s2 = fmaf(S[i][j], sh[i][j], s2);
        }
      }
      sums(s1, s2);
      const float c1 = A.kind_out == LS3D_NORM_LAYER ? s1 * inv_c : 0.0f, c2 = s2 * inv_c;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) S[i][j] = st.w * (S[i][j] - c1 - sh[i][j] * c2);
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) S[i][j] = 0.0f;
    }
    if (A.ds) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float d[8];
        M::template unpack<TR>(rs[i], m0 - i * LPR * 8, d);
#pragma unroll
        for (int j = 0; j < 8; ++j) S[i][j] += d[j];
      }
    }
    if (A.dres) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = A.alpha * S[i][j];
        M::template store<TR, NT>(A.dres, row, lane, i, c, o, m0 - i * LPR * 8);
      }
    }
    if (FULL && A.gate_kind) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float o[8];
        LS3D_OPAQUE(keep[i]);  // (the dropped t is formed again from xh: kept from above it would be 8 more registers a chunk)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float d = ((keep[i] >> j) & 1u) ? (A.kind_in ? fmaf(xh[i][j], wi[i][j], bi[i][j]) : xh[i][j]) * A.inv : 0.0f;
          o[j] = S[i][j] * d;
          S[i][j] *= g[i][j];
        }
        if (A.gate_kind == LS3D_GATE_FULL) {
          if (A.dgate) M::template store<TX, NT>(A.dgate, row, lane, i, c, o, m0 - i * LPR * 8);
        } else if (m0 - i * LPR * 8 > 0) {  // (S is not zero behind the row's end; columns there are never stored, a dead row's must not be added)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[4][i][j] += o[j];
        }
      }
    }
    if (A.thr) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        LS3D_OPAQUE(keep[i]);  // (lane masks of its bits are made again rather than parked)
#pragma unroll
        for (int j = 0; j < 8; ++j) S[i][j] = ((keep[i] >> j) & 1u) ? S[i][j] * A.inv : 0.0f;  // dt
      }
    }
    if (FULL && A.kind_in) {
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const bool in = m0 - i * LPR * 8 > 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (in) {
            acc[2][i][j] = fmaf(S[i][j], xh[i][j], acc[2][i][j]);
            acc[3][i][j] += S[i][j];
          }
          S[i][j] *= wi[i][j];  // zero behind the row's end
          s1 += S[i][j];
          s2 = fmaf(S[i][j], xh[i][j], s2);
        }
      }
      sums(s1, s2);
      const float c1 = A.kind_in == LS3D_NORM_LAYER ? s1 * inv_c : 0.0f, c2 = s2 * inv_c;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) S[i][j] = st.y * (S[i][j] - c1 - xh[i][j] * c2);
    }
    if (A.dx) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) M::template store<TX, NT>(A.dx, row, lane, i, c, S[i], m0 - i * LPR * 8);
    }
  }
  // the block's column sums: the row groups of a wave by lane exchange, what is left through LDS in order; a fixed tree, no atomics
#pragma unroll
  for (int k = 0; k < NSUM; ++k) {
    if (A.slot[k] < 0) continue;
    float *__restrict__ dst = A.partial + ((size_t)blockIdx.x * A.nsum + A.slot[k]) * c;
    if (PARTS == 1) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) M::template store<float, false>(dst, 0, lane, i, c, acc[k][i], c - M::first(lane, i));
      continue;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float a = acc[k][i][j];
#pragma unroll
        for (int d = LPR; d < 64; d <<= 1) a += __shfl_xor(a, d);
        if (LPR > 64 || (threadIdx.x & 63) < LPR) s_col[(LPR > 64 ? sub : threadIdx.x >> 6) * WIDTH + M::column(lane, i, j)] = a;
      }
    __syncthreads();
    for (int i = threadIdx.x; i < c; i += THREADS) {
      float s = s_col[i];
#pragma unroll
      for (int q = 1; q < PARTS; ++q) s += s_col[q * WIDTH + i];
      dst[i] = s;
    }
    __syncthreads();
  }
}

// lanes per row and chunks per lane (the rule that picks one: rn_shape in resnorm.hip)
#define LS3D_RN_SIMPLE_WIDE(GO) GO(16, 2) GO(32, 2) GO(64, 2) GO(128, 2) GO(256, 2) GO(512, 2)
#define LS3D_RN_SIMPLE(GO) GO(4, 1) GO(4, 2) GO(4, 3) GO(8, 2) LS3D_RN_SIMPLE_WIDE(GO)
#define LS3D_RN_FULL_WIDE(GO) GO(16, 1) GO(32, 1) GO(64, 1) GO(128, 1) GO(256, 1) GO(512, 1) GO(1024, 1)
#define LS3D_RN_FULL(GO) GO(4, 1) GO(8, 1) LS3D_RN_FULL_WIDE(GO)

template <typename TX, typename TR>
static bool ls3d_rn_launch_types(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream) {
#define LS3D_RN_GO(L_, V_, F_, NT_)                                                                                                                        \
  if (lpr == L_ && vpt == V_) {                                                                                                                            \
    if (fwd) hipLaunchKernelGGL((k_resnorm_fwd<TX, TR, L_, V_, F_, NT_>), dim3((unsigned)blocks), dim3(ls3d_rn_threads<L_>()), 0, stream, a);              \
    else hipLaunchKernelGGL((k_resnorm_bwd<TX, TR, L_, V_, F_, NT_>), dim3((unsigned)blocks), dim3(ls3d_rn_threads<L_>()), 0, stream, a);                  \
    return true;                                                                                                                                           \
  }
#define LS3D_RN_GO_SIMPLE(L_, V_) LS3D_RN_GO(L_, V_, false, false)
#define LS3D_RN_GO_FULL(L_, V_) LS3D_RN_GO(L_, V_, true, false)
#define LS3D_RN_GO_SIMPLE_NT(L_, V_) LS3D_RN_GO(L_, V_, false, true)
#define LS3D_RN_GO_FULL_NT(L_, V_) LS3D_RN_GO(L_, V_, true, true)
  if constexpr (sizeof(TX) == sizeof(TR)) {
    if (nt && full) { LS3D_RN_FULL_WIDE(LS3D_RN_GO_FULL_NT) }
    else if (nt) { LS3D_RN_SIMPLE_WIDE(LS3D_RN_GO_SIMPLE_NT) }
  }
  if (full) { LS3D_RN_FULL(LS3D_RN_GO_FULL) }
  else { LS3D_RN_SIMPLE(LS3D_RN_GO_SIMPLE) }
#undef LS3D_RN_GO_FULL_NT
#undef LS3D_RN_GO_SIMPLE_NT
#undef LS3D_RN_GO_FULL
#undef LS3D_RN_GO_SIMPLE
#undef LS3D_RN_GO
  return false;
}

bool ls3d_rn_launch_f32(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream);
bool ls3d_rn_launch_bf16(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream);
bool ls3d_rn_launch_f16(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream);
bool ls3d_rn_launch_bf16_f32(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream);
bool ls3d_rn_launch_f16_f32(bool fwd, bool full, bool nt, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream);
