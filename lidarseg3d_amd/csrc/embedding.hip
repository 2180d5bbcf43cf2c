// embedding.hip — row lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[i] = scale * sum_k weight[i][k] * table[idx[i][k]]          (no weights: 1)
//   backward  dtable[v] = scale * sum over the entries e = (i, k) with idx = v of weight[e] * dout[i], entries in input order;
//             dweight[i][k] = scale * <dout[i], table[idx[i][k]]>
// An index outside [0, rows) names no row: it adds nothing and takes no gradient.  Sums in f32, rounded to the table's type once.
//
// The gradient: the entries are sorted by row (stable), cut into tiles of `tile` entries, and a group of lanes walks each tile, adding up dout rows as
// long as the table row stays the same.  A row whose entries lie within one tile is written at once; one that crosses tiles leaves a partial sum
// per tile, which k_emb_join adds in order.  So the work per group is the same whether every token is another one or all are the same, and the
// order of the additions is fixed: no atomics, the same bits every time.  Rows without entries: the table's gradient is cleared first.
// Bound by memory: n rows of dout in, the whole gradient table out.
#include "blocks_common.h"

int ls3d_radix_sort_pairs(const uint32_t *keys_in, const int32_t *vals_in, int n, const int32_t *n_dev, int bits, uint32_t *keys_out, int32_t *vals_out,
                          void *workspace, size_t workspace_bytes, hipStream_t stream);

__device__ __forceinline__ long long emb_index(const void *__restrict__ idx, int is64, size_t e) {
  return is64 ? ((const long long *)idx)[e] : (long long)((const int32_t *)idx)[e];
}

// one chunk of 8 columns of one output row per thread and trip
template <typename T>
__global__ __launch_bounds__(256) void k_emb_fwd(const T *__restrict__ table, size_t table_ld, long long rows, int c, const void *__restrict__ idx, int is64, int n, int k,
                                                 const float *__restrict__ weight, float scale, T *__restrict__ out) {
  const uint32_t groups = (uint32_t)(c + 7) / 8;
  const long long total = (long long)n * groups;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
    const uint32_t i = (uint32_t)(t / groups), g = (uint32_t)(t - (long long)i * groups);
    const int col = (int)g * 8, m = c - col;
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
    for (int q = 0; q < k; ++q) {
      const size_t e = (size_t)i * k + q;
      const long long v = emb_index(idx, is64, e);
      if (v < 0 || v >= rows) continue;
      const float w = weight ? weight[e] : 1.0f;
      float r[8];
      ls3d_unpack8<T>(ls3d_load8<T>(table + (size_t)v * table_ld, col, c), m, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = weight ? fmaf(w, r[j], acc[j]) : acc[j] + r[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= scale;
    ls3d_store8<T>(out + (size_t)i * c + col, acc, m);
  }
}

// sort keys (the table row; `rows` for an entry without one) and the cleared gradient
template <typename T>
__global__ __launch_bounds__(256) void k_emb_keys(const void *__restrict__ idx, int is64, int entries, long long rows, long long padding, uint32_t *__restrict__ keys,
                                                  T *__restrict__ dtable, size_t elems) {
  const size_t t0 = (size_t)blockIdx.x * 256 + threadIdx.x, step = (size_t)gridDim.x * 256;
  for (size_t e = t0; e < (size_t)entries; e += step) {
    const long long v = emb_index(idx, is64, e);
    keys[e] = (uint32_t)(v < 0 || v >= rows || v == padding ? rows : v);
  }
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (size_t g = t0; g * 8 < elems; g += step) ls3d_store8<T>(dtable + g * 8, zero, elems - g * 8 < 8 ? (int)(elems - g * 8) : 8);
}

// grid (groups of tiles, column slabs): `lpr` lanes per tile, a chunk of 8 columns each
template <typename T>
__global__ __launch_bounds__(256) void k_emb_tiles(const uint32_t *__restrict__ keys, const int32_t *__restrict__ order, int entries, int tile, int lpr, long long rows, int c,
                                                   int k, const float *__restrict__ weight, float scale, const T *__restrict__ dout, size_t dout_ld,
                                                   T *__restrict__ dtable, float *__restrict__ partial) {
  const int lane = threadIdx.x % lpr, per = 256 / lpr;
  const long long j = (long long)blockIdx.x * per + threadIdx.x / lpr;
  const long long lo = j * tile;
  const int col = ((int)blockIdx.y * lpr + lane) * 8, m = c - col;
  if (lo >= entries || m <= 0) return;
  const int hi = lo + tile < entries ? (int)(lo + tile) : entries;
  uint32_t cur = keys[lo];
  bool from_before = lo > 0 && keys[lo - 1] == cur;  // the open row began in an earlier tile
  float acc[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
  for (int e = (int)lo; e < hi; ++e) {
    const uint32_t key = keys[e];
    if (key != cur) {
      if (cur < (uint32_t)rows) {
        if (from_before) ls3d_store8<float>(partial + ((size_t)j * 2) * c + col, acc, m);
        else {
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] *= scale;
          ls3d_store8<T>(dtable + (size_t)cur * c + col, acc, m);
        }
      }
      cur = key;
      from_before = false;
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
    }
    if (key >= (uint32_t)rows) break;  // sorted: entries without a row come last
    const int ent = order[e];
    float g[8];
    ls3d_unpack8<T>(ls3d_load8<T>(dout + (size_t)(k == 1 ? ent : ent / k) * dout_ld, col, c), m, g);
    const float w = weight ? weight[ent] : 1.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = fmaf(w, g[q], acc[q]);
  }
  if (cur >= (uint32_t)rows) return;
  const bool goes_on = hi < entries && keys[hi] == cur;
  if (from_before) ls3d_store8<float>(partial + ((size_t)j * 2) * c + col, acc, m);
  else if (goes_on) ls3d_store8<float>(partial + ((size_t)j * 2 + 1) * c + col, acc, m);
  else {
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] *= scale;
    ls3d_store8<T>(dtable + (size_t)cur * c + col, acc, m);
  }
}

// a workgroup for each tile in which a row begins that goes on in the next one: partial[j][1] + partial[j + 1][0] + ... while the tiles begin with that row.
// `lpr` lanes per partial row, the 256 / lpr groups take the tiles in turn (one wave walking the 700 tiles of a row one after the other took 210 us), their
// sums are added in order.
template <typename T>
__global__ __launch_bounds__(256) void k_emb_join(const uint32_t *__restrict__ keys, int entries, int tile, int ntiles, int lpr, long long rows, int c, float scale,
                                                  const float *__restrict__ partial, T *__restrict__ dtable) {
  __shared__ float s_sum[256][9];
  const int j = (int)blockIdx.x;
  const long long hi = (long long)(j + 1) * tile;
  const uint32_t cur = keys[hi - 1];
  if (cur >= (uint32_t)rows || keys[hi] != cur) return;  // nothing goes on (uniform over the workgroup, like the next line)
  if (j > 0 && keys[hi - tile] == cur && keys[hi - tile - 1] == cur) return;  // it began in an earlier tile
  int last = j + 1;  // the last tile that begins with this row: sorted keys, so those that do are the first of any run of tiles
  for (;;) {
    const long long t = (long long)last + 1 + threadIdx.x;
    const int on = __syncthreads_count(t < ntiles && keys[t < ntiles ? t * tile : 0] == cur);
    last += on;
    if (on < 256) break;
  }
  const int lane = (int)threadIdx.x % lpr, grp = (int)threadIdx.x / lpr, ngrp = 256 / lpr;
  const int col = ((int)blockIdx.y * lpr + lane) * 8, m = c - col;
  float acc[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
  if (m > 0) {
#pragma unroll 4
    for (int t = j + 1 + grp; t <= last; t += ngrp) {
      float p[8];
      ls3d_unpack8<float>(ls3d_load8<float>(partial + ((size_t)t * 2) * c, col, c), m, p);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += p[q];
    }
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) s_sum[threadIdx.x][q] = acc[q];
  __syncthreads();
  if (grp == 0 && m > 0) {
    ls3d_unpack8<float>(ls3d_load8<float>(partial + ((size_t)j * 2 + 1) * c, col, c), m, acc);
    for (int g = 0; g < ngrp; ++g)
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += s_sum[g * lpr + lane][q];
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] *= scale;
    ls3d_store8<T>(dtable + (size_t)cur * c + col, acc, m);
  }
}

// dweight: a wave per output row, its dout row read once per 512 columns and entry
template <typename T>
__global__ __launch_bounds__(256) void k_emb_dweight(const T *__restrict__ table, size_t table_ld, long long rows, int c, const void *__restrict__ idx, int is64, int n, int k,
                                                     float scale, const T *__restrict__ dout, size_t dout_ld, float *__restrict__ dweight) {
  const int lane = threadIdx.x & 63;
  for (long long e = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); e < (long long)n * k; e += (long long)gridDim.x * 4) {
    const long long v = emb_index(idx, is64, (size_t)e);
    float s = 0.0f;
    if (v >= 0 && v < rows) {
      const size_t i = (size_t)(e / k);
      for (int col = lane * 8; col < c; col += 512) {
        float a[8], b[8];
        ls3d_unpack8<T>(ls3d_load8<T>(table + (size_t)v * table_ld, col, c), c - col, a);
        ls3d_unpack8<T>(ls3d_load8<T>(dout + i * dout_ld, col, c), c - col, b);
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fmaf(a[q], b[q], s);
      }
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0) dweight[e] = s * scale;
  }
}

static int emb_check(const void *table, long long table_ld, long long rows, int c, int dtype, const void *idx, int idx_dtype, int n, int k, const float *weight) {
  if (rows < 0 || rows > 0x7FFFFFFEll || c < 0 || n < 0 || k < 1 || !ls3d_dtype_ok(dtype) || (idx_dtype != LS3D_INDEX_I32 && idx_dtype != LS3D_INDEX_I64)) return LS3D_ERR_ARG;
  if ((long long)n * k > 0x3FFFFFFFll) return LS3D_ERR_UNSUPPORTED;
  if (n == 0 || c == 0) return LS3D_OK;
  if (!idx || ((uintptr_t)idx & (idx_dtype == LS3D_INDEX_I64 ? 7 : 3)) || ((uintptr_t)weight & 3)) return LS3D_ERR_ARG;
  if (rows && (!table || table_ld < c || ((uintptr_t)table & (ls3d_dtype_size(dtype) - 1)))) return LS3D_ERR_ARG;
  return LS3D_OK;
}

#define EMB_TYPES(dtype, CALL)                                    \
  do {                                                            \
    if ((dtype) == LS3D_DTYPE_F32) { typedef float T; CALL; }     \
    else if ((dtype) == LS3D_DTYPE_BF16) { typedef ls3d_bf16 T; CALL; } \
    else { typedef ls3d_f16 T; CALL; }                            \
  } while (0)

extern "C" int ls3d_embedding_forward(const void *table, long long table_ld, long long rows, int c, int dtype, const void *idx, int idx_dtype, int n, int k,
                                      const float *weight, float scale, void *out, ls3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int rc = emb_check(table, table_ld, rows, c, dtype, idx, idx_dtype, n, k, weight);
  if (rc != LS3D_OK || n == 0 || c == 0) return rc;
  if (!out || ((uintptr_t)out & (ls3d_dtype_size(dtype) - 1))) return LS3D_ERR_ARG;
  const dim3 grid = ls3d_grid((long long)n * ((c + 7) / 8));
  EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_fwd<T>), grid, dim3(256), 0, stream, (const T *)table, (size_t)table_ld, rows, c, idx, (int)(idx_dtype == LS3D_INDEX_I64), n, k,
                                      weight, scale, (T *)out));
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}

// entries per tile: about 2^18 lanes at work on the tiles of a large call, but no fewer than 16 entries
static inline int emb_tile(long long entries, int c) {
  const long long want = entries * ((c + 7) / 8) / 262144;
  int t = 16;
  while (t < want && t < 4096) t *= 2;
  return t;
}

extern "C" size_t ls3d_embedding_workspace_bytes(int n, int k, int c) {
  if (n < 0 || k < 1 || c < 0 || (long long)n * k > 0x3FFFFFFFll) return 0;
  const long long e = (long long)n * k;
  const int tile = emb_tile(e, c);
  const size_t part = (size_t)((e + tile - 1) / tile) * 2 * c * sizeof(float);
  return ((size_t)e * 4 + 255) / 256 * 256 * 3 + (part + 255) / 256 * 256 + ls3d_radix_sort_workspace_bytes((int)e) + 256;
}

extern "C" int ls3d_embedding_backward(const void *table, long long table_ld, long long rows, int c, int dtype, const void *idx, int idx_dtype, int n, int k,
                                       const float *weight, float scale, long long padding, const void *dout, long long dout_ld, void *dtable, float *dweight,
                                       void *workspace, size_t workspace_bytes, ls3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  int rc = emb_check(table, table_ld, dweight ? rows : 0, c, dtype, idx, idx_dtype, n, k, weight);
  if (rc == LS3D_OK && (rows < 0 || rows > 0x7FFFFFFEll)) rc = LS3D_ERR_ARG;
  if (rc != LS3D_OK) return rc;
  const size_t elem = ls3d_dtype_size(dtype);
  if ((n > 0 && c > 0 && (!dout || dout_ld < c || ((uintptr_t)dout & (elem - 1)))) || ((uintptr_t)dtable & (elem - 1)) || ((uintptr_t)dweight & 3)) return LS3D_ERR_ARG;
  const int is64 = idx_dtype == LS3D_INDEX_I64, entries = n * k, groups = (c + 7) / 8;
  if (dweight && entries > 0 && c > 0)
    EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_dweight<T>), ls3d_grid(entries, 4), dim3(256), 0, stream, (const T *)table, (size_t)table_ld, rows, c, idx, is64, n, k, scale,
                                        (const T *)dout, (size_t)dout_ld, dweight));
  if (dtable && rows > 0 && c > 0) {
    if (entries > 0 && (!workspace || ((uintptr_t)workspace & 15))) return LS3D_ERR_ARG;
    if (entries > 0 && workspace_bytes < ls3d_embedding_workspace_bytes(n, k, c)) return LS3D_ERR_WORKSPACE;
    const size_t seg = ((size_t)entries * 4 + 255) / 256 * 256;
    uint32_t *keys = (uint32_t *)workspace, *skeys = (uint32_t *)((char *)workspace + seg);
    int32_t *order = (int32_t *)((char *)workspace + 2 * seg);
    const int tile = emb_tile(entries, c), ntiles = (entries + tile - 1) / tile;
    float *partial = (float *)((char *)workspace + 3 * seg);
    const size_t part = ((size_t)ntiles * 2 * c * sizeof(float) + 255) / 256 * 256;
    void *sort_ws = (char *)workspace + 3 * seg + part;
    const size_t elems = (size_t)rows * c;
    const long long work = (long long)(elems / 8 + 1) > entries ? (long long)(elems / 8 + 1) : entries;
    EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_keys<T>), ls3d_grid(work), dim3(256), 0, stream, idx, is64, entries, rows, padding, keys, (T *)dtable, elems));
    if (entries > 0) {
      int bits = 1;
      while ((rows >> bits) != 0) ++bits;  // keys 0 .. rows
      rc = ls3d_radix_sort_pairs(keys, nullptr, entries, nullptr, bits, skeys, order, sort_ws, ls3d_radix_sort_workspace_bytes(entries), stream);
      if (rc != LS3D_OK) return rc;
      int lpr = 1;
      while (lpr < groups && lpr < 64) lpr *= 2;
      const dim3 grid((unsigned)((ntiles + 256 / lpr - 1) / (256 / lpr)), (unsigned)((groups + lpr - 1) / lpr));
      EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_tiles<T>), grid, dim3(256), 0, stream, (const uint32_t *)skeys, (const int32_t *)order, entries, tile, lpr, rows, c, k, weight,
                                          scale, (const T *)dout, (size_t)dout_ld, (T *)dtable, partial));
      if (ntiles > 1)
        EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_join<T>), dim3((unsigned)(ntiles - 1), grid.y), dim3(256), 0, stream, (const uint32_t *)skeys, entries, tile,
                                            ntiles, lpr, rows, c, scale, (const float *)partial, (T *)dtable));
    }
  }
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}
