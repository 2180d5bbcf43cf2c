// resnorm.hip — entry points of the residual-norm kernels (resnorm.h): argument checks, the launch rule, the reduction of the column sums.
#include "resnorm.h"

constexpr int RN_MAX_C = 8192;      // 512 lanes x 2 chunks of 8 columns, 1024 x 1
constexpr long long RN_NT_BYTES = 256ll << 20;
constexpr int RN_BWD_BLOCKS = 512;  // workgroups of a backward pass: two per CU; each writes one row of column sums

// lanes and chunks per lane of a row: few lanes (few exchanges a sum, more rows a wave), two chunks each, three where that fills four lanes.  With a norm before or
// a gate (`full`) one chunk: its five column sums and four parameters are 72 registers a chunk, and with two the backward pass spills.
static inline void rn_shape(int c, bool full, int *lpr, int *vpt) {
  const int chunks = (c + 7) / 8;
  *lpr = 4;
  *vpt = full ? 1 : chunks <= 12 ? (chunks + 3) / 4 : 2;
  if (*vpt < 1) *vpt = 1;
  while (*lpr * *vpt < chunks) *lpr *= 2;
}

static inline int rn_rows(int lpr) { return lpr >= 256 ? 1 : 256 / lpr; }  // rows of a workgroup

static inline int rn_bwd_blocks(int n, int lpr) {
  const long long b = ((long long)n + rn_rows(lpr) - 1) / rn_rows(lpr);
  return (int)(b < 1 ? 1 : b < RN_BWD_BLOCKS ? b : RN_BWD_BLOCKS);
}

// out[k][c] = sum over the blocks' partial rows, for each wanted sum k: 32 columns a workgroup, 32 row groups that each add every 32nd block in order, eight loads in
// flight (with 8 groups and one load after the other: 18 us for 512 blocks, all latency), then the groups in order
struct rn_outs { void *p[5]; int type[5]; int slot[5]; };
__global__ __launch_bounds__(1024) void k_resnorm_columns(const float *__restrict__ partial, int nblocks, int nsum, int c, rn_outs o) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane, slot = blockIdx.y;
  const float *__restrict__ src = partial + (size_t)slot * c + (col < c ? col : 0);
  float s = 0.0f;
  for (int b = grp; b < nblocks; b += 256) {
    float v[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = src[(size_t)(b + 32 * q < nblocks ? b + 32 * q : 0) * nsum * c];
#pragma unroll
    for (int q = 0; q < 8; ++q) s += b + 32 * q < nblocks ? v[q] : 0.0f;
  }
  red[grp][lane] = s;
  __syncthreads();
  if (grp == 0 && col < c) {
    s = 0.0f;
#pragma unroll
    for (int q = 0; q < 32; ++q) s += red[q][lane];
#pragma unroll
    for (int k = 0; k < 5; ++k)
      if (o.slot[k] == slot) ls3d_param_store(o.p[k], o.type[k], col, s);
  }
}

static inline bool rn_aligned(const void *p, int dtype) { return ((uintptr_t)p & (ls3d_dtype_size(dtype) - 1)) == 0; }

// the part of a descriptor that forward and backward read alike
static int rn_fill(const ls3d_residual_norm_t *d, const void *x, long long x_ld, const void *res, long long res_ld, int n, int c, ls3d_rn_args *a) {
  if (!d || n < 0 || c < 0 || !ls3d_dtype_ok(d->dtype) || !ls3d_dtype_ok(d->stream_dtype)) return LS3D_ERR_ARG;
  if (d->stream_dtype != d->dtype && d->stream_dtype != LS3D_DTYPE_F32) return LS3D_ERR_UNSUPPORTED;
  for (const ls3d_norm_t *m : {&d->in, &d->out}) {
    if (m->kind != LS3D_NORM_NONE && m->kind != LS3D_NORM_LAYER && m->kind != LS3D_NORM_RMS) return LS3D_ERR_ARG;
    if ((m->weight && (!ls3d_dtype_ok(m->weight_dtype) || !rn_aligned(m->weight, m->weight_dtype))) ||
        (m->bias && (!ls3d_dtype_ok(m->bias_dtype) || !rn_aligned(m->bias, m->bias_dtype))))
      return LS3D_ERR_ARG;
    if (m->kind && !(m->eps >= 0.0f)) return LS3D_ERR_ARG;
  }
  if (d->gate_kind != LS3D_GATE_NONE && d->gate_kind != LS3D_GATE_CHANNEL && d->gate_kind != LS3D_GATE_FULL) return LS3D_ERR_ARG;
  if (d->gate_kind && (!ls3d_dtype_ok(d->gate_dtype) || (d->gate_kind == LS3D_GATE_FULL && d->gate_dtype != d->dtype))) return LS3D_ERR_ARG;
  if (!ls3d_dropout_threshold(d->p, &a->thr, &a->inv)) return LS3D_ERR_ARG;
  if (c > RN_MAX_C) return LS3D_ERR_UNSUPPORTED;
  if (n == 0 || c == 0) return LS3D_OK;
  if (!x || x_ld < c || !rn_aligned(x, d->dtype) || (res && (res_ld < c || !rn_aligned(res, d->stream_dtype)))) return LS3D_ERR_ARG;
  if (d->gate_kind && (!d->gate || !rn_aligned(d->gate, d->gate_dtype) || (d->gate_kind == LS3D_GATE_FULL && d->gate_ld < c))) return LS3D_ERR_ARG;
  if (a->thr && (!d->state || ((uintptr_t)d->state & 7))) return LS3D_ERR_ARG;
  a->x = x; a->x_ld = (size_t)x_ld;
  a->res = res; a->res_ld = (size_t)res_ld;
  a->gate = d->gate; a->gate_kind = d->gate_kind; a->gate_t = d->gate_dtype; a->gate_ld = (size_t)d->gate_ld;
  a->n = n; a->c = c;
  a->kind_in = d->in.kind; a->w_in = d->in.weight; a->b_in = d->in.bias; a->w_in_t = d->in.weight_dtype; a->b_in_t = d->in.bias_dtype; a->eps_in = d->in.eps;
  a->kind_out = d->out.kind; a->w_out = d->out.weight; a->b_out = d->out.bias; a->w_out_t = d->out.weight_dtype; a->b_out_t = d->out.bias_dtype; a->eps_out = d->out.eps;
  a->share = 1.0f;
  while ((float)c * a->share > 1.0f) a->share *= 0.5f;
  a->whole = (float)c * a->share;
  a->alpha = d->alpha; a->state = d->state; a->call = d->call;
  return LS3D_OK;
}

// Non-temporal accesses where a pass moves more than any cache keeps until the next one (256 MB) and every access of a wave covers whole lines of a row: 16 lanes or
// more, and no f32 rows beside 2-byte ones.  Measured, without / with: 100000 x 256 f32 208 / 191 us forward and backward, 16384 x 4096 bf16 forward 110 / 103 (100
// on up to 16384 workgroups instead of 2048); narrower rows, 360000 x 96: f32 226 / 233, bf16 125 / 136; under 256 MB, 16384 x 1024 bf16: 74 / 77.
static inline bool rn_streams(const ls3d_residual_norm_t *d, int lpr, long long elems, int of_x, int of_stream) {
  const long long bytes = elems * ((long long)ls3d_dtype_size(d->dtype) * of_x + (long long)ls3d_dtype_size(d->stream_dtype) * of_stream);
  return d->dtype == d->stream_dtype && lpr >= 16 && bytes > RN_NT_BYTES;
}

static bool rn_launch(bool fwd, bool full, bool nt, int dtype, int stream_dtype, const ls3d_rn_args &a, int lpr, int vpt, int blocks, hipStream_t stream) {
  if (dtype == LS3D_DTYPE_F32) return ls3d_rn_launch_f32(fwd, full, nt, a, lpr, vpt, blocks, stream);
  if (dtype == LS3D_DTYPE_BF16)
    return stream_dtype == LS3D_DTYPE_F32 ? ls3d_rn_launch_bf16_f32(fwd, full, nt, a, lpr, vpt, blocks, stream) : ls3d_rn_launch_bf16(fwd, full, nt, a, lpr, vpt, blocks, stream);
  return stream_dtype == LS3D_DTYPE_F32 ? ls3d_rn_launch_f16_f32(fwd, full, nt, a, lpr, vpt, blocks, stream) : ls3d_rn_launch_f16(fwd, full, nt, a, lpr, vpt, blocks, stream);
}

extern "C" int ls3d_residual_norm_forward(const void *x, long long x_ld, const void *residual, long long res_ld, int n, int c, const ls3d_residual_norm_t *d,
                                          void *y, void *sum, float *stats, ls3d_stream_t stream) {
  ls3d_rn_args a = {};
  const int rc = rn_fill(d, x, x_ld, residual, res_ld, n, c, &a);
  if (rc != LS3D_OK || n == 0 || c == 0) return rc;
  if ((a.kind_out && !y) || (!a.kind_out && !sum) || ((uintptr_t)stats & 15) || (y && !rn_aligned(y, d->dtype)) || (sum && !rn_aligned(sum, d->stream_dtype)))
    return LS3D_ERR_ARG;
  a.y = y; a.s = sum; a.stats = stats;
  int lpr, vpt;
  const bool full = a.kind_in || a.gate_kind;
  rn_shape(c, full, &lpr, &vpt);
  const bool nt = rn_streams(d, lpr, (long long)n * c, 1 + (a.y != nullptr) + (a.gate_kind == LS3D_GATE_FULL), (a.res != nullptr) + (a.s != nullptr));
  const int rows = rn_rows(lpr);
  if (!rn_launch(true, full, nt, d->dtype, d->stream_dtype, a, lpr, vpt, (int)ls3d_grid(((long long)n + rows - 1) / rows, 1, nt ? 16384 : 2048).x, (hipStream_t)stream)) return LS3D_ERR_UNSUPPORTED;
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}

extern "C" size_t ls3d_residual_norm_workspace_bytes(int n, int c) {
  if (n < 0 || c < 0 || c > RN_MAX_C) return 0;
  int lpr, vpt;
  int blocks = 0;  // of the shape with the fewest rows a workgroup
  for (int full = 0; full < 2; ++full) {
    rn_shape(c, full != 0, &lpr, &vpt);
    const int b = rn_bwd_blocks(n, lpr);
    blocks = b > blocks ? b : blocks;
  }
  return (size_t)blocks * 5 * c * sizeof(float) + 256;
}

extern "C" int ls3d_residual_norm_backward(const void *x, long long x_ld, const void *residual, long long res_ld, int n, int c, const ls3d_residual_norm_t *d,
                                           const float *stats, const void *dy, long long dy_ld, const void *ds, long long ds_ld, void *dx, void *dresidual,
                                           void *dgate, void *dw_in, void *db_in, void *dw_out, void *db_out, void *workspace, size_t workspace_bytes,
                                           ls3d_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  ls3d_rn_args a = {};
  const int rc = rn_fill(d, x, x_ld, residual, res_ld, n, c, &a);
  if (rc != LS3D_OK || c == 0) return rc;
  // column sums in the order of ls3d_rn_args::slot; a sum without a place to go is not formed
  const bool chan = d->gate_kind == LS3D_GATE_CHANNEL;
  rn_outs o = {{dw_out, db_out, dw_in, db_in, chan ? dgate : nullptr},
               {d->out.weight_dtype, d->out.bias_dtype, d->in.weight_dtype, d->in.bias_dtype, d->gate_dtype}, {-1, -1, -1, -1, -1}};
  const int kinds[5] = {d->out.kind, d->out.kind, d->in.kind, d->in.kind, chan ? 1 : 0};
  int nsum = 0;
  for (int k = 0; k < 5; ++k) {
    if (o.p[k] && (!kinds[k] || !ls3d_dtype_ok(o.type[k]) || !rn_aligned(o.p[k], o.type[k]))) return LS3D_ERR_ARG;
    if (o.p[k]) o.slot[k] = nsum++;
  }
  if (nsum && (!workspace || ((uintptr_t)workspace & 15))) return LS3D_ERR_ARG;
  if (nsum && workspace_bytes < ls3d_residual_norm_workspace_bytes(n, c)) return LS3D_ERR_WORKSPACE;
  int blocks = 0;
  if (n > 0) {
    if ((!dy && !ds) || (dy && !a.kind_out) || (dy && (dy_ld < c || !rn_aligned(dy, d->dtype))) || (ds && (ds_ld < c || !rn_aligned(ds, d->stream_dtype))) ||
        !stats || ((uintptr_t)stats & 15) || (dx && !rn_aligned(dx, d->dtype)) || (dresidual && (!residual || !rn_aligned(dresidual, d->stream_dtype))) ||
        (dgate && (!d->gate_kind || !rn_aligned(dgate, d->gate_dtype))))
      return LS3D_ERR_ARG;
    a.stats = const_cast<float *>(stats);
    a.dy = dy; a.dy_ld = (size_t)dy_ld;
    a.ds = ds; a.ds_ld = (size_t)ds_ld;
    a.dx = dx; a.dres = dresidual; a.dgate = d->gate_kind == LS3D_GATE_FULL ? dgate : nullptr;
    a.partial = (float *)workspace;
    a.nsum = nsum;
    for (int k = 0; k < 5; ++k) a.slot[k] = o.slot[k];
    int lpr, vpt;
    const bool full = a.kind_in || a.gate_kind;
    rn_shape(c, full, &lpr, &vpt);
    const bool nt = rn_streams(d, lpr, (long long)n * c, 1 + (dy != nullptr) + (dx != nullptr) + (a.gate_kind == LS3D_GATE_FULL) + (a.dgate != nullptr),
                      (a.res != nullptr) + (ds != nullptr) + (dresidual != nullptr));
    blocks = rn_bwd_blocks(n, lpr);
    if (!rn_launch(false, full, nt, d->dtype, d->stream_dtype, a, lpr, vpt, blocks, stream)) return LS3D_ERR_UNSUPPORTED;
  }
  if (nsum) hipLaunchKernelGGL(k_resnorm_columns, dim3((unsigned)((c + 31) / 32), (unsigned)nsum), dim3(1024), 0, stream, (const float *)workspace, blocks, nsum, c, o);
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}
