// embedding.hip — row lookup with scaling, and its gradient by sorted tokens.
//
//   forward   out[i] = scale * sum_k weight[i][k] * table[idx[i][k]]          (no weights: 1)
//   backward  dtable[v] = scale * sum over the entries e = (i, k) with idx = v of weight[e] * dout[i], entries in input order;
//             dweight[i][k] = scale * <dout[i], table[idx[i][k]]>
// An index outside [0, rows) names no row: it adds nothing and takes no gradient.  Sums in f32, rounded to the table's type once.
//
// The gradient: the entries that name a row are sorted by it (stable), cut into tiles of `tile` entries, and a group of lanes walks each tile, adding up
// dout rows as long as the table row stays the same.  The group in whose tile a row begins finishes it, into the next tile if need be; only a row that
// covers a whole tile leaves a partial sum per tile, which k_emb_join adds in order.  So a group walks at most two tiles whether every token is another
// one or all are the same, and the order of the additions is fixed: no atomics on sums, the same bits every time.  Rows without entries: the table's
// gradient is cleared first.
// Bound by memory: dout rows in, the whole gradient table out; the sort moves 8 bytes an entry and pass.
#include "blocks_common.h"

__device__ __forceinline__ long long emb_index(const void *__restrict__ idx, int is64, size_t e) {
  return is64 ? ((const long long *)idx)[e] : (long long)((const int32_t *)idx)[e];
}

// One chunk of 8 columns of one output row per thread; I: 32 bits where the chunk count allows.  A lookup is a chain of two round trips (index, table row), so
// U entries of a row that sums several are kept in flight.  Up to 16384 workgroups, few trips a thread: with 2048, 360000 x 64 f32, k = 1 took 26.5 us instead of
// 24.8, and 360000 x 48 f32, k = 8 took 7 us longer (eight entries in flight are no faster than four).
template <typename T, typename I, int U>
__global__ __launch_bounds__(256) void k_emb_fwd(const T *__restrict__ table, size_t table_ld, long long rows, int c, const void *__restrict__ idx, int is64, I total, int k,
                                                 const float *__restrict__ weight, float scale, T *__restrict__ out) {
  const uint32_t groups = (uint32_t)(c + 7) / 8;
  for (I t = (I)blockIdx.x * 256 + threadIdx.x; t < total; t += (I)gridDim.x * 256) {
    const uint32_t i = (uint32_t)(t / groups), g = (uint32_t)(t - (I)i * groups);
    const int col = (int)g * 8, m = c - col;
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
    for (int q0 = 0; q0 < k; q0 += U) {
      long long v[U];
      float w[U];
      ls3d_raw8<T> r[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const size_t e = (size_t)i * k + (q0 + q < k ? q0 + q : k - 1);
        v[q] = emb_index(idx, is64, e);
        w[q] = weight ? weight[e] : 1.0f;
        if (q0 + q >= k) v[q] = -1;
      }
#pragma unroll
      for (int q = 0; q < U; ++q) {
        r[q] = ls3d_raw8<T>{};
        if (v[q] >= 0 && v[q] < rows) r[q] = ls3d_load8<T>(table + (size_t)v[q] * table_ld, col, c);
      }
#pragma unroll
      for (int q = 0; q < U; ++q) {
        if (v[q] < 0 || v[q] >= rows) continue;
        float x[8];
        ls3d_unpack8<T>(r[q], m, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = fmaf(w[q], x[j], acc[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] *= scale;
    ls3d_store8<T>(out + (size_t)i * c + col, acc, m);
  }
}

// ---- the entries sorted by table row: pairs (row, entry), stable, the entries without a row left out; *n_valid = how many there are.
//      LSD radix passes of up to 11 bits (a table of up to 4 M rows: two), the first one straight from the indices.
constexpr int ES_MAX_DIGITS = 2048;
// entries per thread of a 256-thread workgroup: 8, or 4 where that leaves CUs without one
static inline int es_items(long long entries) { return entries > 1048576 ? 8 : 4; }
static inline int es_tiles(long long entries) { return (int)((entries + 256 * es_items(entries) - 1) / (256 * es_items(entries))); }

struct emb_keys { const void *idx; int is64; long long rows, padding; };  // where an entry's row comes from in the first pass
__device__ __forceinline__ uint32_t emb_key(const emb_keys &K, size_t e) {  // 0xFFFFFFFF: no row
  const long long v = emb_index(K.idx, K.is64, e);
  return v < 0 || v >= K.rows || v == K.padding ? 0xFFFFFFFFu : (uint32_t)v;
}

// clears the gradient table, a share per workgroup (rides along with the launches that only read the indices)
template <typename T>
__device__ __forceinline__ void emb_clear(T *__restrict__ dtable, size_t elems, size_t t0, size_t step) {
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (size_t g = t0; g * 8 < elems; g += step) ls3d_store8<T>(dtable + g * 8, zero, elems - g * 8 < 8 ? (int)(elems - g * 8) : 8);
}

// per-workgroup digit counts -> hist[workgroup][digit]; FIRST: from the indices, and the gradient table is cleared by the same launch
template <typename T, bool FIRST, int ITEMS>
__global__ __launch_bounds__(256) void k_es_hist(emb_keys K, const uint2 *__restrict__ pairs, int entries, const int32_t *__restrict__ n_valid, int shift, int digits, int ntiles,
                                                 int32_t *__restrict__ hist, T *__restrict__ dtable, size_t elems) {
  __shared__ int s_h[ES_MAX_DIGITS];
  if ((int)blockIdx.x < ntiles) {
    const int N = FIRST ? entries : *n_valid;
    const long long lo = (long long)blockIdx.x * (256 * ITEMS);
    for (int d = threadIdx.x; d < digits; d += 256) s_h[d] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const long long e = lo + i * 256 + threadIdx.x;
      if (e < N) {
        const uint32_t key = FIRST ? emb_key(K, (size_t)e) : pairs[e].x;
        if (!FIRST || key != 0xFFFFFFFFu) atomicAdd(&s_h[(key >> shift) & (digits - 1)], 1);
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += 256) hist[(size_t)blockIdx.x * digits + d] = s_h[d];
  }
  if (FIRST) emb_clear<T>(dtable, elems, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
}

// hist[workgroup][digit] -> the digit's count in the workgroups before, totals[digit]: 16 digits x 64 segments of workgroups per workgroup
__global__ __launch_bounds__(1024) void k_es_scan(int32_t *__restrict__ hist, int ntiles, int digits, int32_t *__restrict__ totals) {
  __shared__ int s_seg[64][17];
  const int dig = threadIdx.x & 15, d = blockIdx.x * 16 + dig, seg = threadIdx.x >> 4, per = (ntiles + 63) / 64;
  const int lo = seg * per, hi = lo + per < ntiles ? lo + per : ntiles;
  const bool on = d < digits;
  int s = 0;
  for (int b = lo; b < hi; b += 16) {
    int v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = on && b + q < hi ? hist[(size_t)(b + q) * digits + d] : 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) s += v[q];
  }
  s_seg[seg][dig] = s;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int q = 0; q < 64; ++q) {
    const int x = s_seg[q][dig];
    before += q < seg ? x : 0;
    total += x;
  }
  for (int b = lo; b < hi; b += 16) {
    int v[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = on && b + q < hi ? hist[(size_t)(b + q) * digits + d] : 0;
#pragma unroll
    for (int q = 0; q < 16; ++q)
      if (on && b + q < hi) { hist[(size_t)(b + q) * digits + d] = before; before += v[q]; }
  }
  if (on && seg == 0) totals[d] = total;
}

// lanes of the wave that hold a live item with this lane's digit
__device__ __forceinline__ unsigned long long emb_peers(bool live, uint32_t d, int bits) {
  unsigned long long peers = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long m = __ballot((d >> b) & 1u);
    peers &= ((d >> b) & 1u) ? m : ~m;
  }
  return peers;
}

// exclusive sums of v over the workgroup's 64 * W threads, in thread order; *total: their sum (s_w: W ints)
template <int W>
__device__ __forceinline__ int emb_block_scan(int v, int *s_w, int *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(s, d);
    s += lane >= d ? u : 0;
  }
  if (lane == 63) s_w[wave] = s;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    before += w < wave ? s_w[w] : 0;
    sum += s_w[w];
  }
  *total = sum;
  return before + s - v;
}

// places a tile's items: a wave takes 64 * ITEMS consecutive ones, 64 at a time; an item's rank among its wave's equal digits from ballots and a count per
// wave and digit, the waves' and workgroups' shares on top.  Equal digits keep their order.
template <bool FIRST, int ITEMS>
__global__ __launch_bounds__(256) void k_es_scatter(emb_keys K, const uint2 *__restrict__ pairs, int entries, int32_t *__restrict__ n_valid, int shift, int digits, int bits,
                                                    const int32_t *__restrict__ hist, const int32_t *__restrict__ totals, uint2 *__restrict__ out) {
  __shared__ int s_cnt[4][ES_MAX_DIGITS];
  __shared__ int s_w[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int N = FIRST ? entries : *n_valid;
  const long long lo = (long long)blockIdx.x * (256 * ITEMS);
  if (lo >= N) return;  // (the first pass: every workgroup has items)
  for (int d = threadIdx.x; d < digits; d += 256) s_cnt[0][d] = s_cnt[1][d] = s_cnt[2][d] = s_cnt[3][d] = 0;
  uint2 item[ITEMS];
  int rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const long long e = lo + (wave * ITEMS + i) * 64 + lane;
    item[i].x = 0xFFFFFFFFu;
    item[i].y = (unsigned)e;
    if (e < N) {
      if (FIRST) item[i].x = emb_key(K, (size_t)e);
      else item[i] = pairs[e];
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool live = item[i].x != 0xFFFFFFFFu;
    const uint32_t d = (item[i].x >> shift) & (uint32_t)(digits - 1);
    const unsigned long long peers = emb_peers(live, d, bits);
    const int before = __popcll(peers & ((1ull << lane) - 1ull));
    rank[i] = before + (live ? s_cnt[wave][d] : 0);
    LS3D_WAVE_SYNC();
    if (live && before == 0) s_cnt[wave][d] += __popcll(peers);
    LS3D_WAVE_SYNC();
  }
  __syncthreads();
  // where each digit starts: the digits below in all workgroups, the digit itself in the workgroups and waves before
  const int per = (digits + 255) / 256, d0 = (int)threadIdx.x * per;
  int mine = 0, total;
  for (int q = 0; q < per; ++q) mine += d0 + q < digits ? totals[d0 + q] : 0;
  int base = emb_block_scan<4>(mine, s_w, &total);
  for (int q = 0; q < per; ++q) {
    const int d = d0 + q;
    if (d >= digits) break;
    int s = base + hist[(size_t)blockIdx.x * digits + d];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int x = s_cnt[w][d];
      s_cnt[w][d] = s;
      s += x;
    }
    base += totals[d];
  }
  if (FIRST && blockIdx.x == 0 && threadIdx.x == 0) *n_valid = total;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (item[i].x != 0xFFFFFFFFu) out[s_cnt[wave][(item[i].x >> shift) & (uint32_t)(digits - 1)] + rank[i]] = item[i];
}

// few entries (<= 1024 * ITEMS): workgroup 0 sorts them all in LDS, 8 bits a pass, while the others clear the gradient table - one launch
template <typename T, int ITEMS>
__global__ __launch_bounds__(1024) void k_es_small(emb_keys K, int entries, int bits, int32_t *__restrict__ n_valid, uint2 *__restrict__ out, T *__restrict__ dtable, size_t elems) {
  HIP_DYNAMIC_SHARED(char, smem)
  uint2 *s_item = (uint2 *)smem;                                    // [1024 * ITEMS]
  int (*s_cnt)[256] = (int (*)[256])(smem + 1024 * ITEMS * sizeof(uint2));  // [16 waves][256 digits]
  __shared__ int s_w[16];
  if (blockIdx.x > 0 || gridDim.x == 1) {
    const size_t first = gridDim.x == 1 ? 0 : blockIdx.x - 1, others = gridDim.x == 1 ? 1 : gridDim.x - 1;
    emb_clear<T>(dtable, elems, first * 1024 + threadIdx.x, others * 1024);
    if (blockIdx.x > 0) return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint2 item[ITEMS];
  int rank[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int e = (wave * ITEMS + i) * 64 + lane;
    item[i].x = e < entries ? emb_key(K, (size_t)e) : 0xFFFFFFFFu;
    item[i].y = (unsigned)e;
  }
  int total = 0;
  for (int shift = 0; shift < bits; shift += 8) {
    for (int d = threadIdx.x; d < 16 * 256; d += 1024) s_cnt[d >> 8][d & 255] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool live = item[i].x != 0xFFFFFFFFu;
      const uint32_t d = (item[i].x >> shift) & 255u;
      const unsigned long long peers = emb_peers(live, d, 8);
      const int before = __popcll(peers & ((1ull << lane) - 1ull));
      rank[i] = before + (live ? s_cnt[wave][d] : 0);
      LS3D_WAVE_SYNC();
      if (live && before == 0) s_cnt[wave][d] += __popcll(peers);
      LS3D_WAVE_SYNC();
    }
    __syncthreads();
    int mine = 0;
    if (threadIdx.x < 256)
      for (int w = 0; w < 16; ++w) mine += s_cnt[w][threadIdx.x];
    int s = emb_block_scan<16>(mine, s_w, &total);
    if (threadIdx.x < 256)
      for (int w = 0; w < 16; ++w) {
        const int x = s_cnt[w][threadIdx.x];
        s_cnt[w][threadIdx.x] = s;
        s += x;
      }
    __syncthreads();
    uint2 *dst = shift + 8 >= bits ? out : s_item;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (item[i].x != 0xFFFFFFFFu) dst[s_cnt[wave][(item[i].x >> shift) & 255u] + rank[i]] = item[i];
    if (shift + 8 >= bits) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int e = (wave * ITEMS + i) * 64 + lane;
      item[i].x = 0xFFFFFFFFu;
      if (e < total) item[i] = s_item[e];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *n_valid = total;
}

// grid (groups of tiles, column slabs): `lpr` lanes per tile, a chunk of 8 columns each; U entries' rows in flight.
// A row is LONG where it covers a whole tile; the sums of a long row's tiles go to partial[tile][0 | 1] (0: it began in an earlier tile).  A row that
// begins in a tile and is not long is finished by that tile's group, and the next tile's group passes over its entries there.
template <typename T, int U>
__global__ __launch_bounds__(256) void k_emb_tiles(const uint2 *__restrict__ pairs, const int32_t *__restrict__ n_valid, int tile, int lpr, int c, int k,
                                                   const float *__restrict__ weight, float scale, const T *__restrict__ dout, size_t dout_ld,
                                                   T *__restrict__ dtable, float *__restrict__ partial) {
  const int lane = threadIdx.x % lpr, per = 256 / lpr, N = *n_valid;
  const long long j = (long long)blockIdx.x * per + threadIdx.x / lpr, lo = j * tile;
  const int col = ((int)blockIdx.y * lpr + lane) * 8, m = c - col;
  if (lo >= N || m <= 0) return;
  const int hi = lo + tile < N ? (int)(lo + tile) : N;
  auto row_at = [&](long long e) { return e >= 0 && e < N ? pairs[e].x : 0xFFFFFFFFu; };  // (behind either end: no row has this number)
  const uint32_t first = pairs[lo].x, last = pairs[hi - 1].x;
  const uint32_t b1 = row_at(lo - 1), b2 = row_at(lo - tile - 1), n0 = row_at(hi), n1 = row_at((long long)hi + tile);
  uint32_t cur = first;
  bool from_before = b1 == first;                             // the open row began in an earlier tile,
  bool skip = from_before && b2 != first && n0 != first;      // in the one before, whose group finishes it here (it covers neither that tile nor this one)
  const bool spills = n0 == last && (hi - lo == tile);        // the last row goes on in the next tile,
  const bool finish = spills && n1 != last && !(from_before && first == last);  // and ends there: this group goes after it
  float acc[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
  auto close = [&]() {  // the open row is complete
    if (!skip) {
      if (from_before) ls3d_store8<float>(partial + ((size_t)j * 2) * c + col, acc, m);
      else {
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] *= scale;
        ls3d_store8<T>(dtable + (size_t)cur * c + col, acc, m);
      }
    }
  };
  const int end = finish ? (hi + tile < N ? hi + tile : N) : hi;
  bool over = false;
  for (int e0 = (int)lo; e0 < end && !over; e0 += U) {
    uint2 pr[U];
    float w[U];
    ls3d_raw8<T> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) pr[u] = pairs[e0 + u < end ? e0 + u : end - 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = weight ? weight[pr[u].y] : 1.0f;
      r[u] = ls3d_load8<T>(dout + (size_t)(k == 1 ? pr[u].y : pr[u].y / (unsigned)k) * dout_ld, col, c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (e0 + u >= end || over) continue;
      if (pr[u].x != cur) {  // the same for every lane of the group
        if (e0 + u >= hi) { over = true; continue; }  // behind the tile: only the open row is followed
        close();
        cur = pr[u].x;
        from_before = skip = false;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
      }
      float g[8];
      ls3d_unpack8<T>(r[u], m, g);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = fmaf(w[u], g[q], acc[q]);
    }
  }
  if (spills && !finish && !from_before) ls3d_store8<float>(partial + ((size_t)j * 2 + 1) * c + col, acc, m);
  else close();
}

// The long rows: partial[j][1] + partial[j + 1][0] + ... from the tile j in which the row begins, while the tiles begin with it.  A workgroup looks at EJ_TILES
// tiles (few are such a j) and takes what it finds one after the other, all its threads together: `lpr` lanes per partial row, the 256 / lpr groups take the tiles in
// turn (one wave walking the 700 tiles of a row one after the other took 210 us), their sums are added in order.
constexpr int EJ_TILES = 16;  // at most; `span`: fewer where there are few tiles
template <typename T>
__global__ __launch_bounds__(256) void k_emb_join(const uint2 *__restrict__ pairs, const int32_t *__restrict__ n_valid, int tile, int span, int lpr, int c, float scale,
                                                  const float *__restrict__ partial, T *__restrict__ dtable) {
  __shared__ float s_sum[4][64][9];
  __shared__ int s_begin[EJ_TILES], s_rest;
  const int N = *n_valid;
  const long long j0 = (long long)blockIdx.x * span, mine = (j0 + threadIdx.x + 1) * tile;  // `mine`: where this thread's tile ends
  if (j0 * tile >= N) return;
  bool begins = false;
  if ((int)threadIdx.x < span && mine + tile < N) {  // a long row that begins in the tile covers the next one and goes on (or ends) behind it
    const uint32_t row = pairs[mine - 1].x;
    begins = pairs[mine].x == row && pairs[mine + tile].x == row && !(mine > tile && pairs[mine - tile].x == row && pairs[mine - tile - 1].x == row);
  }
  if ((int)threadIdx.x < span) s_begin[threadIdx.x] = begins;
  if (__syncthreads_count(begins) == 0) return;
  const int lane = (int)threadIdx.x % lpr, grp = (int)threadIdx.x / lpr, ngrp = 256 / lpr;
  const int col = ((int)blockIdx.y * lpr + lane) * 8, m = c - col;
  const int ntiles = (int)(((long long)N + tile - 1) / tile);
  for (int q0 = 0; q0 < span; ++q0) {
    if (!s_begin[q0]) continue;  // uniform
    const int j = (int)j0 + q0;
    const uint32_t cur = pairs[((long long)j + 1) * tile - 1].x;
    int last = j + 1;  // the last tile that begins with this row: sorted, so those that do are the first of any run of tiles
    for (;;) {  // 2048 tiles a step, a thread eight of them next to each other
      int on = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const long long t = (long long)last + 1 + threadIdx.x * 8 + u;
        on += t < ntiles && pairs[t < ntiles ? t * tile : 0].x == cur;
      }
      const int full = __syncthreads_count(on == 8), some = __syncthreads_count(on > 0);  // `some` threads, all but the last of them full
      last += full * 8;
      if (full == 256) continue;
      if (some > full && (int)threadIdx.x == full) s_rest = on;
      __syncthreads();
      if (some > full) last += s_rest;
      break;
    }
    float acc[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = 0.0f;
    if (m > 0) {
#pragma unroll 8
      for (int t = j + 1 + grp; t <= last; t += ngrp) {
        float p[8];
        ls3d_unpack8<float>(ls3d_load8<float>(partial + ((size_t)t * 2) * c, col, c), m, p);
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += p[q];
      }
    }
    // the wave's groups by lane exchange, the four waves through LDS, in order
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      for (int d = lpr; d < 64; d <<= 1) acc[q] += __shfl_xor(acc[q], d);
      s_sum[threadIdx.x >> 6][threadIdx.x & 63][q] = acc[q];
    }
    __syncthreads();
    if (grp == 0 && m > 0) {
      ls3d_unpack8<float>(ls3d_load8<float>(partial + ((size_t)j * 2 + 1) * c, col, c), m, acc);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = (acc[q] + ((s_sum[0][lane][q] + s_sum[1][lane][q]) + (s_sum[2][lane][q] + s_sum[3][lane][q]))) * scale;
      ls3d_store8<T>(dtable + (size_t)cur * c + col, acc, m);
    }
    __syncthreads();
  }
}

// dweight: `lpr` lanes per entry
template <typename T>
__global__ __launch_bounds__(256) void k_emb_dweight(const T *__restrict__ table, size_t table_ld, long long rows, int c, const void *__restrict__ idx, int is64, long long entries,
                                                     int k, int lpr, float scale, const T *__restrict__ dout, size_t dout_ld, float *__restrict__ dweight) {
  const int lane = threadIdx.x % lpr, per = 256 / lpr;
  for (long long e0 = (long long)blockIdx.x * per; e0 < entries; e0 += (long long)gridDim.x * per) {  // the same trips for every lane of a wave
    const long long e = e0 + threadIdx.x / lpr;
    const long long v = e < entries ? emb_index(idx, is64, (size_t)e) : -1;
    float s = 0.0f;
    if (v >= 0 && v < rows) {
      const size_t i = (size_t)(e / k);
      for (int col = lane * 8; col < c; col += lpr * 8) {
        float a[8], b[8];
        const ls3d_raw8<T> ra = ls3d_load8<T>(table + (size_t)v * table_ld, col, c), rb = ls3d_load8<T>(dout + i * dout_ld, col, c);
        ls3d_unpack8<T>(ra, c - col, a);
        ls3d_unpack8<T>(rb, c - col, b);
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fmaf(a[q], b[q], s);
      }
    }
    for (int d = lpr >> 1; d >= 1; d >>= 1) s += __shfl_xor(s, d);
    if (lane == 0 && e < entries) dweight[e] = s * scale;
  }
}

constexpr int EMB_MAX_C = 1 << 24;  // (a grid has at most 65535 slabs of 512 columns)
static int emb_check(const void *table, long long table_ld, long long rows, int c, int dtype, const void *idx, int idx_dtype, int n, int k, const float *weight) {
  if (rows < 0 || rows > 0x7FFFFFFEll || c < 0 || n < 0 || k < 1 || !ls3d_dtype_ok(dtype) || (idx_dtype != LS3D_INDEX_I32 && idx_dtype != LS3D_INDEX_I64)) return LS3D_ERR_ARG;
  if ((long long)n * k > 0x3FFFFFFFll || c > EMB_MAX_C) return LS3D_ERR_UNSUPPORTED;
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
  const long long total = (long long)n * ((c + 7) / 8);
  const int is64 = idx_dtype == LS3D_INDEX_I64;
#define EMB_FWD(I_, U_)                                                                                                                                                   \
  EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_fwd<T, I_, U_>), ls3d_grid(total, 256, 16384), dim3(256), 0, stream, (const T *)table, (size_t)table_ld, rows, c, idx, is64, (I_)total, k, \
                                      weight, scale, (T *)out))
  if (total < (1ll << 30)) {  // (the strides on top stay below 2^32)
    if (k == 1) EMB_FWD(uint32_t, 1);
    else EMB_FWD(uint32_t, 4);
  } else EMB_FWD(unsigned long long, 4);
#undef EMB_FWD
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}

// entries per tile: the lanes of a large call fill the card four times over even if two thirds of its entries name no row; 8 to 64 entries.  (360000 entries of 32
// rows x 64 f32: 19 us in tiles of 16, 39 in tiles of 64, where the join has a quarter of the partial sums and is 5 us shorter.)
static inline int emb_tile(long long entries, int c) {
  const long long want = entries * ((c + 7) / 8) / 262144;
  int t = 8;
  while (t < want && t < 64) t *= 2;
  return t;
}

// the sorting of a call: up to ES_SMALL entries in one workgroup, else radix passes of at most 11 bits, as even as they come
constexpr int ES_SMALL = 4096;
static inline int emb_passes(int bits) { return (bits + 10) / 11; }

struct emb_space { size_t pairs[2], partial, hist, totals, n_valid, bytes; };  // byte offsets in the workspace
static emb_space emb_layout(long long entries, int c) {
  emb_space s;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t p = at; at += (bytes + 255) / 256 * 256; return p; };
  const int tile = emb_tile(entries, c);
  s.n_valid = take(4);
  s.totals = take(ES_MAX_DIGITS * 4);
  s.pairs[0] = take((size_t)entries * 8);
  s.pairs[1] = take(entries > ES_SMALL ? (size_t)entries * 8 : 0);
  s.hist = take(entries > ES_SMALL ? (size_t)es_tiles(entries) * ES_MAX_DIGITS * 4 : 0);
  s.partial = take((size_t)((entries + tile - 1) / tile) * 2 * c * sizeof(float));
  s.bytes = at + 256;
  return s;
}

extern "C" size_t ls3d_embedding_workspace_bytes(int n, int k, int c) {
  if (n < 0 || k < 1 || c < 0 || (long long)n * k > 0x3FFFFFFFll) return 0;
  return emb_layout((long long)n * k, c).bytes;
}

template <typename T, int ITEMS>
static void emb_sort_small(const emb_keys &K, int entries, int bits, int32_t *n_valid, uint2 *out, T *dtable, size_t elems, hipStream_t stream) {
  const int lds = 1024 * ITEMS * (int)sizeof(uint2) + 16 * 256 * 4;
  static_assert(1024 * ITEMS * sizeof(uint2) + 16 * 256 * 4 <= 65536, "dynamic LDS without an opt-in");
  hipLaunchKernelGGL((k_es_small<T, ITEMS>), dim3(1 + ls3d_grid((long long)(elems / 8 + 1), 1024, 1024).x), dim3(1024), lds, stream, K, entries, bits, n_valid, out, dtable, elems);
}

// sorts the entries and clears the gradient table; -> the sorted pairs
template <typename T>
static const uint2 *emb_sort(const emb_keys &K, int entries, const emb_space &S, char *ws, T *dtable, size_t elems, hipStream_t stream) {
  int bits = 1;
  while (((K.rows - 1) >> bits) != 0) ++bits;
  int32_t *n_valid = (int32_t *)(ws + S.n_valid), *totals = (int32_t *)(ws + S.totals), *hist = (int32_t *)(ws + S.hist);
  uint2 *buf[2] = {(uint2 *)(ws + S.pairs[0]), (uint2 *)(ws + S.pairs[1])};
  if (entries <= ES_SMALL) {
    if (entries <= 1024) emb_sort_small<T, 1>(K, entries, bits, n_valid, buf[0], dtable, elems, stream);
    else emb_sort_small<T, 4>(K, entries, bits, n_valid, buf[0], dtable, elems, stream);
    return buf[0];
  }
  const int passes = emb_passes(bits), per = (bits + passes - 1) / passes, ntiles = es_tiles(entries), digits = 1 << per, items = es_items(entries);
  const unsigned clear = ls3d_grid((long long)(elems / 8 + 1)).x;
#define ES_PASS(FIRST_, ITEMS_, GRID_)                                                                                                                                  \
  do {                                                                                                                                                                  \
    hipLaunchKernelGGL((k_es_hist<T, FIRST_, ITEMS_>), dim3(GRID_), dim3(256), 0, stream, K, (const uint2 *)in, entries, (const int32_t *)n_valid, p * per, digits,      \
                       ntiles, hist, dtable, elems);                                                                                                                    \
    hipLaunchKernelGGL(k_es_scan, dim3((unsigned)((digits + 15) / 16)), dim3(1024), 0, stream, hist, ntiles, digits, totals);                                            \
    hipLaunchKernelGGL((k_es_scatter<FIRST_, ITEMS_>), dim3((unsigned)ntiles), dim3(256), 0, stream, K, (const uint2 *)in, entries, n_valid, p * per, digits, per,       \
                       (const int32_t *)hist, (const int32_t *)totals, out);                                                                                            \
  } while (0)
  for (int p = 0; p < passes; ++p) {
    uint2 *out = buf[p & 1], *in = buf[1 - (p & 1)];
    const unsigned first = (unsigned)ntiles > clear ? (unsigned)ntiles : clear;
    if (p == 0 && items == 4) ES_PASS(true, 4, first);
    else if (p == 0) ES_PASS(true, 8, first);
    else if (items == 4) ES_PASS(false, 4, (unsigned)ntiles);
    else ES_PASS(false, 8, (unsigned)ntiles);
  }
#undef ES_PASS
  return buf[(passes - 1) & 1];
}

template <typename T>
static void emb_table_gradient(const emb_keys &K, int entries, int c, int k, const float *weight, float scale, const T *dout, size_t dout_ld, T *dtable, char *ws, hipStream_t stream) {
  const size_t elems = (size_t)K.rows * c;
  const emb_space S = emb_layout(entries, c);
  const uint2 *pairs = emb_sort<T>(K, entries, S, ws, dtable, elems, stream);
  const int groups = (c + 7) / 8, tile = emb_tile(entries, c), ntiles = (entries + tile - 1) / tile;
  int lpr = 1;
  while (lpr < groups && lpr < 64) lpr *= 2;
  const dim3 grid((unsigned)((ntiles + 256 / lpr - 1) / (256 / lpr)), (unsigned)((groups + lpr - 1) / lpr));
  const int32_t *n_valid = (const int32_t *)(ws + S.n_valid);
  float *partial = (float *)(ws + S.partial);
  hipLaunchKernelGGL((k_emb_tiles<T, 8>), grid, dim3(256), 0, stream, pairs, n_valid, tile, lpr, c, k, weight, scale, dout, dout_ld, dtable, partial);
  if (ntiles > 1) {  // (16384 tokens of text in 8-entry tiles: 14 us on 16 tiles a workgroup, where several frequent tokens meet in one, 12 on 2)
    const int span = ntiles <= 4096 ? 2 : EJ_TILES;
    hipLaunchKernelGGL((k_emb_join<T>), dim3((unsigned)((ntiles + span - 1) / span), grid.y), dim3(256), 0, stream, pairs, n_valid, tile, span, lpr, c, scale, (const float *)partial,
                       dtable);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_emb_clear(T *__restrict__ dtable, size_t elems) {
  emb_clear<T>(dtable, elems, (size_t)blockIdx.x * 256 + threadIdx.x, (size_t)gridDim.x * 256);
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
  const int is64 = idx_dtype == LS3D_INDEX_I64, entries = n * k;
  if (dtable && rows > 0 && c > 0 && entries > 0) {
    if (!workspace || ((uintptr_t)workspace & 15)) return LS3D_ERR_ARG;
    if (workspace_bytes < ls3d_embedding_workspace_bytes(n, k, c)) return LS3D_ERR_WORKSPACE;
  }
  if (dweight && entries > 0 && (!idx || ((uintptr_t)idx & (is64 ? 7 : 3)))) return LS3D_ERR_ARG;
  if (dweight && entries > 0) {  // (c = 0: the products of no columns, zeros; no row is read)
    int lpr = 1;
    while (lpr * 8 < c && lpr < 64) lpr *= 2;
    EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_dweight<T>), ls3d_grid(entries, 256 / lpr), dim3(256), 0, stream, (const T *)table, (size_t)table_ld, rows, c, idx, is64,
                                        (long long)entries, k, lpr, scale, (const T *)dout, (size_t)dout_ld, dweight));
  }
  if (dtable && rows > 0 && c > 0) {
    const emb_keys K = {idx, is64, rows, padding};
    if (entries > 0) {
      EMB_TYPES(dtype, emb_table_gradient<T>(K, entries, c, k, weight, scale, (const T *)dout, (size_t)dout_ld, (T *)dtable, (char *)workspace, stream));
    } else {
      const size_t elems = (size_t)rows * c;
      EMB_TYPES(dtype, hipLaunchKernelGGL((k_emb_clear<T>), ls3d_grid((long long)(elems / 8 + 1)), dim3(256), 0, stream, (T *)dtable, elems));
    }
  }
  LS3D_RETURN_IF_LAUNCH_FAILED();
  return LS3D_OK;
}
