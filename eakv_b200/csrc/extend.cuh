// extend.cuh - attention of several new tokens per cache: launch arguments,
// the work items and the masks, shared by its kernels.
//
// A row is a (token, query head) pair of one KV head: row r of a cache's KV
// head h is token r / G, query head h*G + r % G (G query heads per KV head).
// A work item is (cache, KV head, tile of rows, split): the rows of a tile are
// neighbours, so their causal limits nearly agree, and every row of the tile
// is served by the one read of a page.
#pragma once
#include "decode_common.cuh"
#include "tokens.cuh"

namespace eakv {

struct ExtendArgs {
  PageGeom geom;
  int n_caches, layer, n_q, G;
  int dtype;
  Rows q, out;
  float scale_log2;          // scale * log2(e)
  int window;                // 0: none
  const unsigned long long *tree;
  float *lse;                // [token][n_q] or NULL
  int *status;
  unsigned wait_budget;
  int test_stall;
  // plan
  int tile_rows;             // rows of a work item
  int tile_lo, tile_hi;      // row tiles of this launch
  int n_splits, split_pages;
  unsigned *cnt;             // one counter per item, zero between calls
  float *part_o, *part_m, *part_l;   // [item][split][row of the tile]..., see part_row
};

// The caches of one launch, all with new tokens.
struct ExtendBatch {
  const uint8_t *base[kMaxBatch];
  int old[kMaxBatch];        // position of the first new token
  int first[kMaxBatch];      // its index in the packed rows
  int n_new[kMaxBatch];
  int tile0[kMaxBatch + 1];  // first row tile of each cache, over one KV head
};

struct ExtItem {
  int b, h, split;
  int item;        // index without the split
  int row0, rows;  // rows of the tile, within the (cache, KV head)
  int old, tok0;   // position of the cache's first new token, its packed index
  int n_new;
  int lo, hi;      // positions that some row of the tile may attend: [lo, hi)
  int all_lo, all_hi;   // positions every row attends: [all_lo, all_hi)
  int pg0, npages; // pages of this split
};

// blockIdx.x -> (tile, head, split), splits fastest, then heads; the last
// tiles of a prompt, which attend the most, start first.
__device__ __forceinline__ ExtItem extend_item(const ExtendArgs &a, const ExtendBatch &batch) {
  ExtItem it;
  int bid = blockIdx.x;
  it.split = bid % a.n_splits;
  it.item = bid / a.n_splits;
  bid = it.item;
  it.h = bid % a.geom.n_heads;
  const int tile = a.tile_hi - 1 - bid / a.geom.n_heads;
  int lo = 0, hi = a.n_caches - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (batch.tile0[mid] <= tile) lo = mid;
    else hi = mid - 1;
  }
  it.b = lo;
  it.old = batch.old[lo];
  it.tok0 = batch.first[lo];
  it.n_new = batch.n_new[lo];
  it.row0 = (tile - batch.tile0[lo]) * a.tile_rows;
  it.rows = min(a.tile_rows, it.n_new * a.G - it.row0);
  const int t_first = it.row0 / a.G, t_last = (it.row0 + it.rows - 1) / a.G;
  it.lo = a.window > 0 ? max(0, it.old + t_first + 1 - a.window) : 0;
  it.hi = a.tree ? it.old + it.n_new : it.old + t_last + 1;
  it.all_lo = a.window > 0 ? max(0, it.old + t_last + 1 - a.window) : 0;
  it.all_hi = a.tree ? it.old : it.old + t_first + 1;
  const int P0 = it.lo / kPagePositions;
  const int P1 = (it.hi + kPagePositions - 1) / kPagePositions;
  it.pg0 = min(P0 + it.split * a.split_pages, P1);
  const int pg1 = min(P1, it.pg0 + a.split_pages);
  it.npages = pg1 > it.pg0 ? pg1 - it.pg0 : 0;
  return it;
}

__device__ __forceinline__ bool extend_item_ok(const ExtendArgs &a, const ExtItem &it) {
  const bool ok = it.b >= 0 && it.b < a.n_caches && it.h < a.geom.n_heads && it.rows >= 1 &&
                  it.row0 >= 0 && it.pg0 >= 0 && it.pg0 + it.npages <= a.geom.n_pages;
  if (!ok && threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
  return ok;
}

// What one row attends: positions [lo, hi), and with a tree, of those from
// `old` on only the ones whose bit is set.
struct RowMask {
  int lo, hi, old;
  unsigned long long bits;
  __device__ __forceinline__ bool attends(int pos) const {
    if (pos < lo || pos >= hi) return false;
    return pos < old || ((bits >> (pos - old)) & 1);
  }
};

// Mask of row r of the (cache, KV head); rows behind the last repeat it.
__device__ __forceinline__ RowMask row_mask(const ExtendArgs &a, const ExtItem &it, int r) {
  RowMask m;
  const int t = min(r, it.n_new * a.G - 1) / a.G;
  m.lo = a.window > 0 ? max(0, it.old + t + 1 - a.window) : 0;
  if (a.tree) {
    m.hi = it.old + it.n_new;
    m.old = it.old;
    m.bits = __ldg(a.tree + it.tok0 + t);
  } else {
    m.hi = m.old = it.old + t + 1;
    m.bits = 0;
  }
  return m;
}

// Partial records of a split: row r of (item, split).
__device__ __forceinline__ size_t part_row(const ExtendArgs &a, const ExtItem &it, int split, int r) {
  return ((size_t)it.item * a.n_splits + split) * a.tile_rows + r;
}

// Arrival of a work item's CTA on its counter, as in decode_common.cuh: true
// for the last of the item's splits, with the other splits' records visible.
__device__ __forceinline__ bool extend_arrive_last(const ExtendArgs &a, int item) {
  __shared__ int s_last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned n = (unsigned)a.n_splits;
    s_last = atomicInc(a.cnt + item, n - 1) == n - 1;
  }
  __syncthreads();
  const bool last = s_last != 0;
  if (last) __threadfence();
  return last;
}

// Weight of a record with maximum m under the common maximum M. A record
// without a finite score has m = -inf: it holds zeros, or NaN where a NaN was
// attended, and counts with weight 1 so that the NaN is kept.
__device__ __forceinline__ float part_weight(float m, float M) {
  return m == -INFINITY ? 1.0f : ex2(m - M);
}

// Output row of row r of the item's tile.
template <typename T>
__device__ __forceinline__ T *extend_out(const ExtendArgs &a, const ExtItem &it, int r) {
  const int row = it.row0 + r;
  return reinterpret_cast<T *>(a.out.data) + (long long)(it.tok0 + row / a.G) * a.out.token_stride +
         (long long)(it.h * a.G + row % a.G) * a.out.head_stride;
}

// LSE of row r from its base-2 maximum and sum.
__device__ __forceinline__ void extend_lse(const ExtendArgs &a, const ExtItem &it, int r, float M, float L) {
  const int row = it.row0 + r;
  a.lse[(long long)(it.tok0 + row / a.G) * a.n_q + it.h * a.G + row % a.G] =
      L == 0.0f ? -INFINITY : ((M == -INFINITY ? 0.0f : M) + log2f(L)) * kLn2;
}

// Four neighbouring dims of the finished row r (unnormalized sums O, base-2
// maximum M, sum L) to the output; the lane with d == 0 writes the LSE.
template <typename T>
__device__ __forceinline__ void extend_store(const ExtendArgs &a, const ExtItem &it, int r, int d,
                                             const float (&O)[4], float M, float L, bool vec) {
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;   // nothing attended: zeros
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = O[e] * inv;
  T *p = extend_out<T>(a, it, r) + d;
  if (vec) store4<T, true>(p, y);
  else store4<T, false>(p, y);
  if (a.lse && d == 0) extend_lse(a, it, r, M, L);
}

// The last CTA of an item: rows merged over the splits, in split order, four
// dims per thread at a time. `ws` is free shared memory of ws_floats: the
// splits' weights of a row are worked out once into it, and the records' loads
// then depend on nothing.
template <int HD, typename T, int NT>
__device__ __forceinline__ void extend_merge(const ExtendArgs &a, const ExtItem &it, bool vec, float *ws,
                                             int ws_floats) {
  const int ns = a.n_splits;
  float *m_s = ws, *l_s = ws + it.rows, *f_s = ws + 2 * it.rows;   // [rows], [rows], [rows][ns]
  const bool staged = (ns + 2) * it.rows <= ws_floats;
  __syncthreads();
  if (staged) {
    for (int x = threadIdx.x; x < it.rows * ns; x += NT)
      f_s[x] = __ldcg(a.part_m + part_row(a, it, x % ns, x / ns));
    __syncthreads();
    for (int r = threadIdx.x; r < it.rows; r += NT) {
      float M = -INFINITY, L = 0.0f;
      for (int s = 0; s < ns; s++) M = fmaxf(M, f_s[r * ns + s]);
#pragma unroll 4
      for (int s = 0; s < ns; s++) {
        const float f = part_weight(f_s[r * ns + s], M);
        f_s[r * ns + s] = f;
        L = fmaf(f, __ldcg(a.part_l + part_row(a, it, s, r)), L);
      }
      m_s[r] = M;
      l_s[r] = L;
    }
    __syncthreads();
  }
  for (int x = threadIdx.x; x < it.rows * (HD / 4); x += NT) {
    const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
    float M = -INFINITY, L = 0.0f;
    if (staged) {
      M = m_s[r];
      L = l_s[r];
    } else {
      for (int s = 0; s < ns; s++) M = fmaxf(M, __ldcg(a.part_m + part_row(a, it, s, r)));
    }
    float O[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int s = 0; s < ns; s++) {
      const size_t pr = part_row(a, it, s, r);
      const float4 o = __ldcg(reinterpret_cast<const float4 *>(a.part_o + pr * HD + d));
      float f;
      if (staged) {
        f = f_s[r * ns + s];
      } else {
        f = part_weight(__ldcg(a.part_m + pr), M);
        L = fmaf(f, __ldcg(a.part_l + pr), L);
      }
      O[0] = fmaf(f, o.x, O[0]);
      O[1] = fmaf(f, o.y, O[1]);
      O[2] = fmaf(f, o.z, O[2]);
      O[3] = fmaf(f, o.w, O[3]);
    }
    extend_store<T>(a, it, r, d, O, M, L, vec);
  }
}

// extend_mma.cu
constexpr int kExtendMmaRows = 16;
int extend_mma_resident(int head_dim, int dtype);
int extend_mma_launch(const ExtendArgs &a, const ExtendBatch &b, int n_blocks, bool vec,
                      cudaStream_t s);
// extend_umma.cu: 16-bit types
constexpr int kExtendUmmaRows = 256;
int extend_umma_launch(const ExtendArgs &a, const ExtendBatch &b, int n_blocks, bool vec,
                       cudaStream_t s);

}  // namespace eakv
