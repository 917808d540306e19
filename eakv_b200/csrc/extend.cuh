// extend.cuh - attention of several new tokens per cache: launch arguments,
// the work items and the masks, shared by its kernels.
//
// A row is a (token, query head) pair of one KV head: row r of a cache's KV
// head h is token r / G, query head h*G + r % G (G query heads per KV head).
// An item is (tile of rows, KV head): the rows of a tile are neighbours, so
// their causal limits nearly agree, and every row of the tile is served by the
// one read of a page. An item's positions are counted in units of unit_pages
// pages.
//
// Two ways of cutting the items up. Balanced: all units of all items in one
// row, cut into as many equal runs as CTAs fit on the GPU at once; a CTA works
// through the (parts of) items in its run. With whole waves of equal splits
// instead, the last wave is rarely full: 2048 tokens behind 32768 positions ran
// 1.40 ms (4 splits, 7 rounds), 1.35 (1 split, 1.7 rounds), 1.06 balanced. An item
// starts with `overhead' units of nothing, its set-up and results, so that a run of
// many short items is no longer than one of few long ones. Splits: every item cut
// into n_splits parts, one CTA each, where these fit on the GPU at once and
// are no longer than a run would be, or where a run would be longer than the
// precision of the sums allows.
// Parts of an item that is cut leave records, which the part that finishes
// last merges.
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
  int tile_rows;             // rows of a tile
  int unit_pages;
  int run;                   // balanced: units of a CTA's run (0: splits)
  int overhead;              // balanced: units that an item counts beyond its own
  long long units;           // balanced: of all items
  int tile_lo, tile_hi;      // splits: row tiles of this launch
  int n_splits, split_units;
  unsigned *cnt;             // counters of cut items, zero between calls
  float *part_o, *part_m, *part_l;   // records [slot][row of the tile]...
  const int32_t *depth;      // of a tree's tokens, or NULL: their slots
};

// The caches of one launch, all with new tokens. (What one cache needs lies
// together: a kernel's first look at each line of its arguments takes about as
// long as a load from memory.)
struct ExtendCache {
  const uint8_t *base;
  int old;      // position of the first new token
  int first;    // its index in the packed rows
  int n_new;
  int tile0;    // first row tile, over one KV head
};
struct ExtendBatch {
  ExtendCache c[kMaxBatch + 1];   // tile0 of the caches behind the last: all tiles
};

// Where the runs of a balanced launch start: row tile, and units behind the
// start of its KV head 0.
constexpr int kMaxRuns = 768;
struct ExtendRuns {
  int2 start[kMaxRuns];
};

// Masks of the new tokens: none, a tree's, a tree's with depths that windows go by.
enum { kCausal = 0, kTree = 1, kTreeDepths = 2 };

// Positions [lo, hi) that some row of rows [row0, row0 + rows) of a cache may
// attend, and the pages that hold them. (A depth may be anything up to the slot.)
struct ExtRange {
  int lo, hi, pg0, pages;
};
__host__ __device__ inline ExtRange extend_range(int row0, int rows, int G, int old, int n_new,
                                                 int window, int tree) {
  ExtRange r;
  const int t_first = tree == kTreeDepths ? 0 : row0 / G, t_last = (row0 + rows - 1) / G;
  r.lo = window > 0 && old + t_first + 1 > window ? old + t_first + 1 - window : 0;
  r.hi = tree ? old + n_new : old + t_last + 1;
  r.pg0 = r.lo / kPagePositions;
  r.pages = (r.hi + kPagePositions - 1) / kPagePositions - r.pg0;
  return r;
}

// A CTA's part of an item.
struct ExtItem {
  const uint8_t *base;   // the cache's slab
  int b, h;
  int row0, rows;  // rows of the tile, within the (cache, KV head)
  int old, tok0;   // position of the cache's first new token, its packed index
  int n_new;
  int lo, hi;      // positions that some row of the tile may attend: [lo, hi)
  int all_lo, all_hi;   // positions every row attends: [all_lo, all_hi)
  int pg0, npages; // pages of this part
  // records: the item's parts, this one's slot, the slots of part p > 0
  // (slot_p0 + p * slot_step) and of part 0, its counter
  int n_parts, slot, slot0, slot_p0, slot_step, counter;
  int state;       // 1: a part, 0: behind the last one, -1: addresses outside the cache
};

// A CTA's walk through its parts of items, in shared memory: thread 0 takes the
// steps, the next one ahead of the barrier that ends a part, so that all threads
// find it behind that.
struct ExtWalk {
  int tile, rem, left;   // next: tile, units behind its KV head 0; units left of the run
  ExtItem item[2];       // of even and odd parts

  __device__ __forceinline__ void begin(const ExtendArgs &a, const ExtendBatch &batch,
                                        const ExtendRuns &runs) {
    if (a.run > 0) {
      const int2 s = runs.start[blockIdx.x];
      tile = s.x;
      rem = s.y;
      left = (int)min((long long)a.run, a.units - (long long)blockIdx.x * a.run);
    } else {
      left = 1;
    }
    next(a, batch, 0);
  }

  // Part `p` into item[p & 1]; false behind the last one.
  __device__ __forceinline__ bool next(const ExtendArgs &a, const ExtendBatch &batch, int p) {
    ExtItem &out = item[p & 1];
    ExtItem it;
    for (;;) {
      if (left <= 0) {
        out.state = 0;
        return false;
      }
      int split = 0, item = 0;
      if (a.run == 0) {
        // splits fastest, then heads; the last tiles of a prompt, which attend the
        // most, start first
        split = blockIdx.x % a.n_splits;
        item = blockIdx.x / a.n_splits;
        it.h = item % a.geom.n_heads;
        tile = a.tile_hi - 1 - item / a.geom.n_heads;
      }
      int lo = 0, hi = a.n_caches - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (batch.c[mid].tile0 <= tile) lo = mid;
        else hi = mid - 1;
      }
      it.b = lo;
      const ExtendCache &c = batch.c[lo];
      it.base = c.base;
      it.old = c.old;
      it.tok0 = c.first;
      it.n_new = c.n_new;
      it.row0 = (tile - c.tile0) * a.tile_rows;
      it.rows = min(a.tile_rows, it.n_new * a.G - it.row0);
      const ExtRange r = extend_range(it.row0, it.rows, a.G, it.old, it.n_new, a.window,
                                      a.tree ? (a.depth ? kTreeDepths : kTree) : kCausal);
      const int t_first = it.row0 / a.G, t_last = (it.row0 + it.rows - 1) / a.G;
      it.lo = r.lo;
      it.hi = r.hi;
      it.all_lo = a.window > 0 ? max(0, it.old + t_last + 1 - a.window) : 0;
      it.all_hi = a.tree ? it.old : it.old + t_first + 1;
      const int units = (r.pages + a.unit_pages - 1) / a.unit_pages;
      int u0, u1;
      if (a.run > 0) {
        // [overhead | units], head after head
        const int len = a.overhead + units;
        it.h = rem / len;
        const int x0 = rem - it.h * len, x1 = min(len, x0 + left);
        // the item's place in the row of all units: this run's end less what is left
        const long long end = min((long long)(blockIdx.x + 1) * a.run, a.units);
        const long long at = end - left - x0 + a.overhead;
        left -= x1 - x0;
        rem += x1 - x0;
        if (rem >= len * a.geom.n_heads) {
          tile++;
          rem = 0;
        }
        u0 = max(x0 - a.overhead, 0);
        u1 = x1 - a.overhead;
        if (u1 <= 0) continue;   // only the item's overhead: another run has its units
        const int first = (int)(at / a.run), last = (int)((at + units - 1) / a.run);
        it.n_parts = last - first + 1;
        // two slots per CTA: a part that begins inside its item, and one that begins it
        it.slot0 = 2 * first + 1;
        it.slot_p0 = 2 * first;
        it.slot_step = 2;
        it.slot = u0 == 0 ? it.slot0 : 2 * blockIdx.x;
        it.counter = first;   // only the last item that starts in a run is cut at its end
      } else {
        u0 = min(split * a.split_units, units);
        u1 = min(u0 + a.split_units, units);
        it.n_parts = a.n_splits;
        it.slot0 = it.slot_p0 = item * a.n_splits;
        it.slot_step = 1;
        it.slot = it.slot0 + split;
        it.counter = item;
        left = 0;
      }
      // the last unit may be half a one: a part behind it starts at the last page's end
      const int p0 = min(u0 * a.unit_pages, r.pages);
      it.pg0 = r.pg0 + p0;
      it.npages = min(u1 * a.unit_pages, r.pages) - p0;
      const bool ok = it.b >= 0 && it.b < a.n_caches && it.h >= 0 && it.h < a.geom.n_heads && it.rows >= 1 &&
                      it.row0 >= 0 && it.pg0 >= 0 && it.pg0 + it.npages <= a.geom.n_pages;
      if (!ok) atomicOr(a.status, kStatusBadIndex);
      it.state = ok ? 1 : -1;
      out = it;
      return true;
    }
  }

  // Parts from p on that nobody works on, after a wait ran out or at a bad item:
  // they arrive all the same, without records, so that the counters are back at
  // zero after the launch.
  // item[p & 1] stays as it is: other threads may still look at it.
  __device__ __forceinline__ void abandon(const ExtendArgs &a, const ExtendBatch &batch, int p) {
    for (const ExtItem *it = &item[p & 1]; it->state != 0; it = &item[(p + 1) & 1]) {
      if (it->n_parts > 1) atomicInc(a.cnt + it->counter, (unsigned)it->n_parts - 1);
      next(a, batch, p + 1);
    }
  }
};

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

// Mask of row r of the (cache, KV head), but for depths; rows behind the last repeat it.
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

// Depth of the cache's new token t: one outside [0, t] is reported and counts as t.
__device__ __forceinline__ int token_depth(const ExtendArgs &a, const ExtItem &it, int t) {
  const int d = __ldg(a.depth + it.tok0 + t);
  if (d >= 0 && d <= t) return d;
  atomicOr(a.status, kStatusBadIndex);
  return t;
}

// The mask m of row r with its window by depths.
__device__ __forceinline__ void depth_window(const ExtendArgs &a, const ExtItem &it, int r, RowMask &m) {
  const int t = min(r, it.n_new * a.G - 1) / a.G;
  // what lies in the window by its depth lies in it by its slot, depths being no larger
  const int d = token_depth(a, it, t);
  m.lo = max(0, it.old + d + 1 - a.window);
  if (d >= a.window)   // new tokens may lie before the window
    for (int j = 0; j < it.n_new; j++)
      if (((m.bits >> j) & 1) && token_depth(a, it, j) <= d - a.window) m.bits &= ~(1ull << j);
}

// (w & mask) | magic
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}
// Two values as f16 in one word.
__device__ __forceinline__ uint32_t pack_f16(float x0, float x1) {
  const __half2 h = __floats2half2_rn(x0, x1);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Record of row r in a slot, and the slot of part p of the item.
__device__ __forceinline__ size_t part_row(const ExtendArgs &a, int slot, int r) {
  return (size_t)slot * a.tile_rows + r;
}
__device__ __forceinline__ int part_slot(const ExtItem &it, int p) {
  return p == 0 ? it.slot0 : it.slot_p0 + p * it.slot_step;
}

// Arrival of a part on its item's counter, as in decode_common.cuh: true for
// the last of the item's parts, with the other parts' records visible. Called
// by NT threads that meet on named barrier `id`; *last is shared.
template <int NT>
__device__ __forceinline__ bool extend_arrive_last(const ExtendArgs &a, const ExtItem &it, int *last,
                                                   int id) {
  __threadfence();
  named_sync(id, NT);
  if (threadIdx.x == 0) {
    const unsigned n = (unsigned)it.n_parts;
    *reinterpret_cast<volatile int *>(last) = atomicInc(a.cnt + it.counter, n - 1) == n - 1;
  }
  named_sync(id, NT);
  const bool r = *reinterpret_cast<volatile int *>(last) != 0;
  if (r) __threadfence();
  return r;
}

// Weight of a record with maximum m under the common maximum M. A record
// without a finite score has m = -inf: it holds zeros, or NaN where a NaN was
// attended, and counts with weight 1 so that the NaN is kept.
__device__ __forceinline__ float part_weight(float m, float M) {
  return m == -INFINITY ? 1.0f : ex2(m - M);
}

// Element offset of every n-th row of the item's tile in a buffer of rows, from
// row r on (the last row when that lies behind it), without a division per row.
struct RowWalk {
  long long at, plain, wrapped;   // offset; its step, and the step into another token
  int h, dh, G;                   // query head within the KV head's group, its step
  __device__ __forceinline__ RowWalk(const ExtendArgs &a, const ExtItem &it, const Rows &b, int r, int n) {
    const int row = it.row0 + min(r, it.rows - 1), t = row / a.G;
    G = a.G;
    h = row - t * G;
    at = (long long)(it.tok0 + t) * b.token_stride + (long long)(it.h * G + h) * b.head_stride;
    const int dt = n / G;
    dh = n - dt * G;
    plain = dt * b.token_stride + dh * b.head_stride;
    wrapped = plain + b.token_stride - G * b.head_stride;
  }
  __device__ __forceinline__ void step() {
    const bool wrap = h + dh >= G;
    at += wrap ? wrapped : plain;
    h += wrap ? dh - G : dh;
  }
};

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

// ROWS times NT elements of four dims from x0 on (row of the chunk x / (HD/4)),
// merged over the parts, PARTS parts' loads at a time.
template <int HD, typename T, int NT, int ROWS, int PARTS>
__device__ __forceinline__ void merge_rows(const ExtendArgs &a, const ExtItem &it, bool vec, int r0, int n,
                                           const float *m_s, const float *l_s, const float *f_s) {
  const int ns = it.n_parts;
  for (int x0 = threadIdx.x; x0 < n; x0 += ROWS * NT) {
    float O[ROWS][4];
#pragma unroll
    for (int k = 0; k < ROWS; k++) O[k][0] = O[k][1] = O[k][2] = O[k][3] = 0.0f;
#pragma unroll 1
    for (int s0 = 0; s0 < ns; s0 += PARTS) {
      float4 o[PARTS][ROWS];
#pragma unroll
      for (int s = 0; s < PARTS; s++) {   // the last part, the last element again behind the end
        const float *po = a.part_o + part_row(a, part_slot(it, min(s0 + s, ns - 1)), r0) * HD;
#pragma unroll
        for (int k = 0; k < ROWS; k++)
          o[s][k] = __ldcg(reinterpret_cast<const float4 *>(po + 4 * min(x0 + k * NT, n - 1)));
      }
#pragma unroll
      for (int s = 0; s < PARTS; s++) {
        if (s0 + s >= ns) break;
#pragma unroll
        for (int k = 0; k < ROWS; k++) {
          const float f = f_s[min(x0 + k * NT, n - 1) / (HD / 4) * ns + s0 + s];
          O[k][0] = fmaf(f, o[s][k].x, O[k][0]);
          O[k][1] = fmaf(f, o[s][k].y, O[k][1]);
          O[k][2] = fmaf(f, o[s][k].z, O[k][2]);
          O[k][3] = fmaf(f, o[s][k].w, O[k][3]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; k++) {
      const int x = x0 + k * NT, r = x / (HD / 4), d = 4 * (x % (HD / 4));
      if (x < n) extend_store<T>(a, it, r0 + r, d, O[k], m_s[r], l_s[r], vec);
    }
  }
}

// The last part of an item: rows merged over the parts, in their order, by NT
// threads that meet on named barrier `id`. `ws` is free shared memory of ws_floats,
// more than twice the parts of any item: the weights of a row's parts are worked out
// once into it. What this takes is the loads' time, so that eight are on their way
// per thread: of four rows, or of eight parts where the rows are few (with one row
// and part at a time 3 parts of 256 rows took 27 us, 19 parts of 16 rows 9 us).
template <int HD, typename T, int NT>
__device__ __forceinline__ void extend_merge(const ExtendArgs &a, const ExtItem &it, bool vec, float *ws,
                                             int ws_floats, int id) {
  const int ns = it.n_parts, most = min(it.rows, ws_floats / (2 * ns + 2));
  for (int r0 = 0; r0 < it.rows; r0 += most) {
    const int rows = min(most, it.rows - r0);
    float *m_s = ws, *l_s = ws + rows;                          // [rows]
    float *f_s = ws + 2 * rows, *p_s = f_s + rows * ns;         // [rows][ns]
    for (int x = threadIdx.x; x < rows * ns; x += NT) {
      const int r = x / ns;
      const size_t pr = part_row(a, part_slot(it, x - r * ns), r0 + r);
      f_s[x] = __ldcg(a.part_m + pr);
      p_s[x] = __ldcg(a.part_l + pr);
    }
    named_sync(id, NT);
    for (int r = threadIdx.x; r < rows; r += NT) {
      float M = -INFINITY, L = 0.0f;
      for (int s = 0; s < ns; s++) M = fmaxf(M, f_s[r * ns + s]);
      for (int s = 0; s < ns; s++) {
        const float f = part_weight(f_s[r * ns + s], M);
        f_s[r * ns + s] = f;
        L = fmaf(f, p_s[r * ns + s], L);
      }
      m_s[r] = M;
      l_s[r] = L;
    }
    named_sync(id, NT);
    const int n = rows * (HD / 4);
    if (n <= NT) merge_rows<HD, T, NT, 1, 8>(a, it, vec, r0, n, m_s, l_s, f_s);
    else merge_rows<HD, T, NT, 4, 2>(a, it, vec, r0, n, m_s, l_s, f_s);
    named_sync(id, NT);   // ws is used again
  }
}

// extend_mma.cu: tiles of 8, 16 or 24 rows
int extend_mma_resident(int head_dim, int dtype, int tile_rows);
int extend_mma_launch(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks,
                      bool vec, cudaStream_t s);
// extend_umma.cu: 16-bit types, where the kernel can run (current device)
constexpr int kExtendUmmaRows = 256;
bool extend_umma_usable(int head_dim, int dtype);
int extend_umma_launch(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks,
                       bool vec, cudaStream_t s);

}  // namespace eakv
