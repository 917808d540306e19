// extend.cu - entry points and plan of the attention of several new tokens per
// cache (eakv_extend_attention): argument checks, the cut of each row tile
// into sequence splits, and the workspace of their records.
#include <math.h>
#include <string.h>

#include "extend.cuh"

namespace eakv {
namespace {

// Items (row tile x KV head) of one launch whose rows are split: bounds the
// counters, which have a fixed place in a workspace, and its records. A call
// with more runs as several launches.
constexpr int kSplitItems = 16384;
constexpr size_t kCounterBytes = kSplitItems * sizeof(unsigned);

// Longest part of an item in pages. The tensor core adds into its f32 sums by
// truncation, a drift of up to 2^-24 of the sum per step of 16 positions. In
// the warp-level kernel four warps take pages in turn: 64 pages are 64 steps of a
// warp (2^-18 at worst, 2^-19 on average, below what f32 results ask for), and
// 1024 pages 2^-14; in the tcgen05 kernel one sum takes every step, and 1024 pages
// are 2^-12, 2^-13 on average: both below the 2^-9 or 2^-12 of 16-bit outputs (and the
// latter below what K's rounding to f16 does there, 2^-10). (With 256
// pages for the warp-level kernel 16 caches of up to 32768 positions were kept from
// equal runs by tiles of 8 rows: 303 us, in runs 231.)
constexpr int kPartPagesF32 = 64, kPartPages16 = 1024;

// Rows (new tokens x query heads per KV head) up to which 16-bit calls take the
// warp-level kernel. 16 caches of 8192 positions, 8 KV heads of 128: at 24, 32, 40, 64
// rows 112, 128, 173, 256 us, the tcgen05 kernel 171 each; head_dim 64 at 32, 40, 64
// rows 81, 107, 160 against 118, 120, 120; 64 caches of 512 positions 73, 112, 166
// against 99 each.
constexpr int kMmaRows = 32;
// A page's time for tiles of 8, 16 and 24 rows of the warp-level kernel, 16-bit
// types: 16 caches of 8192 positions (8 KV heads of 128) took 58, 81 and 112 us with
// one tile each, 15 us of it set-up. A second tile of 8 rows costs as much again (84
// us), so 16 rows go to one tile, 17 to 24 to one of 24. In f32 the two limbs double
// the operands and larger tiles lose: 104 rows per head (13, 7, 5 tiles) 73, 78, 86 us.
constexpr int kTileCost[3] = {10, 16, 21};
// Shortest parts worth a CTA, and what an item costs beyond its positions (set-up,
// results), in pages of the warp-level kernel and tiles of the tcgen05 kernel.
constexpr int kLeastPages = 6, kLeastTiles = 4;
constexpr int kOverheadPages = 6, kOverheadTiles = 5;

// What the cuts of a balanced run cost a CTA, its records and merges: in pages of the
// warp-level kernel, in tiles of the tcgen05 kernel per 64 dims of the head.
// Measured in runs / as whole items, us (8 KV heads, 32 query heads):
// 512-token prompts of the tcgen05 kernel, head_dim 128, at 1.7, 3.0, 4.3 items per CTA:
// no earlier positions 62/45, 90/70, 120/102; 2048 of them 141/111, 214/207, 304/277;
// 8192: 328/324, 590/639, 834/802 (at 2.2 403/475); head_dim 64: 45/35, 64/52, 82/72;
// 102/96, 158/173, 215/225; 257/277, 437/540, 613/685. Single tokens of the warp-level
// kernel, head_dim 128, at 1.2, 2.3, 3.5 items per CTA: 512 positions 33/31, 49/47, 72/63;
// 2048: 59/60, 103/95, 147/135; head_dim 64, at 1.3, 2.2, 3.5: 27/26, 41/38, 58/52; 54/49,
// 75/72, 115/102.
constexpr int kCutPages = 28, kCutTiles = 14;

// Parts of an item, at most: a merge keeps two words of each in shared memory.
constexpr int kMaxParts = 4096;

// One launch's caches and plan: a call's caches with few rows and those with
// many go to different kernels.
struct Part {
  bool umma;
  int tiles, launch_tiles;   // row tiles in all and per launch
  int slots;                 // records of one launch (0: nothing is cut)
  int tile_rows, unit_pages, run, n_runs, overhead, n_splits, split_units, n_caches;
  long long units;
  ExtendBatch b;
  ExtendRuns runs;
};

int sm_count(int dev) {
  int n = 0;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// The caches of `t` that belong to the part, their row tiles, splits and record
// bytes. Call with the caches' device current.
int plan_part(const ExtendArgs &a, const TokenBatch &t, int device, int tree, bool many_ok, bool umma,
              Part &p) {
  p.umma = umma;
  p.tile_rows = kExtendUmmaRows;
  auto mine = [&](int i) {
    const long long rows = (long long)(t.first[i + 1] - t.first[i]) * a.G;
    return rows > 0 && (many_ok && (rows > kMmaRows || t_force_path == 3)) == umma;
  };
  p.n_caches = 0;
  p.slots = p.run = p.n_runs = p.overhead = 0;
  p.units = 0;
  p.n_splits = p.split_units = 1;
  p.unit_pages = umma ? 2 : 1;   // the tcgen05 kernel's tiles are two pages
  const int heads = a.geom.n_heads;
  // the tile size that takes least; 8 rows in f32, and where the parts are as
  // short as they get even so (2 tokens of 32 + 4 heads of 64 behind 2046
  // positions: 14.8 us, with tiles of 16 rows 18)
  long long best = 0;
  for (int size = 8; size <= (a.dtype == EAKV_F32 ? 8 : 24) && !umma; size += 8) {
    long long cost = 0;
    for (int i = 0; i < a.n_caches; i++) {
      if (!mine(i)) continue;
      const int n = t.first[i + 1] - t.first[i];
      const ExtRange r = extend_range(0, n * a.G, a.G, t.pos[i], n, a.window, tree);
      cost += ((long long)n * a.G + size - 1) / size * (r.pages + kOverheadPages) * kTileCost[size / 8 - 1];
    }
    if (size == 8 || cost < best) {
      best = cost;
      p.tile_rows = size;
    }
    const long long least_cost = 3ll * sm_count(device) * (kLeastPages + kOverheadPages) * kTileCost[0];
    if (size == 8 && cost * heads <= least_cost) break;
  }
  long long tiles = 0;
  for (int i = 0; i < a.n_caches; i++) {
    if (!mine(i)) continue;
    const int n = t.first[i + 1] - t.first[i];
    const int k = p.n_caches++;
    p.b.c[k] = {t.base[i], t.pos[i], t.first[i], n, (int)tiles};
    tiles += ((long long)n * a.G + p.tile_rows - 1) / p.tile_rows;
    if (tiles * heads > (1ll << 30)) {
      set_error(EAKV_ERR_INVALID, "extend_attention: more than 2^30 tiles of rows");
      return EAKV_ERR_INVALID;
    }
  }
  for (int i = p.n_caches; i <= kMaxBatch; i++) p.b.c[i] = {nullptr, 0, 0, 0, (int)tiles};
  p.tiles = p.launch_tiles = (int)tiles;
  if (p.tiles == 0) return EAKV_OK;
  // units of a tile's items, and of all
  auto units_of = [&](int k, int tile) {
    const int row0 = (tile - p.b.c[k].tile0) * p.tile_rows, all = p.b.c[k].n_new * a.G;
    const int rows = all - row0 < p.tile_rows ? all - row0 : p.tile_rows;
    const ExtRange r = extend_range(row0, rows, a.G, p.b.c[k].old, p.b.c[k].n_new, a.window, tree);
    return (r.pages + p.unit_pages - 1) / p.unit_pages;
  };
  const int overhead = umma ? kOverheadTiles : kOverheadPages;
  long long units = 0;   // with the items' overheads
  int max_units = 1;
  for (int k = 0; k < p.n_caches; k++)
    for (int i = p.b.c[k].tile0; i < p.b.c[k + 1].tile0; i++) {
      const int u = units_of(k, i);
      units += (long long)(u + overhead) * heads;
      if (u > max_units) max_units = u;
    }
  const int per_sm = umma ? 1 : extend_mma_resident(a.geom.gpd * 64, a.dtype, p.tile_rows);
  if (per_sm <= 0) return EAKV_ERR_INVALID;   // recorded by the lookup
  const int cap = (a.dtype == EAKV_F32 ? kPartPagesF32 : kPartPages16) / p.unit_pages;
  const int least = umma ? kLeastTiles : kLeastPages;
  const long long resident = (long long)per_sm * sm_count(device), items = tiles * heads;
  long long run = (units + resident - 1) / resident;
  if (run < least + overhead) run = least + overhead;
  // splits that fit on the GPU at once, no longer than a run
  long long fit = resident / items;
  if (fit > max_units / least) fit = max_units / least;
  if (fit < 1) fit = 1;
  const bool splits = items * fit <= resident && (max_units + fit - 1) / fit + overhead <= run + run / 8 &&
                      (max_units + fit - 1) / fit <= cap;
  // or whole items, where the last round's idle CTAs cost less than the cuts of runs:
  // rounds of the mean item, and what the longest has beyond it, against a run
  const double mean = (double)units / items, rounds = (double)((items + resident - 1) / resident);
  const bool whole = max_units <= cap && rounds * mean + (max_units + overhead - mean) <=
                                             run + (umma ? kCutTiles * a.geom.gpd : kCutPages);
  const bool even = splits || whole;
  if (!splits) fit = 1;
  if (t_force_splits == 0 && !even && run <= cap && (units + run - 1) / run <= kMaxRuns) {
    p.overhead = overhead;
    p.units = units;
    p.run = (int)run;
    p.n_runs = (int)((units + run - 1) / run);
    // start of every run: walk the tiles
    long long at = 0;   // units before the tile
    int r = 0;
    for (int k = 0; k < p.n_caches; k++)
      for (int i = p.b.c[k].tile0; i < p.b.c[k + 1].tile0; i++) {
        const long long u = (long long)(units_of(k, i) + overhead) * heads;
        for (; r < p.n_runs && (long long)r * p.run < at + u; r++)
          p.runs.start[r] = make_int2(i, (int)((long long)r * p.run - at));
        at += u;
      }
    p.slots = p.n_runs > 1 ? 2 * p.n_runs : 0;
    return EAKV_OK;
  }
  int ns = t_force_splits > 0 ? t_force_splits : even ? (int)fit : (max_units + cap - 1) / cap;
  if (ns > max_units) ns = max_units;
  if (ns > kMaxParts) ns = kMaxParts;
  p.split_units = (max_units + ns - 1) / ns;
  p.n_splits = (max_units + p.split_units - 1) / p.split_units;
  if (p.n_splits > 1) {
    if (p.launch_tiles > kSplitItems / heads) p.launch_tiles = kSplitItems / heads;
    // bounds the records of a launch
    while ((long long)p.launch_tiles * heads * p.n_splits * p.tile_rows > (1ll << 22) && p.launch_tiles > 1)
      p.launch_tiles = (p.launch_tiles + 1) / 2;
    p.slots = p.launch_tiles * heads * p.n_splits;
  }
  return EAKV_OK;
}

// Both parts of a call: the caches with many rows, which the tcgen05 kernel takes where
// it can, and the others.
int plan(const ExtendArgs &a, const TokenBatch &t, int device, int tree, Part (&p)[2]) {
  const bool many_ok = a.dtype != EAKV_F32 && t_force_path != 2 &&
                       extend_umma_usable(a.geom.gpd * 64, a.dtype);
  int rc = plan_part(a, t, device, tree, many_ok, true, p[0]);
  return rc ? rc : plan_part(a, t, device, tree, many_ok, false, p[1]);
}

size_t record_bytes(const ExtendArgs &a, const Part &p) {
  return (size_t)p.slots * p.tile_rows * (a.geom.gpd * 64 + 2) * sizeof(float);
}

// Workspace bytes of both parts, which run one after the other on it.
size_t workspace_of(const ExtendArgs &a, const Part (&p)[2]) {
  const size_t r0 = record_bytes(a, p[0]), r1 = record_bytes(a, p[1]), r = r0 > r1 ? r0 : r1;
  return r ? kCounterBytes + r : 0;
}

int refuse(const char *what) {
  set_error(EAKV_ERR_INVALID, "extend_attention: %s", what);
  return EAKV_ERR_INVALID;
}

// Checks shared by the call and its workspace query.
int check_call(const eakv_cache_t *const *caches, int n_caches, const int *n_new, int dtype, int n_q,
               int window, bool tree, ExtendArgs &a, TokenBatch &b, int &total) {
  int rc = token_batch(caches, n_caches, n_q, nullptr, n_new, "extend_attention", b, total);
  if (rc) return rc;
  if (dtype < EAKV_F32 || dtype > EAKV_BF16) return refuse("unknown element type");
  if (window < 0) return refuse("negative window");
  if (caches[0]->n_kv_heads > kSplitItems) return refuse("more than 16384 KV heads");
  if ((long long)total * (n_q / caches[0]->n_kv_heads) > (1ll << 30))
    return refuse("more than 2^30 (token, query head) rows per KV head");
  for (int i = 0; i < n_caches && tree; i++)
    if (n_new[i] > 64) return refuse("a tree mask holds 64 new tokens per cache at most");
  memset(&a, 0, sizeof a);
  a.geom = caches[0]->geom;
  a.n_caches = n_caches;
  a.n_q = n_q;
  a.G = n_q / caches[0]->n_kv_heads;
  a.dtype = dtype;
  a.window = window;
  return EAKV_OK;
}

}  // namespace
}  // namespace eakv

using namespace eakv;

extern "C" {

int eakv_extend_workspace(const eakv_cache_t *const *caches, int n_caches, const int *n_new,
                          int dtype, int n_q_heads, int window, int tree, size_t *bytes) {
  clear_error();
  if (!bytes) return refuse("NULL result");
  *bytes = 0;
  ExtendArgs a;
  TokenBatch b;
  int total = 0;
  int rc = check_call(caches, n_caches, n_new, dtype, n_q_heads, window, tree != 0, a, b, total);
  if (rc || total == 0) return rc;
  DeviceGuard g(caches[0]->device);
  Part p[2];
  rc = plan(a, b, caches[0]->device, tree == 2 ? kTreeDepths : tree ? kTree : kCausal, p);
  if (!rc) *bytes = workspace_of(a, p);
  return rc;
}

int eakv_extend_attention(const eakv_cache_t *const *caches, int n_caches, int layer,
                          const int *n_new, const eakv_rows_t *q, const eakv_rows_t *out,
                          int n_q_heads, float scale, int window, const uint64_t *tree, float *lse,
                          void *workspace, size_t workspace_bytes, void *stream) {
  return eakv_extend_attention_depths(caches, n_caches, layer, n_new, q, out, n_q_heads, scale, window,
                                      tree, nullptr, lse, workspace, workspace_bytes, stream);
}

int eakv_extend_attention_depths(const eakv_cache_t *const *caches, int n_caches, int layer,
                                 const int *n_new, const eakv_rows_t *q, const eakv_rows_t *out,
                                 int n_q_heads, float scale, int window, const uint64_t *tree,
                                 const int32_t *depth, float *lse, void *workspace,
                                 size_t workspace_bytes, void *stream) {
  clear_error();
  ExtendArgs a;
  TokenBatch b;
  int total = 0;
  if (!q || !out) return refuse("NULL q or out");
  int rc = check_call(caches, n_caches, n_new, q->dtype, n_q_heads, window, tree != nullptr, a, b, total);
  if (rc || total == 0) return rc;
  const eakv_cache_t *c0 = caches[0];
  if ((rc = check_rows(q, "q", "extend_attention")) ||
      (rc = check_out_rows(out, "out", "extend_attention", total, n_q_heads, c0->head_dim)))
    return rc;
  if (q->dtype != out->dtype) return refuse("q and out differ in element type");
  if (layer < 0 || layer >= c0->n_layers) return refuse("layer out of range");
  // 2.3e38 log2 e is below f32's largest number
  if (!(fabsf(scale) <= 2.3e38f)) return refuse("scale is not a number below 2.3e38");
  if ((uintptr_t)tree % 8 || (uintptr_t)lse % 4 || (uintptr_t)depth % 4)
    return refuse("misaligned tree, depth or lse");
  if (depth && !tree) return refuse("depths without a tree");
  if ((uintptr_t)workspace % 16) return refuse("workspace must be 16-byte aligned");
  a.layer = layer;
  a.q = rows_of(q);
  a.out = rows_of(out);
  a.scale_log2 = (scale == 0.0f ? 1.0f / sqrtf((float)c0->head_dim) : scale) * kLog2e;
  a.tree = (const unsigned long long *)tree;
  a.depth = depth;
  a.lse = lse;
  a.wait_budget = t_wait_budget ? t_wait_budget : kWaitBudget;
  a.test_stall = t_test_stall;
  DeviceGuard g(c0->device);
  a.status = device_status_ptr();
  if (!a.status) return refuse("device status word unavailable");
  Part p[2];
  rc = plan(a, b, c0->device, tree ? (depth ? kTreeDepths : kTree) : kCausal, p);
  if (rc) return rc;
  cudaStream_t s = stream ? (cudaStream_t)stream : c0->stream;
  const size_t need = workspace_of(a, p);
  void *data = nullptr;
  if (need && workspace) {
    if (workspace_bytes < need) {
      set_error(EAKV_ERR_INVALID, "extend_attention: workspace of %zu bytes, %zu needed",
                workspace_bytes, need);
      return EAKV_ERR_INVALID;
    }
    a.cnt = (unsigned *)workspace;
    data = (uint8_t *)workspace + kCounterBytes;
  } else if (need) {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    rc = check_cuda(cudaStreamIsCapturing(s, &cap), "extend_attention: stream");
    if (rc) return rc;
    if (cap != cudaStreamCaptureStatusNone)
      return refuse("a captured call needs a workspace of its own (eakv_extend_workspace)");
    rc = cache_parts_workspace(c0, kSplitItems, need - kCounterBytes, &a.cnt, &data);
    if (rc) return rc;
  }
  const bool vec = rows_vec(q) && rows_vec(out);
  for (int k = 0; k < 2; k++) {   // the long ones first
    a.n_caches = p[k].n_caches;
    a.tile_rows = p[k].tile_rows;
    a.unit_pages = p[k].unit_pages;
    a.run = p[k].run;
    a.units = p[k].units;
    a.overhead = p[k].overhead;
    a.n_splits = p[k].n_splits;
    a.split_units = p[k].split_units;
    const size_t rows = (size_t)p[k].slots * a.tile_rows;
    a.part_o = (float *)data;
    a.part_m = a.part_o + rows * c0->head_dim;
    a.part_l = a.part_m + rows;
    for (int t0 = 0; t0 < p[k].tiles && !rc; t0 += p[k].launch_tiles) {
      a.tile_lo = t0;
      a.tile_hi = t0 + p[k].launch_tiles < p[k].tiles ? t0 + p[k].launch_tiles : p[k].tiles;
      const int blocks = a.run ? p[k].n_runs : (a.tile_hi - a.tile_lo) * a.geom.n_heads * a.n_splits;
      rc = p[k].umma ? extend_umma_launch(a, p[k].b, p[k].runs, blocks, vec, s)
                     : extend_mma_launch(a, p[k].b, p[k].runs, blocks, vec, s);
    }
  }
  return rc;
}

}  // extern "C"
