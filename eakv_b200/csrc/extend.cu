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

// Longest split in pages. The tensor core adds into its f32 sums by
// truncation, a drift of up to 2^-24 of the sum per step of 16 positions. In
// the warp-level kernel four warps take pages in turn: 64 pages are 64 steps of a
// warp (2^-18 at worst, 2^-19 on average, below what f32 results ask for), and 256
// pages 2^-16, below 16-bit results' own rounding; in the tcgen05 kernel one
// sum takes every step, and 1024 pages are 2^-12, 2^-13 on average, against the
// 2^-9 of its outputs.
constexpr int kSplitPagesF32 = 64, kSplitPages16 = 256, kSplitPagesUmma = 1024;

// Rows (new tokens x query heads per KV head) up to which 16-bit calls take the
// warp-level kernel.
constexpr int kMmaRows = 32;

// One launch's caches and plan: a call's caches with few rows and those with
// many go to different kernels.
struct Part {
  bool umma;
  int tiles, launch_tiles;   // row tiles in all and per launch
  size_t records;            // bytes of split records of one launch
  int tile_rows, n_splits, split_pages, n_caches;
  ExtendBatch b;
};

int sm_count(int dev) {
  int n = 0;
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

// The caches of `t` that belong to the part, their row tiles, splits and record
// bytes. Call with the caches' device current.
int plan(const ExtendArgs &a, const TokenBatch &t, int device, bool tree, bool umma, Part &p) {
  p.umma = umma;
  p.tile_rows = umma ? kExtendUmmaRows : kExtendMmaRows;
  p.n_caches = 0;
  p.records = 0;
  p.n_splits = p.split_pages = 1;
  const int heads = a.geom.n_heads;
  long long tiles = 0;
  int max_pages = 1;
  for (int i = 0; i < a.n_caches; i++) {
    const int n = t.first[i + 1] - t.first[i];
    const bool many = a.dtype != EAKV_F32 && t_force_path != 2 &&
                      ((long long)n * a.G > kMmaRows || t_force_path == 3);
    if (n == 0 || many != umma) continue;
    const int k = p.n_caches++;
    p.b.base[k] = t.base[i];
    p.b.old[k] = t.pos[i];
    p.b.first[k] = t.first[i];
    p.b.n_new[k] = n;
    p.b.tile0[k] = (int)tiles;
    tiles += ((long long)n * a.G + p.tile_rows - 1) / p.tile_rows;
    long long span = (long long)t.pos[i] + n;   // positions a tile may attend
    if (a.window > 0) {
      // its tokens' windows (a tree's tokens may look ahead within n)
      const long long w = (long long)a.window + (tree ? n : p.tile_rows / a.G + 1);
      if (w < span) span = w + kPagePositions;    // not page-aligned
    }
    const int pages = (int)((span + kPagePositions - 1) / kPagePositions);
    if (pages > max_pages) max_pages = pages;
  }
  for (int i = p.n_caches; i <= kMaxBatch; i++) p.b.tile0[i] = (int)tiles;
  p.tiles = p.launch_tiles = (int)tiles;
  if (p.tiles == 0) return EAKV_OK;
  if (tiles * heads > (1ll << 30)) {
    set_error(EAKV_ERR_INVALID, "extend_attention: more than 2^30 tiles of rows");
    return EAKV_ERR_INVALID;
  }
  const int per_sm = umma ? 1 : extend_mma_resident(a.geom.gpd * 64, a.dtype);
  if (per_sm <= 0) return EAKV_ERR_INVALID;   // recorded by the lookup
  const int cap = umma ? kSplitPagesUmma : a.dtype == EAKV_F32 ? kSplitPagesF32 : kSplitPages16;
  const int lo = (max_pages + cap - 1) / cap;
  int hi = max_pages / 2;   // two pages at least: one per warp, or one tile
  if (hi < lo) hi = lo;
  if (hi > 4096) hi = 4096;
  int ns = t_force_splits > 0 ? t_force_splits
                              : choose_splits(tiles * heads, max_pages, lo, hi, per_sm, sm_count(device));
  if (ns > max_pages) ns = max_pages;
  if (ns < 1) ns = 1;
  p.split_pages = (max_pages + ns - 1) / ns;
  if (umma) p.split_pages += p.split_pages & 1;   // tiles of two pages
  p.n_splits = (max_pages + p.split_pages - 1) / p.split_pages;
  if (p.n_splits > 1) {
    if (p.launch_tiles > kSplitItems / heads) p.launch_tiles = kSplitItems / heads;
    p.records = (size_t)p.launch_tiles * heads * p.n_splits * p.tile_rows *
                (a.geom.gpd * 64 + 2) * sizeof(float);
  }
  // a launch's blocks: fewer row tiles per launch where splits would pass 2^30
  while ((long long)p.launch_tiles * heads * p.n_splits > (1ll << 30) && p.launch_tiles > 1)
    p.launch_tiles = (p.launch_tiles + 1) / 2;
  return EAKV_OK;
}

// Workspace bytes of both parts, which run one after the other on it.
size_t workspace_of(const Part (&p)[2]) {
  const size_t r = p[0].records > p[1].records ? p[0].records : p[1].records;
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
  for (int k = 0; k < 2 && !rc; k++) rc = plan(a, b, caches[0]->device, tree != 0, k == 0, p[k]);
  if (!rc) *bytes = workspace_of(p);
  return rc;
}

int eakv_extend_attention(const eakv_cache_t *const *caches, int n_caches, int layer,
                          const int *n_new, const eakv_rows_t *q, const eakv_rows_t *out,
                          int n_q_heads, float scale, int window, const uint64_t *tree, float *lse,
                          void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  ExtendArgs a;
  TokenBatch b;
  int total = 0;
  if (!q || !out) return refuse("NULL q or out");
  int rc = check_call(caches, n_caches, n_new, q->dtype, n_q_heads, window, tree != nullptr, a, b, total);
  if (rc || total == 0) return rc;
  if ((rc = check_rows(q, "q", "extend_attention")) ||
      (rc = check_rows(out, "out", "extend_attention")))
    return rc;
  const eakv_cache_t *c0 = caches[0];
  if (q->dtype != out->dtype) return refuse("q and out differ in element type");
  if (layer < 0 || layer >= c0->n_layers) return refuse("layer out of range");
  if (!(fabsf(scale) <= 3.0e38f)) return refuse("scale is not a finite number");
  if ((uintptr_t)tree % 8 || (uintptr_t)lse % 4) return refuse("misaligned tree or lse");
  if ((uintptr_t)workspace % 16) return refuse("workspace must be 16-byte aligned");
  a.layer = layer;
  a.q = rows_of(q);
  a.out = rows_of(out);
  a.scale_log2 = (scale == 0.0f ? 1.0f / sqrtf((float)c0->head_dim) : scale) * kLog2e;
  a.tree = (const unsigned long long *)tree;
  a.lse = lse;
  a.wait_budget = t_wait_budget ? t_wait_budget : kWaitBudget;
  a.test_stall = t_test_stall;
  DeviceGuard g(c0->device);
  a.status = device_status_ptr();
  if (!a.status) return refuse("device status word unavailable");
  Part p[2];
  for (int k = 0; k < 2 && !rc; k++) rc = plan(a, b, c0->device, tree != nullptr, k == 0, p[k]);
  if (rc) return rc;
  cudaStream_t s = stream ? (cudaStream_t)stream : c0->stream;
  const size_t need = workspace_of(p);
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
    rc = cache_workspace(c0, kSplitItems, need - kCounterBytes, &a.cnt, &data);
    if (rc) return rc;
  }
  const bool vec = rows_vec(q) && rows_vec(out);
  for (int k = 0; k < 2; k++) {   // the long ones first
    a.n_caches = p[k].n_caches;
    a.tile_rows = p[k].tile_rows;
    a.n_splits = p[k].n_splits;
    a.split_pages = p[k].split_pages;
    const size_t rows = (size_t)p[k].launch_tiles * a.geom.n_heads * a.n_splits * a.tile_rows;
    a.part_o = (float *)data;
    a.part_m = a.part_o + rows * c0->head_dim;
    a.part_l = a.part_m + rows;
    for (int t0 = 0; t0 < p[k].tiles && !rc; t0 += p[k].launch_tiles) {
      a.tile_lo = t0;
      a.tile_hi = t0 + p[k].launch_tiles < p[k].tiles ? t0 + p[k].launch_tiles : p[k].tiles;
      const int blocks = (a.tile_hi - a.tile_lo) * a.geom.n_heads * a.n_splits;
      rc = p[k].umma ? extend_umma_launch(a, p[k].b, blocks, vec, s)
                     : extend_mma_launch(a, p[k].b, blocks, vec, s);
    }
  }
  return rc;
}

}  // extern "C"
