// move.cu - positions moved between caches as they are (copy to several,
// gather by a list, compact in place), and positions of several caches read
// back as values.
//
// move_kernel: a position of one (layer, K/V, head) unit is gpd*32 bytes of
// nibbles and gpd (scale, bias) pairs in its page, both contiguous; a block
// takes kMovePos positions of a unit, each thread 16-byte pieces of them with
// all its loads issued before its first store, and writes every destination
// from one read. Bound: HBM, 40 bytes per group read and, per destination,
// written. Offsets between source and destination need no special case: a
// position is moved whole and its pieces are 16-byte aligned in both pages
// (8-byte for the one (scale, bias) pair of head_dim 64). Measured at 32 layers of
// 8 heads of 128 and 8192 positions, half of them moved: a copy runs at the rate of a
// plain device copy (58 us), a gather by a list at 0.75 of it (73), a compaction in place at
// 0.49 (111), whose block per (layer, K/V, head) needs many of these: 58 us for 2 layers
// of 16384, where the copy takes 8.
//
// In place, a place below its source may be the source of an earlier place
// (index >= its place is required and checked): one block walks a unit's
// places in order, and the loads of a tile come before a barrier, its stores
// behind it; the next tile's loads go out ahead of those stores, which they
// cannot meet, since its sources lie at or above its own places.
#include <string.h>

#include "pipeline.cuh"
#include "tokens.cuh"

namespace eakv {
namespace {

constexpr int kThreads = 256;
constexpr int kMovePos = 256;   // positions per block (or tile)

struct MoveTargets {
  uint8_t *base[kMaxBatch];
  int n_pages[kMaxBatch];
};

struct MoveArgs {
  PageGeom src;              // geometry of the source (the destinations differ in n_pages)
  const uint8_t *src_base;
  int n_dst, dst_pos, src_pos, n;
  const int32_t *index;      // or NULL: src_pos + j
  long long layer_stride, head_stride;
  int limit;                 // index values lie in [0, limit)
  int *status;
};

__device__ __forceinline__ size_t vexp_offset(const PageGeom &g, int n_pages) {
  return ((size_t)g.n_layers * 2 * g.n_heads * n_pages * g.page_bytes + 255) & ~(size_t)255;
}

// The pieces of kMovePos positions that one thread moves: GPD 1 or 2 groups
// per position (0: any number, one piece at a time).
template <int GPD> struct Pieces {
  static constexpr int NIB = 2 * GPD * kMovePos / kThreads;   // 16-byte nibble pieces
  uint4 w[NIB];
  int wj[NIB];          // place within the call, -1: none
  float4 sb;            // (scale, bias) pairs of one position
  int sbj;
};

// Source position of place j, or -1 (beyond the range, or a bad index, which
// is reported).
template <bool kInPlace>
__device__ __forceinline__ int source(const MoveArgs &a, const int32_t *list, int j) {
  if (j >= a.n) return -1;
  if (!list) return a.src_pos + j;
  const int s = __ldg(list + j);
  if (s < 0 || s >= a.limit || (kInPlace && s < a.dst_pos + j)) {
    atomicOr(a.status, kStatusBadIndex);
    return -1;
  }
  return s;
}

template <int GPD, bool kInPlace>
__device__ __forceinline__ void fetch(const MoveArgs &a, const uint8_t *unit, const int32_t *list,
                                      int j0, Pieces<GPD> &p) {
  int sp[Pieces<GPD>::NIB], ss;
#pragma unroll
  for (int k = 0; k < Pieces<GPD>::NIB; k++) {
    const int j = j0 + (threadIdx.x + k * kThreads) / (2 * GPD);
    sp[k] = source<kInPlace>(a, list, j);
    p.wj[k] = sp[k] >= 0 ? j : -1;
  }
  ss = source<kInPlace>(a, list, j0 + threadIdx.x);
  p.sbj = ss >= 0 ? j0 + (int)threadIdx.x : -1;
#pragma unroll
  for (int k = 0; k < Pieces<GPD>::NIB; k++)
    if (p.wj[k] >= 0)
      p.w[k] = *reinterpret_cast<const uint4 *>(
          unit + (size_t)(sp[k] / kPagePositions) * a.src.page_bytes +
          (size_t)(sp[k] % kPagePositions) * (GPD * 32) + 16 * (threadIdx.x % (2 * GPD)));
  if (p.sbj >= 0) {
    const uint8_t *at = unit + (size_t)(ss / kPagePositions) * a.src.page_bytes + a.src.nib_bytes +
                        (size_t)(ss % kPagePositions) * (GPD * 8);
    if constexpr (GPD == 2) {
      p.sb = *reinterpret_cast<const float4 *>(at);
    } else {
      const float2 v = *reinterpret_cast<const float2 *>(at);
      p.sb = make_float4(v.x, v.y, 0.0f, 0.0f);
    }
  }
}

template <int GPD>
__device__ __forceinline__ void put(const MoveArgs &a, uint8_t *unit, const Pieces<GPD> &p) {
#pragma unroll
  for (int k = 0; k < Pieces<GPD>::NIB; k++)
    if (p.wj[k] >= 0) {
      const int d = a.dst_pos + p.wj[k];
      *reinterpret_cast<uint4 *>(unit + (size_t)(d / kPagePositions) * a.src.page_bytes +
                                 (size_t)(d % kPagePositions) * (GPD * 32) +
                                 16 * (threadIdx.x % (2 * GPD))) = p.w[k];
    }
  if (p.sbj >= 0) {
    const int d = a.dst_pos + p.sbj;
    uint8_t *at = unit + (size_t)(d / kPagePositions) * a.src.page_bytes + a.src.nib_bytes +
                  (size_t)(d % kPagePositions) * (GPD * 8);
    if constexpr (GPD == 2) *reinterpret_cast<float4 *>(at) = p.sb;
    else *reinterpret_cast<float2 *>(at) = make_float2(p.sb.x, p.sb.y);
  }
}

// Grid (chunks of positions, units).
template <int GPD>
__global__ void __launch_bounds__(kThreads)
move_kernel(const __grid_constant__ MoveArgs a, const __grid_constant__ MoveTargets to) {
  const int u = blockIdx.y;   // (layer * 2 + kv) * heads + head
  const int h = u % a.src.n_heads, lkv = u / a.src.n_heads;
  const int32_t *list =
      a.index ? a.index + (lkv >> 1) * a.layer_stride + h * a.head_stride : nullptr;
  const uint8_t *unit = a.src_base + (size_t)u * a.src.n_pages * a.src.page_bytes;
  Pieces<GPD> p;
  fetch<GPD, false>(a, unit, list, blockIdx.x * kMovePos, p);
  for (int i = 0; i < a.n_dst; i++)
    put<GPD>(a, to.base[i] + (size_t)u * to.n_pages[i] * a.src.page_bytes, p);
  if (blockIdx.x == 0 && (lkv & 1)) {
    // the V-scale exponent bound of the source covers every position moved
    const int e = vexp_table(a.src_base, a.src)[(lkv >> 1) * a.src.n_heads + h];
    for (int i = threadIdx.x; i < a.n_dst; i += kThreads)
      atomicMax(reinterpret_cast<int *>(to.base[i] + vexp_offset(a.src, to.n_pages[i])) +
                    (lkv >> 1) * a.src.n_heads + h, e);
  }
}

// The same for any number of groups per position, one 8-byte piece at a time:
// head_dims that only quantize, files and these moves serve.
__global__ void __launch_bounds__(kThreads)
move_any_kernel(const __grid_constant__ MoveArgs a, const __grid_constant__ MoveTargets to) {
  const int u = blockIdx.y;
  const int h = u % a.src.n_heads, lkv = u / a.src.n_heads;
  const int32_t *list =
      a.index ? a.index + (lkv >> 1) * a.layer_stride + h * a.head_stride : nullptr;
  const uint8_t *unit = a.src_base + (size_t)u * a.src.n_pages * a.src.page_bytes;
  const int per = 5 * a.src.gpd;   // 8-byte pieces of a position: 4 of nibbles, 1 pair per group
  for (int x = threadIdx.x; x < kMovePos * per; x += kThreads) {
    const int j = blockIdx.x * kMovePos + x / per, c = x % per;
    const int s = source<false>(a, list, j);
    if (s < 0) continue;
    const int d = a.dst_pos + j;
    const bool nib = c < 4 * a.src.gpd;
    auto off = [&](int pos) {
      return (size_t)(pos / kPagePositions) * a.src.page_bytes +
             (nib ? (size_t)(pos % kPagePositions) * a.src.gpd * 32 + 8 * c
                  : a.src.nib_bytes + (size_t)(pos % kPagePositions) * a.src.gpd * 8 +
                        8 * (c - 4 * a.src.gpd));
    };
    const uint2 v = *reinterpret_cast<const uint2 *>(unit + off(s));
    for (int i = 0; i < a.n_dst; i++)
      *reinterpret_cast<uint2 *>(to.base[i] + (size_t)u * to.n_pages[i] * a.src.page_bytes + off(d)) = v;
  }
  if (blockIdx.x == 0 && (lkv & 1)) {
    const int e = vexp_table(a.src_base, a.src)[(lkv >> 1) * a.src.n_heads + h];
    for (int i = threadIdx.x; i < a.n_dst; i += kThreads)
      atomicMax(reinterpret_cast<int *>(to.base[i] + vexp_offset(a.src, to.n_pages[i])) +
                    (lkv >> 1) * a.src.n_heads + h, e);
  }
}

// In place: one block per unit, tile after tile.
template <int GPD>
__global__ void __launch_bounds__(kThreads)
compact_kernel(const __grid_constant__ MoveArgs a, uint8_t *base) {
  const int u = blockIdx.x;
  const int h = u % a.src.n_heads, lkv = u / a.src.n_heads;
  const int32_t *list = a.index + (lkv >> 1) * a.layer_stride + h * a.head_stride;
  uint8_t *unit = base + (size_t)u * a.src.n_pages * a.src.page_bytes;
  Pieces<GPD> p, next;
  fetch<GPD, true>(a, unit, list, 0, p);
  for (int j0 = 0; j0 < a.n; j0 += kMovePos) {
    __syncthreads();   // the whole tile is read
    fetch<GPD, true>(a, unit, list, j0 + kMovePos, next);
    put<GPD>(a, unit, p);
    p = next;
  }
}

// ---- read back ------------------------------------------------------------------

struct ReadArgs {
  PageGeom geom;
  int n_caches, layer0, total;
  Rows out[2];               // K, V
  long long layer_stride;    // elements
};

constexpr int kReadTok = 8;   // positions per warp, their loads first

// Four nibbles of a word (from bit sh, every eighth) as f32: each byte placed in
// the mantissa of 2^23, and 2^23 taken off.
__device__ __forceinline__ void nibbles4(uint32_t word, int sh, float (&n)[4]) {
  const uint32_t w = (word >> sh) & 0x0F0F0F0Fu;
#pragma unroll
  for (int e = 0; e < 4; e++)
    n[e] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 + e)) - 8388608.0f;
}

// Warp: kReadTok neighbouring tokens of one (layer, K/V, head) (two heads at
// head_dim 64): 128 elements per token, four per lane. Bound: HBM, mostly the
// values written: 8192 positions of 4 layers as f32 in 53 us (310 MB, 0.90 of the
// copy rate).
template <int HD, typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
read_kernel(const __grid_constant__ ReadArgs a, const __grid_constant__ TokenBatch batch) {
  constexpr int HPW = 128 / HD, LPR = HD / 4, GPD = HD / 64;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hsets = (a.geom.n_heads + HPW - 1) / HPW;
  const int lkv = blockIdx.y;                 // layer row * 2 + kv
  const Rows out = a.out[lkv & 1];
  if (!out.data) return;
  const int layer = a.layer0 + (lkv >> 1);
  const unsigned w = blockIdx.x * (kThreads / 32) + warp;
  const int run = w / hsets;   // heads vary fastest: a block's stores are near
  const int t0 = run * kReadTok, h = (int)(w - run * hsets) * HPW + lane / LPR;
  if (t0 >= a.total || h >= a.geom.n_heads) return;
  const int d0 = 4 * (lane % LPR), grp = d0 >> 6, k = d0 & 63;
  uint32_t word[kReadTok];
  float2 sb[kReadTok];
  int cache = token_cache(batch, a.n_caches, t0);
  // the head's pages of the cache that the tokens are in, and where it ends
  const uint8_t *unit = batch.base[cache] + page_index(a.geom, layer, lkv & 1, h, 0) * a.geom.page_bytes;
  int end = batch.first[cache + 1], shift = batch.pos[cache] - batch.first[cache];
#pragma unroll
  for (int r = 0; r < kReadTok; r++) {
    const int t = t0 + r;
    if (t < a.total) {
      while (t >= end) {   // first[n_caches] = total > t
        cache++;
        unit = batch.base[cache] + page_index(a.geom, layer, lkv & 1, h, 0) * a.geom.page_bytes;
        end = batch.first[cache + 1];
        shift = batch.pos[cache] - batch.first[cache];
      }
      const int at = t + shift, slot = (at % kPagePositions) * GPD + grp;
      const uint8_t *pp = unit + (size_t)(at / kPagePositions) * a.geom.page_bytes;
      word[r] = *reinterpret_cast<const uint32_t *>(pp + slot * 32 + (k & 31));
      sb[r] = *reinterpret_cast<const float2 *>(pp + a.geom.nib_bytes + slot * 8);
    }
  }
  const int sh = k < 32 ? 0 : 4;
  T *base = reinterpret_cast<T *>(out.data) + (long long)(lkv >> 1) * a.layer_stride +
            (long long)h * out.head_stride + d0 + (long long)t0 * out.token_stride;
#pragma unroll
  for (int r = 0; r < kReadTok; r++) {
    if (t0 + r >= a.total) break;
    float v[4];
    nibbles4(word[r], sh, v);
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = fmaf(v[e], sb[r].x, sb[r].y);
    store4<T, kVec>(base, v);
    base += out.token_stride;
  }
}

template <int HD, typename T>
cudaError_t read_launch(const ReadArgs &a, const TokenBatch &b, int n_layers, bool vec,
                        cudaStream_t s) {
  constexpr int HPW = 128 / HD;
  const long long warps = (long long)((a.total + kReadTok - 1) / kReadTok) *
                          ((a.geom.n_heads + HPW - 1) / HPW);
  if (warps > (1ll << 31)) return cudaErrorInvalidValue;   // a warp's number is 32 bits
  const dim3 grid((unsigned)((warps + kThreads / 32 - 1) / (kThreads / 32)), 2 * n_layers);
  if (vec) read_kernel<HD, T, true><<<grid, kThreads, 0, s>>>(a, b);
  else read_kernel<HD, T, false><<<grid, kThreads, 0, s>>>(a, b);
  return cudaGetLastError();
}

int refuse(const char *who, const char *what) {
  set_error(EAKV_ERR_INVALID, "%s: %s", who, what);
  return EAKV_ERR_INVALID;
}

int units_of(const eakv_cache_t *c) { return c->n_layers * 2 * c->n_kv_heads; }

int move_launch(const MoveArgs &a, const MoveTargets &to, int units, cudaStream_t s) {
  const dim3 grid((a.n + kMovePos - 1) / kMovePos, units);
  if (a.src.gpd == 1) move_kernel<1><<<grid, kThreads, 0, s>>>(a, to);
  else if (a.src.gpd == 2) move_kernel<2><<<grid, kThreads, 0, s>>>(a, to);
  else move_any_kernel<<<grid, kThreads, 0, s>>>(a, to);
  return check_cuda(cudaGetLastError(), "move: launch");
}

// What copy and gather ask of a source and a destination.
int check_pair(const eakv_cache_t *dst, const eakv_cache_t *src, int dst_pos, int n,
               const char *who) {
  if (!dst || dst == src) return refuse(who, "NULL destination, or the source itself");
  if (dst->n_layers != src->n_layers || dst->n_kv_heads != src->n_kv_heads ||
      dst->head_dim != src->head_dim || dst->device != src->device)
    return refuse(who, "caches differ in layers, heads, head_dim or device");
  if (dst_pos < 0 || dst_pos > dst->seq_len || (long long)dst_pos + n > dst->max_seq_len)
    return refuse(who, "destination range outside the cache or beyond its seq_len");
  return EAKV_OK;
}

int check_units(const eakv_cache_t *c, const char *who) {
  if ((long long)c->n_layers * 2 * c->n_kv_heads > 65535)   // grid y
    return refuse(who, "more than 65535 (layer, K/V, head) units");
  return EAKV_OK;
}

}  // namespace
}  // namespace eakv

using namespace eakv;

extern "C" {

int eakv_cache_copy(eakv_cache_t *const *dsts, int n_dst, int dst_pos, const eakv_cache_t *src,
                    int src_pos, int n, void *stream) {
  clear_error();
  const char *who = "cache_copy";
  if (!dsts || n_dst <= 0 || n_dst > kMaxBatch || !src)
    return refuse(who, "need a source and 1..256 destinations");
  if (n < 0 || src_pos < 0 || (long long)src_pos + n > src->seq_len)
    return refuse(who, "source range outside the cache's seq_len");
  int rc = check_units(src, who);
  for (int i = 0; i < n_dst && !rc; i++) {
    rc = check_pair(dsts[i], src, dst_pos, n, who);
    for (int j = 0; j < i && !rc; j++)
      if (dsts[i] == dsts[j]) rc = refuse(who, "the same destination twice");
  }
  if (rc) return rc;
  if (n > 0 && src->geom.gpd > 0) {
    DeviceGuard g(src->device);
    MoveArgs a = {};
    MoveTargets to;
    a.src = src->geom;
    a.src_base = src->d_buf;
    a.n_dst = n_dst;
    a.dst_pos = dst_pos;
    a.src_pos = src_pos;
    a.n = n;
    for (int i = 0; i < n_dst; i++) {
      to.base[i] = dsts[i]->d_buf;
      to.n_pages[i] = dsts[i]->geom.n_pages;
    }
    rc = move_launch(a, to, units_of(src), stream ? (cudaStream_t)stream : src->stream);
    if (rc) return rc;
  }
  for (int i = 0; i < n_dst; i++) dsts[i]->seq_len = dst_pos + n;
  return EAKV_OK;
}

int eakv_cache_fork(const eakv_cache_t *src, int n, int max_seq_len, eakv_cache_t **out) {
  clear_error();
  const char *who = "cache_fork";
  if (!out) return refuse(who, "NULL result");
  *out = nullptr;
  if (!src || n < 0 || n > src->seq_len || max_seq_len <= 0 || n > max_seq_len)
    return refuse(who, "invalid argument");
  DeviceGuard g(src->device);
  eakv_cache_t *c = eakv_cache_create(src->n_layers, src->n_kv_heads, src->head_dim, max_seq_len);
  if (!c) return eakv_last_error();
  int rc = eakv_cache_copy(&c, 1, 0, src, 0, n, src->stream);
  if (!rc && n > 0) {
    // the new cache's own stream goes on behind the copy
    cudaEvent_t ev = nullptr;
    rc = check_cuda(cudaEventCreateWithFlags(&ev, cudaEventDisableTiming), "cache_fork: event");
    if (!rc) rc = check_cuda(cudaEventRecord(ev, src->stream), "cache_fork: event");
    if (!rc) rc = check_cuda(cudaStreamWaitEvent(c->stream, ev, 0), "cache_fork: event");
    if (ev) cudaEventDestroy(ev);
  }
  if (rc) {
    cudaStreamSynchronize(src->stream);   // the copy may still be writing
    eakv_cache_free(c);
    return rc;
  }
  *out = c;
  return EAKV_OK;
}

int eakv_cache_gather(eakv_cache_t *dst, int dst_pos, const eakv_cache_t *src, const int32_t *index,
                      int64_t layer_stride, int64_t head_stride, int n, void *stream) {
  clear_error();
  const char *who = "cache_gather";
  if (!src || (!index && n > 0) || n < 0 || layer_stride < 0 || head_stride < 0)
    return refuse(who, "invalid argument");
  if ((uintptr_t)index % 4) return refuse(who, "misaligned index");
  int rc = check_units(src, who);
  if (!rc) rc = check_pair(dst, src, dst_pos, n, who);
  if (rc) return rc;
  if (n > 0 && src->geom.gpd > 0) {
    DeviceGuard g(src->device);
    MoveArgs a = {};
    MoveTargets to;
    a.src = src->geom;
    a.src_base = src->d_buf;
    a.n_dst = 1;
    a.dst_pos = dst_pos;
    a.n = n;
    a.index = index;
    a.layer_stride = layer_stride;
    a.head_stride = head_stride;
    a.limit = src->seq_len;
    a.status = device_status_ptr();
    if (!a.status) return refuse(who, "device status word unavailable");
    to.base[0] = dst->d_buf;
    to.n_pages[0] = dst->geom.n_pages;
    rc = move_launch(a, to, units_of(src), stream ? (cudaStream_t)stream : src->stream);
    if (rc) return rc;
  }
  dst->seq_len = dst_pos + n;
  return EAKV_OK;
}

int eakv_cache_compact(eakv_cache_t *c, int begin, const int32_t *index, int64_t layer_stride,
                       int64_t head_stride, int n, void *stream) {
  clear_error();
  const char *who = "cache_compact";
  if (!c || (!index && n > 0) || n < 0 || layer_stride < 0 || head_stride < 0 || begin < 0 ||
      begin > c->seq_len || (long long)begin + n > c->max_seq_len)
    return refuse(who, "invalid argument");
  if ((uintptr_t)index % 4) return refuse(who, "misaligned index");
  if (c->geom.gpd > 2) return refuse(who, "head_dim above 128");
  if (n > 0 && c->geom.gpd > 0) {
    DeviceGuard g(c->device);
    MoveArgs a = {};
    a.src = c->geom;
    a.src_base = c->d_buf;
    a.dst_pos = begin;
    a.n = n;
    a.index = index;
    a.layer_stride = layer_stride;
    a.head_stride = head_stride;
    a.limit = c->max_seq_len;
    a.status = device_status_ptr();
    if (!a.status) return refuse(who, "device status word unavailable");
    cudaStream_t s = stream ? (cudaStream_t)stream : c->stream;
    if (c->geom.gpd == 1) compact_kernel<1><<<units_of(c), kThreads, 0, s>>>(a, c->d_buf);
    else compact_kernel<2><<<units_of(c), kThreads, 0, s>>>(a, c->d_buf);
    int rc = check_cuda(cudaGetLastError(), "cache_compact: launch");
    if (rc) return rc;
  }
  c->seq_len = begin + n;
  return EAKV_OK;
}

int eakv_cache_read(const eakv_cache_t *const *caches, int n_caches, int layer0, int n_layers,
                    const int *begin, const int *n, const eakv_rows_t *k, const eakv_rows_t *v,
                    int64_t layer_stride, void *stream) {
  clear_error();
  const char *who = "cache_read";
  if (!caches || n_caches <= 0 || !caches[0] || !begin) return refuse(who, "invalid argument");
  TokenBatch b;
  ReadArgs a = {};
  const eakv_cache_t *c0 = caches[0];
  int rc = token_batch(caches, n_caches, c0->n_kv_heads, begin, n, who, b, a.total);
  if (rc || a.total == 0) return rc;
  if (!k && !v) return refuse(who, "neither k nor v");
  if ((k && (rc = check_out_rows(k, "k", who, a.total, c0->n_kv_heads, c0->head_dim))) ||
      (v && (rc = check_out_rows(v, "v", who, a.total, c0->n_kv_heads, c0->head_dim))))
    return rc;
  if (k && v && k->dtype != v->dtype) return refuse(who, "k and v differ in element type");
  if (layer0 < 0 || n_layers < 1 || (long long)layer0 + n_layers > c0->n_layers || n_layers > 32767 ||
      layer_stride < 0)
    return refuse(who, "layers out of range");
  if (n_layers > 1 && layer_stride < c0->head_dim) return refuse(who, "layers' rows overlap");
  DeviceGuard g(c0->device);
  a.geom = c0->geom;
  a.n_caches = n_caches;
  a.layer0 = layer0;
  a.out[0] = rows_of(k);
  a.out[1] = rows_of(v);
  a.layer_stride = layer_stride;
  const bool vec = rows_vec(k) && rows_vec(v) && layer_stride % 4 == 0;
  const int dtype = k ? k->dtype : v->dtype;
  cudaStream_t s = stream ? (cudaStream_t)stream : c0->stream;
  cudaError_t e;
  if (c0->head_dim == 128)
    e = dtype == EAKV_F32   ? read_launch<128, float>(a, b, n_layers, vec, s)
        : dtype == EAKV_F16 ? read_launch<128, __half>(a, b, n_layers, vec, s)
                            : read_launch<128, __nv_bfloat16>(a, b, n_layers, vec, s);
  else
    e = dtype == EAKV_F32   ? read_launch<64, float>(a, b, n_layers, vec, s)
        : dtype == EAKV_F16 ? read_launch<64, __half>(a, b, n_layers, vec, s)
                            : read_launch<64, __nv_bfloat16>(a, b, n_layers, vec, s);
  return check_cuda(e, "cache_read: launch");
}

}  // extern "C"
