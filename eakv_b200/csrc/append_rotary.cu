// append_rotary.cu - the new tokens of one layer of a batch of caches: q and
// k turned by their rotary positions, k and v quantized into the pages.
//
// Mathematics. A pair (a, b) of a row turns by the angle of (position, pair):
//   a' = a c - b s,   b' = b c + a s.
// Keys: both products are exact in f64 (24 + 24 bits), so a' is rounded to
// f64 and then to f32, and what is quantized is that f32 value; a nibble
// depends on its whole group's minimum and maximum, so a last-bit difference
// in a key could move a nibble by one, a whole quantum, and the keys are held
// to one defined rounding. Queries leave in their own type and are turned in
// f32 with one fma (error 1.5 ulp of f32).
// The quantizer is the cache's own (quantize.cu): the same minimum, maximum,
// signed-zero, NaN and truncation rules, so that the pages equal
// eakv_cache_append's on the same f32 rows bit for bit.
//
// Mapping. A warp takes 128 elements (one row of head_dim 128, two of 64),
// four neighbouring ones per lane (8- or 16-byte loads); a 64-element group
// is 16 lanes. The partner of a rotated element is in the same lane
// (interleaved) or rot_dim/8 lanes away (halves), one shuffle per element;
// group minima and maxima are four shuffle steps; the high nibbles come from
// eight lanes up, so a group's 32 bytes leave as eight 4-byte stores. A warp
// takes kRowSets sets of heads of one token with their loads issued first,
// and reads the token's cosines and sines once for all of them.
//
// Bound: HBM for long chunks (q, k, v in, q out, 40 bytes per group), and
// the launch plus one round trip to memory (positions, then tables) for a
// step of single tokens.
#include "tokens.cuh"
#include "pipeline.cuh"

namespace eakv {
namespace {

constexpr int kThreads = 256;
constexpr int kRowSets = 4;   // sets of 128 elements per warp

struct RotaryArgs {
  PageGeom geom;
  int n_caches, layer, n_q, n_kv, total;
  int head_dim;
  Rows q, k, v, qo;
  const float *cos_t, *sin_t;
  int n_rows, pairs, interleaved, n_axes;
  const int32_t *positions;
  long long axis_stride;
  int bound[EAKV_MAX_AXES];   // first pair behind axis a
  int *status;
};

// One element's nibble: the rule of quantize.cu (NaN and what lies outside
// the int32 range become 0).
__device__ __forceinline__ int nibble(float x, float mn, float inv) {
  const float t = __fadd_rn(__fmul_rn(__fsub_rn(x, mn), inv), 0.5f);
  const int q = (t < 2147483648.0f) ? __float2int_rz(t) : 0;
  return q < 0 ? 0 : (q > 15 ? 15 : q);
}

// Quantizes the group that 16 neighbouring lanes hold (lane j of them:
// elements 4j..4j+3) into slot `slot` of page pp. Every lane of the warp
// calls this; `live` lanes write. Returns the scale.
__device__ __forceinline__ float quantize16(const float (&x)[4], uint8_t *pp, uint32_t nib_bytes,
                                            int slot, bool live, int lane) {
  const int j = lane & 15;
  float mn = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
  float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const float x0 = __shfl_sync(0xffffffffu, x[0], lane & 16);
  // a zero minimum or maximum has the sign of the group's first zero
  const bool zero = (x0 == x0) && (mn == 0.0f || mx == 0.0f);
  if (__any_sync(0xffffffffu, zero)) {
    int fz = 64;
    float zv = 0.0f;
#pragma unroll
    for (int e = 3; e >= 0; e--)
      if (x[e] == 0.0f) {
        fz = 4 * j + e;
        zv = x[e];
      }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      const int ofz = __shfl_xor_sync(0xffffffffu, fz, o);
      const float ozv = __shfl_xor_sync(0xffffffffu, zv, o);
      if (ofz < fz) {
        fz = ofz;
        zv = ozv;
      }
    }
    if (zero) {
      if (mn == 0.0f) mn = zv;
      if (mx == 0.0f) mx = zv;
    }
  }
  if (x0 != x0) {   // a NaN in element 0 stays
    mn = x0;
    mx = x0;
  }
  const float range = __fsub_rn(mx, mn);
  float scale = 1.0f, inv = 0.0f;
  if (range > 0.0f) {
    scale = __fdiv_rn(range, 15.0f);
    inv = __fdiv_rn(15.0f, range);
  }
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; e++) w |= (uint32_t)nibble(x[e], mn, inv) << (8 * e);
  // lanes 0..7 of the group hold the low nibbles, 8..15 the high ones
  const uint32_t hi = __shfl_down_sync(0xffffffffu, w, 8);
  if (live) {
    if (j < 8) *reinterpret_cast<uint32_t *>(pp + (size_t)slot * 32 + 4 * j) = w | (hi << 4);
    if (j == 0)
      *reinterpret_cast<float2 *>(pp + nib_bytes + (size_t)slot * 8) = make_float2(scale, mn);
  }
  return scale;
}

template <int HD, typename T, bool kVec>
__global__ void __launch_bounds__(kThreads)
append_rotary_kernel(const __grid_constant__ RotaryArgs a, const __grid_constant__ TokenBatch batch) {
  constexpr int HPW = 128 / HD;          // heads per set of 128 elements
  constexpr int LPR = HD / 4;            // lanes per row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x;
  const int sub = lane / LPR;            // head within the set
  const int d0 = 4 * (lane % LPR);       // first dim of this lane
  // head slots of a token: k heads, v heads, q heads, each padded to whole sets
  const int kv_sets = (a.n_kv + HPW - 1) / HPW, q_sets = (a.n_q + HPW - 1) / HPW;
  const int sets = 2 * kv_sets + q_sets;
  const int s0 = (blockIdx.y * (kThreads / 32) + warp) * kRowSets;
  if (s0 >= sets) return;

  // rows of this warp, their loads first
  float x[kRowSets][4];
  int head[kRowSets], part[kRowSets];    // part 0 k, 1 v, 2 q; head < 0: none
#pragma unroll
  for (int r = 0; r < kRowSets; r++) {
    const int s = s0 + r;
    part[r] = s < kv_sets ? 0 : (s < 2 * kv_sets ? 1 : 2);
    const int first = part[r] == 0 ? 0 : (part[r] == 1 ? kv_sets : 2 * kv_sets);
    const int h = (s - first) * HPW + sub;
    head[r] = (s < sets && h < (part[r] == 2 ? a.n_q : a.n_kv)) ? h : -1;
    const Rows &src = part[r] == 0 ? a.k : (part[r] == 1 ? a.v : a.q);
#pragma unroll
    for (int e = 0; e < 4; e++) x[r][e] = 0.0f;
    if (head[r] >= 0)
      load4<T, kVec>(reinterpret_cast<const T *>(src.data) + (long long)t * src.token_stride +
                         (long long)head[r] * src.head_stride + d0, x[r]);
  }

  // this lane's angles: pair of element d0 + e
  float c[4], sn[4];
  const bool turned = a.pairs > 0 && d0 < 2 * a.pairs;
  bool ok = true;
  if (a.pairs > 0) {
    int pos[EAKV_MAX_AXES];
#pragma unroll
    for (int ax = 0; ax < EAKV_MAX_AXES; ax++) {
      pos[ax] = ax < a.n_axes ? __ldg(a.positions + ax * a.axis_stride + t) : 0;
      ok = ok && pos[ax] >= 0 && pos[ax] < a.n_rows;
    }
    if (ok && turned) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int d = d0 + e;
        const int pair = a.interleaved ? d >> 1 : (d < a.pairs ? d : d - a.pairs);
        int p = pos[0];
#pragma unroll
        for (int ax = 1; ax < EAKV_MAX_AXES; ax++)
          if (ax < a.n_axes && pair >= a.bound[ax - 1]) p = pos[ax];
        c[e] = __ldg(a.cos_t + (long long)p * a.pairs + pair);
        sn[e] = __ldg(a.sin_t + (long long)p * a.pairs + pair);
      }
    }
  }
  if (!ok) {   // uniform: every lane read the same positions
    if (lane == 0) atomicOr(a.status, kStatusBadIndex);
    return;
  }

  // where the token's K and V go
  int cache = 0, at = 0;
  if (s0 < 2 * kv_sets) {
    cache = token_cache(batch, a.n_caches, t);
    at = batch.pos[cache] + (t - batch.first[cache]);
  }
  // lane that holds the partners of this lane's elements (halves)
  const bool second = !a.interleaved && d0 >= a.pairs;
  const int partner = second ? lane - a.pairs / 4 : lane + a.pairs / 4;

#pragma unroll
  for (int r = 0; r < kRowSets; r++) {
    if (s0 + r >= sets) break;   // uniform
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = x[r][e];
    if (part[r] != 1 && a.pairs > 0) {
      float o[4];
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = x[r][e ^ 1];
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = __shfl_sync(0xffffffffu, x[r][e], partner & 31);
      }
      if (turned) {
        // first of a pair: a c - b s; second: b c + a s
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const bool sec = a.interleaved ? (e & 1) : second;
          const float s = sec ? sn[e] : -sn[e];
          if (part[r] == 0)
            y[e] = (float)__dadd_rn(__dmul_rn((double)x[r][e], (double)c[e]),
                                    __dmul_rn((double)o[e], (double)s));
          else
            y[e] = fmaf(x[r][e], c[e], __fmul_rn(o[e], s));
        }
      }
    }
    if (part[r] == 2) {
      if (head[r] >= 0)
        store4<T, kVec>(reinterpret_cast<T *>(a.qo.data) + (long long)t * a.qo.token_stride +
                            (long long)head[r] * a.qo.head_stride + d0, y);
    } else {
      const int h = head[r] >= 0 ? head[r] : 0;
      const int page = at / kPagePositions, pip = at - page * kPagePositions;
      uint8_t *pp = batch.base[cache] +
                    page_index(a.geom, a.layer, part[r], h, page) * a.geom.page_bytes;
      const int slot = pip * (HD / 64) + d0 / 64;
      const float scale = quantize16(y, pp, a.geom.nib_bytes, slot, head[r] >= 0, lane);
      if (part[r] == 1 && head[r] >= 0 && (lane & 15) == 0)
        vexp_raise(vexp_table(batch.base[cache], a.geom), a.layer * a.geom.n_heads + h, scale);
    }
  }
}

template <int HD, typename T>
cudaError_t launch(const RotaryArgs &a, const TokenBatch &b, bool vec, cudaStream_t s) {
  constexpr int HPW = 128 / HD;
  const int sets = 2 * ((a.n_kv + HPW - 1) / HPW) + (a.n_q + HPW - 1) / HPW;
  const int per_block = kThreads / 32 * kRowSets;
  const dim3 grid(a.total, (sets + per_block - 1) / per_block);
  if (vec) append_rotary_kernel<HD, T, true><<<grid, kThreads, 0, s>>>(a, b);
  else append_rotary_kernel<HD, T, false><<<grid, kThreads, 0, s>>>(a, b);
  return cudaGetLastError();
}

int refuse(const char *what) {
  set_error(EAKV_ERR_INVALID, "append_rotary: %s", what);
  return EAKV_ERR_INVALID;
}

}  // namespace

int check_rows(const eakv_rows_t *r, const char *name, const char *who) {
  if (!r || !r->data || r->dtype < EAKV_F32 || r->dtype > EAKV_BF16 || r->token_stride < 0 ||
      r->head_stride < 0 || (uintptr_t)r->data % dtype_size(r->dtype) != 0) {
    set_error(EAKV_ERR_INVALID, "%s: %s rows: NULL, an unknown element type, a negative stride or "
              "an address that is no multiple of the element size", who, name);
    return EAKV_ERR_INVALID;
  }
  return EAKV_OK;
}

int token_batch(const eakv_cache_t *const *caches, int n_caches, int n_q, const int *pos0,
                const int *n, const char *who, TokenBatch &b, int &total) {
  int rc = check_batch(caches, n_caches, n_q, who);
  if (rc) return rc;
  if (!n) {
    set_error(EAKV_ERR_INVALID, "%s: NULL counts", who);
    return EAKV_ERR_INVALID;
  }
  long long sum = 0;
  for (int i = 0; i < n_caches; i++) {
    const eakv_cache_t *c = caches[i];
    const int p = pos0 ? pos0[i] : c->seq_len;
    if (n[i] < 0 || p < 0 || (long long)p + n[i] > c->max_seq_len) {
      set_error(EAKV_ERR_INVALID, "%s: cache %d: positions %d .. %lld outside 0 .. %d", who, i, p,
                (long long)p + n[i], c->max_seq_len);
      return EAKV_ERR_INVALID;
    }
    b.base[i] = c->d_buf;
    b.pos[i] = p;
    b.first[i] = (int)sum;
    sum += n[i];
    if (sum > (1 << 30)) {
      set_error(EAKV_ERR_INVALID, "%s: more than 2^30 tokens", who);
      return EAKV_ERR_INVALID;
    }
  }
  for (int i = n_caches; i <= kMaxBatch; i++) b.first[i] = (int)sum;
  total = (int)sum;
  return EAKV_OK;
}

}  // namespace eakv

using namespace eakv;

extern "C" int eakv_append_rotary(eakv_cache_t *const *caches, int n_caches, int layer,
                                  const int *n_new, const eakv_rows_t *k, const eakv_rows_t *v,
                                  const eakv_rows_t *q, const eakv_rows_t *q_out, int n_q_heads,
                                  const eakv_rotary_t *rotary, void *stream) {
  clear_error();
  TokenBatch b;
  RotaryArgs a = {};
  const char *who = "append_rotary";
  if (!caches || n_caches <= 0 || !caches[0]) return refuse("need 1..256 caches");
  const int n_kv = caches[0]->n_kv_heads;
  int rc = token_batch(caches, n_caches, q ? n_q_heads : n_kv, nullptr, n_new, who, b, a.total);
  if (rc || a.total == 0) return rc;
  if ((rc = check_rows(k, "k", who)) || (rc = check_rows(v, "v", who))) return rc;
  if (layer < 0 || layer >= caches[0]->n_layers) return refuse("layer out of range");
  if (!q != !q_out) return refuse("q and q_out go together");
  if (q && ((rc = check_rows(q, "q", who)) || (rc = check_rows(q_out, "q_out", who)))) return rc;
  if (v->dtype != k->dtype || (q && (q->dtype != k->dtype || q_out->dtype != k->dtype)))
    return refuse("k, v, q and q_out differ in element type");
  // the same cache twice would write the same positions twice
  for (int i = 0; i < n_caches; i++)
    for (int j = 0; j < i; j++)
      if (caches[i] == caches[j]) return refuse("the same cache twice");
  const eakv_cache_t *c0 = caches[0];
  a.geom = c0->geom;
  a.n_caches = n_caches;
  a.layer = layer;
  a.head_dim = c0->head_dim;
  a.n_kv = n_kv;
  a.n_q = q ? n_q_heads : 0;
  a.k = rows_of(k);
  a.v = rows_of(v);
  a.q = rows_of(q);
  a.qo = rows_of(q_out);
  if (rotary) {
    if (!rotary->cos_table || !rotary->sin_table || !rotary->positions)
      return refuse("NULL rotary table or positions");
    if (rotary->rot_dim <= 0 || rotary->rot_dim % 8 != 0 || rotary->rot_dim > c0->head_dim)
      return refuse("rot_dim must be a multiple of 8 within head_dim");
    if (rotary->n_rows <= 0 || rotary->n_axes < 1 || rotary->n_axes > EAKV_MAX_AXES ||
        rotary->axis_stride < 0)
      return refuse("bad rotary table rows, axes or axis stride");
    int sum = 0;
    for (int i = 0; i < rotary->n_axes; i++) {
      if (rotary->sections[i] < 0 || rotary->sections[i] > rotary->rot_dim)
        return refuse("sections must add up to rot_dim / 2");
      sum += rotary->sections[i];
      a.bound[i] = sum;
    }
    if (sum != rotary->rot_dim / 2) return refuse("sections must add up to rot_dim / 2");
    a.cos_t = rotary->cos_table;
    a.sin_t = rotary->sin_table;
    a.n_rows = rotary->n_rows;
    a.pairs = rotary->rot_dim / 2;
    a.interleaved = rotary->interleaved ? 1 : 0;
    a.n_axes = rotary->n_axes;
    a.positions = rotary->positions;
    a.axis_stride = rotary->axis_stride;
  }
  DeviceGuard g(c0->device);
  a.status = device_status_ptr();
  if (!a.status) return refuse("device status word unavailable");
  const bool vec = rows_vec(k) && rows_vec(v) && rows_vec(q) && rows_vec(q_out);
  cudaStream_t s = stream ? (cudaStream_t)stream : c0->stream;
  cudaError_t e;
  if (c0->head_dim == 128)
    e = k->dtype == EAKV_F32   ? launch<128, float>(a, b, vec, s)
        : k->dtype == EAKV_F16 ? launch<128, __half>(a, b, vec, s)
                               : launch<128, __nv_bfloat16>(a, b, vec, s);
  else
    e = k->dtype == EAKV_F32   ? launch<64, float>(a, b, vec, s)
        : k->dtype == EAKV_F16 ? launch<64, __half>(a, b, vec, s)
                               : launch<64, __nv_bfloat16>(a, b, vec, s);
  return check_cuda(e, "append_rotary: launch");
}
