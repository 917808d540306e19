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
// Mapping. Four lanes hold a 64-element group: lane j elements 8j..8j+7 (the low
// nibbles of bytes 8j..8j+7) and 32+8j..32+8j+7 (their high nibbles), so packing is
// local, minimum and maximum are two shuffle steps, and a lane stores its eight
// bytes at once. A warp holds 512 elements (four heads of 128, eight of 64) and
// takes kPasses of them, of one token and one kind (q, k or v), with their loads
// issued first; the token's cosines and sines are read once for all. The partners
// of rotated halves are loaded again (they are in L1 by then). With four elements
// per lane, sixteen lanes to a group, the reductions and the packing were ten times
// the arithmetic: 16384 tokens of 32 + 16 heads 199-258 us.
//
// Bound: for long chunks HBM (q, k, v in, q out, 40 bytes per group: 55 us for 16384
// tokens of 32 + 16 heads of 128, bf16), from which it is far: 171 us with cold
// caches, of which K and V as they are take 45, the keys' rotation (f64, their
// partners loaded again) 32, the queries as they are 63 (0.65 of HBM's rate: positions,
// tables and rows are a warp's one round trip, two heads' sets at a time) and their
// rotation 31. 2048 tokens 31 us. For a step of single tokens the launch plus a round
// trip to memory (positions, then tables): 16 caches of one token 11 us.
#include "tokens.cuh"
#include "pipeline.cuh"

namespace eakv {
namespace {

constexpr int kThreads = 256;
constexpr int kPasses = 2;    // sets of 512 elements per warp, at most

struct RotaryArgs {
  PageGeom geom;
  int n_caches, layer, n_q, n_kv, total, tokens_y;
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

// Quantizes the group that four neighbouring lanes hold into slot `slot` of page
// pp. Every lane of the warp calls this; `live` lanes write. Returns the scale.
__device__ __forceinline__ float quantize4(const float (&x)[16], uint8_t *pp, uint32_t nib_bytes,
                                           int slot, bool live, int lane) {
  const int j = lane & 3;
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int e = 1; e < 16; e++) {
    mn = fminf(mn, x[e]);
    mx = fmaxf(mx, x[e]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  const float x0 = __shfl_sync(0xffffffffu, x[0], lane & ~3);
  // a zero minimum or maximum has the sign of the group's first zero
  const bool zero = (x0 == x0) && (mn == 0.0f || mx == 0.0f);
  if (__any_sync(0xffffffffu, zero)) {
    int fz = 64;
    float zv = 0.0f;
#pragma unroll
    for (int e = 15; e >= 0; e--) {
      const int k = e < 8 ? 8 * j + e : 24 + 8 * j + e;
      if (x[e] == 0.0f && k < fz) {
        fz = k;
        zv = x[e];
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
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
  uint32_t w[2] = {0u, 0u};
  // A finite inv keeps every t = (x - mn) inv + 1/2 of finite x within [1/2, 16):
  // added to 2^23 with truncation, its integer part is the sum's last bits.
  // (range / 15 < 2^125 as well: x - mn does not overflow; NaN in x has no place.)
  const bool tame = range < 3.0e38f && inv < 3.0e38f && x0 == x0;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 16; e++) nan = nan || x[e] != x[e];
  if (__all_sync(0xffffffffu, tame && !nan)) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float q0 = __fadd_rn(__fmul_rn(__fsub_rn(x[e], mn), inv), 0.5f);
      const float q1 = __fadd_rn(__fmul_rn(__fsub_rn(x[8 + e], mn), inv), 0.5f);
      const uint32_t lo = __float_as_uint(__fadd_rz(q0, 8388608.0f));
      const uint32_t hi = __float_as_uint(__fadd_rz(q1, 8388608.0f));
      // lo and hi are 0x4B00000q: byte e of the word is 16 q_hi + q_lo
      w[e >> 2] += ((hi << 4) + lo) << (8 * (e & 3));
    }
    // what the 0x4B000000s left in the upper byte: 17 * 0x4B000000, from e & 3 == 0
    w[0] -= 0xFB000000u;
    w[1] -= 0xFB000000u;
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++)
      w[e >> 2] |= (uint32_t)(nibble(x[8 + e], mn, inv) * 16 + nibble(x[e], mn, inv)) << (8 * (e & 3));
  }
  if (live) {
    *reinterpret_cast<uint2 *>(pp + (size_t)slot * 32 + 8 * j) = make_uint2(w[0], w[1]);
    if (j == 0)
      *reinterpret_cast<float2 *>(pp + nib_bytes + (size_t)slot * 8) = make_float2(scale, mn);
  }
  return scale;
}

// The warps of a token: K, V, then Q.
struct Sets {
  int kv_warps, warps;   // of K (or V), of all
};
template <int HD>
__host__ __device__ inline Sets sets_of(int n_kv, int n_q) {
  constexpr int HPW = 512 / HD * kPasses;   // heads of a warp
  Sets s;
  s.kv_warps = (n_kv + HPW - 1) / HPW;
  s.warps = 2 * s.kv_warps + (n_q + HPW - 1) / HPW;
  return s;
}

// Four chunks of four elements: dims d0 + 0, 4, 32, 36.
template <typename T> struct Raw16 { Vec4<T> v[4]; };

template <typename T, bool kVec>
__device__ __forceinline__ Vec4<T> fetch4(const T *p) {
  Vec4<T> r;
  if constexpr (kVec) {
    r = *reinterpret_cast<const Vec4<T> *>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) r.v[e] = p[e];
  }
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void put4(T *p, const Vec4<T> &v) {
  if constexpr (kVec) {
    *reinterpret_cast<Vec4<T> *>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) p[e] = v.v[e];
  }
}

template <int HD, typename T, bool kVec>
__global__ void __launch_bounds__(kThreads, 3)
append_rotary_kernel(const __grid_constant__ RotaryArgs a, const __grid_constant__ TokenBatch batch) {
  constexpr int LPR = HD / 16;           // lanes per head
  constexpr int HPP = 32 / LPR;          // heads per pass
  const int lane = threadIdx.x & 31;
  const Sets sets = sets_of<HD>(a.n_kv, a.n_q);
  // blockIdx.y: runs of tokens whose warps an int counts
  const int wid = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int tw = wid / sets.warps, t = blockIdx.y * a.tokens_y + tw;
  if (tw >= a.tokens_y || t >= a.total) return;
  int w = wid - tw * sets.warps;
  const int part = w < sets.kv_warps ? 0 : (w < 2 * sets.kv_warps ? 1 : 2);   // k, v, q
  w -= part * sets.kv_warps;
  const Rows &src = part == 0 ? a.k : (part == 1 ? a.v : a.q);
  const int heads = part == 2 ? a.n_q : a.n_kv;
  const int h0 = w * HPP * kPasses + lane / LPR;          // head of this lane in pass 0
  const int grp = (lane % LPR) >> 2, d0 = 64 * grp + 8 * (lane & 3);   // its first dim

  const T *in = reinterpret_cast<const T *>(src.data) + (long long)t * src.token_stride;
  // Lanes without a head repeat the last. Rows of this warp, their loads first:
  // keys and values, and queries whose pairs do not come in eights, as quantize4
  // wants them; queries as eight pairs.
  const bool eights = part == 2 && a.pairs % 8 == 0;
  const int unit = lane % LPR, n_turned = a.pairs / 8;
  const int da = !eights ? d0 : (a.interleaved || unit >= n_turned ? 16 * unit : 8 * unit);
  const int db = !eights ? d0 + 32 : (a.interleaved || unit >= n_turned ? 16 * unit + 8 : 8 * unit + a.pairs);
  Raw16<T> raw[kPasses];
#pragma unroll
  for (int r = 0; r < kPasses; r++) {
    const T *p = in + (long long)min(h0 + r * HPP, heads - 1) * src.head_stride;
#pragma unroll
    for (int k = 0; k < 4; k++) raw[r].v[k] = fetch4<T, kVec>(p + (k < 2 ? da : db) + 4 * (k & 1));
  }

  int pos[EAKV_MAX_AXES];
  if (a.pairs > 0) {
    bool ok = true;
#pragma unroll
    for (int ax = 0; ax < EAKV_MAX_AXES; ax++) {
      pos[ax] = ax < a.n_axes ? __ldg(a.positions + ax * a.axis_stride + t) : 0;
      ok = ok && pos[ax] >= 0 && pos[ax] < a.n_rows;
    }
    if (!ok) {   // uniform: every lane read the same positions
      if (lane == 0) atomicOr(a.status, kStatusBadIndex);
      return;
    }
  }
  T *out = reinterpret_cast<T *>(a.qo.data) + (long long)t * a.qo.token_stride;
  if (eights) {
    // pairs 8 unit .. 8 unit + 7 of this lane; the angles serve every head
    float c[8], sn[8];
    const bool turned = unit < n_turned;
    if (turned) {
      if (a.n_axes == 1) {   // tables are 16-byte aligned
        const long long at = (long long)pos[0] * a.pairs + 8 * unit;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 c4 = __ldg(reinterpret_cast<const float4 *>(a.cos_t + at + e));
          const float4 s4 = __ldg(reinterpret_cast<const float4 *>(a.sin_t + at + e));
          c[e] = c4.x; c[e + 1] = c4.y; c[e + 2] = c4.z; c[e + 3] = c4.w;
          sn[e] = s4.x; sn[e + 1] = s4.y; sn[e + 2] = s4.z; sn[e + 3] = s4.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int pair = 8 * unit + e;
          int p = pos[0];
#pragma unroll
          for (int ax = 1; ax < EAKV_MAX_AXES; ax++)
            if (ax < a.n_axes && pair >= a.bound[ax - 1]) p = pos[ax];
          c[e] = __ldg(a.cos_t + (long long)p * a.pairs + pair);
          sn[e] = __ldg(a.sin_t + (long long)p * a.pairs + pair);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kPasses; r++) {
      const int h = h0 + r * HPP;
      if (turned) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
          // halves: element i of the two eights; interleaved: neighbours of the sixteen
          T &ra = a.interleaved ? raw[r].v[i >> 1].v[(2 * i) & 3] : raw[r].v[i >> 2].v[i & 3];
          T &rb = a.interleaved ? raw[r].v[i >> 1].v[(2 * i + 1) & 3] : raw[r].v[2 + (i >> 2)].v[i & 3];
          const float x = to_f32<T>(ra), y = to_f32<T>(rb);
          ra = from_f32<T>(fmaf(x, c[i], -__fmul_rn(y, sn[i])));
          rb = from_f32<T>(fmaf(y, c[i], __fmul_rn(x, sn[i])));
        }
      }
      if (h >= heads) continue;
      T *p = out + (long long)h * a.qo.head_stride;
#pragma unroll
      for (int k = 0; k < 4; k++) put4<T, kVec>(p + (k < 2 ? da : db) + 4 * (k & 1), raw[r].v[k]);
    }
    return;
  }
  // dims of chunk k: 0 not turned, 1 first of pairs, 2 second
  auto dim = [&](int k) { return d0 + 4 * (k & 1) + 32 * (k >> 1); };
  auto kind = [&](int k) {
    return dim(k) >= 2 * a.pairs ? 0 : (a.interleaved || dim(k) < a.pairs ? 1 : 2);
  };
  // angles of chunk k, signed: first of a pair a c - b s, second b c + a s (in L1
  // after the first pass; kept in registers they would cost a third of the warps)
  auto angles = [&](int k, float (&c)[4], float (&sn)[4]) {
    const int d = dim(k), second = kind(k) == 2;
    if (a.n_axes == 1 && !a.interleaved) {   // four neighbouring pairs (tables are 16-byte aligned)
      const long long at = (long long)pos[0] * a.pairs + (second ? d - a.pairs : d);
      const float4 c4 = __ldg(reinterpret_cast<const float4 *>(a.cos_t + at));
      const float4 s4 = __ldg(reinterpret_cast<const float4 *>(a.sin_t + at));
      c[0] = c4.x; c[1] = c4.y; c[2] = c4.z; c[3] = c4.w;
      sn[0] = s4.x; sn[1] = s4.y; sn[2] = s4.z; sn[3] = s4.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int pair = a.interleaved ? (d + e) >> 1 : (second ? d + e - a.pairs : d + e);
        int p = pos[0];
#pragma unroll
        for (int ax = 1; ax < EAKV_MAX_AXES; ax++)
          if (ax < a.n_axes && pair >= a.bound[ax - 1]) p = pos[ax];
        c[e] = __ldg(a.cos_t + (long long)p * a.pairs + pair);
        sn[e] = __ldg(a.sin_t + (long long)p * a.pairs + pair);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (a.interleaved ? !(e & 1) : !second) sn[e] = -sn[e];
  };
  // chunk k of pass r, and its elements' partners
  auto chunk = [&](int r, int k, float (&x)[4], float (&o)[4]) {
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = to_f32<T>(raw[r].v[k].v[e]);
    if (a.interleaved) {
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = x[e ^ 1];
    } else {
      const int h = min(h0 + r * HPP, heads - 1);
      const int d = dim(k) + (kind(k) == 2 ? -a.pairs : a.pairs);
      const Vec4<T> v = fetch4<T, kVec>(in + (long long)h * src.head_stride + d);
#pragma unroll
      for (int e = 0; e < 4; e++) o[e] = to_f32<T>(v.v[e]);
    }
  };

  if (part == 2) {
    // every pass is turned before the first is stored: q_out may be q
    Raw16<T> res[kPasses];
#pragma unroll
    for (int r = 0; r < kPasses; r++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        res[r].v[k] = raw[r].v[k];
        if (a.pairs > 0 && kind(k)) {
          float x[4], o[4], c[4], sn[4];
          chunk(r, k, x, o);
          angles(k, c, sn);
#pragma unroll
          for (int e = 0; e < 4; e++)
            res[r].v[k].v[e] = from_f32<T>(fmaf(x[e], c[e], __fmul_rn(o[e], sn[e])));
        }
      }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < kPasses; r++) {
      const int h = h0 + r * HPP;
      if (h >= heads) continue;
      T *p = out + (long long)h * a.qo.head_stride + d0;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        put4<T, kVec>(p + 4 * (k & 1) + 32 * (k >> 1), res[r].v[k]);
      }
    }
    return;
  }
  // where the token's K and V go
  const int cache = token_cache(batch, a.n_caches, t);
  const int at = batch.pos[cache] + (t - batch.first[cache]);
  const int page = at / kPagePositions, slot = (at - page * kPagePositions) * (HD / 64) + grp;
  uint8_t *base = batch.base[cache];
#pragma unroll
  for (int r = 0; r < kPasses; r++) {
    if ((w * kPasses + r) * HPP >= heads) break;   // uniform: a pass without heads
    float x[16];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float y[4], o[4];
      if (part == 0 && a.pairs > 0 && kind(k)) {
        float c[4], sn[4];
        chunk(r, k, y, o);
        angles(k, c, sn);
#pragma unroll
        for (int e = 0; e < 4; e++)
          y[e] = (float)__dadd_rn(__dmul_rn((double)y[e], (double)c[e]),
                                  __dmul_rn((double)o[e], (double)sn[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = to_f32<T>(raw[r].v[k].v[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) x[4 * k + e] = y[e];
    }
    const bool live = h0 + r * HPP < heads;
    const int h = live ? h0 + r * HPP : 0;
    uint8_t *pp = base + page_index(a.geom, a.layer, part, h, page) * a.geom.page_bytes;
    const float scale = quantize4(x, pp, a.geom.nib_bytes, slot, live, lane);
    if (part == 1 && live && (lane & 3) == 0)
      vexp_raise(vexp_table(base, a.geom), a.layer * a.geom.n_heads + h, scale);
  }
}

template <int HD, typename T>
cudaError_t launch(const RotaryArgs &a, const TokenBatch &b, bool vec, cudaStream_t s) {
  RotaryArgs r = a;
  const int per_token = sets_of<HD>(a.n_kv, a.n_q).warps, most = (1 << 30) / per_token;
  r.tokens_y = a.total < most ? a.total : most;
  const dim3 grid((unsigned)(((long long)r.tokens_y * per_token + kThreads / 32 - 1) / (kThreads / 32)),
                  (unsigned)((a.total + r.tokens_y - 1) / r.tokens_y));
  if (vec) append_rotary_kernel<HD, T, true><<<grid, kThreads, 0, s>>>(r, b);
  else append_rotary_kernel<HD, T, false><<<grid, kThreads, 0, s>>>(r, b);
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

int check_out_rows(const eakv_rows_t *r, const char *name, const char *who, int tokens, int heads,
                   int head_dim) {
  int rc = check_rows(r, name, who);
  if (rc) return rc;
  if ((tokens > 1 && r->token_stride < head_dim) || (heads > 1 && r->head_stride < head_dim)) {
    set_error(EAKV_ERR_INVALID, "%s: %s rows overlap (token stride %lld, head stride %lld)", who, name,
              (long long)r->token_stride, (long long)r->head_stride);
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
  if (q && ((rc = check_rows(q, "q", who)) ||
            (rc = check_out_rows(q_out, "q_out", who, a.total, n_q_heads, caches[0]->head_dim))))
    return rc;
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
  a.n_kv = n_kv;
  a.n_q = q ? n_q_heads : 0;
  a.k = rows_of(k);
  a.v = rows_of(v);
  a.q = rows_of(q);
  a.qo = rows_of(q_out);
  if (rotary) {
    if (!rotary->cos_table || !rotary->sin_table || !rotary->positions ||
        ((uintptr_t)rotary->cos_table | (uintptr_t)rotary->sin_table) % 16 ||
        (uintptr_t)rotary->positions % 4)
      return refuse("a rotary table or positions NULL, a table not 16-byte aligned or positions not 4-byte");
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
