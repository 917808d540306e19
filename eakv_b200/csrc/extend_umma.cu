// extend_umma.cu - attention of many new tokens per cache (prompt chunks) over
// the Q4 pages on the fifth-generation tensor cores: tcgen05.mma kind::f16,
// f32 accumulators in tensor memory.
//
// Mathematics. A CTA holds up to 256 (token, query head) rows of one KV head as
// two tiles of 128 (tensor-memory lane = row) and walks its positions in tiles
// of 128 (two pages):
//   S[row][pos]  = Q'[row][dim] K'[pos][dim]^T        (SS, both K-major)
//   O[row][dim] += P'[row][pos] V'[pos][dim]          (P' in tensor memory, V' MN-major)
// with an online softmax in base 2 between them, whose maximum moves lazily
// (when a score passes it by more than 8).
//
// Operands are f16. Q' is q times a power of two per row (exact for bf16 and
// f16 but for elements 2^-18 below the row's largest). K' and V' are the
// dequantized values s (n - 8) + (b + 8 s): n - 8 is exact, s and b + 8 s are rounded
// to f16 and the result once more (3 roundings of 2^-12 relative to the
// value's own size, against the 2^-9 of a bf16 output; keeping the nibbles
// exact instead needs a second accumulator per 64-dim group, for which tensor
// memory has no room, and four more FMAs per score). P' = 2^7 p is at most
// 2^15, one f16.
//
// Ranges. K and V are divided by powers of two taken from the first tile
// (eref): then 128 values of a row lie in f16's range for rows within 2^-10 and
// 2^12 of it. A run of 32 positions with a row outside of that is marked: its rows
// are divided by powers of their own, which go to the softmax threads beside
// it, and these scale the scores and the weights column by column, with
// a V reference of their own per row, taken from attended positions only. So a
// position that a row does not attend has no influence on it, however large.
// Non-finite V groups are kept out of the products (0 NaN is NaN) and
// listed by position; a row that attends one gets NaN in the group's dims.
//
// Roles (13 warps). Warps 0-3 and 4-7: softmax of row tile 0 and 1, one thread
// per row; they read S twice (maximum, then weights), write P' over S, and
// scale O when a maximum moves. Warps 8-11: dequantize, one thread per position
// row: the raw row comes from global memory a tile ahead in registers
// and leaves as sixteen 16-byte stores in the 128-byte swizzle. A
// 32-bit word of nibbles becomes one 16-byte chunk [d, d+2, d+1, d+3, d+32, d+34, d+33,
// d+35] (the pairs that one mask selects); Q' is stored in the same order and
// the output's columns are read back in it, so the order costs nothing. Warp
// 12: one thread issues the MMAs: for tile i, PV of row tile 0, S(i+1) of row tile 0,
// the same for row tile 1, so one row tile's softmax runs under the other's
// MMAs. P' of a tile lies over its S; the tensor pipe runs the MMAs in order.
//
// All hand-overs are mbarriers with bounded, suspending waits; one that runs
// out sets the status word, and every role leaves at its next wait.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "extend.cuh"
#include "umma.cuh"

namespace eakv {
namespace {

using namespace umma;

constexpr int BN = 128;                       // positions per tile
constexpr int kSoftWarps = 8, kConvWarps = 4;
constexpr int kThreads = (kSoftWarps + kConvWarps + 1) * 32;
constexpr int kUnset = -100000;
constexpr int kUp = 12, kDown = 10;           // rows within 2^kUp, 2^-kDown of eref need no mark
constexpr float kPShift = 7.0f;               // P' = 2^7 p
constexpr uint32_t kLayoutSW128 = 2;

template <int HD>
struct WCfg {
  static constexpr int NG = HD / 64;
  static constexpr int PB = kPagePositions * NG * 40;
  static constexpr int NIB = kPagePositions * NG * 32;
  static constexpr int TILE = 128 * HD * 2;   // bytes of a 128 x HD f16 operand
  static constexpr int HALF = 128 * 128;      // bytes of its 64-dim half
  static constexpr int Q = 0;                 // two row tiles
  static constexpr int K = Q + 2 * TILE;      // two stages
  static constexpr int V = K + 2 * TILE;      // two stages
  static constexpr int EXPS = V + 2 * TILE;   // short2 [4][BN]: exponents of marked rows
  static constexpr int INFO = EXPS + 4 * BN * 4;   // int4 [4 tiles][4 warps]
  static constexpr int BARS = INFO + 4 * 4 * 16;
  // barriers: kfull[2] vfull[2] kfree[2] vfree[2] sfull[2] pfull[2] odone[2] drain
  static constexpr int N_BARS = 15;
  static constexpr int REF = BARS + 8 * N_BARS + 8;    // int2: eref of K, V
  static constexpr int SLOT = REF + 8;
  static constexpr int RED = SLOT + 8;                 // int2 [4]
  static constexpr int END = RED + 32;
  static constexpr int SMEM = END + 1024;              // alignment slack
  // tensor memory columns
  static constexpr int S_COL = 0, O_COL = 256, COLS = 512;
  static_assert(REF % 8 == 0 && SLOT % 8 == 0 && RED % 8 == 0, "alignment");
};

enum { kKFull = 0, kVFull = 2, kKFree = 4, kVFree = 6, kSFull = 8, kPFull = 10, kODone = 12, kDrain = 14 };

// D[128 x N] (+)= A B, f16 operands, f32 accumulate: A in shared memory
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc,
                                           uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
// A in tensor memory
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t bd, uint32_t idesc,
                                           uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
// f16 x f16 -> f32, M = 128; B MN-major when b_mn
__host__ __device__ constexpr uint32_t idesc_f16(int N, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ uint32_t pack_f16(float x0, float x1) {
  return as_u32(__floats2half2_rn(x0, x1));
}
__device__ __forceinline__ uint4 ldg_row(const void *p) {
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ float pow2i(int e) {   // 2^e, 0 below the normal range
  return __uint_as_float((uint32_t)min(max(127 + e, 0), 254) << 23);
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// One nibble row (HD/2 bytes) with its (scale, bias) pairs.
template <int HD> struct RawRow {
  uint4 w[HD / 32];
  float sb[2 * (HD / 64)];
};

template <int HD>
__device__ __forceinline__ void load_row(RawRow<HD> &r, const uint8_t *page, int pip) {
  using C = WCfg<HD>;
#pragma unroll
  for (int k = 0; k < HD / 32; k++) r.w[k] = ldg_row(page + (size_t)pip * (HD / 2) + 16 * k);
  if constexpr (HD == 128) {
    const uint4 s = ldg_row(page + C::NIB + pip * 16);
    r.sb[0] = __uint_as_float(s.x); r.sb[1] = __uint_as_float(s.y);
    r.sb[2] = __uint_as_float(s.z); r.sb[3] = __uint_as_float(s.w);
  } else {
    const float2 s = __ldg(reinterpret_cast<const float2 *>(page + C::NIB + pip * 8));
    r.sb[0] = s.x; r.sb[1] = s.y;
  }
}

// Exponent e with every |value| of the row's finite groups below 2^(e+1);
// kUnset when they are all zero or none is finite. Bit g of `bad`: group g is
// not finite.
template <int HD>
__device__ __forceinline__ int row_exp(const RawRow<HD> &r, uint32_t &bad) {
  float m = 0.0f;
  bad = 0;
#pragma unroll
  for (int g = 0; g < HD / 64; g++) {
    // |n - 8| <= 8: 8 |s| + |b + 8 s|
    const float x = fmaf(8.0f, fabsf(r.sb[2 * g]), fabsf(fmaf(8.0f, r.sb[2 * g], r.sb[2 * g + 1])));
    if (x <= 3.0e38f) m = fmaxf(m, x);
    else bad |= 1u << g;
  }
  return m > 0.0f ? (int)(__float_as_uint(m) >> 23) - 127 : kUnset;
}

// The row's values divided by 2^e as f16 into row `row` of an operand: 16-byte
// chunk j of half g holds word j of group g. A group in `zero` is stored as 0.
template <int HD>
__device__ __forceinline__ void store_row(const RawRow<HD> &r, uint8_t *op, int row, int e,
                                          uint32_t zero) {
  using C = WCfg<HD>;
  // 2^-e in two factors: e spans more than the exponents of one float
  const float f0 = pow2i(-(e >> 1)), f1 = pow2i(-(e - (e >> 1)));
#pragma unroll
  for (int g = 0; g < HD / 64; g++) {
    const float s = r.sb[2 * g] * f0 * f1, b = fmaf(8.0f, r.sb[2 * g], r.sb[2 * g + 1]) * f0 * f1;
    __half2 sl = __float2half2_rn(s), sh = __float2half2_rn(s * 0.0625f), bb = __float2half2_rn(b);
    const bool z = (zero >> g) & 1;
    if (z) sl = sh = bb = __float2half2_rn(0.0f);
    const uint32_t words[8] = {r.w[2 * g].x, r.w[2 * g].y, r.w[2 * g].z, r.w[2 * g].w,
                               r.w[2 * g + 1].x, r.w[2 * g + 1].y, r.w[2 * g + 1].z, r.w[2 * g + 1].w};
    uint8_t *base = op + g * C::HALF + row * 128;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t w = words[j], y = w >> 8;
      const __half2 lo0 = __hsub2(as_half2(and_or(w, 0x000F000Fu, 0x64006400u)), as_half2(0x64086408u));
      const __half2 lo1 = __hsub2(as_half2(and_or(y, 0x000F000Fu, 0x64006400u)), as_half2(0x64086408u));
      const __half2 hi0 = __hsub2(as_half2(and_or(w, 0x00F000F0u, 0x64006400u)), as_half2(0x64806480u));
      const __half2 hi1 = __hsub2(as_half2(and_or(y, 0x00F000F0u, 0x64006400u)), as_half2(0x64806480u));
      const uint4 v = make_uint4(as_u32(__hfma2(lo0, sl, bb)), as_u32(__hfma2(lo1, sl, bb)),
                                 as_u32(__hfma2(hi0, sh, bb)), as_u32(__hfma2(hi1, sh, bb)));
      *reinterpret_cast<uint4 *>(base + ((j ^ (row & 7)) << 4)) = v;
    }
  }
}

// Bits of the positions c0 .. c0 + 31 that the row attends, clipped to `end`.
__device__ __forceinline__ uint32_t mask32(const RowMask &m, int c0, int end) {
  const int lo = max(m.lo - c0, 0), hi = min(min(m.hi, end) - c0, 32);
  if (hi <= lo) return 0u;
  uint32_t b = (hi >= 32 ? 0xffffffffu : (1u << hi) - 1u) & ~(lo >= 32 ? 0xffffffffu : (1u << lo) - 1u);
  const int t = m.old - c0;   // columns from t on are new tokens 0, 1, ...
  if (t < 32 && m.old < m.hi) {
    const uint32_t tree = t >= 0 ? (uint32_t)(m.bits << t) : (-t < 64 ? (uint32_t)(m.bits >> -t) : 0u);
    const uint32_t before = t <= 0 ? 0u : (1u << t) - 1u;
    b &= before | tree;
  }
  return b;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1)
extend_umma_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExtendBatch batch,
                   const int vec) {
  using C = WCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t bars = smem_u32(smem + C::BARS);
  auto bar = [&](int i) { return bars + 8 * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ExtItem it = extend_item(a, batch);
  if (!extend_item_ok(a, it)) {
    if (a.n_splits > 1) extend_arrive_last(a, it.item);
    return;
  }
  const uint32_t budget = min(a.wait_budget, 1u << 18);
  const int base_pos = it.pg0 * kPagePositions;
  const int end_pos = (it.pg0 + it.npages) * kPagePositions;   // of this split
  // positions and tiles of each row tile
  const int n_mt = it.rows > 128 ? 2 : 1;
  int nt[2];
#pragma unroll
  for (int m = 0; m < 2; m++) {
    const int last = min(it.row0 + 128 * m + 127, it.row0 + it.rows - 1);
    const int hi = min(a.tree ? it.hi : it.old + last / a.G + 1, end_pos);
    nt[m] = (m < n_mt && hi > base_pos) ? (hi - base_pos + BN - 1) / BN : 0;
  }
  const int n_tiles = max(nt[0], nt[1]);

  if (warp == 12) {
    tmem_alloc(smem_u32(smem + C::SLOT), C::COLS);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(bar(kKFull + i), kConvWarps);
      mbar_init(bar(kVFull + i), kConvWarps);
      mbar_init(bar(kKFree + i), 1);
      mbar_init(bar(kVFree + i), 1);
      mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kPFull + i), 4);
      mbar_init(bar(kODone + i), 1);
    }
    mbar_init(bar(kDrain), 1);
    fence_mbar_init();
  }

  // ---- Q' (softmax threads: one row each) --------------------------------------
  float c_row = 0.0f;      // score factor: |scale| log2 e / 2^(q exponent)
  RowMask mask = {};
  const int mt = warp >> 2;                       // row tile of a softmax warp
  const int r_loc = 128 * mt + (threadIdx.x & 127);   // row within the item
  if (warp < kSoftWarps) {
    mask = row_mask(a, it, it.row0 + min(r_loc, it.rows - 1));
    const int row = it.row0 + min(r_loc, it.rows - 1);
    const T *qp = reinterpret_cast<const T *>(a.q.data) +
                  (long long)(it.tok0 + row / a.G) * a.q.token_stride +
                  (long long)(it.h * a.G + row % a.G) * a.q.head_stride;
    float mx = 0.0f;
    bool bad = false;
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
      float v[4];
      if (vec) load4<T, true>(qp + d, v);
      else load4<T, false>(qp + d, v);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        mx = fmaxf(mx, fabsf(v[e]));
        bad = bad || v[e] != v[e];
      }
    }
    const bool fine = !bad && mx <= 3.0e38f;
    int qe = 0;
    frexpf(mx > 0.0f && fine ? mx : 1.0f, &qe);   // mx in [2^(qe-1), 2^qe)
    qe = max(min(5 - qe, 126), -126);
    const float up = fine ? (a.scale_log2 < 0.0f ? -1.0f : 1.0f) * pow2i(qe) : 0.0f;
    c_row = fine ? fabsf(a.scale_log2) * pow2i(-qe) : __uint_as_float(0x7fc00000u);
    uint8_t *op = smem + C::Q + mt * C::TILE;
    const int rr = threadIdx.x & 127;
#pragma unroll 2
    for (int j = 0; j < HD / 8; j++) {
      const int g = j >> 3, d = 64 * g + 4 * (j & 7);
      float lo[4], hi[4];
      if (vec) {
        load4<T, true>(qp + d, lo);
        load4<T, true>(qp + d + 32, hi);
      } else {
        load4<T, false>(qp + d, lo);
        load4<T, false>(qp + d + 32, hi);
      }
      if (!fine) {
#pragma unroll
        for (int e = 0; e < 4; e++) lo[e] = hi[e] = 0.0f;
      }
      *reinterpret_cast<uint4 *>(op + g * C::HALF + rr * 128 + (((j & 7) ^ (rr & 7)) << 4)) =
          make_uint4(pack_f16(lo[0] * up, lo[2] * up), pack_f16(lo[1] * up, lo[3] * up),
                     pack_f16(hi[0] * up, hi[2] * up), pack_f16(hi[1] * up, hi[3] * up));
    }
    fence_proxy_async_smem();
  }

  // ---- dequantizing threads: the first tile, and the references -----------------
  const int crow = threadIdx.x & 127;             // position row of a converter thread
  const uint8_t *kpages = batch.base[it.b] + page_index(a.geom, a.layer, 0, it.h, 0) * C::PB;
  const uint8_t *vpages = kpages + (size_t)a.geom.n_heads * a.geom.n_pages * C::PB;
  RawRow<HD> kr, vr;
  // row of tile i held by this thread: live when some row of the item may attend it
  auto live = [&](int i) {
    const int p = base_pos + i * BN + crow;
    return i < n_tiles && p >= it.lo && p < it.hi && p < end_pos;
  };
  auto fetch = [&](RawRow<HD> &r, const uint8_t *pages, int i) {
    if (live(i)) {
      const int p = base_pos + i * BN + crow;
      load_row<HD>(r, pages + (size_t)(p / kPagePositions) * C::PB, p % kPagePositions);
    } else {
#pragma unroll
      for (int k = 0; k < HD / 32; k++) r.w[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < 2 * C::NG; k++) r.sb[k] = 0.0f;
    }
  };
  if (warp >= kSoftWarps && warp < kSoftWarps + kConvWarps) {
    fetch(kr, kpages, 0);
    fetch(vr, vpages, 0);
    uint32_t bad;
    const int ek = __reduce_max_sync(0xffffffffu, row_exp<HD>(kr, bad));
    const int ev = __reduce_max_sync(0xffffffffu, row_exp<HD>(vr, bad));
    if (lane == 0) reinterpret_cast<int2 *>(smem + C::RED)[warp - kSoftWarps] = make_int2(ek, ev);
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  int kref = kUnset, vref = kUnset;
#pragma unroll
  for (int w = 0; w < kConvWarps; w++) {
    const int2 e = reinterpret_cast<const int2 *>(smem + C::RED)[w];
    kref = max(kref, e.x);
    vref = max(vref, e.y);
  }
  if (kref == kUnset) kref = 0;
  if (vref == kUnset) vref = 0;
  const uint32_t tm = *reinterpret_cast<const uint32_t *>(smem + C::SLOT);

  bool ok = true;
  auto wait = [&](int b, int use) {   // `use`: how often this barrier was waited for before
    if (!ok) return false;
    if (mbar_wait_sleep(bar(b), use & 1, budget)) return true;
    atomicOr(a.status, kStatusWaitTimeout);
    ok = false;
    return false;
  };

  // the same for a whole warp: its lanes go on, or leave, together
  auto wait_warp = [&](int b, int use) {
    wait(b, use);
    ok = __all_sync(0xffffffffu, ok);
    return ok;
  };

  float m_run = -INFINITY, l_run = 0.0f;
  int eref = kUnset;
  bool poison[2] = {false, false};

  if (warp >= kSoftWarps && warp < kSoftWarps + kConvWarps) {
    // ================= dequantize ================================================
    const int cw = warp - kSoftWarps;
    for (int i = 0; i < n_tiles; i++) {
      const int st = i & 1;
      if (i >= 2 && !wait_warp(kKFree + st, (i >> 1) - 1)) break;
      uint32_t kbad, vbad;
      const int ke = row_exp<HD>(kr, kbad), ve = row_exp<HD>(vr, vbad);
      // a non-finite K group keeps its NaN: it reaches its own score only
      const bool kout = ke != kUnset && (ke > kref + kUp || ke < kref - kDown);
      const bool vout = ve != kUnset && (ve > vref + kUp || ve < vref - kDown);
      const bool mark = __any_sync(0xffffffffu, kout || vout);
      const int kx = mark && ke != kUnset ? ke : kref, vx = mark && ve != kUnset ? ve : vref;
      const uint32_t n0 = __ballot_sync(0xffffffffu, vbad & 1), n1 = __ballot_sync(0xffffffffu, vbad & 2);
      if (mark) reinterpret_cast<short2 *>(smem + C::EXPS)[(i & 3) * BN + crow] = make_short2(kx, vx);
      if (lane == 0)
        reinterpret_cast<int4 *>(smem + C::INFO)[(i & 3) * 4 + cw] = make_int4(mark, n0, n1, 0);
      store_row<HD>(kr, smem + C::K + st * C::TILE, crow, kx, 0u);
      fetch(kr, kpages, i + 1);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kKFull + st));
      if (i >= 2 && !wait_warp(kVFree + st, (i >> 1) - 1)) break;
      store_row<HD>(vr, smem + C::V + st * C::TILE, crow, vx, vbad);
      fetch(vr, vpages, i + 1);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kVFull + st));
    }
  } else if (warp == 12) {
    // ================= MMAs ======================================================
    if (lane == 0) {
      const uint32_t sb = smem_u32(smem);
      auto scores = [&](int m, int i) {
        const uint32_t q0 = sb + C::Q + m * C::TILE, k0 = sb + C::K + (i & 1) * C::TILE;
        const uint32_t d = tm + C::S_COL + 128 * m;
#pragma unroll
        for (int k = 0; k < HD / 16; k++) {
          const uint32_t off = (k >> 2) * C::HALF + (k & 3) * 32;
          mma_f16_ss(d, sdesc(q0 + off, 16, 1024, kLayoutSW128), sdesc(k0 + off, 16, 1024, kLayoutSW128),
                     idesc_f16(BN, 0), k > 0);
        }
        if (i != a.test_stall - 1) mma_commit(bar(kSFull + m));   // test hook: never ready
      };
      auto outputs = [&](int m, int i) {
        const uint32_t v0 = sb + C::V + (i & 1) * C::TILE;
        const uint32_t p = tm + C::S_COL + 128 * m, d = tm + C::O_COL + HD * m;
#pragma unroll
        for (int k = 0; k < BN / 16; k++)
          mma_f16_ts(d, p + 8 * k, sdesc(v0 + k * 2048, C::HALF, 1024, kLayoutSW128),
                     idesc_f16(HD, 1), i > 0 || k > 0);
        if (i == nt[m] - 1) mma_commit(bar(kODone + m));
      };
      // tile i's K (V) is released by the last row tile that uses it
      auto last_user = [&](int i) { return i < nt[1] ? 1 : 0; };
      if (n_tiles > 0 && wait(kKFull, 0)) {
        fence_after_sync();
        for (int m = 0; m < 2; m++)
          if (nt[m] > 0) scores(m, 0);
        mma_commit(bar(kKFree));
      }
      for (int i = 0; i < n_tiles && ok; i++) {
        for (int m = 0; m < 2 && ok; m++) {
          if (i < nt[m]) {
            if (!wait(kPFull + m, i)) break;
            // each tile's V is waited for once
            if (m == (nt[0] > i ? 0 : 1) && !wait(kVFull + (i & 1), i >> 1)) break;
            fence_after_sync();
            outputs(m, i);
            if (m == last_user(i)) mma_commit(bar(kVFree + (i & 1)));
          }
          if (i + 1 < nt[m]) {
            if (m == (nt[0] > i + 1 ? 0 : 1) && !wait(kKFull + ((i + 1) & 1), (i + 1) >> 1)) break;
            fence_after_sync();
            scores(m, i + 1);
            if (m == last_user(i + 1)) mma_commit(bar(kKFree + ((i + 1) & 1)));
          }
        }
      }
      // every MMA has ended before the tensor memory is given back
      mma_commit(bar(kDrain));
      if (!mbar_wait_sleep(bar(kDrain), 0, budget)) {
        atomicOr(a.status, kStatusWaitTimeout);
        ok = false;
      }
    }
    __syncwarp();
  } else {
    // ================= softmax: one row per thread ===============================
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // tensor-memory lane 32 (warp % 4)
    const uint32_t ts = tm + lanes + C::S_COL + 128 * mt, to = tm + lanes + C::O_COL + HD * mt;
    // positions that every row of this row tile attends
    const int first = it.row0 + 128 * mt, last = min(first + 127, it.row0 + it.rows - 1);
    const int all_hi = min(a.tree ? it.old : it.old + first / a.G + 1, end_pos);
    const int all_lo = a.window > 0 ? max(0, it.old + last / a.G + 1 - a.window) : 0;
    const int my_tiles = mt ? nt[1] : nt[0];

    // O times f. Called between S(i) and P'(i): the commit that announced S(i)
    // covers the MMAs before it, the tile before's PV among them, and tile i's is
    // not issued yet.
    auto scale_out = [&](float f) {
#pragma unroll 1
      for (int k = 0; k < HD; k += 32) {
        uint32_t v[32];
        tmem_ld32(to + k, v);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
        uint32_t h0[16], h1[16];
#pragma unroll
        for (int e = 0; e < 16; e++) {
          h0[e] = v[e];
          h1[e] = v[16 + e];
        }
        tmem_st16(to + k, h0);
        tmem_st16(to + k + 16, h1);
      }
      tmem_wait_st();
    };

    auto tile = [&](auto masked_tag, auto slow_tag, int i, int marks) {
      constexpr bool MASKED = decltype(masked_tag)::value, SLOW = decltype(slow_tag)::value;
      const int c0 = base_pos + i * BN;
      const short2 *ex = reinterpret_cast<const short2 *>(smem + C::EXPS) + (i & 3) * BN;
      float mx = -INFINITY;
      int emax = kUnset;
#pragma unroll 1
      for (int ch = 0; ch < 4; ch++) {
        uint32_t v[32];
        tmem_ld32(ts + 32 * ch, v);
        const uint32_t on = MASKED ? mask32(mask, c0 + 32 * ch, end_pos) : 0xffffffffu;
        tmem_wait_ld();
        if constexpr (SLOW) {
          const bool mk = (marks >> ch) & 1;
#pragma unroll 4
          for (int e = 0; e < 32; e++) {
            const short2 x = mk ? ex[32 * ch + e] : make_short2(kref, vref);
            if ((on >> e) & 1) {
              mx = fmaxf(mx, __uint_as_float(v[e]) * pow2i(x.x - kref));
              emax = max(emax, (int)x.y);
            }
          }
        } else {
          float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float x0 = (!MASKED || ((on >> e) & 1)) ? __uint_as_float(v[e]) : -INFINITY;
            const float x1 = (!MASKED || ((on >> (e + 1)) & 1)) ? __uint_as_float(v[e + 1]) : -INFINITY;
            t[(e >> 1) & 3] = max3(t[(e >> 1) & 3], x0, x1);
          }
          mx = fmaxf(mx, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
        }
      }
      // c_row carries 2^kref; the maximum of nothing stays -inf (-inf * 0 is NaN)
      const float xm = mx == -INFINITY ? mx : mx * c_row;
      float f = 1.0f;
      bool move = false;
      if (xm > m_run + 8.0f) {
        f = ex2(m_run - xm);
        m_run = xm;
        l_run *= f;
        move = true;
      }
      if constexpr (SLOW) {
        if (emax != kUnset && (eref == kUnset || emax > eref)) {
          if (eref != kUnset) f *= pow2i(eref - emax);
          eref = emax;
          move = true;
        }
      } else if (eref == kUnset) {
        eref = vref;
      }
      if (i > 0 && __any_sync(0xffffffffu, move)) scale_out(f);
      // weights of unmarked tiles carry 2^(vref - eref) whole; the sum takes it off
      float off = kPShift - (m_run == -INFINITY ? 0.0f : m_run);
      if (!SLOW) off += (float)(vref - eref);
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for (int ch = 0; ch < 4; ch++) {
        uint32_t v[32], p16[16];
        tmem_ld32(ts + 32 * ch, v);
        const uint32_t on = MASKED ? mask32(mask, c0 + 32 * ch, end_pos) : 0xffffffffu;
        tmem_wait_ld();
        if constexpr (SLOW) {
          const bool mk = (marks >> ch) & 1;
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float w[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
              const short2 x = mk ? ex[32 * ch + e + u] : make_short2(kref, vref);
              const bool at = (on >> (e + u)) & 1;
              const float p = at ? ex2(fmaf(__uint_as_float(v[e + u]) * pow2i(x.x - kref), c_row, off)) : 0.0f;
              sum.x += p;
              w[u] = at ? p * pow2i(x.y - eref) : 0.0f;
            }
            p16[e >> 1] = pack_f16(w[0], w[1]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])),
                                        make_float2(c_row, c_row), make_float2(off, off));
            float2 p = make_float2(ex2(x.x), ex2(x.y));
            if (MASKED) {
              if (!((on >> e) & 1)) p.x = 0.0f;
              if (!((on >> (e + 1)) & 1)) p.y = 0.0f;
            }
            sum = __fadd2_rn(sum, p);
            p16[e >> 1] = pack_f16(p.x, p.y);
          }
        }
        tmem_st16(ts + 16 * ch, p16);
      }
      l_run += SLOW ? sum.x + sum.y : (sum.x + sum.y) * pow2i(eref - vref);
      tmem_wait_st();
    };

    c_row *= pow2i(kref >> 1);   // 2^kref in two factors
    c_row *= pow2i(kref - (kref >> 1));
    for (int i = 0; i < my_tiles; i++) {
      if (!wait_warp(kSFull + mt, i)) break;
      fence_after_sync();
      const int c0 = base_pos + i * BN;
      const bool full = c0 >= all_lo && c0 + BN <= all_hi;
      int marks = 0;
      uint32_t nan_any = 0;
      const int4 *info = reinterpret_cast<const int4 *>(smem + C::INFO) + (i & 3) * 4;
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const int4 x = info[w];
        marks |= x.x << w;
        nan_any |= (uint32_t)x.y | (uint32_t)x.z;
      }
      if (nan_any) {
        for (int w = 0; w < 4; w++) {
          const uint32_t on = mask32(mask, c0 + 32 * w, end_pos);
          poison[0] = poison[0] || (on & (uint32_t)info[w].y);
          poison[1] = poison[1] || (on & (uint32_t)info[w].z);
        }
      }
      const bool plain = !marks && __all_sync(0xffffffffu, eref == kUnset || (eref >= vref && eref <= vref + 30));
      if (!plain) tile(std::true_type{}, std::true_type{}, i, marks);
      else if (full) tile(std::false_type{}, std::false_type{}, i, 0);
      else tile(std::true_type{}, std::false_type{}, i, 0);
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kPFull + mt));
    }
  }

  // ---- results --------------------------------------------------------------------
  if (warp < kSoftWarps && ok) {
    const int my_tiles = mt ? nt[1] : nt[0];
    if (my_tiles > 0) {
      wait_warp(kODone + mt, 0);
      fence_after_sync();
    }
  }
  const bool all_ok = __syncthreads_and(ok);
  if (all_ok && warp < kSoftWarps) {
    const int my_tiles = mt ? nt[1] : nt[0];
    const uint32_t to = tm + ((uint32_t)(warp & 3) << 21) + C::O_COL + HD * mt;
    const bool mine = r_loc < it.rows;
    const float down = 0.0078125f;   // 2^-kPShift
    const float L = l_run * down;
    // O carries 2^(kPShift - eref); in two factors
    const int e = eref == kUnset ? 0 : eref;
    const float f0 = pow2i(e >> 1) * down, f1 = pow2i(e - (e >> 1));
#pragma unroll 1
    for (int j = 0; j < HD / 8; j++) {
      uint32_t v[8];
      if (my_tiles > 0) {
        tmem_ld8(to + 8 * j, v);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = 0u;
      }
      const int g = j >> 3;
      float o[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float x = __uint_as_float(v[k]) * f0 * f1;
        o[k] = poison[g] ? __uint_as_float(0x7fc00000u) : x;
      }
      const float lo[4] = {o[0], o[2], o[1], o[3]}, hi[4] = {o[4], o[6], o[5], o[7]};
      const int d = 64 * g + 4 * (j & 7);
      if (mine) {
        if (a.n_splits == 1) {
          extend_store<T>(a, it, r_loc, d, lo, m_run, L, vec);
          extend_store<T>(a, it, r_loc, d + 32, hi, m_run, L, vec);
        } else {
          const size_t pr = part_row(a, it, it.split, r_loc);
          *reinterpret_cast<float4 *>(a.part_o + pr * HD + d) = make_float4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<float4 *>(a.part_o + pr * HD + d + 32) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        }
      }
    }
    if (mine && a.n_splits > 1) {
      const size_t pr = part_row(a, it, it.split, r_loc);
      a.part_m[pr] = m_run;
      a.part_l[pr] = L;
    }
    fence_before_sync();
  }
  __syncthreads();
  fence_after_sync();
  if (warp == 12) tmem_dealloc(tm, C::COLS);
  if (a.n_splits > 1) {
    const bool last = extend_arrive_last(a, it.item);
    if (last && all_ok) extend_merge<HD, T, kThreads>(a, it, vec);
  }
}

template <int HD, typename T>
int launch_one(const ExtendArgs &a, const ExtendBatch &b, int n_blocks, bool vec, cudaStream_t s) {
  using C = WCfg<HD>;
  auto fn = extend_umma_kernel<HD, T>;
  static std::atomic<unsigned long long> attr_done{0};   // one bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(attr_done.load(std::memory_order_acquire) >> (dev & 63) & 1)) {
    int rc = check_cuda(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM),
                        "extend_umma: smem attribute");
    if (rc) return rc;
    attr_done.fetch_or(1ull << (dev & 63), std::memory_order_acq_rel);
  }
  fn<<<n_blocks, kThreads, C::SMEM, s>>>(a, b, vec ? 1 : 0);
  return check_cuda(cudaGetLastError(), "extend_umma launch");
}

}  // namespace

int extend_umma_launch(const ExtendArgs &a, const ExtendBatch &b, int n_blocks, bool vec,
                       cudaStream_t s) {
  if (a.geom.gpd == 2)
    return a.dtype == EAKV_F16 ? launch_one<128, __half>(a, b, n_blocks, vec, s)
                               : launch_one<128, __nv_bfloat16>(a, b, n_blocks, vec, s);
  return a.dtype == EAKV_F16 ? launch_one<64, __half>(a, b, n_blocks, vec, s)
                             : launch_one<64, __nv_bfloat16>(a, b, n_blocks, vec, s);
}

}  // namespace eakv
