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
// f16 but for elements 2^-18 below the row's largest). K' and V' are the dequantized
// values in f16. K' is rounded once (half a step, 2^-11 of the value): with b + 8 s =
// j s + r, j whole, and s = s_hi + s_lo it is m s_hi + (m s_lo + r), m = n - 8 + j, whose first
// product is exact and whose second term is small. With s and b + 8 s rounded to f16
// first, one FMA less, all dims of a position are off alike, which adds up in its
// score: f16 outputs were off by 1.3e-3 of their size in all, now by 0.7e-3, where the
// rounding of a bf16 output alone is 1.7e-3 and that of an f16 one 0.2e-3. In V', whose errors
// are independent from position to position, s is one f16. Keeping K's nibbles
// exact instead needs a second accumulator per 64-dim group, for which tensor memory
// has no room, and four more FMAs per score; f32 rows, which the warp-level kernel
// serves, have them exact. P' = 2^7 p is at most 2^15, one f16.
//
// Ranges. K and V are multiplied by powers of two that take the largest row of the
// first tile (eref) to 2^10. Rows up to 2^4 above it stay in f16's range, and a group's
// scale is a normal f16 number down to groups 2^-21 of the reference (each factor of two
// below costs a bit). A run of 32 positions with a row above that, or 2^-10 below the
// reference, or with V of zeros, is marked: its rows have powers of their own, which go to
// the softmax threads beside it, and these scale the scores and the weights column by column, with
// a V reference of their own per row, taken from attended positions only (of zeros:
// none). So a position that a row does not attend has no influence on it, however large.
// (With the reference at 2^0 and high nibbles held times 16 with a sixteenth of the
// scale, groups 2^-12 of their neighbour lost all but 3 to 5 bits.)
// Non-finite V groups are kept out of the products (0 NaN is NaN) and
// listed by position; a row that attends one gets NaN in the group's dims.
//
// Roles (16 warps). Warps 0-3 and 4-7: softmax of row tile 0 and 1, one thread
// per row, its 128 scores in registers; the weights go over S, and O is scaled
// when a maximum moves. Warps 8-11: dequantize, one thread per position: its K and
// V rows come from global memory a tile ahead in registers and leave as 16-byte
// stores in the 128-byte swizzle. A 32-bit word of nibbles becomes one 16-byte
// chunk [d, d+2, d+1, d+3, d+32, d+34, d+33, d+35] (the pairs that one mask selects);
// Q' is stored in the same order and the output's columns are read back in it, so
// the order costs nothing. Warp 12 issues the MMAs: for tile i, PV of row tile 0,
// S(i+1) of row tile 0, the same for row tile 1, so one row tile's softmax runs
// under the other's MMAs; PV starts on the first half of a tile's weights. Warp 13
// finds the CTA's next part while this one is worked on; the last two only fill
// their warpgroup. P' of a tile lies over its S (tensor memory: 2 x 128 columns of S,
// 2 x 128 of O: all 512); the tensor pipe runs the MMAs in order. The softmax
// warpgroups take registers from the other two.
//
// Bound: the tensor pipe, whose operands come from shared memory at its full rate
// (S = Q'K' reads 128 bytes a cycle) next to the dequantizing stores: 2048 tokens
// of 32 heads (8 KV heads, head_dim 128) behind 32768 positions in 1.19 to 1.24 ms,
// 0.92 to 0.95 PFLOP/s, box to box. Tried and slower: tiles of 64 positions with two S buffers (its
// MMAs are 1.4 times slower per value), one pass over the scores in place of the
// registers, exponentials by polynomial on the FMA pipe for a quarter or half of
// them (the exponentials are not what it waits for).
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
constexpr int kStages = 2;                    // K and V operands in flight
// Tiles whose marks are kept: those of tile i+2 are written when S(i) is done,
// and the softmax threads look at tile i's, and i-1's, until P'(i) is.
constexpr int kInfo = 4;
constexpr int kSoftWarps = 8, kConvWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kConvWarps;
constexpr int kWalkWarp = kMmaWarp + 1;
constexpr int kWorkThreads = (kWalkWarp + 1) * 32;
constexpr int kThreads = (kSoftWarps + kConvWarps + 4) * 32;   // four warpgroups, the last mostly idle
// Registers per thread: the launch gives each thread kRegs, and the warpgroups
// trade them (512 threads x 128 = 128 x (2 kRegsSoft + kRegsConv + kRegsMma)).
constexpr int kRegs = 128, kRegsSoft = 176, kRegsConv = 104, kRegsMma = 56;
static_assert(2 * kRegsSoft + kRegsConv + kRegsMma == 4 * kRegs, "register split");
constexpr int kUnset = -100000;
constexpr int kZeroRow = -1000;               // exponent of a row of zeros, below every other
constexpr int kTop = 10;                      // a row's values below 2^(e+1) are held below 2^(kTop+1)
constexpr int kUp = 4, kDown = 10;            // rows within 2^kUp, 2^-kDown of eref need no mark
static_assert(kTop + 1 + kUp <= 15, "rows without a mark fit f16");
constexpr float kPShift = 7.0f;               // P' = 2^7 p
constexpr uint32_t kLayoutSW128 = 2;

template <int HD>
struct WCfg {
  static constexpr int NG = HD / 64;
  static constexpr int PB = kPagePositions * NG * 40;
  static constexpr int NIB = kPagePositions * NG * 32;
  static constexpr int QTILE = 128 * HD * 2;  // bytes of a row tile of Q'
  static constexpr int QHALF = 128 * 128;     // bytes of its 64-dim half
  static constexpr int TILE = BN * HD * 2;    // bytes of a tile's K' or V'
  static constexpr int HALF = BN * 128;
  static constexpr int Q = 0;                 // two row tiles
  static constexpr int K = Q + 2 * QTILE;
  static constexpr int V = K + kStages * TILE;
  // marked rows' exponents and the warps' marks of kInfo tiles
  static constexpr int EXPS = V + kStages * TILE;            // short2 [kInfo][BN]: K, V
  static constexpr int INFO = EXPS + kInfo * BN * 4;         // int [kInfo][4 warps]
  static constexpr int NANS = INFO + kInfo * 16;             // uint2 [kInfo][4 warps]
  static constexpr int ROWC = NANS + kInfo * 32;             // float [256]: score factor of a row
  static constexpr int BARS = ROWC + 256 * 4;
  // tensor-memory base, `a wait ran out', the item's last part, `its arrival is said'
  static constexpr int SLOT = BARS + 8 * 18;
  static constexpr int RED = SLOT + 16;                      // int2 [4 warps]: largest exponents
  static constexpr int WALK = RED + 32;                      // ExtWalk
  static constexpr int END = WALK + 256;
  static constexpr int SMEM = END + 1024;                    // alignment slack
  static_assert(sizeof(ExtWalk) <= 256, "room for the walk");
  // tensor memory columns
  static constexpr int S_COL = 0, O_COL = 256, COLS = 512;
  static_assert(BARS % 8 == 0 && ROWC % 16 == 0 && SLOT % 8 == 0, "alignment");
};

// Barriers: per stage K and V filled and free; per row tile scores there, each
// half of the weights there, all outputs summed.
enum { kKFull = 0, kVFull = 2, kKFree = 4, kVFree = 6, kSFull = 8, kPFull = 10, kODone = 14, kDrain = 16 };

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

__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ uint4 ldg_row(const void *p) {
  uint4 r;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ float pow2i(int e) {   // 2^e, 0 below the normal range
  return __uint_as_float((uint32_t)min(max(127 + e, 0), 254) << 23);
}
// Two values as T in one word.
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) { return pack_f16(x, y); }
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Waits for the warp's tensor-memory loads, and ties the registers of one to
// the wait: what reads them cannot be moved ahead of it.
__device__ __forceinline__ void wait_ld_of(uint32_t (&v)[32]) {
#define EAKV_T8(i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), \
                   "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7])
  asm volatile("tcgen05.wait::ld.sync.aligned;" : EAKV_T8(0), EAKV_T8(8), EAKV_T8(16), EAKV_T8(24)::"memory");
#undef EAKV_T8
}

// The first trade ends with a barrier of the whole CTA: a warpgroup that has
// little to do would otherwise ask for its registers back before the softmax
// warps have got theirs, and both would wait for good.
__device__ __forceinline__ void regs_traded() { named_sync(2, kThreads); }
template <int N> __device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
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

// A group with a scale of 1 and only zero nibbles, the quantizer's form of 64 equal
// values, gets a scale of 0: b + 8 s and the row's power of two are the values' own.
template <int HD>
__device__ __forceinline__ void drop_idle_scales(RawRow<HD> &r) {
#pragma unroll
  for (int g = 0; g < HD / 64; g++)
    if (r.sb[2 * g] == 1.0f) {
      const uint4 x = r.w[2 * g], y = r.w[2 * g + 1];
      if (((x.x | x.y | x.z | x.w) | (y.x | y.y | y.z | y.w)) == 0) r.sb[2 * g] = 0.0f;
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

// The row's values times 2^(kTop - e) as f16 into row `row` of an operand: 16-byte
// chunk k of half g holds word k of group g. A group in `zero` is stored as 0.
// KEY: with s in two limbs; else s is rounded first.
template <int HD, bool KEY>
__device__ __forceinline__ void store_row(const RawRow<HD> &r, uint8_t *op, int row, int e,
                                          uint32_t zero) {
  using C = WCfg<HD>;
  // in two factors: e spans more than the exponents of one float
  const int up = kTop - e;
  const float f0 = pow2i(up >> 1), f1 = pow2i(up - (up >> 1));
#pragma unroll
  for (int g = 0; g < HD / 64; g++) {
    const float s = r.sb[2 * g] * f0 * f1, b = fmaf(8.0f, r.sb[2 * g], r.sb[2 * g + 1]) * f0 * f1;
    // b = j s + r, and s in two limbs: m s_hi is exact for m = n - 8 + j (6 and 5 bits),
    // m s_lo + r is small. (s = 0 gives j of either end and r = b.)
    const float j = fminf(fmaxf(rintf(__fdividef(b, s)), -16.0f), 16.0f);
    const float hi = KEY ? __uint_as_float(__float_as_uint(s) & 0xFFFC0000u) : s;
    __half2 sh = __float2half2_rn(hi), sl = __float2half2_rn(s - hi), rr = __float2half2_rn(fmaf(-j, s, b));
    if ((zero >> g) & 1) sh = sl = rr = __float2half2_rn(0.0f);
    // n of a low nibble lies in 1024 + n, of a high one in 1024 + 16 n, a sixteenth of
    // which is 64 + n: all exact
    const __half2 off_lo = __float2half2_rn(1032.0f - j), off_hi = __float2half2_rn(j - 72.0f);
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const uint32_t words[8] = {r.w[2 * g].x, r.w[2 * g].y, r.w[2 * g].z, r.w[2 * g].w,
                               r.w[2 * g + 1].x, r.w[2 * g + 1].y, r.w[2 * g + 1].z, r.w[2 * g + 1].w};
    uint8_t *base = op + g * C::HALF + row * 128;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const uint32_t w = words[k], y = w >> 8;
      const __half2 lo0 = __hsub2(as_half2(and_or(w, 0x000F000Fu, 0x64006400u)), off_lo);
      const __half2 lo1 = __hsub2(as_half2(and_or(y, 0x000F000Fu, 0x64006400u)), off_lo);
      const __half2 hi0 = __hfma2(as_half2(and_or(w, 0x00F000F0u, 0x64006400u)), sixteenth, off_hi);
      const __half2 hi1 = __hfma2(as_half2(and_or(y, 0x00F000F0u, 0x64006400u)), sixteenth, off_hi);
      auto value = [&](__half2 m) { return as_u32(__hfma2(m, sh, KEY ? __hfma2(m, sl, rr) : rr)); };
      *reinterpret_cast<uint4 *>(base + ((k ^ (row & 7)) << 4)) =
          make_uint4(value(lo0), value(lo1), value(hi0), value(hi1));
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

// Out of line: hardly any call has depths.
__device__ __noinline__ RowMask depth_mask(const ExtendArgs &a, const ExtItem &it, int r) {
  RowMask m = row_mask(a, it, r);
  depth_window(a, it, r, m);
  return m;
}

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, 1)
extend_umma_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExtendBatch batch,
                   const __grid_constant__ ExtendRuns runs, const int vec) {
  using C = WCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t bars = smem_u32(smem + C::BARS);
  auto bar = [&](int i) { return bars + 8 * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t budget = min(a.wait_budget, 1u << 18);
  ExtWalk &walk = *reinterpret_cast<ExtWalk *>(smem + C::WALK);
  volatile int *failed = reinterpret_cast<volatile int *>(smem + C::SLOT + 4);

  if (warp == kMmaWarp) {
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
      mbar_init(bar(kPFull + 2 + i), 4);
      mbar_init(bar(kODone + i), 1);
    }
    mbar_init(bar(kDrain), 1);
    fence_mbar_init();
    *failed = 0;
    walk.begin(a, batch, runs);
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tm = *reinterpret_cast<const uint32_t *>(smem + C::SLOT);

  // Bounded wait of a whole warp for use `use` of barrier b (how often it was
  // waited for before): its lanes go on, or leave, together.
  bool ok = true;
  auto wait_warp = [&](int b, int use) {
    if (!__all_sync(0xffffffffu, mbar_wait_sleep(bar(b), use & 1, budget))) {
      if (lane == 0) {
        atomicOr(a.status, kStatusWaitTimeout);
        *failed = 1;
      }
      ok = false;
    }
    return ok;
  };
  // Every role walks the same parts of items. They meet twice in each: when Q'
  // and the references are there, and when nothing of the part is in use any
  // more.
  auto meet = [&] { named_sync(3, kWorkThreads); };
  // Positions of part p, and its tiles for each row tile; false behind the last
  // part, or at one outside its cache.
  int base_pos, end_pos, nt0, nt1, n_tiles;
  auto begin_part = [&](const ExtItem &it) {
    if (it.state <= 0) return false;
    base_pos = it.pg0 * kPagePositions;
    end_pos = (it.pg0 + it.npages) * kPagePositions;
    auto tiles_of = [&](int m) {
      if (it.rows <= 128 * m) return 0;
      const int last = min(it.row0 + 128 * m + 127, it.row0 + it.rows - 1);
      const int hi = min(a.tree ? it.hi : it.old + last / a.G + 1, end_pos);
      return hi > base_pos ? (hi - base_pos + BN - 1) / BN : 0;
    };
    nt0 = tiles_of(0);
    nt1 = tiles_of(1);
    n_tiles = max(nt0, nt1);
    return true;
  };
  // references of the part, from the dequantizing warps' maxima
  int kref, vref;
  auto references = [&] {
    kref = vref = kUnset;
#pragma unroll
    for (int w = 0; w < kConvWarps; w++) {
      const int2 e = reinterpret_cast<const int2 *>(smem + C::RED)[w];
      kref = max(kref, e.x);
      vref = max(vref, e.y);
    }
    if (kref == kUnset) kref = 0;
    if (vref == kUnset) vref = 0;
  };

  if (warp >= kSoftWarps && warp < kMmaWarp) {
    // ================= dequantize ================================================
    regs_down<kRegsConv>();
    regs_traded();
    const int cw = warp - kSoftWarps, crow = threadIdx.x & 127;   // its position in a tile
    int done = 0;   // tiles of the parts before
    for (int part = 0;; part++) {
      const ExtItem &it = walk.item[part & 1];
      if (!begin_part(it)) break;
      const uint8_t *kpages = it.base + page_index(a.geom, a.layer, 0, it.h, it.pg0) * C::PB +
                              (size_t)(crow / kPagePositions) * C::PB;
      const uint8_t *vpages = kpages + (size_t)a.geom.n_heads * a.geom.n_pages * C::PB;
      RawRow<HD> kr, vr;
      // This thread's row of tile i, zeros when no row of the item may attend it.
      auto fetch = [&](RawRow<HD> &r, const uint8_t *pages, int i) {
        const int p = base_pos + i * BN + crow;
        if (i < n_tiles && p >= it.lo && p < it.hi && p < end_pos) {
          load_row<HD>(r, pages + (size_t)i * (2 * C::PB), crow % kPagePositions);
        } else {
#pragma unroll
          for (int k = 0; k < HD / 32; k++) r.w[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int k = 0; k < 2 * C::NG; k++) r.sb[k] = 0.0f;
        }
      };
      fetch(kr, kpages, 0);
      fetch(vr, vpages, 0);
      drop_idle_scales<HD>(kr);
      drop_idle_scales<HD>(vr);
      uint32_t bad;
      const int ek = __reduce_max_sync(0xffffffffu, row_exp<HD>(kr, bad));
      const int ev = __reduce_max_sync(0xffffffffu, row_exp<HD>(vr, bad));
      if (lane == 0) reinterpret_cast<int2 *>(smem + C::RED)[cw] = make_int2(ek, ev);
      meet();
      references();
      for (int i = 0; i < n_tiles; i++) {
        const int n = done + i, st = n & 1;
        if (i > 0) {
          drop_idle_scales<HD>(kr);
          drop_idle_scales<HD>(vr);
        }
        uint32_t kbad, vbad;
        const int ke = row_exp<HD>(kr, kbad), ve = row_exp<HD>(vr, vbad);
        const int pos = base_pos + i * BN + crow;
        const bool in = pos >= it.lo && pos < it.hi && pos < end_pos;   // zeros outside are not attended
        const bool mark = __any_sync(0xffffffffu, (ke != kUnset && (ke > kref + kUp || ke < kref - kDown)) ||
                                                      (ve != kUnset && (ve > vref + kUp || ve < vref - kDown)) ||
                                                      (ve == kUnset && !vbad && in));
        const int kx = mark && ke != kUnset ? ke : kref;
        const int vx = !mark ? vref : ve != kUnset ? ve : kZeroRow;
        // a non-finite K group keeps its NaN, which reaches its own score only; a V
        // group is listed instead
        const uint32_t n0 = __ballot_sync(0xffffffffu, vbad & 1), n1 = __ballot_sync(0xffffffffu, vbad & 2);
        if (n >= 2 && !wait_warp(kKFree + st, (n >> 1) - 1)) break;
        if (mark) reinterpret_cast<short2 *>(smem + C::EXPS)[(n % kInfo) * BN + crow] = make_short2(kx, vx);
        if (lane == 0) {
          reinterpret_cast<int *>(smem + C::INFO)[(n % kInfo) * 4 + cw] = (mark ? 1 : 0) | ((n0 | n1) ? 2 : 0);
          reinterpret_cast<uint2 *>(smem + C::NANS)[(n % kInfo) * 4 + cw] = make_uint2(n0, n1);
        }
        store_row<HD, true>(kr, smem + C::K + st * C::TILE, crow, kx, 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kKFull + st));
        fetch(kr, kpages, i + 1);
        if (n >= 2 && !wait_warp(kVFree + st, (n >> 1) - 1)) break;
        store_row<HD, false>(vr, smem + C::V + st * C::TILE, crow, vx, vbad);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kVFull + st));
        fetch(vr, vpages, i + 1);
      }
      done += n_tiles;
      meet();
      if (*failed) break;
    }
  } else if (warp >= kMmaWarp) {
    // ================= MMAs ======================================================
    regs_down<kRegsMma>();
    regs_traded();
    if (warp == kMmaWarp) {
      int done = 0, done0 = 0, done1 = 0;   // tiles of the parts before, of each row tile
      // The whole warp walks the tiles, so that descriptors stay in uniform
      // registers; one lane issues.
      const bool issuer = elect_one();
      const uint32_t sb = smem_u32(smem);
      const uint64_t qd = sdesc(sb + C::Q, 16, 1024, kLayoutSW128);
      const uint64_t kd = sdesc(sb + C::K, 16, 1024, kLayoutSW128);
      const uint64_t vd = sdesc(sb + C::V, C::HALF, 1024, kLayoutSW128);
      // a descriptor's address field counts 16 bytes
      auto scores = [&](int m, int i) {
        const uint64_t q = qd + (uint64_t)(m * (C::QTILE >> 4));
        const uint64_t k = kd + (uint64_t)(((done + i) & 1) * (C::TILE >> 4));
        const uint32_t d = tm + C::S_COL + 128 * m;
        if (issuer) {
#pragma unroll
          for (int s = 0; s < HD / 16; s++) {
            const uint64_t off = ((s >> 2) * C::HALF + (s & 3) * 32) >> 4;
            mma_f16_ss(d, q + off, k + off, idesc_f16(BN, 0), s > 0);
          }
          if (i != a.test_stall - 1) mma_commit(bar(kSFull + m));   // test hook: never ready
          // the tile's K is free when the last row tile that uses it has its scores
          if (m == (i < nt1 ? 1 : 0)) mma_commit(bar(kKFree + ((done + i) & 1)));
        }
      };
      // PV of tile i, half by half as the weights come; false when a wait ran out
      auto outputs = [&](int m, int i, int n) {
        const uint64_t v = vd + (uint64_t)(((done + i) & 1) * (C::TILE >> 4));
        const uint32_t p = tm + C::S_COL + 128 * m, d = tm + C::O_COL + HD * m;
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if (!wait_warp(kPFull + 2 * m + h, (m ? done1 : done0) + i)) return false;
          fence_after_sync();
          if (issuer) {
#pragma unroll
            for (int s = h * (BN / 32); s < (h + 1) * (BN / 32); s++)
              mma_f16_ts(d, p + 8 * s, v + (uint64_t)(s * (2048 >> 4)), idesc_f16(HD, 1), i > 0 || s > 0);
          }
        }
        if (issuer) {
          if (m == (i < nt1 ? 1 : 0)) mma_commit(bar(kVFree + ((done + i) & 1)));
          if (i == n - 1) mma_commit(bar(kODone + m));
        }
        return true;
      };
      // Each tile's K and V is waited for once, ahead of the weights that it is
      // used behind, so that nothing stands between these and their MMAs.
      for (int part = 0;; part++) {
        const ExtItem &it = walk.item[part & 1];
        if (!begin_part(it)) break;
        meet();
        if (n_tiles > 0 && wait_warp(kKFull + (done & 1), done >> 1)) {
          fence_after_sync();
          if (nt0 > 0) scores(0, 0);
          if (nt1 > 0) scores(1, 0);
        }
        for (int i = 0; i < n_tiles && ok; i++) {
          if (i + 1 < n_tiles && !wait_warp(kKFull + ((done + i + 1) & 1), (done + i + 1) >> 1)) break;
          if (!wait_warp(kVFull + ((done + i) & 1), (done + i) >> 1)) break;
          if (i < nt0) {
            if (!outputs(0, i, nt0)) break;
            if (i + 1 < nt0) scores(0, i + 1);
          }
          if (i < nt1) {
            if (!outputs(1, i, nt1)) break;
            if (i + 1 < nt1) scores(1, i + 1);
          }
        }
        done += n_tiles;
        done0 += nt0;
        done1 += nt1;
        meet();
        if (*failed) break;
      }
      // every MMA has ended before the tensor memory is given back
      if (issuer) mma_commit(bar(kDrain));
      __syncwarp();
      wait_warp(kDrain, 0);
    } else if (warp == kWalkWarp) {
      // ================= walk: the next part, while this one is worked on ===========
      int part = 0;
      for (; walk.item[part & 1].state > 0; part++) {
        meet();
        if (lane == 0) walk.next(a, batch, part + 1);
        meet();
        if (*failed) {
          const ExtItem &it = walk.item[part & 1];
          const bool arrived = it.n_parts == 1 || *reinterpret_cast<volatile int *>(smem + C::SLOT + 12);
          if (lane == 0 && !arrived) atomicInc(a.cnt + it.counter, (unsigned)it.n_parts - 1);
          part++;
          break;
        }
      }
      if (lane == 0) walk.abandon(a, batch, part);
    }
  } else {
    // ================= softmax: one row per thread ===============================
    regs_up<kRegsSoft>();
    regs_traded();
    const int mt = warp >> 2;                            // row tile
    // tiles of the parts before: of this row tile, of both; parts with tiles
    int done = 0, all_done = 0, parts = 0;
    for (int part = 0;; part++) {
      const ExtItem &it = walk.item[part & 1];
      if (!begin_part(it)) break;
      // ---- Q' ----------------------------------------------------------------------
      // A row is HD/8 lanes of eight dims each; its power of two goes into ROWC
      // with the scale. Rows behind the last repeat it.
      {
        constexpr int LPR = HD / 8, RPW = 32 / LPR;   // lanes per row, rows per warp and step
        const int d = 8 * (lane % LPR);
        const int rl0 = 32 * warp + lane / LPR;
        RowWalk row(a, it, a.q, rl0, RPW);
        const float sign = a.scale_log2 < 0.0f ? -1.0f : 1.0f;
        const int j = (d & 31) >> 2;
        uint8_t *op = smem + C::Q + mt * C::QTILE + (d >> 6) * C::QHALF + ((d & 32) >> 2);
        // kBatch rows' loads before the first is looked at
        auto rows = [&](auto vec_tag) {
          constexpr int kBatch = 8;
#pragma unroll 1
          for (int s0 = 0; s0 < 32 / RPW; s0 += kBatch) {
            float v[kBatch][2][4];
#pragma unroll
            for (int s = 0; s < kBatch; s++) {
              const T *qp = reinterpret_cast<const T *>(a.q.data) + row.at + d;
              load4<T, decltype(vec_tag)::value>(qp, v[s][0]);
              load4<T, decltype(vec_tag)::value>(qp + 4, v[s][1]);
              if (rl0 + (s0 + s + 1) * RPW < it.rows) row.step();
            }
#pragma unroll
            for (int s = 0; s < kBatch; s++) {
              const int rl = rl0 + (s0 + s) * RPW, rr = rl & 127;
              float (&v0)[4] = v[s][0], (&v1)[4] = v[s][1];
              // largest magnitude as bits: infinities and NaN come out on top
              uint32_t mx = 0;
#pragma unroll
              for (int e = 0; e < 4; e++)
                mx = max(mx, max(__float_as_uint(v0[e]) & 0x7fffffffu, __float_as_uint(v1[e]) & 0x7fffffffu));
#pragma unroll
              for (int o = 1; o < LPR; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
              const bool fine = mx < 0x7f800000u;
              // mx in [2^(e-1), 2^e), e = (mx >> 23) - 126; times 2^(5 - e)
              const int qe = mx == 0 || !fine ? 0 : max(min(131 - (int)(mx >> 23), 126), -126);
              const float up = fine ? sign * pow2i(qe) : 0.0f;
              if (d == 0)
                reinterpret_cast<float *>(smem + C::ROWC)[rl] =
                    fine ? fabsf(a.scale_log2) * pow2i(-qe) : __uint_as_float(0x7fc00000u);
              if (!fine) {
#pragma unroll
                for (int e = 0; e < 4; e++) v0[e] = v1[e] = 0.0f;
              }
              // dims d..d+3 and d+4..d+7: the low or high halves of chunks j and j + 1
              *reinterpret_cast<uint2 *>(op + rr * 128 + ((j ^ (rr & 7)) << 4)) =
                  make_uint2(pack_f16(v0[0] * up, v0[2] * up), pack_f16(v0[1] * up, v0[3] * up));
              *reinterpret_cast<uint2 *>(op + rr * 128 + (((j + 1) ^ (rr & 7)) << 4)) =
                  make_uint2(pack_f16(v1[0] * up, v1[2] * up), pack_f16(v1[1] * up, v1[3] * up));
            }
          }
        };
        if (vec) rows(std::true_type{});
        else rows(std::false_type{});
        fence_proxy_async_smem();
      }
      meet();
      references();
      const int r_loc = 128 * mt + (threadIdx.x & 127);    // row within the item
      RowMask mask = row_mask(a, it, it.row0 + min(r_loc, it.rows - 1));
      if (a.depth && a.window > 0) mask = depth_mask(a, it, it.row0 + min(r_loc, it.rows - 1));
      // score factor: |scale| log2 e / 2^(q exponent), with K's 2^(kref - kTop)
      float c_row = reinterpret_cast<const float *>(smem + C::ROWC)[r_loc];
      c_row *= pow2i((kref - kTop) >> 1);
      c_row *= pow2i(kref - kTop - ((kref - kTop) >> 1));
      float m_run = -INFINITY, l_run = 0.0f;
      int eref = kUnset;
      bool poison0 = false, poison1 = false;   // a non-finite V group was attended
      bool steady = true;   // of the warp: no row's eref is far from vref
      const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // tensor-memory lane 32 (warp % 4)
      const uint32_t ts = tm + lanes + C::S_COL + 128 * mt, to = tm + lanes + C::O_COL + HD * mt;
      // positions that every row of this row tile attends
      const int first = it.row0 + 128 * mt, last = min(first + 127, it.row0 + it.rows - 1);
      const int all_hi = min(a.tree ? it.old : it.old + first / a.G + 1, end_pos);
      const int all_lo = a.window > 0 ? max(0, it.old + last / a.G + 1 - a.window) : 0;
      const int my_tiles = mt ? nt1 : nt0;

      // O times f. Called between S(i) and P'(i): the commit that announced S(i)
      // covers the MMAs before it, the tile before's PV among them, and tile i's is
      // not issued yet.
      auto scale_out = [&](float f) {
#pragma unroll 1
        for (int k = 0; k < HD; k += 16) {
          uint32_t v[16];
          tmem_ld16(to + k, v);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
          tmem_st16(to + k, v);
        }
      };
      // Half h of the tile's weights is in tensor memory (and O is scaled).
      auto announce = [&](int h) {
        tmem_wait_st();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPFull + 2 * mt + h));
      };
      // The scores' maximum xm of a tile (base 2, -inf: none) moves the running
      // maximum when it passes it by 8; `f` is what the sums so far are scaled by.
      auto new_max = [&](float xm, float &f) {
        f = 1.0f;
        if (xm > m_run + 8.0f) {
          f = ex2(m_run - xm);
          m_run = xm;
          l_run *= f;
          return true;
        }
        return false;
      };

      // A tile without marked rows: the row's 128 scores in registers.
      auto tile_fast = [&](auto masked_tag, int i) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        const int c0 = base_pos + i * BN;
        uint32_t v[4][32];
#pragma unroll
        for (int ch = 0; ch < 4; ch++) tmem_ld32(ts + 32 * ch, v[ch]);
#pragma unroll
        for (int ch = 0; ch < 4; ch++) wait_ld_of(v[ch]);
        if constexpr (MASKED) {
#pragma unroll
          for (int ch = 0; ch < 4; ch++) {
            const uint32_t on = mask32(mask, c0 + 32 * ch, end_pos);
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (!((on >> e) & 1)) v[ch][e] = 0xff800000u;   // -inf
          }
        }
        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int ch = 0; ch < 4; ch++)
#pragma unroll
          for (int e = 0; e < 32; e += 8)
#pragma unroll
            for (int k = 0; k < 4; k++)
              t[k] = max3(t[k], __uint_as_float(v[ch][e + 2 * k]), __uint_as_float(v[ch][e + 2 * k + 1]));
        const float mx = fmaxf(max3(t[0], t[1], t[2]), t[3]);
        // the maximum of nothing stays -inf (-inf * 0 is NaN)
        const float xm = mx == -INFINITY ? mx : mx * c_row;
        // the first positions that the row attends (of each their V is within vref's range)
        if (eref == kUnset && mx > -INFINITY) eref = vref;
        const int e_off = eref == kUnset ? 0 : vref - eref;
        if (__any_sync(0xffffffffu, xm > m_run + 8.0f)) {
          float f;
          new_max(xm, f);
          if (i > 0) scale_out(f);
        }
        // the weights carry 2^(vref - eref) whole; the sum takes it off
        const float off = kPShift - (m_run == -INFINITY ? 0.0f : m_run) + (float)e_off;
        const float2 c2 = make_float2(c_row, c_row), o2 = make_float2(off, off);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int ch = 0; ch < 4; ch++) {
          uint32_t p16[16];
          const uint32_t (&x)[32] = v[ch];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 y = __ffma2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), c2, o2);
            float2 p = make_float2(ex2(y.x), ex2(y.y));
            if (MASKED) {   // -inf * 0 where c_row is 0
              if (x[e] == 0xff800000u) p.x = 0.0f;
              if (x[e + 1] == 0xff800000u) p.y = 0.0f;
            }
            sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], p);
            p16[e >> 1] = pack_f16(p.x, p.y);
          }
          tmem_st16(ts + 16 * ch, p16);
          if (ch == 1) announce(0);
        }
        l_run += (sum[0].x + sum[0].y + sum[1].x + sum[1].y) * pow2i(-e_off);
        announce(1);
      };

      // Any tile: every position with its own powers of two.
      auto tile_slow = [&](int i, int marks) {
        const int c0 = base_pos + i * BN;
        const short2 *ex = reinterpret_cast<const short2 *>(smem + C::EXPS) + ((all_done + i) % kInfo) * BN;
        float mx = -INFINITY;
        int emax = kZeroRow;
#pragma unroll 1
        for (int ch = 0; ch < 4; ch++) {
          uint32_t v[32];
          tmem_ld32(ts + 32 * ch, v);
          const uint32_t on = mask32(mask, c0 + 32 * ch, end_pos);
          const bool mk = (marks >> ch) & 1;
          wait_ld_of(v);
#pragma unroll
          for (int e = 0; e < 32; e++) {
            const short2 x = mk ? ex[32 * ch + e] : make_short2(kref, vref);
            if ((on >> e) & 1) {
              mx = fmaxf(mx, __uint_as_float(v[e]) * pow2i(x.x - kref));
              emax = max(emax, (int)x.y);
            }
          }
        }
        float f;
        bool move = new_max(mx == -INFINITY ? mx : mx * c_row, f);
        if (emax > kZeroRow && (eref == kUnset || emax > eref)) {
          if (eref != kUnset) f *= pow2i(eref - emax);
          eref = emax;
          move = true;
        }
        if (i > 0 && __any_sync(0xffffffffu, move)) scale_out(f);
        const float off = kPShift - (m_run == -INFINITY ? 0.0f : m_run);
#pragma unroll 1
        for (int ch = 0; ch < 4; ch++) {
          uint32_t v[32], p16[16];
          tmem_ld32(ts + 32 * ch, v);
          const uint32_t on = mask32(mask, c0 + 32 * ch, end_pos);
          const bool mk = (marks >> ch) & 1;
          wait_ld_of(v);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float w[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
              const short2 x = mk ? ex[32 * ch + e + u] : make_short2(kref, vref);
              const bool at = (on >> (e + u)) & 1;
              const float p = at ? ex2(fmaf(__uint_as_float(v[e + u]) * pow2i(x.x - kref), c_row, off)) : 0.0f;
              l_run += p;
              w[u] = at && x.y > kZeroRow ? p * pow2i(x.y - eref) : 0.0f;
            }
            p16[e >> 1] = pack_f16(w[0], w[1]);
          }
          tmem_st16(ts + 16 * ch, p16);
        }
        announce(0);
        announce(1);
      };

      for (int i = 0; i < my_tiles; i++) {
        if (!wait_warp(kSFull + mt, done + i)) break;
        fence_after_sync();
        const int c0 = base_pos + i * BN;
        const bool full = c0 >= all_lo && c0 + BN <= all_hi;
        // bit 0 of a warp's word: marked rows, bit 1: non-finite V groups
        const int4 sum = *reinterpret_cast<const int4 *>(smem + C::INFO + ((all_done + i) % kInfo) * 16);
        const int any = sum.x | sum.y | sum.z | sum.w;
        if (any & 2) {
          const uint2 *bad = reinterpret_cast<const uint2 *>(smem + C::NANS) + ((all_done + i) % kInfo) * 4;
          for (int w = 0; w < 4; w++) {
            const uint32_t on = mask32(mask, c0 + 32 * w, end_pos);
            poison0 = poison0 || (on & bad[w].x);
            poison1 = poison1 || (on & bad[w].y);
          }
        }
        if ((any & 1) || !steady) {
          tile_slow(i, (sum.x & 1) | (sum.y & 1) << 1 | (sum.z & 1) << 2 | (sum.w & 1) << 3);
          steady = __all_sync(0xffffffffu, eref == kUnset || (eref >= vref && eref <= vref + 30));
        } else if (full) {
          tile_fast(std::false_type{}, i);
        } else {
          tile_fast(std::true_type{}, i);
        }
      }

      // ---- results ----------------------------------------------------------------
      if (ok && my_tiles > 0) wait_warp(kODone + mt, parts);
      // both row tiles are through with K' and V': their space takes the rows on
      // their way out
      named_sync(1, kSoftWarps * 32);
      if (ok) {
        fence_after_sync();
        const float down = 0.0078125f;   // 2^-kPShift
        const float L = l_run * down;
        // O carries 2^(kPShift + kTop - eref); in two factors. Finished rows are divided here.
        const int e = eref == kUnset ? 0 : eref - kTop;
        const float inv = it.n_parts > 1 ? 1.0f : (L == 0.0f ? 0.0f : 1.0f / L);
        const float f0 = pow2i(e >> 1) * down, f1 = pow2i(e - (e >> 1)) * inv;
        if (r_loc < it.rows) {
          if (it.n_parts > 1) {
            const size_t pr = part_row(a, it.slot, r_loc);
            a.part_m[pr] = m_run;
            a.part_l[pr] = L;
          } else if (a.lse) {
            extend_lse(a, it, r_loc, m_run, L);
          }
        }
        // A thread's row leaves by way of shared memory, so that whole lines are
        // stored: up to 256 bytes of a row at a time, 32 rows per warp.
        uint8_t *stage = smem + C::K + warp * (32 * 256);
        static_assert(8 * 32 * 256 <= 2 * kStages * C::TILE, "room for the rows of eight warps");
        const int per_pass = it.n_parts > 1 ? 64 : HD;
        const bool spoiled = __any_sync(0xffffffffu, poison0 || poison1);
#pragma unroll 1
        for (int d0 = 0; d0 < HD; d0 += per_pass) {
          // 16 columns: dims 4j..4j+7 and 32 on of a 64-dim group
#pragma unroll 2
          for (int j = d0 / 8; j < (d0 + per_pass) / 8; j += 2) {
            uint32_t v[16];
            if (my_tiles > 0) {
              tmem_ld16(to + 8 * j, v);
              tmem_wait_ld();
            } else {
#pragma unroll
              for (int k = 0; k < 16; k++) v[k] = 0u;
            }
            float o[16];
#pragma unroll
            for (int k = 0; k < 16; k++) o[k] = __uint_as_float(v[k]) * f0 * f1;
            if (spoiled && (j < 8 ? poison0 : poison1)) {
#pragma unroll
              for (int k = 0; k < 16; k++) o[k] = __uint_as_float(0x7fc00000u);
            }
            const float lo[8] = {o[0], o[2], o[1], o[3], o[8], o[10], o[9], o[11]};
            const float hi[8] = {o[4], o[6], o[5], o[7], o[12], o[14], o[13], o[15]};
            const int d = 64 * (j >> 3) + 4 * (j & 7) - d0;   // within the pass
            // 16-byte chunks of the row, rotated by the lane
            auto put = [&](int byte, uint4 x) {
              *reinterpret_cast<uint4 *>(stage + lane * 256 + ((byte + 16 * lane) & 255)) = x;
            };
            if (it.n_parts > 1) {
#pragma unroll
              for (int k = 0; k < 8; k += 4) {
                put(4 * (d + k), make_uint4(__float_as_uint(lo[k]), __float_as_uint(lo[k + 1]),
                                            __float_as_uint(lo[k + 2]), __float_as_uint(lo[k + 3])));
                put(4 * (d + 32 + k), make_uint4(__float_as_uint(hi[k]), __float_as_uint(hi[k + 1]),
                                                 __float_as_uint(hi[k + 2]), __float_as_uint(hi[k + 3])));
              }
            } else {
              put(2 * d, make_uint4(pack2<T>(lo[0], lo[1]), pack2<T>(lo[2], lo[3]), pack2<T>(lo[4], lo[5]),
                                    pack2<T>(lo[6], lo[7])));
              put(2 * d + 64, make_uint4(pack2<T>(hi[0], hi[1]), pack2<T>(hi[2], hi[3]), pack2<T>(hi[4], hi[5]),
                                         pack2<T>(hi[6], hi[7])));
            }
          }
          __syncwarp();
          // whole rows again: a lane's chunk of rows rr0, rr0 + rows per step, ...
          const bool record = it.n_parts > 1;
          const int cpr = record ? 16 : HD / 8;   // chunks of a row
          const int ch = lane & (cpr - 1), step = 32 / cpr, rr0 = lane / cpr;
          const int n_rows = it.rows - 32 * warp;   // of this warp (row tiles are 4 warps of 32 rows)
          float *po = a.part_o + part_row(a, it.slot, 32 * warp) * HD + d0 + 4 * ch;
          RowWalk row(a, it, a.out, 32 * warp + rr0, step);
          auto chunk = [&](int rr) {
            return *reinterpret_cast<const uint4 *>(stage + rr * 256 + ((16 * ch + 16 * rr) & 255));
          };
          if (record) {
#pragma unroll 4
            for (int rr = rr0; rr < min(32, n_rows); rr += step)
              *reinterpret_cast<uint4 *>(po + rr * HD) = chunk(rr);
          } else {
#pragma unroll 4
            for (int rr = rr0; rr < min(32, n_rows); rr += step) {
              T *p = reinterpret_cast<T *>(a.out.data) + row.at + 8 * ch;
              const uint4 y = chunk(rr);
              if (vec) {
                // 8-byte pieces: rows start on 4-element boundaries
                reinterpret_cast<uint2 *>(p)[0] = make_uint2(y.x, y.y);
                reinterpret_cast<uint2 *>(p)[1] = make_uint2(y.z, y.w);
              } else {
                const T *e8 = reinterpret_cast<const T *>(&y);
#pragma unroll
                for (int k = 0; k < 8; k++) p[k] = e8[k];
              }
              row.step();
            }
          }
          __syncwarp();
        }
      }
      if (it.n_parts > 1) {
        // warps that gave up leave their mark ahead of this barrier
        volatile int *said = reinterpret_cast<volatile int *>(smem + C::SLOT + 12);
        named_sync(1, kSoftWarps * 32);
        if (threadIdx.x == 0) *said = !*failed;
        named_sync(1, kSoftWarps * 32);
        if (*said && extend_arrive_last<kSoftWarps * 32>(a, it, reinterpret_cast<int *>(smem + C::SLOT + 8), 1))
          extend_merge<HD, T, kSoftWarps * 32>(a, it, vec, reinterpret_cast<float *>(smem + C::K),
                                               2 * kStages * C::TILE / 4, 1);
      }
      done += my_tiles;
      all_done += n_tiles;
      parts += my_tiles > 0;
      fence_before_sync();
      meet();
      fence_after_sync();
      if (*failed) break;
    }
    regs_down<kRegs>();
  }
  if (warp >= kSoftWarps) regs_up<kRegs>();   // given back by the softmax warps
  __syncthreads();
  if (warp == kMmaWarp) tmem_dealloc(tm, C::COLS);
}

// Registers per thread that the kernel was built with (0: unknown).
template <int HD, typename T>
int built_registers() {
  static std::atomic<int> known[64];   // per device
  int dev = 0;
  cudaGetDevice(&dev);
  int regs = known[dev & 63].load(std::memory_order_relaxed);
  if (regs) return regs;
  cudaFuncAttributes at;
  if (cudaFuncGetAttributes(&at, extend_umma_kernel<HD, T>) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  known[dev & 63].store(at.numRegs, std::memory_order_relaxed);
  return at.numRegs;
}

template <int HD, typename T>
int launch_one(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks, bool vec,
               cudaStream_t s) {
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
  fn<<<n_blocks, kThreads, C::SMEM, s>>>(a, b, runs, vec ? 1 : 0);
  return check_cuda(cudaGetLastError(), "extend_umma launch");
}

}  // namespace

thread_local int t_extend_registers = 0;

// The warpgroups trade the launch's registers, which have to add up: a compiler (or a
// debug build) that takes another number per thread leaves this kernel out.
bool extend_umma_usable(int head_dim, int dtype) {
  const int regs = t_extend_registers ? t_extend_registers
                   : head_dim == 128  ? (dtype == EAKV_F16 ? built_registers<128, __half>()
                                                           : built_registers<128, __nv_bfloat16>())
                                      : (dtype == EAKV_F16 ? built_registers<64, __half>()
                                                           : built_registers<64, __nv_bfloat16>());
  return regs == kRegs;
}

int extend_umma_launch(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks,
                       bool vec, cudaStream_t s) {
  if (a.geom.gpd == 2)
    return a.dtype == EAKV_F16 ? launch_one<128, __half>(a, b, runs, n_blocks, vec, s)
                               : launch_one<128, __nv_bfloat16>(a, b, runs, n_blocks, vec, s);
  return a.dtype == EAKV_F16 ? launch_one<64, __half>(a, b, runs, n_blocks, vec, s)
                             : launch_one<64, __nv_bfloat16>(a, b, runs, n_blocks, vec, s);
}

}  // namespace eakv

extern "C" int eakv_test_extend_registers(int n) {
  eakv::t_extend_registers = n > 0 ? n : 0;
  return EAKV_OK;
}
