// extend_mma.cu - attention of a few new tokens per cache over the Q4 pages,
// on the warp-level tensor-core instructions (mma.sync, f16 operands, f32
// sums): tiles of 8, 16 or 24 (token, query head) rows of one KV head.
//
// Mathematics. With a group's centred nibbles n' = n - 8 and b' = b + 8 s,
//   q.k = sum_g s_g (q_g . n'_g) + b'_g sum(q_g)
//   o  += sum_j (p_j s_j) n'_j + p_j b'_j                      (per group)
// n' is exact in f16, so only q and p s are rounded as operands. Centring
// matters on the V side: sum_j p_j s_j n_j of raw nibbles carries an offset of
// 7.5 quanta that p_j b_j takes out again, and over 10^4 positions the rest is
// hundreds of times smaller than the offset; of centred ones it is not.
// Every row of q is scaled by a power of two into [2^12, 2^13), of which the operands
// that meet nibbles held times 16 take a sixteenth: 16-bit q (8 or 11 bits) is then
// exact in f16 but for elements 2^-22 below the row's largest; f32 q becomes two
// f16 limbs (hi, x - hi: 22 bits of elements down to 2^-11 of the row's largest). p s
// is one f16 for 16-bit types (2^-12 of each term, below the output's own rounding)
// and two limbs for f32. Sums of scores, softmax and outputs are f32; the maximum moves
// lazily, from below a score to 8 above it (base 2), a whole number, so that p <= 1.
//
// Tiles. Both products are transposed, rows the n8 of the instructions: scores
// S^T[16 positions][8 rows] take K as A operand straight from its bytes (a 32-bit
// word holds dims d..d+3 and d+32..d+35; the pairs that one mask selects are (d,
// d+2) and (d+32, d+34), and the dims of a k-step are taken in that order on both
// sides), O^T[16 dims][8 rows] takes V as A operand from one transposed ldmatrix
// per group and 16 positions, and the weights as B operand by one transposition of
// 8 x 8 pairs (movmatrix). So a page is converted once for a tile, and a tile of few
// rows costs few products: with rows as the m16 one token of four heads behind each
// of 16 x 8192 positions took 71 us, transposed 55. Each warp takes whole pages in
// turn; the page ring, its waits and the split merge are those of the decode kernels.
//
// Bound: the chain of a step's dependent instructions (two to four warps per
// scheduler, as the registers allow), and the set-up and merge of an item, about 15
// us. 16 caches of 8192 positions (168 MB, 26 us at HBM's rate): 58 us for 8 rows,
// 81 for 16, 112 for 24.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "extend.cuh"

namespace eakv {
namespace {

// NT: tiles of eight rows per CTA.
template <int HD, int LIMBS, int NT>
struct XCfg {
  static constexpr int R = 8 * NT, PAIRS = (NT + 1) / 2, QR = 16 * PAIRS;   // rows, and as q's operands lie
  static constexpr int NG = HD / 64;
  static constexpr int NW = 4;
  static constexpr int THREADS = NW * 32;
  static constexpr int MINB = NT == 3 ? 2 : NT == 1 && HD == 64 ? 4 : 3;   // CTAs per SM
  // Positions of a lane per step (g + 8 j). A step's time is its chain of dependent
  // instructions: two of 16 positions side by side where the registers are there.
  static constexpr int J = NT == 1 ? 4 : 2;
  static constexpr int NIB = kPagePositions * NG * 32;
  static constexpr int PB = kPagePositions * NG * 40;
  static constexpr int NSTAGE = HD == 128 ? 5 : 8;              // pages in flight
  static constexpr int STAGE_BYTES = 2 * PB;
  static constexpr int RING = NSTAGE * STAGE_BYTES;
  static constexpr int OS = HD + 8;                             // floats from row to row of the warps' sums
  static constexpr int MERGE = NW * R * (OS + 2) * 4;
  static constexpr int MAIN = RING > MERGE ? RING : MERGE;
  static constexpr int QOFF = MAIN + 2 * NSTAGE * 8;            // q rows [QR][HD] f32
  // [QR] powers of two, [QR] score factors, [NG][QR] sums
  static constexpr int STATOFF = QOFF + QR * HD * 4;
  // K enters as 16 (64 + n), the offset taken off by the sums' start: four
  // operations per two pairs less than centring, and the sums run within
  // 64 sum |q| of zero, 2^-18 of it lost (one-limb types)
  static constexpr bool KRAW = LIMBS == 1;
  static constexpr int STARTOFF = STATOFF + QR * (2 + NG) * 4;  // [NG][QR][warp] starts
  static constexpr int MASKOFF = STARTOFF + QR * NG * NW * 4;   // RowMask [R]
  static constexpr int FRAGOFF = MASKOFF + QR * 32;             // [pair][step][limb][lane]
  static_assert(NW == 4, "a warp per step of a group");
  static constexpr int FRAGS = PAIRS * LIMBS * 4 * NG * 32 * 16;
  static constexpr int SMEM = FRAGOFF + FRAGS;
  static_assert(MAIN % 16 == 0 && FRAGOFF % 16 == 0 && sizeof(RowMask) <= 32, "alignment");
};

__device__ __forceinline__ uint32_t sub_f16x2(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
// Centred nibbles of bytes 0 and 2 as f16 pairs: low ones n - 8, high ones
// 16 (n - 8). A nibble in the low bits of 1024.0 (0x6400) is 1024 + n (+ 16 n in
// place), and 1032 (1024 + 128) comes off exactly.
__device__ __forceinline__ uint32_t nib_lo(uint32_t w) {
  return sub_f16x2(and_or(w, 0x000F000Fu, 0x64006400u), 0x64086408u);
}
__device__ __forceinline__ uint32_t nib_hi(uint32_t w) {
  return sub_f16x2(and_or(w, 0x00F000F0u, 0x64006400u), 0x64806480u);
}

// High nibbles of bytes 0 and 2 with the offset left in: 1024 + 16 n = 16 (64 + n).
__device__ __forceinline__ uint32_t raw_hi(uint32_t w) { return and_or(w, 0x00F000F0u, 0x64006400u); }

// x - f16(x) of both halves, as f16
__device__ __forceinline__ uint32_t pack_rest(float x0, float x1, uint32_t hi) {
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
  return pack_f16(x0 - b.x, x1 - b.y);
}

__device__ __forceinline__ void mma(float *d, const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// The 8 x 8 matrix of f16 pairs that the warp's words hold, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// Units of p s. The products of weight and scale of a row and group are held times a
// power of two that takes the largest of them to [1, 2) when it is set, and keeps it from
// kRefLeast (above, two f16 limbs hold 22 bits) to below kRefMost later. A row's two
// powers share a word, as the upper halves of their f32. kPowerMost, the exponent field
// of the largest power (its inverse is a normal number too), is the first.
constexpr int kPowerMost = 253;
constexpr float kRefMost = 16384.0f, kRefLeast = 0.125f;
template <int NG> __device__ __forceinline__ void set_power(uint32_t &word, int group, int field) {
  if (NG == 1) word = (uint32_t)field << 23;
  else if (group == 0) word = (word & 0xFFFF0000u) | (uint32_t)field << 7;
  else word = (word & 0xFFFFu) | (uint32_t)field << 23;
}
// 2^e, 0 below the normal range
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)max(127 + e, 0) << 23); }
template <int NG> __device__ __forceinline__ float ref_power(uint32_t word, int group) {
  return __uint_as_float(group + 1 < NG ? word << 16 : word & 0xFFFF0000u);
}

// Whether a group with a scale of 1 has only zero nibbles: the quantizer's form of 64
// equal values. Its offset b + 8 s would carry the scale of 1 into sums of values of any
// size (zero vectors among V of 1e-3: outputs off by several times their size), so such
// groups get a scale of 0 in the copy of their page.
__device__ __forceinline__ bool constant_group(const uint8_t *page, int slot) {
  const uint4 x = *reinterpret_cast<const uint4 *>(page + slot * 32);
  const uint4 y = *reinterpret_cast<const uint4 *>(page + slot * 32 + 16);
  return ((x.x | x.y | x.z | x.w) | (y.x | y.y | y.z | y.w)) == 0;
}

// Out of line: between two parts, with few registers to keep over the call.
__device__ __noinline__ void step_walk(ExtWalk &walk, const ExtendArgs &a, const ExtendBatch &batch, int p) {
  walk.next(a, batch, p);
}
__device__ __noinline__ void abandon_walk(ExtWalk &walk, const ExtendArgs &a, const ExtendBatch &batch, int p) {
  walk.abandon(a, batch, p);
}

template <int HD, int LIMBS, int NT, typename T>
__global__ void __launch_bounds__(XCfg<HD, LIMBS, NT>::THREADS, XCfg<HD, LIMBS, NT>::MINB)
extend_mma_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExtendBatch batch,
                  const __grid_constant__ ExtendRuns runs, const int vec) {
  using C = XCfg<HD, LIMBS, NT>;
  constexpr int NG = C::NG, R = C::R, QR = C::QR, J = C::J;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int last_part;
  __shared__ ExtWalk walk;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::MAIN);
  float *q_s = reinterpret_cast<float *>(smem + C::QOFF);
  float *up_s = reinterpret_cast<float *>(smem + C::STATOFF), *fac_s = up_s + QR, *sum_s = fac_s + QR;
  RowMask *mask_s = reinterpret_cast<RowMask *>(smem + C::MASKOFF);
  float *start_s = reinterpret_cast<float *>(smem + C::STARTOFF);
  uint4 *frag_s = reinterpret_cast<uint4 *>(smem + C::FRAGOFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::NSTAGE; s++) {
      mbar_init(smem_u32(&bars[s]), 1);
      reinterpret_cast<int *>(&bars[C::NSTAGE])[s] = 0;               // release count
      reinterpret_cast<int *>(&bars[C::NSTAGE])[C::NSTAGE + s] = -1;  // last page requested
    }
    fence_mbar_init();
    walk.begin(a, batch, runs);
  }
  __syncthreads();
  int *last_req = reinterpret_cast<int *>(&bars[C::NSTAGE]) + C::NSTAGE;
  int done = 0;   // pages of the parts before: stages and phases go on
  for (int part = 0;; part++) {
    const ExtItem &it = walk.item[part & 1];
    if (it.state <= 0) {
      if (threadIdx.x == 0 && it.state < 0) abandon_walk(walk, a, batch, part);
      return;
    }
    const uint8_t *kpages = it.base + page_index(a.geom, a.layer, 0, it.h, 0) * C::PB;
    const uint8_t *vpages = kpages + (size_t)a.geom.n_heads * a.geom.n_pages * C::PB;
    auto issue = [&](int i) {
      if (i == a.test_stall - 1) return;   // test hook: this stage's wait runs out
      const int st = (done + i) % C::NSTAGE;
      const uint32_t full = smem_u32(&bars[st]);
      mbar_arrive_expect_tx(full, 2 * C::PB);
      const uint32_t dst = smem_u32(smem + st * C::STAGE_BYTES);
      bulk_g2s(dst, kpages + (size_t)(it.pg0 + i) * C::PB, C::PB, full);
      bulk_g2s(dst + C::PB, vpages + (size_t)(it.pg0 + i) * C::PB, C::PB, full);
      publish_requested(&last_req[st], done + i);
    };
    // ---- the tile's q rows: f32 in shared memory, row maxima and group sums ------
    // (all loads, then the first pages' requests, then the stores)
    if (threadIdx.x < R) {
      const int r = it.row0 + threadIdx.x;
      RowMask m = row_mask(a, it, r);
      if (a.depth && a.window > 0) depth_window(a, it, r, m);
      mask_s[threadIdx.x] = m;
    }
    {
      constexpr int LOADS = QR * (HD / 4) / C::THREADS, STEP = C::THREADS / (HD / 4);
      const int r0 = threadIdx.x / (HD / 4), d = 4 * (threadIdx.x % (HD / 4));
      float v[LOADS][4];
      auto load = [&](auto vec_tag) {
#pragma unroll
        for (int k = 0; k < LOADS; k++) {
          const int row = it.row0 + r0 + STEP * k, tok = row / a.G;
          v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.0f;
          if (r0 + STEP * k < it.rows)
            load4<T, decltype(vec_tag)::value>(
                reinterpret_cast<const T *>(a.q.data) + (long long)(it.tok0 + tok) * a.q.token_stride +
                    (long long)(it.h * a.G + row - tok * a.G) * a.q.head_stride + d, v[k]);
        }
      };
      if (vec) load(std::true_type{});
      else load(std::false_type{});
      if (threadIdx.x == 0)
        for (int i = 0; i < it.npages && i < C::NSTAGE; i++) issue(i);
#pragma unroll
      for (int k = 0; k < LOADS; k++)
        *reinterpret_cast<float4 *>(q_s + (r0 + STEP * k) * HD + d) =
            make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
    }
    __syncthreads();
    // a warp's rows together, step by step
    {
      constexpr int RW = QR / C::NW;
      float mx[RW], sm[RW][NG];
      bool bad[RW];
#pragma unroll
      for (int i = 0; i < RW; i++) {
        const float *p = q_s + (warp + C::NW * i) * HD + lane;
        mx[i] = 0.0f;
        bad[i] = false;
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          const float v0 = p[64 * gg], v1 = p[64 * gg + 32];
          mx[i] = fmaxf(mx[i], fmaxf(fabsf(v0), fabsf(v1)));
          bad[i] = bad[i] || v0 != v0 || v1 != v1;
          sm[i][gg] = v0 + v1;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < RW; i++) {
          mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
#pragma unroll
          for (int gg = 0; gg < NG; gg++) sm[i][gg] += __shfl_xor_sync(0xffffffffu, sm[i][gg], o);
        }
#pragma unroll
      for (int i = 0; i < RW; i++) {
        const bool fine = !__any_sync(0xffffffffu, bad[i]) && mx[i] <= 3.0e38f;
        const int r = warp + C::NW * i;
        int e = 0;
        frexpf(mx[i] > 0.0f && fine ? mx[i] : 1.0f, &e);          // in [2^(e-1), 2^e)
        const int qe = max(min(13 - e, 126), -126);
        if (lane == 0) {
          const float up = fine ? __uint_as_float((uint32_t)(127 + qe) << 23) : 0.0f;
          up_s[r] = up;
          // a row with an infinity or NaN in q has NaN scores
          fac_s[r] = fine ? a.scale_log2 * __uint_as_float((uint32_t)(127 - qe) << 23)
                          : __uint_as_float(0x7fc00000u);
#pragma unroll
          for (int gg = 0; gg < NG; gg++) sum_s[gg * QR + r] = fine ? sm[i][gg] * up : 0.0f;
        }
      }
    }
    __syncthreads();
    // q's operands: for k-step s = (word j, byte parity par) of group gg the dims
    // d = 64 gg + 8c + 4j + par and d + 2 (low nibbles), d + 32 and d + 34 (high
    // nibbles, held times 16) of rows g, g + 8 of a pair of tiles; each warp one step
    // of every group
#pragma unroll
    for (int pr = 0; pr < C::PAIRS; pr++) {
      const float up[2] = {up_s[16 * pr + g], up_s[16 * pr + g + 8]};
#pragma unroll
      for (int gg = 0; gg < NG; gg++) {
        const int s = 4 * gg + warp;
        const int d = 64 * gg + 8 * c + 4 * ((s >> 1) & 1) + (s & 1);
        uint32_t hi[4], lo[4];
        float start[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 4; k++) {   // k & 1: row, k >> 1: high nibbles
          const int r = k & 1;
          const float *p = q_s + (16 * pr + g + 8 * r) * HD + d + 32 * (k >> 1);
          const float f = up[r] * (C::KRAW || (k >> 1) ? 0.0625f : 1.0f);
          const float x0 = up[r] == 0.0f ? 0.0f : p[0] * f;   // inf * 0
          const float x1 = up[r] == 0.0f ? 0.0f : p[2] * f;
          hi[k] = pack_f16(x0, x1);
          if (C::KRAW) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi[k]));
            start[r] -= 1024.0f * (h.x + h.y);
          }
          lo[k] = LIMBS == 2 ? pack_rest(x0, x1, hi[k]) : 0u;
        }
        uint4 *f = frag_s + (pr * 4 * NG + s) * LIMBS * 32 + lane;
        f[0] = make_uint4(hi[0], hi[2], hi[1], hi[3]);
        if (LIMBS == 2) f[32] = make_uint4(lo[0], lo[2], lo[1], lo[3]);
        if (C::KRAW) {
#pragma unroll
          for (int r = 0; r < 2; r++) {
            start[r] += __shfl_xor_sync(0xffffffffu, start[r], 1);
            start[r] += __shfl_xor_sync(0xffffffffu, start[r], 2);
            if (c == 0) start_s[(gg * QR + 16 * pr + g + 8 * r) * C::NW + warp] = start[r];
          }
        }
      }
    }
    __syncthreads();
    // rows 8 n + 2 c + e of this lane
    float rowfac[NT][2], qsum[NT][2][NG], kstart[NT][2][NG];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int r = 8 * n + 2 * c + e;
        rowfac[n][e] = fac_s[r];
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          qsum[n][e][gg] = sum_s[gg * QR + r];
          const float4 k4 = *reinterpret_cast<const float4 *>(start_s + (gg * QR + r) * C::NW);
          kstart[n][e][gg] = (k4.x + k4.y) + (k4.z + k4.w);
        }
      }

    // O transposed: [group][dims 16w + 2g + parity, low and high nibbles][row tile]
    float o[NG][4][NT][4];
#pragma unroll
    for (int gg = 0; gg < NG; gg++)
#pragma unroll
      for (int m = 0; m < 4; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) o[gg][m][n][k] = 0.0f;
    float m_run[NT][2], l_run[NT][2], pb[NT][2][NG];
    // The products p s, f16 operands, are held times a power of two of the row's and
    // group's own (vref), and the group's o with them; p itself and the sums l and p b' are
    // not. What sets it is the largest p s that the row has attended, not the largest s: a
    // weight near 1 on V of zeros, or on V much smaller than the rest, leaves the others their
    // bits. (One power for both groups lost bits of the smaller: with one 2^-16 of the
    // other f32 outputs were off by 2^-9.) When the maximum moves, p shrinks by a power of
    // two, and o with it, or if what moved it has hardly any V, vref grows by it; when p s comes
    // to kRefMost in these units, vref and o shrink. It starts at the largest: denormal
    // scales need nothing of their own.
    uint32_t vref[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        m_run[n][e] = -INFINITY;
        l_run[n][e] = 0.0f;
        vref[n][e] = (uint32_t)(kPowerMost << 7) * 0x10001u;
#pragma unroll
        for (int gg = 0; gg < NG; gg++) pb[n][e][gg] = 0.0f;
      }

    // (scale, b + 8 scale when centred) of the lane's positions p0 + g + 8 j
    auto scales = [&](const uint8_t *sb, int p0, bool centred, float (&s)[J][NG], float (&b)[J][NG]) {
#pragma unroll
      for (int j = 0; j < J; j++) {
        const int tp = p0 + g + 8 * j;
        if constexpr (NG == 2) {
          const float4 v4 = *reinterpret_cast<const float4 *>(sb + tp * 16);
          s[j][0] = v4.x; b[j][0] = v4.y; s[j][NG - 1] = v4.z; b[j][NG - 1] = v4.w;
        } else {
          const float2 v2 = *reinterpret_cast<const float2 *>(sb + tp * 8);
          s[j][0] = v2.x; b[j][0] = v2.y;
        }
#pragma unroll
        for (int gg = 0; gg < NG; gg++)
          if (centred) b[j][gg] = fmaf(8.0f, s[j][gg], b[j][gg]);
      }
    };

    float page_s[NG];   // largest finite V scale of each group of the page (full pages)
    auto step = [&](auto full_tag, const uint8_t *ks, int page_pos0, int p0) {
      constexpr bool FULL = decltype(full_tag)::value;
      const uint8_t *vsm = ks + C::PB;
      bool on[NT][2][J];   // [row tile][row][position]
      if (!FULL) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const RowMask m = mask_s[8 * n + 2 * c + e];
#pragma unroll
            for (int j = 0; j < J; j++) on[n][e][j] = m.attends(page_pos0 + p0 + g + 8 * j);
          }
      }
      // ---- scores, transposed: [position g + 8 j][row 2 c + e] ------------------
      float sc[NT][2][J];
      {
        float sk[J][NG], bk[J][NG], dk[NT][NG][2 * J];   // dk: of 16 positions after the other
        scales(ks + C::NIB, p0, !C::KRAW, sk, bk);
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          uint2 wv[J];
#pragma unroll
          for (int j = 0; j < J; j++)
            wv[j] = *reinterpret_cast<const uint2 *>(ks + (p0 + 8 * j + g) * (HD / 2) + 8 * c + 32 * gg);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int k = 0; k < 2 * J; k++) dk[n][gg][k] = C::KRAW ? kstart[n][k & 1][gg] : 0.0f;
#pragma unroll
          for (int s = 0; s < 4; s++) {
            uint32_t af[J / 2][4];
#pragma unroll
            for (int j = 0; j < J; j++) {
              const uint32_t w = (s >> 1) ? wv[j].y : wv[j].x;
              const uint32_t y = (s & 1) ? w >> 8 : w;
              af[j >> 1][j & 1] = C::KRAW ? raw_hi((s & 1) ? w >> 4 : w << 4) : nib_lo(y);
              af[j >> 1][2 + (j & 1)] = C::KRAW ? raw_hi(y) : nib_hi(y);
            }
#pragma unroll
            for (int pr = 0; pr < C::PAIRS; pr++)
#pragma unroll
              for (int l = 0; l < LIMBS; l++) {
                const uint4 f = frag_s[((pr * 4 * NG + 4 * gg + s) * LIMBS + l) * 32 + lane];
#pragma unroll
                for (int u = 0; u < J / 2; u++) {
                  mma(dk[2 * pr][gg] + 4 * u, af[u], f.x, f.y);
                  if (2 * pr + 1 < NT) mma(dk[2 * pr + 1 < NT ? 2 * pr + 1 : 0][gg] + 4 * u, af[u], f.z, f.w);
                }
              }
          }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++)
#pragma unroll
            for (int j = 0; j < J; j++) {
              float u = 0.0f;
#pragma unroll
              for (int gg = 0; gg < NG; gg++) {
                u = fmaf(dk[n][gg][2 * j + e], sk[j][gg], u);
                u = fmaf(qsum[n][e][gg], bk[j][gg], u);
              }
              u *= rowfac[n][e];
              sc[n][e][j] = (FULL || on[n][e][j]) ? u : -INFINITY;
            }
      }
      float sv[J][NG], bv[J][NG];
      scales(vsm + C::NIB, p0, true, sv, bv);
      // ---- online softmax, base 2, lazy maximum -----------------------------------
      // (Scales are negative only in damaged files; NaN is passed over.)
      bool move = false;
      float lm[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          lm[n][e] = sc[n][e][0];
#pragma unroll
          for (int j = 1; j < J; j++) lm[n][e] = fmaxf(lm[n][e], sc[n][e][j]);
          move = move || lm[n][e] > m_run[n][e];
#pragma unroll
          for (int gg = 0; gg < NG; gg++) {   // p is at most 1
            float s = FULL ? page_s[gg] : 0.0f;
#pragma unroll
            for (int j = 0; j < J; j++)
              if (!FULL && on[n][e][j]) s = fmaxf(s, fabsf(sv[j][gg]));
            move = move || s * ref_power<NG>(vref[n][e], gg) >= kRefMost;
          }
        }
      if (__any_sync(0xffffffffu, move)) {
        // largest p s of the lane's positions, without infinite scales
        auto most = [&](int n, int e, int gg) {
          const float m = m_run[n][e] == -INFINITY ? 0.0f : m_run[n][e];
          float y = 0.0f;
#pragma unroll
          for (int j = 0; j < J; j++) {
            const float s = fabsf(sv[j][gg]);
            if ((FULL || on[n][e][j]) && s < INFINITY) y = fmaxf(y, ex2(sc[n][e][j] - m) * s);
          }
          return y;
        };
        auto scale_out = [&](int gg, int n, int e, float f) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            o[gg][k][n][e] *= f;
            o[gg][k][n][2 + e] *= f;
          }
        };
        // per row and group: p s too large for its units (lower bits), large enough (upper)
        static_assert(2 * NT * NG <= 16, "room for the bits");
        uint32_t bits = 0;
        int d[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            float t = lm[n][e];
#pragma unroll
            for (int b = 4; b < 32; b <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, b));
            d[n][e] = 0;
            if (t > m_run[n][e]) {
              t = ceilf(t) + 8.0f;
              d[n][e] = (int)fminf(t - m_run[n][e], 1000.0f);   // from -inf: sums of nothing
              m_run[n][e] = t;
              l_run[n][e] *= pow2i(-d[n][e]);
            }
#pragma unroll
            for (int gg = 0; gg < NG; gg++) {
              const float v = most(n, e, gg) * ref_power<NG>(vref[n][e], gg);
              const int k = (2 * n + e) * NG + gg;
              bits |= (v >= kRefMost ? 1u << k : 0u) | (v >= kRefLeast ? 0x10000u << k : 0u);
            }
          }
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, b);
        bool again = (bits & 0xFFFFu) != 0;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 2; e++)
            if (d[n][e] > 0) {
#pragma unroll
              for (int gg = 0; gg < NG; gg++) {
                const float alpha = pow2i(-d[n][e]);
                pb[n][e][gg] *= alpha;
                if (bits & (0x10000u << ((2 * n + e) * NG + gg))) {
                  scale_out(gg, n, e, alpha);
                } else {   // the new largest weight stands on hardly any V
                  const int was = (int)(__float_as_uint(ref_power<NG>(vref[n][e], gg)) >> 23);
                  const int now = min(was + d[n][e], kPowerMost);
                  set_power<NG>(vref[n][e], gg, now);
                  scale_out(gg, n, e, pow2i(now - was - d[n][e]));
                  again = true;
                }
              }
            }
        if (__any_sync(0xffffffffu, again)) {
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
              for (int gg = 0; gg < NG; gg++) {
                float y = most(n, e, gg);
#pragma unroll
                for (int b = 4; b < 32; b <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, b));
                const float f = ref_power<NG>(vref[n][e], gg);
                if (y * f >= kRefMost) {
                  const int was = (int)(__float_as_uint(f) >> 23);
                  const int now = min(max(254 - (int)(__float_as_uint(y) >> 23), 1), kPowerMost);
                  set_power<NG>(vref[n][e], gg, now);
                  scale_out(gg, n, e, pow2i(now - was));
                }
              }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float m = m_run[n][e] == -INFINITY ? 0.0f : m_run[n][e];
#pragma unroll
          for (int j = 0; j < J; j++) {
            sc[n][e][j] = ex2(sc[n][e][j] - m);   // the weights from here on
            l_run[n][e] += sc[n][e][j];
          }
        }
      // ---- outputs -------------------------------------------------------------
#pragma unroll
      for (int gg = 0; gg < NG; gg++) {
        uint32_t bh[NT][J], bl[NT][J];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int j = 0; j < J; j++) {
            float x[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
              // what is not attended adds nothing, whatever its scale and bias are
              x[e] = (FULL || on[n][e][j]) ? sc[n][e][j] * sv[j][gg] * ref_power<NG>(vref[n][e], gg) : 0.0f;
              if (FULL || on[n][e][j]) pb[n][e][gg] = fmaf(sc[n][e][j], bv[j][gg], pb[n][e][gg]);
            }
            const uint32_t h = pack_f16(x[0], x[1]);
            bh[n][j] = transpose8(h);
            bl[n][j] = LIMBS == 2 ? transpose8(pack_rest(x[0], x[1], h)) : 0u;
          }
        // V bytes: lane (g, c) receives bytes 16w + 2g, + 1 of positions 2c, 2c+1
        // (x[2w]) and 2c+8, 2c+9 (x[2w+1])
#pragma unroll
        for (int u = 0; u < J / 2; u++) {
          uint32_t x[4];
          {
            const int t = lane >> 3, r = lane & 7;
            const int at = p0 + 16 * u + 8 * (t & 1) + r;
            ldsm_x4_trans(x, smem_u32(vsm + at * (HD / 2) + 32 * gg + 16 * (t >> 1)));
          }
#pragma unroll
          for (int m = 0; m < 4; m++) {   // m = 2w + parity
            const int w = m >> 1;
            const uint32_t y0 = (m & 1) ? x[2 * w] >> 8 : x[2 * w];
            const uint32_t y1 = (m & 1) ? x[2 * w + 1] >> 8 : x[2 * w + 1];
            const uint32_t af[4] = {nib_lo(y0), nib_hi(y0), nib_lo(y1), nib_hi(y1)};
#pragma unroll
            for (int n = 0; n < NT; n++) {
              mma(o[gg][m][n], af, bh[n][2 * u], bh[n][2 * u + 1]);
              if constexpr (LIMBS == 2) mma(o[gg][m][n], af, bl[n][2 * u], bl[n][2 * u + 1]);
            }
          }
        }
      }
    };

    bool ok = true;
    for (int i = warp; i < it.npages; i += C::NW) {
      const int st = (done + i) % C::NSTAGE;
      if (!wait_requested(&last_req[st], done + i, a.wait_budget) ||
          !mbar_wait(smem_u32(&bars[st]), ((done + i) / C::NSTAGE) & 1, a.wait_budget)) {
        atomicOr(a.status, kStatusWaitTimeout);
        ok = false;
        break;
      }
      uint8_t *ks = smem + st * C::STAGE_BYTES;
      const int page_pos0 = (it.pg0 + i) * kPagePositions;
      const bool full = page_pos0 >= it.all_lo && page_pos0 + kPagePositions <= it.all_hi;
      bool one = false;
#pragma unroll
      for (int k = 0; k < 4 * NG; k++)   // K, then V
        one = one || *reinterpret_cast<const float *>(ks + (k / (2 * NG)) * C::PB + C::NIB +
                                                      8 * (lane + 32 * (k % (2 * NG)))) == 1.0f;
      if (__any_sync(0xffffffffu, one)) {   // groups of equal values: this warp alone has the page
        for (int x = lane; x < 2 * kPagePositions * NG; x += 32) {
          uint8_t *page = ks + x / (kPagePositions * NG) * C::PB;
          float *s = reinterpret_cast<float *>(page + C::NIB + 8 * (x % (kPagePositions * NG)));
          if (*s == 1.0f && constant_group(page, x % (kPagePositions * NG))) *s = 0.0f;
        }
        fence_proxy_async_smem();   // ahead of the copy that fills the stage next
        __syncwarp();
      }
      if (full) {
        // finite scales only: what an infinite one reaches is NaN anyway
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < 2 * NG; k++) {   // with two groups a lane's are of group lane % 2
          const uint32_t b =
              *reinterpret_cast<const uint32_t *>(ks + C::PB + C::NIB + 8 * (lane + 32 * k)) & 0x7fffffffu;
          if (b < 0x7f800000u) most = max(most, b);
        }
#pragma unroll
        for (int gg = 0; gg < NG; gg++)
          page_s[gg] = __uint_as_float(__reduce_max_sync(0xffffffffu, lane % NG == gg ? most : 0u));
#pragma unroll 1
        for (int p0 = 0; p0 < kPagePositions; p0 += 8 * J) step(std::true_type{}, ks, page_pos0, p0);
      } else {
#pragma unroll 1
        for (int p0 = 0; p0 < kPagePositions; p0 += 8 * J) step(std::false_type{}, ks, page_pos0, p0);
      }
      __syncwarp();
      if (lane == 0 && stage_release_last(reinterpret_cast<int *>(&bars[C::NSTAGE]) + st, 1) &&
          i + C::NSTAGE < it.npages)
        issue(i + C::NSTAGE);
    }
    if (!__syncthreads_and(ok)) {
      if (threadIdx.x == 0) {
        drain_stages(bars, last_req, C::NSTAGE, a.wait_budget);
        abandon_walk(walk, a, batch, part);
      }
      return;
    }
    if (threadIdx.x == 0 && !stages_idle(bars, last_req, C::NSTAGE)) {
      atomicOr(a.status, kStatusLateCopy);
      drain_stages(bars, last_req, C::NSTAGE, a.wait_budget);
    }

    // ---- the warps' sums meet in the (now idle) ring ---------------------------------
    __syncthreads();
    float *mw = reinterpret_cast<float *>(smem);   // [NW][R]
    float *lw = mw + C::NW * R;
    float *ow = lw + C::NW * R;                    // [NW][R][OS]
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) {
          l_run[n][e] += __shfl_xor_sync(0xffffffffu, l_run[n][e], b);
#pragma unroll
          for (int gg = 0; gg < NG; gg++) pb[n][e][gg] += __shfl_xor_sync(0xffffffffu, pb[n][e][gg], b);
        }
        const int row = warp * R + 8 * n + 2 * c + e;
        if (g == 0) {
          mw[row] = m_run[n][e];
          lw[row] = l_run[n][e];
        }
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          const float vs = __uint_as_float((254u << 23) - __float_as_uint(ref_power<NG>(vref[n][e], gg)));
#pragma unroll
          for (int w = 0; w < 2; w++)
#pragma unroll
            for (int hi = 0; hi < 2; hi++) {
              const float f = hi ? vs * 0.0625f : vs, b = pb[n][e][gg];
              *reinterpret_cast<float2 *>(ow + row * C::OS + 64 * gg + 32 * hi + 16 * w + 2 * g) =
                  make_float2(fmaf(o[gg][2 * w][n][2 * hi + e], f, b),
                              fmaf(o[gg][2 * w + 1][n][2 * hi + e], f, b));
            }
        }
      }
    __syncthreads();
    for (int x = threadIdx.x; x < it.rows * (HD / 4); x += C::THREADS) {
      const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < C::NW; w++) M = fmaxf(M, mw[w * R + r]);
      float O[4] = {0.0f, 0.0f, 0.0f, 0.0f}, L = 0.0f;
#pragma unroll
      for (int w = 0; w < C::NW; w++) {
        const float f = part_weight(mw[w * R + r], M);
        const float4 v = *reinterpret_cast<const float4 *>(ow + (w * R + r) * C::OS + d);
        L = fmaf(f, lw[w * R + r], L);
        O[0] = fmaf(f, v.x, O[0]);
        O[1] = fmaf(f, v.y, O[1]);
        O[2] = fmaf(f, v.z, O[2]);
        O[3] = fmaf(f, v.w, O[3]);
      }
      if (it.n_parts == 1) {
        extend_store<T>(a, it, r, d, O, M, L, vec);
      } else {
        const size_t pr = part_row(a, it.slot, r);
        *reinterpret_cast<float4 *>(a.part_o + pr * HD + d) = make_float4(O[0], O[1], O[2], O[3]);
        if (d == 0) {
          a.part_m[pr] = M;
          a.part_l[pr] = L;
        }
      }
    }
    if (it.n_parts > 1 && extend_arrive_last<C::THREADS>(a, it, &last_part, 1))
      extend_merge<HD, T, C::THREADS>(a, it, vec, reinterpret_cast<float *>(smem), C::MAIN / 4, 1);
    // the ring takes copies again
    done += it.npages;
    fence_proxy_async_smem();
    if (threadIdx.x == 0) step_walk(walk, a, batch, part + 1);
    __syncthreads();
  }
}

template <int HD, int LIMBS, int NT, typename T>
int resident_one() {
  using C = XCfg<HD, LIMBS, NT>;
  static std::atomic<int> cached[64];
  int dev = 0;
  cudaGetDevice(&dev);
  const int hit = cached[dev & 63].load(std::memory_order_relaxed);
  if (hit) return hit;
  auto fn = extend_mma_kernel<HD, LIMBS, NT, T>;
  if (check_cuda(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM),
                 "extend: smem attribute"))
    return 0;
  int per_sm = 1;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, C::THREADS, C::SMEM);
  if (per_sm < 1) per_sm = 1;
  cached[dev & 63].store(per_sm, std::memory_order_relaxed);
  return per_sm;
}

template <int HD, int LIMBS, int NT, typename T>
int launch_one(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks, bool vec,
               cudaStream_t s) {
  using C = XCfg<HD, LIMBS, NT>;
  extend_mma_kernel<HD, LIMBS, NT, T><<<n_blocks, C::THREADS, C::SMEM, s>>>(a, b, runs, vec ? 1 : 0);
  return check_cuda(cudaGetLastError(), "extend_mma launch");
}

// f(launch or resident functions of the instance that serves the arguments)
template <int HD, typename T, typename F>
int pick_rows(int rows, F f) {
  if (rows == 8) return f.template operator()<HD, 1, 1, T>();
  if (rows == 16) return f.template operator()<HD, 1, 2, T>();
  return f.template operator()<HD, 1, 3, T>();
}
template <int HD, typename F>
int pick(int dtype, int rows, F f) {
  if (dtype == EAKV_F32) return f.template operator()<HD, 2, 1, float>();
  if (dtype == EAKV_F16) return pick_rows<HD, __half>(rows, f);
  return pick_rows<HD, __nv_bfloat16>(rows, f);
}

struct Resident {
  template <int HD, int LIMBS, int NT, typename T> int operator()() const {
    return resident_one<HD, LIMBS, NT, T>();
  }
};
struct Launch {
  const ExtendArgs &a;
  const ExtendBatch &b;
  const ExtendRuns &runs;
  int n_blocks;
  bool vec;
  cudaStream_t s;
  template <int HD, int LIMBS, int NT, typename T> int operator()() const {
    return launch_one<HD, LIMBS, NT, T>(a, b, runs, n_blocks, vec, s);
  }
};

}  // namespace

// CTAs per SM of the kernel for this shape on the current device (0: error).
// Sets the kernel's shared-memory limit, so it comes before the launch.
int extend_mma_resident(int head_dim, int dtype, int tile_rows) {
  return head_dim == 128 ? pick<128>(dtype, tile_rows, Resident{}) : pick<64>(dtype, tile_rows, Resident{});
}

int extend_mma_launch(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks,
                      bool vec, cudaStream_t s) {
  const Launch f{a, b, runs, n_blocks, vec, s};
  return a.geom.gpd == 2 ? pick<128>(a.dtype, a.tile_rows, f) : pick<64>(a.dtype, a.tile_rows, f);
}

}  // namespace eakv
