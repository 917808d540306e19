// extend_mma.cu - attention of a few new tokens per cache over the Q4 pages,
// on the warp-level tensor-core instructions (mma.sync, f16 operands, f32
// sums): tiles of 16 (token, query head) rows of one KV head.
//
// Mathematics. With a group's centred nibbles n' = n - 8 and b' = b + 8 s,
//   q.k = sum_g s_g (q_g . n'_g) + b'_g sum(q_g)
//   o  += sum_j (p_j s_j) n'_j + p_j b'_j                      (per group)
// n' is exact in f16, so only q and p s are rounded as operands. Centring
// matters on the V side: sum_j p_j s_j n_j of raw nibbles carries an offset of
// 7.5 quanta that p_j b_j takes out again, and over 10^4 positions the rest is
// hundreds of times smaller than the offset; of centred ones it is not.
// Every row of q is scaled by a power of two into [16, 32): 16-bit q (8 or 11
// bits) is then exact in f16 but for elements 2^-18 below the row's largest;
// f32 q becomes two f16 limbs (hi, x - hi: 22 bits). p s is one f16 for 16-bit
// types (2^-12 of each term, below the output's own rounding) and two limbs
// for f32. Sums of scores, softmax and outputs are f32; the maximum moves
// lazily, when a score passes it by more than 8 (base 2), so p <= 256.
//
// Tiles. Rows are the m16 of both products, so a page is converted once for
// 16 rows: scores S[16 rows][8 positions] take K as B operand straight from
// its bytes (a 32-bit word holds dims d..d+3 and d+32..d+35; the pairs that
// one mask selects are (d, d+2) and (d+32, d+34), and the dims of a k-step are
// taken in that order on both sides), the score fragments are, pair by pair,
// the A fragments of the output product, and V comes as B operand from one
// transposed ldmatrix per group and 16 positions. Each warp takes whole pages
// in turn; the page ring, its waits and the split merge are those of the
// decode kernels.
//
// Bound: HBM for up to 16 rows (about 21 instructions per KV position of a
// KV head), instruction issue from there on: every further tile of 16 rows
// repeats the conversion.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "extend.cuh"

namespace eakv {
namespace {

template <int HD, int LIMBS>
struct XCfg {
  static constexpr int R = kExtendMmaRows;
  static constexpr int NG = HD / 64;
  static constexpr int NW = 4;
  static constexpr int THREADS = NW * 32;
  static constexpr int MINB = 3;                                // CTAs per SM
  static constexpr int NIB = kPagePositions * NG * 32;
  static constexpr int PB = kPagePositions * NG * 40;
  static constexpr int NSTAGE = HD == 128 ? 5 : 8;              // pages in flight
  static constexpr int STAGE_BYTES = 2 * PB;
  static constexpr int RING = NSTAGE * STAGE_BYTES;
  static constexpr int MERGE = NW * R * (HD + 2) * 4;
  static constexpr int MAIN = RING > MERGE ? RING : MERGE;
  static constexpr int QOFF = MAIN + 2 * NSTAGE * 8;            // q rows [R][HD] f32
  static constexpr int STATOFF = QOFF + R * HD * 4;             // [R] max|q|, [R][NG] sums
  // K enters as 16 (64 + n), the offset taken off by the sums' start: four
  // operations per two pairs less than centring, and the sums run within
  // 64 sum |q| of zero, 2^-18 of it lost (one-limb types)
  static constexpr bool KRAW = LIMBS == 1;
  static constexpr int STARTOFF = STATOFF + R * (1 + NG) * 4;   // [R][NG][warp] starts
  static constexpr int FRAGOFF = STARTOFF + R * NG * NW * 4;    // [step][limb][lane]
  static_assert(NW == 4, "a warp per step of a group");
  static constexpr int FRAGS = LIMBS * 4 * NG * 32 * 16;
  static constexpr int SMEM = FRAGOFF + FRAGS;
  static_assert(MAIN % 16 == 0 && FRAGOFF % 16 == 0, "alignment");
};

__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
  return r;
}
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

__device__ __forceinline__ uint32_t pack_f16(float x0, float x1) {
  const __half2 h = __floats2half2_rn(x0, x1);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// x - f16(x) of both halves, as f16
__device__ __forceinline__ uint32_t pack_rest(float x0, float x1, uint32_t hi) {
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
  return pack_f16(x0 - b.x, x1 - b.y);
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
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

// Out of line: between two parts, with few registers to keep over the call.
__device__ __noinline__ void step_walk(ExtWalk &walk, const ExtendArgs &a, const ExtendBatch &batch, int p) {
  walk.next(a, batch, p);
}
__device__ __noinline__ void abandon_walk(ExtWalk &walk, const ExtendArgs &a, const ExtendBatch &batch, int p) {
  walk.abandon(a, batch, p);
}

template <int HD, int LIMBS, typename T>
__global__ void __launch_bounds__(XCfg<HD, LIMBS>::THREADS, XCfg<HD, LIMBS>::MINB)
extend_mma_kernel(const __grid_constant__ ExtendArgs a, const __grid_constant__ ExtendBatch batch,
                  const __grid_constant__ ExtendRuns runs, const int vec) {
  using C = XCfg<HD, LIMBS>;
  constexpr int NG = C::NG, R = C::R, NR = 2;   // NR: rows of a lane, g + 8 r
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int last_part;
  __shared__ ExtWalk walk;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::MAIN);
  float *q_s = reinterpret_cast<float *>(smem + C::QOFF);
  float *stat_s = reinterpret_cast<float *>(smem + C::STATOFF);
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
    if (threadIdx.x == 0)
      for (int i = 0; i < it.npages && i < C::NSTAGE; i++) issue(i);

    // ---- the tile's q rows: f32 in shared memory, row maxima and group sums ------
    for (int x = threadIdx.x; x < R * (HD / 4); x += C::THREADS) {
      const int r = x / (HD / 4), d = 4 * (x % (HD / 4));
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (r < it.rows) {
        const int row = it.row0 + r;
        const T *p = reinterpret_cast<const T *>(a.q.data) +
                     (long long)(it.tok0 + row / a.G) * a.q.token_stride +
                     (long long)(it.h * a.G + row % a.G) * a.q.head_stride + d;
        if (vec) load4<T, true>(p, v);
        else load4<T, false>(p, v);
      }
      *reinterpret_cast<float4 *>(q_s + r * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    // a warp's rows together, step by step
    {
      constexpr int RW = R / C::NW;
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
        const bool any = __any_sync(0xffffffffu, bad[i]);
        const int r = warp + C::NW * i;
        if (lane == 0) {
          stat_s[r] = any ? INFINITY : mx[i];
#pragma unroll
          for (int gg = 0; gg < NG; gg++) stat_s[R + r * NG + gg] = sm[i][gg];
        }
      }
    }
    __syncthreads();
    // rows g + 8 r of this lane
    float rowfac[NR], qsum[NR][NG], kstart[NR][NG];
    RowMask mask[NR];
    {
      float up[NR];
#pragma unroll
      for (int r = 0; r < NR; r++) {
        const float hmax = stat_s[g + 8 * r];
        const bool fine = hmax <= 3.0e38f;
        int e = 0;
        frexpf(hmax > 0.0f && fine ? hmax : 1.0f, &e);          // hmax in [2^(e-1), 2^e)
        const int qe = max(min(5 - e, 126), -126);
        up[r] = fine ? __uint_as_float((uint32_t)(127 + qe) << 23) : 0.0f;
        // a row with an infinity or NaN in q has NaN scores
        rowfac[r] = fine ? a.scale_log2 * __uint_as_float((uint32_t)(127 - qe) << 23)
                         : __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int gg = 0; gg < NG; gg++)
          qsum[r][gg] = fine ? stat_s[R + (g + 8 * r) * NG + gg] * up[r] : 0.0f;
        mask[r] = row_mask(a, it, it.row0 + g + 8 * r);
      }
      // A fragments of k-step s = (word j, byte parity par) of group gg: dims
      // d = 64 gg + 8c + 4j + par and d + 2 (low nibbles), d + 32 and d + 34 (high
      // nibbles, held times 16)
#pragma unroll
      for (int r = 0; r < NR; r++)
#pragma unroll
        for (int gg = 0; gg < NG; gg++) kstart[r][gg] = 0.0f;
      // each warp one step of every group
#pragma unroll
      for (int gg = 0; gg < NG; gg++) {
        const int s = 4 * gg + warp;
        const int d = 64 * gg + 8 * c + 4 * ((s >> 1) & 1) + (s & 1);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {   // k & 1: row, k >> 1: high nibbles
          const int r = k & 1;
          const float *p = q_s + (g + 8 * r) * HD + d + 32 * (k >> 1);
          const float f = up[r] * (C::KRAW || (k >> 1) ? 0.0625f : 1.0f);
          const float x0 = up[r] == 0.0f ? 0.0f : p[0] * f;   // inf * 0
          const float x1 = up[r] == 0.0f ? 0.0f : p[2] * f;
          hi[k] = pack_f16(x0, x1);
          if (C::KRAW) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi[k]));
            kstart[r][gg] -= 1024.0f * (h.x + h.y);
          }
          lo[k] = LIMBS == 2 ? pack_rest(x0, x1, hi[k]) : 0u;
        }
        uint4 *f = frag_s + s * LIMBS * 32 + lane;
        f[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (LIMBS == 2) f[32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    if (C::KRAW) {
#pragma unroll
      for (int r = 0; r < NR; r++)
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          kstart[r][gg] += __shfl_xor_sync(0xffffffffu, kstart[r][gg], 1);
          kstart[r][gg] += __shfl_xor_sync(0xffffffffu, kstart[r][gg], 2);
          if (c == 0) start_s[((g + 8 * r) * NG + gg) * C::NW + warp] = kstart[r][gg];
        }
    }
    __syncthreads();
    if (C::KRAW) {
#pragma unroll
      for (int r = 0; r < NR; r++)
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          const float4 k4 = *reinterpret_cast<const float4 *>(start_s + ((g + 8 * r) * NG + gg) * C::NW);
          kstart[r][gg] = (k4.x + k4.y) + (k4.z + k4.w);
        }
    }

    float o[NG][8][4];
#pragma unroll
    for (int gg = 0; gg < NG; gg++)
#pragma unroll
      for (int n = 0; n < 8; n++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[gg][n][k] = 0.0f;
    float m_run[NR], m_eff[NR], l_run[NR], pb[NR][NG];
    // Everything a row sums is divided by a power of two near the largest V scale
    // the row has attended (eref: its biased exponent, -6 before the first), by
    // way of the exponential's argument (m_eff); it moves like the maximum, when a
    // scale passes it by 2^6, so that p s stays below 2^8 2^7.
    int eref[NR];
#pragma unroll
    for (int r = 0; r < NR; r++) {
      m_run[r] = -INFINITY;
      m_eff[r] = l_run[r] = 0.0f;
      eref[r] = -6;
#pragma unroll
      for (int gg = 0; gg < NG; gg++) pb[r][gg] = 0.0f;
    }

    // page_ex: largest exponent of a V scale of the page (full pages)
    auto step = [&](auto full_tag, const uint8_t *ks, int page_pos0, int p0, int page_ex) {
      constexpr bool FULL = decltype(full_tag)::value;
      const uint8_t *vsm = ks + C::PB;
      bool on[NR][4];
      float sk[4][NG], bk[4][NG];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int tp = p0 + 2 * c + (j & 1) + (j >> 1) * 8;
        if (!FULL) {
#pragma unroll
          for (int r = 0; r < NR; r++) on[r][j] = mask[r].attends(page_pos0 + tp);
        }
        if constexpr (NG == 2) {
          const float4 k4 = *reinterpret_cast<const float4 *>(ks + C::NIB + tp * 16);
          sk[j][0] = k4.x; bk[j][0] = k4.y; sk[j][1] = k4.z; bk[j][1] = k4.w;
        } else {
          const float2 k2 = *reinterpret_cast<const float2 *>(ks + C::NIB + tp * 8);
          sk[j][0] = k2.x; bk[j][0] = k2.y;
        }
#pragma unroll
        for (int gg = 0; gg < NG && !C::KRAW; gg++) bk[j][gg] = fmaf(8.0f, sk[j][gg], bk[j][gg]);
      }
      // ---- scores --------------------------------------------------------------
      float sc[NR][4];
      {
        float dk[2][NG][4];
#pragma unroll
        for (int gg = 0; gg < NG; gg++) {
          uint2 wv[2];
#pragma unroll
          for (int tile = 0; tile < 2; tile++) {
            wv[tile] = *reinterpret_cast<const uint2 *>(ks + (p0 + 8 * tile + g) * (HD / 2) + 8 * c + 32 * gg);
#pragma unroll
            for (int k = 0; k < 4; k++) dk[tile][gg][k] = C::KRAW ? kstart[k >> 1][gg] : 0.0f;
          }
#pragma unroll
          for (int s = 0; s < 4; s++) {
            uint32_t b0[2], b1[2];
#pragma unroll
            for (int tile = 0; tile < 2; tile++) {
              const uint32_t w = (s >> 1) ? wv[tile].y : wv[tile].x;
              const uint32_t y = (s & 1) ? w >> 8 : w;
              b0[tile] = C::KRAW ? raw_hi((s & 1) ? w >> 4 : w << 4) : nib_lo(y);
              b1[tile] = C::KRAW ? raw_hi(y) : nib_hi(y);
            }
#pragma unroll
            for (int l = 0; l < LIMBS; l++) {
              const uint4 f = frag_s[((4 * gg + s) * LIMBS + l) * 32 + lane];
              const uint32_t af[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
              for (int tile = 0; tile < 2; tile++) mma(dk[tile][gg], af, b0[tile], b1[tile]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int r = 0; r < NR; r++) {
            float u = 0.0f;
#pragma unroll
            for (int gg = 0; gg < NG; gg++) {
              u = fmaf(dk[j >> 1][gg][2 * r + (j & 1)], sk[j][gg], u);
              u = fmaf(qsum[r][gg], bk[j][gg], u);
            }
            u *= rowfac[r];
            sc[r][j] = (FULL || on[r][j]) ? u : -INFINITY;
          }
      }
      float sv[4][NG], bv[4][NG];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int tp = p0 + 2 * c + (j & 1) + (j >> 1) * 8;
        if constexpr (NG == 2) {
          const float4 v4 = *reinterpret_cast<const float4 *>(vsm + C::NIB + tp * 16);
          sv[j][0] = v4.x; bv[j][0] = v4.y; sv[j][1] = v4.z; bv[j][1] = v4.w;
        } else {
          const float2 v2 = *reinterpret_cast<const float2 *>(vsm + C::NIB + tp * 8);
          sv[j][0] = v2.x; bv[j][0] = v2.y;
        }
#pragma unroll
        for (int gg = 0; gg < NG; gg++) bv[j][gg] = fmaf(8.0f, sv[j][gg], bv[j][gg]);
      }
      // ---- online softmax, base 2, lazy maximum -----------------------------------
      // A row moves when a score passes its maximum by 8, or a V scale that it
      // attends passes its reference by 2^6 (scales are negative only in damaged
      // files; NaN is passed over).
      bool move = false;
      float lm[NR];
      int ex[NR];
#pragma unroll
      for (int r = 0; r < NR; r++) {
        lm[r] = fmaxf(fmaxf(sc[r][0], sc[r][1]), fmaxf(sc[r][2], sc[r][3]));
        if (FULL) {
          ex[r] = page_ex;
        } else {
          float sx = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            float s = fabsf(sv[j][0]);
            if (NG == 2) s = fmaxf(s, fabsf(sv[j][NG - 1]));
            if (on[r][j]) sx = fmaxf(sx, s);
          }
          ex[r] = (int)(__float_as_uint(sx) >> 23);
        }
        move = move || lm[r] > m_run[r] + 8.0f || ex[r] > eref[r] + 6;
      }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int r = 0; r < NR; r++) {
          float t = lm[r];
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
          t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
          int x = ex[r];
          if (!FULL && x >= 253) {   // without the infinite ones
            x = 0;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
              for (int gg = 0; gg < NG; gg++) {
                const int e1 = (int)(__float_as_uint(sv[j][gg]) >> 23) & 255;
                if (on[r][j] && e1 < 255) x = max(x, min(e1, 252));
              }
          }
          x = max(x, __shfl_xor_sync(0xffffffffu, x, 1));
          x = max(x, __shfl_xor_sync(0xffffffffu, x, 2));
          const bool mv = t > m_run[r] + 8.0f, me = x > eref[r] + 6;
          if (mv || me) {
            float alpha = mv ? ex2(m_run[r] - t) : 1.0f;
            if (mv) m_run[r] = t;
            // before the first reference all sums are zero, or NaN
            if (me && eref[r] > 0) alpha *= __uint_as_float((uint32_t)max(127 + eref[r] - x, 0) << 23);
            if (me) eref[r] = x;
            m_eff[r] = (m_run[r] == -INFINITY ? 0.0f : m_run[r]) +
                       (eref[r] > 0 ? (float)(eref[r] - 127) : 0.0f);
            l_run[r] *= alpha;
#pragma unroll
            for (int gg = 0; gg < NG; gg++) {
              pb[r][gg] *= alpha;
#pragma unroll
              for (int n = 0; n < 8; n++) {
                o[gg][n][2 * r] *= alpha;
                o[gg][n][2 * r + 1] *= alpha;
              }
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < NR; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          sc[r][j] = ex2(sc[r][j] - m_eff[r]);   // the weights from here on
          l_run[r] += sc[r][j];
        }
      // ---- outputs -------------------------------------------------------------
#pragma unroll
      for (int gg = 0; gg < NG; gg++) {
        uint32_t ah[4], al[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {   // k & 1: row, k >> 1: positions 2c+8, 2c+9
          const int r = k & 1;
          float x[2];
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int j = 2 * (k >> 1) + e;
            // what is not attended adds nothing, whatever its scale and bias are
            x[e] = (FULL || on[r][j]) ? sc[r][j] * sv[j][gg] : 0.0f;
            if (FULL || on[r][j]) pb[r][gg] = fmaf(sc[r][j], bv[j][gg], pb[r][gg]);
          }
          ah[k] = pack_f16(x[0], x[1]);
          al[k] = LIMBS == 2 ? pack_rest(x[0], x[1], ah[k]) : 0u;
        }
        // V bytes: lane (g, c) receives bytes 16w + 2g, + 1 of positions 2c, 2c+1
        // (x[2w]) and 2c+8, 2c+9 (x[2w+1])
        uint32_t x[4];
        {
          const int t = lane >> 3, r = lane & 7;
          ldsm_x4_trans(x, smem_u32(vsm + (p0 + 8 * (t & 1) + r) * (HD / 2) + 32 * gg + 16 * (t >> 1)));
        }
#pragma unroll
        for (int n = 0; n < 8; n++) {   // n = 4w + 2 parity + (high nibbles)
          const int w = n >> 2, par = (n >> 1) & 1;
          const uint32_t y0 = par ? x[2 * w] >> 8 : x[2 * w];
          const uint32_t y1 = par ? x[2 * w + 1] >> 8 : x[2 * w + 1];
          const uint32_t b0 = (n & 1) ? nib_hi(y0) : nib_lo(y0);
          const uint32_t b1 = (n & 1) ? nib_hi(y1) : nib_lo(y1);
          mma(o[gg][n], ah, b0, b1);
          if constexpr (LIMBS == 2) mma(o[gg][n], al, b0, b1);
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
      const uint8_t *ks = smem + st * C::STAGE_BYTES;
      const int page_pos0 = (it.pg0 + i) * kPagePositions;
      const bool full = page_pos0 >= it.all_lo && page_pos0 + kPagePositions <= it.all_hi;
      if (full) {
        // finite scales only: what an infinite one reaches is NaN anyway
        int ex = 0;
#pragma unroll
        for (int k = 0; k < 2 * NG; k++) {
          const uint32_t b = *reinterpret_cast<const uint32_t *>(ks + C::PB + C::NIB + 8 * (lane + 32 * k));
          const int e = (int)(b >> 23) & 255;
          ex = max(ex, e < 255 ? min(e, 252) : 0);
        }
        ex = __reduce_max_sync(0xffffffffu, ex);
#pragma unroll 1
        for (int s = 0; s < kPagePositions / 16; s++) step(std::true_type{}, ks, page_pos0, 16 * s, ex);
      } else {
#pragma unroll 1
        for (int s = 0; s < kPagePositions / 16; s++) step(std::false_type{}, ks, page_pos0, 16 * s, 0);
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
    float *ow = lw + C::NW * R;                    // [NW][R][HD]
#pragma unroll
    for (int r = 0; r < NR; r++) {
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
      l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
#pragma unroll
      for (int gg = 0; gg < NG; gg++) {
        pb[r][gg] += __shfl_xor_sync(0xffffffffu, pb[r][gg], 1);
        pb[r][gg] += __shfl_xor_sync(0xffffffffu, pb[r][gg], 2);
      }
      const int row = warp * R + g + 8 * r;
      const float vs = eref[r] > 0 ? __uint_as_float((uint32_t)eref[r] << 23) : 1.0f;
      if (c == 0) {
        mw[row] = m_run[r];
        lw[row] = l_run[r] * vs;
      }
#pragma unroll
      for (int gg = 0; gg < NG; gg++)
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
          for (int hi = 0; hi < 2; hi++) {
            const float f = hi ? vs * 0.0625f : vs, b = pb[r][gg] * vs;
            const float (&e0)[4] = o[gg][4 * w + hi], (&e1)[4] = o[gg][4 * w + 2 + hi];
            const int k = 2 * r;
            *reinterpret_cast<float4 *>(ow + row * HD + 64 * gg + 32 * hi + 16 * w + 4 * c) =
                make_float4(fmaf(e0[k], f, b), fmaf(e1[k], f, b), fmaf(e0[k + 1], f, b), fmaf(e1[k + 1], f, b));
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
        const float4 v = *reinterpret_cast<const float4 *>(ow + (w * R + r) * HD + d);
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

template <int HD, int LIMBS, typename T>
int resident_one() {
  using C = XCfg<HD, LIMBS>;
  static std::atomic<int> cached[64];
  int dev = 0;
  cudaGetDevice(&dev);
  const int hit = cached[dev & 63].load(std::memory_order_relaxed);
  if (hit) return hit;
  auto fn = extend_mma_kernel<HD, LIMBS, T>;
  if (check_cuda(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM),
                 "extend: smem attribute"))
    return 0;
  int per_sm = 1;
  cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, C::THREADS, C::SMEM);
  if (per_sm < 1) per_sm = 1;
  cached[dev & 63].store(per_sm, std::memory_order_relaxed);
  return per_sm;
}

template <int HD, int LIMBS, typename T>
int launch_one(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks, bool vec,
               cudaStream_t s) {
  using C = XCfg<HD, LIMBS>;
  extend_mma_kernel<HD, LIMBS, T><<<n_blocks, C::THREADS, C::SMEM, s>>>(a, b, runs, vec ? 1 : 0);
  return check_cuda(cudaGetLastError(), "extend_mma launch");
}

// f(launch or resident functions of the instance that serves the arguments)
template <int HD, typename F>
int pick(int dtype, F f) {
  if (dtype == EAKV_F32) return f.template operator()<HD, 2, float>();
  if (dtype == EAKV_F16) return f.template operator()<HD, 1, __half>();
  return f.template operator()<HD, 1, __nv_bfloat16>();
}

struct Resident {
  template <int HD, int LIMBS, typename T> int operator()() const {
    return resident_one<HD, LIMBS, T>();
  }
};
struct Launch {
  const ExtendArgs &a;
  const ExtendBatch &b;
  const ExtendRuns &runs;
  int n_blocks;
  bool vec;
  cudaStream_t s;
  template <int HD, int LIMBS, typename T> int operator()() const {
    return launch_one<HD, LIMBS, T>(a, b, runs, n_blocks, vec, s);
  }
};

}  // namespace

// CTAs per SM of the kernel for this shape on the current device (0: error).
// Sets the kernel's shared-memory limit, so it comes before the launch.
int extend_mma_resident(int head_dim, int dtype) {
  return head_dim == 128 ? pick<128>(dtype, Resident{}) : pick<64>(dtype, Resident{});
}

int extend_mma_launch(const ExtendArgs &a, const ExtendBatch &b, const ExtendRuns &runs, int n_blocks,
                      bool vec, cudaStream_t s) {
  const Launch f{a, b, runs, n_blocks, vec, s};
  return a.geom.gpd == 2 ? pick<128>(a.dtype, f) : pick<64>(a.dtype, f);
}

}  // namespace eakv
