// tokens.cuh - shared by the calls that take several tokens per cache: the
// per-call table of caches, rows of 16- or 32-bit elements, and argument
// checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "internal.cuh"

namespace eakv {

// Caches of a call and where their tokens start in the packed rows. Passed by
// value, so a captured launch keeps the lengths it was captured with.
struct TokenBatch {
  uint8_t *base[kMaxBatch];     // device slab
  int pos[kMaxBatch];           // position of the first token
  int first[kMaxBatch + 1];     // packed index of the first token; [n_caches] = total
};

// Cache of packed token t: the last i with first[i] <= t (caches without
// tokens share their start with the next one, which the search prefers).
__device__ __forceinline__ int token_cache(const TokenBatch &b, int n_caches, int t) {
  int lo = 0, hi = n_caches - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.first[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

struct Rows {
  void *data;
  long long token_stride, head_stride;
};

inline Rows rows_of(const eakv_rows_t *r) {
  return r ? Rows{r->data, (long long)r->token_stride, (long long)r->head_stride}
           : Rows{nullptr, 0, 0};
}

inline int dtype_size(int dtype) { return dtype == EAKV_F32 ? 4 : 2; }

// Whether every row starts on a 4-element boundary (vector loads and stores).
inline bool rows_vec(const eakv_rows_t *r) {
  return !r || (((uintptr_t)r->data % (4 * dtype_size(r->dtype))) == 0 && r->token_stride % 4 == 0 &&
                r->head_stride % 4 == 0);
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

template <typename T> struct alignas(4 * sizeof(T)) Vec4 { T v[4]; };

template <typename T, bool kVec>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
  if constexpr (kVec) {
    const Vec4<T> a = *reinterpret_cast<const Vec4<T> *>(p);
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = to_f32<T>(a.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = to_f32<T>(p[e]);
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ void store4(T *p, const float (&x)[4]) {
  if constexpr (kVec) {
    Vec4<T> a;
#pragma unroll
    for (int e = 0; e < 4; e++) a.v[e] = from_f32<T>(x[e]);
    *reinterpret_cast<Vec4<T> *>(p) = a;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) p[e] = from_f32<T>(x[e]);
  }
}

// Checks of a batch of caches and its token counts: the shape checks of the
// decode's batches, counts >= 0, and a total that fits an int. Fills `b`
// (positions from `pos0`, or each cache's seq_len when NULL) and `total`.
int token_batch(const eakv_cache_t *const *caches, int n_caches, int n_q, const int *pos0,
                const int *n, const char *who, TokenBatch &b, int &total);
// A rows argument: pointer, element type, strides that are not negative.
int check_rows(const eakv_rows_t *r, const char *name, const char *who);
// The same of rows that are written: neighbouring ones may not overlap.
int check_out_rows(const eakv_rows_t *r, const char *name, const char *who, int tokens, int heads,
                   int head_dim);

}  // namespace eakv
