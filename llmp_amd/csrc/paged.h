// What the kernels over the paged 8-bit KV cache share: host checks, element loads, and the requests' rows and lengths as
// a kernel may use them whatever the arrays hold.
#ifndef LLMP_AMD_CSRC_PAGED_H_
#define LLMP_AMD_CSRC_PAGED_H_

#include <hip/hip_runtime.h>

#include <climits>

#include "common.h"
#include "llmp_hip.h"

namespace llmp_hip {

// 0, or the refusal: what every operator asks of a cache.
int CheckPagedCache(const char* who, const llmp_paged_cache& cache, bool needs_edges);
// ... of `tokens` times `heads` rows of head_dim values at element strides, 16-byte boundaries. (What one token or one head has for a stride
// is not used.)
int CheckPagedRows(const char* who, const char* name, const void* rows, int tokens, int heads, int64_t token_stride, int64_t head_stride, int type);

inline int PagedElementBytes(int type) { return type == LLMP_X_F32 ? 4 : 2; }
// (At most half of what an int counts: sums of a position and a tile's size stay in range.)
constexpr int64_t kMostPagedLength = 1 << 30;

// ---- device.
typedef int I32x4 __attribute__((ext_vector_type(4)));
typedef int I32x2 __attribute__((ext_vector_type(2)));
typedef int I32x16 __attribute__((ext_vector_type(16)));
typedef float F32x4 __attribute__((ext_vector_type(4)));
typedef float F32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 F16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));

// Eight consecutive values at a 16-byte boundary as floats.
template <int TYPE>
__device__ __forceinline__ void LoadEight(const void* base, int64_t element, float (&x)[8]) {
  if constexpr (TYPE == LLMP_X_F32) {
    const F32x4* p = reinterpret_cast<const F32x4*>(static_cast<const float*>(base) + element);
    const F32x4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
  } else {
    const U32x4 a = *reinterpret_cast<const U32x4*>(static_cast<const uint16_t*>(base) + element);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = (i & 1) ? a[i / 2] >> 16 : a[i / 2] & 0xFFFFu;
      x[i] = TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(bits) : HalfBitsToFloat(bits);
    }
  }
}
template <int TYPE>
__device__ __forceinline__ float LoadOne(const void* base, int64_t element) {
  if constexpr (TYPE == LLMP_X_F32) return static_cast<const float*>(base)[element];
  const uint32_t bits = static_cast<const uint16_t*>(base)[element];
  return TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(bits) : HalfBitsToFloat(bits);
}
// N consecutive floats rounded once to the type (N a multiple of 4, at a boundary of N elements or 16 bytes).
template <int TYPE, int N>
__device__ __forceinline__ void StoreValues(void* base, int64_t element, const float (&x)[N]) {
  static_assert(N % 4 == 0, "whole 8- or 16-byte stores");
  if constexpr (TYPE == LLMP_X_F32) {
    F32x4* p = reinterpret_cast<F32x4*>(static_cast<float*>(base) + element);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) p[i] = F32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
  } else {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint32_t lo = TYPE == LLMP_X_BF16 ? FloatToBf16Bits(x[2 * i]) : FloatToHalfBits(x[2 * i]);
      const uint32_t hi = TYPE == LLMP_X_BF16 ? FloatToBf16Bits(x[2 * i + 1]) : FloatToHalfBits(x[2 * i + 1]);
      w[i] = lo | (hi << 16);
    }
    uint16_t* p = static_cast<uint16_t*>(base) + element;
    if constexpr (N % 8 == 0) {
#pragma unroll
      for (int i = 0; i < N / 8; ++i) reinterpret_cast<U32x4*>(p)[i] = U32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint2*>(p)[i] = make_uint2(w[2 * i], w[2 * i + 1]);
    }
  }
}

template <int TYPE>
__device__ __forceinline__ void StoreOne(void* base, int64_t element, float x) {
  if constexpr (TYPE == LLMP_X_F32) static_cast<float*>(base)[element] = x;
  if constexpr (TYPE == LLMP_X_BF16) static_cast<uint16_t*>(base)[element] = static_cast<uint16_t>(FloatToBf16Bits(x));
  if constexpr (TYPE == LLMP_X_F16) static_cast<uint16_t*>(base)[element] = static_cast<uint16_t>(FloatToHalfBits(x));
}

// Eight values' codes at a scale: the IEEE quotients rounded to nearest even, at most 127 in magnitude, 0 for NaN. By products with
// the reciprocal, whose errors (below 2^-15 at 127) matter only near the middle between two codes: there, and at scales without a
// reciprocal, by divisions.
__device__ __forceinline__ void CodesOf(const float (&x)[8], float scale, float inverse, int (&code)[8]) {
  bool near = !(scale > 0x1p-120f);
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float y = x[e] * inverse;
    r[e] = rintf(y);
    near = near || fabsf(y - r[e]) > 0.5f - 0x1p-14f;
  }
  if (__any(near)) {
    asm volatile("" ::: "memory");  // (a branch: it is rarely taken)
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = scale > 0.0f ? rintf(x[e] / scale) : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) code[e] = __builtin_isnan(r[e]) ? 0 : static_cast<int>(fminf(fmaxf(r[e], -127.0f), 127.0f));
}

// A request's new tokens, the tokens that it holds and the position of the first new one, whatever the device arrays hold: `n` 0 where its
// rows are not rows of the call. Where `before` is given a token may be past all that is held (it found no page): its position stays,
// what it sees ends at `length`. Positions stay below 2^31: fewer than 2^30 tokens from at most 2^30 on.
struct PagedRequest {
  int start, n, length, base;
};
__device__ __forceinline__ PagedRequest RequestOf(const int32_t* starts, const int32_t* lengths, const int32_t* before, int r, int tokens, int most_length) {
  const int a = starts[r], b = starts[r + 1];
  PagedRequest q;
  q.start = a;
  q.n = (a >= 0 && b <= tokens && b > a) ? b - a : 0;
  q.length = min(max(lengths[r], 0), most_length);
  q.base = before != nullptr ? min(max(before[r], 0), static_cast<int>(kMostPagedLength)) : q.length - q.n;
  return q;
}
// The end of what the request's token at `position` sees.
__device__ __forceinline__ int SeenTo(const PagedRequest& q, int position) { return min(position + 1, q.length); }

}  // namespace llmp_hip

#endif  // LLMP_AMD_CSRC_PAGED_H_
