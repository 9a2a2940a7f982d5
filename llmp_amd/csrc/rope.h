// Rotary positions: the rotation by an angle that a table holds as a fraction of a turn a position.
#ifndef LLMP_AMD_CSRC_ROPE_H_
#define LLMP_AMD_CSRC_ROPE_H_

#include "common.h"

namespace llmp_hip {

// cos and sin of position * turns, where `turns` is a 64-bit fraction of a whole turn: the product modulo 2^64 is the angle's own
// fraction, exactly, at any position. Its upper 32 bits (2^-32 of a turn off at most) are split into quarter turns and a rest
// within an eighth of a turn, whose sine and cosine are their Taylor sums through x^9 and x^10: the terms left out are
// below 2^-28. Off by 2^-23 at most in all.
__device__ __forceinline__ void Turn(uint64_t turns, int32_t position, float* cosine, float* sine) {
  const uint64_t phase = turns * static_cast<uint64_t>(static_cast<int64_t>(position));
  const uint32_t t = static_cast<uint32_t>(phase >> 32);
  const uint32_t quarter = (t + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(t - (quarter << 30))) * 0x1.921fb6p-30f;  // pi / 2^31, to F32
  const float y = x * x;
  const float s = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), 1.0f);
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f), -1.0f / 720.0f), 1.0f / 24.0f), -0.5f), 1.0f);
  const float a = quarter & 1u ? s : c, b = quarter & 1u ? c : s;
  *cosine = (quarter + 1u) & 2u ? -a : a;
  *sine = quarter & 2u ? -b : b;
}

}  // namespace llmp_hip

#endif  // LLMP_AMD_CSRC_ROPE_H_
