// What the two forms of llmp.paged.attend share: the launch's arguments, the queries as whole-number digits, a page's place, and
// the softmax's numbers in the units the kernels hold them in.
//
// A logit is s = scale * q . k with k = c * ks. A query row is whole numbers: x = f * (256 hi + lo), f = max|x| / 32639 (three
// digits and 8355584 for F32), so hi . c and lo . c are integer products and s = (256 (hi . c) + lo . c) * (f * ks * scale) is exact up
// to x's own rounding: 2^-16 of the row's largest magnitude, 2^-24 for F32.
// V's scale vs differs from page to page, so the sum's weights are w = exp(s) * vs. The running maximum is of t = log2(e) s + log2(vs)
// (vs at least 2^-100 there): p = exp2(log2(e) s - E) goes to the sum of probabilities, p * vs <= 1 is rounded to F16 for the
// product with V's codes, and the F16's exponent range is used whatever the scales are. The common factor 2^E leaves at the end.
#ifndef LLMP_AMD_CSRC_PAGED_ATTEND_H_
#define LLMP_AMD_CSRC_PAGED_ATTEND_H_

#include "paged.h"

namespace llmp_hip {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kTileTokens = 64;

struct PagedAttendArgs {
  llmp_paged_attend op;
  float* partial;       // the few rows' form: [2 * workgroups][16][D + 2]: E, sum, values
  int32_t* parts;       // [workgroups][4]
  uint32_t page_magic;  // n / (page / 16) by a multiplication: PagedDivide
  int group;            // query heads a KV head
  int most_length;      // tokens a table row can name
  int few_rows;         // requests of more (token, head) rows than these are the many rows' form's
};

// n / d for n < 2^26 and d from 1 to 16, magic = 2^32 / d + 1 (0 for d = 1): n times the magic's excess stays below 2^32 / d.
__device__ __forceinline__ uint32_t PagedDivide(uint32_t n, uint32_t magic) { return magic == 0 ? n : __umulhi(n, magic); }

// Over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the same column of a 16-column matrix tile): x in two registers, the odd rows of
// 16 lanes of one swapped with the even rows of the other, then the upper halves with the lower ones. (As instructions: the
// compiler's builtin gives one of the two results for both. The wait states are those between a vector write and the swap.)
__device__ __forceinline__ void SwapRows16(float& a, float& b) { asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void SwapHalves(float& a, float& b) { asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ float AcrossHalvesMax(float v) {
  float w = v;
  SwapHalves(v, w);
  return fmaxf(v, w);
}
__device__ __forceinline__ float AcrossHalvesSum(float v) {
  float w = v;
  SwapHalves(v, w);
  return v + w;
}
__device__ __forceinline__ float AcrossGroupsMax(float v) {
  float w = v;
  SwapRows16(v, w);
  return AcrossHalvesMax(fmaxf(v, w));
}
__device__ __forceinline__ float AcrossGroupsSum(float v) {
  float w = v;
  SwapRows16(v, w);
  return AcrossHalvesSum(v + w);
}

template <int TYPE>
constexpr int kDigits = TYPE == LLMP_X_F32 ? 3 : 2;
template <int TYPE>
constexpr float kDigitMax = TYPE == LLMP_X_F32 ? 8355584.0f : 32639.0f;  // 0x7F7F00: a rounding up still fits three digits; 0x7F7F

// Whole numbers' balanced digits, the highest first: each in -128 to 127.
template <int DIGITS>
__device__ __forceinline__ void SplitDigits(int x, int (&digit)[DIGITS]) {
#pragma unroll
  for (int i = DIGITS - 1; i > 0; --i) {
    digit[i] = static_cast<int8_t>(x);
    x = (x - digit[i]) >> 8;
  }
  digit[0] = x;
}

// The sums of the digits' products as one float: three digits' pass 2^31.
template <int DIGITS>
__device__ __forceinline__ float JoinDigits(int hi, int mid, int lo) {
  if constexpr (DIGITS == 2) return static_cast<float>((hi << 8) + lo);
  return fmaf(static_cast<float>(hi), 65536.0f, static_cast<float>((mid << 8) + lo));
}

// Sixteen V codes (bytes) as F16, exactly: a byte c + 128 under 0x64 is the F16 1024 + c + 128.
__device__ __forceinline__ F16x2 TwoCodes(uint32_t biased, uint32_t select) {
  const F16x2 v = __builtin_bit_cast(F16x2, __builtin_amdgcn_perm(biased, 0x64646464u, select));
  return v - F16x2{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
}
__device__ __forceinline__ F16x8 EightCodes(uint32_t a, uint32_t b) {
  a ^= 0x80808080u, b ^= 0x80808080u;
  const F16x2 v0 = TwoCodes(a, 0x00050004u), v1 = TwoCodes(a, 0x00070006u), v2 = TwoCodes(b, 0x00050004u), v3 = TwoCodes(b, 0x00070006u);
  return F16x8{v0.x, v0.y, v1.x, v1.y, v2.x, v2.y, v3.x, v3.y};
}

// softcap * tanh(s / softcap). F32 results take the library's tanh; 16-bit ones 1 - 2 / (e^2x + 1), whose error (2^-23 of the
// softcap) is far below their rounding.
template <int TYPE>
__device__ __forceinline__ float Capped(float s, float softcap, float inverse) {
  if constexpr (TYPE == LLMP_X_F32) return softcap * tanhf(s * inverse);
  const float e = __builtin_amdgcn_exp2f(s * inverse * (2.0f * kLog2E));
  return softcap * (1.0f - 2.0f * __builtin_amdgcn_rcpf(e + 1.0f));
}

// log2 of a page's V scale, as the running maximum takes it.
__device__ __forceinline__ float ScaleLog(float vs) { return __builtin_amdgcn_logf(fmaxf(vs, 0x1p-100f)); }

// The many rows' form (its own file), for requests of more than few_rows rows.
size_t PagedManyScratch(const llmp_paged_attend& op, int cus);
void PagedManyRows(const PagedAttendArgs& args, void* scratch, int cus, hipStream_t stream);

}  // namespace llmp_hip

#endif  // LLMP_AMD_CSRC_PAGED_ATTEND_H_
