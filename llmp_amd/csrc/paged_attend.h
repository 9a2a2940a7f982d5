// What the two forms of llmp.paged.attend share: the launch's arguments, the queries as whole-number digits, a page's place, and
// the softmax's numbers in the units the kernels hold them in.
//
// A logit is s = scale * q . k with k = c * ks. A query row is whole numbers: x = f * (256 hi + lo), f = max|x| / 32639 (three
// digits and 8355584 for F32), so hi . c and lo . c are integer products and s = (256 (hi . c) + lo . c) * (f * ks * scale) is exact up
// to x's own rounding: 2^-16 of the row's largest magnitude, 2^-24 for F32.
// V's scale vs differs from page to page, so the sum's weights are w = exp(s) * vs. The running maximum is of t = log2(e) s + log2(vs)
// (vs at least 2^-80 there: p below then stays below 2^95, and its sums below 2^127 over all the tokens that a row can have):
// p = exp2(log2(e) s - E) goes to the sum of probabilities, p * vs is rounded to F16 for the product with V's codes. E is set kLift below
// the maximum and follows it once that is kSlack further, so a weight is at most 2^15 and the row's largest at least 2^kLift: the
// whole of F16's range (largest 2^16, smallest step 2^-24) lies under the largest. A weight is off by 2^-11 of itself, or by
// 2^-(25 + kLift) of the row's largest where that is more. For F32 what the F16 leaves of a weight goes into a second product, 2^11 times
// as large (a code times 2^-11 is exact in F16): off by 2^-22 of itself or 2^-(36 + kLift) of the largest. The common factor 2^E leaves at the end.
#ifndef LLMP_AMD_CSRC_PAGED_ATTEND_H_
#define LLMP_AMD_CSRC_PAGED_ATTEND_H_

#include "paged.h"

namespace llmp_hip {

constexpr float kLog2E = 1.4426950408889634f;
constexpr int kTileTokens = 64;
// In log2, 15 together. (By a slack of 8, 5, 3, 2: a chunk of 2048 tokens behind 2048 156.0, 156.2, 157.5, 158.9 us, 6 ragged prompts at head
// size 256 108.9, 109.6, 110.9, 111.8.)
constexpr float kLift = 10.0f, kSlack = 5.0f;

struct PagedAttendArgs {
  llmp_paged_attend op;
  float* partial;       // the few rows' form: [2 * workgroups][16][D + 2]: E, sum, values
  int32_t* parts;       // [workgroups][4]
  uint32_t page_magic;   // n / (page / 16) by a multiplication: PagedDivide
  uint32_t group_magic;  // n / group
  int group;            // query heads a KV head
  int most_length;      // tokens a table row can name
  int shift;            // the few rows' form: a unit of the line is 2^shift tiles
  int whole_units;  // the few rows' form: units a workgroup takes where it takes whole segments, 0 where the line is cut evenly
  int few_rows;         // requests of more (token, head) rows than these are the many rows' form's
  const int32_t* all_taken;  // in memory, not zero: by the many rows' form; null: none is
};

// n / d for n * d < 2^32, magic = 2^32 / d + 1 (0 for d = 1): n times the magic's excess stays below 2^32 / d.
__device__ __forceinline__ uint32_t PagedDivide(uint32_t n, uint32_t magic) { return magic == 0 ? n : __umulhi(n, magic); }

// Over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the same column of a 16-column matrix tile): x in two registers, the odd rows of
// 16 lanes of one swapped with the even rows of the other, then the upper halves with the lower ones. (As instructions: the
// compiler's builtin gives one of the two results for both. The wait states are those between a vector write and the swap.)
__device__ __forceinline__ void SwapRows16(float& a, float& b) { asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void SwapHalves(float& a, float& b) { asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ uint32_t AcrossHalvesMost(uint32_t v) {
  float a = __builtin_bit_cast(float, v), b = a;
  SwapHalves(a, b);
  return max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}
__device__ __forceinline__ uint32_t AcrossGroupsMost(uint32_t v) {
  float a = __builtin_bit_cast(float, v), b = a;
  SwapRows16(a, b);
  return AcrossHalvesMost(max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)));
}
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

// Over the lanes of a column of a ROWS-column tile.
template <int ROWS>
__device__ __forceinline__ float Across(float v) { return ROWS == 32 ? AcrossHalvesMax(v) : AcrossGroupsMax(v); }
template <int ROWS>
__device__ __forceinline__ uint32_t Across(uint32_t v) { return ROWS == 32 ? AcrossHalvesMost(v) : AcrossGroupsMost(v); }
template <int ROWS>
__device__ __forceinline__ float AcrossSum(float v) { return ROWS == 32 ? AcrossHalvesSum(v) : AcrossGroupsSum(v); }
// Inclusive sums over the wave's lanes: within rows of 16 by shifts, then each row's last to the next row, the lower half's to the
// upper one.
__device__ __forceinline__ uint32_t WaveSums(uint32_t v) {
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x111, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x112, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x114, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x118, 0xF, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xA, 0xF, false));
  v += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xC, 0xF, false));
  return v;
}

template <int TYPE>
constexpr int kDigits = TYPE == LLMP_X_F32 ? 3 : 2;
template <int TYPE>
constexpr float kDigitMax = TYPE == LLMP_X_F32 ? 8355584.0f : 32639.0f;  // 0x7F7F00: a rounding up still fits three digits; 0x7F7F

// Part of a query row: N eights of values as they lie in memory.
template <int TYPE, int N>
struct QueryPart {
  static constexpr int kWords = TYPE == LLMP_X_F32 ? 2 : 1;  // 16-byte words an eight
  U32x4 raw[N * kWords];
  __device__ __forceinline__ void Load(const void* base, int i, int64_t element) {
    const U32x4* from = TYPE == LLMP_X_F32 ? reinterpret_cast<const U32x4*>(static_cast<const float*>(base) + element)
                                           : reinterpret_cast<const U32x4*>(static_cast<const uint16_t*>(base) + element);
#pragma unroll
    for (int w = 0; w < kWords; ++w) raw[i * kWords + w] = from[w];
  }
  // The largest magnitude as bits: their order is the magnitudes', infinities and NaN the largest.
  __device__ __forceinline__ uint32_t MostBits() const {
    typedef unsigned short U16x2 __attribute__((ext_vector_type(2)));
    if constexpr (TYPE == LLMP_X_F32) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < N * kWords; ++i) {
#pragma unroll
        for (int w = 0; w < 4; ++w) most = max(most, raw[i][w] & 0x7FFFFFFFu);
      }
      return most;
    } else {
      U16x2 most = {0, 0};
#pragma unroll
      for (int i = 0; i < N * kWords; ++i) {
#pragma unroll
        for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(U16x2, raw[i][w] & 0x7FFF7FFFu));
      }
      return max(most.x, most.y);
    }
  }
  __device__ __forceinline__ void Four(int i, int half, float (&v)[4]) const {
    if constexpr (TYPE == LLMP_X_F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t word = raw[2 * i + half][e];  // (a copy: the cast of the element itself reads the vector's first)
        v[e] = __builtin_bit_cast(float, word);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t word = raw[i][2 * half + e / 2], bits = e % 2 ? word >> 16 : word & 0xFFFFu;
        v[e] = TYPE == LLMP_X_BF16 ? (e % 2 ? __builtin_bit_cast(float, word & 0xFFFF0000u) : Bf16BitsToFloat(bits)) : HalfBitsToFloat(bits);
      }
    }
  }
};
// A row's unit from its largest magnitude's bits, and what takes values to whole numbers of it.
struct QueryUnit {
  float unit, inverse;
};
template <int TYPE>
__device__ __forceinline__ QueryUnit UnitOf(uint32_t most_bits) {
  constexpr uint32_t kInfinity = TYPE == LLMP_X_F32 ? 0x7F800000u : TYPE == LLMP_X_BF16 ? 0x7F80u : 0x7C00u;
  const float most = TYPE == LLMP_X_F32 ? __builtin_bit_cast(float, most_bits) : TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(most_bits) : HalfBitsToFloat(most_bits);
  // (A row of zeros, or of magnitudes whose reciprocal is none, is zeros; one with an infinity or a NaN has no logits.)
  const bool bad = most_bits >= kInfinity, small = !(most > 0x1p-100f);
  return {bad ? __builtin_nanf("") : small ? 0.0f : most / kDigitMax<TYPE>, bad || small ? 0.0f : kDigitMax<TYPE> / most};
}
// Four values' digits, the highest first, each balanced (-128 to 127): the bytes of the whole number once what the lower digits
// borrow is added.
template <int DIGITS>
__device__ __forceinline__ void PackDigits(const float (&v)[4], float inverse, uint32_t (&packed)[DIGITS]) {
  uint32_t q[4], up[4];
  const auto bytes = [](const uint32_t (&x)[4], uint32_t low_pair, uint32_t high_pair) {
    return __builtin_amdgcn_perm(x[1], x[0], low_pair) | __builtin_amdgcn_perm(x[3], x[2], high_pair);
  };
  if constexpr (DIGITS == 2) {
    // (Added to 1.5 * 2^23 a value is rounded to a whole number, and that is what the float's low bits are.)
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = __builtin_bit_cast(uint32_t, fmaf(v[e], inverse, 12582912.0f)), up[e] = q[e] + 0x80u;
    packed[0] = bytes(up, 0x0C0C0501u, 0x05010C0Cu);
    packed[1] = bytes(q, 0x0C0C0400u, 0x04000C0Cu);
  } else {
    uint32_t top[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float whole = rintf(v[e] * inverse);
      q[e] = static_cast<uint32_t>(static_cast<int>(whole == whole ? whole : 0.0f));
      up[e] = q[e] + 0x80u, top[e] = q[e] + 0x8080u;
    }
    packed[0] = bytes(top, 0x0C0C0602u, 0x06020C0Cu);
    packed[1] = bytes(up, 0x0C0C0501u, 0x05010C0Cu);
    packed[2] = bytes(q, 0x0C0C0400u, 0x04000C0Cu);
  }
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

// What a weight's F16 leaves of it, and the codes that it multiplies. (Without the factor an F32 prompt of 2000 tokens behind 2000 takes 207
// us at head size 256, 158 at 128, 102 at 64, with it 229, 167, 107; a product of its own, added once a tile, 226 at 256.)
constexpr float kRestUp = 0x1p11f;
__device__ __forceinline__ _Float16 RestOf(float weight, _Float16 held) { return static_cast<_Float16>((weight - static_cast<float>(held)) * kRestUp); }
__device__ __forceinline__ F16x8 RestCodes(F16x8 codes) { return codes * static_cast<_Float16>(1.0f / kRestUp); }

// Where in a row of LDS a piece of 16 bytes lies (and which piece lies there). A wave's read of 16 bytes a lane takes lanes 0 to 3, 12 to
// 15 and 20 to 27 at once, then the others of the first half, and the second half likewise; each 16 lanes are to find their pieces at 16 places
// of the 256 bytes that the banks hold. So lanes 4 to 11 of a group of 16, whose rows these are (tokens 16a + 4t + b for K, dimensions
// in order for V), stand beside the others of the group before or after, who read the neighbouring piece. (Reads with two lanes a place
// measured 1.6 times as long.)
template <int D>
__device__ __forceinline__ int KPiece(int token, int piece) {
  if constexpr (D == 64) return piece ^ ((token >> 4) & 2);
  if constexpr (D == 128) return piece ^ (((token >> 1) & 1) | ((token >> 4) & 3) << 1);
  return piece ^ ((token & 3) | ((token >> 4) & 3) << 2);
}
__device__ __forceinline__ int VPiece(int d, int piece) { return piece ^ ((d >> 2) & 2); }

// A lane's 16 bytes from memory to LDS at `to` (the same in every lane) + 16 lane.
__device__ __forceinline__ void ToLds(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(reinterpret_cast<uintptr_t>(from)),
                                   reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(reinterpret_cast<uintptr_t>(to)), 16, 0, 0);
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
__device__ __forceinline__ float ScaleLog(float vs) { return __builtin_amdgcn_logf(fmaxf(vs, 0x1p-80f)); }

// The many rows' form (its own file), for requests of more than few_rows rows, and those of fewer where they are little work beside
// them: the number that it gives the place of is then not zero.
size_t PagedManyScratch(const llmp_paged_attend& op, int cus);
const int32_t* PagedManyRows(const PagedAttendArgs& args, void* scratch, int cus, hipStream_t stream);

}  // namespace llmp_hip

#endif  // LLMP_AMD_CSRC_PAGED_ATTEND_H_
