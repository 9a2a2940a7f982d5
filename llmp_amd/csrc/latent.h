// What the kernels over latent vectors share: host checks, and 16-bit values as the matrix instructions take them.
#ifndef LLMP_AMD_CSRC_LATENT_H_
#define LLMP_AMD_CSRC_LATENT_H_

#include "paged.h"

namespace llmp_hip {

// 0, or the refusal: what every operator asks of a latent cache.
int CheckLatentCache(const char* who, const llmp_latent_cache& cache);

// ---- device.
typedef __bf16 B16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 B16x8 __attribute__((ext_vector_type(8)));

template <int TYPE>
struct Sixteen;
template <>
struct Sixteen<LLMP_X_BF16> {
  typedef B16x8 Eight;
  typedef B16x2 Two;
  typedef __bf16 One;
  static __device__ __forceinline__ F32x16 Product32(Eight a, Eight b, F32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ F32x4 Product16(Eight a, Eight b, F32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ float AddTwo(Two v, float sum) {
    const __bf16 one = static_cast<__bf16>(1.0f);
    return __builtin_amdgcn_fdot2_f32_bf16(v, Two{one, one}, sum, false);
  }
  template <bool HIGH>
  static __device__ __forceinline__ Two OfE4m3(uint32_t codes) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, HIGH); }
};
template <>
struct Sixteen<LLMP_X_F16> {
  typedef F16x8 Eight;
  typedef F16x2 Two;
  typedef _Float16 One;
  static __device__ __forceinline__ F32x16 Product32(Eight a, Eight b, F32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ F32x4 Product16(Eight a, Eight b, F32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ float AddTwo(Two v, float sum) {
    const _Float16 one = static_cast<_Float16>(1.0f);
    return __builtin_amdgcn_fdot2(v, Two{one, one}, sum, false);
  }
  template <bool HIGH>
  static __device__ __forceinline__ Two OfE4m3(uint32_t codes) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HIGH); }
};

// Eight E4M3 codes as 16-bit values (exact: both types hold every one of them).
template <int TYPE>
__device__ __forceinline__ typename Sixteen<TYPE>::Eight EightE4m3(uint32_t low, uint32_t high) {
  using S = Sixteen<TYPE>;
  const typename S::Two a = S::template OfE4m3<false>(low), b = S::template OfE4m3<true>(low);
  const typename S::Two c = S::template OfE4m3<false>(high), d = S::template OfE4m3<true>(high);
  return typename S::Eight{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// Infinities and NaN as zeros: of 16-bit values, of E4M3 codes.
template <int TYPE>
__device__ __forceinline__ U32x4 Finite(U32x4 w) {
  constexpr uint32_t kExponent = TYPE == LLMP_X_BF16 ? 0x7F80u : 0x7C00u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] &= (w[i] & kExponent) == kExponent ? 0xFFFF0000u : ~0u;
    w[i] &= (w[i] >> 16 & kExponent) == kExponent ? 0x0000FFFFu : ~0u;
  }
  return w;
}
__device__ __forceinline__ U32x4 FiniteCodes(U32x4 w) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i / 4] &= (w[i / 4] >> (8 * (i & 3)) & 0x7Fu) == 0x7Fu ? ~(0xFFu << (8 * (i & 3))) : ~0u;
  return w;
}

// A scalar address and a 32-bit lane offset; the lanes' 16 (4) bytes go to LDS one after the other from byte `to` on. Written as an instruction:
// the compiler, which knows the builtin's write to LDS, waits for it before every later read of LDS. A wait of the caller's own stands before what landed is read.
__device__ __forceinline__ void LineToLds(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void WordToLds(const void* base, uint32_t offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory", "m0");
}
// ... from an address of each lane's own.
__device__ __forceinline__ void LaneLineToLds(const void* from, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
template <int LEFT>
__device__ __forceinline__ void WaitLoads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
// A row of COUNT products whose operands come from LDS, in groups: a group's reads stand before the products of the group before it. (Left to itself the
// compiler saves registers, reads for one product at a time and waits for it: about 130 cycles a product of 32.) read(i) gives product i's operand,
// multiply(i, operand) makes it.
template <int COUNT, int GROUP, class Eight, class Read, class Multiply>
__device__ __forceinline__ void ProductsInGroups(const Read& read, const Multiply& multiply) {
  Eight held[2][GROUP];
#pragma unroll
  for (int i = 0; i < GROUP && i < COUNT; ++i) held[0][i] = read(i);
#pragma unroll
  for (int g = 0; g * GROUP < COUNT; ++g) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < GROUP; ++i) {
      if ((g + 1) * GROUP + i < COUNT) held[(g + 1) & 1][i] = read((g + 1) * GROUP + i);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < GROUP; ++i) {
      if (g * GROUP + i < COUNT) multiply(g * GROUP + i, held[g & 1][i]);
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}
// All the wave's reads of LDS have been answered, and every wave of the workgroup is here.
__device__ __forceinline__ void MeetLds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A column of four 16-bit values, one of each of four rows: lane i of 16 gives the address of row i / 4's values 4 (i % 4) to 4 (i % 4) + 3 and
// gets column i. Of eight bytes: row i / 2's 8 (i % 2) to 8 (i % 2) + 7.
typedef short S16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ S16x4 Column4(const uint8_t* at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) S16x4*>(reinterpret_cast<uintptr_t>(at)));
}
__device__ __forceinline__ I32x2 Column8(const uint8_t* at) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32(reinterpret_cast<__attribute__((address_space(3))) I32x2*>(reinterpret_cast<uintptr_t>(at)));
}
template <class Eight>
__device__ __forceinline__ Eight JoinFours(S16x4 a, S16x4 b) {
  typedef short S16x8 __attribute__((ext_vector_type(8)));
  return __builtin_bit_cast(Eight, S16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

}  // namespace llmp_hip

#endif  // LLMP_AMD_CSRC_LATENT_H_
