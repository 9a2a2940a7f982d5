// llmp.latent.store and llmp.latent.read: rows of a token's latent vector and rotated key into and out of the paged latent cache.
//
// A wave takes a token: eight latent values a lane, then the key's pairs one a lane. What bounds both is memory, and for a decode
// step's few rows the chain of a launch, the slot, the row and its sums. (64 rows to codes 3.3 us, back 3.6; 4900 rows of F32 with the normalisation and the
// rotation 4.9 us; 16900 rows back 9.7 us, 4.0 TB/s.)
#include "latent.h"
#include "rope.h"

namespace llmp_hip {

int CheckLatentCache(const char* who, const llmp_latent_cache& c) {
  if (c.latent == nullptr || c.rope == nullptr) return Refuse(1, "%s: null cache", who);
  if (c.type != LLMP_X_BF16 && c.type != LLMP_X_F16) return Refuse(1, "%s: a cache of BF16 or F16 values, not type %d", who, c.type);
  if (c.width != 256 && c.width != 512) return Refuse(1, "%s: latent vectors of 256 or 512 values, not %d", who, c.width);
  if (c.rope_width != 32 && c.rope_width != 64) return Refuse(1, "%s: rotated keys of 32 or 64 values, not %d", who, c.rope_width);
  if (c.page < 16 || c.page > 256 || c.page % 16 != 0) return Refuse(1, "%s: pages of 16 to 256 tokens, a multiple of 16, not %d", who, c.page);
  if (c.pages < 1 || static_cast<int64_t>(c.pages) * c.page > kMostPagedLength) return Refuse(1, "%s: at least one page, at most 2^30 tokens (%d pages)", who, c.pages);
  if ((reinterpret_cast<uintptr_t>(c.latent) | reinterpret_cast<uintptr_t>(c.rope) | reinterpret_cast<uintptr_t>(c.scale)) % 16 != 0)
    return Refuse(1, "%s: the cache's arrays lie at 16-byte boundaries", who);
  return 0;
}

namespace {

constexpr int kRowThreads = 256, kRowWaves = kRowThreads / kWave;
constexpr int kMostRows = 1 << 25;  // a call's: a grid has less than 2^32 threads

__device__ __forceinline__ float WaveSum(float v) {
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) v += ShflXor(v, m);
  return v;
}

// The smallest power of two s = 2^(e - 127) with most <= 448 s (as the product with F32(1 / 448) has it, whose rounding does not
// change it where most is 448 times a power of two).
__device__ __forceinline__ uint32_t ScaleOf(float most) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, most * (1.0f / 448.0f));
  if (bits <= 0x00400000u) return 0;  // 2^-127, a subnormal
  const uint32_t e = (bits >> 23) + ((bits & 0x7FFFFFu) != 0u ? 1u : 0u);
  return min(e, 253u);
}

template <int TYPE, int KEPT>
__global__ __launch_bounds__(kRowThreads) void LatentStoreKernel(const llmp_latent_store op) {
  const llmp_latent_cache& c = op.cache;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRowWaves + threadIdx.x / kWave;
  if (token >= op.tokens) return;
  const int slot = op.slots[token];
  if (slot < 0 || slot >= c.pages * c.page) return;
  const int d0 = 8 * lane;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.0f;
  if (d0 < c.width) LoadEight<TYPE>(op.latent, token * op.latent_stride + d0, v);
  if (op.weight != nullptr) {
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) squares = fmaf(v[i], v[i], squares);
    squares = WaveSum(squares);
    const float by = 1.0f / sqrtf(squares / static_cast<float>(c.width) + op.eps);
    if (d0 < c.width) {
      const F32x4 w0 = *reinterpret_cast<const F32x4*>(op.weight + d0), w1 = *reinterpret_cast<const F32x4*>(op.weight + d0 + 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * by * (i < 4 ? w0[i & 3] : w1[i & 3]);
    }
  }
  if (c.scale != nullptr) {
    // (Magnitudes as bits: infinities are the largest; a NaN is left out of the scale and becomes a NaN.)
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __builtin_isnan(v[i]) ? 0u : __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    const uint32_t e = ScaleOf(__builtin_bit_cast(float, WaveMaxU32(most)));
    const float inverse = __builtin_bit_cast(float, (254u - e) << 23);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = v[4 * i + j] * inverse;
        y[j] = fabsf(y[j]) > 448.0f ? copysignf(448.0f, y[j]) : y[j];  // (the instruction makes a NaN of more)
      }
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], static_cast<int>(w[i]), true);
    }
    if (d0 < c.width) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(c.latent) + static_cast<int64_t>(slot) * c.width + d0) = make_uint2(w[0], w[1]);
    if (lane == 0) static_cast<uint8_t*>(c.scale)[slot] = static_cast<uint8_t>(e);
  } else if (d0 < c.width) {
    StoreValues<KEPT, 8>(c.latent, static_cast<int64_t>(slot) * c.width + d0, v);
  }
  const int pairs = c.rope_width / 2;
  if (lane < pairs) {
    const bool between = op.interleaved != 0;
    const int a = between ? 2 * lane : lane, b = between ? a + 1 : a + pairs;
    const int64_t from = token * op.rope_stride, to = static_cast<int64_t>(slot) * c.rope_width;
    float x = LoadOne<TYPE>(op.rope, from + a), y = LoadOne<TYPE>(op.rope, from + b);
    if (op.turns != nullptr) {
      float cosine, sine;
      Turn(op.turns[lane], op.positions[token], &cosine, &sine);
      cosine *= op.magnitude, sine *= op.magnitude;
      const float z = x * cosine - y * sine;
      y = x * sine + y * cosine;
      x = z;
    }
    StoreOne<KEPT>(c.rope, to + a, x);
    StoreOne<KEPT>(c.rope, to + b, y);
  }
}

// A wave a row; a slot outside the cache gives zeros.
template <int KEPT, int OUT>
__global__ __launch_bounds__(kRowThreads) void LatentReadKernel(const llmp_latent_cache c, const int32_t* slots, int64_t count, void* latent, void* rope) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowWaves + threadIdx.x / kWave;
  if (row >= count) return;
  const int at = slots[row];
  const bool real = at >= 0 && at < c.pages * c.page;
  const int64_t slot = real ? at : 0;
  const int d0 = 8 * lane;
  if (d0 < c.width) {
    float v[8];
    if (c.scale != nullptr) {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(c.latent) + slot * c.width + d0);
      const uint32_t e = static_cast<const uint8_t*>(c.scale)[slot];
      // (2^(e - 127) in two factors: at e = 0 it is a subnormal.)
      const float by = __builtin_bit_cast(float, max(e, 1u) << 23), rest = e == 0 ? 0.5f : 1.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = E4m3ToFloat((i < 4 ? w.x : w.y) >> (8 * (i & 3)) & 0xFFu) * rest * by;
        if constexpr (OUT == LLMP_X_F16) asm("" : "+v"(v[i]));  // (the F32 product is the value: not one rounding of it to F16 by itself)
      }
    } else {
      LoadEight<KEPT>(c.latent, slot * c.width + d0, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = real ? v[i] : 0.0f;
    StoreValues<OUT, 8>(latent, row * c.width + d0, v);
  }
  // The key by the lanes from the last on: at 256 values they are others than the latent's.
  const int r0 = 8 * (kWave - 1 - lane);
  if (r0 < c.rope_width) {
    float v[8];
    LoadEight<KEPT>(c.rope, slot * c.rope_width + r0, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = real ? v[i] : 0.0f;
    StoreValues<OUT, 8>(rope, row * c.rope_width + r0, v);
  }
}

template <class F>
void WithType(int type, F&& f) {
  if (type == LLMP_X_F32) f(std::integral_constant<int, LLMP_X_F32>{});
  if (type == LLMP_X_BF16) f(std::integral_constant<int, LLMP_X_BF16>{});
  if (type == LLMP_X_F16) f(std::integral_constant<int, LLMP_X_F16>{});
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" int llmp_hip_latent_store(const llmp_latent_store* op, void* stream) {
  if (op == nullptr) return Refuse(1, "latent_store: null operands");
  if (const int bad = CheckLatentCache("latent_store", op->cache); bad != 0) return bad;
  if (op->tokens < 0 || op->tokens > kMostRows) return Refuse(1, "latent_store: %d tokens (at most 2^25)", op->tokens);
  if (op->tokens == 0) return 0;
  if (const int bad = CheckPagedRows("latent_store", "latent", op->latent, op->tokens, 1, op->latent_stride, 0, op->type); bad != 0) return bad;
  const int64_t element = PagedElementBytes(op->type);
  if (op->rope == nullptr || op->slots == nullptr) return Refuse(1, "latent_store: null operand");
  if (reinterpret_cast<uintptr_t>(op->rope) % element != 0 || (op->tokens > 1 && op->rope_stride < 0)) return Refuse(1, "latent_store: rope's rows lie at their elements' boundaries");
  if (reinterpret_cast<uintptr_t>(op->slots) % 4 != 0 || reinterpret_cast<uintptr_t>(op->positions) % 4 != 0 || reinterpret_cast<uintptr_t>(op->turns) % 8 != 0)
    return Refuse(1, "latent_store: slots, positions and the table at their elements' boundaries");
  if (op->turns != nullptr && op->positions == nullptr) return Refuse(1, "latent_store: a rotation needs positions");
  if (reinterpret_cast<uintptr_t>(op->weight) % 16 != 0) return Refuse(1, "latent_store: the weight lies at a 16-byte boundary");
  if (op->weight != nullptr && !(op->eps >= 0.0f)) return Refuse(1, "latent_store: eps %g", op->eps);
  BeginLaunches();
  WithType(op->type, [&](auto type) {
    const dim3 grid((op->tokens + kRowWaves - 1) / kRowWaves);
    if (op->cache.type == LLMP_X_BF16) hipLaunchKernelGGL((LatentStoreKernel<decltype(type)::value, LLMP_X_BF16>), grid, dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), *op);
    if (op->cache.type == LLMP_X_F16) hipLaunchKernelGGL((LatentStoreKernel<decltype(type)::value, LLMP_X_F16>), grid, dim3(kRowThreads), 0, static_cast<hipStream_t>(stream), *op);
  });
  return LaunchStatus("latent_store");
}

extern "C" int llmp_hip_latent_read(const llmp_latent_cache* cache, const int32_t* slots, int64_t count, int type, void* latent_out, void* rope_out, void* stream) {
  if (cache == nullptr) return Refuse(1, "latent_read: null operands");
  if (const int bad = CheckLatentCache("latent_read", *cache); bad != 0) return bad;
  if (count < 0 || count > kMostRows) return Refuse(1, "latent_read: %lld rows (at most 2^25)", (long long)count);
  if (count == 0) return 0;
  if (slots == nullptr || reinterpret_cast<uintptr_t>(slots) % 4 != 0) return Refuse(1, "latent_read: slots at a 4-byte boundary");
  if (const int bad = CheckPagedRows("latent_read", "latent_out", latent_out, 1, 1, 0, 0, type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("latent_read", "rope_out", rope_out, 1, 1, 0, 0, type); bad != 0) return bad;
  BeginLaunches();
  WithType(type, [&](auto out) {
    const dim3 grid(static_cast<unsigned>((count + kRowWaves - 1) / kRowWaves));
    const auto s = static_cast<hipStream_t>(stream);
    if (cache->type == LLMP_X_BF16) hipLaunchKernelGGL((LatentReadKernel<LLMP_X_BF16, decltype(out)::value>), grid, dim3(kRowThreads), 0, s, *cache, slots, count, latent_out, rope_out);
    if (cache->type == LLMP_X_F16) hipLaunchKernelGGL((LatentReadKernel<LLMP_X_F16, decltype(out)::value>), grid, dim3(kRowThreads), 0, s, *cache, slots, count, latent_out, rope_out);
  });
  return LaunchStatus("latent_read");
}
