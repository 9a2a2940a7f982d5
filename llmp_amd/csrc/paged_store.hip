// llmp.paged.store and llmp.paged.read: new K and V rows into the pages of the 8-bit cache, and pages back as values.
//
// A scale belongs to a page and a KV head, so a workgroup takes one (page, head) of K or of V: the new rows' largest magnitude,
// the scale it makes with the one the page has, the held codes rounded again if the scale rises, the new codes. Rows are
// read twice (the second time from the caches); each code is written once. Every page is one workgroup's, so nothing is
// ordered by atomics. V's codes lie with the tokens innermost: a workgroup turns them through LDS and writes 16 tokens of
// a dimension at a time, the bytes of other tokens among them kept as they are.
//
// A scale is F32(largest magnitude * F32(1 / 127)), a code the nearest to the IEEE quotient value / scale: single roundings, so
// that the definition is the same in any program, bit for bit.
//
// Measured: a decode step of 63 tokens, 8 KV heads of 128, 5.8 us, the chain of item, rows, barrier and codes; prompts of 3139 tokens,
// 8 heads of 256 in F16, 18.8 us for 39 MB, 2.1 TB/s (the chain again, with every workgroup on the device at once: rows kept in
// registers, four a thread, took 20.0 us and the decode step 8.6, with code for four rows' divisions where one row is). Reading 13 MB of
// codes back as 27 MB of F16 values 8.6 us, 4.7 TB/s; 8 MB as 17 MB of BF16 8.2 us, 3.0 TB/s, its launch and chain being most of it.
#include "paged.h"

namespace llmp_hip {
namespace {

constexpr int kStoreThreads = 256;

struct StoreItem {
  int page, row, held, count;
};

// The item if it fits the cache and the rows.
__device__ __forceinline__ bool ItemOf(const int32_t* work, int index, int pages, int page, int tokens, StoreItem* item) {
  const I32x4 w = *reinterpret_cast<const I32x4*>(work + 4 * static_cast<int64_t>(index));
  item->page = w.x, item->row = w.y, item->held = w.z, item->count = w.w;
  return w.x >= 0 && w.x < pages && w.w >= 1 && w.z >= 0 && w.w <= page && w.z <= page - w.w && w.y >= 0 && w.w <= tokens && w.y <= tokens - w.w;
}

__device__ __forceinline__ float BlockMax(float v, float* shared) {
#pragma unroll
  for (int step = 1; step < kWave; step <<= 1) v = fmaxf(v, __shfl_xor(v, step));
  if ((threadIdx.x & (kWave - 1)) == 0) shared[threadIdx.x / kWave] = v;
  __syncthreads();
  float all = shared[0];
#pragma unroll
  for (int w = 1; w < kStoreThreads / kWave; ++w) all = fmaxf(all, shared[w]);
  return all;
}

// A held code's at a higher scale (`factor`, the old scale over the new).
__device__ __forceinline__ int CodeAgain(int code, float factor) { return static_cast<int>(rintf(static_cast<float>(code) * factor)); }
__device__ __forceinline__ int ByteOf(uint32_t word, int i) { return static_cast<int8_t>(word >> (8 * i)); }

__device__ __forceinline__ uint32_t WordAgain(uint32_t word, float factor) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) out |= static_cast<uint32_t>(CodeAgain(ByteOf(word, i), factor) & 0xFF) << (8 * i);
  return out;
}

// The largest finite magnitude of the item's rows of this head.
template <int TYPE, int D>
__device__ __forceinline__ float RowsMax(const void* x, int64_t first, int64_t token_stride, int count) {
  constexpr int kLanes = D / 8, kRows = kStoreThreads / kLanes;  // lanes a row, rows a sweep
  float most = 0.0f;
#pragma unroll 4
  for (int i = threadIdx.x / kLanes; i < count; i += kRows) {
    float v[8];
    LoadEight<TYPE>(x, first + i * token_stride + 8 * (threadIdx.x % kLanes), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float size = fabsf(v[e]);
      if (size <= 3.402823466e38f) most = fmaxf(most, size);  // (neither infinities nor NaN)
    }
  }
  return most;
}

// grid (work items, KV heads, 2: K and V).
template <int TYPE, int D>
__global__ __launch_bounds__(kStoreThreads) void StoreKernel(const llmp_paged_store op) {
  constexpr int kLanes = D / 8, kRows = kStoreThreads / kLanes;
  extern __shared__ __attribute__((aligned(16))) uint8_t turned[];  // V: [D][pitch] codes, a dimension's tokens together
  __shared__ float shared[kStoreThreads / kWave];
  __shared__ int edges[2][D];
  const llmp_paged_cache& c = op.cache;
  const int tid = threadIdx.x, head = blockIdx.y;
  const bool values = blockIdx.z != 0;
  StoreItem it;
  if (!ItemOf(op.work, blockIdx.x, c.pages, c.page, op.tokens, &it)) return;
  const void* x = values ? op.v : op.k;
  const int64_t token_stride = values ? op.v_token_stride : op.k_token_stride;
  const int64_t first = it.row * token_stride + head * (values ? op.v_head_stride : op.k_head_stride);
  const int64_t page_head = static_cast<int64_t>(it.page) * c.kv_heads + head;
  float* const scale_at = (values ? c.v_scale : c.k_scale) + page_head;
  if (!values && tid < D) edges[0][tid] = 127, edges[1][tid] = -127;

  const float before = it.held > 0 ? *scale_at : 0.0f;
  const float most = BlockMax(RowsMax<TYPE, D>(x, first, token_stride, it.count), shared);  // (its barrier: every thread has read *scale_at)
  const float scale = fmaxf(before, most * (1.0f / 127.0f));
  const bool rises = it.held > 0 && scale > before;
  const float factor = rises ? before / scale : 1.0f, inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
  if (tid == 0) *scale_at = scale;

  const int d0 = 8 * (tid % kLanes);
  if (!values) {
    uint8_t* const codes = static_cast<uint8_t*>(c.k) + page_head * c.page * D;
    if (rises) {
      for (int i = tid / kLanes; i < it.held; i += kRows) {
        uint2* at = reinterpret_cast<uint2*>(codes + i * D + d0);
        const uint2 w = *at;
        *at = make_uint2(WordAgain(w.x, factor), WordAgain(w.y, factor));
      }
    }
    int low[8], high[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) low[e] = 127, high[e] = -127;
    for (int i = tid / kLanes; i < it.count; i += kRows) {
      float v[8];
      LoadEight<TYPE>(x, first + i * token_stride + d0, v);
      int code[8];
      CodesOf(v, scale, inverse, code);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        low[e] = min(low[e], code[e]), high[e] = max(high[e], code[e]);
        w[e / 4] |= static_cast<uint32_t>(code[e] & 0xFF) << (8 * (e % 4));
      }
      *reinterpret_cast<uint2*>(codes + (it.held + i) * D + d0) = make_uint2(w[0], w[1]);
    }
    if (c.low == nullptr) return;
    if (tid / kLanes < it.count) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // (whole numbers' least and most: the order of the atomics does not matter)
        atomicMin(&edges[0][d0 + e], low[e]);
        atomicMax(&edges[1][d0 + e], high[e]);
      }
    }
    __syncthreads();
    if (tid < D) {
      int8_t* const low_at = static_cast<int8_t*>(c.low) + page_head * D + tid;
      int8_t* const high_at = static_cast<int8_t*>(c.high) + page_head * D + tid;
      int least = edges[0][tid], largest = edges[1][tid];
      // (Rounding to a higher scale keeps the order: the edges of the codes rounded again are the edges, rounded again.)
      if (it.held > 0) least = min(least, CodeAgain(*low_at, factor)), largest = max(largest, CodeAgain(*high_at, factor));
      *low_at = static_cast<int8_t>(least);
      *high_at = static_cast<int8_t>(largest);
    }
    return;
  }
  // V: the new codes to LDS, a dimension's 16-token pieces whole; then piece by piece into the page.
  const int pitch = c.page + 4;  // (four bytes on: a token's lanes write dimensions eight apart, 8 * pitch bytes, which are eight banks at every page size)
  for (int i = tid / kLanes; i < it.count; i += kRows) {
    float v[8];
    LoadEight<TYPE>(x, first + i * token_stride + d0, v);
    int code[8];
    CodesOf(v, scale, inverse, code);
#pragma unroll
    for (int e = 0; e < 8; ++e) turned[(d0 + e) * pitch + it.held + i] = static_cast<uint8_t>(code[e]);
  }
  __syncthreads();
  uint8_t* const codes = static_cast<uint8_t*>(c.v) + page_head * c.page * D;
  const int end = it.held + it.count;
  const int piece0 = rises ? 0 : it.held / 16, pieces = (end + 15) / 16 - piece0;
  for (int i = tid; i < D * pieces; i += kStoreThreads) {
    const int d = i / pieces, t0 = 16 * (piece0 + i % pieces);
    U32x4* at = reinterpret_cast<U32x4*>(codes + d * c.page + t0);
    U32x4 w = {0, 0, 0, 0};
    if (t0 < it.held || t0 + 16 > end) w = *at;  // tokens of it stay, or lie past the new ones
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t fresh = *reinterpret_cast<const uint32_t*>(turned + d * pitch + t0 + 4 * j);
      uint32_t word = w[j];
      const int t = t0 + 4 * j;
      if (rises && t < it.held) {
        const uint32_t again = WordAgain(word, factor);
        const int n = min(it.held - t, 4);
        const uint32_t mask = n == 4 ? ~0u : (1u << (8 * n)) - 1u;
        word = (word & ~mask) | (again & mask);
      }
      uint32_t mask = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) mask |= t + b >= it.held && t + b < end ? 0xFFu << (8 * b) : 0u;
      w[j] = (word & ~mask) | (fresh & mask);
    }
    *at = w;
  }
}

// grid (pages asked for, KV heads, 2: K and V): a page's codes of a head times its scale.
template <int TYPE, int D>
__global__ __launch_bounds__(kStoreThreads) void ReadKernel(const llmp_paged_cache c, const int32_t* pages, int64_t page_stride, void* k_out, void* v_out) {
  extern __shared__ __attribute__((aligned(16))) uint8_t turned[];  // V: [page][D + 4] codes, a token's dimensions together
  const int tid = threadIdx.x, head = blockIdx.y;
  const bool values = blockIdx.z != 0;
  const int at = pages[blockIdx.x * page_stride];
  const bool real = at >= 0 && at < c.pages;
  const int64_t page_head = real ? static_cast<int64_t>(at) * c.kv_heads + head : 0;
  const float scale = real ? (values ? c.v_scale : c.k_scale)[page_head] : 0.0f;
  const uint8_t* const codes = static_cast<const uint8_t*>(values ? c.v : c.k) + page_head * c.page * D;
  const int64_t out = (static_cast<int64_t>(blockIdx.x) * c.kv_heads + head) * c.page * D;
  constexpr int kPitch = D + 4;
  if (values) {
    for (int i = tid; i < D * c.page / 16; i += kStoreThreads) {
      const int d = i / (c.page / 16), t0 = 16 * (i % (c.page / 16));
      const U32x4 w = *reinterpret_cast<const U32x4*>(codes + d * c.page + t0);
#pragma unroll
      for (int j = 0; j < 16; ++j) turned[(t0 + j) * kPitch + d] = static_cast<uint8_t>(w[j / 4] >> (8 * (j % 4)));
    }
    __syncthreads();
  }
  for (int i = tid; i < D * c.page / 8; i += kStoreThreads) {
    const int t = i / (D / 8), d0 = 8 * (i % (D / 8));
    const uint32_t* from = reinterpret_cast<const uint32_t*>(values ? turned + t * kPitch + d0 : codes + t * D + d0);
    const uint32_t w[2] = {from[0], from[1]};
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = real ? static_cast<float>(ByteOf(w[e / 4], e % 4)) * scale : 0.0f;
      // (A value is the F32 product; without this the compiler rounds the product itself to F16 in one instruction.)
      if constexpr (TYPE == LLMP_X_F16) asm("" : "+v"(v[e]));
    }
    StoreValues<TYPE, 8>(values ? v_out : k_out, out + t * D + d0, v);
  }
}

template <int TYPE, int D>
void LaunchStore(const llmp_paged_store& op, hipStream_t stream) {
  const int lds = D * (op.cache.page + 4);
  static bool sized = false;
  if (lds > 32768 && !AllowLds(reinterpret_cast<const void*>(&StoreKernel<TYPE, D>), D * (256 + 4), &sized)) return;
  hipLaunchKernelGGL((StoreKernel<TYPE, D>), dim3(op.work_items, op.cache.kv_heads, 2), dim3(kStoreThreads), lds, stream, op);
}
template <int TYPE, int D>
void LaunchRead(const llmp_paged_cache& c, const int32_t* pages, int64_t page_stride, int count, void* k_out, void* v_out, hipStream_t stream) {
  const int lds = (D + 4) * c.page;
  static bool sized = false;
  if (lds > 32768 && !AllowLds(reinterpret_cast<const void*>(&ReadKernel<TYPE, D>), (D + 4) * 256, &sized)) return;
  hipLaunchKernelGGL((ReadKernel<TYPE, D>), dim3(count, c.kv_heads, 2), dim3(kStoreThreads), lds, stream, c, pages, page_stride, k_out, v_out);
}

// f with the type and the head size as constants.
template <class F>
void WithTypeAndHead(int type, int head_dim, F&& f) {
  const auto with_head = [&](auto t) {
    if (head_dim == 64) f(t, std::integral_constant<int, 64>{});
    if (head_dim == 128) f(t, std::integral_constant<int, 128>{});
    if (head_dim == 256) f(t, std::integral_constant<int, 256>{});
  };
  if (type == LLMP_X_F32) with_head(std::integral_constant<int, LLMP_X_F32>{});
  if (type == LLMP_X_BF16) with_head(std::integral_constant<int, LLMP_X_BF16>{});
  if (type == LLMP_X_F16) with_head(std::integral_constant<int, LLMP_X_F16>{});
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" int llmp_hip_paged_store(const llmp_paged_store* op, void* stream) {
  if (op == nullptr) return Refuse(1, "paged_store: null operands");
  if (const int bad = CheckPagedCache("paged_store", op->cache, false); bad != 0) return bad;
  if (op->tokens < 0 || op->work_items < 0) return Refuse(1, "paged_store: tokens %d, work items %d", op->tokens, op->work_items);
  if (op->tokens == 0 || op->work_items == 0) return 0;
  if (const int bad = CheckPagedRows("paged_store", "k", op->k, op->tokens, op->cache.kv_heads, op->k_token_stride, op->k_head_stride, op->type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_store", "v", op->v, op->tokens, op->cache.kv_heads, op->v_token_stride, op->v_head_stride, op->type); bad != 0) return bad;
  if (op->work == nullptr || reinterpret_cast<uintptr_t>(op->work) % 16 != 0) return Refuse(1, "paged_store: work items at a 16-byte boundary");
  BeginLaunches();
  WithTypeAndHead(op->type, op->cache.head_dim, [&](auto type, auto head) { LaunchStore<decltype(type)::value, decltype(head)::value>(*op, static_cast<hipStream_t>(stream)); });
  return LaunchStatus("paged_store");
}

extern "C" int llmp_hip_paged_read(const llmp_paged_cache* cache, const int32_t* pages, int64_t page_stride, int count, int type, void* k_out, void* v_out,
                                   void* stream) {
  if (cache == nullptr) return Refuse(1, "paged_read: null operands");
  if (const int bad = CheckPagedCache("paged_read", *cache, false); bad != 0) return bad;
  if (count < 0 || page_stride < 0) return Refuse(1, "paged_read: %d pages every %lld", count, (long long)page_stride);
  if (count == 0) return 0;
  if (pages == nullptr || reinterpret_cast<uintptr_t>(pages) % 4 != 0) return Refuse(1, "paged_read: page numbers at a 4-byte boundary");
  if (const int bad = CheckPagedRows("paged_read", "k_out", k_out, 1, 1, 0, 0, type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_read", "v_out", v_out, 1, 1, 0, 0, type); bad != 0) return bad;
  BeginLaunches();
  WithTypeAndHead(type, cache->head_dim, [&](auto t, auto head) {
    LaunchRead<decltype(t)::value, decltype(head)::value>(*cache, pages, page_stride, count, k_out, v_out, static_cast<hipStream_t>(stream));
  });
  return LaunchStatus("paged_read");
}
