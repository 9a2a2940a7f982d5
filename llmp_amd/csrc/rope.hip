// llmp.rope: part of every head's channels rotated by the token's position.
//
// What bounds it is memory: a value is read and written once, for about three operations. A token's cosines and sines are the same for
// all its heads, so a workgroup makes them once in LDS (a thread a pair; about 30 operations each) and goes over the heads of its
// tokens 16 bytes at a time: eight channels and the eight that they turn with. (8192 tokens of 32 heads of 128: 21.4 us, 6.3 TB/s, for part of what is read is
// still in the last cache; 64 tokens in place 3.5 us.)
#include <algorithm>
#include <cmath>

#include "paged.h"
#include "rope.h"

namespace llmp_hip {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMostPairs = 512;  // of a head: n_dims up to 1024
constexpr int kMostTokens = (1 << 24) - 1;  // a call's: a grid has less than 2^32 threads

struct RopeArgs {
  llmp_rope op;
  int tokens_a_group;  // of a workgroup
  int heads_a_group;
  bool copies;  // channels outside the rotation go from x to out
};

template <int TYPE, int N>
__device__ __forceinline__ void LoadSome(const void* base, int64_t element, float (&x)[N]) {
  if constexpr (N == 8) {
    LoadEight<TYPE>(base, element, x);
  } else {
    x[0] = LoadOne<TYPE>(base, element);
  }
}
template <int TYPE, int N>
__device__ __forceinline__ void StoreSome(void* base, int64_t element, const float (&x)[N]) {
  if constexpr (N == 8) {
    StoreValues<TYPE, 8>(base, element, x);
  } else {
    StoreOne<TYPE>(base, element, x[0]);
  }
}

// grid (token groups, head groups). N: channels a step, 8 where everything lies at their boundaries, else 1.
template <int TYPE, int N, bool INTERLEAVED>
__global__ __launch_bounds__(kRopeThreads) void RopeKernel(const RopeArgs a) {
  __shared__ float2 turned[kMostPairs];
  const llmp_rope& op = a.op;
  const int tid = threadIdx.x, pairs = op.n_dims / 2;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.tokens_a_group;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(a.tokens_a_group), op.tokens - token0));
  const int head0 = blockIdx.y * a.heads_a_group, heads = min(a.heads_a_group, op.heads - head0);
  for (int i = tid; i < tokens * pairs; i += kRopeThreads) {
    const int t = i / pairs, p = i - t * pairs;
    float c, s;
    Turn(op.turns[p], op.positions[token0 + t], &c, &s);
    turned[i] = make_float2(c * op.magnitude, (op.inverse ? -s : s) * op.magnitude);
  }
  __syncthreads();
  // A head's work items: N pairs each, then the channels that stay.
  const int turns = pairs / N, stays = a.copies ? (op.head_dim - op.n_dims) / N : 0, items = turns + stays;
  for (int i = tid; i < tokens * heads * items; i += kRopeThreads) {
    const int row = i / items, item = i - row * items;
    const int t = row / heads, h = head0 + row - t * heads;
    const int64_t from = (token0 + t) * op.x_token_stride + h * op.x_head_stride, to = (token0 + t) * op.out_token_stride + h * op.out_head_stride;
    if (item >= turns) {
      int c = (item - turns) * N;
      c += c >= op.first ? op.n_dims : 0;
      float v[N];
      LoadSome<TYPE>(op.x, from + c, v);
      StoreSome<TYPE>(op.out, to + c, v);
      continue;
    }
    const int p0 = item * N;
    const int ca = op.first + (INTERLEAVED ? 2 * p0 : p0), cb = INTERLEAVED ? ca + N : ca + pairs;
    float va[N], vb[N];
    LoadSome<TYPE>(op.x, from + ca, va);
    LoadSome<TYPE>(op.x, from + cb, vb);
    const float2* const by = turned + t * pairs + p0;
    if constexpr (INTERLEAVED && N == 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 r = by[j], q = by[4 + j];
        const float x0 = va[2 * j], y0 = va[2 * j + 1], x1 = vb[2 * j], y1 = vb[2 * j + 1];
        va[2 * j] = x0 * r.x - y0 * r.y, va[2 * j + 1] = x0 * r.y + y0 * r.x;
        vb[2 * j] = x1 * q.x - y1 * q.y, vb[2 * j + 1] = x1 * q.y + y1 * q.x;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 r = by[j];
        const float x = va[j], y = vb[j];
        va[j] = x * r.x - y * r.y, vb[j] = x * r.y + y * r.x;
      }
    }
    StoreSome<TYPE>(op.out, to + ca, va);
    StoreSome<TYPE>(op.out, to + cb, vb);
  }
}

template <int TYPE>
void LaunchRope(const RopeArgs& a, bool wide, dim3 grid, hipStream_t stream) {
  const bool between = a.op.interleaved != 0;
  if (wide) {
    if (between) hipLaunchKernelGGL((RopeKernel<TYPE, 8, true>), grid, dim3(kRopeThreads), 0, stream, a);
    if (!between) hipLaunchKernelGGL((RopeKernel<TYPE, 8, false>), grid, dim3(kRopeThreads), 0, stream, a);
  } else {
    if (between) hipLaunchKernelGGL((RopeKernel<TYPE, 1, true>), grid, dim3(kRopeThreads), 0, stream, a);
    if (!between) hipLaunchKernelGGL((RopeKernel<TYPE, 1, false>), grid, dim3(kRopeThreads), 0, stream, a);
  }
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" int llmp_hip_rope_table(int n_dims, double base, double freq_scale, double ext_factor, double corr_low, double corr_high,
                                   const float* freq_factors, uint64_t* turns) {
  if (turns == nullptr) return Refuse(1, "rope_table: null operand");
  if (n_dims <= 0 || n_dims % 2 != 0 || n_dims > 2 * kMostPairs) return Refuse(1, "rope_table: %d channels (an even number up to %d)", n_dims, 2 * kMostPairs);
  if (!(base > 0.0) || !std::isfinite(base) || !std::isfinite(freq_scale) || !std::isfinite(ext_factor) || !std::isfinite(corr_low) || !std::isfinite(corr_high)) {
    return Refuse(1, "rope_table: a positive base and finite factors");
  }
  for (int p = 0; p < n_dims / 2; ++p) {
    const double factor = freq_factors != nullptr ? freq_factors[p] : 1.0;
    if (!(std::fabs(factor) > 0.0) || !std::isfinite(factor)) return Refuse(1, "rope_table: frequency factor %d is %g", p, factor);
    const double far = std::pow(base, -2.0 * p / n_dims) / factor;
    double f = far * freq_scale;
    if (ext_factor != 0.0) {
      const double at = (p - corr_low) / std::fmax(0.001, corr_high - corr_low);
      const double mix = (1.0 - std::fmin(1.0, std::fmax(0.0, at))) * ext_factor;
      f = f * (1.0 - mix) + far * mix;
    }
    if (!(std::fabs(f) < 0x1p32)) return Refuse(1, "rope_table: frequency %d is %g", p, f);
    const double part = f / (2.0 * M_PI) - std::floor(f / (2.0 * M_PI));  // in [0, 1]: whole turns do nothing
    const double high = std::floor(part * 0x1p32), low = std::floor((part * 0x1p32 - high) * 0x1p32);
    turns[p] = (static_cast<uint64_t>(high) << 32) + static_cast<uint64_t>(low);
  }
  return 0;
}

extern "C" int llmp_hip_rope(const llmp_rope* op, void* stream) {
  if (op == nullptr) return Refuse(1, "rope: null operands");
  if (op->type != LLMP_X_F32 && op->type != LLMP_X_BF16 && op->type != LLMP_X_F16) return Refuse(1, "rope: element type %d", op->type);
  if (op->tokens < 0 || op->tokens > kMostTokens || op->heads <= 0 || op->heads > 65535) return Refuse(1, "rope: %lld tokens, %d heads", (long long)op->tokens, op->heads);
  if (op->head_dim <= 0 || op->head_dim > 65536 || op->n_dims <= 0 || op->n_dims % 2 != 0 || op->n_dims > 2 * kMostPairs || op->first < 0 ||
      op->first + op->n_dims > op->head_dim) {
    return Refuse(1, "rope: channels %d to %d of %d (an even number up to %d)", op->first, op->first + op->n_dims, op->head_dim, 2 * kMostPairs);
  }
  if (!std::isfinite(op->magnitude)) return Refuse(1, "rope: a magnitude that is not finite");
  if (op->tokens == 0) return 0;
  if (op->x == nullptr || op->out == nullptr || op->positions == nullptr || op->turns == nullptr) return Refuse(1, "rope: null operand");
  const int64_t element = PagedElementBytes(op->type);
  if (reinterpret_cast<uintptr_t>(op->x) % element != 0 || reinterpret_cast<uintptr_t>(op->out) % element != 0 ||
      reinterpret_cast<uintptr_t>(op->positions) % 4 != 0 || reinterpret_cast<uintptr_t>(op->turns) % 8 != 0) {
    return Refuse(1, "rope: operands at their elements' boundaries");
  }
  const bool same_strides = (op->tokens == 1 || op->x_token_stride == op->out_token_stride) && (op->heads == 1 || op->x_head_stride == op->out_head_stride);
  if (op->x == op->out && !same_strides) return Refuse(1, "rope: in place with other strides");
  RopeArgs a = {*op, 1, 1, op->x != op->out};
  const int64_t bounds = reinterpret_cast<uintptr_t>(op->x) | reinterpret_cast<uintptr_t>(op->out) |
                         (op->tokens > 1 ? (op->x_token_stride | op->out_token_stride) * element : 0) |
                         (op->heads > 1 ? (op->x_head_stride | op->out_head_stride) * element : 0);
  const bool wide = op->head_dim % 8 == 0 && op->first % 8 == 0 && op->n_dims % 16 == 0 && bounds % 16 == 0;
  // Tokens side by side as the table in LDS has room for, but 1024 workgroups where the call has the work for them; with few tokens
  // the heads are dealt out too, down to a workgroup's own threads' worth.
  const int pairs = op->n_dims / 2, fit = std::max(1, kRopeThreads / pairs);
  a.tokens_a_group = static_cast<int>(std::min<int64_t>(fit, std::max<int64_t>(1, op->tokens / 1024)));
  const int64_t groups = (op->tokens + a.tokens_a_group - 1) / a.tokens_a_group;
  const int items = (op->head_dim - (a.copies ? 0 : op->head_dim - op->n_dims)) / (wide ? 8 : 1);
  const int least = std::max(1, kRopeThreads / std::max(1, items));
  a.heads_a_group = static_cast<int>(std::min<int64_t>(op->heads, std::max<int64_t>(least, op->heads * groups / 1024)));
  a.heads_a_group = std::max(1, std::min(a.heads_a_group, (1 << 22) / (a.tokens_a_group * max(1, items))));  // (a workgroup's items in an int)
  const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>((op->heads + a.heads_a_group - 1) / a.heads_a_group));
  BeginLaunches();
  const auto s = static_cast<hipStream_t>(stream);
  if (op->type == LLMP_X_F32) LaunchRope<LLMP_X_F32>(a, wide, grid, s);
  if (op->type == LLMP_X_BF16) LaunchRope<LLMP_X_BF16>(a, wide, grid, s);
  if (op->type == LLMP_X_F16) LaunchRope<LLMP_X_F16>(a, wide, grid, s);
  return LaunchStatus("rope");
}
