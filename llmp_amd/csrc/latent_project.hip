// llmp.latent.project: every head's rows times that head's matrix, y = x W^T.
//
// With few tokens what bounds it is the matrices' bytes, each read once; with many the rows in and out, for the products' inner
// index is short (128 to 512). A workgroup of four waves takes 128 of a head's outputs and 32 or 128 tokens; 64 of the inner index
// at a time go through LDS, the next under this one's products, rows of 128 bytes in pieces turned so that the 16 lanes that a 16-byte read
// takes at once find them in all banks (KPiece in paged_attend.h says which lanes). The products are W X^T, so that a lane ends with four
// outputs of one token side by side; the tile goes back through LDS and out by whole rows. (64 tokens, 128 heads of 128 to 512: 7.8 us, 3.5 TB/s; 2001
// tokens, 32 heads of 512 to 128: 17.5 us, 4.9 TB/s. 32 tokens a workgroup up to 64 tokens, so that the matrices' reads are spread over all units; 128 beyond, so
// that a matrix is read a sixteenth as often.)
#include "latent.h"

namespace llmp_hip {
namespace {

constexpr int kProjectThreads = 256, kInnerBytes = 128;  // 64 values

__device__ __forceinline__ int ProjectPiece(int row, int piece) { return piece ^ ((row >> 1) & 7); }

// TOKENS: of a workgroup. Waves: four by 32 outputs, or two by 64 outputs times two by 64 tokens.
template <int TYPE, int TOKENS>
__global__ __launch_bounds__(kProjectThreads) void ProjectKernel(const llmp_latent_project op) {
  using S = Sixteen<TYPE>;
  constexpr int kOutputs = 128;
  constexpr int kWaveOutputs = TOKENS == 32 ? 32 : 64, kWaveTokens = TOKENS == 32 ? 32 : 64;
  constexpr int kA = kWaveOutputs / 32, kB = kWaveTokens / 32;
  constexpr int kStage = (kOutputs + TOKENS) * kInnerBytes;
  constexpr int kLoads = kStage / 1024 / 4;  // a wave's
  constexpr int kRing = TOKENS == 32 ? 3 : 2;
  constexpr int kOutPitch = kOutputs * 2 + 16;
  static_assert(TOKENS * kOutPitch <= kRing * kStage, "the result's tile fits");
  __shared__ __attribute__((aligned(16))) uint8_t lds[kRing * kStage];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane / 32, column = lane % 32;
  const int n0 = blockIdx.x * kOutputs, head = blockIdx.y, t0 = blockIdx.z * TOKENS;
  const uint16_t* const w = static_cast<const uint16_t*>(op.w) + head * op.w_head_stride;
  const uint16_t* const x = static_cast<const uint16_t*>(op.x) + head * op.x_head_stride;
  const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));

  // A load's eight rows: outputs, then tokens (past the last one: the last).
  const uint16_t* from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = 8 * (wave * kLoads + i) + lane / 8, piece = ProjectPiece(row, lane % 8);
    const bool output = row < kOutputs;
    const int64_t at = output ? static_cast<int64_t>(min(n0 + row, op.n - 1)) * op.w_row_stride
                              : static_cast<int64_t>(min(t0 + row - kOutputs, op.tokens - 1)) * op.x_token_stride;
    from[i] = (output ? w : x) + at + 8 * piece;
  }
  const int steps = (op.k + 63) / 64;
  const auto fetch = [&](int step) {
    const uint32_t to = lds_at + (step % kRing) * kStage + wave * kLoads * 1024;
    // (Pieces past k: those of the step's first half again; their products are not made.)
    const int back = op.k - 64 * step < 64 ? 32 : 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = 8 * (wave * kLoads + i) + lane / 8;
      LaneLineToLds(from[i] + 64 * step - (ProjectPiece(row, lane % 8) >= 4 ? back : 0), to + 1024 * i);
    }
  };
  F32x16 sums[kA][kB];
#pragma unroll
  for (int a = 0; a < kA; ++a) {
#pragma unroll
    for (int b = 0; b < kB; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[a][b][i] = 0.0f;
    }
  }
  const int first_output = TOKENS == 32 ? 32 * wave : 64 * (wave % 2), first_token = TOKENS == 32 ? 0 : 64 * (wave / 2);
  for (int step = 0; step < kRing - 1 && step < steps; ++step) fetch(step);
  for (int step = 0; step < steps; ++step) {
    if (kRing == 3 && step + 1 < steps) {
      WaitLoads<kLoads>();
    } else {
      WaitLoads<0>();
    }
    MeetLds();
    if (step + kRing - 1 < steps) fetch(step + kRing - 1);
    const uint8_t* const stage = lds + (step % kRing) * kStage;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s == 2 && op.k - 64 * step < 64) break;
      typename S::Eight a[kA], b[kB];
#pragma unroll
      for (int i = 0; i < kA; ++i) {
        const int row = first_output + 32 * i + column;
        a[i] = *reinterpret_cast<const typename S::Eight*>(stage + row * kInnerBytes + 16 * ProjectPiece(row, 2 * s + half));
      }
#pragma unroll
      for (int i = 0; i < kB; ++i) {
        const int row = kOutputs + first_token + 32 * i + column;
        b[i] = *reinterpret_cast<const typename S::Eight*>(stage + row * kInnerBytes + 16 * ProjectPiece(row, 2 * s + half));
      }
#pragma unroll
      for (int i = 0; i < kA; ++i) {
#pragma unroll
        for (int j = 0; j < kB; ++j) sums[i][j] = S::Product32(a[i], b[j], sums[i][j]);
      }
    }
  }
  MeetLds();
  // Element 4a + b of a lane is output 8a + 4 half + b of its block.
#pragma unroll
  for (int i = 0; i < kA; ++i) {
#pragma unroll
    for (int j = 0; j < kB; ++j) {
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const float v[4] = {sums[i][j][4 * a], sums[i][j][4 * a + 1], sums[i][j][4 * a + 2], sums[i][j][4 * a + 3]};
        StoreValues<TYPE, 4>(lds + (first_token + 32 * j + column) * kOutPitch, first_output + 32 * i + 8 * a + 4 * half, v);
      }
    }
  }
  MeetLds();
  uint16_t* const y = static_cast<uint16_t*>(op.y) + head * op.y_head_stride;
  for (int i = tid; i < TOKENS * 16; i += kProjectThreads) {
    const int t = i / 16, n = 8 * (i % 16);
    if (t0 + t < op.tokens && n0 + n < op.n)
      *reinterpret_cast<U32x4*>(y + (t0 + t) * op.y_token_stride + n0 + n) = *reinterpret_cast<const U32x4*>(lds + t * kOutPitch + 2 * n);
  }
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" int llmp_hip_latent_project(const llmp_latent_project* op, void* stream) {
  if (op == nullptr) return Refuse(1, "latent_project: null operands");
  if (op->type != LLMP_X_BF16 && op->type != LLMP_X_F16) return Refuse(1, "latent_project: BF16 or F16 values, not type %d", op->type);
  if (op->k < 32 || op->n < 32 || op->k % 32 != 0 || op->n % 32 != 0 || op->k > 65536 || op->n > 65536)
    return Refuse(1, "latent_project: matrices of %d times %d (multiples of 32 up to 65536)", op->n, op->k);
  if (op->heads < 1 || op->heads > 65535 || op->tokens < 0) return Refuse(1, "latent_project: %d heads, %d tokens", op->heads, op->tokens);
  if (op->tokens == 0) return 0;
  if (const int bad = CheckPagedRows("latent_project", "x", op->x, op->tokens, op->heads, op->x_token_stride, op->x_head_stride, op->type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("latent_project", "w", op->w, op->n, op->heads, op->w_row_stride, op->w_head_stride, op->type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("latent_project", "y", op->y, op->tokens, op->heads, op->y_token_stride, op->y_head_stride, op->type); bad != 0) return bad;
  const auto s = static_cast<hipStream_t>(stream);
  const unsigned outputs = (op->n + 127) / 128;
  const int64_t groups = op->tokens <= 64 ? (op->tokens + 31) / 32 : (op->tokens + 127) / 128;
  if (groups > 65535) return Refuse(1, "latent_project: %d tokens", op->tokens);
  const dim3 grid(outputs, op->heads, static_cast<unsigned>(groups));
  BeginLaunches();
  const auto launch = [&](auto type) {
    constexpr int kType = decltype(type)::value;
    if (op->tokens <= 64) hipLaunchKernelGGL((ProjectKernel<kType, 32>), grid, dim3(kProjectThreads), 0, s, *op);
    if (op->tokens > 64) hipLaunchKernelGGL((ProjectKernel<kType, 128>), grid, dim3(kProjectThreads), 0, s, *op);
  };
  if (op->type == LLMP_X_BF16) launch(std::integral_constant<int, LLMP_X_BF16>{});
  if (op->type == LLMP_X_F16) launch(std::integral_constant<int, LLMP_X_F16>{});
  return LaunchStatus("latent_project");
}
