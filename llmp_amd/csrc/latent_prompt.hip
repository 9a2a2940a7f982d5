// llmp.latent.prompt: the expanded form over ragged requests. A head's keys are its own values beside the rotated key that all heads share, so
// that the shared part is read from one place and never copied to the heads.
//
// What bounds it is the matrix instructions (2 * (nope + rope + value) operations a logit) and beside them a softmax's exponential and six operations
// a logit. A workgroup of four waves has 128 rows of one head, 32 a wave, two workgroups a compute unit; 64 keys at a time go through LDS by loads that
// pass no register, the next tile under this one's work:
//   S^T = K Q^T, P = exp2(S - E), O^T += V^T P^T, all by 32 x 32 products.
// Row 8a + 4h + b of the first product is key 16h + 4a + b of its 32, so that a lane (half h) ends with 16 keys in order of one row, which is what the
// second product takes; V's columns come by transposing reads. Where rows are few for the device, the keys are cut in equal runs, and a
// second launch joins them.
#include <algorithm>
#include <cmath>

#include "latent.h"
#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kKeys = 64;  // a tile's
constexpr int kPromptRows = 128, kPromptThreads = 256;
constexpr float kUp = 8.0f, kFollow = 6.0f;  // log2: as in latent_attend.hip
constexpr int kMostRuns = 64;

struct PromptArgs {
  llmp_latent_prompt op;
  float* values;   // [runs][row tiles of all][kPromptRows][value]
  float* numbers;  // [runs][row tiles of all][kPromptRows][2]: maximum, sum
  int tiles;       // row tiles a request, at most
  int runs;        // that a row tile's keys are cut into
};

// A request's rows of q and its keys, none where the arrays name rows outside the call's.
struct PromptRequest {
  int start, n, key_start, keys;
};
__device__ __forceinline__ PromptRequest PromptOf(const llmp_latent_prompt& op, int r) {
  PromptRequest q;
  q.start = op.starts[r];
  const int end = op.starts[r + 1];
  q.n = q.start >= 0 && end > q.start && end <= op.tokens ? end - q.start : 0;
  const int32_t* const keys = op.key_starts != nullptr ? op.key_starts : op.starts;
  q.key_start = keys[r];
  const int key_end = keys[r + 1];
  q.keys = q.key_start >= 0 && key_end > q.key_start && key_end <= op.keys ? key_end - q.key_start : 0;
  return q;
}

// Pieces of 16 bytes of rows of 256, 128 or 64 bytes, turned by the row: for reads of 16 bytes, and for the transposing reads of values.
template <int BYTES>
__device__ __forceinline__ int KeyTurn(int row) {
  if constexpr (BYTES == 256) return (row & 3) << 2 | (row >> 2 & 3);
  if constexpr (BYTES == 128) return (row >> 1 & 1) | (row >> 2 & 3) << 1;
  return row >> 2 & 3;
}
template <int BYTES>
__device__ __forceinline__ int ValueTurn(int row) {
  if constexpr (BYTES == 256) return (row & 3) << 2 | (row >> 2 & 3);
  return (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

template <int N, int P>
struct PromptGeo {
  static constexpr int kKeyPitch = 2 * N, kRopePitch = 2 * P, kValuePitch = 2 * N;
  static constexpr int kKeyBytes = kKeys * kKeyPitch, kRopeBytes = kKeys * kRopePitch, kValueBytes = kKeys * kValuePitch;
  static constexpr int kTile = kKeyBytes + kRopeBytes + kValueBytes;
  static constexpr int kRing = 2;
  static constexpr int kLds = kRing * kTile;
};

// grid: row tiles, requests and heads and runs in an order that keeps a head's row tiles on one chiplet, the longest first.
template <int TYPE, int N, int P>
__global__ __launch_bounds__(kPromptThreads, 2) void LatentPromptKernel(const PromptArgs a) {
  using G = PromptGeo<N, P>;
  using S = Sixteen<TYPE>;
  typedef typename S::Eight Eight;
  constexpr int kSteps = N / 16, kRopeSteps = P / 16, kBlocks = N / 32;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const llmp_latent_prompt& op = a.op;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane / 32, column = lane % 32;
  const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));

  // Eight workgroups in a row go to eight chiplets: a chiplet takes every eighth (run, head, request).
  const uint32_t index = blockIdx.x, turn = index / 8;
  const uint32_t set = turn / a.tiles * 8 + index % 8;
  const int tile_index = a.tiles - 1 - static_cast<int>(turn % a.tiles);
  const uint32_t request_head = set / a.runs;
  const int run = static_cast<int>(set % a.runs);
  if (request_head >= static_cast<uint32_t>(op.requests) * op.heads) return;
  const int request = request_head / op.heads, head = request_head % op.heads;
  const PromptRequest r = PromptOf(op, request);
  const int first = tile_index * kPromptRows;
  if (first >= r.n) return;

  const int row = first + wave * 32 + column;
  const bool real = row < r.n, busy = first + wave * 32 < r.n;
  const int token = real ? row : first;
  const int base = r.keys - r.n;  // the first query's position
  const int see_to = real ? max(base + row + 1, 0) : 0;
  const int all_to = max(base + first + wave * 32 + 1, 0);        // seen by all of the wave's rows
  const int all_rows_to = max(base + first + 1, 0);               // of the workgroup's
  const int any_to = max(base + min(first + kPromptRows, r.n), 0);  // seen by any
  const int tiles = (any_to + kKeys - 1) / kKeys;
  const int tile_from = static_cast<int>(static_cast<int64_t>(tiles) * run / a.runs), tile_to = static_cast<int>(static_cast<int64_t>(tiles) * (run + 1) / a.runs);

  Eight q[kSteps + kRopeSteps];
  {
    const uint32_t flip = op.scale < 0.0f ? 0x80008000u : 0u;  // (a negative scale goes into the queries: the largest product is the largest logit)
    const uint16_t* const from = static_cast<const uint16_t*>(op.q) + static_cast<int64_t>(r.start + token) * op.q_token_stride + head * op.q_head_stride + 8 * half;
#pragma unroll
    for (int x = 0; x < kSteps + kRopeSteps; ++x) {
      U32x4 v = *reinterpret_cast<const U32x4*>(from + 16 * x);
      v ^= U32x4{flip, flip, flip, flip};
      q[x] = __builtin_bit_cast(Eight, v);
    }
  }
  const float worth = fabsf(op.scale) * kLog2E;
  F32x16 out[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) out[b][i] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;

  const auto fetch = [&](int tile, int slot) {
    const uint32_t to = lds_at + slot * G::kTile;
    int lane_now = lane;
    asm volatile("" : "+v"(lane_now));  // (as something new: the compiler otherwise keeps every load's place)
    const auto part = [&](auto pitch, auto is_value, uint32_t area, const void* rows, int64_t stride) {
      constexpr int kPitch = decltype(pitch)::value, kLanes = kPitch / 16, kRowsALoad = kWave / kLanes, kCount = kKeys / kRowsALoad / 4;
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        const int n = wave * kCount + i, in = n * kRowsALoad + lane_now / kLanes;
        const int turned = decltype(is_value)::value ? ValueTurn<kPitch>(in) : KeyTurn<kPitch>(in);
        const int key = min(tile * kKeys + in, r.keys - 1);  // (past the last one: the last one again)
        const uint16_t* const from = static_cast<const uint16_t*>(rows) + static_cast<int64_t>(r.key_start + key) * stride + 8 * ((lane_now % kLanes) ^ turned);
        LaneLineToLds(from, to + area + 1024 * n);
      }
    };
    part(std::integral_constant<int, G::kKeyPitch>{}, std::false_type{}, 0, static_cast<const uint16_t*>(op.k) + head * op.k_head_stride, op.k_token_stride);
    part(std::integral_constant<int, G::kRopePitch>{}, std::false_type{}, G::kKeyBytes, op.k_rope, op.k_rope_token_stride);
    part(std::integral_constant<int, G::kValuePitch>{}, std::true_type{}, G::kKeyBytes + G::kRopeBytes, static_cast<const uint16_t*>(op.v) + head * op.v_head_stride, op.v_token_stride);
  };

  const int k_row = 16 * (column >> 2 & 1) + 4 * (column >> 3) + (column & 3);
  const int i16 = lane & 15, v_row = 16 * half + (i16 >> 2);
  const uint32_t key_lane = k_row * G::kKeyPitch + 16 * (KeyTurn<G::kKeyPitch>(k_row) ^ half);
  const uint32_t rope_lane = G::kKeyBytes + k_row * G::kRopePitch + 16 * (KeyTurn<G::kRopePitch>(k_row) ^ half);
  const uint32_t value_lane = G::kKeyBytes + G::kRopeBytes + v_row * G::kValuePitch + 16 * ((2 * (lane >> 4 & 1) + (i16 >> 1 & 1)) ^ ValueTurn<G::kValuePitch>(v_row)) + 8 * (i16 & 1);
  // Keys 32 k + 16 half + 8 s to + 7 of dimension 32 b + column.
  const auto value = [&](uint32_t at, int b, int k, int s) {
    constexpr int kTurn8 = 2, kTurn4 = 1;  // of eight rows on, of four
    const uint32_t rows = (32 * k + 8 * s) * G::kValuePitch;
    const S16x4 v = Column4(lds + (at ^ 16 * (4 * b ^ kTurn8 * s)) + rows);
    return JoinFours<Eight>(v, Column4(lds + (at ^ 16 * (4 * b ^ kTurn8 * s ^ kTurn4)) + rows + 4 * G::kValuePitch));
  };

  if (tile_from < tile_to) fetch(tile_from, 0);
  for (int tile = tile_from; tile < tile_to; ++tile) {
    const int slot = (tile - tile_from) & 1;
    WaitLoads<0>();
    MeetLds();
    if (tile + 1 < tile_to) fetch(tile + 1, slot ^ 1);
    const uint32_t at = slot * G::kTile;
    const int p0 = tile * kKeys;
    const bool works = busy && p0 < base + min(first + wave * 32 + 32, r.n);
    F32x16 dots[2];
    if (works) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) dots[k][i] = 0.0f;
#pragma unroll
        for (int x = 0; x < kSteps + kRopeSteps; ++x) {
          const Eight key = x < kSteps ? *reinterpret_cast<const Eight*>(lds + ((at + key_lane) ^ 32 * x) + 32 * k * G::kKeyPitch)
                                       : *reinterpret_cast<const Eight*>(lds + ((at + rope_lane) ^ 32 * (x - kSteps)) + 32 * k * G::kRopePitch);
          dots[k] = S::Product32(key, q[x], dots[k]);
        }
      }
    }
    float worth_now = worth;
    if (p0 + kKeys > all_rows_to) {
      // ---- a tile that some row does not see all of. Infinities and NaN among values that a row does not see are not kept out by a weight of zero:
      // where there are any, they become zeros here, and what they are to the rows that see them is added by itself.
      MeetLds();  // (nobody reads the keys any more: the flags lie there)
      uint8_t* const values = lds + at + G::kKeyBytes + G::kRopeBytes;
      bool odd = false;
      for (int i = 16 * tid; i < G::kValueBytes; i += 16 * kPromptThreads) {
        const U32x4 v = *reinterpret_cast<const U32x4*>(values + i), f = Finite<TYPE>(v);
        odd = odd || v[0] != f[0] || v[1] != f[1] || v[2] != f[2] || v[3] != f[3];
      }
      if (lane == 0) reinterpret_cast<int*>(lds + at)[wave] = 0;
      if (__any(odd) && lane == 0) reinterpret_cast<int*>(lds + at)[wave] = 1;
      MeetLds();
      const int* const flags = reinterpret_cast<const int*>(lds + at);
      if ((flags[0] | flags[1] | flags[2] | flags[3]) != 0) {
        // (A value that is no number makes every row that sees its key none in that dimension, whatever its weight; an infinity does with
        // it what the product of the weight is: either way the row's sum in that dimension ends as weight * value added to it.)
        if (works) {
#pragma unroll 1
          for (int t = 0; t < kKeys; ++t) {
            const bool sees = p0 + t < see_to;
            if (!__any(sees)) continue;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              // Four dimensions of a lane's element group at a time: 8 i + 4 half + e.
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int piece = (4 * b + i) ^ ValueTurn<G::kValuePitch>(t);
                const uint16_t* const v = reinterpret_cast<const uint16_t*>(values + t * G::kValuePitch + 16 * piece + 8 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float x = TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(v[e]) : HalfBitsToFloat(v[e]);
                  if (sees && !(fabsf(x) < INFINITY)) out[b][4 * i + e] += x;
                }
              }
            }
          }
        }
        MeetLds();
        for (int i = 16 * tid; i < G::kValueBytes; i += 16 * kPromptThreads) {
          U32x4* const v = reinterpret_cast<U32x4*>(values + i);
          *v = Finite<TYPE>(*v);
        }
        MeetLds();
      }
      if (p0 + kKeys > all_to) {
        asm volatile("" ::: "memory");  // (a branch: selects would be in every tile's way)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int to = see_to - p0 - 32 * k - 16 * half;
#pragma unroll
          for (int i = 0; i < 16; ++i) dots[k][i] = i < to ? dots[k][i] * worth : -INFINITY;
        }
        worth_now = 1.0f;
      }
    }
    if (!works) continue;
    float peak = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 16; ++i) peak = fmaxf(peak, dots[k][i]);
    }
    peak = AcrossHalvesMax(peak) * worth_now;
    if (__any(peak > top + (kUp + kFollow))) {
      const float higher = fmaxf(top, peak - kUp);
      const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
      top = higher;
      sum *= keep;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) out[b] *= keep;
    }
    const float less = top == -INFINITY ? 0.0f : top;
    Eight weights[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(fmaf(dots[k][i], worth_now, -less));
        sum += p;
        weights[2 * k + i / 8][i % 8] = static_cast<typename S::One>(p);
      }
    }
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int k = 0; k < 4; ++k) out[b] = S::Product32(value(at + value_lane, b, k / 2, k % 2), weights[k], out[b]);
    }
  }
  sum = AcrossHalvesSum(sum);
  if (!real) return;
  // ---- out, or a run for the join. Element 4i + e of block b is dimension 32b + 8i + 4 half + e.
  if (a.runs == 1) {
    const float by = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    const int64_t to = static_cast<int64_t>(r.start + row) * op.out_token_stride + head * op.out_head_stride + 4 * half;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v[4] = {out[b][4 * i] * by, out[b][4 * i + 1] * by, out[b][4 * i + 2] * by, out[b][4 * i + 3] * by};
        StoreValues<TYPE, 4>(op.out, to + 32 * b + 8 * i, v);
      }
    }
  } else {
    const int64_t at = (static_cast<int64_t>(request_head * a.tiles + tile_index) * a.runs + run) * kPromptRows + wave * 32 + column;
    if (half == 0) reinterpret_cast<float2*>(a.numbers)[at] = make_float2(top, sum);
    float* const to = a.values + at * N + 4 * half;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<F32x4*>(to + 32 * b + 8 * i) = F32x4{out[b][4 * i], out[b][4 * i + 1], out[b][4 * i + 2], out[b][4 * i + 3]};
    }
  }
}

// The runs of a row joined: 16 (32) lanes a row, eight (four) values a lane... a thread eight values. grid (row tiles of all).
template <int TYPE, int N>
__global__ __launch_bounds__(kPromptThreads) void LatentPromptJoinKernel(const PromptArgs a) {
  constexpr int kLanes = N / 8, kRowsAGo = kPromptThreads / kLanes;
  const llmp_latent_prompt& op = a.op;
  const uint32_t request_head = blockIdx.x / a.tiles;
  const int tile_index = blockIdx.x % a.tiles, request = request_head / op.heads, head = request_head % op.heads;
  const PromptRequest r = PromptOf(op, request);
  const int first = tile_index * kPromptRows, rows = min(r.n - first, kPromptRows);
  for (int row = threadIdx.x / kLanes; row < rows; row += kRowsAGo) {
    const int d0 = 8 * (threadIdx.x % kLanes);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * a.runs * kPromptRows + row;
    float most = -INFINITY;
    for (int i = 0; i < a.runs; ++i) most = fmaxf(most, a.numbers[2 * (at + i * kPromptRows)]);
    const float less = most == -INFINITY ? 0.0f : most;
    float sum = 0.0f, v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int i = 0; i < a.runs; ++i) {
      const float2 n = reinterpret_cast<const float2*>(a.numbers)[at + i * kPromptRows];
      const float by = __builtin_amdgcn_exp2f(n.x - less);
      sum = fmaf(n.y, by, sum);
      const F32x4* const from = reinterpret_cast<const F32x4*>(a.values + (at + i * kPromptRows) * N + d0);
      const F32x4 x = from[0], y = from[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], by, v[e]), v[4 + e] = fmaf(y[e], by, v[4 + e]);
    }
    const float by = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= by;
    StoreValues<TYPE, 8>(op.out, static_cast<int64_t>(r.start + first + row) * op.out_token_stride + head * op.out_head_stride + d0, v);
  }
}

int CheckLatentPrompt(const llmp_latent_prompt* op, int cus) {
  if (op == nullptr) return Refuse(1, "latent_prompt: null operands");
  if (op->type != LLMP_X_BF16 && op->type != LLMP_X_F16) return Refuse(1, "latent_prompt: BF16 or F16 values, not type %d", op->type);
  if ((op->nope != 64 && op->nope != 128) || op->value != op->nope || (op->rope_width != 32 && op->rope_width != 64))
    return Refuse(1, "latent_prompt: heads of 64 or 128 values for keys and values alike, rotated keys of 32 or 64 (%d, %d, %d)", op->nope, op->value, op->rope_width);
  if (op->heads < 1 || op->heads > 65535 || op->requests < 1 || op->requests > 1 << 24 || op->tokens < 1 || op->keys < 0 || op->most_tokens < 1 ||
      op->keys > 1 << 30 || op->tokens > 1 << 30)
    return Refuse(1, "latent_prompt: 1 to 2^24 requests, 1 to 65535 heads, 1 to 2^30 tokens, at most 2^30 keys (%d, %d, %d, %d, %d)", op->requests, op->heads, op->tokens, op->keys, op->most_tokens);
  if (const int bad = CheckPagedRows("latent_prompt", "q", op->q, op->tokens, op->heads, op->q_token_stride, op->q_head_stride, op->type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("latent_prompt", "out", op->out, op->tokens, op->heads, op->out_token_stride, op->out_head_stride, op->type); bad != 0) return bad;
  if (op->keys > 0) {
    if (const int bad = CheckPagedRows("latent_prompt", "k", op->k, op->keys, op->heads, op->k_token_stride, op->k_head_stride, op->type); bad != 0) return bad;
    if (const int bad = CheckPagedRows("latent_prompt", "v", op->v, op->keys, op->heads, op->v_token_stride, op->v_head_stride, op->type); bad != 0) return bad;
    if (const int bad = CheckPagedRows("latent_prompt", "k_rope", op->k_rope, op->keys, 1, op->k_rope_token_stride, 0, op->type); bad != 0) return bad;
  }
  if (op->starts == nullptr || (reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->key_starts)) % 4 != 0)
    return Refuse(1, "latent_prompt: I32 arrays at 4-byte boundaries");
  if (!std::isfinite(op->scale)) return Refuse(1, "latent_prompt: a scale that is not finite");
  if (cus < 1 || cus > 4096) return Refuse(1, "latent_prompt: %d compute units", cus);
  const int64_t tiles = (std::min(op->most_tokens, op->tokens) + kPromptRows - 1) / kPromptRows;
  if ((static_cast<int64_t>(op->requests) * op->heads + 8) * tiles * kMostRuns > INT_MAX) return Refuse(1, "latent_prompt: %d requests of %d heads with up to %d rows are too many", op->requests, op->heads, op->most_tokens);
  return 0;
}

// How the keys are cut: the least runs that give every compute unit two workgroups, none shorter than four tiles of the longest request that there can be.
int RunsOf(const llmp_latent_prompt& op, int cus, int tiles) {
  const int64_t sets = static_cast<int64_t>(op.requests) * op.heads * tiles;
  const int64_t most = std::max<int64_t>(1, op.keys / (4 * kKeys));
  return static_cast<int>(std::min<int64_t>({most, kMostRuns, std::max<int64_t>(1, 2 * cus / sets)}));
}
int TilesOf(const llmp_latent_prompt& op) { return (std::min(op.most_tokens, op.tokens) + kPromptRows - 1) / kPromptRows; }

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" size_t llmp_hip_latent_prompt_scratch(const llmp_latent_prompt* op, int cus) {
  if (CheckLatentPrompt(op, cus) != 0) return 0;
  const int tiles = TilesOf(*op), runs = RunsOf(*op, cus, tiles);
  if (runs == 1) return 16;
  return static_cast<size_t>(op->requests) * op->heads * tiles * runs * kPromptRows * (8 + 4 * static_cast<size_t>(op->value));
}

extern "C" int llmp_hip_latent_prompt(const llmp_latent_prompt* op, void* scratch, size_t scratch_bytes, int cus, void* stream) {
  if (const int bad = CheckLatentPrompt(op, cus); bad != 0) return bad;
  const size_t need = llmp_hip_latent_prompt_scratch(op, cus);
  if (scratch == nullptr || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
    return Refuse(1, "latent_prompt: %zu bytes of scratch at a 16-byte boundary, not %zu", need, scratch_bytes);
  PromptArgs a;
  a.op = *op;
  a.tiles = TilesOf(*op);
  a.runs = RunsOf(*op, cus, a.tiles);
  const size_t sets = static_cast<size_t>(op->requests) * op->heads;
  a.numbers = static_cast<float*>(scratch);
  a.values = a.numbers + sets * a.tiles * a.runs * kPromptRows * 2;
  const dim3 grid(static_cast<unsigned>((sets * a.runs + 7) / 8 * 8 * a.tiles));
  const auto s = static_cast<hipStream_t>(stream);
  BeginLaunches();
  const auto launch = [&](auto type, auto n, auto p) {
    constexpr int kType = decltype(type)::value, kN = decltype(n)::value, kP = decltype(p)::value;
    static bool sized = false;
    constexpr int kLds = PromptGeo<kN, kP>::kLds;
    if (!AllowLds(reinterpret_cast<const void*>(&LatentPromptKernel<kType, kN, kP>), kLds, &sized)) return;
    hipLaunchKernelGGL((LatentPromptKernel<kType, kN, kP>), grid, dim3(kPromptThreads), kLds, s, a);
    if (a.runs > 1) hipLaunchKernelGGL((LatentPromptJoinKernel<kType, kN>), dim3(static_cast<unsigned>(sets * a.tiles)), dim3(kPromptThreads), 0, s, a);
  };
  const auto sizes = [&](auto type) {
    const auto rope = [&](auto n) {
      if (op->rope_width == 32) launch(type, n, std::integral_constant<int, 32>{});
      if (op->rope_width == 64) launch(type, n, std::integral_constant<int, 64>{});
    };
    if (op->nope == 64) rope(std::integral_constant<int, 64>{});
    if (op->nope == 128) rope(std::integral_constant<int, 128>{});
  };
  if (op->type == LLMP_X_BF16) sizes(std::integral_constant<int, LLMP_X_BF16>{});
  if (op->type == LLMP_X_F16) sizes(std::integral_constant<int, LLMP_X_F16>{});
  return LaunchStatus("latent_prompt");
}
