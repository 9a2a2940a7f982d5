// llmp.latent.prompt: the expanded form over ragged requests. A head's keys are its own values beside the rotated key that all heads share, so
// that the shared part is read from one place and never copied to the heads.
//
// What bounds it is the matrix instructions (2 * (nope + rope + value) operations a logit) and beside them a softmax's exponential and six operations
// a logit. A workgroup of four waves has 128 rows of one head, 32 a wave, two workgroups a compute unit; 64 keys at a time go through LDS by loads that
// pass no register, the next tile under this one's work:
//   S^T = K Q^T, P = exp2(S - E), O^T += V^T P^T, all by 32 x 32 products.
// Row 8a + 4h + b of the first product is key 16h + 4a + b of its 32, so that a lane (half h) ends with 16 keys in order of one row, which is what the
// second product takes; V's columns come by transposing reads.
//
// Where pairs of (head, 128 rows) are many for the device, a workgroup takes one whole, a head's pairs on one chiplet, the longest first (a prompt of 4096, 32 heads:
// 194 us, 215 in the rows' order; of 64 + 32 and 64 values 105 and 128). Elsewhere the pairs' keys are cut evenly (latent_line.h).
// (Times in this file are passes of one call after the other, host and join with them. That prompt, nope 128, rope 64, values of 128: 0.89 PFLOP/s; the matrix
// instructions are busy 52 % of the cycles, other vector instructions 36 %, and a wave's products and softmax wait for each other. Six ragged ones of 12 heads, up to
// 700 rows of 64 + 32 behind 3500 keys: the kernel 35 us and 9 the join, 41.6 the call.)
#include <algorithm>
#include <cmath>

#include "latent_line.h"

namespace llmp_hip {
namespace {

constexpr int kKeys = 64;  // a tile's
constexpr int kPromptRows = 128, kPromptThreads = 256;
constexpr int kAUnit = 2;                            // workgroups a compute unit
// Of the line, to a workgroup: finer parts cost more to write and to join (six ragged prompts of 12 heads: 41.6 us, 44.0 at 128, 44.0 at 512; 100 rows behind 3000,
// 4 heads: 26.3, 23.0 and 30.2; one row behind 4000 keys, 8 heads: 19.6, 17.9 and 26.4).
constexpr int kLeast = 256;

struct PromptArgs {
  llmp_latent_prompt op;
  LatentParts parts;
  int tiles;  // row tiles a request, at most
};

// A request's rows of q and its keys, none where the arrays name rows outside the call's.
struct PromptRequest {
  LatentRequest l;
  int key_start;
};
__device__ __forceinline__ PromptRequest PromptOf(const llmp_latent_prompt& op, int r) {
  PromptRequest q;
  q.l.start = op.starts[r];
  const int end = op.starts[r + 1];
  q.l.n = q.l.start >= 0 && end > q.l.start && end <= op.tokens ? end - q.l.start : 0;
  const int32_t* const keys = op.key_starts != nullptr ? op.key_starts : op.starts;
  q.key_start = keys[r];
  const int key_end = keys[r + 1];
  q.l.length = q.key_start >= 0 && key_end > q.key_start && key_end <= op.keys ? key_end - q.key_start : 0;
  q.l.base = q.l.length - q.l.n;
  q.l.groups = (q.l.n + kPromptRows - 1) / kPromptRows;
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

template <int N, int P, int V>
struct PromptGeo {
  static constexpr int kKeyPitch = 2 * N, kRopePitch = 2 * P, kValuePitch = 2 * V;
  static constexpr int kKeyBytes = kKeys * kKeyPitch, kRopeBytes = kKeys * kRopePitch, kValueBytes = kKeys * kValuePitch;
  static constexpr int kTile = kKeyBytes + kRopeBytes + kValueBytes;
  static constexpr int kRing = 2;
  static constexpr int kKeyLoads = kKeyBytes / 4096, kRopeLoads = kRopeBytes / 4096, kValueLoads = kValueBytes / 4096;  // a wave's
  static constexpr int kLds = kRing * kTile;
};

// LINE: the grid is the device's, each workgroup a run of the line; else a block a (request, head, row tile).
template <int TYPE, int N, int P, int V, bool LINE>
__global__ __launch_bounds__(kPromptThreads, kAUnit) void LatentPromptKernel(const PromptArgs a) {
  using G = PromptGeo<N, P, V>;
  using S = Sixteen<TYPE>;
  typedef typename S::Eight Eight;
  constexpr int kSteps = N / 16, kRopeSteps = P / 16, kBlocks = V / 32;
  constexpr int kKeyGroup = 4, kValueGroup = 4;  // products that are read for at a time
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const llmp_latent_prompt& op = a.op;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane / 32, column = lane % 32;
  const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const uint32_t flip = op.scale < 0.0f ? 0x80008000u : 0u;  // (a negative scale goes into the queries: the largest product is the largest logit)
  const float worth = Scalar(fabsf(op.scale) * kLog2E);

  // Eight workgroups in a row go to eight chiplets: a chiplet takes every eighth (request, head), or an eighth of the line, so that its L2 holds the keys that
  // neighbouring pairs share (one prompt of 4096, 8 heads: 79 us, of 64 + 32 and 64 values 57; runs in the order of the workgroups 92 and 64).
  const int groups = gridDim.x;
  int index = 0;
  int request, head = 0, k = 0;
  int64_t u = 0, u_end = 1, before = 0, per = 1, pair_from = 0;
  if constexpr (LINE) {
    const LatentRun run = RunOf<true>(op.requests, blockIdx.x, groups, kLeast, [&](int r) {
      const LatentRequest l = PromptOf(op, r).l;
      return LineBefore(l, kPromptRows, l.groups) * op.heads;
    });
    u = run.from, u_end = run.to, before = run.before, request = run.request, per = run.per, index = run.index;
    if (tid < 2) a.parts.which[(2 * index + tid) * 4] = -1;
  } else {
    const uint32_t sets = static_cast<uint32_t>(op.requests) * op.heads, padded = (sets + 7) / 8 * 8, set = blockIdx.x % padded;
    if (set >= sets) return;
    request = set / op.heads, head = set % op.heads, k = a.tiles - 1 - static_cast<int>(blockIdx.x / padded);
  }
  for (; u < u_end;) {
  // ---- the next pair, or part of one.
  PromptRequest r = PromptOf(op, request);
  r = {Scalar(r.l), Scalar(r.key_start)};
  LatentPiece piece = {};
  int any_to;
  if constexpr (LINE) {
    const int64_t a_head = LineBefore(r.l, kPromptRows, r.l.groups);
    if (u >= before + a_head * op.heads) {
      before += a_head * op.heads;
      ++request;
      continue;
    }
    head = static_cast<int>(Over(u - before, a_head));
    const int64_t head_from = before + head * a_head;
    k = GroupAt(r.l, kPromptRows, u - head_from);
    any_to = SeenOf(r.l, kPromptRows, k);
    pair_from = head_from + LineBefore(r.l, kPromptRows, k);
    const int x0 = static_cast<int>(u - pair_from), x1 = static_cast<int>(min(u_end - pair_from, static_cast<int64_t>(any_to + kVisit)));
    u = pair_from + x1;
    piece = PieceOf(any_to, kKeys, x0, x1);
    if (!piece.any) continue;
  } else {
    u = u_end;
    if (k >= r.l.groups) return;
    any_to = SeenOf(r.l, kPromptRows, k);
    piece = {0, (any_to + kKeys - 1) / kKeys, true, true, true};
  }
  head = Scalar(head), k = Scalar(k);
  const int tile_from = Scalar(piece.from), tile_to = Scalar(piece.to);
  const int first = k * kPromptRows, base = r.l.base;
  const int row = first + wave * 32 + column;
  const bool real = row < r.l.n, busy = first + wave * 32 < r.l.n;
  const int token = real ? row : first;
  const int see_to = real ? max(base + row + 1, 0) : 0;
  const int all_to = max(base + first + wave * 32 + 1, 0);  // seen by all of the wave's rows
  const int all_rows_to = max(base + first + 1, 0);         // of the workgroup's

  Eight q[kSteps + kRopeSteps];
  {
    const uint16_t* const from = static_cast<const uint16_t*>(op.q) + static_cast<int64_t>(r.l.start + token) * op.q_token_stride + head * op.q_head_stride + 8 * half;
#pragma unroll
    for (int x = 0; x < kSteps + kRopeSteps; ++x) {
      U32x4 v = *reinterpret_cast<const U32x4*>(from + 16 * x);
      v ^= U32x4{flip, flip, flip, flip};
      q[x] = __builtin_bit_cast(Eight, v);
    }
  }
  F32x16 out[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) out[b][i] = 0.0f;
  }
  float top = -INFINITY, sum = 0.0f;

  // A lane's places in a tile's rows, for every load of the wave's (row strides stay below 2^24 values: the host looks; one
  // key's takes itself off again). A load's rows follow the one's before it.
  uint32_t k_places[G::kKeyLoads], r_places[G::kRopeLoads], v_places[G::kValueLoads];
  const auto place = [&](auto pitch, auto turn, uint32_t* places, int count, int64_t stride) {
    constexpr int kLanes = decltype(pitch)::value / 16, kRowsALoad = kWave / kLanes;
#pragma unroll
    for (int i = 0; i < count; ++i) {
      const int in = (wave * count + i) * kRowsALoad + lane / kLanes;
      places[i] = static_cast<uint32_t>(in) * static_cast<uint32_t>(2 * stride) + 16 * ((lane % kLanes) ^ turn(in));
    }
  };
  place(std::integral_constant<int, G::kKeyPitch>{}, KeyTurn<G::kKeyPitch>, k_places, G::kKeyLoads, op.k_token_stride);
  place(std::integral_constant<int, G::kRopePitch>{}, KeyTurn<G::kRopePitch>, r_places, G::kRopeLoads, op.k_rope_token_stride);
  place(std::integral_constant<int, G::kValuePitch>{}, ValueTurn<G::kValuePitch>, v_places, G::kValueLoads, op.v_token_stride);
  const uint16_t* const k_base = static_cast<const uint16_t*>(op.k) + head * op.k_head_stride;
  const uint16_t* const r_base = static_cast<const uint16_t*>(op.k_rope);
  const uint16_t* const v_base = static_cast<const uint16_t*>(op.v) + head * op.v_head_stride;
  const auto fetch = [&](int tile, int slot) {
    const int64_t key = r.key_start + static_cast<int64_t>(tile) * kKeys;
    const int left = r.l.length - tile * kKeys;  // at least one; past them the last one again
    const auto part = [&](auto pitch, const uint32_t* places, int count, uint32_t area, const uint16_t* rows, int64_t stride) {
      constexpr int kLanes = decltype(pitch)::value / 16, kRowsALoad = kWave / kLanes;
      const uint16_t* const from = rows + key * stride;
      const uint32_t to = Scalar(lds_at + slot * G::kTile + area + 1024 * wave * count);
      if (left >= kKeys) {
#pragma unroll
        for (int i = 0; i < count; ++i) LineToLds(from, places[i], to + 1024 * i);
      } else {
#pragma unroll
        for (int i = 0; i < count; ++i) {
          const int in = (wave * count + i) * kRowsALoad + lane / kLanes;
          LineToLds(from, places[i] - static_cast<uint32_t>(max(in - left + 1, 0)) * static_cast<uint32_t>(2 * stride), to + 1024 * i);
        }
      }
    };
    part(std::integral_constant<int, G::kKeyPitch>{}, k_places, G::kKeyLoads, 0, k_base, op.k_token_stride);
    part(std::integral_constant<int, G::kRopePitch>{}, r_places, G::kRopeLoads, G::kKeyBytes, r_base, op.k_rope_token_stride);
    part(std::integral_constant<int, G::kValuePitch>{}, v_places, G::kValueLoads, G::kKeyBytes + G::kRopeBytes, v_base, op.v_token_stride);
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
    const bool works = busy && p0 < base + min(first + wave * 32 + 32, r.l.n);
    F32x16 dots[2];
    if (works) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < 16; ++i) dots[k][i] = 0.0f;
      }
      // (The two blocks of 32 keys in turn: their places differ by a constant.)
      ProductsInGroups<2 * (kSteps + kRopeSteps), kKeyGroup, Eight>(
          [&](int i) {
            const int x = i / 2, k = i % 2;
            return x < kSteps ? *reinterpret_cast<const Eight*>(lds + ((at + key_lane) ^ 32 * x) + 32 * k * G::kKeyPitch)
                              : *reinterpret_cast<const Eight*>(lds + ((at + rope_lane) ^ 32 * (x - kSteps)) + 32 * k * G::kRopePitch);
          },
          [&](int i, Eight key) { dots[i % 2] = S::Product32(key, q[i / 2], dots[i % 2]); });
    }
    uint8_t* const values = lds + at + G::kKeyBytes + G::kRopeBytes;
    float worth_now = worth;
    int odd = 0;
    if (p0 + kKeys > all_rows_to) {
      // ---- a tile that some row does not see all of. Infinities and NaN among values that a row does not see are not kept out by a weight of zero:
      // where there are any, they become zeros before the second product, and what they are to the rows that see them is added by itself.
      MeetLds();  // (nobody reads the keys any more: the flags lie there)
      bool mine = false;
      for (int i = 16 * tid; i < G::kValueBytes; i += 16 * kPromptThreads) {
        const U32x4 v = *reinterpret_cast<const U32x4*>(values + i), f = Finite<TYPE>(v);
        mine = mine || v[0] != f[0] || v[1] != f[1] || v[2] != f[2] || v[3] != f[3];
      }
      if (lane == 0) reinterpret_cast<int*>(lds + at)[wave] = 0;
      if (__any(mine) && lane == 0) reinterpret_cast<int*>(lds + at)[wave] = 1;
      MeetLds();
      const int* const flags = reinterpret_cast<const int*>(lds + at);
      odd = Scalar(flags[0] | flags[1] | flags[2] | flags[3]);
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
    // (All four waves, or none.)
    const auto clean = [&]() {
      MeetLds();
      for (int i = 16 * tid; i < G::kValueBytes; i += 16 * kPromptThreads) {
        U32x4* const v = reinterpret_cast<U32x4*>(values + i);
        *v = Finite<TYPE>(*v);
      }
      MeetLds();
    };
    if (!works) {
      if (odd != 0) clean();
      continue;
    }
    float peak = -INFINITY;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) peak = fmaxf(fmaxf(peak, dots[k][i]), dots[k][i + 1]);
    }
    peak = AcrossHalvesMax(peak) * worth_now;
    if (__any(peak > top + (kUp + kFollow))) {
      const float higher = peak > top + (kUp + kFollow) ? peak - kUp : top;  // (a row's own: what other rows see changes no bit of it)
      const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
      top = higher;
      sum *= keep;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) out[b] *= keep;
    }
    const float less = top == -INFINITY ? 0.0f : top;
    if (odd != 0) {
      // What the second product would add, weight * value, is the value where the weight is not zero and no number where it is. (Here the row's
      // scale has followed. The weights are worked out by themselves: beside the branch everything stays in one piece, the weights with the second product's first reads.)
      uint32_t own = 0;  // the lane's keys with a weight: 16 of the first 32, 16 of the others
      float less_again = less;
      asm volatile("" : "+v"(less_again));
#pragma unroll
      for (int i = 31; i >= 0; --i) {
        const auto weight = static_cast<typename S::One>(__builtin_amdgcn_exp2f(fmaf(dots[i / 16][i % 16], worth_now, -less_again)));
        own = own * 2 + (weight != static_cast<typename S::One>(0.0f) ? 1u : 0u);
      }
      const uint32_t other = ShflXor(own, 32), low = half == 0 ? own : other, high = half == 0 ? other : own;
      const uint32_t heavy[2] = {(low & 0xFFFFu) | high << 16, low >> 16 | (high & 0xFFFF0000u)};  // of the row's 64
#pragma unroll 1
      for (int t = 0; t < kKeys; ++t) {
        const bool sees = p0 + t < see_to;
        const float weight = ((t < 32 ? heavy[0] : heavy[1]) >> (t & 31) & 1u) != 0 ? 1.0f : 0.0f;
        if (!__any(sees)) continue;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          // Four dimensions of a lane's element group at a time: 8 i + 4 half + e.
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int place = (4 * b + i) ^ ValueTurn<G::kValuePitch>(t);
            const uint16_t* const v = reinterpret_cast<const uint16_t*>(values + t * G::kValuePitch + 16 * place + 8 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x = TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(v[e]) : HalfBitsToFloat(v[e]);
              if (sees && !(fabsf(x) < INFINITY)) out[b][4 * i + e] = fmaf(x, weight, out[b][4 * i + e]);
            }
          }
        }
      }
      clean();
    }
    Eight weights[4];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float p = __builtin_amdgcn_exp2f(fmaf(dots[k][i], worth_now, -less)), p1 = __builtin_amdgcn_exp2f(fmaf(dots[k][i + 1], worth_now, -less));
        // (Rounded to the type, for the matrix instructions that take 16-bit values: 2^-8 of a weight, F16 2^-11, beside the result's own rounding, which is as large.)
        weights[2 * k + i / 8][i % 8] = static_cast<typename S::One>(p), weights[2 * k + i / 8][i % 8 + 1] = static_cast<typename S::One>(p1);
        // (The sum is of the weights as they are rounded, two in an instruction.)
        sum = S::AddTwo(typename S::Two{weights[2 * k + i / 8][i % 8], weights[2 * k + i / 8][i % 8 + 1]}, sum);
      }
    }
    // (Two blocks of dimensions in turn: a product does not wait for the one before it.)
    const uint32_t value_at = at + value_lane;
    ProductsInGroups<4 * kBlocks, kValueGroup, Eight>([&](int i) { return value(value_at, 2 * (i / 8) + i % 2, i / 2 % 2, i / 4 % 2); },
                                                      [&](int i, Eight v) { const int b = 2 * (i / 8) + i % 2; out[b] = S::Product32(v, weights[2 * (i / 2 % 2) + i / 4 % 2], out[b]); });
  }
  sum = AcrossHalvesSum(sum);
  if constexpr (LINE) MeetLds();  // (the next pair's tiles come where this one's were)
  // ---- out, or a part for the join. Element 4i + e of block b is dimension 32b + 8i + 4 half + e.
  if (!LINE || (piece.begins && piece.ends)) {
    if (real) {
      const float by = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
      const int64_t to = static_cast<int64_t>(r.l.start + row) * op.out_token_stride + head * op.out_head_stride + 4 * half;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v[4] = {out[b][4 * i] * by, out[b][4 * i + 1] * by, out[b][4 * i + 2] * by, out[b][4 * i + 3] * by};
          StoreValues<TYPE, 4>(op.out, to + 32 * b + 8 * i, v);
        }
      }
    }
  } else {
    const int which = 2 * index + (piece.begins ? 1 : 0);
    if (tid == 0) {
      const LatentOwners owners = OwnersOf(pair_from, any_to, kKeys, per);
      *reinterpret_cast<I32x4*>(a.parts.which + 4 * which) = I32x4{owners.first, k * op.heads + head, min(r.l.n - first, kPromptRows) | owners.count << 8, r.l.start + first};
    }
    if (busy) {
      const int64_t unit = static_cast<int64_t>(which) * (kPromptRows / 32) + wave;
      if (half == 0) a.parts.numbers[unit * 32 + column] = make_float2(top, sum);
      F32x4* const to = reinterpret_cast<F32x4*>(a.parts.values) + unit * (V / 8) * kWave + lane;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(4 * b + i) * kWave] = F32x4{out[b][4 * i], out[b][4 * i + 1], out[b][4 * i + 2], out[b][4 * i + 3]};
      }
    }
  }
  }
}

int TilesOf(const llmp_latent_prompt& op) { return (std::min(op.most_tokens, op.tokens) + kPromptRows - 1) / kPromptRows; }

int CheckLatentPrompt(const llmp_latent_prompt* op, int cus) {
  if (op == nullptr) return Refuse(1, "latent_prompt: null operands");
  if (op->type != LLMP_X_BF16 && op->type != LLMP_X_F16) return Refuse(1, "latent_prompt: BF16 or F16 values, not type %d", op->type);
  if ((op->nope != 64 && op->nope != 128) || (op->value != 64 && op->value != 128) || (op->rope_width != 32 && op->rope_width != 64))
    return Refuse(1, "latent_prompt: heads of 64 or 128 values for keys and for values, rotated keys of 32 or 64 (%d, %d, %d)", op->nope, op->value, op->rope_width);
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
  const int64_t most_stride = 1 << 24;
  if (op->keys > 1 && (op->k_token_stride >= most_stride || op->v_token_stride >= most_stride || op->k_rope_token_stride >= most_stride))
    return Refuse(1, "latent_prompt: keys and values at most 2^24 values apart");
  if ((static_cast<int64_t>(op->requests) * op->heads + 8) * TilesOf(*op) > INT_MAX)
    return Refuse(1, "latent_prompt: %d requests of %d heads with up to %d rows are too many", op->requests, op->heads, op->most_tokens);
  return 0;
}

// Of the line: an eighth of them on every chiplet.
int LineGroups(int cus) { return (kAUnit * cus + 7) / 8 * 8; }

// Blocks where pairs are taken whole: (request, head) by eights, so that a chiplet has all row tiles of its own.
int64_t WholeBlocks(const llmp_latent_prompt& op) { return (static_cast<int64_t>(op.requests) * op.heads + 7) / 8 * 8 * TilesOf(op); }

// Whether pairs are taken whole. Then a call lasts as long as its longest pair (1.5 us a key tile of 128 + 64 and 128 values, a workgroup alone on its unit; 1.1 of 64 + 32 and
// 64) or as a workgroup's share (2.9 and 1.6 us a tile, two of them on it), and cut into runs as long as the share and 25 to 50 us, for the parts. As far as the sizes
// tell those: half of the last row tile of a request is empty, a request has an equal part of the keys and no more than twice that, a row sees all of them, or half where
// all of them are new. The 2.5 and 15 tiles below were found by such calls as these. (Whole and cut, heads of 128 + 64 and 128, then of 64 + 32 and 64: a prompt of 4096, 32 heads 194 and 247 us, 105 and 154, 8 heads 100 and 78, 72 and 52; one of 1000, 8
// heads 30 and 32, 22 and 24; 16 of up to 1000, 32 heads 58 and 82, 37 and 55; six ragged ones of 12 heads, up to 700 rows behind 3500 keys 118 and 59, 82 and 41: the rule
// takes the shorter each time. Of those with 32 heads, wide, it takes them whole: 119 and 108.)
bool WholePairs(const llmp_latent_prompt& op, int cus) {
  const bool fresh = op.key_starts == nullptr || op.keys == op.tokens;
  const double requests = op.requests, tiles = op.keys / static_cast<double>(kKeys) + 1.0, share = tiles / requests + 1.0;
  const double longest = fresh ? std::min(tiles, op.most_tokens / static_cast<double>(kKeys) + 1.0) : std::min(tiles, 2.0 * share);
  const double row_tiles = op.tokens / static_cast<double>(kPromptRows) + 0.5 * requests;
  if (WholeBlocks(op) >= (int64_t{1} << 32) / kPromptThreads) return false;  // (a launch has less than 2^32 threads)
  // (Blocks are dealt by the largest number of queries that the caller says: where that says little, most would have no pair.)
  if (static_cast<double>(TilesOf(op)) * requests > 4.0 * (op.tokens / static_cast<double>(kPromptRows) + requests)) return false;
  const double each = row_tiles * op.heads * share * (fresh ? 0.5 : 1.0) / (kAUnit * cus);
  return longest <= 2.5 * each + 15.0;
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" size_t llmp_hip_latent_prompt_scratch(const llmp_latent_prompt* op, int cus) {
  if (CheckLatentPrompt(op, cus) != 0) return 0;
  return WholePairs(*op, cus) ? 16 : LatentPartsBytes(LineGroups(cus), kPromptRows, op->value);
}

extern "C" int llmp_hip_latent_prompt(const llmp_latent_prompt* op, void* scratch, size_t scratch_bytes, int cus, void* stream) {
  if (const int bad = CheckLatentPrompt(op, cus); bad != 0) return bad;
  const size_t need = llmp_hip_latent_prompt_scratch(op, cus);
  if (scratch == nullptr || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
    return Refuse(1, "latent_prompt: %zu bytes of scratch at a 16-byte boundary, not %zu", need, scratch_bytes);
  const bool whole = WholePairs(*op, cus);
  const int line_groups = LineGroups(cus);
  PromptArgs a;
  a.op = *op;
  a.tiles = TilesOf(*op);
  a.parts = LatentPartsAt(scratch, line_groups, kPromptRows);
  const JoinArgs join = {a.parts, op->out, op->out_token_stride, op->out_head_stride, op->heads, line_groups, 0};
  const auto s = static_cast<hipStream_t>(stream);
  BeginLaunches();
  const auto launch = [&](auto type, auto n, auto p, auto v) {
    constexpr int kType = decltype(type)::value, kN = decltype(n)::value, kP = decltype(p)::value, kV = decltype(v)::value;
    constexpr int kLds = PromptGeo<kN, kP, kV>::kLds;
    static bool sized[2] = {false, false};
    if (whole) {
      if (!AllowLds(reinterpret_cast<const void*>(&LatentPromptKernel<kType, kN, kP, kV, false>), kLds, &sized[0])) return;
      hipLaunchKernelGGL((LatentPromptKernel<kType, kN, kP, kV, false>), dim3(static_cast<unsigned>(WholeBlocks(*op))), dim3(kPromptThreads), kLds, s, a);
    } else {
      if (!AllowLds(reinterpret_cast<const void*>(&LatentPromptKernel<kType, kN, kP, kV, true>), kLds, &sized[1])) return;
      hipLaunchKernelGGL((LatentPromptKernel<kType, kN, kP, kV, true>), dim3(line_groups), dim3(kPromptThreads), kLds, s, a);
      hipLaunchKernelGGL((LatentJoinKernel<kType, kV, 32, kPromptRows>), dim3(line_groups, 2), dim3(kJoinWaves * kWave), 0, s, join);
    }
  };
  const auto sizes = [&](auto type) {
    const auto value = [&](auto n, auto p) {
      if (op->value == 64) launch(type, n, p, std::integral_constant<int, 64>{});
      if (op->value == 128) launch(type, n, p, std::integral_constant<int, 128>{});
    };
    const auto rope = [&](auto n) {
      if (op->rope_width == 32) value(n, std::integral_constant<int, 32>{});
      if (op->rope_width == 64) value(n, std::integral_constant<int, 64>{});
    };
    if (op->nope == 64) rope(std::integral_constant<int, 64>{});
    if (op->nope == 128) rope(std::integral_constant<int, 128>{});
  };
  if (op->type == LLMP_X_BF16) sizes(std::integral_constant<int, LLMP_X_BF16>{});
  if (op->type == LLMP_X_F16) sizes(std::integral_constant<int, LLMP_X_F16>{});
  return LaunchStatus("latent_prompt");
}
