// How the attentions over latent vectors cut a call's work evenly: pairs (a request's rows, some at a time, and the keys that they see) lie on one
// line, a request's after the other's, and every workgroup takes an equal run of it, so that one long request and many short ones fill the device alike.
// A run's first pair may have begun and its last one end in other workgroups: their parts are joined by a second launch. The line is counted in keys, kVisit more for
// a pair's beginning; a tile of keys is the workgroup's in whose run its first key lies.
#ifndef LLMP_AMD_CSRC_LATENT_LINE_H_
#define LLMP_AMD_CSRC_LATENT_LINE_H_

#include "latent.h"
#include "paged_attend.h"

namespace llmp_hip {

constexpr int kVisit = 64;  // what a pair's beginning and end cost, in keys

// The running maximum follows once it is kFollow (log2) behind; weights stay kUp above it, for F16's range.
constexpr float kUp = 8.0f, kFollow = 6.0f;

// Where parts go: a workgroup's later part of a pair that another began (0) and its first part of one that another ends (1).
struct LatentParts {
  float* values;    // [2 * workgroups][rows of a pair][width], in the order of the lanes' registers
  float2* numbers;  // [2 * workgroups][rows of a pair]: maximum, sum
  int32_t* which;   // [2 * workgroups][4]: the workgroup of its pair's first part (-1: no part here), pair, rows and 256 times the pair's parts, first row of the call's
};
inline size_t LatentPartsBytes(int groups, int rows, int width) { return static_cast<size_t>(2 * groups) * (16 + rows * (8 + 4 * static_cast<size_t>(width))); }
inline LatentParts LatentPartsAt(void* scratch, int groups, int rows) {
  LatentParts p;
  p.which = static_cast<int32_t*>(scratch);
  p.numbers = reinterpret_cast<float2*>(p.which + static_cast<size_t>(2 * groups) * 4);
  p.values = reinterpret_cast<float*>(p.numbers + static_cast<size_t>(2 * groups) * rows);
  return p;
}

// ---- device: a request's rows in groups of `t` tokens, the first at position `base`; a token sees the keys up to its position, of `length`.
struct LatentRequest {
  int start, n, length, base;  // PagedRequest's
  int groups;
};
// a / b, for a >= 0 and b > 0. (A division of 64 bits is 0.3 us where a wave waits for it, and hardly any line is that long.)
__device__ __forceinline__ int64_t Over(int64_t a, int64_t b) { return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b; }
// What group k's last token sees.
__device__ __forceinline__ int SeenOf(const LatentRequest& l, int t, int k) { return max(min(l.base + min((k + 1) * t, l.n), l.length), 0); }
// The line before group k, of one pair a group: the sum of min(base + (i + 1) t, most), none below 0, over i < k, and the visits.
__device__ __forceinline__ int64_t LineBefore(const LatentRequest& l, int64_t t, int k) {
  const int64_t most = max(min(l.length, l.base + l.n), 0);
  const int64_t low = l.base < 0 ? min(static_cast<int64_t>(k), Over(-static_cast<int64_t>(l.base), t)) : 0;
  const int64_t high = max(low, min(static_cast<int64_t>(k), most > l.base ? Over(most - static_cast<int64_t>(l.base), t) : 0));
  const int64_t risen = (high - low) * l.base + t * ((high * (high + 1) - low * (low + 1)) / 2);
  return risen + (k - high) * most + static_cast<int64_t>(k) * kVisit;
}
// The last group that begins at or before `u`.
__device__ __forceinline__ int GroupAt(const LatentRequest& l, int64_t t, int64_t u) {
  int k = 0, above = l.groups;
  while (above - k > 1) {
    const int mid = (k + above) / 2;
    if (LineBefore(l, t, mid) <= u) {
      k = mid;
    } else {
      above = mid;
    }
  }
  return k;
}

// Every wave by itself, a lane a request: length_of(r) is a request's of the line. The run [from, to) of this workgroup (`block` of `groups`), the request that
// holds its beginning, and the line before that. Eight workgroups in a row go to eight chiplets: runs side by side are on eight of them, or on one (CHIPLETS).
struct LatentRun {
  int64_t from, to, before, per;
  int request, index;
};
template <bool CHIPLETS, class LengthOf>
__device__ __forceinline__ LatentRun RunOf(int requests, int block, int groups, int64_t least, const LengthOf& length_of) {
  const int lane = threadIdx.x & (kWave - 1);
  const auto sums = [&](int64_t v) {  // inclusive
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
      const int64_t up = __shfl_up(v, m);
      v += lane >= m ? up : 0;
    }
    return v;
  };
  const auto from_lane = [](int64_t v, int l) {
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(v), l);
    return static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), l)) << 32 | low;
  };
  // (The first 64 requests' lengths are kept: most calls have no more.)
  const int64_t first = lane < requests ? length_of(lane) : 0, first_upto = sums(first);
  int64_t total = from_lane(first_upto, kWave - 1);
  for (int r0 = kWave; r0 < requests; r0 += kWave) total += from_lane(sums(r0 + lane < requests ? length_of(r0 + lane) : 0), kWave - 1);
  const int64_t per = max(Over(total + groups - 1, groups), least);
  int index = block;
  if constexpr (CHIPLETS) {
    // An eighth of the runs that there are to each chiplet, and so of the others (`groups` is a multiple of 8).
    const int chiplet = block % 8, i = block / 8, share = static_cast<int>((Over(total + per - 1, per) + 7) / 8);
    index = i < share ? chiplet * share + i : 8 * share + chiplet * (groups / 8 - share) + i - share;
  }
  LatentRun run = {index * per, min((index + 1) * per, total), 0, per, 0, index};
  if (run.from >= run.to) return run;
  for (int r0 = 0; r0 < requests; r0 += kWave) {
    const int64_t mine = r0 == 0 ? first : r0 + lane < requests ? length_of(r0 + lane) : 0;
    const int64_t upto = run.before + (r0 == 0 ? first_upto : sums(mine));
    const int passed = __popcll(__ballot(upto <= run.from));
    if (passed < kWave) {
      run.before = from_lane(upto - mine, passed);
      run.request = r0 + passed;
      break;
    }
    run.before = from_lane(upto, kWave - 1);
  }
  return run;
}

// What of a pair that sees `seen` keys lies in [x0, x1) of its kVisit + seen: tiles [from, to) of `tile` keys, whether they are its first and its last. A pair
// that sees nothing is its beginning's.
struct LatentPiece {
  int from, to;
  bool begins, ends, any;
};
__device__ __forceinline__ LatentPiece PieceOf(int seen, int tile, int x0, int x1) {
  const int tiles = (seen + tile - 1) / tile;
  LatentPiece p;
  p.from = (max(x0 - kVisit, 0) + tile - 1) / tile;
  p.to = x1 == seen + kVisit ? tiles : (max(x1 - kVisit, 0) + tile - 1) / tile;
  p.begins = p.from == 0 && (p.to > 0 || x0 == 0);
  p.ends = p.to == tiles;
  p.any = tiles == 0 ? x0 == 0 : p.from < p.to;
  return p;
}

template <class T>
__device__ __forceinline__ T Scalar(T v) {
  static_assert(sizeof(T) == 4, "32 bits");
  return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ LatentRequest Scalar(const LatentRequest& l) { return {Scalar(l.start), Scalar(l.n), Scalar(l.length), Scalar(l.base), Scalar(l.groups)}; }

// Which workgroups hold parts of a pair at `from` of the line: those from its first tile's to its last one's, each of which has a tile (a run is at least as long).
struct LatentOwners {
  int first, count;
};
__device__ __forceinline__ LatentOwners OwnersOf(int64_t from, int seen, int tile, int64_t per) {
  const int64_t first = Over(from + kVisit, per), last = Over(from + kVisit + static_cast<int64_t>(seen - 1) / tile * tile, per);
  return {static_cast<int>(first), static_cast<int>(last - first) + 1};
}

// ---- the parts of a pair, joined. They are as the lanes held them: an item is UNIT rows by 256 / UNIT dimensions, lane l four of them, 4 (l / UNIT) on, of row
// l % UNIT. The pair's items are dealt to the workgroups (one for each of the first launch's) that hold its parts, so that what one reads is
// about the same whatever the number of parts. A wave takes an item, or where there are many parts a workgroup one together, the waves' parts in turn. Bound by the
// parts' bytes where they are many (256 of 128 rows of 512 values, 67 MB: 17 to 27 us), else by four loads one after the other (16 rows: 5.6 us): a wave reads a
// part's numbers with its values and scales by a running maximum (the numbers first, for the maximum: 33 and 10 us). (One wave an item: 180 us.)
constexpr int kJoinWaves = 16, kJoinAhead = 4;
struct JoinArgs {
  LatentParts parts;
  void* out;
  int64_t out_token_stride, out_head_stride;
  int heads, groups;
  int pairs_a_token;  // 0: a pair is `heads`' of them: rows are tokens; 1: rows are (token, head); more: rows are heads
};
// grid (the first launch's workgroups, 2: by its later part of a pair, by its first one of another)
template <int TYPE, int WIDTH, int UNIT, int ROWS>
__global__ __launch_bounds__(kJoinWaves * kWave) void LatentJoinKernel(const JoinArgs a) {
  constexpr int kItemValues = 256 / UNIT, kBlocks = WIDTH / kItemValues;
  __shared__ F32x4 met[kJoinWaves - 1][kWave];
  __shared__ float2 met_numbers[kJoinWaves - 1][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, column = lane % UNIT, part_of = lane / UNIT;
  const int x = blockIdx.x;
  const int which = blockIdx.y;
  const I32x4 mine = *reinterpret_cast<const I32x4*>(a.parts.which + 8 * x + 4 * which);
  const int leader = mine[0], pair = mine[1], rows = mine[2] & 0xFF, count = mine[2] >> 8, token0 = mine[3];
  if (leader < 0) return;
  const auto unit = [&](int i, int u) { return static_cast<int64_t>(i == 0 ? 2 * leader + 1 : 2 * (leader + i)) * (ROWS / UNIT) + u; };
  const int items = (rows + UNIT - 1) / UNIT * kBlocks;
  // In loads that wait for each other; a meeting of the waves counts as one.
  const auto over = [](int n, int d) { return (n + d - 1) / d; };
  const bool together = over(items, count) * (over(count, kJoinAhead * kJoinWaves) + 1) < over(items, count * kJoinWaves) * over(count, kJoinAhead);
  const int waves = together ? 1 : kJoinWaves;
  for (int item = (x - leader) * waves + (together ? 0 : wave); item < items; item += count * waves) {
    const int u = item / kBlocks, block = item % kBlocks;
    float most = -INFINITY, sum = 0.0f;
    F32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    // (Four parts' loads at a time, the last one's again past the end, and nothing that they wait for: one after the other each waits for memory.)
    const int from = together ? wave : 0, step = together ? kJoinWaves : 1;
    for (int i0 = from; i0 < count; i0 += kJoinAhead * step) {
      float2 n[kJoinAhead];
      F32x4 x[kJoinAhead];
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const int64_t at = unit(min(i0 + j * step, count - 1), u);
        n[j] = a.parts.numbers[at * UNIT + column];
        x[j] = reinterpret_cast<const F32x4*>(a.parts.values)[(at * kBlocks + block) * kWave + lane];
      }
      const float before = most;
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) most = fmaxf(most, n[j].x);
      const float less = most == -INFINITY ? 0.0f : most, keeps = __builtin_amdgcn_exp2f(before - less);
      sum *= keeps, v *= keeps;
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        if (i0 + j * step < count) {
          const float by = __builtin_amdgcn_exp2f(n[j].x - less);
          sum = fmaf(n[j].y, by, sum), v += x[j] * by;
        }
      }
    }
    if (together) {
      if (wave > 0) met[wave - 1][lane] = v, met_numbers[wave - 1][lane] = make_float2(most, sum);
      __syncthreads();
      if (wave == 0) {
        const float own = most;
        for (int i = 0; i < kJoinWaves - 1; ++i) most = fmaxf(most, met_numbers[i][lane].x);
        const float less = most == -INFINITY ? 0.0f : most, keeps = __builtin_amdgcn_exp2f(own - less);
        sum *= keeps, v *= keeps;
        for (int i = 0; i < kJoinWaves - 1; ++i) {
          const float by = __builtin_amdgcn_exp2f(met_numbers[i][lane].x - less);
          sum = fmaf(met_numbers[i][lane].y, by, sum), v += met[i][lane] * by;
        }
      }
      __syncthreads();
    }
    const int row = UNIT * u + column;
    if (row < rows && (!together || wave == 0)) {
      const float by = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
      const float out[4] = {v[0] * by, v[1] * by, v[2] * by, v[3] * by};
      const int token = token0 + (a.pairs_a_token == 0 ? row : a.pairs_a_token == 1 ? row / a.heads : 0);
      const int head = a.pairs_a_token == 0 ? pair % a.heads : a.pairs_a_token == 1 ? row % a.heads : pair % a.pairs_a_token * ROWS + row;
      StoreValues<TYPE, 4>(a.out, token * a.out_token_stride + head * a.out_head_stride + kItemValues * block + 4 * part_of, out);
    }
  }
}

}  // namespace llmp_hip

#endif  // LLMP_AMD_CSRC_LATENT_LINE_H_
