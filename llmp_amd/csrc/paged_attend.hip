// llmp.paged.attend, the form for few rows: decode steps, drafted tokens, and queries with page lists of their own.
//
// What bounds it is the cache's bytes: every K and V byte a request sees is read once for all the query heads of its KV head (up to
// 16 (token, head) rows together). The work is cut evenly: all requests' tiles of 64 tokens, of every KV head, lie on one
// line, and each of a fixed number of workgroups takes an equal run of it, so one long request or many short ones fill the
// device alike. A workgroup's part of a (rows, head) segment that others share goes to scratch and a second launch joins the
// parts; a segment that one workgroup has whole is finished there.
//
// A wave takes a tile alone, its operands straight from memory into the matrix instructions' registers, no LDS:
//   S^T = K Q^T by v_mfma_i32_16x16x64_i8: a lane brings 16 bytes of a token's K row. Row 4a + b of the t-th product is token
//   16a + 4t + b of the tile, so that a lane ends with 16 consecutive tokens (16 g to 16 g + 15, g its group of lanes) of one
//   query row. That is the order in which
//   O^T += V^T P^T by v_mfma_f32_16x16x32_f16 takes P from the same lane's registers, and in which V, stored with the tokens
//   innermost, is 16 bytes of one dimension a lane.
// A lane's 16 tokens are of one page (pages are multiples of 16): one scale each for K and V.
#include <cmath>
#include <type_traits>

#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kFewWaves = 4;
constexpr int kFewThreads = kFewWaves * kWave;
constexpr int kRows = 16;  // rows of a segment: (token, head) pairs

// A request's segments and tiles in this form; units = segments * tiles.
struct FewRequest {
  PagedRequest q;
  int segments;    // row chunks times KV heads
  int first_tile;  // tiles before it lie before every row's window
  int tiles;
  int64_t units;
};
template <bool LISTS>
__device__ __forceinline__ FewRequest FewOf(const PagedAttendArgs& a, int r) {
  const llmp_paged_attend& op = a.op;
  FewRequest f;
  f.q = RequestOf(op.starts, op.lengths, r, op.tokens, a.most_length);
  f.first_tile = 0;
  int chunks;
  if constexpr (LISTS) {
    chunks = f.q.n * ((a.group + kRows - 1) / kRows);
    f.tiles = (op.list_pages * op.cache.page + kTileTokens - 1) / kTileTokens;
  } else {
    const int64_t rows = static_cast<int64_t>(f.q.n) * a.group;
    chunks = rows > a.few_rows ? 0 : static_cast<int>((rows + kRows - 1) / kRows);
    if (op.window > 0) f.first_tile = max(f.q.length - f.q.n - op.window + 1, 0) / kTileTokens;
    f.tiles = max((f.q.length + kTileTokens - 1) / kTileTokens - f.first_tile, 1);  // (a row that sees nothing is written too)
  }
  f.segments = chunks * op.cache.kv_heads;
  f.units = static_cast<int64_t>(f.segments) * f.tiles;
  return f;
}

// Where a lane's 16 tokens lie.
struct Place {
  int page;  // in the cache, -1: none
  int position;
  int offset;  // in the page
};

__device__ __forceinline__ int64_t WaveSum64(int64_t v) {
#pragma unroll
  for (int step = 1; step < kWave; step <<= 1) v += __shfl_xor(v, step);
  return v;
}

// grid (workgroups).
template <int TYPE, int D, bool LISTS>
__global__ __launch_bounds__(kFewThreads, 2) void FewKernel(const PagedAttendArgs a) {
  constexpr int kDig = kDigits<TYPE>;
  constexpr int kSteps = D / 64, kBlocks = D / 16;  // inner steps of K's product, row blocks of V's
  constexpr int kPitch = D + 4;
  extern __shared__ __attribute__((aligned(16))) float meet[];  // [wave][row][kPitch]
  __shared__ float tops[kFewWaves][kRows], sums[kFewWaves][kRows];
  const llmp_paged_attend& op = a.op;
  const llmp_paged_cache& c = op.cache;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int group_of = lane >> 4, column = lane & 15;

  // ---- this workgroup's run of the line of units.
  int64_t total = 0;
  for (int base = 0; base < op.requests; base += kWave) total += WaveSum64(base + lane < op.requests ? FewOf<LISTS>(a, base + lane).units : 0);
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  per = (per + kFewWaves - 1) / kFewWaves * kFewWaves;  // whole rounds of the waves
  int64_t u = blockIdx.x * per;
  const int64_t u_end = min(u + per, total);
  I32x4 part = {-1, 0, 0, 0};
  if (u >= u_end) {
    if (tid == 0) *reinterpret_cast<I32x4*>(a.parts + 4 * blockIdx.x) = part;
    return;
  }
  // The request that holds unit u, and the units before it.
  int r = 0;
  int64_t before = 0;
  for (int base = 0, found = 0; base < op.requests && !found; base += kWave) {
    const int64_t mine = base + lane < op.requests ? FewOf<LISTS>(a, base + lane).units : 0;
    int64_t upto = mine;
#pragma unroll
    for (int step = 1; step < kWave; step <<= 1) {
      const int64_t other = __shfl_up(upto, step);
      if (lane >= step) upto += other;
    }
    const uint64_t past = __ballot(before + upto > u);
    if (past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      r = base + at;
      before += __shfl(upto - mine, at);
      found = 1;
    } else {
      before += __shfl(upto, kWave - 1);
    }
  }
  r = __builtin_amdgcn_readfirstlane(r);

  while (u < u_end && r < op.requests) {
    const FewRequest f = FewOf<LISTS>(a, r);
    if (u >= before + f.units) {
      before += f.units;
      ++r;
      continue;
    }
    const int segment = __builtin_amdgcn_readfirstlane(static_cast<int>((u - before) / f.tiles));
    const int t_first = __builtin_amdgcn_readfirstlane(static_cast<int>((u - before) % f.tiles));
    const int t_count = static_cast<int>(min(static_cast<int64_t>(f.tiles - t_first), u_end - u));
    const int head = segment % c.kv_heads, chunk = segment / c.kv_heads;

    // ---- this lane's query row, and what the segment's rows see.
    int token, query_head, first_token, last_token;
    bool real;
    if constexpr (LISTS) {
      const int a_token = (a.group + kRows - 1) / kRows;
      first_token = last_token = token = chunk / a_token;
      query_head = kRows * (chunk % a_token) + column;
      real = query_head < a.group;
    } else {
      const int row = kRows * chunk + column;
      token = row / a.group;
      query_head = row % a.group;
      real = row < f.q.n * a.group;
      first_token = kRows * chunk / a.group;
      last_token = min((kRows * chunk + kRows - 1) / a.group, f.q.n - 1);
    }
    const int base_position = f.q.length - f.q.n;  // of the request's first new token
    const int position = base_position + token;
    const int window = op.window > 0 ? op.window : INT_MAX / 2;
    const int see_from = max(position - window + 1, 0), see_to = real ? position + 1 : 0;
    const int all_from = max(base_position + last_token - window + 1, 0), all_to = base_position + first_token + 1;  // seen by every row
    const int any_from = max(base_position + first_token - window + 1, 0), any_to = base_position + last_token + 1;  // seen by any

    I32x4 digits[kDig][kSteps];
    float unit;  // a digit product's worth in log2 units, but for K's scale
    {
      float x[kSteps][16];
      const int64_t from = (f.q.start + (real ? token : 0)) * op.q_token_stride + (head * a.group + (real ? query_head : 0)) * op.q_head_stride;
      float most = 0.0f;
      bool finite = true;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float v[8];
          LoadEight<TYPE>(op.q, from + 64 * s + 16 * group_of + 8 * half, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[s][8 * half + e] = v[e];
            finite = finite && fabsf(v[e]) <= 3.402823466e38f;
            most = fmaxf(most, fabsf(v[e]));
          }
        }
      }
      most = AcrossGroupsMax(most);
      const float bad = AcrossGroupsMax(finite ? 0.0f : 1.0f);
      // (A row of zeros, or of magnitudes whose reciprocal is none, is zeros; one with an infinity or a NaN has no logits.)
      const bool small = !(most > 0x1p-100f);
      const float inverse = small ? 0.0f : kDigitMax<TYPE> / most;
      unit = bad > 0.0f ? __builtin_nanf("") : small ? 0.0f : most / kDigitMax<TYPE>;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t packed[kDig];
#pragma unroll
          for (int k = 0; k < kDig; ++k) packed[k] = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            int digit[kDig];
            SplitDigits<kDig>(bad > 0.0f || !real ? 0 : static_cast<int>(rintf(x[s][4 * w + e] * inverse)), digit);
#pragma unroll
            for (int k = 0; k < kDig; ++k) packed[k] |= static_cast<uint32_t>(digit[k] & 0xFF) << (8 * e);
          }
#pragma unroll
          for (int k = 0; k < kDig; ++k) digits[k][s][w] = static_cast<int>(packed[k]);
        }
      }
      unit *= op.softcap != 0.0f ? op.scale : op.scale * kLog2E;
    }
    const float cap_inverse = op.softcap != 0.0f ? 1.0f / op.softcap : 0.0f;

    // ---- the places of a tile's tokens.
    const int32_t* const table = op.table + r * op.table_stride;
    const int32_t* const list =
        LISTS ? op.lists + (static_cast<int64_t>(f.q.start + token) * c.kv_heads + head) * op.list_pages : nullptr;
    const int p16 = c.page / 16;
    const auto place_of = [&](int tile) {
      Place at;
      const int n16 = 4 * tile + group_of;
      int entry = static_cast<int>(PagedDivide(n16, a.page_magic));
      at.offset = 16 * (n16 - entry * p16);
      if constexpr (LISTS) entry = entry < op.list_pages ? list[entry] : -1;
      at.page = -1;
      at.position = 0;
      if (entry >= 0 && entry < op.table_width) {
        at.position = entry * c.page + at.offset;
        if (at.position < f.q.length) at.page = table[entry];
      }
      if (at.page >= c.pages) at.page = -1;
      return at;
    };
    const int tile_end = t_first + t_count + f.first_tile;
    int tile = t_first + f.first_tile + wave;
    int stop = tile_end;
    if constexpr (!LISTS) {  // tiles that no row of this chunk sees
      while (tile < stop && (tile + 1) * kTileTokens <= any_from) tile += kFewWaves;
      stop = min(stop, max(any_to + kTileTokens - 1, 0) / kTileTokens);
    }

    float top = -INFINITY, sum = 0.0f;
    F32x4 out[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) out[b] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // ---- the loads of a tile: K by (token row, inner step), V by block of dimensions, the scales of the lane's page.
    I32x4 k[4][kSteps];
    U32x4 v[kBlocks];
    float ks = 0.0f, vs = 0.0f;
    const int64_t page_bytes = static_cast<int64_t>(c.kv_heads) * c.page * D;
    const uint8_t* const k_base = static_cast<const uint8_t*>(c.k) + static_cast<int64_t>(head) * c.page * D + 16 * group_of + (column & 3) * D;
    const uint8_t* const v_base = static_cast<const uint8_t*>(c.v) + static_cast<int64_t>(head) * c.page * D + column * c.page;
    const auto load_k = [&](const Place& at) {
      // K's row `column` of product t is token 16 (column / 4) + 4 t + column % 4: of another group's page.
      const int page = max(__shfl(at.page, (column >> 2) * 16), 0), offset = __shfl(at.offset, (column >> 2) * 16);
      const uint8_t* from = k_base + page * page_bytes + offset * D;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) k[t][s] = *reinterpret_cast<const I32x4*>(from + 4 * t * D + 64 * s);
      }
    };
    const auto load_v = [&](const Place& at) {
      const uint8_t* from = v_base + max(at.page, 0) * page_bytes + at.offset;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) v[b] = *reinterpret_cast<const U32x4*>(from + 16 * b * c.page);
    };
    const auto load_scales = [&](const Place& at, float* to_k, float* to_v) {
      const int64_t i = static_cast<int64_t>(max(at.page, 0)) * c.kv_heads + head;
      *to_k = c.k_scale[i], *to_v = c.v_scale[i];
    };
    Place here = {-1, 0, 0}, next = {-1, 0, 0};
    if (tile < stop) {
      here = place_of(tile);
      load_k(here);
      load_scales(here, &ks, &vs);
      load_v(here);
      if (tile + kFewWaves < stop) next = place_of(tile + kFewWaves);
    }
    for (; tile < stop; tile += kFewWaves) {
      const bool more = tile + kFewWaves < stop;
      float next_ks = 0.0f, next_vs = 0.0f;
      // ---- S^T = K Q^T
      I32x4 dots[kDig][4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int d = 0; d < kDig; ++d) {
          I32x4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < kSteps; ++s) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][s], digits[d][s], acc, 0, 0, 0);
          dots[d][t] = acc;
        }
      }
      if (more) load_k(next), load_scales(next, &next_ks, &next_vs);
      Place after = {-1, 0, 0};
      if (tile + 2 * kFewWaves < stop) after = place_of(tile + 2 * kFewWaves);
      // ---- the tile's softmax
      float s[16];
      const float worth = unit * ks;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = JoinDigits<kDig>(dots[0][i / 4][i % 4], kDig == 3 ? dots[1][i / 4][i % 4] : 0, dots[kDig - 1][i / 4][i % 4]);
      }
      if (op.softcap != 0.0f) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = Capped<TYPE>(s[i] * worth, op.softcap, cap_inverse) * kLog2E;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] *= worth;
      }
      bool whole = __all(here.page >= 0);
      if constexpr (LISTS) {
        whole = whole && __all(here.position + 16 <= all_to && here.position >= all_from);
      } else {
        whole = whole && (tile + 1) * kTileTokens <= all_to && tile * kTileTokens >= all_from;
      }
      uint32_t seen = 0xFFFFu;
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int p = here.position + i;
          const bool sees = here.page >= 0 && p >= see_from && p < see_to;
          seen |= sees ? 1u << i : 0u;
          s[i] = sees ? s[i] : -INFINITY;
        }
        if (here.page < 0) vs = 0.0f;
      }
      float peak = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) peak = fmaxf(peak, s[i]);
      peak = AcrossGroupsMax(peak + ScaleLog(vs));
      if (__any(peak > top)) {
        const float higher = fmaxf(top, peak);
        const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
        top = higher;
        sum *= keep;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) out[b] *= keep;
      }
      const float from = top == -INFINITY ? 0.0f : top;
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(s[i] - from);
        sum += p[i];
        p[i] *= vs;
      }
      if (!whole) {  // (a hidden token's weight is zero whatever its page's scale is)
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = (seen >> i) & 1u ? p[i] : 0.0f;
      }
      F16x8 w[2], w_low[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        w[i / 8][i % 8] = static_cast<_Float16>(p[i]);
        if constexpr (kDig == 3) w_low[i / 8][i % 8] = static_cast<_Float16>(p[i] - static_cast<float>(w[i / 8][i % 8]));
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const F16x8 v0 = EightCodes(v[b][0], v[b][1]), v1 = EightCodes(v[b][2], v[b][3]);
        out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w[0], out[b], 0, 0, 0);
        out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w[1], out[b], 0, 0, 0);
        if constexpr (kDig == 3) {
          out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w_low[0], out[b], 0, 0, 0);
          out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w_low[1], out[b], 0, 0, 0);
        }
      }
      if (more) load_v(next);
      here = next, next = after, ks = next_ks, vs = next_vs;
    }
    sum = AcrossGroupsSum(sum);

    // ---- the waves' results meet.
    if (group_of == 0) tops[wave][column] = top, sums[wave][column] = sum;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      *reinterpret_cast<F32x4*>(meet + (wave * kRows + column) * kPitch + 16 * b + 4 * group_of) = out[b];
    __syncthreads();
    const bool begins = t_first == 0, ends = t_first + t_count == f.tiles;
    float* const slot = a.partial + (2 * static_cast<int64_t>(blockIdx.x) + (begins ? 1 : 0)) * kRows * (D + 2);
    for (int i = tid; i < kRows * D / 4; i += kFewThreads) {
      const int row = i / (D / 4), d = 4 * (i % (D / 4));
      float high = -INFINITY, all = 0.0f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) high = fmaxf(high, tops[w][row]);
      F32x4 value = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        const float keep = tops[w][row] == -INFINITY ? (high == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(tops[w][row] - high);
        all += sums[w][row] * keep;
        value += *reinterpret_cast<const F32x4*>(meet + (w * kRows + row) * kPitch + d) * keep;
      }
      if (begins && ends) {
        int to_token, to_head;
        bool is_real;
        if constexpr (LISTS) {
          to_token = token, to_head = kRows * (chunk % ((a.group + kRows - 1) / kRows)) + row, is_real = to_head < a.group;
        } else {
          const int at = kRows * chunk + row;
          to_token = at / a.group, to_head = at % a.group, is_real = at < f.q.n * a.group;
        }
        if (is_real) {
          const int h = head * a.group + to_head;
          if (op.sinks != nullptr) all += __builtin_amdgcn_exp2f(fmaf(op.sinks[h], kLog2E, -(high == -INFINITY ? 0.0f : high)));
          const float inverse = all == 0.0f ? 0.0f : 1.0f / all;
          const float x[4] = {value[0] * inverse, value[1] * inverse, value[2] * inverse, value[3] * inverse};
          StoreValues<TYPE, 4>(op.out, (f.q.start + to_token) * op.out_token_stride + h * op.out_head_stride + d, x);
        }
      } else {
        float* const to = slot + row * (D + 2);
        if (d == 0) to[0] = high, to[1] = all;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[2 + d + e] = value[e];
      }
    }
    if (begins && !ends) part = I32x4{static_cast<int>((before + static_cast<int64_t>(segment + 1) * f.tiles - 1) / per), r, segment, 0};
    __syncthreads();
    u += t_count;
  }
  if (tid == 0) *reinterpret_cast<I32x4*>(a.parts + 4 * blockIdx.x) = part;
}

// grid (workgroups of the first launch, 4): the parts of the segment that begins in workgroup x and ends in another, a
// wave a row.
template <int TYPE, int D, bool LISTS>
__global__ __launch_bounds__(kFewThreads) void FewJoinKernel(const PagedAttendArgs a) {
  constexpr int kPer = D / kWave;
  const llmp_paged_attend& op = a.op;
  const I32x4 part = *reinterpret_cast<const I32x4*>(a.parts + 4 * blockIdx.x);
  if (part.x < 0) return;
  const int lane = threadIdx.x & (kWave - 1), row = 4 * blockIdx.y + threadIdx.x / kWave;
  const int r = part.y, head = part.z % op.cache.kv_heads, chunk = part.z / op.cache.kv_heads;
  const PagedRequest q = RequestOf(op.starts, op.lengths, r, op.tokens, a.most_length);
  int token, query_head;
  bool real;
  if constexpr (LISTS) {
    const int a_token = (a.group + kRows - 1) / kRows;
    token = chunk / a_token, query_head = kRows * (chunk % a_token) + row, real = query_head < a.group;
  } else {
    const int at = kRows * chunk + row;
    token = at / a.group, query_head = at % a.group, real = at < q.n * a.group;
  }
  if (!real) return;
  constexpr int64_t kSlot = kRows * (D + 2);
  const int first = blockIdx.x, last = part.x;
  const auto slot_of = [&](int w) { return a.partial + (2 * static_cast<int64_t>(w) + (w == first ? 1 : 0)) * kSlot + row * (D + 2); };
  float high = -INFINITY;
  for (int w = first + lane; w <= last; w += kWave) high = fmaxf(high, slot_of(w)[0]);
#pragma unroll
  for (int step = 1; step < kWave; step <<= 1) high = fmaxf(high, __shfl_xor(high, step));
  float all = 0.0f, value[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) value[e] = 0.0f;
#pragma unroll 8
  for (int w = first; w <= last; ++w) {
    const float* from = slot_of(w);
    const float top = from[0];
    const float keep = top == -INFINITY ? (high == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(top - high);
    all += from[1] * keep;
#pragma unroll
    for (int e = 0; e < kPer; ++e) value[e] += from[2 + kPer * lane + e] * keep;
  }
  const int h = head * a.group + query_head;
  if (op.sinks != nullptr) all += __builtin_amdgcn_exp2f(fmaf(op.sinks[h], kLog2E, -(high == -INFINITY ? 0.0f : high)));
  const float inverse = all == 0.0f ? 0.0f : 1.0f / all;
  const int64_t to = (q.start + token) * op.out_token_stride + h * op.out_head_stride + kPer * lane;
#pragma unroll
  for (int e = 0; e < kPer; ++e) StoreOne<TYPE>(op.out, to + e, value[e] * inverse);
}

// Workgroups of the few rows' launch: two a compute unit (their registers' limit), a wave of each a SIMD.
int FewGroups(int cus) { return 2 * (cus > 0 ? cus : 256); }

size_t PartBytes(int groups) { return static_cast<size_t>(groups) * 4 * sizeof(int32_t); }
size_t FewScratch(int head_dim, int cus) {
  const int groups = FewGroups(cus);
  return PartBytes(groups) + 2 * static_cast<size_t>(groups) * kRows * (head_dim + 2) * sizeof(float);
}

// Requests of more rows than this are the many rows' form's, where the call has any.
constexpr int kFewRows = 64;
bool HasMany(const llmp_paged_attend& op) {
  return op.lists == nullptr && static_cast<int64_t>(op.most_tokens < op.tokens ? op.most_tokens : op.tokens) * (op.heads / op.cache.kv_heads) > kFewRows;
}
size_t AttendScratch(const llmp_paged_attend& op, int cus) {
  return FewScratch(op.cache.head_dim, cus) + (HasMany(op) ? PagedManyScratch(op, cus) : 0);
}

template <int TYPE, int D, bool LISTS>
void LaunchFew(const PagedAttendArgs& args, int groups, hipStream_t stream) {
  constexpr int kLds = kFewWaves * kRows * (D + 4) * static_cast<int>(sizeof(float));
  static bool sized = false;
  if (kLds > 32768 && !AllowLds(reinterpret_cast<const void*>(&FewKernel<TYPE, D, LISTS>), kLds, &sized)) return;
  hipLaunchKernelGGL((FewKernel<TYPE, D, LISTS>), dim3(groups), dim3(kFewThreads), kLds, stream, args);
  hipLaunchKernelGGL((FewJoinKernel<TYPE, D, LISTS>), dim3(groups, kRows / 4), dim3(kFewThreads), 0, stream, args);
}

template <int TYPE, int D>
void LaunchFewFor(const PagedAttendArgs& args, int groups, hipStream_t stream) {
  if (args.op.lists != nullptr) {
    LaunchFew<TYPE, D, true>(args, groups, stream);
  } else {
    LaunchFew<TYPE, D, false>(args, groups, stream);
  }
}
template <int TYPE>
void LaunchFewOf(const PagedAttendArgs& args, int groups, hipStream_t stream) {
  if (args.op.cache.head_dim == 64) LaunchFewFor<TYPE, 64>(args, groups, stream);
  if (args.op.cache.head_dim == 128) LaunchFewFor<TYPE, 128>(args, groups, stream);
  if (args.op.cache.head_dim == 256) LaunchFewFor<TYPE, 256>(args, groups, stream);
}

int CheckAttend(const llmp_paged_attend* op) {
  if (op == nullptr) return Refuse(1, "paged_attend: null operands");
  if (const int bad = CheckPagedCache("paged_attend", op->cache, false); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_attend", "q", op->q, op->q_token_stride, op->q_head_stride, op->type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_attend", "out", op->out, op->out_token_stride, op->out_head_stride, op->type); bad != 0) return bad;
  if (op->requests < 1 || op->requests > 1 << 24 || op->tokens < 1 || op->most_tokens < 1 || op->table_width < 1)
    return Refuse(1, "paged_attend: 1 to 2^24 requests, at least one token and one page a table row (%d, %d, %d, %d)", op->requests, op->tokens,
                  op->most_tokens, op->table_width);
  if (op->heads < 1 || op->heads % op->cache.kv_heads != 0 || static_cast<int64_t>(op->heads) * op->tokens > INT_MAX)
    return Refuse(1, "paged_attend: a whole number of query heads a KV head (%d, %d), at most 2^31 of them in all tokens", op->heads, op->cache.kv_heads);
  if (op->lengths == nullptr || op->starts == nullptr || op->table == nullptr) return Refuse(1, "paged_attend: null operand");
  if ((reinterpret_cast<uintptr_t>(op->lengths) | reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->table) |
       reinterpret_cast<uintptr_t>(op->lists) | reinterpret_cast<uintptr_t>(op->sinks)) % 4 != 0)
    return Refuse(1, "paged_attend: I32 and F32 arrays at 4-byte boundaries");
  if (op->table_stride < op->table_width) return Refuse(1, "paged_attend: a table row of %d entries every %lld", op->table_width, (long long)op->table_stride);
  if (static_cast<int64_t>(op->table_width) * op->cache.page > kMostPagedLength) return Refuse(1, "paged_attend: a table row of at most 2^30 tokens");
  if (op->lists != nullptr && (op->list_pages < 1 || static_cast<int64_t>(op->list_pages) * op->cache.page > kMostPagedLength))
    return Refuse(1, "paged_attend: lists of one to 2^30 tokens' pages, not %d pages", op->list_pages);
  if (op->window < 0) return Refuse(1, "paged_attend: a window of no or some tokens, not %d", op->window);
  if (!std::isfinite(op->scale)) return Refuse(1, "paged_attend: a finite scale");
  if (!(op->softcap >= 0.0f) || !std::isfinite(op->softcap)) return Refuse(1, "paged_attend: a finite softcap, 0 for none");
  return 0;
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" size_t llmp_hip_paged_attend_scratch(const llmp_paged_attend* op, int cus) {
  if (CheckAttend(op) != 0) return 0;
  return AttendScratch(*op, cus);
}

extern "C" int llmp_hip_paged_attend(const llmp_paged_attend* op, void* scratch, size_t scratch_bytes, int cus, void* stream) {
  if (const int bad = CheckAttend(op); bad != 0) return bad;
  const size_t needs = AttendScratch(*op, cus);
  if (scratch == nullptr || scratch_bytes < needs || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
    return Refuse(1, "paged_attend: %zu bytes of scratch at a 16-byte boundary, %zu given", needs, scratch_bytes);
  BeginLaunches();
  PagedAttendArgs args;
  args.op = *op;
  const int groups = FewGroups(cus);
  args.parts = static_cast<int32_t*>(scratch);
  args.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + PartBytes(groups));
  const uint32_t p16 = static_cast<uint32_t>(op->cache.page / 16);
  args.page_magic = p16 == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / p16 + 1);
  args.group = op->heads / op->cache.kv_heads;
  args.most_length = op->table_width * op->cache.page;
  const bool many = HasMany(*op);
  args.few_rows = many ? kFewRows : INT_MAX;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (many) PagedManyRows(args, static_cast<uint8_t*>(scratch) + FewScratch(op->cache.head_dim, cus), cus, on);
  if (many && op->requests == 1 && op->most_tokens == op->tokens) return LaunchStatus("paged_attend");  // the one request has been answered
  if (op->type == LLMP_X_F32) LaunchFewOf<LLMP_X_F32>(args, groups, on);
  if (op->type == LLMP_X_BF16) LaunchFewOf<LLMP_X_BF16>(args, groups, on);
  if (op->type == LLMP_X_F16) LaunchFewOf<LLMP_X_F16>(args, groups, on);
  return LaunchStatus("paged_attend");
}
