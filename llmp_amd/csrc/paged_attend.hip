// llmp.paged.attend, the form for few rows: decode steps, drafted tokens, and queries with page lists of their own.
//
// What bounds it is the cache's bytes: every K and V byte a request sees is read once for all the query heads of its KV head (up to
// 16 (token, head) rows together). The work is cut evenly: all requests' tiles of 64 tokens, of every KV head, lie on one
// line, and each of a fixed number of workgroups takes an equal run of it, so one long request or many short ones fill the
// device alike. A workgroup's part of a (rows, head) segment that others share goes to scratch and a second launch joins the
// parts; a segment that one workgroup has whole is finished there.
//
// A wave takes a tile alone. Its K and V come to the wave's own part of LDS without a register waiting for them (a whole tile is on its
// way under another's work), and from there into the matrix instructions' registers:
//   S^T = K Q^T by v_mfma_i32_16x16x64_i8: a lane brings 16 bytes of a token's K row. Row 4a + b of the t-th product is token
//   16a + 4t + b of the tile, so that a lane ends with 16 consecutive tokens (16 g to 16 g + 15, g its group of lanes) of one
//   query row. That is the order in which
//   O^T += V^T P^T by v_mfma_f32_16x16x32_f16 takes P from the same lane's registers, and in which V, stored with the tokens
//   innermost, is 16 bytes of one dimension a lane.
// A lane's 16 tokens are of one page (pages are multiples of 16): one scale each for K and V.
//
// Measured (both launches, 8 KV heads): 131072 tokens of one request at head size 128, 268 MB, 61.6 us, 4.4 TB/s (a large copy reaches
// 4.9, a read alone 7.0); 32 requests of up to 16384 tokens, 453 MB, 98 us, 4.6 TB/s; 8192 tokens at 256 in F32, 34 MB, a tile a
// wave, 19.7 us: that is the chain of a launch, the lengths, the table, one tile and the waves' meeting, and the join's.
#include <cmath>
#include <type_traits>

#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kFewWaves = 4;
constexpr int kFewThreads = kFewWaves * kWave;
constexpr int kRows = 16;  // rows of a segment: (token, head) pairs
constexpr uint32_t kVisit = 8;  // what a segment's beginning and end cost a workgroup, in tiles

// A request's segments and tiles in this form. A unit of the line is 2^shift tiles of a segment (shift 0 but where the line would
// pass 2^31).
struct FewRequest {
  PagedRequest q;
  int segments;    // row chunks times KV heads
  int first_tile;  // tiles before it lie before every row's window
  int tiles;
  uint32_t units;
};
// A segment's units: whole rounds of the workgroup's waves, so that a run of rounds ends where a segment does (a workgroup with the
// end of one and the beginning of another takes both their visits: 217 tokens of a request and two shorter ones, 25 us and 13).
__device__ __forceinline__ uint32_t SegmentUnits(int tiles, int shift, uint32_t round) {
  if (shift > 0) return static_cast<uint32_t>(((tiles - 1) >> shift) + 1);
  return round == kFewWaves ? (static_cast<uint32_t>(tiles) + kFewWaves - 1) / kFewWaves * kFewWaves : (static_cast<uint32_t>(tiles) + round - 1) / round * round;
}
template <bool LISTS>
__device__ __forceinline__ FewRequest FewOf(const PagedAttendArgs& a, int r, uint32_t round) {
  const llmp_paged_attend& op = a.op;
  FewRequest f;
  f.q = RequestOf(op.starts, op.lengths, op.before, r, op.tokens, a.most_length);
  f.first_tile = 0;
  int chunks;
  if constexpr (LISTS) {
    chunks = f.q.n * ((a.group + kRows - 1) / kRows);
    f.tiles = (op.list_pages * op.cache.page + kTileTokens - 1) / kTileTokens;
  } else {
    const int64_t rows = static_cast<int64_t>(f.q.n) * a.group;
    chunks = rows > a.few_rows ? 0 : static_cast<int>((rows + kRows - 1) / kRows);
    if (op.window > 0) f.first_tile = max(f.q.base - op.window + 1, 0) / kTileTokens;
    f.tiles = max((f.q.length + kTileTokens - 1) / kTileTokens - f.first_tile, 1);  // (a row that sees nothing is written too)
  }
  f.segments = chunks * op.cache.kv_heads;
  f.units = static_cast<uint32_t>(f.segments) * SegmentUnits(f.tiles, a.shift, round);
  return f;
}
// Lane `lane`'s in every lane.
__device__ __forceinline__ FewRequest FewFrom(const FewRequest& f, int lane) {
  const auto from = [&](int v) { return __builtin_amdgcn_readlane(v, lane); };
  return {{from(f.q.start), from(f.q.n), from(f.q.length), from(f.q.base)}, from(f.segments), from(f.first_tile), from(f.tiles), static_cast<uint32_t>(from(static_cast<int>(f.units)))};
}

// A tile of K and V of a head.
constexpr int TileBytes(int head_dim) { return 2 * kTileTokens * head_dim; }
constexpr int FewLds(int head_dim) {
  const int land = kFewWaves * TileBytes(head_dim), meet = kFewWaves * kRows * (head_dim + 4) * 4;
  return land > meet ? land : meet;
}
// Workgroups a compute unit: by registers and LDS, 128 KB of tiles on their way either way (96 KB at 64).
constexpr int FewAUnit(int head_dim) { return head_dim == 64 ? 3 : head_dim == 128 ? 2 : 1; }
// Where a lane's 16 tokens of a tile lie.
struct Place {
  int page;  // in the cache, -1: none
  int position;
  int offset;  // in the page
  bool there;
};
struct Entry {
  int entry;  // of the table row
  int offset;
  bool there;
};

// Workgroup `block` of `blocks`, of which `used` have work, on the line: the device deals the workgroups to its eight chiplets in
// turn, each with an L2 of its own, and a chiplet's take a run of the line, since the rows of a (request, KV head), which share its
// pages, lie side by side there.
constexpr uint32_t kChiplets = 8;
__device__ __forceinline__ uint32_t OnChiplet(uint32_t block, uint32_t blocks, uint32_t used) {
  if (blocks % kChiplets != 0) return block;
  const uint32_t chiplet = block % kChiplets, slot = block / kChiplets, run = (used + kChiplets - 1) / kChiplets;
  return slot < run ? chiplet * run + slot : block;  // (run slots of every chiplet come first: the others keep their places)
}

// grid (workgroups).
template <int TYPE, int D, bool LISTS>
__global__ __launch_bounds__(kFewThreads, FewAUnit(D)) void FewKernel(const PagedAttendArgs a) {
  constexpr int kDig = kDigits<TYPE>;
  constexpr int kSteps = D / 64, kBlocks = D / 16;  // inner steps of K's product, row blocks of V's
  constexpr int kMine = kTileTokens / 4, kProducts = kTileTokens / 16;  // a lane's tokens of a tile, products of 16 tokens
  constexpr int kPitch = D + 4;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  float* const meet = reinterpret_cast<float*>(lds);  // [wave][row][kPitch]
  __shared__ float tops[kFewWaves][kRows], sums[kFewWaves][kRows];
  const llmp_paged_attend& op = a.op;
  const llmp_paged_cache& c = op.cache;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int group_of = lane >> 4, column = lane & 15;
  uint8_t* const landing = lds + wave * TileBytes(D);

  if (!LISTS && a.all_taken != nullptr && *a.all_taken != 0) {
    if (tid == 0) *reinterpret_cast<I32x4*>(a.parts + 4 * blockIdx.x) = I32x4{-1, 0, 0, 0};
    return;
  }
  // ---- this workgroup's run of the line of units: the requests 64 at a time, a lane each.
  uint32_t round = kFewWaves;
  const auto block = [&](int base) {
    FewRequest f = {};
    if (base + lane < op.requests) f = FewOf<LISTS>(a, base + lane, round);
    return f;
  };
  FewRequest mine = block(0);
  uint32_t upto = WaveSums(mine.units);
  // f(request) summed over all requests; the first 64 are at hand.
  const auto over_all = [&](auto&& f) {
    uint32_t sum = __builtin_amdgcn_readlane(WaveSums(f(mine)), kWave - 1);
    for (int base = kWave; base < op.requests; base += kWave) sum += __builtin_amdgcn_readlane(WaveSums(f(block(base))), kWave - 1);
    return sum;
  };
  const auto units_of = [](const FewRequest& f) { return f.units; };
  uint32_t total = over_all(units_of);
  const uint32_t even = (total + gridDim.x - 1) / gridDim.x;
  uint32_t per = (even + kFewWaves - 1) / kFewWaves * kFewWaves;
  // A run a little longer may let every workgroup stay in one segment: a second's visit costs about kVisit tiles. (12 requests of up to
  // 2000 tokens at head size 256 26.4 us without, 23.1 with; 30 of up to 3000 at 128 28.8 and 27.0.)
  if (!LISTS && a.shift == 0 && per > kFewWaves) {
    const auto fits = [&](uint32_t run) {
      return over_all([&](const FewRequest& f) { return f.segments * ((static_cast<uint32_t>(f.tiles) + run - 1) / run); }) <= gridDim.x;
    };
    if (fits(per + kVisit)) {
      while (!fits(per)) per += kFewWaves;  // (at the latest there)
      round = per;
      mine = block(0);
      upto = WaveSums(mine.units);
      total = over_all(units_of);
    }
  }
  if (LISTS && a.whole_units > 0) per = a.whole_units;
  const uint32_t group = OnChiplet(blockIdx.x, gridDim.x, (total + per - 1) / max(per, 1u));
  uint32_t u = group * per;
  const uint32_t u_end = min(u + per, total);
  I32x4 part = {-1, 0, 0, 0};
  if (u >= u_end || total >= 1u << 31) {
    if (tid == 0) *reinterpret_cast<I32x4*>(a.parts + 4 * group) = part;
    return;
  }
  // The request that holds unit u, and the units before it.
  int base = 0, r = 0;
  uint32_t before = 0;
  for (;;) {
    const uint64_t past = __ballot(before + upto > u);
    if (past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      r = base + at;
      before += __builtin_amdgcn_readlane(upto - mine.units, at);
      break;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
    base += kWave;
    if (base >= op.requests) break;  // (not reached: u is below the sum)
    mine = block(base);
    upto = WaveSums(mine.units);
  }

  while (u < u_end && r < op.requests) {
    if (r - base >= kWave) {
      base += kWave;
      mine = block(base);
    }
    const FewRequest f = FewFrom(mine, r - base);
    if (u - before >= f.units) {
      before += f.units;
      ++r;
      continue;
    }
    const uint32_t a_segment = SegmentUnits(f.tiles, a.shift, round);
    const int segment = __builtin_amdgcn_readfirstlane(static_cast<int>((u - before) / a_segment));
    const uint32_t in_segment = u - before - segment * a_segment, u_count = min(a_segment - in_segment, u_end - u);
    const int t_first = static_cast<int>(in_segment << a.shift), t_count = min(f.tiles - t_first, static_cast<int>(u_count << a.shift));
    const int chunks = f.segments / c.kv_heads, head = segment / chunks, chunk = segment - head * chunks;

    // ---- this lane's query row, and what the segment's rows see.
    int token, query_head, first_token, last_token;
    bool real;
    if constexpr (LISTS) {
      const int a_token = (a.group + kRows - 1) / kRows;
      first_token = last_token = token = chunk / a_token;
      query_head = kRows * (chunk - token * a_token) + column;
      real = query_head < a.group;
    } else {
      const int row = kRows * chunk + column;
      token = static_cast<int>(PagedDivide(row, a.group_magic));
      query_head = row - token * a.group;
      real = row < f.q.n * a.group;
      first_token = static_cast<int>(PagedDivide(kRows * chunk, a.group_magic));
      last_token = min(static_cast<int>(PagedDivide(kRows * chunk + kRows - 1, a.group_magic)), f.q.n - 1);
    }
    const int base_position = f.q.base;  // of the request's first new token
    const int position = base_position + token;
    const int window = op.window > 0 ? op.window : INT_MAX / 2;
    const int see_from = max(position - window + 1, 0), see_to = real ? SeenTo(f.q, position) : 0;
    const int all_from = max(base_position + last_token - window + 1, 0), all_to = SeenTo(f.q, base_position + first_token);  // seen by every row
    const int any_from = max(base_position + first_token - window + 1, 0), any_to = SeenTo(f.q, base_position + last_token);  // seen by any

    // The row's loads before all others: its digits are made while the first tile is on its way.
    QueryPart<TYPE, 2 * kSteps> row;
    {
      const int64_t from = (f.q.start + (real ? token : 0)) * op.q_token_stride + (head * a.group + (real ? query_head : 0)) * op.q_head_stride + 16 * group_of;
#pragma unroll
      for (int i = 0; i < 2 * kSteps; ++i) row.Load(op.q, i, from + 64 * (i / 2) + 8 * (i % 2));
    }
    I32x4 digits[kDig][kSteps];
    float unit;  // a digit product's worth in log2 units, but for K's scale
    const auto query = [&]() {
      const QueryUnit made = UnitOf<TYPE>(AcrossGroupsMost(row.MostBits()));
      const float inverse = real ? made.inverse : 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * kSteps; ++i) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float v[4];
          row.Four(i, half, v);
          uint32_t packed[kDig];
          PackDigits<kDig>(v, inverse, packed);
#pragma unroll
          for (int k = 0; k < kDig; ++k) digits[k][i / 2][2 * (i % 2) + half] = static_cast<int>(packed[k]);
        }
      }
      unit = made.unit * (op.softcap != 0.0f ? op.scale : op.scale * kLog2E);
    };
    const float cap_inverse = op.softcap != 0.0f ? 1.0f / op.softcap : 0.0f;

    const int32_t* const table = op.table + r * op.table_stride;
    const int32_t* const list =
        LISTS ? op.lists + (static_cast<int64_t>(f.q.start + token) * c.kv_heads + head) * op.list_pages : nullptr;
    // ---- this wave's tiles, four apart.
    int tile_from = t_first + f.first_tile + wave, tile_to = t_first + t_count + f.first_tile;
    if constexpr (!LISTS) {  // (not those that no row of this chunk sees)
      while (tile_from < tile_to && (tile_from + 1) * kTileTokens <= any_from) tile_from += kFewWaves;
      tile_to = min(tile_to, max(any_to + kTileTokens - 1, 0) / kTileTokens);
    }
    const int tiles = tile_from < tile_to ? (tile_to - tile_from + kFewWaves - 1) / kFewWaves : 0;
    // ---- the places of a tile's tokens.
    const int p16 = c.page / 16;
    // What a place is read from is asked for a tile or two before it is looked at (a look waits for all loads before it, the
    // tiles' among them): the list's entry, then the table's, then the place.
    const auto entry_of = [&](int i) {
      const int n16 = 4 * (tile_from + i * kFewWaves) + group_of;
      Entry e;
      e.entry = static_cast<int>(PagedDivide(n16, a.page_magic));
      e.offset = 16 * (n16 - e.entry * p16);
      if constexpr (LISTS) {
        e.there = e.entry < op.list_pages;
        e.entry = list[min(e.entry, op.list_pages - 1)];
      } else {
        e.there = true;
      }
      return e;
    };
    const auto page_of = [&](const Entry& e) {
      Place at;
      at.position = e.entry * c.page + e.offset;
      at.there = e.there && e.entry >= 0 && e.entry < op.table_width && at.position < f.q.length;
      at.offset = e.offset;
      at.page = table[at.there ? e.entry : 0];
      return at;
    };
    const auto check = [&](Place& at) {
      if (!at.there || at.page < 0 || at.page >= c.pages) at.page = -1;
    };
    // ---- the loads of a tile, to the wave's part of LDS: no registers wait for memory, so a whole tile is on its way under
    // another's work. A load takes 1024 bytes, in memory's order but for the pieces of 16 bytes of a row, which KPiece and VPiece turn.
    const int64_t page_bytes = static_cast<int64_t>(c.kv_heads) * c.page * D;
    const uint8_t* const k_base = static_cast<const uint8_t*>(c.k) + static_cast<int64_t>(head) * c.page * D;
    const uint8_t* const v_base = static_cast<const uint8_t*>(c.v) + static_cast<int64_t>(head) * c.page * D;
    constexpr int kPieces = D / 16, kLoadTokens = kWave / kPieces;  // 16-byte pieces of a K row, rows a load
    const int v_piece = VPiece(lane >> 2, lane & 3);
    const auto load = [&](const Place& at, float* ks, float* vs) {
#pragma unroll
      for (int j = 0; j < kTileTokens / kLoadTokens; ++j) {
        // (A load's tokens are of one group of 16, so of one page: the same for every lane.)
        constexpr int kLoads = 16 / kLoadTokens;
        const int group = j / kLoads, in_group = j % kLoads * kLoadTokens;
        const int page = max(__builtin_amdgcn_readlane(at.page, 16 * group), 0), offset = __builtin_amdgcn_readlane(at.offset, 16 * group);
        const int token = kLoadTokens * j + lane / kPieces;
        ToLds(k_base + page * page_bytes + (offset + in_group) * D + static_cast<uint32_t>(lane / kPieces * D + 16 * KPiece<D>(token, lane % kPieces)),
              landing + 1024 * j);
      }
      const int page = max(__shfl(at.page, 16 * v_piece), 0), offset = __shfl(at.offset, 16 * v_piece);
      const uint8_t* from = v_base + page * page_bytes + (lane >> 2) * c.page + offset;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) ToLds(from + 16 * b * c.page, landing + kTileTokens * D + 1024 * b);
      const int64_t i = static_cast<int64_t>(max(at.page, 0)) * c.kv_heads + head;
      *ks = c.k_scale[i], *vs = c.v_scale[i];
    };
    // What has landed, into registers.
    struct Landed {
      I32x4 k[kProducts][kSteps];
      U32x4 v[kBlocks];
    };
    const auto take = [&](Landed& in) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      asm volatile("" ::: "memory");
#pragma unroll
      for (int t = 0; t < kProducts; ++t) {
        const int token = 16 * (column >> 2) + 4 * t + (column & 3);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) in.k[t][s] = *reinterpret_cast<const I32x4*>(landing + token * D + 16 * KPiece<D>(token, 4 * s + group_of));
      }
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int d = 16 * b + column;
        in.v[b] = *reinterpret_cast<const U32x4*>(landing + kTileTokens * D + d * kTileTokens + 16 * VPiece(d, group_of));
      }
      // (The place is filled again at once: everything has to have left it.)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    float top = -INFINITY, sum = 0.0f;
    F32x4 out[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) out[b] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto attend = [&](const Landed& in, const Place& at, float ks, float vs) {
      // ---- S^T = K Q^T
      float s[kMine];
      {
        I32x4 dots[kDig][kProducts];
#pragma unroll
        for (int t = 0; t < kProducts; ++t) {
#pragma unroll
          for (int d = 0; d < kDig; ++d) {
            I32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < kSteps; ++x) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(in.k[t][x], digits[d][x], acc, 0, 0, 0);
            dots[d][t] = acc;
          }
        }
#pragma unroll
        for (int i = 0; i < kMine; ++i) s[i] = JoinDigits<kDig>(dots[0][i / 4][i % 4], kDig == 3 ? dots[1][i / 4][i % 4] : 0, dots[kDig - 1][i / 4][i % 4]);
      }
      // ---- the tile's softmax
      const float worth = unit * ks;
#pragma unroll
      for (int i = 0; i < kMine; ++i) s[i] *= worth;
      if (op.softcap != 0.0f) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) s[i] = Capped<TYPE>(s[i], op.softcap, cap_inverse) * kLog2E;
      }
      const bool whole = __all(at.page >= 0 && at.position + kMine <= all_to && at.position >= all_from);
      uint32_t seen = 0xFFFFu;
      if (!whole) {
        seen = 0;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
          const int p = at.position + i;
          const bool sees = at.page >= 0 && p >= see_from && p < see_to;
          seen |= sees ? 1u << i : 0u;
          s[i] = sees ? s[i] : -INFINITY;
        }
        if (at.page < 0) vs = 0.0f;
      }
      float peak = s[0];
#pragma unroll
      for (int i = 1; i < kMine; ++i) peak = fmaxf(peak, s[i]);
      peak = AcrossGroupsMax(peak + ScaleLog(vs));
      if (__any(peak > top + (kLift + kSlack))) {
        const float higher = fmaxf(top, peak - kLift);
        const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
        top = higher;
        sum *= keep;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) out[b] *= keep;
      }
      const float from = top == -INFINITY ? 0.0f : top;
      float p[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        p[i] = __builtin_amdgcn_exp2f(s[i] - from);
        sum += p[i];
        p[i] *= vs;
      }
      if (!whole) {  // (a hidden token's weight is zero whatever its page's scale is)
#pragma unroll
        for (int i = 0; i < kMine; ++i) p[i] = (seen >> i) & 1u ? p[i] : 0.0f;
      }
      F16x8 w[2], w_low[2];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        w[i / 8][i % 8] = static_cast<_Float16>(p[i]);
        if constexpr (kDig == 3) w_low[i / 8][i % 8] = RestOf(p[i], w[i / 8][i % 8]);
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const F16x8 v = EightCodes(in.v[b][2 * x], in.v[b][2 * x + 1]);
          out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[x], out[b], 0, 0, 0);
          if constexpr (kDig == 3) out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(RestCodes(v), w_low[x], out[b], 0, 0, 0);
        }
      }
    };

    // ---- the tiles, the next one's loads in flight under each.
    Place here = {}, next = {};
    Entry after = {};
    float ks = 0.0f, vs = 0.0f;
    if (tiles > 0) {
      here = page_of(entry_of(0));
      check(here);
      load(here, &ks, &vs);
      if (tiles > 1) next = page_of(entry_of(1));
      if (tiles > 2) after = entry_of(2);
    }
    query();
    for (int i = 0; i < tiles; ++i) {
      Landed in;
      take(in);
      const Place now = here;
      const float now_ks = ks, now_vs = vs;
      if (i + 1 < tiles) {
        here = next;
        check(here);
        load(here, &ks, &vs);
        if (i + 2 < tiles) next = page_of(after);
        if (i + 3 < tiles) after = entry_of(i + 3);
      }
      attend(in, now, now_ks, now_vs);
    }
    sum = AcrossGroupsSum(sum);

    // ---- the waves' results meet, where the tiles landed.
    __syncthreads();
    if (group_of == 0) tops[wave][column] = top, sums[wave][column] = sum;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
      *reinterpret_cast<F32x4*>(meet + (wave * kRows + column) * kPitch + 16 * b + 4 * group_of) = out[b];
    __syncthreads();
    const bool begins = t_first == 0, ends = t_first + t_count == f.tiles;
    float* const slot = a.partial + (2 * static_cast<int64_t>(group) + (begins ? 1 : 0)) * kRows * (D + 2);
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
          to_token = static_cast<int>(PagedDivide(at, a.group_magic)), to_head = at - to_token * a.group, is_real = at < f.q.n * a.group;
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
    if (begins && !ends) part = I32x4{static_cast<int>((before + (segment + 1) * a_segment - 1) / per), f.q.start, chunk * c.kv_heads + head, f.q.n};
    __syncthreads();
    u += u_count;
  }
  if (tid == 0) *reinterpret_cast<I32x4*>(a.parts + 4 * group) = part;
}

// Parts p from 0 to `count` - 1 of a row (top, sum, D values at part_of(p)) as one, the waves taking
// every fourth; all of a wave's next eight are asked for at once, since such a launch is a chain of round trips. Every thread
// of the first wave gets D / 64 of the row's values, times one over its sum.
template <int D, class F>
__device__ __forceinline__ bool JoinParts(int count, const float* sink, F&& part_of, float (&value)[D / kWave]) {
  constexpr int kPer = D / kWave, kBatch = 8;
  __shared__ float tops[kFewWaves], totals[kFewWaves], values[kFewWaves][D];
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  float high = -INFINITY, all = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) value[e] = 0.0f;
  for (int p0 = wave; p0 < count; p0 += kFewWaves * kBatch) {
    float top[kBatch], total[kBatch], v[kBatch][kPer];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float* from = part_of(min(p0 + kFewWaves * i, count - 1));
      top[i] = from[0], total[i] = from[1];
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[i][e] = from[2 + kPer * lane + e];
    }
    float higher = high;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) higher = fmaxf(higher, top[i]);  // (a part asked for twice changes no maximum)
    const float keep = high == -INFINITY ? (higher == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(high - higher);
    all *= keep;
#pragma unroll
    for (int e = 0; e < kPer; ++e) value[e] *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      // (A row without a logit has a top of -infinity and sums of zero, or no numbers, which stay.)
      float weight = top[i] == -INFINITY ? (higher == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(top[i] - higher);
      if (p0 + kFewWaves * i < count) {
        all += total[i] * weight;
#pragma unroll
        for (int e = 0; e < kPer; ++e) value[e] += v[i][e] * weight;
      }
    }
    high = higher;
  }
  if (lane == 0) tops[wave] = high, totals[wave] = all;
#pragma unroll
  for (int e = 0; e < kPer; ++e) values[wave][kPer * lane + e] = value[e];
  __syncthreads();
  if (wave != 0) return false;
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) top = fmaxf(top, tops[w]);
  all = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) value[e] = 0.0f;
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) {
    const float weight = tops[w] == -INFINITY ? (top == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(tops[w] - top);
    all += totals[w] * weight;
#pragma unroll
    for (int e = 0; e < kPer; ++e) value[e] += values[w][kPer * lane + e] * weight;
  }
  if (sink != nullptr) all += __builtin_amdgcn_exp2f(fmaf(*sink, kLog2E, -(top == -INFINITY ? 0.0f : top)));
  const float inverse = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
  for (int e = 0; e < kPer; ++e) value[e] *= inverse;
  return true;
}

// grid (workgroups of the first launch, rows of a segment): the parts of the segment that begins in workgroup x and ends in another.
// 4 to 5 us, what a launch with two reads after each other takes; 7.6 us for rows of 64 parts.
template <int TYPE, int D, bool LISTS>
__global__ __launch_bounds__(kFewThreads) void FewJoinKernel(const PagedAttendArgs a) {
  constexpr int kPer = D / kWave;
  const llmp_paged_attend& op = a.op;
  const I32x4 part = *reinterpret_cast<const I32x4*>(a.parts + 4 * blockIdx.x);
  if (part.x < 0) return;
  const int row = blockIdx.y, first = blockIdx.x, chunk = part.z / op.cache.kv_heads, head = part.z - chunk * op.cache.kv_heads;
  int token, query_head;
  bool real;
  if constexpr (LISTS) {
    const int a_token = (a.group + kRows - 1) / kRows;
    token = chunk / a_token, query_head = kRows * (chunk % a_token) + row, real = query_head < a.group;
  } else {
    const int at = kRows * chunk + row;
    token = static_cast<int>(PagedDivide(at, a.group_magic)), query_head = at - token * a.group, real = at < part.w * a.group;
  }
  if (!real) return;
  const int h = head * a.group + query_head;
  float value[kPer];
  const bool mine = JoinParts<D>(part.x - first + 1, op.sinks != nullptr ? op.sinks + h : nullptr,
                                 [&](int p) { return a.partial + ((2 * static_cast<int64_t>(first + p) + (p == 0 ? 1 : 0)) * kRows + row) * (D + 2); }, value);
  if (!mine) return;
  const int64_t to = (part.y + token) * op.out_token_stride + h * op.out_head_stride + kPer * (threadIdx.x & (kWave - 1));
#pragma unroll
  for (int e = 0; e < kPer; ++e) StoreOne<TYPE>(op.out, to + e, value[e]);
}

int FewGroups(int head_dim, int cus) { return FewAUnit(head_dim) * (cus > 0 ? cus : 256); }

size_t PartBytes(int groups) { return static_cast<size_t>(groups) * 4 * sizeof(int32_t); }
size_t FewScratch(int head_dim, int cus) {
  const int groups = FewGroups(head_dim, cus);
  return PartBytes(groups) + 2 * static_cast<size_t>(groups) * kRows * (head_dim + 2) * sizeof(float);
}

template <int TYPE, int D, bool LISTS>
void LaunchFew(const PagedAttendArgs& args, int groups, hipStream_t stream) {
  constexpr int kLds = FewLds(D);
  static bool sized = false;
  if (kLds > 32768 && !AllowLds(reinterpret_cast<const void*>(&FewKernel<TYPE, D, LISTS>), kLds, &sized)) return;
  hipLaunchKernelGGL((FewKernel<TYPE, D, LISTS>), dim3(groups), dim3(kFewThreads), kLds, stream, args);
  if (args.whole_units > 0) return;  // no segment is shared
  const int64_t rows = static_cast<int64_t>(LISTS ? 1 : args.op.most_tokens) * args.group;  // at most, of a segment
  hipLaunchKernelGGL((FewJoinKernel<TYPE, D, LISTS>), dim3(groups, rows < kRows ? static_cast<unsigned>(rows) : kRows), dim3(kFewThreads), 0, stream, args);
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

// Requests of more rows than this are the many rows' form's, where the call has any and is work enough: rows times their most tokens
// times head size. In us, this form against that one, bf16, 8 KV heads of 128, groups of 4: of 1000 tokens, 128 and 512 and 1000 new
// 24/41, 36/49, 58/50; of 2000, 32, 256, 512, 1000 24/42, 32/53, 52/57, 93/73; of 8000, 32, 128, 256, 512 31/60, 60/77, 98/90, 168/117;
// groups of 2 at 256, of 2000 128, 256, 512 31/54, 40/55, 70/61; groups of 7 at 64, 64, 512, 1000 21/34, 38/38, 42/43. (The tables there were
// as wide as the request is long: the lengths are the device's to know, so a wider table moves calls of fewer tokens to the other
// form, at the cost that the figures of its left sides show.)
constexpr int kFewRows = 64;
constexpr int64_t kFewWork = 4000000ll * 128;
constexpr int kMostGroup = 1024, kMostFewRows = 1 << 20;  // (PagedDivide's range together)
// Tiles a unit of the line, as a power of two: a call's units stay below 2^31.
int FewShift(const llmp_paged_attend& op) {
  const int64_t group = op.heads / op.cache.kv_heads, chunks_a_token = (group + kRows - 1) / kRows;
  const int64_t segments = op.tokens * chunks_a_token * op.cache.kv_heads;
  const int64_t tokens = op.lists != nullptr ? static_cast<int64_t>(op.list_pages) * op.cache.page : static_cast<int64_t>(op.table_width) * op.cache.page;
  const int64_t tiles = tokens / kTileTokens + 1;
  int shift = 0;
  while (segments * ((tiles >> shift) + kFewWaves) >= 1ll << 31 && shift < 24) ++shift;
  return shift;
}
// With page lists all segments are of one size. Workgroups take whole ones (this many units) where an even cut would save less than
// what it costs: a second segment's beginning and end, and the joining launch. In us, cut evenly against whole, 4 KV heads of 128, groups
// of 4, 512 workgroups: 16 segments of 2, 12, 16 tiles 8.5/6.8, 10.7/10.3, 10.9/12.0; 64 of 8, 16, 64 10.4/8.8, 11.5/12.2, 19/30;
// 256 of 8, 24 14.3/9.4, 20.6/16.6; 400 of 12, 24, 64 17.4/15.1, 29.2/22.1, 49/44; 800 of 24, 64 44.2/39.4, 80/83.
constexpr int kSaving = 12;
int WholeUnits(const PagedAttendArgs& args, int groups) {
  const llmp_paged_attend& op = args.op;
  if (op.lists == nullptr || args.shift > 0) return 0;
  const int64_t segments = static_cast<int64_t>(op.tokens) * ((args.group + kRows - 1) / kRows) * op.cache.kv_heads;
  const int64_t tiles = (static_cast<int64_t>(op.list_pages) * op.cache.page + kTileTokens - 1) / kTileTokens;
  const int64_t a_segment = (tiles + kFewWaves - 1) / kFewWaves * kFewWaves;
  const int64_t even = (segments * a_segment + groups - 1) / groups, whole = a_segment * ((segments + groups - 1) / groups);
  return whole <= even + even / 8 + kSaving ? static_cast<int>(whole) : 0;
}
bool HasMany(const llmp_paged_attend& op) {
  const int64_t group = op.heads / op.cache.kv_heads, rows = op.tokens * group;  // (the heads of all tokens: at most 2^30)
  return op.lists == nullptr && (op.most_tokens < op.tokens ? op.most_tokens : op.tokens) * group > kFewRows &&
         rows * op.table_width > kFewWork / op.cache.head_dim / op.cache.page;
}
size_t AttendScratch(const llmp_paged_attend& op, int cus) {
  return FewScratch(op.cache.head_dim, cus) + (HasMany(op) ? PagedManyScratch(op, cus) : 0);
}

int CheckAttend(const llmp_paged_attend* op) {
  if (op == nullptr) return Refuse(1, "paged_attend: null operands");
  if (const int bad = CheckPagedCache("paged_attend", op->cache, false); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_attend", "q", op->q, op->tokens, op->heads, op->q_token_stride, op->q_head_stride, op->type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_attend", "out", op->out, op->tokens, op->heads, op->out_token_stride, op->out_head_stride, op->type); bad != 0) return bad;
  if (op->requests < 1 || op->requests > 1 << 24 || op->tokens < 1 || op->most_tokens < 1 || op->table_width < 1)
    return Refuse(1, "paged_attend: 1 to 2^24 requests, at least one token and one page a table row (%d, %d, %d, %d)", op->requests, op->tokens,
                  op->most_tokens, op->table_width);
  if (op->heads < 1 || op->heads % op->cache.kv_heads != 0 || static_cast<int64_t>(op->heads) * op->tokens > INT_MAX / 2)
    return Refuse(1, "paged_attend: a whole number of query heads a KV head (%d, %d), at most 2^30 of them in all tokens", op->heads, op->cache.kv_heads);
  if (op->heads / op->cache.kv_heads > kMostGroup) return Refuse(1, "paged_attend: at most %d query heads a KV head, not %d", kMostGroup, op->heads / op->cache.kv_heads);
  if (op->lengths == nullptr || op->starts == nullptr || op->table == nullptr) return Refuse(1, "paged_attend: null operand");
  if ((reinterpret_cast<uintptr_t>(op->lengths) | reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->table) |
       reinterpret_cast<uintptr_t>(op->lists) | reinterpret_cast<uintptr_t>(op->sinks) | reinterpret_cast<uintptr_t>(op->before)) % 4 != 0)
    return Refuse(1, "paged_attend: I32 and F32 arrays at 4-byte boundaries");
  if (op->table_stride < op->table_width) return Refuse(1, "paged_attend: a table row of %d entries every %lld", op->table_width, (long long)op->table_stride);
  if (static_cast<int64_t>(op->table_width) * op->cache.page > kMostPagedLength) return Refuse(1, "paged_attend: a table row of at most 2^30 tokens");
  // (A prompt's tiles of all KV heads are counted in an int.)
  if (static_cast<int64_t>(op->table_width) * op->cache.page * op->cache.kv_heads > 1ll << 36)
    return Refuse(1, "paged_attend: a table row of at most 2^36 tokens of all KV heads together (%d pages of %d, %d heads)", op->table_width, op->cache.page,
                  op->cache.kv_heads);
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
  // (A window that no position passes is none: with one, a position before 0 less the window would pass an int.)
  if (args.op.window >= kMostPagedLength) args.op.window = 0;
  const int groups = FewGroups(op->cache.head_dim, cus);
  args.parts = static_cast<int32_t*>(scratch);
  args.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + PartBytes(groups));
  const uint32_t p16 = static_cast<uint32_t>(op->cache.page / 16);
  args.page_magic = p16 == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / p16 + 1);
  args.group = op->heads / op->cache.kv_heads;
  args.group_magic = args.group == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / args.group + 1);
  args.most_length = op->table_width * op->cache.page;
  const bool many = HasMany(*op);
  const bool alone = many && op->requests == 1 && op->most_tokens >= op->tokens;  // one request: of whatever rows, the many rows' form's
  args.few_rows = alone ? 0 : many ? kFewRows : kMostFewRows;
  args.shift = FewShift(*op);
  args.whole_units = WholeUnits(args, groups);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  args.all_taken = nullptr;
  if (many) args.all_taken = PagedManyRows(args, static_cast<uint8_t*>(scratch) + FewScratch(op->cache.head_dim, cus), cus, on);
  if (alone) return LaunchStatus("paged_attend");
  if (op->type == LLMP_X_F32) LaunchFewOf<LLMP_X_F32>(args, groups, on);
  if (op->type == LLMP_X_BF16) LaunchFewOf<LLMP_X_BF16>(args, groups, on);
  if (op->type == LLMP_X_F16) LaunchFewOf<LLMP_X_F16>(args, groups, on);
  return LaunchStatus("paged_attend");
}
