// llmp.paged.attend, the form for many rows: prompts, whole or in chunks.
//
// What bounds it is the vector units: per logit about seven operations and an exponential, against the matrix instructions' 4 D
// operations; the cache's bytes come from L2 (a head's pages are read by every workgroup of its rows). A workgroup of four
// waves takes 128 rows of one KV head, (token, head) pairs in order, so that a group's query heads share the tile; a
// wave has 32 rows (16 at head size 256). A tile of 64 tokens goes through LDS, double-buffered, its loads in flight under the previous tile's
// work: K as its codes, V turned into F16 once for all the waves. Products as in the few rows' form, 32 x 32:
//   S^T = K Q^T by v_mfma_i32_32x32x32_i8. Row 8a + 4h + b of a product is token 16h + 4a + b of its 32, so that a lane (half h) ends
//   with 16 consecutive tokens of one query row, all of one page;
//   O^T += V^T P^T by v_mfma_f32_32x32x16_f16, P from the same lane's registers.
// LDS rows are 16-byte pieces in an order turned by the row (Turn), so that the 32 rows a matrix operand reads lie in
// different banks.
//
// A first small launch lists the (request, 128 rows) pairs and their tiles. With at least as many (pair, head) segments as workgroups,
// none of them longer than a compute unit's share, each is one workgroup's, longest first, dealt to the compute units there and
// back so that a unit's two workgroups together have about the same; otherwise all segments' tiles lie on one line that the workgroups
// share evenly, and a third launch joins the parts. In us, whole against shared, 8 KV heads: a chunk of 2048 behind 2048 tokens
// (groups of 4 at 128) 154/172, behind 6000 319/346, a prompt of 4000 (groups of 2 at 256) 196/216; of 2000 there, whose last 128
// rows are nearly twice the share, 102/90, 6 ragged prompts 147/109.
//
// Measured at the chunk of 2048 behind 2048, 103 GFLOP: 154 us with the list's and the join's launches, 0.67 PFLOP/s (a large F16 product
// by the library reaches 1.15): 388 vector operations a wave's 32 x 64 logits, about 1800 cycles beside the products' 1024, at two
// waves a SIMD. The products stand apart from the softmax by fences that the compiler's scheduling does not cross; without
// them it is 155.7 us where it is 155.3.
#include <type_traits>

#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kManyRows = 128;  // of a workgroup
constexpr int kJoinThreads = 256;
constexpr int kListThreads = 1024;
constexpr int kBuckets = 1024;  // of the segments' lengths, for their order

// What a segment's beginning and end cost a workgroup, in tiles: where the line is cut evenly, a segment has that many places on it
// before its tiles (a workgroup with eleven short segments otherwise ends last by far).
constexpr int kVisit = 4;

// The list: a header, the pairs, the line's length before each pair (all KV heads'), the pairs' order by length.
struct ListHeader {
  int64_t total;   // tiles of all segments, and kVisit for each
  int pairs, whole;  // whole: every segment is one workgroup's
  int all;           // the few rows' form has nothing left to do
};
struct Pair {
  int request, chunk, first_tile, tiles;
  PagedRequest q;
};
static_assert(sizeof(Pair) == 32);
struct List {
  ListHeader* header;
  Pair* pairs;
  int64_t* before;  // [pairs + 1]
  int32_t* order;
};

struct ManyArgs {
  PagedAttendArgs a;
  List list;
  float* partial;  // [2 * workgroups][kManyRows][D + 2]
  int32_t* parts;  // [workgroups][4]
  int most_pairs;
  int a_unit;  // workgroups a compute unit holds
};

// A few-row request (a prompt's neighbours that decode) is taken along where all of them make the line no longer than this many
// tiles a compute unit, about what the few rows' two launches cost: there a row's tile is 128 rows' work. In us, taken along and by
// the few rows' form: 8 of 500 tokens beside a prompt of 1000 52/57, 4 of 60000 beside 256 180/141, 10 of 20000 beside 2000
// 623/188 (8 KV heads of 128); 6 ragged requests at 256 109/123.
constexpr int kTakeAlong = 8, kTakeAlongRequests = kListThreads;

__device__ __forceinline__ int ChunksOf(const PagedAttendArgs& a, const PagedRequest& q, int few_rows) {
  const int64_t rows = static_cast<int64_t>(q.n) * a.group;
  return rows > few_rows ? static_cast<int>((rows + kManyRows - 1) / kManyRows) : 0;
}
// The tiles that a chunk of a request's rows sees.
__device__ __forceinline__ void TilesOf(const PagedAttendArgs& a, Pair* pair) {
  const PagedRequest& q = pair->q;
  const int first_token = pair->chunk * kManyRows / a.group, last_token = min((pair->chunk * kManyRows + kManyRows - 1) / a.group, q.n - 1);
  const int to = max(SeenTo(q, q.base + last_token), 0), window = a.op.window > 0 ? a.op.window : INT_MAX / 2;
  pair->first_tile = max(q.base + first_token - window + 1, 0) / kTileTokens;
  pair->tiles = max((to + kTileTokens - 1) / kTileTokens - pair->first_tile, 1);  // (rows that see nothing are written too)
}

// One workgroup: the pairs in the order of the requests, their sums, and their order by length, a thread a pair. 6 to 7 us, a chain of
// reads and barriers.
__global__ __launch_bounds__(kListThreads) void ListKernel(const ManyArgs m, int groups) {
  __shared__ int64_t wave_sums[kListThreads / kWave];
  __shared__ int buckets[kBuckets], first_pair[kListThreads];
  __shared__ PagedRequest requests[kListThreads];
  __shared__ int longest;
  if (threadIdx.x == 0) longest = 0;
  const PagedAttendArgs& a = m.a;
  const llmp_paged_attend& op = a.op;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const auto block_sum = [&](int64_t v, int64_t* all) {  // inclusive
#pragma unroll
    for (int step = 1; step < kWave; step <<= 1) {
      const int64_t up = __shfl_up(v, step);
      if (lane >= step) v += up;
    }
    if (lane == kWave - 1) wave_sums[wave] = v;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w < kListThreads / kWave; ++w) {
      const int64_t s = wave_sums[w];
      v += w < wave ? s : 0;
      total += s;
    }
    __syncthreads();
    *all = total;
    return v;
  };
  // The pairs: a request's by all threads where it has many.
  buckets[tid] = 0;
  int64_t count = 0, before = 0;
  bool all_taken = false;
  for (int base = 0; base < op.requests; base += kListThreads) {
    const int here = min(op.requests - base, kListThreads);
    requests[tid] = tid < here ? RequestOf(op.starts, op.lengths, op.before, base + tid, op.tokens, a.most_length) : PagedRequest{};
    int64_t pairs;
    int few_rows = a.few_rows;
    if (op.requests <= kTakeAlongRequests) {
      Pair pair = {};
      pair.q = requests[tid];
      TilesOf(a, &pair);
      const bool few = pair.q.n > 0 && ChunksOf(a, pair.q, few_rows) == 0;
      int64_t along;
      block_sum(few ? static_cast<int64_t>(pair.tiles + kVisit) * op.cache.kv_heads : 0, &along);
      if (along <= static_cast<int64_t>(kTakeAlong) * (groups / m.a_unit)) few_rows = 0;
    }
    all_taken = few_rows == 0;
    const int mine = tid < here ? ChunksOf(a, requests[tid], few_rows) : 0;
    first_pair[tid] = static_cast<int>(block_sum(mine, &pairs)) - mine;
    pairs = min(pairs, m.most_pairs - count);
    __syncthreads();
    // A thread a pair: its request is the last whose pairs begin at or before it (one without pairs begins where the next does).
    for (int64_t p0 = 0; p0 < pairs; p0 += kListThreads) {
      const int p = static_cast<int>(p0) + tid;
      Pair pair = {};
      int64_t length = 0;
      if (p < pairs) {
        int low = 0, high = here;
        while (high - low > 1) {
          const int mid = (low + high) >> 1;
          if (first_pair[mid] <= p) {
            low = mid;
          } else {
            high = mid;
          }
        }
        pair.request = base + low, pair.chunk = p - first_pair[low], pair.q = requests[low];
        TilesOf(a, &pair);
        length = static_cast<int64_t>(pair.tiles + kVisit) * op.cache.kv_heads;
        m.list.pairs[count + p] = pair;
        atomicAdd(&buckets[kBuckets - 1 - min(pair.tiles / 4, kBuckets - 1)], 1);
        atomicMax(&longest, pair.tiles + kVisit);
      }
      int64_t all;
      const int64_t upto = block_sum(length, &all);
      if (p < pairs) m.list.before[count + p] = before + upto - length;
      before += all;
    }
    count += pairs;
    __syncthreads();
  }
  __syncthreads();
  int64_t all;
  const int mine = buckets[tid];
  const int upto = static_cast<int>(block_sum(mine, &all));
  buckets[tid] = upto - mine;
  __syncthreads();
  // (The order within a bucket is any: a segment's result does not depend on its turn.)
  for (int p = tid; p < count; p += kListThreads) m.list.order[atomicAdd(&buckets[kBuckets - 1 - min(m.list.pairs[p].tiles / 4, kBuckets - 1)], 1)] = p;
  if (tid == 0) {
    m.list.before[count] = before;
    m.list.header->total = before;
    m.list.header->pairs = static_cast<int>(count);
    m.list.header->all = all_taken;
    m.list.header->whole = count * op.cache.kv_heads >= groups && longest * static_cast<int64_t>(groups / m.a_unit) <= before;
  }
}

// Where a 16-byte piece of a row of `PIECES` lies: 256 bytes of rows side by side hold a piece number once.
template <int PIECES>
__device__ __forceinline__ int Turn(int row, int piece) { return piece ^ ((row / (16 / PIECES)) & (PIECES - 1)); }

// By head size: four waves of 32 rows, or at 256, where 32 rows' values alone would be half a lane's registers and the
// compiler then carries them to and fro, eight of 16 with 16 x 16 products (twice the reads of LDS).
template <int D>
struct ManyGeo {
  static constexpr int kWaveRows = D == 256 ? 16 : 32;
  static constexpr int kWaves = kManyRows / kWaveRows, kThreads = kWaves * kWave;
  static constexpr int kInner = 1024 / kWaveRows;              // K's dimensions a product: 32, 64
  static constexpr int kTurns = kWaveRows == 32 ? 2 : 1;       // a tile's tokens by 32 or all at once: 16 of them a lane either way
  static constexpr int kKBytes = kTileTokens * D;
  static constexpr int kVBytes = D * kTileTokens * 2;
  static constexpr int kBuffer = kKBytes + kVBytes;
  static constexpr int kLds = 2 * kBuffer + 2 * 4 * 16;  // and the four 16-token groups' scales
  static constexpr int kAUnit = D == 256 ? 1 : 2;        // workgroups a compute unit
  // The token of a row of K in LDS, and where a piece of it lies: rows in the products' order, or as KPiece has them.
  static __device__ __forceinline__ int KToken(int row) {
    if constexpr (kWaveRows == 16) return row;
    return (row & 32) + 16 * ((row >> 2) & 1) + 4 * ((row >> 3) & 3) + (row & 3);
  }
  static __device__ __forceinline__ int KSlot(int row, int piece) {
    if constexpr (kWaveRows == 16) return KPiece<D>(row, piece);
    return Turn<D / 16>(row, piece);
  }
  // Of V's rows of eight pieces: 32 rows are read at once, or 16 and, by other lanes, their pieces' neighbours but one.
  static __device__ __forceinline__ int VSlot(int d, int piece) {
    if constexpr (kWaveRows == 16) return piece ^ ((d >> 1) & 5);
    return Turn<8>(d, piece);
  }
};

template <int TYPE, int D, bool CAPPED>
__global__ __launch_bounds__(ManyGeo<D>::kThreads, 2) void ManyKernel(const ManyArgs m) {
  using G = ManyGeo<D>;
  constexpr int kDig = kDigits<TYPE>;
  constexpr int kWaveRows = G::kWaveRows, kThreads = G::kThreads, kInner = G::kInner;
  constexpr int kSteps = D / kInner, kBlocks = D / kWaveRows, kPieces = D / 16, kLoads = 4 * D / kThreads;
  typedef std::conditional_t<kWaveRows == 32, F32x16, F32x4> Values;  // a lane's of a block of dimensions
  constexpr int kValues = kWaveRows * kWaveRows / kWave;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const PagedAttendArgs& a = m.a;
  const llmp_paged_attend& op = a.op;
  const llmp_paged_cache& c = op.cache;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane / kWaveRows, column = lane % kWaveRows;  // (`half` a quarter where rows are 16)
  const int groups = gridDim.x, w = blockIdx.x;
  const ListHeader header = *m.list.header;
  F32x4* const group_scales = reinterpret_cast<F32x4*>(lds + 2 * G::kBuffer);  // [buffer][group]: K's and V's scale, V's log2 and reciprocal

  int64_t u = 0, u_end = 0, per = 1, pair_from = 0;  // (where on the line the pair begins)
  int turn = 0, pair_index = -1;
  Pair pair = {};
  const auto load_pair = [&]() {
    const I32x4* const from = reinterpret_cast<const I32x4*>(m.list.pairs + pair_index);
    const I32x4 x = from[0], y = from[1];
    const auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    pair = {one(x[0]), one(x[1]), one(x[2]), one(x[3]), {one(y[0]), one(y[1]), one(y[2]), one(y[3])}};
  };
  const int units = groups / m.a_unit, unit_of = w % units;
  const int64_t segments = static_cast<int64_t>(header.pairs) * c.kv_heads;
  if (header.whole) {
    turn = w / units;
  } else {
    // (No fewer than a visit and as many tiles: finer parts cost more to write and to join.)
    per = max((header.total + groups - 1) / groups, static_cast<int64_t>(2 * kVisit));
    u = w * per;
    u_end = min(u + per, header.total);
    if (u < u_end) {  // the pair that holds unit u: the last that begins at or before it
      for (int base = 0; base < header.pairs; base += kWave) {
        const int64_t before = base + lane < header.pairs ? m.list.before[base + lane] : INT64_MAX;
        const int at = __popcll(__ballot(before <= u));
        if (at > 0) {
          const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(before), at - 1);
          pair_index = base + at - 1;
          pair_from = static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(before >> 32), at - 1)) << 32 | low;
        }
        if (at < kWave) break;
      }
      load_pair();
    }
  }
  I32x4 part = {-1, 0, 0, 0};

  for (;;) {
    // ---- the next segment, or part of one.
    int head, t_first, t_count;
    if (header.whole) {
      const int64_t index = turn % 2 == 0 ? static_cast<int64_t>(turn) * units + unit_of : static_cast<int64_t>(turn + 1) * units - 1 - unit_of;
      if (static_cast<int64_t>(turn) * units >= segments) break;
      turn += m.a_unit;
      if (index >= segments) continue;
      pair_index = __builtin_amdgcn_readfirstlane(m.list.order[index / c.kv_heads]);
      head = static_cast<int>(index % c.kv_heads);
      load_pair();
      t_first = 0;
      t_count = pair.tiles;
    } else {
      if (u >= u_end) break;
      const int length = pair.tiles + kVisit;
      if (u >= pair_from + static_cast<int64_t>(length) * c.kv_heads) {
        pair_from += static_cast<int64_t>(length) * c.kv_heads;
        ++pair_index;
        load_pair();
        continue;
      }
      const int in = static_cast<int>(u - pair_from);
      head = in / length;
      const int from = in - head * length, to = static_cast<int>(min(static_cast<int64_t>(length), from + u_end - u));
      u += to - from;
      t_first = max(from - kVisit, 0);
      t_count = max(to - kVisit, 0) - t_first;
      if (t_count == 0) continue;  // the next workgroup begins it
    }
    head = __builtin_amdgcn_readfirstlane(head);
    t_first = __builtin_amdgcn_readfirstlane(t_first);
    t_count = __builtin_amdgcn_readfirstlane(t_count);
    const PagedRequest q = pair.q;
    const int32_t* const table = op.table + pair.request * op.table_stride;

    // ---- this lane's query row, and what the wave's rows see.
    const int row0 = pair.chunk * kManyRows + wave * kWaveRows;
    const int row = row0 + column, rows = q.n * a.group;
    const bool real = row < rows;
    const int token0 = row0 / a.group, in_token0 = row0 - token0 * a.group;  // the wave's first row's
    const int in_tokens = PagedDivide(in_token0 + column, a.group_magic);
    const int token = token0 + in_tokens, query_head = in_token0 + column - in_tokens * a.group;
    const int base_position = q.base;
    const int position = base_position + token;
    const int window = op.window > 0 ? op.window : INT_MAX / 2;
    const int see_from = max(position - window + 1, 0), see_to = real ? SeenTo(q, position) : 0;
    const int first_position = base_position + token0;
    const int last_position = base_position + min(token0 + static_cast<int>(PagedDivide(in_token0 + kWaveRows - 1, a.group_magic)), q.n - 1);
    const int all_from = max(last_position - window + 1, 0), all_to = SeenTo(q, first_position);
    const int any_from = max(first_position - window + 1, 0), any_to = row0 < rows ? SeenTo(q, last_position) : 0;

    const float cap_inverse = op.softcap != 0.0f ? 1.0f / op.softcap : 0.0f;

    // ---- the tiles' loads. A lane knows the page of the tile's 16-token group `lane & 3`; it is looked at a tile after it was
    // asked for (a look waits for all loads before it).
    const int p16 = c.page / 16;
    struct Group {
      int page, offset;
      bool there;
    };
    const auto group_of = [&](int tile) {
      Group g;
      const int n16 = 4 * tile + (lane & 3);
      const int entry = static_cast<int>(PagedDivide(n16, a.page_magic));
      g.offset = 16 * (n16 - entry * p16);
      g.there = entry < op.table_width && 16 * n16 < q.length;
      g.page = table[g.there ? entry : 0];
      return g;
    };
    const int64_t page_bytes = static_cast<int64_t>(c.kv_heads) * c.page * D;
    const uint8_t* const k_base = static_cast<const uint8_t*>(c.k) + static_cast<int64_t>(head) * c.page * D;
    const uint8_t* const v_base = static_cast<const uint8_t*>(c.v) + static_cast<int64_t>(head) * c.page * D;
    // K goes from memory to LDS by itself (a lane's 16 bytes of a load to 16 lane: the row and piece that belong there), V through
    // registers, where it becomes F16. Where a tile is of one page, places are the same for every lane but for constants.
    U32x4 v_in[kLoads];
    F32x4 scales_in;
    bool page_in;
    constexpr int kLoadRows = kWave / kPieces, kWaveKRows = kTileTokens / G::kWaves;  // K's rows a load, a wave
    uint32_t k_from[kLoads];  // from the token group's first row
    int k_group[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int k_row = wave * kWaveKRows + kLoadRows * j + lane / kPieces, t = G::KToken(k_row);
      k_group[j] = t >> 4;
      k_from[j] = (t & 15) * D + 16 * G::KSlot(k_row, lane % kPieces);
    }
    const uint32_t v_from = (tid >> 2) * c.page;
    const bool one_page = p16 % 4 == 0;
    const auto fetch = [&](const Group& g, int buffer) {
      page_in = g.there && g.page >= 0 && g.page < c.pages;
      const int page = page_in ? g.page : 0;
      uint8_t* const k_to = lds + buffer * G::kBuffer + wave * kWaveKRows * D;
      if (one_page) {
        const int64_t at = __builtin_amdgcn_readfirstlane(page) * page_bytes;
        const int offset = __builtin_amdgcn_readfirstlane(g.offset);
        const uint8_t* const k_tile = k_base + at + offset * D;
        const uint8_t* const v_tile = v_base + at + offset;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          ToLds(k_tile + static_cast<uint32_t>(k_from[j] + 16 * k_group[j] * D), k_to + 1024 * j);
          v_in[j] = *reinterpret_cast<const U32x4*>(v_tile + kThreads / 4 * j * c.page + static_cast<uint32_t>(v_from + 16 * (lane & 3)));
        }
      } else {
        const int64_t at = page * page_bytes;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
          const int k_page = __shfl(page, k_group[j]), k_offset = __shfl(g.offset, k_group[j]);
          ToLds(k_base + k_page * page_bytes + k_offset * D + k_from[j], k_to + 1024 * j);
          v_in[j] = *reinterpret_cast<const U32x4*>(v_base + at + g.offset + kThreads / 4 * j * c.page + v_from);  // (a lane's piece of V is of its group)
        }
      }
      if (tid < 4) {
        const int64_t i = static_cast<int64_t>(page) * c.kv_heads + head;
        scales_in = F32x4{c.k_scale[i], c.v_scale[i], 0.0f, 0.0f};
      }
    };
    const auto place = [&](int buffer) {
      uint8_t* const v_at = lds + buffer * G::kBuffer + G::kKBytes;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = tid + kThreads * j;
        const int d = i >> 2, piece = 2 * (i & 3);
        *reinterpret_cast<F16x8*>(v_at + d * 128 + 16 * G::VSlot(d, piece)) = EightCodes(v_in[j][0], v_in[j][1]);
        *reinterpret_cast<F16x8*>(v_at + d * 128 + 16 * G::VSlot(d, piece + 1)) = EightCodes(v_in[j][2], v_in[j][3]);
      }
      if (tid < 4) {  // (a logarithm of -infinity: no page)
        const float vs = scales_in[1];
        group_scales[buffer * 4 + tid] = F32x4{scales_in[0], vs, page_in ? ScaleLog(vs) : -INFINITY, page_in ? 1.0f / vs : 0.0f};
      }
    };

    float top = -INFINITY, sum = 0.0f;
    Values out[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
      for (int i = 0; i < kValues; ++i) out[b][i] = 0.0f;
    }
    const int tile_from = pair.first_tile + t_first, tile_to = tile_from + t_count;
    // A tile is whole in LDS once every wave's loads have landed.
    const auto meet = [&]() {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
    };
    Group next = group_of(tile_from);
    // The row's loads before the first tile's: its digits are made while that is on its way.
    QueryPart<TYPE, 2 * kSteps> part_of_row;
    {
      const int64_t from = (q.start + (real ? token : 0)) * op.q_token_stride + (head * a.group + (real ? query_head : 0)) * op.q_head_stride + 16 * half;
#pragma unroll
      for (int i = 0; i < 2 * kSteps; ++i) part_of_row.Load(op.q, i, from + kInner * (i / 2) + 8 * (i % 2));
    }
    fetch(next, 0);
    next = group_of(tile_from + 1);
    I32x4 digits[kDig][kSteps];
    float unit;
    {
      const QueryUnit made = UnitOf<TYPE>(Across<kWaveRows>(part_of_row.MostBits()));
      // (A negative scale goes into the digits: the units stay positive, so the largest product is the largest logit.)
      const float inverse = !real ? 0.0f : op.scale < 0.0f ? -made.inverse : made.inverse;
#pragma unroll
      for (int i = 0; i < 2 * kSteps; ++i) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float v[4];
          part_of_row.Four(i, k, v);
          uint32_t packed[kDig];
          PackDigits<kDig>(v, inverse, packed);
#pragma unroll
          for (int d = 0; d < kDig; ++d) digits[d][i / 2][2 * (i % 2) + k] = static_cast<int>(packed[d]);
        }
      }
      unit = made.unit * fabsf(op.scale) * (op.softcap != 0.0f ? 1.0f : kLog2E);
    }
    place(0);
    meet();
    for (int tile = tile_from; tile < tile_to; ++tile) {
      const int buffer = (tile - tile_from) & 1;
      const bool more = tile + 1 < tile_to;
      if (more) {
        fetch(next, buffer ^ 1);
        next = group_of(tile + 2);
      }
      if (tile * kTileTokens < any_to && (tile + 1) * kTileTokens > any_from) {
        const uint8_t* const k_at = lds + buffer * G::kBuffer;
        const uint8_t* const v_at = k_at + G::kKBytes;
        const bool inside = (tile + 1) * kTileTokens <= all_to && tile * kTileTokens >= all_from;
        // ---- 32 tokens at a time (all 64 where rows are 16): S^T = K Q^T, their softmax, O^T += V^T P^T
#pragma unroll
        for (int h = 0; h < G::kTurns; ++h) {
          float s[16];
          if constexpr (kWaveRows == 32) {
            I32x16 dots[kDig];
#pragma unroll
            for (int d = 0; d < kDig; ++d) {
#pragma unroll
              for (int i = 0; i < 16; ++i) dots[d][i] = 0;
            }
            const int k_row = 32 * h + column;
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
              const I32x4 k = *reinterpret_cast<const I32x4*>(k_at + k_row * D + 16 * G::KSlot(k_row, 2 * x + half));
#pragma unroll
              for (int d = 0; d < kDig; ++d) dots[d] = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, digits[d][x], dots[d], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = JoinDigits<kDig>(dots[0][i], kDig == 3 ? dots[1][i] : 0, dots[kDig - 1][i]);
          } else {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              I32x4 dots[kDig];
#pragma unroll
              for (int d = 0; d < kDig; ++d) dots[d] = I32x4{0, 0, 0, 0};
              const int k_row = 16 * (column >> 2) + 4 * t + (column & 3);
#pragma unroll
              for (int x = 0; x < kSteps; ++x) {
                const I32x4 k = *reinterpret_cast<const I32x4*>(k_at + k_row * D + 16 * G::KSlot(k_row, 4 * x + half));
#pragma unroll
                for (int d = 0; d < kDig; ++d) dots[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, digits[d][x], dots[d], 0, 0, 0);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) s[4 * t + i] = JoinDigits<kDig>(dots[0][i], kDig == 3 ? dots[1][i] : 0, dots[kDig - 1][i]);
            }
          }
          const int token_group = kWaveRows == 32 ? 2 * h + half : half;  // of the tile's four: the lane's tokens
          // (V's operands are asked for here, before the softmax that makes them useful: a read's latency is the softmax's.)
          F16x8 v_half[2][kBlocks];
          const auto read_v = [&](int x) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              const int d = kWaveRows * b + column;
              v_half[x][b] = *reinterpret_cast<const F16x8*>(v_at + d * 128 + 16 * G::VSlot(d, 2 * token_group + x));
            }
          };
          if constexpr (kWaveRows == 32) {
            read_v(0);
            read_v(1);
          }
          const F32x4 scales = group_scales[buffer * 4 + token_group];  // K's, V's, log2 of V's, 1 / V's
          float worth = unit * scales[0];
          const float value_log = scales[2];
          if constexpr (CAPPED) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = Capped<TYPE>(s[i] * worth, op.softcap, cap_inverse) * kLog2E;
            worth = 1.0f;
          }
          // The short way: every row sees all 32 tokens, and V's scales have logarithms and reciprocals that no exponent runs out of.
          const bool whole = inside && __all(scales[3] > 0x1p-60f && scales[3] < 0x1p60f);
          if (!whole) {
            asm volatile("" ::: "memory");  // (a branch: selects would be in every tile's way)
            const int p0 = tile * kTileTokens + 16 * token_group;
            const int from = value_log == -INFINITY ? 16 : max(see_from - p0, 0), to = see_to - p0;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = i >= from && i < to ? s[i] * worth : -INFINITY;
            worth = 1.0f;
          }
          float peak = s[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) peak = fmaxf(peak, s[i]);
          peak = Across<kWaveRows>(fmaf(peak, worth, value_log));
          // (The maximum follows once it is kSlack behind: the sums rarely turn.)
          if (__any(peak > top + (kLift + kSlack))) {
            const float higher = fmaxf(top, peak - kLift);
            const float keep = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - higher);
            top = higher;
            sum *= keep;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) out[b] *= keep;
          }
          F16x8 p[2], p_low[2];
          const auto pack = [&](int i, float weight) {
            p[i / 8][i % 8] = static_cast<_Float16>(weight);
            if constexpr (kDig == 3) p_low[i / 8][i % 8] = RestOf(weight, p[i / 8][i % 8]);
          };
          if (whole) {  // V's scale in the exponent: the weights at once, and the probabilities' sum from theirs
            const float less = value_log - top;
            float weights = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float v = __builtin_amdgcn_exp2f(fmaf(s[i], worth, less));
              weights += v;
              pack(i, v);
            }
            sum = fmaf(weights, scales[3], sum);
          } else {
            asm volatile("" ::: "memory");
            const float less = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float v = __builtin_amdgcn_exp2f(s[i] - less);
              sum += v;
              pack(i, s[i] == -INFINITY ? 0.0f : v * scales[1]);  // (a hidden token's weight is zero whatever its page's scales are)
            }
          }
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if constexpr (kWaveRows == 16) read_v(x);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
              const F16x8 v = v_half[x][b];
              if constexpr (kWaveRows == 32) {
                out[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[x], out[b], 0, 0, 0);
                if constexpr (kDig == 3) out[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(RestCodes(v), p_low[x], out[b], 0, 0, 0);
              } else {
                out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[x], out[b], 0, 0, 0);
                if constexpr (kDig == 3) out[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(RestCodes(v), p_low[x], out[b], 0, 0, 0);
              }
            }
          }
        }
      }
      if (more) place(buffer ^ 1);
      meet();
    }
    sum = AcrossSum<kWaveRows>(sum);

    // ---- the rows' values, or this part's.
    const bool begins = t_first == 0, ends = t_first + t_count == pair.tiles;
    if (begins && ends) {
      if (real) {
        const int h = head * a.group + query_head;
        if (op.sinks != nullptr) sum += __builtin_amdgcn_exp2f(fmaf(op.sinks[h], kLog2E, -(top == -INFINITY ? 0.0f : top)));
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int64_t to = (q.start + token) * op.out_token_stride + h * op.out_head_stride;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
          for (int i = 0; i < kValues / 4; ++i) {
            const float x[4] = {out[b][4 * i] * inverse, out[b][4 * i + 1] * inverse, out[b][4 * i + 2] * inverse, out[b][4 * i + 3] * inverse};
            StoreValues<TYPE, 4>(op.out, to + kWaveRows * b + 8 * i + 4 * half, x);
          }
        }
      }
    } else {
      float* const to = m.partial + ((2 * static_cast<int64_t>(w) + (begins ? 1 : 0)) * kManyRows + wave * kWaveRows + column) * (D + 2);
      if (half == 0) to[0] = top, to[1] = sum;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) to[2 + kWaveRows * b + 8 * (i / 4) + 4 * half + i % 4] = out[b][i];
      }
      if (begins) {
        const int64_t segment_end = m.list.before[pair_index] + static_cast<int64_t>(head + 1) * (pair.tiles + kVisit);
        part = I32x4{static_cast<int>((segment_end - 1) / per), pair_index, head, 0};
      }
    }
  }
  if (tid == 0) *reinterpret_cast<I32x4*>(m.parts + 4 * w) = part;
}

// grid (workgroups of the launch before, kManyRows / 16): the parts of the segment that begins in workgroup x and ends in
// another, a wave four rows, asked for together, two parts at a time. (Parts are few here and rows many: 208 segments in 213
// workgroups at head size 256, 28 MB of parts, 12.8 us.)
template <int TYPE, int D>
__global__ __launch_bounds__(kJoinThreads) void ManyJoinKernel(const ManyArgs m) {
  constexpr int kPer = D / kWave;
  const PagedAttendArgs& a = m.a;
  const llmp_paged_attend& op = a.op;
  const I32x4 part = *reinterpret_cast<const I32x4*>(m.parts + 4 * blockIdx.x);
  if (part.x < 0) return;
  const Pair pair = m.list.pairs[part.y];
  const int lane = threadIdx.x & (kWave - 1), first = blockIdx.x, last = part.x;
  constexpr int kJoinRows = 4, kBatch = 2;  // rows a wave, parts asked for at once
  const int slot0 = 16 * blockIdx.y + kJoinRows * (threadIdx.x / kWave), row0 = pair.chunk * kManyRows + slot0, rows = pair.q.n * a.group;
  if (row0 >= rows) return;
  float high[kJoinRows], all[kJoinRows], value[kJoinRows][kPer];
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) {
    high[i] = -INFINITY, all[i] = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) value[i][e] = 0.0f;
  }
  for (int w0 = first; w0 <= last; w0 += kBatch) {
    float top[kBatch][kJoinRows], total[kBatch][kJoinRows], v[kBatch][kJoinRows][kPer];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int w = min(w0 + k, last);
#pragma unroll
      for (int i = 0; i < kJoinRows; ++i) {  // (rows past the request's last have slots too, whose values go nowhere)
        const float* from = m.partial + ((2 * static_cast<int64_t>(w) + (w == first ? 1 : 0)) * kManyRows + slot0 + i) * (D + 2);
        top[k][i] = from[0], total[k][i] = from[1];
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[k][i][e] = from[2 + kPer * lane + e];
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (w0 + k > last) break;
#pragma unroll
      for (int i = 0; i < kJoinRows; ++i) {
        const float higher = fmaxf(high[i], top[k][i]);
        const auto weight = [&](float of) { return of == -INFINITY ? (higher == -INFINITY ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(of - higher); };
        const float keep = weight(high[i]), add = weight(top[k][i]);
        all[i] = all[i] * keep + total[k][i] * add;
#pragma unroll
        for (int e = 0; e < kPer; ++e) value[i][e] = value[i][e] * keep + v[k][i][e] * add;
        high[i] = higher;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kJoinRows; ++i) {
    const int row = row0 + i;
    if (row >= rows) return;
    const int token = row / a.group, h = part.z * a.group + row - token * a.group;
    float sum = all[i];
    if (op.sinks != nullptr) sum += __builtin_amdgcn_exp2f(fmaf(op.sinks[h], kLog2E, -(high[i] == -INFINITY ? 0.0f : high[i])));
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t to = (pair.q.start + token) * op.out_token_stride + h * op.out_head_stride + kPer * lane;
#pragma unroll
    for (int e = 0; e < kPer; ++e) StoreOne<TYPE>(op.out, to + e, value[i][e] * inverse);
  }
}

int ManyGroups(int head_dim, int cus) { return (head_dim == 256 ? 1 : 2) * (cus > 0 ? cus : 256); }
int64_t MostPairs(const llmp_paged_attend& op, int group) {
  // (Requests of more than few_rows rows only, and few_rows is at least half of kManyRows: two pairs of every kManyRows rows at most.
  // A request alone, of any rows, has one for every kManyRows and one more; one taken along has one.)
  return 2 * (static_cast<int64_t>(op.tokens) * group / kManyRows + 1) + (op.requests <= kTakeAlongRequests ? op.requests : 0);
}
size_t Up(size_t bytes) { return (bytes + 15) & ~static_cast<size_t>(15); }

template <int TYPE, int D>
void LaunchMany(const ManyArgs& m, int groups, hipStream_t stream) {
  using G = ManyGeo<D>;
  static bool sized = false, sized_capped = false;
  const bool capped = m.a.op.softcap != 0.0f;
  if (G::kLds > 32768 && !AllowLds(reinterpret_cast<const void*>(&ManyKernel<TYPE, D, false>), G::kLds, &sized)) return;
  if (G::kLds > 32768 && !AllowLds(reinterpret_cast<const void*>(&ManyKernel<TYPE, D, true>), G::kLds, &sized_capped)) return;
  hipLaunchKernelGGL(ListKernel, dim3(1), dim3(kListThreads), 0, stream, m, groups);
  if (capped) {
    hipLaunchKernelGGL((ManyKernel<TYPE, D, true>), dim3(groups), dim3(G::kThreads), G::kLds, stream, m);
  } else {
    hipLaunchKernelGGL((ManyKernel<TYPE, D, false>), dim3(groups), dim3(G::kThreads), G::kLds, stream, m);
  }
  hipLaunchKernelGGL((ManyJoinKernel<TYPE, D>), dim3(groups, kManyRows / 16), dim3(kJoinThreads), 0, stream, m);
}
template <int TYPE>
void LaunchManyOf(const ManyArgs& m, int groups, hipStream_t stream) {
  if (m.a.op.cache.head_dim == 64) LaunchMany<TYPE, 64>(m, groups, stream);
  if (m.a.op.cache.head_dim == 128) LaunchMany<TYPE, 128>(m, groups, stream);
  if (m.a.op.cache.head_dim == 256) LaunchMany<TYPE, 256>(m, groups, stream);
}

}  // namespace

size_t PagedManyScratch(const llmp_paged_attend& op, int cus) {
  const int groups = ManyGroups(op.cache.head_dim, cus);
  const size_t pairs = static_cast<size_t>(MostPairs(op, op.heads / op.cache.kv_heads));
  return Up(sizeof(ListHeader)) + Up(pairs * sizeof(Pair)) + Up((pairs + 1) * sizeof(int64_t)) + Up(pairs * sizeof(int32_t)) + 16 * static_cast<size_t>(groups) +
         2 * static_cast<size_t>(groups) * kManyRows * (op.cache.head_dim + 2) * sizeof(float);
}

const int32_t* PagedManyRows(const PagedAttendArgs& args, void* scratch, int cus, hipStream_t stream) {
  const int groups = ManyGroups(args.op.cache.head_dim, cus);
  ManyArgs m;
  m.a = args;
  m.most_pairs = static_cast<int>(MostPairs(args.op, args.group));
  m.a_unit = args.op.cache.head_dim == 256 ? 1 : 2;
  uint8_t* at = static_cast<uint8_t*>(scratch);
  const auto take = [&](size_t bytes) {
    void* p = at;
    at += Up(bytes);
    return p;
  };
  m.list.header = static_cast<ListHeader*>(take(sizeof(ListHeader)));
  m.list.pairs = static_cast<Pair*>(take(m.most_pairs * sizeof(Pair)));
  m.list.before = static_cast<int64_t*>(take((m.most_pairs + 1) * sizeof(int64_t)));
  m.list.order = static_cast<int32_t*>(take(m.most_pairs * sizeof(int32_t)));
  m.parts = static_cast<int32_t*>(take(16 * static_cast<size_t>(groups)));
  m.partial = reinterpret_cast<float*>(at);
  if (args.op.type == LLMP_X_F32) LaunchManyOf<LLMP_X_F32>(m, groups, stream);
  if (args.op.type == LLMP_X_BF16) LaunchManyOf<LLMP_X_BF16>(m, groups, stream);
  if (args.op.type == LLMP_X_F16) LaunchManyOf<LLMP_X_F16>(m, groups, stream);
  return &m.list.header->all;
}

}  // namespace llmp_hip
