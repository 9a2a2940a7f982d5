// llmp.paged.select: for every new token and KV head, the pages of its request whose keys could have the largest logits.
//
// A page keeps every dimension's least and largest K code. With the query as whole numbers c, the sum over the dimensions of
// c * (c > 0 ? high : low) is at least c . k for every key k of the page: the bound that ranks the pages. It is whole-number
// arithmetic up to two F32 products (the query's unit, the page's scale), so every program that follows the definition picks
// the same pages.
//
// First launch, the scores: as products of max(c, 0) with the high codes and of min(c, 0) with the low ones they are matrix
// products of whole numbers, pages as rows and (token, head) pairs of one KV head as columns
// (v_mfma_i32_16x16x64_i8); a wave takes 16 pages at a time. A page that is not in the cache has no score and is never chosen. What bounds it is the codes' bytes, 2 * head_dim a page and head.
// Second launch, the choice: a workgroup a (token, KV head) finds the keep-th largest score by its bits, eight at a time
// (a histogram a pass), and writes the pages at or above it in order; ties go to the lower page. Where there are workgroups enough
// for the card, both are one launch and the scores stay in LDS.
//
// Measured: 8 requests of up to 65536 tokens, pages of 64, 8 KV heads of 128: the scores 9.6 us for 7 MB of codes (a chain: lengths, table,
// codes, products), the choice 6.3 us.
#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kScoreWaves = 4;
constexpr int kScoreThreads = kScoreWaves * kWave;
constexpr int kWholeWaves = 16;
constexpr int kWholeThreads = kWholeWaves * kWave;
constexpr int kPickThreads = 256;
constexpr int kPickKeys = 8192;  // scores a workgroup keeps in LDS; more are read from scratch again
constexpr int kMostKeep = 4096;

struct SelectArgs {
  llmp_paged_select op;
  float* scores;  // [tokens][KV heads][table_width]
  int group, most_length;
  int tokens_a_tile;  // tokens whose heads fill the 16 columns
};

__device__ __forceinline__ bool IsPage(const llmp_paged_cache& c, int page) { return page >= 0 && page < c.pages; }
// How many of its request's pages the token at `position` sees tokens of.
__device__ __forceinline__ int PagesSeen(const llmp_paged_select& op, const PagedRequest& q, int position) {
  const int seen = SeenTo(q, position);
  return seen <= 0 ? 0 : min((seen - 1) / op.cache.page + 1, op.table_width);
}
// A tile of a request's tokens: which, and how many pages its last one has.
struct TokenTile {
  PagedRequest q;
  int request, first, last, pages;
};
// Tile `index` of all requests' (request -1: none).
__device__ __forceinline__ TokenTile TileOf(const SelectArgs& a, uint32_t index) {
  const llmp_paged_select& op = a.op;
  const int lane = threadIdx.x & (kWave - 1);
  TokenTile t = {};
  t.request = -1;
  uint32_t before = 0;
  for (int base = 0; base < op.requests; base += kWave) {
    uint32_t tiles = 0;
    PagedRequest q = {};
    if (base + lane < op.requests) {
      q = RequestOf(op.starts, op.lengths, op.before, base + lane, op.tokens, a.most_length);
      tiles = (q.n + a.tokens_a_tile - 1) / a.tokens_a_tile;
    }
    const uint32_t upto = WaveSums(tiles);
    const uint64_t past = __ballot(before + upto > index);
    if (past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      t.request = base + at;
      t.first = static_cast<int>(index - before - __builtin_amdgcn_readlane(upto - tiles, at)) * a.tokens_a_tile;
      t.q = {__builtin_amdgcn_readlane(q.start, at), __builtin_amdgcn_readlane(q.n, at), __builtin_amdgcn_readlane(q.length, at),
             __builtin_amdgcn_readlane(q.base, at)};
      t.last = min(t.first + a.tokens_a_tile, t.q.n) - 1;
      t.pages = PagesSeen(op, t.q, t.q.base + t.last);
      break;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return t;
}

// A wave's scores of 16 pages at a time; TAKEN: with queries that the workgroup's waves made once, a group of at most 16 heads.
template <int TYPE, int D, bool TAKEN>
struct Scorer {
  static constexpr int kSteps = D / 64;
  const SelectArgs& a;
  const TokenTile& t;
  const int head, lane, group_of, column;
  const int32_t* const table;
  I32x4 up[kSteps], down[kSteps];  // the columns' queries as codes, those above zero and those below apart
  float unit;
  bool real, again = false;  // again: the first heads' codes have made way for others'
  struct Pages {
    I32x4 low[kSteps], high[kSteps];
    float scale;
    bool there;
  };

  __device__ __forceinline__ Scorer(const SelectArgs& args, const TokenTile& tile, int kv_head)
      : a(args), t(tile), head(kv_head), lane(threadIdx.x & (kWave - 1)), group_of(lane >> 4), column(lane & 15),
        table(args.op.table + tile.request * args.op.table_stride) {}

  __device__ __forceinline__ int Entry(int from) const { return table[min(from + column, t.pages - 1)]; }
  // The lane's page row: its low and high codes.
  __device__ __forceinline__ void Load(int page, Pages* to) const {
    const llmp_paged_cache& c = a.op.cache;
    to->there = IsPage(c, page);
    if (!to->there) page = 0;  // (any that can be read)
    const int64_t page_head = static_cast<int64_t>(page) * c.kv_heads + head, at = page_head * D + 16 * group_of;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      to->low[s] = *reinterpret_cast<const I32x4*>(static_cast<const uint8_t*>(c.low) + at + 64 * s);
      to->high[s] = *reinterpret_cast<const I32x4*>(static_cast<const uint8_t*>(c.high) + at + 64 * s);
    }
    to->scale = c.k_scale[page_head];
  }
  // The columns' queries, heads h0 on of the group: asked for, and as codes.
  __device__ __forceinline__ void Ask(int h0, QueryPart<TYPE, 2 * kSteps>* part) {
    const llmp_paged_select& op = a.op;
    const int token = t.first + (a.tokens_a_tile > 1 ? column / a.group : 0);
    const int query_head = a.tokens_a_tile > 1 ? column % a.group : h0 + column;
    real = token <= t.last && query_head < a.group;
    const int64_t start = (t.q.start + (real ? token : t.first)) * op.q_token_stride + (head * a.group + (real ? query_head : 0)) * op.q_head_stride + 16 * group_of;
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) part->Load(op.q, i, start + 64 * (i / 2) + 8 * (i % 2));
  }
  __device__ __forceinline__ void Codes(const QueryPart<TYPE, 2 * kSteps>& part) {
    const uint32_t bits = AcrossGroupsMost(part.MostBits());
    constexpr uint32_t kInfinity = TYPE == LLMP_X_F32 ? 0x7F800000u : TYPE == LLMP_X_BF16 ? 0x7F80u : 0x7C00u;
    const float most = TYPE == LLMP_X_F32 ? __builtin_bit_cast(float, bits) : TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(bits) : HalfBitsToFloat(bits);
    const float scale = bits >= kInfinity ? 0.0f : most * (1.0f / 127.0f), inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    unit = bits >= kInfinity ? __builtin_nanf("") : scale;
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      float v[8];
      int code[8];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float four[4];
        part.Four(i, k, four);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * k + e] = four[e];
      }
      CodesOf(v, scale, inverse, code);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t positive = 0, negative = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          positive |= static_cast<uint32_t>(max(code[4 * k + e], 0)) << (8 * e);
          negative |= static_cast<uint32_t>(min(code[4 * k + e], 0) & 0xFF) << (8 * e);
        }
        up[i / 2][2 * (i % 2) + k] = static_cast<int>(positive), down[i / 2][2 * (i % 2) + k] = static_cast<int>(negative);
      }
    }
  }
  // The queries from LDS: [column][D] codes above zero, then those below, and the columns' units.
  __device__ __forceinline__ void Take(const uint8_t* codes, const float* units) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      up[s] = *reinterpret_cast<const I32x4*>(codes + column * D + 64 * s + 16 * group_of);
      down[s] = *reinterpret_cast<const I32x4*>(codes + 16 * D + column * D + 64 * s + 16 * group_of);
    }
    unit = units[column];
    real = column < a.tokens_a_tile * a.group && t.first + (a.tokens_a_tile > 1 ? column / a.group : 0) <= t.last;
  }
  // The scores of pages `from` to from + 15 through `tile` ([column][page], the wave's own): give(token of the tile, page, score), NaN
  // for a page that is not there.
  template <class F>
  __device__ __forceinline__ void Score(int from, const Pages& pages, float (*tile)[17], F&& give) {
    float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // of column groups, more than one where a KV head has over 16 heads
    for (int h0 = 0; h0 < (TAKEN ? 1 : a.group); h0 += 16) {
      if constexpr (!TAKEN) {
        if (h0 > 0 || again) {
          QueryPart<TYPE, 2 * kSteps> part;
          Ask(h0, &part);
          Codes(part);
          again = true;
        }
      }
      I32x4 sum = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(pages.high[s], up[s], sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(pages.low[s], down[s], sum, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (The scale is the page's of the sum's row: row 4 group_of + i's, that lane holds it.)
        float score = (static_cast<float>(sum[i]) * unit) * __shfl(pages.scale, 4 * group_of + i);
        if (!real || score != score) score = -INFINITY;
        best[i] = fmaxf(best[i], score);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[column][4 * group_of + i] = best[i];
    __builtin_amdgcn_wave_barrier();
    // A lane a (token, page): the largest of the token's columns.
    const int columns = a.tokens_a_tile > 1 ? a.group : 16;
    for (int i = lane; i < a.tokens_a_tile * 16; i += kWave) {
      const int token = i / 16, p = i % 16;
      if (t.first + token > t.last || from + p >= t.pages) continue;
      float top = -INFINITY;
      for (int k = 0; k < columns; ++k) top = fmaxf(top, tile[token * columns + k][p]);
      give(token, from + p, pages.there ? top : __builtin_nanf(""));  // (p is the lane's column: the page whose row it loaded)
    }
    __builtin_amdgcn_wave_barrier();
  }
};

// grid (tiles of tokens, KV heads, blocks of pages).
template <int TYPE, int D>
__global__ __launch_bounds__(kScoreThreads) void ScoreKernel(const SelectArgs a) {
  __shared__ float tile[kScoreWaves][16][17];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), head = blockIdx.y;
  const TokenTile t = TileOf(a, blockIdx.x);
  if (t.request < 0 || static_cast<int>(blockIdx.z) * kScoreWaves * 16 >= t.pages) return;
  int from = (blockIdx.z * kScoreWaves + wave) * 16;
  if (from >= t.pages) return;
  Scorer<TYPE, D, false> scorer(a, t, head);
  typename Scorer<TYPE, D, false>::Pages pages;
  QueryPart<TYPE, D / 32> part;
  int entry = scorer.Entry(from);
  scorer.Ask(0, &part);
  scorer.Load(entry, &pages);
  scorer.Codes(part);
  while (true) {
    scorer.Score(from, pages, tile[wave], [&](int token, int page, float score) {
      a.scores[(static_cast<int64_t>(t.q.start + t.first + token) * a.op.cache.kv_heads + head) * a.op.table_width + page] = score;
    });
    from += gridDim.z * kScoreWaves * 16;
    if (from >= t.pages) break;
    scorer.Load(scorer.Entry(from), &pages);
  }
}

// A score's bits in an order that whole numbers have: larger scores larger keys, 0 for a page that is not there.
__device__ __forceinline__ uint32_t KeyOf(float score) {
  if (score != score) return 0;
  const uint32_t bits = __builtin_bit_cast(uint32_t, score == 0.0f ? 0.0f : score);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// What the threads of a share of a workgroup know together in a choice.
struct Choice {
  int bins[2][256], found[3];
  uint32_t least[kWholeWaves], most[kWholeWaves], least_there[kWholeWaves];
  int others[kWholeWaves], forced[kWholeWaves], sums[2][kWholeWaves];
};
// The sum of `value` over a share's threads before the caller, and all of it; `sums` [waves], written here.
__device__ __forceinline__ int SumBefore(int value, int* sums, int lane, int wave, int waves, int* all) {
  const int upto = static_cast<int>(WaveSums(static_cast<uint32_t>(value)));
  if (lane == kWave - 1) sums[wave] = upto;
  __syncthreads();
  const int of_waves = static_cast<int>(WaveSums(lane < waves ? static_cast<uint32_t>(sums[lane]) : 0u));
  *all = __builtin_amdgcn_readlane(of_waves, kWave - 1);
  return upto - value + (wave > 0 ? __builtin_amdgcn_readlane(of_waves, max(wave - 1, 0)) : 0);
}
// All of a token's `count` pages, at most op.keep, that are there: what is chosen where none has to be left out. By a share of a workgroup, as
// the choice below; `most` pages in any share: where that is a wave's, the share's first wave needs no barrier.
__device__ __forceinline__ void TakeAll(const llmp_paged_select& op, int count, int most, int me, int threads, int* sums, const int32_t* table, int32_t* list) {
  const int lane = me & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(me / kWave), waves = threads / kWave;
  const int run = ((count + kWave - 1) / kWave + waves - 1) / waves * kWave, from = min(wave * run, count), to = min(from + run, count);
  const auto there = [&](int j) { return j < to && IsPage(op.cache, table[j]); };
  if (most <= kWave) {
    if (list == nullptr || wave > 0) return;
    const uint64_t mask = __ballot(there(lane));
    if ((mask >> lane) & 1) list[__popcll(mask & ((1ull << lane) - 1))] = lane;
    for (int i = __popcll(mask) + lane; i < op.keep; i += kWave) list[i] = -1;
    return;
  }
  int mine = 0, all;
  for (int j = from; j < to; j += kWave) mine += __popcll(__ballot(there(j + lane)));
  int at = SumBefore(lane == 0 ? mine : 0, sums, lane, wave, waves, &all);
  if (list == nullptr) return;
  at = __builtin_amdgcn_readfirstlane(at);  // (lane 0's: what lies before the wave)
  for (int j = from; j < to; j += kWave) {
    const uint64_t mask = __ballot(there(j + lane));
    if (there(j + lane)) list[at + __popcll(mask & ((1ull << lane) - 1))] = j + lane;
    at += __popcll(mask);
  }
  for (int i = all + me; i < op.keep; i += threads) list[i] = -1;
}
// The choice of op.keep of `count` pages by a share of a workgroup, `threads` threads (whole waves) of which the caller is number `me`:
// the first and the recent pages, and of the others those with the largest keys, of each those that are there (a key other than
// 0), written in order with -1 past them (list null: nothing is). The workgroup's shares call it together, they meet at its barriers.
template <class F>
__device__ __forceinline__ void Choose(const llmp_paged_select& op, int count, int me, int threads, Choice* all, int share, int shares, F&& key_at, int32_t* list) {
  const int lane = me & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(me / kWave), waves = threads / kWave;
  Choice& my = all[share];
  const int begin = min(op.first, count), end = max(count - op.recent, begin);
  for (int i = me; i < 512; i += threads) my.bins[0][i] = 0;
  uint32_t least = ~0u, most = 0;
  for (int j = me; j < count; j += threads) {  // (the first and the recent ones for whether they are there: then the least is not 0)
    const uint32_t key = key_at(j);
    const bool other = (j >= begin) & (j < end);
    least = min(least, (other | (key == 0)) ? key : ~0u), most = max(most, other ? key : 0u);
  }
  least = WaveMinU32(least), most = WaveMaxU32(most);
  if (lane == 0) my.least[wave] = least, my.most[wave] = most;
  int want = op.keep - op.first - op.recent;
  bool every = count <= op.keep;
  if (me == 0) my.found[2] = every || want == 0;
  __syncthreads();
  for (int w = 0; w < waves; ++w) least = min(least, my.least[w]), most = max(most, my.most[w]);
  if (__any(lane < shares * waves && all[lane / waves].least[lane % waves] == 0)) {  // pages of some share are not there: those that are, counted
    uint32_t low_key = ~0u;
    int others = 0, forced = 0;
    for (int j = me; j < count; j += threads) {
      const uint32_t key = key_at(j);
      const bool other = j >= begin && j < end;
      if (key != 0 && other) low_key = min(low_key, key);
      others += key != 0 && other, forced += key != 0 && !other;
    }
    low_key = WaveMinU32(low_key);
    if (lane == 0) my.least_there[wave] = low_key;
    others = static_cast<int>(WaveSums(static_cast<uint32_t>(others))), forced = static_cast<int>(WaveSums(static_cast<uint32_t>(forced)));
    if (lane == kWave - 1) my.others[wave] = others, my.forced[wave] = forced;
    __syncthreads();
    least = ~0u, others = forced = 0;
    for (int w = 0; w < waves; ++w) least = min(least, my.least_there[w]), others += my.others[w], forced += my.forced[w];
    want = op.keep - forced;
    every = others <= want;
    if (me == 0) my.found[2] = every || want == 0;
    __syncthreads();
  }
  // The want-th largest distance from the least key, its highest bits first (the bounds are mostly of one sign and near each other:
  // eight bits of the distances tell them apart, where eight bits of the keys are the same few), until all that share the bits
  // found so far are chosen.
  uint32_t prefix = ~0u;  // (none wanted: no distance lies above)
  int low = every || want == 0 || most <= least ? 0 : 32 - __clz(most - least);
#pragma unroll 1
  for (int pass = 0;; ++pass) {
    if (__all(lane >= shares || all[lane].found[2] != 0)) break;
    const bool mine = my.found[2] == 0;
    const int upper = low, next = max(upper - 8, 0);
    if (mine) {
      const uint32_t digits = (1u << (upper - next)) - 1;
      for (int j = begin + me; j < end; j += threads) {
        const uint32_t key = key_at(j), d = key - least;
        if ((key != 0) & ((pass == 0) | ((d >> min(upper, 31)) == prefix))) atomicAdd(&my.bins[pass & 1][(d >> next) & digits], 1);
      }
    }
    if (pass > 0) {
      for (int i = me; i < 256; i += threads) my.bins[(pass + 1) & 1][i] = 0;
    }
    __syncthreads();
    if (mine && wave == 0) {  // from the top bin down: the one in which the count passes `want`
      int four[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) four[e] = my.bins[pass & 1][255 - 4 * lane - e], sum += four[e];
      const int upto = static_cast<int>(WaveSums(static_cast<uint32_t>(sum)));
      int above = upto - sum;
      if (above < want && upto >= want) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (above < want && above + four[e] >= want) {
            my.found[0] = 255 - 4 * lane - e, my.found[1] = want - above;
            my.found[2] = above + four[e] == want || next == 0;
          }
          above += four[e];
        }
      }
    }
    __syncthreads();
    if (mine) {
      prefix = (pass == 0 ? 0u : prefix << (upper - next)) | static_cast<uint32_t>(my.found[0]);
      want = my.found[1];
      low = next;
    }
  }
  // In order, a run of pages a thread: all above the bits found, and the first `want` of those that have them.
  const auto look = [&](int j, bool* is_equal) {
    const uint32_t key = key_at(j), d = (key - least) >> low;
    const bool there = key != 0, always = every | (j < begin) | (j >= end);
    *is_equal = there & !always & (d == prefix);
    return there & (always | (d > prefix));
  };
  const int run = (count + threads - 1) / threads, from = min(me * run, count), to = min(from + run, count);
  int equal = 0, larger = 0;
  for (int j = from; j < to; ++j) {
    bool is_equal;
    larger += look(j, &is_equal), equal += is_equal;
  }
  int all_equal, all_chosen;
  int rank = SumBefore(equal, my.sums[0], lane, wave, waves, &all_equal);
  int at = SumBefore(larger + min(max(want - rank, 0), equal), my.sums[1], lane, wave, waves, &all_chosen);
  if (list == nullptr) return;
  for (int j = from; j < to; ++j) {
    bool is_equal;
    const bool is_larger = look(j, &is_equal);
    if ((is_larger || (is_equal && rank < want)) && at < op.keep) list[at++] = j;
    rank += is_equal;
  }
  for (int i = all_chosen + me; i < op.keep; i += threads) list[i] = -1;
}

// grid (tokens, KV heads).
__global__ __launch_bounds__(kPickThreads) void PickKernel(const SelectArgs a) {
  __shared__ uint32_t kept[kPickKeys];
  __shared__ Choice choice;
  const llmp_paged_select& op = a.op;
  const int token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
  int32_t* const list = op.lists + (static_cast<int64_t>(token) * op.cache.kv_heads + head) * op.keep;
  // The token's request: the last that starts at or before it.
  int low = 0, high = op.requests;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (op.starts[mid] <= token) {
      low = mid;
    } else {
      high = mid;
    }
  }
  const PagedRequest q = RequestOf(op.starts, op.lengths, op.before, low, op.tokens, a.most_length);
  const int pages = token >= q.start && token < q.start + q.n ? PagesSeen(op, q, q.base + token - q.start) : 0;
  if (pages <= op.keep) {  // (no scores: all that are there)
    const int32_t* const table = op.table + low * op.table_stride;
    TakeAll(op, pages, pages, tid, kPickThreads, choice.sums[0], table, list);
    return;
  }
  const float* const scores = a.scores + (static_cast<int64_t>(token) * op.cache.kv_heads + head) * op.table_width;
  if (pages <= kPickKeys) {
    // (A thread reads its own keys only until the choice's first barrier.)
#pragma unroll 4
    for (int j = tid; j < pages; j += kPickThreads) kept[j] = KeyOf(scores[j]);
    __syncthreads();
    Choose(op, pages, tid, kPickThreads, &choice, 0, 1, [&](int j) { return kept[j]; }, list);
  } else {
    Choose(op, pages, tid, kPickThreads, &choice, 0, 1, [&](int j) { return KeyOf(scores[j]); }, list);
  }
}

// One launch: a workgroup scores a tile of tokens in one KV head, its keys in LDS ([token][table_width]), and picks from them, a
// token of the tile a share of the waves. grid (tiles of tokens, KV heads).
template <int TYPE, int D>
__global__ __launch_bounds__(kWholeThreads) void WholeKernel(const SelectArgs a, int shares) {
  extern __shared__ __attribute__((aligned(16))) uint32_t keys[];
  __shared__ float tile[kWholeWaves][16][17];
  __shared__ Choice choices[16];
  __shared__ __attribute__((aligned(16))) uint8_t codes[2 * 16 * D];
  __shared__ float units[kWholeWaves];
  const llmp_paged_select& op = a.op;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave), head = blockIdx.y;
  {  // rows of no request, a share of them each workgroup's
    const int begin = op.starts[0], end = op.starts[op.requests];
    for (int token = blockIdx.x; token < op.tokens; token += gridDim.x) {
      if (token >= begin && token < end) continue;
      for (int i = tid; i < op.keep; i += kWholeThreads) op.lists[(static_cast<int64_t>(token) * op.cache.kv_heads + head) * op.keep + i] = -1;
    }
  }
  const TokenTile t = TileOf(a, blockIdx.x);
  if (t.request < 0) return;
  if (t.pages > op.keep) {
    Scorer<TYPE, D, true> scorer(a, t, head);
    // A wave a column: its query's codes, for all the waves (one launch: no group of more than 16).
    constexpr int kPer = D / kWave;
    const int token = t.first + wave / a.group;
    const bool real = wave < a.tokens_a_tile * a.group && token <= t.last;
    const int64_t at = (t.q.start + (real ? token : t.first)) * op.q_token_stride + (head * a.group + (real ? wave % a.group : 0)) * op.q_head_stride + kPer * lane;
    float v[kPer];
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      v[e] = LoadOne<TYPE>(op.q, at + e);
      bits = max(bits, __builtin_bit_cast(uint32_t, v[e]) & 0x7FFFFFFFu);
    }
    bits = WaveMaxU32(bits);
    const bool bad = bits >= 0x7F800000u;
    const float unit = bad ? 0.0f : __builtin_bit_cast(float, bits) * (1.0f / 127.0f);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int code = unit > 0.0f ? static_cast<int>(fminf(fmaxf(rintf(v[e] / unit), -127.0f), 127.0f)) : 0;
      codes[wave * D + kPer * lane + e] = static_cast<uint8_t>(max(code, 0));
      codes[16 * D + wave * D + kPer * lane + e] = static_cast<uint8_t>(min(code, 0));
    }
    if (lane == 0) units[wave] = bad ? __builtin_nanf("") : unit;
    __syncthreads();
    if (16 * wave < t.pages) {
      typename Scorer<TYPE, D, true>::Pages pages;
      scorer.Take(codes, units);
      int entry = scorer.Entry(16 * wave);
      for (int from = 16 * wave; from < t.pages; from += 16 * kWholeWaves) {
        scorer.Load(entry, &pages);
        entry = scorer.Entry(from + 16 * kWholeWaves);
        scorer.Score(from, pages, tile[wave], [&](int token, int page, float score) { keys[token * op.table_width + page] = KeyOf(score); });
      }
    }
  }
  __syncthreads();
  const int threads = kWholeThreads / shares, share = tid / threads, me = tid - share * threads;
  const bool mine = t.first + share <= t.last;
  const int pages = mine ? PagesSeen(op, t.q, t.q.base + t.first + share) : 0;
  int32_t* const list = mine ? op.lists + (static_cast<int64_t>(t.q.start + t.first + share) * op.cache.kv_heads + head) * op.keep : nullptr;
  const uint32_t* const key = keys + share * op.table_width;
  const int32_t* const table = op.table + t.request * op.table_stride;
  if (t.pages <= op.keep) {  // (every token's: the tile's last has the most)
    TakeAll(op, pages, t.pages, me, threads, choices[share].sums[0], table, list);
    return;
  }
  Choose(op, pages, me, threads, choices, share, shares, [&](int j) { return key[j]; }, list);
}

// One launch where its workgroups, one a (tile of tokens, KV head), are at least half as many as the card's 256 compute units and hold
// their keys in LDS: fewer leave the card idle while one reads a whole row's codes, and more spare the scores' way through memory
// and each (token, page)'s part of a wave. In us, two launches against one, 8 KV heads of 128, pages of 16, 1024 a row: groups of 8, one
// token of 1, 8, 32, 64 requests 12.6/18.0, 18.3/18.3, 38.6/25.6, 63.7/37.6 (8 requests of unlike lengths 17/24); groups of 4,
// 4 tokens of 8 and 32 requests 25.3/22.4, 46.2/34.6, 100 of 8 215/97; groups of 1, 16 tokens of 8 and 64 28.5/37.0, 122/79.
constexpr int kWholeWorkgroups = 128, kWholeKeys = 16384;
bool IsWhole(const SelectArgs& a, int64_t tiles) {
  return a.group <= 16 && tiles * a.op.cache.kv_heads >= kWholeWorkgroups && static_cast<int64_t>(a.tokens_a_tile) * a.op.table_width <= kWholeKeys;
}

// How a call is answered, from its sizes alone.
struct SelectForm {
  int64_t tiles;
  bool scored, whole;  // scored: not every page is chosen; whole: in one launch, the scores in LDS
  bool ScoresInMemory() const { return scored && !whole; }
};
SelectForm FormOf(const llmp_paged_select& op, SelectArgs* args) {
  args->op = op;
  args->group = op.heads / op.cache.kv_heads;
  args->most_length = op.table_width * op.cache.page;
  // (A request of one token fills no more columns than its heads.)
  args->tokens_a_tile = args->group >= 16 ? 1 : 16 / args->group;
  if (args->tokens_a_tile > op.most_tokens) args->tokens_a_tile = op.most_tokens;
  const int64_t most_tiles = static_cast<int64_t>(op.requests) + op.tokens / args->tokens_a_tile;
  SelectForm form;
  form.tiles = most_tiles < op.tokens ? most_tiles : op.tokens;
  form.scored = op.table_width > op.keep;
  form.whole = form.scored && IsWhole(*args, form.tiles);
  return form;
}
size_t SelectScratch(const llmp_paged_select& op, const SelectForm& form) {
  return form.ScoresInMemory() ? static_cast<size_t>(op.tokens) * op.cache.kv_heads * op.table_width * sizeof(float) : 16;
}

template <int TYPE, int D>
void LaunchSelect(const SelectArgs& args, const SelectForm& form, hipStream_t stream) {
  const llmp_paged_select& op = args.op;
  if (form.whole) {
    const int lds = args.tokens_a_tile * op.table_width * 4;
    static bool sized = false;
    if (!AllowLds(reinterpret_cast<const void*>(&WholeKernel<TYPE, D>), kWholeKeys * 4, &sized)) return;
    int shares = 1;
    while (shares < args.tokens_a_tile) shares *= 2;
    hipLaunchKernelGGL((WholeKernel<TYPE, D>), dim3(static_cast<unsigned>(form.tiles), op.cache.kv_heads), dim3(kWholeThreads), lds, stream, args, shares);
    return;
  }
  const int blocks = (op.table_width + 16 * kScoreWaves - 1) / (16 * kScoreWaves);
  hipLaunchKernelGGL((ScoreKernel<TYPE, D>), dim3(static_cast<unsigned>(form.tiles), op.cache.kv_heads, blocks < 1024 ? blocks : 1024), dim3(kScoreThreads), 0, stream,
                     args);
}
template <int TYPE>
void LaunchSelectOf(const SelectArgs& args, const SelectForm& form, hipStream_t stream) {
  if (args.op.cache.head_dim == 64) LaunchSelect<TYPE, 64>(args, form, stream);
  if (args.op.cache.head_dim == 128) LaunchSelect<TYPE, 128>(args, form, stream);
  if (args.op.cache.head_dim == 256) LaunchSelect<TYPE, 256>(args, form, stream);
}

int CheckSelect(const llmp_paged_select* op) {
  if (op == nullptr) return Refuse(1, "paged_select: null operands");
  if (const int bad = CheckPagedCache("paged_select", op->cache, true); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_select", "q", op->q, op->tokens, op->heads, op->q_token_stride, op->q_head_stride, op->type); bad != 0) return bad;
  if (op->requests < 1 || op->requests > 1 << 24 || op->tokens < 1 ||  op->most_tokens < 1 || op->table_width < 1)
    return Refuse(1, "paged_select: 1 to 2^24 requests, at least one token and one page a table row (%d, %d, %d, %d)", op->requests, op->tokens,
                  op->most_tokens, op->table_width);
  if (op->heads < 1 || op->heads % op->cache.kv_heads != 0)
    return Refuse(1, "paged_select: a whole number of query heads a KV head (%d, %d)", op->heads, op->cache.kv_heads);
  if (op->lengths == nullptr || op->starts == nullptr || op->table == nullptr || op->lists == nullptr) return Refuse(1, "paged_select: null operand");
  if ((reinterpret_cast<uintptr_t>(op->lengths) | reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->table) |
       reinterpret_cast<uintptr_t>(op->lists) | reinterpret_cast<uintptr_t>(op->before)) % 4 != 0)
    return Refuse(1, "paged_select: I32 arrays at 4-byte boundaries");
  if (op->table_stride < op->table_width) return Refuse(1, "paged_select: a table row of %d entries every %lld", op->table_width, (long long)op->table_stride);
  if (static_cast<int64_t>(op->table_width) * op->cache.page > kMostPagedLength) return Refuse(1, "paged_select: a table row of at most 2^30 tokens");
  if (op->keep < 1 || op->keep > kMostKeep || op->first < 0 || op->recent < 0 || static_cast<int64_t>(op->first) + op->recent > op->keep)
    return Refuse(1, "paged_select: 1 to %d pages, the first and the recent ones among them (%d, %d, %d)", kMostKeep, op->keep, op->first, op->recent);
  return 0;
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" size_t llmp_hip_paged_select_scratch(const llmp_paged_select* op) {
  if (CheckSelect(op) != 0) return 0;
  SelectArgs args;
  return SelectScratch(*op, FormOf(*op, &args));
}

extern "C" int llmp_hip_paged_select(const llmp_paged_select* op, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int bad = CheckSelect(op); bad != 0) return bad;
  SelectArgs args;
  const SelectForm form = FormOf(*op, &args);
  const size_t needs = SelectScratch(*op, form);
  if (scratch == nullptr || scratch_bytes < needs || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
    return Refuse(1, "paged_select: %zu bytes of scratch at a 16-byte boundary, %zu given", needs, scratch_bytes);
  BeginLaunches();
  args.scores = static_cast<float*>(scratch);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (form.scored) {
    if (op->type == LLMP_X_F32) LaunchSelectOf<LLMP_X_F32>(args, form, on);
    if (op->type == LLMP_X_BF16) LaunchSelectOf<LLMP_X_BF16>(args, form, on);
    if (op->type == LLMP_X_F16) LaunchSelectOf<LLMP_X_F16>(args, form, on);
  }
  if (!form.whole) hipLaunchKernelGGL(PickKernel, dim3(op->tokens, op->cache.kv_heads), dim3(kPickThreads), 0, on, args);
  return LaunchStatus("paged_select");
}
