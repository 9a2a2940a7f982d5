// llmp.paged.select: for every new token and KV head, the pages of its request whose keys could have the largest logits.
//
// A page keeps every dimension's least and largest K code. With the query as whole numbers c, the sum over the dimensions of
// c * (c > 0 ? high : low) is at least c . k for every key k of the page: the bound that ranks the pages. It is whole-number
// arithmetic up to two F32 products (the query's unit, the page's scale), so every program that follows the definition picks
// the same pages.
//
// First launch, the scores: as products of max(c, 0) with the high codes and of min(c, 0) with the low ones they are matrix
// products of whole numbers, pages as rows and (token, head) pairs of one KV head as columns
// (v_mfma_i32_16x16x64_i8); a wave takes 16 pages at a time. What bounds it is the codes' bytes, 2 * head_dim a page and head.
// Second launch, the choice: a workgroup a (token, KV head) finds the keep-th largest score by its bits, eight at a time
// (a histogram a pass), and writes the pages at or above it in order; ties go to the lower page.
#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kScoreWaves = 4;
constexpr int kScoreThreads = kScoreWaves * kWave;
constexpr int kPickThreads = 256;
constexpr int kPickKeys = 8192;  // scores a workgroup keeps in LDS; more are read from scratch again
constexpr int kMostKeep = 4096;

struct SelectArgs {
  llmp_paged_select op;
  float* scores;  // [tokens][KV heads][table_width]
  int group, most_length;
  int tokens_a_tile;  // tokens whose heads fill the 16 columns
};

// grid (tiles of tokens, KV heads, blocks of pages).
template <int TYPE, int D>
__global__ __launch_bounds__(kScoreThreads) void ScoreKernel(const SelectArgs a) {
  constexpr int kSteps = D / 64;
  __shared__ float tile[kScoreWaves][16][17];  // [column][page]
  const llmp_paged_select& op = a.op;
  const llmp_paged_cache& c = op.cache;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int group_of = lane >> 4, column = lane & 15, head = blockIdx.y;
  // The request and the tile of its tokens.
  int r = -1, first = 0;
  uint32_t before = 0;
  for (int base = 0; base < op.requests; base += kWave) {
    uint32_t tiles = 0;
    if (base + lane < op.requests) tiles = (RequestOf(op.starts, op.lengths, base + lane, op.tokens, a.most_length).n + a.tokens_a_tile - 1) / a.tokens_a_tile;
    const uint32_t upto = WaveSums(tiles);
    const uint64_t past = __ballot(before + upto > blockIdx.x);
    if (past != 0) {
      const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
      r = base + at;
      first = static_cast<int>(blockIdx.x - before - __builtin_amdgcn_readlane(upto - tiles, at)) * a.tokens_a_tile;
      break;
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  if (r < 0) return;
  const PagedRequest q = RequestOf(op.starts, op.lengths, r, op.tokens, a.most_length);
  const int last = min(first + a.tokens_a_tile, q.n) - 1;
  const int pages = min((q.length - q.n + last) / c.page + 1, op.table_width);  // the last token's
  if (q.length - q.n + last < 0 || static_cast<int>(blockIdx.z) * kScoreWaves * 16 >= pages) return;
  const int32_t* const table = op.table + r * op.table_stride;

  // The columns' queries as codes, those above zero and those below apart.
  I32x4 up[kSteps], down[kSteps];
  float unit;
  bool real;
  const auto query = [&](int h0) {
    const int token = first + (a.tokens_a_tile > 1 ? column / a.group : 0);
    const int query_head = a.tokens_a_tile > 1 ? column % a.group : h0 + column;
    real = token <= last && query_head < a.group;
    QueryPart<TYPE, 2 * kSteps> part;
    const int64_t start = (q.start + (real ? token : first)) * op.q_token_stride + (head * a.group + (real ? query_head : 0)) * op.q_head_stride + 16 * group_of;
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) part.Load(op.q, i, start + 64 * (i / 2) + 8 * (i % 2));
    const uint32_t bits = AcrossGroupsMost(part.MostBits());
    constexpr uint32_t kInfinity = TYPE == LLMP_X_F32 ? 0x7F800000u : TYPE == LLMP_X_BF16 ? 0x7F80u : 0x7C00u;
    const float most = TYPE == LLMP_X_F32 ? __builtin_bit_cast(float, bits) : TYPE == LLMP_X_BF16 ? Bf16BitsToFloat(bits) : HalfBitsToFloat(bits);
    const float scale = bits >= kInfinity ? 0.0f : most * (1.0f / 127.0f), inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    unit = bits >= kInfinity ? __builtin_nanf("") : scale;
#pragma unroll
    for (int i = 0; i < 2 * kSteps; ++i) {
      float v[8];
      int code[8];
      float four[4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
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
  };
  bool made = false;
  for (int from = (blockIdx.z * kScoreWaves + wave) * 16; from < pages; from += gridDim.z * kScoreWaves * 16) {
    // The lane's page row: its low and high codes.
    const int row = min(from + column, pages - 1);
    int page = table[row];
    if (page < 0 || page >= c.pages) page = 0;
    const int64_t at = (static_cast<int64_t>(page) * c.kv_heads + head) * D + 16 * group_of;
    I32x4 low[kSteps], high[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      low[s] = *reinterpret_cast<const I32x4*>(static_cast<const uint8_t*>(c.low) + at + 64 * s);
      high[s] = *reinterpret_cast<const I32x4*>(static_cast<const uint8_t*>(c.high) + at + 64 * s);
    }
    const float page_scale = c.k_scale[static_cast<int64_t>(page) * c.kv_heads + head];
    float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // of column groups, more than one where a KV head has over 16 heads
    for (int h0 = 0; h0 < a.group; h0 += 16) {
      if (!made || a.group > 16) query(h0);
      made = true;
      I32x4 sum = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(high[s], up[s], sum, 0, 0, 0);
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(low[s], down[s], sum, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (The scale is the page's of the sum's row: row 4 group_of + i's, that lane holds it.)
        float score = (static_cast<float>(sum[i]) * unit) * __shfl(page_scale, 4 * group_of + i);
        if (!real || score != score) score = -INFINITY;
        best[i] = fmaxf(best[i], score);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[wave][column][4 * group_of + i] = best[i];
    __builtin_amdgcn_wave_barrier();
    // A lane a (token, page): the largest of the token's columns.
    const int columns = a.tokens_a_tile > 1 ? a.group : 16;
    for (int i = lane; i < a.tokens_a_tile * 16; i += kWave) {
      const int t = i / 16, p = i % 16;
      if (first + t > last || from + p >= pages) continue;
      float top = -INFINITY;
      for (int k = 0; k < columns; ++k) top = fmaxf(top, tile[wave][t * columns + k][p]);
      a.scores[(static_cast<int64_t>(q.start + first + t) * c.kv_heads + head) * op.table_width + from + p] = top;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// A score's bits in an order that whole numbers have: larger scores larger keys, 0 kept for none.
__device__ __forceinline__ uint32_t KeyOf(float score) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, score == 0.0f ? 0.0f : score);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// A count's exclusive sum over the workgroup in thread order, and the whole; `shared` another four words each time.
__device__ __forceinline__ int BlockSum(int count, int* shared, int* all) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int upto = static_cast<int>(WaveSums(static_cast<uint32_t>(count)));
  if (lane == kWave - 1) shared[wave] = upto;
  __syncthreads();
  int before = upto - count, total = 0;
#pragma unroll
  for (int w = 0; w < kPickThreads / kWave; ++w) {
    before += w < wave ? shared[w] : 0;
    total += shared[w];
  }
  *all = total;
  return before;
}

// grid (tokens, KV heads).
__global__ __launch_bounds__(kPickThreads) void PickKernel(const SelectArgs a) {
  __shared__ uint32_t kept[kPickKeys];
  __shared__ int bins[4][256], shared[2][kPickThreads / kWave], found[4][3];
  const llmp_paged_select& op = a.op;
  const int token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & (kWave - 1);
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
  const PagedRequest q = RequestOf(op.starts, op.lengths, low, op.tokens, a.most_length);
  const int position = token >= q.start && token < q.start + q.n ? q.length - q.n + token - q.start : -1;
  const int pages = position < 0 ? 0 : min(position / op.cache.page + 1, op.table_width);
  if (pages <= op.keep) {
    for (int i = tid; i < op.keep; i += kPickThreads) list[i] = i < pages ? i : -1;
    return;
  }
  const float* const scores = a.scores + (static_cast<int64_t>(token) * op.cache.kv_heads + head) * op.table_width;
  const auto key_of = [&](int j) { return j < op.first || j >= pages - op.recent ? ~0u : KeyOf(scores[j]); };
  const bool in_lds = pages <= kPickKeys;
#pragma unroll
  for (int i = 0; i < 4; ++i) bins[i][tid] = 0;
  if (in_lds) {
#pragma unroll 4
    for (int j = tid; j < pages; j += kPickThreads) kept[j] = key_of(j);
  }
  __syncthreads();
  const auto key_at = [&](int j) { return in_lds ? kept[j] : key_of(j); };
  // The keep-th largest key, its highest bits first, until all of the keys that share the bits found so far are to be chosen:
  // `want` of them are.
  uint32_t prefix = 0, mask = 0;
  int want = op.keep;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int shift = 24 - 8 * i;
    for (int j = tid; j < pages; j += kPickThreads) {
      const uint32_t key = key_at(j);
      if ((key & mask) == prefix) atomicAdd(&bins[i][(key >> shift) & 0xFF], 1);
    }
    __syncthreads();
    if (tid < kWave) {  // from the top bin down: the one in which the count passes `want`
      int four[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) four[e] = bins[i][255 - 4 * lane - e], sum += four[e];
      const int upto = static_cast<int>(WaveSums(static_cast<uint32_t>(sum)));
      int above = upto - sum;
      if (above < want && upto >= want) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (above < want && above + four[e] >= want) found[i][0] = 255 - 4 * lane - e, found[i][1] = want - above, found[i][2] = four[e];
          above += four[e];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[i][0]) << shift;
    mask |= 0xFFu << shift;
    want = found[i][1];
    if (found[i][2] == want) break;
  }
  // In order, a run of pages a thread: all above the bits found, and the first `want` of those that have them.
  const int run = (pages + kPickThreads - 1) / kPickThreads, from = min(tid * run, pages), to = min(from + run, pages);
  int equal = 0, larger = 0, all;
  for (int j = from; j < to; ++j) {
    const uint32_t key = key_at(j) & mask;
    equal += key == prefix, larger += key > prefix;
  }
  int rank = BlockSum(equal, shared[0], &all);
  const int chosen = larger + min(max(want - rank, 0), equal);
  int at = BlockSum(chosen, shared[1], &all);
  for (int j = from; j < to; ++j) {
    const uint32_t key = key_at(j) & mask;
    if ((key > prefix || (key == prefix && rank < want)) && at < op.keep) list[at++] = j;
    rank += key == prefix;
  }
}

template <int TYPE, int D>
void LaunchScore(const SelectArgs& args, dim3 grid, hipStream_t stream) {
  hipLaunchKernelGGL((ScoreKernel<TYPE, D>), grid, dim3(kScoreThreads), 0, stream, args);
}
template <int TYPE>
void LaunchScoreOf(const SelectArgs& args, dim3 grid, hipStream_t stream) {
  if (args.op.cache.head_dim == 64) LaunchScore<TYPE, 64>(args, grid, stream);
  if (args.op.cache.head_dim == 128) LaunchScore<TYPE, 128>(args, grid, stream);
  if (args.op.cache.head_dim == 256) LaunchScore<TYPE, 256>(args, grid, stream);
}

int CheckSelect(const llmp_paged_select* op) {
  if (op == nullptr) return Refuse(1, "paged_select: null operands");
  if (const int bad = CheckPagedCache("paged_select", op->cache, true); bad != 0) return bad;
  if (const int bad = CheckPagedRows("paged_select", "q", op->q, op->q_token_stride, op->q_head_stride, op->type); bad != 0) return bad;
  if (op->requests < 1 || op->requests > 1 << 24 || op->tokens < 1 ||  op->most_tokens < 1 || op->table_width < 1)
    return Refuse(1, "paged_select: 1 to 2^24 requests, at least one token and one page a table row (%d, %d, %d, %d)", op->requests, op->tokens,
                  op->most_tokens, op->table_width);
  if (op->heads < 1 || op->heads % op->cache.kv_heads != 0)
    return Refuse(1, "paged_select: a whole number of query heads a KV head (%d, %d)", op->heads, op->cache.kv_heads);
  if (op->lengths == nullptr || op->starts == nullptr || op->table == nullptr || op->lists == nullptr) return Refuse(1, "paged_select: null operand");
  if ((reinterpret_cast<uintptr_t>(op->lengths) | reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->table) |
       reinterpret_cast<uintptr_t>(op->lists)) % 4 != 0)
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
  return static_cast<size_t>(op->tokens) * op->cache.kv_heads * op->table_width * sizeof(float);
}

extern "C" int llmp_hip_paged_select(const llmp_paged_select* op, void* scratch, size_t scratch_bytes, void* stream) {
  if (const int bad = CheckSelect(op); bad != 0) return bad;
  const size_t needs = llmp_hip_paged_select_scratch(op);
  if (scratch == nullptr || scratch_bytes < needs || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
    return Refuse(1, "paged_select: %zu bytes of scratch at a 16-byte boundary, %zu given", needs, scratch_bytes);
  BeginLaunches();
  SelectArgs args;
  args.op = *op;
  args.scores = static_cast<float*>(scratch);
  args.group = op->heads / op->cache.kv_heads;
  args.most_length = op->table_width * op->cache.page;
  // (A request of one token fills no more columns than its heads.)
  args.tokens_a_tile = args.group >= 16 ? 1 : 16 / args.group;
  if (args.tokens_a_tile > op->most_tokens) args.tokens_a_tile = op->most_tokens;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (op->table_width > op->keep) {  // otherwise every page is chosen
    const int64_t tiles = static_cast<int64_t>(op->requests) + op->tokens / args.tokens_a_tile;
    const int blocks = (op->table_width + 16 * kScoreWaves - 1) / (16 * kScoreWaves);
    const dim3 grid(static_cast<unsigned>(tiles < op->tokens ? tiles : op->tokens), op->cache.kv_heads, blocks < 1024 ? blocks : 1024);
    if (op->type == LLMP_X_F32) LaunchScoreOf<LLMP_X_F32>(args, grid, on);
    if (op->type == LLMP_X_BF16) LaunchScoreOf<LLMP_X_BF16>(args, grid, on);
    if (op->type == LLMP_X_F16) LaunchScoreOf<LLMP_X_F16>(args, grid, on);
  }
  hipLaunchKernelGGL(PickKernel, dim3(op->tokens, op->cache.kv_heads), dim3(kPickThreads), 0, on, args);
  return LaunchStatus("paged_select");
}
