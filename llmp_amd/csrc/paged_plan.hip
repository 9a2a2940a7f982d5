// llmp.paged.plan: the requests' lengths before and after a step, in; the pages that change hands, the new tokens' slots
// and the pages they touch, out. Four exclusive sums over the requests (new tokens, pages wanted, pages given back, pages
// touched) say where everything goes; every output is then an index of its own, found by a binary search in those sums, so
// nothing is ordered by atomics and the same lengths give the same answer.
//
// The kernel is latency: a decode step of 64 requests moves some kilobytes. Sizes whose outputs one workgroup writes in a few
// sweeps are one launch, the sums and what is known of each request in LDS; the kinds of outputs lie on one line, so that
// they are written beside each other and not one after another. Larger sizes sum in a first launch of one workgroup (a pass of
// the requests, 1024 at a time, to scratch) and write in a second of many, a workgroup one kind's, its sums in LDS.
#include "paged_attend.h"

namespace llmp_hip {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kOneLaunchRequests = 1024;  // their sums in LDS
// Tokens and work items together: a few sweeps. (One launch and two, us: 1000 requests of a token 8.9 and 8.6, 300 of 4 6.5 and 7.2, 8
// of 250 5.6 and 6.5, of 500, past this, 13 in one workgroup of 256 and 6.5 in two launches.)
constexpr int kOneLaunchOutputs = 4096;
constexpr int kSearchRequests = 4096;     // the second launch's sums in LDS

// A request's numbers before the sums.
struct PlanRequest {
  int before, after, have, want;
};
__device__ __forceinline__ int CeilPages(int tokens, int page) { return (tokens + page - 1) / page; }
__device__ __forceinline__ PlanRequest ReadPlanRequest(const llmp_paged_plan& op, int r) {
  PlanRequest q;
  const int most = static_cast<int>(kMostPagedLength);
  q.before = min(max(op.before[r], 0), most);
  q.after = min(max(op.after[r], 0), most);
  q.have = min(CeilPages(q.before, op.page), op.table_width);
  q.want = min(CeilPages(q.after, op.page), op.table_width);
  return q;
}
// Pages a request gets, and its length after the step, once the wants before it are known.
__device__ __forceinline__ int PagesGot(const PlanRequest& q, int wants_before, int free) {
  return min(max(q.want - q.have, 0), max(free - wants_before, 0));
}
__device__ __forceinline__ int LengthAfter(const PlanRequest& q, int got, int page) {
  if (q.after <= q.before) return q.after;
  // (64 bits: a table's width times a page may pass an int.)
  return static_cast<int>(min(static_cast<int64_t>(q.after), max(static_cast<int64_t>(q.before), static_cast<int64_t>(q.have + got) * page)));
}
__device__ __forceinline__ int PagesTouched(const PlanRequest& q, int length, int page) {
  return length > q.before ? (length - 1) / page - q.before / page + 1 : 0;
}

// What the sums leave: the ring as it was, and the totals.
struct PlanTotals {
  int head, free, wants, gives, touched, tokens;
};
constexpr int kTotalInts = 8;
// What the outputs need of a request.
struct PlanRecord {
  int before, length, have, want;
};
// The sums' and the records' places, in LDS or in scratch.
struct PlanSums {
  int *starts, *wants, *gives, *touched;  // [requests + 1], exclusive
  I32x4* records;
};

// Inclusive sums over a workgroup of N values at once; `carry` the running totals, known to every thread.
template <int THREADS, int N>
__device__ void BlockSums(int (&v)[N], int (&carry)[N], int* wave_sums) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  constexpr int kWaves = THREADS / kWave;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = static_cast<int>(WaveSums(static_cast<uint32_t>(v[i])));
  if (lane == kWave - 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) wave_sums[i * kWaves + wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int s = wave_sums[i * kWaves + w];
      before += w < wave ? s : 0;
      all += s;
    }
    v[i] += before + carry[i];
    carry[i] += all;
  }
  __syncthreads();
}

// The sums' pass by one workgroup: starts, lengths and counters written, the sums and records left in `to`.
template <int THREADS>
__device__ PlanTotals SumRequests(const llmp_paged_plan& op, const PlanSums& to, int* wave_sums) {
  PlanTotals t;
  t.head = op.counters_in[0];
  t.free = min(max(op.counters_in[1], 0), op.ring_size);
  if (t.head < 0 || t.head >= op.ring_size) {
    t.head %= op.ring_size;
    if (t.head < 0) t.head += op.ring_size;
  }
  int carry[3] = {0, 0, 0}, carry_touched[2] = {0, 0};
  for (int base = 0; base < op.requests; base += THREADS) {
    const int r = base + threadIdx.x;
    const bool real = r < op.requests;
    PlanRequest q = {0, 0, 0, 0};
    if (real) q = ReadPlanRequest(op, r);
    const int fresh = max(q.after - q.before, 0), wants = max(q.want - q.have, 0), gives = max(q.have - q.want, 0);
    int v[3] = {fresh, wants, gives};
    BlockSums<THREADS>(v, carry, wave_sums);
    const int got = PagesGot(q, v[1] - wants, t.free);
    const int length = LengthAfter(q, got, op.page);
    const int touched = PagesTouched(q, length, op.page);
    int u[2] = {touched, max(q.after - length, 0)};
    BlockSums<THREADS>(u, carry_touched, wave_sums);
    if (real) {
      op.starts[r] = v[0] - fresh;
      op.lengths[r] = length;
      if (to.starts != op.starts) to.starts[r] = v[0] - fresh;
      to.wants[r] = v[1] - wants;
      to.gives[r] = v[2] - gives;
      to.touched[r] = u[0] - touched;
      to.records[r] = I32x4{q.before, length, q.have, q.want};
    }
  }
  t.tokens = carry[0];
  t.wants = carry[1];
  t.gives = carry[2];
  t.touched = carry_touched[0];
  if (threadIdx.x == 0) {
    op.starts[op.requests] = t.tokens;
    to.starts[op.requests] = t.tokens;
    to.wants[op.requests] = t.wants;
    to.gives[op.requests] = t.gives;
    to.touched[op.requests] = t.touched;
    const int taken = min(t.wants, t.free);
    op.counters[0] = static_cast<int>((static_cast<int64_t>(t.head) + taken) % op.ring_size);
    op.counters[1] = min(t.free - taken + t.gives, op.ring_size);
    op.counters[2] = carry_touched[1];
  }
  return t;
}

// The request whose share of the sums holds `index`: the last r with sums[r] <= index (requests with nothing are passed over).
__device__ __forceinline__ int OwnerOf(const int* sums, int requests, int index) {
  int low = 0, high = requests;  // sums[low] <= index < sums[high]
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (sums[mid] <= index) {
      low = mid;
    } else {
      high = mid;
    }
  }
  return low;
}
// The ring's entry `index` past its head (head and index both below its size).
__device__ __forceinline__ uint32_t RingPlace(const llmp_paged_plan& op, int head, int index) {
  const uint32_t at = static_cast<uint32_t>(head) + static_cast<uint32_t>(index), size = static_cast<uint32_t>(op.ring_size);
  return at >= size ? (at - size >= size ? 0 : at - size) : at;
}
__device__ __forceinline__ PlanRecord RecordOf(const PlanSums& s, int r) {
  const I32x4 w = s.records[r];
  return {w.x, w.y, w.z, w.w};
}
// Page j of request r: an old entry of the table, or the ring's (the new entry itself is another thread's to write).
__device__ __forceinline__ int PageOf(const llmp_paged_plan& op, const PlanTotals& t, const PlanRecord& q, int r, int wants_before, int j) {
  return j < q.have ? op.table[r * op.table_stride + j] : op.ring[RingPlace(op, t.head, wants_before + j - q.have)];
}

// The outputs, each by its index. What the ring takes back lies past all that it gives out, and new entries of the table past all
// that are read, so the order does not matter. (The ranges are checked where they index memory: lengths whose sums
// pass an int give wrong numbers, not accesses outside the arrays.)
__device__ __forceinline__ void WriteToken(const llmp_paged_plan& op, const PlanTotals& t, const PlanSums& s, int i) {
  int slot = -1, position = -1, owner = -1;
  if (i < t.tokens) {
    owner = OwnerOf(s.starts, op.requests, i);
    const PlanRecord q = RecordOf(s, owner);
    position = q.before + i - s.starts[owner];
    if (position >= 0 && position < q.length) {
      const int j = position / op.page;
      slot = PageOf(op, t, q, owner, s.wants[owner], j) * op.page + position - j * op.page;
    }
  }
  op.slots[i] = slot;
  op.positions[i] = position;
  op.owners[i] = owner;
}
__device__ __forceinline__ void WriteItem(const llmp_paged_plan& op, const PlanTotals& t, const PlanSums& s, int i) {
  I32x4 item = {-1, 0, 0, 0};
  if (i < t.touched) {
    const int r = OwnerOf(s.touched, op.requests, i);
    const PlanRecord q = RecordOf(s, r);
    const int j = q.before / op.page + i - s.touched[r];
    if (j >= 0 && j < CeilPages(q.length, op.page)) {
      const int low = max(j * op.page, q.before), high = static_cast<int>(min(static_cast<int64_t>(q.length), static_cast<int64_t>(j + 1) * op.page));
      item = I32x4{PageOf(op, t, q, r, s.wants[r], j), s.starts[r] + low - q.before, low - j * op.page, high - low};
    }
  }
  *reinterpret_cast<I32x4*>(op.work + 4 * static_cast<int64_t>(i)) = item;
}
__device__ __forceinline__ void WriteTaken(const llmp_paged_plan& op, const PlanTotals& t, const PlanSums& s, int i) {
  const int r = OwnerOf(s.wants, op.requests, i);
  const PlanRecord q = RecordOf(s, r);
  const int j = q.have + i - s.wants[r];
  if (j >= q.have && j < q.want) op.table[r * op.table_stride + j] = op.ring[RingPlace(op, t.head, i)];
}
__device__ __forceinline__ void WriteBack(const llmp_paged_plan& op, const PlanTotals& t, const PlanSums& s, int i) {
  const int r = OwnerOf(s.gives, op.requests, i);
  const PlanRecord q = RecordOf(s, r);
  const int j = q.want + i - s.gives[r];
  if (j >= q.want && j < q.have) op.ring[RingPlace(op, t.head, t.free + i)] = op.table[r * op.table_stride + j];
}
__device__ __forceinline__ int TakenOf(const PlanTotals& t) { return min(t.wants, t.free); }
// (All of them, unless the ring's count was wrong.)
__device__ __forceinline__ int BackOf(const llmp_paged_plan& op, const PlanTotals& t) { return min(t.gives, op.ring_size - t.free); }

// THREADS: 256 for a decode step's few outputs, whose barriers four waves then meet at, or 1024 (64 requests of a token 3.3 us and
// 4.4, 200 5.2 and 5.4, 256 5.3 and 4.6). What a launch costs at all is 2 to 3 us of that.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void PlanOneKernel(const llmp_paged_plan op) {
  constexpr int kMost = THREADS;  // requests
  __shared__ int starts[kMost + 1], wants[kMost + 1], gives[kMost + 1], touched[kMost + 1], wave_sums[3 * THREADS / kWave];
  __shared__ I32x4 records[kMost];
  const PlanSums s = {starts, wants, gives, touched, records};
  const PlanTotals t = SumRequests<THREADS>(op, s, wave_sums);
  __syncthreads();
  const int items = op.tokens, taken = items + op.work_items, back = taken + TakenOf(t), end = back + BackOf(op, t);
  for (int i = threadIdx.x; i < end; i += THREADS) {
    if (i < items) {
      WriteToken(op, t, s, i);
    } else if (i < taken) {
      WriteItem(op, t, s, i - items);
    } else if (i < back) {
      WriteTaken(op, t, s, i - taken);
    } else {
      WriteBack(op, t, s, i - back);
    }
  }
}

__device__ __forceinline__ PlanSums ScratchSums(const llmp_paged_plan& op) {
  int* const at = static_cast<int*>(op.scratch) + kTotalInts;
  const int n1 = op.requests + 1;
  I32x4* const records = reinterpret_cast<I32x4*>(at);
  int* const sums = at + 4 * static_cast<int64_t>(op.requests);
  return {op.starts, sums, sums + n1, sums + 2 * static_cast<int64_t>(n1), records};
}

__global__ __launch_bounds__(kPlanThreads) void PlanSumKernel(const llmp_paged_plan op) {
  __shared__ int wave_sums[3 * kPlanThreads / kWave];
  int* totals = static_cast<int*>(op.scratch);
  const PlanTotals t = SumRequests<kPlanThreads>(op, ScratchSums(op), wave_sums);
  // (The counters may be overwritten in place: the second launch takes what they were from here.)
  if (threadIdx.x == 0) {
    totals[0] = t.head, totals[1] = t.free, totals[2] = t.wants, totals[3] = t.gives, totals[4] = t.touched, totals[5] = t.tokens;
  }
}

constexpr int kWriteThreads = 256;
// grid (blocks for tokens, then for items, then `moves` for the pages that move).
__global__ __launch_bounds__(kWriteThreads) void PlanWriteKernel(const llmp_paged_plan op, int token_blocks, int item_blocks) {
  __shared__ int search[kSearchRequests + 1];
  const int* totals = static_cast<const int*>(op.scratch);
  const PlanTotals t = {totals[0], totals[1], totals[2], totals[3], totals[4], totals[5]};
  PlanSums s = ScratchSums(op);
  const int block = blockIdx.x, kind = block < token_blocks ? 0 : block < token_blocks + item_blocks ? 1 : 2;
  // The sums that this kind's outputs are searched in.
  const auto stage = [&](int*& sums) {
    if (op.requests > kSearchRequests) return;
    __syncthreads();
    for (int r = threadIdx.x; r <= op.requests; r += kWriteThreads) search[r] = sums[r];
    sums = search;
    __syncthreads();
  };
  if (kind == 0) {
    stage(s.starts);
    for (int i = block * kWriteThreads + threadIdx.x; i < op.tokens; i += token_blocks * kWriteThreads) WriteToken(op, t, s, i);
  } else if (kind == 1) {
    stage(s.touched);
    for (int i = (block - token_blocks) * kWriteThreads + threadIdx.x; i < op.work_items; i += item_blocks * kWriteThreads) WriteItem(op, t, s, i);
  } else {
    const int first = (block - token_blocks - item_blocks) * kWriteThreads + threadIdx.x, step = (gridDim.x - token_blocks - item_blocks) * kWriteThreads;
    const PlanSums from = s;
    stage(s.wants);
    for (int i = first; i < TakenOf(t); i += step) WriteTaken(op, t, s, i);
    s = from;
    stage(s.gives);
    for (int i = first; i < BackOf(op, t); i += step) WriteBack(op, t, s, i);
  }
}

}  // namespace

int CheckPagedCache(const char* who, const llmp_paged_cache& c, bool needs_edges) {
  if (c.k == nullptr || c.v == nullptr || c.k_scale == nullptr || c.v_scale == nullptr) return Refuse(1, "%s: null array of the cache", who);
  if ((c.low == nullptr) != (c.high == nullptr) || (needs_edges && c.low == nullptr))
    return Refuse(1, "%s: the cache's low and high codes come together%s", who, needs_edges ? ", and are needed here" : "");
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return Refuse(1, "%s: head sizes 64, 128 and 256, not %d", who, c.head_dim);
  if (c.page < 16 || c.page > 256 || c.page % 16 != 0) return Refuse(1, "%s: pages of 16 to 256 tokens, a multiple of 16, not %d", who, c.page);
  if (c.pages < 1 || c.kv_heads < 1 || c.kv_heads > 65535) return Refuse(1, "%s: at least one page and 1 to 65535 KV heads (%d, %d)", who, c.pages, c.kv_heads);
  const uintptr_t all = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | reinterpret_cast<uintptr_t>(c.k_scale) |
                        reinterpret_cast<uintptr_t>(c.v_scale) | reinterpret_cast<uintptr_t>(c.low) | reinterpret_cast<uintptr_t>(c.high);
  if (all % 16 != 0) return Refuse(1, "%s: the cache's arrays lie at 16-byte boundaries", who);
  return 0;
}

int CheckPagedRows(const char* who, const char* name, const void* rows, int tokens, int heads, int64_t token_stride, int64_t head_stride, int type) {
  if (rows == nullptr) return Refuse(1, "%s: null %s", who, name);
  if (type != LLMP_X_F32 && type != LLMP_X_BF16 && type != LLMP_X_F16) return Refuse(1, "%s: F32, BF16 or F16 rows, not type %d", who, type);
  const int per = 16 / PagedElementBytes(type);
  const auto bad = [&](int count, int64_t stride) { return count > 1 && (stride < 0 || stride % per != 0); };
  if (reinterpret_cast<uintptr_t>(rows) % 16 != 0 || bad(tokens, token_stride) || bad(heads, head_stride))
    return Refuse(1, "%s: %s's rows lie at 16-byte boundaries (strides %lld, %lld)", who, name, (long long)token_stride, (long long)head_stride);
  return 0;
}

}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" int64_t llmp_hip_paged_work_items(int requests, int tokens, int page) {
  if (requests < 1 || tokens < 0 || page < 1) return 0;
  // n new tokens touch at most (n - 2) / page + 2 pages, and never more than n.
  const int64_t most = 2 * static_cast<int64_t>(requests) + tokens / page;
  return most < tokens ? most : tokens;
}

extern "C" size_t llmp_hip_paged_plan_scratch(int requests) {
  return requests < 1 ? 0 : (kTotalInts + 4 * static_cast<size_t>(requests) + 3 * (static_cast<size_t>(requests) + 1)) * sizeof(int);
}

extern "C" int llmp_hip_paged_plan(const llmp_paged_plan* op, void* stream) {
  if (op == nullptr) return Refuse(1, "paged_plan: null operands");
  if (op->requests < 1 || op->requests > 1 << 24 || op->table_width < 1 || op->ring_size < 1 || op->tokens < 0 || op->work_items < 0)
    return Refuse(1, "paged_plan: 1 to 2^24 requests, a table and a ring of at least one page (%d, %d, %d), tokens %d, work items %d", op->requests,
                  op->table_width, op->ring_size, op->tokens, op->work_items);
  // (An index of an output and the step to its thread's next one stay an int together.)
  if (op->tokens > kMostPagedLength || op->work_items > kMostPagedLength || op->ring_size > kMostPagedLength)
    return Refuse(1, "paged_plan: at most 2^30 tokens, work items and pages of the ring (%d, %d, %d)", op->tokens, op->work_items, op->ring_size);
  if (op->page < 1 || op->page > 65536) return Refuse(1, "paged_plan: pages of 1 to 65536 tokens, not %d", op->page);
  if (op->before == nullptr || op->after == nullptr || op->table == nullptr || op->ring == nullptr || op->counters_in == nullptr ||
      op->counters == nullptr || op->starts == nullptr || op->lengths == nullptr || op->scratch == nullptr ||
      (op->tokens > 0 && (op->slots == nullptr || op->positions == nullptr || op->owners == nullptr)) || (op->work_items > 0 && op->work == nullptr))
    return Refuse(1, "paged_plan: null operand");
  if (op->table_stride < op->table_width) return Refuse(1, "paged_plan: a table row of %d entries every %lld", op->table_width, (long long)op->table_stride);
  const uintptr_t words = reinterpret_cast<uintptr_t>(op->before) | reinterpret_cast<uintptr_t>(op->after) | reinterpret_cast<uintptr_t>(op->table) |
                          reinterpret_cast<uintptr_t>(op->ring) | reinterpret_cast<uintptr_t>(op->counters_in) | reinterpret_cast<uintptr_t>(op->counters) |
                          reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->lengths) | reinterpret_cast<uintptr_t>(op->slots) |
                          reinterpret_cast<uintptr_t>(op->positions) | reinterpret_cast<uintptr_t>(op->owners);
  if (words % 4 != 0 || (reinterpret_cast<uintptr_t>(op->work) | reinterpret_cast<uintptr_t>(op->scratch)) % 16 != 0)
    return Refuse(1, "paged_plan: I32 arrays at 4-byte boundaries, the work items and the scratch at 16");
  if (op->work_items < llmp_hip_paged_work_items(op->requests, op->tokens, op->page))
    return Refuse(1, "paged_plan: %d work items, %lld may be needed", op->work_items, (long long)llmp_hip_paged_work_items(op->requests, op->tokens, op->page));
  BeginLaunches();
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const int64_t outputs = static_cast<int64_t>(op->tokens) + op->work_items;
  if (op->requests <= kOneLaunchRequests && outputs <= kOneLaunchOutputs) {
    if (op->requests <= 256 && outputs < 512) {
      hipLaunchKernelGGL(PlanOneKernel<256>, dim3(1), dim3(256), 0, on, *op);
    } else {
      hipLaunchKernelGGL(PlanOneKernel<kPlanThreads>, dim3(1), dim3(kPlanThreads), 0, on, *op);
    }
  } else {
    const auto blocks = [](int64_t n) { return static_cast<int>(n < 1 ? 1 : (n + kWriteThreads - 1) / kWriteThreads < 512 ? (n + kWriteThreads - 1) / kWriteThreads : 512); };
    const int tokens = blocks(op->tokens), items = blocks(op->work_items), moves = blocks(op->ring_size);  // (no more pages can move)
    hipLaunchKernelGGL(PlanSumKernel, dim3(1), dim3(kPlanThreads), 0, on, *op);
    hipLaunchKernelGGL(PlanWriteKernel, dim3(tokens + items + moves), dim3(kWriteThreads), 0, on, *op, tokens, items);
  }
  return LaunchStatus("paged_plan");
}
