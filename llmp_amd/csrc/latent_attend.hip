// llmp.latent.attend: the absorbed form over the paged latent cache. All heads share a token's latent vector, which is key and value, so
// the rows of a request are its (token, head) pairs and one read of a tile serves all of them:
//   S^T = C Q^T (latent and rotated part), P = exp2(S - E), O^T += C^T P^T, out = O / sum of P.
//
// What bounds it: with few heads the cache's bytes (1152 a token at 512 + 64 values against 2 * 1088 operations a row; 32 requests of up to 65536, 16 heads: 213 us the
// call, 5.2 TB/s; of codes 136 us, 4.5 TB/s); from about 128 rows a token on the matrix instructions take as long (128 heads: 357 us,
// 0.75 PFLOP/s, of codes 488 us: a wave reads 68 KB of LDS a tile for 1088 cycles of products, and about as many of other instructions stand beside them). A tile is 32 tokens, brought into LDS by loads that pass no register; the rows' queries and
// results stay in registers. Two forms:
//   few rows   (no request has more than 16) every wave of a workgroup's four has all rows and a ring of tiles of its own; it waits for nobody, and the
//              waves' results are added up at the end;
//   many rows  a workgroup takes 128 rows of one request, 16 a wave (128 registers of results and 64 of queries at width 512: two waves a SIMD), all
//              waves the same ring of tiles; at width 256 also 32 a wave, two workgroups a unit.
// Both products take the tile from LDS as it lies. A product's rows are tokens in an order that leaves a lane with consecutive tokens of one row, in the
// order in which the second product takes them; the values' columns come by transposing reads.
// The work is cut evenly over the workgroups (latent_line.h).
#include <algorithm>
#include <cmath>

#include "latent_line.h"

namespace llmp_hip {
namespace {

constexpr int kTokens = 32;  // a tile's
constexpr int kFewRows = 16, kManyRows = 128;
constexpr int kLdsBytes = 160 * 1024;
constexpr int kLeast = 128;  // of the line, to a workgroup: finer parts cost more to write and to join (chunks of 20 heads at width 256: 90.3 us so, 91.8 at 64, 91.5 at 256; one
                             // request of 2000, 16 rows: 19.5, 18.1 and 22.0)

// The forms: up to 16 rows a request, each wave a tile by itself; 128 rows a workgroup, 16 a wave; so, 32 a wave, two workgroups a compute unit.
enum Form { kFewForm, kManyForm, kWideForm };

struct LatentArgs {
  llmp_latent_attend op;
  LatentParts parts;
  int most_length;
  int tokens_a_pair, pairs_a_token;  // rows of several whole tokens, or of part of one
};

template <int R, int P, bool EIGHT, Form FORM>
struct LatentGeo {
  static constexpr bool kFew = FORM == kFewForm;
  static constexpr int kSets = FORM == kWideForm ? 2 : 1;  // groups of 16 rows that a wave has
  static constexpr int kAUnit = kSets;                     // workgroups a compute unit
  static constexpr int kWaves = kFew ? 4 : 8 / kSets, kThreads = kWaves * kWave;
  static constexpr int kRows = kFew ? kFewRows : kManyRows;
  static constexpr int kPitch = EIGHT ? R : 2 * R, kRopePitch = 2 * P;
  static constexpr int kLatentBytes = kTokens * kPitch, kRopeBytes = kTokens * kRopePitch, kScaleBytes = EIGHT && !kFew ? 256 : 0;
  static constexpr int kTile = kLatentBytes + kRopeBytes + kScaleBytes;
  static constexpr int kQueries = kFew ? 0 : kManyRows * 2 * P;  // the queries' rotated part, where registers are short
  static constexpr int kRing = kFew ? std::min(2, kLdsBytes / 4 / kTile) : std::min(5, (kLdsBytes / kAUnit - kQueries) / kTile);
  static constexpr int kSharing = kFew ? 1 : kWaves;  // waves that bring a tile in
  static constexpr int kLatentLoads = kLatentBytes / 1024 / kSharing, kRopeLoads = (kRopeBytes / 1024 + kSharing - 1) / kSharing;
  static constexpr int kLoads = kLatentLoads + kRopeLoads + (kScaleBytes > 0 ? 1 : 0);  // a wave's for a tile
  static constexpr int kArea = kFewRows * R * 4 + 2 * kFewRows * 4;  // the few rows' form: a wave's results for the others
  static constexpr int kLds = kFew ? std::max(4 * kRing * kTile, 4 * kArea) : kRing * kTile + kQueries;

  // What the pieces (of 16 bytes) of a token's row are turned by: the 16 lanes that a 16-byte read takes at once (KPiece in paged_attend.h), and the 32
  // that a transposing read does, then find theirs in all banks.
  static __device__ __forceinline__ int Turn(int token) {
    if constexpr (EIGHT) return (token & 7) << 1 | (token >> 3 & 1);
    return (token & 3) << 2 | (0x1320 >> (4 * (token >> 3 & 3)) & 3);  // (0, 2, 3, 1)
  }
  static __device__ __forceinline__ int RopeTurn(int token) {
    const int eight = 0x1320 >> (4 * (token >> 3 & 3)) & 3;
    return P == 64 ? ((token >> 1 & 1) << 2 | eight) : eight;
  }
};

__device__ __forceinline__ LatentRequest AttendRequest(const LatentArgs& a, int r) {
  const PagedRequest q = RequestOf(a.op.starts, a.op.lengths, a.op.before, r, a.op.tokens, a.most_length);
  return {q.start, q.n, q.length, q.base, (q.n + a.tokens_a_pair - 1) / a.tokens_a_pair};
}

template <int TYPE, int R, int P, bool EIGHT, Form FORM>
__global__ __launch_bounds__((LatentGeo<R, P, EIGHT, FORM>::kThreads), (FORM == kFewForm ? 1 : 2)) void LatentAttendKernel(const LatentArgs a) {
  using G = LatentGeo<R, P, EIGHT, FORM>;
  constexpr bool FEW = G::kFew;
  using S = Sixteen<TYPE>;
  typedef typename S::Eight Eight;
  constexpr int kSteps = R / 32, kRopeSteps = P / 32, kBlocks = R / 16, kSets = G::kSets;
  constexpr int kLogits = 8;  // a lane's of a tile
  constexpr int kKeyGroup = FEW ? 8 : 2, kValueGroup = FEW ? 8 : 2;  // products that are read for at a time
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const llmp_latent_attend& op = a.op;
  const llmp_latent_cache& c = op.cache;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // (All that depends on the lane alone is worked out where it is needed, from a lane number as something new: kept, it is the registers too many, and what the
  // compiler then brings back from memory waits for the tiles under way. 32 rows a wave over codes have ten or eleven registers too many all the same, of which one comes
  // back between every tile's first products, and waits so.)
  const auto lane_anew = [&]() {
    if constexpr (FEW) return static_cast<int>(threadIdx.x & (kWave - 1));
    uint32_t all = ~0u;
    asm volatile("" : "+s"(all));
    return static_cast<int>(__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0)));
  };
  const int groups = gridDim.x, w = blockIdx.x;
  const uint32_t ring_off = FEW ? wave * G::kRing * G::kTile : 0;
  const uint32_t ring_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds)) + ring_off;

  // ---- this workgroup's run of the line
  const int64_t t = a.tokens_a_pair;
  if (threadIdx.x < 2) a.parts.which[(2 * w + threadIdx.x) * 4] = -1;
  // (The few rows' form keeps the first 64 requests, a lane each: looked up again, what its chain of loads begins with is one load longer.)
  LatentRequest first = {};
  if (FEW && lane_anew() < op.requests) first = AttendRequest(a, lane_anew());
  const LatentRun run = RunOf<false>(op.requests, w, groups, kLeast, [&](int r) {
    const LatentRequest l = FEW && r < kWave ? first : AttendRequest(a, r);
    return LineBefore(l, t, l.groups) * a.pairs_a_token;
  });
  int64_t u = run.from, before = run.before;
  const int64_t u_end = run.to;
  if (u >= u_end) return;

  const float sign_scale = Scalar(fabsf(op.scale) * kLog2E);
  const uint32_t flip = op.scale < 0.0f ? 0x80008000u : 0u;  // (a negative scale goes into the queries: the largest product is the largest logit)

  for (int request = run.request; u < u_end; ++request) {
    LatentRequest l;
    if (FEW && request < kWave) {
      l.start = __builtin_amdgcn_readlane(first.start, request), l.n = __builtin_amdgcn_readlane(first.n, request);
      l.length = __builtin_amdgcn_readlane(first.length, request), l.base = __builtin_amdgcn_readlane(first.base, request);
      l.groups = __builtin_amdgcn_readlane(first.groups, request);
    } else {
      l = Scalar(AttendRequest(a, request));
    }
    const int64_t all = LineBefore(l, t, l.groups) * a.pairs_a_token;
    if (u >= before + all) {
      before += all;
      continue;
    }
    for (int k = GroupAt(l, t, Over(u - before, a.pairs_a_token)); k < l.groups && u < u_end; ++k) {
      const int seen = SeenOf(l, a.tokens_a_pair, k), whole = seen + kVisit;
      const int64_t group_from = before + LineBefore(l, t, k) * a.pairs_a_token;
      for (int part = static_cast<int>(Over(u - group_from, whole)); part < a.pairs_a_token && u < u_end; ++part) {
        const int64_t from = group_from + static_cast<int64_t>(part) * whole;
        const int x0 = static_cast<int>(u - from), x1 = static_cast<int>(min(u_end - from, static_cast<int64_t>(whole)));
        u = from + x1;
        const LatentPiece piece = PieceOf(seen, kTokens, x0, x1);
        if (!piece.any) continue;
        const int tile_from = piece.from, tile_to = piece.to;

        // ---- the lane's row.
        const int first_token = k * a.tokens_a_pair;
        const int row0 = FEW ? 0 : 16 * kSets * wave;
        const int rows = a.pairs_a_token == 1 ? min(a.tokens_a_pair, l.n - first_token) * op.heads : min(G::kRows, op.heads - part * G::kRows);
        struct Row {
          int token, head, see_to;
          bool real;
        };
        const auto row_of = [&](int s) {
          const int row = row0 + 16 * s + lane_anew() % 16;
          Row r = {first_token, 0, 0, row < rows};
          if (r.real && a.pairs_a_token == 1) r.token = first_token + row / op.heads, r.head = row % op.heads;
          if (r.real && a.pairs_a_token != 1) r.head = part * G::kRows + row;
          if (r.real) r.see_to = max(min(l.base + r.token + 1, l.length), 0);
          return r;
        };
        const bool busy = row0 < rows;
        const int all_rows_to = max(min(l.base + first_token + 1, l.length), 0);  // seen by all rows of the pair
        const int all_to = max(min(l.base + first_token + 1 + (a.pairs_a_token == 1 ? row0 / op.heads : 0), l.length), 0);  // seen by all of the wave's rows

        constexpr bool kRopeInLds = G::kQueries > 0;
        Eight q[kSets][kSteps + (kRopeInLds ? 0 : kRopeSteps)];
        const uint32_t q_rope = G::kRing * G::kTile + wave * kSets * kRopeSteps * 1024;
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const Row row = row_of(s);
          const int lane = lane_anew(), quarter = lane / 16;
          const uint16_t* const ql = static_cast<const uint16_t*>(op.q_latent) + (l.start + row.token) * op.q_latent_token_stride + row.head * op.q_latent_head_stride + 8 * quarter;
          const uint16_t* const qr = static_cast<const uint16_t*>(op.q_rope) + (l.start + row.token) * op.q_rope_token_stride + row.head * op.q_rope_head_stride + 8 * quarter;
#pragma unroll
          for (int x = 0; x < kSteps + kRopeSteps; ++x) {
            U32x4 v = *reinterpret_cast<const U32x4*>(x < kSteps ? ql + 32 * x : qr + 32 * (x - kSteps));
            v ^= U32x4{flip, flip, flip, flip};
            if (kRopeInLds && x >= kSteps) {
              *reinterpret_cast<U32x4*>(lds + q_rope + (s * kRopeSteps + x - kSteps) * 1024 + 16 * lane) = v;
            } else {
              q[s][x] = __builtin_bit_cast(Eight, v);
            }
          }
        }
        F32x4 out[kSets][kBlocks];
        float top[kSets], sum[kSets];
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) out[s][b] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
          top[s] = -INFINITY, sum[s] = 0.0f;
        }

        // ---- the tiles. A lane holds the cache's row of the first token of one 16-token group of the line (-1: no page); they are looked up 64
        // at a time.
        const int32_t* const table = op.table + request * op.table_stride;
        int held_from = -1, held = 0;
        const auto look_up = [&](int tile) {
          held_from = tile;
          const uint32_t position = static_cast<uint32_t>(2 * tile + lane_anew()) * 16u, entry = position / static_cast<uint32_t>(c.page);
          held = -1;
          if (position < static_cast<uint32_t>(seen) && entry < static_cast<uint32_t>(op.table_width)) {
            const int page = table[entry];
            if (page >= 0 && page < c.pages) held = page * c.page + static_cast<int>(position - entry * c.page);
          }
        };
        const int step = FEW ? G::kWaves : 1;
        const int my_from = tile_from + (FEW ? wave : 0);
        // The few rows' form holds a tile's scales in scalar registers: with them there two tiles a wave fill LDS (32 requests of up to 65536 tokens, rope 32:
        // one tile 135 us, two 128).
        struct TileScales {
          U32x4 a, b;
        };
        TileScales scales_now = {}, scales_next = {};
        const auto tile_scales = [&](int row) { return *(const __attribute__((address_space(4))) U32x4*)(static_cast<const uint8_t*>(c.scale) + row); };
        uint32_t absent = 0;  // two bits a slot of the ring: the tile's groups without a page
        const auto fetch = [&](int tile, int slot) -> TileScales {
          if (held_from < 0 || tile >= held_from + 32) look_up(tile);
          const int at0 = __builtin_amdgcn_readlane(held, 2 * (tile - held_from)), at1 = __builtin_amdgcn_readlane(held, 2 * (tile - held_from) + 1);
          absent = (absent & ~(3u << (2 * slot))) | ((at0 < 0 ? 1u : 0u) | (at1 < 0 ? 2u : 0u)) << (2 * slot);
          const int left = seen - tile * kTokens;  // tokens of the tile, at least one; past them the last one again
          const int row_a = max(at0, 0), row_b = left > 16 ? max(at1, 0) : row_a;
          const int last_a = min(left - 1, 15), last_b = left > 16 ? min(left - 17, 15) : last_a;
          const uint8_t* const latent_a = static_cast<const uint8_t*>(c.latent) + static_cast<int64_t>(row_a) * G::kPitch;
          const uint8_t* const latent_b = static_cast<const uint8_t*>(c.latent) + static_cast<int64_t>(row_b) * G::kPitch;
          const uint8_t* const rope_a = static_cast<const uint8_t*>(c.rope) + static_cast<int64_t>(row_a) * G::kRopePitch;
          const uint8_t* const rope_b = static_cast<const uint8_t*>(c.rope) + static_cast<int64_t>(row_b) * G::kRopePitch;
          const uint32_t to = Scalar(ring_at + slot * G::kTile);
          // (Lanes and waves as something new at every tile: the compiler otherwise keeps every load's offsets, and then spills them.)
          int lane_now = lane_anew(), wave_now = FEW ? 0 : wave;
          asm volatile("" : "+v"(lane_now));
          asm volatile("" : "+s"(wave_now));
          const auto load = [&](auto whole) {
            constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
            for (int i = 0; i < G::kLatentLoads; ++i) {
              constexpr int kLanes = G::kPitch / 16, kRowsALoad = kWave / kLanes;
              const int n = i * G::kSharing + wave_now, row0 = n * kRowsALoad, row = row0 + lane_now / kLanes;
              const bool second = G::kSharing * kRowsALoad > 16 ? row0 >= 16 : i * G::kSharing * kRowsALoad >= 16;
              const uint32_t piece = 16 * ((lane_now % kLanes) ^ G::Turn(row));
              if constexpr (kWhole) {
                LineToLds((second ? latent_b : latent_a) + (row0 & 15) * G::kPitch, lane_now / kLanes * G::kPitch + piece, to + 1024 * n);
              } else {
                LineToLds(second ? latent_b : latent_a, min(row & 15, second ? last_b : last_a) * G::kPitch + piece, to + 1024 * n);
              }
            }
#pragma unroll
            for (int i = 0; i < G::kRopeLoads; ++i) {
              constexpr int kLanes = G::kRopePitch / 16, kRowsALoad = kWave / kLanes;
              const int n = FEW ? i : wave_now % (G::kRopeBytes / 1024);  // (where there are fewer than waves some come twice)
              const int row0 = n * kRowsALoad, row = row0 + lane_now / kLanes;
              const bool second = row0 >= 16;
              const uint32_t piece = 16 * ((lane_now % kLanes) ^ G::RopeTurn(row));
              LineToLds(second ? rope_b : rope_a, (kWhole ? row & 15 : min(row & 15, second ? last_b : last_a)) * G::kRopePitch + piece, to + G::kLatentBytes + 1024 * n);
            }
            // The scales: four tokens a lane, eight lanes of them.
            if constexpr (G::kScaleBytes > 0) WordToLds(c.scale, (lane_now & 4 ? row_b : row_a) + 4 * (lane_now & 3), to + G::kLatentBytes + G::kRopeBytes);
          };
          if (left >= kTokens) {
            load(std::true_type{});
          } else {
            load(std::false_type{});
          }
          if constexpr (EIGHT && FEW) return {tile_scales(row_a), tile_scales(row_b)};
          return {};
        };

        // What a lane reads of a tile. Rows are whole 256 bytes, so that a place is the lane's own (its row, its piece turned) with a constant's bits turned
        // in and a constant added. Keys: row m of the first or second product of 16 tokens (`block`) is token 8 (m / 4) + 4 block + m % 4. Values: a column's lanes name
        // their rows, of four tokens (eight where they are bytes).
        struct Places {
          uint32_t key, rope, value;
        };
        const auto places = [&]() {
          const int l = lane_anew(), quarter = l / 16, i16 = l % 16;
          const int k_token = 8 * (i16 >> 2) + (i16 & 3), v_token = 8 * quarter + (EIGHT ? i16 >> 1 : i16 >> 2);
          Places p;
          p.key = k_token * G::kPitch + (EIGHT ? 16 * (G::Turn(k_token) ^ (quarter >> 1)) + 8 * (quarter & 1) : 16 * (G::Turn(k_token) ^ quarter));
          p.rope = G::kLatentBytes + k_token * G::kRopePitch + 16 * (G::RopeTurn(k_token) ^ quarter);
          p.value = v_token * G::kPitch + 16 * (EIGHT ? G::Turn(v_token) : (i16 >> 1 & 1) ^ G::Turn(v_token)) + 8 * (i16 & 1);
          return p;
        };
        const auto key = [&](uint32_t at, uint32_t rope_at, int x, int block) {
          constexpr int kPieces = EIGHT ? 2 : 4;  // a step's
          if (x >= kSteps) return *reinterpret_cast<const Eight*>(lds + (rope_at ^ 64 * (x - kSteps)) + 4 * block * G::kRopePitch);
          const uint32_t place = (at ^ 16 * ((kPieces * x & 15) ^ (EIGHT ? 8 * block : 0))) + 256 * (kPieces * x >> 4) + 4 * block * G::kPitch;
          if constexpr (EIGHT) {
            const uint2 v = *reinterpret_cast<const uint2*>(lds + place);
            return EightE4m3<TYPE>(v.x, v.y);
          } else {
            return *reinterpret_cast<const Eight*>(lds + place);
          }
        };
        // Tokens 8 quarter to + 7 of dimension 16 b + column.
        const auto value = [&](uint32_t at, int b) {
          constexpr int kPieces = EIGHT ? 1 : 2;
          const uint32_t place = (at ^ 16 * (kPieces * b & 15)) + 256 * (kPieces * b >> 4);
          if constexpr (EIGHT) {
            const I32x2 v = Column8(lds + place);
            return EightE4m3<TYPE>(v.x, v.y);
          } else {
            const S16x4 v = Column4(lds + place);
            return JoinFours<Eight>(v, Column4(lds + place + 4 * G::kPitch));
          }
        };

        // A tile's logits of a wave's rows: element i is token 8 quarter + i.
        float dots[kSets][kLogits];
        const auto scales = [&](uint32_t tile, float (&scale)[kLogits]) {
          uint2 e;
          if constexpr (FEW) {
            const int quarter = lane_anew() / 16;
            const U32x4 a4 = scales_now.a, b4 = scales_now.b;  // (a choice of places would keep them in memory)
            const uint32_t x = quarter < 2 ? a4.x : b4.x, y = quarter < 2 ? a4.y : b4.y, z = quarter < 2 ? a4.z : b4.z, w4 = quarter < 2 ? a4.w : b4.w;
            e = make_uint2(quarter % 2 == 0 ? x : z, quarter % 2 == 0 ? y : w4);
          } else {
            e = *reinterpret_cast<const uint2*>(lds + tile + G::kLatentBytes + G::kRopeBytes + 8 * (lane_anew() / 16));
          }
#pragma unroll
          for (int i = 0; i < kLogits; ++i) {
            const uint32_t bits = (i < 4 ? e.x : e.y) >> (8 * (i & 3)) & 0xFFu;
            scale[i] = __builtin_bit_cast(float, bits == 0 ? 0x00400000u : bits << 23);
          }
        };
        const auto keys = [&](uint32_t tile) {
          const Places p = places();
          const uint32_t key_at = tile + p.key, rope_at = tile + p.rope, query_at = kRopeInLds ? q_rope + 16 * lane_anew() : 0;
          F32x4 sums[kSets][2];
#pragma unroll
          for (int s = 0; s < kSets; ++s) sums[s][0] = sums[s][1] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
          const auto steps = [&](auto from, auto to) {
            constexpr int kFrom = decltype(from)::value;
            // (Steps 256 bytes apart side by side: their places are one with two constants.)
            const auto step_of = [](int i) {
              constexpr int kSame = EIGHT ? kSteps / 8 : kSteps / 4;
              const int x = kFrom + i / 2;
              return x >= kSteps ? x : x / kSame + kSteps / kSame * (x % kSame);
            };
            ProductsInGroups<2 * (decltype(to)::value - kFrom), kKeyGroup, Eight>(
                [&](int i) { return key(key_at, rope_at, step_of(i), i % 2); },
                [&](int i, Eight k) {
                  const int x = step_of(i);
#pragma unroll
                  for (int s = 0; s < kSets; ++s) {
                    const Eight query = kRopeInLds && x >= kSteps ? *reinterpret_cast<const Eight*>(lds + query_at + (s * kRopeSteps + x - kSteps) * 1024) : q[s][kRopeInLds && x >= kSteps ? 0 : x];
                    sums[s][i % 2] = S::Product16(k, query, sums[s][i % 2]);
                  }
                });
          };
          constexpr std::integral_constant<int, 0> kBegin{};
          constexpr std::integral_constant<int, kSteps> kMiddle{};
          constexpr std::integral_constant<int, kSteps + kRopeSteps> kEnd{};
          if constexpr (EIGHT) {
            // Codes' products first: their scale is the token's, the rotated part's is one.
            steps(kBegin, kMiddle);
            float scale8[kLogits];
            scales(tile, scale8);
#pragma unroll
            for (int i = 0; i < kSets * kLogits; ++i) sums[i / kLogits][i / 4 % 2][i % 4] *= scale8[i % kLogits];
            steps(kMiddle, kEnd);
          } else {
            steps(kBegin, kEnd);
          }
#pragma unroll
          for (int i = 0; i < kSets * kLogits; ++i) dots[i / kLogits][i % kLogits] = sums[i / kLogits][i / 4 % 2][i % 4];
        };
        // A token of infinities has a weight of zero for a row that sees it with a logit of minus infinity (with another logit the row is no number altogether), which is no
        // number where it is infinite. The second product makes it so, but not of a tile whose infinities become zeros for other rows' sake (below): so it is done here, before
        // any wave does that, and then they do become zeros, whatever the others see.
        const auto keep_infinities = [&](int tile_number, uint32_t tile, uint32_t gone) -> bool {
          const int p0 = tile_number * kTokens, lane_token = 8 * (lane_anew() / 16);
          bool none = false;  // a logit that is no finite number
#pragma unroll
          for (int s = 0; s < kSets; ++s) {
            const int to = (gone >> (lane_token >> 4) & 1) != 0 ? 0 : row_of(s).see_to - p0 - lane_token;
#pragma unroll
            for (int i = 0; i < kLogits; ++i) none |= (i < to) & !(fabsf(dots[s][i]) < INFINITY);
          }
          if (!__any(none)) return false;
          // How many tokens that a row sees are odd in a dimension: a product of zeros and ones, laid out as the results are. (Without constants that the compiler would keep
          // in registers all along.)
          constexpr uint32_t kExponents = TYPE == LLMP_X_BF16 ? 0x7F807F80u : 0x7C007C00u, kLast = kExponents & (0u - kExponents);
          const auto ones = [](uint32_t two) { return (two << 14) - (TYPE == LLMP_X_BF16 ? two << 7 : two << 10); };  // of 1 or 0 in both halves
          uint32_t value_at = tile + places().value;
          asm volatile("" : "+v"(value_at));
          int to[kSets];
#pragma unroll
          for (int s = 0; s < kSets; ++s) to[s] = (gone >> (lane_token >> 4) & 1) != 0 ? 0 : row_of(s).see_to - p0 - lane_token;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) {
            U32x4 odd = __builtin_bit_cast(U32x4, value(value_at, b));
#pragma unroll
            for (int i = 0; i < 4; ++i) odd[i] = ones(((odd[i] & kExponents) + (kLast | kLast << 16)) >> 15 & 0x00010001u);
#pragma unroll
            for (int s = 0; s < kSets; ++s) {
              asm volatile("" : "+v"(to[s]));  // (anew for every product, for the same reason)
              U32x4 sees;
#pragma unroll
              for (int i = 0; i < 4; ++i) sees[i] = ones((2 * i < to[s] ? 1u : 0u) | (2 * i + 1 < to[s] ? 1u : 0u) << 16);
              const F32x4 many = S::Product16(__builtin_bit_cast(Eight, odd), __builtin_bit_cast(Eight, sees), F32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float keeps = fmaxf(1.0f - many[e], 0.0f);
                out[s][b][e] *= __builtin_amdgcn_rcpf(keeps) * keeps;  // 1, or no number
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
          return true;
        };
        const auto values = [&](int tile_number, uint32_t tile, uint32_t gone, bool alone, bool kept) {
          const uint32_t value_at = tile + places().value;
          const int p0 = tile_number * kTokens;
          float scale8[kLogits];
          if constexpr (EIGHT) scales(tile, scale8);
          bool garbage = kept;
          Eight weights[kSets];
          const bool masked = p0 + kTokens > all_to || gone != 0;
          const float worth = masked ? 1.0f : sign_scale;
#pragma unroll
          for (int s = 0; s < kSets; ++s) {
            // ---- what the rows see
            float (&dot)[kLogits] = dots[s];
            float copy8[kLogits];
            float (&seen8)[kLogits] = kSets == 1 ? scale8 : copy8;
            if constexpr (EIGHT && kSets > 1) {
#pragma unroll
              for (int i = 0; i < kLogits; ++i) seen8[i] = scale8[i];
            }
            if (masked) {
              asm volatile("" ::: "memory");  // (a branch: selects would be in every tile's way)
              const int lane_token = 8 * (lane_anew() / 16);
              const int to = (gone >> (lane_token >> 4) & 1) != 0 ? 0 : row_of(s).see_to - p0 - lane_token;
#pragma unroll
              for (int i = 0; i < kLogits; ++i) {
                // (A value that is no number, or one that a product with zero would make none, has no finite product with any query.)
                garbage |= (i >= to) & !(fabsf(dot[i]) < INFINITY);
                dot[i] = i < to ? dot[i] * sign_scale : -INFINITY;
                if constexpr (EIGHT) seen8[i] = i < to ? seen8[i] : 0.0f;
              }
            }
            // ---- softmax. Eight-bit weights take the token's scale along; the maximum is of both.
            float peak = -INFINITY;
            if constexpr (EIGHT) {
#pragma unroll
              for (int i = 0; i < kLogits; ++i) peak = fmaxf(peak, fmaf(dot[i], worth, __builtin_amdgcn_logf(fmaxf(seen8[i], 0x1p-80f))));
            } else {
#pragma unroll
              for (int i = 0; i < kLogits; i += 2) peak = fmaxf(fmaxf(peak, dot[i]), dot[i + 1]);
              peak *= worth;
            }
            peak = AcrossGroupsMax(peak);
            if (__any(peak > top[s] + (kUp + kFollow))) {
              const float higher = peak > top[s] + (kUp + kFollow) ? peak - kUp : top[s];  // (a row's own: what other rows see changes no bit of it)
              const float keep = top[s] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[s] - higher);
              top[s] = higher;
              sum[s] *= keep;
#pragma unroll
              for (int b = 0; b < kBlocks; ++b) out[s][b] *= keep;
            }
            const float less = top[s] == -INFINITY ? 0.0f : top[s];
#pragma unroll
            for (int i = 0; i < kLogits; i += 2) {
              const float p = __builtin_amdgcn_exp2f(fmaf(dot[i], worth, -less)), p1 = __builtin_amdgcn_exp2f(fmaf(dot[i + 1], worth, -less));
              if constexpr (EIGHT) {
                // (Rounded with the token's scale in them, for the reason below; the sum is of what they are before that, and so a weight's rounding is in it once.)
                sum[s] += p + p1;
                weights[s][i] = static_cast<typename S::One>(p * seen8[i]), weights[s][i + 1] = static_cast<typename S::One>(p1 * seen8[i + 1]);
              } else {
                // (Rounded to the cache's type, for the matrix instructions that take 16-bit values: 2^-8 of a weight, F16 2^-11, beside the result's own rounding, which
                // is as large. Weights of 32 bits as two of 16 would be twice the second product.)
                weights[s][i] = static_cast<typename S::One>(p), weights[s][i + 1] = static_cast<typename S::One>(p1);
                // (The sum is of the weights as they are rounded, two in an instruction.)
                sum[s] = S::AddTwo(typename S::Two{weights[s][i], weights[s][i + 1]}, sum[s]);
              }
            }
          }
          if (alone && __any(garbage)) {
            // A token that some row must not see holds infinities or NaN, which a weight of zero does not keep out: they become zeros in LDS. (A row that
            // sees them is no number, or has been seen to. `alone`: nobody reads the tile as keys any more. Elsewhere all rows see the same.)
#pragma unroll 1
            for (uint32_t i = 16 * lane_anew(); i < G::kLatentBytes; i += 1024) {
              U32x4* const at = reinterpret_cast<U32x4*>(lds + tile + i);
              *at = EIGHT ? FiniteCodes(*at) : Finite<TYPE>(*at);
            }
          }
          if (!FEW && alone) MeetLds();
          // (Blocks 256 bytes apart side by side, for the same reason as the keys' steps.)
          const auto block_of = [](int i) {
            constexpr int kSame = EIGHT ? kBlocks / 16 : kBlocks / 8;
            return i / kSame + kBlocks / kSame * (i % kSame);
          };
          ProductsInGroups<kBlocks, kValueGroup, Eight>([&](int i) { return value(value_at, block_of(i)); },
                                                        [&](int i, Eight v) {
#pragma unroll
                                                          for (int s = 0; s < kSets; ++s) out[s][block_of(i)] = S::Product16(v, weights[s], out[s][block_of(i)]);
                                                        });
        };

        if constexpr (FEW) {
          // A wave's own ring: nobody waits for anybody.
          const int count = tile_to > my_from ? (tile_to - my_from + step - 1) / step : 0;
          if (count > 0) scales_now = fetch(my_from, 0);
          if (G::kRing == 2 && count > 1) scales_next = fetch(my_from + step, 1);
          for (int i = 0; i < count; ++i) {
            if (G::kRing == 2 && i + 1 < count) {
              WaitLoads<G::kLoads>();
            } else {
              WaitLoads<0>();
            }
            const int tile = my_from + i * step;
            const uint32_t at = ring_off + i % G::kRing * G::kTile, gone = absent >> (2 * (i % G::kRing)) & 3u;
            keys(at);
            values(tile, at, gone, true, !EIGHT && ((tile + 1) * kTokens > all_to || gone != 0) && keep_infinities(tile, at, gone));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            scales_now = scales_next;
            if (i + G::kRing < count) (G::kRing == 1 ? scales_now : scales_next) = fetch(my_from + (i + G::kRing) * step, i % G::kRing);
          }
        } else {
          const int count = Scalar(tile_to - tile_from);
          constexpr int kAhead = G::kRing - 1;
          for (int i = 0; i < kAhead && i < count; ++i) fetch(tile_from + i, i);
          const bool early = wave < G::kWaves / 2;
          const bool one_token = a.tokens_a_pair == 1 || rows <= op.heads;
          for (int i = 0; i < count; ++i) {
            // Tile i has landed: of the tiles asked for only later ones are under way.
            const int later = min(kAhead - 1, count - 1 - i);
            if (later >= 3) {
              WaitLoads<3 * G::kLoads>();
            } else if (later == 2) {
              WaitLoads<2 * G::kLoads>();
            } else if (later == 1) {
              WaitLoads<G::kLoads>();
            } else {
              WaitLoads<0>();
            }
            MeetLds();
            // (Half of the waves ask for their part now, half between the products: all at once they wait for each other's loads to be taken.)
            const bool more = i + kAhead < count;
            if (more && early) fetch(tile_from + i + kAhead, (i + kAhead) % G::kRing);
            const uint32_t at = i % G::kRing * G::kTile, gone = absent >> (2 * (i % G::kRing)) & 3u;
            // (Values that some row must not see may have to be changed in LDS: once nobody multiplies them as keys any more.)
            const bool careful = gone != 0 || (!one_token && (tile_from + i + 1) * kTokens > all_rows_to);
            if (busy) keys(at);
            if (more && !early) fetch(tile_from + i + kAhead, (i + kAhead) % G::kRing);
            bool kept = false;
            if (careful) {
              kept = !EIGHT && busy && keep_infinities(tile_from + i, at, gone);
              MeetLds();
            }
            if (busy) values(tile_from + i, at, gone, careful, kept);
            if (!busy && careful) MeetLds();  // (with the others, before they read the values)
          }
          MeetLds();
        }
#pragma unroll
        for (int s = 0; s < kSets; ++s) sum[s] = AcrossGroupsSum(sum[s]);

        // ---- the few rows' form: the waves' results added up, a quarter of the dimensions each.
        const int lane = lane_anew(), quarter = lane / 16, column = lane % 16;
        constexpr int kMine = FEW ? kBlocks / 4 : kBlocks;  // blocks that the wave writes
        const int first_block = FEW ? wave * kMine : 0;
        if constexpr (FEW) {
          F32x4 result[kMine];
          MeetLds();
          uint8_t* const area = lds + wave * G::kArea;
#pragma unroll
          for (int b = 0; b < kBlocks; ++b) reinterpret_cast<F32x4*>(area)[b * kWave + lane] = out[0][b];
          if (quarter == 0) reinterpret_cast<float2*>(area + kFewRows * R * 4)[column] = make_float2(top[0], sum[0]);
          MeetLds();
          float2 numbers[4];
          top[0] = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) numbers[i] = reinterpret_cast<const float2*>(lds + i * G::kArea + kFewRows * R * 4)[column], top[0] = fmaxf(top[0], numbers[i].x);
          sum[0] = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            numbers[i].x = __builtin_amdgcn_exp2f(numbers[i].x - (top[0] == -INFINITY ? 0.0f : top[0]));
            sum[0] = fmaf(numbers[i].x, numbers[i].y, sum[0]);
          }
#pragma unroll
          for (int b = 0; b < kMine; ++b) {
            result[b] = F32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) result[b] += reinterpret_cast<const F32x4*>(lds + i * G::kArea)[(first_block + b) * kWave + lane] * numbers[i].x;
          }
          MeetLds();
#pragma unroll
          for (int b = 0; b < kMine; ++b) out[0][b] = result[b];
        }

        // ---- out, or a part for the join. Element e of a block is dimension 4 quarter + e of it.
        if (piece.begins && piece.ends) {
#pragma unroll
          for (int s = 0; s < kSets; ++s) {
            const Row row = row_of(s);
            if (!row.real) continue;
            const float by = sum[s] > 0.0f || sum[s] != sum[s] ? 1.0f / sum[s] : 0.0f;
            const int64_t to = (l.start + row.token) * op.out_token_stride + row.head * op.out_head_stride + 16 * first_block + 4 * quarter;
#pragma unroll
            for (int b = 0; b < kMine; ++b) {
              const float v[4] = {out[s][b][0] * by, out[s][b][1] * by, out[s][b][2] * by, out[s][b][3] * by};
              StoreValues<TYPE, 4>(op.out, to + 16 * b, v);
            }
          }
        } else {
          const int which = 2 * w + (piece.begins ? 1 : 0);
          if (wave == 0 && lane == 0) {
            const LatentOwners owners = OwnersOf(from, seen, kTokens, run.per);
            *reinterpret_cast<I32x4*>(a.parts.which + 4 * which) = I32x4{owners.first, k * a.pairs_a_token + part, rows | owners.count << 8, l.start + first_token};
          }
#pragma unroll
          for (int s = 0; s < kSets; ++s) {
            if (row0 + 16 * s >= rows) continue;
            const int64_t rows16 = static_cast<int64_t>(which) * (G::kRows / 16) + row0 / 16 + s;
            if (quarter == 0) a.parts.numbers[rows16 * 16 + column] = make_float2(top[s], sum[s]);
            F32x4* const to = reinterpret_cast<F32x4*>(a.parts.values) + (rows16 * kBlocks + first_block) * kWave + lane;
#pragma unroll
            for (int b = 0; b < kMine; ++b) to[b * kWave] = out[s][b];
          }
        }
      }
    }
    before += all;
  }
}

// f with the type, width, rope width, 8 bits or not and the form as constants.
template <class F>
void WithForm(const llmp_latent_attend& op, Form which, F&& f) {
  const auto form = [&](auto type, auto r, auto p) {
    const auto forms = [&](auto eight) {
      if (which == kFewForm) f(type, r, p, eight, std::integral_constant<Form, kFewForm>{});
      if (which == kManyForm) f(type, r, p, eight, std::integral_constant<Form, kManyForm>{});
      if constexpr (decltype(r)::value == 256) {
        if (which == kWideForm) f(type, r, p, eight, std::integral_constant<Form, kWideForm>{});
      }
    };
    if (op.cache.scale != nullptr) forms(std::true_type{});
    if (op.cache.scale == nullptr) forms(std::false_type{});
  };
  const auto widths = [&](auto type) {
    const auto rope = [&](auto r) {
      if (op.cache.rope_width == 32) form(type, r, std::integral_constant<int, 32>{});
      if (op.cache.rope_width == 64) form(type, r, std::integral_constant<int, 64>{});
    };
    if (op.cache.width == 256) rope(std::integral_constant<int, 256>{});
    if (op.cache.width == 512) rope(std::integral_constant<int, 512>{});
  };
  if (op.cache.type == LLMP_X_BF16) widths(std::integral_constant<int, LLMP_X_BF16>{});
  if (op.cache.type == LLMP_X_F16) widths(std::integral_constant<int, LLMP_X_F16>{});
}

// 32 rows a wave read LDS half as often and share what is worked out a tile, but there are twice the parts to join: where requests have more rows than one pair.
// (Width 256, 20 heads, three chunks of up to 300 tokens behind 5000: 90 us, 104 with
// 16 rows a wave; of codes 116 and 138; 32 requests of two tokens and 128 heads behind up to 9000: 67 and 73, of codes 81 and 90; of one token, a single pair a
// request, 63 and 56.)
Form FormOf(const llmp_latent_attend& op) {
  const int64_t rows = static_cast<int64_t>(std::min(op.most_tokens, op.tokens)) * op.heads;
  return rows <= kFewRows ? kFewForm : op.cache.width == 256 && rows > kManyRows ? kWideForm : kManyForm;
}
int RowsOf(const llmp_latent_attend& op) { return FormOf(op) == kFewForm ? kFewRows : kManyRows; }
int GroupsOf(const llmp_latent_attend& op, int cus) { return FormOf(op) == kWideForm ? 2 * cus : cus; }

int CheckLatentAttend(const llmp_latent_attend* op, int cus) {
  if (op == nullptr) return Refuse(1, "latent_attend: null operands");
  if (const int bad = CheckLatentCache("latent_attend", op->cache); bad != 0) return bad;
  if (op->heads < 1 || op->requests < 1 || op->requests > 1 << 24 || op->tokens < 1 || op->most_tokens < 1 || op->table_width < 1 ||
      static_cast<int64_t>(op->heads) * op->tokens > INT_MAX / 2 || op->heads > 65535)
    return Refuse(1, "latent_attend: 1 to 2^24 requests, at least one token and one page a table row, at most 65535 heads and 2^30 of them in all tokens (%d, %d, %d, %d, %d)",
                  op->requests, op->tokens, op->most_tokens, op->table_width, op->heads);
  const int type = op->cache.type;
  if (const int bad = CheckPagedRows("latent_attend", "q_latent", op->q_latent, op->tokens, op->heads, op->q_latent_token_stride, op->q_latent_head_stride, type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("latent_attend", "q_rope", op->q_rope, op->tokens, op->heads, op->q_rope_token_stride, op->q_rope_head_stride, type); bad != 0) return bad;
  if (const int bad = CheckPagedRows("latent_attend", "out", op->out, op->tokens, op->heads, op->out_token_stride, op->out_head_stride, type); bad != 0) return bad;
  if (op->lengths == nullptr || op->starts == nullptr || op->table == nullptr) return Refuse(1, "latent_attend: null operand");
  if ((reinterpret_cast<uintptr_t>(op->lengths) | reinterpret_cast<uintptr_t>(op->starts) | reinterpret_cast<uintptr_t>(op->table) |
       reinterpret_cast<uintptr_t>(op->before)) % 4 != 0)
    return Refuse(1, "latent_attend: I32 arrays at 4-byte boundaries");
  if (op->requests > 1 && op->table_stride < op->table_width)
    return Refuse(1, "latent_attend: a table row of %d entries every %lld", op->table_width, (long long)op->table_stride);
  if (static_cast<int64_t>(op->table_width) * op->cache.page > kMostPagedLength) return Refuse(1, "latent_attend: a table row of at most 2^30 tokens");
  if (!std::isfinite(op->scale)) return Refuse(1, "latent_attend: a scale that is not finite");
  if (cus < 1 || cus > 4096) return Refuse(1, "latent_attend: %d compute units", cus);
  return 0;
}

}  // namespace
}  // namespace llmp_hip

using namespace llmp_hip;

extern "C" size_t llmp_hip_latent_attend_scratch(const llmp_latent_attend* op, int cus) {
  if (CheckLatentAttend(op, cus) != 0) return 0;
  return LatentPartsBytes(GroupsOf(*op, cus), RowsOf(*op), op->cache.width);
}

extern "C" int llmp_hip_latent_attend(const llmp_latent_attend* op, void* scratch, size_t scratch_bytes, int cus, void* stream) {
  if (const int bad = CheckLatentAttend(op, cus); bad != 0) return bad;
  const size_t need = llmp_hip_latent_attend_scratch(op, cus);
  if (scratch == nullptr || scratch_bytes < need || reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
    return Refuse(1, "latent_attend: %zu bytes of scratch at a 16-byte boundary, not %zu", need, scratch_bytes);
  const int rows = RowsOf(*op), groups = GroupsOf(*op, cus);
  LatentArgs a;
  a.op = *op;
  a.parts = LatentPartsAt(scratch, groups, rows);
  a.most_length = op->table_width * op->cache.page;
  a.tokens_a_pair = std::max(1, rows / op->heads);
  a.pairs_a_token = (op->heads + rows - 1) / rows;
  const JoinArgs join = {a.parts, op->out, op->out_token_stride, op->out_head_stride, op->heads, groups, a.pairs_a_token};
  BeginLaunches();
  const auto s = static_cast<hipStream_t>(stream);
  WithForm(*op, FormOf(*op), [&](auto type, auto r, auto p, auto eight, auto form) {
    constexpr int kType = decltype(type)::value, kR = decltype(r)::value, kP = decltype(p)::value;
    constexpr bool kEight = decltype(eight)::value;
    constexpr Form kForm = decltype(form)::value;
    using G = LatentGeo<kR, kP, kEight, kForm>;
    static_assert(G::kRing >= (G::kFew ? 1 : 3) && G::kLds <= kLdsBytes / G::kAUnit, "a ring of tiles");
    constexpr int kLds = G::kLds;
    static bool sized = false;
    if (!AllowLds(reinterpret_cast<const void*>(&LatentAttendKernel<kType, kR, kP, kEight, kForm>), kLds, &sized)) return;
    hipLaunchKernelGGL((LatentAttendKernel<kType, kR, kP, kEight, kForm>), dim3(groups), dim3(G::kThreads), kLds, s, a);
    hipLaunchKernelGGL((LatentJoinKernel<kType, kR, 16, G::kRows>), dim3(groups, 2), dim3(kJoinWaves * kWave), 0, s, join);
  });
  return LaunchStatus("latent_attend");
}
