// Attention of a few query rows over the 4-bit cache, on tensor cores.
//
// For one sequence and cache head with rows r (new tokens x query heads that share the head), tokens t:
//   S[t][r] = sum_g ks[t,g] sum_{d in g} (kc[t,d] - kz[t,g]) q[r,d]
//   O[d][r] = sum_t (vc[t,d] - vz[t,g]) P[t,r],   P[t,r] = vs[t,g] exp2(f[r] S[t][r] - m[r])
// Both products take the codes as the 16-row operand A of m16n8k16 (tokens x channels, then channels x tokens)
// and the rows as its 8 columns, so 8 rows cost one instruction per 256 codes.
//   Keys' operands: a nibble put into the low bits of the fp16 1024 is 1024 + code, and one place higher 1024 + 16 code; less the
//   same of the zero point it is exact and normal.  (The bare nibble, a subnormal, saves the subtraction, 3 % of the time, but
//   the adder lines subnormals up by their exponent field and loses about 10 of the sum's bits: log-sums of short sequences
//   off by 1.7e-6, 5e-8 so.)
//   Keys: every second query value is divided by 16 for the codes one place higher.  Query rows are scaled by a power of
//   two to a maximum in [2^14, 2^15), so that they fit fp16 whatever their type; fp32 rows are split into two fp16 terms (22 bits).
//   Values: 128 + code less 128 + zero point in bf16, exact. P is fp32's value in bf16 terms, each of which has fp32's range:
//   two (17 bits or more) in 16-bit calls, three (24) in fp32 ones, for every token, however small its weight or its scale beside
//   the others'.  (fp16 weights of 11 and 22 bits take 71 and 92 us below, but on a step of 2^-24 of the largest they put 16-bit
//   outputs off by 2e-4 before their own rounding, and fp32 ones by 1e-5 to 6e-2 where one token or one group of channels
//   outweighs the rest by 2^10 to 2^20.)
//   The adder truncates, always towards 0, so a tile's sums are added up outside of it (3 % of the time below, but 131072 tokens
//   that one block adds up leave outputs 5e-5 low, and it grows with the length).
//   P leaves the first product as (token, row) and must enter the second as (row, token): movmatrix.
// The maximum m[r] is a running reference, raised (and the sums rescaled) only when a score passes it by more than
// 2^8: a warp-wide maximum is taken a few times per sequence, not per tile.
//
// Work: a unit is (sequence, cache head, tile of rows), in steps of kWarps tiles of kTile tokens.  All units' steps lie
// end to end, and each block takes the same number of them, whatever the lengths (which only the device knows): none waits
// for a last wave.  The parts of a unit that several blocks share go to
// the scratch, and the block that finishes last joins them in order.
//
// What bounds it: bytes, D / 2 + 4 D / G for each of K and V per token and head; and, as measured, the latency of about 855
// instructions per warp and tile with 12 warps an SM.  48 sequences of up to 8192 tokens, 32 / 8 heads x 128, bf16: 79.5 us,
// 2.8 TB/s; 2 x 131072, fp16: 102 us, 3.0 TB/s; 1 x 77 fp32: 6 us, all latency.
//   Each warp owns a ring of kStages tiles of kTile tokens that it fills with 16-byte asynchronous copies and empties on its
// own: no block-wide barrier until the end.  A row of codes is padded by 16 bytes in shared memory: then lanes (g, t)
// reading 4 bytes at g rows down, and 2t rows down, both touch 32 banks once.
#pragma once
#include <type_traits>

#include "host.h"
#include "lowbit.cuh"

namespace b200q {

struct Cache {
  uint8_t* codes[2];
  uint32_t* params[2];
  int pages, heads, page_size, d, group;
  int64_t slots;
  Divisor page, both_heads;  // by the page size, by 2 * heads
};

struct AttnArgs {
  const void* q;
  long long q_bs, q_ts, q_hs;
  const int32_t* table;
  long long table_stride;
  const int32_t* lens;
  void* out;
  float* lse;
  int ftype, b, tq, hq, max_pages;
  float scale;
  int row_tiles;        // tiles of 8 * NT rows of a cache head
  float* partial;       // [block][2][8 NT][d] sums of a part: of a unit begun by an earlier block, of one begun here
  float* partial_ml;    // [block][2][8 NT][2] maximum and total
  unsigned* counters;   // [block], for the unit begun here
  int* err;
};

constexpr int kMinSteps = 2;  // steps of a unit's first and last part at least
// What a unit costs besides its steps (its queries, its first tiles' way, its join), in steps: 48 sequences of 128 to 8192
// tokens 79.5 us with 2, 80.9 with 1, 81.3 with 3, 84.6 with 5; 1 x 1024 10.5 us, 12.0, 11.7 and 12.0.
constexpr int kUnitSteps = 2;

constexpr int kTile = 32;    // tokens of a warp's step
constexpr int kWarps = 4;    // a block's warps take tiles in turn
constexpr int kStages = 2;   // tiles of a warp's ring: a third one costs a block an SM for heads of 256 (85 against 60 us)
constexpr int kStepTokens = kWarps * kTile;

// How far a weight may pass 1 before its row's reference is raised, and its logarithm.
constexpr float kLag = 256.0f, kLagLog = 8.0f;

template <int D, int G, int NT, bool F32>
struct AttnShape {
  static constexpr int kPitch = D / 2 + 16;
  static constexpr int kGroups = D / G;
  static constexpr int kCodes = kTile * kPitch;
  static constexpr int kParams = kTile * kGroups * 4;
  static constexpr int kStage = 2 * (kCodes + kParams);
  static constexpr int kTerms = F32 ? 2 : 1;                       // fp16 terms of a query value
  static constexpr int kQuery = (D / 32) * kTerms * NT * 32 * 16;  // operand B of the first product
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kJoin = kWarps * 8 * NT * (D + 4) * 4;      // the warps' sums, over the ring
  static constexpr int kBody = kRing > kJoin ? kRing : kJoin;
  static constexpr int kTileParams = kTile * kGroups * 14;        // a warp's tile: what its lanes unpack for one another
  static constexpr int kRowsMl = kWarps * 8 * NT * 2 * 4;
  static constexpr int kSmem = kBody + kQuery + kWarps * kTileParams + kRowsMl + 8 * NT * 24;
};

// Row of the cache that holds token `tok`, or ~0 where there is none to read.
__device__ __forceinline__ uint32_t token_row(const Cache& c, const AttnArgs& a, const int32_t* pages, int head, int tok,
                                              int until) {
  if (tok >= until) return ~0u;
  const int at = static_cast<int>(c.page.of(static_cast<uint32_t>(tok)));
  const int page = __ldg(pages + at);
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(c.pages)) {
    atomicCAS(a.err, 0, kDevErrBadPage);
    return ~0u;
  }
  return (static_cast<uint32_t>(page) * c.heads + head) * c.page_size + (tok - at * c.page_size);
}

// Tokens of a sequence; none where the length is not one that the block table can hold.
__device__ __forceinline__ int valid_length(const Cache& c, const AttnArgs& a, int seq) {
  const int len = __ldg(a.lens + seq);
  if (len >= 0 && len <= static_cast<long long>(a.max_pages) * c.page_size) return len;
  atomicCAS(a.err, 0, kDevErrBadLength);
  return 0;
}

// Four channels of an output that may begin at any element.
__device__ __forceinline__ void store_four(int ftype, void* p, long long i, float4 v) {
  if (ftype == B200Q_F32) {
    float* to = static_cast<float*>(p) + i;
    if (reinterpret_cast<uintptr_t>(p) % 16 == 0)
      *reinterpret_cast<float4*>(to) = v;
    else
      to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
  } else {
    uint16_t* to = static_cast<uint16_t*>(p) + i;
    const uint2 w = ftype == B200Q_F16 ? make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w)) : make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
    if (reinterpret_cast<uintptr_t>(p) % 8 == 0)
      *reinterpret_cast<uint2*>(to) = w;
    else
      to[0] = w.x & 0xffff, to[1] = w.x >> 16, to[2] = w.y & 0xffff, to[3] = w.y >> 16;
  }
}

// Issues the copies of one tile: lane l holds the cache row of token l.
template <int D, int G>
__device__ __forceinline__ void load_tile(const Cache& c, uint32_t stage, uint32_t row, int lane) {
  constexpr int kChunks = D / 32, kPitch = D / 2 + 16, kCodes = kTile * kPitch, kGroups = D / G;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int i = j * 32 + lane, tok = i / kChunks, chunk = i % kChunks;
    const uint32_t r = __shfl_sync(~0u, row, tok);
    if (r != ~0u) {
      const size_t from = static_cast<size_t>(r) * (D / 2) + chunk * 16;
      const uint32_t to = stage + tok * kPitch + chunk * 16;
      copy_async<16>(to, c.codes[0] + from);
      copy_async<16>(to + kCodes, c.codes[1] + from);
    }
  }
  if (row != ~0u) {
    constexpr int kBytes = kGroups * 4 < 16 ? kGroups * 4 : 16;
    const uint32_t to = stage + 2 * kCodes + lane * kGroups * 4;
#pragma unroll
    for (int b = 0; b < kGroups * 4; b += kBytes) {
      copy_async<kBytes>(to + b, reinterpret_cast<const uint8_t*>(c.params[0]) + static_cast<size_t>(row) * kGroups * 4 + b);
      copy_async<kBytes>(to + kTile * kGroups * 4 + b,
                         reinterpret_cast<const uint8_t*>(c.params[1]) + static_cast<size_t>(row) * kGroups * 4 + b);
    }
  }
}

// The same where a tile's tokens lie in one page (pages of a multiple of kTile tokens): `row` is that of the tile's first
// token in every lane, and what is copied is contiguous.  n: tokens to copy.
template <int D, int G>
__device__ __forceinline__ void load_tile_page(const Cache& c, uint32_t stage, uint32_t row, int n, int lane) {
  constexpr int kChunks = D / 32, kPitch = D / 2 + 16, kCodes = kTile * kPitch, kGroups = D / G, kRows = 32 / kChunks;
  const size_t from = static_cast<size_t>(row) * (D / 2) + lane * 16;
  const uint8_t* k = c.codes[0] + from;
  const uint8_t* v = c.codes[1] + from;
  const uint32_t to = stage + lane / kChunks * kPitch + lane % kChunks * 16;
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
    if (n >= kTile || j * kRows + lane / kChunks < n) {
      copy_async<16>(to + j * kRows * kPitch, k + j * 512);
      copy_async<16>(to + j * kRows * kPitch + kCodes, v + j * 512);
    }
  if (lane < n) {
    constexpr int kBytes = kGroups * 4 < 16 ? kGroups * 4 : 16;
    const size_t param = (static_cast<size_t>(row) + lane) * (kGroups * 4);
    const uint32_t at = stage + 2 * kCodes + lane * kGroups * 4;
#pragma unroll
    for (int b = 0; b < kGroups * 4; b += kBytes) {
      copy_async<kBytes>(at + b, reinterpret_cast<const uint8_t*>(c.params[0]) + param + b);
      copy_async<kBytes>(at + kTile * kGroups * 4 + b, reinterpret_cast<const uint8_t*>(c.params[1]) + param + b);
    }
  }
}

// Where a block stands: in shared memory, so that it takes no registers while tiles are computed.
struct Plan {
  uint32_t total, stop, at, base;  // steps of all units, the block's end, its next step, its sequence's first
  int seq, len, n;                 // the sequence, its length, the steps of each of its units
  // the unit at hand: its sequence, cache head and tile of rows, whether its first part is here, the block of that,
  // how many parts it has
  int unit_seq, head, tile, begins, owner, parts;
};

// Blocks an SM: three at up to 168 registers a thread for heads of 128 (2 x 131072 tokens: 102 us, 128 with four and spills,
// 111 with two), four for heads of 64 (48 sequences of up to 8192: 51.7 us, 53.6 with three); 16 rows a pass or 256 channels take what they need.
template <int D, int G, int NT, bool F32>
__global__ void __launch_bounds__(kWarps * 32, NT > 1 || D == 256 ? 1 : D == 128 ? 3 : 4) kv4_attention_kernel(Cache c, AttnArgs a) {
  using Shape = AttnShape<D, G, NT, F32>;
  constexpr int kGroups = Shape::kGroups, kPitch = Shape::kPitch, kRows = 8 * NT, kTerms = Shape::kTerms;
  constexpr uint32_t kMagic = 0x64006400u;  // two fp16 1024: with a code in the low bits 1024 + code
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned arrived;
  __shared__ Plan plan;
  wait_for_previous();
  uint4* const query = reinterpret_cast<uint4*>(smem + Shape::kBody);
  uint8_t* const prepared = smem + Shape::kBody + Shape::kQuery + (threadIdx.x / 32) * Shape::kTileParams;
  float* const row_ml = reinterpret_cast<float*>(smem + Shape::kBody + Shape::kQuery + kWarps * Shape::kTileParams);
  float* const row_f = row_ml + kWarps * kRows * 2;
  int64_t* const row_out = reinterpret_cast<int64_t*>(row_f + kRows);
  float2* const row_all = reinterpret_cast<float2*>(row_out + kRows);
  int* const row_limit = reinterpret_cast<int*>(row_all + kRows);  // tokens that a row sees
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;

  const int units = c.heads * a.row_tiles, ratio = a.hq / c.heads;
  auto steps_of = [&](int len) { return kUnitSteps + max(1, (len + kStepTokens - 1) / kStepTokens); };
  // Block i takes total / blocks steps, and one more while i is below the remainder.  A cut that would leave a part of less
  // than kMinSteps steps at a unit's start or end moves there.
  auto blocks_for = [&](uint32_t total) { return min(gridDim.x, total); };
  // (By one warp, and each length that a unit goes by is read once: a block's threads agree, stay in bounds and end even if a
  // program changes the lengths meanwhile.)
  auto plan_block = [&]() -> Plan {
    uint32_t total = 0;
    for (int i = lane; i < a.b; i += 32) total += steps_of(valid_length(c, a, i));
#pragma unroll
    for (int x = 16; x; x >>= 1) total += __shfl_xor_sync(~0u, total, x);
    total *= units;
    const uint32_t blocks = blocks_for(total);
    if (blockIdx.x >= blocks) return Plan{};
    const uint32_t per = total / blocks, more = total - per * blocks;
    int seq = 0, len = 0, n = 0;
    uint32_t base = 0;
    // the sequence of a step; none only where lengths were changed since they were added up: the block then ends
    auto find = [&](uint32_t step) {
      base = 0;
      for (seq = 0; seq < a.b; seq += 32) {
        const int own = seq + lane < a.b ? valid_length(c, a, seq + lane) : 0, mine = seq + lane < a.b ? steps_of(own) : 0;
        uint32_t sum = mine * units;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const uint32_t v = __shfl_up_sync(~0u, sum, x);
          if (lane >= x) sum += v;
        }
        const unsigned past = __ballot_sync(~0u, base + sum > step);
        if (past) {
          const int first = __ffs(past) - 1;
          len = __shfl_sync(~0u, own, first);
          n = steps_of(len);
          base += __shfl_sync(~0u, sum, first) - n * units;
          seq += first;
          return true;
        }
        base += __shfl_sync(~0u, sum, 31);
      }
      return false;
    };
    auto cut = [&](uint32_t i) {
      const uint32_t step = i * per + min(i, more);
      if (step >= total || !find(step)) return total;
      const uint32_t unit_at = base + (step - base) / n * n;
      return step - unit_at < kUnitSteps + kMinSteps ? unit_at : unit_at + n - step < kMinSteps ? unit_at + n : step;
    };
    const uint32_t stop = cut(blockIdx.x + 1), at = cut(blockIdx.x);
    if (at >= stop || seq >= a.b) return Plan{};
    if (at == base + static_cast<uint32_t>(n) * units) {
      if (++seq >= a.b) return Plan{};
      base = at, len = valid_length(c, a, seq), n = steps_of(len);
    }
    return Plan{total, stop, at, base, seq, len, n};
  };
  if (warp == 0) {
    const Plan mine = plan_block();
    if (lane == 0) plan = mine;
  }
  __syncthreads();
  if (plan.at >= plan.stop) return;

  for (;;) {
    // steps [off, off + count) of the unit; its first kUnitSteps steps stand for what it costs besides
    const int seq = plan.seq, len = plan.len, unit = static_cast<int>((plan.at - plan.base) / plan.n);
    const uint32_t unit_at = plan.base + unit * plan.n, end = min(unit_at + plan.n, plan.stop);
    const int off = max(0, static_cast<int>(plan.at - unit_at) - kUnitSteps), count = static_cast<int>(end - unit_at) - kUnitSteps - off;
    const int tile = unit % a.row_tiles, head = unit / a.row_tiles, rows = min(kRows, a.tq * ratio - tile * kRows);
    // the query rows are on their way first, in their own type
    constexpr int kPer = D / 32, kRowsWarp = kRows / kWarps;
    using Raw = std::conditional_t<F32, float, uint16_t>;
    Raw q[kRowsWarp][kPer];
#pragma unroll
    for (int j = 0; j < kRowsWarp; ++j) {
      const int r = warp + j * kWarps, rr = tile * kRows + r;
      const Raw* from = static_cast<const Raw*>(a.q) + seq * a.q_bs + (rr / ratio) * a.q_ts + (head * ratio + rr % ratio) * a.q_hs + lane;
#pragma unroll
      for (int i = 0; i < kPer; ++i) q[j][i] = r < rows ? __ldg(from + 32 * i) : Raw(0);  // channel 32 i + lane
    }
    __syncthreads();
    if (tid == kWarps * 32 - 1) {
      // the cuts inside the unit, and the block that its first part lies with: the one after the last cut before them
      const uint32_t total = plan.total, blocks = blocks_for(total), per = total / blocks, more = total - per * blocks;
      auto cuts_to = [&](uint32_t step) {  // how many cuts lie at or before `step`
        const uint32_t longer = more * (per + 1);
        return step < longer ? step / (per + 1) + 1 : more + (step - longer) / per + 1;
      };
      const uint32_t before = min(cuts_to(unit_at + kUnitSteps + kMinSteps - 1), blocks);
      plan.owner = static_cast<int>(before) - 1;
      plan.parts = plan.n >= kUnitSteps + 2 * kMinSteps ? 1 + static_cast<int>(min(cuts_to(unit_at + plan.n - kMinSteps), blocks) - before) : 1;
      plan.unit_seq = seq;
      plan.head = head;
      plan.tile = tile;
      plan.begins = off == 0;
      plan.at = end;
      if (end == plan.base + static_cast<uint32_t>(plan.n) * units && end < plan.stop) {
        plan.base = end;
        if (++plan.seq < a.b)
          plan.len = valid_length(c, a, plan.seq), plan.n = steps_of(plan.len);
        else
          plan.stop = end;
      }
    }
    // the last row of the tile sees the most tokens
    const int seen = max(0, len - a.tq + (tile * kRows + rows - 1) / ratio + 1);
    const int begin = off * kStepTokens, until = min(seen, begin + count * kStepTokens);
    const int32_t* pages = a.table + seq * a.table_stride;

    // ring: the first tiles are on their way before the query is looked at
    const uint32_t ring = shared_address(smem) + warp * (kStages * Shape::kStage);
    const int tiles = max(0, (until - begin + kTile - 1) / kTile);
    const int mine = tiles > warp ? (tiles - warp + kWarps - 1) / kWarps : 0;
    // this lane's token of the warp's tile i, or the tile's first where its tokens lie in one page: first + i * step
    const bool paged = c.page_size % kTile == 0;
    const int first = begin + warp * kTile + (paged ? 0 : lane);
    constexpr int kStep = kWarps * kTile;
    uint32_t held[kStages];  // which tokens of the tiles on their way are there
    uint32_t row = token_row(c, a, pages, head, first, until);
    auto load = [&](int i, uint32_t stage, bool ok) {  // tile i, whose row was looked up; the tokens that are there
      if (paged) {
        const int n = row == ~0u ? 0 : min(kTile, until - first - i * kStep);
        if (ok) load_tile_page<D, G>(c, stage, row, n, lane);
        return n >= kTile ? ~0u : (1u << max(0, n)) - 1;
      }
      const uint32_t there = __ballot_sync(~0u, row != ~0u);
      if (ok) load_tile<D, G>(c, stage, row, lane);
      return there;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      held[i] = load(i, ring + i * Shape::kStage, i < mine);
      copy_commit();
      row = token_row(c, a, pages, head, first + (i + 1) * kStep, until);
    }

    // query rows: scaled to fp16, laid out as operand B
#pragma unroll
    for (int j = 0; j < kRowsWarp; ++j) {
      const int r = warp + j * kWarps;
      float v[kPer], top = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if constexpr (F32)
          v[i] = q[j][i];
        else
          v[i] = a.ftype == B200Q_F16 ? __half2float(__ushort_as_half(q[j][i])) : __uint_as_float(static_cast<uint32_t>(q[j][i]) << 16);
        top = fmaxf(top, fabsf(v[i]));
      }
      const Power power = power_for(warp_max(top));
      if (lane == 0) {
        row_f[r] = power.down * a.scale * 1.4426950408889634f;
        row_limit[r] = len - a.tq + (tile * kRows + min(r, rows - 1)) / ratio + 1;
      }
      // lane: channel p = lane % 8 of the 8 that thread lane / 8 of a quad holds; pairs are (0,4) (1,5) (2,6) (3,7)
      const int p = lane % 8, holder = (r % 8) * 4 + lane / 8;
      __half* to = reinterpret_cast<__half*>(query);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float x = v[i] * power.up;
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
          const __half hv = __float2half_rn(x);
          const float back = __half2float(hv);
          x -= back;
          to[(((i * kTerms + term) * NT + r / 8) * 32 + holder) * 8 + (p % 4) * 2 + p / 4] =
              p % 2 ? __float2half_rn(back * 0.0625f) : hv;
        }
      }
    }
    __syncthreads();

    // this lane's columns: rows 2t, 2t + 1 of each 8
    float2 l[NT];
    float m[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n] = both(0.0f);
    }
    const int all_see = len - a.tq + tile * kRows / ratio + 1;  // tokens that every row of the tile sees
    float o[D / 16][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;

    int slot = 0, fill = kStages - 1;
    for (int it = 0; it < mine; ++it) {
      copy_wait<kStages - 2>();
      __syncwarp();
      held[kStages - 1] = load(it + kStages - 1, ring + fill * Shape::kStage, it + kStages - 1 < mine);
      copy_commit();
      row = token_row(c, a, pages, head, first + (it + kStages) * kStep, until);
      const uint8_t* stage = smem + warp * (kStages * Shape::kStage) + slot * Shape::kStage;
      const uint8_t* kc = stage;
      const uint8_t* vc = stage + Shape::kCodes;
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(stage + 2 * Shape::kCodes);
      const uint32_t* vp = kp + kTile * kGroups;
      const uint32_t here = held[0];
      const int base = begin + (it * kWarps + warp) * kTile;
      const bool whole = here == ~0u && base + kTile <= all_see;

      // lane l unpacks token l's scales and zero points for the lanes that use them: [group][token] (key scale, key zero
      // point z as a pair of the fp16 1024 + z), then value scales over kLag, then value zero points z as the bf16 128 + z
      float2* const k_prep = reinterpret_cast<float2*>(prepared);
      float* const v_prep = reinterpret_cast<float*>(prepared + kTile * kGroups * 8);
      uint16_t* const z_prep = reinterpret_cast<uint16_t*>(prepared + kTile * kGroups * 12);
      bool unbounded = false;
      {
        const bool there = here >> lane & 1;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          const uint32_t p = kp[lane * kGroups + k], q = there ? vp[lane * kGroups + k] : 0u;  // places that hold nothing hold any bits
          k_prep[k * kTile + lane] = make_float2(param_scale(p), __uint_as_float((p >> 16 & 15u) * 0x00010001u | kMagic));
          z_prep[k * kTile + lane] = static_cast<uint16_t>(q >> 16 & 15u | 0x4300u);
          const float vs = param_scale(q);
          unbounded |= !(fabsf(vs) < INFINITY);
          v_prep[k * kTile + lane] = vs * (1.0f / kLag);
        }
      }
      unbounded = __any_sync(~0u, unbounded);
      __syncwarp();

      // scores
      float2 s[2][NT][2];  // [tokens g, g + 8], rows 2t and 2t + 1
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        float part[2][NT][4];
#pragma unroll
        for (int i = k * (G / 32); i < (k + 1) * (G / 32); ++i) {
          uint4 b[kTerms][NT];
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int n = 0; n < NT; ++n) b[term][n] = query[((i * kTerms + term) * NT + n) * 32 + lane];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            uint32_t c[2][4];  // pairs (0,4) (1,5) (2,6) (3,7) of tokens g and g + 8
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t w = *reinterpret_cast<const uint32_t*>(kc + (mt * 16 + u * 8 + g) * kPitch + 16 * i + 4 * t);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t mask = j % 2 ? 0x00F000F0u : 0x000F000Fu;
                const uint32_t z = __float_as_uint(k_prep[k * kTile + mt * 16 + u * 8 + g].y);
                c[u][j] = sub_f16x2(and_or(w >> (j / 2 * 8), mask, kMagic), j % 2 ? and_or(z << 4, 0x00F000F0u, kMagic) : z);
              }
            }
#pragma unroll
            for (int term = 0; term < kTerms; ++term)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (i == k * (G / 32) && term == 0)
                  mma_f16_first(part[mt][n], c[0][0], c[1][0], c[0][1], c[1][1], b[term][n].x, b[term][n].y);
                else
                  mma_f16(part[mt][n], c[0][0], c[1][0], c[0][1], c[1][1], b[term][n].x, b[term][n].y);
                mma_f16(part[mt][n], c[0][2], c[1][2], c[0][3], c[1][3], b[term][n].z, b[term][n].w);
              }
          }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float2 ks = both(k_prep[k * kTile + mt * 16 + u * 8 + g].x);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const float* at = part[mt][n] + 2 * u;
              const float2 v = make_float2(at[0], at[1]);
              s[mt][n][u] = k == 0 ? mul2(ks, v) : fma2(ks, v, s[mt][n][u]);
            }
          }
      }

      // weights
      bool raise = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float2& x = s[mt][n][u];
            x = mul2(x, *reinterpret_cast<const float2*>(row_f + n * 8 + 2 * t));
            if (!whole) {
              const int tok = mt * 16 + u * 8 + g;
              const int2 limit = *reinterpret_cast<const int2*>(row_limit + n * 8 + 2 * t);
              if (!(here >> tok & 1) || base + tok >= limit.x) x.x = -INFINITY;
              if (!(here >> tok & 1) || base + tok >= limit.y) x.y = -INFINITY;
            }
          }
        top[n][0] = fmaxf(fmaxf(s[0][n][0].x, s[0][n][1].x), fmaxf(s[1][n][0].x, s[1][n][1].x));
        top[n][1] = fmaxf(fmaxf(s[0][n][0].y, s[0][n][1].y), fmaxf(s[1][n][0].y, s[1][n][1].y));
        raise |= top[n][0] > m[n][0] + kLagLog || top[n][1] > m[n][1] + kLagLog;
      }
      if (__any_sync(~0u, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(~0u, top[n][e], x));
            const float now = fmaxf(m[n][e], top[n][e]);
            const float keep = now == -INFINITY ? 1.0f : exp2_approx(m[n][e] - now);
            m[n][e] = now;
            (e ? l[n].y : l[n].x) *= keep;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) o[j][n][e] *= keep, o[j][n][2 + e] *= keep;
          }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 ref = make_float2(m[n][0] == -INFINITY ? 0.0f : -m[n][0], m[n][1] == -INFINITY ? 0.0f : -m[n][1]);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float2& x = s[mt][n][u];
            x = add2(x, ref);
            x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
            l[n] = add2(l[n], x);
          }
      }

      // values; a tile's sums are made apart and added with rounding
      constexpr int kPTerms = F32 ? 3 : 2;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        float part[G / 16][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          // operand B: P of this group, as (row g, tokens 2t, 2t + 1) of each 8 tokens
          uint32_t b[kPTerms][NT][2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float2 scale = both(v_prep[k * kTile + mt * 16 + u * 8 + g]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float2 x = mul2(s[mt][n][u], scale);
              if (unbounded) {  // an infinite or NaN scale is for the rows that see its token
                if (s[mt][n][u].x == 0.0f) x.x = 0.0f;
                if (s[mt][n][u].y == 0.0f) x.y = 0.0f;
              }
#pragma unroll
              for (int term = 0; term < kPTerms; ++term) {
                const uint32_t v = pack_bf16(x.x, x.y);
                if (term + 1 < kPTerms) {
                  x = fma2(make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)), both(-1.0f), x);
                  if (unbounded) {  // what is left of an infinity
                    if (x.x != x.x) x.x = 0.0f;
                    if (x.y != x.y) x.y = 0.0f;
                  }
                }
                b[term][n][u] = transpose_8x8(v);
              }
            }
          }
          // operand A: tokens 2t, 2t + 1 (u = 0) and 2t + 8, 2t + 9 (u = 1) of this lane's G / 8 channels, the lower
          // half of them as row g of the group's G / 16 products, the upper as row g + 8
          uint32_t lower[2], upper[2], zero[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int tok = mt * 16 + u * 8 + 2 * t;
            const uint8_t* at = vc + tok * kPitch + k * (G / 2) + g * (G / 16);
            if constexpr (G == 64) {
              const uint32_t x = *reinterpret_cast<const uint32_t*>(at), y = *reinterpret_cast<const uint32_t*>(at + kPitch);
              lower[u] = __byte_perm(x, y, 0x5410);
              upper[u] = __byte_perm(x, y, 0x7632);
            } else {
              const uint32_t x = *reinterpret_cast<const uint16_t*>(at), y = *reinterpret_cast<const uint16_t*>(at + kPitch);
              lower[u] = x | y << 16;
              upper[u] = lower[u] >> 8;
            }
            zero[u] = *reinterpret_cast<const uint32_t*>(z_prep + k * kTile + tok);
          }
#pragma unroll
          for (int j = 0; j < G / 16; ++j) {
            constexpr uint32_t kMask = 0x000F000Fu, kMagic128 = 0x43004300u;  // two bf16 128: with a code in the low bits 128 + code
            const uint32_t a0 = sub_bf16x2(and_or(lower[0] >> 4 * j, kMask, kMagic128), zero[0]);
            const uint32_t a1 = sub_bf16x2(and_or(upper[0] >> 4 * j, kMask, kMagic128), zero[0]);
            const uint32_t a2 = sub_bf16x2(and_or(lower[1] >> 4 * j, kMask, kMagic128), zero[1]);
            const uint32_t a3 = sub_bf16x2(and_or(upper[1] >> 4 * j, kMask, kMagic128), zero[1]);
#pragma unroll
            for (int term = 0; term < kPTerms; ++term)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (mt == 0 && term == 0)
                  mma_bf16_first(part[j][n], a0, a1, a2, a3, b[term][n][0], b[term][n][1]);
                else
                  mma_bf16(part[j][n], a0, a1, a2, a3, b[term][n][0], b[term][n][1]);
              }
          }
        }
#pragma unroll
        for (int j = 0; j < G / 16; ++j)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k * (G / 16) + j][n][e] += part[j][n][e];
      }
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) held[i] = held[i + 1];
      slot = slot + 1 == kStages ? 0 : slot + 1;
      fill = fill + 1 == kStages ? 0 : fill + 1;
    }

    // join the warps: maxima and totals, then the sums through shared memory (the rings are done with)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float all = e ? l[n].y : l[n].x;
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) all += __shfl_xor_sync(~0u, all, x);
        if (g == 0) {
          float* ml = row_ml + (warp * kRows + n * 8 + 2 * t + e) * 2;
          ml[0] = m[n][e];
          ml[1] = all;
        }
      }
    copy_wait<0>();
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(smem);  // [kWarps][kRows][D + 4]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * t + e;
        float now = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) now = fmaxf(now, row_ml[(w * kRows + r) * 2]);
        const float keep = m[n][e] == -INFINITY ? 0.0f : exp2_approx(m[n][e] - now);
        float* to = sums + (warp * kRows + r) * (D + 4);
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float v[G / 16];
#pragma unroll
            for (int j = 0; j < G / 16; ++j) v[j] = o[k * (G / 16) + j][n][2 * u + e] * kLag * keep;
            float* p = to + k * G + g * (G / 8) + u * (G / 16);
            if constexpr (G == 64)
              *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            else
              *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
          }
      }
    __syncthreads();

    const int parts = plan.parts, unit_tile = plan.tile, unit_rows = min(kRows, a.tq * ratio - unit_tile * kRows);
    // rows' places in the output, and their maxima and totals
    constexpr int kThreads = kWarps * 32;
    if (tid < kRows) {
      const int rr = unit_tile * kRows + min(tid, unit_rows - 1);
      row_out[tid] = (static_cast<int64_t>(plan.unit_seq) * a.tq + rr / ratio) * a.hq + plan.head * ratio + rr % ratio;
      float now = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) now = fmaxf(now, row_ml[(w * kRows + tid) * 2]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float mw = row_ml[(w * kRows + tid) * 2];
        sum += row_ml[(w * kRows + tid) * 2 + 1] * (mw == -INFINITY ? 1.0f : exp2_approx(mw - now));  // none: 0, or NaN from scores that are
      }
      row_all[tid] = make_float2(now, sum);
    }
    __syncthreads();

    // the block's rows: straight to the output, or to the scratch for the unit's last block to join
    auto finish = [&](int r, int d, float4 v) {
      const float2 ml = row_all[r];
      const float over = ml.y > 0.0f ? 1.0f / ml.y : 0.0f;  // no tokens: 0
      const bool sound = ml.y >= 0.0f;                       // else a NaN to hand on
      v = make_float4(v.x * over, v.y * over, v.z * over, v.w * over);
      if (!sound) v = make_float4(ml.y, ml.y, ml.y, ml.y);
      store_four(a.ftype, a.out, row_out[r] * D + d, v);
      if (d == 0 && a.lse) a.lse[row_out[r]] = ml.y > 0.0f ? (ml.x + log2f(ml.y)) * 0.69314718055994531f : sound ? -INFINITY : ml.y;
    };
    const int mine_at = (2 * blockIdx.x + plan.begins) * kRows;
    for (int i = tid; i < unit_rows * D / 4; i += kThreads) {
      const int r = i / (D / 4), d = i % (D / 4) * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(sums + (w * kRows + r) * (D + 4) + d);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
      if (parts == 1) {
        finish(r, d, v);
      } else {
        __stcg(reinterpret_cast<float4*>(a.partial + static_cast<size_t>(mine_at + r) * D + d), v);
        if (d == 0) __stcg(reinterpret_cast<float2*>(a.partial_ml) + mine_at + r, row_all[r]);
      }
    }
    if (parts > 1) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        arrived = atomicAdd(a.counters + plan.owner, 1u);
        if (arrived + 1 == static_cast<unsigned>(parts)) a.counters[plan.owner] = 0;  // for the next launch
      }
      __syncthreads();
      if (arrived + 1 == static_cast<unsigned>(parts)) {
        __threadfence();
        const int owner = plan.owner;
        // part j lies with block owner + j: the first as the unit begun there, the others as the one begun before
        auto part_row = [&](int j, int r) { return static_cast<size_t>(2 * (owner + j) + (j == 0)) * kRows + r; };
        auto part_four = [&](int j, int r, int d) { return __ldcg(reinterpret_cast<const float4*>(a.partial + part_row(j, r) * D + d)); };
        constexpr int kFirst = 8;  // parts of the thread's first four that are read along with the maxima
        float4 first[kFirst];
#pragma unroll
        for (int j = 0; j < kFirst; ++j)
          if (j < parts && tid < unit_rows * D / 4) first[j] = part_four(j, tid / (D / 4), tid % (D / 4) * 4);
        // what each part counts for, [row][part], and the rows' totals
        float* const share = reinterpret_cast<float*>(smem);
        for (int r = warp; r < unit_rows; r += kWarps) {
          const float2* ml = reinterpret_cast<const float2*>(a.partial_ml);
          const float2 mine = lane < parts ? __ldcg(ml + part_row(lane, r)) : make_float2(-INFINITY, 0.0f);
          float now = mine.x, sum = 0.0f;
          for (int j = lane + 32; j < parts; j += 32) now = fmaxf(now, __ldcg(ml + part_row(j, r)).x);
          now = warp_max(now);
          for (int j = lane; j < parts; j += 32) {
            const float2 x = j == lane ? mine : __ldcg(ml + part_row(j, r));
            const float keep = x.x == -INFINITY ? 0.0f : exp2_approx(x.x - now);
            share[r * parts + j] = keep;
            sum += keep * x.y;
          }
          sum = warp_sum(sum);
          if (lane == 0) row_all[r] = make_float2(now, sum);
        }
        __syncthreads();
        for (int i = tid; i < unit_rows * D / 4; i += kThreads) {
          const int r = i / (D / 4), d = i % (D / 4) * 4;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          auto add = [&](int j, float4 x) {
            const float keep = share[r * parts + j];
            v.x = fmaf(keep, x.x, v.x), v.y = fmaf(keep, x.y, v.y), v.z = fmaf(keep, x.z, v.z), v.w = fmaf(keep, x.w, v.w);
          };
          int j0 = 0;
          if (i == tid) {
#pragma unroll
            for (int j = 0; j < kFirst; ++j)
              if (j < parts) add(j, first[j]);
            j0 = kFirst;
          }
#pragma unroll 8
          for (int j = j0; j < parts; ++j) add(j, part_four(j, r, d));
          finish(r, d, v);
        }
      }
    }
    if (plan.at >= plan.stop) return;
    __syncthreads();  // shared memory is free for the next unit
  }
}

}  // namespace b200q
