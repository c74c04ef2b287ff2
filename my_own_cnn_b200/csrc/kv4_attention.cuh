// Attention of a few query rows over the 4-bit cache, on tensor cores.
//
// For one sequence and cache head with rows r (new tokens x query heads that share the head), tokens t:
//   S[t][r] = sum_g ks[t,g] (sum_{d in g} kc[t,d] q[r,d]  -  kz[t,g] sum_{d in g} q[r,d])
//   O[d][r] = sum_t vc[t,d] P[t,r]  -  sum_t vz[t,g] P[t,r],   P[t,r] = vs[t,g] exp2(f[r] S[t][r] - m[r])
// Both products take the codes as the 16-row operand A of m16n8k16 (tokens x channels, then channels x tokens)
// and the rows as its 8 columns, so 8 rows cost one instruction per 256 codes.
//   Keys: a nibble in the low bits of an fp16 is the subnormal code * 2^-24, exactly, and one place higher
//   code * 2^-20: a word of 8 codes becomes four operands by masking, and every second query value is divided
//   by 16 instead.  Query rows are scaled by a power of two to a maximum in [2^14, 2^15), so that they fit
//   fp16 whatever their type; fp32 rows are split into two fp16 terms (22 bits).
//   Values: the same subnormals, channels as rows: a channel whose nibble lies one place higher has its sum divided by
//   16 at the end, the zero points go through the same instruction as a 16-row operand of their own and are
//   subtracted last.  P is fp16 (11 bits; two terms, 22 bits, in fp32 calls) times a power of two that follows the largest
//   vs that the warp has met, so that full precision holds for tokens whose vs is up to 2^20 below that.
//   P leaves the first product as (token, row) and must enter the second as (row, token): movmatrix.
// The maximum m[r] is a running reference, raised (and the sums rescaled) only when a score passes it by more than
// 2^8: a warp-wide maximum is taken a few times per sequence, not per tile.
//
// Work: a unit is (sequence, cache head, tile of rows), in steps of kWarps tiles of kTile tokens.  All units' steps lie
// end to end, and block i takes steps [i * per, (i + 1) * per) of them, whatever the lengths (which only the device knows):
// every block has the same work, and none waits for a last wave.  The parts of a unit that several blocks share go to
// the workspace, and the block that finishes last joins them in order.
//
// What bounds it: bytes, D / 2 + 4 D / G for each of K and V per token and head.  Each warp owns a ring of kStages tiles of
// kTile tokens that it fills with 16-byte asynchronous copies and empties on its own: no block-wide barrier until
// the end.  A row of codes is padded by 16 bytes in shared memory: then lanes (g, t) reading 4 bytes at g rows down,
// and 2t rows down, both touch 32 banks once.
#pragma once
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

constexpr int kMinSteps = 2;  // steps of a block at least
constexpr int kUnitSteps = 3; // what a unit costs besides its steps (its queries, its first tiles' way, its join), in steps

constexpr int kTile = 32;    // tokens of a warp's step
constexpr int kWarps = 4;    // a block's warps take tiles in turn
constexpr int kStages = 3;
constexpr int kStepTokens = kWarps * kTile;

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
  static constexpr int kRowsMl = kWarps * 8 * NT * 2 * 4;
  static constexpr int kSmem = kBody + kQuery + kRowsMl + (8 * NT * (kGroups + 1)) * 4;
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

template <typename T>
__device__ __forceinline__ float load_as_f32(const void* p, long long i) {
  return to_f32(static_cast<const T*>(p)[i]);
}
__device__ __forceinline__ float load_any(int ftype, const void* p, long long i) {
  return ftype == B200Q_F32   ? load_as_f32<float>(p, i)
         : ftype == B200Q_F16 ? load_as_f32<__half>(p, i)
                              : load_as_f32<__nv_bfloat16>(p, i);
}
__device__ __forceinline__ void store_any(int ftype, void* p, long long i, float v) {
  if (ftype == B200Q_F32)
    static_cast<float*>(p)[i] = v;
  else if (ftype == B200Q_F16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
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

template <int D, int G, int NT, bool F32>
__global__ void __launch_bounds__(kWarps * 32, D <= 128 && NT == 1 ? 3 : 1) kv4_attention_kernel(Cache c, AttnArgs a) {
  using Shape = AttnShape<D, G, NT, F32>;
  constexpr int kGroups = Shape::kGroups, kPitch = Shape::kPitch, kRows = 8 * NT, kTerms = Shape::kTerms;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ unsigned arrived;
  wait_for_previous();
  uint4* const query = reinterpret_cast<uint4*>(smem + Shape::kBody);
  float* const row_ml = reinterpret_cast<float*>(smem + Shape::kBody + Shape::kQuery);
  float* const row_sum = row_ml + kWarps * kRows * 2;  // [kGroups][kRows] sums of the scaled query, times 2^-24
  float* const row_f = row_sum + kRows * kGroups;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, t = lane % 4;

  const int units = c.heads * a.row_tiles, ratio = a.hq / c.heads;
  auto steps_of = [&](int i) { return kUnitSteps + max(1, (valid_length(c, a, i) + kStepTokens - 1) / kStepTokens); };
  long long total = 0;
  for (int i = lane; i < a.b; i += 32) total += steps_of(i);
#pragma unroll
  for (int x = 16; x; x >>= 1) total += __shfl_xor_sync(~0u, total, x);
  total *= units;
  const long long per = max(static_cast<long long>(kMinSteps), (total + gridDim.x - 1) / gridDim.x);
  long long at = blockIdx.x * per;  // the block's next step
  const long long stop = min(total, at + per);
  if (at >= stop) return;
  int seq = 0;
  long long base = 0;  // first step of the sequence
  for (;; seq += 32) {
    long long sum = seq + lane < a.b ? static_cast<long long>(steps_of(seq + lane)) * units : 0;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const long long v = __shfl_up_sync(~0u, sum, x);
      if (lane >= x) sum += v;
    }
    const unsigned past = __ballot_sync(~0u, base + sum > at);
    const int first = past ? __ffs(past) - 1 : 31;
    const long long before = __shfl_sync(~0u, sum, past ? first - 1 : 31);  // lane -1 is lane 31, and not used
    if (!past || first > 0) base += before;
    if (past) {
      seq += first;
      break;
    }
  }

 for (; at < stop;) {
  // steps [off, off + count) of the unit; its first kUnitSteps steps stand for what it costs besides
  const int n = steps_of(seq), len = valid_length(c, a, seq);
  const int unit = static_cast<int>((at - base) / n);
  const long long unit_at = base + static_cast<long long>(unit) * n;
  const long long end = min(unit_at + n, stop);
  const int off = max(0, static_cast<int>(at - unit_at) - kUnitSteps), count = static_cast<int>(end - unit_at) - kUnitSteps - off;
  at = end;
  if (count <= 0) break;  // all of it lies with the next block
  const int tile = unit % a.row_tiles, head = unit / a.row_tiles, rows = min(kRows, a.tq * ratio - tile * kRows);
  const long long owner = (unit_at + kUnitSteps) / per;  // the block that its first step lies with
  const int parts = static_cast<int>((unit_at + n - 1) / per - owner) + 1;
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

  // query rows: scaled to fp16, laid out as operand B; a warp takes rows in turn
  for (int r = warp; r < kRows; r += kWarps) {
    constexpr int kPer = D / 32;
    const int rr = tile * kRows + r;
    float v[kPer];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {  // channel 32 i + lane
      v[i] = r < rows ? load_any(a.ftype, a.q, seq * a.q_bs + (rr / ratio) * a.q_ts + (head * ratio + rr % ratio) * a.q_hs + 32 * i + lane)
                      : 0.0f;
      top = fmaxf(top, fabsf(v[i]));
    }
    const Power power = power_for(warp_max(top));
    if (lane == 0) row_f[r] = power.down * a.scale * 1.4426950408889634f * 16777216.0f;
    // lane: channel p = lane % 8 of the 8 that thread lane / 8 of a quad holds; pairs are (0,4) (1,5) (2,6) (3,7)
    const int p = lane % 8, holder = (r % 8) * 4 + lane / 8;
    __half* to = reinterpret_cast<__half*>(query);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float x = v[i] * power.up;
#pragma unroll
      for (int term = 0; term < kTerms; ++term) {
        const __half hv = __float2half_rn(x);
        const float back = __half2float(hv);
        sum += back;
        x -= back;
        to[(((i * kTerms + term) * NT + r / 8) * 32 + holder) * 8 + (p % 4) * 2 + p / 4] =
            p % 2 ? __float2half_rn(back * 0.0625f) : hv;
      }
      if ((i + 1) % (G / 32) == 0) {
        sum = warp_sum(sum);
        if (lane == 0) row_sum[(i / (G / 32)) * kRows + r] = sum * (1.0f / 16777216.0f);
        sum = 0.0f;
      }
    }
  }
  __syncthreads();

  // this lane's columns: rows 2t, 2t + 1 of each 8
  float2 f[NT], qsum[NT][kGroups], l[NT];
  float m[NT][2];
  int limit[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = n * 8 + 2 * t + e;
      (e ? f[n].y : f[n].x) = row_f[r];
#pragma unroll
      for (int k = 0; k < kGroups; ++k) (e ? qsum[n][k].y : qsum[n][k].x) = row_sum[k * kRows + r];
      m[n][e] = -INFINITY;
      l[n] = both(0.0f);
      limit[n][e] = len - a.tq + (tile * kRows + min(r, rows - 1)) / ratio + 1;
    }
  const int all_see = len - a.tq + tile * kRows / ratio + 1;  // tokens that every row of the tile sees
  float o[D / 16][NT][4], z[kGroups][NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) z[j][n][0] = z[j][n][1] = z[j][n][2] = z[j][n][3] = 0.0f;
  }

  // P's power of two: 2^(127 - v_exp), for a largest vs of 2^(v_exp - 127)
  int v_exp = 127;
  float v_factor = 1.0f, v_limit = -1.0f;
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
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(kc + (mt * 16 + g) * kPitch + 16 * i + 4 * t);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(kc + (mt * 16 + g + 8) * kPitch + 16 * i + 4 * t);
          const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (i == k * (G / 32) && term == 0)
                mma_f16_first(part[mt][n], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u,
                              b[term][n].x, b[term][n].y);
              else
                mma_f16(part[mt][n], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u,
                        b[term][n].x, b[term][n].y);
              mma_f16(part[mt][n], v0 & 0x000F000Fu, v1 & 0x000F000Fu, v0 & 0x00F000F0u, v1 & 0x00F000F0u,
                      b[term][n].z, b[term][n].w);
            }
        }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t p = kp[(mt * 16 + u * 8 + g) * kGroups + k];
          const float2 ks = both(param_scale(p)), kz = both(-zero_point(p));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float* at = part[mt][n] + 2 * u;
            const float2 v = fma2(kz, qsum[n][k], make_float2(at[0], at[1]));
            s[mt][n][u] = k == 0 ? mul2(ks, v) : fma2(ks, v, s[mt][n][u]);
          }
        }
    }

    // this lane's scales of the values, tokens mt * 16 + u * 8 + g
    float vs[2][2][kGroups], v_top = 0.0f;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
          const int tok = mt * 16 + u * 8 + g;
          vs[mt][u][k] = param_scale(vp[tok * kGroups + k]);
          if (!whole && !(here >> tok & 1)) vs[mt][u][k] = 0.0f;
          v_top = fmaxf(v_top, vs[mt][u][k]);
        }

    // weights
    bool raise = v_top > v_limit;
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float2& x = s[mt][n][u];
          x = mul2(x, f[n]);
          if (!whole) {
            const int tok = mt * 16 + u * 8 + g;
            if (!(here >> tok & 1) || base + tok >= limit[n][0]) x.x = -INFINITY;
            if (!(here >> tok & 1) || base + tok >= limit[n][1]) x.y = -INFINITY;
          }
        }
      top[n][0] = fmaxf(fmaxf(s[0][n][0].x, s[0][n][1].x), fmaxf(s[1][n][0].x, s[1][n][1].x));
      top[n][1] = fmaxf(fmaxf(s[0][n][0].y, s[0][n][1].y), fmaxf(s[1][n][0].y, s[1][n][1].y));
      raise |= top[n][0] > m[n][0] + 8.0f || top[n][1] > m[n][1] + 8.0f;
    }
    if (__any_sync(~0u, raise)) {
      float v_keep = 1.0f;
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) v_top = fmaxf(v_top, __shfl_xor_sync(~0u, v_top, x));
      if (v_top > v_limit) {
        const int now = max(1, min(247, static_cast<int>(__float_as_uint(v_top) >> 23)));
        v_keep = now - v_exp < 127 ? __uint_as_float(static_cast<uint32_t>(127 + v_exp - now) << 23) : 0.0f;
        if (v_limit < 0.0f) v_keep = 1.0f;  // no sums yet
        v_exp = now;
        v_factor = __uint_as_float(static_cast<uint32_t>(254 - now) << 23);
        v_limit = __uint_as_float(static_cast<uint32_t>(now + 6) << 23);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[n][e] = fmaxf(top[n][e], __shfl_xor_sync(~0u, top[n][e], x));
          const float now = fmaxf(m[n][e], top[n][e]);
          float keep = now == -INFINITY ? 1.0f : exp2_approx(m[n][e] - now);
          m[n][e] = now;
          (e ? l[n].y : l[n].x) *= keep;
          keep *= v_keep;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) o[j][n][e] *= keep, o[j][n][2 + e] *= keep;
#pragma unroll
          for (int j = 0; j < kGroups; ++j) z[j][n][e] *= keep, z[j][n][2 + e] *= keep;
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

    // values
    constexpr int kPTerms = F32 ? 2 : 1;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        // operand B: P of this group, as (row g, tokens 2t, 2t + 1) of each 8 tokens
        uint32_t b[kPTerms][NT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float2 scale = both(vs[mt][u][k] * v_factor);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float2 x = mul2(s[mt][n][u], scale);
#pragma unroll
            for (int term = 0; term < kPTerms; ++term) {
              const uint32_t v = pack_f16(x.x, x.y);
              if (term + 1 < kPTerms) {
                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&v));
                x = make_float2(x.x - back.x, x.y - back.y);
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
          zero[u] = __byte_perm(vp[tok * kGroups + k], vp[(tok + 1) * kGroups + k], 0x7632);
          if (!whole) zero[u] &= 0x00FF00FFu;  // places that hold nothing hold any bits
        }
#pragma unroll
        for (int j = 0; j < G / 16; ++j) {
          const int down = j / 2 * 8;
          const uint32_t mask = j % 2 ? 0x00F000F0u : 0x000F000Fu;
          const uint32_t a0 = lower[0] >> down & mask, a1 = upper[0] >> down & mask;
          const uint32_t a2 = lower[1] >> down & mask, a3 = upper[1] >> down & mask;
#pragma unroll
          for (int term = 0; term < kPTerms; ++term)
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[k * (G / 16) + j][n], a0, a1, a2, a3, b[term][n][0], b[term][n][1]);
        }
#pragma unroll
        for (int term = 0; term < kPTerms; ++term)
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(z[k][n], zero[0], zero[0], zero[1], zero[1], b[term][n][0], b[term][n][1]);
      }
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
      const float value = __uint_as_float(static_cast<uint32_t>(v_exp) << 23);
      float* to = sums + (warp * kRows + r) * (D + 4);
#pragma unroll
      for (int k = 0; k < kGroups; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float v[G / 16];
#pragma unroll
          for (int j = 0; j < G / 16; ++j) v[j] = fmaf(o[k * (G / 16) + j][n][2 * u + e], j % 2 ? 0.0625f : 1.0f, -z[k][n][2 * u + e]) * 16777216.0f * value * keep;
          float* p = to + k * G + g * (G / 8) + u * (G / 16);
          if constexpr (G == 64)
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
          else
            *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
        }
    }
  __syncthreads();

  // the block's rows: straight to the output, or to the workspace for the unit's last block to join
  auto out_index = [&](int r) {
    const int rr = tile * kRows + r;
    return (static_cast<long long>(seq) * a.tq + rr / ratio) * a.hq + head * ratio + rr % ratio;
  };
  auto finish = [&](int r, int d, float v, float sum, float now) {
    store_any(a.ftype, a.out, out_index(r) * D + d, sum > 0.0f ? v / sum : sum == 0.0f ? 0.0f : sum);
    if (d == 0 && a.lse) a.lse[out_index(r)] = sum > 0.0f ? (now + log2f(sum)) * 0.69314718055994531f : sum == 0.0f ? -INFINITY : sum;
  };
  constexpr int kThreads = kWarps * 32;
  const int mine_at = (2 * blockIdx.x + (off == 0)) * kRows;
  for (int i = tid; i < rows * D; i += kThreads) {
    const int r = i / D, d = i % D;
    float now = -INFINITY, sum = 0.0f, v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) now = fmaxf(now, row_ml[(w * kRows + r) * 2]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = row_ml[(w * kRows + r) * 2];
      sum += mw == -INFINITY ? 0.0f : row_ml[(w * kRows + r) * 2 + 1] * exp2_approx(mw - now);
      v += sums[(w * kRows + r) * (D + 4) + d];
    }
    if (parts == 1) {
      finish(r, d, v, sum, now);
    } else {
      a.partial[static_cast<size_t>(mine_at + r) * D + d] = v;
      if (d == 0) {
        float* ml = a.partial_ml + static_cast<size_t>(mine_at + r) * 2;
        ml[0] = now;
        ml[1] = sum;
      }
    }
  }
  if (parts > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      arrived = atomicAdd(a.counters + owner, 1u);
      if (arrived + 1 == static_cast<unsigned>(parts)) a.counters[owner] = 0;  // for the next launch
    }
    __syncthreads();
    if (arrived + 1 == static_cast<unsigned>(parts)) {
      __threadfence();
      // part j lies with block owner + j: the first as the unit begun there, the others as the one begun before
      auto part_row = [&](int j, int r) { return static_cast<size_t>((2 * (owner + j) + (j == 0)) * kRows + r); };
      // what each part counts for, [row][part], and the rows' totals
      float* const share = reinterpret_cast<float*>(smem);
      for (int r = warp; r < rows; r += kWarps) {
        float now = -INFINITY, sum = 0.0f;
        for (int j = lane; j < parts; j += 32) now = fmaxf(now, __ldcg(a.partial_ml + part_row(j, r) * 2));
#pragma unroll
        for (int x = 16; x; x >>= 1) now = fmaxf(now, __shfl_xor_sync(~0u, now, x));
        for (int j = lane; j < parts; j += 32) {
          const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.partial_ml + part_row(j, r) * 2));
          const float keep = ml.x == -INFINITY ? 0.0f : exp2_approx(ml.x - now);
          share[r * parts + j] = keep;
          sum += keep * ml.y;
        }
        sum = warp_sum(sum);
        if (lane == 0) row_ml[2 * r] = now, row_ml[2 * r + 1] = sum;
      }
      __syncthreads();
      for (int i = tid; i < rows * D / 4; i += kThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int j = 0; j < parts; ++j) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(a.partial + part_row(j, r) * D + d));
          const float keep = share[r * parts + j];
          v.x = fmaf(keep, x.x, v.x), v.y = fmaf(keep, x.y, v.y), v.z = fmaf(keep, x.z, v.z), v.w = fmaf(keep, x.w, v.w);
        }
        const float now = row_ml[2 * r], sum = row_ml[2 * r + 1];
        finish(r, d, v.x, sum, now);
        finish(r, d + 1, v.y, sum, now);
        finish(r, d + 2, v.z, sum, now);
        finish(r, d + 3, v.w, sum, now);
      }
    }
  }
  __syncthreads();  // shared memory is free for the next unit
  if (at == base + static_cast<long long>(n) * units) base = at, ++seq;
 }
}

}  // namespace b200q
