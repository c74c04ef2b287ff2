// What the kernels of prompt attention share: arguments, the order of the work, rows that are done with care.
#pragma once
#include "host.h"
#include "lowbit.cuh"

namespace b200q {

struct PromptArgs {
  const void* q;
  long long q_ts, q_hs;
  const void* k;
  long long k_ts, k_hs;
  const void* v;
  long long v_ts, v_hs;
  const int32_t* starts;
  const int32_t* k_starts;
  void* out;   // [tq][hq][d]
  float* lse;  // [tq][hq], or null
  int b, tq, tk, hq, hk, d;
  Divisor ratio;   // hq / hk
  int row_scale;   // a tile holds tile.d whole tokens (1), or tile.d rows (token, head of the group; hq / hk)
  Divisor tile;
  long long most_units;  // key heads times tiles times parts, as many as there may be
  int parts;             // of each tile's keys; with more than one the sums meet in part_*, [parts][tq * hq]
  float4* part_heads;    // reference (of base 2; -inf: sees none here), sum of weights, the bits of the row's first key and of how many it sees
  float* part_sums;      // [..][d]
  unsigned* arrived;     // [tq * hq] parts that have been written: zero before and after
  float scale;
  int* err;
  long long limit;
};

constexpr float kLog2e = 1.4426950408889634f;

// A row's log-sum from its reference (base 2) and its sum.  With a score of +inf the sum is NaN.
__device__ __forceinline__ float log_sum(float top, float sum) {
  return top == INFINITY ? top : (top + log2f(sum)) * (1.0f / kLog2e);
}

// A sequence's rows; empty where its starts are not in order or pass the tensors.
struct Sequence {
  int q0, lq, k0, lk;
  bool bad;
  __device__ __forceinline__ int tiles(const PromptArgs& a) const {
    return static_cast<int>(a.tile.of(static_cast<uint32_t>(lq * a.row_scale + static_cast<int>(a.tile.d) - 1)));
  }
};
__device__ __forceinline__ Sequence sequence(const PromptArgs& a, int i) {
  Sequence s{};
  if (i >= a.b) return s;
  const int q0 = a.starts[i], q1 = a.starts[i + 1], k0 = a.k_starts[i], k1 = a.k_starts[i + 1];
  s.bad = q0 < 0 || q1 < q0 || q1 > a.tq || k0 < 0 || k1 < k0 || k1 > a.tk;
  if (!s.bad) s = {q0, q1 - q0, k0, k1 - k0, false};
  return s;
}

// Tile `tile` of a sequence.
struct PromptUnit {
  Sequence s;
  int tile;
  bool ok;
};
__device__ __forceinline__ int warp_total(int v) { return __reduce_add_sync(~0u, v); }
// The sum of the lanes up to this one.
__device__ __forceinline__ int warp_running(int v) {
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int x = __shfl_up_sync(~0u, v, o);
    if (static_cast<int>(threadIdx.x % 32) >= o) v += x;
  }
  return v;
}

// A sequence's units, the last `above(l)` of which have more than l steps of 128 keys.
constexpr int kUnitKeys = 128;
struct Units {
  int tiles, lq, shift, most;  // keys less queries; steps of the last unit
  __device__ __forceinline__ Units(const PromptArgs& a, const Sequence& s)
      : tiles(s.tiles(a)), lq(s.lq), shift(s.lk - s.lq), most(tiles ? (s.lk + kUnitKeys - 1) / kUnitKeys : 0) {}
  // all at l < 0; from the first tile whose end passes l steps on
  __device__ __forceinline__ int above(const PromptArgs& a, int l) const {
    if (l < 0) return tiles;
    if (l >= most) return 0;
    const int tokens = l * kUnitKeys - shift;  // that l steps reach
    if (tokens < 0) return tiles;
    return tiles - min(tiles, static_cast<int>(a.tile.of(static_cast<uint32_t>(min(tokens, lq) * a.row_scale))));
  }
};

// Steps [from, to) of `steps` that are part `part`'s.
__device__ __forceinline__ int2 part_steps(const PromptArgs& a, int steps, int part) {
  return make_int2(static_cast<int>(static_cast<long long>(steps) * part / a.parts),
                   static_cast<int>(static_cast<long long>(steps) * (part + 1) / a.parts));
}
// What a part says of a row; the join counts on all of them.  `saw`: the row sees some of its keys.  Where it does and their scores are
// all -inf the sum is zero and the reference any number; where not, it is -inf.
__device__ __forceinline__ void part_head(const PromptArgs& a, int part, long long row, bool saw, float ref, float sum, int k0, int seen) {
  const float from = !saw ? -INFINITY : sum == 0.0f ? 0.0f : ref;
  a.part_heads[part * static_cast<long long>(a.tq) * a.hq + row] = make_float4(from, sum, __int_as_float(k0), __int_as_float(seen));
  atomicAdd(a.arrived + row, 1u);
}

// Finds units, each call a later one than the last; a warp's work.  Of up to 32 sequences, one a lane, the units are in falling order of
// their steps, so that the longest start first and the short ones fill up the end (six sequences with earlier parts 80 us by tile
// number, 67 so); found by bisection over the units with more than l steps.  Of more sequences they are in the sequences'
// order, which a search from where the last one ended finds in one pass over all of them.
class Finder {
 public:
  __device__ __forceinline__ Finder(const PromptArgs& args, bool report) : a(args), lane(threadIdx.x % 32) {
    bool bad = false;
    if (a.b <= 32) {
      s = sequence(a, lane), bad = s.bad;
    } else if (report) {
      for (int i = lane; i < a.b; i += 32) bad |= sequence(a, i).bad;
    }
    if (report && bad) atomicCAS(a.err, 0, kDevErrBadStarts);
  }
  __device__ __forceinline__ PromptUnit operator()(int unit) { return a.b <= 32 ? by_length(unit) : by_sequence(unit); }

 private:
  __device__ __forceinline__ PromptUnit by_length(int unit) {
    const Units u(a, s);
    auto above = [&](int l) { return warp_total(u.above(a, l)); };
    if (unit >= above(-1)) return PromptUnit{};
    // above(lo) > unit >= above(hi) = longer: the unit has hi steps
    int lo = -1, hi = __reduce_max_sync(~0u, u.most), longer = 0;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2, n = above(mid);
      if (n > unit)
        lo = mid;
      else
        hi = mid, longer = n;
    }
    const int left = unit - longer;  // of the units with hi steps
    const int past = u.above(a, hi), n = u.above(a, lo) - past, upto = warp_running(n);
    const unsigned have = __ballot_sync(~0u, upto > left);
    return have ? at(s, u.tiles - past - 1 - (left - (upto - n)), __ffs(have) - 1) : PromptUnit{};
  }
  __device__ __forceinline__ PromptUnit by_sequence(int unit) {
    constexpr int kEach = 4;  // sequences a lane: their loads are one wait
    for (; first < a.b; first += 32 * kEach) {
      Sequence q[kEach];
      int n = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) q[i] = sequence(a, first + kEach * lane + i);
#pragma unroll
      for (int i = 0; i < kEach; ++i) n += q[i].tiles(a);
      const int upto = warp_running(n), left = unit - before;
      if (const unsigned have = __ballot_sync(~0u, upto > left)) {
        int tile = left - (upto - n);
        Sequence mine = q[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) {
          const int t = mine.tiles(a);
          if (tile >= t) tile -= t, mine = q[i];
          else break;
        }
        return at(mine, tile, __ffs(have) - 1);
      }
      before += __shfl_sync(~0u, upto, 31);
    }
    return PromptUnit{};
  }
  __device__ __forceinline__ PromptUnit at(const Sequence& q, int tile, int from) const {
    PromptUnit u;
    u.s = {__shfl_sync(~0u, q.q0, from), __shfl_sync(~0u, q.lq, from), __shfl_sync(~0u, q.k0, from), __shfl_sync(~0u, q.lk, from), false};
    u.tile = __shfl_sync(~0u, tile, from);
    u.ok = u.tile >= 0;  // not so where the starts change meanwhile
    return u;
  }
  const PromptArgs& a;
  int lane;
  Sequence s;
  int first = 0, before = 0;  // the sequences from here on; units of those before
};

// One row of attention by one warp, from memory and with what the row sees alone.  A product of a weight of zero and a masked value is
// zero only while the value is finite, so the fast kernels come here with the rows that they found not finite.  Lanes share out the
// channels, four keys at a time are on their way.
template <typename T>
__device__ __forceinline__ void prompt_row_with_care(const PromptArgs& a, int q_row, int head, int k0, int seen) {
  const int lane = threadIdx.x % 32, kv = static_cast<int>(a.ratio.of(head));
  const T* k = static_cast<const T*>(a.k) + k0 * a.k_ts + kv * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + k0 * a.v_ts + kv * a.v_hs;
  float q[8], o[8] = {}, top = -INFINITY, total = 0.0f;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    q[c] = lane + 32 * c < a.d ? to_f32(static_cast<const T*>(a.q)[q_row * a.q_ts + head * a.q_hs + lane + 32 * c]) : 0.0f;
  for (int j0 = 0; j0 < seen; j0 += 4) {
    T y[4][8], x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        y[i][c] = x[i][c] = from_f32<T>(0.0f);
        if (j0 + i < seen && lane + 32 * c < a.d) {
          y[i][c] = k[(j0 + i) * a.k_ts + lane + 32 * c];
          x[i][c] = v[(j0 + i) * a.v_ts + lane + 32 * c];
        }
      }
    float s[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < 8; ++c) s[i] = fmaf(q[c], to_f32(y[i][c]), s[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (j0 + i >= seen) break;
      const float score = warp_sum(s[i]) * a.scale, now = max_nan(top, score);
      const bool nothing = now == -INFINITY;  // all scores so far
      const float keep = nothing ? 1.0f : expf(top - now), w = nothing ? 0.0f : expf(score - now);
      top = now;
      total = fmaf(total, keep, w);
#pragma unroll
      for (int c = 0; c < 8; ++c) o[c] = fmaf(w, to_f32(x[i][c]), o[c] * keep);
    }
    if (top != top) break;  // and stays so
  }
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(q_row) * a.hq + head) * a.d;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < a.d) out[lane + 32 * c] = from_f32<T>(o[c] / total);
  if (a.lse && lane == 0)
    a.lse[static_cast<long long>(q_row) * a.hq + head] = fabsf(top) < INFINITY ? top + logf(total) : top;
}

// What warp_scan() looks for, a bit for each of a lane's channels (lane, lane + 32, ..).
struct Odd {
  unsigned nan = 0, plus = 0, minus = 0, large = 0;  // NaN, +inf, -inf; magnitudes of 2^100 and more
};
// Some keys (or values) of one head from row `at` on, of `n`.
constexpr int kScanRows = 2;
template <typename T>
__device__ __forceinline__ void warp_scan(Odd& found, const T* base, long long ts, int at, int n, int d) {
  const int lane = threadIdx.x % 32;
  T x[kScanRows][8];
#pragma unroll
  for (int i = 0; i < kScanRows; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      x[i][c] = from_f32<T>(0.0f);
      if (at + i < n && lane + 32 * c < d) x[i][c] = base[(at + i) * ts + lane + 32 * c];
    }
#pragma unroll
  for (int i = 0; i < kScanRows; ++i)
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float f = to_f32(x[i][c]);
      found.nan |= f != f ? 1u << c : 0u;
      found.plus |= f == INFINITY ? 1u << c : 0u;
      found.minus |= f == -INFINITY ? 1u << c : 0u;
      found.large |= fabsf(f) >= 0x1p100f ? 1u << c : 0u;
    }
}

// A row that a fast kernel wrote and found not finite, by one warp.  Most such results are right as they are, and looking for the reason
// takes a read of the values up to the first NaN (or all that the row sees), where a row with care costs all keys and values: 8192 tokens,
// 32 / 8 heads of 128, bf16 take 0.53 ms; with a NaN in the first key as long, in the first value 0.66 ms, in value 4096 79 ms, with an
// infinity in the first value 170 ms; all rows with care would be minutes.
//   - The sum of the weights is NaN.  So is the row's reference where a score is, and all of the row.  A reference of +inf: a score is, and none
//     is NaN; the row is NaN, its log-sum +inf.  (A score may also pass fp32 by the factor |scale| log2(e), where that is above 1: such a row
//     is done with care.)  In fp32 a score is NaN also where a factor is infinite: its terms are.
//   - A channel is NaN or infinite, and the values that the row sees have the NaN or the infinities that make it so.
enum { kSumOdd = 0, kSumFine = 1, kSumNaN = 2, kSettled = 3 };
template <typename T>
__device__ __forceinline__ int prompt_sums(const PromptArgs& a, float top, float sum) {
  if (top != top) return sizeof(T) == 4 ? kSumNaN : kSettled;
  if (top == INFINITY) return fabsf(a.scale) * kLog2e <= 1.0f ? kSettled : kSumOdd;
  return sum > 0.0f && sum < INFINITY ? kSumFine : kSumOdd;
}
template <typename T>
__device__ __forceinline__ bool prompt_row_right(const PromptArgs& a, int q_row, int head, int k0, int seen, int sums) {
  const int lane = threadIdx.x % 32, kv = static_cast<int>(a.ratio.of(head));
  bool right = false;
  if (sums == kSumFine) {
    const T* out = static_cast<const T*>(a.out) + (static_cast<long long>(q_row) * a.hq + head) * a.d;
    float y[8];
    unsigned open = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      y[c] = lane + 32 * c < a.d ? to_f32(out[lane + 32 * c]) : 0.0f;
      open |= fabsf(y[c]) < INFINITY ? 0u : 1u << c;
    }
    Odd values;
    for (int at = 0; at < seen && __any_sync(~0u, open & ~values.nan); at += kScanRows)
      warp_scan(values, static_cast<const T*>(a.v) + k0 * a.v_ts + kv * a.v_hs, a.v_ts, at, seen, a.d);
    right = true;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const unsigned why = y[c] != y[c] ? values.nan | (values.plus & values.minus)
                                        : (y[c] > 0.0f ? values.plus & ~values.minus : values.minus & ~values.plus) & ~values.nan;
      right = right && !((open & ~why) >> c & 1);
    }
    right = __all_sync(~0u, right);
  } else if (sums == kSumNaN) {
    Odd query, keys;
    warp_scan(query, static_cast<const T*>(a.q) + head * a.q_hs, a.q_ts, q_row, q_row + 1, a.d);
    bool nan = __any_sync(~0u, query.nan != 0);
    for (int at = 0; at < seen && !nan; at += kScanRows) {
      warp_scan(keys, static_cast<const T*>(a.k) + k0 * a.k_ts + kv * a.k_hs, a.k_ts, at, seen, a.d);
      nan = __any_sync(~0u, keys.nan != 0);
    }
    right = nan || !__any_sync(~0u, (query.large | keys.large) != 0);
  }
  return right;
}
template <typename T>
__device__ __noinline__ void prompt_row_again(const PromptArgs& a, int q_row, int head, int k0, int seen_and_sums) {
  const int seen = seen_and_sums & 0x3fffffff;
  if (!prompt_row_right<T>(a, q_row, head, k0, seen, static_cast<int>(static_cast<unsigned>(seen_and_sums) >> 30)))
    prompt_row_with_care<T>(a, q_row, head, k0, seen);
}
// The rows of a warp, each in the lane of its bit.
template <typename T>
__device__ __forceinline__ void prompt_rows_again(const PromptArgs& a, unsigned rows, int q_row, int head, int k0, int seen, int sums) {
  for (rows &= ~__ballot_sync(~0u, sums == kSettled); rows; rows &= rows - 1) {
    const int from = __ffs(rows) - 1;
    prompt_row_again<T>(a, __shfl_sync(~0u, q_row, from), __shfl_sync(~0u, head, from), k0,
                        __shfl_sync(~0u, static_cast<int>(static_cast<unsigned>(seen) | static_cast<unsigned>(sums) << 30), from));
  }
}

// Adds up the parts of a row: one warp a row, lanes over channels.
template <typename T>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ PromptArgs a) {
  wait_for_previous();
  const long long rows = static_cast<long long>(a.tq) * a.hq, row = blockIdx.x * 8ll + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= rows) return;
  const unsigned arrived = a.arrived[row];
  __syncwarp();
  if (arrived && lane == 0) a.arrived[row] = 0;
  if (arrived != static_cast<unsigned>(a.parts)) return;  // a row outside every sequence
  // a lane has a part's head; up to 32 parts
  float4 head = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
  if (lane < a.parts) head = a.part_heads[lane * rows + row];
  const bool saw = head.x != -INFINITY;
  float top = head.y == 0.0f ? -INFINITY : head.x;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
  const float w = head.y == 0.0f ? 0.0f : exp2_approx(head.x - top);
  const float total = warp_sum(head.y == 0.0f ? 0.0f : w * head.y);
  float o[8] = {};
#pragma unroll 2
  for (int p = 0; p < a.parts; ++p) {
    const float wp = __shfl_sync(~0u, w, p);
    if (!__shfl_sync(~0u, saw, p)) continue;  // no sums; a weight that is zero alone lets a NaN or an infinity through, as in one part
    const float* from = a.part_sums + (p * rows + row) * a.d;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (lane + 32 * c < a.d) o[c] = fmaf(wp, from[lane + 32 * c], o[c]);
  }
  const int k0 = __float_as_int(__shfl_sync(~0u, head.z, 0)), seen = __float_as_int(__shfl_sync(~0u, head.w, 0));
  bool fine = total > 0.0f && total < INFINITY;
  T* out = static_cast<T*>(a.out) + row * a.d;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < a.d) {
      const float y = seen ? o[c] / total : 0.0f;
      fine = fine && fabsf(y) < INFINITY;
      out[lane + 32 * c] = from_f32<T>(y);
    }
  if (a.lse && lane == 0) a.lse[row] = seen ? log_sum(top, total) : -INFINITY;
  __syncwarp();
  // (where starts that are not in order gave rows to two sequences, the heads may be of neither)
  if (seen > 0 && k0 >= 0 && seen <= a.tk - k0 && !__all_sync(~0u, fine)) {
    const int q_row = static_cast<int>(row / a.hq);
    prompt_rows_again<T>(a, 1u, q_row, static_cast<int>(row - static_cast<long long>(q_row) * a.hq), k0, seen,
                         prompt_sums<T>(a, top, total));
  }
}

}  // namespace b200q
