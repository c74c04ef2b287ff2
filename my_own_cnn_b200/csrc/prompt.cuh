// What the kernels of prompt attention share: arguments, the order of the work, rows that are done with care.
#pragma once
#include <climits>
#include <type_traits>

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

// A row's log-sum from its reference (base 2) and its sum, which is 2^LIFT times as large.  With a score of +inf the sum is NaN.
template <int LIFT = 0>
__device__ __forceinline__ float log_sum(float top, float sum) {
  return top == INFINITY ? top : (top + log2f(sum * (1.0f / static_cast<float>(1 << LIFT)))) * (1.0f / kLog2e);
}

// A result is an average, no larger than the largest value; weights that are rounded for the second product and a sum of weights that are
// not can bring it past fp16's range all the same, by a part in 2^11.
constexpr float kHalfMost = 65504.0f;
__device__ __forceinline__ float to_half_range(float y) {
  return fabsf(y) < INFINITY ? fminf(fmaxf(y, -kHalfMost), kHalfMost) : y;
}
template <typename T>
__device__ __forceinline__ T result(float y) {
  return from_f32<T>(std::is_same<T, __half>::value ? to_half_range(y) : y);
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
// zero only while the value is finite, so the fast kernels come here with rows that they found not finite and prompt_rows_right() cannot
// explain.  C channels a lane (32 apart), 32 / C keys at a time: their partial sums are added up over the lanes and shared out to them in
// one exchange, which leaves the score of a key in each C-th of the lanes.
template <typename T, int C>
__device__ __noinline__ void prompt_row_with_care(const PromptArgs& a, int q_row, int head, int k0, int seen) {
  constexpr int kKeys = 32 / C;
  const int lane = threadIdx.x % 32, kv = static_cast<int>(a.ratio.of(head)), d = a.d;
  const long long k_ts = a.k_ts, v_ts = a.v_ts;
  const float scale = a.scale;
  const T* k = static_cast<const T*>(a.k) + k0 * k_ts + kv * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + k0 * v_ts + kv * a.v_hs;
  const T* q_at = static_cast<const T*>(a.q) + q_row * a.q_ts + head * a.q_hs;
  const T none = from_f32<T>(0.0f);
  int col[C];  // what lies past d or past the keys is read from a place that there is, and left out
  float q[C], o[C] = {}, top = -INFINITY, total = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = min(lane + 32 * c, d - 1);
    q[c] = lane + 32 * c < d ? to_f32(q_at[col[c]]) : 0.0f;
  }
  for (int j0 = 0; j0 < seen; j0 += kKeys) {
    T x[kKeys][C], y[kKeys][C];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int at = min(j0 + i, seen - 1);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        x[i][c] = k[at * k_ts + col[c]];
        y[i][c] = v[at * v_ts + col[c]];
      }
    }
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (lane + 32 * c >= d) x[i][c] = none;
        if (j0 + i >= seen) y[i][c] = none;
      }
    float s[kKeys] = {};
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) s[i] = fmaf(q[c], to_f32(x[i][c]), s[i]);
    // lane l keeps key l / C
#pragma unroll
    for (int o2 = 16, n = kKeys / 2; o2 >= C; o2 >>= 1, n >>= 1) {
      const bool upper = lane & o2;
#pragma unroll
      for (int i = 0; i < kKeys / 2; ++i)
        if (i < n) {
          const float keep = upper ? s[i + n] : s[i], give = upper ? s[i] : s[i + n];
          s[i] = keep + __shfl_xor_sync(~0u, give, o2);
        }
    }
#pragma unroll
    for (int o2 = C / 2; o2; o2 >>= 1) s[0] += __shfl_xor_sync(~0u, s[0], o2);
    const bool here = j0 + lane / C < seen;
    const float score = here ? s[0] * scale : -INFINITY;
    float now = score;
#pragma unroll
    for (int o2 = 16; o2 >= C; o2 >>= 1) now = max_nan(now, __shfl_xor_sync(~0u, now, o2));
    now = max_nan(now, top);
    const bool nothing = now == -INFINITY;  // all scores so far
    const float keep = nothing ? 1.0f : expf(top - now), w = nothing || !here ? 0.0f : expf(score - now);
    float sum = w;
#pragma unroll
    for (int o2 = 16; o2 >= C; o2 >>= 1) sum += __shfl_xor_sync(~0u, sum, o2);
    top = now;
    total = fmaf(total, keep, sum);
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] *= keep;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const float wi = __shfl_sync(~0u, w, i * C);
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = fmaf(wi, to_f32(y[i][c]), o[c]);
    }
    if (top != top) break;  // and stays so
  }
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(q_row) * a.hq + head) * a.d + lane;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (lane + 32 * c < d) out[32 * c] = result<T>(o[c] / total);
  if (a.lse && lane == 0)
    a.lse[static_cast<long long>(q_row) * a.hq + head] = fabsf(top) < INFINITY ? top + logf(total) : top;
}

// Where a channel of some keys (or values) of one head has its first NaN, +inf, -inf and magnitude of 2^100 or more.
struct FirstOdd {
  int nan = INT_MAX, plus = INT_MAX, minus = INT_MAX, large = INT_MAX;
  __device__ __forceinline__ void see(float x, int at) {
    if (fabsf(x) < 0x1p100f) return;
    large = min(large, at);
    if (x != x) nan = min(nan, at);
    if (x == INFINITY) plus = min(plus, at);
    if (x == -INFINITY) minus = min(minus, at);
  }
};

// Rows that a fast kernel wrote and found not finite, those of one warp: of one sequence and key head, each in the lane of its bit.
// Returns the ones that are not right as they are.  Most are, and looking for the reason takes one read of the values for all of them
// (up to where it is found), where a row with care costs all of its keys and values: 2048 tokens, 32 / 8 heads of 128, bf16 take
// 0.09 ms, with a NaN or an infinity in value 3 0.23, in value 1024 0.32.
//   - The sum of the weights is NaN.  So is the row's reference where a score is, and all of the row.  A reference of +inf: a score is,
//     and none is NaN; the row is NaN, its log-sum +inf.  (A score may also pass fp32 by the factor |scale| log2(e), where that is above 1:
//     such a row is done with care.)  In fp32 a score may be NaN also where a factor is infinite and the other one's first term is zero.
//   - A channel is NaN, and a value that the row sees is, or two are infinities of both signs.  Or it is infinite, and a value that
//     the row sees is the same (others would have made it NaN; what it does not see gives NaN or nothing).
enum { kSumOdd = 0, kSumFine = 1, kSumNaN = 2, kSettled = 3 };
template <typename T>
__device__ __forceinline__ int prompt_sums(const PromptArgs& a, float top, float sum) {
  if (top != top) return sizeof(T) == 4 ? kSumNaN : kSettled;
  if (top == INFINITY) return fabsf(a.scale) * kLog2e <= 1.0f ? kSettled : kSumOdd;
  return sum > 0.0f && sum < INFINITY ? kSumFine : kSumOdd;
}
// The first odd places of a head's rows from k0 on, up to `n` or where `enough` (of every lane) says so.
template <typename T, int C, typename F>
__device__ __forceinline__ void scan_rows(FirstOdd (&first)[C], const T* base, long long ts, int n, int d, F enough) {
  constexpr int kRows = 32 / C;
  const int lane = threadIdx.x % 32;
  int col[C];
#pragma unroll
  for (int c = 0; c < C; ++c) col[c] = min(lane + 32 * c, d - 1);
  for (int at = 0; at < n && !__all_sync(~0u, enough()); at += kRows) {
    T x[kRows][C];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) x[i][c] = base[min(at + i, n - 1) * ts + col[c]];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int c = 0; c < C; ++c) first[c].see(to_f32(x[i][c]), min(at + i, n - 1));
  }
}
template <typename T, int C>
__device__ __noinline__ unsigned prompt_rows_right(const PromptArgs& a, unsigned rows, int q_row, int head, int k0, int seen, int sums) {
  const int lane = threadIdx.x % 32, kv = static_cast<int>(a.ratio.of(__shfl_sync(~0u, head, __ffs(rows) - 1)));
  const unsigned fine = rows & __ballot_sync(~0u, sums == kSumFine), nan = rows & __ballot_sync(~0u, sums == kSumNaN);
  unsigned left = rows & ~fine & ~nan;
  const auto each = [](unsigned of, auto&& f) {
    for (; of; of &= of - 1) f(__ffs(of) - 1);
  };
  if (fine) {
    // a lane's channels that are NaN (bit c), +inf (8 + c), -inf (16 + c) in a row
    const auto odd = [&](int row) {
      const int at = __shfl_sync(~0u, q_row, row), h = __shfl_sync(~0u, head, row);
      const T* out = static_cast<const T*>(a.out) + (static_cast<long long>(at) * a.hq + h) * a.d + lane;
      unsigned r = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float y = lane + 32 * c < a.d ? to_f32(out[32 * c]) : 0.0f;
        r |= y != y ? 1u << c : y == INFINITY ? 0x100u << c : y == -INFINITY ? 0x10000u << c : 0u;
      }
      return r;
    };
    unsigned open = 0;
    each(fine, [&](int row) { open |= odd(row); });
    FirstOdd first[C];
    // whether a channel's reasons lie before `n`
    const auto explained = [&](unsigned of, int n) {
      bool yes = true;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (of >> c & 1) yes = yes && (first[c].nan < n || max(first[c].plus, first[c].minus) < n);
        if (of >> (8 + c) & 1) yes = yes && first[c].plus < n;
        if (of >> (16 + c) & 1) yes = yes && first[c].minus < n;
      }
      return yes;
    };
    const int most = __reduce_max_sync(~0u, fine >> lane & 1 ? seen : 0);
    scan_rows<T, C>(first, static_cast<const T*>(a.v) + k0 * a.v_ts + kv * a.v_hs, a.v_ts, most, a.d, [&] { return explained(open, INT_MAX); });
    each(fine, [&](int row) {
      if (!__all_sync(~0u, explained(odd(row), __shfl_sync(~0u, seen, row)))) left |= 1u << row;
    });
  }
  if (nan) {
    FirstOdd keys[C];
    const auto any = [&](auto&& get) {
      int at = INT_MAX;
#pragma unroll
      for (int c = 0; c < C; ++c) at = min(at, get(keys[c]));
      return __reduce_min_sync(~0u, at);
    };
    const int most = __reduce_max_sync(~0u, nan >> lane & 1 ? seen : 0);
    scan_rows<T, C>(keys, static_cast<const T*>(a.k) + k0 * a.k_ts + kv * a.k_hs, a.k_ts, most, a.d,
                    [&] { return any([](const FirstOdd& f) { return f.nan; }) != INT_MAX; });
    const int first_nan = any([](const FirstOdd& f) { return f.nan; }), first_large = any([](const FirstOdd& f) { return f.large; });
    each(nan, [&](int row) {
      const int at = __shfl_sync(~0u, q_row, row), h = __shfl_sync(~0u, head, row), n = __shfl_sync(~0u, seen, row);
      const T* q = static_cast<const T*>(a.q) + at * a.q_ts + h * a.q_hs + lane;
      FirstOdd query;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (lane + 32 * c < a.d) query.see(to_f32(q[32 * c]), 0);
      if (__any_sync(~0u, query.nan == 0) || first_nan < n) return;
      if (__any_sync(~0u, query.large == 0) || first_large < n) left |= 1u << row;
    });
  }
  return left;
}
// The rows of a warp that are not finite, each in the lane of its bit.
template <typename T, int C>
__device__ __forceinline__ void prompt_rows_again_of(const PromptArgs& a, unsigned rows, int q_row, int head, int k0, int seen, int sums) {
  rows = prompt_rows_right<T, C>(a, rows, q_row, head, k0, seen, sums);
  for (; rows; rows &= rows - 1) {
    const int from = __ffs(rows) - 1;
    prompt_row_with_care<T, C>(a, __shfl_sync(~0u, q_row, from), __shfl_sync(~0u, head, from), k0, __shfl_sync(~0u, seen, from));
  }
}
template <typename T>
__device__ __forceinline__ void prompt_rows_again(const PromptArgs& a, unsigned rows, int q_row, int head, int k0, int seen, int sums) {
  rows &= ~__ballot_sync(~0u, sums == kSettled);
  if (!rows) return;
  if (a.d <= 64)
    prompt_rows_again_of<T, 2>(a, rows, q_row, head, k0, seen, sums);
  else if (a.d <= 128)
    prompt_rows_again_of<T, 4>(a, rows, q_row, head, k0, seen, sums);
  else
    prompt_rows_again_of<T, 8>(a, rows, q_row, head, k0, seen, sums);
}

// Adds up the parts of a row: one warp a row, lanes over channels.
template <typename T>
__global__ void __launch_bounds__(256, 2) prompt_join_kernel(const __grid_constant__ PromptArgs a) {
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
      out[lane + 32 * c] = result<T>(y);
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
