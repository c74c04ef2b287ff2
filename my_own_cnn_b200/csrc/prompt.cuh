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
  long long most_units;  // key heads times tiles, as many as there may be
  float scale;
  int* err;
  long long limit;
};

constexpr float kLog2e = 1.4426950408889634f;

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

// Tile `tile` of a sequence; the units are in falling order of the keys that they see, in steps of 128, so that the longest start first and the
// short ones fill up the end.  Found by bisection over the number of units with more than l steps.  A warp's work; a lane
// keeps the first 32 sequences in registers.
struct PromptUnit {
  Sequence s;
  int tile;
  bool ok;
};
__device__ __forceinline__ int warp_total(int v) { return __reduce_add_sync(~0u, v); }
// A sequence's units, the last `above(l)` of which have more than l steps.
struct Units {
  int tiles, lq, shift, most;  // keys less queries; steps of the last unit
  __device__ __forceinline__ Units(const PromptArgs& a, const Sequence& s)
      : tiles(s.tiles(a)), lq(s.lq), shift(s.lk - s.lq), most(tiles ? max(0, s.lk + kUnitKeys - 1) / kUnitKeys : 0) {}
  static constexpr int kUnitKeys = 128;
  // all at l < 0; from the first tile whose end passes l steps on
  __device__ __forceinline__ int above(const PromptArgs& a, int l) const {
    if (l < 0) return tiles;
    if (l >= most) return 0;
    const int tokens = l * kUnitKeys - shift;  // that l steps reach
    if (tokens < 0) return tiles;
    return tiles - min(tiles, static_cast<int>(a.tile.of(static_cast<uint32_t>(min(tokens, lq) * a.row_scale))));
  }
};
__device__ inline PromptUnit prompt_unit(const PromptArgs& a, int unit, bool report) {
  const int lane = threadIdx.x % 32;
  const Sequence first = sequence(a, lane);
  const Units mine(a, first);
  bool bad = first.bad;
  int most = mine.most, all = mine.tiles;
  for (int i = 32 + lane; i < a.b; i += 32) {
    const Sequence s = sequence(a, i);
    const Units u(a, s);
    bad |= s.bad;
    most = max(most, u.most);
    all += u.tiles;
  }
  if (report && bad) atomicCAS(a.err, 0, kDevErrBadStarts);
  PromptUnit u{};
  if (unit >= warp_total(all)) return u;
  auto units_above = [&](int l) {
    int n = mine.above(a, l);
    for (int i = 32 + lane; i < a.b; i += 32) n += Units(a, sequence(a, i)).above(a, l);
    return warp_total(n);
  };
  // units_above(lo) > unit >= units_above(hi) = longer: the unit has hi steps
  int lo = -1, hi = __reduce_max_sync(~0u, most), longer = 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2, n = units_above(mid);
    if (n > unit)
      lo = mid;
    else
      hi = mid, longer = n;
  }
  int left = unit - longer;  // of the units with hi steps
  for (int i0 = 0; i0 < a.b; i0 += 32) {
    const Sequence s = i0 ? sequence(a, i0 + lane) : first;
    const Units v(a, s);
    const int end = v.tiles - v.above(a, hi), n = v.above(a, lo) - v.above(a, hi);
    int upto = n;  // with the sequences before
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned have = __ballot_sync(~0u, upto > left);
    if (have) {
      const int from = __ffs(have) - 1;
      u.s = {__shfl_sync(~0u, s.q0, from), __shfl_sync(~0u, s.lq, from), __shfl_sync(~0u, s.k0, from), __shfl_sync(~0u, s.lk, from),
             false};
      u.tile = __shfl_sync(~0u, end - 1 - (left - (upto - n)), from);
      u.ok = u.tile >= 0;
      return u;
    }
    left -= __shfl_sync(~0u, upto, 31);
  }
  return u;  // the starts changed meanwhile
}

// One row of attention by one warp, from memory and with what the row sees alone.  A product of a weight of zero and a masked value is
// zero only while the value is finite, so the fast kernels come here with the rows that they found not finite.
template <typename T>
__device__ __noinline__ void prompt_row_with_care(const PromptArgs& a, int q_row, int head, int k0, int seen) {
  const int lane = threadIdx.x % 32, kv = static_cast<int>(a.ratio.of(head));
  const T* q = static_cast<const T*>(a.q) + q_row * a.q_ts + head * a.q_hs;
  const T* k = static_cast<const T*>(a.k) + k0 * a.k_ts + kv * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + k0 * a.v_ts + kv * a.v_hs;
  auto score = [&](int j) {
    const T* kj = k + j * a.k_ts;
    float s = 0.0f;
    for (int c = 0; c < a.d; ++c) s = fmaf(to_f32(q[c]), to_f32(kj[c]), s);
    return s * a.scale;
  };
  float top = -INFINITY;
  for (int j = lane; j < seen; j += 32) top = max_nan(top, score(j));
  for (int o = 16; o; o >>= 1) top = max_nan(top, __shfl_xor_sync(~0u, top, o));
  float total = 0.0f, o[8] = {};
  for (int j0 = 0; j0 < seen; j0 += 32) {
    const float p = j0 + lane < seen ? expf(score(j0 + lane) - top) : 0.0f;
    total += p;
    for (int i = 0; i < min(32, seen - j0); ++i) {
      const float w = __shfl_sync(~0u, p, i);
      const T* vj = v + (j0 + i) * a.v_ts;
      for (int c = 0; c < 8; ++c)
        if (lane + 32 * c < a.d) o[c] = fmaf(w, to_f32(vj[lane + 32 * c]), o[c]);
    }
  }
  total = warp_sum(total);
  T* out = static_cast<T*>(a.out) + (static_cast<long long>(q_row) * a.hq + head) * a.d;
  for (int c = 0; c < 8; ++c)
    if (lane + 32 * c < a.d) out[lane + 32 * c] = from_f32<T>(o[c] / total);
  if (a.lse && lane == 0)
    a.lse[static_cast<long long>(q_row) * a.hq + head] = fabsf(top) < INFINITY ? top + logf(total) : top;
}

}  // namespace b200q
