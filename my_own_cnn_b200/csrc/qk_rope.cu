// Per-head RMS norm of queries and keys with the position rotation, and its gradient
// (b200q_qk_norm_rope, b200q_qk_norm_rope_bprop).
//
//   n = x r w, r = (mean x^2 + eps)^-1/2;  y = R(pos) n
//   dn = R^T dy;  dw = sum dn x r;  with v = dn w: dx = r (v - x r^2 mean(v x))
//
// Bytes bound both: x in, y out; the gradient reads x and dy and writes dx.  8192 tokens x 40 heads x 128 fp16: 32.5 us, 5.3
// TB/s; gradient of 4097 x 32 x 64 fp32: 22.2 us, 4.6 TB/s.  A row of up to 256 channels lies in the
// registers of 8, 16 or 32 lanes, 8 channels each, from one read to one write.  Which 8: four pairs that rotate
// together, so that a rotation needs no other lane (half and half: 4 channels of the first half of the rotated ones and
// the 4 that they turn with; interleaved: 8 in a row), and four cosines and sines.  The mean is a few shuffles.  A group
// of lanes takes several heads of one token, so that it reads the token's angles and the weights once, and has
// kAhead rows on their way at a time.  Rows that are not aligned, and sizes that are no multiple of 8, go one warp per row
// through strided loops.
#include <algorithm>

#include "host.h"
#include "lowbit.cuh"

namespace b200q {
namespace {

// One of the two tensors (queries or keys): rows (token, head) of d channels.
struct NormSide {
  const void* x;
  long long ts, hs;
  const void* w;  // may be null
  void* y;        // output (forward), input gradient (bprop)
  long long yts, yhs;
  const void* dy;  // bprop: contiguous
  int heads;
};

struct NormArgs {
  NormSide side[2];
  const float* table;
  const int32_t* pos;
  int positions, t, d, rot, interleaved;
  float eps;
  int* err;
  float* partial;  // bprop: [blocks][2][d] weight-gradient sums
};

constexpr int kNormWarps = 8;

// The rotation of a pair lies in row pos[t] of the table; null for a position outside it.
__device__ __forceinline__ const float* table_row(const NormArgs& a, int t) {
  const int p = a.pos[t];
  if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.positions)) {
    atomicCAS(a.err, 0, kDevErrBadPosition);
    return nullptr;
  }
  return a.table + static_cast<size_t>(p) * a.rot;
}

// Channels of pair i of a row's rotated part.
__device__ __forceinline__ int2 pair_of(const NormArgs& a, int i) {
  return a.interleaved ? make_int2(2 * i, 2 * i + 1) : make_int2(i, i + a.rot / 2);
}

template <typename T>
__device__ __forceinline__ float weight(const T* w, int i) {
  return w ? to_f32(w[i]) : 1.0f;
}

// One warp per row.  A lane writes only the channels that it has read, so y may be x.
template <typename T>
__global__ void qk_norm_rope_kernel(NormArgs a) {
  wait_for_previous();
  const int heads = a.side[0].heads + a.side[1].heads;
  const long long row = static_cast<long long>(blockIdx.x) * kNormWarps + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (row >= static_cast<long long>(a.t) * heads) return;
  const int t = static_cast<int>(row / heads);
  int h = static_cast<int>(row % heads);
  const int which = h >= a.side[0].heads;
  const NormSide& s = a.side[which];
  if (which) h -= a.side[0].heads;
  const T* x = static_cast<const T*>(s.x) + t * s.ts + h * s.hs;
  T* y = static_cast<T*>(s.y) + t * s.yts + h * s.yhs;
  const T* w = static_cast<const T*>(s.w);
  float sq = 0.0f;
  for (int i = lane; i < a.d; i += 32) {
    const float v = to_f32(x[i]);
    sq += v * v;
  }
  const float r = rsqrtf(warp_sum(sq) / a.d + a.eps);
  const float* tab = a.rot ? table_row(a, t) : nullptr;
  if (a.rot && !tab) return;
  for (int i = lane; i < a.rot / 2; i += 32) {
    const int2 p = pair_of(a, i);
    const float u = to_f32(x[p.x]) * r * weight(w, p.x), v = to_f32(x[p.y]) * r * weight(w, p.y);
    const float c = tab[i], sn = tab[a.rot / 2 + i];
    y[p.x] = from_f32<T>(u * c - v * sn);
    y[p.y] = from_f32<T>(v * c + u * sn);
  }
  for (int i = a.rot + lane; i < a.d; i += 32) y[i] = from_f32<T>(to_f32(x[i]) * r * weight(w, i));
}

// One warp per row, a block over many rows; lanes own channels, so each warp's weight-gradient sums in
// shared memory need no atomics.
template <typename T>
__global__ void qk_norm_rope_bprop_kernel(NormArgs a) {
  wait_for_previous();
  extern __shared__ float sums[];  // [kNormWarps][2][d]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  float* mine = sums + warp * 2 * a.d;
  for (int i = lane; i < 2 * a.d; i += 32) mine[i] = 0.0f;
  __syncwarp();
  const int heads = a.side[0].heads + a.side[1].heads;
  for (long long row = static_cast<long long>(blockIdx.x) * kNormWarps + warp; row < static_cast<long long>(a.t) * heads;
       row += static_cast<long long>(gridDim.x) * kNormWarps) {
    const int t = static_cast<int>(row / heads);
    int h = static_cast<int>(row % heads);
    const int which = h >= a.side[0].heads;
    const NormSide& s = a.side[which];
    if (which) h -= a.side[0].heads;
    const T* x = static_cast<const T*>(s.x) + t * s.ts + h * s.hs;
    const long long flat = (static_cast<long long>(t) * s.heads + h) * a.d;
    const T* dy = static_cast<const T*>(s.dy) + flat;
    T* dx = static_cast<T*>(s.y) + flat;
    const T* w = static_cast<const T*>(s.w);
    float* dw = mine + which * a.d;
    const float* tab = a.rot ? table_row(a, t) : nullptr;
    if (a.rot && !tab) continue;
    float sq = 0.0f, gx = 0.0f;
    for (int i = lane; i < a.d; i += 32) sq += to_f32(x[i]) * to_f32(x[i]);
    const float r = rsqrtf(warp_sum(sq) / a.d + a.eps);
    auto back = [&](int i, int2* p, float* u, float* v) {
      *p = pair_of(a, i);
      const float c = tab[i], sn = tab[a.rot / 2 + i], du = to_f32(dy[p->x]), dv = to_f32(dy[p->y]);
      *u = du * c + dv * sn;
      *v = dv * c - du * sn;
    };
    for (int i = lane; i < a.rot / 2; i += 32) {
      int2 p;
      float u, v;
      back(i, &p, &u, &v);
      const float xa = to_f32(x[p.x]), xb = to_f32(x[p.y]);
      gx += u * weight(w, p.x) * xa + v * weight(w, p.y) * xb;
      dw[p.x] += u * xa * r;
      dw[p.y] += v * xb * r;
    }
    for (int i = a.rot + lane; i < a.d; i += 32) {
      const float u = to_f32(dy[i]), xa = to_f32(x[i]);
      gx += u * weight(w, i) * xa;
      dw[i] += u * xa * r;
    }
    const float k = r * r * (warp_sum(gx) / a.d);
    for (int i = lane; i < a.rot / 2; i += 32) {
      int2 p;
      float u, v;
      back(i, &p, &u, &v);
      dx[p.x] = from_f32<T>(r * (u * weight(w, p.x) - to_f32(x[p.x]) * k));
      dx[p.y] = from_f32<T>(r * (v * weight(w, p.y) - to_f32(x[p.y]) * k));
    }
    for (int i = a.rot + lane; i < a.d; i += 32)
      dx[i] = from_f32<T>(r * (to_f32(dy[i]) * weight(w, i) - to_f32(x[i]) * k));
    __syncwarp();
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.d; i += blockDim.x) {
    float v = 0.0f;
    for (int j = 0; j < kNormWarps; ++j) v += sums[j * 2 * a.d + i];
    a.partial[static_cast<size_t>(blockIdx.x) * 2 * a.d + i] = v;
  }
}

constexpr int kFastThreads = 128;
constexpr int kAhead = 4;

// Four channels in memory, as two fp32 pairs.
template <typename T>
struct Four;
template <>
struct Four<float> {
  using Bits = uint4;
  static __device__ __forceinline__ void get(const Bits& v, float2 (&x)[2]) {
    x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ Bits put(const float2 (&x)[2]) {
    return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x), __float_as_uint(x[1].y));
  }
};
template <>
struct Four<__half> {
  using Bits = uint2;
  static __device__ __forceinline__ void get(const Bits& v, float2 (&x)[2]) {
    x[0] = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    x[1] = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  }
  static __device__ __forceinline__ Bits put(const float2 (&x)[2]) {
    return make_uint2(pack_f16(x[0].x, x[0].y), pack_f16(x[1].x, x[1].y));
  }
};
template <>
struct Four<__nv_bfloat16> {
  using Bits = uint2;
  static __device__ __forceinline__ void get(const Bits& v, float2 (&x)[2]) {
    x[0] = make_float2(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u));
    x[1] = make_float2(__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
  }
  static __device__ __forceinline__ Bits put(const float2 (&x)[2]) {
    return make_uint2(pack_bf16(x[0].x, x[0].y), pack_bf16(x[1].x, x[1].y));
  }
};

// A lane's 8 channels of a row: two fours at `at[0]` and `at[1]`.
struct Lane {
  int at[2];
  bool there;    // a row of fewer channels than its lanes can hold leaves the last lanes empty
  bool rotated;
};
template <bool INTERLEAVED>
__device__ __forceinline__ Lane lane_of(const NormArgs& a, int l) {
  Lane r;
  r.rotated = 8 * l < a.rot;
  r.there = 8 * l < a.d;
  r.at[0] = !INTERLEAVED && r.rotated ? 4 * l : 8 * l;
  r.at[1] = !INTERLEAVED && r.rotated ? a.rot / 2 + 4 * l : 8 * l + 4;
  return r;
}

// The two fours as pairs that turn together: x[i].x with y[i].x, x[i].y with y[i].y, angles 2 i and 2 i + 1.
template <bool INTERLEAVED>
__device__ __forceinline__ void to_pairs(const float2 (&f0)[2], const float2 (&f1)[2], float2 (&x)[2], float2 (&y)[2]) {
  if constexpr (INTERLEAVED) {
    x[0] = make_float2(f0[0].x, f0[1].x), y[0] = make_float2(f0[0].y, f0[1].y);
    x[1] = make_float2(f1[0].x, f1[1].x), y[1] = make_float2(f1[0].y, f1[1].y);
  } else {
    x[0] = f0[0], x[1] = f0[1], y[0] = f1[0], y[1] = f1[1];
  }
}
template <bool INTERLEAVED>
__device__ __forceinline__ void from_pairs(const float2 (&x)[2], const float2 (&y)[2], float2 (&f0)[2], float2 (&f1)[2]) {
  if constexpr (INTERLEAVED) {
    f0[0] = make_float2(x[0].x, y[0].x), f0[1] = make_float2(x[0].y, y[0].y);
    f1[0] = make_float2(x[1].x, y[1].x), f1[1] = make_float2(x[1].y, y[1].y);
  } else {
    f0[0] = x[0], f0[1] = x[1], f1[0] = y[0], f1[1] = y[1];
  }
}

template <typename T, bool INTERLEAVED>
struct Row {
  typename Four<T>::Bits bits[2];
  __device__ __forceinline__ void load(const T* p, const Lane& l, bool ok) {
    bits[0] = bits[1] = {};
    if (ok) {
      bits[0] = *reinterpret_cast<const typename Four<T>::Bits*>(p + l.at[0]);
      bits[1] = *reinterpret_cast<const typename Four<T>::Bits*>(p + l.at[1]);
    }
  }
  __device__ __forceinline__ void get(float2 (&x)[2], float2 (&y)[2]) const {
    float2 f0[2], f1[2];
    Four<T>::get(bits[0], f0);
    Four<T>::get(bits[1], f1);
    to_pairs<INTERLEAVED>(f0, f1, x, y);
  }
  static __device__ __forceinline__ void store(T* p, const Lane& l, const float2 (&x)[2], const float2 (&y)[2]) {
    float2 f0[2], f1[2];
    from_pairs<INTERLEAVED>(x, y, f0, f1);
    *reinterpret_cast<typename Four<T>::Bits*>(p + l.at[0]) = Four<T>::put(f0);
    *reinterpret_cast<typename Four<T>::Bits*>(p + l.at[1]) = Four<T>::put(f1);
  }
};

// Angles of a lane's four pairs (none: cosine 1, sine 0).
struct Angles {
  float2 c[2], s[2];
  __device__ __forceinline__ void load(const NormArgs& a, const float* row, const Lane& lane, int l) {
    c[0] = c[1] = both(1.0f);
    s[0] = s[1] = both(0.0f);
    if (row && lane.rotated) {
      const float4 cv = __ldg(reinterpret_cast<const float4*>(row + 4 * l));
      const float4 sv = __ldg(reinterpret_cast<const float4*>(row + a.rot / 2 + 4 * l));
      c[0] = make_float2(cv.x, cv.y), c[1] = make_float2(cv.z, cv.w);
      s[0] = make_float2(sv.x, sv.y), s[1] = make_float2(sv.z, sv.w);
    }
  }
};

template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void lane_weights(const void* w, const Lane& lane, float2 (&x)[2], float2 (&y)[2]) {
  x[0] = x[1] = y[0] = y[1] = both(1.0f);
  if (w) {
    Row<T, INTERLEAVED> r;
    r.load(static_cast<const T*>(w), lane, lane.there);
    r.get(x, y);
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float2 v) {
  float s = v.x + v.y;
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}

// A token's units: `per` heads each of the queries, then of the keys.
struct Split {
  int per, parts_q;
  Divisor parts;
};

// Unit: one side's heads [begin, end) of token t.
struct Unit {
  int t, which, begin, end;
  const float* table;
  bool ok;
};
__device__ __forceinline__ Unit unit_of(const NormArgs& a, uint32_t unit, const Split& split) {
  Unit u;
  u.t = static_cast<int>(split.parts.of(unit));
  int part = static_cast<int>(unit - static_cast<uint32_t>(u.t) * split.parts.d);
  u.which = part >= split.parts_q;
  if (u.which) part -= split.parts_q;
  u.ok = u.t < a.t;
  u.begin = part * split.per;
  u.end = u.ok ? min(a.side[u.which].heads, u.begin + split.per) : u.begin;
  u.table = nullptr;
  if (u.ok && a.rot) u.ok = (u.table = table_row(a, u.t)) != nullptr;
  return u;
}

// A group of LPR lanes takes `per` heads of one token's queries or keys.
template <typename T, int LPR, bool INTERLEAVED>
__global__ void __launch_bounds__(kFastThreads) qk_norm_rope_rows_kernel(NormArgs a, Split split) {
  wait_for_previous();
  const int l = threadIdx.x % LPR;
  const Lane lane = lane_of<INTERLEAVED>(a, l);
  const Unit unit = unit_of(a, blockIdx.x * (kFastThreads / LPR) + threadIdx.x / LPR, split);
  const NormSide& s = a.side[unit.which];
  const T* x = static_cast<const T*>(s.x) + unit.t * s.ts;
  T* y = static_cast<T*>(s.y) + unit.t * s.yts;
  const float over = 1.0f / static_cast<float>(a.d);
  Angles angles;
  float2 w[2], wy[2];
  Row<T, INTERLEAVED> row[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) row[u].load(x + (unit.begin + u) * s.hs, lane, lane.there && unit.begin + u < unit.end);
  angles.load(a, unit.table, lane, l);
  lane_weights<T, INTERLEAVED>(s.w, lane, w, wy);
  for (int h0 = unit.begin; __any_sync(~0u, h0 < unit.end); h0 += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float2 p[2], q[2];
      row[u].get(p, q);
      row[u].load(x + (h0 + u + kAhead) * s.hs, lane, lane.there && h0 + u + kAhead < unit.end);
      const float2 sq = fma2(p[0], p[0], fma2(p[1], p[1], fma2(q[0], q[0], mul2(q[1], q[1]))));
      const float2 r = both(rsqrtf(row_sum<LPR>(sq) * over + a.eps));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 v = mul2(p[i], mul2(r, w[i])), z = mul2(q[i], mul2(r, wy[i]));
        p[i] = fma2(make_float2(-z.x, -z.y), angles.s[i], mul2(v, angles.c[i]));
        q[i] = fma2(v, angles.s[i], mul2(z, angles.c[i]));
      }
      if (unit.ok && lane.there && h0 + u < unit.end) Row<T, INTERLEAVED>::store(y + (h0 + u) * s.yhs, lane, p, q);
    }
  }
}

// The gradient: groups of lanes walk over units, the weights' sums stay in registers.
template <typename T, int LPR, bool INTERLEAVED>
__global__ void __launch_bounds__(kFastThreads) qk_norm_rope_bprop_rows_kernel(NormArgs a, Split split, uint32_t units) {
  wait_for_previous();
  constexpr int kGroups = kFastThreads / LPR, kRowsAhead = 2;
  __shared__ float sums[kGroups][2][LPR * 8];
  const int l = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane lane = lane_of<INTERLEAVED>(a, l);
  const float over = 1.0f / static_cast<float>(a.d);
  float2 dw[2][2][2];  // [side][x or y][pair]
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i / 4][i / 2 % 2][i % 2] = both(0.0f);
  for (uint32_t first = blockIdx.x * kGroups; first < units; first += gridDim.x * kGroups) {
    const Unit unit = unit_of(a, first + group, split);
    const NormSide& s = a.side[unit.which];
    const T* x = static_cast<const T*>(s.x) + unit.t * s.ts;
    const long long flat = static_cast<long long>(unit.t) * s.heads * a.d;
    const T* dy = static_cast<const T*>(s.dy) + flat;
    T* dx = static_cast<T*>(s.y) + flat;
    const bool live = unit.ok && lane.there;
    Angles angles;
    float2 w[2], wy[2], add[2][2];
    add[0][0] = add[0][1] = add[1][0] = add[1][1] = both(0.0f);
    Row<T, INTERLEAVED> row[kRowsAhead], grad[kRowsAhead];
    auto load = [&](int u, int h) {
      row[u].load(x + h * s.hs, lane, live && h < unit.end);
      grad[u].load(dy + h * a.d, lane, live && h < unit.end);
    };
#pragma unroll
    for (int u = 0; u < kRowsAhead; ++u) load(u, unit.begin + u);
    angles.load(a, unit.table, lane, l);
    lane_weights<T, INTERLEAVED>(s.w, lane, w, wy);
    for (int h0 = unit.begin; __any_sync(~0u, h0 < unit.end); h0 += kRowsAhead) {
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        float2 p[2], q[2], dp[2], dq[2];
        row[u].get(p, q);
        grad[u].get(dp, dq);
        load(u, h0 + u + kRowsAhead);
        const float2 sq = fma2(p[0], p[0], fma2(p[1], p[1], fma2(q[0], q[0], mul2(q[1], q[1]))));
        float2 vx = both(0.0f), v[2], z[2], np[2], nq[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 back = make_float2(-angles.s[i].x, -angles.s[i].y);
          const float2 dn = fma2(dq[i], angles.s[i], mul2(dp[i], angles.c[i]));
          const float2 dm = fma2(dp[i], back, mul2(dq[i], angles.c[i]));
          np[i] = mul2(dn, p[i]);
          nq[i] = mul2(dm, q[i]);
          v[i] = mul2(dn, w[i]);
          z[i] = mul2(dm, wy[i]);
          vx = fma2(v[i], p[i], fma2(z[i], q[i], vx));
        }
        const float r = rsqrtf(row_sum<LPR>(sq) * over + a.eps), k = -r * r * (row_sum<LPR>(vx) * over);
        const float2 rr = both(live && h0 + u < unit.end ? r : 0.0f);  // empty lanes: no 0 times infinity
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          add[0][i] = fma2(rr, np[i], add[0][i]);
          add[1][i] = fma2(rr, nq[i], add[1][i]);
          p[i] = mul2(rr, fma2(both(k), p[i], v[i]));
          q[i] = mul2(rr, fma2(both(k), q[i], z[i]));
        }
        if (live && h0 + u < unit.end) Row<T, INTERLEAVED>::store(dx + (h0 + u) * a.d, lane, p, q);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = add[i / 2][i % 2];
      if (unit.which)
        dw[1][i / 2][i % 2] = add2(dw[1][i / 2][i % 2], v);
      else
        dw[0][i / 2][i % 2] = add2(dw[0][i / 2][i % 2], v);
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float2 f0[2], f1[2];
    from_pairs<INTERLEAVED>(dw[which][0], dw[which][1], f0, f1);
    if (lane.there) {
      *reinterpret_cast<float4*>(&sums[group][which][lane.at[0]]) = make_float4(f0[0].x, f0[0].y, f0[1].x, f0[1].y);
      *reinterpret_cast<float4*>(&sums[group][which][lane.at[1]]) = make_float4(f1[0].x, f1[0].y, f1[1].x, f1[1].y);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.d; i += kFastThreads) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) v += sums[j][i / a.d][i % a.d];
    a.partial[static_cast<size_t>(blockIdx.x) * 2 * a.d + i] = v;
  }
}

// Adds the blocks' weight gradients up in a fixed order: 32 columns a block, the partial sums shared out to 32 warps.
template <typename T>
__global__ void norm_weight_grad_kernel(const float* partial, int blocks, int d, T* dqw, T* dkw) {
  wait_for_previous();
  __shared__ float sums[32][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, i = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (i < 2 * d) {
#pragma unroll 10
    for (int b = warp; b < blocks; b += 32) v += partial[static_cast<size_t>(b) * 2 * d + i];
  }
  sums[warp][lane] = v;
  __syncthreads();
  const float all = warp_sum(sums[lane][warp]);  // column `warp` of the block's 32
  const int c = blockIdx.x * 32 + warp;
  if (lane == 0 && c < 2 * d) {
    T* out = c < d ? dqw : dkw;
    if (out) out[c % d] = from_f32<T>(all);
  }
}

// Lanes of a row, 0 where the rows kernels do not take the call: channels, rotated ones and strides are multiples of
// what a lane moves at a time.
int row_lanes(const NormArgs& a, int size, bool back) {
  const unsigned mask = 4 * size - 1;  // alignment of four channels
  if (a.d > 256 || a.d % 8 || a.rot % 8 || (a.rot && (reinterpret_cast<uintptr_t>(a.table) & 15u))) return 0;
  for (const NormSide& s : a.side) {
    uintptr_t bits = reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y) | reinterpret_cast<uintptr_t>(s.w);
    long long strides = s.ts | s.hs;
    if (back)
      bits |= reinterpret_cast<uintptr_t>(s.dy);
    else
      strides |= s.yts | s.yhs;
    if (s.heads && ((bits & mask) || strides % 4)) return 0;
  }
  return a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32;
}

// Heads that one group of lanes takes: many when there are enough rows to fill the GPU with eights (angles
// and weights are read less often), one when there are few (a row's latency is all there is).
Split split_heads(const NormArgs& a, int lanes, int sms) {
  const int hq = a.side[0].heads, hk = a.side[1].heads;
  const long long lanes_of_all = static_cast<long long>(a.t) * (hq + hk) * lanes, full = 1024ll * sms;
  Split s;
  s.per = lanes_of_all >= 16 * full ? 8 : lanes_of_all >= 4 * full ? 4 : 1;
  s.parts_q = (hq + s.per - 1) / s.per;
  s.parts = Divisor(s.parts_q + (hk + s.per - 1) / s.per);
  return s;
}

#define B200Q_NORM_ROWS(kernel)                                                                                  \
  (a.interleaved ? (lanes == 8 ? kernel<T, 8, true> : lanes == 16 ? kernel<T, 16, true> : kernel<T, 32, true>)   \
                 : (lanes == 8 ? kernel<T, 8, false> : lanes == 16 ? kernel<T, 16, false> : kernel<T, 32, false>))

// Checks what both directions share and fills in the kernels' arguments.
int norm_args(const b200q_qk_norm_args* p, NormArgs* a, int* sms) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const int ftype = p->ftype, t = p->t, hq = p->hq, hk = p->hk, d = p->d, rot = p->rot;
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (t < 0 || hq < 0 || hk < 0 || d <= 0) return host_fail(B200Q_ERR_INVALID_ARG, "bad head dimensions");
  if (rot < 0 || rot > d || rot % 2)
    return host_fail(B200Q_ERR_INVALID_ARG, "rotated channels must be even and at most %d, got %d", d, rot);
  if (d > 1024) return host_fail(B200Q_ERR_UNSUPPORTED, "heads of more than 1024 channels");
  if (hq + hk > (1 << 20)) return host_fail(B200Q_ERR_UNSUPPORTED, "too many heads");
  if (t > 0) {
    if ((hq && (!p->q || !p->q_out)) || (hk && (!p->k || !p->k_out)))
      return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
    if (rot && (!p->table || !p->pos || p->positions <= 0))
      return host_fail(B200Q_ERR_INVALID_ARG, "a rotation needs its table and positions");
  }
  a->side[0] = {p->q, p->q_ts, p->q_hs, p->q_w, p->q_out, p->qo_ts, p->qo_hs, p->q_grad, hq};
  a->side[1] = {p->k, p->k_ts, p->k_hs, p->k_w, p->k_out, p->ko_ts, p->ko_hs, p->k_grad, hk};
  a->table = p->table;
  a->pos = p->pos;
  a->positions = p->positions;
  a->t = t;
  a->d = d;
  a->rot = rot;
  a->interleaved = p->interleaved;
  a->eps = p->eps;
  if (t == 0 || hq + hk == 0) return B200Q_OK;
  return host_device(sms, &a->err);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_qk_norm_rope(const b200q_qk_norm_args* args, void* stream) {
  NormArgs a{};
  int sms = 0;
  int rc = norm_args(args, &a, &sms);
  if (rc) return rc;
  const int ftype = args->ftype, t = a.t, hq = args->hq, hk = args->hk, d = a.d;
  if (t == 0 || hq + hk == 0) return B200Q_OK;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const int size = ftype == B200Q_F32 ? 4 : 2;
  if (const int lanes = row_lanes(a, size, false)) {
    const Split split = split_heads(a, lanes, sms);
    const long long units = static_cast<long long>(t) * split.parts.d;
    const long long blocks = (units * lanes + kFastThreads - 1) / kFastThreads;
    if (units > 0x7ffffff0ll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
    B200Q_DISPATCH_FTYPE(ftype, rc = host_launch("qk_norm_rope_kernel launch", B200Q_NORM_ROWS(qk_norm_rope_rows_kernel), dim3(static_cast<unsigned>(blocks)),
                                                 kFastThreads, 0, cs, 1, a, split));
  } else {
    const long long blocks = (static_cast<long long>(t) * (hq + hk) + kNormWarps - 1) / kNormWarps;
    if (blocks > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
    B200Q_DISPATCH_FTYPE(ftype, rc = host_launch("qk_norm_rope_kernel launch", qk_norm_rope_kernel<T>, dim3(static_cast<unsigned>(blocks)),
                                                 kNormWarps * 32, 0, cs, 1, a));
  }
  if (rc == B200Q_OK) host_set_path(18);
  return rc;
}

extern "C" int b200q_qk_norm_rope_bprop(const b200q_qk_norm_args* args, void* stream) {
  NormArgs a{};
  int sms = 0;
  int rc = norm_args(args, &a, &sms);
  if (rc) return rc;
  const int ftype = args->ftype, t = a.t, hq = args->hq, hk = args->hk, d = a.d;
  if (t > 0 && ((hq && !args->q_grad) || (hk && !args->k_grad)))
    return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if ((rc = host_device(&sms, &a.err))) return rc;  // no tokens still mean weight gradients of zero
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const int size = ftype == B200Q_F32 ? 4 : 2;
  const int lanes = row_lanes(a, size, true);
  const Split split = split_heads(a, lanes ? lanes : 32, sms);
  const long long units = static_cast<long long>(t) * (lanes ? static_cast<int>(split.parts.d) : hq + hk);
  if (units > 0x7f000000ll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
  const int units_per_block = lanes ? kFastThreads / lanes : kNormWarps;
  const int room = static_cast<int>(kScratchBytes / (2 * d * sizeof(float)));  // at least 1024 blocks' partial sums
  const int blocks = static_cast<int>(
      std::max(1ll, std::min<long long>((units + units_per_block - 1) / units_per_block, std::min(sms * 4, room))));
  ScratchHold scratch;  // until both kernels are in the stream
  if ((rc = host_scratch(cs, &scratch))) return rc;
  a.partial = static_cast<float*>(scratch.bytes);
  const size_t smem = static_cast<size_t>(kNormWarps) * 2 * d * sizeof(float);
  B200Q_DISPATCH_FTYPE(ftype, {
    if (lanes) {
      rc = host_launch("qk_norm_rope_bprop_kernel launch", B200Q_NORM_ROWS(qk_norm_rope_bprop_rows_kernel), dim3(blocks),
                       kFastThreads, 0, cs, 1, a, split, static_cast<uint32_t>(units));
    } else {
      if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(qk_norm_rope_bprop_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
        if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(qk_norm_rope_bprop_kernel)");
      }
      rc = host_launch("qk_norm_rope_bprop_kernel launch", qk_norm_rope_bprop_kernel<T>, dim3(blocks), kNormWarps * 32,
                       smem, cs, 1, a);
    }
    if (rc) return rc;
    rc = host_launch("norm_weight_grad_kernel launch", norm_weight_grad_kernel<T>, dim3((2 * d + 31) / 32), 1024, 0, cs, 1,
                     a.partial, blocks, d, static_cast<T*>(args->q_w_grad), static_cast<T*>(args->k_w_grad));
  });
  scratch.launched();
  if (rc == B200Q_OK) host_set_path(18);
  return rc;
}
