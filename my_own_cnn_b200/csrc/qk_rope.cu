// Per-head RMS norm of queries and keys with the position rotation, and its gradient
// (b200q_qk_norm_rope, b200q_qk_norm_rope_bprop).
//
//   n = x r w, r = (mean x^2 + eps)^-1/2;  y = R(pos) n
//   dn = R^T dy;  dw = sum dn x r;  with v = dn w: dx = r (v - x r^2 mean(v x))
//
// Bytes bound both: x in, y out; the gradient reads x and dy and writes dx.  A row of 64, 128 or 256 channels lies
// in the registers of 8 to 32 lanes, 16 bytes or D / 32 channels each, from one read to one write: the mean is a
// few shuffles, a rotation partner one more.  A group of lanes takes several heads of one token, so that it
// reads the token's cosines and sines once, and has kUnroll rows on their way at a time.  Other head sizes, rotations
// that are no power of two and unaligned rows go one warp per row through strided loops.
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

// Rows of D channels in LPR lanes of V channels.
template <typename T, int D>
struct RowShape {
  static constexpr int V = 16 / sizeof(T) > D / 32 ? 16 / sizeof(T) : D / 32;
  static constexpr int LPR = D / V;
};
constexpr int kFastThreads = 128;
constexpr int kUnroll = 4;

template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, bool ok, T (&v)[V]) {
  uint4* to = reinterpret_cast<uint4*>(v);
#pragma unroll
  for (int i = 0; i < static_cast<int>(V * sizeof(T) / 16); ++i)
    to[i] = ok ? *(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const float (&v)[V]) {
  alignas(16) T out[V];
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = from_f32<T>(v[j]);
#pragma unroll
  for (int i = 0; i < static_cast<int>(V * sizeof(T) / 16); ++i)
    *(reinterpret_cast<uint4*>(p) + i) = reinterpret_cast<const uint4*>(out)[i];
}

// The rotation of a lane's V channels: y = x c + (partner) s, where the partner is the channel rot / 2 away, in lane
// `lane ^ dist`, or the neighbour in the lane itself (interleaved).  The sine carries the sign.
template <int V>
struct Rotation {
  float c[V], s[V];
  int dist;
  bool interleaved;

  // Lane l of a row; `row` null: no rotation.
  __device__ __forceinline__ void load(const NormArgs& a, const float* row, int l) {
    interleaved = a.interleaved;
    dist = interleaved ? 0 : a.rot / 2 / V;
    const int ch = l * V;
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = 1.0f, s[j] = 0.0f;
    if (!row || ch >= a.rot) return;
    if (interleaved) {
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        c[j] = c[j + 1] = __ldg(row + (ch + j) / 2);
        s[j + 1] = __ldg(row + a.rot / 2 + (ch + j) / 2);
        s[j] = -s[j + 1];
      }
    } else {
      const int at = ch & (a.rot / 2 - 1);
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 cv = __ldg(reinterpret_cast<const float4*>(row + at + j));
        const float4 sv = __ldg(reinterpret_cast<const float4*>(row + a.rot / 2 + at + j));
        c[j] = cv.x, c[j + 1] = cv.y, c[j + 2] = cv.z, c[j + 3] = cv.w;
        s[j] = sv.x, s[j + 1] = sv.y, s[j + 2] = sv.z, s[j + 3] = sv.w;
      }
      if (ch < a.rot / 2) {
#pragma unroll
        for (int j = 0; j < V; ++j) s[j] = -s[j];
      }
    }
  }
  // Every lane of the warp takes part.
  template <bool BACK>
  __device__ __forceinline__ void apply(float (&v)[V]) const {
    float other[V];
#pragma unroll
    for (int j = 0; j < V; ++j) other[j] = interleaved ? v[j ^ 1] : __shfl_xor_sync(~0u, v[j], dist);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = fmaf(other[j], BACK ? -s[j] : s[j], v[j] * c[j]);
  }
};

template <typename T, int V>
__device__ __forceinline__ void load_weights(const NormArgs& a, int which, int l, float (&w)[V]) {
  const T* p = static_cast<const T*>(a.side[which].w);
  if (p) {
    alignas(16) T raw[V];
    load_row<T, V>(p + l * V, true, raw);
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = to_f32(raw[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = 1.0f;
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// A group of LPR lanes takes `per` heads (queries first, then keys) of one token.
template <typename T, int D>
__global__ void __launch_bounds__(kFastThreads) qk_norm_rope_rows_kernel(NormArgs a, int per) {
  constexpr int V = RowShape<T, D>::V, LPR = RowShape<T, D>::LPR;
  const int l = threadIdx.x % LPR, hq = a.side[0].heads, heads = hq + a.side[1].heads;
  const int parts = (heads + per - 1) / per;
  const long long unit = static_cast<long long>(blockIdx.x) * (kFastThreads / LPR) + threadIdx.x / LPR;
  const int t = static_cast<int>(unit / parts);
  bool ok = t < a.t;
  const int begin = static_cast<int>(unit % parts) * per, end = ok ? min(heads, begin + per) : begin;
  const float* tab = nullptr;
  if (ok && a.rot) ok = (tab = table_row(a, t)) != nullptr;
  Rotation<V> rotation;
  bool known = false;  // the rotation is loaded behind the first rows
  for (int h0 = begin; __any_sync(~0u, h0 < end); h0 += kUnroll) {
    alignas(16) T raw[kUnroll][V];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u, which = h >= hq;
      const NormSide& s = a.side[which];
      load_row<T, V>(static_cast<const T*>(s.x) + t * s.ts + (h - (which ? hq : 0)) * s.hs + l * V, h < end, raw[u]);
    }
    if (!known) rotation.load(a, tab, l);
    known = true;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u, which = h >= hq;
      float v[V], w[V], sq = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[j] = to_f32(raw[u][j]);
        sq = fmaf(v[j], v[j], sq);
      }
      load_weights<T, V>(a, which, l, w);
      const float r = rsqrtf(row_sum<LPR>(sq) * (1.0f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = v[j] * r * w[j];
      rotation.template apply<false>(v);
      const NormSide& s = a.side[which];
      if (ok && h < end)
        store_row<T, V>(static_cast<T*>(s.y) + t * s.yts + (h - (which ? hq : 0)) * s.yhs + l * V, v);
    }
  }
}

// The gradient: groups of lanes walk over (token, head) rows, the weights' sums stay in registers.
template <typename T, int D>
__global__ void __launch_bounds__(kFastThreads) qk_norm_rope_bprop_rows_kernel(NormArgs a, int per) {
  constexpr int V = RowShape<T, D>::V, LPR = RowShape<T, D>::LPR, kGroups = kFastThreads / LPR;
  constexpr int kRowsAhead = V > 4 ? 2 : 4;
  __shared__ float sums[kGroups][2][D];
  const int l = threadIdx.x % LPR, group = threadIdx.x / LPR, hq = a.side[0].heads, heads = hq + a.side[1].heads;
  const int parts = (heads + per - 1) / per;
  const long long units = static_cast<long long>(a.t) * parts;
  float dw[2][V];
#pragma unroll
  for (int j = 0; j < V; ++j) dw[0][j] = dw[1][j] = 0.0f;
  for (long long first = static_cast<long long>(blockIdx.x) * kGroups; first < units;
       first += static_cast<long long>(gridDim.x) * kGroups) {
    const long long unit = first + group;
    const int t = static_cast<int>(unit / parts);
    bool ok = unit < units;
    const int begin = static_cast<int>(unit % parts) * per, end = ok ? min(heads, begin + per) : begin;
    const float* tab = nullptr;
    if (ok && a.rot) ok = (tab = table_row(a, t)) != nullptr;
    Rotation<V> rotation;
    bool known = false;
    for (int h0 = begin; __any_sync(~0u, h0 < end); h0 += kRowsAhead) {
      alignas(16) T raw[kRowsAhead][V], grad[kRowsAhead][V];
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        const int h = h0 + u, which = h >= hq, hh = h - (which ? hq : 0);
        const NormSide& s = a.side[which];
        load_row<T, V>(static_cast<const T*>(s.x) + t * s.ts + hh * s.hs + l * V, ok && h < end, raw[u]);
        load_row<T, V>(static_cast<const T*>(s.dy) + (static_cast<long long>(t) * s.heads + hh) * D + l * V, ok && h < end,
                       grad[u]);
      }
      if (!known) rotation.load(a, tab, l);
      known = true;
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        const int h = h0 + u, which = h >= hq, hh = h - (which ? hq : 0);
        const NormSide& s = a.side[which];
        float x[V], v[V], w[V], sq = 0.0f, vx = 0.0f;
        load_weights<T, V>(a, which, l, w);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = to_f32(raw[u][j]);
          v[j] = to_f32(grad[u][j]);
          sq = fmaf(x[j], x[j], sq);
        }
        rotation.template apply<true>(v);
        const float r = rsqrtf(row_sum<LPR>(sq) * (1.0f / D) + a.eps);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float add = ok && h < end ? v[j] * x[j] * r : 0.0f;
          dw[0][j] += which ? 0.0f : add;
          dw[1][j] += which ? add : 0.0f;
          v[j] *= w[j];
          vx = fmaf(v[j], x[j], vx);
        }
        const float k = r * r * (row_sum<LPR>(vx) * (1.0f / D));
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = r * fmaf(-k, x[j], v[j]);
        if (ok && h < end)
          store_row<T, V>(static_cast<T*>(s.y) + (static_cast<long long>(t) * s.heads + hh) * D + l * V, v);
      }
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int j = 0; j < V; ++j) sums[group][which][l * V + j] = dw[which][j];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kFastThreads) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < kGroups; ++j) v += (&sums[j][0][0])[i];
    a.partial[static_cast<size_t>(blockIdx.x) * 2 * D + i] = v;
  }
}

// Adds the blocks' weight gradients up in a fixed order: 32 columns a block, the partial sums shared out to 32 warps.
template <typename T>
__global__ void norm_weight_grad_kernel(const float* partial, int blocks, int d, T* dqw, T* dkw) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, i = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (i < 2 * d) {
#pragma unroll 4
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

// Whether the rows kernels take the call: d and rot in their shapes, and every row 16-byte aligned.
bool rows_fit(const NormArgs& a, int size, bool back) {
  const int v = std::max(16 / size, a.d / 32);
  if (a.d != 64 && a.d != 128 && a.d != 256) return false;
  if (a.rot && ((a.rot & (a.rot - 1)) || a.rot < 2 * v || (reinterpret_cast<uintptr_t>(a.table) & 15u))) return false;
  for (const NormSide& s : a.side) {
    uintptr_t bits = reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y) | reinterpret_cast<uintptr_t>(s.w);
    long long strides = s.ts | s.hs;
    if (back)
      bits |= reinterpret_cast<uintptr_t>(s.dy);
    else
      strides |= s.yts | s.yhs;
    if (s.heads && ((bits & 15u) || (strides * size) % 16)) return false;
  }
  return true;
}

// Heads of a token that one group of lanes takes: many when there are enough rows to fill the GPU with eights (the
// cosines are read less often), one when there are few (a row's latency is all there is).
int heads_per_group(const NormArgs& a, int lanes, int sms) {
  const long long lanes_of_all = static_cast<long long>(a.t) * (a.side[0].heads + a.side[1].heads) * lanes;
  const long long full = 1024ll * sms;
  return lanes_of_all >= 16 * full ? 8 : lanes_of_all >= 4 * full ? 4 : 1;
}

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
  if (rows_fit(a, size, false)) {
    const int lanes = d / std::max(16 / size, d / 32), per = heads_per_group(a, lanes, sms);
    const long long blocks = (static_cast<long long>(t) * ((hq + hk + per - 1) / per) * lanes + kFastThreads - 1) / kFastThreads;
    if (blocks > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
    B200Q_DISPATCH_FTYPE(ftype, (d == 64    ? qk_norm_rope_rows_kernel<T, 64>
                                 : d == 128 ? qk_norm_rope_rows_kernel<T, 128>
                                            : qk_norm_rope_rows_kernel<T, 256>)<<<static_cast<int>(blocks), kFastThreads, 0, cs>>>(a, per));
  } else {
    const long long blocks = (static_cast<long long>(t) * (hq + hk) + kNormWarps - 1) / kNormWarps;
    if (blocks > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
    B200Q_DISPATCH_FTYPE(ftype, (qk_norm_rope_kernel<T><<<static_cast<int>(blocks), kNormWarps * 32, 0, cs>>>(a)));
  }
  rc = host_check_launch("qk_norm_rope_kernel launch");
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
  const bool fast = rows_fit(a, size, true);
  const int lanes = fast ? d / std::max(16 / size, d / 32) : 32, per = fast ? heads_per_group(a, lanes, sms) : 1;
  const int threads = fast ? kFastThreads : kNormWarps * 32;
  const long long want = (static_cast<long long>(t) * ((hq + hk + per - 1) / per) * lanes + threads - 1) / threads;
  const int blocks = static_cast<int>(std::max(1ll, std::min<long long>(want, sms * (fast ? 8 : 4))));
  void* ws = nullptr;
  if ((rc = host_workspace(static_cast<size_t>(blocks) * 2 * d * sizeof(float), cs, &ws))) return rc;
  a.partial = static_cast<float*>(ws);
  const size_t smem = static_cast<size_t>(kNormWarps) * 2 * d * sizeof(float);
  B200Q_DISPATCH_FTYPE(ftype, {
    if (fast) {
      (d == 64    ? qk_norm_rope_bprop_rows_kernel<T, 64>
       : d == 128 ? qk_norm_rope_bprop_rows_kernel<T, 128>
                  : qk_norm_rope_bprop_rows_kernel<T, 256>)<<<blocks, kFastThreads, 0, cs>>>(a, per);
    } else {
      if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(qk_norm_rope_bprop_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
        if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(qk_norm_rope_bprop_kernel)");
      }
      qk_norm_rope_bprop_kernel<T><<<blocks, kNormWarps * 32, smem, cs>>>(a);
    }
    if ((rc = host_check_launch("qk_norm_rope_bprop_kernel launch"))) return rc;
    norm_weight_grad_kernel<T><<<(2 * d + 31) / 32, 1024, 0, cs>>>(a.partial, blocks, d, static_cast<T*>(args->q_w_grad),
                                                                 static_cast<T*>(args->k_w_grad));
  });
  rc = host_check_launch("norm_weight_grad_kernel launch");
  if (rc == B200Q_OK) host_set_path(18);
  return rc;
}
