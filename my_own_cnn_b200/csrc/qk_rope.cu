// Per-head RMS norm of queries and keys with the position rotation, and its gradient
// (b200q_qk_norm_rope, b200q_qk_norm_rope_bprop).
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

template <typename T>
__global__ void norm_weight_grad_kernel(const float* partial, int blocks, int d, T* dqw, T* dkw) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= 2 * d) return;
  float v = 0.0f;
  for (int b = 0; b < blocks; ++b) v += partial[static_cast<size_t>(b) * 2 * d + i];
  T* out = i < d ? dqw : dkw;
  if (out) out[i % d] = from_f32<T>(v);
}

int check_norm(const void* q, const void* k, const float* table, int positions, const int32_t* pos, int ftype, int t,
               int hq, int hk, int d, int rot) {
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (t < 0 || hq < 0 || hk < 0 || d <= 0) return host_fail(B200Q_ERR_INVALID_ARG, "bad head dimensions");
  if (rot < 0 || rot > d || rot % 2)
    return host_fail(B200Q_ERR_INVALID_ARG, "rotated channels must be even and at most %d, got %d", d, rot);
  if (d > 1024) return host_fail(B200Q_ERR_UNSUPPORTED, "heads of more than 1024 channels");
  if (hq + hk > (1 << 20)) return host_fail(B200Q_ERR_UNSUPPORTED, "too many heads");
  if (t == 0) return B200Q_OK;
  if ((hq && !q) || (hk && !k)) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (rot && (!table || !pos || positions <= 0))
    return host_fail(B200Q_ERR_INVALID_ARG, "a rotation needs its table and positions");
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_qk_norm_rope(const void* q, long long q_ts, long long q_hs, const void* k, long long k_ts,
                                  long long k_hs, const void* q_w, const void* k_w, const float* table, int positions,
                                  const int32_t* pos, void* q_out, long long qo_ts, long long qo_hs, void* k_out,
                                  long long ko_ts, long long ko_hs, int ftype, int t, int hq, int hk, int d, int rot,
                                  int interleaved, float eps, void* stream) {
  int rc = check_norm(q, k, table, positions, pos, ftype, t, hq, hk, d, rot);
  if (rc) return rc;
  if (t == 0 || hq + hk == 0) return B200Q_OK;
  if ((hq && !q_out) || (hk && !k_out)) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  NormArgs a{};
  int sms = 0;
  if ((rc = host_device(&sms, &a.err))) return rc;
  a.side[0] = {q, q_ts, q_hs, q_w, q_out, qo_ts, qo_hs, nullptr, hq};
  a.side[1] = {k, k_ts, k_hs, k_w, k_out, ko_ts, ko_hs, nullptr, hk};
  a.table = table;
  a.pos = pos;
  a.positions = positions;
  a.t = t;
  a.d = d;
  a.rot = rot;
  a.interleaved = interleaved;
  a.eps = eps;
  const long long blocks = (static_cast<long long>(t) * (hq + hk) + kNormWarps - 1) / kNormWarps;
  if (blocks > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
  B200Q_DISPATCH_FTYPE(ftype, (qk_norm_rope_kernel<T><<<static_cast<int>(blocks), kNormWarps * 32, 0,
                                                        static_cast<cudaStream_t>(stream)>>>(a)));
  rc = host_check_launch("qk_norm_rope_kernel launch");
  if (rc == B200Q_OK) host_set_path(18);
  return rc;
}

extern "C" int b200q_qk_norm_rope_bprop(const void* dq_out, const void* dk_out, const void* q, long long q_ts,
                                        long long q_hs, const void* k, long long k_ts, long long k_hs, const void* q_w,
                                        const void* k_w, const float* table, int positions, const int32_t* pos,
                                        void* dq, void* dk, void* dq_w, void* dk_w, int ftype, int t, int hq, int hk,
                                        int d, int rot, int interleaved, float eps, void* stream) {
  int rc = check_norm(q, k, table, positions, pos, ftype, t, hq, hk, d, rot);
  if (rc) return rc;
  if (t > 0 && ((hq && (!dq_out || !dq)) || (hk && (!dk_out || !dk))))
    return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  NormArgs a{};
  int sms = 0;
  if ((rc = host_device(&sms, &a.err))) return rc;
  a.side[0] = {q, q_ts, q_hs, q_w, dq, 0, 0, dq_out, hq};
  a.side[1] = {k, k_ts, k_hs, k_w, dk, 0, 0, dk_out, hk};
  a.table = table;
  a.pos = pos;
  a.positions = positions;
  a.t = t;
  a.d = d;
  a.rot = rot;
  a.interleaved = interleaved;
  a.eps = eps;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const long long want = (static_cast<long long>(t) * (hq + hk) + kNormWarps - 1) / kNormWarps;
  const int blocks = static_cast<int>(std::max(1ll, std::min<long long>(want, sms * 4)));
  void* ws = nullptr;
  if ((rc = host_workspace(static_cast<size_t>(blocks) * 2 * d * sizeof(float), cs, &ws))) return rc;
  a.partial = static_cast<float*>(ws);
  const size_t smem = static_cast<size_t>(kNormWarps) * 2 * d * sizeof(float);
  B200Q_DISPATCH_FTYPE(ftype, {
    if (smem > 48 * 1024) {
      cudaError_t e = cudaFuncSetAttribute(qk_norm_rope_bprop_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(smem));
      if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(qk_norm_rope_bprop_kernel)");
    }
    qk_norm_rope_bprop_kernel<T><<<blocks, kNormWarps * 32, smem, cs>>>(a);
    if ((rc = host_check_launch("qk_norm_rope_bprop_kernel launch"))) return rc;
    norm_weight_grad_kernel<T><<<(2 * d + 127) / 128, 128, 0, cs>>>(a.partial, blocks, d, static_cast<T*>(dq_w),
                                                                  static_cast<T*>(dk_w));
  });
  rc = host_check_launch("norm_weight_grad_kernel launch");
  if (rc == B200Q_OK) host_set_path(18);
  return rc;
}
