// Linear layers with 4-bit weights and group scales (b200q_linear_w4).
#include "host.h"
#include "lowbit.cuh"

namespace b200q {
namespace {

struct W4Args {
  const void* x;
  long long ldx;
  const uint8_t* codes;
  const __nv_bfloat16* scales;
  const uint8_t* zeros;
  const void* bias;
  void* y;
  long long ldy;
  int m, n, k, group;
};

constexpr int kRowsX = 4;

// One warp per weight row: y[m][n] = sum over the lanes' 8-code words of (c - z) s x[m].
template <typename T>
__global__ void linear_w4_kernel(W4Args a) {
  const int n = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (n >= a.n) return;
  const int words = (a.k + 7) / 8;
  const size_t pitch = static_cast<size_t>((a.k + 31) / 32) * 4;
  const uint32_t* row = reinterpret_cast<const uint32_t*>(a.codes) + n * pitch;
  const T* x = static_cast<const T*>(a.x);
  const int m0 = blockIdx.y * kRowsX;
  float acc[kRowsX] = {};
  for (int w = lane; w < words; w += 32) {
    const uint32_t c = row[w];
    const size_t g = static_cast<size_t>(w * 8 / a.group) * a.n + n;
    const float s = __bfloat162float(a.scales[g]), z = a.zeros ? static_cast<float>(a.zeros[g]) : 8.0f;
    for (int j = 0; j < 8; ++j) {
      const int k = w * 8 + j;
      if (k >= a.k) break;
      const float v = (static_cast<float>((c >> (4 * j)) & 15u) - z) * s;
      for (int i = 0; i < kRowsX; ++i)
        if (m0 + i < a.m) acc[i] += v * to_f32(x[(m0 + i) * a.ldx + k]);
    }
  }
  for (int i = 0; i < kRowsX; ++i) {
    const float v = warp_sum(acc[i]);
    if (lane == 0 && m0 + i < a.m)
      static_cast<T*>(a.y)[(m0 + i) * a.ldy + n] =
          from_f32<T>(a.bias ? v + to_f32(static_cast<const T*>(a.bias)[n]) : v);
  }
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_linear_w4(const void* x, long long ldx, const uint8_t* codes, const void* scales,
                               const uint8_t* zeros, const void* bias, void* y, long long ldy, int ftype, int m, int n,
                               int k, int group, void* stream) {
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (m < 0 || n < 0 || k < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative linear dimension");
  if (group != 32 && group != 64 && group != 128)
    return host_fail(B200Q_ERR_INVALID_ARG, "weight group must be 32, 64 or 128, got %d", group);
  if (m == 0 || n == 0) return B200Q_OK;
  if (!y || (k > 0 && (!x || !codes || !scales))) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if ((m > 1 && ldx < k) || (m > 1 && ldy < n)) return host_fail(B200Q_ERR_INVALID_ARG, "row stride below row length");
  if (reinterpret_cast<uintptr_t>(codes) & 15u)
    return host_fail(B200Q_ERR_INVALID_ARG, "4-bit weight codes must be 16-byte aligned");
  if (n > (1 << 28) || k > (1 << 28) || m > (1 << 20)) return host_fail(B200Q_ERR_UNSUPPORTED, "linear too large");
  W4Args a{x, ldx, codes, static_cast<const __nv_bfloat16*>(scales), zeros, bias, y, ldy, m, n, k, group};
  const dim3 grid((n + 7) / 8, (m + kRowsX - 1) / kRowsX);
  if (grid.y > 65535) return host_fail(B200Q_ERR_UNSUPPORTED, "linear too large");
  B200Q_DISPATCH_FTYPE(ftype, (linear_w4_kernel<T><<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a)));
  const int rc = host_check_launch("linear_w4_kernel launch");
  if (rc == B200Q_OK) host_set_path(17);
  return rc;
}
