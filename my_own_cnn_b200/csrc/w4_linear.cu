// Linear layers with 4-bit weights and group scales (b200q_linear_w4).
//
//   y[m][n] = sum_g s[g][n] (sum_{k in g} c[n][k] x[m][k]  -  z[g][n] sum_{k in g} x[m][k])
//
// Bytes bound it: K / 2 of codes and 2 or 3 per group for each weight row.  The codes are the 16-row operand A of
// m16n8k16 (weight rows x K) and up to 16 rows of x its 8 columns, once or twice; m16n8k16 from registers because a
// code leaves its word as an operand in about one instruction, while tcgen05 operands would have to be written to
// shared memory first, four times the bytes that were read.
//
// A block owns kRowsW rows and one slice of K; the blocks of a cluster have the same rows and the other slices, and
// add their sums up through each other's shared memory in a fixed order.  Each warp streams its 32 rows through a
// ring of its own (kStages steps of 256 columns, 16-byte asynchronous copies), so nothing but x is shared:
// x lies in shared memory in the order of operand B, put there once per kilobyte or so of every row.
//
// How a lane's word of 8 codes becomes operands: pairs (0,4) (1,5) (2,6) (3,7) by shift and mask, with
//   fp16: the code in the low bits of an fp16 is the subnormal code * 2^-24, exactly; 2^24 goes into the scale;
//   bf16: under the exponent of 128 it is 128 + code; the 128 is taken off with the zero point, as (128 + z) sum x;
//   fp32: 128 + code less 128 + z, exactly, and x as three bf16 terms, which hold all its 24 bits.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "host.h"
#include "lowbit.cuh"

namespace b200q {
namespace {

struct W4Args {
  const void* x;
  long long ldx;
  const uint8_t* codes;
  const uint16_t* scales;  // bf16 bits
  const uint8_t* zeros;
  const void* bias;
  void* y;
  long long ldy;
  int m, n, k;
  int steps;        // of the whole K
  int slice;        // steps of a block
  int phase;        // steps whose x is in shared memory at a time
  int x_vec;        // x rows may be read 16 bytes at a time
};

constexpr int kWarps = 4;
constexpr int kRowsW = 32 * kWarps;  // weight rows of a block
constexpr int kStep = 256;           // columns of a step: 128 bytes of codes per row
constexpr int kStages = 4;
constexpr int kRing = kWarps * kStages * 32 * (kStep / 2);
constexpr int kXBytes = 36 * 1024;   // for x: with the ring, two blocks an SM
constexpr int kMaxSplit = 8;

template <typename T>
struct Terms {
  static constexpr int n = 1;
};
template <>
struct Terms<float> {
  static constexpr int n = 3;
};

// Shared memory: the rings, the sums [8 NT][kRowsW], x, and x's sums per group.
template <int G, int NT>
struct Layout {
  static constexpr int kSums = kRing, kX = kSums + 8 * NT * kRowsW * 4, kXSum = kX + kXBytes;
  static constexpr int kBytes = kXSum + kXBytes / (2 * G) * 2 * 4 + 64;
};

// Where 16-byte piece `piece` of row `row` of a step lies: lanes (g, t) that read pieces of 4, 8 or 16 bytes at
// row g, t pieces on, touch every bank once.
__device__ __forceinline__ int piece_at(int row, int piece) {
  const int flip = (row & 1) << 2 | (row & 2) | (row >> 2 & 1);
  return row * (kStep / 2) + ((piece ^ flip) << 4);
}

__device__ __forceinline__ float peer_load(uint32_t addr, int rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Puts columns [k0, k0 + columns) of up to 8 NT rows of x into shared memory as operand B, and the rows' sums over
// each group beside it (fp32 calls do without).
template <typename T, int G>
__device__ __forceinline__ void stage_x(const W4Args& a, uint4* xs, float* xsum, int m0, int rows, int k0, int columns) {
  constexpr int kTerms = Terms<T>::n, kWords = G / 32;
  const int chunks = columns / 8;
  for (int i = threadIdx.x; i < chunks * rows; i += kWarps * 32) {
    const int m = i / chunks, q = i % chunks, k = k0 + 8 * q;
    const T* from = static_cast<const T*>(a.x) + (m0 + m) * a.ldx + k;
    float v[8];
    if (a.x_vec && k + 8 <= a.k) {
      T raw[8];
#pragma unroll
      for (int b = 0; b < static_cast<int>(sizeof(raw)) / 16; ++b)
        reinterpret_cast<uint4*>(raw)[b] = __ldg(reinterpret_cast<const uint4*>(from) + b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f32(raw[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < a.k ? to_f32(from[j]) : 0.0f;
    }
    // thread t of a quad owns G / 4 columns of a group, kWords words of 8
    const int group = q / (G / 8), t = q % (G / 8) / kWords, word = q % kWords;
    const int block = group * kWords + word;
    if constexpr (kTerms == 1) {
      float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
#pragma unroll
      for (int o = 1; o < G / 8; o <<= 1) sum += __shfl_xor_sync(~0u, sum, o);
      if (q % (G / 8) == 0) xsum[group * ((rows + 1) & ~1) + m] = sum;
    }
#pragma unroll
    for (int term = 0; term < kTerms; ++term) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value) {
          w[j] = pack_f16(v[j], v[j + 4]);
        } else {
          w[j] = pack_bf16(v[j], v[j + 4]);
          v[j] -= __uint_as_float(w[j] << 16);
          v[j + 4] -= __uint_as_float(w[j] & 0xFFFF0000u);
        }
      }
      xs[((block * kTerms + term) * rows + m) * 4 + t] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <typename T, int G, int NT>
__global__ void __launch_bounds__(kWarps * 32) linear_w4_kernel(W4Args a) {
  constexpr bool kHalf = std::is_same<T, __half>::value, kF32 = std::is_same<T, float>::value;
  constexpr int kTerms = Terms<T>::n, kWords = G / 32, kGroups = kStep / G;
  extern __shared__ __align__(128) uint8_t smem[];
  float* const sums = reinterpret_cast<float*>(smem + Layout<G, NT>::kSums);
  uint4* const xs = reinterpret_cast<uint4*>(smem + Layout<G, NT>::kX);
  float* const xsum = reinterpret_cast<float*>(smem + Layout<G, NT>::kXSum);  // [group][rows, made even]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int splits = max(1, (a.steps + a.slice - 1) / a.slice);  // the cluster
  const int rank = blockIdx.x % splits, n0 = blockIdx.x / splits * kRowsW;
  const int m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, a.m - m0);
  const int step0 = rank * a.slice, steps = min(a.slice, a.steps - step0);

  // copies: lane l brings piece l % 8 of rows l / 8, 4 rows on each time; rows past the last repeat it
  const long long pitch = static_cast<long long>((a.k + 31) / 32) * 16;
  const uint32_t ring = shared_address(smem) + warp * (kStages * 32 * (kStep / 2));
  const int piece = lane % 8;
  const int row0 = n0 + warp * 32;
  auto load_step = [&](int s) {
    const long long at = static_cast<long long>(step0 + s) * (kStep / 2) + piece * 16;
    const uint32_t to = ring + (s % kStages) * (32 * (kStep / 2));
    if (at < pitch) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = j * 4 + lane / 8;
        copy_async<16>(to + piece_at(r, piece), a.codes + min(row0 + r, a.n - 1) * pitch + at);
      }
    }
  };
  // scales and zero points: lane l holds those of row l, two steps ahead of their use
  const int my_row = min(row0 + lane, a.n - 1), groups = (a.k + G - 1) / G;
  uint32_t scale[3][kGroups], zero[3][kGroups];
  auto load_params = [&](int s, uint32_t (&sc)[kGroups], uint32_t (&zp)[kGroups]) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const long long at = static_cast<long long>(min((step0 + s) * kGroups + i, groups - 1)) * a.n + my_row;
      sc[i] = __ldg(a.scales + at);
      zp[i] = a.zeros ? __ldg(a.zeros + at) : 8u;
    }
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (s < steps) load_step(s);
    copy_commit();
  }
  if (steps > 0) {
    load_params(0, scale[0], zero[0]);
    load_params(1, scale[1], zero[1]);
  }

  float acc[2][NT][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[mt][n][0] = acc[mt][n][1] = acc[mt][n][2] = acc[mt][n][3] = 0.0f;

  for (int s = 0; s < steps; ++s) {
    if (s % a.phase == 0) {
      if (s) __syncthreads();
      stage_x<T, G>(a, xs, xsum, m0, rows, (step0 + s) * kStep, min(a.phase, steps - s) * kStep);
      __syncthreads();
    }
    copy_wait<kStages - 2>();
    __syncwarp();
    if (s + kStages - 1 < steps) load_step(s + kStages - 1);
    copy_commit();
    load_params(s + 2, scale[2], zero[2]);
    const uint8_t* stage = smem + warp * (kStages * 32 * (kStep / 2)) + (s % kStages) * (32 * (kStep / 2));
    const int block0 = s % a.phase * (kStep / 32);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      float part[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int n = 0; n < NT; ++n) part[mt][n][0] = part[mt][n][1] = part[mt][n][2] = part[mt][n][3] = 0.0f;
      uint32_t w[4][kWords];  // rows g, g + 8, g + 16, g + 24
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = i * (G / 2) + t * (G / 8);  // byte of the row
        const uint8_t* p = stage + piece_at(r * 8 + g, at / 16) + at % 16;
        if constexpr (kWords == 1) {
          w[r][0] = *reinterpret_cast<const uint32_t*>(p);
        } else if constexpr (kWords == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(p);
          w[r][0] = v.x, w[r][1] = v.y;
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(p);
          w[r][0] = v.x, w[r][1] = v.y, w[r][2] = v.z, w[r][3] = v.w;
        }
      }
      uint32_t par[4];  // scale bits, zero point << 16
#pragma unroll
      for (int r = 0; r < 4; ++r) par[r] = __shfl_sync(~0u, scale[0][i] | zero[0][i] << 16, r * 8 + g);
      uint32_t zpair[4];
      if constexpr (kF32) {
#pragma unroll
        for (int r = 0; r < 4; ++r) zpair[r] = (par[r] >> 16) * 0x00010001u + 0x43004300u;
      }
#pragma unroll
      for (int word = 0; word < kWords; ++word) {
        uint4 b[kTerms][NT];
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            b[term][n] = n * 8 + g < rows ? xs[(((block0 + i * kWords + word) * kTerms + term) * rows + n * 8 + g) * 4 + t]
                                          : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t c[2][4];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t v = w[2 * mt + u][word] >> (4 * j);
              if constexpr (kHalf) {
                c[u][j] = v & 0x000F000Fu;
              } else {
                c[u][j] = and_or(v, 0x000F000Fu, 0x43004300u);
                if constexpr (kF32) c[u][j] = sub_bf16x2(c[u][j], zpair[2 * mt + u]);
              }
            }
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (kHalf) {
                mma_f16(part[mt][n], c[0][0], c[1][0], c[0][1], c[1][1], b[term][n].x, b[term][n].y);
                mma_f16(part[mt][n], c[0][2], c[1][2], c[0][3], c[1][3], b[term][n].z, b[term][n].w);
              } else {
                mma_bf16(part[mt][n], c[0][0], c[1][0], c[0][1], c[1][1], b[term][n].x, b[term][n].y);
                mma_bf16(part[mt][n], c[0][2], c[1][2], c[0][3], c[1][3], b[term][n].z, b[term][n].w);
              }
            }
        }
      }
      // the group's scale, and its zero point times the sum of x (columns 2t, 2t + 1)
      const int group = block0 / kWords + i;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float2 sx = make_float2(0.0f, 0.0f);
        if constexpr (!kF32) sx = *reinterpret_cast<const float2*>(xsum + group * ((rows + 1) & ~1) + n * 8 + 2 * t);
        if constexpr (kHalf) sx.x *= 1.0f / 16777216.0f, sx.y *= 1.0f / 16777216.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float sc = __uint_as_float(par[r] << 16);
          const float zr = static_cast<float>(par[r] >> 16) + (kHalf ? 0.0f : 128.0f);
          float* p = part[r / 2][n] + r % 2 * 2;
          float* to = acc[r / 2][n] + r % 2 * 2;
          to[0] = fmaf(sc, kF32 ? p[0] : fmaf(-zr, sx.x, p[0]), to[0]);
          to[1] = fmaf(sc, kF32 ? p[1] : fmaf(-zr, sx.y, p[1]), to[1]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      scale[0][i] = scale[1][i], scale[1][i] = scale[2][i];
      zero[0][i] = zero[1][i], zero[1][i] = zero[2][i];
    }
  }
  copy_wait<0>();

#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sums[(n * 8 + 2 * t + e % 2) * kRowsW + warp * 32 + mt * 16 + e / 2 * 8 + g] =
            kHalf ? acc[mt][n][e] * 16777216.0f : acc[mt][n][e];
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  // block `rank` of the cluster adds up its share of the rows
  const int share = (kRowsW + splits - 1) / splits, from = rank * share, wide = min(share, kRowsW - from);
  const uint32_t mine = shared_address(sums);
  for (int i = threadIdx.x; i < wide * rows; i += kWarps * 32) {
    const int m = i / wide, r = from + i % wide, n = n0 + r;
    if (n >= a.n) continue;
    float v = 0.0f;
    if (splits > 1) {
      for (int j = 0; j < splits; ++j) v += peer_load(mine + (m * kRowsW + r) * 4, j);
    } else {
      v = sums[m * kRowsW + r];
    }
    if (a.bias) v += to_f32(static_cast<const T*>(a.bias)[n]);
    static_cast<T*>(a.y)[(m0 + m) * a.ldy + n] = from_f32<T>(v);
  }
  if (splits > 1) cluster_sync();  // a block's sums stay until all have read them
}

template <typename T, int G, int NT>
int launch_linear(W4Args a, int sms, cudaStream_t stream) {
  constexpr int kSmem = Layout<G, NT>::kBytes;
  auto kernel = linear_w4_kernel<T, G, NT>;
  static std::atomic<bool> ready{false};
  if (!ready.load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(linear_w4_kernel)");
    ready.store(true, std::memory_order_relaxed);
  }
  // K is split so that two blocks an SM are busy, and no further: fewer, longer streams read faster
  const int tiles = (a.n + kRowsW - 1) / kRowsW, passes = (a.m + 8 * NT - 1) / (8 * NT);
  a.steps = (a.k + kStep - 1) / kStep;
  const int want = std::max(1, std::min(kMaxSplit, static_cast<int>(2ll * sms / (static_cast<long long>(tiles) * passes))));
  a.slice = std::max(1, (a.steps + want - 1) / want);
  const int splits = std::max(1, (a.steps + a.slice - 1) / a.slice);
  const int rows = std::min(a.m, 8 * NT);
  a.phase = std::max(1, std::min(a.slice, kXBytes / (rows * kStep * 2 * Terms<T>::n)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles * splits, passes);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {static_cast<unsigned>(splits), 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) return host_cuda_fail(e, "linear_w4_kernel launch");
  return host_check_launch("linear_w4_kernel launch");
}

template <typename T, int G>
int launch_linear_rows(const W4Args& a, int sms, cudaStream_t stream) {
  return a.m <= 8 ? launch_linear<T, G, 1>(a, sms, stream) : launch_linear<T, G, 2>(a, sms, stream);
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
  if (n > (1 << 28) || k > (1 << 28) || m > (1 << 19)) return host_fail(B200Q_ERR_UNSUPPORTED, "linear too large");
  int sms = 0, *err = nullptr;
  int rc = host_device(&sms, &err);
  if (rc) return rc;
  W4Args a{x, ldx, codes, static_cast<const uint16_t*>(scales), zeros, bias, y, ldy, m, n, k};
  const size_t size = ftype == B200Q_F32 ? 4 : 2;
  a.x_vec = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && (m == 1 || ldx * size % 16 == 0);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  B200Q_DISPATCH_FTYPE(ftype, rc = group == 32   ? launch_linear_rows<T, 32>(a, sms, cs)
                                   : group == 64 ? launch_linear_rows<T, 64>(a, sms, cs)
                                                 : launch_linear_rows<T, 128>(a, sms, cs));
  if (rc == B200Q_OK) host_set_path(17);
  return rc;
}
