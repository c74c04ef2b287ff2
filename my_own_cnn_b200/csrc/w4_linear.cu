// Linear layers with 4-bit weights and group scales (b200q_linear_w4).
//
//   y[m][n] = sum_g s[g][n] sum_{k in g} (c[n][k] - z[g][n]) x[m][k]
//
// Bytes bound it: K / 2 of codes and 2 or 3 per group for each weight row; and, as measured, the latency of its instructions
// with 16 warps an SM.  1 x 8192 x 8192 bf16: 11.3 us, 3.1 TB/s; 16 x 16384 x 8192: 35.3 us, 2.1 TB/s; 1 x 768 x 768: 3.0 us.
// The codes are the 16-row operand A of m16n8k16 (weight rows x K) and up to 16 rows of x its 8 columns, once or twice;
// m16n8k16 from registers because a code leaves its word as an operand in two instructions, while tcgen05
// operands would have to be written to shared memory first, four times the bytes that were read.
//   Operands: a nibble put into the low bits of the fp16 1024 is 1024 + code, and one place higher 1024 + 16 code; less the
//   same of the zero point it is exact and normal.  A word of 8 codes becomes four operands, the pairs (0,4) (1,5) (2,6) (3,7),
//   and every second value of x is divided by 16 instead.  x is scaled by a power of two per row and step to a maximum in
//   [2^14, 2^15), so that it fits fp16 whatever its type; fp32 becomes two fp16 terms (22 bits).
//   (The bare nibble, a subnormal, with the zero points' sum kept apart, saves the subtraction: 10.6 against 11.3 us for one
//   row of 8192 x 8192, 34.9 against 35.3 for 16 rows.  But the adder lines subnormals up by their exponent field and truncates
//   about 10 of the sum's bits, and where x has one sign the two sums are many times their difference: fp16 results after a
//   squared ReLU were off by 6e-5, all one way.)
//
// Each warp streams 32 rows through a ring of its own (16-byte asynchronous copies) in steps of kStep columns.  x is
// shared by the block's warps, in the order of operand B; the blocks of a cluster have the same rows and other slices
// of K, and add their sums up through each other's shared memory in a fixed order.
//   Several rows of x: a block owns 8 x 32 weight rows, so that x is brought in once per 32 KB of codes; while a
//   step is computed the next one's x is written to the other of two buffers, from registers that it was read into a
//   step before.
//   One row (and up to kFewRows, where there are few weight rows): a block owns 32 weight rows and its warps share out K: x is small enough to lie in shared memory whole, no
//   barrier is met between the first step and the last, and a cluster is needed only for few weight rows.
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
  int steps;  // of the whole K
  int slice;  // steps of a block
  int x_vec;  // x rows may be read 16 bytes at a time
};

constexpr int kWarps = 8;
constexpr int kFewRows = 4;
constexpr int kStep = 256;           // columns of a step: 128 bytes of codes per row
constexpr int kStage = 32 * (kStep / 2);
constexpr int kMaxSplit = 8;

// FEW: 0, or how many rows of x at most a block has that keeps all of them in shared memory.
// Shared memory: the rings (over them at the end the sums), then x: two steps of it, or (FEW) every step of the block's
// slice.  A step of x: operand B [block of 32 columns][term][row][t] 16 bytes, powers [row].
template <typename T, int G, int NT, int FEW>
struct Layout {
  static constexpr int kTerms = std::is_same<T, float>::value ? 2 : 1;
  static constexpr int kRowsX = FEW ? FEW : 8 * NT;    // rows of x that there is room for
  static constexpr int kRowsW = FEW ? 32 : 32 * kWarps;     // weight rows of a block
  static constexpr int kX = kStep * 2 * kTerms * kRowsX;
  static constexpr int kBuffer = (kX + kRowsX * 4 + 15) / 16 * 16;
  // Three stages where two blocks still fit an SM (228 KB, 1 KB of it taken per block); 16 rows of fp32 leave room for two:
  // 16 x 11000 x 12000 fp32 47 us, 69 with one block and three.
  static constexpr int kStages = FEW || kWarps * 3 * kStage + 2 * kBuffer > 113 * 1024 ? 2 : 3;
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kBuffers = FEW ? (46 * 1024) / kBuffer : 2;
  static constexpr int kBytes = kRing + kBuffers * kBuffer;
};

// Where 16-byte piece `piece` of row `row` of a step lies: lanes (g, t) that read pieces of 4, 8 or 16 bytes at
// row g, t pieces on, touch every bank once.
__device__ __forceinline__ int piece_at(int row, int piece) {
  const int flip = (row & 1) << 2 | (row & 2) | (row >> 2 & 1);
  return row * (kStep / 2) + ((piece ^ flip) << 4);
}

// 1024 + 16 z of 1024 + z, on two fp16 values; exact for every z below 256.
__device__ __forceinline__ uint32_t times_16(uint32_t v) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(16.0f), __float2half2_rn(-15360.0f));
  return *reinterpret_cast<const uint32_t*>(&r);
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

// One row's columns of a step on their way: lane l has columns 8 l to 8 l + 7.
template <typename T>
struct XRow {
  alignas(16) T v[8];

  __device__ __forceinline__ void load(const W4Args& a, int m, int k0) {
    const int k = k0 + threadIdx.x % 32 * 8;
    const T* from = static_cast<const T*>(a.x) + m * a.ldx + k;
    if (a.x_vec && k + 8 <= a.k) {
#pragma unroll
      for (int b = 0; b < static_cast<int>(sizeof(T)) / 2; ++b)
        reinterpret_cast<uint4*>(v)[b] = __ldg(reinterpret_cast<const uint4*>(from) + b);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < a.k ? from[j] : from_f32<T>(0.0f);
    }
  }

  // Into row m of a step's buffer; the whole warp takes part.
  template <int G, typename L>
  __device__ __forceinline__ void store(uint8_t* buffer, int m) const {
    constexpr int kWords = G / 32;
    uint4* const xs = reinterpret_cast<uint4*>(buffer);
    float* const xpower = reinterpret_cast<float*>(buffer + L::kX);
    const int q = threadIdx.x % 32;
    // thread t of a quad owns G / 4 columns of a group, kWords words of 8
    const int group = q / (G / 8), t = q % (G / 8) / kWords, block = group * kWords + q % kWords;
    float2 f[4];  // pairs (j, j + 4)
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = make_float2(to_f32(v[j]), to_f32(v[j + 4]));
      top = fmaxf(fmaxf(fabsf(f[j].x), fabsf(f[j].y)), top);
    }
    const Power p = power_for(warp_max(top));
    if (q == 0) xpower[m] = p.down;
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = mul2(f[j], both(p.up));
#pragma unroll
    for (int term = 0; term < L::kTerms; ++term) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = pack_f16(f[j].x, f[j].y);
        __half2& h = *reinterpret_cast<__half2*>(&w[j]);
        if (term + 1 < L::kTerms) {
          const float2 back = __half22float2(h);
          f[j] = make_float2(f[j].x - back.x, f[j].y - back.y);
        }
        if (j % 2) h = __hmul2(h, __float2half2_rn(0.0625f));
      }
      xs[((block * L::kTerms + term) * L::kRowsX + m) * 4 + t] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

template <typename T, int G, int NT, int FEW>
__global__ void __launch_bounds__(kWarps * 32, 2) linear_w4_kernel(W4Args a) {
  using L = Layout<T, G, NT, FEW>;
  constexpr int kTerms = L::kTerms, kWords = G / 32, kGroups = kStep / G, kStages = L::kStages, kRowsW = L::kRowsW;
  constexpr int kRowsX = L::kRowsX;
  extern __shared__ __align__(128) uint8_t smem[];
  wait_for_previous();
  uint8_t* const buffers = smem + L::kRing;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int splits = max(1, (a.steps + a.slice - 1) / a.slice);  // the cluster
  const int rank = blockIdx.x % splits, n0 = blockIdx.x / splits * kRowsW;
  const int m0 = blockIdx.y * kRowsX, rows = min(kRowsX, a.m - m0);
  // the block's steps are step0 to step0 + count; the warp's are its first, its first + stride, ...
  const int step0 = rank * a.slice, count = min(a.slice, a.steps - step0);
  constexpr int kStride = FEW ? kWarps : 1;
  const int first = step0 + (FEW ? warp : 0), steps = FEW ? (count - warp + kWarps - 1) / kWarps : count;

  // copies: lane l brings piece l % 8 of rows l / 8, l / 8 + 4, ...
  const long long pitch = static_cast<long long>((a.k + 31) / 32) * 16;
  const int row0 = n0 + (FEW ? 0 : warp * 32), here = min(32, a.n - row0) - lane / 8;  // rows past the last are left out
  const uint32_t ring = shared_address(smem) + warp * (kStages * kStage);
  const long long piece0 = static_cast<long long>(first) * (kStep / 2) + lane % 8 * 16;
  const uint8_t* const codes = a.codes + (row0 + lane / 8) * pitch + piece0;
  auto load_step = [&](int s, int slot) {
    const int at = s * kStride * (kStep / 2);
    if (piece0 + at < pitch) {
      const uint8_t* from = codes + at;
      const uint32_t to = ring + slot * kStage;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j * 4 < here) copy_async<16>(to + piece_at(j * 4 + lane / 8, lane % 8), from);
        from += 4 * pitch;
      }
    }
  };
  // scales and zero points: lane l holds those of row l, read a step before their use; past K's last group it repeats
  const int my_row = min(row0 + lane, a.n - 1), groups = (a.k + G - 1) / G;
  uint32_t scale[kGroups], zero[kGroups], next_scale[kGroups], next_zero[kGroups];
  auto load_params = [&](int s) {
    const int group0 = (first + s * kStride) * kGroups;
    const long long at = static_cast<long long>(group0) * a.n + my_row;
    const uint16_t* sp = a.scales + at;
    const uint8_t* zp = a.zeros + at;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      next_scale[i] = __ldg(sp);
      next_zero[i] = a.zeros ? __ldg(zp) : 8u;
      if (group0 + i + 1 < groups) sp += a.n, zp += a.n;
    }
  };

  // sums of products, [16 rows][8 columns][row g or g + 8] for columns 2t, 2t + 1
  float2 acc[2][NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[0][n][0] = acc[0][n][1] = acc[1][n][0] = acc[1][n][1] = both(0.0f);
  constexpr int kRowsWarp = FEW ? 4 : NT;  // rows of a step that a warp has on their way at a time
  XRow<T> x[kRowsWarp];
  auto load_x = [&](int step) {  // rows w, w + 8 of one step
#pragma unroll
    for (int i = 0; i < kRowsWarp; ++i)
      if (i * kWarps + warp < rows) x[i].load(a, m0 + i * kWarps + warp, (step0 + step) * kStep);
  };
  auto store_x = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < kRowsWarp; ++i)
      if (i * kWarps + warp < rows) x[i].template store<G, L>(buffers + buffer * L::kBuffer, i * kWarps + warp);
  };
  if constexpr (!FEW)
    if (steps > 0) load_x(0);  // before the codes: it is needed first
  if (steps > 0) load_params(0);
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (s < steps) load_step(s, s);
    copy_commit();
  }
  if constexpr (FEW) {  // every row of every step, dealt out to the warps
    for (int p0 = warp; p0 < rows * count; p0 += kWarps * kRowsWarp) {
#pragma unroll
      for (int i = 0; i < kRowsWarp; ++i) {
        const int p = p0 + i * kWarps;
        if (p < rows * count) x[i].load(a, m0 + p % rows, (step0 + p / rows) * kStep);
      }
#pragma unroll
      for (int i = 0; i < kRowsWarp; ++i) {
        const int p = p0 + i * kWarps;
        if (p < rows * count) x[i].template store<G, L>(buffers + p / rows * L::kBuffer, p % rows);
      }
    }
  } else {
    if (steps > 0) store_x(0);
    if (steps > 1) load_x(1);
  }
  __syncthreads();
  const int column = min(g, rows - 1);  // columns that no row of x has repeat one that has, and are not used

  int slot = 0, fill = kStages - 1;
  for (int s = 0; s < steps; ++s) {
    const uint8_t* const buffer = buffers + (FEW ? warp + s * kWarps : s & 1) * L::kBuffer;
    if constexpr (!FEW) {
      if (s + 1 < steps) store_x(~s & 1);
      if (s + 2 < steps) load_x(s + 2);
    }
    copy_wait<kStages - 2>();
    __syncwarp();
    if (s + kStages - 1 < steps) load_step(s + kStages - 1, fill);
    copy_commit();
#pragma unroll
    for (int i = 0; i < kGroups; ++i) scale[i] = next_scale[i] << 16, zero[i] = next_zero[i];
    if (s + 1 < steps) load_params(s + 1);
    const uint4* const xs = reinterpret_cast<const uint4*>(buffer);
    const float* const xpower = reinterpret_cast<const float*>(buffer + L::kX);
    const uint8_t* const stage = smem + warp * (kStages * kStage) + slot * kStage;
    float2 sum[2][NT][2];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
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
      constexpr uint32_t kMagic = 0x64006400u;  // two fp16 1024
      uint32_t zpair[4];  // 1024 + the rows' zero points, twice
#pragma unroll
      for (int r = 0; r < 4; ++r) zpair[r] = __shfl_sync(~0u, zero[i], r * 8 + g) * 0x00010001u | kMagic;
      float part[2][NT][4];
#pragma unroll
      for (int word = 0; word < kWords; ++word) {
        uint4 b[kTerms][NT];
#pragma unroll
        for (int term = 0; term < kTerms; ++term)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            b[term][n] = xs[(((i * kWords + word) * kTerms + term) * kRowsX + (FEW ? column : n * 8 + g)) * 4 + t];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t c[2][4];  // pairs (0,4) (1,5) (2,6) (3,7) of rows g and g + 8
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t v = w[2 * mt + u][word] >> (j / 2 * 8), mask = j % 2 ? 0x00F000F0u : 0x000F000Fu;
              c[u][j] = sub_f16x2(and_or(v, mask, kMagic), j % 2 ? times_16(zpair[2 * mt + u]) : zpair[2 * mt + u]);
            }
#pragma unroll
          for (int term = 0; term < kTerms; ++term)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (word == 0 && term == 0)
                mma_f16_first(part[mt][n], c[0][0], c[1][0], c[0][1], c[1][1], b[term][n].x, b[term][n].y);
              else
                mma_f16(part[mt][n], c[0][0], c[1][0], c[0][1], c[1][1], b[term][n].x, b[term][n].y);
              mma_f16(part[mt][n], c[0][2], c[1][2], c[0][3], c[1][3], b[term][n].z, b[term][n].w);
            }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float2 sc = both(__uint_as_float(__shfl_sync(~0u, scale[i], r * 8 + g)));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float* p = part[r / 2][n] + r % 2 * 2;
          float2& to = sum[r / 2][n][r % 2];
          to = i == 0 ? mul2(sc, make_float2(p[0], p[1])) : fma2(sc, make_float2(p[0], p[1]), to);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float2 p = *reinterpret_cast<const float2*>(xpower + (FEW ? 2 * t % kRowsX : n * 8 + 2 * t));
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) acc[mt][n][u] = fma2(p, sum[mt][n][u], acc[mt][n][u]);
    }
    slot = slot + 1 == kStages ? 0 : slot + 1;
    fill = fill + 1 == kStages ? 0 : fill + 1;
    if constexpr (!FEW) __syncthreads();  // this step's x has been read, the next one's is there
  }
  copy_wait<0>();
  if constexpr (FEW) __syncthreads();  // the rings are done with

  constexpr int kPitch = 36;  // of 32 weight rows: stores of rows 2 t, columns g touch every bank once
  static_assert(kWarps * kRowsX * kPitch * 4 <= L::kRing, "the sums lie over the rings");
  float* const all = reinterpret_cast<float*>(smem);  // [warp][kRowsX][kPitch]
  float* const sums = all + warp * (kRowsX * kPitch);
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (FEW && 2 * t >= kRowsX) continue;
        float* to = sums + (n * 8 + 2 * t) * kPitch + mt * 16 + u * 8 + g;
        to[0] = acc[mt][n][u].x;
        if (kRowsX > 1) to[kPitch] = acc[mt][n][u].y;
      }
  if (splits > 1)
    cluster_sync();
  else
    __syncthreads();
  // block `rank` of the cluster adds up its share of the weight rows, over the blocks and (FEW) their warps
  const int share = (kRowsW + splits - 1) / splits, from = rank * share, wide = max(0, min(share, kRowsW - from));
  const uint32_t mine = shared_address(all);
  for (int i = threadIdx.x; i < wide * rows; i += kWarps * 32) {
    const int m = i / wide, r = from + i % wide, n = n0 + r;
    if (n >= a.n) continue;
    const int at = (FEW ? 0 : r / 32 * (kRowsX * kPitch)) + m * kPitch + r % 32;
    float v = 0.0f;
    constexpr int kEach = FEW ? kWarps : 1;
    if (splits > 1) {
      constexpr int kTogether = 4;  // blocks whose sums are on their way at a time
      for (int j = 0; j < splits; j += kTogether) {
        float part[kTogether][kEach];
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
#pragma unroll
          for (int w = 0; w < kEach; ++w)
            part[u][w] = j + u < splits ? peer_load(mine + (at + w * (kRowsX * kPitch)) * 4, j + u) : 0.0f;
#pragma unroll
        for (int u = 0; u < kTogether; ++u)
#pragma unroll
          for (int w = 0; w < kEach; ++w) v += part[u][w];
      }
    } else {
#pragma unroll
      for (int w = 0; w < kEach; ++w) v += all[at + w * (kRowsX * kPitch)];
    }
    if (a.bias) v += to_f32(static_cast<const T*>(a.bias)[n]);
    static_cast<T*>(a.y)[(m0 + m) * a.ldy + n] = from_f32<T>(v);
  }
  if (splits > 1) cluster_sync();  // a block's sums stay until all have read them
}

template <typename T, int G, int NT, int FEW>
int launch_linear(W4Args a, int sms, int device, cudaStream_t stream) {
  using L = Layout<T, G, NT, FEW>;
  constexpr int kSmem = L::kBytes;
  auto kernel = linear_w4_kernel<T, G, NT, FEW>;
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[device].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(linear_w4_kernel)");
    ready[device].store(true, std::memory_order_relaxed);
  }
  // K is split so that two blocks an SM are busy (FEW: and every warp has a step), and no further: fewer, longer streams
  // read faster
  const int tiles = (a.n + L::kRowsW - 1) / L::kRowsW, passes = (a.m + L::kRowsX - 1) / L::kRowsX;
  a.steps = (a.k + kStep - 1) / kStep;
  int want = static_cast<int>(std::min<long long>(kMaxSplit, 2ll * sms / (static_cast<long long>(tiles) * passes)));
  if (FEW) want = std::max(std::min(want, a.steps / kWarps), (a.steps + L::kBuffers - 1) / L::kBuffers);
  want = std::max(1, want);
  a.slice = std::max(1, (a.steps + want - 1) / want);
  const int splits = std::max(1, (a.steps + a.slice - 1) / a.slice);
  return host_launch("linear_w4_kernel launch", kernel, dim3(tiles * splits, passes), kWarps * 32, kSmem, stream, splits, a);
}

template <typename T, int G>
int launch_linear_rows(const W4Args& a, int sms, int device, cudaStream_t stream) {
  // (In a graph, weights that L2 does not hold.)  One row of x: 1 x 8192 x 8192 bf16 11.9 us, 12.2 with blocks of 256 weight
  // rows; 1 x 16000 x 1000 8.2, 8.3 with kFewRows rows of room; 1 x 768 x 768 fp16 3.36 and 3.44.  Two to four: only while blocks of
  // 256, K split eight ways, would leave SMs idle (2 x 16000 x 1000 fp32 9.6 us, 16.8 with those, 4 x 16000 x 1000 bf16 10.3 and
  // 14.2, but 4 x 8192 x 8192 bf16 22.7 and 13.8: each block brings x in).
  if (a.m == 1 && a.k <= kMaxSplit * kStep * Layout<T, G, 1, 1>::kBuffers) return launch_linear<T, G, 1, 1>(a, sms, device, stream);
  if (a.m <= kFewRows && (a.n + 255) / 256 * kMaxSplit < sms && a.k <= kMaxSplit * kStep * Layout<T, G, 1, kFewRows>::kBuffers)
    return launch_linear<T, G, 1, kFewRows>(a, sms, device, stream);
  return a.m <= 8 ? launch_linear<T, G, 1, 0>(a, sms, device, stream) : launch_linear<T, G, 2, 0>(a, sms, device, stream);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_linear_w4(const b200q_linear_w4_args* p, void* stream) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const int ftype = p->ftype, m = p->m, n = p->n, k = p->k, group = p->group;
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (m < 0 || n < 0 || k < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative linear dimension");
  if (group != 32 && group != 64 && group != 128)
    return host_fail(B200Q_ERR_INVALID_ARG, "weight group must be 32, 64 or 128, got %d", group);
  if (m == 0 || n == 0) return B200Q_OK;
  if (!p->y || (k > 0 && (!p->x || !p->codes || !p->scales))) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (m > 1 && (p->ldx < k || p->ldy < n)) return host_fail(B200Q_ERR_INVALID_ARG, "row stride below row length");
  if (reinterpret_cast<uintptr_t>(p->codes) & 15u)
    return host_fail(B200Q_ERR_INVALID_ARG, "4-bit weight codes must be 16-byte aligned");
  if (n > (1 << 28) || k > (1 << 28) || m > (1 << 19)) return host_fail(B200Q_ERR_UNSUPPORTED, "linear too large");
  int sms = 0, device = 0, *err = nullptr;
  int rc = host_device(&sms, &err, &device);
  if (rc) return rc;
  W4Args a{p->x, p->ldx, p->codes, static_cast<const uint16_t*>(p->scales), p->zeros, p->bias, p->y, p->ldy, m, n, k};
  const size_t size = ftype == B200Q_F32 ? 4 : 2;
  a.x_vec = (reinterpret_cast<uintptr_t>(p->x) & 15u) == 0 && (m == 1 || p->ldx * size % 16 == 0);
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  B200Q_DISPATCH_FTYPE(ftype, rc = group == 32   ? launch_linear_rows<T, 32>(a, sms, device, cs)
                                   : group == 64 ? launch_linear_rows<T, 64>(a, sms, device, cs)
                                                 : launch_linear_rows<T, 128>(a, sms, device, cs));
  if (rc == B200Q_OK) host_set_path(17);
  return rc;
}
