// Linear layers of 8-bit rows (b200q_linear_s8).
//
//   y[m][n] = (sum_k x[m][k] w[n][k]) xs[m] ws[n] + bias[n]: the sum exact in int32, the rest fp32.
//
// tcgen05.mma.kind::i8 with the weights as the rows of the product (128 channels, TMEM lanes) and the tokens as its columns: a
// decode step of one token needs 16 columns, not 128 rows, and the same orientation serves a prompt.  A thread of the epilogue
// owns one channel: its scale and bias are registers, the tokens' scales broadcasts from shared memory.
//
// Two kernels.  linear_s8_split_kernel: one tile of 128 channels and up to 256 tokens a cluster, the reduction shared out to its
// 1 to 8 blocks, whose int32 sums meet in shared memory (integers: any order gives the same bits).  It takes the calls whose tiles do
// not fill the GPU: few tokens (bound by the weights' stream from DRAM), short prompts.  linear_s8_pair_kernel: persistent pairs of SMs,
// 256 channels x 256 tokens a tile, M = 256 instructions, the epilogue of a tile under the products of the next.
#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "host.h"
#include "lowbit.cuh"
#include "ptx.cuh"

namespace b200q {
namespace {

constexpr int kBM = 128;  // channels of a block's tile
constexpr int kBK = 128;  // bytes of a step: one 128-byte swizzle row
constexpr int kMaxStages = 16;
constexpr int kSmemMost = 227 * 1024;
constexpr int kRing = 2048;                    // the tokens' scales and the barriers lie before it
constexpr int kSmemFixed = 1024 + kRing;       // and the alignment
// More than half: no two blocks that hold tensor memory share an SM, this library's other kernels' among them.  Blocks of a cluster
// wait for each other; one that held tensor memory while its partner waited for some could wait for good.
constexpr int kSmemAlone = kSmemMost / 2 + 1024;
constexpr int kSplitThreads = 192;
constexpr int kPairThreads = 320;

struct LinArgs {
  const float* xs;
  const float* ws;
  const void* bias;
  void* y;
  long long ldy;
  int m, n, kblocks;
  int bn, stages, split;
  int c_tiles, t_tiles;
  uint32_t idesc, tmem_cols;
  long long limit;
  int* err;
};

// A thread's channel.
template <typename T>
struct Channel {
  T* y;  // of token 0
  float scale, bias;
  bool ok;
  __device__ __forceinline__ Channel(const LinArgs& a, int c) {
    ok = c < a.n;
    y = static_cast<T*>(a.y) + c;
    scale = ok ? __ldg(a.ws + c) : 0.0f;
    bias = ok && a.bias ? to_f32(static_cast<const T*>(a.bias)[c]) : 0.0f;
  }
  __device__ __forceinline__ void put(const LinArgs& a, int token, int sum, float xs) const {
    if (ok && token < a.m) y[token * a.ldy] = from_f32<T>(fmaf(static_cast<float>(sum) * scale, xs, bias));
  }
};

__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) { return make_smem_desc(saddr, 16u, 8u * kBK, 2u); }

__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ uint32_t load_shared_cluster(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
  return r;
}

// One tile a cluster of `split` blocks.  Warp 0 loads, warp 1 issues, warps 2 to 5 write (warp w reads TMEM lanes 32 (w % 4)).
template <typename T>
__global__ void __launch_bounds__(kSplitThreads)
    linear_s8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const LinArgs a) {
  extern __shared__ uint8_t smem_raw[];
  float* s_xs = reinterpret_cast<float*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_xs + 256);
  uint8_t* smem = reinterpret_cast<uint8_t*>(s_xs) + kRing;
  const uint32_t stage_w = kBM * kBK, stage_x = a.bn * kBK, stage = stage_w + stage_x;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, done = full0 + 16 * kMaxStages;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = static_cast<int>(blockIdx.x % a.split), tile = static_cast<int>(blockIdx.x / a.split);
  const int t0 = tile / a.c_tiles * a.bn, c0 = tile % a.c_tiles * kBM;
  const int kb0 = static_cast<int>(static_cast<long long>(a.kblocks) * rank / a.split);
  const int kb1 = static_cast<int>(static_cast<long long>(a.kblocks) * (rank + 1) / a.split);

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(slot), a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t acc = __shfl_sync(~0u, *slot, 0);
  wait_for_previous();

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_bounded(empty0 + 8 * s, ph ^ 1u, a.limit, a.err, kDevErrTimeoutProducer)) break;
        mbar_arrive_expect_tx(full0 + 8 * s, stage);
        const uint32_t at = smem_u32(smem) + s * stage;
        tma_load_3d(at, &tm_w, full0 + 8 * s, kb * kBK, c0, 0);
        tma_load_3d(at + stage_w, &tm_x, full0 + 8 * s, kb * kBK, t0, 0);
        if (++s == a.stages) s = 0, ph ^= 1u;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    int s = 0;
    uint32_t ph = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(~0u, mbar_wait_bounded(full0 + 8 * s, ph, a.limit, a.err, kDevErrTimeoutMma))) break;
      const uint32_t at = smem_u32(smem) + s * stage;
      const uint64_t dw = operand_desc(at), dx = operand_desc(at + stage_w);
#pragma unroll
      for (int j = 0; j < kBK / 32; ++j) tc_mma_i8_elect(acc, dw + 2 * j, dx + 2 * j, a.idesc, kb > kb0 || j ? 1u : 0u);
      tc_commit_elect(empty0 + 8 * s);
      if (++s == a.stages) s = 0, ph ^= 1u;
    }
    tc_commit_elect(done);
    mbar_wait_bounded(done, 0, a.limit, a.err, kDevErrTimeoutMma);
    __syncwarp();
  } else {
    const int mine = (warp % 4) * 32 + lane;  // channel of the tile
    for (int i = threadIdx.x - 64; i < a.bn; i += 128) s_xs[i] = t0 + i < a.m ? __ldg(a.xs + t0 + i) : 0.0f;
    const Channel<T> ch(a, c0 + mine);
    asm volatile("bar.sync 1, 128;" ::: "memory");
    mbar_wait_bounded(done, 0, a.limit, a.err, kDevErrTimeoutEpilogue);
    __syncwarp();
    tc_fence_after();
    const uint32_t from = acc + (static_cast<uint32_t>((warp % 4) * 32) << 16);
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);  // [bn][128]: the ring has been read by now
    for (int c = 0; c < a.bn; c += 16) {
      uint32_t v[16];
      tmem_ld_32x32b_x16(from + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (a.split == 1)
          ch.put(a, t0 + c + j, static_cast<int>(v[j]), s_xs[c + j]);
        else
          part[(c + j) * kBM + mine] = v[j];
      }
    }
    if (a.split > 1) {
      cluster_sync_all();
      const int j0 = a.bn * rank / a.split, j1 = a.bn * (rank + 1) / a.split;
      for (int j = j0; j < j1 && t0 + j < a.m; ++j) {
        const uint32_t at = smem_u32(part + j * kBM + mine);
        int sum = 0;
        for (int r = 0; r < a.split; ++r) sum += static_cast<int>(load_shared_cluster(mapa_shared(at, r)));
        ch.put(a, t0 + j, sum, s_xs[j]);
      }
      cluster_sync_all();
    }
  }
  if (warp < 2 && a.split > 1) {
    cluster_sync_all();
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(acc, a.tmem_cols);
  }
}

// Persistent pairs of blocks: each loads its 128 channels and half of the tokens, the leader issues, both write their channels.
// Two accumulators of bn columns.
template <typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    linear_s8_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const LinArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  uint8_t* smem = reinterpret_cast<uint8_t*>(bars) + kRing;
  const uint32_t stage_w = kBM * kBK, stage_x = a.bn / 2 * kBK, stage = stage_w + stage_x;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, accf0 = full0 + 16 * kMaxStages, acce0 = accf0 + 16;
  const uint32_t drain = acce0 + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 5);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = static_cast<int>(cluster_ctarank()), unit = static_cast<int>(blockIdx.x / 2);
  const int units = static_cast<int>(gridDim.x / 2), tiles = a.c_tiles * a.t_tiles;

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(full0 + 8 * i, 2);  // one expectation from each block of the pair
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accf0 + 8 * i, 1);
      mbar_init(acce0 + 8 * i, 16);  // epilogue warps of both blocks
    }
    mbar_init(drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(slot), a.tmem_cols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both blocks' barriers are there
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, *slot, 0);
  wait_for_previous();

  // Tiles go through bands of 8 channel tiles, so that the pairs at work share weights and tokens in L2.
  auto tile_at = [&](int i, int* ct, int* tt) {
    const int band = 8 * a.t_tiles, b = i / band, in = i - b * band;
    const int wide = min(8, a.c_tiles - 8 * b);
    *tt = in / wide;
    *ct = 8 * b + in % wide;
  };

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t full_leader = mapa_shared(full0, 0);
      for (int i = unit; i < tiles && ok; i += units) {
        int ct, tt;
        tile_at(i, &ct, &tt);
        const int c0 = (2 * ct + rank) * kBM, t0 = tt * a.bn + rank * (a.bn / 2);
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!mbar_wait_bounded(empty0 + 8 * s, ph ^ 1u, a.limit, a.err, kDevErrTimeoutProducer)) {
            ok = false;
            break;
          }
          const uint32_t bar = full_leader + 8 * s, at = smem_u32(smem) + s * stage;
          if (rank == 0)
            mbar_arrive_expect_tx(full0 + 8 * s, stage);
          else
            mbar_arrive_expect_tx_cluster_relaxed(bar, stage);
          tma_load_3d_pair(at, &tm_w, bar, kb * kBK, c0, 0);
          tma_load_3d_pair(at + stage_w, &tm_x, bar, kb * kBK, t0, 0);
          if (++s == a.stages) s = 0, ph ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int i = unit; i < tiles && ok; i += units) {
        if (!__all_sync(~0u, mbar_wait_bounded(acce0 + 8 * buf, acc_ph ^ 1u, a.limit, a.err, kDevErrTimeoutMma))) break;
        tc_fence_after();
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!__all_sync(~0u, mbar_wait_bounded(full0 + 8 * s, ph, a.limit, a.err, kDevErrTimeoutMma))) {
            ok = false;
            break;
          }
          const uint32_t at = smem_u32(smem) + s * stage;
          tc_mma_i8_pair_kblock4(tmem + buf * a.bn, operand_desc(at), operand_desc(at + stage_w), a.idesc, kb ? 1u : 0u);
          tc_commit_pair_elect(empty0 + 8 * s);
          if (++s == a.stages) s = 0, ph ^= 1u;
        }
        if (!ok) break;
        tc_commit_pair_elect(accf0 + 8 * buf);
        buf ^= 1;
        if (buf == 0) acc_ph ^= 1u;
      }
      tc_commit_pair_elect(drain);
      mbar_wait_bounded(drain, 0, a.limit, a.err, kDevErrTimeoutMma);
      __syncwarp();
    }
  } else {
    const int quarter = warp % 4, half = (warp - 2) / 4;
    const uint32_t acce_leader = mapa_shared(acce0, 0);
    int buf = 0;
    uint32_t acc_ph = 0;
    for (int i = unit; i < tiles; i += units) {
      int ct, tt;
      tile_at(i, &ct, &tt);
      const Channel<T> ch(a, (2 * ct + rank) * kBM + quarter * 32 + lane);
      if (!__all_sync(~0u, mbar_wait_bounded(accf0 + 8 * buf, acc_ph, a.limit, a.err, kDevErrTimeoutEpilogue))) break;
      tc_fence_after();
      const uint32_t from = tmem + buf * a.bn + (static_cast<uint32_t>(quarter * 32) << 16);
      for (int c = 32 * half; c < a.bn; c += 64) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(from + c, v);
        const int t = tt * a.bn + c;
        const float mine = t + lane < a.m ? __ldg(a.xs + t + lane) : 0.0f;
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) ch.put(a, t + j, static_cast<int>(v[j]), __shfl_sync(~0u, mine, j));
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acce_leader + 8 * buf);
      buf ^= 1;
      if (buf == 0) acc_ph ^= 1u;
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // nothing reaches the other block's memory after this
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, a.tmem_cols);
  }
}

// How a call is laid out.
struct Plan {
  bool pair;
  int bn, split;
};

int round_up(int v, int to) { return (v + to - 1) / to * to; }

Plan plan_for(int m, int n, int kblocks, int sms) {
  Plan p{false, std::min(256, round_up(m, 16)), 1};
  const int pair_tiles = (n + 255) / 256 * ((m + 255) / 256);
  if (m > 128 && pair_tiles * 2 >= sms) return {true, 256, 1};
  const int tiles = (n + kBM - 1) / kBM * ((m + p.bn - 1) / p.bn);
  while (p.split < 8 && tiles * p.split * 2 <= sms && kblocks >= 2 * p.split) p.split *= 2;
  return p;
}

template <typename T>
int launch_plan(const Plan& p, LinArgs a, const CUtensorMap& tm_w, const CUtensorMap& tm_x, int sms, int device,
                cudaStream_t cs) {
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[device].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(linear_s8_split_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_s8_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(linear_s8_kernel)");
    ready[device].store(true, std::memory_order_relaxed);
  }
  a.bn = p.bn;
  a.split = p.split;
  const int stage = kBM * kBK + (p.pair ? p.bn / 2 : p.bn) * kBK;
  const int steps = p.pair ? a.kblocks : (a.kblocks + p.split - 1) / p.split;
  a.stages = std::max(2, std::min({kMaxStages, (kSmemMost - kSmemFixed) / stage, p.pair ? kMaxStages : steps}));
  a.t_tiles = (a.m + p.bn - 1) / p.bn;
  a.c_tiles = (a.n + (p.pair ? 255 : 127)) / (p.pair ? 256 : 128);
  const uint32_t rows = p.pair ? 256 : 128;
  a.idesc = (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(p.bn >> 3) << 17) | ((rows >> 4) << 24);  // s32 += s8 s8
  for (a.tmem_cols = 32; a.tmem_cols < static_cast<uint32_t>(p.pair ? 2 * p.bn : p.bn);) a.tmem_cols *= 2;
  size_t smem = static_cast<size_t>(a.stages) * stage + kSmemFixed;
  const long long tiles = static_cast<long long>(a.t_tiles) * a.c_tiles;
  if (tiles * 8 > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many tiles");
  smem = std::max(smem, static_cast<size_t>(kSmemAlone));
  if (p.pair) {
    const int pairs = static_cast<int>(std::min<long long>(tiles, sms / 2));
    return host_launch("linear_s8_pair_kernel launch", linear_s8_pair_kernel<T>, dim3(2 * pairs), kPairThreads, smem, cs, 1, tm_w,
                       tm_x, a);
  }
  if (p.split > 1) smem = std::max(smem, static_cast<size_t>(p.bn) * kBM * 4 + kSmemFixed);
  return host_launch("linear_s8_split_kernel launch", linear_s8_split_kernel<T>, dim3(static_cast<unsigned>(tiles * p.split)),
                     kSplitThreads, smem, cs, p.split, tm_w, tm_x, a);
}

int linear_s8(const b200q_linear_s8_args* p, const Plan* fixed, cudaStream_t cs) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const int ftype = p->ftype, m = p->m, n = p->n, k = p->k;
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (m < 0 || n < 0 || k < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative dimensions");
  if (m == 0 || n == 0) return B200Q_OK;
  if (k == 0) return host_fail(B200Q_ERR_INVALID_ARG, "rows of no elements");
  if (k > 131071) return host_fail(B200Q_ERR_UNSUPPORTED, "k = %d: sums of more than 131071 products may pass 32 bits", k);
  if (n > (1 << 28)) return host_fail(B200Q_ERR_UNSUPPORTED, "n = %d is too large", n);
  if (!p->x || !p->w || !p->x_scales || !p->w_scales || !p->y) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if ((p->ldx < k && m > 1) || (p->ldw < k && n > 1) || (p->ldy < n && m > 1))
    return host_fail(B200Q_ERR_INVALID_ARG, "row stride smaller than a row");
  if (((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->w)) & 15u) || (m > 1 && p->ldx % 16) || (n > 1 && p->ldw % 16))
    return host_fail(B200Q_ERR_INVALID_ARG, "codes must be 16-byte aligned, with row strides that are multiples of 16");
  int sms = 0, *err = nullptr, device = 0;
  int rc = host_device(&sms, &err, &device);
  if (rc) return rc;
  LinArgs a{};
  a.xs = p->x_scales;
  a.ws = p->w_scales;
  a.bias = p->bias;
  a.y = p->y;
  a.ldy = p->ldy;
  a.m = m;
  a.n = n;
  a.kblocks = (k + kBK - 1) / kBK;
  a.limit = host_wait_limit();
  a.err = err;
  const Plan plan = fixed ? *fixed : plan_for(m, n, a.kblocks, sms);
  CUtensorMap tm_w, tm_x;
  const auto stride = [&](int rows, int64_t ld) { return static_cast<uint64_t>(rows > 1 ? ld : round_up(k, 16)); };
  if ((rc = host_tensor_map(&tm_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p->w, {static_cast<uint64_t>(k), static_cast<uint64_t>(n), 1},
                            stride(n, p->ldw), stride(n, p->ldw) * n, {kBK, kBM, 1})))
    return rc;
  const uint32_t box = static_cast<uint32_t>(plan.pair ? plan.bn / 2 : plan.bn);
  if ((rc = host_tensor_map(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, p->x, {static_cast<uint64_t>(k), static_cast<uint64_t>(m), 1},
                            stride(m, p->ldx), stride(m, p->ldx) * m, {kBK, box, 1})))
    return rc;
  B200Q_DISPATCH_FTYPE(ftype, rc = launch_plan<T>(plan, a, tm_w, tm_x, sms, device, cs));
  if (rc == B200Q_OK) host_set_path(22);
  return rc;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_linear_s8(const b200q_linear_s8_args* args, void* stream) {
  return linear_s8(args, nullptr, static_cast<cudaStream_t>(stream));
}
