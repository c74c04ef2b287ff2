// Linear layers of 8-bit rows (b200q_linear_s8).
//
//   y[m][n] = (sum_k x[m][k] w[n][k]) ws[n] xs[m] + bias[n]: the sum exact in int32, the rest fp32.
//
// tcgen05.mma.kind::i8 with the weights as the rows of the product (128 channels, TMEM lanes) and the tokens as its columns: a
// decode step of one token needs 16 columns, not 128 rows, and the same orientation serves a prompt.  A thread of the epilogue
// owns one channel: its scale and bias are registers, the tokens' scales broadcasts from shared memory.
//
// Two kernels.  linear_s8_split_kernel: one tile of 128 channels and up to 256 tokens a cluster, the reduction shared out to its
// 1 to 8 blocks, whose int32 sums meet in shared memory (integers: any order gives the same bits).  It takes the calls whose tiles do
// not fill the GPU: few tokens (bound by the weights' stream from DRAM), short prompts.  linear_s8_pair_kernel: persistent pairs of SMs,
// 256 channels x 256 tokens a tile, M = 256 instructions, the epilogue of a tile under the products of the next.
// Measured: 8192 x 8192 x 8192 in 324 to 329 us in a replayed graph, 3340 TOP/s, twice the bf16 rate that cuBLAS reaches (tensor pipe 88 %
// busy): the tensor core bounds it; call after call 383 to 395, as the power limit lowers the clock.  16 x 16384 x 8192 bf16 in 23.7 to 26.8 us,
// 5.7 TB/s (88 % of a copy) at best: DRAM.  1 x 4096 x 4096 in 5.4 to 6.9 us and 77 x 5003 x 4091 fp32 in 8.2 us: a launch, the first bytes'
// latency and the join of the blocks' sums.
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
constexpr int kSteps = 2;  // steps of a stage in the split kernel: one barrier for both
constexpr int kMaxStages = 16;
constexpr int kSmemMost = 227 * 1024;
constexpr int kRing = 2048;                    // the tokens' scales and the barriers lie before it
constexpr int kSmemFixed = 1024 + kRing;       // and the alignment
// Blocks of a cluster take more than half: no two that hold tensor memory then share an SM, this library's other kernels' among
// them.  They wait for each other; one that held tensor memory while its partner waited for some could wait for good.  A block without
// a cluster waits for no other once it has its tensor memory.
constexpr int kSmemAlone = kSmemMost / 2 + 1024;
constexpr int kTwosMost = 48;  // tokens of blocks that share an SM
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
  // N tokens from t on.  All values first, then all stores: one after another a column took 136 clocks.
  template <int N>
  __device__ __forceinline__ void put(const LinArgs& a, int t, const uint32_t (&sum)[N], const float (&xs)[N]) const {
    T v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = from_f32<T>(fmaf(static_cast<float>(static_cast<int>(sum[j])) * scale, xs[j], bias));
    if (!ok) return;
    T* p = y + t * a.ldy;
    if (t + N <= a.m) {
#pragma unroll
      for (int j = 0; j < N; ++j, p += a.ldy) *p = v[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j, p += a.ldy)
        if (t + j < a.m) *p = v[j];
    }
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_shared_cluster(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// A producer that gave up: what it asked for lands before the block ends.
__device__ __forceinline__ void land(uint32_t full0, int stages, int issued, const LinArgs& a) {
  for (int i = max(0, issued - stages); i < issued; ++i)
    mbar_wait_bounded(full0 + 8 * (i % stages), (i / stages) & 1, a.limit, a.err, kDevErrTimeoutProducer);
}

// One tile a cluster of `split` blocks.  Warp 0 loads, warp 1 issues, warps 2 to 5 write (warp w reads TMEM lanes 32 (w % 4)).
template <typename T>
__global__ void __launch_bounds__(kSplitThreads)
    linear_s8_split_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const LinArgs a) {
  extern __shared__ uint8_t smem_raw[];
  float* s_xs = reinterpret_cast<float*>(smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u));
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_xs + 256);
  uint8_t* smem = reinterpret_cast<uint8_t*>(s_xs) + kRing;
  const uint32_t step = (kBM + a.bn) * kBK, stage = kSteps * step;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxStages, done = full0 + 16 * kMaxStages;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 1);
  uint32_t* landing = reinterpret_cast<uint32_t*>(smem + a.stages * stage);  // [split][bn / split][128]: the blocks' sums of my columns
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = static_cast<int>(blockIdx.x % a.split), tile = static_cast<int>(blockIdx.x / a.split);
  const int t0 = tile / a.c_tiles * a.bn, c0 = tile % a.c_tiles * kBM;
  const int kb0 = static_cast<int>(static_cast<long long>(a.kblocks) * rank / a.split);
  const int kb1 = static_cast<int>(static_cast<long long>(a.kblocks) * (rank + 1) / a.split);

  // Loads a stage: steps kb, kb + 1.
  const auto load = [&](int s, int kb) {
    const uint32_t bar = full0 + 8 * s, n = min(kSteps, kb1 - kb);
    uint32_t at = smem_u32(smem) + s * stage;
    mbar_arrive_expect_tx_elect(bar, n * step);
    for (uint32_t i = 0; i < n; ++i, at += step) {
      tma_load_3d_elect(at, &tm_w, bar, (kb + i) * kBK, c0, 0);
      tma_load_3d_elect(at + kBM * kBK, &tm_x, bar, (kb + i) * kBK, t0, 0);
    }
  };
  int first = kb0;  // the ring is filled while the others set up
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < a.stages; ++i) {
        mbar_init(full0 + 8 * i, 1);
        mbar_init(empty0 + 8 * i, 1);
      }
      mbar_init(done, 1);
      fence_mbar_init();
    }
    __syncwarp();
    wait_for_previous();
    for (int s = 0; s < a.stages && first < kb1; ++s, first += kSteps) load(s, first);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(slot), a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (a.split > 1) cluster_arrive();
  const uint32_t acc = __shfl_sync(~0u, *slot, 0);
  wait_for_previous();

  if (warp == 0) {
    int s = 0, kb = first;
    uint32_t ph = 0;
    bool free = false;
    for (; kb < kb1; kb += kSteps) {
      if (!__all_sync(~0u, free || mbar_wait_bounded(empty0 + 8 * s, ph, a.limit, a.err, kDevErrTimeoutProducer))) break;
      const int at = s;
      if (++s == a.stages) s = 0, ph ^= 1u;
      free = mbar_test(empty0 + 8 * s, ph);
      load(at, kb);
    }
    if (kb < kb1) land(full0, a.stages, (kb - kb0) / kSteps, a);
  } else if (warp == 1) {
    int s = 0;
    uint32_t ph = 0;
    bool full = false;
    for (int kb = kb0; kb < kb1; kb += kSteps) {
      if (!__all_sync(~0u, full || mbar_wait_bounded(full0 + 8 * s, ph, a.limit, a.err, kDevErrTimeoutMma))) break;
      const uint32_t at = smem_u32(smem) + s * stage, bar = empty0 + 8 * s;
      if (++s == a.stages) s = 0, ph ^= 1u;
      full = mbar_test(full0 + 8 * s, ph);  // an answer takes 130 clocks, as long as the products of a step of few tokens
      tc_mma_i8_kblock4(acc, operand_desc(at), operand_desc(at + kBM * kBK), a.idesc, kb > kb0 ? 1u : 0u);
      if (kb + 1 < kb1) tc_mma_i8_kblock4(acc, operand_desc(at + step), operand_desc(at + step + kBM * kBK), a.idesc, 1u);
      tc_commit_elect(bar);
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
    const auto xs_at = [&](int c, float (&xs)[16]) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 x = *reinterpret_cast<const float4*>(s_xs + c + j);
        xs[j] = x.x, xs[j + 1] = x.y, xs[j + 2] = x.z, xs[j + 3] = x.w;
      }
    };
    if (a.split == 1) {
      for (int c = 0; c < a.bn && t0 + c < a.m; c += 16) {
        uint32_t v[16];
        float xs[16];
        tmem_ld_32x32b_x16(from + c, v);
        xs_at(c, xs);
        tmem_ld_wait();
        ch.put(a, t0 + c, v, xs);
      }
    } else {
      const int share = a.bn / a.split;  // columns that a block adds up, at least 2
      const uint32_t to = smem_u32(landing + rank * share * kBM + mine);
      cluster_wait();  // the others have started
      for (int c = 0; c < a.bn && t0 + c < a.m; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(from + c, v);
        tmem_ld_wait();
        int owner = c / share, in = c - owner * share;
#pragma unroll
        for (int j = 0; j < 16; j += 2) {  // two columns go to one block
          const uint32_t at = mapa_shared(to, owner) + in * (kBM * 4);
          store_shared_cluster(at, v[j]);
          store_shared_cluster(at + kBM * 4, v[j + 1]);
          if ((in += 2) == share) in = 0, ++owner;
        }
      }
      cluster_sync_all();  // every block's sums have arrived
      const int j0 = share * rank;
      const uint32_t* mine_at = landing + mine;
      for (int j = 0; j < share && t0 + j0 + j < a.m; j += 2) {
        uint32_t v[2] = {0u, 0u};
        const float xs[2] = {s_xs[j0 + j], s_xs[j0 + j + 1]};
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < a.split) {
            v[0] += mine_at[(r * share + j) * kBM];
            v[1] += mine_at[(r * share + j + 1) * kBM];
          }
        ch.put(a, t0 + j0 + j, v, xs);
      }
    }
  }
  if (warp < 2 && a.split > 1) {
    cluster_wait();
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
      int issued = 0;
      bool ok = true, free = true;
      const uint32_t full_leader = mapa_shared(full0, 0);
      for (int i = unit; i < tiles && ok; i += units) {
        int ct, tt;
        tile_at(i, &ct, &tt);
        const int c0 = (2 * ct + rank) * kBM, t0 = tt * a.bn + rank * (a.bn / 2);
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!free && !mbar_wait_bounded(empty0 + 8 * s, ph ^ 1u, a.limit, a.err, kDevErrTimeoutProducer)) {
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
          ++issued;
          if (++s == a.stages) s = 0, ph ^= 1u;
          free = mbar_test(empty0 + 8 * s, ph ^ 1u);
        }
      }
      if (!ok && rank == 0) land(full0, a.stages, issued, a);  // both blocks' copies count there; the other waits for the leader below
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      int s = 0, buf = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true, full = false;
      for (int i = unit; i < tiles && ok; i += units) {
        if (!__all_sync(~0u, mbar_wait_bounded(acce0 + 8 * buf, acc_ph ^ 1u, a.limit, a.err, kDevErrTimeoutMma))) break;
        tc_fence_after();
        for (int kb = 0; kb < a.kblocks; ++kb) {
          if (!__all_sync(~0u, full || mbar_wait_bounded(full0 + 8 * s, ph, a.limit, a.err, kDevErrTimeoutMma))) {
            ok = false;
            break;
          }
          const uint32_t at = smem_u32(smem) + s * stage, bar = empty0 + 8 * s;
          if (++s == a.stages) s = 0, ph ^= 1u;
          full = mbar_test(full0 + 8 * s, ph);
          tc_mma_i8_pair_kblock4(tmem + buf * a.bn, operand_desc(at), operand_desc(at + stage_w), a.idesc, kb ? 1u : 0u);
          tc_commit_pair_elect(bar);
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
      for (int c = 32 * half; c < a.bn && tt * a.bn + c < a.m; c += 64) {
        uint32_t v[32];
        float xs[32];
        tmem_ld_32x32b_x32(from + c, v);
        const int t = tt * a.bn + c;
        const float one = t + lane < a.m ? __ldg(a.xs + t + lane) : 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) xs[j] = __shfl_sync(~0u, one, j);
        tmem_ld_wait();
        ch.put(a, t, v, xs);
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
  int bn, split, stages;
};

int round_up(int v, int to) { return (v + to - 1) / to * to; }

int stage_bytes(const Plan& p) { return p.pair ? (kBM + p.bn / 2) * kBK : kSteps * (kBM + p.bn) * kBK; }
int landing_bytes(const Plan& p) { return p.split > 1 ? p.bn * kBM * 4 : 0; }

// Clocks that a plan takes, from timed calls: what a step of a block costs (its barriers and copies, and more with every token), what a
// tile costs beside its steps, what joining costs, and the bytes at what DRAM gives (4 KB a clock).  The plans differ most where few
// tiles leave SMs idle: 64 x 4096 x 4096 8.7 us on 2 x 32 tokens, 9.6 on 64, 9.4 on 64 split in four; 1 x 4096 x 4096 5.9 split in four,
// 7.6 whole; 512 x 4096 x 4096 13.1 on 128 tokens, 17.6 on pairs of 256; 1024 x 4096 x 4096 21.4 on 256 tokens, 18.2 on pairs.
// `room`: blocks that the GPU holds at once, by the size of their cluster (1, 2, 4, 8: 148, 148, 132, 120 with one a SM).
double plan_clocks(const Plan& p, int m, int n, int kblocks, const int (&room)[4]) {
  const long long t_tiles = (m + p.bn - 1) / p.bn;
  if (p.pair) {
    const long long tiles = t_tiles * ((n + 255) / 256), waves = (tiles + room[0] / 2 - 1) / (room[0] / 2);
    return 9000.0 + 30.0 * p.bn + static_cast<double>(waves) * kblocks * (440.0 + 0.9 * p.bn);
  }
  const long long blocks = t_tiles * ((n + kBM - 1) / kBM) * p.split;
  const int steps = (kblocks + p.split - 1) / p.split;
  // blocks of few tokens share an SM in twos and hide part of each other's steps
  const bool twos = p.split == 1 && p.bn <= kTwosMost && blocks > room[0];
  const long long most = twos ? 2ll * room[0] : room[p.split == 1 ? 0 : p.split == 2 ? 1 : p.split == 4 ? 2 : 3];
  const double waves = static_cast<double>((blocks + most - 1) / most), at_once = twos ? 1.6 : 1.0;
  const double join = p.split > 1 ? 1700.0 + 300.0 * p.split + 15.0 * p.bn : 0.0;
  const double clocks = waves * at_once * (steps * (210.0 + 2.8 * p.bn) + 27.0 * p.bn) + 4500.0 + join;
  return std::max(clocks, (static_cast<double>(n) + m) * kblocks * kBK / 4096.0 + 5000.0 + join);
}

Plan search_plan(int m, int n, int kblocks, const int (&room)[4]) {
  Plan best{false, 16, 1, 0};
  double least = 1e300;
  const auto offer = [&](Plan p) {
    const double c = plan_clocks(p, m, n, kblocks, room);
    if (c < least) least = c, best = p;
  };
  const int most = std::min(256, round_up(m, 16));
  for (int bn = 16; bn <= most; bn += bn < 128 ? 16 : 32)
    for (int split = 1; split <= 8 && split <= kblocks && (split == 1 || bn <= 128); split *= 2) offer({false, bn, split, 0});
  offer({false, most, 1, 0});
  if (m > 64)
    for (int bn = 64; bn <= 256; bn += 32) offer({true, bn, 1, 0});
  const int steps = best.pair ? kblocks : ((kblocks + best.split - 1) / best.split + kSteps - 1) / kSteps;
  const long long blocks = static_cast<long long>((m + best.bn - 1) / best.bn) * ((n + kBM - 1) / kBM);
  const int smem = !best.pair && best.split == 1 && best.bn <= kTwosMost && blocks > room[0] ? kSmemMost / 2 - 1024 : kSmemMost;
  best.stages = std::max(2, std::min({kMaxStages, steps, (smem - kSmemFixed - landing_bytes(best)) / stage_bytes(best)}));
  return best;
}

// The search takes a microsecond: a thread keeps the plans of its last sizes.
Plan plan_for(int m, int n, int kblocks, int device, const int (&room)[4]) {
  struct Kept {
    int m = -1, n, kblocks, device;
    Plan plan;
  };
  static thread_local Kept kept[64];
  Kept& at = kept[(static_cast<unsigned>(m) * 31u + static_cast<unsigned>(n) * 7u + static_cast<unsigned>(kblocks)) % 64u];
  if (at.m != m || at.n != n || at.kblocks != kblocks || at.device != device)
    at = {m, n, kblocks, device, search_plan(m, n, kblocks, room)};
  return at.plan;
}

template <typename T>
int launch_plan(const Plan& p, LinArgs a, const CUtensorMap& tm_w, const CUtensorMap& tm_x, int sms, int device, cudaStream_t cs) {
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[device].load(std::memory_order_relaxed)) {
    cudaError_t e = cudaFuncSetAttribute(linear_s8_split_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(linear_s8_pair_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(linear_s8_kernel)");
    ready[device].store(true, std::memory_order_relaxed);
  }
  a.bn = p.bn;
  a.split = p.split;
  a.stages = p.stages;
  a.t_tiles = (a.m + p.bn - 1) / p.bn;
  a.c_tiles = (a.n + (p.pair ? 255 : 127)) / (p.pair ? 256 : 128);
  const uint32_t rows = p.pair ? 256 : 128;
  a.idesc = (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(p.bn >> 3) << 17) | ((rows >> 4) << 24);  // s32 += s8 s8
  for (a.tmem_cols = 32; a.tmem_cols < static_cast<uint32_t>(p.pair ? 2 * p.bn : p.bn);) a.tmem_cols *= 2;
  size_t smem = static_cast<size_t>(p.stages) * stage_bytes(p) + landing_bytes(p) + kSmemFixed;
  if (p.pair || p.split > 1) smem = std::max(smem, static_cast<size_t>(kSmemAlone));
  const long long tiles = static_cast<long long>(a.t_tiles) * a.c_tiles;
  if (tiles * 8 > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many tiles");
  if (p.pair)
    return host_launch("linear_s8_pair_kernel launch", linear_s8_pair_kernel<T>,
                       dim3(2 * static_cast<unsigned>(std::min<long long>(tiles, sms / 2))), kPairThreads, smem, cs, 1, tm_w, tm_x, a);
  return host_launch("linear_s8_split_kernel launch", linear_s8_split_kernel<T>, dim3(static_cast<unsigned>(tiles * p.split)),
                     kSplitThreads, smem, cs, p.split, tm_w, tm_x, a);
}

// Found once for a device: clusters lie in one part of the GPU each, whose SMs they do not use up.
int block_room(int device, int sms, int (*room)[4]) {
  static std::atomic<int> of[kMaxDevices][4];
  (*room)[0] = sms;
  for (int i = 1; i < 4; ++i) {
    int blocks = of[device][i].load(std::memory_order_relaxed);
    if (!blocks) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(1024);
      cfg.blockDim = dim3(kSplitThreads);
      cfg.dynamicSmemBytes = kSmemAlone;
      cudaLaunchAttribute attr[1] = {};
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim = {1u << i, 1, 1};
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      cudaError_t e = cudaFuncSetAttribute(linear_s8_split_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
      int clusters = 0;
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, linear_s8_split_kernel<float>, &cfg);
      if (e != cudaSuccess) return host_cuda_fail(e, "cudaOccupancyMaxActiveClusters(linear_s8_split_kernel)");
      blocks = std::max(1, clusters) << i;
      of[device][i].store(blocks, std::memory_order_relaxed);
    }
    (*room)[i] = blocks;
  }
  return B200Q_OK;
}

int linear_s8(const b200q_linear_s8_args* p, cudaStream_t cs) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const int ftype = p->ftype, m = p->m, n = p->n, k = p->k;
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (m < 0 || n < 0 || k < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative dimensions");
  if (m == 0 || n == 0) return B200Q_OK;
  if (k == 0) return host_fail(B200Q_ERR_INVALID_ARG, "rows of no elements");
  if (k > 131071) return host_fail(B200Q_ERR_UNSUPPORTED, "k = %d: sums of more than 131071 products may pass 32 bits", k);
  if (m > (1 << 28) || n > (1 << 28)) return host_fail(B200Q_ERR_UNSUPPORTED, "%d x %d results: too large", m, n);
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
  int room[4];
  if ((rc = block_room(device, sms, &room))) return rc;
  const Plan plan = plan_for(m, n, a.kblocks, device, room);
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
  return linear_s8(args, static_cast<cudaStream_t>(stream));
}
