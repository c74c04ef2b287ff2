// Prompt attention of 16-bit types on tcgen05 (prompt_tc_kernel).
//
// A block has two tiles of 128 rows (token, query head of one key head) and goes through the keys 128 at a time.  Warps 0 to 3 and 4
// to 7 hold a tile each, one row a thread: scores from TMEM, weights back over them as 16-bit operands of the second product; warp 8 loads by TMA, warp
// 9 issues.  While one tile's scores become weights the tensor core has the other tile's products:
//   PV_A(j), QK_A(j + 1), PV_B(j), QK_B(j + 1), ...
// Tensor memory: scores of A and B (128 columns each; weights take the first 64), then the sums O of A and B (D columns each).
// A row's reference is not its maximum but one that may lie up to 2^8 below it: O is then rescaled a few times in a row of any length, by
// the threads that own it, and not with every tile.  fp16 weights are lifted by 2^6: they stay normal down to 2^-20 of the reference,
// and below 2^14 above it.
#pragma once
#include "common.cuh"
#include "prompt.cuh"
#include "ptx.cuh"

namespace b200q {

constexpr int kTcKeys = 128;
constexpr int kTcPromptThreads = 320;
constexpr int kTcMaxStages = 8;
constexpr float kSlack = 8.0f;  // log2 of how far a row's maximum may pass its reference

template <int D>
struct TcShape {
  static constexpr int kTile = 128 * D * 2;  // bytes of 128 rows
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kHead = 1024;  // barriers
  static constexpr int kSmem = 1024 + kHead + (2 + kStages) * kTile;
};

// D (+)= A B with A from shared memory or from tensor memory: fp16 or bf16 operands, fp32 sums.
__device__ __forceinline__ void tc_mma_f16_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ts_elect(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value)
    return pack_f16(lo, hi);
  else
    return pack_bf16(lo, hi);
}

// What one block does: its sequence and tokens, read once by warp 0.
struct TcUnit {
  Sequence s;
  int token0;  // of tile A in the sequence
  int ok;
};

template <typename T, int D>
__global__ void __launch_bounds__(kTcPromptThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PromptArgs a, const uint32_t negate) {
  using S = TcShape<D>;
  constexpr int kChunks = D / 64;  // 128-byte columns of a tile
  constexpr float kLift = std::is_same<T, __half>::value ? 6.0f : 0.0f;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kTcMaxStages;
  const uint32_t q_full = full0 + 16 * kTcMaxStages, s_full = q_full + 16, p_full = s_full + 16, o_done = p_full + 16;
  const uint32_t drain = o_done + 16;
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 2 * kTcMaxStages + 9);
  TcUnit* shared_unit = reinterpret_cast<TcUnit*>(slot + 2);
  const uint32_t s_q = smem_u32(smem) + S::kHead, s_ring = s_q + 2 * S::kTile;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int ratio = static_cast<int>(a.ratio.d), tokens = a.tile_tokens / 2;  // of one tile

  if (threadIdx.x == 256) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(o_done + 8 * i, 1);
    }
    mbar_init(drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(slot), 512);
    tmem_relinquish();
  }
  wait_for_previous();
  const int kv = static_cast<int>(blockIdx.x % a.hk);
  if (warp == 0) {
    const PromptUnit u = prompt_unit(a, static_cast<int>(blockIdx.x / a.hk), blockIdx.x == 0);
    if (lane == 0) *shared_unit = {u.s, u.tile * a.tile_tokens, u.ok};
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, *slot, 0);
  const TcUnit u = *shared_unit;
  const int shift = u.s.lk - u.s.lq;
  // keys that a tile needs, in steps: its last token's
  int steps[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = u.token0 + i * tokens, last = min(u.s.lq, first + tokens) - 1;
    steps[i] = u.ok && first < u.s.lq ? (max(0, last + shift + 1) + kTcKeys - 1) / kTcKeys : 0;
  }
  const int all = max(steps[0], steps[1]);

  if (warp == 8) {
    if (lane == 0 && all) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (steps[i]) {
          const uint32_t bytes = static_cast<uint32_t>(tokens * ratio) * 128u;
          mbar_arrive_expect_tx(q_full + 8 * i, kChunks * bytes);
          for (int c = 0; c < kChunks; ++c)
            tma_load_3d(s_q + i * S::kTile + c * 16384, &tm_q, q_full + 8 * i, 64 * c, kv * ratio, u.s.q0 + u.token0 + i * tokens);
        }
      int s = 0, issued = 0;
      uint32_t ph = 0;
      for (; issued < 2 * all; ++issued) {  // K 0, V 0, K 1, V 1, ...
        if (!mbar_wait_bounded(empty0 + 8 * s, ph ^ 1u, a.limit, a.err, kDevErrTimeoutProducer)) break;
        mbar_arrive_expect_tx(full0 + 8 * s, S::kTile);
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d(s_ring + s * S::kTile + c * 16384, issued & 1 ? &tm_v : &tm_k, full0 + 8 * s, 64 * c, kv,
                      u.s.k0 + issued / 2 * kTcKeys);
        if (++s == S::kStages) s = 0, ph ^= 1u;
      }
      if (issued < 2 * all)  // given up: what is on its way lands before the block ends
        for (int i = max(0, issued - S::kStages); i < issued; ++i)
          mbar_wait_bounded(full0 + 8 * (i % S::kStages), (i / S::kStages) & 1, a.limit, a.err, kDevErrTimeoutProducer);
    }
    __syncwarp();
  } else if (warp == 9) {
    constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
    constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) | ((128u >> 4) << 24);
    const uint32_t qk_desc = kDesc | ((kTcKeys >> 3) << 17) | (negate << 13);
    const uint32_t pv_desc = kDesc | ((static_cast<uint32_t>(D) >> 3) << 17) | (1u << 16);  // V: channels contiguous
    bool ok = all > 0;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = ok && __all_sync(~0u, mbar_wait_bounded(bar, parity, a.limit, a.err, kDevErrTimeoutMma));
    };
    auto tile_at = [&](int n) { return s_ring + n % S::kStages * S::kTile; };
    auto tile_wait = [&](int n) { wait(full0 + 8 * (n % S::kStages), (n / S::kStages) & 1); };
    auto release = [&](int n) { tc_commit_elect(empty0 + 8 * (n % S::kStages)); };
    auto qk = [&](int i, int j) {
      if (!ok) return;
      const uint32_t q = s_q + i * S::kTile, k = tile_at(2 * j);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        const uint32_t off = c / 4 * 16384 + c % 4 * 32;
        tc_mma_f16_elect(tmem + i * 128, make_smem_desc(q + off, 16, 1024, 2), make_smem_desc(k + off, 16, 1024, 2), qk_desc, c ? 1u : 0u);
      }
      tc_commit_elect(s_full + 8 * i);
    };
    auto pv = [&](int i, int j) {
      wait(p_full + 8 * i, j & 1);
      if (!ok) return;
      tc_fence_after();
      const uint32_t v = tile_at(2 * j + 1);
#pragma unroll
      for (int c = 0; c < kTcKeys / 16; ++c)
        tc_mma_f16_ts_elect(tmem + 256 + i * D, tmem + i * 128 + c * 8, make_smem_desc(v + c * 2048, 16384, 1024, 2), pv_desc, j | c ? 1u : 0u);
      tc_commit_elect(o_done + 8 * i);
    };
    if (ok) tile_wait(0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (steps[i]) {
        wait(q_full + 8 * i, 0);
        qk(i, 0);
      }
    if (ok) release(0);
    for (int j = 0; j < all && ok; ++j) {
      tile_wait(2 * j + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (j < steps[i]) pv(i, j);
        if (i == 1 && ok) release(2 * j + 1);
        if (j + 1 < steps[i]) {
          if (i == 0 || steps[0] <= j + 1) tile_wait(2 * j + 2);
          wait(o_done + 8 * i, j & 1);  // the weights have been read: new scores may take their place
          qk(i, j + 1);
        }
      }
      if (ok && j + 1 < all) release(2 * j + 2);
    }
    tc_commit_elect(drain);
    mbar_wait_bounded(drain, 0, a.limit, a.err, kDevErrTimeoutMma);
    __syncwarp();
  } else {
    const int i = warp / 4, row = (warp % 4) * 32 + lane, n = steps[i];
    const uint32_t quarter = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + i * 128 + quarter, t_o = tmem + 256 + i * D + quarter;
    const int of = static_cast<int>(a.ratio.of(row)), token = u.token0 + i * tokens + of, head = kv * ratio + row - of * ratio;
    const bool mine = u.ok && of < tokens && token < u.s.lq;
    const int seen = mine ? max(0, token + shift + 1) : 0;
    const float c = fabsf(a.scale) * kLog2e;
    float ref = 0.0f, sum = 0.0f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = __all_sync(~0u, mbar_wait_bounded(s_full + 8 * i, j & 1, a.limit, a.err, kDevErrTimeoutEpilogue));
      if (!ok) break;
      tc_fence_after();
      uint32_t raw[4][32];
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_ld_32x32b_x32(t_s + 32 * k, raw[k]);
      tmem_ld_wait();
      auto s = [&](int k) { return __uint_as_float(raw[k / 32][k % 32]); };
      const int limit = seen - j * kTcKeys;
      if (__any_sync(~0u, limit < kTcKeys)) {
#pragma unroll
        for (int k = 0; k < 128; ++k)
          if (k >= limit) raw[k / 32][k % 32] = 0xFF800000u;
      }
      float m[4] = {s(0), s(1), s(2), s(3)};
#pragma unroll
      for (int k = 4; k < 128; k += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = k + e + 4 < 128 ? max3(m[e], s(k + e), s(k + e + 4)) : fmaxf(m[e], s(k + e));
      const float top = fmaxf(max3(m[0], m[1], m[2]), m[3]) * c;  // -inf: nothing seen in this step
      if (j == 0) {
        ref = top == -INFINITY ? 0.0f : top;
      } else if (__any_sync(~0u, top - ref > kSlack)) {
        const float now = top - ref > kSlack ? top : ref, keep = exp2_approx(ref - now);
        ok = __all_sync(~0u, mbar_wait_bounded(o_done + 8 * i, (j - 1) & 1, a.limit, a.err, kDevErrTimeoutEpilogue));
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int k = 0; k < D; k += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + k, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
          tmem_st_32x32b_x32(t_o + k, o);
        }
        sum *= keep;
        ref = now;
      }
      const float2 by = both(c), less = both(kLift - ref);
      float2 add[2] = {both(0.0f), both(0.0f)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float2 x = fma2(make_float2(s(64 * h + 2 * k), s(64 * h + 2 * k + 1)), by, less);
          const float2 p = make_float2(exp2_approx(x.x), exp2_approx(x.y));
          add[k & 1] = add2(add[k & 1], p);
          w[k] = pack_16<T>(p.x, p.y);
        }
        tmem_st_32x32b_x32(t_s + 32 * h, w);
      }
      const float2 both_sums = add2(add[0], add[1]);
      sum += both_sums.x + both_sums.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + 8 * i);
    }
    if (n && ok) ok = __all_sync(~0u, mbar_wait_bounded(o_done + 8 * i, (n - 1) & 1, a.limit, a.err, kDevErrTimeoutEpilogue));
    tc_fence_after();
    if (ok && u.ok) {
      T* out = static_cast<T*>(a.out) + (static_cast<long long>(u.s.q0 + token) * a.hq + head) * a.d;
      const float scale = seen ? 1.0f / sum : 0.0f;
      bool fine = sum > 0.0f && sum < INFINITY;
      const bool wide = a.d % 16 == 0 && !(reinterpret_cast<uintptr_t>(a.out) & 31u);
#pragma unroll 1
      for (int k = 0; k < D; k += 32) {
        uint32_t o[32];
        if (n) {
          tmem_ld_32x32b_x32(t_o + k, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 16) {
          uint32_t y[8];
#pragma unroll
          for (int f = 0; f < 8; ++f) {
            const float2 v = seen ? make_float2(__uint_as_float(o[e + 2 * f]) * scale, __uint_as_float(o[e + 2 * f + 1]) * scale) : both(0.0f);
            if (k + e + 2 * f < a.d) fine = fine && fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY;
            y[f] = pack_16<T>(v.x, v.y);
          }
          if (mine && k + e < a.d) {
            if (wide) {
              store_32(out + k + e, y);
            } else {
              *reinterpret_cast<uint4*>(out + k + e) = make_uint4(y[0], y[1], y[2], y[3]);
              if (k + e + 8 < a.d) *reinterpret_cast<uint4*>(out + k + e + 8) = make_uint4(y[4], y[5], y[6], y[7]);
            }
          }
        }
      }
      if (a.lse && mine)
        a.lse[static_cast<long long>(u.s.q0 + token) * a.hq + head] = seen ? (ref - kLift + log2f(sum)) * (1.0f / kLog2e) : -INFINITY;
      unsigned again = __ballot_sync(~0u, seen && !fine);
      for (; again; again &= again - 1) {
        const int from = __ffs(again) - 1;
        prompt_row_with_care<T>(a, u.s.q0 + __shfl_sync(~0u, token, from), __shfl_sync(~0u, head, from), u.s.k0,
                                __shfl_sync(~0u, seen, from));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace b200q
