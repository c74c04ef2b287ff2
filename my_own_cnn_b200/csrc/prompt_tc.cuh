// Prompt attention of 16-bit types on tcgen05 (prompt_tc_kernel).
//
// One block an SM takes unit after unit: two tiles of 128 rows (token, query head of one key head), all their keys, tiles of 128 in a
// ring.  Warps 0 to 3 and 4 to 7 hold a tile of rows each, one row a thread: scores of 64 keys from TMEM, weights back over them as
// 16-bit operands of the second product; warp 8 loads by TMA, warps 9 and 11 issue a tile's products each, warp 10 finds the units.
// While a half's scores become weights the tensor core has the other half's and the other tile's products, and while the last sums of a
// unit are scaled and stored, the next one's queries and keys are on their way.
// Tensor memory: scores of A and B (two halves of 64 columns each; weights take the first 32 of a half), then the sums O of A and B (D
// columns each).
// A row's reference is not its maximum but one that may lie up to 2^8 (fp16: 2^4) below it: O is then rescaled a few times in a row of any
// length, by the threads that own it, and not with every tile.  fp16 weights are lifted by 2^11: they stay normal down to 2^-25 of
// the reference, and no more than 2^15 above it.
//
// Weights are rounded to the inputs' type for the second product, by up to 2^-11 or 2^-8 of each: results are 0.0019 off where their own
// rounding makes 0.0016 (8192 tokens bf16; fp16 0.00022 and 0.0002).  A second term a weight would leave that alone and be a second
// product over the same values: 596 us where this takes 462.
//
// 8192 tokens of one prompt, 32 / 8 heads of 128, bf16: 462 to 485 us in a replayed graph, 1160 TFLOP/s (70 % of what cuBLAS reaches in
// a burst); call after call 553 to 566, as the power limit lowers the clock.  Three things bound it at once: a product of 64 keys takes
// 48 clocks where its flops take 32 (operands from shared memory; all products alone take 400 us), a warp's exponentials 8.4 clocks
// each, and the answers between the two.  So scores come in halves of 64 keys, two of them in TMEM for each tile: a half's products run
// while the warps have the other one (whole tiles of 128 keys without a second buffer: 583 us).
#pragma once
#include "common.cuh"
#include "prompt.cuh"
#include "ptx.cuh"

namespace b200q {

constexpr int kTcKeys = 128;  // of a tile of K or V; scores and weights come in halves
constexpr int kHalf = 64;
constexpr int kTcPromptThreads = 384;
constexpr int kTcMaxStages = 8;
// Halves that the tensor core adds up: its adder truncates, some 1e-7 of a sum for 16 keys (131072 keys 8e-4 low, nearly two roundings to
// fp16).  After so many a thread adds its row's sums to those before, in fp32 with rounding: 5e-5 low at any length.
constexpr int kSegment = 128;

template <int D>
struct TcShape {
  static constexpr int kTile = 128 * D * 2;  // bytes of 128 rows
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kHead = 1024;  // barriers and units
  static constexpr int kSmem = 1024 + kHead + (2 + kStages) * kTile + 8 * 4096;  // queries, ring, results
};

// Four products of 16 of K in one elected block, fp16 or bf16 operands, fp32 sums: D (+)= A B.  Both operands 32 bytes on from slice to
// slice (K-major tiles); or A in tensor memory, 8 columns a slice, and B 16 rows of 128 bytes on (a tile of V).
__device__ __forceinline__ void tc_mma_f16_x4_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
      "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_f16_ts_x4_elect(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e, t;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\t"
      "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d),
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
// Nothing that uses these registers comes before this place: tmem_ld_wait() does not name them.
__device__ __forceinline__ void loaded(uint32_t (&v)[32]) {
  asm volatile(""
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                 "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]),
                 "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value)
    return pack_f16(lo, hi);
  else
    return pack_bf16(lo, hi);
}

// What one block does next: a sequence and the tokens of it.
struct TcUnit {
  Sequence s;
  int token0;  // of tile A in the sequence
  int kv;      // key head
  int part, from, to;  // part of the keys: steps of 128
  int ok;
};

// Halves (of 64 keys) that tile i of a unit has to do: its last token's, as far as they are the part's.
__device__ __forceinline__ int unit_halves(const TcUnit& u, int i, int tokens) {
  const int first = u.token0 + i * tokens, last = min(u.s.lq, first + tokens) - 1;
  const int all = first < u.s.lq ? (max(0, last + u.s.lk - u.s.lq + 1) + kHalf - 1) / kHalf : 0;
  return max(0, min(all, 2 * u.to) - 2 * u.from);
}

// before = before keep + O of this thread's row; O alone the first time.
template <int D>
__device__ __noinline__ void take_sums(float (&before)[D], uint32_t t_o, bool first, float keep) {
#pragma unroll 1
  for (int k = 0; k < D; k += 32) {
    uint32_t o[32];
    tmem_ld_32x32b_x32(t_o + k, o);
    tmem_ld_wait();
    loaded(o);
#pragma unroll
    for (int e = 0; e < 32; ++e) before[k + e] = first ? __uint_as_float(o[e]) : fmaf(before[k + e], keep, __uint_as_float(o[e]));
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcPromptThreads, 1)
    prompt_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PromptArgs a, const uint32_t negate) {
  using S = TcShape<D>;
  constexpr int kChunks = D / 64;  // 128-byte columns of a tile
  constexpr float kSlack = std::is_same<T, __half>::value ? 4.0f : 8.0f;  // log2 of how far a row's maximum may pass its reference
  constexpr int kLift = std::is_same<T, __half>::value ? 11 : 0;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kTcMaxStages;
  const uint32_t q_full = full0 + 16 * kTcMaxStages, q_empty = q_full + 16, o_done = q_empty + 16;
  const uint32_t s_full = o_done + 16, p_full = s_full + 32;  // [tile][half]
  const uint32_t u_full = p_full + 32, u_empty = u_full + 16, drain = u_empty + 16;
  const uint32_t ended = drain + 16;  // a tile's last product of a unit
  uint32_t* slot = reinterpret_cast<uint32_t*>(bars + 2 * kTcMaxStages + 22);
  TcUnit* units = reinterpret_cast<TcUnit*>(bars + 2 * kTcMaxStages + 23);  // two
  const uint32_t s_q = smem_u32(smem) + S::kHead, s_ring = s_q + 2 * S::kTile, s_out = s_ring + S::kStages * S::kTile;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int ratio = static_cast<int>(a.ratio.d), tokens = static_cast<int>(a.tile.d) / 2;  // of one tile

  if (threadIdx.x == 256) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 2);  // both tiles' products
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(o_done + 8 * i, 1);
      mbar_init(ended + 8 * i, 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(s_full + 16 * i + 8 * b, 1);
        mbar_init(p_full + 16 * i + 8 * b, 4);
      }
      mbar_init(u_full + 8 * i, 1);
      mbar_init(u_empty + 8 * i, 11);  // loader, issuers, the tiles' eight warps
      mbar_init(drain + 8 * i, 1);
    }
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
  // The block's r-th unit in the units' order, every other round backwards.
  auto find = [&](Finder& finder, int r, TcUnit* to) {
    const long long n = static_cast<long long>(r) * gridDim.x + (r & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    PromptUnit u{};
    const long long whole = n / a.parts;
    if (n < a.most_units) u = finder(static_cast<int>(whole / a.hk));
    if (lane == 0) {
      TcUnit v{u.s, u.tile * static_cast<int>(a.tile.d), static_cast<int>(whole % a.hk), static_cast<int>(n - whole * a.parts), 0, 0, u.ok};
      const int last = min(u.s.lq, v.token0 + static_cast<int>(a.tile.d)) + u.s.lk - u.s.lq;  // keys of the unit's last token
      const int2 steps = part_steps(a, (max(0, last) + kTcKeys - 1) / kTcKeys, v.part);
      v.from = steps.x, v.to = steps.y;
      *to = v;
    }
    return u.ok;
  };
  if (warp == 10) {
    Finder finder(a, blockIdx.x == 0);
    find(finder, 0, units);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(~0u, *slot, 0);

  bool ok = true;  // no wait has run out
  auto wait = [&](uint32_t bar, uint32_t parity, int code) {
    ok = ok && __all_sync(~0u, mbar_wait_bounded(bar, parity, a.limit, a.err, code));
    return ok;
  };
  // The block's r-th unit (every warp that works on units asks for each of them once); ok == 0: there is none.
  auto unit_at = [&](int r, int code) {
    TcUnit u{};
    if (!wait(u_full + 8 * (r & 1), (r >> 1) & 1, code)) return u;
    u = units[r & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(u_empty + 8 * (r & 1));
    return u;
  };

  // The tiles' threads hold a row's 128 scores: registers go to them, 12 warps x 168 = 8 x 200 + 4 x 104.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    constexpr int kCode = kDevErrTimeoutEpilogue;
    const int i = warp / 4, row = (warp % 4) * 32 + lane;
    const uint32_t quarter = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + i * 128 + quarter, t_o = tmem + 256 + i * D + quarter;
    const int of = static_cast<int>(a.ratio.of(row));
    const float c = fabsf(a.scale) * kLog2e;
    const uint32_t stage = s_out + warp * 4096;  // 64 channels of the warp's rows
    uint32_t done = 0, units_of = 0, used = 0;  // halves and units so far; a bit for each half's buffer: its next phase
    for (int r = 0;; ++r) {
      const TcUnit u = unit_at(r, kCode);
      if (!u.ok) break;
      const int n = unit_halves(u, i, tokens), shift = u.s.lk - u.s.lq;
      const int first = u.token0 + i * tokens, token = first + of, head = u.kv * ratio + row - of * ratio;
      if (first >= u.s.lq) continue;
      const bool mine = of < tokens && token < u.s.lq;
      const int seen = mine ? max(0, token + shift + 1) : 0;
      float ref = 0.0f, sum = 0.0f;
      float before[D], held = -INFINITY;  // sums of the segments before (indexed as it runs: local memory), at this reference
      for (int t = 0;;) {
        for (const int stop = min(n, t + kSegment); t < stop; ++t) {
          const uint32_t half = t & 1, t_h = t_s + 64 * half;
          if (!wait(s_full + 16 * i + 8 * half, used >> half & 1, kCode)) break;
          used ^= 1u << half;
          tc_fence_after();
          uint32_t raw[2][32];
          tmem_ld_32x32b_x32(t_h, raw[0]);
          tmem_ld_32x32b_x32(t_h + 32, raw[1]);
          tmem_ld_wait();
          loaded(raw[0]);
          loaded(raw[1]);
          const auto s = [&](int k) { return __uint_as_float(raw[k / 32][k % 32]); };
          const int limit = seen - 2 * u.from * kHalf - t * kHalf;
          if (__any_sync(~0u, limit < kHalf)) {
#pragma unroll
            for (int k = 0; k < kHalf; ++k)
              if (k >= limit) raw[k / 32][k % 32] = 0xFF800000u;
          }
          float m[2] = {s(0), s(1)};
#pragma unroll
          for (int k = 2; k < kHalf - 2; k += 4) m[0] = max3(m[0], s(k), s(k + 1)), m[1] = max3(m[1], s(k + 2), s(k + 3));
          const float top = max3(max_nan(m[0], m[1]), s(kHalf - 2), s(kHalf - 1)) * c;  // -inf: nothing seen here
          // nothing but scores of -inf so far: the sums are zero at any reference
          if (sum == 0.0f) ref = top == -INFINITY ? 0.0f : top;
          if (__any_sync(~0u, top - ref > kSlack)) {  // never at t = 0: there are no sums yet
            const float now = top - ref > kSlack ? top : ref, keep = exp2_approx(ref - now);
            if (!wait(o_done + 8 * i, (done + t - 1) & 1, kCode)) break;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D; k += 32) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(t_o + k, o);
              tmem_ld_wait();
              loaded(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmem_st_32x32b_x32(t_o + k, o);
            }
            sum *= keep;
            ref = now;
          }
          if (top != top) ref = top;  // a score that is NaN: the row's, whatever else there is
          const float less = kLift - ref;
          float add[4] = {};
          uint32_t w[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            const float x = exp2_approx(fmaf(s(2 * k), c, less)), y = exp2_approx(fmaf(s(2 * k + 1), c, less));
            add[2 * (k & 1)] += x;
            add[2 * (k & 1) + 1] += y;
            w[k] = pack_16<T>(x, y);
          }
          tmem_st_32x32b_x32(t_h, w);
          sum += (add[0] + add[1]) + (add[2] + add[3]);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full + 16 * i + 8 * half);
        }
        if (t >= n || !ok) break;
        // The next scores, which are waited for again below, come after the last product but one: so the barrier is in the last one's phase, or
        // past it by one.
        if (!wait(s_full + 16 * i + 8 * (t & 1), used >> (t & 1) & 1, kCode) || !wait(o_done + 8 * i, (done + t - 1) & 1, kCode)) break;
        tc_fence_after();
        take_sums<D>(before, t_o, t == kSegment, exp2_approx(held - ref));
        held = sum == 0.0f ? -INFINITY : ref;
      }
      const float keep = exp2_approx(held - ref);
      const auto with_before = [&](uint32_t (&o)[32], int k) {
        if (n <= kSegment) return;
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(fmaf(before[k + e], keep, __uint_as_float(o[e])));
      };
      done += n;
      if (n) wait(ended + 8 * i, units_of++ & 1, kCode);
      if (!ok) break;
      tc_fence_after();
      if (a.parts > 1) {
        const long long row_at = static_cast<long long>(u.s.q0 + token) * a.hq + head;
        if (mine) part_head(a, u.part, row_at, n && seen > u.from * kTcKeys, ref - kLift, sum, u.s.k0, seen);
        float* sums = a.part_sums + (u.part * static_cast<long long>(a.tq) * a.hq + row_at) * a.d;
#pragma unroll 1
        for (int k = 0; n && k < a.d; k += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(t_o + k, o);
          tmem_ld_wait();
          loaded(o);
          with_before(o, k);
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (mine && k + e < a.d) *reinterpret_cast<uint4*>(sums + k + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
        continue;
      }
      // Results: whole rows by way of the warp's own shared memory (16-byte piece p of a row's 128 bytes at p ^ (row % 8)), so that
      // 8 lanes write 128 bytes together; a thread that writes its own row takes as many cycles as it has sectors.
      const float scale = seen ? 1.0f / sum : 0.0f;
      const long long at = (static_cast<long long>(u.s.q0 + token) * a.hq + head) * a.d;
      float most = 0.0f;  // in size; NaN if one is
#pragma unroll 1
      for (int ch = 0; 64 * ch < a.d; ++ch) {
#pragma unroll
        for (int k = 0; k < 64; k += 32) {
          uint32_t o[32], y[16];
          if (n) {
            tmem_ld_32x32b_x32(t_o + 64 * ch + k, o);
            tmem_ld_wait();
            loaded(o);
            with_before(o, 64 * ch + k);
          }
          const auto at_scale = [&](int f) { return mul2(make_float2(__uint_as_float(o[2 * f]), __uint_as_float(o[2 * f + 1])), both(scale)); };
#pragma unroll
          for (int f = 0; f < 16; ++f) {
            const float2 v = at_scale(f);
            most = max3(most, fabsf(v.x), fabsf(v.y));
            y[f] = seen ? pack_16<T>(v.x, v.y) : 0u;
          }
          if (std::is_same<T, __half>::value && __any_sync(~0u, seen && most > kHalfMost)) {
#pragma unroll
            for (int f = 0; f < 16; ++f) {
              const float2 v = at_scale(f);
              y[f] = seen ? pack_16<T>(to_half_range(v.x), to_half_range(v.y)) : 0u;
            }
          }
#pragma unroll
          for (int f = 0; f < 4; ++f)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + (((k / 8 + f) ^ (lane & 7)) << 4)),
                         "r"(y[4 * f]), "r"(y[4 * f + 1]), "r"(y[4 * f + 2]), "r"(y[4 * f + 3])
                         : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int from = 4 * k + lane / 8, piece = lane & 7;
          const long long to = __shfl_sync(~0u, mine ? at : -1, from);
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(stage + from * 128 + ((piece ^ (from & 7)) << 4))
                       : "memory");
          if (to >= 0 && 64 * ch + 8 * piece < a.d) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + to + 64 * ch + 8 * piece) = v;
        }
        __syncwarp();
      }
      const bool fine = !seen || (sum > 0.0f && sum < INFINITY && most < INFINITY);
      if (a.lse && mine)
        a.lse[static_cast<long long>(u.s.q0 + token) * a.hq + head] = seen ? log_sum<kLift>(ref, sum) : -INFINITY;
      if (const unsigned rows = __ballot_sync(~0u, !fine); __builtin_expect(rows != 0, 0)) {
        __syncwarp();  // these results and log-sums before those that other lanes write in their place
        prompt_rows_again<T>(a, rows, u.s.q0 + token, head, u.s.k0, seen, prompt_sums<T>(a, ref, sum));
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 10) {
      Finder finder(a, false);
      bool more = units[0].ok;
      if (lane == 0) mbar_arrive(u_full);
      for (int r = 1; more; ++r) {
        if (r > 1 && !wait(u_empty + 8 * (r & 1), ((r >> 1) - 1) & 1, kDevErrTimeoutProducer)) break;
        more = find(finder, r, units + (r & 1));
        if (lane == 0) mbar_arrive(u_full + 8 * (r & 1));
        __syncwarp();
      }
    } else if (warp == 8) {
      uint32_t n = 0, loads[2] = {0, 0};
      for (int r = 0;; ++r) {
        const TcUnit u = unit_at(r, kDevErrTimeoutProducer);
        if (!u.ok) break;
        const int kv = u.kv;
        int all = 0;
        bool go = true;
  #pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int halves = unit_halves(u, i, tokens);
          all = max(all, (halves + 1) / 2);
          if (!halves || !go) continue;
          if (loads[i]) go = wait(q_empty + 8 * i, (loads[i] - 1) & 1, kDevErrTimeoutProducer);
          if (!go) continue;
          mbar_arrive_expect_tx_elect(q_full + 8 * i, static_cast<uint32_t>(kChunks * tokens * ratio) * 128u);
          for (int c = 0; c < kChunks; ++c)
            tma_load_3d_elect(s_q + i * S::kTile + c * 16384, &tm_q, q_full + 8 * i, 64 * c, kv * ratio, u.s.q0 + u.token0 + i * tokens);
          ++loads[i];
        }
        for (int k = 0; k < 2 * all && go; ++k, ++n) {  // K 0, V 0, K 1, V 1, ...
          const uint32_t st = n % S::kStages;
          if (n >= S::kStages) go = wait(empty0 + 8 * st, (n / S::kStages - 1) & 1, kDevErrTimeoutProducer);
          if (!go) break;
          mbar_arrive_expect_tx_elect(full0 + 8 * st, S::kTile);
          for (int c = 0; c < kChunks; ++c)
            tma_load_3d_elect(s_ring + st * S::kTile + c * 16384, k & 1 ? &tm_v : &tm_k, full0 + 8 * st, 64 * c, kv, u.s.k0 + (u.from + k / 2) * kTcKeys);
        }
        if (!go) break;
      }
      if (!ok) {  // given up: what is on its way lands before the block ends
        for (uint32_t i = n > S::kStages ? n - S::kStages : 0; i < n; ++i)
          mbar_wait_bounded(full0 + 8 * (i % S::kStages), (i / S::kStages) & 1, a.limit, a.err, kDevErrTimeoutProducer);
        for (int i = 0; i < 2; ++i)
          if (loads[i]) mbar_wait_bounded(q_full + 8 * i, (loads[i] - 1) & 1, a.limit, a.err, kDevErrTimeoutProducer);
        __syncwarp();
      }
    } else {
      // A warp for each tile issues its products: QK of the next half while the weights of this one are made, then PV.
      constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
      constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) | ((128u >> 4) << 24);
      const uint32_t qk_desc = kDesc | ((kHalf >> 3) << 17) | (negate << 13);
      const uint32_t pv_desc = kDesc | ((static_cast<uint32_t>(D) >> 3) << 17) | (1u << 16);  // V: channels contiguous
      constexpr int kCode = kDevErrTimeoutMma;
      const uint64_t q_at = make_smem_desc(s_q, 16, 1024, 2), k_at = make_smem_desc(s_ring, 16, 1024, 2),
                     v_at = make_smem_desc(s_ring, 16384, 1024, 2);
      const int i = warp == 9 ? 0 : 1;
      const uint32_t t_s = tmem + i * 128, t_o = tmem + 256 + i * D;
      const uint64_t q = q_at + i * (S::kTile / 16);
      uint32_t base = 0, done = 0, units_of = 0, used = 0;  // ring tiles, halves and units so far; the buffers' phases
      auto tile_wait = [&](uint32_t n) { return wait(full0 + 8 * (n % S::kStages), (n / S::kStages) & 1, kCode); };
      auto release = [&](uint32_t n) { tc_commit_elect(empty0 + 8 * (n % S::kStages)); };
      for (int r = 0; ok; ++r) {
        const TcUnit u = unit_at(r, kCode);
        if (!u.ok) break;
        const int n = unit_halves(u, i, tokens), all = (max(n, unit_halves(u, 1 - i, tokens)) + 1) / 2;
        // end of the keys that the unit sees, and the half that it cuts
        const int end = min(u.s.lq, u.token0 + 2 * tokens) + u.s.lk - u.s.lq, cut = end % kHalf ? end / kHalf - 2 * u.from : -1;
        auto qk = [&](int t) {
          const uint32_t at = base + (t & ~1);
          if (!(t & 1) && !tile_wait(at)) return;
          const uint64_t k = k_at + at % S::kStages * (S::kTile / 16) + (t & 1) * (kHalf * 8);
#pragma unroll
          for (int c = 0; c < kChunks; ++c) tc_mma_f16_x4_elect(t_s + (t & 1) * kHalf, q + c * 1024, k + c * 1024, qk_desc, c);
          tc_commit_elect(s_full + 16 * i + 8 * (t & 1));
          if ((t & 1) || t + 1 == n) release(at);
          if (t + 1 == n) tc_commit_elect(q_empty + 8 * i);
        };
        if (n) {
          // the last unit's weights have been read: scores may take their place
          if (units_of) wait(ended + 8 * i, (units_of - 1) & 1, kCode);
          if (wait(q_full + 8 * i, units_of++ & 1, kCode)) qk(0);
        }
        for (int t = 0; t < n && ok; ++t) {
          if (t + 1 < n) {  // in the place of the weights before the last
            if (t && !wait(o_done + 8 * i, (done + t - 1) & 1, kCode)) break;
            qk(t + 1);
          }
          if (!(t & 1) && !tile_wait(base + t + 1)) break;
          if (t == cut) {
            // Values behind that end (another sequence's, or nobody's) become zeros while the weights are made: weights of zero would let a
            // NaN or an infinity there through.  Both tiles' warps do so, each before its own product; until both have issued theirs the
            // ring's tile stays.
            const uint32_t v = s_ring + (base + (t | 1)) % S::kStages * S::kTile + (t & 1) * (kHalf * 128);
#pragma unroll 1
            for (int k = end % kHalf * 8 + lane; k < kHalf * 8; k += 32)
#pragma unroll
              for (int c = 0; c < kChunks; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v + c * 16384 + k * 16), "r"(0) : "memory");
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (!wait(p_full + 16 * i + 8 * (t & 1), used >> (t & 1) & 1, kCode)) break;
          used ^= 1u << (t & 1);
          tc_fence_after();
          tc_mma_f16_ts_x4_elect(t_o, t_s + (t & 1) * kHalf, v_at + (base + (t | 1)) % S::kStages * (S::kTile / 16) + (t & 1) * 512,
                                 pv_desc, t % kSegment);
          tc_commit_elect(o_done + 8 * i);
          if ((t & 1) || t + 1 == n) release(base + (t | 1));
          if (t + 1 == n) tc_commit_elect(ended + 8 * i);
        }
        for (int k = (n + 1) / 2 * 2; k < 2 * all && ok; ++k)  // the other tile's alone
          if (tile_wait(base + k)) release(base + k);
        base += 2 * all;
        done += n;
      }
      tc_commit_elect(drain + 8 * i);
      mbar_wait_bounded(drain + 8 * i, 0, a.limit, a.err, kCode);
      __syncwarp();
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
