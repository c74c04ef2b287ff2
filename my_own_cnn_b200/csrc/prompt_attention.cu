// Causal attention over packed prompts (b200q_prompt_attention).
//
//   o_i = sum_j p_ij v_j / l_i,  p_ij = exp(s_ij - m_i),  s_ij = scale q_i k_j,  m_i = max_j s_ij,  l_i = sum_j p_ij,  j <= i + lk - lq
//
// prompt_mma_kernel: mma.sync.m16n8k16, for fp32 and for rows that TMA cannot take.  A block has 64 rows (token, query
// head of one key head) in four warps and goes through the keys 64 at a time; scores, weights and sums stay in registers, the
// maximum and the sum of a row run along.  fp32 operands are three bf16 terms, cut off one after another: 8 + 8 + 8
// bits, so the terms are the value; six products (0 0, 0 1, 1 0, 1 1, 0 2, 2 0) leave 2^-24 of it out.  The first is added with
// rounding.  Five prompts of 1531 tokens in all, 16 heads of 64, fp32: 65 us (the six products take 8 GFLOP): latency, one block of
// four warps a tile and as many blocks as tiles; 1024 tokens of 16 heads run the tensor pipe at 30 %, issue slots at 29 %.  16-bit types round
// weights to theirs, as prompt_tc_kernel does: 8192 tokens, 16 / 8 heads of 256, bf16 10.8 ms (51 TFLOP/s).
#include <algorithm>
#include <atomic>
#include <cmath>

#include "prompt.cuh"
#include "prompt_tc.cuh"

namespace b200q {
namespace {

constexpr int kRows = 64;
constexpr int kMmaThreads = 128;

// Operand words: two 16-bit values in every term.
template <typename T>
struct Terms {
  static constexpr int kCount = 1;
  // log2 of what weights are multiplied by, up to 1 without: fp16's are normal down to 2^-29 so (the largest is 2^15).
  static constexpr int kLift = std::is_same<T, __half>::value ? 15 : 0;
  static __device__ __forceinline__ void cut(float a, float b, uint32_t (&w)[1]) {
    if constexpr (sizeof(T) == 2) w[0] = std::is_same<T, __half>::value ? pack_f16(a, b) : pack_bf16(a, b);
  }
};
template <>
struct Terms<float> {
  static constexpr int kCount = 3;
  static constexpr int kLift = 0;
  static __device__ __forceinline__ void cut(float a, float b, uint32_t (&w)[3]) {
    float x[2] = {a, b};
    uint32_t t[3][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      t[0][i] = __float_as_uint(x[i]) & 0xFFFF0000u;
      const float r = fabsf(x[i]) < INFINITY ? x[i] - __uint_as_float(t[0][i]) : 0.0f;
      t[1][i] = __float_as_uint(r) & 0xFFFF0000u;
      t[2][i] = __float_as_uint(r - __uint_as_float(t[1][i]));
      // a NaN may have its bits among those cut off
      if (x[i] != x[i]) t[0][i] = 0x7FC00000u;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i] = __byte_perm(t[i][0], t[i][1], 0x7632);
  }
};

template <typename T>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
  else
    mma_bf16(c, a[0], a[1], a[2], a[3], b0, b1);
}
// c += a b on bf16 with the addition rounded: the instruction's own adder truncates, which in 24 additions of a row of
// scores adds up to 2e-6 of fp32 outputs (4e-7 so).  16-bit types add the sums of 64 values that way: 131072 keys were 8e-4 low without.
__device__ __forceinline__ void add_product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  float r[4];
  mma_bf16_first(r, a[0], a[1], a[2], a[3], b0, b1);
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] += r[e];
}
// The sum of the first terms' products and the others'.  Where a factor is infinite the others are NaN (its term times a zero) and the first
// has the value.
__device__ __forceinline__ float with_less(float first, float less) { return fabsf(first) == INFINITY ? first : first + less; }
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T, int D>
struct MmaShape {
  static constexpr int kTerms = Terms<T>::kCount;
  static constexpr int kKeys = kTerms == 3 && D == 256 ? 32 : 64;
  static constexpr int kPitch = D * 2 + 16;  // bytes: eight rows of a matrix in eight bank groups
  static constexpr int kQ = kRows * kPitch, kK = kKeys * kPitch;  // one term
  static constexpr int kSmem = kTerms * (kQ + 2 * kK);
};

// Four channels from c on of a row (null: zeros; past d too).
template <typename T>
__device__ __forceinline__ float4 four_of(const T* p, int c, int d, bool wide) {
  float x[4] = {};
  if (p) {
    if (wide && c + 4 <= d) {
      if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4*>(p + c);
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p + c);
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = to_f32(e[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < d) x[j] = to_f32(p[c + j]);
    }
  }
  return make_float4(x[0], x[1], x[2], x[3]);
}

// A thread's pieces of `ROWS` rows of D channels: from memory into registers, and cut into the terms' tiles.
template <typename T, int D, int ROWS>
struct Tile {
  static constexpr int kPieces = ROWS * (D / 4) / kMmaThreads;
  template <typename P>
  static __device__ __forceinline__ void fetch(float4 (&x)[kPieces], int d, bool wide, P row_at) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int i = threadIdx.x + k * kMmaThreads;
      x[k] = four_of<T>(row_at(i / (D / 4)), i % (D / 4) * 4, d, wide);
    }
  }
  static __device__ __forceinline__ void put(uint32_t to, int term, const float4& x, int i) {
    constexpr int kTerms = Terms<T>::kCount;
    uint32_t lo[kTerms], hi[kTerms];
    Terms<T>::cut(x.x, x.y, lo);
    Terms<T>::cut(x.z, x.w, hi);
#pragma unroll
    for (int t = 0; t < kTerms; ++t)
      asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + t * term + i / (D / 4) * (D * 2 + 16) + i % (D / 4) * 8), "r"(lo[t]),
                   "r"(hi[t])
                   : "memory");
  }
  static __device__ __forceinline__ void put(uint32_t to, int term, const float4 (&x)[kPieces]) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) put(to, term, x[k], threadIdx.x + k * kMmaThreads);
  }
  // From memory to the tiles, eight pieces on their way at a time.
  template <typename P>
  static __device__ __forceinline__ void load(uint32_t to, int term, int d, bool wide, P row_at) {
    constexpr int kAtOnce = kPieces < 8 ? kPieces : 8;
#pragma unroll 1
    for (int k0 = 0; k0 < kPieces; k0 += kAtOnce) {
      float4 x[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int i = threadIdx.x + (k0 + k) * kMmaThreads;
        x[k] = four_of<T>(row_at(i / (D / 4)), i % (D / 4) * 4, d, wide);
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) put(to, term, x[k], threadIdx.x + (k0 + k) * kMmaThreads);
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kMmaThreads) prompt_mma_kernel(const __grid_constant__ PromptArgs a, int wide) {
  using S = MmaShape<T, D>;
  constexpr int kTerms = S::kTerms, kKeys = S::kKeys;
  // The products of the terms but for the first ones'.
  constexpr int kA[5] = {2, 0, 1, 1, 0}, kB[5] = {0, 2, 1, 0, 1};
  extern __shared__ __align__(16) uint8_t smem[];
  wait_for_previous();
  const int part = static_cast<int>(blockIdx.x % a.parts), whole = static_cast<int>(blockIdx.x / a.parts);
  const int kv = whole % a.hk, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Finder finder(a, blockIdx.x == 0 && threadIdx.x < 32);
  const PromptUnit u = finder(whole / a.hk);
  if (!u.ok) return;
  const int ratio = static_cast<int>(a.ratio.d), shift = u.s.lk - u.s.lq;
  const int rows = u.s.lq * ratio, row0 = u.tile * kRows;  // of this key head's rows in the sequence
  const uint32_t s_q = shared_address(smem), s_k = s_q + kTerms * S::kQ, s_v = s_k + kTerms * S::kK;
  Tile<T, D, kRows>::load(s_q, S::kQ, a.d, wide, [&](int r) -> const T* {
    if (row0 + r >= rows) return nullptr;
    const int token = static_cast<int>(a.ratio.of(row0 + r)), head = kv * ratio + row0 + r - token * ratio;
    return static_cast<const T*>(a.q) + (u.s.q0 + token) * a.q_ts + head * a.q_hs;
  });
  // keys that a row of this lane sees: rows g and g + 8 of the warp's 16
  const int g = lane / 4, t = lane % 4, last_row = min(rows, row0 + kRows) - 1;
  int seen[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = row0 + warp * 16 + g + 8 * h;
    seen[h] = r < rows ? max(0, static_cast<int>(a.ratio.of(r)) + shift + 1) : 0;
  }
  const int all = max(0, min(u.s.lk, static_cast<int>(a.ratio.of(last_row)) + shift + 1));
  const int2 steps = part_steps(a, (all + kKeys - 1) / kKeys, part);
  const int least = steps.x * kKeys, most = min(all, steps.y * kKeys);
  const float c = a.scale * kLog2e;
  constexpr int kLift = Terms<T>::kLift;
  float o[D / 8][4] = {}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {};
  // Heads of up to 64 channels: the next keys and values are on their way, in registers, while these are worked on.
  using KV = Tile<T, D, kKeys>;
  constexpr bool kAhead = D == 64;
  float4 next_k[kAhead ? KV::kPieces : 1], next_v[kAhead ? KV::kPieces : 1];
  // what lies behind the last key that the tile sees is zeros: a weight of zero would let a NaN or an infinity there through
  const auto key_rows = [&](const void* base, long long ts, long long hs, int j0) {
    return [=](int r) -> const T* {
      return j0 + r < all ? static_cast<const T*>(base) + (u.s.k0 + j0 + r) * ts + kv * hs : nullptr;
    };
  };
  if constexpr (kAhead) {
    if (most > least) {
      KV::fetch(next_k, a.d, wide, key_rows(a.k, a.k_ts, a.k_hs, least));
      KV::fetch(next_v, a.d, wide, key_rows(a.v, a.v_ts, a.v_hs, least));
    }
  }
  for (int j0 = least; j0 < most; j0 += kKeys) {
    __syncthreads();
    if constexpr (kAhead) {
      KV::put(s_k, S::kK, next_k);
      KV::put(s_v, S::kK, next_v);
      if (j0 + kKeys < most) {
        KV::fetch(next_k, a.d, wide, key_rows(a.k, a.k_ts, a.k_hs, j0 + kKeys));
        KV::fetch(next_v, a.d, wide, key_rows(a.v, a.v_ts, a.v_hs, j0 + kKeys));
      }
    } else {
      KV::load(s_k, S::kK, a.d, wide, key_rows(a.k, a.k_ts, a.k_hs, j0));
      KV::load(s_v, S::kK, a.d, wide, key_rows(a.v, a.v_ts, a.v_hs, j0));
    }
    __syncthreads();
    float s[kKeys / 8][4] = {}, less[kTerms == 3 ? kKeys / 8 : 1][4] = {};
#pragma unroll 2
    for (int kc = 0; kc < D; kc += 16) {
      uint32_t q[kTerms][4];
#pragma unroll
      for (int i = 0; i < kTerms; ++i)
        load_matrices(q[i], s_q + i * S::kQ + (warp * 16 + lane % 16) * S::kPitch + (kc + lane / 16 * 8) * 2);
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {
        uint32_t k[kTerms][4];
#pragma unroll
        for (int i = 0; i < kTerms; ++i)
          load_matrices(k[i], s_k + i * S::kK + (n * 16 + lane % 8 + lane / 16 * 8) * S::kPitch + (kc + lane / 8 % 2 * 8) * 2);
        if constexpr (kTerms == 1) {
          mma_16<T>(s[2 * n], q[0], k[0][0], k[0][1]);
          mma_16<T>(s[2 * n + 1], q[0], k[0][2], k[0][3]);
        } else {
#pragma unroll
          for (int p = 0; p < 5; ++p) {
            mma_16<T>(less[2 * n], q[kA[p]], k[kB[p]][0], k[kB[p]][1]);
            mma_16<T>(less[2 * n + 1], q[kA[p]], k[kB[p]][2], k[kB[p]][3]);
          }
          add_product(s[2 * n], q[0], k[0][0], k[0][1]);
          add_product(s[2 * n + 1], q[0], k[0][2], k[0][3]);
        }
      }
    }
    if constexpr (kTerms == 3) {
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = with_less(s[n][e], less[n][e]);
    }
    // softmax: the exponent's base is 2, the scale is in it
    float now[2] = {top[0], top[1]}, from[2];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = j0 + n * 8 + 2 * t + (e & 1) < seen[e / 2] ? s[n][e] * c : -INFINITY;
        now[e / 2] = max_nan(now[e / 2], s[n][e]);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      now[h] = max_nan(now[h], __shfl_xor_sync(~0u, now[h], 1));
      now[h] = max_nan(now[h], __shfl_xor_sync(~0u, now[h], 2));
      from[h] = now[h] == -INFINITY ? 0.0f : now[h];
      const float keep = exp2_approx(top[h] - from[h]);
      from[h] -= kLift;
      top[h] = now[h];
      sum[h] *= keep;
#pragma unroll
      for (int n = 0; n < D / 8; ++n) o[n][2 * h] *= keep, o[n][2 * h + 1] *= keep;
    }
    float add[2] = {};  // of few keys alone, then to the sum: a long row's small weights are not rounded off one by one
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2_approx(s[n][e] - from[e / 2]);
        add[e / 2] += s[n][e];
      }
    sum[0] += add[0], sum[1] += add[1];
    uint32_t p[kKeys / 16][kTerms][4];
#pragma unroll
    for (int kc = 0; kc < kKeys / 16; ++kc)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[kTerms];
        Terms<T>::cut(s[2 * kc + e / 2][e % 2 * 2], s[2 * kc + e / 2][e % 2 * 2 + 1], w);
#pragma unroll
        for (int i = 0; i < kTerms; ++i) p[kc][i][e] = w[i];
      }
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      float small[2][4] = {};
#pragma unroll
      for (int kc = 0; kc < kKeys / 16; ++kc) {
        uint32_t v[kTerms][4];
#pragma unroll
        for (int i = 0; i < kTerms; ++i)
          load_matrices_t(v[i], s_v + i * S::kK + (kc * 16 + lane % 16) * S::kPitch + (n * 16 + lane / 16 * 8) * 2);
        if constexpr (kTerms == 1) {
          mma_16<T>(small[0], p[kc][0], v[0][0], v[0][1]);
          mma_16<T>(small[1], p[kc][0], v[0][2], v[0][3]);
        } else {
#pragma unroll
          for (int i = 0; i < 5; ++i) {
            mma_16<T>(small[0], p[kc][kA[i]], v[kB[i]][0], v[kB[i]][1]);
            mma_16<T>(small[1], p[kc][kA[i]], v[kB[i]][2], v[kB[i]][3]);
          }
          add_product(o[2 * n], p[kc][0], v[0][0], v[0][1]);
          add_product(o[2 * n + 1], p[kc][0], v[0][2], v[0][3]);
        }
      }
      if constexpr (kTerms == 1) {  // added with rounding, as below
#pragma unroll
        for (int e = 0; e < 4; ++e) o[2 * n][e] += small[0][e], o[2 * n + 1][e] += small[1][e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[2 * n][e] = with_less(o[2 * n][e], small[0][e]);
          o[2 * n + 1][e] = with_less(o[2 * n + 1][e], small[1][e]);
        }
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = row0 + warp * 16 + g + 8 * h;
    float l = sum[h];
    l += __shfl_xor_sync(~0u, l, 1);
    l += __shfl_xor_sync(~0u, l, 2);
    const int token = static_cast<int>(a.ratio.of(min(r, rows - 1))), head = kv * ratio + min(r, rows - 1) - token * ratio;
    const long long at = static_cast<long long>(u.s.q0 + token) * a.hq + head;
    if (a.parts > 1) {
      if (r < rows) {
        if (t == 0) part_head(a, part, at, most > least && seen[h] > least, top[h] - kLift, l, u.s.k0, min(u.s.lk, seen[h]));
        float* sums = a.part_sums + (part * static_cast<long long>(a.tq) * a.hq + at) * a.d;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (n * 8 + 2 * t + e < a.d) sums[n * 8 + 2 * t + e] = o[n][2 * h + e];
      }
      continue;
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    bool fine = l > 0.0f && l < INFINITY;
    if (r < rows) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float y = o[n][2 * h + e] * by;
          fine = fine && fabsf(y) < INFINITY;
          if (n * 8 + 2 * t + e < a.d) static_cast<T*>(a.out)[at * a.d + n * 8 + 2 * t + e] = result<T>(seen[h] ? y : 0.0f);
        }
      if (a.lse && t == 0) a.lse[at] = seen[h] ? log_sum<Terms<T>::kLift>(top[h], l) : -INFINITY;
    }
    unsigned again = __ballot_sync(~0u, r < rows && seen[h] && !fine);
    again |= again >> 1;
    again = (again | again >> 2) & 0x11111111u;  // one bit a row
    __syncwarp();
    if (again) prompt_rows_again<T>(a, again, u.s.q0 + token, head, u.s.k0, min(u.s.lk, seen[h]), prompt_sums<T>(a, top[h], l));
  }
}

template <typename T, int D>
int launch_mma(const PromptArgs& a, bool wide, long long units, int device, cudaStream_t cs) {
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[device].load(std::memory_order_relaxed)) {
    const cudaError_t e =
        cudaFuncSetAttribute(prompt_mma_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, MmaShape<T, D>::kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(prompt_mma_kernel)");
    ready[device].store(true, std::memory_order_relaxed);
  }
  return host_launch("prompt_mma_kernel launch", prompt_mma_kernel<T, D>, dim3(static_cast<unsigned>(units)), kMmaThreads,
                     MmaShape<T, D>::kSmem, cs, 1, a, wide ? 1 : 0);
}

// 16-bit heads of up to 128 channels whose addresses and strides a tensor map takes.  A scale of zero would multiply the
// masked scores' infinities.
bool tensor_core_takes(const b200q_prompt_attention_args& p, long long ratio) {
  if (p.ftype == B200Q_F32 || p.d > 128 || p.d % 8 || ratio > 128 || p.scale == 0.0f || p.tk == 0) return false;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                         reinterpret_cast<uintptr_t>(p.out);
  if (bits & 15u) return false;
  const auto fits = [](int64_t stride, int count) { return count == 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); };
  return fits(p.q_ts, p.tq) && fits(p.q_hs, p.hq) && fits(p.k_ts, p.tk) && fits(p.k_hs, p.hk) && fits(p.v_ts, p.tk) && fits(p.v_hs, p.hk);
}

// Parts that the keys are cut into, 1 where there are tiles enough for half of the SMs or few keys: as many as give every SM one, of no
// less than 256 keys of an average sequence (128 on mma.sync, four times as slow), as the scratch holds.  28 rows of one key head
// over 7000 keys in fp32: 254 us in one part, 89 in 4.
int parts_of(const b200q_prompt_attention_args& p, long long units, int sms, bool tensor) {
  const long long rows = static_cast<long long>(p.tq) * p.hq, bytes = rows * (p.d * sizeof(float) + sizeof(float4));
  const long long parts = std::min({sms / std::max(1ll, units), static_cast<long long>(p.tk) / p.b / (tensor ? 256 : 128),
                                    static_cast<long long>(kScratchBytes) / bytes, 32ll});
  return rows <= kSplitCounters && parts > 1 ? static_cast<int>(parts) : 1;
}

template <typename T, int D>
int launch_tc(const PromptArgs& a, int sms, int device, cudaStream_t cs) {
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[device].load(std::memory_order_relaxed)) {
    const cudaError_t e =
        cudaFuncSetAttribute(prompt_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<D>::kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(prompt_tc_kernel)");
    ready[device].store(true, std::memory_order_relaxed);
  }
  const auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const auto map = [&](CUtensorMap* m, const void* base, int heads, int rows, long long ts, long long hs, uint32_t box_heads,
                       uint32_t box_rows) {
    const uint64_t one = static_cast<uint64_t>(a.d) * 2;  // a dimension of one row or head: any stride
    return host_tensor_map(m, type, base, {static_cast<uint64_t>(a.d), static_cast<uint64_t>(heads), static_cast<uint64_t>(rows)},
                           heads == 1 ? one : 2 * static_cast<uint64_t>(hs), rows == 1 ? one : 2 * static_cast<uint64_t>(ts),
                           {64, box_heads, box_rows});
  };
  CUtensorMap tm_q, tm_k, tm_v;
  int rc = map(&tm_q, a.q, a.hq, a.tq, a.q_ts, a.q_hs, a.ratio.d, a.tile.d / 2);
  if (rc == B200Q_OK) rc = map(&tm_k, a.k, a.hk, a.tk, a.k_ts, a.k_hs, 1, kTcKeys);
  if (rc == B200Q_OK) rc = map(&tm_v, a.v, a.hk, a.tk, a.v_ts, a.v_hs, 1, kTcKeys);
  if (rc) return rc;
  return host_launch("prompt_tc_kernel launch", prompt_tc_kernel<T, D>, dim3(static_cast<unsigned>(std::min<long long>(a.most_units, sms))),
                     kTcPromptThreads, TcShape<D>::kSmem, cs, 1, tm_q, tm_k, tm_v, a, a.scale < 0.0f ? 1u : 0u);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_prompt_attention(const b200q_prompt_attention_args* p, void* stream) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  if (p->ftype < B200Q_F32 || p->ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", p->ftype);
  if (p->b < 0 || p->tq < 0 || p->tk < 0 || p->hq < 0 || p->hk < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative dimensions");
  if (p->d < 1 || p->d > 256) return host_fail(B200Q_ERR_UNSUPPORTED, "heads of 1 to 256 channels, got %d", p->d);
  if (!std::isfinite(p->scale * kLog2e))  // exponents are of base 2
    return host_fail(B200Q_ERR_INVALID_ARG, "the scale must be finite, its product with log2(e) too, got %g", static_cast<double>(p->scale));
  if (p->b == 0 || p->tq == 0 || p->hq == 0) return B200Q_OK;
  if (p->hk == 0 || p->hq % p->hk)
    return host_fail(B200Q_ERR_INVALID_ARG, "%d key heads do not divide %d query heads", p->hk, p->hq);
  if (!p->q || !p->out || !p->starts || (p->tk && (!p->k || !p->v))) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (!p->k_starts && p->tk != p->tq)
    return host_fail(B200Q_ERR_INVALID_ARG, "%d query and %d key rows without starts of the keys", p->tq, p->tk);
  const long long ratio = p->hq / p->hk;
  if (p->tq * ratio > 0x3fffffffll || p->tk > 0x3fffffff || p->b > 0x3fffffff)
    return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
  int sms = 0, device = 0;
  PromptArgs a{};
  if (int rc = host_device(&sms, &a.err, &device)) return rc;
  a.q = p->q, a.q_ts = p->q_ts, a.q_hs = p->q_hs;
  a.k = p->k, a.k_ts = p->k_ts, a.k_hs = p->k_hs;
  a.v = p->v, a.v_ts = p->v_ts, a.v_hs = p->v_hs;
  a.starts = p->starts;
  a.k_starts = p->k_starts ? p->k_starts : p->starts;
  a.out = p->out;
  a.lse = p->lse;
  a.b = p->b, a.tq = p->tq, a.tk = p->tk, a.hq = p->hq, a.hk = p->hk, a.d = p->d;
  a.ratio = Divisor(static_cast<uint32_t>(ratio));
  a.scale = p->scale;
  // a warp whose 32 rows are done with care (see prompt_row_with_care) keeps others waiting: 300 clocks a row and key (2048 tokens), and
  // 1024 allowed for
  a.limit = host_wait_limit() + 32ll * 1024 * p->tk;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  const int size = p->ftype == B200Q_F32 ? 4 : 2;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
  const bool tensor = tensor_core_takes(*p, ratio);
  a.tile = Divisor(tensor ? 2 * static_cast<uint32_t>(128 / ratio) : kRows);
  a.row_scale = tensor ? 1 : static_cast<int>(ratio);
  // as many units as there may be: every sequence's last tile may be short
  const long long tiles = p->tq * static_cast<long long>(a.row_scale) / a.tile.d + std::min<long long>(p->b, p->tq);
  ScratchHold scratch;  // until both kernels are in the stream
  a.parts = parts_of(*p, tiles * p->hk, sms, tensor);
  if (a.parts > 1) {
    if (int rc = host_scratch(cs, &scratch)) return rc;
    a.arrived = scratch.counters;
    a.part_heads = static_cast<float4*>(scratch.bytes);
    a.part_sums = reinterpret_cast<float*>(a.part_heads + a.parts * static_cast<long long>(p->tq) * p->hq);
  }
  const long long units = a.most_units = tiles * p->hk * a.parts;
  if (units > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many rows");
  int rc = B200Q_OK;
  if (tensor) {
    if (p->ftype == B200Q_F16)
      rc = a.d <= 64 ? launch_tc<__half, 64>(a, sms, device, cs) : launch_tc<__half, 128>(a, sms, device, cs);
    else
      rc = a.d <= 64 ? launch_tc<__nv_bfloat16, 64>(a, sms, device, cs) : launch_tc<__nv_bfloat16, 128>(a, sms, device, cs);
  } else {
    const long long strides = p->q_ts | p->q_hs | p->k_ts | p->k_hs | p->v_ts | p->v_hs;
    const bool wide = !(bits & (4 * size - 1)) && strides % 4 == 0;
    B200Q_DISPATCH_FTYPE(p->ftype, rc = a.d <= 64    ? launch_mma<T, 64>(a, wide, units, device, cs)
                                        : a.d <= 128 ? launch_mma<T, 128>(a, wide, units, device, cs)
                                                     : launch_mma<T, 256>(a, wide, units, device, cs));
  }
  if (rc == B200Q_OK && a.parts > 1) {
    const long long rows = static_cast<long long>(p->tq) * p->hq;
    B200Q_DISPATCH_FTYPE(p->ftype, rc = host_launch("prompt_join_kernel launch", prompt_join_kernel<T>,
                                                    dim3(static_cast<unsigned>((rows + 7) / 8)), 256, 0, cs, 1, a));
    scratch.launched();
  }
  if (rc == B200Q_OK) host_set_path(tensor ? 23 : 24);
  return rc;
}
