// The 4-bit paged key / value cache and the attention over it (b200q_kv4_append, b200q_kv4_read,
// b200q_kv4_attention).
#include <algorithm>
#include <atomic>

#include "host.h"
#include "kv4_attention.cuh"
#include "lowbit.cuh"

namespace b200q {
namespace {

// Row (slot, head) of the cache: offset in units of one token's head.
__device__ __forceinline__ size_t cache_row(const Cache& c, uint32_t slot, int h) {
  const uint32_t page = c.page.of(slot);
  return (static_cast<size_t>(page) * c.heads + h) * c.page_size + (slot - page * c.page_size);
}

__device__ __forceinline__ bool slot_ok(const Cache& c, long long slot, int* err) {
  if (slot < 0) return false;
  if (slot >= c.slots) {
    atomicCAS(err, 0, kDevErrBadSlot);
    return false;
  }
  return true;
}

struct AppendArgs {
  const void* x[2];
  long long ts[2], hs[2];
  const int64_t* slots;
  int t;
  bool vec;  // rows may be moved 8 channels at a time
  int* err;
};

// Appending and reading move bytes: a row (one token's head, of the keys or the values) lies in D / 8 lanes of 8
// channels, one word of codes; a lane has AHEAD rows on their way at a time, and a block's lanes take rows side by side
// in memory.  8191 tokens x 4 heads x 256 fp32: append 26 us and read 16, 75 MB each.
constexpr int kMoveThreads = 128;

// Row i of a call: token, keys or values, head.
struct MoveRow {
  int t, which, h;
  long long slot;
};
__device__ __forceinline__ MoveRow move_row(const Cache& c, uint32_t i, int t, const int64_t* slots) {
  MoveRow r;
  r.t = static_cast<int>(c.both_heads.of(i));
  const int rest = static_cast<int>(i - static_cast<uint32_t>(r.t) * (2 * c.heads));
  r.which = rest >= c.heads;
  r.h = rest - (r.which ? c.heads : 0);
  r.slot = r.t < t ? __ldg(slots + r.t) : -1;
  return r;
}

// Eight channels; `vec`: whole rows may be moved 8 channels at a time.
template <typename T>
__device__ __forceinline__ void load_eight(T (&v)[8], const T* p, bool ok, bool vec) {
  if (!ok) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from_f32<T>(0.0f);
  } else if (!vec) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j];
  } else if constexpr (sizeof(T) == 4) {
    uint32_t bits[8];
    load_32(bits, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(bits[j]);
  } else {
    const uint4 bits = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned short half = static_cast<unsigned short>(w[j / 2] >> (16 * (j % 2)));
      v[j] = *reinterpret_cast<const T*>(&half);
    }
  }
}
__device__ __forceinline__ void store_eight(float* p, const float (&v)[8]) {
  uint32_t bits[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) bits[j] = __float_as_uint(v[j]);
  store_32(p, bits);
}
__device__ __forceinline__ void store_eight(__half* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_f16(v[0], v[1]), pack_f16(v[2], v[3]), pack_f16(v[4], v[5]), pack_f16(v[6], v[7]));
}
__device__ __forceinline__ void store_eight(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

template <typename T, int D, int G, int AHEAD>
__global__ void __launch_bounds__(kMoveThreads) kv4_append_kernel(Cache c, AppendArgs a) {
  wait_for_previous();
  constexpr int V = 8, kLanes = D / V, kRows = kMoveThreads / kLanes, kPerGroup = G / V;
  const int l = threadIdx.x % kLanes;
  const uint32_t first = blockIdx.x * (kRows * AHEAD) + threadIdx.x / kLanes;
  MoveRow row[AHEAD];
  T raw[AHEAD][V];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    row[u] = move_row(c, first + u * kRows, a.t, a.slots);
    const MoveRow& r = row[u];
    const T* from = static_cast<const T*>(a.x[r.which]) + r.t * a.ts[r.which] + r.h * a.hs[r.which] + l * V;
    load_eight(raw[u], from, r.t < a.t, a.vec);
  }
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    const MoveRow& r = row[u];
    float x[V], lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = to_f32(raw[u][j]);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      lo = min_nan(min_nan(x[j], x[j + 1]), lo);
      hi = max_nan(max_nan(x[j], x[j + 1]), hi);
    }
#pragma unroll
    for (int o = kPerGroup / 2; o; o >>= 1) {
      lo = min_nan(lo, __shfl_xor_sync(~0u, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(~0u, hi, o));
    }
    // the format's own fp32 steps, each rounded once; bf16 scales keep fp32's range
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
    float s = __bfloat162float(sb);
    uint32_t bits = __bfloat16_as_ushort(sb);
    if (!(s >= 1.17549435e-38f)) s = 0.0f, bits = 0;
    if (!(hi - lo < INFINITY)) s = 0.0f, bits = 0x7FC0u;  // a range that is infinite or NaN has no codes: the scale says so
    const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
    const float z = fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f);
    // rint(v) + z in the low bits of 1.5 2^23 + rint(v) + z (the sum rounds half to even, as rint does); v + z >= 0, since
    // x >= lo and z = rint(-lo / s).  The words add up, the exponents' bits with them.
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float v = __fadd_rn(__fadd_rn(__fmul_rn(x[j], inv), 12582912.0f), z);
      word += __float_as_uint(fminf(v, 12582927.0f)) << (4 * j);
    }
    word -= 0x4B400000u * 0x11111111u;
    if (slot_ok(c, r.slot, a.err)) {
      const size_t at = cache_row(c, static_cast<uint32_t>(r.slot), r.h);
      reinterpret_cast<uint32_t*>(c.codes[r.which])[at * kLanes + l] = word;
      if (l % kPerGroup == 0)
        c.params[r.which][at * (D / G) + l / kPerGroup] = bits | static_cast<uint32_t>(z) << 16;
    }
  }
}

template <typename T, int D, int G, int AHEAD>
__global__ void __launch_bounds__(kMoveThreads) kv4_read_kernel(Cache c, const int64_t* slots, T* k, T* v, int t, int* err) {
  wait_for_previous();
  constexpr int V = 8, kLanes = D / V, kRows = kMoveThreads / kLanes, kPerGroup = G / V;
  const int l = threadIdx.x % kLanes;
  const uint32_t first = blockIdx.x * (kRows * AHEAD) + threadIdx.x / kLanes;
  MoveRow row[AHEAD];
  uint32_t word[AHEAD], param[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    row[u] = move_row(c, first + u * kRows, t, slots);
    const MoveRow& r = row[u];
    word[u] = param[u] = 0;  // a scale of zero
    if (slot_ok(c, r.slot, err)) {
      const size_t at = cache_row(c, static_cast<uint32_t>(r.slot), r.h);
      word[u] = __ldg(reinterpret_cast<const uint32_t*>(c.codes[r.which]) + at * kLanes + l);
      param[u] = __ldg(c.params[r.which] + at * (D / G) + l / kPerGroup);
    }
  }
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    const MoveRow& r = row[u];
    if (r.t >= t) continue;
    const float s = param_scale(param[u]);
    // 1024 + code and 1024 + 16 code as fp16 pairs of the codes 16 bits apart, less 1024 + zero point (a sixteenth of the
    // latter: 64 + zero point): exact, and so is its product with the scale in fp32
    const uint32_t z = (param[u] >> 16 & 0xFFu) * 0x00010001u | 0x64006400u;
    const __half2 less = *reinterpret_cast<const __half2*>(&z), less_64 = __hsub2(__float2half2_rn(960.0f), less);
    float out[V];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const uint32_t bits = and_or(word[u] >> (j / 2 * 8), j % 2 ? 0x00F000F0u : 0x000F000Fu, 0x64006400u);
      const __half2 h = j % 2 ? __hfma2(*reinterpret_cast<const __half2*>(&bits), __float2half2_rn(0.0625f), less_64)
                              : __hsub2(*reinterpret_cast<const __half2*>(&bits), less);
      const float2 f = mul2(__half22float2(h), both(s));
      out[j] = f.x;
      out[j + V / 2] = f.y;
    }
    store_eight((r.which ? v : k) + (static_cast<long long>(r.t) * c.heads + r.h) * D + l * V, out);
  }
}

int check_cache(const b200q_kv4_cache* p, Cache* c) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  if (p->pages < 0 || p->heads <= 0 || p->page_size <= 0) return host_fail(B200Q_ERR_INVALID_ARG, "bad cache shape");
  if (p->d != 64 && p->d != 128 && p->d != 256)
    return host_fail(B200Q_ERR_UNSUPPORTED, "4-bit cache heads have 64, 128 or 256 channels, got %d", p->d);
  if (p->group != 32 && p->group != 64)
    return host_fail(B200Q_ERR_UNSUPPORTED, "4-bit cache groups are 32 or 64 channels, got %d", p->group);
  if (p->page_size > (1 << 20) || p->heads > (1 << 16)) return host_fail(B200Q_ERR_UNSUPPORTED, "cache too large");
  if (static_cast<long long>(p->pages) * p->page_size > 0x7fffffffll)
    return host_fail(B200Q_ERR_UNSUPPORTED, "cache of more than 2^31 slots");
  if (static_cast<long long>(p->pages) * p->page_size * p->heads >= 0xffffffffll)  // rows are numbered in 32 bits
    return host_fail(B200Q_ERR_UNSUPPORTED, "cache of more than 2^32 rows");
  if (p->pages > 0 && (!p->k_codes || !p->k_params || !p->v_codes || !p->v_params))
    return host_fail(B200Q_ERR_INVALID_ARG, "null cache pointer");
  if ((reinterpret_cast<uintptr_t>(p->k_codes) | reinterpret_cast<uintptr_t>(p->v_codes) |
       reinterpret_cast<uintptr_t>(p->k_params) | reinterpret_cast<uintptr_t>(p->v_params)) & 15u)
    return host_fail(B200Q_ERR_INVALID_ARG, "cache tensors must be 16-byte aligned");
  *c = Cache{{p->k_codes, p->v_codes}, {p->k_params, p->v_params}, p->pages, p->heads, p->page_size, p->d, p->group,
             static_cast<int64_t>(p->pages) * p->page_size, Divisor(p->page_size), Divisor(2 * p->heads)};
  return B200Q_OK;
}

#define B200Q_MOVE_D(kernel, G, A) (c.d == 64 ? kernel<T, 64, G, A> : c.d == 128 ? kernel<T, 128, G, A> : kernel<T, 256, G, A>)
#define B200Q_MOVE(kernel)                                                                         \
  (ahead == 1 ? c.group == 32 ? B200Q_MOVE_D(kernel, 32, 1) : B200Q_MOVE_D(kernel, 64, 1)          \
              : c.group == 32 ? B200Q_MOVE_D(kernel, 32, 4) : B200Q_MOVE_D(kernel, 64, 4))

// Rows that a lane has on their way: four when there are rows for many blocks (append and read of 8191 tokens x 4 heads x
// 256 fp32: 42 us, 46 with two; 2048 x 8 x 128 bf16: 13.0, 18.6 with one), one when a call is all latency (64 x 8 x 128:
// 4.2 us, 6.2 with four).  Up to kMoveSmall blocks an SM of one row per lane count as such (4 to 16 time alike).
constexpr int kMoveSmall = 8;
int move_blocks(const Cache& c, int t, int sms, int* ahead, int* blocks) {
  const long long rows = 2ll * t * c.heads, per = kMoveThreads / (c.d / 8);
  *ahead = (rows + per - 1) / per <= static_cast<long long>(kMoveSmall) * sms ? 1 : 4;
  const long long n = (rows + per * *ahead - 1) / (per * *ahead);
  if (n * per * *ahead > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many tokens");
  *blocks = static_cast<int>(n);
  return B200Q_OK;
}

template <int D, int G, int NT, bool F32>
int launch_attention(const Cache& c, AttnArgs a, int sms, int device, cudaStream_t stream) {
  using Shape = AttnShape<D, G, NT, F32>;
  auto kernel = kv4_attention_kernel<D, G, NT, F32>;
  // blocks that an SM holds, found once (and on the way, leave for the shared memory that they take)
  static std::atomic<int> per_sm[kMaxDevices];
  int resident = per_sm[device].load(std::memory_order_relaxed);
  if (resident == 0) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(kv4_attention_kernel)");
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kWarps * 32, Shape::kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
    resident = std::max(1, resident);
    per_sm[device].store(resident, std::memory_order_relaxed);
  }
  a.row_tiles = (a.tq * (a.hq / c.heads) + 8 * NT - 1) / (8 * NT);
  // one block for each that the GPU holds at once; fewer when even the longest lengths have fewer steps
  const long long steps = (static_cast<long long>(a.max_pages) * c.page_size + kStepTokens - 1) / kStepTokens;
  const long long most = static_cast<long long>(a.b) * c.heads * a.row_tiles * std::max(1ll, steps);
  if (static_cast<long long>(a.b) * c.heads * a.row_tiles * (steps + kUnitSteps + 1) > 0x7fffffffll)
    return host_fail(B200Q_ERR_UNSUPPORTED, "attention too large");
  // (a unit's parts, one per block at most, leave their shares in shared memory when they are joined; the scratch holds
  // the parts of five hundred blocks or more)
  constexpr int kPartRows = 2 * 8 * NT, kRoom = static_cast<int>(kScratchBytes / (kPartRows * (D + 2) * sizeof(float)));
  const int blocks = static_cast<int>(
      std::min<long long>(std::min({sms * resident, Shape::kBody / (8 * NT * 4), kSplitCounters, kRoom}), most));
  const size_t rows = static_cast<size_t>(blocks) * kPartRows;
  ScratchHold scratch;
  int rc = host_scratch(stream, &scratch);
  if (rc) return rc;
  a.counters = scratch.counters;
  a.partial = static_cast<float*>(scratch.bytes);
  a.partial_ml = a.partial + rows * D;
  rc = host_launch("kv4_attention_kernel launch", kernel, dim3(blocks), kWarps * 32, Shape::kSmem, stream, 1, c, a);
  scratch.launched();
  return rc;
}

int check_ftype(int ftype) {
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_kv4_append(const b200q_kv4_cache* cache, const void* k, long long k_ts, long long k_hs,
                                const void* v, long long v_ts, long long v_hs, const int64_t* slots, int ftype, int t,
                                void* stream) {
  Cache c;
  int rc = check_cache(cache, &c);
  if (rc || (rc = check_ftype(ftype))) return rc;
  if (t < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative token count");
  if (t == 0) return B200Q_OK;
  if (!k || !v || !slots) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  const int size = ftype == B200Q_F32 ? 4 : 2;
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & (8 * size - 1)) == 0 &&
                   (k_ts | k_hs | v_ts | v_hs) % 8 == 0;
  AppendArgs a{{k, v}, {k_ts, v_ts}, {k_hs, v_hs}, slots, t, vec, nullptr};
  int sms = 0;
  if ((rc = host_device(&sms, &a.err))) return rc;
  int ahead = 0, blocks = 0;
  if ((rc = move_blocks(c, t, sms, &ahead, &blocks))) return rc;
  B200Q_DISPATCH_FTYPE(ftype, rc = host_launch("kv4_append_kernel launch", B200Q_MOVE(kv4_append_kernel), dim3(blocks),
                                               kMoveThreads, 0, static_cast<cudaStream_t>(stream), 1, c, a));
  if (rc == B200Q_OK) host_set_path(19);
  return rc;
}

extern "C" int b200q_kv4_read(const b200q_kv4_cache* cache, const int64_t* slots, void* k, void* v, int ftype, int t,
                              void* stream) {
  Cache c;
  int rc = check_cache(cache, &c);
  if (rc || (rc = check_ftype(ftype))) return rc;
  if (t < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative token count");
  if (t == 0) return B200Q_OK;
  if (!k || !v || !slots) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  int sms = 0, *err = nullptr;
  if ((rc = host_device(&sms, &err))) return rc;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 31u)
    return host_fail(B200Q_ERR_INVALID_ARG, "kv4_read outputs must be 32-byte aligned");
  int ahead = 0, blocks = 0;
  if ((rc = move_blocks(c, t, sms, &ahead, &blocks))) return rc;
  B200Q_DISPATCH_FTYPE(ftype, rc = host_launch("kv4_read_kernel launch", B200Q_MOVE(kv4_read_kernel), dim3(blocks),
                                               kMoveThreads, 0, static_cast<cudaStream_t>(stream), 1, c, slots,
                                               static_cast<T*>(k), static_cast<T*>(v), t, err));
  if (rc == B200Q_OK) host_set_path(19);
  return rc;
}

extern "C" int b200q_kv4_attention(const b200q_kv4_cache* cache, const b200q_kv4_attention_args* p, void* stream) {
  Cache c;
  int rc = check_cache(cache, &c);
  if (rc) return rc;
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const int ftype = p->ftype, b = p->b, tq = p->tq, hq = p->hq, max_pages = p->max_pages;
  if ((rc = check_ftype(ftype))) return rc;
  if (b < 0 || tq < 0 || hq < 0 || max_pages < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative attention dimension");
  if (hq % c.heads) return host_fail(B200Q_ERR_INVALID_ARG, "%d query heads do not divide over %d cache heads", hq, c.heads);
  if (b == 0 || tq == 0 || hq == 0) return B200Q_OK;
  if (!p->q || !p->out || !p->lens || (max_pages > 0 && !p->block_table)) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (static_cast<long long>(max_pages) * c.page_size > (1 << 30) || b > (1 << 20) || tq > (1 << 16) || hq > (1 << 16))
    return host_fail(B200Q_ERR_UNSUPPORTED, "attention too large");
  if (static_cast<long long>(b) * tq * hq > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "attention too large");
  AttnArgs a{p->q,   p->q_bs, p->q_ts, p->q_hs, p->block_table, p->bt_stride, p->lens, p->out,
             p->lse, ftype,   b,       tq,      hq,             max_pages,    p->scale};
  int sms = 0, device = 0;
  if ((rc = host_device(&sms, &a.err, &device))) return rc;
  // 16 rows a pass where a head has more than 8; heads of 256 channels keep to 8, whose sums fill the registers
  const int rows = tq * (hq / c.heads);
  const bool two = rows > 8 && c.d <= 128;
  const bool f32 = ftype == B200Q_F32;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
#define B200Q_ATTN(D, G)                                                      \
  (two ? f32 ? launch_attention<D, G, D == 256 ? 1 : 2, true>(c, a, sms, device, cs)  \
             : launch_attention<D, G, D == 256 ? 1 : 2, false>(c, a, sms, device, cs) \
       : f32 ? launch_attention<D, G, 1, true>(c, a, sms, device, cs)                 \
             : launch_attention<D, G, 1, false>(c, a, sms, device, cs))
  rc = c.d == 64    ? c.group == 32 ? B200Q_ATTN(64, 32) : B200Q_ATTN(64, 64)
       : c.d == 128 ? c.group == 32 ? B200Q_ATTN(128, 32) : B200Q_ATTN(128, 64)
                    : c.group == 32 ? B200Q_ATTN(256, 32) : B200Q_ATTN(256, 64);
#undef B200Q_ATTN
  if (rc == B200Q_OK) host_set_path(20);
  return rc;
}
