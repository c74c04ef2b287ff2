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
__device__ __forceinline__ size_t cache_row(const Cache& c, long long slot, int h) {
  const long long page = slot / c.page_size;
  return (static_cast<size_t>(page) * c.heads + h) * c.page_size + static_cast<size_t>(slot - page * c.page_size);
}

__device__ __forceinline__ bool slot_ok(const Cache& c, long long slot, int* err) {
  if (slot < 0) return false;
  if (slot >= static_cast<long long>(c.pages) * c.page_size) {
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
  bool vec;  // rows are 16-byte aligned
  int* err;
};

// Appending and reading move bytes: a row (one token's head, of the keys or the values) lies in D / 8 lanes of 8
// channels, one word of codes; a lane has kAhead rows on their way at a time, and a block's lanes take rows side by
// side in memory.
constexpr int kMoveThreads = 128;
constexpr int kAhead = 4;

// Row i of a call: token, keys or values, head.
struct MoveRow {
  int t, which, h;
  bool ok;
  long long slot;
};
__device__ __forceinline__ MoveRow move_row(const Cache& c, long long i, int t, const int64_t* slots, int* err) {
  MoveRow r;
  r.t = static_cast<int>(i / (2 * c.heads));
  const int rest = static_cast<int>(i - static_cast<long long>(r.t) * 2 * c.heads);
  r.which = rest >= c.heads;
  r.h = rest - (r.which ? c.heads : 0);
  r.ok = r.t < t;
  r.slot = r.ok ? slots[r.t] : -1;
  if (r.ok) r.ok = slot_ok(c, r.slot, err);
  return r;
}

// Eight channels as fp32; `vec`: rows are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load_eight(const T* p, bool ok, bool vec, T (&v)[8]) {
  uint4* to = reinterpret_cast<uint4*>(v);
  if (vec || !ok) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
      to[i] = ok ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[j];
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_append_kernel(Cache c, AppendArgs a) {
  constexpr int kLanes = D / 8, kRows = kMoveThreads / kLanes;
  const int l = threadIdx.x % kLanes;
  const long long first = static_cast<long long>(blockIdx.x) * (kRows * kAhead) + threadIdx.x / kLanes;
  MoveRow row[kAhead];
  alignas(16) T raw[kAhead][8];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    row[u] = move_row(c, first + u * kRows, a.t, a.slots, a.err);
    const MoveRow& r = row[u];
    load_eight(static_cast<const T*>(a.x[r.which]) + r.t * a.ts[r.which] + r.h * a.hs[r.which] + l * 8, r.ok, a.vec, raw[u]);
  }
  const int per_group = c.group / 8;  // lanes of a group
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const MoveRow& r = row[u];
    float x[8], lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = to_f32(raw[u][j]);
      lo = fminf(lo, x[j]);
      hi = fmaxf(hi, x[j]);
    }
    for (int o = per_group / 2; o; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
    }
    // the format's own fp32 steps, each rounded once; bf16 scales keep fp32's range
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
    float s = __bfloat162float(sb);
    uint32_t bits = __bfloat16_as_ushort(sb);
    if (!(s >= 1.17549435e-38f)) s = 0.0f, bits = 0;
    const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
    const float z = fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f);
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      word |= static_cast<uint32_t>(fminf(fmaxf(rintf(__fmul_rn(x[j], inv)) + z, 0.0f), 15.0f)) << (4 * j);
    if (r.ok) {
      const size_t at = cache_row(c, r.slot, r.h);
      reinterpret_cast<uint32_t*>(c.codes[r.which])[at * (D / 8) + l] = word;
      if (l % per_group == 0)
        c.params[r.which][at * (D / c.group) + l / per_group] = bits | static_cast<uint32_t>(z) << 16;
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kMoveThreads) kv4_read_kernel(Cache c, const int64_t* slots, T* k, T* v, int t, int* err) {
  constexpr int kLanes = D / 8, kRows = kMoveThreads / kLanes;
  const int l = threadIdx.x % kLanes;
  const long long first = static_cast<long long>(blockIdx.x) * (kRows * kAhead) + threadIdx.x / kLanes;
  MoveRow row[kAhead];
  uint32_t word[kAhead], param[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    row[u] = move_row(c, first + u * kRows, t, slots, err);
    const MoveRow& r = row[u];
    word[u] = param[u] = 0;  // a scale of zero
    if (r.ok) {
      const size_t at = cache_row(c, r.slot, r.h);
      word[u] = __ldg(reinterpret_cast<const uint32_t*>(c.codes[r.which]) + at * (D / 8) + l);
      param[u] = __ldg(c.params[r.which] + at * (D / c.group) + l * 8 / c.group);
    }
  }
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const MoveRow& r = row[u];
    if (r.t >= t) continue;
    const float s = param_scale(param[u]), z = param_zero(param[u]);
    alignas(16) T out[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = from_f32<T>((static_cast<float>((word[u] >> (4 * j)) & 15u) - z) * s);
    uint4* to = reinterpret_cast<uint4*>((r.which ? v : k) + (static_cast<long long>(r.t) * c.heads + r.h) * D + l * 8);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) to[i] = reinterpret_cast<const uint4*>(out)[i];
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
  if (p->pages > 0 && (!p->k_codes || !p->k_params || !p->v_codes || !p->v_params))
    return host_fail(B200Q_ERR_INVALID_ARG, "null cache pointer");
  if ((reinterpret_cast<uintptr_t>(p->k_codes) | reinterpret_cast<uintptr_t>(p->v_codes) |
       reinterpret_cast<uintptr_t>(p->k_params) | reinterpret_cast<uintptr_t>(p->v_params)) & 15u)
    return host_fail(B200Q_ERR_INVALID_ARG, "cache tensors must be 16-byte aligned");
  *c = Cache{{p->k_codes, p->v_codes}, {p->k_params, p->v_params}, p->pages, p->heads, p->page_size, p->d, p->group};
  return B200Q_OK;
}

int move_blocks(const Cache& c, int t, int* blocks) {
  const int rows = kMoveThreads / (c.d / 8) * kAhead;
  const long long n = (2ll * t * c.heads + rows - 1) / rows;
  if (n > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many tokens");
  *blocks = static_cast<int>(n);
  return B200Q_OK;
}

template <int D, int G, int NT, bool F32>
int launch_attention(const Cache& c, AttnArgs a, int sms, cudaStream_t stream) {
  using Shape = AttnShape<D, G, NT, F32>;
  auto kernel = kv4_attention_kernel<D, G, NT, F32>;
  // blocks that an SM holds, found once (and on the way, leave for the shared memory that they take)
  static std::atomic<int> per_sm{0};
  int resident = per_sm.load(std::memory_order_relaxed);
  if (resident == 0) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaFuncSetAttribute(kv4_attention_kernel)");
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kWarps * 32, Shape::kSmem);
    if (e != cudaSuccess) return host_cuda_fail(e, "cudaOccupancyMaxActiveBlocksPerMultiprocessor");
    resident = std::max(1, resident);
    per_sm.store(resident, std::memory_order_relaxed);
  }
  a.row_tiles = (a.tq * (a.hq / c.heads) + 8 * NT - 1) / (8 * NT);
  // one block for each that the GPU holds at once; fewer when even the longest lengths have fewer steps
  const long long steps = (static_cast<long long>(a.max_pages) * c.page_size + kStepTokens - 1) / kStepTokens;
  const long long most = static_cast<long long>(a.b) * c.heads * a.row_tiles * std::max(1ll, (steps + kMinSteps - 1) / kMinSteps);
  // (a unit's parts, one per block at most, leave their shares in shared memory when they are joined)
  const int blocks = static_cast<int>(std::min<long long>(std::min(sms * resident, Shape::kBody / (8 * NT * 4)), most));
  const size_t rows = static_cast<size_t>(blocks) * 2 * 8 * NT;
  void* ws = nullptr;
  int rc = host_workspace(rows * (D + 2) * sizeof(float), stream, &ws);
  if (rc || (rc = host_counters(stream, &a.counters))) return rc;
  a.partial = static_cast<float*>(ws);
  a.partial_ml = a.partial + rows * D;
  if (blocks > kSplitCounters) return host_fail(B200Q_ERR_UNSUPPORTED, "attention too large");
  kernel<<<blocks, kWarps * 32, Shape::kSmem, stream>>>(c, a);
  return host_check_launch("kv4_attention_kernel launch");
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
  const bool vec = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u) == 0 &&
                   ((k_ts | k_hs | v_ts | v_hs) * size) % 16 == 0;
  AppendArgs a{{k, v}, {k_ts, v_ts}, {k_hs, v_hs}, slots, t, vec, nullptr};
  int sms = 0;
  if ((rc = host_device(&sms, &a.err))) return rc;
  int blocks = 0;
  if ((rc = move_blocks(c, t, &blocks))) return rc;
  B200Q_DISPATCH_FTYPE(ftype, (c.d == 64    ? kv4_append_kernel<T, 64>
                               : c.d == 128 ? kv4_append_kernel<T, 128>
                                            : kv4_append_kernel<T, 256>)<<<blocks, kMoveThreads, 0,
                                                                           static_cast<cudaStream_t>(stream)>>>(c, a));
  rc = host_check_launch("kv4_append_kernel launch");
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
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u)
    return host_fail(B200Q_ERR_INVALID_ARG, "kv4_read outputs must be 16-byte aligned");
  int blocks = 0;
  if ((rc = move_blocks(c, t, &blocks))) return rc;
  B200Q_DISPATCH_FTYPE(ftype, (c.d == 64    ? kv4_read_kernel<T, 64>
                               : c.d == 128 ? kv4_read_kernel<T, 128>
                                            : kv4_read_kernel<T, 256>)<<<blocks, kMoveThreads, 0,
                                                                         static_cast<cudaStream_t>(stream)>>>(
                                  c, slots, static_cast<T*>(k), static_cast<T*>(v), t, err));
  rc = host_check_launch("kv4_read_kernel launch");
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
  AttnArgs a{p->q,   p->q_bs, p->q_ts, p->q_hs, p->block_table, p->bt_stride, p->lens, p->out,
             p->lse, ftype,   b,       tq,      hq,             max_pages,    p->scale};
  int sms = 0;
  if ((rc = host_device(&sms, &a.err))) return rc;
  a.page_shift = -1;
  for (int i = 0; i <= 20; ++i)
    if (c.page_size == 1 << i) a.page_shift = i;
  // 16 rows a pass where a head has more than 8; heads of 256 channels keep to 8, whose sums fill the registers
  const int rows = tq * (hq / c.heads);
  const bool two = rows > 8 && c.d <= 128;
  const bool f32 = ftype == B200Q_F32;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
#define B200Q_ATTN(D, G)                                                      \
  (two ? f32 ? launch_attention<D, G, D == 256 ? 1 : 2, true>(c, a, sms, cs)  \
             : launch_attention<D, G, D == 256 ? 1 : 2, false>(c, a, sms, cs) \
       : f32 ? launch_attention<D, G, 1, true>(c, a, sms, cs)                 \
             : launch_attention<D, G, 1, false>(c, a, sms, cs))
  rc = c.d == 64    ? c.group == 32 ? B200Q_ATTN(64, 32) : B200Q_ATTN(64, 64)
       : c.d == 128 ? c.group == 32 ? B200Q_ATTN(128, 32) : B200Q_ATTN(128, 64)
                    : c.group == 32 ? B200Q_ATTN(256, 32) : B200Q_ATTN(256, 64);
#undef B200Q_ATTN
  if (rc == B200Q_OK) host_set_path(20);
  return rc;
}
