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
  int* err;
};

// One thread per group.
template <typename T>
__global__ void kv4_append_kernel(Cache c, AppendArgs a) {
  const int groups = c.d / c.group;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= 2ll * a.t * c.heads * groups) return;
  const int g = static_cast<int>(i % groups), h = static_cast<int>(i / groups % c.heads);
  const long long r = i / groups / c.heads;
  const int which = static_cast<int>(r % 2), t = static_cast<int>(r / 2);
  const long long slot = a.slots[t];
  if (!slot_ok(c, slot, a.err)) return;
  const T* x = static_cast<const T*>(a.x[which]) + t * a.ts[which] + h * a.hs[which] + g * c.group;
  float lo = 0.0f, hi = 0.0f;
  for (int j = 0; j < c.group; ++j) {
    const float v = to_f32(x[j]);
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f));
  float s = __bfloat162float(sb);
  uint32_t bits = __bfloat16_as_ushort(sb);
  if (!(s >= 1.17549435e-38f)) {
    s = 0.0f;
    bits = 0;
  }
  const float inv = s > 0.0f ? __frcp_rn(s) : 0.0f;
  const float z = fminf(fmaxf(rintf(__fmul_rn(-lo, inv)), 0.0f), 15.0f);
  const size_t row = cache_row(c, slot, h);
  c.params[which][row * groups + g] = bits | static_cast<uint32_t>(z) << 16;
  uint8_t* out = c.codes[which] + row * (c.d / 2) + g * c.group / 2;
  for (int j = 0; j < c.group; j += 2) {
    uint32_t q[2];
    for (int u = 0; u < 2; ++u)
      q[u] = static_cast<uint32_t>(fminf(fmaxf(rintf(__fmul_rn(to_f32(x[j + u]), inv)) + z, 0.0f), 15.0f));
    out[j / 2] = static_cast<uint8_t>(q[0] | q[1] << 4);
  }
}

template <typename T>
__global__ void kv4_read_kernel(Cache c, const int64_t* slots, T* k, T* v, int t, int* err) {
  const int bytes = c.d / 2;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= 2ll * t * c.heads * bytes) return;
  const int b = static_cast<int>(i % bytes), h = static_cast<int>(i / bytes % c.heads);
  const long long r = i / bytes / c.heads;
  const int which = static_cast<int>(r % 2), tok = static_cast<int>(r / 2);
  T* out = (which ? v : k) + (static_cast<long long>(tok) * c.heads + h) * c.d + 2 * b;
  const long long slot = slots[tok];
  if (!slot_ok(c, slot, err)) {
    out[0] = out[1] = from_f32<T>(0.0f);
    return;
  }
  const size_t row = cache_row(c, slot, h);
  const uint32_t byte = c.codes[which][row * bytes + b];
  const uint32_t p = c.params[which][row * (c.d / c.group) + 2 * b / c.group];
  out[0] = from_f32<T>((static_cast<float>(byte & 15u) - param_zero(p)) * param_scale(p));
  out[1] = from_f32<T>((static_cast<float>(byte >> 4) - param_zero(p)) * param_scale(p));
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
  const long long units = static_cast<long long>(a.b) * c.heads * a.row_tiles;
  long long blocks = units;
  const int target = sms * resident * kWaves;
  const long long most = (static_cast<long long>(a.max_pages) * c.page_size + kMinChunk - 1) / kMinChunk;
  if (most > 1 && units < target) {
    // units split so that each block has 1 / target of the tokens: at most one block more per unit
    blocks = std::min<long long>(target + units, units * most);
    a.target = target;
    const size_t rows = static_cast<size_t>(blocks) * 8 * NT;
    void* ws = nullptr;
    int rc = host_workspace(rows * (D + 2) * sizeof(float), stream, &ws);
    if (rc || (rc = host_counters(stream, &a.counters))) return rc;
    a.partial = static_cast<float*>(ws);
    a.partial_ml = a.partial + rows * D;
  }
  if (blocks > (a.target ? kSplitCounters : 0x7fffffffll)) return host_fail(B200Q_ERR_UNSUPPORTED, "attention too large");
  kernel<<<static_cast<int>(blocks), kWarps * 32, Shape::kSmem, stream>>>(c, a);
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
  AppendArgs a{{k, v}, {k_ts, v_ts}, {k_hs, v_hs}, slots, t, nullptr};
  int sms = 0;
  if ((rc = host_device(&sms, &a.err))) return rc;
  const long long blocks = (2ll * t * c.heads * (c.d / c.group) + 127) / 128;
  if (blocks > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many tokens");
  B200Q_DISPATCH_FTYPE(ftype, (kv4_append_kernel<T><<<static_cast<int>(blocks), 128, 0,
                                                      static_cast<cudaStream_t>(stream)>>>(c, a)));
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
  const long long blocks = (2ll * t * c.heads * (c.d / 2) + 255) / 256;
  if (blocks > 0x7fffffffll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many tokens");
  B200Q_DISPATCH_FTYPE(ftype, (kv4_read_kernel<T><<<static_cast<int>(blocks), 256, 0,
                                                    static_cast<cudaStream_t>(stream)>>>(
                                  c, slots, static_cast<T*>(k), static_cast<T*>(v), t, err)));
  rc = host_check_launch("kv4_read_kernel launch");
  if (rc == B200Q_OK) host_set_path(19);
  return rc;
}

extern "C" int b200q_kv4_attention(const b200q_kv4_cache* cache, const void* q, long long q_bs, long long q_ts,
                                   long long q_hs, const int32_t* block_table, long long bt_stride,
                                   const int32_t* lens, void* out, float* lse, int ftype, int b, int tq, int hq,
                                   int max_pages, float scale, void* stream) {
  Cache c;
  int rc = check_cache(cache, &c);
  if (rc || (rc = check_ftype(ftype))) return rc;
  if (b < 0 || tq < 0 || hq < 0 || max_pages < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative attention dimension");
  if (hq % c.heads) return host_fail(B200Q_ERR_INVALID_ARG, "%d query heads do not divide over %d cache heads", hq, c.heads);
  if (b == 0 || tq == 0 || hq == 0) return B200Q_OK;
  if (!q || !out || !lens || (max_pages > 0 && !block_table)) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (static_cast<long long>(max_pages) * c.page_size > (1 << 30) || b > (1 << 20) || tq > (1 << 16) || hq > (1 << 16))
    return host_fail(B200Q_ERR_UNSUPPORTED, "attention too large");
  AttnArgs a{q, q_bs, q_ts, q_hs, block_table, bt_stride, lens, out, lse, ftype, b, tq, hq, max_pages, scale};
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
