// 8-bit rows with one fp32 scale each (b200q_quantize_s8, b200q_rms_norm_s8, b200q_read_s8).
//
//   h = T(x + residual);  u = fp32(h w);  a = max |u|;  r = (mean h^2 + eps)^-1/2
//   code = rint(u fl(127 fl(1 / a))), the product exact;  scale = a r / 127;  value = code scale
//
// The norm's factor r cancels in u r / (max |u| r), so the codes need only the largest |u|: they are the same bits whatever the order
// of the sum of squares.  fma(u, fl(127 fl(1 / a)), 1.5 2^23) rounds the exact product to a whole number, half to even, and leaves the code
// in the low byte of its bits.
//
// Bytes bound it: x (and the residual) in, the sum and one byte an element out.  A row lies in the registers of W warps from its only
// read to its writes, 16 bytes a load and 16 or 32 elements a lane; both reductions meet in one
// barrier.  8192 x 4096 fp16 with a residual: 44 us for 235 MB, 5.3 TB/s (82 % of what a copy reaches), at 61 % of the issue
// slots; read_s8 of the same 18.5 us for 101 MB, 5.4 TB/s.  Few rows are one latency chain (4 x 4096: 3.5 us); rows that do not
// start on 16 bytes are read by elements (1021 x 5003 fp32 and its read: 15.5 us, half of the copy rate).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "host.h"
#include "lowbit.cuh"

namespace b200q {
namespace {

struct RowsArgs {
  const void* x;
  long long ldx;
  const void* w;         // null: all ones
  const void* residual;  // null: none
  long long ldr;
  void* sum;  // T(x + residual); may be x or the residual
  long long lds;
  int8_t* codes;
  long long ldc;
  float* scales;
  int t, n;
  float eps;
};

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kSmallest = 0x1p-119f;  // rows with nothing larger are zeros: 127 / a stays finite

// VEC elements in memory: one, or 16 bytes.
template <typename T, int VEC>
struct Chunk {
  static __device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
  static __device__ __forceinline__ void load(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
      v[0] = to_f32(*p);
    } else {
      const uint4 b = *reinterpret_cast<const uint4*>(p);
      unpack({b.x, b.y, b.z, b.w}, v);
    }
  }
  // Stores v rounded to T, and leaves what was stored in v.
  static __device__ __forceinline__ void store(T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
      const T kept = from_f32<T>(v[0]);
      *p = kept;
      v[0] = to_f32(kept);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4)
          w[i] = __float_as_uint(v[i]);
        else if constexpr (std::is_same<T, __half>::value)
          w[i] = pack_f16(v[2 * i], v[2 * i + 1]);
        else
          w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      }
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      unpack(w, v);
    }
  }
};

// Four codes: the low bytes of the shifted products.
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                     __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&v)[VEC], float inv) {
  constexpr float kShift = 12582912.0f;
  float s[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) s[i] = __fmaf_rn(v[i], inv, kShift);
  if constexpr (VEC == 1) {
    *p = static_cast<int8_t>(__float_as_uint(s[0]) & 255u);
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<uint32_t*>(p) = four_codes(s[0], s[1], s[2], s[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(four_codes(s[0], s[1], s[2], s[3]), four_codes(s[4], s[5], s[6], s[7]));
  }
}

// A row's two reductions over its warps.  Every thread of the block calls it.
struct RowSums {
  uint32_t top;  // bits of max |u|, a NaN above all
  float squares;
};
template <int W>
__device__ __forceinline__ RowSums row_sums(float top, float squares, uint32_t (*tops)[32], float (*sums)[32], int half) {
  RowSums r{__reduce_max_sync(~0u, __float_as_uint(top)), warp_sum(squares)};
  if constexpr (W > 1) {
    const int warp = threadIdx.x / 32, first = warp / W * W;
    if (threadIdx.x % 32 == 0) {
      tops[half][warp] = r.top;
      sums[half][warp] = r.squares;
    }
    __syncthreads();
    r = {0u, 0.0f};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      r.top = max(r.top, tops[half][first + i]);
      r.squares += sums[half][first + i];
    }
  }
  return r;
}

// The factor that brings a sum of squares which left fp32's range back into it (1: it did not).
__device__ __forceinline__ float rescue(float squares, float eps) {
  if (!(squares < __uint_as_float(kInfBits))) return 0x1p-70f;
  return squares < 0x1p-90f && eps < 0x1p-80f ? 0x1p70f : 1.0f;
}
__device__ __forceinline__ float norm_factor(float squares, int n, float eps, float f) {
  return f * rsqrtf(squares / static_cast<float>(n) + eps * f * f);
}

// What a row's largest |u| says: 127 / a for the codes, a / 127 for the scale.
struct RowScale {
  float inv, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float a = __uint_as_float(top);
  if (top >= kInfBits) return {0.0f, __uint_as_float(0x7fc00000u)};
  if (a < kSmallest) return {0.0f, 0.0f};
  return {__fmul_rn(127.0f, __frcp_rn(a)), __fdiv_rn(a, 127.0f)};
}

// NV chunks a lane; max(8, W) warps a block, W of them a row.
template <typename T, int VEC, int NV, int W, bool NORM>
__global__ void __launch_bounds__(32 * (W > 8 ? W : 8)) rows_s8_kernel(RowsArgs a) {
  constexpr int kRows = (W > 8 ? W : 8) / W;
  __shared__ uint32_t tops[2][32];
  __shared__ float sums[2][32];
  wait_for_previous();
  const int row = blockIdx.x * kRows + threadIdx.x / (32 * W);
  const int lane = threadIdx.x % (32 * W);
  const bool live = row < a.t;
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.ldx;
  const T* res = static_cast<const T*>(a.residual) + (live ? row : 0) * a.ldr;
  const T* w = static_cast<const T*>(a.w);
  float v[NV][VEC];
  float top = 0.0f, squares = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 32 * W + lane) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
    if (live && c < a.n) Chunk<T, VEC>::load(x + c, v[i]);
  }
  if (a.residual) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * 32 * W + lane) * VEC;
      if (live && c < a.n) {
        float r[VEC];
        Chunk<T, VEC>::load(res + c, r);
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = __fadd_rn(v[i][j], r[j]);
        Chunk<T, VEC>::store(static_cast<T*>(a.sum) + row * a.lds + c, v[i]);
      }
    }
  }
  // max.NaN: a NaN stays
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 32 * W + lane) * VEC;
    float g[VEC];
    if constexpr (NORM) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) g[j] = 1.0f;
      if (w && c < a.n) Chunk<T, VEC>::load(w + c, g);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (NORM) squares = fmaf(v[i][j], v[i][j], squares);
      const float u = NORM ? __fmul_rn(v[i][j], g[j]) : v[i][j];
      top = max_nan(top, fabsf(u));
      if constexpr (NORM) v[i][j] = u;
    }
  }
  const RowSums s = row_sums<W>(top, squares, tops, sums, 0);
  const RowScale q = row_scale(s.top);
  float scale = q.scale;
  if constexpr (NORM) {
    float f = rescue(s.squares, a.eps), all = s.squares;
    // The same for all lanes of a row; a block of several rows goes there together.
    if (kRows > 1 ? __syncthreads_or(f != 1.0f) : f != 1.0f) {
      float again = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * 32 * W + lane) * VEC;
        if (live && c < a.n) {
          const T* from = a.residual ? static_cast<const T*>(a.sum) + row * a.lds : x;
          float h[VEC];
          Chunk<T, VEC>::load(from + c, h);
#pragma unroll
          for (int j = 0; j < VEC; ++j) again = fmaf(h[j] * f, h[j] * f, again);
        }
      }
      all = row_sums<W>(0.0f, again, tops, sums, 1).squares;
    }
    scale = q.scale > 0.0f ? q.scale * norm_factor(all, a.n, a.eps, f) : q.scale;
  }
  if (!live) return;
  int8_t* codes = a.codes + row * a.ldc;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * 32 * W + lane) * VEC;
    if (c < a.n) {
      if (q.inv == 0.0f) {  // no 0 times infinity
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = 0.0f;
      }
      store_codes<VEC>(codes + c, v[i], q.inv);
    }
  }
  if (lane == 0) a.scales[row] = scale;
}

// Rows that do not fit the registers of 32 warps: one block a row, read again for the codes.
template <typename T, bool NORM>
__global__ void __launch_bounds__(1024) long_rows_s8_kernel(RowsArgs a) {
  __shared__ uint32_t tops[2][32];
  __shared__ float sums[2][32];
  wait_for_previous();
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = static_cast<const T*>(a.residual) + row * a.ldr;
  T* sum = static_cast<T*>(a.sum) + row * a.lds;
  const T* w = static_cast<const T*>(a.w);
  float top = 0.0f, squares = 0.0f;
  for (int c = threadIdx.x; c < a.n; c += 1024) {
    float h = to_f32(x[c]);
    if (a.residual) {
      const T kept = from_f32<T>(__fadd_rn(h, to_f32(res[c])));
      sum[c] = kept;
      h = to_f32(kept);
    }
    squares = fmaf(h, h, squares);
    top = max_nan(top, fabsf(NORM && w ? __fmul_rn(h, to_f32(w[c])) : h));
  }
  const RowSums s = row_sums<32>(top, squares, tops, sums, 0);
  const RowScale q = row_scale(s.top);
  const T* from = a.residual ? sum : x;
  float scale = q.scale;
  if constexpr (NORM) {
    const float f = rescue(s.squares, a.eps);
    float all = s.squares;
    if (f != 1.0f) {
      float again = 0.0f;
      for (int c = threadIdx.x; c < a.n; c += 1024) {
        const float h = to_f32(from[c]) * f;
        again = fmaf(h, h, again);
      }
      all = row_sums<32>(0.0f, again, tops, sums, 1).squares;
    }
    scale = q.scale > 0.0f ? q.scale * norm_factor(all, a.n, a.eps, f) : q.scale;
  }
  for (int c = threadIdx.x; c < a.n; c += 1024) {
    float u[1] = {to_f32(from[c])};
    if (NORM && w) u[0] = __fmul_rn(u[0], to_f32(w[c]));
    if (q.inv == 0.0f) u[0] = 0.0f;
    store_codes<1>(a.codes + row * a.ldc + c, u, q.inv);
  }
  if (threadIdx.x == 0) a.scales[row] = scale;
}

struct ReadArgs {
  const int8_t* codes;
  long long ldc;
  const float* scales;
  void* y;
  long long ldy;
  int t, n;
  Divisor chunks;  // of a row
};

// A thread has one piece of VEC codes; where rows are not aligned 8 codes that lie 32 apart.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) read_s8_kernel(ReadArgs a, uint32_t units) {
  wait_for_previous();
  constexpr int kApart = VEC == 1 ? 8 : 1;
  const uint32_t unit = VEC == 1 ? blockIdx.x * 8u + threadIdx.x / 32 : blockIdx.x * 256u + threadIdx.x;  // fewer than 2^31
  if (unit >= units) return;
  const uint32_t row = a.chunks.of(unit);
  const int c = VEC == 1 ? static_cast<int>(unit - row * a.chunks.d) * 256 + threadIdx.x % 32 : static_cast<int>(unit - row * a.chunks.d) * VEC;
  const int8_t* p = a.codes + static_cast<long long>(row) * a.ldc + c;
  T* y = static_cast<T*>(a.y) + static_cast<long long>(row) * a.ldy + c;
  const float s = __ldg(a.scales + row);
  if constexpr (VEC == 1) {
    int8_t code[kApart];
#pragma unroll
    for (int i = 0; i < kApart; ++i) code[i] = c + 32 * i < a.n ? p[32 * i] : int8_t{0};
#pragma unroll
    for (int i = 0; i < kApart; ++i)
      if (c + 32 * i < a.n) y[32 * i] = from_f32<T>(static_cast<float>(code[i]) * s);
  } else {
    uint32_t words[VEC / 4];
    if constexpr (VEC == 8) {
      const uint2 b = *reinterpret_cast<const uint2*>(p);
      words[0] = b.x, words[1] = b.y;
    } else {
      words[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    // 2^23 + 128 + code in an fp32's bits, exact; the conversion unit takes four times as long as the bytes
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      v[j] = (__uint_as_float(__byte_perm(words[j / 4] ^ 0x80808080u, 0x4B000000u, 0x7440 + j % 4)) - 8388736.0f) * s;
    Chunk<T, VEC>::store(y, v);
  }
}

template <typename T, int VEC, int NV, int W>
int launch_rows(const RowsArgs& a, bool norm, cudaStream_t cs) {
  constexpr int kRows = (W > 8 ? W : 8) / W;
  const dim3 grid(static_cast<unsigned>((a.t + kRows - 1) / kRows));
  return host_launch("rows_s8_kernel launch", norm ? rows_s8_kernel<T, VEC, NV, W, true> : rows_s8_kernel<T, VEC, NV, W, false>,
                     grid, 32 * (W > 8 ? W : 8), 0, cs, 1, a);
}

// The fewest warps that hold a row.
template <typename T, int VEC, int NV>
int launch_warps(const RowsArgs& a, bool norm, cudaStream_t cs) {
  const int per = 32 * VEC * NV;
  if (a.n <= per) return launch_rows<T, VEC, NV, 1>(a, norm, cs);
  if (a.n <= 2 * per) return launch_rows<T, VEC, NV, 2>(a, norm, cs);
  if (a.n <= 4 * per) return launch_rows<T, VEC, NV, 4>(a, norm, cs);
  if (a.n <= 8 * per) return launch_rows<T, VEC, NV, 8>(a, norm, cs);
  if (a.n <= 16 * per) return launch_rows<T, VEC, NV, 16>(a, norm, cs);
  if (a.n <= 32 * per) return launch_rows<T, VEC, NV, 32>(a, norm, cs);
  return host_launch("long_rows_s8_kernel launch", norm ? long_rows_s8_kernel<T, true> : long_rows_s8_kernel<T, false>,
                     dim3(static_cast<unsigned>(a.t)), 1024, 0, cs, 1, a);
}

int rows_s8(const b200q_rows_s8_args* p, bool norm, void* stream) {
  if (!p) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const int ftype = p->ftype;
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (p->t < 0 || p->n < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative dimensions");
  if (norm && !(p->eps >= 0.0f && p->eps < INFINITY))
    return host_fail(B200Q_ERR_INVALID_ARG, "eps must be finite and not negative, got %g", static_cast<double>(p->eps));
  if (p->t == 0 || p->n == 0) {
    if (p->t > 0) return host_fail(B200Q_ERR_INVALID_ARG, "rows of no elements have no scale");
    return B200Q_OK;
  }
  if (p->t > (1 << 30) || p->n > (1 << 30)) return host_fail(B200Q_ERR_UNSUPPORTED, "%d rows of %d: too large", p->t, p->n);
  if (!p->x || !p->codes || !p->scales || (p->residual && !p->sum)) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (!norm && (p->w || p->residual)) return host_fail(B200Q_ERR_INVALID_ARG, "a weight or a residual without a norm");
  if (p->ldc < p->n && p->t > 1) return host_fail(B200Q_ERR_INVALID_ARG, "row stride of the codes smaller than a row");
  if (p->residual && p->lds < p->n && p->t > 1) return host_fail(B200Q_ERR_INVALID_ARG, "row stride of the sum smaller than a row");
  int sms = 0, *err = nullptr;
  if (int rc = host_device(&sms, &err)) return rc;
  const RowsArgs a{p->x, p->ldx, p->w, p->residual, p->ldr, p->sum, p->lds, p->codes, p->ldc, p->scales, p->t, p->n, p->eps};
  const int size = ftype == B200Q_F32 ? 4 : 2, vec = 16 / size;
  uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w);
  long long ld = a.ldx;
  if (a.residual) {
    bits |= reinterpret_cast<uintptr_t>(a.residual) | reinterpret_cast<uintptr_t>(a.sum);
    ld |= a.ldr | a.lds;
  }
  const bool wide = !(bits & 15u) && a.n % vec == 0 && (a.t == 1 || ld % vec == 0) &&
                    !((reinterpret_cast<uintptr_t>(a.codes) | (a.t == 1 ? 0 : a.ldc)) & (vec - 1));
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  int rc = B200Q_OK;
  // 16 elements a lane up to eight warps a row, then 32: a block of 16 or 32 warps waits long at its barrier for the row's slowest (us:
  // 500 x 16384 bf16 10.2 with 16, 7.0 with 32; 30000 x 512 fp16 11.9 with 16, 16.5 with 32; 1021 x 5004 fp32 8.1 and 6.6).
  constexpr int kFew = 4096;
  B200Q_DISPATCH_FTYPE(ftype, rc = !wide          ? launch_warps<T, 1, 16>(a, norm, cs)
                                   : a.n <= kFew ? launch_warps<T, 16 / sizeof(T), sizeof(T)>(a, norm, cs)
                                                 : launch_warps<T, 16 / sizeof(T), 2 * sizeof(T)>(a, norm, cs));
  if (rc == B200Q_OK) host_set_path(21);
  return rc;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_quantize_s8(const b200q_rows_s8_args* args, void* stream) { return rows_s8(args, false, stream); }
extern "C" int b200q_rms_norm_s8(const b200q_rows_s8_args* args, void* stream) { return rows_s8(args, true, stream); }

extern "C" int b200q_read_s8(const b200q_read_s8_args* args, void* stream) {
  if (!args) return host_fail(B200Q_ERR_INVALID_ARG, "null argument");
  const auto [codes, ldc, scales, y, ldy, ftype, t, n] = *args;
  if (ftype < B200Q_F32 || ftype > B200Q_BF16) return host_fail(B200Q_ERR_INVALID_ARG, "bad floating type %d", ftype);
  if (t < 0 || n < 0) return host_fail(B200Q_ERR_INVALID_ARG, "negative dimensions");
  if (t == 0 || n == 0) return B200Q_OK;
  if (!codes || !scales || !y) return host_fail(B200Q_ERR_INVALID_ARG, "null tensor pointer");
  if (ldy < n && t > 1) return host_fail(B200Q_ERR_INVALID_ARG, "row stride of the values smaller than a row");
  int sms = 0, *err = nullptr;
  if (int rc = host_device(&sms, &err)) return rc;
  const int size = ftype == B200Q_F32 ? 4 : 2, vec = 16 / size;
  const bool aligned = n % vec == 0 && !(reinterpret_cast<uintptr_t>(y) & 15u) && (t == 1 || ldy % vec == 0) &&
                       !((reinterpret_cast<uintptr_t>(codes) | (t == 1 ? 0 : ldc)) & (vec - 1));
  const int chunks = aligned ? n / vec : (n + 255) / 256, per_block = aligned ? 256 : 8;
  const long long units = static_cast<long long>(t) * chunks;
  if (units > 0x7fffff00ll) return host_fail(B200Q_ERR_UNSUPPORTED, "too many elements");
  const ReadArgs a{codes, ldc, scales, y, ldy, t, n, Divisor(static_cast<uint32_t>(chunks))};
  const dim3 grid(static_cast<unsigned>((units + per_block - 1) / per_block));
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  int rc = B200Q_OK;
  B200Q_DISPATCH_FTYPE(ftype, rc = host_launch("read_s8_kernel launch", aligned ? read_s8_kernel<T, 16 / sizeof(T)> : read_s8_kernel<T, 1>,
                                               grid, 256, 0, cs, 1, a, static_cast<uint32_t>(units)));
  if (rc == B200Q_OK) host_set_path(21);
  return rc;
}
