/*
 * b200q -- B200-native (sm_100a) int8 / quantized-int32 NHWC convolution and
 * batched GEMM behind a plain C ABI.
 *
 * Every entry point takes device pointers, plain sizes and a CUDA stream passed
 * as `void*` (a cudaStream_t; NULL = legacy default stream), returns an int
 * status (B200Q_OK on success) and never throws.  The message of the last
 * failure on the calling thread is returned by b200q_last_error().
 * Launches are asynchronous on `stream` unless stated otherwise.
 *
 * Drop-in mapping (reference = NikitaYak02/my_own_cnn):
 *   b200q_fprop_nhwc_qi32        replaces conv_quant_detail::launch_fprop_nhwc_qi32_{u8,s5}
 *                                (src/conv_types.h:232-241, src/cuda_kernels.cu:1336-1392,1465-1481)
 *   b200q_block_fprop_nhwc_qi32  replaces conv_quant_detail::launch_block_fprop_nhwc_qi32_{u8,s5}
 *                                (src/conv_types.h:242-251, src/cuda_kernels.cu:1394-1461,1483-1497)
 *   b200q_bmm_matmul_i32         replaces bmm_matmul_i32 (bmm.h:69-74, bmm.cu:298-322)
 *   b200q_conv_fprop_f32         replaces launch_fprop_nhwc / launch_block_fprop_nhwc
 *                                (src/conv_types.h:287-299, src/cuda_kernels.cu:767-823, 939-998)
 *   b200q_conv_bprop_f32         replaces launch_bprop_nhwc / launch_block_bprop_nhwc
 *                                (src/conv_types.h:290-302, src/cuda_kernels.cu:825-872, 1000-1057)
 *   b200q_conv_grad_f32          replaces launch_grad_nhwc / launch_block_grad_nhwc
 *                                (src/conv_types.h:293-306, src/cuda_kernels.cu:874-937, 1059-1136)
 *   b200q_bmm_f32                replaces bmm_matmul (bmm.h:36-39, bmm.cu:270-296); the layer API
 *                                bmm_fprop / bmm_bprop* (bmm.h:41-66) is defined over it by the shim
 * New entry points (int8 storage, fused requantization; no reference counterpart):
 *   b200q_conv2d_s8, b200q_bmm_s8.
 * The C++ shim my_own_cnn_b200/shim/reference_shim.cpp defines the reference's
 * own symbols on top of these, so reference callers link unchanged.
 */
#ifndef B200Q_H_
#define B200Q_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---- */
enum b200q_status {
  B200Q_OK = 0,
  B200Q_ERR_INVALID_ARG = 1,  /* bad shape / pointer / parameter (the reference throws here) */
  B200Q_ERR_UNSUPPORTED = 2,  /* valid request this build cannot run */
  B200Q_ERR_CUDA = 3,         /* a CUDA runtime / driver call failed */
  B200Q_ERR_TIMEOUT = 4       /* a device-side wait ran out; the kernel returned early */
};

/* ---- quantized input types: same values as nnalgebra::DataType (src/nnalgebra_quantization.h:19-24) ---- */
enum b200q_qtype { B200Q_LINQUANT_U8 = 1, B200Q_LINQUANT_S5 = 2 };

/* Same layout as Conv2DParams (src/conv_types.h:21-29). */
typedef struct b200q_conv_params {
  int pad_h, pad_w, stride_h, stride_w, dilation_h, dilation_w, groups;
} b200q_conv_params;

/* Same layouts as QuantizationParameters<LinQuantU8/LinQuantS5>
 * (src/nnalgebra_quantization.h:29-41).  Only zero_point is read. */
typedef struct b200q_qparams_u8 {
  uint8_t zero_point;
  float scale;
  uint8_t symmetric; /* C++ bool */
} b200q_qparams_u8;
typedef struct b200q_qparams_s5 {
  int8_t zero_point;
  uint8_t n_bins;
  float scale;
} b200q_qparams_s5;

/* ---- output epilogue of the int8 entry points ----
 * out_kind B200Q_OUT_S32 : y[m][k] = acc + bias[k]                       (int32, wrapping; bias may be NULL)
 * out_kind B200Q_OUT_S8  : t = acc + bias[k] (int32 wrap); p = (float)t * scale[k] (fp32, RNE);
 *                          q = rint(clamp(p, clamp_lo - zp_out, clamp_hi - zp_out)) + zp_out  (half to even);
 *                          stored as int8.  ReLU = clamp_lo = zp_out; ReLU6 = clamp_hi = q6.
 * out_kind B200Q_OUT_F32 : y = (float)(acc + bias[k]) * scale[k]        (fp32, RNE)
 * For bmm, "k" is the output column n (per-column bias / scale). */
enum b200q_out_kind { B200Q_OUT_S32 = 0, B200Q_OUT_S8 = 1, B200Q_OUT_F32 = 2 };
typedef struct b200q_epilogue {
  int out_kind;
  int zp_out;
  int clamp_lo;
  int clamp_hi;
} b200q_epilogue;

/* ---- drop-in entry points ---- */

/* Quantized NHWC conv forward, int32 accumulators.
 * d_x: [n,h,w,c] float codes, d_w: [k,r,s,c/groups] float codes (cast with truncation
 * like static_cast<int32_t>), d_y: [n,ho,wo,k] int32, every element written.
 * d_in_qp: device array of n qparams (per image), d_f_qp: device pointer to one qparams,
 * of the struct type selected by qtype.
 * y = sum over valid taps of (x - zp_in[img]) * (w - zp_f), int32 wrapping.
 * Runs on tcgen05 tensor cores (raw 8-bit codes, zero points restored by per-row / per-column terms;
 * codes outside the 8-bit range fall back to a direct computation on the device), except groups of
 * (c/groups) * (k/groups) <= 16 channel pairs, which run on a direct CUDA-core kernel.  Uses the
 * stream's workspace for the 8-bit operands.
 * Replaces conv_quant_detail::launch_fprop_nhwc_qi32_{u8,s5} (src/conv_types.h:232-241). */
int b200q_fprop_nhwc_qi32(int qtype, const float* d_x, const float* d_w, int32_t* d_y, int n, int h,
                          int w, int c, int r, int s, int k, const b200q_conv_params* p,
                          const void* d_in_qp, const void* d_f_qp, void* stream);

/* Blocked variant: the filter slice is chosen by the output block
 * (by = ho / (ho_total / block_by), bx = wo / (wo_total / block_bx));
 * d_w: [k, block_by, block_bx, r, s, c/groups].
 * Replaces conv_quant_detail::launch_block_fprop_nhwc_qi32_{u8,s5} (src/conv_types.h:242-251). */
int b200q_block_fprop_nhwc_qi32(int qtype, const float* d_x, const float* d_w, int32_t* d_y, int n,
                                int h, int w, int c, int r, int s, int k,
                                const b200q_conv_params* p, int block_by, int block_bx,
                                const void* d_in_qp, const void* d_f_qp, void* stream);

/* Row-major int32 batched GEMM, C_b = op(A_b) @ op(B_b), int32 wrap-around.
 * Layouts as bmm.h:9-29.  Replaces bmm_matmul_i32 (bmm.h:69-74).
 * With 16-byte aligned A, B and C, K < 2^17 and the contiguous dimensions of A and B multiples of
 * 16, the operands are first copied to int8 in the stream's workspace and multiplied by the
 * tcgen05 GEMM (path 16); if any value lies outside [-128, 127] a device flag makes the CUDA-core
 * kernel recompute C from the int32 operands, so every input gives the same C without a host
 * round trip.  Other shapes run the CUDA-core kernel directly (path 6). */
int b200q_bmm_matmul_i32(const int32_t* A, const int32_t* B, int32_t* C, int batch, int M, int N,
                         int K, int trans_a, int trans_b, void* stream);

/* ---- fp32 drop-ins (tensor cores, 3 x TF32 split products) ----
 * All tensors fp32 in the reference's layouts: x / dx [n,h,w,c], y / dy [n,ho,wo,k],
 * w / dw [k, block_by, block_bx, r, s, c/groups] (block_by = block_bx = 1: the regular KRSC filter).
 * Each operand is split as hi + lo (hi = the value rounded to TF32's 10-bit mantissa, lo = the exact
 * remainder) and the products hi*hi + hi*lo + lo*hi are summed in fp32 by kind::tf32 tcgen05 MMAs,
 * so results agree with an fp32 loop to about 1e-6 of sum(|x||w|) per output (the tests bound the
 * difference to an exact float64 sum by 1e-5 * sum(|x||w|)).  Summation order differs from the
 * reference's loops, so results are not bit-identical to them.  Inputs are assumed finite.
 * Workspace: a per-(device, stream) grow-only buffer holding the split operands.  Groups with
 * (c/groups) * (k/groups) <= 16 (depthwise and the like) run on CUDA-core fp32 kernels instead:
 * a GEMM per group would have 1-4 rows or columns. */

/* y = conv(x, w) (+ bias of the output block).  d_bias: NULL or [k * block_by * block_bx];
 * bias_mode 0 = one bias per (k, block), 1 = one per k shared by all blocks, at index
 * k * block_by * block_bx (BlockBiasMode, src/conv_types.h:36-39, 184-188). */
int b200q_conv_fprop_f32(const float* d_x, const float* d_w, const float* d_bias, int bias_mode, float* d_y, int n,
                         int h, int w, int c, int r, int s, int k, const b200q_conv_params* p, int block_by,
                         int block_bx, void* stream);

/* dx = data gradient of the conv for dy (n, h, w, c are dx's dimensions, as in the reference). */
int b200q_conv_bprop_f32(const float* d_dy, const float* d_w, float* d_dx, int n, int h, int w, int c, int r, int s,
                         int k, const b200q_conv_params* p, int block_by, int block_bx, void* stream);

/* dw = filter gradient; d_dbias (NULL or [k * block_by * block_bx]) receives the blocked bias
 * gradient with the reference's rule (src/cpu_ref.cpp:318-371): dy summed over the block's output
 * pixels whose tap (0, 0) input lies inside the image. */
int b200q_conv_grad_f32(const float* d_x, const float* d_dy, float* d_dw, float* d_dbias, int bias_mode, int n, int h,
                        int w, int c, int r, int s, int k, const b200q_conv_params* p, int block_by, int block_bx,
                        void* stream);

/* Row-major fp32 batched GEMM, C_b = op(A_b) @ op(B_b), layouts as bmm.h:9-29. */
int b200q_bmm_f32(const float* A, const float* B, float* C, int batch, int M, int N, int K, int trans_a, int trans_b,
                  void* stream);

/* ---- new int8 entry points ---- */

/* int8 NHWC conv: d_x [n,h,w,c] int8, d_w [k,r,s,c/groups] int8, zero points 0,
 * int32 accumulation, fused epilogue (see b200q_epilogue).  d_y element type per out_kind.
 * d_bias: [k] int32 or NULL; d_scale: [k] fp32 (required for S8 / F32 outputs). */
int b200q_conv2d_s8(const int8_t* d_x, const int8_t* d_w, const int32_t* d_bias,
                    const float* d_scale, void* d_y, int n, int h, int w, int c, int r, int s,
                    int k, const b200q_conv_params* p, const b200q_epilogue* epi, void* stream);

/* b200q_conv2d_s8 with a residual add fused into the int8 epilogue (the shortcut of a ResNet /
 * MobileNetV2 block; no reference counterpart):
 *   p = fp32(acc + bias[k]) * scale[k] + fp32(res[pixel][k]) * res_scale   (IEEE steps, no fma)
 *   q = clamp(rint(p), lo - zp, hi - zp) + zp
 * d_res: int8 NHWC with the output's shape, 16-byte aligned for the tensor-core paths.  int8 outputs
 * only (B200Q_ERR_INVALID_ARG otherwise). */
int b200q_conv2d_s8_add(const int8_t* d_x, const int8_t* d_w, const int32_t* d_bias, const float* d_scale,
                        const int8_t* d_res, float res_scale, int8_t* d_y, int n, int h, int w, int c, int r,
                        int s, int k, const b200q_conv_params* p, const b200q_epilogue* epi, void* stream);

/* int8 NHWC max pool (R x S window, stride, zero-free padding: padded positions take no part).
 * Output [n, (h + 2*pad_h - r)/stride_h + 1, (w + 2*pad_w - s)/stride_w + 1, c]. */
int b200q_maxpool_s8(const int8_t* d_x, int8_t* d_y, int n, int h, int w, int c, int r, int s, int stride_h,
                     int stride_w, int pad_h, int pad_w, void* stream);

/* int8 NHWC global average pool -> [n][c]: q = clamp(rint(fp32(sum) / fp32(h*w)), -128, 127). */
int b200q_global_avgpool_s8(const int8_t* d_x, int8_t* d_y, int n, int h, int w, int c, void* stream);

/* int8 batched GEMM, layouts as bmm.h:9-29, int32 accumulation, per-column epilogue.
 * d_bias: [N] int32 or NULL; d_col_scale: [N] fp32 (required for S8 / F32 outputs). */
int b200q_bmm_s8(const int8_t* A, const int8_t* B, const int32_t* d_bias, const float* d_col_scale,
                 void* C, int batch, int M, int N, int K, int trans_a, int trans_b,
                 const b200q_epilogue* epi, void* stream);

/* ---- decoder operators with 4-bit storage (no reference counterpart) ----
 * Floating tensors are fp32, fp16 or bf16, one type per call (b200q_ftype); sums, norms and softmax
 * statistics are held in fp32.  Strides are in elements; the last dimension is contiguous.
 * A 4-bit code pair is one byte, low nibble first.  Positions, slots, page numbers and lengths live on
 * the device: one that is out of range is left out of the result (nothing is read or written for it)
 * and reported by the next b200q_device_error() as B200Q_ERR_INVALID_ARG.
 * Attention and the gradient use 8 MiB of scratch: a stream's, which the first of their calls on it makes (not while the
 * stream is captured: B200Q_ERR_UNSUPPORTED), or, for calls that are captured, the graph's own, which is given back when the
 * graph and what was instantiated from it are destroyed.  A destroyed stream's is used again for later streams.  Graphs
 * may be replayed beside one another and beside eager calls; two instances of one graph may not. */
enum b200q_ftype { B200Q_F32 = 0, B200Q_F16 = 1, B200Q_BF16 = 2 };

/* y[m][n] = sum_k x[m][k] * (code[n][k] - zero[k / group][n]) * scale[k / group][n] (+ bias[n]).
 * codes: [n][16 * ceil(k / 32)] bytes, 16-byte aligned (the nibbles past k are not used);
 * scales: bf16 [ceil(k / group)][n]; zeros: uint8 (0 to 255), same shape, or NULL for 8 everywhere;
 * group 32, 64 or 128.  x [m][k] with row stride ldx, y [m][n] with row stride ldy; bias [n] or NULL.
 * Made for the few rows of a decode step: weights are read once per 16 rows of x.  A NaN or an
 * infinity in a row of x makes that row's results NaN or infinite.  y shares no memory with x. */
typedef struct b200q_linear_w4_args {
  const void* x;
  int64_t ldx;
  const uint8_t* codes;
  const void* scales;
  const uint8_t* zeros;
  const void* bias;
  void* y;
  int64_t ldy;
  int ftype, m, n, k, group;
} b200q_linear_w4_args;
int b200q_linear_w4(const b200q_linear_w4_args* args, void* stream);

/* Per-head RMS norm of queries and keys, then the position rotation of each head's first `rot`
 * channels, in one pass:  y = R(pos[t]) (x * rsqrt(mean(x^2) + eps) * w).
 * q [t][hq][d], k [t][hk][d] with token / head strides; q_w, k_w [d] or NULL (all ones).
 * table: fp32 [positions][rot], cos of the rot / 2 angles, then sin; rot even, <= d, 0 for none.
 * Pairs are (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved.  q_out / k_out (with strides) may be
 * q / k.  The gradient's fields are not read. */
typedef struct b200q_qk_norm_args {
  const void *q, *k, *q_w, *k_w;
  const float* table;
  const int32_t* pos;
  void *q_out, *k_out;
  const void *q_grad, *k_grad;
  void *q_w_grad, *k_w_grad;
  int64_t q_ts, q_hs, k_ts, k_hs, qo_ts, qo_hs, ko_ts, ko_hs;
  int positions, ftype, t, hq, hk, d, rot, interleaved;
  float eps;
} b200q_qk_norm_args;
int b200q_qk_norm_rope(const b200q_qk_norm_args* args, void* stream);

/* Gradient of b200q_qk_norm_rope: q_grad / k_grad are the gradients of its outputs, contiguous
 * [t][h][d]; q_out / k_out (contiguous, their strides not read) receive those of its inputs, q_w_grad /
 * k_w_grad [d] (NULL: not wanted) those of the weights, summed over tokens and heads in a fixed order.
 * Recomputes the norms from q and k.  Uses the stream's scratch. */
int b200q_qk_norm_rope_bprop(const b200q_qk_norm_args* args, void* stream);

/* 4-bit paged key / value cache.  codes: [pages][heads][page_size][d / 2] bytes, 16-byte aligned;
 * params: [pages][heads][page_size][d / group] words (bits 0-15 the bf16 scale, 16-23 the zero point, 0 to 15);
 * value = (code - zero) * scale.  d 64, 128 or 256; group 32 or 64.  Slot = page * page_size + place. */
typedef struct b200q_kv4_cache {
  uint8_t* k_codes;
  uint32_t* k_params;
  uint8_t* v_codes;
  uint32_t* v_params;
  int pages, heads, page_size, d, group;
} b200q_kv4_cache;

/* Quantizes k, v [t][heads][d] into slots[t] (int64; negative: not stored).  Per group, in fp32:
 *   lo = min(0, x), hi = max(0, x), s = bf16((hi - lo) * (1 / 15)) (0 when below the smallest normal),
 *   zero = clamp(rint(-lo * (1 / s)), 0, 15), code = clamp(rint(x * (1 / s)) + zero, 0, 15).
 * A group with a NaN or an infinity in it (or whose hi - lo passes fp32's range) gets the scale NaN: its values read back as
 * NaN, and attention rows that see it are NaN.
 * Every slot is named at most once in a call. */
int b200q_kv4_append(const b200q_kv4_cache* c, const void* k, long long k_ts, long long k_hs, const void* v,
                     long long v_ts, long long v_hs, const int64_t* slots, int ftype, int t, void* stream);

/* The values held in slots[t], contiguous [t][heads][d], 32-byte aligned; zeros for negative slots. */
int b200q_kv4_read(const b200q_kv4_cache* c, const int64_t* slots, void* k, void* v, int ftype, int t, void* stream);

/* Attention of tq new tokens per sequence over the cache, which already holds them:
 * token i of sequence b sees the first lens[b] - tq + i + 1 places of its pages
 * block_table[b][0 .. max_pages), row stride bt_stride; none seen: output 0, lse -inf.
 * q [b][tq][hq][d] with strides; query head h reads cache head h / (hq / heads).
 * out contiguous [b][tq][hq][d]; lse fp32 [b][tq][hq] or NULL: log of the sum of exp(scale * q.k).
 * Uses the stream's scratch: sequences are split over blocks.  Lengths and tables stay as they are until the call has run: what
 * changes them is put into the same stream, or waits. */
typedef struct b200q_kv4_attention_args {
  const void* q;
  int64_t q_bs, q_ts, q_hs;
  const int32_t* block_table;
  int64_t bt_stride;
  const int32_t* lens;
  void* out;
  float* lse;
  int ftype, b, tq, hq, max_pages;
  float scale;
} b200q_kv4_attention_args;
int b200q_kv4_attention(const b200q_kv4_cache* c, const b200q_kv4_attention_args* args, void* stream);

/* 8-bit rows: codes int8 [t][n] with row stride ldc and one fp32 scale a row; value = code * scale.
 * b200q_quantize_s8 rounds rows u = x; b200q_rms_norm_s8 rows
 *   u = h * w (w [n] or NULL for all ones), h = x + residual (residual NULL: x), both sums and products rounded
 *   once, h to the rows' own type: it is written to `sum`, which may be x or the residual.
 * code = rint(u * fl(127 * fl(1 / max|u|))), the product exact, ties to even; scale = max|u| / 127, for the norm times
 * (mean(h^2) + eps)^-1/2.  A row with a NaN or an infinity among u has the scale NaN (its values read as NaN) and codes 0; one
 * with nothing above 2^-119 has scale and codes 0.  b200q_quantize_s8 reads x, codes, scales and sizes alone (the other pointers NULL). */
typedef struct b200q_rows_s8_args {
  const void* x;
  int64_t ldx;
  const void* w;
  const void* residual;
  int64_t ldr;
  void* sum;
  int64_t lds;
  int8_t* codes;
  int64_t ldc;
  float* scales;
  int ftype, t, n;
  float eps;
} b200q_rows_s8_args;
int b200q_quantize_s8(const b200q_rows_s8_args* args, void* stream);
int b200q_rms_norm_s8(const b200q_rows_s8_args* args, void* stream);

/* y[t][n] (row stride ldy, of ftype) = codes * scales, rounded once. */
typedef struct b200q_read_s8_args {
  const int8_t* codes;
  int64_t ldc;
  const float* scales;
  void* y;
  int64_t ldy;
  int ftype, t, n;
} b200q_read_s8_args;
int b200q_read_s8(const b200q_read_s8_args* args, void* stream);

/* y[m][n] = (sum_k x[m][k] * w[n][k]) * w_scale[n] * x_scale[m] (+ bias[n]) for 8-bit rows x [m][k] and w [n][k]: the sum exact in
 * 32-bit integers (k <= 131071), the rest in fp32 in this order, y of ftype with row stride ldy; bias [n] of ftype or NULL.  Codes lie on
 * 16-byte boundaries with row strides that are multiples of 16; what lies past k is not used.  A row or a channel with
 * the scale NaN gives NaN.  y shares no memory with the other tensors. */
typedef struct b200q_linear_s8_args {
  const int8_t* x;
  int64_t ldx;
  const float* x_scales;
  const int8_t* w;
  int64_t ldw;
  const float* w_scales;
  const void* bias;
  void* y;
  int64_t ldy;
  int ftype, m, n, k;
} b200q_linear_s8_args;
int b200q_linear_s8(const b200q_linear_s8_args* args, void* stream);

/* Causal attention over packed prompts.  Sequence i has the query rows starts[i] .. starts[i + 1] of q [tq][hq][d] and the key rows
 * k_starts[i] .. k_starts[i + 1] of k, v [tk][hk][d] (k_starts NULL: starts; all with token and head strides, channels
 * contiguous); starts int32 [b + 1] on the device.  The last query is in line with the last key: row j of lq
 * sees the first lk - lq + j + 1 keys; where that is none the output is 0 (lse -inf).  Query head h reads head
 * h / (hq / hk).  out contiguous [tq][hq][d]; lse fp32 [tq][hq] or NULL: log of the sum of exp(scale * q.k).
 * Rows outside every sequence are left as they are.  A sequence whose starts decrease or pass the rows is left out and
 * reported by b200q_device_error().  What a row does not see has no part in it, NaN and infinities among it.
 * d up to 256; scale and its product with log2(e) finite.  Uses the stream's scratch where few rows see many keys: their parts are
 * joined by a second kernel. */
typedef struct b200q_prompt_attention_args {
  const void* q;
  int64_t q_ts, q_hs;
  const void* k;
  int64_t k_ts, k_hs;
  const void* v;
  int64_t v_ts, v_hs;
  const int32_t* starts;
  const int32_t* k_starts;
  void* out;
  float* lse;
  int ftype, b, tq, tk, hq, hk, d;
  float scale;
} b200q_prompt_attention_args;
int b200q_prompt_attention(const b200q_prompt_attention_args* args, void* stream);

/* Packed low-channel int8 conv that allocates nothing (no counterpart in the reference).
 * For callers that may not allocate device memory at all: for example plugins inside a runtime
 * that owns and budgets every byte of GPU memory itself, or latency-critical loops where a
 * cudaMalloc (which can synchronise the device) is not acceptable.  Same arguments, arithmetic
 * and results as b200q_conv2d_s8 on its packed path (im2col matrix + tcgen05 GEMM), for any
 * groups == 1 conv; the im2col matrix and padded weights live in one fixed 32 MiB device array
 * of this library instead of a workspace (every GPU that loads the library holds that array
 * until the process exits).  Limit: round256(N*Ho*Wo*kp) + round256(K*kp) <= 32 MiB with
 * kp = round_up(R*S*C, 32) <= 16384 (the packed path's own limit; a larger kp returns
 * B200Q_ERR_UNSUPPORTED); larger scratch requests return B200Q_ERR_INVALID_ARG with the sizes
 * in b200q_last_error().  The first call on a device looks up the array's device address
 * (cudaGetSymbolAddress) and keeps it for the life of the process; make that first call before
 * any stream capture, and do not reset the device (cudaDeviceReset) between calls.  All calls on a
 * device share the array: every byte the kernels read is rewritten by the same call, but calls
 * that overlap on the GPU (different streams, or host threads sharing a device) race. */
int b200q_conv2d_s8_packed_noalloc(const int8_t* d_x, const int8_t* d_w, const int32_t* d_bias,
                                   const float* d_scale, void* d_y, int n, int h, int w, int c, int r,
                                   int s, int k, const b200q_conv_params* p,
                                   const b200q_epilogue* epi, void* stream);

/* Size in bytes of the fixed scratch array behind b200q_conv2d_s8_packed_noalloc. */
size_t b200q_noalloc_scratch_bytes(void);

/* ---- host utilities ---- */

/* Kernel family (b200q_last_path code) that b200q_conv2d_s8 / b200q_conv2d_s8_add
 * (has_residual != 0) would dispatch this conv to, assuming 16-byte aligned tensor pointers and
 * the current path policy; decided on the host without launching anything (the SM count of the
 * current device, or 148 when no GPU is visible).  The same decision drives the dispatch. */
int b200q_conv2d_s8_plan(int n, int h, int w, int c, int r, int s, int k, const b200q_conv_params* p,
                         const b200q_epilogue* epi, int has_residual, int* path);

/* Output shape with the checks of infer_conv_shape (src/conv_types.h:125-146). */
int b200q_conv_out_shape(int h, int w, int c, int r, int s, int k, const b200q_conv_params* p,
                         int* ho, int* wo);

/* Message of the last failed call on this thread ("" if none). */
const char* b200q_last_error(void);

/* Synchronizes the device, then reads and clears the device-side error word that
 * kernels set when a bounded wait runs out (B200Q_ERR_TIMEOUT) or when they meet a position, slot,
 * page or length that is out of range (B200Q_ERR_INVALID_ARG).  B200Q_OK when it is clear. */
int b200q_device_error(void);

/* Which kernel family the last conv / bmm call on this thread dispatched to:
 * 1 tcgen05 im2col conv, 2 tcgen05 tiled GEMM (for both: GEMMs of at least 2^36 MACs first prepack
 * their weights into per-stage images in the stream's workspace), 3 CUDA-core generic, 4 CUDA-core depthwise,
 * 5 CUDA-core quantized-int32 (drop-in), 6 CUDA-core int32 bmm, 7 tcgen05 GEMM over an im2col matrix
 * packed into the stream's workspace (low channel counts), 8 tcgen05 tiled GEMM on 2-SM pairs
 * (256-row tiles, one M = 256 MMA per K slice across a cluster of two CTAs), 9 tcgen05 row-tile
 * 3x3 conv (one input-window load per tile serves all nine taps), 10 tcgen05 row tiles over a
 * space-to-depth copy of a stride-2 low-channel input (network stems; the input and weights are
 * rearranged into the stream's workspace), 11 tcgen05 quantized-int32 drop-in (raw 8-bit codes and
 * zero-point correction terms), 12 CUDA-core depthwise with TMA-staged tiles, 13 tcgen05 fp32
 * (3 x TF32 split GEMM), 14 CUDA-core fp32 (groups of a few channels, e.g. depthwise), 15 tcgen05
 * pixel-grouped 1x1 GEMM (G pixels per row against block-diagonal weights built in the stream's
 * workspace, for layers with G * K <= 256 and G * C <= 256), 16 tcgen05 int32 bmm (operands copied
 * to int8, CUDA-core recompute only when a value does not fit), 17 4-bit weights linear, 18 per-head norm
 * and rotation (either direction), 19 4-bit cache append / read, 20 4-bit cache attention, 21 8-bit rows (quantized, normed or
 * read), 22 linear of 8-bit rows, 23 prompt attention on tcgen05, 24 prompt attention on mma.sync (fp32; rows and heads that TMA
 * cannot take). */
int b200q_last_path(void);

/* 0 = automatic dispatch (default); 1 = force the CUDA-core kernels (cross-checks). */
void b200q_set_path_policy(int policy);

/* Number of tcgen05 GEMM launches, and of the weight-prepack launches that feed them, issued since
   load (for launch accounting). */
long long b200q_tc_launch_count(void);

/* ---- seeded synthetic data (counter-based splitmix64; the CPU oracle regenerates any slice) ---- */
int b200q_fill_s8_uniform(int8_t* d_out, size_t count, uint64_t seed, uint64_t tensor_id, int lo,
                          int hi, void* stream);
int b200q_fill_i32_uniform(int32_t* d_out, size_t count, uint64_t seed, uint64_t tensor_id,
                           int32_t lo, int32_t hi, void* stream);
/* d_table: 65536 int8 codes in device memory (quantiles of the wanted distribution). */
int b200q_fill_s8_table(int8_t* d_out, size_t count, uint64_t seed, uint64_t tensor_id,
                        const int8_t* d_table, void* stream);

/* Failure-path self test: one CTA waits on an mbarrier that nothing completes, with a
 * limit of `cycles` SM clocks, then records a timeout and returns.  Synchronous.
 * Returns B200Q_ERR_TIMEOUT when the bounded wait behaved (the expected result). */
int b200q_selftest_wait_timeout(long long cycles);

#ifdef __cplusplus
}
#endif

#endif /* B200Q_H_ */
