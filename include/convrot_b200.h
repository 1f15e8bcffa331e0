/*
 * convrot_b200.h -- C ABI of libconvrot_b200.so, the sm_100a (B200) ConvRot
 * W4A4 linear.
 *
 * Every entry point takes device pointers, element counts and a cudaStream_t
 * (passed as void*, NULL = legacy default stream), enqueues its kernels on
 * that stream and returns at once.  No entry point allocates device memory:
 * the caller owns every buffer.  The library itself holds two device arrays
 * per device it is loaded on, for as long as the process lives: a 4-byte
 * error word, and the fixed CONVROT_LINEAR_STATIC_SCRATCH_BYTES (64 MiB)
 * intermediate of convrot_w4a4_linear_static.  Return value: CONVROT_OK (0)
 * or a negative status; convrot_last_error() then gives a message
 * (thread-local).
 *
 * Each function names the reference interface it replaces, as
 * path:line in Lumenbeing/convrot-mlx (src/convrot_mlx/core.py).
 *
 * Conventions shared by all entry points
 *   - matrices are row-major and densely packed (leading dimension = columns);
 *   - "dtype" codes: CONVROT_F32, CONVROT_F16, CONVROT_BF16;
 *   - int4 packing: two's-complement nibbles, element 2j in the low nibble
 *     and 2j+1 in the high nibble of byte j (core.py:97-120);
 *   - weight layouts: CONVROT_LAYOUT_NK = (N, K/2) bytes, packed along K
 *     ("packed-nk-low-nibble-even-feature", core.py:1253-1254);
 *     CONVROT_LAYOUT_KN = (K, N/2) bytes, packed along N
 *     ("packed-kn-low-nibble-even-output", core.py:1248-1250).
 */
#ifndef CONVROT_B200_H
#define CONVROT_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define CONVROT_OK 0
#define CONVROT_ERR_INVALID (-1)     /* bad shape, pointer, alignment or argument */
#define CONVROT_ERR_UNSUPPORTED (-2) /* valid for the reference, not for this build */
#define CONVROT_ERR_CUDA (-3)        /* a CUDA runtime / driver call failed */

/* dtype codes */
#define CONVROT_F32 0
#define CONVROT_F16 1
#define CONVROT_BF16 2

/* weight layouts */
#define CONVROT_LAYOUT_NK 0
#define CONVROT_LAYOUT_KN 1

/* ABI version of this header (major * 100 + minor). */
#define CONVROT_ABI_VERSION 100
int convrot_abi_version(void);

/* Message for the last non-zero status returned on this thread. */
const char* convrot_last_error(void);

/*
 * Fused rotate + row quantize, int8 codes.
 * Replaces metal_fused_prepare_convrot_activation_i8 (core.py:456-484; Metal
 * kernel core.py:307-327).  x: (rows, features) of `dtype`; q_i8: (rows,
 * features) int8 codes in [-7, 7]; scales: (rows,) float32 row scales.
 * group_size in {16, 64, 256, 1024} (the reference fuses 64 and 256 and
 * rotates any power of four eagerly, core.py:50-94); features % group_size == 0.
 * group_size 1 skips the rotation (quantize_signed_int4_rowwise,
 * core.py:149-158; then features % 32 == 0).
 */
int convrot_prepare_i8(const void* x, int dtype, int64_t rows, int64_t features,
                       int group_size, int8_t* q_i8, float* scales, void* stream);

/*
 * Fused rotate + row quantize, packed int4 codes.
 * Replaces metal_fused_prepare_convrot_activation (core.py:425-453; Metal
 * kernel core.py:205-304), prepare_convrot_activation (core.py:161-167),
 * compiled_prepare_convrot_activation (core.py:174) and, applied to a dense
 * (out, in) weight, quantize_convrot_weight (core.py:514-527).
 * q_packed: (rows, features / 2) bytes.
 */
int convrot_prepare_packed(const void* x, int dtype, int64_t rows, int64_t features,
                           int group_size, uint8_t* q_packed, float* scales, void* stream);

/*
 * Normalized regular-Hadamard rotation only, output in the input dtype.
 * Replaces metal_fused_rotate_convrot_activation (core.py:487-511; Metal
 * kernel core.py:330-370) and regular_hadamard (core.py:64-94).
 */
int convrot_rotate(const void* x, int dtype, int64_t rows, int64_t features,
                   int group_size, void* out, void* stream);

/*
 * Modulated LayerNorm fused into the prep: the int8 codes and row scales of
 * convrot_prepare_i8 applied to xm = bf16(fma(bf16(LayerNorm(x)),
 * bf16(1 + scale), shift)), the input of a FLUX-style DiT projection, with x
 * read once.  LayerNorm has no affine terms: mean and variance of the row in
 * float32, y = bf16((x - mean) * rsqrt(var + eps)).  shift / scale: one
 * bfloat16 vector of `features` per sample, sample s at s * mod_stride
 * elements (mod_stride % 8 == 0); row r belongs to sample r / rows_per_mod.
 * x bfloat16 only; group_size 64 or 256.  Bit for bit convrot_prepare_i8 of
 * the same xm; against a separate layer_norm + addcmul only the float32 order
 * of the row statistics differs, which can move a code by one.
 * No reference counterpart: it fuses the activation-preparation pass into the
 * producing op, the cost the reference names in docs/design.md:54-64 (its
 * prep alone is core.py:456-484).
 */
int convrot_modnorm_prepare_i8(const void* x, int dtype, int64_t rows, int64_t features, int group_size,
                               const void* shift, const void* scale, int64_t rows_per_mod, int64_t mod_stride,
                               float eps, int8_t* q_i8, float* scales, void* stream);

/*
 * The prep of a FLUX single block's output-projection input fused into its
 * producer: the int8 codes and row scales of convrot_prepare_i8 applied to
 * row r = [a[r, 0:da], gelu_tanh(m[r, 0:dm])] -- the attention output and
 * the MLP half of the block's input projection -- read straight from the two
 * tensors (row strides a_stride and m_stride elements, multiples of 8;
 * da % 16 == 0).  gelu_tanh(x) = 0.5 x (1 + tanh(0.7978845608028654 (x +
 * 0.044715 x^3))) in float32 with each product and sum rounded separately,
 * then one bf16 rounding.  bfloat16 only; group_size 64 or 256.  Bit for bit
 * convrot_prepare_i8 of the concatenated row.  No reference counterpart: the
 * same fusion of the preparation pass into the producing op as
 * convrot_modnorm_prepare_i8.
 */
int convrot_gelu_concat_prepare_i8(const void* a, int64_t a_stride, int64_t da, const void* m, int64_t m_stride,
                                   int64_t dm, int64_t rows, int group_size, int8_t* q_i8, float* scales,
                                   void* stream);

/*
 * Packed int4 -> int8.  Replaces metal_unpack_signed_int4 (core.py:1014-1027;
 * Metal kernel core.py:915-922) and unpack_signed_int4 (core.py:108-120).
 * packed: n_bytes bytes; out: 2 * n_bytes int8 values in [-8, 7].
 */
int convrot_unpack_int4(const uint8_t* packed, int64_t n_bytes, int8_t* out, void* stream);

/*
 * int8 -> packed int4 (values are taken modulo 16).  Replaces
 * pack_signed_int4 (core.py:97-105).  n_values must be even.
 */
int convrot_pack_int4(const int8_t* values, int64_t n_values, uint8_t* out, void* stream);

/*
 * Transpose a packed (rows, 2 * packed_cols) int4 matrix into a packed
 * (2 * packed_cols, rows) one: NK -> KN (repack_nk_weight_for_mpp,
 * core.py:123-133) and KN -> NK (repack_mpp_weight_to_nk, core.py:136-146).
 * rows must be even.  out: (2 * packed_cols, rows / 2) bytes.
 */
int convrot_repack_int4_transpose(const uint8_t* in, int64_t rows, int64_t packed_cols,
                                  uint8_t* out, void* stream);

/*
 * W4A4 linear: out[m, n] = T(float(sum_k a[m,k] w[n,k]) * xscales[m] *
 * wscales[n] + bias[n]) with an exact int32 dot (tcgen05 kind::i8) and the
 * epilogue fused.  Replaces mpp_w4a4_int8_matmul (core.py:1088-1120; Metal
 * K6 core.py:839-874 + epilogue K9 core.py:925-937), and, with layout NK,
 * the math of packed_w4a4_matmul* (core.py:745-828), expanded_fp32 /
 * reference_w4a4_matmul (core.py:1155-1207).
 * act: (m, k) int8 codes; qweight: packed `layout`; xscales (m,), wscales
 * (n,), bias (n,) float32 (bias may be NULL = zeros); out: (m, n) of
 * out_dtype.  k % 32 == 0; layout KN needs n even.
 */
int convrot_w4a4_gemm(const int8_t* act, const uint8_t* qweight, int layout,
                      const float* xscales, const float* wscales, const float* bias,
                      void* out, int out_dtype, int64_t m, int64_t n, int64_t k,
                      void* stream);

/*
 * W4A16 linear: out[m, n] = T(fl(dots[m, n] * wscales[n]) + bias[n]) with
 * dots = sum_k act[m, k] * w[k, n] accumulated in float32 (tcgen05
 * kind::f16; the nibbles are expanded to exact 16-bit integers in shared
 * memory).  Replaces mpp_w4a16_matmul (core.py:1123-1152; Metal K7
 * core.py:877-912, launched at core.py:961-969).  act: (m, k) rotated activations of act_dtype (bfloat16
 * or float16); qweight: packed `layout` (the reference passes K x packed-N);
 * wscales / bias (n,) float32 (bias may be NULL); out: (m, n) of out_dtype.
 * k % 64 == 0; layout KN needs n % 32 == 0 (16-byte weight rows for TMA).
 * The summation order differs from the reference's float32 matmul: results
 * agree to float32 rounding, not bit for bit.
 */
int convrot_w4a16_gemm(const void* act, int act_dtype, const uint8_t* qweight, int layout,
                       const float* wscales, const float* bias, void* out, int out_dtype,
                       int64_t m, int64_t n, int64_t k, void* stream);

/*
 * Tensor-parallel W4A4 (column split of N across the GPUs of one node): the
 * GEMM of this rank's shard -- qweight / wscales / bias hold columns
 * [col_offset, col_offset + n) of the full layer -- whose epilogue writes
 * every output tile into each of the n_outs (1..8) destinations at
 * dst[i * ldc + col_offset + j]: this GPU's full (m, ldc) output and the
 * peers' (device pointers valid on this GPU, e.g. symmetric memory), so the
 * all-gather of the outputs over NVLink overlaps the GEMM tile by tile.
 * Follow it with convrot_peer_barrier before any rank reads its full output.
 * No reference counterpart: the reference runs on one Apple GPU; this is the
 * multi-GPU form of mpp_w4a4_int8_matmul (core.py:1088-1120).  Needs
 * k % 128 == 0 and, for KN, n % 32 == 0.  outs: host array of n_outs device
 * pointers.
 */
int convrot_w4a4_gemm_gather(const int8_t* act, const uint8_t* qweight, int layout,
                             const float* xscales, const float* wscales, const float* bias,
                             void* const* outs, int n_outs, int64_t ldc, int64_t col_offset,
                             int out_dtype, int64_t m, int64_t n, int64_t k, void* stream);

/*
 * Flag barrier across `world` (1..8) GPUs of one node.  flag_arrays: host
 * array of `world` device pointers, valid on this GPU, to each rank's
 * (world,) uint32 flag array (zero-initialised, mapped by every rank).
 * Writes `epoch` (> 0, increasing per call) into slot `rank` of every array
 * with system-scope release stores, then waits, bounded by 2 s, until this
 * rank's array holds `epoch` in every slot (device error code 31 on time-out,
 * see convrot_take_device_error).  No reference counterpart.
 */
int convrot_peer_barrier(uint32_t* const* flag_arrays, int world, int rank, uint32_t epoch,
                         void* stream);

/*
 * A strided block copy on a copy engine (cudaMemcpy2DAsync, device to
 * device): rows x width_bytes, pitches in bytes.  dst may be a peer GPU's
 * memory mapped into this one (symmetric memory).  The tensor-parallel layer
 * pushes each M-chunk of its column shard into every rank's output with it,
 * overlapping the next chunk's GEMM; follow the copies with
 * convrot_peer_barrier.  No reference counterpart.
 */
int convrot_copy_2d(void* dst, int64_t dst_pitch, const void* src, int64_t src_pitch, int64_t width_bytes,
                    int64_t rows, void* stream);

/*
 * The W4A4 linear in one call that allocates nothing: convrot_prepare_i8
 * followed by convrot_w4a4_gemm, with the int8 codes and row scales between
 * them kept in a fixed device array inside the library instead of a buffer
 * from the caller.  It is for callers that cannot allocate device memory: a
 * plugin that its host engine hands only input and output buffers, or code
 * whose host framework reserves the device's memory for its own allocator.
 * No counterpart in the reference (there the framework allocates).
 *   - The array holds CONVROT_LINEAR_STATIC_SCRATCH_BYTES: the codes of
 *     m x k (rounded up to 256 bytes) plus 4 * m bytes of scales must fit
 *     (m x k up to about 67 million), else CONVROT_ERR_UNSUPPORTED.  Every
 *     GPU that loads the library holds the array until the process exits.
 *   - The first call on a device looks up the array's device address on
 *     that device; made while `stream` is capturing, it is refused with
 *     CONVROT_ERR_UNSUPPORTED (make one call outside capture first).
 *   - Every argument check of convrot_w4a4_gemm runs before anything is
 *     enqueued: a rejected call touches neither the GPU nor the array.
 *   - All calls share the one array: calls whose work overlaps on the GPU
 *     (different streams, or other host threads) race and must not overlap.
 *     Every call rewrites all of the array it reads, so nothing from an
 *     earlier call carries over.
 * Arguments as convrot_prepare_i8 (x, x_dtype, group_size) and
 * convrot_w4a4_gemm (qweight ... stream).
 */
#define CONVROT_LINEAR_STATIC_SCRATCH_BYTES (64LL << 20)
int convrot_w4a4_linear_static(const void* x, int x_dtype, int group_size,
                               const uint8_t* qweight, int layout, const float* wscales,
                               const float* bias, void* out, int out_dtype, int64_t m, int64_t n,
                               int64_t k, void* stream);

/*
 * Diagnostics: which kernel convrot_w4a4_gemm runs.  route 0 (the default):
 * the register-fragment GEMV kernel for m <= 8 (K x packed-N with n % 16 ==
 * 0, or N x packed-K), else the swap-AB kernel for m <= 8 (k % 128 == 0;
 * K x packed-N with n % 32 == 0), else the CTA-pair kernel where it applies
 * (k % 128 == 0; K x packed-N with n % 32 == 0), else the one-CTA kernel;
 * route 1: the one-CTA kernel
 * for every shape; route 2: the CTA-pair kernel wherever it applies (never
 * a small-m one); route 3: the swap-AB kernel wherever it applies (m <=
 * 64); route 4: the register-fragment GEMV kernel wherever it applies
 * (m <= 8; K x packed-N with n % 16 == 0, or N x packed-K).  All give the
 * same bits.  Process-wide; for tests and A/B timing.  No reference
 * counterpart.
 */
int convrot_set_gemm_route(int route);

/*
 * Diagnostics: every wait inside the tcgen05 kernels is bounded; a kernel
 * whose wait times out stops early and records a non-zero code in a
 * device-side word.  This reads and clears that word (0 = no time-out).  It
 * synchronizes the current device.  No reference counterpart (the reference
 * has no failure detection beyond shape checks).  Codes (the first recorded
 * wins): 1-7 one-CTA W4A4 GEMM; 11-19 CTA-pair GEMM (11/12 copy slot free
 * for A / packed weights, 13 accumulator buffer free, 14 A stage landed,
 * 15 expanded weights ready, 16 final MMA drain, 17 packed weights landed,
 * 18 expanded-weight slot free, 19 accumulator ready); 31 peer flag barrier;
 * 41 staged prep row copy; 51-57 swap-AB small-m GEMM (51 packed-weight
 * slot free, 52 activation stage landed, 53 expanded weights ready, 54
 * packed weights landed, 55 expanded-weight slot free, 56 final MMA drain,
 * 57 activation slot free); 61-65 8-bit pair GEMM (61 copy slot free, 62
 * accumulator buffer free, 63 stage landed, 64 final MMA drain, 65
 * accumulator ready); 71-74 8-bit swap GEMM (71 copy slot free, 72 weight
 * stage landed, 73 activation stage landed, 74 final MMA drain); 81-87 8-bit
 * float pair GEMM (81 copy slot free, 82 accumulator free, 83 stage with its
 * scales landed, 85 accumulator ready, 86 scale slot free, 87 final MMA drain);
 * 91-96 8-bit float
 * swap GEMM (91 copy slot free, 92 weight stage landed, 93 activation stage
 * landed, 94 final MMA drain, 95 scale slot free, 96 scales landed).
 */
int convrot_take_device_error(int* code);

/*
 * 8-bit row quantizer: for each row, top = max |v|, scale = top / 127 and
 * codes rne(127 v / top) in [-127, 127], with v = x, or the float32 product
 * x[r, c] * col_scale[c] when col_scale is not NULL (the gradient of the
 * 8-bit linear folds its weight scales in).  A zero row has codes 0 and scale
 * 0; a row that holds an infinity or a NaN has codes 0 and scale NaN, so that
 * what is computed from it is NaN.  Row r of x starts at r * x_stride
 * elements, of the codes at r * q_stride bytes.  No reference counterpart
 * (the 4-bit form is convrot_prepare_packed with group_size 1).
 */
int convrot_quantize_i8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride,
                        const float* col_scale, int8_t* q, int64_t q_stride, float* scales, void* stream);

/*
 * 8-bit linear: out[i, j] = T(fl(fl(fl(dot[i, j]) * xscales[i]) * wscales[j])
 * + bias[j]) with dot[i, j] = sum over k of act[i, k] w[j, k], exact in int32
 * (k <= 131072; tcgen05 kind::i8).  act: (m, k) int8 codes, row i at
 * i * act_stride bytes.  weight: int8, layout CONVROT_LAYOUT_NK = (n, k) rows
 * or CONVROT_LAYOUT_KN = (k, n) rows (the same matrix contracted over its
 * rows: the gradient of the input), row r at r * weight_stride bytes.
 * Strides are multiples of 16 and cover the rows; m and n are below 2^22.
 * wscales and bias may be NULL (ones, zeros).  Codes are in [-127, 127].  No
 * reference counterpart.
 */
int convrot_i8_gemm(const int8_t* act, int64_t act_stride, const int8_t* weight, int64_t weight_stride, int layout,
                    const float* xscales, const float* wscales, const float* bias, void* out, int out_dtype,
                    int64_t m, int64_t n, int64_t k, void* stream);

/*
 * convrot_quantize_i8 of x, then convrot_i8_gemm of its codes, in one call:
 * the 8-bit linear (layout NK), or with col_scale and layout KN the gradient
 * of its input.  `codes` (m, k) and `scales` (m,) are workspace; what they hold
 * afterwards is not specified (for one or two tokens the product forms the
 * codes itself).  The product starts reading the weight while the quantizer
 * runs: `codes` and `scales` may not overlap the weight.
 */
int convrot_i8_linear(const void* x, int x_dtype, int64_t x_stride, const float* col_scale, const int8_t* weight,
                      int64_t weight_stride, int layout, const float* wscales, const float* bias, void* out,
                      int out_dtype, int64_t m, int64_t n, int64_t k, int8_t* codes, int64_t codes_stride,
                      float* scales, void* stream);

/*
 * Rotary positions with several axes for queries and keys, in one launch.
 * Tensors are (batch, heads, tokens, dim), dim <= 256, with unit stride along
 * dim; strides: host array of the element strides {batch, head, token} of q,
 * q_out, k and k_out in this order.  k_heads (or q_heads) may be 0.  The first sum(widths) values of a head are pairs, adjacent
 * (interleaved) or sum(widths) / 2 apart; pair j of axis a turns by
 * positions[token, a] * theta^(-2 j / widths[a]); the rest is copied.
 * inverse turns back: the gradient of the input from that of the output.
 * positions: (tokens, axes) float32, that of sample b at b *
 * position_batch_stride elements (0: shared).  widths: host array, positive
 * and even.  Outputs may not overlap inputs, except that each may be exactly
 * its own input.  No reference counterpart.
 */
int convrot_axial_rotary(int dtype, int64_t batch, int64_t tokens, int64_t dim, const void* q, void* q_out,
                         int64_t q_heads, const void* k, void* k_out, int64_t k_heads, const int64_t* strides,
                         const float* positions, int64_t position_batch_stride, int axes, const int32_t* widths,
                         double theta, int interleaved, int inverse, void* stream);

/*
 * Layer norm of the rows of x (rows, features), packed, features <= 2^20:
 * y = (x - mean) * rsqrt(var + eps) * w + bias in float32, one rounding; w =
 * weight, or 1 + weight with add_one.  Rows r with the same r /
 * rows_per_weight share a weight and a bias vector, at weight_stride elements
 * from one another: all rows (affine norm), or those of a sample (modulated
 * norm), of which there are at most 65535.  weight_dtype: that of x, or
 * CONVROT_F32.  weight and bias may be NULL (w = 1, bias 0).  mean and rstd:
 * (rows,) float32 for the backward pass, or both NULL.  No reference
 * counterpart.
 */
int convrot_layer_norm(const void* x, int dtype, int64_t rows, int64_t features, const void* weight,
                       const void* bias, int weight_dtype, int64_t rows_per_weight, int64_t weight_stride,
                       int add_one, float eps, void* y, float* mean, float* rstd, void* stream);

/*
 * Gradients of convrot_layer_norm: dx (rows, features) of x's dtype, and the
 * sums over the rows that share a weight, dweight = sum dy h and dbias = sum
 * dy with h the normalized row, (rows / rows_per_weight, features) packed, of
 * weight_dtype, either NULL when not wanted.  Sums are float32, in an order
 * fixed by the shape, the types, the addresses' alignment and the number of
 * SMs (no atomics).  mean, rstd: from the forward pass.  workspace:
 * convrot_layer_norm_workspace bytes, 16-byte aligned (not used when neither
 * sum is wanted).  With 0 rows nothing is written.
 */
int64_t convrot_layer_norm_workspace(int64_t rows, int64_t features, int64_t rows_per_weight);
int convrot_layer_norm_backward(const void* x, const void* dy, int dtype, int64_t rows, int64_t features,
                                const void* weight, int weight_dtype, int64_t rows_per_weight,
                                int64_t weight_stride, int add_one, const float* mean, const float* rstd, void* dx,
                                void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Tanh GELU whose input is saved in 8 bits for the backward pass.  Forward:
 * y = gelu_tanh(x) (rows, features), and the codes (rows, features) int8 with
 * scales (rows, ceil(features / 128)) float32 of x in groups of 128 features,
 * as convrot_quantize_i8 forms them; codes and scales may both be NULL (no
 * backward pass wanted).  Backward: dx = dy * gelu_tanh'(codes * scale).  All
 * packed; y, dy and dx have x's dtype.  No reference counterpart.
 */
int convrot_gelu_saved8(const void* x, int dtype, int64_t rows, int64_t features, void* y, int8_t* codes,
                        float* scales, void* stream);
int convrot_gelu_saved8_backward(const void* dy, int dtype, int64_t rows, int64_t features, const int8_t* codes,
                                 const float* scales, void* dx, void* stream);

/*
 * Quantizers of the 8-bit floating-point linear: e4m3 codes and one scale 2^e
 * for each block of 128 consecutive values of a row (convrot_quantize_fp8), or
 * for each block of 128 x 128 (convrot_quantize_fp8_weight), with e the least
 * exponent, at least -127, for which max|x| <= 448 * 2^e, stored as the byte
 * e + 127; code = e4m3(x * 2^-e), to nearest even.  A block of zeros has codes
 * and byte 0; one that holds an infinity or a NaN has codes 0 and byte 255,
 * which stands for NaN.  Blocks at the ends of rows (and of the rows) are of
 * what is there.  Row r of x starts at r * x_stride elements, of the codes at
 * r * codes_stride bytes (a multiple of 16; the bytes of a row past its
 * features up to a multiple of 16 are overwritten), of the scales at r *
 * scales_stride (or r / 128 times it).  No reference counterpart.
 */
int convrot_quantize_fp8(const void* x, int dtype, int64_t rows, int64_t features, int64_t x_stride, uint8_t* codes,
                         int64_t codes_stride, uint8_t* scales, int64_t scales_stride, void* stream);
int convrot_quantize_fp8_weight(const void* w, int dtype, int64_t rows, int64_t features, int64_t w_stride,
                                uint8_t* codes, int64_t codes_stride, uint8_t* scales, int64_t scales_stride,
                                void* stream);

/*
 * 8-bit floating-point linear: out[i, j] = T(sum over blocks b of 128 of k of
 * xscale[i, b] * wscale[j / 128, b] * sum over k in b of act[i, k] w[j, k], +
 * bias[j]), sums in float32 (tcgen05 kind::mxf8f6f4).  act: (m, k) e4m3 codes
 * with scales (m, ceil(k / 128)), rows of scales at multiples of 4 bytes.
 * weight: e4m3, layout CONVROT_LAYOUT_NK = (n, k) rows or CONVROT_LAYOUT_KN =
 * (k, n) rows (the same matrix contracted over its rows: the gradient of the
 * input); wscales: one byte for each 128 x 128 block of the matrix as it
 * lies, rows of them at wscales_stride bytes.  Scales are the bytes of the
 * quantizers above.  Row strides of codes are multiples of 16 and cover the
 * rows, and the rows are read in whole 16 bytes, the last one too (what is
 * behind its end is not used); m, n and k are below 2^22.  bias may be NULL (zeros).  A float32
 * output over more than 8192 k is summed in ranges of that many, one launch
 * after another, except where up to 8 tokens of layout NK fit one launch that
 * adds up blocks.  The order of the sums is fixed by the shape, the layout and the
 * number of SMs.  No reference counterpart.
 */
int convrot_fp8_gemm(const uint8_t* act, int64_t act_stride, const uint8_t* xscales, int64_t xscales_stride,
                     const uint8_t* weight, int64_t weight_stride, int layout, const uint8_t* wscales,
                     int64_t wscales_stride, const float* bias, void* out, int out_dtype, int64_t m, int64_t n,
                     int64_t k, void* stream);

/*
 * convrot_quantize_fp8 of x, then convrot_fp8_gemm of its codes, in one call.
 * `codes` (m, k) and `scales` (m, ceil(k / 128), rows at multiples of 4 bytes)
 * are workspace; what they hold afterwards is not specified.  The product
 * starts reading the weight while the quantizer runs: the workspace may not
 * overlap the weight.
 */
int convrot_fp8_linear(const void* x, int x_dtype, int64_t x_stride, const uint8_t* weight, int64_t weight_stride,
                       int layout, const uint8_t* wscales, int64_t wscales_stride, const float* bias, void* out,
                       int out_dtype, int64_t m, int64_t n, int64_t k, uint8_t* codes, int64_t codes_stride,
                       uint8_t* scales, int64_t scales_stride, void* stream);

/*
 * Sums of squares of many tensors of one dtype, for their norm.  `tensors` is
 * a host array.  Writes `sums_count` partial sums (float64) that add up to the
 * total; convrot_square_sums_count gives a good number of them for these
 * tensors.  Which values a sum holds depends on the sizes and sums_count alone.
 * convrot_norm_of_sums: sqrt of the total of sums (of several dtypes, one
 * after another in memory) as float32.  With `norm` not NULL (at most 8 sums of at
 * most 1024 tensors) convrot_square_sums writes the norm itself and no sums,
 * which may then be NULL.  No reference counterpart.
 */
typedef struct {
  const void* grad;
  int64_t numel;
} convrot_grad_tensor;
int64_t convrot_square_sums_count(int64_t count, const convrot_grad_tensor* tensors);
int convrot_square_sums(int64_t count, const convrot_grad_tensor* tensors, int dtype, double* sums,
                        int64_t sums_count, float* norm, void* stream);
int convrot_norm_of_sums(const double* sums, int64_t sums_count, float* norm, void* stream);

/*
 * One AdamW step (decoupled weight decay) over many tensors of one dtype, in
 * one launch for each 512 of them; `tensors` is a host array.  state_bits 32:
 * exp_avg and exp_avg_sq are float32 (m and v).  state_bits 8: they are e4m3
 * codes of m and of sqrt(v), and scales holds {scale of m, scale of sqrt(v)}
 * for each 256 values of the tensor, float32; codes are rounded to nearest, which
 * roots follow their averages with for beta2 up to 0.95; a block that is not
 * finite gets scales NaN.  Values are taken in memory order, so a tensor and its moments
 * have to be laid out alike.  step counts from 1; step_device and lr_device, where not NULL, are
 * one float32 each on the device and take the place of step and lr (for a
 * captured step).  With sums (of convrot_square_sums) gradients are scaled by
 * min(1, max_norm / (norm + 1e-6)) as they are read, and the norm is written
 * to `norm` if that is not NULL.  Gradients are not written.  No tensor may overlap
 * another.  No reference counterpart.
 */
typedef struct {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* scales;
  int64_t numel;
} convrot_adamw_tensor;
typedef struct {
  double step, lr, beta1, beta2, eps, weight_decay;
  const float* step_device;
  const float* lr_device;
  const double* sums;
  int64_t sums_count;
  double max_norm;
  float* norm;
} convrot_adamw_options;
int convrot_adamw(int64_t count, const convrot_adamw_tensor* tensors, int dtype, int state_bits,
                  const convrot_adamw_options* options, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CONVROT_B200_H */
