/*
 * tilec.h — C ABI of libtilec_hip.so, the MI355X (gfx950) implementation of
 * tilec's matmul op.
 *
 * The reference crosses its host→device boundary in one place: the launch of
 * the tile kernel `_matmul_tiled[(cdiv(M,BM), cdiv(N,BN))](a, b, c, M, N, K,
 * BM=, BN=, BK=)` issued by `_matrix_mul_tiled` (tilec/ext.py:54-63), which
 * goes through `JITFunction.run` / `_launch` (tilec/jit.py:81-105) into
 * `torch.mps.compile_shader(...)(*buffers, threads=..., group_size=...)`.
 * Every entry point below replaces a piece of that path; the Python caller is
 * tilec/ext.py (via ctypes), which keeps the reference's public signature
 * `matrix_mul(x1, x2)` (tilec/ext.py:66-67).
 *
 * Conventions shared by all entry points
 *   - The output is row-major with unit column stride; ldo is its row stride
 *     in elements (>= N).  Each input is row-major (ld* = row stride >= its
 *     number of columns) or, when its `layout` bit is set, column-major
 *     (ld* = column stride >= its number of rows) — the transposed view
 *     x.T of a contiguous matrix, read in place.  The reference makes every
 *     input row-major contiguous first (`.contiguous()`, tilec/ext.py:59-60;
 *     then ld == the number of columns); strided and transposed views skip
 *     that copy here.
 *   - Outputs of products and sums are float32 (the training operators say
 *     their own types).  Inputs are float32, or bfloat16 (fp32 accumulate).
 *   - Nothing here allocates device memory, synchronizes, or reads the device
 *     back: work is enqueued on `stream` (a hipStream_t; NULL = the legacy
 *     default stream) and returns at once, like the reference's asynchronous
 *     MPS launch (tilec/jit.py:105).
 *   - Functions return a status code (TILEC_OK == 0).  On failure
 *     tilec_last_error() returns a message for the calling thread.  The Python
 *     caller maps TILEC_ERR_VALUE to ValueError (the reference's shape error,
 *     tilec/ext.py:57-58), TILEC_ERR_TYPE to TypeError (tilec/jit.py:34-39)
 *     and the rest to RuntimeError.
 */
#ifndef TILEC_H
#define TILEC_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes. */
#define TILEC_OK 0
#define TILEC_ERR_VALUE 1       /* bad shape, stride, pointer or split   */
#define TILEC_ERR_TYPE 2        /* unsupported dtype                      */
#define TILEC_ERR_UNSUPPORTED 3 /* variant unknown or not valid for shape */
#define TILEC_ERR_WORKSPACE 4   /* workspace missing or too small         */
#define TILEC_ERR_HIP 5         /* HIP runtime error at launch            */

/* Element types (the output of a product or a sum is always float32). */
#define TILEC_F32 0
#define TILEC_BF16 1
/* 8-bit floating point, for operands with scales (below). */
#define TILEC_F8E4M3 2 /* 4 bits of exponent, largest 448, no infinities */
#define TILEC_F8E5M2 3 /* 5 bits of exponent, largest 57344              */

/* Kernel families (tilec_variant_info, info[0]). */
#define TILEC_FAMILY_SKINNY 0 /* output-stationary streaming kernel, split K:   */
                              /* M <= 16, or outputs of few 64x64 tiles         */
#define TILEC_FAMILY_GEMM 1   /* LDS-staged MFMA tile GEMM                      */
#define TILEC_FAMILY_DIRECT 2 /* fp32 MFMA on operands loaded straight into     */
                              /* registers, split K: GEMV and small outputs     */

/* Operand layouts: bits of tilec_matmul's `layout` (0 = both row-major). */
#define TILEC_X1_COL_MAJOR 1 /* x1 element (m, k) at x1[m + k * ldx1], ldx1 >= M */
#define TILEC_X2_COL_MAJOR 2 /* x2 element (k, n) at x2[k + n * ldx2], ldx2 >= K */

/* Pass as `variant` to let the library pick with its built-in rule. */
#define TILEC_VARIANT_AUTO (-1)

/*
 * out[M,N] = x1[M,K] · x2[K,N]
 *
 * Replaces the launch `_matmul_tiled[grid](x1, x2, out, M, N, K, BM, BN, BK)`
 * (tilec/ext.py:62; kernel semantics tilec/ext.py:13-24; launch
 * tilec/jit.py:88-105).  `variant` selects a compiled kernel (see
 * tilec_num_variants / tilec_variant_info) the way the reference's constexpr
 * tile sizes select a compiled specialization (tilec/jit.py:66-76);
 * `split_k` (0 = automatic) splits the reduction dimension across
 * workgroups, the role of the legacy `split` config (tilec/ext.py:37,48-51).
 *
 * `layout` (TILEC_X1_COL_MAJOR | TILEC_X2_COL_MAJOR) says how x1 and x2 are
 * stored; every variant takes every layout.  The reference has no such
 * argument: it copies each input to row-major first (tilec/ext.py:59-60).
 *
 * M == 0 or N == 0 enqueues nothing.  K == 0 writes zeros (the reference's
 * accumulator starts at zero and its K loop runs no iterations).
 *
 * A split K needs two device buffers (NULL/0 when their size is 0):
 *   `workspace` — tilec_matmul_workspace_bytes(...) bytes of scratch for the
 *                 partial sums; any contents;
 *   `counters`  — tilec_matmul_counter_bytes(...) bytes of completion
 *                 counters that must be zero before the call.  Every call
 *                 that completes leaves them zero again, so a buffer zeroed
 *                 once at allocation serves all later calls on one stream,
 *                 whatever their shapes, as long as it is large enough.
 * Calls that run concurrently (different streams) need their own buffers.
 */
int tilec_matmul(const void* x1, const void* x2, float* out,
                 int64_t M, int64_t N, int64_t K,
                 int64_t ldx1, int64_t ldx2, int64_t ldo, int32_t layout,
                 int32_t dtype, int32_t variant, int32_t split_k,
                 void* workspace, size_t workspace_bytes,
                 void* counters, size_t counter_bytes, void* stream);

/*
 * Bytes of scratch (`workspace`) tilec_matmul needs for these arguments
 * with both operands row-major and contiguous (0 if none).  For a named
 * variant the size is the same for every layout; TILEC_VARIANT_AUTO may pick
 * another variant for another layout or stride, which
 * tilec_matmul_scratch_bytes accounts for.  Replaces nothing in the
 * reference (its kernel needs no scratch); the caller allocates it the way
 * `_matrix_mul_tiled` allocates `out` (tilec/ext.py:61).
 */
size_t tilec_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K,
                                    int32_t dtype, int32_t variant,
                                    int32_t split_k);

/* Bytes of zero-initialised completion counters (`counters`) it needs. */
size_t tilec_matmul_counter_bytes(int64_t M, int64_t N, int64_t K,
                                  int32_t dtype, int32_t variant,
                                  int32_t split_k);

/*
 * Both scratch sizes for exactly the arguments tilec_matmul gets (layout
 * bits and strides included; ldx1 / ldx2 <= 0: contiguous), so that
 * TILEC_VARIANT_AUTO is resolved as the call will resolve it.  Returns
 * TILEC_OK, or the status tilec_matmul would return for an argument it
 * rejects (sizes are then 0).  Like the two queries above it replaces
 * nothing in the reference; it cannot see pointers, so for the row-dot and
 * row-tile variants it counts the scratch of their streaming fallback.
 */
int tilec_matmul_scratch_bytes(int64_t M, int64_t N, int64_t K,
                               int64_t ldx1, int64_t ldx2, int32_t layout,
                               int32_t dtype, int32_t variant, int32_t split_k,
                               size_t* workspace_bytes, size_t* counter_bytes);

/*
 * tilec_matmul without the caller's scratch: for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid allocation).  No counterpart in the reference, whose
 * kernel needs no scratch.  Same arguments, semantics and status codes as
 * tilec_matmul, minus the four buffer arguments.
 *
 * A split K uses a static array of the library on the current device: at
 * most 16 MiB of partial sums and 1 MiB of counters (each GPU the library
 * runs on holds 17 MiB until the process ends).  A call that needs more
 * (tilec_matmul_scratch_bytes for the same arguments) fails with
 * TILEC_ERR_WORKSPACE before anything is enqueued; use tilec_matmul then.
 * The first call on a device looks the array up and enqueues a small kernel
 * that clears its counters.  Nothing is allocated.
 *
 * Every call on one GPU shares that GPU's array and leaves its counters at
 * zero: calls that overlap on one GPU (concurrent streams, host threads)
 * race and must be serialized by the caller.
 */
int tilec_matmul_noalloc(const void* x1, const void* x2, float* out,
                         int64_t M, int64_t N, int64_t K,
                         int64_t ldx1, int64_t ldx2, int64_t ldo, int32_t layout,
                         int32_t dtype, int32_t variant, int32_t split_k,
                         void* stream);

/*
 * The variant the library's built-in rule picks for a shape with both
 * operands row-major and contiguous (what TILEC_VARIANT_AUTO runs for layout
 * 0), or a negative status.  The reference's equivalent is the fixed
 * BM=BN=64, BK=16 default of `_matrix_mul_tiled` (tilec/ext.py:54); the
 * trained per-shape choice lives host-side in tilec/tune.py, as
 * `tune.pick` does in the reference (tilec/tune.py:143-151).
 */
int32_t tilec_select_variant(int64_t M, int64_t N, int64_t K, int32_t dtype);

/*
 * The same for any layout and strides (ldx1 / ldx2 <= 0: contiguous): what
 * TILEC_VARIANT_AUTO runs for tilec_matmul with these arguments (x @ W.T,
 * for instance, takes the row-dot or row-tile kernels).  No counterpart in
 * the reference, whose operands are always made contiguous
 * (tilec/ext.py:59-60).
 */
int32_t tilec_select_variant_layout(int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t layout,
                                    int64_t ldx1, int64_t ldx2);

/* The split_k that split_k == 0 resolves to for this variant and shape. */
int32_t tilec_auto_split_k(int64_t M, int64_t N, int64_t K, int32_t dtype,
                           int32_t variant);

/*
 * Variant enumeration, for the tuner (the reference enumerates its config
 * space in Python: `mm_configs`, tilec/ext.py:48-51).
 *   info[0] family (TILEC_FAMILY_*)  info[1] dtype (TILEC_F32/BF16)
 *   info[2] BM     info[3] BN        info[4] BK
 *   info[5] waves per workgroup      info[6] max M (0 = unbounded)
 *   info[7] unroll / pipeline depth
 * `name` (may be NULL) receives a static string.
 */
int32_t tilec_num_variants(void);
int tilec_variant_info(int32_t variant, int32_t info[8], const char** name);

/*
 * Row or column sums of a matrix, fp32 accumulate, fp32 out:
 *   axis 1:  out[r] = sum_c x[r][c]   (R outputs)
 *   axis 0:  out[c] = sum_r x[r][c]   (C outputs)
 * x is R x C, float32 or bfloat16, row-major with row stride ldx (>= C), or
 * column-major when `layout` is TILEC_X1_COL_MAJOR (column stride ldx >= R).
 * A sum over zero elements is 0.
 *
 * The reduction the reference plans as `tl.sum` (README.md:88) and shows as
 * the `row_sum` kernel (kernel1.py:8-15: out[r] = tl.sum(x[r, :]); the
 * op-level spelling `tl.ext.sum(x_ptr, axis=1)` at kernel1.py:15).  Long
 * reductions with few outputs are split across workgroups and combined in
 * a fixed order, so results do not depend on scheduling; they need the
 * `workspace` and zeroed `counters` that tilec_sum_workspace_bytes /
 * tilec_sum_counter_bytes give (0 when not split), under the same rules as
 * tilec_matmul's (counters are left zero; concurrent calls need their own).
 */
int tilec_sum(const void* x, float* out, int64_t R, int64_t C, int64_t ldx,
              int32_t layout, int32_t dtype, int32_t axis,
              void* workspace, size_t workspace_bytes,
              void* counters, size_t counter_bytes, void* stream);
size_t tilec_sum_workspace_bytes(int64_t R, int64_t C, int32_t layout,
                                 int32_t dtype, int32_t axis);
size_t tilec_sum_counter_bytes(int64_t R, int64_t C, int32_t layout,
                               int32_t dtype, int32_t axis);

/*
 * The HBM read floor, a measurement aid with no counterpart in the
 * reference: one pass over `bytes` of x (a multiple of 16 KiB, 16-byte
 * aligned), in the order the GEMV kernels are measured against —
 * `workgroups` workgroups (<= 0: two per CU; at most one per 16 KiB piece)
 * read the 16 KiB pieces g, g + G, g + 2G, ... with non-temporal 16-byte
 * loads (four waves per workgroup), so the chip reads one moving window.
 * Wave w of workgroup g writes the fp32 sum of the floats it read to
 * sink[4 g + w] (the caller provides four floats per workgroup); nothing is
 * combined across workgroups.  Asynchronous on `stream`, allocates nothing.
 */
int tilec_read_floor(const void* x, size_t bytes, float* sink, int32_t workgroups, void* stream);

/*
 * Training operators.  The reference has none; they are what a training step
 * needs beside its products (tilec_matmul) and sums (tilec_sum), under the
 * same conventions: asynchronous on `stream`, nothing allocated, a status
 * code, caller-owned scratch.
 */

/*
 * Layer norm over the rows of x [R, D], D >= 1:
 *   y = (x - mean) rstd weight + bias,   rstd = 1 / sqrt(var + eps)
 * with var the mean of the squared deviations.  x and y are float32 or
 * bfloat16, each with its own dtype code and row stride (>= D elements, any
 * alignment of the element); weight and bias [D], contiguous, share w_dtype
 * and may each be NULL (1 and 0).  mean and rstd [R], float32, are written
 * where not NULL.  Statistics are float32.  y may be x (same dtype and
 * stride); otherwise outputs must not overlap inputs.
 */
int tilec_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd,
                     int64_t R, int64_t D, int64_t ldx, int64_t ldy, int32_t x_dtype, int32_t y_dtype,
                     int32_t w_dtype, float eps, void* stream);

/*
 * Its gradients, from the mean and rstd [R] of the forward pass:
 *   dx = rstd (dy weight - c1 - xhat c2),  c1 = mean(dy weight),  c2 = mean(dy weight xhat)
 *   dweight = sum over rows of dy xhat,    dbias = sum over rows of dy
 * dy and dx have y_dtype; dweight and dbias [D] are float32 and may each be
 * NULL.  Column sums are added in a fixed order: the same bits on every call
 * on one device.  `workspace`: tilec_layer_norm_backward_workspace_bytes, any
 * contents; 16-byte aligned.  dx may be dy.
 */
int tilec_layer_norm_backward(const void* dy, const void* x, const float* mean, const float* rstd,
                              const void* weight, void* dx, float* dweight, float* dbias,
                              int64_t R, int64_t D, int64_t lddy, int64_t ldx, int64_t lddx,
                              int32_t x_dtype, int32_t y_dtype, int32_t w_dtype,
                              void* workspace, size_t workspace_bytes, void* stream);
size_t tilec_layer_norm_backward_workspace_bytes(int64_t R, int64_t D, int32_t x_dtype);

/*
 * Cross entropy of logits = x weight^T, which are not given out: x [N, H],
 * weight [V, H] (both float32 or both bfloat16, row-major with row strides ldx,
 * ldw >= H), target [N] int64.
 *   loss_r = log(sum_v exp(logits[r, v])) - logits[r, target_r]
 * float32: `loss` [N] with TILEC_REDUCE_NONE, else one value, the sum or the
 * mean over the rows that count.  Rows whose target is ignore_index do not:
 * their loss and gradients are 0 whatever x holds there and whatever grad_loss
 * is (dx of float32 inputs: where weight is finite), and a mean over no rows is
 * 0.  A target that is neither that nor a class in [0, V) makes its
 * loss, and every gradient it reaches, NaN.
 *
 * grad != 0 also writes the gradients dx [N, H] and dweight [V, H],
 * contiguous, of x's type, of
 *   TILEC_REDUCE_NONE:       sum_r grad_loss[r] loss_r  (grad_loss [N] float32, NULL: ones)
 *   TILEC_REDUCE_SUM, _MEAN: grad_loss[0] loss          (one float32 on the device, NULL: 1)
 * Rows are worked through in chunks of chunk_rows (0: as many as keep the
 * chunk's values, one per row and class, within 2 GiB); more than one chunk
 * adds a float32 [V, H] to the workspace.  Those values are 16-bit ones that
 * gradients of bfloat16 inputs need, or the float32 logits of float32 inputs,
 * losses alone included; losses alone of bfloat16 inputs keep 8 bytes per row
 * and 64 classes.
 *
 * tilec_linear_ce_scratch_bytes gives the workspace (any contents, 16-byte
 * aligned) and counters (zeroed once, left zero) for exactly these arguments;
 * of x and weight it reads the addresses' alignment only.  rows_per_chunk
 * (may be NULL) receives the rows of a chunk.  Every sum is float32 or wider,
 * in a fixed order.
 *
 * configs (float32 only; NULL: the built-in rule): the variant and split_k, as
 * tilec_matmul takes them, of a whole chunk's three products: the logits
 * (chunk rows x V, K = H, x2 column-major), dx (chunk rows x H, K = V) and
 * dweight (V x H, K = chunk rows, x1 column-major).
 */
#define TILEC_REDUCE_NONE 0
#define TILEC_REDUCE_SUM 1
#define TILEC_REDUCE_MEAN 2
int tilec_linear_ce(const void* x, const void* weight, const int64_t* target, float* loss,
                    const float* grad_loss, void* dx, void* dweight, int64_t N, int64_t H, int64_t V,
                    int64_t ldx, int64_t ldw, int32_t dtype, int32_t reduction, int64_t ignore_index,
                    int32_t grad, int64_t chunk_rows, const int32_t* configs,
                    void* workspace, size_t workspace_bytes, void* counters, size_t counter_bytes, void* stream);
int tilec_linear_ce_scratch_bytes(const void* x, const void* weight, int64_t N, int64_t H, int64_t V,
                                  int64_t ldx, int64_t ldw, int32_t dtype, int32_t reduction, int32_t grad,
                                  int64_t chunk_rows, const int32_t* configs, size_t* workspace_bytes,
                                  size_t* counter_bytes, int64_t* rows_per_chunk);

/*
 * One AdamW step over `count` tensors, in place:
 *   g = grad * grad_scale;  p = p (1 - lr weight_decay)
 *   m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   p = p - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)
 * with `step` counted from 1 and grad_scale one float32 on the device (NULL:
 * 1).  `step` and the other numbers are read on the host: a HIP graph repeats
 * those it was recorded with.  The descriptions in `tensors` (host memory) are
 * read before the call returns.  Every tensor is contiguous, of n elements, at any alignment of
 * its element type; no two of them may overlap.
 *
 * state_bits 32: exp_avg and exp_avg_sq are float32 [n].  state_bits 8: they
 * are codes, int8 and uint8 [n], with one float32 scale per 256 consecutive
 * elements (ceil(n / 256) of them), the block's largest magnitude:
 *   m = sign(c) (c / 127)^2 scale        v = (c / 255)^4 scale
 * Zero codes and scales are zero states.
 */
typedef struct tilec_adamw_tensor {
  void* param;              /* float32 or bfloat16 [n], read and written     */
  const void* grad;         /* float32 or bfloat16 [n]                       */
  void* exp_avg;            /* m                                             */
  void* exp_avg_sq;         /* v                                             */
  float* exp_avg_scale;     /* state_bits 8                                  */
  float* exp_avg_sq_scale;  /* state_bits 8                                  */
  void* copy;               /* bfloat16 [n] that gets the new param, or NULL */
  int64_t n;
  int32_t param_dtype, grad_dtype;
} tilec_adamw_tensor;
int tilec_adamw(const tilec_adamw_tensor* tensors, int32_t count, int32_t state_bits, int64_t step, double lr,
                double beta1, double beta2, double eps, double weight_decay, const float* grad_scale, void* stream);

/*
 * The float32 values that 8-bit states stand for, into `param` [n] of each
 * description: of exp_avg with its scales, or, where exp_avg is NULL, of
 * exp_avg_sq.
 */
int tilec_adamw_values(const tilec_adamw_tensor* tensors, int32_t count, void* stream);

/*
 * Operators of 8-bit linear layers.  An 8-bit operand is a matrix of codes
 * [R, C] (TILEC_F8E4M3 or TILEC_F8E5M2, row-major, row stride >= C) and float32
 * scales of its blocks of `block` x 128 values, block 1 or 128:
 *   value[r, c] = code[r, c] * scale[r / block, c / 128]
 * The scales [ceil(R / block), ceil(C / 128)] have strides of their own, *_row and
 * *_group elements (in a product *_row <= 2^21); a matrix's last blocks may be
 * smaller.
 *
 * out [M, N] = x weight^T over the values, x [M, K], weight [N, K]:
 *   out[m, n] = sum_g scale_x[m, g] scale_w[n, g] sum over k of group g of x[m, k] weight[n, k]
 * out is float32 or bfloat16 with row stride ldo >= N.  The sums over groups are
 * float32.  For a float32 out so are those within a group, of exact products;
 * for a bfloat16 out they are the 8-bit matrix instructions', which cut every
 * product at 2^-13 of the largest among eight consecutive k (1.5e-5 of the result
 * for normal values).  The product of two scales is a float32 of its own, formed
 * before it multiplies a group's sum: rounded, below 2^-126 to multiples of 2^-149
 * (0 below 2^-150), and infinite from 2^128 on.  The same bits on every call on one
 * device.  K <= 2^22; K == 0 writes zeros.
 *
 * Operands are read in place where their rows begin at multiples of 16 bytes,
 * and otherwise copied into the workspace first; scales of rows are read fastest
 * with a row stride of 1 (8192^3: 2 %).  tilec_linear_fp8_scratch_bytes says for
 * the same arguments (of x and weight it reads the addresses' alignment only) how
 * much `workspace` (any contents, 16-byte aligned) and `counters` (4-byte aligned,
 * zero before the call and left zero) it takes; concurrent calls need their own.
 */
int tilec_linear_fp8(const void* x, const float* x_scale, const void* weight, const float* w_scale, void* out,
                     int64_t M, int64_t N, int64_t K, int64_t ldx, int64_t ldw, int64_t ldo, int64_t x_scale_row,
                     int64_t x_scale_group, int64_t w_scale_row, int64_t w_scale_group, int32_t x_dtype, int32_t w_dtype,
                     int32_t out_dtype, int32_t x_block, int32_t w_block, void* workspace, size_t workspace_bytes,
                     void* counters, size_t counter_bytes, void* stream);
int tilec_linear_fp8_scratch_bytes(const void* x, const void* weight, int64_t M, int64_t N, int64_t K, int64_t ldx,
                                   int64_t ldw, int32_t x_dtype, int32_t w_dtype, int32_t out_dtype,
                                   size_t* workspace_bytes, size_t* counter_bytes);

/*
 * 8-bit operands.  A block's scale and codes, each operation a float32 one that
 * rounds to nearest, L the largest value of the type (448 or 57344):
 *   a = max(largest magnitude, 2^-100);  scale = a / L;  code = round(x * (L / a))
 * A block that holds a NaN or an infinity has a NaN for its scale and its codes.
 *
 * x [R, C], float32 or bfloat16, is row-major with row stride ldx (>= C) or, with
 * layout TILEC_X1_COL_MAJOR, column-major (column stride ldx >= R): the transpose
 * of a row-major matrix, quantised in blocks of its own columns.  Rows of codes
 * begin at multiples of 16 bytes (codes 16-byte aligned, ldq a multiple of 16);
 * the bytes from C to the next multiple of 16 are set to zero.
 */
int tilec_quantize_fp8(const void* x, void* codes, float* scales, int64_t R, int64_t C, int64_t ldx, int64_t ldq,
                       int64_t scale_row, int64_t scale_group, int32_t layout, int32_t x_dtype, int32_t q_dtype,
                       int32_t block, void* stream);

/* The values that codes stand for, in float32 or bfloat16: out[r, c] = code[r, c] * scale. */
int tilec_dequantize_fp8(const void* codes, const float* scales, void* out, int64_t R, int64_t C, int64_t ldq,
                         int64_t ldo, int64_t scale_row, int64_t scale_group, int32_t q_dtype, int32_t out_dtype,
                         int32_t block, void* stream);

/*
 * Root mean square norm over the rows of h [R, D], D >= 1:
 *   h = x + residual, rounded to the residual's type (residual NULL: h = x, not written)
 *   rstd = 1 / sqrt(sum(h^2) / D + eps);  y = h rstd weight
 * x, residual and weight [D] (NULL: ones) are float32 or bfloat16 each, h has the
 * residual's type.  y is float32, bfloat16, or 8-bit codes with y_scale
 * [R, ceil(D / 128)] for blocks of 1 x 128, as tilec_quantize_fp8 writes them of
 * the float32 y.  rstd [R] float32 is written where not NULL.  h may be the
 * residual, rows and all (ldh == ldr); otherwise outputs must not overlap inputs.
 */
int tilec_rms_norm(const void* x, const void* residual, const void* weight, void* y, float* y_scale, void* h,
                   float* rstd, int64_t R, int64_t D, int64_t ldx, int64_t ldr, int64_t ldy, int64_t ldh,
                   int64_t scale_row, int64_t scale_group, int32_t x_dtype, int32_t r_dtype, int32_t y_dtype,
                   int32_t w_dtype, float eps, void* stream);

/*
 * Its gradients, hhat = h rstd:
 *   dx = rstd (dy weight - hhat mean(dy weight hhat)) + dh;  dweight = sum over rows of dy hhat
 * dx is the gradient of x and of the residual alike; dh (NULL: zeros) is that of h
 * from its other reader.  dx has dh's type, or dy's without it; dweight [D],
 * float32, may be NULL and is added in a fixed order.  `workspace`:
 * tilec_rms_norm_backward_workspace_bytes, any contents, 16-byte aligned.  dx may
 * be dh, rows and all (lddx == lddh), and overlaps nothing else.
 */
int tilec_rms_norm_backward(const void* dy, const void* h, const float* rstd, const void* weight, const void* dh,
                            void* dx, float* dweight, int64_t R, int64_t D, int64_t lddy, int64_t ldh, int64_t lddh,
                            int64_t lddx, int32_t dy_dtype, int32_t h_dtype, int32_t dh_dtype, int32_t w_dtype,
                            void* workspace, size_t workspace_bytes, void* stream);
size_t tilec_rms_norm_backward_workspace_bytes(int64_t R, int64_t D, int32_t h_dtype);

/*
 * The norm of a list of gradients and the factor that clips it to max_norm
 * (negative or infinite: no limit), both one float32 on the device:
 *   norm = |grad_scale| sqrt(sum of all g^2);  scale = grad_scale min(1, max_norm / (norm + 1e-6))
 * grad_scale: one float32 on the device (NULL: 1); scale may be NULL.  Squares
 * and sums are float64, in a fixed order.  An infinite norm gives a scale of 0, a
 * NaN one NaN.  Tensors are contiguous, at any alignment of their type; the
 * descriptions (host memory) are read before the call returns.  `workspace`:
 * tilec_grad_norm_workspace_bytes, any contents, 16-byte aligned.  `counter`: 4
 * bytes, zero before the call and left zero; concurrent calls need their own.
 *
 * tilec_scale_grads multiplies every value by *scale in place, rounding once; it
 * touches none where *scale is 1.  No two tensors may overlap.
 */
typedef struct tilec_grad {
  void* data; /* float32 or bfloat16 [n] */
  int64_t n;
  int32_t dtype;
} tilec_grad;
int tilec_grad_norm(const tilec_grad* grads, int32_t count, const float* grad_scale, double max_norm, float* norm,
                    float* scale, void* workspace, size_t workspace_bytes, void* counter, size_t counter_bytes,
                    void* stream);
size_t tilec_grad_norm_workspace_bytes(const tilec_grad* grads, int32_t count);
int tilec_scale_grads(const tilec_grad* grads, int32_t count, const float* scale, void* stream);

/* Message describing the last failure on this thread ("" if none). */
const char* tilec_last_error(void);

/* ABI version (major * 10000 + minor * 100 + patch). */
int32_t tilec_version(void);

#ifdef __cplusplus
}
#endif

#endif /* TILEC_H */
