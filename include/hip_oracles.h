/*
 * hip_oracles.h -- C ABI of libhip_oracles.so, the MI355X (gfx950) kernel
 * library behind the gfx950 oracle registrations.
 *
 * In better-benchmark an oracle is `oracle_forward(inputs, **cfg)` in a
 * canonical repro's oracle.py, registered with `@oracle_impl(...)`
 * (reference: oracle_harness.py:468-549); its body launches Triton kernels.
 * Each entry point below replaces one such body: the Python oracle
 * allocates the outputs with torch, then calls here with raw device pointers,
 * sizes and the caller's HIP stream.
 *
 * Conventions shared by every entry point:
 *   - Pointers are device pointers.  bf16 tensors are passed as uint16_t*
 *     (raw bfloat16 bit patterns).  Tensors are dense and row-major
 *     (contiguous) unless a stride argument says otherwise.
 *   - `stream` is the caller's stream (torch.cuda.current_stream()); every
 *     launch goes on it.  Calls only enqueue work: no allocation, no
 *     synchronisation, no host<->device copies, so they are safe under
 *     hipStreamBeginCapture / torch.cuda.graph.
 *   - Return 0 on success.  Non-zero is a hipError_t from the launch, or
 *     HIPO_EINVAL (argument check failed before anything was launched).
 *     hipo_last_error() then holds a message (per calling thread).
 *   - Re-entrant.  The only global state is a per-device cache of device
 *     properties, filled on first use.
 */
#ifndef HIP_ORACLES_H_
#define HIP_ORACLES_H_

#include <stddef.h>
#include <stdint.h>

#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HIPO_ABI_VERSION 4
#define HIPO_EINVAL 1000

/* ABI version of the loaded library (HIPO_ABI_VERSION at build time). */
int hipo_abi_version(void);

/* Message describing the last failed call on this thread ("" if none). */
const char* hipo_last_error(void);

/*
 * Row mean: out[r] = mean(x[r, 0:cols]) in fp32.
 * x is [rows, cols] with row stride `row_stride` elements (>= cols).
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/mean_c9e1a8113328/oracle.py:95 (_spatial_mean_row_kernel,
 * same file :45) for the row-reduction form `x.mean(dim=-1)`.
 */
int hipo_row_mean_f32(const float* x, float* out, int64_t rows, int64_t cols,
                      int64_t row_stride, hipStream_t stream);

/*
 * Channel bias + GELU(tanh) + NCHW -> NHWC:
 *   t = bf16(x[n,c,hw] + bias[c])       (eager order: the add rounds to bf16)
 *   y = 0.5 t (1 + tanh(sqrt(2/pi) (t + 0.044715 t^3)))
 *   out[n,hw,c] = bf16(y), correctly rounded (t is bf16: a table of the
 *                 exactly rounded results by bit pattern)
 * x is contiguous NCHW [n, c, hw]; out is the same logical tensor stored
 * channels-last (physical [n, hw, c]).
 * Replaces the Triton bodies of oracle_forward in
 * repros/canonical/pointwise_2d969ac9ad59/oracle.py:47 (tanh GELU) and
 * repros/canonical/pointwise_021e90d9c17d/oracle.py:58 (permute + clone),
 * fused into one pass.
 */
int hipo_bias_gelu_nchw_to_nhwc_bf16(const uint16_t* x, const uint16_t* bias,
                                     uint16_t* out, int64_t n, int64_t c,
                                     int64_t hw, hipStream_t stream);

/*
 * Scaled, additively masked softmax over the last dim (bf16 in/out):
 *   s[b,q,k] = fma(x[b,q,k], scale, mask[q,k])     (fp32 scores)
 *   out[b,q,:] = bf16(softmax_fp32(s[b,q,:]))
 * (eager's bf16 roundings of x * scale and of the sum are exact for a
 * power-of-two scale and a 0 / -inf mask, the causal softmax.)
 * x/out are [batch, q, k] contiguous; mask is [q, k] with row stride
 * `mask_row_stride` elements, broadcast over batch.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/amax_sum_20ccc18dda60/oracle.py:63
 * (_broadcast_add_softmax_kernel, same file :12), and -- with q = 1, one
 * zero mask row and scale 1 -- the plain softmax of
 * repros/canonical/amax_sum_fa4cc85fe5ad/oracle.py:68 (_bf16_softmax_kernel,
 * same file :12).
 */
int hipo_scaled_masked_softmax_bf16(const uint16_t* x, const uint16_t* mask,
                                    uint16_t* out, int64_t batch, int64_t q,
                                    int64_t k, int64_t mask_row_stride,
                                    float scale, hipStream_t stream);

/*
 * Residual add + LayerNorm forward over the last dim (bf16 in/out):
 *   h = bf16(x + residual);  mean, var = fp32 stats of h (population var)
 *   rstd = 1/sqrt(var + eps);  y = bf16((h - mean) * rstd * gamma + beta)
 * x, residual, h, y are [rows, cols] contiguous; gamma, beta are [cols];
 * mean, rstd are fp32 [rows].  h, and y, may be x or the residual itself
 * (not both of them the same tensor), and overlap no operand otherwise.
 * h, mean and rstd may be NULL: that output is
 * not written (the reference's var_mean_80e7ff4dee7f returns y only).
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/var_mean_80e7ff4dee7f/oracle.py:122
 * (_residual_layernorm_kernel, same file :51), and of the residual-LayerNorm
 * families var_mean_0ada225c0a04, var_mean_96edf0542ecd,
 * var_mean_f4578c128d74, var_mean_b19e82f2a47b, var_mean_393456b916a6 and
 * var_mean_45f7dfd4a983 (oracle.py, oracle_forward).
 */
int hipo_residual_layernorm_bf16(const uint16_t* x, const uint16_t* residual,
                                 const uint16_t* gamma, const uint16_t* beta,
                                 uint16_t* h, uint16_t* y, float* mean,
                                 float* rstd, int64_t rows, int64_t cols,
                                 float eps, hipStream_t stream);

/*
 * RMSNorm forward over the last dim (bf16 in/out):
 *   rstd = 1/sqrt(mean(x^2) + eps)   (fp32)
 *   y = bf16(x * rstd * gamma)       (fp32 arithmetic, one rounding)
 * x, y are [rows, cols] contiguous; gamma is [cols]; rstd is fp32 [rows].
 * y may be x itself, and does not overlap it otherwise.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/mean_4462ce967d63/oracle.py:65.
 */
int hipo_rmsnorm_bf16(const uint16_t* x, const uint16_t* gamma, uint16_t* y,
                      float* rstd, int64_t rows, int64_t cols, float eps,
                      hipStream_t stream);

/*
 * RMSNorm with the options the corpus variants use:
 *   h = residual ? bf16(x + residual) : x       (the eager bf16 add)
 *   rstd = 1/sqrt(mean(h^2) + eps)             (fp32)
 *   mode 0: y = bf16(h * rstd * gamma * scale)  (torch rms_norm, one rounding)
 *   mode 1: t = bf16(h * rstd); u = bf16(gamma * t);
 *           y = scale == 1 ? u : bf16(u * scale)   (HF T5 LayerNorm op order)
 * residual, h and rstd may be NULL (h, the bf16 sum, only with a
 * residual).  Shapes as hipo_rmsnorm_bf16; h and y may be x or the residual
 * as in hipo_residual_layernorm_bf16.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/mean_4462ce967d63/oracle.py:65 (T5: residual, eps 1e-6,
 * mode 1, scale 0.04419417382415922) and of the residual-RMSNorm families
 * mean_f08c75b5f21f, mean_db9733790220, mean_8818e35b12aa,
 * mean_c033ad4c69ca, mean_f21cc667fe83 (mode 0), mean_426e2409482e,
 * mean_4dace6865eee, mean_bf2ed36e56df, mean_d28c6a07654f and
 * mean_41e8bba10b8b (oracle.py, oracle_forward).
 */
int hipo_rmsnorm_ex_bf16(const uint16_t* x, const uint16_t* residual,
                         const uint16_t* gamma, uint16_t* h, uint16_t* y, float* rstd,
                         int64_t rows, int64_t cols, float eps, float scale,
                         int mode, hipStream_t stream);

/*
 * Softmax over the last dim with an additive bias shared by groups of
 * `heads` consecutive batch entries:
 *   s[b,q,k] = fma(x[b,q,k], scale, bias[b / heads][q, k])   (fp32 scores,
 *              as the reference's Triton oracle builds them)
 *   out[b,q,:] = bf16(softmax_fp32(s[b,q,:]))
 * bias row of (b, q): bias + (b / heads) * bias_batch_stride
 *                          + q * bias_row_stride   (elements).
 * hipo_scaled_masked_softmax_bf16 is the case bias_batch_stride = 0.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/amax_sum_20ccc18dda60/oracle.py:63 (x viewed
 * [64, 16, 256, 256] + bias [64, 1, 256, 256]: heads = 16, scale = 1).
 */
int hipo_scaled_bias_softmax_bf16(const uint16_t* x, const uint16_t* bias,
                                  uint16_t* out, int64_t batch, int64_t q,
                                  int64_t k, int64_t bias_row_stride,
                                  int64_t bias_batch_stride, int64_t heads,
                                  float scale, hipStream_t stream);

/*
 * Bytes of fp32 workspace hipo_spatial_mean_nhwc_bf16 needs (0: none).
 */
size_t hipo_spatial_mean_workspace_bytes(int64_t n, int64_t hw, int64_t c);

/*
 * Spatial mean of a channels-last bf16 tensor (a reduction over a
 * non-innermost axis):
 *   out[n, c] = bf16(sum_p x[n, p, c] / hw)     (fp32 accumulation)
 * x is [n, c, h, w] stored channels-last, i.e. physical [n, hw, c] with c
 * contiguous; out is [n, c] contiguous ([n, c, 1, 1] keepdim).  `workspace`
 * holds fp32 partial sums when the kernel splits positions; size from
 * hipo_spatial_mean_workspace_bytes (may be NULL when that is 0).
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/mean_c9e1a8113328/oracle.py:95
 * (_spatial_mean_cl_kernel, same file :11).
 */
int hipo_spatial_mean_nhwc_bf16(const uint16_t* x, uint16_t* out, int64_t n,
                                int64_t hw, int64_t c, void* workspace,
                                size_t workspace_bytes, hipStream_t stream);

/*
 * BatchNorm training forward on bf16 activations, fp32 statistics, in the
 * op order of the reference's bf16 BN graphs:
 *   mean[c], var[c] = var_mean(fp32(x), dims (0, 2, 3), correction 0)
 *   save_mean = mean;  save_rstd = 1 / sqrt(var + eps)
 *   y = act(bf16(((x - mean) * save_rstd) * gamma + beta))     (fp32 ops)
 *       act: 0 none, 1 ReLU, 2 SiLU (t / (1 + e^-t), rounded to bf16)
 *   running_mean = mean * momentum + running_mean * (1 - momentum)
 *   running_var  = (var * var_scale) * momentum
 *                  + running_var * (1 - momentum)             (in place)
 * var_scale is the graph's Bessel constant (N/(N-1) at the shape the graph
 * was captured at); it is applied as given.  gamma, beta, running_*,
 * save_* are fp32 [c].  The statistics pass writes (mean, M2) per slice and
 * channel into `workspace` (16-byte aligned, at least the size the matching
 * *_workspace_bytes call returns; no initialisation needed); calls that
 * share a workspace must be ordered.  Deterministic (fixed merge order).
 */

/* Workspace bytes of hipo_batchnorm_nhwc_act_pad_bf16 (0: empty shape). */
size_t hipo_batchnorm_nhwc_workspace_bytes(int64_t n, int64_t h, int64_t w, int64_t c);

/*
 * x is [n, c, h, w] stored channels-last (physical [n, h, w, c]); out is
 * [n, c, h + pad_bottom, w + pad_right] stored channels-last, y in the
 * top-left h x w window and zeros in the padding.  Without padding out may be
 * x itself; it does not overlap x otherwise.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/var_mean_ceb5c315290a/oracle.py:238 (split-K statistics,
 * then the normalise + SiLU + pad epilogue; eps 1e-3, SiLU, pad 1).
 */
int hipo_batchnorm_nhwc_act_pad_bf16(const uint16_t* x, const float* gamma,
                                     const float* beta, float* running_mean,
                                     float* running_var, float* save_mean,
                                     float* save_rstd, uint16_t* out, int64_t n,
                                     int64_t h, int64_t w, int64_t c,
                                     int64_t pad_bottom, int64_t pad_right,
                                     float momentum, float eps, float var_scale,
                                     int act, void* workspace,
                                     size_t workspace_bytes, hipStream_t stream);

/* Workspace bytes of hipo_batchnorm_nchw_act_mean_bf16 (0: empty shape). */
size_t hipo_batchnorm_nchw_mean_workspace_bytes(int64_t n, int64_t c, int64_t hw);

/*
 * x is contiguous NCHW [n, c, hw]; out[n, c] = bf16(mean over hw of y)
 * (fp32 sum), a contiguous [n, c] bf16 tensor.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/var_mean_mean_19ffdb35cc67/oracle.py:167 (one CTA per
 * channel, then the normalise + ReLU + spatial-mean epilogue; eps 1e-5).
 */
int hipo_batchnorm_nchw_act_mean_bf16(const uint16_t* x, const float* gamma,
                                      const float* beta, float* running_mean,
                                      float* running_var, float* save_mean,
                                      float* save_rstd, uint16_t* out, int64_t n,
                                      int64_t c, int64_t hw, float momentum,
                                      float eps, float var_scale, int act,
                                      void* workspace, size_t workspace_bytes,
                                      hipStream_t stream);

/*
 * Bytes of device workspace hipo_batchnorm_train_fwd_f32 needs for this
 * shape (0 if a size is not positive).
 */
size_t hipo_batchnorm_workspace_bytes(int64_t n, int64_t c, int64_t hw);

/*
 * BatchNorm training forward over dims (0, 2, 3) of NCHW fp32, fused with
 * the affine transform, an optional ReLU and the running-stat update:
 *   mean[c], var[c] = population stats of x[:, c, :]   (correction 0)
 *   save_mean = mean;  save_invstd = 1/sqrt(var + eps)
 *   y = relu?((x - mean) * save_invstd * gamma + beta)
 *   running_mean = (1 - momentum) running_mean + momentum mean
 *   running_var  = (1 - momentum) running_var
 *                  + momentum var * count / (count - 1)     (in place)
 * x, y are contiguous [n, c, hw]; y may be x itself (in place), and does
 * not overlap it otherwise; gamma, beta, running_*, save_* are [c].
 * Channels of at most 16384 values (n * hw), and of up to 28672 (49152 where
 * hw is not a multiple of 4) where that is faster, run as one launch with a
 * workgroup per channel that holds it in registers (reads x once, uses no
 * workspace); larger ones as one persistent kernel that reads x once (HW a
 * multiple of 4, 16-byte aligned x / y, x under 4 GiB), others as two
 * split-K launches that read x twice.
 * `workspace` is caller-allocated device memory, 8-byte aligned, of at
 * least hipo_batchnorm_workspace_bytes(n, c, hw) bytes.  It must be
 * zero-filled before its first use and then passed unmodified to later
 * calls: the single-pass kernel keeps its cross-workgroup exchange state
 * there (a completion count, a launch epoch, tagged partial statistics).
 * Calls that share a workspace must be ordered (one stream); bytes 8..11
 * hold a sticky error word, nonzero after an exchange wait timed out (the
 * affected channels' outputs are then NaN).
 * Replaces the Triton bodies of oracle_forward in
 * repros/canonical/var_mean_mean_19ffdb35cc67/oracle.py:167 (one CTA per
 * channel) and repros/canonical/var_mean_ceb5c315290a/oracle.py:238
 * (split-K sum/sum-of-squares, then an epilogue that re-reads x).
 */
int hipo_batchnorm_train_fwd_f32(const float* x, const float* gamma,
                                 const float* beta, float* running_mean,
                                 float* running_var, float* y,
                                 float* save_mean, float* save_invstd,
                                 int64_t n, int64_t c, int64_t hw,
                                 float momentum, float eps, int relu,
                                 void* workspace, size_t workspace_bytes,
                                 hipStream_t stream);

/*
 * hipo_batchnorm_train_fwd_f32 without a caller workspace and without any
 * allocation: no counterpart in the reference.  For callers that cannot
 * allocate device memory or pass a workspace (code under hipGraph capture,
 * tight serving loops, harnesses that forbid hipMalloc).  Same arguments,
 * semantics, kernels and results as hipo_batchnorm_train_fwd_f32, minus the
 * workspace: it uses a 4 MiB file-scope device array per device instead,
 * held until the process ends.  Shapes whose
 * hipo_batchnorm_workspace_bytes(n, c, hw) exceeds 4 MiB are rejected with
 * HIPO_EINVAL (config [128, 256, 56, 56] needs about 96 KiB).  The first
 * call on a device looks up the array's address and clears it with a fill
 * kernel on `stream`; that first call must not be under stream capture
 * (HIPO_EINVAL), later ones may be.  Every call on a device shares that
 * device's array: calls that overlap on one device (several streams) race
 * and must not be issued.
 */
int hipo_batchnorm_train_fwd_f32_noalloc(const float* x, const float* gamma,
                                         const float* beta, float* running_mean,
                                         float* running_var, float* y,
                                         float* save_mean, float* save_invstd,
                                         int64_t n, int64_t c, int64_t hw,
                                         float momentum, float eps, int relu,
                                         hipStream_t stream);

/*
 * The sticky error word of the allocation-free path's static scratch array
 * on `device`: nonzero once an exchange wait of the single-pass kernel
 * timed out there (that call's outputs and running statistics are then
 * NaN).  *word = 0 if hipo_batchnorm_train_fwd_f32_noalloc never ran on the
 * device.  Waits for the device's work to finish (a host query, not a launch:
 * never call it under stream capture); with `clear`, a nonzero word is reset
 * to zero.  No counterpart in the reference: the fault channel of the
 * allocation-free entry point, whose workspace the caller cannot inspect.
 */
int hipo_batchnorm_noalloc_error(int device, uint32_t* word, int clear);

/*
 * Flat stream copy (a measurement yardstick, not an oracle): reads
 * read_bytes from src and writes write_bytes to dst in one launch with the
 * oracle kernels' access style (16-byte non-temporal accesses, 1 KiB per
 * wave, one-shot grid in memory order); chunk i of dst receives chunk i of
 * src where both exist.  Sizes are multiples of 1024 (write_bytes >= 1024),
 * pointers 16-byte aligned.  The time of this copy at a config's read and
 * write bytes is the ceiling the config's kernel is compared with.
 * Counterpart of the reference's memcopy speed-of-light construction
 * (repro_harness.py:952-958, an fp32 add(src, 1, out=dst) over the same
 * bytes), written for MI355X with the stores that kernel lacks.
 */
int hipo_flat_copy(const void* src, int64_t read_bytes, void* dst,
                   int64_t write_bytes, hipStream_t stream);

/*
 * Yardstick for two-input, two-output streaming kernels (the residual
 * LayerNorm: x, residual -> h, y): copies bytes of src0 to dst0 and of src1
 * to dst1 in one launch, each wave moving one 1 KiB chunk of all four
 * buffers with 16-byte non-temporal accesses.  bytes: a positive multiple
 * of 1024; pointers 16-byte aligned.  No counterpart in the reference (its
 * memcopy SOL is one stream each way, repro_harness.py:952-958); used only
 * to price a kernel's access pattern.
 */
int hipo_flat_copy2(const void* src0, const void* src1, void* dst0, void* dst1,
                    int64_t bytes, hipStream_t stream);

/*
 * Yardstick for the single-pass BatchNorm (hipo_batchnorm_train_fwd_f32's
 * fused kernel): y = x for fp32 [n, c, hw] NCHW, with that kernel's exact
 * access pattern -- the same slabs and rounds, each workgroup holding its
 * slab in registers from its loads to its stores, the same per-thread
 * statistics (they wait for each round's loads) and barriers -- but no
 * exchange between workgroups and no normalisation.  Its time is the
 * ceiling of that pattern.  Applies where the fused kernel does (hw a
 * multiple of 4, x and y 16-byte aligned, at most 64 slabs per channel and
 * 64 rounds); other shapes are rejected.  No counterpart in the reference;
 * used only to price a kernel's access pattern.
 */
int hipo_hold_copy_f32(const float* x, float* y, int64_t n, int64_t c, int64_t hw,
                       hipStream_t stream);


/*
 * GELU(tanh) of a contiguous tensor of n elements, element by element:
 *   bf16: y = the correctly rounded bf16 of 0.5 x (1 + tanh(sqrt(2/pi)
 *         (x + 0.044715 x^3))) for every bf16 x (no intermediate rounding);
 *   fp32: the same function as x / (1 + e^(-2u)), u = sqrt(2/pi) (x +
 *         0.044715 x^3), with an extended-precision exp and an IEEE division
 *         (a few fp32 ulps from the exact value; no cancellation).
 * x and y are 16-byte aligned and do not overlap.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/pointwise_2d969ac9ad59/oracle.py:44-62 (_tanh_gelu_kernel,
 * same file :12-26), whose view-reshape wrapper stays in Python.
 */
int hipo_gelu_tanh_bf16(const uint16_t* x, uint16_t* y, int64_t n, hipStream_t stream);
int hipo_gelu_tanh_f32(const float* x, float* y, int64_t n, hipStream_t stream);

/*
 * Batched transpose of the last two dimensions, bit for bit:
 *   y[b, c, r] = x[b, r, c],  x [batch, rows, cols], y [batch, cols, rows],
 * both contiguous, elements of elem_size bytes (2 or 4), x and y distinct.
 * permute(0, 1, 3, 2) + clone of a contiguous 4-D tensor is the case
 * batch = d0 * d1.  Replaces the Triton body of oracle_forward in
 * repros/canonical/pointwise_021e90d9c17d/oracle.py:55-80
 * (_visformer_attention_to_image_kernel, same file :23).
 */
int hipo_transpose_last2(const void* x, void* y, int64_t batch, int64_t rows,
                         int64_t cols, int elem_size, hipStream_t stream);

/*
 * bf16 row mean with an optional ReLU (relu != 0; NaN propagates):
 *   out[r] = bf16(sum_j act(x[r, j]) / cols), fp32 sum, one rounding.
 * x is contiguous [rows, cols] (cols >= 1); out is [rows].  The NCHW
 * spatial mean relu(x).mean([-1, -2]) is the case rows = N * C, cols = H * W.
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/mean_b402ee209d0b/oracle.py:53-80
 * (_relu_spatial_mean_kernel, same file :23-50).
 */
int hipo_row_mean_bf16(const uint16_t* x, uint16_t* out, int64_t rows, int64_t cols,
                       int relu, hipStream_t stream);

/* Workspace bytes of hipo_gelu_erf_bwd_colsum_bf16 (0: empty shape). */
size_t hipo_gelu_erf_bwd_colsum_workspace_bytes(int64_t rows, int64_t cols);

/*
 * GELU(erf) backward with the column sum of its output (a bias gradient):
 *   y[r, c]   = bf16(grad[r, c] * d(x[r, c])),
 *               d(t) = Phi(t) + t phi(t), the derivative of t Phi(t), taken
 *               as the correctly rounded fp32 value for each bf16 t (one
 *               fp32 product, one rounding; inf and NaN t give NaN);
 *   colsum[c] = bf16(sum_r y[r, c]) stored as fp32 (fp32 sums of the bf16 y,
 *               in a fixed order for a given shape).
 * grad, x, y are contiguous [rows, cols] bf16, 16-byte aligned, cols a
 * multiple of 8; colsum is [cols] fp32.  `workspace` holds fp64 partial sums:
 * at least hipo_gelu_erf_bwd_colsum_workspace_bytes(rows, cols) bytes,
 * 16-byte aligned, no initialisation needed; NULL when that is 0 (up to 256
 * rows, a single launch; rows == 0 sets colsum to zero).
 * Replaces the Triton body of oracle_forward in
 * repros/canonical/sum_139a3020e8bf/oracle.py:101-152
 * (_materialize_partial_kernel :13, _final_sum_kernel :62) for the graph of
 * repros/canonical/sum_139a3020e8bf/repro.py:24-48.
 */
int hipo_gelu_erf_bwd_colsum_bf16(const uint16_t* grad, const uint16_t* x, uint16_t* y,
                                  float* colsum, int64_t rows, int64_t cols,
                                  void* workspace, size_t workspace_bytes,
                                  hipStream_t stream);

/*
 * Log probabilities of given tokens.  With s_j = scale * x[r, j]:
 *   lse[r]     = ln sum_j e^(s_j)
 *   logprob[r] = s_t - lse[r],  t = tokens[r]
 *   entropy[r] = -sum_j p_j ln p_j,  p_j = e^(s_j - lse)   (0 where p_j = 0)
 *   top_token[r, 0:top], top_logprob[r, 0:top]: the `top` largest logits of
 *                the row in falling order (of equal ones the lower index
 *                first; NaN above all) and their s - lse
 * in fp32 (one pass over the row).  logits is [rows, vocab] with row stride
 * `row_stride` (>= vocab), of bf16 (elem_size 2) or fp32 (4), at any element
 * alignment; tokens is [rows] of int32 (token_size 4) or int64 (8); the
 * outputs are contiguous.  entropy may be NULL; top is at most 64 and at
 * most vocab, its outputs NULL where it is 0; scale is from 2^-100 to 2^100.
 * A row whose token is ignore_index is left out, whatever its logits hold:
 * 0, 0, 0, and for the alternatives -inf and -1.  A token outside [0, vocab)
 * otherwise has logprob NaN.  A row with nothing above -inf has lse -inf, one
 * with +inf lse +inf, one with NaN lse NaN; their logprobs are s - lse, their
 * entropy NaN.  In the others no logprob is above 0 and no entropy below; where
 * one value is above -inf, its logprob and the entropy are 0.  `workspace`: at
 * least hipo_token_logprobs_workspace_bytes bytes, 16-byte aligned, no
 * initialisation needed (NULL when that is 0); calls that share one must be
 * ordered.  A call with top <= 33 takes about twice the time of one without,
 * with more alternatives or many equal values several times as long; where the
 * largest values crowd into a few runs of 16-byte vectors, up to a pass over
 * the row for each alternative.
 * No counterpart among the reference's oracles; beside
 * hipo_scaled_masked_softmax_bf16 as the softmax of a whole vocabulary.
 */
size_t hipo_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top);
int hipo_token_logprobs(const void* logits, int elem_size, const void* tokens,
                        int token_size, float* logprob, float* lse, float* entropy,
                        float* top_logprob, int64_t* top_token, int64_t rows,
                        int64_t vocab, int64_t row_stride, float scale,
                        int64_t ignore_index, int64_t top, void* workspace,
                        size_t workspace_bytes, hipStream_t stream);

/*
 * Gradient of hipo_token_logprobs with respect to the logits, for the
 * gradients grad of logprob, grad_entropy of entropy and grad_lse of lse
 * (each fp32 [rows]; the latter two may be NULL):
 *   dx[r, j] = scale * (grad [j = t]
 *              + p_j (grad_lse - grad - grad_entropy (ln p_j + entropy)))
 * fp32 arithmetic, one rounding to the logits' type.  lse, and entropy (with
 * grad_entropy), are the forward's results.  logits and dlogits are [rows,
 * vocab] with row strides of their own; dlogits may be logits itself (one
 * stride), and does not overlap it otherwise, nor the other inputs.  Rows of
 * ignore_index are zero, whatever they hold; rows of another token outside
 * [0, vocab) are NaN, and so are rows with NaN or with nothing above -inf, and
 * a +inf's own place.  p_j is e^(s_j - lse) of the fp32 lse: off by a factor of
 * about 1 + |lse| 2^-24, and no probability where |lse| is 2^24 and more (a row
 * of nothing but a mask of -1e9): leave such rows out.
 * No counterpart among the reference's oracles; beside
 * hipo_gelu_erf_bwd_colsum_bf16 as a training gradient.
 */
int hipo_token_logprobs_bwd(const float* grad, const void* logits, int elem_size,
                            const void* tokens, int token_size, const float* lse,
                            const float* entropy, const float* grad_entropy,
                            const float* grad_lse, void* dlogits, int64_t rows,
                            int64_t vocab, int64_t row_stride,
                            int64_t dlogits_row_stride, float scale,
                            int64_t ignore_index, hipStream_t stream);

/*
 * Embedding lookup with a scale:
 *   out[i, :] = scale * weight[tokens[i], :]   (fp32 product, one rounding)
 * weight is [vocab, width] with row stride `row_stride` (>= width), of bf16
 * (elem_size 2) or fp32 (4), out [count, width] contiguous of the same type,
 * both at any element alignment; tokens is [count] of int32 (token_size 4)
 * or int64 (8).  A token outside [0, vocab) gives a row of NaN.
 * No counterpart among the reference's oracles; the input of the
 * residual-RMSNorm and LayerNorm families.
 */
int hipo_embedding(const void* weight, int elem_size, const void* tokens,
                   int token_size, void* out, int64_t count, int64_t width,
                   int64_t vocab, int64_t row_stride, float scale,
                   hipStream_t stream);

/*
 * Gradient of hipo_embedding with respect to the weight:
 *   dweight[v, :] = scale * sum_{i: tokens[i] = v} grad[i, :]
 * in fp32, in an order that the tokens alone fix (the same call gives the
 * same bits), rounded once.  Every row of dweight is written, zeros where no
 * token is; with accumulate != 0 the sum is added to what dweight holds
 * (before the rounding) and rows without tokens are not touched.  Tokens
 * equal to padding_idx, and tokens outside [0, vocab), add nothing (an index
 * outside [0, vocab): no padding).  grad is contiguous [count, width] of bf16
 * (elem_size 2) or fp32 (4), dweight contiguous [vocab, width] of bf16
 * (out_size 2) or fp32 (4), the two apart; count and width are at most
 * 2^31 - 4097, vocab 2^30.  The time grows with vocab also where accumulate
 * leaves rows alone: every 512 rows past 65536 scan the tokens once more (2048
 * tokens: 12 us into 65536 rows, 262 into 10^7).  `workspace`: at least
 * hipo_embedding_bwd_workspace_bytes bytes, 16-byte aligned, no
 * initialisation needed (NULL when that is 0); calls that share one must be
 * ordered.
 * No counterpart among the reference's oracles.
 */
size_t hipo_embedding_bwd_workspace_bytes(int64_t count, int64_t width, int64_t vocab);
int hipo_embedding_bwd(const void* grad, int elem_size, const void* tokens,
                       int token_size, void* dweight, int out_size, int64_t count,
                       int64_t width, int64_t vocab, float scale,
                       int64_t padding_idx, int accumulate, void* workspace,
                       size_t workspace_bytes, hipStream_t stream);

/*
 * The norms around a block of a residual network, fused with its gate and the
 * residual sum.  With norm(v; w, b) = (v - m) r (offset + w) + b, r = 1 /
 * sqrt(mean((v - m)^2) + eps), m the row's mean (layer = 1, LayerNorm) or 0
 * (layer = 0, RMSNorm, without biases):
 *   n = post ? norm(x; post, post_bias) : x
 *   h = residual + scale * gate * n        (one rounding to the tensors' type)
 *   y = norm(h; pre, pre_bias)             (of h as it is stored; pre only)
 *   stats[r] = (mean, r) of x, then of h   (0 and 1 where there is no norm)
 * in fp32.  x, residual, h, y are [rows, cols] contiguous of bf16 (elem_size
 * 2) or fp32 (4), the vectors [cols] of the same type, all at any element
 * alignment; cols is from 8 to 16384.  gate is [gate_rows, cols], row r taking
 * gate row r / (rows / gate_rows): 1 for a vector that all rows share, rows
 * for a gate per value, between them one per sample (gate_rows divides rows);
 * NULL with gate_rows 0 for none.  One of post and pre may be NULL, and so may
 * the biases; y is NULL where pre is.  The outputs overlap no operand.
 * No counterpart among the reference's oracles; beside
 * hipo_residual_layernorm_bf16 and hipo_rmsnorm_ex_bf16, which have the second
 * norm alone, of bf16, and are quicker where that is all and no gradient follows
 * ([8192, 4096] 46 and 45 us, here 53 and 47; [16, 2048] 11 and 8, here 11 and 10).
 */
int hipo_block_norms(const void* x, const void* residual, int elem_size,
                     const void* post, const void* post_bias, const void* pre,
                     const void* pre_bias, const void* gate, void* h, void* y,
                     float* stats, int64_t rows, int64_t cols, int64_t gate_rows,
                     float scale, float offset, float eps, int layer,
                     hipStream_t stream);

/*
 * Gradient of hipo_block_norms for grad_h and grad_y, the gradients of h and y
 * (grad_h may be NULL where pre is not, grad_y is NULL where pre is): with T the
 * gradient of h from both,
 *   dresidual = T,  dgate = scale sum(T n) over the rows of each gate row,
 *   dx, dpost, dpost_bias from scale * gate * T, dpre, dpre_bias from grad_y
 * of x, h and stats as the forward left them.  fp32 sums in an order that the
 * sizes and the GPU fix (the same call gives the same bits), one rounding to
 * the tensors' type.  Sizes and types as in hipo_block_norms; x may be NULL
 * without post and gate, h without pre; each operand's gradient is given where
 * the operand is (dpost_bias with post_bias, ...).  The outputs overlap neither
 * each other nor an operand; with rows == 0 nothing is written.  `workspace`:
 * at least hipo_block_norms_bwd_workspace_bytes bytes, 16-byte aligned, no
 * initialisation needed; calls that share one must be ordered.
 * No counterpart among the reference's oracles.
 */
size_t hipo_block_norms_bwd_workspace_bytes(int64_t rows, int64_t cols);
int hipo_block_norms_bwd(const void* grad_h, const void* grad_y, const void* x,
                         const void* h, const float* stats, int elem_size,
                         const void* post, const void* post_bias, const void* pre,
                         const void* pre_bias, const void* gate, void* dx,
                         void* dresidual, void* dgate, void* dpost,
                         void* dpost_bias, void* dpre, void* dpre_bias,
                         int64_t rows, int64_t cols, int64_t gate_rows, float scale,
                         float offset, int layer, void* workspace,
                         size_t workspace_bytes, hipStream_t stream);

/*
 * Softmax cross entropy of the output layer without its logits: with
 * s_j = scale * sum_k hidden[r, k] weight[j, k],
 *   lse[r]  = ln sum_j e^(s_j)
 *   loss[r] = lse[r] - s_t,  t = tokens[r]
 * in fp32 sums of exact products (fp32 operands: of three bf16 parts each,
 * products below 2^-24 of the largest left out; parts end at 2^-133, so values
 * below 2^-110 are held to fewer bits than 24).  hidden is [rows, width],
 * weight [vocab, width], with row strides of their own (>= width), both of bf16
 * (elem_size 2) or fp32 (4), at any element alignment; tokens is [rows] of
 * int32 (token_size 4) or int64 (8); loss and lse are [rows]; scale is from
 * 2^-100 to 2^100.  At most 2^22 - 256 rows, width 2^20, weight_row_stride 2^21,
 * a vocabulary of 2^31 - 65536, and rows * width 2^38.  A row whose token is
 * ignore_index is left out, whatever it holds: 0 and 0.  A token outside [0,
 * vocab) otherwise has loss NaN.  A row with a NaN logit has lse NaN, one with a
 * logit of +infinity no finite lse; a logit of -infinity adds nothing to the sum,
 * and is a loss of +infinity for its own token (an infinite value in fp32 operands:
 * where those that it is multiplied with are below 128, else the logit may be NaN).
 * Up to 64 rows weight is read where it lies, and so
 * is one that is bf16, 16-byte aligned, of a width and a row stride that are
 * multiples of 8; others are copied into the workspace piece by piece.
 * `workspace`: at least hipo_linear_cross_entropy_workspace_bytes bytes (weight is
 * looked at for its alignment only), 16-byte aligned, no initialisation needed;
 * calls that share one must be ordered.  The same call gives the same bits; a row's
 * may differ in the last ones between batches of other sizes.
 * No counterpart among the reference's oracles; hipo_token_logprobs for logits
 * that are never in memory.
 */
size_t hipo_linear_cross_entropy_workspace_bytes(const void* weight, int elem_size,
                                                 int64_t rows, int64_t width,
                                                 int64_t vocab, int64_t weight_row_stride);
int hipo_linear_cross_entropy(const void* hidden, const void* weight, int elem_size,
                              const void* tokens, int token_size, float* loss,
                              float* lse, int64_t rows, int64_t width, int64_t vocab,
                              int64_t hidden_row_stride, int64_t weight_row_stride,
                              float scale, int64_t ignore_index, void* workspace,
                              size_t workspace_bytes, hipStream_t stream);

/*
 * Gradients of hipo_linear_cross_entropy for grad, the gradient of loss, and
 * grad_lse, of lse (fp32 [rows]; grad_lse may be NULL), lse being the forward's:
 *   d[r, j]  = scale * ((grad + grad_lse) e^(s_j - lse) - grad [j = t])
 *   dhidden  = d weight,  dweight = d^T hidden
 * the logits computed once more in pieces of the vocabulary, the products
 * accumulated in fp32 and rounded once to the operands' type; e^(s_j - lse) of
 * the fp32 lse is off by a factor of about 1 + |lse| 2^-24.  d itself is rounded to
 * bf16 where the operands are bf16 (the matrix cores' type): up to 64 rows, and
 * with _two_parts at any number of rows, to two bf16 parts, some 2^-17 of it, so
 * that the gradients are off by their own rounding alone, at twice the products of
 * dhidden and dweight.
 * dhidden is contiguous [rows, width], dweight [vocab, width]; they overlap
 * neither each other nor an operand.  Rows of ignore_index are zero in dhidden
 * and add nothing to dweight, whatever they hold; a row of another token outside
 * [0, vocab) is NaN and makes dweight NaN.  With rows == 0 dweight (where it is
 * given) is zero and no other pointer is looked at.  Operands and workspace as
 * above.
 * No counterpart among the reference's oracles.
 */
size_t hipo_linear_cross_entropy_bwd_workspace_bytes(const void* weight, int elem_size,
                                                     int64_t rows, int64_t width,
                                                     int64_t vocab,
                                                     int64_t weight_row_stride);
int hipo_linear_cross_entropy_bwd(const float* grad, const void* hidden,
                                  const void* weight, int elem_size,
                                  const void* tokens, int token_size,
                                  const float* lse, const float* grad_lse,
                                  void* dhidden, void* dweight, int64_t rows,
                                  int64_t width, int64_t vocab,
                                  int64_t hidden_row_stride,
                                  int64_t weight_row_stride, float scale,
                                  int64_t ignore_index, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream);
size_t hipo_linear_cross_entropy_bwd_two_parts_workspace_bytes(
    const void* weight, int elem_size, int64_t rows, int64_t width, int64_t vocab,
    int64_t weight_row_stride);
int hipo_linear_cross_entropy_bwd_two_parts(
    const float* grad, const void* hidden, const void* weight, int elem_size,
    const void* tokens, int token_size, const float* lse, const float* grad_lse,
    void* dhidden, void* dweight, int64_t rows, int64_t width, int64_t vocab,
    int64_t hidden_row_stride, int64_t weight_row_stride, float scale,
    int64_t ignore_index, void* workspace, size_t workspace_bytes,
    hipStream_t stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* HIP_ORACLES_H_ */
