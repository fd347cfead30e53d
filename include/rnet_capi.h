/*
 * rnet_capi.h — the C ABI of the B200 (sm_100a) ResonanceNet library
 * (librnet_b200.so). Plain pointers and sizes only; every entry point returns
 * RNET_OK (0) or a negative status and records a message for rnet_last_error().
 *
 * Pointers named d_* / documented as "device" are CUDA device pointers on the
 * current device; `stream` is a cudaStream_t passed as void* (NULL = legacy
 * default stream). Work is asynchronous on that stream unless stated.
 *
 * The C++ drop-in headers (layers.h, resonance_net.h, dist.h) are implemented
 * on top of these functions; a ctypes/cffi binding needs only this file.
 */
#ifndef RNET_CAPI_H
#define RNET_CAPI_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RNET_OK 0
#define RNET_ERR_ARG -1         /* invalid argument / unsupported shape */
#define RNET_ERR_CUDA -2        /* CUDA runtime error (message has details) */
#define RNET_ERR_NCCL -3        /* NCCL error or NCCL library not loadable */
#define RNET_ERR_TIMEOUT -4     /* host-side rendezvous / collective deadline */
#define RNET_ERR_IO -5          /* checkpoint file error, short or malformed file */
#define RNET_ERR_DEVICE -6      /* a kernel raised the device error word */
#define RNET_ERR_UNSUPPORTED -7 /* configuration not implemented */

/* ------------------------------------------------------------------ status */

/* Message of the most recent failing call on this thread ("" if none). */
const char* rnet_last_error(void);

/* Library ABI version (major*100 + minor). */
int rnet_abi_version(void);

/* Number of CUDA kernels this library has launched in this process. */
int rnet_kernel_launches(unsigned long long* n);

/* Read (and optionally clear) the device error word of the current device:
 * bit 0 = a bounded wait timed out, bit 1 = out-of-range index seen,
 * bit 2 = TMEM allocation failed, bit 3 = a selection gave up (its result is
 * incomplete; not expected on any input). Synchronises the device. */
int rnet_device_error(unsigned* word, int clear);

/* Self-test of the bounded-wait failure path (no reference counterpart): runs
 * n_ctas CTAs shaped like the pipelined kernels (a TMEM-owning warp and
 * waiters on an mbarrier) and waits on a barrier that nothing arrives on
 * (arrive = 0) or that one thread arrives on (arrive = 1), with a wait limit
 * of timeout_us. A run-out wait sets bit 0 of the device error word, the CTA
 * frees its TMEM and returns; *timed_out_ctas receives how many CTAs gave up.
 * Synchronises the device. */
int rnet_selftest_bounded_wait(int arrive, unsigned timeout_us, int n_ctas,
                               unsigned* timed_out_ctas);

/* ------------------------------------------------------------------ GEMM engine
 * C[M,N] (op)= alpha * A[M,K] * B[N,K]^T on the tcgen05 3xTF32 engine.
 * a_mn_major = 0: A(i,k) = A[i*lda + k]; 1: A(i,k) = A[k*lda + i]  (same for B).
 * op: 0 = store, 1 = accumulate (C += ...), 2 = residual (C = R + ...).
 * lda/ldb must be multiples of 4 and A/B 16-byte aligned. */
int rnet_gemm_f32(int M, int N, int K, const float* A, int lda, int a_mn_major, const float* B,
                  int ldb, int b_mn_major, float* C, int ldc, const float* R, int ldr, int op,
                  float alpha, void* stream);

/* C[M,N] (op)= alpha * A[M,K] * B[N,K]^T with bf16 A and B (same majors as
 * rnet_gemm_f32; row pitch a multiple of 8 elements, 16-byte aligned) on the
 * tcgen05 kind::f16 path: bf16 tiles staged by TMA straight from memory, fp32
 * accumulation, fp32 C. C16 (optional, op 0 / 2): also store the result as
 * bf16 with row pitch ldc. No counterpart in the reference (fp32 only). */
int rnet_gemm_bf16(int M, int N, int K, const void* A, int lda, int a_mn_major, const void* B,
                   int ldb, int b_mn_major, float* C, int ldc, const float* R, int ldr, int op,
                   float alpha, void* C16, void* stream);

/* Tile shape selection of the GEMM engine for every later call in this
 * process: 0 = automatic (CTA pairs, one 256-row MMA over two SMs, whenever
 * M > 128; single-CTA 128-row tiles otherwise), 1 = always single-CTA,
 * 2 = always CTA pairs. Results are identical up to fp32 summation order.
 * No counterpart in the reference (its GEMMs are cuBLAS calls). */
int rnet_gemm_set_cta_group(int cta_group);

/* Arithmetic of later rnet_gemm_f32 calls in this process: 0 = fp32-accurate
 * (default), 1 = bf16 operands with fp32 accumulation. */
int rnet_gemm_set_precision(int precision);

/* ------------------------------------------------------------------ layer ops
 * One entry per function of the reference's include/layers.h:28-153, same
 * argument meaning, same accumulate/overwrite contract:
 *   overwrite: every *_forward output and cache, rms_norm_backward dx,
 *              cross_entropy loss (sum over tokens) and dlogits;
 *   accumulate (+=): every parameter gradient, and dx of causal_conv /
 *              min_gru / slot_memory / swiglu backward.
 * All pointers are device pointers; temporaries are stream-ordered. The
 * cuBLAS handle of the reference signatures has no counterpart here. */
int rnet_rms_norm_forward(const float* x, const float* w, float* y, float* rms_cache,
                          int batch_seq, int dim, float eps, void* stream);
int rnet_rms_norm_backward(const float* dy, const float* x, const float* w,
                           const float* rms_cache, float* dx, float* dw, int batch_seq, int dim,
                           void* stream);
int rnet_embed_forward(const int* tokens, const float* table, float* output, int batch_seq,
                       int vocab, int dim, void* stream);
int rnet_embed_backward(const float* dout, const int* tokens, float* dtable, int batch_seq,
                        int vocab, int dim, void* stream);
/* output[M,N] = input[M,K] * weight[N,K]^T */
int rnet_linear_forward(const float* input, const float* weight, float* output, int M, int N,
                        int K, void* stream);
/* conv_buf [3, B*T, D] receives {S = c3+c7+c15, c7, c15} like the reference. */
int rnet_causal_conv_forward(const float* x, float* y, const float* conv3_w,
                             const float* conv7_w, const float* conv15_w, const float* mix_w,
                             float* conv_buf, int batch, int seq_len, int dim, void* stream);
/* dmix_quirk = 1 reproduces the reference's mix-weight gradient, which uses
 * S + c7 + c15 (src/causal_conv.cu:155-168); 0 uses S (the exact gradient). */
int rnet_causal_conv_backward(const float* dy, const float* x, const float* conv3_w,
                              const float* conv7_w, const float* conv15_w, const float* mix_w,
                              const float* conv_buf, float* dx, float* d_conv3_w,
                              float* d_conv7_w, float* d_conv15_w, float* d_mix_w, int batch,
                              int seq_len, int dim, int dmix_quirk, void* stream);
int rnet_min_gru_forward(const float* x, float* y, const float* Wz, const float* Wh,
                         const float* bz, const float* bh, float* z_cache, float* h_cache,
                         int batch, int seq_len, int dim, void* stream);
int rnet_min_gru_backward(const float* dy, const float* x, const float* Wz, const float* Wh,
                          const float* bz, const float* bh, const float* z_cache,
                          const float* h_cache, float* dx, float* dWz, float* dWh, float* dbz,
                          float* dbh, int batch, int seq_len, int dim, void* stream);
/* scores_cache may be NULL (scores are then not materialised; top_k == 2). */
int rnet_slot_memory_forward(const float* x, float* y, const float* slot_keys,
                             const float* slot_values, const float* proj_q,
                             const float* proj_out, float* q_cache, float* scores_cache,
                             int* topk_idx_cache, float* topk_w_cache, int batch, int seq_len,
                             int dim, int n_slots, int top_k, void* stream);
int rnet_slot_memory_backward(const float* dy, const float* x, const float* slot_keys,
                              const float* slot_values, const float* proj_q,
                              const float* proj_out, const float* q_cache,
                              const float* scores_cache, const int* topk_idx_cache,
                              const float* topk_w_cache, float* dx, float* d_slot_keys,
                              float* d_slot_values, float* d_proj_q, float* d_proj_out,
                              int batch, int seq_len, int dim, int n_slots, int top_k,
                              void* stream);
int rnet_swiglu_forward(const float* x, float* y, const float* gate_w, const float* up_w,
                        const float* down_w, float* gate_cache, float* up_cache, int batch_seq,
                        int dim, int d_ff, void* stream);
int rnet_swiglu_backward(const float* dy, const float* x, const float* gate_w,
                         const float* up_w, const float* down_w, const float* gate_cache,
                         const float* up_cache, float* dx, float* d_gate_w, float* d_up_w,
                         float* d_down_w, int batch_seq, int dim, int d_ff, void* stream);
int rnet_cross_entropy_forward(const float* logits, const int* targets, float* loss,
                               float* dlogits, int batch_seq, int vocab, void* stream);
/* Same result as rnet_cross_entropy_forward, but allocates nothing: for
 * callers that cannot allocate device memory while they run (a framework that
 * owns all device memory through its own pool, or a context where a
 * cudaMalloc/cudaMallocAsync is not allowed). No counterpart in the reference.
 * Scratch is a fixed 256 KiB array inside the library's device image, held on
 * every GPU that loads the library until exit, which limits batch_seq to
 * 524,280 tokens (larger sizes return RNET_ERR_ARG). The first call on each
 * device looks up that array's device address; make that first call before
 * any stream capture. All calls share the array, so calls that overlap on the
 * GPU (different streams, no ordering between them) race; calls ordered on
 * one stream are safe. The address is cached per device, so do not use this
 * entry point on a device after cudaDeviceReset. Out-of-range targets are
 * clamped to class 0 without
 * setting the device error word. */
int rnet_cross_entropy_forward_noalloc(const float* logits, const int* targets, float* loss,
                                       float* dlogits, int batch_seq, int vocab, void* stream);
int rnet_residual_add(float* x, const float* y, size_t n, void* stream);
int rnet_scale_grads(float* grads, float scale, size_t n, void* stream);

/* ------------------------------------------------------------------ logits
 * Operators on the logits of a model (no counterpart in the reference). Rows
 * of logits are fp32 or bf16 with a pitch of `ld` elements (ld >= vocab, any
 * alignment of the element size). All arithmetic is fp32 or wider. A
 * temperature lies within 1e-4 and 1e4. Nothing is kept from one call for the
 * next, and calls on different streams share nothing but the device error word;
 * that is set up by a device's first call, which is made outside any stream
 * capture. */
#define RNET_DTYPE_F32 0
#define RNET_DTYPE_BF16 1

/* The record a teacher keeps of each row: its top_k (1..64, <= vocab) largest
 * logits, sorted, ties to the lowest index. top_logits / top_idx are [rows,
 * top_k]; lse (may be NULL) is [rows]: log sum exp(logit / temperature) over
 * the whole row. A NaN logit counts as -inf, +inf as the largest finite fp32.
 * Places beyond the row's logits above -inf hold -inf / -1 (padding that the
 * distillation skips). vocab is at most 2^30. */
int rnet_topk_logits_forward(const void* logits, int dtype, long long ld, float temperature,
                             float* top_logits, int* top_idx, float* lse, int rows, int vocab,
                             int top_k, void* stream);

/* Distillation from such records, loss and gradient in one call, like
 * rnet_cross_entropy_forward. With z a row's logits, q = softmax(z /
 * temperature), p_k the teacher's probabilities and w = row_weight[row]:
 *   row_loss = w * (soft_weight * temperature^2 * sum_k p_k (log p_k - log q[i_k])
 *                   + hard_weight * (log sum exp(z) - z[target]))
 *   dlogits  = grad_scale * d row_loss / d z
 *   loss     = sum of row_loss (one float; a fixed order, may be NULL)
 * teacher_idx / teacher_logits [rows, top_k]: an index < 0 is padding, the same
 * index may come twice. teacher_lse NULL: p = softmax(teacher_logits /
 * temperature) over the row's entries (a row without entries has no soft
 * part); else p_k = exp(teacher_logits / temperature - teacher_lse), as
 * recorded at the same temperature, and the mass outside the record is left
 * out of the sum. targets [rows] (needed when hard_weight != 0): a negative
 * target has no hard part. row_weight [rows] (NULL = 1): a row of weight 0
 * gives exactly 0 loss and gradient whatever its logits and record hold. A row
 * whose logits are all -inf has no distribution and gives 0; a NaN or +inf
 * logit makes its row NaN. A teacher index or target >= vocab is skipped and
 * sets the device error word (bit 1). dlogits (may be NULL: loss only) has the
 * logits' type and a pitch of ld_dlogits; it may be the logits themselves
 * (same pointer and pitch). vocab <= 262144, top_k 1..64. */
int rnet_distill_topk_forward(const void* logits, int dtype, long long ld, const int* teacher_idx,
                              const float* teacher_logits, const float* teacher_lse,
                              const int* targets, const float* row_weight, float temperature,
                              float soft_weight, float hard_weight, float grad_scale,
                              float* row_loss, float* loss, void* dlogits, long long ld_dlogits,
                              int rows, int vocab, int top_k, void* stream);

/* ------------------------------------------------------------------ beam search
 * Streams are [batch * beams]: the beams of a sequence lie together, beams
 * 1..32. (No counterpart in the reference.)
 *
 * One selection: per sequence, the `beams` candidates (b, v) with the largest
 * scores_in[b] + log softmax(logits[b])[v], sorted. Totals are formed and compared in
 * 64 bits; equal ones go to the lower beam, then the larger logit, then the lower
 * token (a score may be so large, or logits so small, that unequal logits give equal
 * totals). A chosen total beyond fp32 is stored as infinity. finished_in[b] != 0 (NULL =
 * none finished; needs eos >= 0): the beam has ended and offers only
 * (b, eos) at its own score. Outputs [batch * beams]: scores, tokens, parents
 * (the beam 0..beams-1 each one continues) and finished (may be NULL without
 * finished_in) = the parent had finished, or token == eos (eos = -1: no token
 * ends a beam). A NaN logit or score counts as -inf, +inf as the largest
 * finite fp32; candidates at -inf are never taken. A sequence with fewer
 * candidates than beams fills the places left with score -inf, parent = the
 * place itself and token = eos (0 without one). So a search starts with scores
 * {0, -inf, ...}. scores / finished may be scores_in / finished_in. vocab is at
 * most 2^30. */
int rnet_beam_select(const void* logits, int dtype, long long ld, const float* scores_in,
                     const int* finished_in, int eos, float* scores, int* tokens, int* parents,
                     int* finished, int batch, int beams, int vocab, void* stream);

/* States follow their beams: in each of `outer` planes (outer_pitch bytes
 * apart) of batch * beams rows (row_pitch bytes apart, row_bytes long), row j of
 * a sequence becomes its old row parents[j]. dst may be src (in place: rows
 * that stay are not touched); otherwise the two must not overlap, and share
 * the pitches. Rows, pitches and pointers are multiples of 4 bytes. A parent
 * outside 0..beams-1 leaves its row as it is and sets the device error word
 * (bit 1). Bytes between the rows are not touched. */
int rnet_beam_reorder(const void* src, void* dst, size_t row_bytes, size_t row_pitch, size_t outer,
                      size_t outer_pitch, const int* parents, int batch, int beams, void* stream);

/* The sequences behind the last beams. tokens / parents [n_steps, batch *
 * beams] are the recorded outputs of n_steps (1..2^30) selections, scores [batch *
 * beams] the last one's. sequences [batch * beams, n_steps]: per sequence the
 * beams sorted by score / length^length_alpha (in 64 bits, from the fp32 numbers
 * given; ties to the lower beam; any finite length_alpha, and a score of 0 or -inf
 * stays as it is; NaN counts as -inf, +inf as the largest finite fp32); length
 * counts the tokens up to and including the first eos (n_steps without one, or with
 * eos < 0), and eos fills what follows. lengths and ranked_scores [batch * beams]
 * are in the same order (ranked_scores may be scores). A parent outside
 * 0..beams-1 counts as the beam itself and sets the device error word (bit 1). */
int rnet_beam_backtrack(const int* tokens, const int* parents, const float* scores, int eos,
                        float length_alpha, int* sequences, int* lengths, float* ranked_scores,
                        int n_steps, int batch, int beams, void* stream);

/* ------------------------------------------------------------------ data
 * Training batches of the reference's DataLoader (src/data_loader.cpp:31-52
 * as driven by src/main.cpp:117-133) with the corpus resident on the GPU.
 * rnet_data_create uploads n corpus bytes once (n = 0: the reference's
 * synthetic tokens); seed seeds the std::mt19937 the reference's training
 * loop passes to get_batch (42 + rank * 10007 there). rnet_data_batch makes
 * the reference's draws on the host (window starts, 8 bytes per sequence)
 * and gathers the windows into device int32 inputs / targets [batch *
 * seq_len] on `stream`, asynchronously; the batches equal the reference
 * loader's byte for byte. Not thread-safe per handle. */
typedef struct rnet_data rnet_data;
int rnet_data_create(const unsigned char* host_bytes, size_t n, int device, unsigned seed,
                     rnet_data** out);
int rnet_data_destroy(rnet_data* d);
int rnet_data_batch(rnet_data* d, int batch, int seq_len, int* d_inputs, int* d_targets,
                    void* stream);

/* ------------------------------------------------------------------ model
 * The reference's ResonanceNet class (include/resonance_net.h:56-130).
 * Parameters and gradients are single flat fp32 device buffers in checkpoint
 * tensor order (embed, output, final_norm, then per layer norm1..4, conv3,
 * conv7, conv15, mix, Wz, Wh, bz, bh, slot_keys, slot_values, proj_q,
 * proj_out, gate, up, down). */
typedef struct rnet_model_config {
  int d_model, n_layers, d_ff, n_heads, gru_dim, n_slots, slot_top_k, vocab_size, seq_len;
  float rms_eps;
} rnet_model_config; /* byte-identical to the 40-byte checkpoint header */

typedef struct rnet_model rnet_model;
typedef struct rnet_dist rnet_dist;

/* reference_init = 1: the reference's own initialisation (seeded uniform
 * Xavier, norm gains 1, biases 0); 0: all parameters zero. */
int rnet_model_create(const rnet_model_config* cfg, int device, int reference_init,
                      rnet_model** out);
/* Create a model from a checkpoint file (config read from its header). */
int rnet_model_create_from_checkpoint(const char* path, int device, rnet_model** out);
int rnet_model_destroy(rnet_model* m);
int rnet_model_get_config(const rnet_model* m, rnet_model_config* out);
int rnet_model_param_count(const rnet_model* m, size_t* n);
int rnet_model_device_buffers(rnet_model* m, float** d_params, float** d_grads);
int rnet_model_stream(rnet_model* m, void** stream);
int rnet_model_set_params(rnet_model* m, const float* host, size_t n);
/* Same as rnet_model_set_params from a device buffer (any stream order: the
 * call synchronises the model's stream). No counterpart in the reference. */
int rnet_model_set_params_device(rnet_model* m, const float* d_params, size_t n);
int rnet_model_get_params(rnet_model* m, float* host, size_t n);
int rnet_model_get_grads(rnet_model* m, float* host, size_t n);
/* Re-derive internal layouts after the caller wrote d_params directly. */
int rnet_model_params_updated(rnet_model* m);
int rnet_model_set_conv_quirk(rnet_model* m, int on);
/* GEMM arithmetic of the model: 0 = fp32-accurate (3xTF32 tcgen05, default),
 * 1 = bf16: every GEMM of the train step reads bf16 operands from memory
 * (tcgen05 kind::f16, fp32 accumulation): a bf16 shadow of the fp32 master
 * weights that the SGD update rewrites, and bf16 copies of the activations
 * and gradients that feed GEMMs, written by their producers. Master weights,
 * gradients, norms, scan, conv, slot selection and the optimizer stay fp32.
 * Parity with fp32 within 2e-2. */
int rnet_model_set_precision(rnet_model* m, int precision);
/* Activation recompute (no counterpart in the reference): 1 = keep only each
 * layer's input from the forward and recompute the layer's caches right
 * before its backward (one layer of caches resident instead of n_layers, at
 * the cost of one more forward per step); results are unchanged. With it on,
 * rnet_model_topk is unavailable. Default 0. */
int rnet_model_set_recompute(rnet_model* m, int on);
/* Optimizer extensions (no counterpart in the reference, whose step is plain
 * SGD with global-norm clipping; all three default to off, which keeps that
 * step): momentum (v = momentum * v + g, p -= lr * v), weight decay (wd * p
 * added to the clipped gradient) and a linear learning-rate warmup
 * (lr * min(1, (t + 1) / warmup_steps) at the t-th step after this call; the
 * reference parses TrainConfig::warmup_steps but never applies it). Resets
 * the step count and the velocity. */
int rnet_model_set_optimizer(rnet_model* m, float momentum, float weight_decay,
                             int warmup_steps);
int rnet_model_forward(rnet_model* m, const int* d_tokens, float* d_logits, int batch,
                       int seq_len);
int rnet_model_backward(rnet_model* m, const float* d_dlogits, const int* d_tokens, int batch,
                        int seq_len);
int rnet_model_zero_grad(rnet_model* m);
int rnet_model_step(rnet_model* m, float lr, float grad_clip);
/* zero_grad + forward + cross-entropy (dlogits scaled by 1/(batch*seq_len))
 * + backward + (all-reduce) + clipped SGD, all on the model stream.
 * d_loss_sum (device, may be NULL) receives the summed token loss. Without a
 * data-parallel group, repeated calls with the same batch, seq_len, lr,
 * grad_clip and model configuration replay a CUDA graph of the step captured
 * on the second such call (RNET_TRAIN_GRAPH=0 in the environment at model
 * creation keeps every step eager); the tokens are copied first, so the
 * buffers may differ from call to call. */
int rnet_model_train_step(rnet_model* m, const int* d_inputs, const int* d_targets, int batch,
                          int seq_len, float lr, float grad_clip, float* d_loss_sum);
/* The same step with rnet_distill_topk_forward's loss in the place of the
 * cross-entropy: the teacher's records d_teacher_idx / d_teacher_logits
 * [batch * seq_len, top_k], d_teacher_lse (may be NULL), d_targets (may be NULL
 * without hard_weight) and d_row_weight (may be NULL) as there, all device
 * pointers; dlogits scaled by 1/(batch*seq_len), d_loss_sum (may be NULL) the
 * sum of the rows' losses. Runs on the model stream, always eager (no graph).
 * No counterpart in the reference. */
int rnet_model_train_step_distill(rnet_model* m, const int* d_inputs, const int* d_teacher_idx,
                                  const float* d_teacher_logits, const float* d_teacher_lse,
                                  const int* d_targets, const float* d_row_weight, int batch,
                                  int seq_len, int top_k, float temperature, float soft_weight,
                                  float hard_weight, float lr, float grad_clip,
                                  float* d_loss_sum);
/* Same as rnet_model_train_step with host token buffers; copies in, steps,
 * copies the loss sum out and waits for it. */
int rnet_model_train_step_host(rnet_model* m, const int* h_inputs, const int* h_targets,
                               int batch, int seq_len, float lr, float grad_clip,
                               float* h_loss_sum);
/* Device pointers to the last cached forward's top-k indices / weights of a
 * layer ([batch*seq_len, top_k], reference slot order). */
int rnet_model_topk(rnet_model* m, int layer, const int** d_idx, const float** d_w);
/* Host copies of the same ([batch*seq_len*top_k] each; waits for the stream). */
int rnet_model_topk_host(rnet_model* m, int layer, int* h_idx, float* h_w, size_t n);
int rnet_model_save(rnet_model* m, const char* path);
/* Checkpoint without stalling training (no counterpart in the reference,
 * whose save() blocks on a device-to-host copy): the parameters are
 * snapshotted on the model stream (a device copy ordered after all queued
 * work, so a later SGD step cannot change what is saved), then copied to
 * pinned host memory on a side stream and written by a host thread in the
 * reference byte layout. rnet_model_save_wait joins the write and returns
 * its status; a second save_async first waits for the previous one. Costs
 * one parameter-sized device buffer and one pinned host buffer. */
int rnet_model_save_async(rnet_model* m, const char* path);
int rnet_model_save_wait(rnet_model* m);
int rnet_model_load_weights(rnet_model* m, const char* path);
/* Wait for the model stream and report any device error word bits. */
int rnet_model_synchronize(rnet_model* m);

/* Per-kernel-class timing with CUDA events on the model stream. Classes
 * (index order): gemm, scan_fwd, scan_bwd, conv_fwd, conv_bwd, rms_fwd,
 * rms_bwd, slot_gather, slot_sparse_bwd, embed, cross_entropy, sgd, other.
 * read() fills arrays of n_kinds entries: total ms, algorithmic FLOPs and
 * bytes, number of timed launch groups; reset clears the record. */
#define RNET_PROFILE_KINDS 13
int rnet_model_profile_enable(rnet_model* m, int on);
int rnet_model_profile_read(rnet_model* m, double* ms, double* flops, double* bytes,
                            long long* launches, int n_kinds, int reset);

/* ------------------------------------------------------------------ decode
 * Recurrent inference with the O(1) per-stream state (per layer: the last 14
 * causal-conv inputs and the MinGRU h; 15 * d_model floats per layer per
 * stream). n_streams advance in lock step. The reference has no counterpart
 * (its `generate()` is declared, never defined; `infer` recomputes the whole
 * prefix per token). A decoder is destroyed before its model. */
typedef struct rnet_decoder rnet_decoder;
int rnet_decoder_create(rnet_model* m, int n_streams, rnet_decoder** out);
int rnet_decoder_destroy(rnet_decoder* d);
/* d_tokens [n_streams, seq_len] (device). Runs the chunked-scan forward and
 * keeps the state; the last-position logits / argmax become available. Also
 * folds the slot keys / values with proj_q / proj_out for the decode steps,
 * from the weights of this moment: prefill again after changing weights. */
int rnet_decoder_prefill(rnet_decoder* d, const int* d_tokens, int seq_len);
/* Prefill for a beam search: d_tokens [n_streams / beams, seq_len], one prompt
 * per sequence; its `beams` streams (in a row) all start from its state. */
int rnet_decoder_prefill_beams(rnet_decoder* d, const int* d_tokens, int seq_len, int beams);
/* Beam search of n_steps (1..2^30) tokens from the current logits and states:
 * n_streams / beams sequences of `beams` streams each, beams 1..32 dividing
 * n_streams; a sequence starts from its first stream. Per step: rnet_beam_select
 * on the logits, rnet_beam_reorder of the recurrent states by the parents, one
 * decode step. eos = -1: no token ends a beam. Outputs (device) as
 * rnet_beam_backtrack with n_steps: d_sequences [n_streams, n_steps],
 * d_lengths and d_scores [n_streams], ranked per sequence by
 * score / length^length_alpha. use_graph = 1 replays one captured CUDA graph per
 * step. Asynchronous on the model stream, except that it waits when the record
 * of steps has to grow. Afterwards the streams hold the beams of the last
 * selection, unranked, and rnet_decoder_step(d, NULL) feeds their last tokens; the
 * logits are still those that the last selection chose from. A search without a
 * prefill, step or generation since the last one is refused (RNET_ERR_ARG). */
int rnet_decoder_beam_search(rnet_decoder* d, int beams, int n_steps, int eos, float length_alpha,
                             int* d_sequences, int* d_lengths, float* d_scores, int use_graph);
/* One token per stream: d_tokens [n_streams] (device) or NULL to feed back
 * the previous argmax. */
int rnet_decoder_step(rnet_decoder* d, const int* d_tokens);
/* n_steps greedy steps (fed back on the device); d_out [n_steps, n_streams]
 * (device, may be NULL). use_graph = 1 replays one captured CUDA graph per step. */
int rnet_decoder_generate(rnet_decoder* d, int n_steps, int* d_out, int use_graph);
/* Next-token rule of prefill / step / generate: temperature <= 0 = greedy
 * argmax (default); otherwise the reference infer loop's temperature + top-p
 * sampling (src/main.cpp:327-360: softmax at `temperature`, probabilities
 * sorted descending, smallest prefix reaching `top_p`, sample within it),
 * computed on the device. The uniform for stream m at the sampled token's
 * position pos is a splitmix64 hash of (seed, m, pos), so runs are
 * reproducible and independent of batching; it is not the reference CLI's
 * std::mt19937 stream. Ties in probability order by token id. */
int rnet_decoder_set_sampling(rnet_decoder* d, float temperature, float top_p,
                              unsigned long long seed);
/* Device pointers to the current logits [n_streams, vocab] and next tokens
 * [n_streams], and the state buffer with its size per stream in floats. */
int rnet_decoder_outputs(rnet_decoder* d, const float** d_logits, const int** d_next);
/* Host copies of the same (either pointer may be NULL); waits for the stream. */
int rnet_decoder_outputs_host(rnet_decoder* d, float* h_logits, int* h_next);
int rnet_decoder_state(rnet_decoder* d, float** d_state, size_t* floats_per_stream);

/* ------------------------------------------------------------------ data parallel
 * The reference's include/dist.h:12-36 over NCCL (loaded at run time). */
int rnet_dist_unique_id(unsigned char uid[128]);
int rnet_dist_create(int rank, int world, int local_rank, const unsigned char uid[128],
                     int timeout_ms, rnet_dist** out);
int rnet_dist_destroy(rnet_dist* d);
int rnet_dist_allreduce_sum(rnet_dist* d, float* d_buf, size_t count, void* stream);
int rnet_dist_group_start(rnet_dist* d);
int rnet_dist_group_end(rnet_dist* d);
/* File rendezvous of the 128-byte unique id (reference src/dist.cpp:53-93):
 * write = write "<path>.tmp" then rename (readers never see a partial file);
 * read = poll until a complete file appears, RNET_ERR_TIMEOUT after
 * timeout_ms, RNET_ERR_IO on a short/unreadable file. Host only. */
int rnet_dist_uid_file_write(const char* path, const unsigned char uid[128]);
int rnet_dist_uid_file_read(const char* path, int timeout_ms, unsigned char uid[128]);
/* Attach (or detach with NULL): backward then all-reduces gradient buckets
 * as they complete and step() uses the reference's world-size scaling. */
int rnet_model_set_dist(rnet_model* m, rnet_dist* d);

#ifdef __cplusplus
}
#endif

#endif /* RNET_CAPI_H */
