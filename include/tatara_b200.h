/*
 * tatara_b200 — C ABI of the sm_100a NNUE training step.
 *
 * The library replaces the device side of tatara's trainer backends.  One handle
 * corresponds to one `GpuTrainer` (LayerStack) or `SimpleGpuTrainer` (Simple) of the
 * reference; the entry points below are what an `impl TrainerBackend` over FFI binds.
 * Paths in the comments are relative to the reference project root.
 *
 * Conventions (the reference's, kept):
 *  - every call returns TB_OK or a negative error code; nothing aborts.  The text of
 *    the last error is available from tb_last_error() (bins/nnue_train/src/trainer_common.rs:313
 *    maps such errors to io::Error::other).
 *  - one caller thread per handle (the reference's trainers are Send, not Sync).
 *  - pageable host input arrays are copied into the library's own pinned ring before a
 *    call returns, so the caller may reuse them immediately (InputUploadRing,
 *    bins/nnue_train/src/trainer_common.rs:1041-1097).  Page-locked arrays (tb_host_alloc,
 *    cudaHostAlloc) are read by the copy engine directly: keep batch k untouched until
 *    tb_train_step(k+1) returns, the recycling rule of the reference's training loop
 *    (crates/nnue-train/src/trainer.rs:925-994).
 *  - tb_train_step reports the loss sum of the PREVIOUS step; the first call reports 0.0
 *    (AsyncLossRing, bins/nnue_train/src/trainer_common.rs:909-976).
 */
#ifndef TATARA_B200_H
#define TATARA_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TB_OK 0
#define TB_ERR_INVALID_ARGUMENT (-1)
#define TB_ERR_CUDA (-2)
#define TB_ERR_OUT_OF_MEMORY (-3)
#define TB_ERR_UNSUPPORTED (-4)
#define TB_ERR_NCCL (-5)
#define TB_ERR_NO_DEVICE (-6)
#define TB_ERR_TIMEOUT (-7) /* a data-parallel step did not finish within the deadline: a peer is gone; the handle is poisoned */

enum { TB_ARCH_LAYERSTACK = 0, TB_ARCH_SIMPLE = 1 };
/* SimpleActivation (bins/nnue_train/src/trainer_simple.rs): Pairwise is the FT-output pairwise product of the LayerStack
 * net (the L1 input is then ft_out wide instead of 2 * ft_out); L1 and L2 are CReLU then */
enum { TB_ACT_CRELU = 0, TB_ACT_SCRELU = 1, TB_ACT_PAIRWISE = 2 };
/* crates/nnue-train/src/optimizer.rs:32-37 OptimizerKind */
enum { TB_OPT_RANGER = 0, TB_OPT_RADAM = 1, TB_OPT_ADAMW = 2 };
/* bins/nnue_train/src/cli.rs:623-638 precision flags; --all-optim sets all four.  Accepted for LayerStack with l1_out of 8,
 * 16 or 32 (TB_ERR_UNSUPPORTED otherwise).  TF32: the L1 forward product runs on the tensor cores with TF32 operands (the
 * reference: cuBLAS TF32 tensor-op mode); FT_FP16: fp16 forward table; FT_FP16_OUT (needs FT_FP16): fp16 pre-activations and
 * fp16 FT gradient rows scaled by 2^14 * batch and clamped to +-65504; FP16_OPT_STATE: fp16 moments of the FT table, scaled
 * by 2^28 / 2^40 (bins/nnue_train/src/arch.rs:72-93).  Uploads and downloads stay fp32. */
enum { TB_PREC_TF32 = 1, TB_PREC_FT_FP16 = 2, TB_PREC_FT_FP16_OUT = 4, TB_PREC_FP16_OPT_STATE = 8 };
enum { TB_LOSS_SIGMOID = 0, TB_LOSS_WRM = 1 };

typedef struct tb_trainer tb_trainer;

/*
 * Construction parameters.  Replaces the argument lists of GpuTrainer::new
 * (bins/nnue_train/src/trainer_layerstack.rs:781-796) and SimpleGpuTrainer::new
 * (bins/nnue_train/src/trainer_simple.rs:392-402).  The feature set is passed by its
 * dimensions (crates/shogi-features/src/feature_set.rs:1031-1038) instead of by name.
 */
#define TB_DP_NCCL 0
#define TB_DP_PEER_COPY 1
#define TB_DP_PEER_KERNEL 2

typedef struct tb_config {
    int32_t struct_size;    /* sizeof(tb_config) of the caller */
    int32_t device;         /* CUDA device ordinal */
    int32_t arch;           /* TB_ARCH_* */
    int32_t batch_capacity; /* largest n_pos a step may carry; multiple of 16 */
    int32_t ft_in;          /* N: real feature rows */
    int32_t piece_inputs;   /* pi: rows per king bucket (N = king_buckets * pi) */
    int32_t ft_factorize;   /* 1: pi virtual rows are trained on top (train rows = N + pi) */
    int32_t max_active;     /* A: slots per position and perspective */
    int32_t ft_out;         /* F: multiple of 128 (bins/nnue_train/src/arch.rs:13-19) */
    int32_t l1_out;         /* LayerStack: includes the skip output; Simple: hidden 1 */
    int32_t l2_out;
    int32_t num_buckets;    /* LayerStack: 2..9; ignored for Simple */
    int32_t activation;     /* Simple: TB_ACT_* (CReLU, SCReLU, Pairwise); LayerStack is always pairwise CReLU */
    int32_t optimizer;      /* TB_OPT_* */
    int32_t precision;      /* bit mask of TB_PREC_* */
    float wd_ft, wd_dense, wd_bias;                /* OptimGroupConfig, trainer_layerstack.rs:640-705 */
    float lr_mult_ft, lr_mult_dense, lr_mult_bias; /* Simple uses wd_ft / lr_mult_ft for every group */
    int32_t world_size;     /* data-parallel ranks (1 = single GPU, NCCL not loaded) */
    int32_t rank;
    uint8_t nccl_unique_id[128]; /* from tb_nccl_unique_id() on rank 0, same bytes on every rank */
    int32_t nccl_ctas;      /* > 0: this handle's communicator is created by ncclCommInitRankConfig with minCTAs = maxCTAs =
                               this value (a fixed channel count); 0: ncclCommInitRank, NCCL chooses.  Algorithm, protocol and
                               NVLS have no per-communicator setting in NCCL: they are the application's NCCL_ALGO, NCCL_PROTO
                               and NCCL_NVLS_ENABLE, which this library neither sets nor changes. */
    int32_t dp_exchange;    /* TB_DP_NCCL (0): the gradient parts are summed by ncclAllReduce.  TB_DP_PEER_COPY (1): ranks of
                               one node, one process each: reduce-scatter and all-gather by the copy engines over peer
                               mappings (CUDA IPC) with stream memory operations as signals and a small summing kernel in
                               rank order; NCCL then only carries the start-up handshake and batches off the fast path.
                               TB_DP_PEER_KERNEL (2): the same signals, the data moved by one kernel per part that reads every
                               rank's shard over the peer mappings, sums in rank order and stores the sum to every rank */
} tb_config;

/* nnue_train::trainer::LossKind, crates/nnue-train/src/trainer.rs:75-95 */
typedef struct tb_loss {
    int32_t kind; /* TB_LOSS_* */
    float scale;  /* sigmoid: 1 / scale_param */
    float nnue2score, in_scaling, in_offset, target_offset, target_scaling;
    float pow_exp, qp_asymmetry, weight_boost_w1, weight_boost_w2;
} tb_loss;

/* BatchData, bins/nnue_train/src/trainer_common.rs:142-151.  All pointers are HOST memory. */
typedef struct tb_batch {
    int32_t n_pos;               /* multiple of 16, <= batch_capacity */
    const int32_t* stm_indices;  /* [n_pos, A]; slots >= nnz are ignored; out-of-range values are skipped */
    const int32_t* nstm_indices; /* [n_pos, A] */
    const int32_t* nnz;          /* [n_pos], shared by both perspectives */
    const int32_t* bucket_idx;   /* [n_pos] LayerStack; NULL for Simple */
    const float* score;          /* [n_pos] raw centipawns */
    const float* wdl;            /* [n_pos] 0 / 0.5 / 1 */
    float per_pos_norm;          /* 0 selects the reference's 1 / (n_pos * world_size) */
} tb_batch;

/* ---- life cycle ------------------------------------------------------------------ */
int tb_create(const tb_config* cfg, tb_trainer** out);
/* synchronises both streams before freeing (Drop, trainer_layerstack.rs:335-347) */
void tb_destroy(tb_trainer* t);
/* text of the last error on this handle; with NULL, of the last failed tb_create on this thread */
const char* tb_last_error(const tb_trainer* t);

/* ---- parameter groups -------------------------------------------------------------
 * Names and order follow raw_ckpt_group_sources / uniform_optim_group_layout
 * (trainer_layerstack.rs:740-762): ft_w, ft_b, l1_w, l1_b, l1_shared_weight,
 * l1_shared_bias, l2_w, l2_b, l3_w, l3_b; Simple: ft_w, ft_b, l1_w ([2 * ft_out, l1]; Pairwise [ft_out, l1]), l1_b, l2_w,
 * l2_b, l3_w, l3_b.  Initial weights always come from the host (init.rs or a checkpoint). */
int tb_num_groups(const tb_trainer* t);
const char* tb_group_name(const tb_trainer* t, int group);
int64_t tb_group_len(const tb_trainer* t, const char* name);
/* NULL pointers are skipped.  Re-derives the forward table (factorizer fold) like
 * sync_ft_forward_weights.  Moments are true f32 values (MomentBuf::to_host_f32,
 * trainer_common.rs:89-126). */
int tb_upload_group(tb_trainer* t, const char* name, const float* w, const float* m, const float* v,
                    const float* slow, int64_t len);
int tb_download_group(tb_trainer* t, const char* name, float* w, float* m, float* v, float* slow, int64_t len);
int tb_get_step_count(const tb_trainer* t, uint64_t* step_count);
int tb_set_step_count(tb_trainer* t, uint64_t step_count);

/* ---- the step (trait TrainerBackend, crates/nnue-train/src/trainer.rs:273-374) ------ */
/* train_step -> GpuTrainer::step (trainer_layerstack.rs:1885) / SimpleGpuTrainer::step
 * (trainer_simple.rs:742).  n_pos == 0 returns loss 0 without work. */
int tb_train_step(tb_trainer* t, const tb_batch* batch, float lr, float wdl_lambda, const tb_loss* loss,
                  double* loss_prev);
/* train_step fed with PackedSfenValue records instead of extracted indices: `psv` is n_pos 40-byte records in HOST
 * memory (crates/shogi-format/src/packed_sfen.rs:251-271); 40 bytes per position cross the bus and the work of the
 * reference's dataloader workers (decode, feature extraction of both perspectives, kingrank9 bucket, score and wdl:
 * crates/nnue-train/src/dataloader.rs:444-500, 1303-1407) runs on the device on the copy stream, overlapped with the
 * previous step.  feature_set as in tb_psv_extract; it must be the set the trainer was created for.  The step is
 * bit-identical to tb_train_step on the batch tb_psv_extract returns for the same records.  per_pos_norm is the
 * reference's 1 / (n_pos * world_size). */
int tb_train_step_psv(tb_trainer* t, int feature_set, const uint8_t* psv, int n_pos, float lr, float wdl_lambda,
                      const tb_loss* loss, double* loss_prev);
/* flush_pending_loss: the lagged loss of the last step, then re-arms the ring */
int tb_flush_pending_loss(tb_trainer* t, double* loss);
/* validate_step -> GpuTrainer::validate (trainer_layerstack.rs:1963): forward + loss only, no state
 * change; net_output receives n_pos values */
int tb_validate_step(tb_trainer* t, const tb_batch* batch, float wdl_lambda, const tb_loss* loss,
                     double* sum_sq_err, float* net_output);
/* read_fp16_clamp_count (trainer.rs:368-373): fp16 FT gradient elements that hit the clamp, and elements written, since
 * the handle was created; both 0 without TB_PREC_FT_FP16_OUT */
int tb_read_fp16_clamp_count(tb_trainer* t, uint64_t* clamps, uint64_t* elems);

/* ---- device-resident batches -------------------------------------------------------
 * A batch may be uploaded once into one of TB_NUM_SLOTS device slots and stepped on
 * repeatedly (the reference's native-bench runs a fixed in-memory batch,
 * bins/nnue_train/src/native_bench.rs:550-576). */
#define TB_NUM_SLOTS 4 /* slots 0..2 are the caller's; the last one is the library's scratch batch */
int tb_stage_batch(tb_trainer* t, int slot, const tb_batch* batch);
int tb_train_step_staged(tb_trainer* t, int slot, float lr, float wdl_lambda, const tb_loss* loss,
                         double* loss_prev);

/* ---- diagnostics used by the parity tests ------------------------------------------- */
/* forward + backward (+ gradient all-reduce when world_size > 1) without the optimizer; returns this
 * step's own loss sum, synchronously */
int tb_forward_backward(tb_trainer* t, const tb_batch* batch, float wdl_lambda, const tb_loss* loss,
                        double* loss_now);
/* runs the optimizer on the gradients currently held (completes a tb_forward_backward) */
int tb_apply_optimizer(tb_trainer* t, float lr);
/* gradient of a group after tb_forward_backward */
int tb_download_grad(tb_trainer* t, const char* name, float* grad, int64_t len);
/* an intermediate of the last step in the caller's position order: "ft_stm", "ft_nstm", "combined",
 * "l1_total", "net_output", "dy", "dl1_total", "dft_stm", "dft_nstm", "comb" */
int tb_read_buffer(tb_trainer* t, const char* name, float* out, int64_t len);

/* ---- timing --------------------------------------------------------------------------
 * CUDA events on the library's compute stream.  With profiling on, every kernel phase of a step is
 * bracketed by events; tb_profile_read returns the accumulated milliseconds and launch counts. */
int tb_timer_start(tb_trainer* t);
int tb_timer_stop(tb_trainer* t, float* elapsed_ms);
int tb_profile_enable(tb_trainer* t, int on);
int tb_profile_num_phases(const tb_trainer* t);
int tb_profile_read(tb_trainer* t, int phase, const char** name, double* total_ms, int64_t* launches);
int tb_profile_reset(tb_trainer* t);
/* kernels launched by this handle since creation */
int64_t tb_launch_count(const tb_trainer* t);
int tb_synchronize(tb_trainer* t);

/* ---- FT kernels alone (the reference's per-kernel microbenchmark shapes) ---------------
 * Device-resident single-perspective runs of the three FT kernels on caller-provided HOST data.
 * forward: out[b, :] = sum of table rows (native_kernels.cu:162 sparse_ft_forward);
 * backward: grad[f, :] = sum of dft rows whose position lists f (native_kernels.cu:1630-1840);
 * adam: one fused AdamW + clamp pass (native_kernels.cu:1291 radam_step with scalars (1, 1)).
 * `iters` launches are timed with events; results are copied back when the output pointer is not NULL. */
int tb_ft_forward_bench(int device, const float* table, const int32_t* indices, const int32_t* nnz,
                        int batch, int ft_out, int ft_in, int max_active, int iters, float* out, float* ms_per_iter);
int tb_ft_backward_bench(int device, const float* dft, const int32_t* indices, const int32_t* nnz,
                         int batch, int ft_out, int ft_in, int max_active, int iters, float* grad, float* ms_per_iter);
int tb_adam_clamp_bench(int device, float* w, float* m, float* v, const float* grad, int64_t n, float lr,
                        float decay, float min_w, float max_w, int iters, float* ms_per_iter);

/* The three FT kernels on DEVICE-resident data, one perspective (the reference's microbenchmark protocol:
 * a fixed in-memory batch, warm-up, timed launches, bins/nnue_train/src/native_bench.rs:550-576,
 * docs/native-cuda-benchmark.md:11-33).  Only the index lists come from the host; table, incoming gradient rows and
 * moments are filled on the device.  Every launch group is timed with its own pair of CUDA events; with flush_l2 a
 * 256 MB buffer is written before each one.  fwd / bwd / adam: the generic kernels (L2 gather; global inverse index +
 * per-row sums; AdamW with the +-32767/127 clamp).  With rows_per_slice > 0 and king-sliced lists (every row of a
 * position inside one slice of rows_per_slice table rows) the slice-resident kernels of the training step are timed
 * too, sorts and plans included; otherwise those two fields are negative. */
typedef struct tb_ft_microbench_result {
    float fwd_ms, bwd_ms, adam_ms;
    float fwd_slice_ms, bwd_slice_ms;
    int32_t iters;
} tb_ft_microbench_result;
int tb_ft_microbench(int device, const int32_t* indices, const int32_t* nnz, int batch, int ft_out, int ft_in,
                     int rows_per_slice, int max_active, int iters, int flush_l2, tb_ft_microbench_result* out);

/* ---- FT weight gradient without any allocation -------------------------------------------
 * No counterpart in the reference (its trainers allocate their workspace in the constructor).
 * For hosts that must not allocate device memory once they run — a framework whose allocator owns the
 * whole GPU, a process with a fixed memory plan — this variant of the FT backward keeps the working
 * memory of the inverse index and of the long-list partial sums in a static device array inside the
 * library (about 20.5 MB per GPU, held until exit) and calls no cudaMalloc / cudaFree.  ALL pointers are DEVICE memory owned by the caller;
 * the work is enqueued on `stream` (a cudaStream_t, NULL = default stream) and not synchronised.
 * Limits: ft_in <= TB_STATIC_SCRATCH_MAX_FT_IN and batch * max_active <= TB_STATIC_SCRATCH_MAX_PAIRS;
 * beyond them the call fails and writes the reason to err (may be NULL).  Calls share the one array:
 * never let two of them overlap on a GPU.  The first call on a device resolves the array's address;
 * issue it before any stream capture.  d_dft and d_grad must be 16-byte aligned (rows move as 128-bit
 * vectors).  Same kernels and same summation order as tb_ft_backward_bench (lists of more than 4096 entries are
 * summed in parts of 4096), so the two agree bit for bit. */
#define TB_STATIC_SCRATCH_MAX_FT_IN 131072
#define TB_STATIC_SCRATCH_MAX_PAIRS 655360
int tb_ft_backward_static_scratch(const float* d_dft, const int32_t* d_indices, const int32_t* d_nnz, int batch,
                                  int ft_out, int ft_in, int max_active, float* d_grad, void* stream, char* err,
                                  size_t err_len);

/* ---- operators on the caller's device tensors ----------------------------------------------
 * No counterpart in the reference.  What a trainer with learned buckets needs beside the step: normalised rows in
 * front of a gate, the choice of a bucket (expert) per row with a balance loss, the rows sorted by expert and back, rows of a table by token with the table's gradient, and the
 * matrix optimizer of hidden weights.  ALL tensor pointers are DEVICE memory of the
 * current device, owned by the caller; the work is enqueued on `stream` (a cudaStream_t, NULL = default stream) and not synchronised; nothing is
 * allocated and nothing is kept between calls, so calls on different streams may overlap as long as each has its own workspace.
 * A call's kernels may be started while the kernel ahead of them on the stream is ending; they wait for its end before they touch memory.
 * A failed call returns a code, writes the reason to err (may be NULL) and launches nothing when an argument is refused.
 * Workspaces: tb_*_workspace returns the bytes a call of these sizes needs on the current device (negative: invalid sizes).
 * Row strides count elements; they may exceed the row (columns of a wider buffer).  Where a function says so, a result may be the memory of an
 * input element by element (same address and strides): y that of x, dx of dy or x, dlogits of the logits, an orthogonalised matrix of its input, the Muon step's of what they replace.
 * Any other element in common with an input or another result is refused.  Sums are fp32 in a fixed order
 * (repeated calls agree bit for bit), results are rounded once to the tensors' type. */
enum { TB_TYPE_F32 = 0, TB_TYPE_F16 = 1, TB_TYPE_BF16 = 2 };

/* y = (x - mean) * rstd * weight + bias per row of n; weight, bias (fp32 [n]) may be NULL (1 and 0), mean, rstd (fp32 [rows], kept
 * for the backward pass) may be NULL.  x and y have the same type. */
int tb_layer_norm_forward(const void* d_x, int64_t x_stride, const float* d_weight, const float* d_bias, float eps, int type, int64_t rows,
                          int n, void* d_y, int64_t y_stride, float* d_mean, float* d_rstd, void* stream, char* err, size_t err_len);
int64_t tb_layer_norm_backward_workspace(int64_t rows, int n);
/* dx, and dweight, dbias (fp32 [n], written, not added to; either may be NULL, both NULL need no workspace).  dx may be dy or x. */
int tb_layer_norm_backward(const void* d_dy, int64_t dy_stride, const void* d_x, int64_t x_stride, const float* d_mean, const float* d_rstd,
                           const float* d_weight, int type, int64_t rows, int n, void* d_dx, int64_t dx_stride, float* d_dweight,
                           float* d_dbias, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len);

/* The k largest of every row's `experts` logits (1 <= k <= min(experts, 16), experts <= 1024), ties to the lowest index, with
 * the gates, per-expert counts and losses.  mask: NULL or a byte per row, 0 = the row takes no part.  A logit of -inf forbids its
 * expert; a NaN counts as the largest and makes its row's gates and the losses NaN.  Writes index [rows, k] (-1 where no expert is left),
 * gate [rows, k] (softmax over the chosen with renormalise, else over the row; 0 beside -1), counts [experts], rows [1] (rows N that
 * take part and have an expert), prob_mean [experts] (P: the mean softmax over those), losses [2]: the balance loss
 * experts * sum_e counts_e / (N k) * P_e and the z loss, the mean squared log-sum-exp (0 where N is 0). */
int64_t tb_route_forward_workspace(int64_t rows, int experts);
int tb_route_forward(const void* d_logits, int64_t stride, int type, int64_t rows, int experts, int k, int renormalise, const uint8_t* d_mask,
                     int32_t* d_index, float* d_gate, int32_t* d_counts, int32_t* d_rows, float* d_prob_mean, float* d_losses, void* d_work,
                     int64_t work_bytes, void* stream, char* err, size_t err_len);
/* The logits' gradient from dgate [rows, k] and dlosses [2] (the gradients of the gates and of the two losses; either may be NULL: zero) and
 * what the forward call wrote; the choice and the counts are constants.  Rows that take no part get zeros.  dlogits may be the logits. */
int tb_route_backward(const void* d_logits, int64_t stride, int type, int64_t rows, int experts, int k, int renormalise, const uint8_t* d_mask,
                      const int32_t* d_index, const float* d_gate, const float* d_dgate, const int32_t* d_counts, const int32_t* d_rows,
                      const float* d_dlosses, void* d_dlogits, int64_t dstride, void* stream, char* err, size_t err_len);

/* Newton-Schulz orthogonalisation of every matrix of a batch: X = x / (|x| + eps) (Frobenius norm), then `steps` (1 .. 32) times
 * X = (a I + b A + c A^2) X with A = X X^T taken over the shorter side; coefficients = {a, b, c} on the HOST.  x and out have the same
 * type; x_batch and out_batch are the strides between matrices.  Coefficients for which a singular value of at most 1
 * could grow beyond 4 (or |a| + |b| s^2 + |c| s^4 beyond 31) are refused.  64-bit throughout where the shorter side is at most 64.  Above: fp32 and fp16
 * are products of 22-bit operands (elements below 2^-25 of the norm to 2^-47 of it), bf16 of 11-bit ones (2^-36; 1e-3 of the result beside its own rounding: give
 * fp32 for more), with fp32 sums.  A matrix with an infinity or a NaN comes out NaN. */
int64_t tb_orthogonalise_workspace(int type, int batch, int rows, int cols);
int tb_orthogonalise(const void* d_x, int64_t x_batch, int64_t x_stride, int type, int batch, int rows, int cols, int steps,
                     const float* coefficients, float eps, void* d_out, int64_t out_batch, int64_t out_stride, void* d_work,
                     int64_t work_bytes, void* stream, char* err, size_t err_len);

/* The Muon step of a batch of weight matrices, all contiguous [batch, rows, cols]: m' = beta m + g; u = nesterov ? g + beta m' : m';
 * w' = clamp(w (1 - lr weight_decay) - lr scale orthogonalise(u), -clip, clip).  w, m and their results are fp32 (each result may be its
 * input's memory and must not overlap any other tensor), g any type. */
typedef struct tb_muon {
    int32_t struct_size; /* sizeof(tb_muon) of the caller */
    int32_t steps, nesterov;
    float a, b, c, eps;  /* of the orthogonalisation */
    float lr, beta, weight_decay, scale, clip; /* clip: INFINITY for none */
} tb_muon;
int64_t tb_muon_step_workspace(int batch, int rows, int cols);
int tb_muon_step(const tb_muon* cfg, const float* d_w, const float* d_m, const void* d_g, int g_type, int batch, int rows, int cols,
                 float* d_w_out, float* d_m_out, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len);

/* Root-mean-square norm on a residual stream: h = x + residual, y = h * rstd * weight per row of n, rstd = 1 / sqrt(mean(h^2) + eps).  The norm is that of the fp32 sum;
 * d_h receives the sum rounded to the tensors' type, for the next layer and the backward pass.  residual may be NULL (h is x; d_h must be NULL then), weight (fp32 [n]), d_h and d_rstd
 * (fp32 [rows], kept for the backward pass) may be NULL.  All rows have the same type.  y and h may each be the memory of x or of the residual (not the same one); the
 * backward pass takes h, which is x where there is no residual: not for a y in its place.  Rows go by 16-byte accesses where they all start on such a boundary and n is a multiple, and the weight starts on 16 bytes for
 * fp32 and 32 bytes for 16-bit rows (backward 16); otherwise by single elements, at two to three times the time. */
int tb_rms_norm_forward(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const float* d_weight, float eps, int type,
                        int64_t rows, int n, void* d_y, int64_t y_stride, void* d_h, int64_t h_stride, float* d_rstd, void* stream, char* err, size_t err_len);
/* The same with y in 8 bits: q [rows, n] (e4m3 bytes) and scale [rows, ceil(n / group)] (fp32, contiguous) with y ~ q * scale; group: 32, 64, 128 columns, or n (a scale
 * per row).  scale = max(largest |y| of the group / 448, 2^-126), q = y / scale rounded to nearest.  A group whose y holds an infinity or a NaN has q NaN throughout.  q overlaps no other
 * tensor; h may be the memory of x or of the residual. */
int tb_rms_norm_quantised(const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const float* d_weight, float eps, int type,
                          int64_t rows, int n, int group, void* d_q, int64_t q_stride, float* d_scale, void* d_h, int64_t h_stride, float* d_rstd, void* stream,
                          char* err, size_t err_len);
int64_t tb_rms_norm_backward_workspace(int64_t rows, int n);
/* dx (the gradient of x and of the residual alike) from dy, h and rstd, plus dresidual, the gradient that arrives at h from elsewhere (may be NULL), and dweight (fp32 [n], written, not
 * added to; NULL: not wanted, and no workspace).  dx may be the memory of dy, h or dresidual. */
int tb_rms_norm_backward(const void* d_dy, int64_t dy_stride, const void* d_h, int64_t h_stride, const float* d_rstd, const float* d_weight,
                         const void* d_dresidual, int64_t dresidual_stride, int type, int64_t rows, int n, void* d_dx, int64_t dx_stride, float* d_dweight,
                         void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len);

/* Rows to their experts and back.  index [rows, k] holds the experts of every row (as tb_route_forward writes it: 1 <= k <= 16, experts <= 1024; anything outside
 * [0, experts) is no choice).  tb_expert_order sorts the choices by expert, within one by row and then choice: expert e has the places [offsets[e], offsets[e + 1]), a multiple of
 * `align` of them; position [rows, k] is the place of every choice (-1: none), source [slots] the choice r * k + j of every place, -1 at the places that align or missing choices
 * leave over.  slots is what tb_expert_slots returns (negative: invalid sizes), enough for any choice; offsets [experts + 1] ends at the last place in use. */
int64_t tb_expert_slots(int64_t rows, int k, int experts, int align);
int64_t tb_expert_order_workspace(int64_t rows, int k, int experts);
int tb_expert_order(const int32_t* d_index, int64_t rows, int k, int experts, int align, int32_t* d_position, int32_t* d_source, int64_t slots,
                    int32_t* d_offsets, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len);
/* out [slots, n]: x[r] at the places of its choices, zeros at places without a choice.  position and source as tb_expert_order wrote them (a place outside [0, slots) is skipped); n <= 2^30
 * here and below.  The results of these three overlap no other tensor, the gaps between rows of a wider buffer included. */
int tb_dispatch_forward(const void* d_x, int64_t x_stride, int type, int64_t rows, int n, int k, const int32_t* d_position, const int32_t* d_source,
                        int64_t slots, void* d_out, int64_t out_stride, void* stream, char* err, size_t err_len);
/* out[r] = sum over j of gate[r, j] * y[position[r, j]]; a choice without a place adds nothing, whatever its gate.  gate (fp32 [rows, k]) NULL: 1, which makes this the gradient
 * of tb_dispatch_forward. */
int tb_combine_forward(const void* d_y, int64_t y_stride, int type, int64_t slots, int64_t rows, int n, int k, const int32_t* d_position, const float* d_gate,
                       void* d_out, int64_t out_stride, void* stream, char* err, size_t err_len);
/* dy [slots, n] (zeros at places without a choice) and dgate [rows, k] (0 without a place) of tb_combine_forward from the gradient dout [rows, n] of its result. */
int tb_combine_backward(const void* d_dout, int64_t dout_stride, const void* d_y, int64_t y_stride, int type, int64_t slots, int64_t rows, int n, int k,
                        const int32_t* d_position, const int32_t* d_source, const float* d_gate, void* d_dy, int64_t dy_stride, float* d_dgate, void* stream,
                        char* err, size_t err_len);

/* out [count, n] = scale * table[token]; tokens are 32- or 64-bit whole numbers (token_bytes 4 or 8), one outside [0, rows) has a row of zeros.  out and table have the same type;
 * results overlap no other tensor, gaps included. */
int tb_embedding_forward(const void* d_tokens, int token_bytes, int64_t count, const void* d_table, int64_t table_stride, int type, int64_t rows, int n, float scale,
                         void* d_out, int64_t out_stride, void* stream, char* err, size_t err_len);
int64_t tb_embedding_backward_workspace(int64_t count, int64_t rows, int n);
/* dtable [rows, n] = scale * the sum of dy over the tokens of every row, written (not added to), zeros where there are none; of type dtable_type: that of dy, or TB_TYPE_F32.  The
 * 16-byte pieces of memory that hold a row of dy may be read whole. */
int tb_embedding_backward(const void* d_dy, int64_t dy_stride, int type, const void* d_tokens, int token_bytes, int64_t count, int64_t rows, int n, float scale,
                          void* d_dtable, int64_t dtable_stride, int dtable_type, void* d_work, int64_t work_bytes, void* stream, char* err, size_t err_len);

/* ---- inputs: PackedSfenValue records -> step inputs, on the device ---------------------
 * Decodes 40-byte records (crates/shogi-format/src/packed_sfen.rs:387-448) and extracts the active
 * feature indices of both perspectives (crates/shogi-features/src/feature_set.rs:655-808), the
 * kingrank9 bucket (crates/shogi-features/src/kingrank9.rs:11-24), score and wdl
 * (crates/nnue-train/src/dataloader.rs:444-500).  feature_set: 0 halfkp, 4 halfka-hm-merged.
 * All pointers are HOST memory; bucket may be NULL. */
int tb_psv_extract(int device, int feature_set, const uint8_t* psv, int64_t n_records, int32_t* stm_indices,
                   int32_t* nstm_indices, int32_t* nnz, int32_t* bucket, float* score, float* wdl);
/* seeded synthetic PackedSfenValue records (host): full 40-piece sets, see the generator's comment */
int tb_psv_synthesize(uint64_t seed, int64_t n_records, uint8_t* psv_out);
/* encodes one position (host); arrays as in the decoder's board: piece type 0..14, colour 0/1 */
int tb_psv_encode(const uint8_t* board_pt, const uint8_t* board_color, const uint8_t* hand_black7,
                  const uint8_t* hand_white7, int side_to_move, int black_king_sq, int white_king_sq,
                  int score, int ply, int result, uint8_t* psv40_out);

/* ---- weight initialisation (host) --------------------------------------------------------
 * The reference's deterministic sampler (crates/nnue-train/src/init.rs:111-210), for callers that have
 * no Rust host to draw the initial weights.  dist: 0 zeroed, 1 uniform.  scale_kind: 0 absolute half
 * width, 1 sqrt(scale_value / fan_in). */
int tb_init_sample(float* out, int64_t n, int64_t num_buckets, int64_t fan_in, int dist, int scale_kind,
                   float scale_value, int per_bucket_repeat, uint64_t seed);

/* page-locked host memory for step inputs (pinned_host_alloc of the reference's runtime,
 * crates/cuda-native-runtime/src/runtime.rs:701-769).  Any thread may call.  tb_host_free returns at once; a freed block is
 * handed out again only after everything that any GPU of this process has been given to do by then, on the
 * caller's streams as on the library's.  Freed blocks are kept for later calls: at most 256 MB of them, back to the system
 * when 256 allocations have not matched them or when memory runs out.  Likewise tb_psv_extract keeps up to four sets of
 * buffers per GPU, each of at most 96 MB of device memory and as much page-locked memory, until memory runs out. */
int tb_host_alloc(void** out, size_t bytes);
int tb_host_free(void* p);

/* ---- data parallel ---------------------------------------------------------------------- */
/* rank 0 creates the id, every rank passes the same bytes in tb_config.nccl_unique_id */
int tb_nccl_unique_id(uint8_t out[128]);

int tb_device_count(void);
const char* tb_version(void);

#ifdef __cplusplus
}
#endif
#endif
