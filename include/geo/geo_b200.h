/*
 * geo/geo_b200.h -- additive C ABI of libgeo_b200.so (no reference header has
 * these symbols; each block names the reference code whose semantics it
 * batches).
 *
 *  1. Trainer: a parameter multivector and its optimizer state resident on one
 *     GPU, trained by the fused full cycle (forward -> residual -> 0.5|r|^2 ->
 *     parameter VJP -> optimizer) in one streaming pass per minibatch.
 *     Optimizer semantics are the reference V8 graph runtime's for the graph
 *     x*w (or w*x) -> add(., scale(t, -1)) -> squared_norm
 *     (reference src/full_cycle_v8.c:942-1041): g = sum_s grad_s * scale,
 *     SGD w -= lr g, Adam m = b1 m + (1-b1) g, v = b2 v + (1-b2) g^2,
 *     w -= lr (m / (1-b1^t)) / (sqrt(v / (1-b2^t)) + eps); transactional
 *     (nothing changes when any candidate value is non-finite).
 *  2. Data parallelism: one process (or thread) per GPU; each rank trains on
 *     its own slice of the global batch and the per-rank gradient/loss record
 *     (2^n + 8 doubles) is all-gathered over NCCL and summed in rank order, so
 *     every rank applies the identical update to its replica.
 *  3. Pairwise products with both operands varying per element (reference
 *     src/operator_kernel.c:412-539, geo_operator_gp_f64 and its JVP/VJP),
 *     float64, plus a float32 build of the forward.
 *  4. Sparse fixed-multivector operators over a batch (reference
 *     src/operator_kernel.c:191-334, geo_operator_apply_*_f64 and VJPs).
 *  5. Layer operators over rows of coefficients (no counterpart in the
 *     reference): layer norm, dropout, the two fused with a residual, and
 *     rotary positions, each with its VJP; float64, float32, bfloat16, float16.
 *
 * All device-pointer calls are asynchronous on the given stream; host-pointer
 * calls are synchronous. Arrays are sample-major [batch][2^n].
 */
#ifndef GEO_B200_H
#define GEO_B200_H

#include "geo/operator_kernel.h"

#include <cuda_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GEO_B200_ABI_VERSION 0x00010000u

/* Status of the per-multivector geo_operator_*_f64 calls (geo/operator_kernel.h)
 * when the GPU call itself fails (no device, launch or copy error); the
 * reference's geo_operator_status_t has no such value. */
#define GEO_OPERATOR_B200_DEVICE_FAILURE 100

typedef enum {
    GEO_B200_OK = 0,
    GEO_B200_INVALID_ARGUMENT = 1,
    GEO_B200_UNSUPPORTED_DIMENSION = 2,
    GEO_B200_NUMERIC_FAILURE = 3,
    GEO_B200_RUNTIME_FAILURE = 4,
    GEO_B200_ALLOCATION_FAILURE = 5,
    GEO_B200_COMM_FAILURE = 6,
    GEO_B200_TIMEOUT = 7
} geo_b200_status_t;

typedef enum {
    GEO_B200_OPTIMIZER_SGD = 1,  /* same values as GEO_V8_OPTIMIZER_* */
    GEO_B200_OPTIMIZER_ADAM = 2
} geo_b200_optimizer_t;

typedef struct {
    uint32_t optimizer;      /* geo_b200_optimizer_t */
    double learning_rate;
    double beta1;
    double beta2;
    double epsilon;
} geo_b200_optimizer_config_t;

typedef struct geo_b200_trainer geo_b200_trainer_t;
typedef struct geo_b200_comm geo_b200_comm_t;

uint32_t geo_b200_abi_version(void);
const char *geo_b200_status_string(geo_b200_status_t status);

/* ---- 1. trainer ------------------------------------------------------- */

/* Creates the trainer on the current CUDA device. initial_parameter is a host
 * array of 2^dimension doubles; moments start at zero and the step count at 0
 * (like geo_v8_set_value on a PARAMETER, reference src/full_cycle_v8.c:559-563). */
geo_b200_status_t geo_b200_trainer_create(geo_b200_trainer_t **trainer, uint8_t dimension,
                                          const int8_t *signature, int parameter_on_left,
                                          const double *initial_parameter,
                                          const geo_b200_optimizer_config_t *config);
void geo_b200_trainer_destroy(geo_b200_trainer_t *trainer);

/* One training step on a device-resident minibatch (inputs/targets
 * [batch][2^n] in device memory). gradient_scale multiplies the summed
 * gradient (1/global_batch gives the mean, as geo_v8_optimizer_step's
 * gradient_scale). Asynchronous on `stream`; numeric status accumulates until
 * geo_b200_trainer_sync. With a communicator attached, every rank must call it
 * the same number of times. */
geo_b200_status_t geo_b200_trainer_step_device(geo_b200_trainer_t *trainer, const double *device_inputs,
                                               const double *device_targets, size_t batch,
                                               double gradient_scale, cudaStream_t stream);

/* The two halves of a step, for gradient accumulation over micro-batches
 * (the batched form of geo_v8_backward(accumulate) + geo_v8_optimizer_step):
 * accumulate adds the micro-batch's gradient and loss sums to the trainer's
 * running record; apply reduces the record across ranks (when a communicator
 * is attached), applies the optimizer with `gradient_scale` and clears the
 * record. step_device == accumulate + apply. */
geo_b200_status_t geo_b200_trainer_accumulate_device(geo_b200_trainer_t *trainer, const double *device_inputs,
                                                     const double *device_targets, size_t batch,
                                                     cudaStream_t stream);
geo_b200_status_t geo_b200_trainer_apply(geo_b200_trainer_t *trainer, double gradient_scale, cudaStream_t stream);

/* Same step from host (pageable or pinned) buffers: copies in, trains, waits,
 * and returns the step's status; *loss_sum receives sum_s 0.5 |r_s|^2 over
 * the global batch (may be NULL). */
geo_b200_status_t geo_b200_trainer_step_host(geo_b200_trainer_t *trainer, const double *inputs,
                                             const double *targets, size_t batch, double gradient_scale,
                                             double *loss_sum);

/* Waits for all queued steps (bounded by the communicator timeout when one is
 * attached) and returns the first failure since the previous sync.
 * *loss_sum (may be NULL) receives the last step's global loss sum. */
geo_b200_status_t geo_b200_trainer_sync(geo_b200_trainer_t *trainer, double *loss_sum);

/* Host copies of the parameter and Adam moments (any pointer may be NULL). */
geo_b200_status_t geo_b200_trainer_get_state(geo_b200_trainer_t *trainer, double *parameter,
                                             double *first_moment, double *second_moment,
                                             uint64_t *step_count);
/* Replaces the parameter and resets moments and step count. */
geo_b200_status_t geo_b200_trainer_set_parameter(geo_b200_trainer_t *trainer, const double *parameter);
/* Restores a full optimizer state (checkpoint resume). */
geo_b200_status_t geo_b200_trainer_set_state(geo_b200_trainer_t *trainer, const double *parameter,
                                             const double *first_moment, const double *second_moment,
                                             uint64_t step_count);
/* Kernel family used by the trainer's streaming pass.
 *  CAYLEY: the 2^n x 2^n sign-folded Cayley matrix on FP64 FMA units (any n).
 *  REPRESENTATION: a D x D real matrix representation of Cl(p,q) (D = 8 or 16
 *    for n = 5, 6) on FP64 tensor cores; S*D*D instead of 4^n multiply-adds.
 *  AUTO (default): REPRESENTATION where available for n >= 5, else CAYLEY.
 * Both are parity-checked against the reference to 1e-12. */
typedef enum {
    GEO_B200_ALGORITHM_AUTO = 0,
    GEO_B200_ALGORITHM_CAYLEY = 1,
    GEO_B200_ALGORITHM_REPRESENTATION = 2
} geo_b200_algorithm_t;

/* Selects the kernel family; INVALID_ARGUMENT when REPRESENTATION is not
 * available for this algebra and side. */
geo_b200_status_t geo_b200_trainer_set_algorithm(geo_b200_trainer_t *trainer, geo_b200_algorithm_t algorithm);
/* The family the next step will use (never AUTO). */
geo_b200_algorithm_t geo_b200_trainer_algorithm(const geo_b200_trainer_t *trainer);

/* Device pointer to the resident parameter (2^n doubles). */
const double *geo_b200_trainer_device_parameter(const geo_b200_trainer_t *trainer);

/* ---- 1b. fixed-parameter forward on a chosen kernel family ------------ */

/* outputs[s] = inputs[s] * parameter (parameter_on_left = 0) or
 * parameter * inputs[s]: the product of geo_batch_gp_cuda_planned_forward_f64
 * (reference src/batch_gp_cuda.cu:252-286, src/batch_gp.c:107-161) without a
 * plan object. All arrays are device memory; asynchronous on `stream`;
 * reports argument and launch errors only, like the device ABI.
 *  CAYLEY: the 2^n x 2^n sign-folded Cayley matrix on FP64 FMA units (any n).
 *  REPRESENTATION (n = 5, 6; inputs and outputs 16-byte aligned): X' = P x,
 *    Y' = X' W' on FP64 tensor cores, y = P^-1 Y'. Equal to the Cayley product
 *    up to rounding (within 1e-12 relative); INVALID_ARGUMENT where it is not
 *    available.
 *  AUTO: REPRESENTATION where available, else CAYLEY; bit-identical to
 *    geo_batch_gp_cuda_planned_forward_f64 on the same arrays (the same kernel).
 * device_parameter may be geo_b200_trainer_device_parameter(). Outputs may be
 * the inputs (in place) but must not overlap them otherwise. A non-finite
 * input coefficient makes every output coefficient of its sample non-finite
 * on both families, as in the reference (which of Inf and NaN may differ). */
geo_b200_status_t geo_b200_forward_f64(uint8_t dimension, const int8_t *signature, int parameter_on_left,
                                       geo_b200_algorithm_t algorithm, const double *device_inputs,
                                       const double *device_parameter, double *device_outputs, size_t batch_size,
                                       cudaStream_t stream);

/* ---- 2. data parallelism ---------------------------------------------- */

#define GEO_B200_COMM_ID_BYTES 128

/* Rank 0 creates the id and shares the bytes with the other ranks out of band. */
geo_b200_status_t geo_b200_comm_unique_id(unsigned char id[GEO_B200_COMM_ID_BYTES]);
/* Collective over `world` ranks; uses the current CUDA device. Returns
 * GEO_B200_TIMEOUT if the ranks have not all joined within timeout_ms. */
geo_b200_status_t geo_b200_comm_create(geo_b200_comm_t **comm, int rank, int world,
                                       const unsigned char id[GEO_B200_COMM_ID_BYTES], int timeout_ms);
void geo_b200_comm_destroy(geo_b200_comm_t *comm);
/* Aborts in-flight collectives (use after a peer failed). */
void geo_b200_comm_abort(geo_b200_comm_t *comm);
geo_b200_status_t geo_b200_trainer_attach_comm(geo_b200_trainer_t *trainer, geo_b200_comm_t *comm);

/* ---- 2b. batched V8 programs ------------------------------------------ */

/* One optimizer step of a compiled V8 program over a device-resident
 * minibatch, equal to: geo_v8_zero_grad; for every sample s: set the INPUT
 * node `input_node` to inputs[s] and the TARGET node `target_node` to
 * targets[s], geo_v8_forward, geo_v8_backward(accumulate = s != 0); then
 * geo_v8_optimizer_step(optimizer, ..., gradient_scale)
 * (reference src/full_cycle_v8.c:569-1041, per sample). Any compiled program:
 *   - the graph gp = GEOMETRIC_PRODUCT(input, w) or (w, input);
 *     neg = SCALE(target, -1); residual = ADD(gp, neg) (either order);
 *     loss = SQUARED_NORM(residual), with `w` its only PARAMETER and no
 *     constraint, runs as one fused streaming pass on the tensor cores;
 *   - every other graph (all node kinds, constraints, several parameters,
 *     STATE leaves held fixed across the batch) runs per sample on the GPU with
 *     the reference's arithmetic, gradients summed over the batch.
 * target_node may be GEO_V8_INVALID_NODE (device_targets then unused) for the
 * general path. Parameters and Adam moments are updated in place
 * (transactional), the step count advances, gradients are cleared; node
 * values other than the parameters are left unchanged. *loss_sum (may be
 * NULL) receives the sum over the batch of the loss node's value.
 * Synchronous; returns geo_v8_status_t values (declared in
 * geo/full_cycle_v8.h, passed here as int to keep this header independent). */
int geo_b200_v8_batch_train_step(void *program, uint32_t input_node, uint32_t target_node,
                                 const double *device_inputs, const double *device_targets, size_t batch,
                                 int optimizer, double learning_rate, double beta1, double beta2, double epsilon,
                                 double gradient_scale, double *loss_sum);

/* Batched inference: for every sample s, set `input_node` to inputs[s], run
 * geo_v8_forward and write the value of `output_node` to outputs[s]
 * ([batch][2^n] device arrays). Every other leaf keeps its value; node values
 * in the program are not modified. Synchronous; geo_v8_status_t values. */
int geo_b200_v8_batch_forward(void *program, uint32_t input_node, const double *device_inputs, size_t batch,
                              uint32_t output_node, double *device_outputs);

/* The graph runtime's exp and tanh (TANH nodes; SIGMOID nodes through exp,
 * reference src/full_cycle_v8.c:181-190, 651) are correctly rounded (round to
 * nearest, ties to even) for every binary64 argument: a table-driven
 * double-double evaluation with Ziv's rounding test, and an exact 256-bit
 * fixed-point evaluation when that test cannot decide. The reference calls the
 * C library's exp and tanh; wherever those are correctly rounded the results
 * agree bit for bit, elsewhere the value here is the closer one.
 * geo_b200_cr_math_f64 applies one of them to `count` doubles of a device array
 * (device_out may equal device_in), asynchronously on `stream`; the *_EXACT_PATH
 * values run the fixed-point evaluation for every argument it covers (a check
 * of that path). */
typedef enum {
    GEO_B200_CR_EXP = 0,
    GEO_B200_CR_TANH = 1,
    GEO_B200_CR_EXP_EXACT_PATH = 2,
    GEO_B200_CR_TANH_EXACT_PATH = 3
} geo_b200_cr_function_t;
geo_b200_status_t geo_b200_cr_math_f64(int function, const double *device_in, double *device_out, size_t count,
                                       cudaStream_t stream);

/* ---- 2c. parameter VJP that allocates nothing -------------------------- */

/* This entry point has no counterpart in the reference.
 *
 * Same result as geo_batch_gp_cuda_parameter_vjp_f64 (the summed parameter
 * cotangent of the batched geometric product), for callers that cannot call
 * cudaMalloc: hosts whose own allocator has reserved the device memory up
 * front (so a further cudaMalloc fails), latency-critical loops that must not
 * take the implicit device synchronisation of cudaMalloc/cudaFree, and plugin
 * hosts that forbid device allocation after start-up. It takes no plan (a plan
 * upload allocates); dimension and signature are given directly, all arrays
 * are device memory supplied by the caller, and the call is asynchronous on
 * `stream`.
 *
 * Its reduction scratch is one fixed array compiled into the library
 * (GEO_B200_NOALLOC_RECORDS records of 576 bytes, about 1.2 MB), which every
 * GPU that loads the library holds until the process exits. That bounds the
 * batch: batch_size must not exceed GEO_B200_NOALLOC_MAX_BATCH (131072
 * samples, any dimension); larger batches are rejected with
 * GEO_B200_INVALID_ARGUMENT before anything is launched. The first call on each
 * device looks up the array's device address (a one-time set-up per device,
 * repeated only if the device's context was recreated, e.g. after
 * cudaDeviceReset); make that first call before any stream capture. All calls share the one
 * array and every call overwrites the part it uses, so calls whose kernels
 * overlap on the GPU (different streams without ordering) race; order them on
 * one stream. */
#define GEO_B200_NOALLOC_RECORDS 2048u
#define GEO_B200_NOALLOC_MAX_BATCH 131072u
geo_b200_status_t geo_b200_parameter_vjp_noalloc_f64(uint8_t dimension, const int8_t *signature,
                                                     int parameter_on_left, const double *device_inputs,
                                                     const double *device_output_cotangents, size_t batch_size,
                                                     double *device_parameter_cotangent, cudaStream_t stream);

/* ---- 3. pairwise products (both operands vary per element) ------------ */

/* out[s] = left[s] * right[s]. */
geo_b200_status_t geo_b200_pairwise_gp_f64(uint8_t dimension, const int8_t *signature, const double *device_left,
                                           const double *device_right, double *device_out, size_t batch,
                                           cudaStream_t stream);
/* Per-element VJP: left_bar[s], right_bar[s] from out_bar[s]
 * (reference src/operator_kernel.c:494-539). Either output may be NULL. */
geo_b200_status_t geo_b200_pairwise_gp_vjp_f64(uint8_t dimension, const int8_t *signature,
                                               const double *device_left, const double *device_right,
                                               const double *device_out_cotangent, double *device_left_cotangent,
                                               double *device_right_cotangent, size_t batch, cudaStream_t stream);
/* Per-element JVP (reference src/operator_kernel.c:449-492). */
geo_b200_status_t geo_b200_pairwise_gp_jvp_f64(uint8_t dimension, const int8_t *signature,
                                               const double *device_left, const double *device_right,
                                               const double *device_left_tangent, const double *device_right_tangent,
                                               double *device_out_tangent, size_t batch, cudaStream_t stream);
/* float32 build of the forward. When left_even_compact is non-zero, `left`
 * holds only the 2^(n-1) even-grade coefficients of each element, in
 * increasing blade order (compact storage); otherwise 2^n dense values. */
geo_b200_status_t geo_b200_pairwise_gp_f32(uint8_t dimension, const int8_t *signature, const float *device_left,
                                           int left_even_compact, const float *device_right, float *device_out,
                                           size_t batch, cudaStream_t stream);

/* Bounded waits of the n = 6 TMA pairwise kernels (no counterpart in the
 * reference, whose products run on the CPU). Every wait of those kernels on a
 * load or on a ring stage gives up after a fixed number of polls; a CTA whose
 * wait gave up stops loading, waits (bounded) for its loads in flight, writes
 * NaN into every output row it had not stored and ends, so the context stays
 * usable. This call synchronizes the current device and reports how many
 * give-ups (one per CTA of the float32 kernel, one per warp of the float64
 * kernel) were recorded since the last reset (*count); reset != 0 clears it.
 * Returns GEO_B200_TIMEOUT when the count is non-zero. */
geo_b200_status_t geo_b200_pairwise_wait_failures(unsigned *count, int reset);
/* Self-test of that failure path: runs the float64 (precision 64) or float32
 * (precision 32) TMA pairwise kernel over `batch` rows of device_out with no
 * load issued at all, so every first wait runs out after wait_limit polls with
 * no copy in flight. Synchronizes the stream; returns GEO_B200_TIMEOUT when the
 * kernel reported its give-up (device_out then holds NaN in every row). */
geo_b200_status_t geo_b200_pairwise_wait_selftest(int precision, void *device_out, size_t batch,
                                                  uint32_t wait_limit, cudaStream_t stream);

/* ---- 4. sparse fixed-multivector plans over a batch ------------------- */

/* out[s] = plan applied to in[s] (integer coefficients of the plan). */
geo_b200_status_t geo_b200_sparse_apply_f64(const geo_operator_plan_i32_t *plan, const double *device_in,
                                            double *device_out, size_t batch, cudaStream_t stream);
/* Coefficients replaced by real parameters[term_count] (device array). */
geo_b200_status_t geo_b200_sparse_apply_parametric_f64(const geo_operator_plan_i32_t *plan,
                                                       const double *device_parameters, const double *device_in,
                                                       double *device_out, size_t batch, cudaStream_t stream);
/* in_bar[s] = M^T out_bar[s] (integer plan). */
geo_b200_status_t geo_b200_sparse_apply_vjp_f64(const geo_operator_plan_i32_t *plan,
                                                const double *device_out_cotangent, double *device_in_cotangent,
                                                size_t batch, cudaStream_t stream);
/* Parametric VJP: per-element input cotangents (may be NULL) and the
 * parameter cotangents summed over the batch (term_count doubles, device). */
geo_b200_status_t geo_b200_sparse_apply_parametric_vjp_f64(const geo_operator_plan_i32_t *plan,
                                                           const double *device_parameters, const double *device_in,
                                                           const double *device_out_cotangent,
                                                           double *device_in_cotangent,
                                                           double *device_parameter_cotangent, size_t batch,
                                                           cudaStream_t stream);

/* ---- 5. layer operators over rows of coefficients ---------------------- */

/* What a model of several layers does between its products, on arrays of
 * `rows` rows of `cols` values in device memory (a row: the coefficients of
 * one or several multivectors, or of any other layer). None of these has a
 * counterpart in the reference. Common to all of section 5:
 *   - asynchronous on `stream`, which belongs to the current device, as does
 *     every array (device memory, managed memory, or pinned host memory);
 *     other pointers are refused with GEO_B200_INVALID_ARGUMENT, as is an array
 *     that is not aligned to its value type, before anything is launched. Only
 *     argument and launch errors are reported. Nothing is allocated and nothing
 *     is kept between calls; calls may be captured into a CUDA graph, and made by
 *     several host threads at once.
 *   - strides are in values; 0 means packed rows, otherwise stride >= cols.
 *     Nothing is written between the rows; what lies there may be read along
 *     with its neighbours and has no effect.
 *   - an output may be the same array (pointer and stride) as an input of the
 *     call that it overwrites; arrays must not overlap otherwise.
 *   - arithmetic and sums are float64 for GEO_B200_F64 and float32 otherwise
 *     (epsilon, the scale of dropout and the amplitude of rotary positions are
 *     rounded to it, and what leaves its range is infinite), rounded once (to
 *     nearest, ties to even) to the array's type. Sums are taken in a fixed
 *     order: the same call gives the same bits.
 *   - infinities and NaN reach every output that depends on them. */
typedef enum {
    GEO_B200_F64 = 1,
    GEO_B200_F32 = 2,
    GEO_B200_BF16 = 3,
    GEO_B200_F16 = 4
} geo_b200_type_t;

#define GEO_B200_LAYER_MAX_COLS 16777216u  /* 2^24 values a row */
#define GEO_B200_LAYER_MAX_ROWS 4294967296ull

/* Layer norm over each row: with mean m and variance v (divided by cols),
 *   rstd = 1 / sqrt(v + epsilon),  y = (x - m) rstd weight + bias.
 * The mean over a multivector's coefficients, and a weight and bias for each, do
 * not commute with rotors: on rows of multivectors this is a norm of channels. */
typedef struct {
    uint32_t type;              /* geo_b200_type_t of x, y and their cotangents */
    uint32_t parameter_type;    /* of weight, bias and their cotangents: `type`, or F32 for the 16-bit types */
    size_t rows, cols;          /* 1 .. GEO_B200_LAYER_MAX_ROWS, 1 .. GEO_B200_LAYER_MAX_COLS */
    size_t x_stride, y_stride, y_cotangent_stride, x_cotangent_stride;
    double epsilon;             /* finite, >= 0 */
} geo_b200_layer_norm_config_t;

/* weight, bias (cols values each) may be NULL: 1 and 0. mean and rstd (rows
 * values each, float64 for GEO_B200_F64, else float32; what the VJP needs) may
 * be NULL. The statistics of a row are taken about its own mean (no difference
 * of large squares). */
geo_b200_status_t geo_b200_layer_norm(const geo_b200_layer_norm_config_t *config, const void *device_x,
                                      const void *device_weight, const void *device_bias, void *device_y,
                                      void *device_mean, void *device_rstd, cudaStream_t stream);

/* Bytes of device workspace of the VJP of `config` on the current device (the
 * partial sums of the weight's and the bias's cotangent); 0 for a config that
 * the VJP would refuse. */
size_t geo_b200_layer_norm_vjp_workspace(const geo_b200_layer_norm_config_t *config);

/* VJP: with xh = (x - mean) rstd, g = y_bar weight (means over the row),
 *   x_bar = rstd (g - mean(g) - xh mean(g xh)),
 *   weight_bar = sum over the rows of y_bar xh, bias_bar = sum of y_bar.
 * Any of the three outputs may be NULL, not all; outputs are overwritten.
 * workspace: geo_b200_layer_norm_vjp_workspace bytes, 16-byte aligned, not
 * needed (may be NULL) when weight_bar and bias_bar are both NULL. Calls that
 * may overlap on the GPU, captured graphs among them, need a workspace each. */
geo_b200_status_t geo_b200_layer_norm_vjp(const geo_b200_layer_norm_config_t *config, const void *device_x,
                                          const void *device_weight, const void *device_mean,
                                          const void *device_rstd, const void *device_y_cotangent,
                                          void *device_x_cotangent, void *device_weight_cotangent,
                                          void *device_bias_cotangent, void *device_workspace,
                                          size_t workspace_bytes, cudaStream_t stream);

/* Rows of more than 4096 values, up to 32768 (half of that in float64) lie in a
 * cluster of thread blocks that send one another their sums. Every wait for those
 * gives up after a fixed number of polls (seconds, where a row takes microseconds;
 * it cannot happen unless a block of the cluster failed). A warp whose wait gave up
 * waits and sends no more: what it writes from then on is NaN (its part of the rows,
 * their statistics, its columns of weight_bar and bias_bar), and so it is for the
 * cluster's other warps from their next row on. The call ends and the context stays
 * usable.
 * Self-test of that path, float32, packed and 16-byte aligned rows that fill their
 * cluster (cols a multiple of 8192 that is a power of two), without a weight: layer
 * norm of device_x into device_out (device_y_cotangent NULL, mean and rstd
 * written), or its VJP (device_out: x_bar; mean and rstd read). In round `round` of
 * the rows that a cluster takes one after another, its last block sends nothing;
 * waits give up after wait_limit polls, 1 .. 2^22. Later rows, and the column sums,
 * are NaN. */
geo_b200_status_t geo_b200_layer_norm_wait_selftest(
    const geo_b200_layer_norm_config_t *config, const void *device_x, const void *device_y_cotangent, void *device_out,
    void *device_mean, void *device_rstd, void *device_weight_cotangent, void *device_bias_cotangent,
    void *device_workspace, size_t workspace_bytes, uint32_t round, uint32_t wait_limit, cudaStream_t stream);

/* Dropout, y = [residual +] keep x / (1 - rate), whose mask is computed from a
 * counter and never stored. What is kept or dropped as one is a unit of
 * 2^dimension consecutive values of a row: a single value (dimension 0), or a
 * whole multivector, which keeps a layer of multivectors equivariant (dropping
 * coefficients one by one does not commute with a rotor).
 * Unit u = (row cols + col) >> dimension (strides do not enter) draws 16 bits:
 * half u & 1 (0: the low one) of word (u & 7) / 2 of the block
 *   Philox4x32-10(counter = {lo, hi of u >> 3, lo, hi of the offset}, key = {lo, hi of the seed})
 * (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC
 * 2011), and is kept when they are >= T = rate in steps of 2^-16, rounded to
 * the nearest (ties to even); x is scaled by 65536 / (65536 - T), so the mean
 * over masks is x at the rounded rate, and T = 65536 drops everything.
 * A dropped unit gives 0 (or the residual) whatever its x holds, NaN included. */
typedef struct {
    uint32_t type;              /* geo_b200_type_t of all arrays */
    uint32_t dimension;         /* 0 .. 6; cols is a multiple of 2^dimension */
    size_t rows, cols;
    size_t x_stride, residual_stride, y_stride, y_cotangent_stride, x_cotangent_stride;
    double rate;                /* 0 .. 1 */
    uint64_t seed;
    uint64_t offset;            /* another mask for each call of a training run */
} geo_b200_dropout_config_t;

/* residual may be NULL. device_offset may be NULL; else the value it points to
 * when the kernel runs is added to config->offset (modulo 2^64), so that a
 * captured graph draws another mask at each replay. */
geo_b200_status_t geo_b200_dropout(const geo_b200_dropout_config_t *config, const void *device_x,
                                   const void *device_residual, const uint64_t *device_offset, void *device_y,
                                   cudaStream_t stream);
/* x_bar = keep y_bar / (1 - rate), of the forward's seed and offset (the
 * residual's cotangent is y_bar itself). */
geo_b200_status_t geo_b200_dropout_vjp(const geo_b200_dropout_config_t *config, const uint64_t *device_offset,
                                       const void *device_y_cotangent, void *device_x_cotangent,
                                       cudaStream_t stream);

/* Both in one pass over a residual stream: z = residual + dropout(x) and
 * y = layer_norm(z). z is dropout's y (dropout->y_stride) and layer norm's x
 * (norm->x_stride, the same value); type, rows and cols agree. The statistics
 * and y are taken from z before it is rounded to its type. */
geo_b200_status_t geo_b200_residual_dropout_layer_norm(
    const geo_b200_layer_norm_config_t *norm, const geo_b200_dropout_config_t *dropout, const void *device_x,
    const void *device_residual, const uint64_t *device_offset, const void *device_weight, const void *device_bias,
    void *device_z, void *device_y, void *device_mean, void *device_rstd, cudaStream_t stream);
/* VJP from y_bar (norm->y_cotangent_stride) and, where z is used further on,
 * its own cotangent z_bar (dropout->y_cotangent_stride; may be NULL):
 *   residual_bar = layer_norm_vjp(y_bar) + z_bar  (norm->x_cotangent_stride),
 *   x_bar = keep residual_bar / (1 - rate)        (dropout->x_cotangent_stride).
 * Any output may be NULL, not all. Workspace as geo_b200_layer_norm_vjp, from
 * geo_b200_layer_norm_vjp_workspace(norm). */
geo_b200_status_t geo_b200_residual_dropout_layer_norm_vjp(
    const geo_b200_layer_norm_config_t *norm, const geo_b200_dropout_config_t *dropout,
    const uint64_t *device_offset, const void *device_z, const void *device_weight, const void *device_mean,
    const void *device_rstd, const void *device_y_cotangent, const void *device_z_cotangent,
    void *device_residual_cotangent, void *device_x_cotangent, void *device_weight_cotangent,
    void *device_bias_cotangent, void *device_workspace, size_t workspace_bytes, cudaStream_t stream);

/* Rotary positions: the vector of a token's head is turned, pair of
 * coordinates by pair, by the rotor of its position,
 *   (a, b) -> amplitude (a cos t - b sin t, a sin t + b cos t), t = position f_i,
 * which makes the product of two turned vectors a function of the difference
 * of their positions. Pairs i < rotary_dim / 2 are coordinates (2i, 2i + 1)
 * (INTERLEAVED) or (i, i + rotary_dim / 2) (HALF); coordinates from rotary_dim
 * on are copied. f_i = base^(-2i / rotary_dim) radians per position, and for
 * contexts longer than a model was trained on:
 *   LINEAR: f_i / factor;
 *   BASE:   base replaced by base factor^(d / (d - 2)), d = rotary_dim > 2
 *           (d = 2 has the single frequency 1 and is left alone);
 *   BANDED: f_i k_i + f_i / factor (1 - k_i), k_i = (r_i - low) / (high - low)
 *           clamped to [0, 1], r_i = original_length f_i / (2 pi) the turns
 *           that pair i makes over the original context. */
typedef enum { GEO_B200_ROTARY_INTERLEAVED = 0, GEO_B200_ROTARY_HALF = 1 } geo_b200_rotary_layout_t;
typedef enum {
    GEO_B200_ROTARY_SCALING_NONE = 0,
    GEO_B200_ROTARY_SCALING_LINEAR = 1,
    GEO_B200_ROTARY_SCALING_BASE = 2,
    GEO_B200_ROTARY_SCALING_BANDED = 3
} geo_b200_rotary_scaling_t;
typedef enum { GEO_B200_I32 = 1, GEO_B200_I64 = 2 } geo_b200_position_type_t;

#define GEO_B200_ROTARY_MAX_DIM 256u

typedef struct {
    uint32_t layout;            /* geo_b200_rotary_layout_t */
    uint32_t rotary_dim;        /* even, 2 .. GEO_B200_ROTARY_MAX_DIM */
    double base;                /* finite, > 0 */
    uint32_t scaling;           /* geo_b200_rotary_scaling_t */
    double factor;              /* finite, > 0; unless NONE */
    double original_length;     /* BANDED: finite, > 0 */
    double low_rotations;       /* BANDED: finite, < high_rotations */
    double high_rotations;
    double amplitude;           /* finite */
} geo_b200_rotary_config_t;

/* Filled by geo_b200_rotary_plan_init (host code, no GPU), owned by the caller:
 * turns per position of each pair, as the sum of two float64, so that the
 * angle of a far position keeps its accuracy (an error of at most
 * 2^-63 |position| turns times the pair's own turns per position, next to
 * float64 rounding). */
typedef struct {
    uint32_t abi_version;       /* GEO_B200_ABI_VERSION */
    uint32_t layout;
    uint32_t rotary_dim;
    uint32_t reserved;
    double amplitude;
    double turns[GEO_B200_ROTARY_MAX_DIM / 2];
    double turns_low[GEO_B200_ROTARY_MAX_DIM / 2];
} geo_b200_rotary_plan_t;

geo_b200_status_t geo_b200_rotary_plan_init(geo_b200_rotary_plan_t *plan, const geo_b200_rotary_config_t *config);

/* Arrays [batch][tokens][heads][head_dim] with any strides between batches,
 * tokens and heads (0: packed, in that order); the head_dim values of a head
 * are adjacent, and heads must not overlap. Queries and keys that lie side by
 * side in one projection are one call. */
typedef struct {
    uint32_t type;              /* geo_b200_type_t of x and y */
    uint32_t position_type;     /* geo_b200_position_type_t */
    size_t batch, tokens, heads, head_dim;  /* >= 1; rotary_dim <= head_dim <= 65536 */
    size_t x_batch_stride, x_token_stride, x_head_stride;
    size_t y_batch_stride, y_token_stride, y_head_stride;
    size_t position_batch_stride;  /* 0: every sequence has the same positions */
    int64_t first_position;     /* position of token t is first_position + t when no positions are given */
} geo_b200_rotary_shape_t;

/* device_positions (may be NULL) holds the position of token t of sequence b
 * at [b position_batch_stride + t]; positions may be negative, in any order and
 * repeated, |position| <= 2^31. */
geo_b200_status_t geo_b200_rotary(const geo_b200_rotary_plan_t *plan, const geo_b200_rotary_shape_t *shape,
                                  const void *device_x, const void *device_positions, void *device_y,
                                  cudaStream_t stream);
/* x_bar from y_bar: the reversed rotor. The shape's x strides describe
 * device_y_cotangent, its y strides device_x_cotangent. */
geo_b200_status_t geo_b200_rotary_vjp(const geo_b200_rotary_plan_t *plan, const geo_b200_rotary_shape_t *shape,
                                      const void *device_y_cotangent, const void *device_positions,
                                      void *device_x_cotangent, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif
