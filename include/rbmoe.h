/*
 * rbmoe.h — C ABI of the MI355X (gfx950) mixture-of-experts layer.
 *
 * Drop-in boundary for RustingBrain's `MoeLayer`: the forward pass with the two
 * auxiliary losses (reference src/moe.rs:203-341), the backward pass
 * (src/moe.rs:348-489) and the block's RMSNorm and residual add either side of
 * the layer (src/transformer_block.rs:216-222, 257-263); and, on their own,
 * operators of a training or serving step around it: a sub-layer joined to the
 * residual stream, orthogonalised weight updates, and the attention half of a
 * block with a paged cache of keys and values.  The reference
 * has no FFI seam for this layer; each entry point below names the reference
 * interface it stands in for, so that a Rust `extern "C"` block can bind them
 * one to one.  Plain pointers and sizes only.  Every function returns an
 * `rbmoe_status`; none throws, aborts or falls back to a CPU path.
 *
 * Matrices are row-major and contiguous, exactly like the reference `Matrix`
 * (src/matrix.rs:13-18).  A `Linear` weight is `[out_features, in_features]`
 * (src/param.rs:620-633): router `[E, d]`, gate/up `[F, d]`, down `[d, F]`.
 */
#ifndef RBMOE_H
#define RBMOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Mirrors the `NetworkError` variants that can leave this path
 * (reference src/network.rs:19-83). */
typedef enum rbmoe_status {
    RBMOE_OK = 0,
    RBMOE_INVALID_INPUT = 1,      /* NetworkError::InvalidInput{expected, actual}      */
    RBMOE_INVALID_CONFIG = 2,     /* NetworkError::InvalidConfig(String)               */
    RBMOE_DEVICE_ERROR = 3,       /* NetworkError::Cuda(String): a HIP call failed     */
    RBMOE_BACKEND_UNAVAILABLE = 4,/* NetworkError::CudaFeatureDisabled: no usable GPU  */
    RBMOE_MEMORY_BUDGET = 5,      /* NetworkError::CudaMemoryBudget{estimated, budget} */
    RBMOE_OUT_OF_MEMORY = 6,      /* NetworkError::CudaOutOfMemory{requested, free}    */
    RBMOE_UNSUPPORTED = 7,        /* NetworkError::UnsupportedCuda(String)             */
    RBMOE_NULL_POINTER = 8        /* a required pointer argument was NULL              */
} rbmoe_status;

typedef enum rbmoe_dtype {
    RBMOE_F32 = 0,
    RBMOE_BF16 = 1,  /* raw 16-bit patterns, round-to-nearest-even from f32 */
    RBMOE_I8 = 2     /* weights only: symmetric int8 + one f32 scale per output row */
} rbmoe_dtype;

/* Which weight of the layer; the order is the reference's parameter traversal
 * (src/moe.rs:516-525 with src/ffn.rs:126-131). */
typedef enum rbmoe_weight {
    RBMOE_W_ROUTER = 0,       /* [E, d]              Router.projection  (src/moe.rs:91-100) */
    RBMOE_W_GATE = 1,         /* [F, d]  per expert  SwiGlu.gate        (src/ffn.rs:19-23)  */
    RBMOE_W_UP = 2,           /* [F, d]  per expert  SwiGlu.up                              */
    RBMOE_W_DOWN = 3,         /* [d, F]  per expert  SwiGlu.down                            */
    RBMOE_W_SHARED_GATE = 4,  /* [Fs, d]             MoeLayer.shared    (src/moe.rs:210)    */
    RBMOE_W_SHARED_UP = 5,    /* [Fs, d]                                                    */
    RBMOE_W_SHARED_DOWN = 6,  /* [d, Fs]                                                    */
    RBMOE_W_NORM = 7,         /* [1, d]  feed_forward_norm.weight: rbmoe_get_weight_grad only  */
    RBMOE_W_POST_NORM = 8,    /* [1, d]  rbmoe_set_block_join's weight: likewise                 */
    RBMOE_W_BLOCK_GATE = 9    /* [1, d]  rbmoe_set_block_join's gate: likewise                   */
} rbmoe_weight;

/* `MoeConfig` (reference src/moe.rs:25-39) plus what a device layer must know
 * up front.  `shared_d_ff` exists because the reference's `shared` field is
 * public and may hold an expert of another width (src/moe.rs:210, used that way
 * at src/moe.rs:841-843); 0 means "same as d_ff". */
typedef struct rbmoe_config {
    int32_t d_model;
    int32_t num_experts;
    int32_t experts_per_token;
    int32_t d_ff;
    int32_t shared_expert;         /* 0 / 1 */
    int32_t shared_d_ff;           /* 0 = d_ff */
    float aux_loss_weight;         /* DEFAULT_AUX_LOSS_WEIGHT = 0.01 (src/moe.rs:20)           */
    float router_z_loss_weight;    /* DEFAULT_ROUTER_Z_LOSS_WEIGHT = 1e-3 (src/moe.rs:23)      */
    int32_t weight_dtype;          /* rbmoe_dtype of the expert weights                        */
    int32_t act_dtype;             /* rbmoe_dtype of x / out: RBMOE_F32 or RBMOE_BF16          */
    int32_t max_tokens;            /* workspace is sized for this many rows; forward allocates nothing */
} rbmoe_config;

/* Routing tables of the last forward, the bit-exact comparands.
 * Slot s = token * k + rank (rank 0 = highest probability), as the reference's
 * `assignments` (src/moe.rs:142-145).  All pointers are optional (NULL = skip)
 * and must be host memory. */
typedef struct rbmoe_routing {
    int32_t* expert_of;   /* [T*k]  expert per slot, -1 = UNROUTED (src/moe.rs:190-191) */
    float* gate_of;       /* [T*k]  renormalised gate per slot                          */
    int32_t* counts;      /* [E]    expert_tokens[e].len() (src/moe.rs:266-274)         */
    int32_t* offsets;     /* [E+1]  exclusive prefix of counts                          */
    int32_t* perm_slot;   /* [T*k]  expert_slots, experts concatenated; first offsets[E] valid  */
    int32_t* perm_token;  /* [T*k]  expert_tokens, experts concatenated                 */
    float* probabilities; /* [T*E]  MoeCache.probabilities (src/moe.rs:137-140)         */
    float* log_sum_exp;   /* [T]    MoeCache.log_sum_exp   (src/moe.rs:141-142)         */
} rbmoe_routing;

typedef struct rbmoe_ctx rbmoe_ctx;
typedef struct rbmoe_layer rbmoe_layer;

/* MoeConfig::new (src/moe.rs:41-51): defaults for everything but the three
 * arguments; dtypes default to f32, max_tokens to 0 (must be set). */
int rbmoe_config_init(rbmoe_config* cfg, int32_t d_model, int32_t num_experts,
                      int32_t experts_per_token, int32_t d_ff);

/* MoeConfig::validate (src/moe.rs:68-86) plus dtype/limit checks.  Touches no
 * GPU.  On failure writes a message (same wording as the reference where one
 * exists) into `msg` if `msg_cap` > 0. */
int rbmoe_validate(const rbmoe_config* cfg, char* msg, size_t msg_cap);

/* TransformerConfig::parameter_counts restricted to one layer
 * (src/transformer.rs:194-227; MoeLayer::num_parameters / active_parameters,
 * src/moe.rs:527-545). */
int rbmoe_parameter_counts(const rbmoe_config* cfg, uint64_t* total, uint64_t* active);

/* Opens device `device` with a memory budget in MiB (0 = unlimited): the role of
 * `CudaDevice::open` + `GpuContext` (src/param.rs:86-190,
 * src/gpu_transformer.rs:45-76).  Fails closed with RBMOE_BACKEND_UNAVAILABLE
 * when no GPU can be used. */
int rbmoe_ctx_create(int32_t device, size_t budget_mib, rbmoe_ctx** out);
void rbmoe_ctx_destroy(rbmoe_ctx* ctx);

/* Use the caller's HIP stream (a `hipStream_t` passed as void*) instead of the
 * context's own; NULL restores the context's own stream. */
int rbmoe_ctx_set_stream(rbmoe_ctx* ctx, void* hip_stream);

/* GpuContext::synchronize (src/gpu_transformer.rs:179-187). */
int rbmoe_synchronize(rbmoe_ctx* ctx);

/* Message of the last failure on this context (owned by the context). */
const char* rbmoe_last_error(const rbmoe_ctx* ctx);
/* Message of the last failure of a call that had no context to attach it to
 * (thread-local). */
const char* rbmoe_last_global_error(void);

/* MoeLayer::new (src/moe.rs:215-231) + TransformerLm::to_cuda's upload of the
 * layer (src/transformer.rs:1263-1296): validates, checks the budget BEFORE
 * allocating (src/param.rs:172-189), allocates weights (zeroed) and workspace.
 * Expert widths between two multiples of a matrix-core tile are stored rounded up (bf16 rows: to 64, at most four
 * times the width; all-f32 layers: to 32, at most twice), which takes that much more memory.  f32 rows over bf16 or int8
 * weights keep f32 accuracy at widths off 64 (stored rounded up to 32, at most twice the width, where the context has no
 * memory budget, and as they are under one); at multiples of 64 the
 * products take a bf16 copy of the rows (RBMOE_OPT_FORCE_GENERIC: f32 accuracy there too, at a thirtieth of the rate).  A layer whose rounded
 * widths are over the budget - here, or when the norm or training mode is added before the first weight - or over a limit
 * of the backward products keeps its true widths instead (bf16 rows then take the any-shape kernels).  Layers that already hold
 * weights stay as they are: a budget shared by several layers has to allow for their rounded widths.
 * Small calls share a long down product's reduction out over workgroups, whose f32 sums are added in a fixed order; the rule looks at
 * the call's shape alone, so a call's bits do not depend on max_tokens.  Under a memory budget, in the layout of true widths
 * and in training mode, whose backward pass reads the rows, no reduction is shared out: the same call's rows may there differ in their last
 * bits (f32 sums in another order; bf16 rows by a rounding now and then). */
int rbmoe_layer_create(rbmoe_ctx* ctx, const rbmoe_config* cfg, rbmoe_layer** out);
void rbmoe_layer_destroy(rbmoe_layer* layer);

/* Behaviour switches of a layer, the counterpart of the reference's test hooks and environment switches
 * (CHUNK_ROWS_OVERRIDE src/gpu_model.rs:2948, cuda_flash::DISABLED src/cuda_flash.rs:898-907): every default is
 * the fast path, the other settings exist for A/B measurements and for tests that hold one kernel set against
 * another.  The library itself reads no environment variable. */
typedef enum rbmoe_option {
    RBMOE_OPT_FORCE_GENERIC = 0,   /* 1: the any-shape kernels for every product; only before the first weight is set */
    RBMOE_OPT_EXPLICIT_GATHER = 1, /* 1: gathered rows are written out instead of gathered inside the gate/up product */
    RBMOE_OPT_GROUP_M = 2,         /* row tiles that walk the column tiles together on one XCD; 0: each product's default */
    RBMOE_OPT_DECODE_PATH = 3,     /* 0: a few tokens take the large-batch kernels too */
    RBMOE_OPT_DECODE_FRONT = 4,    /* 0: decode-shaped calls route in a launch of their own */
    RBMOE_OPT_FUSED_ROUTER = 5,    /* 0: router logits and the routing behind them in separate launches */
    RBMOE_OPT_SIDE_STREAM = 6,     /* 0: everything on the context's one stream */
    RBMOE_OPT_WGRAD_MODE = 7,      /* cut experts' weight gradients: 0 fixed order (default), 1 f32 atomics, 2 never cut */
    RBMOE_OPT_WGRAD_GENERIC = 8,   /* 1: the plain kernel for the weight gradients */
    RBMOE_OPT_DECODE_COMBINE_FOLD = 9, /* 0: decode-shaped calls combine in a launch of their own */
    /* (not switches of a kernel choice, but of what rbmoe_set_weight does with f32 data) */
    RBMOE_OPT_QUANT_RULE = 10,     /* f32 -> int8 per row, scale = absmax / 127: 0 q = round(w / scale), the checkpoint
                                      writer's rule (src/transformer.rs:512-519); 1 q = round(w * (1 / scale)), the
                                      in-memory rule of Quantized::from_matrix (src/quantized.rs:29-51) */
    RBMOE_OPT_QUANTIZE_ROUTER = 11,/* 1: an f32 router is quantized at upload as well, as TransformerLm::quantize does
                                      (src/transformer.rs:899-910 via src/moe.rs:491-500), and the layer routes with the
                                      quantized product (sum x * q in 32 lanes) * scale (src/quantized.rs:55-62, :154-177) */
    RBMOE_OPT_DECODE_DOWN_BY_EXPERT = 12 /* (a kernel choice again) 0: the down launch of a decode-shaped call always
                                      finds its experts through the tile table, also behind RBMOE_OPT_DECODE_FRONT */
} rbmoe_option;
int rbmoe_layer_set_option(rbmoe_layer* layer, int32_t option, int32_t value);

/* DeviceParam::new (src/gpu_transformer.rs:471-490): copies one weight matrix
 * from HOST memory to the device (the caller keeps its buffer).  `dtype` is the
 * dtype of `data`; f32 data is converted to the layer's weight dtype (bf16 by
 * RNE; int8 by the checkpoint rule scale = absmax/127, q = round(w/scale),
 * src/transformer.rs:512-519, or the in-memory rule with RBMOE_OPT_QUANT_RULE).  For
 * RBMOE_I8 data, `scales` holds one f32 per row.  `expert` is ignored for the router and
 * the shared expert.  The router is kept in f32 whatever the experts' dtype, unless it is given
 * as RBMOE_I8 data or RBMOE_OPT_QUANTIZE_ROUTER is set: the layer then routes with the
 * quantized product of src/quantized.rs:55-62 (inference only). */
int rbmoe_set_weight(rbmoe_layer* layer, int32_t which, int32_t expert, const void* data,
                     int32_t dtype, const float* scales, int32_t rows, int32_t cols);

/* MoeLayer::forward_train (src/moe.rs:243-341) on DEVICE pointers, enqueued on
 * the context's stream; returns without synchronising.
 *   x        [T, cols] act_dtype; cols must equal d_model (else InvalidInput)
 *   valid    [T] bytes, 0 = padding row (Layout.valid, src/batch.rs:224-269), or NULL
 *   router_bias [E] f32 added to the logits, or NULL (the reference router is
 *            bias-free; this is a benchmark hook for skewed loads)
 *   residual [T, d] act_dtype added to the result (the block's residual add,
 *            src/transformer_block.rs:221-222), or NULL
 *   out      [T, d] act_dtype
 * Rows may start at any element; off a 16-byte boundary the matrix-core kernels work on a copy of them.
 * Auxiliary losses and routing tables stay on the device until fetched. */
int rbmoe_forward(rbmoe_layer* layer, const void* x, int32_t T, int32_t cols, const uint8_t* valid,
                  const float* router_bias, const void* residual, void* out);

/* rbmoe_forward for callers that cannot allocate device memory and want no allocation made on their behalf
 * either: code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc.  It has no
 * counterpart in the reference.  Same arguments and same results as rbmoe_forward (bit for bit: the same
 * kernels run), but every intermediate buffer of the call (probabilities, routing tables, tile table, losses,
 * hidden and expert output rows) lies in a static device array of RBMOE_STATIC_SCRATCH_BYTES that is part of
 * the library's code object, instead of in the workspace that rbmoe_layer_create allocated.  The call makes
 * no hipMalloc, hipFree or other allocating call.  (A few tokens over many or wide experts, which rbmoe_forward hands to
 * the large-batch kernels, stay decode-shaped here: same routing bit for bit, rows equal to their rounding.)
 * Limits: decode-shaped calls only, i.e. 1 to 32 tokens with tokens * num_experts <= 2048 on a layer with bf16
 * or int8 weights on the matrix-core path (bf16 rows, or f32 rows whose bf16 copy then lies in the
 * array as well), not in training mode; and the buffers of the call (about tokens * experts_per_token *
 * (d_ff + d_model) * 2 bytes, plus the shared expert's rows and the tables) must fit the array.  Anything else is RBMOE_UNSUPPORTED with a message that says which limit was hit.
 * Every call on one GPU, from any layer or context, uses that GPU's one array: calls that overlap in time on
 * one GPU race, and rbmoe_get_losses / rbmoe_get_routing / rbmoe_get_expert_rows after this call read the array,
 * so they describe this call only until the next static call on the same GPU. */
#define RBMOE_STATIC_SCRATCH_BYTES (8u << 20)
int rbmoe_forward_static(rbmoe_layer* layer, const void* x, int32_t T, int32_t cols, const uint8_t* valid,
                         const float* router_bias, const void* residual, void* out);

/* Same on HOST pointers: copies in, runs, synchronises, copies out. */
int rbmoe_forward_host(rbmoe_layer* layer, const void* x, int32_t T, int32_t cols,
                       const uint8_t* valid, const float* router_bias, const void* residual,
                       void* out);

/* forward_train on HOST matrices together with its MoeCache (src/moe.rs:243-341), in two halves.  _begin copies the
 * rows in, enqueues the forward (block != 0: the block step of rbmoe_forward_block, `residual` is then ignored) and
 * returns when `routing` and `losses` ([2]: auxiliary, z; either may be NULL) are filled, which is while the expert
 * products are still under way; `out` is complete after _finish.  `x_dtype` is the dtype of x, residual and out: the
 * layer's own, or RBMOE_F32 on a bf16 layer (rows are rounded to nearest even on the way in and widened on the way
 * out).  x, residual and out belong to the call until _finish.  Between the two calls no other call may
 * be made on the layer. */
int rbmoe_forward_train_begin(rbmoe_layer* layer, const void* x, int32_t x_dtype, int32_t T, int32_t cols,
                              const uint8_t* valid, const float* router_bias, const void* residual, int32_t block,
                              void* out, rbmoe_routing* routing, float* losses);
int rbmoe_forward_train_finish(rbmoe_layer* layer);

/* MoeCache::aux_loss / z_loss (src/moe.rs:158-172) of the last forward.
 * Synchronises the stream. */
int rbmoe_get_losses(rbmoe_layer* layer, float* aux_loss, float* z_loss);

/* Routing tables of the last forward into host buffers.  Synchronises. */
int rbmoe_get_routing(rbmoe_layer* layer, rbmoe_routing* routing);

/* Expert hidden rows H [offsets[E], F] and expert output rows Y [offsets[E], d]
 * of the last forward, in permuted order, converted to f32, into host buffers
 * (either may be NULL) — the reference keeps both in MoeCache
 * (src/moe.rs:150-152, src/ffn.rs:27-33).  Synchronises. */
int rbmoe_get_expert_rows(rbmoe_layer* layer, float* hidden, float* expert_out);

/* ---- the block's steps either side of the layer ------------------------------------------
 * TransformerBlock::forward_train's feed-forward half (src/transformer_block.rs:216-222):
 *   normed = feed_forward_norm.forward(residual)   RmsNorm::forward, src/norm.rs:41-61
 *   output = moe.forward_train(normed) + residual  add_in_place, src/transformer_block.rs:310-323
 * rbmoe_set_feed_forward_norm uploads the norm's weight [d_model] (f32, host) and eps
 * (TransformerConfig::rmsnorm_eps, src/transformer.rs:42); the first call allocates the normed rows. */
int rbmoe_set_feed_forward_norm(rbmoe_layer* layer, const float* weight, int32_t cols, float eps);
/* out = x + layer(rmsnorm(x)) on DEVICE pointers ([T, d] act_dtype; `out` may be `x` itself).  The norm
 * runs as a prologue kernel with the reference's sequential sum of squares, so routing is decided on the
 * same normed rows as on the CPU; the residual add is part of the combine kernel.  Routing, losses and
 * the backward pass's state refer to the NORMED rows (rbmoe_backward then returns the gradient with
 * respect to them).  Other arguments as rbmoe_forward. */
int rbmoe_forward_block(rbmoe_layer* layer, const void* x, int32_t tokens, int32_t cols, const uint8_t* valid,
                        const float* router_bias, void* out);
/* Same on HOST pointers; synchronises. */
int rbmoe_forward_block_host(rbmoe_layer* layer, const void* x, int32_t tokens, int32_t cols,
                             const uint8_t* valid, const float* router_bias, void* out);

/* The block step's join, where it is more than the residual add: out = x + scale * gate * RmsNorm(layer(rmsnorm(x))) * post_weight, as
 * rbmoe_join_forward has it (below), of the layer's rows rounded to its dtype.  post_weight and gate are HOST [d_model] f32 or NULL; both
 * NULL with scale 1 is the residual add again.  From then on rbmoe_forward_block and rbmoe_backward_block (and their host forms) include it; padding rows pass x through, the
 * shared expert's rows included.  In training mode the gradients of post_weight and gate accumulate like the norm's
 * (RBMOE_W_POST_NORM, RBMOE_W_BLOCK_GATE).  Needs the feed-forward norm; a backward pass for a forward from before this call is refused.
 * (rbmoe_backward behind a joined block step is the layer's alone: its grad_output is that of the layer's rows.) */
int rbmoe_set_block_join(rbmoe_layer* layer, const float* post_weight, const float* gate, int32_t cols, float eps, float scale);

/* ---- backward pass (MoeLayer::backward, src/moe.rs:348-489) ------------------------------
 * Training mode makes the forward keep what MoeCache keeps for the backward pass (the input,
 * src/moe.rs:133-135; gate and up pre-activations, src/ffn.rs:27-33) and allocates f32 gradient
 * accumulators, the role of Param.grad (src/param.rs).  For every f32 / bf16 layer: bf16 layers with a d_model
 * that is a multiple of 64 and all-f32 layers (32) differentiate on the matrix cores, their expert widths rounded up
 * (rbmoe_layer_create); f32 rows over bf16 weights do where every width is a multiple of 64; any other shape or dtype
 * mix on plain kernels; int8 layers report RBMOE_UNSUPPORTED, as the reference has no backward for quantized
 * experts (src/ffn.rs:87-93).
 * Call it before the weights are set.  A training layer always takes the large-batch kernels.  A forward from before it has kept no
 * input, so rbmoe_backward behind one is RBMOE_INVALID_INPUT (but for large-batch calls behind the norm, whose rows are the layer's). */
int rbmoe_layer_enable_training(rbmoe_layer* layer);

/* MoeLayer::backward on DEVICE pointers for the last forward: `grad_output` [tokens, cols] act_dtype in,
 * `grad_input` [tokens, cols] act_dtype out; weight gradients are ACCUMULATED (as Param.grad is) until
 * rbmoe_zero_grads.  The gradients of the two auxiliary losses reach the router here, as in the
 * reference (src/moe.rs:343-347).  `tokens` and `cols` are the shape of both buffers and must be the
 * last forward's (the reference sizes the gradient from the cached input, src/moe.rs:349-350):
 * anything else is RBMOE_INVALID_INPUT and neither buffer is touched.  Enqueued on the context's stream. */
int rbmoe_backward(rbmoe_layer* layer, const void* grad_output, int32_t tokens, int32_t cols, void* grad_input);
/* Same on HOST pointers; synchronises. */
int rbmoe_backward_host(rbmoe_layer* layer, const void* grad_output, int32_t tokens, int32_t cols,
                        void* grad_input);
/* The same (block != 0: rbmoe_backward_block) on host gradients of dtype `dtype`: the layer's own, or RBMOE_F32 on a
 * bf16 layer.  Synchronises. */
int rbmoe_backward_train_host(rbmoe_layer* layer, const void* grad_output, int32_t dtype, int32_t tokens, int32_t cols,
                              int32_t block, void* grad_input);
/* Param::zero_grad for every weight of the layer. */
int rbmoe_zero_grads(rbmoe_layer* layer);
/* One accumulated weight gradient as f32 [rows, cols] into host memory (same ids and shapes as
 * rbmoe_set_weight).  Synchronises. */
int rbmoe_get_weight_grad(rbmoe_layer* layer, int32_t which, int32_t expert, float* host, int32_t rows,
                          int32_t cols);

/* The feed-forward half of TransformerBlock::backward (src/transformer_block.rs:257-263) after
 * rbmoe_forward_block, on DEVICE pointers:
 *   grad_projected = moe.backward(cache, grad_output)
 *   grad_input     = feed_forward_norm.backward(residual, grad_projected) + grad_output
 * (RmsNorm::backward, src/norm.rs:63-121).  The norm's scale gradient accumulates like the other weight
 * gradients and is read with rbmoe_get_weight_grad(layer, RBMOE_W_NORM, 0, host, 1, d_model).  `grad_input`
 * may be `grad_output` itself.  Needs training mode and a norm (in either order).  `tokens` and `cols` as
 * for rbmoe_backward. */
int rbmoe_backward_block(rbmoe_layer* layer, const void* grad_output, int32_t tokens, int32_t cols,
                         void* grad_input);
/* Same on HOST pointers; synchronises. */
int rbmoe_backward_block_host(rbmoe_layer* layer, const void* grad_output, int32_t tokens, int32_t cols,
                              void* grad_input);

/* ---- a sub-layer joined to the residual stream ----------------------------------------------------
 * What stands between a sub-layer's output and the next sub-layer's input, in one call each way: a norm behind the sub-layer,
 * a gate, a residual scale, the residual add and the next norm.  The reference's block has the add and the norm in front
 * (src/transformer_block.rs:216-222); with a norm behind, a gate or a scale it has no counterpart.
 *   b      = RmsNorm(y) * post_weight      (y itself where post_weight is NULL)
 *   out    = x + scale * gate * b
 *   normed = RmsNorm(out) * next_weight    (of the rows as they are stored; only with next_weight)
 * Rows [rows, cols] are of the join's dtype, weights [cols] f32; a gate by channel is [cols] f32, one by row [rows, cols] of the join's
 * dtype.  All of them DEVICE pointers.  `valid` [rows] bytes or NULL: a padding row (0) takes y as zero, so its `out` is its x; what
 * lies in its y and gate is not used, and it adds nothing to the gradients of weights and gate (its `normed` is that of its x, and
 * grad_normed reaches its grad_x).  Statistics and sums are f32, each output is rounded once; a row's sum of squares is taken in f32, so
 * a row whose squares pass its range has a norm of zeros, and with eps 0 one whose squares are below it none.  `out` may be x, `normed` may
 * be y; apart from that outputs must not overlap inputs or one another. */
typedef enum rbmoe_gate {
    RBMOE_GATE_NONE = 0,
    RBMOE_GATE_CHANNEL = 1, /* [cols] f32, a parameter */
    RBMOE_GATE_ROW = 2      /* [rows, cols] of the rows' dtype */
} rbmoe_gate;
typedef struct rbmoe_join rbmoe_join;
/* Holds the workspace of the backward pass (counted against the context's budget), up to 12 bytes a column for each of 512 workgroups; weights
 * come with a call, so one join serves every sub-layer of its width, dtype and gate, one call after the other.  1 to 65536 columns; calls take up
 * to 2^30 rows. */
int rbmoe_join_create(rbmoe_ctx* ctx, int32_t cols, int32_t dtype, int32_t gate, rbmoe_join** out);
void rbmoe_join_destroy(rbmoe_join* join);
/* Enqueued on the context's stream; allocates nothing. */
int rbmoe_join_forward(rbmoe_join* join, int32_t rows, const void* x, const void* y, const uint8_t* valid,
                       const float* post_weight, const void* gate, float scale, const float* next_weight, float eps,
                       void* out, void* normed);
/* Gradients of both inputs (grad_x, grad_y, required), and of post_weight, gate and next_weight (each may be NULL).  y, valid, weights,
 * gate, scale and eps are the forward's, `out` the rows that it wrote (read with next_weight only).  grad_out is what reaches `out`
 * from elsewhere (NULL: nothing), grad_normed what reaches `normed` (with next_weight).  Gradients of [cols] parameters are
 * written, or with accumulate != 0 added to what is there; a gate's by row is always written.  A gradient of an input may lie where
 * grad_out or grad_normed lies.  The same call gives the same bits.  Calls on one join must not overlap in time. */
int rbmoe_join_backward(rbmoe_join* join, int32_t rows, const void* y, const void* out, const uint8_t* valid,
                        const float* post_weight, const void* gate, float scale, const float* next_weight, float eps,
                        const void* grad_out, const void* grad_normed, int32_t accumulate, void* grad_x, void* grad_y,
                        float* grad_post, void* grad_gate, float* grad_next);

/* ---- orthogonalised weight updates -----------------------------------------------------------------
 * The reference's optimisers run on the host over Param.grad; this is a step on the device for weight matrices.  A handle
 * takes a stack of `count` matrices [rows, cols] (row-major, contiguous, at most 16384 a side) and holds the workspace: about 12 bytes an element
 * and 8 bytes a squared shorter side, counted against the context's budget.
 * rbmoe_orthogonalize brings the singular values of every matrix near one: X = U / (|U|_F + 1e-7), then `steps` times
 *   A = X X^T, B = b A + c A A, X = a X + B X,  (a, b, c) = (3.4445, -4.7750, 2.0315)
 * (five steps: values from 0.003 |U|_F up end in [0.68, 1.21]; elements below 2^-38 |U|_F count as zero).  Accuracy is f32's whatever the types of `in` and `out`, each RBMOE_F32 or
 * RBMOE_BF16, and whatever |U|_F is, from 1e-35 up: one far below 1e-7 gives a small result, exact relative to itself.  `out` may be `in`.  A
 * matrix of zeros stays one.
 * rbmoe_muon_step is an optimiser step with it (decoupled weight decay):
 *   M = momentum_factor M + G,  U = G + momentum_factor M (nesterov != 0) or M,
 *   W = (1 - lr weight_decay) W - lr update_scale O,  O the orthogonalised U;  update_scale 0 stands for sqrt(max(1, rows / cols)).
 * M and W are f32 and updated in place.  DEVICE pointers, enqueued on the context's stream, nothing is allocated; the same call
 * gives the same bits.  Calls on one handle must not overlap in time.  A matrix with infinities or NaN among its gradients ends as NaN,
 * the others of the stack do not. */
typedef struct rbmoe_muon rbmoe_muon;
int rbmoe_muon_create(rbmoe_ctx* ctx, int32_t count, int32_t rows, int32_t cols, rbmoe_muon** out);
void rbmoe_muon_destroy(rbmoe_muon* muon);
int rbmoe_orthogonalize(rbmoe_muon* muon, const void* in, int32_t in_dtype, int32_t steps, void* out, int32_t out_dtype);
int rbmoe_muon_step(rbmoe_muon* muon, const void* grad, int32_t grad_dtype, float* momentum, float* weight, float lr,
                    float momentum_factor, float weight_decay, float update_scale, int32_t nesterov, int32_t steps);

/* The same step for a layer's expert matrices, from its own accumulated gradients: every gate, up and down matrix of the routed
 * and the shared expert gets one, and the stored weights (operand order and the backward pass's transposed copies included) follow on the
 * device.  rbmoe_layer_enable_muon, after rbmoe_layer_enable_training and before the weights are set, allocates momentum (zeros), for a bf16
 * layer f32 weights that the stored ones are rounded from, and the workspace.  The router, the norm and the join keep their
 * weights: they are vectors or nearly so, and the host updates them.  rbmoe_layer_muon_step enqueues kernels only (it can be captured);
 * RBMOE_INVALID_INPUT where no backward pass has run since rbmoe_zero_grads.  The gradients stay as they are. */
int rbmoe_layer_enable_muon(rbmoe_layer* layer);
int rbmoe_layer_muon_step(rbmoe_layer* layer, float lr, float momentum_factor, float weight_decay, float update_scale,
                          int32_t nesterov, int32_t steps);
/* One expert matrix as f32 [rows, cols] (ids and shapes as rbmoe_set_weight; f32 layers, or with updates enabled) into HOST memory: what
 * a checkpoint holds.  Synchronises. */
int rbmoe_get_weight(rbmoe_layer* layer, int32_t which, int32_t expert, float* host, int32_t rows, int32_t cols);

/* ---- attention ------------------------------------------------------------------------------------
 * The attention half of a block, between its projections: whole sequences both ways (the reference's src/attention.rs, and
 * src/cuda_flash.rs on its device), a paged cache of keys and values, and one new row a sequence over it.  Rows are [rows, heads, head_dim] of
 * RBMOE_F32 or RBMOE_BF16 with consecutive elements; a stride says how many elements lie between two rows (0: no gap), so that
 * q, k and v may lie side by side as one projection leaves them.  kv_heads divides heads: head h reads kv head
 * h / (heads / kv_heads).  head_dim is a multiple of 8 up to 128, heads at most 1024.  Everything below are DEVICE pointers but the handles; every call is
 * enqueued on the context's stream and allocates nothing, and the same call gives the same bits.  Outputs must not overlap inputs or one another.  Rows of 16-byte
 * pieces (addresses and strides) are staged the fast way; any other element is as good a start. */

/* Attention of whole sequences.  Sequence i has the queries query_begin[i] .. + query_count[i] and the keys key_begin[i] .. +
 * key_count[i] (key arrays NULL: the queries'), of arrays of query_rows and key_rows rows: packed one behind the other, or padded,
 * with rows between them that are left as they are.  Counts go up to longest_queries and longest_keys, which a launch is
 * sized by (a longer sequence counts as that long).  With causal != 0 query r of a sequence sees its keys up to
 * r + key_count - query_count: the queries are the last of the keys, whose first may come from a cache.  Rows and keys of a sequence that lie outside the
 * arrays are left out, and the others see what they would see beside them.
 *   s_ij = scale q_i . k_j,   lse_i = log sum_j exp s_ij,   out_i = sum_j exp(s_ij - lse_i) v_j    over the keys that row i sees
 * A row that sees no key is zeros, its lse -inf; a key whose score is -inf counts as not seen.  What is not seen has no effect, whatever it
 * holds; infinities and NaN that are seen have the effect that f32 arithmetic gives them.  scale is positive.  Two sequences may share keys
 * (forward only), not queries.
 *   out  [query_rows, heads, head_dim] without gaps      lse [heads, query_rows] f32 or NULL
 * Sums and statistics are f32.  f32 rows are multiplied in parts that keep their 24 bits, and results are as exact as with f32 products; bf16 rows
 * round exp(s_ij - m) to bf16 for the product with v, and p and ds for the gradients (sequences of up to 32 rows or keys: to 16 bits). */
typedef struct rbmoe_attention rbmoe_attention;
/* backward_rows: the most query rows of a backward pass (0: forward only): 8 bytes a row and head, and for the first 16384 / kv_heads rows of
 * heads in groups 8 * head_dim bytes a row and head more, counted against the budget. */
int rbmoe_attention_create(rbmoe_ctx* ctx, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t backward_rows,
                           rbmoe_attention** out);
void rbmoe_attention_destroy(rbmoe_attention* attention);
int rbmoe_attention_forward(rbmoe_attention* attention, int32_t sequences, int32_t longest_queries, int32_t longest_keys,
                            const int32_t* query_begin, const int32_t* query_count, const int32_t* key_begin, const int32_t* key_count,
                            int32_t query_rows, int32_t key_rows, const void* q, int32_t q_stride, const void* k, int32_t k_stride,
                            const void* v, int32_t v_stride, int32_t causal, float scale, void* out, float* lse);
/* Gradients of q, k and v, each with its input's stride and of its type; the arguments up to scale are the forward's, out and lse
 * what it wrote, grad_out is without gaps like out.  A kv head's gradients are the sums over its group;
 * keys that no row sees get zeros.  Every sequence has keys of its own.  Calls on one attention must not overlap in time (the forward may be called
 * any way). */
int rbmoe_attention_backward(rbmoe_attention* attention, int32_t sequences, int32_t longest_queries, int32_t longest_keys,
                             const int32_t* query_begin, const int32_t* query_count, const int32_t* key_begin, const int32_t* key_count,
                             int32_t query_rows, int32_t key_rows, const void* q, int32_t q_stride, const void* k, int32_t k_stride,
                             const void* v, int32_t v_stride, int32_t causal, float scale, const void* out, const float* lse,
                             const void* grad_out, void* grad_q, void* grad_k, void* grad_v);

/* A cache of keys and values in pages.  Slot page * page_rows + r is row r of a page; which pages belong to which sequence is the
 * caller's affair.  Rows are of `dtype`, the cache holds them as they are (cache_dtype = dtype) or in 8 bits (RBMOE_I8): a scale max |x| / 127 a
 * row and head, round(127 x / max |x|) with ties to even; a row with an infinity or NaN reads back as NaN.  page_rows is a power of two from 16 to
 * 4096.  The pages (zeros at first, head_dim rounded up to 64 or 128, 8 bytes more a row and head in 8 bits) count against the budget. */
typedef struct rbmoe_kv_cache rbmoe_kv_cache;
int rbmoe_kv_cache_create(rbmoe_ctx* ctx, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t cache_dtype, int32_t page_rows,
                          int32_t pages, rbmoe_kv_cache** out);
void rbmoe_kv_cache_destroy(rbmoe_kv_cache* cache);
/* Rows k and v [rows, kv_heads, head_dim] (up to 2^28 a call) to their slots.  A row whose slot is negative or behind the last page is left out (padding).  The
 * rows of one call go to different slots: two rows for one slot leave a mixture of both there. */
int rbmoe_kv_cache_write(rbmoe_kv_cache* cache, int32_t rows, const void* k, int32_t k_stride, const void* v, int32_t v_stride,
                         const int64_t* slots);
/* And back, to any rows; those without a slot are zeros. */
int rbmoe_kv_cache_read(rbmoe_kv_cache* cache, int32_t rows, void* k, int32_t k_stride, void* v, int32_t v_stride, const int64_t* slots);

/* One query row a sequence over the cache: out[i] = attention of q[i] over the first lengths[i] rows of sequence i, whose pages are
 * tables[i][0 .. table_pages).  The new row's own key is written before, and counts.  Lengths go up to `longest` (longer ones are cut), by which a
 * launch is sized: a captured graph takes the longest that its replays will see.  A table entry that is no page of the cache has no rows; a
 * sequence without any gives zeros.  Infinities and NaN have the effect that f32 arithmetic gives them.  The handle holds the workspace for up to max_sequences sequences, joins parts of long sequences in
 * it, and serves any number of caches, one call after the other.  Where the parts end depends on all lengths of a call, and the last bits of its f32
 * sums with it. */
typedef struct rbmoe_decode rbmoe_decode;
int rbmoe_decode_create(rbmoe_ctx* ctx, int32_t heads, int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t max_sequences,
                        rbmoe_decode** out);
void rbmoe_decode_destroy(rbmoe_decode* decode);
int rbmoe_decode_attention(rbmoe_decode* decode, rbmoe_kv_cache* cache, int32_t sequences, const void* q, int32_t q_stride,
                           const int32_t* tables, int32_t table_pages, const int32_t* lengths, int32_t longest, float scale, void* out);

/* Per-stage timing of one forward with HIP events on the context's stream.
 * `ms` receives RBMOE_NUM_STAGES durations in milliseconds.  Synchronises.
 * Every stage has launches of its own here, one behind the other: a call that is not timed may have the dispatch inside the
 * gate/up launch, and the shared expert's products inside the routed experts' launches or beside them on a second stream,
 * and is then shorter than the stages' sum.
 * Stage 1 brackets no work at all: it reads what one pair of event records adds to
 * every other stage (about 5 us), so callers can subtract it. */
#define RBMOE_NUM_STAGES 8
enum {
    RBMOE_STAGE_ROUTER = 0,   /* logits, softmax, top-k, block histograms       */
    RBMOE_STAGE_EMPTY = 1,    /* nothing: the cost of one event interval        */
    RBMOE_STAGE_DISPATCH = 2, /* layout scan, losses, permutation (+ row gather) */
    RBMOE_STAGE_GATE_UP = 3,  /* grouped gate/up product + SwiGLU               */
    RBMOE_STAGE_DOWN = 4,     /* grouped down product                           */
    RBMOE_STAGE_SHARED = 5,   /* shared expert (both products)                  */
    RBMOE_STAGE_COMBINE = 6,  /* gate-weighted combine (+ shared, + residual)   */
    RBMOE_STAGE_TOTAL = 7
};
int rbmoe_forward_timed(rbmoe_layer* layer, const void* x, int32_t T, int32_t cols,
                        const uint8_t* valid, const float* router_bias, const void* residual,
                        void* out, float* ms);

/* Kernel durations of one forward the way a kernel trace reports them: every launch of the forward carries its own
 * start and stop events, which receive the begin and end time stamps of that dispatch itself (no launch gap, no
 * event-pair overhead, no events between the stages).  `ms` receives RBMOE_NUM_STAGES values in milliseconds: per
 * stage the sum over its launches (RBMOE_STAGE_EMPTY: 0), RBMOE_STAGE_TOTAL: their sum - the time the device spent
 * inside kernels, which is less than the forward took by the gaps between the launches.  Synchronises.  Where the
 * gate/up launch does the dispatch's work, RBMOE_STAGE_DISPATCH is 0.  A large-batch call's shared expert has launches of its
 * own on the main stream here, like rbmoe_forward_timed's; one that is not timed may have it inside the routed experts'
 * launches or beside them.  A reduction that the call shares out over workgroups is shared out alike in both. */
int rbmoe_forward_kernel_times(rbmoe_layer* layer, const void* x, int32_t T, int32_t cols,
                               const uint8_t* valid, const float* router_bias, const void* residual,
                               void* out, float* ms);

/* Launch time of one stage by itself: enqueues the launches of stage `stage` (RBMOE_STAGE_ROUTER, _DISPATCH,
 * _GATE_UP, _DOWN or _COMBINE) of the LAST forward again, on the same buffers, once untimed and then `launches`
 * times back to back between ONE pair of events, and returns the average in milliseconds.  Synchronises.  The
 * stages read their inputs and overwrite their outputs with the same values, so the layer's state is unchanged.
 * A figure taken this way contains no event-pair overhead (one pair over many launches) and cannot fall below
 * what a kernel trace shows for the launch; the operands a stage shares with its neighbours in a forward may sit
 * in other cache levels here.  With ms_per_launch == NULL the launches are only enqueued (no warm-up, no events, no
 * synchronisation): for a caller that times a sequence of its own, e.g. the same stage of several layers in
 * rotation.  RBMOE_UNSUPPORTED when the last forward had nothing to do for the stage, or did it in a decode-shaped launch; a
 * dispatch inside a gate/up launch is replayed as the launch it would be, and gate/up and down as the routed experts' alone. */
int rbmoe_replay_stage(rbmoe_layer* layer, int32_t stage, int32_t launches, float* ms_per_launch);

/* Name of the kernels the last forward used for the expert products, for reports: "mfma_bf16_stream" (large
 * batches), "mfma_bf16_decode_front" (a few tokens, routing beside the gate/up products), "mfma_bf16_decode" (a few
 * tokens, routing in a launch of its own), each with "_int8w" behind it for int8 weights, "mfma_f32" (all-f32 layers
 * at widths of whole slices), "generic" (every other layer: f32 rows, whose products run on the matrix cores like mfma_f32's
 * unless RBMOE_OPT_FORCE_GENERIC is set, and bf16 rows on the any-shape kernels); "none" before the first.  Static storage. */
const char* rbmoe_expert_kernel_name(const rbmoe_layer* layer);

/* Device memory helpers for hosts without their own HIP binding. */
int rbmoe_device_alloc(rbmoe_ctx* ctx, size_t bytes, void** out);
int rbmoe_device_free(rbmoe_ctx* ctx, void* ptr);
/* Host memory the GPU writes to and reads from directly (57 GB/s over the link here, against 4 to 30 for a copy to or
 * from memory that is not pinned): every entry point above that fills or reads a host array recognises these blocks.
 * They come from a pool of at most 1 GiB that keeps freed blocks for the next caller while a context lives; RBMOE_OUT_OF_MEMORY when it is exhausted (use ordinary memory then).  Any thread may free. */
int rbmoe_host_alloc(rbmoe_ctx* ctx, size_t bytes, void** out);
void rbmoe_host_free(void* ptr);
int rbmoe_copy_to_device(rbmoe_ctx* ctx, void* dst, const void* src, size_t bytes);
int rbmoe_copy_to_host(rbmoe_ctx* ctx, void* dst, const void* src, size_t bytes);
/* Device-to-device copy on the context's stream, then synchronise (also serves as the
 * plain copy of known size that hardware-counter readings are calibrated against). */
int rbmoe_copy_device(rbmoe_ctx* ctx, void* dst, const void* src, size_t bytes);


const char* rbmoe_version(void);

#ifdef __cplusplus
}
#endif
#endif /* RBMOE_H */
