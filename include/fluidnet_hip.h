/*
 * fluidnet_hip.h -- C ABI of libfluidnet_hip.so, the MI355X (gfx950) compute library behind
 * the FluidNet hot path (UNet forward/backward, physics loss, K-step rollout loss, clip+Adam,
 * autoregressive rollout).
 *
 * The reference (ohmatheus/FluidNet) has no FFI for this path: its boundary is the Python module
 * API of ml/ (SURVEY.md section 8b).  This header is what a binding for that API would call; every
 * entry point cites the reference interface it replaces (paths relative to the reference root).
 * All pointers are DEVICE pointers unless named host_*; no torch types appear here.  Every launch
 * goes to the hipStream_t passed in (as void*); nothing here allocates, frees or synchronises
 * unless the comment says so.  Return value: 0 = ok, negative = FNET_E_* (see fnet_strerror).
 *
 * Data layout ("P-tensor"): activations live in HBM as channels-last, spatially PADDED arrays
 *     [B][H+2][W+2][ldc]   element type fp32 or bf16,
 * one ring of padding pixels filled according to the conv padding mode (zeros / replicate /
 * reflect / circular), so that every 3x3 convolution is a "valid" convolution over the
 * flattened pixel axis f = (n*(H+2)+y)*(W+2)+x with nine constant offsets.  A view selects
 * channels [coff, coff+C) of a buffer with ldc channels (this is how skip-connection concat
 * costs nothing).  Field planes at the API surface (inputs, targets, predictions) are plain
 * fp32 NCHW like the reference's tensors.
 */
#ifndef FLUIDNET_HIP_H
#define FLUIDNET_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FNET_ABI_VERSION 2        /* 2: FnetOp slot meanings of round 2 (CONV3X3 mode, lanes in slot 29), fnet_set_knob */

/* error codes */
#define FNET_OK 0
#define FNET_E_BADARG (-1)   /* shape / alignment / enum violation (host-side check, nothing launched) */
#define FNET_E_HIP (-2)      /* a HIP runtime call failed; fnet_last_hip_error() has the code */
#define FNET_E_UNSUPPORTED (-3)
#define FNET_E_TOO_LARGE (-4)  /* the input exceeds the stated maximum of an allocation-free entry point (nothing launched) */
#define FNET_E_OVERLAP (-5)    /* two tensors of a list that is written share memory (nothing launched) */

/* element type of P-tensors */
#define FNET_F32 0
#define FNET_BF16 1
#define FNET_F16 2            /* block norms and tensor lists only */

/* padding mode (ml/models/unet.py:13 PaddingType; ml/training/physics_loss.py:32-33) */
#define FNET_PAD_ZEROS 0
#define FNET_PAD_REPLICATE 1
#define FNET_PAD_REFLECT 2
#define FNET_PAD_CIRCULAR 3

/* activation (ml/models/unet.py:31-39) */
#define FNET_ACT_RELU 0
#define FNET_ACT_LEAKY 1
#define FNET_ACT_GELU 2
#define FNET_ACT_SILU 3
#define FNET_ACT_IDENTITY 4

/* output activation (ml/models/unet.py:296-301) */
#define FNET_OUT_LINEAR_CLAMP 0
#define FNET_OUT_SIGMOID_TANH 1

/* stencil (ml/training/physics_loss.py:16) */
#define FNET_STENCIL_FORWARD 0
#define FNET_STENCIL_CENTRAL 1

/* conv implementation selector */
#define FNET_CONV_REF 0   /* plain fp32-accumulate FMA kernels, any dtype: the debugging / exact path */
#define FNET_CONV_MFMA 1  /* bf16 MFMA implicit GEMM (32x32x16), LDS-staged halo rows */

/* ---- op records ------------------------------------------------------------------------
 * A "plan" is an array of FnetOp executed in order on one stream by fnet_plan_run().  The host
 * side (fluidnet_amd/engine/plan.py) builds one plan per (UNetConfig, B, H, W, K) and replays
 * it every step; slot meaning per opcode is documented in include/fluidnet_ops.h.
 */
typedef struct FnetOp {
    int32_t op;       /* FNET_OP_* */
    int32_t dtype;    /* FNET_F32 / FNET_BF16 for the P-tensors of this op */
    int32_t i[30];    /* integer arguments */
    float f[8];       /* float arguments */
    uint64_t p[10];   /* device pointers (0 = absent) */
} FnetOp;

enum FnetOpCode {
    FNET_OP_NOP = 0,
    FNET_OP_PACK_INPUT = 1,
    FNET_OP_CONV3X3 = 2,
    FNET_OP_WGRAD = 3,
    FNET_OP_IN_STATS = 4,
    FNET_OP_APPLY = 5,
    FNET_OP_UPSAMPLE2X = 6,
    FNET_OP_SUBSAMPLE_BIAS = 7,
    FNET_OP_PAD_RING = 8,
    FNET_OP_HEAD_FWD = 9,
    FNET_OP_LOSS_REDUCE = 10,
    FNET_OP_LOSS_FINALIZE = 11,
    FNET_OP_LOSS_GRAD = 12,
    FNET_OP_HEAD_BWD = 13,
    FNET_OP_INACT_BWD_REDUCE = 14,
    FNET_OP_INACT_BWD_APPLY = 15,
    FNET_OP_AFFINE_GRAD = 16,
    FNET_OP_FOLD_SUM = 17,
    FNET_OP_BIAS_GRAD = 18,
    FNET_OP_ZERO_INSERT = 19,
    FNET_OP_UPSAMPLE2X_BWD = 20,
    FNET_OP_UNPACK_GRAD = 21,
    FNET_OP_ZERO = 22,
    FNET_OP_PREP_WEIGHTS = 23,
    FNET_OP_GRAD_NORM = 24,
    FNET_OP_ADAM = 25,
    FNET_OP_COPY_PLANES = 26,
    FNET_OP_UNPREP_WGRAD = 27,
    FNET_OP_STENCIL = 28,
    FNET_OP_AFFINE_GRAD_MULTI = 29,
    FNET_OP_METRICS = 30,
    FNET_OP_GATHER_BATCH = 31,
    FNET_OP_POOL2X = 32,          /* 2x2 average / max pooling of the pooled `down` variants (unet.py:93-94) */
    FNET_OP_POOL2X_BWD = 33,
    FNET_OP_NORM_COMBINE = 34,    /* BatchNorm2d / GroupNorm statistics pooled from the per-(n,c) ones (unet.py:20-28) */
    FNET_OP_NORM_COMBINE_BWD = 35,
    FNET_OP_DEPTH2SPACE = 36,     /* phase interleave + bias of the transposed-conv upsample (unet.py:150) */
    FNET_OP_SPACE2DEPTH = 37,
    FNET_OP_EVENT_RECORD = 38,    /* lanes: record event i[0] on the op's lane (see FNET_LANE_SLOT) */
    FNET_OP_EVENT_WAIT = 39,      /* lanes: the op's lane waits for the last record of event i[0] */
    FNET_OP_COUNT_
};

/* Lanes.  Every op runs on lane op.i[FNET_LANE_SLOT]: lane 0 is the stream passed to fnet_plan_run, lanes 1..FNET_MAX_LANES-1 are
 * side streams the library creates once per device (hipStreamNonBlocking).  EVENT_RECORD / EVENT_WAIT (event ids 0 .. 2^20-1, a
 * per-device pool shared by all plans: an id is recorded before it is waited for inside one fnet_plan_run) order lanes against
 * each other.  The plan builder joins every side lane back into lane 0 before the plan ends.  Used to run the weight-gradient
 * kernels (MFMA-bound) beside the normalisation / activation adjoint kernels (HBM- and VALU-bound) of the backward pass. */
#define FNET_LANE_SLOT 29
#define FNET_MAX_LANES 4

/* Library identity / diagnostics. */
int fnet_abi_version(void);
const char* fnet_strerror(int code);
int fnet_last_hip_error(void);
/* Device properties the host uses to size grids: [0]=CU count, [1]=max LDS per block, [2]=warp size, [3]=gfx major*100+minor. */
int fnet_device_info(int32_t out[4]);

/*
 * Execute a plan: ops[0..n) in order on `stream`.  Replaces the chain of ATen calls under
 * UNet.forward (ml/models/unet.py:281-303), PhysicsAwareLoss.forward
 * (ml/training/physics_loss.py:210-278), Trainer._compute_rollout_loss
 * (ml/training/trainer.py:311-385), loss.backward()/clip_grad_norm_/Adam.step
 * (ml/training/trainer.py:190-195) and the rollout loop body (ml/scripts/simple_infer.py:226-260).
 * Every op validates its arguments on the host before launching; on the first failure nothing
 * further is launched and *failed_index (if non-null) receives the op index.
 * The executor may issue adjacent records as one launch where that is the same computation: a run of PREP_WEIGHTS records (one launch
 * per 32), IN_STATS immediately followed by the APPLY of the same InstanceNorm unit on an image of at most 64 x 64, and
 * INACT_BWD_REDUCE immediately followed by the INACT_BWD_APPLY of the same single-source unit on at most 32 x 32 (ml/models/unet.py:65-69
 * and its autograd adjoint in one kernel each; statistics summed in a fixed order, outputs within one bf16 ulp of the separate
 * launches); HEAD_FWD immediately followed by the LOSS_REDUCE of its prediction, and LOSS_GRAD immediately followed by the HEAD_BWD that
 * consumes its dpred (ml/models/unet.py:294-303 + ml/training/physics_loss.py:210-278 in one pass each: z, pred, dpred and the activation
 * gradient bit-identical to the separate launches, the fp64 loss sums and the head weight / bias gradients to summation order); a run of
 * UNPREP_WGRAD records of one lane (one launch per 32).  Records that do not qualify, or that would fail their own checks, take the ordinary
 * launchers; results and error reporting are otherwise those of record-by-record execution.
 */
int fnet_plan_run(const FnetOp* ops, int32_t n_ops, void* stream, int32_t* failed_index);
/* The hipStream_t behind side lane `lane` (1 .. FNET_MAX_LANES-1) of the current device, created on first use and owned by the
 * library.  No reference counterpart (the reference is single-stream): the data-parallel host uses it to order a gradient
 * bucket's RCCL all-reduce behind the lane that produced the bucket's last piece (fluidnet_amd/training/dp.py). */
int fnet_lane_stream(int32_t lane, void** stream_out);
/* Development / test control with no reference counterpart: overrides one of the launch heuristics that the library otherwise reads
 * from the environment once per process ("sa_minitems", "sa_cs", "sb_maxhw", "wg_px", "fuse_head", "wg_xcd" = FNET_SA_MINITEMS, FNET_SA_CS,
 * FNET_SB_MAXHW, FNET_WG_PX, FNET_FUSE_HEAD, FNET_WG_XCD; INTEGRATION.md "Development knobs").  value < 0 restores the environment's value or the default.  FNET_E_BADARG for an
 * unknown name.  Results never depend on a knob beyond summation order; production code does not call this. */
int fnet_set_knob(const char* name, int32_t value);

/*
 * hipGraph form of fnet_plan_run for launch-bound loops (the 600-frame rollout of
 * ml/scripts/simple_infer.py:226-260).  fnet_graph_create captures the plan on
 * a private capture stream (this call allocates the graph objects and synchronises nothing else);
 * fnet_graph_launch replays it `repeat` times on `stream`; fnet_graph_destroy frees it.
 */
int fnet_graph_create(const FnetOp* ops, int32_t n_ops, void** graph_out);
int fnet_graph_launch(void* graph, void* stream, int32_t repeat);
int fnet_graph_destroy(void* graph);

/*
 * Single-op conveniences used by the host mirror of the reference's free functions and by the
 * parity tests (each is fnet_plan_run on a one-element plan):
 *   fnet_spatial_gradients  <- compute_spatial_gradients  (ml/training/physics_loss.py:19-50)
 *   fnet_divergence         <- compute_divergence         (ml/training/physics_loss.py:53-91)
 * field planes are fp32 [B][H][W] contiguous.
 */
int fnet_spatial_gradients(const float* field, float* grad_x, float* grad_y, int32_t B, int32_t H, int32_t W,
                           float dx, float dy, int32_t padding_mode, int32_t stencil_mode, void* stream);
int fnet_divergence(const float* velx, const float* vely, float* div, int32_t B, int32_t H, int32_t W, float dx,
                    float dy, int32_t padding_mode, int32_t stencil_mode, void* stream);

/*
 * Allocation-free physics-loss terms.  NO counterpart in the reference: it exists for callers that cannot call hipMalloc -- code
 * under hipGraph capture, the viewer's per-frame loop, harnesses that forbid allocation.  Computes the forward terms of
 * PhysicsAwareLoss (ml/training/physics_loss.py:210-278) exactly as fnet_plan_run does for the op sequence ZERO(sums) + LOSS_REDUCE +
 * LOSS_FINALIZE, but the eight fp64 sums those kernels need live in a 256-byte static __device__ array of the library (one copy per
 * GPU, held until the process ends) instead of a caller buffer; no hipMalloc / hipFree / allocating routine is called.
 *   pred [B,3,H,W]; target / density_in / emitter / collider: planes with the given batch strides (floats), as LOSS_REDUCE;
 *   flags bit0 divergence, bit1 gradient, bit2 emitter term; terms_out: DEVICE float[8] = mse, divergence, gradient, emitter, total,
 *   fluid-cell count (written on `stream`).
 * Limit: B*H*W <= 2^30 cells, else FNET_E_TOO_LARGE.  All calls on one GPU share the array (cleared at the start of every call):
 * calls that overlap on one GPU -- two streams or two threads -- race on it; serialise them.
 */
int fnet_physics_loss_terms_noalloc(const float* pred, const float* target, const float* density_in, const float* emitter,
                                    const float* collider, int32_t B, int32_t H, int32_t W, int32_t target_bstride, int32_t density_bstride,
                                    int32_t emitter_bstride, int32_t collider_bstride, int32_t padding_mode, int32_t stencil_mode, int32_t flags,
                                    float grid_spacing, float w_mse, float w_div, float w_grad, float w_emit, float* terms_out, void* stream);

/*
 * HIP-event timing of a stream region, on the stream the kernels were launched on (bench.py
 * uses this for roofline.achieved; torch.cuda.Event only sees torch's current stream).
 * fnet_timer_create allocates two events; start/stop record them; elapsed_ms synchronises on the
 * stop event and returns milliseconds.
 */
int fnet_timer_create(void** timer_out);
int fnet_timer_start(void* timer, void* stream);
int fnet_timer_stop(void* timer, void* stream);
int fnet_timer_elapsed_ms(void* timer, float* ms_out);
int fnet_timer_destroy(void* timer);

/*
 * Native inference rollout: the per-step work of the reference's C++ viewer
 * (engine/src/Simulation.cpp:236-367: pack six planes, Ort::Session::Run, copy the output into
 * the back buffer) as one device-resident loop.  Model family: the four shipped architectures' block
 * types (instance / batch / group norm, stride or pooled downsample, nearest or bilinear upsample);
 * weights = the float tensors of a reference checkpoint in state-dict order (ml/models/unet.py:204-279;
 * BatchNorm2d: weight, bias, running_mean, running_var -- not its int64 counter), concatenated as fp32;
 * bf16 MFMA arithmetic.
 *   fnet_unet_param_count   number of floats fnet_rollout_create expects for a configuration
 *   fnet_rollout_create     allocates every device buffer (hipMalloc), uploads and re-lays the weights,
 *                           captures one frame in a hipGraph; synchronises
 *   fnet_rollout_set_weights / set_masks / set_state   host -> device uploads (null = zeros); synchronise
 *   fnet_rollout_add_impulse  velx += ix, vely += iy from a host [B][2][H][W] array (Simulation.cpp:263-271) on `stream`; synchronises
 *                           `stream` before returning, so the host array may be reused or freed at once
 *   fnet_rollout_step       `frames` graph replays on `stream`: state_prev <- density, state <- UNet(state, prev, masks)
 *   fnet_rollout_state_ptr  device pointers of the state [B][3][H][W] and the previous density [B][H][W]
 *   fnet_rollout_read_state device -> host copy of the state; synchronises `stream`
 */
typedef struct FnetUNetConfig {
    int32_t in_channels;        /* 6 */
    int32_t out_channels;       /* 3 */
    int32_t base_channels;      /* multiple of 4, <= 64 (not a multiple of 8: those tensors run zero-padded) */
    int32_t depth;
    int32_t act;                /* FNET_ACT_* */
    int32_t padding_mode;       /* FNET_PAD_* */
    int32_t upsample;           /* 0 nearest, 1 bilinear */
    int32_t use_residual;       /* 0 / 1 */
    int32_t bottleneck_blocks;
    int32_t output_activation;  /* FNET_OUT_* */
    int32_t norm;               /* 0 instance, 1 batch (eval mode: running statistics), 2 group */
    int32_t downsample;         /* 0 stride-2 conv, 1 avgpool + conv, 2 maxpool + conv */
    int32_t group_norm_groups;  /* norm == 2: the reference's `groups` (largest divisor of the channel count <= it is used) */
} FnetUNetConfig;
int fnet_unet_param_count(const FnetUNetConfig* cfg, int64_t* n_floats);
int fnet_rollout_create(const FnetUNetConfig* cfg, const float* host_params, int64_t n_params, int32_t B, int32_t H, int32_t W,
                        void** handle_out);
int fnet_rollout_set_weights(void* handle, const float* host_params, int64_t n_params);
int fnet_rollout_set_masks(void* handle, const float* host_emitter, const float* host_collider);
int fnet_rollout_set_state(void* handle, const float* host_state, const float* host_prev_density);
int fnet_rollout_add_impulse(void* handle, const float* host_impulse_xy, void* stream);
int fnet_rollout_step(void* handle, int32_t frames, void* stream);
int fnet_rollout_state_ptr(void* handle, float** device_state, float** device_prev_density);
int fnet_rollout_read_state(void* handle, float* host_state, void* stream);
int fnet_rollout_destroy(void* handle);

/*
 * Norms around a residual block, with its gate and residual scale, over the last axis of row-major operands (a row = one token, or one
 * pixel of a channels-last image).  No reference counterpart (its blocks normalise over pixels, ml/models/unet.py:17-28); the host
 * mirror is fluidnet_amd/models/block_norm.py.
 *   N(v) = v / sqrt(mean v^2 + eps)  or  (v - mean) / sqrt(var + eps)
 *   u = POST ? N(branch) * post_weight + post_bias : branch
 *   y = x + residual_scale * scale[c] * act(gate) * u           (branch == 0: y = x, nothing written)
 *   h = N(y) * pre_weight + pre_bias                            (h == 0: not computed; y is taken before it is rounded)
 * Row r of an operand starts at r * its row stride (elements); the elements of a row are adjacent.  y, h, dx, dbranch and an elementwise
 * dgate are dense.  Any alignment of the element size.  Absent pointers are 0 (an absent weight is 1, an absent bias 0).  Statistics, sums
 * and products are 32-bit; sums over rows are taken in a fixed order.
 * Backward recomputes y from x, branch and gate, and reads the forward's stats.  Gradients whose pointer is 0 are not computed.
 */
#define FNET_NORM_RMS 0
#define FNET_NORM_LAYER 1
#define FNET_GATE_NONE 0
#define FNET_GATE_ELEMENT 1   /* a value per element */
#define FNET_GATE_TOKEN 2     /* a value per row */
#define FNET_GATE_SAMPLE 3    /* a row of values per `tokens` consecutive rows */
#define FNET_GATE_CHANNEL 4   /* one row of values for all rows */
#define FNET_GATE_IDENTITY 0
#define FNET_GATE_SIGMOID 1
#define FNET_GATE_TANH 2
#define FNET_BLOCK_NORM_MAX_WIDTH 16384
typedef struct FnetBlockNorm {
    int64_t rows;             /* < 2^31 */
    int64_t tokens;           /* rows per sample (FNET_GATE_SAMPLE; divides rows) */
    int64_t x_stride, branch_stride, gate_stride, dy_stride, dh_stride;   /* row strides; gate_stride: of a row / sample of the gate */
    int32_t width;            /* 1 .. FNET_BLOCK_NORM_MAX_WIDTH */
    int32_t dtype;            /* x, branch, y, h and their gradients */
    int32_t param_dtype;      /* weights, biases, scale and their gradients: FNET_F32 or dtype */
    int32_t gate_dtype;       /* gate and its gradient: FNET_F32 or dtype */
    int32_t kind, post;       /* FNET_NORM_*; 1: the branch is normalised */
    int32_t gate_kind, gate_act;
    float residual_scale, eps;
    uint64_t x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias;
    uint64_t y, h;            /* forward results */
    uint64_t stats;           /* float [4][rows]: mean and 1/deviation of the branch, then of y; 0: not kept (forward only) */
    uint64_t dy, dh;          /* 0: zero */
    uint64_t dx, dbranch, dgate, dscale, dpost_weight, dpost_bias, dpre_weight, dpre_bias;
    uint64_t workspace;       /* backward: fnet_block_norm_workspace bytes, 16-byte aligned */
    int64_t workspace_bytes;
} FnetBlockNorm;
int fnet_block_norm_fwd(const FnetBlockNorm* host_args, void* stream);
int fnet_block_norm_bwd(const FnetBlockNorm* host_args, void* stream);
/* bytes of workspace that fnet_block_norm_bwd needs for these arguments (0 if none); host only */
int fnet_block_norm_workspace(const FnetBlockNorm* host_args, int64_t* bytes);

/*
 * Lists of tensors: the global gradient norm, clipping in place and a clipped Adam step, for any number of separate tensors of the three
 * element types (ml/training/trainer.py:190-195; FNET_OP_GRAD_NORM / FNET_OP_ADAM are the same for one flat fp32 buffer).  The list
 * is given by host arrays of device addresses, element counts and types, read during the call and passed on as kernel arguments; a dense
 * tensor of any layout is its memory in order.  Entries of no elements are skipped.  All of it is capturable.
 *   fnet_list_norm_partials  sums of squares / of absolutes / maxima of the list's parts in 64 bits, *n_partials of them (at most `capacity`,
 *                            which 2048 + n / 64 + 256 * n_strided + 8 always covers); `clock`, if not 0, is advanced as one Adam step
 *   fnet_list_clock          advances clock = (t, beta1^t, beta2^t) alone
 *   fnet_list_norm_finish    the norm itself from the partials
 *   fnet_list_scale          g *= min(1, max_norm / (norm + 1e-6)), the norm taken from the partials, or from *norm if those are 0; the
 *                            norm is also stored to *norm_out if that is not 0, for a list of no elements too.  FNET_E_OVERLAP if two
 *                            dense tensors share memory
 *   fnet_list_adam           one whole step: norm, clock, update.  Parameters that are not fp32 have an fp32 master that is updated and of
 *                            which they are the rounding.  FNET_E_OVERLAP if what is written shares memory, with itself or with a gradient
 */
#define FNET_LIST_MAXDIM 6
#define FNET_LIST_NORM_2 0
#define FNET_LIST_NORM_1 1
#define FNET_LIST_NORM_INF 2
typedef struct FnetStridedTensor {    /* a tensor that is no dense block: sizes and strides (elements, positive, no overlap) */
    uint64_t ptr;
    int32_t dtype, ndim;
    int64_t size[FNET_LIST_MAXDIM], stride[FNET_LIST_MAXDIM];
} FnetStridedTensor;
typedef struct FnetAdamList {
    double lr, beta1, beta2, eps, weight_decay;
    double max_norm;          /* < 0: no clipping */
    double* partials;         /* device, for clipping: `capacity` values of workspace, as in fnet_list_norm_partials */
    double* clock;            /* device: t, beta1^t, beta2^t of the steps done so far; advanced */
    const double* lr_device;  /* device, or 0: lr */
    float* norm_out;          /* device, or 0: the 2-norm of the gradients before clipping */
    int32_t capacity;
} FnetAdamList;
int fnet_list_norm_partials(int32_t n, const uint64_t* host_ptr, const int64_t* host_numel, const int32_t* host_dtype, int32_t n_strided,
                            const FnetStridedTensor* host_strided, int32_t norm_kind, double* partials, int32_t capacity,
                            int32_t* n_partials, double* clock, double beta1, double beta2, void* stream);
int fnet_list_clock(double* clock, double beta1, double beta2, void* stream);
int fnet_list_norm_finish(const double* partials, int32_t n_partials, int32_t norm_kind, float* norm_out, void* stream);
int fnet_list_scale(int32_t n, const uint64_t* host_ptr, const int64_t* host_numel, const int32_t* host_dtype, int32_t n_strided,
                    const FnetStridedTensor* host_strided, const double* partials, int32_t n_partials, int32_t norm_kind, const float* norm,
                    double max_norm, float* norm_out, void* stream);
int fnet_list_adam(int32_t n, const uint64_t* host_param, const uint64_t* host_grad, const uint64_t* host_exp_avg, const uint64_t* host_exp_avg_sq,
                   const uint64_t* host_master, const int64_t* host_numel, const int32_t* host_dtype, const FnetAdamList* host_args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FLUIDNET_HIP_H */
