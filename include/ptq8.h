/*
 * ptq8.h - C ABI of the B200-native (sm_100a) W8A8 / W4A8 quantized-conv engine and of its
 * token operators (per-token quantization, linear layers, experts).
 *
 * Drop-in boundary for the reference's int8 engine (PaperTigerL/ptq-int8-lab,
 * 06-gpu-int8/cpp).  Each entry point names the reference interface it
 * replaces.  Conventions: plain pointers and sizes; no entry point exits the
 * process (the reference's CUDA_CHECK calls std::exit, int8_engine.cuh:109-117);
 * every failure returns a nonzero status and the message is available from
 * ptq8_engine_last_error() or the caller's err buffer.  The engine owns its
 * device memory; the caller owns input / logits buffers and may provide the
 * CUDA stream.  One engine per device per host thread.
 */
#ifndef PTQ8_H
#define PTQ8_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PTQ8_ABI_VERSION 1

/* status codes */
#define PTQ8_OK 0
#define PTQ8_ERR_INVALID 1  /* bad argument / state / unsupported topology */
#define PTQ8_ERR_FORMAT 2   /* malformed PTQ2 / PTQW / PTQC file */
#define PTQ8_ERR_CUDA 3     /* CUDA runtime error */
#define PTQ8_ERR_TIMEOUT 4  /* a bounded device wait ran out; outputs invalid */

/* graph passes (ptq8_engine_build `passes` bit mask) */
#define PTQ8_PASS_CENTER_TAP 1 /* 07-tensorrt-deploy/scripts/push_optimize_onnx.py:36-93 */
#define PTQ8_PASS_DECOMPOSE 2  /* 07-tensorrt-deploy/scripts/push_decompose.py:99-202  */
/* generalised positional decomposition: per-position sub-convs of convs whose output
 * positions read different kernel slices (push_decompose.py:50-80 computes the slices; its
 * decompose() declines such geometries); taps that only read padding are skipped */
#define PTQ8_PASS_POSITIONAL 4

/* activation range modes (06-gpu-int8/cpp/ptq_quant.h:163) */
#define PTQ8_ACT_ABSMAX 0
#define PTQ8_ACT_MINMAX 1

typedef struct ptq8_model ptq8_model;
typedef struct ptq8_engine ptq8_engine;

int ptq8_abi_version(void);

/* ---- calibrated-model files ------------------------------------------------ */

/* Model::load(path, err) - 06-gpu-int8/cpp/ptq_model.h:72-91.
 * PTQW or PTQ2 by magic, strict EOF, topology validation (ptq_model.h:104-203);
 * also PTQ8, this engine's native package (weight codes, f32 scales and bits per conv,
 * W4 two codes per byte; layout in csrc/ptq8_model.hpp), which builds without
 * re-quantizing.  Returns NULL on failure with the reason in err. */
ptq8_model* ptq8_model_load(const char* path, char* err, size_t errlen);
void ptq8_model_free(ptq8_model* m);

/* Counters of Model (ptq_model.h:65-70,205-229): out[11] = {n_conv, n_block,
 * stem_pool, fc_in, fc_out, n_depthwise, n_grouped, n_relu6, n_residual2,
 * format (1 PTQW, 2 PTQ2, 3 PTQ8), convs per block}. */
int ptq8_model_info(const ptq8_model* m, int* out);
/* ConvSpec of conv i (ptq_model.h:46-55): {cout, cin, kh, kw, sh, sw, ph, pw, relu, groups}. */
int ptq8_model_conv(const ptq8_model* m, int i, int* meta10);
/* BlockSpec of block i (ptq_model.h:57-63). */
int ptq8_model_block(const ptq8_model* m, int i, int* convs, int cap, int* n_convs, int* ds, int* stride,
                     int* residual);
/* Borrowed pointers to conv i's fp32 weight/bias (i = -1: the FC).  A PTQ8 conv has no
 * fp32 weights (n_weight 0). */
int ptq8_model_weights(const ptq8_model* m, int i, const float** weight, size_t* n_weight, const float** bias);
/* Borrowed pointers to conv i's stored codes ([cout][cin*kh*kw], one per byte) and f32
 * per-channel scales, and its bits (8 / 4), from a PTQ8 package; bits 0 and NULL
 * pointers for a PTQ2 / PTQW conv.  No counterpart in the reference (its files hold fp32
 * weights that Int8Engine::build quantizes, int8_engine.cuh:208). */
int ptq8_model_codes(const ptq8_model* m, int i, const int8_t** codes, size_t* n_codes, const float** scales,
                     int* bits);

/* load_ptqc(path, n_expected, out, err) - 06-gpu-int8/cpp/ptq_model.h:425-503.
 * Writes n (lo, hi) pairs to lohi[2n] (cap = number of floats available). */
int ptq8_load_ptqc(const char* path, size_t n_expected, float* lohi, size_t cap, char* err, size_t errlen);

/* tensor_quant_from_range scale (ptq_quant.h:195-214), returned in float64 as the
 * reference oracle uses it (09-ptq-toolkit/ptq_toolkit/ref_int8.py:69-87). */
double ptq8_act_scale(float lo, float hi, int bits, int mode);
/* quantize_weight_per_channel_sym (ptq_quant.h:72-110): w[cout][k] -> codes, f32 scales. */
int ptq8_quantize_weight(const float* w, int cout, int k, int bits, int8_t* codes, float* scale32);

/* Activation codes computed on `device` by the engine's own device quantizer
 * (the epilogue path): codes[i] = clip(round_half_away(double(x[i]) / s), -128, 127)
 * with s = ptq8_act_scale(lo, hi, 8, mode) (ref_int8.py:89-91).  Test entry point.
 * The range is checked like load_ptqc checks PTQC entries (ptq_model.h:425-503):
 * non-finite lo/hi, lo > hi, or a mode other than PTQ8_ACT_ABSMAX / PTQ8_ACT_MINMAX
 * return PTQ8_ERR_INVALID before any device work. */
int ptq8_quantize_device(int device, const float* x_host, size_t n, float lo, float hi, int mode, int8_t* codes);

/* Same codes as ptq8_quantize_device, but the call allocates no device memory
 * (no cudaMalloc / cudaFree, no allocating library routine).  No counterpart in
 * the reference.  For callers that cannot allocate: a process whose free device
 * memory is held by another allocator (a framework's caching pool, a serving
 * process at its memory cap) where a cudaMalloc may fail, and code that cannot
 * take the device-wide synchronisation cudaFree implies while other streams run.
 *
 * The input and output stay the caller's host buffers.  The device staging for
 * them is a fixed array inside the library, one per device, holding at most
 * PTQ8_NOALLOC_MAX_VALUES values (4 MiB of floats + 1 MiB of codes); a larger n
 * is rejected with PTQ8_ERR_INVALID and a message in err, and so is a range or mode
 * that ptq8_quantize_device rejects.  Every call looks the array's device address up
 * (cudaGetSymbolAddress, with the device current), so the first call on a device
 * loads the module there: make it before any stream capture.  All calls on a device
 * share the array and leave their data in it, so calls that overlap in time (two host
 * threads on the same device) race and must be serialised by the caller.  Copies and
 * the kernel run on the legacy default stream; the call returns when the codes are on
 * the host.  err (may be NULL) receives "" on success. */
#define PTQ8_NOALLOC_MAX_VALUES (1u << 20)
int ptq8_quantize_device_noalloc(int device, const float* x_host, size_t n, float lo, float hi, int mode,
                                 int8_t* codes, char* err, size_t errlen);

/* ---- engine ---------------------------------------------------------------- */

/* Int8Engine construction on CUDA device `device` (int8_engine.cuh:130). */
ptq8_engine* ptq8_engine_create(int device);
void ptq8_engine_destroy(ptq8_engine* e);
const char* ptq8_engine_last_error(const ptq8_engine* e);

/* Int8Engine::build(model, w_bits, a_bits) - int8_engine.cuh:132-349.
 * layer_bits (nullable, n_layer_bits == n_conv): per-conv weight bits 8/4 from a
 * layer plan (09-ptq-toolkit/ptq_toolkit/quant/mixed.py:126-212).  `passes` is a
 * PTQ8_PASS_* mask applied to the quantized layers.  The model must outlive the
 * engine (the reference keeps a raw pointer, int8_engine.cuh:134). */
int ptq8_engine_build(ptq8_engine* e, const ptq8_model* m, int w_bits, int a_bits, const int* layer_bits,
                      int n_layer_bits, int passes);
/* Int8Engine::set_act_mode - int8_engine.cuh:353. */
int ptq8_engine_set_act_mode(ptq8_engine* e, int mode);
/* Int8Engine::set_calib(ranges) - int8_engine.cuh:362-406; lohi[2n]. */
int ptq8_engine_set_calib(ptq8_engine* e, const float* lohi, size_t n);
/* Network input geometry (default 3x32x32, ptq_model.h:104 validates with 32x32). */
int ptq8_engine_set_input_shape(ptq8_engine* e, int c, int h, int w);
/* Int8Engine::alloc_scratch(n) - int8_engine.cuh:807-833: plan the launches and
 * allocate every activation buffer for batches up to max_batch. */
int ptq8_engine_alloc_scratch(ptq8_engine* e, int max_batch);
/* Int8Engine::set_stream - int8_engine.cuh:771 (NULL: engine-owned stream). */
int ptq8_engine_set_stream(ptq8_engine* e, void* stream);
/* Cap the persistent grid of every tensor-core conv at max_ctas CTAs (0: one per SM,
 * the default) -- e.g. to leave SMs to other work.  No counterpart in the reference
 * (its kernels are launched per tile).  Drops captured graphs. */
int ptq8_engine_set_max_ctas(ptq8_engine* e, int max_ctas);
void* ptq8_engine_stream(ptq8_engine* e);

/* Int8Engine::forward(x_host, n, c, h, w, logits_host) - int8_engine.cuh:429-645.
 * Host buffers: H2D, the whole forward as one CUDA graph, D2H, synchronize. */
int ptq8_engine_forward(ptq8_engine* e, const float* x_host, int n, int c, int h, int w, float* logits_host);
/* Pipelined host-buffer forward (no counterpart in the reference, whose forward is
 * synchronous): enqueues the H2D copy of x_host into one of two engine input slots on
 * an engine-owned copy stream, the forward (CUDA graph) on the engine stream once that
 * copy has landed, and the D2H copy of the logits; returns without waiting.  The H2D of
 * call k+1 overlaps the forward of call k.  ptq8_engine_sync() waits for every enqueued
 * call.  x_host (pinned, for the copies to overlap) must stay unchanged and logits_host
 * unread until then.  Same logits as ptq8_engine_forward.  The engine's other calls
 * that take or run on an input (forward, forward_device, run, input_buffer, profile,
 * ptq8_forward / ptq8_forward_debug) first wait for pipelined copies still in flight. */
int ptq8_engine_forward_async(ptq8_engine* e, const float* x_host, int n, float* logits_host);
/* Device-pointer forward (fp32 NCHW input, fp32 [n][fc_out] logits); enqueued
 * on the engine stream, not synchronized. */
int ptq8_engine_forward_device(ptq8_engine* e, const float* x_dev, int n, float* logits_dev);
/* ---- 8-bit pixel input (CIFAR-10 records) ----------------------------------
 * The reference decodes CIFAR-10 records and normalises them on the host, then
 * uploads fp32 (ref_e2e.py:261-276; main.cpp:178-198,245-261).  These calls upload the
 * 8-bit pixels (1 byte per value instead of 4) and the stem kernel does the
 * normalisation and the exact quantization on the device: the same network input
 * codes, bit for bit, as the reference's fp32 path, given the same normalisation.
 * Pixels are [n][c][h][w] bytes per image; image i starts at x + i * record_bytes
 * (record_bytes 0: c*h*w, packed; a raw CIFAR-10 batch file is x = file + 1,
 * record_bytes = 3073, skipping each record's label byte).  At most 4 channels. */
#define PTQ8_NORM_DIV 0 /* x = (px - mean*255) / (std*255): ref_e2e.py:272-274 (the default) */
#define PTQ8_NORM_MUL 1 /* x = ((px/255)*255 - mean*255) * (1/(std*255)): main.cpp:245-261 */
/* Normalisation of 8-bit input (mode PTQ8_NORM_*; mean/std: float[c], or both NULL for the
 * CIFAR-10 constants of main.cpp:25-26).  Every operation in float32, rounded to nearest.
 * Drops captured 8-bit-input graphs. */
int ptq8_engine_set_input_norm(ptq8_engine* e, int mode, const float* mean, const float* std_);
/* Int8Engine::forward (int8_engine.cuh:429) from 8-bit host pixels: H2D of the pixels,
 * the forward as one CUDA graph, D2H of the logits, synchronize. */
int ptq8_engine_forward_u8(ptq8_engine* e, const uint8_t* x_host, int n, size_t record_bytes, float* logits_host);
/* Pipelined form of ptq8_engine_forward_u8, with the semantics of ptq8_engine_forward_async
 * (same two input slots and copy stream; wait with ptq8_engine_sync). */
int ptq8_engine_forward_u8_async(ptq8_engine* e, const uint8_t* x_host, int n, size_t record_bytes,
                                 float* logits_host);
/* Device-pointer form (8-bit pixels on the device, fp32 logits [n][fc_out]); enqueued on
 * the engine stream, not synchronized. */
int ptq8_engine_forward_device_u8(ptq8_engine* e, const uint8_t* x_dev, int n, size_t record_bytes,
                                  float* logits_dev);

/* Engine-resident buffers: callers may write inputs straight into the input
 * buffer and run ptq8_engine_run() with no copies. */
float* ptq8_engine_input_buffer(ptq8_engine* e);
float* ptq8_engine_logits_buffer(ptq8_engine* e);
int ptq8_engine_run(ptq8_engine* e, int n, int use_graph);
/* Async device-to-device copy of the last forward's logits ([n][fc_out]) on the engine stream. */
int ptq8_engine_copy_logits(ptq8_engine* e, int n, float* dst_dev);
int ptq8_engine_sync(ptq8_engine* e);
/* Reads and clears this engine's device error word, set by bounded waits that ran out
 * (PTQ8_ERR_TIMEOUT; each engine has its own word, so one engine's timeout never
 * aborts or reports through another).  No counterpart in the reference (its kernels
 * have no waits; CUDA errors exit, int8_engine.cuh:109-117). */
int ptq8_engine_check_device_error(ptq8_engine* e);
/* Failure-detection test hook, no counterpart in the reference.  Sets the limit of
 * every bounded device wait of this engine's kernels in clock cycles (0: the default,
 * about 2 s) and, when stall_first_load is nonzero, makes the first operand load of
 * the forward's first tensor-core conv (CTA 0) never arrive, so that the waits on it
 * run out: the forward then reports PTQ8_ERR_TIMEOUT through
 * ptq8_engine_check_device_error / ptq8_engine_sync / ptq8_engine_forward instead of
 * hanging, and the context stays usable.  Drops captured graphs. */
int ptq8_engine_set_wait_test(ptq8_engine* e, long long wait_limit_cycles, int stall_first_load);

/* Parity dumps (replaces forward(..., stop_after_block, mid_out),
 * int8_engine.cuh:429 and locate_block.cpp): what 0 = int8 input codes of conv
 * `index` (NHWC, row pitch shape4[3]; the stem's are its im2col rows), what 1 =
 * the fp32 map fed to the pooling head (NHWC).  shape4 = {N_max, H, W, ld}. */
int ptq8_engine_tensor_info(ptq8_engine* e, int what, int index, int* shape4);
int ptq8_engine_dump(ptq8_engine* e, int what, int index, int n, void* host_dst, size_t bytes);
/* The same for images [n0, n0 + n) of the last forward (the reference oracle runs and
 * dumps a batch chunk by chunk, 06-gpu-int8/cpp/ref_e2e.py:308-329): parity checks of a
 * full-size batch without copying whole multi-GB maps to the host. */
int ptq8_engine_dump_range(ptq8_engine* e, int what, int index, int n0, int n, void* host_dst, size_t bytes);
/* Per-launch timing (CUDA events on the engine stream, `iters` back-to-back
 * launches of each step, not graph-captured) with each step's algorithmic work:
 * ms[i], macs[i], bytes[i], kind[i] (0 stem im2col + GEMM, 1 tensor-core conv,
 * 2 depthwise, 3 maxpool, 4 pooling head) for i < *n_steps (cap entries available).
 * Replaces the reference's PROF_LAYERS per-conv events (int8_engine.cuh:168-176,901-931). */
int ptq8_engine_profile(ptq8_engine* e, int n, int iters, float* ms, double* macs, double* bytes, int* kind,
                        int cap, int* n_steps);
/* Number of kernel launches in one forward (the CUDA graph's kernel nodes). */
int ptq8_engine_n_launches(const ptq8_engine* e);
/* Conv weight bytes the planned engine keeps in device memory, the bytes the same
 * weights take as int8 codes, and how many convs hold W4 codes packed two per byte
 * (W4 convs whose weight slab stays resident in shared memory, and depthwise W4
 * tables).  No counterpart in the reference, whose PTQ2 stores W4 layers as fp32 QDQ
 * values (09-ptq-toolkit/ptq_toolkit/pipeline.py:272-279) and whose engine holds
 * every code as a byte (int8_engine.cuh:211-276). */
int ptq8_engine_weight_bytes(const ptq8_engine* e, size_t* device_bytes, size_t* int8_bytes, int* packed_convs);
/* Human-readable record of what the graph passes did. */
int ptq8_engine_passes_log(const ptq8_engine* e, char* out, size_t cap);

/* ---- one-call interface ----------------------------------------------------
 * The same engine behind five calls, for callers that do not need the steps
 * above.  Status codes only (the reference's forward exits on CUDA errors,
 * int8_engine.cuh:109-117); messages via ptq8_last_error. */

typedef struct ptq8_opts {
    int device;      /* CUDA device ordinal */
    int w_bits;      /* weight bits (8 or 4) when no layer plan is given (Int8Engine::build w_bits) */
    int a_bits;      /* activation bits: 8 */
    int act_mode;    /* PTQ8_ACT_ABSMAX (default, ref_int8.py:69-87) or PTQ8_ACT_MINMAX */
    int passes;      /* PTQ8_PASS_* bits: graph passes on the quantized layers */
    int max_batch;   /* device scratch for this many images; 0: sized by the first forward */
} ptq8_opts;

/* Model::load (ptq_model.h:72) + load_ptqc (:425) + layer plan (mixed_check.py:62-81,
 * per-layer bits 4/8, per_channel only) + Int8Engine::build / set_act_mode /
 * set_calib / alloc_scratch (int8_engine.cuh:132,353,362,807) in one call.  PTQ2
 * and PTQW files are accepted unchanged; plan_json may be NULL.  opts NULL means
 * {device 0, W8, A8, AbsMax, no passes, max_batch 0}.  The engine owns the model.
 * On failure *out is NULL and err holds the message. */
int ptq8_load(const char* model_path, const char* calib_path, const char* plan_json, const ptq8_opts* opts,
              ptq8_engine** out, char* err, size_t errlen);
/* Forward of n images (fp32 NCHW at x_dev) into logits_dev [n][fc_out], both device
 * pointers, asynchronous on `stream` (NULL: the engine's stream).  Replaces
 * Int8Engine::forward (int8_engine.cuh:429) without its host copies. */
int ptq8_forward(ptq8_engine* e, const float* x_dev, int n, float* logits_dev, void* stream);
/* ptq8_forward, then (synchronously) the int8 input codes of every conv, handed to
 * dump(user, conv, codes, n, h, w, ld) as a host array [n][h][w][ld] (the stem's
 * are its im2col rows) -- the parity hook that replaces forward(...,
 * stop_after_block, mid_out) and locate_block.cpp. */
typedef void (*ptq8_dump_fn)(void* user, int conv, const int8_t* codes, int n, int h, int w, int ld);
int ptq8_forward_debug(ptq8_engine* e, const float* x_dev, int n, float* logits_dev, void* stream,
                       ptq8_dump_fn dump, void* user);
/* Capture (and cache) the CUDA graph of a forward at batch n ahead of the first
 * forward (the reference launches kernel by kernel with no graph). */
int ptq8_capture_graph(ptq8_engine* e, int n);
/* Destroy an engine and, when it came from ptq8_load, its model. */
void ptq8_destroy(ptq8_engine* e);
const char* ptq8_last_error(const ptq8_engine* e);

/* ---- token operators ---------------------------------------------------------
 *
 * The engine's arithmetic for a language model's layers: int8 activations with one
 * scale per token, int8 (or packed int4) weights with one scale per output channel,
 * exact int32 sums.  No reference counterpart (its engine runs convolutions with
 * static activation ranges).  All tensors are device memory of the handle's device;
 * every call only enqueues work on `stream` (a cudaStream_t, NULL: the legacy default
 * stream), allocates nothing and may be captured in a CUDA graph.  Row pitches are in
 * elements of the tensor, and may exceed the row's width.  A tensor is aligned to its
 * element type, or the call is refused.  One handle per device per
 * host thread; handles are independent of engines.  Forward only. */

typedef struct ptq8_ops ptq8_ops;

/* element types */
#define PTQ8_F32 0
#define PTQ8_F16 1
#define PTQ8_BF16 2

/* what a product does with its channels */
#define PTQ8_EPI_NONE 0
#define PTQ8_EPI_SWIGLU 1 /* weights hold 2*out_features channels, gate then up: y = silu(gate) * up */

/* int32 sums of in_features products of codes of magnitude <= 128 never overflow up to here */
#define PTQ8_MAX_IN_FEATURES 131071
#define PTQ8_MAX_GROUPS 1024
/* widest row of quantize_rows: its vectors of 4 or 8 values end within an int */
#define PTQ8_MAX_ROW_WIDTH 0x7FFFFFF0

ptq8_ops* ptq8_ops_create(int device, char* err, size_t errlen);
/* Waits for nothing: kernels of the handle may still run, and graphs that hold them may be replayed.  What a device
 * wait of theirs that runs out would report is lost with the handle; ptq8_ops_check_device_error comes before. */
void ptq8_ops_destroy(ptq8_ops* ops);
const char* ptq8_ops_last_error(const ptq8_ops* ops);
/* Waits for `stream`, then reports (and clears) a bounded device wait that ran out: PTQ8_ERR_TIMEOUT.
 * Until it is cleared here, every further call on the handle returns PTQ8_ERR_TIMEOUT too. */
int ptq8_ops_check_device_error(ptq8_ops* ops, void* stream);
/* Failure-detection test hook: wait limit in clock cycles (0: the default, about 2 s), and a switch that makes
 * a kernel with such waits (tensor-core products, cache_attention) announce its first operand load without issuing it. */
int ptq8_ops_set_wait_test(ptq8_ops* ops, long long wait_limit_cycles, int stall_first_load);

/* int8 codes with one scale per row (token):
 *   scale[r] = max(fl32(max_k |x[row(r)][k]| / 127), 1e-8)
 *   codes[r][k] = round_half_away(x[row(r)][k] / scale[r])   (the exact quotient; within +-127)
 * row(r) = rows[r], or r where rows is NULL.  A row whose index is outside [0, x_rows) gets codes 0 and scale 0.
 * A row that holds NaN or an infinity gets codes 0 and scale NaN or infinity, so that its products are NaN. */
typedef struct {
    const void* x;       /* [x_rows][width], pitch ldx */
    long long ldx;
    long long x_rows;
    const int* rows;     /* [n_rows] or NULL (then n_rows == x_rows) */
    long long n_rows;
    int8_t* codes;       /* [n_rows][width], pitch ldc; must not overlap x */
    long long ldc;
    float* scale;        /* [n_rows] */
    int width;
    int x_type;          /* PTQ8_F32 / F16 / BF16 */
} ptq8_rows_args;
int ptq8_quantize_rows(ptq8_ops* ops, const ptq8_rows_args* args, void* stream);

/* y[t][c] = fl(fl(float(sum_k x[t][k] * w[c][k]) * fl(x_scale[t] * w_scale[c])) + bias[c]), then the epilogue,
 * then one rounding to y's type.  w_bits 4: codes two per byte, code k in the low (k even) or high half of byte k/2.
 * The tensor-core kernels need x, w (and a group's weights) to start at multiples of 16 bytes and row pitches that
 * are multiples of 16 bytes; any other layout runs on a slower kernel.
 * ptq8_linear_grouped: rows offsets[g] .. offsets[g+1]-1 meet group g's weights (offsets: device memory, groups+1
 * values, not decreasing, within [0, rows]; values outside are clamped, and where they decrease no access leaves the
 * tensors, but rows of two groups may hold either's product); rows of no group are not written. */
typedef struct {
    const int8_t* x;       /* [rows][in_features], pitch ldx */
    long long ldx;
    const float* x_scale;  /* [rows] */
    const void* w;         /* [groups][channels][in_features], pitch ldw bytes, groups w_group_stride bytes apart */
    long long ldw;
    long long w_group_stride;
    const float* w_scale;  /* [groups][channels] */
    const float* bias;     /* [groups][channels] or NULL */
    void* y;               /* [rows][out_features], pitch ldy; must not overlap the inputs */
    long long ldy;
    const int* offsets;    /* ptq8_linear_grouped only */
    long long rows;
    int in_features;
    int out_features;      /* channels = out_features, or twice that with PTQ8_EPI_SWIGLU */
    int groups;            /* ptq8_linear_grouped only */
    int w_bits;            /* 8 or 4 */
    int epilogue;          /* PTQ8_EPI_* */
    int y_type;            /* PTQ8_F32 / F16 / BF16 */
} ptq8_linear_args;
int ptq8_linear(ptq8_ops* ops, const ptq8_linear_args* args, void* stream);
int ptq8_linear_grouped(ptq8_ops* ops, const ptq8_linear_args* args, void* stream);

/* Which kernel a product runs on.  Host only: no handle, no device, and the tensors are not read (their addresses'
 * alignment counts).  The answer is the one that a call with these arguments takes on a device of `sms` SMs. */
#define PTQ8_KERNEL_ANY 0   /* any layout */
#define PTQ8_KERNEL_FEW 1   /* a few tokens, weights streamed to registers */
#define PTQ8_KERNEL_TILES 2 /* tensor-core tiles: the fields below */
typedef struct {
    int kernel;             /* PTQ8_KERNEL_* */
    int variant;            /* index of the tile variant, 0 up to ptq8_linear_variants() - 1 */
    int ctas, tokens;       /* CTAs and tokens of a tile */
    int w_bits, epilogue;   /* what the variant serves */
    int split;              /* CTAs that share a tile's sum */
    int stages, turns;      /* shared-memory stages of a CTA; sets of int4 unpacking warps that take turns at them */
    int operand_tiles;      /* int4: widened weight tiles in TMEM */
    int smem_bytes;         /* dynamic shared memory of a CTA */
} ptq8_linear_choice;
int ptq8_linear_variants(void);
int ptq8_linear_choose(int sms, const ptq8_linear_args* args, int grouped, ptq8_linear_choice* choice);
/* The same for one variant and split, whatever the call would choose: PTQ8_ERR_INVALID where that pair cannot serve it. */
int ptq8_linear_choose_as(int sms, const ptq8_linear_args* args, int grouped, int variant, int split, ptq8_linear_choice* choice);
/* Test hook: products of this handle run as `variant` with `split` (-1: as they choose), or are refused where that pair
 * cannot serve them. */
int ptq8_ops_set_choice_test(ptq8_ops* ops, int variant, int split);

/* y[t][c] = sum_g w_scale[c][g] * (sum_{k in group g} code[c][k] * x[t][k]) + bias[c], then the epilogue, then one rounding to
 * y's type: float activations, 4-bit weights with a scale per `group` consecutive input features (the last group may be
 * shorter).  Codes lie as ptq8_linear's do with w_bits 4.  Sums are f32.
 * On the tensor cores an activation is an f16 number times a power of two that goes by the largest, top, of the 128 that it lies
 * among (from a multiple of 128 on): off by at most 2^-39 top, or 2^-35 top where its feature's number is odd.  f16 and bf16 ones
 * within 2^-24 of top are exact; f32 ones take two f16 numbers and are off by at most 2^-22 of themselves more.  (A top below 2^-100
 * counts as 2^-100.)  Outputs of a token that holds NaN or an infinity are NaN or infinite.
 * Groups of a multiple of 32 features (or of all) with weights and pitches at multiples of 16 bytes run on the tensor cores;
 * any other group and layout on a slower kernel. */
typedef struct {
    const void* x;         /* [rows][in_features], pitch ldx elements */
    long long ldx;
    const void* w;         /* [channels][in_features], two codes per byte, pitch ldw bytes */
    long long ldw;
    const void* w_scale;   /* [channels][groups], pitch lds elements */
    long long lds;
    const float* bias;     /* [channels] or NULL */
    void* y;               /* [rows][out_features], pitch ldy elements; must not overlap the inputs */
    long long ldy;
    long long rows;
    int in_features;
    int out_features;      /* channels = out_features, or twice that with PTQ8_EPI_SWIGLU */
    int group;
    int epilogue;          /* PTQ8_EPI_* */
    int x_type, scale_type, y_type;   /* PTQ8_F32 / F16 / BF16 */
    int reserved;
} ptq8_linear_w4_args;
int ptq8_linear_w4(ptq8_ops* ops, const ptq8_linear_w4_args* args, void* stream);

/* ---- the cache of keys and values in 4 bits --------------------------------------
 *
 * A row (one token, one head; of the keys or the values) is head_dim codes of 4 bits, code 2 i in the low and 2 i + 1 in the
 * high half of byte i, and a pair of bf16 numbers: step, then least.  Code c stands for least + step * c.  The rows of a
 * head lie one after another in pages of `page` tokens.  A sequence's positions 0, 1, .. lie in the pages that its row of
 * the table names, one after another; its length counts its positions, those of the new tokens among them, which are the
 * last ones: of n new tokens, token i has position length - n + i.  New tokens of all sequences lie one after another:
 * sequence b's are starts[b] .. starts[b + 1] - 1, or token b alone where starts is NULL.
 *
 * Table, lengths and starts are device memory and read on the device.  starts must not decrease; values outside
 * [0, tokens] are clamped, and where they decrease no access leaves the tensors, but a token may be taken for another
 * sequence's.  A position without a page (behind the table's row, before 0, or where the table names no page of the cache)
 * is not written, reads as zeros and is not attended to.  Codes and pairs, and all of their page and head strides, are
 * aligned to 16 bytes. */
#define PTQ8_MAX_SEQUENCES 1024
typedef struct {
    uint8_t* k;             /* codes [pages][kv_heads][page][head_dim / 2] */
    uint8_t* v;
    uint16_t* k_scale;      /* bf16 (step, least) [pages][kv_heads][page][2] */
    uint16_t* v_scale;
    long long k_page, k_head, v_page, v_head;                                 /* strides in bytes */
    long long k_scale_page, k_scale_head, v_scale_page, v_scale_head;
    const int* table;       /* [sequences][table_width], pitch table_pitch elements */
    long long table_pitch;
    const int* lengths;     /* [sequences] */
    const int* starts;      /* [sequences + 1] or NULL (then tokens == sequences) */
    long long pages;
    int table_width;
    int page;               /* tokens of a page: 16, 32, 64, .. 4096 */
    int kv_heads;
    int head_dim;           /* 64, 128 or 256 */
    int sequences;          /* up to PTQ8_MAX_SEQUENCES */
    int reserved;
} ptq8_cache;

/* ptq8_cache_write: the new tokens' keys and values into the cache, for each row x
 *   least = the largest bf16 number <= min x
 *   step = max(the smallest bf16 number >= fl32(fl32(max x - least) / 15), 2^-100)
 *   code = rint(fl32(fl32(x - least) * fl32(1 / step))) (halves to even), within 0 .. 15
 * A row that holds NaN or an infinity, or whose spread no float holds, gets codes 0 and NaN for both: whatever attends to
 * it is NaN.  A page that is written belongs to one sequence; where two write the same row it holds a mixture of theirs.
 * ptq8_cache_read: what the cache holds at the new tokens' positions, fl32(least + step * code), rounded once more to
 * `type`.  Tokens of no sequence are left as they were. */
typedef struct {
    ptq8_cache cache;
    void* k;                /* [tokens][kv_heads][head_dim], head_dim consecutive; read by ptq8_cache_write, */
    void* v;                /* written by ptq8_cache_read */
    long long k_token, k_head, v_token, v_head;   /* strides in elements */
    long long tokens;
    int type;               /* PTQ8_F32 / F16 / BF16 */
    int reserved;
} ptq8_cache_rows_args;
int ptq8_cache_write(ptq8_ops* ops, const ptq8_cache_rows_args* args, void* stream);
int ptq8_cache_read(ptq8_ops* ops, const ptq8_cache_rows_args* args, void* stream);

/* out[token][h] = sum_j p_j v_j, p = softmax_j(scale * q[token][h] . k_j), over the positions j up to the token's own, keys and
 * values of head h / (heads / kv_heads).  A token that sees no position gets zeros; tokens of no sequence are left as they
 * were.  Queries are f16 or bf16, the output has their type; sums and the softmax are f32, p (times the value's step) is rounded
 * to f16's 11 bits for its product with the codes less eight, 2^-30 of the largest step that the token sees being the finest.  Rows of keys or values that a token does not see have no part in its
 * output, whatever they hold.  Queries are f16 numbers times a power of two that goes by a row's largest: off by at most 2^-39 of it,
 * or 2^-35 in dimensions of odd number.  Any finite query is taken; keys up to 2^115, and scores (times log2(e)) as well as sums of p v
 * (p up to 2^8 a position, before they are divided by the sum of p), that f32 numbers hold.
 * workspace: device memory of ptq8_cache_attention_workspace() bytes, aligned to 16 bytes, which this call alone uses until its
 * kernels have run: calls on one stream may share it, calls on two streams or of two graphs that may run at once may not. */
typedef struct {
    ptq8_cache cache;
    const void* q;          /* [tokens][heads][head_dim], head_dim consecutive */
    void* out;              /* the same shape; must not overlap the inputs */
    long long q_token, q_head, out_token, out_head;   /* strides in elements */
    long long tokens;
    void* workspace;
    long long workspace_bytes;
    float scale;
    int heads;              /* a multiple of kv_heads */
    int type;               /* PTQ8_F16 / BF16 */
    int reserved;
} ptq8_cache_attention_args;
int ptq8_cache_attention(ptq8_ops* ops, const ptq8_cache_attention_args* args, void* stream);
/* Bytes that a call with these arguments needs (0: it needs none), or -1 where it is refused (see ptq8_ops_last_error).
 * Neither the tensors' addresses nor their contents count. */
long long ptq8_cache_attention_workspace(ptq8_ops* ops, const ptq8_cache_attention_args* args);

#ifdef __cplusplus
}
#endif

#endif /* PTQ8_H */
