/*
 * persistent_lstm_hip.h -- C ABI of the MI355X (gfx950) stacked LSTM + Linear inference forward and of the operators of
 * a residual block around a recurrence that is parallel over time (at the end).
 *
 * Library: persistent_lstm_hip_amd/lib/libpersistent_lstm_hip.so
 *
 * Conventions
 *   - Every pointer named *_dev, and every tensor argument, is device memory on the current HIP
 *     device.  fp16 tensors are IEEE binary16 (torch.float16), row-major, contiguous.
 *   - `stream` is a hipStream_t (may be NULL for the null stream).  Entry points only enqueue
 *     work on that stream; none of them synchronises except plh_status().
 *   - Return value: PLH_OK, or an error code; plh_last_error() gives the calling thread's message.
 *     PLH_ERR_INVALID and PLH_ERR_UNSUPPORTED correspond to the reference's std::invalid_argument
 *     (Python ValueError, persistent_lstm_op.cpp:7-11); PLH_ERR_HIP to its std::runtime_error with
 *     the hipGetErrorString text (Python RuntimeError, persistent_lstm_hip.cu:1730-1735).
 *   - Model geometry: I = input size, H = hidden size, L = layers, O = Linear output size
 *     (O = 0: no head).  Gate order along the 4H axis is i, f, g, o as in torch.nn.LSTM.
 *   - Numerics: fp16 weights and activations, fp32 MFMA accumulation, c kept in fp32, h rounded
 *     to fp16 every step, fused bias b_ih + b_hh summed in fp32, head accumulated in fp32 and
 *     written as fp16.
 *
 * Reference interface each entry point replaces (mantuoluozk/persistent_lstm_hip):
 *   bindings.cpp:154-165 exports the pybind functions the Python dispatcher calls.  The weight
 *   repacking that model.py:542-582 / :20-27 does on the Python side becomes plh_pack_regressor,
 *   and the family of fixed-shape forwards collapses into plh_forward.
 */
#ifndef PERSISTENT_LSTM_HIP_H
#define PERSISTENT_LSTM_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PLH_OK 0
#define PLH_ERR_INVALID 1     /* bad argument (shape, size, null pointer)        -> ValueError   */
#define PLH_ERR_UNSUPPORTED 2 /* geometry outside what the kernels implement      -> ValueError   */
#define PLH_ERR_HIP 3         /* HIP runtime error                                -> RuntimeError */
#define PLH_ERR_DEVICE 4      /* the persistent kernel reported a failure status  -> RuntimeError */

/* Bits of the device status word read by plh_status(). */
#define PLH_STATUS_TIMEOUT 1u /* a layer hand-off wait exceeded its time limit; outputs are NaN */

/* ABI version of this header. */
int plh_abi_version(void);

/* Message describing the last error raised on the calling thread ("" if none). */
const char* plh_last_error(void);

/* 1 if plh_forward implements this geometry, else 0 (plh_last_error() says why): 1 <= H <= 1024, any
 * input size up to 65536, L <= 64, O <= 4096 (the reference's generic entry point serves
 * 1 <= H <= 1024 and any input size, model.py:154-165, persistent_lstm_hip.cu:2981-2991).
 * Replaces the shape predicates PersistentLSTMRegressor._can_use_specialized_regressor_hip
 * (model.py:432-441) and NativeModuleFallback._can_use_generic_projected_module (model.py:131-165). */
int plh_supports(int input_size, int hidden_size, int num_layers, int output_size);

/* Bytes of the packed-weight blob for a geometry (negative on invalid geometry). */
int64_t plh_packed_bytes(int input_size, int hidden_size, int num_layers, int output_size);

/*
 * Pack torch-layout fp16 parameters into the kernel's resident-weight layout.
 *   w_ih[l]: weight_ih_l{l} [4H, l == 0 ? I : H]      w_hh[l]: weight_hh_l{l} [4H, H]
 *   b_ih[l], b_hh[l]: [4H] (b_hh[l] or the whole b_hh array may be NULL: treated as zero, which also
 *                     lets a caller pass the reference's pre-fused bias b_ih + b_hh in b_ih)
 *   lin_w [O, H], lin_b [O] (ignored when O == 0)
 * w_ih, w_hh, b_ih, b_hh are HOST arrays of L device pointers.
 * Replaces the repack cache fill of model.py:542-582 (kpairs packing, model.py:20-27) and the
 * per-call weight handling of persistent_lstm_regressor_forward_generic_projected_hip
 * (persistent_lstm_hip.cu:2923-3000).
 */
int plh_pack_regressor(int input_size, int hidden_size, int num_layers, int output_size,
                       const void* const* w_ih, const void* const* w_hh, const void* const* b_ih,
                       const void* const* b_hh, const void* lin_w, const void* lin_b,
                       void* packed_dev, int64_t packed_bytes, void* stream);

/* Bytes of device workspace plh_forward needs for (geometry, batch, seq_len).  At padded H 512 it
 * depends on the path the launch plan picks for that batch and length (the layer-sequential one
 * holds a layer's input projection for every step: about 3 MB per step at 512 rows). */
int64_t plh_workspace_bytes(int input_size, int hidden_size, int num_layers, int output_size, int batch,
                            int seq_len);

/*
 * Stacked LSTM (+ optional Linear head) forward over x [batch, seq_len, I] fp16 (batch_first).
 *   lengths   device int32 [batch] or NULL.  NULL: every row runs seq_len steps.  Otherwise
 *             packed-sequence semantics: row b runs lengths[b] steps, its state is frozen after,
 *             out_seq is zero past its length and the head reads its state at its last step.
 *   h0, c0    device fp16 [L, batch, H] initial state, or NULL for zeros (nn.LSTM hx).
 *   out       device fp16 [batch, O]: Linear(h_n[L-1]) (= Linear(out_seq[:, -1]) for full rows).
 *   out_seq   device fp16 [batch, seq_len, H]: last layer's outputs, or NULL.
 *   h_n, c_n  device fp16 [L, batch, H] final states, or NULL.
 *   probe_steps device int32 [n_probe], strictly increasing step counts in [1, seq_len];
 *             probe_h / probe_c device fp32 [n_probe, L, batch, H] receive every layer's state
 *             after that many steps (h as rounded to fp16, c in fp32).  n_probe = 0: no probes.
 *   workspace device memory of at least plh_workspace_bytes(...) bytes, 256-byte aligned.
 * Any output pointer may be NULL.  Asynchronous on `stream`; forwards on different streams of one
 * device are ordered by the library (each needs the whole device co-resident): the first forward
 * on a second stream synchronises the device once, later ones wait on an event of the previous
 * forward when it was on another stream (not inside a stream capture).  Hidden sizes 513..1024, inputs wider
 * than the padded hidden size above 128, and at padded H 512 a batch that needs more wavefront launches than
 * there are layers run layer by layer: per layer the input projection of every step as one fp16
 * MFMA GEMM (plh_input_projection's kernel; for layer 0 with input_size <= 32 at H > 256 inside the
 * recurrent kernel), then a W_hh-only persistent kernel.  That path rounds the GEMM's x_t W_ih^T to
 * fp16 before the recurrent sum, as the reference's generic path does (persistent_lstm_hip.cu:
 * 2988-2994); the all-layers path keeps it in fp32, so at padded H 512 the batch size decides which
 * of the two roundings a row gets (both are within the tolerance; the rows after the last full launch of
 * a batch take the all-layers path where that is faster for their number).  At padded H 128 an input
 * wider than that has its layer-0 projections from the same GEMM, rounded to fp16, in front of launches
 * of all layers (short sequences of more than three layers, or of many layers in several launches:
 * layer by layer).
 * Replaces persistent_lstm4_forward_interleaved (bindings.cpp:157, persistent_lstm_hip.cu:2126-2254)
 * and persistent_lstm_regressor_forward_generic_projected (bindings.cpp:163,
 * persistent_lstm_hip.cu:2923-3181), whose signatures return only the [batch, O] head output;
 * the state/sequence/probe outputs serve the nn.LSTM drop-in (model.py:323-395) and drift checks.
 */
int plh_forward(const void* packed_dev, int input_size, int hidden_size, int num_layers, int output_size,
                const void* x, int batch, int seq_len, const int32_t* lengths, const void* h0,
                const void* c0, void* out, void* out_seq, void* h_n, void* c_n,
                const int32_t* probe_steps, int n_probe, float* probe_h, float* probe_c, void* workspace,
                int64_t workspace_bytes, void* stream);

/*
 * plh_forward of the head alone ([batch, O], full-length rows, zero initial state) for a batch whose rows
 * may all be equal, which the reference's dispatcher looks for on the host before every forward
 * (model.py:493-520) to run one row of it (model.py:628-645).  Where plh_detects_uniform() is 1 the forward
 * finds out on the device while it packs x, without a host synchronisation, and a batch of equal rows then
 * keeps one tile of the device busy; the outputs are those of plh_forward either way.  Where it is 0 every
 * row is computed (a caller that looks first saves more there: one row runs a smaller launch).
 */
int plh_detects_uniform(int input_size, int hidden_size, int num_layers, int output_size, int batch, int seq_len);
int plh_forward_detect(const void* packed_dev, int input_size, int hidden_size, int num_layers, int output_size,
                       const void* x, int batch, int seq_len, void* out, void* workspace, int64_t workspace_bytes,
                       void* stream);

/*
 * Time-parallel input projection: out[m][n] = sum_{j < k} x[m][j] * w[n][j] for m < rows, n < cols,
 * fp16 operands and result, fp32 accumulation (MFMA), e.g. one layer's x_t W_ih^T for all T steps
 * of a batch at once (rows = T * batch).
 *   w   device fp16 [cols][k] row-major
 *   blocked = 0: x device fp16 [rows][ldx], out [rows][ldo], row-major
 *   blocked = 1: x and out fragment-blocked, [rows / 16][ld / 32][64][8] halfs: element (r, c) at
 *            (((r / 16) * (ld / 32) + c / 32) * 64 + ((c % 32) / 8) * 16 + r % 16) * 8 + c % 8, so that
 *            every 16 rows x 32 columns are one contiguous 1 KB block (the layout of the
 *            layer-sequential path's layer inputs and projections; the faster form)
 * Requires k % 128 == 0, k <= 65536, cols % 128 == 0, ldx >= k and ldo >= cols multiples of 8
 * (blocked: of 32, and rows % 16 == 0), 16-byte aligned pointers (PLH_ERR_INVALID otherwise;
 * zero-pad K to meet them).  Asynchronous on `stream`.
 * Replaces the reference's torch::matmul input projections of fp16 tensors (the generic path's
 * x.matmul(W_ih^T), persistent_lstm_hip.cu:2988-2994; the projected path's, :2329-2379).
 */
int plh_input_projection(const void* x, int64_t ldx, const void* w, int k, void* out, int64_t ldo, int64_t rows,
                         int cols, int blocked, void* stream);

/*
 * plh_forward without a workspace argument, for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid allocation).  It uses a device
 * scratch array inside the library, PLH_NOALLOC_SCRATCH_BYTES (64 MiB, plh_noalloc_scratch_bytes()),
 * one per GPU, held until the process ends; it calls no allocating routine.  A forward whose
 * plh_workspace_bytes(...) exceeds it is rejected with PLH_ERR_INVALID before anything is enqueued
 * (e.g. the C2 shape fits up to about 64 rows at 1000 steps).  All calls on one GPU share its scratch:
 * calls that overlap on one GPU (different streams or threads) race; calls ordered on one stream do
 * not.  Everything the kernels read from the scratch is written or cleared by the same call.
 * No counterpart in the reference; outputs and arguments as plh_forward.
 */
#define PLH_NOALLOC_SCRATCH_BYTES ((int64_t)64 << 20)
int plh_forward_noalloc(const void* packed_dev, int input_size, int hidden_size, int num_layers, int output_size,
                        const void* x, int batch, int seq_len, const int32_t* lengths, const void* h0,
                        const void* c0, void* out, void* out_seq, void* h_n, void* c_n,
                        const int32_t* probe_steps, int n_probe, float* probe_h, float* probe_c, void* stream);
int64_t plh_noalloc_scratch_bytes(void);
/* plh_status for plh_forward_noalloc: synchronise `stream` and read the status word the last
 * plh_forward_noalloc on the current device left in its scratch (0 = success, else PLH_STATUS_*
 * bits).  Like the scratch, shared by every caller on that device.  No counterpart in the reference. */
int plh_noalloc_status(uint32_t* status, void* stream);

/* Synchronise `stream` and read the status word the last plh_forward left in `workspace`
 * (0 = success, else PLH_STATUS_* bits).  Returns PLH_OK or PLH_ERR_HIP. */
int plh_status(const void* workspace, uint32_t* status, void* stream);

/*
 * Optional timing of the persistent kernel alone (for benchmarks and profilers of the caller).
 * plh_kernel_timing(n) with n > 0 arms n pairs of HIP events for the calling thread: each later
 * plh_forward on this thread records one pair around its persistent launch(es) (on the
 * layer-sequential H512 path: around all its projection GEMMs and launches), until the n pairs
 * are used.  plh_kernel_timing(0) disarms.  Called again with the n it was armed with, it re-arms
 * the same events without creating any (no HIP call: a caller can arm before its warm-ups and
 * re-arm right before its timed forwards).  plh_kernel_timing_read synchronises on the recorded
 * events and returns the summed elapsed milliseconds and the number of timed forwards.
 * No counterpart in the reference (it only timed whole forwards from Python, LSTM-hip.py:80-91).
 */
int plh_kernel_timing(int max_forwards);
int plh_kernel_timing_read(double* total_ms, int* forwards);

/*
 * Bound on every wait between workgroups of the calling thread's later plh_forward calls, in
 * microseconds (default 2000000; limit_us <= 0 restores the default).  A wait that exceeds it sets
 * PLH_STATUS_TIMEOUT, fails every other wait of the launch and poisons the outputs with NaN, so
 * the kernel always ends.  Failure detection for hung co-resident workgroups; no counterpart in the
 * reference (its kernels spin without bound).
 */
int plh_set_wait_limit_us(int64_t limit_us);

/*
 * Failure injection for tests of the failure path: with step >= 0, the calling thread's later
 * plh_forward calls that run the layer-sequential path make one workgroup of each launch treat its
 * exchange wait at that step as timed out (PLH_STATUS_TIMEOUT, outputs NaN where not computed, every
 * kernel still ends normally).  step < 0 turns it off.  The other paths' first hand-off wait can be
 * made to time out with a small plh_set_wait_limit_us; this path's per-step waits finish too fast
 * for that.  No counterpart in the reference.
 */
int plh_inject_wait_failure(int step);

/* out[r, c] = in[0, c] for r < rows (fp16).  Replaces repeat_first_row
 * (bindings.cpp:164, persistent_lstm_hip.cu:1684-1695, :1784-1809). */
int plh_repeat_first_row(const void* in, void* out, int rows, int cols, void* stream);

/*
 * Diagnostic for benchmarks: the dense fp16 MFMA rate this GPU sustains with
 * v_mfma_f32_16x16x32_f16 (the recurrent kernels' instruction) on every CU, in TFLOP/s, and the
 * shader clock during that run, in GHz (about 30 ms on the current device and the null stream;
 * allocates and frees its own buffers).  No counterpart in the reference, which quotes no peak.
 */
int plh_probe_mfma_f16(double* tflops, double* clock_ghz);

/*
 * Operators of a residual block around a recurrence that is parallel over time, y = x + dropout(W_o scan(W_g norm(x))),
 * for training and serving.  No counterpart in the reference, whose recurrence is the LSTM's alone.
 *   - dtype names the element type of the activations (PLH_F16, PLH_BF16, PLH_F32); sums, statistics and states are
 *     fp32, rounded once where an activation is written.
 *   - Pointers need the alignment of their elements only (the workspaces: 16 bytes); strides are in elements.
 *   - Asynchronous on `stream`; no atomics, so that results are the same from call to call.  All can be captured in a
 *     HIP graph.
 */
#define PLH_F16 0
#define PLH_BF16 1
#define PLH_F32 2

/*
 * Gated linear recurrence over gates [batch][seq_len][parts * hidden], parts = 3 with an output gate (f, g, o), 2
 * without (f, g):
 *     a_t = sigmoid(f_t)   c_t = a_t c_{t-1} + (1 - a_t) g_t   out_t = sigmoid(o_t) c_t, or c_t
 *   gates     element (b, t, k) at b * stride_b + t * stride_t + k
 *   lengths   device int32 [batch] or NULL (every row runs seq_len steps): row b runs min(max(lengths[b], 0), seq_len)
 *             steps, its c stays as it is after them and its out is zero there.  What gates hold there is not read.
 *   c0        device fp32 [batch][hidden] or NULL for zeros
 *   out       [batch][seq_len][hidden], contiguous
 *   c_n       device fp32 [batch][hidden] or NULL: c after the last step
 *   states    device fp32 [plh_gated_scan_states(seq_len)][batch][hidden] or NULL: what the backward pass needs
 *   workspace device memory of plh_gated_scan_workspace_bytes(...) bytes (0 for many channels), 16-byte aligned,
 *             used until the call's work on `stream` is done; nothing is kept in it
 * seq_len = 1 is the step of a serving loop; c_n may then be c0 (in place).
 * Limits: hidden <= 2^24, batch * hidden <= 2^29, seq_len <= 2^30.
 */
int64_t plh_gated_scan_states(int64_t seq_len);
int64_t plh_gated_scan_workspace_bytes(int64_t batch, int64_t seq_len, int hidden);
int plh_gated_scan_forward(int dtype, int output_gate, const void* gates, int64_t stride_b, int64_t stride_t,
                           int64_t batch, int64_t seq_len, int hidden, const int32_t* lengths, const float* c0,
                           void* out, float* c_n, float* states, void* workspace, int64_t workspace_bytes,
                           void* stream);
/*
 * Its gradient: d_gates [batch][seq_len][parts * hidden] (contiguous; zero past a row's length) and d_c0 [batch][hidden]
 * (fp32, or NULL) from d_out [batch][seq_len][hidden] (contiguous; not read past a row's length) and d_cn (fp32
 * [batch][hidden], or NULL for zeros).  gates, lengths and states as in the forward call that wrote states.
 */
int plh_gated_scan_backward(int dtype, int output_gate, const void* gates, int64_t stride_b, int64_t stride_t,
                            int64_t batch, int64_t seq_len, int hidden, const int32_t* lengths, const float* states,
                            const void* d_out, const float* d_cn, void* d_gates, float* d_c0, void* workspace,
                            int64_t workspace_bytes, void* stream);

/*
 * Layer norm over the last dimension of x [rows][cols] (row r at r * stride):
 *     y = (x - mean) * rstd * weight + bias,   rstd = 1 / sqrt(variance + eps), the variance over cols elements
 *   weight, bias  [cols] of wdtype (PLH_F32 or dtype), either may be NULL (1 and 0)
 *   y             [rows][cols], contiguous
 *   mean, rstd    device fp32 [rows] or NULL: what the backward pass needs
 * Limits: cols <= 2^24.
 */
int plh_layer_norm_forward(int dtype, int wdtype, const void* x, int64_t stride, int64_t rows, int64_t cols,
                           const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                           void* stream);
/*
 * Its gradient: d_x [rows][cols] (contiguous), d_weight and d_bias [cols] of wdtype, each of the three or NULL.
 * d_y [rows][cols] contiguous.  workspace as above, of plh_layer_norm_workspace_bytes(...) bytes (partial sums of d_weight
 * and d_bias: at most 1024 rows, 64 where cols > 16384).
 */
int64_t plh_layer_norm_workspace_bytes(int64_t rows, int64_t cols);
int plh_layer_norm_backward(int dtype, int wdtype, const void* x, int64_t stride, int64_t rows, int64_t cols,
                            const void* weight, const float* mean, const float* rstd, const void* d_y, void* d_x,
                            void* d_weight, void* d_bias, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * out[e] = residual[e] + (keep(e) ? x[e] * 65536 / (65536 - threshold) : 0) for e < n (residual NULL: 0).  keep(e) is
 * r(e) >= threshold, 0 <= threshold <= 65536: an element is dropped with probability threshold / 65536, and then it
 * is not read into the result, infinity and NaN included.  r(e) are 16 bits of Philox4x32-10 with the key `seed` and
 * the counter (e / 8, offset), 64 bits each: the low (e even) or high half of output word (e % 8) / 2.  So a mask is
 * a function of (seed, offset, e) alone, needs no storage, and the gradient is the same call with d_out for x and no
 * residual.  offset_dev: NULL, or a device int64 that is added to `offset` when the kernel runs (a captured graph's
 * replays then get masks of their own).
 */
int plh_dropout_add(int dtype, const void* x, const void* residual, void* out, int64_t n, int threshold, uint64_t seed,
                    uint64_t offset, const int64_t* offset_dev, void* stream);

/*
 * Operators of a block around a selective state space scan, y = x + W_out scan(silu(conv(u)), dt, A, B, C, D, z), for
 * training and serving.  Conventions as above.
 */

/*
 * Causal convolution along time, a filter of `width` taps (1 to 8) per channel:
 *     acc[b, t, c] = bias[c] + sum_k weight[c, k] x[b, t - width + 1 + k, c]      y = silu(acc), or acc (silu = 0)
 *   x             element (b, t, c) at b * stride_b + t * stride_t + c
 *   weight, bias  [channels][width] and [channels] of wdtype (PLH_F32 or dtype); bias may be NULL (zeros)
 *   state         [batch][width - 1][channels]: the inputs before the first step, the oldest first, or NULL for zeros
 *   lengths       device int32 [batch] or NULL, as for the gated scan: y is zero past a row's length, x is not read there
 *   y             [batch][seq_len][channels], contiguous
 *   state_n       [batch][width - 1][channels]: the last width - 1 inputs of every row (of its state, where it is shorter);
 *                 not the memory of state
 * The step takes one input per row and a state; its state_n may be state (in place).
 * Limits: channels <= 2^22, seq_len <= 2^30, batch * channels <= 2^28, batch * channels * seq_len <= 2^35.
 */
int plh_causal_conv_forward(int dtype, int wdtype, const void* x, int64_t stride_b, int64_t stride_t, int64_t batch,
                            int64_t seq_len, int64_t channels, int width, const void* weight, const void* bias,
                            const void* state, const int32_t* lengths, int silu, void* y, void* state_n, void* stream);
int plh_causal_conv_step(int dtype, int wdtype, const void* x, int64_t stride_b, int64_t batch, int64_t channels,
                         int width, const void* weight, const void* bias, const void* state, int silu, void* y,
                         void* state_n, void* stream);
/*
 * Its gradient from d_y [batch][seq_len][channels] (contiguous; not read past a row's length) and d_state_n (or NULL for
 * zeros): d_x [batch][seq_len][channels] (contiguous, zero past a row's length), d_weight, d_bias (of wdtype) and d_state
 * (seq_len > 0), each of the four or NULL.  The workspace holds partial sums of d_weight and d_bias.
 */
int64_t plh_causal_conv_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int width);
int plh_causal_conv_backward(int dtype, int wdtype, const void* x, int64_t stride_b, int64_t stride_t, int64_t batch,
                             int64_t seq_len, int64_t channels, int width, const void* weight, const void* bias,
                             const void* state, const int32_t* lengths, int silu, const void* d_y,
                             const void* d_state_n, void* d_x, void* d_weight, void* d_bias, void* d_state,
                             void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Selective state space scan, for every row b, channel d and state n:
 *     dt = softplus(raw + dt_bias[d]), or raw + dt_bias[d] (softplus = 0)
 *     h_n <- exp(dt A[d, n]) h_n + dt u B[n]      y = sum_n C[n] h_n + D[d] u      out = y silu(z), or y (z NULL)
 *   u, dt, z       [batch][seq_len][channels], element (b, t, d) at b * stride[0] + t * stride[1] + d; dt holds raw
 *   B, C           [batch][seq_len][states], likewise
 *   A              [channels][states], not positive (a decay); D, dt_bias [channels], either may be NULL (zeros);
 *                  all of wdtype (PLH_F32 or dtype)
 *   lengths        device int32 [batch] or NULL, as for the gated scan: h stays as it is past a row's length, out is
 *                  zero there, and nothing is read
 *   h0, h_n        device fp32 [batch][channels][states], either may be NULL (zeros; not wanted)
 *   out            [batch][seq_len][channels], contiguous
 *   states_out     device fp32 [plh_selective_scan_states(seq_len)][batch][channels][states] or NULL: what the backward
 *                  pass needs
 * The step is seq_len = 1 without lengths, from h to h_n, which may be the same memory.
 * Limits: 1 <= states <= 64, channels <= 2^20, seq_len <= 2^30, batch * ceil(channels / 8) < 2^23 and, from 2^21 rows on,
 * <= 2^21, batch * seq_len * states <= 2^30; of the step batch * channels * lanes <= 2^32 - 256 with ceil(states / 4)
 * lanes, rounded up to a power of two.
 */
typedef struct plh_selective_scan_args {
  int dtype, wdtype;
  const void *u, *dt, *z, *B, *C;
  int64_t u_stride[2], dt_stride[2], z_stride[2], B_stride[2], C_stride[2];
  const void *A, *D, *dt_bias;
  const int32_t* lengths;
  int64_t batch, seq_len, channels;
  int states, softplus;
} plh_selective_scan_args;

int64_t plh_selective_scan_states(int64_t seq_len);
int64_t plh_selective_scan_workspace_bytes(int64_t batch, int64_t seq_len, int64_t channels, int states, int backward);
int plh_selective_scan_forward(const plh_selective_scan_args* args, const float* h0, void* out, float* h_n,
                               float* states_out, void* workspace, int64_t workspace_bytes, void* stream);
int plh_selective_scan_step(const plh_selective_scan_args* args, const float* h, void* out, float* h_n, void* stream);
/*
 * Its gradient from d_out [batch][seq_len][channels] (contiguous; not read past a row's length) and d_hn (fp32, or NULL for
 * zeros), with the args and the states of the forward call.  d_u, d_dt, d_z (required with z) [batch][seq_len][channels],
 * contiguous; d_B, d_C [batch][seq_len][states], contiguous; all zero past a row's length.  d_A, d_D, d_dt_bias of wdtype;
 * d_h0 fp32.  All but d_u, d_dt and d_z may be NULL.
 */
typedef struct plh_selective_scan_grads {
  void *d_u, *d_dt, *d_z, *d_B, *d_C;
  void *d_A, *d_D, *d_dt_bias;
  float* d_h0;
} plh_selective_scan_grads;
int plh_selective_scan_backward(const plh_selective_scan_args* args, const float* states, const void* d_out,
                                const float* d_hn, const plh_selective_scan_grads* grads, void* workspace,
                                int64_t workspace_bytes, void* stream);

/*
 * The Euclidean norm of all elements of `count` tensors together, and the tensors times min(1, max_norm / (norm + 1e-6)).
 *   dtypes, in, out, numel   host arrays of `count`; tensor i has numel[i] elements of dtypes[i], dense.  out[i] may be
 *                            in[i] (in place); out NULL: only the norm is wanted.  Tensors must not overlap otherwise.
 *   max_norm                 infinity: no limit
 *   norm                     device fp32
 * Squares are summed in 64 bits.  A norm of infinity scales by zero, of NaN by NaN.
 */
int64_t plh_clip_grad_norm_workspace_bytes(int64_t count, const int64_t* numel);
int plh_clip_grad_norm(int64_t count, const int* dtypes, const void* const* in, void* const* out, const int64_t* numel,
                       double max_norm, float* norm, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PERSISTENT_LSTM_HIP_H */
