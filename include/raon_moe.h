/*
 * raon_moe.h -- C ABI of librmoe.so, the MI355X (gfx950) quantized-MoE hot path.
 *
 * The library replaces the device side of raon-npu's NPU backend for the q4nx
 * mixture-of-experts path.  Every entry point below names the reference
 * interface it stands in for (paths inside the reference tree).  The Python
 * host mirror (raon-npu_amd/backend.py, class GpuBackend) binds these entry
 * points with ctypes and keeps the reference's Backend method signatures.
 *
 * Conventions
 *  - Every function returns an int status (RMOE_OK on success).  No C++
 *    exception crosses the ABI.  rmoe_last_error() returns the message of the
 *    last failure on the calling thread.
 *  - bf16 values are uint16_t bit patterns; fp32 values are float.
 *  - "Host" entry points take host pointers, borrow them for the call only,
 *    and are synchronous.  "_dev" entry points take device pointers and a
 *    hipStream_t passed as void* (NULL = the context's stream); they are
 *    asynchronous and never allocate, so they can be captured in a HIP graph.
 *  - Device memory (weights, scratch) is owned by the context.  A context is
 *    not thread-safe: calls that overlap on one context race on its scratch.
 *
 * Weight format at the boundary is the reference's q4nx pack_gemv layout
 * (quant/q4nx.py:335-393); per-expert bundles are the concatenations of
 * kernels/moe/pack.py:136-224 (expert e at offset e * expert_bytes; gate rows
 * then up rows in one [2I, H] matrix; down [H, Ipad]).  Uploads re-lay the
 * bytes on the device into the library's own tile layout.
 */
#ifndef RAON_MOE_H
#define RAON_MOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes; the Python mirror maps them to the reference's exception types. */
#define RMOE_OK 0
#define RMOE_EINVAL 1   /* ValueError: shape/dtype/contract violation (npu/backend.py:4864-4897) */
#define RMOE_ENOTFOUND 2 /* KeyError: unknown weight or layer (npu/backend.py:3609)               */
#define RMOE_EDEVICE 3  /* RuntimeError: HIP/device failure (npu/backend.py:1429-1437)            */
#define RMOE_ENOMEM 4   /* RuntimeError: device allocation failed                                 */

/* Activations (host/backend.py:47-62 SiTU-GLU; kernels/moe/reference.py:127-180 SwiGLU). */
#define RMOE_ACT_SITU 0
#define RMOE_ACT_SWIGLU 1
/* Activations of one value, for the products with an epilogue only (rmoe_linear_act_dev,
 * rmoe_experts_linear_dev): the value itself, z sigmoid(z), z times the normal distribution
 * function of z, and that with 0.5 (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) in its place. */
#define RMOE_ACT_NONE 2
#define RMOE_ACT_SILU 3
#define RMOE_ACT_GELU 4
#define RMOE_ACT_GELU_TANH 5

/* Router score functions (host/raon.py:1233-1234 sigmoid; softmax for BASELINE configs). */
#define RMOE_SCORE_SIGMOID 0
#define RMOE_SCORE_SOFTMAX 1

/* Weight formats of a dense matrix (BundleMeta.fmt, npu/backend.py:104-117). */
#define RMOE_FMT_Q4NX 0  /* "q4nx_gemv": 5 bits per weight (quant/q4nx.py:335-393)       */
#define RMOE_FMT_BFP16 1 /* "bfp16_gemv": bfp16ebs8, 9 bits per weight (quant/bfp16.py) */

/* Element types of token rows. */
#define RMOE_DT_BF16 0
#define RMOE_DT_F16 1
#define RMOE_DT_F32 2

/* Gates of a block's result in the norms around it: none, one value a column (fp32 [H]), one a row (fp32 [T]), or
 * one an element (rows' type, [T, H]). */
#define RMOE_GATE_NONE 0
#define RMOE_GATE_COLUMN 1
#define RMOE_GATE_ROW 2
#define RMOE_GATE_FULL 3

typedef struct rmoe_ctx rmoe_ctx;

/* Message of the last failed call on this thread ("" if none). */
const char* rmoe_last_error(void);

/* Library version string. */
const char* rmoe_version(void);

/* Context lifetime.  Replaces NpuBackend.__init__ device set-up (npu/backend.py:2404-2521)
 * and the XRT device/runner it opens. */
int rmoe_create(int device, rmoe_ctx** out);
int rmoe_destroy(rmoe_ctx* ctx);
/* Wait for all work queued on the device (the context's stream and the streams of _dev calls;
 * run.wait(), npu/backend.py:2236-2244), then report any error the kernels flagged since the
 * last synchronous call (e.g. device expert ids out of range, a decode-stack timeout). */
int rmoe_synchronize(rmoe_ctx* ctx);
/* The context's HIP stream, as void*. */
void* rmoe_stream(rmoe_ctx* ctx);

/* --------------------------------------------------------------- dense matrices --
 * Dense q4nx or bfp16 matrices ("bundles" of npu/backend.py:360-392, e.g. dense_gu) served by
 * rmoe_linear.  M % 128 == 0 and K % 256 == 0 (quant/q4nx.py:358-366).          */

/* Upload pack_gemv bytes of an [M, K] matrix; returns a handle.  Replaces the bundle
 * upload of NpuBackend.preload / _get_weight_tensor (npu/backend.py:3265). */
int rmoe_matrix_upload(rmoe_ctx* ctx, const void* pack_gemv_bytes, size_t nbytes, int M, int K, int* handle);
/* Allocate an [M, K] matrix and fill it by quantizing fp32 device weights w_dev [M, K]
 * row-major on the device (quant/q4nx.py:127-200, bit-exact).  Synchronous; with stream NULL
 * it first waits for whatever the device still runs, which may be writing the weights. */
int rmoe_matrix_quantize_dev(rmoe_ctx* ctx, const float* w_dev, int M, int K, int* handle, void* stream);
/* Read a matrix back as pack_gemv bytes (inverse re-layout; used for round trips). */
int rmoe_matrix_download(rmoe_ctx* ctx, int handle, void* pack_gemv_bytes, size_t nbytes);
int rmoe_matrix_free(rmoe_ctx* ctx, int handle);
int rmoe_matrix_shape(rmoe_ctx* ctx, int handle, int* M, int* K);

/* Upload the 9-bit bfp16ebs8 GEMV bytes of an [M, K] matrix (pack_bfp16_gemv with the
 * NPU's 4 core rows, quant/bfp16.py:216-329; M*K*9/8 bytes, M % 128 == 0, K % 256 == 0);
 * returns a handle served by rmoe_linear / rmoe_linear_dev / rmoe_matrix_download like a
 * q4nx matrix.  Replaces the "bfp16_gemv" bundle load (npu/backend.py:744-746) and the
 * GEMV_BFP16 operator's weight argument (kernels/gemv_bfp16/op.py:93-103); the GEMV
 * decodes m * 2^(max(e,7) - 133) exactly (kernels/gemv_bfp16/bfp16_gemv.cc:8-22). */
int rmoe_matrix_upload_bfp16(rmoe_ctx* ctx, const void* gemv_bytes, size_t nbytes, int M, int K, int* handle);
/* RMOE_FMT_* of a matrix (rmoe_matrix_download returns that format's bytes). */
int rmoe_matrix_format(rmoe_ctx* ctx, int handle, int* fmt);
/* Dense q4nx matrix [M, K] straight from a row-major llama.cpp Q4_K tensor (block_q4_K:
 * 144 bytes per 256 weights of a row; M*K/256*144 bytes; M % 128 == 0, K % 256 == 0),
 * converted on the device: every 4-bit code is kept and each 32-column group gets
 * scale = RTNE_bf16(d*sc), min = RTNE_bf16(-dmin*mn).  Replaces GGUFReader.q4nx_components
 * for a Q4_K tensor (quant/gguf_q4k.py:160-186, 228-233) followed by pack_gemv and the
 * bundle load; rmoe_matrix_download returns the equivalent pack_gemv bytes. */
int rmoe_matrix_upload_q4k(rmoe_ctx* ctx, const void* q4k_bytes, size_t nbytes, int M, int K, int* handle);

/* y[T, M] = RTNE_bf16(x[T, K] @ W^T), fp32 accumulation.  Replaces NpuBackend.linear /
 * _execute_gemv for a q4nx or bfp16 bundle (npu/backend.py:3569-3721, 3908-4021) and
 * Backend.linear_batch (host/backend.py:71-74).  K_in <= K: columns past K_in are zero
 * padding (comp.padded_k > comp.orig_k, npu/backend.py:3680-3684).  rmoe_linear gives a
 * token the same bytes alone and in a batch; rmoe_linear_dev does so except for T = 1 of a
 * q4nx matrix with M < 2048 and K = 512, 1024, 2048 or 4096, whose fp32 sums are added in
 * another order (a faster kernel), so that last bits may differ. */
int rmoe_linear(rmoe_ctx* ctx, int handle, const uint16_t* x, int T, int K_in, uint16_t* y);
int rmoe_linear_dev(rmoe_ctx* ctx, int handle, const void* x_dev, int T, void* y_dev, void* stream);
/* Size the scratch that rmoe_linear_dev needs for up to T tokens on this matrix. */
int rmoe_reserve_linear(rmoe_ctx* ctx, int handle, int T);

/* Dense product with an epilogue, on device operands:
 *   y = RTNE(act(x W^T + bias) + residual),
 * sums and epilogue in fp32, rounded once.  x bf16 [T, K_in], K_in <= K a multiple of 8, 16-byte
 * aligned; W's columns past K_in take no part, whatever they hold, nor do those past I of an
 * expert's down, which are padding (x's columns there count for nothing).  bias fp32 [M] or NULL;
 * residual bf16 of y's shape or NULL (y itself: added in place); y bf16 [T, M'].  act
 * RMOE_ACT_NONE, _SILU, _GELU, _GELU_TANH: M' = M; RMOE_ACT_SWIGLU, _SITU (gate_beta, value_beta,
 * 2^-100 to 2^100 in magnitude): M' = M / 2, row i of W the gate and row M/2 + i the up of output
 * i, bias added to both.
 * (rmoe_linear_dev followed by the activation rounds gate and up to bf16 first; this call does
 * not.)  Products of weights and values are exact; many rows are multiplied in fp16 with a power
 * of two per row of x and of W, where weights below 2^-27 of their row's largest (values of x:
 * 2^-30) keep fewer bits.  Sums of many rows are added in another order, so that a row's last
 * bits may depend on how many rows the call has (rmoe_linear_dev's do not).  Asynchronous on
 * `stream`, never allocates; products of many rows use context scratch, so that overlapping ones
 * need a context each.  The reference adds bias, activation and residual on the host
 * (host/raon.py:1314-1330). */
int rmoe_linear_act_dev(rmoe_ctx* ctx, int handle, const void* x_dev, int T, int K_in, const float* bias_dev, int act,
                        float gate_beta, float value_beta, const void* residual_dev, void* y_dev, void* stream);
/* Size the scratch that rmoe_linear_act_dev needs for up to T tokens on this matrix.  Graphs
 * captured before stay valid: scratch that was too small is kept until rmoe_destroy, and the next
 * has twice its size where that fits, else what was asked for.  Reserve for the largest call first. */
int rmoe_reserve_linear_act(rmoe_ctx* ctx, int handle, int T);

/* ------------------------------------------------------------ tokens by expert --
 * The steps around the experts' products on device operands, for an engine that puts work of
 * its own between them.  T tokens (at least one) of width H in RMOE_DT_* elements, any H from 1 to
 * 2^30, contiguous rows at any address of their type; k (1..16) routes per token, A = T k < 2^31
 * assignments a = t k + r.  Asynchronous on `stream`; nothing is allocated and no scratch of the
 * context is used, so that calls on several streams or captured graphs share only the buffers the
 * caller gives them.  Inputs and outputs of a call must not overlap. */

/* Sort: rows[inv[a]] = x[t] for every assignment whose expert ids[a] is in 0..n_experts-1
 * (n_experts <= 256), by expert and within an expert in ascending a; order[inv[a]] = a, and
 * expert e's rows are [offsets[e], offsets[e+1]) (offsets int32 [n_experts + 1]).  A negative
 * id is a route without an expert (padding, a dropped route, an expert of another GPU):
 * inv[a] = -1 and no row.  The same expert may appear twice in a token.  rows [A, H], order
 * [A] and inv [T, k] are written in full except rows and order from offsets[n_experts] on,
 * which stay as they were.  An id past the experts has no row either, and the next
 * synchronous call reports it.  The permutation is rmoe_dispatch's
 * (kernels/moe_grouped/planner.py:76-108), the gather its jobs' (:184-240). */
int rmoe_sort_tokens_dev(rmoe_ctx* ctx, const void* x_dev, int dtype, int T, int H, const void* ids_dev, int k,
                         int n_experts, void* rows_dev, void* order_dev, void* inv_dev, void* offsets_dev,
                         void* stream);
/* The sort's gradient: dx[t] = sum of drows[inv[t][r]] over the routes with a row (none: zeros),
 * fp32 in ascending sorted position, rounded once.  drows [A, H], dx [T, H]. */
int rmoe_sort_tokens_backward_dev(rmoe_ctx* ctx, const void* drows_dev, int dtype, int T, int H, const void* inv_dev,
                                  int k, void* dx_dev, void* stream);
/* Combine: out[t] = sum of weights[t][r] rows[inv[t][r]] over the routes with a row, fp32 in
 * ascending sorted position (= expert id, the order of rmoe_moe_experts_grouped), rounded
 * once.  rows [A, H], weights fp32 [T, k], out [T, H].  A route without a row takes no part,
 * whatever its weight. */
int rmoe_combine_tokens_dev(rmoe_ctx* ctx, const void* rows_dev, int dtype, int T, int H, const void* inv_dev,
                            const void* weights_dev, int k, void* out_dev, void* stream);
/* Combine's gradient: drows[inv[t][r]] = weights[t][r] dout[t] (rows no route names stay as
 * they were), dweights[t][r] = <dout[t], rows[inv[t][r]]> in fp32, 0 without a row.  inv as
 * rmoe_sort_tokens_dev writes it: no position twice. */
int rmoe_combine_tokens_backward_dev(rmoe_ctx* ctx, const void* dout_dev, const void* rows_dev, int dtype, int T, int H,
                                     const void* inv_dev, const void* weights_dev, int k, void* drows_dev,
                                     void* dweights_dev, void* stream);

/* --------------------------------------------------------------- MoE layers --
 * One MoE layer: n_routed experts + n_shared (0 or 1) shared expert, hidden H,
 * intermediate I (down input padded to Ipad = ceil(I/256)*256), router [n_routed, H].
 * H % 256 == 0, (2I) % 128 == 0, I % 64 == 0 (kernels/moe/pack.py:40-87). */
int rmoe_layer_create(rmoe_ctx* ctx, int layer, int hidden, int inter, int n_routed, int n_shared, int top_k);
/* Size the context scratch so that the "_dev" entry points of this layer accept up to
 * max_tokens tokens (they never allocate).  Replaces NpuBackend._prepared_buffer set-up. */
int rmoe_reserve(rmoe_ctx* ctx, int layer, int max_tokens);
/* Expert bundles in kernels/moe/pack.py geometry: (n_routed + n_shared) experts back to back.
 * gate_up: expert_bytes = 2I*H*5/8; down: H*Ipad*5/8.  Replaces moe_b1/moe_b2 uploads. */
int rmoe_layer_upload_experts(rmoe_ctx* ctx, int layer, const void* gate_up, size_t gu_nbytes,
                              const void* down, size_t dn_nbytes);
/* One part of expert `expert` from a row-major Q4_K tensor, converted on the device as in
 * rmoe_matrix_upload_q4k: part RMOE_PART_GATE (rows [0, I) of gate_up) and RMOE_PART_UP
 * (rows [I, 2I)) take [I, H]; RMOE_PART_DOWN takes [H, I] (I % 256 == 0; the columns up
 * to Ipad are the zero padding of kernels/moe/pack.py).  Replaces the per-expert
 * q4nx_components(name, outer_index=e) of quant/gguf_q4k.py:160-186 for the
 * ffn_{gate,up,down}_exps tensors feeding moe_b1/moe_b2. */
#define RMOE_PART_GATE 0
#define RMOE_PART_UP 1
#define RMOE_PART_DOWN 2
int rmoe_layer_upload_expert_q4k(rmoe_ctx* ctx, int layer, int expert, int part, const void* q4k_bytes,
                                 size_t nbytes);
/* A matrix handle that views one expert's weights in place (no copy, no upload):
 * part RMOE_PART_GATE_UP gives the expert's gate/up [2I, H] (q4nx; gate rows, then up
 * rows), RMOE_PART_DOWN its down [H, Ipad] (q4nx, or bfp16 in a weights-d layer; input
 * columns past I are the zero padding).  The handle is served by rmoe_linear /
 * rmoe_linear_dev / rmoe_matrix_download like an uploaded matrix; rmoe_matrix_free drops
 * the handle only, and freeing or re-creating the layer invalidates it.  Replaces the
 * component lookup that serves the shared expert's projections
 * model.layers.{L}.moe.shared_experts.{gate,up,down}_proj.weight by name
 * (npu/backend.py:360-392 specs, :3575-3609 lookup; called by RaonModel._moe_token,
 * host/raon.py:1314-1323, and the prefill shared precompute, :1570-1577) -- here from the
 * shared expert that a q4nx layer holds as expert n_routed (kernels/moe/pack.py:40-44),
 * or from moe_b2's last expert in a weights-d layer (npu/backend.py:4068-4107). */
#define RMOE_PART_GATE_UP 3
int rmoe_layer_expert_matrix(rmoe_ctx* ctx, int layer, int expert, int part, int* handle);
/* Quantize one expert from fp32 device weights (gate_up [2I, H], down [H, I] row-major;
 * the down input columns past I are zero-padded to Ipad).  Bit-exact quant/q4nx.py:127-200.
 * Synchronous; stream as in rmoe_matrix_quantize_dev. */
int rmoe_layer_quantize_expert_dev(rmoe_ctx* ctx, int layer, int expert, const float* gate_up_dev,
                                   const float* down_dev, void* stream);
/* Fill every expert of the layer with seeded synthetic weights N(0, std) generated on
 * the device (counter-based RNG, one stream per expert matrix) and quantized with the
 * same bit-exact q4nx quantizer.  For benchmarks at full depth; synchronous.  No
 * reference counterpart (the reference quantizes host arrays, quant/q4nx.py:127-200). */
int rmoe_layer_synthesize_dev(rmoe_ctx* ctx, int layer, uint64_t seed, float std, void* stream);
/* A MoE layer in the reference's weights-d layout (npu/backend.py:624-700), the format the
 * released model ships in:
 *   moe_b1  "q4nx_gemv_bundle": n_routed experts of [2I, H] (gate rows, then up rows),
 *           expert_bytes = 2I*H*5/8 (3,481,600 B for H=2560, I=1088);
 *   moe_b2  "bfp16_gemv_bundle": n_routed + 1 experts of [H, Ipad] bfp16ebs8, the last one
 *           the shared expert's down projection (component fmt "shared_down", expert_id
 *           128), expert_bytes = H*Ipad*9/8 (3,686,400 B).
 * The shared expert's gate/up (shared_gu, a dense "bfp16_gemv" matrix) stays outside the
 * layer, as in the reference: serve it with rmoe_matrix_upload_bfp16 + rmoe_linear.
 * Such a layer serves rmoe_route, rmoe_moe_experts (routed experts: q4nx gate/up, bfp16
 * down, ordered combine) and rmoe_moe_experts_grouped (routed sums + shared down from
 * shared_gu); the entry points that compute the shared gate/up inside the layer (decode,
 * decode stack, prefill_dev) reject it with RMOE_EINVAL. */
int rmoe_layer_create_d(rmoe_ctx* ctx, int layer, int hidden, int inter, int n_routed, int top_k);
/* Experts [expert0, expert0 + n) of one bundle of a weights-d layer: bytes are n
 * consecutive expert slices of moe_b1.bin (RMOE_BUNDLE_B1, offset expert*expert_bytes) or
 * moe_b2.bin (RMOE_BUNDLE_B2), as DWeights._read_expert_slice (npu/backend.py:1006-1034)
 * reads them; re-laid out on the device.  Lets a loader stream a bundle file in pieces. */
#define RMOE_BUNDLE_B1 1
#define RMOE_BUNDLE_B2 2
int rmoe_layer_upload_d(rmoe_ctx* ctx, int layer, int bundle, int expert0, int n, const void* bytes, size_t nbytes);
/* Read one expert back in its bundle's GEMV bytes (round trips, oracle cross-checks).
 * For a weights-d layer down is bfp16 (H*Ipad*9/8 bytes) and the shared expert
 * (expert n_routed) has no gate/up: pass gate_up = NULL, gu_nbytes = 0. */
int rmoe_layer_download_expert(rmoe_ctx* ctx, int layer, int expert, void* gate_up, size_t gu_nbytes,
                               void* down, size_t dn_nbytes);
/* Router of the layer (host/raon.py:1224-1247): weight bf16 [n_routed, H]; bias fp32
 * [n_routed] or NULL (selection-only e_score_correction_bias); score RMOE_SCORE_*;
 * renormalize 0/1; scaling = routed_scaling_factor.  Synchronous; the _dev form first waits
 * for whatever the device still runs, which may be writing the weights. */
int rmoe_layer_set_router(rmoe_ctx* ctx, int layer, const uint16_t* weight, const float* bias,
                          int score, int renormalize, float scaling);
int rmoe_layer_set_router_dev(rmoe_ctx* ctx, int layer, const void* weight_dev, const float* bias_host,
                              int score, int renormalize, float scaling);
int rmoe_layer_free(rmoe_ctx* ctx, int layer);

/* Router + top-k for T tokens (RaonModel._route_token, host/raon.py:1224-1247).
 * top_ids int32 [T, k], weights fp32 [T, k], logits fp32 [T, n_routed] (may be NULL).
 * Top-k ties keep the lower expert id first. */
int rmoe_route(rmoe_ctx* ctx, int layer, const uint16_t* x, int T, int32_t* top_ids, float* weights,
               float* logits);

/* Routed experts for one token: Backend.moe_experts (host/backend.py:98-117,466-510;
 * npu/backend.py:5029-5322).  Ascending-expert-id fp32 combine, RTNE.  act RMOE_ACT_*. */
int rmoe_moe_experts(rmoe_ctx* ctx, int layer, const uint16_t* x, const int32_t* top_ids,
                     const float* top_weights, int k, int act, float gate_beta, float value_beta,
                     uint16_t* out);
/* Device-pointer form of rmoe_moe_experts for any layer (q4nx or weights-d): x_dev bf16
 * [H], top_ids_dev int32 [k] (distinct, in 0..n_routed-1: not checked on the device beyond
 * clamping into range), top_weights_dev fp32 [k], out_dev bf16 [H].  Queued on `stream`
 * (NULL: the context stream); never allocates, so it can be captured in a HIP graph after
 * rmoe_reserve(layer, 1) with k <= top_k.  Replaces NpuBackend.moe_experts' direct decode
 * runner (npu/backend.py:5098-5229) for an engine that keeps activations on the device. */
int rmoe_moe_experts_dev(rmoe_ctx* ctx, int layer, const void* x_dev, const void* top_ids_dev,
                         const void* top_weights_dev, int k, int act, float gate_beta, float value_beta,
                         void* out_dev, void* stream);

/* rmoe_moe_experts_dev without context scratch: the same kernels and results, with their
 * working memory (the activations of the k slots, k x Ipad bf16) in a file-scope device
 * array of 256 KiB that each GPU holds until the process ends, its address looked up
 * once per device by rmoe_create.  It allocates nothing and needs no rmoe_reserve, for
 * callers that cannot allocate: code under HIP graph capture, tight serving loops,
 * harnesses that forbid allocation.  A layer and k whose scratch exceeds 256 KiB, or whose
 * k slots exceed the decode kernels' shape limits, is rejected with RMOE_EINVAL (the
 * BASELINE shape at k=8 needs 12 KiB, the reference model's at k=6 15 KiB).  All calls
 * on one GPU share the array: calls that overlap on
 * one GPU (any context, any stream) race.  No counterpart in the reference. */
int rmoe_moe_experts_static_dev(rmoe_ctx* ctx, int layer, const void* x_dev, const void* top_ids_dev,
                                const void* top_weights_dev, int k, int act, float gate_beta, float value_beta,
                                void* out_dev, void* stream);

/* Router + routed + shared expert + combine for one decode token, all on the device:
 * RaonModel._moe_token (host/raon.py:1288-1330) with the router moved onto the GPU.
 * out = RTNE(f32(routed) + f32(shared)); with residual != 0 also adds x:
 * out = RTNE(f32(x) + f32(out)).  top_ids/top_weights (device, may be NULL) receive
 * the routing of the token. */
int rmoe_moe_decode_dev(rmoe_ctx* ctx, int layer, const void* x_dev, void* out_dev, int residual,
                        int act, float gate_beta, float value_beta, void* top_ids_dev,
                        void* top_weights_dev, void* stream);
/* One stage of rmoe_moe_decode_dev: 0 = router (ids/weights into context scratch),
 * 1 = gate/up of all slots + activation, 2 = down of all slots + ordered combine into
 * out_dev.  Stages read the previous stage's context scratch; the split mirrors the
 * reference's moe_start("b1") / moe_start("b2") phases (npu/backend.py:5167-5284). */
int rmoe_moe_decode_stage_dev(rmoe_ctx* ctx, int layer, int stage, const void* x_dev, void* out_dev, int residual,
                              int act, float gate_beta, float value_beta, void* stream);
int rmoe_moe_decode(rmoe_ctx* ctx, int layer, const uint16_t* x, uint16_t* out, int residual,
                    int act, float gate_beta, float value_beta, int32_t* top_ids, float* top_weights);

/* One decode token through n_layers (1..64) MoE layers of one geometry in ONE persistent
 * launch: the per-layer loop of RaonModel.advance (host/raon.py:862-909) restricted to its
 * MoE sublayers, each layer as rmoe_moe_decode_dev with x_{l+1} = out_l (residual != 0:
 * x_{l+1} = RTNE(f32(x_l) + f32(out_l))).  layers is a host array of layer ids read during
 * the call.  top_ids/top_weights (device, may be NULL) receive [n_layers, k].  The kernel
 * keeps one workgroup per CU resident; its waits are bounded (a timeout is reported as
 * RMOE_EDEVICE by the next synchronous call).  Every layer must have a router and a
 * shared expert.  rmoe_reserve_decode_stack sizes the hand-off buffers (host call,
 * allocates); the _dev call never allocates.  The host form rmoe_moe_decode_stack (and
 * rmoe_moe_decode) first waits for all of this process's work on the device, so that no
 * kernel queued earlier on another stream holds CUs; with the _dev form that is the
 * caller's to ensure. */
int rmoe_reserve_decode_stack(rmoe_ctx* ctx, const int* layers, int n_layers);
/* Diagnostic, no counterpart in the reference: the number of polls (about a microsecond
 * each) after which a wait of the persistent decode kernel gives up (0 restores the default,
 * about two seconds).  A wait that gives up abandons the launch (every workgroup leaves),
 * and the next synchronous call returns RMOE_EDEVICE naming the first wait that gave up:
 * its workgroup, layer and hand-off (the layer's input, a down unit's h, or a combiner's d).
 * For callers that need a shorter bound, and for tests of the error report. */
int rmoe_set_stack_wait_limit(rmoe_ctx* ctx, unsigned polls);
int rmoe_moe_decode_stack_dev(rmoe_ctx* ctx, const int* layers, int n_layers, const void* x_dev, void* out_dev,
                              int residual, int act, float gate_beta, float value_beta, void* top_ids_dev,
                              void* top_weights_dev, void* stream);
int rmoe_moe_decode_stack(rmoe_ctx* ctx, const int* layers, int n_layers, const uint16_t* x, uint16_t* out,
                          int residual, int act, float gate_beta, float value_beta, int32_t* top_ids,
                          float* top_weights);

/* Dispatch permutation (kernels/moe_grouped/planner.py:76-108 flattened): top_ids int32
 * [T, k] -> order int32 [T*k] (assignment index t*k + r at each expert-sorted position;
 * ascending expert, then token, then route) and offsets int32 [n_experts + 1]. */
int rmoe_dispatch(rmoe_ctx* ctx, const int32_t* top_ids, int T, int k, int n_experts, int32_t* order,
                  int32_t* offsets);

/* rmoe_linear_act_dev over sorted rows, each row with the matrix of its expert: for e in
 * 0..n_routed-1 and offsets[e] <= p < offsets[e+1] (rmoe_sort_tokens_dev's offsets)
 *   y[p] = RTNE(act(rows[p] W_e^T + bias[e]) + residual[p]).
 * part RMOE_PART_GATE_UP: W_e [2I, H]; RMOE_PART_DOWN: W_e [H, I], rows of K_in = I columns or
 * more, up to Ipad: what they and the padded weights hold past I takes no part.  rows bf16 [n, K_in], 16-byte aligned, K_in a multiple of 8; bias
 * fp32 [n_routed, M] or NULL; residual and y bf16 [n, M'].  Rows from offsets[n_routed] on
 * stay as they were.  Both layer layouts (q4nx and weights-d) are served. */
int rmoe_experts_linear_dev(rmoe_ctx* ctx, int layer, int part, const void* rows_dev, int n, int K_in,
                            const void* offsets_dev, const float* bias_dev, int act, float gate_beta, float value_beta,
                            const void* residual_dev, void* y_dev, void* stream);
/* Size the scratch that rmoe_experts_linear_dev needs for up to n rows on this layer (the same
 * scratch as rmoe_reserve_linear_act's). */
int rmoe_reserve_experts_linear(rmoe_ctx* ctx, int layer, int n);

/* Grouped prefill MoE: NpuBackend.moe_experts_grouped (npu/backend.py:4845-4979).
 * x [T, H], top_ids [T, k] (distinct per token, 0..n_routed-1), top_weights fp32 [T, k],
 * shared_gu [T, 2I] -> routed [T, H] and shared_down [T, H]. */
int rmoe_moe_experts_grouped(rmoe_ctx* ctx, int layer, const uint16_t* x, int T, const int32_t* top_ids,
                             const float* top_weights, const uint16_t* shared_gu, int act, float gate_beta,
                             float value_beta, uint16_t* routed, uint16_t* shared_down);

/* rmoe_moe_experts_grouped on device-resident operands (the same contract,
 * npu/backend.py:4845-4979): x_dev bf16 [T, H], top_ids_dev int32 [T, k], top_weights_dev
 * fp32 [T, k], shared_gu_dev bf16 [T, 2I] -> routed_dev and shared_down_dev bf16 [T, H], on
 * `stream` (null: the context's stream), asynchronously.  T must not exceed the tokens
 * reserved with rmoe_reserve; an expert id out of range is reported by the next
 * synchronous call. */
int rmoe_moe_experts_grouped_dev(rmoe_ctx* ctx, int layer, const void* x_dev, int T, const void* top_ids_dev,
                                 const void* top_weights_dev, const void* shared_gu_dev, int act, float gate_beta,
                                 float value_beta, void* routed_dev, void* shared_down_dev, void* stream);

/* Full prefill MoE layer on the device (host/raon.py:1565-1602 grouped branch): router,
 * dispatch, grouped gate/up + activation, grouped down, ordered combine, shared expert.
 * out [T, H] = RTNE(f32(routed) + f32(shared_down)) (+ x when residual != 0). */
int rmoe_moe_prefill_dev(rmoe_ctx* ctx, int layer, const void* x_dev, int T, void* out_dev, int residual,
                         int act, float gate_beta, float value_beta, void* top_ids_dev,
                         void* top_weights_dev, void* stream);

/* ------------------------------------------------------ microscaled 4-bit rows --
 * A third weight format and the one quantized form of activations: blocks of 32 columns that share a power of two 2^s,
 * s = clamp(floor(log2 max|x|) - 2, -127, 127) (zeros: -127), held as the byte s + 127, and per column a 4-bit code, bit
 * 3 its sign and bits 0..2 an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6: the nearest to x 2^-s, ties to the even index,
 * magnitudes above 6 to 6.  (The published microscaling format with e2m1 elements and e8m0 scales.)  A block that
 * holds NaN or an infinity has byte 255 and codes 0 and stands for NaN.  A row of K columns has P = K rounded up to 32 of
 * them, zeros past K: P/2 bytes of codes, the even column in a byte's low half, and P/32 scale bytes.  Codes and scales
 * are plain row-major arrays of the caller, weights [M, K] and activations [T, K] alike: weights are quantized by the
 * same call, and nothing is uploaded or laid out again.  All calls are asynchronous on `stream`, allocate nothing and
 * use no scratch of the context: calls on several streams and captured graphs share only the buffers the caller gives
 * them.  At least one row. */

/* x [T, K] in RMOE_DT_* elements, contiguous, at any address of their type, K from 1 to 2^30 -> codes [T, P/2] (16-byte
 * aligned), scales [T, P/32], and values [T, K] in x's type, what they stand for (exact; NULL: not written; x itself: in
 * place).  For a forward pass that trains: compute with the values, and pass their gradient on to x unchanged. */
int rmoe_mx_quantize_dev(rmoe_ctx* ctx, const void* x_dev, int dtype, int T, int K, void* codes_dev, void* scales_dev,
                         void* values_dev, void* stream);
/* y[T, M'] = RTNE(act(x W^T + bias) + residual) of quantized rows x [T, K] and weights [M, K], K a multiple of 32 (of
 * another width: quantized rows end in zeros, so both sides' P is the K here): products exact, sums and epilogue fp32,
 * rounded once to bf16.  act, bias, residual and M' as in rmoe_linear_act_dev; any M (even when gated).  A scale byte
 * of 255 in a row of x or W makes its results NaN.  Codes 16-byte aligned; scales at any address (at one that is not a
 * multiple of 16 calls of many rows and of a K that is a multiple of 512 take the kernel of other K, which is slower).
 * Sums may be added in another order for another number of rows or such scales, so that a row's last bits may depend on
 * them.  T x M below 2^28 always fits a launch; larger calls whose tiles would take 2^32 threads are refused. */
int rmoe_mx_linear_dev(rmoe_ctx* ctx, const void* x_codes_dev, const void* x_scales_dev, int T, int K,
                       const void* w_codes_dev, const void* w_scales_dev, int M, const float* bias_dev, int act,
                       float gate_beta, float value_beta, const void* residual_dev, void* y_dev, void* stream);
/* The same over sorted rows, each with the matrix of its expert: for e in 0..n_experts-1 (at most 256) and offsets[e] <=
 * p < offsets[e+1] (rmoe_sort_tokens_dev's offsets) W_e of codes [n_experts, M, K/2] and scales [n_experts, M, K/32], bias
 * [n_experts, M] or NULL.  Rows from offsets[n_experts] on stay as they were. */
int rmoe_mx_experts_linear_dev(rmoe_ctx* ctx, const void* x_codes_dev, const void* x_scales_dev, int n, int K,
                               const void* w_codes_dev, const void* w_scales_dev, int M, const void* offsets_dev,
                               int n_experts, const float* bias_dev, int act, float gate_beta, float value_beta,
                               const void* residual_dev, void* y_dev, void* stream);

/* ------------------------------------------------------- norms around a block --
 * What stands between two blocks (attention, a dense MLP or the experts) of a residual stream:
 *   n = (mean_j b_j^2 + eps)^-1/2,  u = n b wpost  (post NULL: u = b)
 *   y = R(scale r + g u)
 *   m = (mean_j y_j^2 + eps)^-1/2,  h = R(m y wpre)
 * block b, residual r, y and h [T, H] in RMOE_DT_* elements at any address of their type, H from 1 to 8192; sums and
 * products fp32 (rows whose sum of squares passes its range give zeros), R one rounding to the rows' type; h is the
 * norm of y as stored.  wpost and wpre fp32 [H]; gate g as gate_kind (RMOE_GATE_*) says, NULL for none.  block
 * NULL: no y, post or gate, and h is the norm of residual (the norm before the first block).  h NULL: not wanted;
 * codes [T, P/2] (16-byte aligned) and scales [T, P/32], both or neither: h as microscaled 4-bit rows, the bytes that
 * rmoe_mx_quantize_dev makes of it.  eps > 0.  Asynchronous, allocates nothing, no scratch.  y may be residual or block,
 * h may be block, nothing else may overlap.  The reference normalises on the host (host/raon.py:904-909). */
int rmoe_residual_norm_dev(rmoe_ctx* ctx, const void* block_dev, const void* residual_dev, int dtype, int T, int H,
                           const float* post_weight_dev, const void* gate_dev, int gate_kind, float scale,
                           const float* pre_weight_dev, float eps, void* y_dev, void* h_dev, void* codes_dev,
                           void* scales_dev, void* stream);
/* Floats of work memory that rmoe_residual_norm_backward_dev takes for T rows of width H. */
int rmoe_norm_backward_work(int T, int H, size_t* floats);
/* Its gradients from dy (of y where the stream goes on; NULL: none) and dh (of h; NULL: none), at least one of them:
 *   a = dh wpre,  D = dy + m a - y m^3 (sum_j a_j y_j) / H,  dresidual = scale D,  du = g D,  v = du wpost,
 *   dblock = n v - b n^3 (sum_j v_j b_j) / H  (post NULL: du),
 *   dpre_weight = sum_t dh y m,  dpost_weight = sum_t du b n,  dgate = D u summed over what a gate's value is shared by.
 * block, y (as computed), gate, scale and eps as in the forward call; block NULL: the gradient of the norm of y alone,
 * with scale 1 for the plain sum dy + norm's.  dpre_weight, dpost_weight fp32 [H], dgate as the gate; NULL: not wanted.
 * dresidual may be dy, dblock may be dh.  work: fp32, rmoe_norm_backward_work, of the call alone while it runs.  Column
 * sums are added in a fixed order. */
int rmoe_residual_norm_backward_dev(rmoe_ctx* ctx, const void* dy_dev, const void* dh_dev, const void* block_dev,
                                    const void* y_dev, int dtype, int T, int H, const float* post_weight_dev,
                                    const void* gate_dev, int gate_kind, float scale, const float* pre_weight_dev,
                                    float eps, void* dblock_dev, void* dresidual_dev, float* dpost_weight_dev,
                                    void* dgate_dev, float* dpre_weight_dev, float* work_dev, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RAON_MOE_H */
