/*
 * hm_moe.h -- C ABI of the MI355X (gfx950) MoE-block engine.
 *
 * This is the boundary between the C++20 host layer (HipBackend,
 * HipTensorBackend, HipMoEBlock) and the hand-written HIP kernels in
 * libhm_kernels.so.  It replaces, for the device-resident MoE block, what the
 * reference reaches through its C++ virtual interfaces and its CUDA kernel
 * free functions (SHOnnay/hypermoe-engine):
 *
 *   ComputeBackend            src/backend/Backend.hpp:36-71
 *   TensorBackend             src/tensor/backend/TensorBackend.hpp:11-39
 *   MoERuntime::executeBatch  src/core/runtime/MoERuntime.hpp:57-60
 *   CUDA kernels              src/backend/cuda/CudaKernels.hpp:10-46
 *
 * Conventions
 *   - Every pointer argument is a DEVICE pointer unless its comment says
 *     host.  The caller owns all memory; nothing here allocates device memory
 *     except hm_device_alloc/hm_host_alloc.
 *   - `stream` is a hipStream_t passed as void* (NULL = default stream).
 *     Launchers are asynchronous on that stream and never synchronise.
 *   - Every function returns an hm_status.  HM_ERR_INVALID, HM_ERR_OVERFLOW
 *     and HM_ERR_RUNTIME map to the reference's std::invalid_argument,
 *     std::overflow_error and std::runtime_error.  A HIP failure returns
 *     HM_ERR_RUNTIME and hm_last_hip_error() gives the hipError_t.
 *   - Conditions only the device can see (a non-finite router score, a
 *     softmax/renormalisation failure) are reported through the device
 *     status word `status` (int32, HM_STATUS_* bits), which the caller reads
 *     back; the reference throws std::runtime_error for them
 *     (src/router/CpuRouterBackend.cpp:47,57-59,83-85).  A token whose
 *     softmax or renormalisation failed gets placeholder ids 0..top_k-1 with
 *     zero scores, so that the launches queued after it stay in range.
 *   - No function throws.
 */
#ifndef HM_MOE_H
#define HM_MOE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HM_ABI_VERSION 1

typedef enum hm_status {
    HM_OK = 0,
    HM_ERR_INVALID = 1,   /* std::invalid_argument */
    HM_ERR_OVERFLOW = 2,  /* std::overflow_error   */
    HM_ERR_RUNTIME = 3,   /* std::runtime_error (HIP or launch failure) */
    HM_ERR_UNSUPPORTED = 4
} hm_status;

/* Device status word bits (written by kernels, read by the host). */
#define HM_STATUS_NONFINITE_SCORE 1u   /* CpuRouterBackend.cpp:47        */
#define HM_STATUS_SOFTMAX_FAILED 2u    /* CpuRouterBackend.cpp:57-59     */
#define HM_STATUS_RENORM_FAILED 4u     /* CpuRouterBackend.cpp:83-85     */

/* Routing flags, RouterConfig (src/router/RouterConfig.hpp:22-29). */
#define HM_ROUTE_SOFTMAX 1u  /* RoutingNormalization::Softmax, else None */
#define HM_ROUTE_RENORM 2u   /* renormalizeSelected                       */
/* Execution flag for hm_moe_block_forward: run the INT8 expert GEMMs on the
 * scalar reference kernels instead of MFMA (identical integers and float
 * operation sequence; used to pin the MFMA kernels). */
#define HM_EXEC_GENERIC 0x100u
/* Execution flag for hm_moe_block_forward: INT8 experts always take the
 * integer-limb GEMMs.  Without it a block of at most HM_GEMV_MAX_TOKENS
 * tokens and HM_GEMV_MAX_PAIRS (token, expert) pairs (decode) takes the
 * W8A32 GEMV kernels instead, which stream each selected expert's weights
 * once and compute in FP32 (within 1e-4 of the reference, not bit-identical
 * to the limb arithmetic); larger blocks, decode ones included, take the
 * limb GEMMs. */
#define HM_EXEC_LIMBS 0x200u
#define HM_GEMV_MAX_TOKENS 16
#define HM_GEMV_MAX_PAIRS 64
/* Execution flag for hm_router_topk / hm_moe_block_forward: every router
 * logit of a decode batch (up to 16 tokens) is computed with the reference's
 * sequential FP64 chain instead of certifying the parallel sums (the results
 * are identical; the flag exercises the fallback).  Larger batches run the
 * chains with and without it. */
#define HM_EXEC_ROUTE_SEQUENTIAL 0x400u
/* Execution flag for hm_moe_block_forward: INT8 prefill experts with at most
 * 32 grouped rows take the bounded split-K GEMM (K split over a workgroup's
 * waves, exact integer partials; the same bits as without it) instead of
 * the tile GEMMs' partial tiles.  Off by default: on this GPU it is slower
 * at every batch size measured (the tiles stream the same weights faster). */
#define HM_EXEC_SPLIT_K 0x800u

/* Element types (src/tensor/DType.hpp:9-14 numbering; FP8 has no counterpart
 * there).  Expert weights are FP32, INT8 or FP8. */
#define HM_DTYPE_FP32 0
#define HM_DTYPE_FP16 1
#define HM_DTYPE_BF16 2
#define HM_DTYPE_INT8 3
#define HM_DTYPE_FP8 4 /* e4m3 bytes with a float scale per block (F1) */

int hm_abi_version(void);
const char* hm_status_string(int status);
/* Last hipError_t seen by a launcher on this host thread (0 = none). */
int hm_last_hip_error(void);

/* ---- Device runtime (ComputeBackend surface, src/backend/Backend.hpp:36-71) */
int hm_device_count(int* count_out /* host */);
int hm_set_device(int ordinal);
int hm_device_alloc(void** ptr_out /* host */, size_t bytes);
int hm_device_free(void* ptr);
int hm_host_alloc(void** ptr_out /* host */, size_t bytes); /* pinned */
int hm_host_free(void* ptr);
int hm_memcpy_h2d(void* dst, const void* src_host, size_t bytes, void* stream);
int hm_memcpy_d2h(void* dst_host, const void* src, size_t bytes, void* stream);
int hm_memcpy_d2d(void* dst, const void* src, size_t bytes, void* stream);
int hm_stream_create(void** stream_out /* host */);
int hm_stream_destroy(void* stream);
int hm_stream_synchronize(void* stream);
int hm_event_create(void** event_out /* host */);
int hm_event_destroy(void* event);
int hm_event_record(void* event, void* stream);
int hm_event_synchronize(void* event);
int hm_stream_wait_event(void* stream, void* event);
int hm_event_elapsed_ms(float* ms_out /* host */, void* start, void* stop);
int hm_mem_info(size_t* free_out /* host */, size_t* total_out /* host */);

/* ---- A1  RMSNorm (src/transformer/norm/RMSNorm.cpp:65-77) ----------------
 * y[r,i] = float(double(x[r,i]) * inv_r * double(gamma[i])),
 * inv_r = 1/sqrt(sum_i double(x)^2 / width + double(eps)), the sum taken in
 * ascending i exactly as the reference's sequential loop.  Bit-exact. */
int hm_rmsnorm(const float* x, const float* gamma, float* y, int64_t rows,
               int64_t width, float eps, void* stream);

/* ---- A2  Router (src/router/CpuRouterBackend.cpp:35-91) -----------------
 * logits[t,e] = float(sum_k double(h[t,k]) * double(w[k,e])), k ascending;
 * softmax with glibc-expf-exact float exp and double denominator; top-k by
 * (score desc, expert id asc); optional renormalisation by the double sum of
 * the selected scores in rank order.  ids/scores are [tokens x top_k] in
 * rank order.  Bit-exact.  The logits go to logits_out, or, when it is NULL,
 * to `route_ws` (hm_route_workspace_bytes(tokens, hidden, experts) bytes, 16-byte
 * aligned).  Batches of more than 16 tokens run the reference's chain of
 * every logit on the FP64 matrix cores; with route_ws given, smaller ones
 * (hidden % 32 == 0) take FP64 block sums whose partials live in route_ws, and
 * a logit whose float their error bound does not settle is recomputed by the
 * sequential chain.  (For larger batches the size counts more than the logits
 * they use.)  `flags`: HM_ROUTE_* bits, optionally HM_EXEC_ROUTE_SEQUENTIAL. */
size_t hm_route_workspace_bytes(int64_t tokens, int64_t hidden, int64_t experts);
int hm_router_topk(const float* h, const float* w, int64_t tokens,
                   int64_t hidden, int64_t experts, int32_t top_k,
                   uint32_t flags, uint32_t* ids, float* scores,
                   float* logits_out, int32_t* status, void* route_ws,
                   void* stream);

/* ---- A3  Token permute (src/router/CpuRouterBackend.cpp:140-159) ---------
 * Stable counting sort of the tokens*top_k (token, rank) pairs by expert id:
 * counts[E], offsets[E+1], perm_tokens/perm_weights[tokens*top_k] in group
 * order (groups by ascending expert id, tokens ascending inside a group),
 * slots[tokens*top_k]: the grouped row of pair (t, r).  Bit-exact.  No
 * global atomics: per-chunk LDS histograms, then each chunk ranks its pairs.
 * `workspace`: hm_permute_workspace_bytes(...) bytes (may be NULL when that
 * is 0, i.e. tokens*top_k <= 1024). */
size_t hm_permute_workspace_bytes(int64_t tokens, int32_t top_k, int64_t experts);
int hm_permute(const uint32_t* ids, const float* scores, int64_t tokens,
               int32_t top_k, int64_t experts, int32_t* counts,
               int32_t* offsets, int32_t* perm_tokens, float* perm_weights,
               int32_t* slots, void* workspace, void* stream);

/* ---- A4  Gather rows (src/core/runtime/MoERuntime.cpp:282-299) ----------
 * out[r,:] = in[rows[r],:]. */
int hm_gather_rows(const float* in, const int32_t* rows, int64_t count,
                   int64_t width, float* out, void* stream);

/* ---- A5/A5' op level (TensorBackend::matmulInt8Weights / matmul,
 * src/tensor/backend/CpuTensorBackend.cpp:87-190).  x [M x K] FP32,
 * q / w [K x N] row-major INPUT_OUTPUT, y [M x N].
 * hm_matmul_w8a32, mode 1 (reference): the reference's loop,
 * acc += x * (float(q - zp) * scale) in FP32, bit-exact.  Mode 2
 * (cooperative): the terms x (q - zp) exactly, summed in FP32 in another,
 * fixed order, times the scale: within (K + 32) 2^-24 sum_k |x w| of the exact
 * sum, as the loop is within K 2^-24 of that, so the two differ by up to both
 * (on the reference's own test inputs by less than 1e-5 + 1e-5|ref|).  Non-finite
 * activations and weights past the float range give what the loop gives.
 * The plan (hm_plan_int8_gemm) is the reference's: its partition and block
 * counts and the scratch it asks of the caller are part of the interface,
 * though the cooperative kernel splits K inside a workgroup and leaves the
 * scratch untouched. */
typedef struct hm_int8_gemm_plan {
    int32_t implementation; /* 1 = Reference (one lane per output),
                               2 = Cooperative (split-K partitions) */
    int64_t partitions;     /* bounded split-K: min(8, ceil(K/512)) */
    int64_t blocks;         /* workgroups of the reference's launch */
    int64_t scratch_elements; /* FP32 scratch the call asks for, M*N*P if P > 1 */
} hm_int8_gemm_plan;
/* Launch plan, src/backend/cuda/Int8GemmPlan.cpp:29-53 (mode: 0 auto,
 * 1 reference, 2 cooperative). */
int hm_plan_int8_gemm(int64_t rows, int64_t inner, int64_t cols, int32_t mode,
                      hm_int8_gemm_plan* plan_out /* host */);
int hm_matmul_w8a32(const float* x, const int8_t* q, float scale, int32_t zp,
                    float* y, int64_t rows, int64_t inner, int64_t cols,
                    int32_t mode, float* scratch, size_t scratch_bytes,
                    void* stream);
int hm_matmul_f32(const float* x, const float* w, float* y, int64_t rows,
                  int64_t inner, int64_t cols, void* stream);

/* ---- A6  elementwise (Activation.cpp:44, CpuTensorBackend.cpp:192-220) */
int hm_silu(const float* x, float* y, int64_t n, void* stream);
int hm_mul(const float* a, const float* b, float* y, int64_t n, void* stream);
int hm_add(const float* a, const float* b, float* y, int64_t n, void* stream);

/* ---- A7  Combine (src/core/runtime/MoERuntime.cpp:308-325) --------------
 * out[t,:] = sum over the token's pairs in ascending expert id of
 * w * y_grouped[slot,:], float multiply then float add, starting from 0.
 * Bit-exact given y_grouped.  If residual != NULL, out = residual + sum
 * (TransformerBlock.cpp:101-104), the add done last. */
int hm_combine(const float* y_grouped, const uint32_t* ids,
               const int32_t* slots, const float* scores, int64_t tokens,
               int32_t top_k, int64_t width, const float* residual,
               float* out, void* stream);

/* ---- A8  INT8 packer (src/tensor/quantization/Quantization.cpp:45-79) on
 * the host: scale = max|w|/127 (1 if all zero), zp = 0,
 * q = int8(clamp(round(w/scale), -127, 127)).  Host pointers. */
int hm_quantize_int8_host(const float* w /* host */, int64_t n,
                          int8_t* q /* host */, float* scale /* host */,
                          int32_t* zero_point /* host */,
                          float* max_abs_error /* host, may be NULL */);

/* ---- A10  Device-resident expert table --------------------------------
 * The reference payload for expert e is gate [H x I] | up [H x I] |
 * down [I x H], row-major INPUT_OUTPUT (ExpertPacker.cpp:228-230,
 * WeightConverter.cpp:31-42).  hm_pack_layer re-lays it out once on the
 * device into the kernels' layout: each projection transposed to [N x K]
 * (K contiguous), experts back to back.  The packed table holds
 * 3*E*H*I elements of the same dtype. */
typedef struct hm_layer {
    int64_t experts, hidden, intermediate;
    int32_t dtype;              /* HM_DTYPE_INT8, HM_DTYPE_FP32 or HM_DTYPE_FP8 */
    const void* packed;         /* output of hm_pack_layer; FP8: see F2 */
    const float* scale;         /* INT8: [E x 3] {gate, up, down}; FP8: block scales (F2) */
    const int32_t* zero_point;  /* [E x 3], INT8 only */
} hm_layer;
size_t hm_packed_layer_bytes(int64_t experts, int64_t hidden,
                             int64_t intermediate, int32_t dtype);
int hm_pack_layer(const void* reference_payload, int64_t experts,
                  int64_t hidden, int64_t intermediate, int32_t dtype,
                  void* packed, void* stream);

/* ---- A5 block level + A11: the fused MoE block ------------------------
 * MoERuntime::executeBatch (src/core/runtime/MoERuntime.cpp:58-349) with all
 * experts device resident: route -> permute -> grouped SwiGLU experts ->
 * combine.  hidden [T x H] (post-RMSNorm), router_w [H x E].
 *
 * INT8 experts use the integer-limb arithmetic: activations are written as
 * per-row (gate/up) or per-128-column (down) fixed point split into
 * `limbs_x` / `limbs_z` balanced signed INT8 digits; every int32 partial is
 * exact; the FP32 result is within 1e-4 of the reference W8A32 path for
 * limbs >= 2 and bit-exact against the build's CPU restatement.
 * FP32 experts use FP32 arithmetic (within 1e-3 of the reference).
 * FP8 experts run as hm_fp8_experts does from FP32 rows to FP32 rows (F2);
 * the limb arguments and the HM_EXEC_* bits of INT8 experts do not apply.
 *
 * Outputs (device, caller-owned; all but `out` may be NULL, in which case
 * the workspace copy is used):
 *   out [T x H]; ids, scores [T x k]; counts [E]; offsets [E+1];
 *   perm_tokens, perm_weights [T*k]; expert_out [T*k x H] (grouped order,
 *   the per-group expert outputs of BatchLayerExecutionResult);
 *   status: HM_STATUS_* bits (must be zeroed by the caller once; kernels
 *   only OR bits in).
 * The workspace must hold hm_moe_block_workspace_bytes(...) bytes. */
typedef struct hm_block_io {
    float* out;
    uint32_t* ids;
    float* scores;
    int32_t* counts;
    int32_t* offsets;
    int32_t* perm_tokens;
    float* perm_weights;
    float* expert_out;
    int32_t* status;
    const float* residual; /* optional: out = residual + MoE(hidden) */
    /* Optional profiling spans (the role of the reference's GpuEventQueue,
     * src/profiling/GpuEventQueue.hpp:17-69): HM_BLOCK_EVENTS hipEvent_t
     * handles recorded on `stream` at the stage boundaries
     * [start, routed, permuted, quantised, gate/up done, down done,
     * combined].  Events 3 and 4 bracket the gate/up kernels themselves:
     * they are taken at the first kernel's start and the last kernel's end
     * (hipExtLaunchKernelGGL), so their span is the stage's kernel time.
     * NULL = no recording. */
    void* const* events;
} hm_block_io;
#define HM_BLOCK_EVENTS 7
/* exec_flags: the HM_EXEC_* bits the calls will pass (the generic path needs
 * an extra [T*k x I] float buffer). */
size_t hm_moe_block_workspace_bytes(const hm_layer* layer, int64_t tokens,
                                    int32_t top_k, int32_t limbs_x,
                                    int32_t limbs_z, uint32_t exec_flags);
int hm_moe_block_forward(const hm_layer* layer, const float* hidden,
                         const float* router_w, int64_t tokens, int32_t top_k,
                         uint32_t route_flags, int32_t limbs_x,
                         int32_t limbs_z, const hm_block_io* io,
                         void* workspace, size_t workspace_bytes,
                         void* stream);

/* One MoE sub-layer of the transformer block
 * (src/transformer/runtime/TransformerBlock.cpp:88-104: RMSNorm.cpp:65-77
 * on the layer input, the MoE block on the normalised rows, the input added
 * back): io->out = h + MoE(RMSNorm(h; gamma, eps)).  normed [tokens x
 * hidden] receives RMSNorm(h) (hm_rmsnorm's values); it must not overlap h.
 * io->residual must be NULL or h.  Decode batches normalise inside the
 * router's first kernel (one launch fewer than hm_rmsnorm followed by
 * hm_moe_block_forward); other batches launch hm_rmsnorm first.  Same
 * workspace as hm_moe_block_forward. */
int hm_moe_layer_forward(const hm_layer* layer, const float* h,
                         const float* gamma, float eps, float* normed,
                         const float* router_w, int64_t tokens, int32_t top_k,
                         uint32_t route_flags, int32_t limbs_x,
                         int32_t limbs_z, const hm_block_io* io,
                         void* workspace, size_t workspace_bytes,
                         void* stream);

/* ---- The block without allocation ------------------------------------
 * No counterpart in the reference.  For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): hm_moe_block_forward with its workspace in a
 * library-owned device array of HM_NOALLOC_WORKSPACE_BYTES per GPU (held
 * from first use until the process ends).  Same arguments and results as
 * hm_moe_block_forward without the workspace; the caller still passes the
 * inputs and the outputs in `io`.  Returns HM_ERR_UNSUPPORTED, without
 * launching anything, when the call needs a larger workspace
 * (hm_moe_block_workspace_bytes > HM_NOALLOC_WORKSPACE_BYTES: decode
 * batches always fit, prefill batches up to a few hundred tokens at the
 * Qwen3-30B-A3B shape).  It allocates nothing and calls no allocating
 * routine.  All calls on one GPU share the array: calls that overlap on a
 * GPU (other streams, other host threads) race and must be serialised by
 * the caller. */
#define HM_NOALLOC_WORKSPACE_BYTES ((size_t)64 << 20)
int hm_moe_block_forward_noalloc(const hm_layer* layer, const float* hidden,
                                 const float* router_w, int64_t tokens,
                                 int32_t top_k, uint32_t route_flags,
                                 int32_t limbs_x, int32_t limbs_z,
                                 const hm_block_io* io, void* stream);

/* ---- Limb arithmetic at op level (build-owned, no reference counterpart):
 * quantise rows to digit planes and return exact int32 partials, so tests
 * can pin "INT8 int32 partials bit-exact" directly.
 * digits: [limbs x rows x inner] int8; scales [rows];
 * partials: [limbs x rows x cols] int32 of sum_k d * (q[k,c] - zp) with q in
 * the packed [cols x inner] (transposed) layout. */
int hm_limb_quantize_rows(const float* x, int64_t rows, int64_t inner,
                          int32_t limbs, int8_t* digits, float* scales,
                          void* stream);
int hm_limb_partials(const int8_t* digits, int64_t rows, int64_t inner,
                     int32_t limbs, const int8_t* q_packed, int32_t zp,
                     int64_t cols, int32_t* partials, void* stream);

/* ---- F1  Block-scaled FP8 (no counterpart in the reference) -------------
 * A matrix [rows x width] in FP8 is rows of hm_fp8_pitch(width) bytes (width
 * rounded up to 128): e4m3 (OCP, largest 448), zeros past the width, 16-byte
 * aligned.  Each block of block_rows rows (1: activations, 128: weights) x
 * 128 columns has a float scale, scale[ceil(rows / block_rows) x
 * ceil(width / 128)]; a byte stands for its e4m3 value times that scale.
 * Checkpoints in this format whose inner dimension is a multiple of 128 are
 * read as they are.
 *
 * hm_fp8_quantize: x (FP32, FP16 or BF16; element (r, k) at x[r row_stride +
 * k col_stride], one of the strides 1) to that form.  With amax = max(|x|,
 * 2^-100) over a block, scale = amax / 448 and each byte is the e4m3 value
 * nearest to 448 x / amax, ties to even (decided exactly for 16-bit x).  A
 * block that holds an infinity or a NaN becomes NaN throughout.  q and scale
 * must not overlap x.  The blocks of a transposed matrix are the transposed
 * blocks, so quantising the transposed view of a weight gives the operand of
 * its input's gradient.
 *
 * hm_fp8_matmul: y[m, n] = sum_b xs[m, b] ws[n / w_block_rows, b]
 * sum_{k in block b} x[m, k] w[n, k], x [rows x inner] with a scale per row
 * and block, w [cols x inner] with w_block_rows 128 or 1, y [rows x cols] in
 * y_dtype (FP32, FP16, BF16).  A layer's product: x W^T.  Its input's
 * gradient: dY times the quantised transposed view of W.  Its weight's
 * gradient: the transposed views of dY and x, both with a scale per row
 * (w_block_rows 1).  y must not overlap the operands.
 * Sums: the sizes and y_dtype fix their order, so a call repeats its bits, but
 * a row's may differ with the number of rows beside it.  FP32 results are FP32
 * sums of the exact products (1.1e-7 of the result's norm over 4096 columns).
 * FP16 and BF16 results of many rows take the FP8 matrix instruction, which
 * aligns eight consecutive products to the largest and drops what lies more
 * than 13 bits below it: at most 2^-10 of sum |x w|; 1.5e-5 of the result's
 * norm for normally distributed operands, 5.1e-5 for bytes spread evenly over
 * the format (FP16's own rounding: 2.1e-4).  A caller that needs the FP32 sums
 * asks for FP32 results, at half the rate.
 * Scales: xs ws is one FP32 product.  Where it passes the largest float (the
 * blocks' maxima multiply to over 6.8e43) the outputs that it enters are
 * infinite or NaN, also where the block's sum is small enough for a finite
 * one; below 2^-126 it has the bits of a subnormal.
 *
 * HM_ERR_OVERFLOW: to quantise rows of contiguous columns with block_rows 1,
 * over 2^42 blocks, 2^40 rows or 2^31 columns; otherwise over 65535 x 128 rows
 * or 2^29 - 128 columns.  To multiply, over 2^31 - 1 rows or inner columns or
 * 67 million columns (rows of w). */
int64_t hm_fp8_pitch(int64_t width);
int hm_fp8_quantize(const void* x, int32_t dtype, int64_t rows, int64_t width,
                    int64_t row_stride, int64_t col_stride, int32_t block_rows,
                    uint8_t* q, float* scale, void* stream);
int hm_fp8_matmul(const uint8_t* xq, const float* xs, const uint8_t* wq,
                  const float* ws, int32_t w_block_rows, int64_t rows,
                  int64_t inner, int64_t cols, void* y, int32_t y_dtype,
                  void* stream);

/* ---- F2  FP8 experts ---------------------------------------------------
 * The SwiGLU experts of a routed batch (ExpertExecutor.cpp:43-138 over the
 * groups of MoERuntime.cpp:282-306) with the weights of an FP8 layer:
 * grouped row g of expert e, offsets[e] <= g < offsets[e + 1], is
 *   y[g] = z D_e^T,  z = silu(x[perm_tokens[g]] G_e^T) * (x[..] U_e^T),
 * x and z each quantised to a scale per row and 128 columns before their
 * product: x as by hm_fp8_quantize, z from FP32 values, scale and quotients
 * within two units in the last place of hm_fp8_quantize's.  y's sums are those
 * of F1.  z's are FP32 sums of the exact products, except for BF16 y and at
 * least 128 pairs an expert: there gate and up take the FP8 instruction, and a
 * byte of z next to a border may move by a step (an error of 2.0e-3 of y's
 * norm in all, where FP32 sums leave 1.7e-3, BF16's own rounding; FP32 or FP16
 * y avoids it).  layer->packed holds, expert after expert, gate [I x pitch(H)],
 * up [I x pitch(H)] and down [H x pitch(I)] bytes, layer->scale [E x 3 x
 * ceil(H / 128) ceil(I / 128)] their block scales, each projection's in its
 * own [ceil(N / 128) x ceil(K / 128)] order; zero_point is unused.  x
 * [tokens x H], y [pairs x H]; offsets [E + 1] and perm_tokens [pairs] as
 * hm_permute gives them (a token outside 0 .. tokens - 1 reads token 0).
 * Rows of y from offsets[E] on are left as they were.  At most 1024 experts.
 * The workspace holds hm_fp8_experts_workspace_bytes(...) bytes; calls that
 * overlap in time need one each. */
size_t hm_fp8_experts_workspace_bytes(const hm_layer* layer, int64_t tokens,
                                      int64_t pairs);
/* An FP8 layer from a payload in the reference's layout (gate [H x I] | up
 * [H x I] | down [I x H] per expert, as for hm_pack_layer; FP32, FP16 or
 * BF16, on the device): `packed` (hm_packed_layer_bytes(..., HM_DTYPE_FP8)
 * bytes, 16-byte aligned) and `scale` as above. */
int hm_fp8_pack_layer(const void* payload, int32_t dtype, int64_t experts,
                      int64_t hidden, int64_t intermediate, void* packed,
                      float* scale, void* stream);
int hm_fp8_experts(const hm_layer* layer, const void* x, int32_t x_dtype,
                   int64_t tokens, const int32_t* offsets,
                   const int32_t* perm_tokens, int64_t pairs, void* y,
                   int32_t y_dtype, void* workspace, size_t workspace_bytes,
                   void* stream);

/* ---- F3  Token rows to the experts and back, and the gradients -----------
 * hm_gather_rows and hm_combine for FP32, FP16 and BF16 rows (`dtype`), with
 * weights either way, pairs that no expert took, and backward passes.
 * slots [tokens x top_k] is hm_permute's: the grouped row of a token's r-th
 * expert, below `rows`, each row named once.  A slot outside 0 .. rows - 1
 * marks a pair that was dropped (a full expert, an expert on another GPU):
 * it is written nowhere, adds nothing and its weight's gradient is 0.
 * Grouped rows that no slot names are left as they were.  weights and their
 * gradients are FP32 [tokens x top_k]; sums are FP32, ranks ascending, and
 * rounded once.
 *   hm_dispatch_rows       out[slots[t,r]] = w[t,r] x[t] (weights NULL: x[t])
 *   hm_dispatch_rows_grad  dx[t] = sum_r w[t,r] dout[slots[t,r]],
 *                          dweights[t,r] = <dout[slots[t,r]], x[t]>
 *   hm_combine_rows        out[t] = sum_r w[t,r] y[slots[t,r]], plus
 *                          residual[t] last (weights NULL: 1; residual NULL:
 *                          none; out may be residual)
 *   hm_combine_rows_grad   dy[slots[t,r]] = w[t,r] dout[t],
 *                          dweights[t,r] = <dout[t], y[slots[t,r]]>
 * (the residual's gradient is dout).  dweights may be NULL, then x and y may
 * be too; asking for it needs the weights.  Outputs must not overlap inputs
 * otherwise. */
int hm_dispatch_rows(const void* x, const int32_t* slots, const float* weights,
                     int64_t tokens, int32_t top_k, int64_t rows, int64_t width,
                     int32_t dtype, void* out, void* stream);
int hm_dispatch_rows_grad(const void* dout, const void* x, const int32_t* slots,
                          const float* weights, int64_t tokens, int32_t top_k,
                          int64_t rows, int64_t width, int32_t dtype, void* dx,
                          float* dweights, void* stream);
int hm_combine_rows(const void* y, const int32_t* slots, const float* weights,
                    const void* residual, int64_t tokens, int32_t top_k,
                    int64_t rows, int64_t width, int32_t dtype, void* out,
                    void* stream);
int hm_combine_rows_grad(const void* dout, const void* y, const int32_t* slots,
                         const float* weights, int64_t tokens, int32_t top_k,
                         int64_t rows, int64_t width, int32_t dtype, void* dy,
                         float* dweights, void* stream);

/* ---- F4  Experts held in 16 bits, and their training ---------------------
 * Grouped products: rows in expert order (hm_dispatch_rows; offsets [groups +
 * 1] as hm_permute gives them), each group times its own matrix.  Operands
 * FP16 or BF16 (`dtype`), sums FP32, rounded once to the result's type: dtype,
 * or FP32 where a result type is asked for.  Matrices are row-major, one after
 * another: w [groups x cols x inner].  Rows before offsets[0] and from
 * offsets[groups] on are read by nothing and their results left as they were;
 * a group may have no rows.  Offsets ascend; what they name past `rows` is left
 * out.  At most 1024 groups, 2^31 - 1 rows, 2^26 columns and 2^40 values a
 * matrix.  Outputs must not overlap inputs.
 *   hm_grouped_matmul       y[g] = x[g] w_e^T, x [rows x inner], y [rows x
 *                           cols].  w_transposed: w [groups x inner x cols],
 *                           y[g] = x[g] w_e, which is the input's gradient of
 *                           the product by the same matrices
 *   hm_grouped_swiglu       the gate and up products and z[g] = silu(gate) up,
 *                           from FP32 sums: w [groups x 2 intermediate x
 *                           hidden], gate rows first; z [rows x intermediate].
 *                           perm_tokens [rows]: row g reads x[perm_tokens[g]],
 *                           x [x_rows x hidden] (outside it: row 0); NULL: x's
 *                           own rows.  pre [rows x 2 intermediate] receives
 *                           gate | up for the backward pass; may be NULL
 *   hm_grouped_swiglu_grad  dz[g] = dy[g] w_e (w the down matrices [groups x
 *                           hidden x intermediate]) kept in FP32, and from it
 *                           and pre, with s = 1 / (1 + e^-gate): dpre = dz up
 *                           s (1 + gate (1 - s)) | dz gate s, and z = gate s up
 *                           again for the down matrices' gradient (NULL: not)
 *   hm_grouped_weight_grad  dw[e] = sum over the group's rows of dy[g]^T x[g]
 *                           [cols x inner], zeros for a group without rows;
 *                           accumulate: added to what dw holds (in FP32, then
 *                           rounded once).  The workspace holds
 *                           hm_grouped_weight_grad_workspace_bytes(...) bytes
 *                           (may be 0); calls that overlap in time need one
 *                           each.
 * A sum's order is fixed by the sizes and offsets: no atomics, the same bits
 * every run. */
#define HM_GROUPED_MAX_GROUPS 1024
int hm_grouped_matmul(const void* x, int32_t dtype, const void* w,
                      int32_t w_transposed, const int32_t* offsets,
                      int64_t groups, int64_t rows, int64_t inner, int64_t cols,
                      void* y, int32_t y_dtype, void* stream);
int hm_grouped_swiglu(const void* x, int32_t dtype, int64_t x_rows,
                      const int32_t* perm_tokens, const void* w,
                      const int32_t* offsets, int64_t groups, int64_t rows,
                      int64_t hidden, int64_t intermediate, void* z, void* pre,
                      void* stream);
int hm_grouped_swiglu_grad(const void* dy, int32_t dtype, const void* w,
                           const void* pre, const int32_t* offsets,
                           int64_t groups, int64_t rows, int64_t hidden,
                           int64_t intermediate, void* dpre, void* z,
                           void* stream);
size_t hm_grouped_weight_grad_workspace_bytes(int64_t groups, int64_t rows,
                                              int64_t cols, int64_t inner);
int hm_grouped_weight_grad(const void* dy, const void* x, int32_t dtype,
                           const int32_t* offsets, int64_t groups, int64_t rows,
                           int64_t cols, int64_t inner, void* dw,
                           int32_t dw_dtype, int32_t accumulate,
                           void* workspace, size_t workspace_bytes,
                           void* stream);

/* ---- F5  Low-rank adapters beside a shared projection --------------------
 * A projection that all rows share, W, and for each row its own adapter a =
 * ids[row] (outside 0 .. adapters - 1: none), in any order:
 *   mid[t] = scale[a] x[t] A_a^T,   y[t] = x[t] W^T + mid[t] B_a^T
 * x [rows x inner], W [cols x inner], down = A [adapters x rank x inner], up =
 * B [adapters x cols x rank], FP16 or BF16 (`dtype`), scale [adapters] FP32.
 * mid [rows x rank] (zeros for a row without adapter) and y [rows x cols] have
 * that type; sums are FP32, mid is rounded once before its product.  Adapters
 * of smaller rank are padded with zeros.
 * w_transposed: W [inner x cols], down [adapters x inner x rank], up [adapters
 * x rank x cols], y = x W + mid up_a.  That is the input's gradient: pass dy,
 * the same W, B as `down` and A as `up`; mid is then the gradient of mid, with
 * the scale.
 * hm_adapter_weight_grad: dw[a] = sum over the rows t with ids[t] = a of
 * left[t]^T right[t], [left_cols x right_cols]: A's gradient of the gradient of
 * mid and x, B's of dy and mid.  Zeros for an adapter without rows; accumulate,
 * dw_dtype and workspace as F4's (at most 1 GB); every adapter goes through
 * the ids of all rows, so its time grows with adapters times rows.  mid and y
 * must not overlap anything.  Rank up to 256, up to 65535 adapters and 2^23 - 1
 * rows.
 * Rows of one adapter side by side are fastest.  An infinity or a NaN in an
 * adapter's matrices reaches the rows of that adapter only: others have the
 * bits that they have without it, at up to some 25 times the call's time. */
#define HM_ADAPTER_MAX_RANK 256
int hm_adapter_matmul(const void* x, int32_t dtype, const void* w,
                      int32_t w_transposed, const void* down, const void* up,
                      const float* scale, const int32_t* ids, int64_t adapters,
                      int64_t rank, int64_t rows, int64_t inner, int64_t cols,
                      void* mid, void* y, void* stream);
size_t hm_adapter_weight_grad_workspace_bytes(int64_t adapters, int64_t rows,
                                              int64_t left_cols,
                                              int64_t right_cols);
int hm_adapter_weight_grad(const void* left, const void* right, int32_t dtype,
                           const int32_t* ids, int64_t adapters, int64_t rows,
                           int64_t left_cols, int64_t right_cols, void* dw,
                           int32_t dw_dtype, int32_t accumulate,
                           void* workspace, size_t workspace_bytes,
                           void* stream);

/* ---- Test hooks --------------------------------------------------------
 * The device restatement of glibc expf used by the router softmax and SiLU,
 * evaluated elementwise (parity of the libm boundary). */
int hm_debug_expf(const float* x, float* y, int64_t n, void* stream);
/* Which kernel an FP8 call of these sizes takes, so that a test of one is a
 * test of that one.  Products: rows of x << 16 | rows of w of a tile, 0 the
 * kernel that streams w.  Experts: 16 the kernels for few rows, 0 streamed
 * weights, else the rows of a tile (<< 16 where gate and up use the exact
 * products).  -1: not a call. */
int hm_debug_fp8_matmul_form(int64_t rows, int64_t inner, int64_t cols,
                             int32_t y_dtype);
int hm_debug_fp8_experts_form(const hm_layer* layer, int64_t tokens,
                              int64_t pairs, int32_t y_dtype);

/* The same for F4 and F5.  kind 0, 1: hm_grouped_matmul, w_transposed; 2:
 * hm_grouped_swiglu (its own rows); 3: hm_grouped_swiglu_grad (inner: hidden,
 * cols: intermediate); 4: hm_grouped_weight_grad; 5, 6: hm_adapter_matmul,
 * w_transposed (groups 1).  m << 16: the kernel that streams w for 16 m rows
 * at a time; 256, 128, 64: tiles of 256 x 256, 128 x 256 and 128 x
 * 128; 32: tiles of 128 x 128 for operands off 16 bytes; 0: the generic kernel.
 * -1: not a call. */
int hm_debug_grouped_form(int32_t kind, int64_t groups, int64_t rows,
                          int64_t inner, int64_t cols, int32_t rank,
                          int32_t aligned16);

#ifdef __cplusplus
}
#endif
#endif /* HM_MOE_H */
