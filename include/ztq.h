/*
 * ztq.h -- C ABI of libztq_sm100a.so: B200 (sm_100a) weight-quantized GEMV kernels
 * behind ztensor's kernel-library calling convention.
 *
 * Conventions (the ones ztensor's zero-CGo binding layer relies on,
 * internal/cuda/purego.go:237 `Ccall(fn, args ...uintptr)`):
 *   - every argument is an integer-class machine word (pointers, int, cudaStream_t);
 *   - the return value is a cudaError_t, 0 = success;
 *   - all pointers are DEVICE pointers owned by the caller; a launcher allocates
 *     nothing, keeps nothing, never synchronises and never reads device memory,
 *     so it can be recorded into a CUDA graph;
 *   - launches are asynchronous on `stream` (NULL = legacy default stream);
 *   - argument errors are reported as cudaErrorInvalidValue before any launch.
 *     There is no CPU fallback: the caller decides what to do with an error.
 *
 * Packed-weight layouts on the device ("residency layouts"):
 *   Q4_0     separated, exactly Q4Storage.RawBytesGPU (tensor/quantized.go:158-187):
 *            [fp16 scale x nBlocks][pad to 16 B][16 data bytes x nBlocks]
 *   IQ4_NL   the same separated layout (built from the 18-byte blocks by
 *            ztq_repack_blocks18)
 *   Q8_0     Q8Storage.RawBytes (tensor/quantized.go:427-438): 36-byte blocks
 *            {f32 scale, 32 x int8}, unchanged
 *   W4G      GPTQ 4-bit / AWQ, one layout for both (their packed bytes are
 *            identical): [data: K/2 bytes per row] + [half2 {scale, zero} per group]
 *   ternary  TernaryStorage bytes with every row starting on a byte
 *            (ceil(K/4) bytes per row; identical to RawBytes when K % 4 == 0),
 *            the layout internal/cuda/kernels/ternary_gemv.cu:21-29 expects
 */
#ifndef ZTQ_H
#define ZTQ_H

#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* flags for the ztq_gemv_* entry points */
#define ZTQ_X_F32   1   /* activations are float32 (default: fp16)            */
#define ZTQ_Y_F32   2   /* outputs are float32 (default: fp16, round-nearest)  */
#define ZTQ_X_KB    4   /* activations laid out [K, batch] (default [batch,K]) */
#define ZTQ_Y_NB    8   /* outputs laid out [N, batch] (default [batch, N])    */
#define ZTQ_NO_PDL 16   /* launch without the programmatic-dependent-launch attribute.  With it (the default) a kernel
                           starts fetching the packed WEIGHTS before it waits for the preceding kernel of the stream;
                           activations, workspaces and outputs are ordered after that kernel.  Kernels of this
                           library that write weight layouts never release their dependents early, so sequences of
                           ztq calls are safe; a caller whose own kernel writes weights and triggers its dependents
                           early (griddepcontrol.launch_dependents) directly in front of a ztq launch passes this flag. */
#define ZTQ_PLAIN  32   /* force the plain (non-streaming) kernel              */
#define ZTQ_ROPE_PAIRS 128 /* rotary positions turn interleaved pairs (2i, 2i+1) instead of halves (i, i + rot_dim/2) */
#define ZTQ_FP32_DECODE 64 /* decode codes to fp32 in registers instead of the exact integer block dot */

/* ---- drop-in replacements: same names, arguments and meaning as the
 * ---- reference's launchers ------------------------------------------------ */

/* Replaces internal/cuda/kernels/gemm_q4.h:29-33 (gemm_q4.cu:163-201).
 * C[M,N] = dequant(A_q4[M,K]) * B[K,N]; A in the separated layout, data region
 * at byte `data_offset`; B, C float32 row-major.  K % 32 must be 0. */
cudaError_t gemm_q4_f32(const void* A_q4, const float* B, float* C, int M, int K, int N, int data_offset,
                        cudaStream_t stream);

/* Replaces internal/cuda/kernels/gemm_q8.h (gemm_q8.cu:156-182): A is M*K/32
 * 36-byte Q8_0 blocks. */
cudaError_t gemm_q8_f32(const void* A_q8, const float* B, float* C, int M, int K, int N, cudaStream_t stream);

/* Replaces internal/cuda/kernels/ternary_gemv.h:33-37 (ternary_gemv.cu:85-99):
 * y[m] = sum_k decode(W[m,k]) * x[k], W row-aligned 2-bit codes, x, y float32. */
cudaError_t ternary_gemv_f32(const void* W_ternary, const float* x, float* y, int M, int K, cudaStream_t stream);

/* ---- fp16-activation entry points (the W4A16 path and its siblings).
 * y[b, n] = sum_k dequant(W[n, k]) * x[b, k], 1 <= batch.  These are what
 * GPUEngine.MatMul's B-weight branches (compute/gpu_engine.go:2127-2204 for Q4,
 * :2617-2686 for Q8) and a GPUEngine.MatMulW4A16 (the optional interface of
 * compute/w4a16.go:139-143) bind instead of transposing around gemm_q4_f32. */
cudaError_t ztq_gemv_q4_0(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch,
                          int flags, cudaStream_t stream);
cudaError_t ztq_gemv_iq4nl(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch,
                           int flags, cudaStream_t stream);
cudaError_t ztq_gemv_q8_0(const void* w_blocks36, const void* x, void* y, int N, int K, int batch, int flags,
                          cudaStream_t stream);
/* GPTQ 4-bit / AWQ: qdata = N*K/2 bytes, meta = half2 {scale, zero} per group,
 * groups of `group` consecutive k inside a row (a power of two >= 32 dividing K;
 * 128 is the tuned case). */
cudaError_t ztq_gemv_w4g(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                         int batch, int flags, cudaStream_t stream);
/* Three or more activation rows (any batch >= 1 is accepted): the same product as ztq_gemv_w4g, group 128, fp16
 * activations [batch, K], outputs [batch, N], computed as a skinny GEMM on the tcgen05 tensor cores with TMEM
 * accumulators (weights as the M operand, batch padded to 8, 16 or 32 as the N operand, 32 activation vectors per
 * pass over the weights).  Default operands: the 4-bit codes and the activations as three int8 digit planes of a
 * 21-bit block fixed point (exact integer group sums); ZTQ_FP32_DECODE: fp16 operands, nothing rounded.
 * This is the batched form of the W4A16 entry a GPUEngine.MatMulW4A16 (compute/w4a16.go:139-143) binds when
 * m >= 3; the reference has no tensor-core path for quantized weights (its batch path is the naive 16x16 tile
 * kernel of gemm_q4.cu:119-159).  `workspace` (>= ztq_gemm_w4g_tc_workspace_bytes(N, K, batch), 256-byte aligned,
 * caller-owned, overwritten) receives the activations rearranged into tensor-core tiles by a small first kernel.
 * K % 512 == 0.  Flags: ZTQ_Y_F32, ZTQ_NO_PDL, ZTQ_FP32_DECODE. */
size_t ztq_gemm_w4g_tc_workspace_bytes(int N, int K, int batch);
cudaError_t ztq_gemm_w4g_tc(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group, int batch,
                            void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream);
/* The same for Q4_0 weights (a scale per block of 32, zero point 8): the batched form of ztq_gemv_q4_0, which the
 * B-weight branch of GPUEngine.MatMul binds from three activation rows on, where the reference transposes, runs its
 * 16x16 tile kernel and transposes back (compute/gpu_engine.go:2166-2203, gemm_q4.cu:119-159).  Each of a group's
 * four tensor-core steps (32 k = one block) keeps an accumulator of its own and the epilogue applies the block
 * scales; 16 activation vectors per pass over the weights.  w_sep / data_offset as for ztq_gemv_q4_0
 * (data_offset > 0), fp16 activations [batch, K], outputs [batch, N]; K % 512 == 0.  Flags: ZTQ_Y_F32, ZTQ_NO_PDL. */
size_t ztq_gemm_q4_0_tc_workspace_bytes(int N, int K, int batch);
cudaError_t ztq_gemm_q4_0_tc(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch, void* workspace,
                             size_t workspace_bytes, int flags, cudaStream_t stream);

/* Q8_0 with 3 or more activation rows, on the storage's own bytes (Q8Storage.RawBytes: 36-byte blocks {float32 scale,
 * 32 int8}, 16-byte aligned base): the same tensor-core kernel with the int8 codes as the signed operand, the scales
 * taken from the blocks as they stream through shared memory, activations as 18-bit block fixed point (a block's 32
 * products with codes up to +-127 stay inside int32).  K % 512 == 0, fp16 activations [batch, K], y [batch, N] fp16
 * (or fp32 with ZTQ_Y_F32); replaces the tile kernel of gemm_q8.cu:113-152 for batches. */
size_t ztq_gemm_q8_0_tc_workspace_bytes(int N, int K, int batch);
cudaError_t ztq_gemm_q8_0_tc(const void* blocks36, const void* x, void* y, int N, int K, int batch, void* workspace,
                             size_t workspace_bytes, int flags, cudaStream_t stream);
/* Ternary with an optional fp16 scale per output row (row_scale may be NULL). */
cudaError_t ztq_gemv_ternary(const void* w_rows, const void* row_scale, const void* x, void* y, int N, int K,
                             int batch, int flags, cudaStream_t stream);

/* ---- split-K for narrow outputs (few rows, long K), batch 1.  The K axis is cut into `splits`
 * (2..64) equal slices handled by separate groups of CTAs; each writes fp32 partial sums of all N rows
 * to `workspace` (>= ztq_splitk_workspace_bytes(N, splits), 16-byte aligned, caller-owned, contents
 * overwritten), and a second kernel adds the slices in slice order: deterministic, no atomics.
 * Completes the "split-K with a deterministic second-pass reduction" the reference's kernels lack
 * (gemm_q4.cu:163-191 launches ceil(M/16) blocks whatever K is).  K/splits must be a multiple of
 * 256 (Q4_0) or of 4*group (W4G).  Activations are one contiguous vector [K], outputs [N].
 * Flags: ZTQ_X_F32, ZTQ_Y_F32, ZTQ_NO_PDL, ZTQ_FP32_DECODE; any other flag (the layout flags ZTQ_X_KB /
 * ZTQ_Y_NB, ZTQ_PLAIN) returns cudaErrorInvalidValue. */
size_t ztq_splitk_workspace_bytes(int N, int splits);
cudaError_t ztq_gemv_w4g_splitk(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                                int splits, void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream);
cudaError_t ztq_gemv_q4_0_splitk(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int splits,
                                 void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream);

/* Split-K GEMV for callers that must not allocate.  No counterpart in the reference.
 *
 * Who needs it: an engine that hands out every device buffer from an arena it sized at start-up and
 * treats a cudaMalloc after that point as a bug, or a caller that is already recording a CUDA graph,
 * where allocating is not allowed.  Such a caller has nowhere to get the split-K workspace from, so
 * this variant brings its own: the fp32 partial sums go into a fixed array inside the library
 * (ZTQ_STATIC_SCRATCH_BYTES, resident on every GPU that loads the library until the process ends).
 * The call allocates nothing and frees nothing; inputs and the output are still the caller's.
 *
 * Limits and rules:
 *   - N * splits * 4 bytes must not exceed ZTQ_STATIC_SCRATCH_BYTES, otherwise cudaErrorInvalidValue
 *     is returned and nothing is launched (use ztq_gemv_w4g_splitk with your own workspace instead);
 *   - the first call on each device looks up the array's device address (the device must be
 *     current); make that first call before starting any stream capture on that device.  A first
 *     call made on a capturing stream returns cudaErrorStreamCaptureUnsupported and leaves no trace:
 *     a later call outside capture does the set-up;
 *   - all calls share the one array and it keeps whatever the last call left in it.  Nothing in it
 *     has to start at zero: every call overwrites the N * splits partial sums it later reads.  Two
 *     calls whose kernels can overlap on the GPU (different streams, no dependency) race on the array:
 *     keep calls to this entry point ordered on one stream or otherwise serialised.
 * Arguments and results are those of ztq_gemv_w4g_splitk. */
#define ZTQ_STATIC_SCRATCH_BYTES (1 << 20)
cudaError_t ztq_gemv_w4g_splitk_static(const void* qdata, const void* meta, const void* x, void* y, int N, int K,
                                       int group, int splits, int flags, cudaStream_t stream);

/* ---- tensor-parallel row shards: GEMV with the all-reduce of its outputs fused in.
 * No counterpart in the reference (its all-reduce, internal/nccl/nccl_purego.go:267-285,
 * has no caller); this is the shard path of a row-parallel
 * projection.  Every rank (one process per GPU) calls the same sequence of
 * *_allreduce launchers with the same shapes.  The kernel pushes every fp32
 * partial output as an 8-byte {value, tag} cell into every rank's slot buffer
 * with one plain peer store (no multicast, no fences), then waits a bounded time
 * until its own rank's cells of that row carry the tag of this launch and adds
 * them in rank order, so y is the full sum and is bit-identical on all ranks.
 * If a peer never arrives the kernel gives up, sets the device error word
 * (ztq_device_error() == 4) and returns; the context stays usable.
 * The all-reduce exists in the integer-arithmetic kernels only: ZTQ_FP32_DECODE and ZTQ_PLAIN are refused
 * (cudaErrorInvalidValue) by the *_allreduce entry points. */
typedef struct ZtqAllReduce {
    int world, rank;      /* 2..8 ranks */
    int slot_stride;      /* cells per (parity, rank) slot: >= batch * N of the largest reduced output */
    int reserved;
    void* slots[8];       /* slots[r]: rank r's slot buffer as mapped in THIS process:
                             2 * world * slot_stride cells of 8 bytes, zero-initialised */
    void* state;          /* this rank's {launch sequence, finished CTAs}: 2 unsigned, zero-initialised */
} ZtqAllReduce;

cudaError_t ztq_gemv_w4g_allreduce(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                                   int batch, int flags, const ZtqAllReduce* ar, cudaStream_t stream);
/* The same for 3 or more activation rows: ztq_gemm_w4g_tc with the all-reduce in its epilogue.  The warp that holds
 * a row tile's final sums pushes them as cells and goes on with its next tile; the peers' cells are collected after
 * the CTA's last tile.  Integer operands only (ZTQ_FP32_DECODE is refused); passes of 16 activation rows, each one
 * launch of the sequence every rank counts; slot_stride >= min(batch, 16) * N.  GEMV and tensor-core launchers of
 * one ZtqAllReduce may alternate freely as long as every rank issues the same sequence. */
cudaError_t ztq_gemm_w4g_tc_allreduce(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group,
                                      int batch, void* workspace, size_t workspace_bytes, int flags, const ZtqAllReduce* ar,
                                      cudaStream_t stream);
cudaError_t ztq_gemv_q4_0_allreduce(const void* w_sep, int data_offset, const void* x, void* y, int N, int K, int batch,
                                    int flags, const ZtqAllReduce* ar, cudaStream_t stream);

/* ---- Q4_K (tensor/quantized_kquant.go: super-blocks of 256 weights in 144 bytes) --------------------
 * y[b, n] = sum_k dequant(W[n, k]) * x[b, k], the product xblas.GemmF32Q4KNT / GemmQ4KF32 compute on the CPU engine
 * (internal/xblas/gemm_q4k.go:15-140) and gemv_q4k_f32 on the reference's GPU path (compute/gpu_engine.go:2209-2330).
 * w_sep is the separated device layout made by ztq_repack_blocks144: the 16 header bytes {fp16 d, fp16 dmin, 12
 * bytes of 6-bit scales and mins} of every super-block, then at data_offset = 16 * nblocks the 128 nibble bytes of
 * every super-block.  K % 256 == 0 and K >= 2048; batch <= 8 (one pass over the weights per row).
 * Flags: ZTQ_X_F32, ZTQ_Y_F32, ZTQ_NO_PDL. */
cudaError_t ztq_gemv_q4k(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch, int flags,
                         cudaStream_t stream);
/* RawBytes() of a Q4KStorage (144-byte super-blocks, 16-byte aligned) -> the separated layout above. */
cudaError_t ztq_repack_blocks144(const void* aos, void* sep, long long nblocks, cudaStream_t stream);
/* Q5_K (tensor/quantized_kquant.go:489-621; CPU product xblas.GemmF32Q5KNT, internal/xblas/gemm_quant.go:273-360;
 * the reference's GPU path is gemv_q5k_f32): as Q4_K with a fifth bit per weight.  Separated layout made by
 * ztq_repack_blocks176: per super-block 48 side bytes {16 header bytes, the 32 qh bytes}, then at data_offset =
 * 48 * nblocks the 128 low-nibble bytes of every super-block.  Same limits and flags as ztq_gemv_q4k. */
cudaError_t ztq_gemv_q5k(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch, int flags,
                         cudaStream_t stream);
cudaError_t ztq_repack_blocks176(const void* aos, void* sep, long long nblocks, cudaStream_t stream);
/* Q6_K (tensor/quantized_kquant.go:335-483; CPU product xblas.GemmF32Q6KNT, internal/xblas/gemm_quant.go:384-470;
 * the reference's GPU path is gemv_q6k_f32): 6-bit codes, one int8 scale per 16 weights, one fp16 d per 256.
 * Separated layout made by ztq_repack_blocks210 (the 210-byte source blocks need no alignment): per super-block 96
 * side bytes {64 bytes qh, 16 scales, fp16 d, 14 zero bytes}, then at data_offset = 96 * nblocks the 128 ql bytes
 * of every super-block.  Same limits and flags as ztq_gemv_q4k. */
cudaError_t ztq_gemv_q6k(const void* w_sep, long long data_offset, const void* x, void* y, int N, int K, int batch, int flags,
                         cudaStream_t stream);
cudaError_t ztq_repack_blocks210(const void* aos, void* sep, long long nblocks, cudaStream_t stream);

/* ---- the steps either side of a projection, folded into the GEMV (batch 1) ---------------------
 * The reference runs RMSNorm and SwiGLU as kernels of their own around MatMul
 * (internal/cuda/kernels/fused_add_rmsnorm.cu:13-50, fused_swiglu.cu:10-21).  Here, for W4A16 weights (group
 * 128, K >= 2048, K % 256 == 0):
 *   norm_weight != NULL:  the GEMV reads  v = x + residual  (residual may be NULL), normalises it on the way
 *                         in, activation[k] = v[k] * rsqrt(mean(v^2) + eps) * norm_weight[k], and writes v to
 *                         sum_out when that is not NULL (sum_out must not alias x or residual: other CTAs
 *                         still read them).  x, residual, sum_out share x's element type (fp16, or fp32 with
 *                         ZTQ_X_F32); norm_weight is float32, 16-byte aligned; eps travels as its bit pattern.
 *   swiglu != 0:          rows of the matrix are (gate_i, up_i) pairs (ztq_interleave_rows lays them out so);
 *                         y has N / 2 entries, y[i] = gate_i * sigmoid(gate_i) * up_i.
 * Flags: ZTQ_X_F32, ZTQ_Y_F32, ZTQ_NO_PDL. */
typedef struct ZtqGemvFusion {
    const void* residual;
    const void* norm_weight;
    void* sum_out;
    unsigned int eps_bits;
    int swiglu;
} ZtqGemvFusion;
cudaError_t ztq_gemv_w4g_fused(const void* qdata, const void* meta, const void* x, void* y, int N, int K, int group, int flags,
                               const ZtqGemvFusion* fz, cudaStream_t stream);
/* out row 2i = a row i, out row 2i+1 = b row i; rows of row_bytes bytes (a multiple of 16), 16-byte aligned
 * pointers.  Applied to the packed codes and to the {scale, zero} rows of a gate and an up projection it gives
 * the pair layout the SwiGLU epilogue wants (tensor.MergeQ4Storage, tensor/quantized.go:227, concatenates instead). */
cudaError_t ztq_interleave_rows(const void* a, const void* b, void* out, long long rows, int row_bytes, cudaStream_t stream);

/* Set-up helpers for the buffers above (not for the hot path: they allocate
 * and map memory).  ztq_symm_alloc returns zeroed device memory that can be
 * exported; the 64-byte handle travels to the peer processes by any host
 * channel; ztq_ipc_open maps a peer's buffer and enables peer access. */
cudaError_t ztq_symm_alloc(void** ptr, size_t bytes);
cudaError_t ztq_symm_free(void* ptr);
/* Zeroes a buffer of ztq_symm_alloc and waits for the device.  Used to bring the ranks back in step after a
 * launch that gave up on a peer (ztq_device_error() == 4): all ranks stop launching, meet on the host, zero
 * their slot buffer and state words, meet again, and carry on from sequence number 0. */
cudaError_t ztq_symm_zero(void* ptr, size_t bytes);
cudaError_t ztq_ipc_export(void* ptr, void* handle64);
cudaError_t ztq_ipc_open(const void* handle64, void** ptr);
cudaError_t ztq_ipc_close(void* ptr);

/* ---- residency: repack and quantize on the device -------------------------
 * One-off helpers for UploadWeights (compute/gpu_engine.go:778-1058). */

/* 18-byte AoS blocks (Q4Storage.RawBytes / IQ4NLStorage.RawBytes) -> separated layout. */
cudaError_t ztq_repack_blocks18(const void* aos, void* sep, long long n_blocks, cudaStream_t stream);
/* GPTQ/AWQ group scales and zeros (two fp16 arrays) -> interleaved half2 meta. */
cudaError_t ztq_pack_w4g_meta(const void* scales, const void* zeros, void* meta, long long n_groups,
                              cudaStream_t stream);
/* Flat TernaryStorage bytes -> row-aligned rows (a copy when K % 4 == 0). */
cudaError_t ztq_repack_ternary_rows(const void* flat, void* rows, int M, int K, cudaStream_t stream);

/* float32 -> packed, bit-identical to tensor.QuantizeQ4 / QuantizeQ8 /
 * QuantizeGPTQ(.,group,4) / QuantizeAWQ (n multiple of 32 / group). */
cudaError_t ztq_quantize_q4_0(const float* src, void* sep, long long n, cudaStream_t stream);
cudaError_t ztq_quantize_q8_0(const float* src, void* blocks36, long long n, cudaStream_t stream);
cudaError_t ztq_quantize_w4g(const float* src, void* qdata, void* meta, long long n, int group, int awq_rounding,
                             cudaStream_t stream);

/* packed -> float32, bit-identical to the storages' Dequantize(). fmt: 0 Q4_0,
 * 1 IQ4_NL, 2 W4G, 3 Q8_0, 4 ternary (row-aligned, aux = K). */
cudaError_t ztq_dequantize(int fmt, const void* w, const void* meta_or_null, float* dst, long long n, int aux,
                           cudaStream_t stream);

/* y[M, N] = x[M, K] * w[K, N] with w float32 row-major, as ztq_dequantize leaves the Slice() of a 4-bit storage:
 * the product of compute.MatMulW4A16 when the weights are the B operand (compute/w4a16.go:107-119), where the
 * dequantized slice is multiplied as a literal [K, N] matrix by CPUEngine.MatMul -> SgemmSimd
 * (internal/xblas/gemm_simd_amd64.go:16-36).  Summation over k ascending, fused multiply-add except in the last
 * N % 4 columns (multiply, then add), which is the order of that routine.  x: fp16, or float32 with ZTQ_X_F32.
 * A correctness path for that operand layout, not a tuned kernel.  Flags: ZTQ_X_F32, ZTQ_NO_PDL. */
cudaError_t ztq_matmul_wkn_f32(const void* x, const float* w_kn, float* y, int M, int K, int N, int flags, cudaStream_t stream);

/* ==== the decode step around the projections ================================
 * What stands between two quantized projections of a decode step: the plan of the step (block tables, slots), rotary
 * positions with the append of keys and values to a paged 8-bit cache, attention over that cache, and the token drawn
 * from the logits.  No counterpart on the reference's quantized path (its rope, paged attention and argmax kernels,
 * internal/cuda/kernels/, work on float32 caches with host-built tables).  All pointers belong to the current device.
 * All of these are safe to capture; lengths, tables and slots are read on the device, so one captured graph serves steps
 * of any lengths within the sizes given on the host. */

/* The plan of a step.  Per sequence b: ctx_len[b] tokens are cached, new_len[b] >= 0 tokens come in this step, or
 * new_len[b] == -1 ends the sequence and gives its blocks back.
 *   block_table [sequences][table_width]  blocks of a sequence in order; the entries this step needs are filled in, all
 *                                         others are left as they were
 *   ring [pool_blocks], ring_state {head, count}   free blocks: `count` of them from `head` on, wrapping around.  New
 *                                         blocks are taken from the head in the order of the sequences; blocks given
 *                                         back go behind the last one and are used from the next step on.
 *   ring_state_out {head, count}          may be ring_state itself
 *   query_start [sequences + 1]           first row of each sequence among the step's rows, then the number of rows
 *   positions, slots [max_tokens]         per row: position, and block * block_size + offset in the cache; rows behind
 *                                         the last sequence get position 0 and slot -1 (the append skips them)
 *   kv_len [sequences]                    tokens in the cache after the append (0: not in this step)
 *   next_len [sequences]                  ctx_len of the next step (may be ctx_len itself)
 *   status [sequences]                    0, or why a sequence gets nothing in this step (slots -1, kv_len 0, next_len =
 *                                         ctx_len): 1 not enough free blocks, 2 table_width too small, 3 max_tokens
 *                                         too small, 4 a negative or impossible length
 * When blocks run short, a sequence is refused if its blocks and those of all sequences before it that ask for any
 * exceed the free ones.  block_size: 16, 32, 64 or 128; sequences <= 4096.  Flags: ZTQ_NO_PDL. */
cudaError_t ztq_kv_plan(const int* ctx_len, const int* new_len, int* block_table, int* ring, const int* ring_state, int* ring_state_out,
                        int* next_len, int* kv_len, int* query_start, int* positions, int* slots, int* status, int sequences, int table_width,
                        int block_size, int pool_blocks, int max_tokens, int flags, cudaStream_t stream);

/* Rotary positions.  table [rows][rot_dim / 2] of float32 {cos, sin} of position * frequency, times `magnitude` (0: 1);
 * made once per model by ztq_rope_table (angles in 64 bits) for positions first .. first + rows - 1.
 * frequency i = base^(-2i / rot_dim), then
 *   ZTQ_ROPE_LINEAR    divided by factor
 *   ZTQ_ROPE_BY_TURNS  kept where it makes turns_high turns or more over original_positions, divided by factor where it
 *                      makes turns_low or fewer, a linear blend in the number of turns between
 *   ZTQ_ROPE_BY_DIM    the same, the blend linear in the dimension between those of turns_high (rounded down) and
 *                      turns_low (rounded up): "NTK-by-parts" (Peng et al., YaRN, 2023)
 * rot_dim: a multiple of 16 up to 256 and the head; what lies behind it in a head passes unchanged. */
#define ZTQ_ROPE_UNSCALED 0
#define ZTQ_ROPE_LINEAR   1
#define ZTQ_ROPE_BY_TURNS 2
#define ZTQ_ROPE_BY_DIM   3
typedef struct ZtqRopeSpec {
    double base, factor, turns_low, turns_high, original_positions, magnitude;
    int rot_dim, scaling;
} ZtqRopeSpec;
cudaError_t ztq_rope_table(void* table, int first, int rows, const ZtqRopeSpec* spec, int flags, cudaStream_t stream);
/* y[t, h] = x[t, h] rotated to positions[t]; strides in elements, head_dim contiguous and a multiple of 16 up to 256.
 * y may be x (same strides and type).  A position outside the table makes the rotated part of its row NaN and sets the
 * device error word to 6.  Flags: ZTQ_X_F32, ZTQ_Y_F32, ZTQ_ROPE_PAIRS, ZTQ_NO_PDL. */
cudaError_t ztq_rope(const void* x, void* y, int tokens, int heads, int head_dim, long long x_token, long long x_head, long long y_token,
                     long long y_head, const void* table, int table_rows, int rot_dim, const int* positions, int flags, cudaStream_t stream);

/* One layer's paged cache: int8 codes, a value is its code times the scale of its (block, head).  Element d of token o of
 * head h of block b stands at b * block_stride + (h * block_size + o) * head_dim + d of k and of v (block_stride in bytes, a
 * multiple of 16, so blocks of several layers, or of k and v, may interleave); scales are [blocks][kv_heads].
 * block_size 16, 32, 64 or 128; head_dim a multiple of 16 up to 256 (attention: 64, 128 or 256); k, v 16-byte aligned. */
typedef struct ZtqKvCache {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    long long block_stride;
    int blocks, kv_heads, block_size, head_dim;
} ZtqKvCache;

/* Rotates the queries into q_out (q_heads 0: none; q_out may be q) and appends the step's keys (rotated) and values to the
 * cache at `slots` (negative: the row is skipped, and a position outside the table is no error).  table NULL: nothing is rotated.  Strides in elements.
 * The scale of a (block, head) becomes the smallest power of two that holds the new rows' largest value in 127 steps, or
 * stays if it is larger already and the block held rows of the sequence (slot offset > 0); codes in the block are rounded
 * to a grown scale.  A block whose new rows are not finite gets the scale NaN until it is begun anew.
 * The rows of one block stand one after the other with consecutive slots, as ztq_kv_plan lays them out, and no slot comes
 * twice; a row out of order behind one of its block, or a slot behind the cache, is skipped and sets the device error
 * word to 5.  Flags: ZTQ_X_F32 (q, k, v), ZTQ_Y_F32 (q_out), ZTQ_ROPE_PAIRS, ZTQ_NO_PDL. */
cudaError_t ztq_rope_append_q8(const void* q, const void* k, const void* v, void* q_out, long long q_token, long long q_head, long long k_token,
                               long long k_head, long long v_token, long long v_head, long long qo_token, long long qo_head, int tokens, int q_heads,
                               const void* table, int table_rows, int rot_dim, const int* positions, const int* slots, const ZtqKvCache* cache,
                               int flags, cudaStream_t stream);
/* The cache's dequantizer: k_out, v_out [tokens][kv_heads][head_dim] (either may be NULL; fp16, or float32 with ZTQ_Y_F32)
 * = the cache's rows at `slots`; a slot outside the cache leaves its row as it was. */
cudaError_t ztq_kv_read_q8(const ZtqKvCache* cache, const int* slots, int tokens, void* k_out, void* v_out, int flags, cudaStream_t stream);

/* y[t, h] = attention of query row t, head h over its sequence's cached tokens: causal (the last row of a sequence stands
 * at position kv_len - 1), and with window > 0 only over the last `window` positions up to its own.  q_heads is a multiple
 * of kv_heads; head h reads kv head h / (q_heads / kv_heads).  Rows of sequence b: query_start[b] .. query_start[b + 1];
 * rows behind the last sequence are left as they were; a row that sees nothing becomes 0.  scale_bits: the softmax
 * scale's float32 bits.  max_new: most rows of one sequence (a sequence with more is left out and sets the device error
 * word to 8).  A block table entry outside the cache hides its tokens and sets the error word to 7; entries in front of the
 * window of a sequence's first row are not looked at.  A scale that is not finite makes the rows that see its tokens NaN.
 * workspace: >= ztq_attn_q8_workspace_bytes(...) of the same sizes, 16-byte aligned, overwritten; calls that share one must not overlap on the GPU
 * (two captured graphs that may run at once need one each).  sequences <= 4096.
 * With ZTQ_X_F32 or ZTQ_Y_F32 queries (of any size) and weights enter the products with 22 bits, else weights with 11; scores,
 * softmax sums and outputs are summed in fp32.  A weight times its V scale keeps these bits down to 2^-15 (else 2^-18) of the row's
 * largest such product and is held to 2^-36 (2^-28) of it; V scales below 2^-90 count as that.  Flags: ZTQ_X_F32, ZTQ_Y_F32, ZTQ_NO_PDL. */
size_t ztq_attn_q8_workspace_bytes(int tokens, int sequences, int max_new, int q_heads, int kv_heads, int head_dim);
cudaError_t ztq_attn_q8(const void* q, void* y, long long q_token, long long q_head, long long y_token, long long y_head, int tokens, int q_heads,
                        const int* query_start, const int* kv_len, const int* block_table, int sequences, int table_width, int max_new, int window,
                        unsigned scale_bits, const ZtqKvCache* cache, void* workspace, size_t workspace_bytes, int flags, cudaStream_t stream);

/* One token per row of logits [rows][vocab] (row_stride in elements; fp16, or float32 with ZTQ_X_F32) from uniform[row] in
 * [0, 1).  Tokens in order of (logit descending, index ascending), w = exp((logit - largest) / temperature); the first
 * top_k stay (<= 0: all), of those the shortest prefix with top_p of their mass (at least one token; >= 1: all), of those
 * the ones with w >= min_p; the token is the first by index whose running sum of w exceeds uniform times the sum.
 * temperature 0 takes the first of the order.  Per-row arrays; temperature, top_k, top_p, min_p may be NULL (1, all,
 * all, all).  w is held in steps of 2^-44 of the largest: a token below 2^-45 counts as 0 and is not drawn, not even for
 * uniform 0.  logprob (may be NULL): log of the token's share of what was kept.  -inf and NaN are never drawn; a row
 * with nothing else gives token -1 and logprob NaN.  vocab <= ZTQ_SAMPLE_MAX_VOCAB.  Flags: ZTQ_X_F32, ZTQ_NO_PDL. */
#define ZTQ_SAMPLE_MAX_VOCAB 327680
cudaError_t ztq_sample(const void* logits, long long row_stride, int rows, int vocab, const float* temperature, const int* top_k,
                       const float* top_p, const float* min_p, const float* uniform, int* token, float* logprob, int flags, cudaStream_t stream);

/* ---- probes ---------------------------------------------------------------- */
/* The launch plan the first launch of a call with these arguments gets on a device of `sms` SMs (host
 * arithmetic only, no device needed).  fmt: 0 Q4_0, 1 IQ4_NL, 2 W4G, 3 Q8_0, 4 ternary, 5 Q4_K, 6 Q5_K, 7 Q6_K
 * (the ztq_gemv_* entry points), 8 ztq_gemm_w4g_tc.  out[12]:
 *   GEMV    {kernel: 0 plain / 1 streaming / 2 chunk-pair, activation rows per launch, rows per team per stage,
 *            rows per stage, stages, overlay stages, rows per pass, grid, tiles of the busiest CTA, passes of
 *            the busiest CTA, warps per team, teams}
 *   tensor  {3, padded columns, K slices, groups per slice, row tiles, work items, grid, items of the busiest
 *            CTA, 0, 0, 0, 0}
 * Returns 0, or 1 for arguments no entry point accepts.  Tests use it to state which code path a shape runs. */
int ztq_describe_plan(int fmt, int N, int K, int group, int batch, int sms, int* out);
int ztq_check_sm100(void);          /* 1 when the current device is compute capability 10.x */
/* Launches a kernel that does nothing, with the grid, block size, dynamic shared memory and (unless ZTQ_NO_PDL)
 * the programmatic-dependent-launch attribute of a GEMV launch.  A stream of these measures the floor of a
 * dependent launch on the device at hand: the part of a small GEMV's time that no kernel change can remove. */
cudaError_t ztq_probe_launch(int grid, int threads, int smem_bytes, int flags, cudaStream_t stream);
int ztq_abi_version(void);
/* Reads and clears the device-side error word (0 = none; see ztq_common.cuh): the first error of one of the operators that had any.
 * Synchronises the device: a diagnostic call, not for the hot path. */
int ztq_device_error(void);

#ifdef __cplusplus
}
#endif
#endif /* ZTQ_H */
