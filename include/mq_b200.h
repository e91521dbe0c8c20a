/*
 * mq_b200 — B200 (sm_100a) quantized-linear engine behind a plain C ABI.
 *
 * Drop-in device path for mini_ai's quantized linear: y = x · Wᵀ over GGUF
 * Q8_0 / Q4_0 / Q4_1 weights. Every entry point takes plain pointers and
 * sizes, returns MQ_OK (0) or a negative MQ_ERR_* code, and leaves a message
 * in mq_last_error() for the calling thread. No C++ exception crosses this
 * boundary. Device pointers are CUDA device addresses on the handle's device;
 * `stream` is a cudaStream_t (NULL = the legacy default stream) and every
 * device call is stream-ordered and asynchronous unless stated otherwise.
 *
 * Reference interfaces replaced (paths in the mini_ai project):
 *   - QuantizeTensor / TensorFromQuantized / DequantizeTensor,
 *     include/mini_llama/quantized_tensor.h:21-24
 *   - QuantizedDotRow, include/mini_llama/quantized_tensor.h:25
 *   - LinearDispatch (quantized branch), include/mini_llama/matmul_dispatch.h:28
 *   - CudaModelState::UploadWeight + LinearKernel, src/cuda_backend.cu:94-110,275-283
 *   - CudaDeviceInfo, include/mini_llama/backend.h:10
 */
#ifndef MQ_B200_H_
#define MQ_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* GGML block types; the numeric values are the reference's QuantType ids
 * (include/mini_llama/quantized_tensor.h:10 == gguf.h:15-17). */
enum {
  MQ_Q4_0 = 2, /* 18-byte block: fp16 d, 16 bytes of nibbles; w = d*(q-8)   */
  MQ_Q4_1 = 3, /* 20-byte block: fp16 d, fp16 m, 16 bytes;     w = d*q + m   */
  MQ_Q8_0 = 8  /* 34-byte block: fp16 d, 32 int8;              w = d*q       */
};

enum {
  MQ_OK = 0,
  MQ_ERR_INVALID = -1,     /* bad argument: type, shape, pointer, stride     */
  MQ_ERR_CUDA = -2,        /* a CUDA runtime call failed                     */
  MQ_ERR_SIZE = -3,        /* byte count does not match rows x cols x type   */
  MQ_ERR_NONFINITE = -4,   /* quantize input holds Inf/NaN                   */
  MQ_ERR_RANGE = -5,       /* quantize scale or min overflows fp16           */
  MQ_ERR_TIMEOUT = -6,     /* a bounded device wait on a peer ran out        */
  MQ_ERR_UNSUPPORTED = -7  /* not built for this device / configuration      */
};

typedef struct mq_weight mq_weight; /* opaque device-resident packed weight */

/* Message for the last failing call on this thread ("" if none). */
const char *mq_last_error(void);

/* Library version string. */
const char *mq_version(void);

/* Bytes of the GGUF block stream for a rows x cols matrix: rows *
 * ceil(cols/32) * {34|18|20}; 0 for an unknown type or a non-positive shape.
 * Mirrors the size rule of TensorFromQuantized, src/quantized_tensor.cc:88-96. */
size_t mq_quantized_bytes(int qtype, int rows, int cols);

/* Bit-exact host quantizer: packs a row-major F32 rows x cols matrix into
 * GGUF blocks exactly as QuantizeTensor does (src/quantized_tensor.cc:104-159),
 * using `threads` host threads (0 = all hardware threads). Errors:
 * MQ_ERR_NONFINITE for Inf/NaN input, MQ_ERR_RANGE when a scale or Q4_1 min
 * overflows fp16, MQ_ERR_SIZE when dst_bytes is not mq_quantized_bytes(). */
int mq_quantize(int qtype, const float *src, int rows, int cols, void *dst, size_t dst_bytes, int threads);

/* Host decoder, DequantizeTensor (src/quantized_tensor.cc:193-206). */
int mq_dequantize(int qtype, const void *blocks, size_t nbytes, int rows, int cols, float *dst);

/* Device quantizer: the same bit-exact packing as mq_quantize, run on the GPU
 * over a device F32 matrix into a device GGUF block buffer. Input errors
 * (non-finite values, fp16 overflow) are reported when the call returns, so
 * this call synchronizes `stream`. */
int mq_quantize_device(int device, int qtype, const float *d_src, int rows, int cols, void *d_dst,
                       size_t dst_bytes, void *stream);

/* Upload a packed weight. `blocks` is the GGUF block stream (host memory when
 * blocks_on_device == 0, a device pointer on `device` otherwise) of a rows x
 * cols matrix. The weight is re-laid out on the device for 16-byte vector
 * loads (quants and fp16 scales in separate, aligned planes); the number of
 * bytes per weight is unchanged. Replaces CudaModelState::UploadWeight
 * (src/cuda_backend.cu:275-283). Synchronizes `stream` before returning. */
int mq_weight_create(int device, int qtype, int rows, int cols, const void *blocks, size_t nbytes,
                     int blocks_on_device, void *stream, mq_weight **out);

/* Upload rows [row_begin, row_end) of a rows x cols packed weight as its own
 * handle: the output-row shard one GPU holds when a projection is split
 * across GPUs. `blocks` is the FULL matrix's block stream (host or device). */
int mq_weight_shard_create(int device, int qtype, int rows, int cols, int row_begin, int row_end,
                           const void *blocks, size_t nbytes, int blocks_on_device, void *stream,
                           mq_weight **out);

/* Release a handle and its device memory (NULL is a no-op). */
void mq_weight_destroy(mq_weight *w);

/* Shape, type, device and device bytes of a handle (any out-pointer may be NULL). */
int mq_weight_info(const mq_weight *w, int *qtype, int *rows, int *cols, int *device, size_t *device_bytes);

/* Write the handle's weight back as a GGUF block stream to host memory
 * (round-trip check of the device layout). Synchronous. */
int mq_weight_export(const mq_weight *w, void *dst, size_t dst_bytes);

/* y[i, n] = sum_k x[i, k] * W[n, k] (+ bias[n]) for i in [0, m).
 * x: device F32 [m, ldx] with ldx >= cols; y: device F32 [m, ldy] with
 * ldy >= rows; bias: device F32 [rows] or NULL. Small m runs a streaming
 * GEMV, larger m the tcgen05 tensor-core GEMMs (see mq_set_path). The tensor-
 * core paths keep per-(device, stream) scratch for the split activations,
 * allocated on first use and grown as needed (the growth synchronizes the
 * stream). A bounded wait that runs out inside a GEMM launch is reported as
 * MQ_ERR_TIMEOUT by the next mq_linear call on that device. Accumulation is
 * fp32; results
 * match the reference's sequential fp32 dot (QuantizedDotRow,
 * src/quantized_tensor.cc:161-191) to within accumulation-order rounding.
 * The quantized branch of LinearDispatch (src/matmul_optimized.cc:172-174)
 * and LinearKernel (src/cuda_backend.cu:94-110) accept m == 1 only; here any
 * m >= 0 works (m == 0 is a no-op). */
int mq_linear(const mq_weight *w, const float *x, int m, int ldx, const float *bias, float *y, int ldy,
              void *stream);

/* The gate/up half of the Llama FFN in one call: y = SwiGlu(x * W_gateᵀ,
 * x * W_upᵀ), i.e. y[i, n] = g / (1 + exp(-g)) * u with g, u the two products,
 * as FfnForward's `Linear(h, w_gate)`, `Linear(h, w_up)`, `SwiGlu(gate, up)`
 * (src/forward.cc:105-110; SwiGluKernel, src/cuda_backend.cu:241-245; Silu,
 * src/ops.cc:85-91). The gate product goes to a per-(device, stream) scratch
 * buffer and the up product's kernel applies the SwiGLU in its output write,
 * so the separate elementwise pass and one round trip of both outputs are
 * gone. Both weights must have the same shape and device; x, y as mq_linear. */
int mq_linear_swiglu(const mq_weight *w_gate, const mq_weight *w_up, const float *x, int m, int ldx, float *y,
                     int ldy, void *stream);

/* y = residual + (x * Wᵀ + bias): the linear followed by the residual add of
 * ForwardCuda (`AddKernel(x, o)` after the wo and w_down projections,
 * src/cuda_backend.cu:236-240), in the kernel's own output write. residual:
 * device F32 [m, ldy] with y's stride; it may be y itself (the usual
 * in-place residual stream). Otherwise as mq_linear. */
int mq_linear_residual(const mq_weight *w, const float *x, int m, int ldx, const float *bias, const float *residual,
                       float *y, int ldy, void *stream);

/* Same product for a ragged batch: `offsets` (host, n_seqs + 1 entries,
 * offsets[0] == 0, non-decreasing) delimits each request's rows inside the
 * contiguous [offsets[n_seqs], ldx] activation matrix. The rows are
 * independent, so the result equals mq_linear with m = offsets[n_seqs]; the
 * offsets are validated and kept for callers that need per-request slices. */
int mq_linear_ragged(const mq_weight *w, const float *x, const int *offsets, int n_seqs, int ldx,
                     const float *bias, float *y, int ldy, void *stream);

/* Same product as mq_linear for decode-sized batches, for callers that cannot
 * allocate device memory: they own every device byte through their own pool,
 * run under a fixed memory budget, or call from a hot loop where cudaMalloc's
 * device-wide synchronisation and latency are not acceptable. It has no
 * counterpart in the reference. This call allocates nothing: its scratch is a
 * fixed 3.6 MiB device array that every GPU loading the library holds until
 * the process exits. Limits: 1 <= m <= 16 (m == 0 is a no-op), weight cols
 * <= 16384 and rows <= 131072; larger requests fail with MQ_ERR_INVALID. The
 * first call on a device resolves the array's device address there, so make
 * that first call before any stream capture. All calls on a device share the
 * array, so calls that overlap on the GPU (other streams, other host threads)
 * race and must be serialised by the caller. A bounded device wait that runs
 * out writes NaN to the outputs. */
int mq_linear_noalloc(const mq_weight *w, const float *x, int m, int ldx, const float *bias, float *y, int ldy,
                      void *stream);

/* ---- Paged 4-bit key/value cache for serving: what a forward over ragged
 * requests needs between its projections (mq_linear_ragged). A cache holds,
 * for each layer, `pages` pages of `page_size` consecutive tokens of one
 * request; page ids are shared by the layers. Every 32 elements of a key or
 * value row are a Q4_0 block, c * d with c in [-8, 7]: for the block's first
 * element s of largest |x|, d = fp16(bf16(s / -8)), and c = x / d rounded to
 * nearest even and clamped. (d has 8 significant bits, so that every c * d
 * is an fp16 number; mq_quantize keeps 11, so its blocks hold other values.)
 * A block with a non-finite element, or whose |d| would pass 8160, is stored
 * as NaN, and attention that sees it answers NaN. 4.5 bits an element. No
 * counterpart in the reference, whose forward keeps one max_seq_len F32
 * cache per context (src/forward.cc).
 *
 * A step: mq_pages_plan once, then for each layer mq_kv4_store and
 * mq_kv4_attention on the same stream. All lengths, offsets and tables are
 * int32 device arrays, read by the kernels when they run: a captured graph
 * serves every step of its buffers' sizes. No call allocates device memory or
 * synchronises, except a creation that is given none and its destruction. */
typedef struct mq_kv4 mq_kv4;

/* Device bytes of a cache: layers * pages * page_size * kv_heads * head_dim *
 * 9 / 8; 0 (and mq_last_error) for a shape that mq_kv4_create refuses. */
size_t mq_kv4_bytes(int layers, int pages, int page_size, int kv_heads, int head_dim);

/* A cache of zeros on `device`. page_size: a multiple of 16 up to 1024;
 * head_dim: 32, 64, 96 or 128; kv_heads up to 65536; pages * page_size <
 * 2^31. `memory` is the caller's device memory for it (at least
 * mq_kv4_bytes(), 16-byte aligned), which must outlive the handle and is
 * cleared on `stream`; NULL allocates it, which synchronizes `stream`.
 * MQ_KV4_WAIT_NS in the environment limits each wait inside the cache's
 * attention (nanoseconds, default 1 s, at most 10 s); with
 * MQ_KV4_LOSE_COPIES=1 every such wait runs out, so that a program's
 * handling of MQ_ERR_TIMEOUT can be tried. */
int mq_kv4_create(int device, int layers, int pages, int page_size, int kv_heads, int head_dim, void *memory,
                  size_t memory_bytes, void *stream, mq_kv4 **out);
void mq_kv4_destroy(mq_kv4 *c);

/* Shape, device and device bytes of a handle (any out-pointer may be NULL). */
int mq_kv4_info(const mq_kv4 *c, int *device, int *layers, int *pages, int *page_size, int *kv_heads, int *head_dim,
                size_t *device_bytes);

/* Packs key and value rows into `layer` at `slots` (slot = page id *
 * page_size + place in the page; a row whose slot is negative or past the
 * cache is skipped). Head h of row i: device F32 k + i * ld_k + h * hs_k,
 * head_dim elements (the rows of a fused [q | k | v] projection: ld its row
 * length, hs = head_dim); any alignment to 4 bytes works, 16-byte pointers
 * and strides run faster. The slots of one call must differ: of two rows for
 * one slot, either may win each block. */
int mq_kv4_store(const mq_kv4 *c, int layer, const float *k, int64_t ld_k, int64_t hs_k, const float *v, int64_t ld_v,
                 int64_t hs_v, const int *slots, int rows, void *stream);

/* The values that `layer` holds at `slots`, into k and v [rows][kv_heads]
 * [head_dim]; rows of a negative slot or one past the cache are 0. */
int mq_kv4_load(const mq_kv4 *c, int layer, const int *slots, int rows, float *k, float *v, void *stream);

/* Workspace bytes of mq_kv4_attention for this cache, head count and
 * max_new, whatever the batch; 0 for a NULL handle. */
size_t mq_kv4_attention_workspace(const mq_kv4 *c, int heads, int max_new);

/* Causal attention over the cache: row i of request r (rows offsets[r] ..
 * offsets[r + 1] - 1 of q and out; offsets[0] = 0, non-decreasing) stands at
 * position seq_lens[r] - (offsets[r + 1] - offsets[r]) + i of its request and
 * sees positions 0 up to its own, at most seq_lens[r] of them:
 *   out = softmax(scale * q . k) v, query head h with KV head h / (heads / kv_heads).
 * seq_lens counts the step's own rows, which mq_kv4_store has written.
 * block_tables [n_seqs][max_pages] page ids, max_pages * page_size <= 2^31 -
 * 4097; lengths past max_pages * page_size count as that, and tokens of a
 * page id outside the cache are not seen. A row that sees nothing is 0; rows
 * past offsets[n_seqs] stay as they are, and no row past `rows` is touched.
 * max_new: the most rows that a request brings, as far as the caller knows;
 * it selects kernels and a lower or higher value costs time only. q and out
 * as in mq_kv4_store, no two heads of out sharing memory; out may be q only
 * if it has q's strides. F32 softmax and sums; q and the softmax weights
 * enter the tensor cores as fp16 hi + lo pairs (22 bits). workspace: device
 * memory of at least mq_kv4_attention_workspace() bytes, 16-byte aligned,
 * not shared with a call that may run at the same time; its contents do not
 * matter. The summation order is fixed: equal inputs give equal bits. Every
 * wait of the kernels is bounded: where one runs out, all rows that its CTA
 * had still to write are NaN, and so are the cut rows that it had a part in;
 * the device's error flag (mq_device_error_flag) is raised, and the next
 * call returns MQ_ERR_TIMEOUT without launching anything. */
int mq_kv4_attention(const mq_kv4 *c, int layer, const float *q, int64_t ld_q, int64_t hs_q, int rows, int heads,
                     const int *offsets, const int *seq_lens, const int *block_tables, int n_seqs, int max_pages,
                     int max_new, float scale, float *out, int64_t ld_out, int64_t hs_out, void *workspace,
                     size_t workspace_bytes, void *stream);

/* Block tables and slot map of a step, from the lengths of its requests
 * (n_seqs <= 8192). Request r holds ctx_lens[r] tokens, in the pages of its
 * row of block_tables [n_seqs][max_pages], and brings new_lens[r] rows. The
 * further pages that it needs are taken from the top of the stack free_pages
 * (capacity n_pages, *n_free of them valid) in request order and entered in
 * its row. Out: offsets [n_seqs + 1], the rows before each request;
 * seq_lens [n_seqs] = ctx + new (may be ctx_lens); slots and positions
 * [rows], -1 behind the last request; *n_free_out (may be n_free).
 * A request is refused when a length is negative, when ctx + new passes
 * max_pages * page_size, when its rows (or, where it brings none, the rows
 * before it) pass `rows`, or when it needs pages and it and the requests
 * before it need more than *n_free: its table, length and the stack stay as
 * they were, and its rows get slot -1. *refused counts them. The rows of a
 * refused request keep their place in offsets, and mq_kv4_attention, which
 * knows only lengths, takes them for the request's last cached tokens: finite
 * values that mean nothing. Tell them by their slots or positions of -1. */
int mq_pages_plan(int device, const int *ctx_lens, const int *new_lens, int n_seqs, int page_size, int *block_tables,
                  int max_pages, const int *free_pages, int n_pages, const int *n_free, int rows, int *offsets,
                  int *seq_lens, int *slots, int *positions, int *n_free_out, int *refused, void *stream);

/* Ends requests: pushes the pages of requests[0..n) (indices of the rows of
 * block_tables; those outside [0, n_seqs) are skipped, one named twice counts
 * once) onto the stack and sets their seq_lens to 0. The stack never passes
 * its capacity n_pages. */
int mq_pages_release(int device, const int *requests, int n, int n_seqs, int page_size, int *seq_lens,
                     const int *block_tables, int max_pages, int *free_pages, int n_pages, int *n_free, void *stream);

/* ---- Row-sharded linear across GPUs (one process or host thread per GPU).
 * A weight of N = G*R rows is split into G equal output-row shards
 * (mq_weight_shard_create with rows [r*R, (r+1)*R) on rank r). Each rank
 * computes its R outputs and an NCCL all-gather over NVLink assembles the
 * full [m, N] output on every rank. The result equals mq_linear on the whole
 * weight up to fp32 summation order: the kernels split each tile's K range
 * across CTAs by the launch's total work, so a shard may sum in another order
 * (bit-identical where both launches split alike, e.g. when neither has more
 * (128-row tile, K step) chunks than SMs). No counterpart in the reference, which runs every
 * linear on one device (`--device N`, src/main.cc:249-250); new surface for
 * the multi-GPU row of the hot path. NCCL is loaded at run time
 * (libnccl.so.2). */
typedef struct mq_comm mq_comm;
#define MQ_COMM_ID_BYTES 128

/* A fresh communicator id (rank 0 creates it and shares it with the other
 * ranks through the caller's own host channel). len >= MQ_COMM_ID_BYTES. */
int mq_comm_unique_id(void *id, size_t len);

/* Join the communicator of `nranks` ranks as `rank`, on `device`. Collective:
 * every rank must call it with the same id. With MQ_P2P_GATHER=1 in every
 * rank's environment (and 2..8 ranks) it also allocates a staging region of
 * 2 * nranks * 4 MiB on `device` and maps every peer's region through CUDA
 * IPC, so that mq_linear_sharded_allgather gathers over NVLink peer memory
 * instead of NCCL; if any rank cannot map every peer, all ranks use NCCL.
 * Destroy the communicators only after every rank's last gather completed
 * (for example after a barrier). */
int mq_comm_create(int device, int nranks, int rank, const void *id, size_t len, mq_comm **out);
void mq_comm_destroy(mq_comm *c);

/* 1 when the communicator gathers over NVLink peer memory (MQ_P2P_GATHER=1
 * and every rank mapped every peer), 0 when it uses NCCL's all-gather, a
 * negative code for a NULL handle. */
int mq_comm_uses_peer_gather(const mq_comm *c);

/* y[i, n] for all n in [0, N) on every rank: this rank's shard product
 * (+ bias[rank*R .. rank*R+R) when bias, the full [N] vector, is given) and
 * an all-gather of the slices. x: device F32 [m, ldx] (full K); y: device F32
 * [m, ldy] with ldy >= N. Stream-ordered on `stream`; every rank must call it
 * with the same m, in the same order relative to its other collectives. The
 * peer-memory gather (see mq_comm_create) takes outputs with m * R <= 2^20 and
 * may be captured in a CUDA graph. A peer that does not arrive within the wait
 * limit (MQ_P2P_WAIT_NS nanoseconds in the environment at mq_comm_create,
 * default 1 s) leaves NaN in that peer's output columns and poisons the
 * communicator: its next call and every later peer-memory gather on it fail
 * with MQ_ERR_TIMEOUT (replays of a captured graph write NaN without
 * waiting); destroy it and create a new one. */
int mq_linear_sharded_allgather(const mq_weight *shard, const float *x, int m, int ldx, const float *bias,
                                float *y, int ldy, mq_comm *comm, void *stream);

/* Kernel selection for the next mq_linear calls on this thread:
 * 0 = automatic (default): the tcgen05 int8 decode GEMV for m <= 4, the
 *     tcgen05 scale-folded decode GEMM for m <= 32 (the fp16 decode GEMM for
 *     weights whose block scales exceed the fold's fp16 range), the tcgen05
 *     prefill GEMM above;
 * 1 = force the stream-K SIMT GEMV, 2 = force the tcgen05 prefill GEMM,
 * 3 = force the tcgen05 int8 decode GEMV, 4 = force the tcgen05 fp16 decode
 * GEMM, 5 = force the SIMT dp4a decode GEMV, 6 = force the tcgen05
 * scale-folded decode GEMM (MQ_ERR_UNSUPPORTED for weights outside its
 * range), 7 = force the scale-folded decode GEMM on CTA pairs (tcgen05
 * cta_group::2; MQ_ERR_UNSUPPORTED for weights outside the fold's range or
 * with an odd number of 128-row tiles); other values are ignored. Returns the
 * previous mode. */
int mq_set_path(int mode);

/* Number of kernels this library has launched in this process (all devices,
 * all threads): the evidence a benchmark reports as its kernel count. */
uint64_t mq_kernel_launches(void);

/* Human-readable device list, like CudaDeviceInfo (src/cuda_backend.cu:355-369). */
int mq_device_info(char *buf, size_t len);

/* The bounded-wait error flag of `device` as its kernels see it: a device
 * pointer to an int in mapped host memory. A tensor-core kernel whose wait ran
 * out stores 1 there; the next tensor-core call on that device then returns
 * MQ_ERR_TIMEOUT and clears it. Exposed so that a monitor or a test can read
 * the flag or raise it from the device (cudaMemset, or a kernel's store). */
int mq_device_error_flag(int device, int **flag);

#ifdef __cplusplus
}
#endif
#endif /* MQ_B200_H_ */
