#ifndef QWN_HIP_EXT_H
#define QWN_HIP_EXT_H

/*
 * qwn_hip extensions beyond the reference's qwnrun ABI.
 *
 * None of these has a counterpart in c/cuda/qwn_cuda_abi.h.  They exist for
 * callers that keep activations on the device: a resident decode loop, a
 * benchmark that times kernels with inputs already in HBM, HIP graph
 * capture.  They take DEVICE pointers, enqueue on the caller's stream
 * (a hipStream_t passed as void*; NULL = the context's own stream, a
 * blocking stream, so ordered with work on the null stream), never
 * synchronise and never allocate, so they are safe to record into a graph.
 * The library advertises them with QWN_CUDA_CAP_DEVICE_POINTERS.
 *
 * Contexts, tensors and KV caches are the handles of qwn_cuda_abi.h.
 * Device pointer alignment: int8 activation rows and fp32 activation rows
 * must start on 16-byte boundaries (pointer and row stride).
 */

#include "qwn_cuda_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    QwnCudaAbiHeader header;
    uint32_t dtype;          /* QwnCudaTensorDType */
    uint32_t rows;
    uint32_t cols;
    uint32_t units_per_row;  /* lane work units: HyperVSQ-2 block, 4 Q4_0 blocks, 8 halves */
    uint64_t logical_bytes;  /* bytes in the on-disk format (what the ABI was given) */
    uint64_t device_bytes;   /* bytes resident in the device layout */
    uint32_t lanes_per_row;  /* launch plan for batch 1 */
    uint32_t units_per_lane;
    uint32_t rows_per_wave;
    uint32_t grid;
    uint64_t mfma_copy_bytes; /* the batched GEMM's MFMA-order copy (0: none), charged to the
                                 context's budget and gpu_resident_bytes with logical_bytes */
} QwnHipTensorInfo;

/* Shape, byte counts and batch-1 launch plan of a resident tensor. */
QWN_CUDA_ABI_API int qwn_hip_ext_tensor_info(const QwnCudaTensorHandle *tensor,
                                             QwnHipTensorInfo *info);

/* Activation images.  The GEMV reads activations from an "image": per token
 * the exact LDS layout its dot products use (int8 values split into signed
 * high and unsigned low nibbles in the order the weight unpack produces,
 * plus per-32 correction sums; fp32 for F16 tensors).  Images depend only
 * on the tensor's dtype and column count, so one image serves every tensor
 * with the same input (q/k/v, gate/up).  Image strides and pointers must be
 * 16-byte aligned. */
QWN_CUDA_ABI_API uint64_t qwn_hip_ext_activation_image_bytes(const QwnCudaTensorHandle *tensor);

/* Image from int8 tokens (HyperVSQ-2, Q4_0 tensors) or fp32 tokens (F16
 * tensors): x [batch][x_stride elements] -> image [batch][image_stride]. */
QWN_CUDA_ABI_API int qwn_hip_ext_prepare_image_device(QwnCudaContextHandle *context,
                                                      const QwnCudaTensorHandle *tensor,
                                                      const void *x, uint32_t batch,
                                                      uint32_t x_stride, void *image,
                                                      uint32_t image_stride, void *stream);

/* Per-token int8 quantization of fp32 x (the activation step of
 * c/qwanto_kernels.c:354-433) fused with the image build: writes scales
 * [batch], the images and, if q8 is not NULL, the int8 tokens
 * [batch][q8_stride] zero padded. */
QWN_CUDA_ABI_API int qwn_hip_ext_quantize_image_device(QwnCudaContextHandle *context,
                                                       const QwnCudaTensorHandle *tensor,
                                                       const float *x, uint32_t batch,
                                                       uint32_t x_stride, void *image,
                                                       uint32_t image_stride, float *scales,
                                                       int8_t *q8, uint32_t q8_stride,
                                                       void *stream);

/* GEMV/GEMM on images: output [batch][output_stride] = W x_t * scale_t
 * (scales[t], or `scale` when scales is NULL; ignored for F16).  Weights
 * are read once per 16 tokens. */
QWN_CUDA_ABI_API int qwn_hip_ext_gemm_image_device(QwnCudaContextHandle *context,
                                                   const QwnCudaTensorHandle *tensor,
                                                   const void *image, uint32_t image_stride,
                                                   const float *scales, float scale,
                                                   float *output, uint32_t batch,
                                                   uint32_t output_stride, void *stream);

/* Grouped GEMV: up to 4 tensors of one dtype and column count that share
 * one input (q/k/v, gate/up) in a single launch.  Input modes:
 *   IMAGE    prebuilt activation images [batch][image_stride], scales
 *   F32      one fp32 token x [cols] (cols a multiple of 32); every
 *            workgroup quantizes it per token itself (c/qwanto_kernels.c:
 *            354-433) into its LDS image -- no separate quantize launch
 *   RMSNORM  y = (x * 1/sqrt(mean(x^2) + eps)) * norm, then as F32
 *            (c/qwanto_decode.c:627-652)
 *   SWIGLU   y = (x / (1 + exp(-x))) * x2, then as F32
 *            (c/qwanto_decode.c:1946-1949)
 * Output modes: STORE; ADD (outputs += result, one token: the residual
 * stream); ARGMAX (store, and one packed key per workgroup in
 * argmax_partials -- qwn_hip_ext_gemv_group_partials() of them -- reduced
 * by qwn_hip_ext_argmax_device to the first index of the largest output);
 * SWIGLU (two tensors of one shape, gate and up, one token: outputs[0] =
 * (g / (1 + exp(-g))) * u per row, c/qwanto_decode.c:1946-1949; outputs[1]
 * is not written).
 * Device pointers, caller's stream, no allocation. */
#define QWN_HIP_GEMV_INPUT_IMAGE 0u
#define QWN_HIP_GEMV_INPUT_F32 1u
#define QWN_HIP_GEMV_INPUT_RMSNORM 2u
#define QWN_HIP_GEMV_INPUT_SWIGLU 3u
#define QWN_HIP_GEMV_OUTPUT_STORE 0u
#define QWN_HIP_GEMV_OUTPUT_ADD 1u
#define QWN_HIP_GEMV_OUTPUT_ARGMAX 2u
#define QWN_HIP_GEMV_OUTPUT_SWIGLU 3u
#define QWN_HIP_GEMV_MAX_GROUP 4u

typedef struct {
    QwnCudaAbiHeader header;
    uint32_t count;                       /* tensors, 1..4 */
    uint32_t input_mode;                  /* QWN_HIP_GEMV_INPUT_* */
    uint32_t output_mode;                 /* QWN_HIP_GEMV_OUTPUT_* */
    uint32_t batch;                       /* tokens (image input); 1 otherwise */
    const QwnCudaTensorHandle *tensors;   /* [count] */
    float *const *outputs;                /* [count] device fp32 [batch][output_stride] */
    uint32_t output_stride;               /* 0: rows of each tensor */
    uint32_t image_stride;
    const void *image;
    const float *scales;                  /* image input: per-token scales or NULL */
    float scale;                          /* image input without scales */
    float eps;                            /* RMSNORM */
    const float *x;                       /* fp32 input [cols] */
    const float *x2;                      /* SWIGLU: the up projection [cols] */
    const float *norm;                    /* RMSNORM weights [cols] */
    float *scale_out;                     /* optional: the activation scale (one float) */
    uint64_t *argmax_partials;            /* ARGMAX */
} QwnHipGemvGroupRequest;

QWN_CUDA_ABI_API uint32_t qwn_hip_ext_gemv_group_partials(QwnCudaContextHandle *context,
                                                          const QwnHipGemvGroupRequest *request);
QWN_CUDA_ABI_API int qwn_hip_ext_gemv_group_device(QwnCudaContextHandle *context,
                                                   const QwnHipGemvGroupRequest *request, void *stream);
QWN_CUDA_ABI_API int qwn_hip_ext_argmax_device(QwnCudaContextHandle *context, const uint64_t *partials,
                                               uint32_t count, int32_t *index, void *stream);

/* int8 MFMA batch GEMM of a HyperVSQ-2 or Q4_0 tensor, 1..16 tokens per
 * call (the ABI's GEMM uses it by itself from 2 HyperVSQ-2 / 3 Q4_0
 * tokens on the MFMA-order copy, from 3 / 6 without it): HyperVSQ-2 blocks are exact int8 dot products with the octant
 * multipliers folded into the weights (v_mfma_i32_16x16x64_i8), Q4_0 blocks
 * one v_mfma_i32_16x16x32_i8 each on the signed codes n - 8, on tiles of 16
 * rows x 16 tokens.  The activations are read from an "MFMA image" of the
 * int8 tokens (qwn_hip_ext_mfma_image_bytes() bytes, 16-byte aligned;
 * 0 for F16 tensors), built by qwn_hip_ext_mfma_image_device from q8
 * [batch][q8_stride].  output [batch][output_stride] = W x_t * scales[t]. */
QWN_CUDA_ABI_API uint64_t qwn_hip_ext_mfma_image_bytes(const QwnCudaTensorHandle *tensor);
QWN_CUDA_ABI_API int qwn_hip_ext_mfma_image_device(QwnCudaContextHandle *context,
                                                   const QwnCudaTensorHandle *tensor, const int8_t *q8,
                                                   uint32_t batch, uint32_t q8_stride, void *image,
                                                   void *stream);
QWN_CUDA_ABI_API int qwn_hip_ext_gemm_mfma_device(QwnCudaContextHandle *context,
                                                  const QwnCudaTensorHandle *tensor, const void *image,
                                                  const float *scales, float *output, uint32_t batch,
                                                  uint32_t output_stride, void *stream);
/* The same GEMM over `count` (1..4) tensors of one kind with the same
 * column count that share one MFMA image (q/k/v, gate/up), in one launch:
 * outputs[i] [batch][output_stride or the tensor's rows]; accumulate != 0
 * adds the product to the outputs (a residual stream) instead. */
QWN_CUDA_ABI_API int qwn_hip_ext_gemm_mfma_group_device(QwnCudaContextHandle *context,
                                                        const QwnCudaTensorHandle *tensors, uint32_t count,
                                                        const void *image, const float *scales,
                                                        float *const *outputs, uint32_t batch,
                                                        uint32_t output_stride, uint32_t accumulate,
                                                        void *stream);

/* Upload `count` tensors, each as qwn_cuda_abi_upload_tensor
 * (c/cuda/qwn_cuda_abi.h:244-246), through one pipeline: whole-row chunks
 * of each host buffer (an mmap'd .qwn payload, say) are copied into one of
 * two pinned staging slots while the other slot's DMA and repack run; the
 * call synchronises once for the batch.  out[i] receives tensor i's handle;
 * on failure nothing of the batch stays resident.  (No counterpart in the
 * reference: its host uploads tensor by tensor, c/qwanto_decode.c:790-830.) */
QWN_CUDA_ABI_API int qwn_hip_ext_upload_batch(QwnCudaContextHandle *context,
                                              const QwnCudaTensorUpload *uploads, uint32_t count,
                                              QwnCudaTensorHandle *out);

/* Tensor placement with a GPU tier, as the reference's qwn_plan_residency
 * (c/qwanto_native.c:379-435, replaced here): tensors in the order of their
 * name's priority (embedding / LM head 255, norms 245, attention 230, dense
 * gate 210, other 160, experts 80), then smaller first, then index; each
 * goes to the GPU while the GPU budget has room, else to RAM while the RAM
 * budget has room, else stays file-backed.  items[count] receive the plan
 * in that order (the reference's QwnPlacement layout), totals[3] the GPU,
 * RAM and file bytes.  gpu_budget QWN_HIP_GPU_BUDGET_AUTO: 90% of the free
 * memory of the context's device (context required), as the reference host
 * sizes its GPU tier (c/qwanto_decode.c:202-216); otherwise context may be
 * NULL. */
#define QWN_HIP_TIER_GPU 0u
#define QWN_HIP_TIER_RAM 1u
#define QWN_HIP_TIER_FILE 2u
#define QWN_HIP_GPU_BUDGET_AUTO UINT64_MAX
typedef struct {
    uint64_t name_hash;       /* FNV-1a 64 of the name (the .qwn index hash) */
    uint64_t byte_offset;
    uint64_t byte_size;
    uint32_t tensor_index;
    uint8_t tier;             /* QWN_HIP_TIER_* */
    uint8_t priority;
    uint16_t reserved;
} QwnHipPlacement;
QWN_CUDA_ABI_API int qwn_hip_ext_plan_residency(QwnCudaContextHandle *context, const char *const *names,
                                                const uint64_t *byte_offsets, const uint64_t *byte_sizes,
                                                uint32_t count, uint64_t gpu_budget, uint64_t ram_budget,
                                                QwnHipPlacement *items, uint64_t *totals);

/* Per-token int8 quantization on the device without an image:
 * x fp32 [batch][x_stride] -> q8 [batch][q8_stride] (zero padded past
 * cols), scales [batch]. */
QWN_CUDA_ABI_API int qwn_hip_ext_quantize_device(QwnCudaContextHandle *context,
                                                 const float *x, uint32_t batch,
                                                 uint32_t cols, uint32_t x_stride,
                                                 int8_t *q8, uint32_t q8_stride,
                                                 float *scales, void *stream);

/* Append `count` tokens of fp32 K and V ([count][n_channels], device) at
 * position cache.tokens; synchronous bookkeeping, asynchronous kernels. */
QWN_CUDA_ABI_API int qwn_hip_ext_kv_append_device(QwnCudaContextHandle *context,
                                                  QwnCudaKvCacheHandle *cache,
                                                  const float *keys,
                                                  const float *values,
                                                  uint32_t count, void *stream);

/* Attention over tokens [0, position] with a device query and output
 * ([query_heads][head_dim] fp32).  `workspace` is a device buffer of at
 * least qwn_hip_ext_attention_workspace_bytes() bytes. */
QWN_CUDA_ABI_API uint64_t qwn_hip_ext_attention_workspace_bytes(
    QwnCudaKvCacheHandle *cache, uint32_t query_heads, uint32_t position);
QWN_CUDA_ABI_API int qwn_hip_ext_kv_attention_device(QwnCudaContextHandle *context,
                                                     QwnCudaKvCacheHandle *cache,
                                                     const float *query, float *output,
                                                     uint32_t query_heads,
                                                     uint32_t position, float scale,
                                                     void *workspace, void *stream);

/* The same attention with no workspace argument and no allocation: the
 * split partials live in a file-scope device array of 4 MiB per GPU (its
 * address looked up once per device at context creation).  No counterpart
 * in the reference; for callers that cannot allocate (code under HIP graph
 * capture, serving loops that forbid hipMalloc).  A request whose partials
 * exceed the array (qwn_hip_ext_attention_workspace_bytes() > 4 MiB) is
 * refused with QWN_CUDA_STATUS_INVALID_ARGUMENT.  Every call on one GPU
 * shares that GPU's array, so calls must not run at the same time on one
 * GPU: a call is refused with QWN_CUDA_STATUS_UNAVAILABLE while the
 * previous call on that GPU, enqueued on a different stream (another
 * stream of the caller, another context's stream), has not finished.
 * Calls on one stream are ordered and always accepted.  Calls recorded
 * into a HIP graph are not tracked: a graph that replays them on two
 * streams at once races. */
QWN_CUDA_ABI_API int qwn_hip_ext_kv_attention_device_noalloc(QwnCudaContextHandle *context,
                                                             QwnCudaKvCacheHandle *cache,
                                                             const float *query, float *output,
                                                             uint32_t query_heads, uint32_t position,
                                                             float scale, void *stream);

/* ---- operators of a batched serving step --------------------------------
 * What lies between the projections when many sequences are decoded at once:
 * the residual's addition with RMSNorm and the projections' int8 input, the
 * paged 4-bit KV cache, and the logits' penalties and masks.  Each takes a
 * request struct of device pointers that a caller builds once and passes
 * every step; strides are in elements (0: rows back to back), and no pointer
 * needs more alignment than its element.  A request's outputs may not overlap
 * its inputs, the workspace or each other except where it says so: such a request
 * is refused (columns of one wider buffer do not overlap).  Sizes that only the device
 * knows (a batch's row starts, cached lengths, page numbers, token ids) are read
 * there, so a captured step replays with new ones; each is checked there, and
 * what points outside the buffers that the host described is left out.  No
 * counterpart in the reference. */
#define QWN_HIP_DTYPE_F32 0u
#define QWN_HIP_DTYPE_F16 1u
#define QWN_HIP_DTYPE_BF16 2u

/* h = x + residual (rounded to dtype; residual NULL: h = x)
 * y = h * norm / sqrt(mean(h^2) + eps), rounded once to fp32 from 64 bits
 * scales[t] = amax / 127 (1 where amax is 0), q8 = rint(y / scale): the
 * per-token quantization of qwn_hip_ext_quantize_device on y, bit for bit.
 * A token whose y are not all finite has the scale NaN and zeros in q8. */
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t tokens;
    uint32_t cols;
    uint32_t dtype;                /* of x, residual, residual_out and y */
    uint32_t x_stride;
    uint32_t residual_stride;
    uint32_t residual_out_stride;
    uint32_t y_stride;
    uint32_t q8_stride;            /* q8 is zero from cols to here */
    float eps;
    uint32_t reserved;
    const void *x;                 /* [tokens][x_stride] */
    const void *residual;          /* NULL, or [tokens][residual_stride] */
    void *residual_out;            /* NULL, or h [tokens][residual_out_stride]; may be x or residual
                                      with that one's stride */
    const float *norm;             /* [cols] */
    void *y;                       /* NULL, or [tokens][y_stride] */
    int8_t *q8;                    /* NULL, or [tokens][q8_stride] (then scales too) */
    float *scales;                 /* [tokens] */
} QwnHipNormRequest;
QWN_CUDA_ABI_API int qwn_hip_ext_norm_quantize_device(QwnCudaContextHandle *context,
                                                      const QwnHipNormRequest *request, void *stream);

/* A paged KV cache held in 4 bits: `pages` pages of page_tokens tokens (a
 * power of two from 16 to 1024), handed to sequences by the caller through a
 * page table.  A token's K or V of one head (head_dim up to 256) is held per
 * group of 64 channels as an f16 minimum, an f16 step = (max - min) / 15 and
 * codes rint((x - minimum) / step) in 0 .. 15; it stands for minimum + step *
 * code.  Values that are not finite are held as zero, finite ones clamped to
 * the range of f16.  rope_dims (even, 0: none) channels of every key, as
 * pairs (i, i + rope_dims / 2), are rotated by position * rope_theta^(-2 i /
 * rope_dims) on the way in, in 64 bits.  Charged to the context's budget; one
 * cache per layer. */
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t pages;
    uint32_t page_tokens;
    uint32_t kv_heads;
    uint32_t head_dim;
    uint32_t rope_dims;
    float rope_theta;
} QwnHipPagedKvOptions;
typedef struct {
    QwnCudaAbiHeader header;
    void *opaque;
} QwnHipPagedKvHandle;
QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_create(QwnCudaContextHandle *context, const QwnHipPagedKvOptions *options,
                                                 QwnHipPagedKvHandle *out);
/* Waits for the device: no call of any stream may still use the cache. */
QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_destroy(QwnCudaContextHandle *context, QwnHipPagedKvHandle *cache);

/* A ragged batch.  Sequence s brings the rows starts[s] .. starts[s + 1] - 1
 * of the step's tensors (none, one, or many), its tokens past[s], past[s] + 1,
 * ...; slot t of it lies in page page_table[s][t / page_tokens].  Rows behind
 * starts[sequences] belong to no sequence: they are not read, and outputs keep
 * what they held there.  A sequence whose past is negative or whose rows do
 * not lie in 0 .. tokens is left out; slots whose page is not one of the
 * cache's (or lies past table_stride) are not stored, and not attended to. */
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t sequences;
    uint32_t tokens;               /* rows of the step's tensors */
    uint32_t table_stride;         /* pages of a row of the table */
    uint32_t reserved;
    const int32_t *starts;         /* device [sequences + 1], ascending */
    const int32_t *past;           /* device [sequences]: tokens before this step's */
    const int32_t *page_table;     /* device [sequences][table_stride] */
} QwnHipPagedBatch;

/* Stores the batch's keys (rotated) and values at their slots, and, if query
 * is given, writes the rotated queries.  A position is the token's slot, or
 * positions[row].  Sequences may share pages (a common prefix), but a slot may
 * be named once in a call. */
typedef struct {
    QwnCudaAbiHeader header;
    const QwnHipPagedBatch *batch;
    uint32_t dtype;                /* of key, value, query and query_out */
    uint32_t query_heads;
    uint32_t key_stride;
    uint32_t value_stride;
    uint32_t query_stride;
    uint32_t query_out_stride;
    const void *key;               /* [tokens][key_stride]: [kv_heads][head_dim] */
    const void *value;             /* [tokens][value_stride] */
    const void *query;             /* NULL, or [tokens][query_stride]: [query_heads][head_dim] */
    void *query_out;               /* [tokens][query_out_stride]; may be query with its stride */
    const int32_t *positions;      /* NULL, or [tokens] */
} QwnHipPagedAppendRequest;
QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_append_device(QwnCudaContextHandle *context, QwnHipPagedKvHandle *cache,
                                                        const QwnHipPagedAppendRequest *request, void *stream);

/* The values that the batch's tokens (its rows, as the append stored them)
 * stand for, fp32 [tokens][stride] of keys and values (either may be NULL). */
QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_read_device(QwnCudaContextHandle *context, QwnHipPagedKvHandle *cache,
                                                      const QwnHipPagedBatch *batch, float *keys, float *values,
                                                      uint32_t stride, void *stream);

/* Causal attention of the batch's rows over the cache, the batch's own tokens
 * appended before: token past[s] + i of sequence s attends to its slots 0 ..
 * past[s] + i, query head h to KV head h / (query_heads / kv_heads).  A row
 * that attends to nothing is zeros; a row whose query (or the scale) is not
 * finite is NaN.  Scores may be of any size, past fp32's too.
 * fp32 queries are computed to fp32 (22 bits of query and probability in the
 * matrix products), f16 and bf16 ones with f16 probabilities, and bf16 batches
 * of many rows (80 of a KV head a sequence and more on average) with the keys and
 * values rounded to f16.  The kernels are chosen by `tokens`, `sequences` and
 * table_stride: prompts go best in a call apart from single tokens.  The output may not be the query.
 * The workspace (qwn_hip_ext_paged_kv_attention_workspace_bytes, the same for
 * every batch of a cache; 0 for a request that is refused; 16-byte aligned)
 * holds nothing between calls, and may not be shared by calls that run at the
 * same time. */
typedef struct {
    QwnCudaAbiHeader header;
    const QwnHipPagedBatch *batch;
    uint32_t dtype;                /* of query and output */
    uint32_t query_heads;          /* a multiple of the cache's kv_heads */
    uint32_t query_stride;
    uint32_t output_stride;
    const void *query;             /* [tokens][query_stride]: [query_heads][head_dim] */
    void *output;                  /* [tokens][output_stride] */
    void *workspace;
    float scale;
    uint32_t reserved;
} QwnHipPagedAttentionRequest;
QWN_CUDA_ABI_API uint64_t qwn_hip_ext_paged_kv_attention_workspace_bytes(QwnCudaContextHandle *context,
                                                                         QwnHipPagedKvHandle *cache,
                                                                         const QwnHipPagedAttentionRequest *request);
QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_attention_device(QwnCudaContextHandle *context, QwnHipPagedKvHandle *cache,
                                                           const QwnHipPagedAttentionRequest *request, void *stream);

/* The logits of a batch before the greedy choice (or a caller's sampler):
 * tokens of the row's history: l > 0 ? l / repetition : l * repetition, and
 * for those it holds `count` > 0 times behind its first prompt_counts[row]
 * entries l -= frequency * count + presence; l += the sum of the token's
 * biases (a token may come several times); l = -inf where the token's bit of
 * the row's mask is 0.  In 64 bits, rounded to fp32 and then to dtype.  ids: the first
 * index of the largest value, -1 for a row that nothing is left of (every
 * value -inf or NaN).  Tokens outside 0 .. vocab - 1 in a list are padding.
 * A row's part of a list is list[starts[row]] .. list[starts[row + 1] - 1],
 * none if that does not lie in the list's capacity.  Row r reads mask row
 * mask_index[r] (none if that is not one), or r where mask_index is NULL. */
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t rows;                 /* up to 65535 */
    uint32_t vocab;
    uint32_t dtype;                /* of logits and out */
    uint32_t in_stride;
    uint32_t out_stride;
    uint32_t history_capacity;     /* entries of history, under 2^29 */
    uint32_t bias_capacity;        /* entries of bias_tokens and bias_values */
    uint32_t mask_rows;
    uint32_t mask_stride;          /* words of a mask row */
    uint32_t reserved;
    const void *logits;            /* [rows][in_stride] */
    void *out;                     /* [rows][out_stride]; may be logits with its stride */
    const int32_t *history;        /* NULL, or token ids, every row's prompt and what it generated */
    const int32_t *history_starts; /* [rows + 1] */
    const int32_t *prompt_counts;  /* NULL (none), or [rows] */
    const float *repetition;       /* NULL (1), or [rows] */
    const float *presence;         /* NULL (0), or [rows] */
    const float *frequency;        /* NULL (0), or [rows] */
    const int32_t *bias_tokens;    /* NULL, or token ids */
    const float *bias_values;
    const int32_t *bias_starts;    /* [rows + 1] */
    const uint32_t *mask;          /* NULL, or [mask_rows][mask_stride]: bit t % 32 of word t / 32 */
    const int32_t *mask_index;     /* NULL, or [rows] */
    int32_t *ids;                  /* NULL, or [rows] */
    void *workspace;               /* for ids: qwn_hip_ext_logits_workspace_bytes(), 8-byte aligned */
} QwnHipLogitsRequest;
QWN_CUDA_ABI_API uint64_t qwn_hip_ext_logits_workspace_bytes(uint32_t rows, uint32_t vocab);
QWN_CUDA_ABI_API int qwn_hip_ext_logits_process_device(QwnCudaContextHandle *context,
                                                       const QwnHipLogitsRequest *request, void *stream);

/* ---- operators of packed prompts and of beams ------------------------------
 * Requests and their rules are those of a batched serving step (above). */

/* Queries and keys of a step's tokens: each head normed where weights are given,
 *   y = x * norm / sqrt(mean(x^2) + eps)
 * then its first rope_dims (even, 0: none) channels rotated as pairs (i, i +
 * rope_dims / 2) by positions[axis][token] * rope_theta^(-2 i / rope_dims).  Of
 * the pairs, sections[0] belong to axis 0, sections[1] to axis 1, ... (they add
 * up to rope_dims / 2): one section after the other, or, with in_turn not 0,
 * dealt to the axes in turn, past those that have all of theirs.  Axes 0, 1 and 2
 * may be time, height and width; text has the same position in all.  Angles are
 * computed in 64 bits; fp32 rows are, too, and rounded once, 16-bit ones in fp32 (norms
 * of heads whose mean square is no number of fp32 in 64 bits).
 * An output may be its input with that one's stride. */
#define QWN_HIP_ROTARY_AXES 4u
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t tokens;
    uint32_t dtype;
    uint32_t query_heads;          /* 0: no queries */
    uint32_t key_heads;            /* 0: no keys */
    uint32_t head_dim;             /* up to 256 */
    uint32_t rope_dims;
    uint32_t sections[4];
    uint32_t in_turn;
    uint32_t query_stride;
    uint32_t key_stride;
    uint32_t query_out_stride;
    uint32_t key_out_stride;
    uint32_t position_stride;      /* 0: tokens */
    float rope_theta;
    float eps;
    const void *query;             /* [tokens][query_stride]: [query_heads][head_dim] */
    const void *key;               /* [tokens][key_stride]: [key_heads][head_dim] */
    void *query_out;
    void *key_out;
    const float *query_norm;       /* NULL, or [head_dim] */
    const float *key_norm;
    const int32_t *positions;      /* [axis][position_stride], axes up to the last that has a section */
} QwnHipRotaryRequest;
QWN_CUDA_ABI_API int qwn_hip_ext_rotary_device(QwnCudaContextHandle *context, const QwnHipRotaryRequest *request, void *stream);

/* Causal attention of packed sequences over their own keys and values: row
 * starts[s] + i of sequence s attends to the rows starts[s] .. starts[s] + i,
 * query head h to KV head h / (query_heads / kv_heads).  Rows behind
 * starts[sequences] belong to no sequence: they are not read, and the output
 * keeps what it held there; a sequence whose rows do not lie in 0 .. tokens is
 * left out.  Scores and sums are fp32, probabilities are rounded to dtype (f16: below 2^-20 of
 * the row's largest to steps of 2^-30 of that); fp32 is fp32 throughout.  Finite queries, keys and scale have their softmax whatever the
 * scores' size, past fp32's too (of fp32 and bf16, a channel counts as zero where the
 * key times the query, taken as its share of its row's largest, is below 2^-116).  A key or query
 * with an infinity: a score of -inf has probability 0, a row with one that is +inf or
 * NaN, and a row with a scale that is not finite, is NaN.  A value that is not finite
 * makes its channel so in the rows that attend to it, and in no other; of finite values, up to
 * the type's largest, the average is finite.  For single
 * tokens behind a cache:
 * qwn_hip_ext_paged_kv_attention_device. */
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t sequences;
    uint32_t tokens;               /* rows of the tensors */
    uint32_t dtype;
    uint32_t query_heads;          /* a multiple of kv_heads */
    uint32_t kv_heads;
    uint32_t head_dim;             /* up to 256 */
    uint32_t query_stride;
    uint32_t key_stride;
    uint32_t value_stride;
    uint32_t output_stride;
    float scale;
    uint32_t reserved;
    const int32_t *starts;         /* device [sequences + 1], ascending */
    const void *query;             /* [tokens][query_stride]: [query_heads][head_dim] */
    const void *key;               /* [tokens][key_stride]: [kv_heads][head_dim] */
    const void *value;             /* [tokens][value_stride] */
    void *output;                  /* [tokens][output_stride] */
} QwnHipPromptAttentionRequest;
QWN_CUDA_ABI_API int qwn_hip_ext_prompt_attention_device(QwnCudaContextHandle *context,
                                                         const QwnHipPromptAttentionRequest *request, void *stream);

/* The best continuations of each sequence's beams.  Row s * beams + b of the
 * logits is beam b of sequence s, whose log probabilities so far add up to
 * scores[s][b]; token t continues it to
 *   scores[s][b] + logits[t] - log(sum of exp(logits))
 * Of a sequence's beams and tokens the `count` largest, in order (ties: the lower
 * beam, then the lower token), as value, row and token: -inf, -1, -1 past the
 * last.  next_*: of those the first `beams` whose token is none of end_tokens, the
 * same way.  No candidates come from a beam whose score is not finite, from
 * logits that are -inf or NaN (they do not count in the sum), or from a row with a
 * logit of +inf.  A row's sum is one of fp32 powers; values are added up in 64 bits,
 * ordered there (a beam's that are one number there, by their logits), and rounded to fp32.
 * The workspace (qwn_hip_ext_beam_select_workspace_bytes, 0 for sizes that are
 * refused; 16-byte aligned) holds nothing between calls, and may not be shared by
 * calls that run at the same time. */
#define QWN_HIP_BEAM_MAX_BEAMS 32u
#define QWN_HIP_BEAM_MAX_COUNT 64u
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t sequences;
    uint32_t beams;                /* 1..32 */
    uint32_t vocab;
    uint32_t count;                /* candidates of a sequence, 1..64 */
    uint32_t dtype;                /* of logits */
    uint32_t in_stride;
    uint32_t end_count;            /* of end_tokens, up to 4 */
    int32_t end_tokens[4];
    uint32_t reserved;
    const void *logits;            /* [sequences * beams][in_stride] */
    const float *scores;           /* [sequences][beams] */
    float *values;                 /* [sequences][count] */
    int32_t *parents;              /* [sequences][count]: rows of the logits */
    int32_t *tokens;               /* [sequences][count] */
    float *next_scores;            /* NULL (then all three), or [sequences][beams]; may be scores */
    int32_t *next_parents;
    int32_t *next_tokens;
    void *workspace;
} QwnHipBeamSelectRequest;
QWN_CUDA_ABI_API uint64_t qwn_hip_ext_beam_select_workspace_bytes(uint32_t sequences, uint32_t beams, uint32_t vocab,
                                                                  uint32_t count);
QWN_CUDA_ABI_API int qwn_hip_ext_beam_select_device(QwnCudaContextHandle *context, const QwnHipBeamSelectRequest *request,
                                                    void *stream);

/* What the beams keep follows them: row r (of sequence r / beams) goes on from
 * row parents[r] of its sequence, with that one's length past[p] + added, its
 * history, to which tokens[r] comes as entry past[p] + added, and its pages.  Pages
 * that are full are shared; the one in use goes on with the first row that has
 * this parent, and each further one takes the page `spare` that it holds, to
 * which the slots are copied in every cache given, and in exchange the page in
 * use of a row that nothing goes on from becomes its spare, as long as there are such
 * rows (a row of a negative length leaves no page).  Where the page in
 * use has just become full, the row takes its spare as the next one, and has
 * none (-1) until the caller hands it another, or gets a page in use that no
 * copy has taken, which only a row of another length leaves; where its table ends there, the spare
 * stays what it is.  So a row owns two pages, one in
 * use and one spare, no row's table names another's, and none in use is lost that a row has
 * room for; the caller takes back full pages that no table names any more.  Table entries past the page in use are
 * -1.  A row whose parent is none of its sequence (-1) goes on from itself, with no
 * token; one whose parent's length is negative, too (its own negative: nothing of
 * it changes).  Pages that are not the caches' are not copied to or from.  Tables and histories may be in
 * place, lengths and spares may not. */
#define QWN_HIP_BEAM_MAX_CACHES 256u
typedef struct {
    QwnCudaAbiHeader header;
    uint32_t sequences;
    uint32_t beams;                /* 1..32 */
    uint32_t page_tokens;          /* of the caches */
    uint32_t table_stride;         /* pages of a row of the tables */
    uint32_t added;                /* tokens the step brought to each row */
    uint32_t history_length;       /* entries of a row's history */
    const int32_t *parents;        /* [rows] */
    const int32_t *past;           /* [rows] */
    int32_t *past_out;             /* [rows] */
    const int32_t *page_table;     /* [rows][table_stride] */
    int32_t *page_table_out;       /* may be page_table */
    const int32_t *spare;          /* [rows] */
    int32_t *spare_out;            /* [rows] */
    const int32_t *tokens;         /* NULL, or [rows] */
    const int32_t *history;        /* NULL, or [rows][history_length] */
    int32_t *history_out;          /* may be history */
} QwnHipBeamAdvanceRequest;
/* `caches`: count handles of one shape (up to 256; 0: no pages are copied). */
QWN_CUDA_ABI_API int qwn_hip_ext_paged_kv_beam_advance_device(QwnCudaContextHandle *context, const QwnHipPagedKvHandle *caches,
                                                              uint32_t count, const QwnHipBeamAdvanceRequest *request,
                                                              void *stream);

/* Debug: the integer sums of the GEMV for one token, computed by the same
 * device code as the GEMV (host pointers, synchronous).  HyperVSQ-2:
 * out[row][block*8 + octant] = sum (code-1)*a; Q4_0: out[row][block] =
 * sum (nibble-8)*a.  out_capacity counts int32 elements. */
QWN_CUDA_ABI_API int qwn_hip_ext_debug_int_sums(QwnCudaContextHandle *context,
                                                const QwnCudaTensorHandle *tensor,
                                                const int8_t *host_q8,
                                                int32_t *host_out,
                                                uint64_t out_capacity);

/* Debug: the exact int32 block dot products of the int8 MFMA GEMM
 * (qwn_hip_ext_gemm_mfma_device's kernel, the same plan and operand code)
 * for batch (1..16) int8 tokens host_q8 [batch][cols] (host pointers,
 * synchronous).  out[token][row][block]: HyperVSQ-2 per 256-weight block
 * sum over octants of multiplier * sum (code-1)*a; Q4_0 per 32-weight block
 * sum (nibble-8)*a.  out_capacity counts int32 elements. */
QWN_CUDA_ABI_API int qwn_hip_ext_debug_mfma_int_sums(QwnCudaContextHandle *context,
                                                     const QwnCudaTensorHandle *tensor,
                                                     const int8_t *host_q8, uint32_t batch,
                                                     int32_t *host_out, uint64_t out_capacity);

/* Debug: cached tokens [first, first + count) of a Q8 KV cache in the CPU
 * cache's token-major layout (c/qwanto_turboquant.h:78-94): keys/values
 * [count][kv_heads*head_dim] int8, scales [count][ceil(channels/64)] fp32
 * (host pointers, synchronous). */
QWN_CUDA_ABI_API int qwn_hip_ext_debug_kv_read(QwnCudaContextHandle *context,
                                               const QwnCudaKvCacheHandle *cache, uint32_t first,
                                               uint32_t count, int8_t *host_keys, int8_t *host_values,
                                               float *host_key_scales, float *host_value_scales);

#ifdef __cplusplus
}
#endif

#endif /* QWN_HIP_EXT_H */
