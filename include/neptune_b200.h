/*
 * neptune_b200.h -- C ABI of the B200 (sm_100a) backend for neptune-opt's fused
 * dependent-reduction hot path.
 *
 * Every entry point takes plain device pointers, element counts and element strides,
 * launches on the caller's CUDA stream and returns 0 (NB200_OK) or a negative
 * nb200_status. No C++ exception crosses this boundary. Inputs are never written.
 * Outputs and scratch are allocated by the caller; the library allocates no device
 * memory. nb200_last_error() returns a message for the last failing call on the
 * calling host thread.
 *
 * The entry points mirror the kernel launch signatures of the reference backend
 * (Defyli/neptune-opt, package neptune_codegen); each declaration names the launch it
 * replaces as file:line within that project.
 */
#ifndef NEPTUNE_B200_H
#define NEPTUNE_B200_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ status / types */
typedef enum {
    NB200_OK = 0,
    NB200_ERR_ARG = -1,         /* bad pointer, size, stride, dtype or parameter       */
    NB200_ERR_CAPACITY = -2,    /* request exceeds a documented capacity               */
    NB200_ERR_LAUNCH = -3,      /* the CUDA launch itself failed                       */
    NB200_ERR_TIMEOUT = -4,     /* a bounded device wait ran out                       */
    NB200_ERR_UNSUPPORTED = -5  /* valid request this build does not implement         */
} nb200_status;

/* Element types of row data (the reference accepts exactly these three:
 * neptune_codegen/template.py:346). */
typedef enum { NB200_F32 = 0, NB200_BF16 = 1, NB200_F16 = 2 } nb200_dtype;

/* Index types of segment descriptors (neptune_codegen/torch_op.py:358). */
typedef enum { NB200_I32 = 0, NB200_I64 = 1 } nb200_index_dtype;

/* The eleven scalar skeletons of neptune_codegen/library.py:19-177, compiled in. */
typedef enum {
    NB200_LOGSUMEXP = 0,    /* m + log(sum exp(x - m) + tiny)           library.py:19  */
    NB200_LSE_BIASED = 1,   /* logsumexp(x + alpha)                     library.py:100 */
    NB200_LSE_SCALED = 2,   /* logsumexp(x / T)                         library.py:157 */
    NB200_SOFTCAP_LSE = 3,  /* logsumexp(tanh(beta x))                  library.py:59  */
    NB200_STABLE_L2 = 4,    /* m sqrt(sum (x/m)^2), m = max|x|          library.py:32  */
    NB200_LINEAR_ATTN = 5,  /* sum x / max|x|                           library.py:40  */
    NB200_DECAY_RENORM = 6, /* sum x / (N + max|x|)                     library.py:49  */
    NB200_SUMSQ_DIV = 7,    /* sum x^2 / max|x|                         library.py:92  */
    NB200_RMSNORM_MAX = 8,  /* max x / sqrt(mean x^2 + eps)             library.py:72  */
    NB200_VARIANCE = 9,     /* two-pass mean((x - mean)^2)              library.py:114 */
    NB200_STD = 10,         /* two-pass sqrt(variance)                  library.py:143 */
    NB200_NUM_SKELETONS = 11
} nb200_skeleton;

/* Scalar parameters of a skeleton. Only the fields the skeleton declares are read
 * (library.py: tiny, alpha, T, beta, N, eps). Values arrive as binary64 exactly as the
 * reference bakes them into its source (emitters.py:300-327) and are narrowed to fp32
 * where the kernel computes. */
typedef struct {
    double tiny;
    double alpha;
    double T;
    double beta;
    double N;
    double eps;
} nb200_params;

/* Launch policy chosen by the host (neptune_codegen/autotune.py:222-250 picks Triton
 * (BLOCK, num_warps); here it picks a CUDA variant). Pass NULL for the library default. */
typedef enum {
    NB200_VARIANT_AUTO = 0,
    NB200_VARIANT_WARP_ROW = 1, /* one warp folds one row, register-resident chunks     */
    NB200_VARIANT_CTA_ROW = 2,  /* one CTA folds one row                                 */
    NB200_VARIANT_STREAM = 3,   /* bulk-copy staged rows (contiguous, 16-byte aligned)   */
    NB200_VARIANT_CLUSTER = 4   /* one thread-block cluster per row, CTA states merged   */
                                /* through distributed shared memory (contiguous,        */
                                /* 16-byte aligned rows; folds and RMSNorm)              */
} nb200_variant;

typedef struct {
    int32_t variant;        /* nb200_variant                                          */
    int32_t threads;        /* CTA size (64..512, x32); for NB200_VARIANT_STREAM the   */
                            /* number of warps, each owning its own ring of stages    */
    int32_t ctas_per_sm;    /* persistent grid = SMs * ctas_per_sm (0: default)       */
    int32_t stages;         /* NB200_VARIANT_STREAM: stages per warp ring (0: fit);   */
                            /* NB200_VARIANT_CLUSTER: CTAs per row, 2..16 (0: chosen) */
} nb200_launch;

/* One partial state of the repaired fold (emitters.py:436-519): raw producer value,
 * fp32 accumulator, "seen" flag and nonfinite status bits (bit 0 NaN, bit 1 +inf). */
typedef struct {
    float m;
    float acc;
    int32_t seen;
    int32_t status;
} nb200_state;

/* ------------------------------------------------------------------ library info */
const char* nb200_last_error(void);
const char* nb200_version(void);
/* Number of nb200 kernel launches issued by this process (for launch accounting). */
uint64_t nb200_launch_count(void);
/* Reads and clears the fault bits of the kernels with device-side waits or checks (bit 0: a bounded wait
 * on a bulk copy ran out; a streaming kernel stopped early, the gated norm's backward wrote the rows it
 * could not read, and its sums over rows, as NaN; bit 1: a bounded wait in an attention kernel, forward or
 * backward, ran out and its output was left unwritten, or (behind a shared prefix) written as NaN; bit 2: the peer merge's bounded wait for the ranks'
 * states ran out, those rows written as NaN; bit 3: a peer push or merge found a buffer whose recorded
 * layout differs from the call's, nothing stored or read).
 * Synchronous. No counterpart in the reference, whose Triton kernels have no device-side waits. */
int nb200_stream_fault(uint32_t* bits);

/* ------------------------------------------------------------------ a1: serial fold
 * Row-last repaired fold of one skeleton over a strided 2-D view x[rows, ncols]
 * (element strides stride_row, stride_col; any sign-free layout torch can express).
 * out[rows] is contiguous, in the input dtype. Replaces the serial launch
 * `kernel[(rows,)](x, out, rows, ncols, stride_row, stride_col, BLOCK=...)` of
 * neptune_codegen/template.py:376-378 (kernel body template.py:41-54 and the
 * two-pass body template.py:62-103). */
int nb200_fold(int skeleton, const nb200_params* params,
               const void* x, int dtype, int64_t rows, int64_t ncols,
               int64_t stride_row, int64_t stride_col,
               void* out, const nb200_launch* launch, void* stream);

/* Softmax-family readout fused into the log fold (the lowering of
 * neptune_recognize/lowering.py:80-99): mode 0 softmax exp(x - m) / s, mode 1
 * log_softmax (x - m) - log(s) with the reference's row-wide NaN for +inf rows.
 * y[rows, ncols] is contiguous in the input dtype; lse (nullable) receives the
 * logsumexp per row in the input dtype. */
int nb200_softmax(int mode, const void* x, int dtype, int64_t rows, int64_t ncols,
                  int64_t stride_row, int64_t stride_col,
                  void* y, void* lse, const nb200_launch* launch, void* stream);

/* Row L2 normalisation built on the stable_l2 fold (library.py:32-38): norm[rows]
 * (nullable) = m * sqrt(sum (x/m)^2) and y = x / norm, both in the input dtype. */
int nb200_l2_normalize(const void* x, int dtype, int64_t rows, int64_t ncols,
                       int64_t stride_row, int64_t stride_col,
                       void* y, void* norm, const nb200_launch* launch, void* stream);

/* ------------------------------------------------------------------ a2: split plan
 * Explicit split of each row into nparts column chunks of chunk_cols columns
 * (neptune_codegen/template.py:114-125, :137-165, launch :380-390). Chunk states go to
 * caller-owned scratch of nb200_fold_split_scratch_bytes(rows, nparts) bytes and are
 * merged in ascending chunk order. nparts = ceil(ncols / chunk_cols) <= 4096. */
int64_t nb200_fold_split_scratch_bytes(int64_t rows, int64_t nparts);
int nb200_fold_split(int skeleton, const nb200_params* params,
                     const void* x, int dtype, int64_t rows, int64_t ncols,
                     int64_t stride_row, int64_t stride_col, int64_t chunk_cols,
                     void* scratch, int64_t scratch_bytes, void* out,
                     const nb200_launch* launch, void* stream);

/* The split plan for callers that cannot allocate device memory (a host that hands over only its
 * input and output buffers, a fixed device-memory budget, a path where an allocation would
 * synchronise). Same arguments and result as nb200_fold_split minus the scratch: the chunk states
 * live in a 4 MiB array built into the library, which every GPU that loads the library holds until
 * exit. Limit: rows * ceil(ncols / chunk_cols) <= NB200_NOALLOC_MAX_STATES, else NB200_ERR_CAPACITY.
 * The first call on a device resolves the array's device address (make it before any stream
 * capture). Calls share the array: calls that overlap on the GPU race. Allocates nothing.
 * No counterpart in the reference, whose split plan always allocates its scratch with torch. */
#define NB200_NOALLOC_MAX_STATES 262144
int nb200_fold_split_noalloc(int skeleton, const nb200_params* params,
                             const void* x, int dtype, int64_t rows, int64_t ncols,
                             int64_t stride_row, int64_t stride_col, int64_t chunk_cols,
                             void* out, void* stream);

/* The two halves of the split plan, for callers that move states between devices.
 * nb200_fold_partial folds columns [col_begin, col_begin + ncols_shard) of every row in
 * chunk_cols chunks into states[rows * nparts] (nparts = ceil(ncols_shard / chunk_cols)).
 * nb200_fold_merge merges states laid out [rows][nparts] with element stride part_stride
 * between consecutive parts of a row and row_stride between rows, in ascending part
 * order, and finalises into out[rows] (input dtype). ncols_total is the full row width
 * (read by skeletons whose algebra uses N = ncols). */
int nb200_fold_partial(int skeleton, const nb200_params* params,
                       const void* x, int dtype, int64_t rows, int64_t ncols_total,
                       int64_t col_begin, int64_t ncols_shard,
                       int64_t stride_row, int64_t stride_col, int64_t chunk_cols,
                       nb200_state* states, const nb200_launch* launch, void* stream);
int nb200_fold_merge(int skeleton, const nb200_params* params,
                     const nb200_state* states, int64_t rows, int64_t nparts,
                     int64_t row_stride, int64_t part_stride,
                     void* out, int dtype, void* stream);

/* The split plan across GPUs without a collective (no counterpart in the reference, which has no
 * multi-GPU path): column shards' chunk states move through NVLink peer memory. Each rank owns an
 * exchange buffer of nb200_peer_buffer_bytes(rows, world, nparts) bytes (device memory, 256-byte
 * aligned, reused across calls), initialises it once with nb200_peer_init (which records the
 * (rows, world, nparts) layout in the buffer's header, clears its epoch and zeroes its slots), and maps
 * every other rank's buffer with nb200_ipc_handle / nb200_ipc_open (CUDA IPC; the library only
 * maps, it allocates nothing). Every rank initialises before any rank's first push (a barrier
 * between them). Per call, in this order on one stream:
 *   nb200_fold_partial  -> states[rows][nlocal] of this rank's shard;
 *   nb200_peer_push     -> writes them into slot `rank` (nparts wide, parts past nlocal empty) of
 *                          every rank's buffer (peers[r] = rank r's buffer as mapped here,
 *                          peers[rank] = buffer), each state tagged with the call's epoch inside
 *                          its 16 bytes (no fence, no flag);
 *   nb200_peer_merge    -> reads each state until it carries the call's epoch (bounded: about a
 *                          second, then bit 2 of nb200_stream_fault and the row reads NaN), merges
 *                          each row's world * nparts states in ascending (rank, part) order into
 *                          out[rows] -- the result of nb200_fold_merge on the gathered states.
 * Every rank makes the same calls in the same order with the same rows and nparts; a call's epoch
 * lives in the buffer, so the sequence may be captured in a CUDA graph and replayed. world <= 8.
 * Layout checks: before storing into a destination, the push kernel compares the call's
 * (rows, world, nparts) with the layout recorded in this rank's and the destination's header; the
 * merge compares its own. On a mismatch (or a buffer never initialised) nothing is stored or read,
 * bit 3 of nb200_stream_fault is set and the merge writes every row as NaN. After fault bit 2 or 3 the
 * ranks' epochs no longer agree: close the exchange on every rank and set it up again. */
int64_t nb200_peer_buffer_bytes(int64_t rows, int64_t world, int64_t nparts);
int nb200_peer_init(void* buffer, int64_t rows, int world, int64_t nparts, void* stream);
int nb200_peer_push(const nb200_state* states, int64_t rows, int64_t nlocal, int64_t nparts,
                    void* const* peers, int world, int rank, void* buffer, void* stream);
int nb200_peer_merge(int skeleton, const nb200_params* params, void* buffer, int64_t rows,
                     int64_t nparts, int world, void* out, int dtype, void* stream);
/* The same call in TWO launches (no counterpart in the reference): the partial fold of this rank's
 * column shard x[rows, ncols_shard] (contiguous rows, 16-byte aligned, row stride, width and
 * chunk_cols multiples of 16 bytes, chunks wider than 4 KB -- narrower ones return
 * NB200_ERR_UNSUPPORTED: use the push form) storing its tagged chunk states straight into every rank's
 * buffer (nb200_fold_partial + nb200_peer_push in one kernel), then the
 * merge of nb200_peer_merge. ncols_total (all ranks' columns) sets the skeletons' 1/N as in
 * nb200_fold_partial. Same buffers, layout checks, fault bits, epochs, parities and protocol as
 * the push/merge pair (the two forms may be mixed, across ranks and across calls), and the same
 * result bit for bit. */
int nb200_peer_fold(int skeleton, const nb200_params* params, const void* x, int dtype, int64_t rows,
                    int64_t ncols_total, int64_t ncols_shard, int64_t stride_row, int64_t chunk_cols, int64_t nparts,
                    void* const* peers, int world, int rank, void* buffer, void* out, void* stream);
/* CUDA IPC of a device allocation: handle (64 bytes) and the byte offset of ptr inside it; open
 * maps a peer's allocation (base; add the peer's offset), close unmaps it. */
int nb200_ipc_handle(const void* ptr, void* handle, int64_t* offset);
int nb200_ipc_open(const void* handle, void** base);
int nb200_ipc_close(void* base);

/* ------------------------------------------------------------------ a3: RMSNorm
 * out = round_in(x * rsqrt_rn(div_rn(sum x^2, ncols) + eps)) * gamma, rounded to the
 * input dtype; fp32 stages with no contraction (neptune_codegen/emitters.py:549-627,
 * launch template.py:294-319). out is contiguous [rows, ncols]. */
int nb200_rms_norm(const void* x, const void* gamma, int dtype, int64_t rows, int64_t ncols,
                   int64_t stride_row, int64_t stride_col, int64_t stride_gamma,
                   double eps, void* out, const nb200_launch* launch, void* stream);

/* RMSNorm over rows held in HOST memory (no counterpart in the reference, whose ops take device
 * tensors): x[rows, ncols] and gamma[ncols] contiguous host buffers (page-locked for the copies to
 * overlap), y[rows, ncols] a host buffer. Rows move through the device in chunks of chunk_rows
 * (0: about 16 MiB per chunk): while chunk k runs on `stream`, chunk k+1 is copied in and chunk
 * k-1 copied back on two helper streams, so both PCIe directions are busy at once. The rows of y
 * equal nb200_rms_norm's on the same rows. work: device memory, 256-byte aligned, of
 * nb200_rms_norm_host_work_bytes(dtype, ncols, chunk_rows) bytes (gamma plus two input and two
 * output chunks). The copies wait for earlier work on `stream`, and `stream` waits for the last
 * copy back: y is complete once `stream` is. Calls on one device serialise their enqueueing. */
int64_t nb200_rms_norm_host_work_bytes(int dtype, int64_t ncols, int64_t chunk_rows);
int nb200_rms_norm_host(const void* x, const void* gamma, int dtype, int64_t rows, int64_t ncols,
                        double eps, void* y, int64_t chunk_rows, void* work, int64_t work_bytes,
                        void* stream);

/* ------------------------------------------------------------------ a4/a5: segments
 * Descriptor status bits, ORed into a caller-owned device word (never a device assert):
 * 1 a length is negative or > nrows, 2 lengths do not cover nrows (checked unless unsafe),
 * 4 a boundary lies outside [0, nrows], 8 boundaries decrease. The word is sticky: the library
 * only sets bits, the caller clears it. */

/* Span construction from lengths (neptune_codegen/torch_op.py:370-387: cat(0, cumsum(lengths))
 * and its assertions): int64 spans[nsegments + 1] from lengths with element stride length_stride.
 * Offsets need no construction: nb200_segment_pool reads them directly. */
int nb200_segment_spans(const void* lengths, int index_dtype, int64_t nsegments, int64_t length_stride,
                        int unsafe, int64_t nrows, int64_t* spans, uint32_t* status, void* stream);

/* Ordered storage-dtype pooling (neptune_codegen/torch_op.py:254-306, launch :390-410): for each
 * segment s and channel c, acc = initial, then for every row r in [bounds[s], bounds[s+1]) in order
 * acc = round_storage(acc + data[r, c]); reduce 0 sum, 1 mean = div_rn(acc,
 * float(round_storage(count))). Empty mean without initial and malformed boundaries give NaN.
 * bounds are nsegments + 1 CSR boundaries (int32 or int64, element stride bound_stride), validated
 * in the kernel into *status (nullable). initial_bits is the fp32 bit pattern of `initial`. out is
 * contiguous [nsegments, channels]. */
int nb200_segment_pool(const void* data, int dtype, int64_t nrows, int64_t channels,
                       int64_t stride_row, int64_t stride_channel,
                       const void* bounds, int index_dtype, int64_t bound_stride, int64_t nsegments,
                       int reduce, int has_initial, uint32_t initial_bits, void* out,
                       uint32_t* status, void* stream);

/* ------------------------------------------------------------------ a9: attention
 * O = softmax(scale * Q K^T [+ causal mask]) V per (batch, head), bf16 in/out with
 * fp32 online max/sum repair; lse (nullable) receives fp32 natural log-sum-exp of the scaled
 * scores per query row, [B, H, S]. Q, K, V, O are contiguous [B, H, S, D], 16-byte aligned;
 * head_dim must be 128 (else NB200_ERR_UNSUPPORTED) and scale > 0. causal != 0 masks key > query.
 * No counterpart in the reference (its roadmap declares attention out of scope:
 * docs/roadmap.md:28-31). */
int nb200_attention(const void* q, const void* k, const void* v, void* o, float* lse,
                    int64_t batch, int64_t heads, int64_t seq, int64_t head_dim,
                    int causal, float scale, void* stream);

/* The same attention with shared key/value heads, strided tensors and per-batch lengths, and its
 * backward pass. q, o are [batch, heads, seq, head_dim], k, v [batch, kv_heads, seq, head_dim] with
 * heads a multiple of kv_heads (query head h reads key/value head h / (heads / kv_heads)); the last
 * dimension is contiguous, the others have element strides. Every base is 16-byte aligned and every
 * stride of a dimension longer than one is a positive multiple of 8 elements (else NB200_ERR_ARG).
 * seq_lens (nullable, device memory): tokens of each batch element, read as clamped to [0, seq];
 * queries and keys at or past it are masked whatever they hold: their rows of o and of the gradients
 * are zero, their lse is -inf. lse is contiguous [batch, heads, seq]. head_dim must be 128. */
typedef struct {
    int64_t batch, heads, kv_heads, seq, head_dim;
    const int32_t* seq_lens;
    int32_t causal;
    float scale;
} nb200_attn_args;
typedef struct {
    int64_t batch, head, seq; /* elements */
} nb200_attn_strides;

/* strides: of q, k, v, o. lse nullable. */
int nb200_attention_fwd(const nb200_attn_args* args, const nb200_attn_strides* strides,
                        const void* q, const void* k, const void* v, void* o, float* lse, void* stream);

/* Gradients of the forward pass's o with respect to q, k, v, given o, lse and grad_o: with
 * P = exp(scale q k^T - lse) recomputed, dv = P^T grad_o, dS = P * (grad_o v^T - rowsum(grad_o * o)),
 * dq = scale dS k, dk = scale dS^T q; dk and dv of a shared head sum over its query heads. P and dS
 * are rounded to bf16 for the products, whose sums are fp32. The result does not depend on
 * scheduling. strides: of q, k, v, o, grad_o, dq, dk, dv. work: device memory, 16-byte aligned, of
 * nb200_attention_bwd_work_bytes(args) bytes. */
int64_t nb200_attention_bwd_work_bytes(const nb200_attn_args* args);
int nb200_attention_bwd(const nb200_attn_args* args, const nb200_attn_strides* strides,
                        const void* q, const void* k, const void* v, const void* o, const float* lse,
                        const void* grad_o, void* dq, void* dk, void* dv, void* work, int64_t work_bytes,
                        void* stream);

/* ------------------------------------------------------------------ norms around a block
 * y = residual + scale a(gate) z with z = post_weight * x rsqrt(mean x^2 + eps) (z = x without a
 * post weight), and h = pre_weight * y rsqrt(mean y^2 + eps) (not computed without a pre weight).
 * x and residual are [rows, width] with unit column stride; gate (nullable) holds one row per
 * rows_per_gate consecutive rows; weights are contiguous [width]; everything is of one dtype. y, h and
 * every gradient are contiguous; pointers need their elements' alignment only, and each its own (the
 * rows move faster where all start on a 16-byte boundary, or alike). All of it is computed in fp32 and rounded once, h from the
 * unrounded y. rstd is fp32 [rows, 2], 8-byte aligned: the two reciprocal norms (1 where a weight is absent).
 * width <= 16384 (else NB200_ERR_CAPACITY); rows a multiple of rows_per_gate. No counterpart in the
 * reference, whose RMSNorm is forward only (neptune_codegen/emitters.py:549-627). */
typedef enum { NB200_GATE_NONE = 0, NB200_GATE_TANH = 1, NB200_GATE_SIGMOID = 2 } nb200_gate_act;
typedef struct {
    const void *x, *residual, *gate, *post_weight, *pre_weight;
    int64_t rows, width;
    int64_t stride_x, stride_residual, stride_gate;     /* elements between rows */
    int64_t stride_grad_y, stride_grad_h;               /* of the backward pass's inputs */
    int64_t rows_per_gate;
    int32_t gate_act;
    double scale, eps;
} nb200_norm_args;
int nb200_gated_norm(const nb200_norm_args* args, int dtype, void* y, void* h, float* rstd, void* stream);

/* Gradients given rstd of the forward pass, grad_y and grad_h (each nullable: zero). dx and dresidual
 * are required; dgate (one row per gate row), dpost and dpre are nullable. work: device memory,
 * 16-byte aligned, of nb200_gated_norm_bwd_work_bytes(args) bytes: fp32 column sums per chunk of
 * rows, added in a fixed order. */
int64_t nb200_gated_norm_bwd_work_bytes(const nb200_norm_args* args);
int nb200_gated_norm_bwd(const nb200_norm_args* args, int dtype, const float* rstd, const void* grad_y,
                         const void* grad_h, void* dx, void* dresidual, void* dgate, void* dpost, void* dpre,
                         void* work, int64_t work_bytes, void* stream);

/* ------------------------------------------------------------------ distillation loss
 * Per row: p_j = exp(teacher_j / T - Z) over the kept entries, Z = logsumexp of their teacher_j / T
 * (teacher_lse null) or teacher_lse[row]; q = softmax(x / T); loss = sum_j p_j (log p_j - log q at
 * index_j); stats = {logsumexp(x / T), Z, sum_j p_j}. An index outside [0, vocab), or a teacher logit
 * of -inf, marks an entry that is not kept; a row without kept entries has loss 0 and gradient 0. x is
 * [rows, vocab] and teacher, index [rows, top], unit column stride; top <= 256 (else
 * NB200_ERR_CAPACITY). loss and teacher_lse are fp32 [rows], stats fp32 [rows, 3], contiguous. Built on
 * the reference's logsumexp skeleton (neptune_codegen/library.py:19), which has no loss and no gradient. */
typedef struct {
    const void *x, *teacher, *index;
    int64_t rows, vocab, top;
    int64_t stride_x, stride_teacher, stride_index;     /* elements between rows */
    int32_t dtype, teacher_dtype, index_dtype;
    double temperature;
} nb200_distill_args;
int nb200_distill_loss(const nb200_distill_args* args, const float* teacher_lse, float* loss, float* stats,
                       void* stream);

/* dx[r, c] = grad[r * stride_grad] / T * (stats mass * q_c - sum of p_j with index_j == c), contiguous, in x's dtype. */
int nb200_distill_loss_bwd(const nb200_distill_args* args, const float* grad, int64_t stride_grad,
                           const float* stats, void* dx, void* stream);

/* ------------------------------------------------------------------ attention behind a shared prefix
 * A few new tokens per sequence against a prefix that all sequences share and each sequence's own cache:
 * o = softmax(scale q K^T) V with K, V the whole prefix followed by the sequence's own tokens up to the
 * query's position. q is [batch, heads, tokens, head_dim], prefix_k, prefix_v [kv_heads, prefix, head_dim]
 * (the batch stride is not used), k, v [batch, kv_heads, cache, head_dim], o contiguous like q, lse
 * (nullable) fp32 [batch, heads, tokens], contiguous, the natural log-sum-exp of the scaled scores.
 * seq_lens (nullable, device memory: every sequence fills its cache): own tokens of each sequence, the new
 * ones included, read as clamped to [0, cache]. Query t stands at own position seq_lens[b] - tokens + t;
 * one before its sequence's first token (a free slot) has a zero row of o and an lse of -inf, as has a row
 * whose every score is -inf. What the caches hold at or past seq_lens does not matter, nor
 * what a later new token holds to an earlier one. dtype NB200_BF16 or
 * NB200_F16 for all tensors; probabilities are rounded to it for the product with V, all sums are fp32.
 * head_dim 64 or 128 (else NB200_ERR_UNSUPPORTED); heads a multiple of kv_heads; bases and strides as for
 * nb200_attention_fwd. prefix or cache may be 0. o, lse and work share no memory with the inputs. work: device memory,
 * 16-byte aligned, of nb200_prefix_attention_work_bytes(args) bytes. The result does not depend on scheduling. No counterpart in
 * the reference; the merge of partial results is its split plan's (neptune_codegen/algebra.py:348-403). */
typedef struct {
    int64_t batch, heads, kv_heads, tokens, head_dim, prefix, cache;
    const int32_t* seq_lens;
    int32_t dtype;
    float scale;
} nb200_prefix_attn_args;
/* strides: of q, prefix_k, prefix_v, k, v. */
int64_t nb200_prefix_attention_work_bytes(const nb200_prefix_attn_args* args);
int nb200_prefix_attention(const nb200_prefix_attn_args* args, const nb200_attn_strides* strides, const void* q,
                           const void* prefix_k, const void* prefix_v, const void* k, const void* v, void* o, float* lse,
                           void* work, int64_t work_bytes, void* stream);

/* ------------------------------------------------------------------ RMSNorm to 8 bits
 * y = x + residual (y = x without a residual), h = weight * y rsqrt(mean y^2 + eps), and per row (group 0) or per
 * group of `group` consecutive columns scale = max(max |h| / most, 2^-126), q = round(h / scale), saturating, with
 * most = 448 (NB200_E4M3), 57344 (NB200_E5M2) or 127 (NB200_I8). All in fp32; y (written only with a residual) is
 * rounded to dtype, h is taken from the unrounded y. A NaN in a row makes its scales NaN and its bytes NaN (0 in
 * int8). x and residual are [rows, width] with unit column stride, weight contiguous [width], all of one dtype; q, y
 * and scale ([rows] or [rows, width / group], fp32) are contiguous. Pointers need their elements' alignment only
 * (rows that all start on 16-byte boundaries move faster); q, scale and y share no memory with the inputs. group is 0, 16, 32, 64 or 128 and divides width;
 * width <= 16384 (else NB200_ERR_CAPACITY). The norm is the reference's (neptune_codegen/emitters.py:549-627)
 * without its intermediate rounding; the reference has no 8-bit output. */
typedef enum { NB200_E4M3 = 0, NB200_E5M2 = 1, NB200_I8 = 2 } nb200_byte_kind;
typedef struct {
    const void *x, *residual, *weight;
    int64_t rows, width, group;
    int64_t stride_x, stride_residual;                  /* elements between rows */
    int32_t dtype, kind;
    double eps;
} nb200_norm8_args;
int nb200_norm8(const nb200_norm8_args* args, void* q, float* scale, void* y, void* stream);

/* ------------------------------------------------------------------ logits before sampling
 * Per row, for each token of the vocabulary, in this order and in fp32, rounded once:
 *   x > 0 ? x / repetition : x * repetition   if the token is in the row's history,
 *   x - frequency * count - presence          if it is among the history's output tokens, count times,
 *   x + the sum of its biases                 (in the order they are given),
 *   x / temperature,
 *   -inf                                      where its bit of allowed is 0.
 * tokens (nullable with history = 0) is [rows, history]: the first token_lens[row] (null: all) are the row's
 * history, of which the first prompt_lens[row] (null: none) are its prompt and the others its output. A token or
 * bias index outside [0, vocab) is skipped. repetition, presence, frequency, temperature: fp32 [rows], each
 * nullable (no such step); the caller keeps repetition and temperature positive (of one below 2^-128 fp32 does not
 * hold the reciprocal: its largest value stands in, so that 0 stays 0). allowed (nullable) is
 * [rows, ceil(vocab / 32)] int32, bit v % 32 of word v / 32. logits is [rows, vocab], out contiguous like it, of one
 * dtype, and no memory of logits; every tensor has unit column stride. biases <= 1024 (else NB200_ERR_CAPACITY).
 * work: device memory, 16-byte aligned, of nb200_penalize_logits_work_bytes(args) bytes (0 without history and
 * biases). No counterpart in the
 * reference. */
typedef struct {
    const void *logits, *tokens, *bias_index;
    const float* bias_value;
    const int32_t *token_lens, *prompt_lens, *allowed;
    const float *repetition, *presence, *frequency, *temperature;
    int64_t rows, vocab, history, biases;
    int64_t stride_logits, stride_tokens, stride_bias_index, stride_bias_value, stride_allowed; /* elements */
    int32_t dtype, token_dtype, bias_dtype;
} nb200_logits_args;
int64_t nb200_penalize_logits_work_bytes(const nb200_logits_args* args);
int nb200_penalize_logits(const nb200_logits_args* args, void* out, void* work, int64_t work_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* NEPTUNE_B200_H */
