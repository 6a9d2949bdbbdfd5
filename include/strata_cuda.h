/*
 * libstrata_cuda — B200 (sm_100a) backend for StrataCuda's mixture-of-experts path.
 *
 * A C ABI (plain pointers, sizes and opaque 64-bit buffer handles; no CUDA or torch types)
 * that a host language binds through its FFI. It replaces the reference's backend object
 * protocol (src/backend.js:58-206: kind, alloc, write, read, copy, zero, run, free, idle,
 * flush, info, dispose) with one context per device, and adds fused entry points for the
 * whole MoE layer so that no routing result crosses to the host.
 *
 * Conventions
 *  - Every call returns a status (STRATA_OK = 0). The message of the last failure on a
 *    context is available from strata_last_error().
 *  - Buffers hold 4-byte elements (src/backend.js:84-92, 128-134): lengths and offsets are
 *    counted in elements, never bytes.
 *  - Calls on one context are stream-ordered and asynchronous; strata_read and strata_idle
 *    synchronise (src/backend.js:94, 117). One thread drives a context at a time.
 *  - Host memory passed in is borrowed only for the duration of the call.
 *  - Kernels never fault on bad indices: a data-dependent index outside its buffer is
 *    skipped and recorded, and the next synchronising call returns STRATA_ERR_DEVICE.
 */
#ifndef STRATA_CUDA_H
#define STRATA_CUDA_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

#define STRATA_OK 0
#define STRATA_ERR_RANGE 1   /* argument outside the supported range: RangeError, src/backend.js:6-9 */
#define STRATA_ERR_LAYOUT 2  /* buffer/shape layout violated: Error, src/backend.js:22-36 */
#define STRATA_ERR_UNKNOWN 3 /* unknown kernel or missing argument: src/backend.js:102; wasm/runtime.js:12 */
#define STRATA_ERR_HANDLE 4  /* not a live buffer of this context: src/backend.js:138-143 */
#define STRATA_ERR_ALLOC 5   /* device allocation failed: wasm/runtime.js:7 "WASM allocation failed" */
#define STRATA_ERR_CUDA 6    /* CUDA runtime error (the message names it) */
#define STRATA_ERR_DEVICE 7  /* a kernel recorded an out-of-range index, an invalid routing, a timed-out wait, a non-finite PLE scale or cache value, cache scales too far apart */

#define STRATA_F32 0
#define STRATA_I32 1
#define STRATA_U32 2

#define STRATA_ARG_BUF 0
#define STRATA_ARG_I32 1
#define STRATA_ARG_F32 2

typedef struct strata_ctx strata_ctx;
typedef uint64_t strata_buf; /* opaque; 0 is never a valid handle */

/* One named argument of strata_run: the reference passes buffers and numbers in one object
 * keyed by the kernel's parameter names (src/backend.js:101-113). */
typedef struct {
    const char *name;
    int32_t kind; /* STRATA_ARG_* */
    int32_t i32;
    float f32;
    strata_buf buf;
} strata_arg;

/* ---- context (GpuBackend.create / dispose, src/backend.js:59-71, 121) ---- */
int strata_create(int device, strata_ctx **out);
int strata_destroy(strata_ctx *ctx);
/* Copies the last error message (NUL-terminated, truncated to cap). Returns its full length. */
int strata_last_error(strata_ctx *ctx, char *buf, size_t cap);
/* The CUDA stream the context issues work on (a cudaStream_t, as an opaque pointer). */
int strata_stream(strata_ctx *ctx, void **stream);

/* ---- buffers (src/backend.js:84-100, 114-118) ---- */
/* alloc(length, type, {zero}); length in 4-byte elements, >= 1. */
int strata_alloc(strata_ctx *ctx, uint64_t length, int type, int zero, strata_buf *out);
int strata_free(strata_ctx *ctx, strata_buf buf);
/* write(buffer, data, offset): count elements from host memory at element offset. */
int strata_write(strata_ctx *ctx, strata_buf buf, const void *data, uint64_t count, uint64_t offset);
/* read(buffer): count elements from element offset into host memory; synchronises. */
int strata_read(strata_ctx *ctx, strata_buf buf, void *out, uint64_t count, uint64_t offset);
/* copy(source, destination, count, sourceOffset, destinationOffset), stream-ordered. */
int strata_copy(strata_ctx *ctx, strata_buf src, strata_buf dst, uint64_t count, uint64_t src_offset, uint64_t dst_offset);
/* zero(buffer), stream-ordered (src/backend.js:93). */
int strata_zero(strata_ctx *ctx, strata_buf buf);
/* Length (elements), type and device address of a live buffer. */
int strata_buffer_info(strata_ctx *ctx, strata_buf buf, uint64_t *length, int *type, void **device_ptr);

/* ---- dispatch (run, src/backend.js:101-113; validateDispatch :10-56) ----
 * Runs one reference entry of kernels/strata.cu by name, with the reference's parameter names and
 * its grid of 64-lane workgroups: all 49 entries that src/engine.js, src/ops.js and src/prefill.js
 * dispatch (mixture of experts, projections, norms, embeddings, RoPE, hyper-connections, the gated
 * delta rule, convolution, attention, per-layer embeddings, argmax; their prompt-batch forms).
 * Results are bit-identical to the reference's F32 CPU path; the RoPE table's cosf / sinf and the
 * softplus's logf, which the reference leaves to its C library, agree with it within one ulp.
 * Validation mirrors src/backend.js:10-56. It also rejects zero divisors and loop extents larger
 * than their buffers, which the reference leaves unchecked.
 *
 * Four further names have no counterpart in the reference. They read a token list or a position
 * from device memory instead of a kernel argument, so that one captured CUDA graph can replay
 * every decode step or full prompt chunk:
 *   strata_embed_token  (Table, Token, Residual, width, streams, vocab, tokens)
 *   strata_rope_at      (X, Cos, Sin, Y, Position, dim, heads, rotary, tokens)
 *   strata_kv_append_at (K, V, Keys, Values, Position, width, tokens)
 *   strata_attention_at (Q, Keys, Values, Position, Y, dim, heads, kvHeads, scale; query tokens = groups[2])
 * Each computes what strata_embedding, strata_rope_position, strata_kv_append_batch and
 * strata_attention_batch compute for the same values.
 *
 * Two more have no counterpart either. They run the decode step's hyper-connection block
 * (src/engine.js:78-84) in two launches instead of six, with each value formed by the same
 * operations in the same order:
 *   strata_hc_in  (Residual, NormW, DownW, InjectW, Norm, Down, Inject, width, streams, rank, epsilon):
 *                 strata_norm of the streams rows, then the down and inject projections of the norm
 *   strata_hc_out (Norm, Down, UpW, Mixed, width, streams, rank, scale):
 *                 strata_elementwise mode 1, the up projection and strata_hc_mix
 *
 * Six more serve decode of many independent sequences at once (a serving batch; the reference
 * holds one session per engine, src/engine.js:53-72). Token t of a dispatch belongs to sequence t,
 * which has its own position Positions[t] and its own slice of the cache, history or state
 * buffer; each gives sequence t what the one-sequence entry in brackets gives it alone:
 *   strata_rope_seqs      (X, Cos, Sin, Y, Positions, dim, heads, rotary, tokens)   [strata_rope_position]
 *   strata_kv_append_seqs (K, V, Keys, Values, Positions, width, cells, tokens)     [strata_kv_append;
 *                          sequence t's cache is cells [t cells, (t + 1) cells) of Keys / Values]
 *   strata_attention_seqs (Q, Keys, Values, Positions, Y, dim, heads, kvHeads, cells, scale;
 *                          sequences = groups[2])                                   [strata_attention_batch]
 *   strata_conv_seqs      (History, X, W, Y, channels, taps, dilation, activation, tokens)  [strata_conv]
 *   strata_gdn_seqs       (State, Q, K, V, Decay, Beta, Y, dim, keyHeads, valueHeads, tokens) [strata_gdn_step]
 *   strata_argmax_rows    (Logits, Tokens, count, rows)                             [strata_argmax per row]
 * A position outside [0, cells) is reported as an index error, never written.
 *
 * Two more run parts of the delta-rule layer in one launch each, with the same values as the
 * dispatches they replace:
 *   strata_gdn_prep (History, X, W, Q, K, V, keyDim, valueDim, headDim, qScale, epsilon): one
 *     token's strata_conv (4 taps, dilation 1, SiLU) over the [q | k | v] projection, the three
 *     strata_slice and the two strata_norm mode 1 (q heads times qScale, k heads);
 *   strata_gdn_gates_fused (X, AlphaW, BetaW, A, Dt, Decay, Strength, width, heads, tokens): the
 *     alpha and beta projections of each token, then strata_gdn_gates (src/engine.js; the batch
 *     forms of src/prefill.js for tokens > 1). */
int strata_run(strata_ctx *ctx, const char *name, const strata_arg *args, int nargs, const uint32_t groups[3]);

/* ---- synchronisation and introspection (idle, flush, info: src/backend.js:119-120) ---- */
int strata_idle(strata_ctx *ctx);
int strata_flush(strata_ctx *ctx);
/* JSON object: device, SMs, bytes resident, buffers, dispatches, fused calls. */
int strata_info(strata_ctx *ctx, char *json, size_t cap);

/* ---- fused mixture-of-experts layer ----
 * One layer's weights, as resident buffers. The routed experts are the layer's slice of
 * experts.bin: `experts` consecutive Q2 blobs (vendor/strata/tools/pack_layer.py:54-65 with
 * H = width, FF = ff: gate/up codes with rows interleaved g0,u0,g1,..., down codes,
 * gate/up FP16 scales, down FP16 scales; 3*ff*width*9/32 bytes per blob), read by
 * src/model.js:160-167. Replaces the per-layer sequence of src/engine.js:133-156 (decode)
 * and src/prefill.js:52-78 (prompt batches). */
typedef struct {
    int32_t width;           /* hidden size H; multiple of 64 */
    int32_t ff;              /* expert intermediate size; multiple of 64 */
    int32_t experts;         /* 1..512 */
    int32_t top_k;           /* 1..min(experts, 32) */
    strata_buf router;       /* f32 [experts * width]: blk.L.ffn_gate_inp.weight, row-major */
    strata_buf router_bias;  /* 0, or f32 [experts] added to the logits (strata_elementwise mode 5) */
    strata_buf experts_blob; /* u32 [experts * blob_bytes / 4] */
    strata_buf shared_blob;  /* u32 [blob_bytes / 4]: the shared expert as one Q2 blob */
    strata_buf shared_gate;  /* f32 [width]: blk.L.ffn_gate_inp_shexp.weight */
} strata_moe_layer;

/* Whole layer for `tokens` rows of x (f32 [tokens * width]) into y (f32 [tokens * width]),
 * routed ids (i32 [tokens * top_k]) and weights (f32 [tokens * top_k]). Routing is
 * bit-identical to strata_router_batch; y follows the reference's combine order.
 *   mode 0: exact — every dot product in the reference's reduction order (bit-identical y).
 *   mode 1: fast — at H/F = 2048/512 or 2560/640 (other shapes run the exact mode):
 *           tokens <= 8: one persistent integer tensor-core launch (decode);
 *           9 .. 64: the exact router kernels, then one integer tensor-core launch;
 *           above 64: the tcgen05 prefill path (FP16 operands).
 *           Routing is still bit-identical. y is within 1e-5 relative L2 up to 64 tokens and
 *           the same bits run to run (fixed summation order); within 2e-3 above 64 tokens,
 *           where the GEMM epilogues add with atomics.
 * Stream-ordered; does not synchronise. */
#define STRATA_MOE_EXACT 0
#define STRATA_MOE_FAST 1
int strata_moe_forward(strata_ctx *ctx, const strata_moe_layer *layer, strata_buf x, int32_t tokens, strata_buf y, strata_buf ids,
                       strata_buf weights, int32_t mode);

/* Replaces the per-blob check of PackStore.readExpertBlob (src/model.js:160-167), which the
 * whole-model upload skips: every FP16 scale of `count` consecutive Q2 blobs in `blobs` (gate/up
 * and down scale planes) must be finite. Returns STRATA_ERR_LAYOUT "Non-finite expert scales
 * (blob i)" naming the lowest offending blob. Synchronises. The fused kernels convert scales
 * with the hardware FP16 conversion and rely on this check having passed on upload. */
int strata_validate_experts(strata_ctx *ctx, strata_buf blobs, int32_t count, int32_t width, int32_t ff);

/* ---- allocation-free fused layer ----
 * No counterpart in the reference. For callers that must not allocate device memory: a host
 * engine that has already carved HBM into its own arenas and forbids allocations behind its
 * accounting; code running during CUDA stream capture, where cudaMalloc is not allowed;
 * processes that may not grow their device footprint. strata_moe_forward grows a workspace
 * with cudaMalloc. This variant takes caller-owned device pointers and a stream (a
 * cudaStream_t as void*; NULL = the default stream), computes exactly what
 * strata_moe_forward computes in mode STRATA_MOE_EXACT, and keeps all temporaries in one
 * static device array of STRATA_NOALLOC_SCRATCH_BYTES compiled into the library.
 *  - Calls needing more scratch are rejected with STRATA_ERR_RANGE (up to 73 tokens at
 *    H 2048 / E 512 / k 10 / F 512).
 *  - The first call on each device looks the array's address up, so make it before any
 *    stream capture.
 *  - Calls share the array: calls that overlap on the GPU race, so order them on one stream.
 *  - The calling thread's current device must own `stream`, the pointers and the layer, in
 *    the runtime's primary context (the array's address is cached per device ordinal); a
 *    stream of another device is rejected with STRATA_ERR_RANGE.
 *  - A token whose routing fails (NaN probabilities) gets id -1; that pair adds nothing to y.
 *    strata_moe_forward reports it as an error at the next synchronising call; this entry
 *    cannot without synchronising, so check `ids` for -1.
 *  - Never allocates or frees. `msg` (optional) receives the reason for a non-zero status. */
#define STRATA_NOALLOC_SCRATCH_BYTES (8u << 20)
typedef struct {
    int32_t width, ff, experts, top_k;   /* as in strata_moe_layer */
    const float *router;                 /* device f32 [experts * width] */
    const float *router_bias;            /* device f32 [experts], or NULL */
    const uint32_t *experts_blob;        /* device u32: experts Q2 blobs */
    const uint32_t *shared_blob;         /* device u32: one Q2 blob */
    const float *shared_gate;            /* device f32 [width] */
} strata_moe_layer_dev;
int strata_moe_forward_noalloc(const strata_moe_layer_dev *layer, const float *x, int32_t tokens, float *y, int32_t *ids,
                               float *weights, void *stream, char *msg, size_t msg_cap);

/* ---- expert-parallel layer over NCCL (one process per GPU) ----
 * The fused entry point strata_moe_ep (the expert-parallel path of BASELINE's north star; the
 * reference has no multi-GPU path). The 512 (layer.experts) routed experts are sharded evenly:
 * rank r owns the experts its placement gives it (strata_ep_set_placement; by default
 * [r E/n, (r + 1) E/n)), and its layer.experts_blob holds exactly those blobs in ascending id;
 * router, shared gate and shared expert are replicated. A rank passes its own tokens and
 * receives their y, ids and weights (routing over all E experts, bit-exact; y within 2e-3
 * relative L2, the tensor-core path's tolerance).
 * Setup: rank 0 calls strata_ep_unique_id, the 128 bytes are shared by the caller (e.g. a
 * torch.distributed broadcast), every rank calls strata_ep_init. NCCL (libnccl.so.2) is bound
 * at run time. Each forward reads the per-peer row counts back to the host once.
 * Failure detection (no reference counterpart; the reference's nearest is its failed-session
 * state, src/engine.js:147-151, and worker-crash rejection, src/backend.js:165-168): the
 * communicator is non-blocking, and every host wait on the peers (the forward's count read,
 * strata_sync/strata_read and friends, strata_destroy) is bounded by strata_ep_set_timeout
 * (default 60 s). A wait that runs out, or an NCCL asynchronous error, aborts the communicator
 * (ncclCommAbort) and returns STRATA_ERR_CUDA naming the cause; later expert-parallel calls
 * fail until strata_ep_init is called again. The context itself stays usable. */
#define STRATA_EP_ID_BYTES 128
int strata_ep_unique_id(strata_ctx *ctx, uint8_t *id, size_t cap);
int strata_ep_init(strata_ctx *ctx, int32_t rank, int32_t n_ranks, const uint8_t *id);
int strata_ep_set_timeout(strata_ctx *ctx, int32_t milliseconds);
/* Expert placement (no reference counterpart): owner[e] is the rank that holds expert e, for
 * e < experts; every rank must own at least one expert, and every rank must set the same
 * placement. A rank's layer.experts_blob then holds the experts it owns in ascending id order.
 * Without a call (or with owner = NULL) rank r owns experts [r E/n, (r + 1) E/n). A placement
 * balanced by the experts' routed rows keeps a skewed router from loading one rank with the
 * popular experts. Synchronises. strata_ep_local_experts gives this rank's blob count under
 * the placement in force for `experts` (setting the contiguous one if none is). */
int strata_ep_set_placement(strata_ctx *ctx, int32_t experts, const int32_t *owner);
int strata_ep_local_experts(strata_ctx *ctx, int32_t experts, int32_t *count);
int strata_moe_ep_forward(strata_ctx *ctx, const strata_moe_layer *layer, strata_buf x, int32_t tokens, strata_buf y, strata_buf ids,
                          strata_buf weights);
/* Same-device loopback transport (no reference counterpart): n virtual ranks on ONE GPU, one
 * context each, driven by n host threads; the exchanges become device-to-device copies
 * between the ranks' buffers, ordered by stream events (no kernel waits on another rank).
 * Tests the expert-parallel layer at 2, 4 or 8 ranks on a single GPU. The hub's creator calls
 * strata_ep_loopback_create once, every rank's context strata_ep_init_loopback(rank, hub);
 * strata_ep_loopback_release drops the creator's reference (the ranks keep theirs). */
int strata_ep_loopback_create(strata_ctx *ctx, int32_t n_ranks, uint64_t *hub);
int strata_ep_init_loopback(strata_ctx *ctx, int32_t rank, uint64_t hub);
int strata_ep_loopback_release(strata_ctx *ctx, uint64_t hub);

/* ---- per-layer embeddings (PLE) on the device ----
 * Replaces the host-side row gather of src/model.js:230-242 (plePackedRows) followed by the
 * strata_ple_decode dispatch of src/ops.js:79-83. The IQ4_NL table (rows of head_dim values,
 * head_dim / 32 * 18 bytes each: per 32 values an FP16 scale and 16 code bytes) stays resident
 * in `table` (u32 words); the host still computes the n-gram row ids (src/model.js ngramRows)
 * and writes them to `ids` (i32). Values[h * head_dim + j] receive exactly what
 * strata_ple_decode gives for the same rows packed one after another. head_dim must be a
 * multiple of 32 ("Invalid packed PLE layout"). A row outside the table reads zeros and a
 * non-finite scale ("Non-finite PLE scales", src/model.js:241) are reported by the next
 * synchronising call. Stream-ordered. */
int strata_ple_gather_decode(strata_ctx *ctx, strata_buf table, strata_buf ids, int32_t rows, int32_t head_dim, strata_buf values);

/* ---- attention over a paged key/value cache held in 8 bits (no reference counterpart) ----
 * The reference keeps F32 caches of at most 2048 cells and leaves sparse selection out
 * (src/model.js:13). These entries serve longer sessions and more of them: a cache of one byte
 * per value, attention over it, and a selection of the blocks that a query attends to.
 *
 * Format. A page holds STRATA_KV8_BLOCK = 64 consecutive tokens (a block) of one sequence for every
 * key/value head. With P = dim padded to 64, 128 or 256:
 *   codes   int8 [pages][kv_heads][2][P * 64]: keys as [P / 64][64 tokens][64 channels], then values as
 *           [P channels][64 tokens]; channels past dim are zero
 *   marks   int8 [pages][kv_heads][2][P]: the lowest and the highest key code of each channel
 *   scales  f32  [pages][kv_heads][2]: key scale, value scale; value = code * scale
 *   open    f32  [sequences][2][64][kv_heads][dim]: the rows of each sequence's last, unfilled block,
 *           from which its codes are formed again when a larger value makes its scale grow
 *   table   i32  [sequences][blocks]: the page of each block (a page belongs to one sequence)
 * With handles the codes and marks are u32 buffers of a quarter as many elements. `workspace` is
 * scratch of STRATA_KV8_WORKSPACE_BYTES, zero-filled once by the caller and then left to these
 * entries; calls that may overlap on the GPU need caches with workspaces of their own.
 *
 * Runs. A call works on segments * count tokens, `count` for each of `segments` runs. Run i belongs
 * to sequence[i] and its first token stands at position start[i]; both are read on the device, so a
 * captured graph can replay the call. sequence -1 marks an idle slot: nothing is appended, nothing is
 * picked, its output is zero. Decode of a batch is count = 1; a prompt chunk is segments = 1.
 * Rows of q, k and v are `row_stride` floats apart (0: contiguous).
 *
 * append: scale = amax / 127 over a block's rows so far (0 below 2^-100), code = x times the
 *   reciprocal of scale, rounded to nearest even. A block's codes depend on its rows alone, not on how they
 *   were split over calls. Appending goes on where the sequence ends; a run that starts at a block's
 *   first token starts that block afresh, and one that starts inside the open block drops its rows from there on (a block
 *   that has been filled is not open any more: only its first token starts it anew).
 *   A value that is not finite is stored as zero and reported. Runs of one call name different sequences.
 * select: for each token and key/value head the `top` blocks (of those at or before the token) with the
 *   largest score, in ascending order, -1 past the last: i32
 *   picks [tokens][kv_heads][top]. The score is sum_d p_d hi_d + n_d lo_d times the block's key scale, where hi, lo
 *   are the marks and p, n the group's positive and negative query parts: queries are rounded to
 *   multiples of amax / 32767, added up as whole numbers and rounded to 8 bits, so that the choice does not
 *   depend on the order of any sum. Without the rounding it is an upper bound on the summed logits of the group's queries;
 *   rounding p and n moves it by half of sum_d |hi_d| + |lo_d| units at most. The `first` first and `last` last blocks
 *   are always picked; equal scores go to the lower block. A query value that is not finite counts as zero. Tables of at most
 *   STRATA_KV8_SELECT_BLOCKS blocks.
 * attend: y [tokens][heads * dim] = softmax(scale * q . k) v over the keys at or before the token's position, of
 *   every block (picks null / 0) or of the blocks that picks [tokens][kv_heads][top] lists (distinct, -1 for
 *   none; top at most 33554431, the blocks that a table can have). Query head h uses key/value head
 *   h / (heads / kv_heads). A token that sees no key gets zeros.
 *   F32 in and out. Queries and weights keep 22 bits or more of their row's largest (8-bit digits or two FP16
 *   halves, by the kernel's form) and meet the codes without rounding these; maxima, sums and results are F32 or wider.
 *   Prompt chunks keep weights times their page's value scale to 2^-31 of the row's largest such product; values of a page
 *   whose scale is below 2^-90 of the largest in sight of the 128 rows of a tile count as zeros there. Tokens
 *   taken one by one refer to the largest value scale of the first 32 pages of a list (of each part that a CTA has): scales
 *   below 2^-40 of it lose bits, and one above 2^80 times it is reported. A query value that is not finite makes its own row NaN.
 *
 * heads / kv_heads is any whole number, dim is 1 .. 256. A run that attends to every block has at most 2^31 - 128 rows
 * (count * heads / kv_heads). A sequence, page or position outside the cache
 * is skipped and reported by the next synchronising call (STRATA_ERR_DEVICE), or, in the pointer forms, by
 * bit 0 of *status (bit 1: a bounded wait in a kernel ran out, bit 4: a value that was not finite, bit 5: value scales too
 * far apart), which the caller clears. */
#define STRATA_KV8_BLOCK 64
#define STRATA_KV8_WORKSPACE_BYTES (32u << 20)
#define STRATA_KV8_SELECT_BLOCKS 32768
typedef struct {
    int32_t kv_heads, dim, pages, sequences, blocks;
    strata_buf codes, marks, scales, open, table, workspace;
} strata_kv8_cache;
int strata_kv8_append(strata_ctx *ctx, const strata_kv8_cache *cache, strata_buf k, strata_buf v, uint64_t row_stride, int32_t segments,
                      int32_t count, strata_buf sequence, strata_buf start);
int strata_kv8_select(strata_ctx *ctx, const strata_kv8_cache *cache, strata_buf q, uint64_t row_stride, int32_t heads, int32_t segments,
                      int32_t count, strata_buf sequence, strata_buf start, int32_t top, int32_t first, int32_t last, strata_buf picks);
int strata_kv8_attend(strata_ctx *ctx, const strata_kv8_cache *cache, strata_buf q, uint64_t row_stride, int32_t heads, int32_t segments,
                      int32_t count, strata_buf sequence, strata_buf start, strata_buf picks, int32_t top, float scale, strata_buf y);
/* The same on caller-owned device memory and a stream (a cudaStream_t as void*; NULL = the default
 * stream) of the calling thread's current device. Nothing is allocated. codes, marks and workspace
 * start on 16-byte boundaries, everything else on its element's. `status` (optional) is a device word
 * that errors are added to; `msg` (optional) receives the reason for a non-zero return. */
typedef struct {
    int32_t kv_heads, dim, pages, sequences, blocks;
    int8_t *codes, *marks;
    float *scales, *open;
    const int32_t *table;
    void *workspace;
    uint32_t *status;
} strata_kv8_cache_dev;
int strata_kv8_append_dev(const strata_kv8_cache_dev *cache, const float *k, const float *v, uint64_t row_stride, int32_t segments,
                          int32_t count, const int32_t *sequence, const int32_t *start, void *stream, char *msg, size_t msg_cap);
int strata_kv8_select_dev(const strata_kv8_cache_dev *cache, const float *q, uint64_t row_stride, int32_t heads, int32_t segments,
                          int32_t count, const int32_t *sequence, const int32_t *start, int32_t top, int32_t first, int32_t last,
                          int32_t *picks, void *stream, char *msg, size_t msg_cap);
int strata_kv8_attend_dev(const strata_kv8_cache_dev *cache, const float *q, uint64_t row_stride, int32_t heads, int32_t segments,
                          int32_t count, const int32_t *sequence, const int32_t *start, const int32_t *picks, int32_t top, float scale,
                          float *y, void *stream, char *msg, size_t msg_cap);
/* The same three with their arguments in a structure, for bindings that pay for each argument. `rows` is k or q; members
 * that an operator does not take are ignored. */
#define STRATA_KV8_APPEND 0
#define STRATA_KV8_SELECT 1
#define STRATA_KV8_ATTEND 2
typedef struct {
    const strata_kv8_cache_dev *cache;
    const float *rows, *v;
    uint64_t row_stride;
    const int32_t *sequence, *start;
    int32_t *picks; /* select: written; attend: read, or null */
    float *y;
    void *stream;
    char *msg;
    uint64_t msg_cap;
    int32_t op, segments, count, heads, top, first, last;
    float scale;
} strata_kv8_call;
int strata_kv8_call_dev(const strata_kv8_call *call);

/* ---- token mixers over runs of many sequences (no reference counterpart) ----
 * The reference walks the delta rule token after token (kernels/strata.cu:304-313, :432-444) and dispatches its inputs and the
 * queries and keys of attention in five steps each (src/engine.js, src/prefill.js). These entries take several tokens of
 * several sequences in one call, single tokens and long prompts alike. F32 in and out, every sum in F32; results agree with the
 * reference's entries to F32 rounding, not bit for bit.
 *
 * Runs. A call works on segments * count rows, `count` for each of `segments` runs; run i belongs to sequence[i], and has
 * lengths[i] tokens (lengths null / 0: count each). Both are read on the device, so a captured graph can replay a call. Rows
 * behind a run's tokens are left as they were. sequence -1 marks an idle slot: its rows become zero, what it holds stays. Runs
 * of one call name different sequences: one that an earlier run has too is reported and treated as idle. Rows of x, q, k and v
 * are `..._stride` floats apart (0: contiguous); results are contiguous and do not overlap what is read.
 *
 * delta_inputs: from a layer's [q | k | v] projection x [rows][channels], channels = (2 key_heads + value_heads) * dim, a causal
 *   convolution of each channel, c_t = sum_m weight[c][m] x_{t - (taps - 1) + m}, which goes on from the sequence's last
 *   taps - 1 inputs (history, oldest first) and leaves the new ones there; s = c / (1 + exp(-c)); for each head of q and k
 *   s / sqrt(sum s^2 + epsilon), q's times q_scale (0: 1 / sqrt(dim)); v = s.
 * delta_rule: with the state S [dim key][dim value] of each value head of the run's sequence, token after token
 *     S <- decay S;  d = beta (v - S^T k);  S <- S + k d^T;  y = S^T q
 *   Value head h reads key head h % key_heads. decay, beta [rows][value_heads]; y [rows][value_heads * dim]. Runs of many
 *   tokens over heads of at most 128 channels are taken in chunks of 64 on the tensor cores, all others token by token. A chunk's factors keep
 *   22 bits down to 2^-27 of what is largest in their row (a token's k or q; a value channel's state over its keys), sums are F32: a token's
 *   result is off by what 22 bits lose of what its state holds, not by the size of what comes later or of what a decay has taken away. A chunk
 *   where that would not hold, or in which a value is not finite (or past 2^60 in magnitude), is walked token by token, so that no token before
 *   it sees it; 0.05 to 0.4 ms a chunk. How a call is taken goes by its segments, count, heads and dim, and by the values: it repeats bit for
 *   bit, and tokens that are cut into other calls differ in their last bits. Token by token S^T k and S^T q are formed before the decay
 *   and have to stay in F32's range there.
 * qk_rope: for each head of q and k x / sqrt(mean x^2 + epsilon) times the kind's weight [dim], its first `rotary` channels
 *   rotated (channel d with d + rotary / 2) by the row start[i] + j of cos and sin [cells][rotary / 2], as strata_norm and then
 *   strata_rope_position. Heads of q may lie q_head_stride floats apart (0: dim), as in a projection of [q | gate] for each head.
 *   A position outside the tables gives a row of zeros and is reported. sequence may be null / 0: no idle slots. y may be what is
 *   read where that is contiguous.
 *
 * dim is 1 .. 256 and value_heads a multiple of key_heads; taps is 1 .. 8. The workspace is scratch of delta_rule of
 * STRATA_DELTA_WORKSPACE_BYTES; calls that may overlap on the GPU need workspaces of their own, calls that follow one another on
 * a stream may share one. A sequence outside [-1, sequences), a length outside [0, count] or a position outside the tables is
 * reported by the next synchronising call (STRATA_ERR_DEVICE), or, in the pointer forms, by bit 0 of *status (bit 1: a bounded
 * wait in a kernel ran out), which the caller clears. */
#define STRATA_DELTA_WORKSPACE_BYTES (128u << 20)
typedef struct {
    int32_t key_heads, value_heads, dim, taps, sequences;
    strata_buf state;     /* f32 [sequences][dim key][value_heads][dim value]; delta_rule */
    strata_buf history;   /* f32 [sequences][channels][taps - 1]; delta_inputs with taps > 1 */
    strata_buf weight;    /* f32 [channels][taps]; delta_inputs */
    strata_buf workspace; /* delta_rule */
} strata_delta_net;
int strata_delta_inputs(strata_ctx *ctx, const strata_delta_net *net, strata_buf x, uint64_t row_stride, int32_t segments, int32_t count,
                        strata_buf sequence, strata_buf lengths, float q_scale, float epsilon, strata_buf q, strata_buf k, strata_buf v);
int strata_delta_rule(strata_ctx *ctx, const strata_delta_net *net, strata_buf q, uint64_t q_stride, strata_buf k, uint64_t k_stride,
                      strata_buf v, uint64_t v_stride, strata_buf decay, strata_buf beta, int32_t segments, int32_t count,
                      strata_buf sequence, strata_buf lengths, strata_buf y);
typedef struct {
    int32_t heads, kv_heads, dim, rotary, cells, sequences;
    strata_buf q_weight, k_weight; /* f32 [dim] */
    strata_buf cos, sin;           /* f32 [cells][rotary / 2]; ignored where rotary is 0 */
} strata_qk_rope_weights;
int strata_qk_rope(strata_ctx *ctx, const strata_qk_rope_weights *weights, strata_buf q, uint64_t q_stride, uint64_t q_head_stride,
                   strata_buf k, uint64_t k_stride, int32_t segments, int32_t count, strata_buf sequence, strata_buf start,
                   strata_buf lengths, float epsilon, strata_buf yq, strata_buf yk);
/* The same on caller-owned device memory and a stream (a cudaStream_t as void*; NULL = the default stream) of the calling
 * thread's current device, with the arguments in a structure. Nothing is allocated. The workspace starts on a 128-byte boundary,
 * everything else on its element's. `status` (optional) is a device word that errors are added to; `msg` (optional) receives
 * the reason for a non-zero return. */
typedef struct {
    int32_t key_heads, value_heads, dim, taps, sequences;
    float *state, *history;
    const float *weight;
    void *workspace;
    uint32_t *status;
} strata_delta_net_dev;
typedef struct {
    const strata_delta_net_dev *net;
    const float *x;
    uint64_t row_stride;
    const int32_t *sequence, *lengths;
    float *q, *k, *v;
    void *stream;
    char *msg;
    uint64_t msg_cap;
    int32_t segments, count;
    float q_scale, epsilon;
} strata_delta_inputs_call;
typedef struct {
    const strata_delta_net_dev *net;
    const float *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride;
    const float *decay, *beta;
    const int32_t *sequence, *lengths;
    float *y;
    void *stream;
    char *msg;
    uint64_t msg_cap;
    int32_t segments, count;
} strata_delta_rule_call;
typedef struct {
    int32_t heads, kv_heads, dim, rotary, cells, sequences;
    const float *q_weight, *k_weight, *cos, *sin;
    uint32_t *status;
} strata_qk_rope_weights_dev;
typedef struct {
    const strata_qk_rope_weights_dev *weights;
    const float *q, *k;
    uint64_t q_stride, q_head_stride, k_stride;
    const int32_t *sequence, *start, *lengths;
    float *yq, *yk;
    void *stream;
    char *msg;
    uint64_t msg_cap;
    int32_t segments, count;
    float epsilon;
} strata_qk_rope_call;
int strata_delta_inputs_dev(const strata_delta_inputs_call *call);
int strata_delta_rule_dev(const strata_delta_rule_call *call);
int strata_qk_rope_dev(const strata_qk_rope_call *call);

/* ---- CUDA graphs of the context's stream (no reference counterpart: the B200 runtime replays
 * captured work instead of relaunching it from the host) ----
 * strata_capture_begin starts capturing the context's stream (thread-local mode): the calls
 * that follow on this thread are recorded, not run. Calls that synchronise (read, idle, free)
 * or that would grow the layer workspace fail while capturing, so run a layer once before
 * capturing it. strata_capture_end instantiates the recorded work and returns a graph handle;
 * strata_graph_launch replays it on the stream (stream-ordered, asynchronous);
 * strata_graph_free synchronises and releases it. The graph keeps the buffers it was captured
 * with: free a graph before freeing its buffers. */
int strata_capture_begin(strata_ctx *ctx);
int strata_capture_end(strata_ctx *ctx, uint64_t *graph);
int strata_graph_launch(strata_ctx *ctx, uint64_t graph);
int strata_graph_free(strata_ctx *ctx, uint64_t graph);

/* ---- device-time profile of the fused layer (diagnostics; no reference counterpart) ----
 * While enabled, strata_moe_forward records CUDA events around its phases on the context's
 * stream. strata_profile_read synchronises, adds the phase times (milliseconds) of every call
 * since the last read into ms[0..n) and resets them; *calls receives the number of calls.
 * Phases: 0 routing (prefill path: router logits, top-k, permutation, activation rows),
 * 1 gate/up tensor-core GEMM, 2 down tensor-core GEMM (prefill and expert-parallel paths),
 * 3 fused decode kernel (decode path), 4 expert-parallel dispatch (counts and rows exchange,
 * regrouping by local expert), 5 expert-parallel return (outputs back to their ranks, combine).
 * strata_moe_ep_forward records phases 0, 4, 1, 2, 5. */
#define STRATA_PHASES 6
int strata_profile(strata_ctx *ctx, int32_t enable);
int strata_profile_read(strata_ctx *ctx, double *ms, int32_t n, uint64_t *calls);

/* ---- seeded synthetic workload (device generator; same bytes as stratacuda_b200/synth.py) ---- */
/* `count` expert blobs of one layer starting at `first_expert` into buf at element offset.
 * `shared` is a flag word: 1 = the shared expert's random streams, 2 = signed FP16 scales
 * N(0, 0.02) instead of |N(0, 0.02)|. */
int strata_synth_blobs(strata_ctx *ctx, strata_buf buf, uint64_t offset, uint64_t seed, int32_t layer, int32_t first_expert,
                       int32_t count, int32_t width, int32_t ff, int32_t shared);
/* `count` normals N(0,1)*scale of stream (seed, tag, sub) from draw `start` into buf at offset. */
int strata_synth_normals(strata_ctx *ctx, strata_buf buf, uint64_t offset, uint64_t seed, uint64_t tag, uint64_t sub, uint64_t start,
                         uint64_t count, double scale);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif
#endif
