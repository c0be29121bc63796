/* fyodor_b200.h - C ABI of the B200 provider for the Fyodor inference engine.
 *
 * The engine binds exactly one symbol, the provider vtable:
 *
 *   const nya_backend_interface *nya_cuda_backend(void);
 *
 * which replaces the reference provider's export in CUDA/cuda.c:457-462 and is
 * registered by backend/core/compute.c:7-9,25-27 when the engine is built with
 * NYA_ENABLE_CUDA. Its fields follow backend/include/compute_backend.h:12-29;
 * every return convention is the engine's (0 = output ready, -1 = decline or
 * failure, NULL plan = run the CPU reference).
 *
 * The fyb_* functions below are extensions for tools, tests and benchmarks
 * that need device-level access (no counterpart in the reference unless a
 * line says otherwise). They take plain pointers and sizes; "stream" is a
 * cudaStream_t passed as void* (NULL = the legacy default stream). Device
 * entry points return 0 on success, -1 for invalid arguments (nothing is
 * launched) and -2 for a CUDA launch failure.
 */
#ifndef FYODOR_B200_H
#define FYODOR_B200_H

#include "fyodor_b200_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Provider vtable. Replaces CUDA/cuda.c:457-462 (nya_cuda_backend). */
const nya_backend_interface *nya_cuda_backend(void);

/* Library identification (no counterpart in the reference). */
const char *fyb_version(void);
/* Number of CUDA devices visible to this process; 0 when none. */
int fyb_device_count(void);

/* ---- device-level kernels ---------------------------------------------- */

/* out[i] = value i of a GGUF tensor, bit-exact with the engine's
   nya_llm_tensor_value (backend/core/llm_quant.c:91-142). Device pointers. */
int fyb_dequantize(const void *weights, size_t count, unsigned type, float *out, void *stream);

/* Scratch needed by fyb_quant_matmul for one shape (bytes; 0 when none). */
size_t fyb_quant_matmul_workspace(size_t rows, size_t columns, unsigned type, size_t batch);

/* Y[b][r] = sum_k W[r][k] * X[b][k] on the device, the batched form of the
   engine's nya_compute_matmul_typed (backend/include/compute.h:80-83): W in
   GGUF row-major block storage, X batch-major [batch][columns], Y
   [batch][rows]. Q4_K/Q6_K run the tensor-core GEMV at batch 1-2 and the
   small-batch GEMM above it (up to 16 vectors per launch, every weight unit
   read once); Q8_0 with columns a multiple of 256 (and 16-byte aligned W and
   X) runs the bulk-staged Q8_0 kernel (up to 8 vectors per launch); every
   other case runs the type-generic kernel. `workspace` must hold
   fyb_quant_matmul_workspace() bytes: [counters][stream-K partials][repacked
   units][small-batch GEMM scratch], the counters zero before the first call
   (calls return them to zero). K-quant weights are repacked into the
   workspace on every call, so this entry point is for testing, not a hot
   loop (plans repack once). The layout depends on the device's SM count:
   use a workspace on the device it was sized for. */
int fyb_quant_matmul(const void *weights, size_t rows, size_t columns, unsigned type,
    const float *x, float *y, size_t batch, void *workspace, size_t workspace_bytes, void *stream);

/* fyb_quant_matmul in two halves (Q4_K/Q6_K only, -1 for other types): the
   repack of W into the workspace's units, once per weight matrix, then any
   number of products from the repacked workspace (the timed path of the
   matvec sweep). Same workspace size and results as fyb_quant_matmul. */
int fyb_quant_repack(const void *weights, size_t rows, size_t columns, unsigned type, void *workspace,
    size_t workspace_bytes, void *stream);
int fyb_quant_matmul_prepared(size_t rows, size_t columns, unsigned type, const float *x, float *y, size_t batch,
    void *workspace, size_t workspace_bytes, void *stream);

/* Decode attention over an fp16 KV cache for a ragged batch of sequences
   (no reference counterpart at this level; the engine's semantics are
   backend/core/llm_cpu.c:510-535 with an F32 cache).
   q   [nseq][heads][head_dim] f32, out [nseq][heads][head_dim] f32
   k,v per sequence s at k + s*seq_stride: [kv_heads][capacity][head_dim] f16
   lengths[s] = attended positions of sequence s (device array, 1..capacity).
   splits = context partitions per (sequence, kv head); 0 picks a default.
   workspace: fyb_attention_workspace() bytes, zero before the first call.
   With 2..64 query heads per KV head one CTA computes all of them on tensor
   cores (fp16 MMAs on hi/lo splits of q and of the probabilities, fp32
   accumulation), reading each K/V tile once. */
size_t fyb_attention_workspace(unsigned nseq, unsigned heads, unsigned kv_heads, unsigned head_dim, unsigned splits);
int fyb_attention_decode(const float *q, const void *k_cache, const void *v_cache, size_t seq_stride,
    const unsigned *lengths, unsigned nseq, unsigned heads, unsigned kv_heads, unsigned head_dim,
    unsigned capacity, float scale, float *out, unsigned splits, void *workspace, size_t workspace_bytes,
    void *stream);

/* Speculative verification: `queries` query rows per sequence (the draft
   tokens), causal within the draft (no counterpart in the reference, whose
   verification runs the drafts one decode step at a time,
   backend/core/llm_cpu.c:1274-1305). q and out are
   [nseq][queries][heads][head_dim]; lengths[s] counts sequence s's cached
   positions including its draft (>= queries), and query j attends positions
   0 .. lengths[s] - queries + j. workspace: fyb_attention_workspace(nseq *
   queries, ...) bytes, zero before the first call. nseq * queries <= 65535.
   When queries x (heads / kv_heads) <= 64 one CTA takes all draft rows of a
   KV head and reads each K/V tile once for them (the tensor-core kernel of
   fyb_attention_decode); otherwise every row streams the cache on its own. */
int fyb_attention_verify(const float *q, const void *k_cache, const void *v_cache, size_t seq_stride,
    const unsigned *lengths, unsigned nseq, unsigned queries, unsigned heads, unsigned kv_heads, unsigned head_dim,
    unsigned capacity, float scale, float *out, unsigned splits, void *workspace, size_t workspace_bytes,
    void *stream);

/* fyb_attention_decode without a workspace argument and without allocating
   anything (no counterpart in the reference). Same arguments and results as
   fyb_attention_decode; the scratch is a fixed array of
   FYB_ATTENTION_STATIC_SCRATCH_BYTES per device inside the library. Meant
   for callers that cannot allocate device memory where they call: a hook
   that runs under a device-memory budget it has already used up
   (NYA_CUDA_MEMORY_MIB), or a latency path that must not take cudaFree's
   implicit device synchronization.
   - The first call on a device (that device current) looks up the array's
     address; make that first call before any stream capture on the device.
   - Returns -3, launching nothing, when the problem needs more scratch than
     the array holds (fyb_attention_workspace() gives the need).
   - One array per device: calls that overlap in time on one device (other
     streams or threads) race on it and must be serialized by the caller.
   - The array is resident on every device that loads the library (4 MiB,
     outside the NYA_CUDA_MEMORY_MIB budget), and the address found at the
     first call assumes the device's primary context is never reset. */
#define FYB_ATTENTION_STATIC_SCRATCH_BYTES ((size_t)4 << 20)
int fyb_attention_decode_static(const float *q, const void *k_cache, const void *v_cache, size_t seq_stride,
    const unsigned *lengths, unsigned nseq, unsigned heads, unsigned kv_heads, unsigned head_dim,
    unsigned capacity, float scale, float *out, unsigned splits, void *stream);

/* ---- resident plans ---------------------------------------------------- */

/* Greedy decode entirely on the device: starting from `token` at `position`,
   run `steps` tokens, each taking the argmax of the previous logits (first
   index of the maximum, as nya_llm_sample with temperature 0 does,
   backend/core/llm_cpu.c:896-905). tokens_out[i] receives the i-th generated
   token. `plan` is a state returned by the vtable's plan_create. */
int fyb_plan_decode_greedy(void *plan, uint32_t token, size_t position, size_t steps, uint32_t *tokens_out);

/* Speculative verification (the engine's serial draft check,
   backend/core/llm_cpu.c:1274-1305, as one pass): count (1..16) draft tokens
   at positions [position, position + count) of a single-GPU plan's sequence
   (position <= the valid prefix), causal attention inside the draft, every
   weight read once for all of them; the logits of every draft position to
   logits [count][V] (suppressed ids -inf). The draft's K/V rows stay in the
   cache: the caller continues from the accepted prefix, whose later positions
   the next call rewrites. 0 / -1 invalid or no chunker (tensor-parallel
   shards, NYA_CUDA_CHUNKED_PREFILL=0) / -1 and a failed plan on a device
   error. */
int fyb_plan_verify(void *plan, const uint32_t *tokens, size_t count, size_t position, float *logits);

/* Times `steps` device-side greedy steps with CUDA events on the plan's
   stream (no host synchronization between steps); returns milliseconds or
   a negative value on failure. */
double fyb_plan_time_greedy(void *plan, uint32_t token, size_t position, size_t steps);

/* Kernel launches of one plan_token step: the request update plus the
   persistent decode kernel (2), or 3 + 5 per layer when the plan runs
   one kernel per operation. */
unsigned long long fyb_plan_launches_per_token(const void *plan);

/* Which decode step the plan runs: 0 one kernel per operation
   (NYA_CUDA_PERSISTENT=0 or an unsupported geometry), 1 the persistent
   kernel with CTA barriers between phases (default), 2 its dataflow form
   (NYA_CUDA_DATAFLOW=1: phases start per 256-column input block as its
   producers finish, no CTA barrier inside matrix phases; single GPU). -1 for
   a null plan. */
int fyb_plan_decode_form(const void *plan);

/* Average duration (ms) of each kernel class of one decode step measured
   with CUDA events around eager launches: out[0] matrix kernels, out[1]
   attention, out[2] other. Returns 0 on success. */
int fyb_plan_profile(void *plan, uint32_t token, size_t position, size_t steps, double *out);

/* Profiling of the persistent decode kernel (no reference counterpart): runs
   one decode step of `token` at `position` with per-CTA trace points and
   copies them to out[point * grid + cta] (globaltimer nanoseconds). Points
   per CTA: start; per layer, for the QKV, attention, O, gate/up and down
   phases, (CTA idle, dependency met) pairs, with a point after each input
   preparation and after the CTA's attention items; logits (idle, met,
   prepared); exit (idle, met). Returns the number of points per CTA and
   stores the grid in *grid_out, or -1 (plan without the persistent kernel,
   invalid arguments, out_count too small). With warp_out (may be NULL),
   also per-warp records of every GEMV phase: warp_out[((layer*5 + phase) *
   warps + warp) * 8 + k] (phase 0 QKV, 1 O, 2 gate/up, 3 down; layers*5 for
   the logits), k = 0 entry (ns), 1 SM clock cycles spent waiting for
   weights, 2 units computed (ns), 3 done (ns); then the default form's
   times (ns) after 4 the CTA barrier that follows the units, 5 the outputs
   of tiles shared between warps, 6 the fence, 7 the second CTA barrier; the
   dataflow form's 4 input preparation at phase entry done (ns), 5 cycles
   waiting for input blocks between units, 6 cycles in tile outputs;
   warp_count >= (layers*5 + 1) * grid * 16 * 8. The dataflow form has
   fewer CTA points (start; per layer the CTA idle and ready points before
   attention and the end of attention; exit idle and ready) and leaves the
   rest 0. */
long fyb_plan_trace(void *plan, uint32_t token, size_t position, unsigned long long *out, size_t out_count,
    unsigned *grid_out, unsigned long long *warp_out, size_t warp_count);

/* Average milliseconds of one stand-alone launch of a fused projection
   kernel of `layer` (which: 0 QKV+RoPE+KV append, 1 attention output,
   2 gate/up+SwiGLU, 3 down, 4 logits+argmax), timed over `reps` launches
   with CUDA events; *bytes receives the kernel's algorithmic bytes per
   launch (weights, input vector, norm weights, outputs). Timed launch i
   uses layer (layer + 1 + i) % layers, so with many layers consecutive
   launches read different weights (more bytes than L2 holds). */
double fyb_plan_time_projection(void *plan, unsigned layer, unsigned which, unsigned reps, size_t *bytes);

/* ---- batched decode (the engine's per-token step, reference
   CUDA/resident.inc:434-595 and backend/core/llm_cpu.c:424-578, applied to
   B sequences at once; the reference plan decodes one sequence) ----------
   fyb_batch_create: B (1..16) sequences of a resident plan's model, each with
   its own fp16 KV cache of the plan's capacity and its own position; they
   share the plan's weights (the plan must outlive the batch; single-GPU
   plans only). NULL if declined. Every step multiplies each weight once for
   all B sequences (batches of 9..16 on the tcgen05 small-batch GEMM).
   fyb_batch_step: one step of every sequence b at positions[b] with
   tokens[b] (position + 1 <= capacity); logits [B][V] (raw, no suppressed
   ids) and argmax [B] (first index of the maximum) copied out when
   non-null. 0 / -1 invalid / -2 device failure.
   fyb_batch_decode_greedy: `steps` greedy steps on the device from
   tokens / positions (each position + steps <= capacity); out [steps][B].
   fyb_batch_time_greedy: milliseconds per greedy step over `steps` graph
   replays (CUDA events) from tokens / positions (each position + steps <=
   capacity), after two untimed steps from the same start; < 0 on error.
   fyb_batch_launches_per_step: kernels in the last step enqueued. */
void *fyb_batch_create(void *plan, unsigned batch);
/* The same over a paged 8-bit cache: the sequences share `blocks` blocks of
   block_size tokens per layer (FYB_KV8_INT8 or FYB_KV8_E4M3; fyb_kv_blocks,
   fyb_kv8_append and fyb_kv8_attention make the step's cache part). Sequence
   b's position may be at most the tokens it holds; an earlier one gives the
   blocks past it back first. A step, or a run of greedy steps, that needs more
   blocks than there are is refused (-1) before anything is launched. */
void *fyb_batch_create_kv8(void *plan, unsigned batch, uint32_t blocks, uint32_t block_size, uint32_t format);
/* The same over a paged 4-bit cache (fyb_kv4_append, fyb_kv4_attention; head
   dimension 64 or 128): 0.56 of its bytes. */
void *fyb_batch_create_kv4(void *plan, unsigned batch, uint32_t blocks, uint32_t block_size);
/* Blocks of a paged batch that no sequence holds (-1 for other batches). */
long fyb_batch_free_blocks(const void *batch);
void fyb_batch_free(void *batch);
int fyb_batch_step(void *batch, const uint32_t *tokens, const uint32_t *positions, float *logits, uint32_t *argmax);
/* fyb_batch_step whose logits stay on the device (raw, no suppressed ids): of
   each sequence b the log probability and rank of targets[b] (the token that
   follows tokens[b] in a text; negative: none), the entropy, and the top (0..32)
   most probable tokens, as fyb_logprobs gives them (host arrays [B], [B][top]).
   targets, logprob, rank and entropy may be NULL, logprob and rank need targets.
   What scores a text, or a cache of fewer bits by what it costs. */
int fyb_batch_score(void *batch, const uint32_t *tokens, const uint32_t *positions, const int32_t *targets,
    float *logprob, int32_t *rank, float *entropy, uint32_t top, int32_t *top_tokens, float *top_logprobs);
int fyb_batch_decode_greedy(void *batch, const uint32_t *tokens, const uint32_t *positions, size_t steps,
    uint32_t *out);
double fyb_batch_time_greedy(void *batch, const uint32_t *tokens, const uint32_t *positions, size_t steps);
unsigned long long fyb_batch_launches_per_step(const void *batch);

/* ---- paged 8-bit KV cache (no counterpart in the reference, whose cache is
   one F32 array per sequence, backend/core/llm_cpu.c:510-535) --------------
   The cache is a pool of blocks of block_size tokens. A request's tokens lie
   in the blocks its row of a block table names, token t in block
   table[t / block_size] at offset t % block_size, so requests of any length
   share the pool. K and V are stored in 8 bits with one F32 scale for each
   (block, KV head): value = stored * scale. A serving step runs
   fyb_kv_blocks once, then per layer fyb_kv8_append (with RoPE) and
   fyb_kv8_attention; all of them read lengths, tables and slots on the
   device, so a CUDA graph of the step serves every later step.

   q, k, v rows are `type` F32, F16 or BF16 (GGML ids 0, 1, 30), strides in
   elements; a row's heads are contiguous. A call of no rows does nothing and may
   pass NULL for the rows. Every pointer below is a device
   pointer unless a line says otherwise; `error` (may be NULL) is a device
   word that receives 4 when an index read on the device is out of range (the
   row or position concerned is then left out) and 2 for non-finite values
   given to the cache; kernels set it and never clear it. */
#define FYB_KV8_INT8 0u /* signed integers -127..127 */
#define FYB_KV8_E4M3 1u /* 8-bit floats, 4 exponent and 3 mantissa bits, largest 448 */
typedef struct fyb_kv8_cache {
    void *k, *v;              /* [blocks][kv_heads][block_size][head_dim] bytes, 16-byte aligned */
    float *k_scale, *v_scale; /* [blocks][kv_heads] */
    uint32_t blocks, kv_heads;
    uint32_t block_size;      /* 16, 32, 64, 128 or 256 tokens */
    uint32_t head_dim;        /* 64 or 128 */
    uint32_t format;          /* FYB_KV8_INT8 or FYB_KV8_E4M3 */
} fyb_kv8_cache;

/* One step's block tables and slot maps from request lengths, in one launch.
   Request r holds lengths[r] tokens and brings new_tokens[r] more; its blocks
   are table[r * table_stride ..]. The blocks it needs beyond those it has are
   popped, requests in order, from the stack free_list[0 .. free_count[0]):
   the j-th block of the step is free_list[free_count[0] - 1 - j], written to
   the table. Requests are served whole or not at all: status[r] 0 served, 1
   too few free blocks (all later requests that need one are refused too), 2
   invalid (negative counts, more tokens than the table holds or than 2^31 - 1,
   rows beyond max_rows). Outputs: lengths_out[r] (lengths + new when served),
   free_count_out[0], row_start [requests + 1] (the step's rows, request after
   request, clamped to max_rows) and, per row 0..max_rows, slots (block *
   block_size + offset; -1 for rows of refused requests and rows beyond the
   last), positions (token index in its request, 0 beyond the last row) and
   row_request (-1 beyond the last row). lengths_out and free_count_out are
   buffers of their own (-1 when they are the inputs): a step can be repeated.
   requests <= 16384, max_rows < 2^30, block_size a power of two. */
int fyb_kv_blocks(const int32_t *lengths, const int32_t *new_tokens, uint32_t requests, int32_t *table,
    size_t table_stride, uint32_t block_size, const int32_t *free_list, const int32_t *free_count,
    int32_t *lengths_out, int32_t *free_count_out, int32_t *row_start, int32_t *slots, int32_t *positions,
    int32_t *row_request, uint32_t max_rows, int32_t *status, void *stream);
/* Shortens every request r to keep[r] tokens (longer than it is: nothing; 0 or
   less: finished): the blocks it needs no more are pushed on free_list (of
   free_capacity entries; a request whose blocks do not fit stays as it is, and
   so do all after it) in request order, their table entries set to -1,
   lengths[r] set, free_count[0] raised. What rejects drafts and ends requests.
   In place. requests <= 16384. */
int fyb_kv_release(int32_t *lengths, const int32_t *keep, uint32_t requests, int32_t *table, size_t table_stride,
    uint32_t block_size, int32_t *free_list, int32_t *free_count, uint32_t free_capacity, void *stream);

/* Rotary positions. The engine's frequencies (backend/core/llm_cpu.c:216-229)
   scaled for long contexts, on the host: freq[j], j < dims / 2, and in
   *magnitude what cos and sin are multiplied by. */
#define FYB_ROPE_PLAIN 0u  /* base^(-2j/dims) */
#define FYB_ROPE_LINEAR 1u /* divided by factor */
#define FYB_ROPE_NTK 2u    /* base grown to base * factor^(dims / (dims - 2)) */
#define FYB_ROPE_YARN 3u   /* between plain and linear by the turns a dimension makes over original_context (beta_fast,
                              beta_slow); magnitude 0.1 ln(factor) + 1 */
#define FYB_ROPE_BANDS 4u  /* plain above high_freq turns, linear below low_freq turns, blended between */
typedef struct fyb_rope_scaling {
    uint32_t kind;
    float factor, original_context;
    float beta_fast, beta_slow; /* YARN (32 and 1 where 0) */
    float low_freq, high_freq;  /* BANDS (1 and 4 where 0) */
} fyb_rope_scaling;
/* scaling may be NULL (plain); factors (may be NULL): dims / 2 divisors of the
   frequencies (a model's rope_freqs tensor). Host pointers. */
int fyb_rope_frequencies(uint32_t dims, float base, const fyb_rope_scaling *scaling, const float *factors,
    float *freq, float *magnitude);
/* cos / sin [rows][dims / 2] of the angles (float)(first + row) * freq[j], times
   magnitude (freq on the device). */
int fyb_rope_tables(const float *freq, uint32_t dims, float magnitude, uint32_t first, uint32_t rows, float *cos_table,
    float *sin_table, void *stream);

#define FYB_ROPE_INTERLEAVED 0u /* pairs (2j, 2j + 1) */
#define FYB_ROPE_HALF 1u        /* pairs (j, j + dims / 2) */
typedef struct fyb_rope_desc {
    const float *cos_table, *sin_table; /* [table_rows][dims / 2], 16-byte aligned */
    uint32_t table_rows;
    uint32_t dims;                      /* the first dims (even) of every head are rotated, the rest is copied */
    uint32_t layout;
} fyb_rope_desc;
/* q_out / k_out = q / k [rows][heads][head_dim] rotated to positions[row] (k may be
   NULL with kv_heads 0, q with heads 0, not both). An output may be its input (same stride). A row whose
   position is outside the table is not written. */
int fyb_rope(const fyb_rope_desc *rope, const int32_t *positions, size_t rows, uint32_t head_dim, uint32_t type,
    const void *q, size_t q_stride, void *q_out, size_t q_out_stride, uint32_t heads, const void *k, size_t k_stride,
    void *k_out, size_t k_out_stride, uint32_t kv_heads, uint32_t *error, void *stream);

/* Append K and V rows [rows][kv_heads][head_dim] at slots[row] (a negative slot
   is skipped). Rows of one block follow one another in the list and ascend (what
   fyb_kv_blocks makes of each request); rows without a slot may lie between
   them, all rows of a block within block_size of each other. Tokens are
   appended: those below the first new one of a block stay, those above it are
   no longer valid. A row whose position is out of the table is left out of K,
   its neighbours in the block are not; a block none of whose rows is stored
   stays as it is. The
   block's scale becomes max(old scale, max|x| * (1 / 127 or 1 / 448)) (the old
   scale counts only if the block holds older tokens); where it grows the older
   tokens are stored anew, q' = round(q * (old / new)); new ones are
   round(x / scale), to nearest even, every step in F32. Infinities are stored as the largest
   value, NaN as 0, neither counts for the scale. With `rope` K is rotated to
   positions[row] first, and q (may be NULL with heads 0) to q_out as by
   fyb_rope, in the same call; half pairs then need dims a multiple of 8. */
int fyb_kv8_append(const fyb_kv8_cache *cache, const int32_t *slots, size_t rows, uint32_t type, const void *k,
    size_t k_stride, const void *v, size_t v_stride, const fyb_rope_desc *rope, const int32_t *positions,
    const void *q, size_t q_stride, void *q_out, size_t q_out_stride, uint32_t heads, uint32_t *error, void *stream);
/* k_out / v_out [rows][kv_heads][head_dim] F32 = the values held at slots[row] (0 for a
   negative slot), as plan_read_kv returns a plan's rows. */
int fyb_kv8_read(const fyb_kv8_cache *cache, const int32_t *slots, size_t rows, float *k_out, float *v_out,
    uint32_t *error, void *stream);

/* Causal attention of the newest rows of each request over its blocks.
   Request r has lengths[r] tokens in the cache (its rows of this step among
   them) and the rows row_start[r] .. row_start[r + 1] of q and out, at most
   max_rows each (row_start NULL: one row per request, row r); row j of n
   attends tokens 0 .. lengths[r] - n + j, scores q.k * scale, softmax and sums
   in F32. A row that attends nothing is 0. q [rows][heads][head_dim] and out
   of `type`; heads a multiple of kv_heads, at most 64 per KV head. Infinities
   and NaN in slots past a request's length have no effect.
   workspace: fyb_kv8_attention_workspace() bytes on this device, zero before
   the first call (calls leave it so); calls that overlap in time need
   workspaces of their own. Results do not depend on timing. */
size_t fyb_kv8_attention_workspace(uint32_t requests, uint32_t max_rows, uint32_t heads, uint32_t kv_heads,
    uint32_t head_dim);
int fyb_kv8_attention(const fyb_kv8_cache *cache, const int32_t *lengths, const int32_t *row_start, uint32_t requests,
    uint32_t max_rows, size_t rows, const int32_t *table, size_t table_stride, uint32_t type, const void *q,
    size_t q_stride, void *out, size_t out_stride, uint32_t heads, float scale, void *workspace,
    size_t workspace_bytes, uint32_t *error, void *stream);

/* ---- paged 4-bit KV cache (no counterpart in the reference) ---------------
   The cache of the section above in 4.5 bits a value: blocks, tables, slots,
   lengths, row types, strides and error words as there (fyb_kv_blocks and
   fyb_kv_release serve both). Each group of 64 values of a head of a token is
   held as low + scale * n, n = 0..15, scale and low F16. Of the group's finite
   values, those beyond +-61440 taken as +-61440, low and high are the least (-0
   less than 0) and the greatest rounded to F16, scale is (high - low) / 15
   rounded to F16, and n is the whole number nearest to (x - low) / scale, ties
   to even, in 0..15 (0 where scale is 0). Infinities are held as 0 or 15, NaN as
   0 would be; both raise 2 in `error`. A group without a finite value has low
   and scale 0. A row depends on no other: tokens may be written in any order,
   and again.
   A token's row of a head is head_dim / 8 words of 32 bits, each eight values,
   the first in the lowest bits: word w holds dimensions 8w.. of a head of 64;
   of a head of 128 word 2j holds dimensions 8j.., word 2j + 1 64 + 8j... */
typedef struct fyb_kv4_cache {
    void *k, *v;             /* [blocks][kv_heads][block_size][head_dim / 2] bytes, 16-byte aligned */
    void *k_scale, *v_scale; /* [blocks][kv_heads][block_size][head_dim / 64][2] F16: scale, low; 16-byte aligned */
    uint32_t blocks, kv_heads;
    uint32_t block_size;     /* 16, 32, 64, 128 or 256 tokens */
    uint32_t head_dim;       /* 64 or 128 */
} fyb_kv4_cache;
/* Append K and V rows at slots[row] (a negative slot is skipped, every other
   occurs once in a call). A row whose slot is out of range is left out, one
   whose position is out of the table is left out of K. With `rope` K is rotated
   in F32 to positions[row] first, and q (may be NULL with heads 0) to q_out as
   by fyb_rope, in the same call. */
int fyb_kv4_append(const fyb_kv4_cache *cache, const int32_t *slots, size_t rows, uint32_t type, const void *k,
    size_t k_stride, const void *v, size_t v_stride, const fyb_rope_desc *rope, const int32_t *positions,
    const void *q, size_t q_stride, void *q_out, size_t q_out_stride, uint32_t heads, uint32_t *error, void *stream);
/* k_out / v_out [rows][kv_heads][head_dim] F32, 16-byte aligned = the values held at slots[row] (0 for a negative slot). */
int fyb_kv4_read(const fyb_kv4_cache *cache, const int32_t *slots, size_t rows, float *k_out, float *v_out,
    uint32_t *error, void *stream);
/* Causal attention of the newest rows of each request over its blocks:
   fyb_kv8_attention's arguments, workspace rules and results over this cache.
   Rows of 16 bits are computed with weights of one fp16 half from five rows per
   KV head on (max_rows x heads of a group), from nine on with K and V rounded to
   fp16 too: fp16 rows are then some 3e-4 and 4e-4 of the norm off, where rounding
   the output alone is 2e-4. F32 rows are not (3e-6), whatever their number, but
   each eight of them read the cache once. */
size_t fyb_kv4_attention_workspace(uint32_t requests, uint32_t max_rows, uint32_t heads, uint32_t kv_heads,
    uint32_t head_dim);
int fyb_kv4_attention(const fyb_kv4_cache *cache, const int32_t *lengths, const int32_t *row_start, uint32_t requests,
    uint32_t max_rows, size_t rows, const int32_t *table, size_t table_stride, uint32_t type, const void *q,
    size_t q_stride, void *out, size_t out_stride, uint32_t heads, float scale, void *workspace,
    size_t workspace_bytes, uint32_t *error, void *stream);

/* ---- log probabilities (the engine's callers take them from whole logits on
   the host; no counterpart in the reference) --------------------------------
   Of each row x of logits [rows][vocabulary] (`type` F32, F16 or BF16, stride in
   elements), in F32 and natural units:
     logprob[r]       x[t] - ln sum exp x, t = tokens[r]
     rank[r]          logits above x[t], and equal ones before it
     entropy[r]       - sum p ln p
     top_tokens, top_logprobs [rows][top]   the most probable tokens, of equal
                      ones the first; -1 and -inf beyond those of probability > 0
   tokens and logprob may be NULL together, rank (needs tokens) and entropy
   alone, top_tokens and top_logprobs with top 0. A negative token asks for none
   (logprob 0, rank -1); one past the vocabulary is taken so and raises 4 in
   `error`. A logit of -inf is a token that cannot be answered: logprob -inf, no
   part in the entropy; a row of nothing else has logprob -inf and entropy 0. A
   row with NaN or +inf raises 2: its logprob, entropy and top_logprobs are NaN,
   NaN is not among its alternatives.
   top <= 32, rows <= 2^31 - 1. workspace: fyb_logprobs_workspace() bytes, 16-byte aligned,
   zero before the first call (calls leave it so); calls that overlap in time
   need workspaces of their own. Results do not depend on timing. */
#define FYB_LOGPROBS_TOP 32u
size_t fyb_logprobs_workspace(size_t rows, uint32_t vocabulary, uint32_t top);
int fyb_logprobs(uint32_t type, const void *logits, size_t stride, size_t rows, uint32_t vocabulary,
    const int32_t *tokens, float *logprob, int32_t *rank, float *entropy, uint32_t top, int32_t *top_tokens,
    float *top_logprobs, void *workspace, size_t workspace_bytes, uint32_t *error, void *stream);

/* ---- tensor parallelism across processes (no reference counterpart) -----
   A process whose environment holds NYA_CUDA_TP_SIZE=N (2..8) and
   NYA_CUDA_TP_RANK=r (and NYA_CUDA_DEVICE for its GPU) creates plans that hold
   rank r's shard of the model: its H/N query and Hkv/N KV heads (rows of
   q/k/v, columns of the attention output), its FFN/N rows of gate/up and
   columns of down, and its V/N rows of the output head. The persistent decode
   kernel adds the ranks' partial attention-output and down rows over NVLink
   in every rank's exchange region (one exchange per attention block and one
   per MLP block), every rank gets the whole logits vector and the same greedy
   token. Before the first step each rank exports its exchange region with
   fyb_plan_tp_handle, the handles of all ranks are gathered (in rank order)
   by the caller, and every rank passes them to fyb_plan_tp_connect. The ranks
   must then run the same steps (plan_token, plan_prefill, greedy decoding)
   together; a rank that stops makes the others fail their next step after a
   bounded wait. plan_read_kv declines (a rank holds only its KV heads). */
#define FYB_IPC_HANDLE_BYTES 64
/* rank and size of the plan's shard (size 1 without tensor parallelism). */
int fyb_plan_tp_info(const void *plan, unsigned *rank, unsigned *size);
/* this rank's exchange region handle (FYB_IPC_HANDLE_BYTES bytes). */
int fyb_plan_tp_handle(void *plan, void *handle, size_t bytes);
/* opens the other ranks' regions; handles = count (= size) handles in rank order. */
int fyb_plan_tp_connect(void *plan, const void *handles, size_t count);
/* marks a connected plan unconnected again, so plan_token, plan_prefill and
   the greedy loop return -1 without launching: what every rank does when
   another rank could not create its plan or open the regions. */
int fyb_plan_tp_disconnect(void *plan);
/* connects plans that live in this one process (one thread per GPU, or
   several shards on one GPU): plans[j] is rank j's plan, count = size; the
   regions are used through their device pointers (peer access is enabled
   between different devices) instead of IPC handles. Connects `plan` only;
   call it once per plan. 0, -1 invalid arguments, -2 peer access refused. */
int fyb_plan_tp_connect_local(void *plan, void *const *plans, size_t count);
/* the plan's device error word: 0 none, 1 a bounded wait ran out (a peer or
   a producer never arrived), 2 non-finite logits, 4 an index out of range;
   -1 for a NULL plan. A plan with a non-zero word has failed. */
int fyb_plan_error(const void *plan);

/* ---- synthetic GGUF-layout models (no reference counterpart) -------------
   Builds an in-memory model in the engine's own binding layout
   (backend/core/llm_gguf.c:1013-1118): LLaMA tensors, block formats as
   given, random contents drawn from a seeded counter-based generator. */
typedef struct fyb_synth_config {
    uint32_t layers, embedding, heads, kv_heads, feed_forward, vocabulary, context;
    uint32_t matrix_type;   /* type of q/k/v/o/gate/up/down */
    uint32_t embed_type;    /* token_embd */
    uint32_t output_type;   /* output */
    float rope_base, epsilon;
    uint64_t seed;
    int norm_mode;          /* 0: all ones, 1: N(1, 0.01), 2: N(0, 1) */
    int threads;            /* host threads for filling; 0 = all cores */
    int centered;           /* Q4_K only: choose each group's min so its mean
                               weight is near zero (mins then are not uniform) */
    const char *path;       /* null: private memory. Otherwise the tensor bytes
                               live in this file, mapped shared: the first
                               process to create it fills it, later ones (same
                               configuration) wait until it is complete and map
                               it read-only, so ranks on one host share one copy,
                               as processes mapping one GGUF file do. */
} fyb_synth_config;
nya_llm_context *fyb_synth_create(const fyb_synth_config *config);
void fyb_synth_free(nya_llm_context *model);
/* Fill `bytes` of one tensor the way fyb_synth_create does (type-aware
   values: uniform quants, |N(0,1)|*0.01 fp16 scales). */
void fyb_synth_fill(void *data, size_t rows, size_t columns, uint32_t type, uint64_t seed, uint64_t stream_id);

#ifdef __cplusplus
}
#endif
#endif
