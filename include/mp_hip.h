/*
 * mp_hip.h -- C ABI of the MI355X (gfx950) device backend for MiniPrefix's
 * FP32 generation path.
 *
 * The reference keeps its device forward inside CudaRunner
 * (miniprefix/src/backend/cuda/llama_runner.cu:51-186); the host side
 * (Engine, Scheduler, KVManager, ExactPrefixCache) talks to it only through
 * the ModelRunner virtual interface (miniprefix/include/miniprefix/model.h:35-58).
 * This header is the thin layer below a ModelRunner: weights resident in HBM,
 * paged K/V pools, device block tables, the copy-on-write tail copy and the
 * chunk forward. It has no C++, torch or HIP types in its signatures.
 *
 * Conventions:
 *  - every function returns 0 on success or a negative MP_* status; the
 *    message of the last failure on a context is mp_hip_last_error();
 *  - host pointers are borrowed for the duration of the call only;
 *  - every call that takes a context is synchronous (device work is complete
 *    when it returns) unless documented otherwise, matching the reference's
 *    synchronous append (llama_runner.cu:170);
 *  - a context is single-threaded, like the reference's KVManager
 *    (miniprefix/include/miniprefix/kv_manager.h:18-19).
 *
 * Arithmetic: in the exact mode every kernel reproduces the reference CPU
 * path's floating-point evaluation order (sequential-k projections with
 * separate multiply and add, sequential RMSNorm and softmax sums, two-pass
 * softmax, glibc-compatible expf, host-computed RoPE angles), so logits are
 * bit-identical to miniprefix/src/backend/cpu/llama_runner.cpp:60-104; the
 * fast mode trades that for matrix cores (MP_ARITHMETIC_FAST below).
 */
#ifndef MP_HIP_H
#define MP_HIP_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
    MP_OK = 0,
    MP_INVALID_ARGUMENT = -1, /* std::invalid_argument in the reference */
    MP_DEVICE_ERROR = -2,     /* runtime_error("what: "+error string), resources.cpp:6-8 */
    MP_OUT_OF_MEMORY = -3,
    MP_NONFINITE = -4         /* runtime_error("nonfinite ... logits"), llama_runner.cu:173 */
};

/* Arithmetic of a context (mp_model_desc.arithmetic):
 * - MP_ARITHMETIC_EXACT: every sum in the reference CPU path's order
 *   (sequential k, separate multiply and add, two-pass softmax): logits
 *   bit-identical to miniprefix/src/backend/cpu/llama_runner.cpp:60-104;
 * - MP_ARITHMETIC_FAST: projections and the LM head on FP32 matrix cores,
 *   decode attention split over the context (flash-decoding) and prefill
 *   attention on the matrix cores (flash attention), in their own summation
 *   order: logits within 1e-3 relative and decode attention within 1e-4
 *   absolute of the reference, greedy tokens checked against it. The
 *   attention paths need 16-token pages, 64-wide heads and at most 4 query
 *   heads per KV head (else they run the exact kernels). Needs hidden,
 *   intermediate, q+2*kv width and vocabulary multiples of 16, else the
 *   context computes exactly. */
enum { MP_ARITHMETIC_EXACT = 0, MP_ARITHMETIC_FAST = 1 };

/* Model shape; same fields and limits as ModelConfig (model.h:9-16,
 * model.cpp:9-15), plus the arithmetic mode (no counterpart in the reference). */
typedef struct mp_model_desc {
    int32_t layers, hidden, intermediate, heads, kv_heads, vocabulary, context;
    float rms_epsilon, rope_theta;
    int32_t tied;
    int32_t arithmetic;
} mp_model_desc;

/* Paged KV geometry (KvCacheConfig, paged_kv.h:13-17) plus the device block
 * table arena: max_sequences tables of max_sequence_blocks int32 entries
 * (KVManager::max_sequence_blocks, kv_manager.cpp:16-18). */
typedef struct mp_kv_desc {
    int32_t block_tokens, max_blocks, max_sequences, max_sequence_blocks;
} mp_kv_desc;

/* Strided tail region in float elements of ONE pool (K or V); rows are
 * layers (KVManager::TailCopyRegion, kv_manager.h:40-41). */
typedef struct mp_tail_region {
    uint64_t destination, source, pitch, width, rows;
} mp_tail_region;

/* One sequence's slice of a forward call: `count` new tokens starting at
 * committed position `used`, block table in arena slot `table_slot`. */
typedef struct mp_seq_step {
    int32_t table_slot, used, count;
} mp_seq_step;

typedef struct mp_hip_counters {
    uint64_t device_weight_bytes, weight_uploaded_bytes, token_uploaded_bytes;
    uint64_t kv_uploaded_bytes, logits_downloaded_bytes, device_allocations;
    uint64_t device_workspace_bytes, block_table_uploaded_bytes, block_table_device_bytes;
    uint64_t kv_pool_bytes, forward_calls, forward_rows, cow_copies, cow_bytes;
} mp_hip_counters;

typedef struct mp_hip mp_hip;

/* Replaces the CudaRunner constructor's device half (llama_runner.cu:78-87):
 * selects the current device, creates one stream, allocates the K and V pools
 * (max_blocks*layers*block_tokens*kv_width floats each, zeroed), the table
 * arena and the RoPE table for `context` positions. Weights follow with
 * mp_hip_upload_tensor. */
int mp_hip_create(const mp_model_desc* model, const mp_kv_desc* kv, mp_hip** out);
/* Synchronizes and frees everything (CudaRunner::~CudaRunner, :88). */
int mp_hip_destroy(mp_hip* h);
/* Message of the last failure on `h`; for h = NULL, of the last failed
 * context-free call (the stand-alone attention entry points) on this thread. */
const char* mp_hip_last_error(const mp_hip* h);

/* Tensor slots, canonical per-layer order. layer = -1 for the model-level
 * tensors. Data is FP32 in the reference's stored layout: projections
 * [in,out] row-major (model.cpp:33-37), embedding [vocab,hidden], norms
 * [hidden], untied head [hidden,vocab]. Replaces upload_parameter (:72-76). */
enum {
    MP_TENSOR_INPUT_NORM = 0, MP_TENSOR_Q, MP_TENSOR_K, MP_TENSOR_V, MP_TENSOR_O,
    MP_TENSOR_POST_NORM, MP_TENSOR_GATE, MP_TENSOR_UP, MP_TENSOR_DOWN,
    MP_TENSOR_EMBEDDING = 100, MP_TENSOR_FINAL_NORM = 101, MP_TENSOR_LM_HEAD = 102
};
int mp_hip_upload_tensor(mp_hip* h, int32_t layer, int32_t slot, const float* data, size_t count);
/* Reports whether every tensor the model needs has been uploaded. */
int mp_hip_ready(const mp_hip* h, int32_t* ready);

/* Writes table entries [first, first+count) of arena slot `slot`
 * (block-table H2D, llama_runner.cu:110-117,139-143). */
int mp_hip_table_write(mp_hip* h, int32_t slot, int32_t first, const int32_t* blocks, int32_t count);

/* Copy-on-write of a shared partial tail: copies the region in BOTH the K
 * and the V pool with one kernel (llama_runner.cu:130-137). The region must
 * be one KVManager forms: pitch = block_tokens*kv_width, rows = layers,
 * width = valid tokens * kv_width, source and destination page bases.
 * Inside a page the pools use the device order, and the copy moves the
 * valid tokens' K and V in that order (the same bytes the reference's 2-D
 * copy moves, counted the same way in the COW statistics). Other regions
 * are MP_INVALID_ARGUMENT. Queued: the copies queued since the last
 * forward run as one launch at the start of the next forward (or at
 * mp_hip_sync), before any kernel touches the pools; a copy that would read
 * or write a page a queued copy writes (or write a page one reads) first
 * flushes the queue, so the result is that of the calls in order. */
int mp_hip_copy_tail(mp_hip* h, const mp_tail_region* region);

/* Same copy, timed with device events around it (the reference's opt-in
 * COW timing, llama_runner.cu:129-138,171-172): flushes the queue first
 * (untimed), then launches and times this copy alone. Synchronous. */
int mp_hip_copy_tail_timed(mp_hip* h, const mp_tail_region* region, uint64_t* nanoseconds);

/* Chunk forward of `nseq` sequences (CpuRunner::append's device half,
 * llama_runner.cpp:70-102): embeds `tokens` (sum of counts, sequence-major),
 * runs every layer writing K/V at positions used..used+count-1 through each
 * sequence's table, and produces for each sequence the logits of its LAST
 * token. `logits` (nseq*vocab floats) may be NULL; `argmax` (nseq) receives
 * the first index of the maximum logit (std::max_element, engine.cpp:99);
 * `nonfinite` (nseq, may be NULL) receives 1 for a sequence with any
 * non-finite logit. Returns MP_NONFINITE if any produced logit is not
 * finite (llama_runner.cu:173); outputs are still written. Synchronous. */
int mp_hip_forward(mp_hip* h, const mp_seq_step* steps, int32_t nseq, const int32_t* tokens,
                   float* logits, int32_t* argmax, int32_t* nonfinite);

/* Stand-alone paged GQA decode attention on caller-owned DEVICE buffers
 * (the attention of llama_runner.cpp:85-93 for one query row of length
 * `length`). q: [heads*dim]; pools: [blocks][layers][block_tokens][kv_heads*dim];
 * table: device int32 page table; out: [heads*dim]. `stream` is a
 * hipStream_t or NULL for the null stream. Asynchronous. */
int mp_hip_paged_attention_decode(const float* q, const float* keys, const float* values,
                                  const int32_t* table, int32_t length, int32_t layer,
                                  int32_t layers, int32_t block_tokens, int32_t heads,
                                  int32_t kv_heads, int32_t dim, float* out, void* stream);

/* The decode attention of the fast arithmetic (MP_ARITHMETIC_FAST): the
 * kernels a fast-mode forward runs for its one-token rows, on caller-owned
 * DEVICE buffers, for `rows` query rows at once (the attention of
 * llama_runner.cpp:85-93 in the flash-decoding order: splits of
 * 16-256 tokens, each with a running maximum, denominator and weighted sum,
 * combined at the end; within 1e-4 absolute of the reference on its scale of
 * inputs). q: [rows][heads*dim]; out: [rows][heads*dim]; row r attends
 * lengths[r] tokens (host array) through its page table at
 * tables + r*table_stride (device int32). The pools hold the forward's
 * device page order (mp_hip_kv_pools; layout.h: per (block, layer) KV head
 * major, K as [d/4][slot][4], V as [slot/4][d][4]), not the reference's
 * [slot][kv_width]. Needs block_tokens 16, dim 64 and at most 4 query heads
 * per KV head, else MP_INVALID_ARGUMENT (message:
 * mp_hip_last_error(NULL)). Its work lists and partials come from memory that
 * the library keeps between calls (at most 256 MiB of device and as much of
 * pinned memory; destroying any context frees it). Synchronous on `stream`
 * (NULL: the null stream). */
int mp_hip_paged_attention_decode_fast(const float* q, const float* keys, const float* values,
                                       const int32_t* tables, int32_t table_stride, const int32_t* lengths,
                                       int32_t rows, int32_t layer, int32_t layers, int32_t block_tokens,
                                       int32_t heads, int32_t kv_heads, int32_t dim, float* out, void* stream);

/* The same attention as mp_hip_paged_attention_decode with no allocation of
 * any kind: no counterpart in the reference; for callers that cannot
 * allocate (code under HIP graph capture, serving loops that forbid
 * allocation). The scores of a long row (heads / kv_heads *
 * round_up(length, 16) > 10240) go to a 1 MiB device array of the library
 * (one per GPU, held until the process ends) instead of a per-call
 * hipMalloc; a row must satisfy heads * round_up(length, 16) <= 262144, or
 * the call returns MP_INVALID_ARGUMENT (message: mp_hip_last_error(NULL)).
 * Calls for long rows that overlap on one GPU share the array and race;
 * others may overlap. Asynchronous on `stream`. */
int mp_hip_paged_attention_decode_noalloc(const float* q, const float* keys, const float* values,
                                          const int32_t* table, int32_t length, int32_t layer,
                                          int32_t layers, int32_t block_tokens, int32_t heads,
                                          int32_t kv_heads, int32_t dim, float* out, void* stream);

/* ---- A paged K/V cache in 8 bits -----------------------------------------
 * (no counterpart in the reference, whose pools are FP32). Stand-alone like
 * the attention calls above: caller-owned DEVICE buffers, a caller's stream
 * (NULL: the null stream), asynchronous, no allocation, no state kept between
 * calls, lengths read on the device, so that a call can be captured into a
 * HIP graph and replayed with new lengths. Calls run on the stream's device.
 * Refusals are MP_INVALID_ARGUMENT with a message in mp_hip_last_error(NULL).
 *
 * Format. A page is block_tokens tokens (16, 32, 64 or 128) of one layer. Per
 * KV head it holds dim bytes a token (dim 64, 128 or 256) in each of `keys`
 * and `values`, [blocks][layers][kv_heads][block_tokens * dim], and in
 * `scales`, [blocks][layers][kv_heads][2], the scale of the head's keys and
 * that of its values. A byte b stands for scale * (b - 128) (MP_KV8_INT8; 0
 * is not written) or scale times the E4M3 number b (MP_KV8_E4M3: 448 largest,
 * 0x7F and 0xFF NaN). Scales are powers of two from 2^-126 on, so that raising
 * one moves codes without another rounding of the scale, and every value is
 * exact in FP32, BF16 and (in its range) FP16. A block takes less than 2 GiB
 * of keys. Order of a head's bytes: tiles
 * of 16 tokens; inside a tile keys are [dim/16][slot][16 dims], values
 * [dim/64][slot/4][dim%16][dim%64/16][slot%4]: the matrix cores' operands,
 * 16 bytes a lane. A block is contiguous in all three arrays: copying one on
 * write is three plain copies. keys and values are 16-byte aligned, scales
 * 8-byte.
 *
 * Rows. q, k, v and out are FP32, BF16 or FP16 (MP_TYPE_*), one row a token,
 * heads adjacent, `stride` elements from row to row (a fused q|k|v matrix is
 * three pointers with one stride); any alignment of their type, 16 bytes for
 * full speed. Rows are packed: sequence s has rows starts[s] ..
 * starts[s+1]-1 (device int32, sequences + 1 of them, not decreasing), at
 * positions used[s], used[s]+1, ... (device int32), and page table tables +
 * s*table_stride (device int32). Rows outside starts[0] .. starts[sequences]-1
 * are not touched. A sequence without rows is nothing. One with used[s]
 * outside 0 .. 2^30 has no tokens: append writes and read reads none of it (an
 * append's q_out has its queries, NaN where they are to turn). rows and
 * sequences are at most 2^20 each. Refused as too large for a launch: attention
 * of more than 2^22 rows times query heads; append and read of more than 2^21
 * pages times KV heads (2^22 with 32 tokens a page, 2^23 with 16), where every
 * sequence is taken to begin and end inside a page.
 *
 * What the device finds: a token whose page id is not in 0 .. blocks-1 or
 * whose page lies past table_stride is not written; an attention row that
 * needs such a page is NaN, as is one longer than max_length, one with a NaN
 * or an infinity in q, and one that sees a NaN key or scale; one that sees a
 * NaN among the value bytes is NaN in its dim. Rows that do not see them are
 * as without them. */
enum { MP_TYPE_F32 = 0, MP_TYPE_BF16 = 1, MP_TYPE_F16 = 2 };
enum { MP_KV8_INT8 = 0, MP_KV8_E4M3 = 1 };

typedef struct mp_kv8_cache {
    uint8_t* keys;
    uint8_t* values;
    float* scales;
    int32_t blocks, layers, block_tokens, kv_heads, dim, format;
} mp_kv8_cache;

/* Rotary positions: cos and sin of `positions` positions, device FP32
 * [positions][dims/2], whatever angles the model has (a context stretched by
 * interpolation is a matter of these tables). The first `dims` dims of every
 * head turn, the rest pass: pairs are (i, i + dims/2), or with `interleaved`
 * (2i, 2i + 1); a' = a cos - b sin, b' = b cos + a sin, each operation rounded
 * to FP32. dims is even; 0: no rotation, and the tables may be NULL. */
typedef struct mp_rope {
    const float* cos;
    const float* sin;
    int32_t positions, dims, interleaved;
} mp_rope;

/* Appends the rows' keys (rotated) and values to their pages of `layer`, and
 * writes the rotated queries to q_out (which may be q; q NULL: none; `heads`
 * query heads). Per page, head and kind: where the first new token takes slot
 * 0 the page starts anew; otherwise the slots before it are kept. The scale
 * is the smallest power of two that holds the new tokens, not smaller than
 * that of the kept ones; where it grows, the kept codes are rounded again
 * (nearest, ties to even, as are the new ones). Slots behind the last new
 * token keep their bytes. After a step that was taken back its positions are
 * simply appended again; a scale that the step had raised stays as it is.
 * A NaN or infinity in the new tokens makes the scale NaN, and with it the
 * head's keys (or values) of the page, until the page is written from slot 0.
 * Rows at or past rope->positions are not written (their slots keep what was
 * there), and their q_out is NaN. `rope` may be NULL. k and v must not overlap
 * the cache; sequences that write must not share the page that they write. */
int mp_hip_kv8_append(const mp_kv8_cache* cache, int32_t layer, const void* k, int64_t k_stride, const void* v,
                      int64_t v_stride, const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride,
                      int32_t heads, int32_t type, const mp_rope* rope, const int32_t* tables, int32_t table_stride,
                      const int32_t* starts, const int32_t* used, int32_t sequences, int32_t rows, void* stream);

/* Reads tokens back as rows of values: row i of sequence s is the token at
 * position used[s] + i - starts[s], as the pages hold it (rotated keys).
 * NaN for tokens without a valid page. Values outside the range of FP16 are
 * rounded as its conversion does. */
int mp_hip_kv8_read(const mp_kv8_cache* cache, int32_t layer, const int32_t* tables, int32_t table_stride,
                    const int32_t* starts, const int32_t* used, int32_t sequences, int32_t rows, int32_t type,
                    void* k, int64_t k_stride, void* v, int64_t v_stride, void* stream);

/* Bytes of workspace with which both attention calls below run `rows` rows of
 * `sequences` sequences (decode: as many as rows) of up to max_length tokens,
 * and any of fewer or shorter ones. 0 is possible, and then the pointer may be
 * NULL; else it is 16-byte aligned. A workspace holds nothing between calls;
 * calls that may overlap, replayed graphs among them, need workspaces of their
 * own. */
int mp_hip_kv8_attention_workspace(const mp_kv8_cache* cache, int32_t rows, int32_t sequences, int32_t heads,
                                   int32_t max_length, size_t* bytes);

/* Decode attention: row r, at position lengths[r] - 1, attends the
 * lengths[r] tokens of its page table tables + r*table_stride (device int32,
 * at most max_length): out = sum_t softmax_t(scale * q.k_t) v_t, query head h
 * on KV head h / (heads / kv_heads), at most 16 query heads per KV head. A
 * row of no tokens (length 0 or less) gives zeros. `scale` is finite (to
 * 2.3e38) and not negative. out may be q, with its stride; with another one
 * and more than one row the call is refused. The result, before it is rounded
 * to the rows' type, is off by about 1e-6 of the largest value that the row
 * sees, as FP32 sums are; pages whose value scale is more than 2^24 (INT8) or
 * 2^15 (E4M3) below that of such a page are held to 2^-31 of the largest
 * value. Pages that a row does not see do not touch this. */
int mp_hip_kv8_attention_decode(const mp_kv8_cache* cache, int32_t layer, const void* q, int64_t q_stride,
                                int32_t type, const int32_t* tables, int32_t table_stride, const int32_t* lengths,
                                int32_t rows, int32_t heads, int32_t max_length, float scale, void* out,
                                int64_t out_stride, void* workspace, size_t workspace_bytes, void* stream);

/* Prefill attention of packed rows, causal: the row at position p attends
 * tokens 0 .. p of its sequence, all of them in the pages already (append
 * first); used[s] + the rows of s is at most max_length. Any mix of counts,
 * single tokens among them. Rows of every type have the accuracy of FP32 sums,
 * as in decode, and are rounded once, to their type. out may be q, as there. */
int mp_hip_kv8_attention_prefill(const mp_kv8_cache* cache, int32_t layer, const void* q, int64_t q_stride,
                                 int32_t type, const int32_t* tables, int32_t table_stride, const int32_t* starts,
                                 const int32_t* used, int32_t sequences, int32_t rows, int32_t heads,
                                 int32_t max_length, float scale, void* out, int64_t out_stride, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* ---- Weights in 4 bits, rows in 8 bits ------------------------------------
 * (no counterpart in the reference, whose weights are FP32). What a model
 * needs around the 8-bit cache above: its weights packed to 4 bits, products
 * of rows with them, the norm between layers, and rows of 8 bits for prompts.
 * Stand-alone calls of the same manner: the caller's DEVICE buffers and stream
 * (NULL: the null stream), asynchronous, no allocation, no state kept between
 * calls, capturable into a HIP graph; on the stream's device. Refusals are
 * MP_INVALID_ARGUMENT with a message in mp_hip_last_error(NULL).
 *
 * Rows. FP32, BF16 or FP16 as above, any alignment of their type (16 bytes of
 * base and stride for full speed), or MP_TYPE_I8: a whole number, -127 to 127,
 * per element in `data`, `stride` bytes from row to row, times a power of two
 * per 32 elements, the byte b in `scales` for 2^(b - 127) (27 to 247; 255: NaN),
 * `scale_stride` bytes from row to row. 8-bit rows are whole groups of 32
 * elements; data and stride are 16-byte aligned, scales and their stride 4-byte
 * (the scales' rows are whole words, also the last, whose rest may be anything).
 * A group is written with the smallest power of two, from 2^-100 on, that holds
 * its largest magnitude, elements rounded to nearest, ties to even; a group with
 * a NaN, an infinity or a magnitude above 127 * 2^120 has the scale NaN. For
 * float rows scales and scale_stride are not looked at. At most 2^20 rows a call,
 * and rows, conversions and reads of at most 2^33 elements.
 *
 * Rows that a call writes may not overlap what it reads unless it says so.
 *
 * Matrices. `rows` (1 to 2^24) by `depth` (a multiple of 32 up to 2^20)
 * weights; each is an E2M1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6, or their
 * negatives) times a power of two per 32 weights along the row, chosen like
 * that of 8-bit rows (a magnitude above 6 * 2^120 makes it NaN). Codes lie by
 * tiles of 16 rows and 128 columns,
 * [rows/16][depth/128][column%128/32][row%16][16 bytes], even columns in the
 * low halves of the bytes, code 8 + c the negative of c; scale bytes as above (27
 * to 247; 255: NaN) are
 * [rows/16][depth/512][column%128/32][row%16][column%512/128]: the matrix cores'
 * operands. Tiles are whole, filled up with zeros. Both are 16-byte aligned and
 * of the sizes that mp_hip_w4_sizes says. */
enum { MP_TYPE_I8 = 3 };

typedef struct mp_rows {
    void* data;
    int64_t stride;
    uint8_t* scales;
    int64_t scale_stride;
    int32_t type;
} mp_rows;

typedef struct mp_w4_matrix {
    uint8_t* codes;
    uint8_t* scales;
    int32_t rows, depth;
} mp_w4_matrix;

int mp_hip_w4_sizes(int32_t rows, int32_t depth, size_t* code_bytes, size_t* scale_bytes);

/* Packs float rows into rows first .. first+rows-1 of a matrix (query, key and
 * value weights go into one matrix by three calls). The other rows stay as they
 * are; the call that packs the last row writes the zeros behind it. */
int mp_hip_w4_pack(const mp_w4_matrix* w, int32_t first, const mp_rows* x, int32_t rows, void* stream);

/* Rows ids[0 .. count-1] (device int32) of a matrix as float rows: an embedding
 * lookup in a 4-bit table. An id that is no row of the matrix gives NaN. */
int mp_hip_w4_read(const mp_w4_matrix* w, const int32_t* ids, int32_t count, const mp_rows* out, void* stream);

/* Rows of `width` elements from one type to another, float rows to 8 bits and
 * back among them. out may be x, as the same rows. */
int mp_hip_convert_rows(const mp_rows* x, int32_t rows, int32_t width, const mp_rows* out, void* stream);

/* Root-mean-square norm with the residual's addition: t = x + residual
 * (residual NULL: t = x), out = t * weight / sqrt(mean(t^2) + epsilon) per row of
 * `width` elements, and t itself to `sum` (NULL: not written; not without a
 * residual). x, residual and sum are float rows of one type, out rows of any,
 * weight FP32. Everything is computed in 64 bits and rounded once, out from the
 * exact t, not from the rounded sum. A row of zeros with epsilon 0 is NaN. sum
 * may be x or the residual, and out may be x, as the same rows. */
int mp_hip_rms_norm(const mp_rows* x, const mp_rows* residual, const mp_rows* sum, const float* weight, float epsilon,
                    int32_t rows, int32_t width, const mp_rows* out, void* stream);

/* Products: out[r][n] = sum_k x[r][k] w[n][k], or with a `gate` matrix of w's
 * size the gated pair g / (1 + exp(-g)) * u of g = x gate^T and u = x w^T. x and
 * out are rows of any type (8-bit results need w->rows to be a multiple of 32).
 * One to 2^20 rows: single tokens read the weights' 4 bits once, prompts are the
 * matrix cores' work. Rows and weights count as they are (an FP32 element below
 * 2^-110 without what of it lies below 2^-133), sums are FP32 (nothing below
 * 2^-149), and the result is rounded once, to out's type. A row with a NaN or an
 * infinity has no finite result, and a NaN scale of a matrix's row none in its
 * column; other rows and columns are as without them. Refused are products of more
 * than 2^22 tiles of 128 rows by 256 results (by 128 of a gated pair), and of more
 * than 2^22 blocks of 128 rows by 64 elements in 8 bits. The workspace (16-byte
 * aligned; mp_hip_w4_product_workspace says its size for the same or more rows; 0
 * is possible, and then it may be NULL) holds nothing between calls; calls that
 * may overlap, replayed graphs among them, need workspaces of their own. */
int mp_hip_w4_product_workspace(const mp_w4_matrix* w, int32_t type, int32_t rows, int32_t gated, size_t* bytes);
int mp_hip_w4_product(const mp_w4_matrix* w, const mp_w4_matrix* gate, const mp_rows* x, int32_t rows,
                      const mp_rows* out, void* workspace, size_t workspace_bytes, void* stream);

/* Applies queued table entries and copies, then waits for all work on the
 * context's stream (StreamBlas::synchronize). */
int mp_hip_sync(mp_hip* h);
int mp_hip_stats(const mp_hip* h, mp_hip_counters* out);

/* Device pointers of the K and V pools (for tests and profiling); their
 * contents include queued copies after mp_hip_sync. */
int mp_hip_kv_pools(const mp_hip* h, float** keys, float** values, size_t* elements);

/* The context's stream (hipStream_t), e.g. for recording events around calls. */
void* mp_hip_stream(const mp_hip* h);

/* Kernel timing of forward calls with HIP events on the context's stream
 * (instrumentation; no counterpart in the reference). `classes` is a mask of
 * MP_TIME_* bits; each enabled class brackets its launches with events and
 * accumulates their elapsed time when the forward call completes. Setting
 * the mask resets the totals. One ATTENTION launch is one layer's attention
 * (score, softmax and value kernels); one PROJECTION launch is one GEMM
 * (QKV, O, gate/up or down); one HEAD launch is final norm, LM head and
 * argmax of a call. Attention events ride on the kernel dispatches; the
 * others are stream markers between kernels. With MP_TIME_SAMPLED only one
 * layer per forward call is timed (layer = call count modulo layers), which
 * keeps the instrumentation's own cost out of a throughput measurement. */
enum { MP_TIME_ATTENTION = 1, MP_TIME_PROJECTION = 2, MP_TIME_HEAD = 4, MP_TIME_SAMPLED = 8 };
typedef struct mp_hip_timing_totals {
    uint64_t attention_ns, attention_launches;
    uint64_t projection_ns, projection_launches;
    uint64_t head_ns, head_launches;
} mp_hip_timing_totals;
int mp_hip_set_timing(mp_hip* h, uint32_t classes);
int mp_hip_kernel_times(const mp_hip* h, mp_hip_timing_totals* out);

/* Graph replay of fast-arithmetic decode steps (no counterpart in the
 * reference, which launches every kernel of every step): a decode step
 * (every sequence one token) of up to 16 sequences and of a shape seen in
 * the previous call -- the same number of sequences, logits wanted or not,
 * rows longer and shorter than 256 tokens present or not -- is captured
 * once as a HIP graph of its launches and replayed at later steps of that
 * shape, with the step's metadata uploaded before the replay; results are
 * bit-identical to direct launches. On by default; off while kernel timing
 * (mp_hip_set_timing) is on. mp_hip_set_graphs(h, 0) switches it off (and retires the graphs);
 * mp_hip_graphs_captured reports how many graphs the context holds. */
int mp_hip_set_graphs(mp_hip* h, int32_t enabled);
int mp_hip_graphs_captured(const mp_hip* h, int32_t* count);

#ifdef __cplusplus
}
#endif
#endif
