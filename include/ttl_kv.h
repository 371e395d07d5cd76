/*
 * ttl_kv.h -- C ABI of the paged key/value cache and its attention on the B200.
 *
 * ttl_attn (ttl_attn.h) keeps one contiguous f32 cache and takes one token of
 * one sequence per call, as tt-lab does (store_kv, src/model.cpp:247-253;
 * attention_from_cache, :255-290).  ttl_kv serves many sequences: K and V live
 * in pages of a pool, a batch brings any number of new rows per sequence (a
 * token, a chunk of a prompt, a whole prompt), and the cache may be held in
 * 4 bits.  The projections stay with the caller: the rows come in as Q, K, V.
 *
 * One step is: ttl_kv_batch_async (which rows belong to which sequence; once
 * per step, shared by all layers), then per layer ttl_kv_append_async (rotate,
 * store) and ttl_kv_attend_async.
 *
 * Conventions as in ttl_moe.h: TTL_OK or a negative status, messages from
 * ttl_kv_last_error (of the calling thread when the handle is NULL).  All
 * device memory is allocated in ttl_kv_create.  The _async calls take device
 * pointers of the handle's GPU, enqueue on the handle's stream, allocate
 * nothing, never wait, and may be captured into a CUDA graph (capture on the
 * handle's stream).  Calls on one handle, and graphs captured from them, share
 * the handle's plan and workspace: they must run one after another, never at
 * the same time on two streams.
 *
 * Graphs.  A graph that holds an append, read or attend without its batch call
 * uses the plan of the last batch call that ran on the device.  It reads as
 * many rows of its arrays as the batch had when it was captured; where the plan
 * has another number of rows, ttl_kv_sync reports it, and only the rows that
 * both have are stored or written (a call captured with no rows is not in the
 * graph).  Where an attend's plan asks for other kernels than the captured ones
 * (max_new and the number of sequences choose them), ttl_kv_sync reports it and
 * out is left as it was.  A batch call inside a capture sets the row count and
 * the kernels of the calls that follow it, captured or not, though the plan on
 * the device is still the earlier one until the graph runs.
 *
 * What only the device can see (row_start, length, page ids) is checked there:
 * a sequence with bad numbers is skipped (its rows are left as they were), a
 * page id outside the pool is skipped on append and read, and read as page 0
 * on attend; ttl_kv_sync then returns TTL_ERR_DEVICE with the reason, once.
 */
#ifndef TTL_KV_H
#define TTL_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ttl_kv ttl_kv;

enum {
    TTL_KV_F32 = 0,
    TTL_KV_F16 = 1,
    TTL_KV_BF16 = 2,
    TTL_KV_MXFP4 = 3 /* cache only: E2M1 codes, one E8M0 scale per 32 values of a head */
};

typedef struct {
    uint32_t layers;      /* 1..256 */
    uint32_t pages;       /* pages of the pool (per layer; a page id is good in every layer) */
    uint32_t page_tokens; /* 16, 32, 64 or 128 */
    uint32_t q_heads;     /* a multiple of kv_heads, at most 256 */
    uint32_t kv_heads;
    uint32_t head_dim;    /* 64 or 128 */
    uint32_t rows_type;   /* of q, k, v and out rows: TTL_KV_F32, _F16 or _BF16 */
    uint32_t cache_type;  /* rows_type or TTL_KV_MXFP4 */
    uint32_t max_seqs;    /* sequences of a batch, 1..4096 */
    uint32_t max_rows;    /* rows of a batch, 1..2^20 */
    uint32_t window;      /* positions a sliding call attends to (0: no sliding calls) */
    uint32_t rope_dims;   /* leading values of a head that are rotated: 0 or a multiple of 16 <= head_dim */
    uint32_t rope_interleaved; /* 0: pairs (i, i + rope_dims/2), as apply_rope (src/model.cpp:230-245); 1: (2i, 2i + 1) */
    const double *rope_freq;   /* host, rope_dims/2 values: radians per position of each pair */
    double rope_scale;         /* factor on cos and sin; 0 means 1 */
    int32_t device;            /* CUDA device ordinal, -1 = the calling thread's current device */
    void *stream;              /* cudaStream_t to enqueue on, NULL = own (cudaStreamLegacy for the default stream) */
} ttl_kv_config;

int ttl_kv_create(const ttl_kv_config *config, ttl_kv **handle_out);
void ttl_kv_destroy(ttl_kv *handle);
const char *ttl_kv_last_error(const ttl_kv *handle);

/* Device bytes one page takes in one layer. */
size_t ttl_kv_page_bytes(const ttl_kv *handle);

/* The batch: `seqs` sequences and `rows` rows in all.  Device arrays:
 *   row_start [seqs + 1]  rows [row_start[s], row_start[s+1]) are sequence s's
 *                         new tokens, in order (none, one or many); rows past
 *                         row_start[seqs] are padding and left as they were
 *   length    [seqs]      tokens of sequence s including its new rows, at most
 *                         2^29 - 128: the rows' positions are length - new ..
 *                         length - 1
 *   pages     [seqs][page_stride]  page ids: position p is in slot
 *                         p % page_tokens of page pages[s][p / page_tokens].
 *                         Sequences may share pages that they only read.
 *                         Entries of pages that no call reaches (an attend those
 *                         whose positions no row sees, an append or read those
 *                         without rows) may hold anything, -1 for instance
 *   first     [rows] or NULL  lowest position a row may see (a packed
 *                         document's start)
 *   prefix    [seqs] or NULL  every row sees all positions below prefix
 * Row i at position p sees positions max(first, p - window + 1 if sliding) ..
 * max(p, prefix - 1).  max_new is an upper bound on the new rows of any one
 * sequence (it selects the kernels); a sequence above it is an error.
 * row_start, length, first and prefix are read by this call's kernel, pages
 * by every later append, read and attend: keep it until the next batch. */
int ttl_kv_batch_async(ttl_kv *handle, uint32_t seqs, uint32_t rows, uint32_t max_new, const int32_t *row_start,
                       const int32_t *length, const int32_t *pages, uint32_t page_stride, const int32_t *first,
                       const int32_t *prefix);

/* Stores K and V [rows][kv_heads][head_dim] of the batch's rows in layer
 * `layer`, K rotated by its position (rotate != 0), and writes Q
 * [rows][q_heads][head_dim], rotated, to q_out (q and q_out NULL: no Q;
 * q_out == q with the same stride rotates in place).  Strides are elements
 * between rows; base pointers and strides are multiples of 16 bytes.  What a
 * call writes must not overlap the rows that it reads, nor one output another
 * (views of one array with one stride may lie side by side).  With a
 * 4-bit cache a block's scale is 2^(floor(log2 max|x|) - 2), codes round to
 * nearest, ties to even; a block that holds an infinity or NaN becomes NaN.
 * Two rows must not share a slot. */
int ttl_kv_append_async(ttl_kv *handle, int layer, int rotate, const void *k, size_t k_stride, const void *v,
                        size_t v_stride, const void *q, size_t q_stride, void *q_out, size_t q_out_stride);

/* The batch's rows as the cache holds them: K and V [rows][kv_heads][head_dim]
 * in rows_type (a batch whose rows are a whole sequence reads it back). */
int ttl_kv_read_async(ttl_kv *handle, int layer, void *k, size_t k_stride, void *v, size_t v_stride);

#define TTL_KV_SLIDING 1u /* flags: the layer attends to the window only */

/* out [rows][q_heads][head_dim] = attention of Q over layer `layer`'s cache:
 *   score = q.k * scale            (scale 0: 1 / sqrt(head_dim))
 *   cap > 0: score = cap * tanh(score / cap)
 *   slopes (device f32 [q_heads] or NULL): score -= slope * |p - j|
 *   softmax over the visible j and, with sinks (device f32 [q_heads] or NULL),
 *   the head's sink, which adds to the sum and has no value row
 * A row that sees nothing is zero.  Values of positions a row does not see
 * never reach it, infinities and NaN included.  f16 and bf16 rows: products
 * on the tensor cores, sums in 32 bits (over n keys of one CTA's part good to
 * n * 2^-24 of their size), weights rounded to the rows' type.  Over
 * a 4-bit cache they are rounded to f16 where few rows of a sequence are new and
 * to bf16 in bf16 prompts, so a row's last bits may depend on the batch that it
 * is in; of the cache's values, those below 2^-124 may count as zero.  A column
 * that meets an infinity or NaN in a place that it does not see (but for slots
 * behind the sequence's end, which cost nothing) or sees one is computed again
 * in 32-bit arithmetic, which takes up to 300 times as long. */
int ttl_kv_attend_async(ttl_kv *handle, int layer, uint32_t flags, const void *q, size_t q_stride, void *out,
                        size_t out_stride, float scale, float cap, const float *sinks, const float *slopes);

/* Waits for the handle's stream, then reports and clears the device status. */
int ttl_kv_sync(ttl_kv *handle);
void *ttl_kv_stream(ttl_kv *handle);

#ifdef __cplusplus
}
#endif

#endif
